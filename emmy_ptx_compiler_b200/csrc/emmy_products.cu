// Matrix products whose sizes are known only on the device, and products of
// 8-bit integers (C ABI: include/emmy_b200.h):
//
//   emmy_grouped_matmul     out[r, :]  = x[r, :] W_e^T            (r in group e)
//   emmy_grouped_matmul_dw  dw[e]      = dy_e^T x_e
//   emmy_int8_matmul        out[r, n]  = (xq[r, :] . wq[e, n, :]) x_scale[r] w_scale[e, n] + bias[e, n]
//   emmy_quantize_rows      scale = max |x| / 127,  q = round(x / scale)
//
// Every product is one form:  out(c, m) = sum_k A(m, k) B(c, k), where m runs along the output's
// contiguous axis and c along its rows:
//
//   forward  A = W_e (m: channels),       B = x   (c: rows of the group, ragged), k: channels
//   dw       A = x_e (m: input channels), B = dy  (c: output channels),           k: rows, ragged
//
// The group boundaries are read on the device; a launch covers any of them, so no call waits for
// the host and a recorded graph follows new boundaries.  Sums of 16-bit products are held in f32 and
// rounded once, to the output's type; tensor cores truncate where they align addends, so long sums are
// joined from segments.  Sums of 8-bit products are exact in s32; scaling rounds them to f32 (a 24-bit significand, for sums beyond 2^24),
// then once for each scale, the bias and the output's type.

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <cstdarg>
#include <cstdio>

#include "emmy_b200.h"
#include "emmy_launch_record.h"

extern "C" int emmy_record_error(int code, const char *msg);  // emmy_runtime.cpp (not exported)

// Status bits of this file's kernels, one word for each device; private to this file.
static __device__ unsigned int emmy_status = 0u;
#define EMMY_STATUS_DEFINED

#include "emmy_products_dev.cuh"
#include "emmy_products_tc.cuh"

namespace {

// ---------------------------------------------------------------- row quantization
//
// Reads a row once: its values wait in registers while the block agrees on their largest
// magnitude.  Bound by memory (k values read, k bytes written), as long as a value costs few
// instructions, so nothing is converted to or from integers one by one:
//
// * the largest magnitude is a maximum of sign-less bit patterns, which order like the values
//   and put infinities and NaN on top;
// * fma(x, 1 / s, 1.5 * 2^23) rounds the exact product to an integer, ties to even, and leaves
//   that integer in the low byte of the result's bits;
// * 1 / s is off by half a step, so below 128 the product is off by less than 1e-5 and decides
//   every quotient but those that close to a half (16-bit rows meet exact halves often: a row whose
//   peak is a power of two has one in a few hundred values).  For these the residual x - q s tells:
//   it is a multiple of half a step of s and at most about s / 2, so the FMA that computes it is
//   exact, and comparing it with s / 2 settles the side and the ties.
//
// 16381 x 8192 f32 rows take 107 us (6.2 TB/s), 16-bit rows 72 to 82 us (4.9 to 5.6 TB/s), which issue
// instructions in 7 of 10 cycles: the more of their quotients lie near a half, the longer (rows of small
// integers, where most packs hold one, 100 us).  One row takes 2 us.

constexpr float kRoundMagic = 12582912.0f;  // 1.5 * 2^23
constexpr float kNearHalf = 0.49999f;  // below: off by less than 127.5 * 2^-24 = 7.6e-6

// x / s to the nearest integer, exact ties to even, for the quotient of the two f32 values.
__device__ __noinline__ int quantize_exact(float x, float s, float inv) {
    const float q = fmaf(x, inv, kRoundMagic) - kRoundMagic;
    const float d = fmaf(x, inv, -q);
    float r = q;
    if (fabsf(d) > kNearHalf) {
        const float step = d > 0.0f ? 1.0f : -1.0f;
        const float past = fmaf(-(q + 0.5f * step), s, x) * step;  // > 0: beyond the half, away from q
        if (past > 0.0f || (past == 0.0f && (static_cast<int>(q) & 1))) r = q + step;
    }
    return static_cast<int>(fminf(fmaxf(r, -127.0f), 127.0f));
}

template <typename T>
struct Bits;
template <>
struct Bits<float> {
    using U = uint32_t;
    static constexpr uint32_t kInf = 0x7f800000u, kAbs = 0x7fffffffu;
    static __device__ __forceinline__ float value(uint32_t u) { return __uint_as_float(u); }
};
template <>
struct Bits<__nv_bfloat16> {
    using U = uint16_t;
    static constexpr uint32_t kInf = 0x7f80u, kAbs = 0x7fffu;
    static __device__ __forceinline__ float value(uint32_t u) { return __uint_as_float(u << 16); }
};
template <>
struct Bits<__half> {
    using U = uint16_t;
    static constexpr uint32_t kInf = 0x7c00u, kAbs = 0x7fffu;
    static __device__ __forceinline__ float value(uint32_t u) {
        return __half2float(__ushort_as_half(static_cast<unsigned short>(u)));
    }
};

// VEC values as they are loaded: 16 bytes, or a single value where rows are not aligned to that.
template <typename T, int VEC>
struct Pack {
    using U = typename Bits<T>::U;
    U v[VEC];
    __device__ __forceinline__ void load(const T *p) {
        if constexpr (VEC == 1) v[0] = *reinterpret_cast<const U *>(p);
        else *reinterpret_cast<uint4 *>(v) = __ldcs(reinterpret_cast<const uint4 *>(p));
    }
    __device__ __forceinline__ uint32_t peak() const {
        uint32_t m = 0;
        if constexpr (VEC == 8) {
            uint32_t m2 = 0;
            #pragma unroll
            for (int i = 0; i < 4; ++i) m2 = __vmaxu2(m2, reinterpret_cast<const uint32_t *>(v)[i] & 0x7fff7fffu);
            m = max(m2 & 0xffffu, m2 >> 16);
        } else {
            #pragma unroll
            for (int i = 0; i < VEC; ++i) m = max(m, static_cast<uint32_t>(v[i]) & Bits<T>::kAbs);
        }
        return m;
    }
    // exact: every value goes the long way (a scale so small that its reciprocal needs lifting)
    __device__ __forceinline__ void store(int8_t *q, float s, float inv, float lift, bool zero, bool exact) const {
        uint32_t r[VEC];
        float rest[VEC], near = 0.0f;
        #pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const float x = Bits<T>::value(v[i]), f = fmaf(x, inv, kRoundMagic);
            r[i] = __float_as_uint(f);
            rest[i] = fmaf(kRoundMagic - f, s, x);
            near = fmaxf(near, fabsf(rest[i]));
        }
        if (exact) {
            #pragma unroll
            for (int i = 0; i < VEC; ++i) r[i] = static_cast<uint32_t>(quantize_exact(Bits<T>::value(v[i]) * lift, s, inv));
        } else if (near > kNearHalf * s) {
            const uint32_t half = __float_as_uint(0.5f * s);
            #pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const uint32_t bits = __float_as_uint(rest[i]);
                // beyond the half, or on it beside an odd integer: one further
                if ((bits & 0x7fffffffu) + (r[i] & 1u) > half) r[i] += 1u | static_cast<uint32_t>(static_cast<int>(bits) >> 31);
            }
        }
        if constexpr (VEC == 1) {
            *q = zero ? 0 : static_cast<int8_t>(r[0]);
        } else {
            uint32_t w[VEC / 4];
            #pragma unroll
            for (int i = 0; i < VEC / 4; ++i)
                w[i] = zero ? 0u
                            : __byte_perm(__byte_perm(r[4 * i], r[4 * i + 1], 0x0040),
                                          __byte_perm(r[4 * i + 2], r[4 * i + 3], 0x0040), 0x5410);
            if constexpr (VEC == 8) *reinterpret_cast<uint2 *>(q) = make_uint2(w[0], w[1]);
            else *reinterpret_cast<uint32_t *>(q) = w[0];
        }
    }
};

// GROUP threads for each row, PER packs of it in each thread's registers; what a longer row has
// beyond them is read again from L2.
template <typename T, int VEC, int GROUP, int PER>
__global__ void __launch_bounds__(GROUP == 32 ? 256 : GROUP) quantize_rows_kernel(const T *__restrict__ x, int64_t x_stride,
                                                            int8_t *__restrict__ q, int64_t q_stride,
                                                            float *__restrict__ scale, int64_t rows, int64_t k) {
    constexpr int THREADS = GROUP == 32 ? 256 : GROUP;
    const int tid = threadIdx.x % GROUP;
    const int64_t r = static_cast<int64_t>(blockIdx.x) * (THREADS / GROUP) + threadIdx.x / GROUP;
    const bool live = r < rows;
    emmy::wait_for_prior_grid();
    emmy::let_next_grid_start();
    const T *xr = x + (live ? r : 0) * x_stride;
    const int64_t packs = live ? k / VEC : 0;
    Pack<T, VEC> held[PER];
    uint32_t peak = 0;
    #pragma unroll
    for (int i = 0; i < PER; ++i)
        if (tid + i * GROUP < packs) held[i].load(xr + (tid + i * GROUP) * static_cast<int64_t>(VEC));
    #pragma unroll
    for (int i = 0; i < PER; ++i)
        if (tid + i * GROUP < packs) peak = max(peak, held[i].peak());
    for (int64_t i = tid + PER * GROUP; i < packs; i += GROUP) {
        Pack<T, VEC> more;
        more.load(xr + i * VEC);
        peak = max(peak, more.peak());
    }
    peak = __reduce_max_sync(0xffffffffu, peak);
    if constexpr (GROUP > 32) {
        __shared__ uint32_t s_peak[GROUP / 32];
        if ((threadIdx.x & 31) == 0) s_peak[threadIdx.x >> 5] = peak;
        __syncthreads();
        peak = __reduce_max_sync(0xffffffffu, s_peak[threadIdx.x % (GROUP / 32)]);
    }
    if (!live) return;
    const bool bad = peak >= Bits<T>::kInf;
    const float s = __fdiv_rn(Bits<T>::value(peak), 127.0f);
    const bool tiny = s < 1e-30f;  // lifted by a power of two, with its row, before the reciprocal
    const float lift = tiny ? 0x1p64f : 1.0f, ls = s * lift, inv = 1.0f / ls;
    const bool zero = bad || s == 0.0f;
    if (tid == 0) scale[r] = bad ? __int_as_float(0x7fffffff) : s;
    int8_t *qr = q + r * q_stride;
    #pragma unroll
    for (int i = 0; i < PER; ++i)
        if (tid + i * GROUP < packs)
            held[i].store(qr + (tid + i * GROUP) * static_cast<int64_t>(VEC), ls, inv, lift, zero, tiny);
    for (int64_t i = tid + PER * GROUP; i < packs; i += GROUP) {
        Pack<T, VEC> more;
        more.load(xr + i * VEC);
        more.store(qr + i * VEC, ls, inv, lift, zero, tiny);
    }
}

// ---------------------------------------------------------------- host side

int report(int code, const char *fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    return emmy_record_error(code, buf);
}

// The call's device, made current for the launch and put back afterwards.  It is set even where it
// is the thread's device already: a thread that has not used it yet has no context, which encoding
// a tensor map needs.
struct DeviceScope {
    int prev = -1;
    cudaError_t err;
    explicit DeviceScope(int dev) {
        err = cudaGetDevice(&prev);
        if (err == cudaSuccess) err = cudaSetDevice(dev);
        if (prev == dev) prev = -1;
    }
    ~DeviceScope() {
        if (prev >= 0) cudaSetDevice(prev);
    }
};

constexpr int64_t kMaxExtent = (1ll << 31) - 1024;  // 32-bit extents, with room to round them up to tiles
constexpr int64_t kMaxTiles = 1ll << 30;

bool bad_extent(int64_t v) { return v < 0 || v > kMaxExtent; }

// ---- tensor maps

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                  const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_tiled() {
    static const EncodeTiledFn fn = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            f = nullptr;
        return reinterpret_cast<EncodeTiledFn>(f);
    }();
    return fn;
}

// An operand as TMA sees it: `inner` contiguous values, then one or two strided extents (elements).
struct Operand {
    const void *base;
    int64_t inner, rows, row_stride, mats, mat_stride;
};

// TMA takes 16-byte aligned bases and strides; where an extent is 1 its stride is free, so any
// valid one stands in for it.
bool tma_ready(Operand &o, int esize) {
    if (o.inner < 1 || o.rows < 1 || o.mats < 1) return false;
    const int64_t unit = 16 / esize;
    if (o.rows == 1) o.row_stride = (o.inner + unit - 1) / unit * unit;
    if (o.mats == 1) o.mat_stride = (o.rows * o.row_stride + unit - 1) / unit * unit;
    return reinterpret_cast<uintptr_t>(o.base) % 16 == 0 && o.row_stride % unit == 0 && o.mat_stride % unit == 0 &&
           o.row_stride >= o.inner && o.mat_stride > 0 && o.row_stride * esize < (1ll << 40) &&
           o.mat_stride * esize < (1ll << 40);
}

bool encode(CUtensorMap *map, const Operand &o, CUtensorMapDataType type, int esize, int rank, uint32_t box_inner,
            uint32_t box_rows) {
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(o.inner), static_cast<cuuint64_t>(o.rows),
                                static_cast<cuuint64_t>(o.mats)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(o.row_stride) * esize,
                                   static_cast<cuuint64_t>(o.mat_stride) * esize};
    const cuuint32_t box[3] = {box_inner, box_rows, 1}, step[3] = {1, 1, 1};
    return encode_tiled()(map, type, rank, const_cast<void *>(o.base), dims, strides, box, step,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// ---- launches

constexpr int kSms = 148;

struct Call {
    const char *name;
    int dev;
    cudaStream_t stream;
};

int launched(const Call &call, cudaError_t err) {
    if (err == cudaSuccess) return EMMY_OK;
    cudaGetLastError();  // the launch's own error does not stay behind for the caller's next check
    return report(EMMY_ERR_CUDA, "%s: launch: %s", call.name, cudaGetErrorString(err));
}

cudaLaunchConfig_t config(const Call &call, int64_t blocks, int threads, uint32_t smem) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(blocks));
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = call.stream;
    return cfg;
}

// The kernel may be set up while the one before it on the stream still runs.  Every kernel here
// waits for that one's end before it touches a buffer, so the order on the stream holds.
cudaLaunchAttribute early_start() {
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    return attr;
}

using TcKernel = void (*)(Product, Flags, CUtensorMap, CUtensorMap);

// What every variant's launch takes.
struct Launch {
    const Call &call;
    const Product &p;
    Flags flags;
    const CUtensorMap &ta, &tb;
    int64_t clusters;
    int cluster;
};

// `ready` marks the devices on which the kernel's shared-memory limit has been raised.
int launch_clusters(const Launch &l, TcKernel kernel, std::atomic<uint64_t> &ready, int threads, uint32_t smem) {
    if (!(ready.load(std::memory_order_acquire) >> l.call.dev & 1)) {
        const cudaError_t err =
            cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
        if (err != cudaSuccess) return launched(l.call, err);
        ready.fetch_or(1ull << l.call.dev, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg = config(l.call, l.clusters * l.cluster, threads, smem);
    cudaLaunchAttribute attrs[2] = {early_start(), {}};
    attrs[1].id = cudaLaunchAttributeClusterDimension;
    attrs[1].val.clusterDim = {static_cast<unsigned>(l.cluster), 1, 1};
    cfg.attrs = attrs;
    cfg.numAttrs = 2;
    return launched(l.call, cudaLaunchKernelEx(&cfg, kernel, l.p, l.flags, l.ta, l.tb));
}

template <bool I8, int LAYOUT, int BN, bool TMA, bool JOIN>
int launch_single(const Launch &l) {
    using Cfg = TcConfig<I8, BN, TMA>;
    static std::atomic<uint64_t> ready{0};
    return launch_clusters(l, product_tc_kernel<I8, LAYOUT, BN, TMA, JOIN>, ready, Cfg::kThreads, Cfg::kSmem);
}

template <bool I8, int LAYOUT, int BN, bool JOIN>
int launch_pair(const Launch &l) {
    using Cfg = PairConfig<BN>;
    static std::atomic<uint64_t> ready{0}, ready_direct{0};
    if constexpr (JOIN && BN == 256)
        if (l.p.out_type == EMMY_F32)
            return launch_clusters(l, product_pair_kernel<I8, LAYOUT, BN, JOIN, true>, ready_direct,
                                   Cfg::kThreads + (LAYOUT == kMM ? Cfg::kTailThreads : 0), Cfg::kSmem);
    return launch_clusters(l, product_pair_kernel<I8, LAYOUT, BN, JOIN>, ready,
                           Cfg::kThreads + (LAYOUT == kMM ? Cfg::kTailThreads : 0), Cfg::kSmem);
}

template <bool I8, int LAYOUT, bool JOIN>
int launch_variant(const Launch &l, bool tma, int pair, int bn) {
    if (pair) return pair == 256 ? launch_pair<I8, LAYOUT, 256, JOIN>(l) : launch_pair<I8, LAYOUT, 128, JOIN>(l);
    if constexpr (LAYOUT == kMM) {
        return tma ? launch_single<I8, LAYOUT, 128, true, JOIN>(l) : launch_single<I8, LAYOUT, 128, false, JOIN>(l);
    } else {
        if (!tma)
            return bn == 32   ? launch_single<I8, LAYOUT, 32, false, JOIN>(l)
                   : bn == 64 ? launch_single<I8, LAYOUT, 64, false, JOIN>(l)
                              : launch_single<I8, LAYOUT, 128, false, JOIN>(l);
        switch (bn) {
            case 16: return launch_single<I8, LAYOUT, 16, true, JOIN>(l);
            case 32: return launch_single<I8, LAYOUT, 32, true, JOIN>(l);
            case 64: return launch_single<I8, LAYOUT, 64, true, JOIN>(l);
            default: return launch_single<I8, LAYOUT, 128, true, JOIN>(l);
        }
    }
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Behind the last value of an operand.
const void *end_of(const Operand &o, int esize) {
    if (o.inner < 1 || o.rows < 1 || o.mats < 1) return o.base;
    const int64_t last = (o.mats - 1) * o.mat_stride + (o.rows - 1) * o.row_stride + o.inner;
    return static_cast<const uint8_t *>(o.base) + last * esize;
}

// The kernel that a product runs on.
struct Variant {
    int pair = 0;      // 256 or 128: pairs of CTAs on tiles of as many output rows
    int bn = 0;        // output rows of a tile
    int split = 1;     // CTAs that divide a sum
    int64_t clusters = 0;  // of the launch
};

// Chooses it by the extents, the operands' size and whether TMA can take both of them (`tma`); false where
// the output has more tiles than are supported.
bool choose(const Product &p, int esize, bool tma, Variant &v) {
    // groups that can hold rows, and the rows of an even one
    const int64_t groups = p.experts < p.rows ? p.experts : (p.rows ? p.rows : 1), bk = 128 / esize;
    const int64_t even = ceil_div(p.rows, groups), kblocks = ceil_div(p.dw ? even : p.k, bk);
    // tiles of even groups, and the most that any grouping can have
    auto tiles = [&](int64_t tm, int64_t tc) {
        return ceil_div(p.m, tm) * (p.dw ? p.experts * ceil_div(p.c, tc) : groups * ceil_div(even, tc));
    };
    auto most = [&](int64_t tm, int64_t tc) {
        return ceil_div(p.m, tm) * (p.dw ? p.experts * ceil_div(p.c, tc) : p.rows / tc + groups);
    };
    if (most(kTileM, p.dw ? 64 : 16) > kMaxTiles) return false;
    const int64_t cext = p.dw ? p.c : even;
    // Pairs of CTAs where groups have rows for them and there are tiles enough, and, for dw, where the
    // sums are long enough to cover a wide tile's way out (32 experts, dw [512, 1024]: 256 rows each 22
    // against a single CTA's 19 us, 1000 rows each of 16 [1024, 1024] 36 against 47 us).
    if (tma && p.m > 128 && cext > 64 && !(p.dw && kblocks < 8)) {
        if (cext > 128 && tiles(256, 256) >= kSms / 4) v.pair = 256;
        else if (tiles(256, 128) >= kSms / 4) v.pair = 128;
    }
    // Output rows of a single CTA's tile: a few more than an even group has, so that an uneven one
    // still fits; 64 until there are tiles for every SM (300 rows, [512, 1024]: 7.5 against 8.3 us at 128).
    v.bn = 128;
    if (v.pair) v.bn = v.pair;
    else if (!p.dw && !tma) {
        // What a block costs the warps that cut it, relative to 128 wide: 0.63 and 0.48 (8787 rows, int8
        // [639, 809]: 3 waves of tiles 128 wide in 68 us, 5 of 64 in 71, 10 of 32 in 108; 1022 rows, 8
        // experts [777, 1001]: one wave of 128 in 50, one of 64 in 38, two of 32 in 52).
        const struct { int bn; double cost; } widths[] = {{128, 1.0}, {64, 0.63}, {32, 0.48}};
        double best = 1e300;
        for (const auto &w : widths) {
            const double cost = static_cast<double>(ceil_div(tiles(kTileM, w.bn), kSms)) * w.cost;
            if (cost < best) best = cost, v.bn = w.bn;
        }
    }
    else if (!p.dw) v.bn = even <= 12 ? 16 : even <= 24 ? 32 : even <= 48 || tiles(kTileM, 128) <= kSms ? 64 : 128;
    // CTAs that run at once: clusters of 4 and 8 leave some of a GPC's SMs over
    auto resident = [&](int cluster) {
        const int per_sm = !v.pair && tma && v.bn <= 32 ? 2 : 1;
        return per_sm * (cluster <= 2 ? kSms : cluster == 4 ? 132 : 120);
    };
    // Idle SMs take parts of the sums, as long as a part is worth the exchange: 4 blocks of it for
    // the few columns of a narrow tile, 8 (of 32 or more) and 16 for wider ones (1022 rows, 8 experts, dx
    // [1000, 776], 13 blocks at 128 wide: 11 us whole, 18 in halves; 90 rows, [768, 8192]: 11 us in
    // eighths, 13 in quarters; 60000 rows, dw [256, 256]: 275 us whole, 42 in eighths).
    const int64_t part = v.bn <= 32 ? 4 : v.bn == 64 ? 8 : 16;
    if (!v.pair && (v.bn != 64 || kblocks >= 32))
        while (v.split < 8 && tiles(kTileM, v.bn) * v.split * 2 <= resident(v.split * 2) && kblocks >= v.split * 2 * part)
            v.split *= 2;
    const int cluster = v.pair ? 2 : v.split;
    v.clusters = v.pair ? most(2 * kTileM, v.pair) : most(kTileM, v.bn);
    if (v.clusters > resident(cluster) / cluster) v.clusters = resident(cluster) / cluster;
    return true;
}

template <bool I8>
int launch_product(const Call &call, Product p, bool bf16) {
    constexpr int esize = I8 ? 1 : 2, bk = 128 / esize;
    const bool a_mn = p.dw || p.a_k != 1;
    Operand a{p.a, 0, 0, 0, 1, 0}, b{p.b, 0, 0, 0, 1, 0};
    if (p.dw) {
        a.inner = p.m, a.rows = p.rows, a.row_stride = p.a_k;
        b.inner = p.c, b.rows = p.rows, b.row_stride = p.b_k;
    } else {
        a.inner = a_mn ? p.m : p.k, a.rows = a_mn ? p.k : p.m, a.row_stride = a_mn ? p.a_k : p.a_m;
        a.mats = p.experts, a.mat_stride = p.a_e;
        b.inner = p.k, b.rows = p.rows, b.row_stride = p.b_c;
    }
    p.a_end = end_of(a, esize);
    p.b_end = end_of(b, esize);
    const Flags flags{bf16, encode_tiled() && tma_ready(a, esize), encode_tiled() && tma_ready(b, esize)};
    const bool tma = flags.tma_a && flags.tma_b;
    Variant v;
    if (!choose(p, esize, tma, v))
        return report(EMMY_ERR_INVALID, "%s: an output of more than 2^30 tiles is not supported", call.name);
    CUtensorMap ta{}, tb{};
    const CUtensorMapDataType type = I8     ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                     : bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                            : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    if ((flags.tma_a && !encode(&ta, a, type, esize, 3, bk, a_mn ? 64 : kTileM)) ||
        (flags.tma_b && !encode(&tb, b, type, esize, 2, bk, p.dw ? 64 : v.pair ? v.pair / 2 : v.bn)))
        return report(EMMY_ERR_CUDA, "%s: cuTensorMapEncodeTiled failed", call.name);
    const Launch l{call, p, flags, ta, tb, v.clusters, v.pair ? 2 : v.split};
    if constexpr (I8) {
        return launch_variant<true, kKK, false>(l, tma, v.pair, v.bn);
    } else {
        // the longest sum that a CTA may have
        const bool join = ceil_div(ceil_div(p.dw ? p.rows : p.k, bk), v.split) > segment_blocks(p.out_type);
        auto go = [&](auto kernels) {
            constexpr bool JOIN = decltype(kernels)::value;
            return p.dw ? launch_variant<false, kMM, JOIN>(l, tma, v.pair, v.bn)
                   : a_mn ? launch_variant<false, kMK, JOIN>(l, tma, v.pair, v.bn)
                          : launch_variant<false, kKK, JOIN>(l, tma, v.pair, v.bn);
        };
        return join ? go(std::true_type{}) : go(std::false_type{});
    }
}

bool no_output(const Product &p) { return p.m == 0 || p.experts == 0 || (p.dw ? p.c : p.rows) == 0; }

int run_product(const char *name, int dev, int operands, const Product &p, uint64_t stream) {
    if (no_output(p)) return EMMY_OK;
    DeviceScope scope(dev);
    if (scope.err != cudaSuccess)
        return report(EMMY_ERR_CUDA, "%s: device %d: %s", name, dev, cudaGetErrorString(scope.err));
    const Call call{name, dev, reinterpret_cast<cudaStream_t>(stream)};
    return operands == kS8 ? launch_product<true>(call, p, false) : launch_product<false>(call, p, operands == EMMY_BF16);
}

// A warp for each row while its registers hold the row, else a block of 128 or 256 threads.
template <typename T>
int launch_quantize(const Call &call, const T *x, int64_t x_stride, int8_t *q, int64_t q_stride, float *scale,
                    int64_t rows, int64_t k) {
    constexpr int VEC = 16 / sizeof(T);
    const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && reinterpret_cast<uintptr_t>(q) % VEC == 0 &&
                     x_stride % VEC == 0 && q_stride % VEC == 0 && k % VEC == 0;
    auto go = [&](auto kernel, int group) {
        const int threads = group == 32 ? 256 : group;
        cudaLaunchConfig_t cfg = config(call, ceil_div(rows, threads / group), threads, 0);
        cudaLaunchAttribute attr = early_start();
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        return launched(call, cudaLaunchKernelEx(&cfg, kernel, x, x_stride, q, q_stride, scale, rows, k));
    };
    if (vec) {
        if (k <= 32 * 4 * VEC) return go(quantize_rows_kernel<T, VEC, 32, 4>, 32);
        if (k <= 128 * 4 * VEC) return go(quantize_rows_kernel<T, VEC, 128, 4>, 128);
        if (k <= 256 * 4 * VEC) return go(quantize_rows_kernel<T, VEC, 256, 4>, 256);
        return go(quantize_rows_kernel<T, VEC, 256, 8>, 256);
    }
    if (k <= 32 * 32) return go(quantize_rows_kernel<T, 1, 32, 32>, 32);
    if (k <= 128 * 32) return go(quantize_rows_kernel<T, 1, 128, 32>, 128);
    return go(quantize_rows_kernel<T, 1, 256, 32>, 256);
}

int check_common(const char *name, int dev, int64_t rows, int64_t experts, int64_t n, int64_t k) {
    if (dev < 0 || dev >= 64) return report(EMMY_ERR_INVALID, "%s: bad device %d", name, dev);
    if (bad_extent(rows) || bad_extent(n) || bad_extent(k))
        return report(EMMY_ERR_INVALID, "%s: rows, n and k must be within 0 and 2^31 - 1024", name);
    if (experts < 0 || experts > kMaxExperts)
        return report(EMMY_ERR_INVALID, "%s: experts must be within 0 and %d", name, kMaxExperts);
    return EMMY_OK;
}

int check_types(const char *name, int dtype, int out_dtype) {
    if (dtype != EMMY_BF16 && dtype != EMMY_F16)
        return report(EMMY_ERR_INVALID, "%s: operands must be EMMY_BF16 or EMMY_F16", name);
    if (out_dtype != dtype && out_dtype != EMMY_F32)
        return report(EMMY_ERR_INVALID, "%s: the output must be of the operands' type or EMMY_F32", name);
    return EMMY_OK;
}

}  // namespace

extern "C" int emmy_grouped_matmul(int dev, int dtype, int out_dtype, const void *x, int64_t x_stride, const void *w,
                                   int64_t w_stride_e, int64_t w_stride_n, int64_t w_stride_k,
                                   const int32_t *offsets, void *out, int64_t out_stride, int64_t rows,
                                   int64_t experts, int64_t n, int64_t k, uint64_t stream) {
    static const char name[] = "emmy_grouped_matmul";
    if (int rc = check_common(name, dev, rows, experts, n, k)) return rc;
    if (int rc = check_types(name, dtype, out_dtype)) return rc;
    if (w_stride_n != 1 && w_stride_k != 1)
        return report(EMMY_ERR_INVALID, "%s: one of w's strides over n and k must be 1", name);
    if (x_stride < 0 || w_stride_e < 0 || w_stride_n < 0 || w_stride_k < 0 || out_stride < n)
        return report(EMMY_ERR_INVALID, "%s: negative stride, or output rows that overlap", name);
    if (rows && experts && n && (!offsets || !out || (k && (!x || !w))))
        return report(EMMY_ERR_INVALID, "%s: NULL pointer", name);
    Product p{};
    p.a = w, p.b = x, p.out = out, p.offsets = offsets;
    p.a_e = w_stride_e, p.a_m = w_stride_n, p.a_k = w_stride_k;
    p.b_c = x_stride, p.b_k = 1, p.out_c = out_stride;
    p.m = n, p.k = k, p.rows = rows;
    p.experts = static_cast<int>(experts), p.out_type = out_dtype;
    return run_product(name, dev, dtype, p, stream);
}

extern "C" int emmy_grouped_matmul_dw(int dev, int dtype, int out_dtype, const void *dy, int64_t dy_stride,
                                      const void *x, int64_t x_stride, const int32_t *offsets, void *dw,
                                      int64_t dw_stride_e, int64_t dw_stride_n, int64_t rows, int64_t experts,
                                      int64_t n, int64_t k, uint64_t stream) {
    static const char name[] = "emmy_grouped_matmul_dw";
    if (int rc = check_common(name, dev, rows, experts, n, k)) return rc;
    if (int rc = check_types(name, dtype, out_dtype)) return rc;
    if (dy_stride < 0 || x_stride < 0 || dw_stride_n < k || dw_stride_e < 0)
        return report(EMMY_ERR_INVALID, "%s: negative stride, or output rows that overlap", name);
    if (experts > 1 && n && k && dw_stride_e < (n - 1) * dw_stride_n + k)
        return report(EMMY_ERR_INVALID, "%s: output matrices overlap", name);
    if (experts && n && k && (!dw || !offsets || (rows && (!dy || !x))))
        return report(EMMY_ERR_INVALID, "%s: NULL pointer", name);
    Product p{};
    p.a = x, p.b = dy, p.out = dw, p.offsets = offsets;
    p.a_m = 1, p.a_k = x_stride;
    p.b_c = 1, p.b_k = dy_stride, p.out_e = dw_stride_e, p.out_c = dw_stride_n;
    p.m = k, p.c = n, p.rows = rows;
    p.experts = static_cast<int>(experts), p.out_type = out_dtype, p.dw = true;
    return run_product(name, dev, dtype, p, stream);
}

extern "C" int emmy_int8_matmul(int dev, int out_dtype, const int8_t *xq, int64_t x_stride, const float *x_scale,
                                const int8_t *wq, int64_t w_stride_e, int64_t w_stride_n, const float *w_scale,
                                const float *bias, const int32_t *offsets, void *out, int64_t out_stride,
                                int64_t rows, int64_t experts, int64_t n, int64_t k, uint64_t stream) {
    static const char name[] = "emmy_int8_matmul";
    if (int rc = check_common(name, dev, rows, experts, n, k)) return rc;
    if (out_dtype != EMMY_F32 && out_dtype != EMMY_BF16 && out_dtype != EMMY_F16)
        return report(EMMY_ERR_INVALID, "%s: the output must be EMMY_F32, EMMY_BF16 or EMMY_F16", name);
    if (k > EMMY_PRODUCTS_MAX_K8)
        return report(EMMY_ERR_INVALID, "%s: k must be at most %d: a longer sum could pass 32 bits", name,
                      EMMY_PRODUCTS_MAX_K8);
    if (!offsets && experts != 1)
        return report(EMMY_ERR_INVALID, "%s: without offsets there is one expert", name);
    if (x_stride < 0 || w_stride_e < 0 || w_stride_n < 0 || out_stride < n)
        return report(EMMY_ERR_INVALID, "%s: negative stride, or output rows that overlap", name);
    if (rows && experts && n && (!out || !x_scale || !w_scale || (k && (!xq || !wq))))
        return report(EMMY_ERR_INVALID, "%s: NULL pointer", name);
    Product p{};
    p.a = wq, p.b = xq, p.out = out, p.offsets = offsets;
    p.x_scale = x_scale, p.w_scale = w_scale, p.bias = bias;
    p.a_e = w_stride_e, p.a_m = w_stride_n, p.a_k = 1;
    p.b_c = x_stride, p.b_k = 1, p.out_c = out_stride;
    p.m = n, p.k = k, p.rows = rows;
    p.experts = static_cast<int>(experts), p.out_type = out_dtype;
    return run_product(name, dev, kS8, p, stream);
}

extern "C" int emmy_quantize_rows(int dev, int dtype, const void *x, int64_t x_stride, int8_t *q, int64_t q_stride,
                                  float *scale, int64_t rows, int64_t k, uint64_t stream) {
    static const char name[] = "emmy_quantize_rows";
    if (int rc = check_common(name, dev, rows, 1, 0, k)) return rc;
    if (dtype != EMMY_F32 && dtype != EMMY_BF16 && dtype != EMMY_F16)
        return report(EMMY_ERR_INVALID, "%s: rows must be EMMY_F32, EMMY_BF16 or EMMY_F16", name);
    if (x_stride < 0 || q_stride < k)
        return report(EMMY_ERR_INVALID, "%s: negative stride, or output rows that overlap", name);
    if (rows == 0) return EMMY_OK;
    if (!scale || (k && (!x || !q))) return report(EMMY_ERR_INVALID, "%s: NULL pointer", name);
    DeviceScope scope(dev);
    if (scope.err != cudaSuccess) return report(EMMY_ERR_CUDA, "%s: device %d: %s", name, dev, cudaGetErrorString(scope.err));
    const Call call{name, dev, reinterpret_cast<cudaStream_t>(stream)};
    if (dtype == EMMY_BF16) return launch_quantize(call, static_cast<const __nv_bfloat16 *>(x), x_stride, q, q_stride, scale, rows, k);
    if (dtype == EMMY_F16) return launch_quantize(call, static_cast<const __half *>(x), x_stride, q, q_stride, scale, rows, k);
    return launch_quantize(call, static_cast<const float *>(x), x_stride, q, q_stride, scale, rows, k);
}

extern "C" int emmy_products_variant(int esize, int dw, int aligned, int64_t rows, int64_t experts, int64_t n,
                                     int64_t k, int32_t *variant) {
    static const char name[] = "emmy_products_variant";
    if (int rc = check_common(name, 0, rows, experts, n, k)) return rc;
    if ((esize != 1 && esize != 2) || (dw && esize == 1))
        return report(EMMY_ERR_INVALID, "%s: operands of 2 bytes, or of 1 where dw is 0", name);
    if (!variant) return report(EMMY_ERR_INVALID, "%s: NULL pointer", name);
    Product p{};
    p.m = dw ? k : n, p.c = dw ? n : 0, p.k = dw ? 0 : k, p.rows = rows;
    p.experts = static_cast<int>(experts), p.dw = dw != 0;
    Variant v;
    // without rows or terms of a sum there is nothing for TMA to load
    if (!no_output(p) && !choose(p, esize, aligned && rows && k, v))
        return report(EMMY_ERR_INVALID, "%s: an output of more than 2^30 tiles is not supported", name);
    variant[0] = v.pair != 0, variant[1] = v.bn, variant[2] = v.split;
    return EMMY_OK;
}

extern "C" int emmy_products_status(int dev, uint32_t *status) {
    if (!status) return report(EMMY_ERR_INVALID, "emmy_products_status: NULL pointer");
    if (dev < 0 || dev >= 64) return report(EMMY_ERR_INVALID, "emmy_products_status: bad device %d", dev);
    DeviceScope scope(dev);
    cudaError_t err = scope.err;
    const unsigned int zero = 0u;
    if (err == cudaSuccess) err = cudaDeviceSynchronize();
    if (err == cudaSuccess) err = cudaMemcpyFromSymbol(status, emmy_status, sizeof *status);
    if (err == cudaSuccess && *status) err = cudaMemcpyToSymbol(emmy_status, &zero, sizeof zero);
    if (err != cudaSuccess) return report(EMMY_ERR_CUDA, "emmy_products_status: %s", cudaGetErrorString(err));
    return EMMY_OK;
}
