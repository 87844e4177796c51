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
// the host and a recorded graph follows new boundaries.

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

// x / s rounded to the nearest integer, exact ties to even, for the quotient of the two f32 values.
// The product with the rounded reciprocal is off by less than 1e-4 below 128, so only a quotient
// that close to a half is settled by the sign of x - (q +- 1/2) s, which one FMA gives exactly.
__device__ __forceinline__ float quantize_one(float x, float s, float inv) {
    const float t = x * inv;
    float q = rintf(t);
    const float d = t - q;
    if (fabsf(d) > 0.4999f) {
        const float step = d > 0.0f ? 1.0f : -1.0f;
        const float past = fmaf(-(q + 0.5f * step), s, x) * step;  // > 0: beyond the half, away from q
        const float even = q * 0.5f;
        if (past > 0.0f || (past == 0.0f && rintf(even) != even)) q += step;
    }
    return fminf(fmaxf(q, -127.0f), 127.0f);
}

// One row for each block at a time: its largest magnitude, then its integers.
template <typename T>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const T *__restrict__ x, int64_t x_stride,
                                                            int8_t *__restrict__ q, int64_t q_stride,
                                                            float *__restrict__ scale, int64_t rows, int64_t k) {
    __shared__ float s_peak[8];
    __shared__ int s_bad[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const T *xr = x + r * x_stride;
        float peak = 0.0f;
        bool bad = false;
        for (int64_t i = threadIdx.x; i < k; i += 256) {
            const float v = fabsf(to_float(xr[i]));
            bad |= !(v <= 3.402823466e38f);  // infinity or NaN
            peak = fmaxf(peak, v);
        }
        for (int d = 16; d > 0; d >>= 1) peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, d));
        const int any = __any_sync(0xffffffffu, bad);
        __syncthreads();
        if (lane == 0) {
            s_peak[warp] = peak;
            s_bad[warp] = any;
        }
        __syncthreads();
        bad = false;
        for (int i = 0; i < 8; ++i) {
            peak = fmaxf(peak, s_peak[i]);
            bad |= s_bad[i] != 0;
        }
        const float s = __fdiv_rn(peak, 127.0f);
        // a scale whose reciprocal could overflow is lifted, with its row, by a power of two
        const float lift = s < 1e-30f ? 0x1p64f : 1.0f;
        const float ls = s * lift, inv = 1.0f / ls;
        for (int64_t i = threadIdx.x; i < k; i += 256)
            q[r * q_stride + i] =
                bad || s == 0.0f ? 0 : static_cast<int8_t>(quantize_one(to_float(xr[i]) * lift, ls, inv));
        if (threadIdx.x == 0) scale[r] = bad ? __int_as_float(0x7fffffff) : s;
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

// The call's device, made current for the launch and put back afterwards.
struct DeviceScope {
    int prev = -1;
    cudaError_t err;
    explicit DeviceScope(int dev) {
        err = cudaGetDevice(&prev);
        if (err == cudaSuccess && prev != dev) err = cudaSetDevice(dev);
        if (prev == dev) prev = -1;
    }
    ~DeviceScope() {
        if (prev >= 0) cudaSetDevice(prev);
    }
};

constexpr int64_t kMaxExtent = (1ll << 31) - 1;

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

using TcKernel = void (*)(Product, Layout, CUtensorMap, CUtensorMap);

// A launch of clusters of `cluster` CTAs.  `ready` marks the devices on which the kernel's
// shared-memory limit has been raised.
int launch_clusters(const Call &call, TcKernel kernel, std::atomic<uint64_t> &ready, const Product &p, const Layout &lay,
                    const CUtensorMap &ta, const CUtensorMap &tb, int64_t clusters, int cluster, int threads,
                    uint32_t smem) {
    if (!(ready.load(std::memory_order_acquire) >> call.dev & 1)) {
        const cudaError_t err =
            cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
        if (err != cudaSuccess) return launched(call, err);
        ready.fetch_or(1ull << call.dev, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim = {static_cast<unsigned>(cluster), 1, 1};
    cfg.gridDim = dim3(static_cast<unsigned>(clusters * cluster));
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = call.stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return launched(call, cudaLaunchKernelEx(&cfg, kernel, p, lay, ta, tb));
}

template <bool I8, int BN, bool TMA>
int launch_single(const Call &call, const Product &p, const Layout &lay, const CUtensorMap &ta, const CUtensorMap &tb,
                  int64_t clusters, int split) {
    using Cfg = TcConfig<I8, BN, TMA>;
    static std::atomic<uint64_t> ready{0};
    return launch_clusters(call, product_tc_kernel<I8, BN, TMA>, ready, p, lay, ta, tb, clusters, split, Cfg::kThreads,
                           Cfg::kSmem);
}

template <bool I8, int BN>
int launch_pair(const Call &call, const Product &p, const Layout &lay, const CUtensorMap &ta, const CUtensorMap &tb,
                int64_t pairs) {
    static std::atomic<uint64_t> ready{0};
    return launch_clusters(call, product_pair_kernel<I8, BN>, ready, p, lay, ta, tb, pairs, 2, 192,
                           PairConfig<BN>::kSmem);
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

template <bool I8>
int launch_product(const Call &call, const Product &p, bool bf16) {
    constexpr int esize = I8 ? 1 : 2, bk = 128 / esize;
    Layout lay{};
    lay.a_mn = p.dw || p.a_k != 1;
    lay.b_mn = p.dw;
    lay.bf16 = bf16;
    Operand a{p.a, 0, 0, 0, 1, 0}, b{p.b, 0, 0, 0, 1, 0};
    if (p.dw) {
        a.inner = p.m, a.rows = p.rows, a.row_stride = p.a_k;
        b.inner = p.c, b.rows = p.rows, b.row_stride = p.b_k;
    } else {
        a.inner = lay.a_mn ? p.m : p.k, a.rows = lay.a_mn ? p.k : p.m, a.row_stride = lay.a_mn ? p.a_k : p.a_m;
        a.mats = p.experts, a.mat_stride = p.a_e;
        b.inner = p.k, b.rows = p.rows, b.row_stride = p.b_c;
    }
    bool tma = encode_tiled() && tma_ready(a, esize) && tma_ready(b, esize);

    // groups that can hold rows, and the rows of an even one
    const int64_t groups = p.experts < p.rows ? p.experts : (p.rows ? p.rows : 1);
    const int64_t even = ceil_div(p.rows, groups), kblocks = ceil_div(p.dw ? even : p.k, bk);
    // tiles of even groups, and the most that any grouping can have
    auto tiles = [&](int64_t tm, int64_t tc) {
        return ceil_div(p.m, tm) * (p.dw ? p.experts * ceil_div(p.c, tc) : groups * ceil_div(even, tc));
    };
    auto most = [&](int64_t tm, int64_t tc) {
        return ceil_div(p.m, tm) * (p.dw ? p.experts * ceil_div(p.c, tc) : p.rows / tc + groups);
    };
    const int64_t cext = p.dw ? p.c : even;
    int pair = 0;
    if (tma && p.m > 128 && cext > 64) {
        if (cext > 192 && tiles(256, 256) >= kSms / 4) pair = 256;
        else if (tiles(256, 128) >= kSms / 4) pair = 128;
    }
    const int bn = pair ? pair : p.dw ? 128 : even <= 12 ? 16 : even <= 24 ? 32 : even <= 48 ? 64 : 128;

    CUtensorMap ta{}, tb{};
    if (tma) {
        const CUtensorMapDataType type = I8     ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                         : bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
        if (!encode(&ta, a, type, esize, 3, bk, lay.a_mn ? 64 : kTileM) ||
            !encode(&tb, b, type, esize, 2, bk, lay.b_mn ? 64 : pair ? pair / 2 : bn))
            return report(EMMY_ERR_CUDA, "%s: cuTensorMapEncodeTiled failed", call.name);
    }
    if (pair) {
        int64_t pairs = most(256, pair);
        if (pairs > kSms / 2) pairs = kSms / 2;
        return pair == 256 ? launch_pair<I8, 256>(call, p, lay, ta, tb, pairs)
                           : launch_pair<I8, 128>(call, p, lay, ta, tb, pairs);
    }
    const int resident = kSms * (bn <= 32 ? 2 : 1);
    int split = 1;
    while (split < 8 && tiles(kTileM, bn) * split * 2 <= resident && kblocks >= split * 2 * 4) split *= 2;
    int64_t clusters = most(kTileM, bn);
    if (clusters > resident / split) clusters = resident / split;
    if (!tma)
        return bn <= 32 ? launch_single<I8, 32, false>(call, p, lay, ta, tb, clusters, split)
                        : launch_single<I8, 128, false>(call, p, lay, ta, tb, clusters, split);
    switch (bn) {
        case 16: return launch_single<I8, 16, true>(call, p, lay, ta, tb, clusters, split);
        case 32: return launch_single<I8, 32, true>(call, p, lay, ta, tb, clusters, split);
        case 64: return launch_single<I8, 64, true>(call, p, lay, ta, tb, clusters, split);
        default: return launch_single<I8, 128, true>(call, p, lay, ta, tb, clusters, split);
    }
}

int run_product(const char *name, int dev, int operands, const Product &p, uint64_t stream) {
    if (p.m == 0 || p.experts == 0 || (p.dw ? p.c : p.rows) == 0) return EMMY_OK;
    DeviceScope scope(dev);
    if (scope.err != cudaSuccess)
        return report(EMMY_ERR_CUDA, "%s: device %d: %s", name, dev, cudaGetErrorString(scope.err));
    const Call call{name, dev, reinterpret_cast<cudaStream_t>(stream)};
    return operands == kS8 ? launch_product<true>(call, p, false) : launch_product<false>(call, p, operands == EMMY_BF16);
}

int check_common(const char *name, int dev, int64_t rows, int64_t experts, int64_t n, int64_t k) {
    if (dev < 0 || dev >= 64) return report(EMMY_ERR_INVALID, "%s: bad device %d", name, dev);
    if (bad_extent(rows) || bad_extent(n) || bad_extent(k))
        return report(EMMY_ERR_INVALID, "%s: rows, n and k must be within 0 and 2^31 - 1", name);
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
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const unsigned grid = static_cast<unsigned>(rows < 148 * 8 ? rows : 148 * 8);
    if (dtype == EMMY_BF16)
        quantize_rows_kernel<<<grid, 256, 0, s>>>(static_cast<const __nv_bfloat16 *>(x), x_stride, q, q_stride, scale, rows, k);
    else if (dtype == EMMY_F16)
        quantize_rows_kernel<<<grid, 256, 0, s>>>(static_cast<const __half *>(x), x_stride, q, q_stride, scale, rows, k);
    else
        quantize_rows_kernel<<<grid, 256, 0, s>>>(static_cast<const float *>(x), x_stride, q, q_stride, scale, rows, k);
    const cudaError_t err = cudaGetLastError();
    if (err != cudaSuccess) return report(EMMY_ERR_CUDA, "%s: launch: %s", name, cudaGetErrorString(err));
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
