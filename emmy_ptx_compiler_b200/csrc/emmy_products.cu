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

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <cstdarg>
#include <cstdio>

#include "emmy_b200.h"
#include "emmy_launch_record.h"

extern "C" int emmy_record_error(int code, const char *msg);  // emmy_runtime.cpp (not exported)

// Status bits of this file's kernels, one word for each device (the name is private to this file).
#define emmy_status g_products_status
extern "C" {
static __device__ unsigned int g_products_status = 0u;
}

namespace {

constexpr int kMaxExperts = EMMY_PRODUCTS_MAX_EXPERTS;
constexpr int kS8 = 3;  // operand code of 8-bit products beside EMMY_F32, EMMY_BF16 and EMMY_F16

// One product, as the kernels see it.  Strides are in elements.
struct Product {
    const void *a;  // A(m, k) of expert e at a[e * a_e + m * a_m + k * a_k]  (dw: k counts from the group's start)
    const void *b;  // B(c, k): forward b[(begin_e + c) * b_c + k], dw b[(begin_e + k) * b_k + c]
    void *out;      // forward out[(begin_e + c) * out_c + m], dw out[e * out_e + c * out_c + m]
    const int32_t *offsets;
    const float *x_scale;  // [rows], or NULL: plain sums
    const float *w_scale;  // [experts, m]
    const float *bias;     // [experts, m], or NULL
    int64_t a_e, a_m, a_k, b_c, b_k, out_e, out_c;
    int64_t m, c, k;  // extents; c counts only for dw, k only for the forward form
    int64_t rows;
    int experts;
    int out_type;
    bool dw;
};

// ---------------------------------------------------------------- groups

// Boundaries of the groups in shared memory: row[e] .. row[e + 1] are expert e's rows, after every
// offset was brought into [0, rows] and up to the largest before it; tiles[e] counts the column
// tiles of the experts before e.
struct Groups {
    int row[kMaxExperts + 1];
    int tiles[kMaxExperts + 1];
};

// Filled by one whole warp: each lane takes a run of consecutive experts; running maxima and sums
// cross the lanes in two warp scans.
__device__ __forceinline__ void load_groups(Groups &g, const Product &p, int col_tile) {
    const int lane = threadIdx.x & 31, e = p.experts, rows = static_cast<int>(p.rows);
    if (!p.offsets) {
        if (lane == 0) {
            g.row[0] = 0;
            g.row[1] = rows;
        }
    } else {
        const int per = (e + 1 + 31) / 32, i0 = lane * per, i1 = min(e + 1, i0 + per);
        int top = 0;
        for (int i = i0; i < i1; ++i) {
            top = max(top, min(max(p.offsets[i], 0), rows));
            g.row[i] = top;
        }
        for (int d = 1; d < 32; d <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, top, d);
            if (lane >= d) top = max(top, up);
        }
        const int before = __shfl_up_sync(0xffffffffu, top, 1);
        if (lane > 0)
            for (int i = i0; i < i1; ++i) g.row[i] = max(g.row[i], before);
    }
    __syncwarp();
    const int per = (e + 31) / 32, i0 = min(e, lane * per), i1 = min(e, i0 + per);
    auto tiles_of = [&](int i) {
        return p.dw ? static_cast<int>((p.c + col_tile - 1) / col_tile)
                    : (g.row[i + 1] - g.row[i] + col_tile - 1) / col_tile;
    };
    int sum = 0;
    for (int i = i0; i < i1; ++i) sum += tiles_of(i);
    int upto = sum;
    for (int d = 1; d < 32; d <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += up;
    }
    int at = upto - sum;
    for (int i = i0; i < i1; ++i) {
        g.tiles[i] = at;
        at += tiles_of(i);
    }
    if (lane == 31) g.tiles[e] = upto;
    __syncwarp();
}

__device__ __forceinline__ void store_out(void *out, int type, int64_t i, float v) {
    if (type == EMMY_BF16) {
        static_cast<__nv_bfloat16 *>(out)[i] = __float2bfloat16_rn(v);
    } else if (type == EMMY_F16) {
        static_cast<__half *>(out)[i] = __float2half_rn(v);
    } else {
        static_cast<float *>(out)[i] = v;
    }
}

__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(float v) { return v; }

template <typename Acc, typename T>
__device__ __forceinline__ Acc load_as(T v) {
    if constexpr (sizeof(T) == 1) return v;
    else return to_float(v);
}

// ---------------------------------------------------------------- products on CUDA cores

// 64 x 64 tiles on 256 threads, 16 of k at a time through shared memory: any stride, alignment and
// extent.  Sums are held in f32 (s32 for 8-bit operands).
template <typename T, typename Acc>
__global__ void __launch_bounds__(256) product_simt_kernel(const Product p) {
    constexpr int TM = 64, TC = 64, TK = 16;
    __shared__ Groups g;
    __shared__ Acc sa[TK][TM + 1];
    __shared__ Acc sb[TK][TC + 1];
    if (threadIdx.x < 32) load_groups(g, p, TC);
    __syncthreads();
    const int64_t mt = (p.m + TM - 1) / TM, total = mt * g.tiles[p.experts];
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const T *a = static_cast<const T *>(p.a), *b = static_cast<const T *>(p.b);
    int e = 0;
    for (int64_t t = blockIdx.x; t < total; t += gridDim.x) {
        while (t >= mt * g.tiles[e + 1]) ++e;
        const int64_t r = t - mt * g.tiles[e];
        const int64_t m0 = r % mt * TM, c0 = r / mt * TC;
        const int64_t begin = g.row[e], count = g.row[e + 1] - g.row[e];
        const int64_t cend = p.dw ? p.c : count, kend = p.dw ? count : p.k;
        const T *ae = a + (p.dw ? begin * p.a_k : e * p.a_e);
        const T *be = b + begin * (p.dw ? p.b_k : p.b_c);
        Acc acc[4][4] = {};
        for (int64_t k0 = 0; k0 < kend; k0 += TK) {
            for (int i = threadIdx.x; i < TK * TM; i += 256) {
                // neighbouring threads follow the axis that is contiguous in memory
                const int mm = p.a_k == 1 ? i / TK : i % TM, kk = p.a_k == 1 ? i % TK : i / TM;
                const int64_t gm = m0 + mm, gk = k0 + kk;
                sa[kk][mm] = gm < p.m && gk < kend ? load_as<Acc>(ae[gm * p.a_m + gk * p.a_k]) : Acc(0);
            }
            for (int i = threadIdx.x; i < TK * TC; i += 256) {
                const int cc = p.b_k == 1 ? i / TK : i % TC, kk = p.b_k == 1 ? i % TK : i / TC;
                const int64_t gc = c0 + cc, gk = k0 + kk;
                sb[kk][cc] = gc < cend && gk < kend ? load_as<Acc>(be[gc * p.b_c + gk * p.b_k]) : Acc(0);
            }
            __syncthreads();
            for (int kk = 0; kk < TK; ++kk) {
                Acc av[4], bv[4];
                #pragma unroll
                for (int i = 0; i < 4; ++i) av[i] = sa[kk][tx + 16 * i];
                #pragma unroll
                for (int i = 0; i < 4; ++i) bv[i] = sb[kk][ty + 16 * i];
                #pragma unroll
                for (int i = 0; i < 4; ++i)
                    #pragma unroll
                    for (int j = 0; j < 4; ++j) acc[i][j] += av[i] * bv[j];
            }
            __syncthreads();
        }
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            #pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t m = m0 + tx + 16 * i, c = c0 + ty + 16 * j;
                if (m >= p.m || c >= cend) continue;
                float v = static_cast<float>(acc[i][j]);
                if (p.x_scale) {
                    v = v * p.x_scale[begin + c] * p.w_scale[e * p.m + m];
                    if (p.bias) v += p.bias[e * p.m + m];
                }
                store_out(p.out, p.out_type, (p.dw ? e * p.out_e : begin * p.out_c) + c * p.out_c + m, v);
            }
        }
    }
}

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

int launch_product(const char *name, int dev, int operands, const Product &p, uint64_t stream) {
    if (p.m == 0 || p.experts == 0 || (p.dw ? p.c : p.rows) == 0) return EMMY_OK;
    DeviceScope scope(dev);
    if (scope.err != cudaSuccess) return report(EMMY_ERR_CUDA, "%s: device %d: %s", name, dev, cudaGetErrorString(scope.err));
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const int64_t mt = (p.m + 63) / 64;
    const int64_t ct = p.dw ? p.experts * ((p.c + 63) / 64) : p.rows / 64 + (p.rows < p.experts ? p.rows : p.experts);
    const unsigned grid = static_cast<unsigned>(mt * ct < 148 * 4 ? mt * ct : 148 * 4);
    switch (operands) {
        case EMMY_BF16: product_simt_kernel<__nv_bfloat16, float><<<grid, 256, 0, s>>>(p); break;
        case EMMY_F16: product_simt_kernel<__half, float><<<grid, 256, 0, s>>>(p); break;
        default: product_simt_kernel<int8_t, int><<<grid, 256, 0, s>>>(p); break;
    }
    const cudaError_t err = cudaGetLastError();
    if (err != cudaSuccess) return report(EMMY_ERR_CUDA, "%s: launch: %s", name, cudaGetErrorString(err));
    return EMMY_OK;
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
    return launch_product(name, dev, dtype, p, stream);
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
    return launch_product(name, dev, dtype, p, stream);
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
    return launch_product(name, dev, kS8, p, stream);
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
    if (err == cudaSuccess) err = cudaMemcpyFromSymbol(status, g_products_status, sizeof *status);
    if (err == cudaSuccess && *status) err = cudaMemcpyToSymbol(g_products_status, &zero, sizeof zero);
    if (err != cudaSuccess) return report(EMMY_ERR_CUDA, "emmy_products_status: %s", cudaGetErrorString(err));
    return EMMY_OK;
}
