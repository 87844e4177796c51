// Device pieces that the product kernels share: the description of a product, the boundaries of
// its groups, and the conversion of a finished sum.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "emmy_b200.h"

namespace {

constexpr int kMaxExperts = EMMY_PRODUCTS_MAX_EXPERTS;
constexpr int kS8 = 3;  // operand code of 8-bit products beside EMMY_F32, EMMY_BF16 and EMMY_F16

// One product, as the kernels see it.  Strides are in elements.
struct Product {
    const void *a;  // A(m, k) of expert e at a[e * a_e + m * a_m + k * a_k]  (dw: k counts from the group's start)
    const void *b;  // B(c, k): forward b[(begin_e + c) * b_c + k], dw b[(begin_e + k) * b_k + c]
    const void *a_end, *b_end;  // behind the operands' last values (plain loads stay below them)
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

}  // namespace
