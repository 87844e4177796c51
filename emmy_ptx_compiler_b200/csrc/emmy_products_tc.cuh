// Products on the 5th-generation tensor cores: out(c, m) = sum_k A(m, k) B(c, k).
//
// The output's contiguous axis m (the channels) lies on the 128 lanes of tensor memory and the
// output's rows c (the tokens of a group) on the N columns of the instruction, 16 to 128 of them.
// So a group of a few tokens costs a few columns, not a padded tile of 128 rows, and a warp's
// 32 lanes store 32 neighbouring channels of one output row.
#pragma once

#include "emmy_products_dev.cuh"
#include "emmy_sm100.cuh"

#include <type_traits>

namespace emmy {

// tcgen05.mma and tcgen05.commit predicated on `elected`, for a warp that runs its loop together and
// issues from one lane.  The operands have to be in uniform registers: they stay there while the
// control flow is the whole warp's, and have to be moved there for each instruction inside a
// branch that one lane takes.
template <bool I8, bool PAIR>
__device__ __forceinline__ void umma_if(uint32_t elected, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                        uint32_t idesc, uint32_t accumulate) {
#define EMMY_UMMA_IF(GROUP, KIND)                                                              \
    asm volatile(                                                                              \
        "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"               \
        " @q tcgen05.mma.cta_group::" GROUP ".kind::" KIND " [%0], %1, %2, %3, p;\n}\n" ::"r"( \
            d_tmem),                                                                           \
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(elected)                    \
        : "memory")
    if constexpr (I8 && PAIR) EMMY_UMMA_IF("2", "i8");
    else if constexpr (I8) EMMY_UMMA_IF("1", "i8");
    else if constexpr (PAIR) EMMY_UMMA_IF("2", "f16");
    else EMMY_UMMA_IF("1", "f16");
#undef EMMY_UMMA_IF
}

// Arrive on this CTA's `bar` (PAIR: on the barrier at that place of both CTAs) once every MMA issued
// before has completed.
template <bool PAIR>
__device__ __forceinline__ void umma_commit_if(uint32_t elected, uint32_t bar) {
    if constexpr (PAIR)
        asm volatile(
            "{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n"
            " @q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %2;\n}\n"
            ::"r"(bar), "r"(elected), "h"(static_cast<uint16_t>(3))
            : "memory");
    else
        asm volatile(
            "{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n"
            " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(bar),
            "r"(elected)
            : "memory");
}

// 32 lanes x 16 consecutive 32-bit columns.
__device__ __forceinline__ void tmem_ld_32x32b_x16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}

// 16 lanes x 32 consecutive 32-bit columns in matrix-fragment order: register 4 g + i of thread t
// holds lane t / 4 + 8 (i / 2) and column 8 g + 2 (t % 4) + i % 2.
__device__ __forceinline__ void tmem_ld_16x256b_x4(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}

// Four 8 x 8 matrices of 16-bit values in fragment order, stored transposed: lane 8 i + j gives the
// address of column j of matrix i.
__device__ __forceinline__ void stmatrix_x4_trans(uint32_t smem_addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(smem_addr), "r"(a),
                 "r"(b), "r"(c), "r"(d)
                 : "memory");
}

// 3-D tiled load into this CTA's shared memory, completion counted on the mbarrier at
// shared::cluster address `bar_cluster` (the leader's).
__device__ __forceinline__ void tma_load_3d_pair(void *dst, const CUtensorMap *map, uint32_t bar_cluster, int32_t x,
                                                 int32_t y, int32_t z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar_cluster), "r"(x), "r"(y), "r"(z)
        : "memory");
}

// 3-D tiled load into this CTA's shared memory, completion signalled on `bar`.
__device__ __forceinline__ void tma_load_3d(void *dst, const CUtensorMap *map, uint64_t *bar, int32_t x, int32_t y,
                                            int32_t z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
        : "memory");
}

// Orders this thread's plain shared-memory accesses before later ones of the async proxy (TMA, UMMA).
__device__ __forceinline__ void fence_proxy_async() {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// Programmatic launches: a kernel may start while the one before it on the stream still runs; it
// waits here, before its first access to memory that others write, until that one has finished.
__device__ __forceinline__ void wait_for_prior_grid() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_grid_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t cluster_addr) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(cluster_addr) : "memory");
    return v;
}

// Instruction descriptors: kind::f16 with either operand MN-major, and kind::i8 (s8 x s8 -> s32).
__host__ __device__ constexpr uint32_t idesc_f16_major(uint32_t ab_fmt, uint32_t a_mn, uint32_t b_mn, uint32_t m,
                                                       uint32_t n) {
    return idesc_f16(ab_fmt, b_mn, m, n) | (a_mn << 15);
}
__host__ __device__ constexpr uint32_t idesc_s8(uint32_t m, uint32_t n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((m >> 4) << 24);
}

}  // namespace emmy

namespace {

constexpr uint64_t kWaitNs = 2000000000ull;  // per wait: orders of magnitude above any legal one
constexpr int kTileM = 128;
constexpr uint32_t kBlockBytes = 128;                  // one 128-byte swizzle row of k (or of m, c)
constexpr uint32_t kPanel = 64 * kBlockBytes;          // 64 k x 64 m (or c) of an MN-major 16-bit operand
constexpr uint32_t kStageA = kTileM * kBlockBytes;

// The operands' layouts: which of them are contiguous along m (c) instead of along k.
enum : int { kKK = 0, kMK = 1, kMM = 2 };  // kMM: dw

// One block's MMAs (128 bytes of k, or the first `steps` quarters of it) over the operands whose
// descriptors for stage 0 are `a`, `b`.  The stage and the quarter only add to the descriptors' low
// words, and everything else is known at compile time: a single thread issues all of this, and a
// block of 256 x 256 leaves it 512 clocks.
template <bool I8, int LAYOUT, bool PAIR>
struct Issue {
    static constexpr bool kAmn = LAYOUT != kKK, kBmn = LAYOUT == kMM;
    static constexpr uint32_t kStepA = (kAmn ? 16 * kBlockBytes : 32) >> 4, kStepB = (kBmn ? 16 * kBlockBytes : 32) >> 4;

    uint32_t a_lo, b_lo, a_hi, b_hi, idesc, elected;

    __device__ __forceinline__ Issue(const uint8_t *a, const uint8_t *b, bool bf16, int n) {
        const uint64_t da = emmy::smem_desc_sw128(emmy::smem_u32(a), kAmn ? kPanel : 16, 1024);
        const uint64_t db = emmy::smem_desc_sw128(emmy::smem_u32(b), kBmn ? kPanel : 16, 1024);
        a_lo = static_cast<uint32_t>(da), a_hi = static_cast<uint32_t>(da >> 32);
        b_lo = static_cast<uint32_t>(db), b_hi = static_cast<uint32_t>(db >> 32);
        elected = emmy::elect_one();
        const uint32_t m = PAIR ? 2 * kTileM : kTileM;
        idesc = I8 ? emmy::idesc_s8(m, n) : emmy::idesc_f16_major(bf16 ? 1u : 0u, kAmn, kBmn, m, n);
    }
    __device__ __forceinline__ void mma(uint32_t d_tmem, uint32_t a, uint32_t b, uint32_t more) const {
        emmy::umma_if<I8, PAIR>(elected, d_tmem, static_cast<uint64_t>(a_hi) << 32 | a,
                                static_cast<uint64_t>(b_hi) << 32 | b, idesc, more);
    }
    // the whole warp calls these
    __device__ __forceinline__ void block(uint32_t d_tmem, uint32_t a_off, uint32_t b_off, uint32_t more, int steps) const {
        const uint32_t a = a_lo + (a_off >> 4), b = b_lo + (b_off >> 4);
        if (LAYOUT != kMM || steps == 4) {
            mma(d_tmem, a, b, more);
            #pragma unroll
            for (int kk = 1; kk < 4; ++kk) mma(d_tmem, a + kk * kStepA, b + kk * kStepB, 1u);
        } else {
            for (int kk = 0; kk < steps; ++kk) mma(d_tmem, a + kk * kStepA, b + kk * kStepB, more | (kk > 0));
        }
    }
    __device__ __forceinline__ void commit(uint64_t *bar) const {
        emmy::umma_commit_if<PAIR>(elected, emmy::smem_u32(bar));
    }
};

// A value that is the same on every lane, in a form the compiler knows to be.
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

struct Tile {
    int e, begin;   // expert and its first row
    int m0, c0;     // first channel, first output row (of the group; dw: of the matrix)
    int cols;       // output rows in the tile
    int kend;       // extent of the sum
    int kb0, kb1;   // blocks of it that this CTA sums
};

// MMAs (of 16 k) in the block before kb1: 4, or those up to the end of the sum.
__device__ __forceinline__ int last_block_steps(const Tile &w, int kb1, int bk) {
    const int have = w.kend - (kb1 - 1) * bk;
    return have < bk ? (have + 15) / 16 : 4;
}

// Channel tiles that go over all rows of their expert together: what they read of the rows stays
// in L2 from one to the next.
constexpr int kSweep = 8;

// Tile t of the launch (tm x col_tile; host code keeps the tiles within 31 bits).  `e` is a cursor:
// tiles of one caller come in ascending order.  A cluster of `split` CTAs divides the sum.
__device__ __forceinline__ Tile tile_at(const Product &p, const Groups &g, int t, int mt, int &e, int tm, int col_tile,
                                        int bk, uint32_t rank, uint32_t split) {
    while (t >= mt * g.tiles[e + 1]) ++e;
    const int begin = g.row[e], count = g.row[e + 1] - begin;
    const uint32_t r = t - mt * g.tiles[e], sweep_tiles = kSweep * (g.tiles[e + 1] - g.tiles[e]);
    const uint32_t sweep = r / sweep_tiles, in = r - sweep * sweep_tiles, first = sweep * kSweep;
    const uint32_t wide = min(static_cast<uint32_t>(kSweep), mt - first), ci = in / wide;
    Tile o;
    o.e = e;
    o.begin = begin;
    o.m0 = static_cast<int>(first + in - ci * wide) * tm;
    o.c0 = static_cast<int>(ci) * col_tile;
    o.cols = min(col_tile, (p.dw ? static_cast<int>(p.c) : count) - o.c0);
    o.kend = p.dw ? count : static_cast<int>(p.k);
    const uint32_t nkb = o.kend / bk + (o.kend % bk != 0);
    o.kb0 = static_cast<int>(nkb * rank / split);
    o.kb1 = static_cast<int>(nkb * (rank + 1) / split);
    return o;
}

// Operands that TMA cannot address (rows that start off a 16-byte boundary) are loaded in units of
// 64 bytes of a row, as the five aligned 16-byte words that cover them; the bytes are shifted into
// place in registers.  A word is read whole where it lies inside the operand, whichever of its
// bytes are wanted; at the operand's two ends it is put together from its bytes.
struct Unit {
    uint4 w[5];
};

__device__ __noinline__ uint4 load_edge_word(const uint8_t *at, const uint8_t *lo, const uint8_t *hi) {
    alignas(16) uint8_t v[16];
    for (int i = 0; i < 16; ++i) v[i] = at + i >= lo && at + i < hi ? at[i] : 0;
    return *reinterpret_cast<const uint4 *>(v);
}

// `bytes` (at most 64, may be negative) of the unit at `src` are wanted.
__device__ __forceinline__ void load_unit(Unit &u, const uint8_t *src, int64_t bytes, const uint8_t *lo,
                                          const uint8_t *hi) {
    const uint8_t *at = reinterpret_cast<const uint8_t *>(reinterpret_cast<uintptr_t>(src) & ~uintptr_t(15));
    const uint8_t *end = src + (bytes < 64 ? bytes : 64);
    #pragma unroll
    for (int i = 0; i < 5; ++i, at += 16) {
        u.w[i] = make_uint4(0, 0, 0, 0);
        if (bytes > 0 && at < end) {
            if (at >= lo && at + 16 <= hi) u.w[i] = *reinterpret_cast<const uint4 *>(at);
            else u.w[i] = load_edge_word(at, lo, hi);
        }
    }
}

// The first `keep` bytes of a word (any value; below 0 counts as 0).
__device__ __forceinline__ uint32_t keep_bytes(uint32_t v, int64_t keep) {
    return keep >= 4 ? v : keep <= 0 ? 0u : v & ((1u << (8 * static_cast<int>(keep))) - 1u);
}

// Shift a unit into place and store its four 16-byte chunks, zeros behind `bytes`, into row `row` of a
// swizzled panel; `half`: which 64 bytes of the 128-byte row.
__device__ __forceinline__ void store_unit(const Unit &u, const uint8_t *src, int64_t bytes, uint8_t *panel, int row,
                                           int half) {
    const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(src)) & 15u, bits = (off & 3u) * 8u;
    const uint32_t *w = reinterpret_cast<const uint32_t *>(&u);
    uint32_t v[17];
    #pragma unroll
    for (int i = 0; i < 17; ++i) {
        // word off / 4 + i of the 20, without indexing registers by a variable
        const uint32_t near = off & 4u ? w[i + 1] : w[i], far = off & 4u ? w[i + 3] : w[i + 2];
        v[i] = off & 8u ? far : near;
    }
    #pragma unroll
    for (int j = 0; j < 4; ++j) {
        uint32_t c[4];
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            c[i] = __funnelshift_r(v[4 * j + i], v[4 * j + i + 1], bits);
            if (bytes < 64) c[i] = keep_bytes(c[i], bytes - 16 * j - 4 * i);
        }
        *reinterpret_cast<uint4 *>(panel + row * kBlockBytes + (((half * 4 + j) ^ (row & 7)) << 4)) =
            make_uint4(c[0], c[1], c[2], c[3]);
    }
}

// Rows [from, to) of a 64-row panel become zeros (whole 128-byte rows, so the swizzle does not matter).
__device__ __forceinline__ void zero_panel_rows(uint8_t *panel, int from, int to, int lane) {
    for (int i = from * 8 + lane; i < to * 8; i += 32) reinterpret_cast<uint4 *>(panel)[i] = make_uint4(0, 0, 0, 0);
}

template <bool I8>
__device__ __forceinline__ float sum_value(uint32_t bits) {
    if constexpr (I8) return __int2float_rn(static_cast<int>(bits));
    else return __uint_as_float(bits);
}

// Where channel m of output row c of the tile goes.
__device__ __forceinline__ int64_t out_index(const Product &p, const Tile &t, int64_t m, int c) {
    return (p.dw ? t.e * p.out_e : t.begin * p.out_c) + (t.c0 + static_cast<int64_t>(c)) * p.out_c + m;
}

// Scale of a channel, and its bias.
struct Channel {
    float scale = 0.0f, bias = 0.0f;
};
__device__ __forceinline__ Channel channel(const Product &p, const Tile &t, int64_t m) {
    Channel c;
    if (m < p.m) {
        c.scale = p.w_scale[t.e * p.m + m];
        if (p.bias) c.bias = p.bias[t.e * p.m + m];
    }
    return c;
}
template <bool I8>
__device__ __forceinline__ float scaled(uint32_t bits, float row_scale, const Channel &c) {
    if constexpr (I8) return sum_value<true>(bits) * row_scale * c.scale + c.bias;
    else return sum_value<false>(bits);
}

// Staging of a warp's 32 channels x 32 output rows: 64 bytes a row, 80 apart, so that neither the
// transposed 8 x 8 stores nor the 16-byte reads meet bank conflicts.
constexpr uint32_t kStoreRow = 80, kStoreBytes = 32 * kStoreRow;

__device__ __forceinline__ uint32_t pack16(bool bf16, float lo, float hi) {
    if (bf16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&v);
    }
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}

// Output rows [from, to) of a warp's 32 channels, from the accumulator at `taddr`.  Its channels lie
// on lanes, the output's along a row.  16-bit outputs are transposed on the way: fragments of 8 x 8
// go to shared memory through stmatrix, and 4 lanes then write each 64-byte piece of an output row
// 16 bytes at a time (4 stores for 32 rows instead of 32, and the conversion packs two values).  f32
// outputs need no help: 32 lanes write 128 bytes of a row.  `empty`: the sum had no terms.
template <bool I8>
__device__ __forceinline__ void store_tile(const Product &p, const Tile &w, int mq, uint32_t taddr, bool empty, int from,
                                           int to, uint8_t *buf, int lane) {
    if (to > w.cols) to = w.cols;
    if (from >= to) return;
    if (p.out_type == EMMY_F32) {
        const int64_t m = mq + lane;
        Channel ch;
        if constexpr (I8) ch = channel(p, w, m);
        float *out = static_cast<float *>(p.out) + out_index(p, w, m, from);
        #pragma unroll 1
        for (int c = from; c < to; c += 32, out += 32 * p.out_c) {
            uint32_t r[32];
            emmy::tmem_ld_32x32b_x32(taddr + c, r);
            float xs = 0.0f;
            if (I8 && c + lane < to) xs = p.x_scale[w.begin + w.c0 + c + lane];
            emmy::tmem_ld_wait();
            if (empty) {
                #pragma unroll
                for (int j = 0; j < 32; ++j) r[j] = 0u;
            }
            float *o = out;
            #pragma unroll
            for (int j = 0; j < 32; ++j, o += p.out_c) {
                const float v = scaled<I8>(r[j], I8 ? __shfl_sync(0xffffffffu, xs, j) : 0.0f, ch);
                if (m < p.m && c + j < to) *o = v;
            }
        }
        return;
    }
    const int piece = lane & 3;
    uint16_t *out = static_cast<uint16_t *>(p.out) + out_index(p, w, mq, from);
    const bool vec = (reinterpret_cast<uintptr_t>(p.out) & 15) == 0 && ((p.out_c | p.out_e | p.m) & 7) == 0;
    const bool bf16 = p.out_type == EMMY_BF16, piece_in = mq + piece * 8 < p.m;
    Channel ch[4];
    if constexpr (I8) {
        #pragma unroll
        for (int i = 0; i < 4; ++i) ch[i] = channel(p, w, mq + lane / 4 + 8 * i);
    }
    #pragma unroll 1
    for (int c = from; c < to; c += 32, out += 32 * p.out_c) {
        uint32_t r[2][16];
        emmy::tmem_ld_16x256b_x4(taddr + c, r[0]);
        emmy::tmem_ld_16x256b_x4(taddr + (16u << 16) + c, r[1]);
        float xs[8];
        if constexpr (I8) {
            #pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int col = c + 8 * (i >> 1) + 2 * piece + (i & 1);
                xs[i] = col < to ? p.x_scale[w.begin + w.c0 + col] : 0.0f;
            }
        }
        emmy::tmem_ld_wait();
        if (empty) {
            #pragma unroll
            for (int i = 0; i < 16; ++i) r[0][i] = r[1][i] = 0u;
        }
        #pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t v[8];
            #pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int row = 2 * h + (i & 1), col = i >> 1 << 1;
                v[i] = pack16(bf16, scaled<I8>(r[h][2 * i], I8 ? xs[col] : 0.0f, ch[row]),
                              scaled<I8>(r[h][2 * i + 1], I8 ? xs[col + 1] : 0.0f, ch[row]));
            }
            const uint32_t at = emmy::smem_u32(buf) + ((lane >> 4) * 8 + (lane & 7)) * kStoreRow +
                                (16 * h + 8 * ((lane >> 3) & 1)) * 2;
            emmy::stmatrix_x4_trans(at, v[0], v[1], v[2], v[3]);
            emmy::stmatrix_x4_trans(at + 16 * kStoreRow, v[4], v[5], v[6], v[7]);
        }
        __syncwarp();
        if (vec) {
            #pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = i * 8 + (lane >> 2);
                if (piece_in && c + row < to)
                    *reinterpret_cast<uint4 *>(out + row * p.out_c + piece * 8) =
                        *reinterpret_cast<const uint4 *>(buf + row * kStoreRow + piece * 16);
            }
        } else if (mq + lane < p.m) {
            for (int row = 0; row < 32 && c + row < to; ++row)
                out[row * p.out_c + lane] = *reinterpret_cast<const uint16_t *>(buf + row * kStoreRow + lane * 2);
        }
        __syncwarp();
    }
}

template <bool I8, int BN, bool TMA>
struct TcConfig {
    static constexpr uint32_t kStageB = BN * kBlockBytes;
    static constexpr uint32_t kStage = kStageA + kStageB;
    static constexpr uint32_t kRed = BN * kTileM * 4;  // partial sums for the cluster
    static constexpr int kStages = BN == 16 ? 5 : BN == 32 ? 4 : BN == 64 ? 7 : 4;
    static constexpr int kOut = BN >= 64 ? 8 : 4;  // warps that turn sums into output
    static constexpr int kLoaders = TMA ? 1 : 8;   // warps that fill the stages
    static constexpr int kThreads = 64 + 32 * kOut + (TMA ? 0 : 32 * kLoaders);
    static constexpr uint32_t kSmem = 1024 + kStages * kStage + kRed + 256;
    static constexpr uint32_t kTmemCols = 2 * BN < 32 ? 32 : 2 * BN;
};

// Warp 0 loads operand tiles by TMA (TMA false: the last 8 warps do, with plain loads, for
// rows TMA cannot take), warp 1 issues the MMAs into one of two accumulators, the warps from 2 on
// turn the other into output, 4 or 8 of them: a warp reaches 32 of the 128 lanes.  In a cluster of several CTAs every CTA sums its part of k, and the parts are
// added in rank order through distributed shared memory, each CTA finishing its share of columns:
// the result depends on neither timing nor the number of SMs.
template <bool I8, int LAYOUT, int BN, bool TMA>
__global__ void __launch_bounds__(TcConfig<I8, BN, TMA>::kThreads, 1)
    product_tc_kernel(const Product p, const bool bf16, const __grid_constant__ CUtensorMap tm_a,
                      const __grid_constant__ CUtensorMap tm_b) {
    using Cfg = TcConfig<I8, BN, TMA>;
    using T = std::conditional_t<I8, int8_t, uint16_t>;
    static_assert(LAYOUT != kMM || BN % 64 == 0, "dw's B comes in panels of 64");
    constexpr int STAGES = Cfg::kStages;
    constexpr int BK = I8 ? 128 : 64;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ Groups g;
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *sA = smem;
    uint8_t *sB = sA + STAGES * kStageA;
    uint32_t *red = reinterpret_cast<uint32_t *>(sB + STAGES * Cfg::kStageB);
    uint64_t *full = reinterpret_cast<uint64_t *>(reinterpret_cast<uint8_t *>(red) + Cfg::kRed);
    uint64_t *empty = full + STAGES;
    uint64_t *tfull = empty + STAGES;
    uint64_t *tempty = tfull + 2;
    uint64_t *drain = tempty + 2;
    uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(drain + 1);
    volatile uint32_t *abort_flag = tmem_holder + 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = emmy::cluster_ctarank(), split = emmy::cluster_nctarank();

    if (threadIdx.x == 64) {
        for (int s = 0; s < STAGES; ++s) {
            emmy::mbar_init(&full[s], Cfg::kLoaders);
            emmy::mbar_init(&empty[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            emmy::mbar_init(&tfull[a], 1);
            emmy::mbar_init(&tempty[a], Cfg::kOut);
        }
        emmy::mbar_init(drain, 1);
        *abort_flag = 0u;
        emmy::fence_barrier_init();
    }
    if (warp == 1) {
        emmy::tmem_alloc(tmem_holder, Cfg::kTmemCols);
        emmy::tmem_relinquish();
    }
    if (warp == 0) {
        if (TMA && lane == 0) {
            emmy::tma_prefetch(&tm_a);
            emmy::tma_prefetch(&tm_b);
        }
    }
    emmy::wait_for_prior_grid();
    if (warp == 0) load_groups(g, p, BN);
    emmy::tc_fence_before();
    __syncthreads();
    emmy::tc_fence_after();
    emmy::let_next_grid_start();
    const uint32_t tmem_base = *tmem_holder;

    const int mt = static_cast<int>((p.m + kTileM - 1) / kTileM), total = mt * g.tiles[p.experts];
    const int step = static_cast<int>(gridDim.x / split);
    uint32_t stage = 0, phase = 0, it = 0;
    uint32_t issued = 0u, parity_bits = 0u;  // producer: loads in flight for each stage and their parity
    bool ok = true;
    int e = 0;
    // Without a cluster each role runs through all of the CTA's tiles at its own pace; a cluster
    // takes one tile at a time, because its CTAs meet after each.
    for (int first = static_cast<int>(blockIdx.x / split); first < total; first += split > 1 ? step : total) {
        const int last = split > 1 ? first + 1 : total;
        if (TMA && warp == 0) {
            if (lane == 0) {
                for (int t = first; t < last && ok; t += step) {
                    const Tile w = tile_at(p, g, t, mt, e, kTileM, BN, BK, rank, split);
                    for (int kb = w.kb0; kb < w.kb1; ++kb) {
                        if (!emmy::mbar_wait(&empty[stage], phase ^ 1u, abort_flag, EMMY_STATUS_TIMEOUT_PRODUCER, kWaitNs)) {
                            ok = false;
                            break;
                        }
                        emmy::mbar_arrive_expect_tx(&full[stage], Cfg::kStage);
                        uint8_t *a = sA + stage * kStageA, *b = sB + stage * Cfg::kStageB;
                        const int k0 = kb * BK;
                        if constexpr (LAYOUT == kKK) {
                            emmy::tma_load_3d(a, &tm_a, &full[stage], k0, w.m0, w.e);
                        } else {
                            const int ka = LAYOUT == kMM ? w.begin + k0 : k0, ez = LAYOUT == kMM ? 0 : w.e;
                            emmy::tma_load_3d(a, &tm_a, &full[stage], w.m0, ka, ez);
                            emmy::tma_load_3d(a + kPanel, &tm_a, &full[stage], w.m0 + 64, ka, ez);
                        }
                        if constexpr (LAYOUT == kMM) {
                            #pragma unroll
                            for (int j = 0; j < BN / 64; ++j)
                                emmy::tma_load_2d(b + j * kPanel, &tm_b, &full[stage], w.c0 + 64 * j, w.begin + k0);
                        } else {
                            emmy::tma_load_2d(b, &tm_b, &full[stage], k0, w.begin + w.c0);
                        }
                        issued |= 1u << stage;
                        parity_bits = (parity_bits & ~(1u << stage)) | (phase << stage);
                        if (++stage == STAGES) {
                            stage = 0;
                            phase ^= 1u;
                        }
                    }
                }
            }
            __syncwarp();
        } else if (!TMA && warp >= 2 + Cfg::kOut) {
            // 256 threads: one unit of A (128 rows x 2 halves) and at most one of B each, the next
            // block's loads in flight while this block's are stored
            const int th = threadIdx.x - 64 - 32 * Cfg::kOut, half = th & 1;
            const uint8_t *a_lo = static_cast<const uint8_t *>(p.a), *a_hi = static_cast<const uint8_t *>(p.a_end);
            const uint8_t *b_lo = static_cast<const uint8_t *>(p.b), *b_hi = static_cast<const uint8_t *>(p.b_end);
            const bool has_b = th < 2 * BN;
            for (int t = first; t < last && ok; t += step) {
                const Tile w = tile_at(p, g, t, mt, e, kTileM, BN, BK, rank, split);
                const T *ae = static_cast<const T *>(p.a) + (p.dw ? w.begin * p.a_k : w.e * p.a_e);
                const T *be = static_cast<const T *>(p.b) + w.begin * (p.dw ? p.b_k : p.b_c);
                Unit ua, ub;
                const uint8_t *pa = nullptr, *pb = nullptr;
                int64_t na = 0, nb = 0;
                // where this thread's units of block kb lie, and how many of their bytes are wanted
                auto load = [&](int kb) {
                    const int64_t k0 = static_cast<int64_t>(kb) * BK, kleft = w.kend - k0;
                    const int64_t row = th >> 1, krow = row & 63, panel = row >> 6;
                    if constexpr (LAYOUT != kKK) {
                        const int64_t m = w.m0 + 64 * panel;
                        pa = reinterpret_cast<const uint8_t *>(ae + (k0 + krow) * p.a_k + m);
                        na = krow < kleft ? (p.m - m) * static_cast<int64_t>(sizeof(T)) : 0;
                    } else {
                        pa = reinterpret_cast<const uint8_t *>(ae + (w.m0 + row) * p.a_m + k0);
                        na = row < p.m - w.m0 ? kleft * static_cast<int64_t>(sizeof(T)) : 0;
                    }
                    pa += 64 * half;
                    na -= 64 * half;
                    load_unit(ua, pa, na, a_lo, a_hi);
                    if (!has_b) return;
                    if constexpr (LAYOUT == kMM) {
                        pb = reinterpret_cast<const uint8_t *>(be + (k0 + krow) * p.b_k + w.c0 + 64 * panel);
                        nb = krow < kleft ? (w.cols - 64 * panel) * static_cast<int64_t>(sizeof(T)) : 0;
                    } else {
                        pb = reinterpret_cast<const uint8_t *>(be + (w.c0 + row) * p.b_c + k0);
                        nb = row < w.cols ? kleft * static_cast<int64_t>(sizeof(T)) : 0;
                    }
                    pb += 64 * half;
                    nb -= 64 * half;
                    load_unit(ub, pb, nb, b_lo, b_hi);
                };
                if (w.kb0 < w.kb1) load(w.kb0);
                for (int kb = w.kb0; kb < w.kb1; ++kb) {
                    if (!emmy::mbar_wait(&empty[stage], phase ^ 1u, abort_flag, EMMY_STATUS_TIMEOUT_PRODUCER, kWaitNs)) {
                        ok = false;
                        break;
                    }
                    // a 128-row K-major tile and two 64-row panels are laid out alike
                    store_unit(ua, pa, na, sA + stage * kStageA, th >> 1, half);
                    if (has_b) store_unit(ub, pb, nb, sB + stage * Cfg::kStageB, th >> 1, half);
                    emmy::fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) emmy::mbar_arrive(&full[stage]);
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                    if (kb + 1 < w.kb1) load(kb + 1);
                }
            }
        } else if (warp == 1) {
            const Issue<I8, LAYOUT, false> issue(sA, sB, bf16, BN);
            for (int t = first; t < last && ok; t += step, ++it) {
                const Tile w = tile_at(p, g, t, mt, e, kTileM, BN, BK, rank, split);
                const uint32_t acc = it & 1u, aphase = (it >> 1) & 1u;
                ok = __all_sync(0xffffffffu, emmy::mbar_wait(&tempty[acc], aphase ^ 1u, abort_flag,
                                                             EMMY_STATUS_TIMEOUT_MMA, kWaitNs));
                if (!ok) break;
                emmy::tc_fence_after();
                const uint32_t d_tmem = tmem_base + acc * BN;
                const int blocks = uniform(w.kb1 - w.kb0), last_steps = uniform(last_block_steps(w, w.kb1, BK));
                for (int i = 0; i < blocks; ++i) {
                    ok = __all_sync(0xffffffffu, emmy::mbar_wait(&full[stage], phase, abort_flag,
                                                                 EMMY_STATUS_TIMEOUT_MMA, kWaitNs));
                    if (!ok) break;
                    const int steps = LAYOUT == kMM && i == blocks - 1 ? last_steps : 4;
                    if (LAYOUT == kMM && TMA && i == blocks - 1) {
                        // a block that ends inside: later rows belong to the next group (or hold
                        // anything), so what the last MMA takes of them becomes zero in both operands
                        const int have = min(BK, w.kend - (w.kb1 - 1) * BK);
                        if (have < steps * 16) {
                            uint8_t *a = sA + stage * kStageA, *b = sB + stage * Cfg::kStageB;
                            for (int j = 0; j < 2; ++j) zero_panel_rows(a + j * kPanel, have, steps * 16, lane);
                            for (int j = 0; j < BN / 64; ++j) zero_panel_rows(b + j * kPanel, have, steps * 16, lane);
                            emmy::fence_proxy_async();
                        }
                        __syncwarp();
                    }
                    emmy::tc_fence_after();
                    issue.block(d_tmem, stage * kStageA, stage * Cfg::kStageB, i > 0, steps);
                    issue.commit(&empty[stage]);
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (!ok) break;
                issue.commit(&tfull[acc]);
            }
            __syncwarp();
        } else if (warp >= 2 && warp < 2 + Cfg::kOut) {
            const int q = warp & 3, part = (warp - 2) >> 2;
            constexpr int PARTS = Cfg::kOut / 4, SPAN = BN / PARTS;
            for (int t = first; t < last && ok; t += step, ++it) {
                const Tile w = tile_at(p, g, t, mt, e, kTileM, BN, BK, rank, split);
                const uint32_t acc = it & 1u, aphase = (it >> 1) & 1u;
                if (!emmy::mbar_wait(&tfull[acc], aphase, abort_flag, EMMY_STATUS_TIMEOUT_EPILOGUE, kWaitNs)) {
                    ok = false;
                    break;
                }
                emmy::tc_fence_after();
                const uint32_t taddr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + acc * BN;
                const bool none = w.kb0 == w.kb1;  // nothing was accumulated
                if (BN >= 64 && split == 1) {
                    // the sums' exchange buffer is free without a cluster
                    store_tile<I8>(p, w, w.m0 + q * 32, taddr, none, part * SPAN, (part + 1) * SPAN,
                                   reinterpret_cast<uint8_t *>(red) + (warp - 2) * kStoreBytes, lane);
                } else {
                    // few columns, or parts of sums: channels of a column are neighbours either way
                    const int64_t m = w.m0 + q * 32 + lane;
                    Channel ch;
                    if (I8 && split == 1) ch = channel(p, w, m);
                    #pragma unroll 1
                    for (int c = part * SPAN; c < min((part + 1) * SPAN, w.cols); c += 16) {
                        uint32_t r[16];
                        emmy::tmem_ld_32x32b_x16(taddr + c, r);
                        emmy::tmem_ld_wait();
                        #pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            if (c + j >= w.cols) break;
                            const uint32_t v = none ? 0u : r[j];
                            if (split > 1)
                                red[(c + j) * kTileM + q * 32 + lane] = v;
                            else if (m < p.m)
                                store_out(p.out, p.out_type, out_index(p, w, m, c + j),
                                          scaled<I8>(v, I8 ? p.x_scale[w.begin + w.c0 + c + j] : 0.0f, ch));
                        }
                    }
                }
                emmy::tc_fence_before();
                __syncwarp();
                if (lane == 0) emmy::mbar_arrive(&tempty[acc]);
            }
        }
        if (split > 1) {
            __syncwarp();
            emmy::cluster_sync();  // every CTA's partial sums are in its shared memory
            if (warp >= 2 && warp < 2 + Cfg::kOut && ok) {
                const Tile w = tile_at(p, g, first, mt, e, kTileM, BN, BK, rank, split);
                const int lm = (warp & 3) * 32 + lane, part = (warp - 2) >> 2, parts = Cfg::kOut / 4;
                const int64_t m = w.m0 + lm;
                if (m < p.m) {
                    Channel ch;
                    if constexpr (I8) ch = channel(p, w, m);
                    for (int c = rank + split * part; c < w.cols; c += split * parts) {
                        uint32_t sum = 0u;  // 0 of either type
                        for (uint32_t s = 0; s < split; ++s) {
                            const uint32_t v = emmy::ld_cluster_u32(emmy::mapa(&red[c * kTileM + lm], s));
                            sum = I8 ? sum + v : __float_as_uint(__uint_as_float(sum) + __uint_as_float(v));
                        }
                        store_out(p.out, p.out_type, out_index(p, w, m, c),
                                  scaled<I8>(sum, I8 ? p.x_scale[w.begin + w.c0 + c] : 0.0f, ch));
                    }
                }
            }
            __syncwarp();
            emmy::cluster_sync();  // and may be overwritten
        }
    }

    if (TMA && warp == 0 && lane == 0 && !ok) {
        // this CTA's own loads still in flight land before it leaves (bounded)
        volatile uint32_t never = 0u;
        for (int s = 0; s < STAGES; ++s)
            if (issued & (1u << s)) emmy::mbar_wait(&full[s], (parity_bits >> s) & 1u, &never, 0u, 20000000ull);
    }
    if (warp == 1) {
        // every MMA has finished before tensor memory is released (bounded); committed by the lane
        // that issued them
        emmy::umma_commit_if<false>(emmy::elect_one(), emmy::smem_u32(drain));
        volatile uint32_t never = 0u;
        emmy::mbar_wait(drain, 0u, &never, 0u, 20000000ull);
        __syncwarp();
    }
    emmy::tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        emmy::tc_fence_after();
        emmy::tmem_dealloc(tmem_base, Cfg::kTmemCols);
    }
}

// ---------------------------------------------------------------- CTA pairs
//
// For groups of many rows: 256 channels x BN rows of output on a pair of CTAs.  Each CTA loads its
// 128 channels of A and its half of B's rows, the leader issues cta_group::2 MMAs over both CTAs'
// shared memory, and each CTA turns its own 128 lanes into output while the next tile accumulates.
// A pair moves 64 bytes into shared memory per SM and clock of MMA (BN = 256), half of what a
// single CTA's 128 x 128 tile needs - more than L2 delivers.

template <int BN>
struct PairConfig {
    static constexpr uint32_t kStageB = BN / 2 * kBlockBytes;
    static constexpr uint32_t kStage = kStageA + kStageB;
    static constexpr int kStages = BN == 256 ? 6 : 8;
    static constexpr int kOut = 8;  // warps that turn sums into output
    static constexpr int kThreads = 64 + 32 * kOut;
    static constexpr uint32_t kSmem = 1024 + kStages * kStage + kOut * kStoreBytes + 512;
};

template <bool I8, int LAYOUT, int BN>
__global__ void __launch_bounds__(PairConfig<BN>::kThreads, 1)
    product_pair_kernel(const Product p, const bool bf16, const __grid_constant__ CUtensorMap tm_a,
                        const __grid_constant__ CUtensorMap tm_b) {
    using Cfg = PairConfig<BN>;
    constexpr int STAGES = Cfg::kStages, BK = I8 ? 128 : 64, CN = BN / 2;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ Groups g;
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *sA = smem;
    uint8_t *sB = sA + STAGES * kStageA;
    uint8_t *sStore = sB + STAGES * Cfg::kStageB;
    uint64_t *full = reinterpret_cast<uint64_t *>(sStore + Cfg::kOut * kStoreBytes);
    uint64_t *empty = full + STAGES;
    uint64_t *tfull = empty + STAGES;
    uint64_t *tempty = tfull + 2;
    uint64_t *drain = tempty + 2;
    uint64_t *tail = drain + 1;       // this CTA's loads of a block that ends inside
    // the peer's are in and their spare rows zeroed (leader only); one for each stage, because the
    // peer may be several blocks ahead, but never twice on one stage
    uint64_t *tail_peer = tail + 1;
    uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(tail_peer + STAGES);
    volatile uint32_t *abort_flag = tmem_holder + 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = emmy::cluster_ctarank();

    if (threadIdx.x == 64) {
        for (int s = 0; s < STAGES; ++s) {
            emmy::mbar_init(&full[s], 1);
            emmy::mbar_init(&empty[s], 1);
            emmy::mbar_init(&tail_peer[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            emmy::mbar_init(&tfull[a], 1);
            emmy::mbar_init(&tempty[a], 2 * Cfg::kOut);
        }
        emmy::mbar_init(drain, 1);
        emmy::mbar_init(tail, 1);
        *abort_flag = 0u;
        emmy::fence_barrier_init();
    }
    if (warp == 1) {
        emmy::tmem_alloc_pair(tmem_holder, 2 * BN);
        emmy::tmem_relinquish_pair();
    }
    if (warp == 0) {
        if (lane == 0) {
            emmy::tma_prefetch(&tm_a);
            emmy::tma_prefetch(&tm_b);
        }
    }
    emmy::wait_for_prior_grid();
    if (warp == 0) load_groups(g, p, BN);
    emmy::tc_fence_before();
    __syncthreads();
    emmy::cluster_sync();  // the peer signals the leader's barriers only after both are initialised
    emmy::tc_fence_after();
    const uint32_t tmem_base = *tmem_holder;
    emmy::let_next_grid_start();
    const int mt = static_cast<int>((p.m + 2 * kTileM - 1) / (2 * kTileM)), total = mt * g.tiles[p.experts];
    const int pair = static_cast<int>(blockIdx.x >> 1), npairs = static_cast<int>(gridDim.x >> 1);
    int e = 0;
    auto tile = [&](int t) {
        Tile o = tile_at(p, g, t, mt, e, 2 * kTileM, BN, BK, 0, 1);
        o.m0 += static_cast<int>(rank) * kTileM;  // this CTA's channels
        return o;
    };

    if (warp == 0) {
        // ---------------- loads (both CTAs; completion counted on the leader's barrier)
        uint32_t stage = 0, phase = 0, tails = 0;
        uint32_t peer_parity = 0u;  // of tail_peer, one bit for each stage
        uint32_t issued = 0u, parity_bits = 0u;
        bool ok = true;
        const uint32_t leader_full = emmy::mapa(&full[0], 0), own_tail = emmy::mapa(tail, rank);
        // One block's loads, completing on the barrier at cluster address `bar`; one thread.
        auto load = [&](const Tile &w, int kb, uint32_t bar) {
            uint8_t *a = sA + stage * kStageA, *b = sB + stage * Cfg::kStageB;
            const int k0 = kb * BK, c0 = w.c0 + static_cast<int>(rank) * CN;
            if constexpr (LAYOUT == kKK) {
                emmy::tma_load_3d_pair(a, &tm_a, bar, k0, w.m0, w.e);
            } else {
                const int ka = LAYOUT == kMM ? w.begin + k0 : k0, ez = LAYOUT == kMM ? 0 : w.e;
                emmy::tma_load_3d_pair(a, &tm_a, bar, w.m0, ka, ez);
                emmy::tma_load_3d_pair(a + kPanel, &tm_a, bar, w.m0 + 64, ka, ez);
            }
            if constexpr (LAYOUT == kMM) {
                #pragma unroll
                for (int j = 0; j < CN / 64; ++j)
                    emmy::tma_load_2d_pair(b + j * kPanel, &tm_b, bar, c0 + 64 * j, w.begin + k0);
            } else {
                emmy::tma_load_2d_pair(b, &tm_b, bar, k0, w.begin + c0);
            }
        };
        auto next = [&]() {
            if (++stage == STAGES) {
                stage = 0;
                phase ^= 1u;
            }
        };
        for (int t = pair; t < total && ok; t += npairs) {
            const Tile w = tile(t);
            const int whole = LAYOUT == kMM ? w.kend / BK : w.kb1;
            if (lane == 0) {
                for (int kb = 0; kb < whole; ++kb) {
                    if (!emmy::mbar_wait_cluster(&empty[stage], phase ^ 1u, abort_flag, EMMY_STATUS_TIMEOUT_PRODUCER, kWaitNs)) {
                        ok = false;
                        break;
                    }
                    if (rank == 0) {
                        emmy::mbar_arrive_expect_tx(&full[stage], 2u * Cfg::kStage);
                        issued |= 1u << stage;
                        parity_bits = (parity_bits & ~(1u << stage)) | (phase << stage);
                    }
                    load(w, kb, leader_full + stage * 8u);
                    next();
                }
            }
            if constexpr (LAYOUT == kMM) {
                // A last block that ends inside: later rows belong to the next group (or hold
                // anything), and what the last MMA takes of them becomes zero in both operands
                // before the leader's barrier completes.  The whole warp does that.
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                stage = __shfl_sync(0xffffffffu, stage, 0);
                phase = __shfl_sync(0xffffffffu, phase, 0);
                if (whole == w.kb1) continue;
                ok = emmy::mbar_wait_cluster(&empty[stage], phase ^ 1u, abort_flag, EMMY_STATUS_TIMEOUT_PRODUCER, kWaitNs);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                if (lane == 0) {
                    emmy::mbar_arrive_expect_tx(tail, Cfg::kStage);
                    load(w, whole, own_tail);
                }
                __syncwarp();
                ok = emmy::mbar_wait_cluster(tail, tails & 1u, abort_flag, EMMY_STATUS_TIMEOUT_PRODUCER, kWaitNs);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                ++tails;
                const int have = w.kend - whole * BK, upto = (have + 15) / 16 * 16;
                for (int j = 0; j < 2; ++j) zero_panel_rows(sA + stage * kStageA + j * kPanel, have, upto, lane);
                for (int j = 0; j < CN / 64; ++j)
                    zero_panel_rows(sB + stage * Cfg::kStageB + j * kPanel, have, upto, lane);
                emmy::fence_proxy_async();
                __syncwarp();
                if (rank == 1) {
                    if (lane == 0) emmy::mbar_arrive_cluster(emmy::mapa(&tail_peer[stage], 0));
                } else {
                    ok = emmy::mbar_wait_cluster(&tail_peer[stage], peer_parity >> stage & 1u, abort_flag,
                                                 EMMY_STATUS_TIMEOUT_PRODUCER, kWaitNs);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    peer_parity ^= 1u << stage;
                    if (lane == 0) emmy::mbar_arrive(&full[stage]);
                }
                next();
            }
        }
        if (!ok && rank == 0 && lane == 0) {
            // loads still in flight land before the pair leaves (bounded)
            volatile uint32_t never = 0u;
            for (int s = 0; s < STAGES; ++s)
                if (issued & (1u << s)) emmy::mbar_wait_cluster(&full[s], (parity_bits >> s) & 1u, &never, 0u, 20000000ull);
        }
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0) {
            // ---------------- MMA issuer (leader only)
            const Issue<I8, LAYOUT, true> issue(sA, sB, bf16, BN);
            uint32_t stage = 0, phase = 0, it = 0;
            bool ok = true;
            for (int t = pair; t < total && ok; t += npairs, ++it) {
                const Tile w = tile(t);
                const uint32_t acc = it & 1u, aphase = (it >> 1) & 1u;
                ok = __all_sync(0xffffffffu, emmy::mbar_wait_cluster(&tempty[acc], aphase ^ 1u, abort_flag,
                                                                     EMMY_STATUS_TIMEOUT_MMA, kWaitNs));
                if (!ok) break;
                emmy::tc_fence_after();
                const uint32_t d_tmem = tmem_base + acc * BN;
                const int blocks = uniform(w.kb1), last_steps = uniform(last_block_steps(w, w.kb1, BK));
                for (int i = 0; i < blocks; ++i) {
                    ok = __all_sync(0xffffffffu, emmy::mbar_wait_cluster(&full[stage], phase, abort_flag,
                                                                         EMMY_STATUS_TIMEOUT_MMA, kWaitNs));
                    if (!ok) break;
                    emmy::tc_fence_after();
                    issue.block(d_tmem, stage * kStageA, stage * Cfg::kStageB, i > 0,
                                LAYOUT == kMM && i == blocks - 1 ? last_steps : 4);
                    issue.commit(&empty[stage]);
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (!ok) break;
                issue.commit(&tfull[acc]);
            }
            // arrives on both CTAs once every pair MMA has finished
            issue.commit(drain);
        }
        __syncwarp();
    } else {
        // ---------------- output (both CTAs): own 128 channels of the tile
        const int q = warp & 3, part = (warp - 2) >> 2;
        constexpr int SPAN = BN / (Cfg::kOut / 4);
        const uint32_t leader_tempty = emmy::mapa(&tempty[0], 0);
        uint32_t it = 0;
        for (int t = pair; t < total; t += npairs, ++it) {
            const Tile w = tile(t);
            const uint32_t acc = it & 1u, aphase = (it >> 1) & 1u;
            if (!emmy::mbar_wait_cluster(&tfull[acc], aphase, abort_flag, EMMY_STATUS_TIMEOUT_EPILOGUE, kWaitNs)) break;
            emmy::tc_fence_after();
            store_tile<I8>(p, w, w.m0 + q * 32, tmem_base + (static_cast<uint32_t>(q * 32) << 16) + acc * BN, w.kb1 == 0,
                           part * SPAN, (part + 1) * SPAN, sStore + (warp - 2) * kStoreBytes, lane);
            emmy::tc_fence_before();
            __syncwarp();
            if (lane == 0) emmy::mbar_arrive_cluster(leader_tempty + acc * 8u);
        }
    }
    emmy::tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        // the last MMA, and the leader's last commit into this CTA, have landed (bounded)
        if (lane == 0) {
            volatile uint32_t never = 0u;
            emmy::mbar_wait_cluster(drain, 0u, &never, 0u, kWaitNs);
        }
        __syncwarp();
    }
    emmy::cluster_sync();  // no CTA leaves while its peer may still signal or read it
    if (warp == 1) {
        emmy::tc_fence_after();
        emmy::tmem_dealloc_pair(tmem_base, 2 * BN);
    }
}

}  // namespace
