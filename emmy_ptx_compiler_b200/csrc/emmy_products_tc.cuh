// Products on the 5th-generation tensor cores: out(c, m) = sum_k A(m, k) B(c, k).
//
// The output's contiguous axis m (the channels) lies on the 128 lanes of tensor memory and the
// output's rows c (the tokens of a group) on the N columns of the instruction, 16 to 256 of them.
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

// 32 lanes x 16 consecutive 32-bit columns, back into tensor memory.
__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void st_cluster_u32(uint32_t cluster_addr, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr), "r"(v) : "memory");
}

// The two halves of cluster_sync().
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

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

constexpr uint64_t kWaitNs = 2000000000ull;  // a wait for one block or one tile's way out: orders of magnitude above any legal one
// A wait for whole sums may last as long as their blocks do, at 20 us each (0.3 to 2 us measured).
__device__ __forceinline__ uint64_t sum_wait_ns(uint64_t blocks) { return kWaitNs + blocks * 20000ull; }
constexpr int kTileM = 128;
constexpr uint32_t kBlockBytes = 128;                  // one 128-byte swizzle row of k (or of m, c)
constexpr uint32_t kPanel = 64 * kBlockBytes;          // 64 k x 64 m (or c) of an MN-major 16-bit operand
constexpr uint32_t kStageA = kTileM * kBlockBytes;

struct Flags {
    bool bf16;            // 16-bit operands are bf16, else f16
    bool tma_a, tma_b;    // TMA can load the operand
};

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

// Tile t of the launch (tm x col_tile; host code keeps the tiles within 31 bits), for a whole warp.
// `e` is a cursor: tiles of one caller come in ascending order, and each step looks 32 experts
// ahead.  A cluster of `split` CTAs divides the sum.
__device__ __forceinline__ Tile tile_at(const Product &p, const Groups &g, int t, int mt, int &e, int tm, int col_tile,
                                        int bk, uint32_t rank, uint32_t split) {
    for (const int lane = threadIdx.x & 31;; e += 32) {
        const int i = e + 1 + lane;
        const uint32_t past = __ballot_sync(0xffffffffu, i > p.experts || t < mt * g.tiles[min(i, p.experts)]);
        if (past) {
            e += __ffs(past) - 1;
            break;
        }
    }
    const int begin = g.row[e], count = g.row[e + 1] - begin;
    const uint32_t r = t - mt * g.tiles[e], ct = g.tiles[e + 1] - g.tiles[e];
    const uint32_t sweep = ct == 1 ? r / kSweep : r / kSweep / ct, in = r - sweep * kSweep * ct, first = sweep * kSweep;
    const uint32_t wide = min(static_cast<uint32_t>(kSweep), mt - first);
    const uint32_t ci = ct == 1 ? 0 : wide == kSweep ? in / kSweep : in / wide;
    Tile o;
    o.e = e;
    o.begin = begin;
    o.m0 = static_cast<int>(first + in - ci * wide) * tm;
    o.c0 = static_cast<int>(ci) * col_tile;
    o.cols = min(col_tile, (p.dw ? static_cast<int>(p.c) : count) - o.c0);
    o.kend = p.dw ? count : static_cast<int>(p.k);
    const uint32_t nkb = static_cast<uint32_t>(o.kend + bk - 1) / bk;
    // split is a power of two
    o.kb0 = static_cast<int>(nkb * rank >> (31 - __clz(split)));
    o.kb1 = static_cast<int>(nkb * (rank + 1) >> (31 - __clz(split)));
    return o;
}

// Operands that TMA cannot address (rows that start off a 16-byte boundary): each 16-byte chunk of the
// swizzled operand is cut out of the two aligned 16-byte words that it lies in.  A word is read
// whole where it lies inside the operand, whichever of its bytes are wanted; at the operand's two
// ends it is put together from its bytes.
__device__ __noinline__ uint4 load_edge_word(const uint8_t *at, const uint8_t *lo, const uint8_t *hi) {
    alignas(16) uint8_t v[16];
    for (int i = 0; i < 16; ++i) v[i] = at + i >= lo && at + i < hi ? at[i] : 0;
    return *reinterpret_cast<const uint4 *>(v);
}

// Rows of an operand's block: row r at `src` + r * `stride` bytes, of which `valid` bytes are wanted in
// the first `rows` of them.
struct Rows {
    const uint8_t *src, *lo, *hi;
    int64_t stride, valid, rows;
};

// The first `keep` bytes of a word (below 0 counts as 0).
__device__ __forceinline__ uint32_t keep_bytes(uint32_t v, int keep) {
    return keep >= 4 ? v : keep <= 0 ? 0u : v & ((1u << (8 * keep)) - 1u);
}

// N rows from `r0` on into the swizzled 128-byte rows of `operand`, zeros where nothing is wanted; one
// warp, 8 lanes to a row.  All loads are issued before the first is used, unless some word of the
// warp lies across an end of the operand.
template <int N>
__device__ __forceinline__ void copy_rows(const Rows &b, int r0, uint8_t *operand, int lane) {
    constexpr int K = N / 4;
    const int valid = static_cast<int>(b.valid < 128 ? b.valid : 128), j = lane & 7, have = valid - 16 * j;
    const int rows = static_cast<int>(b.rows < r0 + N ? b.rows : r0 + N);
    const uint32_t low = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(b.src)), low_stride = static_cast<uint32_t>(b.stride);
    uint4 w0[K], w1[K];
    bool edge = false;
    const uint8_t *src = b.src + (r0 + (lane >> 3)) * b.stride + 16 * j;
    #pragma unroll
    for (int k = 0; k < K; ++k, src += 4 * b.stride) {
        const int row = r0 + (lane >> 3) + 4 * k, off = static_cast<int>(low + row * low_stride) & 15;
        const uint8_t *at = src - off;
        const bool first = row < rows && have > 0, second = first && off + have > 16 && off > 0;
        edge |= first && (at < b.lo || at + (second ? 32 : 16) > b.hi);
    }
    if (!__any_sync(0xffffffffu, edge)) {
        src = b.src + (r0 + (lane >> 3)) * b.stride + 16 * j;
        #pragma unroll
        for (int k = 0; k < K; ++k, src += 4 * b.stride) {
            const int row = r0 + (lane >> 3) + 4 * k, off = static_cast<int>(low + row * low_stride) & 15;
            const uint4 *at = reinterpret_cast<const uint4 *>(src - off);
            const bool first = row < rows && have > 0, second = first && off + have > 16 && off > 0;
            w0[k] = first ? __ldg(at) : make_uint4(0, 0, 0, 0);
            w1[k] = second ? __ldg(at + 1) : make_uint4(0, 0, 0, 0);
        }
    } else {
        #pragma unroll
        for (int k = 0; k < K; ++k) {
            const int row = r0 + (lane >> 3) + 4 * k, off = static_cast<int>(low + row * low_stride) & 15;
            const uint8_t *at = b.src + row * b.stride + 16 * j - off;
            const bool first = row < rows && have > 0;
            w0[k] = first ? load_edge_word(at, b.lo, b.hi) : make_uint4(0, 0, 0, 0);
            w1[k] = first ? load_edge_word(at + 16, b.lo, b.hi) : make_uint4(0, 0, 0, 0);
        }
    }
    #pragma unroll
    for (int k = 0; k < K; ++k) {
        const int row = r0 + (lane >> 3) + 4 * k;
        const uint32_t off = low + row * low_stride;  // its low 4 bits count
        const uint32_t a[8] = {w0[k].x, w0[k].y, w0[k].z, w0[k].w, w1[k].x, w1[k].y, w1[k].z, w1[k].w};
        uint32_t h[6], v[5], c[4];
        #pragma unroll
        for (int q = 0; q < 6; ++q) h[q] = off & 8u ? a[q + 2] : a[q];
        #pragma unroll
        for (int q = 0; q < 5; ++q) v[q] = off & 4u ? h[q + 1] : h[q];
        #pragma unroll
        for (int q = 0; q < 4; ++q) {
            c[q] = __funnelshift_r(v[q], v[q + 1], (off & 3u) * 8u);
            if (have < 16) c[q] = keep_bytes(c[q], have - 4 * q);
        }
        *reinterpret_cast<uint4 *>(operand + row * kBlockBytes + ((j ^ (row & 7)) << 4)) = make_uint4(c[0], c[1], c[2], c[3]);
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

// Scale of a channel, and its bias; loaded before the sums are ready.
struct Channel {
    float scale = 0.0f, bias = 0.0f;
};
template <bool I8>
__device__ __forceinline__ Channel channel(const Product &p, const Tile &t, int64_t m) {
    Channel c;
    if (I8 && m < p.m) {
        c.scale = p.w_scale[t.e * p.m + m];
        if (p.bias) c.bias = p.bias[t.e * p.m + m];
    }
    return c;
}

// Scales of N x 32 output rows from `from` on, lane l holding those of rows 32 i + l.
template <bool I8, int N>
struct RowScales {
    float v[N];
    __device__ __forceinline__ RowScales(const Product &p, const Tile &t, int from, int lane) {
        #pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = from + 32 * i + lane;
            v[i] = I8 && c < t.cols ? p.x_scale[t.begin + t.c0 + c] : 0.0f;
        }
    }
    // of row `i` of the first 32
    __device__ __forceinline__ float at(int i) const { return I8 ? __shfl_sync(0xffffffffu, v[0], i) : 0.0f; }
    __device__ __forceinline__ void next() {
        #pragma unroll
        for (int i = 0; i + 1 < N; ++i) v[i] = v[i + 1];
    }
};

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
// 16 bytes at a time (4 stores for 32 rows instead of 32, and the conversion packs two values).
// f32 outputs need no help: 32 lanes write 128 bytes of a row.  The next columns come from tensor
// memory while these are stored.  A 32 x 32 piece takes a warp about 800 cycles (300 to convert, 180
// through stmatrix, 330 for the reads and stores); TMA stores of two 32 x 16 pieces took 1250, most of
// it in issuing them from one lane.
// `empty`: the sum had no terms.
template <bool I8, int N>
__device__ __forceinline__ void store_tile(const Product &p, const Tile &w, int mq, uint32_t taddr, bool empty, int from,
                                           int to, const Channel &own, RowScales<I8, N> xs, uint8_t *buf, int lane) {
    if (p.out_type == EMMY_F32) {
        const int64_t m = mq + lane;
        float *out = static_cast<float *>(p.out) + out_index(p, w, m, from);
        uint32_t r[32];
        if (from < to) emmy::tmem_ld_32x32b_x32(taddr + from, r);
        #pragma unroll 1
        for (int c = from; c < to; c += 32, out += 32 * p.out_c, xs.next()) {
            float v[32];
            emmy::tmem_ld_wait();
            #pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = scaled<I8>(empty ? 0u : r[j], xs.at(j), own);
            if (c + 32 < to) emmy::tmem_ld_32x32b_x32(taddr + c + 32, r);  // on their way while these are stored
            float *o = out;
            #pragma unroll
            for (int j = 0; j < 32; ++j, o += p.out_c)
                if (m < p.m && c + j < to) *o = v[j];
        }
        return;
    }
    const int piece = lane & 3, row4 = lane >> 2;
    const bool vec = (reinterpret_cast<uintptr_t>(p.out) & 15) == 0 && ((p.out_c | p.out_e | p.m) & 7) == 0;
    const bool bf16 = p.out_type == EMMY_BF16, in = vec ? mq + piece * 8 < p.m : mq + lane < p.m;
    const int64_t step8 = 8 * p.out_c;
    uint16_t *out = static_cast<uint16_t *>(p.out) +
                    (vec ? out_index(p, w, mq + piece * 8, from + row4) : out_index(p, w, mq + lane, from));
    Channel ch[4];
    if constexpr (I8) {
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            ch[i].scale = __shfl_sync(0xffffffffu, own.scale, lane / 4 + 8 * i);
            ch[i].bias = __shfl_sync(0xffffffffu, own.bias, lane / 4 + 8 * i);
        }
    }
    const uint32_t put = emmy::smem_u32(buf) + ((lane >> 4) * 8 + (lane & 7)) * kStoreRow + 16 * ((lane >> 3) & 1);
    const uint8_t *get = buf + row4 * kStoreRow + piece * 16;
    uint32_t r[2][16];
    if (from < to) {
        emmy::tmem_ld_16x256b_x4(taddr + from, r[0]);
        emmy::tmem_ld_16x256b_x4(taddr + (16u << 16) + from, r[1]);
    }
    #pragma unroll 1
    for (int c = from; c < to; c += 32, xs.next()) {
        uint32_t v[2][8];
        float x[8];
        #pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = xs.at(8 * (i >> 1) + 2 * piece + (i & 1));
        emmy::tmem_ld_wait();
        if (empty) {
            #pragma unroll
            for (int i = 0; i < 16; ++i) r[0][i] = r[1][i] = 0u;
        }
        #pragma unroll
        for (int h = 0; h < 2; ++h) {
            #pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int row = 2 * h + (i & 1), col = i >> 1 << 1;
                v[h][i] = pack16(bf16, scaled<I8>(r[h][2 * i], x[col], ch[row]), scaled<I8>(r[h][2 * i + 1], x[col + 1], ch[row]));
            }
        }
        if (c + 32 < to) {  // on their way while these are stored
            emmy::tmem_ld_16x256b_x4(taddr + c + 32, r[0]);
            emmy::tmem_ld_16x256b_x4(taddr + (16u << 16) + c + 32, r[1]);
        }
        #pragma unroll
        for (int h = 0; h < 2; ++h) {
            emmy::stmatrix_x4_trans(put + 32 * h, v[h][0], v[h][1], v[h][2], v[h][3]);
            emmy::stmatrix_x4_trans(put + 32 * h + 16 * kStoreRow, v[h][4], v[h][5], v[h][6], v[h][7]);
        }
        __syncwarp();
        if (vec) {
            uint4 q[4];
            #pragma unroll
            for (int i = 0; i < 4; ++i) q[i] = *reinterpret_cast<const uint4 *>(get + i * 8 * kStoreRow);
            #pragma unroll
            for (int i = 0; i < 4; ++i, out += step8)
                if (in && c + i * 8 + row4 < to) *reinterpret_cast<uint4 *>(out) = q[i];
        } else {
            for (int i = 0; i < 32; ++i, out += p.out_c)
                if (in && c + i < to) *out = *reinterpret_cast<const uint16_t *>(buf + i * kStoreRow + lane * 2);
        }
        __syncwarp();
    }
}

// Tensor cores cut off what lies below the last bit of a running sum, so a long sum of one sign would
// lose up to half a step for each MMA (262144 rows of positive values: 1.5e-3 of their sum).  So sums of
// 16-bit products are joined from segments, added in f32 to nearest by the warps that turn sums into
// output: up to 768 terms for an f32 output (0.7e-6 off for bf16 and 1.0e-6 for f16 values of either sign, 1.3e-6 and
// 4.4e-6 for values of one), up to 8192 where rounding to 16 bits follows (5e-5 of a sum of one sign; half a
// step is 4.9e-4 or 3.9e-3).  Kernels with JOIN do so, at 0 to 6 % more time (dw of 16384 rows each of 4
// experts [2048, 2048]: 383 against 377 us to bf16, 386 against 381 to f32; 7108 rows, 24 experts [1416, 1000] to
// f32: 44 against 41 us); where no sum of a launch can be that long the others run.
constexpr int kShortSegment = 12, kLongSegment = 128;  // blocks
__host__ __device__ constexpr int segment_blocks(int out_type) { return out_type == EMMY_F32 ? kShortSegment : kLongSegment; }
// Segments of a sum after the first, and the blocks of each: as equal as they can be.
__device__ __forceinline__ int more_segments(int blocks, int segment) { return blocks > segment ? (blocks - 1) / segment : 0; }
__device__ __forceinline__ int equal_segment(int blocks, int segment) {
    const int n = more_segments(blocks, segment) + 1;
    return (blocks + n - 1) / n;
}

// The barriers of a tile's accumulators: segment `it` of a CTA's tiles arrives in accumulator `it` & 1.
template <bool PAIR>
struct Accumulators {
    uint64_t *full, *empty;  // it is complete; it may be overwritten (PAIR: the leader's counts)
    volatile uint32_t *abort_flag;

    __device__ __forceinline__ bool wait(uint32_t it, int blocks) const {
        uint64_t *bar = &full[it & 1u];
        const uint32_t phase = (it >> 1) & 1u;
        const bool ok = PAIR ? emmy::mbar_wait_cluster(bar, phase, abort_flag, EMMY_STATUS_TIMEOUT_EPILOGUE, sum_wait_ns(blocks))
                             : emmy::mbar_wait(bar, phase, abort_flag, EMMY_STATUS_TIMEOUT_EPILOGUE, sum_wait_ns(blocks));
        if (!__all_sync(0xffffffffu, ok)) return false;
        emmy::tc_fence_after();
        return true;
    }
    __device__ __forceinline__ void release(uint32_t it, int lane) const {
        emmy::tc_fence_before();
        __syncwarp();
        if (lane == 0) {
            if constexpr (PAIR) emmy::mbar_arrive_cluster(emmy::mapa(&empty[it & 1u], 0));
            else emmy::mbar_arrive(&empty[it & 1u]);
        }
    }
};

// The sum of the segments `it` to `it` + `more` of a tile, for a warp's 32 channels and the SPAN columns
// from `taddr` of the first accumulator on (the second one is BN columns further), left in the columns behind
// both.  Every accumulator is released.
template <int BN, int SPAN, bool PAIR>
__device__ __forceinline__ bool join_segments(uint32_t taddr, const Accumulators<PAIR> acc, uint32_t it, int more, int lane) {
    const uint32_t whole = taddr + 2 * BN;
    #pragma unroll 1
    for (int s = 0; s <= more; ++s, ++it) {
        if (!acc.wait(it, kLongSegment)) return false;
        #pragma unroll 1
        for (int c = 0; c < SPAN; c += 16) {
            uint32_t r[16], sum[16];
            emmy::tmem_ld_32x32b_x16(taddr + (it & 1u) * BN + c, r);
            if (s > 0) emmy::tmem_ld_32x32b_x16(whole + c, sum);
            emmy::tmem_ld_wait();
            #pragma unroll
            for (int j = 0; j < 16; ++j)
                if (s > 0) r[j] = __float_as_uint(__uint_as_float(sum[j]) + __uint_as_float(r[j]));
            emmy::tmem_st_32x32b_x16(whole + c, r);
        }
        emmy::tmem_st_wait();
        acc.release(it, lane);
    }
    return true;
}

// Out of line, for kernels whose warps that load leave few registers.
template <int BN, int SPAN, bool PAIR>
__device__ __noinline__ bool join_segments_apart(uint32_t taddr, const Accumulators<PAIR> acc, uint32_t it, int more, int lane) {
    return join_segments<BN, SPAN, PAIR>(taddr, acc, it, more, lane);
}

// The same where two accumulators take all of tensor memory: the sum waits in registers.  The last segment's
// accumulator is not released.  STEP: columns of a read (the compiler keeps all in registers at 16 where the sum
// is stored from there, and at 32 where it goes back).
template <int BN, int SPAN, int STEP, bool PAIR>
__device__ __forceinline__ bool sum_segments(float (&sum)[SPAN], uint32_t taddr, const Accumulators<PAIR> &acc, uint32_t it, int more,
                                             int lane) {
    #pragma unroll
    for (int c = 0; c < SPAN; ++c) sum[c] = 0.0f;
    #pragma unroll 1
    for (int s = 0;; ++s, ++it) {
        if (!acc.wait(it, kLongSegment)) return false;
        #pragma unroll
        for (int c = 0; c < SPAN; c += STEP) {
            uint32_t r[STEP];
            if constexpr (STEP == 32) emmy::tmem_ld_32x32b_x32(taddr + (it & 1u) * BN + c, r);
            else emmy::tmem_ld_32x32b_x16(taddr + (it & 1u) * BN + c, r);
            emmy::tmem_ld_wait();
            #pragma unroll
            for (int j = 0; j < STEP; ++j) sum[c + j] += __uint_as_float(r[j]);
        }
        if (s == more) return true;
        acc.release(it, lane);
    }
}

// And put back into the last segment's accumulator.
template <int BN, int SPAN, bool PAIR>
__device__ __forceinline__ bool join_segments_wide(uint32_t taddr, const Accumulators<PAIR> &acc, uint32_t it, int more, int lane) {
    float sum[SPAN];
    if (!sum_segments<BN, SPAN, 32, PAIR>(sum, taddr, acc, it, more, lane)) return false;
    #pragma unroll
    for (int c = 0; c < SPAN; c += 16) {
        uint32_t r[16];
        #pragma unroll
        for (int j = 0; j < 16; ++j) r[j] = __float_as_uint(sum[c + j]);
        emmy::tmem_st_32x32b_x16(taddr + ((it + more) & 1u) * BN + c, r);
    }
    emmy::tmem_st_wait();
    return true;
}

// Send 16 columns' sums from `c` on, for one channel, to the CTAs that finish them: 16 / G columns to
// each of G.  `own`: this rank's place in a CTA's exchange buffer, in bytes.
template <int G>
__device__ __forceinline__ void send_columns(const uint32_t *red, uint32_t own, uint32_t share, int share_log, int c,
                                             int cols, const uint32_t (&r)[16], bool none) {
    #pragma unroll
    for (int d = 0; d < G; ++d) {
        const int first = c + d * (16 / G);
        if (first >= cols) break;
        const uint32_t at = emmy::mapa(red, first >> share_log) + own + (first & (share - 1)) * kTileM * 4;
        #pragma unroll
        for (int j = 0; j < 16 / G; ++j)
            if (first + j < cols) emmy::st_cluster_u32(at + j * kTileM * 4, none ? 0u : r[d * (16 / G) + j]);
    }
}

template <bool I8, int BN, bool TMA>
struct TcConfig {
    static constexpr uint32_t kStageB = BN * kBlockBytes;
    static constexpr uint32_t kStage = kStageA + kStageB;
    static constexpr uint32_t kRed = BN * kTileM * 4;  // partial sums for the cluster
    static constexpr uint32_t kOutStage = BN >= 64 ? 4 * kStoreBytes * (TMA ? 2 : 1) : 0;
    static constexpr int kStages = BN == 16 ? 5 : BN == 32 ? 4 : BN == 64 ? 6 : 4;
    static constexpr int kOut = BN >= 64 && TMA ? 8 : 4;  // warps that turn sums into output
    // two teams on alternate blocks hide more of the loads' latency (8 rows of 8 experts, int8 [3425,
    // 4057]: 94 against 125 us); with both operands 128 rows high they lack the registers (dw
    // [777, 1001] of 1022 rows: 54 against 38 us)
    static constexpr int kTeams = BN <= 64 ? 2 : 1;
    static constexpr int kLoaders = TMA ? 0 : 8 * kTeams;  // warps that load without TMA, 8 to a block
    static constexpr int kThreads = 64 + 32 * (kOut + kLoaders);
    static constexpr uint32_t kSmem = 1024 + kStages * kStage + kRed + kOutStage + 256;
    static constexpr int kPerSm = TMA && BN <= 32 ? 2 : 1;  // CTAs that share an SM
    // two accumulators and the columns of a third, in a power of two
    static constexpr uint32_t kTmemCols = 4 * BN;
};

// One CTA on 128 channels x BN rows of output.  Warp 0 loads operand tiles by TMA (TMA false: the
// last warps load those operands whose rows TMA cannot take), warp 1 issues the MMAs into one of two
// accumulators, the warps from 2 on turn the other into output, 4 or 8 of them: a warp reaches 32 of
// the 128 lanes.
//
// With BN of 16 or 32, for groups of a few rows, this is bound by reading the weights: 64 experts
// [2048, 4096] for 512 rows take 168 us, 6.4 TB/s.  Two CTAs share an SM, so that one's loads cover
// the other's start and end.  Where there are fewer tiles than SMs a cluster of CTAs divides each
// sum: one token of 8 experts [1024, 2048] takes 10 us in quarters against 13 undivided.  Each CTA
// sums its part of k and the parts are added in rank order: a CTA finishes its share of the
// columns, for which the others send their parts through distributed shared memory, so the result
// depends on no timing.
//
// Tensor memory is held from start to end, and the CTAs of a cluster wait for each other.  Two
// kernels that did so with more than 512 columns between them on one SM could block each other.  Shared
// memory rules that out: a CTA with tiles of 16 or 32 rows (64 or 128 columns, up to 108 KB) leaves room for one
// more of them or for one CTA of the attention family with at most 256 columns, and every CTA with
// wider tiles, of the GEMM family or of the attention family with 512 columns takes 129 KB or more.
template <bool I8, int LAYOUT, int BN, bool TMA, bool JOIN>
__global__ void __launch_bounds__(TcConfig<I8, BN, TMA>::kThreads, TcConfig<I8, BN, TMA>::kPerSm)
    product_tc_kernel(const Product p, const Flags flags, const __grid_constant__ CUtensorMap tm_a,
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
    uint8_t *out_stage = reinterpret_cast<uint8_t *>(red) + Cfg::kRed;
    uint64_t *full = reinterpret_cast<uint64_t *>(out_stage + Cfg::kOutStage);
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
            emmy::mbar_init(&full[s], 1 + Cfg::kLoaders / Cfg::kTeams);
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
        if (lane == 0) {
            if (TMA || flags.tma_a) emmy::tma_prefetch(&tm_a);
            if (TMA || flags.tma_b) emmy::tma_prefetch(&tm_b);
        }
    }
    emmy::wait_for_prior_grid();
    if (warp == 0) load_groups(g, p, BN);
    emmy::tc_fence_before();
    __syncthreads();
    emmy::tc_fence_after();
    emmy::let_next_grid_start();
    const uint32_t tmem_base = *tmem_holder;
    bool met = split == 1;  // the cluster's other CTAs have started: their shared memory may be written
    if (!met) emmy::cluster_arrive();

    const int mt = static_cast<int>((p.m + kTileM - 1) / kTileM), total = mt * g.tiles[p.experts];
    const int step = static_cast<int>(gridDim.x / split);
    uint32_t stage = 0, phase = 0, it = 0;
    uint32_t issued = 0u, parity_bits = 0u;  // producer: loads in flight for each stage and their parity
    bool ok = true;
    const uint32_t share = BN / split, share_log = 31 - __clz(share);  // columns of a tile that each CTA finishes
    int e = 0;
    // Without a cluster each role runs through all of the CTA's tiles at its own pace; a cluster
    // takes one tile at a time, because its CTAs meet after each.
    for (int first = static_cast<int>(blockIdx.x / split); first < total; first += split > 1 ? step : total) {
        const int last = split > 1 ? first + 1 : total;
        if (warp == 0) {
            const bool ta = TMA || flags.tma_a, tb = TMA || flags.tma_b;
            const uint32_t bytes = (ta ? kStageA : 0) + (tb ? Cfg::kStageB : 0);
            for (int t = first; t < last && ok; t += step) {
                const Tile w = tile_at(p, g, t, mt, e, kTileM, BN, BK, rank, split);
                if (lane == 0) {
                    for (int kb = w.kb0; kb < w.kb1; ++kb) {
                        if (!emmy::mbar_wait(&empty[stage], phase ^ 1u, abort_flag, EMMY_STATUS_TIMEOUT_PRODUCER, kWaitNs)) {
                            ok = false;
                            break;
                        }
                        emmy::mbar_arrive_expect_tx(&full[stage], bytes);
                        uint8_t *a = sA + stage * kStageA, *b = sB + stage * Cfg::kStageB;
                        const int k0 = kb * BK;
                        if constexpr (LAYOUT == kKK) {
                            if (ta) emmy::tma_load_3d(a, &tm_a, &full[stage], k0, w.m0, w.e);
                        } else if (ta) {
                            const int ka = LAYOUT == kMM ? w.begin + k0 : k0, ez = LAYOUT == kMM ? 0 : w.e;
                            emmy::tma_load_3d(a, &tm_a, &full[stage], w.m0, ka, ez);
                            emmy::tma_load_3d(a + kPanel, &tm_a, &full[stage], w.m0 + 64, ka, ez);
                        }
                        if constexpr (LAYOUT != kMM) {
                            if (tb) emmy::tma_load_2d(b, &tm_b, &full[stage], k0, w.begin + w.c0);
                        } else if (tb) {
                            #pragma unroll
                            for (int j = 0; j < BN / 64; ++j)
                                emmy::tma_load_2d(b + j * kPanel, &tm_b, &full[stage], w.c0 + 64 * j, w.begin + k0);
                        }
                        issued |= 1u << stage;
                        parity_bits = (parity_bits & ~(1u << stage)) | (phase << stage);
                        if (++stage == STAGES) {
                            stage = 0;
                            phase ^= 1u;
                        }
                    }
                }
                ok = __all_sync(0xffffffffu, ok);
            }
        } else if (!TMA && warp >= 2 + Cfg::kOut) {
            // Two teams of 8 warps take every other block, so that one's loads are on their way while
            // the other's are put in place.  A warp has 16 rows of A and BN / 8 of B; rows run along
            // m (c), or along k in panels of 64.
            const int lw = warp - 2 - Cfg::kOut, slot0 = (lw & 7) * 16, slotb0 = (lw & 7) * (BN / 8);
            const uint32_t team = lw >> 3;
            const bool has_a = !flags.tma_a, has_b = !flags.tma_b;
            constexpr int64_t ES = sizeof(T);
            for (int t = first; t < last && ok; t += step) {
                const Tile w = tile_at(p, g, t, mt, e, kTileM, BN, BK, rank, split);
                const T *ae = static_cast<const T *>(p.a) + (p.dw ? w.begin * p.a_k : w.e * p.a_e);
                const T *be = static_cast<const T *>(p.b) + w.begin * (p.dw ? p.b_k : p.b_c);
                auto rows_a = [&](int kb) {
                    const int64_t k0 = static_cast<int64_t>(kb) * BK, kleft = w.kend - k0;
                    Rows r;
                    r.lo = static_cast<const uint8_t *>(p.a);
                    r.hi = static_cast<const uint8_t *>(p.a_end);
                    if constexpr (LAYOUT == kKK) {
                        r.src = reinterpret_cast<const uint8_t *>(ae + w.m0 * p.a_m + k0);
                        r.stride = p.a_m * ES, r.valid = kleft * ES, r.rows = p.m - w.m0;
                    } else {
                        // this warp's 16 rows lie in one panel
                        const int64_t m = w.m0 + (slot0 & 64);
                        r.src = reinterpret_cast<const uint8_t *>(ae + (k0 - (slot0 & 64)) * p.a_k + m);
                        r.stride = p.a_k * ES, r.valid = (p.m - m) * ES, r.rows = kleft + (slot0 & 64);
                    }
                    return r;
                };
                auto rows_b = [&](int kb) {
                    const int64_t k0 = static_cast<int64_t>(kb) * BK, kleft = w.kend - k0;
                    Rows r;
                    r.lo = static_cast<const uint8_t *>(p.b);
                    r.hi = static_cast<const uint8_t *>(p.b_end);
                    if constexpr (LAYOUT != kMM) {
                        r.src = reinterpret_cast<const uint8_t *>(be + w.c0 * p.b_c + k0);
                        r.stride = p.b_c * ES, r.valid = kleft * ES, r.rows = w.cols;
                    } else {
                        const int64_t c = slotb0 & 64;
                        r.src = reinterpret_cast<const uint8_t *>(be + (k0 - c) * p.b_k + w.c0 + c);
                        r.stride = p.b_k * ES, r.valid = (w.cols - c) * ES, r.rows = kleft + c;
                    }
                    return r;
                };
                for (int kb = w.kb0; kb < w.kb1; ++kb, ++it) {
                    // `it` counts this CTA's blocks
                    const uint32_t s = it % STAGES, sphase = it / STAGES & 1u;
                    if (it % Cfg::kTeams != team) continue;
                    ok = __all_sync(0xffffffffu, emmy::mbar_wait(&empty[s], sphase ^ 1u, abort_flag,
                                                                 EMMY_STATUS_TIMEOUT_PRODUCER, kWaitNs));
                    if (!ok) break;
                    if (has_a) copy_rows<16>(rows_a(kb), slot0, sA + s * kStageA, lane);
                    if (has_b) copy_rows<(BN >= 32 ? BN / 8 : 4)>(rows_b(kb), slotb0, sB + s * Cfg::kStageB, lane);
                    emmy::fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) emmy::mbar_arrive(&full[s]);
                }
            }
        } else if (warp == 1) {
            const Issue<I8, LAYOUT, false> issue(sA, sB, flags.bf16, BN);
            uint32_t d_tmem = tmem_base;
            // waits for the accumulator of the tile's (segment's) sum
            auto begin = [&] {
                ok = __all_sync(0xffffffffu, emmy::mbar_wait(&tempty[it & 1u], (it >> 1 & 1u) ^ 1u, abort_flag,
                                                             EMMY_STATUS_TIMEOUT_MMA, kWaitNs));
                emmy::tc_fence_after();
                d_tmem = tmem_base + (it & 1u) * BN;
            };
            for (int t = first; t < last && ok; t += step, ++it) {
                const Tile w = tile_at(p, g, t, mt, e, kTileM, BN, BK, rank, split);
                const int blocks = uniform(w.kb1 - w.kb0), last_steps = uniform(last_block_steps(w, w.kb1, BK));
                const int segment = JOIN ? uniform(equal_segment(blocks, segment_blocks(p.out_type))) : 0;
                begin();
                if (!ok) break;
                for (int i = 0, from = 0; i < blocks; ++i) {
                    if (JOIN && i == from + segment) {
                        issue.commit(&tfull[it & 1u]);
                        ++it;
                        from = i;
                        begin();
                        if (!ok) break;
                    }
                    ok = __all_sync(0xffffffffu, emmy::mbar_wait(&full[stage], phase, abort_flag,
                                                                 EMMY_STATUS_TIMEOUT_MMA, kWaitNs));
                    if (!ok) break;
                    const int steps = LAYOUT == kMM && i == blocks - 1 ? last_steps : 4;
                    if (LAYOUT == kMM && i == blocks - 1) {
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
                    issue.block(d_tmem, stage * kStageA, stage * Cfg::kStageB, i > from, steps);
                    issue.commit(&empty[stage]);
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (!ok) break;
                issue.commit(&tfull[it & 1u]);
            }
            __syncwarp();
        } else if (warp >= 2 && warp < 2 + Cfg::kOut) {
            const int q = warp & 3, part = (warp - 2) >> 2;
            constexpr int SPAN = BN / (Cfg::kOut / 4);
            const Accumulators<false> acc{tfull, tempty, abort_flag};
            for (int t = first; t < last && ok; t += step, ++it) {
                const Tile w = tile_at(p, g, t, mt, e, kTileM, BN, BK, rank, split);
                const int64_t m = w.m0 + q * 32 + lane;
                const Channel ch = channel<I8>(p, w, m);
                RowScales<I8, (SPAN + 31) / 32> xs(p, w, part * SPAN, lane);
                const uint32_t lanes = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
                const int more = JOIN ? more_segments(w.kb1 - w.kb0, segment_blocks(p.out_type)) : 0;
                if constexpr (JOIN)
                    ok = TMA ? join_segments<BN, SPAN, false>(lanes + part * SPAN, acc, it, more, lane)
                             : join_segments_apart<BN, SPAN, false>(lanes + part * SPAN, acc, it, more, lane);
                else
                    ok = acc.wait(it, w.kb1 - w.kb0);
                if (!ok) break;
                it += more;
                const uint32_t taddr = lanes + (JOIN ? 2u : it & 1u) * BN;
                const bool none = w.kb0 == w.kb1;  // nothing was accumulated
                if (BN >= 64 && split == 1) {
                    store_tile<I8>(p, w, w.m0 + q * 32, taddr, none, part * SPAN, min((part + 1) * SPAN, w.cols), ch, xs,
                                   out_stage + (warp - 2) * kStoreBytes, lane);
                } else {
                    // few columns, or parts of sums: channels of a column are neighbours either way
                    if (!met) {
                        emmy::cluster_wait();
                        met = true;
                    }
                    const uint32_t own = (rank * share * kTileM + q * 32 + lane) * 4;
                    #pragma unroll 1
                    for (int c = part * SPAN; c < min((part + 1) * SPAN, w.cols); c += 16) {
                        uint32_t r[16];
                        emmy::tmem_ld_32x32b_x16(taddr + c, r);
                        emmy::tmem_ld_wait();
                        if (split > 1) {
                            if (share >= 16) send_columns<1>(red, own, share, share_log, c, w.cols, r, none);
                            else if (share == 8) send_columns<2>(red, own, share, share_log, c, w.cols, r, none);
                            else if (share == 4) send_columns<4>(red, own, share, share_log, c, w.cols, r, none);
                            else send_columns<8>(red, own, share, share_log, c, w.cols, r, none);
                        } else {
                            #pragma unroll
                            for (int j = 0; j < 16; ++j) {
                                const float v = scaled<I8>(none ? 0u : r[j], xs.at((c & 16) + j), ch);
                                if (m < p.m && c + j < w.cols)
                                    store_out(p.out, p.out_type, out_index(p, w, m, c + j), v);
                            }
                        }
                    }
                }
                if (!JOIN) acc.release(it, lane);
            }
        }
        if (split > 1) {
            // the columns that this CTA finishes, their scales loaded before the parts arrive
            const bool out_warp = warp >= 2 && warp < 2 + Cfg::kOut && ok;
            const int lm = (warp & 3) * 32 + lane, part = (warp - 2) >> 2, parts = Cfg::kOut / 4;
            const int from = static_cast<int>(rank * share);
            Tile w{};
            Channel ch;
            float xs = 0.0f;
            if (out_warp) {
                w = tile_at(p, g, first, mt, e, kTileM, BN, BK, rank, split);
                ch = channel<I8>(p, w, w.m0 + lm);
                if (I8 && from + lane < w.cols) xs = p.x_scale[w.begin + w.c0 + from + lane];
            }
            __syncwarp();
            if (!met) {
                emmy::cluster_wait();
                met = true;
            }
            emmy::cluster_sync();  // this CTA's columns have arrived from every rank
            if (out_warp && BN >= 64) {
                // sums go back to tensor memory, where a whole tile's would be, and leave the same way
                const uint32_t acc = (it - 1) & 1u;
                const uint32_t taddr = tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16) + acc * BN;
                const int span = max(static_cast<int>(share) / parts, 32), begin = from + part * span;
                const int to = min(min(begin + span, from + static_cast<int>(share)), w.cols);
                #pragma unroll 1
                for (int c = begin; c < to; c += 16) {
                    uint32_t sum[16];
                    const uint32_t *at = red + (c - from) * kTileM + lm;
                    #pragma unroll
                    for (int j = 0; j < 16; ++j) sum[j] = at[j * kTileM];
                    for (uint32_t s = 1; s < split; ++s) {
                        at += share * kTileM;
                        #pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const uint32_t v = at[j * kTileM];
                            sum[j] = I8 ? sum[j] + v : __float_as_uint(__uint_as_float(sum[j]) + __uint_as_float(v));
                        }
                    }
                    emmy::tmem_st_32x32b_x16(taddr + c, sum);
                }
                emmy::tmem_st_wait();
                __syncwarp();
                if (begin < to) {
                    const RowScales<I8, 2> scales(p, w, begin, lane);
                    store_tile<I8>(p, w, w.m0 + (warp & 3) * 32, taddr, false, begin, to, ch, scales,
                                   out_stage + (warp - 2) * kStoreBytes, lane);
                }
            } else if (out_warp) {
                const int64_t m = w.m0 + lm;
                const int to = min(from + static_cast<int>(share), w.cols);
                #pragma unroll 4
                for (int c = from; c < to; ++c) {
                    const uint32_t *at = red + (c - from) * kTileM + lm;
                    uint32_t v[8], sum = 0u;  // 0 of either type
                    #pragma unroll
                    for (int s = 0; s < 8; ++s) v[s] = s < split ? at[s * share * kTileM] : 0u;
                    #pragma unroll
                    for (int s = 0; s < 8; ++s)
                        if (s < split)
                            sum = I8 ? sum + v[s] : __float_as_uint(__uint_as_float(sum) + __uint_as_float(v[s]));
                    const float x = I8 ? __shfl_sync(0xffffffffu, xs, c - from) : 0.0f;
                    if (m < p.m) store_out(p.out, p.out_type, out_index(p, w, m, c), scaled<I8>(sum, x, ch));
                }
            }
            if (first + step < total) {
                __syncwarp();
                emmy::cluster_sync();  // and may be overwritten
            }
        }
    }
    if (!met) {
        __syncwarp();
        emmy::cluster_wait();
    }

    if (warp == 0 && lane == 0 && !ok) {
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
// single CTA's 128 x 128 tile needs.
//
// Bound by the tensor cores where sums are long: 16384 rows, 4 experts [4096, 4096], take 347 us (1.58
// PFLOP/s bf16), int8 8192^3 takes 326 us (3.38 POP/s).  Sums of a few blocks are bound by the way
// out (a 32 x 32 piece of a tile takes its warp 800 cycles): 8192 rows, 32 experts, dx [1024, 512] 20 us.
// Measured on the way: 6 stages against 4, 352 against 382 us for the first of these; MMAs issued
// from a branch of one lane, with their operands moved to uniform registers one by one, 590 cycles a
// block against 512 of MMA.

template <int BN>
struct PairConfig {
    static constexpr uint32_t kStageB = BN / 2 * kBlockBytes;
    static constexpr uint32_t kStage = kStageA + kStageB;
    static constexpr int kStages = BN == 256 ? 6 : 8;
    static constexpr uint32_t kTmemCols = 512;  // two accumulators, and the columns of a third of 128
    static constexpr int kOut = 8;  // warps that turn sums into output
    static constexpr int kThreads = 64 + 32 * kOut;
    static constexpr int kTailThreads = 32;  // dw: one more warp
    static constexpr uint32_t kSmem = 1024 + kStages * kStage + kOut * kStoreBytes + 512;
};

// DIRECT: f32 outputs of kernels with JOIN whose sums wait in registers.
template <bool I8, int LAYOUT, int BN, bool JOIN, bool DIRECT = false>
__global__ void __launch_bounds__(PairConfig<BN>::kThreads + (LAYOUT == kMM ? PairConfig<BN>::kTailThreads : 0), 1)
    product_pair_kernel(const Product p, const Flags flags, const __grid_constant__ CUtensorMap tm_a,
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
    uint64_t *tail = drain + 1;  // for each stage: this CTA's loads of a block that ends inside
    uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(tail + STAGES);
    volatile uint32_t *abort_flag = tmem_holder + 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = emmy::cluster_ctarank();

    if (threadIdx.x == 64) {
        for (int s = 0; s < STAGES; ++s) {
            emmy::mbar_init(&full[s], LAYOUT == kMM ? 2 : 1);  // dw: one arrival for each CTA
            emmy::mbar_init(&empty[s], 1);
            emmy::mbar_init(&tail[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            emmy::mbar_init(&tfull[a], 1);
            emmy::mbar_init(&tempty[a], 2 * Cfg::kOut);
        }
        emmy::mbar_init(drain, 1);
        *abort_flag = 0u;
        emmy::fence_barrier_init();
    }
    if (warp == 1) {
        emmy::tmem_alloc_pair(tmem_holder, Cfg::kTmemCols);
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
        uint32_t stage = 0, phase = 0;
        uint32_t issued = 0u, parity_bits = 0u, tail_issued = 0u, tail_uses = 0u;
        bool ok = true;
        const uint32_t leader_full = emmy::mapa(&full[0], 0), own_tail = emmy::mapa(&tail[0], rank);
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
        for (int t = pair; t < total && ok; t += npairs) {
            const Tile w = tile(t);
            if (lane == 0) {
                for (int kb = 0; kb < w.kb1; ++kb) {
                    if (!emmy::mbar_wait_cluster(&empty[stage], phase ^ 1u, abort_flag, EMMY_STATUS_TIMEOUT_PRODUCER, kWaitNs)) {
                        ok = false;
                        break;
                    }
                    if (LAYOUT == kMM && w.kend - kb * BK < BK) {
                        // ends inside: the tail warp passes it on
                        emmy::mbar_arrive_expect_tx(&tail[stage], Cfg::kStage);
                        load(w, kb, own_tail + stage * 8u);
                        tail_issued |= 1u << stage;
                        tail_uses ^= 1u << stage;
                    } else {
                        if (rank == 0) {
                            emmy::mbar_arrive_expect_tx(&full[stage], 2u * Cfg::kStage);
                            if (LAYOUT == kMM) emmy::mbar_arrive(&full[stage]);
                            issued |= 1u << stage;
                            parity_bits = (parity_bits & ~(1u << stage)) | (phase << stage);
                        }
                        load(w, kb, leader_full + stage * 8u);
                    }
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            ok = __all_sync(0xffffffffu, ok);
        }
        if (!ok && lane == 0) {
            // loads still in flight land before the pair leaves (bounded)
            volatile uint32_t never = 0u;
            for (int s = 0; s < STAGES; ++s) {
                if (issued & (1u << s)) emmy::mbar_wait_cluster(&full[s], (parity_bits >> s) & 1u, &never, 0u, 20000000ull);
                if (tail_issued & (1u << s))
                    emmy::mbar_wait_cluster(&tail[s], (tail_uses >> s & 1u) ^ 1u, &never, 0u, 20000000ull);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0) {
            // ---------------- MMA issuer (leader only)
            const Issue<I8, LAYOUT, true> issue(sA, sB, flags.bf16, BN);
            uint32_t stage = 0, phase = 0, it = 0;
            bool ok = true;
            uint32_t d_tmem = tmem_base;
            auto begin = [&] {
                ok = __all_sync(0xffffffffu, emmy::mbar_wait_cluster(&tempty[it & 1u], (it >> 1 & 1u) ^ 1u, abort_flag,
                                                                     EMMY_STATUS_TIMEOUT_MMA, kWaitNs));
                emmy::tc_fence_after();
                d_tmem = tmem_base + (it & 1u) * BN;
            };
            for (int t = pair; t < total && ok; t += npairs, ++it) {
                const Tile w = tile(t);
                const int blocks = uniform(w.kb1), last_steps = uniform(last_block_steps(w, w.kb1, BK));
                const int segment = JOIN ? uniform(equal_segment(blocks, segment_blocks(p.out_type))) : 0;
                begin();
                if (!ok) break;
                for (int i = 0, from = 0; i < blocks; ++i) {
                    if (JOIN && i == from + segment) {
                        issue.commit(&tfull[it & 1u]);
                        ++it;
                        from = i;
                        begin();
                        if (!ok) break;
                    }
                    ok = __all_sync(0xffffffffu, emmy::mbar_wait_cluster(&full[stage], phase, abort_flag,
                                                                         EMMY_STATUS_TIMEOUT_MMA, kWaitNs));
                    if (!ok) break;
                    emmy::tc_fence_after();
                    issue.block(d_tmem, stage * kStageA, stage * Cfg::kStageB, i > from,
                                LAYOUT == kMM && i == blocks - 1 ? last_steps : 4);
                    issue.commit(&empty[stage]);
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (!ok) break;
                issue.commit(&tfull[it & 1u]);
            }
            // arrives on both CTAs once every pair MMA has finished
            issue.commit(drain);
        }
        __syncwarp();
    } else if (LAYOUT == kMM && warp == 2 + Cfg::kOut) {
        // ---------------- blocks that end inside (both CTAs): the rows behind the end belong to the
        // next group, or hold anything.  What the last MMA takes of them becomes zero in both
        // operands before the leader's barrier completes, while the loads run on.
        uint32_t blocks = 0, tail_parity = 0u;  // of `tail`, one bit for each stage
        uint64_t span = 0;  // what a wait lasts: every sum since the last tile that ended inside, and its way out
        for (int t = pair; t < total; t += npairs) {
            const Tile w = tile(t);
            blocks += w.kb1;
            span += w.kb1 + 1;
            const int have = w.kend % BK;
            if (have == 0) continue;
            const uint32_t stage = (blocks - 1) % STAGES;
            if (!__all_sync(0xffffffffu, emmy::mbar_wait_cluster(&tail[stage], tail_parity >> stage & 1u, abort_flag,
                                                                 EMMY_STATUS_TIMEOUT_PRODUCER, sum_wait_ns(span))))
                break;
            span = 0;
            tail_parity ^= 1u << stage;
            const int upto = (have + 15) / 16 * 16;
            for (int j = 0; j < 2; ++j) zero_panel_rows(sA + stage * kStageA + j * kPanel, have, upto, lane);
            for (int j = 0; j < CN / 64; ++j) zero_panel_rows(sB + stage * Cfg::kStageB + j * kPanel, have, upto, lane);
            emmy::fence_proxy_async();
            __syncwarp();
            if (lane == 0) emmy::mbar_arrive_cluster(emmy::mapa(&full[stage], 0));
        }
        __syncwarp();
    } else {
        // ---------------- output (both CTAs): own 128 channels of the tile
        const int q = warp & 3, part = (warp - 2) >> 2;
        constexpr int SPAN = BN / (Cfg::kOut / 4);
        const Accumulators<true> acc{tfull, tempty, abort_flag};
        uint32_t it = 0;
        for (int t = pair; t < total; t += npairs, ++it) {
            const Tile w = tile(t);
            const Channel ch = channel<I8>(p, w, w.m0 + q * 32 + lane);
            const RowScales<I8, SPAN / 32> xs(p, w, part * SPAN, lane);
            const uint32_t lanes = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
            const int more = JOIN ? more_segments(w.kb1, segment_blocks(p.out_type)) : 0, from = part * SPAN, m = w.m0 + q * 32;
            if constexpr (DIRECT) {
                // f32 sums leave from registers while the next tile's segments go on
                float sum[SPAN], *out = static_cast<float *>(p.out) + out_index(p, w, m + lane, from);
                const int cols = m + lane < p.m ? w.cols - from : 0;
                if (!sum_segments<BN, SPAN, 16, true>(sum, lanes + from, acc, it, more, lane)) break;
                it += more;
                acc.release(it, lane);
                #pragma unroll
                for (int c = 0; c < SPAN; ++c, out += p.out_c)
                    if (c < cols) *out = w.kb1 == 0 ? 0.0f : sum[c];
            } else {
                constexpr bool WIDE = 3 * BN > 512;
                bool ok;
                if constexpr (JOIN && !WIDE)
                    ok = join_segments<BN, SPAN, true>(lanes + from, acc, it, more, lane);
                else if (JOIN && more)
                    ok = join_segments_wide<BN, SPAN, true>(lanes + from, acc, it, more, lane);
                else
                    ok = acc.wait(it, w.kb1);
                if (!ok) break;
                it += more;
                store_tile<I8>(p, w, m, lanes + (JOIN && !WIDE ? 2u : it & 1u) * BN, w.kb1 == 0, from, min(from + SPAN, w.cols), ch,
                               xs, sStore + (warp - 2) * kStoreBytes, lane);
                if (!JOIN || WIDE) acc.release(it, lane);
            }
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
        emmy::tmem_dealloc_pair(tmem_base, Cfg::kTmemCols);
    }
}

}  // namespace
