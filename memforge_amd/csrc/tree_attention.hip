// Attention for trees of drafted tokens over the paged cache.
//
// Sequence s has ctx tokens in the pool and n nodes whose keys and values are rows
// of the call. Node i sees the context, itself and its ancestors:
//     out = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q.k_j)
// with grouped heads. A (node, head) pair is a column; the G heads of a kv head
// share its K/V rows, so a kv head's n G columns are one matrix product with them.
//
// Work. A sequence's keys are tiles of 32: the context's, then the nodes'. All
// sequences' tiles stand in one line, which is cut into equal shares; each share has
// a workgroup for every lane, a (kv head, group of columns). It runs the pieces of
// the sequences that the share covers, writes the whole ones out and leaves the
// others' unnormalised sums for merge_tree_kernel. So one long context and a batch
// of uneven ones both fill the GPU, from lengths that only the device knows: the
// plan (tree_plan_kernel, once for all layers of a step) is made there. The lanes of
// a share stand side by side, so that the kv heads of a slot, which lie together in
// memory, are read at the same time (a share of one head's tiles of its own: 377 us
// for 358 in the first case below, 145 for 133 in the second).
//
// Bound. Two layers with their plan, by graph replay on an MI355X: 64 contexts (median
// 2,048, 16 nodes each, bf16, 40/8 heads of 128) 360 us, 327 with loads and merges
// alone; their keys and values at the 4.9 TB/s of a large copy take 304. One context
// of 32,001 under 48 nodes (fp16, the same heads) 132 us, 93 without the products and
// 123 without the loads, floor 54: 240 columns a kv head, whose chain of product,
// softmax, product the two waves of a SIMD do not hide from each other.
//
// Tiles. Four or eight waves, WC side by side on blocks of 32 columns and WK along
// the keys: a stage of WK or more tiles goes from global memory straight into LDS once
// for all columns; a ring of stages keeps loads in flight. S^T = K Q^T, softmax with
// a lazily moved maximum, O^T += V^T P^T in 32x32 MFMA blocks whose operands need no
// move between lanes: as attn_wide_body (attn_kernels.h) lays them out.
#include <algorithm>
#include <cmath>

#include "attn_kernels.h"

namespace mf {
namespace {

typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;

// As ld_lds16, for rows that are read once: past what the caches hold (two layers of 64
// contexts of a median of 2048 at 40/8 x 128: 428 -> 381 us with plan and merges).
__device__ __forceinline__ void ld_lds16_nt(const void* gsrc, uint32_t lds_addr) {
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, off nt" ::"{m0}"(lds_addr), "v"(gsrc) : "memory");
}

constexpr int kTreeThreads = 256;
constexpr int kTile = 32;            // keys
constexpr int kMaxSeqs = 4096;
constexpr int kWindow = 1024;        // block-table entries held in LDS
constexpr int kMaxWild = 1 + MF_TREE_MAX_NODES / kTile;  // a context's last tile, and the nodes' tiles
constexpr int kSeqInts = 8;          // context, nodes, first row, tiles, column groups, context tiles, -, -
constexpr int kWorkInts = 16;        // a worker's first sequence, kv head, first tile, tiles, the sequence's six, column group

struct TreePlanArgs {
    const int32_t* parents;
    const int32_t* cu_nodes;
    const int32_t* ctx_lens;
    int num_seqs;
    int64_t num_rows;
    int max_nodes, mask_words;
    int64_t max_context;
    int group;        // query heads of a kv head
    int num_kv_heads;
    int group_cols;   // columns of one column group
    int lanes;        // (kv head, column group)s: workers of one share
    int num_shares, min_share;
    int64_t* head;      // share, all tiles
    int32_t* seqs;
    int64_t* seq_first; // first tile of each sequence in the line
    int32_t* work;
    uint32_t* masks;
    int64_t* positions;
};

__device__ __forceinline__ void seq_shape(const TreePlanArgs& a, int s, int& ctx, int& n, int64_t& row0) {
    row0 = a.cu_nodes[s];
    const int64_t rows = a.cu_nodes[s + 1] - row0;
    n = (int)min(rows, (int64_t)a.max_nodes);
    if (row0 < 0 || rows < 0 || row0 + n > a.num_rows) n = 0;
    ctx = (int)min((int64_t)max(a.ctx_lens[s], 0), a.max_context);
}

// Positions of no sequence's rows.
__global__ __launch_bounds__(kTreeThreads) void clear_positions_kernel(int64_t* positions, int64_t num_rows) {
    for (int64_t r = (int64_t)blockIdx.x * kTreeThreads + threadIdx.x; r < num_rows; r += (int64_t)gridDim.x * kTreeThreads)
        positions[r] = 0;
}

// Block 0 lays the tiles out; block 1 + s writes sequence s's masks and positions. Rows that are no
// node's have position 0, so that what follows may look it up: block 1 + s writes those of its
// own rows (past max_nodes, or of a tree that has none), block 0 those before and behind all trees.
__global__ __launch_bounds__(kTreeThreads) void tree_plan_kernel(TreePlanArgs a) {
    __shared__ int64_t first[kMaxSeqs + 1];
    __shared__ int64_t waves[kTreeThreads / 64];
    __shared__ int rows_lo[kTreeThreads / 64], rows_hi[kTreeThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (blockIdx.x > 0) {
        int* up = (int*)first;
        const int s = blockIdx.x - 1;
        int ctx, n;
        int64_t row0;
        seq_shape(a, s, ctx, n, row0);
        for (int i = tid; i < n; i += kTreeThreads) {
            const int p = a.parents[row0 + i];
            up[i] = p >= 0 && p < i ? p : -1;
        }
        __syncthreads();
        // ancestors come in falling order, so a node's words are finished one after the other
        for (int i = tid; i < n; i += kTreeThreads) {
            uint32_t* row = a.masks + (row0 + i) * a.mask_words;
            for (int w = a.mask_words - 1; w > i >> 5; --w) row[w] = 0;
            int depth = 0, word = i >> 5;
            uint32_t bits = 0;
            for (int at = i;; at = up[at]) {
                while (at < 0 ? word >= 0 : at >> 5 < word) {
                    row[word--] = bits;
                    bits = 0;
                }
                if (at < 0) break;
                bits |= 1u << (at & 31);
                ++depth;
            }
            a.positions[row0 + i] = (int64_t)ctx + depth - 1;
        }
        const int64_t last = min((int64_t)a.cu_nodes[s + 1], a.num_rows);
        for (int64_t r = max(row0, (int64_t)0) + n + tid; r < last; r += kTreeThreads) a.positions[r] = 0;
        return;
    }
    const int per = (a.num_seqs + kTreeThreads - 1) / kTreeThreads;
    const int s0 = min(tid * per, a.num_seqs), s1 = min(s0 + per, a.num_seqs);
    int64_t mine = 0;
    int row_lo = INT_MAX, row_hi = INT_MIN;  // of the numbers in cu_nodes
    for (int s = s0; s < s1; ++s) {
        int ctx, n;
        int64_t row0;
        seq_shape(a, s, ctx, n, row0);
        const int row1 = a.cu_nodes[s + 1];
        row_lo = min(row_lo, min((int)row0, row1));
        row_hi = max(row_hi, max((int)row0, row1));
        const int held = (ctx + kTile - 1) / kTile;
        const int tiles = n > 0 ? held + (n + kTile - 1) / kTile : 0;
        const int groups = (n * a.group + a.group_cols - 1) / a.group_cols;
        int32_t* q = a.seqs + (int64_t)s * kSeqInts;
        q[0] = ctx;
        q[1] = n;
        q[2] = (int)row0;
        q[3] = tiles;
        q[4] = groups;
        q[5] = held;
        first[s] = mine;
        mine += tiles;
    }
    int64_t incl = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t up = __shfl_up(incl, o, 64);
        if (lane >= o) incl += up;
        row_lo = min(row_lo, __shfl_xor(row_lo, o, 64));
        row_hi = max(row_hi, __shfl_xor(row_hi, o, 64));
    }
    if (lane == 63) {
        waves[wave] = incl;
        rows_lo[wave] = row_lo;
        rows_hi[wave] = row_hi;
    }
    __syncthreads();
    int64_t base = incl - mine, total = 0;
    for (int w = 0; w < kTreeThreads / 64; ++w) {
        if (w < wave) base += waves[w];
        total += waves[w];
        row_lo = min(row_lo, rows_lo[w]);
        row_hi = max(row_hi, rows_hi[w]);
    }
    for (int s = s0; s < s1; ++s) {
        first[s] += base;
        a.seq_first[s] = first[s];
    }
    if (tid == 0) first[a.num_seqs] = total;
    const int64_t share = min(max((total + a.num_shares - 1) / a.num_shares, (int64_t)a.min_share), (int64_t)INT_MAX);
    if (tid == 0) {
        a.head[0] = share;
        a.head[1] = total;
    }
    __syncthreads();
    const int column_groups = a.lanes / a.num_kv_heads;
    for (int w = tid; w < a.num_shares * a.lanes; w += kTreeThreads) {
        const int i = w / a.lanes, lane_of = w - i * a.lanes, h = lane_of / column_groups;
        const int64_t at = (int64_t)i * share;
        int lo = 0, hi = a.num_seqs - 1;  // the last sequence that starts at or before `at`: it has tiles
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (first[mid] <= at) lo = mid;
            else hi = mid - 1;
        }
        const int32_t* q = a.seqs + (int64_t)lo * kSeqInts;
        const int left = (int)max(min(share, total - at), (int64_t)0);
        int4* to = (int4*)(a.work + (int64_t)w * kWorkInts);
        to[0] = make_int4(lo, h, (int)(at - first[lo]), left);
        to[1] = make_int4(q[0], q[1], q[2], q[3]);
        to[2] = make_int4(q[4], q[5], lane_of - h * column_groups, 0);
    }
    const int64_t before = min((int64_t)row_lo, a.num_rows);
    for (int64_t r = tid; r < before; r += kTreeThreads) a.positions[r] = 0;
    for (int64_t r = max((int64_t)row_hi, (int64_t)0) + tid; r < a.num_rows; r += kTreeThreads) a.positions[r] = 0;
}

struct TreeArgs {
    const int64_t* head;
    const int32_t* work;
    const int32_t* seqs;
    const int64_t* seq_first;
    const uint32_t* masks;
    int mask_words;
    int num_seqs;
    const char* q;
    int64_t q_sr, q_sh;
    char* out;
    int64_t o_sr, o_sh;
    const char *k_pool, *v_pool;
    int64_t p_sb, p_ss, p_sh;
    int block_size, block_shift;  // shift -1: not a power of two
    uint32_t num_blocks;
    const int32_t* tables;
    int64_t table_stride;
    const char *new_k, *new_v;
    int64_t n_sr, n_sh;
    int group, num_kv_heads;
    float scale_log2, inv_scale_log2;
    uint32_t q_sign;
    float* partials;
};

template <int DT, int D, int WC, int WK>
struct TreeShape {
    static constexpr int ES = DT == MF_F32 ? 4 : 2;
    static constexpr int WAVES = WC * WK;
    static constexpr int RB = D * ES;                      // bytes of a key row
    static constexpr int NCH = RB / 16;                    // its 16-byte chunks
    static constexpr int RPB = RB >= 256 ? 1 : 256 / RB;   // rows in 256 bytes (every LDS bank once)
    static constexpr int TILE = kTile * RB;
    static constexpr int SUB = WK * TILE >= 8192 ? 1 : 8192 / (WK * TILE);  // tiles of a wave in a stage
    static constexpr int ST = WK * SUB;                    // tiles of a stage
    static constexpr int HALF = ST * TILE;                 // its K rows, then its V rows
    static constexpr int STG = 2 * HALF;
    static constexpr int RING = STG * 4 <= 64 * 1024 ? 4 : 2;
    static constexpr int PAIRS = HALF / 1024 / WAVES;      // 1 KB pieces of K, and of V, per wave and stage
    static constexpr int NLD = 2 * PAIRS;
    static constexpr int NQ = RB / 32;                     // 16-byte pieces of a query row per lane half
    static constexpr int ND = D / 32;
    static constexpr int PER_CU = WAVES == 8 || RB > 256 || RING * STG > 72 * 1024 ? 1 : 2;  // workgroups
    // Weights are 2^(score - maximum + UP), the maximum moved when a score passes it by more than
    // 2^SLACK, and UP cancels in out = sum w v / sum w. fp16 keeps weights for the second product in
    // steps of 2^-24 at the least, which are then 2^-34 of the largest: all rounded off together are
    // at most keys * 2^-35 of the sum. (With UP 0 the tail of 32,001 keys could lose 2^-10 of
    // it.) The price is a maximum that moves more often: the second case above 117.8 us a call with
    // SLACK 8 and UP 0, 120.8 so, 123.5 with SLACK 3.
    static constexpr float UP = DT == MF_F16 ? 10.f : 0.f;
    static constexpr float SLACK = DT == MF_F16 ? 5.f : kLazyLog2;
    static constexpr int COLS = WC * 32;
    static constexpr int SLOT = COLS * (D + 2);            // floats of a piece's sums
    static_assert(PAIRS >= 1 && HALF % (1024 * WAVES) == 0, "whole pieces for every wave");
};

// Sum and maximum of a column live in two lanes (lane halves); O^T's lane (hf, column)
// holds head_dim elements 32 d + 8 b + 4 hf + 0..3 in acc[d][4 b ..].
template <int DT, int ND>
__device__ __forceinline__ void store_column(char* dst, bool live, const f32x16 (&acc)[ND], float inv, int hf) {
    if constexpr (DT == MF_F32) {
        if (!live) return;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int b = 0; b < 4; ++b)
                *(float4*)(dst + (32 * d + 8 * b + 4 * hf) * 4) =
                    make_float4(acc[d][4 * b] * inv, acc[d][4 * b + 1] * inv, acc[d][4 * b + 2] * inv, acc[d][4 * b + 3] * inv);
    } else {
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int b = 0; b < 4; b += 2) {
                uint32_t w[2][2];
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        w[e][k] = f32_to_bits<DT>(acc[d][4 * (b + e) + 2 * k] * inv) |
                                  (f32_to_bits<DT>(acc[d][4 * (b + e) + 2 * k + 1] * inv) << 16);
                auto x = __builtin_amdgcn_permlane32_swap(w[0][0], w[1][0], false, false);
                auto y = __builtin_amdgcn_permlane32_swap(w[0][1], w[1][1], false, false);
                if (live) *(uint4*)(dst + (32 * d + 8 * (b + hf)) * 2) = make_uint4(x[0], y[0], x[1], y[1]);
            }
    }
}

__device__ __forceinline__ f32x16 mfma32_f32(float a, float b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0);
}

// The sum over both lane halves, in both.
__device__ __forceinline__ float both_halves_sum(float v) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Infinities and NaN are the elements whose exponent is all ones.
template <int DT>
__device__ __forceinline__ bool not_finite(uint32_t element) {
    constexpr uint32_t inf = DT == MF_F32 ? 0x7f800000u : DT == MF_BF16 ? 0x7f80u : 0x7c00u;
    return (element & inf) == inf;
}
// 0 in their place, in an element or in a pair.
template <int DT>
__device__ __forceinline__ uint32_t finite_of(uint32_t x) {
    if constexpr (DT == MF_F32) return not_finite<DT>(x) ? 0u : x;
    else return (not_finite<DT>(x & 0xffffu) ? 0u : x & 0xffffu) | (not_finite<DT>(x >> 16) ? 0u : x & 0xffff0000u);
}
// Adds an element to a sum if it is not finite.
template <int DT>
__device__ __forceinline__ float with(float sum, uint32_t element) {
    return not_finite<DT>(element) ? sum + bits_to_f32<DT>(element) : sum;
}

template <int DT, int D, int WC, int WK>
__global__ __launch_bounds__(WC * WK * 64, (TreeShape<DT, D, WC, WK>::PER_CU * WC * WK / 4)) void tree_kernel(TreeArgs a) {
    using S = TreeShape<DT, D, WC, WK>;
    constexpr int ES = S::ES, RB = S::RB, NCH = S::NCH, RPB = S::RPB, NQ = S::NQ, ND = S::ND, ST = S::ST;
    constexpr int AHEAD = S::RING - 1;  // stages in flight
    constexpr float kNegInf = -__builtin_huge_valf();
    __shared__ __align__(1024) char ring[S::RING * S::STG];
    __shared__ int tab[kWindow];
    // Rows of the tiles that not all columns see whole (the context's last, and the nodes') whose V is not all
    // finite: a word of 32 rows for each tile, then whether there are any.
    __shared__ uint32_t wild[kMaxWild + 1];
    static_assert(WK == 1 || (WK - 1) * WC * (ND * 16 + 2) * 256 <= S::RING * S::STG, "the key waves' sums fit the ring");

    const int32_t* at = a.work + (int64_t)blockIdx.x * kWorkInts;
    const int h = at[1], grp = at[10];
    int s = at[0], tile0 = at[2], left = at[3];
    int ctx = at[4], n = at[5], row0 = at[6], tiles = at[7], groups = at[8], held = at[9];
    if (left <= 0) return;
    const int tid = threadIdx.x, lane = tid & 63, hf = lane >> 5, j = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wc = wave % WC, wk = wave / WC;
    const uint32_t ring_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)ring;
    auto sync = [&]() {
        __builtin_amdgcn_s_waitcnt((15) | (3 << 14) | (7 << 4) | (0 << 8));  // lgkmcnt(0)
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    // lane addresses inside a tile: K rows (key lane & 31), V rows
    uint32_t kaddr[NQ], vaddr[ND];
#pragma unroll
    for (int c = 0; c < NQ; ++c)
        kaddr[c] = (uint32_t)((lane & 31) * RB + (((2 * c + hf) ^ ((j / RPB) & (NCH - 1))) << 4));
#pragma unroll
    for (int d = 0; d < ND; ++d) {
        if constexpr (DT == MF_F32)
            vaddr[d] = (uint32_t)(S::HALF + 4 * hf * RB + (32 * d + (lane & 31)) * 4);
        else
            vaddr[d] = (uint32_t)(S::HALF + (4 * hf + (j >> 2)) * RB +
                                  (((4 * d + 2 * ((lane & 31) >> 4) + ((j & 3) >> 1)) ^ (((j >> 2) / RPB) << 2)) << 4) +
                                  8 * (j & 1));
    }
    // 1 KB pieces of a stage: this wave's i-th K piece holds row_of(i) of the stage in this
    // lane's 16 bytes, its V piece the same row; rows are swizzled in 16-byte chunks
    auto k_swizzle = [](int in) { return ((in & 15) / RPB) & (NCH - 1); };
    auto v_swizzle = [](int in) { return DT == MF_F32 ? 0 : ((in & 3) / RPB) << 2; };
    auto row_of = [&](int i) { return (wave + S::WAVES * i) * (1024 / RB) + lane * 16 / RB; };
    auto k_piece = [&](int i) { return ((lane & (NCH - 1)) ^ k_swizzle(row_of(i))) << 4; };
    auto v_piece = [&](int i) { return ((lane & (NCH - 1)) ^ v_swizzle(row_of(i))) << 4; };
    const int64_t v_delta = a.v_pool - a.k_pool, nv_delta = a.new_v - a.new_k;
    auto block_of = [&](int key) -> int {
        return a.block_shift >= 0 ? key >> a.block_shift : (int)((unsigned)key / (unsigned)a.block_size);
    };

    bool first = true;
    for (;;) {
        const int run = min(left, tiles - tile0);
        if (grp < groups) {
            // ---- one sequence: its block-table entries, or a window of them, in LDS
            const int32_t* trow = a.tables + (int64_t)s * a.table_stride;
            int window = 0, window_lo = 0, window_hi = 0;  // first block, and the keys it covers
            auto fill_window = [&](int from_key) {
                const int blocks = ctx > 0 ? block_of(ctx - 1) + 1 : 0;
                window = blocks <= kWindow ? 0 : block_of(from_key);
                window_lo = window * a.block_size;
                window_hi = blocks - window <= kWindow ? ctx : (window + kWindow) * a.block_size;
                const int end = min(window + kWindow, blocks);
                for (int i = window + tid; i < end; i += S::WAVES * 64) tab[i - window] = trow[i];
            };
            fill_window(tile0 * kTile);
            if (tid <= kMaxWild) wild[tid] = 0;
            sync();
            const int part_seen = ctx / kTile;  // the first of those tiles

            int f_tile = tile0, f_left = run;
            int in_flight = 0, head_buf = 0, next_buf = 0;
            auto fetch = [&]() __attribute__((always_inline)) {
                const int take = min(ST, f_left);
                const int st0 = f_tile, t_end = st0 + take;
                const uint32_t dst0 = ring_at + (uint32_t)(next_buf * S::STG);
                const int first_key = st0 * kTile, end_key = min(t_end * kTile, ctx);
                if (first_key < end_key && (first_key < window_lo || end_key > window_hi)) {
                    sync();
                    fill_window(first_key);
                    sync();
                }
                if (st0 + ST <= min(held, t_end) && a.block_shift >= 0) {
                    // all keys in the pool; rows past the context's end read its last one: masked, and every
                    // column sees that row
                    const char* kh = a.k_pool + (int64_t)h * a.p_sh * ES;
                    uint32_t e[S::PAIRS];
                    int key[S::PAIRS];
#pragma unroll
                    for (int i = 0; i < S::PAIRS; ++i) {
                        key[i] = min(first_key + row_of(i), ctx - 1);
                        e[i] = (uint32_t)tab[(key[i] >> a.block_shift) - window];
                    }
#pragma unroll
                    for (int i = 0; i < S::PAIRS; ++i) {
                        const char* src = kh + ((int64_t)min(e[i], a.num_blocks - 1) * a.p_sb +
                                                (int64_t)(key[i] & (a.block_size - 1)) * a.p_ss) * ES;
                        ld_lds16_nt(src + k_piece(i), dst0 + (uint32_t)((wave + S::WAVES * i) * 1024));
                        ld_lds16_nt(src + v_delta + v_piece(i), dst0 + (uint32_t)(S::HALF + (wave + S::WAVES * i) * 1024));
                    }
                } else {
#pragma unroll 1
                    for (int i = 0; i < S::PAIRS; ++i) {
                        const int r = row_of(i), in = r & 31;
                        const int t = min(st0 + (r >> 5), t_end - 1);
                        const char* src;
                        int64_t to_v;
                        if (t < held) {
                            const int key = min(t * kTile + in, ctx - 1), blk = block_of(key);
                            const uint32_t e = min((uint32_t)tab[blk - window], a.num_blocks - 1);
                            src = a.k_pool + ((int64_t)e * a.p_sb + (int64_t)(key - blk * a.block_size) * a.p_ss +
                                              (int64_t)h * a.p_sh) * ES;
                            to_v = v_delta;
                        } else {
                            const int node = min((t - held) * kTile + in, n - 1);
                            src = a.new_k + ((int64_t)(row0 + node) * a.n_sr + (int64_t)h * a.n_sh) * ES;
                            to_v = nv_delta;
                        }
                        ld_lds16_nt(src + k_piece(i), dst0 + (uint32_t)((wave + S::WAVES * i) * 1024));
                        ld_lds16_nt(src + to_v + v_piece(i), dst0 + (uint32_t)(S::HALF + (wave + S::WAVES * i) * 1024));
                    }
                }
                f_left -= take;
                f_tile += take;
                ++in_flight;
                next_buf = next_buf + 1 == S::RING ? 0 : next_buf + 1;
            };
#pragma unroll 1
            for (int u = 0; u < AHEAD && f_left > 0; ++u) fetch();

            {
                // ---- this lane's column and query
                const int t0 = tile0, t1 = t0 + run;
                const int cidx = grp * S::COLS + wc * 32 + (lane & 31);
                const bool valid = cidx < n * a.group;
                const int node = (int)((unsigned)(valid ? cidx : 0) / (unsigned)a.group);
                const int64_t prow = row0 + node;
                const int qhead = h * a.group + (valid ? cidx : 0) - node * a.group;
                const bool busy = grp * S::COLS + wc * 32 < n * a.group;  // a wave of padding columns only loads
                uint4 qf[NQ];
                const char* qp = a.q + (prow * a.q_sr + (int64_t)qhead * a.q_sh) * ES;
#pragma unroll
                for (int c = 0; c < NQ; ++c) {
                    const uint4 v = *(const uint4*)(qp + (2 * c + hf) * 16);
                    qf[c] = make_uint4(v.x ^ a.q_sign, v.y ^ a.q_sign, v.z ^ a.q_sign, v.w ^ a.q_sign);
                }
                float m = kMinM, l = 0.f, thr = (kMinM + S::SLACK) * a.inv_scale_log2;
                f32x16 acc[ND];
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;

                auto tile = [&](const char* stg, int t) __attribute__((always_inline)) {
                    f32x16 st;
#pragma unroll
                    for (int i = 0; i < 16; ++i) st[i] = 0.f;
#pragma unroll
                    for (int c = 0; c < NQ; ++c) {
                        const uint4 kf = *(const uint4*)(stg + kaddr[c]);
                        if constexpr (DT == MF_F32) {
                            st = mfma32_f32(__uint_as_float(kf.x), __uint_as_float(qf[c].x), st);
                            st = mfma32_f32(__uint_as_float(kf.y), __uint_as_float(qf[c].y), st);
                            st = mfma32_f32(__uint_as_float(kf.z), __uint_as_float(qf[c].z), st);
                            st = mfma32_f32(__uint_as_float(kf.w), __uint_as_float(qf[c].w), st);
                        } else {
                            st = mfma32<DT>(kf, qf[c], st);
                        }
                    }
                    if ((t + 1) * kTile > ctx) {  // the context's last tile, and the nodes'
                        uint32_t seen;
                        if (t < held) seen = 0xffffffffu >> ((t + 1) * kTile - ctx);
                        else seen = valid ? a.masks[prow * a.mask_words + (t - held)] : 0u;
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const int key = 8 * (i >> 2) + 4 * hf + (i & 3);
                            st[i] = seen >> key & 1u ? st[i] : kNegInf;
                        }
                    }
                    // lazy rescale: the maximum moves when a score passes it by more than 2^SLACK
                    float lmax = st[0];
#pragma unroll
                    for (int i = 1; i < 16; ++i) lmax = fmax_prop(lmax, st[i]);
                    if (__builtin_amdgcn_ballot_w64(lmax > thr) != 0) {
                        auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(lmax), __float_as_uint(lmax), false, false);
                        float mn = fmax_prop(__uint_as_float(r[0]), __uint_as_float(r[1])) * a.scale_log2;
                        // fp16's weights end at 2^16: roundings of scores of any size (here, and four in thr) go the other way
                        if constexpr (DT == MF_F16) mn += fabsf(mn) * 0x1p-23f;
                        mn = fmaxf(m, mn);
                        const float alpha = __builtin_amdgcn_exp2f(m - mn);
                        l *= alpha;
#pragma unroll
                        for (int d = 0; d < ND; ++d)
#pragma unroll
                            for (int i = 0; i < 16; ++i) acc[d][i] *= alpha;
                        m = mn;
                        thr = (mn + S::SLACK - (DT == MF_F16 ? fabsf(mn) * 0x1p-21f : 0.f)) * a.inv_scale_log2;
                    }
                    float sum = 0.f;
                    const float zero = DT == MF_F16 ? S::UP - m : -m;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        st[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[i], a.scale_log2, zero));
                        sum += st[i];
                    }
                    l += sum;
                    if constexpr (DT == MF_F32) {
#pragma unroll
                        for (int i = 0; i < 16; ++i)
#pragma unroll
                            for (int d = 0; d < ND; ++d)
                                acc[d] = mfma32_f32(*(const float*)(stg + vaddr[d] + (8 * (i >> 2) + (i & 3)) * RB), st[i],
                                                    acc[d]);
                    } else {
                        // 16-bit operands of the second product: each weight off by half a step of the type (fp16's
                        // smallest weights by half of its least step, see UP; its largest are 2^15)
                        uint32_t pw[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const f32x2 pair = {st[2 * i], st[2 * i + 1]};
                            if constexpr (DT == MF_BF16)
                                pw[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(pair, bf16x2));
                            else
                                pw[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(pair, f16x2));
                        }
#pragma unroll
                        for (int k = 0; k < 2; ++k)
#pragma unroll
                            for (int d = 0; d < ND; ++d) {
                                const uint2 v0 = ld_tr16(stg + vaddr[d] + 16 * k * RB);
                                const uint2 v1 = ld_tr16(stg + vaddr[d] + (16 * k + 8) * RB);
                                acc[d] = mfma32<DT>(make_uint4(v0.x, v0.y, v1.x, v1.y),
                                                    make_uint4(pw[4 * k], pw[4 * k + 1], pw[4 * k + 2], pw[4 * k + 3]), acc[d]);
                            }
                    }
                };

                for (int st0 = t0; st0 < t1; st0 += ST) {
                    if (in_flight == AHEAD) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((AHEAD - 1) * S::NLD) : "memory");
                    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                    --in_flight;
                    sync();  // the oldest stage is whole, and the one before it has been read
                    if (f_left > 0) fetch();
                    if (st0 + ST > part_seen) {
                        // the product below gives a column 0 times the rows it does not see, which would be NaN for
                        // an infinity: there the rows hold 0 instead, and who sees them gets it at the end
                        char* v = ring + head_buf * S::STG + S::HALF + wave * 1024 + lane * 16;
#pragma unroll
                        for (int i = 0; i < S::PAIRS; ++i) {
                            uint4* at_v = (uint4*)(v + i * S::WAVES * 1024);
                            const uint4 x = *at_v;
                            const uint4 y = make_uint4(finite_of<DT>(x.x), finite_of<DT>(x.y), finite_of<DT>(x.z), finite_of<DT>(x.w));
                            const int t = st0 + (row_of(i) >> 5);
                            if (((x.x ^ y.x) | (x.y ^ y.y) | (x.z ^ y.z) | (x.w ^ y.w)) != 0 && t >= part_seen && t < t1) {
                                *at_v = y;
                                atomicOr(&wild[t - part_seen], 1u << (row_of(i) & 31));
                                wild[kMaxWild] = 1;
                            }
                        }
                        sync();
                    }
                    if (busy) {
                        const char* stg = ring + head_buf * S::STG;
#pragma unroll 1
                        for (int x = 0; x < S::SUB; ++x) {
                            const int t = st0 + x * WK + wk;
                            if (t < t1) tile(stg + (x * WK + wk) * S::TILE, t);
                        }
                    }
                    head_buf = head_buf + 1 == S::RING ? 0 : head_buf + 1;
                }

                // ---- the key waves' sums in one, then the piece's result
                l = both_halves_sum(l);
                if constexpr (WK > 1) {
                    constexpr int PART = (ND * 16 + 2) * 64;
                    sync();
                    if (wk > 0) {
                        float* to = (float*)ring + ((wk - 1) * WC + wc) * PART;
#pragma unroll
                        for (int d = 0; d < ND; ++d)
#pragma unroll
                            for (int i = 0; i < 16; i += 4)
                                *(float4*)(to + (d * 16 + i) * 64 + 4 * lane) =
                                    make_float4(acc[d][i], acc[d][i + 1], acc[d][i + 2], acc[d][i + 3]);
                        to[ND * 1024 + lane] = m;
                        to[ND * 1024 + 64 + lane] = l;
                    }
                    sync();
                    if (wk == 0) {
#pragma unroll
                        for (int o = 0; o < WK - 1; ++o) {
                            const float* from = (const float*)ring + (o * WC + wc) * PART;
                            const float m1 = from[ND * 1024 + lane], l1 = from[ND * 1024 + 64 + lane];
                            const float mn = fmaxf(m, m1);
                            const float w0 = __builtin_amdgcn_exp2f(m - mn), w1 = __builtin_amdgcn_exp2f(m1 - mn);
                            m = mn;
                            l = l * w0 + l1 * w1;
#pragma unroll
                            for (int d = 0; d < ND; ++d)
#pragma unroll
                                for (int i = 0; i < 16; i += 4) {
                                    const float4 v = *(const float4*)(from + (d * 16 + i) * 64 + 4 * lane);
                                    acc[d][i] = acc[d][i] * w0 + v.x * w1;
                                    acc[d][i + 1] = acc[d][i + 1] * w0 + v.y * w1;
                                    acc[d][i + 2] = acc[d][i + 2] * w0 + v.z * w1;
                                    acc[d][i + 3] = acc[d][i + 3] * w0 + v.w * w1;
                                }
                        }
                    }
                }
                if (wild[kMaxWild] != 0 && wk == 0 && busy) {
                    for (int t = max(t0, part_seen); t < t1; ++t) {
                        uint32_t rows = __builtin_amdgcn_readfirstlane(wild[t - part_seen]);
                        const uint32_t seen = !valid ? 0u : t >= held ? a.masks[prow * a.mask_words + (t - held)]
                                                                      : 0xffffffffu >> ((t + 1) * kTile - ctx);
                        for (; rows != 0; rows &= rows - 1) {
                            const int r = __builtin_ctz(rows), key = t * kTile + r;
                            if (!(seen >> r & 1u)) continue;
                            const char* src;
                            if (t < held) {
                                const int blk = block_of(key);
                                const uint32_t e = min((uint32_t)trow[blk], a.num_blocks - 1);
                                src = a.v_pool + ((int64_t)e * a.p_sb + (int64_t)(key - blk * a.block_size) * a.p_ss +
                                                  (int64_t)h * a.p_sh) * ES;
                            } else {
                                src = a.new_v + ((int64_t)(row0 + (key - held * kTile)) * a.n_sr + (int64_t)h * a.n_sh) * ES;
                            }
#pragma unroll
                            for (int d = 0; d < ND; ++d)
#pragma unroll
                                for (int b = 0; b < 4; ++b) {
                                    const char* piece = src + (32 * d + 8 * b + 4 * hf) * ES;
                                    if constexpr (DT == MF_F32) {
                                        const uint4 x = *(const uint4*)piece;
                                        acc[d][4 * b] = with<DT>(acc[d][4 * b], x.x);
                                        acc[d][4 * b + 1] = with<DT>(acc[d][4 * b + 1], x.y);
                                        acc[d][4 * b + 2] = with<DT>(acc[d][4 * b + 2], x.z);
                                        acc[d][4 * b + 3] = with<DT>(acc[d][4 * b + 3], x.w);
                                    } else {
                                        const uint2 x = *(const uint2*)piece;
                                        acc[d][4 * b] = with<DT>(acc[d][4 * b], x.x & 0xffffu);
                                        acc[d][4 * b + 1] = with<DT>(acc[d][4 * b + 1], x.x >> 16);
                                        acc[d][4 * b + 2] = with<DT>(acc[d][4 * b + 2], x.y & 0xffffu);
                                        acc[d][4 * b + 3] = with<DT>(acc[d][4 * b + 3], x.y >> 16);
                                    }
                                }
                        }
                    }
                }
                if (wk == 0 && busy) {
                    if (t0 == 0 && t1 == tiles) {
                        store_column<DT, ND>(a.out + (prow * a.o_sr + (int64_t)qhead * a.o_sh) * ES, valid, acc, 1.f / l, hf);
                    } else {
                        float* to = a.partials + (2 * (int64_t)blockIdx.x + (first ? 0 : 1)) * S::SLOT + wc * 32 * (D + 2);
#pragma unroll
                        for (int d = 0; d < ND; ++d)
#pragma unroll
                            for (int i = 0; i < 16; i += 4)
                                if (valid)
                                    *(float4*)(to + (d * 16 + i) * 64 + 4 * lane) =
                                        make_float4(acc[d][i], acc[d][i + 1], acc[d][i + 2], acc[d][i + 3]);
                        if (hf == 0) {
                            to[32 * D + lane] = m;
                            to[32 * D + 32 + lane] = l;
                        }
                    }
                }
            }
            sync();  // the ring and the window have been read
        }
        left -= run;
        if (left <= 0) return;
        first = false;
        tile0 = 0;
        do {
            ++s;
            const int32_t* info = a.seqs + (int64_t)s * kSeqInts;
            ctx = info[0];
            n = info[1];
            row0 = info[2];
            tiles = info[3];
            groups = info[4];
            held = info[5];
        } while (tiles == 0);  // the line has `left` more tiles, so a sequence with tiles comes
    }
}

// The cut (sequence, kv head, column group)s' results. SPLIT: a workgroup for 32 columns and
// 32 head_dim elements, whose four waves take every fourth piece; otherwise one for 32
// columns, a wave for every 32 elements, which walks the two or three pieces itself.
template <int DT, int D, int WC, int WK, bool SPLIT>
__global__ __launch_bounds__(kTreeThreads) void merge_tree_kernel(TreeArgs a, int units_per_seq) {
    using S = TreeShape<DT, D, WC, WK>;
    constexpr int ES = S::ES;
    __shared__ float sums[SPLIT ? 3 : 1][SPLIT ? 18 * 64 : 1];
    const int64_t share = a.head[0];
    const int u = blockIdx.x, s = u / units_per_seq, unit = u - s * units_per_seq;
    const int lane = threadIdx.x & 63, hf = lane >> 5, wave = threadIdx.x >> 6;
    const int blk = SPLIT ? blockIdx.y / S::ND : blockIdx.y;
    const int32_t* info = a.seqs + (int64_t)s * kSeqInts;
    const int n = info[1], row0 = info[2], tiles = info[3], groups = info[4];
    const int64_t begin = a.seq_first[s];
    const int column_groups = units_per_seq / a.num_kv_heads, h = unit / column_groups, grp = unit - h * column_groups;
    if (tiles == 0 || grp >= groups) return;
    if (grp * S::COLS + blk * 32 >= n * a.group) return;
    const int64_t w0 = begin / share, w1 = (begin + tiles - 1) / share;
    if (w0 == w1) return;
    const int c = grp * S::COLS + blk * 32 + (lane & 31);
    const bool valid = c < n * a.group;
    for (int d = SPLIT ? blockIdx.y % S::ND : wave; d < S::ND; d += SPLIT ? S::ND : 4) {
        float m = kMinM, l = 0.f;
        f32x16 acc[1];
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[0][i] = 0.f;
#pragma unroll 2
        for (int64_t w = w0 + (SPLIT ? wave : 0); w <= w1; w += SPLIT ? 4 : 1) {
            const int64_t slot = 2 * (w * units_per_seq + unit) + (w * share < begin ? 1 : 0);
            const float* from = a.partials + slot * S::SLOT + blk * 32 * (D + 2);
            const float m1 = from[32 * D + (lane & 31)], l1 = from[32 * D + 32 + (lane & 31)];
            float4 v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = *(const float4*)(from + (d * 16 + 4 * i) * 64 + 4 * lane);
            const float mn = fmaxf(m, m1);
            const float e0 = __builtin_amdgcn_exp2f(m - mn), e1 = __builtin_amdgcn_exp2f(m1 - mn);
            m = mn;
            l = l * e0 + l1 * e1;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                acc[0][4 * i] = acc[0][4 * i] * e0 + v[i].x * e1;
                acc[0][4 * i + 1] = acc[0][4 * i + 1] * e0 + v[i].y * e1;
                acc[0][4 * i + 2] = acc[0][4 * i + 2] * e0 + v[i].z * e1;
                acc[0][4 * i + 3] = acc[0][4 * i + 3] * e0 + v[i].w * e1;
            }
        }
        if constexpr (SPLIT) {
            if (wave > 0) {
                float* to = sums[wave - 1];
#pragma unroll
                for (int i = 0; i < 16; ++i) to[i * 64 + lane] = acc[0][i];
                to[16 * 64 + lane] = m;
                to[17 * 64 + lane] = l;
            }
            __syncthreads();
            if (wave > 0) return;
#pragma unroll
            for (int o = 0; o < 3; ++o) {
                const float m1 = sums[o][16 * 64 + lane], l1 = sums[o][17 * 64 + lane];
                const float mn = fmaxf(m, m1);
                const float e0 = __builtin_amdgcn_exp2f(m - mn), e1 = __builtin_amdgcn_exp2f(m1 - mn);
                m = mn;
                l = l * e0 + l1 * e1;
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[0][i] = acc[0][i] * e0 + sums[o][i * 64 + lane] * e1;
            }
        }
        const int node = (int)((unsigned)(valid ? c : 0) / (unsigned)a.group);
        const int qhead = h * a.group + (valid ? c : 0) - node * a.group;
        store_column<DT, 1>(a.out + ((int64_t)(row0 + node) * a.o_sr + (int64_t)qhead * a.o_sh + 32 * d) * ES, valid, acc,
                            1.f / l, hf);
    }
}

// The waves' arrangement for a call and the least tiles of a share. wc waves stand side by
// side on blocks of 32 columns, 4 / wc along the keys; 8 waves where 8 blocks share their keys.
//
// Each tile is loaded once for all columns of its group, so a group is as wide as the columns
// are. The rule by its sides (layers as in the comment above, us a call with the plan):
// 20 columns, 64 contexts of up to 4,000 at 40/8 x 128: two blocks 202, four 205, one block
// with four waves along the keys 222; 60 columns there: two 232, four 237. 80 columns, the
// first case above: four blocks 358, eight 400. 240 columns, the second: eight blocks 133,
// two groups of four 153; 192 at 15/5 x 64, four layers: 116, 126.
//
// Shares of few tiles spread a short line over more of the GPU and leave more sums to merge.
// 4 contexts of up to 700 tokens at 15/5 x 64, least shares of 8, 4, 2 and 1: 24 columns (four
// layers) -, 53, 44, 48; 72 columns 71, 65, 63, -; 192 columns 82, 73, 77, -; 24 in fp32 (two
// layers) 63, 46, 38, -.
struct TreeConfig {
    int wc, per_cu, min_share;
};

TreeConfig tree_config(int dtype, int head_dim, int max_nodes, int group) {
    const int64_t cols = (int64_t)max_nodes * group;
    const int rb = head_dim * dtype_size(dtype);
    if (dtype == MF_F32 || rb > 256) return {4, rb > 256 ? 1 : 2, 2};
    if (cols <= 64) return {2, 2, 2};
    if (cols <= 128) return {4, 2, 2};
    return {8, 1, 4};
}

template <int DT, int D, int WC, int WK>
int launch_tree(const TreeArgs& a, int workers, int units_per_seq, hipStream_t st) {
    hipLaunchKernelGGL((tree_kernel<DT, D, WC, WK>), dim3((unsigned)workers), dim3(WC * WK * 64), 0, st, a);
    if (int e = check_launch()) return e;
    const int units = a.num_seqs * units_per_seq;
    // Few units for the workers are cut into many pieces each: their sums are spread over more
    // workgroups (4 contexts of up to 700, the 24 columns above: 43 us, unsplit 53; one of 32,001:
    // 133, 146; 16 at 15/5 x 64 and 192 columns: 114, 116). Where most units are whole, the larger
    // grid has nothing to do (1,024 contexts of up to 200 at 40/8 x 128, 20 columns: 492, unsplit 418).
    if ((int64_t)units * 2 <= workers)
        hipLaunchKernelGGL((merge_tree_kernel<DT, D, WC, WK, true>), dim3((unsigned)units, WC * (D / 32)),
                           dim3(kTreeThreads), 0, st, a, units_per_seq);
    else
        hipLaunchKernelGGL((merge_tree_kernel<DT, D, WC, WK, false>), dim3((unsigned)units, WC), dim3(kTreeThreads), 0, st, a,
                           units_per_seq);
    return check_launch();
}

template <int DT, int D>
int launch_tree(const TreeArgs& a, const TreeConfig& c, int workers, int units_per_seq, hipStream_t st) {
    if constexpr (DT != MF_F32 && D <= 128) {
        if (c.wc == 2) return launch_tree<DT, D, 2, 2>(a, workers, units_per_seq, st);
        if (c.wc == 8) return launch_tree<DT, D, 8, 1>(a, workers, units_per_seq, st);
    }
    return launch_tree<DT, D, 4, 1>(a, workers, units_per_seq, st);
}

bool tree_shape_ok(int num_seqs, int64_t num_rows, int max_nodes, int num_q_heads, int num_kv_heads, int head_dim, int dtype) {
    return num_seqs >= 0 && num_seqs <= kMaxSeqs && num_rows >= 0 && num_rows <= INT_MAX && max_nodes >= 1 &&
           max_nodes <= MF_TREE_MAX_NODES && num_kv_heads >= 1 && num_q_heads >= num_kv_heads &&
           num_q_heads % num_kv_heads == 0 && num_q_heads <= (1 << 16) && dtype_ok(dtype) && head_dim > 0;
}
bool tree_dim_ok(int head_dim) { return head_dim == 32 || head_dim == 64 || head_dim == 128 || head_dim == 256; }

// Where a plan's parts lie in its buffer, in 32-bit words.
struct TreeLayout {
    int64_t head, seq_first, work, seqs, masks, total;
    int shares, lanes, workers, mask_words;
};
TreeLayout tree_layout(int num_seqs, int64_t num_rows, int max_nodes, int group, int num_kv_heads, const TreeConfig& c,
                       int num_cus) {
    TreeLayout l;
    const int64_t lanes = num_kv_heads * (((int64_t)max_nodes * group + c.wc * 32 - 1) / (c.wc * 32));
    l.lanes = (int)lanes;
    l.shares = (int)std::max<int64_t>(num_cus * c.per_cu / lanes, 1);
    l.workers = l.shares * l.lanes;
    l.mask_words = (max_nodes + 31) / 32;
    l.head = 0;
    l.seq_first = 4;
    l.work = l.seq_first + 2 * (((int64_t)num_seqs + 1) & ~1ll);
    l.seqs = l.work + kWorkInts * (int64_t)l.workers;
    l.masks = l.seqs + (int64_t)kSeqInts * num_seqs;
    l.total = l.masks + num_rows * l.mask_words;
    return l;
}

}  // namespace
}  // namespace mf

extern "C" int mf_tree_plan_sizes(int num_seqs, int64_t num_rows, int max_nodes, int num_q_heads, int num_kv_heads,
                                  int head_dim, int dtype, int num_cus, int64_t* plan_words, int64_t* partials_floats) {
    using namespace mf;
    if (!tree_shape_ok(num_seqs, num_rows, max_nodes, num_q_heads, num_kv_heads, head_dim, dtype) || num_cus < 1 ||
        num_cus > 4096 || !plan_words || !partials_floats)
        return MF_ERR_ARG;
    if (!tree_dim_ok(head_dim)) return MF_ERR_UNSUPPORTED;
    const TreeConfig c = tree_config(dtype, head_dim, max_nodes, num_q_heads / num_kv_heads);
    const TreeLayout l = tree_layout(num_seqs, num_rows, max_nodes, num_q_heads / num_kv_heads, num_kv_heads, c, num_cus);
    *plan_words = l.total;
    *partials_floats = 2 * (int64_t)l.workers * (c.wc * 32) * (head_dim + 2);
    return MF_OK;
}

extern "C" int mf_tree_plan(const int32_t* parents, const int32_t* cu_nodes, const int32_t* context_lens, int num_seqs,
                            int64_t num_rows, int max_nodes, int64_t max_context, int num_q_heads, int num_kv_heads,
                            int head_dim, int dtype, int num_cus, int32_t* plan, int64_t plan_words, int64_t* positions,
                            mf_stream_t stream) {
    using namespace mf;
    int64_t words = 0, floats = 0;
    if (int e = mf_tree_plan_sizes(num_seqs, num_rows, max_nodes, num_q_heads, num_kv_heads, head_dim, dtype, num_cus,
                                   &words, &floats))
        return e;
    if (max_context < 0 || max_context > (1 << 30)) return MF_ERR_ARG;
    if (num_seqs == 0) {
        if (num_rows == 0) return MF_OK;
        if (!positions) return MF_ERR_ARG;
        const int64_t blocks = std::min<int64_t>((num_rows + kTreeThreads - 1) / kTreeThreads, 1024);
        hipLaunchKernelGGL(clear_positions_kernel, dim3((unsigned)blocks), dim3(kTreeThreads), 0, (hipStream_t)stream,
                           positions, num_rows);
        return check_launch();
    }
    if (!cu_nodes || !context_lens || !plan || ((uintptr_t)plan & 15) || (num_rows > 0 && (!parents || !positions)))
        return MF_ERR_ARG;
    if (plan_words < words) return MF_ERR_WORKSPACE;
    const int group = num_q_heads / num_kv_heads;
    const TreeConfig c = tree_config(dtype, head_dim, max_nodes, group);
    const TreeLayout l = tree_layout(num_seqs, num_rows, max_nodes, num_q_heads / num_kv_heads, num_kv_heads, c, num_cus);
    TreePlanArgs a{parents, cu_nodes, context_lens, num_seqs, num_rows, max_nodes, l.mask_words, max_context, group,
                   num_kv_heads, c.wc * 32, l.lanes, l.shares, c.min_share, (int64_t*)(plan + l.head), plan + l.seqs,
                   (int64_t*)(plan + l.seq_first), plan + l.work, (uint32_t*)(plan + l.masks), positions};
    hipLaunchKernelGGL(tree_plan_kernel, dim3((unsigned)num_seqs + 1), dim3(kTreeThreads), 0, (hipStream_t)stream, a);
    return check_launch();
}

extern "C" int mf_tree_attention(const void* q, int64_t q_stride_row, int64_t q_stride_head, void* out,
                                 int64_t out_stride_row, int64_t out_stride_head, int dtype, const void* k_pool,
                                 const void* v_pool, int64_t pool_stride_block, int64_t pool_stride_slot,
                                 int64_t pool_stride_head, int block_size, int64_t num_blocks,
                                 const int32_t* block_tables, int64_t block_table_stride, const void* new_k,
                                 const void* new_v, int64_t new_stride_row, int64_t new_stride_head, int num_seqs,
                                 int64_t num_rows, int max_nodes, int num_q_heads, int num_kv_heads, int head_dim,
                                 float scale, int num_cus, const int32_t* plan, int64_t plan_words, float* partials,
                                 int64_t partials_floats, mf_stream_t stream) {
    using namespace mf;
    if (!(std::fabs(scale) < INFINITY)) return MF_ERR_ARG;
    int64_t words = 0, floats = 0;
    if (int e = mf_tree_plan_sizes(num_seqs, num_rows, max_nodes, num_q_heads, num_kv_heads, head_dim, dtype, num_cus,
                                   &words, &floats))
        return e;
    if (block_size < 1 || num_blocks < 1 || num_blocks > INT_MAX || block_table_stride < 0) return MF_ERR_ARG;
    if (num_seqs == 0 || num_rows == 0) return MF_OK;
    if (!q || !out || !k_pool || !v_pool || !block_tables || !new_k || !new_v || !plan || !partials) return MF_ERR_ARG;
    if (plan_words < words || partials_floats < floats) return MF_ERR_WORKSPACE;
    const int es = dtype_size(dtype);
    const int64_t strides[] = {q_stride_row, q_stride_head, out_stride_row, out_stride_head, pool_stride_block,
                               pool_stride_slot, pool_stride_head, new_stride_row, new_stride_head};
    for (int64_t x : strides)
        if (x % (16 / es)) return MF_ERR_ARG;  // rows are read and written in 16-byte pieces
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)new_k | (uintptr_t)new_v |
         (uintptr_t)plan | (uintptr_t)partials) & 15)
        return MF_ERR_ARG;
    const int group = num_q_heads / num_kv_heads;
    const TreeConfig c = tree_config(dtype, head_dim, max_nodes, group);
    const TreeLayout l = tree_layout(num_seqs, num_rows, max_nodes, num_q_heads / num_kv_heads, num_kv_heads, c, num_cus);
    TreeArgs a{};
    a.head = (const int64_t*)(plan + l.head);
    a.work = plan + l.work;
    a.seqs = plan + l.seqs;
    a.seq_first = (const int64_t*)(plan + l.seq_first);
    a.masks = (const uint32_t*)(plan + l.masks);
    a.mask_words = l.mask_words;
    a.num_seqs = num_seqs;
    a.q = (const char*)q;
    a.q_sr = q_stride_row;
    a.q_sh = q_stride_head;
    a.out = (char*)out;
    a.o_sr = out_stride_row;
    a.o_sh = out_stride_head;
    a.k_pool = (const char*)k_pool;
    a.v_pool = (const char*)v_pool;
    a.p_sb = pool_stride_block;
    a.p_ss = pool_stride_slot;
    a.p_sh = pool_stride_head;
    a.block_size = block_size;
    a.block_shift = -1;
    for (int b = 0; b < 31; ++b)
        if (1 << b == block_size) a.block_shift = b;
    a.num_blocks = (uint32_t)num_blocks;
    a.tables = block_tables;
    a.table_stride = block_table_stride;
    a.new_k = (const char*)new_k;
    a.new_v = (const char*)new_v;
    a.n_sr = new_stride_row;
    a.n_sh = new_stride_head;
    a.group = group;
    a.num_kv_heads = num_kv_heads;
    // a negative scale flips the queries' signs; 2^-100 for 0 makes every weight exactly 1
    a.q_sign = scale < 0.f ? (es == 4 ? 0x80000000u : 0x80008000u) : 0u;
    a.scale_log2 = scale == 0.f ? 0x1p-100f : std::fabs(scale) * 1.4426950408889634f;
    a.inv_scale_log2 = 1.f / a.scale_log2;
    a.partials = partials;
    if ((int64_t)num_seqs * l.lanes > INT_MAX) return MF_ERR_ARG;
    hipStream_t st = (hipStream_t)stream;
#define MF_TREE_CASE(DT, DV) \
    if (dtype == DT && head_dim == DV) return launch_tree<DT, DV>(a, c, l.workers, l.lanes, st);
    MF_TREE_CASE(MF_BF16, 32)
    MF_TREE_CASE(MF_BF16, 64)
    MF_TREE_CASE(MF_BF16, 128)
    MF_TREE_CASE(MF_BF16, 256)
    MF_TREE_CASE(MF_F16, 32)
    MF_TREE_CASE(MF_F16, 64)
    MF_TREE_CASE(MF_F16, 128)
    MF_TREE_CASE(MF_F16, 256)
    MF_TREE_CASE(MF_F32, 32)
    MF_TREE_CASE(MF_F32, 64)
    MF_TREE_CASE(MF_F32, 128)
    MF_TREE_CASE(MF_F32, 256)
#undef MF_TREE_CASE
    return MF_ERR_UNSUPPORTED;
}
