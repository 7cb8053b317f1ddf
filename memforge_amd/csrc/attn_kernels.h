// Varlen paged attention for gfx950: one code path for decode, chunked
// prefill and the (k+1)-query speculative verify.
//
// Work decomposition. A "column" is one (query row, query head) pair; the G
// query heads that share a KV head are adjacent columns, so a decode row of a
// GQA group-5 model is 5 columns and a 5-token verify row of a group-3 model is
// 15. One wave owns a work item = (sequence, kv head, up to NT tiles of 16
// columns, a range of 16-key tiles), reads every K/V tile of that range exactly
// once and shares it across all of its columns.
//
// Per 16-key tile the wave computes S^T = K Q^T with MFMA (A = K rows straight
// from the pool, B = the Q fragment kept in registers), applies the per-column
// causal rule key <= position(row), runs the online softmax with the column
// max reduced across the four 16-lane groups by xor shuffles, and accumulates
// O^T = V^T P^T with a second MFMA whose B operand is the exponentiated S^T
// tile exactly as the first MFMA left it in registers. V arrives with
// fully coalesced 16-token x 16-byte row loads and is transposed into the MFMA
// A layout with byte permutes. 16-bit prefill runs in workgroups that share
// each K/V row through LDS instead (attn_wide_body).
//
// Long contexts are split into key partitions (the plan decides); each leaves
// its running maximum and sum in fp32 and its normalised output in the launch's
// type (or in fp32, see the split-K merge), and a merge kernel combines them
// with the log-sum-exp rule.
#pragma once

#include <algorithm>
#include <array>
#include <cfloat>
#include <climits>
#include <cmath>
#include <type_traits>

#include "mf_common.h"

#ifndef MF_MAX_ITEM_TILES
#define MF_MAX_ITEM_TILES 128
#endif
namespace mf {

struct AttnArgs {
    const char* q;
    int64_t q_sr, q_sh;
    char* out;
    int64_t o_sr, o_sh;
    const char* k_pool;
    const char* v_pool;
    int64_t p_sb, p_ss, p_sh;
    int block_size;
    const int32_t* block_tables;
    int64_t bt_stride;
    const int32_t* cu_seqlens;
    const int32_t* kv_lens;
    const int64_t* positions;
    const int32_t* row_map;
    const int32_t* pool_lens;
    const char* new_k;
    const char* new_v;
    int64_t n_sr, n_sh;
    int G;
    int head_dim;
    float scale_log2;    // |scale| * log2(e), > 0
    float inv_scale_log2;
    uint32_t q_sign;     // xor applied to every Q word: flips the sign for a negative scale
    const int32_t* items;
    int num_items;
    const int32_t* dev_count;  // when set, the live item / merge count (the grid is a capacity)
    float* partials;
    int part_dstride;  // floats per column of a partial slot's output block
    const int32_t* merges;  // plan merge records (fused split-K merge)
    int32_t* counters;      // per-group arrival counters; null = separate merge kernel
    // Written-in-flight launch (mf_paged_attention_kv_write; the kernels'
    // TAIL instances): a sequence's keys at or above kv_len - rows are its own
    // new rows, read from new_k/new_v (row cu_seqlens[s] + key - (kv_len -
    // rows)), and the launch's first w_blocks workgroups copy new rows
    // [0, w_rows) into the pool through w_slots (a slot < 0 or >= w_num_slots
    // is skipped). No item reads a slot that this launch writes, so nothing
    // waits on the copy.
    int num_kv_heads;
    const int64_t* w_slots;
    int w_rows;
    int w_blocks;
    int64_t w_num_slots;
};

// What a scored launch (mf_scoring; the kernels' SC instances) takes besides.
struct ScoredArgs : AttnArgs {
    const float* slopes;          // per query head, or null
    const int32_t* first_keys;    // per sequence, or null
    const int32_t* prefix_lens;   // per sequence, or null
    float cap_in;    // 2 * log2(e) * |scale| / softcap, 0: scores are not capped
    float cap_log2;  // softcap * log2(e)
    float cap_x;     // |scale| / softcap
    float cap_top, cap_top4;     // largest raw scores of score_all's polynomials of three and four terms
    float cap_p3[3], cap_p4[4];  // their coefficients, raw scores to capped log2 units
};

// The launches of scored_attention.hip, as launch_attention's: padded head_dim
// dp, written in flight or not.
int launch_scored(int dtype, int dp, bool tail, const ScoredArgs& a, const int32_t* items, int64_t n_narrow,
                  int64_t n_wide, const int32_t* merges, int64_t n_merges, bool fast, const int32_t* dev_counts,
                  hipStream_t stream);

namespace {

typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(2))) float f32x2;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) short i16x4;
typedef __attribute__((ext_vector_type(4))) _Float16 f16x4;

constexpr int kWaves = 4;  // waves per workgroup; each wave runs its own item
constexpr int kMaxItemTiles = MF_MAX_ITEM_TILES;  // key tiles per work item (two block-table entries per lane)
#ifndef MF_NARROW_ITEMS
#define MF_NARROW_ITEMS 4096  // planner: target item count that sets the narrow key partition
#endif
// Wave priority (s_setprio) of the workgroup-shared wide loop. In a mixed
// launch a CU holds single-tile (decode) waves beside the wide (prefill) ones;
// at equal priority the decode waves' issue slowed the wide workgroups sharing
// their CU by about 40% (per-workgroup timestamps on the C2 step: 31.4 against
// 22.0 us median life), and the CUs holding a decode workgroup finished last.
// Raised, the wide waves issue first and the decode waves take the slots they
// leave while they wait on memory. Measured on the C2 engine layer: 53.7 us at
// equal priority, 49.3-49.8 us at 1, 49.4-49.8 at 2.
#ifndef MF_WIDE_PRIO
#define MF_WIDE_PRIO 1
#endif
// XCD-local order of the wide workgroups (1). The dispatcher sends
// workgroup b of a launch to XCD b mod 8, so the
// consecutive wide workgroups of one key range (the column groups of one
// sequence, kv head and key partition, which read the same K/V tiles) land on
// eight XCDs whose L2s each fetch the tiles. The planner instead deals whole
// ranges to eight queues (least causal work first) and interleaves them, so
// workgroup 8k + x comes from queue x and a range stays on one XCD; each
// queue runs its workgroups most causal work first. Measured on the C2
// prefill items alone: 38.2-38.8 us -> 35.1-35.5 us between events, PMC
// FETCH 74 MB -> 24 MB (1.4x the K/V and query bytes). In a mixed launch the
// wide workgroups follow the single-tile ones, which only rotates the XCDs
// (a range still shares one). There, at 32-tile wide partitions, the order
// was slower (C2 engine layer 49.2 -> 50.2 us); at 64-tile equal-stride
// partitions it was faster: 45.71-45.75 against 45.85-45.94 us, and the mixed
// plan's prefill items alone 34.7-34.9 against 39.6-39.8 us. Mixed plans now
// cut each column quad on its own (quad partitions, in the planner) and keep
// a (sequence, kv head)'s workgroups on one XCD.
#ifndef MF_WIDE_XCD
#define MF_WIDE_XCD 1
#endif
#ifndef MF_WIDE_ITEMS
#define MF_WIDE_ITEMS 4096  // planner: most wide items before partitions grow
#endif
constexpr float kLazyLog2 = 8.f;  // running-max slack of the online softmax (log2 units)
// Running maximum before any key is seen: finite, so exponent arguments never
// need a -inf guard; 2^(kMinM - x) is 0 for every score x.
constexpr float kMinM = -1e30f;

// 16-column tiles one wave carries for multi-tile (prefill / wide verify)
// items.
__host__ __device__ constexpr int wide_tiles(int dt, int dp) {
    // 16-bit: the 32 columns of one MFMA block (attn_wide_body)
    return dt == MF_F32 ? (dp >= 128 ? 2 : 4) : (dp >= 256 ? 1 : 2);
}

template <bool SC>
using ArgsOf = std::conditional_t<SC, ScoredArgs, AttnArgs>;

// Raw scores q.k brought to log2 units (what the exponent takes): the scored launch's
// scale, cap and distance bias; dist(i) is position - key of score i, either sign.
//
// tanh(x) = 1 - 2 / (e^2x + 1): one exponential and one reciprocal, exact at both
// infinities, NaN for NaN, its error about 1e-7 of the cap. Both instructions run at a
// quarter of the rate, and prefill is bound by the VALU, so where every score of the
// wave's block lies below half the cap (most do) 16-bit types take an odd polynomial
// instead, in the raw score: s (p0 + p1 z + p2 z^2 [+ p3 z^3]), z = s^2, fitted to
// tanh(x) / x for the least relative error: three terms over |x| <= 0.25 (4.0e-7), four
// over |x| <= 0.5 (5.4e-7). One test of the block's largest magnitude picks. With four
// terms alone and x formed first, two chunks of 2048 rows after up to 6144 keys took 707
// us at a cap that no score comes near (40/8 heads x 128, 475 GFLOP), 665 with both; at
// one whose quarter many pass 746 and 752 us. Slots that no row sees are cleared and pick
// nothing; where another row's score of the block passes half the cap, a row's scores are
// off by 1e-7 of the cap, 2e-7 of that score. fp32 takes the series to x^11 below 0.35 (the
// next term is 2e-8 of x there) score by score: its launches are not bound by this.
template <int DT, int N, class Dist>
__device__ __forceinline__ void score_all(float (&s)[N], const ScoredArgs& a, float slope_log2, Dist dist) {
    if (a.cap_in != 0.f) {
        float top = __builtin_huge_valf();
        if constexpr (DT != MF_F32) {
            top = __builtin_fabsf(s[0]);
#pragma unroll
            for (int i = 1; i < N; ++i) top = fmax_prop(top, __builtin_fabsf(s[i]));
        }
        if (DT != MF_F32 && __builtin_amdgcn_ballot_w64(!(top <= a.cap_top)) == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float z = s[i] * s[i];
                const float c = __builtin_fmaf(z, a.cap_p3[2], a.cap_p3[1]);
                s[i] *= __builtin_fmaf(z, c, a.cap_p3[0]);
            }
        } else if (DT != MF_F32 && __builtin_amdgcn_ballot_w64(!(top <= a.cap_top4)) == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float z = s[i] * s[i];
                float c = __builtin_fmaf(z, a.cap_p4[3], a.cap_p4[2]);
                c = __builtin_fmaf(z, c, a.cap_p4[1]);
                s[i] *= __builtin_fmaf(z, c, a.cap_p4[0]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float y = s[i] * a.cap_in;
                float th = 1.f - 2.f * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(y) + 1.f);
                if constexpr (DT == MF_F32) {
                    const float h = s[i] * a.cap_x, z = h * h;
                    float c = __builtin_fmaf(z, -1382.f / 155925.f, 62.f / 2835.f);
                    c = __builtin_fmaf(z, c, -17.f / 315.f);
                    c = __builtin_fmaf(z, c, 2.f / 15.f);
                    c = __builtin_fmaf(z, c, -1.f / 3.f);
                    th = z < 0.1225f ? __builtin_fmaf(h * z, c, h) : th;
                }
                s[i] = th * a.cap_log2;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] *= a.scale_log2;
    }
    if (a.slopes) {
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] = __builtin_fmaf(-slope_log2, __builtin_fabsf(dist(i)), s[i]);
    }
}

// The copy of a written-in-flight launch: workgroup `wblock` of the leading
// w_blocks. Every new row's K and V, head by head, go to the pool slot of
// w_slots in 16-byte pieces: consecutive lanes take consecutive pieces of one
// row (its heads are adjacent), so loads and stores coalesce.
template <int DT>
__device__ __forceinline__ void write_new_rows(const AttnArgs& a, int wblock) {
    constexpr int ES = DT == MF_F32 ? 4 : 2;
    const int cpr = a.head_dim * ES / 16;  // 16-byte pieces of one head's row
    const int per_row = 2 * a.num_kv_heads * cpr;
    const int total = a.w_rows * per_row;
    for (int u = wblock * 256 + (int)threadIdx.x; u < total; u += a.w_blocks * 256) {
        const int row = u / per_row;
        int rest = u - row * per_row;
        const int isv = rest >= a.num_kv_heads * cpr;
        rest -= isv * a.num_kv_heads * cpr;
        const int head = rest / cpr;
        const int piece = rest - head * cpr;
        const int64_t slot = a.w_slots[row];
        if (slot < 0 || slot >= a.w_num_slots) continue;
        const int64_t blk = slot / a.block_size;
        const int64_t off = slot - blk * a.block_size;
        const char* src = (isv ? a.new_v : a.new_k) + ((int64_t)row * a.n_sr + (int64_t)head * a.n_sh) * ES + piece * 16;
        char* dst = const_cast<char*>(isv ? a.v_pool : a.k_pool) +
                    (blk * a.p_sb + off * a.p_ss + (int64_t)head * a.p_sh) * ES + piece * 16;
        *(uint4*)dst = *(const uint4*)src;
    }
}

// ------------------------------------------------------------- MFMA wrappers
// S^T tile: 16 keys x 16 columns, contraction over one 16-byte chunk of
// head_dim per lane (8 x 16-bit or 4 x fp32 elements).
template <int DT>
__device__ __forceinline__ f32x4 mfma_qk(uint4 a, uint4 b, f32x4 c) {
    if constexpr (DT == MF_BF16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                       __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    } else if constexpr (DT == MF_F16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                      __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    } else {
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.x), __uint_as_float(b.x), c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.y), __uint_as_float(b.y), c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.z), __uint_as_float(b.z), c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.w), __uint_as_float(b.w), c, 0, 0, 0);
        return c;
    }
}

// O^T tile: 16 head_dim rows x 16 columns, contraction over 16 keys
// (4 per lane) for 16-bit types.
template <int DT>
__device__ __forceinline__ f32x4 mfma_pv16(uint2 a, uint2 b, f32x4 c) {
    if constexpr (DT == MF_BF16) {
        return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(i16x4, a),
                                                         __builtin_bit_cast(i16x4, b), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, a),
                                                     __builtin_bit_cast(f16x4, b), c, 0, 0, 0);
    }
}

// ---------------------------------------------------------- memory helpers

template <int N>
__device__ __forceinline__ void ld_words(const char* p, uint32_t* w) {
    if constexpr (N == 4) {
        w[0] = *(const uint32_t*)p;
    } else if constexpr (N == 8) {
        const uint2 v = *(const uint2*)p;
        w[0] = v.x; w[1] = v.y;
    } else {
        static_assert(N % 16 == 0, "chunk");
#pragma unroll
        for (int k = 0; k < N / 16; ++k) {
            const uint4 v = *(const uint4*)(p + 16 * k);
            w[4 * k] = v.x; w[4 * k + 1] = v.y; w[4 * k + 2] = v.z; w[4 * k + 3] = v.w;
        }
    }
}

// The same loads marked non-temporal (streamed, not kept in cache): pool
// tiles of single-column-tile items are read by exactly one wave.
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ uint4 ld_nt16(const char* p) {
    const u32x4 v = __builtin_nontemporal_load((const u32x4*)p);
    return make_uint4(v.x, v.y, v.z, v.w);
}
// 16 bytes per lane from global memory straight into LDS (gfx950's
// global_load_lds_dwordx4): lane i's bytes land at lds_addr + 16 i, lds_addr
// being the same for the whole wave. Written as inline assembly because the
// builtin makes the compiler wait for the transfer before every later LDS
// read; the caller waits for it (vmcnt) before the barrier that publishes it.
// The LDS address is bound to m0 by the operand constraint, so the compiler
// writes m0 itself and knows what it holds (a clobber of the reserved m0
// would not be honoured); the s_nop gives the write its one wait state before
// the load reads it.
__device__ __forceinline__ void ld_lds16(const void* gsrc, uint32_t lds_addr) {
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"{m0}"(lds_addr), "v"(gsrc) : "memory");
}

template <int N>
__device__ __forceinline__ void ld_words_nt(const char* p, uint32_t* w) {
    if constexpr (N == 4) {
        w[0] = __builtin_nontemporal_load((const uint32_t*)p);
    } else if constexpr (N == 8) {
        const u32x2 v = __builtin_nontemporal_load((const u32x2*)p);
        w[0] = v.x; w[1] = v.y;
    } else {
        static_assert(N % 16 == 0, "chunk");
#pragma unroll
        for (int k = 0; k < N / 16; ++k) {
            const uint4 v = ld_nt16(p + 16 * k);
            w[4 * k] = v.x; w[4 * k + 1] = v.y; w[4 * k + 2] = v.z; w[4 * k + 3] = v.w;
        }
    }
}

template <int N>
__device__ __forceinline__ void st_words(char* p, const uint32_t* w) {
    if constexpr (N == 4) {
        *(uint32_t*)p = w[0];
    } else if constexpr (N == 8) {
        *(uint2*)p = make_uint2(w[0], w[1]);
    } else {
        static_assert(N % 16 == 0, "chunk");
#pragma unroll
        for (int k = 0; k < N / 16; ++k)
            *(uint4*)(p + 16 * k) = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
    }
}

// Writes NE contiguous output elements (value e is vals[e]) in dtype DT.
template <int DT, int NE>
__device__ __forceinline__ void store_elems(char* p, const float* vals) {
    if constexpr (DT == MF_F32) {
        uint32_t w[NE];
#pragma unroll
        for (int e = 0; e < NE; ++e) w[e] = __float_as_uint(vals[e]);
        st_words<NE * 4>(p, w);
    } else {
        uint32_t w[NE / 2];
#pragma unroll
        for (int e = 0; e < NE / 2; ++e)
            w[e] = f32_to_bits<DT>(vals[2 * e]) | (f32_to_bits<DT>(vals[2 * e + 1]) << 16);
        st_words<NE * 2>(p, w);
    }
}

// Writes the lane's contiguous chunk of 4*VCH output elements.
template <int DT, int VCH>
__device__ __forceinline__ void store_out_chunk(char* p, const float* vals) {
    store_elems<DT, 4 * VCH>(p, vals);
}

// ------------------------------------------------------------- split-K merge
// Partials of one 16-column tile (merge record `mg`) live in slots
// slot0 + p*sstride, p < np. A slot holds, per column, the partition's
// normalised output o_p / l_p in the launch's element type (column c at
// element c*part_dstride), then 16 running maxima m_p and 16 sums l_p (fp32,
// at float 16*part_dstride). The merged output is
// sum_p w_p l_p (o_p / l_p) / sum_p w_p l_p with w_p = 2^(m_p - max_p m_p).
// A normalised output is a convex combination of V rows, so it keeps the
// output type's range; 16-bit partials halve the bytes written and merged
// against fp32 ones, for one more rounding to that type.
// Records and items flagged MF_PLAN_FP32_PARTIALS hold the outputs in fp32
// instead (the slot has the room): a device's decode plan cuts ranges that the
// general plan runs as one cooperative unit, whose waves combine in fp32, and the
// cut must not round what the whole unit does not. 16-bit launches of 256-byte
// rows and more only, as that rule. Scored launches and those over a 4-bit pool keep
// every partial in fp32.
template <int DT, int DP>
constexpr bool has_fp32_partials() { return DT != MF_F32 && DP >= 128; }
template <int DT>
__device__ __forceinline__ char* partial_out(const AttnArgs& a, int64_t slot, int col, int elem) {
    constexpr int ES = DT == MF_F32 ? 4 : 2;
    return (char*)(a.partials + slot * (16 * (int64_t)(a.part_dstride + 2))) +
           ((int64_t)col * a.part_dstride + elem) * ES;
}
__device__ __forceinline__ float* partial_ml(const AttnArgs& a, int64_t slot) {
    return a.partials + slot * (16 * (int64_t)(a.part_dstride + 2)) + 16 * a.part_dstride;
}

// merge_range accumulates partitions p0, p0+pinc, ... relative to their own
// maximum `mx` (lane (g, j): column j, head_dim range [4g*VCH, 4g*VCH+4*VCH)).
// Partitions go four at a time with every load of a batch issued before any
// is used (a batch past the last partition loads only what exists; the
// condition is wave-uniform), and the running maximum moves batch to batch:
// a merge of n partitions per wave costs ceil(n/4) memory round trips. PT: the
// type of the partial outputs; B: partitions per batch.
template <int DT, int DP, int PT = DT, int B = 4>
__device__ __forceinline__ void merge_range(const AttnArgs& a, const int32_t* mg, int p0, int pinc, int j,
                                            int dbase, float& mx, float& L, float (&o)[DP / 4]) {
    constexpr int VCH = DP / 16;
    constexpr int ES = PT == MF_F32 ? 4 : 2;
    constexpr int NW = 4 * VCH * ES / 4;  // words of the lane's chunk
    const int np = mg[3], slot0 = mg[4], sstride = mg[5];
    mx = kMinM;
    L = 0.f;
#pragma unroll
    for (int e = 0; e < 4 * VCH; ++e) o[e] = 0.f;
    for (int p = p0; p < np; p += B * pinc) {
        uint32_t raw[B][NW];
        float mb[B], lb[B];
#pragma unroll
        for (int b = 0; b < B; ++b) {
            if (p + b * pinc < np) {
                const int64_t slot = slot0 + (int64_t)(p + b * pinc) * sstride;
                ld_words<4 * VCH * ES>(partial_out<PT>(a, slot, j, dbase), raw[b]);
                const float* ml = partial_ml(a, slot);
                mb[b] = ml[j];
                lb[b] = ml[16 + j];
            } else {
#pragma unroll
                for (int e = 0; e < NW; ++e) raw[b][e] = 0u;
                mb[b] = kMinM;
                lb[b] = 0.f;
            }
        }
        float bm = mx;
#pragma unroll
        for (int b = 0; b < B; ++b) bm = fmaxf(bm, mb[b]);
        const float keep = __builtin_amdgcn_exp2f(mx - bm);
        L *= keep;
#pragma unroll
        for (int e = 0; e < 4 * VCH; ++e) o[e] *= keep;
#pragma unroll
        for (int b = 0; b < B; ++b) {
            const float wl = __builtin_amdgcn_exp2f(mb[b] - bm) * lb[b];
            L += wl;
#pragma unroll
            for (int e = 0; e < 4 * VCH; ++e) {
                float v;
                if constexpr (PT == MF_F32) v = __uint_as_float(raw[b][e]);
                else v = bits_to_f32<PT>((raw[b][e >> 1] >> (16 * (e & 1))) & 0xffffu);
                o[e] += wl * v;
            }
        }
        mx = bm;
    }
}

// Output row/head of column tile ct's column j, or false for a padding column.
// mg: a merge record (s, h, column tile, parts, slot0, slot stride, first row,
// rows and flag)
__device__ __forceinline__ bool merge_column(const AttnArgs& a, const int32_t* mg, int j, int& prow, int& qhead) {
    const int h = mg[1], ct = mg[2];
    const int row0 = mg[6];
    const int ncols = (mg[7] & ~MF_PLAN_FP32_PARTIALS) * a.G;
    const int cidx = ct * 16 + j;
    if (cidx >= ncols) return false;
    const int r = cidx / a.G;
    prow = row0 + r;
    if (a.row_map) prow = a.row_map[prow];
    qhead = h * a.G + (cidx - r * a.G);
    return true;
}

// Single-wave merge of one record. FP32B: partitions per batch of a record of
// fp32 partials, 0 where the caller's records have none (prefill items). ALL32: every
// record's are.
template <int DT, int DP, int FP32B = 0, bool ALL32 = false>
__device__ __forceinline__ void merge_tile(const AttnArgs& a, const int32_t* mg, int g, int j) {
    constexpr int VCH = DP / 16;
    constexpr int ES = DT == MF_F32 ? 4 : 2;
    int prow, qhead;
    const int dbase = 4 * g * VCH;
    if (!merge_column(a, mg, j, prow, qhead) || dbase >= a.head_dim) return;
    float mx, L, o[4 * VCH];
    bool merged = false;
    if constexpr (ALL32) {
        merge_range<DT, DP, MF_F32, FP32B>(a, mg, 0, 1, j, dbase, mx, L, o);
        merged = true;
    } else if constexpr (has_fp32_partials<DT, DP>() && FP32B > 0) {
        if (mg[7] & MF_PLAN_FP32_PARTIALS) {
            merge_range<DT, DP, MF_F32, FP32B>(a, mg, 0, 1, j, dbase, mx, L, o);
            merged = true;
        }
    }
    if (!merged) merge_range<DT, DP>(a, mg, 0, 1, j, dbase, mx, L, o);
    const float inv = L > 0.f ? 1.f / L : 0.f;
#pragma unroll
    for (int e = 0; e < 4 * VCH; ++e) o[e] *= inv;
    store_out_chunk<DT, VCH>(a.out + ((int64_t)prow * a.o_sr + (int64_t)qhead * a.o_sh + dbase) * ES, o);
}

// Fused split-K merge: the last partition of a group to arrive merges the
// group. Release the partials (agent-scope fence: the L2s of the XCDs are not
// coherent with each other), count the arrival, and on the last arrival
// acquire everyone else's partials and reset the counter for the next call.
// Every wave runs to the end; nothing waits on another wave.
template <int DT, int DP>
__device__ __forceinline__ void arrive_and_merge(const AttnArgs& a, int m0, int nct, int lane) {
    if (a.counters == nullptr) return;
    __threadfence();
    int prev = 0;
    if (lane == 0) prev = atomicAdd(a.counters + m0, 1);
    prev = __shfl(prev, 0, 64);
    const int32_t* mg0 = a.merges + (int64_t)m0 * MF_PLAN_MERGE_INTS;
    if (prev == mg0[3] - 1) {
        __threadfence();
        if (lane == 0) a.counters[m0] = 0;
        for (int o = 0; o < nct; ++o) merge_tile<DT, DP>(a, mg0 + o * MF_PLAN_MERGE_INTS, lane >> 4, lane & 15);
    }
}

// -------------------------------------------------------------- main kernel
// Waves per SIMD the register allocator must leave room for: two where the
// kernel fits in 256 registers without spilling (key rows up to 128 bytes,
// or up to 256 bytes for single-tile items), else one. 16-bit wide kernels are
// held to what the shared loop gains from, four (three at 256-byte rows). There
// the whole kernel, with the wave-by-wave body beside the loop, spills at 168
// registers: 61 to 67 vector and 22 to 24 scalar ones, 236 to 244 bytes of
// scratch (50 to 55 vector ones on other block sizes than 16). Compiled without
// that body the loop spills 1 or 2 (9).
#ifndef MF_WIDE_WAVES
#define MF_WIDE_WAVES(dp) ((dp) == 128 ? 3 : 4)
#endif
// Scored wide launches at 256-byte rows run two waves of 64-key stages and softmax steps
// (two score chains at once, one test of the maximum for both): the transforms' registers
// spill at three. Two chunks of 2048 rows after up to 6144 keys, 40/8 heads x 128, capped
// scores (475 GFLOP): 836 us at three waves and 32 keys, 778 at two, 698 with stages of
// 64, 689 with steps of 64 (since then the cap's polynomials and the stages' addresses:
// 648 to 685 over several cards). At 128-byte rows four waves and 32-key steps stay the
// faster (8 packed prompts of documents 49 us, 57 at three waves with steps of 64).
constexpr int scored_waves(int dp) { return dp == 128 ? 2 : 4; }
constexpr int scored_step(int dp) { return dp == 128 ? 2 : 1; }  // 32-key blocks
template <int DT, int DP, int NT, bool SC = false>
constexpr int attn_waves_per_eu() {
    constexpr int row_bytes = DP * (DT == MF_F32 ? 4 : 2);
    if (DT != MF_F32 && NT > 1) return SC ? scored_waves(DP) : MF_WIDE_WAVES(DP);
    return (row_bytes <= 128 || (row_bytes <= 256 && NT == 1)) ? 2 : 1;
}

// Register buffers of the single-column-tile key pipeline: the tile being
// processed plus the two in flight. Measured on MI355X for 128-byte rows
// (bf16 D 64): four and six buffers were no faster than three, and eight
// slower (they cost waves per SIMD); a 256-byte row's buffer is 32 registers,
// and three fit the two-waves-per-SIMD budget.
// One launch for plans holding both single-tile and wide items (see
// attn_mixed_kernel); 0 launches them one after the other.
#ifndef MF_MIXED_LAUNCH
#define MF_MIXED_LAUNCH 1
#endif

// Tiles of extra work the planner charges to the last wave of a cooperative
// unit that holds a multi-row sequence's last tile. Measured on C3's verify
// layer (graph replays): 0 13.2 us, 2 12.96-12.99, 4 12.93-12.94, 6
// 12.36-12.37, 8 12.34-12.37, 10 13.22-13.24, 12 13.18-13.19, 16 13.0. In an
// instrumented build's timeline those waves started their key loop 1.1 us
// after the unit's other waves and ran the boundary and in-flight tiles after
// it, while the others waited at the combine.
#ifndef MF_TAIL_WAVE_TILES
#define MF_TAIL_WAVE_TILES 6
#endif

#ifndef MF_NARROW_DEPTH
#define MF_NARROW_DEPTH 3
#endif

// LDS of the attention kernels: one dynamically sized arena per workgroup.
// A workgroup uses at most one of its two layouts -- the wide items'
// double-buffered K/V stages (workgroup-shared key loop) or the cooperative
// units' softmax states (narrow items) -- so a launch that runs both kinds of
// workgroup (attn_mixed_kernel) sizes the arena for the larger, not for both.
extern __shared__ __attribute__((aligned(16))) char attn_lds[];

// Workgroup-shared prefill loop (attn_wide_body): keys per LDS stage (two
// stage buffers: the stage being computed and the one arriving).
#ifndef MF_WIDE_KEYS
#define MF_WIDE_KEYS(dp) ((dp) == 128 ? 32 : 64)
#endif
constexpr int wide_keys(int dp, bool sc) { return sc ? 64 : MF_WIDE_KEYS(dp); }
template <int DT, int DP, bool SC>
constexpr int wide_lds_bytes() {
    if constexpr (DT == MF_F32) return 0;  // the workgroup-shared loop is 16-bit only
    else return 2 * 2 * wide_keys(DP, SC) * DP * 2;
}
template <int DP>
constexpr int coop_lds_bytes() {
    return (kWaves * 4 * (DP / 16) * 64 + 2 * kWaves * 16) * 4;
}
template <int DT, int DP, int NT, bool FAST, bool SC = false>
constexpr int attn_lds_bytes() {
    if constexpr (NT == 1) return coop_lds_bytes<DP>();
    else return wide_lds_bytes<DT, DP, SC>();
}

// The body of one workgroup of the attention kernel: `block` is its index
// among the workgroups that run items of this column-tile width.
// TAIL: a written-in-flight launch (compiled apart, so the other launches
// keep their register budget). SC: a scored launch, likewise: scores are taken
// to log2 units before the mask (scored()) instead of inside the exponent, and
// keys below the sequence's first are masked and their V rows cleared, a row's
// last key is the later of its position and the sequence's prefix.
template <int DT, int DP, int NT, bool FAST, bool TAIL = false, bool SC = false>
__device__ __forceinline__ void attn_body(const ArgsOf<SC>& a, const int block) {
    constexpr int ES = DT == MF_F32 ? 4 : 2;
    constexpr int EPL = 16 / ES;      // elements per 16-byte chunk
    constexpr int NL = DP * ES / 64;  // 16-byte K/Q chunks per lane
    constexpr int VCH = DP / 16;      // V elements per lane per key (= d tiles)
    constexpr int VB = VCH * ES;      // bytes of one lane's V chunk
    constexpr int VWD = VB / 4;       // 32-bit words of one lane's V chunk
    static_assert(NL >= 1 && VWD >= 1, "head_dim too small for this dtype");
    constexpr float kNegInf = -__builtin_huge_valf();

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int item = block * kWaves + wave;
    // The item carries its sequence's first row, row count and kv length (the
    // planner's copies of cu_seqlens / kv_lens), so nothing waits on loading
    // them before the row positions and block table are fetched.
    const int32_t* it = a.items + (int64_t)item * MF_PLAN_ITEM_INTS;
    int4 iv0, iv1, iv2;
    if constexpr (NT == 1) {
        // Single-tile items load their item before the count check, together
        // with the argument block that the check reads (the item list's
        // address needs no argument load when it is preloaded), instead of
        // one round trip after it. The item is in bounds past the live count:
        // plans fill whole workgroups and counted launches size the list by
        // its capacity. The empty asm keeps the loads ahead of the check.
        // Wide items keep the order below: their setup issues the item with
        // the workgroup's other items' keys in one batch after the check.
        iv0 = *(const int4*)it;
        iv1 = *(const int4*)(it + 4);
        iv2 = *(const int4*)(it + 8);
        asm volatile("" ::"s"(iv0.x), "s"(iv0.y), "s"(iv0.z), "s"(iv0.w), "s"(iv1.x), "s"(iv1.y), "s"(iv1.z),
                     "s"(iv1.w), "s"(iv2.x), "s"(iv2.y), "s"(iv2.z), "s"(iv2.w));
        // ... and so do the argument fields the next batch of loads (block
        // table, row positions, Q) is addressed from, which otherwise come
        // from argument cache lines fetched after the check
        asm volatile("" ::"s"(a.block_tables), "s"(a.bt_stride), "s"(a.positions), "s"(a.pool_lens), "s"(a.q),
                     "s"(a.q_sr), "s"(a.q_sh), "s"(a.G), "s"(a.row_map), "s"(a.q_sign));
    }
    const int num_items = a.dev_count ? *a.dev_count : a.num_items;
    if (item >= num_items) return;
    if constexpr (NT != 1) {
        iv0 = make_int4(it[0], it[1], it[2], it[3]);
        iv1 = make_int4(it[4], it[5], it[6], it[7]);
        iv2 = make_int4(it[8], it[9], it[10], it[11]);
    }
    const int lane = threadIdx.x & 63;
    const int g = lane >> 4;  // 16-lane group: MFMA k-group / output row group
    const int j = lane & 15;  // MFMA column (query column) and A-row (key) index

    const int s = iv0.x, h = iv0.y, c0 = iv0.z, nct = iv0.w;
    const int kt0 = iv1.x, kt1 = iv1.y, pslot = iv1.z;
    const int row0 = iv2.x;
    const int ncols = iv2.y * a.G;
    const int kv_len = iv2.z;
    // Keys below pool_len are in the pool; the rest are in-flight rows of the
    // sequence's own new tokens (a verify pass: pool_lens; a written-in-flight
    // step: everything past the keys before the sequence's rows).
    const bool inflight = TAIL || a.pool_lens != nullptr;
    const int pool_len = TAIL ? kv_len - iv2.y : (a.pool_lens != nullptr ? a.pool_lens[s] : kv_len);
    const int D = a.head_dim;
    int first = 0, prefix = 0;
    if constexpr (SC) {
        if (a.first_keys) first = a.first_keys[s];
        if (a.prefix_lens) prefix = a.prefix_lens[s];
    }

    // The loads that need nothing but the item go out together -- block-table
    // entries first (loads retire in issue order, and the first K/V tiles
    // wait only on them), then row positions, then Q -- so the setup costs
    // one round trip before the K/V stream starts, not three.
    //
    // ---- block-table entries of the item's tiles, two per lane (tile kt0+l
    // and kt0+64+l; fast path, at most kMaxItemTiles), read back with
    // readlane. On a verify pass
    // that is every tile holding a pool key (the boundary tile included);
    // pool_end is the end of the tiles lying wholly in the pool.
    const int tbl_end = inflight ? max(kt0, min(kt1, (pool_len + 15) >> 4)) : kt1;
    const int pool_end = inflight ? max(kt0, min(kt1, pool_len >> 4)) : kt1;
    int tbl = 0, tbl_hi = 0;
    const int tbl_base = kt0;
    if constexpr (FAST) {
        // Every lane loads (a clamped entry past the item's tiles, entry 0 of
        // the row for an item without tiles; only entries of the item's own
        // tiles are ever read back), so no branch skips a load and nothing
        // consumes the values before the other setup loads are issued: the
        // count of loads in flight is the same on every path and later waits
        // stay exact.
        const int idx = kt0 + lane;
        const int32_t* row = a.block_tables + (int64_t)s * a.bt_stride;
        const bool any = tbl_end > kt0;
        tbl = row[any ? min(idx, tbl_end - 1) : 0];
        if constexpr (kMaxItemTiles > 64) tbl_hi = row[any ? min(idx + 64, tbl_end - 1) : 0];
    }
    // physical block of the item's tile i (wave-uniform i)
    auto tbl_at = [&](int i) -> int {
        const int lo = __builtin_amdgcn_readlane(tbl, i & 63);
        if constexpr (kMaxItemTiles > 64) return i < 64 ? lo : __builtin_amdgcn_readlane(tbl_hi, i & 63);
        return lo;
    };

    // ---- columns owned by this lane (one per tile)
    int prow[NT], qhead[NT], qpos[NT];
    bool qvalid[NT];
    int at_pos[NT];   // SC: the row's own position, which the distance counts from
    float slope[NT];  // SC: in log2 units
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        // padding columns read row0's position and query (unconditional
        // loads, results discarded)
        const int cidx = (c0 + nt) * 16 + j;
        const bool valid = nt < nct && cidx < ncols;
        const int r = valid ? cidx / a.G : 0;
        const int gq = valid ? cidx - r * a.G : 0;
        int pr = row0 + r;
        if (a.row_map) pr = a.row_map[pr];
        // the low word of the little-endian int64 position (what the int
        // conversion keeps): a 64-bit load's unused high register would be
        // reused as a temporary, and that write waits for the load
        const int pos = reinterpret_cast<const int32_t*>(a.positions)[2 * (int64_t)pr];
        prow[nt] = pr;
        qhead[nt] = h * a.G + gq;
        qpos[nt] = valid ? (SC ? max(pos, prefix - 1) : pos) : -1;
        qvalid[nt] = valid;
        if constexpr (SC) {
            at_pos[nt] = pos;
            slope[nt] = a.slopes ? a.slopes[qhead[nt]] * 1.4426950408889634f : 0.f;
        }
    }

    // ---- Q fragments (MFMA B operand of S^T = K Q^T): lane (g, j) holds
    // column j's head_dim chunk (c*4 + g) for c < NL.
    uint4 qf[NT][NL];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int c = 0; c < NL; ++c) {
            const int d0 = (c * 4 + g) * EPL;
            // A padding column holds row0's query (its scores are computed
            // and never stored; every column has its own softmax state).
            uint4 v = make_uint4(0, 0, 0, 0);
            if (FAST || d0 < D)  // the fast path has head_dim == DP: every chunk exists
                v = *(const uint4*)(a.q + ((int64_t)prow[nt] * a.q_sr + (int64_t)qhead[nt] * a.q_sh + d0) * ES);
            qf[nt][c] = make_uint4(v.x ^ a.q_sign, v.y ^ a.q_sign, v.z ^ a.q_sign, v.w ^ a.q_sign);
        }
    }

    // General path: address of key `key`'s row for this kv head, or null.
    auto key_row = [&](const char* pool, const char* inflight, int key) -> const char* {
        if (key >= kv_len) return nullptr;
        if (key < pool_len) {
            const int blk = key / a.block_size;
            const int off = key - blk * a.block_size;
            const int phys = a.block_tables[(int64_t)s * a.bt_stride + blk];
            return pool + ((int64_t)phys * a.p_sb + (int64_t)off * a.p_ss + (int64_t)h * a.p_sh) * ES;
        }
        int nr = row0 + (key - pool_len);
        if (a.row_map) nr = a.row_map[nr];
        return inflight + ((int64_t)nr * a.n_sr + (int64_t)h * a.n_sh) * ES;
    };

    // byte offsets of this lane's K chunk (key j, chunk g) and V chunk (keys
    // 4g.., head_dim j*VCH..) inside one block of one kv head
    const uint32_t k_lane_off = (uint32_t)(((int64_t)j * a.p_ss + g * EPL) * ES);
    const uint32_t v_row_bytes = (uint32_t)(a.p_ss * ES);
    const uint32_t v_lane_off = (uint32_t)(((int64_t)(4 * g) * a.p_ss + j * VCH) * ES);
    // Per-key loads of tile kt (the verify boundary and in-flight tiles, and
    // every tile off the fast path). On the fast path a tile's pool keys all
    // lie in one block, whose entry is already in tbl.
    // has_map: the launch has a row map (a compile-time copy of each case:
    // with the map read behind a runtime test, the five row lookups below
    // each ended in a wait for every load in flight, row map or not -- on a
    // verify pass the boundary tile's wave then started its key loop 2.3 us
    // after the others and held up its cooperative unit)
    auto load_general_m = [&](int kt, uint4 (&kf)[NL], uint32_t (&vf)[4][VWD], auto has_map) {
        int phys = 0;
        if constexpr (FAST) phys = kt < tbl_end ? tbl_at(kt - tbl_base) : 0;
        auto row = [&](const char* pool, const char* inflight, int key) -> const char* {
            if constexpr (FAST) {
                if (key >= kv_len) return nullptr;
                if (key < pool_len)
                    return pool + ((int64_t)phys * a.p_sb + (int64_t)(key & 15) * a.p_ss + (int64_t)h * a.p_sh) * ES;
                int nr = row0 + (key - pool_len);
                if constexpr (decltype(has_map)::value) nr = a.row_map[nr];
                return inflight + ((int64_t)nr * a.n_sr + (int64_t)h * a.n_sh) * ES;
            } else {
                return key_row(pool, inflight, key);
            }
        };
        const char* kp = row(a.k_pool, a.new_k, kt * 16 + j);
#pragma unroll
        for (int c = 0; c < NL; ++c) {
            const int d0 = (c * 4 + g) * EPL;
            kf[c] = (kp && d0 < D) ? *(const uint4*)(kp + (int64_t)d0 * ES) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const char* vp = row(a.v_pool, a.new_v, kt * 16 + 4 * g + r);
            if (vp && j * VCH < D) {
                ld_words<VB>(vp + (int64_t)j * VCH * ES, vf[r]);
            } else {
#pragma unroll
                for (int w = 0; w < VWD; ++w) vf[r][w] = 0;
            }
        }
    };
    auto load_general = [&](int kt, uint4 (&kf)[NL], uint32_t (&vf)[4][VWD]) {
        if (FAST && a.row_map) load_general_m(kt, kf, vf, std::true_type{});
        else load_general_m(kt, kf, vf, std::false_type{});
    };
    // Lane byte offsets of the V rows 4g..4g+3 inside a block, computed once.
    uint32_t v_off[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) v_off[r] = v_lane_off + (uint32_t)r * v_row_bytes;
    // A dummy load (a prefetch slot past the item's last tile) keeps the
    // chunk offsets but drops the lane offsets: the wave reads the block's
    // first few lines instead of the whole tile again. `none` (wave-uniform):
    // the item has no pool tile at all, and the dummy reads the start of Q,
    // which every call has.
    auto load_tile = [&](int kt, uint4 (&kf)[NL], uint32_t (&vf)[4][VWD], bool dummy = false, bool none = false) {
        if constexpr (FAST) {
            // block base is wave-uniform (scalar registers); the lane's byte
            // offsets inside a block never change
            const int phys = tbl_at(kt - tbl_base);
            const int64_t boff = ((int64_t)phys * a.p_sb + (int64_t)h * a.p_sh) * ES;
            const char* kb = none ? a.q : a.k_pool + boff;
            const char* vb = none ? a.q : a.v_pool + boff;
            const uint32_t sel = (dummy || none) ? 0u : 0xffffffffu;
            const uint32_t ko = k_lane_off & sel;
            if constexpr (NT == 1 && DP * ES >= 256) {
                // non-temporal only for rows of 256 bytes or more: measured
                // faster there (bf16 D 128) and slower for 128-byte rows
#pragma unroll
                for (int c = 0; c < NL; ++c) kf[c] = ld_nt16(kb + ko + c * 4 * 16);
#pragma unroll
                for (int r = 0; r < 4; ++r) ld_words_nt<VB>(vb + (v_off[r] & sel), vf[r]);
            } else {
#pragma unroll
                for (int c = 0; c < NL; ++c) kf[c] = *(const uint4*)(kb + ko + c * 4 * 16);
#pragma unroll
                for (int r = 0; r < 4; ++r) ld_words<VB>(vb + (v_off[r] & sel), vf[r]);
            }
        } else {
            load_general(kt, kf, vf);
        }
    };

    // The first NB-1 tiles of a single-column-tile (decode) item go out with
    // the setup loads: positions only trim the item's key range, and these
    // tiles lie in it whenever the item has any. Slots past the item's tiles
    // take a one-line dummy load.
    // The loads are unconditional -- an item without pool tiles issues dummy
    // ones -- so the count of loads in flight is the same on every path and
    // the first use of Q waits for Q alone, not for these tiles too.
    constexpr int NB = NT == 1 ? MF_NARROW_DEPTH : 2;
    uint4 kR[NB][NL];
    uint32_t vR[NB][4][VWD];
    if constexpr (FAST && NT == 1) {
        const bool none = kt0 >= pool_end;
#pragma unroll
        for (int i = 0; i < NB - 1; ++i)
            load_tile(max(kt0, min(kt0 + i, pool_end - 1)), kR[i], vR[i], kt0 + i > pool_end - 1, none);
    }

    int maxpos = -1;
    int minpos = INT_MAX;  // over the item's real columns
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        maxpos = max(maxpos, qpos[nt]);
        if (qvalid[nt]) minpos = min(minpos, qpos[nt]);
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
        maxpos = max(maxpos, __shfl_xor(maxpos, off, 64));
        minpos = min(minpos, __shfl_xor(minpos, off, 64));
    }
    minpos = __builtin_amdgcn_readfirstlane(minpos);
    // last key each lane's column may see (-1 for padding columns)
    int lim[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) lim[nt] = qpos[nt] >= 0 ? min(qpos[nt], kv_len - 1) : -1;
    // Tiles past the last key any column may see are never read.
    int kt_end = min(kt1, (min(maxpos, kv_len - 1) >> 4) + 1);
    if (maxpos < 0 || kv_len <= 0) kt_end = kt0;
    kt_end = __builtin_amdgcn_readfirstlane(kt_end);

    // m: running max of the scaled scores (log2 units); thr: the raw score
    // above which a column's running max must move, (m + kLazyLog2) / scale.
    float m[NT], l[NT], thr[NT];
    f32x4 acc[NT][VCH];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        m[nt] = kMinM;
        thr[nt] = SC ? kMinM + kLazyLog2 : (kMinM + kLazyLog2) * a.inv_scale_log2;
        l[nt] = 0.f;
#pragma unroll
        for (int c = 0; c < VCH; ++c) acc[nt][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    // K: lane (g, j) loads key j's head_dim chunks (c*4 + g).
    // V: lane (g, j) loads keys 4g..4g+3, head_dim elements [j*VCH, j*VCH+VCH).
    // FAST path (16-token blocks, head_dim == DP): every
    // load is unconditional, so the compiler can keep the next tile's loads in
    // flight while the current tile is processed.
    // Tiles [kt0, fast_end) run through the pipelined loop. On the fast path
    // with in-flight keys (a verify pass) that is only the tiles lying wholly
    // in the pool; the one or two tiles holding the boundary and the in-flight
    // candidates follow through the general per-key loads.
    int fast_end = kt_end;
    if constexpr (FAST) {
        if (inflight) fast_end = max(kt0, min(kt_end, pool_len >> 4));
    }
    // Per-tile work is branch-free apart from wave-uniform decisions: every
    // column tile's MFMAs run (tiles past nct hold zero queries and are never
    // stored), and masking is a select, so the scheduler sees one straight
    // block per tile, in four parts: scores, the lazy rescale, exponentials
    // and the PV product.
    //
    // Slots past the context in the last block may hold anything, NaN
    // included; p = 0 there, but 0 * NaN is NaN, so clear them.
    auto clear_v_tail = [&](int kt, uint32_t (&vf)[4][VWD]) {
        if constexpr (SC) {
            if ((FAST && (kt + 1) * 16 > kv_len) || kt * 16 < first) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int key = kt * 16 + 4 * g + r;
                    const bool live = key >= first && key < kv_len;
#pragma unroll
                    for (int w = 0; w < VWD; ++w) vf[r][w] = live ? vf[r][w] : 0u;
                }
            }
        } else if constexpr (FAST) {
            if ((kt + 1) * 16 > kv_len) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const bool live = kt * 16 + 4 * g + r < kv_len;
#pragma unroll
                    for (int w = 0; w < VWD; ++w) vf[r][w] = live ? vf[r][w] : 0u;
                }
            }
        }
    };
    // S^T = K Q^T for every column tile (lane (g, j): keys 4g..4g+3 of
    // column j), masked. Scores stay raw; the scale is applied inside the
    // exponent, p = 2^(s * scale - m), one fma.
    auto scores = [&](int kt, const uint4 (&kf)[NL], float (&sv)[NT][4]) {
        f32x4 st[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            st[nt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < NL; ++c) st[nt] = mfma_qk<DT>(kf[c], qf[nt][c], st[nt]);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int r = 0; r < 4; ++r) sv[nt][r] = st[nt][r];
        // Every key of a tile wholly inside the context and at or before every
        // column's position is visible to all columns: no mask to apply.
        const bool edge = !(kt * 16 + 15 <= minpos && (kt + 1) * 16 <= kv_len && (!SC || kt * 16 >= first));
        if constexpr (SC) {
            // a block's largest score picks how it is capped (score_all): no hidden one does
            if (edge) {
                asm volatile("");
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        sv[nt][r] = kt * 16 + 4 * g + r <= lim[nt] && kt * 16 + 4 * g + r >= first ? sv[nt][r] : 0.f;
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float dist = (float)(kt * 16 + 4 * g - at_pos[nt]);
                score_all<DT>(sv[nt], a, slope[nt], [&](int i) { return dist + i; });
            }
        }
        if (edge) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    sv[nt][r] = kt * 16 + 4 * g + r <= lim[nt] && (!SC || kt * 16 + 4 * g + r >= first) ? sv[nt][r]
                                                                                                     : kNegInf;
        }
    };
    // Lazy rescaling: a column's running max m moves (and l, acc are
    // rescaled) only when one of its scores exceeds m by more than
    // kLazyLog2, so p = 2^(s - m) stays below 2^kLazyLog2; l and acc always
    // share the m they were built with, so the result is the same softmax.
    // Each lane tests its own four scores; the max across the column's
    // four lane groups is only formed when some lane asks for a move.
    auto needs_rescale = [&](const float (&sv)[NT][4], float (&lmax)[NT]) -> bool {
        bool grow = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            lmax[nt] = fmax_prop(fmax_prop(sv[nt][0], sv[nt][1]), fmax_prop(sv[nt][2], sv[nt][3]));
            grow |= lmax[nt] > thr[nt];
        }
        return __builtin_amdgcn_ballot_w64(grow) != 0;
    };
    auto rescale = [&](const float (&lmax)[NT]) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const float mn = fmaxf(m[nt], SC ? group_max4(lmax[nt]) : group_max4(lmax[nt]) * a.scale_log2);
            const float alpha = __builtin_amdgcn_exp2f(m[nt] - mn);
            l[nt] *= alpha;
#pragma unroll
            for (int c = 0; c < VCH; ++c) acc[nt][c] *= alpha;
            m[nt] = mn;
            thr[nt] = SC ? mn + kLazyLog2 : (mn + kLazyLog2) * a.inv_scale_log2;
        }
    };
    // p = 2^(s * scale - m) against the current running max, l += row sums;
    // packed to the 16-bit dtype for the PV MFMA, which takes both operands in
    // one type (fp32 kept as is). That rounds a weight by at most 2^-8 of it in
    // bf16, 2^-11 in fp16: an output error of 0.0019 to 0.0022 of its norm in
    // bf16 where weights kept in 32 bits leave 0.0017. l sums them unrounded.
    auto exps = [&](const float (&sv)[NT][4], uint2 (&p16)[NT], float (&p32)[NT][4]) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float p[4];
#pragma unroll
            for (int r = 0; r < 4; ++r)
                p[r] = __builtin_amdgcn_exp2f(SC ? sv[nt][r] - m[nt] : __builtin_fmaf(sv[nt][r], a.scale_log2, -m[nt]));
            l[nt] += (p[0] + p[1]) + (p[2] + p[3]);
            if constexpr (DT == MF_F32) {
#pragma unroll
                for (int r = 0; r < 4; ++r) p32[nt][r] = p[r];
            } else if constexpr (DT == MF_BF16) {
                // hardware round-to-nearest-even pack (v_cvt_pk_bf16_f32)
                p16[nt] = make_uint2(
                    __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){p[0], p[1]}, bf16x2)),
                    __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){p[2], p[3]}, bf16x2)));
            } else {
                p16[nt] = make_uint2(f32_to_bits<DT>(p[0]) | (f32_to_bits<DT>(p[1]) << 16),
                                     f32_to_bits<DT>(p[2]) | (f32_to_bits<DT>(p[3]) << 16));
            }
        }
    };
    // MFMA A operand (16-bit) of head_dim tile c: element c of keys
    // 4g..4g+3, the low (c even) or high halves of word c/2, paired by byte
    // permutes. Row i of tile c is head_dim element i*VCH + c.
    auto va16 = [&](const uint32_t (&vf)[4][VWD], int c) -> uint2 {
        const int wd = c >> 1;
        const uint32_t sel = (c & 1) ? 0x07060302u : 0x05040100u;
        return make_uint2(__builtin_amdgcn_perm(vf[1][wd], vf[0][wd], sel),
                          __builtin_amdgcn_perm(vf[3][wd], vf[2][wd], sel));
    };
    // O^T += V^T P^T for one tile, one MFMA per 16-row head_dim tile c.
    auto pv = [&](const uint32_t (&vf)[4][VWD], const uint2 (&p16)[NT], const float (&p32)[NT][4]) {
#pragma unroll
        for (int c = 0; c < VCH; ++c) {
            if constexpr (DT == MF_F32) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float va = __uint_as_float(vf[r][c]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        acc[nt][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(va, p32[nt][r], acc[nt][c], 0, 0, 0);
                }
            } else {
                const uint2 va = va16(vf, c);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) acc[nt][c] = mfma_pv16<DT>(va, p16[nt], acc[nt][c]);
            }
        }
    };
    auto process = [&](int kt, const uint4 (&kf)[NL], uint32_t (&vf)[4][VWD]) {
        clear_v_tail(kt, vf);
        float sv[NT][4];
        scores(kt, kf, sv);
        float lmax[NT];
        if (needs_rescale(sv, lmax)) rescale(lmax);
        uint2 p16[NT];
        float p32[NT][4];
        exps(sv, p16, p32);
        pv(vf, p16, p32);
    };

    // ---- key loops. Single-column-tile items (decode, verify) stream their
    // own tiles through the NB-buffer register ring below; wide items pooled
    // four to a workgroup with unrelated items stream theirs through two
    // buffers (attn_wide_body runs the ones that share a key range). Every
    // prefetch is unconditional (past the end it is a dummy or a clamped
    // re-read) because a conditional load makes the compiler drain every
    // outstanding load at the join and serialises the pipeline.
    // The first tile past the pipelined range (a verify pass's boundary or
    // candidate tile) is fetched before the loop, so its per-key loads
    // overlap the pool tiles instead of following them.
    uint4 kT[NL];
    uint32_t vT[4][VWD];
    if constexpr (FAST && NT == 1) {
        if (fast_end < kt_end) load_general(fast_end, kT, vT);
    }
    if (kt0 < fast_end) {
        // Ring of NB register buffers: each step issues the tile NB-1 ahead
        // into the slot freed last and processes the oldest. The loop runs
        // whole rounds of NB steps and the last n % NB tiles (already in
        // slots 0..) follow after it: an exit from inside a round would give
        // the loop a latch that some paths reach with a slot's loads still
        // in flight, and the compiler then drains every load at the top of
        // each round. Prefetches past the last tile still issue (a
        // conditional load would drain the pipeline as well), but as a
        // single line: for 256-byte rows these loads bypass L2, so a full
        // re-read would cost HBM.
        const int last = fast_end - 1;
        int kt = kt0;
        if constexpr (NT == 1) {
            if constexpr (!FAST) {
                // (fast items issued these with the setup loads)
#pragma unroll
                for (int i = 0; i < NB - 1; ++i) load_tile(min(kt0 + i, last), kR[i], vR[i]);
            }
            for (int r = (fast_end - kt0) / NB; r > 0; --r) {
#pragma unroll
                for (int u = 0; u < NB; ++u) {
                    const int nx = kt + NB - 1;
                    load_tile(min(nx, last), kR[(u + NB - 1) % NB], vR[(u + NB - 1) % NB], nx > last);
                    process(kt, kR[u], vR[u]);
                    ++kt;
                }
            }
            // The last (n mod NB) tiles, as nested tests: the flat form (one
            // test per slot) keeps every slot live through the tail and
            // spills at 256-byte rows.
            auto tail = [&](auto self, auto U) {
                constexpr int u = decltype(U)::value;
                if constexpr (u < NB - 1) {
                    if (kt + u <= last) {
                        process(kt + u, kR[u], vR[u]);
                        self(self, std::integral_constant<int, u + 1>{});
                    }
                }
            };
            tail(tail, std::integral_constant<int, 0>{});
        } else {
            // wide items without LDS sharing (a few pooled workgroups): two
            // buffers, which keeps the D 64 kernel at four waves per SIMD
            load_tile(kt, kR[0], vR[0]);
            for (;;) {
                load_tile(min(kt + 1, last), kR[1], vR[1]);
                process(kt, kR[0], vR[0]);
                if (++kt > last) break;
                load_tile(min(kt + 1, last), kR[0], vR[0]);
                process(kt, kR[1], vR[1]);
                if (++kt > last) break;
            }
        }
    }

    if constexpr (FAST) {
        int kt = fast_end;
        if constexpr (NT == 1) {
            if (kt < kt_end) process(kt++, kT, vT);
        }
        for (; kt < kt_end; ++kt) {
            load_general(kt, kR[0], vR[0]);
            process(kt, kR[0], vR[0]);
        }
    }

    // ---- cooperative items: the workgroup's four waves took consecutive key
    // ranges of one (sequence, kv head, column tile) and combine their
    // softmax states through LDS. Every lane (g, j) of every wave holds the
    // same column j and head_dim elements (4g + r)*VCH + c; wave w combines
    // the elements with r == w across the four waves and stores them -- the
    // normalised output, or one partial of a longer split.
    if constexpr (NT == 1) {
        if (iv2.w != 0) {  // the planner flags all four items of a cooperative workgroup
            static_assert(coop_lds_bytes<DP>() == (kWaves * 4 * VCH * 64 + 2 * kWaves * 16) * 4, "LDS arena layout");
            auto s_acc = reinterpret_cast<float (*)[4 * VCH][64]>(attn_lds);
            auto s_m = reinterpret_cast<float (*)[16]>(attn_lds + kWaves * 4 * VCH * 64 * 4);
            auto s_l = reinterpret_cast<float (*)[16]>(attn_lds + (kWaves * 4 * VCH * 64 + kWaves * 16) * 4);
            const float lt = group_sum4(l[0]);
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int c = 0; c < VCH; ++c) s_acc[wave][r * VCH + c][lane] = acc[0][c][r];
            if (g == 0) {
                s_m[wave][j] = m[0];
                s_l[wave][j] = lt;
            }
            __syncthreads();
            float mw[kWaves], M = kMinM;
#pragma unroll
            for (int u = 0; u < kWaves; ++u) {
                mw[u] = s_m[u][j];
                M = fmaxf(M, mw[u]);
            }
            float L = 0.f, o[VCH];
#pragma unroll
            for (int c = 0; c < VCH; ++c) o[c] = 0.f;
#pragma unroll
            for (int u = 0; u < kWaves; ++u) {
                const float w = __builtin_amdgcn_exp2f(mw[u] - M);
                L += s_l[u][j] * w;
#pragma unroll
                for (int c = 0; c < VCH; ++c) o[c] += w * s_acc[u][wave * VCH + c][lane];
            }
            const int d0 = (4 * g + wave) * VCH;
            if (nct > 0 && (SC ? qvalid[0] : qpos[0] >= 0)) {
                if (pslot < 0) {
                    if (d0 < D) {
                        const float inv = L > 0.f ? 1.f / L : 0.f;
#pragma unroll
                        for (int c = 0; c < VCH; ++c) o[c] *= inv;
                        store_elems<DT, VCH>(a.out + ((int64_t)prow[0] * a.o_sr + (int64_t)qhead[0] * a.o_sh + d0) * ES, o);
                    }
                } else {
                    const float inv = L > 0.f ? 1.f / L : 0.f;
#pragma unroll
                    for (int c = 0; c < VCH; ++c) o[c] *= inv;
                    bool fp32 = SC;
                    if constexpr (!SC && has_fp32_partials<DT, DP>()) fp32 = (iv1.w & MF_PLAN_FP32_PARTIALS) != 0;
                    if (fp32) store_elems<MF_F32, VCH>(partial_out<MF_F32>(a, pslot, j, d0), o);
                    else store_elems<DT, VCH>(partial_out<DT>(a, pslot, j, d0), o);
                    if (g == 0 && wave == 0) {
                        float* ml = partial_ml(a, pslot);
                        ml[j] = M;
                        ml[16 + j] = L;
                    }
                }
            }
            // fused split-K merge: every wave releases its part of the
            // partial, then wave 0 counts the workgroup's arrival
            if (pslot >= 0 && a.counters != nullptr) {
                __threadfence();
                __syncthreads();
                if (wave == 0) {
                    const int m0 = iv1.w & ~MF_PLAN_FP32_PARTIALS;
                    int prev = 0;
                    if (lane == 0) prev = atomicAdd(a.counters + m0, 1);
                    prev = __shfl(prev, 0, 64);
                    const int32_t* mg0 = a.merges + (int64_t)m0 * MF_PLAN_MERGE_INTS;
                    if (prev == mg0[3] - 1) {
                        __threadfence();
                        if (lane == 0) a.counters[m0] = 0;
                        merge_tile<DT, DP, 2>(a, mg0, g, j);
                    }
                }
            }
            return;
        }
    }

    // ---- finish: the lane holds O^T[d = (4g + r)*VCH + c][column j], i.e. the
    // contiguous head_dim range [4g*VCH, 4g*VCH + 4*VCH) of its column.
    const int dbase = 4 * g * VCH;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const float lt = group_sum4(l[nt]);
        if (nt >= nct || (SC ? !qvalid[nt] : qpos[nt] < 0)) continue;
        if (pslot < 0) {
            if (dbase < D) {
                const float inv = lt > 0.f ? 1.f / lt : 0.f;
                float vals[4 * VCH];
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int c = 0; c < VCH; ++c) vals[r * VCH + c] = acc[nt][c][r] * inv;
                char* op = a.out + ((int64_t)prow[nt] * a.o_sr + (int64_t)qhead[nt] * a.o_sh + dbase) * ES;
                store_out_chunk<DT, VCH>(op, vals);
            }
        } else {
            const float inv = lt > 0.f ? 1.f / lt : 0.f;
            float vals[4 * VCH];
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int c = 0; c < VCH; ++c) vals[r * VCH + c] = acc[nt][c][r] * inv;
            constexpr int PT = SC ? MF_F32 : DT;
            store_out_chunk<PT, VCH>(partial_out<PT>(a, pslot + nt, j, dbase), vals);
            if (g == 0) {
                float* ml = partial_ml(a, pslot + nt);
                ml[j] = m[nt];
                ml[16 + j] = lt;
            }
        }
    }

    if (pslot >= 0) arrive_and_merge<DT, DP>(a, iv1.w, nct, lane);
}

// ------------------------------------------------- workgroup-shared wide items
typedef __attribute__((ext_vector_type(16))) float f32x16;

// S^T / O^T block: 32 rows x 32 columns, contraction over 16 elements (8 per
// lane half).
template <int DT>
__device__ __forceinline__ f32x16 mfma32(uint4 a, uint4 b, f32x16 c) {
    if constexpr (DT == MF_BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c,
                                                      0, 0, 0);
}

// 4 keys x 16 head_dim elements per 16-lane group, transposed on the way out
// of LDS: lane i of the group gets element i of the four rows.
__device__ __forceinline__ uint2 ld_tr16(const char* lds) {
    typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)lds));
}

// ld_lds16 from a wave-uniform base and a 32-bit lane offset: no vector
// address arithmetic per load. The five wait states cover a base that a vector
// instruction (v_readfirstlane) wrote just before, which the compiler cannot
// see to do inside the assembly, and the m0 write's one.
__device__ __forceinline__ void ld_lds16_base(const char* base_, uint32_t lane_off, uint32_t lds_addr) {
    const uint64_t u = (uint64_t)(uintptr_t)base_;
    const uint64_t base = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)u) |
                          ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(u >> 32)) << 32);
    asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" ::"{m0}"(lds_addr), "v"(lane_off), "s"(base) : "memory");
}

// A workgroup whose four wide items are column groups of one (sequence, kv
// head, key range): each wave owns 32 columns, and every K/V row of the range
// is staged in LDS once for the four waves.
//
// Per 32 keys the wave forms S^T = K Q^T and O^T += V^T P^T as 32x32x16 MFMA
// blocks (the full-rate shape: 1.85 PFLOP/s over the chip on this card against
// 1.17 for 16x16x32 and half that for 16x16x16). S^T leaves lane (half hf,
// column c) with keys 8b + 4hf + r of its column; P^T's B operand takes those
// registers as they are, and V^T's A operand is read in the same key order by
// the transposing LDS read, so neither P nor V moves between lanes.
//
// Stages of 64 keys (32 at 256-byte rows) go from global memory straight into
// LDS (two buffers, one barrier per stage). Each wave loads the same few 1 KB pieces of every
// 16-key block, so a piece is one scalar base plus a lane offset that never
// changes: new rows of a written-in-flight step are just another base and
// offset. K rows are xor-swizzled by key in 16-byte chunks (32 keys x one
// chunk read conflict-free), V rows by key mod 4 in pairs of 32-byte granules
// (the transposing read's four rows x 64 bytes hit distinct banks): the
// conflict counter reads zero.
//
// Measured on MI355X against the 16x16 loop this replaces (one layer, KV write
// and merge included): two chunks of 2048 rows after up to 6144 keys, 40/8
// heads x 128, 333 GFLOP: 817 -> 388 us (860 TFLOP/s); 16 prompts of up to 1024
// tokens, 15/5 heads x 64: 32.9 -> 29.1 us. What bounds it: MFMA is busy a third
// of the time and the VALU (exponentials, maxima, packing) as long, in turn
// rather than together -- timing copies without the exponentials, the PV
// products or the LDS reads each gained 10-25%, none more. So waves per SIMD
// count: at 256-byte rows 32-key stages leave room for three (168 registers,
// with spills, and 32 KB of LDS a workgroup), 373 us against 403 with two and
// 64-key stages;
// two score chains at a time took 430 against 436. Scalar registers count too:
// a base computed for every load apart, with a branch each, took 630 us.
//
// Blocks of another size than 16 tokens (BLK16 false) change only where a stage's
// rows are read from: each lane looks up the block of its own key, one stage
// ahead. The planner cuts wide work for workgroups that share their tiles and
// does not see the block size; run wave by wave, its plans took up to 1.7 times
// as long there as the narrower per-wave ranges of the 16x16 loop. Graph
// replays, us, 32-token blocks, that loop, wave by wave, and this: 12 verifies
// of 8 rows at 15/5 heads x 64 33, 50, 20; 6 prompts of up to 900 at 8/2 x 32
// 24, 39, 13; chunks of 512 and 700 after 2000 and 500 at 40/8 x 128 295, 302, 88.
//
// cols holds the first column tile and the tile count of the workgroup's four
// items, in scalar registers: only the block table's round trip stands before
// the first stage. Two to three more did -- the other items' columns by vector
// loads, and a wait for every load in flight behind each test of the row map --
// which beside decode streams cost a mixed step up to 14%. Graph replays, us,
// before and after (and with the 16x16 loop): 2 chunks of 512 rows and 24
// decodes of up to 4700 keys at 15/5 heads x 64 30.6, 26.5 (26.0); 1 chunk of
// 370 and 29 decodes of up to 1150 15.1, 13.6 (13.5); 4 chunks of 512 and 28
// decodes of up to 4096 29.4, 28.7 (31.5); 60 decodes of up to 500 keys and 4
// chunks of about 100 16.0, 15.1 (14.3); 16 prompts of up to 1024 31.5, 30.0
// (35.8). The wave's own item is read again rather than kept: its registers,
// held over the caller's comparison, made the 256-byte kernel spill scalars in
// its loop (two chunks of 2048 rows 409 us against 397).
template <int DT, int DP, bool TAIL, bool BLK16, bool SC>
__device__ __forceinline__ void attn_wide_body(const ArgsOf<SC>& a, const int block,
                                               const int (&cols)[kWaves][2]) {
    constexpr int RB = DP * 2;       // bytes of one key row
    constexpr int NCH = RB / 16;     // 16-byte chunks per row
    constexpr int KEYS = wide_keys(DP, SC), TS = KEYS / 16;  // keys and 16-key blocks per stage
    constexpr int NS = SC ? scored_step(DP) : 1;
    constexpr int RPB = 256 / RB;    // rows per 256 bytes (all LDS banks once)
    constexpr int NQ = DP / 16;      // MFMA steps of S^T
    constexpr int ND = DP / 32;      // 32-row blocks of O^T
    constexpr int PK = RB / 64;      // 1 KB pieces of 16 K rows (V: as many)
    constexpr int NLD = TS * 2 * PK / 4;  // pieces per wave and stage
    constexpr int NOFF = DP == 128 ? 2 : 1;  // a wave's distinct pieces of a block
    constexpr int HALF = KEYS * RB;     // K rows of a stage, then its V rows
    constexpr int STG = 2 * HALF;
    static_assert(DT != MF_F32 && RPB >= 1 && wide_lds_bytes<DT, DP, SC>() == 2 * STG, "stage layout");
    constexpr float kNegInf = -__builtin_huge_valf();

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    const int hf = lane >> 5;
    const char *k_pool = a.k_pool, *v_pool = a.v_pool, *new_k = a.new_k, *new_v = a.new_v;
    const int32_t* it = a.items + ((int64_t)block * kWaves + wave) * MF_PLAN_ITEM_INTS;
    const int s = it[0], h = it[1], c0 = it[2], nct = it[3], kt0 = it[4], kt1 = it[5], pslot = it[6], m0 = it[7];
    const int row0 = it[8], nrows = it[9], kv_len = it[10];
    const bool inflight = TAIL || a.pool_lens != nullptr;
    const int pool_len = TAIL ? kv_len - nrows : (a.pool_lens != nullptr ? a.pool_lens[s] : kv_len);

    // block-table entries of the 64 tiles from tbl_base (one per lane), and of
    // the 64 after them (16-token blocks)
    const int32_t* trow = a.block_tables + (int64_t)s * a.bt_stride;
    const int tbl_end = inflight ? min(kt1, (pool_len + 15) >> 4) : kt1;
    const int tbl_last = max(tbl_end - 1, 0);  // tiles past it are new rows: never read through the table
    int tbl_base = kt0;
    int tbl = 0, tbl_next = 0;
    if constexpr (BLK16) {
        tbl = trow[min(kt0 + lane, tbl_last)];
        tbl_next = trow[min(kt0 + 64 + lane, tbl_last)];
    }
    auto tbl_at = [&](int t) -> int { return __builtin_amdgcn_readlane(tbl, t - tbl_base); };  // wave-uniform t

    // other block sizes: the key this lane fetches with its i-th piece of stage u
    // (clamped to the range and the context, whose last row then stands in: it is
    // masked there), and the entries of the blocks that hold a stage's keys
    const unsigned bsz = (unsigned)a.block_size;
    auto piece_key = [&](int u, int i) -> int {
        const int x = wave + 4 * i;
        const int p = x % (2 * PK);
        const int k16 = (p >= PK ? p - PK : p) * (1024 / RB) + lane * 16 / RB;
        return min(min(kt0 + TS * u + x / (2 * PK), kt1 - 1) * 16 + k16, kv_len - 1);
    };
    auto look = [&](int u, int (&phys)[NLD]) {
        if constexpr (!BLK16) {
#pragma unroll
            for (int i = 0; i < NLD; ++i)
                phys[i] = trow[(unsigned)max(min(piece_key(u, i), pool_len - 1), 0) / bsz];
        }
    };
    int ph0[NLD], ph1[NLD];
    look(0, ph0);
    look(1, ph1);

    // ---- this lane's column: position and query (padding columns read
    // row0's and are never stored)
    const int ct = (lane & 31) >> 4, j = lane & 15;
    const int cidx = c0 * 16 + (lane & 31);
    const bool valid = ct < nct && cidx < nrows * a.G;
    const int col = valid ? cidx : 0;
    const int crow = (int)((unsigned)col / (unsigned)a.G);
    const int qhead = h * a.G + col - crow * a.G;
    // its own row and those of the workgroup's other columns (two per lane),
    // whose positions say how far the stages run, without an exchange between
    // the waves. One test of the row map for all three: each one joins behind a
    // wait for every load in flight.
    int rows[3] = {row0 + crow, row0, row0};
    bool other[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int c = (hf ? cols[2 * k + 1][0] : cols[2 * k][0]) * 16 + (lane & 31);
        other[k] = ct < (hf ? cols[2 * k + 1][1] : cols[2 * k][1]) && c < nrows * a.G;
        rows[1 + k] = row0 + (int)((unsigned)(other[k] ? c : 0) / (unsigned)a.G);
    }
    if (!TAIL && a.row_map) {
#pragma unroll
        for (int k = 0; k < 3; ++k) rows[k] = a.row_map[rows[k]];
    }
    int rpos[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) rpos[k] = reinterpret_cast<const int32_t*>(a.positions)[2 * (int64_t)rows[k]];
    const int prow = rows[0];
    int first_key = 0, prefix = 0;
    float slope = 0.f;
    if constexpr (SC) {
        if (a.first_keys) first_key = a.first_keys[s];
        if (a.prefix_lens) prefix = a.prefix_lens[s];
        if (a.slopes) slope = a.slopes[qhead] * 1.4426950408889634f;
    }
    // the last key of the context a row may see, by position (SC: or prefix)
    auto reach = [&](int pos) { return SC ? max(pos, prefix - 1) : pos; };
    const int qpos = valid ? reach(rpos[0]) : -1;
    const int wpos = max(other[0] ? reach(rpos[1]) : -1, other[1] ? reach(rpos[2]) : -1);
    uint4 qf[NQ];
#pragma unroll
    for (int c = 0; c < NQ; ++c) {
        const uint4 v = *(const uint4*)(a.q + ((int64_t)prow * a.q_sr + (int64_t)qhead * a.q_sh + c * 16 + hf * 8) * 2);
        qf[c] = make_uint4(v.x ^ a.q_sign, v.y ^ a.q_sign, v.z ^ a.q_sign, v.w ^ a.q_sign);
    }

    // ---- stages
    const uint32_t lds_base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)attn_lds;
    uint32_t off[NOFF], ioff[NOFF];  // this lane's 16 bytes inside a 16-key block: pool rows, new rows
#pragma unroll
    for (int n = 0; n < NOFF; ++n) {
        const int p = (wave + 4 * n) % (2 * PK);
        const bool isv = p >= PK;
        const int k16 = (isv ? p - PK : p) * (1024 / RB) + lane * 16 / RB;
        const int swz = isv ? ((k16 & 3) / RPB) << 2 : (k16 / RPB) & (NCH - 1);
        const uint32_t piece = (uint32_t)(((lane & (NCH - 1)) ^ swz) << 4);
        off[n] = (uint32_t)(k16 * a.p_ss * 2) + piece;
        ioff[n] = (uint32_t)(k16 * a.n_sr * 2) + piece;
    }
    const int64_t blk_bytes = a.p_sb * 2;
    const char* kp_h = k_pool + (int64_t)h * a.p_sh * 2;  // this kv head's rows
    const char* nk_h = new_k + ((int64_t)(row0 - pool_len) * a.n_sr + (int64_t)h * a.n_sh) * 2;
    const int64_t v_delta = v_pool - k_pool, nv_delta = new_v - new_k;
    const int64_t tile_bytes = 16 * a.n_sr * 2;
    // Where this kv head's K rows of tile t begin. Scored launches, whose loop has few
    // scalar registers left, keep the 64 tiles' addresses in lanes rather than form each
    // from its entry: a stage's fetch is 60 scalar instructions shorter (the two chunks
    // above 667 -> 659 us).
    uint32_t base_lo = 0, base_hi = 0;
    auto set_bases = [&]() {
        if constexpr (SC && BLK16) {
            const uint64_t b = (uint64_t)kp_h + (uint64_t)((int64_t)tbl * blk_bytes);
            base_lo = (uint32_t)b;
            base_hi = (uint32_t)(b >> 32);
        }
    };
    set_bases();
    auto rows_at = [&](int t) -> const char* {
        if constexpr (SC && BLK16) {
            const uint32_t lo = __builtin_amdgcn_readlane(base_lo, t - tbl_base);
            const uint32_t hi = __builtin_amdgcn_readlane(base_hi, t - tbl_base);
            return (const char*)((uint64_t)hi << 32 | lo);
        } else {
            return kp_h + (int64_t)tbl_at(t) * blk_bytes;
        }
    };
    // tiles the fetches clamp to: the item's range for the first stage, the
    // workgroup's last read tile once the positions are in
    int fetch_end = kt1;
    auto fetch = [&](int u, int buf, const int (&phys)[NLD]) __attribute__((always_inline)) {
        const int t0 = kt0 + TS * u;
        if constexpr (!BLK16) {
#pragma unroll
            for (int i = 0; i < NLD; ++i) {
                const int x = wave + 4 * i;
                const int b = x / (2 * PK), p = x % (2 * PK);
                const bool isv = p >= PK;
                const int k16 = (isv ? p - PK : p) * (1024 / RB) + lane * 16 / RB;
                const int swz = isv ? ((k16 & 3) / RPB) << 2 : (k16 / RPB) & (NCH - 1);
                const int key = piece_key(u, i);
                const char* src;
                if (!inflight || key < pool_len) {
                    src = k_pool + (isv ? v_delta : 0) + ((int64_t)phys[i] * a.p_sb +
                                                          (int64_t)((unsigned)key % bsz) * a.p_ss + (int64_t)h * a.p_sh) * 2;
                } else {
                    int nr = row0 + key - pool_len;
                    if (a.row_map) nr = a.row_map[nr];
                    src = new_k + (isv ? nv_delta : 0) + ((int64_t)nr * a.n_sr + (int64_t)h * a.n_sh) * 2;
                }
                ld_lds16(src + (((lane & (NCH - 1)) ^ swz) << 4),
                         lds_base + (uint32_t)(buf * STG + b * 16 * RB + (isv ? HALF + (p - PK) * 1024 : p * 1024)));
            }
            return;
        }
        if (t0 - tbl_base >= 64) {
            tbl_base += 64;
            tbl = tbl_next;
            tbl_next = trow[min(tbl_base + 64 + lane, tbl_last)];
            set_bases();
        }
        const uint32_t dst0 = lds_base + (uint32_t)(buf * STG);
        const int key1 = (t0 + TS) * 16;
        const bool whole = t0 + TS <= fetch_end;
        // A stage wholly in the pool or wholly of new rows takes a scalar base
        // per block; the boundary stage, the range's last one, and rows behind
        // a row map take the general form below.
        const bool in_pool = whole & (!inflight | (key1 <= pool_len));
        const bool in_new = whole & inflight & (t0 * 16 >= pool_len) & (key1 <= kv_len) & (a.row_map == nullptr);
        auto piece = [&](int i, const char* block_base, int64_t to_v, uint32_t lane_off) {
            const int p = (wave + 4 * i) % (2 * PK), b = (wave + 4 * i) / (2 * PK);
            const bool isv = p >= PK;
            ld_lds16_base(block_base + (isv ? to_v : 0), lane_off,
                          dst0 + (uint32_t)(b * 16 * RB + (isv ? HALF + (p - PK) * 1024 : p * 1024)));
        };
        if (in_pool) {
#pragma unroll
            for (int i = 0; i < NLD; ++i)
                piece(i, rows_at(t0 + (wave + 4 * i) / (2 * PK)), v_delta, off[i % NOFF]);
        } else if (in_new) {
#pragma unroll
            for (int i = 0; i < NLD; ++i)
                piece(i, nk_h + (t0 + (wave + 4 * i) / (2 * PK)) * tile_bytes, nv_delta, ioff[i % NOFF]);
        } else {
#pragma unroll 1
            for (int i = 0; i < NLD; ++i) {
                const int x = wave + 4 * i;
                const int b = x / (2 * PK), p = x % (2 * PK);
                const bool isv = p >= PK;
                const int t = min(t0 + b, fetch_end - 1);
                const uint32_t dst = dst0 + (uint32_t)(b * 16 * RB + (isv ? HALF + (p - PK) * 1024 : p * 1024));
                const int k16 = (isv ? p - PK : p) * (1024 / RB) + lane * 16 / RB;
                const int swz = isv ? ((k16 & 3) / RPB) << 2 : (k16 / RPB) & (NCH - 1);
                const int piece = ((lane & (NCH - 1)) ^ swz) << 4;
                // In a block of the pool every slot exists; a new row past the
                // context reads the last one. Either is masked, and its V row
                // cleared.
                const int key = inflight ? min(t * 16 + k16, kv_len - 1) : t * 16 + k16;
                const char* src;
                if (!inflight || key < pool_len) {
                    if constexpr (SC) {
                        src = rows_at(t) + (isv ? v_delta : 0) + (int64_t)k16 * a.p_ss * 2;
                    } else {
                        const int64_t blk = tbl_at(t);
                        src = k_pool + (isv ? v_delta : 0) + (blk * a.p_sb + (int64_t)k16 * a.p_ss + (int64_t)h * a.p_sh) * 2;
                    }
                } else {
                    int nr = row0 + key - pool_len;
                    if (a.row_map) nr = a.row_map[nr];
                    src = new_k + (isv ? nv_delta : 0) + ((int64_t)nr * a.n_sr + (int64_t)h * a.n_sh) * 2;
                }
                ld_lds16(src + piece, dst);
            }
        }
    };
    if constexpr (MF_WIDE_PRIO > 0) __builtin_amdgcn_s_setprio(MF_WIDE_PRIO);
    if (kt1 > kt0) fetch(0, 0, ph0);

    // ---- the columns' causal limits; tiles past the workgroup's last visible
    // key are not read
    const int end_key = min(kv_len, kt1 * 16);
    const int lim = qpos >= 0 ? min(qpos, end_key - 1) : -1;  // last key the column may see here
    int maxlim = lim, minlim = valid ? lim : INT_MAX, wglim = min(wpos, end_key - 1);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        maxlim = max(maxlim, __shfl_xor(maxlim, o, 64));
        minlim = min(minlim, __shfl_xor(minlim, o, 64));
        wglim = max(wglim, __shfl_xor(wglim, o, 64));
    }
    maxlim = __builtin_amdgcn_readfirstlane(maxlim);
    minlim = __builtin_amdgcn_readfirstlane(minlim);
    wglim = __builtin_amdgcn_readfirstlane(wglim);
    auto sync = [&]() {
        // this wave's LDS reads and writes are done, then all waves'
        __builtin_amdgcn_s_waitcnt((15) | (3 << 14) | (7 << 4) | (0 << 8));  // lgkmcnt(0)
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    const int wg_end = wglim < kt0 * 16 ? kt0 : (wglim >> 4) + 1;
    fetch_end = wg_end;
    const int nst = (wg_end - kt0 + TS - 1) / TS;

    float m = kMinM, l = 0.f;
    float thr = SC ? kMinM + kLazyLog2 : (kMinM + kLazyLog2) * a.inv_scale_log2;
    f32x16 acc[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;

    // lane addresses inside a stage: K rows (key lane & 31), V rows (key 4hf +
    // (lane & 15) / 4 of each group of 8)
    uint32_t kaddr[NQ], vaddr[ND];
#pragma unroll
    for (int c = 0; c < NQ; ++c)
        kaddr[c] = (uint32_t)((lane & 31) * RB + (((2 * c + hf) ^ ((j / RPB) & (NCH - 1))) << 4));
#pragma unroll
    for (int d = 0; d < ND; ++d)
        vaddr[d] = (uint32_t)(HALF + (4 * hf + (j >> 2)) * RB +
                              (((4 * d + 2 * ct + ((j & 3) >> 1)) ^ (((j >> 2) / RPB) << 2)) << 4) + 8 * (j & 1));

    // NS blocks of 32 keys, one softmax step
    auto tile = [&](const char* stg, int key0) __attribute__((always_inline)) {
        f32x16 st[NS];
#pragma unroll
        for (int n = 0; n < NS; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) st[n][i] = 0.f;
#pragma unroll
        for (int c = 0; c < NQ; ++c)
#pragma unroll
            for (int n = 0; n < NS; ++n) st[n] = mfma32<DT>(*(const uint4*)(stg + n * 32 * RB + kaddr[c]), qf[c], st[n]);
        if constexpr (SC) {
            const float dist = (float)(key0 + 4 * hf - rpos[0]);
            float x[16 * NS];
#pragma unroll
            for (int i = 0; i < 16 * NS; ++i) x[i] = st[i >> 4][i & 15];
            score_all<DT>(x, a, slope, [&](int i) { return dist + (32 * (i >> 4) + 8 * ((i & 15) >> 2) + (i & 3)); });
#pragma unroll
            for (int i = 0; i < 16 * NS; ++i) st[i >> 4][i & 15] = x[i];
        }
        if (key0 + 32 * NS - 1 > minlim || (SC && key0 < first_key)) {
#pragma unroll
            for (int n = 0; n < NS; ++n)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int key = key0 + 32 * n + 8 * (i >> 2) + 4 * hf + (i & 3);
                    st[n][i] = key <= lim && (!SC || key >= first_key) ? st[n][i] : kNegInf;
                }
        }
        // lazy rescale, as in attn_body; a column's keys lie in two lanes
        float lmax = st[0][0];
#pragma unroll
        for (int n = 0; n < NS; ++n)
#pragma unroll
            for (int i = n ? 0 : 1; i < 16; ++i) lmax = fmax_prop(lmax, st[n][i]);
        if (__builtin_amdgcn_ballot_w64(lmax > thr) != 0) {
            auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(lmax), __float_as_uint(lmax), false, false);
            const float cm = fmax_prop(__uint_as_float(r[0]), __uint_as_float(r[1]));
            const float mn = fmaxf(m, SC ? cm : cm * a.scale_log2);
            const float alpha = __builtin_amdgcn_exp2f(m - mn);
            l *= alpha;
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[d][i] *= alpha;
            m = mn;
            thr = SC ? mn + kLazyLog2 : (mn + kLazyLog2) * a.inv_scale_log2;
        }
#pragma unroll
        for (int n = 0; n < NS; ++n) {
            uint32_t pw[8];
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float s0 = st[n][2 * i], s1 = st[n][2 * i + 1];
                const float p0 = __builtin_amdgcn_exp2f(SC ? s0 - m : __builtin_fmaf(s0, a.scale_log2, -m));
                const float p1 = __builtin_amdgcn_exp2f(SC ? s1 - m : __builtin_fmaf(s1, a.scale_log2, -m));
                sum += p0 + p1;
                if constexpr (DT == MF_BF16)
                    pw[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){p0, p1}, bf16x2));
                else
                    pw[i] = f32_to_bits<DT>(p0) | (f32_to_bits<DT>(p1) << 16);
            }
            l += sum;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const uint4 pf = make_uint4(pw[4 * k], pw[4 * k + 1], pw[4 * k + 2], pw[4 * k + 3]);
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    const uint2 v0 = ld_tr16(stg + vaddr[d] + (32 * n + 16 * k) * RB);
                    const uint2 v1 = ld_tr16(stg + vaddr[d] + (32 * n + 16 * k + 8) * RB);
                    acc[d] = mfma32<DT>(make_uint4(v0.x, v0.y, v1.x, v1.y), pf, acc[d]);
                }
            }
        }
    };

    if (nst > 0) {
        if (nst > 1) fetch(1, 1, ph1);
        const int live_end = min(kv_len, wg_end * 16);  // rows past it may hold anything, NaN included
        if (nst > 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NLD) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        sync();
        look(2, ph0);
        for (int u = 0; u < nst; ++u) {
            char* stg = attn_lds + (u & 1) * STG;
            const int key0 = (kt0 + TS * u) * 16;
            if (key0 + KEYS > live_end) {
                // the last stage: p is 0 for its rows past the context, and 0 * NaN is NaN
                // (SC: nor may their scores pick how the rest is capped)
                const int first = live_end - key0;
                for (int x = first * NCH + (int)threadIdx.x; x < KEYS * NCH; x += 256) {
                    *(uint4*)(stg + HALF + x * 16) = make_uint4(0, 0, 0, 0);
                    if constexpr (SC) *(uint4*)(stg + x * 16) = make_uint4(0, 0, 0, 0);
                }
                sync();
            }
            if (SC && key0 < first_key) {  // likewise the keys no row of the sequence sees
                for (int x = (int)threadIdx.x; x < min(first_key - key0, KEYS) * NCH; x += 256) {
                    *(uint4*)(stg + HALF + x * 16) = make_uint4(0, 0, 0, 0);
                    *(uint4*)(stg + x * 16) = make_uint4(0, 0, 0, 0);
                }
                sync();
            }
#pragma unroll
            for (int v = 0; v < KEYS / (32 * NS); ++v)
                if (key0 + 32 * NS * v <= maxlim) tile(stg + v * 32 * NS * RB, key0 + 32 * NS * v);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            sync();
            if (u + 2 < nst) {
                fetch(u + 2, u & 1, ph0);
                look(u + 3, ph0);
            }
        }
    } else {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the first stage still lands in this workgroup's LDS
    }

    // ---- finish: lane (hf, column) holds head_dim elements 32d + 8b + 4hf ..
    // + 3; the halves trade blocks so that each lane stores 16 bytes
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
    const float lt = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    const float inv = lt > 0.f ? 1.f / lt : 0.f;
    const bool live = SC ? valid : qpos >= 0;  // scored rows that see no key get zeros
    if (SC && pslot >= 0) {
        if (live) {
            char* part = partial_out<MF_F32>(a, pslot + ct, j, 0);
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    float4 o;
                    o.x = acc[d][4 * b] * inv;
                    o.y = acc[d][4 * b + 1] * inv;
                    o.z = acc[d][4 * b + 2] * inv;
                    o.w = acc[d][4 * b + 3] * inv;
                    *(float4*)(part + (32 * d + 8 * b + 4 * hf) * 4) = o;
                }
            if (hf == 0) {
                float* ml = partial_ml(a, pslot + ct);
                ml[j] = m;
                ml[16 + j] = lt;
            }
        }
        return;
    }
    char* dst = nullptr;
    if (live)
        dst = pslot < 0 ? a.out + ((int64_t)prow * a.o_sr + (int64_t)qhead * a.o_sh) * 2
                        : partial_out<DT>(a, pslot + ct, j, 0);
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
    if (pslot >= 0) {
        if (live && hf == 0) {
            float* ml = partial_ml(a, pslot + ct);
            ml[j] = m;
            ml[16 + j] = lt;
        }
        arrive_and_merge<DT, DP>(a, m0, nct, lane);
    }
}

// One workgroup of a launch's items. 16-bit wide items share their key range
// through LDS: the planner gives every such workgroup one (sequence, kv head,
// key range); one whose items differ runs them wave by wave. The four items'
// fields are loaded together and compared without short-circuit: chained &&
// made the compiler issue one load per comparison, each behind a full wait,
// which beside a decode workgroup's streams took 12.7 us of a prefill
// workgroup's setup (4.0 us alone).
template <int DT, int DP, int NT, bool FAST, bool TAIL = false, bool SC = false>
__device__ __forceinline__ void attn_block(const ArgsOf<SC>& a, const int block) {
    if constexpr (DT != MF_F32 && NT > 1) {
        const int num_items = a.dev_count ? *a.dev_count : a.num_items;
        const int32_t* i0 = a.items + (int64_t)block * kWaves * MF_PLAN_ITEM_INTS;
        int32_t key[kWaves][4];
        int cols[kWaves][2];
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const int32_t* iw = i0 + w * MF_PLAN_ITEM_INTS;
            key[w][0] = iw[0];
            key[w][1] = iw[1];
            key[w][2] = iw[4];
            key[w][3] = iw[5];
            cols[w][0] = iw[2];
            cols[w][1] = iw[3];
        }
        bool same = (FAST || a.head_dim == DP) & ((block + 1) * kWaves <= num_items);
#pragma unroll
        for (int w = 1; w < kWaves; ++w)
            same = same & (key[w][0] == key[0][0]) & (key[w][1] == key[0][1]) & (key[w][2] == key[0][2]) &
                   (key[w][3] == key[0][3]);
        if (same) {
            attn_wide_body<DT, DP, TAIL, FAST, SC>(a, block, cols);
            return;
        }
    }
    attn_body<DT, DP, NT, FAST, TAIL, SC>(a, block);
}

// The item list comes as a separate first argument, which the build has the
// hardware preload into scalar registers: a wave's first item load then
// needs no load of the argument block (see attn_body).
template <int DT, int DP, int NT, bool FAST, bool TAIL = false, bool SC = false>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(attn_waves_per_eu<DT, DP, NT, SC>())))
void attn_kernel(const int32_t* items, ArgsOf<SC> a) {
    a.items = items;
    if constexpr (TAIL) {
        // the copy workgroups first (measured on the C2 step: 53.7 us per
        // layer against 55.7 with them last)
        const int b = blockIdx.x;
        if (b < a.w_blocks) write_new_rows<DT>(a, b);
        else attn_block<DT, DP, NT, FAST, true, SC>(a, b - a.w_blocks);
    } else {
        attn_block<DT, DP, NT, FAST, false, SC>(a, blockIdx.x);
    }
}

// In a mixed launch the single-tile (decode) waves start their loads after a
// short sleep, about the time the dispatcher takes to hand out the launch's
// workgroups. Per-workgroup timestamps of the C2 launch showed a prefill
// workgroup beside a decode workgroup spend 14.6 us (median) from its start
// to its first staged tile, against 6.1 us on a CU without one: its setup
// loads (block table, Q, the first K/V stages) queued behind the decode
// waves' streams, while the decode workgroups themselves finished at 14 us
// and the prefill ones at 34-41 us. With the decode waves held back by one
// s_sleep(32) (2,048 cycles) the prefill setup loads go out first: C2 engine
// layer 43.0-43.6 us against 44.6-45.1 (graph replays, alternating builds);
// two to four sleeps gave 43.3-44.1, six 44.9-45.1, nine 46.0-46.4.
#ifndef MF_MIXED_NARROW_SLEEPS
#define MF_MIXED_NARROW_SLEEPS 1
#endif
__device__ __forceinline__ void narrow_start_delay() {
#pragma unroll
    for (int i = 0; i < MF_MIXED_NARROW_SLEEPS; ++i) __builtin_amdgcn_s_sleep(32);
}

// Single-tile and wide items of one plan in one launch: the first
// workgroups run the single-tile items (decode rows: chains of dependent
// loads, latency-bound), the last `wide_blocks` the wide ones (prefill rows:
// MFMA and softmax work), which fill the slots the single-tile workgroups
// leave and overlap their load latency. Two back-to-back launches would leave
// the chip half idle for the length of the shorter one. Measured on the C2
// step (bf16, D 64, 382 single-tile and 900 wide workgroups): 67.9 us per
// layer as two launches, 62.7 us with the wide workgroups first, 58.6 us with
// the single-tile ones first. Each workgroup is entirely one kind, so the
// barriers of either body stay workgroup-uniform.
//
// Occupancy: with 16-bit rows of 128 bytes (D 64) the launch asks
// for four waves per SIMD. Its LDS is one arena sized for the larger of the
// two bodies (32.8 KB at D 64, so four workgroups fit a CU), and the compiler
// then keeps it to 128 registers with a few spills; three waves per SIMD, the
// single-tile body's own need (140 registers), left the C2 step's 1,104
// workgroups in more than one round of three per CU. Measured on the C2
// engine layer as graph replays: 55.1-56.3 us at four, 56.0-57.3 at three.
template <int DT, int DP, int NTW, bool SC = false>
constexpr int mixed_waves_per_eu() {
    if constexpr (SC && DT != MF_F32) return scored_waves(DP);
    else if constexpr (DT != MF_F32 && DP == 64) return 4;
    else return attn_waves_per_eu<DT, DP, NTW>() < attn_waves_per_eu<DT, DP, 1>() ? attn_waves_per_eu<DT, DP, NTW>()
                                                                                 : attn_waves_per_eu<DT, DP, 1>();
}
template <int DT, int DP, int NTW, bool SC = false>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(mixed_waves_per_eu<DT, DP, NTW, SC>())))
void attn_mixed_kernel(ArgsOf<SC> narrow, ArgsOf<SC> wide, int wide_blocks) {
    const int b = blockIdx.x;
    const int narrow_blocks = (int)gridDim.x - wide_blocks;
    if (b < narrow_blocks) {
        narrow_start_delay();
        attn_body<DT, DP, 1, true, false, SC>(narrow, b);
    } else {
        attn_block<DT, DP, NTW, true, false, SC>(wide, b - narrow_blocks);
    }
}

// The written-in-flight form: the copy workgroups first, then the narrow and
// wide ones. One argument block (the wide items differ only in their list):
// the larger body needs the scalar registers a second block would take.
template <int DT, int DP, int NTW, bool SC = false>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(mixed_waves_per_eu<DT, DP, NTW, SC>())))
void attn_mixed_tail_kernel(ArgsOf<SC> a, const int32_t* wide_items, int wide_num_items,
                            const int32_t* wide_dev_count, int wide_blocks) {
    const int b = blockIdx.x - a.w_blocks;
    const int narrow_blocks = (int)gridDim.x - a.w_blocks - wide_blocks;
    if (b < 0) {
        write_new_rows<DT>(a, blockIdx.x);
    } else if (b < narrow_blocks) {
        narrow_start_delay();
        attn_body<DT, DP, 1, true, true, SC>(a, b);
    } else {
        ArgsOf<SC> w = a;
        w.items = wide_items;
        w.num_items = wide_num_items;
        w.dev_count = wide_dev_count;
        attn_block<DT, DP, NTW, true, true, SC>(w, b - narrow_blocks);
    }
}

// ------------------------------------------------------------ decode slices
// A large decode launch as one resident round of waves (mf_attention_plan_slices).
// The plan cuts the concatenated (sequence, 16-key tile) order into equal
// slices; one wave per (slice, kv head) streams the slice's tiles for its head
// and the waves of a slice sit next to each other in the grid (four to a
// workgroup), so every block's rows are read for all kv heads at about the
// same time and no workgroup waits for another to leave. Measured on MI355X
// with a load-only kernel over the C5 block tables: the per-range plan
// (cooperative units: one CU reading one head's quarters, several rounds of
// workgroups) streams at 5.9 TB/s, the same tiles in one round with a
// workgroup per four heads of a range at 6.5-6.8 TB/s. The plan counts one
// workgroup per CU (one wave per SIMD, MF_SLICE_WAVES_PER_CU): with two per
// CU the C5 layer took 521 us against 505, fewer streams keeping the HBM
// busier (three per CU at head_dim 64: 303 against 287 us).
//
// A slice is a list of segments, each one sequence's tiles [kt0, kt1) (a
// whole range or a piece of one; pieces leave split-K partials for the merge
// kernel). Each lane holds eight of the slice's block-table entries (tile
// lane + 64k), so the register ring below runs across segment boundaries
// without a drain: every segment is padded to a multiple of the ring depth
// with dummy tiles (entry stored as ~block: a one-line load, every key
// masked), which keeps the ring's slot of a tile fixed at tile % depth. Lane
// i holds segment i's record and query position, and each segment start
// loads the next segment's query.
constexpr int kSliceRecordInts = MF_SLICE_INTS;
constexpr int kSliceMaxTiles = MF_SLICE_MAX_TILES;        // table entries per lane: tiles / 64
constexpr int kSliceTableRegs = kSliceMaxTiles / 64;
constexpr int kSliceMaxSegments = MF_SLICE_MAX_SEGMENTS;  // one record per lane at set-up
static_assert(kSliceMaxTiles % 64 == 0 && kSliceMaxSegments <= 64, "slice limits");

template <int DT, int DP>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(attn_waves_per_eu<DT, DP, 1>())))
void attn_slice_kernel(AttnArgs a, int num_slices, int hkv) {
    constexpr int ES = DT == MF_F32 ? 4 : 2;
    constexpr int EPL = 16 / ES;
    constexpr int NL = DP * ES / 64;
    constexpr int VCH = DP / 16;
    constexpr int VB = VCH * ES;
    constexpr int VWD = VB / 4;
    constexpr int NB = MF_NARROW_DEPTH;
    constexpr float kNegInf = -__builtin_huge_valf();

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int w = blockIdx.x * kWaves + wave;
    if (w >= num_slices * hkv) return;
    const int sl = w / hkv;
    const int h = w - sl * hkv;
    const int lane = threadIdx.x & 63;
    const int g = lane >> 4;
    const int j = lane & 15;

    // ---- set-up: the slice's segment records, one per lane, then its
    // block-table entries (4 per lane) and the first ring tiles
    const int32_t* hdr = a.items + (int64_t)sl * kSliceRecordInts;
    const int seg0 = hdr[0], nseg = hdr[1], ntiles = hdr[2];
    if (nseg <= 0 || ntiles <= 0) return;  // (the planner makes no empty slice)
    const int32_t* segs = a.items + ((int64_t)num_slices + seg0) * kSliceRecordInts;
    // Lane i keeps segment i's record (and its query position) for the whole
    // slice: a segment start reads it with readlane, no memory wait.
    const int32_t* rec = segs + (int64_t)min(lane, nseg - 1) * kSliceRecordInts;
    const int4 r0 = *(const int4*)rec;        // s, kt0, kt1, row
    const int4 r1 = *(const int4*)(rec + 4);  // kv_len, slot0, pieces, piece
    int tbl[kSliceTableRegs];
    {
        const int len = lane < nseg ? r0.z - r0.y : 0;
        const int plen = (len + NB - 1) / NB * NB;
        int pend = plen;  // inclusive scan of the padded lengths
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int v = __shfl_up(pend, off, 64);
            if (lane >= off) pend += v;
        }
        const int pstart = pend - plen;
#pragma unroll
        for (int k = 0; k < kSliceTableRegs; ++k) {
            const int t = min(lane + 64 * k, ntiles - 1);
            int idx = 0;  // last segment starting at or before t
#pragma unroll
            for (int step = 32; step >= 1; step >>= 1) {
                const int c = idx + step;
                const int ps = __shfl(pstart, min(c, 63), 64);
                if (c < nseg && ps <= t) idx = c;
            }
            const int ts = __shfl(r0.x, idx, 64);
            const int tk0 = __shfl(r0.y, idx, 64);
            const int tlen = __shfl(len, idx, 64);
            const int o = t - __shfl(pstart, idx, 64);
            const bool real = o < tlen;
            const int e = a.block_tables[(int64_t)ts * a.bt_stride + tk0 + (real ? o : tlen - 1)];
            tbl[k] = real ? e : ~e;
        }
    }
    auto tbl_at = [&](int i) -> int {  // wave-uniform i
        const int k = i >> 6;
        const int l = i & 63;
        int e = __builtin_amdgcn_readlane(tbl[0], l);
#pragma unroll
        for (int q = 1; q < kSliceTableRegs; ++q) e = k == q ? __builtin_amdgcn_readlane(tbl[q], l) : e;
        return e;
    };

    const uint32_t k_lane_off = (uint32_t)(((int64_t)j * a.p_ss + g * EPL) * ES);
    const uint32_t v_row_bytes = (uint32_t)(a.p_ss * ES);
    const uint32_t v_lane_off = (uint32_t)(((int64_t)(4 * g) * a.p_ss + j * VCH) * ES);
    uint32_t v_off[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) v_off[r] = v_lane_off + (uint32_t)r * v_row_bytes;
    // Tile i of the slice; `past` (wave-uniform): a prefetch slot beyond the
    // slice's last tile. Dummy and past tiles load one line per chunk.
    auto load_tile = [&](int i, uint4 (&kf)[NL], uint32_t (&vf)[4][VWD], bool past) {
        const int e = tbl_at(i);
        const int phys = e < 0 ? ~e : e;
        const int64_t boff = ((int64_t)phys * a.p_sb + (int64_t)h * a.p_sh) * ES;
        const char* kb = a.k_pool + boff;
        const char* vb = a.v_pool + boff;
        const uint32_t sel = (past || e < 0) ? 0u : 0xffffffffu;
        const uint32_t ko = k_lane_off & sel;
        if constexpr (DP * ES >= 256) {
#pragma unroll
            for (int c = 0; c < NL; ++c) kf[c] = ld_nt16(kb + ko + c * 4 * 16);
#pragma unroll
            for (int r = 0; r < 4; ++r) ld_words_nt<VB>(vb + (v_off[r] & sel), vf[r]);
        } else {
#pragma unroll
            for (int c = 0; c < NL; ++c) kf[c] = *(const uint4*)(kb + ko + c * 4 * 16);
#pragma unroll
            for (int r = 0; r < 4; ++r) ld_words<VB>(vb + (v_off[r] & sel), vf[r]);
        }
    };

    // Query position of lane i's segment; then the first segment's query
    // (MFMA B operand: lane (g, j) holds column j's head_dim chunks c*4 + g;
    // padding columns j >= G read column 0's, whose scores are never stored)
    // and the first ring tiles. A segment loads the next one's query when it
    // starts, so no segment start waits on memory.
    const int lpos = reinterpret_cast<const int32_t*>(a.positions)[2 * (int64_t)r0.w];
    const bool colv = j < a.G;  // decode: one row, columns 0..G-1 are its heads
    const int qhead = h * a.G + (colv ? j : 0);
    uint4 qn[NL];
    auto load_q = [&](int row) {
#pragma unroll
        for (int c = 0; c < NL; ++c)
            qn[c] = *(const uint4*)(a.q + ((int64_t)row * a.q_sr + (int64_t)qhead * a.q_sh + (c * 4 + g) * EPL) * ES);
    };
    load_q(__builtin_amdgcn_readlane(r0.w, 0));
    uint4 kR[NB][NL];
    uint32_t vR[NB][4][VWD];
#pragma unroll
    for (int i = 0; i < NB - 1; ++i) load_tile(min(i, ntiles - 1), kR[i], vR[i], i > ntiles - 1);

    // ---- per-segment state (the lambdas below read it by reference)
    uint4 qf[NL];
    float m, l, thr;
    f32x4 acc[VCH];
    int lim = -1, minpos = -1, key_end = 0;

    auto process = [&](int kt, const uint4 (&kf)[NL], uint32_t (&vf)[4][VWD]) {
        if ((kt + 1) * 16 > key_end) {
            // keys past the segment (padding, or slots past the context,
            // which may hold anything): p = 0 there, and 0 * NaN is NaN
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const bool live = kt * 16 + 4 * g + r < key_end;
#pragma unroll
                for (int x = 0; x < VWD; ++x) vf[r][x] = live ? vf[r][x] : 0u;
            }
        }
        f32x4 st = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < NL; ++c) st = mfma_qk<DT>(kf[c], qf[c], st);
        float sv[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) sv[r] = st[r];
        if (!(kt * 16 + 15 <= minpos && (kt + 1) * 16 <= key_end)) {
#pragma unroll
            for (int r = 0; r < 4; ++r) sv[r] = kt * 16 + 4 * g + r <= lim ? sv[r] : kNegInf;
        }
        // lazy rescale, exactly as the per-range kernel does it
        const float lmax = fmax_prop(fmax_prop(sv[0], sv[1]), fmax_prop(sv[2], sv[3]));
        if (__builtin_amdgcn_ballot_w64(lmax > thr) != 0) {
            const float mn = fmaxf(m, group_max4(lmax) * a.scale_log2);
            const float alpha = __builtin_amdgcn_exp2f(m - mn);
            l *= alpha;
#pragma unroll
            for (int c = 0; c < VCH; ++c) acc[c] *= alpha;
            m = mn;
            thr = (mn + kLazyLog2) * a.inv_scale_log2;
        }
        float p[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) p[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[r], a.scale_log2, -m));
        l += (p[0] + p[1]) + (p[2] + p[3]);
        if constexpr (DT == MF_F32) {
#pragma unroll
            for (int c = 0; c < VCH; ++c)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    acc[c] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vf[r][c]), p[r], acc[c], 0, 0, 0);
        } else {
            uint2 p16;
            if constexpr (DT == MF_BF16) {
                p16 = make_uint2(__builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){p[0], p[1]}, bf16x2)),
                                 __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){p[2], p[3]}, bf16x2)));
            } else {
                p16 = make_uint2(f32_to_bits<DT>(p[0]) | (f32_to_bits<DT>(p[1]) << 16),
                                 f32_to_bits<DT>(p[2]) | (f32_to_bits<DT>(p[3]) << 16));
            }
#pragma unroll
            for (int c = 0; c < VCH; ++c) {
                const int wd = c >> 1;
                const uint32_t sel = (c & 1) ? 0x07060302u : 0x05040100u;
                const uint2 va = make_uint2(__builtin_amdgcn_perm(vf[1][wd], vf[0][wd], sel),
                                            __builtin_amdgcn_perm(vf[3][wd], vf[2][wd], sel));
                acc[c] = mfma_pv16<DT>(va, p16, acc[c]);
            }
        }
    };

    const int dbase = 4 * g * VCH;
    int t = 0;  // slice index of the next tile to process
    for (int si = 0; si < nseg; ++si) {
        const int kt0 = __builtin_amdgcn_readlane(r0.y, si);
        const int kt1 = __builtin_amdgcn_readlane(r0.z, si);
        const int row = __builtin_amdgcn_readlane(r0.w, si);
        const int kv_len = __builtin_amdgcn_readlane(r1.x, si);
        const int pos = __builtin_amdgcn_readlane(lpos, si);
#pragma unroll
        for (int c = 0; c < NL; ++c)
            qf[c] = make_uint4(qn[c].x ^ a.q_sign, qn[c].y ^ a.q_sign, qn[c].z ^ a.q_sign, qn[c].w ^ a.q_sign);
        // the next segment's query (the last segment re-reads its own, so
        // every segment issues the same loads)
        load_q(__builtin_amdgcn_readlane(r0.w, min(si + 1, nseg - 1)));
        key_end = min(kv_len, kt1 * 16);
        lim = colv && pos >= 0 ? min(pos, key_end - 1) : -1;
        minpos = pos;
        m = kMinM;
        thr = (kMinM + kLazyLog2) * a.inv_scale_log2;
        l = 0.f;
#pragma unroll
        for (int c = 0; c < VCH; ++c) acc[c] = f32x4{0.f, 0.f, 0.f, 0.f};

        const int seg_start = t;
        const int rounds = (kt1 - kt0 + NB - 1) / NB;
        for (int r = rounds; r > 0; --r) {
#pragma unroll
            for (int u = 0; u < NB; ++u) {
                const int nx = t + NB - 1;
                load_tile(min(nx, ntiles - 1), kR[(u + NB - 1) % NB], vR[(u + NB - 1) % NB], nx > ntiles - 1);
                process(kt0 + (t - seg_start), kR[u], vR[u]);
                ++t;
            }
        }

        // ---- finish the segment: the normalised output, or its partial
        const float lt = group_sum4(l);
        if (colv && pos >= 0) {
            const int slot0 = __builtin_amdgcn_readlane(r1.y, si);
            if (slot0 < 0) {
                const float inv = lt > 0.f ? 1.f / lt : 0.f;
                float vals[4 * VCH];
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int c = 0; c < VCH; ++c) vals[r * VCH + c] = acc[c][r] * inv;
                store_out_chunk<DT, VCH>(a.out + ((int64_t)row * a.o_sr + (int64_t)qhead * a.o_sh + dbase) * ES, vals);
            } else {
                const int pslot = slot0 + h * __builtin_amdgcn_readlane(r1.z, si) + __builtin_amdgcn_readlane(r1.w, si);
                const float inv = lt > 0.f ? 1.f / lt : 0.f;
                float vals[4 * VCH];
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int c = 0; c < VCH; ++c) vals[r * VCH + c] = acc[c][r] * inv;
                store_out_chunk<DT, VCH>(partial_out<DT>(a, pslot, j, dbase), vals);
                if (g == 0) {
                    float* ml = partial_ml(a, pslot);
                    ml[j] = m;
                    ml[16 + j] = lt;
                }
            }
        }
    }
}

// --------------------------------------------------------------- merge kernel
// A merge launch's record mi, loaded before its count check (record
// min(mi, num_merges - 1): in bounds for every workgroup of the grid), so the
// load goes out with the argument block's instead of one round trip after it;
// the record list's address and num_merges are the preloaded first arguments.
// The argument fields the merge addresses its partials, row map and output
// from are loaded in the same batch. The empty asm keeps the loads ahead of
// the check.
__device__ __forceinline__ void load_merge_record(const AttnArgs& a, const int32_t* merges, int mi, int num_merges,
                                                  int32_t (&mg)[MF_PLAN_MERGE_INTS]) {
    const int32_t* rec = merges + (int64_t)min(mi, num_merges - 1) * MF_PLAN_MERGE_INTS;
    const int4 r0 = *(const int4*)rec, r1 = *(const int4*)(rec + 4);
    asm volatile("" ::"s"(r0.x), "s"(r0.y), "s"(r0.z), "s"(r0.w), "s"(r1.x), "s"(r1.y), "s"(r1.z), "s"(r1.w));
    asm volatile("" ::"s"(a.G), "s"(a.out), "s"(a.o_sr), "s"(a.o_sh), "s"(a.row_map), "s"(a.partials),
                 "s"(a.part_dstride), "s"(a.head_dim));
    mg[0] = r0.x; mg[1] = r0.y; mg[2] = r0.z; mg[3] = r0.w;
    mg[4] = r1.x; mg[5] = r1.y; mg[6] = r1.z; mg[7] = r1.w;
}

// One wave per merge record, each record a workgroup of its own: the wave
// loads its record's partitions four at a time (merge_range) and writes the
// output directly, with no LDS combine or barrier. Measured on MI355X against
// the two earlier forms (four waves per record splitting its partitions and
// combining them in LDS below 128 records, four records per workgroup above):
// C3's verify layer (75 records) 11.36-11.38 us against 12.29-12.40, the C2
// layer (1,955 records) 37.9-38.1 against 38.2-38.3, C5 (824) the same.
template <int DT, int DP, bool ALL32 = false>
__global__ __launch_bounds__(64) void merge_kernel(const int32_t* merges, int num_merges, AttnArgs a) {
    const int mi = blockIdx.x;
    int32_t mg[MF_PLAN_MERGE_INTS];
    load_merge_record(a, merges, mi, num_merges, mg);
    if (mi >= (a.dev_count ? *a.dev_count : num_merges)) return;
    const int lane = threadIdx.x & 63;
    merge_tile<DT, DP, (DP > 128 ? 2 : 4), ALL32>(a, mg, lane >> 4, lane & 15);
}

// Fp32 partials of decode ranges: one workgroup per record, its partitions dealt to the
// four waves, whose results are combined through LDS as the cooperative units' states
// are. A long range is cut into some thirty, which one wave reads four at a time: 32
// records of up to 36 partitions, 19 us that way, 8 this way.
constexpr int merge_quad_lds(int dp) { return (kWaves * (dp / 4) * 64 + 2 * kWaves * 64) * 4; }
template <int DT, int DP>
__global__ __launch_bounds__(256) void merge_quad_kernel(const int32_t* merges, int num_merges, AttnArgs a) {
    constexpr int VCH = DP / 16;
    const int mi = blockIdx.x;
    int32_t mg[MF_PLAN_MERGE_INTS];
    load_merge_record(a, merges, mi, num_merges, mg);
    if (mi >= (a.dev_count ? *a.dev_count : num_merges)) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63, g = lane >> 4, j = lane & 15;
    int prow = 0, qhead = 0;
    const bool valid = merge_column(a, mg, j, prow, qhead) && 4 * g * VCH < a.head_dim;
    float mx = kMinM, L = 0.f, o[4 * VCH];
#pragma unroll
    for (int e = 0; e < 4 * VCH; ++e) o[e] = 0.f;
    if (valid && wave < mg[3])
        merge_range<DT, DP, MF_F32, (DP > 128 ? 2 : 4)>(a, mg, wave, kWaves, j, 4 * g * VCH, mx, L, o);
    auto s_o = reinterpret_cast<float (*)[4 * VCH][64]>(attn_lds);
    auto s_m = reinterpret_cast<float (*)[64]>(attn_lds + kWaves * 4 * VCH * 64 * 4);
    auto s_l = s_m + kWaves;
#pragma unroll
    for (int e = 0; e < 4 * VCH; ++e) s_o[wave][e][lane] = o[e];
    s_m[wave][lane] = mx;
    s_l[wave][lane] = L;
    __syncthreads();
    const int d0 = (4 * g + wave) * VCH;
    if (!valid || d0 >= a.head_dim) return;
    float M = kMinM;
#pragma unroll
    for (int u = 0; u < kWaves; ++u) M = fmaxf(M, s_m[u][lane]);
    L = 0.f;
    float r[VCH];
#pragma unroll
    for (int c = 0; c < VCH; ++c) r[c] = 0.f;
#pragma unroll
    for (int u = 0; u < kWaves; ++u) {
        const float w = __builtin_amdgcn_exp2f(s_m[u][lane] - M);
        L += s_l[u][lane] * w;
#pragma unroll
        for (int c = 0; c < VCH; ++c) r[c] += w * s_o[u][wave * VCH + c][lane];
    }
    const float inv = L > 0.f ? 1.f / L : 0.f;
#pragma unroll
    for (int c = 0; c < VCH; ++c) r[c] *= inv;
    constexpr int ES = DT == MF_F32 ? 4 : 2;
    store_elems<DT, VCH>(a.out + ((int64_t)prow * a.o_sr + (int64_t)qhead * a.o_sh + d0) * ES, r);
}

// The split-K merge launch: one single-wave workgroup per record.
template <int DT, int DP>
int launch_merge(const AttnArgs& a, const int32_t* merges, int64_t n_merges, hipStream_t stream) {
    hipLaunchKernelGGL((merge_kernel<DT, DP>), dim3((unsigned)n_merges), dim3(64), 0, stream, merges, (int)n_merges,
                       a);
    return check_launch();
}

// The merge of a launch whose partials are all fp32: four waves a record where all its
// items are decode ranges, one where prefill items leave many records of two or three
// partitions.
template <int DT, int DP>
int launch_merge32(const AttnArgs& a, const int32_t* merges, int64_t n_merges, bool decode, hipStream_t stream) {
    if (decode)
        hipLaunchKernelGGL((merge_quad_kernel<DT, DP>), dim3((unsigned)n_merges), dim3(256), merge_quad_lds(DP), stream,
                           merges, (int)n_merges, a);
    else
        hipLaunchKernelGGL((merge_kernel<DT, DP, true>), dim3((unsigned)n_merges), dim3(64), 0, stream, merges,
                           (int)n_merges, a);
    return check_launch();
}

// TAIL: a written-in-flight launch (16-token blocks and unpadded head_dim
// only: `fast`); its copy workgroups ride in the first launch, or in a
// copy-only launch when there are no items.
template <int DT, int DP, bool TAIL = false, bool SC = false>
int launch_attention(ArgsOf<SC> a, const int32_t* items, int64_t n_narrow, int64_t n_wide,
                     const int32_t* merges, int64_t n_merges, bool fast, const int32_t* dev_counts,
                     hipStream_t stream) {
    // With arrival counters the attention kernel merges its own partitions;
    // a merges-only call (no items) still runs the separate merge kernel.
    const bool fused = a.counters != nullptr && (n_narrow + n_wide) > 0;
    const bool decode = n_wide == 0;
    constexpr int NTW = wide_tiles(DT, DP);
    if constexpr (TAIL) {
        if (!fast) return MF_ERR_UNSUPPORTED;
        if (a.w_blocks > 0 && n_narrow + n_wide == 0) {
            ArgsOf<SC> aw = a;
            aw.items = items;
            aw.num_items = 0;
            aw.dev_count = nullptr;
            hipLaunchKernelGGL((attn_kernel<DT, DP, 1, true, true, SC>), dim3((unsigned)a.w_blocks), dim3(256),
                               (attn_lds_bytes<DT, DP, 1, true>()), stream, aw.items, aw);
            if (int st = check_launch()) return st;
        }
    } else {
        a.w_blocks = 0;
    }
#if MF_MIXED_LAUNCH
    if constexpr (NTW > 1 && DT != MF_F32) {
        if (fast && n_narrow > 0 && n_wide > 0) {
            ArgsOf<SC> an = a, aw = a;
            an.items = items;
            an.num_items = (int)n_narrow;
            an.dev_count = dev_counts ? dev_counts + 0 : nullptr;
            aw.items = items + n_narrow * MF_PLAN_ITEM_INTS;
            aw.num_items = (int)n_wide;
            aw.dev_count = dev_counts ? dev_counts + 1 : nullptr;
            const int64_t wide_blocks = (n_wide + kWaves - 1) / kWaves;
            const dim3 grid((unsigned)(a.w_blocks + wide_blocks + (n_narrow + kWaves - 1) / kWaves));
            constexpr int lds = attn_lds_bytes<DT, DP, 1, true>() > attn_lds_bytes<DT, DP, NTW, true, SC>()
                                    ? attn_lds_bytes<DT, DP, 1, true>() : attn_lds_bytes<DT, DP, NTW, true, SC>();
            if constexpr (TAIL)
                hipLaunchKernelGGL((attn_mixed_tail_kernel<DT, DP, NTW, SC>), grid, dim3(256), lds, stream, an,
                                   aw.items, aw.num_items, aw.dev_count, (int)wide_blocks);
            else
                hipLaunchKernelGGL((attn_mixed_kernel<DT, DP, NTW, SC>), grid, dim3(256), lds, stream, an, aw,
                                   (int)wide_blocks);
            if (int st = check_launch()) return st;
            n_narrow = n_wide = 0;
            a.w_blocks = 0;
        }
    }
#endif
    if (n_narrow > 0) {
        a.items = items;
        a.num_items = (int)n_narrow;
        a.dev_count = dev_counts ? dev_counts + 0 : nullptr;
        const dim3 grid((unsigned)(a.w_blocks + (n_narrow + kWaves - 1) / kWaves));
        if (fast)
            hipLaunchKernelGGL((attn_kernel<DT, DP, 1, true, TAIL, SC>), grid, dim3(256),
                               (attn_lds_bytes<DT, DP, 1, true>()), stream, a.items, a);
        else if constexpr (!TAIL)
            hipLaunchKernelGGL((attn_kernel<DT, DP, 1, false, false, SC>), grid, dim3(256), (attn_lds_bytes<DT, DP, 1, false>()),
                               stream, a.items, a);
        if (int st = check_launch()) return st;
        a.w_blocks = 0;
    }
    if constexpr (NTW > 1) {
        if (n_wide > 0) {
            a.items = items + n_narrow * MF_PLAN_ITEM_INTS;
            a.num_items = (int)n_wide;
            a.dev_count = dev_counts ? dev_counts + 1 : nullptr;
            const dim3 grid((unsigned)(a.w_blocks + (n_wide + kWaves - 1) / kWaves));
            if (fast)
                hipLaunchKernelGGL((attn_kernel<DT, DP, NTW, true, TAIL, SC>), grid, dim3(256),
                                   (attn_lds_bytes<DT, DP, NTW, true, SC>()), stream, a.items, a);
            else if constexpr (!TAIL)
                hipLaunchKernelGGL((attn_kernel<DT, DP, NTW, false, false, SC>), grid, dim3(256),
                                   (attn_lds_bytes<DT, DP, NTW, false, SC>()), stream, a.items, a);
            if (int st = check_launch()) return st;
        }
    } else {
        if (n_wide > 0) return MF_ERR_ARG;  // the plan was made for another dtype
    }
    if (n_merges > 0 && !fused) {
        a.dev_count = dev_counts ? dev_counts + 2 : nullptr;
        if constexpr (SC) return launch_merge32<DT, DP>(a, merges, n_merges, decode, stream);
        else if (int st = launch_merge<DT, DP>(a, merges, n_merges, stream)) return st;
    }
    return MF_OK;
}

// A slice plan (mf_attention_plan_slices): one wave per (slice, kv head),
// then the merge of the sequences split across slices.
template <int DT, int DP>
int launch_slices(AttnArgs a, const int32_t* slices, int64_t n_slices, int hkv, const int32_t* merges,
                  int64_t n_merges, hipStream_t stream) {
    if (n_slices > 0) {
        a.items = slices;
        const int64_t waves = n_slices * hkv;
        const dim3 grid((unsigned)((waves + kWaves - 1) / kWaves));
        hipLaunchKernelGGL((attn_slice_kernel<DT, DP>), grid, dim3(256), 0, stream, a, (int)n_slices, hkv);
        if (int st = check_launch()) return st;
    }
    if (n_merges > 0) {
        if (int st = launch_merge<DT, DP>(a, merges, n_merges, stream)) return st;
    }
    return MF_OK;
}

// A scored launch's fields; a.scale_log2 is set. A cap so small or so large against
// the scale that their quotient leaves fp32's normal numbers is refused.
inline int set_scoring(ScoredArgs& a, const mf_scoring& s) {
    if (!(s.softcap >= 0.f) || !(s.softcap < INFINITY)) return MF_ERR_ARG;
    a.slopes = s.slopes;
    a.first_keys = s.first_keys;
    a.prefix_lens = s.prefix_lens;
    a.cap_in = s.softcap > 0.f ? 2.f * a.scale_log2 / s.softcap : 0.f;
    a.cap_log2 = s.softcap * 1.4426950408889634f;
    a.cap_x = s.softcap > 0.f ? a.scale_log2 / a.cap_log2 : 0.f;
    // The polynomials' coefficients by powers of cap_x, so that they take raw scores. Where
    // one leaves fp32's normal numbers: four terms are not used; three lose the last (2e-8 of
    // the score at a fiftieth of the cap) or the last two (1.2e-5 at 6e-3 of it, for caps past
    // 1e17), and are used below that; a cap so small that they overflow is left to the
    // exponential (1e-7 of it is nothing).
    const double p3[3] = {0.9999996, -0.33321908, 0.12841609};
    const double p4[4] = {0.99999946, -0.33326318, 0.13190299, -0.04440228};
    double power = (double)a.cap_log2 * a.cap_x;
    float reach = 0.25f;
    bool high = false;
    for (int i = 0; i < 4; ++i, power *= (double)a.cap_x * a.cap_x) {
        const double c = power * (i < 3 ? p3[i] : p4[i]);
        high |= std::abs(c) > 1e37;
        if (i < 3) {
            if (std::abs(c) < FLT_MIN) reach = std::fmin(reach, i == 2 ? 0.02f : 6e-3f);
            a.cap_p3[i] = std::abs(c) < FLT_MIN ? 0.f : (float)c;
        }
        a.cap_p4[i] = (float)(power * p4[i]);
    }
    // z = s^2 stays finite
    a.cap_top = high ? -1.f : std::fmin(reach / a.cap_x, 1e18f);
    a.cap_top4 = high || std::abs(a.cap_p4[3]) < FLT_MIN ? -1.f : 0.5f / a.cap_x;
    if (s.softcap > 0.f && !(a.cap_in >= FLT_MIN && a.cap_in < INFINITY && a.cap_log2 < INFINITY)) return MF_ERR_ARG;
    return MF_OK;
}

// Padded head_dim the kernels are built for, or 0 if unsupported.
int padded_head_dim(int dtype, int d) {
    if (d <= 0 || (d & (d - 1)) != 0) return 0;  // powers of two only
    if (dtype == MF_F32) {
        if (d > 128) return 0;
        return d < 16 ? 16 : d;
    }
    if (d > 256) return 0;
    return d < 32 ? 32 : d;
}

inline int part_dstride_for(int head_dim) { return head_dim < 32 ? 32 : head_dim; }

}  // namespace
}  // namespace mf
