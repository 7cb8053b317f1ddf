// Varlen paged attention over a 4-bit pool (mf_pool4), with or without capped,
// biased and masked scores, on the plans of the 16-bit kernels (attn_kernels.h).
//
// The mathematics is theirs: columns are (row, query head) pairs of one kv head,
// S^T = K Q^T, an online softmax in log2 units with a lazy running maximum,
// O^T += V^T P^T. What differs is where K and V come from: codes go through
// gfx950's scaled conversions (two elements an instruction, the group's scale
// applied, exact in fp16 and bf16) on their way into the MFMA operands, so the
// products run on the 16-bit matrix rate with q and p unchanged.
//
// Decode items (attn4_narrow): a wave takes 32 keys at a time of 16 columns. Of the
// contraction over head_dim, lane (g, j) holds elements [g D/4, (g + 1) D/4) of key j
// -- for K one load of D/8 bytes, contiguous over the wave, whose scale is (D 128)
// the lane's own byte -- and Q's fragments are read in the same order. V lies
// token-minor in the pool, so a lane's 16 bytes are four keys of eight head_dim
// elements, which four conversions a key and a byte permute a pair turn into the
// operand of the 32-key product.
//
// Prefill items (attn4_wide): the four waves of a workgroup share a key range; each
// stage's codes are converted once, while they pass from registers to LDS, and the
// loop over the stage is the 16-bit kernels'.
#include "attn_kernels.h"
#include "kv4.h"

namespace mf {
namespace {

struct Attn4Args : ScoredArgs {
    const uint32_t* kc;
    const uint8_t* ks;
    const uint32_t* vc;
    const uint8_t* vs;
    int H;               // kv heads
    int tpb;             // 16-key tiles of a block
    uint32_t tpb_magic;  // ceil(2^32 / tpb), unused for 1
    uint32_t blk_bytes;  // codes of one block, K or V, all heads; its scales take a sixteenth
};

// Block index of tile t in its sequence's table.
__device__ __forceinline__ int block_of(const Attn4Args& a, int t) {
    return a.tpb == 1 ? t : (int)__umulhi((uint32_t)t, a.tpb_magic);
}

// Two softmax weights for the product with V, in the launch's 16-bit type, which the matrix
// instructions take both operands in. Rounding them (at most 2^-8 of a weight in bf16, 2^-11
// in fp16) is what the output's error has over one whose weights stay in 32 bits: 0.0022 of
// its norm against 0.0017 in bf16, 0.00025 against 0.00021 in fp16. The sums of weights and
// outputs are fp32.
template <int DT>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
    if constexpr (DT == MF_BF16) return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){x, y}, bf16x2));
    else return f32_to_bits<DT>(x) | (f32_to_bits<DT>(y) << 16);
}

constexpr int kDepth4 = 2;  // register buffers of the decode loop, 32 keys each

// One wave: the 16-column tile and the keys of its item. BLK16: 16-token blocks, where
// a tile is a block and the addresses of its slots fall away (of a pair of tiles, 81
// scalar instructions with them).
template <int DT, int DP, bool SC, bool BLK16>
__device__ __forceinline__ void attn4_narrow(const Attn4Args& a, const int32_t* it, const int wave, const bool coop) {
    constexpr int KW = DP / 32;                // words of a lane's K per 16 keys
    constexpr int VCH = DP / 16;               // head_dim elements of a lane's V per key
    constexpr int VW = DP == 256 ? 8 : 4;      // words of its V per 16 keys
    constexpr int XW = VCH / 2;                // 16-bit pairs of a lane's V per key
    constexpr float kNegInf = -__builtin_huge_valf();
    const int lane = threadIdx.x & 63;
    const int g = lane >> 4, j = lane & 15;
    const int s = it[0], h = it[1], c0 = it[2], kt0 = it[4], kt1 = it[5], pslot = it[6];
    const int row0 = it[8], ncols = it[9] * a.G, kv_len = it[10];
    int first = 0, prefix = 0;
    if constexpr (SC) {
        if (a.first_keys) first = a.first_keys[s];
        if (a.prefix_lens) prefix = a.prefix_lens[s];
    }
    // ---- the item's blocks (at most as many as its 128 tiles), two a lane
    const int32_t* trow = a.block_tables + (int64_t)s * a.bt_stride;
    const int last_block = block_of(a, max(kt1 - 1, 0)), block0 = min(block_of(a, kt0), last_block);
    const int tbl = trow[min(block0 + lane, last_block)];
    const int tbl_hi = trow[min(block0 + 64 + lane, last_block)];

    // ---- this lane's column
    const int cidx = c0 * 16 + j;
    const bool valid = cidx < ncols && it[3] > 0;
    const int r = valid ? cidx / a.G : 0;
    int prow = row0 + r;
    if (a.row_map) prow = a.row_map[prow];
    const int qhead = h * a.G + (valid ? cidx - r * a.G : 0);
    const int pos = reinterpret_cast<const int32_t*>(a.positions)[2 * (int64_t)prow];
    float slope = 0.f;
    if constexpr (SC) {
        if (a.slopes) slope = a.slopes[qhead] * 1.4426950408889634f;
    }
    uint4 qf[KW];
#pragma unroll
    for (int c = 0; c < KW; ++c) {
        const uint4 v = *(const uint4*)(a.q + ((int64_t)prow * a.q_sr + (int64_t)qhead * a.q_sh + g * (DP / 4) + c * 8) * 2);
        qf[c] = make_uint4(v.x ^ a.q_sign, v.y ^ a.q_sign, v.z ^ a.q_sign, v.w ^ a.q_sign);
    }
    const int reach = valid ? (SC ? max(pos, prefix - 1) : pos) : -1;
    const int lim = reach >= 0 ? min(min(reach, kv_len - 1), kt1 * 16 - 1) : -1;  // last key of the item the column sees

    // ---- the stream. A tile's addresses are scalar: the head's bases, the block and
    // the 16 slots of it; a lane's byte offsets never change.
    struct Tile {
        uint32_t kw[KW], ks, vw[VW], vs;
    };
    const int bs = BLK16 ? 16 : a.tpb * 16;
    constexpr int VSH = DP == 64 ? 1 : DP == 32 ? 2 : 0;  // lanes that share a word's eight elements: 2^VSH
    const int vchunk = DP == 256 ? 2 * j : j >> VSH;
    const uint32_t k_lane = (uint32_t)(j * (DP / 8) + g * KW) * 4;
    const uint32_t v_lane = (uint32_t)(vchunk * bs + 4 * g) * 4;
    const uint32_t ks_lane = (uint32_t)(j * (DP / 32) + (DP == 256 ? 2 * g : DP == 128 ? g : DP == 64 ? g >> 1 : 0));
    const uint32_t vs_lane = (uint32_t)((vchunk >> 2) * bs + 4 * g);
    const char* kc_h = (const char*)a.kc + (int64_t)h * bs * (DP / 2);
    const char* ks_h = (const char*)a.ks + (int64_t)h * bs * (DP / 32);
    const char* vc_h = (const char*)a.vc + (int64_t)h * bs * (DP / 2);
    const char* vs_h = (const char*)a.vs + (int64_t)h * bs * (DP / 32);
    int at_block = 0, at_off = 0;  // of the next tile to load: table entry, first slot
    auto load = [&](Tile& x) __attribute__((always_inline)) {
        const int e0 = __builtin_amdgcn_readlane(tbl, at_block & 63), e1 = __builtin_amdgcn_readlane(tbl_hi, at_block & 63);
        const uint64_t o = (uint64_t)(uint32_t)(at_block < 64 ? e0 : e1) * a.blk_bytes;
        const char *kc = kc_h + o, *ks = ks_h + (o >> 4), *vc = vc_h + o, *vs = vs_h + (o >> 4);
        if constexpr (!BLK16) {
            kc += (uint32_t)(at_off * (DP / 2));
            ks += (uint32_t)(at_off * (DP / 32));
            vc += (uint32_t)(at_off * 4);
            vs += (uint32_t)at_off;
        }
        ld_words<KW * 4>(kc + k_lane, x.kw);
        if constexpr (DP == 256) x.ks = *(const uint16_t*)(ks + ks_lane);
        else x.ks = *(const uint8_t*)(ks + ks_lane);
        ld_words<16>(vc + v_lane, x.vw);
        if constexpr (DP == 256) ld_words<16>(vc + (v_lane + 4 * (uint32_t)bs), x.vw + 4);
        x.vs = *(const uint32_t*)(vs + vs_lane);
    };

    float m = kMinM, l = 0.f;
    float thr = SC ? kMinM + kLazyLog2 : (kMinM + kLazyLog2) * a.inv_scale_log2;
    f32x4 acc[VCH];
#pragma unroll
    for (int c = 0; c < VCH; ++c) acc[c] = f32x4{0.f, 0.f, 0.f, 0.f};

    if (kt1 > kt0) {
        int maxlim = lim, minlim = valid ? lim : INT_MAX;
#pragma unroll
        for (int o = 8; o >= 1; o >>= 1) {  // the four lane groups hold the same columns
            maxlim = max(maxlim, __shfl_xor(maxlim, o, 64));
            minlim = min(minlim, __shfl_xor(minlim, o, 64));
        }
        maxlim = __builtin_amdgcn_readfirstlane(maxlim);
        minlim = __builtin_amdgcn_readfirstlane(minlim);
        const int tb = SC ? min(max(kt0, first >> 4), kt1) : kt0;
        const int te = maxlim < 0 ? tb : max(tb, min(kt1, (maxlim >> 4) + 1));

        auto process = [&](int t, Tile& x, Tile& y) __attribute__((always_inline)) {
            const int key0 = t * 16 + 4 * g;  // this lane's keys: key0 + r, key0 + 16 + r
            // a key's V scale: its byte among the bits the conversion reads
            uint32_t vscale[8];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                vscale[k] = k < 3 ? x.vs << (23 - 8 * k) : x.vs >> 1;
                vscale[4 + k] = k < 3 ? y.vs << (23 - 8 * k) : y.vs >> 1;
            }
            // keys no column sees may hold anything: their V is cleared, and with it
            // a scale that makes zeros NaN
            if (t * 16 + 31 > maxlim || (SC && t * 16 < first)) {
                asm volatile("");  // a branch: one tile in a range takes it, as selects all would
                const int end = maxlim - key0, begin = first - key0;
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const int key = (k & 3) + 16 * (k >> 2);
                    const bool live = key <= end && (!SC || key >= begin);
                    vscale[k] = live ? vscale[k] : 0x3f800000u;
#pragma unroll
                    for (int u = 0; u < VW / 4; ++u) {
                        uint32_t& w = (k < 4 ? x : y).vw[4 * u + (k & 3)];
                        w = live ? w : 0u;
                    }
                }
                // K likewise in a scored launch: a block's largest score picks how it is
                // capped (score_all)
                if constexpr (SC) {
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        Tile& z = u ? y : x;
                        const int key = t * 16 + 16 * u + j;
                        const bool live = key <= maxlim && key >= first;
                        z.ks = live ? z.ks : 0x7f7fu;
#pragma unroll
                        for (int c = 0; c < KW; ++c) z.kw[c] = live ? z.kw[c] : 0u;
                    }
                }
            }
            f32x4 st[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const Tile& z = u ? y : x;
                st[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < KW; ++c) {
                    const float ks = scale4(DP == 256 ? (c < 4 ? z.ks & 255u : z.ks >> 8) : z.ks);
                    st[u] = mfma_qk<DT>(octet4<DT>(z.kw[c], ks), qf[c], st[u]);
                }
            }
            float sv[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) sv[k] = st[k >> 2][k & 3];
            if constexpr (SC) {
                const float dist = (float)(key0 - pos);
                score_all<DT>(sv, a, slope, [&](int k) { return dist + ((k & 3) + 16 * (k >> 2)); });
            }
            if (t * 16 + 31 > minlim || (SC && t * 16 < first)) {
                asm volatile("");
                const int end = lim - key0, begin = first - key0;
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const int key = (k & 3) + 16 * (k >> 2);
                    sv[k] = key <= end && (!SC || key >= begin) ? sv[k] : kNegInf;
                }
            }
            float lmax = sv[0];
#pragma unroll
            for (int k = 1; k < 8; ++k) lmax = fmax_prop(lmax, sv[k]);
            if (__builtin_amdgcn_ballot_w64(lmax > thr) != 0) {
                const float cm = group_max4(lmax);
                const float mn = fmaxf(m, SC ? cm : cm * a.scale_log2);
                const float alpha = __builtin_amdgcn_exp2f(m - mn);
                l *= alpha;
#pragma unroll
                for (int c = 0; c < VCH; ++c) acc[c] *= alpha;
                m = mn;
                thr = SC ? mn + kLazyLog2 : (mn + kLazyLog2) * a.inv_scale_log2;
            }
            float p[8];
#pragma unroll
            for (int k = 0; k < 8; ++k)
                p[k] = __builtin_amdgcn_exp2f(SC ? sv[k] - m : __builtin_fmaf(sv[k], a.scale_log2, -m));
            l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
            const uint4 pf = make_uint4(pack2<DT>(p[0], p[1]), pack2<DT>(p[2], p[3]), pack2<DT>(p[4], p[5]),
                                        pack2<DT>(p[6], p[7]));
            // V: XW pairs of the lane's elements for each of its eight keys, then
            // pairs of keys per element
            uint32_t v[8][XW];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const uint32_t* w = (k < 4 ? x : y).vw + (k & 3);
                if constexpr (VCH >= 8) {
#pragma unroll
                    for (int u = 0; u < VW / 4; ++u) {
                        const uint4 o = octet4<DT>(w[4 * u], __uint_as_float(vscale[k]));
                        v[k][4 * u] = o.x; v[k][4 * u + 1] = o.y; v[k][4 * u + 2] = o.z; v[k][4 * u + 3] = o.w;
                    }
                } else if constexpr (VCH == 4) {
                    const uint32_t half = w[0] >> (16 * (j & 1));
                    v[k][0] = pair4<DT, 0>(half, __uint_as_float(vscale[k]));
                    v[k][1] = pair4<DT, 1>(half, __uint_as_float(vscale[k]));
                } else {
                    v[k][0] = pair4<DT, 0>(w[0] >> (8 * (j & 3)), __uint_as_float(vscale[k]));
                }
            }
#pragma unroll
            for (int u = 0; u < XW; ++u) {
                uint32_t lo[4], hi[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    lo[k] = __builtin_amdgcn_perm(v[2 * k + 1][u], v[2 * k][u], 0x05040100u);
                    hi[k] = __builtin_amdgcn_perm(v[2 * k + 1][u], v[2 * k][u], 0x07060302u);
                }
                acc[2 * u] = mfma_qk<DT>(make_uint4(lo[0], lo[1], lo[2], lo[3]), pf, acc[2 * u]);
                acc[2 * u + 1] = mfma_qk<DT>(make_uint4(hi[0], hi[1], hi[2], hi[3]), pf, acc[2 * u + 1]);
            }
        };
        if (tb < te) {
            // a ring of kDepth4 buffers of two tiles; loads past the range's end
            // read its last tile again, masked
            Tile ring[kDepth4][2];
            const int last = te - 1;
            int next = tb;
            at_block = block_of(a, tb) - block0;
            at_off = (tb - block_of(a, tb) * a.tpb) * 16;
            auto step = [&]() __attribute__((always_inline)) {
                if constexpr (BLK16) {
                    at_block = min(at_block + 1, last - block0);
                } else {
                    const bool more = next < last, wrap = more && at_off + 16 == bs;
                    at_off = wrap ? 0 : more ? at_off + 16 : at_off;
                    at_block += wrap ? 1 : 0;
                    ++next;
                }
            };
            auto fetch = [&](Tile (&x)[2]) __attribute__((always_inline)) {
                load(x[0]);
                step();
                load(x[1]);
                step();
            };
            int t = tb;
#pragma unroll
            for (int i = 0; i < kDepth4 - 1; ++i) fetch(ring[i]);
            for (int n = (te - tb + 1) / 2 / kDepth4; n > 0; --n) {
#pragma unroll
                for (int u = 0; u < kDepth4; ++u) {
                    fetch(ring[(u + kDepth4 - 1) % kDepth4]);
                    process(t, ring[u][0], ring[u][1]);
                    t += 2;
                }
            }
            auto tail = [&](auto self, auto U) {
                constexpr int u = decltype(U)::value;
                if constexpr (u < kDepth4 - 1) {
                    if (t <= last) {
                        process(t, ring[u][0], ring[u][1]);
                        t += 2;
                        self(self, std::integral_constant<int, u + 1>{});
                    }
                }
            };
            tail(tail, std::integral_constant<int, 0>{});
        }
    }

    // ---- finish: lane (g, j) holds column j's elements (4g + r) VCH + c in acc[c][r]
    l = group_sum4(l);
    float M = m, L = l;
    if (coop) {
        // the four waves took quarters of one range: each combines the elements of
        // its own r over the waves' states, left in LDS
        auto s_acc = reinterpret_cast<float (*)[4 * VCH][64]>(attn_lds);
        auto s_m = reinterpret_cast<float (*)[16]>(attn_lds + kWaves * 4 * VCH * 64 * 4);
        auto s_l = s_m + kWaves;
#pragma unroll
        for (int rr = 0; rr < 4; ++rr)
#pragma unroll
            for (int c = 0; c < VCH; ++c) s_acc[wave][rr * VCH + c][lane] = acc[c][rr];
        if (g == 0) {
            s_m[wave][j] = m;
            s_l[wave][j] = l;
        }
        __syncthreads();
        float o[VCH];
        M = kMinM;
        L = 0.f;
#pragma unroll
        for (int u = 0; u < kWaves; ++u) M = fmaxf(M, s_m[u][j]);
#pragma unroll
        for (int c = 0; c < VCH; ++c) o[c] = 0.f;
#pragma unroll
        for (int u = 0; u < kWaves; ++u) {
            const float w = __builtin_amdgcn_exp2f(s_m[u][j] - M);
            L += s_l[u][j] * w;
#pragma unroll
            for (int c = 0; c < VCH; ++c) o[c] += w * s_acc[u][wave * VCH + c][lane];
        }
        if (!valid) return;
        const float inv = L > 0.f ? 1.f / L : 0.f;
#pragma unroll
        for (int c = 0; c < VCH; ++c) o[c] *= inv;
        const int d0 = (4 * g + wave) * VCH;
        if (pslot < 0) {
            store_elems<DT, VCH>(a.out + ((int64_t)prow * a.o_sr + (int64_t)qhead * a.o_sh + d0) * 2, o);
        } else {
            store_elems<MF_F32, VCH>(partial_out<MF_F32>(a, pslot, j, d0), o);
            if (g == 0 && wave == 0) {
                partial_ml(a, pslot)[j] = M;
                partial_ml(a, pslot)[16 + j] = L;
            }
        }
        return;
    }
    if (!valid) return;
    const float inv = L > 0.f ? 1.f / L : 0.f;
    float o[4 * VCH];
#pragma unroll
    for (int rr = 0; rr < 4; ++rr)
#pragma unroll
        for (int c = 0; c < VCH; ++c) o[rr * VCH + c] = acc[c][rr] * inv;
    if (pslot < 0) {
        store_out_chunk<DT, VCH>(a.out + ((int64_t)prow * a.o_sr + (int64_t)qhead * a.o_sh + 4 * g * VCH) * 2, o);
    } else {
        store_out_chunk<MF_F32, VCH>(partial_out<MF_F32>(a, pslot, j, 4 * g * VCH), o);
        if (g == 0) {
            partial_ml(a, pslot)[j] = M;
            partial_ml(a, pslot)[16 + j] = L;
        }
    }
}

// ------------------------------------------------------- workgroup-shared items
// Keys of a stage (two buffers of K and V rows, 64 KB of LDS at D 128) and of one
// softmax step. Two chunks of 2048 rows after up to 6144 keys, 40/8 heads x 128 (450
// GFLOP): 541 us with stages and steps of 32 keys at three waves per SIMD, 487 with
// stages of 64 at two, 472 with steps of 64 as well (952 TFLOP/s): two score chains at
// once, one test of the maximum for both, half the barriers.
constexpr int kWideKeys4 = 64;
template <int DP>
constexpr int wide_lds4() { return 2 * 2 * kWideKeys4 * DP * 2; }

// `it` is this wave's item, nct the column tiles it takes of it; cols holds the first
// column tile and the tiles of all four.
template <int DT, int DP, bool SC>
__device__ __forceinline__ void attn4_wide(const Attn4Args& a, const int32_t* it, const int nct,
                                           const int (&cols)[kWaves][2]) {
    constexpr int RB = DP * 2;       // bytes of a key's row in LDS
    constexpr int NCH = RB / 16;     // 16-byte chunks of a row: the eight elements of a word
    constexpr int KEYS = kWideKeys4, TS = KEYS / 16;
    constexpr int RPB = 256 / RB;    // rows in 256 bytes
    constexpr int NQ = DP / 16, ND = DP / 32;
    constexpr int HALF = KEYS * RB, STG = 2 * HALF;
    constexpr int NW = KEYS * (DP / 8) / 256;  // words of a thread's K (and V) per stage
    static_assert(NW == 1 || NW == 2 || NW == 4, "stage layout");
    constexpr float kNegInf = -__builtin_huge_valf();
    const int lane = threadIdx.x & 63;
    const int hf = lane >> 5;
    const int s = it[0], h = it[1], c0 = it[2], kt0 = it[4], kt1 = it[5], pslot = it[6];
    const int row0 = it[8], nrows = it[9], kv_len = it[10];
    int first = 0, prefix = 0;
    if constexpr (SC) {
        if (a.first_keys) first = a.first_keys[s];
        if (a.prefix_lens) prefix = a.prefix_lens[s];
    }
    const int32_t* trow = a.block_tables + (int64_t)s * a.bt_stride;

    // ---- this lane's column, and two of the workgroup's other columns, whose
    // positions say how far the stages run
    const int ct = (lane & 31) >> 4, j = lane & 15;
    const int cidx = c0 * 16 + (lane & 31);
    const bool valid = ct < nct && cidx < nrows * a.G;
    const int col = valid ? cidx : 0;
    const int crow = (int)((unsigned)col / (unsigned)a.G);
    const int qhead = h * a.G + col - crow * a.G;
    int rows[3] = {row0 + crow, row0, row0};
    bool other[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int c = (hf ? cols[2 * k + 1][0] : cols[2 * k][0]) * 16 + (lane & 31);
        other[k] = ct < (hf ? cols[2 * k + 1][1] : cols[2 * k][1]) && c < nrows * a.G;
        rows[1 + k] = row0 + (int)((unsigned)(other[k] ? c : 0) / (unsigned)a.G);
    }
    if (a.row_map) {
#pragma unroll
        for (int k = 0; k < 3; ++k) rows[k] = a.row_map[rows[k]];
    }
    int rpos[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) rpos[k] = reinterpret_cast<const int32_t*>(a.positions)[2 * (int64_t)rows[k]];
    const int prow = rows[0];
    float slope = 0.f;
    if constexpr (SC) {
        if (a.slopes) slope = a.slopes[qhead] * 1.4426950408889634f;
    }
    auto reach = [&](int pos) { return SC ? max(pos, prefix - 1) : pos; };
    const int qpos = valid ? reach(rpos[0]) : -1;
    const int wpos = max(other[0] ? reach(rpos[1]) : -1, other[1] ? reach(rpos[2]) : -1);
    uint4 qf[NQ];
#pragma unroll
    for (int c = 0; c < NQ; ++c) {
        const uint4 v = *(const uint4*)(a.q + ((int64_t)prow * a.q_sr + (int64_t)qhead * a.q_sh + c * 16 + hf * 8) * 2);
        qf[c] = make_uint4(v.x ^ a.q_sign, v.y ^ a.q_sign, v.z ^ a.q_sign, v.w ^ a.q_sign);
    }
    const int end_key = min(kv_len, kt1 * 16);
    const int lim = qpos >= 0 ? min(qpos, end_key - 1) : -1;
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
    const int te = wglim < kt0 * 16 ? kt0 : (wglim >> 4) + 1;
    const int nst = (te - kt0 + TS - 1) / TS;

    // ---- staging: this thread's words of a stage. K: NW words of one key; V: NW
    // tokens of one word's elements. A 16-key tile belongs to whole waves, so a
    // stage's addresses are scalar bases and lane offsets that never change.
    const int x = (int)threadIdx.x;
    const int tt = __builtin_amdgcn_readfirstlane(x / (256 / TS));  // tile of the stage
    const int xi = x % (256 / TS);                                  // thread of the tile
    constexpr int KT = (DP / 8) / NW;                               // threads of a key
    const int kkey = xi / KT, kword = (xi % KT) * NW;
    const int vword = xi % (DP / 8), vtok = xi / (DP / 8) * NW;
    const int bs = a.tpb * 16;
    const uint32_t kc_lane = (uint32_t)(kkey * (DP / 8) + kword) * 4, ks_lane = (uint32_t)(kkey * (DP / 32) + (kword >> 2));
    const uint32_t vc_lane = (uint32_t)(vword * bs + vtok) * 4, vs_lane = (uint32_t)((vword >> 2) * bs + vtok);
    uint32_t k_dst[NW], v_dst[NW];  // bytes inside a stage
#pragma unroll
    for (int k = 0; k < NW; ++k) {
        k_dst[k] = (uint32_t)((tt * 16 + kkey) * RB + (((kword + k) ^ ((kkey / RPB) & (NCH - 1))) << 4));
        v_dst[k] = (uint32_t)(HALF + (tt * 16 + vtok + k) * RB + ((vword ^ ((((vtok + k) & 3) / RPB) << 2)) << 4));
    }
    struct Codes {
        uint32_t kw[NW], vw[NW], ks, vs;
    };
    auto entry = [&](int u) { return trow[block_of(a, min(kt0 + TS * u + tt, te - 1))]; };
    auto fetch = [&](int u, int entry_, Codes& c) __attribute__((always_inline)) {
        const int t = min(kt0 + TS * u + tt, te - 1);
        const int off = (t - block_of(a, t) * a.tpb) * 16;
        const int64_t row = (int64_t)__builtin_amdgcn_readfirstlane(entry_) * a.H + h;
        ld_words<NW * 4>((const char*)(a.kc + (row * bs + off) * (DP / 8)) + kc_lane, c.kw);
        c.ks = (a.ks + (row * bs + off) * (DP / 32))[ks_lane];
        ld_words<NW * 4>((const char*)(a.vc + row * (DP / 8) * bs + off) + vc_lane, c.vw);
        const uint8_t* vs = a.vs + row * (DP / 32) * bs + off;
        if constexpr (NW == 4) c.vs = *(const uint32_t*)(vs + vs_lane);
        else if constexpr (NW == 2) c.vs = *(const uint16_t*)(vs + vs_lane);
        else c.vs = vs[vs_lane];
    };
    auto stage = [&](int u, char* stg, Codes& c) __attribute__((always_inline)) {
        uint32_t vs[NW];
#pragma unroll
        for (int k = 0; k < NW; ++k) vs[k] = ((c.vs >> (8 * k)) << 23) & 0x7f800000u;
        const int key0 = (kt0 + TS * u + tt) * 16;
        if (key0 + 15 > wglim || (SC && key0 < first)) {
            // keys no row sees may hold anything: cleared, and a scale that makes
            // zeros NaN with them
#pragma unroll
            for (int k = 0; k < NW; ++k) {
                const int key = key0 + vtok + k;
                const bool live = key <= wglim && (!SC || key >= first);
                vs[k] = live ? vs[k] : 0x3f800000u;
                c.vw[k] = live ? c.vw[k] : 0u;
            }
            if constexpr (SC) {  // K too, as in attn4_narrow
                const bool live = key0 + kkey <= wglim && key0 + kkey >= first;
                c.ks = live ? c.ks : 127u;
#pragma unroll
                for (int k = 0; k < NW; ++k) c.kw[k] = live ? c.kw[k] : 0u;
            }
        }
        const float ks = scale4(c.ks);
#pragma unroll
        for (int k = 0; k < NW; ++k) *(uint4*)(stg + k_dst[k]) = octet4<DT>(c.kw[k], ks);
#pragma unroll
        for (int k = 0; k < NW; ++k) *(uint4*)(stg + v_dst[k]) = octet4<DT>(c.vw[k], __uint_as_float(vs[k]));
    };
    auto sync = [&]() {
        __builtin_amdgcn_s_waitcnt((15) | (3 << 14) | (7 << 4) | (0 << 8));  // lgkmcnt(0)
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };

    float m = kMinM, l = 0.f;
    float thr = SC ? kMinM + kLazyLog2 : (kMinM + kLazyLog2) * a.inv_scale_log2;
    f32x16 acc[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;
    uint32_t kaddr[NQ], vaddr[ND];
#pragma unroll
    for (int c = 0; c < NQ; ++c)
        kaddr[c] = (uint32_t)((lane & 31) * RB + (((2 * c + hf) ^ ((j / RPB) & (NCH - 1))) << 4));
#pragma unroll
    for (int d = 0; d < ND; ++d)
        vaddr[d] = (uint32_t)(HALF + (4 * hf + (j >> 2)) * RB +
                              (((4 * d + 2 * ct + ((j & 3) >> 1)) ^ (((j >> 2) / RPB) << 2)) << 4) + 8 * (j & 1));

    // NS blocks of 32 keys, one softmax step
    constexpr int NS = KEYS / 32;
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
        if (key0 + KEYS - 1 > minlim || (SC && key0 < first)) {
#pragma unroll
            for (int n = 0; n < NS; ++n)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int key = key0 + 32 * n + 8 * (i >> 2) + 4 * hf + (i & 3);
                    st[n][i] = key <= lim && (!SC || key >= first) ? st[n][i] : kNegInf;
                }
        }
        float lmax = st[0][0];
#pragma unroll
        for (int n = 0; n < NS; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) lmax = fmax_prop(lmax, st[n][i]);
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
                const float p0 =
                    __builtin_amdgcn_exp2f(SC ? st[n][2 * i] - m : __builtin_fmaf(st[n][2 * i], a.scale_log2, -m));
                const float p1 =
                    __builtin_amdgcn_exp2f(SC ? st[n][2 * i + 1] - m : __builtin_fmaf(st[n][2 * i + 1], a.scale_log2, -m));
                sum += p0 + p1;
                pw[i] = pack2<DT>(p0, p1);
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
        Codes c;
        fetch(0, entry(0), c);
        int blk = entry(1);
        stage(0, attn_lds, c);
        fetch(1, blk, c);
        blk = entry(2);
        sync();
        // the buffer being written was read in the round before, which every wave
        // has left; the codes in flight meanwhile are two stages ahead
        auto round = [&](int u, auto odd) __attribute__((always_inline)) {
            constexpr int B = decltype(odd)::value;
            if (u + 1 < nst) {
                stage(u + 1, attn_lds + (1 - B) * STG, c);
                fetch(u + 2, blk, c);
                blk = entry(u + 3);
            }
            const int key0 = (kt0 + TS * u) * 16;
            if (key0 <= maxlim) tile(attn_lds + B * STG, key0);
            sync();
        };
        for (int u = 0; u < nst; u += 2) {
            round(u, std::integral_constant<int, 0>{});
            if (u + 1 < nst) round(u + 1, std::integral_constant<int, 1>{});
        }
    }

    // ---- finish: lane (hf, column) holds elements 32d + 8b + 4hf .. + 3
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
    const float lt = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    const float inv = lt > 0.f ? 1.f / lt : 0.f;
    if (!valid) return;
    if (pslot >= 0) {
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
            partial_ml(a, pslot + ct)[j] = m;
            partial_ml(a, pslot + ct)[16 + j] = lt;
        }
        return;
    }
    char* dst = a.out + ((int64_t)prow * a.o_sr + (int64_t)qhead * a.o_sh) * 2;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int b = 0; b < 4; b += 2) {
            // the column's two lanes trade blocks, so that each stores 16 bytes (both
            // are valid or neither)
            uint32_t w[2][2];
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    w[e][k] = f32_to_bits<DT>(acc[d][4 * (b + e) + 2 * k] * inv) |
                              (f32_to_bits<DT>(acc[d][4 * (b + e) + 2 * k + 1] * inv) << 16);
            auto y = __builtin_amdgcn_permlane32_swap(w[0][0], w[1][0], false, false);
            auto z = __builtin_amdgcn_permlane32_swap(w[0][1], w[1][1], false, false);
            *(uint4*)(dst + (32 * d + 8 * (b + hf)) * 2) = make_uint4(y[0], z[0], y[1], z[1]);
        }
}

template <int DP>
constexpr int lds4(bool wide) {
    if constexpr (DP == 256) return coop_lds_bytes<DP>();
    else return wide && wide_lds4<DP>() > coop_lds_bytes<DP>() ? wide_lds4<DP>() : coop_lds_bytes<DP>();
}

// What a launch holds: narrow items, wide ones, or both (the narrow ones' workgroups
// first).
enum { kNarrow4, kWide4, kBoth4 };

// Waves per SIMD the register allocator leaves room for. A wide workgroup at D 128
// takes 245 registers; held to the 168 of three waves it spills.
template <int DP, int KIND>
constexpr int waves4() {
    return DP == 256 ? 1 : KIND == kNarrow4 || DP == 128 ? 2 : 3;
}

template <int DT, int DP, bool SC, int KIND, bool BLK16>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(waves4<DP, KIND>())))
void attn4_kernel(const int32_t* items, Attn4Args a, int narrow_blocks, const int32_t* wide_items, int wide_num,
                  const int32_t* wide_count) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int b = blockIdx.x;
    if (KIND == kNarrow4 || (KIND == kBoth4 && b < narrow_blocks)) {
        const int item = b * kWaves + wave;
        const int32_t* it = items + (int64_t)item * MF_PLAN_ITEM_INTS;
        if (item >= (a.dev_count ? *a.dev_count : a.num_items)) return;
        const bool coop = it[11] != 0;  // of the whole workgroup
        if (!coop && it[3] == 0) return;  // padding
        attn4_narrow<DT, DP, SC, BLK16>(a, it, wave, coop);
        return;
    }
    if constexpr (KIND != kNarrow4 && DP < 256) {
        const int block = KIND == kBoth4 ? b - narrow_blocks : b;
        const int num = wide_count ? *wide_count : wide_num;
        if (block * kWaves >= num) return;
        const int32_t* i0 = wide_items + (int64_t)block * kWaves * MF_PLAN_ITEM_INTS;
        bool same = true;
#pragma unroll
        for (int w = 1; w < kWaves; ++w) {
            const int32_t* iw = i0 + w * MF_PLAN_ITEM_INTS;
            same = same & (iw[0] == i0[0]) & (iw[1] == i0[1]) & (iw[4] == i0[4]) & (iw[5] == i0[5]);
        }
        // A workgroup of unrelated items (plans that are not made for a device pool
        // short ones) runs them one after the other, each the columns of one wave.
#pragma unroll 1
        for (int k = 0; k < (same ? 1 : kWaves); ++k) {
            int cols[kWaves][2];
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const int32_t* iw = i0 + (same ? w : k) * MF_PLAN_ITEM_INTS;
                const int2 tiles = *(const int2*)(iw + 2);
                cols[w][0] = tiles.x;
                cols[w][1] = same | (w == k) ? tiles.y : 0;
            }
            const int32_t* it = i0 + (same ? wave : k) * MF_PLAN_ITEM_INTS;
            attn4_wide<DT, DP, SC>(a, it, same | (wave == k) ? it[3] : 0, cols);
        }
    }
}

template <int DT, int DP, bool SC>
int launch4(Attn4Args a, const int32_t* items, int64_t n_narrow, int64_t n_wide, const int32_t* merges,
            int64_t n_merges, const int32_t* dev_counts, hipStream_t stream) {
    if (DP == 256 && n_wide > 0) return MF_ERR_ARG;  // the plan was made for another head_dim
    if (n_narrow + n_wide > 0) {
        a.num_items = (int)n_narrow;
        a.dev_count = dev_counts;
        const int32_t* wide = items + n_narrow * MF_PLAN_ITEM_INTS;
        const int nb = (int)(n_narrow / kWaves);
        const dim3 grid((unsigned)((n_narrow + n_wide) / kWaves));
        const int32_t* wide_count = dev_counts ? dev_counts + 1 : nullptr;
        const bool blk16 = a.tpb == 1;
#define MF_LAUNCH4(KIND, B16, LDS)                                                                                   \
    hipLaunchKernelGGL((attn4_kernel<DT, DP, SC, KIND, B16>), grid, dim3(256), LDS, stream, items, a, nb, wide,      \
                       (int)n_wide, wide_count)
        if (n_wide == 0) {
            if (blk16) MF_LAUNCH4(kNarrow4, true, lds4<DP>(false));
            else MF_LAUNCH4(kNarrow4, false, lds4<DP>(false));
        } else if constexpr (DP < 256) {
            if (n_narrow == 0) MF_LAUNCH4(kWide4, false, wide_lds4<DP>());
            else if (blk16) MF_LAUNCH4(kBoth4, true, lds4<DP>(true));
            else MF_LAUNCH4(kBoth4, false, lds4<DP>(true));
        }
#undef MF_LAUNCH4
        if (int st = check_launch()) return st;
    }
    if (n_merges > 0) {
        a.dev_count = dev_counts ? dev_counts + 2 : nullptr;
        return launch_merge32<DT, DP>(a, merges, n_merges, n_wide == 0, stream);
    }
    return MF_OK;
}

}  // namespace
}  // namespace mf

extern "C" int mf_paged_attention4(const mf_scoring* scoring, const void* q, int64_t q_stride_row,
                                   int64_t q_stride_head, void* out, int64_t out_stride_row, int64_t out_stride_head,
                                   int dtype, const mf_pool4* pool, const int32_t* block_tables,
                                   int64_t block_table_stride, const int32_t* cu_seqlens, const int32_t* kv_lens,
                                   const int64_t* positions, const int32_t* row_map, int num_q_heads, float scale,
                                   const int32_t* plan_items, int64_t num_items_narrow, int64_t num_items_wide,
                                   const int32_t* plan_merges, int64_t num_merges, const int32_t* device_counts,
                                   float* partials, int64_t partials_floats, mf_stream_t stream) {
    using namespace mf;
    if (int st = check_pool4(pool)) return st;
    if (!dtype_ok(dtype) || dtype == MF_F32) return MF_ERR_UNSUPPORTED;
    if (dtype != pool->dtype) return MF_ERR_ARG;
    if (!(std::fabs(scale) < INFINITY) || num_q_heads <= 0 || num_q_heads % pool->num_heads) return MF_ERR_ARG;
    if (num_items_narrow < 0 || num_items_wide < 0 || num_merges < 0 || num_items_narrow % kWaves ||
        num_items_wide % kWaves)
        return MF_ERR_ARG;
    if (num_items_narrow + num_items_wide == 0 && num_merges == 0) return MF_OK;
    if (!q || !out || !block_tables || !cu_seqlens || !kv_lens || !positions) return MF_ERR_ARG;
    if (num_items_narrow + num_items_wide > 0 && !plan_items) return MF_ERR_ARG;
    if (num_merges > 0 && (!plan_merges || !partials || partials_floats <= 0)) return MF_ERR_WORKSPACE;
    if ((q_stride_row | q_stride_head) % 8 || (uintptr_t)q % 16) return MF_ERR_ARG;
    const int out_align = std::min(16, 4 * (pool->head_dim / 16) * 2);
    if ((out_stride_row * 2) % out_align || (out_stride_head * 2) % out_align || (uintptr_t)out % out_align)
        return MF_ERR_ARG;
    Attn4Args a{};
    a.q = (const char*)q;
    a.q_sr = q_stride_row;
    a.q_sh = q_stride_head;
    a.out = (char*)out;
    a.o_sr = out_stride_row;
    a.o_sh = out_stride_head;
    a.block_size = pool->block_size;
    a.block_tables = block_tables;
    a.bt_stride = block_table_stride;
    a.positions = positions;
    a.row_map = row_map;
    a.H = a.num_kv_heads = pool->num_heads;
    a.G = num_q_heads / pool->num_heads;
    a.head_dim = pool->head_dim;
    a.kc = pool->key_codes;
    a.ks = pool->key_scales;
    a.vc = pool->value_codes;
    a.vs = pool->value_scales;
    a.tpb = pool->block_size / 16;
    const int64_t blk_bytes = (int64_t)pool->num_heads * pool->block_size * (pool->head_dim / 2);
    if (blk_bytes > INT_MAX) return MF_ERR_ARG;
    a.blk_bytes = (uint32_t)blk_bytes;
    a.tpb_magic = a.tpb > 1 ? (uint32_t)(((1ull << 32) + a.tpb - 1) / a.tpb) : 0u;
    // as in mf_paged_attention: a negative scale turns q's signs, a zero one becomes
    // 2^-100
    a.q_sign = scale < 0.f ? 0x80008000u : 0u;
    a.scale_log2 = scale == 0.f ? 0x1p-100f : std::fabs(scale) * 1.4426950408889634f;
    a.inv_scale_log2 = 1.f / a.scale_log2;
    a.partials = partials;
    a.part_dstride = part_dstride_for(pool->head_dim);
    a.merges = plan_merges;
    if (scoring) {
        if (int st = set_scoring(a, *scoring)) return st;
    }
    hipStream_t st = (hipStream_t)stream;
#define MF_ATTN4_CASE(DT, DPV)                                                                                       \
    if (dtype == DT && pool->head_dim == DPV)                                                                        \
        return scoring ? launch4<DT, DPV, true>(a, plan_items, num_items_narrow, num_items_wide, plan_merges,        \
                                                num_merges, device_counts, st)                                       \
                       : launch4<DT, DPV, false>(a, plan_items, num_items_narrow, num_items_wide, plan_merges,       \
                                                 num_merges, device_counts, st);
    MF_ATTN4_CASE(MF_BF16, 32)
    MF_ATTN4_CASE(MF_BF16, 64)
    MF_ATTN4_CASE(MF_BF16, 128)
    MF_ATTN4_CASE(MF_BF16, 256)
    MF_ATTN4_CASE(MF_F16, 32)
    MF_ATTN4_CASE(MF_F16, 64)
    MF_ATTN4_CASE(MF_F16, 128)
    MF_ATTN4_CASE(MF_F16, 256)
#undef MF_ATTN4_CASE
    return MF_ERR_UNSUPPORTED;
}
