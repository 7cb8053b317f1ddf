// Writing rows to the 4-bit pool and gathering them back.
//
// A group is 32 elements x_i of one token and head. With top = max |x_i| its scale is
// 2^E, E = floor(log2 top) - 2, one more where top exceeds 1.75 * 2^floor(log2 top):
// top then lies in (3.5, 7] * 2^E, where no element is off by more than 2^E (6 stands
// for up to 7). E is bounded by what the pool's type can hold (kv4.h). A code is the
// nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 times 2^E, ties to the even code, with the
// sign: gfx950's conversion, checked against that definition. A group holding NaN or
// an infinity gets the scale byte 255 and reads as NaN.
//
// Both kernels are bound by the bytes they move. A lane takes one word (eight elements)
// of four consecutive rows, key and value: neighbouring lanes neighbouring words of a
// row, so the rows' side and the key codes are contiguous, and the four value words,
// which lie side by side in the pool, are one 16-byte access where the rows' slots
// follow each other from a multiple of four. The four lanes of a group find its maximum
// with two lane exchanges. 16001 rows of 8 heads x 128 written and 20097 gathered (187
// MB): 62.7 us with a thread per word and row, which spent it on 64-bit divisions and
// 4-byte value accesses; 38.3 with this, 4.9 TB/s, what a large copy reaches.
#include <climits>

#include "kv4.h"

namespace mf {
namespace {

struct Cache4Args {
    const char* k_rows;
    const char* v_rows;
    int64_t row_st, row_sh;  // elements
    uint32_t* kc;
    uint8_t* ks;
    uint32_t* vc;
    uint8_t* vs;
    const int64_t* slots;
    int64_t num_tokens, num_slots;
    int bs, heads;
    int word_bits;  // log2 of a row's words
    int lo, hi;     // bounds of a scale byte
};

// Eight elements from p; VEC: p is 16-byte aligned.
template <int DT, bool VEC>
__device__ __forceinline__ void load8(const char* p, float (&x)[8]) {
    constexpr int ES = DT == MF_F32 ? 4 : 2;
    if constexpr (VEC) {
        uint4 w[ES / 2];
#pragma unroll
        for (int k = 0; k < ES / 2; ++k) w[k] = *(const uint4*)(p + 16 * k);
        const uint32_t* u = (const uint32_t*)w;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if constexpr (ES == 4) x[e] = __uint_as_float(u[e]);
            else x[e] = bits_to_f32<DT>((u[e >> 1] >> (16 * (e & 1))) & 0xffffu);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if constexpr (ES == 4) x[e] = *(const float*)(p + 4 * e);
            else x[e] = bits_to_f32<DT>(*(const uint16_t*)(p + 2 * e));
        }
    }
}
template <int DT, bool VEC>
__device__ __forceinline__ void store8(char* p, const float (&x)[8]) {
    constexpr int ES = DT == MF_F32 ? 4 : 2;
    if constexpr (VEC) {
        uint32_t u[2 * ES];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if constexpr (ES == 4) u[e] = __float_as_uint(x[e]);
            else u[e >> 1] = (e & 1) ? u[e >> 1] | (f32_to_bits<DT>(x[e]) << 16) : f32_to_bits<DT>(x[e]);
        }
#pragma unroll
        for (int k = 0; k < ES / 2; ++k)
            *(uint4*)(p + 16 * k) = make_uint4(u[4 * k], u[4 * k + 1], u[4 * k + 2], u[4 * k + 3]);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if constexpr (ES == 4) *(float*)(p + 4 * e) = x[e];
            else *(uint16_t*)(p + 2 * e) = (uint16_t)f32_to_bits<DT>(x[e]);
        }
    }
}

// This lane's eight codes and its group's scale byte; the group's other elements
// are in the lanes that differ in the two low bits of `lane`.
__device__ __forceinline__ uint32_t encode8(const float (&x)[8], int lo, int hi, uint32_t& byte) {
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
    top = max(top, (uint32_t)__shfl_xor((int)top, 1, 64));
    top = max(top, (uint32_t)__shfl_xor((int)top, 2, 64));
    if (top >= 0x7f800000u) {
        byte = kNaNScale4;
        return 0u;
    }
    // the exponent, carried over where the mantissa is above 1.75
    byte = (uint32_t)min(max((int)((top + 0x1fffffu) >> 23) - 2, lo), hi);
    const float s = scale4(byte);
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], s, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], s, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], s, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], s, 3);
    return w;
}

__device__ __forceinline__ void decode8(uint32_t w, uint32_t byte, float (&x)[8]) {
    const float s = scale4(byte);
    const uint4 v = octet4<MF_BF16>(w, s);  // bf16 holds every value exactly
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = bf16_bits_to_f32((u[e >> 1] >> (16 * (e & 1))) & 0xffffu);
}

// A lane's place: word c of rows t0 .. t0 + 3 of head h. A wave covers the 64 / words
// of four rows of one head that its lanes hold; a workgroup's waves take four heads.
struct Place {
    int h, c;
    int64_t t0;
    int64_t slot[4];  // -1: no such row, or its slot lies outside the pool
    bool any, run;    // some row exists; all four, in slots that follow each other from a multiple of four
};
__device__ __forceinline__ bool find_place(const Cache4Args& a, Place& p) {
    const int lane = threadIdx.x & 63;
    p.h = (int)blockIdx.y * 4 + (int)(threadIdx.x >> 6);
    if (p.h >= a.heads) return false;
    p.c = lane & ((1 << a.word_bits) - 1);
    p.t0 = ((int64_t)blockIdx.x * (64 >> a.word_bits) + (lane >> a.word_bits)) * 4;
    p.any = false;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int64_t s = p.t0 + k < a.num_tokens ? a.slots[p.t0 + k] : -1;
        p.slot[k] = s >= 0 && s < a.num_slots ? s : -1;
        p.any |= p.slot[k] >= 0;
    }
    p.run = p.slot[0] >= 0 && (p.slot[0] & 3) == 0;
#pragma unroll
    for (int k = 1; k < 4; ++k) p.run = p.run && p.slot[k] == p.slot[0] + k;
    return p.any;  // the same in a group's four lanes
}
// Row (block, head) and slot in the block of pool slot s. Slots of one layer fit 31
// bits but for pools of more than 2^31 tokens.
__device__ __forceinline__ void slot_place(const Cache4Args& a, int64_t s, int h, int64_t& row, int& off) {
    const int64_t blk = s < (1ll << 31) ? (int64_t)((uint32_t)s / (uint32_t)a.bs) : s / a.bs;
    off = (int)(s - blk * a.bs);
    row = blk * a.heads + h;
}

template <int DT, bool VEC>
__global__ __launch_bounds__(256) void kv4_write_kernel(Cache4Args a) {
    constexpr int ES = DT == MF_F32 ? 4 : 2;
    Place p;
    if (!find_place(a, p)) return;
    const int words = 1 << a.word_bits, groups = words >> 2;
    const int64_t src = (p.t0 * a.row_st + (int64_t)p.h * a.row_sh + p.c * 8) * ES;
    float k[4][8], v[4][8];
    const int some = p.slot[0] >= 0 ? 0 : p.slot[1] >= 0 ? 1 : p.slot[2] >= 0 ? 2 : 3;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        // in the place of a row that is not written, one that is
        const int64_t at = src + (int64_t)(p.slot[i] >= 0 ? i : some) * a.row_st * ES;
        load8<DT, VEC>(a.k_rows + at, k[i]);
        load8<DT, VEC>(a.v_rows + at, v[i]);
    }
    uint32_t vw[4], vb[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t byte;
        const uint32_t w = encode8(k[i], a.lo, a.hi, byte);
        vw[i] = encode8(v[i], a.lo, a.hi, vb[i]);
        if (p.slot[i] < 0) continue;
        int64_t row;
        int off;
        slot_place(a, p.slot[i], p.h, row, off);
        a.kc[((row * a.bs + off) << a.word_bits) + p.c] = w;
        if ((p.c & 3) == 0) a.ks[(row * a.bs + off) * groups + (p.c >> 2)] = (uint8_t)byte;
        if (!p.run) {
            a.vc[((row << a.word_bits) + p.c) * a.bs + off] = vw[i];
            if ((p.c & 3) == 0) a.vs[(row * groups + (p.c >> 2)) * a.bs + off] = (uint8_t)vb[i];
        }
    }
    if (p.run) {
        int64_t row;
        int off;
        slot_place(a, p.slot[0], p.h, row, off);
        *(uint4*)(a.vc + ((row << a.word_bits) + p.c) * a.bs + off) = make_uint4(vw[0], vw[1], vw[2], vw[3]);
        if ((p.c & 3) == 0)
            *(uint32_t*)(a.vs + (row * groups + (p.c >> 2)) * a.bs + off) =
                vb[0] | (vb[1] << 8) | (vb[2] << 16) | (vb[3] << 24);
    }
}

template <int DT, bool VEC>
__global__ __launch_bounds__(256) void kv4_gather_kernel(Cache4Args a) {
    constexpr int ES = DT == MF_F32 ? 4 : 2;
    Place p;
    if (!find_place(a, p)) return;
    const int words = 1 << a.word_bits, groups = words >> 2;
    const int64_t dst = (p.t0 * a.row_st + (int64_t)p.h * a.row_sh + p.c * 8) * ES;
    uint32_t kw[4] = {}, kb[4] = {}, vw[4] = {}, vb[4] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (p.slot[i] < 0) continue;
        int64_t row;
        int off;
        slot_place(a, p.slot[i], p.h, row, off);
        kw[i] = a.kc[((row * a.bs + off) << a.word_bits) + p.c];
        kb[i] = a.ks[(row * a.bs + off) * groups + (p.c >> 2)];
        const uint32_t* vc = a.vc + ((row << a.word_bits) + p.c) * a.bs + off;
        const uint8_t* vs = a.vs + (row * groups + (p.c >> 2)) * a.bs + off;
        if (!p.run) {
            vw[i] = *vc;
            vb[i] = *vs;
        } else if (i == 0) {
            const uint4 w = *(const uint4*)vc;
            const uint32_t b = *(const uint32_t*)vs;
            vw[0] = w.x; vw[1] = w.y; vw[2] = w.z; vw[3] = w.w;
            vb[0] = b & 255u; vb[1] = (b >> 8) & 255u; vb[2] = (b >> 16) & 255u; vb[3] = b >> 24;
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (p.slot[i] < 0) continue;
        float x[8];
        decode8(kw[i], kb[i], x);
        store8<DT, VEC>((char*)a.k_rows + dst + (int64_t)i * a.row_st * ES, x);
        decode8(vw[i], vb[i], x);
        store8<DT, VEC>((char*)a.v_rows + dst + (int64_t)i * a.row_st * ES, x);
    }
}

template <bool GATHER>
int launch_cache4(const void* k, const void* v, int dtype, int64_t st, int64_t sh, const int64_t* slots, int64_t n,
                  const mf_pool4* p, hipStream_t stream) {
    if (int e = check_pool4(p)) return e;
    if (!dtype_ok(dtype) || n < 0) return MF_ERR_ARG;
    if (n == 0) return MF_OK;
    if (!k || !v || !slots) return MF_ERR_ARG;
    Cache4Args a{(const char*)k, (const char*)v, st, sh, p->key_codes, p->key_scales, p->value_codes, p->value_scales,
                 slots, n, p->num_blocks * p->block_size, p->block_size, p->num_heads,
                 __builtin_ctz(p->head_dim / 8), min_scale4(p->dtype), max_scale4(p->dtype)};
    const int64_t rows = 4 * (64 / (p->head_dim / 8));  // of a wave
    const int64_t blocks = (n + rows - 1) / rows;
    if (blocks > INT_MAX || p->num_heads > 4 * 65535) return MF_ERR_ARG;
    const dim3 grid((unsigned)blocks, (unsigned)((p->num_heads + 3) / 4));
    const int es = dtype_size(dtype);
    const bool vec = ((((uintptr_t)k | (uintptr_t)v) & 15) == 0) && (st * es) % 16 == 0 && (sh * es) % 16 == 0;
#define MF_CACHE4(DT)                                                                                       \
    if (dtype == DT) {                                                                                      \
        if constexpr (GATHER) {                                                                             \
            if (vec) hipLaunchKernelGGL((kv4_gather_kernel<DT, true>), grid, dim3(256), 0, stream, a);      \
            else hipLaunchKernelGGL((kv4_gather_kernel<DT, false>), grid, dim3(256), 0, stream, a);         \
        } else {                                                                                            \
            if (vec) hipLaunchKernelGGL((kv4_write_kernel<DT, true>), grid, dim3(256), 0, stream, a);       \
            else hipLaunchKernelGGL((kv4_write_kernel<DT, false>), grid, dim3(256), 0, stream, a);          \
        }                                                                                                   \
    }
    MF_CACHE4(MF_F32)
    MF_CACHE4(MF_F16)
    MF_CACHE4(MF_BF16)
#undef MF_CACHE4
    return check_launch();
}

}  // namespace
}  // namespace mf

extern "C" int mf_kv4_write(const void* k_src, const void* v_src, int src_dtype, int64_t src_stride_t,
                            int64_t src_stride_h, const int64_t* slot_mapping, int64_t num_tokens,
                            const mf_pool4* pool, mf_stream_t stream) {
    return mf::launch_cache4<false>(k_src, v_src, src_dtype, src_stride_t, src_stride_h, slot_mapping, num_tokens, pool,
                                    (hipStream_t)stream);
}

extern "C" int mf_kv4_gather(const mf_pool4* pool, const int64_t* slot_mapping, int64_t num_tokens, void* k_dst,
                             void* v_dst, int dst_dtype, int64_t dst_stride_t, int64_t dst_stride_h,
                             mf_stream_t stream) {
    return mf::launch_cache4<true>(k_dst, v_dst, dst_dtype, dst_stride_t, dst_stride_h, slot_mapping, num_tokens, pool,
                                   (hipStream_t)stream);
}
