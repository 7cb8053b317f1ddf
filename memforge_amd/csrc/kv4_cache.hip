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
// Both kernels are bound by the bytes they move. One thread handles eight elements
// (a word of codes) of a row's key and value; the four lanes of a group find its
// maximum with two lane exchanges.
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
    int bs, heads, dim;
    int lo, hi;  // bounds of a scale byte
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

template <int DT, bool VEC>
__global__ __launch_bounds__(256) void kv4_write_kernel(Cache4Args a) {
    constexpr int ES = DT == MF_F32 ? 4 : 2;
    const int chunks = a.dim / 8;
    const int64_t per_tok = (int64_t)a.heads * chunks;
    const int64_t total = a.num_tokens * per_tok;  // a multiple of four: a group's lanes leave together
    for (int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x; idx < total; idx += (int64_t)gridDim.x * 256) {
        const int64_t t = idx / per_tok;
        const int rem = (int)(idx - t * per_tok);
        const int h = rem / chunks, c = rem - h * chunks;
        const int64_t slot = a.slots[t];
        if (slot < 0 || slot >= a.num_slots) continue;
        const int64_t src = (t * a.row_st + (int64_t)h * a.row_sh + c * 8) * ES;
        const int64_t blk = slot / a.bs;
        const int off = (int)(slot - blk * a.bs);
        const int64_t row = blk * a.heads + h;
        float x[8];
        uint32_t byte;
        load8<DT, VEC>(a.k_rows + src, x);
        uint32_t w = encode8(x, a.lo, a.hi, byte);
        a.kc[(row * a.bs + off) * chunks + c] = w;
        if ((c & 3) == 0) a.ks[(row * a.bs + off) * (chunks / 4) + c / 4] = (uint8_t)byte;
        load8<DT, VEC>(a.v_rows + src, x);
        w = encode8(x, a.lo, a.hi, byte);
        a.vc[(row * chunks + c) * a.bs + off] = w;
        if ((c & 3) == 0) a.vs[(row * (chunks / 4) + c / 4) * a.bs + off] = (uint8_t)byte;
    }
}

template <int DT, bool VEC>
__global__ __launch_bounds__(256) void kv4_gather_kernel(Cache4Args a) {
    constexpr int ES = DT == MF_F32 ? 4 : 2;
    const int chunks = a.dim / 8;
    const int64_t per_tok = (int64_t)a.heads * chunks;
    const int64_t total = a.num_tokens * per_tok;
    for (int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x; idx < total; idx += (int64_t)gridDim.x * 256) {
        const int64_t t = idx / per_tok;
        const int rem = (int)(idx - t * per_tok);
        const int h = rem / chunks, c = rem - h * chunks;
        const int64_t slot = a.slots[t];
        if (slot < 0 || slot >= a.num_slots) continue;
        const int64_t dst = (t * a.row_st + (int64_t)h * a.row_sh + c * 8) * ES;
        const int64_t blk = slot / a.bs;
        const int off = (int)(slot - blk * a.bs);
        const int64_t row = blk * a.heads + h;
        float x[8];
        decode8(a.kc[(row * a.bs + off) * chunks + c], a.ks[(row * a.bs + off) * (chunks / 4) + c / 4], x);
        store8<DT, VEC>((char*)a.k_rows + dst, x);
        decode8(a.vc[(row * chunks + c) * a.bs + off], a.vs[(row * (chunks / 4) + c / 4) * a.bs + off], x);
        store8<DT, VEC>((char*)a.v_rows + dst, x);
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
                 slots, n, p->num_blocks * p->block_size, p->block_size, p->num_heads, p->head_dim,
                 min_scale4(p->dtype), max_scale4(p->dtype)};
    const int64_t total = n * p->num_heads * (p->head_dim / 8);
    const int64_t blocks = (total + 255) / 256;
    const dim3 grid((unsigned)(blocks < (1 << 20) ? blocks : (1 << 20)));
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
