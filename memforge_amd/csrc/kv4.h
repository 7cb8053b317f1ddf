// The 4-bit pool (mf_pool4): e2m1 codes, one e8m0 scale byte for 32 elements of a
// token's head (the OCP microscaling format), and gfx950's conversions.
#pragma once

#include "mf_common.h"

namespace mf {

constexpr int kGroup4 = 32;  // elements of one scale

// Scale bytes of a pool whose attention runs in `dtype`: every value a code can
// stand for, 0.5 to 6 times the scale, is then a normal number of that type (fp16:
// at least a subnormal one that it holds exactly), and finite.
inline int min_scale4(int dtype) { return dtype == MF_F16 ? 127 - 23 : 127 - 125; }
inline int max_scale4(int dtype) { return dtype == MF_F16 ? 127 + 13 : 127 + 125; }
constexpr int kNaNScale4 = 255;

// The scale a byte stands for, as the operand of the conversions (255 makes every code
// NaN). They read bits 30 to 23 alone, whatever stands in the others (checked over
// random words).
__device__ __forceinline__ float scale4(uint32_t byte) { return __uint_as_float(byte << 23); }

// Byte B of w, two codes, as two elements of the 16-bit type: one instruction, the
// scale applied, exact (checked over all codes and scale bytes).
template <int DT, int B>
__device__ __forceinline__ uint32_t pair4(uint32_t w, float scale) {
    if constexpr (DT == MF_BF16)
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, B));
    else
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, B));
}
// All eight codes of w.
template <int DT>
__device__ __forceinline__ uint4 octet4(uint32_t w, float scale) {
    return make_uint4(pair4<DT, 0>(w, scale), pair4<DT, 1>(w, scale), pair4<DT, 2>(w, scale), pair4<DT, 3>(w, scale));
}

// What mf_pool4 must satisfy; MF_OK or a status.
inline int check_pool4(const mf_pool4* p) {
    if (!p || !p->key_codes || !p->key_scales || !p->value_codes || !p->value_scales) return MF_ERR_ARG;
    if (p->num_blocks <= 0 || p->num_heads <= 0 || p->block_size <= 0 || p->block_size % 16 || p->block_size > 512)
        return MF_ERR_ARG;
    if (!dtype_ok(p->dtype)) return MF_ERR_ARG;
    if (p->head_dim != 32 && p->head_dim != 64 && p->head_dim != 128 && p->head_dim != 256) return MF_ERR_UNSUPPORTED;
    if (((uintptr_t)p->key_codes | (uintptr_t)p->value_codes) & 15) return MF_ERR_ARG;
    if (((uintptr_t)p->key_scales | (uintptr_t)p->value_scales) & 3) return MF_ERR_ARG;
    return MF_OK;
}

}  // namespace mf
