// Device helpers of the paged 8- and 16-bit cache: conversions between held codes, f32 and bf16.
#pragma once
#include "device_utils.hpp"
#include "kv_index.hpp"

namespace qtts {

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));  // register arrays of HIP's uint4 end in scratch memory

// biased exponent of a block's scale from the largest |x| (as bits): see KvFormat.  448 = 1.75 2^8 and 127 = 1.984375 2^6.
template <int FMT>
__device__ __forceinline__ int kv_scale_exp(unsigned amax_bits) {
    constexpr int TOP_EXP = FMT == KV_E4M3 ? 8 : 6;
    constexpr unsigned TOP_FRAC = FMT == KV_E4M3 ? 0x600000u : 0x7e0000u;
    const int e = (int)(amax_bits >> 23) - TOP_EXP + ((amax_bits & 0x7fffffu) > TOP_FRAC ? 1 : 0);
    return max(e, KV_MIN_EXP + 127);
}
// four f32 -> four codes; inv = 2^-e
template <int FMT>
__device__ __forceinline__ unsigned kv_encode4(const float* x, float inv) {
    if constexpr (FMT == KV_E4M3) {
        int r = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * inv, x[1] * inv, 0, false);
        return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(x[2] * inv, x[3] * inv, r, true);
    } else {
        unsigned r = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) r |= ((unsigned)(int)__builtin_rintf(x[i] * inv) & 0xffu) << (8 * i);
        return r;
    }
}
// What a block with an infinity or a NaN holds, so that every element reads back as NaN: e4m3 has a NaN of its own; int8 codes are 0
// under the biased exponent 255, which as a scale is infinity, and 0 * infinity is NaN.
template <int FMT>
__device__ __forceinline__ unsigned kv_bad_codes() { return FMT == KV_E4M3 ? 0x7f7f7f7fu : 0u; }
template <int FMT>
__device__ __forceinline__ int kv_bad_exp() { return FMT == KV_E4M3 ? 127 : 255; }

__device__ __forceinline__ float kv_scale(unsigned biased) { return __uint_as_float(biased << 23); }

// four codes -> f32 values
template <int FMT>
__device__ __forceinline__ void kv_decode4(unsigned c, float scale, float* o) {
    if constexpr (FMT == KV_E4M3) {
        o[0] = __builtin_amdgcn_cvt_f32_fp8((int)c, 0) * scale;
        o[1] = __builtin_amdgcn_cvt_f32_fp8((int)c, 1) * scale;
        o[2] = __builtin_amdgcn_cvt_f32_fp8((int)c, 2) * scale;
        o[3] = __builtin_amdgcn_cvt_f32_fp8((int)c, 3) * scale;
    } else {
        // the four codes stay one register until here: the compiler would carry them around the callers' loops as separate bytes
        asm("" : "+v"(c));
        // written with byte casts: the compiler takes a byte out, extends its sign and converts it in one instruction
        o[0] = (float)(signed char)(c & 0xffu) * scale;
        o[1] = (float)(signed char)((c >> 8) & 0xffu) * scale;
        o[2] = (float)(signed char)((c >> 16) & 0xffu) * scale;
        o[3] = (float)(signed char)(c >> 24) * scale;
    }
}
__device__ __forceinline__ unsigned pack_bf16(float a, float b) {  // one conversion for both (round to nearest even)
    typedef float f32x2_t __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2_t{a, b}, bf16x2_t));
}
// eight codes -> eight bf16 in operand order, exact (see KvFormat)
template <int FMT>
__device__ __forceinline__ u32x4_t kv_decode8(unsigned c0, unsigned c1, float scale) {
    if constexpr (FMT == KV_E4M3) {  // one instruction converts, scales and packs two codes
        const auto two = [&](bf16x2_t v) { return __builtin_bit_cast(unsigned, v); };
        return u32x4_t{two(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c0, scale, false)), two(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c0, scale, true)),
                       two(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c1, scale, false)), two(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c1, scale, true))};
    } else {
        float f[8];
        kv_decode4<FMT>(c0, scale, f);
        kv_decode4<FMT>(c1, scale, f + 4);
        return u32x4_t{pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7])};
    }
}

}  // namespace qtts
