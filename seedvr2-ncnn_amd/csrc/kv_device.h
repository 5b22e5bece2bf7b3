// Device helpers of the key/value cache kernels (gfx950): 4-bit rows.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace awa
{
namespace dev
{

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

// The power of two behind a scale byte: 2^(byte - 127); 255 stands for NaN.
__device__ __forceinline__ float four_unit(unsigned byte)
{
    const unsigned b = byte == 0u ? 0x00400000u : byte << 23;
    return __uint_as_float(byte == 255u ? 0x7fc00000u : b);
}

// The eight values of a word of codes.
__device__ __forceinline__ void four_values(unsigned word, float unit, float (&v)[8])
{
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, 1.f, 0);
    const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, 1.f, 1);
    const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, 1.f, 2);
    const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, 1.f, 3);
    v[0] = a[0] * unit, v[1] = a[1] * unit, v[2] = b[0] * unit, v[3] = b[1] * unit;
    v[4] = c[0] * unit, v[5] = c[1] * unit, v[6] = d[0] * unit, v[7] = d[1] * unit;
}

// The same as bf16, of which every such value is one.
__device__ __forceinline__ uint4 four_bf16(unsigned word, float unit)
{
    return make_uint4(__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, unit, 0)),
                      __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, unit, 1)),
                      __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, unit, 2)),
                      __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, unit, 3)));
}

} // namespace dev
} // namespace awa
