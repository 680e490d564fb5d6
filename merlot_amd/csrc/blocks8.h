// 8-bit float blocks: 128 values along the reduction share one power-of-two scale, stored as its biased exponent (a byte b stands for 2^(b - 127), 255 for NaN).
// A power of two because (a) the gfx950 matrix instruction takes exactly that beside its 8-bit operands -- the product needs no vector work and no second set
// of accumulators for the scales --, and (b) dividing by it is exact: ONE rounding stands between a value and its 8-bit copy, and the copy's values are bf16 values.
#pragma once
#include "common.h"

constexpr int E4M3_TOP = 8, E5M2_TOP = 15;               // the format's largest value is 1.75 * 2^TOP (448, 57 344)

// bits of a block's max |v| -> scale byte: the least e with max |v| <= 1.75 * 2^(TOP + e).  Not finite: 255.  All zeros: 2^0.  e is at least -127.
__device__ __forceinline__ int block_scale_byte(uint32_t amax_bits, int top) {
    if (amax_bits > 0x7f7fffffu) return 255;
    const int e = (int)(amax_bits >> 23) - 127 - top + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return amax_bits == 0u ? 127 : max(e + 127, 0);
}
// 2^-e of a scale byte, exactly (bytes 0 ... 247 of finite blocks: the result's own exponent field is 254 - byte)
__device__ __forceinline__ float block_inverse(int byte) { return __uint_as_float((uint32_t)(254 - byte) << 23); }

// max over each aligned group of G lanes (G = 16 or 32): rotations inside rows of 16 lanes (data-parallel primitives, no LDS), one exchange between two rows
template <int G>
__device__ __forceinline__ uint32_t group_umax(uint32_t m) {
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x128, 0xf, 0xf, true));      // row_ror:8
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x124, 0xf, 0xf, true));      // row_ror:4
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x122, 0xf, 0xf, true));      // row_ror:2
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x121, 0xf, 0xf, true));      // row_ror:1
    if constexpr (G == 32) m = max(m, (uint32_t)__shfl_xor((int)m, 16, 64));
    return m;
}

// four fp32 values -> four codes (nearest, ties to even), FMT 0 = e4m3, 1 = e5m2
template <int FMT>
__device__ __forceinline__ uint32_t pack_codes(float a, float b, float c, float d) {
    int w = 0;
    if constexpr (FMT == 0) {
        w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, w, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
    } else {
        w = __builtin_amdgcn_cvt_pk_bf8_f32(a, b, w, false);
        w = __builtin_amdgcn_cvt_pk_bf8_f32(c, d, w, true);
    }
    return (uint32_t)w;
}

// the codes of VEC values under their block's scale byte; a block that is not finite becomes NaN as a whole (a code that cannot be mistaken for a number)
template <int FMT, int VEC>
__device__ __forceinline__ void store_codes(uint8_t* p, const float (&v)[VEC], int byte) {
    const float inv = block_inverse(byte == 255 ? 254 : byte);
    uint32_t w[VEC / 4];
#pragma unroll
    for (int k = 0; k < VEC / 4; ++k)
        w[k] = byte == 255 ? 0x7f7f7f7fu : pack_codes<FMT>(v[4 * k] * inv, v[4 * k + 1] * inv, v[4 * k + 2] * inv, v[4 * k + 3] * inv);
    if constexpr (VEC == 8) *reinterpret_cast<u32x2*>(p) = u32x2{w[0], w[1]};
    else *reinterpret_cast<uint32_t*>(p) = w[0];
}
