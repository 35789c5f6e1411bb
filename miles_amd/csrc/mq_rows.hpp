// Row access shared by the norm kernels and the linear layers' epilogues: elements of any of the three types as floats, sums
// over lanes, and the 8-bit copies (e4m3 codes, one E8M0 exponent byte per 32 columns) that stand for an activation.
#pragma once
#include "mq_api_internal.hpp"
#include "mq_common.hpp"

namespace mq {

// elements of one 16-byte access
template <int D>
constexpr int kVec = D == MQ_F32 ? 4 : 8;
template <int D>
constexpr int kElem = D == MQ_F32 ? 4 : 2;

template <int D>
__device__ __forceinline__ float one_elem(const void* p, int64_t i) { return load_f32(p, i, D); }

// kVec elements as floats
template <int D>
__device__ __forceinline__ void unpack(u32x4 v, float* f) {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (D == MQ_F32) f[i] = u2f(u[i]);
        else {
            f[2 * i] = elem_lo<D == MQ_F16>(u[i]);
            f[2 * i + 1] = elem_hi<D == MQ_F16>(u[i]);
        }
    }
}
// two floats as two 16-bit elements, rounded to nearest even
template <int D>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if (D == MQ_F16) {
        const _Float16 x = (_Float16)a, y = (_Float16)b;
        return (uint32_t)__builtin_bit_cast(uint16_t, x) | ((uint32_t)__builtin_bit_cast(uint16_t, y) << 16);
    }
    return hw_bf16x2(a, b);
}
template <int D>
__device__ __forceinline__ u32x4 pack(const float* f) {
    if (D == MQ_F32) return u32x4{f2u(f[0]), f2u(f[1]), f2u(f[2]), f2u(f[3])};
    return u32x4{pack2<D>(f[0], f[1]), pack2<D>(f[2], f[3]), pack2<D>(f[4], f[5]), pack2<D>(f[6], f[7])};
}
// the kVec elements of a row from column c on, zero from column n on
template <int D>
__device__ __forceinline__ u32x4 ld_row(const void* row, int64_t c, int64_t n) {
    constexpr int V = kVec<D>;
    if (c + V <= n) return ld16_at2((const char*)row + c * kElem<D>);
    u32x4 v = {0u, 0u, 0u, 0u};
    if (c < n) {
        uint32_t u[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int j = 0; j < V; j++) {
            if (c + j < n) {
                if (D == MQ_F32) u[j & 3] = ((const uint32_t*)row)[c + j];
                else u[j / 2] |= (uint32_t)((const uint16_t*)row)[c + j] << (16 * (j & 1));
            }
        }
        v = u32x4{u[0], u[1], u[2], u[3]};
    }
    return v;
}
template <int D>
__device__ __forceinline__ void st_row(void* row, int64_t c, int64_t n, u32x4 v) {
    constexpr int V = kVec<D>;
    if (c + V <= n) {
        st16_at2((char*)row + c * kElem<D>, v);
        return;
    }
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < V; j++) {
        if (c + j < n) {
            if (D == MQ_F32) ((uint32_t*)row)[c + j] = u[j & 3];
            else ((uint16_t*)row)[c + j] = (uint16_t)(u[j / 2] >> (16 * (j & 1)));
        }
    }
}

// ---- sums over lanes ---------------------------------------------------------------------------------------------------
template <int CTRL>
__device__ __forceinline__ float dpp_f32(float v) { return u2f(dpp_u32<CTRL>(f2u(v))); }
// the same order of additions in every lane, so that a result does not depend on which lane reads it
__device__ __forceinline__ float wave_sum(float v) {
    v += dpp_f32<kDppQuadXor1>(v);
    v += dpp_f32<kDppQuadXor2>(v);
    v += dpp_f32<kDppRowHalfMirror>(v);
    v += dpp_f32<kDppRowMirror>(v);
    const float a = u2f((uint32_t)__builtin_amdgcn_readlane((int)f2u(v), 0)), b = u2f((uint32_t)__builtin_amdgcn_readlane((int)f2u(v), 16));
    const float c = u2f((uint32_t)__builtin_amdgcn_readlane((int)f2u(v), 32)), d = u2f((uint32_t)__builtin_amdgcn_readlane((int)f2u(v), 48));
    return (a + b) + (c + d);
}

// ---- 8-bit copies --------------------------------------------------------------------------------------------------------
// 2^(e - 127)
__device__ __forceinline__ float e8m0_value(uint32_t e) { return e ? u2f(e == 255 ? 0x7FC00000u : e << 23) : u2f(0x00400000u); }
// The larger of a running maximum and a magnitude; a NaN has no part in it (the arithmetic of mxfp8_quantize).
__device__ __forceinline__ float keep_larger(float m, float v) { return __builtin_fmaxf(m, __builtin_fabsf(v)); }
// Four values over their group's power of two, which leaves none above 448 but an infinity, in a group whose maximum is one
// (infinite != 0): that becomes 448.  A NaN goes through.
__device__ __forceinline__ uint32_t keep_codes4(float a, float b, float c, float d, float inv, bool infinite) {
    if (infinite)
        return hw_e4m3x4(clamp_keep_nan(a * inv, -kFp8Max, kFp8Max), clamp_keep_nan(b * inv, -kFp8Max, kFp8Max),
                         clamp_keep_nan(c * inv, -kFp8Max, kFp8Max), clamp_keep_nan(d * inv, -kFp8Max, kFp8Max));
    return hw_e4m3x4(a * inv, b * inv, c * inv, d * inv);
}
constexpr uint32_t kInfinity = 0x7F800000u;
__device__ __forceinline__ uint32_t keep_exponent(uint32_t group_magnitude) { return e8m0_ceil(u2f(group_magnitude) * u2f(0x3B124925u)); }
// four codes as floats: exact, a power of two away from three bits of mantissa
__device__ __forceinline__ void kept_values4(uint32_t codes, float scale, float* f) {
    const f32x2 lo = hw_e4m3x2_decode<false>(codes), hi = hw_e4m3x2_decode<true>(codes);
    f[0] = lo.x * scale;
    f[1] = lo.y * scale;
    f[2] = hi.x * scale;
    f[3] = hi.y * scale;
}

// The same as four 16-bit values, two to an instruction: equal to the product rounded once for every code and every exponent
// (all 256 x 255 compared on the device by the dequantizer's test and the weight gradient's), except that in fp16 a finite value
// above 65504, a code of 256 and more in a group whose maximum lies close below that, becomes 65504.
template <int D>
__device__ __forceinline__ u32x2 kept_pack4(uint32_t codes, uint32_t e) {
    const float s = e8m0_value(e);
    if (D == MQ_F16) {
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
        if (e >= 127 + 8) {
            float f[4];
            kept_values4(codes, s, f);
#pragma unroll
            for (int i = 0; i < 4; i++) f[i] = clamp_keep_nan(f[i], -65504.0f, 65504.0f);
            return u32x2{pack2<D>(f[0], f[1]), pack2<D>(f[2], f[3])};
        }
        const f16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, s, false), hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, s, true);
        return u32x2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
    }
    const bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, s, false), hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, s, true);
    return u32x2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
}

}  // namespace mq
