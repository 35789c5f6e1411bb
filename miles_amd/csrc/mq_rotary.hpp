// Rotary positions: pairs of a vector's elements turned by position x inv_freq, shared by the operator of that name and by the paged cache,
// which rotates keys and queries on the way.
//
//   angle = position inv_freq, c = fl32(scale cos(angle)), s = fl32(scale sin(angle)), (a, b) -> (a c - b s, b c + a s)
//
// Angle, cosine and sine are computed in 64 bits: at position 10^6 an angle of 32 bits is off by 0.03 of a radian.  One rounding makes c and
// s, and products and sums are rounded one by one (no fused operation), so that a result is what the same expression on tensors gives.
#pragma once
#include "mq_rows.hpp"

namespace mq {

typedef float f32x2_t __attribute__((ext_vector_type(2)));

// cos and sin of x, |x| < 2^50 or so: x less the nearest multiple n of pi/2, which two 53-bit pieces of pi/2 give to 2^-53 of
// a radian while n < 2^52, then the Taylor series on [-pi/4, pi/4], whose first terms left out are (pi/4)^17 / 17! = 5e-17 and
// (pi/4)^18 / 18! = 2e-18.  Some 30 operations of 64 bits, at the rate of 32-bit ones here, for each pair and token, not for each head.
__device__ __forceinline__ void cos_sin(double x, double& c, double& s) {
    const double n = __builtin_rint(x * 0.63661977236758134308);                  // 2 / pi
    const double r = __builtin_fma(-n, 6.1232339957367659e-17, __builtin_fma(-n, 1.5707963267948966, x));
    const double z = r * r;
    double p = -1.0 / 1307674368000.0;                                           // 15!
    p = __builtin_fma(p, z, 1.0 / 6227020800.0);
    p = __builtin_fma(p, z, -1.0 / 39916800.0);
    p = __builtin_fma(p, z, 1.0 / 362880.0);
    p = __builtin_fma(p, z, -1.0 / 5040.0);
    p = __builtin_fma(p, z, 1.0 / 120.0);
    p = __builtin_fma(p, z, -1.0 / 6.0);
    const double sine = __builtin_fma(p * z, r, r);
    double q = 1.0 / 20922789888000.0;                                           // 16!
    q = __builtin_fma(q, z, -1.0 / 87178291200.0);
    q = __builtin_fma(q, z, 1.0 / 479001600.0);
    q = __builtin_fma(q, z, -1.0 / 3628800.0);
    q = __builtin_fma(q, z, 1.0 / 40320.0);
    q = __builtin_fma(q, z, -1.0 / 720.0);
    q = __builtin_fma(q, z, 1.0 / 24.0);
    q = __builtin_fma(q, z, -0.5);
    const double cosine = __builtin_fma(q, z, 1.0);
    // n modulo 4, also where n has no 32 bits
    const int quarter = (int)(n - 4.0 * __builtin_floor(n * 0.25));
    const double u = quarter & 1 ? sine : cosine, v = quarter & 1 ? cosine : sine;
    c = quarter == 1 || quarter == 2 ? -u : u;
    s = quarter & 2 ? -v : v;
}

struct RotaryTurn {
    const void* positions;           // int32 or int64
    const void* inv_freq;            // [pairs] fp32 or fp64
    double scale;
    int pairs, positions64, freq64, back;
};
__device__ __forceinline__ int64_t index_at(const void* p, int64_t i, int is64) { return is64 ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i]; }
__device__ __forceinline__ f32x2_t turn_of(const RotaryTurn& a, int64_t position, int pair) {
    const double f = a.freq64 ? ((const double*)a.inv_freq)[pair] : (double)((const float*)a.inv_freq)[pair];
    double c, s;
    cos_sin((double)position * f, c, s);
    const float sine = (float)(s * a.scale);
    return f32x2_t{(float)(c * a.scale), a.back ? -sine : sine};
}

// The elements of one 16-byte access, as pairs: halves a and b of the vector (INTER 0), or neighbours (INTER 1)
template <int D>
__device__ __forceinline__ void turn_halves(u32x4& a, u32x4& b, const f32x2_t* cs) {
    constexpr int V = kVec<D>;
    float x[V], y[V], u[V], w[V];
    unpack<D>(a, x);
    unpack<D>(b, y);
#pragma unroll
    for (int i = 0; i < V; i++) {
        u[i] = x[i] * cs[i].x - y[i] * cs[i].y;
        w[i] = y[i] * cs[i].x + x[i] * cs[i].y;
    }
    a = pack<D>(u);
    b = pack<D>(w);
}
template <int D>
__device__ __forceinline__ void turn_neighbours(u32x4& a, const f32x2_t* cs) {
    constexpr int V = kVec<D>;
    float x[V], u[V];
    unpack<D>(a, x);
#pragma unroll
    for (int i = 0; i < V; i += 2) {
        u[i] = x[i] * cs[i / 2].x - x[i + 1] * cs[i / 2].y;
        u[i + 1] = x[i + 1] * cs[i / 2].x + x[i] * cs[i / 2].y;
    }
    a = pack<D>(u);
}

// i / d by one multiplication, for i d < 2^32
struct SmallDivisor {
    uint32_t d, m;
};
inline SmallDivisor small_divisor(uint32_t d) { return SmallDivisor{d, d == 1 ? 0u : (uint32_t)((1ull << 32) / d + 1)}; }
__device__ __forceinline__ uint32_t divide(uint32_t i, const SmallDivisor& v) { return v.d == 1 ? i : __umulhi(i, v.m); }

}  // namespace mq
