// The 8-bit rule shared by the int8 products (p2n_int8.hip) and the 8-bit activation checkpoints (p2n_act8.hip).
//   scale  s = float32(max|v| / 127)
//   code   q = clamp(round_half_even(v / s), -127, 127), the quotient taken exactly
//   s = 0 (all zero, or a maximum so small that the division underflows): q = 0
//   a NaN or an infinity among the v: s = NaN, and with it everything that is multiplied by it
#pragma once
#include "p2n_common.h"

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

#ifdef __HIPCC__
// running maximum of |v| as a bit pattern: unsigned order puts the infinities and the NaNs on top
__device__ __forceinline__ unsigned p2n_absbits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// amax / 127, correctly rounded: a first quotient with the rounded reciprocal is off by at most one step, its residual is exact, and
// one correction step with a correctly rounded reciprocal gives the rounded quotient (Markstein) -- as long as nothing
// underflows, below that the division itself.
__device__ __forceinline__ float p2n_q8_scale(unsigned amax_bits) {
    const float a = __uint_as_float(amax_bits), y = 1.0f / 127.0f, q = a * y;
    float s = fmaf(fmaf(-127.0f, q, a), y, q);
    if (__any(a > 0.f && a < 7.9e-31f)) s = a < 7.9e-31f ? a / 127.0f : s;
    return amax_bits >= 0x7F800000u ? __uint_as_float(0x7FC00000u) : s;
}

// What the codes of one scale are formed with: s and v times `up` (2^100 where s is under 2^-100 and has no reciprocal in
// float32, else 1; the product is exact), and 1/(s * up) to one step; 0 where there is nothing to divide by (s = 0, NaN).
struct P2nQ8 {
    float s, up, inv;
};
__device__ __forceinline__ P2nQ8 p2n_q8_make(float s) {
    P2nQ8 Q;
    Q.up = s < 7.9e-31f ? 1.2676506e30f : 1.f;
    Q.s = s * Q.up;
    Q.inv = Q.s > 0.f ? __builtin_amdgcn_rcpf(Q.s) : 0.f;
    return Q;
}

// The code next to a tie.  v * inv is off by less than 1.6e-5 and may sit on the other side of a tie than the true
// quotient; the residual v - q*s decides: there it is a multiple of ulp(s)/2 below 2^25 of them, so the fma gives it exactly.
__device__ __forceinline__ float p2n_q8_decide(float v, const P2nQ8 &Q) {
    v *= Q.up;
    float q = rintf(v * Q.inv);
    const float r = fmaf(-q, Q.s, v), d = 2.f * fabsf(r) - Q.s;
    const bool past = (d > 0.f) | ((d == 0.f) & (((int)q & 1) != 0));
    q += past ? (r < 0.f ? -1.f : 1.f) : 0.f;
    return fminf(fmaxf(q, -127.f), 127.f);
}

// Codes of NV values (a multiple of 4) of one scale, packed four to a dword in order.  v * inv is off by less than 1.6e-5 (inv by
// 2^-23, at up to 127.5), so its rounding to even is the code unless it lies within that of a tie.  The rounding is the addition
// of 1.5 * 2^23 in one fma (one rounding to a whole number, whose low byte is the code).  Any lane near a tie sends its wave
// through the decision for these values: one time in 16 for 16 values of 64 lanes.
#define P2N_Q8_MAGIC 12582912.0f
// four values: their dword, and into `near` how far the farthest lies from its code
__device__ __forceinline__ int p2n_q8_four(const float *v, const P2nQ8 &Q, float &near) {
    unsigned m[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float a = fmaf(v[i], Q.inv, P2N_Q8_MAGIC);
        m[i] = __float_as_uint(a);
        near = fmaxf(near, fabsf(fmaf(v[i], Q.inv, P2N_Q8_MAGIC - a)));
    }
    const unsigned lo = __builtin_amdgcn_perm(m[1], m[0], 0x0C0C0400u);        // bytes 0,1 = low bytes of v0, v1
    const unsigned hi = __builtin_amdgcn_perm(m[3], m[2], 0x04000C0Cu);        // bytes 2,3 = low bytes of v2, v3
    return (int)(lo | hi);
}
__device__ __forceinline__ bool p2n_q8_tie(float near, const P2nQ8 &Q) { return __any((near > 0.49997f) | (Q.up > 1.f)); }
__device__ __forceinline__ int p2n_q8_decide4(const float *v, const P2nQ8 &Q) {
    unsigned c = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) c |= ((unsigned)(int)p2n_q8_decide(v[i], Q) & 0xFFu) << (8 * i);
    return (int)c;
}
template <int NV>
__device__ __forceinline__ void p2n_q8_pack(const float (&v)[NV], const P2nQ8 &Q, int (&code)[NV / 4]) {
    float near = 0.f;
#pragma unroll
    for (int i = 0; i < NV / 4; ++i) code[i] = p2n_q8_four(v + 4 * i, Q, near);
    if (p2n_q8_tie(near, Q)) {
#pragma unroll
        for (int i = 0; i < NV / 4; ++i) code[i] = p2n_q8_decide4(v + 4 * i, Q);
    }
}
#endif
