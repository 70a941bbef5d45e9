// vy_quant.cuh -- int8 codes of a row from its largest magnitude (device helpers).
#pragma once

#include "vy_common.cuh"

namespace vy {

// A code is the nearest integer of the exact quotient x / s, ties to even.  With 1 / s rounded down
// and up, one fused multiply-add each rounds x lo and x hi to the nearest integer (adding 1.5 * 2^23,
// which leaves the integer's two's complement in the low bits); x / s lies between the two products
// and rounding is monotone, so where both give one integer it is the code.  Where they differ (about
// one value in 10^5: a tie c lies between), the sign of x - c s decides, exact under one fused
// multiply-add.  Two FFMAs and a LOP3 a value; rint and float-to-int conversions run at an eighth of
// that rate and would bound the kernel; following the distance to the nearest tie instead took some 20
// instructions a value in all (4096 x 14336, bf16: 46 us, 36 this way).
constexpr float kRound = 12582912.f;

struct RowScale {
    float s, lo, hi;
    float up;           // 1, or 2^100 where 1 / s is out of range: x and s are scaled by it, exactly
    uint32_t odd;       // not zero when up is not 1: every value takes the long way
    uint32_t keep;      // 0 for a zero row or a NaN scale: all codes 0; else all ones
};

__device__ __forceinline__ float quant_long(float v, const RowScale& r) {
    const float x = v * r.up, s = r.s * r.up;
    const float t = x * __frcp_rn(s);
    const float near = (t + kRound) - kRound, d = t - near;
    float q = near;
    if (fabsf(d) > 0.499f) {                      // t is off by 2^-23 relative at most
        const float c = near + copysignf(0.5f, d);
        const float e = fmaf(-c, s, x);           // c s has 32 bits, nothing underflows: the sign is exact
        q = e > 0.f ? c + 0.5f : e < 0.f ? c - 0.5f : c;     // c + kRound goes to the even one
    }
    // a subnormal s may be so coarse that amax / s passes 127
    return fminf(fmaxf(q, -127.f), 127.f) + kRound;
}

// The codes of N values, N / 4 words.
template <int N>
__device__ __forceinline__ void quant_words(const float (&v)[N], const RowScale& r, uint32_t (&w)[N / 4]) {
    uint32_t m[N], differ = r.odd;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        m[j] = __float_as_uint(fmaf(v[j], r.lo, kRound));
        differ |= m[j] ^ __float_as_uint(fmaf(v[j], r.hi, kRound));
    }
    if (differ) {
#pragma unroll
        for (int j = 0; j < N; ++j) m[j] = __float_as_uint(quant_long(v[j], r));
    }
#pragma unroll
    for (int q = 0; q < N / 4; ++q) {
        const uint32_t lo = __byte_perm(m[4 * q], m[4 * q + 1], 0x0040);
        const uint32_t hi = __byte_perm(m[4 * q + 2], m[4 * q + 3], 0x0040);
        w[q] = __byte_perm(lo, hi, 0x5410) & r.keep;
    }
}

// Plain (coherent) 16-byte load: x may come from the kernel in front, which this one overlaps.
__device__ __forceinline__ uint4 ld_piece(const uint4* p) {
    uint4 v;
    asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// Values of one 16-byte piece, and their largest magnitude's bit pattern (magnitudes order like
// their patterns, NaN above infinity: an integer maximum).
template <int DT>
struct Piece {
    static constexpr int N = DT == VY_F32 ? 4 : 8;
    static __device__ __forceinline__ void values(const uint4& u, float (&v)[N]) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (DT == VY_F32) {
                v[j] = __uint_as_float(w[j]);
            } else if constexpr (DT == VY_BF16) {
                v[2 * j] = __uint_as_float(w[j] << 16);
                v[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
            } else {
                v[2 * j] = act_from_bits<VY_F16>(w[j] & 0xFFFFu);
                v[2 * j + 1] = act_from_bits<VY_F16>(w[j] >> 16);
            }
        }
    }
    // 16-bit types: of each half in place, fp32: of the word
    static __device__ __forceinline__ uint32_t top(uint32_t t, const uint4& u) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (DT == VY_F32)
                t = max(t, w[j] & 0x7FFFFFFFu);
            else if constexpr (DT == VY_BF16)
                asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(t) : "r"(w[j] & 0x7FFF7FFFu));
            else
                asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(t) : "r"(w[j] & 0x7FFF7FFFu));
        }
        return t;
    }
    // the fp32 magnitude's pattern from top's
    static __device__ __forceinline__ uint32_t wide(uint32_t t) {
        if constexpr (DT == VY_F32) return t;
        const uint32_t a = __float_as_uint(act_from_bits<DT>(t & 0xFFFFu)) & 0x7FFFFFFFu;
        return max(a, __float_as_uint(act_from_bits<DT>(t >> 16)) & 0x7FFFFFFFu);
    }
};

// The scale of a row whose largest magnitude has the pattern `top`.
__device__ __forceinline__ RowScale row_scale(uint32_t top) {
    RowScale r;
    r.s = top < 0x7F800000u ? __fdiv_rn(__uint_as_float(top), 127.f) : __uint_as_float(0x7FC00000u);
    const bool zero = !(r.s > 0.f), tiny = r.s < 1e-30f && !zero;
    r.up = tiny ? 0x1p100f : 1.f;
    r.odd = tiny;
    r.keep = zero ? 0u : 0xFFFFFFFFu;
    r.lo = zero || tiny ? 0.f : __frcp_rd(r.s);
    r.hi = zero || tiny ? 0.f : __frcp_ru(r.s);
    return r;
}
// Codes of a row's 16-byte piece `at`.
template <int DT>
__device__ __forceinline__ void put_piece(int8_t* out, int64_t at, const uint4& u, const RowScale& r) {
    using P = Piece<DT>;
    float v[P::N];
    uint32_t w[P::N / 4];
    P::values(u, v);
    quant_words<P::N>(v, r, w);
    if constexpr (P::N == 8)
        reinterpret_cast<uint2*>(out)[at] = make_uint2(w[0], w[1]);
    else
        reinterpret_cast<uint32_t*>(out)[at] = w[0];
}
// Codes of single values k, k + step, ... below cols (rows that are no whole pieces, or not aligned).
template <int DT>
__device__ __forceinline__ void put_tail(int8_t* out, const void* src, int64_t k, int64_t cols, int step, const RowScale& r) {
    for (; k < cols; k += step) {
        const float v[4] = {load_as_float(src, DT, k), 0.f, 0.f, 0.f};
        uint32_t w[1];
        quant_words<4>(v, r, w);
        out[k] = static_cast<int8_t>(w[0] & 0xFFu);
    }
}

}  // namespace vy
