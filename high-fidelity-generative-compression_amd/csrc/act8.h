// Activations held in 8 bits: number formats, token addressing and reductions shared by act8.hip (checkpoints) and norm8.hip
// (norms that write or read them).
//
// A token is one position of an activation [N, C, HW]; its C values share ONE exponent.  q is int8 or e4m3 (finite-only,
// largest value 448), shape of the tensor; qe [N, HW] holds exponent + 127 in a byte:
//     value = q * 2^(qe - 127),   qe = smallest exponent with max|v| <= QMAX * 2^(qe - 127),  QMAX = 127 or 448
// Powers of two, not max|v| / QMAX: q * 2^e then has at most 8 significant bits, so a restored value is EXACT in bfloat16 and a
// product over restored values carries the one rounding of q and no second one; the price is up to one bit of int8's range
// (e4m3 loses nothing: it has its own exponent).  qe = 255 marks a token with an infinity or NaN: it restores to NaN as a
// whole, so that a diverged activation never comes back finite.  A token of zeros has qe = 1 (2^-126).
#pragma once
#include "common.h"

enum { HIFIC_Q_INT8 = 0, HIFIC_Q_E4M3 = 1 };

typedef unsigned char u8_t;
typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2_t __attribute__((ext_vector_type(2)));

// |v| as unsigned bits: ordered like the magnitudes, infinities above every number and NaN above those (fmaxf would lose a NaN)
__device__ __forceinline__ unsigned abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ unsigned umax(unsigned a, unsigned b) { return a > b ? a : b; }

// amax as abs_bits -> the byte of the exponent.  QMAX = 1.984375 * 2^6 (127) or 1.75 * 2^8 (448).
template <int FMT>
__device__ __forceinline__ unsigned q8_code(unsigned amax) {
    if (amax >= 0x7f800000u) return 255u;
    const int k = (int)(amax >> 23);                                 // biased exponent of amax
    const unsigned frac = amax & 0x7fffffu;
    const int e = FMT == HIFIC_Q_INT8 ? k - 6 + (frac > 0x7e0000u ? 1 : 0) : k - 8 + (frac > 0x600000u ? 1 : 0);
    return (unsigned)(e < 1 ? 1 : e);
}
__device__ __forceinline__ float q8_scale(unsigned code) {           // 2^(code - 127); NaN for a token that is not finite
    return __uint_as_float((code << 23) | (code == 255u ? 0x400000u : 0u));
}
__device__ __forceinline__ float q8_inv_scale(unsigned code) {       // 2^(127 - code); 0 for a token that is not finite
    return code == 255u ? 0.f : __uint_as_float((254u - code) << 23);
}

// One value t = v / scale -> its 8 bits (round half to even).  The clamp only acts where max|v| was formed with another rounding
// than v itself (|t| at most one ulp above QMAX).  0 * inf of a token that is not finite is stored as 0.
template <int FMT>
__device__ __forceinline__ unsigned q8_round(float t) {
    if (FMT == HIFIC_Q_INT8) {
        t = __builtin_amdgcn_fmed3f(t, -127.f, 127.f);
        // adding 1.5 * 2^23 leaves round(t) in two's complement in the low bits
        return __float_as_uint(t + 12582912.f) & 0xffu;
    }
    t = __builtin_amdgcn_fmed3f(t, -448.f, 448.f);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(t, t, 0, false) & 0xffu;
}
template <int FMT>
__device__ __forceinline__ float q8_value(unsigned b) {              // the 8 bits as a number, without the exponent
    if (FMT == HIFIC_Q_INT8) return (float)(signed char)b;
    return __builtin_amdgcn_cvt_f32_fp8((int)b, 0);
}
// the format's next value above (up) or below, never beyond +-QMAX: two's complement, or sign and magnitude with one step
// across zero (e4m3's -0 counts as 0)
template <int FMT>
__device__ __forceinline__ unsigned q8_next(unsigned b, bool up) {
    const int top = FMT == HIFIC_Q_INT8 ? 127 : 126;                 // e4m3 code 126 is 448, 127 is NaN
    int key = FMT == HIFIC_Q_INT8 ? (int)(signed char)b : ((b & 0x80u) ? -(int)(b & 0x7fu) : (int)b);
    key += up ? 1 : -1;
    key = key > top ? top : (key < -top ? -top : key);
    return FMT == HIFIC_Q_INT8 ? (unsigned)key & 0xffu : (key < 0 ? 0x80u | (unsigned)(-key) : (unsigned)key);
}

// xh of a norm whose ReLU follows -> 8 bits that are on the same side of the ReLU: the backward pass masks by the value that was
// kept, and with plain rounding a fraction (step / 4) * density(0) ~ 0.3 % of int8 masks would flip - an error of 5 % (its square
// root) in every gradient behind, ten times what the rounding itself costs.  gamma * x + beta is monotone in x, so of the two
// neighbours of xh one is always on xh's side; it is taken where the nearest one is not.  fmaf rounds once, so its sign is the
// sign of the exact sum and forward and backward agree bit for bit.
template <int FMT>
__device__ __forceinline__ unsigned q8_round_masked(float xh, float inv, float scale, float gamma, float beta) {
    const float t = xh * inv;
    unsigned b = q8_round<FMT>(t);
    const float v = q8_value<FMT>(b);
    if ((fmaf(gamma, v * scale, beta) > 0.f) != (fmaf(gamma, xh, beta) > 0.f)) b = q8_next<FMT>(b, t > v);
    return b;
}

static inline bool act8_dtype_ok(int dtype) { return dtype == HIFIC_F32 || dtype == HIFIC_BF16; }
static inline bool act8_fmt_ok(int fmt) { return fmt == HIFIC_Q_INT8 || fmt == HIFIC_Q_E4M3; }
