// Activations held in 8 bits: number formats, token addressing and reductions shared by act8.hip (checkpoints),
// norm8_fwd.hip and norm8_bwd.hip (norms that write or read them).
//
// A token is one position of an activation [N, C, HW]; its C values share ONE exponent.  q is int8 or e4m3 (finite-only,
// largest value 448), shape of the tensor; qe [N, HW] holds exponent + 127 in a byte:
//     value = q * 2^(qe - 127),   qe = smallest exponent with max|v| <= QMAX * 2^(qe - 127),  QMAX = 127 or 448
// Powers of two, not max|v| / QMAX: q * 2^e then has at most 8 significant bits, so a restored value is EXACT in bfloat16 (down to
// 2^-133) and a
// product over restored values carries the one rounding of q and no second one; the price is up to one bit of int8's range
// (e4m3 loses nothing: it has its own exponent).  qe = 255 marks a token with an infinity or NaN: it restores to NaN as a
// whole, so that a diverged activation never comes back finite; a finite token comes back finite (q8_top).  A token of zeros has
// qe = 1 (2^-126).
//
// Times in the comments of these files: one MI355X, bfloat16 unless said, calls of the C entry point back to back (launches and, in a
// backward pass, the column sums included), three sets of operands in turn; variants that are set against each other ran side by side.
#pragma once
#include "common.h"

enum { HIFIC_Q_INT8 = 0, HIFIC_Q_E4M3 = 1 };

typedef unsigned char u8_t;
typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2_t __attribute__((ext_vector_type(2)));

// |v| as unsigned bits: ordered like the magnitudes, infinities above every number and NaN above those
__device__ __forceinline__ unsigned abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ unsigned umax(unsigned a, unsigned b) { return a > b ? a : b; }
// a maximum that keeps a NaN (fmaxf drops it; one instruction either way)
__device__ __forceinline__ float nmax(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ unsigned umin(unsigned a, unsigned b) { return a < b ? a : b; }

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

// v, limited to what rounds to a number of float32: at the largest exponent (2^122 for int8, 2^120 for e4m3) half way to 64 and 256 and
// beyond, the nearest value would be 2^128, and a finite token would come back infinite.  The constants are the numbers below
// 63.5 * 2^122 and 248 * 2^120; no token of a smaller exponent holds more than 127 * 2^121 (which still rounds to itself) or 448 * 2^119.
template <int FMT> __device__ __forceinline__ float q8_top(float v) {
    const float m = __uint_as_float(FMT == HIFIC_Q_INT8 ? 0x7f7dffffu : 0x7f77ffffu);
    return __builtin_amdgcn_fmed3f(v, -m, m);
}

// the same as a limit of t = v / scale for a token of exponent byte `code`: 63 and 240 at the largest exponent
template <int FMT> __device__ __forceinline__ float q8_limit(unsigned code) {
    return FMT == HIFIC_Q_INT8 ? (code == 249u ? 63.f : 127.f) : (code == 247u ? 240.f : 448.f);
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

// the ReLU is open at v (at a NaN too, which then passes forward and backward)
__device__ __forceinline__ bool relu_on(float v) { return !(v <= 0.f); }
__device__ __forceinline__ float relu_nan(float v) { return relu_on(v) ? v : 0.f; }

// xh of a norm whose ReLU follows -> 8 bits that are on the same side of the ReLU: the backward pass masks by the value that was
// kept, and with plain rounding a fraction (step / 4) * density(0) ~ 0.3 % of int8 masks would flip - an error of 5 % (its square
// root) in every gradient behind, ten times what the rounding itself costs.  gamma * x + beta is monotone in x, so of the two
// neighbours of xh one is always on xh's side; it is taken where the nearest one is not.  fmaf rounds once, so its sign is the
// sign of the exact sum and forward and backward agree bit for bit.
template <int FMT>
__device__ __forceinline__ unsigned q8_round_masked(float xh, float inv, float scale, float gamma, float beta) {
    const float t = xh * inv;
    unsigned b = q8_round<FMT>(t);
    const bool on = relu_on(fmaf(gamma, xh, beta));
    if (relu_on(fmaf(gamma, q8_value<FMT>(b) * scale, beta)) != on) b = q8_next<FMT>(b, on == (gamma > 0.f));
    return b;
}

// the compiler may not carry what it computed from r past this point
template <typename V> __device__ __forceinline__ void forget(V& r) { asm volatile("" : "+v"(r)); }

// ---- eight values at a time ------------------------------------------------------------------------------------------------
// The wide kernels give a lane eight neighbouring values (16 bytes of bfloat16): of a plane (eight positions of a channel) or of a
// row (eight channels of a token).  The types are aligned to one element only, so odd planes and rows take the same path
// (gfx950 loads and stores 16 bytes at any address); a last group of fewer than eight is moved back to end at the plane's or row's
// end, and its first values are then computed twice, with the same result.
typedef u32x4_t u32x4_a2 __attribute__((aligned(2)));
typedef u32x2_t u32x2_a1 __attribute__((aligned(1)));
typedef u32x4_t u32x4_a1 __attribute__((aligned(1)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef f32x4_t f32x4_a4 __attribute__((aligned(4)));

template <typename T> struct V8;
template <> struct V8<bf16_t> {
    u32x4_t r;
    __device__ __forceinline__ void load(const bf16_t* p) { r = *(const u32x4_a2*)p; }
    __device__ __forceinline__ float get(int j) const { return __uint_as_float((j & 1) ? (r[j >> 1] & 0xffff0000u) : (r[j >> 1] << 16)); }
    __device__ __forceinline__ void set(const float* v) {
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j] = f2bf2(v[2 * j], v[2 * j + 1]);
    }
    __device__ __forceinline__ void store(bf16_t* p) const { *(u32x4_a2*)p = r; }
    __device__ __forceinline__ void forget() { ::forget(r); }
};
template <> struct V8<float> {
    f32x4_t r[2];
    __device__ __forceinline__ void load(const float* p) { r[0] = *(const f32x4_a4*)p; r[1] = *(const f32x4_a4*)(p + 4); }
    __device__ __forceinline__ float get(int j) const { return r[j >> 2][j & 3]; }
    __device__ __forceinline__ void set(const float* v) {
#pragma unroll
        for (int j = 0; j < 8; ++j) r[j >> 2][j & 3] = v[j];
    }
    __device__ __forceinline__ void store(float* p) const { *(f32x4_a4*)p = r[0]; *(f32x4_a4*)(p + 4) = r[1]; }
    __device__ __forceinline__ void forget() { ::forget(r[0]); ::forget(r[1]); }
};

// eight values, already divided by their scales -> eight bytes.  CLAMP: only where |t| can exceed QMAX by a rounding (see q8_round).
template <int FMT, bool CLAMP>
__device__ __forceinline__ u32x2_t q8_pack8(const float* t) {
    u32x2_t o;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float m = FMT == HIFIC_Q_INT8 ? 127.f : 448.f;
            v[j] = CLAMP ? __builtin_amdgcn_fmed3f(t[4 * h + j], -m, m) : t[4 * h + j];
        }
        if (FMT == HIFIC_Q_INT8) {
            unsigned b[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) b[j] = __float_as_uint(v[j] + 12582912.f);
            o[h] = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u) | __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu);
        } else {
            int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
            o[h] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], w, true);
        }
    }
    return o;
}
// byte B of u, signed, as a number: one instruction (a sub-dword operand with sign extension; written out because the compiler extends
// bytes that are used in two places in one of their own first: rows of 960 from int8, backward 67 us with it, 69 without)
template <int B>
__device__ __forceinline__ float byte_f32(unsigned u) {
    float v;
    if constexpr (B == 0) asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_0" : "=v"(v) : "v"(u));
    else if constexpr (B == 1) asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_1" : "=v"(v) : "v"(u));
    else if constexpr (B == 2) asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_2" : "=v"(v) : "v"(u));
    else asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_3" : "=v"(v) : "v"(u));
    return v;
}
// eight bytes -> eight values, times scale[j].  A product per value, whose result is the kept value whatever the scale (an offset
// byte and one fused multiply-add would need 128 * scale, which is infinite from 2^121 on).
template <int FMT>
__device__ __forceinline__ void q8_unpack8(u32x2_t q, const float* scale, float* v) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if (FMT == HIFIC_Q_INT8) {
            v[4 * h] = byte_f32<0>(q[h]) * scale[4 * h]; v[4 * h + 1] = byte_f32<1>(q[h]) * scale[4 * h + 1];
            v[4 * h + 2] = byte_f32<2>(q[h]) * scale[4 * h + 2]; v[4 * h + 3] = byte_f32<3>(q[h]) * scale[4 * h + 3];
        } else {
            const hw_f32x2_t a = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[h], false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[h], true);
            v[4 * h] = a[0] * scale[4 * h]; v[4 * h + 1] = a[1] * scale[4 * h + 1];
            v[4 * h + 2] = b[0] * scale[4 * h + 2]; v[4 * h + 3] = b[1] * scale[4 * h + 3];
        }
    }
}
__device__ __forceinline__ void q8_scales(u32x2_t e, float* scale) {
#pragma unroll
    for (int j = 0; j < 8; ++j) scale[j] = q8_scale((e[j >> 2] >> (8 * (j & 3))) & 0xffu);
}

// eight normalised values of a channel whose ReLU follows, as x = xh / scale, with v = fma(gamma, xh, beta) and gs = gamma * scale:
// q8_round_masked of each, and v becomes relu(v).  No clamp: max|xh| gave the exponent, so |x| <= QMAX, and the neighbour
// that is taken lies between x and the nearest value's other side.
template <int FMT>
__device__ __forceinline__ u32x2_t q8_pack8_masked(const float* x, float* v, const float* gs, float beta, float gamma) {
    const float up = gamma > 0.f ? 1.f : -1.f;                   // the step towards the ReLU's open side
    if (FMT == HIFIC_Q_INT8) {
        float t[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float n = rintf(x[j]);
            const bool on = relu_on(v[j]);
            const float other = n + (on ? up : -up);
            t[j] = relu_on(fmaf(gs[j], n, beta)) != on ? other : n;
            v[j] = on ? v[j] : 0.f;
        }
        return q8_pack8<FMT, false>(t);
    }
    u32x2_t q = q8_pack8<FMT, false>(x);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const hw_f32x2_t a = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[h], false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[h], true);
        const float n[4] = {a[0], a[1], b[0], b[1]};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool on = relu_on(v[4 * h + j]);
            if (relu_on(fmaf(gs[4 * h + j], n[j], beta)) != on) {
                const unsigned c = q8_next<FMT>((q[h] >> (8 * j)) & 0xffu, (on ? up : -up) > 0.f);
                q[h] = (q[h] & ~(0xffu << (8 * j))) | (c << (8 * j));
            }
            v[4 * h + j] = on ? v[4 * h + j] : 0.f;
        }
    }
    return q;
}

// base (the same for the whole workgroup) + a byte offset per lane: one 32-bit register addresses every tensor of a tile
template <typename T> __device__ __forceinline__ T* at(T* base, unsigned bytes) { return (T*)((char*)base + bytes); }
template <typename T> __device__ __forceinline__ const T* at(const T* base, unsigned bytes) { return (const T*)((const char*)base + bytes); }

// Planes: lane = (group of eight positions pl = lane % LPX, channel sub-group lane / LPX).  v[j], this lane's partial of position j,
// is combined over the 64 / LPX sub-groups of the wave; out[pl * 8 + j] receives the wave's result.
// Every step halves what a lane carries: the lanes of one half keep the first values, those of the other the last ones.  Across
// 32 and 16 lanes that is one swap instruction and one operation per value that is kept, no select and no address (the swap gives
// {x of the low lanes, y of the low lanes} and {x of the high, y of the high}); across 8 lanes a rotation of the row; what is left
// (LPX < 8) is one value.  Eight values over 4 sub-groups: 12 instructions, where shuffles with selects took about 90 and the two
// or three reductions of a tile more than the arithmetic of its values.
template <bool MAX> __device__ __forceinline__ unsigned tile_op(unsigned x, unsigned y) { return MAX ? umax(x, y) : x + y; }
template <bool MAX> __device__ __forceinline__ float tile_op(float x, float y) { return MAX ? nmax(x, y) : x + y; }
template <bool MAX, typename V>
__device__ __forceinline__ V tile_swap32(V x, V y) {
    const u32x2_t r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, y), false, false);
    return tile_op<MAX>(__builtin_bit_cast(V, (unsigned)r[0]), __builtin_bit_cast(V, (unsigned)r[1]));
}
template <bool MAX, typename V>
__device__ __forceinline__ V tile_swap16(V x, V y) {
    const u32x2_t r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, y), false, false);
    return tile_op<MAX>(__builtin_bit_cast(V, (unsigned)r[0]), __builtin_bit_cast(V, (unsigned)r[1]));
}
template <int CTRL, typename V>                                  // a data-parallel-primitive move within rows of 16 lanes
__device__ __forceinline__ V tile_dpp(V x) {
    return __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
template <int LPX, bool MAX, typename V>
__device__ __forceinline__ void tile_reduce(const V* v, V* out) {
    const int lane = threadIdx.x & 63;
    V a[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] = tile_swap32<MAX>(v[j], v[4 + j]);
    int first = (lane & 32) ? 4 : 0;
    if constexpr (LPX <= 16) {
#pragma unroll
        for (int j = 0; j < 2; ++j) a[j] = tile_swap16<MAX>(a[j], a[2 + j]);
        first += (lane & 16) ? 2 : 0;
    }
    if constexpr (LPX <= 8) {
        const bool hi = lane & 8;
        a[0] = tile_op<MAX>(hi ? a[1] : a[0], tile_dpp<0x128>(hi ? a[0] : a[1]));       // row_ror:8 = the lane 8 further
        first += hi ? 1 : 0;
    }
    if constexpr (LPX <= 4) a[0] = tile_op<MAX>(a[0], __builtin_bit_cast(V, __builtin_amdgcn_ds_swizzle(__builtin_bit_cast(int, a[0]), 0x101f)));  // lane ^ 4
    if constexpr (LPX <= 2) a[0] = tile_op<MAX>(a[0], tile_dpp<0x4e>(a[0]));            // quad_perm 2 3 0 1
    if constexpr (LPX <= 1) a[0] = tile_op<MAX>(a[0], tile_dpp<0xb1>(a[0]));            // quad_perm 1 0 3 2
    constexpr int KEEP = LPX == 32 ? 4 : (LPX == 16 ? 2 : 1);
    if (LPX >= 8 || (lane & 7) < LPX)
#pragma unroll
        for (int j = 0; j < KEEP; ++j) out[(lane % LPX) * 8 + first + j] = a[j];
}

// Workgroups go round-robin to the 8 XCDs, each with its own L2; neighbouring tiles share 128-byte lines where a tile is narrower
// than 64 positions: hand each XCD a contiguous range of them.
__device__ __forceinline__ unsigned xcd_block(unsigned bid, unsigned total) {
    return (total & 7u) == 0 ? (bid & 7u) * (total >> 3) + (bid >> 3) : bid;
}

// Tile of the plane kernels: NW waves, LPX groups of eight positions, 64 NW / LPX channel groups, at most `most` channels per
// thread, images of less than 4 GiB.  The widest LPX that fits the channels (what a tile costs besides its values - reductions,
// scales, barriers - is shared by most values then: norm forward 16x60x256x256 75 us, with LPX <= 8 120), then narrower while
// there are CUs without a workgroup (16x960x16x16: 256 wide tiles 12 us, 512 narrow ones 13.4) or more than an eighth of the lanes
// lies past the planes' ends.  Eight waves in the place of four where four would read less than 128 bytes of a channel at a time
// (four / eight waves, norm forward 4x550x50x68 24 / 16 us, 16x480x64x64 47 / 43, backward 63 / 49; 16x960x16x16 9.3 / 8.6, backward
// 14 / 12; eight for 16x240x64x64 too: forward 16.9 / 16.3, backward 24 / 28), and fewer workgroups of
// those are enough before pieces of 16 or 32 bytes are (bfloat16 15x909x22x8: 330 of LPX 1 13.9 us, 165 of LPX 2 9.8; 13x336x50x8: 325 of
// LPX 2 8.4, 169 of LPX 4 7.0; but 16x960x16x16: 256 of LPX 2 8.6, 128 of LPX 4 9.4).
// lpx = 0: more channels than the registers hold, or images beyond 32-bit byte offsets.
struct TileCfg { int lpx, cpt, nw; unsigned tiles; long long blocks; };  // (tiles per image, less than 2^20; of the batch)
static inline TileCfg tile_waves(long long N, int C, int HW, int most, int bytes, int nw) {
    TileCfg t{0, 0, nw, 0, 0};
    for (int lpx = nw == 4 ? 32 : 8; lpx >= 1; lpx >>= 1) {
        const int cpt = cdiv(C, 64 * nw / lpx);
        if (cpt > most) continue;
        t.lpx = lpx; t.cpt = cpt;
        t.tiles = (unsigned)cdiv(cdiv(HW, 8), lpx);
        t.blocks = (long long)t.tiles * N;
        const long long octs = cdiv(HW, 8);
        const int enough = nw == 4 ? 256 : (lpx * 8 * bytes > 32 ? 150 : 100);
        if ((t.blocks >= enough || cpt <= 1) && (lpx == 1 || (long long)t.tiles * lpx * 8 <= octs * 9)) break;
    }
    return t;
}
static inline TileCfg tile_pick(long long N, int C, int HW, int most, int bytes) {
    if ((long long)(C + 512) * HW > (1ll << 30) - 64) return TileCfg{0, 0, 4, 0, 0};     // (C + 512: a lane's offset is formed before it is dropped)
    const TileCfg t = tile_waves(N, C, HW, most, bytes, 4);
    return t.lpx == 0 || (t.lpx * 8 * bytes < 128 && C > 32 * most) ? tile_waves(N, C, HW, most, bytes, 8) : t;
}
// What tile_pick can return (channels per thread as the class 1, 2, 4 or 8 that holds them).  Four waves with pieces of less than 128
// bytes: at most 32 * most channels.  Eight waves: more than 32 * most channels, and at most twice the width that four waves are left
// for - where eight of a width have enough workgroups, four of half of it have them too.
constexpr bool tile_used(int lpx, int cpt, int nw, int most, int bytes) {
    const int least = cpt <= 2 ? cpt : cpt / 2 + 1;
    if (nw == 4) return lpx * 8 * bytes >= 128 || least <= (most * lpx > 8 ? most * lpx / 8 : 1);
    return lpx * bytes <= 16 && cpt >= most * lpx / 16 + 1;
}
// F(LPX, CPT, NW) for the configuration t of elements of type T; only the kernels that tile_pick can ask for are built
#define TILE_DISPATCH(t, T, MOST, F)                                                                                      \
    do {                                                                                                                  \
        if ((t).nw == 8) {                                                                                                \
            if ((t).lpx == 8) { TILE_CPT(8, t, T, MOST, F, 8); } else if ((t).lpx == 4) { TILE_CPT(4, t, T, MOST, F, 8); } \
            else if ((t).lpx == 2) { TILE_CPT(2, t, T, MOST, F, 8); } else { TILE_CPT(1, t, T, MOST, F, 8); }             \
        } else if ((t).lpx == 32) { TILE_CPT(32, t, T, MOST, F, 4); } else if ((t).lpx == 16) { TILE_CPT(16, t, T, MOST, F, 4); } \
        else if ((t).lpx == 8) { TILE_CPT(8, t, T, MOST, F, 4); } else if ((t).lpx == 4) { TILE_CPT(4, t, T, MOST, F, 4); } \
        else if ((t).lpx == 2) { TILE_CPT(2, t, T, MOST, F, 4); } else { TILE_CPT(1, t, T, MOST, F, 4); }                 \
    } while (0)
#define TILE_CPT(LPX, t, T, MOST, F, NW)                                                                                  \
    if ((t).cpt <= 1) { TILE_ONE(LPX, 1, NW, T, MOST, F) } else if ((t).cpt <= 2) { TILE_ONE(LPX, 2, NW, T, MOST, F) }     \
    else if ((t).cpt <= 4) { TILE_ONE(LPX, 4, NW, T, MOST, F) } else { TILE_ONE(LPX, ((MOST) < 8 ? 4 : 8), NW, T, MOST, F) }
#define TILE_ONE(LPX, CPT, NW, T, MOST, F)                                                                                \
    if constexpr (tile_used(LPX, CPT, NW, MOST, sizeof(T))) { F(LPX, CPT, NW); } else return HIFIC_ERR_UNSUPPORTED;
// sum / maximum over the waves' results of a tile position
template <int NW, int TP> __device__ __forceinline__ float waves_sum(const float (*red)[TP], int i) {
    float s = (red[0][i] + red[1][i]) + (red[2][i] + red[3][i]);
    if constexpr (NW == 8) s += (red[4][i] + red[5][i]) + (red[6][i] + red[7][i]);
    return s;
}
template <int NW, int TP> __device__ __forceinline__ float waves_max(const float (*red)[TP], int i) {
    float m = nmax(nmax(red[0][i], red[1][i]), nmax(red[2][i], red[3][i]));
    if constexpr (NW == 8) m = nmax(m, nmax(nmax(red[4][i], red[5][i]), nmax(red[6][i], red[7][i])));
    return m;
}

// Rows: L lanes and K groups of eight channels per lane hold a row, in workgroups of row_block(L) threads.  Sums and maxima over the
// row's L lanes, through LDS where a row has the whole workgroup.
constexpr int row_block(int L) { return L > 256 ? L : 256; }
template <int L, typename V, typename Op>
__device__ __forceinline__ V row_reduce(V v, Op op) {
#pragma unroll
    for (int o = (L < 64 ? L : 64) >> 1; o > 0; o >>= 1) v = op(v, __builtin_bit_cast(V, __shfl_xor(__builtin_bit_cast(int, v), o, 64)));
    if constexpr (L >= 256) {
        __shared__ V red[L / 64];
        __syncthreads();
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        V part[L / 64];
#pragma unroll
        for (int i = 0; i < L / 64; ++i) part[i] = red[i];
#pragma unroll
        for (int s = L / 128; s > 0; s >>= 1)
#pragma unroll
            for (int i = 0; i < s; ++i) part[i] = op(part[i], part[i + s]);
        v = part[0];
    }
    return v;
}
template <int L> __device__ __forceinline__ float row_sum(float v) { return row_reduce<L>(v, [](float a, float b) { return a + b; }); }
template <int L> __device__ __forceinline__ unsigned row_max(unsigned v) { return row_reduce<L>(v, [](unsigned a, unsigned b) { return umax(a, b); }); }
// As few lanes of a wave as hold the row in one group each (65536x129, both passes: 32 lanes 36 us, 64 lanes 52), the wave with up to 4 groups for
// wider ones, a workgroup of 256 above 2048 channels and where fewer than 1024 rows would leave the other CUs idle, one of 1024
// threads above 8192 (2048x16384, both passes: 130 us, the any-shape kernels 331).  l = 0: more channels than the registers hold.
struct RowCfg { int l, k; };
static inline RowCfg row_pick(long long N, int C) {
    RowCfg r;
    if (C > 2048 || (N < 1024 && C > 512)) r.l = C > 8192 ? 1024 : 256;
    else r.l = C <= 64 ? 8 : (C <= 128 ? 16 : (C <= 256 ? 32 : 64));
    r.k = cdiv(C, 8 * r.l);
    if (r.k > (r.l == 1024 ? 2 : 4)) r.l = 0;
    return r;
}
#define ROW_DISPATCH(r, F)                                                                              \
    do {                                                                                                \
        if ((r).l == 8) { F(8, 1); } else if ((r).l == 16) { F(16, 1); } else if ((r).l == 32) { F(32, 1); } \
        else if ((r).l == 64) { if ((r).k <= 1) { F(64, 1); } else if ((r).k <= 2) { F(64, 2); } else { F(64, 4); } } \
        else if ((r).l == 256) { if ((r).k <= 1) { F(256, 1); } else if ((r).k <= 2) { F(256, 2); } else { F(256, 4); } } \
        else { F(1024, 2); }                                                                            \
    } while (0);

// Lanes on tokens of the any-shape kernels, counted over the batch (the rest of 256 on channels): 64, 16 where they are few, 1 for
// rows of eight channels and more, whose neighbours in memory are channels.  At most 2^20 workgroups, each with its share of the tokens.
static inline int any_px(long long N, int C, int HW) { return HW == 1 && C >= 8 ? 1 : (N * HW < 64 * 512 ? 16 : 64); }
static inline unsigned any_grid(long long blocks) { return (unsigned)(blocks < (1 << 20) ? blocks : 1 << 20); }

// A launch holds less than 2^32 threads: F(first image, images) over parts of the batch of at most 2^21 workgroups (or one image).
template <typename F>
static inline int batch_parts(long long N, long long per_image, F f) {
    const long long step = (1ll << 21) / per_image > 1 ? (1ll << 21) / per_image : 1;
    for (long long n = 0; n < N; n += step) {
        const int rc = f(n, N - n < step ? N - n : step);
        if (rc != HIFIC_OK) return rc;
    }
    return HIFIC_OK;
}
// a null pointer stays one
template <typename T> static inline T* ahead(T* p, long long n) { return p ? p + n : p; }

constexpr int ACT8_MAX_C = 1 << 20;      // channels of a token in what forms its sums or exponent
static inline bool act8_dtype_ok(int dtype) { return dtype == HIFIC_F32 || dtype == HIFIC_BF16; }
static inline bool act8_fmt_ok(int fmt) { return fmt == HIFIC_Q_INT8 || fmt == HIFIC_Q_E4M3; }
