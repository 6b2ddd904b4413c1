// Norms that write or read activations in 8 bits (format: act8.h), and the root-mean-square norm.  Per token t of x [N, C, HW]:
//   RMS norm      h = x (+ resid, rounded to the storage type: the new residual stream),  r = rsqrt(sum_c h^2 / C + eps),
//                 xh = h r,  y = w_c xh
//                 backward: g = w dy,  dx = r (g - xh sum_c(g xh) / C) (+ dstream),  dw_c = sum_t dy xh
//   channel norm  d = x - sum_c x / C,  r = rsqrt(sum_c d^2 / (C - 1) + eps),  xh = d r,
//                 y = relu?(gamma_c xh + beta_c) (+ resid)
//                 backward: dy masked by gamma xh + beta > 0,  g = gamma dy,
//                 dx = r (g - sum_c g / C - xh sum_c(g xh) / (C - 1)),  dgamma_c = sum_t dy xh,  dbeta_c = sum_t dy
// What the backward pass needs of the forward pass is xh and r: xh is kept in 8 bits (1 byte per element in the place of the 2 of
// a bfloat16 input, or of the 4 of input and output), r in float32 per token.  Sums and statistics are float32 throughout.
#include "act8.h"
#include <type_traits>

enum { M_RMS = 0, M_CHAN = 1 };
enum { Q_NONE = 2 };                     // FMT of a forward kernel that writes no 8-bit tensor
enum { SRC_T = 2 };                      // SRC of a backward kernel that reads h in the storage type (0 / 1: int8 / e4m3)

// sums / maxima over the C values of a token: lanes px, px + PX, ... of a wave, then the block's four waves through LDS
template <int PX>
__device__ __forceinline__ float tok_sum(float v, float (*red)[PX]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int o = PX; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
    __syncthreads();
    if (lane < PX) red[wave][lane] = v;
    __syncthreads();
    return (red[0][lane % PX] + red[1][lane % PX]) + (red[2][lane % PX] + red[3][lane % PX]);
}
template <int PX>
__device__ __forceinline__ unsigned tok_max(unsigned v, float (*red)[PX]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int o = PX; o < 64; o <<= 1) v = umax(v, (unsigned)__shfl_xor((int)v, o, 64));
    __syncthreads();
    if (lane < PX) red[wave][lane] = __uint_as_float(v);
    __syncthreads();
    const int p = lane % PX;
    return umax(umax(__float_as_uint(red[0][p]), __float_as_uint(red[1][p])), umax(__float_as_uint(red[2][p]), __float_as_uint(red[3][p])));
}

struct NormFwd {
    const void* x; const void* resid; const float* w; const float* b;
    void* y; void* h; float* rstd;
    u8_t *q, *qe, *q2, *qe2;             // xh (RMS with q_of_y: y) and, with a channel norm's resid, y
    int C, HW; unsigned tiles; float eps; int relu, q_of_y;
    float rc, rv;                        // 1 / C, and 1 / C or 1 / (C - 1): a product in the place of a division per position
};

// Any shape: PX lanes on consecutive positions x 256 / PX channel groups, the tensor re-read by every pass (from L2).
template <typename T, int MODE, int FMT, int PX>
__global__ __launch_bounds__(256) void norm8_fwd_kernel(const NormFwd p) {
    constexpr int G = 256 / PX;
    constexpr int F = FMT == Q_NONE ? HIFIC_Q_INT8 : FMT;
    __shared__ float red[4][PX];
    const int px = threadIdx.x % PX, g = threadIdx.x / PX;
    const unsigned n = blockIdx.x / p.tiles, hw = (blockIdx.x - n * p.tiles) * PX + px;
    const bool ok = hw < (unsigned)p.HW;
    const size_t base = (size_t)n * p.C * p.HW + (ok ? hw : 0), tok = (size_t)n * p.HW + hw;
    const T* x = (const T*)p.x + base;
    const T* rs = p.resid ? (const T*)p.resid + base : nullptr;
    T* y = p.y ? (T*)p.y + base : nullptr;
    T* h = p.h ? (T*)p.h + base : nullptr;
    const size_t cs = p.HW;
    auto stream = [&](int c) {
        float v = DT<T>::ld(x + c * cs);
        if (MODE == M_RMS && rs) { T o; DT<T>::st(&o, v + DT<T>::ld(rs + c * cs)); v = DT<T>::ld(&o); }
        return v;
    };
    float mu = 0.f;
    if (MODE == M_CHAN) {
        float s = 0.f;
        for (int c = g; c < p.C; c += G) s += stream(c);
        mu = tok_sum<PX>(s, red) * p.rc;
    }
    float ss = 0.f;
    for (int c = g; c < p.C; c += G) {
        const float v = stream(c), d = v - mu;
        ss += d * d;
        if (MODE == M_RMS && h && ok) DT<T>::st(h + c * cs, v);
    }
    ss = tok_sum<PX>(ss, red);
    const float r = rsqrtf(ss * p.rv + p.eps);
    if (p.rstd && ok && g == 0) p.rstd[tok] = r;
    unsigned code = 0;
    float inv = 0.f, scale = 0.f;
    if (FMT != Q_NONE) {
        unsigned am = 0;
        for (int c = g; c < p.C; c += G) {
            const float xh = (stream(c) - mu) * r;
            am = umax(am, abs_bits(MODE == M_RMS && p.q_of_y ? xh * p.w[c] : xh));
        }
        code = q8_code<F>(tok_max<PX>(am, red));
        inv = q8_inv_scale(code); scale = q8_scale(code);
        if (ok && g == 0) p.qe[tok] = (u8_t)code;
    }
    unsigned am2 = 0;
    for (int c = g; c < p.C; c += G) {
        const float xh = (stream(c) - mu) * r;
        float o = MODE == M_RMS ? xh * p.w[c] : fmaf(p.w[c], xh, p.b[c]);
        if (FMT != Q_NONE && ok)
            p.q[base + c * cs] = (u8_t)(MODE == M_CHAN && p.relu ? q8_round_masked<F>(xh, inv, scale, p.w[c], p.b[c])
                                                                 : q8_round<F>((MODE == M_RMS && p.q_of_y ? o : xh) * inv));
        if (MODE == M_CHAN && p.relu) o = relu_nan(o);
        if (MODE == M_CHAN && rs) {      // both terms rounded to the storage type first, as norm and add one after the other
            T t; DT<T>::st(&t, o); o = DT<T>::ld(&t) + DT<T>::ld(rs + c * cs);
        }
        if (y && ok) DT<T>::st(y + c * cs, o);
        am2 = umax(am2, abs_bits(o));
    }
    if (MODE == M_CHAN && FMT != Q_NONE && p.q2) {
        const unsigned code2 = q8_code<F>(tok_max<PX>(am2, red));
        const float inv2 = q8_inv_scale(code2);
        if (ok && g == 0) p.qe2[tok] = (u8_t)code2;
        for (int c = g; c < p.C; c += G) {
            float o = fmaf(p.w[c], (stream(c) - mu) * r, p.b[c]);
            if (p.relu) o = relu_nan(o);
            T t; DT<T>::st(&t, o); o = DT<T>::ld(&t) + DT<T>::ld(rs + c * cs);
            if (ok) p.q2[base + c * cs] = (u8_t)q8_round<F>(o * inv2);
        }
    }
}

// Planes of eight positions and more: a workgroup owns LPX * 8 positions x all channels (tile_pick), eight positions and CPT
// channels per lane, kept as they were loaded between the passes: every tensor crosses HBM once.
template <typename T, int MODE, int FMT, int LPX, int CPT>
__global__ __launch_bounds__(256, 2) void norm8_fwd_tile_kernel(const NormFwd p, unsigned blocks) {
    constexpr int SUBS = 64 / LPX, G = 4 * SUBS, TP = LPX * 8;
    constexpr int F = FMT == Q_NONE ? HIFIC_Q_INT8 : FMT;
    __shared__ float red[4][TP], redm[4][TP];
    __shared__ float st_r[TP], st_inv[TP];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, pl = lane % LPX, g = wave * SUBS + lane / LPX;
    const unsigned bid = xcd_block(blockIdx.x, blocks), n = bid / p.tiles, tile = bid - n * p.tiles;
    const unsigned oct = tile * LPX + pl, octs = ((unsigned)p.HW + 7) >> 3;
    const bool ok = oct < octs;
    const unsigned off0 = umin(ok ? oct * 8 : 0u, (unsigned)p.HW - 8), off = (unsigned)g * p.HW + off0;
    const unsigned kst = (unsigned)G * p.HW;                         // channel k of this lane: img + off + k * kst
    const size_t img = (size_t)n * p.C * p.HW;
    // position tid of the tile, for the threads that finish the statistics
    const unsigned so = tile * LPX + (tid >> 3);
    const bool sok = tid < TP && so < octs;
    const size_t stok = (size_t)n * p.HW + umin(so * 8, (unsigned)p.HW - 8) + (tid & 7);
    const T *x = (const T*)p.x + img, *rs = (const T*)p.resid + (p.resid ? img : 0);
    V8<T> xr[CPT], rr[CPT];
    float w[CPT], b[MODE == M_CHAN ? CPT : 1];
#pragma unroll
    for (int k = 0; k < CPT; ++k) {
        const int c = g + G * k < p.C ? g + G * k : 0;               // (a load of channel 0 in the place of a branch around it)
        const unsigned o = (c == 0 ? off0 : off + k * kst) * (unsigned)sizeof(T);
        xr[k].load(at(x, o));
        w[k] = p.w[c];
        if constexpr (MODE == M_CHAN) b[k] = p.b[c];
        if (p.resid) rr[k].load(at(rs, o));
    }
    if (MODE == M_RMS && p.resid) {
#pragma unroll
        for (int k = 0; k < CPT; ++k) {
            float h[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) h[j] = xr[k].get(j) + rr[k].get(j);
            xr[k].set(h);
            if (ok && g + G * k < p.C) xr[k].store(at((T*)p.h + img, (off + k * kst) * (unsigned)sizeof(T)));
        }
    }
    // maxima as floats: a NaN is lost in them, but not in the sum of squares, and r carries it into the exponent
    float mu[8], acc[8], am[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) { mu[j] = 0.f; acc[j] = 0.f; am[j] = 0.f; }
    if constexpr (MODE == M_CHAN) {
#pragma unroll
        for (int k = 0; k < CPT; ++k)
            if (g + G * k < p.C)
#pragma unroll
                for (int j = 0; j < 8; ++j) acc[j] += xr[k].get(j);
        tile_reduce<LPX, false>(acc, red[wave]);
        __syncthreads();
        if (tid < TP) st_r[tid] = ((red[0][tid] + red[1][tid]) + (red[2][tid] + red[3][tid])) * p.rc;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 8; ++j) { mu[j] = st_r[pl * 8 + j]; acc[j] = 0.f; }
    }
    // each pass unpacks again: kept unpacked, the values would take twice the registers
#pragma unroll
    for (int k = 0; k < CPT; ++k) xr[k].forget();
#pragma unroll
    for (int k = 0; k < CPT; ++k)
        if (g + G * k < p.C)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float d = xr[k].get(j) - mu[j];
                acc[j] += d * d;
                if (FMT != Q_NONE) am[j] = fmaxf(am[j], fabsf(MODE == M_RMS && p.q_of_y ? d * w[k] : d));
            }
#pragma unroll
    for (int k = 0; k < CPT; ++k) xr[k].forget();
    tile_reduce<LPX, false>(acc, red[wave]);
    if (FMT != Q_NONE) tile_reduce<LPX, true>(am, redm[wave]);
    __syncthreads();
    if (tid < TP) {
        const float ss = (red[0][tid] + red[1][tid]) + (red[2][tid] + red[3][tid]);
        const float r = rsqrtf(ss * p.rv + p.eps);
        st_r[tid] = r;
        if (p.rstd && sok) p.rstd[stok] = r;
        if (FMT != Q_NONE) {
            // max|d| r = max|d r|: a rounded product is monotone (with q_of_y the weight comes between, and q8_pack8 clamps)
            const float m = fmaxf(fmaxf(redm[0][tid], redm[1][tid]), fmaxf(redm[2][tid], redm[3][tid]));
            const unsigned code = q8_code<F>(abs_bits(m * r));
            st_inv[tid] = q8_inv_scale(code);
            if (sok) p.qe[stok] = (u8_t)code;
        }
    }
    __syncthreads();
    // x = d * (r / scale) is xh / scale: dividing by a power of two commutes with the rounding, and so does gs below
    float r[8], ri[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float inv = FMT != Q_NONE ? st_inv[pl * 8 + j] : 0.f;
        r[j] = st_r[pl * 8 + j]; ri[j] = r[j] * inv; am[j] = 0.f;
        // behind a ReLU only x and gs are formed: r's place holds the scale 1 / inv, a power of two (2^127 for a token that is not
        // finite: its values are NaN)
        if (MODE == M_CHAN && FMT != Q_NONE && p.relu) r[j] = __uint_as_float(0x7f000000u - __float_as_uint(inv));
    }
#pragma unroll
    for (int k = 0; k < CPT; ++k) {
        const int c = g + G * k;
        if (c >= p.C) continue;
        float o[8];
        if (MODE == M_CHAN && FMT != Q_NONE && p.relu) {
            float x[8], gs[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                gs[j] = w[k] * r[j];
                x[j] = (xr[k].get(j) - mu[j]) * ri[j];
                o[j] = fmaf(gs[j], x[j], b[MODE == M_CHAN ? k : 0]);
            }
            const u32x2_t q = q8_pack8_masked<F>(x, o, gs, b[MODE == M_CHAN ? k : 0], w[k]);
            if (ok) *(u32x2_a1*)at(p.q + img, off + k * kst) = q;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float xh = (xr[k].get(j) - mu[j]) * r[j];
                o[j] = MODE == M_RMS ? xh * w[k] : fmaf(w[k], xh, b[MODE == M_CHAN ? k : 0]);
            }
            if constexpr (FMT != Q_NONE) {
                float t[8];
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    t[j] = MODE == M_RMS && p.q_of_y ? o[j] * st_inv[pl * 8 + j] : (xr[k].get(j) - mu[j]) * ri[j];
                const u32x2_t q = q8_pack8<F, MODE == M_RMS>(t);
                if (ok) *(u32x2_a1*)at(p.q + img, off + k * kst) = q;
            }
        }
        if constexpr (MODE == M_CHAN) {
            if (p.resid) {               // both terms rounded to the storage type first, as norm and add one after the other
                V8<T> t; t.set(o);
#pragma unroll
                for (int j = 0; j < 8; ++j) { o[j] = t.get(j) + rr[k].get(j); if (FMT != Q_NONE) am[j] = fmaxf(am[j], fabsf(o[j])); if (o[j] != o[j]) am[j] = INFINITY; }
                xr[k] = t;               // q2 below: the sum again from its two terms, in float32
            }
        }
        if (p.y && ok) { V8<T> t; t.set(o); t.store(at((T*)p.y + img, (off + k * kst) * (unsigned)sizeof(T))); }
    }
    if constexpr (MODE == M_CHAN && FMT != Q_NONE) {
        if (!p.q2) return;
        tile_reduce<LPX, true>(am, redm[wave]);          // (a NaN as an infinity; redm's readers are behind a barrier)
        __syncthreads();
        if (tid < TP) {
            const unsigned code = q8_code<F>(abs_bits(fmaxf(fmaxf(redm[0][tid], redm[1][tid]), fmaxf(redm[2][tid], redm[3][tid]))));
            st_inv[tid] = q8_inv_scale(code);
            if (sok) p.qe2[stok] = (u8_t)code;
        }
        __syncthreads();
        if (!ok) return;
#pragma unroll
        for (int k = 0; k < CPT; ++k) {
            const int c = g + G * k;
            if (c >= p.C) continue;
            float t[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) t[j] = (xr[k].get(j) + rr[k].get(j)) * st_inv[pl * 8 + j];
            *(u32x2_a1*)at(p.q2 + img, off + k * kst) = q8_pack8<F, false>(t);
        }
    }
}

// Rows of eight channels and more (root-mean-square norm): eight channels per lane, L lanes and K groups per lane for a row.
template <typename T, int FMT, int L, int K>
__global__ __launch_bounds__(256) void rms_fwd_rows_kernel(const NormFwd p, int N) {
    constexpr int F = FMT == Q_NONE ? HIFIC_Q_INT8 : FMT;
    const int l = threadIdx.x % L;
    const long long row0 = (long long)blockIdx.x * (256 / L) + threadIdx.x / L;
    const bool ok = row0 < N;
    const size_t base = (size_t)(ok ? row0 : N - 1) * p.C;
    const unsigned C = p.C;
    V8<T> xr[K], rr[K];
    V8<float> w[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const unsigned c = umin((unsigned)(l + L * k) * 8, C - 8);
        xr[k].load((const T*)p.x + base + c);
        if (p.resid) rr[k].load((const T*)p.resid + base + c);
        w[k].load(p.w + c);
    }
    float ss = 0.f, am = 0.f;            // (a NaN is lost in am, not in ss, and r carries it into the exponent)
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const unsigned cn = (unsigned)(l + L * k) * 8, c = umin(cn, C - 8);
        if (p.resid) {
            float h[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) h[j] = xr[k].get(j) + rr[k].get(j);
            xr[k].set(h);
            if (ok && cn < C) xr[k].store((T*)p.h + base + c);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            // a group past the end was moved back: its first values belong to the group before it
            const float v = c + j >= cn ? xr[k].get(j) : 0.f;
            ss += v * v;
            if (FMT != Q_NONE) am = fmaxf(am, fabsf(p.q_of_y ? v * w[k].get(j) : v));
        }
    }
    ss = row_sum<L>(ss);
    const float r = rsqrtf(ss * p.rv + p.eps);
    float inv = 0.f;
    if constexpr (FMT != Q_NONE) {
        const unsigned code = q8_code<F>(abs_bits(__uint_as_float(row_max<L>(__float_as_uint(am))) * r));
        inv = q8_inv_scale(code);
        if (ok && l == 0) p.qe[row0] = (u8_t)code;
    }
    if (!ok) return;
    if (p.rstd && l == 0) p.rstd[row0] = r;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const unsigned cn = (unsigned)(l + L * k) * 8;
        if (cn >= C) continue;
        const size_t at = base + umin(cn, C - 8);
        float xh[8], o[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) { xh[j] = xr[k].get(j) * r; o[j] = xh[j] * w[k].get(j); }
        if constexpr (FMT != Q_NONE) {
            float t[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) t[j] = (p.q_of_y ? o[j] : xh[j]) * inv;
            *(u32x2_a1*)(p.q + at) = q8_pack8<F, true>(t);
        }
        if (p.y) { V8<T> t; t.set(o); t.store((T*)p.y + at); }
    }
}

struct NormBwd {
    const void* h; const u8_t *q, *qe;   // h in the storage type, or xh in 8 bits
    const float* rstd; const void* dy; const void* dstream; const float* w; const float* b;
    void* dx; float* part;
    int C, HW; unsigned tiles; int relu, db;
    long long tokens; int nsplit;
    float rc, rv;                        // as in NormFwd
};

template <typename T, int SRC>
__device__ __forceinline__ float norm8_xh(const NormBwd& p, size_t i, float r, float scale) {
    if (SRC == SRC_T) return DT<T>::ld((const T*)p.h + i) * r;
    return q8_value<SRC>(p.q[i]) * scale;
}

template <typename T, int MODE, int SRC, int PX>
__global__ __launch_bounds__(256) void norm8_bwd_kernel(const NormBwd p) {
    constexpr int G = 256 / PX;
    __shared__ float red[4][PX];
    const int px = threadIdx.x % PX, g = threadIdx.x / PX;
    const unsigned n = blockIdx.x / p.tiles, hw = (blockIdx.x - n * p.tiles) * PX + px;
    const bool ok = hw < (unsigned)p.HW;
    const size_t base = (size_t)n * p.C * p.HW + (ok ? hw : 0), tok = (size_t)n * p.HW + (ok ? hw : 0);
    const T* dy = (const T*)p.dy + base;
    const size_t cs = p.HW;
    const float r = p.rstd[tok], scale = SRC == SRC_T ? 0.f : q8_scale(p.qe[tok]);
    float s1 = 0.f, s2 = 0.f;
    for (int c = g; c < p.C; c += G) {
        const float xh = norm8_xh<T, SRC>(p, base + c * cs, r, scale);
        float d = DT<T>::ld(dy + c * cs);
        if (MODE == M_CHAN && p.relu && !relu_on(fmaf(p.w[c], xh, p.b[c]))) d = 0.f;
        d *= p.w[c];
        s1 += d; s2 += d * xh;
    }
    if (MODE == M_CHAN) s1 = tok_sum<PX>(s1, red) * p.rc;
    s2 = tok_sum<PX>(s2, red) * p.rv;
    if (!ok) return;
    for (int c = g; c < p.C; c += G) {
        const float xh = norm8_xh<T, SRC>(p, base + c * cs, r, scale);
        float d = DT<T>::ld(dy + c * cs);
        if (MODE == M_CHAN && p.relu && !relu_on(fmaf(p.w[c], xh, p.b[c]))) d = 0.f;
        d = d * p.w[c] - xh * s2;
        if (MODE == M_CHAN) d -= s1;
        d *= r;
        if (MODE == M_RMS && p.dstream) d += DT<T>::ld((const T*)p.dstream + base + c * cs);
        DT<T>::st((T*)p.dx + base + c * cs, d);
    }
}

// part[split][0..2][c] = sums over the split's tokens of dy xh, dy and (db) dx as stored
template <typename T, int MODE, int SRC, int PX>
__global__ __launch_bounds__(256) void norm8_param_kernel(const NormBwd p) {
    constexpr int G = 256 / PX;
    const int px = threadIdx.x % PX, g = threadIdx.x / PX, c = blockIdx.x * G + g;
    const long long per = (p.tokens + p.nsplit - 1) / p.nsplit, lo = blockIdx.y * per, hi = lo + per < p.tokens ? lo + per : p.tokens;
    float sg = 0.f, sb = 0.f, sd = 0.f;
    if (c < p.C)
        for (long long t = lo + px; t < hi; t += PX) {
            const long long n = t / p.HW;
            const size_t i = ((size_t)n * p.C + c) * p.HW + (t - n * p.HW);
            const float xh = norm8_xh<T, SRC>(p, i, p.rstd[t], SRC == SRC_T ? 0.f : q8_scale(p.qe[t]));
            float d = DT<T>::ld((const T*)p.dy + i);
            if (MODE == M_CHAN && p.relu && !relu_on(fmaf(p.w[c], xh, p.b[c]))) d = 0.f;
            sg += d * xh; sb += d;
            if (MODE == M_CHAN && p.db) sd += DT<T>::ld((const T*)p.dx + i);
        }
#pragma unroll
    for (int o = PX >> 1; o > 0; o >>= 1) {
        sg += __shfl_xor(sg, o, 64);
        if (MODE == M_CHAN) { sb += __shfl_xor(sb, o, 64); sd += __shfl_xor(sd, o, 64); }
    }
    if (px == 0 && c < p.C) {
        float* out = p.part + (size_t)blockIdx.y * (MODE == M_RMS ? 1 : 2 + p.db) * p.C + c;
        out[0] = sg;
        if (MODE == M_CHAN) { out[p.C] = sb; if (p.db) out[2 * p.C] = sd; }
    }
}

// Planes: as norm8_fwd_tile_kernel.  A workgroup takes `pit` tiles of one image in turn and keeps the sums of its channels in
// registers: part[workgroup][0..2][c] as norm8_param_kernel.
template <typename T, int MODE, int SRC, int LPX, int CPT>
__global__ __launch_bounds__(256, 2) void norm8_bwd_tile_kernel(const NormBwd p, unsigned blocks, unsigned pit) {
    constexpr int SUBS = 64 / LPX, G = 4 * SUBS, TP = LPX * 8;
    __shared__ float red[2][4][TP], st[2][TP];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, pl = lane % LPX, g = wave * SUBS + lane / LPX;
    const unsigned per = (p.tiles + pit - 1) / pit;                  // workgroups per image
    const unsigned bid = xcd_block(blockIdx.x, blocks), n = bid / per, t0 = (bid - n * per) * pit;
    const unsigned octs = ((unsigned)p.HW + 7) >> 3;
    const unsigned kst = (unsigned)G * p.HW;                         // channel k of this lane: img + off + k * kst
    const size_t img = (size_t)n * p.C * p.HW;
    float w[CPT], b[MODE == M_CHAN ? CPT : 1], pg[CPT], pb[MODE == M_CHAN ? CPT : 1], pd[MODE == M_CHAN ? CPT : 1];
#pragma unroll
    for (int k = 0; k < CPT; ++k) {
        const int c = g + G * k, ci = c < p.C ? c : 0;
        w[k] = p.w[ci]; pg[k] = 0.f;
        if constexpr (MODE == M_CHAN) { b[k] = p.b[ci]; pb[k] = 0.f; pd[k] = 0.f; }
    }
    for (unsigned it = 0; it < pit && t0 + it < p.tiles; ++it) {
        const unsigned oct = (t0 + it) * LPX + pl;
        const bool ok = oct < octs;
        const unsigned hw0 = umin(ok ? oct * 8 : 0u, (unsigned)p.HW - 8);
        const int dup = ok ? (int)(oct * 8 - hw0) : 8;               // values that another lane adds to the channels' sums
        const unsigned off = (unsigned)g * p.HW + hw0;
        const size_t tok = (size_t)n * p.HW + hw0;
        V8<T> dy[CPT], hr[SRC == SRC_T ? CPT : 1], ds[MODE == M_RMS ? CPT : 1];
        u32x2_t q[SRC == SRC_T ? 1 : CPT];
#pragma unroll
        for (int k = 0; k < CPT; ++k) {
            const unsigned o = g + G * k < p.C ? off + k * kst : hw0, oT = o * (unsigned)sizeof(T);
            if constexpr (SRC == SRC_T) hr[k].load(at((const T*)p.h + img, oT));
            else q[k] = *(const u32x2_a1*)at(p.q + img, o);
            dy[k].load(at((const T*)p.dy + img, oT));
            if constexpr (MODE == M_RMS) if (p.dstream) ds[k].load(at((const T*)p.dstream + img, oT));
        }
        V8<float> r; r.load(p.rstd + tok);
        float sc[8], s128[8];
        if constexpr (SRC != SRC_T) q8_scales<SRC>(*(const u32x2_a1*)(p.qe + tok), sc, s128);
        auto values = [&](int k, float* xh) {
            if constexpr (SRC == SRC_T) {
#pragma unroll
                for (int j = 0; j < 8; ++j) xh[j] = hr[k].get(j) * r.get(j);
            } else q8_unpack8<SRC>(q[k], sc, s128, xh);
        };
        float s1[8], s2[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) { s1[j] = 0.f; s2[j] = 0.f; }
        auto sums = [&](auto moved) {    // moved: this lane's group was moved back at the plane's end, or is not there
#pragma unroll
            for (int k = 0; k < CPT; ++k) {
                if (g + G * k >= p.C) continue;
                float xh[8];
                values(k, xh);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    float d = dy[k].get(j);
                    if (MODE == M_CHAN && p.relu && !relu_on(fmaf(w[k], xh[j], b[MODE == M_CHAN ? k : 0]))) d = 0.f;
                    const float dk = decltype(moved)::value && j < dup ? 0.f : d;
                    pg[k] += dk * xh[j];
                    if constexpr (MODE == M_CHAN) pb[k] += dk;
                    d *= w[k];
                    if (MODE == M_CHAN) s1[j] += d;
                    s2[j] += d * xh[j];
                }
            }
        };
        if (__any(dup != 0)) sums(std::true_type{}); else sums(std::false_type{});
        // the second pass unpacks again: kept unpacked, the values of more than two channels would cost waves
        if constexpr (CPT > 2)
#pragma unroll
        for (int k = 0; k < CPT; ++k) { dy[k].forget(); if constexpr (SRC == SRC_T) hr[k].forget(); else forget(q[k]); }
        tile_reduce<LPX, false>(s2, red[1][wave]);
        if (MODE == M_CHAN) tile_reduce<LPX, false>(s1, red[0][wave]);
        __syncthreads();
        if (tid < TP) {
            st[1][tid] = ((red[1][0][tid] + red[1][1][tid]) + (red[1][2][tid] + red[1][3][tid])) * p.rv;
            if (MODE == M_CHAN) st[0][tid] = ((red[0][0][tid] + red[0][1][tid]) + (red[0][2][tid] + red[0][3][tid])) * p.rc;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 8; ++j) { s2[j] = st[1][pl * 8 + j]; if (MODE == M_CHAN) s1[j] = st[0][pl * 8 + j]; }
#pragma unroll
        for (int k = 0; k < CPT; ++k) {
            const int c = g + G * k;
            if (c >= p.C) continue;
            float xh[8], o[8];
            values(k, xh);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float d = dy[k].get(j);
                if (MODE == M_CHAN && p.relu && !relu_on(fmaf(w[k], xh[j], b[MODE == M_CHAN ? k : 0]))) d = 0.f;
                d = d * w[k] - xh[j] * s2[j];
                if (MODE == M_CHAN) d -= s1[j];
                o[j] = d * r.get(j);
                if constexpr (MODE == M_RMS) if (p.dstream) o[j] += ds[k].get(j);
            }
            V8<T> t; t.set(o);
            if (ok) t.store(at((T*)p.dx + img, (off + k * kst) * (unsigned)sizeof(T)));
            if constexpr (MODE == M_CHAN)
                if (p.db)
#pragma unroll
                    for (int j = 0; j < 8; ++j) pd[k] += j >= dup ? t.get(j) : 0.f;      // what the tensor holds
        }
    }
    float* part = p.part + (size_t)bid * (MODE == M_RMS ? 1 : 2 + p.db) * p.C;
#pragma unroll
    for (int k = 0; k < CPT; ++k) {
        const int c = g + G * k;
#pragma unroll
        for (int o = LPX >> 1; o > 0; o >>= 1) {
            pg[k] += __shfl_xor(pg[k], o, 64);
            if constexpr (MODE == M_CHAN) { pb[k] += __shfl_xor(pb[k], o, 64); pd[k] += __shfl_xor(pd[k], o, 64); }
        }
        if (pl == 0 && c < p.C) {
            part[c] = pg[k];
            if constexpr (MODE == M_CHAN) { part[p.C + c] = pb[k]; if (p.db) part[2 * p.C + c] = pd[k]; }
        }
    }
}

// Rows: a workgroup takes every gridDim.x-th group of 256 / L rows and keeps the sums of its channels in registers.
template <typename T, int SRC, int L, int K>
__global__ __launch_bounds__(256) void rms_bwd_rows_kernel(const NormBwd p, int N) {
    constexpr int R = 256 / L;
    __shared__ float red[R][L][8];
    const int l = threadIdx.x % L, rg = threadIdx.x / L;
    const unsigned C = p.C;
    V8<float> w[K];
    float pg[K][8];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        w[k].load(p.w + umin((unsigned)(l + L * k) * 8, C - 8));
#pragma unroll
        for (int j = 0; j < 8; ++j) pg[k][j] = 0.f;
    }
    for (long long r0 = (long long)blockIdx.x * R; r0 < N; r0 += (long long)gridDim.x * R) {
        const bool ok = r0 + rg < N;
        const long long row = ok ? r0 + rg : N - 1;
        const size_t base = (size_t)row * C;
        V8<T> dy[K], hr[SRC == SRC_T ? K : 1], ds[K];
        u32x2_t q[SRC == SRC_T ? 1 : K];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const size_t at = base + umin((unsigned)(l + L * k) * 8, C - 8);
            if constexpr (SRC == SRC_T) hr[k].load((const T*)p.h + at); else q[k] = *(const u32x2_a1*)(p.q + at);
            dy[k].load((const T*)p.dy + at);
            if (p.dstream) ds[k].load((const T*)p.dstream + at);
        }
        const float r = p.rstd[row];
        float sc[8], s128[8];
        if constexpr (SRC != SRC_T) { const unsigned e = 0x01010101u * p.qe[row]; q8_scales<SRC>(u32x2_t{e, e}, sc, s128); }
        auto values = [&](int k, float* xh) {
            if constexpr (SRC == SRC_T) {
#pragma unroll
                for (int j = 0; j < 8; ++j) xh[j] = hr[k].get(j) * r;
            } else q8_unpack8<SRC>(q[k], sc, s128, xh);
        };
        float s2 = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const unsigned cn = (unsigned)(l + L * k) * 8, c = umin(cn, C - 8);
            float xh[8];
            values(k, xh);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float d = c + j >= cn ? dy[k].get(j) * xh[j] : 0.f;
                pg[k][j] += ok ? d : 0.f;
                s2 += d * w[k].get(j);
            }
        }
        s2 = row_sum<L>(s2) * p.rv;
        if (!ok) continue;               // (only the last round has rows that are not there, and none of its lanes waits again)
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const unsigned cn = (unsigned)(l + L * k) * 8;
            if (cn >= C) continue;
            float xh[8], o[8];
            values(k, xh);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                o[j] = (dy[k].get(j) * w[k].get(j) - xh[j] * s2) * r;
                if (p.dstream) o[j] += ds[k].get(j);
            }
            V8<T> t; t.set(o);
            t.store((T*)p.dx + base + umin(cn, C - 8));
        }
    }
    float* part = p.part + (size_t)blockIdx.x * C;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const unsigned cn = (unsigned)(l + L * k) * 8, c = umin(cn, C - 8);
        if (R > 1) {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < 8; ++j) red[rg][l][j] = pg[k][j];
            __syncthreads();
            if (rg != 0) continue;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float s = 0.f;
                for (int i = 0; i < R; ++i) s += red[i][l][j];
                pg[k][j] = s;
            }
        }
        if (cn < C)
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c + j >= cn) part[c + j] = pg[k][j];
    }
}

// column sums of part[rows][nr * C] into up to three vectors, each written or added to, in a fixed order: 16 columns x 64 row
// lanes per workgroup (a few hundred columns of ~1000 rows: more row lanes, so that no thread adds more than a few dozen)
__global__ __launch_bounds__(1024) void norm8_colsum_kernel(const float* __restrict__ part, float* __restrict__ d0, float* __restrict__ d1,
                                                            float* __restrict__ d2, int C, int rows, int nr, int acc, int acc2) {
    __shared__ float red[64][17];
    const int cl = threadIdx.x & 15, col = blockIdx.x * 16 + cl, rl = threadIdx.x >> 4, W = nr * C;
    float s = 0.f;
    if (col < W) {
        int r = rl;
        for (; r + 448 < rows; r += 512) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = part[(size_t)(r + 64 * j) * W + col];
            s += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
        }
        for (; r < rows; r += 64) s += part[(size_t)r * W + col];
    }
    red[rl][cl] = s;
    __syncthreads();
    if (threadIdx.x < 64) {
        const int c = threadIdx.x & 15, q = threadIdx.x >> 4;
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) t += red[q * 16 + i][c];
        t += __shfl_xor(t, 16, 64);
        t += __shfl_xor(t, 32, 64);
        if (q == 0 && col < W) {
            float* d = col < C ? d0 + col : (col < 2 * C ? d1 + (col - C) : d2 + (col - 2 * C));
            if (col < 2 * C ? acc : acc2) *d += t; else *d = t;
        }
    }
}

namespace {
int norm8_px(int HW) { return HW == 1 ? 1 : (HW < 48 ? 16 : 64); }
int norm8_nsplit(int N, int C, int HW) {                             // ~1024 workgroups, at least 64 tokens each
    const int px = norm8_px(HW), cb = cdiv(C, 256 / px);
    const long long tokens = (long long)N * HW, most = cdivl(tokens, 64);
    long long s = cdiv(1024, cb);
    if (s > most) s = most;
    return (int)(s < 1 ? 1 : s);
}
// tiles per workgroup of the backward plane kernel: 512 workgroups, two per CU (what its registers allow), each with its share of
// the tiles - one round, few rows of channel sums (16x120x128x128: 43 us, with 1024 workgroups 47.5, with 2048 53)
unsigned norm8_pit(const TileCfg& t, long long N) {
    unsigned pit = (unsigned)(t.blocks / 512);
    return pit < 1 ? 1 : (pit > t.tiles ? t.tiles : pit);
}
// channels per thread that the plane kernels keep in registers
template <typename T> constexpr int tile_most() { return sizeof(T) == 2 ? 8 : 4; }
// rows of channel sums that the backward pass writes
template <typename T>
size_t norm8_rows(int mode, int N, int C, int HW) {
    if (HW >= 8) {
        const TileCfg t = tile_pick(N, C, HW, tile_most<T>());
        if (t.lpx) return (size_t)cdiv((int)t.tiles, (int)norm8_pit(t, N)) * N;
    }
    if (mode == M_RMS && HW == 1 && C >= 8) {
        const RowCfg r = row_pick(N, C);
        if (r.l) { const int g = cdiv(N, 256 / r.l); return (size_t)(g < 1024 ? g : 1024); }
    }
    return (size_t)norm8_nsplit(N, C, HW);
}

template <typename T, int MODE, int FMT>
int norm8_fwd_launch(NormFwd& p, int N, hipStream_t st) {
    p.rc = 1.f / (float)p.C;
    p.rv = 1.f / (float)(MODE == M_RMS ? p.C : p.C - 1);
    if (p.HW >= 8) {
        const TileCfg t = tile_pick(N, p.C, p.HW, tile_most<T>());
        if (t.lpx) {
            if (t.blocks > 0x7fffffffll) return HIFIC_ERR_UNSUPPORTED;
            p.tiles = t.tiles;
#define FWD(LPX, CPT) hipLaunchKernelGGL((norm8_fwd_tile_kernel<T, MODE, FMT, LPX, CPT>), dim3((unsigned)t.blocks), dim3(256), 0, st, p, (unsigned)t.blocks)
            TILE_DISPATCH(t, tile_most<T>(), FWD);
#undef FWD
            return hific_launch_status();
        }
    }
    if constexpr (MODE == M_RMS) {
        RowCfg r;
        if (p.HW == 1 && p.C >= 8 && (r = row_pick(N, p.C)).l) {
#define ROWS(L, K) hipLaunchKernelGGL((rms_fwd_rows_kernel<T, FMT, L, K>), dim3(cdiv(N, 256 / L)), dim3(256), 0, st, p, N)
            ROW_DISPATCH(r, ROWS)
#undef ROWS
            return hific_launch_status();
        }
    }
    const int px = norm8_px(p.HW);
    const long long blocks = cdivl(p.HW, px) * N;
    if (blocks > 0x7fffffffll) return HIFIC_ERR_UNSUPPORTED;
    p.tiles = (unsigned)cdivl(p.HW, px);
    const dim3 grid((unsigned)blocks);
    if (px == 1) hipLaunchKernelGGL((norm8_fwd_kernel<T, MODE, FMT, 1>), grid, dim3(256), 0, st, p);
    else if (px == 16) hipLaunchKernelGGL((norm8_fwd_kernel<T, MODE, FMT, 16>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((norm8_fwd_kernel<T, MODE, FMT, 64>), grid, dim3(256), 0, st, p);
    return hific_launch_status();
}

template <typename T, int MODE, int SRC>
int norm8_bwd_launch(NormBwd& p, int N, float* d0, float* d1, float* d2, int acc, int acc2, size_t ws_bytes, hipStream_t st) {
    p.rc = 1.f / (float)p.C;
    p.rv = 1.f / (float)(MODE == M_RMS ? p.C : p.C - 1);
    const int nr = MODE == M_RMS ? 1 : 2 + p.db;
    const size_t rows = norm8_rows<T>(MODE, N, p.C, p.HW);
    if (rows * nr * p.C * sizeof(float) > ws_bytes) return HIFIC_ERR_WS;
    TileCfg t{0, 0, 0, 0};
    RowCfg r{0, 0};
    if (p.HW >= 8) t = tile_pick(N, p.C, p.HW, tile_most<T>());
    else if (MODE == M_RMS && p.HW == 1 && p.C >= 8) r = row_pick(N, p.C);
    if (rows > 0x7fffffffull) return HIFIC_ERR_UNSUPPORTED;
    if (t.lpx) {
        p.tiles = t.tiles;
        const unsigned pit = norm8_pit(t, N);
#define BWD(LPX, CPT) hipLaunchKernelGGL((norm8_bwd_tile_kernel<T, MODE, SRC, LPX, CPT>), dim3((unsigned)rows), dim3(256), 0, st, p, (unsigned)rows, pit)
        TILE_DISPATCH(t, tile_most<T>(), BWD);
#undef BWD
    } else if (r.l) {
        if constexpr (MODE == M_RMS) {
#define ROWS(L, K) hipLaunchKernelGGL((rms_bwd_rows_kernel<T, SRC, L, K>), dim3((unsigned)rows), dim3(256), 0, st, p, N)
            ROW_DISPATCH(r, ROWS)
#undef ROWS
        }
    } else {
        const int px = norm8_px(p.HW);
        const long long blocks = cdivl(p.HW, px) * N;
        if (blocks > 0x7fffffffll) return HIFIC_ERR_UNSUPPORTED;
        p.tiles = (unsigned)cdivl(p.HW, px);
        p.tokens = (long long)N * p.HW;
        p.nsplit = (int)rows;
        const dim3 grid((unsigned)blocks), pgrid(cdiv(p.C, 256 / px), p.nsplit);
#define BWD(PX)                                                                                                 \
        do {                                                                                                    \
            hipLaunchKernelGGL((norm8_bwd_kernel<T, MODE, SRC, PX>), grid, dim3(256), 0, st, p);               \
            hipLaunchKernelGGL((norm8_param_kernel<T, MODE, SRC, PX>), pgrid, dim3(256), 0, st, p);            \
        } while (0)
        if (px == 1) BWD(1); else if (px == 16) BWD(16); else BWD(64);
#undef BWD
    }
    hipLaunchKernelGGL(norm8_colsum_kernel, dim3(cdiv(nr * p.C, 16)), dim3(1024), 0, st, p.part, d0, d1, d2, p.C, (int)rows, nr, acc, acc2);
    return hific_launch_status();
}
}  // namespace

extern "C" {

int hific_rms_norm_fwd(const void* x, const void* resid, const float* w, void* y, void* h, float* rstd, void* q, void* qe,
                       int fmt, int q_of_y, int N, int C, int HW, float eps, int dtype, hipStream_t st) {
    if (!x || !w || N <= 0 || C <= 0 || HW <= 0 || !act8_dtype_ok(dtype) || !(eps > 0.f)) return HIFIC_ERR_ARG;
    if ((resid != nullptr) != (h != nullptr) || (q != nullptr) != (qe != nullptr) || (!y && !q)) return HIFIC_ERR_ARG;
    if (q && !act8_fmt_ok(fmt)) return HIFIC_ERR_ARG;
    NormFwd p{x, resid, w, nullptr, y, h, rstd, (u8_t*)q, (u8_t*)qe, nullptr, nullptr, C, HW, 0, eps, 0, q_of_y, 0.f, 0.f};
#define RMS(T) (!q ? norm8_fwd_launch<T, M_RMS, Q_NONE>(p, N, st) : fmt == HIFIC_Q_INT8                                     \
                   ? norm8_fwd_launch<T, M_RMS, HIFIC_Q_INT8>(p, N, st) : norm8_fwd_launch<T, M_RMS, HIFIC_Q_E4M3>(p, N, st))
    return dtype == HIFIC_F32 ? RMS(float) : RMS(bf16_t);
#undef RMS
}

size_t hific_norm8_bwd_ws_bytes(int N, int C, int HW) {
    if (N <= 0 || C <= 0 || HW <= 0) return 0;
    size_t rows = 0;
    for (int mode : {M_RMS, M_CHAN}) {
        const size_t a = norm8_rows<float>(mode, N, C, HW), b = norm8_rows<bf16_t>(mode, N, C, HW);
        rows = a > rows ? a : rows;
        rows = b > rows ? b : rows;
    }
    return rows * 3 * C * sizeof(float);
}

int hific_rms_norm_bwd(const void* h, const void* q, const void* qe, int fmt, const float* rstd, const void* dy, const void* dstream,
                       const float* w, void* dx, float* dw, int accumulate, int N, int C, int HW, int dtype, void* ws, size_t ws_bytes,
                       hipStream_t st) {
    if (!rstd || !dy || !w || !dx || !dw || !ws || N <= 0 || C <= 0 || HW <= 0 || !act8_dtype_ok(dtype)) return HIFIC_ERR_ARG;
    if ((h != nullptr) == (q != nullptr) || (q != nullptr) != (qe != nullptr) || (q && !act8_fmt_ok(fmt))) return HIFIC_ERR_ARG;
    NormBwd p{h, (const u8_t*)q, (const u8_t*)qe, rstd, dy, dstream, w, nullptr, dx, (float*)ws, C, HW, 0, 0, 0, 0, 0, 0.f, 0.f};
#define RMS(T) (h ? norm8_bwd_launch<T, M_RMS, SRC_T>(p, N, dw, nullptr, nullptr, accumulate, 0, ws_bytes, st)              \
                  : fmt == HIFIC_Q_INT8                                                                                     \
                  ? norm8_bwd_launch<T, M_RMS, HIFIC_Q_INT8>(p, N, dw, nullptr, nullptr, accumulate, 0, ws_bytes, st)       \
                  : norm8_bwd_launch<T, M_RMS, HIFIC_Q_E4M3>(p, N, dw, nullptr, nullptr, accumulate, 0, ws_bytes, st))
    return dtype == HIFIC_F32 ? RMS(float) : RMS(bf16_t);
#undef RMS
}

int hific_channelnorm8_fwd(const void* x, const float* gamma, const float* beta, const void* resid, void* y, float* rstd, void* q,
                           void* qe, void* q2, void* qe2, int fmt, int N, int C, int HW, float eps, int relu, int dtype, hipStream_t st) {
    if (!x || !gamma || !beta || !y || !rstd || !q || !qe || N <= 0 || C < 2 || HW <= 0 || !(eps > 0.f)) return HIFIC_ERR_ARG;
    if (!act8_dtype_ok(dtype) || !act8_fmt_ok(fmt)) return HIFIC_ERR_ARG;
    if ((q2 != nullptr) != (qe2 != nullptr) || (q2 && !resid)) return HIFIC_ERR_ARG;
    NormFwd p{x, resid, gamma, beta, y, nullptr, rstd, (u8_t*)q, (u8_t*)qe, (u8_t*)q2, (u8_t*)qe2, C, HW, 0, eps, relu, 0, 0.f, 0.f};
#define CN(T) (fmt == HIFIC_Q_INT8 ? norm8_fwd_launch<T, M_CHAN, HIFIC_Q_INT8>(p, N, st) : norm8_fwd_launch<T, M_CHAN, HIFIC_Q_E4M3>(p, N, st))
    return dtype == HIFIC_F32 ? CN(float) : CN(bf16_t);
#undef CN
}

int hific_channelnorm8_bwd(const void* q, const void* qe, int fmt, const float* rstd, const void* dy, const float* gamma,
                           const float* beta, void* dx, float* dgamma, float* dbeta, int accumulate, float* dprev_bias,
                           int accumulate_prev, int N, int C, int HW, int relu, int dtype, void* ws, size_t ws_bytes, hipStream_t st) {
    if (!q || !qe || !rstd || !dy || !gamma || !beta || !dx || !dgamma || !dbeta || !ws || N <= 0 || C < 2 || HW <= 0) return HIFIC_ERR_ARG;
    if (!act8_dtype_ok(dtype) || !act8_fmt_ok(fmt)) return HIFIC_ERR_ARG;
    NormBwd p{nullptr, (const u8_t*)q, (const u8_t*)qe, rstd, dy, nullptr, gamma, beta, dx, (float*)ws, C, HW, 0, relu,
              dprev_bias ? 1 : 0, 0, 0, 0.f, 0.f};
#define CN(T) (fmt == HIFIC_Q_INT8                                                                                                       \
                   ? norm8_bwd_launch<T, M_CHAN, HIFIC_Q_INT8>(p, N, dgamma, dbeta, dprev_bias, accumulate, accumulate_prev, ws_bytes, st) \
                   : norm8_bwd_launch<T, M_CHAN, HIFIC_Q_E4M3>(p, N, dgamma, dbeta, dprev_bias, accumulate, accumulate_prev, ws_bytes, st))
    return dtype == HIFIC_F32 ? CN(float) : CN(bf16_t);
#undef CN
}

}  // extern "C"
