// Forward passes of the norms of norm8.h.
#include "norm8.h"

struct NormFwd {
    const void* x; const void* resid; const float* w; const float* b;
    void* y; void* h; float* rstd;
    u8_t *q, *qe, *q2, *qe2;             // xh (RMS with q_of_y: y) and, with a channel norm's resid, y
    int C, HW; unsigned tiles; float eps; int relu, q_of_y;
    float nc, nv;                        // C, and C or C - 1: divisors (a product with a rounded 1 / C would miss the mean of equal terms)
};

// r of a token whose sum of squares left float32 (values above about 1e19), d(c) its values: the sum again in 64 bits.  One lane walks
// the channels: such tokens are rare, and the kernels keep no register for them.  0 where a value is infinite: it becomes NaN
// (infinity * 0) and the others 0, as in the formula.
template <typename D>
__device__ float norm8_r_far(D d, int C, float nv, float eps) {
    double ss = 0.;
#pragma unroll 1
    for (int c = 0; c < C; ++c) { const double v = d(c); ss += v * v; }
    return (float)(1. / sqrt(ss / nv + eps));
}
__device__ __forceinline__ float norm8_r(float ss, float nv, float eps) { return rsqrtf(ss / nv + eps); }
// max|d w| r does not give the exponent of y = (d r) w where d * w left the range of float32 or lost its bits below it
__device__ __forceinline__ bool norm8_far(float m, float ss) { return m == INFINITY || (m < 0x1p-100f && ss > 0.f); }

// Any shape: PX lanes on consecutive tokens x 256 / PX channel groups, the tensor re-read by every pass (from L2).  Chains of loads
// bound it: channel norm 16x960x2x2 39 us, 16x960x2x3 44, 2x4500x16x16 232 (2x3000x32x32 250, which the tiles below take in 17).
template <typename T, int MODE, int FMT, int PX>
__global__ __launch_bounds__(256) void norm8_fwd_kernel(const NormFwd p, long long tokens) {
    constexpr int G = 256 / PX;
    constexpr int F = FMT == Q_NONE ? HIFIC_Q_INT8 : FMT;
    __shared__ float red[4][PX];
    const int px = threadIdx.x % PX, g = threadIdx.x / PX;
    const size_t cs = p.HW;
    for (long long t0 = (long long)blockIdx.x * PX; t0 < tokens; t0 += (long long)gridDim.x * PX) {
        const bool ok = t0 + px < tokens;
        const long long tok = ok ? t0 + px : tokens - 1, n = tok / p.HW;
        const size_t base = (size_t)n * p.C * p.HW + (size_t)(tok - n * p.HW);
        const T* x = (const T*)p.x + base;
        const T* rs = p.resid ? (const T*)p.resid + base : nullptr;
        T* y = p.y ? (T*)p.y + base : nullptr;
        T* h = p.h ? (T*)p.h + base : nullptr;
        auto stream = [&](int c) {
            float v = DT<T>::ld(x + c * cs);
            if (MODE == M_RMS && rs) { T o; DT<T>::st(&o, v + DT<T>::ld(rs + c * cs)); v = DT<T>::ld(&o); }
            return v;
        };
        float mu = 0.f;
        if (MODE == M_CHAN) {
            float s = 0.f;
            for (int c = g; c < p.C; c += G) s += stream(c);
            mu = tok_sum<PX>(s, red) / p.nc;
        }
        float ss = 0.f;
        for (int c = g; c < p.C; c += G) {
            const float v = stream(c), d = v - mu;
            ss += d * d;
            if (MODE == M_RMS && h && ok) DT<T>::st(h + c * cs, v);
        }
        ss = tok_sum<PX>(ss, red);
        float r = norm8_r(ss, p.nv, p.eps);
        if (ss == INFINITY) r = norm8_r_far([&](int c) { return stream(c) - mu; }, p.C, p.nv, p.eps);
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
                                                                     : q8_round<F>((MODE == M_RMS && p.q_of_y ? q8_top<F>(o) : xh) * inv));
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
                if (ok) p.q2[base + c * cs] = (u8_t)q8_round<F>(q8_top<F>(o) * inv2);
            }
        }
    }
}

// Planes of eight positions and more: a workgroup owns LPX * 8 positions x all channels (tile_pick), eight positions and CPT
// channels per lane, kept as they were loaded between the passes: every tensor crosses HBM once, and that bounds it.  us (TB/s): channel
// norm + ReLU 16x60x256x256 70.5 (4.5), 16x120x128x128 38.6 (4.1), 16x960x16x16 8.8 (2.2: the latency of three dependent passes), with
// a residual and its second 8-bit form 107.6 (4.7), 52.4 (4.8), 11.5 (2.7); root-mean-square norm with residual 108.1 (4.7), 53.4 (4.7),
// 8.8 (3.6), with its normalised form kept 122.6 (4.6), 62.9 (4.5), 10.4 (3.4).
template <typename T, int MODE, int FMT, bool RES, int LPX, int CPT, int NW>
__global__ __launch_bounds__(64 * NW, 2) void norm8_fwd_tile_kernel(const NormFwd p, unsigned blocks) {
    constexpr int SUBS = 64 / LPX, G = NW * SUBS, TP = LPX * 8;
    constexpr int F = FMT == Q_NONE ? HIFIC_Q_INT8 : FMT;
    __shared__ float red[NW][TP], redm[NW][TP];
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
    const T *x = (const T*)p.x + img, *rs = RES ? (const T*)p.resid + img : nullptr;
    V8<T> xr[CPT], rr[RES ? CPT : 1];
    float w[CPT], b[MODE == M_CHAN ? CPT : 1];
#pragma unroll
    for (int k = 0; k < CPT; ++k) {
        const int c = g + G * k < p.C ? g + G * k : 0;               // (a load of channel 0 in the place of a branch around it)
        const unsigned o = (c == 0 ? off0 : off + k * kst) * (unsigned)sizeof(T);
        xr[k].load(at(x, o));
        w[k] = p.w[c];
        if constexpr (MODE == M_CHAN) b[k] = p.b[c];
        if constexpr (RES) rr[k].load(at(rs, o));
    }
    if constexpr (MODE == M_RMS && RES) {
#pragma unroll
        for (int k = 0; k < CPT; ++k) {
            float h[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) h[j] = xr[k].get(j) + rr[k].get(j);
            xr[k].set(h);
            if (ok && g + G * k < p.C) xr[k].store(at((T*)p.h + img, (off + k * kst) * (unsigned)sizeof(T)));
        }
    }
    // maxima as floats, NaN included: r carries one of x into the exponent, but not one of a weight (or of infinity times a zero weight)
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
        if (tid < TP) st_r[tid] = waves_sum<NW, TP>(red, tid) / p.nc;
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
                if (FMT != Q_NONE) am[j] = nmax(am[j], fabsf(MODE == M_RMS && p.q_of_y ? d * w[k] : d));
            }
#pragma unroll
    for (int k = 0; k < CPT; ++k) xr[k].forget();
    tile_reduce<LPX, false>(acc, red[wave]);
    if (FMT != Q_NONE) tile_reduce<LPX, true>(am, redm[wave]);
    __syncthreads();
    if (tid < TP) {
        const float ss = waves_sum<NW, TP>(red, tid);
        const unsigned at0 = umin(so * 8, (unsigned)p.HW - 8) + (tid & 7);       // (of the last tile's lanes past the plane: some position of it)
        auto dev = [&](int c) {
            const size_t i = at0 + (size_t)c * p.HW;
            float v = DT<T>::ld(x + i);
            if (MODE == M_CHAN) return v - st_r[tid];
            if (RES) { T o; DT<T>::st(&o, v + DT<T>::ld(rs + i)); v = DT<T>::ld(&o); }
            return v;
        };
        float r = norm8_r(ss, p.nv, p.eps);
        if (ss == INFINITY) r = norm8_r_far(dev, p.C, p.nv, p.eps);
        if (FMT != Q_NONE) {
            // max|d| r = max|d r|: a rounded product is monotone (with q_of_y the weight comes between, and q8_pack8 clamps)
            const float m = waves_max<NW, TP>(redm, tid);
            float top = m * r;
            if (MODE == M_RMS && p.q_of_y && norm8_far(m, ss)) {
                top = 0.f;
#pragma unroll 1
                for (int c = 0; c < p.C; ++c) top = nmax(top, fabsf(dev(c) * r * p.w[c]));
            }
            const unsigned code = q8_code<F>(abs_bits(top));
            st_inv[tid] = q8_inv_scale(code);
            if (sok) p.qe[stok] = (u8_t)code;
        }
        st_r[tid] = r;
        if (p.rstd && sok) p.rstd[stok] = r;
    }
    __syncthreads();
    // (xh / scale in two products: r / scale overflows where a token's values are all alike or nearly so)
    float r[8], inv[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) { r[j] = st_r[pl * 8 + j]; inv[j] = FMT != Q_NONE ? st_inv[pl * 8 + j] : 0.f; am[j] = 0.f; }
#pragma unroll
    for (int k = 0; k < CPT; ++k) {
        const int c = g + G * k;
        if (c >= p.C) continue;
        float o[8], xh[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            xh[j] = (xr[k].get(j) - mu[j]) * r[j];
            o[j] = MODE == M_RMS ? xh[j] * w[k] : fmaf(w[k], xh[j], b[MODE == M_CHAN ? k : 0]);
        }
        if constexpr (FMT != Q_NONE) {
            float t[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) t[j] = (MODE == M_RMS && p.q_of_y ? q8_top<F>(o[j]) : xh[j]) * inv[j];
            u32x2_t q;
            if (MODE == M_CHAN && p.relu) {
                float gs[8];             // gamma * scale; the scale 1 / inv is a power of two (2^127 for a token that is not finite: its values are NaN)
#pragma unroll
                for (int j = 0; j < 8; ++j) gs[j] = w[k] * __uint_as_float(0x7f000000u - __float_as_uint(inv[j]));
                q = q8_pack8_masked<F>(t, o, gs, b[MODE == M_CHAN ? k : 0], w[k]);
            } else q = q8_pack8<F, MODE == M_RMS>(t);
            if (ok) *(u32x2_a1*)at(p.q + img, off + k * kst) = q;
        }
        if constexpr (MODE == M_CHAN) {
            if constexpr (RES) {         // both terms rounded to the storage type first, as norm and add one after the other
                V8<T> t; t.set(o);
#pragma unroll
                for (int j = 0; j < 8; ++j) { o[j] = t.get(j) + rr[k].get(j); if (FMT != Q_NONE) am[j] = nmax(am[j], fabsf(o[j])); }
                xr[k] = t;               // q2 below: the sum again from its two terms, in float32
            }
        }
        if (p.y && ok) { V8<T> t; t.set(o); t.store(at((T*)p.y + img, (off + k * kst) * (unsigned)sizeof(T))); }
    }
    if constexpr (MODE == M_CHAN && FMT != Q_NONE && RES) {
        if (!p.q2) return;
        tile_reduce<LPX, true>(am, redm[wave]);          // (redm's readers are behind a barrier)
        __syncthreads();
        if (tid < TP) {
            const unsigned code = q8_code<F>(abs_bits(waves_max<NW, TP>(redm, tid)));
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
            for (int j = 0; j < 8; ++j) t[j] = q8_top<F>(xr[k].get(j) + rr[k].get(j)) * st_inv[pl * 8 + j];
            *(u32x2_a1*)at(p.q2 + img, off + k * kst) = q8_pack8<F, false>(t);
        }
    }
}

// Rows of eight channels and more (root-mean-square norm): eight channels per lane, L lanes and K groups per lane for a row.  65536x960
// with residual 87 us (5.8 TB/s: part of it from the memory-side cache), 16384x4096 94 us (5.7), to 8 bits 38 and 40; one row 4.9 us (the launch).
template <typename T, int FMT, int L, int K>
__global__ __launch_bounds__(row_block(L)) void rms_fwd_rows_kernel(const NormFwd p, int N) {
    constexpr int F = FMT == Q_NONE ? HIFIC_Q_INT8 : FMT;
    const int l = threadIdx.x % L;
    const long long row0 = (long long)blockIdx.x * (row_block(L) / L) + threadIdx.x / L;
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
    float ss = 0.f, am = 0.f;            // (am keeps a NaN: it may be a weight's)
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
            if (FMT != Q_NONE) am = nmax(am, fabsf(p.q_of_y ? v * w[k].get(j) : v));
        }
    }
    // the widest rows unpack again below: kept unpacked, their values would cost a workgroup per CU (2048x16384 to 8 bits 28 us, 35)
    if constexpr (sizeof(T) == 2 && (L == 1024 || K == 4))
#pragma unroll
        for (int k = 0; k < K; ++k) xr[k].forget();
    ss = row_sum<L>(ss);
    float r = norm8_r(ss, p.nv, p.eps), m = 0.f, inv = 0.f, lim = 0.f;
    if (FMT != Q_NONE) m = __uint_as_float(row_max<L>(abs_bits(am)));
    float top = m * r;
    const bool far = ss == INFINITY || (FMT != Q_NONE && p.q_of_y && norm8_far(m, ss));
    if (__any(far)) {                    // (from memory again: such rows are rare, and the kernel keeps no register for them)
        auto value = [&](unsigned c) {
            float v = DT<T>::ld((const T*)p.x + base + c);
            if (p.resid) { T o; DT<T>::st(&o, v + DT<T>::ld((const T*)p.resid + base + c)); v = DT<T>::ld(&o); }
            return v;
        };
        // norm8_r_far by all lanes of the row: in float32, scaled by the power of two that takes the largest value to [2, 4)
        unsigned am = 0;
#pragma unroll 1
        for (unsigned c = l; c < C; c += L) am = umax(am, abs_bits(value(c)));
        am = row_max<L>(am);
        const float s = __uint_as_float(am >= 0x7f800000u ? 0u : (255u - (am >> 23)) << 23);
        float sum = 0.f;
#pragma unroll 1
        for (unsigned c = l; c < C; c += L) { const float v = value(c) * s; sum += v * v; }
        sum = row_sum<L>(sum);
        if (ss == INFINITY) r = am >= 0x7f800000u ? 0.f : s * rsqrtf(sum / p.nv + p.eps * s * s);
        if (FMT != Q_NONE) {
            float y = 0.f;
#pragma unroll 1
            for (unsigned c = l; c < C; c += L) y = nmax(y, fabsf(p.q_of_y ? value(c) * r * p.w[c] : value(c) * r));
            y = __uint_as_float(row_max<L>(abs_bits(y)));
            if (far) top = y;            // (a row's result does not depend on its neighbours)
        }
    }
    if constexpr (FMT != Q_NONE) {
        const unsigned code = q8_code<F>(abs_bits(top));
        inv = q8_inv_scale(code);
        lim = q8_limit<F>(code);
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
            for (int j = 0; j < 8; ++j) t[j] = __builtin_amdgcn_fmed3f((p.q_of_y ? o[j] : xh[j]) * inv, -lim, lim);
            *(u32x2_a1*)(p.q + at) = q8_pack8<F, false>(t);
        }
        if (p.y) { V8<T> t; t.set(o); t.store((T*)p.y + at); }
    }
}

namespace {
template <typename T>
NormFwd norm8_part(NormFwd p, long long n0) {                        // from image n0 on
    const long long i = n0 * p.C * p.HW, t = n0 * p.HW;
    p.x = (const T*)p.x + i; p.resid = ahead((const T*)p.resid, i); p.y = ahead((T*)p.y, i); p.h = ahead((T*)p.h, i);
    p.rstd = ahead(p.rstd, t);
    p.q = ahead(p.q, i); p.qe = ahead(p.qe, t); p.q2 = ahead(p.q2, i); p.qe2 = ahead(p.qe2, t);
    return p;
}
template <typename T, int MODE, int FMT>
int norm8_fwd_launch(NormFwd& p, int N, hipStream_t st) {
    p.nc = (float)p.C;
    p.nv = (float)(MODE == M_RMS ? p.C : p.C - 1);
    if (p.HW >= 8) {
        const TileCfg t = tile_pick(N, p.C, p.HW, tile_most<T>(), sizeof(T));
        if (t.lpx) {
            p.tiles = t.tiles;
            return batch_parts(N, t.tiles, [&](long long n0, long long n) {
                const NormFwd part = norm8_part<T>(p, n0);
                const dim3 grid((unsigned)(t.tiles * n));
#define FWD(LPX, CPT, NW)                                                                                                           \
                do {                                                                                                                \
                    if (p.resid) hipLaunchKernelGGL((norm8_fwd_tile_kernel<T, MODE, FMT, true, LPX, CPT, NW>), grid, dim3(64 * NW), 0, st, part, grid.x); \
                    else hipLaunchKernelGGL((norm8_fwd_tile_kernel<T, MODE, FMT, false, LPX, CPT, NW>), grid, dim3(64 * NW), 0, st, part, grid.x); \
                } while (0)
                TILE_DISPATCH(t, T, tile_most<T>(), FWD);
#undef FWD
                return hific_launch_status();
            });
        }
    }
    if constexpr (MODE == M_RMS) {
        RowCfg r;
        if (p.HW == 1 && p.C >= 8 && (r = row_pick(N, p.C)).l) {
            return batch_parts(N, 1, [&](long long n0, long long n) {
                const NormFwd part = norm8_part<T>(p, n0);
#define ROWS(L, K) hipLaunchKernelGGL((rms_fwd_rows_kernel<T, FMT, L, K>), dim3(cdiv((int)n, row_block(L) / L)), dim3(row_block(L)), 0, st, part, (int)n)
                ROW_DISPATCH(r, ROWS)
#undef ROWS
                return hific_launch_status();
            });
        }
    }
    const int px = any_px(N, p.C, p.HW);
    const long long tokens = (long long)N * p.HW;
    const dim3 grid(any_grid(cdivl(tokens, px)));
    if (px == 1) hipLaunchKernelGGL((norm8_fwd_kernel<T, MODE, FMT, 1>), grid, dim3(256), 0, st, p, tokens);
    else if (px == 16) hipLaunchKernelGGL((norm8_fwd_kernel<T, MODE, FMT, 16>), grid, dim3(256), 0, st, p, tokens);
    else hipLaunchKernelGGL((norm8_fwd_kernel<T, MODE, FMT, 64>), grid, dim3(256), 0, st, p, tokens);
    return hific_launch_status();
}
}  // namespace

extern "C" {

int hific_rms_norm_fwd(const void* x, const void* resid, const float* w, void* y, void* h, float* rstd, void* q, void* qe,
                       int fmt, int q_of_y, int N, int C, int HW, float eps, int dtype, hipStream_t st) {
    if (!x || !w || N <= 0 || C <= 0 || HW <= 0 || !act8_dtype_ok(dtype) || !(eps > 0.f)) return HIFIC_ERR_ARG;
    if ((resid != nullptr) != (h != nullptr) || (q != nullptr) != (qe != nullptr) || (!y && !q)) return HIFIC_ERR_ARG;
    if (q && !act8_fmt_ok(fmt)) return HIFIC_ERR_ARG;
    if (C > ACT8_MAX_C) return HIFIC_ERR_UNSUPPORTED;
    NormFwd p{x, resid, w, nullptr, y, h, rstd, (u8_t*)q, (u8_t*)qe, nullptr, nullptr, C, HW, 0, eps, 0, q_of_y, 0.f, 0.f};
#define RMS(T) (!q ? norm8_fwd_launch<T, M_RMS, Q_NONE>(p, N, st) : fmt == HIFIC_Q_INT8                                     \
                   ? norm8_fwd_launch<T, M_RMS, HIFIC_Q_INT8>(p, N, st) : norm8_fwd_launch<T, M_RMS, HIFIC_Q_E4M3>(p, N, st))
    return dtype == HIFIC_F32 ? RMS(float) : RMS(bf16_t);
#undef RMS
}

int hific_channelnorm8_fwd(const void* x, const float* gamma, const float* beta, const void* resid, void* y, float* rstd, void* q,
                           void* qe, void* q2, void* qe2, int fmt, int N, int C, int HW, float eps, int relu, int dtype, hipStream_t st) {
    if (!x || !gamma || !beta || !y || !rstd || !q || !qe || N <= 0 || C < 2 || HW <= 0 || !(eps > 0.f)) return HIFIC_ERR_ARG;
    if (!act8_dtype_ok(dtype) || !act8_fmt_ok(fmt)) return HIFIC_ERR_ARG;
    if ((q2 != nullptr) != (qe2 != nullptr) || (q2 && !resid)) return HIFIC_ERR_ARG;
    if (C > ACT8_MAX_C) return HIFIC_ERR_UNSUPPORTED;
    NormFwd p{x, resid, gamma, beta, y, nullptr, rstd, (u8_t*)q, (u8_t*)qe, (u8_t*)q2, (u8_t*)qe2, C, HW, 0, eps, relu, 0, 0.f, 0.f};
#define CN(T) (fmt == HIFIC_Q_INT8 ? norm8_fwd_launch<T, M_CHAN, HIFIC_Q_INT8>(p, N, st) : norm8_fwd_launch<T, M_CHAN, HIFIC_Q_E4M3>(p, N, st))
    return dtype == HIFIC_F32 ? CN(float) : CN(bf16_t);
#undef CN
}

}  // extern "C"
