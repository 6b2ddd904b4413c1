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
        mu = tok_sum<PX>(s, red) / (float)p.C;
    }
    float ss = 0.f;
    for (int c = g; c < p.C; c += G) {
        const float v = stream(c), d = v - mu;
        ss += d * d;
        if (MODE == M_RMS && h && ok) DT<T>::st(h + c * cs, v);
    }
    ss = tok_sum<PX>(ss, red);
    const float r = rsqrtf(ss / (float)(MODE == M_RMS ? p.C : p.C - 1) + p.eps);
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
        if (MODE == M_CHAN && p.relu) o = o > 0.f || o != o ? o : 0.f;
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
            if (p.relu) o = o > 0.f || o != o ? o : 0.f;
            T t; DT<T>::st(&t, o); o = DT<T>::ld(&t) + DT<T>::ld(rs + c * cs);
            if (ok) p.q2[base + c * cs] = (u8_t)q8_round<F>(o * inv2);
        }
    }
}

struct NormBwd {
    const void* h; const u8_t *q, *qe;   // h in the storage type, or xh in 8 bits
    const float* rstd; const void* dy; const void* dstream; const float* w; const float* b;
    void* dx; float* part;
    int C, HW; unsigned tiles; int relu, db;
    long long tokens; int nsplit;
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
        if (MODE == M_CHAN && p.relu && !(fmaf(p.w[c], xh, p.b[c]) > 0.f)) d = 0.f;
        d *= p.w[c];
        s1 += d; s2 += d * xh;
    }
    if (MODE == M_CHAN) s1 = tok_sum<PX>(s1, red) / (float)p.C;
    s2 = tok_sum<PX>(s2, red) / (float)(MODE == M_RMS ? p.C : p.C - 1);
    if (!ok) return;
    for (int c = g; c < p.C; c += G) {
        const float xh = norm8_xh<T, SRC>(p, base + c * cs, r, scale);
        float d = DT<T>::ld(dy + c * cs);
        if (MODE == M_CHAN && p.relu && !(fmaf(p.w[c], xh, p.b[c]) > 0.f)) d = 0.f;
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
            if (MODE == M_CHAN && p.relu && !(fmaf(p.w[c], xh, p.b[c]) > 0.f)) d = 0.f;
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

// column sums of part[rows][nr * C] into up to three vectors, each written or added to: 64 columns x 16 row lanes, fixed order
__global__ __launch_bounds__(1024) void norm8_colsum_kernel(const float* __restrict__ part, float* __restrict__ d0, float* __restrict__ d1,
                                                            float* __restrict__ d2, int C, int rows, int nr, int acc, int acc2) {
    __shared__ float red[16][64];
    const int col = blockIdx.x * 64 + (threadIdx.x & 63), rl = threadIdx.x >> 6, W = nr * C;
    float s = 0.f;
    if (col < W) {
        int r = rl;
        for (; r + 112 < rows; r += 128) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = part[(size_t)(r + 16 * j) * W + col];
            s += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
        }
        for (; r < rows; r += 16) s += part[(size_t)r * W + col];
    }
    red[rl][threadIdx.x & 63] = s;
    __syncthreads();
    if (rl == 0 && col < W) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) t += red[i][threadIdx.x & 63];
        float* d = col < C ? d0 + col : (col < 2 * C ? d1 + (col - C) : d2 + (col - 2 * C));
        if (col < 2 * C ? acc : acc2) *d += t; else *d = t;
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

template <typename T, int MODE, int FMT>
int norm8_fwd_launch(NormFwd& p, int N, hipStream_t st) {
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
    const int px = norm8_px(p.HW), nr = MODE == M_RMS ? 1 : 2 + p.db;
    const long long blocks = cdivl(p.HW, px) * N;
    if (blocks > 0x7fffffffll) return HIFIC_ERR_UNSUPPORTED;
    p.tiles = (unsigned)cdivl(p.HW, px);
    p.tokens = (long long)N * p.HW;
    p.nsplit = norm8_nsplit(N, p.C, p.HW);
    if ((size_t)p.nsplit * nr * p.C * sizeof(float) > ws_bytes) return HIFIC_ERR_WS;
    const dim3 grid((unsigned)blocks), pgrid(cdiv(p.C, 256 / px), p.nsplit);
#define BWD(PX)                                                                                             \
    do {                                                                                                    \
        hipLaunchKernelGGL((norm8_bwd_kernel<T, MODE, SRC, PX>), grid, dim3(256), 0, st, p);               \
        hipLaunchKernelGGL((norm8_param_kernel<T, MODE, SRC, PX>), pgrid, dim3(256), 0, st, p);            \
    } while (0)
    if (px == 1) BWD(1); else if (px == 16) BWD(16); else BWD(64);
#undef BWD
    hipLaunchKernelGGL(norm8_colsum_kernel, dim3(cdiv(nr * p.C, 64)), dim3(1024), 0, st, p.part, d0, d1, d2, p.C, p.nsplit, nr, acc, acc2);
    return hific_launch_status();
}
}  // namespace

extern "C" {

int hific_rms_norm_fwd(const void* x, const void* resid, const float* w, void* y, void* h, float* rstd, void* q, void* qe,
                       int fmt, int q_of_y, int N, int C, int HW, float eps, int dtype, hipStream_t st) {
    if (!x || !w || N <= 0 || C <= 0 || HW <= 0 || !act8_dtype_ok(dtype) || !(eps > 0.f)) return HIFIC_ERR_ARG;
    if ((resid != nullptr) != (h != nullptr) || (q != nullptr) != (qe != nullptr) || (!y && !q)) return HIFIC_ERR_ARG;
    if (q && !act8_fmt_ok(fmt)) return HIFIC_ERR_ARG;
    NormFwd p{x, resid, w, nullptr, y, h, rstd, (u8_t*)q, (u8_t*)qe, nullptr, nullptr, C, HW, 0, eps, 0, q_of_y};
#define RMS(T) (!q ? norm8_fwd_launch<T, M_RMS, Q_NONE>(p, N, st) : fmt == HIFIC_Q_INT8                                     \
                   ? norm8_fwd_launch<T, M_RMS, HIFIC_Q_INT8>(p, N, st) : norm8_fwd_launch<T, M_RMS, HIFIC_Q_E4M3>(p, N, st))
    return dtype == HIFIC_F32 ? RMS(float) : RMS(bf16_t);
#undef RMS
}

size_t hific_norm8_bwd_ws_bytes(int N, int C, int HW) {
    if (N <= 0 || C <= 0 || HW <= 0) return 0;
    return (size_t)norm8_nsplit(N, C, HW) * 3 * C * sizeof(float);
}

int hific_rms_norm_bwd(const void* h, const void* q, const void* qe, int fmt, const float* rstd, const void* dy, const void* dstream,
                       const float* w, void* dx, float* dw, int accumulate, int N, int C, int HW, int dtype, void* ws, size_t ws_bytes,
                       hipStream_t st) {
    if (!rstd || !dy || !w || !dx || !dw || !ws || N <= 0 || C <= 0 || HW <= 0 || !act8_dtype_ok(dtype)) return HIFIC_ERR_ARG;
    if ((h != nullptr) == (q != nullptr) || (q != nullptr) != (qe != nullptr) || (q && !act8_fmt_ok(fmt))) return HIFIC_ERR_ARG;
    NormBwd p{h, (const u8_t*)q, (const u8_t*)qe, rstd, dy, dstream, w, nullptr, dx, (float*)ws, C, HW, 0, 0, 0, 0, 0};
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
    NormFwd p{x, resid, gamma, beta, y, nullptr, rstd, (u8_t*)q, (u8_t*)qe, (u8_t*)q2, (u8_t*)qe2, C, HW, 0, eps, relu, 0};
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
              dprev_bias ? 1 : 0, 0, 0};
#define CN(T) (fmt == HIFIC_Q_INT8                                                                                                       \
                   ? norm8_bwd_launch<T, M_CHAN, HIFIC_Q_INT8>(p, N, dgamma, dbeta, dprev_bias, accumulate, accumulate_prev, ws_bytes, st) \
                   : norm8_bwd_launch<T, M_CHAN, HIFIC_Q_E4M3>(p, N, dgamma, dbeta, dprev_bias, accumulate, accumulate_prev, ws_bytes, st))
    return dtype == HIFIC_F32 ? CN(float) : CN(bf16_t);
#undef CN
}

}  // extern "C"
