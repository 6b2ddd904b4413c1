// Activation checkpoints in 8 bits (format: act8.h): pack an activation, restore it.  Both are bound by HBM: pack reads T and
// writes 1 byte per element, restore the reverse.  us (TB/s): 16x60x256x256 pack 38.6 (4.9), restore 34.7 (5.4), with
// gamma, beta and ReLU 40.4 (4.7); 16x240x64x64 10.1 (4.7), 8.6 (5.5), 9.7; 16x960x16x16 4.8, 4.9, 5.2, most of it the launch.
#include "act8.h"

// Any shape: PX lanes on consecutive tokens x 256 / PX channel groups, the tensor read twice (the second time from L2).  A few
// workgroups with long chains of loads: 16x960x2x2 17 us, 2x4500x16x16 120 (2x3000x32x32 115, which the tiles below take in 10).
template <typename T, int FMT, int PX>
__global__ __launch_bounds__(256) void act8_pack_kernel(const T* __restrict__ x, u8_t* __restrict__ q, u8_t* __restrict__ qe,
                                                        int C, int HW, long long tokens) {
    constexpr int G = 256 / PX;
    __shared__ unsigned red[G][PX];
    const int px = threadIdx.x % PX, g = threadIdx.x / PX;
    for (long long t0 = (long long)blockIdx.x * PX; t0 < tokens; t0 += (long long)gridDim.x * PX) {
        const bool ok = t0 + px < tokens;
        const long long tok = ok ? t0 + px : tokens - 1, n = tok / HW;
        const size_t base = (size_t)n * C * HW + (size_t)(tok - n * HW);
        unsigned am = 0;
        for (int c = g; c < C; c += G) am = umax(am, abs_bits(DT<T>::ld(x + base + (size_t)c * HW)));
        __syncthreads();
        red[g][px] = am;
        __syncthreads();
        for (int k = 0; k < G; ++k) am = umax(am, red[k][px]);
        const unsigned code = q8_code<FMT>(am);
        const float inv = q8_inv_scale(code);
        if (!ok) continue;               // (the last round only)
        if (g == 0) qe[tok] = (u8_t)code;
        for (int c = g; c < C; c += G) q[base + (size_t)c * HW] = (u8_t)q8_round<FMT>(q8_top<FMT>(DT<T>::ld(x + base + (size_t)c * HW)) * inv);
    }
}

// Planes of eight positions and more: the tile stays in registers between the maximum and the rounding, one pass over HBM (3x220x45x31
// 4.4 us against a floor of 0.5: the launch and latency).
template <typename T, int FMT, int LPX, int CPT, int NW>
__global__ __launch_bounds__(64 * NW) void act8_pack_tile_kernel(const T* __restrict__ x, u8_t* __restrict__ q, u8_t* __restrict__ qe,
                                                             int C, int HW, unsigned tiles, unsigned blocks) {
    constexpr int SUBS = 64 / LPX, G = NW * SUBS, TP = LPX * 8;
    __shared__ unsigned red[NW][TP];
    __shared__ float inv_s[TP];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, pl = lane % LPX, g = wave * SUBS + lane / LPX;
    const unsigned bid = xcd_block(blockIdx.x, blocks), n = bid / tiles, tile = bid - n * tiles;
    const unsigned oct = tile * LPX + pl, octs = ((unsigned)HW + 7) >> 3;
    const bool ok = oct < octs;
    const unsigned hw0 = umin(ok ? oct * 8 : 0u, (unsigned)HW - 8), off = (unsigned)g * HW + hw0;
    const unsigned kst = (unsigned)G * HW;                           // channel k of this lane: img + off + k * kst
    const size_t img = (size_t)n * C * HW;
    V8<T> xr[CPT];
#pragma unroll
    for (int k = 0; k < CPT; ++k) {
        // (channel 0 in the place of one that is not there: it counts once anyway)
        xr[k].load(at(x + img, (g + G * k < C ? off + k * kst : hw0) * (unsigned)sizeof(T)));
    }
    unsigned am[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) am[j] = 0;
#pragma unroll
    for (int k = 0; k < CPT; ++k)
#pragma unroll
        for (int j = 0; j < 8; ++j) am[j] = umax(am[j], abs_bits(xr[k].get(j)));
    tile_reduce<LPX, true>(am, red[wave]);
    __syncthreads();
    if (tid < TP) {                      // (TP <= 256)
        unsigned m = red[0][tid];
#pragma unroll
        for (int i = 1; i < NW; ++i) m = umax(m, red[i][tid]);
        const unsigned code = q8_code<FMT>(m);
        inv_s[tid] = q8_inv_scale(code);
        const unsigned o = tile * LPX + (tid >> 3);
        if (o < octs) qe[(size_t)n * HW + umin(o * 8, (unsigned)HW - 8) + (tid & 7)] = (u8_t)code;
    }
    __syncthreads();
    float inv[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) inv[j] = inv_s[pl * 8 + j];
    if (!ok) return;
#pragma unroll
    for (int k = 0; k < CPT; ++k) {
        const int c = g + G * k;
        if (c < C) {
            float t[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) t[j] = q8_top<FMT>(xr[k].get(j)) * inv[j];
            *(u32x2_a1*)at(q + img, off + k * kst) = q8_pack8<FMT, false>(t);
        }
    }
}

// out = relu?(gamma_c * (q * 2^e) + beta_c), or q * 2^e where gamma is null.  V positions x CH channels per thread: the exponents
// are read once for CH channels.  V = 8 for planes of eight positions and more; V = 1 otherwise (rows of odd shape, tiny planes).
template <typename T, int FMT, int V, int CH>
__global__ __launch_bounds__(256) void act8_restore_kernel(const u8_t* __restrict__ q, const u8_t* __restrict__ qe,
                                                           const float* __restrict__ gamma, const float* __restrict__ beta,
                                                           T* __restrict__ out, int C, int HW, unsigned octs, unsigned cgs, long long n,
                                                           int relu) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const long long rest = i / octs;
    const unsigned oct = (unsigned)(i - rest * octs);
    const long long img = rest / cgs;
    const int c0 = (int)(rest - img * cgs) * CH;
    const unsigned hw0 = V == 1 ? oct : umin(oct * 8, (unsigned)HW - 8);
    const size_t base = ((size_t)img * C + c0) * HW + hw0;
    float s[V];
    if constexpr (V == 8) q8_scales(*(const u32x2_a1*)(qe + (size_t)img * HW + hw0), s);
    else s[0] = q8_scale(qe[(size_t)img * HW + hw0]);
#pragma unroll
    for (int k = 0; k < CH; ++k) {
        if (c0 + k >= C) break;
        float v[V];
        if constexpr (V == 8) q8_unpack8<FMT>(*(const u32x2_a1*)(q + base + (size_t)k * HW), s, v);
        else v[0] = q8_value<FMT>(q[base + (size_t)k * HW]) * s[0];
        if (gamma)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                v[j] = fmaf(gamma[c0 + k], v[j], beta[c0 + k]);
                if (relu) v[j] = relu_nan(v[j]);
            }
        if constexpr (V == 8) { V8<T> o; o.set(v); o.store(out + base + (size_t)k * HW); }
        else DT<T>::st(out + base + (size_t)k * HW, v[0]);
    }
}

// Rows (HW = 1) of eight channels and more: eight channels per lane, L lanes and K groups per lane for a row (row_pick).
template <typename T, int FMT, int L, int K>
__global__ __launch_bounds__(row_block(L)) void act8_pack_rows_kernel(const T* __restrict__ x, u8_t* __restrict__ q, u8_t* __restrict__ qe, int N, int C) {
    const int l = threadIdx.x % L;
    const long long row0 = (long long)blockIdx.x * (row_block(L) / L) + threadIdx.x / L;
    const bool ok = row0 < N;
    const size_t base = (size_t)(ok ? row0 : N - 1) * C;
    V8<T> xr[K];
#pragma unroll
    for (int k = 0; k < K; ++k) xr[k].load(x + base + umin((unsigned)(l + L * k) * 8, (unsigned)C - 8));
    unsigned am = 0;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < 8; ++j) am = umax(am, abs_bits(xr[k].get(j)));
    am = row_max<L>(am);
    const unsigned code = q8_code<FMT>(am);
    const float inv = q8_inv_scale(code);
    if (!ok) return;
    if (l == 0) qe[row0] = (u8_t)code;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const unsigned c = (unsigned)(l + L * k) * 8;
        if (c < (unsigned)C) {
            float t[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) t[j] = q8_top<FMT>(xr[k].get(j)) * inv;
            *(u32x2_a1*)(q + base + umin(c, (unsigned)C - 8)) = q8_pack8<FMT, false>(t);
        }
    }
}
template <typename T, int FMT>
__global__ __launch_bounds__(256) void act8_restore_rows_kernel(const u8_t* __restrict__ q, const u8_t* __restrict__ qe,
                                                                const float* __restrict__ gamma, const float* __restrict__ beta,
                                                                T* __restrict__ out, int C, unsigned octs, long long n, int relu) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const long long row = i / octs;
    const unsigned c = umin((unsigned)(i - row * octs) * 8, (unsigned)C - 8);
    const unsigned e = 0x01010101u * qe[row];
    float s[8], v[8];
    q8_scales(u32x2_t{e, e}, s);
    q8_unpack8<FMT>(*(const u32x2_a1*)(q + (size_t)row * C + c), s, v);
    if (gamma)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[j] = fmaf(gamma[c + j], v[j], beta[c + j]);
            if (relu) v[j] = relu_nan(v[j]);
        }
    V8<T> o; o.set(v); o.store(out + (size_t)row * C + c);
}

namespace {
template <typename T, int FMT>
int pack_launch(const T* x, u8_t* q, u8_t* qe, int N, int C, int HW, hipStream_t st) {
    if (HW >= 8) {
        const TileCfg t = tile_pick(N, C, HW, 8, sizeof(T));
        if (t.lpx) {
            return batch_parts(N, t.tiles, [&](long long n0, long long n) {
                const long long at = n0 * C * HW;
                const unsigned blocks = (unsigned)(t.tiles * n);
#define TILE(LPX, CPT, NW) hipLaunchKernelGGL((act8_pack_tile_kernel<T, FMT, LPX, CPT, NW>), dim3(blocks), dim3(64 * NW), 0, st, x + at, q + at, qe + n0 * HW, C, HW, t.tiles, blocks)
                TILE_DISPATCH(t, T, 8, TILE);
#undef TILE
                return hific_launch_status();
            });
        }
    }
    RowCfg r;
    if (HW == 1 && C >= 8 && (r = row_pick(N, C)).l) {
        return batch_parts(N, 1, [&](long long n0, long long n) {
            const long long at = n0 * C;
#define ROWS(L, K) hipLaunchKernelGGL((act8_pack_rows_kernel<T, FMT, L, K>), dim3(cdiv((int)n, row_block(L) / L)), dim3(row_block(L)), 0, st, x + at, q + at, qe + n0, (int)n, C)
            ROW_DISPATCH(r, ROWS)
#undef ROWS
            return hific_launch_status();
        });
    }
    const int px = any_px(N, C, HW);
    const long long tokens = (long long)N * HW;
    const dim3 grid(any_grid(cdivl(tokens, px)));
    if (px == 1) hipLaunchKernelGGL((act8_pack_kernel<T, FMT, 1>), grid, dim3(256), 0, st, x, q, qe, C, HW, tokens);
    else if (px == 16) hipLaunchKernelGGL((act8_pack_kernel<T, FMT, 16>), grid, dim3(256), 0, st, x, q, qe, C, HW, tokens);
    else hipLaunchKernelGGL((act8_pack_kernel<T, FMT, 64>), grid, dim3(256), 0, st, x, q, qe, C, HW, tokens);
    return hific_launch_status();
}

template <typename T, int FMT>
int restore_launch(const u8_t* q, const u8_t* qe, const float* gamma, const float* beta, int relu, T* out, int N, int C, int HW, hipStream_t st) {
    if (HW == 1 && C >= 8) {
        const unsigned octs = (unsigned)cdiv(C, 8);
        return batch_parts(N, cdivl(octs, 256), [&](long long n0, long long n) {
            const long long at = n0 * C;
            hipLaunchKernelGGL((act8_restore_rows_kernel<T, FMT>), dim3((unsigned)cdivl(octs * n, 256)), dim3(256), 0, st, q + at, qe + n0, gamma, beta,
                               out + at, C, octs, octs * n, relu);
            return hific_launch_status();
        });
    }
    constexpr int CH = 4;
    const unsigned octs = HW >= 8 ? (unsigned)cdivl(HW, 8) : (unsigned)HW, cgs = (unsigned)cdiv(C, CH);
    const long long each = (long long)octs * cgs;                     // threads of an image
    if (cdivl(each, 256) >= 1ll << 24) return HIFIC_ERR_UNSUPPORTED;  // (an image of more than 10^11 values)
    return batch_parts(N, cdivl(each, 256), [&](long long n0, long long n) {
        const long long at = n0 * C * HW, threads = each * n;
        const dim3 grid((unsigned)cdivl(threads, 256));
        if (HW >= 8) hipLaunchKernelGGL((act8_restore_kernel<T, FMT, 8, CH>), grid, dim3(256), 0, st, q + at, qe + n0 * HW, gamma, beta, out + at, C, HW, octs, cgs, threads, relu);
        else hipLaunchKernelGGL((act8_restore_kernel<T, FMT, 1, CH>), grid, dim3(256), 0, st, q + at, qe + n0 * HW, gamma, beta, out + at, C, HW, octs, cgs, threads, relu);
        return hific_launch_status();
    });
}
}  // namespace

extern "C" {

int hific_act8_pack(const void* x, void* q, void* qe, int fmt, int N, int C, int HW, int dtype, hipStream_t st) {
    if (!x || !q || !qe || N <= 0 || C <= 0 || HW <= 0 || !act8_dtype_ok(dtype) || !act8_fmt_ok(fmt)) return HIFIC_ERR_ARG;
    if (C > ACT8_MAX_C) return HIFIC_ERR_UNSUPPORTED;
#define PACK(T) (fmt == HIFIC_Q_INT8 ? pack_launch<T, HIFIC_Q_INT8>((const T*)x, (u8_t*)q, (u8_t*)qe, N, C, HW, st) \
                                     : pack_launch<T, HIFIC_Q_E4M3>((const T*)x, (u8_t*)q, (u8_t*)qe, N, C, HW, st))
    return dtype == HIFIC_F32 ? PACK(float) : PACK(bf16_t);
#undef PACK
}

int hific_act8_restore(const void* q, const void* qe, int fmt, const float* gamma, const float* beta, int relu, void* out,
                       int N, int C, int HW, int dtype, hipStream_t st) {
    if (!q || !qe || !out || N <= 0 || C <= 0 || HW <= 0 || !act8_dtype_ok(dtype) || !act8_fmt_ok(fmt)) return HIFIC_ERR_ARG;
    if ((gamma == nullptr) != (beta == nullptr) || (relu && !gamma)) return HIFIC_ERR_ARG;
#define REST(T) (fmt == HIFIC_Q_INT8 ? restore_launch<T, HIFIC_Q_INT8>((const u8_t*)q, (const u8_t*)qe, gamma, beta, relu, (T*)out, N, C, HW, st) \
                                     : restore_launch<T, HIFIC_Q_E4M3>((const u8_t*)q, (const u8_t*)qe, gamma, beta, relu, (T*)out, N, C, HW, st))
    return dtype == HIFIC_F32 ? REST(float) : REST(bf16_t);
#undef REST
}

}  // extern "C"
