// Backward passes of the norms of norm8.h.
#include "norm8.h"

struct NormBwd {
    const void* h; const u8_t *q, *qe;   // h in the storage type, or xh in 8 bits
    const float* rstd; const void* dy; const void* dstream; const float* w; const float* b;
    void* dx; float* part;
    int C, HW; unsigned tiles; int relu, db;
    long long tokens; int nsplit;        // (tokens: tiles of the batch in norm8_bwd_tile_kernel)
    float nc, nv;                        // as in NormFwd
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
    const size_t cs = p.HW;
    for (long long t0 = (long long)blockIdx.x * PX; t0 < p.tokens; t0 += (long long)gridDim.x * PX) {
        const bool ok = t0 + px < p.tokens;
        const long long tok = ok ? t0 + px : p.tokens - 1, n = tok / p.HW;
        const size_t base = (size_t)n * p.C * p.HW + (size_t)(tok - n * p.HW);
        const T* dy = (const T*)p.dy + base;
        const float r = p.rstd[tok], scale = SRC == SRC_T ? 0.f : q8_scale(p.qe[tok]);
        float s1 = 0.f, s2 = 0.f;
        for (int c = g; c < p.C; c += G) {
            const float xh = norm8_xh<T, SRC>(p, base + c * cs, r, scale);
            float d = DT<T>::ld(dy + c * cs);
            if (MODE == M_CHAN && p.relu && !relu_on(fmaf(p.w[c], xh, p.b[c]))) d = 0.f;
            d *= p.w[c];
            s1 += d; s2 += d * xh;
        }
        if (MODE == M_CHAN) s1 = tok_sum<PX>(s1, red) / p.nc;
        s2 = tok_sum<PX>(s2, red) / p.nv;
        if (!ok) continue;               // (the last round only)
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

// Planes: as norm8_fwd_tile_kernel.  A workgroup takes `pit` tiles in turn (p.tokens counts tiles here) and keeps the sums of its
// channels in registers: part[workgroup][0..2][c] as norm8_param_kernel.  Bound by the issue of its instructions as much as by HBM (about
// 20 per value: two unpackings, mask, two sums, three channel sums; registers allow eight waves per CU).  us (TB/s): channel
// norm + ReLU from int8 16x60x256x256 83.6 (3.8), 16x120x128x128 42.5 (3.7), 16x960x16x16 12.3 (1.6); root-mean-square norm with the stream's
// gradient 115.7 (4.3), 58.7 (4.3), 13.2 (2.4), from int8 without it 83.6, 43.3, 11.8.
template <typename T, int MODE, int SRC, int LPX, int CPT, int NW>
__global__ __launch_bounds__(64 * NW, 2) void norm8_bwd_tile_kernel(const NormBwd p, unsigned blocks, unsigned pit) {
    constexpr int SUBS = 64 / LPX, G = NW * SUBS, TP = LPX * 8;
    __shared__ float red[2][NW][TP], st[2][TP];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, pl = lane % LPX, g = wave * SUBS + lane / LPX;
    const unsigned bid = xcd_block(blockIdx.x, blocks);
    const unsigned octs = ((unsigned)p.HW + 7) >> 3;
    const unsigned kst = (unsigned)G * p.HW;                         // channel k of this lane: img + off + k * kst
    float w[CPT], b[MODE == M_CHAN ? CPT : 1], pg[CPT], pb[MODE == M_CHAN ? CPT : 1], pd[MODE == M_CHAN ? CPT : 1];
#pragma unroll
    for (int k = 0; k < CPT; ++k) {
        const int c = g + G * k, ci = c < p.C ? c : 0;
        w[k] = p.w[ci]; pg[k] = 0.f;
        if constexpr (MODE == M_CHAN) { b[k] = p.b[ci]; pb[k] = 0.f; pd[k] = 0.f; }
    }
    for (unsigned it = 0; it < pit; ++it) {
        const long long lin = (long long)bid * pit + it;             // tile of the batch: small planes share a workgroup
        if (lin >= p.tokens) break;
        const unsigned n = (unsigned)(lin / p.tiles), oct = (unsigned)(lin - (long long)n * p.tiles) * LPX + pl;
        const size_t img = (size_t)n * p.C * p.HW;
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
        float sc[8];
        if constexpr (SRC != SRC_T) q8_scales(*(const u32x2_a1*)(p.qe + tok), sc);
        auto values = [&](int k, float* xh) {
            if constexpr (SRC == SRC_T) {
#pragma unroll
                for (int j = 0; j < 8; ++j) xh[j] = hr[k].get(j) * r.get(j);
            } else q8_unpack8<SRC>(q[k], sc, xh);
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
            st[1][tid] = waves_sum<NW, TP>(red[1], tid) / p.nv;
            if (MODE == M_CHAN) st[0][tid] = waves_sum<NW, TP>(red[0], tid) / p.nc;
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

// Rows: a workgroup takes every gridDim.x-th group of R rows and keeps the sums of its channels in registers.  65536x960 104 us
// (4.8 TB/s), 16384x4096 115 us (4.7); from int8 without the stream's gradient 68 and 79.
template <typename T, int SRC, int L, int K>
__global__ __launch_bounds__(row_block(L)) void rms_bwd_rows_kernel(const NormBwd p, int N) {
    constexpr int R = row_block(L) / L;
    __shared__ float red[R > 1 ? R : 1][R > 1 ? L : 1][8];
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
        float sc[8];
        if constexpr (SRC != SRC_T) { const unsigned e = 0x01010101u * p.qe[row]; q8_scales(u32x2_t{e, e}, sc); }
        auto values = [&](int k, float* xh) {
            if constexpr (SRC == SRC_T) {
#pragma unroll
                for (int j = 0; j < 8; ++j) xh[j] = hr[k].get(j) * r;
            } else q8_unpack8<SRC>(q[k], sc, xh);
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
        if constexpr (K > 1)             // (unpacked again below, as in norm8_bwd_tile_kernel)
#pragma unroll
            for (int k = 0; k < K; ++k) { dy[k].forget(); if constexpr (SRC == SRC_T) hr[k].forget(); else forget(q[k]); }
        s2 = row_sum<L>(s2) / p.nv;
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
        if constexpr (R > 1) {
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
// lanes per workgroup (a few hundred columns of ~1000 rows: more row lanes, so that no thread adds more than a few dozen).  As a launch
// of its own about 4 us for 512 rows of 480 sums; 12 for 1024 of 16384.
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
int norm8_nsplit(int N, int C, int HW) {                             // ~1024 workgroups, at least 64 tokens each
    const int px = any_px(N, C, HW), cb = cdiv(C, 256 / px);
    const long long tokens = (long long)N * HW, most = cdivl(tokens, 64);
    long long s = cdiv(1024, cb);
    if (s > most) s = most;
    return (int)(s < 1 ? 1 : s);
}
// tiles per workgroup of the backward plane kernel: 512 workgroups, two per CU (what its registers allow), each with its share of
// the tiles - one round, few rows of channel sums (16x120x128x128: 43 us, with 1024 workgroups 47.5, with 2048 53); 256 of eight waves
// (16x480x64x64: 49 us, 512 51)
unsigned norm8_pit(const TileCfg& t) {
    const int most = t.nw == 8 ? 256 : 512;
    return (unsigned)(t.blocks < most ? 1 : cdivl(t.blocks, most));
}
// rows of channel sums that the backward pass writes
template <typename T>
size_t norm8_rows(int mode, int N, int C, int HW) {
    if (HW >= 8) {
        const TileCfg t = tile_pick(N, C, HW, tile_most<T>(), sizeof(T));
        if (t.lpx) return (size_t)cdivl(t.blocks, norm8_pit(t));
    }
    if (mode == M_RMS && HW == 1 && C >= 8) {
        const RowCfg r = row_pick(N, C);
        if (r.l) {                       // at least four groups of rows per workgroup once every CU has one: each writes a row of C sums
            const int g = (int)cdivl(N, row_block(r.l) / r.l);
            return (size_t)(g <= 256 ? g : (g < 1024 ? 256 : (g < 4096 ? cdiv(g, 4) : 1024)));
        }
    }
    return (size_t)norm8_nsplit(N, C, HW);
}

template <typename T, int MODE, int SRC>
int norm8_bwd_launch(NormBwd& p, int N, float* d0, float* d1, float* d2, int acc, int acc2, size_t ws_bytes, hipStream_t st) {
    p.nc = (float)p.C;
    p.nv = (float)(MODE == M_RMS ? p.C : p.C - 1);
    const int nr = MODE == M_RMS ? 1 : 2 + p.db;
    const size_t rows = norm8_rows<T>(MODE, N, p.C, p.HW);
    if (rows * nr * p.C * sizeof(float) > ws_bytes) return HIFIC_ERR_WS;
    TileCfg t{0, 0, 4, 0, 0};
    RowCfg r{0, 0};
    if (p.HW >= 8) t = tile_pick(N, p.C, p.HW, tile_most<T>(), sizeof(T));
    else if (MODE == M_RMS && p.HW == 1 && p.C >= 8) r = row_pick(N, p.C);
    if (rows > 0x7fffffffull) return HIFIC_ERR_UNSUPPORTED;
    if (t.lpx) {
        p.tiles = t.tiles;
        const unsigned pit = norm8_pit(t);
        p.tokens = t.blocks;
#define BWD(LPX, CPT, NW) hipLaunchKernelGGL((norm8_bwd_tile_kernel<T, MODE, SRC, LPX, CPT, NW>), dim3((unsigned)rows), dim3(64 * NW), 0, st, p, (unsigned)rows, pit)
        TILE_DISPATCH(t, T, tile_most<T>(), BWD);
#undef BWD
    } else if (r.l) {
        if constexpr (MODE == M_RMS) {
#define ROWS(L, K) hipLaunchKernelGGL((rms_bwd_rows_kernel<T, SRC, L, K>), dim3((unsigned)rows), dim3(row_block(L)), 0, st, p, N)
            ROW_DISPATCH(r, ROWS)
#undef ROWS
        }
    } else {
        const int px = any_px(N, p.C, p.HW);
        p.tokens = (long long)N * p.HW;
        p.nsplit = (int)rows;
        const dim3 grid(any_grid(cdivl(p.tokens, px))), pgrid(cdiv(p.C, 256 / px), p.nsplit);
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

size_t hific_norm8_bwd_ws_bytes(int N, int C, int HW) {
    if (N <= 0 || C <= 0 || HW <= 0 || C > ACT8_MAX_C) return 0;
    size_t rows = 0;                     // of C sums: one kind of them for the root-mean-square norm, up to three for the channel norm
    for (int mode : {M_RMS, M_CHAN}) {
        const size_t a = norm8_rows<float>(mode, N, C, HW), b = norm8_rows<bf16_t>(mode, N, C, HW), m = (a > b ? a : b) * (mode == M_RMS ? 1 : 3);
        rows = m > rows ? m : rows;
    }
    return rows * C * sizeof(float);
}

int hific_rms_norm_bwd(const void* h, const void* q, const void* qe, int fmt, const float* rstd, const void* dy, const void* dstream,
                       const float* w, void* dx, float* dw, int accumulate, int N, int C, int HW, int dtype, void* ws, size_t ws_bytes,
                       hipStream_t st) {
    if (!rstd || !dy || !w || !dx || !dw || !ws || N <= 0 || C <= 0 || HW <= 0 || !act8_dtype_ok(dtype)) return HIFIC_ERR_ARG;
    if ((h != nullptr) == (q != nullptr) || (q != nullptr) != (qe != nullptr) || (q && !act8_fmt_ok(fmt))) return HIFIC_ERR_ARG;
    if (C > ACT8_MAX_C) return HIFIC_ERR_UNSUPPORTED;
    NormBwd p{h, (const u8_t*)q, (const u8_t*)qe, rstd, dy, dstream, w, nullptr, dx, (float*)ws, C, HW, 0, 0, 0, 0, 0, 0.f, 0.f};
#define RMS(T) (h ? norm8_bwd_launch<T, M_RMS, SRC_T>(p, N, dw, nullptr, nullptr, accumulate, 0, ws_bytes, st)              \
                  : fmt == HIFIC_Q_INT8                                                                                     \
                  ? norm8_bwd_launch<T, M_RMS, HIFIC_Q_INT8>(p, N, dw, nullptr, nullptr, accumulate, 0, ws_bytes, st)       \
                  : norm8_bwd_launch<T, M_RMS, HIFIC_Q_E4M3>(p, N, dw, nullptr, nullptr, accumulate, 0, ws_bytes, st))
    return dtype == HIFIC_F32 ? RMS(float) : RMS(bf16_t);
#undef RMS
}

int hific_channelnorm8_bwd(const void* q, const void* qe, int fmt, const float* rstd, const void* dy, const float* gamma,
                           const float* beta, void* dx, float* dgamma, float* dbeta, int accumulate, float* dprev_bias,
                           int accumulate_prev, int N, int C, int HW, int relu, int dtype, void* ws, size_t ws_bytes, hipStream_t st) {
    if (!q || !qe || !rstd || !dy || !gamma || !beta || !dx || !dgamma || !dbeta || !ws || N <= 0 || C < 2 || HW <= 0) return HIFIC_ERR_ARG;
    if (!act8_dtype_ok(dtype) || !act8_fmt_ok(fmt)) return HIFIC_ERR_ARG;
    if (C > ACT8_MAX_C) return HIFIC_ERR_UNSUPPORTED;
    NormBwd p{nullptr, (const u8_t*)q, (const u8_t*)qe, rstd, dy, nullptr, gamma, beta, dx, (float*)ws, C, HW, 0, relu,
              dprev_bias ? 1 : 0, 0, 0, 0.f, 0.f};
#define CN(T) (fmt == HIFIC_Q_INT8                                                                                                       \
                   ? norm8_bwd_launch<T, M_CHAN, HIFIC_Q_INT8>(p, N, dgamma, dbeta, dprev_bias, accumulate, accumulate_prev, ws_bytes, st) \
                   : norm8_bwd_launch<T, M_CHAN, HIFIC_Q_E4M3>(p, N, dgamma, dbeta, dprev_bias, accumulate, accumulate_prev, ws_bytes, st))
    return dtype == HIFIC_F32 ? CN(float) : CN(bf16_t);
#undef CN
}

}  // extern "C"
