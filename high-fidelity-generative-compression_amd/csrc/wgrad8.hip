// Weight gradient of a convolution whose input is held in 8 bits, on planes that the natural-order kernels (gconv_wgrad*.hip: output
// rows of a multiple of 8 positions) do not take:
//     dw[m][c][r][s] = sum over images and positions of a[m][y, x] * b[c][st y - pt + r, st x - pl + s]
// (nn.Conv2d: a = dy, b = the input; nn.ConvTranspose2d: a = the input, b = dy.)  One product of two matrices whose reduction index is
// the position:  A [M][P], B [C R S][P], dw = A B^T.  Odd planes have no 16-byte rows to load, so both operands are first written out
// once in that order as bfloat16, every image's positions padded to a multiple of 8 with zeros: restored values of 8 bits are exact in
// bfloat16, products are exact, and the sum is float32.  The gather costs R S times the input's bytes (read from L2), the product then
// runs without a bounds check or an address in its loop.
#include "act8.h"

typedef __attribute__((ext_vector_type(16))) float wg_acc_t;

struct WgOperand {
    const void* src; const u8_t* qe;     // SRC_BF16: bfloat16 values; else 8 bits and their exponents
    const float* gamma; const float* beta;
    int C, H, W, R, S, st, pt, pl, reflect, relu;
};
enum { SRC_BF16 = 2 };

// out[row][i], row = (c R + r) S + s, i = n Lp + position (Lp = positions padded to a multiple of 8; i < Kp), eight i per thread
template <int SRC>
__device__ __forceinline__ void wgrad8_gather(const WgOperand& p, bf16_t* out, long long idx, int N, int OW, int L, int Lp, int Kp) {
    const unsigned per = (unsigned)Kp >> 3;
    const unsigned row = (unsigned)(idx / per), oct = (unsigned)(idx - (long long)row * per);
    const unsigned img = oct * 8 / (unsigned)Lp, pos = oct * 8 - img * (unsigned)Lp;
    V8<bf16_t> o;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.f;
    if (img < (unsigned)N) {
        const unsigned rs = (unsigned)(p.R * p.S), c = row / rs, t = row - c * rs, r = t / (unsigned)p.S, s = t - r * (unsigned)p.S;
        const size_t plane = ((size_t)img * p.C + c) * p.H * p.W, tok = (size_t)img * p.H * p.W;
        int y = (int)(pos / (unsigned)OW), x = (int)(pos - (unsigned)y * (unsigned)OW);
        const float ga = SRC != SRC_BF16 && p.gamma ? p.gamma[c] : 0.f, be = SRC != SRC_BF16 && p.gamma ? p.beta[c] : 0.f;
        const int iy0 = y * p.st - p.pt + (int)r, ix0 = x * p.st - p.pl + (int)s;
        if (p.st == 1 && x + 8 <= OW && pos + 8 <= (unsigned)L && iy0 >= 0 && iy0 < p.H && ix0 >= 0 && ix0 + 8 <= p.W) {
            // eight neighbours of one input row
            const size_t at = (size_t)iy0 * p.W + ix0;
            if constexpr (SRC == SRC_BF16) {
                o.load((const bf16_t*)p.src + plane + at);
                o.store(out + (size_t)row * Kp + (size_t)oct * 8);
                return;
            } else {
                float sc[8], s128[8];
                q8_scales<SRC>(*(const u32x2_a1*)(p.qe + tok + at), sc, s128);
                q8_unpack8<SRC>(*(const u32x2_a1*)((const u8_t*)p.src + plane + at), sc, s128, v);
                if (p.gamma)
#pragma unroll
                    for (int j = 0; j < 8; ++j) { v[j] = fmaf(ga, v[j], be); if (p.relu) v[j] = relu_nan(v[j]); }
            }
        } else
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                int iy = y * p.st - p.pt + (int)r, ix = x * p.st - p.pl + (int)s;
                if (p.reflect) { iy = reflect_idx(iy, p.H); ix = reflect_idx(ix, p.W); }
                const bool ok = pos + j < (unsigned)L && (unsigned)iy < (unsigned)p.H && (unsigned)ix < (unsigned)p.W;
                const size_t at = ok ? (size_t)iy * p.W + ix : 0;
                float w;
                if constexpr (SRC == SRC_BF16) w = bf2f(((const bf16_t*)p.src)[plane + at]);
                else {
                    w = q8_value<SRC>(((const u8_t*)p.src)[plane + at]) * q8_scale(p.qe[tok + at]);
                    if (p.gamma) { w = fmaf(ga, w, be); if (p.relu) w = relu_nan(w); }
                }
                v[j] = ok ? w : 0.f;
                if (++x == OW) { x = 0; ++y; }
            }
    }
    o.set(v);
    o.store(out + (size_t)row * Kp + (size_t)oct * 8);
}
// both operands in one launch: the first `blocks8` workgroups write the 8-bit one, the rest the bfloat16 one
template <int FMT>
__global__ __launch_bounds__(256) void wgrad8_gather_kernel(const WgOperand p8, bf16_t* __restrict__ out8, long long n8, unsigned blocks8,
                                                            const WgOperand pb, bf16_t* __restrict__ outb, long long nb, int N, int OW, int L,
                                                            int Lp, int Kp) {
    if (blockIdx.x < blocks8) {
        const long long idx = (long long)blockIdx.x * 256 + threadIdx.x;
        if (idx < n8) wgrad8_gather<FMT>(p8, out8, idx, N, OW, L, Lp, Kp);
    } else {
        const long long idx = (long long)(blockIdx.x - blocks8) * 256 + threadIdx.x;
        if (idx < nb) wgrad8_gather<SRC_BF16>(pb, outb, idx, N, OW, L, Lp, Kp);
    }
}

// part[split][m][n] (or dw itself: one split) = sum over the split's 64-wide slices of A[m][k] B[n][k].  T x T tile per workgroup, four
// waves as 2 x 2 of (T / 2) x (T / 2), v_mfma_f32_32x32x16_bf16; both tiles of the next slice travel through registers into the other
// half of LDS while this one is multiplied: one barrier per slice.  Rows of 144 bytes: conflict-free 16-byte fragment reads.
template <int T>
__global__ __launch_bounds__(256) void wgrad8_gemm_kernel(const bf16_t* __restrict__ A, const bf16_t* __restrict__ B, float* __restrict__ out, int M,
                                                          int Nn, int Kp, int mtiles, int slices, int per, int accumulate) {
    constexpr int PITCH = 144, TILE = T * PITCH, PIECES = T * 8 / 256, F = T / 64;      // F x F fragments per wave
    __shared__ __attribute__((aligned(16))) unsigned char lds[2][2][TILE];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave >> 1, wn = wave & 1, l31 = lane & 31, lhi = lane >> 5;
    const int m0 = (blockIdx.x % mtiles) * T, n0 = (blockIdx.x / mtiles) * T, split = blockIdx.y;
    const int lo = split * per, hi = lo + per < slices ? lo + per : slices;
    const bf16_t *ap[PIECES], *bp[PIECES];
    int dst[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int piece = tid + 256 * i, row = piece >> 3, seg = piece & 7;
        const int m = m0 + row < M ? m0 + row : M - 1, n = n0 + row < Nn ? n0 + row : Nn - 1;      // (rows past the end are not written)
        ap[i] = A + (size_t)m * Kp + seg * 8;
        bp[i] = B + (size_t)n * Kp + seg * 8;
        dst[i] = row * PITCH + seg * 16;
    }
    wg_acc_t acc[F][F];
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
        for (int j = 0; j < F; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
    u32x4_t ra[PIECES], rb[PIECES];
    auto load = [&](int t) {
        t = t < hi ? t : hi - 1;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) { ra[i] = *(const u32x4_t*)(ap[i] + (size_t)t * 64); rb[i] = *(const u32x4_t*)(bp[i] + (size_t)t * 64); }
    };
    auto store = [&](int b) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) { *(u32x4_t*)(lds[b][0] + dst[i]) = ra[i]; *(u32x4_t*)(lds[b][1] + dst[i]) = rb[i]; }
    };
    if (lo < hi) {
        load(lo);
        store(0);
        load(lo + 1);
        for (int t = lo; t < hi; ++t) {
            const int cur = (t - lo) & 1;
            __syncthreads();
            store(cur ^ 1);
            load(t + 2);
            const unsigned char *fa = lds[cur][0] + (wm * (T / 2) + l31) * PITCH + lhi * 16, *fb = lds[cur][1] + (wn * (T / 2) + l31) * PITCH + lhi * 16;
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
                bf16x8_t a[F], b[F];
#pragma unroll
                for (int i = 0; i < F; ++i) { a[i] = *(const bf16x8_t*)(fa + i * 32 * PITCH + ks * 32); b[i] = *(const bf16x8_t*)(fb + i * 32 * PITCH + ks * 32); }
#pragma unroll
                for (int i = 0; i < F; ++i)
#pragma unroll
                    for (int j = 0; j < F; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[i], b[j], acc[i][j], 0, 0, 0);
            }
        }
    }
    float* o = out + (size_t)split * M * Nn;
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
        for (int j = 0; j < F; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int m = m0 + wm * (T / 2) + i * 32 + (r & 3) + 8 * (r >> 2) + 4 * lhi, n = n0 + wn * (T / 2) + j * 32 + l31;
                if (m < M && n < Nn) {
                    float* d = o + (size_t)m * Nn + n;
                    *d = accumulate ? *d + acc[i][j][r] : acc[i][j][r];
                }
            }
}

// dw (=|+=) sum of the splits, in order
__global__ __launch_bounds__(256) void wgrad8_sum_kernel(const float* __restrict__ part, float* __restrict__ dw, long long n, int splits, int accumulate) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    float s = 0.f;
    int k = 0;
    for (; k + 4 <= splits; k += 4) {
        const float a = part[(size_t)k * n + i], b = part[(size_t)(k + 1) * n + i], c = part[(size_t)(k + 2) * n + i], d = part[(size_t)(k + 3) * n + i];
        s += (a + b) + (c + d);
    }
    for (; k < splits; ++k) s += part[(size_t)k * n + i];
    dw[i] = accumulate ? dw[i] + s : s;
}

namespace {
struct WgPlan { int L, Lp, Kp, M, Nn, T, mtiles, tiles, slices, per, splits; size_t a_bytes, b_bytes, bytes; };
// N images, a: [M] rows of OH x OW positions, b: C channels x R S taps
bool wg_plan(WgPlan& p, int N, int M, int C, int RS, int OH, int OW) {
    const long long L = (long long)OH * OW, Lp = (L + 7) / 8 * 8, Kp = (Lp * N + 63) / 64 * 64, Nn = (long long)C * RS;
    if (Kp > 0x7fffffff || Nn > 0x7fffffff || (long long)M * Nn > 0x7fffffff) return false;
    if ((Nn + M) * (Kp / 8) > 0x7ffffffell * 256) return false;                              // (the gather's grid)
    p.L = (int)L; p.Lp = (int)Lp; p.Kp = (int)Kp; p.M = M; p.Nn = (int)Nn;
    p.a_bytes = (size_t)M * Kp * 2; p.b_bytes = (size_t)Nn * Kp * 2;
    p.slices = (int)(Kp / 64);
    // 128 x 128 tiles halve the LDS reads per product; 64 x 64 where there would be fewer than 128 of them
    p.T = (long long)cdiv(M, 128) * cdiv(p.Nn, 128) >= 128 ? 128 : 64;
    p.mtiles = cdiv(M, p.T);
    p.tiles = p.mtiles * cdiv(p.Nn, p.T);
    // the reduction is split until ~512 workgroups run, each at least 4 slices, at most 16 partial results
    int s = cdiv(512, p.tiles);
    if (s > p.slices / 4) s = p.slices / 4;
    if (s > 16) s = 16;
    if (s < 1) s = 1;
    p.per = cdiv(p.slices, s);
    p.splits = cdiv(p.slices, p.per);
    p.bytes = p.a_bytes + p.b_bytes + (p.splits > 1 ? (size_t)p.splits * M * Nn * sizeof(float) : 0);
    return true;
}
}  // namespace

extern "C" {

// transposed 0: q [N, C, H, W] is the input of nn.Conv2d, dy [N, K, OH, OW]; 1: of nn.ConvTranspose2d (stride, pt = pl = its padding)
size_t hific_wgrad8_ws_bytes(int transposed, int N, int C, int H, int W, int K, int R, int S, int OH, int OW) {
    WgPlan p;
    if (N <= 0 || C <= 0 || K <= 0 || R <= 0 || S <= 0 || H <= 0 || W <= 0 || OH <= 0 || OW <= 0) return 0;
    const bool ok = transposed ? wg_plan(p, N, C, K, R * S, H, W) : wg_plan(p, N, K, C, R * S, OH, OW);
    return ok ? p.bytes : 0;
}

// 1: this form is the faster one.  The natural-order kernels read the input once, this one writes it R S times, so the bytes of the
// gathered operands decide, against what the other side has for the shape (us, this form / restore + the other):
//   3x3 (stride 2: 4x4 too) on rows of a multiple of 16: 8x16 out, 1 MiB 10.5 / 24; 36x32, 2 MiB 15 / 28; 6x32, 14 MiB 24 / 37;
//     51x16, 26 MiB 34 / 32; 16x16, 52 MiB 53 / 47; 75 MiB 189 / 97
//   other windows, or rows of a multiple of 8: 8x24, 13 MiB 26 / 50; 16x56, 27 MiB 43 / 60; 12x56, 35 MiB 45 / 50
//   any other row: 31x24, 10 MiB 20 / 44; 8x14, 73 MiB 79 / 231; 35x44, 78 MiB 115 / 407
int hific_wgrad8_prefer(int transposed, int N, int C, int H, int W, int K, int R, int S, int OH, int OW, int stride) {
    WgPlan p;
    if (N <= 0 || C <= 0 || K <= 0 || R <= 0 || S <= 0 || H <= 0 || W <= 0 || OH <= 0 || OW <= 0) return 0;
    if (!(transposed ? wg_plan(p, N, C, K, R * S, H, W) : wg_plan(p, N, K, C, R * S, OH, OW))) return 0;
    const int row = transposed ? W : OW;
    const bool natural = row % 16 == 0 && R == S && ((R == 3 && stride <= 2) || (R == 4 && stride == 2));
    const size_t limit = natural ? (size_t)20 << 20 : (row % 8 == 0 ? (size_t)40 << 20 : (size_t)1 << 30);
    return p.a_bytes + p.b_bytes <= limit;
}

int hific_wgrad8(int transposed, const void* q, const void* qe, int fmt, const float* gamma, const float* beta, int relu, const void* dy,
                 float* dw, int N, int C, int H, int W, int K, int R, int S, int OH, int OW, int stride, int pt, int pl, int pad_mode,
                 int accumulate, void* ws, size_t ws_bytes, hipStream_t st) {
    if (!q || !qe || !dy || !dw || !ws || N <= 0 || C <= 0 || H <= 0 || W <= 0 || K <= 0 || R <= 0 || S <= 0 || OH <= 0 || OW <= 0) return HIFIC_ERR_ARG;
    if (stride <= 0 || pt < 0 || pl < 0 || !act8_fmt_ok(fmt) || ((gamma == nullptr) != (beta == nullptr)) || (relu && !gamma)) return HIFIC_ERR_ARG;
    if (pad_mode != PAD_ZERO && pad_mode != PAD_REFLECT) return HIFIC_ERR_ARG;
    if (pad_mode == PAD_REFLECT) {           // one reflection only, and only of an input
        if (transposed || pt >= H || pl >= W || (OH - 1) * stride - pt + R - 1 > 2 * (H - 1) || (OW - 1) * stride - pl + S - 1 > 2 * (W - 1))
            return HIFIC_ERR_ARG;
    }
    WgPlan p;
    if (!(transposed ? wg_plan(p, N, C, K, R * S, H, W) : wg_plan(p, N, K, C, R * S, OH, OW))) return HIFIC_ERR_UNSUPPORTED;
    if (ws_bytes < p.bytes || ((size_t)ws & 15)) return HIFIC_ERR_WS;
    bf16_t* A = (bf16_t*)ws;
    bf16_t* B = (bf16_t*)((char*)ws + p.a_bytes);
    float* part = p.splits > 1 ? (float*)((char*)ws + p.a_bytes + p.b_bytes) : dw;
    const WgOperand x{q, (const u8_t*)qe, gamma, beta, C, H, W, transposed ? 1 : R, transposed ? 1 : S, transposed ? 1 : stride,
                      transposed ? 0 : pt, transposed ? 0 : pl, !transposed && pad_mode == PAD_REFLECT, relu};
    const WgOperand g{dy, nullptr, nullptr, nullptr, K, OH, OW, transposed ? R : 1, transposed ? S : 1, transposed ? stride : 1,
                      transposed ? pt : 0, transposed ? pl : 0, 0, 0};
    const int pw = transposed ? W : OW;
    const long long na = (long long)p.M * (p.Kp / 8), nb = (long long)p.Nn * (p.Kp / 8), n8 = transposed ? na : nb, n16 = transposed ? nb : na;
    const unsigned blocks8 = (unsigned)cdivl(n8, 256), blocks = blocks8 + (unsigned)cdivl(n16, 256);
#define GATHER(F) hipLaunchKernelGGL((wgrad8_gather_kernel<F>), dim3(blocks), dim3(256), 0, st, x, transposed ? A : B, n8, blocks8, g, \
                                     transposed ? B : A, n16, N, pw, p.L, p.Lp, p.Kp)
    if (fmt == HIFIC_Q_INT8) GATHER(HIFIC_Q_INT8); else GATHER(HIFIC_Q_E4M3);
#undef GATHER
    const dim3 grid(p.tiles, p.splits);
    const int acc = p.splits > 1 ? 0 : accumulate;
    if (p.T == 128) hipLaunchKernelGGL((wgrad8_gemm_kernel<128>), grid, dim3(256), 0, st, A, B, part, p.M, p.Nn, p.Kp, p.mtiles, p.slices, p.per, acc);
    else hipLaunchKernelGGL((wgrad8_gemm_kernel<64>), grid, dim3(256), 0, st, A, B, part, p.M, p.Nn, p.Kp, p.mtiles, p.slices, p.per, acc);
    if (p.splits > 1) {
        const long long n = (long long)p.M * p.Nn;
        hipLaunchKernelGGL(wgrad8_sum_kernel, dim3((unsigned)cdivl(n, 256)), dim3(256), 0, st, part, dw, n, p.splits, accumulate);
    }
    return hific_launch_status();
}

}  // extern "C"
