// Weight gradient of a convolution whose input is held in 8 bits, for odd planes and small products (the natural-order kernels of
// gconv_wgrad*.hip need output rows of a multiple of 8 positions, and reach their rate on large products):
//     dw[m][c][r][s] = sum over images and positions of a[m][y, x] * b[c][st y - pt + r, st x - pl + s]
// (nn.Conv2d: a = dy, b = the input; nn.ConvTranspose2d: a = the input, b = dy.)  One product of two matrices whose reduction index is
// the position:  A [M][P], B [C R S][P], dw = A B^T.  A is read where it lies.  The rows of B are written out once as bfloat16 (restored
// values of 8 bits are exact in it, so products are exact; the sum is float32), but only for the S horizontal taps: with rows of exactly
// OW values, a vertical tap is a shift by whole rows of the same copy,
//     T[c][s][py][n][y'][x] = b[c][st y' + py - pt, st x + s - pl],   py = r mod st,   B[c r s][n, y, x] = T[c][s][py][n][y + r / st][x]
// so that eight neighbouring positions of an image are sixteen neighbouring bytes of both operands (at any 2-byte address), and the
// product's loop has no bounds check.  Writing out all R S taps took 20 of 32 us at 7x112x19x69, 3x3, and 52 of 123 us at 12x49x56x74.
#include "act8.h"

typedef __attribute__((ext_vector_type(16))) float wg_acc_t;

extern "C" int hific_act8_restore(const void* q, const void* qe, int fmt, const float* gamma, const float* beta, int relu, void* out,
                                  int N, int C, int HW, int dtype, hipStream_t st);      // act8.hip

enum { SRC_BF16 = 2 };
struct WgTaps {
    const void* src; const u8_t* qe;     // SRC_BF16: bfloat16 values; else 8 bits and their exponents
    const float* gamma; const float* beta;
    int C, H, W, S, py, st, pt, pl, reflect, relu, N, OW, rows;       // rows of T per image
    int window;                          // the bytes of eight neighbours lie in one window of an input row
    unsigned octs;                       // groups of eight of a row
};

// T, eight neighbours of one row (of eight and more) per thread, at the row's end moved back to end with it.  What they are read from
// lies in one window of eight (stride 2: sixteen) bytes of one input row, reflected columns included: a byte permutation picks them,
// and only the lanes at a row's ends form its selectors.  Other shapes (narrow rows, large strides or pads), and the ends of bfloat16
// rows: value by value.  Bound by the latency of its index arithmetic and loads on small planes (2x120x61x47 stride 2: 5.3 us), by its
// instructions on large ones (16x480x32x32 stride 2, 25 MB written: 17 us, value by value 41).
template <int SRC>
__global__ __launch_bounds__(256) void wgrad8_taps_kernel(const WgTaps p, bf16_t* __restrict__ out, unsigned total) {
    const unsigned idx = blockIdx.x * 256 + threadIdx.x;
    if (idx >= total) return;
    const unsigned line = idx / p.octs;                              // ((c, s, py, n), y)
    const int x0 = p.OW < 8 ? 0 : (int)umin((idx - line * p.octs) * 8, (unsigned)p.OW - 8), cnt = p.OW < 8 ? p.OW : 8;
    const unsigned row = line / (unsigned)p.rows;
    const int y = (int)(line - row * (unsigned)p.rows);
    unsigned t = row / (unsigned)p.N;
    const unsigned n = row - t * (unsigned)p.N;
    const int py = (int)(t % (unsigned)p.py);
    t /= (unsigned)p.py;
    const unsigned c = t / (unsigned)p.S;
    const int s = (int)(t - c * (unsigned)p.S);
    int iy = y * p.st + py - p.pt;
    if (p.reflect) iy = reflect_idx(iy, p.H);
    const bool rok = (unsigned)iy < (unsigned)p.H;                   // (a row that only a tap beyond R would read: past the reflection too)
    const int ix0 = x0 * p.st + s - p.pl;
    bf16_t* dst = out + (size_t)line * p.OW + x0;
    V8<bf16_t> o;
    float v[8];
    if (!rok) {
#pragma unroll
        for (int j = 0; j < 8; ++j) if (j < cnt) dst[j] = 0;
        return;
    }
    const size_t at = ((size_t)n * p.C + c) * p.H * p.W + (size_t)iy * p.W, tok = ((size_t)n * p.H + iy) * p.W;
    if constexpr (SRC == SRC_BF16) {
        const bf16_t* src = (const bf16_t*)p.src + at;
        if (p.window && ix0 >= 0 && ix0 + 8 * p.st <= p.W) {
            o.load(src + ix0);
            if (p.st == 2) {
                V8<bf16_t> h; h.load(src + ix0 + 8);
                o.r = u32x4_t{__builtin_amdgcn_perm(o.r[1], o.r[0], 0x05040100u), __builtin_amdgcn_perm(o.r[3], o.r[2], 0x05040100u),
                              __builtin_amdgcn_perm(h.r[1], h.r[0], 0x05040100u), __builtin_amdgcn_perm(h.r[3], h.r[2], 0x05040100u)};
            }
            o.store(dst);
            return;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            int ix = ix0 + j * p.st;
            if (p.reflect) ix = reflect_idx(ix, p.W);
            const bool ok = (unsigned)ix < (unsigned)p.W;
            v[j] = ok ? bf2f(src[ok ? ix : 0]) : 0.f;
        }
    } else {
        const u8_t *src = (const u8_t*)p.src + at, *e = p.qe + tok;
        const float ga = p.gamma ? p.gamma[c] : 0.f, be = p.gamma ? p.beta[c] : 0.f;
        unsigned keep = 0xffu;
        if (p.window) {
            const int base = ix0 < 0 ? 0 : (ix0 + 8 * p.st <= p.W ? ix0 : p.W - 8 * p.st);
            const bool edge = base != ix0;
            u32x2_t q, eb;
            if (p.st == 1) {
                u32x2_t sel{0x03020100u, 0x07060504u};
                if (edge) {
                    sel = u32x2_t{0u, 0u}; keep = 0;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        int ix = ix0 + j;
                        if (p.reflect) ix = reflect_idx(ix, p.W);
                        const bool ok = (unsigned)(ix - base) < 8u;
                        keep |= ok ? 1u << j : 0u;
                        sel[j >> 2] |= (ok ? (unsigned)(ix - base) : 0u) << (8 * (j & 3));
                    }
                }
                const u32x2_t qw = *(const u32x2_a1*)(src + base), ew = *(const u32x2_a1*)(e + base);
                q = u32x2_t{__builtin_amdgcn_perm(qw[1], qw[0], sel[0]), __builtin_amdgcn_perm(qw[1], qw[0], sel[1])};
                eb = u32x2_t{__builtin_amdgcn_perm(ew[1], ew[0], sel[0]), __builtin_amdgcn_perm(ew[1], ew[0], sel[1])};
            } else {
                // a byte of the low half of the window, or (0x0c: a zero byte) of the high one
                u32x2_t sl{0x06040200u, 0x0c0c0c0cu}, sh{0x0c0c0c0cu, 0x06040200u};
                if (edge) {
                    sl = u32x2_t{0u, 0u}; sh = u32x2_t{0u, 0u}; keep = 0;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        int ix = ix0 + 2 * j;
                        if (p.reflect) ix = reflect_idx(ix, p.W);
                        const unsigned i = (unsigned)(ix - base);
                        keep |= i < 16u ? 1u << j : 0u;
                        sl[j >> 2] |= (i < 8u ? i : 0x0cu) << (8 * (j & 3));
                        sh[j >> 2] |= (i >= 8u && i < 16u ? i - 8u : 0x0cu) << (8 * (j & 3));
                    }
                }
                const u32x4_t qw = *(const u32x4_a1*)(src + base), ew = *(const u32x4_a1*)(e + base);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    q[h] = __builtin_amdgcn_perm(qw[1], qw[0], sl[h]) | __builtin_amdgcn_perm(qw[3], qw[2], sh[h]);
                    eb[h] = __builtin_amdgcn_perm(ew[1], ew[0], sl[h]) | __builtin_amdgcn_perm(ew[3], ew[2], sh[h]);
                }
            }
            float sc[8];
            q8_scales(eb, sc);
            q8_unpack8<SRC>(q, sc, v);
        } else {
            keep = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                int ix = ix0 + j * p.st;
                if (p.reflect) ix = reflect_idx(ix, p.W);
                const bool ok = (unsigned)ix < (unsigned)p.W;
                keep |= ok ? 1u << j : 0u;
                v[j] = q8_value<SRC>(src[ok ? ix : 0]) * q8_scale(e[ok ? ix : 0]);
            }
        }
        if (p.gamma)
#pragma unroll
            for (int j = 0; j < 8; ++j) { v[j] = fmaf(ga, v[j], be); if (p.relu) v[j] = relu_nan(v[j]); }
        if (keep != 0xffu)               // the pad's zeros come behind the norm
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = (keep >> j) & 1u ? v[j] : 0.f;
    }
    if (cnt == 8) { o.set(v); o.store(dst); return; }
#pragma unroll
    for (int j = 0; j < 8; ++j) if (j < cnt) DT<bf16_t>::st(dst + j, v[j]);
}

// A [N][M][L] and T, as the product reads them
struct WgGemm {
    const bf16_t *A, *T;
    float* out;
    int N, M, Nn, L, OW, plane;          // plane: of T
    int R, S, st, py;
    int octs, mtiles, tiles, slices, per, accumulate;
    unsigned blocks;
};

// part[split][m][n] (or dw itself: one split) = sum over the split's slices of A[m][k] B[n][k].  A slice is eight groups of eight
// positions; a group stays in its image, the image's last one is moved back to end with it and the positions it repeats are set to
// zero in both operands (zero times an infinity of one would be NaN).  TILE x TILE per workgroup, four waves as 2 x 2,
// v_mfma_f32_32x32x16_bf16; both tiles of the next slice travel through registers into the other half of LDS while this one is
// multiplied: one barrier per slice (two or four slices ahead in registers: 9 to 36 % slower).  Rows of 144 bytes: conflict-free 16-byte
// fragment reads.  The tiles of one split go to one XCD, whose L2 then holds the split's part of both operands (4 to 6 %).
// 3x437x35x44 to 793 channels, 3x3: 56 us, 515 TFLOP/s; 960 x 960 on 16x16x16: 134 us, 507.  By count a slice of the large tile takes 768
// cycles of LDS against 512 of matrix instructions, and at 2-byte addresses about as many in the vector cache.
template <int TILE>
__global__ __launch_bounds__(256) void wgrad8_gemm_kernel(const WgGemm p) {
    constexpr int PITCH = 144, BYTES = TILE * PITCH, PIECES = TILE * 8 / 256, F = TILE / 64;      // F x F fragments per wave
    __shared__ __attribute__((aligned(16))) unsigned char lds[2][2][BYTES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave >> 1, wn = wave & 1, l31 = lane & 31, lhi = lane >> 5;
    const unsigned bid = xcd_block(blockIdx.x, gridDim.x);           // (a multiple of eight workgroups)
    if (bid >= p.blocks) return;
    const int split = (int)(bid / (unsigned)p.tiles), tile = (int)(bid - (unsigned)split * (unsigned)p.tiles);
    const int m0 = (tile % p.mtiles) * TILE, n0 = (tile / p.mtiles) * TILE;
    const int lo = split * p.per, hi = lo + p.per < p.slices ? lo + p.per : p.slices;
    const bf16_t *ap[PIECES], *bp[PIECES];
    int dst[PIECES];
    const int seg = tid & 7;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int row = (tid + 256 * i) >> 3;
        const int m = m0 + row < p.M ? m0 + row : p.M - 1, n = n0 + row < p.Nn ? n0 + row : p.Nn - 1;      // (rows past the end are not written)
        const int rs = p.R * p.S, c = n / rs, r = (n - c * rs) / p.S, s = n - c * rs - r * p.S, ry = r / p.st;
        ap[i] = p.A + (size_t)m * p.L;
        bp[i] = p.T + ((size_t)(c * p.S + s) * p.py + (r - ry * p.st)) * p.N * p.plane + (size_t)ry * p.OW;
        dst[i] = row * PITCH + seg * 16;
    }
    // this thread's group of the next slice that is loaded: image and group in it
    int img = (int)(((long long)lo * 8 + seg) / p.octs), oct = (int)((long long)lo * 8 + seg - (long long)img * p.octs);
    wg_acc_t acc[F][F];
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
        for (int j = 0; j < F; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
    u32x4_t ra[PIECES], rb[PIECES];
    int dup = 0;                         // leading positions of the loaded group that do not count
    auto load = [&]() {
        const bool ok = img < p.N;       // (the last slice, and what is loaded past it)
        const int pos = ok ? (oct * 8 < p.L - 8 ? oct * 8 : p.L - 8) : 0;
        dup = ok ? oct * 8 - pos : 8;
        const size_t im = ok ? img : 0, oa = im * p.M * p.L + pos, ob = im * p.plane + pos;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) { ra[i] = *(const u32x4_a2*)(ap[i] + oa); rb[i] = *(const u32x4_a2*)(bp[i] + ob); }
        oct += 8;
        while (oct >= p.octs) { oct -= p.octs; ++img; }
    };
    auto store = [&](int b) {
        if (dup) {
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                const unsigned keep = dup > 2 * d + 1 ? 0u : (dup > 2 * d ? 0xffff0000u : 0xffffffffu);
#pragma unroll
                for (int i = 0; i < PIECES; ++i) { ra[i][d] &= keep; rb[i][d] &= keep; }
            }
        }
#pragma unroll
        for (int i = 0; i < PIECES; ++i) { *(u32x4_t*)(lds[b][0] + dst[i]) = ra[i]; *(u32x4_t*)(lds[b][1] + dst[i]) = rb[i]; }
    };
    if (lo < hi) {
        load();
        store(0);
        load();
        for (int t = lo; t < hi; ++t) {
            const int cur = (t - lo) & 1;
            __syncthreads();
            store(cur ^ 1);
            load();
            const unsigned char *fa = lds[cur][0] + (wm * (TILE / 2) + l31) * PITCH + lhi * 16, *fb = lds[cur][1] + (wn * (TILE / 2) + l31) * PITCH + lhi * 16;
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
    float* o = p.out + (size_t)split * p.M * p.Nn;
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
        for (int j = 0; j < F; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int m = m0 + wm * (TILE / 2) + i * 32 + (r & 3) + 8 * (r >> 2) + 4 * lhi, n = n0 + wn * (TILE / 2) + j * 32 + l31;
                if (m < p.M && n < p.Nn) {
                    float* d = o + (size_t)m * p.Nn + n;
                    *d = p.accumulate ? *d + acc[i][j][r] : acc[i][j][r];
                }
            }
}

// dw (=|+=) sum of the parts in a fixed order, R threads per value (many parts of few values: 1, or a chain of loads decides)
template <int R>
__global__ __launch_bounds__(256) void wgrad8_sum_kernel(const float* __restrict__ part, float* __restrict__ dw, long long n, int splits, int accumulate) {
    constexpr int COLS = 256 / R;
    __shared__ float red[R > 1 ? R : 1][R > 1 ? COLS : 1];
    const int col = threadIdx.x % COLS, r = threadIdx.x / COLS;
    const long long i = (long long)blockIdx.x * COLS + col;
    float s = 0.f;
    if (i < n) {
        int k = r;
        for (; k + 3 * R < splits; k += 4 * R) {
            const float a = part[(size_t)k * n + i], b = part[(size_t)(k + R) * n + i], c = part[(size_t)(k + 2 * R) * n + i], d = part[(size_t)(k + 3 * R) * n + i];
            s += (a + b) + (c + d);
        }
        for (; k < splits; k += R) s += part[(size_t)k * n + i];
    }
    if constexpr (R > 1) {
        red[r][col] = s;
        __syncthreads();
        if (r != 0) return;
        s = 0.f;
#pragma unroll
        for (int j = 0; j < R; ++j) s += red[j][col];
    }
    if (i < n) dw[i] = accumulate ? dw[i] + s : s;
}

namespace {
struct WgPlan { int L, M, Nn, T, octs, py, plane, mtiles, tiles, slices, per, splits; size_t a_bytes, t_bytes, bytes; };
// N images, a: [M] rows of OH x OW positions (written out as bfloat16 where it is the 8-bit operand), b: C channels x R x S taps
bool wg_plan(WgPlan& p, int N, int M, int C, int R, int S, int OH, int OW, int st, bool a8) {
    const long long L = (long long)OH * OW, Nn = (long long)C * R * S, plane = (OH + (R - 1ll) / st) * OW, py = st < R ? st : R;
    if (L < 8 || plane > 0x7fffffff || Nn > 0x7fffffff || M * Nn > 0x7fffffff) return false;
    const long long octs = (L + 7) / 8, rows = (long long)C * S * py * N;
    if (octs * N > 0x3fffffff || rows * (plane / OW) * ((OW + 7) / 8) > 0x7fffffff) return false;
    p.L = (int)L; p.M = M; p.Nn = (int)Nn; p.octs = (int)octs; p.py = (int)py; p.plane = (int)plane;
    p.a_bytes = a8 ? ((size_t)N * M * L * 2 + 255) / 256 * 256 : 0;
    p.t_bytes = ((size_t)rows * plane * 2 + 255) / 256 * 256;
    p.slices = (int)((octs * N + 7) / 8);
    // 128 x 128 tiles halve the LDS reads per product; 64 x 64 where 256 workgroups of those would have less than 16 slices each
    const long long big = (long long)cdiv(M, 128) * cdiv(p.Nn, 128);
    p.T = big >= 128 || big * p.slices >= 4096 ? 128 : 64;
    p.mtiles = cdiv(M, p.T);
    p.tiles = p.mtiles * cdiv(p.Nn, p.T);
    // How often to split the reduction (at least 4 slices each, at most 32 parts, of few tiles up to 256).  A CU holds two workgroups of the large tile;
    // alone one takes about 1 us per slice, two together 1.55 (217 tiles of 73 slices: not split 67 us, two parts 56, three 70;
    // 12 tiles of 777: 21 parts 39 us, 22 parts - eight CUs with two of them - 48); of the small tile up to four overlap.  The sum over the parts takes
    // 4 us and its bytes.
    const double mn = (double)M * p.Nn * 4e-6 / 4;
    int best = 1;
    double best_us = 1e30;
    const int most = p.tiles <= 8 ? 256 / p.tiles : (p.T == 128 ? 32 : 16);
    for (int s = 1; s <= most && (s == 1 || s * 4 <= p.slices); ++s) {
        const int w = (int)cdivl((long long)p.tiles * s, 256);
        const double share = p.T == 128 ? w / 2 * 1.55 + w % 2 : 0.3 + 0.15 * w;
        const double us = share * (cdiv(p.slices, s) + (p.T == 128 ? 3 : 8)) + (s > 1 ? 4 + (s + 1) * mn : 0.);
        if (us < best_us) { best_us = us; best = s; }
    }
    const int s = best;
    p.per = cdiv(p.slices, s);
    p.splits = cdiv(p.slices, p.per);
    p.bytes = p.a_bytes + p.t_bytes + (p.splits > 1 ? (size_t)p.splits * M * Nn * sizeof(float) : 0);
    return (long long)p.tiles * p.splits < 1 << 23;
}
bool wg_plan_of(WgPlan& p, int transposed, int N, int C, int H, int W, int K, int R, int S, int OH, int OW, int stride) {
    if (N <= 0 || C <= 0 || K <= 0 || R <= 0 || S <= 0 || H <= 0 || W <= 0 || OH <= 0 || OW <= 0 || stride <= 0) return false;
    return transposed ? wg_plan(p, N, C, K, R, S, H, W, stride, true) : wg_plan(p, N, K, C, R, S, OH, OW, stride, false);
}
}  // namespace

extern "C" {

// transposed 0: q [N, C, H, W] is the input of nn.Conv2d, dy [N, K, OH, OW]; 1: of nn.ConvTranspose2d (stride, pt = pl = its padding)
size_t hific_wgrad8_ws_bytes(int transposed, int N, int C, int H, int W, int K, int R, int S, int OH, int OW, int stride) {
    WgPlan p;
    return wg_plan_of(p, transposed, N, C, H, W, K, R, S, OH, OW, stride) ? p.bytes : 0;
}

// 1: this form is the faster one.  Against it: the bytes of T, which few rows of A do not pay for, and where the natural-order kernels
// apply (3x3, 4x4 with stride 2, rows of a multiple of 16) their better rate on large products.  us, this form / restore + the other:
//   natural, 0.15 GFLOP 10 / 26; 1.2, 15 / 27; 4.2, 30 / 40, transposed 36 / 43; 8.5, 37 / 36, transposed 50 / 40; 68 (16x960x16x16
//     3x3, 960 out) 139 / 88
//   rows of a multiple of 8, or other windows: 16x480x24x24 3x3 86 / 126; 16x320x16x16 5x5 65 / 244; 2x60x200x200 3x3 48 / 64;
//     2x60x128x128 7x7 to 3 channels 58 / 41
//   any other row: 2x120x61x47 stride 2 18 / 44; 3x437x35x44 75 / 403; 16x16x255x255 191 / 202; 4x60x255x255 7x7 to 3 channels 436 / 88
int hific_wgrad8_prefer(int transposed, int N, int C, int H, int W, int K, int R, int S, int OH, int OW, int stride) {
    WgPlan p;
    if (!wg_plan_of(p, transposed, N, C, H, W, K, R, S, OH, OW, stride)) return 0;
    const int row = transposed ? W : OW;
    if ((long long)p.M * R < 32 && p.t_bytes > (size_t)4 << 20) return 0;
    const bool natural = row % 16 == 0 && R == S && ((R == 3 && stride <= 2) || (R == 4 && stride == 2));
    if (natural) return p.t_bytes <= (size_t)40 << 20 && 2. * N * p.L * p.M * p.Nn <= (transposed ? 5e9 : 9e9);
    return p.a_bytes + p.t_bytes <= (row % 8 == 0 ? (size_t)256 << 20 : (size_t)1 << 30);
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
    if (!wg_plan_of(p, transposed, N, C, H, W, K, R, S, OH, OW, stride)) return HIFIC_ERR_UNSUPPORTED;
    if (ws_bytes < p.bytes || ((size_t)ws & 15)) return HIFIC_ERR_WS;
    bf16_t* A = (bf16_t*)ws;
    bf16_t* T = (bf16_t*)((char*)ws + p.a_bytes);
    float* part = p.splits > 1 ? (float*)((char*)ws + p.a_bytes + p.t_bytes) : dw;
    if (transposed) {
        const int rc = hific_act8_restore(q, qe, fmt, gamma, beta, relu, A, N, C, H * W, HIFIC_BF16, st);
        if (rc != HIFIC_OK) return rc;
    }
    const int pw = transposed ? W : OW;
    const int bw = transposed ? OW : W;
    const unsigned toct = (unsigned)cdiv(pw, 8), total = (unsigned)((transposed ? K : C) * (long long)S * p.py * N * (p.plane / pw) * toct);
    const int window = pw >= 8 && stride <= 2 && bw >= 8 * stride && pl <= 7 && (long long)(pw - 1) * stride + S - 1 - pl <= bw + 6;
    const WgTaps x{transposed ? dy : q, (const u8_t*)qe, gamma, beta, transposed ? K : C, transposed ? OH : H, bw, S, p.py, stride,
                   pt, pl, pad_mode == PAD_REFLECT, relu, N, pw, p.plane / pw, window, toct};
    const dim3 tgrid((total + 255) / 256);
    if (transposed) hipLaunchKernelGGL((wgrad8_taps_kernel<SRC_BF16>), tgrid, dim3(256), 0, st, x, T, total);
    else if (fmt == HIFIC_Q_INT8) hipLaunchKernelGGL((wgrad8_taps_kernel<HIFIC_Q_INT8>), tgrid, dim3(256), 0, st, x, T, total);
    else hipLaunchKernelGGL((wgrad8_taps_kernel<HIFIC_Q_E4M3>), tgrid, dim3(256), 0, st, x, T, total);
    const WgGemm g{transposed ? A : (const bf16_t*)dy, T, part, N, p.M, p.Nn, p.L, pw, p.plane, R, S, stride, p.py, p.octs, p.mtiles, p.tiles,
                   p.slices, p.per, p.splits > 1 ? 0 : accumulate, (unsigned)(p.tiles * p.splits)};
    if (p.T == 128) hipLaunchKernelGGL((wgrad8_gemm_kernel<128>), dim3((g.blocks + 7) & ~7u), dim3(256), 0, st, g);
    else hipLaunchKernelGGL((wgrad8_gemm_kernel<64>), dim3((g.blocks + 7) & ~7u), dim3(256), 0, st, g);
    if (p.splits > 1) {
        const long long n = (long long)p.M * p.Nn;
        if (p.splits > 32) hipLaunchKernelGGL((wgrad8_sum_kernel<8>), dim3((unsigned)cdivl(n, 32)), dim3(256), 0, st, part, dw, n, p.splits, accumulate);
        else hipLaunchKernelGGL((wgrad8_sum_kernel<1>), dim3((unsigned)cdivl(n, 256)), dim3(256), 0, st, part, dw, n, p.splits, accumulate);
    }
    return hific_launch_status();
}

}  // extern "C"
