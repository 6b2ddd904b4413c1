// Activation checkpoints in 8 bits (format: act8.h): pack an activation, restore it.  Both are bound by HBM: pack reads T and
// writes 1 byte per element, restore the reverse.
#include "act8.h"

// PX lanes on consecutive positions x 256 / PX channel groups; see norm8.hip for the choice of PX.
template <typename T, int FMT, int PX>
__global__ __launch_bounds__(256) void act8_pack_kernel(const T* __restrict__ x, u8_t* __restrict__ q, u8_t* __restrict__ qe,
                                                        int C, int HW, unsigned tiles) {
    constexpr int G = 256 / PX;
    __shared__ unsigned red[G][PX];
    const int px = threadIdx.x % PX, g = threadIdx.x / PX;
    const unsigned n = blockIdx.x / tiles, hw = (blockIdx.x - n * tiles) * PX + px;
    const bool ok = hw < (unsigned)HW;
    const size_t base = (size_t)n * C * HW + (ok ? hw : 0);
    unsigned am = 0;
    for (int c = g; c < C; c += G) am = umax(am, abs_bits(DT<T>::ld(x + base + (size_t)c * HW)));
    red[g][px] = am;
    __syncthreads();
    for (int k = 0; k < G; ++k) am = umax(am, red[k][px]);
    const unsigned code = q8_code<FMT>(am);
    const float inv = q8_inv_scale(code);
    if (!ok) return;
    if (g == 0) qe[(size_t)n * HW + hw] = (u8_t)code;
    for (int c = g; c < C; c += G) q[base + (size_t)c * HW] = (u8_t)q8_round<FMT>(DT<T>::ld(x + base + (size_t)c * HW) * inv);
}

// out = relu?(gamma_c * (q * 2^e) + beta_c), or q * 2^e where gamma is null
template <typename T, int FMT>
__global__ __launch_bounds__(256) void act8_restore_kernel(const u8_t* __restrict__ q, const u8_t* __restrict__ qe,
                                                           const float* __restrict__ gamma, const float* __restrict__ beta,
                                                           T* __restrict__ out, int C, int HW, long long n, int relu) {
    const long long step = (long long)gridDim.x * 256;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += step) {
        const long long plane = i / HW, img = plane / C;
        float v = q8_value<FMT>(q[i]) * q8_scale(qe[img * HW + (i - plane * HW)]);
        if (gamma) {
            const int c = (int)(plane - img * C);
            v = fmaf(gamma[c], v, beta[c]);
            if (relu) v = v > 0.f ? v : (v != v ? v : 0.f);
        }
        DT<T>::st(out + i, v);
    }
}

extern "C" {

int hific_act8_pack(const void* x, void* q, void* qe, int fmt, int N, int C, int HW, int dtype, hipStream_t st) {
    if (!x || !q || !qe || N <= 0 || C <= 0 || HW <= 0 || !act8_dtype_ok(dtype) || !act8_fmt_ok(fmt)) return HIFIC_ERR_ARG;
    const int px = HW == 1 ? 1 : (HW < 48 ? 16 : 64);
    const long long tiles = cdivl(HW, px), blocks = tiles * N;
    if (blocks > 0x7fffffffll) return HIFIC_ERR_UNSUPPORTED;
#define PACK(T, F, PX) hipLaunchKernelGGL((act8_pack_kernel<T, F, PX>), dim3((unsigned)blocks), dim3(256), 0, st, (const T*)x, \
                                          (u8_t*)q, (u8_t*)qe, C, HW, (unsigned)tiles)
#define PACK_P(T, F) do { if (px == 1) PACK(T, F, 1); else if (px == 16) PACK(T, F, 16); else PACK(T, F, 64); } while (0)
#define PACK_F(T) do { if (fmt == HIFIC_Q_INT8) PACK_P(T, HIFIC_Q_INT8); else PACK_P(T, HIFIC_Q_E4M3); } while (0)
    if (dtype == HIFIC_F32) PACK_F(float); else PACK_F(bf16_t);
#undef PACK_F
#undef PACK_P
#undef PACK
    return hific_launch_status();
}

int hific_act8_restore(const void* q, const void* qe, int fmt, const float* gamma, const float* beta, int relu, void* out,
                       int N, int C, int HW, int dtype, hipStream_t st) {
    if (!q || !qe || !out || N <= 0 || C <= 0 || HW <= 0 || !act8_dtype_ok(dtype) || !act8_fmt_ok(fmt)) return HIFIC_ERR_ARG;
    if ((gamma == nullptr) != (beta == nullptr) || (relu && !gamma)) return HIFIC_ERR_ARG;
    const long long n = (long long)N * C * HW;
    const long long want = cdivl(n, 256);
    const unsigned blocks = (unsigned)(want < 65536 ? want : 65536);
#define REST(T, F) hipLaunchKernelGGL((act8_restore_kernel<T, F>), dim3(blocks), dim3(256), 0, st, (const u8_t*)q,           \
                                      (const u8_t*)qe, gamma, beta, (T*)out, C, HW, n, relu)
#define REST_F(T) do { if (fmt == HIFIC_Q_INT8) REST(T, HIFIC_Q_INT8); else REST(T, HIFIC_Q_E4M3); } while (0)
    if (dtype == HIFIC_F32) REST_F(float); else REST_F(bf16_t);
#undef REST_F
#undef REST
    return hific_launch_status();
}

}  // extern "C"
