// norm8_fwd.hip, norm8_bwd.hip: norms that write or read activations in 8 bits (format: act8.h), and the root-mean-square norm.
// Per token t of x [N, C, HW]:
//   RMS norm      h = x (+ resid, rounded to the storage type: the new residual stream),  r = rsqrt(sum_c h^2 / C + eps),
//                 xh = h r,  y = w_c xh
//                 backward: g = w dy,  dx = r (g - xh sum_c(g xh) / C) (+ dstream),  dw_c = sum_t dy xh
//   channel norm  d = x - sum_c x / C,  r = rsqrt(sum_c d^2 / (C - 1) + eps),  xh = d r,
//                 y = relu?(gamma_c xh + beta_c) (+ resid)
//                 backward: dy masked by gamma xh + beta > 0,  g = gamma dy,
//                 dx = r (g - sum_c g / C - xh sum_c(g xh) / (C - 1)),  dgamma_c = sum_t dy xh,  dbeta_c = sum_t dy
// What the backward pass needs of the forward pass is xh and r: xh is kept in 8 bits (1 byte per element in the place of the 2 of
// a bfloat16 input, or of the 4 of input and output), r in float32 per token.  Sums and statistics are float32 throughout.
#pragma once
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

// channels per thread that the plane kernels keep in registers
template <typename T> constexpr int tile_most() { return sizeof(T) == 2 ? 8 : 4; }
