// linear16.cu -- linear layer on 16-bit operands with bias, activation, gate
// and residual in the epilogue: 64 x 64 output tiles, FP32 products and sums.
#include "qi_internal.h"
#include "sm100.cuh"

namespace qi {
namespace {

__device__ int g_linear16_err;

__device__ __forceinline__ float sigmoid_f32(float v) { return 1.0f / (1.0f + __expf(-v)); }

template <typename T>
__device__ __forceinline__ float lf(const void* p, long long i) {
  return static_cast<float>(static_cast<const T*>(p)[i]);
}

template <typename T, typename O>
__global__ void __launch_bounds__(256) linear16_kernel(const __grid_constant__ Linear16Args a) {
  __shared__ float sx[16][65], sw[2][16][65];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const long long m0 = blockIdx.y * 64ll, n0 = blockIdx.x * 64ll;
  const bool wide = a.act == QI_ACT_SWIGLU;
  float acc[2][4][4] = {};
  for (int k0 = 0; k0 < a.K; k0 += 16) {
    for (int i = threadIdx.x; i < 64 * 16; i += 256) {
      const int r = i >> 4, c = i & 15;
      const bool in = k0 + c < a.K;
      sx[c][r] = in && m0 + r < a.M ? lf<T>(a.x, (m0 + r) * a.ldx + k0 + c) : 0.f;
      sw[0][c][r] = in && n0 + r < a.N ? lf<T>(a.w, (n0 + r) * a.ldw + k0 + c) : 0.f;
      if (wide) sw[1][c][r] = in && n0 + r < a.N ? lf<T>(a.w, (a.N + n0 + r) * a.ldw + k0 + c) : 0.f;
    }
    __syncthreads();
    for (int c = 0; c < 16; ++c)
      for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
          acc[0][i][j] += sx[c][ty * 4 + i] * sw[0][c][tx * 4 + j];
          if (wide) acc[1][i][j] += sx[c][ty * 4 + i] * sw[1][c][tx * 4 + j];
        }
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const long long m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
      if (m >= a.M || n >= a.N) continue;
      float y = acc[0][i][j];
      if (a.bias) y += lf<T>(a.bias, n);
      if (a.act == QI_ACT_GELU) {
        y *= sigmoid_f32(1.5957691216057308f * (y + 0.044715f * y * y * y));
      } else if (a.act == QI_ACT_SILU) {
        y *= sigmoid_f32(y);
      } else if (wide) {
        float u = acc[1][i][j];
        if (a.bias) u += lf<T>(a.bias, a.N + n);
        y *= sigmoid_f32(y) * u;
      }
      if (a.gate) y *= a.gate[n];
      if (a.residual) y += lf<O>(a.residual, m * a.ldr + n);
      static_cast<O*>(a.out)[m * a.ldo + n] = static_cast<O>(y);
    }
}

}  // namespace

int linear16_launch(const Linear16Args& a, cudaStream_t stream) {
  const dim3 grid((a.N + 63) / 64, (a.M + 63) / 64);
  if (a.dtype == QI_DT_BF16 && a.out_dtype == QI_DT_F32)
    linear16_kernel<__nv_bfloat16, float><<<grid, 256, 0, stream>>>(a);
  else if (a.dtype == QI_DT_BF16)
    linear16_kernel<__nv_bfloat16, __nv_bfloat16><<<grid, 256, 0, stream>>>(a);
  else if (a.out_dtype == QI_DT_F32)
    linear16_kernel<__half, float><<<grid, 256, 0, stream>>>(a);
  else
    linear16_kernel<__half, __half><<<grid, 256, 0, stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? QI_OK : QI_ERR_CUDA;
}

int linear16_take_error(int* bad) {
  int h = 0;
  if (cudaMemcpyFromSymbol(&h, g_linear16_err, sizeof(int)) != cudaSuccess) return QI_ERR_CUDA;
  if (h) {
    *bad = 1;
    h = 0;
    if (cudaMemcpyToSymbol(g_linear16_err, &h, sizeof(int)) != cudaSuccess) return QI_ERR_CUDA;
  }
  return QI_OK;
}

}  // namespace qi
