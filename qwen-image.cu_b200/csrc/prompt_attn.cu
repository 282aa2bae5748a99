// prompt_attn.cu -- softmax attention over packed sequences with grouped heads.
//
// One warp per (query, head) walks the keys the query sees with a running
// maximum m and sum l (FP32, base 2): for score s = scale * log2(e) * q.k,
//   m' = max(m, s), l' = l 2^(m-m') + 2^(s-m'), o' = o 2^(m-m') + 2^(s-m') v,
// and out = o / l, or 0 when no key is seen.
#include "qi_internal.h"
#include "sm100.cuh"

namespace qi {
namespace {

__device__ int g_prompt_attn_err;

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }

template <typename T>
__global__ void __launch_bounds__(256) prompt_attn_kernel(const __grid_constant__ PromptAttnArgs a) {
  const int b = blockIdx.y, h = blockIdx.z, lane = threadIdx.x & 31;
  const int q0 = min(max(a.q_begin[b], 0), a.total_q), q1 = min(max(a.q_end[b], q0), a.total_q);
  const int k0 = min(max(a.k_begin[b], 0), a.total_k), k1 = min(max(a.k_end[b], k0), a.total_k);
  const int i = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (i >= q1 - q0) return;
  const int seen = a.causal ? min(k1 - k0, max(0, i + 1 + (k1 - k0) - (q1 - q0))) : k1 - k0;
  const int hk = h / (a.heads / a.kv_heads);
  const T* q = static_cast<const T*>(a.q) + static_cast<long long>(q0 + i) * a.q_row + h * a.q_head;
  const T* k = static_cast<const T*>(a.k) + static_cast<long long>(k0) * a.k_row + hk * a.k_head;
  const T* v = static_cast<const T*>(a.v) + static_cast<long long>(k0) * a.v_row + hk * a.v_head;
  const float s2 = a.scale * 1.4426950408889634f;
  float qr[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
  for (int e = 0; e < 4; ++e) qr[e] = lane + 32 * e < a.head_dim ? to_f32(q[lane + 32 * e]) : 0.f;
  for (int j = 0; j < seen; ++j) {
    float s = 0.f;
    for (int e = 0; e < 4; ++e)
      if (lane + 32 * e < a.head_dim) s += qr[e] * to_f32(k[j * a.k_row + lane + 32 * e]);
    for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    s *= s2;
    const float mn = fmaxf(m, s), al = m == -INFINITY ? 0.f : exp2f(m - mn), p = exp2f(s - mn);
    m = mn;
    l = l * al + p;
    for (int e = 0; e < 4; ++e)
      if (lane + 32 * e < a.head_dim) o[e] = o[e] * al + p * to_f32(v[j * a.v_row + lane + 32 * e]);
  }
  T* out = static_cast<T*>(a.out) + static_cast<long long>(q0 + i) * a.o_row + h * a.o_head;
  for (int e = 0; e < 4; ++e)
    if (lane + 32 * e < a.head_dim) out[lane + 32 * e] = from_f32<T>(seen ? o[e] / l : 0.f);
}

}  // namespace

long long prompt_attention_workspace(int heads, int kv_heads, int head_dim, int batch, int total_q, int max_k) {
  return 0;
}

int prompt_attention_launch(const PromptAttnArgs& a, cudaStream_t stream) {
  const dim3 grid((a.total_q + 7) / 8, a.batch, a.heads);
  if (a.dtype == QI_DT_BF16)
    prompt_attn_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>(a);
  else
    prompt_attn_kernel<__half><<<grid, 256, 0, stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? QI_OK : QI_ERR_CUDA;
}

int prompt_attention_take_error(int* bad) {
  int h = 0;
  if (cudaMemcpyFromSymbol(&h, g_prompt_attn_err, sizeof(int)) != cudaSuccess) return QI_ERR_CUDA;
  if (h) {
    *bad = 1;
    h = 0;
    if (cudaMemcpyToSymbol(g_prompt_attn_err, &h, sizeof(int)) != cudaSuccess) return QI_ERR_CUDA;
  }
  return QI_OK;
}

}  // namespace qi
