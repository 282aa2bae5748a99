// prompt_ops.cu -- entry points of the prompt operators: argument checks of
// qi_prompt_attention and qi_linear_16bit, and their common error report.
// Nothing here allocates or keeps state between calls; what is refused is
// refused before anything is launched.
#include "qi_internal.h"

using namespace qi;

namespace {
bool misaligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

// The byte ranges [a, a + na) and [b, b + nb) share a byte.
bool overlap(const void* a, long long na, const void* b, long long nb) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return a && b && na > 0 && nb > 0 && x < y + static_cast<uintptr_t>(nb) && y < x + static_cast<uintptr_t>(na);
}

// Bytes of a [rows, cols] matrix with leading dimension ld.
long long span(long long rows, long long cols, long long ld, int esize) {
  return rows > 0 && cols > 0 ? ((rows - 1) * ld + cols) * esize : 0;
}

// A stride the kernels take: positive, whole 16-byte steps, within a TMA
// descriptor's 40 bits.  A dimension of one element has no stride to check.
int check_stride(long long stride, long long n) {
  if (n <= 1) return QI_OK;
  if (stride <= 0 || stride >= (1ll << 38)) return QI_ERR_ARG;
  return stride % 8 ? QI_ERR_ALIGN : QI_OK;
}

// [rows][heads][dim] elements of 2 bytes at p, stepping row and head elements.
struct Strided {
  const void* p;
  long long rows, heads, dim, row, head;
  long long bytes() const {
    return rows > 0 ? 2 * ((rows > 1 ? (rows - 1) * row : 0) + (heads > 1 ? (heads - 1) * head : 0) + dim) : 0;
  }
};

// Whether two such tensors may share an element.  Apart: disjoint byte ranges,
// or (views into the rows of one buffer) the same row stride, with each row's
// heads of the one clear of the other's.
bool may_share(const Strided& a, const Strided& b) {
  if (!overlap(a.p, a.bytes(), b.p, b.bytes())) return false;
  if (a.rows <= 1 || b.rows <= 1 || a.row != b.row) return true;
  const long long fa = (a.heads > 1 ? (a.heads - 1) * a.head : 0) + a.dim, fb = (b.heads > 1 ? (b.heads - 1) * b.head : 0) + b.dim;
  const long long diff = (static_cast<long long>(reinterpret_cast<uintptr_t>(b.p)) -
                          static_cast<long long>(reinterpret_cast<uintptr_t>(a.p))) / 2;
  const long long d = ((diff % a.row) + a.row) % a.row;  // where b's heads start in a's rows
  return d < fa || d + fb > a.row;
}

constexpr int kMaxExtent = 1 << 30;  // rows, columns: index arithmetic in int with room for a tile

int check_sizes(int heads, int kv_heads, int head_dim, int batch, int total_q, int total_k, int max_k) {
  if (heads < 1 || kv_heads < 1 || heads % kv_heads || head_dim < 1) return QI_ERR_ARG;
  if (batch < 0 || total_q < 0 || total_k < 0 || max_k < 0) return QI_ERR_ARG;
  if (head_dim % 8 || head_dim > 128 || heads > 65535) return QI_ERR_UNSUPPORTED;
  if (total_q > kMaxExtent || total_k > kMaxExtent) return QI_ERR_UNSUPPORTED;
  return QI_OK;
}
}  // namespace

extern "C" long long qi_prompt_attention_workspace(int heads, int kv_heads, int head_dim, int batch, int total_q,
                                                   int total_k, int max_k) {
  const int st = check_sizes(heads, kv_heads, head_dim, batch, total_q, total_k, max_k);
  if (st != QI_OK) return -st;
  return prompt_attention_workspace(heads, kv_heads, head_dim, batch, total_q, max_k);
}

extern "C" int qi_prompt_attention(const void* q, long long q_row, long long q_head, const void* k, long long k_row,
                                   long long k_head, const void* v, long long v_row, long long v_head, void* out,
                                   long long o_row, long long o_head, int dtype, int heads, int kv_heads, int head_dim,
                                   const int* q_begin, const int* q_end, const int* k_begin, const int* k_end,
                                   int batch, int total_q, int total_k, int max_k, float scale, int causal,
                                   void* workspace, long long workspace_bytes, void* stream) {
  int st = check_sizes(heads, kv_heads, head_dim, batch, total_q, total_k, max_k);
  if (st != QI_OK) return st;
  if (dtype != QI_DT_BF16 && dtype != QI_DT_F16) return QI_ERR_ARG;
  if (!(scale > -2.0e38f && scale < 2.0e38f)) return QI_ERR_ARG;  // scale log2(e) is finite
  if (batch == 0 || total_q == 0) return QI_OK;
  if (!q || !out || !q_begin || !q_end || !k_begin || !k_end) return QI_ERR_ARG;
  if (total_k > 0 && (!k || !v)) return QI_ERR_ARG;
  const long long strides[8][2] = {{q_row, total_q}, {q_head, heads},    {k_row, total_k}, {k_head, kv_heads},
                                   {v_row, total_k}, {v_head, kv_heads}, {o_row, total_q}, {o_head, heads}};
  for (const auto& s : strides)
    if ((st = check_stride(s[0], s[1])) != QI_OK) return st;
  // rows and heads of out apart from one another: one of the two dimensions
  // steps over everything the other one spans
  const long long row_span = heads > 1 ? (heads - 1) * o_head + head_dim : head_dim;
  const long long head_span = total_q > 1 ? (total_q - 1) * o_row + head_dim : head_dim;
  if (heads > 1 && o_head < head_dim) return QI_ERR_ARG;
  if (total_q > 1 && o_row < head_dim) return QI_ERR_ARG;
  if (heads > 1 && total_q > 1 && o_row < row_span && o_head < head_span) return QI_ERR_ARG;
  if (misaligned(q) || misaligned(k) || misaligned(v) || misaligned(out)) return QI_ERR_ALIGN;
  if (workspace && misaligned(workspace)) return QI_ERR_ALIGN;
  const Strided sq{q, total_q, heads, head_dim, q_row, q_head}, so{out, total_q, heads, head_dim, o_row, o_head};
  const Strided sk{k, total_k, kv_heads, head_dim, k_row, k_head}, sv{v, total_k, kv_heads, head_dim, v_row, v_head};
  const bool in_place = out == q && (total_q <= 1 || o_row == q_row) && (heads <= 1 || o_head == q_head);
  if ((!in_place && may_share(so, sq)) || may_share(so, sk) || may_share(so, sv)) return QI_ERR_ARG;
  const long long need = prompt_attention_workspace(heads, kv_heads, head_dim, batch, total_q, max_k);
  if (need > 0 && (!workspace || workspace_bytes < need)) return QI_ERR_ARG;
  PromptAttnArgs a{q, k, v, out, q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head, dtype, heads, kv_heads,
                   head_dim, q_begin, q_end, k_begin, k_end, batch, total_q, total_k, max_k, scale, causal != 0,
                   workspace};
  return prompt_attention_launch(a, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int qi_linear_16bit(const void* x, long long ldx, int M, int K, const void* w, long long ldw, int N,
                               int dtype, const void* bias, int act, const float* gate, const void* residual,
                               long long ldr, void* out, long long ldo, int out_dtype, void* stream) {
  if (dtype != QI_DT_BF16 && dtype != QI_DT_F16) return QI_ERR_ARG;
  if (out_dtype != dtype && out_dtype != QI_DT_F32) return QI_ERR_ARG;
  if (act < QI_ACT_NONE || act > QI_ACT_SWIGLU) return QI_ERR_ARG;
  if (M < 0 || N < 1 || K < 1) return QI_ERR_ARG;
  const long long wide = act == QI_ACT_SWIGLU ? 2 : 1;
  if (M > kMaxExtent || K > kMaxExtent || wide * N > kMaxExtent) return QI_ERR_UNSUPPORTED;
  if (M == 0) return QI_OK;
  if (!x || !w || !out) return QI_ERR_ARG;
  const long long lim = 1ll << 38;
  if (ldx < K || ldw < K || ldo < N || (residual && ldr < N)) return QI_ERR_ARG;
  if (ldx >= lim || ldw >= lim || ldo >= lim || (residual && ldr >= lim)) return QI_ERR_ARG;
  const int osize = out_dtype == QI_DT_F32 ? 4 : 2;
  if (ldx % 8 || ldw % 8 || (ldo * osize) % 16 || (residual && (ldr * osize) % 16)) return QI_ERR_ALIGN;
  if (misaligned(x) || misaligned(w) || misaligned(out) || misaligned(bias) || misaligned(gate) || misaligned(residual))
    return QI_ERR_ALIGN;
  const long long no = span(M, N, ldo, osize);
  if (overlap(out, no, x, span(M, K, ldx, 2)) || overlap(out, no, w, span(wide * N, K, ldw, 2)) ||
      overlap(out, no, bias, wide * N * 2) || overlap(out, no, gate, 4ll * N))
    return QI_ERR_ARG;
  if (residual && !(residual == out && ldr == ldo) && overlap(out, no, residual, span(M, N, ldr, osize)))
    return QI_ERR_ARG;
  Linear16Args a{x, w, bias, gate, residual, out, ldx, ldw, ldr, ldo, M, N, K, dtype, out_dtype, act};
  return linear16_launch(a, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int qi_prompt_ops_check(void) {
  if (cudaDeviceSynchronize() != cudaSuccess) return QI_ERR_CUDA;
  int bad = 0;
  if (prompt_attention_take_error(&bad) != QI_OK || linear16_take_error(&bad) != QI_OK) return QI_ERR_CUDA;
  return bad ? QI_ERR_DEVICE : QI_OK;
}
