// Attention of packed prompts of different lengths, keys and values packed beside them or in pages.
#include <math.h>

#define KX_FILE_ID 12
#include "attn_simple.hpp"

namespace kx {

struct PromptArgs {
  PagedView kv;  // table: null for packed keys
  const void* q;
  const void* k;
  const void* v;
  void* out;
  const int32_t* cu_q;
  const int32_t* cu_k;
  int64_t q_stride, k_stride, v_stride, out_stride;
  int32_t batch, head_num, kv_heads, head_size, q_rows, k_rows, causal, window;
  float scale;
};

template <typename T>
__global__ __launch_bounds__(256) void prompt_attn_simple_kernel(const PromptArgs a) {
  const int h = blockIdx.x, row = blockIdx.y, kvh = h / (a.head_num / a.kv_heads);
  if (a.cu_q[0] > row || a.cu_q[a.batch] <= row) return;
  int b = 0, up = a.batch;
  while (up - b > 1) {
    const int mid = (b + up) >> 1;
    if (a.cu_q[mid] <= row) b = mid;
    else up = mid;
  }
  int k0 = 0, keys;
  if (a.kv.table) {
    keys = min(max(a.kv.seq_lens[b], 0), a.kv.capacity());
  } else {
    k0 = min(max(a.cu_k[b], 0), a.k_rows);
    keys = max(min(a.cu_k[b + 1], a.k_rows) - k0, 0);
  }
  const int p = keys - a.cu_q[b + 1] + row;  // position of the row
  const int hi = a.causal ? min(p + 1, keys) : keys;
  const int lo = a.window > 0 ? max(0, p - a.window + 1) : 0;
  const int32_t* table = a.kv.table + b * a.kv.table_stride;
  auto row_of = [&](int t, bool value) -> const T* {
    if (!a.kv.table)
      return value ? static_cast<const T*>(a.v) + (k0 + t) * a.v_stride + kvh * a.head_size
                   : static_cast<const T*>(a.k) + (k0 + t) * a.k_stride + kvh * a.head_size;
    const int col = a.kv.div.page(t), page = table[col];
    if (page < 0 || page >= a.kv.num_pages) return nullptr;
    return reinterpret_cast<const T*>(value ? a.kv.value : a.kv.key) + page * a.kv.page_stride +
           (t - col * a.kv.div.size) * a.kv.row_stride + kvh * a.kv.head_stride;
  };
  attn_row_simple<T, T>(static_cast<const T*>(a.q) + row * a.q_stride + h * a.head_size,
                        static_cast<T*>(a.out) + row * a.out_stride + h * a.head_size, a.head_size, lo, hi, a.scale, row_of);
}

}  // namespace kx

extern "C" int kx_prompt_attention(const kx_prompt_attn_desc* d, void* stream) {
  using namespace kx;
  if (!d || d->batch < 0 || d->q_rows < 0) return KX_EINVAL;
  if (d->batch == 0 || d->q_rows == 0) return KX_OK;
  if (!kind_known(d->type) || d->head_num <= 0 || d->kv_head_num <= 0 || d->head_num % d->kv_head_num) return KX_EINVAL;
  if (!head_size_known(d->head_size)) return KX_EUNSUPPORTED;
  if (d->window < 0 || (d->window > 0 && !d->causal)) return KX_EINVAL;
  const int64_t q_dim = (int64_t)d->head_num * d->head_size, kv_dim = (int64_t)d->kv_head_num * d->head_size;
  const size_t unit = 16 / kind_bytes(d->type);
  if (!d->q || !d->out || !d->cu_q || (uintptr_t)d->cu_q % 4 || !aligned16(d->q) || !aligned16(d->out) ||
      !stride_ok(d->q_stride, q_dim, unit) || !stride_ok(d->out_stride, q_dim, unit))
    return KX_EINVAL;
  PromptArgs a{};
  if (d->pages) {
    if (d->k || d->v || d->cu_k) return KX_EINVAL;
    if (const int rc = paged_check(*d->pages)) return rc;
    if (d->pages->type != d->type) return KX_EUNSUPPORTED;
    if (d->pages->kv_head_num != d->kv_head_num || d->pages->head_size != d->head_size || d->pages->batch != d->batch)
      return KX_EINVAL;
    a.kv = paged_view(*d->pages);
  } else {
    if (!d->k || !d->v || !d->cu_k || (uintptr_t)d->cu_k % 4 || d->k_rows < 0 || !aligned16(d->k) || !aligned16(d->v) ||
        !stride_ok(d->k_stride, kv_dim, unit) || !stride_ok(d->v_stride, kv_dim, unit))
      return KX_EINVAL;
  }
  a.q = d->q; a.k = d->k; a.v = d->v; a.out = d->out; a.cu_q = d->cu_q; a.cu_k = d->cu_k;
  a.q_stride = d->q_stride; a.k_stride = d->k_stride; a.v_stride = d->v_stride; a.out_stride = d->out_stride;
  a.batch = d->batch; a.head_num = d->head_num; a.kv_heads = d->kv_head_num; a.head_size = d->head_size;
  a.q_rows = d->q_rows; a.k_rows = d->k_rows; a.causal = d->causal; a.window = d->window; a.scale = d->scale;
  const dim3 grid(d->head_num, d->q_rows), block(256);
  hipStream_t s = (hipStream_t)stream;
  if (d->type == KX_F16) hipLaunchKernelGGL(prompt_attn_simple_kernel<_Float16>, grid, block, 0, s, a);
  else if (d->type == KX_BF16) hipLaunchKernelGGL(prompt_attn_simple_kernel<__bf16>, grid, block, 0, s, a);
  else hipLaunchKernelGGL(prompt_attn_simple_kernel<float>, grid, block, 0, s, a);
  KX_LAUNCH_CHECK();
  return KX_OK;
}
