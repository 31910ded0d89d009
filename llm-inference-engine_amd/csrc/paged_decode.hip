// Attention of one new token per sequence over the pages of a KV cache.
#include <math.h>

#define KX_FILE_ID 11
#include "attn_simple.hpp"

namespace kx {

struct PagedDecodeArgs {
  PagedView kv;
  const void* q;
  void* out;
  int64_t q_stride, out_stride;
  int32_t head_num, kv_heads, head_size, window;
  float scale;
};

template <typename Q, typename KV>
__global__ __launch_bounds__(256) void paged_decode_simple_kernel(const PagedDecodeArgs a) {
  const int h = blockIdx.x, b = blockIdx.y, kvh = h / (a.head_num / a.kv_heads);
  const int len = min(max(a.kv.seq_lens[b], 0), a.kv.capacity());
  const int lo = a.window > 0 ? max(0, len - a.window) : 0;
  const int32_t* table = a.kv.table + b * a.kv.table_stride;
  auto row_of = [&](int t, bool value) -> const KV* {
    const int col = a.kv.div.page(t), page = table[col];
    if (page < 0 || page >= a.kv.num_pages) return nullptr;
    return reinterpret_cast<const KV*>(value ? a.kv.value : a.kv.key) + page * a.kv.page_stride +
           (t - col * a.kv.div.size) * a.kv.row_stride + kvh * a.kv.head_stride;
  };
  attn_row_simple<Q, KV>(static_cast<const Q*>(a.q) + b * a.q_stride + h * a.head_size,
                         static_cast<Q*>(a.out) + b * a.out_stride + h * a.head_size, a.head_size, lo, len, a.scale, row_of);
}

}  // namespace kx

extern "C" size_t kx_paged_decode_workspace_bytes(int32_t batch, int32_t head_num, int32_t kv_head_num, int32_t head_size) {
  return batch <= 0 || head_num <= 0 || kv_head_num <= 0 || head_num % kv_head_num || head_size <= 0 ? 0 : 256;
}

extern "C" int kx_paged_decode(const kx_paged_decode_desc* d, void* stream) {
  using namespace kx;
  if (!d || d->kv.batch < 0) return KX_EINVAL;
  if (d->kv.batch == 0) return KX_OK;
  if (const int rc = paged_check(d->kv)) return rc;
  if (!kind_known(d->q_type) || d->head_num <= 0 || d->head_num % d->kv.kv_head_num || d->window < 0) return KX_EINVAL;
  if (!kinds_fit(d->q_type, d->kv.type)) return KX_EUNSUPPORTED;
  const int64_t q_dim = (int64_t)d->head_num * d->kv.head_size;
  const size_t unit = 16 / kind_bytes(d->q_type);
  if (!d->q || !d->out || !aligned16(d->q) || !aligned16(d->out) || !stride_ok(d->q_stride, q_dim, unit) ||
      !stride_ok(d->out_stride, q_dim, unit))
    return KX_EINVAL;
  if (!d->workspace || d->workspace_bytes < kx_paged_decode_workspace_bytes(d->kv.batch, d->head_num, d->kv.kv_head_num, d->kv.head_size))
    return KX_EWORKSPACE;
  if ((uintptr_t)d->workspace % 256) return KX_EINVAL;
  PagedDecodeArgs a{paged_view(d->kv), d->q, d->out, d->q_stride, d->out_stride, d->head_num, d->kv.kv_head_num,
                    d->kv.head_size, d->window, d->scale};
  const dim3 grid(d->head_num, d->kv.batch), block(256);
  hipStream_t s = (hipStream_t)stream;
#define KX_GO(Q_, C_) hipLaunchKernelGGL((paged_decode_simple_kernel<Q_, C_>), grid, block, 0, s, a)
  if (d->q_type == KX_F16) KX_GO(_Float16, _Float16);
  else if (d->q_type == KX_BF16) KX_GO(__bf16, __bf16);
  else if (d->kv.type == KX_F16) KX_GO(float, _Float16);
  else if (d->kv.type == KX_BF16) KX_GO(float, __bf16);
  else KX_GO(float, float);
#undef KX_GO
  KX_LAUNCH_CHECK();
  return KX_OK;
}
