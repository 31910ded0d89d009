// New rows of a ragged batch into the pages of a KV cache, rotated for their own positions.
//
// Rotation pair (a, b) = (x[2i], x[2i+1]) or (x[i], x[i + hs/2]) at position p, with the tables' column 2i:
//   a' = a cos - b sin,  b' = a sin + b cos        (rope_kernel.cu:5-36, 98-128)
// One workgroup takes a row: finds its sequence by bisection of cu_rows, its place through the table, and then
// every thread keeps the sin/cos of its four pairs in registers and walks the heads of q, k and v with them.
// Copy bound: each element is read once and written once.
#define KX_FILE_ID 10
#include "paged.hpp"

namespace kx {

enum WriteOperand { PW_KEY, PW_VALUE, PW_TABLE, PW_LENS, PW_CU, PW_K, PW_V, PW_Q, PW_QOUT, PW_SIN, PW_COS };

struct PagedWriteArgs {
  PagedView kv;
  char* key;
  char* value;
  const int32_t* cu;
  const void* k;
  const void* v;
  const void* q;
  void* q_out;
  int64_t k_stride, v_stride, q_stride, q_out_stride;
  const float* sin_cache;
  const float* cos_cache;
  int32_t rows, head_num, kv_heads, head_size, table_rows;
  KX_BFIELD(11)
};

// cu[b] <= row < cu[b + 1], or -1.  `cu` is non-decreasing.
__device__ __forceinline__ int sequence_of_row(const PagedWriteArgs& a, int row) {
  int lo = 0, hi = a.kv.batch;  // cu[lo] <= row (if any), cu[hi] > row
  if (*KX_CK(a, PW_CU, a.cu + hi) <= row || *KX_CK(a, PW_CU, a.cu) > row) return -1;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (*KX_CK(a, PW_CU, a.cu + mid) <= row) lo = mid;
    else hi = mid;
  }
  return lo;
}

template <typename S, typename C, int VARIANT>
__global__ __launch_bounds__(256) void paged_write_kernel(const PagedWriteArgs a) {
  const int row = blockIdx.x;
  const int b = sequence_of_row(a, row);
  if (b < 0) return;
  const int len = min(max(*KX_CK(a, PW_LENS, a.kv.seq_lens + b), 0), a.kv.capacity());
  const int64_t at = (int64_t)row - *KX_CK(a, PW_CU, a.cu + b + 1) + len;
  if (at < 0 || at >= len || (a.sin_cache && at >= a.table_rows)) return;
  const int pos = (int)at, page_col = a.kv.div.page(pos);
  const int page = *KX_CK(a, PW_TABLE, a.kv.table + (b * a.kv.table_stride + page_col));
  const bool filed = page >= 0 && page < a.kv.num_pages;
  const int64_t slot = page * a.kv.page_stride + (pos - page_col * a.kv.div.size) * a.kv.row_stride;

  // a thread's eight elements of a head: two runs of four, the first and the second elements of four pairs, or with
  // interleaved pairs the pairs (0, 1), (2, 3) of each run
  const int hs = a.head_size, per_head = hs / 8;
  const int piece = threadIdx.x % per_head, first = threadIdx.x / per_head, step = blockDim.x / per_head;
  const int d0 = VARIANT == KX_ROPE_INTERLEAVED ? 8 * piece : 4 * piece;
  const int d1 = VARIANT == KX_ROPE_INTERLEAVED ? d0 + 4 : d0 + hs / 2;
  float sn[4], cs[4];
  if (a.sin_cache) {
    const float* st = a.sin_cache + (size_t)pos * hs;
    const float* ct = a.cos_cache + (size_t)pos * hs;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int col = VARIANT == KX_ROPE_INTERLEAVED ? d0 + 2 * i : 2 * (d0 + i);
      sn[i] = *KX_CK(a, PW_SIN, st + col);
      cs[i] = *KX_CK(a, PW_COS, ct + col);
    }
  }
  const int total = a.head_num + 2 * a.kv_heads;
  for (int h = first; h < total; h += step) {
    const S* src;
    int hk = h;  // head within its tensor
    const bool is_q = h < a.head_num, is_k = !is_q && h < a.head_num + a.kv_heads;
    if (is_q) {
      src = static_cast<const S*>(a.q) + row * a.q_stride;
    } else if (is_k) {
      hk = h - a.head_num;
      src = static_cast<const S*>(a.k) + row * a.k_stride;
    } else {
      hk = h - a.head_num - a.kv_heads;
      src = static_cast<const S*>(a.v) + row * a.v_stride;
    }
    if (!is_q && !filed) continue;
    const int operand = is_q ? PW_Q : is_k ? PW_K : PW_V;
    (void)operand;
    src += (int64_t)hk * hs;
    float x[4], y[4];
    load4(KX_CKN(a, operand, src + d0, 4 * sizeof(S)), x);
    load4(KX_CKN(a, operand, src + d1, 4 * sizeof(S)), y);
    if ((is_q || is_k) && a.sin_cache) {
      if (VARIANT == KX_ROPE_INTERLEAVED) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float p = x[2 * i], r = x[2 * i + 1], s = y[2 * i], t = y[2 * i + 1];
          x[2 * i] = p * cs[i] - r * sn[i];
          x[2 * i + 1] = p * sn[i] + r * cs[i];
          y[2 * i] = s * cs[2 + i] - t * sn[2 + i];
          y[2 * i + 1] = s * sn[2 + i] + t * cs[2 + i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p = x[i], r = y[i];
          x[i] = p * cs[i] - r * sn[i];
          y[i] = p * sn[i] + r * cs[i];
        }
      }
    }
    if (is_q) {
      S* dst = static_cast<S*>(a.q_out) + row * a.q_out_stride + (int64_t)hk * hs;
      store4(KX_CKN(a, PW_QOUT, dst + d0, 4 * sizeof(S)), x);
      store4(KX_CKN(a, PW_QOUT, dst + d1, 4 * sizeof(S)), y);
    } else {
      C* dst = reinterpret_cast<C*>(is_k ? a.key : a.value) + slot + hk * a.kv.head_stride;
      store4(KX_CKN(a, is_k ? PW_KEY : PW_VALUE, dst + d0, 4 * sizeof(C)), x);
      store4(KX_CKN(a, is_k ? PW_KEY : PW_VALUE, dst + d1, 4 * sizeof(C)), y);
    }
  }
}

template <typename S, typename C>
static void paged_write_launch(const PagedWriteArgs& a, int variant, hipStream_t stream) {
  if (variant == KX_ROPE_INTERLEAVED)
    hipLaunchKernelGGL((paged_write_kernel<S, C, KX_ROPE_INTERLEAVED>), dim3(a.rows), dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((paged_write_kernel<S, C, KX_ROPE_HALF_SPLIT>), dim3(a.rows), dim3(256), 0, stream, a);
}

}  // namespace kx

extern "C" int kx_paged_write(const kx_paged_write_desc* d, void* stream) {
  using namespace kx;
  if (!d) return KX_EINVAL;
  if (d->rows < 0 || d->kv.batch < 0) return KX_EINVAL;
  if (d->rows == 0 || d->kv.batch == 0) return KX_OK;
  if (const int rc = paged_check(d->kv)) return rc;
  if (!kind_known(d->src_type) || !d->cu_rows || (uintptr_t)d->cu_rows % 4 || !d->k || !d->v) return KX_EINVAL;
  if (!kinds_fit(d->src_type, d->kv.type)) return KX_EUNSUPPORTED;
  if (d->rope_variant != KX_ROPE_INTERLEAVED && d->rope_variant != KX_ROPE_HALF_SPLIT) return KX_EINVAL;
  const bool rope = d->sin_cache != nullptr;
  if (rope != (d->cos_cache != nullptr) || (rope && d->table_rows <= 0)) return KX_EINVAL;
  if ((d->q != nullptr) != (d->q_out != nullptr) || (d->q && (!rope || d->head_num <= 0))) return KX_EINVAL;
  const int64_t kv_dim = (int64_t)d->kv.kv_head_num * d->kv.head_size, q_dim = (int64_t)d->head_num * d->kv.head_size;
  if (!stride_ok(d->k_stride, kv_dim, 4) || !stride_ok(d->v_stride, kv_dim, 4)) return KX_EINVAL;
  if (d->q && (!stride_ok(d->q_stride, q_dim, 4) || !stride_ok(d->q_out_stride, q_dim, 4))) return KX_EINVAL;
  if (!aligned16(d->k) || !aligned16(d->v) || !aligned16(d->q) || !aligned16(d->q_out)) return KX_EINVAL;
  PagedWriteArgs a{};
  a.kv = paged_view(d->kv);
  a.key = static_cast<char*>(d->kv.key);
  a.value = static_cast<char*>(d->kv.value);
  a.cu = d->cu_rows;
  a.k = d->k; a.v = d->v; a.q = d->q; a.q_out = d->q_out;
  a.k_stride = d->k_stride; a.v_stride = d->v_stride; a.q_stride = d->q_stride; a.q_out_stride = d->q_out_stride;
  a.sin_cache = d->sin_cache; a.cos_cache = d->cos_cache;
  a.rows = d->rows; a.head_num = d->q ? d->head_num : 0; a.kv_heads = d->kv.kv_head_num;
  a.head_size = d->kv.head_size; a.table_rows = d->table_rows;
  const void* operands[] = {a.key, a.value, a.kv.table, a.kv.seq_lens, a.cu, a.k, a.v, a.q, a.q_out, a.sin_cache, a.cos_cache};
  for (int i = 0; i < 11; ++i) KX_BSET(a, i, operands[i]);
  (void)operands;
  hipStream_t s = (hipStream_t)stream;
  if (d->src_type == KX_F16) paged_write_launch<_Float16, _Float16>(a, d->rope_variant, s);
  else if (d->src_type == KX_BF16) paged_write_launch<__bf16, __bf16>(a, d->rope_variant, s);
  else if (d->kv.type == KX_F16) paged_write_launch<float, _Float16>(a, d->rope_variant, s);
  else if (d->kv.type == KX_BF16) paged_write_launch<float, __bf16>(a, d->rope_variant, s);
  else paged_write_launch<float, float>(a, d->rope_variant, s);
  KX_LAUNCH_CHECK();
  return KX_OK;
}
