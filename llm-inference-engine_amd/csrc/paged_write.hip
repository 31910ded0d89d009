// New rows of a ragged batch into the pages of a KV cache, rotated for their own positions.
//
// Rotation pair (a, b) = (x[2i], x[2i+1]) or (x[i], x[i + hs/2]) at position p, with the tables' column 2i:
//   a' = a cos - b sin,  b' = a sin + b cos        (rope_kernel.cu:5-36, 98-128)
// One workgroup takes a row.  A thread keeps the sin/cos of its pairs (16 bytes of elements in each half of the pairs) in
// registers and walks the heads of q, k and v with them, the next head's elements requested ahead of the current
// one's stores; the first are requested before anything else, beside the search for the row's sequence, which
// probes cu_rows at 64 places at a time (a bisection of 64 sequences waited six times).
//
// Copy bound: each element is read once and written once; 168 MB of bf16 prompts in 36 us (4.6 TB/s, what a large copy
// reaches here is 4.7).
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

// cu[b] <= row < cu[b + 1], or -1.  `cu` is non-decreasing; any other order ends as well, within its bounds.
__device__ __forceinline__ int sequence_of_row(const PagedWriteArgs& a, int row) {
  const int lane = lane_id();
  int lo = 0, hi = a.kv.batch;
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) / 64, at = lo + (lane + 1) * step;
    const bool behind = at < hi && *KX_CK(a, PW_CU, a.cu + min(at, hi)) <= row;
    lo += __builtin_popcountll(__ballot(behind)) * step;
    hi = min(lo + step, hi);
  }
  const bool inside = *KX_CK(a, PW_CU, a.cu + lo) <= row && *KX_CK(a, PW_CU, a.cu + lo + 1) > row;
  return inside ? lo : -1;
}

// 16 bytes of a source row, widened
template <typename S, int V>
__device__ __forceinline__ void load_run(const S* p, float (&o)[V]) {
  typedef S vec __attribute__((ext_vector_type(V)));
  const vec v = *reinterpret_cast<const vec*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) o[i] = (float)v[i];
}
template <typename C, int V>
__device__ __forceinline__ void store_run(C* p, const float (&x)[V]) {
  typedef C vec __attribute__((ext_vector_type(V)));
  vec v;
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = round_to<C>(x[i]);
  *reinterpret_cast<vec*>(p) = v;
}

template <typename S, typename C, int VARIANT>
__global__ __launch_bounds__(128) void paged_write_kernel(const PagedWriteArgs a) {
  constexpr int V = 16 / sizeof(S);
  const int row = blockIdx.x, hs = a.head_size, per_head = hs / (2 * V);
  // a thread's elements of a head: two runs, the first and the second elements of V pairs, or with interleaved pairs 2 V
  // consecutive elements
  const int piece = threadIdx.x % per_head, first = threadIdx.x / per_head, step = blockDim.x / per_head;
  const int d0 = VARIANT == KX_ROPE_INTERLEAVED ? 2 * V * piece : V * piece;
  const int d1 = VARIANT == KX_ROPE_INTERLEAVED ? d0 + V : d0 + hs / 2;
  const int total = a.head_num + 2 * a.kv_heads;
  auto load_head = [&](int h, float (&x)[V], float (&y)[V]) {
    const S* src;
    int operand = PW_Q;
    (void)operand;
    if (h < a.head_num) {
      src = static_cast<const S*>(a.q) + row * a.q_stride;
    } else if (h < a.head_num + a.kv_heads) {
      src = static_cast<const S*>(a.k) + row * a.k_stride;
      h -= a.head_num;
      operand = PW_K;
    } else {
      src = static_cast<const S*>(a.v) + row * a.v_stride;
      h -= a.head_num + a.kv_heads;
      operand = PW_V;
    }
    src += (int64_t)h * hs;
    load_run<S, V>(KX_CKN(a, operand, src + d0, 16), x);
    load_run<S, V>(KX_CKN(a, operand, src + d1, 16), y);
  };
  float x[V], y[V];
  if (first < total) load_head(first, x, y);

  const int b = __builtin_amdgcn_readfirstlane(sequence_of_row(a, row));
  if (b < 0) return;
  const int64_t at = (int64_t)row - *KX_CK(a, PW_CU, a.cu + b + 1) + *KX_CK(a, PW_LENS, a.kv.seq_lens + b);  // below the length
  if (at < 0 || (a.sin_cache && at >= a.table_rows)) return;
  const int pos = (int)at, page_col = a.kv.div.page(pos);
  int page = -1;
  if (pos < a.kv.capacity()) page = *KX_CK(a, PW_TABLE, a.kv.table + (b * a.kv.table_stride + page_col));
  const bool filed = page >= 0 && page < a.kv.num_pages;
  const int64_t slot = page * a.kv.page_stride + (pos - page_col * a.kv.div.size) * a.kv.row_stride;
  float sn[V], cs[V];
  if (a.sin_cache) {
    const float* st = a.sin_cache + (size_t)pos * hs;
    const float* ct = a.cos_cache + (size_t)pos * hs;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int col = VARIANT == KX_ROPE_INTERLEAVED ? d0 + 2 * i : 2 * (d0 + i);
      sn[i] = *KX_CK(a, PW_SIN, st + col);
      cs[i] = *KX_CK(a, PW_COS, ct + col);
    }
  }
  for (int h = first; h < total; h += step) {
    float nx[V], ny[V];
    if (h + step < total) load_head(h + step, nx, ny);
    const bool is_q = h < a.head_num, is_k = !is_q && h < a.head_num + a.kv_heads;
    if ((is_q || is_k) && a.sin_cache) {
      if (VARIANT == KX_ROPE_INTERLEAVED) {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
          const float p = x[2 * i], r = x[2 * i + 1], s = y[2 * i], t = y[2 * i + 1];
          x[2 * i] = p * cs[i] - r * sn[i];
          x[2 * i + 1] = p * sn[i] + r * cs[i];
          y[2 * i] = s * cs[V / 2 + i] - t * sn[V / 2 + i];
          y[2 * i + 1] = s * sn[V / 2 + i] + t * cs[V / 2 + i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float p = x[i], r = y[i];
          x[i] = p * cs[i] - r * sn[i];
          y[i] = p * sn[i] + r * cs[i];
        }
      }
    }
    if (is_q) {
      S* dst = static_cast<S*>(a.q_out) + row * a.q_out_stride + (int64_t)h * hs;
      store_run<S, V>(KX_CKN(a, PW_QOUT, dst + d0, 16), x);
      store_run<S, V>(KX_CKN(a, PW_QOUT, dst + d1, 16), y);
    } else if (filed) {
      const int hk = is_k ? h - a.head_num : h - a.head_num - a.kv_heads;
      C* dst = reinterpret_cast<C*>(is_k ? a.key : a.value) + slot + hk * a.kv.head_stride;
      store_run<C, V>(KX_CKN(a, is_k ? PW_KEY : PW_VALUE, dst + d0, V * sizeof(C)), x);
      store_run<C, V>(KX_CKN(a, is_k ? PW_KEY : PW_VALUE, dst + d1, V * sizeof(C)), y);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      x[i] = nx[i];
      y[i] = ny[i];
    }
  }
}

template <typename S, typename C>
static void paged_write_launch(const PagedWriteArgs& a, int variant, hipStream_t stream) {
  // Small workgroups that walk several heads keep more rows in flight: 6.9 k rows of 48 bf16 heads of 128 take 36.3 us with
  // 64 threads, 37.4 with 128, 43.7 with 256, 54.4 with one thread per piece; fp32 into fp16, with twice the pieces, 64.5
  // with 64 and 61.8 with 128; 10 fp32 heads 27.2 with 64, 35.0 with 128.
  const int pieces = (a.head_num + 2 * a.kv_heads) * a.head_size * (int)sizeof(S) / 32;
  const dim3 grid(a.rows), block(pieces >= 512 ? 128 : 64);
  if (variant == KX_ROPE_INTERLEAVED)
    hipLaunchKernelGGL((paged_write_kernel<S, C, KX_ROPE_INTERLEAVED>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((paged_write_kernel<S, C, KX_ROPE_HALF_SPLIT>), grid, block, 0, stream, a);
}

}  // namespace kx

extern "C" int kx_paged_write(const kx_paged_write_desc* d, void* stream) {
  using namespace kx;
  if (!d) return KX_EINVAL;
  if (d->rows < 0 || d->kv.batch < 0) return KX_EINVAL;
  if (d->rows == 0 || d->kv.batch == 0) return KX_OK;
  if (const int rc = paged_check(d->kv)) return rc;
  if (!kind_known(d->src_type) || !d->cu_rows || !aligned4(d->cu_rows) || !d->k || !d->v) return KX_EINVAL;
  if (!kinds_fit(d->src_type, d->kv.type)) return KX_EUNSUPPORTED;
  if (d->rope_variant != KX_ROPE_INTERLEAVED && d->rope_variant != KX_ROPE_HALF_SPLIT) return KX_EINVAL;
  const bool rope = d->sin_cache != nullptr;
  if (rope != (d->cos_cache != nullptr) || (rope && d->table_rows <= 0) || !aligned4(d->sin_cache) || !aligned4(d->cos_cache))
    return KX_EINVAL;
  if ((d->q != nullptr) != (d->q_out != nullptr) || (d->q && (!rope || d->head_num <= 0))) return KX_EINVAL;
  const int64_t kv_dim = (int64_t)d->kv.kv_head_num * d->kv.head_size, q_dim = (int64_t)d->head_num * d->kv.head_size;
  const size_t unit = 16 / kind_bytes(d->src_type);
  if (!stride_ok(d->k_stride, kv_dim, unit) || !stride_ok(d->v_stride, kv_dim, unit)) return KX_EINVAL;
  if (d->q && (!stride_ok(d->q_stride, q_dim, unit) || !stride_ok(d->q_out_stride, q_dim, unit))) return KX_EINVAL;
  if (!aligned16(d->k) || !aligned16(d->v) || !aligned16(d->q) || !aligned16(d->q_out)) return KX_EINVAL;
  if (d->q && d->q == d->q_out && d->q_stride != d->q_out_stride) return KX_EINVAL;  // one row's results over another's elements
  if (!grid_fits(d->rows, 128) || (d->q ? q_dim : 0) + 2 * kv_dim > 0x3fffffff) return KX_ELIMIT;
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
