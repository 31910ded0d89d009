// What the kernels of batched serving share: element types, the pages of a KV cache, argument checks.
#pragma once
#include "kx_common.hpp"

namespace kx {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ int wave_scan(int v) {  // inclusive prefix sum over the 64 lanes
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);  // row_shr:1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast:15
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row_bcast:31
  return v;
}

// Four consecutive elements, widened exactly.
__device__ __forceinline__ void load4(const float* p, float (&o)[4]) {
  const f32x4 v = *reinterpret_cast<const f32x4*>(p);
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = v[i];
}
__device__ __forceinline__ void load4(const _Float16* p, float (&o)[4]) {
  const f16x4 v = *reinterpret_cast<const f16x4*>(p);
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = (float)v[i];
}
__device__ __forceinline__ void load4(const __bf16* p, float (&o)[4]) {
  const bf16x4 v = *reinterpret_cast<const bf16x4*>(p);
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = (float)v[i];
}

// The one rounding of a result to its type: to nearest even, fp16 saturating at its largest value.
template <typename T> __device__ __forceinline__ T round_to(float x);
template <> __device__ __forceinline__ float round_to<float>(float x) { return x; }
template <> __device__ __forceinline__ _Float16 round_to<_Float16>(float x) { return x != x ? (_Float16)x : sat_f16(x); }
template <> __device__ __forceinline__ __bf16 round_to<__bf16>(float x) { return (__bf16)x; }

// Division of a position by the page size: n / d = (2n * mul) >> (32 + shift) for n < 2^31, with
// 2^shift >= d and mul = ceil(2^(31 + shift) / d) (the rounded-up reciprocal is off by less than one part in
// 2^31, so the quotient of a 31-bit n is exact).
struct PageDiv {
  uint32_t mul;
  int32_t shift, size;
  __device__ int page(int t) const { return (int)(__umulhi((unsigned)t << 1, mul) >> shift); }
};
inline PageDiv page_div(int32_t d) {
  int s = 0;
  while ((1ll << s) < d) ++s;
  return PageDiv{(uint32_t)(((1ull << (31 + s)) + (uint64_t)d - 1) / (uint64_t)d), s, d};
}

// kx_paged_kv as a kernel sees it
struct PagedView {
  const char* key;
  const char* value;
  const int32_t* table;
  const int32_t* seq_lens;
  int64_t page_stride, row_stride, head_stride, table_stride;  // elements
  PageDiv div;
  int32_t num_pages, table_pages, batch;
  __device__ int capacity() const { return table_pages * div.size; }
};
inline PagedView paged_view(const kx_paged_kv& d) {
  return PagedView{static_cast<const char*>(d.key), static_cast<const char*>(d.value), d.table, d.seq_lens,
                   d.page_stride, d.row_stride, d.head_stride, d.table_stride,
                   page_div(d.page_size), d.num_pages, d.table_pages, d.batch};
}
// Positions of a sequence, and elements of a row of logits: the end of a last tile or step still fits 31 bits.
constexpr int64_t kMostPositions = 0x7fffff00ll;
// The tickets of the workgroups that meet in a workspace (64 bytes each) lie ahead of all records, at the same place for
// every call of every entry, whatever its sizes: no call's records ever lie where another's tickets are, so calls of
// different sizes and kinds can follow each other in one workspace.
constexpr size_t kTicketStride = 64, kTicketBytes = 3 * 1024 * kTicketStride;
// a launch has fewer than 2^32 threads
inline bool grid_fits(int64_t blocks, int threads) { return blocks * threads <= 0xffffffffll; }
inline size_t kind_bytes(int32_t kind) { return kind == KX_F32 ? 4 : 2; }
inline bool kind_known(int32_t kind) { return kind == KX_F32 || kind == KX_F16 || kind == KX_BF16; }
inline bool head_size_known(int32_t hs) { return hs == 32 || hs == 64 || hs == 128; }
// a row stride: whole 16-byte pieces, at least the row
inline bool stride_ok(int64_t stride, int64_t least, size_t unit) {
  return stride >= least && stride % (int64_t)unit == 0;
}
inline bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }
inline bool aligned4(const void* p) { return (uintptr_t)p % 4 == 0; }

inline int paged_check(const kx_paged_kv& d) {
  if (!kind_known(d.type) || d.kv_head_num <= 0 || d.page_size <= 0 || d.num_pages <= 0 || d.table_pages <= 0)
    return KX_EINVAL;
  if (!d.key || !d.value || !d.table || !d.seq_lens || !aligned16(d.key) || !aligned16(d.value)) return KX_EINVAL;
  if (!aligned4(d.table) || !aligned4(d.seq_lens)) return KX_EINVAL;
  if (!head_size_known(d.head_size)) return KX_EUNSUPPORTED;
  const size_t unit = 16 / kind_bytes(d.type);
  if (!stride_ok(d.page_stride, d.head_size, unit) || !stride_ok(d.row_stride, d.head_size, unit) ||
      !stride_ok(d.head_stride, d.head_size, unit) || d.table_stride < d.table_pages)
    return KX_EINVAL;
  if ((int64_t)d.page_size * d.table_pages > kMostPositions) return KX_EINVAL;
  return KX_OK;
}
// queries of a type over a cache of a type: fp32 over any, 16-bit ones over their own
inline bool kinds_fit(int32_t q, int32_t kv) { return q == KX_F32 || q == kv; }

}  // namespace kx
