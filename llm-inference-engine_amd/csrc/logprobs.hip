// Log probabilities of given tokens, entropy and the best alternatives of rows of logits.
#include <math.h>

#define KX_FILE_ID 13
#include "paged.hpp"

namespace kx {

struct LogprobsArgs {
  const void* logits;
  const int32_t* tokens;
  float* logprob;
  float* entropy;
  int32_t* top_ids;
  float* top_logprobs;
  int64_t row_stride;
  int32_t rows, vocab, top_n;
};

// Order of the alternatives as an unsigned whole number: larger value first, the lower index ahead among equal
// ones, NaN below -inf.
__device__ __forceinline__ unsigned long long rank_of(float x, int index) {
  unsigned u = __float_as_uint(x == 0.f ? 0.f : x);
  u = u >> 31 ? ~u : u | 0x80000000u;  // monotone in x
  if (x != x) u = 0u;
  return (unsigned long long)u << 32 | (0xffffffffu - (unsigned)index);
}

__device__ __forceinline__ unsigned long long wave_max_u64(unsigned long long v) {
  for (int off = 32; off; off >>= 1) {
    const unsigned long long o = __shfl_xor(v, off);
    v = o > v ? o : v;
  }
  return v;
}

template <typename T>
__global__ __launch_bounds__(256) void logprobs_simple_kernel(const LogprobsArgs a) {
  __shared__ float red[4], red2[4];
  __shared__ unsigned long long best[4];
  const int row = blockIdx.x, tid = threadIdx.x;
  const T* x = static_cast<const T*>(a.logits) + row * a.row_stride;
  float m = -INFINITY;
  bool odd = false;
  for (int i = tid; i < a.vocab; i += 256) {
    const float v = (float)x[i];
    odd |= v != v || v == INFINITY;
    m = fmaxf(m, v);
  }
  odd = __syncthreads_or(odd);
  m = wave_max(m);
  if ((tid & 63) == 0) red[tid >> 6] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  odd |= m == -INFINITY;
  __syncthreads();
  float z = 0.f, s = 0.f;
  for (int i = tid; i < a.vocab; i += 256) {
    const float d = (float)x[i] - m, e = expf(d);
    z += e;
    if (e > 0.f) s = fmaf(d, e, s);
  }
  z = wave_sum(z);
  s = wave_sum(s);
  if ((tid & 63) == 0) red[tid >> 6] = z, red2[tid >> 6] = s;
  __syncthreads();
  z = (red[0] + red[1]) + (red[2] + red[3]);
  s = (red2[0] + red2[1]) + (red2[2] + red2[3]);
  const float lz = odd ? NAN : logf(z);
  if (tid == 0) {
    if (a.logprob) {
      const int t = a.tokens[row];
      a.logprob[row] = t < 0 ? 0.f : t >= a.vocab ? NAN : ((float)x[t] - m) - lz;
    }
    if (a.entropy) a.entropy[row] = lz - s / z;
  }
  unsigned long long below = ~0ull;
  for (int n = 0; n < a.top_n; ++n) {
    unsigned long long b = 0;
    for (int i = tid; i < a.vocab; i += 256) {
      const unsigned long long r = rank_of((float)x[i], i);
      if (r < below && r > b) b = r;
    }
    b = wave_max_u64(b);
    __syncthreads();
    if ((tid & 63) == 0) best[tid >> 6] = b;
    __syncthreads();
    for (int w = 0; w < 4; ++w) b = best[w] > b ? best[w] : b;
    below = b;
    if (tid == 0) {
      const int i = (int)(0xffffffffu - (unsigned)b);
      a.top_ids[(size_t)row * a.top_n + n] = i;
      a.top_logprobs[(size_t)row * a.top_n + n] = ((float)x[i] - m) - lz;
    }
  }
}

}  // namespace kx

extern "C" size_t kx_token_logprobs_workspace_bytes(int32_t rows, int32_t vocab, int32_t top_n) { return rows <= 0 || vocab <= 0 || top_n < 0 ? 0 : 256; }

extern "C" int kx_token_logprobs(const kx_logprobs_desc* d, void* stream) {
  using namespace kx;
  if (!d || d->rows < 0) return KX_EINVAL;
  if (d->rows == 0) return KX_OK;
  if (!kind_known(d->type) || !d->logits || (uintptr_t)d->logits % kind_bytes(d->type) || d->vocab <= 0 || d->row_stride < d->vocab)
    return KX_EINVAL;
  if ((d->tokens != nullptr) != (d->logprob != nullptr)) return KX_EINVAL;
  if (d->top_n < 0 || d->top_n > KX_LOGPROBS_TOP_MAX || d->top_n > d->vocab) return KX_EINVAL;
  if (d->top_n > 0 && (!d->top_ids || !d->top_logprobs)) return KX_EINVAL;
  if (!d->workspace || d->workspace_bytes < kx_token_logprobs_workspace_bytes(d->rows, d->vocab, d->top_n)) return KX_EWORKSPACE;
  if ((uintptr_t)d->workspace % 256) return KX_EINVAL;
  LogprobsArgs a{d->logits, d->tokens, d->logprob, d->entropy, d->top_ids, d->top_logprobs, d->row_stride, d->rows, d->vocab, d->top_n};
  hipStream_t s = (hipStream_t)stream;
  if (d->type == KX_F16) hipLaunchKernelGGL(logprobs_simple_kernel<_Float16>, dim3(d->rows), dim3(256), 0, s, a);
  else if (d->type == KX_BF16) hipLaunchKernelGGL(logprobs_simple_kernel<__bf16>, dim3(d->rows), dim3(256), 0, s, a);
  else hipLaunchKernelGGL(logprobs_simple_kernel<float>, dim3(d->rows), dim3(256), 0, s, a);
  KX_LAUNCH_CHECK();
  return KX_OK;
}
