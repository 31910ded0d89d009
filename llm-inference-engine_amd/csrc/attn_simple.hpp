// One query head over the key rows lo..hi-1 by one workgroup of 256 threads: the definition with an online
// softmax, 256 keys at a time.  `row_of(t, v)`: the address of key (value) row t, or null for a row that is not there.
#pragma once
#include "paged.hpp"

namespace kx {

template <typename Q, typename KV, typename RowOf>
__device__ void attn_row_simple(const Q* q, Q* out, int hs, int lo, int hi, float scale, const RowOf& row_of) {
  __shared__ float sq[128], sp[256], red[4], so[256];
  const int tid = threadIdx.x;
  if (tid < hs) sq[tid] = (float)q[tid];
  float m = -INFINITY, l = 0.f, o = 0.f;  // o: dim tid % hs, keys of the chunk congruent to tid / hs
  const int parts = 256 / hs, d = tid % hs, part = tid / hs;
  for (int t0 = lo; t0 < hi; t0 += 256) {
    __syncthreads();
    const int t = t0 + tid;
    const KV* kr = t < hi ? reinterpret_cast<const KV*>(row_of(t, false)) : nullptr;
    float s = -INFINITY;
    if (kr) {
      s = 0.f;
      for (int i = 0; i < hs; i += 4) {
        float k4[4];
        load4(kr + i, k4);
        for (int e = 0; e < 4; ++e) s = fmaf(k4[e], sq[i + e], s);
      }
      s *= scale;
    }
    float mx = wave_max(s);
    if ((tid & 63) == 0) red[tid >> 6] = mx;
    __syncthreads();
    mx = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float m_new = fmaxf(m, mx), base = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = expf(m - base), p = expf(s - base);
    m = m_new;
    sp[tid] = p;
    __syncthreads();
    const float sum = wave_sum(p);
    if ((tid & 63) == 0) red[tid >> 6] = sum;
    __syncthreads();
    l = l * alpha + ((red[0] + red[1]) + (red[2] + red[3]));
    o *= alpha;
    for (int j = part; j < 256 && t0 + j < hi; j += parts) {
      const KV* vr = sp[j] != 0.f ? reinterpret_cast<const KV*>(row_of(t0 + j, true)) : nullptr;
      if (vr) o = fmaf(sp[j], (float)vr[d], o);
    }
  }
  so[tid] = o;
  __syncthreads();
  if (tid < hs) {
    float sum = 0.f;
    for (int i = 0; i < parts; ++i) sum += so[i * hs + tid];
    out[tid] = (Q)(l == 0.f ? 0.f : sum / l);
  }
}

}  // namespace kx
