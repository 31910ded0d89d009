// Log probabilities of given tokens, entropy and the best alternatives of rows of logits, in one pass over them.
//
//   m = max x,  z = sum e^{x - m},  s = sum (x - m) e^{x - m}
//   log p_t = (x_t - m) - ln z,   entropy = ln z - s / z
//
// Bound: the row is read once (rows * vocab * element size): 623 MB of 16-bit logits in 116 us, 5.4 TB/s, where a plain sum
// over as much memory reads 5.7.  9.4 vector instructions per element take 71 % of the cycles of that time.  A single row
// of 128 k fp32 logits takes 7.9 us, latencies of loads, of the ticket and of code that runs once.
//
// Split: a workgroup takes a row, or with few rows one of up to 32 parts of it; the parts' sums and lists meet in the
// workspace and the workgroup that arrives last joins them in their order.
//
// Alternatives without a second pass: a lane keeps its largest value of all and of each of eight groups of its loads.  The
// top_n-th largest of 64 of them (the largest of four lanes each) is at most the top_n-th largest value, so only the few
// groups that reach it are read again (they are in the caches), their elements dealt over all threads (a wave that walked
// its lanes' groups by itself did so for 64 lanes each time: 142 us instead of 118; elements kept in registers instead, each
// with its own code: 11.2 us for the single row), and those at or above it (some tens) are ranked by counting.
// Where more of them are alike than the list holds, or fewer than top_n are above -inf, the part is gone through in order of
// index instead (the text with three logits a row that are not banned: 252 us).
//
// The reference m is shared by a wave and is the maximum of what it has seen.  So z >= 1, ln z >= 0 and -s / z >= 0: nothing
// cancels, no probability passes one and no entropy falls below zero.  (A reference that followed only when exceeded by 16
// let ln z and x - m, both up to 16, cancel.  Measured in turn against that: the text 116.5 / 116.2 us, one row 7.96 / 7.92; a
// wave meets a new maximum a few times only.)  e^d is taken as a power of two, d log2 e rounded: off by |d| 2^-24 of
// itself, more the smaller its share.
#include <math.h>

#define KX_FILE_ID 13
#include "paged.hpp"

namespace kx {

enum LogprobsOperand { PL_X, PL_TOKENS, PL_LOGPROB, PL_ENTROPY, PL_IDS, PL_TOP, PL_WS };

constexpr int kLpThreads = 256, kLpWaves = kLpThreads / 64;
constexpr int kLpUnroll = 4;      // vectors of 16 bytes in flight per lane
constexpr int kLpGroups = 8;      // groups of a lane's loads
constexpr int kLpList = 512;      // elements that are ranked at once
constexpr int kLpMaxParts = 32;   // of a row
constexpr int kLpSlots = 1024;    // workgroups that few rows are cut for
constexpr int kLpRecord = 16 + 8 * KX_LOGPROBS_TOP_MAX;  // bytes: m, z, s, -, then the list
static_assert(kLpSlots * kTicketStride <= kTicketBytes, "");

struct LogprobsArgs {
  const void* logits;
  const int32_t* tokens;
  float* logprob;
  float* entropy;
  int32_t* top_ids;
  float* top_logprobs;
  char* records;      // [row][part]
  unsigned* tickets;  // [row], 64 bytes apart
  int64_t row_stride;
  int32_t rows, vocab, top_n, parts;
  KX_BFIELD(7)
};

// fp32 values as whole numbers of the same order
__device__ __forceinline__ unsigned order_of(float x) {
  const unsigned u = __float_as_uint(x);
  return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of_order(unsigned u) { return __uint_as_float(u >> 31 ? u ^ 0x80000000u : ~u); }

// At most the n-th largest of the wave's values: its first 16 bits, found from the top (0 with fewer than n above it).
__device__ __forceinline__ unsigned nth_largest(unsigned v, int n) {
  unsigned t = 0;
#pragma unroll
  for (int bit = 31; bit >= 16; --bit) {
    const unsigned c = t | 1u << bit;
    if (__builtin_popcountll(__ballot(v >= c)) >= n) t = c;
  }
  return t;
}

// Order of the alternatives as an unsigned whole number: larger value first, the lower index ahead among equal ones
// (both zeros are equal), NaN below -inf.  No element has key 0.
__device__ __forceinline__ unsigned long long key_of(float x, int index) {
  const unsigned u = x != x ? 0u : order_of(x == 0.f ? 0.f : x);
  return (unsigned long long)u << 32 | (0xffffffffu - (unsigned)index);
}
__device__ __forceinline__ float value_of_key(unsigned long long k) { return value_of_order((unsigned)(k >> 32)); }
__device__ __forceinline__ int index_of_key(unsigned long long k) { return (int)(0xffffffffu - (unsigned)k); }

template <typename T> struct LogitVec;  // 16 bytes of logits
template <> struct LogitVec<float> {
  static constexpr int N = 4;
  static constexpr unsigned kNone = 0xff800000u;  // -inf
  static __device__ __forceinline__ float get(const u32x4& v, int i) { return __uint_as_float(v[i]); }
};
template <> struct LogitVec<_Float16> {
  static constexpr int N = 8;
  static constexpr unsigned kNone = 0xfc00fc00u;
  static __device__ __forceinline__ float get(const u32x4& v, int i) {
    return (float)__builtin_bit_cast(_Float16, (unsigned short)(v[i / 2] >> (i % 2 * 16)));
  }
};
template <> struct LogitVec<__bf16> {
  static constexpr int N = 8;
  static constexpr unsigned kNone = 0xff80ff80u;
  static __device__ __forceinline__ float get(const u32x4& v, int i) {
    return __uint_as_float(i % 2 ? v[i / 2] & 0xffff0000u : v[i / 2] << 16);
  }
};

// sums relative to m
struct LogSums {
  float m, z, s;
};
// The same sums relative to a larger reference.  m = -inf: nothing but -inf so far (z = 0) or nothing but NaN.
__device__ __forceinline__ void rebase(LogSums& a, float m) {
  if (a.m != -INFINITY) {
    const float d = a.m - m, f = __builtin_amdgcn_exp2f(d * 1.4426950408889634f);
    a.s = d > -150.f ? (a.s + a.z * d) * f : a.s * 0.f;
    a.z *= f;
  }
  a.m = m;
}

// The top_n largest of the `count` keys in LDS, in falling order: a key's place is the number of keys above it, which four
// lanes count together.
__device__ __forceinline__ void rank_keys(const unsigned long long* keys, int count, int top_n, unsigned long long* out) {
  const int part = threadIdx.x % 4;
  for (int i = threadIdx.x / 4; i < count; i += kLpThreads / 4) {
    const unsigned long long mine = keys[i];
    int above = 0;
#pragma unroll 4
    for (int j = part; j < count; j += 4) above += keys[j] > mine;
    above += __builtin_amdgcn_update_dpp(0, above, 0xB1, 0xF, 0xF, true);  // the lane's neighbour of a pair
    above += __builtin_amdgcn_update_dpp(0, above, 0x4E, 0xF, 0xF, true);  // the other pair of four
    if (part == 0 && above < top_n) out[above] = mine;
  }
}

template <typename T>
__global__ __launch_bounds__(kLpThreads, 6) void logprobs_kernel(const LogprobsArgs a) {
  typedef LogitVec<T> Vec;
  constexpr int N = Vec::N;
  // group maxima and the list; in the join the parts' lists, and those of their keys that may be among the best: the
  // lists of top_n parts at most
  __shared__ __attribute__((aligned(16))) unsigned long long sm_raw[2 * kLpMaxParts * KX_LOGPROBS_TOP_MAX];
  unsigned long long* sm_best = sm_raw + kLpMaxParts * KX_LOGPROBS_TOP_MAX;
  static_assert(sizeof(sm_raw) >= kLpGroups * kLpThreads * 4 + kLpList * 8, "");
  float* sm_group = reinterpret_cast<float*>(sm_raw);
  unsigned long long* sm_list = sm_raw + kLpGroups * kLpThreads / 2;
  __shared__ unsigned long long sm_top[KX_LOGPROBS_TOP_MAX];
  __shared__ float sm_sums[kLpWaves][3];
  __shared__ unsigned sm_largest[kLpThreads];
  __shared__ unsigned short sm_hit[kLpList];  // groups to look through: group * threads + thread
  __shared__ int sm_count, sm_hits, sm_last;

  const int tid = threadIdx.x, lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
  const T* x = static_cast<const T*>(a.logits) + row * a.row_stride;
  // the row from its first 16-byte boundary on in vectors; the elements ahead and behind belong to the outer parts
  const int ahead = min(a.vocab, (int)((16 - (uintptr_t)x % 16) % 16 / sizeof(T)));
  const int vectors = (a.vocab - ahead) / N, behind0 = ahead + vectors * N;
  const int v0 = (int)((int64_t)vectors * part / a.parts), v1 = (int)((int64_t)vectors * (part + 1) / a.parts);
  const u32x4* xv = reinterpret_cast<const u32x4*>(x + ahead);
  int extra = -1;  // this thread's element ahead or behind
  if (part == 0 && tid < ahead) extra = tid;
  if (part == a.parts - 1 && tid >= 8 && behind0 + tid - 8 < a.vocab) extra = behind0 + tid - 8;
  const float xe = extra >= 0 ? (float)*KX_CK(a, PL_X, x + extra) : -INFINITY;

  if (tid == 0) sm_count = sm_hits = 0;
  LogSums sums = {wave_max(xe), 0.f, 0.f};
  float largest = fmaxf(xe, -INFINITY);  // (no NaN)
  if (extra >= 0) {
    const float d = xe - (sums.m == -INFINITY ? 0.f : sums.m), e = __builtin_amdgcn_exp2f(d * 1.4426950408889634f);
    sums.z = e;
    sums.s = fmaxf(d, -150.f) * e;
  }
  const int per_step = kLpThreads * kLpUnroll;
  const int steps = (v1 - v0 + per_step - 1) / per_step, group_steps = (steps + kLpGroups - 1) / kLpGroups;
  auto load_step = [&](int step, u32x4 (&v)[kLpUnroll]) {
    const int at = v0 + step * per_step + tid;
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u) {
      const int i = at + u * kLpThreads;
      v[u] = *KX_CK(a, PL_X, xv + min(i, v1 - 1));
    }
    if (step == steps - 1) {
#pragma unroll
      for (int u = 0; u < kLpUnroll; ++u)
        if (at + u * kLpThreads >= v1) v[u] = u32x4{Vec::kNone, Vec::kNone, Vec::kNone, Vec::kNone};
    }
  };
  int step = 0;
  for (int group = 0; step < steps; ++group) {
    float group_max = -INFINITY;
    const int end = min(step + group_steps, steps);
    for (; step < end; ++step) {
      u32x4 v[kLpUnroll];
      load_step(step, v);
      float mx = Vec::get(v[0], 0);
#pragma unroll
      for (int u = 0; u < kLpUnroll; ++u)
#pragma unroll
        for (int i = 0; i < N; ++i) mx = fmaxf(mx, Vec::get(v[u], i));
      mx = fmaxf(mx, -INFINITY);  // (a first element that is NaN)
      group_max = fmaxf(group_max, mx);
      if (__ballot(mx > sums.m)) rebase(sums, fmaxf(sums.m, wave_max(mx)));
      const float m = sums.m == -INFINITY ? 0.f : sums.m;
      float z0 = 0.f, z1 = 0.f, s0 = 0.f, s1 = 0.f;
#pragma unroll
      for (int u = 0; u < kLpUnroll; ++u)
#pragma unroll
        for (int i = 0; i < N; i += 2) {
          const float d0 = Vec::get(v[u], i) - m, d1 = Vec::get(v[u], i + 1) - m;
          const float e0 = __builtin_amdgcn_exp2f(d0 * 1.4426950408889634f), e1 = __builtin_amdgcn_exp2f(d1 * 1.4426950408889634f);
          z0 += e0;
          z1 += e1;
          s0 = fmaf(fmaxf(d0, -150.f), e0, s0);  // (-inf adds nothing: e is zero)
          s1 = fmaf(fmaxf(d1, -150.f), e1, s1);
        }
      sums.z += z0 + z1;
      sums.s += s0 + s1;
    }
    sm_group[group * kLpThreads + tid] = group_max;
    largest = fmaxf(largest, group_max);
  }
  sums.z = wave_sum(sums.z);
  sums.s = wave_sum(sums.s);
  if (lane == 0) {
    sm_sums[wave][0] = sums.m;
    sm_sums[wave][1] = sums.z;
    sm_sums[wave][2] = sums.s;
  }
  if (a.top_n > 0) sm_largest[tid] = order_of(largest);
  __syncthreads();
  LogSums all = {-INFINITY, 0.f, 0.f};
#pragma unroll
  for (int w = 0; w < kLpWaves; ++w) all.m = fmaxf(all.m, sm_sums[w][0]);
#pragma unroll
  for (int w = 0; w < kLpWaves; ++w) {
    LogSums one = {sm_sums[w][0], sm_sums[w][1], sm_sums[w][2]};
    rebase(one, all.m);
    all.z += one.z;
    all.s += one.s;
  }

  if (a.top_n > 0) {
    unsigned of_lanes = sm_largest[lane];
#pragma unroll
    for (int w = 1; w < kLpWaves; ++w) of_lanes = max(of_lanes, sm_largest[w * 64 + lane]);
    // (a bound below every value is a NaN here, which no value is below)
    const float least = value_of_order(nth_largest(of_lanes, a.top_n));
    // not below it (a NaN may be among the best of a row with fewer than top_n others)
    if (extra >= 0 && !(xe < least)) {
      const int at = atomicAdd(&sm_count, 1);
      if (at < kLpList) sm_list[at] = key_of(xe, extra);
    }
    // the groups that reach it, and then all of their elements, dealt over the threads
    for (int group = 0; group * group_steps < steps; ++group)
      if (!(sm_group[group * kLpThreads + tid] < least)) {
        const int at = atomicAdd(&sm_hits, 1);
        if (at < kLpList) sm_hit[at] = (unsigned short)(group * kLpThreads + tid);
      }
    __syncthreads();
    if (sm_hits <= kLpList) {
      constexpr int PER = kLpUnroll * N;  // elements of a step
      constexpr int AT_ONCE = 2;
      const int elements = sm_hits * PER;
      for (int i0 = tid; i0 < elements; i0 += AT_ONCE * kLpThreads) {
        for (int st = 0; st < group_steps; ++st) {
          int index[AT_ONCE];
          float value[AT_ONCE];
#pragma unroll
          for (int k = 0; k < AT_ONCE; ++k) {
            const int i = min(i0 + k * kLpThreads, elements - 1), hit = sm_hit[i / PER], e = i % PER;
            const int step_of = hit / kLpThreads * group_steps + st, vec = v0 + step_of * per_step + e / N * kLpThreads + hit % kLpThreads;
            const bool mine = i0 + k * kLpThreads < elements && vec < v1;
            index[k] = mine ? ahead + vec * N + e % N : -1;
            value[k] = (float)*KX_CK(a, PL_X, x + max(index[k], 0));
          }
#pragma unroll
          for (int k = 0; k < AT_ONCE; ++k)
            if (index[k] >= 0 && !(value[k] < least)) {
              const int at = atomicAdd(&sm_count, 1);
              if (at < kLpList) sm_list[at] = key_of(value[k], index[k]);
            }
        }
      }
    } else if (tid == 0) {
      sm_count = kLpList + 1;  // each of them holds an element of the list at least
    }
    __syncthreads();
    int count = sm_count;
    if (tid < KX_LOGPROBS_TOP_MAX) sm_top[tid] = 0;
    __syncthreads();
    if (count > kLpList) {
      // Too many alike: in order of index, 256 at a time, the best so far kept at the head of the list.  A step without a
      // value above the least of them (an equal one further on ranks below it) is passed over.
      unsigned long long least_key = 0;
      if (tid == 0) sm_count = 0;
      __syncthreads();
      auto look_through = [&](int from, int upto) {
        for (int base = from; base < upto; base += kLpThreads) {
          const int i = base + tid;
          const unsigned long long key = i < upto ? key_of((float)*KX_CK(a, PL_X, x + i), i) : 0;
          if (key > least_key) sm_list[atomicAdd(&sm_count, 1)] = key;  // at most kLpList: see below
          __syncthreads();
          count = sm_count;
          __syncthreads();
          if (count > kLpList - kLpThreads) {
            rank_keys(sm_list, count, a.top_n, sm_top);
            __syncthreads();
            if (tid < a.top_n) sm_list[tid] = sm_top[tid];
            least_key = sm_top[a.top_n - 1];
            if (tid == 0) sm_count = a.top_n;
            __syncthreads();
          }
        }
      };
      // (the pieces one after the other: ahead of the vectors, a step of them each, behind them)
      for (int st = -1; st <= steps; ++st) {
        int from = part == 0 ? 0 : ahead, upto = ahead;
        if (st == steps) {
          from = behind0;
          upto = part == a.parts - 1 ? a.vocab : behind0;
        } else if (st >= 0) {
          u32x4 v[kLpUnroll];
          load_step(st, v);
          float mx = -INFINITY;
#pragma unroll
          for (int u = 0; u < kLpUnroll; ++u)
#pragma unroll
            for (int e = 0; e < N; ++e) mx = fmaxf(mx, Vec::get(v[u], e));
          // (the value of no key is a NaN)
          if (!__syncthreads_or(!(mx <= value_of_key(least_key)))) continue;
          from = ahead + (v0 + st * per_step) * N;
          upto = ahead + min(v0 + (st + 1) * per_step, v1) * N;
        }
        look_through(from, upto);
      }
      count = sm_count;
    }
    rank_keys(sm_list, count, a.top_n, sm_top);
    __syncthreads();
  }

  unsigned long long best = tid < a.top_n ? sm_top[tid] : 0;  // threads 0 .. top_n - 1 of the first wave
  if (a.parts > 1) {
    char* mine = a.records + (int64_t)(row * a.parts) * kLpRecord;
    const __amdgpu_buffer_rsrc_t rec = __builtin_amdgcn_make_buffer_rsrc(mine, 0, 0x7fffffff, 0x00020000);
    // device-scope stores, acknowledged ahead of the ticket; device-scope loads behind it (no cache write-back)
    KX_TOUCH(a, PL_WS, mine + part * kLpRecord, kLpRecord);
    if (tid == 0) {
      const u32x4 s = {__float_as_uint(all.m), __float_as_uint(all.z), __float_as_uint(all.s), 0u};
      __builtin_amdgcn_raw_buffer_store_b128(s, rec, part * kLpRecord, 0, 16);
    }
    if (tid < a.top_n)
      __builtin_amdgcn_raw_buffer_store_b64(u32x2{(unsigned)best, (unsigned)(best >> 32)}, rec, part * kLpRecord + 16 + 8 * tid, 0, 16);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0) {
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
      sm_last = atomicInc(KX_CK(a, PL_WS, a.tickets + row * (kTicketStride / 4)), (unsigned)a.parts - 1u) == (unsigned)a.parts - 1u;  // wraps to 0
    }
    __syncthreads();
    if (!sm_last) return;
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    // the parts' lists, all requested before the first is used
    constexpr int ROUNDS = kLpMaxParts * KX_LOGPROBS_TOP_MAX / kLpThreads;
    const int keys = a.parts * a.top_n;
    u32x2 k[ROUNDS];
#pragma unroll
    for (int j = 0; j < ROUNDS; ++j) {
      const int i = max(min(tid + j * kLpThreads, keys - 1), 0), p = a.top_n ? i / a.top_n : 0;
      k[j] = __builtin_amdgcn_raw_buffer_load_b64(rec, p * kLpRecord + 16 + 8 * (i - p * a.top_n), 0, 16);
    }
    const u32x4 s = __builtin_amdgcn_raw_buffer_load_b128(rec, min(lane, a.parts - 1) * kLpRecord, 0, 16);
    LogSums one = {__uint_as_float(s.x), __uint_as_float(s.y), __uint_as_float(s.z)};
    if (lane >= a.parts) one = LogSums{-INFINITY, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < ROUNDS; ++j)
      if (tid + j * kLpThreads < keys) sm_raw[tid + j * kLpThreads] = (unsigned long long)k[j].y << 32 | k[j].x;
    const float m = wave_max(one.m);
    rebase(one, m);
    all = LogSums{m, wave_sum(one.z), wave_sum(one.s)};
    if (tid == 0) sm_count = 0;
    __syncthreads();
    if (a.top_n > 0) {
      // The parts' lists fall.  With `depth` keys of each list at least top_n: no key below all of those is among the best;
      // with a head of top_n lists or more, none below the top_n-th largest of the heads.
      const int depth = (a.top_n + a.parts - 1) / a.parts;
      const unsigned head = lane < a.parts ? (unsigned)(sm_raw[lane * a.top_n + depth - 1] >> 32) : 0u;
      const unsigned long long bound = (unsigned long long)nth_largest(head, depth == 1 ? a.top_n : a.parts) << 32;
#pragma unroll
      for (int j = 0; j < ROUNDS; ++j) {
        const unsigned long long key = (unsigned long long)k[j].y << 32 | k[j].x;
        if (tid + j * kLpThreads < keys && key >= bound) sm_best[atomicAdd(&sm_count, 1)] = key;
      }
      __syncthreads();
      rank_keys(sm_best, sm_count, a.top_n, sm_top);
      __syncthreads();
      best = tid < a.top_n ? sm_top[tid] : 0;
    }
  }
  if (wave != 0) return;
  const bool odd = !(all.z > 0.f && all.z < INFINITY);
  const float lz = odd ? NAN : logf(all.z);
  if (lane == 0) {
    if (a.logprob) {
      const int t = *KX_CK(a, PL_TOKENS, a.tokens + row);
      *KX_CK(a, PL_LOGPROB, a.logprob + row) =
          t < 0 ? 0.f : t >= a.vocab ? NAN : ((float)*KX_CK(a, PL_X, x + t) - all.m) - lz;
    }
    if (a.entropy) *KX_CK(a, PL_ENTROPY, a.entropy + row) = lz - all.s / all.z;
  }
  if (lane < a.top_n) {
    *KX_CK(a, PL_IDS, a.top_ids + ((int64_t)row * a.top_n + lane)) = index_of_key(best);
    *KX_CK(a, PL_TOP, a.top_logprobs + ((int64_t)row * a.top_n + lane)) = (value_of_key(best) - all.m) - lz;
  }
}

// Parts of a row: enough to fill the chip, each of two vectors per thread at least.
static int logprobs_parts(int rows, int vocab, int kind) {
  const int64_t least = (int64_t)kLpThreads * 2 * 16 / (int64_t)kind_bytes(kind);
  int64_t parts = kLpSlots / rows;
  if (parts > vocab / least) parts = vocab / least;
  return parts < 1 ? 1 : parts > kLpMaxParts ? kLpMaxParts : (int)parts;
}

}  // namespace kx

extern "C" size_t kx_token_logprobs_workspace_bytes(int32_t rows, int32_t vocab, int32_t top_n) {
  using namespace kx;
  if (rows <= 0 || vocab <= 0 || top_n < 0) return 0;
  return kTicketBytes + (size_t)kLpSlots * kLpRecord;
}

extern "C" int kx_token_logprobs(const kx_logprobs_desc* d, void* stream) {
  using namespace kx;
  if (!d || d->rows < 0) return KX_EINVAL;
  if (d->rows == 0) return KX_OK;
  if (!kind_known(d->type) || !d->logits || (uintptr_t)d->logits % kind_bytes(d->type) || d->vocab <= 0 || d->row_stride < d->vocab)
    return KX_EINVAL;
  if ((d->tokens != nullptr) != (d->logprob != nullptr)) return KX_EINVAL;
  if (d->top_n < 0 || d->top_n > KX_LOGPROBS_TOP_MAX || d->top_n > d->vocab) return KX_EINVAL;
  if (d->top_n > 0 && (!d->top_ids || !d->top_logprobs)) return KX_EINVAL;
  if (!aligned4(d->tokens) || !aligned4(d->logprob) || !aligned4(d->entropy) || !aligned4(d->top_ids) || !aligned4(d->top_logprobs))
    return KX_EINVAL;
  if (!d->workspace || d->workspace_bytes < kx_token_logprobs_workspace_bytes(d->rows, d->vocab, d->top_n)) return KX_EWORKSPACE;
  if ((uintptr_t)d->workspace % 256) return KX_EINVAL;
  if (!grid_fits(d->rows, kLpThreads) || d->vocab > kMostPositions) return KX_ELIMIT;
  LogprobsArgs a{};
  a.logits = d->logits;
  a.tokens = d->tokens;
  a.logprob = d->logprob;
  a.entropy = d->entropy;
  a.top_ids = d->top_ids;
  a.top_logprobs = d->top_logprobs;
  a.tickets = static_cast<unsigned*>(d->workspace);
  a.records = static_cast<char*>(d->workspace) + kTicketBytes;
  a.row_stride = d->row_stride;
  a.rows = d->rows;
  a.vocab = d->vocab;
  a.top_n = d->top_n;
  a.parts = logprobs_parts(d->rows, d->vocab, d->type);
  const void* operands[] = {a.logits, a.tokens, a.logprob, a.entropy, a.top_ids, a.top_logprobs, d->workspace};
  for (int i = 0; i < 7; ++i) KX_BSET(a, i, operands[i]);
  (void)operands;
  const dim3 grid((unsigned)a.rows * (unsigned)a.parts), block(kLpThreads);
  hipStream_t s = (hipStream_t)stream;
  if (d->type == KX_F16) hipLaunchKernelGGL(logprobs_kernel<_Float16>, grid, block, 0, s, a);
  else if (d->type == KX_BF16) hipLaunchKernelGGL(logprobs_kernel<__bf16>, grid, block, 0, s, a);
  else hipLaunchKernelGGL(logprobs_kernel<float>, grid, block, 0, s, a);
  KX_LAUNCH_CHECK();
  return KX_OK;
}
