// Attention of packed prompts of different lengths, keys and values packed beside them or in pages.
//
//   row i of n at position p = (keys - n) + i:  s_t = scale q_i . k_t,  out_i = sum_t e^{s_t - m} v_t / sum_t e^{s_t - m}
//   over the t that it sees: t < keys, t <= p when causal, t > p - window with a window.
//
// Bound: 4 hs operations per (head, row, seen key) on the matrix cores; K and V come from L2.
//
// Split: the rows of a sequence times the kv_mul query heads of a kv head are one list of (row, head) pairs; a
// workgroup takes 32 consecutive pairs per wave, so any grouping of heads fills the tiles and a staged K/V tile
// feeds all heads that share it.  A workgroup finds its sequence by a prefix sum over the lengths: no plan from the host.
//
// Tile: 64 keys in LDS, two buffers, filled by LDS-DMA (a wave instruction moves 1 KiB, every lane from an address of
// its own, so rows may come from pages), one barrier per tile.  A row's 16-byte pieces sit exclusive-or-ed with a
// row key, applied to the source address and to the reads, which makes both products' reads conflict-free.
//
// Products: S^T = K Q^T leaves the keys on the register axis and the pair on the lane, so the softmax state is one
// value per lane and the weights are already the B operand of O^T = V^T P^T; the A operand V^T comes out of row-major V by
// transposing LDS reads (16-bit types), or one element per lane (fp32).
//
// Reached: 1.0 PFLOP/s on a prompt of 4096 (32 heads over 8, 128 wide, bf16: 134 us), where a library product of 8192 x 8192 x
// 8192 reaches 1.09.  The clock falls to 2.0 GHz there (2.3 and more in the other kernels of batched serving), and matrix
// instructions take 51 % and vector ones 47 % of the cycles that a CU is busy (64-wide prompts: 30 and 68 %; pieces over pages:
// 34 and 41 %).  Tried and no faster: the two waves of a SIMD half a step apart (150 us), the next scores and the last
// second product between a wave's vector instructions (143, with spills), waiting later for the LDS-DMA (the same), two
// workgroups of four waves and 32-key tiles per CU (154).
// A workgroup takes 7 us beside its tiles (lengths, pages and first tiles 4, joining and storing 2).
//
// Rounding: products of 16-bit operands are exact in fp32 and summed there, softmax in fp32, weights rounded to the
// type for the second product and summed as they were rounded, so a result is a mean of the values and lies among
// them.  (With the sum of the unrounded weights, values of 65504 came out as infinity.  Dot products with ones sum them; measured in
// turn against that, us: a prompt of 4096 143 / 145, packed prompts 52.7 / 52.0, pieces 94.3 / 93.8.)  The running maximum follows only when it is
// exceeded by more than 2^8: weights up to 256 have the same relative precision, and the rescaling pass is rare.
//
// Values that are not finite: hidden from a pair, they meet its weight of zero all the same.  A workgroup with a result that is
// not finite goes through its keys once more; then a tile that a wave sees in part and that holds such a value is taken key by key when
// the others are done (50 - 70 us, all waves side by side): one NaN in a prompt of 4096 0.35 ms, 512 rows over a window
// with pages of NaN standing in for those left behind 59 us for 34.  (Pairs with such results computed anew one by one: 27 ms and
// 8.3 ms.  The edge tiles looked through in every call: 4 % of short prompts' time, 1 % this way.)
#include <math.h>

#include <type_traits>

#define KX_FILE_ID 12
#include "paged.hpp"

namespace kx {

enum PromptOperand { PP_Q, PP_K, PP_V, PP_OUT, PP_CUQ, PP_CUK, PP_TABLE, PP_LENS };

// keys per tile: as many as let two buffers of a tile per group of waves fit LDS
template <typename T> __host__ __device__ constexpr int pa_keys() { return sizeof(T) == 4 ? 32 : 64; }

enum { PA_PACKED = 0, PA_BLOCK_PAGES = 1, PA_ANY_PAGES = 2 };  // where rows are: see row sources below

struct PromptArgs {
  PagedView kv;
  const char* q;
  const char* k;  // packed rows, or the pages
  const char* v;
  char* out;
  const int32_t* cu_q;
  const int32_t* cu_k;
  int64_t q_stride, k_stride, v_stride, out_stride;
  int32_t batch, kv_heads, kv_mul, q_rows, k_rows, causal, window;
  PageDiv mul_div;  // division by kv_mul
  float scale;
  KX_BFIELD(8)
};

// A workgroup's part of the batch.
struct PromptWork {
  int b, q0, n;      // sequence, its first row in q, its rows
  int k0, keys;      // first key row (packed), keys
  int p0;            // position of the first row, below zero with fewer keys than rows
  int block;         // 32 * waves pairs from here
};

__device__ __forceinline__ int clamp_row(int x, int rows) { return min(max(x, 0), rows); }

template <int ROWS, bool PAGED>
__device__ __forceinline__ bool find_prompt(const PromptArgs& a, int item, PromptWork& w) {
  const int lane = lane_id();
  int done = 0;
  for (int base = 0; base < a.batch; base += 64) {
    const int b = base + lane;
    int q0 = 0, n = 0, k0 = 0, keys = 0, length = 0;
    if (b < a.batch) {
      q0 = clamp_row(*KX_CK(a, PP_CUQ, a.cu_q + b), a.q_rows);
      n = max(clamp_row(*KX_CK(a, PP_CUQ, a.cu_q + b + 1), a.q_rows) - q0, 0);
      if (PAGED) {
        length = max(*KX_CK(a, PP_LENS, a.kv.seq_lens + b), 0);
        keys = min(length, a.kv.capacity());
      } else {
        k0 = clamp_row(*KX_CK(a, PP_CUK, a.cu_k + b), a.k_rows);
        length = keys = max(clamp_row(*KX_CK(a, PP_CUK, a.cu_k + b + 1), a.k_rows) - k0, 0);
      }
    }
    // The sequences (64 at a time) in falling order of their keys, each one's last blocks first: long chains of tiles
    // start early.  (Six pieces of 118 .. 1024 rows over 425 .. 4298 keys: 178 us in index order, 146 so, in the form that this was
    // tried with, now 91.)
    const int mine = (int)(((int64_t)n * a.kv_mul + ROWS - 1) / ROWS);
    int blocks = mine, from = lane;
    if (a.batch > 1) {
      int place = 0;
      for (int j = 0; j < min(a.batch - base, 64); ++j) {
        const int other = __builtin_amdgcn_readlane(keys, j);
        place += other > keys || (other == keys && j < lane);
      }
      if (b >= a.batch) place = lane;
      from = __builtin_amdgcn_ds_permute(place << 2, lane);
      blocks = __builtin_amdgcn_ds_permute(place << 2, mine);
    }
    const int upto = wave_scan(blocks);
    const unsigned long long past = __ballot(done + upto > item);
    if (past) {
      const int at = __builtin_ctzll(past), l = __builtin_amdgcn_readlane(from, at);
      w.b = base + l;
      w.q0 = __builtin_amdgcn_readlane(q0, l);
      w.n = __builtin_amdgcn_readlane(n, l);
      w.k0 = __builtin_amdgcn_readlane(k0, l);
      w.keys = __builtin_amdgcn_readlane(keys, l);
      w.p0 = __builtin_amdgcn_readlane(length, l) - w.n;
      w.block = done + __builtin_amdgcn_readlane(upto, at) - 1 - item;
      return true;
    }
    done += __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}

// The 16-byte piece of a K (V) row that sits at position c of its place in LDS is c ^ key.  K rows are read 16 at a
// time at one piece: the 16 positions cover the banks once.  V rows: 4 (16-bit) rows x 64 bytes at a time,
// or two rows four apart x 128 bytes (fp32).
template <int CH>
__device__ __forceinline__ int k_swizzle(int row) { return CH >= 16 ? row % 16 : CH == 8 ? row / 2 % 8 : row / 4 % 4; }
template <int CH, bool F32>
__device__ __forceinline__ int v_swizzle(int row) {
  if (F32) return CH >= 16 ? (row >> 2 & 1) << 3 : 0;
  return CH == 16 ? (row & 3) << 2 : CH == 8 ? (row >> 1 & 1) << 2 : 0;
}

// A transposing LDS read: of the 4 rows x 16 elements that 16 lanes point at (8 bytes each, row i / 4 for lane i), lane i
// gets column i.  The restrict pointer tells the compiler that the read does not meet the LDS-DMA in flight (it fills
// the other buffer); without it every such read waits for all of that first.
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s16x4* lds_tr_ptr;
__device__ __forceinline__ s16x4 read_transposed(lds_tr_ptr __restrict__ p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16(p);
}

template <typename T> struct PromptMma;
template <> struct PromptMma<_Float16> {
  typedef f16x8 frag;
  static __device__ __forceinline__ f32x16 mul(frag a, frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float add_pair(_Float16 x, _Float16 y, float c) {
    typedef _Float16 pair __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2(pair{x, y}, pair{(_Float16)1.f, (_Float16)1.f}, c, false);
  }
};
template <> struct PromptMma<__bf16> {
  typedef bf16x8 frag;
  static __device__ __forceinline__ f32x16 mul(frag a, frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float add_pair(__bf16 x, __bf16 y, float c) {
    typedef __bf16 pair __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16(pair{x, y}, pair{(__bf16)1.f, (__bf16)1.f}, c, false);
  }
};
template <> struct PromptMma<float> { typedef f32x4 frag; };

// c and the products of the elements of two dwords
template <typename T>
__device__ __forceinline__ float dot_dword(unsigned x, unsigned y, float c) {
  if constexpr (sizeof(T) == 4) {
    return fmaf(__uint_as_float(x), __uint_as_float(y), c);
  } else if constexpr (std::is_same<T, _Float16>::value) {
    typedef _Float16 pair __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(pair, x), __builtin_bit_cast(pair, y), c, false);
  } else {
    typedef __bf16 pair __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(pair, x), __builtin_bit_cast(pair, y), c, false);
  }
}
typedef const __attribute__((address_space(3))) u32x4* lds_vec_ptr;
__device__ __forceinline__ u32x4 read_tile(lds_vec_ptr __restrict__ p) { return *p; }  // (restrict: as above)

// NW: waves of the workgroup.  KG: groups of waves that share the pairs and take every KG-th tile of the keys, joined in LDS at the end: shorter
// chains of tiles and more workgroups where there are few pairs.  (Narrower heads of 16-bit types keep to 128 registers: two workgroups
// share a CU.)
// CAREFUL: the second time, for values that are not finite (see above).  A wave whose results all are has stored them the first time;
// the others (`odd`) do so now, from queries that are still whole where the results lie over them.  Returns whether a second time
// is called for, to all waves alike.
template <typename T, int HS, int MODE, int KG, int NW, bool CAREFUL>
__device__ __forceinline__ bool prompt_attn(const PromptArgs& a, bool& odd) {
  constexpr int PW = NW / KG;                    // waves of a group
  constexpr int PAIRS = PW * 32;                 // pairs of the workgroup
  constexpr int KT = pa_keys<T>();
  constexpr bool F32 = sizeof(T) == 4, PAGED = MODE != PA_PACKED;
  constexpr int ROWB = HS * (int)sizeof(T);      // bytes of a row
  constexpr int CH = ROWB / 16;                  // its pieces
  constexpr int RPP = 1024 / ROWB;               // rows per DMA instruction
  constexpr int TILEB = KT * ROWB;               // K (or V) bytes of a tile
  constexpr int KP = TILEB / 1024;               // DMA instructions for them
  constexpr int RP = (KP * KG + NW - 1) / NW;    // of K (and of V) per wave and buffer
  constexpr int DT = HS / 32;                    // output tiles
  // fp16 weights are held 2^7 times as large: at most 2^15, and whole down to 2^-21 of the largest
  constexpr float kShift = std::is_same<T, _Float16>::value ? 7.f : 0.f;
  constexpr int KS = HS * (int)sizeof(T) / 32;   // 32-byte steps of the first product
  static_assert(KP * KG % NW == 0 || KP * KG < NW, "");
  __shared__ int sm_missing[PAGED ? NW : 1], sm_odd[CAREFUL ? 1 : NW];
  extern __shared__ __attribute__((aligned(1024))) char smem[];  // two buffers of KG tiles, K and V each
  typedef __attribute__((address_space(3))) void* lds_ptr;
  typedef const __attribute__((address_space(3))) char* lds_bytes;

  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int qcol = lane & 31, half = lane >> 5;
  const int kvh = blockIdx.x % a.kv_heads;
  PromptWork w;
  if (!find_prompt<PAIRS, PAGED>(a, blockIdx.x / a.kv_heads, w)) return false;
  const int group = KG == 1 ? 0 : wave / PW;

  // ---- this workgroup's and this wave's pairs, and what they see ----
  const int pairs = w.n * a.kv_mul, f0 = w.block * PAIRS;
  auto hi_of = [&](int row) { return a.causal ? max(min(w.p0 + row + 1, w.keys), 0) : w.keys; };
  auto lo_of = [&](int row) { return a.window > 0 ? max(max(w.p0 + row, 0) - a.window + 1, 0) : 0; };
  auto row_of = [&](int f) { return a.mul_div.page(min(f, pairs - 1)); };
  const int hi = hi_of(row_of(f0 + PAIRS - 1)), lo = min(lo_of(row_of(f0)), hi);
  const int t0 = lo / KT, t1 = hi > lo ? (hi + KT - 1) / KT : t0;
  const int wf0 = f0 + wave % PW * 32;
  const int first_row = row_of(wf0), last_row = row_of(wf0 + 31);
  const int w_hi = wf0 < pairs ? hi_of(last_row) : 0, w_lo = lo_of(first_row);
  const int full_hi = hi_of(first_row), full_lo = lo_of(last_row);  // every pair of the wave sees these keys
  const int my_f = min(wf0 + qcol, pairs - 1), my_row = row_of(my_f), my_head = my_f - my_row * a.kv_mul;
  const int my_hi = hi_of(my_row), my_lo = lo_of(my_row);

  // ---- row sources ----
  const int64_t k_stride = PAGED ? a.kv.row_stride : a.k_stride, v_stride = PAGED ? a.kv.row_stride : a.v_stride;
  const T* kbase = reinterpret_cast<const T*>(a.k) + (PAGED ? kvh * a.kv.head_stride : w.k0 * a.k_stride + kvh * HS);
  const T* vbase = reinterpret_cast<const T*>(a.v) + (PAGED ? kvh * a.kv.head_stride : w.k0 * a.v_stride + kvh * HS);
  const int32_t* table = PAGED ? a.kv.table + w.b * a.kv.table_stride : nullptr;
  auto page_ok = [&](int p) { return (unsigned)p < (unsigned)a.kv.num_pages; };
  auto lookup = [&](int t) { return *KX_CK(a, PP_TABLE, table + a.kv.div.page(t)); };
  const unsigned page_bytes = PAGED ? (unsigned)(a.kv.page_stride * sizeof(T)) : 0u, row_bytes = PAGED ? (unsigned)(a.kv.row_stride * sizeof(T)) : 0u;
  // byte offset of position t, whose page is `page` (one that is not there: some page that is)
  auto paged_offset = [&](int page, int t) {
    return (uint64_t)(page_ok(page) ? (unsigned)page : 0u) * page_bytes +
           (uint64_t)(unsigned)(t - a.kv.div.page(t) * a.kv.div.size) * row_bytes;
  };
  // The KG tiles of a buffer are consecutive, so its K rows are KG * KT consecutive keys.  DMA pair j of a wave, one
  // instruction for K and one for V: the first of its rows among the keys, and a lane's.
  auto pair_first = [&](int j) { return (wave + NW * j) * RPP; };
  auto pair_row = [&](int j) { return pair_first(j) + lane / CH; };
  // Pages of the next buffer's rows, requested a step ahead: one per instruction where pages are whole 16-row blocks, else
  // one per lane.  (By vector loads in both cases: the end of a step waits for those anyway, while a scalar load would
  // have the next fragment reads wait for it.)
  int ids[PAGED ? RP : 1];
  auto get_ids = [&](int t) {
    if constexpr (PAGED) {
      int zero;
      asm volatile("v_mov_b32 %0, 0" : "=v"(zero));
#pragma unroll
      for (int j = 0; j < RP; ++j) {
        if constexpr (MODE == PA_BLOCK_PAGES)
          ids[j] = lookup(min(t * KT + pair_first(j), (w.keys - 1) & ~(RPP - 1)) + zero);
        else
          ids[j] = lookup(min(t * KT + pair_row(j), w.keys - 1));
      }
    }
  };
  if (t0 < t1) get_ids(t0);
  // ---- queries: lane (pair, half) holds the pieces of its row that meet its pieces of a K row ----
  typedef typename PromptMma<T>::frag frag;
  frag qf[KS];
  const T* qrow = reinterpret_cast<const T*>(a.q) + (w.q0 + my_row) * a.q_stride + (kvh * a.kv_mul + my_head) * HS;
#pragma unroll
  for (int ks = 0; ks < KS; ++ks)
    qf[ks] = *KX_CK(a, PP_Q, reinterpret_cast<const frag*>(reinterpret_cast<const char*>(qrow) + 32 * ks + 16 * half));
  // A page that is not there is looked for once, beside the first tiles' way here, and tile by tile only if there is one.
  const int last_col = PAGED && t0 < t1 ? a.kv.div.page(hi - 1) : 0, col = PAGED ? a.kv.div.page(lo) + (int)threadIdx.x : 0;
  int probe = 0;
  if (PAGED && t0 < t1) probe = *KX_CK(a, PP_TABLE, table + min(col, last_col));

  const bool has_pair = KP * KG >= NW || wave < KP * KG;
  // a lane's byte offsets from the first row of the buffer (packed), from the first row of the instruction's 16-row block, or
  // within its row (pages); `tail`: those in the last buffer, where rows behind the last key are replaced by it
  unsigned k_off[RP], v_off[RP], k_tail[RP], v_tail[RP];
  const int steps = (t1 - t0 + KG - 1) / KG, tail_key0 = (t0 + (steps - 1) * KG) * KT;
#pragma unroll
  for (int j = 0; j < RP; ++j) {
    const int row = pair_row(j), from = MODE == PA_PACKED ? row : MODE == PA_BLOCK_PAGES ? lane / CH : 0;
    const int block = min(tail_key0 + pair_first(j), (w.keys - 1) & ~(RPP - 1)) + lane / CH;
    const int behind = MODE == PA_PACKED ? max(tail_key0 + row - (w.keys - 1), 0) : MODE == PA_BLOCK_PAGES ? max(block - (w.keys - 1), 0) : 0;
    const unsigned kp = 16u * (lane % CH ^ k_swizzle<CH>(row)), vp = 16u * (lane % CH ^ v_swizzle<CH, F32>(row));
    const unsigned kb = (unsigned)((int)k_stride * (int)sizeof(T)), vb = (unsigned)((int)v_stride * (int)sizeof(T));
    k_off[j] = kp + from * kb;
    v_off[j] = vp + from * vb;
    k_tail[j] = kp + (unsigned)(from - behind) * kb;
    v_tail[j] = vp + (unsigned)(from - behind) * vb;
  }
  auto issue = [&](int t, int buf, int from, int upto) {
    if (!has_pair) return;
    const int key0 = t * KT;
    const bool whole = key0 + KG * KT <= w.keys;
#pragma unroll
    for (int j = 0; j < RP; ++j) {
      if (j < from || j >= upto) continue;
      const char* ks = reinterpret_cast<const char*>(kbase);
      const char* vs = reinterpret_cast<const char*>(vbase);
      if constexpr (MODE == PA_ANY_PAGES) {
        const uint64_t at = paged_offset(ids[j], min(key0 + pair_row(j), w.keys - 1));
        ks += at;
        vs += at;
      } else if constexpr (MODE == PA_BLOCK_PAGES) {
        const uint64_t at = paged_offset(__builtin_amdgcn_readfirstlane(ids[j]), min(key0 + pair_first(j), (w.keys - 1) & ~(RPP - 1)));
        ks += at;
        vs += at;
      } else {
        ks += (int64_t)key0 * k_stride * (int)sizeof(T);
        vs += (int64_t)key0 * v_stride * (int)sizeof(T);
      }
      ks += whole ? k_off[j] : k_tail[j];
      vs += whole ? v_off[j] : v_tail[j];
      const int q = wave + NW * j;
      char* to = smem + buf * KG * 2 * TILEB + q / KP * 2 * TILEB + q % KP * 1024;
      __builtin_amdgcn_global_load_lds(KX_CKN(a, PP_K, ks, 16), (lds_ptr)to, 16, 0, 0);
      __builtin_amdgcn_global_load_lds(KX_CKN(a, PP_V, vs, 16), (lds_ptr)(to + TILEB), 16, 0, 0);
    }
  };

  if (t0 < t1) {
    issue(t0, 0, 0, RP);
    if (t0 + KG < t1) get_ids(t0 + KG);
  }
  // scores in powers of two; a negative scale turns the queries' sign, and a scale of zero still hides (-inf * 0 is NaN)
  if (a.scale < 0.f) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = -qf[ks];
  }
  const float c = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 1.2e-38f);

  // ---- fragment addresses in a buffer ----
  unsigned kfrag[KS], vfrag[DT];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) kfrag[ks] = qcol * ROWB + (((2 * ks + half) ^ k_swizzle<CH>(qcol)) << 4);
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
    if constexpr (F32) {  // element 32 dt + qcol of rows 4 half + ...
      const int row = 4 * half, d = 32 * dt + qcol;
      vfrag[dt] = TILEB + row * ROWB + ((d / 4 ^ v_swizzle<CH, true>(row)) << 4) + d % 4 * 4;
    } else {  // 8 bytes: elements 4 (i % 4) .. of row 4 half + i / 4, i = lane % 16
      const int row = 4 * half + (lane & 15) / 4, d = 32 * dt + (lane & 16) + (lane & 3) * 4;
      vfrag[dt] = TILEB + row * ROWB + ((d / 8 ^ v_swizzle<CH, false>(row)) << 4) + d % 8 * 2;
    }
  }

  f32x16 o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[dt][r] = 0.f;
  float m = -INFINITY, l = 0.f;  // m in units of the raw product
  int odd_first = 0, odd_last = -1;  // first key of the first and of the last tile that is left for the end

  bool missing = false;
  if (PAGED && t0 < t1) {
    missing = !page_ok(probe);
    for (int at = col + NW * 64; at <= last_col; at += NW * 64) missing |= !page_ok(*KX_CK(a, PP_TABLE, table + at));
    const bool any = __ballot(missing) != 0;
    if (lane == 0) sm_missing[wave] = any;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (PAGED && t0 < t1) {
    missing = false;
#pragma unroll
    for (int v = 0; v < NW; ++v) missing |= sm_missing[v] != 0;
    missing = __builtin_amdgcn_readfirstlane(missing);
  }
  for (int t = t0, buf = 0; t < t1; t += KG, buf ^= 1) {
    // The next tiles are requested in two parts beside the scores: the LDS-DMA of a CU takes 64 bytes a cycle, and a wave
    // that sends all of its share at once waits for that.
    const bool more = t + KG < t1;
    const int key0 = (t + group) * KT;  // this wave's tile
    if (key0 < w_hi && key0 + KT > w_lo) {
      const lds_bytes base = (lds_bytes)smem + (buf * KG + group) * 2 * TILEB;
      // ---- scores: register r of s[kt] is key 32 kt + 8 (r / 4) + 4 half + r % 4 ----
      f32x16 s[KT / 32];
      frag kf[KT / 32][KS];
#pragma unroll
      for (int kt = 0; kt < KT / 32; ++kt) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[kt][r] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          kf[kt][ks] = *(const __attribute__((address_space(3))) frag*)(base + kfrag[ks] + kt * 32 * ROWB);
      }
#pragma unroll
      for (int kt = 0; kt < KT / 32; ++kt) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          if constexpr (F32) {
#pragma unroll
            for (int e = 0; e < 4; ++e) s[kt] = __builtin_amdgcn_mfma_f32_32x32x2f32(kf[kt][ks][e], qf[ks][e], s[kt], 0, 0, 0);
          } else {
            s[kt] = PromptMma<T>::mul(kf[kt][ks], qf[ks], s[kt]);
          }
        }
        if constexpr (!F32) {
          if (kt == 0) {
            // half of the fragments ahead of the first product, then one read behind each product
            __builtin_amdgcn_sched_group_barrier(0x100, KS, 0);
#pragma unroll
            for (int i = 0; i < KS; ++i) {
              __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
              __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        constexpr int HALVES = KT / 32;
        if (more) issue(t + KG, buf ^ 1, kt * RP / HALVES, (kt + 1) * RP / HALVES);
      }
      if (t + 2 * KG < t1) get_ids(t + 2 * KG);
      bool left = false;  // for the end
      if (key0 + KT > full_hi || key0 < full_lo || missing) {
        // keys of the tile that are there
        auto pages_there = [&]() {
          const int at = key0 + lane;
          return __ballot(at < w.keys && page_ok(lookup(min(at, w.keys - 1))));
        };
        unsigned long long there = PAGED && missing ? pages_there() : ~0ull;
        const unsigned long long mine = there >> 4 * half;
#pragma unroll
        for (int kt = 0; kt < KT / 32; ++kt)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int k = 32 * kt + 8 * (r / 4) + r % 4, at = key0 + k + 4 * half;
            if (at >= my_hi || at < my_lo || !(mine >> k & 1)) s[kt][r] = -INFINITY;
          }
        if constexpr (CAREFUL) {
          // A value that is not finite must not meet the weight of zero of a pair that does not see it: a tile with such is left
          // for the end.  Values of pages that are not there become zeros instead (every wave that finds some writes these
          // ahead of its own reads; no pair sees them).
          auto look = [&]() {
            float sums[4] = {0.f, 0.f, 0.f, 0.f};  // 0, or NaN (0 times what is not finite)
#pragma unroll 1
            for (int j = 0; j < KP; ++j) {
              const u32x4 x = read_tile((lds_vec_ptr)(base + TILEB + j * 1024 + lane * 16));
#pragma unroll
              for (int e = 0; e < 4; ++e) sums[e] = dot_dword<T>(x[e], 0u, sums[e]);
            }
            return __ballot(sums[0] + sums[1] + sums[2] + sums[3] != 0.f) != 0;
          };
          left = look();
          if (PAGED && left) {
            if (!missing) there = pages_there();
#pragma unroll 1
            for (int j = 0; j < KP; ++j)
              if (!(there >> (j * RPP + lane / CH) & 1))
                *(__attribute__((address_space(3))) u32x4*)(base + TILEB + j * 1024 + lane * 16) = u32x4{0u, 0u, 0u, 0u};
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            left = look();
          }
          if (left) {
            if (odd_last < 0) odd_first = key0;
            odd_last = key0;
          }
        }
      }
      float mx = s[0][0];
#pragma unroll
      for (int kt = 0; kt < KT / 32; ++kt)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[kt][r]);
      mx = xor32_max(mx);
      // (m starts at -inf: the first finite maximum exceeds it by inf)
      if (__ballot((mx - m) * c > 8.f || (m == -INFINITY && mx > m))) {
        const float m_new = fmaxf(m, mx);
        const float alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - m_new) * c);
        l *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[dt][r] *= alpha;
        m = m_new;
      }
      const float mc = (m == -INFINITY ? 0.f : m * c) - kShift;
      if (!left) {
#pragma unroll
        for (int kt = 0; kt < KT / 32; ++kt) {
          float sum = 0.f;
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            s[kt][r] = __builtin_amdgcn_exp2f(fmaf(s[kt][r], c, -mc));
            if constexpr (F32) sum += s[kt][r];
          }
          if constexpr (F32) {
#pragma unroll
            for (int r = 0; r < 16; ++r)
#pragma unroll
              for (int dt = 0; dt < DT; ++dt) {
                const float vf = *(const __attribute__((address_space(3))) float*)(base + vfrag[dt] + (32 * kt + 8 * (r / 4) + r % 4) * ROWB);
                o[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(vf, s[kt][r], o[dt], 0, 0, 0);
              }
          } else {
#pragma unroll
            for (int st = 0; st < 2; ++st) {
              frag pf;
#pragma unroll
              for (int j = 0; j < 8; ++j) pf[j] = (T)s[kt][8 * st + j];
#pragma unroll
              for (int j = 0; j < 8; j += 2) sum = PromptMma<T>::add_pair(pf[j], pf[j + 1], sum);
#pragma unroll
              for (int dt = 0; dt < DT; ++dt) {
                const lds_bytes at = base + vfrag[dt] + (32 * kt + 16 * st) * ROWB;
                const s16x4 lo4 = read_transposed((lds_tr_ptr)at);
                const s16x4 hi4 = read_transposed((lds_tr_ptr)(at + 8 * ROWB));
                const s16x8 both = __builtin_shufflevector(lo4, hi4, 0, 1, 2, 3, 4, 5, 6, 7);
                o[dt] = PromptMma<T>::mul(__builtin_bit_cast(frag, both), pf, o[dt]);
              }
            }
          }
          l += sum;
        }
      }
    } else {
      if (more) issue(t + KG, buf ^ 1, 0, RP);
      if (t + 2 * KG < t1) get_ids(t + 2 * KG);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  }
  if constexpr (CAREFUL) {
    // ---- the tiles that were left: key by key, each pair with those that it sees, from memory.  A lane has half of its pair's
    //      query and of its values ----
    for (int key0 = odd_first; key0 <= odd_last; key0 += KG * KT) {
      if (key0 + KT <= full_hi && key0 >= full_lo && !missing) continue;
      // a row's byte offset; whether it is there
      auto row_at = [&](int t, int64_t stride, bool& there) -> int64_t {
        if constexpr (PAGED) {
          const int page = lookup(t);
          there = page_ok(page);
          return paged_offset(page, t);
        } else {
          there = true;
          return t * stride * (int)sizeof(T);
        }
      };
      float sum = 0.f;
      for (int j = 0; j < KP; ++j) {
        const int t = key0 + j * RPP + lane / CH;
        bool there;
        const char* vr = reinterpret_cast<const char*>(vbase) + row_at(min(t, w.keys - 1), v_stride, there) + lane % CH * 16;
        if (t >= w.keys || !there) continue;
        const u32x4 x = *KX_CK(a, PP_V, reinterpret_cast<const u32x4*>(vr));
#pragma unroll
        for (int e = 0; e < 4; ++e) sum = dot_dword<T>(x[e], 0u, sum);
      }
      if (!__ballot(sum != 0.f)) continue;
      const float mc = (m == -INFINITY ? 0.f : m * c) - kShift;
#pragma unroll 1
      for (int t = max(key0, w_lo); t < min(key0 + KT, w_hi); ++t) {
        bool there;
        const char* kr = reinterpret_cast<const char*>(kbase) + row_at(t, k_stride, there) + 16 * half;
        const char* vr = reinterpret_cast<const char*>(vbase) + row_at(t, v_stride, there) + 4 * half * (int)sizeof(T);
        if (!there) continue;
        float x = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const u32x4 k4 = *KX_CK(a, PP_K, reinterpret_cast<const u32x4*>(kr + 32 * ks)), q4 = __builtin_bit_cast(u32x4, qf[ks]);
#pragma unroll
          for (int e = 0; e < 4; ++e) x = dot_dword<T>(k4[e], q4[e], x);
        }
        x += __shfl_xor(x, 32);
        const bool seen = t >= my_lo && t < my_hi;
        const float weight = seen ? (float)(T)__builtin_amdgcn_exp2f(fmaf(x, c, -mc)) : 0.f;
        l += half == 0 ? weight : 0.f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            float v4[4];
            load4(KX_CKN(a, PP_V, reinterpret_cast<const T*>(vr) + 32 * dt + 8 * q, 4 * sizeof(T)), v4);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[dt][4 * q + e] = seen ? fmaf(weight, v4[e], o[dt][4 * q + e]) : o[dt][4 * q + e];
          }
      }
    }
  }
  l = xor32_sum(l);
  if constexpr (KG > 1) {
    // the groups' results meet in LDS (nothing of the tiles is read any more)
    constexpr int PART = (DT * 16 + 2) * 64 * 4;  // bytes of a wave's o, m, l
    static_assert((KG - 1) * PW * PART <= 2 * KG * 2 * TILEB, "");
    if (group > 0) {
      char* mine = smem + (wave - PW) * PART;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<f32x4*>(mine + ((dt * 4 + q) * 64 + lane) * 16) =
              f32x4{o[dt][4 * q], o[dt][4 * q + 1], o[dt][4 * q + 2], o[dt][4 * q + 3]};
      *reinterpret_cast<float*>(mine + DT * 16 * 64 * 4 + lane * 4) = m;
      *reinterpret_cast<float*>(mine + (DT * 16 + 1) * 64 * 4 + lane * 4) = l;
    }
    __syncthreads();
    if (group == 0) {
#pragma unroll
      for (int g = 1; g < KG; ++g) {
        const char* part = smem + ((g - 1) * PW + wave) * PART;
        const float pm = *reinterpret_cast<const float*>(part + DT * 16 * 64 * 4 + lane * 4);
        const float pl = *reinterpret_cast<const float*>(part + (DT * 16 + 1) * 64 * 4 + lane * 4);
        const float m_new = fmaxf(m, pm);
        // a part without a maximum holds zeros, or NaN: those stay
        const float fa = m == m_new ? 1.f : m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - m_new) * c);
        const float fb = pm == m_new ? 1.f : pm == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((pm - m_new) * c);
        l = l * fa + pl * fb;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const f32x4 po = *reinterpret_cast<const f32x4*>(part + ((dt * 4 + q) * 64 + lane) * 16);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[dt][4 * q + e] = o[dt][4 * q + e] * fa + po[e] * fb;
          }
        m = m_new;
      }
    }
  }
  if (group == 0 && wf0 < pairs) {
    // ---- results: through the wave's part of LDS to whole rows ----
    const float inv = l == 0.f ? 0.f : 1.f / l;
    float sum = 0.f;  // NaN if any result is not finite
    // (with groups: where the first of the parts that this wave alone has read lies)
    char* region = smem + wave * (KG > 1 ? (DT * 16 + 2) * 256 : 32 * ROWB);
    static_assert((DT * 16 + 2) * 256 >= 32 * ROWB, "");
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        typedef T vec __attribute__((ext_vector_type(4)));
        vec y;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = o[dt][4 * q + e] * inv;
          if (!CAREFUL) sum = fmaf(x, 0.f, sum);
          y[e] = !CAREFUL || fabsf(x) < INFINITY ? round_to<T>(x) : (T)x;  // (an infinity that is seen stays one)
        }
        const int byte = (32 * dt + 8 * q + 4 * half) * (int)sizeof(T);
        *reinterpret_cast<vec*>(region + qcol * ROWB + ((byte >> 4 ^ k_swizzle<CH>(qcol)) << 4) + (byte & 15)) = y;
      }
    if (!CAREFUL) odd = __ballot(sum != 0.f) != 0;
    // (a wave's LDS instructions are served in order: it reads what its own lanes wrote)
#pragma unroll
    for (int j = 0; j < 32 / RPP; ++j) {
      const int r = j * RPP + lane / CH, p = lane % CH;
      const u32x4 y = *reinterpret_cast<const u32x4*>(region + r * ROWB + ((p ^ k_swizzle<CH>(r)) << 4));
      const int f = wf0 + r;
      if (f < pairs && odd == CAREFUL) {
        const int row = a.mul_div.page(f);
        char* dst = a.out + ((w.q0 + row) * a.out_stride + (kvh * a.kv_mul + f - row * a.kv_mul) * HS) * (int64_t)sizeof(T) + 16 * p;
        *KX_CKN(a, PP_OUT, reinterpret_cast<u32x4*>(dst), 16) = y;
      }
    }
  }
  if constexpr (CAREFUL) return false;
  if (lane == 0) sm_odd[wave] = odd;
  __syncthreads();
  int any = 0;
#pragma unroll
  for (int v = 0; v < NW; ++v) any |= sm_odd[v];
  return __builtin_amdgcn_readfirstlane(any) != 0;
}

template <typename T, int HS, int MODE, int KG, int NW>
__global__ __launch_bounds__(NW * 64, sizeof(T) == 2 && HS <= 64 ? NW / 2 : NW / 4) void prompt_attn_kernel(const PromptArgs a) {
  bool odd = false;
  if (__builtin_expect(prompt_attn<T, HS, MODE, KG, NW, false>(a, odd), false)) prompt_attn<T, HS, MODE, KG, NW, true>(a, odd);
}

// the two buffers; the rows of the results pass through the same place
template <typename T, int HS, int KG, int NW>
constexpr int prompt_lds() {
  const int row = HS * (int)sizeof(T), tiles = 2 * KG * 2 * pa_keys<T>() * row, rows = KG == 1 ? NW * 32 * row : 0;
  return tiles > rows ? tiles : rows;
}

template <typename T, int HS, int MODE, int KG, int NW>
static int prompt_launch(const PromptArgs& a, hipStream_t s) {
  constexpr int pairs = NW / KG * 32, lds = prompt_lds<T, HS, KG, NW>();
  // blocks of the sequences: an even share of all pairs and one more each
  const int64_t items = (int64_t)a.q_rows * a.kv_mul / pairs + a.batch;
  if (!grid_fits(items * a.kv_heads, NW * 64)) return KX_ELIMIT;
  static OncePerDevice limit;
  if (lds > 32768)
    if (const int rc = limit.raise(reinterpret_cast<const void*>(&prompt_attn_kernel<T, HS, MODE, KG, NW>), lds)) return rc;
  hipLaunchKernelGGL((prompt_attn_kernel<T, HS, MODE, KG, NW>), dim3((unsigned)(items * a.kv_heads)), dim3(NW * 64), lds, s, a);
  KX_LAUNCH_CHECK();
  return KX_OK;
}
template <typename T, int HS, int KG, int NW>
static int prompt_mode(const PromptArgs& a, hipStream_t s) {
  if (!a.kv.table) return prompt_launch<T, HS, PA_PACKED, KG, NW>(a, s);
  if (a.kv.div.size % 16 == 0) return prompt_launch<T, HS, PA_BLOCK_PAGES, KG, NW>(a, s);
  return prompt_launch<T, HS, PA_ANY_PAGES, KG, NW>(a, s);
}
// Groups of waves per workgroup.  Two or more cut a sequence's chain of tiles and give that many times the workgroups, for
// as many times the K/V traffic per product.
//   16-bit: two groups where the call would not fill the chip with workgroups of 256 pairs (`blocks`) otherwise: under 320
//   of them, or with narrower heads, whose smaller tiles let two such workgroups share a CU, under 800 (64 wide) or 600 (32).
//   Measured (us, one group / two; causal, 32 heads over 8): 128 wide, blocks 64: 19.8 / 14.4, 256: 63.5 / 53.1, 346: 34.1 /
//   37.9 (8 prompts), 375: 95.6 / 102, 512 (a prompt of 4096): 143 / 155; 64 wide, 85: 11.0 / 9.1, 473: 36.3 / 30.4, 512: 97.2 /
//   87.7, 1090: 88.2 / 93.2, 2085: 134 / 151; 32 wide, 74: 34.4 / 20.2, 512: 76.9 / 63.0, 674: 51.7 / 57.8.
//   fp32: as many groups as LDS holds buffers for, always: its products take sixteen times as long and hide the traffic
//   (64 wide, blocks 31: one 33.7, two 26.8, four 18.9; 612: one 367, four 303; 128 wide, 512: one 1145, two 1097).  Four waves
//   instead of eight, one per SIMD, where that many more workgroups still find CUs of their own, or nearly: the chain of
//   products of a SIMD is half as long.  Measured (us, eight / four, by the workgroups that eight would take): 128 wide, 23:
//   54.7 / 35.2, 136: 60.2 / 42.1, 280: 49.0 / 38.0, 560: 58.2 / 70.9; 64 wide, 84: 17.3 / 14.4, 180: 27.6 / 20.9, 232: 18.2 /
//   19.4, 384: 76.7 / 96.6; 32 wide, 52: 11.3 / 9.8, 138: 42.7 / 32.8, 348: 51.0 /
//   47.1, 650: 26.3 / 33.8.  (16-bit types: nothing, 26.6 / 25.0 at best.)
template <typename T, int HS>
static int prompt_groups(const PromptArgs& a, hipStream_t s) {
  if constexpr (sizeof(T) == 4) {
    constexpr int KG = prompt_lds<T, HS, 4, 8>() <= 131072 ? 4 : 2;
    const int64_t workgroups = ((int64_t)a.q_rows * a.kv_mul / (8 / KG * 32) + a.batch) * a.kv_heads;  // of eight waves
    return workgroups <= (HS == 64 ? 200 : HS == 32 ? 400 : 320) ? prompt_mode<T, HS, KG, 4>(a, s) : prompt_mode<T, HS, KG, 8>(a, s);
  } else {
    const double blocks = (double)a.q_rows * a.kv_mul / 256 * a.kv_heads;
    return blocks < (HS == 128 ? 320 : HS == 64 ? 800 : 600) ? prompt_mode<T, HS, 2, 8>(a, s) : prompt_mode<T, HS, 1, 8>(a, s);
  }
}
template <typename T>
static int prompt_hs(const PromptArgs& a, int hs, hipStream_t s) {
  return hs == 32 ? prompt_groups<T, 32>(a, s) : hs == 64 ? prompt_groups<T, 64>(a, s) : prompt_groups<T, 128>(a, s);
}

}  // namespace kx

extern "C" int kx_prompt_attention(const kx_prompt_attn_desc* d, void* stream) {
  using namespace kx;
  if (!d || d->batch < 0 || d->q_rows < 0) return KX_EINVAL;
  if (d->batch == 0 || d->q_rows == 0) return KX_OK;
  if (!kind_known(d->type) || d->head_num <= 0 || d->kv_head_num <= 0 || d->head_num % d->kv_head_num) return KX_EINVAL;
  if (!head_size_known(d->head_size)) return KX_EUNSUPPORTED;
  if (d->window < 0 || (d->window > 0 && !d->causal) || !isfinite(d->scale)) return KX_EINVAL;
  const int64_t q_dim = (int64_t)d->head_num * d->head_size, kv_dim = (int64_t)d->kv_head_num * d->head_size;
  const size_t bytes = kind_bytes(d->type), unit = 16 / bytes;
  if (!d->q || !d->out || !d->cu_q || !aligned4(d->cu_q) || !aligned16(d->q) || !aligned16(d->out) ||
      !stride_ok(d->q_stride, q_dim, unit) || !stride_ok(d->out_stride, q_dim, unit))
    return KX_EINVAL;
  PromptArgs a{};
  if (d->pages) {
    if (d->k || d->v || d->cu_k) return KX_EINVAL;
    if (const int rc = paged_check(*d->pages)) return rc;
    if (d->pages->type != d->type) return KX_EUNSUPPORTED;
    if (d->pages->kv_head_num != d->kv_head_num || d->pages->head_size != d->head_size || d->pages->batch != d->batch)
      return KX_EINVAL;
    // (a page's and a row's bytes are counted in 32 bits)
    if ((uint64_t)d->pages->page_stride * bytes > 0xffffffffull || (uint64_t)d->pages->row_stride * bytes * 16 > 0x7fffffffull)
      return KX_EUNSUPPORTED;
    a.kv = paged_view(*d->pages);
    a.k = a.kv.key;
    a.v = a.kv.value;
  } else {
    if (!d->k || !d->v || !d->cu_k || !aligned4(d->cu_k) || d->k_rows < 0 || !aligned16(d->k) || !aligned16(d->v) ||
        !stride_ok(d->k_stride, kv_dim, unit) || !stride_ok(d->v_stride, kv_dim, unit))
      return KX_EINVAL;
    // the rows of a buffer (256 keys at most) are addressed by 31-bit offsets from the first one
    if ((uint64_t)d->k_stride * bytes * 256 > 0x7fffffffull || (uint64_t)d->v_stride * bytes * 256 > 0x7fffffffull)
      return KX_EUNSUPPORTED;
    a.k = static_cast<const char*>(d->k);
    a.v = static_cast<const char*>(d->v);
  }
  const int32_t kv_mul = d->head_num / d->kv_head_num;
  // (row, head) pairs, keys and the elements of a row are counted in 31 bits
  if ((int64_t)d->q_rows * kv_mul > 0x7fff0000ll || (!d->pages && d->k_rows > kMostPositions) || q_dim > 0x7fffffffll) return KX_ELIMIT;
  a.q = static_cast<const char*>(d->q); a.out = static_cast<char*>(d->out); a.cu_q = d->cu_q; a.cu_k = d->cu_k;
  a.q_stride = d->q_stride; a.k_stride = d->k_stride; a.v_stride = d->v_stride; a.out_stride = d->out_stride;
  a.batch = d->batch; a.kv_heads = d->kv_head_num; a.kv_mul = kv_mul; a.mul_div = page_div(kv_mul);
  a.q_rows = d->q_rows; a.k_rows = d->k_rows; a.causal = d->causal; a.window = d->window; a.scale = d->scale;
  const void* operands[] = {a.q, a.k, a.v, a.out, a.cu_q, a.cu_k, a.kv.table, a.kv.seq_lens};
  for (int i = 0; i < 8; ++i) KX_BSET(a, i, operands[i]);
  (void)operands;
  hipStream_t s = (hipStream_t)stream;
  return d->type == KX_F16 ? prompt_hs<_Float16>(a, d->head_size, s)
         : d->type == KX_BF16 ? prompt_hs<__bf16>(a, d->head_size, s) : prompt_hs<float>(a, d->head_size, s);
}
