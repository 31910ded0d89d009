// Attention of one new token per sequence over the pages of a KV cache, one launch for a ragged batch.
//
//   s_t = scale q . k_t,  out = sum_t e^{s_t - m} v_t / sum_t e^{s_t - m},  t in [max(0, len - window), len)
//
// Bound: every K and V row of a kv head is read once for the query heads that share it (2 len hs bytes per element
// size); at 16 heads per kv head the arithmetic is a fifth of what the matrix cores do in that time.  1.24 GB of three
// documents in 238 us (5.2 TB/s, a plain sum reads 5.7), 281 MB of 48 chats in 62.7 us (4.5 with start and end), a chat of
// 137 keys in 6.4 us, of which a launch is the most.
//
// Cut: the 16-key blocks of the whole batch are dealt over the chip.  Every workgroup reads the lengths, sums
// the tiles, derives the same chunk length c from the sum and finds its own (sequence, chunk) by a prefix sum: no
// plan from the host, so a captured launch follows the lengths.  The results of a cut sequence meet in the workspace
// and the workgroup that arrives last joins them in the order of the chunks: results do not depend on arrival.
//
// Tile: 32 keys (16 with an fp32 cache) per wave, in registers, the next one requested ahead.  S^T = K Q^T with keys on the
// rows and heads on the columns of a 16 x 16 tile leaves the weights of 4 keys per 16-key block in a lane, which is
// the B operand of O^T = V^T P^T if V rows are taken in that order; the A operand V^T is made of the loaded
// rows by byte permutes within the lane.  Nothing crosses lanes but the maximum.
//
// Arithmetic: products of 16-bit operands are exact in fp32.  An fp32 query is split into parts of the cache's
// type (fp16: two parts of 11 bits, scaled by a power of two so that the largest element sits at 2^14 and the
// parts of elements 2^14 smaller are still whole; bf16: three parts of 8 bits); the weights likewise: two parts of fp16, e^x scaled to 2^15, three
// of bf16 where the result is fp32, two where it is bf16 (17 bits, far below the result's 8).  Sums, maxima and the join are fp32.
#include <math.h>

#include <type_traits>

#define KX_FILE_ID 11
#include "paged.hpp"

namespace kx {

enum DecodeOperand { PD_KEY, PD_VALUE, PD_TABLE, PD_LENS, PD_Q, PD_OUT, PD_WS };

constexpr int kPdWaves = 4;
// Workgroups that a batch is cut for, two rounds of what the chip holds.  Measured (us, 512 / 768 / 1024 / 1536 / 2048): three
// documents of 60 - 131 k keys 276 / 231 / 237 / 245 / 245, 48 chats of 1 - 8192 keys 66.9 / 65.4 / 62.8 / 64.6 / 64.8.  (512 workgroups
// that take their work from a counter: 249 and 66.3, or with one counter per XCD 254 and 68.6.)
constexpr int kPdSlots = 1024;
constexpr int kPdMaxSplits = 128;   // chunks of one sequence
constexpr int kPdLeastChunk = 16;   // tiles of a chunk at least (16 fp32 sequences of 500-4400 keys: 33.2 us with 8, 29.3 with 16)

struct PagedDecodeArgs {
  PagedView kv;
  const void* q;
  void* out;
  float* records;     // [record][head of the group][HS + 4]
  unsigned* tickets;  // [first record of a sequence][kv head and group], 64 bytes apart
  int64_t q_stride, out_stride;
  int32_t head_num, kv_heads, kv_mul, groups, group_heads, window, items;
  PageDiv heads_div;  // division by kv_heads * groups
  float scale, per_item;  // per_item: 1 / items
  KX_BFIELD(7)
};

// What a workgroup works on.
struct DecodeWork {
  int b, len, lo;        // sequence, its rows, the first one that is seen
  int tile0, tiles;      // this chunk's tiles
  int split, nsplit, record;  // chunk number of how many, and the first chunk's record
};

template <int TK>
__device__ __forceinline__ bool find_work(const PagedDecodeArgs& a, int item, DecodeWork& w) {
  const int lane = lane_id(), batch = a.kv.batch;
  auto length = [&](int b) { return b < batch ? max(*KX_CK(a, PD_LENS, a.kv.seq_lens + b), 0) : 0; };
  auto first = [&](int len) { return a.window > 0 ? max(0, len - a.window) : 0; };
  auto rows = [&](int len) { return min(len, a.kv.capacity()); };  // those that the table has places for
  auto tiles_of = [&](int len) { return rows(len) > first(len) ? (rows(len) - 1) / TK - first(len) / TK + 1 : 0; };
  // The chunk length: an even share, and no sequence in more than kPdMaxSplits.  (Sums past 2^24 tiles are rounded:
  // the grid and the records have one item to spare for the share, the limit gets one tile more.  2^27 tiles hold any sequence.)
  float sum = 0.f, most = 0.f;
  int len = 0, tiles = 0;
  for (int base = 0; base < batch; base += 64) {
    len = length(base + lane);
    tiles = tiles_of(len);
    sum += (float)tiles;
    most = fmaxf(most, (float)tiles);
  }
  sum = wave_sum(sum);
  most = wave_max(most);
  const float share = ceilf(sum * a.per_item), limit = ceilf(most * (1.f / kPdMaxSplits)) + (most >= 16777216.f ? 1.f : 0.f);
  const int chunk = max(kPdLeastChunk, ((int)fminf(fmaxf(share, limit), 134217728.f) + kPdWaves - 1) / kPdWaves * kPdWaves);
  int done = 0, records = 0;
  for (int base = 0; base < batch; base += 64) {
    if (batch > 64) {
      len = length(base + lane);
      tiles = tiles_of(len);
    }
    const int n = base + lane < batch ? max(1, (tiles + chunk - 1) / chunk) : 0;
    const int upto = wave_scan(n), cut = wave_scan(n > 1 ? n : 0);
    const unsigned long long past = __ballot(done + upto > item);
    if (past) {
      const int l = __builtin_ctzll(past);
      w.b = base + l;
      const int length_b = __builtin_amdgcn_readlane(len, l);
      w.len = rows(length_b);
      w.nsplit = __builtin_amdgcn_readlane(n, l);
      w.split = item - (done + __builtin_amdgcn_readlane(upto, l) - w.nsplit);
      w.record = records + __builtin_amdgcn_readlane(cut, l) - w.nsplit;
      w.lo = first(length_b);
      const int all = __builtin_amdgcn_readlane(tiles, l);
      int each = all;
      if (w.nsplit > 1) each = all / w.nsplit;
      const int more = all - each * w.nsplit;
      w.tile0 = w.lo / TK + w.split * each + min(w.split, more);
      w.tiles = each + (w.split < more ? 1 : 0);
      return true;
    }
    done += __builtin_amdgcn_readlane(upto, 63);
    records += __builtin_amdgcn_readlane(cut, 63);
  }
  return false;
}

// ---- the two products by cache type ----
template <typename KVT> struct DecodeMma;
template <> struct DecodeMma<_Float16> {
  typedef f16x8 frag;
  static __device__ __forceinline__ f32x4 mul(frag a, frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
template <> struct DecodeMma<__bf16> {
  typedef bf16x8 frag;
  static __device__ __forceinline__ f32x4 mul(frag a, frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};

template <typename KVT, int HS, bool UNI>
struct DecodeTile16 {  // 32 keys of a 16-bit cache
  static constexpr int VD = HS / 32;  // dwords of a V row in a lane (HS / 16 elements)
  u32x4 k[2][HS / 32];
  unsigned v[8][VD];
};
template <int HS>
struct DecodeTile32 {  // 16 keys of an fp32 cache
  f32x4 k[HS / 16];
  float v[4][HS / 16];
};

// Pages of a tile's rows.  UNI (pages of whole 16-key blocks): one page per block, in a scalar register.  Else a
// lane looks up the rows that it loads: its K row and its four V rows of each block.
template <int SUB, bool UNI>
struct DecodePages {
  int k[SUB];
  int v[UNI ? 1 : SUB * 4];
};

template <typename QT, typename KVT, int HS, bool UNI>
__global__ __launch_bounds__(kPdWaves * 64, 2) void paged_decode_kernel(const PagedDecodeArgs a) {
  constexpr bool F32KV = sizeof(KVT) == 4;
  constexpr int SUB = F32KV ? 1 : 2, TK = 16 * SUB;
  constexpr int VE = HS / 16;            // elements of a V row in a lane
  constexpr int OE = VE;                 // output tiles
  constexpr int ROW = HS + 4;            // floats of a record's head: O, m, l, two unused
  __shared__ __attribute__((aligned(16))) float sm_o[kPdWaves][16][ROW];
  __shared__ float sm_w[kPdWaves][kPdMaxSplits];
  __shared__ int sm_last;

  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int heads_of = a.kv_heads * a.groups;  // workgroups per item
  const int item = a.heads_div.page(blockIdx.x), hv = blockIdx.x - item * heads_of;
  const int kvh = a.groups == 1 ? hv : hv / a.groups, head0 = kvh * a.kv_mul + (hv - kvh * a.groups) * a.group_heads;
  const int heads = min(a.group_heads, (kvh + 1) * a.kv_mul - head0);
  DecodeWork w;
  if (!find_work<TK>(a, item, w)) return;

  // ---- rows ----
  const int32_t* table = a.kv.table + w.b * a.kv.table_stride;
  const KVT* key = reinterpret_cast<const KVT*>(a.kv.key) + kvh * a.kv.head_stride;
  const KVT* value = reinterpret_cast<const KVT*>(a.kv.value) + kvh * a.kv.head_stride;
  const int last = w.len - 1;
  auto page_ok = [&](int p) { return (unsigned)p < (unsigned)a.kv.num_pages; };
  auto lookup = [&](int t) { return *KX_CK(a, PD_TABLE, table + a.kv.div.page(t)); };
  // rows that are not seen are replaced by the nearest one that is: no address outside the sequence is formed
  auto seen_row = [&](int t) { return min(max(t, w.lo), last); };
  typedef DecodePages<SUB, UNI> Pages;
  auto get_pages = [&](Pages& p, int tile) {
#pragma unroll
    for (int i = 0; i < SUB; ++i) {
      const int t0 = tile * TK + 16 * i;
      if constexpr (UNI) {
        p.k[i] = __builtin_amdgcn_readfirstlane(lookup(seen_row(min(max(t0, w.lo & ~15), last & ~15))));
      } else {
        p.k[i] = lookup(seen_row(t0 + n));
#pragma unroll
        for (int r = 0; r < 4; ++r) p.v[4 * i + r] = lookup(seen_row(t0 + 4 * g + r));
      }
    }
  };
  auto row_at = [&](const KVT* base, int page, int t) {
    const int col = a.kv.div.page(t);
    return base + (page_ok(page) ? page : 0) * a.kv.page_stride + (t - col * a.kv.div.size) * a.kv.row_stride;
  };
  // the row that stands in for t: within its 16-key block, or the nearest block that is seen
  auto stand_in = [&](int t0, int j) { return seen_row(min(max(t0, w.lo & ~15), last & ~15) + j); };

  typedef typename std::conditional<F32KV, DecodeTile32<HS>, DecodeTile16<KVT, HS, UNI>>::type Tile;
  auto load_tile = [&](Tile& T, const Pages& p, int tile) {
#pragma unroll
    for (int i = 0; i < SUB; ++i) {
      const int t0 = tile * TK + 16 * i;
      const KVT* kr = row_at(key, p.k[i], UNI ? stand_in(t0, n) : seen_row(t0 + n));
      if constexpr (F32KV) {
#pragma unroll
        for (int j = 0; j < HS / 16; ++j)
          T.k[j] = *KX_CK(a, PD_KEY, reinterpret_cast<const f32x4*>(kr + 16 * j + 4 * g));
      } else {
#pragma unroll
        for (int s = 0; s < HS / 32; ++s)
          T.k[i][s] = *KX_CK(a, PD_KEY, reinterpret_cast<const u32x4*>(kr + 32 * s + 8 * g));
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int page = UNI ? p.k[i] : p.v[UNI ? 0 : 4 * i + r];
        const KVT* vr = row_at(value, page, UNI ? stand_in(t0, 4 * g + r) : seen_row(t0 + 4 * g + r)) + VE * n;
        (void)KX_CKN(a, PD_VALUE, vr, VE * sizeof(KVT));
        if constexpr (F32KV) {
          typedef float vec __attribute__((ext_vector_type(VE < 4 ? VE : 4)));
#pragma unroll
          for (int c = 0; c < VE; c += VE < 4 ? VE : 4) {
            const vec x = *reinterpret_cast<const vec*>(vr + c);
#pragma unroll
            for (int e = 0; e < (VE < 4 ? VE : 4); ++e) T.v[r][c + e] = x[e];
          }
        } else if constexpr (VE == 8) {
          const u32x4 x = *reinterpret_cast<const u32x4*>(vr);
#pragma unroll
          for (int c = 0; c < 4; ++c) T.v[4 * i + r][c] = x[c];
        } else if constexpr (VE == 4) {
          const u32x2 x = *reinterpret_cast<const u32x2*>(vr);
          T.v[4 * i + r][0] = x[0];
          T.v[4 * i + r][1] = x[1];
        } else {
          T.v[4 * i + r][0] = *reinterpret_cast<const unsigned*>(vr);
        }
      }
    }
  };

  f32x4 o[OE];
#pragma unroll
  for (int e = 0; e < OE; ++e) o[e] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;

  int t = w.tile0 + wave;
  const int t_end = w.tile0 + w.tiles;
  if (t < t_end) {
    Pages pg, pg_next;
    Tile cur, nxt;
    // ---- the queries: lane (head n, g) holds the dims of the K fragment that it multiplies ----
    constexpr int QP = F32KV ? 1 : sizeof(QT) == 2 ? 1 : sizeof(KVT) == 2 && std::is_same<KVT, _Float16>::value ? 2 : 3;
    constexpr int PP = F32KV ? 1 : sizeof(QT) == 4 && std::is_same<KVT, __bf16>::value ? 3 : 2;
    const QT* qr = static_cast<const QT*>(a.q) + w.b * a.q_stride + (int64_t)(head0 + min(n, heads - 1)) * HS;
    // scores in powers of two; a negative scale turns the queries' sign, and a scale of zero still hides (-inf * 0 is NaN)
    float unscale = fabsf(a.scale) * 1.4426950408889634f;
    constexpr int QV = F32KV || sizeof(QT) == 4 ? HS / 16 : HS / 32;  // 16-byte pieces
    u32x4 raw[QV];
    auto load_q = [&]() {
#pragma unroll
      for (int j = 0; j < QV; ++j) {
        const int d = F32KV ? 16 * j + 4 * g : sizeof(QT) == 4 ? 32 * (j / 2) + 8 * g + 4 * (j % 2) : 32 * j + 8 * g;
        raw[j] = *KX_CK(a, PD_Q, reinterpret_cast<const u32x4*>(qr + d));
      }
    };
    // queries that are taken apart are requested ahead of the first tile and taken apart beside its way here (one short
    // sequence: 6.4 us, 6.9 otherwise); the others behind it
    constexpr bool Q_FIRST = QP > 1;
    if (Q_FIRST) load_q();
    get_pages(pg, t);
    load_tile(cur, pg, t);
    if (t + kPdWaves < t_end) get_pages(pg_next, t + kPdWaves);
    if (!Q_FIRST) load_q();
    f32x4 qf[F32KV ? HS / 16 : 1];
    u32x4 qh[F32KV ? 1 : QP][F32KV ? 1 : HS / 32];
    if constexpr (F32KV) {
#pragma unroll
      for (int j = 0; j < HS / 16; ++j) qf[j] = __builtin_bit_cast(f32x4, raw[j]) * (a.scale < 0.f ? -1.f : 1.f);
    } else if constexpr (sizeof(QT) == 2) {
#pragma unroll
      for (int s = 0; s < HS / 32; ++s) qh[0][s] = raw[s] ^ (a.scale < 0.f ? 0x80008000u : 0u);
    } else {
      float x[HS / 32][8], big = 0.f;
#pragma unroll
      for (int s = 0; s < HS / 32; ++s)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[s][e] = __uint_as_float(raw[2 * s + e / 4][e % 4]);
          big = fmaxf(big, fabsf(x[s][e]));
        }
      int up = 0;
      if constexpr (std::is_same<KVT, _Float16>::value) {
        big = xor32_max(xor16_max(big));
        up = big > 0.f && big < INFINITY ? min(14 - __builtin_amdgcn_frexp_expf(big), 64) : 0;
        unscale = ldexpf(unscale, -up);
      }
#pragma unroll
      for (int s = 0; s < HS / 32; ++s) {
        typename DecodeMma<typename std::conditional<F32KV, _Float16, KVT>::type>::frag part[QP];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float rest = ldexpf(a.scale < 0.f ? -x[s][e] : x[s][e], up);
#pragma unroll
          for (int p = 0; p < QP; ++p) {
            const KVT h = (KVT)rest;
            part[p][e] = h;
            rest -= (float)h;
          }
        }
#pragma unroll
        for (int p = 0; p < QP; ++p) qh[p][s] = __builtin_bit_cast(u32x4, part[p]);
      }
    }

    unscale = fmaxf(unscale, 1.2e-38f);

    for (;;) {
      const bool more = t + kPdWaves < t_end;
      const Pages pg_now = pg;
      if (more) {
        pg = pg_next;
        load_tile(nxt, pg, t + kPdWaves);
        if (t + 2 * kPdWaves < t_end) get_pages(pg_next, t + 2 * kPdWaves);
      }
      // ---- scores: lane (head n, g) gets keys t0 + 16 i + 4 g + r ----
      float s[SUB][4];
#pragma unroll
      for (int i = 0; i < SUB; ++i) {
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
        if constexpr (F32KV) {
#pragma unroll
          for (int j = 0; j < HS / 16; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              acc = __builtin_amdgcn_mfma_f32_16x16x4f32(cur.k[j][e], qf[j][e], acc, 0, 0, 0);
        } else {
          typedef DecodeMma<KVT> Mma;
#pragma unroll
          for (int p = QP - 1; p >= 0; --p)
#pragma unroll
            for (int st = 0; st < HS / 32; ++st)
              acc = Mma::mul(__builtin_bit_cast(typename Mma::frag, cur.k[i][st]),
                             __builtin_bit_cast(typename Mma::frag, qh[p][st]), acc);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) s[i][r] = acc[r];
      }
      // ---- rows that are not seen: no weight, and no value either (0 x NaN is NaN) ----
      bool all_pages = true;
#pragma unroll
      for (int i = 0; i < SUB; ++i) {
        if constexpr (UNI) {
          all_pages &= page_ok(pg_now.k[i]);
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r) all_pages &= page_ok(pg_now.v[UNI ? 0 : 4 * i + r]);
        }
      }
      if constexpr (!UNI) all_pages = __ballot(all_pages) == ~0ull;
      if (!all_pages || t * TK < w.lo || t * TK + TK > w.len) {
#pragma unroll
        for (int i = 0; i < SUB; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int at = t * TK + 16 * i + 4 * g + r;
            const bool seen = at >= w.lo && at < w.len && page_ok(UNI ? pg_now.k[i] : pg_now.v[UNI ? 0 : 4 * i + r]);
            s[i][r] = seen ? s[i][r] : -INFINITY;
            if constexpr (F32KV) {
#pragma unroll
              for (int e = 0; e < VE; ++e) cur.v[r][e] = seen ? cur.v[r][e] : 0.f;
            } else {
#pragma unroll
              for (int c = 0; c < HS / 32; ++c) cur.v[4 * i + r][c] = seen ? cur.v[4 * i + r][c] : 0u;
            }
          }
      }
      float mx = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3]));
      if constexpr (SUB == 2) mx = fmaxf(mx, fmaxf(fmaxf(s[SUB - 1][0], s[SUB - 1][1]), fmaxf(s[SUB - 1][2], s[SUB - 1][3])));
      mx = xor32_max(xor16_max(mx)) * unscale;
      const float m_new = fmaxf(m, mx);
      if (__ballot(m_new > m)) {
        const float alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - m_new);
        l *= alpha;
#pragma unroll
        for (int e = 0; e < OE; ++e) o[e] *= alpha;
        m = m_new;
      }
      // weights, scaled by 2^15 where fp16 holds them; nothing seen so far: e^(-inf) = 0
      const float base = (m == -INFINITY ? 0.f : m) - (std::is_same<KVT, _Float16>::value ? 15.f : 0.f);
      float p[SUB][4];
#pragma unroll
      for (int i = 0; i < SUB; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          p[i][r] = __builtin_amdgcn_exp2f(fmaf(s[i][r], unscale, -base));
          l += p[i][r];
        }
      // ---- O^T += V^T P^T: output tile e holds dims VE * (4 g + r) + e of head n ----
      if constexpr (F32KV) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int e = 0; e < OE; ++e)
            o[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(cur.v[r][e], p[0][r], o[e], 0, 0, 0);
      } else {
        typedef DecodeMma<KVT> Mma;
        typename Mma::frag pf[PP];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float rest = p[(j >> 2) % SUB][j & 3];
#pragma unroll
          for (int q = 0; q < PP; ++q) {
            const KVT h = (KVT)rest;
            pf[q][j] = h;
            rest -= (float)h;
          }
        }
#pragma unroll
        for (int e = 0; e < OE; ++e) {
          u32x4 vf;  // element e of the eight rows
#pragma unroll
          for (int c = 0; c < 4; ++c)
            vf[c] = __builtin_amdgcn_perm(cur.v[2 * c + 1][e / 2], cur.v[2 * c][e / 2], e & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
          for (int q = PP - 1; q >= 0; --q) o[e] = Mma::mul(__builtin_bit_cast(typename Mma::frag, vf), pf[q], o[e]);
        }
      }
      if (!more) break;
      cur = nxt;
      t += kPdWaves;
    }
  }

  // ---- the waves of the workgroup meet in LDS ----
  l = xor32_sum(xor16_sum(l));
  if (n < heads) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int e = 0; e < OE; ++e) sm_o[wave][n][VE * (4 * g + r) + e] = o[e][r];
    if (g == 0) {
      sm_o[wave][n][HS] = m;
      sm_o[wave][n][HS + 1] = l;
    }
  }
  __syncthreads();
  const int64_t rec_floats = (int64_t)a.group_heads * ROW;
  const __amdgpu_buffer_rsrc_t rec_rsrc =
      __builtin_amdgcn_make_buffer_rsrc(a.records + (int64_t)w.record * heads_of * rec_floats, 0, 0x7fffffff, 0x00020000);
  for (int idx = threadIdx.x; idx < heads * (HS / 4); idx += kPdWaves * 64) {
    const int head = idx / (HS / 4), d = idx % (HS / 4) * 4;
    float M = sm_o[0][head][HS];
#pragma unroll
    for (int v = 1; v < kPdWaves; ++v) M = fmaxf(M, sm_o[v][head][HS]);
    float L = 0.f;
    f32x4 O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int v = 0; v < kPdWaves; ++v) {
      const float f = sm_o[v][head][HS] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sm_o[v][head][HS] - M);
      // a wave that saw nothing holds zeros, or NaN of a NaN key (its maximum is -inf then): those stay
      L += M == -INFINITY ? sm_o[v][head][HS + 1] : sm_o[v][head][HS + 1] * f;
      const f32x4 x = *reinterpret_cast<const f32x4*>(&sm_o[v][head][d]);
      O += M == -INFINITY ? x : x * f;
    }
    if (w.nsplit == 1) {
      QT* dst = static_cast<QT*>(a.out) + w.b * a.out_stride + (int64_t)(head0 + head) * HS + d;
      typedef QT vec __attribute__((ext_vector_type(4)));
      vec y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = (QT)(L == 0.f ? 0.f : O[e] / L);
      *KX_CK(a, PD_OUT, reinterpret_cast<vec*>(dst)) = y;
    } else {
      // device-scope stores: written through to where the joining workgroup reads
      const unsigned at = (unsigned)(((w.split * heads_of + hv) * (int64_t)a.group_heads + head) * ROW) * 4u;
      KX_TOUCH(a, PD_WS, reinterpret_cast<const char*>(a.records + (int64_t)w.record * heads_of * rec_floats) + at + 4 * d, 16);
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, O), rec_rsrc, at + 4u * d, 0, 16);
      if (d == 0) {
        const u32x4 ml = {__float_as_uint(M), __float_as_uint(L), 0u, 0u};
        __builtin_amdgcn_raw_buffer_store_b128(ml, rec_rsrc, at + 4u * HS, 0, 16);
      }
    }
  }
  if (w.nsplit == 1) return;

  // ---- the workgroup that arrives last joins the chunks.  Its partners' records are complete: each storing wave
  //      has waited for the acknowledgement of its write-through stores ahead of the barrier and the ticket; they are
  //      read with device-scope loads, so neither side needs a cache write-back or invalidation ----
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    unsigned* ticket = a.tickets + ((int64_t)w.record * heads_of + hv) * (kTicketStride / 4);
    sm_last = atomicInc(KX_CK(a, PD_WS, ticket), (unsigned)w.nsplit - 1u) == (unsigned)w.nsplit - 1u;  // wraps to 0
  }
  __syncthreads();
  if (!sm_last) return;
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  constexpr int LPR = HS / 4, RG = 64 / LPR, PASS = 8;
  const int c4 = lane % LPR * 4, rg = lane / LPR;
  for (int head = wave; head < heads; head += kPdWaves) {
    auto at = [&](int split) { return (unsigned)(((split * heads_of + hv) * (int64_t)a.group_heads + head) * ROW) * 4u; };
    // weights of the chunks, two per lane
    float cm[kPdMaxSplits / 64], cl[kPdMaxSplits / 64], M = -INFINITY;
    bool odd = false;  // a chunk without a finite maximum but with a sum: NaN keys
#pragma unroll
    for (int c = 0; c < kPdMaxSplits / 64; ++c) {
      const int sp = c * 64 + lane;
      const u32x2 ml = __builtin_amdgcn_raw_buffer_load_b64(rec_rsrc, at(min(sp, w.nsplit - 1)) + 4u * HS, 0, 16);
      cm[c] = sp < w.nsplit ? __uint_as_float(ml.x) : -INFINITY;
      cl[c] = sp < w.nsplit ? __uint_as_float(ml.y) : 0.f;
      odd |= cl[c] != cl[c];
      M = fmaxf(M, cm[c]);
    }
    M = wave_max(M);
    float L = 0.f;
#pragma unroll
    for (int c = 0; c < kPdMaxSplits / 64; ++c) {
      const float f = cm[c] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(cm[c] - M);
      L += f * cl[c];
      sm_w[wave][c * 64 + lane] = f;
    }
    L = wave_sum(L);
    if (__ballot(odd)) L = NAN;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < w.nsplit; s0 += PASS * RG) {
      u32x4 x[PASS];
#pragma unroll
      for (int k = 0; k < PASS; ++k)
        x[k] = __builtin_amdgcn_raw_buffer_load_b128(rec_rsrc, at(min(s0 + k * RG + rg, w.nsplit - 1)) + 4u * c4, 0, 16);
#pragma unroll
      for (int k = 0; k < PASS; ++k) {
        const int sp = s0 + k * RG + rg;
        const float f = sp < w.nsplit ? sm_w[wave][sp] : 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = f == 0.f ? acc[e] : fmaf(__uint_as_float(x[k][e]), f, acc[e]);
      }
    }
#pragma unroll
    for (int off = 32; off >= LPR; off >>= 1)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += __shfl_xor(acc[e], off);
    if (rg == 0) {
      QT* dst = static_cast<QT*>(a.out) + w.b * a.out_stride + (int64_t)(head0 + head) * HS + c4;
      typedef QT vec __attribute__((ext_vector_type(4)));
      vec y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = (QT)(L == 0.f ? 0.f : acc[e] / L);
      *KX_CK(a, PD_OUT, reinterpret_cast<vec*>(dst)) = y;
    }
  }
}

// How the heads of a call are dealt: 16 query heads at most per workgroup, the groups of a kv head of equal size.
struct DecodeHeads {
  int kv_mul, groups, group_heads;
};
static DecodeHeads decode_heads(int head_num, int kv_heads) {
  const int kv_mul = head_num / kv_heads, groups = (kv_mul + 15) / 16;
  return DecodeHeads{kv_mul, groups, (kv_mul + groups - 1) / groups};
}
// Chunks that the batch is cut into per (kv head, group): one workgroup each.
static int decode_items(int kv_heads, int groups) {
  const int n = kPdSlots / (kv_heads * groups);
  return n < 1 ? 1 : n;
}
// Records that a call may use.  A sequence that is cut has more tiles than a chunk, so its chunks are fewer than twice
// its share of `items`; one more for the rounding of the share.
static int decode_records(int items) { return 2 * items + 1; }
// records * (kv heads * groups) <= 2 * slots + kv heads * groups, and those are kPdSlots at most.
static_assert(3 * kPdSlots * kTicketStride <= kTicketBytes, "");

template <typename QT, typename KVT, int HS>
static void paged_decode_launch(const PagedDecodeArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)(a.items + a.kv.batch + 1) * a.kv_heads * a.groups), block(kPdWaves * 64);
  if (a.kv.div.size % 16 == 0)
    hipLaunchKernelGGL((paged_decode_kernel<QT, KVT, HS, true>), grid, block, 0, s, a);
  else
    hipLaunchKernelGGL((paged_decode_kernel<QT, KVT, HS, false>), grid, block, 0, s, a);
}
template <typename QT, typename KVT>
static void paged_decode_hs(const PagedDecodeArgs& a, int hs, hipStream_t s) {
  if (hs == 32) paged_decode_launch<QT, KVT, 32>(a, s);
  else if (hs == 64) paged_decode_launch<QT, KVT, 64>(a, s);
  else paged_decode_launch<QT, KVT, 128>(a, s);
}

}  // namespace kx

extern "C" size_t kx_paged_decode_workspace_bytes(int32_t batch, int32_t head_num, int32_t kv_head_num, int32_t head_size) {
  using namespace kx;
  if (batch <= 0 || head_num <= 0 || kv_head_num <= 0 || head_num % kv_head_num || head_size <= 0) return 0;
  const DecodeHeads h = decode_heads(head_num, kv_head_num);
  return kTicketBytes + (size_t)decode_records(decode_items(kv_head_num, h.groups)) * kv_head_num * h.groups *
                              h.group_heads * (head_size + 4) * sizeof(float);
}

extern "C" int kx_paged_decode(const kx_paged_decode_desc* d, void* stream) {
  using namespace kx;
  if (!d || d->kv.batch < 0) return KX_EINVAL;
  if (d->kv.batch == 0) return KX_OK;
  if (const int rc = paged_check(d->kv)) return rc;
  if (!kind_known(d->q_type) || d->head_num <= 0 || d->head_num % d->kv.kv_head_num || d->window < 0 || !isfinite(d->scale))
    return KX_EINVAL;
  if (!kinds_fit(d->q_type, d->kv.type)) return KX_EUNSUPPORTED;
  const int64_t q_dim = (int64_t)d->head_num * d->kv.head_size;
  const size_t unit = 16 / kind_bytes(d->q_type);
  if (!d->q || !d->out || !aligned16(d->q) || !aligned16(d->out) || !stride_ok(d->q_stride, q_dim, unit) ||
      !stride_ok(d->out_stride, q_dim, unit))
    return KX_EINVAL;
  if (!d->workspace || d->workspace_bytes < kx_paged_decode_workspace_bytes(d->kv.batch, d->head_num, d->kv.kv_head_num, d->kv.head_size))
    return KX_EWORKSPACE;
  if ((uintptr_t)d->workspace % 256) return KX_EINVAL;
  const DecodeHeads h = decode_heads(d->head_num, d->kv.kv_head_num);
  PagedDecodeArgs a{};
  a.kv = paged_view(d->kv);
  a.q = d->q;
  a.out = d->out;
  a.tickets = static_cast<unsigned*>(d->workspace);
  a.records = reinterpret_cast<float*>(static_cast<char*>(d->workspace) + kTicketBytes);
  a.q_stride = d->q_stride;
  a.out_stride = d->out_stride;
  a.head_num = d->head_num;
  a.kv_heads = d->kv.kv_head_num;
  a.kv_mul = h.kv_mul;
  a.groups = h.groups;
  a.group_heads = h.group_heads;
  a.window = d->window;
  if ((int64_t)a.kv_heads * a.groups > kPdSlots) return KX_EUNSUPPORTED;
  a.items = decode_items(a.kv_heads, a.groups);
  a.scale = d->scale;
  a.per_item = 1.f / (float)a.items;
  a.heads_div = page_div(a.kv_heads * a.groups);
  if (!grid_fits(((int64_t)a.items + a.kv.batch + 1) * a.kv_heads * a.groups, kPdWaves * 64)) return KX_ELIMIT;
  const void* operands[] = {a.kv.key, a.kv.value, a.kv.table, a.kv.seq_lens, a.q, a.out, d->workspace};
  for (int i = 0; i < 7; ++i) KX_BSET(a, i, operands[i]);
  (void)operands;
  hipStream_t s = (hipStream_t)stream;
  const int hs = d->kv.head_size;
  if (d->q_type == KX_F16) paged_decode_hs<_Float16, _Float16>(a, hs, s);
  else if (d->q_type == KX_BF16) paged_decode_hs<__bf16, __bf16>(a, hs, s);
  else if (d->kv.type == KX_F16) paged_decode_hs<float, _Float16>(a, hs, s);
  else if (d->kv.type == KX_BF16) paged_decode_hs<float, __bf16>(a, hs, s);
  else paged_decode_hs<float, float>(a, hs, s);
  KX_LAUNCH_CHECK();
  return KX_OK;
}
