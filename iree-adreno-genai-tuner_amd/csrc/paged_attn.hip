// Causal GQA attention over a paged KV cache with a prefix that the whole batch shares (paged_attn).
//
// For the token at position p of a sequence and query head h (KV head h / g): o = sum_j softmax_j(scale q . k_j) v_j over
// its keys j <= p. Any split of the keys into ranges gives the same result: a range yields m = max s, l = sum
// exp(s - m), o = sum exp(s - m) v, and ranges join as M = max m, o = sum e^(m - M) o / sum e^(m - M) l. So the shared keys
// are one range for all tokens of the batch, whose rows (token, head of the group) are stacked: their K and V are
// read once per 16 to 128 rows instead of once per sequence. The keys of a sequence's own are a second kind of range.
// Both run in one launch; a second joins the ranges of each row where there are several.
//
// Whole calls, back to back: one sequence of 700 keys (24/8 heads of 128, fp32) 9.9 us, a chain of dependent loads and two
// launches; 32 sequences behind 2048 shared keys (32/8 heads, fp16) 21 us; 64 behind 16384 (24/8, fp32) 64 us.
#include "q4_common.h"
#include "q4_paged.h"

#include <algorithm>
#include <cmath>

namespace q4 {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kKeys = 32;   // keys of a wave's block (streaming form)
constexpr int kStage = 64;  // keys of a workgroup's stage (shared form)
constexpr int kTurn = kWaves * kKeys;  // keys that the waves of the streaming form take side by side

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
template <int CT>
using vec8 = typename Num<CT>::type __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x4 mfma16(vec8<Q4_F16> a, vec8<Q4_F16> b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(vec8<Q4_BF16> a, vec8<Q4_BF16> b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32(vec8<Q4_F16> a, vec8<Q4_F16> b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32(vec8<Q4_BF16> a, vec8<Q4_BF16> b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
// Transposing LDS read: the lanes of each 16 read a 4 x 16 block of 16-bit values (lane i: row i / 4, columns
// 4 (i % 4) ..) and lane i receives column i.
__device__ __forceinline__ short4v read_tr4(const void* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)p);
}
// A product's result is written to its registers 12 (32x32) or 8 (16x16) wait states after its last instruction was issued. The
// compiler keeps what it emits away from them for so long, but does not look into inline assembly: values that max3 takes
// from a product pass through here first.
__device__ __forceinline__ void settle(f32x16& s) { asm("s_nop 11" : "+v"(s)); }
__device__ __forceinline__ void settle(f32x4& s, f32x4& t) { asm("s_nop 7" : "+v"(s), "+v"(t)); }
// The largest of three (a NaN loses); fmaxf costs an instruction per operand more, to quiet signalling NaNs.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

struct AttnArgs {
  PagedBatch b;
  const void* q;
  int64_t qr, qh;
  const void *kc, *vc;
  void* out;
  // Results of ranges, (m, l) and o: first the shared ones, [T * n_q][shared_splits], then the slots of own ranges, slot_rows
  // rows each. own: of each row the place of its first own range and their number.
  float *ml, *o;
  int2* own;  // null: every row has one range
  const int32_t* shared_pages;
  int T, n_q, n_kv, g, L, shared_len;
  int held;  // keys that the page lists hold, the shared ones or those of page_table (which the prefix may exceed), L at most
  int shared_blocks, shared_splits, shared_tile;  // workgroups of the shared ranges, ranges, rows of a workgroup
  int own_from, slot_rows, own_rows;              // own ranges: their first key, rows of a slot and of all slots
  bool longest_first, refill;
  int turn_from;
  float cs, sign;  // exponents are s * cs in log2 units; sign: that of the scale, taken into q
  int own_whole, own_items, own_most, places;     // items with all of their keys, items, ranges of an item at most and of all
  FastDiv by_g, by_kv, by_shared, by_ranges, by_tiles;
};

// Rows (token, head of the group) of a workgroup where there are `rows` in all. Up to 16 rows are not enough to share the
// keys among waves: each wave streams blocks of its own (paged_stream). Past them the waves share stages of keys
// in LDS (paged_shared), 32 rows a wave: two waves for the rows and two for the keys, or four for the rows. 8 sequences of
// 1000 to 6000 keys, 32/8 heads of 128, f16 (fp32): 4 rows in tiles of 16 and 64 30.7 and 33.6 us (30.8 and 34.1), 24
// rows in tiles of 64 and 128 35.6 and 37.3 (36.6 and 39.3), 160 rows in tiles of 64 and 128 73 and 61 (81 and 68).
__host__ __device__ __forceinline__ int tile_rows(int64_t rows) { return rows <= 16 ? 16 : rows <= 64 ? 64 : 128; }

// The sequence of token t, another in each lane (batch or more: none). Every lane of the wave takes part.
__device__ __forceinline__ int sequence_of_lane(const PagedBatch& b, int t) {
  if (!b.cu) return b.by_rows.div(t);
  int n = 0;
  for (int i = 0; i < b.batch; i += 64) {
    const int left = min(64, b.batch - i);
    const int v = b.cu[i + 1 + min(static_cast<int>(threadIdx.x & 63), left - 1)];
    for (int l = 0; l < left; ++l) n += __builtin_amdgcn_readlane(v, l) <= t;
  }
  return n;
}

// First token and number of tokens of sequence b.
__device__ __forceinline__ int2 tokens_of(const PagedBatch& b, int seq, int T) {
  if (!b.cu) return make_int2(seq * b.rows, b.rows);
  const int c0 = min(max(b.cu[seq], 0), T);
  return make_int2(c0, min(max(b.cu[seq + 1], c0), T) - c0);
}

__host__ __device__ __forceinline__ int tiles_of(int64_t rows) {
  const int h = tile_rows(rows);
  return static_cast<int>((rows + h - 1) / h);
}

constexpr int kMaxKeys = 1 << 30;  // positions of the blocks ahead stay below 2^31
constexpr int kSlots = 512;    // own ranges at once: two workgroups on every compute unit
constexpr int kMaxSplits = 64;  // ranges of a tile's keys

// Ranges of each of `items` that share `places`: as many as fit at once, or, where those leave more than an eighth of the
// places free, as many as fill them twice (the last ones start as the first end; `refill`: of many keys and few rows). One
// token each of 12 / 20 / 24 sequences of 1000 to 6000 keys, 16 heads of 64: 46.9 / 74.4 / 79.6 -> 40.0 / 61.2 / 84.6 us;
// 8 KV heads of 128, 24 / 40 sequences: 78 / 130 -> 70 / 109. Where they do fit (8 / 16 sequences of 16 heads), the second filling
// costs: 31.6 / 53.4 -> 32.4 / 57.8 us; so it does for more than 32 rows (10 tokens each of 40 sequences of 2100 keys, 32/8 heads of
// 128, 78 -> 84, of 80 with 16/4 of 64 43.4 -> 48.3). It gains as much below the limit of 2048 keys as above (40 sequences, 8
// heads of 64: 2000 keys 47.0 -> 42.3, 2100 49.2 -> 44.2), and nothing at 1000.
//
// One each where the free places times the keys are few (no shared ranges, which need a join anyway): what splitting saves of the
// time of an item, the free share of it, has to exceed what ranges cost, about that of 520 keys. 600 keys, 8 KV heads of 128,
// 24 sequences of 1 / 30 / 100 tokens 18.5 / 33.5 / 67.5 -> 15.4 / 27.9 / 55.7 us; 2 of them 10.7 / 16.5 / 23.7 as they are, 11.4 /
// 24.3 / 24.8 in one; 1000 keys, 8 and 24 of 100 tokens 42.7 / 95 -> 37.8 / 86.
__host__ __device__ __forceinline__ int ranges_of(int items, int places, bool refill, int most, int keys) {
  if (places == kSlots && keys > 4 * kTurn && static_cast<int64_t>(places - items) * keys <= places * 520) return 1;
  int n = places / items;
  if (refill && 8 * n * items < 7 * places) n = 2 * places / items;
  return n < 1 ? 1 : n < most ? n : most;
}

// Own items are the tiles of each KV head. As many as fill the compute units whole times take all of their keys at once; the
// rest, which would hold a few units and leave the others waiting, is split over all of them (of few items: all).
struct Own {
  int seq, tile, h;          // sequence, row tile in it, KV head
  int range, ranges, slot0;  // ranges: at most; slot0: that of the item's first range (a single range has one beside
                             // shared ranges only: without them it is the result)
};

// Item and range of own workgroup `idx` (wave-uniform); false: none.
__device__ __forceinline__ bool own_item(const AttnArgs& a, int idx, Own* w) {
  const int lane = threadIdx.x & 63;
  auto count = [&](int i) {  // lane: tiles of sequence i + lane
    const int s = min(i + lane, a.b.batch - 1);
    return i + lane < a.b.batch ? tiles_of(static_cast<int64_t>(tokens_of(a.b, s, a.T).y) * a.g) : 0;
  };
  int whole = a.own_whole, items = a.own_items;
  FastDiv by_ranges = a.by_ranges;
  if (a.b.cu) {
    int tiles = 0;
    for (int i = 0; i < a.b.batch; i += 64) tiles += count(i);
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) tiles += __shfl_xor(tiles, m, 64);
    items = __builtin_amdgcn_readfirstlane(tiles) * a.n_kv;
    whole = items / kSlots * kSlots;
    by_ranges.d = ranges_of(max(items - whole, 1), a.places, a.refill, a.own_most, a.L - a.own_from);
  }
  int item = idx;
  w->range = 0, w->ranges = 1, w->slot0 = idx;
  if (idx >= whole) {
    w->ranges = by_ranges.d;
    const int i = a.b.cu ? (idx - whole) / w->ranges : by_ranges.div(idx - whole);
    w->range = idx - whole - i * w->ranges;
    w->slot0 = (a.shared_splits ? whole : 0) + i * w->ranges;
    item = whole + i;
    if (item >= items) return false;
  }
  int tile = a.by_kv.div(item);
  w->h = item - tile * a.n_kv;
  if (a.longest_first) {
    // Longest first (a batch of 64 at most): those that wait for a place are short. Where none waits and each compute unit gets
    // a second one, the second ones go shortest first, so that the longest and the shortest share a unit.
    int seconds = a.turn_from;
    if (a.b.cu) {
      const int per = a.n_kv * w->ranges;
      seconds = a.shared_blocks == 0 && whole == 0 && items * w->ranges <= kSlots ? (kSlots / 2 + per - 1) / per : INT32_MAX;
    }
    if (tile >= seconds) tile = a.by_kv.div(items) - 1 - (tile - seconds);
    // The sequence that holds this tile of the order, bit by bit of the lengths (in 64 classes: the order need not be exact;
    // counting for each sequence the longer ones took 2 us of 64 sequences beside the shared keys' work).
    const int len = lane < a.b.batch ? a.b.lens[lane] : 0, most = a.L - a.own_from;
    const int n = a.b.cu ? count(0) : lane < a.b.batch ? static_cast<int>(a.by_tiles.d) : 0;
    const int bits = 32 - __builtin_clz(most), key = min(max(len - a.own_from, 0), most) >> max(bits - 6, 0);
    auto tiles_in = [&](uint64_t m) -> int {  // bit by bit of their numbers
      if (!a.b.cu) return __popcll(m) * static_cast<int>(a.by_tiles.d);
      int sum = 0;
      for (int i = 0;; ++i) {
        sum += __popcll(__ballot(n >> i & 1) & m) << i;
        if (!__ballot(n >> (i + 1))) return sum;
      }
    };
    uint64_t m = __ballot(n > 0);
    for (int i = min(bits, 6) - 1; i >= 0; --i) {
      const uint64_t ones = __ballot(key >> i & 1) & m;
      const int t = tiles_in(ones);
      if (tile < t) m = ones;
      else tile -= t, m &= ~ones;
    }
    for (; m; m &= m - 1) {  // equally long
      w->seq = __builtin_ctzll(m);
      const int t = __builtin_amdgcn_readlane(n, w->seq);
      w->tile = tile;
      if (tile < t) return true;
      tile -= t;
    }
    return false;
  }
  if (!a.b.cu) {
    w->seq = a.by_tiles.div(tile);
    w->tile = tile - w->seq * a.by_tiles.d;
    return true;
  }
  int base = 0;
  for (int i = 0; i < a.b.batch; i += 64) {
    const int n = count(i);
    int run = n;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const int o = __shfl_up(run, m, 64);
      if (lane >= m) run += o;
    }
    const uint64_t past = __ballot(base + run > tile);
    if (past) {
      const int l = __builtin_ctzll(past);
      w->seq = i + l;
      w->tile = tile - base - (__builtin_amdgcn_readlane(run, l) - __builtin_amdgcn_readlane(n, l));
      return true;
    }
    base += __builtin_amdgcn_readlane(run, 63);
  }
  return false;
}

// Swizzles of the 16-byte chunks of a key's row in LDS: V so that the four rows of a transposing read fall in different
// banks, K so that 16 rows at one chunk do.
template <int HD>
__device__ __forceinline__ int vswz(int r) {
  return HD == 128 ? (r & 3) << 2 : ((r >> 1) & 1) << 2;
}
template <int HD>
__device__ __forceinline__ int kswz(int r) {
  return HD == 128 ? (r & 15) : ((r >> 1) & 7);
}

// Row of the cache of key j from its page-list entry, -1 for none (past the end, or no page of the pool). No branch: one that
// skips the use of a loaded entry makes the compiler wait for every load in flight before the register is written again.
__device__ __forceinline__ int slot_at(const PagedBatch& b, int entry, int j, int end) {
  const int s = entry * b.page_size + (j - b.by_page.div(max(j, 0)) * b.page_size);
  const int bad = (entry >> 31) | ((b.num_pages - 1 - entry) >> 31) | ((end - 1 - j) >> 31);
  return s | bad;
}

// Address of row s of the cache (row 0 where there is none): one multiplication of 32 by 32 bits into 64.
__device__ __forceinline__ const unsigned char* row_at(const unsigned char* base, int s, uint32_t pitch) {
  return base + static_cast<uint64_t>(static_cast<uint32_t>(max(s, 0))) * pitch;
}

// What a workgroup does: the tile of rows, the keys of its range, and where the range's result goes. Ranges are dealt, not cut:
// range s of n has the blocks s, s + n, .. of the keys (of `turn` keys, as many as a workgroup takes at once), so that its first
// keys, and their page entries, are known before the length of the sequence is.
struct Item {
  bool shared;
  int h, seq, row0, n_rows, tok0;        // rows row0 .. of the n_rows that start at token tok0
  int part, ranges, slot0;               // the range's number, how many there are, their first slot (own ranges)
  int k0, step, k1;                      // blocks at k0, k0 + step, .. below k1
  int own_end;                           // the keys of the sequence (own ranges)
  const int32_t* table;                  // its row of the page table
  int behind;                            // own ranges: position of a token = behind + its index in the sequence
};

// The page-list entry of key j: of the shared keys, or of the sequence's own (past its list: its last entry).
__device__ __forceinline__ int page_at(const AttnArgs& a, const Item& it, int j) {
  const int p = a.b.by_page.div(j);
  return j < a.shared_len ? a.shared_pages[p] : it.table[min(p, a.b.max_pages - 1)];
}

// One row: its token and head, and how many keys of the range's kind it sees (0: none, or no row). Wave-uniform flow.
struct Row {
  int token, head, lim, in_tile;
  bool ok;
};
__device__ __forceinline__ Row row_of(const AttnArgs& a, const Item& it, int r) {
  Row w;
  w.ok = r < it.n_rows;
  const int i = a.by_g.div(r);
  w.token = it.tok0 + i;
  w.head = it.h * a.g + r - i * a.g;
  w.lim = 0;
  w.in_tile = r - it.row0;
  if (it.shared) {
    const int s = sequence_of_lane(a.b, w.ok ? w.token : 0);
    if (w.ok && s < a.b.batch) {
      const int2 tk = tokens_of(a.b, s, a.T);
      w.ok = w.token >= tk.x && w.token < tk.x + tk.y;
      const int len = a.b.lens[s];
      w.lim = min(min(len - tk.y + (w.token - tk.x) + 1, max(len, 0)), a.shared_len);
    } else {
      w.ok = false;
    }
  } else {
    w.lim = min(it.behind + i + 1, it.own_end);
  }
  if (!w.ok) w.lim = 0;
  return w;
}

// Eight consecutive values of a row of q as the B operand (with fp32: two fp16 terms), times the scale's sign; zeros where
// there is no row.
template <int QT, int CT>
__device__ __forceinline__ void load_q(const AttnArgs& a, const Row& w, int d, vec8<CT>* hi_out, vec8<CT>* lo_out) {
  typedef typename Num<QT>::type Q;
  typedef vec8<CT> C8;
  const Q* p = static_cast<const Q*>(a.q) + w.token * a.qr + w.head * a.qh + d;
  if constexpr (QT == Q4_F32) {
    f32x4 x = {}, y = {};
    if (w.ok) {
      x = *reinterpret_cast<const f32x4*>(p);
      y = *reinterpret_cast<const f32x4*>(p + 4);
    }
    const float neg1 = minus_one();
    uint32_t hi[4], lo[4];
    split_f16_pair(a.sign * x.x, a.sign * x.y, neg1, hi[0], lo[0]);
    split_f16_pair(a.sign * x.z, a.sign * x.w, neg1, hi[1], lo[1]);
    split_f16_pair(a.sign * y.x, a.sign * y.y, neg1, hi[2], lo[2]);
    split_f16_pair(a.sign * y.z, a.sign * y.w, neg1, hi[3], lo[3]);
    *hi_out = __builtin_bit_cast(C8, make_uint4(hi[0], hi[1], hi[2], hi[3]));
    *lo_out = __builtin_bit_cast(C8, make_uint4(lo[0], lo[1], lo[2], lo[3]));
  } else {
    uint4 x = make_uint4(0, 0, 0, 0);
    if (w.ok) x = *reinterpret_cast<const uint4*>(p);
    const uint32_t flip = a.sign < 0.0f ? 0x80008000u : 0u, keep = a.sign == 0.0f ? 0u : 0xffffffffu;
    x.x = (x.x ^ flip) & keep, x.y = (x.y ^ flip) & keep, x.z = (x.z ^ flip) & keep, x.w = (x.w ^ flip) & keep;
    *hi_out = __builtin_bit_cast(C8, x);
  }
}

// A weight is exp2(score - (maximum - kOffset)), the maximum being that of the last rescaling, which comes where it has grown by more
// than kGrow. fp16 has 2^-24 for its smallest step, and what a weight loses there the sum of the weights still has: with
// weights up to 1 a key 17.4 (natural units) above 16384 others took their 4.5e-4 of the result with it. With the largest one between 2^12
// and 2^14 a weight is off by 2^-37 of it, and fp16's range (2^16) still holds what the rounding of scores up to 10^7 adds. bf16 has the
// exponents of fp32.
template <int CT>
constexpr float kOffset = CT == Q4_F16 ? 12.0f : 0.0f;
template <int CT>
constexpr float kGrow = CT == Q4_F16 ? 2.0f : 8.0f;

// Eight softmax weights as the B operand of P V, in two terms of the cache's type that are multiplied one after the other: the weights
// rounded, and what that leaves. One term alone put the results of fp16 and bf16 activations 1.35 times as far from the exact ones
// as their own rounding does; two cost half of the matrix products more (prompts behind 4096 shared keys 190 -> 239 us in replayed graphs,
// 5 drafted tokens each of 48 sequences 53 -> 61, single tokens up to 3%). The second term is formed while the first one's products run.
template <int CT>
__device__ __forceinline__ vec8<CT> upper8(const float (&p)[8]) {
  typedef typename Num<CT>::type C2 __attribute__((ext_vector_type(2)));
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{p[2 * i], p[2 * i + 1]}), C2));
  return __builtin_bit_cast(vec8<CT>, make_uint4(w[0], w[1], w[2], w[3]));
}
template <int CT>
__device__ __forceinline__ vec8<CT> lower8(const float (&p)[8], vec8<CT> upper, float neg1) {
  const uint4 u4 = __builtin_bit_cast(uint4, upper);
  const uint32_t u[4] = {u4.x, u4.y, u4.z, u4.w};
  float left[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (CT == Q4_F16)
      left[i] = fmaf(static_cast<float>(upper[i]), neg1, p[i]);  // one instruction that reads the half as it is
    else
      left[i] = p[i] - __builtin_bit_cast(float, i & 1 ? u[i / 2] & 0xffff0000u : u[i / 2] << 16);
  }
  return upper8<CT>(left);
}

// N consecutive values of a range's o; or of the result, where it is the only range of the row.
template <int QT, int HD, int N>
__device__ __forceinline__ void store_o(const AttnArgs& a, const Item& it, const Row& w, int d, const float (&v)[N], float m,
                                        float l) {
  typedef typename Num<QT>::type Q;
  const int64_t row = static_cast<int64_t>(w.token) * a.n_q + w.head, shared = static_cast<int64_t>(a.T) * a.n_q * a.shared_splits;
  const int64_t first = shared + static_cast<int64_t>(it.slot0) * a.slot_rows + w.in_tile;
  if (a.own && d == 0 && !it.shared && it.part == 0) a.own[row] = make_int2(static_cast<int>(first - shared), it.ranges);
  if (!it.shared && it.ranges == 1 && a.shared_splits == 0) {
    const float inv = l > 0.0f ? 1.0f / l : l;  // no keys: zeros; NaN stays
    struct alignas(N * sizeof(Q) < 16 ? N * sizeof(Q) : 16) V {
      Q v[N];
    } y;
#pragma unroll
    for (int i = 0; i < N; ++i) y.v[i] = static_cast<Q>(v[i] * inv);
    *reinterpret_cast<V*>(static_cast<Q*>(a.out) + row * HD + d) = y;
  } else {
    const int64_t i = it.shared ? row * a.shared_splits + it.part : first + static_cast<int64_t>(it.part) * a.slot_rows;
#pragma unroll
    for (int j = 0; j < N; j += 4)
      *reinterpret_cast<f32x4*>(a.o + i * HD + d + j) = f32x4{v[j], v[j + 1], v[j + 2], v[j + 3]};
    if (d == 0) *reinterpret_cast<float2*>(a.ml + 2 * i) = make_float2(m, l);
  }
}

// Streaming form: 16 rows of one KV head, 32-key blocks dealt to the four waves, which keep (m, l, o) of their own and
// join them at the end. What bounds it is the latency and bandwidth of the key loads: 8 sequences of 1000 to 6000 keys of 16
// heads of 64 take 32 us, 3.6 TB/s (a large copy 5.1); two blocks a wave in flight instead of one spill or gain nothing.
//
// Per block and wave: S^T = K Q^T (16x16x32 MFMA; K straight from memory to the A operand: lane r16 + 16 quad holds key
// r16, dims 32 t + 8 quad ..), softmax per column (a lane holds 8 keys of one row, the other quads the rest), O^T +=
// V^T P^T. The S^T accumulators are the P^T operand as they stand: k slots 8 quad + j carry keys 4 quad + j and 16 +
// 4 quad + j - 4, and V^T comes from a row-major copy of the block in LDS in the same order by transposing reads.
// The loads of the next block are issued when this one's registers are free, and cross its softmax and PV.
template <int QT, int CT, int HD>
__device__ __forceinline__ void paged_stream(const AttnArgs& a, const Item& it, int entry, unsigned char* buf0,
                                             unsigned char* buf1, float2 (*wml)[64]) {
  typedef vec8<CT> C8;
  constexpr bool kSplit = QT == Q4_F32;      // q as two fp16 terms
  constexpr int KS = HD / 32, OT = HD / 16;  // MFMA steps over the dims; 16-dim output tiles
  constexpr int kRowB = HD * 2;
  constexpr int kCpr = HD / 8;               // 16-byte chunks per row
  constexpr int kVld = kKeys * kCpr / 64;    // V loads per lane
  constexpr int kRpi = 64 / kCpr;            // rows per load instruction
  constexpr int kBuf = 16 * HD * 4;          // LDS of a wave (two waves a buffer): a V block, then its rows of o
  static_assert(kBuf >= kKeys * kRowB && 2 * kBuf <= 2 * kStage * kRowB, "LDS of a wave");
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, quad = lane >> 4;
  auto buf_of = [&](int wv) { return (wv < 2 ? buf0 : buf1) + (wv & 1) * kBuf; };
  unsigned char* vb = buf_of(wave);

  const int k1 = it.k1;

  // Keys of a block: lane l (and l + 32) looks up key kb + l. The entry is loaded unconditionally, at the last key past the
  // end: chosen or copied behind the key loads, it would wait for them all.
  const int kl = lane & 31;
  auto page_entry = [&](int kb) { return page_at(a, it, min(kb + kl, k1 - 1)); };
  auto slot_of = [&](int entry, int kb) { return slot_at(a.b, entry, kb + kl, k1); };
  const uint32_t pitch = static_cast<uint32_t>(a.n_kv) * kRowB;
  const unsigned char* kbase = static_cast<const unsigned char*>(a.kc) + it.h * kRowB + 16 * quad;
  const unsigned char* vbase = static_cast<const unsigned char*>(a.vc) + it.h * kRowB + 16 * (lane % kCpr);
  u32x4 kr[2][KS], vr[kVld];
  auto load = [&](int slot) {  // keys without a row read row 0: their scores are masked, their values cleared
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int s = __shfl(slot, 16 * u + r16, 64);
      const unsigned char* p = row_at(kbase, s, pitch);
#pragma unroll
      for (int t = 0; t < KS; ++t) kr[u][t] = *reinterpret_cast<const u32x4*>(p + 64 * t);
    }
#pragma unroll
    for (int i = 0; i < kVld; ++i) {
      const int s = __shfl(slot, i * kRpi + lane / kCpr, 64);
      vr[i] = *reinterpret_cast<const u32x4*>(row_at(vbase, s, pitch));
    }
  };

  int kb = it.k0 + wave * kKeys;
  int slot = slot_of(entry, kb);
  if (kb < k1) {
    load(slot);
    entry = page_entry(kb + it.step);
  }

  // The rows, while the first keys are on their way.
  const Row w = row_of(a, it, it.row0 + r16);
  C8 qv[KS], ql[kSplit ? KS : 1];
#pragma unroll
  for (int t = 0; t < KS; ++t) load_q<QT, CT>(a, w, 32 * t + 8 * quad, &qv[t], &ql[kSplit ? t : 0]);
  int least = w.ok ? w.lim : INT32_MAX;  // the keys that every row sees
#pragma unroll
  for (int m = 8; m >= 1; m >>= 1) least = min(least, __shfl_xor(least, m, 64));
  least = __builtin_amdgcn_readfirstlane(least);

  f32x4 o[OT];
  float m = -INFINITY, l = 0.0f;  // m in log2 units; l: over this lane's keys
#pragma unroll
  for (int d = 0; d < OT; ++d) o[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  const float neg1 = minus_one();

  for (; kb < k1; kb += it.step) {
    // S^T: keys 16 u + 4 quad + i, row r16
    f32x4 s[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      s[u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      f32x4 lo = s[u];
#pragma unroll
      for (int t = 0; t < KS; ++t) {
        s[u] = mfma16(__builtin_bit_cast(C8, kr[u][t]), qv[t], s[u]);
        if constexpr (kSplit) lo = mfma16(__builtin_bit_cast(C8, kr[u][t]), ql[t], lo);
      }
      if constexpr (kSplit)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[u][i] += lo[i];
    }
    if constexpr (!kSplit) settle(s[0], s[1]);
    const uint32_t held = static_cast<uint32_t>(__ballot(slot >= 0));
#pragma unroll
    for (int i = 0; i < kVld; ++i) {
      const int r = i * kRpi + lane / kCpr, c = lane % kCpr;
      if (held != 0xffffffffu) vr[i] &= (held >> r) & 1 ? 0xffffffffu : 0u;
      *reinterpret_cast<u32x4*>(vb + r * kRowB + ((c ^ vswz<HD>(r)) << 4)) = vr[i];
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    slot = slot_of(entry, kb + it.step);
    if (kb + it.step < k1) load(slot);
    entry = page_entry(kb + 2 * it.step);
    if (held != 0xffffffffu || kb + kKeys > least) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int k = 16 * u + 4 * quad + i;
          if (kb + k >= w.lim || !((held >> k) & 1)) s[u][i] = -INFINITY;
        }
    }
    float mb = max3(max3(s[0][0], s[0][1], s[0][2]), max3(s[0][3], s[1][0], s[1][1]),
                    max3(s[1][2], s[1][3], s[1][3]));
    mb = swap_combine32<true>(swap_combine16<true>(mb)) * a.cs;
    if (__any(mb > m + kGrow<CT>)) {
      const float m_new = fmaxf(m, mb);
      const float alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - m_new);
      m = m_new;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < OT; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[d][i] *= alpha;
    }
    const float mu = m == -INFINITY ? 0.0f : m - kOffset<CT>;
    float p[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = __builtin_amdgcn_exp2f(fmaf(s[i >> 2][i & 3], a.cs, -mu));
#pragma unroll
    for (int i = 0; i < 8; ++i) l += p[i];
    const C8 ph = upper8<CT>(p), pl = lower8<CT>(p, ph, neg1);
#pragma unroll
    for (int d = 0; d < OT; ++d) {
      short4v v[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int r = 16 * u + 4 * quad + (r16 >> 2), c = 2 * d + ((r16 & 3) >> 1);
        v[u] = read_tr4(vb + r * kRowB + ((c ^ vswz<HD>(r)) << 4) + (r16 & 1) * 8);
      }
      const C8 va = __builtin_bit_cast(C8, __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7));
      o[d] = mfma16(va, ph, o[d]);
      o[d] = mfma16(va, pl, o[d]);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }

  // Join the four waves: (m, l) of each, then the weighted o.
  l = swap_combine32<false>(swap_combine16<false>(l));
  if (l != l && m == -INFINITY) m = 0.0f;  // every score was NaN: not a range without keys
  if (quad == 0) wml[wave][r16] = make_float2(m, l);
  __syncthreads();
  float* jb = reinterpret_cast<float*>(vb);  // rows of HD floats, their 16-byte chunks swizzled by the row
  float M = wml[0][r16].x;
#pragma unroll
  for (int v = 1; v < kWaves; ++v) M = fmaxf(M, wml[v][r16].x);
  const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - M);
  if (w.ok) {
#pragma unroll
    for (int d = 0; d < OT; ++d)
      *reinterpret_cast<f32x4*>(jb + r16 * HD + 4 * ((4 * d + quad) ^ r16)) =
          f32x4{f * o[d][0], f * o[d][1], f * o[d][2], f * o[d][3]};
  }
  __syncthreads();
  // thread: row r, dims 4 c ..; a row's place is that of lane r (all lanes take part in the shuffles: kC4 is 16 or 32)
  constexpr int kC4 = HD / 4;
  for (int e = threadIdx.x; e < 16 * kC4; e += kThreads) {
    const int r = e / kC4, c = e % kC4;
    Row y;
    y.token = __shfl(w.token, r, 64), y.head = __shfl(w.head, r, 64), y.in_tile = r;
    if (!__shfl(static_cast<int>(w.ok), r, 64)) continue;
    float mm = wml[0][r].x;
#pragma unroll
    for (int v = 1; v < kWaves; ++v) mm = fmaxf(mm, wml[v][r].x);
    float den = 0.0f;
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      const float2 z = wml[i][r];
      den += z.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(z.x - mm) * z.y;
      v += *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(buf_of(i)) + r * HD + 4 * (c ^ r));
    }
    const float y4[4] = {v[0], v[1], v[2], v[3]};
    store_o<QT, HD, 4>(a, it, y, 4 * c, y4, mm, den);
  }
}

// 16 bytes per lane from memory straight into LDS (lane i's at dst + 16 i).
__device__ __forceinline__ void load_lds16(const unsigned char* src, unsigned char* dst) {
  __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) void*)(src),
                                   (__attribute__((address_space(3))) void*)(dst), 16, 0, 0);
}

// Shared form: 32 RW rows of one KV head, 32 rows a wave; the waves share stages of 64 keys in LDS (two buffers, one
// barrier a stage). With RW == 2 the two halves of the workgroup take the two 32-key blocks of a stage and join at the
// end; with RW == 4 every wave takes both. What bounds it is the softmax between the two products of a block, which a wave
// runs one after the other, and the two workgroups that the registers leave a compute unit: prompts of 8 sequences behind 4096
// shared keys (32/8 heads of 128, bf16) take 235 us, 0.63 PFLOP/s, or 0.95 with the weights' second term
// (a large product 1.22), the matrix cores busy 44%.
//
// Per block and wave: S^T = K Q^T by 32x32x16 MFMA (lane: one row, half of the keys), softmax as above, O^T += V^T P^T with
// the accumulators of S^T as the operand: lane half h supplies keys 16 u + 8 (i / 4) + 4 h + i % 4, and the transposing
// reads of V follow the same order. Stage b + 1 goes straight to LDS while stage b is computed: a row may come from any
// page; those without a key read row 0 and have their values cleared in LDS before the stage is used (what lies
// there may be NaN, and a weight of zero does not undo that). The buffers are two LDS objects and the loop names them in turn, so
// that the compiler sees that reads of one do not touch the loads into the other and does not wait for them.
template <int QT, int CT, int HD, int RW>
__device__ __forceinline__ void paged_shared(const AttnArgs& a, const Item& it, int entry, unsigned char* buf0,
                                             unsigned char* buf1, float2 (*wml)[64]) {
  typedef vec8<CT> C8;
  constexpr bool kSplit = QT == Q4_F32;
  constexpr int KW = kWaves / RW;
  constexpr int KS = HD / 16, OT = HD / 32;       // MFMA steps over the dims; 32-dim output tiles
  constexpr int kRowB = HD * 2;
  constexpr int kCpr = HD / 8;
  constexpr int kHalf = kStage * kRowB;           // bytes of a stage's K (or V)
  constexpr int kRpi = 64 / kCpr;                 // rows per load instruction of a wave
  constexpr int kLd = kHalf / 1024 / kWaves;      // K (and V) load instructions per wave
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = lane >> 5, ql_ = lane & 31;
  const int rw = wave % RW, kw = wave / RW;

  // Stages: lane l of every wave looks up key kb + l. Load instruction wave + 4 j fills rows (wave + 4 j) kRpi ..; the lane for
  // chunk s of row r fetches chunk s ^ swz(r), the same for every j.
  const int k1 = it.k1;
  auto page_entry = [&](int kb) { return page_at(a, it, min(kb + lane, k1 - 1)); };
  auto slot_of = [&](int entry, int kb) { return slot_at(a.b, entry, kb + lane, k1); };
  const uint32_t pitch = static_cast<uint32_t>(a.n_kv) * kRowB;
  const int lr = wave * kRpi + lane / kCpr, lc = lane % kCpr;
  static_assert(kWaves * kRpi % 16 == 0, "one swizzle for all loads of a lane");
  const unsigned char* kbase = static_cast<const unsigned char*>(a.kc) + it.h * kRowB + ((lc ^ kswz<HD>(lr)) << 4);
  const unsigned char* vbase = static_cast<const unsigned char*>(a.vc) + it.h * kRowB + ((lc ^ vswz<HD>(lr)) << 4);
  auto issue = [&](unsigned char* buf, int slot) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < kLd; ++j) {
      const int s = __shfl(slot, j * kWaves * kRpi + lr, 64);
      unsigned char* dst = buf + (wave + j * kWaves) * 1024;
      load_lds16(row_at(kbase, s, pitch), dst);
      load_lds16(row_at(vbase, s, pitch), dst + kHalf);
    }
  };

  int slot = slot_of(entry, it.k0);
  if (it.k0 < k1) {
    issue(buf0, slot);
    entry = page_entry(it.k0 + it.step);
  }
  // The rows, while the first stage is on its way.
  const Row w = row_of(a, it, it.row0 + 32 * rw + ql_);
  int most = w.lim, least = w.ok ? w.lim : INT32_MAX;
#pragma unroll
  for (int m = 16; m >= 1; m >>= 1) {
    most = max(most, __shfl_xor(most, m, 64));
    least = min(least, __shfl_xor(least, m, 64));
  }
  most = __builtin_amdgcn_readfirstlane(most);
  least = __builtin_amdgcn_readfirstlane(least);
  C8 qv[KS], qlo[kSplit ? KS : 1];
#pragma unroll
  for (int t = 0; t < KS; ++t) load_q<QT, CT>(a, w, 16 * t + 8 * half, &qv[t], &qlo[kSplit ? t : 0]);

  f32x16 o[OT];
#pragma unroll
  for (int d = 0; d < OT; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[d][e] = 0.0f;
  float m = -INFINITY, l = 0.0f;
  const float neg1 = minus_one();
  const int kr4 = (lane & 15) >> 2;
  const int vrow = (4 * half + kr4) * kRowB + (lane & 1) * 8;
  int vcol[OT];
#pragma unroll
  for (int d = 0; d < OT; ++d) vcol[d] = vrow + (((4 * d + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ vswz<HD>(kr4)) << 4);

  // The block of 32 keys from row r0 of a stage on; kb: its first key. (Two blocks at a time, as far as the registers hold them: prompts
  // 240 instead of 238 us.)
  auto compute = [&](const unsigned char* buf, int r0, int kb, uint32_t held) __attribute__((always_inline)) {
    if (kb >= most) return;
    const unsigned char* Ks = buf + r0 * kRowB;
    const unsigned char* Vs = Ks + kHalf;
    C8 ka[KS];
#pragma unroll
    for (int t = 0; t < KS; ++t)
      ka[t] = *reinterpret_cast<const C8*>(Ks + ql_ * kRowB + (((2 * t + half) ^ kswz<HD>(ql_)) << 4));
    f32x16 s = {};
#pragma unroll
    for (int t = 0; t < KS; ++t) {
      if constexpr (kSplit) s = mfma32(ka[t], qlo[t], s);
      s = mfma32(ka[t], qv[t], s);
    }
    settle(s);
    if (held != 0xffffffffu || kb + 32 > least) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int k = 8 * (e >> 2) + 4 * half + (e & 3);
        if (kb + k >= w.lim || !((held >> k) & 1)) s[e] = -INFINITY;
      }
    }
    const float x = max3(max3(s[0], s[1], s[2]), s[3], s[4]);
    const float y = max3(max3(s[5], s[6], s[7]), s[8], s[9]);
    const float z = max3(max3(s[10], s[11], s[12]), max3(s[13], s[14], s[15]), -INFINITY);
    const float mb = swap_combine32<true>(max3(x, y, z)) * a.cs;
    if (__any(mb > m + kGrow<CT>)) {
      const float m_new = fmaxf(m, mb);
      const float alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - m_new);
      m = m_new;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < OT; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] *= alpha;
    }
    const float mu = m == -INFINITY ? 0.0f : m - kOffset<CT>;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      float p[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i] = __builtin_amdgcn_exp2f(fmaf(s[8 * u + i], a.cs, -mu));
      const C8 ph = upper8<CT>(p);
      C8 va[OT];
#pragma unroll
      for (int d = 0; d < OT; ++d) {
        const short4v v0 = read_tr4(Vs + vcol[d] + 16 * u * kRowB);
        const short4v v1 = read_tr4(Vs + vcol[d] + (16 * u + 8) * kRowB);
        va[d] = __builtin_bit_cast(C8, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
      }
#pragma unroll
      for (int d = 0; d < OT; ++d) o[d] = mfma32(va[d], ph, o[d]);
      const C8 pl = lower8<CT>(p, ph, neg1);
#pragma unroll
      for (int i = 0; i < 8; ++i) l += p[i];
#pragma unroll
      for (int d = 0; d < OT; ++d) o[d] = mfma32(va[d], pl, o[d]);
    }
  };

  // All loads of this wave have landed and its reads are done; then all waves'.
  auto turn = [&]() __attribute__((always_inline)) {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(7 << 4);  // vmcnt(0), lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  if (it.k0 < k1) {
    int kb = it.k0;
    uint64_t held = __ballot(slot >= 0);
    // one stage from `cur` while the next one goes to `nxt`; false: it was the last
    auto stage = [&](unsigned char* cur, unsigned char* nxt) __attribute__((always_inline)) {
      const uint64_t now = held;
      const bool more = kb + it.step < k1;
      if (now != ~uint64_t{0}) {
        for (int i = threadIdx.x; i < kStage * kCpr; i += kThreads)
          if (!((now >> (i / kCpr)) & 1)) reinterpret_cast<u32x4*>(cur + kHalf)[i] = u32x4{0, 0, 0, 0};
        turn();
      }
      slot = slot_of(entry, kb + it.step);
      if (more) issue(nxt, slot);
      entry = page_entry(kb + 2 * it.step);
      held = __ballot(slot >= 0);
      if constexpr (KW == 2) {
        compute(cur, 32 * kw, kb + 32 * kw, static_cast<uint32_t>(now >> (32 * kw)));
      } else {
        compute(cur, 0, kb, static_cast<uint32_t>(now));
        compute(cur, 32, kb + 32, static_cast<uint32_t>(now >> 32));
      }
      kb += it.step;
      turn();
      return more;
    };
    turn();
    while (stage(buf0, buf1) && stage(buf1, buf0)) {
    }
  }
  l = swap_combine32<false>(l);
  if (l != l && m == -INFINITY) m = 0.0f;
  if constexpr (KW == 2) {
    // the second half of the workgroup hands its rows over, register by register (the lanes hold the same places)
    float* jb = reinterpret_cast<float*>(buf0) + rw * OT * 16 * 64 + lane;
    if (kw == 1) {
      wml[rw][lane] = make_float2(m, l);
#pragma unroll
      for (int d = 0; d < OT; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) jb[(d * 16 + e) * 64] = o[d][e];
    }
    __syncthreads();
    if (kw == 1) return;
    const float2 x = wml[rw][lane];
    const float M = fmaxf(m, x.x);
    const float f0 = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - M);
    const float f1 = x.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(x.x - M);
    m = M;
    l = f0 * l + f1 * x.y;
#pragma unroll
    for (int d = 0; d < OT; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[d][e] = f0 * o[d][e] + f1 * jb[(d * 16 + e) * 64];
  }
#pragma unroll
  for (int d = 0; d < OT; ++d)
#pragma unroll
    for (int b = 0; b < 4; b += 2) {
      // dims 8 b + 4 half + i and 8 (b + 1) + 4 half + i of the tile -> lane half h gets all of 8 (b + h) ..
      float v[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = o[d][4 * b + i], y = o[d][4 * b + 4 + i];
        const auto t = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, y),
                                                        false, false);
        const unsigned lo = t[0], hi = t[1];  // (a bit cast of a vector element reads element 0 with this compiler)
        v[i] = __builtin_bit_cast(float, lo);
        v[4 + i] = __builtin_bit_cast(float, hi);
      }
      if (w.ok) store_o<QT, HD, 8>(a, it, w, 32 * d + 8 * (b + half), v, m, l);
    }
}

template <int QT, int CT, int HD>
__global__ __launch_bounds__(kThreads, 2) void paged_attn_kernel(AttnArgs a) {
  __shared__ __attribute__((aligned(16))) unsigned char buf0[2 * kStage * HD * 2], buf1[2 * kStage * HD * 2];
  __shared__ float2 wml[kWaves][64];
  int idx = blockIdx.x;
  Item it;
  it.shared = idx < a.shared_blocks;
  if (!it.shared) idx -= a.shared_blocks;
  int tile, height, split;
  it.seq = 0, it.tok0 = 0, it.own_end = 0, it.behind = 0, it.table = a.b.table, it.slot0 = 0;
  if (it.shared) {
    const int hs = a.by_kv.div(idx);
    it.h = idx - hs * a.n_kv;
    tile = a.by_shared.div(hs);
    split = hs - tile * a.shared_splits;
    it.ranges = a.shared_splits;
    height = a.shared_tile;
    it.n_rows = a.T * a.g;
  } else {
    Own w;
    if (!own_item(a, idx, &w)) return;
    it.h = __builtin_amdgcn_readfirstlane(w.h);
    it.seq = __builtin_amdgcn_readfirstlane(w.seq);
    it.ranges = w.ranges, it.slot0 = w.slot0;
    tile = __builtin_amdgcn_readfirstlane(w.tile);
    split = w.range;
    const int2 tk = tokens_of(a.b, it.seq, a.T);
    it.tok0 = tk.x;
    it.n_rows = tk.y * a.g;
    height = tile_rows(it.n_rows);
    it.table += it.seq * a.b.stride;
  }
  const bool stream = height == 16;
  const int turn = stream ? kTurn : kStage;
  it.row0 = tile * height;
  it.k0 = (it.shared ? 0 : a.own_from) + split * turn;
  const int first = it.k0 + (stream ? threadIdx.x >> 6 << 5 | (threadIdx.x & 31) : threadIdx.x & 63);
  const int entry = page_at(a, it, it.shared ? min(first, a.shared_len - 1) : max(first, 0));
  it.part = split;
  it.k1 = a.shared_len;
  if (!it.shared) {
    const int len = a.b.lens[it.seq], tokens = a.b.cu ? it.n_rows / a.g : a.b.rows;
    it.own_end = min(max(len, 0), a.held);
    it.behind = len - tokens;
    // no row of the tile sees more than its last
    const int last = a.by_g.div(min(it.row0 + height, it.n_rows) - 1);
    it.k1 = min(it.own_end, it.behind + last + 1);
    // no range without a block for every wave
    it.ranges = min(it.ranges, max((it.k1 - a.own_from + kTurn - 1) / kTurn, 1));
    if (split >= it.ranges) return;
  }
  it.step = it.ranges * turn;
  if (stream) return paged_stream<QT, CT, HD>(a, it, entry, buf0, buf1, wml);
  if (height == 64) paged_shared<QT, CT, HD, 2>(a, it, entry, buf0, buf1, wml);
  else paged_shared<QT, CT, HD, 4>(a, it, entry, buf0, buf1, wml);
}

// Joins the ranges of each row: PG threads, each for every PG-th range, and those side by side for 4 dims of the row; the first
// kB ranges of a thread are in flight at once. One launch and two dependent loads, 4 to 5 us, for a few rows; 6.6 us for the
// 20 MB of 7680 rows of 128 dims in four shared ranges and one own.
template <int QT, int HD, int PG>
__global__ __launch_bounds__(256) void paged_join_kernel(AttnArgs a) {
  typedef typename Num<QT>::type Q;
  constexpr int kC4 = HD / 4, kB = 4, kRow = kC4 * PG, kRowsWg = 256 / kRow;
  __shared__ float sm[kRowsWg][PG][kC4], sd[kRowsWg][PG][kC4];
  __shared__ f32x4 so[kRowsWg][PG][kC4];
  const int lr = threadIdx.x / kRow, pg = threadIdx.x % kRow / kC4, c = threadIdx.x % kC4;
  const int64_t rows = static_cast<int64_t>(a.T) * a.n_q, row = static_cast<int64_t>(blockIdx.x) * kRowsWg + lr;
  bool ok = row < rows;
  if (a.b.cu) {
    const int64_t t = row / a.n_q;
    ok = ok && t >= a.b.cu[0] && t < a.b.cu[a.b.batch];  // else of no sequence
  }
  int2 own = make_int2(0, 0);
  if (ok && a.L > a.own_from) own = a.own[row];
  if (a.shared_splits == 0 && own.y == 1) ok = false;  // its one range has written the result
  // (where cu_q does not ascend, a row may have no range, and `own` anything)
  if (own.x < 0 || own.y < 0 || own.y > kMaxSplits || own.x >= a.own_rows - (own.y - 1) * a.slot_rows) own.y = 0;
  const int parts = a.shared_splits + own.y;
  auto place = [&](int p) {
    return p < a.shared_splits ? row * a.shared_splits + p
                               : rows * a.shared_splits + own.x + static_cast<int64_t>(p - a.shared_splits) * a.slot_rows;
  };
  const float2* ml = reinterpret_cast<const float2*>(a.ml);
  float M = -INFINITY, den = 0.0f;
  f32x4 num = {0.0f, 0.0f, 0.0f, 0.0f};
  if (ok)
    for (int p0 = pg; p0 < parts; p0 += kB * PG) {
      float2 x[kB];
      f32x4 v[kB];
#pragma unroll
      for (int i = 0; i < kB; ++i) {
        x[i] = make_float2(-INFINITY, 0.0f);
        if (p0 + i * PG < parts) {
          const int64_t at = place(p0 + i * PG);
          x[i] = ml[at];
          v[i] = *reinterpret_cast<const f32x4*>(a.o + at * HD + 4 * c);
        }
      }
      float mb = M;
#pragma unroll
      for (int i = 0; i < kB; ++i) mb = fmaxf(mb, x[i].x);
      const float alpha = M == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(M - mb);
      M = mb;
      den *= alpha;
      num *= alpha;
#pragma unroll
      for (int i = 0; i < kB; ++i)
        if (x[i].x != -INFINITY) {
          const float w = __builtin_amdgcn_exp2f(x[i].x - M);
          den = fmaf(w, x[i].y, den);
#pragma unroll
          for (int j = 0; j < 4; ++j) num[j] = fmaf(w, v[i][j], num[j]);
        }
    }
  if constexpr (PG > 1) {
    sm[lr][pg][c] = M;
    sd[lr][pg][c] = den;
    so[lr][pg][c] = num;
    __syncthreads();
    if (pg != 0) return;
    float all = M;
#pragma unroll
    for (int i = 1; i < PG; ++i) all = fmaxf(all, sm[lr][i][c]);
    den = 0.0f;
    num = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < PG; ++i) {
      const float m = sm[lr][i][c];
      const float w = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - all);
      den = fmaf(w, sd[lr][i][c], den);
      const f32x4 v = so[lr][i][c];
#pragma unroll
      for (int j = 0; j < 4; ++j) num[j] = fmaf(w, v[j], num[j]);
    }
  }
  if (!ok) return;
  const float inv = den > 0.0f ? 1.0f / den : den;
  struct alignas(4 * sizeof(Q)) Q4v {
    Q v[4];
  };
  Q4v y;
#pragma unroll
  for (int j = 0; j < 4; ++j) y.v[j] = static_cast<Q>(num[j] * inv);
  *reinterpret_cast<Q4v*>(static_cast<Q*>(a.out) + row * HD + 4 * c) = y;
}

struct Plan {
  int64_t shared_blocks, own_blocks;  // workgroups (own: an upper bound)
  int64_t partials;                   // results of ranges that the workspace holds (0: none is needed)
  int shared_tile, shared_splits, own_from, slot_rows;
  int places, own_whole, own_items, own_ranges, own_most, own_tiles;  // (without cu_q) tiles of a sequence
  int most;                                                    // ranges of a row at most
  int turn_from;  // the second ones: tiles from here on
  bool longest_first, refill;
};

Plan plan_for(int64_t T, int n_q, int n_kv, int batch, bool ragged, int L, int shared_len) {
  Plan p{};
  if (T == 0) return p;
  const int g = n_q / n_kv;
  const int64_t rows = T * g;
  // The shared keys are a range of their own where that saves reading them once for each sequence: not for one sequence, not
  // for a few keys (they cost their ranges' partial results and join), and not where a sequence's rows alone fill tiles
  // (prompts), which then read them as often either way and join less. One token each of 2 / 8 / 32 sequences, 32/8
  // heads of 128, 200 own keys, apart and not: 256 shared keys 9.2 / 11.6 / 15.8 and 10.1 / 10.0 / 12.2 us, 1024 keys
  // 9.3 / 12.1 / 16.9 and 10.8 / 15.8 / 22.5, 16384 keys 19.0 / 22.3 / 34.3 and 25.1 / 49.5 / 158; 100 tokens each of 8 behind
  // 4096 131 and 107.
  const bool apart = shared_len >= 4 * kTurn && batch > 1 && rows / batch < 128;
  p.own_from = apart ? shared_len : 0;
  if (apart) {
    // One workgroup for every compute unit: the other place of each is left to own ranges, and what ranges write and the join
    // reads stays small (of 48 x 5 tokens x 32 heads and 4096 shared keys, 17 MB; with two 70 us, with one 57).
    p.shared_tile = tile_rows(rows);
    const int64_t items = n_kv * static_cast<int64_t>(tiles_of(rows));
    p.shared_splits = static_cast<int>(std::max<int64_t>(
        1, std::min<int64_t>({kSlots / 2 / items, (shared_len + kTurn - 1) / kTurn, kMaxSplits})));
    p.shared_blocks = items * p.shared_splits;
  }
  p.places = kSlots - static_cast<int>(std::min<int64_t>(p.shared_blocks, kSlots / 2));  // what shared ranges leave
  if (const int64_t keys = L - p.own_from; keys > 0) {
    // (with cu_q, which only the device reads, these go by the mean of the rows and by one tile for each sequence)
    p.refill = rows / batch <= 32 && keys >= 2048;
    p.own_tiles = ragged ? 1 : tiles_of(rows / batch);
    const int64_t items = static_cast<int64_t>(batch) * p.own_tiles * n_kv;
    // Short keys are one range, which needs no join: up to two blocks a wave always, up to four where there are items for a
    // quarter of the units. One token each of 1 / 4 / 12 / 32 sequences, 8 KV heads of 128, one range and as many as fit:
    // 250 keys 7.9 / 8.1 / 8.6 / 10.2 and 10.1 / 10.1 / 10.7 / 13.3 us, 400 keys 9.7 / 10.2 / 11.0 / 13.6 and 10.2 / 10.2 /
    // 12.8 / 16.9.
    const bool one = !apart && keys <= (items >= kSlots / 8 ? 4 : 2) * kTurn;
    p.own_most = one ? 1 : static_cast<int>(std::min<int64_t>((keys + kTurn - 1) / kTurn, kMaxSplits));
    if (ragged) {
      // the number of tiles, and so of ranges, is known on the device alone; at most one tile that is not full a sequence, and
      // a full one has 128 rows
      const int64_t most = (rows / 128 + batch) * n_kv, fill = p.refill ? 2 * p.places : p.places;  // items; what ranges fill
      p.own_blocks = std::max(most, (most < kSlots ? 0 : most) + fill);  // (fewer than kSlots: none is whole)
      p.slot_rows = tile_rows(rows);
    } else {
      const int64_t rest = items % kSlots;
      p.own_ranges = rest ? ranges_of(static_cast<int>(rest), p.places, p.refill, p.own_most, static_cast<int>(keys)) : 1;
      p.own_items = static_cast<int>(items), p.own_whole = static_cast<int>(items - rest);
      p.own_blocks = items - rest + rest * p.own_ranges;
      p.own_most = p.own_ranges;
      p.slot_rows = tile_rows(rows / batch);
    }
    // One token each of 8 / 16 / 28 sequences of 1000 to 6000 keys, 16 heads of 64, the second ones longest first too and
    // shortest first: 34.6 / 60.9 / 99 and 31.5 / 53.3 / 85 us. Up to three tokens each, 8 KV heads of 128, in the batch's order
    // and so: 34.9 / 61.7 / 108 and 33.0 / 53.8 / 88.
    p.longest_first = batch > 1 && batch <= 64 && keys > 4 * kTurn;
    p.turn_from = INT32_MAX;
    if (!apart && !ragged && p.own_blocks <= kSlots) p.turn_from = (kSlots / 2 + n_kv * p.own_ranges - 1) / (n_kv * p.own_ranges);
  }
  p.most = p.shared_splits + p.own_most;
  if (apart) p.most = std::max(p.most, 2);  // shared ranges are joined also where a row has one range in all (L == shared_len)
  if (p.most > 1)
    p.partials = T * n_q * p.shared_splits +
                 p.slot_rows * (apart ? p.own_blocks : std::min<int64_t>(p.own_blocks, p.refill ? 2 * kSlots : kSlots));
  return p;
}

size_t ml_floats(size_t n) { return (2 * n + 3) / 4 * 4; }
size_t workspace_of(const Plan& p, int64_t rows, int hd) {
  const size_t n = static_cast<size_t>(p.partials);
  return n ? (ml_floats(n) + n * hd) * sizeof(float) + rows * sizeof(int2) : 0;
}

int attn_args(int64_t T, int n_q, int n_kv, int hd, int batch, int L, int shared_len) {
  if (T < 0 || T > INT32_MAX || n_q <= 0 || n_kv <= 0 || batch <= 0 || L <= 0 || shared_len < 0 || shared_len > L)
    return Q4_ERR_SHAPE;
  if (L > kMaxKeys) return Q4_ERR_RANGE;
  // row numbers of the last tile, and offsets in a token's heads, stay below 2^31
  if (n_q % n_kv || T * n_q > INT32_MAX - 128 || n_q > INT32_MAX / 2048) return Q4_ERR_SHAPE;
  if (hd != 64 && hd != 128) return Q4_ERR_UNSUPPORTED;
  if (n_q / n_kv > 64) return Q4_ERR_UNSUPPORTED;
  return Q4_OK;
}

template <int QT, int CT, int HD>
int launch(const AttnArgs& a, int64_t blocks, int most, hipStream_t st) {
  const int64_t rows = static_cast<int64_t>(a.T) * a.n_q;
  const int pg = most <= 4 || rows >= 16384 ? 1 : most <= 16 ? 4 : 8, per = 256 / (HD / 4 * pg);
  if (!fits_grid(blocks, kThreads) || (most > 1 && !fits_grid((rows + per - 1) / per, 256))) return Q4_ERR_SHAPE;
  if (blocks > 0)
    hipLaunchKernelGGL((paged_attn_kernel<QT, CT, HD>), dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, st, a);
  if (most > 1) {
    // (pg) a few ranges a thread, so that a row is one round trip; a thread a row where there are rows enough to fill the chip.
    // With 1 / 4 / 8: one sequence of 700 keys 11.0 / 10.3 / 9.6 us, of 16000 29.5 / 20.8 / 19.4, 7680 rows of 5 ranges
    // 57 / 57 / 59, 65000 rows of 2 to 4 ranges 234 / 244 / 257.
    const auto fn = pg == 1 ? paged_join_kernel<QT, HD, 1> : pg == 4 ? paged_join_kernel<QT, HD, 4> : paged_join_kernel<QT, HD, 8>;
    hipLaunchKernelGGL(fn, dim3(static_cast<unsigned>((rows + per - 1) / per)), dim3(256), 0, st, a);
  }
  return launch_status();
}

}  // namespace
}  // namespace q4

using namespace q4;

extern "C" int paged_attn_workspace_bytes_for(int64_t T, int n_q, int n_kv, int head_dim, int batch, int L, int shared_len,
                                              int has_cu_q, size_t* bytes) {
  if (!bytes) return Q4_ERR_NULL;
  if (int st = attn_args(T, n_q, n_kv, head_dim, batch, L, shared_len)) return st;
  if (!has_cu_q && T % batch) return Q4_ERR_SHAPE;
  *bytes = workspace_of(plan_for(T, n_q, n_kv, batch, has_cu_q != 0, L, shared_len), T * n_q, head_dim);
  return Q4_OK;
}

extern "C" int paged_attn_workspace_bytes(int64_t T, int n_q, int n_kv, int head_dim, int batch, int L, int shared_len,
                                          size_t* bytes) {
  if (int st = paged_attn_workspace_bytes_for(T, n_q, n_kv, head_dim, batch, L, shared_len, 1, bytes)) return st;
  size_t even = 0;
  if (T % batch == 0) paged_attn_workspace_bytes_for(T, n_q, n_kv, head_dim, batch, L, shared_len, 0, &even);
  *bytes = std::max(*bytes, even);
  return Q4_OK;
}

extern "C" int paged_attn(const q4_paged_kv* kv, const void* q, int64_t q_row, int64_t q_head, void* out, int dtype, int64_t T,
                          int n_q, int L, const int32_t* shared_pages, int shared_len, float scale, void* workspace,
                          size_t workspace_bytes, void* stream) {
  if (!q || !out || (shared_len > 0 && !shared_pages)) return Q4_ERR_NULL;
  AttnArgs a{};
  if (int st = paged_batch(kv, dtype, T, &a.b)) return st;
  const int hd = kv->head_dim;
  if (int st = attn_args(T, n_q, kv->n_kv, hd, kv->batch, L, shared_len)) return st;
  if (shared_len > kv->num_pages * kv->page_size || !std::isfinite(scale)) return Q4_ERR_RANGE;
  const int e = dtype == Q4_F32 ? 4 : 8;
  if (q_row < 0 || q_head < 0 || q_row % e || q_head % e) return Q4_ERR_SHAPE;
  if (!aligned(q, 16) || !aligned(out, 16) || !aligned(kv->k_cache, 16) || !aligned(kv->v_cache, 16) ||
      !aligned(shared_pages, 4))
    return Q4_ERR_ALIGN;
  if (T == 0) return Q4_OK;
  const int g = n_q / kv->n_kv;
  const Plan p = plan_for(T, n_q, kv->n_kv, kv->batch, kv->cu_q != nullptr, L, shared_len);
  if (p.partials) {
    if (!workspace || workspace_bytes < workspace_of(p, T * n_q, hd)) return Q4_ERR_WORKSPACE;
    if (!aligned(workspace, 16)) return Q4_ERR_ALIGN;
  }
  const int64_t blocks = p.shared_blocks + p.own_blocks;
  if (p.partials > INT32_MAX) return Q4_ERR_SHAPE;
  a.q = q, a.qr = q_row, a.qh = q_head;
  a.kc = kv->k_cache, a.vc = kv->v_cache, a.out = out;
  if (p.partials) {
    a.ml = static_cast<float*>(workspace);
    a.o = a.ml + ml_floats(p.partials);
    a.own = reinterpret_cast<int2*>(a.o + p.partials * hd);
    a.own_rows = static_cast<int>(p.partials - T * n_q * p.shared_splits);
  }
  a.shared_pages = shared_pages;
  a.T = static_cast<int>(T), a.n_q = n_q, a.n_kv = kv->n_kv, a.g = g, a.L = L, a.shared_len = shared_len;
  a.shared_blocks = static_cast<int>(p.shared_blocks), a.shared_splits = p.shared_splits, a.shared_tile = p.shared_tile;
  a.held = static_cast<int>(std::min<int64_t>(std::max<int64_t>(int64_t{kv->max_pages} * kv->page_size, shared_len), L));
  a.own_from = p.own_from, a.slot_rows = p.slot_rows;
  a.longest_first = p.longest_first, a.refill = p.refill, a.turn_from = p.turn_from;
  // a negative scale turns q around and a zero one clears it, so that the exponents' factor is positive
  a.sign = scale < 0.0f ? -1.0f : scale == 0.0f ? 0.0f : 1.0f;
  a.cs = scale == 0.0f ? 1.0f : std::fabs(scale) * 1.44269504088896340736f;
  a.by_g = FastDiv(g), a.by_kv = FastDiv(kv->n_kv);
  a.own_whole = p.own_whole, a.own_items = p.own_items, a.own_most = p.own_most, a.places = p.places;
  a.by_shared = FastDiv(std::max(p.shared_splits, 1)), a.by_ranges = FastDiv(std::max(p.own_ranges, 1));
  a.by_tiles = FastDiv(std::max(p.own_tiles, 1));
  const hipStream_t st = as_stream(stream);
  const auto fn = dtype == Q4_F32    ? (hd == 128 ? launch<Q4_F32, Q4_F16, 128> : launch<Q4_F32, Q4_F16, 64>)
                  : dtype == Q4_F16  ? (hd == 128 ? launch<Q4_F16, Q4_F16, 128> : launch<Q4_F16, Q4_F16, 64>)
                                     : (hd == 128 ? launch<Q4_BF16, Q4_BF16, 128> : launch<Q4_BF16, Q4_BF16, 64>);
  return fn(a, blocks, p.most, st);
}
