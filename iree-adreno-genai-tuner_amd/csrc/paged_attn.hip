// Causal GQA attention over a paged KV cache with a prefix that the whole batch shares (paged_attn).
//
// For the token at position p of a sequence and query head h (KV head h / g): o = sum_j softmax_j(scale q . k_j) v_j over
// its keys j <= p. Any split of the keys into ranges gives the same result: a range yields m = max s, l = sum
// exp(s - m), o = sum exp(s - m) v, and ranges join as M = max m, o = sum e^(m - M) o / sum e^(m - M) l. So the shared keys
// are one range for all tokens of the batch, whose rows (token, head of the group) are stacked: their K and V are
// read once per 16 rows instead of once per sequence. The keys of a sequence's own are a second kind of range.
// Both run in one launch; a second joins the ranges of each row where there are several.
#include "q4_common.h"
#include "q4_paged.h"

#include <algorithm>
#include <cmath>

namespace q4 {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kRows = 16;  // rows (token, query head of the group) of a workgroup
constexpr int kKeys = 32;  // keys of a wave's block

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short short4v __attribute__((ext_vector_type(4)));
template <int CT>
using vec8 = typename Num<CT>::type __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x4 mfma16(vec8<Q4_F16> a, vec8<Q4_F16> b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(vec8<Q4_BF16> a, vec8<Q4_BF16> b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
// Transposing LDS read: the lanes of each 16 read a 4 x 16 block of 16-bit values (lane i: row i / 4, columns
// 4 (i % 4) ..) and lane i receives column i.
__device__ __forceinline__ short4v read_tr4(void* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)p);
}

struct AttnArgs {
  PagedBatch b;
  const void* q;
  int64_t qr, qh;
  const void *kc, *vc;
  void* out;
  float *ml, *o;  // ranges' (m, l) and o of each row: [T * n_q][parts]
  const int32_t* shared_pages;
  int T, n_q, n_kv, g, L, shared_len;
  int shared_blocks, shared_splits, shared_keys;  // workgroups of the shared ranges, ranges, keys of a range
  int own_splits, parts;
  float cs, sign;  // exponents are s * cs in log2 units; sign: that of the scale, taken into q
  FastDiv by_g, by_kv, by_shared, by_own;
};

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

// The sequence and, within it, the row tile of own tile `tile` (wave-uniform); false: past the last.
__device__ __forceinline__ bool own_tile(const AttnArgs& a, int tile, int* seq, int* in_seq) {
  if (!a.b.cu) {
    const int per = (a.b.rows * a.g + kRows - 1) / kRows;
    *seq = tile / per;
    *in_seq = tile - *seq * per;
    return *seq < a.b.batch;
  }
  const int lane = threadIdx.x & 63;
  int base = 0;
  for (int i = 0; i < a.b.batch; i += 64) {
    const int s = min(i + lane, a.b.batch - 1);
    const int n = i + lane < a.b.batch ? (tokens_of(a.b, s, a.T).y * a.g + kRows - 1) / kRows : 0;
    int run = n;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const int o = __shfl_up(run, m, 64);
      if (lane >= m) run += o;
    }
    const uint64_t past = __ballot(base + run > tile);
    if (past) {
      const int l = __builtin_ctzll(past);
      *seq = i + l;
      *in_seq = tile - base - (__builtin_amdgcn_readlane(run, l) - __builtin_amdgcn_readlane(n, l));
      return true;
    }
    base += __builtin_amdgcn_readlane(run, 63);
  }
  return false;
}

// V's 16-byte chunks of a row in LDS, swizzled so that the four rows of a transposing read fall in different banks.
template <int HD>
__device__ __forceinline__ int vswz(int r) {
  return HD == 128 ? (r & 3) << 2 : ((r >> 1) & 1) << 2;
}

// Workgroup: 16 rows of one KV head against one range of keys, 32-key blocks dealt to its four waves, which keep
// (m, l, o) of their own and join them at the end.
//
// Per block and wave: S^T = K Q^T (16x16x32 MFMA; K straight from memory to the A operand: lane r16 + 16 quad holds key
// r16, dims 32 t + 8 quad ..), softmax per column (a lane holds 8 keys of one row, the other quads the rest), O^T +=
// V^T P^T. The S^T accumulators are the P^T operand as they stand: k slots 8 quad + j carry keys 4 quad + j and 16 +
// 4 quad + j - 4, and V^T comes from a row-major copy of the block in LDS in the same order by transposing reads.
// The loads of the next block are issued when this one's registers are free, and cross its softmax and PV.
template <int QT, int CT, int HD>
__global__ __launch_bounds__(kThreads, 2) void paged_attn_kernel(AttnArgs a) {
  typedef typename Num<QT>::type Q;
  typedef typename Num<CT>::type C;
  typedef vec8<CT> C8;
  constexpr bool kSplit = QT == Q4_F32;     // q and P as two fp16 terms
  constexpr int KS = HD / 32, OT = HD / 16;  // MFMA steps over the dims; 16-dim output tiles
  constexpr int kRowB = HD * 2;
  constexpr int kCpr = HD / 8;               // 16-byte chunks per row
  constexpr int kVld = kKeys * kCpr / 64;    // V loads per lane
  constexpr int kRpi = 64 / kCpr;            // rows per load instruction
  constexpr int kPitch = HD + 4;             // floats per row of the join buffer
  constexpr int kBuf = std::max(kKeys * kRowB, kRows * kPitch * 4);
  __shared__ __attribute__((aligned(16))) unsigned char buf[kWaves][kBuf];
  __shared__ float2 wml[kWaves][kRows];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, quad = lane >> 4;

  // What this workgroup does: rows and keys.
  int idx = blockIdx.x;
  const bool shared = idx < a.shared_blocks;
  if (!shared) idx -= a.shared_blocks;
  const int hs = a.by_kv.div(idx), h = idx - hs * a.n_kv;
  const FastDiv by_split = shared ? a.by_shared : a.by_own;
  int tile = by_split.div(hs);
  const int split = hs - tile * static_cast<int>(by_split.d);
  int seq = 0, token, lim = 0, row_g, k0, k1;
  bool row_ok;
  if (shared) {
    const int r = tile * kRows + r16;
    token = a.by_g.div(r);
    row_g = r - token * a.g;
    row_ok = token < a.T;
    const int s = sequence_of_lane(a.b, row_ok ? token : 0);
    row_ok = row_ok && s < a.b.batch;
    if (row_ok) {
      const int2 tk = tokens_of(a.b, s, a.T);
      row_ok = token >= tk.x && token < tk.x + tk.y;
      lim = min(min(a.b.lens[s] - tk.y + (token - tk.x) + 1, a.b.keys(s)), a.shared_len);
    }
    k0 = split * a.shared_keys;
    k1 = min(k0 + a.shared_keys, a.shared_len);
  } else {
    if (!own_tile(a, tile, &seq, &tile)) return;
    seq = __builtin_amdgcn_readfirstlane(seq);
    const int2 tk = tokens_of(a.b, seq, a.T);
    const int r = tile * kRows + r16;
    const int i = a.by_g.div(r);
    row_g = r - i * a.g;
    token = tk.x + i;
    row_ok = i < tk.y;
    const int end = min(a.b.keys(seq), a.L);
    lim = min(a.b.lens[seq] - tk.y + i + 1, end);
    const int n = max(end - a.shared_len, 0);
    const int per = ((n + a.own_splits - 1) / a.own_splits + kKeys - 1) / kKeys * kKeys;
    k0 = a.shared_len + min(split * per, n);
    k1 = min(k0 + per, end);
  }
  if (!row_ok) lim = 0;
  // the last key any row sees, and the first block that some row does not see whole
  int most = lim, least = row_ok ? lim : INT32_MAX;
#pragma unroll
  for (int m = 8; m >= 1; m >>= 1) {
    most = max(most, __shfl_xor(most, m, 64));
    least = min(least, __shfl_xor(least, m, 64));
  }
  k1 = __builtin_amdgcn_readfirstlane(min(k1, most));
  least = __builtin_amdgcn_readfirstlane(least);
  const int head = h * a.g + row_g;

  // Q^T operand: column r16, dims 32 t + 8 quad ..
  C8 qv[KS], ql[kSplit ? KS : 1];
  {
    const Q* qp = static_cast<const Q*>(a.q) + token * a.qr + head * a.qh + 8 * quad;
    const float neg1 = minus_one();
#pragma unroll
    for (int t = 0; t < KS; ++t) {
      if constexpr (kSplit) {
        f32x4 x = {}, y = {};
        if (row_ok) {
          x = *reinterpret_cast<const f32x4*>(qp + 32 * t);
          y = *reinterpret_cast<const f32x4*>(qp + 32 * t + 4);
        }
        uint32_t hi[4], lo[4];
        split_f16_pair(a.sign * x.x, a.sign * x.y, neg1, hi[0], lo[0]);
        split_f16_pair(a.sign * x.z, a.sign * x.w, neg1, hi[1], lo[1]);
        split_f16_pair(a.sign * y.x, a.sign * y.y, neg1, hi[2], lo[2]);
        split_f16_pair(a.sign * y.z, a.sign * y.w, neg1, hi[3], lo[3]);
        qv[t] = __builtin_bit_cast(C8, make_uint4(hi[0], hi[1], hi[2], hi[3]));
        ql[t] = __builtin_bit_cast(C8, make_uint4(lo[0], lo[1], lo[2], lo[3]));
      } else {
        uint4 x = make_uint4(0, 0, 0, 0);
        if (row_ok) x = *reinterpret_cast<const uint4*>(qp + 32 * t);
        const uint32_t flip = a.sign < 0.0f ? 0x80008000u : 0u, keep = a.sign == 0.0f ? 0u : 0xffffffffu;
        x.x = (x.x ^ flip) & keep, x.y = (x.y ^ flip) & keep, x.z = (x.z ^ flip) & keep, x.w = (x.w ^ flip) & keep;
        qv[t] = __builtin_bit_cast(C8, x);
      }
    }
  }

  // Keys of a block: lane l (and l + 32) looks up key kb + l.
  const int32_t* pages = shared ? a.shared_pages : a.b.table + seq * a.b.stride;
  const int kl = lane & 31;
  auto page_entry = [&](int kb) {
    const int j = kb + kl;
    return j < k1 ? pages[a.b.by_page.div(j)] : -1;
  };
  auto slot_of = [&](int entry, int kb) {
    const int j = kb + kl;
    return j < k1 ? a.b.slot(entry, j - a.b.by_page.div(j) * a.b.page_size) : -1;
  };
  const int64_t pitch = static_cast<int64_t>(a.n_kv) * kRowB;
  const unsigned char* kbase = static_cast<const unsigned char*>(a.kc) + h * kRowB + 16 * quad;
  const unsigned char* vbase = static_cast<const unsigned char*>(a.vc) + h * kRowB + 16 * (lane % kCpr);
  uint4 kr[2][KS], vr[kVld];
  auto load = [&](int slot) {  // keys without a row read row 0: their scores are masked, their values cleared
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int s = __shfl(slot, 16 * u + r16, 64);
      const unsigned char* p = kbase + max(s, 0) * pitch;
#pragma unroll
      for (int t = 0; t < KS; ++t) kr[u][t] = *reinterpret_cast<const uint4*>(p + 64 * t);
    }
#pragma unroll
    for (int i = 0; i < kVld; ++i) {
      const int s = __shfl(slot, i * kRpi + lane / kCpr, 64);
      vr[i] = *reinterpret_cast<const uint4*>(vbase + max(s, 0) * pitch);
    }
  };

  f32x4 o[OT];
#pragma unroll
  for (int d = 0; d < OT; ++d) o[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float m = -INFINITY, l = 0.0f;  // m in log2 units; l: over this lane's keys
  unsigned char* vb = buf[wave];
  const float neg1 = minus_one();

  constexpr int kStep = kWaves * kKeys;
  int kb = k0 + wave * kKeys;
  int slot = -1, entry = -1;
  if (kb < k1) {
    slot = slot_of(page_entry(kb), kb);
    load(slot);
    entry = page_entry(kb + kStep);
  }
  for (; kb < k1; kb += kStep) {
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
    const uint32_t held = static_cast<uint32_t>(__ballot(slot >= 0));
#pragma unroll
    for (int i = 0; i < kVld; ++i) {
      const int r = i * kRpi + lane / kCpr, c = lane % kCpr;
      if (held != 0xffffffffu && !((held >> r) & 1)) vr[i] = make_uint4(0, 0, 0, 0);
      *reinterpret_cast<uint4*>(vb + r * kRowB + ((c ^ vswz<HD>(r)) << 4)) = vr[i];
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (kb + kStep < k1) {
      slot = slot_of(entry, kb + kStep);
      load(slot);
      entry = page_entry(kb + 2 * kStep);
    }
    if (held != 0xffffffffu || kb + kKeys > least) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int k = 16 * u + 4 * quad + i;
          if (kb + k >= lim || !((held >> k) & 1)) s[u][i] = -INFINITY;
        }
    }
    float mb = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                     fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
    mb = swap_combine32<true>(swap_combine16<true>(mb)) * a.cs;
    // the sums are rescaled only where a maximum has grown by more than 2^8: weights stay below that
    if (__any(mb > m + 8.0f)) {
      const float m_new = fmaxf(m, mb);
      const float alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - m_new);
      m = m_new;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < OT; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[d][i] *= alpha;
    }
    const float mu = m == -INFINITY ? 0.0f : m;
    float p[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = __builtin_amdgcn_exp2f(fmaf(s[i >> 2][i & 3], a.cs, -mu));
    C8 ph, pl;
    if constexpr (kSplit) {
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) split_f16_pair(p[2 * i], p[2 * i + 1], neg1, hi[i], lo[i]);
      ph = __builtin_bit_cast(C8, make_uint4(hi[0], hi[1], hi[2], hi[3]));
      pl = __builtin_bit_cast(C8, make_uint4(lo[0], lo[1], lo[2], lo[3]));
#pragma unroll
      for (int i = 0; i < 8; ++i) l += p[i];
    } else {
      // weights rounded to the cache's type; the sum is that of the rounded ones, so that a row's weights add to 1
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        ph[i] = static_cast<C>(p[i]);
        l += static_cast<float>(ph[i]);
      }
    }
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
      if constexpr (kSplit) o[d] = mfma16(va, pl, o[d]);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }

  // Join the four waves: (m, l) of each, then the weighted o.
  l = swap_combine32<false>(swap_combine16<false>(l));
  if (l != l && m == -INFINITY) m = 0.0f;  // every score was NaN: not a range without keys
  if (quad == 0) wml[wave][r16] = make_float2(m, l);
  __syncthreads();
  float M = wml[0][r16].x;
#pragma unroll
  for (int w = 1; w < kWaves; ++w) M = fmaxf(M, wml[w][r16].x);
  const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - M);
  float* jb = reinterpret_cast<float*>(buf[wave]);
  if (row_ok) {
#pragma unroll
    for (int d = 0; d < OT; ++d)
      *reinterpret_cast<f32x4*>(jb + r16 * kPitch + 16 * d + 4 * quad) =
          f32x4{f * o[d][0], f * o[d][1], f * o[d][2], f * o[d][3]};
  }
  __syncthreads();
  // thread: row r, dims 4 c ..; a row's token and head are those of lane r
  constexpr int kC4 = HD / 4;
  const int part = shared ? split : a.shared_splits + split;
  for (int e = threadIdx.x; e < kRows * kC4; e += kThreads) {
    const int r = e / kC4, c = e % kC4;
    // (kC4 is 16 or 32: every wave's lanes hold 4 or 2 rows, and all lanes take part in the shuffles)
    const int rt = __shfl(token, r, 64), rh = __shfl(head, r, 64);
    if (!__shfl(static_cast<int>(row_ok), r, 64)) continue;
    float mm = wml[0][r].x;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) mm = fmaxf(mm, wml[w][r].x);
    float den = 0.0f;
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float2 x = wml[w][r];
      den += x.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(x.x - mm) * x.y;
      v += *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(buf[w]) + r * kPitch + 4 * c);
    }
    const int64_t row = static_cast<int64_t>(rt) * a.n_q + rh;
    if (a.parts == 1) {
      const float inv = den > 0.0f ? 1.0f / den : 0.0f;
      Q y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = static_cast<Q>(v[i] * inv);
      struct alignas(4 * sizeof(Q)) Q4v {
        Q v[4];
      };
      *reinterpret_cast<Q4v*>(static_cast<Q*>(a.out) + row * HD + 4 * c) = Q4v{{y[0], y[1], y[2], y[3]}};
    } else {
      const int64_t i = row * a.parts + part;
      *reinterpret_cast<f32x4*>(a.o + i * HD + 4 * c) = v;
      if (c == 0) *reinterpret_cast<float2*>(a.ml + 2 * i) = make_float2(mm, den);
    }
  }
}

// Joins the ranges of each row, a thread for 4 dims of a row; the first kB ranges are in flight at once.
template <int QT, int HD>
__global__ __launch_bounds__(256) void paged_join_kernel(AttnArgs a) {
  typedef typename Num<QT>::type Q;
  constexpr int kC4 = HD / 4, kB = 8;
  const int64_t e = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t row = e / kC4;
  const int c = static_cast<int>(e % kC4);
  if (row >= static_cast<int64_t>(a.T) * a.n_q) return;
  if (a.b.cu) {
    const int64_t t = row / a.n_q;
    if (t < a.b.cu[0] || t >= a.b.cu[a.b.batch]) return;  // of no sequence
  }
  const float2* ml = reinterpret_cast<const float2*>(a.ml) + row * a.parts;
  const float* o = a.o + row * a.parts * HD + 4 * c;
  float M = -INFINITY, den = 0.0f;
  f32x4 num = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int p0 = 0; p0 < a.parts; p0 += kB) {
    float2 x[kB];
    f32x4 v[kB];
#pragma unroll
    for (int i = 0; i < kB; ++i) {
      x[i] = make_float2(-INFINITY, 0.0f);
      if (p0 + i < a.parts) {
        x[i] = ml[p0 + i];
        v[i] = *reinterpret_cast<const f32x4*>(o + static_cast<int64_t>(p0 + i) * HD);
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
  const float inv = den > 0.0f ? 1.0f / den : 0.0f;
  struct alignas(4 * sizeof(Q)) Q4v {
    Q v[4];
  };
  Q4v y;
#pragma unroll
  for (int j = 0; j < 4; ++j) y.v[j] = static_cast<Q>(num[j] * inv);
  *reinterpret_cast<Q4v*>(static_cast<Q*>(a.out) + row * HD + 4 * c) = y;
}

struct Plan {
  int64_t shared_tiles, own_tiles;  // row tiles (own: an upper bound)
  int shared_splits, shared_keys, own_splits, parts;
};

// Ranges: enough workgroups to give every compute unit two, and no range below 128 keys (a block for each wave).
int splits_for(int64_t items, int64_t keys) {
  const int64_t want = std::max<int64_t>(1, 512 / std::max<int64_t>(items, 1));
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({want, (keys + 127) / 128, 64})));
}

Plan plan_for(int64_t T, int g, int n_kv, int batch, bool ragged, int L, int shared_len) {
  Plan p{};
  const int64_t rows = T * g;
  p.own_tiles = ragged ? (rows + static_cast<int64_t>(kRows - 1) * batch) / kRows
                       : batch * ((rows / batch + kRows - 1) / kRows);
  p.own_splits = L > shared_len ? splits_for(n_kv * p.own_tiles, L - shared_len) : 0;
  if (shared_len > 0) {
    p.shared_tiles = (rows + kRows - 1) / kRows;
    const int s = splits_for(n_kv * p.shared_tiles, shared_len);
    p.shared_keys = ((shared_len + s - 1) / s + kKeys - 1) / kKeys * kKeys;
    p.shared_splits = (shared_len + p.shared_keys - 1) / p.shared_keys;
  }
  p.parts = p.shared_splits + p.own_splits;
  return p;
}

size_t ml_floats(size_t n) { return (2 * n + 3) / 4 * 4; }

int attn_args(int64_t T, int n_q, int n_kv, int hd, int batch, int L, int shared_len) {
  if (T < 0 || T > INT32_MAX || n_q <= 0 || n_kv <= 0 || batch <= 0 || L <= 0 || shared_len < 0 || shared_len > L)
    return Q4_ERR_SHAPE;
  if (n_q % n_kv || T * n_q > INT32_MAX) return Q4_ERR_SHAPE;
  if (hd != 64 && hd != 128) return Q4_ERR_UNSUPPORTED;
  if (n_q / n_kv > 64) return Q4_ERR_UNSUPPORTED;
  return Q4_OK;
}

template <int QT, int CT, int HD>
int launch(const AttnArgs& a, int64_t blocks, hipStream_t st) {
  hipLaunchKernelGGL((paged_attn_kernel<QT, CT, HD>), dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, st, a);
  if (a.parts > 1) {
    const int64_t threads = static_cast<int64_t>(a.T) * a.n_q * (HD / 4);
    hipLaunchKernelGGL((paged_join_kernel<QT, HD>), dim3(static_cast<unsigned>((threads + 255) / 256)), dim3(256), 0, st, a);
  }
  return launch_status();
}

}  // namespace
}  // namespace q4

using namespace q4;

extern "C" int paged_attn_workspace_bytes(int64_t T, int n_q, int n_kv, int head_dim, int batch, int L, int shared_len,
                                          size_t* bytes) {
  if (!bytes) return Q4_ERR_NULL;
  if (int st = attn_args(T, n_q, n_kv, head_dim, batch, L, shared_len)) return st;
  size_t most = 0;
  for (const bool ragged : {false, true}) {
    if (!ragged && T % batch) continue;
    const Plan p = plan_for(T, n_q / n_kv, n_kv, batch, ragged, L, shared_len);
    const size_t n = static_cast<size_t>(T) * n_q * p.parts;
    if (p.parts > 1) most = std::max(most, (ml_floats(n) + n * head_dim) * sizeof(float));
  }
  *bytes = most;
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
  const Plan p = plan_for(T, g, kv->n_kv, kv->batch, kv->cu_q != nullptr, L, shared_len);
  const size_t n = static_cast<size_t>(T) * n_q * p.parts;
  if (p.parts > 1) {
    if (!workspace || workspace_bytes < (ml_floats(n) + n * hd) * sizeof(float)) return Q4_ERR_WORKSPACE;
    if (!aligned(workspace, 16)) return Q4_ERR_ALIGN;
  }
  const int64_t shared_blocks = p.shared_tiles * p.shared_splits * kv->n_kv;
  const int64_t blocks = shared_blocks + p.own_tiles * p.own_splits * kv->n_kv;
  if (blocks > INT32_MAX) return Q4_ERR_SHAPE;
  a.q = q, a.qr = q_row, a.qh = q_head;
  a.kc = kv->k_cache, a.vc = kv->v_cache, a.out = out;
  a.ml = static_cast<float*>(workspace);
  a.o = a.ml + ml_floats(n);
  a.shared_pages = shared_pages;
  a.T = static_cast<int>(T), a.n_q = n_q, a.n_kv = kv->n_kv, a.g = g, a.L = L, a.shared_len = shared_len;
  a.shared_blocks = static_cast<int>(shared_blocks), a.shared_splits = p.shared_splits, a.shared_keys = p.shared_keys;
  a.own_splits = p.own_splits, a.parts = p.parts;
  // a negative scale turns q around and a zero one clears it, so that the exponents' factor is positive
  a.sign = scale < 0.0f ? -1.0f : scale == 0.0f ? 0.0f : 1.0f;
  a.cs = scale == 0.0f ? 1.0f : std::fabs(scale) * 1.44269504088896340736f;
  a.by_g = FastDiv(g), a.by_kv = FastDiv(kv->n_kv);
  a.by_shared = FastDiv(std::max(p.shared_splits, 1)), a.by_own = FastDiv(std::max(p.own_splits, 1));
  const hipStream_t st = as_stream(stream);
  const auto fn = dtype == Q4_F32    ? (hd == 128 ? launch<Q4_F32, Q4_F16, 128> : launch<Q4_F32, Q4_F16, 64>)
                  : dtype == Q4_F16  ? (hd == 128 ? launch<Q4_F16, Q4_F16, 128> : launch<Q4_F16, Q4_F16, 64>)
                                     : (hd == 128 ? launch<Q4_BF16, Q4_BF16, 128> : launch<Q4_BF16, Q4_BF16, 64>);
  return fn(a, blocks, st);
}
