// Rotary positions (rope_rotate) and the write of a step's keys and values into a paged cache with the rotation
// applied on the way (paged_kv_append).
//
// Pair i (a, b) of a head at position p: (a c - b s, b c + a s), c = mscale cos(p f_i), s = mscale sin(p f_i). The angle
// is formed in fp64 as revolutions, p f_i / 2 pi, whose fraction alone matters: at position 2^24 an fp32 angle
// is off by up to 0.5 rad, the fraction by 2^-26 revolutions (its rounding to fp32).
//
// A workgroup holds the cos / sin of its tokens in LDS, computed once for all heads (one per thread and pass), and then
// streams the heads: units of one or two 16-byte vectors, the loads of kU units in flight per thread, the
// first of them issued before the angles are formed, so that a small call is one memory round trip behind the
// positions. Sizes whose halves or strides are no whole vectors take the same kernel element by element.
#include "q4_common.h"
#include "q4_paged.h"

#include <algorithm>
#include <initializer_list>

// Which product of a sum is fused is written out: left to the compiler it differs between the kernels of one operator, and
// a token's result would depend on how many are rotated with it.
#pragma clang fp contract(off)

namespace q4 {
namespace {

constexpr int kThreads = 256;
constexpr int kU = 2;  // units in flight per thread (8192 tokens of 40 heads of 128, bf16: 40.7 us with 4, 38.2 with 2)

// Calls past this many bytes (the L2s together) go around the caches: nothing of them would be found there again, and
// what they displace would. 8192 tokens of 40 heads of 128, bf16: 38.2 -> 32 us, which is the time of a copy; with nothing
// to save (a few tokens) the rotated q stays in the cache for the attention that follows.
constexpr int64_t kStream = 32 << 20;

// V at p, around the caches if NT and V is a whole 16 bytes.
template <bool NT, typename V>
__device__ __forceinline__ V load_v(const void* p) {
  if constexpr (NT && sizeof(V) == 16) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(V, __builtin_nontemporal_load(static_cast<const u32x4*>(p)));
  } else {
    return *static_cast<const V*>(p);
  }
}
template <bool NT, typename V>
__device__ __forceinline__ void store_v(void* p, const V& v) {
  if constexpr (NT && sizeof(V) == 16) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    __builtin_nontemporal_store(__builtin_bit_cast(u32x4, v), static_cast<u32x4*>(p));
  } else {
    *static_cast<V*>(p) = v;
  }
}

// One unit of a head: a pair of vectors (half layout, rotated part), or one vector of interleaved pairs or of the
// part that is not rotated. Vectors of VB bytes (16 or 8); VB == 0: pairs of elements, then single ones.
template <int DT, int LAYOUT, int VB>
struct Unit {
  typedef typename Num<DT>::type T;
  static constexpr int E = VB ? VB / static_cast<int>(sizeof(T)) : 1;
  struct alignas(E * sizeof(T)) V {
    T v[E];
  };
  V a, b;

  // Element offsets of a unit's vectors in its head (second: -1 for none).
  static __device__ __forceinline__ int first(int u, int half) {
    if constexpr (LAYOUT == Q4_ROPE_HALF) return u < half / E ? u * E : 2 * half + (u - half / E) * E;
    return VB ? u * E : 2 * u;
  }
  static __device__ __forceinline__ int second(int u, int half) {
    if constexpr (LAYOUT == Q4_ROPE_HALF) return u < half / E ? half + u * E : -1;
    return VB ? -1 : 2 * u + 1;
  }
  // Units of a head of hd dims; those of its rotated part alone.
  static int count(int hd, int half) { return LAYOUT == Q4_ROPE_HALF ? half / E + (hd - 2 * half) / E : VB ? hd / E : hd / 2; }
  static int rotated(int half) { return LAYOUT == Q4_ROPE_HALF ? half / E : VB ? (2 * half + E - 1) / E : half; }

  template <bool NT>
  __device__ __forceinline__ void load(const T* head, int u, int half) {
    a = load_v<NT, V>(head + first(u, half));
    const int s = second(u, half);
    if (s >= 0) b = load_v<NT, V>(head + s);
  }
  // Rotates by the token's table of (cos, sin); pairs past `half` keep their values.
  __device__ __forceinline__ void rotate(const float2* cs, int u, int half) {
    auto pair = [&](T& x, T& y, int i) {
      const float2 w = cs[i];
      const float p = static_cast<float>(x), q = static_cast<float>(y);
      x = static_cast<T>(fmaf(p, w.x, -(q * w.y)));
      y = static_cast<T>(fmaf(q, w.x, p * w.y));
    };
    if constexpr (LAYOUT == Q4_ROPE_HALF) {
      if (u < half / E)
#pragma unroll
        for (int e = 0; e < E; ++e) pair(a.v[e], b.v[e], u * E + e);
    } else if constexpr (VB != 0) {
#pragma unroll
      for (int e = 0; e < E / 2; ++e)
        if (u * (E / 2) + e < half) pair(a.v[2 * e], a.v[2 * e + 1], u * (E / 2) + e);
    } else if (u < half) {
      pair(a.v[0], b.v[0], u);
    }
  }
  template <bool NT, typename C>
  __device__ __forceinline__ void store(C* head, int u, int half) const {
    struct alignas(E * sizeof(C)) W {
      C v[E];
    };
    auto put = [&](const V& x, int off) {
      W w;
#pragma unroll
      for (int e = 0; e < E; ++e) w.v[e] = static_cast<C>(x.v[e]);
      store_v<NT>(head + off, w);
    };
    put(a, first(u, half));
    const int s = second(u, half);
    if (s >= 0) put(b, s);
  }
};

// (cos, sin) of frequency f at position p, times mscale.
__device__ __forceinline__ float2 cos_sin(int p, float f, float mscale) {
  double r = static_cast<double>(p) * static_cast<double>(f) * 0.15915494309189533577;  // 1 / (2 pi)
  r -= rint(r);
  float s, c;
  sincospif(2.0f * static_cast<float>(r), &s, &c);
  return make_float2(mscale * c, mscale * s);
}

struct RopeArgs {
  const float* inv_freq;
  int half;
  float mscale, sign;
};

// The tables of the `n` tokens of this workgroup: cs[token][half], positions in pos (LDS). A barrier follows.
__device__ __forceinline__ void fill_tables(float2* cs, const int* pos, int n, const RopeArgs& r, FastDiv by_half) {
  for (int i = threadIdx.x; i < n * r.half; i += kThreads) {
    const int t = by_half.div(i);
    float2 w = cos_sin(pos[t], r.inv_freq[i - t * r.half], r.mscale);
    w.y *= r.sign;
    cs[i] = w;
  }
}

// x, y: T tokens of H heads; workgroup (x, y): tokens x * tpb .., part y of their units. HBM bound: 8192 tokens of 40 heads of
// 128 dims in bf16 30.1 us, 5.6 TB/s; 8 tokens of 32 heads 3.0 us, the launch and two dependent loads.
template <int DT, int LAYOUT, int VB, bool NT>
__global__ __launch_bounds__(kThreads) void rope_kernel(const void* x_, int64_t xr, int64_t xh, void* y_, int64_t yr,
                                                       int64_t yh, int T, int tpb, int H, int units, int part,
                                                       const int32_t* __restrict__ positions, RopeArgs r, FastDiv by_units,
                                                       FastDiv by_heads, FastDiv by_half) {
  typedef Unit<DT, LAYOUT, VB> U;
  typedef typename U::T E;
  extern __shared__ float2 lds[];
  int* pos = reinterpret_cast<int*>(lds);
  float2* cs = lds + (tpb + 1) / 2;
  const E* x = static_cast<const E*>(x_);
  E* y = static_cast<E*>(y_);
  const int t0 = blockIdx.x * tpb, n = min(tpb, T - t0);
  const int end = min(n * H * units, (static_cast<int>(blockIdx.y) + 1) * part);
  const int mine = blockIdx.y * part + threadIdx.x;
  U w[kU];
  auto load = [&](int base) {
#pragma unroll
    for (int k = 0; k < kU; ++k) {
      const int i = base + k * kThreads;
      if (i < end) {
        const int hh = by_units.div(i), t = by_heads.div(hh);
        w[k].template load<NT>(x + (t0 + t) * xr + (hh - t * H) * xh, i - hh * units, r.half);
      }
    }
  };
  load(mine);
  if (threadIdx.x < n) pos[threadIdx.x] = positions[t0 + threadIdx.x];
  __syncthreads();
  fill_tables(cs, pos, n, r, by_half);
  __syncthreads();
  for (int base = mine; base < end; base += kU * kThreads) {
    if (base != mine) load(base);
#pragma unroll
    for (int k = 0; k < kU; ++k) {
      const int i = base + k * kThreads;
      if (i < end) {
        const int hh = by_units.div(i), t = by_heads.div(hh), u = i - hh * units;
        w[k].rotate(cs + t * r.half, u, r.half);
        w[k].template store<NT>(y + (t0 + t) * yr + (hh - t * H) * yh, u, r.half);
      }
    }
  }
}

struct AppendArgs {
  PagedBatch b;
  const void *k, *v, *q;
  void *kc, *vc, *qo;
  int64_t kr, kh, vr, vh, qr, qh, por, poh;
  int T, tpb, n_kv, heads, hd, units, part;  // heads: n_kv of k, n_kv of v, then those of q
  RopeArgs r;
  FastDiv by_units, by_heads, by_half;
};

// How many sequences end at or before token t (tokens of cu ascending): the sequence that holds t.
// Every lane of the wave passes the same t.
__device__ __forceinline__ int sequence_of(const PagedBatch& b, int t) {
  int n = 0;
  for (int i = 0; i < b.batch; i += 64) {
    const int l = i + (threadIdx.x & 63);
    n += __popcll(__ballot(l < b.batch && b.cu[min(l, b.batch - 1) + 1] <= t));
  }
  return n;
}

// The same over the heads of k, v and q of each token, with the row of the cache looked up beside the tables. HBM bound: prompts
// of 16 sequences (8000 tokens, 32/8 heads of 128 in bf16) 40.1 us, 5.0 TB/s; 32 tokens 4.2 us, three dependent loads.
template <int DT, int CT, int LAYOUT, int VB, bool NT>
__global__ __launch_bounds__(kThreads) void append_kernel(AppendArgs a) {
  typedef Unit<DT, LAYOUT, VB> U;
  typedef typename U::T E;
  typedef typename Num<CT>::type C;
  extern __shared__ float2 lds[];
  int* pos = reinterpret_cast<int*>(lds);      // position of each token, -1 for none
  int* slot = pos + a.tpb;                     // its row of the cache, -1 for none
  float2* cs = lds + a.tpb;
  const int t0 = blockIdx.x * a.tpb, n = min(a.tpb, a.T - t0);
  const int end = min(n * a.heads * a.units, (static_cast<int>(blockIdx.y) + 1) * a.part);
  const int mine = blockIdx.y * a.part + threadIdx.x;
  const int half = a.r.half;
  U w[kU];
  auto head_of = [&](int i, int* t, int* h) {
    const int hh = a.by_units.div(i);
    *t = a.by_heads.div(hh);
    *h = hh - *t * a.heads;
    return i - hh * a.units;
  };
  auto load = [&](int base) {
#pragma unroll
    for (int k = 0; k < kU; ++k) {
      const int i = base + k * kThreads;
      if (i < end) {
        int t, h;
        const int u = head_of(i, &t, &h);
        const int64_t tt = t0 + t;
        const E* p = h < a.n_kv       ? static_cast<const E*>(a.k) + tt * a.kr + h * a.kh
                     : h < 2 * a.n_kv ? static_cast<const E*>(a.v) + tt * a.vr + (h - a.n_kv) * a.vh
                                      : static_cast<const E*>(a.q) + tt * a.qr + (h - 2 * a.n_kv) * a.qh;
        w[k].template load<NT>(p, u, half);
      }
    }
  };
  load(mine);
  // wave i: tokens i, i + 4, ..
  for (int j = threadIdx.x >> 6; j < n; j += kThreads / 64) {
    const int t = t0 + j;
    int b, p = -1, s = -1;
    if (a.b.cu) {
      b = sequence_of(a.b, t);
      if (b < a.b.batch) {
        const int c0 = a.b.cu[b], c1 = a.b.cu[b + 1];
        if (t >= c0 && c0 >= 0 && a.b.lens[b] >= 0) p = a.b.lens[b] - c1 + t;
      }
    } else {
      b = a.b.by_rows.div(t);
      if (a.b.lens[b] >= 0) p = a.b.lens[b] - a.b.rows + (t - b * a.b.rows);
    }
    if (p >= 0) {
      const int page = a.b.by_page.div(p);
      if (page < a.b.max_pages) s = a.b.slot(a.b.table[b * a.b.stride + page], p - page * a.b.page_size);
    }
    if ((threadIdx.x & 63) == 0) {
      pos[j] = max(p, -1);
      slot[j] = s;
    }
  }
  __syncthreads();
  fill_tables(cs, pos, n, a.r, a.by_half);
  __syncthreads();
  for (int base = mine; base < end; base += kU * kThreads) {
    if (base != mine) load(base);
#pragma unroll
    for (int k = 0; k < kU; ++k) {
      const int i = base + k * kThreads;
      if (i < end) {
        int t, h;
        const int u = head_of(i, &t, &h);
        const int64_t s = slot[t];
        if (h < a.n_kv || h >= 2 * a.n_kv) w[k].rotate(cs + t * half, u, half);
        if (h >= 2 * a.n_kv) {
          if (pos[t] >= 0) w[k].template store<NT>(static_cast<E*>(a.qo) + (t0 + t) * a.por + (h - 2 * a.n_kv) * a.poh, u, half);
        } else if (s >= 0) {
          C* c = static_cast<C*>(h < a.n_kv ? a.kc : a.vc);
          w[k].template store<NT>(c + (s * a.n_kv + (h < a.n_kv ? h : h - a.n_kv)) * a.hd, u, half);
        }
      }
    }
  }
}

// Tokens per workgroup and parts per token group: about kU units a thread while that leaves 1024 workgroups (four for
// each compute unit), else a token, whose units are split until there are 512.
struct Split {
  int tpb, part, parts;
};
Split split_for(int64_t T, int per_token, int half) {
  Split s;
  s.tpb = std::max(1, std::min({kU * kThreads / per_token, static_cast<int>(std::min<int64_t>(T / 1024, 16)),
                                2048 / std::max(half, 1)}));
  const int units = s.tpb * per_token;
  const int64_t wgs = (T + s.tpb - 1) / s.tpb;
  s.parts = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>((units + kThreads - 1) / kThreads, 512 / wgs)));
  s.part = (units + s.parts - 1) / s.parts;
  return s;
}

int rope_args(const q4_rope* rope, int hd, RopeArgs* r, int* layout) {
  *r = RopeArgs{nullptr, 0, 1.0f, 1.0f};
  *layout = Q4_ROPE_HALF;
  if (!rope) return Q4_OK;
  if (rope->rot_dim < 0 || rope->rot_dim % 2 || rope->rot_dim > hd) return Q4_ERR_SHAPE;
  if (rope->layout != Q4_ROPE_HALF && rope->layout != Q4_ROPE_INTERLEAVED) return Q4_ERR_RANGE;
  if (rope->rot_dim && !rope->inv_freq) return Q4_ERR_NULL;
  if (!aligned(rope->inv_freq, 4)) return Q4_ERR_ALIGN;
  *r = RopeArgs{rope->inv_freq, rope->rot_dim / 2, rope->mscale, 1.0f};
  *layout = rope->layout;
  return Q4_OK;
}

size_t bytes_of(int dt) { return dt == Q4_F32 ? 4 : 2; }

template <int DT, int LAYOUT, int VB>
int launch_rope(const void* x, int64_t xr, int64_t xh, void* y, int64_t yr, int64_t yh, int64_t T, int heads, int hd,
                const int32_t* positions, const RopeArgs& r, hipStream_t st) {
  typedef Unit<DT, LAYOUT, VB> U;
  const bool in_place = x == y && xr == yr && xh == yh;
  const int units = in_place ? U::rotated(r.half) : U::count(hd, r.half);
  if (units == 0) return Q4_OK;
  const Split s = split_for(T, heads * units, r.half);
  if (!fits_grid((T + s.tpb - 1) / s.tpb, kThreads)) return Q4_ERR_SHAPE;
  const size_t lds = 8 * ((s.tpb + 1) / 2 + static_cast<size_t>(s.tpb) * r.half);
  const bool stream = T * heads * hd * static_cast<int64_t>(sizeof(typename U::T)) > kStream;
  const auto fn = VB == 16 && stream ? rope_kernel<DT, LAYOUT, VB, VB == 16> : rope_kernel<DT, LAYOUT, VB, false>;
  hipLaunchKernelGGL(fn, dim3(static_cast<unsigned>((T + s.tpb - 1) / s.tpb), s.parts),
                     dim3(kThreads), lds, st, x, xr, xh, y, yr, yh, static_cast<int>(T), s.tpb, heads, units, s.part,
                     positions, r, FastDiv(units), FastDiv(heads), FastDiv(std::max(r.half, 1)));
  return launch_status();
}

template <int DT, int LAYOUT>
int launch_rope1(int vb, const void* x, int64_t xr, int64_t xh, void* y, int64_t yr, int64_t yh, int64_t T, int heads, int hd,
                 const int32_t* positions, const RopeArgs& r, hipStream_t st) {
  const auto fn = vb == 16 ? launch_rope<DT, LAYOUT, 16> : vb == 8 ? launch_rope<DT, LAYOUT, 8> : launch_rope<DT, LAYOUT, 0>;
  return fn(x, xr, xh, y, yr, yh, T, heads, hd, positions, r, st);
}

template <int DT, int CT, int LAYOUT, int VB>
int launch_append(AppendArgs& a, hipStream_t st) {
  a.units = Unit<DT, LAYOUT, VB>::count(a.hd, a.r.half);
  const Split s = split_for(a.T, a.heads * a.units, a.r.half);
  if (!fits_grid((int64_t{a.T} + s.tpb - 1) / s.tpb, kThreads)) return Q4_ERR_SHAPE;
  a.tpb = s.tpb;
  a.part = s.part;
  a.by_units = FastDiv(a.units);
  a.by_heads = FastDiv(a.heads);
  a.by_half = FastDiv(std::max(a.r.half, 1));
  const size_t lds = 8 * (s.tpb + static_cast<size_t>(s.tpb) * a.r.half);
  const bool stream = static_cast<int64_t>(a.T) * a.heads * a.hd * static_cast<int64_t>(sizeof(typename Num<DT>::type)) > kStream;
  const auto fn = VB == 16 && stream ? append_kernel<DT, CT, LAYOUT, VB, VB == 16> : append_kernel<DT, CT, LAYOUT, VB, false>;
  hipLaunchKernelGGL(fn, dim3(static_cast<unsigned>((int64_t{a.T} + s.tpb - 1) / s.tpb), s.parts), dim3(kThreads), lds,
                     st, a);
  return launch_status();
}

template <int DT, int CT>
int launch_append1(int vb, int layout, AppendArgs& a, hipStream_t st) {
  const bool half = layout == Q4_ROPE_HALF;
  const auto fn = vb == 16  ? (half ? launch_append<DT, CT, Q4_ROPE_HALF, 16> : launch_append<DT, CT, Q4_ROPE_INTERLEAVED, 16>)
                  : vb == 8 ? (half ? launch_append<DT, CT, Q4_ROPE_HALF, 8> : launch_append<DT, CT, Q4_ROPE_INTERLEAVED, 8>)
                            : (half ? launch_append<DT, CT, Q4_ROPE_HALF, 0> : launch_append<DT, CT, Q4_ROPE_INTERLEAVED, 0>);
  return fn(a, st);
}

// The widest vectors, in bytes, in which heads of hd dims with `half` rotated pairs, operands at these addresses and these
// strides are whole (the interleaved layout needs no boundary between its rotated pairs and the rest on a vector);
// 0: none. Odd halves and starts go element by element (8192 tokens of 40 heads, 62 of 128 dims rotated by halves: 70 us).
int vector_bytes(int hd, int half, int layout, size_t es, std::initializer_list<const void*> at,
                 std::initializer_list<int64_t> strides) {
  for (const int vb : {16, 8}) {
    const int e = vb / static_cast<int>(es);
    bool ok = hd % e == 0 && (layout == Q4_ROPE_INTERLEAVED || half % e == 0);
    for (const void* p : at) ok = ok && aligned(p, vb);
    for (const int64_t s : strides) ok = ok && s % e == 0;
    if (ok) return vb;
  }
  return 0;
}

}  // namespace
}  // namespace q4

using namespace q4;

extern "C" int rope_rotate(const void* x, int64_t x_row, int64_t x_head, void* y, int64_t y_row, int64_t y_head, int dtype,
                           int64_t T, int heads, int head_dim, const int32_t* positions, const q4_rope* rope, int inverse,
                           void* stream) {
  if (!x || !y || !positions || !rope) return Q4_ERR_NULL;
  if (dtype != Q4_F32 && dtype != Q4_F16 && dtype != Q4_BF16) return Q4_ERR_DTYPE;
  if (T < 0 || heads <= 0 || head_dim <= 0 || head_dim % 2 || head_dim > 1024 || T > INT32_MAX ||
      T * heads > INT32_MAX || x_row < 0 || x_head < 0 || y_row < 0 || y_head < 0)
    return Q4_ERR_SHAPE;
  if (static_cast<int64_t>(heads) * head_dim > INT32_MAX / 16) return Q4_ERR_SHAPE;
  RopeArgs r;
  int layout;
  if (int st = rope_args(rope, head_dim, &r, &layout)) return st;
  const size_t es = bytes_of(dtype);
  if (!aligned(x, es) || !aligned(y, es) || !aligned(positions, 4)) return Q4_ERR_ALIGN;
  if (T == 0) return Q4_OK;
  r.sign = inverse ? -1.0f : 1.0f;
  const int vb = vector_bytes(head_dim, r.half, layout, es, {x, y}, {x_row, x_head, y_row, y_head});
  const bool half = layout == Q4_ROPE_HALF;
  const auto fn = dtype == Q4_F32   ? (half ? launch_rope1<Q4_F32, Q4_ROPE_HALF> : launch_rope1<Q4_F32, Q4_ROPE_INTERLEAVED>)
                  : dtype == Q4_F16 ? (half ? launch_rope1<Q4_F16, Q4_ROPE_HALF> : launch_rope1<Q4_F16, Q4_ROPE_INTERLEAVED>)
                                    : (half ? launch_rope1<Q4_BF16, Q4_ROPE_HALF> : launch_rope1<Q4_BF16, Q4_ROPE_INTERLEAVED>);
  return fn(vb, x, x_row, x_head, y, y_row, y_head, T, heads, head_dim, positions, r, as_stream(stream));
}

extern "C" int paged_kv_append(const q4_paged_kv* kv, const void* k, int64_t k_row, int64_t k_head, const void* v,
                               int64_t v_row, int64_t v_head, int dtype, int64_t T, const q4_rope* rope, const void* q,
                               int64_t q_row, int64_t q_head, void* q_out, int64_t qo_row, int64_t qo_head, int n_q,
                               void* stream) {
  if (!k || !v || (q && !q_out)) return Q4_ERR_NULL;
  AppendArgs a;
  if (int st = paged_batch(kv, dtype, T, &a.b)) return st;
  const int hd = kv->head_dim;
  if (hd % 2 || hd > 1024 || k_row < 0 || k_head < 0 || v_row < 0 || v_head < 0) return Q4_ERR_SHAPE;
  if (q ? n_q <= 0 || q_row < 0 || q_head < 0 || qo_row < 0 || qo_head < 0 : n_q != 0) return Q4_ERR_SHAPE;
  const int64_t heads = 2 * static_cast<int64_t>(kv->n_kv) + n_q;
  if (heads * hd > INT32_MAX / 16) return Q4_ERR_SHAPE;
  int layout;
  if (int st = rope_args(rope, hd, &a.r, &layout)) return st;
  const size_t es = bytes_of(dtype), cs = bytes_of(kv->dtype);
  if (!aligned(k, es) || !aligned(v, es) || !aligned(q, es) || !aligned(q_out, es) || !aligned(kv->k_cache, cs) ||
      !aligned(kv->v_cache, cs))
    return Q4_ERR_ALIGN;
  if (T == 0) return Q4_OK;
  const int vb = vector_bytes(hd, a.r.half, layout, es, {k, v, kv->k_cache, kv->v_cache, q, q_out},
                              {k_row, k_head, v_row, v_head, q ? q_row : 0, q ? q_head : 0, q ? qo_row : 0, q ? qo_head : 0});
  a.k = k, a.kr = k_row, a.kh = k_head;
  a.v = v, a.vr = v_row, a.vh = v_head;
  a.q = q, a.qr = q_row, a.qh = q_head;
  a.qo = q_out, a.por = qo_row, a.poh = qo_head;
  a.kc = kv->k_cache, a.vc = kv->v_cache;
  a.T = static_cast<int>(T), a.n_kv = kv->n_kv, a.heads = static_cast<int>(heads), a.hd = hd;
  const hipStream_t st = as_stream(stream);
  if (dtype == Q4_F32) return launch_append1<Q4_F32, Q4_F16>(vb, layout, a, st);
  if (dtype == Q4_F16) return launch_append1<Q4_F16, Q4_F16>(vb, layout, a, st);
  return launch_append1<Q4_BF16, Q4_BF16>(vb, layout, a, st);
}
