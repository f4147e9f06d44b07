// Verification of drafted tokens against the target's probabilities (spec_verify).
//
// Row b accepts its drafted tokens x_i while u_i q_i(x_i) < p_i(x_i); at the first refusal j the next token is drawn from
// w = max(p_j - q_j, 0), after the last acceptance from w = p_n, by inversion: the lowest index whose running sum exceeds
// r sum(w). The product of two fp32 numbers is exact in fp64 and so is nearly every difference, and sums are
// fp64 in a fixed order, so the choice is that of the definition but within about 1e-14 of a border.
//
// Two launches, each one pass: the first decides j (every wave for itself: two dependent round trips instead of a
// launch) and sums w over chunks of kChunk values, a wave each; the second finds the chunk by a scan of the chunk sums, and
// reads that chunk again for the index. Only one row of p and one of q is read in full, whatever the number
// of drafts. Bound: HBM for large batches (64 rows of 128256 values 19.8 us, 3.3 TB/s: the sums 15.6, the pick 4.6; 13.9 without
// draft_probs), the dependent loads and two launches for one sequence (32000 values 9.5 us).
#include "q4_common.h"

#include <algorithm>

namespace q4 {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kChunk = kThreads * 4;              // values of a row that are summed together: a wave's, and 4 a thread of the pick
constexpr int kPer = kChunk / (64 * 4);           // float4s per lane of a wave that sums a chunk

struct VerifyArgs {
  const int32_t* tokens;
  const float* draft;
  const float* target;
  const float* uniforms;
  const int32_t* n_draft;
  int64_t tok_row, draft_batch, draft_row, target_batch, target_row, uni_row;
  int K, V, chunks;
  double2* sums;     // [B][chunks]: of w, and of p alone
  int32_t* out;
  int32_t* accepted;
};

// Tokens of row b that are accepted, and how many were drafted. The same in every lane.
__device__ __forceinline__ int accepted_of(const VerifyArgs& a, int b, int* drafted) {
  const int n = a.n_draft ? min(max(a.n_draft[b], 0), a.K) : a.K;
  *drafted = n;
  const int lane = threadIdx.x & 63;
  for (int base = 0; base < n; base += 64) {
    const int i = base + lane;
    bool ok = false;
    if (i < n) {
      const int x = a.tokens[b * a.tok_row + i];
      if (x >= 0 && x < a.V) {
        const double u = a.uniforms[b * a.uni_row + i];
        const double q = a.draft ? a.draft[b * a.draft_batch + i * a.draft_row + x] : 1.0f;
        ok = u * q < static_cast<double>(a.target[b * a.target_batch + i * a.target_row + x]);
      }
    }
    const uint64_t bad = ~__ballot(ok);
    if (bad) return min(base + __builtin_ctzll(bad), n);
  }
  return n;
}

// The weights of one row: w = max(p - q, 0) of the refused place, p otherwise.
struct Weights {
  const float* p;
  const float* q;  // null: none
  int zero;        // index of no weight (a certain draft that was refused), -1: none
};
__device__ __forceinline__ Weights weights_of(const VerifyArgs& a, int b, int j, int drafted) {
  Weights w{a.target + b * a.target_batch + j * a.target_row, nullptr, -1};
  if (j < drafted) {
    if (a.draft) w.q = a.draft + b * a.draft_batch + j * a.draft_row;
    else w.zero = a.tokens[b * a.tok_row + j];
  }
  return w;
}

// (w, p) of the 4 values from e on (zeros past V); rows start on whole floats, not on whole vectors.
struct alignas(4) Quad {
  float v[4];
};
__device__ __forceinline__ void load4(const float* row, int e, int V, float (&v)[4]) {
  if (e <= V - 4) {
    const Quad q = *reinterpret_cast<const Quad*>(row + e);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = q.v[i];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = e < V - i ? row[e + i] : 0.0f;
  }
}
__device__ __forceinline__ double weight(const Weights& w, int e, float p, float q) {
  const double d = e == w.zero ? 0.0 : static_cast<double>(p) - static_cast<double>(q);
  return d > 0.0 ? d : 0.0;
}
__device__ __forceinline__ double positive(float p) { return p > 0.0f ? static_cast<double>(p) : 0.0; }

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
  return v;
}

// A wave sums a chunk: no barrier.
__global__ __launch_bounds__(kThreads) void verify_sum_kernel(VerifyArgs a) {
  const int groups = (a.chunks + kWaves - 1) / kWaves;
  const int b = blockIdx.x / groups, c = (blockIdx.x - b * groups) * kWaves + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (c >= a.chunks) return;
  int drafted;
  const int j = accepted_of(a, b, &drafted);
  const Weights w = weights_of(a, b, j, drafted);
  float p[kPer][4], q[kPer][4] = {};
#pragma unroll
  for (int k = 0; k < kPer; ++k) load4(w.p, c * kChunk + (k * 64 + lane) * 4, a.V, p[k]);
  if (w.q) {
#pragma unroll
    for (int k = 0; k < kPer; ++k) load4(w.q, c * kChunk + (k * 64 + lane) * 4, a.V, q[k]);
  }
  double s = 0.0, sp = 0.0;
#pragma unroll
  for (int k = 0; k < kPer; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s += weight(w, c * kChunk + (k * 64 + lane) * 4 + i, p[k][i], q[k][i]);
      sp += positive(p[k][i]);
    }
  s = wave_sum(s);
  sp = wave_sum(sp);
  if (lane == 0) {
    a.sums[static_cast<int64_t>(b) * a.chunks + c] = make_double2(s, sp);
    if (c == 0) a.accepted[b] = j;
  }
}

// Inclusive running sums over the threads of the workgroup, of N values at once; total[k]: of all threads. `part`: N doubles
// per wave, free on entry; the caller synchronises before it is used again.
template <int N>
__device__ __forceinline__ void block_scan(double (&v)[N], double (*part)[N], double (&total)[N]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    double o[N];
#pragma unroll
    for (int k = 0; k < N; ++k) o[k] = __shfl_up(v[k], m, 64);
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (lane >= m) v[k] += o[k];
  }
  if (lane == 63)
#pragma unroll
    for (int k = 0; k < N; ++k) part[wave][k] = v[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; ++k) {
    double before = 0.0, all = 0.0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      if (i == wave) before = all;
      all += part[i][k];
    }
    total[k] = all;
    v[k] += before;
  }
}

// The least `lo` and the largest `hi` of the workgroup, in every thread. `part`: free on entry.
__device__ __forceinline__ int2 block_min_max(int lo, int hi, int2* part) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) {
    lo = min(lo, __shfl_xor(lo, m, 64));
    hi = max(hi, __shfl_xor(hi, m, 64));
  }
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = make_int2(lo, hi);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWaves; ++i) lo = min(lo, part[i].x), hi = max(hi, part[i].y);
  return make_int2(lo, hi);
}

__global__ __launch_bounds__(kThreads) void verify_pick_kernel(VerifyArgs a) {
  const int b = blockIdx.x;
  __shared__ double sums_s[kWaves][2], in_s[kWaves][1], before_s;
  __shared__ int2 mm[2][kWaves];
  const int drafted = a.n_draft ? min(max(a.n_draft[b], 0), a.K) : a.K;
  const int j = a.accepted[b];
  const double u = a.uniforms[b * a.uni_row + a.K];
  const double2* sums = a.sums + static_cast<int64_t>(b) * a.chunks;
  auto load = [&](int c) { return c < a.chunks ? sums[c] : make_double2(0.0, 0.0); };
  // the sums of all chunks; one tile of kThreads chunks (256 K values) is kept with its running sums
  const double2 mine = load(threadIdx.x);
  double run[2] = {mine.x, mine.y}, all[2];
  block_scan(run, sums_s, all);
  for (int i = kThreads; i < a.chunks; i += kThreads) {
    const double2 s = load(i + threadIdx.x);
    double v[2] = {s.x, s.y}, t[2];
    __syncthreads();
    block_scan(v, sums_s, t);
    all[0] += t[0], all[1] += t[1];
  }
  const int f = all[0] > 0.0 ? 0 : 1;  // nothing left of p at the refused place: p itself
  const double limit = all[f] * u;
  // the first chunk whose running sum exceeds the limit, else the last one with any weight
  double carry = 0.0;
  int chunk = -1;
  for (int i = 0; i < a.chunks; i += kThreads) {
    const int c = i + threadIdx.x;
    double s = f ? mine.y : mine.x, r = run[f], t = 0.0;
    if (a.chunks > kThreads) {  // more than one tile: again, with the sums of those before
      const double2 s2 = load(c);
      s = f ? s2.y : s2.x;
      double v[1] = {s}, w[1];
      __syncthreads();
      block_scan(v, in_s, w);
      r = carry + v[0];
      t = w[0];
    }
    const int2 at = block_min_max(s > 0.0 && r > limit ? c : INT32_MAX, s > 0.0 ? c : -1, mm[0]);
    const bool found = at.x != INT32_MAX;
    if (found) chunk = at.x;
    else if (at.y >= 0) chunk = at.y;
    if (c == chunk) before_s = r - s;
    __syncthreads();
    if (found) break;
    carry += t;
  }
  int next = -1;
  if (chunk >= 0) {
    Weights w = weights_of(a, b, j, drafted);
    if (f) w.q = nullptr, w.zero = -1;
    const int e = chunk * kChunk + threadIdx.x * 4;
    float p[4], q[4] = {};
    load4(w.p, e, a.V, p);
    if (w.q) load4(w.q, e, a.V, q);
    double v[4], s[1], t[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = weight(w, e + i, p[i], q[i]);
    const double own = ((v[0] + v[1]) + v[2]) + v[3];
    s[0] = own;
    block_scan(s, in_s, t);
    double r = before_s + (s[0] - own);
    int lo = INT32_MAX, hi = -1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      r += v[i];
      if (v[i] > 0.0) {
        if (r > limit) lo = min(lo, e + i);
        hi = max(hi, e + i);
      }
    }
    const int2 at = block_min_max(lo, hi, mm[1]);
    next = at.x != INT32_MAX ? at.x : at.y;
  }
  for (int i = threadIdx.x; i <= a.K; i += kThreads)
    a.out[static_cast<int64_t>(b) * (a.K + 1) + i] = i < j ? a.tokens[b * a.tok_row + i] : i == j ? next : -1;
}

int chunks_of(int64_t V) { return static_cast<int>((V + kChunk - 1) / kChunk); }

}  // namespace
}  // namespace q4

using namespace q4;

extern "C" int spec_verify_workspace_bytes(int B, int K, int64_t V, size_t* bytes) {
  if (!bytes) return Q4_ERR_NULL;
  if (B <= 0 || K < 0 || V <= 0 || V > INT32_MAX - kChunk || static_cast<int64_t>(B) * chunks_of(V) > INT32_MAX)
    return Q4_ERR_SHAPE;
  *bytes = static_cast<size_t>(B) * chunks_of(V) * sizeof(double2);
  return Q4_OK;
}

extern "C" int spec_verify(const int32_t* tokens, int64_t tok_row, const float* draft, int64_t draft_batch,
                           int64_t draft_row, const float* target, int64_t target_batch, int64_t target_row,
                           const float* uniforms, int64_t uni_row, const int32_t* n_draft, int B, int K, int64_t V,
                           int32_t* out_tokens, int32_t* n_accepted, void* workspace, size_t workspace_bytes, void* stream) {
  if ((!tokens && K > 0) || !target || !uniforms || !out_tokens || !n_accepted || !workspace) return Q4_ERR_NULL;
  size_t need = 0;
  if (int st = spec_verify_workspace_bytes(B, K, V, &need)) return st;
  if (tok_row < 0 || draft_batch < 0 || draft_row < 0 || target_batch < 0 || target_row < 0 || uni_row < 0)
    return Q4_ERR_SHAPE;
  if (workspace_bytes < need) return Q4_ERR_WORKSPACE;
  if (!aligned(tokens, 4) || !aligned(draft, 4) || !aligned(target, 4) || !aligned(uniforms, 4) || !aligned(n_draft, 4) ||
      !aligned(out_tokens, 4) || !aligned(n_accepted, 4) || !aligned(workspace, 16))
    return Q4_ERR_ALIGN;
  VerifyArgs a{tokens, draft, target, uniforms, n_draft, tok_row, draft_batch, draft_row, target_batch, target_row, uni_row,
               K, static_cast<int>(V), chunks_of(V), static_cast<double2*>(workspace), out_tokens, n_accepted};
  const hipStream_t st = as_stream(stream);
  const int64_t sums = static_cast<int64_t>(B) * ((a.chunks + kWaves - 1) / kWaves);
  if (!fits_grid(sums, kThreads)) return Q4_ERR_SHAPE;
  hipLaunchKernelGGL(verify_sum_kernel, dim3(static_cast<unsigned>(sums)), dim3(kThreads), 0, st, a);
  hipLaunchKernelGGL(verify_pick_kernel, dim3(B), dim3(kThreads), 0, st, a);
  return launch_status();
}
