// gtk_logprobs.cu -- log probabilities of given tokens, entropy and top alternatives of rows of logits, and the
// gradient of the first two.
#include <cooperative_groups.h>

#include <cfloat>
#include <cmath>
#include <initializer_list>
#include <type_traits>

#include "gtk_rows.cuh"

namespace {

using gtk::Two;

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr float kLn2 = 0.693147180559945309f, kLog2e = 1.44269504088896341f;

// exp2 of a number <= 0 (or NaN)
__device__ __forceinline__ float pow2(float y)
{
  float p;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p) : "f"(y));
  return p;
}

// 16 bytes of a row: its elements as pairs of 32-bit floats, and their maximum (NaN only where all are).
template <class T>
struct Pack16;
template <>
struct Pack16<float> {
  static constexpr int kElems = 4;
  static constexpr uint32_t kMinusInf = 0xFF800000u;
  static constexpr int kLowestBit     = 0;  // below it all numbers of the type agree, written as 32-bit floats
  static __device__ __forceinline__ void pairs(const uint4& r, Two (&x)[2])
  {
    x[0] = Two(__uint_as_float(r.x), __uint_as_float(r.y));
    x[1] = Two(__uint_as_float(r.z), __uint_as_float(r.w));
  }
  template <int N>
  static __device__ __forceinline__ float highest(const uint4 (&r)[N])
  {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i)
      m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(r[i].x), __uint_as_float(r[i].y)), fmaxf(__uint_as_float(r[i].z), __uint_as_float(r[i].w))));
    return m;
  }
};
template <class T, class T2>
struct Pack16Half {
  static constexpr int kElems = 8;
  static __device__ __forceinline__ T2 as(const uint32_t& w) { return *reinterpret_cast<const T2*>(&w); }
  static __device__ __forceinline__ float2 both(T2 w);
  static __device__ __forceinline__ void pairs(const uint4& r, Two (&x)[4])
  {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = both(as(w[i]));
      x[i]           = Two(f.x, f.y);
    }
  }
  template <int N>
  static __device__ __forceinline__ float highest(const uint4 (&r)[N])
  {
    T2 m = __hmax2(__hmax2(as(r[0].x), as(r[0].y)), __hmax2(as(r[0].z), as(r[0].w)));
#pragma unroll
    for (int i = 1; i < N; ++i) m = __hmax2(m, __hmax2(__hmax2(as(r[i].x), as(r[i].y)), __hmax2(as(r[i].z), as(r[i].w))));
    const float2 f = both(m);
    return fmaxf(f.x, f.y);
  }
};
template <>
__device__ __forceinline__ float2 Pack16Half<__nv_bfloat16, __nv_bfloat162>::both(__nv_bfloat162 w) { return __bfloat1622float2(w); }
template <>
__device__ __forceinline__ float2 Pack16Half<__half, __half2>::both(__half2 w) { return __half22float2(w); }
template <>
struct Pack16<__nv_bfloat16> : Pack16Half<__nv_bfloat16, __nv_bfloat162> {
  static constexpr uint32_t kMinusInf = 0xFF80FF80u;
  static constexpr int kLowestBit     = 16;
};
template <>
struct Pack16<__half> : Pack16Half<__half, __half2> {
  static constexpr uint32_t kMinusInf = 0xFC00FC00u;
  static constexpr int kLowestBit     = 13;
};

// A row in memory: elements in front of the first 16-byte boundary, packs of 16 bytes, elements behind the last pack.
template <class T>
struct RowParts {
  static constexpr int kElems = Pack16<T>::kElems;
  const T* x;
  int head, packs, tail;
  __device__ RowParts(const T* row, int vocab) : x(row)
  {
    head  = min(vocab, int((16u - (uint32_t(reinterpret_cast<uintptr_t>(row)) & 15u)) % 16u / sizeof(T)));
    packs = (vocab - head) / kElems;
    tail  = vocab - head - packs * kElems;
  }
  __device__ __forceinline__ const uint4* pack(int p) const { return reinterpret_cast<const uint4*>(x + head) + p; }
  __device__ __forceinline__ int pack_column(int p) const { return head + p * kElems; }
  // the i-th of the head + tail elements outside the packs
  __device__ __forceinline__ int loose_column(int i) const { return i < head ? i : packs * kElems + i; }
};

// What has been seen of a row: m the highest logit so far (starts at the lowest finite number, so that masked places at
// -inf never meet it in a difference of infinities), s the sum of 2^y and t that of 2^y * y with y = (x - m) * k,
// k = scale * log2(e).  y of an element that contributes nothing may be -inf: 0 * -inf is kept out of t.  A NaN stays one
// through 2^y.
struct RowSum {
  float m = -FLT_MAX, s = 0.f, t = 0.f;

  __device__ __forceinline__ void add(float x, float k)
  {
    if (x > m) raise(x, k);
    const float y = (x - m) * k, p = pow2(y);
    s += p;
    t = fmaf(p, fmaxf(y, -1e4f), t);
  }
  __device__ __forceinline__ void raise(float to, float k)
  {
    const float d = fmaxf((m - to) * k, -1e4f), f = pow2(d);
    t = fmaf(s, d, t) * f;
    s *= f;
    m = to;
  }
};

// Logits as whole numbers in their order (-0 as 0); 0 stands for nothing, which -inf is here.
__device__ __forceinline__ uint32_t value_key(float x)
{
  const uint32_t b = __float_as_uint(x + 0.f);
  return x > -INFINITY ? (b & 0x80000000u ? ~b : b | 0x80000000u) : 0u;
}
// with the column behind it, the lower one the higher number among equals
__device__ __forceinline__ uint64_t rank_key(float x, uint32_t column)
{
  const uint32_t v = value_key(x);
  return v ? uint64_t(v) << 32 | ~column : 0u;
}
__device__ __forceinline__ uint32_t key_column(uint64_t key) { return ~uint32_t(key); }
__device__ __forceinline__ float key_value(uint64_t key)
{
  const uint32_t b = uint32_t(key >> 32);
  return __uint_as_float(b & 0x80000000u ? b & 0x7FFFFFFFu : ~b);
}

struct ScoreArgs {
  int vocab;
  int64_t stride;
  float scale;
  const int32_t* targets;
  int top_k;
  float *logprob, *entropy, *lse;
  int32_t* top_ids;
  float* top_logprobs;
};

constexpr int kBatch = 4;              // packs that a thread has in flight
constexpr int kMaxParts = 8;           // CTAs that share a row
constexpr int kMostWinners = 64, kMostCandidates = 1024;

struct TopScratch {
  uint64_t candidate[kMostCandidates];
  uint64_t best[kWarps];
  uint64_t top[GTK_MAX_TOP];  // of this CTA's part of the row, highest first, 0 where there is none
  int winner[kThreads];
  int winners, candidates;
};

// The top_k columns of packs [begin, end) and, for loose, of the elements outside the packs, to S.top.
// Each thread knows the highest element `best` of the packs that it has read (begin + thread, and every kThreads-th from
// there).  The top_k-th highest of those is a bound that at least top_k elements reach; threads whose best is below it
// hold none of the top.  So the packs of about top_k threads are read again (from L2) and what reaches the bound is
// ranked.  Where more threads than kMostWinners reach it, with equal numbers, the columns decide among those: the argument
// holds for (value, column) too.
template <class T>
__device__ __forceinline__ void select_top(const RowParts<T>& row, int begin, int end, bool loose, int top_k, float best, TopScratch& S)
{
  constexpr int E = Pack16<T>::kElems;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t mine = value_key(best);
  uint32_t bound      = 0;
#pragma unroll 1
  for (int bit = 31; bit >= Pack16<T>::kLowestBit; --bit) {
    const uint32_t higher = bound | 1u << bit;
    if (__syncthreads_count(mine >= higher) >= top_k) bound = higher;
  }
  uint64_t floor = uint64_t(bound) << 32;
  if (tid == 0) S.winners = S.candidates = 0;
  if (tid < top_k) S.top[tid] = 0;
  bool wins = mine >= max(bound, 1u);
  if (__syncthreads_count(wins) > kMostWinners && bound) {
    uint64_t key = 0;  // the thread's highest with its column
    if (mine >= bound)
      for (int p = begin + tid; p < end && !key; p += kThreads) {
        const T* x = row.x + row.pack_column(p);
        for (int j = 0; j < E && !key; ++j)
          if (gtk::to_float(x[j]) == best) key = rank_key(best, uint32_t(row.pack_column(p) + j));
      }
#pragma unroll 1
    for (int bit = 31; bit >= 0; --bit) {
      const uint64_t higher = floor | 1u << bit;
      if (__syncthreads_count(key >= higher) >= top_k) floor = higher;
    }
    wins = key >= floor;
  }
  if (wins) S.winner[atomicAdd(&S.winners, 1)] = tid;
  __syncthreads();
  const int each = (end - begin + kThreads - 1) / kThreads, pairs = S.winners * each;  // packs of the winners
  auto offer = [&](uint64_t key) {
    if (key < max(floor, uint64_t(1))) return;
    const int at = atomicAdd(&S.candidates, 1);
    if (at < kMostCandidates) S.candidate[at] = key;
  };
  const int loose_count = loose ? row.head + row.tail : 0;
  for (int i = tid; i < pairs; i += kThreads) {
    const int p = begin + S.winner[i / each] + i % each * kThreads;
    if (p >= end) continue;
    const uint4 raw = __ldg(row.pack(p));
    const T* x      = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int j = 0; j < E; ++j) offer(rank_key(gtk::to_float(x[j]), uint32_t(row.pack_column(p) + j)));
  }
  if (tid < loose_count) offer(rank_key(gtk::to_float(row.x[row.loose_column(tid)]), uint32_t(row.loose_column(tid))));
  __syncthreads();
  const int n = S.candidates;
  if (n <= kMostCandidates) {
    for (int i = tid; i < n; i += kThreads) {
      const uint64_t key = S.candidate[i];
      int above          = 0;
      for (int j = 0; j < n; ++j) above += S.candidate[j] > key;
      if (above < top_k) S.top[above] = key;
    }
  } else {  // few threads own many of the highest: one after the other
    uint64_t below = ~uint64_t(0);
    for (int r = 0; r < top_k; ++r) {
      uint64_t high = 0;
      for (int i = tid; i < pairs; i += kThreads) {
        const int p = begin + S.winner[i / each] + i % each * kThreads;
        if (p >= end) continue;
        const T* x = row.x + row.pack_column(p);
        for (int j = 0; j < E; ++j) {
          const uint64_t key = rank_key(gtk::to_float(x[j]), uint32_t(row.pack_column(p) + j));
          if (key < below) high = max(high, key);
        }
      }
      if (tid < loose_count) {
        const uint64_t key = rank_key(gtk::to_float(row.x[row.loose_column(tid)]), uint32_t(row.loose_column(tid)));
        if (key < below) high = max(high, key);
      }
#pragma unroll
      for (int d = 16; d; d >>= 1) high = max(high, uint64_t(__shfl_xor_sync(0xFFFFFFFFu, high, d)));
      if (lane == 0) S.best[warp] = high;
      __syncthreads();
      for (int w = 0; w < kWarps; ++w) high = max(high, S.best[w]);
      __syncthreads();
      if (tid == 0) S.top[r] = high;
      below = high;
    }
  }
  __syncthreads();
}

struct NoScratch {};

// A row's CTAs (a cluster when there are several) each stream their share of its packs once.
template <class T, bool ENTROPY, bool TOP>
__global__ void __launch_bounds__(kThreads) k_token_logprobs(const T* __restrict__ logits, const ScoreArgs a, int parts)
{
  namespace cg = cooperative_groups;
  constexpr int E = Pack16<T>::kElems;
  __shared__ float s_m[kWarps];
  __shared__ float s_s[kWarps], s_t[kWarps];
  __shared__ RowSum s_part;  // of this CTA, read by the row's first
  __shared__ typename std::conditional<TOP, TopScratch, NoScratch>::type s_top;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t r = blockIdx.x / unsigned(parts);
  const int part  = int(blockIdx.x % unsigned(parts));
  const RowParts<T> row(logits + r * a.stride, a.vocab);
  const int share = (row.packs + parts - 1) / parts;
  const int begin = min(row.packs, part * share), end = min(row.packs, begin + share);
  const float k   = a.scale * kLog2e;
  int target      = -1;
  float at_target = 0.f;
  if (tid == 0 && part == 0 && a.logprob) {
    target = __ldg(a.targets + r);
    if (target >= 0 && target < a.vocab) at_target = gtk::to_float(row.x[target]);
  }
  RowSum sum;
  if (part == 0 && tid < row.head + row.tail) sum.add(gtk::to_float(row.x[row.loose_column(tid)]), k);
  Two s2(sum.s, 0.f), t2(sum.t, 0.f);
  const Two k2(k, k);
  float best = -INFINITY;
  for (int p0 = begin + tid; p0 < end; p0 += kBatch * kThreads) {
    uint4 raw[kBatch];
#pragma unroll
    for (int q = 0; q < kBatch; ++q) {
      constexpr uint32_t w = Pack16<T>::kMinusInf;
      raw[q] = p0 + q * kThreads < end ? __ldg(row.pack(p0 + q * kThreads)) : make_uint4(w, w, w, w);
    }
    const float high = Pack16<T>::highest(raw);
    if (high > best) {
      best = high;
      if (high > sum.m) {
        const float d = fmaxf((sum.m - high) * k, -1e4f), f = pow2(d);
        const Two f2(f, f);
        if (ENTROPY) t2 = fma2(s2, Two(d, d), t2) * f2;
        s2    = s2 * f2;
        sum.m = high;
      }
    }
    const Two m2(-sum.m, -sum.m);
#pragma unroll
    for (int q = 0; q < kBatch; ++q) {
      Two x[E / 2];
      Pack16<T>::pairs(raw[q], x);
#pragma unroll
      for (int j = 0; j < E / 2; ++j) {
        float y0, y1;
        ((x[j] + m2) * k2).get(y0, y1);
        const Two p(pow2(y0), pow2(y1));
        s2 = s2 + p;
        if (ENTROPY) t2 = fma2(p, Two(fmaxf(y0, -1e4f), fmaxf(y1, -1e4f)), t2);
      }
    }
  }
  {
    float lo, hi;
    s2.get(lo, hi);
    sum.s = lo + hi;
    t2.get(lo, hi);
    sum.t = lo + hi;
  }
  // the CTA's maximum, then its sums relative to that
  float m = sum.m;
#pragma unroll
  for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, d));
  sum.raise(m, k);
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    sum.s += __shfl_xor_sync(0xFFFFFFFFu, sum.s, d);
    if (ENTROPY) sum.t += __shfl_xor_sync(0xFFFFFFFFu, sum.t, d);
  }
  if (lane == 0) s_m[warp] = sum.m, s_s[warp] = sum.s, s_t[warp] = sum.t;
  __syncthreads();
  m = s_m[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) m = fmaxf(m, s_m[w]);
  RowSum all;
  all.m = m;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    RowSum o;
    o.m = s_m[w], o.s = s_s[w], o.t = s_t[w];
    o.raise(m, k);
    all.s += o.s;
    all.t += o.t;
  }
  if constexpr (TOP) select_top(row, begin, end, part == 0, a.top_k, best, s_top);
  if (parts > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    if (tid == 0) s_part = all;
    cluster.sync();
    if (part == 0) {
      for (int c = 1; c < parts; ++c) m = fmaxf(m, cluster.map_shared_rank(&s_part, c)->m);
      RowSum joined;
      joined.m = m;
      for (int c = 0; c < parts; ++c) {
        RowSum o = *cluster.map_shared_rank(&s_part, c);
        o.raise(m, k);
        joined.s += o.s;
        joined.t += o.t;
      }
      all = joined;
      if constexpr (TOP) {
        // at most kMaxParts * GTK_MAX_TOP = kThreads keys, one per thread
        uint64_t key = 0;
        if (tid < parts * a.top_k) key = cluster.map_shared_rank(&s_top, tid / a.top_k)->top[tid % a.top_k];
        s_top.candidate[tid] = key;
        __syncthreads();
        if (tid < a.top_k) s_top.top[tid] = 0;
        __syncthreads();
        int above = 0;
        for (int j = 0; j < parts * a.top_k; ++j) above += s_top.candidate[j] > key;
        if (key && above < a.top_k) s_top.top[above] = key;
        __syncthreads();
      }
    }
    cluster.sync();  // nobody leaves while its shared memory is read
    if (part != 0) return;
  }
  const float log_sum = logf(all.s);  // -inf: nothing allowed, NaN: no distribution
  const bool none = all.s == 0.f, broken = isnan(all.s);
  const float nan = __int_as_float(0x7FC00000);
  if (tid == 0) {
    if (a.logprob) {
      float lp = target < 0 ? 0.f : nan;
      if (target >= 0 && target < a.vocab && !broken) lp = none ? -INFINITY : (at_target - all.m) * a.scale - log_sum;
      a.logprob[r] = lp;
    }
    if (a.entropy) a.entropy[r] = none ? 0.f : broken ? nan : fmaxf(log_sum - kLn2 * all.t / all.s, 0.f);
    if (a.lse) a.lse[r] = none ? -INFINITY : broken ? nan : fmaf(all.m, a.scale, log_sum);
  }
  if constexpr (TOP) {
    if (tid < a.top_k) {
      const uint64_t key = broken ? 0 : s_top.top[tid];
      if (a.top_ids) a.top_ids[r * a.top_k + tid] = key ? int32_t(key_column(key)) : -1;
      if (a.top_logprobs) a.top_logprobs[r * a.top_k + tid] = broken ? nan : key ? (key_value(key) - all.m) * a.scale - log_sum : -INFINITY;
    }
  }
}

// How many CTAs share a row: few rows are split until the GPU has a few CTAs per SM.
int row_parts(int64_t rows, int64_t bytes, int sm_count)
{
  int parts = 1;
  while (parts < kMaxParts && rows * parts * 2 <= int64_t(sm_count) * 2 && bytes / (parts * 2) >= 8192) parts *= 2;
  return parts;
}

template <class T, bool ENTROPY, bool TOP>
cudaError_t launch_logprobs(const gtk::HandleView& v, const void* logits, int64_t n_rows, const ScoreArgs& a)
{
  const int parts = row_parts(n_rows, int64_t(a.vocab) * int64_t(sizeof(T)), v.sm_count);
  return gtk::launch_clusters(k_token_logprobs<T, ENTROPY, TOP>, dim3(unsigned(n_rows * parts)), dim3(kThreads), parts, v.stream,
                              static_cast<const T*>(logits), a, parts);
}

struct ScoreGradArgs {
  int vocab;
  int64_t stride, grad_stride;
  float scale;
  const int32_t* targets;
  const float *lse, *entropy, *grad_logprob, *grad_entropy;
};

// d = scale * (g * ([j == t] - p) - e * p * (log p + H)), log p = scale * x - lse.  Every element is read and written once, by
// the same thread, so that grad may be logits.  A row's elements are shared by `parts` CTAs.
template <class T, bool ENTROPY>
struct GradRow {
  float scale, lse, g, e, H;
  int t;
  bool nothing;
  __device__ GradRow(const ScoreGradArgs& a, int64_t r) : scale(a.scale)
  {
    t   = a.grad_logprob ? __ldg(a.targets + r) : -1;
    if (t >= a.vocab) t = -1;
    g   = t >= 0 ? __ldg(a.grad_logprob + r) * -scale : 0.f;
    e   = ENTROPY ? __ldg(a.grad_entropy + r) * -scale : 0.f;
    H   = ENTROPY ? __ldg(a.entropy + r) : 0.f;
    lse = __ldg(a.lse + r);
    nothing = lse == -INFINITY || (t < 0 && !ENTROPY);
  }
  __device__ __forceinline__ float of(float x, int column) const
  {
    const float z = fmaf(x, scale, -lse), p = pow2(z * kLog2e);
    const float d = p * (ENTROPY ? fmaf(e, fmaxf(z, -1e4f) + H, g) : g);
    return column == t ? d - g : d;
  }
};

template <class T, bool ENTROPY>
__global__ void __launch_bounds__(kThreads) k_token_logprobs_grad(const T* logits, T* grad, const ScoreGradArgs a, int parts)
{
  constexpr int E = Pack16<T>::kElems;
  const int64_t r = blockIdx.x / unsigned(parts);
  const int part  = int(blockIdx.x % unsigned(parts)), tid = threadIdx.x;
  const RowParts<T> row(logits + r * a.stride, a.vocab);
  T* to = grad + r * a.grad_stride;
  const GradRow<T, ENTROPY> R(a, r);
  if (part == 0 && tid < row.head + row.tail) {
    const int c = row.loose_column(tid);
    to[c]       = gtk::from_float<T>(R.nothing ? 0.f : R.of(gtk::to_float(row.x[c]), c));
  }
  const int share = (row.packs + parts - 1) / parts;
  const int begin = part * share, end = min(row.packs, begin + share);
  uint4* out = reinterpret_cast<uint4*>(to + row.head);
  if (R.nothing) {
    for (int p = begin + tid; p < end; p += kThreads) out[p] = make_uint4(0u, 0u, 0u, 0u);
    return;
  }
  const Two scale2(R.scale, R.scale), lse2(-R.lse, -R.lse), log2e2(kLog2e, kLog2e), g2(R.g, R.g), e2(R.e, R.e), H2(R.H, R.H);
  for (int p0 = begin + tid; p0 < end; p0 += kBatch * kThreads) {
    uint4 raw[kBatch];
#pragma unroll
    for (int q = 0; q < kBatch; ++q)
      if (p0 + q * kThreads < end) raw[q] = *row.pack(p0 + q * kThreads);
#pragma unroll
    for (int q = 0; q < kBatch; ++q) {
      const int p = p0 + q * kThreads;
      if (p >= end) break;
      Two x[E / 2];
      Pack16<T>::pairs(raw[q], x);
      gtk::Pack<T, E> y;
      const int at = R.t - row.pack_column(p);
#pragma unroll
      for (int j = 0; j < E / 2; ++j) {
        const Two z = fma2(x[j], scale2, lse2);
        float y0, y1;
        (z * log2e2).get(y0, y1);
        const Two p2(pow2(y0), pow2(y1));
        Two d;
        if (ENTROPY) {
          float z0, z1;
          z.get(z0, z1);
          d = p2 * fma2(e2, Two(fmaxf(z0, -1e4f), fmaxf(z1, -1e4f)) + H2, g2);
        } else {
          d = p2 * g2;
        }
        float d0, d1;
        d.get(d0, d1);
        y.e[2 * j]     = gtk::from_float<T>(d0);
        y.e[2 * j + 1] = gtk::from_float<T>(d1);
      }
      if (uint32_t(at) < uint32_t(E)) {  // the target's own element
        const float d = R.of(gtk::to_float(row.x[R.t]), R.t);
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (j == at) y.e[j] = gtk::from_float<T>(d);
      }
      out[p] = *reinterpret_cast<const uint4*>(&y);
    }
  }
}

// The same where logits and gradient lie differently against 16-byte boundaries: element by element.
template <class T, bool ENTROPY>
__global__ void __launch_bounds__(kThreads) k_token_logprobs_grad_plain(const T* logits, T* grad, const ScoreGradArgs a, int parts)
{
  const int64_t r = blockIdx.x / unsigned(parts);
  const int part  = int(blockIdx.x % unsigned(parts));
  const T* x      = logits + r * a.stride;
  T* to           = grad + r * a.grad_stride;
  const GradRow<T, ENTROPY> R(a, r);
  for (int64_t c = part * kThreads + threadIdx.x; c < a.vocab; c += int64_t(parts) * kThreads)
    to[c] = gtk::from_float<T>(R.nothing ? 0.f : R.of(gtk::to_float(x[c]), int(c)));
}

template <class T, bool ENTROPY>
cudaError_t launch_logprobs_grad(const gtk::HandleView& v, const void* logits, void* grad, int64_t n_rows, const ScoreGradArgs& a)
{
  const bool alike = (reinterpret_cast<uintptr_t>(logits) - reinterpret_cast<uintptr_t>(grad)) % 16 == 0 &&
                     (n_rows == 1 || (a.stride - a.grad_stride) * int64_t(sizeof(T)) % 16 == 0);
  const int64_t batches = (a.vocab + kBatch * kThreads * Pack16<T>::kElems - 1) / (kBatch * kThreads * Pack16<T>::kElems);
  const int parts = int(std::max<int64_t>(1, std::min<int64_t>(batches, int64_t(v.sm_count) * 8 / n_rows)));
  return gtk::launch(alike ? k_token_logprobs_grad<T, ENTROPY> : k_token_logprobs_grad_plain<T, ENTROPY>, dim3(unsigned(n_rows * parts)),
                     dim3(kThreads), 0, v.stream, static_cast<const T*>(logits), static_cast<T*>(grad), a, parts);
}

constexpr int64_t kMaxVocab = int64_t(1) << 30, kMaxRows = (int64_t(1) << 31) - 1;

gtk::Refusal refuse_sizes(int type, int64_t n_rows, int64_t vocab, int64_t stride, float scale)
{
  if (!gtk::known_type(type)) return "unknown element type";
  if (n_rows < 0 || vocab <= 0 || stride < 0) return "n_rows and stride must be >= 0, vocab > 0";
  if (n_rows > kMaxRows || vocab > kMaxVocab) return "n_rows of 2^31 and more, or vocab beyond 2^30";
  if (!(scale > 0.f) || std::isinf(scale)) return "scale must be a finite number > 0";
  return nullptr;
}

bool all_aligned4(std::initializer_list<const void*> ps)
{
  for (const void* p : ps)
    if (!gtk::aligned_to(p, 4)) return false;
  return true;
}

}  // namespace

extern "C" GTK_API int gtk_token_logprobs(gtk_tokenizer* h, const void* d_logits, int type, int64_t n_rows, int64_t vocab, int64_t stride,
                                          float scale, const int32_t* d_targets, int top_k, float* d_logprob, float* d_entropy,
                                          float* d_lse, int32_t* d_top_ids, float* d_top_logprobs)
{
  auto check = [&]() -> gtk::Refusal {
    if (const gtk::Refusal why = refuse_sizes(type, n_rows, vocab, stride, scale)) return why;
    if (top_k < 0 || top_k > GTK_MAX_TOP) return "top_k must be 0 .. GTK_MAX_TOP";
    if ((top_k > 0) != (d_top_ids || d_top_logprobs)) return "top_k and the buffers for the alternatives do not go together";
    if (n_rows == 0) return nullptr;
    if (!d_logits || (d_logprob && !d_targets)) return "null device pointer";
    if (!gtk::aligned_to(d_logits, gtk::element_size(type)) ||
        !all_aligned4({d_targets, d_logprob, d_entropy, d_lse, d_top_ids, d_top_logprobs}))
      return "a device pointer is not aligned to its elements";
    return nullptr;
  };
  return gtk::run_operator(h, check, [&](const gtk::HandleView& v) -> cudaError_t {
    if (n_rows == 0) return cudaSuccess;
    const ScoreArgs a{int(vocab), stride, scale, d_targets, top_k, d_logprob, d_entropy, d_lse, d_top_ids, d_top_logprobs};
    return gtk::with_type(type, [&](auto x) {
      using T = decltype(x);
      auto f  = top_k ? (d_entropy ? launch_logprobs<T, true, true> : launch_logprobs<T, false, true>)
                      : (d_entropy ? launch_logprobs<T, true, false> : launch_logprobs<T, false, false>);
      return f(v, d_logits, n_rows, a);
    });
  });
}

extern "C" GTK_API int gtk_token_logprobs_grad(gtk_tokenizer* h, const void* d_logits, int type, int64_t n_rows, int64_t vocab,
                                               int64_t stride, float scale, const int32_t* d_targets, const float* d_lse,
                                               const float* d_entropy, const float* d_grad_logprob, const float* d_grad_entropy,
                                               void* d_grad_logits, int64_t grad_stride)
{
  auto check = [&]() -> gtk::Refusal {
    if (const gtk::Refusal why = refuse_sizes(type, n_rows, vocab, stride, scale)) return why;
    if (grad_stride < vocab) return "grad_stride must be >= vocab";
    if (n_rows == 0) return nullptr;
    if (!d_logits || !d_grad_logits || !d_lse || (d_grad_logprob && !d_targets) || (d_grad_entropy && !d_entropy))
      return "null device pointer";
    if (d_logits == d_grad_logits && stride != grad_stride) return "in place, both strides must be the same";
    if (!gtk::aligned_to(d_logits, gtk::element_size(type)) || !gtk::aligned_to(d_grad_logits, gtk::element_size(type)) ||
        !all_aligned4({d_targets, d_lse, d_entropy, d_grad_logprob, d_grad_entropy}))
      return "a device pointer is not aligned to its elements";
    return nullptr;
  };
  return gtk::run_operator(h, check, [&](const gtk::HandleView& v) -> cudaError_t {
    if (n_rows == 0) return cudaSuccess;
    const ScoreGradArgs a{int(vocab), stride, grad_stride, scale, d_targets, d_lse, d_entropy, d_grad_logprob, d_grad_entropy};
    return gtk::with_type(type, [&](auto x) {
      using T = decltype(x);
      auto f  = d_grad_entropy ? launch_logprobs_grad<T, true> : launch_logprobs_grad<T, false>;
      return f(v, d_logits, d_grad_logits, n_rows, a);
    });
  });
}
