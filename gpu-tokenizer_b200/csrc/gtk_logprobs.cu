// gtk_logprobs.cu -- log probabilities of given tokens, entropy and top alternatives of rows of logits, and the
// gradient of the first two.
//
// With k = scale * log2(e), m a row's maximum and y_j = (x_j - m) k:  S = sum 2^y_j,  lse = scale m + ln S,
// log p_t = scale (x_t - m) - ln S,  H = ln S - ln 2 (sum 2^y_j y_j) / S.  Both sums are formed in one pass with the maximum so
// far and moved when that rises.  dx_j = scale (g ([j = t] - p_j) - e p_j (log p_j + H)) needs lse and H only, where 32 bits of lse
// still hold ln S.
//
// All of it is bound by memory, and just so: an element costs one exponential (16 a clock and SM) and some four further
// instructions.  Measured against a copy (6.45 TB/s):
//   8192 rows of 50257 bf16     130 us, 98 %, with 20 alternatives 167; back to back for a second 150 us: at 1000 W the SMs run at
//                               1.6 GHz, and 412 M exponentials alone then take 108 us
//   4096 rows of the same, f32  121 us, 105 %, with entropy 123; with 20 alternatives 154
//   gradient of 8192 rows       259 us, 98 %
//   one row                     4 us without alternatives, 8.4 with 20 of them and entropy: phases that wait for each other
#include <cooperative_groups.h>

#include <cfloat>
#include <cmath>
#include <initializer_list>
#include <type_traits>

#include "gtk_checked.cuh"
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

// 16 bytes of a row: its elements as pairs of 32-bit floats, and their maxima (NaN only where all are).
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
  // maxima: one of the whole pack
  using Max = float;
  static constexpr int kHalves = 1;
  static __device__ __forceinline__ Max lowest() { return -INFINITY; }
  static __device__ __forceinline__ Max highest(const uint4& r)
  {
    return fmaxf(fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)), fmaxf(__uint_as_float(r.z), __uint_as_float(r.w)));
  }
  static __device__ __forceinline__ Max higher(Max a, Max b) { return fmaxf(a, b); }
  static __device__ __forceinline__ float of(Max m, int) { return m; }
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
  // maxima: one of the even elements, one of the odd ones
  using Max = T2;
  static constexpr int kHalves = 2;
  static __device__ __forceinline__ Max highest(const uint4& r) { return __hmax2(__hmax2(as(r.x), as(r.y)), __hmax2(as(r.z), as(r.w))); }
  static __device__ __forceinline__ Max higher(Max a, Max b) { return __hmax2(a, b); }
  static __device__ __forceinline__ float of(Max m, int half)
  {
    const float2 f = both(m);
    return half ? f.y : f.x;
  }
};
template <>
__device__ __forceinline__ float2 Pack16Half<__nv_bfloat16, __nv_bfloat162>::both(__nv_bfloat162 w) { return __bfloat1622float2(w); }
template <>
__device__ __forceinline__ float2 Pack16Half<__half, __half2>::both(__half2 w) { return __half22float2(w); }
template <>
struct Pack16<__nv_bfloat16> : Pack16Half<__nv_bfloat16, __nv_bfloat162> {
  static __device__ __forceinline__ Max lowest() { return __float2bfloat162_rn(-INFINITY); }
  static constexpr uint32_t kMinusInf = 0xFF80FF80u;
  static constexpr int kLowestBit     = 16;
};
template <>
struct Pack16<__half> : Pack16Half<__half, __half2> {
  static __device__ __forceinline__ Max lowest() { return __float2half2_rn(-INFINITY); }
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
// Sets that are read again and keys that are ranked at most; beyond that the way through ties and crowds is taken.  The keys of
// all parts fit into one CTA's list.
constexpr int kMostSets = 64, kMostKeys = 512, kMostKeysOfPart = kMostKeys / kMaxParts;
static_assert(kMostKeysOfPart >= GTK_MAX_TOP, "a part's own top_k fit into its share");

struct TopScratch {
  uint64_t key[kMostKeys];
  uint64_t best[kWarps];
  int set[kThreads];  // thread << 8 | q << 4 | half
  int sets, keys, crowded;
  uint32_t bound;
};

// The highest value_key that at least `wanted` of the CTA's threads reach with `mine`, or a lower one that exactly so many
// reach; 0 where fewer threads have any.
template <class T>
__device__ __forceinline__ uint32_t find_bound(uint32_t mine, int wanted)
{
  uint32_t bound = 0;
#pragma unroll 1
  for (int bit = 31; bit >= Pack16<T>::kLowestBit; --bit) {
    const uint32_t higher = bound | 1u << bit;
    const int reach       = __syncthreads_count(mine >= higher);
    if (reach >= wanted) bound = higher;
    if (reach == wanted) break;
  }
  // the low bits that are the same in all numbers of the type: ones below a negative one, see value_key
  if (bound && !(bound & 0x80000000u)) bound |= (1u << Pack16<T>::kLowestBit) - 1u;
  return bound;
}

// Leaves in S.key[0 .. S.keys), in any order, keys of packs [begin, end) and, for loose, of the elements outside the packs,
// at most `most` of them, among which are all of the top_k highest that reach the bound.
// A thread has read packs begin + thread, and every blockDim-th from there; of those that were q-th in their batch it knows the
// highest elements best[q], and `mine` is the value_key of its highest of all.  Only packs of sets (a thread, a q, a half of the
// elements) whose highest reaches the bound are read again, from L2.  That is about top_k sets, as long as numbers differ, and then
// collect_few has answered already: this is the way of rows with ties and crowds.
// Where more than kMostSets reach it, the threads whose highest (by value, then by column) are the top_k highest of their
// kind take the sets' place: what the others hold comes behind those.
template <class T>
__device__ __forceinline__ void collect_keys(const RowParts<T>& row, int begin, int end, bool loose, int top_k, int most, uint32_t bound, uint32_t mine,
                                             const typename Pack16<T>::Max (&best)[kBatch], TopScratch& S)
{
  using P         = Pack16<T>;
  constexpr int E = P::kElems;
  const int tid = threadIdx.x, threads = blockDim.x, warp = tid >> 5, lane = tid & 31;
  uint64_t floor = uint64_t(bound) << 32;
  __syncthreads();  // all have seen collect_few's keys
  if (tid == 0) S.sets = S.keys = 0;
  __syncthreads();
  if (mine && mine >= bound) {
#pragma unroll
    for (int q = 0; q < kBatch; ++q)
#pragma unroll
      for (int half = 0; half < P::kHalves; ++half) {
        const uint32_t key = value_key(P::of(best[q], half));
        if (key && key >= bound) {
          const int at = atomicAdd(&S.sets, 1);
          if (at < kMostSets && GTK_IN(at, kThreads, 300)) S.set[at] = tid << 8 | q << 4 | half;
        }
      }
  }
  __syncthreads();
  const bool by_set = S.sets <= kMostSets;
  if (!by_set) {
    bound        = max(bound, find_bound<T>(mine, top_k));
    floor        = uint64_t(bound) << 32;
    uint64_t key = 0;  // the thread's highest with its column
    if (mine && mine >= bound)
      for (int p = begin + tid; p < end && !key; p += threads) {
        const T* x = row.x + row.pack_column(p);
        for (int j = 0; j < E && !key; ++j)
          if (value_key(gtk::to_float(x[j])) == mine) key = rank_key(gtk::to_float(x[j]), uint32_t(row.pack_column(p) + j));
      }
    if (__syncthreads_count(key != 0) >= top_k) {
#pragma unroll 1
      for (int bit = 31; bit >= 0; --bit) {
        const uint64_t higher = floor | 1u << bit;
        if (__syncthreads_count(key >= higher) >= top_k) floor = higher;
      }
    }
    if (tid == 0) S.sets = 0;
    __syncthreads();
    if (key && key >= floor) {
      const int at = atomicAdd(&S.sets, 1);
      if (GTK_IN(at, kThreads, 301)) S.set[at] = tid << 8;
    }
    __syncthreads();
  }
  const int step = by_set ? kBatch * threads : threads;
  const uint32_t each = uint32_t(max(1, (end - begin + step - 1) / step)), packs = uint32_t(S.sets) * each;
  const float reach = bound ? key_value(floor) : -INFINITY;
  // f(key) for the elements of the i-th pack of the sets that reach the bound
  auto each_key = [&](uint32_t i, auto&& f) {
    const uint32_t at = i / each;
    if (!GTK_IN(at, kThreads, 302)) return;
    const int w = S.set[at], p = begin + (w >> 8) + (w >> 4 & 15) * threads + int(i - at * each) * step;
    if (p >= end || !GTK_IN(p, row.packs, 303)) return;
    const uint4 raw = __ldg(row.pack(p));
    const T* x      = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int j = 0; j < E; ++j)
      if (gtk::to_float(x[j]) >= reach && (!by_set || P::kHalves == 1 || (j & 1) == (w & 1))) f(rank_key(gtk::to_float(x[j]), uint32_t(row.pack_column(p) + j)));
  };
  auto each_loose = [&](auto&& f) {
    if (loose && tid < row.head + row.tail) f(rank_key(gtk::to_float(row.x[row.loose_column(tid)]), uint32_t(row.loose_column(tid))));
  };
  auto offer = [&](uint64_t key) {
    if (key == 0 || key < floor) return;
    const int at = atomicAdd(&S.keys, 1);
    if (at < most && GTK_IN(at, kMostKeys, 304)) S.key[at] = key;
  };
#pragma unroll 1
  for (uint32_t i = tid; i < packs; i += threads) each_key(i, offer);
  each_loose(offer);
  __syncthreads();
  if (S.keys <= most) return;
  // few sets hold many of the highest: one after the other
  uint64_t below = ~uint64_t(0);
  int found      = 0;
#pragma unroll 1
  for (; found < top_k; ++found) {
    uint64_t high = 0;
    auto look     = [&](uint64_t key) {
      if (key < below) high = max(high, key);
    };
#pragma unroll 1
    for (uint32_t i = tid; i < packs; i += threads) each_key(i, look);
    each_loose(look);
#pragma unroll
    for (int d = 16; d; d >>= 1) high = max(high, uint64_t(__shfl_xor_sync(0xFFFFFFFFu, high, d)));
    if (lane == 0) S.best[warp] = high;
    __syncthreads();
    for (int w = 0; w < threads / 32; ++w) high = max(high, S.best[w]);
    __syncthreads();
    if (high == 0) break;
    if (tid == 0 && GTK_IN(found, kMostKeysOfPart, 305)) S.key[found] = high;
    below = high;
  }
  if (tid == 0) S.keys = found;
  __syncthreads();
}

// The same where the sets that reach the bound are few in each warp, which then reads its own ones again and waits for no other
// (with the list of all warps at once one row took 9.1 us, now 8.4, 8192 rows of 50257 bf16 with 20 alternatives 171, now 167): false
// where they are not, or hold too many keys.  S.keys and S.crowded are 0 before.
template <int LOOK, class T>
__device__ __forceinline__ bool collect_few(const RowParts<T>& row, int begin, int end, bool loose, int most, uint32_t bound,
                                            const typename Pack16<T>::Max (&best)[kBatch], TopScratch& S)
{
  using P         = Pack16<T>;
  constexpr int E = P::kElems;
  const int tid = threadIdx.x, threads = blockDim.x, warp = tid >> 5, lane = tid & 31;
  const int room     = kThreads * 32 / threads;
  int* const set     = S.set + warp * room;
  const uint64_t floor = uint64_t(bound) << 32;
  const float reach  = bound ? key_value(floor) : -FLT_MAX;  // -inf is no alternative
  auto offer = [&](float x, int column) {
    const int at = atomicAdd(&S.keys, 1);
    if (at < most && GTK_IN(at, kMostKeys, 306)) S.key[at] = rank_key(x, uint32_t(column));
  };
  int sets = 0;
#pragma unroll
  for (int q = 0; q < kBatch; ++q)
#pragma unroll
    for (int half = 0; half < P::kHalves; ++half) {
      const bool reaches  = P::of(best[q], half) >= reach;
      const uint32_t some = __ballot_sync(0xFFFFFFFFu, reaches);
      const int at        = sets + __popc(some & ((1u << lane) - 1u));
      if (reaches && at < room && GTK_IN(set + at - S.set, kThreads, 307)) set[at] = tid << 8 | q << 4 | half;
      sets += __popc(some);
    }
  __syncwarp();
  if (sets > room) {
    if (lane == 0) S.crowded = 1;
  } else {
    // as many threads to the packs of a set as there are for all, and each looks at LOOK packs at a time
    const int share_log2 = sets > 1 ? max(0, 5 - (32 - __clz(sets - 1))) : 5, stride = kBatch * threads << share_log2;
    auto look            = [&](const uint4& raw, int p, int half) {
      const T* x = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (gtk::to_float(x[j]) >= reach && (P::kHalves == 1 || (j & 1) == half)) offer(gtk::to_float(x[j]), row.pack_column(p) + j);
    };
    for (int i = lane >> share_log2; i < sets; i += 32 >> share_log2) {
      if (!GTK_IN(set + i - S.set, kThreads, 308)) break;
      const int w = set[i];
      for (int p = begin + (w >> 8) + ((w >> 4 & 15) + kBatch * (lane & ((1 << share_log2) - 1))) * threads; p < end; p += LOOK * stride) {
        uint4 raw[LOOK];
#pragma unroll
        for (int q = 0; q < LOOK; ++q)
          if (GTK_IN(p + q * stride < end ? p + q * stride : p, row.packs, 309)) raw[q] = __ldg(row.pack(p + q * stride < end ? p + q * stride : p));
#pragma unroll
        for (int q = 0; q < LOOK; ++q)
          if (p + q * stride < end) look(raw[q], p + q * stride, w & 1);
      }
    }
  }
  if (loose && tid < row.head + row.tail) {
    const float x = gtk::to_float(row.x[row.loose_column(tid)]);
    if (x >= reach) offer(x, row.loose_column(tid));
  }
  __syncthreads();
  return !S.crowded && S.keys <= most;
}

// The top_k highest of S.key[0 .. n), each to put(place, key) by one thread, places that remain with key 0.
template <class Put>
__device__ __forceinline__ void rank_keys(const TopScratch& S, int n, int top_k, Put&& put)
{
#pragma unroll 1
  for (int i = threadIdx.x; i < max(n, top_k); i += blockDim.x) {
    const uint64_t key = i < n && GTK_IN(i, kMostKeys, 310) ? S.key[i] : 0u;
    int above          = i < n ? 0 : i;  // nothing comes behind all that there is
    if (i < n)
#pragma unroll 4
      for (int j = 0; j < n; ++j) above += S.key[j] > key;
    if (above < top_k && GTK_IN(above, top_k, 311)) put(above, key);
  }
}

struct NoScratch {};

// A row is streamed once, by a CTA of 64 .. kThreads threads or by a cluster of such CTAs that take a share of its packs each.
// What keeps memory busy here is many CTAs at different places of their rows, so registers are few and a CTA ends with its
// row.  8192 rows of 50257 bf16 took 186 us with CTAs that stay and have the next row's first batch in registers, 147 us with a
// ring of batches in shared memory that runs on into the next row, 138 us as it is but with 256 threads, 130 us with 128.
// Alternatives cost a row its end: the bound and the packs that are read again are waits one after another, in which the CTA asks
// for nothing else (8192 rows of 8192 bf16: 29 us without, 37 with one, 47 with 20).
// CTAs of kThreads per SM that registers are shared out for.  With 4 and 5, us: 8192 rows of 50257 bf16 130 and 133, 4096 of them with
// entropy 80 and 76, with entropy and five alternatives 95 and 90; 999 of f32 with these 40 and 45, 8192 rows of 8192 f32 with
// five alternatives 64 and 60.  fp16, whose conversions want more registers: 4096 rows of 50257 with entropy 72.5 and 73.6, with
// entropy and 20 alternatives 98.6 and 97.8, with 20 alternatives alone 96.7 and 101 (spilled).  Parts of rows, of which an SM has two
// at most: 74 rows of 50257 fp16 with entropy 10.4 and 12.4, with 20 alternatives too 14.4 and 16.4, bf16 14.5 and 16.4.
template <class T, bool ENTROPY, bool TOP, bool SPLIT>
constexpr int kResident =
    !SPLIT && (sizeof(T) == 4 ? TOP && !ENTROPY : ENTROPY || (TOP && std::is_same<T, __nv_bfloat16>::value)) ? 5 : 4;

// Packs that a thread reads again at a time.  8192 rows of 50257 bf16 with 20 alternatives: 167 us with two, 170 with one, 182 with four, for
// want of registers; 4096 of fp16 111 with two, 115 with four.  Where there are more of them, 4096 rows of f32 with entropy too: 154 with
// four, 162 with two; 16 rows of f32 in parts: 14.4 and 16.4.
template <class T, bool ENTROPY, bool SPLIT>
constexpr int kLookAgain = SPLIT || (sizeof(T) == 4 && ENTROPY) ? 4 : 2;

template <class T, bool ENTROPY, bool TOP, bool SPLIT>
__global__ void __launch_bounds__(kThreads, kResident<T, ENTROPY, TOP, SPLIT>) k_token_logprobs(const T* __restrict__ logits, const ScoreArgs a, int n_parts)
{
  const int parts     = SPLIT ? n_parts : 1;
  constexpr int kLook = kLookAgain<T, ENTROPY, SPLIT>;
  namespace cg = cooperative_groups;
  using P         = Pack16<T>;
  constexpr int E = P::kElems;
  __shared__ float s_m[kWarps], s_s[kWarps], s_t[kWarps];
  __shared__ RowSum s_part;  // of this CTA, read by the row's first
  __shared__ typename std::conditional<TOP, TopScratch, NoScratch>::type s_top;
  const int tid = threadIdx.x, threads = blockDim.x, warps = threads >> 5, warp = tid >> 5, lane = tid & 31;
  const int64_t r = blockIdx.x / unsigned(parts);
  const int part  = int(blockIdx.x % unsigned(parts));
  const RowParts<T> row(logits + r * a.stride, a.vocab);
  const int share = (row.packs + parts - 1) / parts;
  const int begin = min(row.packs, part * share), end = min(row.packs, begin + share);
  const float k = a.scale * kLog2e, nan = __int_as_float(0x7FC00000);
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
  typename P::Max best[kBatch];
#pragma unroll
  for (int q = 0; q < kBatch; ++q) best[q] = P::lowest();
  auto take = [&](const uint4 (&raw)[kBatch]) {
    typename P::Max all = P::highest(raw[0]);
    if (TOP) best[0] = P::higher(best[0], all);
#pragma unroll
    for (int q = 1; q < kBatch; ++q) {
      const typename P::Max m = P::highest(raw[q]);
      if (TOP) best[q] = P::higher(best[q], m);
      all = P::higher(all, m);
    }
    const float high = P::kHalves == 2 ? fmaxf(P::of(all, 0), P::of(all, 1)) : P::of(all, 0);
    if (high > sum.m) {
      const float d = fmaxf((sum.m - high) * k, -1e4f), f = pow2(d);
      const Two f2(f, f);
      if (ENTROPY) t2 = fma2(s2, Two(d, d), t2) * f2;
      s2    = s2 * f2;
      sum.m = high;
    }
    const Two m2(-sum.m, -sum.m);
#pragma unroll
    for (int q = 0; q < kBatch; ++q) {
      Two x[E / 2];
      P::pairs(raw[q], x);
#pragma unroll
      for (int j = 0; j < E / 2; ++j) {
        float y0, y1;
        ((x[j] + m2) * k2).get(y0, y1);
        const Two p(pow2(y0), pow2(y1));
        s2 = s2 + p;
        if (ENTROPY) t2 = fma2(p, Two(fmaxf(y0, -1e4f), fmaxf(y1, -1e4f)), t2);
      }
    }
  };
  int p0 = begin + tid;
  // Whole batches by code of their own: 999 rows of f32 take 34 us, 41 with packs asked for one by one in all batches, 4096 of bf16
  // with alternatives 84 and 95.  Parts of a row have few batches, which would wait for both codes to come in (one row: 4.6 us
  // and 4.2).
  if constexpr (!SPLIT)
    for (; p0 < end - (kBatch - 1) * threads; p0 += kBatch * threads) {
      uint4 raw[kBatch];
#pragma unroll
      for (int q = 0; q < kBatch; ++q) raw[q] = __ldg(row.pack(p0 + q * threads));
      take(raw);
    }
  auto take_some = [&]() {
    uint4 raw[kBatch];
#pragma unroll
    for (int q = 0; q < kBatch; ++q) {
      constexpr uint32_t w = P::kMinusInf;
      raw[q] = p0 + q * threads < end ? __ldg(row.pack(p0 + q * threads)) : make_uint4(w, w, w, w);
    }
    take(raw);
  };
  if constexpr (SPLIT)
    for (; p0 < end; p0 += kBatch * threads) take_some();
  else if (p0 < end)
    take_some();
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
  if constexpr (TOP)
    if (tid == 0) s_top.keys = s_top.crowded = 0;
  __syncthreads();
  RowSum all;
  all.m = s_m[0];
  for (int w = 1; w < warps; ++w) all.m = fmaxf(all.m, s_m[w]);
  for (int w = 0; w < warps; ++w) {
    RowSum o;
    o.m = s_m[w], o.s = s_s[w], o.t = s_t[w];
    o.raise(all.m, k);
    all.s += o.s;
    all.t += o.t;
  }
  float log_sum = logf(all.s);  // -inf: nothing allowed, NaN: no distribution
  auto put = [&](int place, uint64_t key) {  // an alternative of the row, once `all` is the whole row's
    const bool broken = isnan(all.s);
    if (key && !GTK_IN(key_column(key), a.vocab, 312)) return;
    if (a.top_ids) a.top_ids[r * a.top_k + place] = key && !broken ? int32_t(key_column(key)) : -1;
    if (a.top_logprobs)
      a.top_logprobs[r * a.top_k + place] = broken ? nan : key ? (key_value(key) - all.m) * a.scale - log_sum : -INFINITY;
  };
  uint32_t mine = 0, bound = 0;  // value_key of the thread's highest, and what the alternatives reach
  if constexpr (TOP) {
    typename P::Max over = best[0];
#pragma unroll
    for (int q = 1; q < kBatch; ++q) over = P::higher(over, best[q]);
    mine = value_key(P::kHalves == 2 ? fmaxf(P::of(over, 0), P::of(over, 1)) : P::of(over, 0));
    // at least top_k elements reach the top_k-th highest of the threads' own; with several parts, the lowest of the parts'
    // (top_k / parts)-th highest
    bound = find_bound<T>(mine, (a.top_k + parts - 1) / parts);
  }
  if constexpr (!SPLIT) {
    if constexpr (TOP) {
      if (!collect_few<kLook>(row, begin, end, true, kMostKeys, bound, best, s_top))
        collect_keys(row, begin, end, true, a.top_k, kMostKeys, bound, mine, best, s_top);
      rank_keys(s_top, s_top.keys, a.top_k, put);
    }
  } else {
    cg::cluster_group cluster = cg::this_cluster();
    if (tid == 0) {
      s_part = all;
      if constexpr (TOP) s_top.bound = bound;
    }
    cluster.sync();
    if constexpr (TOP) {
      // lane c asks part c, here and below: reads of other CTAs' shared memory take long, one after the other too long
      bound = __reduce_min_sync(0xFFFFFFFFu, lane < parts ? cluster.map_shared_rank(&s_top, lane)->bound : bound);
      if (!collect_few<kLook>(row, begin, end, part == 0, kMostKeysOfPart, bound, best, s_top))
        collect_keys(row, begin, end, part == 0, a.top_k, kMostKeysOfPart, bound, mine, best, s_top);
      cluster.sync();
    }
    if (part == 0) {
      RowSum o;
      int keys = 0;
      if (lane < parts) {
        o = *cluster.map_shared_rank(&s_part, lane);
        if constexpr (TOP) keys = cluster.map_shared_rank(&s_top, lane)->keys;
      }
      all.m = o.m;
#pragma unroll
      for (int d = kMaxParts / 2; d; d >>= 1) all.m = fmaxf(all.m, __shfl_xor_sync(0xFFFFFFFFu, all.m, d));
      all.m = __shfl_sync(0xFFFFFFFFu, all.m, 0);
      o.raise(all.m, k);
#pragma unroll
      for (int d = kMaxParts / 2; d; d >>= 1) {
        o.s += __shfl_xor_sync(0xFFFFFFFFu, o.s, d);
        o.t += __shfl_xor_sync(0xFFFFFFFFu, o.t, d);
      }
      all.s   = __shfl_sync(0xFFFFFFFFu, o.s, 0);
      all.t   = __shfl_sync(0xFFFFFFFFu, o.t, 0);
      log_sum = logf(all.s);
      if constexpr (TOP) {  // the others' keys behind its own
        int upto = keys;
#pragma unroll
        for (int d = 1; d < kMaxParts; d *= 2) {
          const int more = __shfl_up_sync(0xFFFFFFFFu, upto, d);
          if (lane >= d) upto += more;
        }
        for (int c = 1 + warp; c < parts; c += warps) {
          const int count = __shfl_sync(0xFFFFFFFFu, keys, c), at = __shfl_sync(0xFFFFFFFFu, upto, c) - count;
          for (int i = lane; i < count; i += 32)
            if (GTK_IN(at + i, kMostKeys, 313) && GTK_IN(i, kMostKeysOfPart, 314)) s_top.key[at + i] = cluster.map_shared_rank(&s_top, c)->key[i];
        }
        __syncthreads();
        rank_keys(s_top, __shfl_sync(0xFFFFFFFFu, upto, parts - 1), a.top_k, put);
      }
    }
    cluster.sync();  // nobody leaves while its shared memory is read
    if (part != 0) return;
  }
  if (tid == 0) {
    const bool none = all.s == 0.f, broken = isnan(all.s);
    if (a.logprob) {
      float lp = target < 0 ? 0.f : nan;
      if (target >= 0 && target < a.vocab && !broken) lp = none ? -INFINITY : (at_target - all.m) * a.scale - log_sum;
      a.logprob[r] = lp;
    }
    if (a.entropy) a.entropy[r] = none ? 0.f : broken ? nan : fmaxf(log_sum - kLn2 * all.t / all.s, 0.f);
    if (a.lse) a.lse[r] = none ? -INFINITY : broken ? nan : fmaf(all.m, a.scale, log_sum);
  }
}

// How many CTAs share a row, and how many threads they have.
// Few rows are split, as long as a CTA keeps 12 KiB and there is an SM for each (for two, of rows from 160 KiB on).  In 1 / 2 / 4 / 8
// parts, us: one row of 50257 bf16 6.4 / 5.5 / 4.6 / 4.0, 74 of them 6.4 / 5.5 / 6.2 / 7.0, 148 of them 6.1 / 6.8 / 8.3 / 10.7; 148 rows of
// 131072 bf16 18.3 / 13.5 / 13.4 / 15.2; one row of 8192 bf16 with five alternatives 6.0 / 8.3 / 8.1 / 8.2.
// Rows in numbers take fewer threads each, so that more of them are under way while others are at their ends.  With 256 / 128 /
// 64, us: 740 rows of 50257 bf16 17.7 / 19.1 / 26.9, 999 of them 24.7 / 22.6 / 29.1, 8192 of them 141 / 130 / 130; of rows of 8192 bf16 with
// five alternatives 148: 6.4 / 6.6 / 7.6, 500: 9.3 / 8.0 / 8.3, 1500: 19.3 / 14.4 / 13.3, 8192: 88 / 56 / 45.
struct Teams {
  int parts, threads;
};
Teams teams_for(int64_t rows, int64_t bytes, int sm_count)
{
  Teams t{1, kThreads};
  const int64_t room = int64_t(sm_count) * (bytes >= (160 << 10) ? 2 : 1);
  while (t.parts < kMaxParts && rows * t.parts * 2 <= room && bytes / (t.parts * 2) >= (12 << 10)) t.parts *= 2;
  if (rows > int64_t(sm_count) * 5 || (bytes <= (24 << 10) && rows > int64_t(sm_count) * 3 / 2)) t.threads = 128;
  if (bytes <= (24 << 10) && rows > int64_t(sm_count) * 8) t.threads = 64;
  return t;
}

template <class T, bool ENTROPY, bool TOP>
cudaError_t launch_logprobs(const gtk::HandleView& v, const void* logits, int64_t n_rows, const ScoreArgs& a)
{
  const Teams t = teams_for(n_rows, int64_t(a.vocab) * int64_t(sizeof(T)), v.sm_count);
  auto kernel   = t.parts > 1 ? k_token_logprobs<T, ENTROPY, TOP, true> : k_token_logprobs<T, ENTROPY, TOP, false>;
  return gtk::launch_clusters(kernel, dim3(unsigned(n_rows * t.parts)), dim3(unsigned(t.threads)), t.parts, 0, v.stream,
                              static_cast<const T*>(logits), a, t.parts);
}

struct ScoreGradArgs {
  int vocab;
  int64_t stride, grad_stride;
  float scale;
  const int32_t* targets;
  const float *lse, *entropy, *grad_logprob, *grad_entropy;
};

// From this size on lse no longer does for p = exp(scale * x - lse): it is scale * m + ln S rounded to 32 bits, off by up to 2^-24 of itself,
// and that is the relative error of p (7.6e-6 below 256, a 64th of what rounding to fp16 costs).  A row filled with the lowest number of
// its type, which is how many a mask is written, keeps nothing of ln S at all, and scale * m may be beyond 32 bits where ln S is a small
// number.  Such rows are summed again from their logits, as k_token_logprobs has done it, which costs a second reading by one CTA
// (8192 rows of 50257 bf16 262 us, all far 362; 4096 of f32 273 and 379; one row 6.1 and 16.4): the limit is above the 100 or so that the
// logits of models in use lie around.
constexpr float kFarLse = 256.f;

// The highest of a row and the sum of 2^((x - highest) k), by all threads of a CTA.
template <class T>
__device__ __noinline__ float2 sum_row(const T* x, int vocab, float k)
{
  using P         = Pack16<T>;
  constexpr int E = P::kElems;
  __shared__ float s_m[kWarps], s_s[kWarps];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const RowParts<T> row(x, vocab);
  RowSum sum;
  if (tid < row.head + row.tail) sum.add(gtk::to_float(row.x[row.loose_column(tid)]), k);
  for (int p0 = tid; p0 < row.packs; p0 += kBatch * kThreads) {
    uint4 raw[kBatch];
#pragma unroll
    for (int q = 0; q < kBatch; ++q) {
      constexpr uint32_t w = P::kMinusInf;
      raw[q] = p0 + q * kThreads < row.packs ? *row.pack(p0 + q * kThreads) : make_uint4(w, w, w, w);
    }
#pragma unroll
    for (int q = 0; q < kBatch; ++q) {
      const typename P::Max all = P::highest(raw[q]);
      const float high          = P::kHalves == 2 ? fmaxf(P::of(all, 0), P::of(all, 1)) : P::of(all, 0);
      if (high > sum.m) sum.raise(high, k);
      Two pairs[E / 2];
      P::pairs(raw[q], pairs);
#pragma unroll
      for (int j = 0; j < E / 2; ++j) {
        float x0, x1;
        pairs[j].get(x0, x1);
        sum.s += pow2((x0 - sum.m) * k) + pow2((x1 - sum.m) * k);
      }
    }
  }
  float high = sum.m;
#pragma unroll
  for (int d = 16; d; d >>= 1) high = fmaxf(high, __shfl_xor_sync(0xFFFFFFFFu, high, d));
  sum.raise(high, k);
#pragma unroll
  for (int d = 16; d; d >>= 1) sum.s += __shfl_xor_sync(0xFFFFFFFFu, sum.s, d);
  if (lane == 0) s_m[warp] = sum.m, s_s[warp] = sum.s;
  __syncthreads();
  float m = s_m[0];
  for (int w = 1; w < kWarps; ++w) m = fmaxf(m, s_m[w]);
  float s = 0.f;
  for (int w = 0; w < kWarps; ++w) {
    RowSum o;
    o.m = s_m[w], o.s = s_s[w];
    o.raise(m, k);
    s += o.s;
  }
  return make_float2(m, s);
}

// d = scale * (g * ([j == t] - p) - e * p * (log p + H)), log p = scale * (x - m) - log_sum.  With m = 0 and log_sum = lse in all rows but
// far ones, where sum_again() finds both.  Every element is read and written once, by
// the same thread, so that grad may be logits.  A row's elements are shared by `parts` CTAs: as many as it has batches, up to 32 CTAs
// per SM in all (1021 rows of 32003 fp16 with entropy: 25 us, with up to 8 28 us; 2000 of them 42 and 46).  A far row is its first CTA's
// alone, which has read all of it before it writes.
template <class T, bool ENTROPY>
struct GradRow {
  float scale, m, log_sum, g, e, H;
  int t;
  bool nothing, far;
  __device__ GradRow(const ScoreGradArgs& a, int64_t r) : scale(a.scale), m(0.f)
  {
    t   = a.grad_logprob ? __ldg(a.targets + r) : -1;
    if (t >= a.vocab) t = -1;
    g   = t >= 0 ? __ldg(a.grad_logprob + r) * -scale : 0.f;
    e   = ENTROPY ? __ldg(a.grad_entropy + r) * -scale : 0.f;
    H   = ENTROPY ? __ldg(a.entropy + r) : 0.f;
    log_sum = __ldg(a.lse + r);
    // Whatever the row holds: padding may be NaN, and 0 * NaN is no zero.  Up to a scale of 1 no number becomes -inf: all are masked
    nothing = (g == 0.f && e == 0.f) || (log_sum == -INFINITY && scale <= 1.f);
    far     = !nothing && fabsf(log_sum) >= kFarLse;
  }
  // for a far row, by all threads of a CTA
  __device__ __forceinline__ void sum_again(const T* x, int vocab)
  {
    const float2 found = sum_row(x, vocab, scale * kLog2e);
    m = found.x, log_sum = logf(found.y);
    nothing = found.y == 0.f;
  }
  template <bool NEAR = false>  // NEAR: m is known to be 0
  __device__ __forceinline__ float of(float x, int column) const
  {
    const float z = fmaf(NEAR ? x : x - m, scale, -log_sum), p = pow2(z * kLog2e);
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
  GradRow<T, ENTROPY> R(a, r);
  if (R.far) {
    if (part != 0) return;
    R.sum_again(row.x, a.vocab);
  }
  if (part == 0 && tid < row.head + row.tail) {
    const int c = row.loose_column(tid);
    to[c]       = gtk::from_float<T>(R.nothing ? 0.f : R.of(gtk::to_float(row.x[c]), c));
  }
  const int share = R.far ? row.packs : (row.packs + parts - 1) / parts;
  const int begin = part * share, end = min(row.packs, begin + share);
  uint4* out = reinterpret_cast<uint4*>(to + row.head);
  if (R.nothing) {
    for (int p = begin + tid; p < end; p += kThreads) out[p] = make_uint4(0u, 0u, 0u, 0u);
    return;
  }
  const Two scale2(R.scale, R.scale), m2(-R.m, -R.m), log_sum2(-R.log_sum, -R.log_sum), log2e2(kLog2e, kLog2e), g2(R.g, R.g), e2(R.e, R.e), H2(R.H, R.H);
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
        const Two z = fma2(x[j] + m2, scale2, log_sum2);
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
        const float d = GTK_IN(R.t, a.vocab, 315) ? R.of(gtk::to_float(row.x[R.t]), R.t) : 0.f;
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (j == at) y.e[j] = gtk::from_float<T>(d);
      }
      out[p] = *reinterpret_cast<const uint4*>(&y);
    }
  }
}

// The same where logits and gradient lie differently against 16-byte boundaries: element by element, with
// kPlainBatch loads in flight (2048 rows of 50257 bf16: 95 us, one load at a time 228, in packs where they lie alike 69; f32 143
// and 134).
constexpr int kPlainBatch = 8;
template <class T, bool ENTROPY>
__global__ void __launch_bounds__(kThreads) k_token_logprobs_grad_plain(const T* logits, T* grad, const ScoreGradArgs a, int parts)
{
  const int64_t r = blockIdx.x / unsigned(parts);
  const int part  = int(blockIdx.x % unsigned(parts));
  const T* x      = logits + r * a.stride;
  T* to           = grad + r * a.grad_stride;
  GradRow<T, ENTROPY> R(a, r);
  auto all = [&](auto near, int first, int step) {
    for (int64_t c0 = int64_t(first) * kPlainBatch * kThreads + threadIdx.x; c0 < a.vocab; c0 += int64_t(step) * kPlainBatch * kThreads) {
      T raw[kPlainBatch];
#pragma unroll
      for (int q = 0; q < kPlainBatch; ++q)
        if (c0 + q * kThreads < a.vocab) raw[q] = x[c0 + q * kThreads];
#pragma unroll
      for (int q = 0; q < kPlainBatch; ++q) {
        const int64_t c = c0 + q * kThreads;
        if (c < a.vocab) to[c] = gtk::from_float<T>(R.nothing ? 0.f : R.template of<decltype(near)::value>(gtk::to_float(raw[q]), int(c)));
      }
    }
  };
  if (!R.far) {
    all(std::true_type{}, part, parts);
  } else if (part == 0) {
    R.sum_again(x, a.vocab);
    all(std::false_type{}, 0, 1);
  }
}

template <class T, bool ENTROPY>
cudaError_t launch_logprobs_grad(const gtk::HandleView& v, const void* logits, void* grad, int64_t n_rows, const ScoreGradArgs& a)
{
  const bool alike = (reinterpret_cast<uintptr_t>(logits) - reinterpret_cast<uintptr_t>(grad)) % 16 == 0 &&
                     (n_rows == 1 || (a.stride - a.grad_stride) * int64_t(sizeof(T)) % 16 == 0);
  const int64_t batches = (a.vocab + kBatch * kThreads * Pack16<T>::kElems - 1) / (kBatch * kThreads * Pack16<T>::kElems);
  const int parts = int(std::max<int64_t>(1, std::min<int64_t>(batches, int64_t(v.sm_count) * 32 / n_rows)));
  return gtk::launch(alike ? k_token_logprobs_grad<T, ENTROPY> : k_token_logprobs_grad_plain<T, ENTROPY>, dim3(unsigned(n_rows * parts)),
                     dim3(kThreads), 0, v.stream, static_cast<const T*>(logits), static_cast<T*>(grad), a, parts);
}

constexpr int64_t kMaxVocab = int64_t(1) << 30, kMaxRows = (int64_t(1) << 31) - 1;
constexpr float kMaxScale = 1e38f;  // times log2(e) it is a number too

gtk::Refusal refuse_sizes(int type, int64_t n_rows, int64_t vocab, int64_t stride, float scale)
{
  if (!gtk::known_type(type)) return "unknown element type";
  if (n_rows < 0 || vocab <= 0 || stride < 0) return "n_rows and stride must be >= 0, vocab > 0";
  if (n_rows > kMaxRows || vocab > kMaxVocab) return "n_rows of 2^31 and more, or vocab beyond 2^30";
  if (!(scale > 0.f && scale <= kMaxScale)) return "scale must be a number > 0, 1e38 at most";
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

#ifdef GTK_CHECKED
cudaError_t gtk::logprobs_check_words(int sum[4], bool reset) { return add_check_words(sum, reset); }
cudaError_t gtk::logprobs_check_selftest() { return check_selftest(399); }
#endif
