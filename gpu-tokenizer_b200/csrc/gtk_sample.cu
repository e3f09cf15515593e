// gtk_sample.cu -- an id drawn per row of logits, with temperature, top-k, top-p and min-p, from a given random number.
//
// With m a row's maximum and w_j = exp((x_j - m) / T), columns ranked by logit, of equal ones the lower first: the first K = top_k are
// looked at; of these the fewest whose weights reach top_p of their sum; of these those with w_j >= min_p.  The id is the first
// column, in the order of columns, at which the sum of the weights that are left exceeds u times the whole of it.
//
// A row is read once.  Its weights are summed in 32 bits, by sections of neighbouring columns, and every decision that hangs on such a
// sum is held against a bound of its error (Row::exponent_error); where a border lies within the bound the row is summed again in 64 bits.
//
// The reading is bound by memory, what follows it by phases that wait for each other.  Measured against a copy (6.57 TB/s), in a graph of calls
// whose inputs together pass L2; logits normal with a head of 64 likely ids, whose lead differs from row to row, "sure" with one far above all:
//   1024 rows of 131072 bf16, no limits   sure 53.7 us, 76 %; where a model is unsure of thousands of ids, some ten of them are looked
//                                         at again, which takes one CTA 80 us each: 137
//   2048 rows of 50257, no limits, sure   f32 71.8 us, 87 %, bf16 47.5, fp16 46.7; unsure 111, 91, 88
//   the same, unsure, with the 50 highest f32 136 us, bf16 90, fp16 87; with min-p 0.05 instead 153, 106, 103
//   512 rows of 50257, the highest        f32 23.4 us, bf16 17.5, fp16 17.2; weights are summed in these too, for the NaN that they tell of
//   one row of 50257 bf16                 6.1 us without limits, 14.7 with top-k and top-p
//   64 rows of 131072 f32, wide nuclei    77 us: three readings, 120 instructions an element, 17 of them in 64 bits
//   64 rows of 131072 bf16, top-p 0.95, normal with deviation 2, T = 1: mean 0 1255 us, mean 10 5370; see Slowly::search
#include <cooperative_groups.h>

#include <cfloat>
#include <climits>
#include <cmath>

#include "gtk_checked.cuh"
#include "gtk_logits.cuh"

namespace {

namespace cg = cooperative_groups;
using gtk::key_column;
using gtk::key_value;
using gtk::Pack16;
using gtk::pow2;
using gtk::rank_key;
using gtk::Two;
using gtk::value_key;

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMaxParts = 8;     // CTAs that share a row
constexpr int kPacks    = 4;     // of 16 bytes that a thread has of a section: 32 * kPacks neighbouring packs, whose sum is kept
constexpr int kBins     = 256;
constexpr int kFine     = 1024;  // bins of a wide row
constexpr int kMostKeys = 512;   // columns that are ranked at most
constexpr int kSetsOfWarp = 32 * kPacks;  // of its columns that a warp knows the highest of, at most
constexpr float kLow    = -0x1p60f;

struct SampleArgs {
  int vocab;
  int64_t stride;
  const double* uniform;
  const float *temperature, *top_p, *min_p;
  const int32_t* top_k;
  int32_t* ids;
  float* logprob;
};

// What a row's request wants.
struct Limits {
  double u;
  float t, p, least;
  int k;
  double inverse;  // of the temperature, 1 for 0
  __device__ Limits(const SampleArgs& a, int64_t r)
  {
    u     = __ldg(a.uniform + r);
    if (u > 1.0) u = 1.0;
    t     = a.temperature ? __ldg(a.temperature + r) : 1.f;
    p     = a.top_p ? __ldg(a.top_p + r) : 1.f;
    least = a.min_p ? fminf(__ldg(a.min_p + r), 1.f) : 0.f;
    if (a.min_p && isnan(__ldg(a.min_p + r))) least = NAN;
    k = a.top_k ? __ldg(a.top_k + r) : 0;
    if (k <= 0 || k >= a.vocab) k = INT_MAX;
    if (t == 0.f) k = 1;
    inverse = t == 0.f ? 1.0 : 1.0 / double(t);
  }
  __device__ bool broken() const { return !(t >= 0.f && t < INFINITY) || isnan(p) || isnan(least) || isnan(u); }
  __device__ bool cut_by_mass() const { return p < 1.f && t > 0.f; }
  __device__ bool all() const { return k == INT_MAX && !cut_by_mass() && !(least > 0.f); }
};

// What the threads of a CTA tell each other, and the columns that are ranked.  Small, for what shared memory takes the loads under way do
// not have: 25 KiB a CTA cost 2048 rows of 50257 f32 a fifth.
struct alignas(16) Scratch {
  union {
    struct {
      uint64_t key[kMostKeys];
      double weight[kMostKeys];
    };
    struct {
      uint32_t fine[kFine], fine_all[kFine];  // of this CTA, of all that share the row
    };
  };
  union {
    uint64_t ranked[kThreads];
    uint32_t by_column[kMostKeys];
  };
  union {
    uint8_t set[kWarps * kSetsOfWarp];
    uint16_t order[kMostKeys];
  };
  double power[64];  // 2^(i / 64)
  double mass[kWarps];
  int count[kWarps];
  float top[kWarps], low[kWarps];
  int hist[kBins], bins[kBins];  // of this CTA, of all that share the row
  double total, part_sum;
  uint64_t floor;
  int column, keys, left, part_count, solved, first, last;
  float run[kFine / 128];
  bool sure;
  float part_top;
};

template <class T>
__device__ __forceinline__ void unpack(const uint4& raw, float (&x)[Pack16<T>::kElems])
{
  Two pairs[Pack16<T>::kElems / 2];
  Pack16<T>::pairs(raw, pairs);
#pragma unroll
  for (int j = 0; j < Pack16<T>::kElems / 2; ++j) pairs[j].get(x[2 * j], x[2 * j + 1]);
}

// their sum, by halves
template <class N, int E>
__device__ __forceinline__ N sum_of(N (&x)[E])
{
#pragma unroll
  for (int d = 1; d < E; d *= 2)
#pragma unroll
    for (int j = 0; j < E; j += 2 * d) x[j] += x[j + d];
  return x[0];
}

// adds to a word of shared memory where `yes`, without a branch
__device__ __forceinline__ void add_shared(uint32_t* p, uint32_t n, bool yes)
{
  asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %2, 0;\n @p red.shared.add.u32 [%0], %1;\n}" ::"r"(uint32_t(__cvta_generic_to_shared(p))), "r"(n),
               "r"(uint32_t(yes))
               : "memory");
}

// Past the first-level cache, in which the loads under way would otherwise take their places (2048 rows of 50257 f32 77 -> 68 us).
__device__ __forceinline__ uint4 load_past(const uint4* p)
{
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// A row as the packs of 16 bytes that it touches; what lies in them outside of it counts as -inf.
template <class T>
struct Row {
  static constexpr int E = Pack16<T>::kElems, kColumns = 32 * kPacks * E;  // of a section
  const uint4* base;
  int vocab, lead, packs, sections;
  __device__ Row(const T* x, int vocab_) : vocab(vocab_)
  {
    lead     = int((uint32_t(reinterpret_cast<uintptr_t>(x)) & 15u) / sizeof(T));
    base     = reinterpret_cast<const uint4*>(x - lead);
    packs    = (lead + vocab + E - 1) / E;
    sections = (packs + 32 * kPacks - 1) / (32 * kPacks);
  }
  __device__ __forceinline__ int column(int p) const { return p * E - lead; }
  __device__ __forceinline__ uint4 load(int p) const
  {
    constexpr uint32_t w = Pack16<T>::kMinusInf;
    if (p >= packs) return make_uint4(w, w, w, w);
    uint4 raw = __ldg(base + p);
    if (p == 0 || p == packs - 1) {
      T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (uint32_t(column(p) + j) >= uint32_t(vocab)) e[j] = gtk::from_float<T>(-INFINITY);
    }
    return raw;
  }
  __device__ __forceinline__ float value(int c) const
  {
    return gtk::to_float(reinterpret_cast<const T*>(base)[lead + c]);
  }
  // The first and the last pack are in no such section.
  __device__ __forceinline__ bool whole(int s) const { return s > 0 && (s + 1) * 32 * kPacks < packs; }
  __device__ __forceinline__ void load_section(int s, uint4 (&raw)[kPacks]) const
  {
    const int p0 = s * 32 * kPacks + int(threadIdx.x & 31);
    if (whole(s)) {
#pragma unroll
      for (int q = 0; q < kPacks; ++q) raw[q] = load_past(base + p0 + q * 32);
    } else {
#pragma unroll
      for (int q = 0; q < kPacks; ++q) raw[q] = load(p0 + q * 32);
    }
  }
  // Bounds of what 32 bits cost, in parts of 2^-24 of the sum of all weights, when that is at least `sum` times the highest's.  A weight 2^y, y =
  // x k - c rounded once, with k rounded once: 2 ln 2 |y| such parts of itself, and 4 for the exponential (2^-22).  The weights' mean of
  // ln 2 |y| is their entropy less ln(sum), ln(vocab / sum) at most, and c, a whole number, adds less than one to |y|.  The sum of a section:
  // ten additions (four or five of a thread's, five of the warp's), and nothing more where sections are added, in 64 bits.  The section that a
  // column lies in: its sum's and its weights' errors, and 16 roundings more of what lies in front of the column (near_column).
  static constexpr float kWeightError = 4.f, kSumError = 10.f, kOwnError = 28.f;
  __device__ __forceinline__ float exponent_error(double sum) const
  {
    return 2.f * 0.6932f * (fmaxf(0.f, log2f(float(vocab) / float(sum))) + 1.1f);
  }
};

__device__ __forceinline__ float warp_max(float x)
{
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xFFFFFFFF;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float warp_min(float x)
{
  float y;
  asm volatile("redux.sync.min.f32 %0, %1, 0xFFFFFFFF;" : "=f"(y) : "f"(x));
  return y;
}
template <class N>
__device__ __forceinline__ N warp_sum(N x)
{
#pragma unroll
  for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xFFFFFFFFu, x, d);
  return x;
}
template <class N>
__device__ __forceinline__ N warp_upto(N x)  // the sum of the lanes up to the own one
{
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const N l = __shfl_up_sync(0xFFFFFFFFu, x, d);
    if (lane >= d) x += l;
  }
  return x;
}

// exp((x - m) / T) in 64 bits: with y = (x - m) log2(e) / T = n / 64 + f the product of 2^(n / 64), by a table of 64 entries, and
// 2^f, |f| <= 1 / 128, whose series is cut behind the fifth power (3e-17).  No branch, so that several are under way at once; 2^e in two
// factors, for the subnormal ones.
struct Weight64 {
  double m, k;  // k: log2(e) / T
  const double* power;
  __device__ __forceinline__ double operator()(float x) const
  {
    const float one[1] = {x};
    double w[1];
    of(one, w);
    return w[0];
  }
  // of N numbers, step by step for all of them: a step waits for the one before it some 30 clocks
  template <int N>
  __device__ __forceinline__ void of(const float (&x)[N], double (&w)[N]) const
  {
    constexpr double l2 = 0.69314718055994531;
    double y[N], a[N];
    int n[N];
#pragma unroll
    for (int i = 0; i < N; ++i) y[i] = double(x[i]) - m;
#pragma unroll
    for (int i = 0; i < N; ++i) y[i] = fmax(y[i] * k, -1990.0);
#pragma unroll
    for (int i = 0; i < N; ++i) a[i] = fma(y[i], 64.0, 0x1.8p52);  // n in the low bits
#pragma unroll
    for (int i = 0; i < N; ++i) n[i] = __double2loint(a[i]), a[i] -= 0x1.8p52;
#pragma unroll
    for (int i = 0; i < N; ++i) y[i] = fma(a[i], -1.0 / 64, y[i]);
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = fma(y[i], l2 * l2 * l2 * l2 * l2 / 120, l2 * l2 * l2 * l2 / 24);
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = fma(y[i], w[i], l2 * l2 * l2 / 6);
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = fma(y[i], w[i], l2 * l2 / 2);
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = fma(y[i], w[i], l2);
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = fma(y[i], w[i], 1.0);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = n[i] >> 6, most = max(e, -1000);
      w[i] *= power[n[i] & 63] * __hiloint2double((most + 1023) << 20, 0);
      n[i] = e - most;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] *= __hiloint2double((n[i] + 1023) << 20, 0);
  }
};

// the table, by all threads
__device__ __forceinline__ Weight64 weight64(const Limits& l, double m, Scratch& S)
{
  if (threadIdx.x < 64) S.power[threadIdx.x] = exp2(double(threadIdx.x) / 64);
  __syncthreads();
  return Weight64{m, 1.4426950408889634 * l.inverse, S.power};
}

struct Sum {
  double mass;
  int count;
};

// The sums of weights by sections, to `section`, and their whole, by all threads.  weigh(x, column, w, count): the weights of some neighbouring
// columns, and how many of them count.
template <class T, class Weigh>
__device__ __forceinline__ Sum sum_row(const Row<T>& row, double* section, Scratch& S, Weigh&& weigh)
{
  const int threads = blockDim.x, warps = threads >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Sum s{0.0, 0};
  __syncthreads();
  uint4 raw[kPacks];
  if (warp < row.sections) row.load_section(warp, raw);
  for (int i = warp; i < row.sections; i += warps) {
    uint4 next[kPacks];
    if (i + warps < row.sections) row.load_section(i + warps, next);
    double sum = 0.0;
#pragma unroll 1
    for (int q = 0; q < kPacks; ++q) {  // one after the other: the code is run few times, and has to come in first
      const int p = (i * kPacks + q) * 32 + lane;
      float all[Row<T>::E];
      unpack<T>(raw[0], all);
#pragma unroll
      for (int j = 0; j < Row<T>::E; j += 4) {
        const float x[4] = {all[j], all[j + 1], all[j + 2], all[j + 3]};
        double w[4];
        weigh(x, row.column(p) + j, w, s.count);
        sum += sum_of(w);
      }
#pragma unroll
      for (int e = 1; e < kPacks; ++e) raw[e - 1] = raw[e];
    }
#pragma unroll
    for (int e = 0; e < kPacks; ++e) raw[e] = next[e];
    sum = warp_sum(sum);
    if (lane == 0 && GTK_IN(i, row.sections, 500)) section[i] = sum;
    s.mass += sum;
  }
  s.count = warp_sum(s.count);
  if (lane == 0) S.mass[warp] = s.mass, S.count[warp] = s.count;
  __syncthreads();
  s = Sum{0.0, 0};
  for (int w = 0; w < warps; ++w) s.mass += S.mass[w], s.count += S.count[w];
  return s;
}

// the same from f(x, column) -> {weight, whether it counts}
template <class T, class F>
__device__ __forceinline__ Sum sum_columns(const Row<T>& row, double* section, Scratch& S, F&& f)
{
  return sum_row(row, section, S, [&](const auto& x, int c, auto& w, int& count) {
    for (int j = 0; j < int(sizeof(x) / sizeof(x[0])); ++j) {
      const Sum o = f(x[j], c + j);
      w[j] = o.mass, count += o.count;
    }
  });
}

// A column with its section and its logit, and the sums of the weights in front of it and with it.
struct Place {
  int column, section;
  double before, upto;
  float x;
};

// The first column at which the sum of the weights exceeds the target, `share` of the sum of all, by one warp: section(s) is a section's sum,
// weigh(s)(x, column, w) the weights of columns in it.  The last one with any weight where rounding leaves none, column -1 where none has any.
template <class T, class Section, class Weigh>
__device__ __forceinline__ Place locate(const Row<T>& row, double share, double& total, Section&& section, Weigh&& weigh)
{
  constexpr uint32_t all = 0xFFFFFFFFu;
  constexpr int kOwn     = kPacks * Row<T>::E;  // neighbouring columns of a lane
  static_assert(kOwn <= 32, "");
  const int lane = threadIdx.x & 31, each = (row.sections + 31) / 32;
  // the lane in whose share the target lies, of those with any weight
  auto lane_of = [&](double mine, double upto, double target) {
    const uint32_t over = __ballot_sync(all, mine > 0.0 && upto > target), some = __ballot_sync(all, mine > 0.0);
    return over ? __ffs(over) - 1 : some ? 31 - __clz(some) : -1;
  };
  const int begin = min(lane * each, row.sections), end = min(begin + each, row.sections);
  double mine = 0.0;
  for (int i = begin; i < end; ++i) mine += section(i);
  double upto = warp_upto(mine);
  total       = __shfl_sync(all, upto, 31);
  const double target = share * total;
  int from = lane_of(mine, upto, target);
  if (from < 0) return Place{-1, -1, 0.0, 0.0, 0.f};
  int s        = -1;
  double front = upto - mine, next = front;
  if (lane == from)
    for (int i = begin; i < end; ++i) {
      const double w = section(i);
      if (!(w > 0.0)) continue;
      s = i, front = next;
      next += w;
      if (next > target) break;
    }
  s     = __shfl_sync(all, s, from);
  front = __shfl_sync(all, front, from);
  // neighbouring packs to a lane
  auto weight = weigh(s);
  mine        = 0.0;
#pragma unroll 1
  for (int q = 0; q < kPacks; ++q) {
    const int p     = (s * 32 + lane) * kPacks + q, c = row.column(p);
    const uint4 raw = row.load(p);
    float all_of[Row<T>::E];
    unpack<T>(raw, all_of);
#pragma unroll
    for (int j = 0; j < Row<T>::E; j += 4) {
      const float x[4] = {all_of[j], all_of[j + 1], all_of[j + 2], all_of[j + 3]};
      double w[4];
      weight(x, c + j, w);
      mine += sum_of(w);
    }
  }
  upto = front + warp_upto(mine);
  from = lane_of(mine, upto, target);
  if (from < 0) return Place{-1, s, 0.0, 0.0, 0.f};
  front = __shfl_sync(all, upto - mine, from);
  // a column to a lane
  const int c = row.column((s * 32 + from) * kPacks) + lane;
  const float own[1] = {lane < kOwn && uint32_t(c) < uint32_t(row.vocab) ? row.value(c) : -INFINITY};
  double w[1];
  weight(own, c, w);
  mine        = own[0] > -INFINITY ? w[0] : 0.0;
  upto        = front + warp_upto(mine);
  from        = lane_of(mine, upto, target);
  if (from < 0) return Place{-1, s, 0.0, 0.0, 0.f};
  return Place{__shfl_sync(all, c, from), s, __shfl_sync(all, upto - mine, from), __shfl_sync(all, upto, from), __shfl_sync(all, own[0], from)};
}

// Everything in 64 bits, by one CTA, in as many readings of the row as it takes: rows of which nothing else is known, or whose borders
// the sums in 32 bits do not tell from each other.
template <class T>
struct Slowly {
  const Row<T>& row;
  const Limits& l;
  double* section;
  Scratch& S;
  double m;
  uint64_t floor;  // what is left reaches it, see rank_key
  Weight64 power;
  double total;  // of the last find

  __device__ double weight(float x) const { return power(x); }
  __device__ bool left(float x, int c) const { return rank_key(x, uint32_t(c)) >= floor; }

  // the first column at which `weigh` exceeds a share of its sum, known to all threads
  template <class Weigh>
  __device__ int find(double share, Weigh&& weigh)
  {
    __syncthreads();
    if (threadIdx.x < 32) {
      double total;
      const Place found = locate(row, share, total, [&](int s) { return section[s]; }, [&](int) {
        return [&](const auto& x, int c, auto& w) {
          for (int j = 0; j < int(sizeof(x) / sizeof(x[0])); ++j) w[j] = weigh(x[j], c + j);
        };
      });
      if (threadIdx.x == 0) S.column = found.column, S.total = total;
    }
    __syncthreads();
    const int column = S.column;
    total            = S.total;
    __syncthreads();
    return column;
  }

  // Raises the floor to the highest value at which enough(sum over the columns that reach it) holds, and there to as many columns of that
  // value as are wanted(sum over those above it).  A reading in 64 bits for each halving, up to 32 of them, and four more: 80 us each for 131072
  // columns.  Rows come here with some hundreds of equal logits at the border of a wide limit, which 16-bit logits away from 0 have (bf16 of
  // mean 10 and deviation 2, 131072 of them, top-p 0.95: 1596), and by a top-k with more than 512 candidates where sets of columns are masked
  // by a finite number far below (64 rows of 50257 f32, top-k 700, 21000 columns at -1e9: 1238 us, at -inf 65).
  template <class Enough, class Wanted>
  __device__ void search(uint32_t most, Enough&& enough, Wanted&& wanted)
  {
    uint32_t lo = 1, hi = most;  // enough at lo
    for (bool first = true; lo < hi; first = false) {
      const uint32_t mid = first ? most : lo + (hi - lo + 1) / 2;  // rows of equal logits end with the first
      const Sum s = sum_columns(row, section, S, [&](float x, int c) { return value_key(x) >= mid && left(x, c) ? Sum{weight(x), 1} : Sum{0.0, 0}; });
      if (enough(s)) lo = mid;
      else hi = mid - 1;
    }
    const Sum above = sum_columns(row, section, S, [&](float x, int c) { return value_key(x) > lo && left(x, c) ? Sum{weight(x), 1} : Sum{0.0, 0}; });
    const float value  = key_value(uint64_t(lo) << 32);
    auto equal         = [&](float x, int c) { return value_key(x) == lo && left(x, c) ? 1.0 : 0.0; };
    const double equals = sum_columns(row, section, S, [&](float x, int c) { return Sum{equal(x, c), 0}; }).mass;
    const int column    = find((wanted(above, weight(value)) - 0.5) / equals, equal);
    floor            = max(floor, rank_key(value, uint32_t(column)));
  }

  // the drawn column and its log probability; -1 for a row without one
  __device__ int run(float& logprob)
  {
    const int threads = blockDim.x, warps = threads >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    bool broken   = false;
    uint32_t most = 0;
    const int some = sum_columns(row, section, S, [&](float x, int c) {
                       if (uint32_t(c) < uint32_t(row.vocab)) broken |= !(x < INFINITY), most = max(most, value_key(x));
                       return Sum{0.0, x > -INFINITY ? 1 : 0};
                     }).count;
    logprob = __int_as_float(0x7FC00000);
    if (__syncthreads_or(broken)) return -1;
    most = __reduce_max_sync(0xFFFFFFFFu, most);
    if (lane == 0) S.count[warp] = int(most);
    __syncthreads();
    for (int w = 0; w < warps; ++w) most = max(most, uint32_t(S.count[w]));
    logprob = -INFINITY;
    if (most == 0) return -1;
    m     = key_value(uint64_t(most) << 32);
    power = weight64(l, m, S);
    if (l.k < some)
      search(most, [&](const Sum& s) { return s.count >= l.k; }, [&](const Sum& s, double) { return double(l.k - s.count); });
    if (l.cut_by_mass()) {
      const double whole = sum_columns(row, section, S, [&](float x, int c) { return left(x, c) ? Sum{weight(x), 1} : Sum{0.0, 0}; }).mass;
      const double reach = fmax(0.0, double(l.p)) * whole;
      search(most, [&](const Sum& s) { return s.mass >= reach; },
             [&](const Sum& s, double w) {
               double n = fmax(1.0, w > 0.0 ? ceil((reach - s.mass) / w) : 1.0);
               if (n > 1.0 && s.mass + (n - 1.0) * w >= reach) n -= 1.0;
               return n;
             });
    }
    const double least_y = l.least > 0.f ? log(double(l.least)) : -INFINITY;
    auto drawn           = [&](float x, int c) { return left(x, c) && (double(x) - m) * l.inverse >= least_y ? weight(x) : 0.0; };
    sum_columns(row, section, S, [&](float x, int c) { return Sum{drawn(x, c), 0}; });
    const int id = find(l.u, drawn);
    if (id < 0) return -1;
    logprob = l.t == 0.f ? 0.f : float((double(row.value(id)) - m) * l.inverse - log(total));
    return id;
  }
};

template <class T>
__device__ __noinline__ int draw_slowly(const Row<T>& row, const Limits& l, double* section, Scratch& S, float& logprob)
{
  Slowly<T> s{row, l, section, S, 0.0, 1, {}, 0.0};
  return s.run(logprob);
}

// The sum of all weights in 64 bits, by sections too.
template <class T>
__device__ __noinline__ double sum_exactly(const Row<T>& row, const Limits& l, double m, double* section, Scratch& S)
{
  const Weight64 weight = weight64(l, m, S);
  return sum_row(row, section, S, [&](const auto& x, int, auto& w, int&) { weight.of(x, w); }).mass;
}

// What is drawn of all columns, with everything in 64 bits.
template <class T>
__device__ __noinline__ int draw_exactly(const Row<T>& row, const Limits& l, double m, double* section, Scratch& S, float& logprob)
{
  sum_exactly(row, l, m, section, S);
  const Weight64 weight{m, 1.4426950408889634 * l.inverse, S.power};
  if (threadIdx.x >= 32) return -1;
  double total;
  const Place found = locate(row, l.u, total, [&](int s) { return section[s]; },
                             [&](int) { return [&](const auto& x, int, auto& w) { weight.of(x, w); }; });
  logprob           = float((double(found.x) - m) * l.inverse - log(total));
  return found.column;
}

// Sorts n numbers, highest first, by all threads; there is room up to the next power of two.
template <class N>
__device__ void sort_down(N* a, int n)
{
  int size = 2;
  while (size < n) size *= 2;
  for (int i = n + int(threadIdx.x); i < size; i += blockDim.x) a[i] = 0;
  __syncthreads();
  for (int run = 2; run <= size; run *= 2)
    for (int d = run / 2; d; d /= 2) {
      for (int i = threadIdx.x; i < size / 2; i += blockDim.x) {
        const int at = 2 * i - (i & (d - 1));
        if (!GTK_IN(at + d, kMostKeys, 501)) continue;
        const N lo = a[at], hi = a[at + d];
        if ((lo < hi) == ((at & run) == 0)) a[at] = hi, a[at + d] = lo;
      }
      __syncthreads();
    }
}

// The ones of n ranked keys that are left, their number and their weights' sum; `whole`: the sum that top-p is a part of, off by `error` at
// most, < 0 where it is the sum of the keys.  By one warp; false where the error leaves it open.
__device__ __forceinline__ bool cut_keys(const Limits& l, double m, const uint64_t* key, const double* weight, int n, double whole, double error,
                                         int& left, double& total)
{
  const int lane = threadIdx.x & 31;
  n              = min(n, l.k);
  const int each = (n + 31) / 32, begin = min(n, lane * each), end = min(n, begin + each);
  double mine = 0.0;
  for (int i = begin; i < end; ++i) mine += weight[i];
  const double upto = warp_upto(mine), front = upto - mine;
  if (whole < 0.0) whole = __shfl_sync(0xFFFFFFFFu, upto, 31), error = 0.0;
  left      = n;
  bool open = false;
  if (l.cut_by_mass()) {
    const double reach = fmax(0.0, double(l.p)) * whole;
    int last           = INT_MAX;
    double so_far      = front;
    for (int i = begin; i < end && last == INT_MAX; ++i)
      if ((so_far += weight[i]) >= reach - error) last = i, open = so_far < reach + error;
    const int first = __reduce_min_sync(0xFFFFFFFFu, last);
    open            = __any_sync(0xFFFFFFFFu, open && last == first);
    if (first != INT_MAX) left = first + 1;
  }
  if (l.least > 0.f) {
    const double least_y = log(double(l.least));
    int allowed          = 0;
    for (int i = begin; i < end; ++i) allowed += (double(key_value(key[i])) - m) * l.inverse >= least_y;
    allowed = max(1, __reduce_add_sync(0xFFFFFFFFu, allowed));
    if (allowed < left) left = allowed, open = false;  // whatever top-p leaves open
  }
  double so_far = front;
  for (int i = begin; i < min(end, left); ++i) so_far += weight[i];
  total = __shfl_sync(0xFFFFFFFFu, so_far, (left - 1) / each);
  return !open;
}

// The rank of the key that is drawn: of n ranks in the order of columns those below `left` count.  By one warp.
__device__ __forceinline__ int draw_key(const uint16_t* order, const double* weight, int n, int left, double target)
{
  const int lane = threadIdx.x & 31, each = (n + 31) / 32, begin = min(n, lane * each), end = min(n, begin + each);
  auto weight_at = [&](int i) { return int(order[i]) < left ? weight[order[i]] : 0.0; };
  double mine    = 0.0;
  for (int i = begin; i < end; ++i) mine += weight_at(i);
  const double upto   = warp_upto(mine);
  const uint32_t over = __ballot_sync(0xFFFFFFFFu, mine > 0.0 && upto > target), some = __ballot_sync(0xFFFFFFFFu, mine > 0.0);
  const int from      = over ? __ffs(over) - 1 : 31 - __clz(some);  // the last one with any weight where rounding leaves none
  int at              = 0;
  if (lane == from) {
    double so_far = upto - mine;
    for (int i = begin; i < end; ++i) {
      const double w = weight_at(i);
      if (!(w > 0.0)) continue;
      at = int(order[i]);
      if ((so_far += w) > target) break;
    }
  }
  return __shfl_sync(0xFFFFFFFFu, at, from);
}

// The CTAs that share a row, and this one's sections of it.
template <bool SPLIT>
struct Team {
  int parts, part, share, begin, end;
  __device__ __forceinline__ void sync() const
  {
    if constexpr (SPLIT) cg::this_cluster().sync();
    else __syncthreads();
  }
  // an object of the c-th CTA that this one has at the same place
  template <class N>
  __device__ __forceinline__ N* of(N* mine, int c) const
  {
    if constexpr (SPLIT) return cg::this_cluster().map_shared_rank(mine, c);
    else return mine;
  }
  // f(s, each_pack) for the warps' sections, where each_pack(g) calls g(p, pack) for the thread's packs of it
  template <class T, class F>
  __device__ __forceinline__ void each_section_packs(const Row<T>& row, F&& f) const
  {
    const int warps = blockDim.x >> 5;
    for (int s = begin + int(threadIdx.x >> 5); s < end; s += warps) {
      uint4 raw[kPacks];  // the next section's too do not fit into the registers (64 rows of 131072 f32: 116 us, as it is 75)
      row.load_section(s, raw);
      f(s, [&](auto&& g) {
#pragma unroll 1
        for (int q = 0; q < kPacks; ++q) {  // one after the other: the code is run few times, and has to come in first
          g((s * kPacks + q) * 32 + int(threadIdx.x & 31), raw[0]);
#pragma unroll
          for (int i = 1; i < kPacks; ++i) raw[i - 1] = raw[i];
        }
      });
    }
  }
};

// The keys of all CTAs behind those of the first: their number, known to all; they are there when it is kMostKeys at most.
template <bool SPLIT>
__device__ __forceinline__ int gather_keys(const Team<SPLIT>& team, Scratch& S)
{
  team.sync();
  if constexpr (!SPLIT) {
    return S.keys;
  } else {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    // lane c asks part c
    const int keys = lane < team.parts ? team.of(&S, lane)->keys : 0;
    const int upto = warp_upto(keys), n = __shfl_sync(0xFFFFFFFFu, upto, 31);
    if (team.part == 0 && n <= kMostKeys)
      for (int c = 1 + warp; c < team.parts; c += warps) {
        const int count = __shfl_sync(0xFFFFFFFFu, keys, c), at = __shfl_sync(0xFFFFFFFFu, upto, c) - count;
        for (int i = lane; i < count; i += 32)
          if (GTK_IN(at + i, kMostKeys, 507)) S.key[at + i] = team.of(&S, c)->key[i];
      }
    team.sync();
    return n;
  }
}

// The lowest of the numbers between those of the keys lo (for which holds() need not) and hi (for which it does) at which holds(); it does
// for all above.
template <class Holds>
__device__ __forceinline__ uint32_t lowest_key(uint32_t lo, uint32_t hi, Holds&& holds)
{
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo) / 2;
    if (holds(key_value(uint64_t(mid) << 32))) hi = mid;
    else lo = mid + 1;
  }
  return hi;
}

// What a pass over a wide row goes by: x is in interval int((hi - x) * scale), or above all of them from `beyond` on.
struct Interval {
  uint64_t floor;
  float hi, scale, beyond;
  float a, b, c, d;
  bool yes, all;
};

// Counts the columns in S.fine, or with v.yes adds their weights, as whole numbers relative to the interval's upper end: v.a the highest
// logit, v.b an exponent's part of a logit, v.c of an interval, v.d the bits of a one.  The sum of the weights from `beyond` on, or of v.all.
// PLAIN: by weight, and no round has been before.
template <bool PLAIN, class T, bool SPLIT>
__device__ __noinline__ double count_columns(const Row<T>& row, const Team<SPLIT>& team, const Interval v, Scratch& S)
{
  constexpr int E = Row<T>::E;
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  double sum = 0.0;
  team.each_section_packs(row, [&](int, auto&& each) {
    float of_section = 0.f;
    each([&](int p, const uint4& raw) {
      float x[E], at[E], part[E];
      unpack<T>(raw, x);
      int b[E];
      bool in[E];
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const bool left = PLAIN || v.floor == 1 || rank_key(x[j], uint32_t(row.column(p) + j)) >= v.floor;
        at[j]   = (v.hi - x[j]) * v.scale;
        in[j]   = left && x[j] < v.beyond;
        b[j]    = int(fminf(at[j], float(kFine)));
        part[j] = (PLAIN || v.yes) && left && (v.all || !in[j]) ? pow2((x[j] - v.a) * v.b) : 0.f;
      }
#pragma unroll
      for (int j = 0; j < E; ++j) at[j] = PLAIN || v.yes ? pow2(fmaf(float(b[j]) - at[j], v.c, v.d)) : 1.f;
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const bool counts = in[j] && b[j] < kFine && GTK_IN(b[j], kFine, 508);
        add_shared(S.fine + (counts ? b[j] : 0), uint32_t(__float2int_rn(at[j])), counts);
      }
      of_section += sum_of(part);
    });
    sum += of_section;
  });
  sum = warp_sum(sum);
  if (lane == 0) S.mass[warp] = sum;
  __syncthreads();
  sum = 0.0;
  for (int w = 0; w < warps; ++w) sum += S.mass[w];
  if (threadIdx.x == 0) S.part_sum = sum;
  return sum;
}

// Sums in 64 bits, of columns that reach v.floor: those above interval v.b (v.yes: all) and at least v.a by sections, all of them together; lists
// those in front of interval v.c, and tells how many are above and whether some of these are below v.a.
struct Above {
  double all;
  int count;
  bool cut_short;
};
// PLAIN: by weight, no round before, no min-p.
template <bool PLAIN, class T, bool SPLIT>
__device__ __noinline__ Above sum_above(const Row<T>& row, const Team<SPLIT>& team, const Weight64 weight, const Interval v, double* section,
                                        Scratch& S)
{
  constexpr int E = Row<T>::E, kOnce = 4;  // columns at a time
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Above found{0.0, 0, false};
  team.each_section_packs(row, [&](int s, auto&& each_pack) {
    double part = 0.0;
    each_pack([&](int p, const uint4& raw) {
      float all[E];
      unpack<T>(raw, all);
      uint32_t hits = 0;
#pragma unroll
      for (int i = 0; i < E; i += kOnce) {
        float x[kOnce];
        double w[kOnce], kept[kOnce];
#pragma unroll
        for (int j = 0; j < kOnce; ++j) x[j] = all[i + j];
        weight.of(x, w);
#pragma unroll
        for (int j = 0; j < kOnce; ++j) {
          const float at = (v.hi - x[j]) * v.scale;
          if constexpr (PLAIN) {  // -inf weighs nothing and lies in no interval
            const bool above = x[j] >= v.beyond || at < v.b;
            hits |= (!above && at < v.c ? 1u : 0u) << (i + j);
            kept[j] = above ? w[j] : 0.0;
          } else {
            const bool in    = rank_key(x[j], uint32_t(row.column(p) + i + j)) >= v.floor;
            const bool above = in && (v.yes || x[j] >= v.beyond || at < v.b), high = x[j] >= v.a;
            hits |= (in && !above && at < v.c ? 1u : 0u) << (i + j);
            w[j]    = in ? w[j] : 0.0;
            kept[j] = above && high ? w[j] : 0.0;
            found.count += above;
            found.cut_short |= above && !high;
          }
        }
        part += sum_of(kept);
        found.all += sum_of(w);
      }
      if (hits) {
        int i = atomicAdd(&S.keys, __popc(hits));
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (hits >> j & 1u) {
            if (i < kMostKeys && GTK_IN(i, kMostKeys, 509)) S.key[i] = rank_key(all[j], uint32_t(row.column(p) + j));
            ++i;
          }
      }
    });
    part = warp_sum(part);
    if (lane == 0 && GTK_IN(s, row.sections, 510)) section[s] = part;
  });
  found.all = warp_sum(found.all), found.count = warp_sum(found.count);
  found.cut_short = __any_sync(0xFFFFFFFFu, found.cut_short);
  if (lane == 0) S.mass[warp] = found.all, S.count[warp] = found.count << 1 | int(found.cut_short);
  __syncthreads();
  found.all = 0.0, found.count = 0;
  for (int w = 0; w < warps; ++w) found.all += S.mass[w], found.count += S.count[w] >> 1, found.cut_short |= S.count[w] & 1;
  if (threadIdx.x == 0) S.part_sum = found.all, S.part_count = found.count << 1 | int(found.cut_short);
  return found;
}

// Rows of which more columns are left than can be ranked.  For a limit by number or by mass the columns are counted by the interval of
// logits that they lie in, kFine of them, with weights as whole numbers (so that their sum is one in whatever order), again in the one that the limit
// falls in while that holds too many; then one pass in 64 bits sums what lies above it, by sections, and lists the columns within.
// Which of these are left is known once they are ranked.
// False where that finds nothing: more equal logits at a limit than can be ranked, or a limit beyond the intervals.  The answer is the
// first CTA's.
template <class T, bool SPLIT>
__device__ __noinline__ bool draw_wide(const Row<T>& row, const Limits& l, const Team<SPLIT>& team, float top, float low, double* section, Scratch& S,
                                       int& id, float& logprob)
{
  const int tid = threadIdx.x, threads = blockDim.x, warps = threads >> 5, warp = tid >> 5, lane = tid & 31;
  const double m        = top;
  const Weight64 weight = weight64(l, m, S);
  const float k         = float(weight.k);
  const uint32_t key_top = value_key(top);
  // what min-p leaves
  const uint32_t key_lowest = value_key(-FLT_MAX);
  uint32_t key_least = key_lowest;
  if (l.least > 0.f) {
    const double least_y = log(double(l.least));
    key_least            = lowest_key(key_lowest, key_top, [&](float x) { return (double(x) - m) * l.inverse >= least_y; });
  }
  uint64_t floor = 1;  // of the rank keys that are left
  const bool by_number = l.k != INT_MAX, by_mass = l.cut_by_mass();
  const int bits = min(15, 30 - (31 - __clz(row.vocab)));  // of the whole numbers, vocab of which 32 bits hold
  for (int round = by_number ? 0 : 1; round < 2 || (round == 2 && !by_number && !by_mass); ++round) {
    const bool mass = round == 1;
    if (mass && !by_mass) {
      if (by_number) break;
      round = 2;  // min-p alone
    }
    // ---- between which logits the limit lies: those from `beyond` on, and those in intervals in front of the first-th, are left; those
    // behind the last-th are not
    float lo = 0.f, hi = top, scale = 0.f, beyond = INFINITY;
    int first = 0, last = -1;
    if (round < 2) {
      // Columns of which vocab together weigh less than half of what is cut away are below the limit by mass.  By number it is among the
      // sets' highest, or not far below.
      lo = mass ? top - (log2f(float(row.vocab) / (1.f - fmaxf(l.p, 0.f))) + 2.f) / k : low - 2.f * (top - low);
      float front = 0.f, whole = 0.f;  // the sums of what lies from `beyond` on, of all that is left of rounds before
      for (int level = 0;; ++level) {
        scale            = float(kFine) / (hi - lo) * 0.9999f;
        const float step = k / scale;
        if (!(scale > 0.f && scale < 0x1p100f) || level == 3) return false;
        for (int i = tid; i < kFine; i += threads) S.fine[i] = 0;
        __syncthreads();
        const Interval v{floor, hi, scale, beyond, top, k, step, float(bits), mass, level == 0};
        double sum = mass && floor == 1 ? count_columns<true>(row, team, v, S) : count_columns<false>(row, team, v, S);
        const uint4* fine = reinterpret_cast<const uint4*>(S.fine);
        if constexpr (SPLIT) {
          team.sync();
          sum = warp_sum(lane < team.parts ? team.of(&S, lane)->part_sum : 0.0);
          for (int i = tid; i < kFine / 4; i += threads) {
            uint4 n = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
            for (int c = 0; c < kMaxParts; ++c)
              if (c < team.parts) {
                const uint4 o = reinterpret_cast<const uint4*>(team.of(&S, c)->fine)[i];
                n = make_uint4(n.x + o.x, n.y + o.y, n.z + o.z, n.w + o.w);
              }
            reinterpret_cast<uint4*>(S.fine_all)[i] = n;
          }
          fine = reinterpret_cast<const uint4*>(S.fine_all);
          team.sync();  // the others' are cleared for the next level only when all have read them
        }
        if (mass && level == 0) whole = float(sum);
        if (mass && level > 0) front = float(sum);
        // the interval that the limit falls in, and those that rounding makes possible: four to a lane, by warps
        const float unit = mass ? ldexpf(1.f, -bits) : 1.f, wanted = mass ? fmaxf(l.p, 0.f) * whole : float(l.k);
        const float lead = (hi - top) * k;
        auto weigh       = [&](uint32_t n, int b) { return float(n) * unit * (mass ? pow2(lead - float(b) * step) : 1.f); };
        for (int i = warp; i < kFine / 128; i += warps) {
          const uint4 n = fine[i * 32 + lane];
          const int b   = (i * 32 + lane) * 4;
          const float w = warp_sum((weigh(n.x, b) + weigh(n.y, b + 1)) + (weigh(n.z, b + 2) + weigh(n.w, b + 3)));
          if (lane == 0) S.run[i] = w;
        }
        if (tid == 0) S.first = kFine, S.last = kFine - 1;
        __syncthreads();
        for (int i = warp; i < kFine / 128; i += warps) {
          const uint4 n = fine[i * 32 + lane];
          const int b   = (i * 32 + lane) * 4;
          float w[4]    = {weigh(n.x, b), weigh(n.y, b + 1), weigh(n.z, b + 2), weigh(n.w, b + 3)};
          float upto    = 0.f;
          for (int j = 0; j < i; ++j) upto += S.run[j];
          upto += warp_upto((w[0] + w[1]) + (w[2] + w[3])) - ((w[0] + w[1]) + (w[2] + w[3]));
          int from = kFine, to = kFine - 1;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            upto += w[j];
            const float off = mass ? upto * unit + 1e-5f * wanted : 0.f;
            if (from == kFine && front + upto + off >= wanted) from = b + j;
            if (to == kFine - 1 && front + upto - off >= wanted) to = b + j;
          }
          from = __reduce_min_sync(0xFFFFFFFFu, from), to = __reduce_min_sync(0xFFFFFFFFu, to);
          if (lane == 0) atomicMin(&S.first, from), atomicMin(&S.last, to);
        }
        __syncthreads();
        first = S.first, last = S.last;
        if (first == kFine) return false;  // the limit is further down
        // how many columns that may be
        int n = 0;
        for (int b = first + lane; b <= last; b += 32)
          n += int(float(reinterpret_cast<const uint32_t*>(fine)[b]) * unit * 1.02f * (mass ? pow2(step * 0.5f) : 1.f)) + 1;
        n = warp_sum(n);
        float so_far = 0.f;  // by number, which front and these are exactly
        if (!mass)
          for (int b = lane; b < first; b += 32) so_far += float(reinterpret_cast<const uint32_t*>(fine)[b]);
        if (n <= kMostKeys - 64) break;
        front += warp_sum(so_far);
        // those intervals alone, from one number to another
        const uint32_t key_lo = value_key(fmaxf(lo - (hi - lo) * 1e-3f, -FLT_MAX)), key_hi = value_key(hi) + 1;
        const uint32_t above  = lowest_key(key_lo, key_hi, [&](float x) { return (hi - x) * scale < float(first); });
        const uint32_t within = lowest_key(key_lo, above, [&](float x) { return (hi - x) * scale < float(last + 1); });
        if (above <= within + 1) return false;  // one number
        if (above < key_hi || beyond == INFINITY) beyond = above <= key_top ? key_value(uint64_t(above) << 32) : INFINITY;
        const float next_lo = key_value(uint64_t(within) << 32);
        hi = key_value(uint64_t(above - 1) << 32), lo = next_lo - (hi - next_lo) * 1e-3f;
        __syncthreads();
      }
    }
    // ---- what lies above it, and the columns within
    __syncthreads();
    if (tid == 0) S.keys = 0;
    __syncthreads();
    const float x_least = key_value(uint64_t(key_least) << 32), from_first = float(first), upto_last = float(last + 1);
    const Interval v{floor, hi, scale, beyond, x_least, from_first, upto_last, 0.f, round == 2, false};
    const Above found = round == 1 && floor == 1 && !(l.least > 0.f) ? sum_above<true>(row, team, weight, v, section, S)
                                                                     : sum_above<false>(row, team, weight, v, section, S);
    double sum_all    = found.all;
    int count         = found.count;
    bool cut_short    = found.cut_short;
    const int n = gather_keys(team, S);
    if (n > kMostKeys) return false;
    if constexpr (SPLIT) {
      if (team.part == 0) {
        sum_all         = warp_sum(lane < team.parts ? team.of(&S, lane)->part_sum : 0.0);
        const int other = lane < team.parts ? team.of(&S, lane)->part_count : 0;
        count           = warp_sum(other >> 1);
        cut_short       = __any_sync(0xFFFFFFFFu, other & 1);
        for (int s = team.end + tid; s < row.sections; s += threads) section[s] = team.of(section, s / team.share)[s];
      }
      team.sync();
    }
    // ---- which of these are left
    if (team.part == 0) {
      int left    = 0;
      bool solved = true;
      if (n > 0) {
        __syncthreads();
        sort_down(S.key, n);
        for (int i = tid; i < n; i += threads) S.weight[i] = weight(key_value(S.key[i]));
      }
      __syncthreads();
      if (round == 0) {
        left   = l.k - count;
        solved = left >= 0 && left <= n;
      } else if (round == 1 && !cut_short) {
        const double reach = fmax(0.0, double(l.p)) * sum_all;
        double above       = 0.0;
        for (int s = lane; s < row.sections; s += 32) above += section[s];
        above = warp_sum(above);
        // the list's weights in front of every lane's share of it, by every warp
        const int each = (n + 31) / 32, begin = min(n, lane * each), end = min(n, begin + each);
        double mine = 0.0;
        for (int i = begin; i < end; ++i) mine += S.weight[i];
        double upto = above + warp_upto(mine) - mine;
        left        = INT_MAX;
        for (int i = begin; i < end && left == INT_MAX; ++i)
          if ((upto += S.weight[i]) >= reach) left = i + 1;
        left   = __reduce_min_sync(0xFFFFFFFFu, left);
        solved = above < reach && left != INT_MAX;  // the limit is neither above nor below
      }
      if (solved && left > 0) {
        floor = max(floor, S.key[left - 1]);
      } else if (solved && (round == 0 || (round == 1 && !cut_short))) {  // as many as lie above it
        const uint32_t above = lowest_key(key_lowest, key_top, [&](float x) { return x >= beyond || (hi - x) * scale < from_first; });
        floor                = max(floor, uint64_t(above) << 32);
      }
      if (solved && !(round == 0 && by_mass)) {
        floor = max(floor, uint64_t(key_least) << 32);
        // the sections with what is left of the list, and the draw
        for (int i = tid; i < left; i += threads)
          S.order[i] = uint16_t(S.key[i] >= floor ? int(key_column(S.key[i]) + row.lead) / Row<T>::kColumns : 0xFFFF);
        __syncthreads();
        for (int s = tid; s < row.sections; s += threads) {
          double sum = 0.0;
#pragma unroll 4
          for (int i = 0; i < left; ++i)
            if (S.order[i] == s) sum += S.weight[i];
          section[s] += sum;
        }
        __syncthreads();
        if (warp == 0) {
          double total;
          const Place found = locate(row, l.u, total, [&](int s) { return section[s]; }, [&](int) {
            return [&](const auto& x, int c, auto& w) {
              weight.of(x, w);
#pragma unroll
              for (int j = 0; j < int(sizeof(x) / sizeof(x[0])); ++j) w[j] = rank_key(x[j], uint32_t(c + j)) >= floor ? w[j] : 0.0;
            };
          });
          if (lane == 0) S.column = found.column, S.total = total;
        }
        __syncthreads();
        id      = S.column;
        logprob = id < 0 ? 0.f : float((double(row.value(id)) - m) * l.inverse - log(S.total));
        solved  = id >= 0;
      }
      if (tid == 0) S.solved = solved, S.floor = floor;
    }
    team.sync();
    const Scratch* leader = team.of(&S, 0);
    const bool solved     = leader->solved;
    floor                 = leader->floor;
    team.sync();
    if (!solved || !(round == 0 && by_mass)) return solved;
  }
  return false;
}

// The highest of a thread's sets: the columns of the packs that are q-th in the sections that it has read.
template <class T>
struct Best {
  using P = Pack16<T>;
  typename P::Max of_set[kPacks];
  __device__ __forceinline__ Best()
  {
#pragma unroll
    for (int q = 0; q < kPacks; ++q) of_set[q] = P::lowest();
  }
  __device__ __forceinline__ float value(int q) const
  {
    return P::kHalves == 2 ? fmaxf(P::of(of_set[q], 0), P::of(of_set[q], 1)) : P::of(of_set[q], 0);
  }
};

// A section's sum, relative to 2^c_top.  A broken section's reference is NaN, so that its sum is one too however far below the highest its numbers
// lie (all masked but one, or nothing left of them by a cold temperature).
__device__ __forceinline__ double of_section(const float2& v, float c_top)
{
  const float d = v.x - c_top;
  return d <= -1000.f ? 0.0 : double(v.y) * __hiloint2double((int(d) + 1023) << 20, 0);
}

// locate() with the sums of the first reading, relative to 2^c_top: sections in 64 bits, within its section in 32.
template <class T>
__device__ __forceinline__ Place near_column(const Row<T>& row, const float2* piece, float c_top, float k, double share, double& total, Scratch& S)
{
  constexpr uint32_t all = 0xFFFFFFFFu;
  constexpr int E = Row<T>::E, kOwn = kPacks * E;
  static_assert(kOwn <= 32 && kPacks == 4, "");
  const int lane = threadIdx.x & 31, each = (row.sections + 31) / 32;
  const int begin = min(lane * each, row.sections), end = min(begin + each, row.sections);
  double mine = 0.0;
  for (int i = begin; i < end; ++i) mine += of_section(piece[i], c_top);
  const double upto = warp_upto(mine);
  total             = __shfl_sync(all, upto, 31);
  const double target = share * total;
  uint32_t over = __ballot_sync(all, mine > 0.0 && upto > target);
  if (over == 0) return Place{-1, -1, 0.0, 0.0, 0.f};  // rounding has left none
  int from     = __ffs(over) - 1, s = -1;
  double front = upto - mine;
  if (lane == from)
    for (s = begin; s + 1 < end; ++s) {
      const double w = of_section(piece[s], c_top);
      if (w > 0.0 && front + w > target) break;
      front += w;
    }
  s     = __shfl_sync(all, s, from);
  front = __shfl_sync(all, front, from);
  // neighbouring packs to a lane
  uint4 raw[kPacks];
#pragma unroll
  for (int q = 0; q < kPacks; ++q) raw[q] = row.load((s * 32 + lane) * kPacks + q);
  const float c   = piece[s].x;
  const int shift = int(c_top - c);  // the section has weight, so that is below 1000
  const float rest = float((target - front) * __hiloint2double((1023 + shift) << 20, 0));
  const Two k2(k, k), c2(-c, -c);
  Two sum[kPacks];
#pragma unroll
  for (int q = 0; q < kPacks; ++q) {
    Two x[E / 2];
    Pack16<T>::pairs(raw[q], x);
#pragma unroll
    for (int j = 0; j < E / 2; ++j) {
      float y0, y1;
      gtk::fma2(x[j], k2, c2).get(y0, y1);
      x[j] = Two(pow2(y0), pow2(y1));
    }
#pragma unroll
    for (int d = 1; d < E / 2; d *= 2)
#pragma unroll
      for (int j = 0; j < E / 2; j += 2 * d) x[j] = x[j] + x[j + d];
    sum[q] = x[0];
  }
  float lo, hi;
  ((sum[0] + sum[1]) + (sum[2] + sum[3])).get(lo, hi);
  float own         = lo + hi;
  const float so_far = warp_upto(own);
  over              = __ballot_sync(all, own > 0.f && so_far > rest);
  if (over == 0) return Place{-1, s, 0.0, 0.0, 0.f};
  from = __ffs(over) - 1;
  // a column to a lane
  uint4* const shared = reinterpret_cast<uint4*>(S.key);
  if (lane == from)
#pragma unroll
    for (int q = 0; q < kPacks; ++q) shared[q] = raw[q];
  __syncwarp();
  const float x = lane < kOwn ? gtk::to_float(reinterpret_cast<const T*>(shared)[lane]) : -INFINITY;
  own           = pow2(fmaf(x, k, -c));
  const float in_front = __shfl_sync(all, so_far, max(from - 1, 0));
  const float now      = (from > 0 ? in_front : 0.f) + warp_upto(own);
  over                 = __ballot_sync(all, own > 0.f && now > rest);
  if (over == 0) return Place{-1, s, 0.0, 0.0, 0.f};
  const int at      = __ffs(over) - 1;
  const double unit = __hiloint2double((1023 - shift) << 20, 0);
  const float here  = __shfl_sync(all, now, at), before = here - __shfl_sync(all, own, at);
  return Place{row.column((s * 32 + from) * kPacks) + at, s, front + double(before) * unit, front + double(here) * unit, __shfl_sync(all, x, at)};
}

// The row's highest logit, from the warps' own.
template <bool SPLIT>
__device__ __forceinline__ float highest(const Team<SPLIT>& team, Scratch& S, float top)
{
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  if (lane == 0) S.top[warp] = top;
  __syncthreads();
  top = warp_max(lane < warps ? S.top[lane] : -INFINITY);
  if constexpr (SPLIT) {
    if (threadIdx.x == 0) S.part_top = top;
    team.sync();
    top = warp_max(lane < team.parts ? team.of(&S, lane)->part_top : -INFINITY);  // lane c asks part c, here and below
  }
  return top;
}

// Whether 32 bits hold a row's numbers and their sum, which is positive and finite then.
__device__ __forceinline__ bool fits(bool ranged, float top, float c_top, double sum)
{
  return ranged && fabsf(top) < 0x1p59f && fabsf(c_top) < 0x1p20f && sum > 0.0 && sum < 1e30;
}

// A row without limits: the answer is its first warp's.
template <class T, bool SPLIT>
__device__ __noinline__ int draw_of_all(const Row<T>& row, const Limits& l, const Team<SPLIT>& team, float top, float k, bool ranged, double* section,
                                        Scratch& S, float& logprob)
{
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  top                = highest(team, S, top);
  const float c_top  = ceilf(fmaxf(top, kLow) * k);
  float2* const piece = reinterpret_cast<float2*>(section);
  if constexpr (SPLIT) {
    if (team.part == 0)  // the others' sections behind its own
      for (int s = team.end + int(threadIdx.x); s < row.sections; s += blockDim.x) piece[s] = team.of(piece, s / team.share)[s];
    team.sync();  // nobody leaves while its shared memory is read
    if (team.part != 0) return -1;
  }
  int id = -1;
  if (warp == 0) {
    double total;
    const Place at = near_column(row, piece, c_top, k, l.u, total, S);
    bool sure = fits(ranged, top, c_top, total) && at.column >= 0;
    if (sure) {
      // u sum - (the weights in front): an error of a weight in front counts 1 - u times, of one behind u times, and those of the
      // sections' sums likewise, but for the column's own section
      const double u = l.u, target = u * total;
      const float shares = fmaxf(float(u), 1.f - float(u)), both = 2.f * float(u) * (1.f - float(u));
      const float of_all = row.exponent_error(total) * shares + (Row<T>::kWeightError + Row<T>::kSumError) * both + 0.1f;
      const double off   = 0x1p-24 * (total * of_all + Row<T>::kOwnError * of_section(piece[at.section], c_top));
      sure             = target - at.before >= off && at.upto - target >= off;
      const double shift = double(top) * double(k) - double(c_top);  // the highest's exponent
      logprob            = float((double(at.x) - double(top)) * l.inverse + 0.6931471805599453 * shift - log(total));
      id                 = at.column;
    }
    if (lane == 0) S.sure = sure, S.solved = fits(ranged, top, c_top, total);
  }
  __syncthreads();
  if (S.sure) return id;
  __syncthreads();
  return S.solved ? draw_exactly(row, l, top, section, S, logprob) : draw_slowly(row, l, section, S, logprob);
}

// A row of which the highest alone is left, of equal ones the lowest column: the answer is its first thread's.
template <class T, bool SPLIT>
__device__ __noinline__ int draw_highest(const Row<T>& row, const Limits& l, const Team<SPLIT>& team, const Best<T>& best, float top, double* section,
                                         Scratch& S, float& logprob)
{
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  if (threadIdx.x == 0) S.column = INT_MAX;
  top = highest(team, S, top);
  const float2* const piece = reinterpret_cast<const float2*>(section);
  bool broken = !(fabsf(top) < 0x1p59f);
  for (int s = team.begin + int(threadIdx.x); s < team.end; s += blockDim.x) broken |= !(piece[s].y < 1e30f);  // a NaN, or +inf
  uint32_t column = INT_MAX;
#pragma unroll
  for (int q = 0; q < kPacks; ++q)
    if (best.value(q) == top) {
#pragma unroll 4
      for (int s = team.begin + warp; s < team.end; s += warps) {
        const int p     = (s * kPacks + q) * 32 + lane;
        const uint4 raw = row.load(p);
#pragma unroll
        for (int j = Row<T>::E - 1; j >= 0; --j)
          if (gtk::to_float(reinterpret_cast<const T*>(&raw)[j]) == top) column = min(column, uint32_t(row.column(p) + j));
      }
    }
  column = __reduce_min_sync(0xFFFFFFFFu, column);
  if (lane == 0 && column != INT_MAX) atomicMin(&S.column, int(column));
  broken = __syncthreads_or(broken);
  column = uint32_t(S.column);
  if constexpr (SPLIT) {
    if (threadIdx.x == 0) S.solved = broken;
    team.sync();
    column = __reduce_min_sync(0xFFFFFFFFu, lane < team.parts ? uint32_t(team.of(&S, lane)->column) : INT_MAX);
    broken = __any_sync(0xFFFFFFFFu, lane < team.parts && team.of(&S, lane)->solved);
    team.sync();  // nobody leaves while its shared memory is read
    if (team.part != 0) return -1;
  }
  if (broken) return draw_slowly(row, l, section, S, logprob);
  logprob = 0.f;
  return int(column);
}

// A row with limits: the answer is its first thread's.
template <class T, bool SPLIT>
__device__ __noinline__ int draw_limited(const Row<T>& row, const Limits& l, const Team<SPLIT>& team, const Best<T>& best, float top, float k,
                                         bool ranged, double* section, Scratch& S, float& logprob)
{
  constexpr int E = Row<T>::E, kAgain = 2;  // packs that a thread reads again at a time
  const int tid = threadIdx.x, threads = blockDim.x, warps = threads >> 5, warp = tid >> 5, lane = tid & 31;
  float low = INFINITY;
#pragma unroll
  for (int q = 0; q < kPacks; ++q)
    if (best.value(q) > -INFINITY) low = fminf(low, best.value(q));
  low = warp_min(low);
  if (lane == 0) S.low[warp] = low;
  for (int i = tid; i < kBins; i += threads) S.hist[i] = 0;
  if (tid == 0) S.keys = 0;
  top = highest(team, S, top);
  low = warp_min(lane < warps ? S.low[lane] : INFINITY);
  if constexpr (SPLIT) {
    // the parts' lowest, by way of all their warps
    for (int c = 0; c < team.parts; ++c) low = fminf(low, warp_min(lane < warps ? team.of(&S, c)->low[lane] : INFINITY));
  }

  // ---- the sum of all weights relative to the highest's, and how the sets' highest are distributed
  const float c_top = ceilf(fmaxf(top, kLow) * k);
  const float scale = fminf(float(kBins) / (top - low), 0x1p100f);
  const float2* const piece = reinterpret_cast<const float2*>(section);
  double sum = 0.0;
  for (int s = team.begin + tid; s < team.end; s += threads) sum += of_section(piece[s], c_top);
  sum = warp_sum(sum);
  if (lane == 0) S.mass[warp] = sum;
#pragma unroll
  for (int q = 0; q < kPacks; ++q) {
    const float v = best.value(q);
    if (v > -INFINITY) {
      const int at = int(fminf((top - v) * scale, float(kBins - 1)));
      if (GTK_IN(at, kBins, 504)) atomicAdd(&S.hist[at], 1);
    }
  }
  __syncthreads();
  sum = 0.0;
  for (int w = 0; w < warps; ++w) sum += S.mass[w];
  const int* hist = S.hist;
  if constexpr (SPLIT) {
    if (tid == 0) S.part_sum = sum;
    team.sync();
    sum = warp_sum(lane < team.parts ? team.of(&S, lane)->part_sum : 0.0);
    for (int i = tid; i < kBins; i += threads) {
      int n = 0;
      for (int c = 0; c < team.parts; ++c) n += team.of(&S, c)->hist[i];
      S.bins[i] = n;
    }
    hist = S.bins;
    __syncthreads();
  }
  // rows whose numbers 32 bits do not hold are looked at again, as are those without a distribution
  if (!fits(ranged, top, c_top, sum)) {
    team.sync();  // nobody leaves while its shared memory is read
    return team.part == 0 ? draw_slowly(row, l, section, S, logprob) : -1;
  }
  const double m     = top;
  // ---- how far down the columns have to be known
  const bool by_mass = l.cut_by_mass(), of_all = by_mass && l.k == INT_MAX;  // top-p of all columns
  double error = 0.0;
  if (of_all) {
    error = 0x1p-24 * double(row.exponent_error(sum) + Row<T>::kWeightError + Row<T>::kSumError + 0.1f);
    sum *= exp2(double(c_top) - double(top) * double(k));  // relative to the highest's
  }
  int reach = kBins;
  {
    constexpr int kEach = kBins / 32;
    int counts[kEach], count = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) count += counts[i] = hist[lane * kEach + i];
    int count_upto = warp_upto(count) - count;
    if (of_all) {
      const float width = k / scale, wanted = fmaxf(l.p, 0.f) * float(sum) * 1.0001f;
      float masses[kEach], mass = 0.f;
#pragma unroll
      for (int i = 0; i < kEach; ++i) mass += masses[i] = counts[i] ? float(counts[i]) * pow2(-float(lane * kEach + i + 1) * width) * 0.999f : 0.f;
      float mass_upto = warp_upto(mass) - mass;  // no less than that lies above
#pragma unroll
      for (int i = 0; i < kEach; ++i)
        if ((mass_upto += masses[i]) >= wanted && reach == kBins && counts[i]) reach = lane * kEach + i;
    } else {
#pragma unroll
      for (int i = 0; i < kEach; ++i)
        if ((count_upto += counts[i]) >= l.k && reach == kBins && counts[i]) reach = lane * kEach + i;
    }
    reach = __reduce_min_sync(0xFFFFFFFFu, reach);
    if (l.least > 0.f && (l.k == INT_MAX || !by_mass))
      reach = min(reach, int(fminf(-logf(l.least) * l.t * scale * 1.0001f + 2.f, float(kBins))));
  }
  const bool everything = reach == kBins;
  const float bound     = reach == kBins - 1 ? float(kBins + 1) : float(reach + 1);  // the last one holds the lowest too, however that is rounded
  bool some             = !everything || row.vocab <= kMostKeys;
  if (everything && !some) {  // where most columns are masked, what is left may be few
    int n = 0;
    for (int i = lane; i < kBins; i += 32) n += hist[i];
    some = warp_sum(n) <= kMostKeys / 4;
  }
  if (some) {
    auto reaches        = [&](float x) { return everything || (top - x) * scale < bound; };
    uint8_t* const set  = S.set + warp * kSetsOfWarp;
    static_assert(kSetsOfWarp <= 256, "");
    int sets = 0;
#pragma unroll
    for (int q = 0; q < kPacks; ++q) {
      const float v       = best.value(q);
      const bool mine     = v > -INFINITY && reaches(v);
      const uint32_t them = __ballot_sync(0xFFFFFFFFu, mine);
      const int at        = sets + __popc(them & ((1u << lane) - 1u));
      if (mine && GTK_IN(at, kSetsOfWarp, 505)) set[at] = uint8_t(q * 32 + lane);
      sets += __popc(them);
    }
    __syncwarp();
    const int sections = (team.end - team.begin - warp + warps - 1) / warps, packs = sets * max(0, sections);
    const float per_set = 1.f / float(max(sets, 1));
    for (int i0 = 0; i0 < packs; i0 += 32 * kAgain) {
      uint4 raw[kAgain];
      int column[kAgain];
      uint32_t hits = 0;
#pragma unroll
      for (int e = 0; e < kAgain; ++e) {
        const int i = i0 + e * 32 + lane, s = int((float(i) + 0.5f) * per_set);  // i / sets
        const int p = i < packs ? (team.begin + warp + s * warps) * 32 * kPacks + int(set[i - s * sets]) : row.packs;
        column[e]   = row.column(p);
        raw[e]      = row.load(p);
      }
#pragma unroll
      for (int e = 0; e < kAgain; ++e)
#pragma unroll
        for (int j = 0; j < E; ++j) {
          const float x = gtk::to_float(reinterpret_cast<const T*>(&raw[e])[j]);
          hits |= (x > -INFINITY && reaches(x) ? 1u : 0u) << (e * E + j);
        }
      const int mine = __popc(hits), upto = warp_upto(mine);
      int at = 0;
      if (lane == 31 && upto > 0) at = atomicAdd(&S.keys, upto);
      at = __shfl_sync(0xFFFFFFFFu, at, 31) + upto - mine;
      if (hits == 0) continue;
#pragma unroll
      for (int e = 0; e < kAgain; ++e)
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (hits >> (e * E + j) & 1u) {
            if (at < kMostKeys && GTK_IN(at, kMostKeys, 506))
              S.key[at] = rank_key(gtk::to_float(reinterpret_cast<const T*>(&raw[e])[j]), uint32_t(column[e] + j));
            ++at;
          }
    }
  }
  const int n = gather_keys(team, S);
  if (!some || n > kMostKeys) {
    int id            = -1;
    const bool solved = draw_wide(row, l, team, top, low, section, S, id, logprob);
    team.sync();  // nobody leaves while its shared memory is read
    if (team.part != 0) return -1;
    return solved ? id : draw_slowly(row, l, section, S, logprob);
  }
  if (team.part != 0) return -1;

  // ---- the columns that are known, ranked
  const bool few = n <= threads;
  if (few) {
    if (tid < n) {
      const uint64_t key = S.key[tid];
      const double w     = exp((double(key_value(key)) - m) * l.inverse);
      int rank = 0, place = 0;
#pragma unroll 4
      for (int j = 0; j < n; ++j) {
        const uint64_t other = S.key[j];
        rank += other > key;
        place += uint32_t(other) > uint32_t(key);  // a lower column
      }
      if (GTK_IN(rank, kThreads, 511) && GTK_IN(place, kThreads, 512)) S.ranked[rank] = key, S.weight[rank] = w, S.order[place] = uint16_t(rank);
    }
  } else {
    sort_down(S.key, n);
    for (int i = tid; i < n; i += threads) S.weight[i] = exp((double(key_value(S.key[i])) - m) * l.inverse);
  }
  __syncthreads();
  const uint64_t* ranked = few ? S.ranked : S.key;
  double whole = of_all && !everything ? sum : -1.0, off = error * sum;
  for (int round = 0; round < 2; ++round) {
    if (warp == 0) {
      int left;
      double total;
      const bool sure = cut_keys(l, m, ranked, S.weight, n, whole, off, left, total);
      if (lane == 0) S.sure = sure, S.left = left, S.total = total;
      if (few && sure) {
        const int at = draw_key(S.order, S.weight, n, left, l.u * total);
        if (lane == 0) S.column = at;
      }
    }
    __syncthreads();
    if (S.sure) break;
    __syncthreads();
    whole = sum_exactly(row, l, m, section, S), off = 0.0;
  }
  if (!few) {
    // 20 bits of column, 9 of rank; the lowest column first
    const int left = S.left;
    for (int i = tid; i < left; i += threads) S.by_column[i] = ~(key_column(S.key[i]) << 9 | uint32_t(i));
    __syncthreads();
    static_assert(kMostKeys == 1 << 9 && GTK_MAX_SAMPLE_VOCAB == 1 << 20, "");
    sort_down(S.by_column, left);
    for (int i = tid; i < left; i += threads) S.order[i] = uint16_t(~S.by_column[i] & (kMostKeys - 1));
    __syncthreads();
    if (warp == 0) {
      const int at = draw_key(S.order, S.weight, left, left, l.u * S.total);
      if (lane == 0) S.column = at;
    }
    __syncthreads();
  }
  if (tid != 0) return -1;
  const uint64_t drawn = ranked[S.column];
  logprob              = l.t == 0.f ? 0.f : float((double(key_value(drawn)) - m) * l.inverse - log(S.total));
  return int(key_column(drawn));
}

template <class T, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 4) k_sample(const T* __restrict__ logits, const SampleArgs a, int n_parts)
{
  using P         = Pack16<T>;
  constexpr int E = P::kElems;
  extern __shared__ double s_section[];  // a whole row's
  __shared__ Scratch S;
  const int parts = SPLIT ? n_parts : 1;
  const int tid = threadIdx.x, warps = blockDim.x >> 5, warp = tid >> 5, lane = tid & 31;
  const int64_t r = blockIdx.x / unsigned(parts);
  const int part  = int(blockIdx.x % unsigned(parts));
  const Row<T> row(logits + r * a.stride, a.vocab);
  const int share = (row.sections + parts - 1) / parts;
  const int begin = min(row.sections, part * share), end = min(row.sections, begin + share);
  uint4 raw[kPacks];
  if (begin + warp < end) row.load_section(begin + warp, raw);  // while the limits come in
  const Limits l(a, r);
  auto put = [&](int id, float logprob) {
    if (tid != 0 || part != 0) return;
    a.ids[r] = id;
    if (a.logprob) a.logprob[r] = logprob;
  };
  if (l.u < 0.0) return put(-1, 0.f);
  if (l.broken()) return put(-1, __int_as_float(0x7FC00000));

  // ---- the row, once: a warp's section is summed relative to 2^c, c a whole number, no less than any exponent so far
  const double k64  = 1.4426950408889634 * l.inverse;
  const bool ranged = k64 > 0x1p-20 && k64 < 0x1p20;
  const float k     = ranged ? float(k64) : 1.f;
  float2* const piece = reinterpret_cast<float2*>(s_section);
  Best<T> best;
  float top = -INFINITY, ref = kLow;
  auto take = [&](int s, const uint4 (&raw)[kPacks]) {
    typename P::Max most = P::highest(raw[0]);
    best.of_set[0]       = P::higher(best.of_set[0], most);
#pragma unroll
    for (int q = 1; q < kPacks; ++q) {
      const typename P::Max m = P::highest(raw[q]);
      best.of_set[q]          = P::higher(best.of_set[q], m);
      most                    = P::higher(most, m);
    }
    top = fmaxf(top, warp_max(P::kHalves == 2 ? fmaxf(P::of(most, 0), P::of(most, 1)) : P::of(most, 0)));
    const float c = ceilf(fmaxf(ref, top) * k);
    const Two k2(k, k), c2(-c, -c);
    Two sum[kPacks];
#pragma unroll
    for (int q = 0; q < kPacks; ++q) {
      Two x[E / 2];
      P::pairs(raw[q], x);
#pragma unroll
      for (int j = 0; j < E / 2; ++j) {
        float y0, y1;
        gtk::fma2(x[j], k2, c2).get(y0, y1);
        x[j] = Two(pow2(y0), pow2(y1));
      }
#pragma unroll
      for (int d = 1; d < E / 2; d *= 2)
#pragma unroll
        for (int j = 0; j < E / 2; j += 2 * d) x[j] = x[j] + x[j + d];
      sum[q] = x[0];
    }
#pragma unroll
    for (int d = 1; d < kPacks; d *= 2)
#pragma unroll
      for (int q = 0; q < kPacks; q += 2 * d) sum[q] = sum[q] + sum[q + d];
    float lo, hi;
    sum[0].get(lo, hi);
    lo = warp_sum(lo + hi);
    // NaN where, and only where, the section has a NaN or +inf: rows are told broken by it
    if (lane == 0 && GTK_IN(s, row.sections, 503)) piece[s] = make_float2(isnan(lo) ? lo : c, lo);
  };
  for (int s = begin + warp; s < end; s += 2 * warps) {
    uint4 next[kPacks];
    if (s + warps < end) row.load_section(s + warps, next);
    take(s, raw);
    if (s + warps >= end) break;
    if (s + 2 * warps < end) row.load_section(s + 2 * warps, raw);
    take(s + warps, next);
  }
  const Team<SPLIT> team{parts, part, share, begin, end};
  float logprob = 0.f;
  const int id  = l.all()    ? draw_of_all(row, l, team, top, k, ranged, s_section, S, logprob)
                  : l.k == 1 ? draw_highest(row, l, team, best, top, s_section, S, logprob)
                             : draw_limited(row, l, team, best, top, k, ranged, s_section, S, logprob);
  put(id, logprob);
}

static_assert(sizeof(Scratch) + (GTK_MAX_SAMPLE_VOCAB / (32 * kPacks * 4) + 1) * sizeof(double) <= 48 << 10, "what a CTA has without asking");

// How many CTAs share a row, and how many threads they have.
// When the rule was chosen, in 1 / 2 / 4 / 8 parts of 256 threads, us: one row of 50257 bf16 without limits - / 9.8 / 8.9 / 8.4, 64 of 131072 f32
// 23.7 / 15.9 / 12.7 / 14, with the 50 highest 42 / 25 / 19 / 22; 148 of 50257 bf16 9.8 / 9.8 / 13.1, with limits 16.7 / 16.9 / 27; 256 of f32
// 21.6 / 23.2 / 28.  A nucleus may be wide, and a wide row is bound by instructions: 256 rows of 50304 f32, a few of them wide, took 102 / 74 / 66,
// with none 27 / 25 / 36; 333 of 32003 fp16, all of them wide, 84 / 119 / 162.
// At its borders now, a row less in two parts and a row more in one: 74 and 75 nuclei of 50257 bf16 (0.95 at T = 0.8) 60 and 72, 0.99 at 1.3
// 67 and 80; 296 and 297 of f32 102 and 112, 112 and 119.  Nuclei of rows between were not measured in both ways.
// Rows in numbers take 128 threads, so that more of them are under way while others are at their ends: of 256 / 128, 2048 rows of 50257 f32
// 80 / 73, bf16 50 / 45, with min-p 73 / 63; 512 of bf16 24 / 28.
struct Teams {
  int parts, threads;
};
Teams teams_for(int64_t rows, int64_t bytes, bool nuclei, int sm_count)
{
  Teams t{1, kThreads};
  const int64_t room = int64_t(sm_count) * (bytes >= (160 << 10) ? 2 : 1);
  while (t.parts < kMaxParts && rows * t.parts * 2 <= room && bytes / (t.parts * 2) >= (12 << 10)) t.parts *= 2;
  if (nuclei && t.parts == 1 && bytes >= (160 << 10) && rows * 2 <= int64_t(sm_count) * 4) t.parts = 2;
  if (rows > int64_t(sm_count) * 8 && bytes <= (256 << 10)) t.threads = 128;
  return t;
}

template <class T>
cudaError_t launch_sample(const gtk::HandleView& v, const void* logits, int64_t n_rows, const SampleArgs& a)
{
  const Teams t         = teams_for(n_rows, int64_t(a.vocab) * int64_t(sizeof(T)), a.top_p != nullptr, v.sm_count);
  const size_t sections = (size_t(a.vocab) + Row<T>::E + Row<T>::kColumns - 1) / Row<T>::kColumns;
  const auto kernel = t.parts > 1 ? k_sample<T, true> : k_sample<T, false>;
  return gtk::launch_clusters(kernel, dim3(unsigned(n_rows * t.parts)), dim3(unsigned(t.threads)),
                              t.parts, sections * sizeof(double), v.stream, static_cast<const T*>(logits), a, t.parts);
}

constexpr int64_t kMaxRows = (int64_t(1) << 31) - 1;

}  // namespace

extern "C" GTK_API int gtk_sample(gtk_tokenizer* h, const void* d_logits, int type, int64_t n_rows, int64_t vocab, int64_t stride,
                                  const double* d_uniform, const float* d_temperature, const int32_t* d_top_k, const float* d_top_p,
                                  const float* d_min_p, int32_t* d_ids, float* d_logprob)
{
  auto check = [&]() -> gtk::Refusal {
    if (!gtk::known_type(type)) return "unknown element type";
    if (n_rows < 0 || vocab <= 0 || stride < 0) return "n_rows and stride must be >= 0, vocab > 0";
    if (n_rows > kMaxRows || vocab > GTK_MAX_SAMPLE_VOCAB) return "n_rows of 2^31 and more, or vocab beyond 2^20";
    if (n_rows == 0) return nullptr;
    if (!d_logits || !d_uniform || !d_ids) return "null device pointer";
    if (!gtk::aligned_to(d_logits, gtk::element_size(type)) || !gtk::aligned_to(d_uniform, 8))
      return "a device pointer is not aligned to its elements";
    for (const void* q : {static_cast<const void*>(d_temperature), static_cast<const void*>(d_top_k), static_cast<const void*>(d_top_p),
                          static_cast<const void*>(d_min_p), static_cast<const void*>(d_ids), static_cast<const void*>(d_logprob)})
      if (!gtk::aligned_to(q, 4)) return "a device pointer is not aligned to its elements";
    return nullptr;
  };
  return gtk::run_operator(h, check, [&](const gtk::HandleView& v) -> cudaError_t {
    if (n_rows == 0) return cudaSuccess;
    const SampleArgs a{int(vocab), stride, d_uniform, d_temperature, d_top_p, d_min_p, d_top_k, d_ids, d_logprob};
    return gtk::with_type(type, [&](auto x) { return launch_sample<decltype(x)>(v, d_logits, n_rows, a); });
  });
}

#ifdef GTK_CHECKED
cudaError_t gtk::sample_check_words(int sum[4], bool reset) { return add_check_words(sum, reset); }
cudaError_t gtk::sample_check_selftest() { return check_selftest(599); }
#endif
