// gtk_sample.cu -- an id drawn per row of logits, with temperature, top-k, top-p and min-p, from a given random number.
//
// With m a row's maximum and w_j = exp((x_j - m) / T), columns ranked by logit, of equal ones the lower first: the first K = top_k are
// looked at; of these the fewest whose weights reach top_p of their sum; of these those with w_j >= min_p.  The id is the first
// column, in the order of columns, at which the sum of the weights that are left exceeds u times the whole of it.
#include <climits>
#include <cmath>

#include "gtk_checked.cuh"
#include "gtk_logits.cuh"

namespace {

using gtk::key_column;
using gtk::key_value;
using gtk::rank_key;
using gtk::value_key;

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kSection = 1024, kMostSections = 1024;  // columns whose sums are kept, and how many of those a row has at most

struct SampleArgs {
  int vocab;
  int64_t stride;
  const double* uniform;
  const float *temperature, *top_p, *min_p;
  const int32_t* top_k;
  int32_t* ids;
  float* logprob;
};

struct Scratch {
  double section[kMostSections];
  double mass[kWarps];
  int count[kWarps];
  double at, total;
  int column;
};

struct Sum {
  double mass;
  int count;
};

// f(x, column) -> {weight, counted} over all columns, by all threads
template <class T, class F>
__device__ Sum sum_row(const T* x, int vocab, Scratch& S, F&& f)
{
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  Sum s{0.0, 0};
  for (int c = tid; c < vocab; c += kThreads) {
    const Sum o = f(gtk::to_float(x[c]), c);
    s.mass += o.mass, s.count += o.count;
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    s.mass += __shfl_xor_sync(0xFFFFFFFFu, s.mass, d);
    s.count += __shfl_xor_sync(0xFFFFFFFFu, s.count, d);
  }
  __syncthreads();
  if (lane == 0) S.mass[warp] = s.mass, S.count[warp] = s.count;
  __syncthreads();
  s = Sum{0.0, 0};
  for (int w = 0; w < kWarps; ++w) s.mass += S.mass[w], s.count += S.count[w];
  return s;
}

// The first column at which the sum of f(x, column) exceeds the target, which is `share` of the whole where `of_whole`; the last column
// with any weight where rounding leaves none, -1 where no column has any.  S.total is the whole.
template <class T, class F>
__device__ int locate(const T* x, int vocab, Scratch& S, bool of_whole, double share, F&& f)
{
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int sections = (vocab + kSection - 1) / kSection;
  __syncthreads();
  for (int s = warp; s < sections; s += kWarps) {
    double sum = 0.0;
    for (int c = s * kSection + lane; c < min(vocab, (s + 1) * kSection); c += 32) sum += f(gtk::to_float(x[c]), c);
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
    if (lane == 0) S.section[s] = sum;
  }
  __syncthreads();
  if (tid == 0) {
    double total = 0.0;
    for (int s = 0; s < sections; ++s) total += S.section[s];
    const double target = of_whole ? share * total : share;
    double front = 0.0;
    int found = -1, last = -1;
    double before_last = 0.0;
    for (int s = 0; s < sections && found < 0; ++s) {
      if (S.section[s] > 0.0) last = s, before_last = front;
      if (front + S.section[s] > target) found = s;
      else front += S.section[s];
    }
    if (found < 0) found = last, front = before_last;
    S.column = found, S.at = front, S.total = total;
  }
  __syncthreads();
  const int s = S.column;
  const double target = of_whole ? share * S.total : share;
  __syncthreads();
  if (s >= 0 && warp == 0) {
    double front = S.at;
    int found = -1, last = -1;
    for (int c0 = s * kSection; c0 < min(vocab, (s + 1) * kSection) && found < 0; c0 += 32) {
      const int c    = c0 + lane;
      const double w = c < vocab ? f(gtk::to_float(x[c]), c) : 0.0;
      double upto    = w;
#pragma unroll
      for (int d = 1; d < 32; d *= 2) {
        const double l = __shfl_up_sync(0xFFFFFFFFu, upto, d);
        if (lane >= d) upto += l;
      }
      const uint32_t over = __ballot_sync(0xFFFFFFFFu, w > 0.0 && front + upto > target), some = __ballot_sync(0xFFFFFFFFu, w > 0.0);
      if (over) found = c0 + __ffs(over) - 1;
      if (some) last = c0 + 31 - __clz(some);
      front += __shfl_sync(0xFFFFFFFFu, upto, 31);
    }
    if (lane == 0) S.column = found >= 0 ? found : last;
  }
  __syncthreads();
  return S.column;
}

template <class T>
__global__ void __launch_bounds__(kThreads) k_sample(const T* __restrict__ logits, const SampleArgs a)
{
  __shared__ Scratch S;
  const int64_t r = blockIdx.x;
  const T* x      = logits + r * a.stride;
  const int tid = threadIdx.x, vocab = a.vocab;
  const float nan = __int_as_float(0x7FC00000);
  auto put        = [&](int id, float logprob) {
    if (tid != 0) return;
    a.ids[r] = id;
    if (a.logprob) a.logprob[r] = logprob;
  };
  const double u = a.uniform[r];
  if (u < 0.0) return put(-1, 0.f);
  const float t = a.temperature ? a.temperature[r] : 1.f, p = a.top_p ? a.top_p[r] : 1.f, least = a.min_p ? a.min_p[r] : 0.f;
  const int k   = t == 0.f ? 1 : a.top_k ? a.top_k[r] : 0;
  // the maximum; a row with a NaN or +inf is none
  bool broken = !(t >= 0.f && t < INFINITY) || isnan(p) || isnan(least) || isnan(u);
  uint32_t most = 0;
  int some = 0;
  for (int c = tid; c < vocab; c += kThreads) {
    const float v = gtk::to_float(x[c]);
    broken |= !(v < INFINITY);
    most = max(most, value_key(v));
    some += v > -INFINITY;
  }
  if (__syncthreads_or(broken)) return put(-1, nan);
#pragma unroll
  for (int d = 16; d; d >>= 1) some += __shfl_xor_sync(0xFFFFFFFFu, some, d);
  most = __reduce_max_sync(0xFFFFFFFFu, most);
  if ((tid & 31) == 0) S.count[tid >> 5] = int(most), S.mass[tid >> 5] = some;
  __syncthreads();
  some = 0;
  for (int w = 0; w < kWarps; ++w) most = max(most, uint32_t(S.count[w])), some += int(S.mass[w]);
  if (some == 0) return put(-1, -INFINITY);
  const double m = key_value(uint64_t(most) << 32), inverse = t == 0.f ? 1.0 : 1.0 / double(t);
  auto weight    = [&](float v) { return v > -INFINITY ? exp((double(v) - m) * inverse) : 0.0; };
  uint64_t floor = 0;  // what is left reaches it, see rank_key
  auto left      = [&](float v, int c) { return rank_key(v, uint32_t(c)) >= max(floor, uint64_t(1)); };
  // Lowers the floor from the highest: to the highest value at which enough(sum over the columns that reach it) holds, then to as many
  // columns of that value as are wanted(sum over those above it).
  auto search = [&](auto&& enough, auto&& wanted) {
    uint32_t lo = 0, hi = most;  // enough at lo
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo + 1) / 2;
      const Sum s = sum_row(x, vocab, S, [&](float v, int c) { return value_key(v) >= mid && left(v, c) ? Sum{weight(v), 1} : Sum{0.0, 0}; });
      if (enough(s)) lo = mid;
      else hi = mid - 1;
    }
    const Sum above = sum_row(x, vocab, S, [&](float v, int c) { return value_key(v) > lo && left(v, c) ? Sum{weight(v), 1} : Sum{0.0, 0}; });
    const float value = key_value(uint64_t(lo) << 32);
    const int column  = locate(x, vocab, S, false, wanted(above, weight(value)) - 1.0,
                               [&](float v, int c) { return value_key(v) == lo && left(v, c) ? 1.0 : 0.0; });
    floor             = max(floor, rank_key(value, uint32_t(column)));
  };
  if (k > 0 && k < some)
    search([&](const Sum& s) { return s.count >= k; }, [&](const Sum& s, double) { return double(k - s.count); });
  if (p < 1.f && t > 0.f) {
    const double whole = sum_row(x, vocab, S, [&](float v, int c) { return left(v, c) ? Sum{weight(v), 1} : Sum{0.0, 0}; }).mass;
    const double reach = max(0.0, double(p)) * whole;
    search([&](const Sum& s) { return s.mass >= reach; },
           [&](const Sum& s, double w) {
             double n = max(1.0, w > 0.0 ? ceil((reach - s.mass) / w) : 1.0);
             if (n > 1.0 && s.mass + (n - 1.0) * w >= reach) n -= 1.0;
             return n;
           });
  }
  const double least_y = least > 0.f ? log(min(1.0, double(least))) : -INFINITY;
  auto drawn           = [&](float v, int c) { return left(v, c) && (double(v) - m) * inverse >= least_y ? weight(v) : 0.0; };
  const int id         = locate(x, vocab, S, true, min(u, 1.0), drawn);
  put(id, t == 0.f ? 0.f : float((double(gtk::to_float(x[id])) - m) * inverse - log(S.total)));
}

constexpr int64_t kMaxVocab = int64_t(kSection) * kMostSections, kMaxRows = (int64_t(1) << 31) - 1;

}  // namespace

extern "C" GTK_API int gtk_sample(gtk_tokenizer* h, const void* d_logits, int type, int64_t n_rows, int64_t vocab, int64_t stride,
                                  const double* d_uniform, const float* d_temperature, const int32_t* d_top_k, const float* d_top_p,
                                  const float* d_min_p, int32_t* d_ids, float* d_logprob)
{
  auto check = [&]() -> gtk::Refusal {
    if (!gtk::known_type(type)) return "unknown element type";
    if (n_rows < 0 || vocab <= 0 || stride < 0) return "n_rows and stride must be >= 0, vocab > 0";
    if (n_rows > kMaxRows || vocab > kMaxVocab) return "n_rows of 2^31 and more, or vocab beyond 2^20";
    if (n_rows == 0) return nullptr;
    if (!d_logits || !d_uniform || !d_ids) return "null device pointer";
    if (!gtk::aligned_to(d_logits, gtk::element_size(type)) || !gtk::aligned_to(d_uniform, 8)) return "a device pointer is not aligned to its elements";
    for (const void* q : {static_cast<const void*>(d_temperature), static_cast<const void*>(d_top_k), static_cast<const void*>(d_top_p),
                          static_cast<const void*>(d_min_p), static_cast<const void*>(d_ids), static_cast<const void*>(d_logprob)})
      if (!gtk::aligned_to(q, 4)) return "a device pointer is not aligned to its elements";
    return nullptr;
  };
  return gtk::run_operator(h, check, [&](const gtk::HandleView& v) -> cudaError_t {
    if (n_rows == 0) return cudaSuccess;
    const SampleArgs a{int(vocab), stride, d_uniform, d_temperature, d_top_p, d_min_p, d_top_k, d_ids, d_logprob};
    return gtk::with_type(type, [&](auto x) {
      using T = decltype(x);
      return gtk::launch(k_sample<T>, dim3(unsigned(n_rows)), dim3(kThreads), 0, v.stream, static_cast<const T*>(d_logits), a);
    });
  });
}

#ifdef GTK_CHECKED
cudaError_t gtk::sample_check_words(int sum[4], bool reset) { return add_check_words(sum, reset); }
cudaError_t gtk::sample_check_selftest() { return check_selftest(599); }
#endif
