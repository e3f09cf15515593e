// gtk_logprobs.cu -- log probabilities of given tokens, entropy and top alternatives of rows of logits, and the
// gradient of the first two.
#include <cfloat>
#include <cmath>
#include <initializer_list>

#include "gtk_rows.cuh"

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr float kLn2 = 0.693147180559945309f, kLog2e = 1.44269504088896341f;

// exp2 of a number <= 0 (or NaN)
__device__ __forceinline__ float pow2(float y)
{
  float p;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p) : "f"(y));
  return p;
}

// What has been seen of a row: m the highest logit so far (starts at the lowest finite number, so that masked places at
// -inf never meet it in a difference of infinities), s the sum of 2^y and t that of 2^y * y with y = (x - m) * k,
// k = scale * log2(e).  Joining two: both are moved to the higher m.
struct RowSum {
  float m = -FLT_MAX, s = 0.f, t = 0.f;

  // y of an element that contributes nothing may be -inf: 0 * -inf is kept out of t.  A NaN stays one through 2^y.
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
  __device__ __forceinline__ void join(RowSum o, float k)
  {
    if (o.m > m) raise(o.m, k);
    else o.raise(m, k);
    s += o.s;
    t += o.t;
  }
};

__device__ __forceinline__ RowSum shuffled(const RowSum& a, int mask)
{
  RowSum b;
  b.m = __shfl_xor_sync(0xFFFFFFFFu, a.m, mask);
  b.s = __shfl_xor_sync(0xFFFFFFFFu, a.s, mask);
  b.t = __shfl_xor_sync(0xFFFFFFFFu, a.t, mask);
  return b;
}

// Logits as whole numbers in their order (-0 as 0), the lower column the higher number among equals.
__device__ __forceinline__ uint64_t rank_key(float x, uint32_t column)
{
  const uint32_t b = __float_as_uint(x + 0.f);
  return uint64_t(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | ~column;
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

template <class T>
__global__ void __launch_bounds__(kThreads) k_token_logprobs(const T* __restrict__ logits, const ScoreArgs a)
{
  __shared__ RowSum s_sum[kWarps];
  __shared__ uint64_t s_key[kWarps];
  const int64_t row = blockIdx.x;
  const T* x        = logits + row * a.stride;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float k = a.scale * kLog2e;
  RowSum sum;
  for (int c = threadIdx.x; c < a.vocab; c += kThreads) sum.add(gtk::to_float(x[c]), k);
#pragma unroll
  for (int d = 16; d; d >>= 1) sum.join(shuffled(sum, d), k);
  if (lane == 0) s_sum[warp] = sum;
  __syncthreads();
  sum = s_sum[0];
  for (int w = 1; w < kWarps; ++w) sum.join(s_sum[w], k);
  const float log_sum = logf(sum.s);  // -inf: nothing allowed, NaN: no distribution
  const bool none = sum.s == 0.f, broken = isnan(sum.s);
  const float nan = __int_as_float(0x7FC00000);
  if (threadIdx.x == 0) {
    if (a.logprob) {
      const int t = a.targets[row];
      float lp    = t < 0 ? 0.f : nan;
      if (t >= 0 && t < a.vocab && !broken) lp = none ? -INFINITY : (gtk::to_float(x[t]) - sum.m) * a.scale - log_sum;
      a.logprob[row] = lp;
    }
    if (a.entropy) a.entropy[row] = none ? 0.f : broken ? nan : fmaxf(log_sum - kLn2 * sum.t / sum.s, 0.f);
    if (a.lse) a.lse[row] = none ? -INFINITY : broken ? nan : fmaf(sum.m, a.scale, log_sum);
  }
  uint64_t below = ~uint64_t(0);
  for (int i = 0; i < a.top_k; ++i) {
    uint64_t best = 0;
    if (!broken)
      for (int c = threadIdx.x; c < a.vocab; c += kThreads) {
        const float v      = gtk::to_float(x[c]);
        const uint64_t key = rank_key(v, uint32_t(c));
        if (v > -INFINITY && key < below && key > best) best = key;
      }
#pragma unroll
    for (int d = 16; d; d >>= 1) best = max(best, uint64_t(__shfl_xor_sync(0xFFFFFFFFu, best, d)));
    __syncthreads();
    if (lane == 0) s_key[warp] = best;
    __syncthreads();
    for (int w = 0; w < kWarps; ++w) best = max(best, s_key[w]);
    below = best;
    if (threadIdx.x == 0) {
      if (a.top_ids) a.top_ids[row * a.top_k + i] = best ? int32_t(key_column(best)) : -1;
      if (a.top_logprobs)
        a.top_logprobs[row * a.top_k + i] = broken ? nan : best ? (key_value(best) - sum.m) * a.scale - log_sum : -INFINITY;
    }
    if (!best) below = 0;
  }
}

struct ScoreGradArgs {
  int vocab;
  int64_t stride, grad_stride;
  float scale;
  const int32_t* targets;
  const float *lse, *entropy, *grad_logprob, *grad_entropy;
};

template <class T>
__global__ void __launch_bounds__(kThreads) k_token_logprobs_grad(const T* logits, T* grad, const ScoreGradArgs a)
{
  const int64_t row = blockIdx.x;
  const T* x        = logits + row * a.stride;
  T* dx             = grad + row * a.grad_stride;
  const int t       = a.grad_logprob ? a.targets[row] : -1;
  const float g     = t >= 0 && t < a.vocab ? a.grad_logprob[row] : 0.f;
  const float e     = a.grad_entropy ? a.grad_entropy[row] : 0.f;
  const float lse   = a.lse[row];
  const bool nothing = lse == -INFINITY || ((t < 0 || t >= a.vocab) && !a.grad_entropy);
  const float H      = a.grad_entropy ? a.entropy[row] : 0.f;
  for (int c = threadIdx.x; c < a.vocab; c += kThreads) {
    float d = 0.f;
    if (!nothing) {
      const float z = fmaf(gtk::to_float(x[c]), a.scale, -lse), p = pow2(z * kLog2e);
      d = -p * fmaf(e, fmaxf(z, -1e4f) + H, g);
      if (c == t) d += g;
      d *= a.scale;
    }
    dx[c] = gtk::from_float<T>(d);
  }
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
      return gtk::launch(k_token_logprobs<T>, dim3(unsigned(n_rows)), dim3(kThreads), 0, v.stream, static_cast<const T*>(d_logits), a);
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
      return gtk::launch(k_token_logprobs_grad<T>, dim3(unsigned(n_rows)), dim3(kThreads), 0, v.stream, static_cast<const T*>(d_logits),
                         static_cast<T*>(d_grad_logits), a);
    });
  });
}
