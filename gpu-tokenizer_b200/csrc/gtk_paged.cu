// gtk_paged.cu -- the bookkeeping of a cache in blocks: which blocks requests hold, and where their new tokens go.
//
// With B tokens per block, a request of L tokens holds ceil(L / B) blocks, and its token j lies in slot
// table[j / B] * B + j % B.  Blocks that nobody holds wait in a ring: taken at its head, given back at its tail.
//
// A step moves little: what it takes is launches, sums over all requests, and loads that wait for each other.  Measured in a graph of calls behind
// each other: blocks of 256 requests 7.9 us, of 8192 of which half are replaced 17 (205 by one CTA that moves all of them); slots of 256
// tokens 4.2, of a million of 512 requests 9.6 (floor 2.6; 18 with a search for each token), of 8192 requests 19.6, of one token each 12.7,
// and of 8193, offsets first, 23.7.
#include <climits>

#include "gtk_checked.cuh"
#include "gtk_rows.cuh"

namespace {

constexpr int kThreads = 1024, kWarps = kThreads / 32;

// Division by a number that stays the same, of numbers below 2^31: a multiplication by ceil(2^(31 + s) / d), s = ceil(log2 d), is off by less
// than one part in 2^31 of the quotient's last place (Granlund and Montgomery 1994).
struct Divisor {
  uint32_t d, m;
  int s;
  __host__ explicit Divisor(int by) : d(uint32_t(by)), s(0)
  {
    while ((uint64_t(1) << s) < d) ++s;
    m = uint32_t(((uint64_t(1) << (31 + s)) + d - 1) / d);
  }
  __device__ __forceinline__ uint32_t of(uint32_t x) const { return uint32_t((uint64_t(x) * m) >> (31 + s)); }
};

struct Requests {
  const int32_t *old_lengths, *new_lengths;
  int64_t n;
  Divisor block;
};

struct StepArgs {
  Requests q;
  int32_t* tables;
  int64_t columns, stride;
  int32_t* queue;
  int64_t capacity;
  const int64_t* state;
  int64_t* state_out;
};

// Blocks that a request holds before the step and after it; none of either where it is no request.
struct Blocks {
  uint32_t have = 0, need = 0;
  __device__ __forceinline__ Blocks(const Requests& q, int64_t r)
  {
    if (r >= q.n) return;
    const int32_t before = __ldg(q.old_lengths + r), after = __ldg(q.new_lengths + r);
    if (before < 0 || after < 0) return;
    have = before ? q.block.of(uint32_t(before) - 1u) + 1u : 0u;
    need = after ? q.block.of(uint32_t(after) - 1u) + 1u : 0u;
  }
  __device__ __forceinline__ uint32_t taken() const { return need > have ? need - have : 0u; }
  __device__ __forceinline__ uint32_t given() const { return have > need ? have - need : 0u; }
};

__device__ __forceinline__ int64_t warp_sum(int64_t x)
{
#pragma unroll
  for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xFFFFFFFFu, x, d);
  return x;
}
__device__ __forceinline__ int64_t warp_upto(int64_t x)
{
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int64_t l = __shfl_up_sync(0xFFFFFFFFu, x, d);
    if (lane >= d) x += l;
  }
  return x;
}

struct Pair {
  int64_t a, b;
};

// Of two numbers per thread the sums up to the own ones, and of all; every thread of the CTA.
__device__ __forceinline__ Pair block_upto(Pair x, Pair& all, Pair (&s_sum)[kWarps])
{
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  x.a = warp_upto(x.a), x.b = warp_upto(x.b);
  __syncthreads();
  if (lane == 31) s_sum[warp] = x;
  __syncthreads();
  const Pair w = s_sum[lane];  // as many warps as lanes
  all          = Pair{warp_sum(w.a), warp_sum(w.b)};
  x.a += warp_sum(lane < warp ? w.a : 0), x.b += warp_sum(lane < warp ? w.b : 0);
  return x;
}
static_assert(kWarps == 32, "");

// Each CTA forms the sums over all requests by itself (they are read from L2: 64 KiB for 8192 of them), and then moves the blocks of a share of
// the requests, in tiles of a thread each; a warp moves those of one request after the other.  The state is written by the kernel behind this
// one, when all have read it.
struct StepStatus {
  int64_t taken, given, status;
};
__device__ __forceinline__ StepStatus look_at_step(const StepArgs& a, int64_t begin, Pair& before, Pair (&s_sum)[kWarps])
{
  const int tid = threadIdx.x;
  Pair front{0, 0}, rest{0, 0};  // of the requests in front of `begin`, and from there on
  bool beyond = false;
#pragma unroll 4
  for (int64_t r = tid; r < a.q.n; r += kThreads) {
    const Blocks b(a.q, r);
    Pair& to = r < begin ? front : rest;
    to.a += b.taken(), to.b += b.given();
    beyond |= int64_t(max(b.have, b.need)) > a.columns;
  }
  beyond = __syncthreads_or(beyond);
  Pair all;
  block_upto(front, before, s_sum);
  block_upto(rest, all, s_sum);
  StepStatus s{before.a + all.a, before.b + all.b, 0};
  // The counts may be anything.  Their difference and sum wrap: with a head and a new tail that are not negative and a difference that is
  // no more than the places for what comes back, neither has.
  const uint64_t head = uint64_t(a.state[0]), tail = uint64_t(a.state[1]), waiting = tail - head;
  const int64_t room = a.capacity - s.given;
  if (beyond) s.status = -1;
  else if ((int64_t(head) | int64_t(tail + uint64_t(s.given)) | room) < 0 || waiting > uint64_t(room)) s.status = -2;
  else if (s.taken > int64_t(waiting)) s.status = s.taken - int64_t(waiting);
  return s;
}

__device__ __forceinline__ void put_state(const StepArgs& a, const StepStatus& s)
{
  const int64_t head = a.state[0], tail = a.state[1];
  a.state_out[0] = s.status ? head : head + s.taken;
  a.state_out[1] = s.status ? tail : tail + s.given;
  a.state_out[2] = s.status;
}

template <bool ALONE>
__global__ void __launch_bounds__(kThreads) k_block_tables(const StepArgs a, int64_t share)
{
  __shared__ Pair s_sum[kWarps];
  __shared__ uint32_t s_have[kThreads], s_need[kThreads], s_from[kThreads];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t begin = min(a.q.n, blockIdx.x * share), end = min(a.q.n, begin + share);
  Pair before;
  const StepStatus s = look_at_step(a, begin, before, s_sum);
  const int64_t head = a.state[0], tail = a.state[1];
  if constexpr (ALONE) {
    __syncthreads();  // all have read the state
    if (tid == 0) put_state(a, s);
  }
  if (s.status) return;
  const uint32_t capacity = uint32_t(a.capacity), at_head = uint32_t(head % a.capacity), at_tail = uint32_t(tail % a.capacity);
  // places in the ring; a step moves no more blocks than it has
  auto place = [&](uint32_t from, uint32_t i) {
    const uint32_t p = from + i;  // both below 2^31
    return p >= capacity ? p - capacity : p;
  };
  for (int64_t first = begin; first < end; first += kThreads) {
    Blocks b(a.q, first + tid);
    if (first + tid >= end) b.have = b.need = 0;
    Pair all;
    const Pair upto = block_upto(Pair{int64_t(b.taken()), int64_t(b.given())}, all, s_sum);
    s_have[tid] = b.have, s_need[tid] = b.need;
    s_from[tid] = b.need > b.have ? place(at_head, uint32_t(before.a + upto.a - b.taken())) : place(at_tail, uint32_t(before.b + upto.b - b.given()));
    before.a += all.a, before.b += all.b;
    __syncthreads();
    const int rows = int(min(int64_t(kThreads), end - first));
    // a warp's requests lie kWarps apart: lane l knows of the l-th of them
    const int own     = warp + lane * kWarps;
    uint32_t some     = __ballot_sync(0xFFFFFFFFu, own < rows && s_have[own] != s_need[own]);
    static_assert(kThreads == 32 * kWarps, "");
    while (some) {
      const int r = warp + (__ffs(some) - 1) * kWarps;
      some &= some - 1;
      const uint32_t have = s_have[r], need = s_need[r], from = s_from[r];
      int32_t* row = a.tables + (first + r) * a.stride;
#pragma unroll 4
      for (uint32_t i = have + lane; i < need; i += 32) {
        const uint32_t p = place(from, i - have);
        if (GTK_IN(p, capacity, 400) && GTK_IN(i, a.columns, 401)) row[i] = __ldcg(a.queue + p);
      }
#pragma unroll 4
      for (uint32_t i = need + lane; i < have; i += 32) {
        const uint32_t p = place(from, i - need);
        if (GTK_IN(p, capacity, 402) && GTK_IN(i, a.columns, 403)) a.queue[p] = row[i];
      }
    }
    __syncthreads();
  }
}

// What k_block_tables<false> has found, again, when all of its CTAs are through.
__global__ void __launch_bounds__(kThreads) k_block_state(const StepArgs a)
{
  __shared__ Pair s_sum[kWarps];
  Pair before;
  const StepStatus s = look_at_step(a, 0, before, s_sum);
  gtk::await_kernel();
  __syncthreads();
  if (threadIdx.x == 0) put_state(a, s);
}

struct SlotArgs {
  Requests q;
  const int32_t* tables;
  int64_t columns, stride;
  const int64_t* state;
  int64_t capacity;
  int64_t* slots;
  int32_t *positions, *requests;
  int64_t* offsets;
};

__device__ __forceinline__ int64_t new_tokens(const SlotArgs& a, int64_t r)
{
  const int32_t before = __ldg(a.q.old_lengths + r), after = __ldg(a.q.new_lengths + r);
  return before >= 0 && after > before ? int64_t(after) - before : 0;
}

// The tokens [begin, end) of the step, those below `total` of requests [first, n), which offset_at(request) tells the owners of, by all threads; a
// warp takes neighbouring ones, and looks for a request among all only where it is not the one of the token 32 places before.
template <class OffsetAt>
__device__ __forceinline__ void put_slots(const SlotArgs& a, int64_t begin, int64_t end, int64_t first, int64_t n, int64_t total,
                                          OffsetAt&& offset_at)
{
  constexpr int kOnce = 4;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t each = ((end - begin + kWarps - 1) / kWarps + 31) / 32 * 32;
  // the last request from lo on that begins at i or before, for i < total
  auto owner = [&](int64_t lo, int64_t i) {
    int64_t hi = n;
    while (hi - lo > 1) {
      const int64_t mid = (lo + hi) / 2;
      if (offset_at(mid) <= i) lo = mid;
      else hi = mid;
    }
    return lo;
  };
  const int64_t from = begin + warp * each, to = min(end, from + each);
  int64_t lo = from < to && from < total ? owner(first, from) : first, next = from < to && from < total ? offset_at(lo + 1) : 0;
  for (int64_t i0 = from; i0 < to; i0 += 32 * kOnce) {
    int32_t position[kOnce], request[kOnce], entry[kOnce];
#pragma unroll
    for (int e = 0; e < kOnce; ++e) {
      const int64_t i = i0 + e * 32 + lane;
      position[e] = request[e] = entry[e] = -1;
      if (i < to && i < total) {
        if (i >= next) lo = owner(lo, i), next = offset_at(lo + 1);
        request[e]  = int32_t(lo);
        position[e] = __ldg(a.q.old_lengths + lo) + int32_t(i - offset_at(lo));
        const uint32_t column = a.q.block.of(uint32_t(position[e]));
        if (int64_t(column) < a.columns) entry[e] = __ldg(a.tables + lo * a.stride + column);
      }
    }
#pragma unroll
    for (int e = 0; e < kOnce; ++e) {
      const int64_t i = i0 + e * 32 + lane;
      if (i >= to) break;
      const uint32_t in_block = uint32_t(position[e]) - a.q.block.of(uint32_t(position[e])) * a.q.block.d;
      a.slots[i] = entry[e] >= 0 ? int64_t(entry[e]) * a.q.block.d + in_block : -1;
      if (a.positions) a.positions[i] = position[e];
      if (a.requests) a.requests[i] = request[e];
    }
  }
}

// Up to kFewRequests: each CTA adds up all of them, in shared memory, and puts a share of the tokens; the first one puts the offsets too.  What
// begins at 2^31 or later is behind every token that has a place.
constexpr int kFewRequests = 8192;
template <int EACH>  // neighbouring requests to a thread
__global__ void __launch_bounds__(kThreads) k_slots_of_few(const SlotArgs a, int64_t share)
{
  constexpr int kMine = EACH * kThreads;  // requests at most
  __shared__ uint32_t s_offset[kMine + 1];
  __shared__ Pair s_sum[kWarps];
  const int tid = threadIdx.x;
  const bool not_done = a.state && __ldg(a.state + 2) != 0;
  const int first     = tid * EACH;
  int64_t more[EACH], mine = 0;
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    more[e] = first + e < a.q.n && !not_done ? new_tokens(a, first + e) : 0;
    mine += more[e];
  }
  Pair all;
  int64_t upto = block_upto(Pair{mine, 0}, all, s_sum).a - mine;
  if (tid == 0) {
    s_offset[0] = 0;
    if (blockIdx.x == 0) a.offsets[0] = 0;
  }
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    upto += more[e];
    if (first + e < a.q.n && GTK_IN(first + e + 1, kMine + 1, 404)) {
      s_offset[first + e + 1] = uint32_t(min(upto, int64_t(1) << 31));
      if (blockIdx.x == 0) a.offsets[first + e + 1] = upto;
    }
  }
  __syncthreads();
  const int64_t begin = blockIdx.x * share;
  put_slots(a, begin, min(a.capacity, begin + share), 0, a.q.n, all.a, [&](int64_t r) { return int64_t(s_offset[r]); });
}

// Many requests: offsets first, then the tokens.
__global__ void __launch_bounds__(kThreads) k_slot_offsets(const SlotArgs a)
{
  __shared__ Pair s_sum[kWarps];
  constexpr int kEach = 8;
  const int tid  = threadIdx.x;
  const bool not_done = a.state && __ldg(a.state + 2) != 0;
  int64_t before = 0;
  if (tid == 0) a.offsets[0] = 0;
  for (int64_t tile = 0; tile < a.q.n; tile += kThreads * kEach) {
    const int64_t first = tile + tid * kEach;
    int64_t more[kEach], mine = 0;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      more[e] = first + e < a.q.n && !not_done ? new_tokens(a, first + e) : 0;
      mine += more[e];
    }
    Pair all;
    int64_t upto = before + block_upto(Pair{mine, 0}, all, s_sum).a - mine;
#pragma unroll
    for (int e = 0; e < kEach; ++e)
      if (first + e < a.q.n) a.offsets[first + e + 1] = upto += more[e];
    before += all.a;
  }
}
__global__ void __launch_bounds__(kThreads) k_slots_of_many(const SlotArgs a, int64_t share)
{
  __shared__ int64_t s_offset[kFewRequests / 2 + 1];
  gtk::await_kernel();
  const int64_t begin = blockIdx.x * share, end = min(a.capacity, begin + share), total = __ldcg(a.offsets + a.q.n);
  auto owner = [&](int64_t i) {
    int64_t lo = 0, hi = a.q.n;
    while (hi - lo > 1) {
      const int64_t mid = (lo + hi) / 2;
      if (__ldcg(a.offsets + mid) <= i) lo = mid;
      else hi = mid;
    }
    return lo;
  };
  // the requests of these tokens, in shared memory where they are few enough
  const int64_t first = begin < total ? owner(begin) : 0, last = begin < total ? owner(min(end, total) - 1) : 0;
  if (last - first + 1 <= kFewRequests / 2) {
    for (int64_t r = first + threadIdx.x; r <= last + 1; r += kThreads) s_offset[r - first] = __ldcg(a.offsets + r);
    __syncthreads();
    put_slots(a, begin, end, first, last + 1, total, [&](int64_t r) { return s_offset[r - first]; });
  } else {
    put_slots(a, begin, end, first, last + 1, total, [&](int64_t r) { return __ldcg(a.offsets + r); });
  }
}

// Requests of a CTA that is the only one, at most, and of one of several, at least.  Alone and with others, us (512 and 513 requests, in a graph): in
// a decoding step 9.3 and 10.5; half of them replaced by others of up to 8192 tokens 17.5 and 10.5.  The rule knows of requests and not of
// their blocks, whose number is in device memory: 512 new ones of 131072 tokens each in blocks of 16, four million blocks, take one CTA 1630,
// 513 take all CTAs 123.
constexpr int64_t kAlone = 512, kShare = 32;
constexpr int64_t kMost = (int64_t(1) << 31) - 1;

gtk::Refusal refuse_step(const void* before, const void* after, int64_t n, int block, const void* tables, int64_t columns, int64_t stride)
{
  if (n < 0 || n > kMost) return "n_requests must be 0 .. 2^31 - 1";
  if (block <= 0 || block > (1 << 20)) return "block_tokens must be 1 .. 2^20";
  if (columns <= 0 || columns > kMost) return "columns must be 1 .. 2^31 - 1";
  if (stride < columns) return "table_stride must be >= columns";
  if (n > 0 && (!before || !after || !tables)) return "null device pointer";
  if (!gtk::aligned_to(before, 4) || !gtk::aligned_to(after, 4) || !gtk::aligned_to(tables, 4))
    return "a device pointer is not aligned to its elements";
  return nullptr;
}

}  // namespace

extern "C" GTK_API int gtk_block_tables(gtk_tokenizer* h, const int32_t* d_old_lengths, const int32_t* d_new_lengths, int64_t n_requests,
                                        int block_tokens, int32_t* d_tables, int64_t columns, int64_t table_stride, int32_t* d_queue,
                                        int64_t queue_capacity, const int64_t* d_state, int64_t* d_state_out)
{
  auto check = [&]() -> gtk::Refusal {
    if (const gtk::Refusal why = refuse_step(d_old_lengths, d_new_lengths, n_requests, block_tokens, d_tables, columns, table_stride)) return why;
    if (queue_capacity <= 0 || queue_capacity > kMost) return "queue_capacity must be 1 .. 2^31 - 1";
    if (!d_queue || !d_state || !d_state_out) return "null device pointer";
    if (!gtk::aligned_to(d_queue, 4) || !gtk::aligned_to(d_state, 8) || !gtk::aligned_to(d_state_out, 8))
      return "a device pointer is not aligned to its elements";
    return nullptr;
  };
  return gtk::run_operator(h, check, [&](const gtk::HandleView& v) -> cudaError_t {
    const StepArgs a{{d_old_lengths, d_new_lengths, n_requests, Divisor(block_tokens)},
                     d_tables, columns, table_stride, d_queue, queue_capacity, d_state, d_state_out};
    const int64_t ctas = n_requests > kAlone ? std::min<int64_t>((n_requests + kShare - 1) / kShare, v.sm_count) : 1;
    if (ctas == 1) return gtk::launch(k_block_tables<true>, dim3(1), dim3(kThreads), 0, v.stream, a, n_requests);
    const int64_t share = (n_requests + ctas - 1) / ctas;
    const cudaError_t e = gtk::launch(k_block_tables<false>, dim3(unsigned(ctas)), dim3(kThreads), 0, v.stream, a, share);
    return e != cudaSuccess ? e : gtk::launch_behind(k_block_state, dim3(1), dim3(kThreads), 0, v.stream, a);
  });
}

extern "C" GTK_API int gtk_slot_map(gtk_tokenizer* h, const int32_t* d_old_lengths, const int32_t* d_new_lengths, int64_t n_requests,
                                    int block_tokens, const int32_t* d_tables, int64_t columns, int64_t table_stride, const int64_t* d_state,
                                    int64_t capacity, int64_t* d_slots, int32_t* d_positions, int32_t* d_requests, int64_t* d_offsets)
{
  auto check = [&]() -> gtk::Refusal {
    if (const gtk::Refusal why = refuse_step(d_old_lengths, d_new_lengths, n_requests, block_tokens, d_tables, columns, table_stride)) return why;
    if (capacity < 0 || capacity > kMost) return "capacity must be 0 .. 2^31 - 1";
    if (!d_offsets || (capacity > 0 && !d_slots)) return "null device pointer";
    if (!gtk::aligned_to(d_state, 8) || !gtk::aligned_to(d_slots, 8) || !gtk::aligned_to(d_offsets, 8) || !gtk::aligned_to(d_positions, 4) ||
        !gtk::aligned_to(d_requests, 4))
      return "a device pointer is not aligned to its elements";
    return nullptr;
  };
  return gtk::run_operator(h, check, [&](const gtk::HandleView& v) -> cudaError_t {
    const SlotArgs a{{d_old_lengths, d_new_lengths, n_requests, Divisor(block_tokens)}, d_tables, columns, table_stride, d_state, capacity,
                     d_slots, d_positions, d_requests, d_offsets};
    const bool few = n_requests <= kFewRequests;
    if (!few)
      if (const cudaError_t e = gtk::launch(k_slot_offsets, dim3(1), dim3(kThreads), 0, v.stream, a); e != cudaSuccess) return e;
    const int64_t ctas  = std::max<int64_t>(1, std::min<int64_t>((capacity + kThreads - 1) / kThreads, int64_t(v.sm_count)));
    const int64_t share = (capacity + ctas - 1) / ctas;
    const auto of_few = n_requests <= kThreads       ? k_slots_of_few<1>
                        : n_requests <= 4 * kThreads ? k_slots_of_few<4>
                                                     : k_slots_of_few<kFewRequests / kThreads>;
    return few ? gtk::launch(of_few, dim3(unsigned(ctas)), dim3(kThreads), 0, v.stream, a, share)
               : gtk::launch_behind(k_slots_of_many, dim3(unsigned(ctas)), dim3(kThreads), 0, v.stream, a, share);
  });
}

#ifdef GTK_CHECKED
cudaError_t gtk::paged_check_words(int sum[4], bool reset) { return add_check_words(sum, reset); }
cudaError_t gtk::paged_check_selftest() { return check_selftest(499); }
#endif
