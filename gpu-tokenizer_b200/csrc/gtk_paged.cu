// gtk_paged.cu -- the bookkeeping of a cache in blocks: which blocks requests hold, and where their new tokens go.
//
// With B tokens per block, a request of L tokens holds ceil(L / B) blocks, and its token j lies in slot
// table[j / B] * B + j % B.  Blocks that nobody holds wait in a ring: taken at its head, given back at its tail.
#include <climits>

#include "gtk_checked.cuh"
#include "gtk_rows.cuh"

namespace {

constexpr int kThreads = 1024, kWarps = kThreads / 32;

struct StepArgs {
  const int32_t *old_lengths, *new_lengths;
  int64_t n;
  int block;
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
  __device__ Blocks(const StepArgs& a, int64_t r)
  {
    if (r >= a.n) return;
    const int32_t before = __ldg(a.old_lengths + r), after = __ldg(a.new_lengths + r);
    if (before < 0 || after < 0) return;
    have = (uint32_t(before) + uint32_t(a.block) - 1u) / uint32_t(a.block);
    need = (uint32_t(after) + uint32_t(a.block) - 1u) / uint32_t(a.block);
  }
  __device__ uint32_t taken() const { return need > have ? need - have : 0u; }
  __device__ uint32_t given() const { return have > need ? have - need : 0u; }
};

__device__ __forceinline__ int64_t warp_sum(int64_t x)
{
#pragma unroll
  for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xFFFFFFFFu, x, d);
  return x;
}

__global__ void __launch_bounds__(kThreads) k_block_tables(const StepArgs a)
{
  __shared__ int64_t s_taken[kWarps], s_given[kWarps];
  __shared__ uint32_t s_have[kThreads], s_need[kThreads];
  __shared__ int64_t s_from[kThreads];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t head = a.state[0], tail = a.state[1];
  int64_t taken = 0, given = 0;
  bool beyond   = false;
  for (int64_t r = tid; r < a.n; r += kThreads) {
    const Blocks b(a, r);
    taken += b.taken(), given += b.given();
    beyond |= int64_t(max(b.have, b.need)) > a.columns;
  }
  taken = warp_sum(taken), given = warp_sum(given);
  if (lane == 0) s_taken[warp] = taken, s_given[warp] = given;
  beyond = __syncthreads_or(beyond);
  taken  = warp_sum(s_taken[lane]);
  given  = warp_sum(s_given[lane]);
  __syncthreads();
  const int64_t waiting = tail - head;
  int64_t status        = 0;
  if (beyond) status = -1;
  else if (head < 0 || waiting < 0 || waiting + given > a.capacity) status = -2;
  else if (taken > waiting) status = taken - waiting;
  if (tid == 0) {
    a.state_out[0] = status ? head : head + taken;
    a.state_out[1] = status ? tail : tail + given;
    a.state_out[2] = status;
  }
  if (status) return;
  int64_t took = 0, gave = 0;  // by the requests in front of the tile
  for (int64_t first = 0; first < a.n; first += kThreads) {
    const Blocks b(a, first + tid);
    int64_t t = b.taken(), g = b.given();
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int64_t tl = __shfl_up_sync(0xFFFFFFFFu, t, d), gl = __shfl_up_sync(0xFFFFFFFFu, g, d);
      if (lane >= d) t += tl, g += gl;
    }
    if (lane == 31) s_taken[warp] = t, s_given[warp] = g;
    s_have[tid] = b.have, s_need[tid] = b.need;
    __syncthreads();
    const int64_t taken_before = warp_sum(lane < warp ? s_taken[lane] : 0), given_before = warp_sum(lane < warp ? s_given[lane] : 0);
    s_from[tid] = b.need > b.have ? head + took + taken_before + t - b.taken() : tail + gave + given_before + g - b.given();
    took += warp_sum(s_taken[lane]), gave += warp_sum(s_given[lane]);
    __syncthreads();
    const int rows = int(min(int64_t(kThreads), a.n - first));
    for (int r = warp; r < rows; r += kWarps) {
      const uint32_t have = s_have[r], need = s_need[r];
      const int64_t at = s_from[r];
      int32_t* row     = a.tables + (first + r) * a.stride;
      for (uint32_t i = have + lane; i < need; i += 32) row[i] = a.queue[(at + (i - have)) % a.capacity];
      for (uint32_t i = need + lane; i < have; i += 32) a.queue[(at + (i - need)) % a.capacity] = row[i];
    }
    __syncthreads();
  }
}

struct SlotArgs {
  const int32_t *old_lengths, *new_lengths;
  int64_t n;
  int block;
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
  if (r >= a.n) return 0;
  const int32_t before = __ldg(a.old_lengths + r), after = __ldg(a.new_lengths + r);
  return before >= 0 && after > before ? int64_t(after) - before : 0;
}

__global__ void __launch_bounds__(kThreads) k_slot_offsets(const SlotArgs a)
{
  __shared__ int64_t s_sum[kWarps];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const bool done = a.state && a.state[2] != 0;
  int64_t before  = 0;
  if (tid == 0) a.offsets[0] = 0;
  for (int64_t first = 0; first < a.n; first += kThreads) {
    int64_t t = done ? 0 : new_tokens(a, first + tid);
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int64_t l = __shfl_up_sync(0xFFFFFFFFu, t, d);
      if (lane >= d) t += l;
    }
    if (lane == 31) s_sum[warp] = t;
    __syncthreads();
    const int64_t front = warp_sum(lane < warp ? s_sum[lane] : 0);
    if (first + tid < a.n) a.offsets[first + tid + 1] = before + front + t;
    before += warp_sum(s_sum[lane]);
    __syncthreads();
  }
}

__global__ void __launch_bounds__(256) k_slots(const SlotArgs a)
{
  for (int64_t i = blockIdx.x * int64_t(blockDim.x) + threadIdx.x; i < a.capacity; i += int64_t(gridDim.x) * blockDim.x) {
    int64_t slot = -1;
    int32_t position = -1, request = -1;
    if (i < a.offsets[a.n]) {
      int64_t lo = 0, hi = a.n;  // offsets[lo] <= i < offsets[hi]
      while (hi - lo > 1) {
        const int64_t mid = (lo + hi) / 2;
        if (a.offsets[mid] <= i) lo = mid;
        else hi = mid;
      }
      request  = int32_t(lo);
      position = __ldg(a.old_lengths + lo) + int32_t(i - a.offsets[lo]);
      const int column = position / a.block;
      const int32_t b  = column < a.columns ? a.tables[lo * a.stride + column] : -1;
      if (b >= 0) slot = int64_t(b) * a.block + position % a.block;
    }
    a.slots[i] = slot;
    if (a.positions) a.positions[i] = position;
    if (a.requests) a.requests[i] = request;
  }
}

constexpr int64_t kMost = (int64_t(1) << 31) - 1;

gtk::Refusal refuse_step(const void* before, const void* after, int64_t n, int block, const void* tables, int64_t columns, int64_t stride)
{
  if (n < 0 || n > kMost) return "n_requests must be 0 .. 2^31 - 1";
  if (block <= 0 || block > (1 << 20)) return "block_tokens must be 1 .. 2^20";
  if (columns <= 0 || columns > kMost) return "columns must be 1 .. 2^31 - 1";
  if (stride < columns) return "table_stride must be >= columns";
  if (n > 0 && (!before || !after || !tables)) return "null device pointer";
  if (!gtk::aligned_to(before, 4) || !gtk::aligned_to(after, 4) || !gtk::aligned_to(tables, 4)) return "a device pointer is not aligned to its elements";
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
    const StepArgs a{d_old_lengths, d_new_lengths, n_requests, block_tokens, d_tables, columns, table_stride, d_queue, queue_capacity, d_state, d_state_out};
    return gtk::launch(k_block_tables, dim3(1), dim3(kThreads), 0, v.stream, a);
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
    const SlotArgs a{d_old_lengths, d_new_lengths, n_requests, block_tokens, d_tables, columns, table_stride, d_state, capacity,
                     d_slots, d_positions, d_requests, d_offsets};
    cudaError_t e = gtk::launch(k_slot_offsets, dim3(1), dim3(kThreads), 0, v.stream, a);
    if (e != cudaSuccess || capacity == 0) return e;
    return gtk::launch(k_slots, dim3(unsigned(std::min<int64_t>((capacity + 255) / 256, int64_t(v.sm_count) * 8))), dim3(256), 0, v.stream, a);
  });
}

#ifdef GTK_CHECKED
cudaError_t gtk::paged_check_words(int sum[4], bool reset) { return add_check_words(sum, reset); }
cudaError_t gtk::paged_check_selftest() { return check_selftest(499); }
#endif
