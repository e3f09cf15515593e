// gtk_embed.cu -- embedding lookup with scaling, and its gradient by sorted tokens.
#include <algorithm>
#include <cmath>

#include "gtk_rows.cuh"

namespace {

using gtk::Pack;
using gtk::Two;

// ------------------------------------------------------------------------------------------------ lookup
// out[i] = scale * table[ids[i]].  A block's threads are split into row groups of 1 << group_log2; a group copies a row
// in packs of V elements, four loads in flight per thread.
constexpr int kEmbedThreads = 256;

template <class T, class O, int V>
__global__ void __launch_bounds__(kEmbedThreads)
k_embed(const int32_t* __restrict__ ids, int64_t n, const T* __restrict__ table, int vocab, int dim, int64_t table_stride,
        float scale, O* __restrict__ out, int64_t out_stride, int group_log2)
{
  const int group = 1 << group_log2, lane = threadIdx.x & (group - 1);
  const int64_t i = int64_t(blockIdx.x) * (kEmbedThreads >> group_log2) + (threadIdx.x >> group_log2);
  if (i >= n) return;
  const int id = __ldg(ids + i);
  O* to        = out + i * out_stride;
  if (uint32_t(id) >= uint32_t(vocab)) {
    const O fill = gtk::from_float<O>(id < 0 ? 0.f : __int_as_float(0x7FC00000));
    for (int c = lane; c < dim; c += group) to[c] = fill;
    return;
  }
  const T* from   = table + int64_t(id) * table_stride;
  const int packs = dim / V;
  for (int u0 = lane; u0 < packs; u0 += 4 * group) {
    Pack<T, V> x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (u0 + k * group < packs) x[k] = gtk::load_pack<T, V>(from + int64_t(u0 + k * group) * V);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (u0 + k * group < packs) {
        Pack<O, V> y;
#pragma unroll
        for (int j = 0; j < V; ++j) y.e[j] = gtk::from_float<O>(gtk::to_float(x[k].e[j]) * scale);
        gtk::store_pack<O, V>(to + int64_t(u0 + k * group) * V, y);
      }
  }
  for (int c = packs * V + lane; c < dim; c += group) to[c] = gtk::from_float<O>(gtk::to_float(from[c]) * scale);
}

template <class T, class O, int V>
cudaError_t launch_embed(const gtk::HandleView& v, const int32_t* ids, int64_t n, const void* table, int64_t vocab, int64_t dim,
                         int64_t table_stride, float scale, void* out, int64_t out_stride)
{
  const int64_t packs = std::max<int64_t>(1, dim / V);
  int group_log2 = 5;  // a warp per row, more for rows of more than four packs a lane
  while (group_log2 < 8 && (int64_t(4) << group_log2) < packs) ++group_log2;
  const int64_t rows = kEmbedThreads >> group_log2;
  return gtk::launch(k_embed<T, O, V>, dim3(unsigned((n + rows - 1) / rows)), dim3(kEmbedThreads), 0, v.stream, ids, n,
                     static_cast<const T*>(table), int(vocab), int(dim), table_stride, scale, static_cast<O*>(out), out_stride,
                     group_log2);
}

// ------------------------------------------------------------------------------------------------ gradient
// grad_table[v] = scale * sum of grad_out[i] over the i with ids[i] == v, in three launches:
//   k_embed_grad_sort   groups the tokens by id, which brings the rows of a sum next to each other in order of i, and
//                       writes the rows that no id points to
//   k_embed_grad_sums   the grouped tokens in blocks of equal length, a row group of threads per block; a sum is kept in
//                       registers.  One that lies in a block or reaches over one boundary is its first block's alone; a
//                       longer one is cut at the boundaries and its parts go to the workspace
//   k_embed_grad_join   adds the parts of the long ones from left to right
// Every sum is thus formed in an order that the ids alone decide.
constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32;
constexpr int kOwnersLog2 = 7, kOwners = 1 << kOwnersLog2;  // CTAs of k_embed_grad_sort
constexpr int kMaxDigitBits = 9;                            // a thread per bin at most
constexpr int64_t kMaxDim = int64_t(1) << 20;

struct GradPlan {
  int passes, digit_bits;
  int block_log2;   // tokens per block of k_embed_grad_sums
  int64_t blocks;
  int64_t pitch;    // 32-bit floats between rows of the parts
  size_t at_tokens[2], at_header, at_parts, bytes;
};

int bits_of(int64_t x)
{
  int b = 0;
  while (x >> b) ++b;
  return b;
}

constexpr size_t kSharedMost = 96 << 10;  // of a CTA
constexpr int kMinBlockLog2 = 3, kMaxBlockLog2 = 10;

GradPlan grad_plan(int64_t n, int64_t vocab, int64_t dim)
{
  GradPlan p{};
  const int bits = std::max(1, bits_of((vocab - 1) >> kOwnersLog2));
  p.passes       = (bits + kMaxDigitBits - 1) / kMaxDigitBits;
  p.digit_bits   = (bits + p.passes - 1) / p.passes;
  p.block_log2   = kMinBlockLog2;
  // blocks as long as still leaves about 1.5 M columns of them: a dozen row groups of 768 columns per SM
  while (p.block_log2 < kMaxBlockLog2 && (n >> (p.block_log2 + 1)) * dim >= int64_t(3) << 19) ++p.block_log2;
  p.blocks    = (n + (int64_t(1) << p.block_log2) - 1) >> p.block_log2;
  p.pitch     = (dim + 7) / 8 * 8;
  size_t at   = 0;
  auto room   = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) & ~size_t(255);
    return here;
  };
  p.at_tokens[0] = room(size_t(n) * sizeof(uint2));
  p.at_tokens[1] = room(size_t(n) * sizeof(uint2));
  p.at_header    = room(size_t(p.blocks + 2) * 4);
  p.at_parts     = room(size_t(p.blocks) * 2 * size_t(p.pitch) * 4);
  p.bytes        = at;
  return p;
}

// Written by k_embed_grad_sort and read by what follows.
struct GradHeader {
  uint32_t tokens;      // that take part
  uint32_t long_sums;   // sums that k_embed_grad_sums has cut
  uint32_t block[1];    // .. and the blocks in which they begin
};

struct SortArgs {
  const int32_t* ids;
  int64_t n;
  uint32_t vocab;
  int passes, digit_bits;
  uint2 *tokens0, *tokens1;  // {id, place}: the grouped tokens end up in tokens0 after an even number of passes
  GradHeader* header;
};

struct SortShared {
  uint32_t at[kSortWarps][1 << kMaxDigitBits];
  uint32_t warp_sum[kSortWarps];
  uint32_t lower[kSortWarps], mine[kSortWarps];
};

// The sum over the warps in front and over all of them, of a number that each warp has put into v.
__device__ __forceinline__ void over_warps(const uint32_t* v, int warp, uint32_t& front, uint32_t& all)
{
  front = all = 0;
#pragma unroll
  for (int w = 0; w < kSortWarps; ++w) {
    const uint32_t x = v[w];
    front += w < warp ? x : 0u;
    all += x;
  }
}

// One digit of a stable sort of the CTA's own `count` tokens.  Each warp takes a stretch of them, counts its digits, and
// moves its tokens to the places that digits in front and stretches in front leave it.
__device__ void sort_digit(const uint2* from, uint2* to, uint32_t count, int shift, int digit_bits, SortShared& S)
{
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int bins         = 1 << digit_bits;
  const uint32_t stretch = (count + kSortThreads - 1) / kSortThreads * 32;
  const int warps        = int((count + stretch - 1) / stretch);  // that have any
  const uint32_t first   = warp * stretch, last = min(count, first + stretch);
  const uint32_t lower   = (1u << lane) - 1u;
  if (warp < warps) {
    for (int b = lane; b < bins; b += 32) S.at[warp][b] = 0;
    __syncwarp();
#pragma unroll 4
    for (uint32_t i = first + lane; i < last; i += 32) atomicAdd(&S.at[warp][(from[i].x >> shift) & (bins - 1)], 1u);
  }
  __syncthreads();
  uint32_t sum = 0;
  if (tid < bins) {
#pragma unroll 4
    for (int w = 0; w < warps; ++w) {
      const uint32_t c = S.at[w][tid];
      S.at[w][tid]     = sum;
      sum += c;
    }
  }
  uint32_t upto = sum;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const uint32_t o = __shfl_up_sync(0xFFFFFFFFu, upto, d);
    if (lane >= d) upto += o;
  }
  if (lane == 31) S.warp_sum[warp] = upto;
  __syncthreads();
  if (tid < bins) {
    uint32_t front, all;
    over_warps(S.warp_sum, warp, front, all);
    front += upto - sum;
#pragma unroll 4
    for (int w = 0; w < warps; ++w) S.at[w][tid] += front;
  }
  __syncthreads();
  if (warp < warps) {
#pragma unroll 2
    for (uint32_t i0 = first; i0 < last; i0 += 32) {
      const bool here      = i0 + lane < last;
      const uint2 x        = here ? from[i0 + lane] : make_uint2(0u, 0u);
      const uint32_t digit = here ? (x.x >> shift) & uint32_t(bins - 1) : 0xFFFFFFFFu;
      const uint32_t peers = __match_any_sync(0xFFFFFFFFu, digit);
      const uint32_t place = here ? S.at[warp][digit] + __popc(peers & lower) : 0u;
      __syncwarp();
      if (here && (peers >> lane) == 1u) S.at[warp][digit] = place + 1u;  // the last of the peers
      __syncwarp();
      if (here) to[place] = x;
    }
  }
  __syncthreads();
}

// CTA c owns the ids with id % kOwners == c: it looks at all ids, learns how many tokens lower owners have, which is where
// its own go, writes them there in order and sorts them.  Nothing is waited for between CTAs.  Returns its share.
__device__ void group_tokens(const SortArgs& a, SortShared& S, uint32_t& begin, uint32_t& count)
{
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t owner  = blockIdx.x;
  const int64_t stretch = (a.n + kSortThreads - 1) / kSortThreads * 32;
  const int64_t first   = min(a.n, warp * stretch), last = min(a.n, first + stretch);
  uint32_t lower = 0, mine = 0;
#pragma unroll 8
  for (int64_t i = first + lane; i < last; i += 32) {
    const uint32_t id = uint32_t(__ldg(a.ids + i)), of = id < a.vocab ? id & (kOwners - 1) : uint32_t(kOwners);
    lower += of < owner;
    mine += of == owner;
  }
  lower = __reduce_add_sync(0xFFFFFFFFu, lower);
  mine  = __reduce_add_sync(0xFFFFFFFFu, mine);
  if (lane == 0) S.lower[warp] = lower, S.mine[warp] = mine;
  __syncthreads();
  uint32_t at;
  over_warps(S.lower, warp, at, begin);
  over_warps(S.mine, warp, at, count);
  if (owner == kOwners - 1 && tid == 0) a.header->tokens = begin + count;
  if (mine) {
    uint2* to = a.tokens0 + begin + at;
    for (int64_t i0 = first; i0 < last; i0 += 8 * 32) {
      uint32_t id[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) id[k] = i0 + k * 32 + lane < last ? uint32_t(__ldg(a.ids + i0 + k * 32 + lane)) : 0xFFFFFFFFu;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const bool is_mine  = id[k] < a.vocab && (id[k] & (kOwners - 1)) == owner;
        const uint32_t mask = __ballot_sync(0xFFFFFFFFu, is_mine);
        if (!mask) continue;
        if (is_mine) to[__popc(mask & ((1u << lane) - 1u))] = make_uint2(id[k], uint32_t(i0 + k * 32 + lane));
        to += __popc(mask);
      }
    }
  }
  __syncthreads();
  if (count == 0) return;
  for (int pass = 0; pass < a.passes; ++pass)
    sort_digit((pass & 1 ? a.tokens1 : a.tokens0) + begin, (pass & 1 ? a.tokens0 : a.tokens1) + begin, count,
               kOwnersLog2 + pass * a.digit_bits, a.digit_bits, S);
}

// zeros over a row, however it lies
template <class T>
__device__ __forceinline__ void clear_row(T* row, int dim, int lane, int lanes)
{
  const int head = min(dim, int((16u - (uint32_t(reinterpret_cast<uintptr_t>(row)) & 15u)) % 16u / sizeof(T)));
  constexpr int E = 16 / int(sizeof(T));
  const int packs = (dim - head) / E;
  uint4* body     = reinterpret_cast<uint4*>(row + head);
  for (int p = lane; p < packs; p += lanes) body[p] = make_uint4(0u, 0u, 0u, 0u);
  const T zero = gtk::from_float<T>(0.f);
  for (int c = lane; c < dim - packs * E; c += lanes) row[c < head ? c : c + packs * E] = zero;
}

template <class T>
__global__ void __launch_bounds__(kSortThreads, 1)
k_embed_grad_sort(const SortArgs a, T* __restrict__ grad_table, int dim, int64_t table_stride, bool clear)
{
  extern __shared__ uint4 s_raw[];
  SortShared& S = *reinterpret_cast<SortShared*>(s_raw);
  uint32_t begin = 0, count = 0;
  if (a.n > 0) {
    if (blockIdx.x == 0 && threadIdx.x == 0) a.header->long_sums = 0;
    group_tokens(a, S, begin, count);
  }
  if (!clear) return;
  // the rows of this owner that have no token, as many at once as the shared memory has bits
  uint32_t* used         = &S.at[0][0];
  constexpr int kAtOnce  = sizeof(S.at) * 8;
  const uint2* tokens    = (a.passes & 1 ? a.tokens1 : a.tokens0) + begin;
  const int64_t rows     = (int64_t(a.vocab) - int64_t(blockIdx.x) + kOwners - 1) >> kOwnersLog2;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int64_t r0 = 0; r0 < rows; r0 += kAtOnce) {
    const int here = int(min(int64_t(kAtOnce), rows - r0));
    for (int w = threadIdx.x; w < (here + 31) / 32; w += kSortThreads) used[w] = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < count; i += kSortThreads) {
      const int64_t r = int64_t(tokens[i].x >> kOwnersLog2) - r0;
      if (r >= 0 && r < here && (i == 0 || tokens[i - 1].x != tokens[i].x)) atomicOr(used + (r >> 5), 1u << (r & 31));
    }
    __syncthreads();
    for (int r = warp; r < here; r += kSortWarps)
      if (!(used[r >> 5] >> (r & 31) & 1u)) clear_row(grad_table + (((r0 + r) << kOwnersLog2) + blockIdx.x) * table_stride, dim, lane, 32);
    __syncthreads();
  }
}

constexpr int kGradThreads = 256;

// V neighbouring columns of a finished sum to their row; packs: they may be stored in one piece
template <class T, int V>
__device__ __forceinline__ void store_sum(T* row, int valid, bool packs, float scale, bool accumulate, const float* sum)
{
  if (packs && valid >= V) {
    Pack<T, V> v;
    if (accumulate) v = gtk::load_pack<T, V>(row);
#pragma unroll
    for (int j = 0; j < V; ++j) v.e[j] = gtk::from_float<T>(accumulate ? fmaf(sum[j], scale, gtk::to_float(v.e[j])) : sum[j] * scale);
    gtk::store_pack<T, V>(row, v);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j < valid) row[j] = gtk::from_float<T>(accumulate ? fmaf(sum[j], scale, gtk::to_float(row[j])) : sum[j] * scale);
  }
}

struct GradArgs {
  const uint2* tokens;  // grouped {id, place}
  GradHeader* header;
  int dim;
  int block_log2;
  int64_t out_stride, table_stride, pitch;
  float scale;
  bool accumulate;
  float* parts;  // [blocks][2][pitch]: of the long sum that begins further left, of the one that begins in the block
};

constexpr uint32_t kNoId = 0xFFFFFFFFu;
constexpr int kChunk = 4, kChunks = 4;  // rows that are waited for together, and such chunks in flight

__device__ __forceinline__ void copy16(uint32_t shared_at, const void* from)
{
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(shared_at), "l"(from) : "memory");
}
__device__ __forceinline__ void end_chunk() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING>
__device__ __forceinline__ void await_chunks() { asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory"); }

// first place in [from, to) whose id is not `id` (where one id follows another it does not come back)
__device__ __forceinline__ int end_of_id(const uint2* tokens, int from, int to, uint32_t id)
{
  while (from < to) {
    const int mid = (from + to) >> 1;
    if (tokens[mid].x == id) from = mid + 1;
    else to = mid;
  }
  return from;
}

// 16 bytes of a row, added to its columns' sums
__device__ __forceinline__ void add_pack(const uint4& r, const float*, Two (&sum)[2])
{
  sum[0] = sum[0] + Two(__uint_as_float(r.x), __uint_as_float(r.y));
  sum[1] = sum[1] + Two(__uint_as_float(r.z), __uint_as_float(r.w));
}
template <class O>
__device__ __forceinline__ void add_pack(const uint4& r, const O*, Two (&sum)[4])
{
  const O* e = reinterpret_cast<const O*>(&r);
#pragma unroll
  for (int j = 0; j < 4; ++j) sum[j] = sum[j] + Two(gtk::to_float(e[2 * j]), gtk::to_float(e[2 * j + 1]));
}

// the 16 bytes that begin `bytes` (a multiple of 2, below 16) behind the first of two packs
__device__ __forceinline__ uint4 shifted(const uint4& a, const uint4& b, uint32_t bytes)
{
  uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  if (bytes & 8)
#pragma unroll
    for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
  if (bytes & 4)
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
  const uint32_t half = (bytes & 2) * 8;
  return make_uint4(__funnelshift_r(w[0], w[1], half), __funnelshift_r(w[1], w[2], half), __funnelshift_r(w[2], w[3], half),
                    __funnelshift_r(w[3], w[4], half));
}

// A group of threads (part of a warp, or the whole CTA) takes a block of tokens.  Every thread has the columns of 16 bytes and
// copies its share of the rows to shared memory, up to kChunk * kChunks rows ahead.
// ALIGNED: rows of both arrays start where 16 bytes of grad_out's elements do.  Otherwise a row's 16-byte pieces are copied as they lie
// between 16-byte boundaries (the outer ones hold bytes of its neighbours, which nobody looks at) and a thread takes its
// columns from two of them; sums go through shared memory to be stored by neighbouring threads side by side.
template <class O, class T, bool ALIGNED>
__global__ void __launch_bounds__(kGradThreads) k_embed_grad_sums(const GradArgs a, const O* __restrict__ grad_out, T* __restrict__ grad_table)
{
  constexpr int E = 16 / int(sizeof(O));
  extern __shared__ uint4 s_raw[];
  const int group = blockDim.x, groups = blockDim.y, lane = threadIdx.x;
  const int length = 1 << a.block_log2, window = 3 * length + 2;
  // [groups][rows][group] pieces, [groups][group * E] sums unless ALIGNED, [groups][window] tokens
  uint4* ring = s_raw + threadIdx.y * (kChunk * kChunks) * group;
  float* sums = reinterpret_cast<float*>(s_raw + groups * (kChunk * kChunks) * group) + threadIdx.y * group * E;
  uint2* P    = reinterpret_cast<uint2*>(s_raw + groups * group * (kChunk * kChunks + (ALIGNED ? 0 : E / 4))) + threadIdx.y * window + length + 1;
  // the block's tokens, its neighbours' and one more at each end
  const int64_t n     = a.header->tokens;
  const int64_t block = int64_t(blockIdx.x) * groups + threadIdx.y;
  const int64_t begin = block << a.block_log2;
  for (int i = lane - length - 1; i <= 2 * length; i += group)
    P[i] = begin + i >= 0 && begin + i < n ? __ldg(a.tokens + begin + i) : make_uint2(kNoId, 0u);  // ids are below 2^31
  __syncthreads();
  // the columns: from `first` on, `own` of them this thread's; `pieces` 16-byte pieces of a row, counted from the one with `first`
  const int slab  = (ALIGNED ? group : group - 1) * E;
  const int first = blockIdx.y * slab, width = min(slab, a.dim - first);
  const int c     = first + lane * E, own = max(0, min(E, first + width - c));
  const uint32_t mask = group >= 32 ? 0xFFFFFFFFu : ((1u << group) - 1u) << (threadIdx.y * group & 31);
  auto meet = [&] {
    if (group > 32) __syncthreads();
    else __syncwarp(mask);
  };
  int at = 0, stop = 0;
  bool from_left = false, to_right = false;
  if (begin < n) {
    const int end      = int(min(int64_t(length), n - begin));
    const uint32_t id0 = P[0].x, id1 = P[end - 1].x;
    stop = end;
    // the sum that begins further left: skipped, or this block's part of a long one
    from_left = P[-1].x == id0;
    if (from_left && P[end].x != id0 && P[-length - 1].x != id0) {
      at        = end_of_id(P, 0, end, id0);
      from_left = false;
    }
    // the sum that reaches over the end: to its end, or up to the boundary when it is a long one
    if (at < end && P[end].x == id1 && !(from_left && id1 == id0)) {
      to_right = P[2 * length].x == id1;
      if (!to_right) stop = end_of_id(P, end, 2 * length, id1);
      else if (c == 0) a.header->block[atomicAdd(&a.header->long_sums, 1u)] = uint32_t(block);
    }
  }
  if (at >= stop) return;  // the whole group
  const uint32_t ring_at = uint32_t(__cvta_generic_to_shared(ring)) + lane * 16;
  const char* column     = reinterpret_cast<const char*>(grad_out + first);
  const int64_t row_bytes = a.out_stride * int64_t(sizeof(O));
  const uint32_t width_bytes = uint32_t(width) * uint32_t(sizeof(O));
  auto request = [&](int chunk) {
#pragma unroll
    for (int k = 0; k < kChunk; ++k) {
      const int i = at + chunk * kChunk + k;
      if (i < stop) {
        const char* row      = column + int64_t(P[i].y) * row_bytes;
        const uint32_t shift = ALIGNED ? 0u : uint32_t(reinterpret_cast<uintptr_t>(row)) & 15u;
        if (uint32_t(lane) * 16u < shift + width_bytes) copy16(ring_at + ((chunk % kChunks) * kChunk + k) * group * 16, row - shift + lane * 16);
      }
    }
    end_chunk();
  };
  Two sum[E / 2];
#pragma unroll
  for (int j = 0; j < E / 2; ++j) sum[j] = Two(0.f, 0.f);
  auto store_part = [&](int which) {
    if (!own) return;
    float* to = a.parts + (block * 2 + which) * a.pitch + c;  // the pitch is a multiple of E
#pragma unroll
    for (int j = 0; j < E / 2; j += 2) {
      float4 v;
      sum[j].get(v.x, v.y);
      sum[j + 1].get(v.z, v.w);
      *reinterpret_cast<float4*>(to + 2 * j) = v;
    }
  };
  auto finish = [&](uint32_t id) {
    if (from_left) {
      store_part(0);
      from_left = false;
      return;
    }
    T* row = grad_table + int64_t(id) * a.table_stride;
    float x[E];
#pragma unroll
    for (int j = 0; j < E / 2; ++j) sum[j].get(x[2 * j], x[2 * j + 1]);
    if constexpr (ALIGNED) {
      store_sum<T, E>(row + c, own, true, a.scale, a.accumulate, x);
    } else {
#pragma unroll
      for (int j = 0; j < E; j += 4) *reinterpret_cast<float4*>(sums + lane * E + j) = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
      meet();
      for (int i = lane; i < width; i += group) store_sum<T, 1>(row + first + i, 1, true, a.scale, a.accumulate, sums + i);
      meet();
    }
  };
#pragma unroll
  for (int q = 0; q < kChunks - 1; ++q) request(q);
  uint32_t id = P[at].x;
  for (int chunk = 0; at + chunk * kChunk < stop; ++chunk) {
    await_chunks<kChunks - 2>();
    if constexpr (!ALIGNED) meet();
    request(chunk + kChunks - 1);  // over the chunk in front, which everybody has added
    const uint4* rows = ring + (chunk % kChunks) * kChunk * group + lane;
#pragma unroll
    for (int k = 0; k < kChunk; ++k) {
      const int i = at + chunk * kChunk + k;
      if (i >= stop) break;
      const uint2 token = P[i];
      if (token.x != id) {
        finish(id);
        id = token.x;
#pragma unroll
        for (int j = 0; j < E / 2; ++j) sum[j] = Two(0.f, 0.f);
      }
      if constexpr (ALIGNED) {
        add_pack(rows[k * group], static_cast<const O*>(nullptr), sum);
      } else if (own) {
        const uint32_t shift = (uint32_t(reinterpret_cast<uintptr_t>(column)) + token.y * uint32_t(row_bytes)) & 15u;
        add_pack(shifted(rows[k * group], rows[k * group + 1], shift), static_cast<const O*>(nullptr), sum);
      }
    }
  }
  if (to_right) store_part(1);
  else finish(id);
}

// The parts of a long sum, 128 columns at a time: each warp adds a run of parts, then the warps' sums are added in order.
template <class T>
__global__ void __launch_bounds__(kGradThreads) k_embed_grad_join(const GradArgs a, T* __restrict__ grad_table, bool packs)
{
  constexpr int kWarps = kGradThreads / 32;
  __shared__ float4 s_sum[kWarps][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t n     = a.header->tokens;
  const int slabs     = (a.dim + 127) / 128;
  const int64_t items = int64_t(a.header->long_sums) * slabs;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t block = a.header->block[item / slabs];
    const int c         = int(item % slabs) * 128 + lane * 4;
    const uint32_t id   = a.tokens[((block + 1) << a.block_log2) - 1].x;
    int64_t more = 0;  // blocks behind this one that begin with the same id
    for (int found = kGradThreads; found == kGradThreads; more += found) {
      const int64_t i = (block + 1 + more + threadIdx.x) << a.block_log2;
      found           = __syncthreads_count(i < n && a.tokens[i].x == id);
    }
    const int64_t each = (more + 1 + kWarps - 1) / kWarps;
    const int64_t from = warp * each, to = min(more + 1, from + each);
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    if (c < a.dim) {
#pragma unroll 8
      for (int64_t i = from; i < to; ++i) {  // part 0 is the one that begins in the block
        const float4 x = *reinterpret_cast<const float4*>(a.parts + ((block + i) * 2 + (i == 0 ? 1 : 0)) * a.pitch + c);
        sum.x += x.x, sum.y += x.y, sum.z += x.z, sum.w += x.w;
      }
    }
    s_sum[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && c < a.dim) {
#pragma unroll
      for (int w = 1; w < kWarps; ++w) {
        const float4 x = s_sum[w][lane];
        sum.x += x.x, sum.y += x.y, sum.z += x.z, sum.w += x.w;
      }
      const float y[4] = {sum.x, sum.y, sum.z, sum.w};
      store_sum<T, 4>(grad_table + int64_t(id) * a.table_stride + c, a.dim - c, packs, a.scale, a.accumulate, y);
    }
    __syncthreads();
  }
}

template <class O, class T, bool ALIGNED>
cudaError_t launch_embed_grad(const gtk::HandleView& v, const GradPlan& p, GradArgs a, const int32_t* ids, int64_t n, int64_t vocab,
                              const void* grad_out, void* grad_table, unsigned char* work)
{
  T* table = static_cast<T*>(grad_table);
  const SortArgs s{ids, n, uint32_t(vocab), p.passes, p.digit_bits, reinterpret_cast<uint2*>(work + p.at_tokens[0]),
                   reinterpret_cast<uint2*>(work + p.at_tokens[1]), a.header};
  cudaError_t e = gtk::launch(k_embed_grad_sort<T>, dim3(kOwners), dim3(kSortThreads), sizeof(SortShared), v.stream, s, table, a.dim,
                              a.table_stride, !a.accumulate);
  if (e != cudaSuccess || n == 0) return e;
  a.tokens = p.passes & 1 ? s.tokens1 : s.tokens0;
  // threads of a group: a power of two below a warp, several groups in a CTA; else whole warps, a CTA's at most
  constexpr int E      = 16 / int(sizeof(O));
  const int64_t wanted = (a.dim + E - 1) / E + (ALIGNED ? 0 : 1);
  unsigned group = 1;
  if (wanted > 32) group = unsigned(std::min<int64_t>(kGradThreads, (wanted + 31) / 32 * 32));
  else
    while (group < wanted) group *= 2;
  const unsigned columns = (ALIGNED ? group : group - 1) * E, slabs = unsigned((a.dim + columns - 1) / columns);
  const size_t bytes     = size_t(group) * 16 * (kChunk * kChunks + (ALIGNED ? 0 : E / 4)) + sizeof(uint2) * ((size_t(3) << a.block_log2) + 2);
  unsigned groups = group > 32 ? 1 : std::max(1u, 128 / group);
  while (groups > 1 && groups * bytes > kSharedMost) groups /= 2;
  e = gtk::launch(k_embed_grad_sums<O, T, ALIGNED>, dim3(unsigned((p.blocks + groups - 1) / groups), slabs), dim3(group, groups), groups * bytes,
                  v.stream, a, static_cast<const O*>(grad_out), table);
  // a sum is long when it holds a whole block and more on both sides
  if (e == cudaSuccess && p.blocks > 2)
    e = gtk::launch(k_embed_grad_join<T>, dim3(unsigned(std::min<int64_t>(p.blocks * ((a.dim + 127) / 128), int64_t(v.sm_count) * 8))),
                    dim3(kGradThreads), 0, v.stream, a, table, ALIGNED);
  return e;
}

constexpr int64_t kMaxCount = (int64_t(1) << 31) - 1;

gtk::Refusal refuse_sizes(int64_t n_ids, int64_t vocab, int64_t dim)
{
  if (n_ids < 0 || vocab <= 0 || dim <= 0) return "n_ids must be >= 0, vocab and dim > 0";
  if (n_ids > kMaxCount || vocab > kMaxCount || dim > kMaxDim) return "n_ids or vocab of 2^31 and more, or dim beyond 2^20";
  return nullptr;
}

}  // namespace

extern "C" GTK_API int gtk_embed(gtk_tokenizer* h, const int32_t* d_ids, int64_t n_ids, const void* d_table, int table_type,
                                 int64_t vocab, int64_t dim, int64_t table_stride, float scale, void* d_out, int out_type,
                                 int64_t out_stride)
{
  auto check = [&]() -> gtk::Refusal {
    if (const gtk::Refusal why = refuse_sizes(n_ids, vocab, dim)) return why;
    if (!gtk::known_type(table_type) || !gtk::known_type(out_type)) return "unknown element type";
    if (table_stride < 0 || out_stride < dim) return "table_stride must be >= 0, out_stride >= dim";
    if (n_ids == 0) return nullptr;
    if (!d_ids || !d_table || !d_out) return "null device pointer";
    if (!gtk::aligned_to(d_ids, 4) || !gtk::aligned_to(d_table, gtk::element_size(table_type)) ||
        !gtk::aligned_to(d_out, gtk::element_size(out_type)))
      return "a device pointer is not aligned to its elements";
    return nullptr;
  };
  return gtk::run_operator(h, check, [&](const gtk::HandleView& v) -> cudaError_t {
    if (n_ids == 0) return cudaSuccess;
    const bool packs = gtk::rows_aligned(d_table, table_stride, table_type, 8) && gtk::rows_aligned(d_out, out_stride, out_type, 8);
    return gtk::with_type(table_type, [&](auto t) {
      return gtk::with_type(out_type, [&](auto o) {
        auto f = packs ? launch_embed<decltype(t), decltype(o), 8> : launch_embed<decltype(t), decltype(o), 1>;
        return f(v, d_ids, n_ids, d_table, vocab, dim, table_stride, scale, d_out, out_stride);
      });
    });
  });
}

extern "C" GTK_API int gtk_embed_grad_workspace(gtk_tokenizer* h, int64_t n_ids, int64_t vocab, int64_t dim, size_t* workspace_bytes)
{
  gtk::HandleView v;
  if (!gtk::handle_view(h, &v)) return GTK_ERR_INVALID_ARG;
  try {
    std::lock_guard<std::mutex> lock(*v.mu);
    const gtk::Refusal why = !workspace_bytes ? "workspace_bytes is null" : refuse_sizes(n_ids, vocab, dim);
    if (why) {
      *v.last_error = why;
      return GTK_ERR_INVALID_ARG;
    }
  } catch (...) {
    return GTK_ERR_MEMORY;
  }
  *workspace_bytes = std::max<size_t>(256, grad_plan(n_ids, vocab, dim).bytes);
  return GTK_OK;
}

extern "C" GTK_API int gtk_embed_grad(gtk_tokenizer* h, const int32_t* d_ids, int64_t n_ids, const void* d_grad_out, int out_type,
                                      int64_t out_stride, float scale, int64_t vocab, int64_t dim, void* d_grad_table, int table_type,
                                      int64_t table_stride, int accumulate, void* d_workspace, size_t workspace_bytes)
{
  auto check = [&]() -> gtk::Refusal {
    if (const gtk::Refusal why = refuse_sizes(n_ids, vocab, dim)) return why;
    if (!gtk::known_type(table_type) || !gtk::known_type(out_type)) return "unknown element type";
    if (out_stride < 0 || table_stride < dim) return "out_stride must be >= 0, table_stride >= dim";
    if (n_ids == 0 && accumulate) return nullptr;
    if (!d_grad_table || (n_ids > 0 && (!d_ids || !d_grad_out || !d_workspace))) return "null device pointer";
    if (!gtk::aligned_to(d_ids, 4) || !gtk::aligned_to(d_grad_out, gtk::element_size(out_type)) ||
        !gtk::aligned_to(d_grad_table, gtk::element_size(table_type)))
      return "a device pointer is not aligned to its elements";
    if (n_ids > 0 && !gtk::aligned_to(d_workspace, 16)) return "d_workspace is not aligned to 16 bytes";
    if (n_ids > 0 && workspace_bytes < grad_plan(n_ids, vocab, dim).bytes)
      return "workspace_bytes is less than gtk_embed_grad_workspace says";
    return nullptr;
  };
  return gtk::run_operator(h, check, [&](const gtk::HandleView& v) -> cudaError_t {
    if (n_ids == 0 && accumulate) return cudaSuccess;
    const GradPlan p = grad_plan(n_ids, vocab, dim);
    unsigned char* work = static_cast<unsigned char*>(d_workspace);
    const GradArgs a{nullptr, reinterpret_cast<GradHeader*>(work + p.at_header), int(dim), p.block_log2, out_stride, table_stride, p.pitch,
                     scale, accumulate != 0, reinterpret_cast<float*>(work + p.at_parts)};
    const bool aligned = gtk::rows_aligned(d_grad_out, out_stride, out_type, 8) && gtk::rows_aligned(d_grad_table, table_stride, table_type, 8);
    return gtk::with_type(out_type, [&](auto o) {
      return gtk::with_type(table_type, [&](auto t) {
        using O = decltype(o);
        using T = decltype(t);
        auto f  = aligned ? launch_embed_grad<O, T, true> : launch_embed_grad<O, T, false>;
        return f(v, p, a, d_ids, n_ids, vocab, d_grad_out, d_grad_table, work);
      });
    });
  });
}
