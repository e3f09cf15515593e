// gtk_embed.cu -- embedding lookup with scaling, and its gradient by sorted tokens.
#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>

#include "gtk_rows.cuh"

namespace {

using gtk::Pack;

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
//   k_embed_grad_sort   one cluster sorts the ids (stable, by digits from the lowest), which brings the rows of a sum next
//                       to each other in order of i; the other CTAs meanwhile write the rows that no id points to
//   k_embed_grad_sums   the sorted positions in blocks of equal length, a row group of threads per block; a sum is kept in
//                       registers.  One that lies in a block or reaches over one boundary is its first block's alone; a
//                       longer one is cut at the boundaries and its parts go to the workspace
//   k_embed_grad_join   adds the parts of the long ones from left to right
// Every sum is thus formed in an order that the ids alone decide.
constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32, kSortCtas = 8;
constexpr int kDigitBits = 8, kBins = 1 << kDigitBits;
constexpr int64_t kMaxDim = int64_t(1) << 20;

struct GradPlan {
  int passes;
  int block_log2;   // sorted positions per block of k_embed_grad_sums
  int64_t blocks;
  int64_t pitch;    // 32-bit floats between rows of the parts
  size_t at_pairs[2], at_long, at_parts, bytes;
};

int bits_of(int64_t x)
{
  int b = 0;
  while (x >> b) ++b;
  return b;
}

constexpr int kMinBlockLog2 = 3, kMaxBlockLog2 = 10;

GradPlan grad_plan(int64_t n, int64_t vocab, int64_t dim)
{
  GradPlan p{};
  // keys are 0 .. vocab, the last one stands for ids that take no part
  p.passes     = (bits_of(vocab) + kDigitBits - 1) / kDigitBits;
  p.block_log2 = kMinBlockLog2;
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
  p.at_pairs[0] = room(size_t(n) * sizeof(uint2));
  p.at_pairs[1] = room(size_t(n) * sizeof(uint2));
  p.at_long     = room(size_t(p.blocks + 1) * 4);
  p.at_parts    = room(size_t(p.blocks) * 2 * size_t(p.pitch) * 4);
  p.bytes       = at;
  return p;
}

struct SortArgs {
  const int32_t* ids;
  int64_t n;
  uint32_t vocab;
  int passes;
  uint2 *pairs0, *pairs1;  // {key, place}: written by the first, third .. and by the second, fourth .. pass
  uint32_t* long_sums;  // [0] how many, behind it the blocks in which they begin (k_embed_grad_sums)
};

struct SortShared {
  uint32_t at[kSortWarps][kBins];
  uint32_t total[kBins];
  uint32_t warp_sum[kBins / 32];
};

// The ids of a CTA are a stretch of the whole, those of a warp a stretch of the CTA's; a pass counts the digits of every
// stretch, turns the counts into places (digits in front, then stretches in front) and moves the pairs there.
__device__ void sort_ids(const SortArgs& a, SortShared& S)
{
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cta         = int(cluster.block_rank());
  const int64_t rounds  = (a.n + int64_t(kSortCtas) * kSortThreads - 1) / (int64_t(kSortCtas) * kSortThreads);
  const int64_t first   = (int64_t(cta) * kSortWarps + warp) * rounds * 32;
  const int64_t last    = min(a.n, first + rounds * 32);
  const uint32_t lower  = (1u << lane) - 1u;
  for (int pass = 0; pass < a.passes; ++pass) {
    const int shift   = pass * kDigitBits;
    const uint2* from = pass & 1 ? a.pairs0 : a.pairs1;
    uint2* to         = pass & 1 ? a.pairs1 : a.pairs0;
    auto load = [&](int64_t i) {
      if (pass == 0) return make_uint2(min(uint32_t(__ldg(a.ids + i)), a.vocab), uint32_t(i));
      return __ldcg(from + i);  // written by other SMs of the cluster
    };
    for (int b = lane; b < kBins; b += 32) S.at[warp][b] = 0;
    __syncwarp();
#pragma unroll 4
    for (int64_t i = first + lane; i < last; i += 32) atomicAdd(&S.at[warp][(load(i).x >> shift) & (kBins - 1)], 1u);
    __syncthreads();
    if (tid < kBins) {
      uint32_t sum = 0;
#pragma unroll 8
      for (int w = 0; w < kSortWarps; ++w) {
        const uint32_t c = S.at[w][tid];
        S.at[w][tid]     = sum;
        sum += c;
      }
      S.total[tid] = sum;
    }
    cluster.sync();
    uint32_t before = 0;
    if (tid < kBins) {
      uint32_t all = 0;
#pragma unroll
      for (int c = 0; c < kSortCtas; ++c) {
        const uint32_t t = cluster.map_shared_rank(S.total, c)[tid];
        before += c < cta ? t : 0u;
        all += t;
      }
      uint32_t upto = all;
#pragma unroll
      for (int d = 1; d < 32; d *= 2) {
        const uint32_t o = __shfl_up_sync(0xFFFFFFFFu, upto, d);
        if (lane >= d) upto += o;
      }
      if (lane == 31) S.warp_sum[warp] = upto;
      before += upto - all;
    }
    __syncthreads();
    if (tid < kBins) {
      for (int w = 0; w < warp; ++w) before += S.warp_sum[w];
#pragma unroll 8
      for (int w = 0; w < kSortWarps; ++w) S.at[w][tid] += before;
    }
    __syncthreads();
#pragma unroll 2
    for (int64_t i0 = first; i0 < last; i0 += 32) {
      const int64_t i      = i0 + lane;
      const bool here      = i < last;
      const uint2 x        = here ? load(i) : make_uint2(0u, 0u);
      const uint32_t digit = here ? (x.x >> shift) & uint32_t(kBins - 1) : 0xFFFFFFFFu;
      const uint32_t peers = __match_any_sync(0xFFFFFFFFu, digit);
      const uint32_t place = here ? S.at[warp][digit] + __popc(peers & lower) : 0u;
      __syncwarp();
      if (here && (peers >> lane) == 1u) S.at[warp][digit] = place + 1u;  // the last of the peers
      __syncwarp();
      if (here) to[place] = x;
    }
    cluster.sync();  // the pairs are where the next pass reads them; nobody reads S.total any more
  }
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

// The first cluster sorts, the CTAs behind it clear the rows that no id points to (accumulate == 0): each looks at all ids
// for those of its own rows.
template <class T>
__global__ void __launch_bounds__(kSortThreads, 2) __cluster_dims__(kSortCtas, 1, 1)
k_embed_grad_sort(const SortArgs a, T* __restrict__ grad_table, int dim, int64_t table_stride)
{
  constexpr int kRowsAtOnce = sizeof(SortShared) / 4 * 32;
  __shared__ union {
    SortShared sort;
    uint32_t used[kRowsAtOnce / 32];
  } S;
  if (blockIdx.x < kSortCtas) {
    if (blockIdx.x == 0 && threadIdx.x == 0 && a.n > 0) a.long_sums[0] = 0;
    if (a.n > 0) sort_ids(a, S.sort);
    return;
  }
  const int64_t ctas = gridDim.x - kSortCtas, cta = blockIdx.x - kSortCtas;
  const int64_t share = (a.vocab + ctas - 1) / ctas, end = min(int64_t(a.vocab), (cta + 1) * share);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int64_t v0 = cta * share; v0 < end; v0 += kRowsAtOnce) {
    const int rows = int(min(int64_t(kRowsAtOnce), end - v0));
    for (int w = threadIdx.x; w < (rows + 31) / 32; w += kSortThreads) S.used[w] = 0;
    __syncthreads();
#pragma unroll 8
    for (int64_t i = threadIdx.x; i < a.n; i += kSortThreads) {
      const int64_t v = int64_t(__ldg(a.ids + i)) - v0;
      if (v >= 0 && v < rows) {
        const uint32_t bit = 1u << (v & 31);
        if (!(S.used[v >> 5] & bit)) atomicOr(&S.used[v >> 5], bit);
      }
    }
    __syncthreads();
    for (int v = warp; v < rows; v += kSortWarps)
      if (!(S.used[v >> 5] >> (v & 31) & 1u)) clear_row(grad_table + (v0 + v) * table_stride, dim, lane, 32);
    __syncthreads();
  }
}

// How a thread sees its V columns of a row, `valid` of them within the row.
// Packs: rows start on 16-byte boundaries (or what V elements take), V = 8.
// Words: 16-bit elements at any address, V = 2: the one or two aligned 32-bit words that hold them.  A word is read only
// if an element of the row lies in it, so nothing is touched that the row does not share four bytes with.
// Singles: 32-bit elements, V = 1.
template <class T, int V>
struct Columns {
  static constexpr bool kWords = V == 2 && sizeof(T) == 2;
  Pack<T, kWords ? 4 : V> raw;
  uint32_t odd;
  __device__ __forceinline__ void load(const T* p, int valid)
  {
    if constexpr (kWords) {
      const uintptr_t at  = reinterpret_cast<uintptr_t>(p);
      const uint32_t* w   = reinterpret_cast<const uint32_t*>(at & ~uintptr_t(3));
      odd                 = uint32_t(at & 2) * 8;
      uint32_t* r         = reinterpret_cast<uint32_t*>(&raw);
      r[0]                = __ldg(w);
      r[1]                = odd && valid > 1 ? __ldg(w + 1) : 0u;
    } else if (valid >= V) {
      raw = gtk::load_pack<T, V>(p);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) raw.e[j] = j < valid ? p[j] : gtk::from_float<T>(0.f);
    }
  }
  __device__ __forceinline__ void add_to(float (&sum)[V]) const
  {
    if constexpr (kWords) {
      const uint32_t* r = reinterpret_cast<const uint32_t*>(&raw);
      const uint32_t w  = __funnelshift_r(r[0], r[1], odd);
      const T* e        = reinterpret_cast<const T*>(&w);
      sum[0] += gtk::to_float(e[0]);
      sum[1] += gtk::to_float(e[1]);  // beyond the row's end: never stored
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) sum[j] += gtk::to_float(raw.e[j]);
    }
  }
};

// a finished sum to its row; packs: all V columns may be stored in one piece
template <class T, int V>
__device__ __forceinline__ void store_sum(T* row, int valid, bool packs, float scale, bool accumulate, const float (&sum)[V])
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
  const uint2* pairs;  // sorted {key, place}
  int64_t n;
  uint32_t vocab;
  int dim;
  int block_log2;
  int64_t blocks;
  int64_t out_stride, table_stride, pitch;
  float scale;
  bool accumulate;
  uint32_t* long_sums;
  float* parts;  // [blocks][2][pitch]: of the long sum that begins further left, of the one that begins in the block
};

constexpr int kGradThreads = 256, kGradBlocksPerSm = 4;

// first place in [from, to) whose key is not `key` (the keys are sorted and from there on >= key)
__device__ __forceinline__ int end_of_key(const uint2* pairs, int from, int to, uint32_t key)
{
  while (from < to) {
    const int mid = (from + to) >> 1;
    if (pairs[mid].x == key) from = mid + 1;
    else to = mid;
  }
  return from;
}

// Positions [at, stop) of the keys and places in P: sums of equal keys, each to finish(key, sum) when the key changes; the
// rows are loaded kRowsInFlight at a time, whole packs of V columns where FULL.  Returns whether a last sum is left over.
template <bool FULL, class O, int V, class Finish>
__device__ __forceinline__ bool sum_rows(const uint2* P, int at, int stop, uint32_t vocab, const O* grad_out, int64_t stride, int valid,
                                         uint32_t& key, float (&sum)[V], Finish&& finish)
{
  constexpr int kRowsInFlight = sizeof(Columns<O, V>) > 20 ? 4 : 8;
  key = P[at].x;
#pragma unroll
  for (int j = 0; j < V; ++j) sum[j] = 0.f;
  for (; at < stop; at += kRowsInFlight) {
    Columns<O, V> x[kRowsInFlight];
#pragma unroll
    for (int k = 0; k < kRowsInFlight; ++k) x[k].load(grad_out + int64_t(P[min(at + k, stop - 1)].y) * stride, FULL ? V : valid);
#pragma unroll
    for (int k = 0; k < kRowsInFlight; ++k) {
      if (at + k >= stop) break;
      const uint32_t now = P[at + k].x;
      if (now != key) {
        finish(key, sum);
        key = now;
#pragma unroll
        for (int j = 0; j < V; ++j) sum[j] = 0.f;
      }
      if (key >= vocab) return false;  // ids that take no part, sorted behind all others
      x[k].add_to(sum);
    }
  }
  return true;
}

template <class O, class T, int V>
__global__ void __launch_bounds__(kGradThreads, kGradBlocksPerSm) k_embed_grad_sums(const GradArgs a, const O* __restrict__ grad_out, T* __restrict__ grad_table)
{
  extern __shared__ uint2 s_pairs[];  // [blockDim.y][3 * block + 2]: the block's, its neighbours' and one more at each end
  const int length    = 1 << a.block_log2, window = 3 * length + 2;
  const int64_t block = int64_t(blockIdx.x) * blockDim.y + threadIdx.y;
  const int64_t begin = block << a.block_log2;
  uint2* P            = s_pairs + threadIdx.y * window + length + 1;
  for (int i = int(threadIdx.x) - length - 1; i <= 2 * length; i += blockDim.x)
    P[i] = begin + i >= 0 && begin + i < a.n ? __ldg(a.pairs + begin + i) : make_uint2(0xFFFFFFFFu, 0u);  // beyond the ends: no key
  __syncthreads();
  const int c = (blockIdx.y * blockDim.x + threadIdx.x) * V;
  if (begin >= a.n || c >= a.dim) return;
  const int valid     = a.dim - c;
  const int end       = int(min(int64_t(length), a.n - begin));
  const uint32_t key0 = P[0].x;
  // the sum that begins further left: skipped, or this block's part of a long one
  bool from_left = P[-1].x == key0;
  int at = 0;
  if (from_left && P[end].x != key0 && P[-length - 1].x != key0) {
    at        = end_of_key(P, 0, end, key0);
    from_left = false;
  }
  if (at >= end) return;
  // the sum that reaches over the end: to its end, or up to the boundary when it is a long one
  const uint32_t key1 = P[end - 1].x;
  int stop            = end;
  bool to_right       = false;
  if (P[end].x == key1 && !(from_left && key1 == key0)) {
    to_right = P[2 * length].x == key1;
    if (!to_right) stop = end_of_key(P, end, 2 * length, key1);
    else if (key1 < a.vocab && c == 0) a.long_sums[1 + atomicAdd(a.long_sums, 1u)] = uint32_t(block);
  }
  uint32_t key;
  float sum[V];
  auto part = [&](int which, const float (&x)[V]) {
    Pack<float, V> p;
#pragma unroll
    for (int j = 0; j < V; ++j) p.e[j] = x[j];
    gtk::store_pack<float, V>(a.parts + (block * 2 + which) * a.pitch + c, p);  // the pitch is a multiple of V
  };
  auto finish = [&](uint32_t of, const float (&x)[V]) {
    if (from_left) part(0, x);
    else store_sum<T, V>(grad_table + int64_t(of) * a.table_stride + c, valid, V == 8, a.scale, a.accumulate, x);
    from_left = false;
  };
  const O* column = grad_out + c;
  const bool rest = valid >= V ? sum_rows<true, O, V>(P, at, stop, a.vocab, column, a.out_stride, valid, key, sum, finish)
                               : sum_rows<false, O, V>(P, at, stop, a.vocab, column, a.out_stride, valid, key, sum, finish);
  if (!rest) return;
  if (to_right) part(1, sum);
  else finish(key, sum);
}

// The parts of a long sum, 128 columns at a time: each warp adds a run of parts, then the warps' sums are added in order.
template <class T>
__global__ void __launch_bounds__(kGradThreads) k_embed_grad_join(const GradArgs a, T* __restrict__ grad_table, bool packs)
{
  constexpr int kWarps = kGradThreads / 32;
  __shared__ float4 s_sum[kWarps][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slabs     = (a.dim + 127) / 128;
  const int64_t items = int64_t(a.long_sums[0]) * slabs;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t block = a.long_sums[1 + item / slabs];
    const int c         = int(item % slabs) * 128 + lane * 4;
    const uint32_t key  = a.pairs[((block + 1) << a.block_log2) - 1].x;
    int64_t more = 0;  // blocks behind this one that begin with the same key
    for (int found = kGradThreads; found == kGradThreads; more += found) {
      const int64_t b = block + 1 + more + threadIdx.x;
      found           = __syncthreads_count(b < a.blocks && a.pairs[b << a.block_log2].x == key);
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
      store_sum<T, 4>(grad_table + int64_t(key) * a.table_stride + c, a.dim - c, packs, a.scale, a.accumulate, y);
    }
    __syncthreads();
  }
}

// columns of a row over the x dimension of a block
unsigned column_threads(int64_t dim, int pack)
{
  const int64_t packs = (dim + pack - 1) / pack;
  if (packs >= kGradThreads) return kGradThreads;
  if (packs >= 32) return unsigned((packs + 31) / 32 * 32);
  unsigned x = 1;
  while (x < packs) x *= 2;
  return x;
}

template <class O, class T, int V>
cudaError_t launch_embed_grad(const gtk::HandleView& v, const GradPlan& p, GradArgs a, const int32_t* ids, const void* grad_out,
                              void* grad_table, unsigned char* work)
{
  T* table = static_cast<T*>(grad_table);
  SortArgs s{ids, a.n, a.vocab, p.passes, reinterpret_cast<uint2*>(work + p.at_pairs[0]), reinterpret_cast<uint2*>(work + p.at_pairs[1]),
             a.long_sums};
  int64_t clear = 0;  // clusters that clear: one CTA per 64 KiB, as many as there are SMs
  if (!a.accumulate)
    clear = std::max<int64_t>(1, std::min<int64_t>(2 * v.sm_count / kSortCtas - 8, int64_t(a.vocab) * a.dim * int64_t(sizeof(T)) / (int64_t(kSortCtas) << 16)));
  cudaError_t e = gtk::launch(k_embed_grad_sort<T>, dim3(unsigned((1 + clear) * kSortCtas)), dim3(kSortThreads), 0, v.stream, s, table, a.dim,
                              a.table_stride);
  if (e != cudaSuccess || a.n == 0) return e;
  a.pairs = p.passes & 1 ? s.pairs0 : s.pairs1;
  const unsigned tx = column_threads(a.dim, V), slabs = unsigned((a.dim + tx * V - 1) / (tx * V));
  const unsigned pairs_bytes = unsigned(sizeof(uint2)) * ((3u << a.block_log2) + 2u);  // of a row group, 24 KiB at most
  const unsigned ty = std::max(1u, std::min(kGradThreads / tx, 49152u / pairs_bytes));
  e = gtk::launch(k_embed_grad_sums<O, T, V>, dim3(unsigned((p.blocks + ty - 1) / ty), slabs), dim3(tx, ty),
                  size_t(ty) * pairs_bytes, v.stream, a, static_cast<const O*>(grad_out), table);
  // a sum is long when it holds a whole block
  if (e == cudaSuccess && p.blocks > 2)
    e = gtk::launch(k_embed_grad_join<T>, dim3(unsigned(std::min<int64_t>(p.blocks * ((a.dim + 127) / 128), int64_t(v.sm_count) * 8))),
                    dim3(kGradThreads), 0, v.stream, a, table, V == 8);
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
    const GradArgs a{nullptr, n_ids, uint32_t(vocab), int(dim), p.block_log2, p.blocks, out_stride, table_stride, p.pitch, scale, accumulate != 0,
                     reinterpret_cast<uint32_t*>(work + p.at_long), reinterpret_cast<float*>(work + p.at_parts)};
    const bool packs = gtk::rows_aligned(d_grad_out, out_stride, out_type, 8) && gtk::rows_aligned(d_grad_table, table_stride, table_type, 8);
    return gtk::with_type(out_type, [&](auto o) {
      return gtk::with_type(table_type, [&](auto t) {
        using O = decltype(o);
        using T = decltype(t);
        auto f  = packs ? launch_embed_grad<O, T, 8> : launch_embed_grad<O, T, sizeof(O) == 2 ? 2 : 1>;
        return f(v, p, a, d_ids, d_grad_out, d_grad_table, work);
      });
    });
  });
}
