// gtk_embed.cu -- embedding lookup with scaling, and its gradient by sorted tokens.
#include <algorithm>
#include <cmath>

#include "gtk_checked.cuh"
#include "gtk_long_sums.hpp"
#include "gtk_rows.cuh"

namespace {

using gtk::LongSum;
using gtk::Pack;
using gtk::Two;

// ------------------------------------------------------------------------------------------------ lookup
// out[i] = scale * table[ids[i]], a product in 32 bits and one rounding.  Each row is read once and written once, so memory bounds
// it: 32768 rows of 1024 bf16 take 18.3 us, 74 % of the measured copy rate over the bytes that differ; a few rows are a
// launch and two waits behind one another, for the id and for the row (1.7 us).  A block's threads are split into groups of 1 << group_log2; a group copies ROWS rows at a time, so
// that the wait for an id and then for its row is shared by several.
// V = 8: rows of both arrays start where 8 elements may be moved at once.  V = 2: any rows, two columns at a time, but where both
// types have 16 bits the 16 bytes between two boundaries of the output come from two such pieces of the table (30000 rows of
// 1601 bf16: 37 us a call, in pairs 45; 20000 rows of 333 f32, which are 14.4 that way, are left at 12.3 in pairs).
constexpr int kEmbedThreads = 256;

// Two neighbouring elements at any address.  16-bit ones come in the one or two aligned 32-bit words that hold them; a word
// is read only if a wanted element lies in it.
template <class T>
__device__ __forceinline__ uint2 load_two(const T* p, bool second)
{
  if constexpr (sizeof(T) == 4) {
    return make_uint2(__ldg(reinterpret_cast<const uint32_t*>(p)), second ? __ldg(reinterpret_cast<const uint32_t*>(p) + 1) : 0u);
  } else {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(reinterpret_cast<uintptr_t>(p) & ~uintptr_t(3));
    const bool odd    = reinterpret_cast<uintptr_t>(p) & 2;
    return make_uint2(__ldg(w), odd && second ? __ldg(w + 1) : 0u);
  }
}
template <class T>
__device__ __forceinline__ void two_floats(uint2 raw, const T* p, float& a, float& b)
{
  if constexpr (sizeof(T) == 4) a = __uint_as_float(raw.x), b = __uint_as_float(raw.y);
  else gtk::word_pair(__funnelshift_r(raw.x, raw.y, uint32_t(reinterpret_cast<uintptr_t>(p) & 2) * 8), T{}).get(a, b);
}
template <class O>
__device__ __forceinline__ void store_two(O* p, bool second, float a, float b)
{
  Pack<O, 2> y;
  y.e[0] = gtk::from_float<O>(a), y.e[1] = gtk::from_float<O>(b);
  if (second && reinterpret_cast<uintptr_t>(p) % sizeof(y) == 0) {
    gtk::store_pack<O, 2>(p, y);
  } else {
    p[0] = y.e[0];
    if (second) p[1] = y.e[1];
  }
}

// the 16 bytes that begin `bytes` (below 16, and even) behind the first of two pieces
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

// A row of any alignment to one of any other, both of 16-bit types.  A piece of 16 bytes is read only if a wanted
// element lies in it.
template <class T, class O>
__device__ __forceinline__ void copy_row(const T* from, O* to, int dim, float scale, int lane, int group)
{
  constexpr int E = 16 / int(sizeof(O)), kAhead = 4;
  const int head  = min(dim, int((16u - (uint32_t(reinterpret_cast<uintptr_t>(to)) & 15u)) % 16u / sizeof(O)));
  const int packs = (dim - head) / E;
  const uintptr_t at    = reinterpret_cast<uintptr_t>(from + head);
  const uint32_t shift  = uint32_t(at & 15);  // the same for all packs
  const uint4* pieces   = reinterpret_cast<const uint4*>(at - shift);
  uint4* out            = reinterpret_cast<uint4*>(to + head);
  for (int p0 = lane; p0 < packs; p0 += kAhead * group) {
    uint4 a[kAhead], b[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (p0 + k * group < packs) {
        a[k] = __ldg(pieces + p0 + k * group);
        b[k] = shift ? __ldg(pieces + p0 + k * group + 1) : make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (p0 + k * group < packs) {
        const uint4 raw = shifted(a[k], b[k], shift);
        const T* x      = reinterpret_cast<const T*>(&raw);
        Pack<O, E> y;
#pragma unroll
        for (int j = 0; j < E; ++j) y.e[j] = gtk::from_float<O>(gtk::to_float(x[j]) * scale);
        out[p0 + k * group] = *reinterpret_cast<const uint4*>(&y);
      }
  }
  for (int i = lane; i < dim - packs * E; i += group) {
    const int c = i < head ? i : i + packs * E;
    to[c]       = gtk::from_float<O>(gtk::to_float(__ldg(from + c)) * scale);
  }
}

template <class T, class O, int V, int ROWS>
__global__ void __launch_bounds__(kEmbedThreads)
k_embed(const int32_t* __restrict__ ids, int64_t n, const T* __restrict__ table, int vocab, int dim, int64_t table_stride,
        float scale, O* __restrict__ out, int64_t out_stride, int group_log2)
{
  const int group = 1 << group_log2, lane = threadIdx.x & (group - 1);
  const int64_t first = (int64_t(blockIdx.x) * (kEmbedThreads >> group_log2) + (threadIdx.x >> group_log2)) * ROWS;
  int id[ROWS];
  const T* from[ROWS];
  O* to[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) id[r] = first + r < n ? __ldg(ids + first + r) : -1;
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const bool has = uint32_t(id[r]) < uint32_t(vocab);
    from[r]        = has ? table + int64_t(id[r]) * table_stride : nullptr;
    to[r]          = out + (first + r) * out_stride;
    if (!has && first + r < n) {
      const O fill = gtk::from_float<O>(id[r] < 0 ? 0.f : __int_as_float(0x7FC00000));
      for (int c = lane; c < dim; c += group) to[r][c] = fill;
    }
  }
  if constexpr (V == 8) {
    constexpr int kAhead = ROWS == 1 ? 4 : sizeof(T) == 2 ? 2 : 1;
    const int packs      = dim / V;
    for (int u0 = lane; u0 < packs; u0 += kAhead * group) {
      Pack<T, V> x[ROWS][kAhead];
#pragma unroll
      for (int r = 0; r < ROWS; ++r)
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
          if (from[r] && u0 + k * group < packs) x[r][k] = gtk::load_pack<T, V>(from[r] + (u0 + k * group) * V);
#pragma unroll
      for (int r = 0; r < ROWS; ++r)
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
          if (from[r] && u0 + k * group < packs) {
            Pack<O, V> y;
#pragma unroll
            for (int j = 0; j < V; ++j) y.e[j] = gtk::from_float<O>(gtk::to_float(x[r][k].e[j]) * scale);
            gtk::store_pack<O, V>(to[r] + (u0 + k * group) * V, y);
          }
    }
    for (int c = packs * V + lane; c < dim; c += group)
#pragma unroll
      for (int r = 0; r < ROWS; ++r)
        if (from[r]) to[r][c] = gtk::from_float<O>(gtk::to_float(from[r][c]) * scale);
  } else if constexpr (sizeof(T) + sizeof(O) == 4) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
      if (from[r]) copy_row(from[r], to[r], dim, scale, lane, group);
  } else {
    constexpr int kAhead = 4;
    const int pairs      = (dim + 1) / 2;
    for (int u0 = lane; u0 < pairs; u0 += kAhead * group) {
      uint2 x[ROWS][kAhead];
#pragma unroll
      for (int r = 0; r < ROWS; ++r)
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          const int c = (u0 + k * group) * 2;
          if (from[r] && c < dim) x[r][k] = load_two(from[r] + c, c + 1 < dim);
        }
#pragma unroll
      for (int r = 0; r < ROWS; ++r)
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          const int c = (u0 + k * group) * 2;
          if (from[r] && c < dim) {
            float a, b;
            two_floats(x[r][k], from[r] + c, a, b);
            store_two(to[r] + c, c + 1 < dim, a * scale, b * scale);
          }
        }
    }
  }
}

template <class T, class O, int V>
cudaError_t launch_embed(const gtk::HandleView& v, const int32_t* ids, int64_t n, const void* table, int64_t vocab, int64_t dim,
                         int64_t table_stride, float scale, void* out, int64_t out_stride)
{
  // Lanes for a row: a quarter as many as it has units, a warp at most; more, up to one per unit, while that keeps the GPU's threads
  // from being used up (2048 rows of 1024 bf16: 2.5 us with 32 lanes, 3.3 with 128; 64 rows of 768: 2.1 and 1.9).  Many rows
  // of packs go two at once (32768 rows of 1024 bf16: 18.1 us, one at once 19.0, four 24.8; 100000 rows of 256: 14.8, with a lane
  // for every pack 34.4), others one.
  const int64_t units = V == 2 && sizeof(T) + sizeof(O) == 4 ? (dim * int64_t(sizeof(O)) + 15) / 16 : (dim + V - 1) / V;
  const bool many     = n >= int64_t(v.sm_count) * 64;
  int group_log2      = 0;
  while (group_log2 < 5 && (int64_t(4) << group_log2) < units) ++group_log2;
  while (group_log2 < 8 && (int64_t(1) << group_log2) < units && n << (group_log2 + 1) <= int64_t(v.sm_count) * 512) ++group_log2;
  const int64_t rows = (kEmbedThreads >> group_log2) * (many && V == 8 ? 2 : 1);
  auto kernel        = k_embed<T, O, V, 1>;
  if constexpr (V == 8)
    if (many) kernel = k_embed<T, O, V, 2>;
  return gtk::launch(kernel, dim3(unsigned((n + rows - 1) / rows)), dim3(kEmbedThreads), 0,
                     v.stream, ids, n, static_cast<const T*>(table), int(vocab), int(dim), table_stride, scale, static_cast<O*>(out), out_stride,
                     group_log2);
}

// ------------------------------------------------------------------------------------------------ gradient
// grad_table[v] = scale * sum of grad_out[i] over the i with ids[i] == v, in three launches:
//   k_embed_grad_sort   groups the tokens by id, which brings the rows of a sum next to each other in order of i, and
//                       clears the rows that no id points to
//   k_embed_grad_sums   the grouped tokens in blocks of equal length, a group of threads per block; a sum is kept in registers.
//                       One that lies in a block or reaches over one boundary is its first block's alone; a longer one is cut
//                       at the boundaries and its parts go to the workspace
//   k_embed_grad_join   adds the parts of the long ones from left to right
// Every sum is thus formed in an order that the ids alone decide, in 32 bits, and rounded once.  A row of grad_out is read once and a
// row of grad_table written once: that traffic is the floor, and the grouping, which the rows wait for, is what comes on top.
// 32768 tokens of 768 bf16 to 50257 rows of f32: 57 us (30, 20 and 6.6 of the three; the last two begin while their predecessor
// ends, which takes 4 us off), at the copy rate 32.  4096 tokens: 42 us, nearly all of it the 154 MB of zeros.  131072 tokens: 108
// (43, 50, 14), at the copy rate 55.
constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32;
// CTAs of k_embed_grad_sort, one to an SM.  All of them read all ids, from the second-level cache: no CTA waits for another and one
// launch does it all, while up to some 100 000 ids the clearing of rows hides it (32768 tokens and 154 MB of table: 30 us, without
// clearing 11.4, clearing all of it without a token 26.7).  Beyond, the reading shows: 1M tokens, 350 us.  An id that a large part of the tokens has is one CTA's work:
// 32768 tokens of which half have one id take 41 us here, all of them 82.
constexpr int kOwnersLog2 = 7, kOwners = 1 << kOwnersLog2;
constexpr int kMaxDigitBits = 9;                            // a thread per bin at most
constexpr int64_t kMaxDim = int64_t(1) << 20;

struct GradPlan {
  int passes, digit_bits;
  int block_log2;   // tokens per block of k_embed_grad_sums
  int64_t blocks;
  int64_t pitch;    // 32-bit floats between rows of the parts
  size_t at_tokens[2], at_long, at_parts, bytes;
};

int bits_of(int64_t x)
{
  int b = 0;
  while (x >> b) ++b;
  return b;
}

constexpr size_t kSharedGroups = 96 << 10;  // of a CTA, where it has the choice of fewer groups
constexpr int kMinBlockLog2 = 3, kMaxBlockLog2 = 10;

GradPlan grad_plan(int64_t n, int64_t vocab, int64_t dim)
{
  GradPlan p{};
  const int bits = std::max(1, bits_of((vocab - 1) >> kOwnersLog2));
  p.passes       = (bits + kMaxDigitBits - 1) / kMaxDigitBits;
  p.digit_bits   = (bits + p.passes - 1) / p.passes;
  p.block_log2   = kMinBlockLog2;
  // Blocks of 8 to 32 tokens: as long as they leave some 600 000 columns of blocks, so that all SMs have work (sums and join of 4096
  // tokens of 768: 12 us with 8, 15 with 32, 20 with 64; of 131072 tokens of 1601: 175, 115, 115), and longer, up to 64, where
  // there were more than 4096 of them, for the parts of the most frequent id's sum are added one after the other (131072 tokens of
  // 64: 33 us with 8, 23 with 32, 34 with 64).  Longer ones only where the parts would take more than 32 MiB.
  while (p.block_log2 < 5 && (n >> (p.block_log2 + 1)) * dim >= 600000) ++p.block_log2;
  while (p.block_log2 < 6 && n >> p.block_log2 > 4096) ++p.block_log2;
  while (p.block_log2 < kMaxBlockLog2 && (n >> p.block_log2) * dim * 8 > (int64_t(32) << 20)) ++p.block_log2;
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
  p.at_long      = room(size_t(p.blocks) * sizeof(LongSum));
  p.at_parts     = room(size_t(p.blocks) * 2 * size_t(p.pitch) * 4);
  p.bytes        = at;
  return p;
}

struct SortArgs {
  const int32_t* ids;
  int64_t n;
  uint32_t vocab;
  int passes, digit_bits, block_log2;
  uint2 *tokens0, *tokens1;  // {id, place}: the grouped tokens end up in tokens0 after an even number of passes
  LongSum* long_sums;  // one per block
};

constexpr uint32_t kNoId = 0xFFFFFFFFu;  // ids are below 2^31
constexpr int kListRoom  = 600;          // tokens of an owner that a warp finds in its part of the text
// Tokens of an owner that are sorted by counting those in front of each: 512 tokens in all take the kernel 6.9 us, with the digits'
// barriers 8.1, 8192 take 28.8 and 30.3; with up to 192 of an owner's instead 32768 took 0.7 longer.
constexpr uint32_t kRankMost = 128;

struct SortShared {
  uint32_t at[kSortWarps][1 << kMaxDigitBits];
  uint2 list[kSortWarps][kListRoom];
  uint32_t warp_sum[kSortWarps];
  uint32_t lower[kSortWarps], mine[kSortWarps];
};

// The sum over the warps in front and over all of them, of a number that each warp has put into v.
__device__ __forceinline__ void over_warps(const uint32_t* v, int warp, int lane, uint32_t& front, uint32_t& all)
{
  const uint32_t mine = v[lane];  // kSortWarps == 32
  uint32_t upto       = mine;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const uint32_t o = __shfl_up_sync(0xFFFFFFFFu, upto, d);
    if (lane >= d) upto += o;
  }
  front = __shfl_sync(0xFFFFFFFFu, upto - mine, warp);
  all   = __shfl_sync(0xFFFFFFFFu, upto, 31);
}

// One digit of a stable sort of the CTA's own tokens, of which this warp has from[0 .. count) (each warp those behind the
// warp in front).  Each warp counts its digits and moves its tokens to the places that digits in front and warps in front leave.
__device__ void sort_digit(const uint2* from, uint32_t count, uint2* to, int shift, int digit_bits, SortShared& S)
{
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int bins       = 1 << digit_bits;
  const uint32_t lower = (1u << lane) - 1u;
  for (int b = lane; b < bins; b += 32) S.at[warp][b] = 0;
  __syncwarp();
  // The lanes of one digit are counted by the last of them: a frequent id would have them wait for each other at one address.
  auto peers_of = [&](uint32_t digit) { return __match_any_sync(0xFFFFFFFFu, digit); };
#pragma unroll 4
  for (uint32_t i0 = 0; i0 < count; i0 += 32) {
    const bool here      = i0 + lane < count;
    const uint32_t digit = here ? (from[i0 + lane].x >> shift) & uint32_t(bins - 1) : 0xFFFFFFFFu;
    const uint32_t peers = peers_of(digit);
    if (here && (peers >> lane) == 1u && GTK_IN(digit, 1 << kMaxDigitBits, 200)) S.at[warp][digit] += __popc(peers);
    __syncwarp();
  }
  __syncthreads();
  uint32_t counts[kSortWarps], sum = 0;
  if (tid < bins) {
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) counts[w] = S.at[w][tid];
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) sum += counts[w];
  }
  uint32_t upto = sum;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const uint32_t o = __shfl_up_sync(0xFFFFFFFFu, upto, d);
    if (lane >= d) upto += o;
  }
  if (lane == 31) S.warp_sum[warp] = upto;
  __syncthreads();
  uint32_t at, all;
  over_warps(S.warp_sum, warp, lane, at, all);
  at += upto - sum;
  if (tid < bins) {
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) {
      S.at[w][tid] = at;
      at += counts[w];
    }
  }
  __syncthreads();
#pragma unroll 2
  for (uint32_t i0 = 0; i0 < count; i0 += 32) {
    const bool here      = i0 + lane < count;
    const uint2 x        = here ? from[i0 + lane] : make_uint2(0u, 0u);
    const uint32_t digit = here ? (x.x >> shift) & uint32_t(bins - 1) : 0xFFFFFFFFu;
    const uint32_t peers = peers_of(digit);
    const uint32_t place = here ? S.at[warp][digit] + __popc(peers & lower) : 0u;
    __syncwarp();
    if (here && (peers >> lane) == 1u) S.at[warp][digit] = place + 1u;  // the last of the peers
    __syncwarp();
    if (here && GTK_IN(place, all, 201)) to[place] = x;
  }
  __syncthreads();
}

// f(id[4], place of the first) for the ids of the warp's part, four per lane at a time.  Ids in front of the array and behind
// it, which share 16 bytes with its ends, are kNoId.
template <class F>
__device__ __forceinline__ void scan_ids(const SortArgs& a, int warp, int lane, F&& f)
{
  const int64_t skip  = int64_t(reinterpret_cast<uintptr_t>(a.ids) & 15u) / 4;
  const uint4* quads  = reinterpret_cast<const uint4*>(a.ids - skip);
  const int64_t count = (a.n + skip + 3) / 4, each = ((count + kSortWarps - 1) / kSortWarps + 31) / 32 * 32;
  const int64_t last  = min(count, (warp + 1) * each);
  constexpr int kAhead = 4;
  for (int64_t q0 = warp * each; q0 < last; q0 += 32 * kAhead) {
    uint4 x[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) x[k] = q0 + k * 32 + lane < last ? __ldg(quads + q0 + k * 32 + lane) : make_uint4(kNoId, kNoId, kNoId, kNoId);
    const bool edge = q0 * 4 < skip || (q0 + 32 * kAhead) * 4 - skip > a.n;  // the same for the warp
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int64_t i = (q0 + k * 32 + lane) * 4 - skip;
      uint32_t id[4]  = {x[k].x, x[k].y, x[k].z, x[k].w};
      if (edge)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (i + j < 0 || i + j >= a.n) id[j] = kNoId;
      f(id, i);
    }
  }
}

// Four ids' owners in the bytes of a word (those that take no part count as the last one's), and from them, as bit 7 of each
// byte, whose owner is lower or this one: bytes below 128 neither borrow from nor carry into their neighbours here.
struct Owners {
  uint32_t of;
  __device__ __forceinline__ Owners(const uint32_t (&id)[4], uint32_t vocab)
  {
    uint32_t x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = id[j] < vocab ? id[j] : uint32_t(kOwners - 1);
    of = __byte_perm(__byte_perm(x[0], x[1], 0x0040), __byte_perm(x[2], x[3], 0x0040), 0x5410) & 0x7F7F7F7Fu;
  }
  __device__ __forceinline__ uint32_t below(uint32_t owner4) const { return ~((of | 0x80808080u) - owner4) & 0x80808080u; }
  __device__ __forceinline__ uint32_t equal(uint32_t owner4) const { return ~((of ^ owner4) + 0x7F7F7F7Fu) & 0x80808080u; }
};
static_assert(kOwners == 128, "an owner is seven bits of a byte");

// CTA c owns the ids with id % kOwners == c: it looks at all ids, learns how many tokens lower owners have, which is where
// its own go, and sorts its own.  Nothing is waited for between CTAs.  Returns its share of the grouped tokens; behind the
// last share are tokens of no id.
__device__ void group_tokens(const SortArgs& a, SortShared& S, uint32_t& begin, uint32_t& count)
{
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t owner = blockIdx.x, lanes_below = (1u << lane) - 1u;
  const uint32_t owner4 = owner * 0x01010101u;
  uint32_t lower = 0, mine = 0;
  // The tokens of one step that are this owner's to to[], in order, as far as there is room; returns how many.
  auto take = [&](const uint32_t (&id)[4], const Owners& o, int64_t i, uint2* to, uint32_t room, const uint2* whole, int64_t size) {
    uint32_t bits = o.equal(owner4);
    if (owner == kOwners - 1)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (id[j] >= a.vocab) bits &= ~(0x80u << 8 * j);
    const uint32_t lanes = __ballot_sync(0xFFFFFFFFu, bits != 0);
    if (!lanes) return 0u;
    if (!__any_sync(0xFFFFFFFFu, bits & (bits - 1))) {  // one per lane at most
      const uint32_t at = __popc(lanes & lanes_below);
      const int j       = __clz(__brev(bits)) >> 3;
      if (bits && at < room && GTK_IN(to + at - whole, size, 202)) to[at] = make_uint2(j == 0 ? id[0] : j == 1 ? id[1] : j == 2 ? id[2] : id[3], uint32_t(i + j));
      return uint32_t(__popc(lanes));
    }
    uint32_t total = 0, at = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t mask = __ballot_sync(0xFFFFFFFFu, bits >> (8 * j + 7) & 1u);
      total += __popc(mask);
      at += __popc(mask & lanes_below);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (bits >> (8 * j + 7) & 1u) {
        if (at < room && GTK_IN(to + at - whole, size, 203)) to[at] = make_uint2(id[j], uint32_t(i + j));
        ++at;
      }
    return total;
  };
  scan_ids(a, warp, lane, [&](const uint32_t (&id)[4], int64_t i) {
    const Owners o(id, a.vocab);
    lower += __popc(o.below(owner4));
    mine += take(id, o, i, S.list[warp] + mine, mine < kListRoom ? kListRoom - mine : 0u, S.list[warp], kListRoom);
  });
  lower = __reduce_add_sync(0xFFFFFFFFu, lower);
  if (lane == 0) S.lower[warp] = lower, S.mine[warp] = mine;
  const bool listed = !__syncthreads_or(mine > kListRoom);
  uint32_t at;
  over_warps(S.lower, warp, lane, at, begin);
  over_warps(S.mine, warp, lane, at, count);
  if (owner == kOwners - 1) {  // behind the last share
    uint2* const last = a.passes & 1 ? a.tokens1 : a.tokens0;
    for (int64_t i = int64_t(begin) + count + tid; i < a.n; i += kSortThreads) {
      last[i] = make_uint2(kNoId, 0u);
      if (i + 1 == a.n || ((i + 1) & ((1 << a.block_log2) - 1)) == 0) a.long_sums[i >> a.block_log2] = LongSum{kNoId, 0u};
    }
  }
  if (count == 0) return;
  if (!listed) {
    uint2* to = a.tokens0 + begin + at;
    scan_ids(a, warp, lane, [&](const uint32_t (&id)[4], int64_t i) { to += take(id, Owners(id, a.vocab), i, to, 128u, a.tokens0, a.n); });
    __syncthreads();
  }
  if (listed && count <= kRankMost) {  // each token's place is the number of those in front of it
    uint64_t* const keys = reinterpret_cast<uint64_t*>(S.at);
    for (uint32_t k = lane; k < mine; k += 32)
      if (GTK_IN(at + k, kRankMost, 204)) keys[at + k] = uint64_t(S.list[warp][k].x) << 32 | S.list[warp][k].y;
    __syncthreads();
    if (tid < int(count)) {
      const uint64_t key = keys[tid];
      uint32_t place     = 0;
#pragma unroll 8
      for (uint32_t k = 0; k < count; ++k) place += keys[k] < key;
      if (GTK_IN(place, count, 205)) (a.passes & 1 ? a.tokens1 : a.tokens0)[begin + place] = make_uint2(uint32_t(key >> 32), uint32_t(key));
    }
    __syncthreads();
    return;
  }
  const uint32_t stretch = (count + kSortThreads - 1) / kSortThreads * 32, first = min(count, warp * stretch), some = min(count - first, stretch);
  for (int pass = 0; pass < a.passes; ++pass) {
    const bool from_list = pass == 0 && listed;
    sort_digit(from_list ? S.list[warp] : (pass & 1 ? a.tokens1 : a.tokens0) + begin + first, from_list ? mine : some,
               (pass & 1 ? a.tokens0 : a.tokens1) + begin, kOwnersLog2 + pass * a.digit_bits, a.digit_bits, S);
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

template <class T>
__global__ void __launch_bounds__(kSortThreads, 1)
k_embed_grad_sort(const SortArgs a, T* __restrict__ grad_table, int dim, int64_t table_stride, bool clear)
{
  extern __shared__ uint4 s_raw[];
  SortShared& S = *reinterpret_cast<SortShared*>(s_raw);
  uint32_t begin = 0, count = 0;
  if (a.n > 0) group_tokens(a, S, begin, count);
  const uint2* tokens = (a.passes & 1 ? a.tokens1 : a.tokens0) + begin;
  gtk::each_long_sum(
      begin, int64_t(begin) + count, a.n, a.block_log2, threadIdx.x, kSortThreads,
      [&](int64_t place) { return GTK_IN(place - begin, count, 206) ? tokens[place - begin].x : kNoId; },
      [&](int64_t block, const LongSum& L) {
        if (GTK_IN(block, (a.n + (int64_t(1) << a.block_log2) - 1) >> a.block_log2, 207)) a.long_sums[block] = L;
      });
  if (!clear) return;
  // the rows of this owner that have no token, as many at once as the shared memory has bits
  uint32_t* used        = &S.at[0][0];
  constexpr int kAtOnce = sizeof(S.at) * 8;
  const int64_t rows    = (int64_t(a.vocab) - int64_t(blockIdx.x) + kOwners - 1) >> kOwnersLog2;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int64_t r0 = 0; r0 < rows; r0 += kAtOnce) {
    const int here = int(min(int64_t(kAtOnce), rows - r0));
    __syncthreads();
    for (int w = threadIdx.x; w < (here + 31) / 32; w += kSortThreads) used[w] = 0;
    __syncthreads();
#pragma unroll 4
    for (uint32_t i = threadIdx.x; i < count; i += kSortThreads) {
      const int64_t r = int64_t(tokens[i].x >> kOwnersLog2) - r0;
      if (r >= 0 && r < here && GTK_IN(r >> 5, kSortWarps << kMaxDigitBits, 208) && !(used[r >> 5] >> (r & 31) & 1u)) atomicOr(used + (r >> 5), 1u << (r & 31));
    }
    __syncthreads();
    for (int r = warp; r < here; r += kSortWarps)
      if (!(used[r >> 5] >> (r & 31) & 1u) && GTK_IN(((r0 + r) << kOwnersLog2) + blockIdx.x, a.vocab, 209)) clear_row(grad_table + (((r0 + r) << kOwnersLog2) + blockIdx.x) * table_stride, dim, lane, 32);
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
  const uint2* tokens;  // grouped {id, place}, those of no id behind them
  int64_t n;
  uint32_t vocab;
  LongSum* long_sums;  // one per block
  int dim;
  int block_log2;
  int64_t out_stride, table_stride, pitch;
  float scale;
  bool accumulate;
  float* parts;  // [blocks][2][pitch]: of the long sum that begins further left, of the one that begins in the block
};

// Rows that are waited for together, and such chunks in flight (131072 rows of 1601 bf16: 4 and 3 102 us, 4 and 2 108, 4 and 4 109,
// 2 and 4 106, 8 and 3 131: what shared memory a group takes is taken from the number of groups).
constexpr int kChunk = 4, kChunks = 3;

// first place in [from, to) whose id is not `id` (where one id follows another it does not come back)
__device__ __forceinline__ int end_of_id(const uint32_t* ids, int from, int to, uint32_t id)
{
  while (from < to) {
    const int mid = (from + to) >> 1;
    if (ids[mid] == id) from = mid + 1;
    else to = mid;
  }
  return from;
}

// how many of the places in front of `length` hold a token
__device__ __forceinline__ int end_of_tokens(const uint32_t* ids, int length)
{
  int from = 0;
  while (from < length) {
    const int mid = (from + length) >> 1;
    if (ids[mid] != kNoId) from = mid + 1;
    else length = mid;
  }
  return from;
}

// How a group's threads share the columns of a slab: a thread has kUnits units of kUnit neighbouring columns.
// ALIGNED (rows of both arrays start where 16 bytes of grad_out's elements do): one unit, the 16 bytes that it copies itself.
// Otherwise: four units of 32 bits each, 32 units apart, so that the threads of a warp read and store neighbouring words
// however a row lies.
template <class O, bool ALIGNED>
struct Share {
  static constexpr int kUnit  = (ALIGNED ? 16 : 4) / int(sizeof(O));
  static constexpr int kUnits = ALIGNED ? 1 : 4;
  static constexpr int kCount = kUnit * kUnits;
};

// sum[u * kUnit ..] += the thread's units of a staged row; `shift` bytes of its first piece belong to what lies in front of it.
// Unless ALIGNED, `mine` counts 32-bit words and the units are kStep words apart.
constexpr int kStep = 32;
template <bool ALIGNED, class O>
__device__ __forceinline__ void add_row(const uint4* row, int mine, uint32_t shift, Two (&sum)[16 / sizeof(O) / 2])
{
  uint4 r;
  if constexpr (ALIGNED) {
    r = row[mine];
  } else {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(row) + (shift >> 2) + mine;
    r = make_uint4(w[0], w[kStep], w[2 * kStep], w[3 * kStep]);
    if (sizeof(O) == 2 && (shift & 2)) {  // the same for the whole group: pairs of elements that lie in two words
      r.x = __funnelshift_r(r.x, w[1], 16);
      r.y = __funnelshift_r(r.y, w[kStep + 1], 16);
      r.z = __funnelshift_r(r.z, w[2 * kStep + 1], 16);
      r.w = __funnelshift_r(r.w, w[3 * kStep + 1], 16);
    }
  }
  if constexpr (sizeof(O) == 4) {
    sum[0] = sum[0] + Two(__uint_as_float(r.x), __uint_as_float(r.y));
    sum[1] = sum[1] + Two(__uint_as_float(r.z), __uint_as_float(r.w));
  } else {
    sum[0] = sum[0] + gtk::word_pair(r.x, O{});
    sum[1] = sum[1] + gtk::word_pair(r.y, O{});
    sum[2] = sum[2] + gtk::word_pair(r.z, O{});
    sum[3] = sum[3] + gtk::word_pair(r.w, O{});
  }
}

// Shared memory of a group: the ring of 16-byte pieces (and one more: whoever takes words from the last piece looks into the
// next one), the addresses of the rows and the ids of two blocks of tokens, and room for a chunk behind them.
struct GroupShared {
  int ring, tokens;
  __host__ __device__ GroupShared(int group, int length) : ring((kChunk * kChunks * group + 1) * 16), tokens(2 * length + kChunk) {}
  __host__ __device__ int bytes() const { return ring + (tokens * 12 + 15) / 16 * 16; }
};

// A group of threads (part of a warp, or the whole CTA) takes a block of tokens.  One addition per element read: memory bounds it
// (131072 rows of 1601 bf16, any alignment, 100 us: 4.2 TB/s over the rows; 131072 of 768 bf16 50 us: 4.0 TB/s; the ids of
// a real text repeat, so the rows come in no order).  The rows come to shared memory in 16-byte pieces,
// a warp copying a row, kChunk * kChunks rows ahead.  The pieces are those between 16-byte boundaries: the outer ones may
// hold bytes of a row's neighbours, which nobody looks at.
template <class O, class T, bool ALIGNED>
__global__ void __launch_bounds__(kGradThreads) k_embed_grad_sums(const GradArgs a, const O* __restrict__ grad_out, T* __restrict__ grad_table)
{
  using S         = Share<O, ALIGNED>;
  constexpr int E = 16 / int(sizeof(O));
  extern __shared__ uint4 s_raw[];
  const int group = blockDim.x, lane = threadIdx.x;
  const int length = 1 << a.block_log2;
  const GroupShared shared(group, length);
  unsigned char* base     = reinterpret_cast<unsigned char*>(s_raw) + threadIdx.y * shared.bytes();
  const uint4* ring       = reinterpret_cast<const uint4*>(base);
  uint64_t* address       = reinterpret_cast<uint64_t*>(base + shared.ring);
  uint32_t* ids           = reinterpret_cast<uint32_t*>(address + shared.tokens);
  // the columns: `width` from `first` on
  gtk::await_kernel();
  const int slab  = (ALIGNED ? group : group - 1) * E;
  const int first = blockIdx.y * slab, width = min(slab, a.dim - first);
  // the tokens of this block and the next, and one at either end of the block in front
  const int64_t block = int64_t(blockIdx.x) * blockDim.y + threadIdx.y;
  const int64_t begin = block << a.block_log2;
  const uint32_t left = begin > 0 && begin < a.n ? __ldcg(&a.tokens[begin - 1].x) : kNoId;
  const uint32_t far_left = begin > length && begin < a.n ? __ldcg(&a.tokens[begin - length - 1].x) : kNoId;
  for (int i = lane; i < shared.tokens; i += group) {
    uint2 token = begin + i < a.n ? __ldcg(a.tokens + begin + i) : make_uint2(kNoId, 0u);
    if (!GTK_IN(token.y, a.n, 210)) token = make_uint2(kNoId, 0u);
    ids[i]     = token.x;
    address[i] = reinterpret_cast<uint64_t>(grad_out + first + int64_t(token.y) * a.out_stride);
  }
  __syncthreads();
  const uint32_t mask = group >= 32 ? 0xFFFFFFFFu : ((1u << group) - 1u) << (threadIdx.y * group & 31);
  int at = 0, stop = 0;
  bool from_left = false, to_right = false;
  if (ids[0] != kNoId) {
    const int end      = ids[length - 1] != kNoId ? length : end_of_tokens(ids, length);
    const uint32_t id0 = ids[0], id1 = ids[end - 1];
    stop = end;
    // the sum that begins further left: skipped, or this block's part of a long one
    from_left = left == id0;
    if (from_left && ids[end] != id0 && far_left != id0) {
      at        = end_of_id(ids, 0, end, id0);
      from_left = false;
    }
    // the sum that reaches over the end: to its end, or up to the boundary when it is a long one
    if (at < end && ids[end] == id1 && !(from_left && id1 == id0)) {
      to_right = ids[2 * length] == id1;
      if (!to_right) stop = end_of_id(ids, end, 2 * length, id1);
    }
  }
  if (at >= stop) return;  // the whole group
  const uint32_t width_bytes = uint32_t(width) * uint32_t(sizeof(O)), slot_bytes = group * 16, chunk_bytes = kChunk * slot_bytes;
  const uint32_t ring_at = uint32_t(__cvta_generic_to_shared(ring));
  uint32_t to = ring_at;  // where the next chunk goes
  // The rows of window places chunk * kChunk ..: each is one warp's to copy, or the group's when that is smaller.
  const int warps = max(1, group >> 5), copier = group > 32 ? lane & 31 : lane, copiers = min(group, 32);
  auto request = [&](int chunk) {
    for (int k = lane >> 5; k < kChunk; k += warps) {
      const int i = chunk * kChunk + k;
      if (i < at || i >= stop || !GTK_IN(i, shared.tokens, 211)) continue;
      const uint64_t row    = address[i];
      const uint32_t shift  = ALIGNED ? 0u : uint32_t(row) & 15u;
      const char* from      = reinterpret_cast<const char*>(row - shift) + copier * 16;
      const uint32_t slot   = to + k * slot_bytes + copier * 16;
      const int pieces      = int((shift + width_bytes + 15u) >> 4) - copier;
#pragma unroll
      for (int p = 0; p < kGradThreads; p += 32)
        if (p < pieces && GTK_IN(to + k * slot_bytes + (copier + p) * 16 - ring_at, kChunk * kChunks * group * 16, 212) && GTK_IN(copier + p, group, 213)) gtk::copy16(slot + p * 16, from + p * 16);
        else break;
    }
    gtk::end_chunk();
    to = to + chunk_bytes == ring_at + kChunks * chunk_bytes ? ring_at : to + chunk_bytes;
  };
  // ALIGNED: the thread's own piece.  Otherwise words, those of a warp next to each other
  const int mine = ALIGNED ? lane : (lane & ~31) * 4 + (lane & 31);
  // the thread's columns from the first of the slab: unit u begins at own + u * kStep units and has valid(u) of them in the row
  const int own  = mine * S::kUnit;
  auto valid     = [&](int u) { return max(0, min(S::kUnit, width - own - u * kStep * S::kUnit)); };
  uint32_t whole = 0, some = 0;
#pragma unroll
  for (int u = 0; u < S::kUnits; ++u) {
    whole |= (valid(u) == S::kUnit ? 1u : 0u) << u;
    some |= (valid(u) > 0 ? 1u : 0u) << u;
  }
  Two sum[S::kCount / 2];
  auto store_part = [&](int which) {
    float* to_part = a.parts + (block * 2 + which) * a.pitch + first + own;
    float x[S::kCount];
#pragma unroll
    for (int j = 0; j < S::kCount / 2; ++j) sum[j].get(x[2 * j], x[2 * j + 1]);
#pragma unroll
    for (int u = 0; u < S::kUnits; ++u)
      if ((some >> u & 1u) && GTK_IN(first + own + u * kStep * S::kUnit + S::kUnit - 1, a.pitch, 214) &&
          GTK_IN(block << a.block_log2, a.n, 215)) {  // whole units: the pitch is a multiple of them
        Pack<float, S::kUnit> p;
#pragma unroll
        for (int j = 0; j < S::kUnit; ++j) p.e[j] = x[u * S::kUnit + j];
        gtk::store_pack<float, S::kUnit>(to_part + u * kStep * S::kUnit, p);
      }
  };
  auto finish = [&](uint32_t id) {
    if (from_left) {
      store_part(0);
      from_left = false;
      return;
    }
    if (!GTK_IN(id, a.vocab, 216)) return;
    T* row           = grad_table + int64_t(id) * a.table_stride + first + own;
    const bool packs = ALIGNED || reinterpret_cast<uintptr_t>(row) % (sizeof(T) * S::kUnit) == 0;
    float x[S::kCount];
    if (whole == (1u << S::kUnits) - 1u && !a.accumulate) {  // nearly all threads, nearly always
      const Two scale(a.scale, a.scale);
#pragma unroll
      for (int j = 0; j < S::kCount / 2; ++j) (sum[j] * scale).get(x[2 * j], x[2 * j + 1]);
#pragma unroll
      for (int u = 0; u < S::kUnits; ++u) {
        T* unit = row + u * kStep * S::kUnit;
        Pack<T, S::kUnit> y;
#pragma unroll
        for (int j = 0; j < S::kUnit; ++j) y.e[j] = gtk::from_float<T>(x[u * S::kUnit + j]);
        if (packs) gtk::store_pack<T, S::kUnit>(unit, y);
        else
#pragma unroll
          for (int j = 0; j < S::kUnit; ++j) unit[j] = y.e[j];
      }
      return;
    }
#pragma unroll
    for (int j = 0; j < S::kCount / 2; ++j) sum[j].get(x[2 * j], x[2 * j + 1]);
#pragma unroll
    for (int u = 0; u < S::kUnits; ++u) store_sum<T, S::kUnit>(row + u * kStep * S::kUnit, valid(u), packs, a.scale, a.accumulate, x + u * S::kUnit);
  };
  int chunk = at / kChunk;
#pragma unroll
  for (int q = 0; q < kChunks - 1; ++q) request(chunk + q);
#pragma unroll
  for (int j = 0; j < S::kCount / 2; ++j) sum[j] = Two(0.f, 0.f);
  uint32_t id = ids[at];
  const uint4* rows = ring;
  for (; chunk * kChunk < stop && GTK_IN(chunk * kChunk + kChunk - 1, shared.tokens, 217); ++chunk) {
    gtk::await_chunks<kChunks - 2>();
    if (group > 32) __syncthreads();
    else __syncwarp(mask);
    request(chunk + kChunks - 1);  // over the chunk in front, which everybody has added
    uint32_t now[kChunk], shift[kChunk];
#pragma unroll
    for (int k = 0; k < kChunk; ++k) {
      now[k]   = ids[chunk * kChunk + k];
      shift[k] = ALIGNED ? 0u : uint32_t(reinterpret_cast<const uint32_t*>(address)[2 * (chunk * kChunk + k)]) & 15u;
    }
    if (now[0] == id && now[kChunk - 1] == id) {  // all of one sum; what lies outside [at, stop) has other ids
#pragma unroll
      for (int k = 0; k < kChunk; ++k) add_row<ALIGNED, O>(rows + k * group, mine, shift[k], sum);
    } else {
#pragma unroll
      for (int k = 0; k < kChunk; ++k) {
        const int i = chunk * kChunk + k;
        if (i < at || i >= stop) continue;
        if (now[k] != id) {
          finish(id);
          id = now[k];
#pragma unroll
          for (int j = 0; j < S::kCount / 2; ++j) sum[j] = Two(0.f, 0.f);
        }
        add_row<ALIGNED, O>(rows + k * group, mine, shift[k], sum);
      }
    }
    rows = rows + kChunk * group == ring + kChunks * kChunk * group ? ring : rows + kChunk * group;
  }
  if (to_right) store_part(1);
  else finish(id);
}

// The parts of long sums (32768 tokens of a text-like distribution: 6.5 us, 131072: 14), 128 columns at a time: a warp per sum; those of more than kJoinAlone parts are all warps' work, each adds
// a run of parts, then the warps' sums are added in order.
constexpr int kJoinThreads = 256, kJoinBlocks = 16, kJoinAlone = 32;
template <class T>
__global__ void __launch_bounds__(kJoinThreads) k_embed_grad_join(const GradArgs a, T* __restrict__ grad_table, bool packs)
{
  constexpr int kWarps = kJoinThreads / 32;
  __shared__ float4 s_sum[kWarps][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c         = blockIdx.y * 128 + lane * 4;
  const int64_t first = int64_t(blockIdx.x) * kJoinBlocks, blocks = (a.n + (int64_t(1) << a.block_log2) - 1) >> a.block_log2;
  gtk::await_kernel();
  LongSum mine{kNoId, 0u};
  if (lane < kJoinBlocks && first + lane < blocks) {
    const uint2 x = __ldcg(reinterpret_cast<const uint2*>(a.long_sums + first + lane));
    mine          = LongSum{x.x, x.y};
  }
  auto add_parts = [&](int at, uint32_t from, uint32_t to) {  // part 0 is the one that begins in the block
    const float* part = a.parts + (first + at) * 2 * a.pitch + c;
    float4 sum        = make_float4(0.f, 0.f, 0.f, 0.f);
    if (c < a.dim)
      for (uint32_t i0 = from; i0 < to; i0 += 8) {
        float4 x[8];
#pragma unroll
        for (uint32_t k = 0; k < 8; ++k) {
          const uint32_t i = min(i0 + k, to - 1);
          if (GTK_IN(first + at + i, blocks, 218)) x[k]             = __ldcg(reinterpret_cast<const float4*>(part + (2 * int64_t(i) + (i == 0 ? 1 : 0)) * a.pitch));
        }
#pragma unroll
        for (uint32_t k = 0; k < 8; ++k)
          if (i0 + k < to) sum.x += x[k].x, sum.y += x[k].y, sum.z += x[k].z, sum.w += x[k].w;
      }
    return sum;
  };
  auto store = [&](uint32_t id, const float4& sum) {
    const float y[4] = {sum.x, sum.y, sum.z, sum.w};
    if (c < a.dim && GTK_IN(id, a.vocab, 219)) store_sum<T, 4>(grad_table + int64_t(id) * a.table_stride + c, a.dim - c, packs, a.scale, a.accumulate, y);
  };
  // the same for every warp
  const uint32_t few = __ballot_sync(0xFFFFFFFFu, mine.parts > 0 && mine.parts <= kJoinAlone), many = __ballot_sync(0xFFFFFFFFu, mine.parts > kJoinAlone);
  int turn = 0;
  for (uint32_t some = few; some; some &= some - 1, ++turn) {
    const int at         = __ffs(some) - 1;
    const uint32_t id    = __shfl_sync(0xFFFFFFFFu, mine.id, at), parts = __shfl_sync(0xFFFFFFFFu, mine.parts, at);
    if (turn % kWarps == warp) store(id, add_parts(at, 0, parts));
  }
  for (uint32_t some = many; some; some &= some - 1) {
    const int at        = __ffs(some) - 1;
    const uint32_t id   = __shfl_sync(0xFFFFFFFFu, mine.id, at), parts = __shfl_sync(0xFFFFFFFFu, mine.parts, at);
    const uint32_t each = (parts + kWarps - 1) / kWarps, from = min(parts, warp * each);
    float4 sum          = add_parts(at, from, min(parts, from + each));
    s_sum[warp][lane]   = sum;
    __syncthreads();
    if (warp == 0) {
#pragma unroll
      for (int w = 1; w < kWarps; ++w) {
        const float4 x = s_sum[w][lane];
        sum.x += x.x, sum.y += x.y, sum.z += x.z, sum.w += x.w;
      }
      store(id, sum);
    }
    __syncthreads();
  }
}

template <class O, class T, bool ALIGNED>
cudaError_t launch_embed_grad(const gtk::HandleView& v, const GradPlan& p, GradArgs a, const int32_t* ids, int64_t n, int64_t vocab,
                              const void* grad_out, void* grad_table, unsigned char* work)
{
  T* table = static_cast<T*>(grad_table);
  const SortArgs s{ids, n, uint32_t(vocab), p.passes, p.digit_bits, p.block_log2, reinterpret_cast<uint2*>(work + p.at_tokens[0]),
                   reinterpret_cast<uint2*>(work + p.at_tokens[1]), a.long_sums};
  cudaError_t e = gtk::launch(k_embed_grad_sort<T>, dim3(kOwners), dim3(kSortThreads), sizeof(SortShared), v.stream, s, table, a.dim,
                              a.table_stride, !a.accumulate);
  if (e != cudaSuccess || n == 0) return e;
  a.tokens = p.passes & 1 ? s.tokens1 : s.tokens0;
  // threads of a group: a power of two from 8 on below a warp when each has 16 bytes of its own; else whole warps, a CTA's at most
  constexpr int E      = 16 / int(sizeof(O));
  const int64_t wanted = (a.dim + E - 1) / E + (ALIGNED ? 0 : 1);
  unsigned group = unsigned(std::min<int64_t>(kGradThreads, (wanted + 31) / 32 * 32));
  while (ALIGNED && group <= 32 && group > 8 && group / 2 >= wanted) group /= 2;
  const unsigned columns = (ALIGNED ? group : group - 1) * E, slabs = unsigned((a.dim + columns - 1) / columns);
  const size_t bytes     = size_t(GroupShared(int(group), 1 << a.block_log2).bytes());
  unsigned groups = group > 32 ? 1 : 128 / group;
  while (groups * group > 32 && groups > 1 && groups * bytes > kSharedGroups) groups /= 2;
  e = gtk::launch_behind(k_embed_grad_sums<O, T, ALIGNED>, dim3(unsigned((p.blocks + groups - 1) / groups), slabs), dim3(group, groups), groups * bytes,
                  v.stream, a, static_cast<const O*>(grad_out), table);
  if (e == cudaSuccess && p.blocks > 2)  // a long sum begins in one block, fills the next and goes on
    e = gtk::launch_behind(k_embed_grad_join<T>, dim3(unsigned((p.blocks + kJoinBlocks - 1) / kJoinBlocks), unsigned((a.dim + 127) / 128)),
                    dim3(kJoinThreads), 0, v.stream, a, table, ALIGNED);
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
        auto f = packs ? launch_embed<decltype(t), decltype(o), 8> : launch_embed<decltype(t), decltype(o), 2>;
        return f(v, d_ids, n_ids, d_table, vocab, dim, table_stride, scale, d_out, out_stride);
      });
    });
  });
}

extern "C" GTK_API int gtk_embed_grad_workspace(gtk_tokenizer* h, int64_t n_ids, int64_t vocab, int64_t dim, size_t* workspace_bytes)
{
  if (!h) return GTK_ERR_INVALID_ARG;
  try {
    std::lock_guard<std::mutex> lock(*gtk::handle_mutex(h));
    gtk::HandleView v;
    gtk::handle_view(h, &v);
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
    const GradArgs a{nullptr, n_ids, uint32_t(vocab), reinterpret_cast<LongSum*>(work + p.at_long), int(dim), p.block_log2, out_stride, table_stride, p.pitch,
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

#ifdef GTK_CHECKED
cudaError_t gtk::embed_check_words(int sum[4], bool reset) { return add_check_words(sum, reset); }
cudaError_t gtk::embed_check_selftest() { return check_selftest(299); }
#endif
