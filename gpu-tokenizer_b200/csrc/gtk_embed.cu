// gtk_embed.cu -- embedding lookup with scaling, and its gradient by sorted tokens.
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
// grad_table[v] = scale * sum of grad_out[i] over the i with ids[i] == v.  The ids are sorted (stable, by digits from the
// lowest), which brings the rows of a sum next to each other in order of i.  The sorted positions are cut into units of
// equal length; a row group walks a unit and keeps the running sum in registers.  A sum that begins and ends inside its
// unit is stored right away; what a unit has of a sum that reaches over its ends goes to the workspace, and a last
// kernel joins those parts from left to right.  Every sum is thus formed in an order that the ids alone decide.
constexpr int kSortThreads = 512, kSortWarps = kSortThreads / 32;
constexpr int kMaxDigitBits = 9;  // bins <= threads
constexpr int64_t kMaxDim = int64_t(1) << 20;

struct GradPlan {
  int passes, digit_bits;
  int rounds;         // a sort tile is rounds * kSortThreads ids
  int64_t tiles;
  int64_t unit_rows, units;
  size_t at_pairs[2], at_counts, at_present, at_parts, bytes;
};

int bits_of(int64_t x)
{
  int b = 0;
  while (x >> b) ++b;
  return b;
}

GradPlan grad_plan(int64_t n, int64_t vocab, int64_t dim)
{
  GradPlan p{};
  const int bits = std::max(1, bits_of(vocab));  // keys are 0 .. vocab, the last one stands for ids that take no part
  p.passes       = (bits + kMaxDigitBits - 1) / kMaxDigitBits;
  p.digit_bits   = (bits + p.passes - 1) / p.passes;
  p.rounds       = 4;
  while (p.rounds < 32 && n > int64_t(64) * p.rounds * kSortThreads) p.rounds *= 2;
  p.tiles = (n + int64_t(p.rounds) * kSortThreads - 1) / (int64_t(p.rounds) * kSortThreads);
  // units: long enough that few sums are cut, short enough that their number times the columns fills the GPU
  const int64_t most_units = std::max<int64_t>(64, (int64_t(4096) * 768) / dim);
  p.unit_rows = std::max<int64_t>(8, (n + most_units - 1) / most_units);
  p.units     = (n + p.unit_rows - 1) / p.unit_rows;
  size_t at   = 0;
  auto room   = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) & ~size_t(255);
    return here;
  };
  p.at_pairs[0] = room(size_t(n) * sizeof(uint2));
  p.at_pairs[1] = room(size_t(n) * sizeof(uint2));
  p.at_counts   = room(size_t(p.tiles) * (size_t(1) << p.digit_bits) * 4);
  p.at_present  = room(size_t(vocab));
  p.at_parts    = room(size_t(p.units) * 2 * size_t(dim) * 4);
  p.bytes       = at;
  return p;
}

// what is sorted: the ids themselves in the first pass, {key, place} pairs in later ones
struct SortInput {
  const int32_t* ids;
  const uint2* pairs;
  int64_t n;
  uint32_t vocab;
  __device__ uint2 at(int64_t i) const
  {
    if (pairs) return pairs[i];
    const uint32_t id = uint32_t(ids[i]);
    return make_uint2(min(id, vocab), uint32_t(i));
  }
};

__global__ void __launch_bounds__(kSortThreads)
k_digit_counts(SortInput in, int shift, int bins, int64_t tile, uint32_t* __restrict__ counts, uint8_t* __restrict__ present)
{
  __shared__ uint32_t s_count[1 << kMaxDigitBits];
  for (int b = threadIdx.x; b < bins; b += kSortThreads) s_count[b] = 0;
  if (present)
    for (int64_t v = int64_t(blockIdx.x) * kSortThreads + threadIdx.x; v < in.vocab; v += int64_t(gridDim.x) * kSortThreads) present[v] = 0;
  __syncthreads();
  const int64_t from = blockIdx.x * tile, to = min(in.n, from + tile);
  for (int64_t i = from + threadIdx.x; i < to; i += kSortThreads) atomicAdd(s_count + ((in.at(i).x >> shift) & (bins - 1)), 1u);
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += kSortThreads) counts[blockIdx.x * int64_t(bins) + b] = s_count[b];
}

template <int ROUNDS>
__global__ void __launch_bounds__(kSortThreads)
k_digit_scatter(SortInput in, int shift, int bins, const uint32_t* __restrict__ counts, uint2* __restrict__ out, uint8_t* __restrict__ present)
{
  __shared__ uint32_t s_at[kSortWarps][1 << kMaxDigitBits];
  __shared__ uint32_t s_warp_sum[kSortWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int b = lane; b < bins; b += 32) s_at[warp][b] = 0;
  __syncwarp();
  // places within the warp's own stretch of the tile
  const int64_t first = int64_t(blockIdx.x) * (ROUNDS * kSortThreads) + warp * (ROUNDS * 32);
  uint2 x[ROUNDS];
  uint32_t place[ROUNDS];
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const int64_t i = first + r * 32 + lane;
    x[r]            = i < in.n ? in.at(i) : make_uint2(0u, 0u);
  }
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const bool here      = first + r * 32 + lane < in.n;
    const uint32_t digit = here ? (x[r].x >> shift) & uint32_t(bins - 1) : 0xFFFFFFFFu;
    const uint32_t peers = __match_any_sync(0xFFFFFFFFu, digit);
    const uint32_t before = here ? s_at[warp][digit] : 0u;
    place[r]              = before + __popc(peers & ((1u << lane) - 1u));
    __syncwarp();
    if (here && (peers >> lane) == 1u) s_at[warp][digit] = before + __popc(peers);  // the last of the peers
    __syncwarp();
  }
  // where every bin of this tile begins: bins in front of it, and the same bin in the tiles in front
  uint32_t total = 0, front = 0;
  const int bin  = threadIdx.x;
  if (bin < bins)
    for (int64_t t = 0; t < gridDim.x; ++t) {
      const uint32_t c = counts[t * bins + bin];
      front += t < blockIdx.x ? c : 0u;
      total += c;
    }
  uint32_t upto = total;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const uint32_t o = __shfl_up_sync(0xFFFFFFFFu, upto, d);
    if (lane >= d) upto += o;
  }
  if (lane == 31) s_warp_sum[warp] = upto;
  __syncthreads();
  if (bin < bins) {
    uint32_t at = upto - total + front;
    for (int w = 0; w < warp; ++w) at += s_warp_sum[w];
    for (int w = 0; w < kSortWarps; ++w) {
      const uint32_t c = s_at[w][bin];
      s_at[w][bin]     = at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r)
    if (first + r * 32 + lane < in.n) {
      out[s_at[warp][(x[r].x >> shift) & uint32_t(bins - 1)] + place[r]] = x[r];
      if (present && x[r].x < in.vocab) present[x[r].x] = 1;  // whoever writes it writes the same
    }
}

// V columns of a row; valid < V at the end of a row that V does not divide
template <class T, int V>
__device__ __forceinline__ void load_row(const T* p, int valid, float (&x)[V])
{
  if (valid == V) {
    const Pack<T, V> v = gtk::load_pack<T, V>(p);
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = gtk::to_float(v.e[j]);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = j < valid ? gtk::to_float(p[j]) : 0.f;
  }
}

template <class T, int V>
__device__ __forceinline__ void store_row(T* p, int valid, const float (&x)[V])
{
  if (valid == V) {
    Pack<T, V> v;
#pragma unroll
    for (int j = 0; j < V; ++j) v.e[j] = gtk::from_float<T>(x[j]);
    gtk::store_pack<T, V>(p, v);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j < valid) p[j] = gtk::from_float<T>(x[j]);
  }
}

// a finished sum to its row
template <class T, int V>
__device__ __forceinline__ void store_sum(T* row, int valid, float scale, bool accumulate, const float (&sum)[V])
{
  float y[V];
  if (accumulate) {
    load_row<T, V>(row, valid, y);
#pragma unroll
    for (int j = 0; j < V; ++j) y[j] = fmaf(sum[j], scale, y[j]);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) y[j] = sum[j] * scale;
  }
  store_row<T, V>(row, valid, y);
}

struct GradArgs {
  const uint2* pairs;  // sorted {key, place}
  int64_t n;
  uint32_t vocab;
  int dim;
  int64_t unit_rows, units;
  int64_t out_stride, table_stride;
  float scale;
  bool accumulate;
  float* parts;  // [units][2][dim]: of the sum that has begun in an earlier unit, of the one that goes on in the next
};

constexpr int kGradThreads = 256, kRowsInFlight = 8;

template <class O, class T, int V>
__global__ void __launch_bounds__(kGradThreads) k_embed_grad_units(const GradArgs a, const O* __restrict__ grad_out, T* __restrict__ grad_table)
{
  const int64_t unit = int64_t(blockIdx.x) * blockDim.y + threadIdx.y;
  const int c        = (blockIdx.y * blockDim.x + threadIdx.x) * V;
  if (unit >= a.units || c >= a.dim) return;
  const int valid     = min(V, a.dim - c);
  const int64_t begin = unit * a.unit_rows, end = min(a.n, begin + a.unit_rows);
  uint32_t key = __ldg(&a.pairs[begin].x);
  bool from_before = begin > 0 && __ldg(&a.pairs[begin - 1].x) == key;
  float sum[V] = {};
  for (int64_t at = begin; at < end; at += kRowsInFlight) {
    uint2 p[kRowsInFlight];
    float x[kRowsInFlight][V];
#pragma unroll
    for (int k = 0; k < kRowsInFlight; ++k) p[k] = at + k < end ? __ldg(a.pairs + at + k) : make_uint2(a.vocab, 0u);
#pragma unroll
    for (int k = 0; k < kRowsInFlight; ++k)
      if (p[k].x < a.vocab) load_row<O, V>(grad_out + int64_t(p[k].y) * a.out_stride + c, valid, x[k]);
#pragma unroll
    for (int k = 0; k < kRowsInFlight; ++k) {
      if (at + k >= end) break;
      if (p[k].x != key) {
        if (from_before) store_row<float, V>(a.parts + unit * 2 * a.dim + c, valid, sum);
        else store_sum<T, V>(grad_table + int64_t(key) * a.table_stride + c, valid, a.scale, a.accumulate, sum);
        from_before = false;
        key         = p[k].x;
#pragma unroll
        for (int j = 0; j < V; ++j) sum[j] = 0.f;
      }
      if (key >= a.vocab) return;  // sorted behind every sum
#pragma unroll
      for (int j = 0; j < V; ++j) sum[j] += x[k][j];
    }
  }
  const bool goes_on = end < a.n && __ldg(&a.pairs[end].x) == key;
  if (from_before) store_row<float, V>(a.parts + unit * 2 * a.dim + c, valid, sum);
  else if (goes_on) store_row<float, V>(a.parts + (unit * 2 + 1) * a.dim + c, valid, sum);
  else store_sum<T, V>(grad_table + int64_t(key) * a.table_stride + c, valid, a.scale, a.accumulate, sum);
}

// A block per unit in which a sum begins that goes on in the next.
template <class T>
__global__ void __launch_bounds__(kGradThreads) k_embed_grad_join(const GradArgs a, T* __restrict__ grad_table)
{
  __shared__ int64_t s_units;
  const int64_t unit  = blockIdx.x;
  const int64_t begin = unit * a.unit_rows, end = min(a.n, begin + a.unit_rows);
  if (end >= a.n) return;
  const uint32_t key = a.pairs[end - 1].x;
  if (key >= a.vocab || a.pairs[end].x != key) return;
  if (a.pairs[begin].x == key && begin > 0 && a.pairs[begin - 1].x == key) return;  // begins further left
  if (threadIdx.x < 32) {  // units behind this one that begin with the same key
    int64_t more = 0;
    for (;;) {
      const int64_t u     = unit + 1 + more + threadIdx.x;
      const uint32_t same = __ballot_sync(0xFFFFFFFFu, u < a.units && a.pairs[u * a.unit_rows].x == key);
      if (same != 0xFFFFFFFFu) {
        more += __ffs(~same) - 1;
        break;
      }
      more += 32;
    }
    if (threadIdx.x == 0) s_units = more;
  }
  __syncthreads();
  const int64_t more = s_units;
  for (int c = threadIdx.x; c < a.dim; c += kGradThreads) {
    float sum[1] = {a.parts[(unit * 2 + 1) * a.dim + c]};
#pragma unroll 8
    for (int64_t u = 1; u <= more; ++u) sum[0] += a.parts[(unit + u) * 2 * a.dim + c];
    store_sum<T, 1>(grad_table + int64_t(key) * a.table_stride + c, 1, a.scale, a.accumulate, sum);
  }
}

// zeros for the rows that no id points to
template <class T, int V>
__global__ void __launch_bounds__(kGradThreads)
k_embed_grad_fill(const uint8_t* __restrict__ present, int64_t vocab, int dim, T* __restrict__ grad_table, int64_t table_stride)
{
  const float zero[V] = {};
  for (int64_t v = int64_t(blockIdx.x) * blockDim.y + threadIdx.y; v < vocab; v += int64_t(gridDim.x) * blockDim.y) {
    if (present && present[v]) continue;
    for (int c = threadIdx.x * V; c < dim; c += blockDim.x * V) store_row<T, V>(grad_table + v * table_stride + c, min(V, dim - c), zero);
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
  uint8_t* present = a.accumulate ? nullptr : work + p.at_present;
  T* table         = static_cast<T*>(grad_table);
  const unsigned tx = column_threads(a.dim, V), ty = kGradThreads / tx;
  cudaError_t e     = cudaSuccess;
  if (a.n > 0) {
    SortInput in{ids, nullptr, a.n, a.vocab};
    uint32_t* counts   = reinterpret_cast<uint32_t*>(work + p.at_counts);
    const int bins     = 1 << p.digit_bits;
    const int64_t tile = int64_t(p.rounds) * kSortThreads;
    uint2* sorted      = nullptr;
    for (int pass = 0; pass < p.passes && e == cudaSuccess; ++pass) {
      const int shift = pass * p.digit_bits;
      sorted          = reinterpret_cast<uint2*>(work + p.at_pairs[pass & 1]);
      e = gtk::launch(k_digit_counts, dim3(unsigned(p.tiles)), dim3(kSortThreads), 0, v.stream, in, shift, bins, tile, counts,
                      pass == 0 ? present : nullptr);
      auto scatter = p.rounds == 4 ? k_digit_scatter<4> : p.rounds == 8 ? k_digit_scatter<8> : p.rounds == 16 ? k_digit_scatter<16>
                                                                                                          : k_digit_scatter<32>;
      if (e == cudaSuccess)
        e = gtk::launch(scatter, dim3(unsigned(p.tiles)), dim3(kSortThreads), 0, v.stream, in, shift, bins, counts, sorted,
                        pass == 0 ? present : nullptr);
      in.pairs = sorted;
    }
    a.pairs = sorted;
    if (e == cudaSuccess)
      e = gtk::launch(k_embed_grad_units<O, T, V>, dim3(unsigned((p.units + ty - 1) / ty), unsigned((a.dim + tx * V - 1) / (tx * V))),
                      dim3(tx, ty), 0, v.stream, a, static_cast<const O*>(grad_out), table);
    if (e == cudaSuccess)
      e = gtk::launch(k_embed_grad_join<T>, dim3(unsigned(p.units)), dim3(kGradThreads), 0, v.stream, a, table);
  }
  if (e == cudaSuccess && !a.accumulate) {
    const int64_t blocks = std::min<int64_t>((a.vocab + ty - 1) / ty, int64_t(v.sm_count) * 8);
    e = gtk::launch(k_embed_grad_fill<T, V>, dim3(unsigned(blocks)), dim3(tx, ty), 0, v.stream, a.n > 0 ? present : nullptr,
                    int64_t(a.vocab), a.dim, table, a.table_stride);
  }
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
    const GradArgs a{nullptr, n_ids, uint32_t(vocab), int(dim), p.unit_rows, p.units, out_stride, table_stride, scale, accumulate != 0,
                     reinterpret_cast<float*>(static_cast<unsigned char*>(d_workspace) + p.at_parts)};
    const bool packs = gtk::rows_aligned(d_grad_out, out_stride, out_type, 8) && gtk::rows_aligned(d_grad_table, table_stride, table_type, 8) &&
                       dim % 4 == 0;  // the workspace's rows are dim 32-bit floats
    return gtk::with_type(out_type, [&](auto o) {
      return gtk::with_type(table_type, [&](auto t) {
        auto f = packs ? launch_embed_grad<decltype(o), decltype(t), 8> : launch_embed_grad<decltype(o), decltype(t), 1>;
        return f(v, p, a, d_ids, d_grad_out, d_grad_table, static_cast<unsigned char*>(d_workspace));
      });
    });
  });
}
