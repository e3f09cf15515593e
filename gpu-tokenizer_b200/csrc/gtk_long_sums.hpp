// gtk_long_sums.hpp -- which sums of the lookup's gradient are cut into parts (gtk_embed.cu).  No CUDA in it but the mark of its
// functions, so that every access it makes can be counted on the CPU.
#pragma once
#include <cstdint>

#ifdef __CUDACC__
#define GTK_OWN_FN __device__ __forceinline__
#else
#define GTK_OWN_FN inline
#endif

namespace gtk {

// Of a block of tokens: the long sum that begins in it, and in how many blocks that has a part; parts == 0: none.
struct alignas(8) LongSum {
  uint32_t id, parts;
};

// The grouped tokens [begin, end) of n are one owner's; those of an id lie next to each other.  put(block, LongSum) for the blocks
// whose last token is the owner's, so that each block is put by one owner: the sum that its last token belongs to is long when it
// reaches over the next boundary too, and begins in the block when no token in front of the block has its id.  Shared by `threads`.
// id_at(place) is asked about the owner's own tokens only; an owner without any has no block, whatever place its share begins at.
template <class IdAt, class Put>
GTK_OWN_FN void each_long_sum(int64_t begin, int64_t end, int64_t n, int block_log2, int thread, int threads, IdAt&& id_at, Put&& put)
{
  if (begin >= end) return;
  for (int64_t block = (begin >> block_log2) + thread; block << block_log2 < end; block += threads) {
    const int64_t after = (block + 1) << block_log2, last = (after < n ? after : n) - 1, third = (block + 2) << block_log2;
    if (last >= end) continue;
    const uint32_t id  = id_at(last);
    const int64_t left = (block << block_log2) - 1;
    LongSum L{id, 0u};
    if (third < end && id_at(third) == id && !(left >= begin && id_at(left) == id)) {
      int64_t from = third, to = end;  // the last place with the id is in [from, to)
      while (to - from > 1) {
        const int64_t mid = (from + to) / 2;
        if (id_at(mid) == id) from = mid;
        else to = mid;
      }
      L.parts = uint32_t((from >> block_log2) - block + 1);
    }
    put(block, L);
  }
}

}  // namespace gtk
