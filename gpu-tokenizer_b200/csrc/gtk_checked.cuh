// gtk_checked.cuh -- the index checks of the checked build (-DGTK_CHECKED).
//
// Every index into shared memory, the lane scratch, the staging buffers, the work buffers and the per-chunk / per-unit arrays that is
// computed from data is compared with its limit before it is used.  A violation is recorded (first failing check, offending
// value, limit, number of violations) and the access is skipped, so a wrong index shows up as a report, never as a fault; read the
// record with gtk_debug_check_words.  Without the flag the checks compile to nothing.  Each source file has a record of its
// own; the checks' numbers are below 100 in gtk_kernels.cu, 200 to 299 in gtk_embed.cu, 300 to 399 in gtk_logprobs.cu,
// 400 to 499 in gtk_paged.cu, 500 to 599 in gtk_sample.cu.
#pragma once
#ifdef GTK_CHECKED
#include <cuda_runtime.h>

namespace {
__device__ int g_check_words[4];
__device__ __noinline__ bool check_failed(int id, long long value, long long limit)
{
  if (atomicAdd(&g_check_words[3], 1) == 0) {
    g_check_words[0] = id;
    g_check_words[1] = int(value);
    g_check_words[2] = int(limit);
  }
  return false;
}

#define GTK_IN(value, limit, id) \
  ((static_cast<unsigned long long>(value) < static_cast<unsigned long long>(limit)) || check_failed((id), (long long)(value), (long long)(limit)))

// a check that must fail
__global__ void k_check_selftest(int* sink, int id)
{
  const int bad = 5 + int(threadIdx.x);
  if (GTK_IN(bad, 4, id)) sink[bad] = 1;
}
cudaError_t check_selftest(int id)
{
  int* sink     = nullptr;
  cudaError_t e = cudaMalloc(&sink, 64);
  if (e != cudaSuccess) return e;
  k_check_selftest<<<1, 1>>>(sink, id);
  e = cudaDeviceSynchronize();
  cudaFree(sink);
  return e;
}

// adds this file's record to `sum`: the words of the first failure anywhere, and the number of all
cudaError_t add_check_words(int sum[4], bool reset)
{
  int mine[4]         = {0, 0, 0, 0};
  const cudaError_t e = cudaMemcpyFromSymbol(mine, g_check_words, sizeof(mine));
  if (e != cudaSuccess) return e;
  if (sum[3] == 0)
    for (int i = 0; i < 3; ++i) sum[i] = mine[i];
  sum[3] += mine[3];
  const int none[4] = {0, 0, 0, 0};
  return reset ? cudaMemcpyToSymbol(g_check_words, none, sizeof(none)) : cudaSuccess;
}
}  // namespace

namespace gtk {
cudaError_t embed_check_words(int sum[4], bool reset);
cudaError_t embed_check_selftest();
cudaError_t logprobs_check_words(int sum[4], bool reset);
cudaError_t logprobs_check_selftest();
cudaError_t paged_check_words(int sum[4], bool reset);
cudaError_t paged_check_selftest();
cudaError_t sample_check_words(int sum[4], bool reset);
cudaError_t sample_check_selftest();
}  // namespace gtk
#else
#define GTK_IN(value, limit, id) true
#endif
