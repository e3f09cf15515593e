// gtk_logits.cuh -- what the operators on rows of logits share (gtk_logprobs.cu, gtk_sample.cu): packs of 16 bytes of a row, the
// exponential, and logits as whole numbers in their order.
#pragma once
#include "gtk_rows.cuh"

namespace gtk {

constexpr float kLog2e = 1.44269504088896341f;

// exp2 of a number <= 0 (or NaN)
__device__ __forceinline__ float pow2(float y)
{
  float p;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p) : "f"(y));
  return p;
}

// 16 bytes of a row: its elements as pairs of 32-bit floats, and their maxima (NaN only where all are).
template <class T>
struct Pack16;
template <>
struct Pack16<float> {
  static constexpr int kElems = 4;
  static constexpr uint32_t kMinusInf = 0xFF800000u;
  static constexpr int kLowestBit     = 0;  // below it all numbers of the type agree, written as 32-bit floats
  static __device__ __forceinline__ void pairs(const uint4& r, Two (&x)[2])
  {
    x[0] = Two(__uint_as_float(r.x), __uint_as_float(r.y));
    x[1] = Two(__uint_as_float(r.z), __uint_as_float(r.w));
  }
  // maxima: one of the whole pack
  using Max = float;
  static constexpr int kHalves = 1;
  static __device__ __forceinline__ Max lowest() { return -INFINITY; }
  static __device__ __forceinline__ Max highest(const uint4& r)
  {
    return fmaxf(fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)), fmaxf(__uint_as_float(r.z), __uint_as_float(r.w)));
  }
  static __device__ __forceinline__ Max higher(Max a, Max b) { return fmaxf(a, b); }
  static __device__ __forceinline__ float of(Max m, int) { return m; }
};
template <class T, class T2>
struct Pack16Half {
  static constexpr int kElems = 8;
  static __device__ __forceinline__ T2 as(const uint32_t& w) { return *reinterpret_cast<const T2*>(&w); }
  static __device__ __forceinline__ float2 both(T2 w);
  static __device__ __forceinline__ void pairs(const uint4& r, Two (&x)[4])
  {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = both(as(w[i]));
      x[i]           = Two(f.x, f.y);
    }
  }
  // maxima: one of the even elements, one of the odd ones
  using Max = T2;
  static constexpr int kHalves = 2;
  static __device__ __forceinline__ Max highest(const uint4& r) { return __hmax2(__hmax2(as(r.x), as(r.y)), __hmax2(as(r.z), as(r.w))); }
  static __device__ __forceinline__ Max higher(Max a, Max b) { return __hmax2(a, b); }
  static __device__ __forceinline__ float of(Max m, int half)
  {
    const float2 f = both(m);
    return half ? f.y : f.x;
  }
};
template <>
__device__ __forceinline__ float2 Pack16Half<__nv_bfloat16, __nv_bfloat162>::both(__nv_bfloat162 w) { return __bfloat1622float2(w); }
template <>
__device__ __forceinline__ float2 Pack16Half<__half, __half2>::both(__half2 w) { return __half22float2(w); }
template <>
struct Pack16<__nv_bfloat16> : Pack16Half<__nv_bfloat16, __nv_bfloat162> {
  static __device__ __forceinline__ Max lowest() { return __float2bfloat162_rn(-INFINITY); }
  static constexpr uint32_t kMinusInf = 0xFF80FF80u;
  static constexpr int kLowestBit     = 16;
};
template <>
struct Pack16<__half> : Pack16Half<__half, __half2> {
  static __device__ __forceinline__ Max lowest() { return __float2half2_rn(-INFINITY); }
  static constexpr uint32_t kMinusInf = 0xFC00FC00u;
  static constexpr int kLowestBit     = 13;
};

// Logits as whole numbers in their order (-0 as 0); 0 stands for nothing, which -inf is here.
__device__ __forceinline__ uint32_t value_key(float x)
{
  const uint32_t b = __float_as_uint(x + 0.f);
  return x > -INFINITY ? (b & 0x80000000u ? ~b : b | 0x80000000u) : 0u;
}
// with the column behind it, the lower one the higher number among equals
__device__ __forceinline__ uint64_t rank_key(float x, uint32_t column)
{
  const uint32_t v = value_key(x);
  return v ? uint64_t(v) << 32 | ~column : 0u;
}
__device__ __forceinline__ uint32_t key_column(uint64_t key) { return ~uint32_t(key); }
__device__ __forceinline__ float key_value(uint64_t key)
{
  const uint32_t b = uint32_t(key >> 32);
  return __uint_as_float(b & 0x80000000u ? b & 0x7FFFFFFFu : ~b);
}

}  // namespace gtk
