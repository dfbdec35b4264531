// The 8-bit paged K/V cache: codes of one byte, int8 or e4m3, with an FP32 scale per block (page) and KV head.
#pragma once

#include "common.cuh"

namespace xdk {
namespace {

struct Int8Codes {};
struct E4m3Codes {};

// How a value becomes a code and a code a value.  `top`: the largest value a code stands for, so a block's scale is its largest
// |value| * (1 / top).
template <typename C> struct Codec;
template <> struct Codec<Int8Codes> {
  static constexpr float kTop = 127.0f;
  // Round half to even: the sum with 1.5 * 2^23 is a whole number, whose low byte is the code's.  |x| <= kTop.
  __device__ static __forceinline__ uint32_t pack4(const float* x) {
    uint32_t v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __float_as_uint(__fadd_rn(x[i], 12582912.0f));
    return __byte_perm(__byte_perm(v[0], v[1], 0x0040), __byte_perm(v[2], v[3], 0x0040), 0x5410);
  }
  __device__ static __forceinline__ void unpack4(uint32_t v, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = static_cast<float>(static_cast<int8_t>(v >> (8 * i)));
  }
  // A whole number of units, so that the sum of a block's codes does not depend on the order.
  static constexpr float kUnits = 1.0f;
  // Four codes as two FP16 pairs.  Centred: the codes, exactly: 1024 + (code + 128) is a half whose low byte is the code with its sign
  // bit flipped.  Not centred: that byte alone, the subnormal (code + 128) * 2^-24, for two instructions less per pair.
  static constexpr float kOffset = 128.0f, kUnit = 5.9604644775390625e-08f;  // not centred: (code + kOffset) * kUnit
  template <bool CENTRED, int P0, int P1>                                    // the bytes of the pair
  __device__ static __forceinline__ uint32_t half_pair(uint32_t flipped) {
    if constexpr (!CENTRED) return __byte_perm(flipped, 0u, P0 | 0x40 | (P1 << 8) | 0x4000);
    const uint32_t biased = __byte_perm(flipped, 0x64646464u, P0 | 0x40 | (P1 << 8) | 0x4000);
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&biased), __half2half2(__ushort_as_half(0x6480)));  // - 1152
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  template <bool CENTRED> __device__ static __forceinline__ void neighbours(uint32_t v, uint32_t& b01, uint32_t& b23) {
    const uint32_t f = v ^ 0x80808080u;
    b01 = half_pair<CENTRED, 0, 1>(f), b23 = half_pair<CENTRED, 2, 3>(f);
  }
  template <bool CENTRED> __device__ static __forceinline__ void alternate(uint32_t v, uint32_t& b02, uint32_t& b13) {
    const uint32_t f = v ^ 0x80808080u;
    b02 = half_pair<CENTRED, 0, 2>(f), b13 = half_pair<CENTRED, 1, 3>(f);
  }
};
template <> struct Codec<E4m3Codes> {
  static constexpr float kTop = 448.0f;
  __device__ static __forceinline__ uint32_t pack2(float lo, float hi) {  // round to nearest even, saturating
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
  }
  __device__ static __forceinline__ uint32_t pack4(const float* x) { return pack2(x[0], x[1]) | (pack2(x[2], x[3]) << 16); }
  __device__ static __forceinline__ uint32_t half_pair(uint16_t v) {  // exact
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(v));
    return r;
  }
  __device__ static __forceinline__ void unpack4(uint32_t v, float* x) {
    uint32_t h[2];
    neighbours<true>(v, h[0], h[1]);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
  }
  static constexpr float kUnits = 512.0f;  // the smallest code stands for 2^-9
  static constexpr float kOffset = 0.0f, kUnit = 1.0f;  // always centred: the conversion is one instruction per pair
  template <bool CENTRED> __device__ static __forceinline__ void neighbours(uint32_t v, uint32_t& b01, uint32_t& b23) {
    b01 = half_pair(static_cast<uint16_t>(v)), b23 = half_pair(static_cast<uint16_t>(v >> 16));
  }
  template <bool CENTRED> __device__ static __forceinline__ void alternate(uint32_t v, uint32_t& b02, uint32_t& b13) {
    neighbours<CENTRED>(__byte_perm(v, 0u, 0x3120), b02, b13);
  }
};

}  // namespace

inline bool kv8_head_dim(int64_t d) { return d == 64 || d == 128 || d == 256; }
constexpr int64_t kKV8MaxPage = 1024;  // rows of a block
// what the kernels index with 32 bits or put on a grid's y and z
inline int kv8_limits(int64_t tokens, int64_t kv_heads, int64_t max_pages, int64_t page_size) {
  if (tokens > (1LL << 26) || kv_heads > 65535 || max_pages > 2147483647LL || page_size > kKV8MaxPage) return XDK_ERR_LIMIT;
  return XDK_OK;
}

}  // namespace xdk
