// Rows of bf16, fp16 or fp32 (or bytes) at any address: conversions, 16-byte pieces, and what rows need that do not start on 16-byte
// boundaries (odd widths, strides, views).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ptx.cuh"

namespace b200 {

DEV float to_f32(float v) { return v; }
DEV float to_f32(__half v) { return __half2float(v); }
DEV float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
DEV T from_f32(float v);
template <>
DEV float from_f32<float>(float v) { return v; }
template <>
DEV __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
DEV __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// 16 bytes as elements.
template <class T>
union Vec {
  static constexpr int E = 16 / sizeof(T);
  uint4 raw;
  T v[E];
};

// The bytes of a tensor, first to last element: what may be read when a row's neighbourhood is fetched; and whether that holds for all vectors
// of a row, as it does but for the first and last few bytes of the tensor.
struct Span {
  const uint8_t *lo, *hi;
  bool inner;
};
template <class T>
DEV Span span_of(const void* p, int64_t rows, int64_t stride, int64_t cols, const void* row) {
  const uint8_t *lo = (const uint8_t*)p, *hi = lo + ((rows - 1) * stride + cols) * (int64_t)sizeof(T), *at = (const uint8_t*)row;
  return {lo, hi, at - 15 >= lo && at + cols * (int64_t)sizeof(T) + 32 <= hi};
}

// Bytes sh .. sh + 15 of the 32 bytes a, b. sh is the same for a whole row, so the branches seldom part a warp.
DEV uint4 shift16(const uint4& a, const uint4& b, uint32_t sh) {
  const uint32_t bits = (sh & 3) * 8;
  const auto cut = [bits](uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3, uint32_t w4) {
    return make_uint4(__funnelshift_r(w0, w1, bits), __funnelshift_r(w1, w2, bits), __funnelshift_r(w2, w3, bits), __funnelshift_r(w3, w4, bits));
  };
  if (sh < 8) return sh < 4 ? cut(a.x, a.y, a.z, a.w, b.x) : cut(a.y, a.z, a.w, b.x, b.y);
  return sh < 12 ? cut(a.z, a.w, b.x, b.y, b.z) : cut(a.w, b.x, b.y, b.z, b.w);
}

// 16 bytes from an address that is aligned to an element only: the two aligned vectors around it (fetch, without a branch, so that a thread's
// loads fly together), later shifted into place (take). Bytes of neighbouring rows come along and are the caller's to ignore. Near the ends
// of the tensor, where an aligned vector would reach past it, take reads element by element, zeros outside.
template <class T>
struct Any16 {
  uint4 a, b;
  DEV static bool whole(const uint8_t* p, const Span& s) {
    const uint32_t sh = (uint32_t)(uintptr_t)p & 15u;
    return s.inner || (p - sh >= s.lo && p - sh + (sh ? 32 : 16) <= s.hi);
  }
  DEV void fetch(const uint8_t* p, const Span& s, bool wanted) {
    const uint32_t sh = (uint32_t)(uintptr_t)p & 15u;
    a = b = make_uint4(0u, 0u, 0u, 0u);
    if (wanted && whole(p, s)) {
      a = *reinterpret_cast<const uint4*>(p - sh);           // plain loads: a neighbour's bytes may be written meanwhile (rows in place)
      b = *reinterpret_cast<const uint4*>(p - sh + (sh ? 16 : 0));
    }
  }
  DEV uint4 take(const uint8_t* p, const Span& s) const {
    if (whole(p, s)) {
      return shift16(a, b, (uint32_t)(uintptr_t)p & 15u);
    }
    uint32_t w[4] = {0u, 0u, 0u, 0u};
    for (int i = 0; i < (int)(16 / sizeof(T)); ++i) {
      const uint8_t* q = p + i * sizeof(T);
      uint32_t v = 0;
      if (q >= s.lo && q + sizeof(T) <= s.hi) {
        if constexpr (sizeof(T) == 4) v = *reinterpret_cast<const uint32_t*>(q);
        else if constexpr (sizeof(T) == 2) v = *reinterpret_cast<const unsigned short*>(q);
        else v = *q;
      }
      const int word = i * (int)sizeof(T) / 4;
      v <<= i * sizeof(T) % 4 * 8;
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] |= word == k ? v : 0u;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
// The same interface for addresses that are aligned. kZero: a vector that is not wanted is zero, which makes the load a predicated one among the
// others (unsort 8192 x 8 x 2048 50 us, 71 without); a warp's row is better without (SwiGLU 65536 x 768 43.4 us, 43.8 with), and its kernel looks at
// no vector that was not wanted.
template <class T, bool kZero>
struct Own16 {
  uint4 a;
  DEV void fetch(const uint8_t* p, const Span&, bool wanted) {
    if (kZero) a = make_uint4(0u, 0u, 0u, 0u);
    if (wanted) a = *reinterpret_cast<const uint4*>(p);
  }
  DEV uint4 take(const uint8_t*, const Span&) const { return a; }
};
template <class T, bool kAny, bool kZero>
struct Fetch16Of {
  using type = Own16<T, kZero>;
};
template <class T, bool kZero>
struct Fetch16Of<T, true, kZero> {
  using type = Any16<T>;
};
template <class T, bool kAny, bool kZero = true>
using Fetch16 = typename Fetch16Of<T, kAny, kZero>::type;

}  // namespace b200
