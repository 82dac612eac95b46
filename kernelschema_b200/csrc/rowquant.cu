// Rows quantised to 8 bits with one fp32 scale per row, in the launch that produces them:
//   RMS norm   h = x + r,  y = h * rsqrt(mean(h^2) + eps) * w
//   SwiGLU     x = [g | u],  y = g * sigmoid(g) * u
//   both       amax = max|y|,  scale = amax / Q,  q = round_to_nearest_even(y * (Q / amax)),  Q = 127 (int8) or 448 (e4m3)
//
// Both are bound by HBM: every input element is read once, every output element written once, and a row stays in registers between its
// reductions. h, the sum of squares, y and amax are fp32; the residual stream h, the normed row y and the code q are each rounded once,
// from the fp32 value (the norm sees h before it is rounded to the stream's type).
// A row holds no scale when it has no finite amax: a NaN or an infinity in it, or a sum of squares beyond fp32, makes the scale NaN and
// the codes zero, so that the row is NaN wherever it is multiplied out. A row whose amax is below 2^-116 counts as zero (scale 0,
// codes 0): Q / amax stays finite for every other one, and scale stays a normal number.
#include <cuda_fp16.h>

#include "kernels.cuh"
#include "ptx.cuh"

namespace b200 {

namespace {

constexpr uint32_t kInfBits = 0x7F800000u;
constexpr float kLeastAmax = 0x1p-116f;

template <class T>
struct Row {                                             // 16-byte vectors of a row's type
  static constexpr int E = 16 / sizeof(T);
};

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

template <class T>
union Vec {
  uint4 raw;
  T v[Row<T>::E];
};

// Weight of the norm: the rows' own type or fp32.
template <class T>
DEV float weight_at(const void* w, bool w_f32, int64_t i) {
  return w_f32 ? __ldg(reinterpret_cast<const float*>(w) + i) : to_f32(reinterpret_cast<const T*>(w)[i]);
}

DEV uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// Reductions over the threads of a row: a warp, or the whole block (32 words of shared memory, one per warp).
template <bool kWarp>
DEV float row_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  if (kWarp) return v;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = (int)(blockDim.x + 31) >> 5;
  if (lane == 0) red[warp] = v;
  __syncthreads();
  v = lane < warps ? red[lane] : 0.f;
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}
template <bool kWarp>
DEV uint32_t row_max(uint32_t v, uint32_t* red) {
  v = __reduce_max_sync(0xFFFFFFFFu, v);
  if (kWarp) return v;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = (int)(blockDim.x + 31) >> 5;
  if (lane == 0) red[warp] = v;
  __syncthreads();
  return __reduce_max_sync(0xFFFFFFFFu, lane < warps ? red[lane] : 0u);
}

// amax of a row (as bits: infinities and NaN compare above every finite value) -> factor of the codes and the row's scale
DEV float code_factor(uint32_t amax_bits, int q_type, float& scale) {
  const float top = q_type == kInt8 ? 127.f : 448.f, amax = __uint_as_float(amax_bits);
  if (amax_bits >= kInfBits) {
    scale = __uint_as_float(0x7FC00000u);
    return 0.f;
  }
  if (amax < kLeastAmax) {
    scale = 0.f;
    return 0.f;
  }
  scale = amax / top;
  return top / amax;
}

// Four codes in a word. With a factor of zero the codes are zero whatever y holds.
DEV uint32_t codes4(float a, float b, float c, float d, float f, int q_type) {
  if (f == 0.f) return 0u;
  a *= f, b *= f, c *= f, d *= f;
  if (q_type == kInt8) {
    const uint32_t lo = __byte_perm(__float2int_rn(a), __float2int_rn(b), 0x0040), hi = __byte_perm(__float2int_rn(c), __float2int_rn(d), 0x0040);
    return __byte_perm(lo, hi, 0x5410);
  }
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return (uint32_t)lo | ((uint32_t)hi << 16);
}

template <int E>
DEV void store_codes(uint8_t* dst, const float* y, float f, int q_type) {
  const uint32_t lo = codes4(y[0], y[1], y[2], y[3], f, q_type);
  if constexpr (E == 8)
    *reinterpret_cast<uint2*>(dst) = make_uint2(lo, codes4(y[4], y[5], y[6], y[7], f, q_type));
  else
    *reinterpret_cast<uint32_t*>(dst) = lo;
}

// Most threads of a block: 64 registers a thread hold up to 16 values of a row and what is loaded for them, 128 the rest.
template <class T, int VPT, bool kWarp>
constexpr int row_threads() { return kWarp ? 128 : VPT * Row<T>::E <= 16 ? 1024 : 512; }

// ----------------------------------------------------------------------------- norm
// A row belongs to one warp (kWarp, up to 128 vectors) or to a block. Vectors v0, v0 + threads, ... of the row are a thread's; it reads
// and writes the same places of x, residual, hidden and normed, so hidden may be x or residual itself.
template <class T, int VPT, bool kWarp>
__global__ void __launch_bounds__(row_threads<T, VPT, kWarp>()) k_rmsnorm_quantize(const RmsNormParams p) {
  constexpr int E = Row<T>::E;
  __shared__ float red_sum[32];
  __shared__ uint32_t red_max[32];
  const int lane = threadIdx.x & 31;
  const int64_t row = kWarp ? (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : (int64_t)blockIdx.x;
  const int v0 = kWarp ? lane : (int)threadIdx.x, step = kWarp ? 32 : (int)blockDim.x;
  const int nvec = p.cols / E;
  pdl_trigger();
  pdl_wait();
  if (kWarp && row >= p.rows) return;
  const T* x = (const T*)p.x + row * p.x_stride;
  const T* r = p.residual ? (const T*)p.residual + row * p.residual_stride : nullptr;
  Vec<T> xv[VPT], rv[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = v0 + i * step;
    xv[i].raw = make_uint4(0u, 0u, 0u, 0u);
    if (v < nvec) xv[i].raw = reinterpret_cast<const uint4*>(x)[v];
  }
  if (r) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = v0 + i * step;
      rv[i].raw = make_uint4(0u, 0u, 0u, 0u);
      if (v < nvec) rv[i].raw = reinterpret_cast<const uint4*>(r)[v];
    }
  }
  float y[VPT][E];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int j = 0; j < E; ++j) {
      y[i][j] = to_f32(xv[i].v[j]);
      if (r) y[i][j] += to_f32(rv[i].v[j]);
      ss = fmaf(y[i][j], y[i][j], ss);
    }
  if (p.hidden) {
    T* h = (T*)p.hidden + row * p.hidden_stride;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = v0 + i * step;
      Vec<T> o;
#pragma unroll
      for (int j = 0; j < E; ++j) o.v[j] = from_f32<T>(y[i][j]);
      if (v < nvec) reinterpret_cast<uint4*>(h)[v] = o.raw;
    }
  }
  ss = row_sum<kWarp>(ss, red_sum);
  // a sum that is no number leaves no finite y either (infinity * 0 would pass for one)
  const float rstd = abs_bits(ss) < kInfBits ? rsqrtf(ss / (float)p.cols + p.eps) : __uint_as_float(0x7FC00000u);
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = v0 + i * step;
    if (v >= nvec) continue;
    if (p.weight_f32) {
      const float4* w = reinterpret_cast<const float4*>(p.weight) + (int64_t)v * (E / 4);
#pragma unroll
      for (int j = 0; j < E / 4; ++j) {
        const float4 c = __ldg(w + j);
        y[i][4 * j] *= rstd * c.x;
        y[i][4 * j + 1] *= rstd * c.y;
        y[i][4 * j + 2] *= rstd * c.z;
        y[i][4 * j + 3] *= rstd * c.w;
      }
    } else {
      Vec<T> c;
      c.raw = __ldg(reinterpret_cast<const uint4*>(p.weight) + v);
#pragma unroll
      for (int j = 0; j < E; ++j) y[i][j] *= rstd * to_f32(c.v[j]);
    }
#pragma unroll
    for (int j = 0; j < E; ++j) amax = max(amax, abs_bits(y[i][j]));
  }
  amax = row_max<kWarp>(amax, red_max);
  float scale;
  const float f = code_factor(amax, p.q_type, scale);
  if (v0 == 0) p.scale[row] = scale;
  uint8_t* q = p.q + row * p.q_stride;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = v0 + i * step;
    if (v < nvec) store_codes<E>(q + (int64_t)v * E, y[i], f, p.q_type);
  }
  if (p.normed) {
    T* n = (T*)p.normed + row * p.normed_stride;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = v0 + i * step;
      Vec<T> o;
#pragma unroll
      for (int j = 0; j < E; ++j) o.v[j] = from_f32<T>(y[i][j]);
      if (v < nvec) reinterpret_cast<uint4*>(n)[v] = o.raw;
    }
  }
}

// Rows that vectors do not fit (odd widths, strides or addresses): the same, element by element.
template <class T, int NPT>
__global__ void __launch_bounds__(1024) k_rmsnorm_quantize_odd(const RmsNormParams p) {
  __shared__ float red_sum[32];
  __shared__ uint32_t red_max[32];
  const int64_t row = blockIdx.x;
  pdl_trigger();
  pdl_wait();
  const T* x = (const T*)p.x + row * p.x_stride;
  const T* r = p.residual ? (const T*)p.residual + row * p.residual_stride : nullptr;
  float y[NPT];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < NPT; ++i) {
    const int c = (int)threadIdx.x + i * (int)blockDim.x;
    y[i] = 0.f;
    if (c < p.cols) {
      y[i] = to_f32(x[c]);
      if (r) y[i] += to_f32(r[c]);
    }
    ss = fmaf(y[i], y[i], ss);
  }
  if (p.hidden) {
    T* h = (T*)p.hidden + row * p.hidden_stride;
#pragma unroll
    for (int i = 0; i < NPT; ++i) {
      const int c = (int)threadIdx.x + i * (int)blockDim.x;
      if (c < p.cols) h[c] = from_f32<T>(y[i]);
    }
  }
  ss = row_sum<false>(ss, red_sum);
  const float rstd = abs_bits(ss) < kInfBits ? rsqrtf(ss / (float)p.cols + p.eps) : __uint_as_float(0x7FC00000u);
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < NPT; ++i) {
    const int c = (int)threadIdx.x + i * (int)blockDim.x;
    if (c < p.cols) {
      y[i] *= rstd * weight_at<T>(p.weight, p.weight_f32, c);
      amax = max(amax, abs_bits(y[i]));
    }
  }
  amax = row_max<false>(amax, red_max);
  float scale;
  const float f = code_factor(amax, p.q_type, scale);
  if (threadIdx.x == 0) p.scale[row] = scale;
  uint8_t* q = p.q + row * p.q_stride;
  T* n = p.normed ? (T*)p.normed + row * p.normed_stride : nullptr;
#pragma unroll
  for (int i = 0; i < NPT; ++i) {
    const int c = (int)threadIdx.x + i * (int)blockDim.x;
    if (c < p.cols) {
      q[c] = (uint8_t)codes4(y[i], 0.f, 0.f, 0.f, f, p.q_type);
      if (n) n[c] = from_f32<T>(y[i]);
    }
  }
}

// ----------------------------------------------------------------------------- SwiGLU
DEV float silu_mul(float g, float u) { return __fdividef(g, 1.f + __expf(-g)) * u; }

template <class T, int VPT, bool kWarp>
__global__ void __launch_bounds__(row_threads<T, VPT, kWarp>()) k_swiglu_quantize(const SwigluParams p) {
  constexpr int E = Row<T>::E;
  __shared__ uint32_t red_max[32];
  const int lane = threadIdx.x & 31;
  const int64_t row = kWarp ? (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : (int64_t)blockIdx.x;
  const int v0 = kWarp ? lane : (int)threadIdx.x, step = kWarp ? 32 : (int)blockDim.x;
  const int nvec = p.cols / E;
  pdl_trigger();
  pdl_wait();
  if (kWarp && row >= p.rows) return;
  const uint4* g = reinterpret_cast<const uint4*>((const T*)p.x + row * p.x_stride);
  const uint4* u = reinterpret_cast<const uint4*>((const T*)p.x + row * p.x_stride + p.cols);
  Vec<T> gv[VPT], uv[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = v0 + i * step;
    gv[i].raw = uv[i].raw = make_uint4(0u, 0u, 0u, 0u);
    if (v < nvec) {
      gv[i].raw = g[v];
      uv[i].raw = u[v];
    }
  }
  float y[VPT][E];
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int j = 0; j < E; ++j) {
      y[i][j] = silu_mul(to_f32(gv[i].v[j]), to_f32(uv[i].v[j]));
      amax = max(amax, abs_bits(y[i][j]));
    }
  amax = row_max<kWarp>(amax, red_max);
  float scale;
  const float f = code_factor(amax, p.q_type, scale);
  if (v0 == 0) p.scale[row] = scale;
  uint8_t* q = p.q + row * p.q_stride;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = v0 + i * step;
    if (v < nvec) store_codes<E>(q + (int64_t)v * E, y[i], f, p.q_type);
  }
}

template <class T, int NPT>
__global__ void __launch_bounds__(1024) k_swiglu_quantize_odd(const SwigluParams p) {
  __shared__ uint32_t red_max[32];
  const int64_t row = blockIdx.x;
  pdl_trigger();
  pdl_wait();
  const T* g = (const T*)p.x + row * p.x_stride;
  const T* u = g + p.cols;
  float y[NPT];
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < NPT; ++i) {
    const int c = (int)threadIdx.x + i * (int)blockDim.x;
    y[i] = c < p.cols ? silu_mul(to_f32(g[c]), to_f32(u[c])) : 0.f;
    amax = max(amax, abs_bits(y[i]));
  }
  amax = row_max<false>(amax, red_max);
  float scale;
  const float f = code_factor(amax, p.q_type, scale);
  if (threadIdx.x == 0) p.scale[row] = scale;
  uint8_t* q = p.q + row * p.q_stride;
#pragma unroll
  for (int i = 0; i < NPT; ++i) {
    const int c = (int)threadIdx.x + i * (int)blockDim.x;
    if (c < p.cols) q[c] = (uint8_t)codes4(y[i], 0.f, 0.f, 0.f, f, p.q_type);
  }
}

// ----------------------------------------------------------------------------- launches
int round_up32(int v) { return (v + 31) / 32 * 32; }

template <class T>
struct NormKernels {
  using P = RmsNormParams;
  template <int VPT, bool kWarp>
  static constexpr auto vec() { return k_rmsnorm_quantize<T, VPT, kWarp>; }
  template <int NPT>
  static constexpr auto odd() { return k_rmsnorm_quantize_odd<T, NPT>; }
};
template <class T>
struct SwigluKernels {
  using P = SwigluParams;
  template <int VPT, bool kWarp>
  static constexpr auto vec() { return k_swiglu_quantize<T, VPT, kWarp>; }
  template <int NPT>
  static constexpr auto odd() { return k_swiglu_quantize_odd<T, NPT>; }
};

// Up to 128 vectors a row is a warp's: no barrier, four rows to a block. Above that a block's, of as many vectors per thread as leave
// every SM several blocks; with fewer rows than that, one vector per thread and more threads, because a row's own latency is the time.
template <class K, int E>
int launch_rows(const typename K::P& p, bool vectors, cudaStream_t st) {
  if (!vectors) {
    const int npt = p.cols <= 8192 ? 8 : 32, threads = round_up32((p.cols + npt - 1) / npt);
    const dim3 grid((unsigned)p.rows), block((unsigned)threads);
    return (int)(npt == 8 ? launch_chain(K::template odd<8>(), grid, block, 0, st, p) : launch_chain(K::template odd<32>(), grid, block, 0, st, p));
  }
  const int nvec = p.cols / E;
  if (nvec <= 128) {
    const dim3 grid((unsigned)((p.rows + 3) / 4)), block(128);
    if (nvec <= 32) return (int)launch_chain(K::template vec<1, true>(), grid, block, 0, st, p);
    if (nvec <= 64) return (int)launch_chain(K::template vec<2, true>(), grid, block, 0, st, p);
    return (int)launch_chain(K::template vec<4, true>(), grid, block, 0, st, p);
  }
  // values of a thread: 8 or 16 in blocks of up to 1024, 32 or 64 in blocks of up to 512 threads
  int values = p.rows >= 2 * sm_count() ? 32 : 8;
  const auto threads = [&] { return round_up32((p.cols + values - 1) / values); };
  while (threads() > (values <= 16 ? 1024 : 512)) values *= 2;
  const dim3 grid((unsigned)p.rows), block((unsigned)threads());
  if (values == 8) return (int)launch_chain(K::template vec<8 / E, false>(), grid, block, 0, st, p);
  if (values == 16) return (int)launch_chain(K::template vec<16 / E, false>(), grid, block, 0, st, p);
  if (values == 32) return (int)launch_chain(K::template vec<32 / E, false>(), grid, block, 0, st, p);
  return (int)launch_chain(K::template vec<64 / E, false>(), grid, block, 0, st, p);
}

// Rows of 16-byte vectors: width, address and stride; nullptr fits everywhere.
bool fits(const void* p, int64_t stride, int64_t size, int64_t align) { return !p || (((uintptr_t)p | (uintptr_t)(stride * size)) % align) == 0; }

}  // namespace

int launch_rmsnorm_quantize(const RmsNormParams& p, cudaStream_t st) {
  if (!p.rows) return 0;
  const int64_t size = p.dtype == kF32 ? 4 : 2, e = 16 / size;
  const bool vec = p.cols % e == 0 && fits(p.x, p.x_stride, size, 16) && fits(p.residual, p.residual_stride, size, 16) && fits(p.weight, 0, 0, 16) &&
                   fits(p.hidden, p.hidden_stride, size, 16) && fits(p.normed, p.normed_stride, size, 16) && fits(p.q, p.q_stride, 1, e);
  if (p.dtype == kBf16) return launch_rows<NormKernels<__nv_bfloat16>, 8>(p, vec, st);
  if (p.dtype == kF16) return launch_rows<NormKernels<__half>, 8>(p, vec, st);
  return launch_rows<NormKernels<float>, 4>(p, vec, st);
}

int launch_swiglu_quantize(const SwigluParams& p, cudaStream_t st) {
  if (!p.rows) return 0;
  const int64_t size = p.dtype == kF32 ? 4 : 2, e = 16 / size;
  const bool vec = p.cols % e == 0 && fits(p.x, p.x_stride, size, 16) && fits(p.q, p.q_stride, 1, e);
  if (p.dtype == kBf16) return launch_rows<SwigluKernels<__nv_bfloat16>, 8>(p, vec, st);
  if (p.dtype == kF16) return launch_rows<SwigluKernels<__half>, 8>(p, vec, st);
  return launch_rows<SwigluKernels<float>, 4>(p, vec, st);
}

}  // namespace b200
