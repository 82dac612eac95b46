// Rows quantised to 8 bits with one fp32 scale per row, in the launch that produces them:
//   RMS norm   h = x + r,  y = h * rsqrt(mean(h^2) + eps) * w
//   SwiGLU     x = [g | u],  y = g * sigmoid(g) * u
//   both       amax = max|y|,  scale = amax / Q,  q = round_to_nearest_even(y * (Q / amax)),  Q = 127 (int8) or 448 (e4m3)
//
// Both are bound by HBM: every input element is read once, every output element written once, and a row stays in registers between its
// reductions, but for a part of the widest ones, which spills (shifted rows above 16384 columns, fp32 above 8192; aligned fp32 above 16384) (norm 8192 x 7168 bf16 68 us = 6.1 TB/s; SwiGLU 65536 x 768 43 us = 5.8, 16384 x 2048 27 = 6.2). h, the sum of squares, y and amax are fp32; the residual stream h, the normed row y and the code q are each rounded once,
// from the fp32 value (the norm sees h before it is rounded to the stream's type).
// A row holds no scale when it has no finite amax: a NaN or an infinity in it, or a sum of squares beyond fp32, makes the scale NaN and
// the codes zero, so that the row is NaN wherever it is multiplied out. A row whose amax is below 2^-116 counts as zero (scale 0,
// codes 0): Q / amax stays finite for every other one, and scale stays a normal number. Without eps the norm of a row of zeros, or of one whose squares
// vanish in fp32, is 0 * infinity: scale NaN. A y on the border between two codes may take either: y * (Q / amax) and y / scale round differently.
//
// Rows that vectors do not fit (odd widths, strides or addresses) are read as vectors shifted into place (Any16), so a thread holds the
// same columns as otherwise, and written through shared memory, from where they go out in aligned vectors with single elements at the two ends.
// They are bound by instructions (8192 x 4099 83 us where 4096 columns take 40). A block that keeps its weights for several rows (88), one barrier for
// three outputs in places of their own (83) gave nothing; element by element it is 140.
#include <type_traits>

#include "kernels.cuh"
#include "rows.cuh"

namespace b200 {

namespace {

constexpr uint32_t kInfBits = 0x7F800000u;
constexpr float kLeastAmax = 0x1p-116f;

DEV uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// Reductions over the threads of a row: `lanes` of a warp (kWarp, a power of two), or the whole block (32 words of shared memory, one per warp).
template <bool kWarp>
DEV float row_sum(float v, float* red, int lanes) {
  if (kWarp && lanes < 32) {
    for (int o = lanes >> 1; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
  }
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
DEV uint32_t row_max(uint32_t v, uint32_t* red, int lanes) {
  if (kWarp && lanes < 32) {
    for (int o = lanes >> 1; o; o >>= 1) v = max(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
    return v;
  }
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

// Rows of one output that vectors do not fit, on their way out through shared memory, by the whole block.
// A run of bytes whose first lies at smem: aligned vectors of the destination, each cut from two of smem, and up to 15 bytes at either end.
// kPhase: smem has the destination's phase, so that nothing is cut.
template <class T, bool kPhase>
DEV void run_out(const uint8_t* smem, uint8_t* dst, int bytes) {
  const int head = min((int)(-(uint32_t)(uintptr_t)dst & 15u), bytes), pieces = (bytes - head) >> 4, tail = head + 16 * pieces;
  for (int i = threadIdx.x; i < pieces; i += blockDim.x) {
    const uint4* from = reinterpret_cast<const uint4*>(smem + (kPhase ? head : 0)) + i;
    reinterpret_cast<uint4*>(dst + head)[i] = kPhase ? from[0] : shift16(from[0], from[1], (uint32_t)head);
  }
  if (threadIdx.x < 32) {
    const int b = ((int)threadIdx.x & 15) * (int)sizeof(T) + (threadIdx.x < 16 ? 0 : tail);
    if (b < (threadIdx.x < 16 ? head : bytes)) *reinterpret_cast<T*>(dst + b) = *reinterpret_cast<const T*>(smem + b);
  }
}
// A block with one row lays it out from the start of `smem`.
template <class T>
DEV void row_out(const uint8_t* smem, uint8_t* dst, int bytes) {
  __syncthreads();
  run_out<T, false>(smem, dst, bytes);
  __syncthreads();
}
// A block with several short rows lays them out in the phase that their destination has. Rows that lie behind one another in memory are one
// run of bytes; others have a place of `pitch` bytes each.
struct Stage {
  uint8_t *smem, *dst;       // dst: the block's first row
  int64_t stride;            // bytes between rows of dst
  int rows, row_bytes;
  DEV bool one_run() const { return stride == row_bytes || rows == 1; }
  DEV int pitch() const { return ((row_bytes + 15) & ~15) + 16; }
  DEV uint8_t* at(int r) const {
    if (one_run()) return smem + ((uint32_t)(uintptr_t)dst & 15u) + r * row_bytes;
    return smem + r * pitch() + ((uint32_t)(uintptr_t)(dst + r * stride) & 15u);
  }
  template <class T>
  DEV void out() const {
    __syncthreads();
    if (one_run()) {
      run_out<T, true>(at(0), dst, rows * row_bytes);
    } else {
      for (int r = 0; r < rows; ++r) run_out<T, true>(at(r), dst + r * stride, row_bytes);
    }
    __syncthreads();
  }
};
int stage_bytes(int rows, int64_t row_bytes) { return rows * (int)((row_bytes + 15) / 16 * 16 + 16) + 16; }

// What a thread of a row kernel works on: vectors v0, v0 + step, ... of a row. kWarp: `lanes` threads of a warp share a row, blockDim.x / lanes
// rows to a block; otherwise a block has one.
template <class T, bool kWarp, bool kAny>
struct Place {
  int64_t row, first;        // this thread's row, the block's first
  int r, v0, step, nvec;
  DEV Place(int cols, int lanes) {
    constexpr int E = Vec<T>::E;
    r = kWarp ? (int)threadIdx.x / lanes : 0;
    first = kWarp ? (int64_t)blockIdx.x * (int)(blockDim.x / lanes) : (int64_t)blockIdx.x;
    row = first + r;
    v0 = kWarp ? (int)threadIdx.x % lanes : (int)threadIdx.x;
    step = kWarp ? lanes : (int)blockDim.x;
    nvec = kAny ? (cols + E - 1) / E : cols / E;
  }
  DEV int rows_here(int64_t rows, int lanes) const {
    return kWarp ? (int)min(rows - first, (int64_t)(blockDim.x / lanes)) : 1;
  }
};

template <class T>
DEV const uint8_t* vec_at(const T* row, int v) { return reinterpret_cast<const uint8_t*>(row) + (int64_t)v * 16; }

// One output's rows: VPT vectors of fp32 values of a thread, rounded to T.
template <class T, int VPT, bool kWarp, bool kAny>
DEV void store_rows(T* out, int64_t stride, const float (&y)[VPT][Vec<T>::E], const Place<T, kWarp, kAny>& at, int cols, int rows, uint8_t* smem) {
  constexpr int E = Vec<T>::E;
  const Stage st{smem, reinterpret_cast<uint8_t*>(out + at.first * stride), stride * (int64_t)sizeof(T), rows, cols * (int)sizeof(T)};
  if (at.r < rows) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = at.v0 + i * at.step;
      if (v >= at.nvec) continue;
      Vec<T> o;
#pragma unroll
      for (int j = 0; j < E; ++j) o.v[j] = from_f32<T>(y[i][j]);
      if constexpr (!kAny) {
        reinterpret_cast<uint4*>(out + at.row * stride)[v] = o.raw;
      } else if constexpr (!kWarp) {
        reinterpret_cast<uint4*>(smem)[v] = o.raw;           // what is past the row's end stays here
      } else {
        T* to = reinterpret_cast<T*>(st.at(at.r)) + v * E;
        const int n = min(E, cols - v * E);
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (j < n) to[j] = o.v[j];
      }
    }
  }
  if constexpr (kAny && !kWarp) row_out<T>(smem, st.dst, st.row_bytes);
  if constexpr (kAny && kWarp) st.template out<T>();
}

// The codes and the scale.
template <class I, int VPT, bool kWarp, bool kAny>
DEV void store_codes(uint8_t* q, int64_t stride, float* scale_out, const float (&y)[VPT][Vec<I>::E], uint32_t amax, int q_type,
                     const Place<I, kWarp, kAny>& at, int cols, int rows, uint8_t* smem) {
  constexpr int E = Vec<I>::E;
  float scale;
  const float f = code_factor(amax, q_type, scale);
  if (at.v0 == 0 && at.r < rows) scale_out[at.row] = scale;
  const Stage st{smem, q + at.first * stride, stride, rows, cols};
  if (at.r < rows) {
    uint8_t* to = !kAny ? q + at.row * stride : kWarp ? st.at(at.r) : smem;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = at.v0 + i * at.step;
      if (v >= at.nvec) continue;
      uint32_t w[E / 4];
#pragma unroll
      for (int j = 0; j < E / 4; ++j) w[j] = codes4(y[i][4 * j], y[i][4 * j + 1], y[i][4 * j + 2], y[i][4 * j + 3], f, q_type);
      if constexpr (!kAny || !kWarp) {
        if constexpr (E == 8) *reinterpret_cast<uint2*>(to + (int64_t)v * E) = make_uint2(w[0], w[1]);
        else *reinterpret_cast<uint32_t*>(to + (int64_t)v * E) = w[0];
      } else {
        const int n = min(E, cols - v * E);
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (j < n) to[v * E + j] = (uint8_t)(w[j / 4] >> (j % 4 * 8));
      }
    }
  }
  if constexpr (kAny && !kWarp) row_out<uint8_t>(smem, st.dst, cols);
  if constexpr (kAny && kWarp) st.template out<uint8_t>();
}

// A vector that ends behind its row: the neighbour's elements become zero. They add nothing to the sums and to amax.
template <class T>
DEV void cut_vec(Vec<T>& x, int v, int cols) {
  if ((v + 1) * Vec<T>::E <= cols) return;
#pragma unroll
  for (int j = 0; j < Vec<T>::E; ++j)
    if (v * Vec<T>::E + j >= cols) x.v[j] = from_f32<T>(0.f);
}

// Most threads of a block: 64 registers a thread hold up to 16 values of a row and what is loaded for them, 128 the rest.
template <class T, int VPT, bool kWarp>
constexpr int row_threads() { return kWarp ? 128 : VPT * Vec<T>::E <= 16 ? 1024 : 512; }

// ----------------------------------------------------------------------------- norm
// A thread reads and writes the same places of x, residual, hidden and normed of its row (through shared memory: after the block has read
// its rows), so hidden may be x or residual itself.
template <class T, int VPT, bool kWarp, bool kAny>
__global__ void __launch_bounds__(row_threads<T, VPT, kWarp>()) k_rmsnorm_quantize(const RmsNormParams p, const int lanes) {
  constexpr int E = Vec<T>::E;
  extern __shared__ uint4 row_smem[];
  __shared__ float red_sum[32];
  __shared__ uint32_t red_max[32];
  const Place<T, kWarp, kAny> at(p.cols, lanes);
  const int rows = at.rows_here(p.rows, lanes);
  uint8_t* smem = reinterpret_cast<uint8_t*>(row_smem);
  pdl_trigger();
  pdl_wait();
  const bool live = at.r < rows;
  const T* x = (const T*)p.x + at.row * p.x_stride;
  const T* r = p.residual ? (const T*)p.residual + at.row * p.residual_stride : nullptr;
  const Span sx = span_of<T>(p.x, p.rows, p.x_stride, p.cols, x), sr = span_of<T>(p.residual, p.rows, p.residual_stride, p.cols, r);
  const T* rows_r = r ? r : x;                               // any address: nothing is fetched without a residual
  Fetch16<T, kAny, !kWarp> xf[VPT], rf[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = at.v0 + i * at.step;
    xf[i].fetch(vec_at(x, v), sx, live && v < at.nvec);
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = at.v0 + i * at.step;
    rf[i].fetch(vec_at(rows_r, v), sr, r && live && v < at.nvec);
  }
  float y[VPT][E];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = at.v0 + i * at.step;
    Vec<T> xv, rv;
    xv.raw = rv.raw = make_uint4(0u, 0u, 0u, 0u);
    if (live && v < at.nvec) {
      xv.raw = xf[i].take(vec_at(x, v), sx);
      if (r) rv.raw = rf[i].take(vec_at(r, v), sr);
      if constexpr (kAny) {
        cut_vec<T>(xv, v, p.cols);
        if (r) cut_vec<T>(rv, v, p.cols);
      }
    }
#pragma unroll
    for (int j = 0; j < E; ++j) {
      y[i][j] = to_f32(xv.v[j]);
      if (r) y[i][j] += to_f32(rv.v[j]);
      ss = fmaf(y[i][j], y[i][j], ss);
    }
  }
  if (p.hidden) store_rows<T, VPT, kWarp, kAny>((T*)p.hidden, p.hidden_stride, y, at, p.cols, rows, smem);
  ss = row_sum<kWarp>(ss, red_sum, lanes);
  // a sum that is no number leaves no finite y either (infinity * 0 would pass for one)
  const float rstd = abs_bits(ss) < kInfBits ? rsqrtf(ss / (float)p.cols + p.eps) : __uint_as_float(0x7FC00000u);
  uint32_t amax = 0;
  if (p.weight_f32) {
    const Span sw = span_of<float>(p.weight, 1, 0, p.cols, p.weight);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = at.v0 + i * at.step;
      if (v >= at.nvec) continue;
#pragma unroll
      for (int j = 0; j < E / 4; ++j) {
        const uint8_t* from = vec_at((const float*)p.weight, v * (E / 4) + j);
        Fetch16<float, kAny> f;
        Vec<float> c;
        f.fetch(from, sw, true);
        c.raw = f.take(from, sw);
#pragma unroll
        for (int k = 0; k < 4; ++k) y[i][4 * j + k] *= rstd * c.v[k];
      }
    }
  } else {
    const Span sw = span_of<T>(p.weight, 1, 0, p.cols, p.weight);
    Fetch16<T, kAny> f[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) f[i].fetch(vec_at((const T*)p.weight, at.v0 + i * at.step), sw, at.v0 + i * at.step < at.nvec);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (at.v0 + i * at.step >= at.nvec) continue;
      Vec<T> c;
      c.raw = f[i].take(vec_at((const T*)p.weight, at.v0 + i * at.step), sw);
#pragma unroll
      for (int j = 0; j < E; ++j) y[i][j] *= rstd * to_f32(c.v[j]);
    }
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int j = 0; j < E; ++j) amax = max(amax, abs_bits(y[i][j]));
  amax = row_max<kWarp>(amax, red_max, lanes);
  store_codes<T, VPT, kWarp, kAny>(p.q, p.q_stride, p.scale, y, amax, p.q_type, at, p.cols, rows, smem);
  if (p.normed) store_rows<T, VPT, kWarp, kAny>((T*)p.normed, p.normed_stride, y, at, p.cols, rows, smem);
}

// ----------------------------------------------------------------------------- SwiGLU
// g * sigmoid(g) * u = g / (1 + exp(-g)) * u, while the quotient is a normal number. (The approximations flush subnormals and meet none.)
constexpr float kFarGate = -87.f;
DEV float silu_mul(float g, float u) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.44269504f));             // log2(e)
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return g * r * u;
}
// The same for any g: with e = exp(-|g| / 2) sigmoid is 1 / (1 + e^2) above zero and e^2 / (1 + e^2) below, where u comes in between the two e. A large u
// lifts y above the least amax down to a gate of -174, and so far e is a normal number. Taken for vectors with a gate below kFarGate: for
// every element it is dearer (65536 x 768 49 us instead of 43).
DEV float silu_mul_far(float g, float u) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fabsf(g) * -0.72134752f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(fmaf(e, e, 1.f)));
  const float f = g < 0.f ? e : 1.f;
  return g * r * (f * u) * f;
}

// The least element of a vector (a NaN is none).
DEV float least(const Vec<float>& x) { return fminf(fminf(x.v[0], x.v[1]), fminf(x.v[2], x.v[3])); }
template <class T>
DEV float least(const Vec<T>& x) {
  using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
  union {
    uint4 raw;
    T2 pair[4];
  } p{x.raw};
  const T2 m = __hmin2(__hmin2(p.pair[0], p.pair[1]), __hmin2(p.pair[2], p.pair[3]));
  return fminf(to_f32(m.x), to_f32(m.y));
}

template <class T, int VPT, bool kWarp, bool kAny>
__global__ void __launch_bounds__(row_threads<T, VPT, kWarp>()) k_swiglu_quantize(const SwigluParams p, const int lanes) {
  constexpr int E = Vec<T>::E;
  extern __shared__ uint4 row_smem[];
  __shared__ uint32_t red_max[32];
  const Place<T, kWarp, kAny> at(p.cols, lanes);
  const int rows = at.rows_here(p.rows, lanes);
  pdl_trigger();
  pdl_wait();
  const bool live = at.r < rows;
  const T* g = (const T*)p.x + at.row * p.x_stride;
  const Span sx = span_of<T>(p.x, p.rows, p.x_stride, 2 * (int64_t)p.cols, g);
  Fetch16<T, kAny, !kWarp> gf[VPT], uf[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = at.v0 + i * at.step;
    gf[i].fetch(vec_at(g, v), sx, live && v < at.nvec);
    uf[i].fetch(vec_at(g + p.cols, v), sx, live && v < at.nvec);
  }
  float y[VPT][E];
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = at.v0 + i * at.step;
    Vec<T> gv, uv;
    gv.raw = uv.raw = make_uint4(0u, 0u, 0u, 0u);
    if (live && v < at.nvec) {
      gv.raw = gf[i].take(vec_at(g, v), sx);
      uv.raw = uf[i].take(vec_at(g + p.cols, v), sx);
      if constexpr (kAny) {
        cut_vec<T>(gv, v, p.cols);
        cut_vec<T>(uv, v, p.cols);
      }
    }
    if (!(least(gv) < kFarGate)) {
#pragma unroll
      for (int j = 0; j < E; ++j) y[i][j] = silu_mul(to_f32(gv.v[j]), to_f32(uv.v[j]));
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j) y[i][j] = silu_mul_far(to_f32(gv.v[j]), to_f32(uv.v[j]));
    }
#pragma unroll
    for (int j = 0; j < E; ++j) amax = max(amax, abs_bits(y[i][j]));
  }
  amax = row_max<kWarp>(amax, red_max, lanes);
  store_codes<T, VPT, kWarp, kAny>(p.q, p.q_stride, p.scale, y, amax, p.q_type, at, p.cols, rows, reinterpret_cast<uint8_t*>(row_smem));
}

// ----------------------------------------------------------------------------- launches
int round_up32(int v) { return (v + 31) / 32 * 32; }

template <class T>
struct NormKernels {
  using P = RmsNormParams;
  using I = T;
  static constexpr int kStageSize = sizeof(T);               // bytes of the widest output element
  // values of a thread where rows are many: 8192 x 7168 bf16 68 us with 32, 72 with 16; 8192 x 2048 fp32 36 with 32, 35 with 16. Shifted
  // vectors take registers: 8192 x 4099 bf16 98 us with 16, 120 with 32; 8192 x 2047 fp32 70 with 8, 88 with 16
  static constexpr int kValues = sizeof(T) == 2 ? 32 : 16, kValuesAny = sizeof(T) == 2 ? 16 : 8;
  template <int VPT, bool kWarp, bool kAny>
  static constexpr auto kernel() { return k_rmsnorm_quantize<T, VPT, kWarp, kAny>; }
};
template <class T>
struct SwigluKernels {
  using P = SwigluParams;
  using I = T;
  static constexpr int kStageSize = 1;
  static constexpr int kValues = 16, kValuesAny = sizeof(T) == 2 ? 16 : 8;         // 16384 x 2048 bf16 27.2 us with 16, 27.7 with 32
  template <int VPT, bool kWarp, bool kAny>
  static constexpr auto kernel() { return k_swiglu_quantize<T, VPT, kWarp, kAny>; }
};

template <class K, int VPT, bool kWarp, bool kAny>
int launch_form(const typename K::P& p, int threads, int lanes, cudaStream_t st) {
  const int rows = kWarp ? threads / lanes : 1;
  const int smem = kAny ? stage_bytes(rows, (int64_t)p.cols * K::kStageSize) : 0;
  if (smem > 32 * 1024) {
    static SmemOptIn opt_in;
    if (int e = opt_in.ensure(K::template kernel<VPT, kWarp, kAny>(), stage_bytes(1, kRowQuantMaxCols * K::kStageSize))) return e;
  }
  return (int)launch_chain(K::template kernel<VPT, kWarp, kAny>(), dim3((unsigned)((p.rows + rows - 1) / rows)), dim3((unsigned)threads), (size_t)smem, st, p, lanes);
}

// Up to 96 vectors (64 where they are shifted) a row is a warp's, or a part's of one: no barrier, 128 threads to a block. Above that a block's, of as
// many vectors per thread as leave every SM several blocks; with fewer rows than that, one vector per thread and more threads, because
// a row's own latency is the time.
template <class K, bool kAny>
int launch_rows(const typename K::P& p, cudaStream_t st) {
  constexpr int E = Vec<typename K::I>::E;
  const int nvec = (p.cols + E - 1) / E;
  if (nvec <= (kAny ? 64 : 96)) {
    int lanes = 1;
    while (lanes < nvec && lanes < 32) lanes *= 2;
    if (nvec <= 32) return launch_form<K, 1, true, kAny>(p, 128, lanes, st);
    if (kAny || nvec <= 64) return launch_form<K, 2, true, kAny>(p, 128, lanes, st);
    if constexpr (!kAny) return launch_form<K, 3, true, false>(p, 128, lanes, st);
  }
  // values of a thread: 8 or 16 in blocks of up to 1024, 32 or 64 in blocks of up to 512 threads
  int values = p.rows < 2 * sm_count() ? 8 : kAny ? K::kValuesAny : nvec <= 128 ? 16 : K::kValues;
  const auto threads = [&] { return round_up32((nvec * E + values - 1) / values); };
  while (threads() > (values <= 16 ? 1024 : 512)) values *= 2;
  if (values == 8) return launch_form<K, 8 / E, false, kAny>(p, threads(), 32, st);
  if (values == 16) return launch_form<K, 16 / E, false, kAny>(p, threads(), 32, st);
  if constexpr (!kAny && K::kValues == 32) {                 // elsewhere the step from 16 values leads past 32: as many columns fit 16
    if (values == 32) return launch_form<K, 32 / E, false, kAny>(p, threads(), 32, st);
  }
  return launch_form<K, 64 / E, false, kAny>(p, threads(), 32, st);
}

// Whether 16-byte vectors fit an address and the stride between rows, in bytes; a null pointer fits everywhere.
bool fits(const void* p, int64_t stride, int64_t align) { return !p || (((uintptr_t)p | (uintptr_t)stride) % align) == 0; }

template <class T>
int launch_norm(const RmsNormParams& p, cudaStream_t st) {
  constexpr int64_t size = sizeof(T), e = 16 / size;
  const bool vec = p.cols % e == 0 && fits(p.x, p.x_stride * size, 16) && fits(p.residual, p.residual_stride * size, 16) && fits(p.weight, 0, 16) &&
                   fits(p.hidden, p.hidden_stride * size, 16) && fits(p.normed, p.normed_stride * size, 16) && fits(p.q, p.q_stride, e);
  return vec ? launch_rows<NormKernels<T>, false>(p, st) : launch_rows<NormKernels<T>, true>(p, st);
}

template <class T>
int launch_swiglu(const SwigluParams& p, cudaStream_t st) {
  constexpr int64_t size = sizeof(T), e = 16 / size;
  const bool vec = p.cols % e == 0 && fits(p.x, p.x_stride * size, 16) && fits(p.q, p.q_stride, e);
  return vec ? launch_rows<SwigluKernels<T>, false>(p, st) : launch_rows<SwigluKernels<T>, true>(p, st);
}

}  // namespace

int launch_rmsnorm_quantize(const RmsNormParams& p, cudaStream_t st) {
  if (!p.rows) return 0;
  if (p.dtype == kBf16) return launch_norm<__nv_bfloat16>(p, st);
  if (p.dtype == kF16) return launch_norm<__half>(p, st);
  return launch_norm<float>(p, st);
}

int launch_swiglu_quantize(const SwigluParams& p, cudaStream_t st) {
  if (!p.rows) return 0;
  if (p.dtype == kBf16) return launch_swiglu<__nv_bfloat16>(p, st);
  if (p.dtype == kF16) return launch_swiglu<__half>(p, st);
  return launch_swiglu<float>(p, st);
}

}  // namespace b200
