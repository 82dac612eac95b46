// GEMM of 8-bit rows for a handful of tokens (the contract of gemm_8bit.cu): a stream over the weights.
//
// N * K bytes of weights are read once and nothing else is of their size, so the kernel is bound by HBM, and below about 20 MB by the latency of
// one pass: launch, first bytes, reduction. Weights go from global memory straight into the A fragments of mma.sync.m16n8k32, tokens into
// the B fragments (8 of them are no padding); no shared memory, no barrier before the reduction.
// K order: a sum may take its k in any order as long as both operands agree. Lane (g = lane / 4, t = lane % 4) reads 16 consecutive bytes at
// 64 * unit + 16 * t of weight rows g and g + 8 and of token g, and two MMAs multiply whatever k's the lane has there.
// A block owns 16 weight rows; its warps take the 64-byte units of K in turn, so neighbouring warps read neighbouring sectors, and their
// partial sums meet in shared memory in warp order (int8: exact; e4m3: reproducible).
#include <cuda_fp16.h>

#include "kernels.cuh"
#include "ptx.cuh"

namespace b200 {

namespace {

constexpr int kD8Rows = 16, kD8Unit = 64;                    // weight rows of a block; bytes of K of a step
constexpr int kD8Batch = 4;                                  // steps whose loads fly together

template <bool kInt>
DEV void mma_k32(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (kInt)
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(*reinterpret_cast<int*>(&d[0])), "+r"(*reinterpret_cast<int*>(&d[1])), "+r"(*reinterpret_cast<int*>(&d[2])),
                   "+r"(*reinterpret_cast<int*>(&d[3]))
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Volatile, so that the compiler keeps a batch's loads in front of its first MMA instead of moving them down to save registers.
DEV uint4 load_once(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
DEV uint4 load_again(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

template <bool kInt, int NT>
__global__ void __launch_bounds__(512) k_gemm_8bit_decode(const uint8_t* __restrict__ a, int64_t a_stride, const uint8_t* __restrict__ b, const Gemm8Params p) {
  extern __shared__ float d8_part[];                         // [warps][8 * NT tokens][16 rows]
  constexpr int kTile = 8 * NT * kD8Rows;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = (int)(blockDim.x >> 5);
  const int g = lane >> 2, t = lane & 3;
  const int64_t row0 = (int64_t)blockIdx.x * kD8Rows;
  const int units = (p.K + kD8Unit - 1) / kD8Unit;
  pdl_trigger();
  pdl_wait();
  // rows and tokens past the end read row 0 instead: their sums are not stored
  const uint8_t* w0 = b + (row0 + g < p.N ? row0 + g : 0) * p.K;
  const uint8_t* w1 = b + (row0 + g + 8 < p.N ? row0 + g + 8 : 0) * p.K;
  const uint8_t* x[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) x[n] = a + (8 * n + g < p.M ? 8 * n + g : 0) * a_stride;
  float acc[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;             // all bits zero: an int32 zero as well

  for (int u0 = warp; u0 < units; u0 += warps * kD8Batch) {
    uint4 wa[kD8Batch], wb[kD8Batch], xb[kD8Batch][NT];
#pragma unroll
    for (int i = 0; i < kD8Batch; ++i) {
      const int k = (u0 + i * warps) * kD8Unit + t * 16;     // K is a multiple of 16: a lane's 16 bytes are in or out
      // Out: the row's first bytes times zero, without a branch among the loads (a NaN there is one of the row's own).
      const int at = k < p.K ? k : 0;
      wa[i] = load_once(w0 + at);
      wb[i] = load_once(w1 + at);
#pragma unroll
      for (int n = 0; n < NT; ++n) xb[i][n] = load_again(x[n] + at);
    }
#pragma unroll
    for (int i = 0; i < kD8Batch; ++i)
      if ((u0 + i * warps) * kD8Unit + t * 16 >= p.K) {
#pragma unroll
        for (int n = 0; n < NT; ++n) xb[i][n] = make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
    for (int i = 0; i < kD8Batch; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        mma_k32<kInt>(acc[n], wa[i].x, wb[i].x, wa[i].y, wb[i].y, xb[i][n].x, xb[i][n].y);
        mma_k32<kInt>(acc[n], wa[i].z, wb[i].z, wa[i].w, wb[i].w, xb[i][n].z, xb[i][n].w);
      }
  }
  // accumulator (row g / g + 8, tokens 8n + 2t, 8n + 2t + 1)
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) d8_part[warp * kTile + (8 * n + 2 * t + (i & 1)) * kD8Rows + g + 8 * (i >> 1)] = acc[n][i];
  __syncthreads();
  for (int i = threadIdx.x; i < p.M * kD8Rows; i += blockDim.x) {
    const int tok = i / kD8Rows;
    const int64_t n = row0 + i % kD8Rows;
    if (n >= p.N) continue;
    float sum;
    if (kInt) {
      int total = 0;
      for (int w = 0; w < warps; ++w) total += __float_as_int(d8_part[w * kTile + i]);
      sum = __int2float_rn(total);
    } else {
      sum = d8_part[i];
      for (int w = 1; w < warps; ++w) sum += d8_part[w * kTile + i];
    }
    const float v = sum * __ldg(p.a_scale + tok) * __ldg(p.b_scale + n);
    const int64_t at = tok * p.out_stride + n;
    if (p.out_type == kBf16) reinterpret_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(v);
    else if (p.out_type == kF16) reinterpret_cast<__half*>(p.out)[at] = __float2half_rn(v);
    else reinterpret_cast<float*>(p.out)[at] = v;
  }
}

template <bool kInt, int NT>
int launch_nt(const void* a, int64_t a_stride, const void* b, const Gemm8Params& p, cudaStream_t st) {
  const int64_t blocks = ((int64_t)p.N + kD8Rows - 1) / kD8Rows;
  const int warps = gemm_8bit_decode_warps(blocks, p.K, sm_count());
  const int smem = warps * 8 * NT * kD8Rows * 4;
  static SmemOptIn opt_in;
  if (int e = opt_in.ensure(k_gemm_8bit_decode<kInt, NT>, 16 * 8 * NT * kD8Rows * 4)) return e;
  return (int)launch_chain(k_gemm_8bit_decode<kInt, NT>, dim3((unsigned)blocks), dim3((unsigned)(32 * warps)), smem, st, (const uint8_t*)a, a_stride,
                           (const uint8_t*)b, p);
}

}  // namespace

int launch_gemm_8bit_decode(const void* a, int64_t a_stride, const void* b, const Gemm8Params& p, cudaStream_t st) {
  if (p.M <= 16) return p.code == kInt8 ? launch_nt<true, 2>(a, a_stride, b, p, st) : launch_nt<false, 2>(a, a_stride, b, p, st);
  return launch_nt<true, 4>(a, a_stride, b, p, st);
}

}  // namespace b200
