// Tokens in the order of their experts, and back, with what a backward pass needs. Unlike the route map of the layer (route_map.cu) the
// segments are tight (no rows of padding) and nothing belongs to a layer.
//
//   order      a stable counting sort of the T * K routes by expert: offsets[e], row_of[t, k], route_of_row[r]. Routes without an expert of
//              this range sort behind all others: row_of = -1, and the rows behind offsets[E] have route_of_row = -1.
//   sort       rows[row_of[t, k]] = x[t], zeros behind offsets[E]
//   unsort     y[t] = sum_k w[t, k] * rows[row_of[t, k]], fp32 in ascending k, rounded once; with w = 1 the gradient of sort
//   gradient   drows[row_of[t, k]] = w[t, k] * dy[t], zeros behind offsets[E];  dw[t, k] = <rows[row_of[t, k]], dy[t]>
//
// No atomics on global memory, every sum in a fixed order: the same inputs give the same bits.
#include <cuda_fp16.h>

#include "kernels.cuh"
#include "ptx.cuh"

namespace b200 {

namespace {

// ----------------------------------------------------------------------------- order
// One thread per route. A chunk is ranked by per-warp histograms (each warp owns a row of `hist`, and within a warp the lanes of one bucket
// find each other with one ballot per bit of the bucket), so positions follow the flat route index. Bucket E takes the routes
// without an expert.
constexpr int kOrdThreads = 1024, kOrdWarps = 32;
// Chunks that one launch ranks: every block counts all ids by itself, eight per thread at most.
constexpr int kOrdFusedChunks = 8;
// Chunks up to which a block adds up the other chunks' counts itself; beyond, a launch of its own turns the counts into prefixes.
constexpr int kOrdDirectChunks = 128;

struct OrderView {
  const int32_t* ids;
  int64_t stride;
  int64_t total;
  int K, E;
};

DEV int bucket_of(const OrderView& v, int64_t f) {
  if (f >= v.total) return -1;
  const int64_t t = v.total <= INT32_MAX ? (int64_t)((uint32_t)f / (uint32_t)v.K) : f / v.K;
  const int e = __ldg(v.ids + t * v.stride + (f - t * v.K));
  return (uint32_t)e < (uint32_t)v.E ? e : v.E;
}

// Lanes whose bucket is this lane's; -1 (no route) matches nothing that is looked at.
DEV unsigned same_bucket(int b, int bits) {
  unsigned m = __ballot_sync(0xFFFFFFFFu, b >= 0);
  for (int i = 0; i < bits; ++i) {
    const bool set = (b >> i) & 1;
    const unsigned bal = __ballot_sync(0xFFFFFFFFu, set);
    m &= set ? bal : ~bal;
  }
  return m;
}

// Shared memory: hist [32 warps][nb] 16-bit, then before[nb], base[nb + 1] (32-bit).
__host__ __device__ inline int ord_hist_bytes(int nb) { return (kOrdWarps * nb * 2 + 15) / 16 * 16; }
inline int ord_smem(int nb) { return ord_hist_bytes(nb) + (2 * nb + 1) * 4; }

DEV void chunk_hist(uint16_t* hist, int b, unsigned same, int nb) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < ord_hist_bytes(nb) / 16; i += kOrdThreads) reinterpret_cast<uint4*>(hist)[i] = make_uint4(0u, 0u, 0u, 0u);
  __syncthreads();
  if (b >= 0 && lane == __ffs(same) - 1) hist[warp * nb + b] = (uint16_t)__popc(same);
  __syncthreads();
}

__global__ void __launch_bounds__(kOrdThreads) k_order_hist(const OrderView v, int bits, int32_t* __restrict__ counts) {
  extern __shared__ uint4 ord_smem_raw[];
  uint16_t* hist = reinterpret_cast<uint16_t*>(ord_smem_raw);
  const int nb = v.E + 1;
  pdl_trigger();
  pdl_wait();
  const int b = bucket_of(v, (int64_t)blockIdx.x * kOrdThreads + threadIdx.x);
  chunk_hist(hist, b, same_bucket(b, bits), nb);
  for (int e = threadIdx.x; e < nb; e += kOrdThreads) {
    int sum = 0;
#pragma unroll
    for (int w = 0; w < kOrdWarps; ++w) sum += hist[w * nb + e];
    counts[(int64_t)blockIdx.x * nb + e] = sum;
  }
}

// counts[c][e] -> counts of the chunks before c; the totals go into row `chunks`.
__global__ void __launch_bounds__(128) k_order_scan(int32_t* counts, int chunks, int nb) {
  const int e = blockIdx.x * 128 + threadIdx.x;
  pdl_trigger();
  pdl_wait();
  if (e >= nb) return;
  int sum = 0;
  for (int c0 = 0; c0 < chunks; c0 += 8) {
    int v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c0 + i < chunks ? counts[(int64_t)(c0 + i) * nb + e] : 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c0 + i < chunks) {
        counts[(int64_t)(c0 + i) * nb + e] = sum;
        sum += v[i];
      }
  }
  counts[(int64_t)chunks * nb + e] = sum;
}

// kForm 0: counts itself (one launch); 1: adds up the chunks' counts; 2: reads prefixes.
template <int kForm>
__global__ void __launch_bounds__(kOrdThreads) k_order_scatter(const OrderView v, int bits, const int32_t* __restrict__ counts, int chunks,
                                                               int32_t* __restrict__ offsets, int32_t* __restrict__ row_of,
                                                               int32_t* __restrict__ route_of_row) {
  extern __shared__ uint4 ord_smem_raw[];
  __shared__ int warp_sum[kOrdWarps];
  const int nb = v.E + 1, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint16_t* hist = reinterpret_cast<uint16_t*>(ord_smem_raw);
  int* before = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(ord_smem_raw) + ord_hist_bytes(nb));
  int* base = before + nb;
  pdl_trigger();
  pdl_wait();
  const int64_t f = (int64_t)blockIdx.x * kOrdThreads + threadIdx.x;
  const int b = bucket_of(v, f);
  if (kForm == 0) {
    for (int e = threadIdx.x; e < 2 * nb; e += kOrdThreads) before[e] = 0;      // before and base
    __syncthreads();
    for (int c = 0; c < chunks; ++c) {
      const int o = c == (int)blockIdx.x ? b : bucket_of(v, (int64_t)c * kOrdThreads + threadIdx.x);
      if (o >= 0) {
        atomicAdd(base + o, 1);                                                  // sums of ones: any order gives the same
        if (c < (int)blockIdx.x) atomicAdd(before + o, 1);
      }
    }
  } else {
    for (int e = threadIdx.x; e < nb; e += kOrdThreads) {
      int sum = 0, mine = 0;
      if (kForm == 1) {
#pragma unroll 8
        for (int c = 0; c < chunks; ++c) {
          if (c == (int)blockIdx.x) mine = sum;
          sum += __ldg(counts + (int64_t)c * nb + e);
        }
      } else {
        mine = __ldg(counts + (int64_t)blockIdx.x * nb + e);
        sum = __ldg(counts + (int64_t)chunks * nb + e);
      }
      before[e] = mine;
      base[e] = sum;
    }
  }
  const unsigned same = same_bucket(b, bits);
  chunk_hist(hist, b, same, nb);
  // base: totals -> first rows, buckets dealt to the threads in order (two where there are more than threads)
  const int per = (nb + kOrdThreads - 1) / kOrdThreads;
  int mine = 0;
  for (int i = 0; i < per; ++i) mine += (int)threadIdx.x * per + i < nb ? base[threadIdx.x * per + i] : 0;
  int run = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xFFFFFFFFu, run, o);
    if (lane >= o) run += u;
  }
  if (lane == 31) warp_sum[warp] = run;
  __syncthreads();
  int lead = lane < warp ? warp_sum[lane] : 0;
#pragma unroll
  for (int o = 16; o; o >>= 1) lead += __shfl_xor_sync(0xFFFFFFFFu, lead, o);
  run += lead - mine;
  for (int i = 0; i < per; ++i) {
    const int e = threadIdx.x * per + i;
    if (e < nb) {
      const int n = base[e];
      base[e] = run;
      if (blockIdx.x == 0) offsets[e] = run;
      run += n;
    }
  }
  // hist: counts of a chunk's warps -> routes of the chunk in front of each warp
  for (int e = threadIdx.x; e < nb; e += kOrdThreads) {
    int sum = 0;
#pragma unroll
    for (int w = 0; w < kOrdWarps; ++w) {
      const int n = hist[w * nb + e];
      hist[w * nb + e] = (uint16_t)sum;
      sum += n;
    }
  }
  __syncthreads();
  if (b < 0) return;
  const int row = base[b] + before[b] + hist[warp * nb + b] + __popc(same & ((1u << lane) - 1));
  row_of[f] = b < v.E ? row : -1;
  route_of_row[row] = b < v.E ? (int32_t)f : -1;
}

// ----------------------------------------------------------------------------- rows
DEV float to_f(float v) { return v; }
DEV float to_f(__half v) { return __half2float(v); }
DEV float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
DEV T from_f(float v);
template <>
DEV float from_f<float>(float v) { return v; }
template <>
DEV __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
DEV __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// E elements of T as one access (16 bytes, or one element where rows do not start on 16-byte boundaries).
template <class T, int E>
struct __align__(sizeof(T) * E) Piece {
  T v[E];
};

constexpr int kRowThreads = 256;

// Zeros in the rows behind the last route: dealt to all threads of the grid.
template <class P>
DEV void zero_behind(P* rows, int64_t pieces, const int32_t* valid, int64_t n_rows) {
  const int64_t first = (int64_t)min(max(__ldg(valid), 0), (int)n_rows) * pieces, end = n_rows * pieces;
  P zero;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(P) / sizeof(zero.v[0])); ++i) zero.v[i] = decltype(zero.v[0] + zero.v[0])(0);
  for (int64_t i = first + (int64_t)blockIdx.x * kRowThreads + threadIdx.x; i < end; i += (int64_t)gridDim.x * kRowThreads) rows[i] = zero;
}

// A thread owns N pieces of one token (pieces p, p + lanes, ...): read once, written to the token's K rows.
// `lanes` threads share a token; the grid covers T * lanes threads.
template <class U, int E, int N>
__global__ void __launch_bounds__(kRowThreads) k_sort_rows(const U* __restrict__ x, int64_t x_stride, int64_t T, int64_t pieces, int64_t lanes,
                                                           const int32_t* __restrict__ row_of, int K, const int32_t* __restrict__ valid,
                                                           U* __restrict__ rows) {
  using P = Piece<U, E>;
  pdl_trigger();
  pdl_wait();
  const int64_t n_rows = T * K;
  const int64_t i = (int64_t)blockIdx.x * kRowThreads + threadIdx.x;
  const int64_t t = i / lanes, p0 = i - t * lanes;
  if (t < T) {
    P v[N];
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (p0 + j * lanes < pieces) v[j] = *(reinterpret_cast<const P*>(x + t * x_stride) + p0 + j * lanes);
    for (int k = 0; k < K; ++k) {
      const int64_t row = __ldg(row_of + t * K + k);
      if (row < 0 || row >= n_rows) continue;
      P* dst = reinterpret_cast<P*>(rows) + row * pieces;
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (p0 + j * lanes < pieces) dst[p0 + j * lanes] = v[j];
    }
  }
  zero_behind(reinterpret_cast<P*>(rows), pieces, valid, n_rows);
}

// y[t] (+ weights): eight slots' rows in flight per thread, one piece of a token each.
template <class T_, int E>
__global__ void __launch_bounds__(kRowThreads) k_unsort_rows(const T_* __restrict__ rows, int64_t rows_stride, int64_t n_rows,
                                                             const int32_t* __restrict__ row_of, const float* __restrict__ weights, int64_t T, int K,
                                                             int64_t pieces, T_* __restrict__ y, int64_t y_stride) {
  using P = Piece<T_, E>;
  pdl_trigger();
  pdl_wait();
  const int64_t i = (int64_t)blockIdx.x * kRowThreads + threadIdx.x;
  const int64_t t = i / pieces, p = i - t * pieces;
  if (t >= T) return;
  float acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  for (int k0 = 0; k0 < K; k0 += 8) {
    int64_t row[8];
    float w[8];
    P v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      row[j] = k0 + j < K ? __ldg(row_of + t * K + k0 + j) : -1;
      w[j] = weights && k0 + j < K ? __ldg(weights + t * K + k0 + j) : 1.f;
      if (row[j] >= n_rows) row[j] = -1;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (row[j] >= 0) v[j] = *(reinterpret_cast<const P*>(rows + row[j] * rows_stride) + p);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (row[j] >= 0) {
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = fmaf(to_f(v[j].v[e]), w[j], acc[e]);
      }
  }
  P o;
#pragma unroll
  for (int e = 0; e < E; ++e) o.v[e] = from_f<T_>(acc[e]);
  *(reinterpret_cast<P*>(y + t * y_stride) + p) = o;
}

// One warp per token: a piece of dy is read once for the token's K rows; their dot products stay in registers, four slots at a time.
template <class T_, int E>
__global__ void __launch_bounds__(kRowThreads) k_unsort_backward(const T_* __restrict__ dy, int64_t dy_stride, const T_* __restrict__ rows,
                                                                 int64_t rows_stride, const int32_t* __restrict__ row_of,
                                                                 const float* __restrict__ weights, int64_t T, int K, int64_t pieces,
                                                                 const int32_t* __restrict__ valid, T_* __restrict__ drows, float* __restrict__ dweights) {
  using P = Piece<T_, E>;
  constexpr int kSlots = 4;
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t t = (int64_t)blockIdx.x * (kRowThreads / 32) + (threadIdx.x >> 5), n_rows = T * K;
  if (t < T) {
    for (int k0 = 0; k0 < K; k0 += kSlots) {
      int64_t row[kSlots];
      float w[kSlots], dot[kSlots];
#pragma unroll
      for (int j = 0; j < kSlots; ++j) {
        row[j] = k0 + j < K ? __ldg(row_of + t * K + k0 + j) : -1;
        w[j] = weights && k0 + j < K ? __ldg(weights + t * K + k0 + j) : 1.f;
        if (row[j] >= n_rows) row[j] = -1;
        dot[j] = 0.f;
      }
      for (int64_t p = lane; p < pieces; p += 32) {
        const P g = *(reinterpret_cast<const P*>(dy + t * dy_stride) + p);
        P v[kSlots];
        if (dweights) {
#pragma unroll
          for (int j = 0; j < kSlots; ++j)
            if (row[j] >= 0) v[j] = *(reinterpret_cast<const P*>(rows + row[j] * rows_stride) + p);
        }
#pragma unroll
        for (int j = 0; j < kSlots; ++j) {
          if (row[j] < 0) continue;
          if (dweights) {
#pragma unroll
            for (int e = 0; e < E; ++e) dot[j] = fmaf(to_f(v[j].v[e]), to_f(g.v[e]), dot[j]);
          }
          if (drows) {
            P o;
#pragma unroll
            for (int e = 0; e < E; ++e) o.v[e] = from_f<T_>(to_f(g.v[e]) * w[j]);
            reinterpret_cast<P*>(drows)[row[j] * pieces + p] = o;
          }
        }
      }
      if (dweights) {
#pragma unroll
        for (int j = 0; j < kSlots; ++j) {
#pragma unroll
          for (int o = 16; o; o >>= 1) dot[j] += __shfl_xor_sync(0xFFFFFFFFu, dot[j], o);
          if (lane == 0 && k0 + j < K) dweights[t * K + k0 + j] = row[j] >= 0 ? dot[j] : 0.f;
        }
      }
    }
  }
  if (drows) zero_behind(reinterpret_cast<P*>(drows), pieces, valid, n_rows);
}

unsigned blocks_of(int64_t n, int64_t per) { return (unsigned)((n + per - 1) / per); }

template <class U, int E>
int launch_sort(const void* x, int64_t x_stride_bytes, int64_t T, int64_t row_bytes, const int32_t* row_of, int K, const int32_t* valid, void* rows,
                cudaStream_t st) {
  const int64_t pieces = row_bytes / (int64_t)(sizeof(U) * E), stride = x_stride_bytes / (int64_t)sizeof(U);
  // four pieces per thread once that still fills the device: fewer index reads for the same bytes
  const bool four = T * pieces >= 4ll * 1024 * sm_count();
  const int64_t lanes = four ? (pieces + 3) / 4 : pieces;
  const dim3 grid(blocks_of(T * lanes, kRowThreads)), block(kRowThreads);
  if (four) return (int)launch_chain(k_sort_rows<U, E, 4>, grid, block, 0, st, (const U*)x, stride, T, pieces, lanes, row_of, K, valid, (U*)rows);
  return (int)launch_chain(k_sort_rows<U, E, 1>, grid, block, 0, st, (const U*)x, stride, T, pieces, lanes, row_of, K, valid, (U*)rows);
}

template <class T_, int E>
int launch_unsort(const UnsortParams& p, cudaStream_t st) {
  const int64_t pieces = p.cols / E;
  return (int)launch_chain(k_unsort_rows<T_, E>, dim3(blocks_of(p.T * pieces, kRowThreads)), dim3(kRowThreads), 0, st, (const T_*)p.rows, p.rows_stride,
                           p.n_rows, p.row_of, p.weights, p.T, p.K, pieces, (T_*)p.y, p.y_stride);
}

template <class T_, int E>
int launch_unsort_back(const UnsortParams& p, const int32_t* valid, void* drows, float* dweights, cudaStream_t st) {
  const int64_t pieces = p.cols / E;
  return (int)launch_chain(k_unsort_backward<T_, E>, dim3(blocks_of(p.T, kRowThreads / 32)), dim3(kRowThreads), 0, st, (const T_*)p.y, p.y_stride,
                           (const T_*)p.rows, p.rows_stride, p.row_of, p.weights, p.T, p.K, pieces, valid, (T_*)drows, dweights);
}

bool on16(const void* p, int64_t stride_bytes) { return (((uintptr_t)p | (uintptr_t)stride_bytes) & 15) == 0; }

}  // namespace

int64_t route_sort_workspace_bytes(int64_t total, int E) {
  const int64_t chunks = (total + kOrdThreads - 1) / kOrdThreads;
  return chunks <= kOrdFusedChunks ? 0 : (chunks + 1) * (E + 1) * 4;
}

int launch_route_sort(const int32_t* ids, int64_t stride, int64_t T, int K, int E, int32_t* offsets, int32_t* row_of, int32_t* route_of_row, void* workspace,
                      cudaStream_t st) {
  const OrderView v{ids, stride, T * K, K, E};
  const int nb = E + 1, smem = ord_smem(nb), chunks = (int)((v.total + kOrdThreads - 1) / kOrdThreads);
  const int bits = 32 - __builtin_clz((unsigned)nb - 1);
  int32_t* counts = (int32_t*)workspace;
  static SmemOptIn opt_hist, opt0, opt1, opt2;
  const int most = ord_smem(kOrderMaxExperts + 1);
  const dim3 grid((unsigned)(chunks ? chunks : 1)), block(kOrdThreads);
  if (chunks <= kOrdFusedChunks) {
    if (int e = opt0.ensure(k_order_scatter<0>, most)) return e;
    return (int)launch_chain(k_order_scatter<0>, grid, block, smem, st, v, bits, counts, chunks, offsets, row_of, route_of_row);
  }
  if (int e = opt_hist.ensure(k_order_hist, most)) return e;
  if (int e = (int)launch_chain(k_order_hist, grid, block, smem, st, v, bits, counts)) return e;
  if (chunks <= kOrdDirectChunks) {
    if (int e = opt1.ensure(k_order_scatter<1>, most)) return e;
    return (int)launch_chain(k_order_scatter<1>, grid, block, smem, st, v, bits, counts, chunks, offsets, row_of, route_of_row);
  }
  if (int e = (int)launch_chain(k_order_scan, dim3((unsigned)((nb + 127) / 128)), dim3(128), 0, st, counts, chunks, nb)) return e;
  if (int e = opt2.ensure(k_order_scatter<2>, most)) return e;
  return (int)launch_chain(k_order_scatter<2>, grid, block, smem, st, v, bits, counts, chunks, offsets, row_of, route_of_row);
}

int launch_sort_rows(const void* x, int64_t x_stride, int64_t T, int64_t row_bytes, const int32_t* row_of, int K, const int32_t* valid, void* rows,
                     cudaStream_t st) {
  if (!T || !row_bytes) return 0;
  const uintptr_t all = (uintptr_t)x | (uintptr_t)rows | (uintptr_t)x_stride | (uintptr_t)row_bytes;
  if (all % 16 == 0) return launch_sort<uint32_t, 4>(x, x_stride, T, row_bytes, row_of, K, valid, rows, st);
  if (all % 4 == 0) return launch_sort<uint32_t, 1>(x, x_stride, T, row_bytes, row_of, K, valid, rows, st);
  if (all % 2 == 0) return launch_sort<uint16_t, 1>(x, x_stride, T, row_bytes, row_of, K, valid, rows, st);
  return launch_sort<uint8_t, 1>(x, x_stride, T, row_bytes, row_of, K, valid, rows, st);
}

int launch_unsort_rows(const UnsortParams& p, cudaStream_t st) {
  if (!p.T || !p.cols) return 0;
  const int64_t size = p.dtype == kF32 ? 4 : 2;
  const bool vec = p.cols * size % 16 == 0 && on16(p.rows, p.rows_stride * size) && on16(p.y, p.y_stride * size);
  if (p.dtype == kBf16) return vec ? launch_unsort<__nv_bfloat16, 8>(p, st) : launch_unsort<__nv_bfloat16, 1>(p, st);
  if (p.dtype == kF16) return vec ? launch_unsort<__half, 8>(p, st) : launch_unsort<__half, 1>(p, st);
  return vec ? launch_unsort<float, 4>(p, st) : launch_unsort<float, 1>(p, st);
}

int launch_unsort_backward(const UnsortParams& p, const int32_t* valid, void* drows, float* dweights, cudaStream_t st) {
  if (!p.T || !p.cols) return 0;
  const int64_t size = p.dtype == kF32 ? 4 : 2;
  const bool vec = p.cols * size % 16 == 0 && on16(p.rows, p.rows_stride * size) && on16(p.y, p.y_stride * size) && on16(drows, 0);
  if (p.dtype == kBf16) return vec ? launch_unsort_back<__nv_bfloat16, 8>(p, valid, drows, dweights, st) : launch_unsort_back<__nv_bfloat16, 1>(p, valid, drows, dweights, st);
  if (p.dtype == kF16) return vec ? launch_unsort_back<__half, 8>(p, valid, drows, dweights, st) : launch_unsort_back<__half, 1>(p, valid, drows, dweights, st);
  return vec ? launch_unsort_back<float, 4>(p, valid, drows, dweights, st) : launch_unsort_back<float, 1>(p, valid, drows, dweights, st);
}

}  // namespace b200
