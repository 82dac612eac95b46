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
// The row kernels are bound by HBM (8192 x 8 routes, 2048 wide bf16: sort 50 us = 6.0 TB/s, mostly writes; unsort 50 = 6.0; gradient 102 = 5.6), the
// order by the latency of its one or two launches (64 routes 3 us, 65536 10).
#include <algorithm>

#include "kernels.cuh"
#include "rows.cuh"

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
  const int64_t t = (uint32_t)f / (uint32_t)v.K;             // fewer than 2^31 routes
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
        for (int c0 = 0; c0 < chunks; c0 += 32) {            // 32 counts in flight: their latency is most of this kernel's time
          int n[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) n[i] = c0 + i < chunks ? __ldg(counts + (int64_t)(c0 + i) * nb + e) : 0;
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            if (c0 + i == (int)blockIdx.x) mine = sum;
            sum += n[i];
          }
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
// A token's row is `pieces` vectors of 16 bytes. Rows on 16-byte boundaries are read and written as they are. Others (kAny) are cut where the vectors
// of the row that is WRITTEN lie: its aligned vectors are filled from source vectors that are shifted into place (Any16), and up to 15
// bytes at either end go element by element, by the first 32 threads of the token.
constexpr int kRowThreads = 256;

// `lanes` consecutive threads of the grid share a token. The division by lanes is a multiplication (n / d for n < 2^31: Granlund and Montgomery,
// "Division by invariant integers using multiplication", 1994).
struct Spread {
  uint32_t lanes, mul, shift;
  int64_t t;
  uint32_t lane;
  DEV void place() {
    const uint32_t i = blockIdx.x * kRowThreads + threadIdx.x, q = (__umulhi(mul, i) + i) >> shift;
    t = q;
    lane = i - q * lanes;
  }
};

// How a row of `bytes` that starts at `at` is written: `head` bytes, whole vectors, the rest.
struct Cut {
  int head, pieces, tail;
  DEV Cut(const void* at, int bytes) {
    head = min((int)(-(uint32_t)(uintptr_t)at & 15u), bytes);
    pieces = (bytes - head) >> 4;
    tail = head + 16 * pieces;
  }
  // byte of the element that thread `lane` has at the ends, or -1
  template <class T>
  DEV int edge(int lane, int bytes) const {
    if (lane >= 32) return -1;
    const int b = (lane & 15) * (int)sizeof(T) + (lane < 16 ? 0 : tail);
    return b < (lane < 16 ? head : bytes) ? b : -1;
  }
};

// Zeros in the rows behind the last route, one run of bytes: vectors dealt to all threads of the grid, elements of T at its ends.
template <class T>
DEV void zero_behind(uint8_t* rows, int row_bytes, const int32_t* valid, int64_t n_rows) {
  const int64_t first = min(max((int64_t)__ldg(valid), (int64_t)0), n_rows);
  if (first == n_rows) return;
  uint8_t* at = rows + first * row_bytes;
  const int64_t bytes = (n_rows - first) * row_bytes, head = min((int64_t)(-(uint32_t)(uintptr_t)at & 15u), bytes), pieces = (bytes - head) >> 4;
  for (int64_t i = (int64_t)blockIdx.x * kRowThreads + threadIdx.x; i < pieces; i += (int64_t)gridDim.x * kRowThreads)
    reinterpret_cast<uint4*>(at + head)[i] = make_uint4(0u, 0u, 0u, 0u);
  if (blockIdx.x == 0 && threadIdx.x < 32) {
    const int64_t b = (int64_t)(threadIdx.x & 15) * (int)sizeof(T) + (threadIdx.x < 16 ? 0 : head + 16 * pieces);
    if (b < (threadIdx.x < 16 ? head : bytes)) *reinterpret_cast<T*>(at + b) = 0;
  }
}

template <class T>
struct Bits;                 // an unsigned integer as wide as T
template <>
struct Bits<__half> { using type = uint16_t; };
template <>
struct Bits<__nv_bfloat16> { using type = uint16_t; };
template <>
struct Bits<float> { using type = uint32_t; };

// A thread has N pieces of one token, lanes apart: read once, written to the token's K rows (kAny: read for each row, from L1).
template <class U, int N, bool kAny>
__global__ void __launch_bounds__(kRowThreads) k_sort_rows(const uint8_t* __restrict__ x, int64_t x_stride, int64_t T, int row_bytes, Spread sp,
                                                           const int32_t* __restrict__ row_of, int K, const int32_t* __restrict__ valid,
                                                           uint8_t* __restrict__ rows) {
  pdl_trigger();
  pdl_wait();
  sp.place();
  const int64_t n_rows = T * K, t = sp.t;
  if (t < T) {
    const uint8_t* from = x + t * x_stride;
    const int lane = (int)sp.lane, all = (int)sp.lanes;
    if constexpr (!kAny) {
      for (int i = lane; i * 16 < row_bytes; i += N * all) {
        uint4 v[N];
#pragma unroll
        for (int j = 0; j < N; ++j)
          if ((i + j * all) * 16 < row_bytes) v[j] = __ldg(reinterpret_cast<const uint4*>(from) + i + j * all);
        for (int k = 0; k < K; ++k) {
          const int row = __ldg(row_of + t * K + k);
          if ((uint32_t)row >= (uint64_t)n_rows) continue;
          uint4* dst = reinterpret_cast<uint4*>(rows + (int64_t)row * row_bytes);
#pragma unroll
          for (int j = 0; j < N; ++j)
            if ((i + j * all) * 16 < row_bytes) dst[i + j * all] = v[j];
        }
      }
    } else {
      const Span sx{x, x + (T - 1) * x_stride + row_bytes, from - 15 >= x && from + row_bytes + 32 <= x + (T - 1) * x_stride + row_bytes};
      for (int k = 0; k < K; ++k) {
        const int row = __ldg(row_of + t * K + k);
        if ((uint32_t)row >= (uint64_t)n_rows) continue;
        uint8_t* dst = rows + (int64_t)row * row_bytes;
        const Cut cut(dst, row_bytes);
        for (int i = lane; i < cut.pieces; i += all) {
          Any16<U> f;
          f.fetch(from + cut.head + 16 * i, sx, true);
          reinterpret_cast<uint4*>(dst + cut.head)[i] = f.take(from + cut.head + 16 * i, sx);
        }
        const int b = cut.template edge<U>(lane, row_bytes);
        if (b >= 0) *reinterpret_cast<U*>(dst + b) = *reinterpret_cast<const U*>(from + b);
      }
    }
  }
  zero_behind<U>(rows, row_bytes, valid, n_rows);
}

// The span of a tensor for each of its rows: every row but the first and the last has its neighbours around it.
template <class T>
struct RowSpans {
  const uint8_t *lo, *hi;
  int64_t last;
  DEV RowSpans(const void* p, int64_t rows, int64_t stride, int64_t cols) {
    lo = (const uint8_t*)p;
    hi = lo + ((rows - 1) * stride + cols) * (int64_t)sizeof(T);
    last = stride >= cols && cols * (int64_t)sizeof(T) >= 32 ? rows - 1 : 0;
  }
  DEV Span of(int64_t row) const { return {lo, hi, row > 0 && row < last}; }
};

// Rows of a few elements (scales): a thread per route.
template <class U>
__global__ void __launch_bounds__(kRowThreads) k_sort_short(const uint8_t* __restrict__ x, int64_t x_stride, int64_t T, int row_bytes,
                                                            const int32_t* __restrict__ row_of, int K, const int32_t* __restrict__ valid,
                                                            uint8_t* __restrict__ rows) {
  pdl_trigger();
  pdl_wait();
  const int64_t n_rows = T * K, i = (int64_t)blockIdx.x * kRowThreads + threadIdx.x;
  if (i < n_rows) {
    const int row = __ldg(row_of + i);
    const uint8_t* from = x + (int64_t)((uint32_t)i / (uint32_t)K) * x_stride;
    if ((uint32_t)row < (uint64_t)n_rows)
      for (int b = 0; b < row_bytes; b += (int)sizeof(U)) *reinterpret_cast<U*>(rows + (int64_t)row * row_bytes + b) = __ldg(reinterpret_cast<const U*>(from + b));
  }
  zero_behind<U>(rows, row_bytes, valid, n_rows);
}

// Rows and weights of up to S slots.
template <int S>
struct Slots {
  int row[S];
  float w[S];
  DEV Slots(const int32_t* row_of, const float* weights, int64_t t, int K, int k0, int64_t n_rows) {
#pragma unroll
    for (int j = 0; j < S; ++j) {
      row[j] = k0 + j < K ? __ldg(row_of + t * K + k0 + j) : -1;
      w[j] = weights && k0 + j < K ? __ldg(weights + t * K + k0 + j) : 1.f;
    }
#pragma unroll
    for (int j = 0; j < S; ++j)
      if ((uint32_t)row[j] >= (uint64_t)n_rows) row[j] = -1;
  }
};

// y[t]: a thread has N pieces of a token, and the rows of S slots in flight for them: eight vectors, or four that are shifted.
template <class T_, int S, int N, bool kAny>
__global__ void __launch_bounds__(kRowThreads) k_unsort_rows(const UnsortParams p, Spread sp) {
  constexpr int E = Vec<T_>::E;
  pdl_trigger();
  pdl_wait();
  sp.place();
  const int64_t t = sp.t;
  if (t >= p.T) return;
  const T_* rows = (const T_*)p.rows;
  T_* y = (T_*)p.y + t * p.y_stride;
  const int lane = (int)sp.lane, all = (int)sp.lanes, bytes = (int)p.cols * (int)sizeof(T_);
  const Cut cut = kAny ? Cut(y, bytes) : Cut(nullptr, bytes);
  const RowSpans<T_> sr(p.rows, p.n_rows, p.rows_stride, p.cols);
  for (int i = lane; i < cut.pieces; i += N * all) {
    float acc[N][E];
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int e = 0; e < E; ++e) acc[n][e] = 0.f;
    for (int k0 = 0; k0 < p.K; k0 += S) {
      const Slots<S> s(p.row_of, p.weights, t, p.K, k0, p.n_rows);
      Fetch16<T_, kAny> f[S][N];
#pragma unroll
      for (int j = 0; j < S; ++j)
#pragma unroll
        for (int n = 0; n < N; ++n) {
          const int at = i + n * all;
          f[j][n].fetch(reinterpret_cast<const uint8_t*>(rows + (int64_t)max(s.row[j], 0) * p.rows_stride) + cut.head + 16 * at,
                        sr.of(s.row[j]), s.row[j] >= 0 && (N == 1 || at < cut.pieces));
        }
#pragma unroll
      for (int j = 0; j < S; ++j) {
        if (s.row[j] < 0) continue;
#pragma unroll
        for (int n = 0; n < N; ++n) {
          Vec<T_> v;
          v.raw = f[j][n].take(reinterpret_cast<const uint8_t*>(rows + (int64_t)s.row[j] * p.rows_stride) + cut.head + 16 * (i + n * all), sr.of(s.row[j]));
#pragma unroll
          for (int e = 0; e < E; ++e) acc[n][e] = fmaf(to_f32(v.v[e]), s.w[j], acc[n][e]);
        }
      }
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int at = i + n * all;
      if (N > 1 && at >= cut.pieces) continue;
      Vec<T_> o;
#pragma unroll
      for (int e = 0; e < E; ++e) o.v[e] = from_f32<T_>(acc[n][e]);
      reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(y) + cut.head)[at] = o.raw;
    }
  }
  if constexpr (kAny) {
    const int b = cut.template edge<T_>(lane, bytes);
    if (b >= 0) {
      const int c = b / (int)sizeof(T_);
      float acc = 0.f;
      for (int k0 = 0; k0 < p.K; k0 += S) {
        const Slots<S> s(p.row_of, p.weights, t, p.K, k0, p.n_rows);
        T_ v[S];
#pragma unroll
        for (int j = 0; j < S; ++j) v[j] = s.row[j] >= 0 ? rows[(int64_t)s.row[j] * p.rows_stride + c] : from_f32<T_>(0.f);
#pragma unroll
        for (int j = 0; j < S; ++j)
          if (s.row[j] >= 0) acc = fmaf(to_f32(v[j]), s.w[j], acc);
      }
      y[c] = from_f32<T_>(acc);
    }
  }
}

// One warp per token, or one block (kBlock: few tokens with long rows). A piece of dy is read once for four of the token's rows; their dot
// products stay in registers until the row's end.
template <class T_, bool kAny, bool kBlock>
__global__ void __launch_bounds__(kRowThreads) k_unsort_backward(const UnsortParams p, const int32_t* __restrict__ valid, T_* __restrict__ drows,
                                                                 float* __restrict__ dweights) {
  constexpr int E = Vec<T_>::E, kSlots = 4, kWarps = kRowThreads / 32;
  __shared__ float part[kWarps][kSlots];
  pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x >> 5;
  const int lane = kBlock ? (int)threadIdx.x : (int)threadIdx.x & 31, all = kBlock ? kRowThreads : 32;
  const int64_t t = kBlock ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * kWarps + warp;
  const int bytes = (int)p.cols * (int)sizeof(T_);
  const T_* rows = (const T_*)p.rows;
  const T_* dy = (const T_*)p.y + t * p.y_stride;
  const RowSpans<T_> rows_of(p.rows, p.n_rows, p.rows_stride, p.cols), grads_of(p.y, p.T, p.y_stride, p.cols);
  const Span sd = grads_of.of(t);
  if (t < p.T) {
    for (int k0 = 0; k0 < p.K; k0 += kSlots) {
      int row[kSlots];
      float w[kSlots], dot[kSlots];
#pragma unroll
      for (int j = 0; j < kSlots; ++j) {
        row[j] = k0 + j < p.K ? __ldg(p.row_of + t * p.K + k0 + j) : -1;
        w[j] = p.weights && k0 + j < p.K ? __ldg(p.weights + t * p.K + k0 + j) : 1.f;
        if ((uint32_t)row[j] >= (uint64_t)p.n_rows) row[j] = -1;
        dot[j] = 0.f;
      }
      if constexpr (!kAny) {
        for (int i = lane; i * 16 < bytes; i += all) {
          Vec<T_> g, v[kSlots];
          g.raw = __ldg(reinterpret_cast<const uint4*>(dy) + i);
          if (dweights) {
#pragma unroll
            for (int j = 0; j < kSlots; ++j)
              if (row[j] >= 0) v[j].raw = __ldg(reinterpret_cast<const uint4*>(rows + (int64_t)row[j] * p.rows_stride) + i);
          }
#pragma unroll
          for (int j = 0; j < kSlots; ++j) {
            if (row[j] < 0) continue;
            if (dweights) {
#pragma unroll
              for (int e = 0; e < E; ++e) dot[j] = fmaf(to_f32(v[j].v[e]), to_f32(g.v[e]), dot[j]);
            }
            if (drows) {
              Vec<T_> o;
#pragma unroll
              for (int e = 0; e < E; ++e) o.v[e] = from_f32<T_>(to_f32(g.v[e]) * w[j]);
              reinterpret_cast<uint4*>(drows + (int64_t)row[j] * p.cols)[i] = o.raw;
            }
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < kSlots; ++j) {
          if (row[j] < 0) continue;
          uint8_t* dst = reinterpret_cast<uint8_t*>(drows + (int64_t)row[j] * p.cols);        // its phase, without gradients of rows as well
          const uint8_t *from = reinterpret_cast<const uint8_t*>(rows + (int64_t)row[j] * p.rows_stride), *grad = reinterpret_cast<const uint8_t*>(dy);
          const Cut cut(dst, bytes);
          const Span sr = rows_of.of(row[j]);
          for (int i = lane; i < cut.pieces; i += all) {
            const int at = cut.head + 16 * i;
            Any16<T_> fg, fv;
            fg.fetch(grad + at, sd, true);
            fv.fetch(from + at, sr, dweights);
            Vec<T_> g, v, o;
            g.raw = fg.take(grad + at, sd);
            if (dweights) {
              v.raw = fv.take(from + at, sr);
#pragma unroll
              for (int e = 0; e < E; ++e) dot[j] = fmaf(to_f32(v.v[e]), to_f32(g.v[e]), dot[j]);
            }
            if (drows) {
#pragma unroll
              for (int e = 0; e < E; ++e) o.v[e] = from_f32<T_>(to_f32(g.v[e]) * w[j]);
              *reinterpret_cast<uint4*>(dst + at) = o.raw;
            }
          }
          const int b = cut.template edge<T_>(lane, bytes);
          if (b >= 0) {
            const int c = b / (int)sizeof(T_);
            const float g = to_f32(dy[c]);
            if (dweights) dot[j] = fmaf(to_f32(rows[(int64_t)row[j] * p.rows_stride + c]), g, dot[j]);
            if (drows) drows[(int64_t)row[j] * p.cols + c] = from_f32<T_>(g * w[j]);
          }
        }
      }
      if (dweights) {
#pragma unroll
        for (int j = 0; j < kSlots; ++j) {
#pragma unroll
          for (int o = 16; o; o >>= 1) dot[j] += __shfl_xor_sync(0xFFFFFFFFu, dot[j], o);
        }
        if constexpr (kBlock) {
          __syncthreads();
          if ((threadIdx.x & 31) == 0) {
#pragma unroll
            for (int j = 0; j < kSlots; ++j) part[warp][j] = dot[j];
          }
          __syncthreads();
#pragma unroll
          for (int j = 0; j < kSlots; ++j) {
            dot[j] = part[0][j];
#pragma unroll
            for (int i = 1; i < kWarps; ++i) dot[j] += part[i][j];
          }
        }
        if (lane == 0) {
#pragma unroll
          for (int j = 0; j < kSlots; ++j)
            if (k0 + j < p.K) dweights[t * p.K + k0 + j] = row[j] >= 0 ? dot[j] : 0.f;
        }
      }
    }
  }
  if (drows) zero_behind<typename Bits<T_>::type>(reinterpret_cast<uint8_t*>(drows), bytes, valid, p.n_rows);
}

unsigned blocks_of(int64_t n, int64_t per) { return (unsigned)((n + per - 1) / per); }

// `threads` for each of T tokens, fewer where the grid's threads would pass 2^31 (a thread then takes more pieces), but not below the 32 that
// write a row's ends: 32 for each of 2^26 - 1 tokens still fit.
Spread spread(int64_t threads, int64_t T) {
  while (threads > 32 && threads * T > INT32_MAX - kRowThreads) threads = std::max<int64_t>(32, (threads + 1) / 2);
  Spread s{};
  s.lanes = (uint32_t)threads;
  while ((1ull << s.shift) < (uint64_t)threads) ++s.shift;
  s.mul = (uint32_t)(((1ull << 32) * ((1ull << s.shift) - (uint64_t)threads)) / (uint64_t)threads + 1);
  return s;
}
dim3 grid_of(const Spread& s, int64_t T) { return dim3(blocks_of(T * s.lanes, kRowThreads)); }

template <class U, bool kAny>
int launch_sort(const void* x, int64_t x_stride, int64_t T, int row_bytes, const int32_t* row_of, int K, const int32_t* valid, void* rows, cudaStream_t st) {
  if (kAny && row_bytes < 32)
    return (int)launch_chain(k_sort_short<U>, dim3(blocks_of(T * K, kRowThreads)), dim3(kRowThreads), 0, st, (const uint8_t*)x, x_stride, T, row_bytes, row_of, K,
                             valid, (uint8_t*)rows);
  const int64_t pieces = (row_bytes + 15) / 16;
  // four pieces per thread once that still fills the device: fewer index reads for the same bytes
  const bool four = T * pieces >= 4ll * 1024 * sm_count();
  const int64_t want = four ? (pieces + 3) / 4 : pieces;
  const Spread sp = spread(kAny && want < 32 ? 32 : want, T);
  const auto kern = four && !kAny ? k_sort_rows<U, 4, kAny> : k_sort_rows<U, 1, kAny>;
  return (int)launch_chain(kern, grid_of(sp, T), dim3(kRowThreads), 0, st, (const uint8_t*)x, x_stride, T, row_bytes, sp, row_of, K, valid, (uint8_t*)rows);
}

template <class T_, int S, int N, bool kAny>
int launch_unsort_form(const UnsortParams& p, cudaStream_t st) {
  const int64_t pieces = (p.cols * (int64_t)sizeof(T_) / 16 + N - 1) / N;
  const Spread sp = spread(kAny && pieces < 32 ? 32 : pieces, p.T);
  return (int)launch_chain(k_unsort_rows<T_, S, N, kAny>, grid_of(sp, p.T), dim3(kRowThreads), 0, st, p, sp);
}
// Few slots: more pieces per thread for the same bytes in flight, while that leaves the device full.
template <class T_, bool kAny>
int launch_unsort(const UnsortParams& p, cudaStream_t st) {
  if constexpr (kAny) {
    return launch_unsort_form<T_, 4, 1, true>(p, st);
  } else {
    const bool full = p.T * p.cols * (int64_t)sizeof(T_) / 16 >= 8ll * 1024 * sm_count();
    if (p.K > 4 || !full) return launch_unsort_form<T_, 8, 1, false>(p, st);
    return p.K > 2 ? launch_unsort_form<T_, 4, 2, false>(p, st) : launch_unsort_form<T_, 2, 4, false>(p, st);
  }
}

template <class T_, bool kAny>
int launch_unsort_back(const UnsortParams& p, const int32_t* valid, void* drows, float* dweights, cudaStream_t st) {
  // a block per token while warps would leave most of the device idle
  if (p.T < 16ll * sm_count() && p.cols * (int64_t)sizeof(T_) >= 1024)
    return (int)launch_chain(k_unsort_backward<T_, kAny, true>, dim3((unsigned)p.T), dim3(kRowThreads), 0, st, p, valid, (T_*)drows, dweights);
  return (int)launch_chain(k_unsort_backward<T_, kAny, false>, dim3(blocks_of(p.T, kRowThreads / 32)), dim3(kRowThreads), 0, st, p, valid, (T_*)drows, dweights);
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
  if (all % 16 == 0) return launch_sort<uint32_t, false>(x, x_stride, T, (int)row_bytes, row_of, K, valid, rows, st);
  if (all % 4 == 0) return launch_sort<uint32_t, true>(x, x_stride, T, (int)row_bytes, row_of, K, valid, rows, st);
  if (all % 2 == 0) return launch_sort<uint16_t, true>(x, x_stride, T, (int)row_bytes, row_of, K, valid, rows, st);
  return launch_sort<uint8_t, true>(x, x_stride, T, (int)row_bytes, row_of, K, valid, rows, st);
}

int launch_unsort_rows(const UnsortParams& p, cudaStream_t st) {
  if (!p.T || !p.cols) return 0;
  const int64_t size = p.dtype == kF32 ? 4 : 2;
  const bool vec = p.cols * size % 16 == 0 && on16(p.rows, p.rows_stride * size) && on16(p.y, p.y_stride * size);
  if (p.dtype == kBf16) return vec ? launch_unsort<__nv_bfloat16, false>(p, st) : launch_unsort<__nv_bfloat16, true>(p, st);
  if (p.dtype == kF16) return vec ? launch_unsort<__half, false>(p, st) : launch_unsort<__half, true>(p, st);
  return vec ? launch_unsort<float, false>(p, st) : launch_unsort<float, true>(p, st);
}

int launch_unsort_backward(const UnsortParams& p, const int32_t* valid, void* drows, float* dweights, cudaStream_t st) {
  if (!p.T || !p.cols) return 0;
  const int64_t size = p.dtype == kF32 ? 4 : 2;
  const bool vec = p.cols * size % 16 == 0 && on16(p.rows, p.rows_stride * size) && on16(p.y, p.y_stride * size) && on16(drows, 0);
  if (p.dtype == kBf16) return vec ? launch_unsort_back<__nv_bfloat16, false>(p, valid, drows, dweights, st) : launch_unsort_back<__nv_bfloat16, true>(p, valid, drows, dweights, st);
  if (p.dtype == kF16) return vec ? launch_unsort_back<__half, false>(p, valid, drows, dweights, st) : launch_unsort_back<__half, true>(p, valid, drows, dweights, st);
  return vec ? launch_unsort_back<float, false>(p, valid, drows, dweights, st) : launch_unsort_back<float, true>(p, valid, drows, dweights, st);
}

}  // namespace b200
