// What the kernels of the 8-bit GEMM share (gemm_8bit.cu, gemm_8bit_clusters.cuh): instructions, the tiles of a call and who takes them, the way of
// an accumulator into the output.
#pragma once
#include <cuda_fp16.h>

#include "kernels.cuh"
#include "ptx.cuh"

namespace b200 {

namespace {

constexpr int kG8EpiWarps = 8;
constexpr int kG8Threads = 32 * (2 + kG8EpiWarps);
constexpr int kG8Group = 8;                                  // token tiles of a raster group (dense)

__host__ __device__ constexpr int g8_table_bytes(int experts) { return experts ? 4 * (3 * experts + 2) : 0; }

// MT = most tokens of a tile. kDeep: one block has an SM's shared memory, otherwise two share it (and its TMEM).
// A stage holds KC steps of 128 bytes of K. A step of few tokens takes the tensor core 128 cycles (its 16 KB of weights at 128 bytes a cycle), and
// the MMA thread's wait and commit about as many: two steps per stage where a long loop of them is the time (16 x 4096 x 7168 12.4 -> 10.3 us,
// 64 rows 13.1 -> 12.0; four steps leave too few stages: 13.0, 14.4; 128 rows, three stages, 14.8 -> 15.7; narrower tiles of 32 or 64
// weight rows, which read less per step, take the same time).
template <int MT, bool kDeep = false>
struct G8Cfg {
  static constexpr int KC = kDeep && MT <= 64 ? 2 : 1;
  static constexpr int kWStep = 128 * 128, kXStep = MT * 128;
  static constexpr int kWBytes = KC * kWStep, kXBytes = KC * kXStep, kStageBytes = kWBytes + kXBytes;
  static constexpr int kStages = kDeep ? (MT == 16 ? 5 : MT == 64 ? 4 : 6) : (MT == 16 ? 5 : MT == 64 ? 4 : 3);
  static constexpr int kTmemCols = 2 * MT;
  static constexpr int kBlocksPerSm = kDeep ? 1 : 2;
  static constexpr int kBarBytes = 256;
  static constexpr int smem(int experts) { return kStages * kStageBytes + 1024 + kBarBytes + g8_table_bytes(experts); }
};

template <bool kInt>
DEV void mma_8bit(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  if (kInt)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// Instruction descriptor: signed 8-bit operands and an int32 accumulator (kind::i8), or E4M3 operands (format 0) and fp32 (kind::f8f6f4);
// both K-major, N >> 3 in [17,23), M >> 4 in [24,29).
template <bool kInt>
DEV constexpr uint32_t idesc_8bit(int m, int n) {
  return (kInt ? (2u << 4) | (1u << 7) | (1u << 10) : (1u << 4)) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

template <bool kInt>
DEV float acc_value(float raw) { return kInt ? __int2float_rn(__float_as_int(raw)) : raw; }

template <class O>
DEV O out_value(float v);
template <>
DEV float out_value<float>(float v) { return v; }
template <>
DEV __half out_value<__half>(float v) { return __float2half_rn(v); }
template <>
DEV __nv_bfloat16 out_value<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

DEV void store_out(void* out, int64_t at, float v, int out_type) {
  if (out_type == kBf16) reinterpret_cast<__nv_bfloat16*>(out)[at] = out_value<__nv_bfloat16>(v);
  else if (out_type == kF16) reinterpret_cast<__half*>(out)[at] = out_value<__half>(v);
  else reinterpret_cast<float*>(out)[at] = v;
}

// One channel (a lane) of kCols tokens: the values first, without a branch among them, then the stores.
template <class O, int kCols>
DEV void store_tokens(const float (&v)[32], void* out, int64_t at, int64_t stride, bool live, int cols) {
  O o[kCols];
#pragma unroll
  for (int j = 0; j < kCols; ++j) o[j] = out_value<O>(v[j]);
  O* dst = reinterpret_cast<O*>(out) + at;
  if (!live) return;
  if (cols >= kCols) {
#pragma unroll
    for (int j = 0; j < kCols; ++j, dst += stride) *dst = o[j];
  } else {
#pragma unroll
    for (int j = 0; j < kCols; ++j, dst += stride)
      if (j < cols) *dst = o[j];
  }
}

// One tile of the output.
struct G8Item {
  int64_t row0;     // first token
  int rows;         // tokens, 1..MT
  int wrow0;        // first weight row of the map
  int n0, expert;   // first channel, expert
};

// Device tables of a grouped call: first row of every segment [experts + 1], cut to the rows there are and to ascending order; the experts
// by the size of their tiles, largest first [experts]; and the token tiles of the experts before each one in that order [experts + 1].
struct G8Tables {
  const int *off, *order, *tiles;
};

// Tiles of a segment, all of one size (a multiple of 32 but for the last).
template <int MT>
DEV int g8_cuts(int rows) { return (rows + MT - 1) / MT; }
template <int MT>
DEV int g8_tile_rows(int rows) {
  const int cuts = g8_cuts<MT>(rows);
  return cuts > 1 ? min(MT, ((rows + cuts - 1) / cuts + 31) & ~31) : rows;
}

// Tile t of a dense call: token tiles in groups of kG8Group, fastest inside a group, so that what runs at once is a compact block of the output.
template <int MT, int BN = 128>
DEV G8Item g8_dense_item(const Gemm8Params& p, int64_t t, int n_nt) {
  G8Item it;
  const int64_t n_mt = (p.M + MT - 1) / MT, per = (int64_t)kG8Group * n_nt, g = t / per, r = t - g * per;
  const int64_t rows = min((int64_t)kG8Group, n_mt - g * kG8Group);
  const int64_t mt = g * kG8Group + r % rows;
  it.n0 = (int)(r / rows) * BN;
  it.row0 = mt * MT;
  it.rows = (int)min((int64_t)MT, p.M - it.row0);
  it.expert = 0;
  it.wrow0 = it.n0;
  return it;
}

// The tiles worker, worker + workers, ... of the call; every role of a worker (a block, or a pair of them) walks them by itself. Grouped:
// channels fastest, so that neighbours read the same tokens and an expert's weights are in use by its token tiles at one time; segments cut
// into tiles of like size, and experts with large tiles first, so that the tiles of a round cost the same and the last round is short
// (tiles of 256 rows and a rest each, in the experts' order: 65536 rows of 128 experts x 1536 x 2048 205 us).
template <int MT, int BN = 128>
struct G8Walk {
  int64_t t, items;
  int step, n_nt;
  DEV G8Walk(const Gemm8Params& p, const G8Tables& tb, int worker, int workers) {
    n_nt = (p.N - 1) / BN + 1;
    t = worker;
    step = workers;
    items = (p.experts ? (int64_t)tb.tiles[p.experts] : ((int64_t)p.M + MT - 1) / MT) * n_nt;
  }
  DEV bool next(const Gemm8Params& p, const G8Tables& tb, G8Item& it) {
    if (t >= items) return false;
    if (!p.experts) {
      it = g8_dense_item<MT, BN>(p, t, n_nt);
    } else {
      const int mt = (int)(t / n_nt);
      int lo = 0, hi = p.experts;                            // last place with tiles[place] <= mt: the one that holds it (empty segments have none)
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (tb.tiles[mid] <= mt) lo = mid; else hi = mid;
      }
      it.expert = tb.order[lo];
      const int first = tb.off[it.expert], rows = tb.off[it.expert + 1] - first, size = g8_tile_rows<MT>(rows), at = (mt - tb.tiles[lo]) * size;
      it.row0 = first + at;
      it.rows = min(size, rows - at);
      it.n0 = (int)(t - (int64_t)mt * n_nt) * BN;
      it.wrow0 = it.expert * p.N + it.n0;
    }
    t += step;
    return true;
  }
};

// Operand maps of the tokens with boxes of 16, 32, 64 and 128 rows: a copy fetches the rows that its tile has, rounded up to a box.
struct TokenMaps {
  CUtensorMap m[4];
};
__host__ DEV int g8_box(int rows) { return rows <= 16 ? 0 : rows <= 32 ? 1 : rows <= 64 ? 2 : 3; }

// Fills the tables, by the whole block; the caller synchronises.
template <int MT>
DEV void g8_tables(const Gemm8Params& p, int* off, int* order, int* tiles) {
  constexpr int kClasses = (MT + 31) / 32;                   // of tile sizes
  __shared__ int s_class[kClasses];
  const int lane = threadIdx.x & 31, warp = warp_uniform();
  for (int e = threadIdx.x; e <= p.experts; e += kG8Threads) off[e] = min(max(__ldg(p.offsets + e), 0), (int)p.M);
  __syncthreads();
  if (warp == 2) {
    int most = 0;                                            // ascending whatever the caller's offsets are
    for (int e0 = 0; e0 <= p.experts; e0 += 32) {
      const int e = e0 + lane;
      int v = max(e <= p.experts ? off[e] : 0, most);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xFFFFFFFFu, v, o);
        if (lane >= o) v = max(v, u);
      }
      if (e <= p.experts) off[e] = v;
      most = __shfl_sync(0xFFFFFFFFu, v, 31);
    }
  }
  __syncthreads();
  // a stable counting sort of the experts by class, one warp per class: warp 0 the largest tiles; empty segments are with the smallest
  const int cls = kClasses - 1 - warp;
  for (int pass = 0; pass < 2; ++pass) {
    if (cls >= 0) {
      int place = 0;
      if (pass) for (int c = kClasses - 1; c > cls; --c) place += s_class[c];
      for (int e0 = 0; e0 < p.experts; e0 += 32) {
        const int e = e0 + lane, rows = e < p.experts ? off[e + 1] - off[e] : 0;
        const bool mine = e < p.experts && max((g8_tile_rows<MT>(rows) + 31) / 32 - 1, 0) == cls;
        const unsigned who = __ballot_sync(0xFFFFFFFFu, mine);
        if (pass && mine) order[place + __popc(who & ((1u << lane) - 1))] = e;
        place += __popc(who);
      }
      if (!pass && lane == 0) s_class[cls] = place;
    }
    __syncthreads();
  }
  if (warp != 2) return;
  int sum = 0;
  for (int e0 = 0; e0 < p.experts; e0 += 32) {
    const int i = e0 + lane, e = i < p.experts ? order[i] : 0;
    int v = i < p.experts ? g8_cuts<MT>(off[e + 1] - off[e]) : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xFFFFFFFFu, v, o);
      if (lane >= o) v += u;
    }
    if (i < p.experts) tiles[i + 1] = sum + v;
    sum += __shfl_sync(0xFFFFFFFFu, v, 31);
  }
  if (lane == 0) tiles[0] = 0;
}

// Rows of no segment, of an output that this call made; `w` of kG8EpiWarps warps of a block.
DEV void g8_zero_rest(const Gemm8Params& p, const int* off, int w, int lane) {
  const int64_t before = off[0], behind = off[p.experts], rest = before + (p.M - behind);
  for (int64_t r = (int64_t)blockIdx.x * kG8EpiWarps + w; r < rest; r += (int64_t)gridDim.x * kG8EpiWarps) {
    const int64_t row = r < before ? r : behind + (r - before);
    for (int n = lane; n < p.N; n += 32) store_out(p.out, row * p.out_stride + n, 0.f, p.out_type);
  }
}

// Half (of the column pairs) of an accumulator: TMEM -> scaled values of this lane's channel n -> output. s_sa: 32 floats of the warp's own.
template <bool kInt, int MT>
DEV void g8_store_tile(const Gemm8Params& p, const G8Item& it, int n, bool live, float sb, uint32_t taddr, int half, float* s_sa) {
  constexpr int kCols = MT < 32 ? MT : 32;
  const int lane = threadIdx.x & 31;
  for (int col = half * kCols; col < it.rows; col += 2 * kCols) {
    float v[32];
    if constexpr (MT >= 32) tmem_ld32(taddr + col, v); else tmem_ld16(taddr + col, v);
    const float sa = lane < it.rows - col ? __ldg(p.a_scale + it.row0 + col + lane) : 0.f;
    __syncwarp();
    s_sa[lane] = sa;                                         // read back four at a time by every lane
    __syncwarp();
    tmem_ld_wait();
#pragma unroll
    for (int j = 0; j < kCols; j += 4) {
      const float4 s = *reinterpret_cast<const float4*>(s_sa + j);
      v[j] = acc_value<kInt>(v[j]) * s.x * sb;
      v[j + 1] = acc_value<kInt>(v[j + 1]) * s.y * sb;
      v[j + 2] = acc_value<kInt>(v[j + 2]) * s.z * sb;
      v[j + 3] = acc_value<kInt>(v[j + 3]) * s.w * sb;
    }
    const int64_t at = (it.row0 + col) * p.out_stride + n;
    if (p.out_type == kBf16) store_tokens<__nv_bfloat16, kCols>(v, p.out, at, p.out_stride, live, it.rows - col);
    else if (p.out_type == kF16) store_tokens<__half, kCols>(v, p.out, at, p.out_stride, live, it.rows - col);
    else store_tokens<float, kCols>(v, p.out, at, p.out_stride, live, it.rows - col);
  }
}

}  // namespace

}  // namespace b200
