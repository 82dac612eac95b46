// GEMM of 8-bit rows: out[m, n] = sa[m] * sb[n] * sum_k a[m, k] * b[n, k], int8 (exact int32 sums) or E4M3 (fp32 sums), one scale per
// token and per output channel; dense, or over the segments of tokens that are sorted by expert (one weight matrix per segment).
//
// The weights are the M side of tcgen05.mma (128 weight rows = 128 TMEM lanes), the tokens its N side, which a tile takes in steps of 16
// or 32: a tile of few tokens is no padding, and an expert's rest of rows costs what it holds. A thread of the epilogue then owns an
// output channel (one sb in a register) and a warp writes 32 consecutive channels of a token, so odd widths, strides and addresses
// need no form of their own.
// kind::i8 and kind::f8f6f4 take 32 bytes of K per instruction: a stage of 128 bytes of K is four of them, 64-byte-per-cycle operand
// reads as for any type. K beyond the last 128-byte step reads as zeros (TMA's fill), so K needs no more than 16-byte rows.
#include <cuda_fp16.h>

#include "kernels.cuh"
#include "ptx.cuh"

namespace b200 {

namespace {

constexpr int kG8EpiWarps = 8;
constexpr int kG8Threads = 32 * (2 + kG8EpiWarps);
constexpr int kG8Group = 8;                                  // token tiles of a raster group (dense)

__host__ __device__ constexpr int g8_table_bytes(int experts) { return experts ? 4 * (3 * experts + 2) : 0; }

// MT = most tokens of a tile. Up to 128 two blocks share an SM (half of its shared memory and TMEM each).
template <int MT, bool kDeep = false>
struct G8Cfg {
  static constexpr int kWBytes = 128 * 128, kXBytes = MT * 128, kStageBytes = kWBytes + kXBytes;
  static constexpr int kStages = kDeep ? (MT == 16 ? 11 : MT == 64 ? 8 : 6) : (MT == 16 ? 5 : MT == 64 ? 4 : 3);
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
DEV int g8_box(int rows) { return rows <= 16 ? 0 : rows <= 32 ? 1 : rows <= 64 ? 2 : 3; }

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

template <bool kInt, int MT, bool kDeep>
__global__ void __launch_bounds__(kG8Threads, G8Cfg<MT, kDeep>::kBlocksPerSm)
k_gemm_8bit(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ TokenMaps tm_x, const Gemm8Params p) {
  using C = G8Cfg<MT, kDeep>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t s_w = base, s_x = s_w + C::kStages * C::kWBytes;
  const uint32_t bar_full = s_x + C::kStages * C::kXBytes, bar_empty = bar_full + 8 * C::kStages;
  const uint32_t bar_acc_full = bar_empty + 8 * C::kStages, bar_acc_empty = bar_acc_full + 16, s_slot = bar_acc_empty + 16;
  int* tab = reinterpret_cast<int*>(smem_raw + (bar_full - smem_u32(smem_raw)) + C::kBarBytes);   // off[E + 1], order[E], tiles[E + 1]
  const int warp = warp_uniform(), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar_acc_full + 8 * b, 1);
      mbar_init(bar_acc_empty + 8 * b, kG8EpiWarps);
    }
    mbar_init_fence();
    tma_prefetch_desc(&tm_w);
  }
  if (warp == 1) tmem_alloc<C::kTmemCols>(s_slot);
  pdl_wait();
  int* off = tab;
  int *order = tab + p.experts + 1, *tiles = order + p.experts;
  if (p.experts) g8_tables<MT>(p, off, order, tiles);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(s_slot));

  const G8Tables tb{off, order, tiles};
  const int nk = (p.K + 127) / 128;
  G8Walk<MT> walk(p, tb, (int)blockIdx.x, (int)gridDim.x);
  G8Item it;

  if (warp == 0) {
    if (elect_one()) {
      uint32_t s = 0, ph = 1;
      bool ok = true;
      while (ok && walk.next(p, tb, it)) {
        const int box = g8_box(it.rows), bytes = 128 * 16 << box;
        for (int ks = 0; ks < nk; ++ks) {
          if (!mbar_wait(bar_empty + 8 * s, ph)) { if (p.status) atomicCAS(p.status, 0, 141); ok = false; break; }
          const uint32_t full = bar_full + 8 * s;
          mbar_expect_tx(full, C::kWBytes + bytes);
          tma_load_2d(s_w + s * C::kWBytes, &tm_w, full, ks * 128, it.wrow0);
          tma_load_2d(s_x + s * C::kXBytes, &tm_x.m[box], full, ks * 128, (int)it.row0);
          if (++s == C::kStages) { s = 0; ph ^= 1; }
        }
      }
      pdl_trigger();                                         // this block has asked for its last bytes, and holds its TMEM
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one()) {
      constexpr uint32_t kHi = (1024u >> 4) | (1u << 14) | (2u << 29);   // SBO 1024, version 1, SWIZZLE_128B
      const uint32_t w_lo0 = ((s_w >> 4) & 0x3FFF) | (1u << 16), x_lo0 = ((s_x >> 4) & 0x3FFF) | (1u << 16);
      uint32_t s = 0, ph = 0, n_it = 0;
      bool ok = true;
      for (; ok && walk.next(p, tb, it); ++n_it) {
        const uint32_t buf = n_it & 1;
        if (!mbar_wait(bar_acc_empty + 8 * buf, ((n_it >> 1) & 1) ^ 1)) { if (p.status) atomicCAS(p.status, 0, 142); break; }
        tc_fence_after();
        const uint32_t acc = tmem + buf * MT;
        const uint32_t idesc = idesc_8bit<kInt>(128, it.rows <= 16 ? 16 : (it.rows + 31) & ~31);
        for (int ks = 0; ks < nk; ++ks) {
          if (!mbar_wait(bar_full + 8 * s, ph)) { if (p.status) atomicCAS(p.status, 0, 143); ok = false; break; }
          tc_fence_after();
          const uint32_t w_lo = w_lo0 + s * (C::kWBytes >> 4), x_lo = x_lo0 + s * (C::kXBytes >> 4);
#pragma unroll
          for (int q = 0; q < 4; ++q)
            mma_8bit<kInt>(acc, ((uint64_t)kHi << 32) | (w_lo + 2 * q), ((uint64_t)kHi << 32) | (x_lo + 2 * q), idesc, (ks | q) ? 1u : 0u);
          mma_commit(bar_empty + 8 * s);
          if (++s == C::kStages) { s = 0; ph ^= 1; }
        }
        if (ok) mma_commit(bar_acc_full + 8 * buf);
      }
    }
    __syncwarp();
  } else {
    const int quad = warp & 3, half = (warp - 2) >> 2;
    __shared__ float4 s_scales[kG8EpiWarps][8];
    float* s_sa = reinterpret_cast<float*>(s_scales[warp - 2]);
    uint32_t n_it = 0;
    for (; walk.next(p, tb, it); ++n_it) {
      const uint32_t buf = n_it & 1;
      int okw = 1;
      if (lane == 0) okw = mbar_wait(bar_acc_full + 8 * buf, (n_it >> 1) & 1, nk) ? 1 : 0;
      okw = __shfl_sync(0xFFFFFFFFu, okw, 0);
      if (!okw) { if (lane == 0 && p.status) atomicCAS(p.status, 0, 144); break; }
      tc_fence_after();
      const int n = it.n0 + quad * 32 + lane;
      const bool live = n < p.N;
      const float sb = live ? __ldg(p.b_scale + (int64_t)it.expert * p.N + n) : 0.f;
      const uint32_t taddr = tmem + ((uint32_t)(quad * 32) << 16) + buf * MT;
      g8_store_tile<kInt, MT>(p, it, n, live, sb, taddr, half, s_sa);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_acc_empty + 8 * buf);
    }
    if (p.experts && p.zero_rest) g8_zero_rest(p, off, warp - 2, lane);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc<C::kTmemCols>(tmem);
  }
}

// ----------------------------------------------------------------------------- CTA pairs
// tcgen05.mma.cta_group::2 on tiles of 256 weight rows x MT tokens: each SM fetches its 128 weight rows and half of the tokens, so a tile of
// twice the work moves MT / 2 token rows less per SM than two tiles of the single kernel do (32 KB per 512 tensor cycles at MT = 256).
template <int MT>
struct G8Pair {
  static constexpr int kWBytes = 128 * 128, kXBytes = MT / 2 * 128, kStageBytes = kWBytes + kXBytes;
  static constexpr int kStages = MT == 256 ? 6 : 8;
  static_assert(MT == 128 || MT == 256, "a CTA's share of the tokens is fetched in one box");
  static constexpr int kTmemCols = 2 * MT;
  static constexpr int kBarBytes = 256;
  static constexpr int smem(int experts) { return kStages * kStageBytes + 1024 + kBarBytes + g8_table_bytes(experts); }
};

template <bool kInt>
DEV void mma_8bit_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  if (kInt)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

template <bool kInt, int MT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kG8Threads, 1)
k_gemm_8bit_pair(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ TokenMaps tm_x, const Gemm8Params p) {
  using C = G8Pair<MT>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t s_w = base, s_x = s_w + C::kStages * C::kWBytes;
  const uint32_t bar_full = s_x + C::kStages * C::kXBytes;   // leader: two producer arrivals and both CTAs' bytes
  const uint32_t bar_empty = bar_full + 8 * C::kStages;      // both CTAs: MMAs of the stage retired
  const uint32_t bar_acc_full = bar_empty + 8 * C::kStages;  // [2] both CTAs
  const uint32_t bar_acc_empty = bar_acc_full + 16;          // [2] leader: the pair's epilogue warps
  const uint32_t s_slot = bar_acc_empty + 16;
  int* off = reinterpret_cast<int*>(smem_raw + (bar_full - smem_u32(smem_raw)) + C::kBarBytes);
  int *order = off + p.experts + 1, *tiles = order + p.experts;
  const int warp = warp_uniform(), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(bar_full + 8 * s, 2);
      mbar_init(bar_empty + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar_acc_full + 8 * b, 1);
      mbar_init(bar_acc_empty + 8 * b, 2 * kG8EpiWarps);
    }
    mbar_init_fence();
    tma_prefetch_desc(&tm_w);
  }
  if (warp == 1) tmem_alloc_pair<C::kTmemCols>(s_slot);
  pdl_wait();
  if (p.experts) g8_tables<MT>(p, off, order, tiles);
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(s_slot));

  const G8Tables tb{off, order, tiles};
  const int nk = (p.K + 127) / 128;
  G8Walk<MT, 256> walk(p, tb, (int)blockIdx.x >> 1, (int)gridDim.x >> 1);
  G8Item it;

  if (warp == 0) {
    if (elect_one()) {
      uint32_t s = 0, ph = 1;
      bool ok = true;
      const uint32_t full0 = map_to_cta(bar_full, 0);
      while (ok && walk.next(p, tb, it)) {
        const int share = ((it.rows + 31) & ~31) / 2, box = g8_box(share), bytes = 128 * 16 << box;
        const int wrow = it.wrow0 + (int)rank * 128, xrow = (int)it.row0 + (int)rank * share;
        for (int ks = 0; ks < nk; ++ks) {
          if (!mbar_wait_cluster(bar_empty + 8 * s, ph)) { if (p.status) atomicCAS(p.status, 0, 148); ok = false; break; }
          const uint32_t full = full0 + 8 * s;
          mbar_expect_tx_remote(full, C::kWBytes + bytes);
          tma_load_2d_pair(s_w + s * C::kWBytes, &tm_w, full, ks * 128, wrow);
          tma_load_2d_pair(s_x + s * C::kXBytes, &tm_x.m[box], full, ks * 128, xrow);
          if (++s == C::kStages) { s = 0; ph ^= 1; }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0 && elect_one()) {
      constexpr uint32_t kHi = (1024u >> 4) | (1u << 14) | (2u << 29);
      const uint32_t w_lo0 = ((s_w >> 4) & 0x3FFF) | (1u << 16), x_lo0 = ((s_x >> 4) & 0x3FFF) | (1u << 16);
      uint32_t s = 0, ph = 0, n_it = 0;
      bool ok = true;
      for (; ok && walk.next(p, tb, it); ++n_it) {
        const uint32_t buf = n_it & 1;
        if (!mbar_wait_cluster(bar_acc_empty + 8 * buf, ((n_it >> 1) & 1) ^ 1)) { if (p.status) atomicCAS(p.status, 0, 149); break; }
        tc_fence_after();
        const uint32_t acc = tmem + buf * MT;
        const uint32_t idesc = idesc_8bit<kInt>(256, (it.rows + 31) & ~31);
        for (int ks = 0; ks < nk; ++ks) {
          if (!mbar_wait_cluster(bar_full + 8 * s, ph)) { if (p.status) atomicCAS(p.status, 0, 150); ok = false; break; }
          tc_fence_after();
          const uint32_t w_lo = w_lo0 + s * (C::kWBytes >> 4), x_lo = x_lo0 + s * (C::kXBytes >> 4);
#pragma unroll
          for (int q = 0; q < 4; ++q)
            mma_8bit_pair<kInt>(acc, ((uint64_t)kHi << 32) | (w_lo + 2 * q), ((uint64_t)kHi << 32) | (x_lo + 2 * q), idesc, (ks | q) ? 1u : 0u);
          mma_commit_pair(bar_empty + 8 * s);
          if (++s == C::kStages) { s = 0; ph ^= 1; }
        }
        if (ok) mma_commit_pair(bar_acc_full + 8 * buf);
      }
    }
    __syncwarp();
  } else {
    const int quad = warp & 3, half = (warp - 2) >> 2;
    __shared__ float4 s_scales[kG8EpiWarps][8];
    float* s_sa = reinterpret_cast<float*>(s_scales[warp - 2]);
    const uint32_t acc_empty0 = map_to_cta(bar_acc_empty, 0);
    uint32_t n_it = 0;
    for (; walk.next(p, tb, it); ++n_it) {
      const uint32_t buf = n_it & 1;
      int okw = 1;
      if (lane == 0) okw = mbar_wait_cluster(bar_acc_full + 8 * buf, (n_it >> 1) & 1, nk) ? 1 : 0;
      okw = __shfl_sync(0xFFFFFFFFu, okw, 0);
      if (!okw) { if (lane == 0 && p.status) atomicCAS(p.status, 0, 151); break; }
      tc_fence_after();
      const int n = it.n0 + (int)rank * 128 + quad * 32 + lane;
      const bool live = n < p.N;
      const float sb = live ? __ldg(p.b_scale + (int64_t)it.expert * p.N + n) : 0.f;
      g8_store_tile<kInt, MT>(p, it, n, live, sb, tmem + ((uint32_t)(quad * 32) << 16) + buf * MT, half, s_sa);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_remote(acc_empty0 + 8 * buf);
    }
    if (p.experts && p.zero_rest) g8_zero_rest(p, off, warp - 2, lane);
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc_pair<C::kTmemCols>(tmem);
  }
}

template <bool kInt, int MT>
int launch_pair(const CUtensorMap& tw, const TokenMaps& tx, const Gemm8Params& p, int64_t items, cudaStream_t st) {
  using C = G8Pair<MT>;
  auto kern = k_gemm_8bit_pair<kInt, MT>;
  static SmemOptIn opt_in;
  if (int e = opt_in.ensure(kern, C::smem(kGemm8MaxExperts))) return e;
  const int64_t pairs = sm_count() / 2;
  // in plain stream order: every SM is taken anyway
  kern<<<dim3((unsigned)(2 * (items < pairs ? items : pairs))), dim3(kG8Threads), C::smem(p.experts), st>>>(tw, tx, p);
  return (int)cudaGetLastError();
}

// Few tiles: K is split over a cluster of C blocks (rank r takes k-steps [nk * r / C, nk * (r + 1) / C)). Each block leaves its sums of the tile
// in its shared memory, and every rank adds up a share of the tile's elements over the ranks, in rank order: one launch, no workspace,
// the same bits every time (int8: the bits of the unsplit sum).
// kDeep: with few blocks, one of them has an SM's whole shared memory for its stages.
template <int MT, bool kDeep>
struct G8Split {
  static constexpr int kStages = kDeep ? (MT == 16 ? 11 : MT == 64 ? 8 : 6) : (MT == 16 ? 6 : MT == 64 ? 4 : 3);
  static constexpr int kTmemCols = MT < 32 ? 32 : MT;
  static constexpr int kSmem = kStages * G8Cfg<MT>::kStageBytes + 1024 + G8Cfg<MT>::kBarBytes;
  static_assert(MT * 128 * 4 <= kStages * G8Cfg<MT>::kStageBytes && kSmem <= 232448 && 16 * kStages + 12 <= G8Cfg<MT>::kBarBytes, "the tile's sums take the stages' place");
};

template <bool kInt, int MT, bool kDeep>
__global__ void __launch_bounds__(kG8Threads, kDeep ? 1 : G8Cfg<MT>::kBlocksPerSm)
k_gemm_8bit_split(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ TokenMaps tm_x, const Gemm8Params p, const int split) {
  using C = G8Cfg<MT>;
  using S = G8Split<MT, kDeep>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t s_w = base, s_x = s_w + S::kStages * C::kWBytes;
  const uint32_t bar_full = s_x + S::kStages * C::kXBytes, bar_empty = bar_full + 8 * S::kStages, bar_acc = bar_empty + 8 * S::kStages, s_slot = bar_acc + 8;
  const int warp = warp_uniform(), lane = threadIdx.x & 31;
  const int rank = (int)blockIdx.x % split;                  // == rank in the cluster
  const int n_nt = (int)(((int64_t)p.N + 127) / 128), nk = (p.K + 127) / 128;
  const int k0 = (int)((int64_t)nk * rank / split), k1 = (int)((int64_t)nk * (rank + 1) / split);
  const G8Item it = g8_dense_item<MT>(p, (int)blockIdx.x / split, n_nt);

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    mbar_init(bar_acc, 1);
    mbar_init_fence();
    tma_prefetch_desc(&tm_w);
  }
  if (warp == 1) tmem_alloc<S::kTmemCols>(s_slot);
  pdl_wait();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(s_slot));

  if (warp == 0) {
    if (elect_one()) {
      const int box = g8_box(it.rows), bytes = 128 * 16 << box;
      uint32_t s = 0, ph = 1;
      for (int ks = k0; ks < k1; ++ks) {
        if (!mbar_wait(bar_empty + 8 * s, ph)) { if (p.status) atomicCAS(p.status, 0, 145); break; }
        const uint32_t full = bar_full + 8 * s;
        mbar_expect_tx(full, C::kWBytes + bytes);
        tma_load_2d(s_w + s * C::kWBytes, &tm_w, full, ks * 128, it.wrow0);
        tma_load_2d(s_x + s * C::kXBytes, &tm_x.m[box], full, ks * 128, (int)it.row0);
        if (++s == S::kStages) { s = 0; ph ^= 1; }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one()) {
      constexpr uint32_t kHi = (1024u >> 4) | (1u << 14) | (2u << 29);
      const uint32_t w_lo0 = ((s_w >> 4) & 0x3FFF) | (1u << 16), x_lo0 = ((s_x >> 4) & 0x3FFF) | (1u << 16);
      const uint32_t idesc = idesc_8bit<kInt>(128, it.rows <= 16 ? 16 : (it.rows + 31) & ~31);
      uint32_t s = 0, ph = 0;
      bool ok = true;
      for (int ks = k0; ks < k1; ++ks) {
        if (!mbar_wait(bar_full + 8 * s, ph)) { if (p.status) atomicCAS(p.status, 0, 146); ok = false; break; }
        tc_fence_after();
        const uint32_t w_lo = w_lo0 + s * (C::kWBytes >> 4), x_lo = x_lo0 + s * (C::kXBytes >> 4);
#pragma unroll
        for (int q = 0; q < 4; ++q)
          mma_8bit<kInt>(tmem, ((uint64_t)kHi << 32) | (w_lo + 2 * q), ((uint64_t)kHi << 32) | (x_lo + 2 * q), idesc, (ks > k0 || q) ? 1u : 0u);
        mma_commit(bar_empty + 8 * s);
        if (++s == S::kStages) { s = 0; ph ^= 1; }
      }
      if (ok) mma_commit(bar_acc);
    }
    __syncwarp();
  } else {
    // sums -> shared memory [token][128 channels], in the stages' place: their last reader is the MMA that bar_acc waits for
    const int quad = warp & 3, half = (warp - 2) >> 2;
    int okw = 1;
    if (lane == 0) okw = mbar_wait(bar_acc, 0, nk) ? 1 : 0;
    okw = __shfl_sync(0xFFFFFFFFu, okw, 0);
    if (!okw && lane == 0 && p.status) atomicCAS(p.status, 0, 147);
    tc_fence_after();
    constexpr int kCols = MT < 32 ? MT : 32;
    const uint32_t taddr = tmem + ((uint32_t)(quad * 32) << 16);
    for (int col = half * kCols; okw && col < it.rows; col += 2 * kCols) {
      float v[32];
      if constexpr (MT >= 32) tmem_ld32(taddr + col, v); else tmem_ld16(taddr + col, v);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < kCols; ++j)
        asm volatile("st.shared.f32 [%0], %1;" ::"r"(base + (uint32_t)(((col + j) * 128 + quad * 32 + lane) * 4)), "f"(v[j]) : "memory");
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                                        // every rank's sums are in place
  const int elements = it.rows * 128;
  for (int i = rank * kG8Threads + (int)threadIdx.x; i < elements; i += split * kG8Threads) {
    const int tok = i >> 7, n = it.n0 + (i & 127);
    float v[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      v[r] = 0.f;
      if (r < split) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v[r]) : "r"(map_to_cta(base + (uint32_t)i * 4u, (uint32_t)r)));
    }
    float sum;
    if (kInt) {
      int total = __float_as_int(v[0]);
#pragma unroll
      for (int r = 1; r < 8; ++r) total += __float_as_int(v[r]);
      sum = __int2float_rn(total);
    } else {
      sum = v[0];
#pragma unroll
      for (int r = 1; r < 8; ++r)
        if (r < split) sum += v[r];
    }
    if (n < p.N) store_out(p.out, (it.row0 + tok) * p.out_stride + n, sum * __ldg(p.a_scale + it.row0 + tok) * __ldg(p.b_scale + n), p.out_type);
  }
  cluster_sync_all();                                        // nobody leaves while a peer still reads its sums
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc<S::kTmemCols>(tmem);
  }
}

template <bool kInt, int MT, bool kDeep>
int launch_split_form(const CUtensorMap& tw, const TokenMaps& tx, const Gemm8Params& p, int64_t items, int split, cudaStream_t st) {
  auto kern = k_gemm_8bit_split<kInt, MT, kDeep>;
  static SmemOptIn opt_in;
  if (int e = opt_in.ensure(kern, G8Split<MT, kDeep>::kSmem)) return e;
  return (int)launch_clusters(kern, dim3((unsigned)(items * split)), dim3(kG8Threads), dim3((unsigned)split), G8Split<MT, kDeep>::kSmem, st, tw, tx, p, split);
}
template <bool kInt, int MT>
int launch_split(const CUtensorMap& tw, const TokenMaps& tx, const Gemm8Params& p, int64_t items, int split, cudaStream_t st) {
  // Half of the SMs at most: with one block per SM the GPCs do not hold as many clusters as there are SMs for (1 x 2010 x 10112, 128 blocks in
  // clusters of eight, 13.7 us in the deep form, 7.8 with two blocks per SM). Clusters of four are never that few where they are chosen.
  const bool deep = split == 8 && items * split <= sm_count() / 2;
  return deep ? launch_split_form<kInt, MT, true>(tw, tx, p, items, split, st) : launch_split_form<kInt, MT, false>(tw, tx, p, items, split, st);
}

template <bool kInt, int MT, bool kDeep>
int launch_mt(const CUtensorMap& tw, const TokenMaps& tx, const Gemm8Params& p, int64_t most_items, cudaStream_t st) {
  using C = G8Cfg<MT, kDeep>;
  auto kern = k_gemm_8bit<kInt, MT, kDeep>;
  static SmemOptIn opt_in;
  if (int e = opt_in.ensure(kern, C::smem(kGemm8MaxExperts))) return e;
  const int64_t slots = (int64_t)sm_count() * C::kBlocksPerSm;
  return (int)launch_chain(kern, dim3((unsigned)(most_items < slots ? most_items : slots)), dim3(kG8Threads), C::smem(p.experts), st, tw, tx, p);
}

// How a call runs: kDecode (gemm_8bit_decode.cu), kSingle (one block per tile of 128 x mt, deep where all tiles run at once), kSplit (K over a
// cluster of `split` blocks), kPair (tiles of 256 x mt on CTA pairs).
enum { kDecode, kSingle, kSplit, kPair };
struct G8Plan {
  int form, mt, split;
};

// Dense: the form whose estimate is the least. An estimate is in microseconds of a call among others, linear in what its form is made of: waves of
// blocks, the k-steps of 128 of a wave (dearer the fuller it is), the bytes of the weights, the sums that a cluster exchanges. Fitted to
// 4400 shapes (1 to 4096 rows, 128 <= N <= 16384, 256 <= K <= 16384, both types, every form timed); choosing by it costs 1 to 2 % on average
// against always taking the fastest form, 11 % or less for 90 of 100 shapes. Some of the times behind it (us, int8):
//   1 x 4096 x 7168      decode 8.4, split 9.2, single 12.0          16 x 16384 x 4096   single 13.7, decode 15.4
//   64 x 1024 x 8192     split 8.0, single 13.6                      256 x 4096 x 7168   single (64 rows) 13.8, split 17.7, pair (256) 23
//   512 x 4096 x 12288   pair (128) 24.7, single 26.9                8192 x 4096 x 12288 pair (256) 255, pair (128) 304, single 362
G8Plan dense_plan(const Gemm8Params& p) {
  const int sms = sm_count();
  const auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
  const int64_t m = p.M, n = p.N, nk = up(p.K, 128);
  G8Plan best{kSingle, 128, 1};
  double least = 1e30;
  const auto offer = [&](double us, G8Plan plan) {
    if (us < least) least = us, best = plan;
  };
  const auto single = [&](int mt) {
    const int64_t items = up(m, mt) * up(n, 128);
    const bool deep = items <= sms;
    const int64_t slots = deep ? sms : 2 * sms, w = up(items, slots);
    const double full = (double)items / (double)(w * slots), steps = (double)(w * nk);
    const double us = mt == 16                ? 2.67 * w + steps * (0.160 + 0.178 * full)
                      : mt == 64 && deep      ? 3.13 * w + steps * (0.189 + 0.086 * full)
                      : mt == 64              ? 3.92 + 0.55 * w + steps * (0.177 + 0.276 * full)
                      : deep                  ? 4.09 * w + steps * (0.240 + 0.075 * full)
                                              : 3.83 + 1.64 * w + steps * (0.347 + 0.222 * full);
    offer(us, {kSingle, mt, 1});
  };
  const auto split = [&](int mt, int by, double wave, double step, double fetch, double exchange) {
    const int64_t items = up(m, mt) * up(n, 128), blocks = items * by;
    if (by > nk || blocks > 600) return;
    const int64_t w = up(blocks, by == 8 ? 256 : 264), steps = up(nk, by);
    const double rows = (double)(m < mt ? m : mt);
    offer(wave * w + step * (double)(steps * w) + fetch * 1e-3 * (double)(blocks * steps) * (16 + rows / 8) + exchange * 1e-4 * (double)blocks * rows,
          {kSplit, mt, by});
  };
  if (m <= 16 || (m <= 32 && p.code == kInt8)) {
    const int64_t blocks = up(n, 16), warps = blocks < 222 ? 16 : blocks < 444 ? 8 : 4;
    const double mb = (double)n * p.K * 1e-6, units = (double)p.K / 64 / (double)warps;
    offer(m > 16 ? 3.17 + 0.182 * mb + 0.313 * units : p.code == kInt8 ? 2.16 + 0.133 * mb + 0.239 * units : 2.50 + 0.149 * mb + 0.306 * units, {kDecode, 0, 1});
  }
  if (m <= 16) {
    single(16);
    split(16, 4, 4.40, 0.153, 0.0906, 4.62);
    split(16, 8, 4.48, 0.143, 0.0968, 2.85);
    return best;
  }
  if (m <= 640) {
    single(64);
    split(64, 4, 5.59, 0.207, 0.0393, 1.43);
    split(64, 8, 5.02, 0.227, 0.0359, 1.40);
  }
  if (m > 64) {
    single(128);
    if (m <= 1500) {
      split(128, 4, 8.18, 0.242, 0.0392, 0.64);
      split(128, 8, 6.29, 0.272, 0.0433, 0.81);
    }
    for (int mt = 128; mt <= (m > 128 ? 256 : 128); mt *= 2) {
      const int64_t items = up(m, mt) * up(n, 256), pairs = sms / 2, w = up(items, pairs);
      const double full = (double)items / (double)(w * pairs), steps = (double)(w * nk);
      offer(mt == 128 ? 3.68 + 1.93 * w + steps * (0.192 + 0.034 * full) : 4.32 + 2.74 * w + steps * (0.288 + 0.060 * full), {kPair, mt, 1});
    }
  }
  return best;
}

// Grouped: by the rows of a segment, on average, which is all that the host knows. Weights stream past few rows whatever the tile; from 32 rows on a
// tile should hold a segment, and from about 160 the pair's tile saves operand traffic, unless K is over before its longer start is made
// up for (us, 128 experts: 1536 x 2048 with 2 rows 43 / 45 / 46 / 46 for 16 / 64 / 128 / pairs, 32 rows 77 / 70 / 70 / 70, 256 rows - / 166 / 140 / 128,
// 1024 rows - / - / 415 / 323; 2048 x 768 with 512 rows 141 for 128, 162 for pairs).
G8Plan grouped_plan(const Gemm8Params& p) {
  const int64_t rows = ((int64_t)p.M + p.experts - 1) / p.experts;
  if (rows <= 4) return {kSingle, 16, 1};
  if (rows <= 32) return {kSingle, 64, 1};
  if (rows <= 160 || p.K < 1536 || p.N <= 128) return {kSingle, 128, 1};
  return {kPair, 256, 1};
}

template <bool kInt>
int launch_plan(const CUtensorMap& tw, const TokenMaps& tx, const Gemm8Params& p, const G8Plan& plan, cudaStream_t st) {
  const int64_t mt = plan.mt, bn = plan.form == kPair ? 256 : 128;
  // a segment ends inside its last tile: at most one tile more than its rows fill, and no tile is empty
  const int64_t m_tiles = p.experts ? p.M / mt + (p.experts < p.M ? p.experts : p.M) : (p.M + mt - 1) / mt;
  const int64_t items = m_tiles * (((int64_t)p.N + bn - 1) / bn);
  if (plan.form == kPair) return mt == 128 ? launch_pair<kInt, 128>(tw, tx, p, items, st) : launch_pair<kInt, 256>(tw, tx, p, items, st);
  if (plan.form == kSplit) {
    if (mt == 16) return launch_split<kInt, 16>(tw, tx, p, items, plan.split, st);
    if (mt == 64) return launch_split<kInt, 64>(tw, tx, p, items, plan.split, st);
    return launch_split<kInt, 128>(tw, tx, p, items, plan.split, st);
  }
  const bool deep = items <= sm_count();
  if (mt == 16) return deep ? launch_mt<kInt, 16, true>(tw, tx, p, items, st) : launch_mt<kInt, 16, false>(tw, tx, p, items, st);
  if (mt == 64) return deep ? launch_mt<kInt, 64, true>(tw, tx, p, items, st) : launch_mt<kInt, 64, false>(tw, tx, p, items, st);
  return deep ? launch_mt<kInt, 128, true>(tw, tx, p, items, st) : launch_mt<kInt, 128, false>(tw, tx, p, items, st);
}

}  // namespace

int launch_gemm_8bit(const void* a, int64_t a_stride, const void* b, const Gemm8Params& p, cudaStream_t st) {
  const G8Plan plan = p.experts ? grouped_plan(p) : dense_plan(p);
  if (plan.form == kDecode) return launch_gemm_8bit_decode(a, a_stride, b, p, st);
  CUtensorMap tw;
  TokenMaps tx;
  int rc = make_operand_map(&tw, b, (uint64_t)(p.experts ? p.experts : 1) * (uint64_t)p.N, (uint64_t)p.K, 128);
  for (int i = 0; i < 4 && !rc; ++i) rc = make_operand_map(&tx.m[i], a, (uint64_t)p.M, (uint64_t)p.K, 16u << i, (uint64_t)a_stride);
  if (rc) return rc;
  return p.code == kInt8 ? launch_plan<true>(tw, tx, p, plan, st) : launch_plan<false>(tw, tx, p, plan, st);
}

}  // namespace b200
