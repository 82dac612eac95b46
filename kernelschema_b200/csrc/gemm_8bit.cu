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

// MT = most tokens of a tile. Up to 128 two blocks share an SM (half of its shared memory and TMEM each).
template <int MT>
struct G8Cfg {
  static constexpr int kWBytes = 128 * 128, kXBytes = MT * 128, kStageBytes = kWBytes + kXBytes;
  static constexpr int kStages = MT == 16 ? 5 : MT == 64 ? 4 : MT == 128 ? 3 : 4;
  static constexpr int kTmemCols = 2 * MT;
  static constexpr int kBlocksPerSm = MT <= 128 ? 2 : 1;
  static constexpr int kBarBytes = 256;
  static constexpr int smem(int experts) { return kStages * kStageBytes + 1024 + kBarBytes + (experts ? 8 * (experts + 1) : 0); }
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

DEV void store_out(void* out, int64_t at, float v, int out_type) {
  if (out_type == kBf16) reinterpret_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(v);
  else if (out_type == kF16) reinterpret_cast<__half*>(out)[at] = __float2half_rn(v);
  else reinterpret_cast<float*>(out)[at] = v;
}

// One tile of the output.
struct G8Item {
  int64_t row0;     // first token
  int rows;         // tokens, 1..MT
  int wrow0;        // first weight row of the map
  int n0, expert;   // first channel, expert
};

// Device tables of a grouped call: first row of every segment, cut to the rows there are and to ascending order, and the token tiles before it.
struct G8Tables {
  const int* off;
  const int* tiles;
};

template <int MT>
DEV G8Item g8_item(const Gemm8Params& p, const G8Tables& tb, int64_t t, int n_nt) {
  G8Item it;
  if (!p.experts) {
    const int64_t n_mt = (p.M + MT - 1) / MT, per = (int64_t)kG8Group * n_nt, g = t / per, r = t - g * per;
    const int64_t rows = min((int64_t)kG8Group, n_mt - g * kG8Group);
    const int64_t mt = g * kG8Group + r % rows;
    it.n0 = (int)(r / rows) * 128;
    it.row0 = mt * MT;
    it.rows = (int)min((int64_t)MT, p.M - it.row0);
    it.expert = 0;
    it.wrow0 = it.n0;
    return it;
  }
  const int mt = (int)(t / n_nt);
  it.n0 = (int)(t - (int64_t)mt * n_nt) * 128;
  int lo = 0, hi = p.experts;                                // last e with tiles[e] <= mt: the segment that holds it (empty ones have none)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (tb.tiles[mid] <= mt) lo = mid; else hi = mid;
  }
  const int first = tb.off[lo] + (mt - tb.tiles[lo]) * MT;
  it.expert = lo;
  it.row0 = first;
  it.rows = min(MT, tb.off[lo + 1] - first);
  it.wrow0 = lo * p.N + it.n0;
  return it;
}

// Token rows that a tile's copies fetch: boxes of 16, 64 or 128 rows.
template <int MT>
DEV int g8_fetch(int rows) { return rows <= 16 ? 16 : MT >= 64 && rows <= 64 ? 64 : rows <= 128 ? 128 : 256; }

template <bool kInt, int MT>
__global__ void __launch_bounds__(kG8Threads, G8Cfg<MT>::kBlocksPerSm)
k_gemm_8bit(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x16, const __grid_constant__ CUtensorMap tm_x64,
            const __grid_constant__ CUtensorMap tm_x128, const Gemm8Params p) {
  using C = G8Cfg<MT>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t s_w = base, s_x = s_w + C::kStages * C::kWBytes;
  const uint32_t bar_full = s_x + C::kStages * C::kXBytes, bar_empty = bar_full + 8 * C::kStages;
  const uint32_t bar_acc_full = bar_empty + 8 * C::kStages, bar_acc_empty = bar_acc_full + 16, s_slot = bar_acc_empty + 16;
  int* tab = reinterpret_cast<int*>(smem_raw + (bar_full - smem_u32(smem_raw)) + C::kBarBytes);   // off[E + 1], tiles[E + 1]
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
    tma_prefetch_desc(&tm_x16);
  }
  if (warp == 1) tmem_alloc<C::kTmemCols>(s_slot);
  pdl_wait();
  const int n_nt = (int)(((int64_t)p.N + 127) / 128);
  int* off = tab;
  int* tiles = tab + p.experts + 1;
  if (p.experts) {
    for (int e = threadIdx.x; e <= p.experts; e += kG8Threads) off[e] = min(max(__ldg(p.offsets + e), 0), (int)p.M);
    __syncthreads();
    if (warp == 2) {
      int most = 0;                                          // ascending whatever the caller's offsets are
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
      __syncwarp();
      int sum = 0;
      for (int e0 = 0; e0 < p.experts; e0 += 32) {
        const int e = e0 + lane;
        int v = e < p.experts ? (off[e + 1] - off[e] + MT - 1) / MT : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int u = __shfl_up_sync(0xFFFFFFFFu, v, o);
          if (lane >= o) v += u;
        }
        if (e < p.experts) tiles[e + 1] = sum + v;
        sum += __shfl_sync(0xFFFFFFFFu, v, 31);
      }
      if (lane == 0) tiles[0] = 0;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(s_slot));

  const G8Tables tb{off, tiles};
  const int nk = (p.K + 127) / 128;
  const int64_t items = (p.experts ? (int64_t)tiles[p.experts] : ((int64_t)p.M + MT - 1) / MT) * n_nt;

  if (warp == 0) {
    if (elect_one()) {
      uint32_t s = 0, ph = 1;
      bool ok = true;
      for (int64_t t = blockIdx.x; ok && t < items; t += gridDim.x) {
        const G8Item it = g8_item<MT>(p, tb, t, n_nt);
        const int fetch = g8_fetch<MT>(it.rows);
        const CUtensorMap* tm_x = fetch == 16 ? &tm_x16 : fetch == 64 ? &tm_x64 : &tm_x128;
        for (int ks = 0; ks < nk; ++ks) {
          if (!mbar_wait(bar_empty + 8 * s, ph)) { if (p.status) atomicCAS(p.status, 0, 141); ok = false; break; }
          const uint32_t full = bar_full + 8 * s;
          mbar_expect_tx(full, C::kWBytes + fetch * 128);
          tma_load_2d(s_w + s * C::kWBytes, &tm_w, full, ks * 128, it.wrow0);
          tma_load_2d(s_x + s * C::kXBytes, tm_x, full, ks * 128, (int)it.row0);
          if (fetch == 256) tma_load_2d(s_x + s * C::kXBytes + 128 * 128, tm_x, full, ks * 128, (int)it.row0 + 128);
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
      for (int64_t t = blockIdx.x; ok && t < items; t += gridDim.x, ++n_it) {
        const G8Item it = g8_item<MT>(p, tb, t, n_nt);
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
    uint32_t n_it = 0;
    for (int64_t t = blockIdx.x; t < items; t += gridDim.x, ++n_it) {
      const G8Item it = g8_item<MT>(p, tb, t, n_nt);
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
      constexpr int kCols = MT < 32 ? MT : 32;
      for (int col = half * kCols; col < it.rows; col += 2 * kCols) {
        float v[32];
        if constexpr (MT >= 32) tmem_ld32(taddr + col, v); else tmem_ld16(taddr + col, v);
        const float sa = lane < it.rows - col ? __ldg(p.a_scale + it.row0 + col + lane) : 0.f;
        tmem_ld_wait();
        const int64_t at = (it.row0 + col) * p.out_stride + n;
        const int cols = min(kCols, it.rows - col);
#pragma unroll
        for (int j = 0; j < kCols; ++j) {
          const float s = __shfl_sync(0xFFFFFFFFu, sa, j);
          if (live && j < cols) store_out(p.out, at + j * p.out_stride, acc_value<kInt>(v[j]) * s * sb, p.out_type);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_acc_empty + 8 * buf);
    }
    if (p.experts && p.zero_rest) {
      // rows of no segment, of an output that this call made
      const int64_t before = off[0], behind = off[p.experts], rest = before + (p.M - behind);
      for (int64_t r = (int64_t)blockIdx.x * kG8EpiWarps + (warp - 2); r < rest; r += (int64_t)gridDim.x * kG8EpiWarps) {
        const int64_t row = r < before ? r : behind + (r - before);
        for (int n = lane; n < p.N; n += 32) store_out(p.out, row * p.out_stride + n, 0.f, p.out_type);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc<C::kTmemCols>(tmem);
  }
}

template <bool kInt, int MT>
int launch_mt(const CUtensorMap& tw, const CUtensorMap (&tx)[3], const Gemm8Params& p, int64_t most_items, cudaStream_t st) {
  using C = G8Cfg<MT>;
  auto kern = k_gemm_8bit<kInt, MT>;
  static SmemOptIn opt_in;
  if (int e = opt_in.ensure(kern, C::smem(kGemm8MaxExperts))) return e;
  const int64_t slots = (int64_t)sm_count() * C::kBlocksPerSm;
  return (int)launch_chain(kern, dim3((unsigned)(most_items < slots ? most_items : slots)), dim3(kG8Threads), C::smem(p.experts), st, tw, tx[0], tx[1],
                           tx[2], p);
}

template <bool kInt>
int launch_any(const CUtensorMap& tw, const CUtensorMap (&tx)[3], const Gemm8Params& p, int mt, int64_t items, cudaStream_t st) {
  if (mt == 16) return launch_mt<kInt, 16>(tw, tx, p, items, st);
  if (mt == 64) return launch_mt<kInt, 64>(tw, tx, p, items, st);
  if (mt == 128) return launch_mt<kInt, 128>(tw, tx, p, items, st);
  return launch_mt<kInt, 256>(tw, tx, p, items, st);
}

}  // namespace

int launch_gemm_8bit(const void* a, int64_t a_stride, const void* b, const Gemm8Params& p, cudaStream_t st) {
  const int64_t experts = p.experts ? p.experts : 1;
  const int64_t rows = p.experts ? (p.M + experts - 1) / experts : p.M;          // of a segment, on average
  const int mt = rows <= 16 ? 16 : rows <= 64 ? 64 : rows <= 128 ? 128 : 256;
  CUtensorMap tw, tx[3];
  int rc = make_operand_map(&tw, b, (uint64_t)(experts * p.N), (uint64_t)p.K, 128);
  const uint32_t boxes[3] = {16, 64, 128};
  for (int i = 0; i < 3 && !rc; ++i) rc = make_operand_map(&tx[i], a, (uint64_t)p.M, (uint64_t)p.K, boxes[i], (uint64_t)a_stride);
  if (rc) return rc;
  // a segment ends inside its last tile: at most one tile more than its rows fill, and no tile is empty
  const int64_t m_tiles = p.experts ? (p.M / mt + (experts < p.M ? experts : p.M)) : (p.M + mt - 1) / mt;
  const int64_t items = m_tiles * (((int64_t)p.N + 127) / 128);
  return p.code == kInt8 ? launch_any<true>(tw, tx, p, mt, items, st) : launch_any<false>(tw, tx, p, mt, items, st);
}

}  // namespace b200
