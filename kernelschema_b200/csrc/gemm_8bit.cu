// GEMM of 8-bit rows: out[m, n] = sa[m] * sb[n] * sum_k a[m, k] * b[n, k], int8 (exact int32 sums) or E4M3 (fp32 sums), one scale per
// token and per output channel; dense, or over the segments of tokens that are sorted by expert (one weight matrix per segment).
//
// The weights are the M side of tcgen05.mma (128 weight rows = 128 TMEM lanes), the tokens its N side, which a tile takes in steps of 16
// or 32: a tile of few tokens is no padding, and an expert's rest of rows costs what it holds. A thread of the epilogue then owns an
// output channel (one sb in a register) and a warp writes 32 consecutive channels of a token, so odd widths, strides and addresses
// need no form of their own.
// kind::i8 and kind::f8f6f4 take 32 bytes of K per instruction, four per step of 128 bytes. K beyond the last step reads as zeros (TMA's fill), so
// rows need no more than 16-byte lengths.
//
// What bounds it: many tokens, the tensor cores (8192 x 4096 x 12288 int8 256 us in a graph = 3.2 P op/s, 96 % busy; in calls among others 297, by the power cap); few, the weight
// stream (64 tokens over 128 experts 305 MB in 53 us = 5.75 TB/s) and, below about 20 MB of weights, launch, first access and
// reduction (100 x 2113 x 7168 10.7 us). The forms and their times are at dense_plan (gemm_8bit_plan.cuh).
#include "gemm_8bit.cuh"
#include "gemm_8bit_clusters.cuh"
#include "gemm_8bit_plan.cuh"

namespace b200 {

namespace {

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
        for (int ks = 0; ks < nk; ks += C::KC) {
          if (!mbar_wait(bar_empty + 8 * s, ph)) { if (p.status) atomicCAS(p.status, 0, 141); ok = false; break; }
          const uint32_t full = bar_full + 8 * s;
          mbar_expect_tx(full, min(C::KC, nk - ks) * (C::kWStep + bytes));
#pragma unroll
          for (int c = 0; c < C::KC; ++c) {
            if (ks + c >= nk) break;
            tma_load_2d(s_w + s * C::kWBytes + c * C::kWStep, &tm_w, full, (ks + c) * 128, it.wrow0);
            tma_load_2d(s_x + s * C::kXBytes + c * C::kXStep, &tm_x.m[box], full, (ks + c) * 128, (int)it.row0);
          }
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
        for (int ks = 0; ks < nk; ks += C::KC) {
          if (!mbar_wait(bar_full + 8 * s, ph)) { if (p.status) atomicCAS(p.status, 0, 143); ok = false; break; }
          tc_fence_after();
          const uint32_t w_lo = w_lo0 + s * (C::kWBytes >> 4), x_lo = x_lo0 + s * (C::kXBytes >> 4);
#pragma unroll
          for (int c = 0; c < C::KC; ++c) {
            if (ks + c >= nk) break;
#pragma unroll
            for (int q = 0; q < 4; ++q)
              mma_8bit<kInt>(acc, ((uint64_t)kHi << 32) | (w_lo + c * (C::kWStep >> 4) + 2 * q), ((uint64_t)kHi << 32) | (x_lo + c * (C::kXStep >> 4) + 2 * q), idesc,
                             (ks | c | q) ? 1u : 0u);
          }
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

template <bool kInt, int MT, bool kDeep>
int launch_split_form(const CUtensorMap& tw, const TokenMaps& tx, const Gemm8Params& p, int64_t items, int split, cudaStream_t st) {
  auto kern = k_gemm_8bit_split<kInt, MT, kDeep>;
  static SmemOptIn opt_in;
  if (int e = opt_in.ensure(kern, G8Split<MT, kDeep>::kSmem)) return e;
  return (int)launch_clusters(kern, dim3((unsigned)(items * split)), dim3(kG8Threads), dim3((unsigned)split), G8Split<MT, kDeep>::kSmem, st, tw, tx, p, split);
}
template <bool kInt, int MT>
int launch_split(const CUtensorMap& tw, const TokenMaps& tx, const Gemm8Params& p, int64_t items, int split, bool deep, cudaStream_t st) {
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

template <bool kInt>
int launch_plan(const CUtensorMap& tw, const TokenMaps& tx, const Gemm8Params& p, const G8Plan& plan, cudaStream_t st) {
  const int64_t mt = plan.mt, items = g8_items(p, plan);
  const bool deep = g8_deep(plan, items, sm_count());
  if (plan.form == kPair) return mt == 128 ? launch_pair<kInt, 128>(tw, tx, p, items, st) : launch_pair<kInt, 256>(tw, tx, p, items, st);
  if (plan.form == kSplit) {
    if (mt == 16) return launch_split<kInt, 16>(tw, tx, p, items, plan.split, deep, st);
    if (mt == 64) return launch_split<kInt, 64>(tw, tx, p, items, plan.split, deep, st);
    return launch_split<kInt, 128>(tw, tx, p, items, plan.split, deep, st);
  }
  if (mt == 16) return deep ? launch_mt<kInt, 16, true>(tw, tx, p, items, st) : launch_mt<kInt, 16, false>(tw, tx, p, items, st);
  if (mt == 64) return deep ? launch_mt<kInt, 64, true>(tw, tx, p, items, st) : launch_mt<kInt, 64, false>(tw, tx, p, items, st);
  return deep ? launch_mt<kInt, 128, true>(tw, tx, p, items, st) : launch_mt<kInt, 128, false>(tw, tx, p, items, st);
}

}  // namespace

int launch_gemm_8bit(const void* a, int64_t a_stride, const void* b, const Gemm8Params& p, cudaStream_t st) {
  const G8Plan plan = p.experts ? grouped_plan(p) : dense_plan(p, sm_count());
  if (plan.form == kDecode) return launch_gemm_8bit_decode(a, a_stride, b, p, st);
  CUtensorMap tw;
  TokenMaps tx;
  int rc = make_operand_map(&tw, b, (uint64_t)(p.experts ? p.experts : 1) * (uint64_t)p.N, (uint64_t)p.K, 128);
  // of the token maps those that a tile of the call can ask for: dense tiles are full but for the last (a map takes 0.2 us to make)
  const auto box = [&](int64_t rows) { return g8_box((int)(plan.form == kPair ? (rows + 31) / 32 * 16 : rows)); };
  const int64_t rest = p.M % plan.mt;
  const unsigned need = p.experts ? 15u : (p.M >= plan.mt ? 1u << box(plan.mt) : 0u) | (rest ? 1u << box(rest) : 0u);
  for (int i = 0; i < 4 && !rc; ++i)
    if (need >> i & 1) rc = make_operand_map(&tx.m[i], a, (uint64_t)p.M, (uint64_t)p.K, 16u << i, (uint64_t)a_stride);
  if (rc) return rc;
  return p.code == kInt8 ? launch_plan<true>(tw, tx, p, plan, st) : launch_plan<false>(tw, tx, p, plan, st);
}

}  // namespace b200
