// The kernels of the 8-bit GEMM that run as clusters: CTA pairs for many tokens, K split over several blocks for few tiles. Neither lets the next
// launch in early (launch_clusters in kernels.cuh).
#pragma once
#include "gemm_8bit.cuh"

namespace b200 {

namespace {

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

// ----------------------------------------------------------------------------- K over clusters
// Few tiles: K is split over a cluster of C blocks (rank r takes k-steps [nk * r / C, nk * (r + 1) / C)). Each block leaves its sums of the tile
// in its shared memory, and every rank adds up a share of the tile's elements over the ranks, in rank order: one launch, no workspace,
// the same bits every time (int8: the bits of the unsplit sum).
// kDeep: with few blocks, one of them has an SM's whole shared memory for its stages.
template <int MT, bool kDeep>
struct G8Split {
  static constexpr int kStages = kDeep ? (MT == 16 ? 11 : MT == 64 ? 8 : 6) : (MT == 16 ? 6 : MT == 64 ? 4 : 3);
  static constexpr int kTmemCols = MT < 32 ? 32 : MT;
  static constexpr int kSmem = kStages * (16384 + MT * 128) + 1024 + G8Cfg<MT>::kBarBytes;
  static_assert(MT * 128 * 4 <= kStages * (16384 + MT * 128) && kSmem <= 232448 && 16 * kStages + 12 <= G8Cfg<MT>::kBarBytes, "the tile's sums take the stages' place");
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

}  // namespace

}  // namespace b200
