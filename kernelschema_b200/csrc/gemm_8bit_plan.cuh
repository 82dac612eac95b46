// Which form of the 8-bit GEMM a call takes: host rules on sizes, type of codes and multiprocessors.
#pragma once
#include "kernels.cuh"

namespace b200 {

// How a call runs: kDecode (gemm_8bit_decode.cu), kSingle (one block per tile of 128 x mt, deep where all tiles run at once), kSplit (K over a
// cluster of `split` blocks), kPair (tiles of 256 x mt on CTA pairs).
enum { kDecode, kSingle, kSplit, kPair };
struct G8Plan {
  int form, mt, split;
};

// Dense: the form whose estimate is the least. An estimate is in microseconds of a call among others, linear in what its form is made of: waves of
// blocks, the k-steps of 128 of a wave (dearer the fuller it is), the bytes of the weights, the sums that a cluster exchanges. Fitted to
// 12000 shapes (1 to 4096 rows, 128 <= N <= 16384, 256 <= K <= 16384, both types, every form timed); choosing by it costs 1 % on average against
// always taking the fastest form, 8 % or less for 95 of 100 shapes. Some of the times behind it (us, int8):
//   1 x 4096 x 7168      decode 8.4, split 9.2, single 10.3          16 x 16384 x 4096   single 13.0, decode 15.4
//   64 x 1024 x 8192     split 8.0, single 12.6                      256 x 4096 x 7168   single (64 rows) 13.8, split 17.7, pair (256) 23
//   512 x 4096 x 12288   pair (128) 24.7, single 26.9                8192 x 4096 x 12288 pair (256) 255, pair (128) 304, single 362
inline G8Plan dense_plan(const Gemm8Params& p, int sms) {
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
    const double us = mt == 16           ? 2.82 * w + steps * (0.137 + 0.185 * full)
                      : mt == 64 && deep ? 3.28 * w + steps * (0.176 + 0.095 * full)
                      : mt == 64         ? 3.84 + 0.65 * w + steps * (0.170 + 0.275 * full)
                      : deep             ? 4.15 * w + steps * (0.236 + 0.062 * full)
                                         : 3.97 + 1.75 * w + steps * (0.233 + 0.357 * full);
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
    // batches of loads of a warp, dearer with the rows; the weights; the blocks
    const int64_t blocks = up(n, 16);
    const double batches = (double)up(up(up(p.K, 64), gemm_8bit_decode_warps(blocks, p.K, sms)), 4), mb = (double)n * p.K * 1e-6, kb = (double)blocks * 1e-3;
    const double r = (double)m / 16;
    offer(m > 16             ? 2.02 + batches * (0.524 + 0.405 * r) + 0.126 * mb + 2.41 * kb
          : p.code == kInt8  ? 1.31 + batches * (0.477 + 0.504 * r) + 0.156 * mb + 1.07 * kb
                             : 1.37 + batches * (0.637 + 0.413 * r) + 0.172 * mb + 0.99 * kb,
          {kDecode, 0, 1});
  }
  if (m <= 16) {
    single(16);
    split(16, 4, 4.40, 0.160, 0.0921, 4.09);
    split(16, 8, 4.52, 0.141, 0.1004, 2.51);
    return best;
  }
  if (m <= 640) {
    single(64);
    split(64, 4, 5.53, 0.247, 0.0294, 1.51);
    split(64, 8, 5.09, 0.209, 0.0509, 1.15);
  }
  if (m > 64) {
    single(128);
    if (m <= 1500) split(128, 8, 6.24, 0.280, 0.0360, 0.84);
    for (int mt = 128; mt <= (m > 128 ? 256 : 128); mt *= 2) {
      const int64_t items = up(m, mt) * up(n, 256), pairs = sms / 2, w = up(items, pairs);
      const double full = (double)items / (double)(w * pairs), steps = (double)(w * nk);
      offer(mt == 128 ? 3.65 + 1.99 * w + steps * (0.187 + 0.034 * full) : 4.22 + 2.82 * w + steps * (0.287 + 0.057 * full), {kPair, mt, 1});
    }
  }
  return best;
}

// Grouped: by the rows of a segment, on average, which is all that the host knows (few segments that hold all rows take tiles as small as the average of all
// segments asks for, and their weights then come from L2 once per tile). Weights stream past few rows whatever the tile; from 32 rows on a
// tile should hold a segment, and from about 160 the pair's tile saves operand traffic, unless K is over before its longer start is made
// up for (us, 128 experts: 1536 x 2048 with 2 rows 43 / 45 / 46 / 46 for 16 / 64 / 128 / pairs, 32 rows 77 / 70 / 70 / 70, 256 rows - / 166 / 140 / 128,
// 1024 rows - / - / 415 / 323; 2048 x 768 with 512 rows 141 for 128, 162 for pairs).
inline G8Plan grouped_plan(const Gemm8Params& p) {
  const int64_t rows = ((int64_t)p.M + p.experts - 1) / p.experts;
  if (rows <= 4) return {kSingle, 16, 1};
  if (rows <= 32) return {kSingle, 64, 1};
  if (rows <= 160 || p.K < 1536 || p.N <= 128) return {kSingle, 128, 1};
  return {kPair, 256, 1};
}

// Tiles of a call, at most. Grouped: a segment ends inside its last tile, so one tile more than its rows fill, and no tile is empty.
inline int64_t g8_items(const Gemm8Params& p, const G8Plan& plan) {
  const int64_t mt = plan.mt, bn = plan.form == kPair ? 256 : 128;
  const int64_t m_tiles = p.experts ? p.M / mt + (p.experts < p.M ? p.experts : p.M) : (p.M + mt - 1) / mt;
  return m_tiles * (((int64_t)p.N + bn - 1) / bn);
}

// Whether a block of kSingle or kSplit has an SM's whole shared memory for its stages: where all tiles run at once so. Of a split one half of the
// SMs at most: with one block per SM the GPCs do not hold as many clusters as there are SMs for (1 x 2010 x 10112, 128 blocks in
// clusters of eight, 13.7 us in the deep form, 7.8 with two blocks per SM). Clusters of four are never that few where they are chosen.
inline bool g8_deep(const G8Plan& plan, int64_t items, int sms) {
  return plan.form == kSplit ? plan.split == 8 && items * plan.split <= sms / 2 : plan.form == kSingle && items <= sms;
}

}  // namespace b200
