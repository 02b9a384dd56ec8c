// linear_plan.h -- which kernel computes a product of the MLP layer, and how it cuts the
// work.  Host code alone.
#pragma once
#include <algorithm>

#include "kernels.h"

namespace mlpg {

constexpr int kKb = 64;            // contraction elements per stage: one 128-byte swizzle row
constexpr int kMaxSplit = 8;       // portable cluster size

// The tensor cores cut low bits when they add to an accumulator: on average about 2^-25 of
// it per step of 16, at most 2^-23, always towards zero, so the loss grows with the
// contraction (2-norm against 64 bits: 6e-7 after 512, 5e-6 after 4096).  The contraction is
// therefore cut into partial sums that start from zero and are added in f32, rounded to
// nearest.  Blocks per partial sum at most: 512 deep for f32 results; for 16-bit ones as much
// as keeps the loss below 1/15 of half a step of the type, 4096 deep for f16 and 32768 for
// bf16.  (2048 x 11008 x 4096 with a residual: 144.6 us with a single sum, 147.9 us every
// 4096, 149.7 us every 1024.)
constexpr int segment_blocks(int out_type) { return out_type == kTypeF32 ? 8 : (out_type == kTypeF16 ? 64 : 512); }

// The split kernel's partial sums per CTA, which fill its share of TMEM, and the blocks of the
// contraction that they hold
constexpr int split_segments(int bn) { return bn == 256 ? 2 : 256 / bn; }
constexpr int split_blocks(int bn, int out_type) { return segment_blocks(out_type) * split_segments(bn); }

// Which kernel, and how it cuts the work.
struct Plan {
  int bn;      // 0: CTA pairs; else rows per CTA of the split kernel
  int split;   // cluster size
};

// CTAs of clusters of S that are resident at once on a B200's 148 SMs (the occupancy
// query's answers), one CTA per SM and two.
inline constexpr int kRoom[2][kMaxSplit] = {{148, 148, 135, 132, 130, 132, 105, 120}, {296, 296, 279, 284, 280, 270, 259, 264}};

// An estimate of the split kernel's time in us in a stream of such calls: loads bound by the
// busiest SM (102 GB/s, 76 where a single CTA of a kind that shares its SM keeps but half
// of the bytes in flight, 0.59 us per block at 256 rows) or by HBM (6.6 TB/s, less with
// fewer CTAs than SMs), or a little longer than either where both are near; then the sums
// over the cluster and the epilogue.  Clusters of more than four cost extra (128 x 4096 x
// 4096 in parts of 128 rows: 13.1 us with four CTAs, 14.0 with eight and half the loads
// each): eight CTAs of one GPC have to be free at once.  The constants are a fit to 156
// products of 1 .. 4096 rows, every bn and cluster size timed: the choice is on average 0.7 %
// slower than the best of them and at most 15 %.
// `limit`: a time that is at least this is not worth working out to the end.
inline double split_time(const LinearArgs& a, int bn, int S, double limit) {
  const int per_sm = bn <= 128 ? 2 : 1, room = kRoom[per_sm - 1][S - 1];
  const int num_kb = (a.depth + kKb - 1) / kKb, kb = (num_kb + S - 1) / S;
  const int ctas = (a.rows + bn - 1) / bn * ((a.cols + 127) / 128) * S;   // at most 16 row tiles: 2^27 x S
  const double on_sm = (double)((ctas * per_sm + room - 1) / room), rounds = (double)((ctas + room - 1) / room);
  // the busiest SM ends a little faster where the others have less
  const double share = on_sm < 2 ? 1 : 0.713 * on_sm + 0.287 * std::max(1.0, (double)(ctas * per_sm) / room);
  const double mb = (128 + bn) * 128e-6;   // a block of both operands
  const double load = share * kb * std::max(mb / (on_sm < 2 && per_sm == 2 ? 0.0755 : 0.102), bn * 0.0023);
  const double hbm = ((double)a.rows + a.cols) * num_kb * kKb * 2e-6 / 6.6 * (1 + 0.54 * std::max(0.0, 1 - ctas / 160.0));
  const double most = std::max(load, hbm);
  if (2.41 + most >= limit) return limit;
  double near = std::min(load, hbm) / most;
  near *= near, near *= near, near *= near;
  const double n = std::min(bn, a.rows);
  static constexpr double kPow57[9] = {0, 1, 1.485, 1.871, 2.204, 2.503, 2.777, 3.032, 3.272};   // on_sm ^ 0.57
  double sums = S > 1 ? 0.248 + n * 0.016 * (S - 1) / S : 0;
  if (S > 4) sums += (0.108 + n * 0.0017) * (S - 4);
  return 2.41 + most * (1 + 0.13 * near) + sums * kPow57[std::min((int)on_sm, 8)] + n / S * 0.0151 * on_sm +
         n * 0.0043 + (rounds - 1) * 2.54;
}

// The same for the pair kernel: rounds of tiles over the pairs, or HBM (few rounds hide
// little of a cold start: 3.35 TB/s).
inline double pair_time(const LinearArgs& a) {
  const long num_kb = (a.depth + kKb - 1) / kKb;
  const long tiles = (long)((a.rows + 255) / 256) * ((a.cols + 255) / 256), pairs = a.num_sms / 2;
  const double rounds = (double)((tiles + pairs - 1) / pairs);
  const double hbm = ((double)a.rows + a.cols) * num_kb * kKb * 2e-6 / 3.35 + (double)a.rows * a.cols * 2e-6 / 5.0;
  return 2.85 + std::max(rounds * std::max(num_kb * 0.392, 0.38) + 2.59, hbm);
}

inline Plan plan(const LinearArgs& a) {
  Plan best = {0, 1};
  const bool f32 = a.out_type == kTypeF32;
  const int num_kb = (a.depth + kKb - 1) / kKb;
  // f32 sums leave TMEM every 8 blocks (dw 2048 x 4096 x 11008: 167 us against 147)
  double t = pair_time(a) * (f32 && num_kb > segment_blocks(kTypeF32) ? 1.15 : 1.0);
  for (int bn = a.op == kOpDw ? 64 : 16; bn <= 256; bn *= 2) {
    const long tiles = (long)((a.rows + bn - 1) / bn) * ((a.cols + 127) / 128);
    if (16L * bn < a.rows) continue;   // the fit's range: up to 16 row tiles, 4 CTAs per SM where split
    for (int S = 1; S <= std::min({kMaxSplit, num_kb, bn == 256 ? 4 : kMaxSplit}); ++S) {
      if (S > 1 && tiles * S > 4L * a.num_sms) break;
      if ((num_kb + S - 1) / S > split_blocks(bn, a.out_type)) continue;
      const double u = split_time(a, bn, S, t);
      if (u < t) t = u, best = {bn, S};
    }
    if (bn >= a.rows) break;
  }
  return best;
}

}  // namespace mlpg
