// linear.cu -- the layer's products: which kernel runs a call, and operands that the
// TMA cannot read.
#include <algorithm>

#include "linear.cuh"

namespace mlpg {

namespace {

// ---- operands that the TMA cannot read ---------------------------------------------------
// Rows of any alignment copied to rows of whole 16 bytes.
__global__ void __launch_bounds__(256) pack_rows_kernel(const uint16_t* __restrict__ src, long ld, uint16_t* __restrict__ dst,
                                                        int rows, int cols, int groups) {
  const long total = (long)rows * groups;
  for (long i = blockIdx.x * 256L + threadIdx.x; i < total; i += gridDim.x * 256L) {
    const int r = (int)(i / groups), g = (int)(i % groups);
    const uint16_t* s = src + (size_t)r * ld + 8 * g;
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t lo = 8 * g + 2 * j < cols ? s[2 * j] : 0u, hi = 8 * g + 2 * j + 1 < cols ? s[2 * j + 1] : 0u;
      w[j] = lo | (hi << 16);
    }
    reinterpret_cast<uint4*>(dst)[i] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

void stored(const LinearArgs& a, Operand& x, Operand& y) {
  const int n = a.op == kOpDw ? a.depth : a.rows;
  x = Operand{a.A, a.lda, n, a.op == kOpDx || a.op == kOpLinear ? a.depth : a.rows};
  y = Operand{a.B, a.ldb, a.op == kOpLinear ? a.depth : (a.op == kOpDx ? a.cols : a.depth),
              a.op == kOpDx ? a.depth : a.cols};
}

cudaError_t pack(Operand& o, unsigned char*& ws, const LinearArgs& a) {
  const size_t bytes = o.packed();
  if (!bytes) return cudaSuccess;
  const int groups = (o.cols + 7) / 8;
  const long grid = std::min(((long)o.rows * groups + 255) / 256, 16L * a.num_sms);
  pack_rows_kernel<<<(unsigned)grid, 256, 0, a.stream>>>(static_cast<const uint16_t*>(o.p), o.ld,
                                                         reinterpret_cast<uint16_t*>(ws), o.rows, o.cols, groups);
  o.p = ws;
  o.ld = 8L * groups;
  ws += bytes;
  return cudaGetLastError();
}

// Which kernel, and how it cuts the work.
struct Plan {
  int bn;      // 0: CTA pairs; else rows per CTA of the split kernel
  int split;   // cluster size
};

// CTAs of clusters of S that are resident at once on a B200's 148 SMs (the occupancy
// query's answers), one CTA per SM and two.
constexpr int kRoom[2][kMaxSplit] = {{148, 148, 135, 132, 130, 132, 105, 120}, {296, 296, 279, 284, 280, 270, 259, 264}};

// An estimate of the split kernel's time in us in a stream of such calls: loads bound by the
// busiest SM (102 GB/s, 76 where a single CTA of a kind that shares its SM keeps but half
// of the bytes in flight, 0.59 us per block at 256 rows) or by HBM (6.6 TB/s, less with
// fewer CTAs than SMs), or a little longer than either where both are near; then the sums
// over the cluster and the epilogue.  Clusters of more than four cost extra (128 x 4096 x
// 4096 in parts of 128 rows: 13.1 us with four CTAs, 14.0 with eight and half the loads
// each): eight CTAs of one GPC have to be free at once.  The constants are a fit to 156
// products of 1 .. 4096 rows, every bn and cluster size timed: the choice is on average 0.7 %
// slower than the best of them and at most 15 %.
double split_time(const LinearArgs& a, int bn, int S) {
  const int per_sm = bn <= 128 ? 2 : 1, room = kRoom[per_sm - 1][S - 1];
  const long num_kb = (a.depth + kKb - 1) / kKb, kb = (num_kb + S - 1) / S;
  const long ctas = (long)((a.rows + bn - 1) / bn) * ((a.cols + 127) / 128) * S;
  const double on_sm = (double)((ctas * per_sm + room - 1) / room), rounds = (double)((ctas + room - 1) / room);
  // the busiest SM ends a little faster where the others have less
  const double share = on_sm < 2 ? 1 : 0.713 * on_sm + 0.287 * std::max(1.0, (double)(ctas * per_sm) / room);
  const double mb = (128 + bn) * 128e-6;   // a block of both operands
  const double load = share * kb * std::max(mb / (on_sm < 2 && per_sm == 2 ? 0.0755 : 0.102), bn * 0.0023);
  const double hbm = ((double)a.rows + a.cols) * num_kb * kKb * 2e-6 / 6.6 * (1 + 0.54 * std::max(0.0, 1 - ctas / 160.0));
  const double most = std::max(load, hbm);
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
double pair_time(const LinearArgs& a) {
  const long num_kb = (a.depth + kKb - 1) / kKb;
  const long tiles = (long)((a.rows + 255) / 256) * ((a.cols + 255) / 256), pairs = a.num_sms / 2;
  const double rounds = (double)((tiles + pairs - 1) / pairs);
  const double hbm = ((double)a.rows + a.cols) * num_kb * kKb * 2e-6 / 3.35 + (double)a.rows * a.cols * 2e-6 / 5.0;
  return 2.85 + std::max(rounds * std::max(num_kb * 0.392, 0.38) + 2.59, hbm);
}

Plan plan(const LinearArgs& a) {
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
      const double u = split_time(a, bn, S);
      if (u < t) t = u, best = {bn, S};
    }
    if (bn >= a.rows) break;
  }
  return best;
}

}  // namespace

size_t linear_workspace(const LinearArgs& a) {
  Operand x, y;
  stored(a, x, y);
  return x.packed() + y.packed();
}

cudaError_t launch_linear(const LinearArgs& a) {
  Operand x, y;
  stored(a, x, y);
  unsigned char* ws = static_cast<unsigned char*>(a.ws);
  cudaError_t e;
  if ((e = pack(x, ws, a)) != cudaSuccess || (e = pack(y, ws, a)) != cudaSuccess) return e;
  const Plan pl = plan(a);
  return pl.bn ? launch_split(a, x, y, pl.bn, pl.split) : launch_pair(a, x, y);
}

}  // namespace mlpg
