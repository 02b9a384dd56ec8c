// linear.cu -- the MLP layer's products: Y = R + drop(act(X W + b)) and the two
// gradient products dX = R + dZ W^T, dW = R + X^T dZ.
#include <cuda_runtime.h>

#include "layer.cuh"

namespace mlpg {

namespace {

// 64 x 64 outputs per CTA, 4 x 4 per thread, f32 sums over 16-deep slices in shared
// memory.  Row[r, c] = A[r * ar + c * ac], Col[c, k] = B[c * bc + k * bk].
constexpr int kT = 64, kD = 16;

__global__ void __launch_bounds__(256) linear_kernel(LinearArgs p, long ar, long ac, long bc, long bk, int tiles_r) {
  __shared__ float sa[kD][kT + 1], sb[kD][kT + 1];
  const int r0 = (int)(blockIdx.x % tiles_r) * kT, c0 = (int)(blockIdx.x / tiles_r) * kT;
  const int t = threadIdx.x, tr = t / 16, tc = t % 16;
  float acc[4][4] = {};
  for (int d0 = 0; d0 < p.depth; d0 += kD) {
    for (int i = t; i < kT * kD; i += 256) {
      const int x = i % kT, d = i / kT;
      sa[d][x] = (r0 + x < p.rows && d0 + d < p.depth) ? load1(p.A, (size_t)(r0 + x) * ar + (size_t)(d0 + d) * ac, p.type) : 0.f;
      sb[d][x] = (c0 + x < p.cols && d0 + d < p.depth) ? load1(p.B, (size_t)(d0 + d) * bc + (size_t)(c0 + x) * bk, p.type) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int d = 0; d < kD; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] += sa[d][tr + 16 * i] * sb[d][tc + 16 * j];
    __syncthreads();
  }
  const uint64_t off = drop_offset(p.drop);
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int r = r0 + tr + 16 * i, c = c0 + tc + 16 * j;
      if (r >= p.rows || c >= p.cols) continue;
      float v = acc[i][j];
      if (p.bias) v += load1(p.bias, c, p.type);
      if (p.pre) store1(p.pre, (size_t)r * p.ldz + c, v, p.type);
      v = act_fwd(v, p.act);
      if (p.drop.thr) v = drop1(v, p.drop, off, r, c);
      if (p.res) v += load1(p.res, (size_t)r * p.ldr + c, p.out_type);
      store1(p.out, (size_t)r * p.ldo + c, v, p.out_type);
    }
}

}  // namespace

size_t linear_workspace(const LinearArgs&) { return 0; }

cudaError_t launch_linear(const LinearArgs& a) {
  const int tiles_r = (a.rows + kT - 1) / kT, tiles_c = (a.cols + kT - 1) / kT;
  const long ar = a.op == kOpDw ? 1 : a.lda, ac = a.op == kOpDw ? a.lda : 1;
  const long bc = a.op == kOpDx ? 1 : a.ldb, bk = a.op == kOpDx ? a.ldb : 1;
  linear_kernel<<<(unsigned)tiles_r * tiles_c, 256, 0, a.stream>>>(a, ar, ac, bc, bk, tiles_r);
  return cudaGetLastError();
}

}  // namespace mlpg
