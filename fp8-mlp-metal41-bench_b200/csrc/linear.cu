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
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(256);
  cfg.stream = a.stream;
  // the launch's own status: cudaGetLastError would answer with another call's
  const cudaError_t e = cudaLaunchKernelEx(&cfg, pack_rows_kernel, static_cast<const uint16_t*>(o.p), o.ld,
                                           reinterpret_cast<uint16_t*>(ws), o.rows, o.cols, groups);
  o.p = ws;
  o.ld = 8L * groups;
  ws += bytes;
  return e;
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
