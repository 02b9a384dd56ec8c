// linear.cuh -- the MLP layer's products on tcgen05: Y = R + drop(act(X W + b)) and the
// two gradient products dX = R + dZ W^T, dW = R + X^T dZ, f16 or bf16 operands, f32
// accumulators in TMEM, one rounding of each result.
//
// Two kernels share the operand layouts (an operand whose contraction index is
// contiguous is K-major, else MN-major; both come straight from the caller's rows by
// TMA with the 128-byte swizzle) and the epilogue's arithmetic:
//
//   linear_pair.cu    persistent, 256 x 256 tiles on CTA pairs, for many tiles
//   linear_split.cu   128 columns x BN rows per CTA, the contraction split over a
//                     cluster: few rows, where the weights' bytes bound the call
//   linear_plan.h     the choice between them
//   linear.cu         operands that the TMA cannot read
//
// Every mbarrier wait is bounded (ptx.cuh); on expiry a kernel records an error
// word, lets its TMA copies land, frees TMEM and returns.  No load uses multicast.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <mutex>

#include "layer.cuh"
#include "linear_plan.h"
#include "ptx.cuh"
#include "tmap.h"

namespace mlpg {

constexpr int kBoxBytes = 64 * 128;   // one MN-major box: 64 contraction rows x 64 elements
constexpr int kSmemMax = 232448;

struct EpiArgs {
  const void *bias, *res;
  void *out, *pre;
  long ldo, ldr, ldz;
  int act;
  int rows, cols, depth;
  DropArgs drop;
  bool bias_vec, out_vec, res_vec, pre_vec;   // 16-byte aligned base and rows
  int* dev_err;
};

// v += bias[c .. c+7]; columns at or past `cols` keep their value
template <int TYPE>
__device__ __forceinline__ void add_bias8(float (&v)[8], const EpiArgs& p, int c) {
  float b[8];
  loadn<TYPE, 8>(b, p.bias, (size_t)c, c, p.cols, p.bias_vec);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] += b[i];
}

__device__ __forceinline__ uint64_t op_desc(uint32_t addr, bool mn, int kk) {
  // 16 deep: 32 bytes along a K-major row, 16 rows of 128 bytes of an MN-major box
  return mn ? sdesc_sw128(addr + kk * 2048, kBoxBytes, 1024) : sdesc_sw128(addr + kk * 32, 16, 1024);
}

// ---- host ---------------------------------------------------------------------------------

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// The TMA reads rows whose base and distance are multiples of 16 bytes (a single row
// has no distance).
inline bool tma_rows(const void* p, long ld, int rows, int es) { return aligned16(p) && (rows == 1 || ld * es % 16 == 0); }

// A stored 16-bit operand [rows, cols].
struct Operand {
  const void* p;
  long ld;
  int rows, cols;
  size_t packed() const {
    return tma_rows(p, ld, rows, 2) ? 0 : ((size_t)rows * ((cols + 7) / 8) * 16 + 255) / 256 * 256;
  }
};

// 2-D map of [rows, cols] elements of es bytes in boxes of 128-byte rows, 128-byte swizzle
inline bool map_rows(CUtensorMap* m, const void* p, long ld, int rows, int cols, int es, int box_rows) {
  const uint64_t pitch = rows == 1 ? ((uint64_t)cols * es + 15) / 16 * 16 : (uint64_t)ld * es;
  return make_map(m, p, es == 2 ? CU_TENSOR_MAP_DATA_TYPE_UINT16 : CU_TENSOR_MAP_DATA_TYPE_UINT32, (uint64_t)cols,
                  (uint64_t)rows, pitch, 128 / es, (uint32_t)box_rows);
}

inline EpiArgs epilogue(const LinearArgs& a) {
  EpiArgs e = {};
  e.bias = a.bias;
  e.res = a.res;
  e.out = a.out;
  e.pre = a.pre;
  e.ldo = a.ldo;
  e.ldr = a.ldr;
  e.ldz = a.ldz;
  e.act = a.act;
  e.rows = a.rows;
  e.cols = a.cols;
  e.depth = a.depth;
  e.drop = a.drop;
  e.bias_vec = aligned16(a.bias);
  const int es = a.out_type == kTypeF32 ? 4 : 2;
  e.out_vec = aligned16(a.out) && a.ldo * es % 16 == 0;
  e.res_vec = aligned16(a.res) && a.ldr * es % 16 == 0;
  e.pre_vec = aligned16(a.pre) && a.ldz % 8 == 0;
  e.dev_err = a.dev_err;
  return e;
}

// Per device: a kernel's dynamic shared memory is set, its co-resident clusters counted.
struct Once {
  std::mutex mu;
  unsigned mask = 0;
  int value[32] = {0};
};

template <typename Kernel>
cudaError_t prepare(Once& once, Kernel k, int smem, cudaLaunchConfig_t& cfg, int* clusters) {
  int dev = 0;
  cudaGetDevice(&dev);
  dev &= 31;
  std::lock_guard<std::mutex> lk(once.mu);
  if (!(once.mask & (1u << dev))) {
    cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    int n = 0;
    if (clusters && (e = cudaOccupancyMaxActiveClusters(&n, k, &cfg)) != cudaSuccess) return e;
    once.value[dev] = n;
    once.mask |= 1u << dev;
  }
  if (clusters) *clusters = once.value[dev];
  return cudaSuccess;
}

// rows_op, cols_op: the stored operands whose rows or columns index the result's rows
// and columns (A and B of LinearArgs, packed where they had to be)
cudaError_t launch_pair(const LinearArgs& a, const Operand& rows_op, const Operand& cols_op);
// bn rows per CTA (16, 32, 64, 128, 256; dW from 64), clusters of `split`; at most split_blocks
// blocks of the contraction per CTA
cudaError_t launch_split(const LinearArgs& a, const Operand& rows_op, const Operand& cols_op, int bn, int split);

}  // namespace mlpg
