// layer_elem.cu -- the MLP layer's elementwise passes: the gradient of the product's
// epilogue (with the bias gradient's column sums) and dropout.
//
// Both are bound by HBM: one pass over the data, eight neighbouring columns (16 bytes)
// per thread and step.
#include <cuda_runtime.h>

#include "layer.cuh"

namespace mlpg {

namespace {

// Eight elements of a row from column c on; those past `cols` read as 0.
__device__ __forceinline__ void load8(float (&v)[8], const void* base, size_t at, int c, int cols, int type, bool vec) {
  if (vec && c + 8 <= cols) {
    const uint4 w = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + at);
    const uint32_t q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack2(q[i], type);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < cols ? load1(base, at + i, type) : 0.f;
  }
}

__device__ __forceinline__ void store8(const float (&v)[8], void* base, size_t at, int c, int cols, int type, bool vec) {
  if (vec && c + 8 <= cols) {
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + at) =
        make_uint4(pack2(v[0], v[1], type), pack2(v[2], v[3], type), pack2(v[4], v[5], type), pack2(v[6], v[7], type));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < cols) store1(base, at + i, v[i], type);
  }
}

// Rows whose 16-byte groups are aligned.
bool vec_rows(const void* p, long ld) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && ld % 8 == 0; }

__global__ void __launch_bounds__(256) dropout_kernel(DropoutArgs p, int groups, bool vx, bool vr, bool vy) {
  const uint64_t off = drop_offset(p.drop);
  const long total = (long)p.N * groups;
  for (long i = blockIdx.x * 256L + threadIdx.x; i < total; i += gridDim.x * 256L) {
    const int r = (int)(i / groups), g = (int)(i % groups), c = 8 * g;
    float v[8];
    load8(v, p.X, (size_t)r * p.ldx + c, c, p.M, p.type, vx);
    if (p.drop.thr) drop8(v, p.drop, off, r, g);
    if (p.res) {
      float q[8];
      load8(q, p.res, (size_t)r * p.ldr + c, c, p.M, p.type, vr);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += q[j];
    }
    store8(v, p.Y, (size_t)r * p.ldy + c, c, p.M, p.type, vy);
  }
}

// One CTA per 64 columns: 8 threads side by side, 32 rows at a time; a thread's eight
// column sums meet in shared memory in a fixed order.
__global__ void __launch_bounds__(256) act_grad_kernel(ActGradArgs p, bool vy, bool vz, bool vd) {
  __shared__ float part[32][64];
  const uint64_t off = drop_offset(p.drop);
  const int g = blockIdx.x * 8 + (threadIdx.x & 7), c = 8 * g, rr = threadIdx.x >> 3;
  float sum[8] = {};
  if (c < p.M)
    for (int r = rr; r < p.N; r += 32) {
      float v[8];
      load8(v, p.dY, (size_t)r * p.lddy + c, c, p.M, p.type, vy);
      if (p.act != kActNone) {
        float z[8];
        load8(z, p.Z, (size_t)r * p.ldz + c, c, p.M, p.type, vz);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= act_slope(z[j], p.act);
      }
      if (p.drop.thr) drop8(v, p.drop, off, r, g);
      if (p.dZ) store8(v, p.dZ, (size_t)r * p.lddz + c, c, p.M, p.type, vd);
#pragma unroll
      for (int j = 0; j < 8; ++j) sum[j] += v[j];
    }
  if (!p.dbias) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) part[rr][(threadIdx.x & 7) * 8 + j] = sum[j];
  __syncthreads();
  const int col = blockIdx.x * 64 + threadIdx.x;
  if (threadIdx.x < 64 && col < p.M) {
    float s = 0.f;
    for (int i = 0; i < 32; ++i) s += part[i][threadIdx.x];
    p.dbias[col] = s;
  }
}

}  // namespace

cudaError_t launch_dropout(const DropoutArgs& a) {
  const int groups = (a.M + 7) / 8;
  long grid = ((long)a.N * groups + 255) / 256;
  if (grid > 16L * a.num_sms) grid = 16L * a.num_sms;
  dropout_kernel<<<(unsigned)grid, 256, 0, a.stream>>>(a, groups, vec_rows(a.X, a.ldx), vec_rows(a.res, a.ldr),
                                                       vec_rows(a.Y, a.ldy));
  return cudaGetLastError();
}

cudaError_t launch_act_grad(const ActGradArgs& a) {
  act_grad_kernel<<<(a.M + 63) / 64, 256, 0, a.stream>>>(a, vec_rows(a.dY, a.lddy), vec_rows(a.Z, a.ldz),
                                                         vec_rows(a.dZ, a.lddz));
  return cudaGetLastError();
}

}  // namespace mlpg
