// layer_elem.cu -- the MLP layer's elementwise passes: the gradient of the product's
// epilogue (with the bias gradient's column sums) and dropout.
//
// Both are bound by HBM: one pass over the data, eight neighbouring columns (16 bytes)
// per thread and step.
#include <cuda_runtime.h>

#include "layer.cuh"

namespace mlpg {

namespace {

// Rows whose 16-byte groups are aligned.
bool vec_rows(const void* p, long ld) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && ld % 8 == 0; }

template <int TYPE>
__global__ void __launch_bounds__(256) dropout_kernel(DropoutArgs p, int groups, bool vx, bool vr, bool vy) {
  const uint64_t off = drop_offset(p.drop);
  const long total = (long)p.N * groups;
  for (long i = blockIdx.x * 256L + threadIdx.x; i < total; i += gridDim.x * 256L) {
    const int r = (int)(i / groups), g = (int)(i % groups), c = 8 * g;
    float v[8];
    loadn<TYPE, 8>(v, p.X, (size_t)r * p.ldx + c, c, p.M, vx);
    if (p.drop.thr) drop8(v, p.drop, off, r, g);
    if (p.res) {
      float q[8];
      loadn<TYPE, 8>(q, p.res, (size_t)r * p.ldr + c, c, p.M, vr);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += q[j];
    }
    storen<TYPE, 8>(v, p.Y, (size_t)r * p.ldy + c, c, p.M, vy);
  }
}

// One CTA per 64 columns: 8 threads side by side, 32 rows at a time; a thread's eight
// column sums meet in shared memory in a fixed order.
template <int TYPE, int ACT>
__global__ void __launch_bounds__(256) act_grad_kernel(ActGradArgs p, bool vy, bool vz, bool vd) {
  __shared__ float part[32][64];
  const uint64_t off = drop_offset(p.drop);
  const int g = blockIdx.x * 8 + (threadIdx.x & 7), c = 8 * g, rr = threadIdx.x >> 3;
  float sum[8] = {};
  if (c < p.M)
    for (int r = rr; r < p.N; r += 32) {
      float v[8];
      loadn<TYPE, 8>(v, p.dY, (size_t)r * p.lddy + c, c, p.M, vy);
      if constexpr (ACT != kActNone) {
        float z[8];
        loadn<TYPE, 8>(z, p.Z, (size_t)r * p.ldz + c, c, p.M, vz);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= act_slope<ACT>(z[j]);
      }
      if (p.drop.thr) drop8(v, p.drop, off, r, g);
      if (p.dZ) storen<TYPE, 8>(v, p.dZ, (size_t)r * p.lddz + c, c, p.M, vd);
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
  const bool vx = vec_rows(a.X, a.ldx), vr = vec_rows(a.res, a.ldr), vy = vec_rows(a.Y, a.ldy);
  if (a.type == kTypeF16) dropout_kernel<kTypeF16><<<(unsigned)grid, 256, 0, a.stream>>>(a, groups, vx, vr, vy);
  else dropout_kernel<kTypeBF16><<<(unsigned)grid, 256, 0, a.stream>>>(a, groups, vx, vr, vy);
  return cudaGetLastError();
}

namespace {

template <int TYPE>
void act_grad_typed(const ActGradArgs& a) {
  const bool vy = vec_rows(a.dY, a.lddy), vz = vec_rows(a.Z, a.ldz), vd = vec_rows(a.dZ, a.lddz);
  const unsigned grid = (a.M + 63) / 64;
  switch (a.act) {
    case kActRelu: act_grad_kernel<TYPE, kActRelu><<<grid, 256, 0, a.stream>>>(a, vy, vz, vd); break;
    case kActGelu: act_grad_kernel<TYPE, kActGelu><<<grid, 256, 0, a.stream>>>(a, vy, vz, vd); break;
    case kActGeluTanh: act_grad_kernel<TYPE, kActGeluTanh><<<grid, 256, 0, a.stream>>>(a, vy, vz, vd); break;
    case kActSilu: act_grad_kernel<TYPE, kActSilu><<<grid, 256, 0, a.stream>>>(a, vy, vz, vd); break;
    default: act_grad_kernel<TYPE, kActNone><<<grid, 256, 0, a.stream>>>(a, vy, vz, vd); break;
  }
}

}  // namespace

cudaError_t launch_act_grad(const ActGradArgs& a) {
  if (a.type == kTypeF16) act_grad_typed<kTypeF16>(a);
  else act_grad_typed<kTypeBF16>(a);
  return cudaGetLastError();
}

}  // namespace mlpg
