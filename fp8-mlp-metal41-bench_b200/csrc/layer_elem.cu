// layer_elem.cu -- the MLP layer's elementwise passes: the gradient of the product's
// epilogue (with the bias gradient's column sums) and dropout.
//
// One pass over the data, eight neighbouring columns (16 bytes) per thread and row.
// The threads of a CTA form 2^lx column groups x 256 / 2^lx rows, so no index needs a
// division.  Each thread walks down its rows behind a ring of its own in shared memory
// that cp.async keeps kDepth - 1 rows ahead: the loads need no registers and no barrier,
// and the arithmetic of one row runs under the loads of the next ones.
#include <cuda_runtime.h>

#include <algorithm>

#include "layer.cuh"
#include "ptx.cuh"

namespace mlpg {

namespace {

constexpr int kThreads = 256;

// Rows whose 16-byte groups are aligned.
bool vec_rows(const void* p, long ld) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && ld % 8 == 0; }

constexpr int kDepth = 4;

// Eight elements from global to shared memory: cp.async where the rows allow it, else
// (and past the row's end, where zeros go) plain loads.  Read once: no L1.
__device__ __forceinline__ void fetch8(uint4* dst, const void* base, size_t at, int c, int cols, bool vec) {
  const uint16_t* p = static_cast<const uint16_t*>(base) + at;
  if (vec && c + 8 <= cols) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(p) : "memory");
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = (c + 2 * i < cols ? p[2 * i] : 0u) | ((uint32_t)(c + 2 * i + 1 < cols ? p[2 * i + 1] : 0u) << 16);
    *dst = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
__device__ __forceinline__ void fetch_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// all but the kDepth - 1 newest groups have landed
__device__ __forceinline__ void fetch_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory"); }

template <int TYPE, bool RES>
__global__ void __launch_bounds__(kThreads) dropout_kernel(const __grid_constant__ DropoutArgs p, int lx, bool vx, bool vr,
                                                           bool vy) {
  __shared__ uint4 ring[kDepth][RES ? 2 : 1][kThreads];
  const int t = (int)threadIdx.x;
  const int g = (int)(blockIdx.x << lx) + (t & ((1 << lx) - 1)), c = 8 * g;
  if (c >= p.M) return;
  const uint64_t off = drop_offset(p.drop);
  const long step = (long)gridDim.y * (kThreads >> lx);
  long next = (long)blockIdx.y * (kThreads >> lx) + (t >> lx);
  auto fetch = [&](int slot) {
    if (next < p.N) {
      fetch8(&ring[slot][0][t], p.X, (size_t)next * p.ldx + c, c, p.M, vx);
      if constexpr (RES) fetch8(&ring[slot][1][t], p.res, (size_t)next * p.ldr + c, c, p.M, vr);
    }
    fetch_commit();
    next += step;
  };
  long r = next;
#pragma unroll
  for (int d = 0; d < kDepth - 1; ++d) fetch(d);
  for (int slot = 0; r < p.N; r += step, slot = (slot + 1) % kDepth) {
    fetch((slot + kDepth - 1) % kDepth);
    const uint4 b = p.drop.on ? drop_bits(p.drop, off, (int)r, g) : make_uint4(0, 0, 0, 0);
    fetch_wait();
    float v[8];
    unpack8<TYPE>(v, ring[slot][0][t]);
    if (p.drop.on) drop8(v, p.drop, b);
    if constexpr (RES) {
      float w[8];
      unpack8<TYPE>(w, ring[slot][1][t]);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += w[j];
    }
    storen<TYPE, 8>(v, p.Y, (size_t)r * p.ldy + c, c, p.M, vy);
  }
}

// A cluster's CTAs share the rows of one slab of columns.  Each thread's eight column
// sums meet the CTA's other rows in shared memory and the other CTAs' over distributed
// shared memory, always in the same order.
template <int TYPE, int ACT>
__global__ void __launch_bounds__(kThreads, 4) act_grad_kernel(const __grid_constant__ ActGradArgs p, int lx, bool vy, bool vz,
                                                               bool vd) {
  __shared__ uint4 ring[kDepth][ACT == kActNone ? 1 : 2][kThreads];
  float* part = reinterpret_cast<float*>(ring);   // the sums, once the ring is drained
  const int t = (int)threadIdx.x, ty = kThreads >> lx, tx = 1 << lx;
  const int S = (int)gridDim.y, rank = (int)blockIdx.y;   // the cluster is the grid's y
  const int g = (int)(blockIdx.x << lx) + (t & (tx - 1)), c = 8 * g;
  float sum[8] = {};
  if (c < p.M) {
    const uint64_t off = drop_offset(p.drop);
    const long step = (long)S * ty;
    long next = (long)rank * ty + (t >> lx);
    auto fetch = [&](int slot) {
      if (next < p.N) {
        fetch8(&ring[slot][0][t], p.dY, (size_t)next * p.lddy + c, c, p.M, vy);
        if constexpr (ACT != kActNone) fetch8(&ring[slot][1][t], p.Z, (size_t)next * p.ldz + c, c, p.M, vz);
      }
      fetch_commit();
      next += step;
    };
    long r = next;
#pragma unroll
    for (int d = 0; d < kDepth - 1; ++d) fetch(d);
    for (int slot = 0; r < p.N; r += step, slot = (slot + 1) % kDepth) {
      fetch((slot + kDepth - 1) % kDepth);
      const uint4 b = p.drop.on ? drop_bits(p.drop, off, (int)r, g) : make_uint4(0, 0, 0, 0);
      fetch_wait();
      float v[8];
      unpack8<TYPE>(v, ring[slot][0][t]);
      if constexpr (ACT != kActNone) {
        float w[8];
        unpack8<TYPE>(w, ring[slot][1][t]);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= act_slope<ACT>(w[j]);
      }
      if (p.drop.on) drop8(v, p.drop, b);
      if (p.dZ) storen<TYPE, 8>(v, p.dZ, (size_t)r * p.lddz + c, c, p.M, vd);
#pragma unroll
      for (int j = 0; j < 8; ++j) sum[j] += v[j];
    }
  }
  if (!p.dbias) return;   // the same for the whole cluster
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 8; ++j) part[threadIdx.x * 8 + j] = sum[j];
  __syncthreads();
  // column i of the slab: thread i adds the rows' sums up
  const int cols = 8 * tx;
  float s = 0.f;
  if ((int)threadIdx.x < cols)
    for (int k = 0; k < ty; ++k) s += part[k * cols + (int)threadIdx.x];
  __syncthreads();
  if ((int)threadIdx.x < cols) part[threadIdx.x] = s;
  cluster_sync();
  const int col = (int)(blockIdx.x << lx) * 8 + (int)threadIdx.x;
  if (rank == 0 && (int)threadIdx.x < cols && col < p.M) {
    float t = 0.f;
    for (int k = 0; k < S; ++k) t += __uint_as_float(ld_dsmem_u32(mapa_shared(&part[threadIdx.x], (uint32_t)k)));
    p.dbias[col] = t;
  }
  cluster_sync_relaxed();   // no CTA leaves while its sums are read
}

int log2_up(int n, int most) {
  int l = 0;
  while (l < most && (1 << l) < n) ++l;
  return l;
}

template <int TYPE, int ACT>
cudaError_t launch_act_grad_typed(const ActGradArgs& a) {
  const int groups = (a.M + 7) / 8;
  // Column groups per CTA (32 to 128 columns) and CTAs per cluster: four CTAs fit an SM,
  // and what counts is that the last round over the SMs is full.
  int lx = log2_up(groups, 4), S = 1;
  double best = 0;
  for (int l = std::min(lx, 2); l <= std::min(lx, 4); ++l)
    for (int k = 1; k <= 8; ++k) {
      if (k > 1 && (long)a.N <= (long)(k - 1) * (kThreads >> l)) break;   // a CTA without rows
      const long slabs = (groups + (1 << l) - 1) >> l, ctas = slabs * k, sms = a.num_sms;
      const long room = 4 * sms, rounds = (ctas + room - 1) / room;
      const long last = ctas - (rounds - 1) * room;
      const double busy = (double)ctas / ((rounds - 1) * room + (last + sms - 1) / sms * sms);
      const double cols = (double)groups / (slabs << l);
      const double score = busy * cols * std::min(1.0, (double)ctas / (3 * sms)) * (l == 2 ? 0.9 : 1.0);
      if (score > best * 1.01) best = score, lx = l, S = k;
    }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = S;
  attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3((groups + (1 << lx) - 1) >> lx, S);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = a.stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, act_grad_kernel<TYPE, ACT>, a, lx, vec_rows(a.dY, a.lddy), vec_rows(a.Z, a.ldz),
                            vec_rows(a.dZ, a.lddz));
}

template <int TYPE>
cudaError_t launch_act_grad_act(const ActGradArgs& a) {
  switch (a.act) {
    case kActRelu: return launch_act_grad_typed<TYPE, kActRelu>(a);
    case kActGelu: return launch_act_grad_typed<TYPE, kActGelu>(a);
    case kActGeluTanh: return launch_act_grad_typed<TYPE, kActGeluTanh>(a);
    case kActSilu: return launch_act_grad_typed<TYPE, kActSilu>(a);
    default: return launch_act_grad_typed<TYPE, kActNone>(a);
  }
}

}  // namespace

cudaError_t launch_dropout(const DropoutArgs& a) {
  const int groups = (a.M + 7) / 8;
  // rows of CTAs: enough to fill the SMs six deep, each with rows left to walk down
  const int lx = log2_up(groups, 5), ty = kThreads >> lx;
  const long slabs = (groups + (1 << lx) - 1) >> lx;
  const long most = std::max(1L, 6L * a.num_sms / slabs);
  const dim3 grid((unsigned)slabs, (unsigned)std::min({((long)a.N + ty - 1) / ty, most, 65535L}));
  const bool vx = vec_rows(a.X, a.ldx), vr = vec_rows(a.res, a.ldr), vy = vec_rows(a.Y, a.ldy);
  if (a.type == kTypeF16) {
    if (a.res) dropout_kernel<kTypeF16, true><<<grid, kThreads, 0, a.stream>>>(a, lx, vx, vr, vy);
    else dropout_kernel<kTypeF16, false><<<grid, kThreads, 0, a.stream>>>(a, lx, vx, vr, vy);
  } else {
    if (a.res) dropout_kernel<kTypeBF16, true><<<grid, kThreads, 0, a.stream>>>(a, lx, vx, vr, vy);
    else dropout_kernel<kTypeBF16, false><<<grid, kThreads, 0, a.stream>>>(a, lx, vx, vr, vy);
  }
  return cudaGetLastError();
}

cudaError_t launch_act_grad(const ActGradArgs& a) {
  return a.type == kTypeF16 ? launch_act_grad_act<kTypeF16>(a) : launch_act_grad_act<kTypeBF16>(a);
}

}  // namespace mlpg
