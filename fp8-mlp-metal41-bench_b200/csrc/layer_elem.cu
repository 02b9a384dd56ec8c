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
#include <cmath>

#include "layer.cuh"
#include "ptx.cuh"

namespace mlpg {

namespace {

constexpr int kThreads = 256;

// Rows whose 16-byte groups are aligned.
bool vec_rows(const void* p, long ld) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && ld % 8 == 0; }

constexpr int kDepth = 4;

// A thread's walk down its rows of one operand: the next row's address, and whether its
// eight columns are one aligned 16-byte unit.
struct Walk {
  const uint16_t* p;
  long step;      // elements from one of the thread's rows to the next
  bool unit;
};

__device__ __forceinline__ Walk walk(const void* base, long ld, bool vec, int r, int rows, int c, int cols) {
  return Walk{static_cast<const uint16_t*>(base) + (size_t)r * ld + c, ld * rows, vec && c + 8 <= cols};
}

// The walk's row to shared memory: cp.async where it is one unit, else plain loads, with
// zeros past the row's end.  Every element is read once: L1 is passed by.
__device__ __forceinline__ void fetch8(uint32_t dst, Walk& w, int c, int cols) {
  if (w.unit) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(w.p) : "memory");
  } else {
    uint32_t q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      q[i] = (c + 2 * i < cols ? w.p[2 * i] : 0u) | ((uint32_t)(c + 2 * i + 1 < cols ? w.p[2 * i + 1] : 0u) << 16);
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(q[0]), "r"(q[1]), "r"(q[2]), "r"(q[3])
                 : "memory");
  }
  w.p += w.step;
}
__device__ __forceinline__ void fetch_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// all but the kDepth - 1 newest groups have landed
__device__ __forceinline__ void fetch_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory"); }

__device__ __forceinline__ uint4 lds16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

template <int TYPE>
__device__ __forceinline__ void put8(const float (&v)[8], Walk& w, int c, int cols) {
  storen<TYPE, 8>(v, const_cast<uint16_t*>(w.p), 0, c, cols, w.unit);
  w.p += w.step;
}

// One or two operands' rows pass through f(row, words of the first, of the second) in
// order, from `r` on in steps of `rows`; `ring` is the thread's 16 bytes of slot 0.
template <int OPS, typename F>
__device__ __forceinline__ void stream_rows(uint32_t ring, Walk a, Walk b, int r, int rows, int n, int c, int cols, F f) {
  constexpr uint32_t kOp = kThreads * 16, kSlot = OPS * kOp, kRing = kDepth * kSlot;
  static_assert((kRing & (kRing - 1)) == 0, "power of two");
  int next = r;
  uint32_t in = 0, out = 0;
  auto fetch = [&] {
    if (next < n) {
      fetch8(ring + in, a, c, cols);
      if constexpr (OPS == 2) fetch8(ring + in + kOp, b, c, cols);
    }
    fetch_commit();
    next += rows;
    in = (in + kSlot) & (kRing - 1);
  };
#pragma unroll
  for (int d = 0; d < kDepth - 1; ++d) fetch();
  for (; r < n; r += rows) {
    fetch();
    f(r, [&] { fetch_wait(); return lds16(ring + out); }, [&] { return lds16(ring + out + kOp); });
    out = (out + kSlot) & (kRing - 1);
  }
}

template <int TYPE, bool RES>
__global__ void __launch_bounds__(kThreads) dropout_kernel(const __grid_constant__ DropoutArgs p, int lx, bool vx, bool vr,
                                                           bool vy) {
  __shared__ uint4 ring[kDepth * (RES ? 2 : 1) * kThreads];
  const int t = (int)threadIdx.x;
  const int g = (int)(blockIdx.x << lx) + (t & ((1 << lx) - 1)), c = 8 * g;
  if (c >= p.M) return;
  griddep_wait();
  const uint64_t off = drop_offset(p.drop);
  const int rows = (int)gridDim.y * (kThreads >> lx), r = (int)blockIdx.y * (kThreads >> lx) + (t >> lx);
  Walk y = walk(p.Y, p.ldy, vy, r, rows, c, p.M);
  stream_rows<RES ? 2 : 1>(smem_u32(ring + t), walk(p.X, p.ldx, vx, r, rows, c, p.M),
                           walk(p.res, p.ldr, vr, r, rows, c, p.M), r, rows, p.N, c, p.M,
                           [&](int row, auto first, auto second) {
    const uint4 b = p.drop.on ? drop_bits(p.drop, off, row, g) : make_uint4(0, 0, 0, 0);
    float v[8];
    unpack8<TYPE>(v, first());
    if (p.drop.on) drop8(v, p.drop, b);
    if constexpr (RES) {
      float w[8];
      unpack8<TYPE>(w, second());
#pragma unroll
      for (int j = 0; j < 8; j += 2) split2(add2(pair2(v[j], v[j + 1]), pair2(w[j], w[j + 1])), v[j], v[j + 1]);
    }
    put8<TYPE>(v, y, c, p.M);
  });
  griddep_launch();
}

// A cluster's CTAs share the rows of one slab of columns.  Each thread's eight column
// sums meet the CTA's other rows in shared memory and the other CTAs' over distributed
// shared memory, always in the same order.
template <int TYPE, int ACT>
__global__ void __launch_bounds__(kThreads, 4) act_grad_kernel(const __grid_constant__ ActGradArgs p, int lx, bool vy, bool vz,
                                                               bool vd) {
  __shared__ uint4 ring[kDepth * (ACT == kActNone ? 1 : 2) * kThreads];
  float* part = reinterpret_cast<float*>(ring);   // the sums, once the ring is drained
  const int t = (int)threadIdx.x, ty = kThreads >> lx, tx = 1 << lx;
  const int S = (int)gridDim.y, rank = (int)blockIdx.y;   // the cluster is the grid's y
  const int g = (int)(blockIdx.x << lx) + (t & (tx - 1)), c = 8 * g;
  float sum[8] = {};
  griddep_wait();
  if (c < p.M) {
    const uint64_t off = drop_offset(p.drop);
    const int rows = S * ty, r = rank * ty + (t >> lx);
    Walk d = walk(p.dZ, p.lddz, vd, r, rows, c, p.M);
    stream_rows<ACT == kActNone ? 1 : 2>(smem_u32(ring + t), walk(p.dY, p.lddy, vy, r, rows, c, p.M),
                                         walk(p.Z, p.ldz, vz, r, rows, c, p.M), r, rows, p.N, c, p.M,
                                         [&](int row, auto first, auto second) {
      const uint4 b = p.drop.on ? drop_bits(p.drop, off, row, g) : make_uint4(0, 0, 0, 0);
      float v[8];
      unpack8<TYPE>(v, first());
      if constexpr (ACT != kActNone) {
        float w[8];
        unpack8<TYPE>(w, second());
#pragma unroll
        for (int j = 0; j < 8; j += 2)
          split2(mul2(pair2(v[j], v[j + 1]), act_slope2<ACT>(pair2(w[j], w[j + 1]))), v[j], v[j + 1]);
      }
      if (p.drop.on) drop8(v, p.drop, b);
      if (p.dZ) put8<TYPE>(v, d, c, p.M);
#pragma unroll
      for (int j = 0; j < 8; j += 2)
        split2(add2(pair2(sum[j], sum[j + 1]), pair2(v[j], v[j + 1])), sum[j], sum[j + 1]);
    });
  }
  griddep_launch();
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
  // Columns per CTA (16 to 128) and CTAs per cluster.  What counts, measured over all
  // pairs at nine shapes: SMs with equal numbers of CTAs, three or four each (2048 x 11008
  // with dropout: 35.2 us with 86 slabs x 8 = 4.65 per SM, 41.6 us with 86 x 4 = 2.3),
  // four rows per thread (300 x 11008: 7.3 us with 86 x 4, 9.3 us with 86 x 8) and rows
  // of whole 128-byte lines (8192 x 1024: 17 us with 32 slabs x 8, 20 us with 64 x 8);
  // clusters of 16 pay for narrow matrices alone (16384 x 64: 7.8 against 12 us), and
  // sizes between the powers of two do not (172 x 6: 38.2 us).
  static const double kLines[5] = {0, 0.6, 0.9, 0.98, 1.0};
  int lx = log2_up(groups, 4), S = 1;
  double best = 0;
  for (int l = std::min(lx, 4); l >= std::min(lx, 1); --l) {
    const long slabs = (groups + (1 << l) - 1) >> l, sms = a.num_sms;
    const int ty = kThreads >> l;
    const int most = slabs * 8 <= sms / 2 ? 16 : 8;
    for (int k = 1; k <= most && (k == 1 || k / 2 * ty < a.N); k *= 2) {
      const long ctas = slabs * k;
      const double even = (double)ctas / ((ctas + sms - 1) / sms * sms);
      const double fill = std::min(1.0, ctas / (3.5 * sms)), depth = std::min(1.0, a.N / (4.0 * ty * k));
      const double score = even * std::sqrt(fill * depth) * kLines[std::max(l, 1)] * groups / (slabs << l);
      if (score > best * 1.005) best = score, lx = l, S = k;
    }
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = S;
  attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3((groups + (1 << lx) - 1) >> lx, S);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = a.stream;
  cfg.attrs = attr;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = 2;
  if (S > 8) {   // clusters above the portable size
    const cudaError_t e = cudaFuncSetAttribute(act_grad_kernel<TYPE, ACT>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
  }
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
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kThreads);
  cfg.stream = a.stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  auto kernel = a.type == kTypeF16 ? (a.res ? dropout_kernel<kTypeF16, true> : dropout_kernel<kTypeF16, false>)
                                   : (a.res ? dropout_kernel<kTypeBF16, true> : dropout_kernel<kTypeBF16, false>);
  return cudaLaunchKernelEx(&cfg, kernel, a, lx, vx, vr, vy);
}

cudaError_t launch_act_grad(const ActGradArgs& a) {
  return a.type == kTypeF16 ? launch_act_grad_act<kTypeF16>(a) : launch_act_grad_act<kTypeBF16>(a);
}

}  // namespace mlpg
