// layer_elem.cu -- the MLP layer's elementwise passes: the gradient of the product's
// epilogue (with the bias gradient's column sums) and dropout.
//
// One pass over the data, eight neighbouring columns (16 bytes) per thread and row.
// A CTA's 256 or 1024 threads form 2^lx column groups by as many rows as that leaves, so no
// index needs a division.  Each thread walks down its rows behind a ring of its own in
// shared memory that cp.async keeps kDepth - 1 rows ahead: the loads need no registers and
// no barrier, and the arithmetic of one row runs under the loads of the next ones.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "layer.cuh"
#include "ptx.cuh"

namespace mlpg {

namespace {

constexpr int kThreads = 256;

// The widest unit (16, 8, 4 or 2 bytes) on which every row of a matrix starts.
int row_unit(const void* p, long ld) {
  const uint64_t x = reinterpret_cast<uintptr_t>(p) | (uint64_t)(2 * ld) | 16u;
  return (int)(x & (~x + 1));
}

constexpr int kDepth = 4;
// act_grad adds the values of a thread's rows one by one.  Where there are more rows than this,
// each such run starts from zero and then joins the others: the roundings of equal values go
// the same way (a column of 270001 of them was 2e-5 off with 2100 in one run).
constexpr int kRun = 128;

// A thread's walk down its rows of one operand: the next row's address, and the unit in
// which its eight columns are read or written (2 for a group that ends behind the row).
struct Walk {
  const uint16_t* p;
  long step;      // elements from one of the thread's rows to the next
  int unit;
};

__device__ __forceinline__ Walk walk(const void* base, long ld, int unit, int r, int rows, int c, int cols) {
  return Walk{static_cast<const uint16_t*>(base) + (size_t)r * ld + c, ld * rows, c + 8 <= cols ? unit : 2};
}

template <int BYTES>
__device__ __forceinline__ void fetch_units(uint32_t dst, const uint16_t* p) {
#pragma unroll
  for (int i = 0; i < 16; i += BYTES)
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst + i), "l"(p + i / 2), "n"(BYTES) : "memory");
}

// The walk's row to shared memory: cp.async in whole units, else plain loads, with zeros
// past the row's end.  Units of 16 bytes are read once by one thread: L1 is passed by.
// WIDE: every operand's unit is 16, so that the narrower ones are not asked for (they cost
// an aligned act_grad 7 %).
template <bool WIDE>
__device__ __forceinline__ void fetch8(uint32_t dst, Walk& w, int c, int cols) {
  if (w.unit == 16) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(w.p) : "memory");
  } else if (!WIDE && w.unit == 8) {
    fetch_units<8>(dst, w.p);
  } else if (!WIDE && w.unit == 4) {
    fetch_units<4>(dst, w.p);
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

template <int TYPE, bool WIDE>
__device__ __forceinline__ void put8(const float (&v)[8], Walk& w, int c, int cols) {
  uint16_t* d = const_cast<uint16_t*>(w.p);
  if (w.unit == 16) {
    *reinterpret_cast<uint4*>(d) = pack8<TYPE>(v);
  } else if (!WIDE && w.unit >= 4) {   // 8 or 4 bytes: four words either way
    const uint4 q = pack8<TYPE>(v);
    uint32_t* d4 = reinterpret_cast<uint32_t*>(d);
    d4[0] = q.x, d4[1] = q.y, d4[2] = q.z, d4[3] = q.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < cols) store1<TYPE>(d, i, v[i]);
  }
  w.p += w.step;
}

// One or two operands' rows pass through f(row, words of the first, of the second) in
// order, from `r` on in steps of `rows`; `ring` is the thread's 16 bytes of slot 0.
template <int THREADS, int OPS, bool WIDE, typename F>
__device__ __forceinline__ void stream_rows(uint32_t ring, Walk a, Walk b, int r, int rows, int n, int c, int cols, F f) {
  constexpr uint32_t kOp = THREADS * 16, kSlot = OPS * kOp, kRing = kDepth * kSlot;
  static_assert((kRing & (kRing - 1)) == 0, "power of two");
  int next = r;
  uint32_t in = 0, out = 0;
  auto fetch = [&] {
    if (next < n) {
      fetch8<WIDE>(ring + in, a, c, cols);
      if constexpr (OPS == 2) fetch8<WIDE>(ring + in + kOp, b, c, cols);
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

// Bound by HBM: 4096 x 4096 bf16 with a residual 18.6 us, 5.4 TB/s (17.1 us without
// dropout); 33 x 4104 1.4 us.
template <int TYPE, bool RES, bool WIDE>
__global__ void __launch_bounds__(kThreads) dropout_kernel(const __grid_constant__ DropoutArgs p, int lx, int vx, int vr,
                                                           int vy) {
  __shared__ uint4 ring[kDepth * (RES ? 2 : 1) * kThreads];
  const int t = (int)threadIdx.x;
  const int g = (int)(blockIdx.x << lx) + (t & ((1 << lx) - 1)), c = 8 * g;
  if (c >= p.M) return;
  griddep_wait();
  const uint64_t off = drop_offset(p.drop);
  const int rows = (int)gridDim.y * (kThreads >> lx), r = (int)blockIdx.y * (kThreads >> lx) + (t >> lx);
  Walk y = walk(p.Y, p.ldy, vy, r, rows, c, p.M);
  stream_rows<kThreads, RES ? 2 : 1, WIDE>(smem_u32(ring + t), walk(p.X, p.ldx, vx, r, rows, c, p.M),
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
    put8<TYPE, WIDE>(v, y, c, p.M);
  });
  griddep_launch();
}

// A cluster's CTAs share the rows of one slab of columns.  Each thread's eight column
// sums meet the CTA's other rows in shared memory and the other CTAs' over distributed
// shared memory, always in the same order.
// 2048 x 11008 bf16 with the sums: 19.2 us without an activation (4.7 TB/s), 28 us with
// gelu (4.9 TB/s), 37 us with gelu and dropout.
// LONG: several runs per thread (in one kernel with the rest, that rest takes 1 to 4 % longer).
template <int TYPE, int ACT, int THREADS, bool WIDE, bool LONG>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) act_grad_kernel(const __grid_constant__ ActGradArgs p, int lx,
                                                                           int vy, int vz, int vd) {
  constexpr int kOps = ACT == kActNone ? 1 : 2;
  extern __shared__ uint4 ring[];                 // kDepth rows of one or two operands, LONG: and the runs' sums
  float* part = reinterpret_cast<float*>(ring);   // the sums, once the ring is drained
  const int t = (int)threadIdx.x, ty = THREADS >> lx, tx = 1 << lx;
  const int S = (int)gridDim.y, rank = (int)blockIdx.y;   // the cluster is the grid's y
  const int g = (int)(blockIdx.x << lx) + (t & (tx - 1)), c = 8 * g;
  float sum[8] = {};
  griddep_wait();
  if (c < p.M) {
    const uint64_t off = drop_offset(p.drop);
    const int rows = S * ty;
    int r = rank * ty + (t >> lx);
    Walk d = walk(p.dZ, p.lddz, vd, r, rows, c, p.M);
    auto run = [&](int end) {
      stream_rows<THREADS, kOps, WIDE>(smem_u32(ring + t), walk(p.dY, p.lddy, vy, r, rows, c, p.M),
                                       walk(p.Z, p.ldz, vz, r, rows, c, p.M), r, rows, end, c, p.M,
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
        if (p.dZ) put8<TYPE, WIDE>(v, d, c, p.M);
#pragma unroll
        for (int j = 0; j < 8; j += 2)
          split2(add2(pair2(sum[j], sum[j + 1]), pair2(v[j], v[j + 1])), sum[j], sum[j + 1]);
      });
    };
    if constexpr (LONG) {
      float4* total = reinterpret_cast<float4*>(ring + kDepth * kOps * THREADS) + 2 * t;
      total[0] = total[1] = make_float4(0.f, 0.f, 0.f, 0.f);
      for (; r < p.N; r += kRun * rows) {
        run(p.N - r > kRun * rows ? r + kRun * rows : p.N);
        const float4 x = total[0], y = total[1];
        total[0] = make_float4(x.x + sum[0], x.y + sum[1], x.z + sum[2], x.w + sum[3]);
        total[1] = make_float4(y.x + sum[4], y.y + sum[5], y.z + sum[6], y.w + sum[7]);
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[j] = 0.f;
      }
      const float4 x = total[0], y = total[1];
      sum[0] = x.x, sum[1] = x.y, sum[2] = x.z, sum[3] = x.w, sum[4] = y.x, sum[5] = y.y, sum[6] = y.z, sum[7] = y.w;
    } else {
      run(p.N);
    }
  }
  griddep_launch();
  if (!p.dbias) return;   // the same for the whole cluster
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 8; ++j) part[threadIdx.x * 8 + j] = sum[j];
  __syncthreads();
  // the rows' sums of one column are added by THREADS / cols threads, then theirs by one
  const int cols = 8 * tx, segs = THREADS >> (lx + 3), i = t & (cols - 1);
  float s = 0.f;
  for (int k = t >> (lx + 3); k < ty; k += segs) s += part[k * cols + i];
  __syncthreads();
  part[t] = s;
  __syncthreads();
  s = 0.f;
  if (t < cols)
    for (int k = 0; k < segs; ++k) s += part[k * cols + t];
  __syncthreads();
  if (t < cols) part[t] = s;
  cluster_sync();
  const int col = (int)blockIdx.x * cols + t;
  if (rank == 0 && t < cols && col < p.M) {
    float sum_all = 0.f;
    for (int k = 0; k < S; ++k) sum_all += __uint_as_float(ld_dsmem_u32(mapa_shared(&part[t], (uint32_t)k)));
    p.dbias[col] = sum_all;
  }
  cluster_sync_relaxed();   // no CTA leaves while its sums are read
}

int log2_up(int n, int most) {
  int l = 0;
  while (l < most && (1 << l) < n) ++l;
  return l;
}

// How a call is cut: 2^lx column groups per CTA, S CTAs (a cluster where there are sums)
// on the rows of a slab, threads per CTA.
struct GradPlan {
  int lx, S, threads;
};

// What counts, measured over all pairs of slab width and S at twelve shapes: SMs with equal
// numbers of CTAs, three or four of 256 threads each (2048 x 11008 with dropout: 1.2
// times as long with 86 slabs x 4 as with 86 x 8), four rows per thread (300 x 11008: 7.5 us with
// 86 x 4, 9.0 us with 86 x 8) and rows of whole 128-byte lines (2048 x 4096: 15.6 us with
// 64 slabs x 8, 18.3 us with 128 x 8).  Sizes of S between the powers of two never paid
// (2048 x 11008: 38.2 us with 172 x 6), clusters of 16 for narrow matrices alone (16384 x
// 64: 7.5 against 11.7 us).  CTAs of 1024 threads fill the SMs where few slabs with at most
// 8 CTAs on each would not (8192 x 1024: 16.0 against 19.7 us, 32768 x 512 without an
// activation: 18.1 against 31.2 us).
GradPlan grad_plan(const ActGradArgs& a) {
  // CTAs of clusters of 1, 2, 4, 8, 16 that are resident at once on 148 SMs
  static const long kRoom[2][5] = {{740, 740, 740, 740, 496}, {148, 148, 132, 120, 112}};
  static const double kLines[5] = {0, 0.6, 0.9, 0.98, 1.0};
  const int groups = (a.M + 7) / 8, most_lx = std::min(log2_up(groups, 4), 4);
  GradPlan best = {most_lx, 1, kThreads};
  if (!a.dbias) {   // rows go to any number of CTAs
    const long slabs = (groups + (1 << most_lx) - 1) >> most_lx, ty = kThreads >> most_lx;
    best.S = (int)std::min({((long)a.N + ty - 1) / ty, std::max(1L, 5L * a.num_sms / slabs), 65535L});
    return best;
  }
  double top = 0;
  for (int threads = kThreads; threads <= 1024; threads *= 4)
    for (int l = most_lx; l >= std::min(most_lx, 1); --l) {
      const long slabs = (groups + (1 << l) - 1) >> l, sms = a.num_sms;
      const int ty = threads >> l, most = slabs * 8 <= sms / 2 && threads == kThreads ? 16 : 8;
      for (int k = 1; k <= most && (k == 1 || k / 2 * ty < a.N); k *= 2) {
        const long ctas = slabs * k, room = kRoom[threads > kThreads][log2_up(k, 4)];
        const double even = ctas <= room ? (double)ctas / ((ctas + sms - 1) / sms * sms)
                                         : (double)ctas / ((ctas + room - 1) / room * (threads > kThreads ? sms : 5 * sms));
        const double fill = std::min(1.0, ctas * (threads / kThreads) / (3.5 * sms));
        const double depth = std::min(1.0, a.N / (4.0 * ty * k));
        const double score = even * std::sqrt(fill * depth) * kLines[std::max(l, 1)] * groups / (slabs << l) *
                             (threads == kThreads ? 1.0 : 0.9);
        if (score > top * 1.005) top = score, best = {l, k, threads};
      }
    }
  return best;
}

template <int TYPE, int ACT, int THREADS, bool WIDE, bool LONG>
cudaError_t launch_act_grad_kernel(const ActGradArgs& a, const GradPlan& pl) {
  auto kernel = act_grad_kernel<TYPE, ACT, THREADS, WIDE, LONG>;
  // the rings; at least, and LONG besides, the sums' 32 bytes a thread
  constexpr int smem = (kDepth * (ACT == kActNone ? 1 : 2) * 16 + (LONG ? 32 : 0)) * THREADS;
  static_assert(smem >= THREADS * 32, "sums");
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 1;
  attr[1].val.clusterDim.y = pl.S;
  attr[1].val.clusterDim.z = 1;
  cfg.gridDim = dim3(((a.M + 7) / 8 + (1 << pl.lx) - 1) >> pl.lx, pl.S);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = a.stream;
  cfg.attrs = attr;
  cfg.numAttrs = a.dbias ? 2 : 1;
  cudaError_t e = cudaSuccess;
  if (smem > 48 * 1024) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess && a.dbias && pl.S > 8)   // clusters above the portable size
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) return e;
  return cudaLaunchKernelEx(&cfg, kernel, a, pl.lx, row_unit(a.dY, a.lddy), row_unit(a.Z, a.ldz),
                            row_unit(a.dZ, a.lddz));
}

template <int TYPE, int ACT, int THREADS, bool WIDE>
cudaError_t launch_act_grad_typed(const ActGradArgs& a, const GradPlan& pl) {
  if (a.dbias && a.N > (long)kRun * pl.S * (THREADS >> pl.lx))
    return launch_act_grad_kernel<TYPE, ACT, THREADS, WIDE, true>(a, pl);
  return launch_act_grad_kernel<TYPE, ACT, THREADS, WIDE, false>(a, pl);
}

template <int TYPE, int ACT>
cudaError_t launch_act_grad_sized(const ActGradArgs& a) {
  const GradPlan pl = grad_plan(a);
  const bool wide = row_unit(a.dY, a.lddy) == 16 && (ACT == kActNone || row_unit(a.Z, a.ldz) == 16) &&
                    (!a.dZ || row_unit(a.dZ, a.lddz) == 16);
  if (pl.threads == 1024)
    return wide ? launch_act_grad_typed<TYPE, ACT, 1024, true>(a, pl) : launch_act_grad_typed<TYPE, ACT, 1024, false>(a, pl);
  return wide ? launch_act_grad_typed<TYPE, ACT, kThreads, true>(a, pl)
              : launch_act_grad_typed<TYPE, ACT, kThreads, false>(a, pl);
}

template <int TYPE>
cudaError_t launch_act_grad_act(const ActGradArgs& a) {
  switch (a.act) {
    case kActRelu: return launch_act_grad_sized<TYPE, kActRelu>(a);
    case kActGelu: return launch_act_grad_sized<TYPE, kActGelu>(a);
    case kActGeluTanh: return launch_act_grad_sized<TYPE, kActGeluTanh>(a);
    case kActSilu: return launch_act_grad_sized<TYPE, kActSilu>(a);
    default: return launch_act_grad_sized<TYPE, kActNone>(a);
  }
}

template <int TYPE>
auto dropout_pick(bool res, bool wide) {
  return res ? (wide ? dropout_kernel<TYPE, true, true> : dropout_kernel<TYPE, true, false>)
             : (wide ? dropout_kernel<TYPE, false, true> : dropout_kernel<TYPE, false, false>);
}

}  // namespace

cudaError_t launch_dropout(const DropoutArgs& a) {
  const int groups = (a.M + 7) / 8;
  // rows of CTAs: enough to fill the SMs six deep, each with rows left to walk down
  const int lx = log2_up(groups, 5), ty = kThreads >> lx;
  const long slabs = (groups + (1 << lx) - 1) >> lx;
  const long most = std::max(1L, 6L * a.num_sms / slabs);
  const dim3 grid((unsigned)slabs, (unsigned)std::min({((long)a.N + ty - 1) / ty, most, 65535L}));
  const int vx = row_unit(a.X, a.ldx), vr = row_unit(a.res, a.ldr), vy = row_unit(a.Y, a.ldy);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kThreads);
  cfg.stream = a.stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const bool wide = vx == 16 && vy == 16 && (!a.res || vr == 16);
  auto kernel = dropout_pick<kTypeBF16>(a.res, wide);
  if (a.type == kTypeF16) kernel = dropout_pick<kTypeF16>(a.res, wide);
  return cudaLaunchKernelEx(&cfg, kernel, a, lx, vx, vr, vy);
}

cudaError_t launch_act_grad(const ActGradArgs& a) {
  return a.type == kTypeF16 ? launch_act_grad_act<kTypeF16>(a) : launch_act_grad_act<kTypeBF16>(a);
}

}  // namespace mlpg
