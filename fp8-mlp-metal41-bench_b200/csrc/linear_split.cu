// linear_split.cu -- the layer's products for few rows: the contraction split over a
// thread-block cluster.
#include "linear.cuh"

namespace mlpg {

namespace {

// ---- few rows -----------------------------------------------------------------------------
// One CTA computes 128 columns x BN rows over its share of the contraction, with the
// columns as the MMA's 128 lanes (so a single row still fills the tensor core's M and
// the epilogue's threads).  The cluster's CTAs split the contraction, put their partial
// sums into their own shared memory, and each then sums and finishes its share of the
// tile over distributed shared memory, in rank order: no workspace, no atomics, the
// same result every time.
//
// Bound by HBM while the weights are read once: 1 x 4096 x 11008 bf16 16.3 us, 5.5 TB/s of
// weights with the launch and the sums in it; 13 x 11008 x 4096 17.5 us.  From 64 rows on by
// what an SM reads from L2 (about 100 GB/s): 256 x 4096 x 4096 15.4 us.
//
// A CTA's partial sums lie side by side in TMEM and are added with rounding when they are
// read out (dW 8192 x 1024 x 1024 in f32: 32.6 us, the pair kernel 47 us).
constexpr int kSplitThreads = 256;

template <int OP, int BN, bool DEEP>
struct SplitCfg {
  static constexpr bool C_MN = OP != kOpDx, R_MN = OP == kOpDw;
  static constexpr int C_BYTES = 128 * 128, R_BYTES = BN * 128;
  static constexpr int STAGE_BYTES = C_BYTES + R_BYTES;
  // BN <= 128: two CTAs per SM, about 100 KB each in flight (one CTA per SM with ten stages
  // streams W more slowly: 1 x 4096 x 11008 18.8 against 16.5 us)
  static constexpr int STAGES = BN <= 32 ? 5 : (BN == 128 ? 3 : 4);
  static constexpr int PER_SM = BN <= 128 ? 2 : 1;
  static constexpr int BAR_OFF = STAGES * STAGE_BYTES;
  static constexpr int SMEM = BAR_OFF + 512 + 1024;
  static constexpr int SEGS = DEEP ? split_segments(BN) : 1;   // accumulators
  static constexpr uint32_t TMEM_COLS = BN < 32 && !DEEP ? 32 : SEGS * BN;
  static constexpr uint32_t IDESC = (1u << 4) | ((C_MN ? 1u : 0u) << 15) | ((R_MN ? 1u : 0u) << 16) |
                                    ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
  static_assert(BN * 512 <= BAR_OFF, "partial sums fit the ring");
  static_assert(SMEM * PER_SM <= kSmemMax, "shared memory budget");
  static_assert(TMEM_COLS * PER_SM <= 512, "TMEM budget");
  static_assert(SMEM > 228 * 1024 - 160 * 1024, "no room beside the peak probe (peak.cu)");
  static_assert((PER_SM + 1) * SMEM > 228 * 1024, "no third CTA on an SM, so none waits for TMEM");
  static_assert(!R_MN || BN % 64 == 0, "whole MN boxes");
};

struct SplitBars {
  uint64_t full[8], empty[8], acc;
  uint32_t tmem_base;
  int abort_flag;
};

template <bool MN>
__device__ __forceinline__ void load_op(unsigned char* dst, const CUtensorMap* m, uint64_t* bar, int at, int kb,
                                        int extent) {
  if constexpr (MN) {
    for (int j = 0; j < extent / 64; ++j) tma_load_2d(dst + j * kBoxBytes, m, bar, at + 64 * j, kb * kKb);
  } else {
    tma_load_2d(dst, m, bar, kb * kKb, at);
  }
}

__device__ __forceinline__ float4 ld_dsmem_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

__device__ __forceinline__ uint32_t cluster_nctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}

// DEEP: several partial sums per CTA (where one will do, the code that adds them costs 2 to 3 %
// all the same: dx 256 x 1024 x 1024 5.24 against 5.08 us)
template <int OP, int TYPE, int BN, bool F32, bool DEEP>
__global__ void __launch_bounds__(kSplitThreads, SplitCfg<OP, BN, DEEP>::PER_SM)
    linear_split_kernel(const __grid_constant__ CUtensorMap tmC, const __grid_constant__ CUtensorMap tmR,
                        const __grid_constant__ EpiArgs p) {
  using C = SplitCfg<OP, BN, DEEP>;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  SplitBars* bars = reinterpret_cast<SplitBars*>(smem + C::BAR_OFF);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_ctarank(), S = (int)cluster_nctarank();
  const int tiles_c = (p.cols + 127) / 128;
  const int tile = blockIdx.x / S;
  const int c0 = tile % tiles_c * 128, r0 = tile / tiles_c * BN;
  const int num_kb = (p.depth + kKb - 1) / kKb;
  // this CTA's run of the contraction; not empty, S <= num_kb (<= 2^24: 32 bits hold the products)
  const int kb0 = num_kb * rank / S, kb1 = num_kb * (rank + 1) / S;
  // blocks per partial sum; no more of them than SEGS, the caller sees to it
  constexpr int seg = segment_blocks(F32 ? (int)kTypeF32 : TYPE);
  AbortCtl ctl{p.dev_err, &bars->abort_flag};

  auto load_stage = [&](uint32_t stage, int kb) {
    unsigned char* dst = smem + stage * C::STAGE_BYTES;
    mbar_arrive_expect_tx(&bars->full[stage], C::STAGE_BYTES);
    load_op<C::C_MN>(dst, &tmC, &bars->full[stage], c0, kb, 128);
    load_op<C::R_MN>(dst + C::C_BYTES, &tmR, &bars->full[stage], r0, kb, BN);
  };
  const int first = min(C::STAGES, kb1 - kb0);   // stages that the ring takes at once
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&bars->full[s], 1);
      mbar_init(&bars->empty[s], 1);
    }
    mbar_init(&bars->acc, 1);
    bars->abort_flag = 0;
    fence_mbar_init();
    fence_proxy_async_smem();
    // the first loads leave before the CTA has its TMEM
    griddep_wait();
    for (int s = 0; s < first; ++s) load_stage((uint32_t)s, kb0 + s);
  }
  if (warp == 1) {
    tmem_alloc(&bars->tmem_base, C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  griddep_wait();
  const uint32_t tmem_base = bars->tmem_base;
  bool aborted_any = false;
  const int nrows = min(BN, p.rows - r0);
  float* part = reinterpret_cast<float*>(smem);   // [row][128 columns], over the drained ring

  if (warp == 0 && lane == 0) {
    uint32_t stage = 0, phase = 0;   // the ring's second round
    for (int kb = kb0 + first; kb < kb1; ++kb) {
      if (!mbar_wait(&bars->empty[stage], phase, ctl, 0x100 + stage)) { aborted_any = true; break; }
      load_stage(stage, kb);
      if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
    }
  } else if (warp == 1 && lane == 0) {
    uint32_t stage = 0, phase = 0;
    const uint32_t smem_base = smem_u32(smem);
    constexpr uint32_t fmt = TYPE == kTypeBF16 ? 1u : 0u;
    const uint32_t idesc = C::IDESC | (fmt << 7) | (fmt << 10);
    uint32_t d = tmem_base;
    for (int kb = kb0, at = 0; kb < kb1; ++kb, ++at) {
      if (DEEP && at == seg) {   // a fresh accumulator
        at = 0;
        d += BN;
      }
      if (!mbar_wait(&bars->full[stage], phase, ctl, 0x300 + stage)) { aborted_any = true; break; }
      tc_fence_after();
      const uint32_t a = smem_base + stage * C::STAGE_BYTES, b = a + C::C_BYTES;
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
        tc_mma<kKindF16>(d, op_desc(a, C::C_MN, kk), op_desc(b, C::R_MN, kk), idesc,
                         (at != 0 || kk != 0) ? 1u : 0u);
      tc_commit(&bars->empty[stage]);
      if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
    }
    if (!aborted_any) tc_commit(&bars->acc);
  } else if (warp >= 4) {
    // every load has landed and every MMA has read it: the ring is free
    const int q = warp & 3;
    const bool ok = __all_sync(0xffffffffu, mbar_wait(&bars->acc, 0, ctl, 0x400));
    aborted_any = !ok;
    if (ok) {
      tc_fence_after();
      const uint32_t acc = tmem_base + ((uint32_t)(q * 32) << 16);
      constexpr int CH = BN < 32 ? 16 : 32;
#pragma unroll 1
      for (int n0 = 0; n0 < nrows; n0 += CH) {
        uint32_t r[CH];
        if constexpr (CH == 16) tmem_ld_32x32b_x16(acc + (uint32_t)n0, r);
        else tmem_ld_32x32b_x32(acc + (uint32_t)n0, r);
        tmem_ld_wait();
        if constexpr (DEEP) {   // the other partial sums, added with rounding
#pragma unroll 1
          for (int g = 1; g * seg < kb1 - kb0; ++g) {
            uint32_t x[CH];
            if constexpr (CH == 16) tmem_ld_32x32b_x16(acc + (uint32_t)(g * BN + n0), x);
            else tmem_ld_32x32b_x32(acc + (uint32_t)(g * BN + n0), x);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < CH; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) + __uint_as_float(x[i]));
          }
        }
#pragma unroll
        for (int i = 0; i < CH; ++i)
          if (n0 + i < nrows) part[(n0 + i) * 128 + q * 32 + lane] = __uint_as_float(r[i]);
      }
      tc_fence_before();
    }
  }
  if (aborted_any || aborted(ctl)) {
    const unsigned long long t0 = global_ns();   // TMA copies still in flight land
    while (global_ns() - t0 < 100000ull) {}
  }
  __syncwarp();
  // The next kernel may be set up once every CTA's partial sums are in shared memory; the first
  // thread of a CTA counts for all, so warps without a part in the sums don't ask.  Asked for
  // right after the set-up, calls take the same time to 1 %; not at all, 1 us more.
  if (warp >= 4) griddep_launch();
  if (S > 1) cluster_sync();
  else __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, C::TMEM_COLS);
  }

  // The tile's rows go round the cluster.  A thread finishes four columns: the 32 lanes
  // then read 512 contiguous bytes of each partial sum, which is what the SM-to-SM
  // network carries best (eight columns per thread, half of the lanes' 16-byte units at
  // a time, took twice as long).
  const uint64_t off = drop_offset(p.drop);
  const int c = c0 + 4 * lane;
  if (c < p.cols) {
    for (int n = rank + S * warp; n < nrows; n += S * (kSplitThreads / 32)) {
      const int row = r0 + n;
      const uint32_t at = smem_u32(part) + (uint32_t)(n * 128 + 4 * lane) * 4u;
      // every partial sum's load is in flight before the first is added
      float4 x[kMaxSplit];
#pragma unroll
      for (int s = 0; s < kMaxSplit; ++s)
        if (s < S) x[s] = ld_dsmem_f4(mapa_addr(at, (uint32_t)s));
      float v[4] = {};
#pragma unroll
      for (int s = 0; s < kMaxSplit; ++s)
        if (s < S) {
          v[0] += x[s].x;
          v[1] += x[s].y;
          v[2] += x[s].z;
          v[3] += x[s].w;
        }
      if constexpr (OP == kOpLinear) {
        float b[4];
        if (p.bias) {
          loadn<TYPE, 4>(b, p.bias, (size_t)c, c, p.cols, p.bias_vec);
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] += b[j];
        }
        if (p.pre) store4<TYPE>(v, p.pre, (size_t)row * p.ldz + c, c, p.cols, p.pre_vec);
        act_fwd_n(v, p.act);
        if (p.drop.on) drop4(v, p.drop, off, row, c);
      }
      const size_t oa = (size_t)row * p.ldo + c, ra = (size_t)row * p.ldr + c;
      if constexpr (F32) {
        float* out = static_cast<float*>(p.out) + oa;
        const float* res = static_cast<const float*>(p.res) + ra;
        if (p.res) {
          float r[4] = {};
          if (p.res_vec && c + 4 <= p.cols) {
            const float4 q = *reinterpret_cast<const float4*>(res);
            r[0] = q.x, r[1] = q.y, r[2] = q.z, r[3] = q.w;
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (c + j < p.cols) r[j] = res[j];
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] += r[j];
        }
        if (p.out_vec && c + 4 <= p.cols) {
          *reinterpret_cast<float4*>(out) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (c + j < p.cols) out[j] = v[j];
        }
      } else {
        if (p.res) {
          float r[4];
          loadn<TYPE, 4>(r, p.res, ra, c, p.cols, p.res_vec);
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] += r[j];
        }
        store4<TYPE>(v, p.out, oa, c, p.cols, p.out_vec);
      }
    }
  }
  // no CTA leaves while another reads its partial sums; nothing is handed over, so the
  // barrier need not wait for the stores above
  __syncwarp();
  if (S > 1) cluster_sync_relaxed();
}

template <int OP, int TYPE, int BN, bool F32, bool DEEP>
cudaError_t launch_kernel(const LinearArgs& a, const Operand& x, const Operand& y, int S) {
  using C = SplitCfg<OP, BN, DEEP>;
  const EpiArgs p = epilogue(a);
  CUtensorMap tmC, tmR;
  if (!map_rows(&tmC, y.p, y.ld, y.rows, y.cols, 2, C::C_MN ? kKb : 128) ||
      !map_rows(&tmR, x.p, x.ld, x.rows, x.cols, 2, C::R_MN ? kKb : BN))
    return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = S;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.blockDim = dim3(kSplitThreads);
  cfg.gridDim = dim3((unsigned)((a.cols + 127) / 128) * ((a.rows + BN - 1) / BN) * S);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = a.stream;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  static Once once;
  auto k = linear_split_kernel<OP, TYPE, BN, F32, DEEP>;
  cudaError_t e = prepare(once, k, C::SMEM, cfg, nullptr);
  if (e != cudaSuccess) return e;
  return cudaLaunchKernelEx(&cfg, k, tmC, tmR, p);
}

template <int OP, int TYPE, int BN, bool F32 = false>
cudaError_t launch_one(const LinearArgs& a, const Operand& x, const Operand& y, int S) {
  if constexpr (!F32)
    if (((a.depth + kKb - 1) / kKb + S - 1) / S <= segment_blocks(TYPE))
      return launch_kernel<OP, TYPE, BN, F32, false>(a, x, y, S);
  return launch_kernel<OP, TYPE, BN, F32, true>(a, x, y, S);
}

template <int OP, int TYPE>
cudaError_t launch_bn(const LinearArgs& a, const Operand& x, const Operand& y, int bn, int S) {
  if constexpr (OP != kOpDw) {
    if (bn == 16) return launch_one<OP, TYPE, 16>(a, x, y, S);
    if (bn == 32) return launch_one<OP, TYPE, 32>(a, x, y, S);
  }
  if constexpr (OP == kOpDw) {
    if (a.out_type == kTypeF32) {
      if (bn == 64) return launch_one<OP, TYPE, 64, true>(a, x, y, S);
      if (bn == 128) return launch_one<OP, TYPE, 128, true>(a, x, y, S);
      return launch_one<OP, TYPE, 256, true>(a, x, y, S);
    }
  }
  if (bn == 64) return launch_one<OP, TYPE, 64>(a, x, y, S);
  if (bn == 128) return launch_one<OP, TYPE, 128>(a, x, y, S);
  return launch_one<OP, TYPE, 256>(a, x, y, S);
}

template <int TYPE>
cudaError_t launch_typed(const LinearArgs& a, const Operand& x, const Operand& y, int bn, int S) {
  if (a.op == kOpLinear) return launch_bn<kOpLinear, TYPE>(a, x, y, bn, S);
  if (a.op == kOpDx) return launch_bn<kOpDx, TYPE>(a, x, y, bn, S);
  return launch_bn<kOpDw, TYPE>(a, x, y, bn, S);
}

}  // namespace

cudaError_t launch_split(const LinearArgs& a, const Operand& rows_op, const Operand& cols_op, int bn, int split) {
  return a.type == kTypeF16 ? launch_typed<kTypeF16>(a, rows_op, cols_op, bn, split)
                            : launch_typed<kTypeBF16>(a, rows_op, cols_op, bn, split);
}

}  // namespace mlpg
