// linear_pair.cu -- the layer's products for many tiles: persistent CTA pairs.
#include "linear.cuh"

namespace mlpg {

namespace {

// ---- CTA pairs ------------------------------------------------------------------------
// 256 x 256 tiles: each CTA holds 128 rows of the accumulator, loads its own rows of the
// row operand and half of the columns of the column operand; the leader issues
// tcgen05.mma.cta_group::2 over both CTAs' shared memory.
//   warp 0      TMA producer, both CTAs
//   warp 1      TMEM allocation; MMA issuer in the leader
//   warps 4-19  epilogue: TMEM lane quadrant w % 4, 64 columns each
// Sixteen epilogue warps, because an epilogue with an activation and dropout issues some
// 35 instructions per element (2048 x 512 x 11008 with gelu, dropout and residual: 50 us,
// with eight warps 55), and because 64 columns per thread leave room for f32 sums.
//
// Partial sums (segment_blocks) leave TMEM while the next one is computed in the other
// accumulator, and are added in registers.  With f32 results (dW alone) the tile is
// finished from there; with 16-bit results the sum goes back over the last accumulator,
// because an epilogue with an activation needs the registers.
//
// Bound by the tensor cores, and over a run of such calls by the board's power: linear
// 2048 x 4096 x 11008 bf16 147 us, 1250 TFLOP/s (76 % of the measured burst, 90 % of the
// sustained rate), with gelu_tanh, bias and Z 151 us; dw 2048 x 4096 x 11008 147 us, in f32
// 167 us.
constexpr int kPairThreads = 640;
constexpr int kEpiWarps = 16;
constexpr int kEpiBuf = 4096;      // a warp's staging: 32 rows x 128 bytes
constexpr int kGroupRows = 8;      // row tiles per group of the tile order

template <int OP>
struct PairCfg {
  static constexpr bool A_MN = OP == kOpDw, B_MN = OP != kOpDx;
  static constexpr int BN = 256, BH = BN / 2;
  static constexpr int STAGES = 5;
  static constexpr int A_BYTES = 128 * 128, B_BYTES = BH * 128;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int EPI_OFF = STAGES * STAGE_BYTES;
  static constexpr int BAR_OFF = EPI_OFF + kEpiWarps * kEpiBuf;
  static constexpr int SMEM = BAR_OFF + 512 + 1024;
  static constexpr uint32_t TMEM_COLS = 2 * BN;
  static constexpr uint32_t IDESC = (1u << 4) | ((A_MN ? 1u : 0u) << 15) | ((B_MN ? 1u : 0u) << 16) |
                                    ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(256 >> 4) << 24);
  static_assert(SMEM <= kSmemMax, "shared memory budget");
};

struct PairBars {
  uint64_t full[8], empty[8];
  uint64_t acc_full[2], acc_empty[2];
  uint64_t res[kEpiWarps];      // a warp's residual tile has landed
  uint32_t tmem_base;
  int abort_flag;
};
static_assert(sizeof(PairBars) <= 512, "barrier block");

struct PairArgs {
  EpiArgs e;
  int tiles_r, tiles_c, num_kb;
  bool out_tma, res_tma, pre_tma;
};

// Tiles in groups of kGroupRows row tiles, rows fastest: the tiles in flight at one
// time then share both operands' blocks in L2 however many rows there are.
__device__ __forceinline__ void tile_at(int t, const PairArgs& p, int& tr, int& tc) {
  const int per = kGroupRows * p.tiles_c;
  const int g = t / per, r0 = g * kGroupRows;
  const int h = min(kGroupRows, p.tiles_r - r0);
  const int i = t - g * per;
  tr = r0 + i % h;
  tc = i / h;
}

// One operand's slice of a stage: `extent` rows (or columns) from `at`, contraction
// block kb.  Box origins are multiples of 64 elements, 128 bytes.
template <bool MN>
__device__ __forceinline__ void load_op_pair(unsigned char* dst, const CUtensorMap* m, uint32_t bar, int at, int kb,
                                             int extent) {
  if constexpr (MN) {
    for (int j = 0; j < extent / 64; ++j) tma_load_2d_pair(dst + j * kBoxBytes, m, bar, at + 64 * j, kb * kKb);
  } else {
    tma_load_2d_pair(dst, m, bar, kb * kKb, at);
  }
}

// A 32-row tile of 128-byte rows between global memory and a warp's staging buffer
// without TMA (rows of any alignment), es bytes per element; lanes take neighbouring
// columns.  16-byte unit u of row r sits at r * 128 + ((u ^ (r & 7)) << 4).
template <bool STORE>
__device__ __forceinline__ void copy_tile(unsigned char* st, void* g, long ld, int es, int row0, int c0, int rows,
                                          int cols) {
  const int lane = threadIdx.x & 31, n = 128 / es;
  const int nr = min(32, rows - row0);
  for (int r = 0; r < nr; ++r)
    for (int i = lane; i < n; i += 32) {
      if (c0 + i >= cols) break;
      const int b = i * es;
      unsigned char* s = st + r * 128 + (((b >> 4) ^ (r & 7)) << 4) + (b & 15);
      const size_t at = (size_t)(row0 + r) * ld + c0 + i;
      if (es == 2) {
        if constexpr (STORE) static_cast<uint16_t*>(g)[at] = *reinterpret_cast<uint16_t*>(s);
        else *reinterpret_cast<uint16_t*>(s) = static_cast<const uint16_t*>(g)[at];
      } else {
        if constexpr (STORE) static_cast<uint32_t*>(g)[at] = *reinterpret_cast<uint32_t*>(s);
        else *reinterpret_cast<uint32_t*>(s) = static_cast<const uint32_t*>(g)[at];
      }
    }
}

// A warp's staging buffer: tiles go out by TMA store (or plain stores), the residual
// comes in by TMA load (or plain loads) into the buffer that its result replaces.
struct Staging {
  unsigned char* buf;
  uint64_t* bar;
  uint32_t phase;          // parity of the bar's next completion
};

__device__ __forceinline__ uint4* unit(unsigned char* st, int row, int u) {
  return reinterpret_cast<uint4*>(st + row * 128 + ((u ^ (row & 7)) << 4));
}

// The stores before it have read the buffer.
__device__ __forceinline__ void staging_free() {
  if ((threadIdx.x & 31) == 0) bulk_wait_read_all();
  __syncwarp();
}

template <bool F32>
__device__ __forceinline__ void res_fetch(Staging& s, const PairArgs& p, const CUtensorMap* m, int row0, int c0) {
  if (p.res_tma) {
    if ((threadIdx.x & 31) == 0) {
      mbar_arrive_expect_tx(s.bar, kEpiBuf);
      tma_load_2d(s.buf, m, s.bar, c0, row0);
    }
  } else {
    copy_tile<false>(s.buf, const_cast<void*>(p.e.res), p.e.ldr, F32 ? 4 : 2, row0, c0, p.e.rows, p.e.cols);
  }
}

__device__ __forceinline__ bool res_wait(Staging& s, const PairArgs& p, const AbortCtl& ctl) {
  bool ok = true;
  if (p.res_tma) {
    ok = mbar_wait(s.bar, s.phase, ctl, 0x500);
    s.phase ^= 1u;
  }
  ok = __all_sync(0xffffffffu, ok);
  __syncwarp();
  return ok;
}

// A TMA store clips at the map's last column in units of 16 bytes (measured: it fills the
// unit with zeros), so a tile that holds a part of a unit goes out by plain stores.
__device__ __forceinline__ void tile_out(unsigned char* st, bool tma, const CUtensorMap* m, void* g, long ld, int es,
                                         int row0, int c0, int rows, int cols) {
  if (tma && (c0 + 128 / es <= cols || ((unsigned)cols * es) % 16u == 0)) {
    fence_proxy_async_smem();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) {
      tma_store_2d(m, smem_u32(st), c0, row0);
      bulk_commit_group();
    }
  } else {
    __syncwarp();
    copy_tile<true>(st, g, ld, es, row0, c0, rows, cols);
    fence_proxy_async_smem();   // before a TMA load into the buffer
    __syncwarp();
  }
}

// DEEP: 16-bit results of more than one partial sum (what that needs in registers would cost
// the others 0.3 to 1.5 %)
template <int OP, int TYPE, bool F32, int ACT, bool DEEP>
__global__ void __launch_bounds__(kPairThreads, 1)
    linear_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                       const __grid_constant__ CUtensorMap tmOut, const __grid_constant__ CUtensorMap tmRes,
                       const __grid_constant__ CUtensorMap tmPre, const __grid_constant__ PairArgs p) {
  using C = PairCfg<OP>;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  PairBars* bars = reinterpret_cast<PairBars*>(smem + C::BAR_OFF);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
  const int num_tiles = p.tiles_r * p.tiles_c;
  constexpr int seg = segment_blocks(F32 ? (int)kTypeF32 : TYPE);
  AbortCtl ctl{p.e.dev_err, &bars->abort_flag};

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&bars->full[s], 1);
      mbar_init(&bars->empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bars->acc_full[b], 1);
      mbar_init(&bars->acc_empty[b], 2 * kEpiWarps);   // the epilogue warps of both CTAs
    }
    for (int w = 0; w < kEpiWarps; ++w) mbar_init(&bars->res[w], 1);
    bars->abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  if (warp == 1) {
    tmem_alloc_pair(&bars->tmem_base, C::TMEM_COLS);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  griddep_wait();
  const uint32_t tmem_base = bars->tmem_base;
  bool aborted_any = false;

  if (warp == 0 && lane == 0) {
    uint32_t stage = 0, phase = 0;
    bool ok = true;
    for (int t = pair; t < num_tiles && ok; t += npairs) {
      int tr, tc;
      tile_at(t, p, tr, tc);
      for (int kb = 0; kb < p.num_kb; ++kb) {
        if (!mbar_wait(&bars->empty[stage], phase ^ 1u, ctl, 0x100 + stage)) { ok = false; break; }
        const uint32_t lfull = mapa_shared(&bars->full[stage], 0);
        unsigned char* dst = smem + stage * C::STAGE_BYTES;
        // the leader expects both CTAs' bytes; the other CTA's loads complete on its barrier
        if (rank == 0) mbar_arrive_expect_tx(&bars->full[stage], 2 * C::STAGE_BYTES);
        load_op_pair<C::A_MN>(dst, &tmA, lfull, tr * 256 + (int)rank * 128, kb, 128);
        load_op_pair<C::B_MN>(dst + C::A_BYTES, &tmB, lfull, tc * C::BN + (int)rank * C::BH, kb, C::BH);
        if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
      }
    }
    aborted_any = !ok;
  } else if (warp == 1 && lane == 0 && rank == 0) {
    uint32_t stage = 0, phase = 0;
    int local = 0;
    bool ok = true;
    const uint32_t smem_base = smem_u32(smem);
    constexpr uint32_t fmt = TYPE == kTypeBF16 ? 1u : 0u;
    const uint32_t idesc = C::IDESC | (fmt << 7) | (fmt << 10);
    for (int t = pair; t < num_tiles && ok; t += npairs)
      for (int s0 = 0; s0 < p.num_kb && ok; s0 += seg, ++local) {
        const int buf = local & 1;
        if (!mbar_wait(&bars->acc_empty[buf], ((uint32_t)(local >> 1) & 1u) ^ 1u, ctl, 0x200 + buf)) { ok = false; break; }
        tc_fence_after();
        const uint32_t d = tmem_base + (uint32_t)(buf * C::BN);
        const int s1 = min(p.num_kb, s0 + seg);
        for (int kb = s0; kb < s1; ++kb) {
          if (!mbar_wait(&bars->full[stage], phase, ctl, 0x300 + stage)) { ok = false; break; }
          tc_fence_after();
          const uint32_t a = smem_base + stage * C::STAGE_BYTES, b = a + C::A_BYTES;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            tc_mma_pair<kKindF16>(d, op_desc(a, C::A_MN, kk), op_desc(b, C::B_MN, kk), idesc,
                                  (kb != s0 || kk != 0) ? 1u : 0u);
          tc_commit_pair(&bars->empty[stage], 0x3);
          if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
        }
        if (ok) tc_commit_pair(&bars->acc_full[buf], 0x3);
      }
    aborted_any = !ok;
  } else if (warp >= 4) {
    const int q = warp & 3, h = (warp - 4) >> 2;
    Staging st{smem + C::EPI_OFF + (warp - 4) * kEpiBuf, &bars->res[warp - 4], 0u};
    const uint64_t off = drop_offset(p.e.drop);
    int local = 0;
    bool ok = true;
    for (int t = pair; t < num_tiles && ok; t += npairs) {
      int tr, tc;
      tile_at(t, p, tr, tc);
      const int row0 = tr * 256 + (int)rank * 128 + q * 32, c0 = tc * C::BN + h * 64;
      const bool live = row0 < p.e.rows && c0 < p.e.cols;
      const bool pre = OP == kOpLinear && p.e.pre != nullptr;
      const uint32_t quad = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(h * 64);
      staging_free();
      // the residual comes while the product is still running (Z has the buffer first)
      if (live && p.e.res && !pre) res_fetch<F32>(st, p, &tmRes, row0, c0);
      auto release = [&](int buf) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster_relaxed(mapa_shared(&bars->acc_empty[buf], 0));
      };
      auto acquire = [&](int buf) {
        ok = __all_sync(0xffffffffu, mbar_wait(&bars->acc_full[buf], (uint32_t)(local >> 1) & 1u, ctl, 0x400 + buf));
        tc_fence_after();
        return ok;
      };
      // adds the partial sum that comes next and hands its accumulator back
      auto drain = [&](float (&sum)[64]) {
        const int buf = local & 1;
        if (!acquire(buf)) return false;
#pragma unroll
        for (int j = 0; j < 64; j += 16) {
          uint32_t ra[16];
          tmem_ld_32x32b_x16(quad + (uint32_t)(buf * C::BN + j), ra);
          tmem_ld_wait();
          if (j == 48) release(buf);
#pragma unroll
          for (int i = 0; i < 16; ++i) sum[j + i] += __uint_as_float(ra[i]);
        }
        ++local;
        return true;
      };
      if constexpr (F32) {
        float sum[64] = {};
        for (int s0 = 0; s0 < p.num_kb; s0 += seg)
          if (!drain(sum)) break;
        if (!ok) break;
        // two staged tiles of 32 columns
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const int cg = c0 + 32 * g;
          if (!live || cg >= p.e.cols) continue;
          if (g) {
            staging_free();
            if (p.e.res) res_fetch<F32>(st, p, &tmRes, row0, cg);
          }
          if (p.e.res && !(ok = res_wait(st, p, ctl))) break;
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            const float* v = sum + 32 * g + 4 * u;
            float4* at = reinterpret_cast<float4*>(unit(st.buf, lane, u));
            const float4 r = p.e.res ? *at : make_float4(0.f, 0.f, 0.f, 0.f);
            *at = make_float4(v[0] + r.x, v[1] + r.y, v[2] + r.z, v[3] + r.w);
          }
          tile_out(st.buf, p.out_tma, &tmOut, p.e.out, p.e.ldo, 4, row0, cg, p.e.rows, p.e.cols);
        }
      } else {
        if constexpr (DEEP) {
          float sum[64] = {};
          for (int s0 = 0; s0 + seg < p.num_kb; s0 += seg)
            if (!drain(sum)) break;
          if (!ok || !acquire(local & 1)) break;
          const uint32_t last = quad + (uint32_t)((local & 1) * C::BN);
#pragma unroll
          for (int j = 0; j < 64; j += 16) {
            uint32_t ra[16];
            tmem_ld_32x32b_x16(last + (uint32_t)j, ra);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) ra[i] = __float_as_uint(sum[j + i] + __uint_as_float(ra[i]));
            tmem_st_32x32b_x16(last + (uint32_t)j, ra);
          }
          tmem_st_wait();
        } else if (!acquire(local & 1)) {
          break;
        }
        const int buf = local & 1;
        ++local;
        const uint32_t acc = quad + (uint32_t)(buf * C::BN);
        if (!live) {
          release(buf);
          continue;
        }
        // Z and Y are two passes over the accumulator through the one staging buffer
#pragma unroll 1
        for (int pass = pre ? 0 : 1; pass < 2; ++pass) {
          if (pass && pre) {
            staging_free();
            if (p.e.res) res_fetch<F32>(st, p, &tmRes, row0, c0);
          }
          if (pass && p.e.res && !(ok = res_wait(st, p, ctl))) break;
          // sixteen columns per step, the next sixteen on their way; with the type and the
          // activation known, a few branches that no lane diverges on are all that is left
          // (with the type and the activation asked at run time a step of eight took
          // 450 cycles, most of them in branches)
          uint32_t ra[16];
          tmem_ld_32x32b_x16(acc, ra);
#pragma unroll 1
          for (int j = 0; j < 8; j += 2) {
            float v[2][8];
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i >> 3][i & 7] = __uint_as_float(ra[i]);
            if (j < 6) tmem_ld_32x32b_x16(acc + (uint32_t)(8 * (j + 2)), ra);
            else if (pass) release(buf);
            uint4 *at0 = unit(st.buf, lane, j), *at1 = unit(st.buf, lane, j + 1);
            if constexpr (OP == kOpLinear) {
              const int c = c0 + 8 * j;
              if (p.e.bias) {
                add_bias8<TYPE>(v[0], p.e, c);
                add_bias8<TYPE>(v[1], p.e, c + 8);
              }
              if (pass) {
                act_fwd_n<ACT, 8>(v[0]);
                act_fwd_n<ACT, 8>(v[1]);
                if (p.e.drop.on) {
                  drop8(v[0], p.e.drop, drop_bits(p.e.drop, off, row0 + lane, c >> 3));
                  drop8(v[1], p.e.drop, drop_bits(p.e.drop, off, row0 + lane, (c >> 3) + 1));
                }
              }
            }
            if (p.e.res && pass) {
              float r[2][8];
              unpack8<TYPE>(r[0], *at0);
              unpack8<TYPE>(r[1], *at1);
#pragma unroll
              for (int i = 0; i < 16; ++i) v[i >> 3][i & 7] += r[i >> 3][i & 7];
            }
            *at0 = pack8<TYPE>(v[0]);
            *at1 = pack8<TYPE>(v[1]);
          }
          if (pass) tile_out(st.buf, p.out_tma, &tmOut, p.e.out, p.e.ldo, 2, row0, c0, p.e.rows, p.e.cols);
          else tile_out(st.buf, p.pre_tma, &tmPre, p.e.pre, p.e.ldz, 2, row0, c0, p.e.rows, p.e.cols);
        }
      }
    }
    if (lane == 0) bulk_wait_all();
    __syncwarp();
    aborted_any = !ok;
  }

  if (aborted_any || aborted(ctl)) {
    const unsigned long long t0 = global_ns();   // TMA copies still in flight land
    while (global_ns() - t0 < 100000ull) {}
  }
  __syncwarp();
  // the next kernel may be set up once every CTA has stored its last tile (linear_split.cu)
  if (warp >= 4) griddep_launch();
  tc_fence_before();
  cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, C::TMEM_COLS);
  }
}

template <int OP, int TYPE, bool F32, int ACT, bool DEEP>
cudaError_t launch_kernel(const LinearArgs& a, const Operand& x, const Operand& y) {
  using C = PairCfg<OP>;
  PairArgs p = {};
  p.e = epilogue(a);
  p.tiles_r = (a.rows + 255) / 256;
  p.tiles_c = (a.cols + C::BN - 1) / C::BN;
  p.num_kb = (a.depth + kKb - 1) / kKb;
  constexpr int es = F32 ? 4 : 2;
  p.out_tma = tma_rows(a.out, a.ldo, a.rows, es);
  p.res_tma = a.res && tma_rows(a.res, a.ldr, a.rows, es);
  p.pre_tma = a.pre && tma_rows(a.pre, a.ldz, a.rows, 2);
  CUtensorMap tmA, tmB, tmO, tmR, tmZ;
  bool ok = map_rows(&tmA, x.p, x.ld, x.rows, x.cols, 2, C::A_MN ? kKb : 128) &&
            map_rows(&tmB, y.p, y.ld, y.rows, y.cols, 2, C::B_MN ? kKb : C::BH);
  tmO = tmR = tmZ = tmA;
  if (ok && p.out_tma) ok = map_rows(&tmO, a.out, a.ldo, a.rows, a.cols, es, 32);
  if (ok && p.res_tma) ok = map_rows(&tmR, a.res, a.ldr, a.rows, a.cols, es, 32);
  if (ok && p.pre_tma) ok = map_rows(&tmZ, a.pre, a.ldz, a.rows, a.cols, 2, 32);
  if (!ok) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.blockDim = dim3(kPairThreads);
  cfg.gridDim = dim3(a.num_sms / 2 * 2);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = a.stream;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  static Once once;
  int pairs = 0;
  auto k = linear_pair_kernel<OP, TYPE, F32, ACT, DEEP>;
  cudaError_t e = prepare(once, k, C::SMEM, cfg, &pairs);
  if (e != cudaSuccess) return e;
  if (pairs <= 0) return cudaErrorInvalidConfiguration;
  pairs = std::min(pairs, p.tiles_r * p.tiles_c);
  cfg.gridDim = dim3(2 * pairs);
  return cudaLaunchKernelEx(&cfg, k, tmA, tmB, tmO, tmR, tmZ, p);
}

template <int OP, int TYPE, bool F32, int ACT>
cudaError_t launch_one(const LinearArgs& a, const Operand& x, const Operand& y) {
  if constexpr (!F32)
    if (a.depth > segment_blocks(TYPE) * kKb) return launch_kernel<OP, TYPE, F32, ACT, true>(a, x, y);
  return launch_kernel<OP, TYPE, F32, ACT, false>(a, x, y);
}

template <int TYPE>
cudaError_t launch_typed(const LinearArgs& a, const Operand& x, const Operand& y) {
  if (a.op == kOpDx) return launch_one<kOpDx, TYPE, false, kActNone>(a, x, y);
  if (a.op == kOpDw)
    return a.out_type == kTypeF32 ? launch_one<kOpDw, TYPE, true, kActNone>(a, x, y)
                                  : launch_one<kOpDw, TYPE, false, kActNone>(a, x, y);
  switch (a.act) {
    case kActRelu: return launch_one<kOpLinear, TYPE, false, kActRelu>(a, x, y);
    case kActGelu: return launch_one<kOpLinear, TYPE, false, kActGelu>(a, x, y);
    case kActGeluTanh: return launch_one<kOpLinear, TYPE, false, kActGeluTanh>(a, x, y);
    case kActSilu: return launch_one<kOpLinear, TYPE, false, kActSilu>(a, x, y);
    default: return launch_one<kOpLinear, TYPE, false, kActNone>(a, x, y);
  }
}

}  // namespace

cudaError_t launch_pair(const LinearArgs& a, const Operand& rows_op, const Operand& cols_op) {
  return a.type == kTypeF16 ? launch_typed<kTypeF16>(a, rows_op, cols_op)
                            : launch_typed<kTypeBF16>(a, rows_op, cols_op);
}

}  // namespace mlpg
