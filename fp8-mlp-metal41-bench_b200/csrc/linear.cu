// linear.cu -- the MLP layer's products on tcgen05: Y = R + drop(act(X W + b)) and the
// two gradient products dX = R + dZ W^T, dW = R + X^T dZ, f16 or bf16 operands, f32
// accumulators in TMEM, one rounding of each result.
//
// Two kernels share the operand layouts (an operand whose contraction index is
// contiguous is K-major, else MN-major; both come straight from the caller's rows by
// TMA with the 128-byte swizzle) and the epilogue's arithmetic (epi8):
//
//   linear_pair_kernel   persistent, 256 x 256 tiles on CTA pairs, for many tiles
//   linear_split_kernel  128 columns x BN rows per CTA, the contraction split over a
//                        cluster: few rows, where the weights' bytes bound the call
//
// Every mbarrier wait is bounded (ptx.cuh); on expiry the kernel records an error
// word, lets its TMA copies land, frees TMEM and returns.  No load uses multicast.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstring>
#include <mutex>

#include "layer.cuh"
#include "ptx.cuh"
#include "tmap.h"

namespace mlpg {

namespace {

constexpr int kKb = 64;            // contraction elements per stage: one 128-byte swizzle row
constexpr int kBoxBytes = 64 * 128;   // one MN-major box: 64 contraction rows x 64 elements
constexpr int kSmemMax = 232448;
constexpr int kEpiBuf = 4096;      // staging of 32 rows x 128 bytes

struct EpiArgs {
  const void *bias, *res;
  void *out, *pre;
  long ldo, ldr, ldz;
  int type, out_type, act;
  int rows, cols, depth;
  DropArgs drop;
  bool bias_vec, out_vec, res_vec, pre_vec;   // 16-byte aligned base and rows
  int* dev_err;
};

// ---- the epilogue's arithmetic on eight neighbouring columns ------------------------

// v += bias[c .. c+7]; columns at or past `cols` keep their value
__device__ __forceinline__ void add_bias8(float (&v)[8], const EpiArgs& p, int c) {
  if (p.bias_vec && c + 8 <= p.cols) {
    const uint4 w = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.bias) + c));
    const uint32_t q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack2(q[i], p.type);
      v[2 * i] += f.x;
      v[2 * i + 1] += f.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < p.cols) v[i] += load1(p.bias, c + i, p.type);
  }
}

__device__ __forceinline__ uint4 pack8(const float (&v)[8], int type) {
  return make_uint4(pack2(v[0], v[1], type), pack2(v[2], v[3], type), pack2(v[4], v[5], type),
                    pack2(v[6], v[7], type));
}

__device__ __forceinline__ void add8(float (&v)[8], uint4 w, int type) {
  const uint32_t q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack2(q[i], type);
    v[2 * i] += f.x;
    v[2 * i + 1] += f.y;
  }
}

// v = drop(act(v)) of row `row`, columns c .. c+7 (c a multiple of 8)
__device__ __forceinline__ void act_drop8(float (&v)[8], const EpiArgs& p, uint64_t off, int row, int c) {
  if (p.act != kActNone) act_fwd8(v, p.act);
  if (p.drop.thr) drop8(v, p.drop, off, row, c >> 3);
}

// ---- CTA pairs ------------------------------------------------------------------------
// 256 x BN tiles: each CTA holds 128 rows of the accumulator, loads its own rows of the
// row operand and half of the columns of the column operand; the leader issues
// tcgen05.mma.cta_group::2 over both CTAs' shared memory.
//   warp 0      TMA producer, both CTAs
//   warp 1      TMEM allocation; MMA issuer in the leader
//   warps 4-11  epilogue: TMEM lane quadrant w % 4, one half of the columns each
//
// F32 results (dW alone): the tensor cores cut low bits when they add to an
// accumulator, about 2^-25 of it per step of 16, which grows with the contraction
// (measured against 64 bits: 6e-7 after 512, 5e-6 after 4096).  So every 512 deep the
// partial sum leaves TMEM and is added in registers, rounded to nearest; the tile is
// 128 columns wide there to leave room for 64 sums per thread.  16-bit results, whose
// own rounding is 2^-12 or 2^-9, keep one accumulation.
constexpr int kPairThreads = 384;
constexpr int kGroupRows = 8;      // row tiles per group of the tile order

template <int OP, bool F32>
struct PairCfg {
  static constexpr bool A_MN = OP == kOpDw, B_MN = OP != kOpDx;
  static constexpr int BN = F32 ? 128 : 256, BH = BN / 2;
  static constexpr int STAGES = F32 ? 6 : 5;
  static constexpr int A_BYTES = 128 * 128, B_BYTES = BH * 128;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int SEG = 8;     // F32: stages per partial sum
  static constexpr int EPI_OFF = STAGES * STAGE_BYTES;
  static constexpr int BAR_OFF = EPI_OFF + 8 * 2 * kEpiBuf;
  static constexpr int SMEM = BAR_OFF + 512 + 1024;
  static constexpr uint32_t TMEM_COLS = 2 * BN;
  static constexpr uint32_t IDESC = (1u << 4) | ((A_MN ? 1u : 0u) << 15) | ((B_MN ? 1u : 0u) << 16) |
                                    ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(256 >> 4) << 24);
  static_assert(SMEM <= kSmemMax, "shared memory budget");
};

struct PairBars {
  uint64_t full[8], empty[8];
  uint64_t acc_full[2], acc_empty[2];
  uint64_t res[8][2];      // a warp's residual tile has landed
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

__device__ __forceinline__ uint64_t op_desc(uint32_t addr, bool mn, int kk) {
  // 16 deep: 32 bytes along a K-major row, 16 rows of 128 bytes of an MN-major box
  return mn ? sdesc_sw128(addr + kk * 2048, kBoxBytes, 1024) : sdesc_sw128(addr + kk * 32, 16, 1024);
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

// A warp's staging buffers: tiles go out by TMA store (or plain stores), the residual
// comes in by TMA load (or plain loads) into the buffer that its result replaces.
struct Staging {
  unsigned char* buf;      // two of kEpiBuf
  uint64_t* bar;           // two
  uint32_t phase;          // bit b: parity of bar[b]'s next completion
};

__device__ __forceinline__ uint4* unit(unsigned char* st, int row, int u) {
  return reinterpret_cast<uint4*>(st + row * 128 + ((u ^ (row & 7)) << 4));
}

__device__ __forceinline__ void res_fetch(Staging& s, int b, const PairArgs& p, const CUtensorMap* m, int row0, int c0) {
  if (p.res_tma) {
    if ((threadIdx.x & 31) == 0) {
      mbar_arrive_expect_tx(&s.bar[b], kEpiBuf);
      tma_load_2d(s.buf + b * kEpiBuf, m, &s.bar[b], c0, row0);
    }
  } else {
    copy_tile<false>(s.buf + b * kEpiBuf, const_cast<void*>(p.e.res), p.e.ldr, p.e.out_type == kTypeF32 ? 4 : 2, row0,
                     c0, p.e.rows, p.e.cols);
  }
}

__device__ __forceinline__ bool res_wait(Staging& s, int b, const PairArgs& p, const AbortCtl& ctl) {
  bool ok = true;
  if (p.res_tma) {
    ok = mbar_wait(&s.bar[b], (s.phase >> b) & 1u, ctl, 0x500 + b);
    s.phase ^= 1u << b;
  }
  ok = __all_sync(0xffffffffu, ok);
  __syncwarp();
  return ok;
}

__device__ __forceinline__ void tile_out(unsigned char* st, bool tma, const CUtensorMap* m, void* g, long ld, int es,
                                         int row0, int c0, int rows, int cols) {
  if (tma) {
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

template <int OP, bool F32>
__global__ void __launch_bounds__(kPairThreads, 1)
    linear_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                       const __grid_constant__ CUtensorMap tmOut, const __grid_constant__ CUtensorMap tmRes,
                       const __grid_constant__ CUtensorMap tmPre, const __grid_constant__ PairArgs p) {
  using C = PairCfg<OP, F32>;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  PairBars* bars = reinterpret_cast<PairBars*>(smem + C::BAR_OFF);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
  const int num_tiles = p.tiles_r * p.tiles_c;
  const int seg = F32 ? C::SEG : p.num_kb;
  AbortCtl ctl{p.e.dev_err, &bars->abort_flag};

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&bars->full[s], 1);
      mbar_init(&bars->empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bars->acc_full[b], 1);
      mbar_init(&bars->acc_empty[b], 2 * 8);   // the epilogue warps of both CTAs
    }
    for (int w = 0; w < 8; ++w)
      for (int b = 0; b < 2; ++b) mbar_init(&bars->res[w][b], 1);
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
    const uint32_t fmt = p.e.type == kTypeBF16 ? 1u : 0u;
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
    Staging st{smem + C::EPI_OFF + (warp - 4) * 2 * kEpiBuf, bars->res[warp - 4], 0u};
    const uint64_t off = drop_offset(p.e.drop);
    int local = 0;
    bool ok = true;
    constexpr int GC = F32 ? 32 : 64;            // columns per staged tile: 128 bytes
    constexpr int NG = C::BH / GC;               // two staged tiles per warp and tile
    static_assert(NG == 2, "two staging buffers");
    for (int t = pair; t < num_tiles && ok; t += npairs) {
      int tr, tc;
      tile_at(t, p, tr, tc);
      const int row0 = tr * 256 + (int)rank * 128 + q * 32, c0 = tc * C::BN + h * C::BH;
      const int row = row0 + lane;
      const bool live0 = row0 < p.e.rows && c0 < p.e.cols, live1 = row0 < p.e.rows && c0 + GC < p.e.cols;
      // with Z both buffers of a group are in use (0: Y, 1: Z), else groups alternate
      const bool two = p.e.pre != nullptr;
      const uint32_t quad = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(h * C::BH);
      // the previous tile's stores have read the buffers; the residual's tiles come
      // while the product is still running
      if (lane == 0) bulk_wait_read_all();
      __syncwarp();
      if (p.e.res && live0) {
        res_fetch(st, 0, p, &tmRes, row0, c0);
        if (!two && live1) res_fetch(st, 1, p, &tmRes, row0, c0 + GC);
      }
      auto release = [&](int buf) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(mapa_shared(&bars->acc_empty[buf], 0));
      };
      if constexpr (F32) {
        float sum[C::BH] = {};
        for (int s0 = 0; s0 < p.num_kb; s0 += seg, ++local) {
          const int buf = local & 1;
          ok = __all_sync(0xffffffffu, mbar_wait(&bars->acc_full[buf], (uint32_t)(local >> 1) & 1u, ctl, 0x400 + buf));
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int j = 0; j < C::BH; j += 32) {
            uint32_t ra[32];
            tmem_ld_32x32b_x32(quad + (uint32_t)(buf * C::BN + j), ra);
            tmem_ld_wait();
            if (j + 32 == C::BH) release(buf);
#pragma unroll
            for (int i = 0; i < 32; ++i) sum[j + i] += __uint_as_float(ra[i]);
          }
        }
        if (!ok) break;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          if (!(g ? live1 : live0)) continue;
          unsigned char* sb = st.buf + g * kEpiBuf;
          if (p.e.res && !(ok = res_wait(st, g, p, ctl))) break;
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            float4 v = make_float4(sum[32 * g + 4 * u], sum[32 * g + 4 * u + 1], sum[32 * g + 4 * u + 2],
                                   sum[32 * g + 4 * u + 3]);
            float4* at = reinterpret_cast<float4*>(unit(sb, lane, u));
            if (p.e.res) {
              const float4 r = *at;
              v = make_float4(v.x + r.x, v.y + r.y, v.z + r.z, v.w + r.w);
            }
            *at = v;
          }
          tile_out(sb, p.out_tma, &tmOut, p.e.out, p.e.ldo, 4, row0, c0 + g * GC, p.e.rows, p.e.cols);
        }
      } else {
        const int buf = local & 1;
        ok = __all_sync(0xffffffffu, mbar_wait(&bars->acc_full[buf], (uint32_t)(local >> 1) & 1u, ctl, 0x400 + buf));
        if (!ok) break;
        ++local;
        tc_fence_after();
        const uint32_t acc = quad + (uint32_t)(buf * C::BN);
        if (!live0) {
          release(buf);
          continue;
        }
#pragma unroll 1
        for (int g = 0; g < NG; ++g) {
          if (g && !live1) {
            release(buf);
            break;
          }
          const int cg = c0 + g * GC, b = two ? 0 : g;
          unsigned char* sb = st.buf + b * kEpiBuf;
          if (two && g) {
            if (lane == 0) bulk_wait_read_all();
            __syncwarp();
            if (p.e.res) res_fetch(st, 0, p, &tmRes, row0, cg);
          }
          if (p.e.res && !(ok = res_wait(st, b, p, ctl))) break;
          uint32_t ra[32];
#pragma unroll 1
          for (int hc = 0; hc < 2; ++hc) {
            tmem_ld_32x32b_x32(acc + (uint32_t)(g * GC + hc * 32), ra);
            tmem_ld_wait();
            if (g == NG - 1 && hc == 1) release(buf);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int c = cg + hc * 32 + 8 * j;
              float v[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(ra[8 * j + i]);
              if (p.e.bias) add_bias8(v, p.e, c);
              if (two) *unit(st.buf + kEpiBuf, lane, hc * 4 + j) = pack8(v, p.e.type);
              act_drop8(v, p.e, off, row, c);
              uint4* at = unit(sb, lane, hc * 4 + j);
              if (p.e.res) add8(v, *at, p.e.type);
              *at = pack8(v, p.e.type);
            }
          }
          tile_out(sb, p.out_tma, &tmOut, p.e.out, p.e.ldo, 2, row0, cg, p.e.rows, p.e.cols);
          if (two) tile_out(st.buf + kEpiBuf, p.pre_tma, &tmPre, p.e.pre, p.e.ldz, 2, row0, cg, p.e.rows, p.e.cols);
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
  tc_fence_before();
  cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, C::TMEM_COLS);
  }
}

// ---- few rows -----------------------------------------------------------------------------
// One CTA computes 128 columns x BN rows over its share of the contraction, with the
// columns as the MMA's 128 lanes (so a single row still fills the tensor core's M and
// the epilogue's threads).  The cluster's CTAs split the contraction, put their partial
// sums into their own shared memory, and each then sums and finishes its share of the
// tile over distributed shared memory, in rank order: no workspace, no atomics, the
// same result every time.
constexpr int kSplitThreads = 256;

template <int OP, int BN>
struct SplitCfg {
  static constexpr bool C_MN = OP != kOpDx, R_MN = OP == kOpDw;
  static constexpr int C_BYTES = 128 * 128, R_BYTES = BN * 128;
  static constexpr int STAGE_BYTES = C_BYTES + R_BYTES;
  // BN <= 64: two CTAs per SM, about 100 KB each in flight
  static constexpr int STAGES = BN <= 32 ? 5 : (BN == 64 ? 4 : (BN == 128 ? 6 : 4));
  static constexpr int PER_SM = BN <= 64 ? 2 : 1;
  static constexpr int BAR_OFF = STAGES * STAGE_BYTES;
  static constexpr int SMEM = BAR_OFF + 512 + 1024;
  static constexpr uint32_t TMEM_COLS = BN < 32 ? 32 : BN;
  static constexpr uint32_t IDESC = (1u << 4) | ((C_MN ? 1u : 0u) << 15) | ((R_MN ? 1u : 0u) << 16) |
                                    ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
  static_assert(BN * 512 <= BAR_OFF, "partial sums fit the ring");
  static_assert(SMEM * PER_SM <= kSmemMax, "shared memory budget");
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

// Eight columns of one row: a 16-byte access where the matrix allows it.
__device__ __forceinline__ void put8(void* base, long ld, bool vec, int row, int c, int cols, const float (&v)[8],
                                     int type) {
  const size_t at = (size_t)row * ld + c;
  if (vec && c + 8 <= cols) {
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + at) = pack8(v, type);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < cols) store1(base, at + i, v[i], type);
  }
}

template <int OP, int BN>
__global__ void __launch_bounds__(kSplitThreads, SplitCfg<OP, BN>::PER_SM)
    linear_split_kernel(const __grid_constant__ CUtensorMap tmC, const __grid_constant__ CUtensorMap tmR,
                        const __grid_constant__ EpiArgs p) {
  using C = SplitCfg<OP, BN>;
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
  const int kb0 = (int)((long)num_kb * rank / S), kb1 = (int)((long)num_kb * (rank + 1) / S);   // kb1 > kb0: S <= num_kb
  AbortCtl ctl{p.dev_err, &bars->abort_flag};

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&bars->full[s], 1);
      mbar_init(&bars->empty[s], 1);
    }
    mbar_init(&bars->acc, 1);
    bars->abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmC);
    tma_prefetch_desc(&tmR);
  }
  if (warp == 1) {
    tmem_alloc(&bars->tmem_base, C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = bars->tmem_base;
  bool aborted_any = false;
  const int nrows = min(BN, p.rows - r0);
  float* part = reinterpret_cast<float*>(smem);   // [row][128 columns], over the drained ring

  if (warp == 0 && lane == 0) {
    uint32_t stage = 0, phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!mbar_wait(&bars->empty[stage], phase ^ 1u, ctl, 0x100 + stage)) { aborted_any = true; break; }
      unsigned char* dst = smem + stage * C::STAGE_BYTES;
      mbar_arrive_expect_tx(&bars->full[stage], C::STAGE_BYTES);
      load_op<C::C_MN>(dst, &tmC, &bars->full[stage], c0, kb, 128);
      load_op<C::R_MN>(dst + C::C_BYTES, &tmR, &bars->full[stage], r0, kb, BN);
      if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
    }
  } else if (warp == 1 && lane == 0) {
    uint32_t stage = 0, phase = 0;
    const uint32_t smem_base = smem_u32(smem);
    const uint32_t fmt = p.type == kTypeBF16 ? 1u : 0u;
    const uint32_t idesc = C::IDESC | (fmt << 7) | (fmt << 10);
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!mbar_wait(&bars->full[stage], phase, ctl, 0x300 + stage)) { aborted_any = true; break; }
      tc_fence_after();
      const uint32_t a = smem_base + stage * C::STAGE_BYTES, b = a + C::C_BYTES;
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
        tc_mma<kKindF16>(tmem_base, op_desc(a, C::C_MN, kk), op_desc(b, C::R_MN, kk), idesc,
                         (kb != kb0 || kk != 0) ? 1u : 0u);
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
  cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, C::TMEM_COLS);
  }

  // this CTA's share of the tile's 8-column groups
  const uint64_t off = drop_offset(p.drop);
  const uint32_t mine = smem_u32(part);
  for (int i = rank * kSplitThreads + (int)threadIdx.x; i < nrows * 16; i += S * kSplitThreads) {
    const int n = i >> 4, row = r0 + n, c = c0 + 8 * (i & 15);
    if (c >= p.cols) continue;
    const uint32_t at = mine + (uint32_t)(n * 128 + 8 * (i & 15)) * 4u;
    float v[8] = {};
    for (int s = 0; s < S; ++s) {
      uint32_t a;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(at), "r"(s));
      const float4 x = ld_dsmem_f4(a), y = ld_dsmem_f4(a + 16u);
      v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
      v[4] += y.x; v[5] += y.y; v[6] += y.z; v[7] += y.w;
    }
    if (p.bias) add_bias8(v, p, c);
    if (p.pre) put8(p.pre, p.ldz, p.pre_vec, row, c, p.cols, v, p.type);
    act_drop8(v, p, off, row, c);
    if (p.res) {
      const size_t ra = (size_t)row * p.ldr + c;
      if (p.res_vec && c + 8 <= p.cols) {
        add8(v, *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.res) + ra), p.type);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (c + j < p.cols) v[j] += load1(p.res, ra + j, p.type);
      }
    }
    put8(p.out, p.ldo, p.out_vec, row, c, p.cols, v, p.type);
  }
  cluster_sync();   // no CTA leaves while another reads its partial sums
}

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

// ---- host ---------------------------------------------------------------------------------

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// The TMA reads rows whose base and distance are multiples of 16 bytes (a single row
// has no distance).
bool tma_rows(const void* p, long ld, int rows, int es) { return aligned16(p) && (rows == 1 || ld * es % 16 == 0); }

// A stored 16-bit operand [rows, cols].
struct Operand {
  const void* p;
  long ld;
  int rows, cols;
  size_t packed() const {
    return tma_rows(p, ld, rows, 2) ? 0 : ((size_t)rows * ((cols + 7) / 8) * 16 + 255) / 256 * 256;
  }
};

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
  pack_rows_kernel<<<(unsigned)grid, 256, 0, a.stream>>>(static_cast<const uint16_t*>(o.p), o.ld,
                                                         reinterpret_cast<uint16_t*>(ws), o.rows, o.cols, groups);
  o.p = ws;
  o.ld = 8L * groups;
  ws += bytes;
  return cudaGetLastError();
}

// 2-D map of [rows, cols] elements of es bytes in boxes of 128-byte rows, 128-byte swizzle
bool map_rows(CUtensorMap* m, const void* p, long ld, int rows, int cols, int es, int box_rows) {
  const uint64_t pitch = rows == 1 ? ((uint64_t)cols * es + 15) / 16 * 16 : (uint64_t)ld * es;
  return make_map(m, p, es == 2 ? CU_TENSOR_MAP_DATA_TYPE_UINT16 : CU_TENSOR_MAP_DATA_TYPE_UINT32, (uint64_t)cols,
                  (uint64_t)rows, pitch, 128 / es, (uint32_t)box_rows);
}

EpiArgs epilogue(const LinearArgs& a) {
  EpiArgs e = {};
  e.bias = a.bias;
  e.res = a.res;
  e.out = a.out;
  e.pre = a.pre;
  e.ldo = a.ldo;
  e.ldr = a.ldr;
  e.ldz = a.ldz;
  e.type = a.type;
  e.out_type = a.out_type;
  e.act = a.act;
  e.rows = a.rows;
  e.cols = a.cols;
  e.depth = a.depth;
  e.drop = a.drop;
  e.bias_vec = aligned16(a.bias);
  e.out_vec = aligned16(a.out) && a.ldo % 8 == 0;
  e.res_vec = aligned16(a.res) && a.ldr % 8 == 0;
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

template <int OP, bool F32>
cudaError_t launch_pair(const LinearArgs& a, const Operand& x, const Operand& y) {
  using C = PairCfg<OP, F32>;
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
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.blockDim = dim3(kPairThreads);
  cfg.gridDim = dim3(a.num_sms / 2 * 2);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = a.stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  static Once once;
  int pairs = 0;
  auto k = linear_pair_kernel<OP, F32>;
  cudaError_t e = prepare(once, k, C::SMEM, cfg, &pairs);
  if (e != cudaSuccess) return e;
  if (pairs <= 0) return cudaErrorInvalidConfiguration;
  pairs = std::min(pairs, p.tiles_r * p.tiles_c);
  cfg.gridDim = dim3(2 * pairs);
  return cudaLaunchKernelEx(&cfg, k, tmA, tmB, tmO, tmR, tmZ, p);
}

template <int OP, int BN>
cudaError_t launch_split_bn(const LinearArgs& a, const Operand& x, const Operand& y, int S) {
  using C = SplitCfg<OP, BN>;
  const EpiArgs p = epilogue(a);
  CUtensorMap tmC, tmR;
  if (!map_rows(&tmC, y.p, y.ld, y.rows, y.cols, 2, C::C_MN ? kKb : 128) ||
      !map_rows(&tmR, x.p, x.ld, x.rows, x.cols, 2, C::R_MN ? kKb : BN))
    return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = S;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.blockDim = dim3(kSplitThreads);
  cfg.gridDim = dim3((unsigned)((a.cols + 127) / 128) * ((a.rows + BN - 1) / BN) * S);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = a.stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  static Once once;
  auto k = linear_split_kernel<OP, BN>;
  cudaError_t e = prepare(once, k, C::SMEM, cfg, nullptr);
  if (e != cudaSuccess) return e;
  return cudaLaunchKernelEx(&cfg, k, tmC, tmR, p);
}

template <int OP>
cudaError_t launch_split(const LinearArgs& a, const Operand& x, const Operand& y, int bn, int S) {
  if constexpr (OP != kOpDw) {
    if (bn == 16) return launch_split_bn<OP, 16>(a, x, y, S);
    if (bn == 32) return launch_split_bn<OP, 32>(a, x, y, S);
  }
  if (bn == 64) return launch_split_bn<OP, 64>(a, x, y, S);
  if (bn == 128) return launch_split_bn<OP, 128>(a, x, y, S);
  return launch_split_bn<OP, 256>(a, x, y, S);
}

// Which kernel, and how it cuts the work.
struct Plan {
  int bn;      // 0: CTA pairs; else rows per CTA of the split kernel
  int split;   // cluster size
};

Plan plan(const LinearArgs& a) {
  if (a.out_type == kTypeF32) return {0, 1};
  const int num_kb = (a.depth + kKb - 1) / kKb;
  const long tiles_c = (a.cols + 127) / 128;
  const long pair_tiles = (long)((a.rows + 255) / 256) * ((a.cols + 255) / 256);
  if (a.rows > 256 && pair_tiles * 2 >= a.num_sms / 2) return {0, 1};
  int bn = a.op == kOpDw ? 64 : 16;
  while (bn < 256 && bn < a.rows) bn *= 2;
  const long tiles = tiles_c * ((a.rows + bn - 1) / bn);
  const long slots = (long)a.num_sms * (bn <= 64 ? 2 : 1);
  int S = 1;
  while (S < 8 && tiles * (S + 1) <= slots && num_kb >= 2 * (S + 1)) ++S;
  return {bn, S};
}

template <int OP>
cudaError_t launch_op(const LinearArgs& a, const Operand& x, const Operand& y) {
  const Plan pl = plan(a);
  if (pl.bn) return launch_split<OP>(a, x, y, pl.bn, pl.split);
  if constexpr (OP == kOpDw) {
    if (a.out_type == kTypeF32) return launch_pair<OP, true>(a, x, y);
  }
  return launch_pair<OP, false>(a, x, y);
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
  switch (a.op) {
    case kOpLinear: return launch_op<kOpLinear>(a, x, y);
    case kOpDx: return launch_op<kOpDx>(a, x, y);
    default: return launch_op<kOpDw>(a, x, y);
  }
}

}  // namespace mlpg
