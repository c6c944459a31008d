// Gated feed-forward block on the sm_100a tensor cores, without its projections in memory.
//
//   forward    act = silu(x Wg^T) * (x Wu^T),   y = residual + act Wd^T
//   backward   da = dy Wd,  s = 1 / (1 + e^-gate),  silu = gate s
//              dgate = da up (s + silu (1 - s)),  dup = da silu,  act again
//              dx = dgate Wg + dup Wu,  dWg = dgate^T x,  dWu = dup^T x,  dWd = dy^T act
//
// x [tokens][width], Wg over Wu in one [2 hidden][width] matrix, Wd [width][hidden], all bf16; in 8 bits x and Wg, Wu are
// e4m3 with one fp32 scale a row, which the epilogue applies (a product of rows scales as its rows do).
//
// gated_ffn_kernel<PAIR, BWD, E4M3> makes everything above the line dx: the gate and the up projection of a tile are two
// halves of one accumulator, so the epilogue holds both factors of the product in fp32 and rounds it once; the backward
// instance forms both again, and da beside them in a third accumulator, instead of reading what forward would have had to
// store (4 bytes per token and hidden channel, and twice that to read it: a layer of 8192 x 4864 keeps 240 MB less). What
// leaves is act and, in backward, dgate and dup, which the plain products of the block read.
// No sum is shared between CTAs and none depends on the order in which tiles finish: a call repeats bit for bit.
//
// act, dgate and dup are rounded to bf16 once: they are operands of tensor-core products. Everything before that is fp32, the
// sigmoid from __expf and __fdividef (off by 2 + 1.17 |gate| and by 2 units in the last place: 2^-18 of itself up to a gate of 20,
// far below bf16's 2^-9). Against 64 bits the rounding of act takes y of 1237 x 1544 x 8936 from 0.0017 of its 2-norm, which is
// y's own rounding, to 0.0019; the gradients of 8192 x 896 x 4864, with that of dgate and dup, to 0.0023.
//
// 8192 tokens x 896 x 4864, one launch each. Forward 92 us, 1550 TFLOP/s, tensor pipe 85 % busy, operands out of L2 at 12.1 TB/s,
// 49 % of its rate; the rest is the epilogue of a last, partly filled round. Backward 158 us, 1360 TFLOP/s, tensor pipe 73 %: its
// epilogue holds three accumulators and writes three outputs, and gate and up have one accumulator only, so the first products
// of a tile wait for the reader of the tile before. Both figures are of short runs; kept up for a second the
// clocks fall at the power limit and a call takes a fifth longer (a library product falls from 1641 to 1371 TFLOP/s).
// 24 tokens x 4096 x 11008 in 8 bits 18 us, 90 MB of weights at 5.0 TB/s: start, first fetch and drain of 14 us of reading.
#include <cuda.h>
#include <cuda_fp8.h>

#include "balanced_gemm.cuh"
#include "common.cuh"
#include "gated_ffn.cuh"
#include "ops.cuh"
#include "ptx.cuh"

namespace srt {

int* tc_status_device_ptr();  // igemm_tcgen05.cu
int tmap_rows(CUtensorMap* tm, const void* base, uint64_t rows, uint64_t cols, uint64_t pitch, int elem_bytes, uint32_t box_cols, uint32_t box_rows);

namespace {

using namespace ptx;
using bf16 = __nv_bfloat16;

constexpr int FM = 128;                  // rows of a CTA's tile (tensor-memory lanes)
constexpr int epi_groups(bool pair) { return pair ? 4 : 2; }                  // of four warps, behind the TMA and the MMA warp
constexpr int ffn_threads(bool pair) { return 64 + 128 * epi_groups(pair); }
constexpr int F_MAX_STAGES = 16;
constexpr int F_SLAB_BYTES = FM * 64;    // 128 x 32 bf16 on the way out, 64-byte swizzle
constexpr int F_NARROW_BYTES = FM * 32;  // 128 x 16 bf16, 32-byte swizzle: three a group of a single CTA, in backward
enum { W_FFN_LOAD = 0x31, W_FFN_FULL = 0x32, W_FFN_ACC = 0x33, W_FFN_EPI = 0x34, W_FFN_DRAIN = 0x35 };

struct FfnParams {
  int T, F, k_blocks;
  int m_units, n_tiles;        // tiles of 128 (256 for a pair) tokens, and of g hidden channels
  int g;                       // hidden channels of a tile; a pair has 128
  int cols;                    // tensor-memory columns: a power of two, at least 4 g
  int stages, stage_bytes;
  uint32_t a_bytes;            // of a stage: with fewer than 128 tokens only their rows; the products read on into what
                               // follows, and the rows of the accumulators that this fills are not stored
  uint32_t gu_bytes, da_bytes; // what one CTA loads a k-block in either phase
  int slab_bytes;              // shared memory that outputs pass through on their way to TMA; 0: straight from registers to
  bf16 *act, *dgu;             // these, rows so far apart
  int act_pitch, dgu_pitch;
  const float *x_scale, *w_scale;
  int* status;
};

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ float sigmoid_f(float v) { return __fdividef(1.f, 1.f + __expf(-v)); }

// Tiles in bands of eight row units, rows fastest: the CTAs at work at one time read about as many rows of x as of the
// weights, both out of L2.
__device__ __forceinline__ void tile_of(const FfnParams& p, int t, int& m, int& n) {
  constexpr int BAND = 8;
  const int band = t / (BAND * p.n_tiles), first = band * BAND;
  const int size = min(BAND, p.m_units - first), r = t - first * p.n_tiles;
  n = r / size;
  m = first + r - n * size;
}

// PAIR: cta_group::2, 256 tokens x 128 hidden channels; rank 0 stages the gate rows of the weights and rank 1 the up rows,
// both halves of the B operand of one 256 x 256 product. Otherwise one CTA has 128 tokens x g channels.
// Tensor memory, in quarters of `cols`: forward two accumulators of two quarters; backward da of even tiles | gate and up |
// da of odd tiles, so that the da product of the next tile runs beside the epilogue of the current one.
template <bool PAIR, bool BWD, bool E4M3>
__global__ void __launch_bounds__(ffn_threads(PAIR), PAIR ? 1 : 2)
gated_ffn_kernel(const FfnParams p, const __grid_constant__ CUtensorMap tx, const __grid_constant__ CUtensorMap tw,
                 const __grid_constant__ CUtensorMap tdy, const __grid_constant__ CUtensorMap twd,
                 const __grid_constant__ CUtensorMap tact, const __grid_constant__ CUtensorMap tgate,
                 const __grid_constant__ CUtensorMap tup) {
  constexpr int NCTA = PAIR ? 2 : 1;
  constexpr int BKE = E4M3 ? 128 : 64;  // reduction elements of a k-block
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const int NS = p.stages;
  uint8_t* sOut = base + NS * p.stage_bytes;
  uint64_t* bars = (uint64_t*)(sOut + p.slab_bytes + (PAIR ? 0 : FM * 128 - (int)p.a_bytes));
  const uint32_t full = smem_u32(bars), empty = full + 8 * F_MAX_STAGES, acc_full = empty + 8 * F_MAX_STAGES, acc_empty = acc_full + 16;
  uint32_t* tmem_ptr = (uint32_t*)(bars + 2 * F_MAX_STAGES + 4);
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const uint32_t rank = PAIR ? cluster_ctarank() : 0u;
  const int unit = (int)blockIdx.x / NCTA, nunits = (int)gridDim.x / NCTA;
  const int total = p.m_units * p.n_tiles, nkb = p.k_blocks, g = p.g;
  const int quarter = p.cols / 4;
  const uint32_t s0 = smem_u32(base);

  if (tid == 0) {
    for (int s = 0; s < NS; ++s) { mbar_init(full + 8 * s, 1); mbar_init(empty + 8 * s, 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(acc_full + 8 * b, 1); mbar_init(acc_empty + 8 * b, 4 * epi_groups(PAIR) * NCTA); }
    mbar_fence_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tx);
    tma_prefetch_desc(&tw);
    if (BWD) { tma_prefetch_desc(&tdy); tma_prefetch_desc(&twd); }
  }
  if (warp == 1) {
    if (PAIR) { tmem_alloc_pair(smem_u32(tmem_ptr), p.cols); tmem_relinquish_pair(); }
    else { tmem_alloc(smem_u32(tmem_ptr), p.cols); tmem_relinquish(); }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (PAIR) cluster_sync_all();  // the peer's barriers and tensor memory exist before anything refers to them
  tc_fence_after_sync();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_ptr, 0);
  pdl_enter();

  if (warp == 0) {
    // The warp walks together and one thread of it issues (see elect_one); what does not change from one k-block to the next
    // stays out of the loops.
    const uint32_t full_to = PAIR ? map_to_cta(full, 0u) : full;  // the leader's barriers
    const uint32_t wrap = (uint32_t)NS * p.stage_bytes, gu_bytes = p.gu_bytes * NCTA, da_bytes = p.da_bytes * NCTA;
    int it = 0;
    uint32_t at = 0, bar = 0, ph = 1;  // offsets of the current stage and of its barriers
    bool ok = true;
    auto load = [&](uint32_t offset, const CUtensorMap* tm, int x, int y) {
      if (PAIR) tma_load_2d_pair(s0 + at + offset, tm, full_to + bar, x, y);
      else tma_load_2d(s0 + at + offset, tm, full_to + bar, x, y);
    };
    auto step = [&]() {
      ++it;
      at += p.stage_bytes;
      bar += 8;
      if (at == wrap) { at = 0; bar = 0; ph ^= 1u; }
    };
    for (int t = unit; t < total && ok; t += nunits) {
      int m, n;
      tile_of(p, t, m, n);
      const int m0 = (m * NCTA + (int)rank) * FM, n0 = n * g;
      if (BWD) {
        const int f0 = n0 + (PAIR ? (int)rank * 64 : 0);
        for (int kb = 0; kb < nkb; ++kb) {
          ok = mbar_wait_warp<false>(empty + bar, ph, p.status, W_FFN_LOAD);
          if (!ok) break;
          if (elect_one()) {
            if (rank == 0) mbar_arrive_expect_tx(full + bar, da_bytes);
            load(0, &tdy, kb * 64, m0);
            load(p.a_bytes, &twd, f0, kb * 64);
            if (!PAIR && g > 64) load(p.a_bytes + 8192, &twd, f0 + 64, kb * 64);
          }
          step();
        }
      }
      const int w0 = n0 + (PAIR ? (int)rank * p.F : 0);
      for (int kb = 0; kb < nkb && ok; ++kb) {
        ok = mbar_wait_warp<false>(empty + bar, ph, p.status, W_FFN_LOAD);
        if (!ok) break;
        if (elect_one()) {
          if (rank == 0) mbar_arrive_expect_tx(full + bar, gu_bytes);
          load(0, &tx, kb * BKE, m0);
          load(p.a_bytes, &tw, kb * BKE, w0);
          if (!PAIR) load(p.a_bytes + (uint32_t)g * 128u, &tw, kb * BKE, p.F + n0);
        }
        step();
      }
    }
    // a wait that gave up: the copies in flight land before the CTA's memory is given back
    if (!ok && rank == 0)
      for (int k = it > NS ? it - NS : 0; k < it; ++k) mbar_wait_warp<false>(full + 8 * (k % NS), (uint32_t)(k / NS) & 1u, p.status, W_FFN_DRAIN);
  } else if (warp == 1) {
    if (rank == 0) {
      const uint32_t i_gu = E4M3 ? make_idesc_e4m3(FM * NCTA, PAIR ? 256 : 2 * g) : make_idesc_bf16(FM * NCTA, PAIR ? 256 : 2 * g, 0, 0);
      const uint32_t i_da = make_idesc_bf16(FM * NCTA, g, 0, 1);
      const uint64_t desc_a = make_smem_desc_sw128(s0, 0, 1024), desc_b = make_smem_desc_sw128(s0 + p.a_bytes, 0, 1024);
      const uint64_t desc_mn = make_smem_desc_sw128(s0 + p.a_bytes, 8192, 1024);
      const uint32_t wrap = (uint32_t)NS * p.stage_bytes;
      int i = 0;
      uint32_t at = 0, bar = 0, ph = 0;
      bool ok = true;
      // b_step: 16 elements along the reduction (32 in 8 bits), in a B tile that is stored along it or across it
      auto product = [&](uint32_t acc, uint32_t idesc, uint64_t db, uint32_t b_step) {
        uint32_t add = 0;
        for (int kb = 0; kb < nkb; ++kb) {
          ok = mbar_wait_warp<PAIR>(full + bar, ph, p.status, W_FFN_FULL);
          if (!ok) return;
          tc_fence_after_sync();
          if (elect_one()) {
            const uint64_t ad = desc_at(desc_a, at), bd = desc_at(db, at);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if (E4M3) {
                if (PAIR) umma_e4m3_pair(acc, desc_at(ad, k * 32), desc_at(bd, k * b_step), idesc, k ? 1u : add);
                else umma_e4m3(acc, desc_at(ad, k * 32), desc_at(bd, k * b_step), idesc, k ? 1u : add);
              } else {
                if (PAIR) umma_bf16_pair(acc, desc_at(ad, k * 32), desc_at(bd, k * b_step), idesc, k ? 1u : add);
                else umma_bf16(acc, desc_at(ad, k * 32), desc_at(bd, k * b_step), idesc, k ? 1u : add);
              }
            }
            if (PAIR) umma_commit_pair(empty + bar, (uint16_t)3);
            else umma_commit(empty + bar);
          }
          add = 1;
          at += p.stage_bytes;
          bar += 8;
          if (at == wrap) { at = 0; bar = 0; ph ^= 1u; }
        }
      };
      for (int t = unit; t < total && ok; t += nunits, ++i) {
        const uint32_t b = (uint32_t)i & 1u;
        // tile i - 2 has been read (parity starts so that the first two waits pass)
        ok = mbar_wait_warp<PAIR>(acc_empty + 8 * b, ((uint32_t)(i >> 1) & 1u) ^ 1u, p.status, W_FFN_ACC);
        if (!ok) break;
        tc_fence_after_sync();
        if (BWD) {
          product(tmem + (b ? 3u * quarter : 0u), i_da, desc_mn, 2048u);
          // gate and up have one accumulator: tile i - 1 has been read
          if (ok && i > 0) ok = mbar_wait_warp<PAIR>(acc_empty + 8 * (b ^ 1u), (uint32_t)((i - 1) >> 1) & 1u, p.status, W_FFN_ACC);
          if (!ok) break;
          tc_fence_after_sync();
          product(tmem + quarter, i_gu, desc_b, 32u);
        } else {
          product(tmem + b * 2u * quarter, i_gu, desc_b, 32u);
        }
        if (!ok) break;
        if (elect_one()) {
          if (PAIR) umma_commit_pair(acc_full + 8 * b, (uint16_t)3);
          else umma_commit(acc_full + 8 * b);
        }
      }
    }
  } else {
    const int grp = (warp - 2) >> 2, q = warp & 3, row = q * 32 + lane;
    const bool issuer = ((warp - 2) & 3) == 0 && lane == 0;
    const uint32_t lanes = (uint32_t)(q * 32) << 16;
    bool ok = true;
    int i = 0;
    for (int t = unit; t < total; t += nunits, ++i) {
      int m, n;
      tile_of(p, t, m, n);
      const int m0 = (m * NCTA + (int)rank) * FM, n0 = n * g;
      const uint32_t b = (uint32_t)i & 1u;
      const uint32_t t_gu = tmem + lanes + (BWD ? (uint32_t)quarter : b * 2u * quarter);
      const uint32_t t_da = tmem + lanes + (b ? 3u * quarter : 0u);
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(acc_full + 8 * b, (uint32_t)(i >> 1) & 1u, p.status, W_FFN_EPI));
      tc_fence_after_sync();
      const int mrow = m0 + row;
      const float xs = E4M3 && mrow < p.T ? p.x_scale[mrow] : 1.f;
      auto done = [&]() {
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          if (PAIR) mbar_arrive_cluster(map_to_cta(acc_empty + 8 * b, 0u));
          else mbar_arrive(acc_empty + 8 * b);
        }
      };
      if constexpr (PAIR) {
        const int c0 = grp * 32;
        const bool live = m0 < p.T && n0 + c0 < p.F;  // the same for the whole group
        uint32_t w[BWD ? 3 : 1][16];
        if (live) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t gv[16], uv[16], dv[BWD ? 16 : 1];
            tmem_ld_32x32b_x16(t_gu + (uint32_t)(c0 + h * 16), gv);
            tmem_ld_32x32b_x16(t_gu + 128u + (uint32_t)(c0 + h * 16), uv);
            if constexpr (BWD) tmem_ld_32x32b_x16(t_da + (uint32_t)(c0 + h * 16), dv);
            tmem_ld_wait();
            const int col = n0 + c0 + h * 16;
#pragma unroll
            for (int c = 0; c < 16; c += 2) {
              float a[2], dg[2], du[2];
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                float gt = __uint_as_float(gv[c + e]), up = __uint_as_float(uv[c + e]);
                if (E4M3) {
                  const int f = min(col + c + e, p.F - 1);
                  gt *= xs * p.w_scale[f];
                  up *= xs * p.w_scale[p.F + f];
                }
                const float sg = sigmoid_f(gt), silu = gt * sg;
                a[e] = silu * up;
                if constexpr (BWD) {
                  const float da = __uint_as_float(dv[c + e]);
                  dg[e] = da * up * (sg + silu * (1.f - sg));
                  du[e] = da * silu;
                }
              }
              w[0][h * 8 + c / 2] = pack_bf16(a[0], a[1]);
              if constexpr (BWD) {
                w[1][h * 8 + c / 2] = pack_bf16(dg[0], dg[1]);
                w[2][h * 8 + c / 2] = pack_bf16(du[0], du[1]);
              }
            }
          }
        }
        done();
        if (live) {
          const uint32_t slab = smem_u32(sOut) + (uint32_t)grp * F_SLAB_BYTES, mine = slab + (uint32_t)row * 64u;
#pragma unroll
          for (int o = 0; o < (BWD ? 3 : 1); ++o) {
            if (issuer) bulk_wait_group_read<0>();  // the store before has read the slab
            named_bar_sync(1 + grp, 128);
#pragma unroll
            for (int c = 0; c < 4; ++c)
              st_shared_v4(mine + (uint32_t)((c ^ ((row >> 1) & 3)) << 4), w[o][c * 4], w[o][c * 4 + 1], w[o][c * 4 + 2], w[o][c * 4 + 3]);
            fence_proxy_async_smem();
            named_bar_sync(1 + grp, 128);
            if (issuer) {
              tma_store_2d(o == 0 ? &tact : o == 1 ? &tgate : &tup, slab, n0 + c0, m0);
              bulk_commit_group();
            }
          }
        }
      } else {
        if (BWD && p.slab_bytes) {
          // sixteen channels at a time, dealt to the two groups in turn
          const uint32_t slab = smem_u32(sOut) + (uint32_t)grp * 3 * F_NARROW_BYTES, mine = slab + (uint32_t)row * 32u;
          const uint32_t flip = (uint32_t)(row >> 2) & 1u;
          if (m0 < p.T)
            for (int c = grp * 16; c < g && n0 + c < p.F; c += 32) {
              uint32_t gv[16], uv[16], dv[16], w[3][8];
              tmem_ld_32x32b_x16(t_gu + (uint32_t)c, gv);
              tmem_ld_32x32b_x16(t_gu + (uint32_t)(g + c), uv);
              tmem_ld_32x32b_x16(t_da + (uint32_t)c, dv);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 16; e += 2) {
                float a[2], dg[2], du[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                  const float gt = __uint_as_float(gv[e + k]), up = __uint_as_float(uv[e + k]), da = __uint_as_float(dv[e + k]);
                  const float sg = sigmoid_f(gt), silu = gt * sg;
                  a[k] = silu * up;
                  dg[k] = da * up * (sg + silu * (1.f - sg));
                  du[k] = da * silu;
                }
                w[0][e / 2] = pack_bf16(a[0], a[1]);
                w[1][e / 2] = pack_bf16(dg[0], dg[1]);
                w[2][e / 2] = pack_bf16(du[0], du[1]);
              }
              if (issuer) bulk_wait_group_read<0>();  // the stores before have read the slabs
              named_bar_sync(1 + grp, 128);
#pragma unroll
              for (int o = 0; o < 3; ++o)
#pragma unroll
                for (int v = 0; v < 2; ++v)
                  st_shared_v4(mine + (uint32_t)o * F_NARROW_BYTES + (((uint32_t)v ^ flip) << 4), w[o][4 * v], w[o][4 * v + 1], w[o][4 * v + 2], w[o][4 * v + 3]);
              fence_proxy_async_smem();
              named_bar_sync(1 + grp, 128);
              if (issuer) {
                tma_store_2d(&tact, slab, n0 + c, m0);
                tma_store_2d(&tgate, slab + F_NARROW_BYTES, n0 + c, m0);
                tma_store_2d(&tup, slab + 2 * F_NARROW_BYTES, n0 + c, m0);
                bulk_commit_group();
              }
            }
        } else {
          // eight channels at a time, dealt to the two groups in turn
          if (m0 < p.T)
            for (int c = grp * 8; c < g; c += 16) {
              uint32_t gv[8], uv[8], dv[8];
              tmem_ld_32x32b_x8(t_gu + (uint32_t)c, gv);
              tmem_ld_32x32b_x8(t_gu + (uint32_t)(g + c), uv);
              if constexpr (BWD) tmem_ld_32x32b_x8(t_da + (uint32_t)c, dv);
              tmem_ld_wait();
              const int f = n0 + c;
              if (mrow < p.T && f < p.F) {
                float a[8], dg[8], du[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                  float gt = __uint_as_float(gv[e]), up = __uint_as_float(uv[e]);
                  if (E4M3) {
                    gt *= xs * p.w_scale[f + e];
                    up *= xs * p.w_scale[p.F + f + e];
                  }
                  const float sg = sigmoid_f(gt), silu = gt * sg;
                  a[e] = silu * up;
                  if constexpr (BWD) {
                    const float da = __uint_as_float(dv[e]);
                    dg[e] = da * up * (sg + silu * (1.f - sg));
                    du[e] = da * silu;
                  }
                }
                Vec16<bf16> o;
                o.pack(a);
                o.store(p.act + (size_t)mrow * p.act_pitch + f);
                if constexpr (BWD) {
                  o.pack(dg);
                  o.store(p.dgu + (size_t)mrow * p.dgu_pitch + f);
                  o.pack(du);
                  o.store(p.dgu + (size_t)mrow * p.dgu_pitch + p.F + f);
                }
              }
            }
        }
        done();
      }
    }
    if ((PAIR || BWD) && issuer) bulk_wait_group_read<0>();  // the slab outlives the last store's read
  }

  tc_fence_before_sync();
  __syncthreads();
  if (PAIR) cluster_sync_all();  // neither CTA leaves while the other can signal its barriers or read its operands
  if (warp == 1) {
    __syncwarp();
    tc_fence_after_sync();
    if (PAIR) tmem_dealloc_pair(tmem, p.cols);
    else tmem_dealloc(tmem, p.cols);
  }
}

int tmap_rows_128b(CUtensorMap* tm, const void* base, uint64_t rows, uint64_t cols, uint64_t pitch, int elem_bytes, uint32_t box_rows) {
  return tmap_rows(tm, base, rows, cols, pitch, elem_bytes, 128u / (uint32_t)elem_bytes, box_rows);
}

constexpr size_t ffn_tail_bytes() { return (2 * F_MAX_STAGES + 4) * 8 + 16; }

// How a call is cut: the least time by the model of balanced_gemm.cu, in microseconds. A k-block of a product with n columns
// takes 0.155 at least, 1.53 ns a column, its bytes at 115 KB out of L2 (half as much again where rows do not begin on 128
// bytes), or at 40 KB out of memory where a single row of tiles reads the weights; an epilogue takes 0.35 and 18 ns a channel,
// in backward 30, beside the next tile's products. Measured, pair against the best single width: 8192 tokens 94 and 110 us,
// 600 x 2048 x 5632 25 and 21, 256 x 896 x 4864 10 and 8; backward, 8192: 168 and 238, 333: 26 and 21.
struct FfnPlan {
  bool pair;
  int g;
};
FfnPlan plan_ffn(int T, int C, int F, bool bwd, int esz) {
  const int sms = sm_count(), kb = ceil_div(C, 128 / esz);
  const int a_rows = T < FM ? (T + 7) / 8 * 8 : FM;
  const double odd_c = C * esz % 128 ? 1.5 : 1.0, odd_f = F % 64 ? 1.5 : 1.0;
  auto k_block = [&](double a, double b, int n, bool once) {
    double t = 0.155;
    auto at_least = [&](double v) { t = v > t ? v : t; };
    at_least(0.00153 * n);
    at_least((a + b) / 115e3);
    if (once) at_least(b / 40e3);
    return t;
  };
  FfnPlan best = {false, 16};
  double best_cost = 1e30;
  auto consider = [&](bool pair, int g) {
    const int m_units = ceil_div(T, pair ? 2 * FM : FM), nc = pair ? g : 2 * g;
    const long long tiles = (long long)m_units * ceil_div(F, g);
    const double a = 128.0 * a_rows * odd_c;
    double t = kb * k_block(a, 128.0 * nc * odd_c, 2 * g, m_units == 1);
    if (bwd) t += kb * k_block(a, 8192.0 * ceil_div(pair ? g / 2 : g, 64) * odd_f, g, m_units == 1);
    const double epi = 0.35 + (bwd ? 0.030 : 0.018) * g;
    const double cost = (double)ceil_div_ll(tiles, pair ? sms / 2 : sms) * (t > epi ? t : epi) + epi;
    if (cost < best_cost) { best_cost = cost; best = {pair, g}; }
  };
  for (int g = 16; g <= 128; g += bwd ? 16 : 8) consider(false, g);
  if (sms >= 2) consider(true, 128);
  return best;
}

template <bool PAIR, bool BWD, bool E4M3>
int launch_ffn(FfnParams& p, const CUtensorMap (&tm)[7], cudaStream_t st) {
  const size_t budget = PAIR || p.cols > 256 ? 232448 : 113 * 1024;  // two single CTAs share an SM where tensor memory allows
  // a single CTA with few tokens reads up to 16 KB beyond a stage's rows
  const size_t fixed = 1024 + (size_t)p.slab_bytes + (PAIR ? 0 : FM * 128 - (int)p.a_bytes) + ffn_tail_bytes();
  p.stages = (int)((budget - fixed) / p.stage_bytes);
  if (p.stages > F_MAX_STAGES) p.stages = F_MAX_STAGES;
  const size_t smem = fixed + (size_t)p.stages * p.stage_bytes;
  static SmemOptIn opt_in;
  SRT_CHECK_CUDA(opt_in.set(gated_ffn_kernel<PAIR, BWD, E4M3>, 232448));
  const int room = PAIR ? sm_count() / 2 : sm_count() * (p.cols > 256 ? 1 : 2);
  const long long total = (long long)p.m_units * p.n_tiles;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((total < room ? total : room) * (PAIR ? 2 : 1)));
  cfg.blockDim = dim3(ffn_threads(PAIR));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = (pdl_big_kernels() && (pdl_classes() & PDL_GEMM) != 0) ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (PAIR) {
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 2;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
  }
  SRT_CHECK_CUDA(cudaLaunchKernelEx(&cfg, gated_ffn_kernel<PAIR, BWD, E4M3>, p, tm[0], tm[1], tm[2], tm[3], tm[4], tm[5], tm[6]));
  SRT_LAUNCH_CHECK();
  return SRT_OK;
}

// The rows of act and dgu begin on 128 bytes, whatever `hidden` is: TMA takes half as much time again for rows that do not
// (1237 x 1544 x 8936, forward: 103.8 us with rows of `hidden`, 96.7 with these).
int act_pitch(const srt_gated_ffn_desc& d) { return (d.hidden + 63) / 64 * 64; }
int dgu_pitch(const srt_gated_ffn_desc& d) { return (2 * d.hidden + 63) / 64 * 64; }

// act, and with dy also dgu = (dgate, dup), from x and the weights.
int gated_products(const srt_gated_ffn_desc& d, const void* x, const float* x_scale, const void* w_gu, const float* w_scale,
                   const void* dy, const void* w_down, void* act, void* dgu, cudaStream_t st) {
  const bool bwd = dy != nullptr, e4m3 = x_scale != nullptr;
  const int T = d.tokens, C = d.width, F = d.hidden, esz = e4m3 ? 1 : 2;
  const FfnPlan plan = plan_ffn(T, C, F, bwd, esz);
  FfnParams p = {};
  p.T = T;
  p.F = F;
  p.g = plan.g;
  p.k_blocks = ceil_div(C, 128 / esz);
  p.m_units = ceil_div(T, plan.pair ? 2 * FM : FM);
  p.n_tiles = ceil_div(F, plan.g);
  p.cols = 32;
  while (p.cols < 4 * plan.g) p.cols *= 2;
  const int a_rows = plan.pair || T >= FM ? FM : (T + 7) / 8 * 8;
  const int b_rows = plan.pair ? 128 : plan.g;  // of the gate or of the up matrix, a CTA and k-block
  const int da_blocks = plan.pair ? 1 : ceil_div(plan.g, 64);
  p.gu_bytes = (uint32_t)(a_rows + (plan.pair ? 1 : 2) * b_rows) * 128u;
  p.da_bytes = (uint32_t)a_rows * 128u + (uint32_t)da_blocks * 8192u;
  int b_bytes = (plan.pair ? 1 : 2) * b_rows * 128;
  if (bwd && da_blocks * 8192 > b_bytes) b_bytes = da_blocks * 8192;
  p.a_bytes = (uint32_t)a_rows * 128u;
  p.stage_bytes = (int)p.a_bytes + b_bytes;
  p.act = (bf16*)act;
  p.dgu = (bf16*)dgu;
  p.act_pitch = act_pitch(d);
  p.dgu_pitch = dgu_pitch(d);
  // A warp that stores 16 bytes of each of its 32 rows takes 32 turns for it, three times in backward. Through slabs instead, single
  // CTAs make a whole backward pass of 333 x 896 x 4864 take 44.7 us and not 45.5, of 777 tokens 71.5 and not 75.9; with fewer
  // rows than a tile's the stages that the slabs cost weigh more: 64 tokens 35.0 and not 32.5.
  const bool slabs = !plan.pair && bwd && T >= FM;
  p.slab_bytes = plan.pair ? epi_groups(true) * F_SLAB_BYTES : slabs ? epi_groups(false) * 3 * F_NARROW_BYTES : 0;
  p.x_scale = x_scale;
  p.w_scale = w_scale;
  p.status = tc_status_device_ptr();
  SRT_REQUIRE(p.status != nullptr, "tcgen05 status word unavailable");
  CUtensorMap tm[7];
  int rc;
  if ((rc = tmap_rows_128b(&tm[0], x, T, C, C, esz, a_rows)) || (rc = tmap_rows_128b(&tm[1], w_gu, 2ull * F, C, C, esz, b_rows))) return rc;
  for (int i = 2; i < 7; ++i) tm[i] = tm[0];
  if (bwd && ((rc = tmap_rows_128b(&tm[2], dy, T, C, C, 2, a_rows)) || (rc = tmap_rows_128b(&tm[3], w_down, C, F, F, 2, 64)))) return rc;
  const int out_cols = plan.pair ? 32 : 16;
  if ((plan.pair || slabs) && (rc = tmap_rows(&tm[4], act, T, F, p.act_pitch, 2, out_cols, FM))) return rc;
  // the two halves of dgu have maps of their own: a store that reaches beyond `hidden` is clipped in either
  if (bwd && (plan.pair || slabs) && ((rc = tmap_rows(&tm[5], dgu, T, F, p.dgu_pitch, 2, out_cols, FM)) ||
                                      (rc = tmap_rows(&tm[6], (bf16*)dgu + F, T, F, p.dgu_pitch, 2, out_cols, FM))))
    return rc;
  if (bwd) return plan.pair ? launch_ffn<true, true, false>(p, tm, st) : launch_ffn<false, true, false>(p, tm, st);
  if (e4m3) return plan.pair ? launch_ffn<true, false, true>(p, tm, st) : launch_ffn<false, false, true>(p, tm, st);
  return plan.pair ? launch_ffn<true, false, false>(p, tm, st) : launch_ffn<false, false, false>(p, tm, st);
}

// ---- a few tokens ---------------------------------------------------------------------------------------
// One to four tokens: the weights are read once and everything else is small, so the products are dot products of weight rows
// on the CUDA cores, without the set-up of tensor memory and tensor maps. A warp has one hidden channel (its gate and its up
// row), or a quarter of one output row; all its loads are in flight together. fp32 sums in a fixed order.
//
// What a token more costs here grows with the weights, and the tensor cores take it for nothing: so the more weights, the fewer
// tokens. Measured with weights out of memory, dot products and tensor cores, us: 896 x 4864 1 token 8.7 and 11.9, 3 11.9 and
// 11.9, 4 13.0 and 12.0; 2048 x 8192 1 token 21.6 and 25.0, 2 25.1 and 25.0, 3 28.6 and 25.0; 4096 x 11008 1 token 50.0 and
// 47.5, in 8 bits 36.0 and 36.0; 1024 x 2816 in 8 bits 1 token 5.6 and 9.6, 4 8.3 and 9.7.
constexpr int TOK_MAX = 4;
bool few_tokens(const srt_gated_ffn_desc& d) {
  return d.tokens <= TOK_MAX && (long long)d.tokens * (d.tokens > 1 ? d.tokens - 1 : 1) * d.width * d.hidden <= 36000000;
}
constexpr int TOK_THREADS = 128;

__device__ __forceinline__ float warp_add(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// 16 bytes of e4m3 as fp32.
__device__ __forceinline__ void unpack_e4m3(const uint4& v, float (&f)[16]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[i] >> (16 * h)), __NV_E4M3);
      const float2 t = __half22float2(__half2(r));
      f[i * 4 + h * 2] = t.x;
      f[i * 4 + h * 2 + 1] = t.y;
    }
}
template <bool E4M3>
__device__ __forceinline__ void unpack_any(const uint4& v, float (&f)[E4M3 ? 16 : 8]) {
  if constexpr (E4M3) {
    unpack_e4m3(v, f);
  } else {
    Vec16<bf16> a;
    a.raw = v;
    a.unpack(f);
  }
}

template <int TT, bool E4M3>
__global__ void __launch_bounds__(TOK_THREADS)
token_gate_kernel(const uint4* __restrict__ x, const uint4* __restrict__ w, const float* __restrict__ x_scale,
                  const float* __restrict__ w_scale, bf16* __restrict__ act, int vecs, int F) {
  constexpr int V = E4M3 ? 16 : 8, U = 4;
  pdl_enter();
  const int lane = threadIdx.x & 31, f = (int)blockIdx.x * (TOK_THREADS / 32) + (threadIdx.x >> 5);
  if (f >= F) return;
  const uint4 *wg = w + (size_t)f * vecs, *wu = w + (size_t)(F + f) * vecs;
  float g[TT], u[TT];
#pragma unroll
  for (int t = 0; t < TT; ++t) g[t] = u[t] = 0.f;
  for (int v0 = lane; v0 < vecs; v0 += 32 * U) {
    uint4 a[U], b[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const bool in = v0 + 32 * i < vecs;
      a[i] = in ? __ldcs(wg + v0 + 32 * i) : make_uint4(0, 0, 0, 0);
      b[i] = in ? __ldcs(wu + v0 + 32 * i) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (v0 + 32 * i >= vecs) break;
      float fa[V], fb[V];
      unpack_any<E4M3>(a[i], fa);
      unpack_any<E4M3>(b[i], fb);
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        float fx[V];
        unpack_any<E4M3>(x[(size_t)t * vecs + v0 + 32 * i], fx);
#pragma unroll
        for (int e = 0; e < V; ++e) { g[t] = fmaf(fa[e], fx[e], g[t]); u[t] = fmaf(fb[e], fx[e], u[t]); }
      }
    }
  }
#pragma unroll
  for (int t = 0; t < TT; ++t) {
    g[t] = warp_add(g[t]);
    u[t] = warp_add(u[t]);
  }
  if (lane == 0) {
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      if (E4M3) {
        g[t] *= x_scale[t] * w_scale[f];
        u[t] *= x_scale[t] * w_scale[F + f];
      }
      act[(size_t)t * F + f] = __float2bfloat16_rn(g[t] * sigmoid_f(g[t]) * u[t]);
    }
  }
}

// One output row of Wd a block, a quarter of it a warp. The first loads of the row leave before the launch in front, the
// gate's, has ended: it does not write weights, and it has waited for whatever did. (They bypass L1.) That holds for the blocks
// that find room beside the gate's: 56 registers a thread there leave an SM with eight of its blocks room for two of these, and
// one with nine for none, so of 896 rows beside 4864 hidden channels some 230 have loads on the way; the others start cold.
template <int TT>
__global__ void __launch_bounds__(TOK_THREADS)
token_down_kernel(const uint4* act, const uint4* __restrict__ w, const bf16* __restrict__ residual, bf16* __restrict__ y, int vecs, int C) {
  constexpr int U = 4, WARPS = TOK_THREADS / 32;
  __shared__ float sh[WARPS][TT];
  const int c = blockIdx.x;
  const uint4* wr = w + (size_t)c * vecs;
  uint4 a[U];
  auto fetch = [&](int v0) {
#pragma unroll
    for (int i = 0; i < U; ++i) a[i] = v0 + TOK_THREADS * i < vecs ? __ldcg(wr + v0 + TOK_THREADS * i) : make_uint4(0, 0, 0, 0);
  };
  fetch(threadIdx.x);
  pdl_enter();
  float s[TT];
#pragma unroll
  for (int t = 0; t < TT; ++t) s[t] = 0.f;
  for (int v0 = threadIdx.x; v0 < vecs; v0 += TOK_THREADS * U) {
    if (v0 != (int)threadIdx.x) fetch(v0);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (v0 + TOK_THREADS * i >= vecs) break;
      float fa[8];
      unpack_any<false>(a[i], fa);
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        float fx[8];
        unpack_any<false>(act[(size_t)t * vecs + v0 + TOK_THREADS * i], fx);
#pragma unroll
        for (int e = 0; e < 8; ++e) s[t] = fmaf(fa[e], fx[e], s[t]);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < TT; ++t) {
    s[t] = warp_add(s[t]);
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5][t] = s[t];
  }
  __syncthreads();
  if (threadIdx.x < TT) {
    const int t = threadIdx.x;
    float r = 0.f;
#pragma unroll
    for (int k = 0; k < WARPS; ++k) r += sh[k][t];
    if (residual) r += __bfloat162float(residual[(size_t)t * C + c]);
    y[(size_t)t * C + c] = __float2bfloat16_rn(r);
  }
}

template <int TT>
int token_ffn(const srt_gated_ffn_desc& d, const void* x, const float* x_scale, const void* w_gu, const float* w_scale, const void* w_down,
              const void* residual, void* act, void* y, cudaStream_t st) {
  const dim3 grid(ceil_div(d.hidden, TOK_THREADS / 32));
  if (x_scale)
    SRT_CHECK_CUDA(launch_pdl(token_gate_kernel<TT, true>, grid, dim3(TOK_THREADS), 0, st, (const uint4*)x, (const uint4*)w_gu, x_scale, w_scale,
                              (bf16*)act, d.width / 16, d.hidden));
  else
    SRT_CHECK_CUDA(launch_pdl(token_gate_kernel<TT, false>, grid, dim3(TOK_THREADS), 0, st, (const uint4*)x, (const uint4*)w_gu, x_scale, w_scale,
                              (bf16*)act, d.width / 8, d.hidden));
  SRT_LAUNCH_CHECK();
  SRT_CHECK_CUDA(launch_pdl(token_down_kernel<TT>, dim3(d.width), dim3(TOK_THREADS), 0, st, (const uint4*)act, (const uint4*)w_down,
                            (const bf16*)residual, (bf16*)y, d.hidden / 8, d.width));
  SRT_LAUNCH_CHECK();
  return SRT_OK;
}

size_t up256(size_t v) { return (v + 255) / 256 * 256; }
int check_ffn(const srt_gated_ffn_desc* d, int width_unit) {
  SRT_REQUIRE(d, "gated_ffn: null descriptor");
  SRT_REQUIRE(d->tokens >= 0 && d->width > 0 && d->hidden > 0, "gated_ffn: sizes %d, %d, %d out of range", d->tokens, d->width, d->hidden);
  SRT_REQUIRE(d->width % width_unit == 0 && d->hidden % 8 == 0, "gated_ffn: width (%d) must be a multiple of %d and hidden (%d) of 8",
              d->width, width_unit, d->hidden);
  SRT_REQUIRE((long long)d->tokens * 2 * d->hidden < (1ll << 31) && (long long)d->tokens * d->width < (1ll << 31) &&
                  2ll * d->hidden * d->width < (1ll << 31),
              "gated_ffn: a matrix of %d tokens x (%d, 2 x %d) exceeds 2^31 elements", d->tokens, d->width, d->hidden);
  return SRT_OK;
}
#define FFN_ALIGNED(...) ffn_aligned({__VA_ARGS__})
int ffn_aligned(std::initializer_list<const void*> ps) {
  for (const void* q : ps) SRT_REQUIRE(((uintptr_t)q & 15) == 0, "gated_ffn: operands must be 16-byte aligned");
  return SRT_OK;
}

// The plain products around the gated one.
GemmProblem down_problem(const srt_gated_ffn_desc& d) { return {d.tokens, d.width, d.hidden, false, false, SRT_BF16, act_pitch(d)}; }  // y
GemmProblem dx_problem(const srt_gated_ffn_desc& d) { return {d.tokens, d.width, 2 * d.hidden, false, true, SRT_BF16, dgu_pitch(d)}; }
GemmProblem dw_problem(const srt_gated_ffn_desc& d, int type) { return {2 * d.hidden, d.width, d.tokens, true, true, type, dgu_pitch(d)}; }  // dWg over dWu
GemmProblem dd_problem(const srt_gated_ffn_desc& d, int type) { return {d.width, d.hidden, d.tokens, true, true, type, 0, act_pitch(d)}; }   // dWd
size_t larger(size_t a, size_t b) { return a > b ? a : b; }

}  // namespace

size_t gated_ffn_fwd_scratch_bytes(const srt_gated_ffn_desc& d) {
  return up256((size_t)d.tokens * act_pitch(d) * 2) + balanced_gemm_scratch_bytes(down_problem(d));
}

int gated_ffn_fwd(const srt_gated_ffn_desc* d, const void* x, const float* x_scale, const void* w_gu, const float* w_scale,
                  const void* w_down, const void* residual, void* y, void* scratch, size_t scratch_bytes, bool e4m3, cudaStream_t st) {
  int rc = check_ffn(d, e4m3 ? 16 : 8);
  if (rc || d->tokens == 0) return rc;
  SRT_REQUIRE(x && w_gu && w_down && y && (!e4m3 || (x_scale && w_scale)), "gated_ffn_fwd: null operand");
  const size_t act_bytes = up256((size_t)d->tokens * act_pitch(*d) * 2);
  SRT_REQUIRE(scratch && scratch_bytes >= act_bytes, "gated_ffn_fwd: scratch too small (%zu < %zu)", scratch_bytes, act_bytes);
  if ((rc = FFN_ALIGNED(x, w_gu, w_down, residual, y, scratch))) return rc;
  SRT_REQUIRE((((uintptr_t)x_scale | (uintptr_t)w_scale) & 3) == 0, "gated_ffn: scales must be aligned to 4 bytes");
  void* act = scratch;
  switch (few_tokens(*d) ? d->tokens : 0) {
    case 1: return token_ffn<1>(*d, x, x_scale, w_gu, w_scale, w_down, residual, act, y, st);
    case 2: return token_ffn<2>(*d, x, x_scale, w_gu, w_scale, w_down, residual, act, y, st);
    case 3: return token_ffn<3>(*d, x, x_scale, w_gu, w_scale, w_down, residual, act, y, st);
    case TOK_MAX: return token_ffn<TOK_MAX>(*d, x, x_scale, w_gu, w_scale, w_down, residual, act, y, st);
  }
  if ((rc = gated_products(*d, x, x_scale, w_gu, w_scale, nullptr, nullptr, act, nullptr, st))) return rc;
  return balanced_gemm(down_problem(*d), act, w_down, residual, y, (char*)scratch + act_bytes, scratch_bytes - act_bytes, true, st);
}

GatedFfnScratch gated_ffn_scratch(const srt_gated_ffn_desc& d, int grad_dtype) {
  GatedFfnScratch s;
  s.dgu = up256((size_t)d.tokens * act_pitch(d) * 2);
  s.slots = s.dgu + up256((size_t)d.tokens * dgu_pitch(d) * 2);
  s.total = s.slots + larger(balanced_gemm_scratch_bytes(dx_problem(d)),
                             larger(balanced_gemm_scratch_bytes(dw_problem(d, grad_dtype)), balanced_gemm_scratch_bytes(dd_problem(d, grad_dtype))));
  return s;
}

int gated_ffn_bwd(const srt_gated_ffn_desc* d, const void* dy, const void* x, const void* w_gu, const void* w_down, int grad_dtype,
                  void* dx, void* dw_gu, void* dw_down, void* scratch, size_t scratch_bytes, cudaStream_t st) {
  int rc = check_ffn(d, 8);
  if (rc) return rc;
  SRT_REQUIRE(grad_dtype == SRT_F32 || grad_dtype == SRT_BF16, "gated_ffn_bwd: gradient type %d is neither SRT_F32 nor SRT_BF16", grad_dtype);
  const size_t CF = (size_t)d->width * d->hidden, gsz = grad_dtype == SRT_F32 ? 4 : 2;
  if (d->tokens == 0) {
    if (dw_gu) SRT_CHECK_CUDA(cudaMemsetAsync(dw_gu, 0, 2 * CF * gsz, st));
    if (dw_down) SRT_CHECK_CUDA(cudaMemsetAsync(dw_down, 0, CF * gsz, st));
    return SRT_OK;
  }
  SRT_REQUIRE(dy && x && w_gu && w_down, "gated_ffn_bwd: null operand");
  const GatedFfnScratch s = gated_ffn_scratch(*d, grad_dtype);
  SRT_REQUIRE(scratch && scratch_bytes >= s.slots, "gated_ffn_bwd: scratch too small (%zu < %zu)", scratch_bytes, s.total);
  if ((rc = FFN_ALIGNED(dy, x, w_gu, w_down, dx, dw_gu, dw_down, scratch))) return rc;
  char* base = (char*)scratch;
  void *act = base, *dgu = base + s.dgu, *slots = base + s.slots;
  const size_t room = scratch_bytes - s.slots;
  if ((rc = gated_products(*d, x, nullptr, w_gu, nullptr, dy, w_down, act, dgu, st))) return rc;
  if (dx && (rc = balanced_gemm(dx_problem(*d), dgu, w_gu, nullptr, dx, slots, room, true, st))) return rc;
  if (dw_gu && (rc = balanced_gemm(dw_problem(*d, grad_dtype), dgu, x, nullptr, dw_gu, slots, room, true, st))) return rc;
  // act comes from the gated kernel, which is directly in front where nothing else was asked for
  if (dw_down && (rc = balanced_gemm(dd_problem(*d, grad_dtype), dy, act, nullptr, dw_down, slots, room, dx || dw_gu, st))) return rc;
  return SRT_OK;
}

}  // namespace srt

using namespace srt;

extern "C" {

size_t srt_gated_ffn_fwd_scratch_bytes(const srt_gated_ffn_desc* d) { return check_ffn(d, 8) ? 0 : gated_ffn_fwd_scratch_bytes(*d); }

int srt_gated_ffn_fwd(const srt_gated_ffn_desc* d, const void* x, const void* w_gate_up, const void* w_down, const void* residual,
                      void* y, void* scratch, size_t scratch_bytes, void* stream) {
  return gated_ffn_fwd(d, x, nullptr, w_gate_up, nullptr, w_down, residual, y, scratch, scratch_bytes, false, (cudaStream_t)stream);
}

int srt_gated_ffn_fwd_e4m3(const srt_gated_ffn_desc* d, const void* x, const float* x_scale, const void* w_gate_up,
                           const float* w_scale, const void* w_down, const void* residual, void* y, void* scratch, size_t scratch_bytes,
                           void* stream) {
  return gated_ffn_fwd(d, x, x_scale, w_gate_up, w_scale, w_down, residual, y, scratch, scratch_bytes, true, (cudaStream_t)stream);
}

size_t srt_gated_ffn_bwd_scratch_bytes(const srt_gated_ffn_desc* d, int grad_dtype) {
  return check_ffn(d, 8) ? 0 : gated_ffn_scratch(*d, grad_dtype).total;
}

int srt_gated_ffn_bwd(const srt_gated_ffn_desc* d, const void* dy, const void* x, const void* w_gate_up, const void* w_down,
                      int grad_dtype, void* dx, void* dw_gate_up, void* dw_down, void* scratch, size_t scratch_bytes, void* stream) {
  return gated_ffn_bwd(d, dy, x, w_gate_up, w_down, grad_dtype, dx, dw_gate_up, dw_down, scratch, scratch_bytes, (cudaStream_t)stream);
}

}  // extern "C"
