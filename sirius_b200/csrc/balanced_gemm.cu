// Products whose work is dealt evenly to all SMs: D = A B (+ addend) with either operand stored along or across the reduction.
//
// The output is cut into tiles; a unit (a CTA, or a CTA pair with cta_group::2) takes whole tiles while there are enough for
// all, and what is left over, fewer tiles than units, is cut along the reduction into as many equal ranges as there are units.
// A unit that has only a part of a tile's reduction leaves fp32 sums in a slot of its own, and a second, small launch adds the
// slots of every such tile in the order of the reduction. So the 152 tiles of a weight gradient take 74 pairs 2.05 rounds and not
// three, a few rows against a long reduction occupy the device, no CTA waits for another, and the sums have a fixed order. With
// few tiles a cluster shares each, and the parts meet in its shared memory instead (split_gemm_kernel).
//
// Warps as in the gated kernels: 0 TMA, 1 MMA, 2-17 four epilogue groups that take the 32-column slabs of a tile in turn. The
// accumulator is double-buffered in tensor memory, so the epilogue of a tile runs beside the products of the next.
//
// Of the feed-forward block of 8192 tokens x 896 x 4864: y 56 us, 1270 TFLOP/s, tensor pipe 65 % busy (128 tiles on 74 pairs, two
// rounds for 1.73 of work; sharing the rest would cost more in slots and a second launch); dx 97 us, 1480, 80 % (one round of whole
// tiles, 54 shared by all pairs, a join of 5 behind it); dWg over dWu 94 us, 1520, 83 % (two rounds, 4 tiles shared, a join); dWd
// 54 us, 1320, 70 % (133 tiles for 148 CTAs). Operands come out of L2 at 11 to 15 TB/s, which is what single CTAs are bound by;
// pairs read half of B each. A library product of these sizes takes 57, 109, 123 and 57 us. Two slabs for the output of an epilogue
// group instead of one cost a stage: dWd 55 -> 67 us.
#include <cuda.h>

#include <atomic>

#include "balanced_gemm.cuh"
#include "ptx.cuh"

namespace srt {

int* tc_status_device_ptr();  // igemm_tcgen05.cu
int tmap_rows(CUtensorMap* tm, const void* base, uint64_t rows, uint64_t cols, uint64_t pitch, int elem_bytes, uint32_t box_cols, uint32_t box_rows);

namespace {

using namespace ptx;
using bf16 = __nv_bfloat16;

constexpr int BM = 128;
constexpr int EPI_GROUPS = 4;                     // of four warps
constexpr int G_THREADS = 64 + 128 * EPI_GROUPS;
constexpr int G_MAX_STAGES = 16;
constexpr int SLAB_BYTES = BM * 64;  // 128 rows x 32 bf16 or 16 fp32, 64-byte swizzle
enum { W_GEMM_LOAD = 0x41, W_GEMM_FULL = 0x42, W_GEMM_ACC = 0x43, W_GEMM_EPI = 0x44, W_GEMM_DRAIN = 0x45 };

struct GemmParams {
  int M, N, k_blocks, n;       // n: columns of a tile, a multiple of 32
  int m_units, n_tiles, band;  // tiles are walked in bands of `band` columns of tiles
  int tiles, units, rounds;    // a unit has up to `rounds` whole tiles ...
  int rest, sharers;           // ... and the first `sharers` units share the `rest` tiles beyond those
  int cols;                    // tensor-memory columns
  int stages, stage_bytes;
  uint32_t a_bytes;            // of a stage: with fewer than 128 rows only those; the products read on into what follows, and
                               // the rows of the accumulator that this fills are not stored
  uint32_t load_bytes;         // of one CTA a k-block
  int f32_out;
  int b_early;                 // B may be read before the launch in front of this one has ended
  const bf16* addend;
  void* D;
  const float* slots;          // [2 sharers][rows of a unit][n]
  int* status;
};

// The walk of a unit over its share: whole tiles first, then its range of the shared ones.
struct Walk {
  int i;
  long long at, end;  // position and end in the shared range, in k-blocks
};
struct Piece {
  int tile, k0, k1, slot;  // slot < 0: the whole reduction
};
__host__ __device__ inline long long share_begin(long long work, int unit, int units) { return work * unit / units; }
__device__ __forceinline__ Walk walk_begin(const GemmParams& p, int unit) {
  if (unit >= p.sharers) return {0, 0, 0};
  const long long work = (long long)p.rest * p.k_blocks;
  return {0, share_begin(work, unit, p.sharers), share_begin(work, unit + 1, p.sharers)};
}
__device__ __forceinline__ bool walk_next(const GemmParams& p, int unit, Walk& w, Piece& o) {
  if (w.i < p.rounds && unit + w.i * p.units < p.tiles) {
    o = {unit + w.i * p.units, 0, p.k_blocks, -1};
    ++w.i;
    return true;
  }
  if (w.at >= w.end) return false;
  const int t = (int)(w.at / p.k_blocks);
  const long long first = (long long)t * p.k_blocks, stop = w.end < first + p.k_blocks ? w.end : first + p.k_blocks;
  o.tile = p.rounds * p.units + t;
  o.k0 = (int)(w.at - first);
  o.k1 = (int)(stop - first);
  o.slot = o.k0 == 0 && o.k1 == p.k_blocks ? -1 : 2 * unit + (o.k0 == 0 ? 1 : 0);
  w.at = stop;
  return true;
}
__host__ __device__ inline void tile_at(const GemmParams& p, int t, int& m, int& n) {
  const int b = t / (p.band * p.m_units), first = b * p.band;
  const int size = p.n_tiles - first < p.band ? p.n_tiles - first : p.band, r = t - first * p.m_units;
  m = r / size;
  n = first + r - m * size;
}

template <bool PAIR, bool A_MN, bool B_MN>
__global__ void __launch_bounds__(G_THREADS, 1)
balanced_gemm_kernel(const GemmParams p, const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tb,
                     const __grid_constant__ CUtensorMap td, const __grid_constant__ CUtensorMap tslot) {
  constexpr int NCTA = PAIR ? 2 : 1;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const int NS = p.stages;
  uint8_t* sOut = base + NS * p.stage_bytes;
  uint64_t* bars = (uint64_t*)(sOut + EPI_GROUPS * SLAB_BYTES);
  const uint32_t full = smem_u32(bars), empty = full + 8 * G_MAX_STAGES, acc_full = empty + 8 * G_MAX_STAGES, acc_empty = acc_full + 16;
  uint32_t* tmem_ptr = (uint32_t*)(bars + 2 * G_MAX_STAGES + 4);
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const uint32_t rank = PAIR ? cluster_ctarank() : 0u;
  const int unit = (int)blockIdx.x / NCTA;
  const int n_cta = p.n / NCTA;  // columns of B that this CTA stages
  const uint32_t s0 = smem_u32(base);

  if (tid == 0) {
    for (int s = 0; s < NS; ++s) { mbar_init(full + 8 * s, 1); mbar_init(empty + 8 * s, 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(acc_full + 8 * b, 1); mbar_init(acc_empty + 8 * b, 4 * EPI_GROUPS * NCTA); }
    mbar_fence_init();
  }
  if (warp == 0 && lane == 0) { tma_prefetch_desc(&ta); tma_prefetch_desc(&tb); tma_prefetch_desc(&td); }
  if (warp == 1) {
    if (PAIR) { tmem_alloc_pair(smem_u32(tmem_ptr), p.cols); tmem_relinquish_pair(); }
    else { tmem_alloc(smem_u32(tmem_ptr), p.cols); tmem_relinquish(); }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (PAIR) cluster_sync_all();  // the peer's barriers and tensor memory exist before anything refers to them
  tc_fence_after_sync();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_ptr, 0);
  // A producer that may fetch B ahead of the launch in front enters later: its first stages travel while that one drains.
  const bool ahead = p.b_early && warp == 0;
  if (!ahead) pdl_enter();

  if (warp == 0) {
    // The warp walks together and one thread of it issues (see elect_one); what does not change from one k-block to the next
    // stays out of the loops.
    const uint32_t bytes = p.load_bytes * NCTA, full_to = PAIR ? map_to_cta(full, 0u) : full;  // the leader's barriers
    const uint32_t wrap = (uint32_t)NS * p.stage_bytes;
    int it = 0, early = 0;
    uint32_t at = 0, bar = 0, ph = 1;  // offsets of the current stage and of its barriers
    bool ok = true;
    auto step = [&]() {
      at += p.stage_bytes;
      bar += 8;
      if (at == wrap) { at = 0; bar = 0; ph ^= 1u; }
    };
    auto load = [&](uint32_t dst, const CUtensorMap* tm, int x, int y) {
      if (PAIR) tma_load_2d_pair(dst, tm, full_to + bar, x, y);
      else tma_load_2d(dst, tm, full_to + bar, x, y);
    };
    auto load_a = [&](int m0, int k0) {
      const uint32_t a = s0 + at;
      if (A_MN) {
        load(a, &ta, m0, k0);
        load(a + 8192u, &ta, m0 + 64, k0);
      } else {
        load(a, &ta, k0, m0);
      }
    };
    auto load_b = [&](int n0, int k0) {
      const uint32_t b = s0 + at + p.a_bytes;
      if (B_MN) {
        load(b, &tb, n0, k0);
        if (n_cta > 64) load(b + 8192u, &tb, n0 + 64, k0);
        if (!PAIR && n_cta > 128) {
          load(b + 16384u, &tb, n0 + 128, k0);
          if (n_cta > 192) load(b + 24576u, &tb, n0 + 192, k0);
        }
      } else {
        load(b, &tb, k0, n0);
      }
    };
    if (ahead) {
      Walk w = walk_begin(p, unit);
      Piece o;
      while (early < NS && walk_next(p, unit, w, o)) {
        int m, n;
        tile_at(p, o.tile, m, n);
        for (int kb = o.k0; kb < o.k1 && early < NS; ++kb, ++early) {
          if (elect_one()) {
            if (rank == 0) mbar_arrive_expect_tx(full + bar, bytes);
            load_b(n * p.n + (int)rank * n_cta, kb * 64);
          }
          step();
        }
      }
      pdl_enter();
      at = bar = 0;
      ph = 1;
    }
    Walk w = walk_begin(p, unit);
    Piece o;
    while (ok && walk_next(p, unit, w, o)) {
      int m, n;
      tile_at(p, o.tile, m, n);
      const int m0 = (m * NCTA + (int)rank) * BM, n0 = n * p.n + (int)rank * n_cta;
      int k0 = o.k0 * 64;
      const int k1 = o.k1 * 64;
      for (; it < early && k0 < k1; k0 += 64, ++it) {
        if (elect_one()) load_a(m0, k0);
        step();
      }
      for (; k0 < k1; k0 += 64, ++it) {
        ok = mbar_wait_warp<false>(empty + bar, ph, p.status, W_GEMM_LOAD);
        if (!ok) break;
        if (elect_one()) {
          if (rank == 0) mbar_arrive_expect_tx(full + bar, bytes);
          load_a(m0, k0);
          load_b(n0, k0);
        }
        step();
      }
    }
    // a wait that gave up: the copies in flight land before the CTA's memory is given back
    if (!ok && rank == 0)
      for (int k = it > NS ? it - NS : 0; k < it; ++k) mbar_wait_warp<false>(full + 8 * (k % NS), (uint32_t)(k / NS) & 1u, p.status, W_GEMM_DRAIN);
  } else if (warp == 1) {
    if (rank == 0) {
      const uint32_t idesc = make_idesc_bf16(BM * NCTA, p.n, A_MN, B_MN);
      constexpr uint32_t a_step = A_MN ? 2048u : 32u, b_step = B_MN ? 2048u : 32u;  // 16 elements along the reduction
      const uint64_t desc_a = make_smem_desc_sw128(s0, A_MN ? 8192 : 0, 1024), desc_b = make_smem_desc_sw128(s0 + p.a_bytes, B_MN ? 8192 : 0, 1024);
      const uint32_t wrap = (uint32_t)NS * p.stage_bytes;
      int i = 0;
      uint32_t at = 0, bar = 0, ph = 0;
      bool ok = true;
      Walk w = walk_begin(p, unit);
      Piece o;
      for (; ok && walk_next(p, unit, w, o); ++i) {
        const uint32_t b2 = (uint32_t)i & 1u, acc = tmem + b2 * (uint32_t)(p.cols / 2);
        ok = mbar_wait_warp<PAIR>(acc_empty + 8 * b2, ((uint32_t)(i >> 1) & 1u) ^ 1u, p.status, W_GEMM_ACC);
        if (!ok) break;
        uint32_t add = 0;
        for (int kb = o.k0; kb < o.k1; ++kb) {
          ok = mbar_wait_warp<PAIR>(full + bar, ph, p.status, W_GEMM_FULL);
          if (!ok) break;
          tc_fence_after_sync();
          if (elect_one()) {
            const uint64_t ad = desc_at(desc_a, at), bd = desc_at(desc_b, at);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if (PAIR) umma_bf16_pair(acc, desc_at(ad, k * a_step), desc_at(bd, k * b_step), idesc, k ? 1u : add);
              else umma_bf16(acc, desc_at(ad, k * a_step), desc_at(bd, k * b_step), idesc, k ? 1u : add);
            }
            if (PAIR) umma_commit_pair(empty + bar, (uint16_t)3);
            else umma_commit(empty + bar);
          }
          add = 1;
          at += p.stage_bytes;
          bar += 8;
          if (at == wrap) { at = 0; bar = 0; ph ^= 1u; }
        }
        if (!ok) break;
        if (elect_one()) {
          if (PAIR) umma_commit_pair(acc_full + 8 * b2, (uint16_t)3);
          else umma_commit(acc_full + 8 * b2);
        }
      }
    }
  } else {
    const int grp = (warp - 2) >> 2, q = warp & 3, row = q * 32 + lane;
    const bool issuer = ((warp - 2) & 3) == 0 && lane == 0;
    const uint32_t lanes = (uint32_t)(q * 32) << 16;
    const uint32_t slab = smem_u32(sOut) + (uint32_t)grp * SLAB_BYTES;
    bool ok = true;
    Walk w = walk_begin(p, unit);
    Piece o;
    for (int i = 0; walk_next(p, unit, w, o); ++i) {
      int m, n;
      tile_at(p, o.tile, m, n);
      const int m0 = (m * NCTA + (int)rank) * BM, n0 = n * p.n, mrow = m0 + row;
      const uint32_t b2 = (uint32_t)i & 1u, acc = tmem + lanes + b2 * (uint32_t)(p.cols / 2);
      const bool whole = o.slot < 0, wide = p.f32_out || !whole;
      // the addend of the first slab travels while the products run
      Vec16<bf16> add[4];
      auto fetch = [&](int c) {
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          add[v].raw = make_uint4(0, 0, 0, 0);
          const int col = n0 + c + v * 8;
          if (whole && p.addend && mrow < p.M && c < p.n && col < p.N) add[v].load(p.addend + (size_t)mrow * p.N + col);
        }
      };
      fetch(grp * 32);
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(acc_full + 8 * b2, (uint32_t)(i >> 1) & 1u, p.status, W_GEMM_EPI));
      tc_fence_after_sync();
      for (int c = grp * 32; c < p.n; c += 32 * EPI_GROUPS) {
        if (m0 >= p.M || n0 + c >= p.N) break;  // the same for the whole group; nothing of the slab exists
        uint32_t f[32];
        tmem_ld_32x32b_x32(acc + (uint32_t)c, f);
        tmem_ld_wait();
        if (p.addend && whole) {
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            float a[8];
            add[v].unpack(a);
#pragma unroll
            for (int e = 0; e < 8; ++e) f[v * 8 + e] = __float_as_uint(__uint_as_float(f[v * 8 + e]) + a[e]);
          }
          fetch(c + 32 * EPI_GROUPS);
        }
        // 64 bytes of every row at a time: all 32 columns in bf16, 16 of them in fp32
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (!wide) {
            if (h == 1) break;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              __nv_bfloat162 v = __floats2bfloat162_rn(__uint_as_float(f[2 * e]), __uint_as_float(f[2 * e + 1]));
              f[e] = *reinterpret_cast<uint32_t*>(&v);
            }
          }
          if (issuer) bulk_wait_group_read<0>();  // the store before has read the slab
          named_bar_sync(1 + grp, 128);
#pragma unroll
          for (int v = 0; v < 4; ++v)
            st_shared_v4(slab + (uint32_t)row * 64u + (uint32_t)((v ^ ((row >> 1) & 3)) << 4), f[h * 16 + v * 4], f[h * 16 + v * 4 + 1],
                         f[h * 16 + v * 4 + 2], f[h * 16 + v * 4 + 3]);
          fence_proxy_async_smem();
          named_bar_sync(1 + grp, 128);
          if (issuer) {
            if (whole) tma_store_2d(&td, slab, n0 + c + h * 16, m0);
            else tma_store_2d(&tslot, slab, c + h * 16, (o.slot * NCTA + (int)rank) * BM);
            bulk_commit_group();
          }
        }
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        if (PAIR) mbar_arrive_cluster(map_to_cta(acc_empty + 8 * b2, 0u));
        else mbar_arrive(acc_empty + 8 * b2);
      }
    }
    if (issuer) bulk_wait_group_read<0>();  // the slab outlives the last store's read
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

// The tiles whose reduction was shared, found by the host: the slots of units u0 ... u1 in the order of the reduction, plus the
// addend. Block (tile, part of its rows); a thread has four columns of a row, eight slots in flight.
// (Blocks that found their tile themselves, by divisions of 64-bit numbers: 10 to 16 us for 54 tiles. Several
// rows a thread, one after the other: 7.6 to 12 us for 54 tiles of two slots, 7.8 us for two tiles of 32.)
constexpr int JOIN_THREADS = 256, JOIN_MAX = 160;
struct JoinList {
  struct { int m, n, u0, u1; } t[JOIN_MAX];
};
__global__ void __launch_bounds__(JOIN_THREADS)
balanced_gemm_join_kernel(const GemmParams p, const __grid_constant__ JoinList list, int unit_rows, int block_rows) {
  pdl_enter();
  const int u0 = list.t[blockIdx.x].u0, u1 = list.t[blockIdx.x].u1;
  const int row0 = list.t[blockIdx.x].m * unit_rows, col0 = list.t[blockIdx.x].n * p.n;
  const int per_row = p.n / 4;
  const size_t step = (size_t)2 * unit_rows * p.n;
  const int ri = threadIdx.x / per_row, r = (int)blockIdx.y * block_rows + ri, c = (threadIdx.x - ri * per_row) * 4;
  if (ri >= block_rows || r >= unit_rows || row0 + r >= p.M || col0 + c >= p.N) return;  // N is a multiple of eight
  const size_t at = (size_t)(row0 + r) * p.N + col0 + c;
  uint2 add = make_uint2(0u, 0u);
  if (p.addend) add = *reinterpret_cast<const uint2*>(p.addend + at);
  const float* f = p.slots + (size_t)u0 * step + (size_t)r * p.n + c;
  float4 s = *reinterpret_cast<const float4*>(f + step / 2);
  f += step;
  for (int k = u0 + 1; k <= u1; k += 8, f += 8 * step) {
    float4 a[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) a[j] = k + j <= u1 ? *reinterpret_cast<const float4*>(f + j * step) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int j = 0; j < 8; ++j) { s.x += a[j].x; s.y += a[j].y; s.z += a[j].z; s.w += a[j].w; }
  }
  s.x += __uint_as_float(add.x << 16);
  s.y += __uint_as_float(add.x & 0xffff0000u);
  s.z += __uint_as_float(add.y << 16);
  s.w += __uint_as_float(add.y & 0xffff0000u);
  if (p.f32_out) {
    *reinterpret_cast<float4*>((float*)p.D + at) = s;
  } else {
    __nv_bfloat162 lo = __floats2bfloat162_rn(s.x, s.y), hi = __floats2bfloat162_rn(s.z, s.w);
    *reinterpret_cast<uint2*>((bf16*)p.D + at) = make_uint2(*reinterpret_cast<uint32_t*>(&lo), *reinterpret_cast<uint32_t*>(&hi));
  }
}

// ---- a tile a cluster -------------------------------------------------------------------------------------
// With few tiles a cluster of c CTAs shares one: each takes a part of the reduction in 128 elements a stage (two blocks of 64),
// leaves its fp32 sums in its own shared memory, and adds a part of the tile from all of them in the order of the reduction.
// One launch, and no slots in memory. What a few tokens need: their products wait for memory and for launches, not for the
// tensor cores.
constexpr int SPLIT_MAX = 8;  // CTAs of a portable cluster
struct SplitParams {
  int M, N, n, c, m_units, steps;  // steps of 128 along the reduction, at least c
  int cols;                        // tensor-memory columns
  int stages;
  uint32_t a_bytes, b_bytes;       // of a block; as in GemmParams, few rows are staged alone
  int f32_out, b_early;
  const bf16* addend;
  void* D;
  int* status;
};
template <bool B_MN>
__global__ void __launch_bounds__(G_THREADS, 1)
split_gemm_kernel(const SplitParams p, const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tb) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const int NS = p.stages;
  const uint32_t stage_bytes = 2u * (p.a_bytes + p.b_bytes);
  uint64_t* bars = (uint64_t*)(base + (uint32_t)NS * stage_bytes + BM * 128 - p.a_bytes);
  const uint32_t full = smem_u32(bars), empty = full + 8 * G_MAX_STAGES, acc_full = empty + 8 * G_MAX_STAGES;
  uint32_t* tmem_ptr = (uint32_t*)(bars + 2 * G_MAX_STAGES + 1);
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const uint32_t s0 = smem_u32(base), rank = cluster_ctarank();
  const int tile = (int)blockIdx.x / p.c, m0 = tile % p.m_units * BM, n0 = tile / p.m_units * p.n;
  const int k0 = p.steps * (int)rank / p.c, k1 = p.steps * ((int)rank + 1) / p.c;

  if (tid == 0) {
    for (int s = 0; s < NS; ++s) { mbar_init(full + 8 * s, 1); mbar_init(empty + 8 * s, 1); }
    mbar_init(acc_full, 1);
    mbar_fence_init();
  }
  if (warp == 0 && lane == 0) { tma_prefetch_desc(&ta); tma_prefetch_desc(&tb); }
  if (warp == 1) { tmem_alloc(smem_u32(tmem_ptr), p.cols); tmem_relinquish(); }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_ptr, 0);
  const bool ahead = p.b_early && warp == 0;
  if (!ahead) pdl_enter();

  if (warp == 0) {
    const uint32_t wrap = (uint32_t)NS * stage_bytes;
    uint32_t at = 0, bar = 0, ph = 1;
    auto step = [&]() {
      at += stage_bytes;
      bar += 8;
      if (at == wrap) { at = 0; bar = 0; ph ^= 1u; }
    };
    auto load_a = [&](int k) {
      tma_load_2d(s0 + at, &ta, full + bar, k * 128, m0);
      tma_load_2d(s0 + at + p.a_bytes, &ta, full + bar, k * 128 + 64, m0);
    };
    auto load_b = [&](int k) {
      mbar_arrive_expect_tx(full + bar, stage_bytes);
      uint32_t b = s0 + at + 2u * p.a_bytes;
      if (B_MN) {
        for (int h = 0; h < 2; ++h)
          for (int x = 0; x < p.n; x += 64, b += 8192u) tma_load_2d(b, &tb, full + bar, n0 + x, k * 128 + h * 64);
      } else {
        tma_load_2d(b, &tb, full + bar, k * 128, n0);
        tma_load_2d(b + p.b_bytes, &tb, full + bar, k * 128 + 64, n0);
      }
    };
    int early = k0;
    if (ahead) {
      for (; early < k1 && early < k0 + NS; ++early) {
        if (elect_one()) load_b(early);
        step();
      }
      pdl_enter();
      at = bar = 0;
      ph = 1;
    }
    int k = k0;
    for (; k < early; ++k) {
      if (elect_one()) load_a(k);
      step();
    }
    bool ok = true;
    for (; k < k1; ++k) {
      ok = mbar_wait_warp<false>(empty + bar, ph, p.status, W_GEMM_LOAD);
      if (!ok) break;
      if (elect_one()) {
        load_b(k);
        load_a(k);
      }
      step();
    }
    // a wait that gave up: the copies in flight land before the CTA's memory is given back
    if (!ok)
      for (int i = k - k0 > NS ? k - k0 - NS : 0; i < k - k0; ++i) mbar_wait_warp<false>(full + 8 * (i % NS), (uint32_t)(i / NS) & 1u, p.status, W_GEMM_DRAIN);
  } else if (warp == 1) {
    const uint32_t idesc = make_idesc_bf16(BM, p.n, 0, B_MN);
    constexpr uint32_t b_step = B_MN ? 2048u : 32u;
    const uint64_t desc_a = make_smem_desc_sw128(s0, 0, 1024), desc_b = make_smem_desc_sw128(s0 + 2u * p.a_bytes, B_MN ? 8192 : 0, 1024);
    const uint32_t wrap = (uint32_t)NS * stage_bytes;
    uint32_t at = 0, bar = 0, ph = 0, add = 0;
    bool ok = true;
    for (int k = k0; k < k1; ++k) {
      ok = mbar_wait_warp<false>(full + bar, ph, p.status, W_GEMM_FULL);
      if (!ok) break;
      tc_fence_after_sync();
      if (elect_one()) {
        const uint64_t ad = desc_at(desc_a, at), bd = desc_at(desc_b, at);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          umma_bf16(tmem, desc_at(ad, (j & 3) * 32 + (j >> 2) * p.a_bytes), desc_at(bd, (j & 3) * b_step + (j >> 2) * p.b_bytes), idesc, j ? 1u : add);
        umma_commit(empty + bar);
      }
      add = 1;
      at += stage_bytes;
      bar += 8;
      if (at == wrap) { at = 0; bar = 0; ph ^= 1u; }
    }
    if (ok && elect_one()) umma_commit(acc_full);
  } else {
    // the sums into shared memory, over the stages that the products have read; rows 16 bytes apart in their banks
    const int grp = (warp - 2) >> 2, q = warp & 3, row = q * 32 + lane;
    __all_sync(0xffffffffu, mbar_wait(acc_full, 0, p.status, W_GEMM_EPI));
    tc_fence_after_sync();
    if (q * 32 < (int)(p.a_bytes >> 7))  // rows that were staged
      for (int c = grp * 32; c < p.n; c += 32 * EPI_GROUPS) {
        uint32_t f[32];
        tmem_ld_32x32b_x32(tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)c, f);
        tmem_ld_wait();
        if (row < (int)(p.a_bytes >> 7)) {
          const uint32_t dst = s0 + (uint32_t)(row * (p.n + 4) + c) * 4u;
#pragma unroll
          for (int v = 0; v < 8; ++v) st_shared_v4(dst + 16u * v, f[4 * v], f[4 * v + 1], f[4 * v + 2], f[4 * v + 3]);
        }
      }
  }
  tc_fence_before_sync();
  __syncwarp();
  cluster_sync_all();  // every CTA's sums are there (and every warp of this CTA is)

  const int per_row = p.n / 4, rows = min(BM, p.M - m0);
  for (int i = (int)rank * G_THREADS + tid; i < rows * per_row; i += p.c * G_THREADS) {
    const int r = i / per_row, col = (i - r * per_row) * 4;
    if (n0 + col >= p.N) continue;  // N is a multiple of eight
    const size_t at = (size_t)(m0 + r) * p.N + n0 + col;
    const uint32_t src = s0 + (uint32_t)(r * (p.n + 4) + col) * 4u;
    float4 v[SPLIT_MAX];
#pragma unroll
    for (int k = 0; k < SPLIT_MAX; ++k)
      if (k < p.c) v[k] = ld_cluster_f4(map_to_cta(src, (uint32_t)k));
    float4 t = v[0];
#pragma unroll
    for (int k = 1; k < SPLIT_MAX; ++k)
      if (k < p.c) { t.x += v[k].x; t.y += v[k].y; t.z += v[k].z; t.w += v[k].w; }
    if (p.addend) {
      const uint2 a = *reinterpret_cast<const uint2*>(p.addend + at);
      t.x += __uint_as_float(a.x << 16);
      t.y += __uint_as_float(a.x & 0xffff0000u);
      t.z += __uint_as_float(a.y << 16);
      t.w += __uint_as_float(a.y & 0xffff0000u);
    }
    if (p.f32_out) {
      *reinterpret_cast<float4*>((float*)p.D + at) = t;
    } else {
      __nv_bfloat162 lo = __floats2bfloat162_rn(t.x, t.y), hi = __floats2bfloat162_rn(t.z, t.w);
      *reinterpret_cast<uint2*>((bf16*)p.D + at) = make_uint2(*reinterpret_cast<uint32_t*>(&lo), *reinterpret_cast<uint32_t*>(&hi));
    }
  }
  cluster_sync_all();  // the sums outlive their readers
  if (warp == 1) {
    __syncwarp();
    tc_fence_after_sync();
    tmem_dealloc(tmem, p.cols);
  }
}

// How a problem is cut: the cut with the least time by this model, in microseconds, of which the constants were measured (with
// both forms, every tile width and all three operand orders, 74 pairs busy). A k-block takes 0.155 at least, 1.53 ns a column
// of the tile for the products, and its bytes at 115 KB out of L2 (rows that do not begin on 128 bytes take half as much again),
// or, where B is read only once, 40 KB out of memory. An epilogue takes 0.7, a pair's 1.0, and 7 ns a column, in fp32 10, and runs beside
// the next tile's products. Sharing the rest of the tiles takes a launch and the slots' way to memory and back, some 3.5 MB.
// Against the best cut found by trying all: within 5 % for 13 of 16 problems of 8 to 8192 rows; for the weight gradients of 18
// shapes and 1 to 2048 tokens, in both types, 2 % behind on the mean (8 with half the time for a tile's beginning and half as
// much again a column: narrow tiles then look too good).
//
// A tile a cluster of c takes 3.6 to begin and end, 0.16 c and 0.195 ns an element of the tile to bring the parts together, and
// a step of 128 along the reduction 0.28 at least, 2.8 ns a column, its bytes at 160 KB and 16.5 TB/s on all of them; where B is
// read only once, at 65 KB and 6.3 TB/s out of memory. (On this scale the other cuts begin with 1.5.) Measured with weights out
// of memory, sharing units and a second launch against clusters: 24 x 4096 x 11008 22.6 and 18.4 us, 5 x 896 x 4864 10.3 and 6.4,
// 128 x 896 x 4864 11.5 and 8.0, 333 x 896 x 9728 (B across) 17.4 and 14.3, 512 x 896 x 4864 13.9 and 11.2, 600 x 2048 x 5632
// 18.7 and 18.4, 1024 x 896 x 4864 15.0 and 15.2. Whole device only: in a partition clusters may not find their SMs.
struct GemmPlan {
  bool pair;
  int n, m_units, n_tiles, tiles, units, rounds, rest, sharers;
  int split;  // CTAs of a cluster that share a tile each, or 0
};
// Clusters of c CTAs of split_gemm_kernel that the device holds at one time, as the driver counts them (0 if it does not); asked
// for once a device.
template <bool B_MN>
int clusters_that_fit(int c) {
  static std::atomic<int> known[16][SPLIT_MAX + 1];  // one more than the count
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 16) return 0;
  const int k = known[dev][c].load(std::memory_order_relaxed);
  if (k) return k - 1;
  constexpr int smem = 232448;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)c);
  cfg.blockDim = dim3(G_THREADS);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)c;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaFuncSetAttribute(split_gemm_kernel<B_MN>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&n, split_gemm_kernel<B_MN>, &cfg) != cudaSuccess || n < 0) {
    cudaGetLastError();
    n = 0;
  }
  known[dev][c].store(n + 1, std::memory_order_relaxed);
  return n;
}
int a_pitch(const GemmProblem& q) { return q.a_pitch ? q.a_pitch : q.a_mn ? q.M : q.K; }
int b_pitch(const GemmProblem& q) { return q.b_pitch ? q.b_pitch : q.b_mn ? q.N : q.K; }
size_t plan_bytes(const GemmPlan& g) { return g.rest ? (size_t)2 * g.sharers * (g.pair ? 2 * BM : BM) * g.n * sizeof(float) : 0; }
// Plans that need more than `room` bytes of slots are left out; one without any is always there.
GemmPlan plan_gemm(const GemmProblem& q, size_t room) {
  constexpr int LEAST = 4;  // k-blocks of a share: less is not worth a slot
  const int sms = sm_count() < JOIN_MAX ? sm_count() : JOIN_MAX, kb = ceil_div(q.K, 64);
  const int a_rows = !q.a_mn && q.M < BM ? (q.M + 7) / 8 * 8 : BM;
  const bool a_odd = a_pitch(q) % 64 != 0, b_odd = b_pitch(q) % 64 != 0;
  GemmPlan best = {};
  double best_cost = 1e30;
  for (int c = 1; c <= (q.a_mn || sm_limit() != 0 ? 0 : SPLIT_MAX); ++c) {
    const int fit = q.b_mn ? clusters_that_fit<true>(c) : clusters_that_fit<false>(c), steps = ceil_div(ceil_div(q.K, 128), c);
    if (steps * (c - 1) >= ceil_div(q.K, 128)) continue;  // a CTA without a step
    for (int n = 32; n <= 256; n += 32) {
      if (n > 32 && n - 32 >= q.N) continue;  // wider than the matrix
      const int m_units = ceil_div(q.M, BM), n_tiles = ceil_div(q.N, n);
      if ((long long)m_units * n_tiles > fit) continue;
      const double all = (double)m_units * n_tiles * c;
      const double a_bytes = 256.0 * a_rows * (a_odd ? 1.5 : 1.0);
      const double b_bytes = 2.0 * (q.b_mn ? 8192.0 * ceil_div(n, 64) : 128.0 * n) * (b_odd ? 1.5 : 1.0);
      double t = 0.28;
      auto at_least = [&](double v) { t = v > t ? v : t; };
      at_least(0.0028 * n);
      at_least((a_bytes + b_bytes) / 160e3);
      at_least((a_bytes + b_bytes) * all / 16.5e6);
      if (m_units == 1) {
        at_least(b_bytes / 65e3);
        at_least(b_bytes * all / 6.3e6);
      }
      const double cost = 3.6 - 1.5 + 0.16 * c + 0.195e-3 * a_rows * n + steps * t;
      if (cost < best_cost) {
        best_cost = cost;
        best = {};
        best.n = n;
        best.m_units = m_units;
        best.n_tiles = n_tiles;
        best.tiles = best.units = m_units * n_tiles;
        best.split = c;
      }
    }
  }
  for (int pair = 0; pair <= (sms >= 2 && q.M > BM ? 1 : 0); ++pair) {
    for (int n = 32; n <= 256; n += 32) {
      if (n > 32 && n - 32 >= q.N) continue;  // wider than the matrix
      GemmPlan g = {};
      g.pair = pair != 0;
      g.n = n;
      g.m_units = ceil_div(q.M, pair ? 2 * BM : BM);
      g.n_tiles = ceil_div(q.N, n);
      g.tiles = g.m_units * g.n_tiles;
      const int all = pair ? sms / 2 : sms, nc = pair ? n / 2 : n;
      const double a_bytes = 128.0 * a_rows * (a_odd ? 1.5 : 1.0);
      const double b_bytes = (q.b_mn ? 8192.0 * ceil_div(nc, 64) : 128.0 * nc) * (b_odd ? 1.5 : 1.0);
      double t_kb = 0.155;
      auto at_least = [&](double t) { t_kb = t > t_kb ? t : t_kb; };
      at_least(0.00153 * n);
      at_least((a_bytes + b_bytes) / 115e3);
      if (g.m_units == 1) at_least(b_bytes / 40e3 + 0.03);
      const double t_epi = (pair ? 1.0 : 0.7) + (q.out_dtype == SRT_F32 ? 0.010 : 0.007) * n;
      for (int share = 0; share < 2; ++share) {
        const long long most = (long long)g.tiles * kb / LEAST;  // units that have something to do
        g.units = share && most > g.tiles ? (most < all ? (int)most : all) : (g.tiles < all ? g.tiles : all);
        g.rounds = g.tiles / g.units;
        g.rest = g.tiles - g.rounds * g.units;
        const long long work = (long long)g.rest * kb;
        g.sharers = work / LEAST < g.units ? (int)(work / LEAST) : g.units;
        if (!share || g.sharers <= g.rest) {
          g.rounds = ceil_div(g.tiles, g.units);
          g.rest = g.sharers = 0;
        }
        if (plan_bytes(g) > room) continue;
        double cost = g.rounds * (kb * t_kb > t_epi ? kb * t_kb : t_epi) + t_epi;
        if (g.rest > 0)
          cost += (double)g.rest * kb / g.sharers * t_kb + 5.0 + (g.sharers + g.rest) * (pair ? 2.0 : 1.0) * a_rows * n * 4.0 / 3.5e6;
        if (cost < best_cost) { best_cost = cost; best = g; }
      }
    }
  }
  return best;
}

// The tiles with more than one part, each with the units that have one: a border between two shares inside a tile makes it
// such a tile, and the first border inside stands for it.
int join_list(const GemmParams& p, JoinList& list) {
  const long long work = (long long)p.rest * p.k_blocks;
  int count = 0, last = -1;
  for (int u = 1; u < p.sharers; ++u) {
    const long long border = share_begin(work, u, p.sharers);
    const int t = (int)(border / p.k_blocks);
    if (border == (long long)t * p.k_blocks) continue;
    if (t == last) {
      list.t[count - 1].u1 = u;
      continue;
    }
    last = t;
    int m, n;
    tile_at(p, p.rounds * p.units + t, m, n);
    list.t[count++] = {m, n, u - 1, u};
  }
  return count;
}

template <bool PAIR, bool A_MN, bool B_MN>
int launch_gemm(GemmParams& p, const GemmPlan& g, const CUtensorMap (&tm)[4], cudaStream_t st) {
  constexpr size_t fixed = 1024 + EPI_GROUPS * SLAB_BYTES + (2 * G_MAX_STAGES + 4) * 8 + 16;
  p.stages = (int)((232448 - fixed) / p.stage_bytes);
  if (p.stages > G_MAX_STAGES) p.stages = G_MAX_STAGES;
  static SmemOptIn opt_in;
  SRT_CHECK_CUDA(opt_in.set(balanced_gemm_kernel<PAIR, A_MN, B_MN>, 232448));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(g.units * (PAIR ? 2 : 1)));
  cfg.blockDim = dim3(G_THREADS);
  cfg.dynamicSmemBytes = fixed + (size_t)p.stages * p.stage_bytes;
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
  SRT_CHECK_CUDA(cudaLaunchKernelEx(&cfg, balanced_gemm_kernel<PAIR, A_MN, B_MN>, p, tm[0], tm[1], tm[2], tm[3]));
  SRT_LAUNCH_CHECK();
  if (g.rest == 0) return SRT_OK;
  JoinList list;
  const int tiles = join_list(p, list);
  if (tiles == 0) return SRT_OK;  // every share ended with a tile
  const int rows = PAIR ? 2 * BM : BM, live = p.M < rows ? p.M : rows;
  const int block_rows = JOIN_THREADS / (g.n / 4);  // one item a thread
  SRT_CHECK_CUDA(launch_pdl(balanced_gemm_join_kernel, dim3(tiles, ceil_div(live, block_rows)), dim3(JOIN_THREADS), 0, st, p, list, rows, block_rows));
  SRT_LAUNCH_CHECK();
  return SRT_OK;
}

template <bool B_MN>
int launch_split(SplitParams& p, const CUtensorMap (&tm)[4], cudaStream_t st) {
  const size_t fixed = 1024 + BM * 128 - p.a_bytes + (2 * G_MAX_STAGES + 1) * 8 + 16, stage = 2 * (size_t)(p.a_bytes + p.b_bytes);
  p.stages = (int)((232448 - fixed) / stage);
  if (p.stages > G_MAX_STAGES) p.stages = G_MAX_STAGES;
  const size_t sums = (size_t)(p.a_bytes >> 7) * (p.n + 4) * 4;
  SRT_REQUIRE(p.stages >= 2 && sums <= p.stages * stage, "balanced_gemm: a tile of %d columns does not fit a cluster", p.n);
  static SmemOptIn opt_in;
  SRT_CHECK_CUDA(opt_in.set(split_gemm_kernel<B_MN>, 232448));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.m_units * ceil_div(p.N, p.n) * p.c));
  cfg.blockDim = dim3(G_THREADS);
  cfg.dynamicSmemBytes = fixed + (size_t)p.stages * stage;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = (pdl_big_kernels() && (pdl_classes() & PDL_GEMM) != 0) ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)p.c;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  SRT_CHECK_CUDA(cudaLaunchKernelEx(&cfg, split_gemm_kernel<B_MN>, p, tm[0], tm[1]));
  SRT_LAUNCH_CHECK();
  return SRT_OK;
}

}  // namespace

size_t balanced_gemm_scratch_bytes(const GemmProblem& q) { return q.M > 0 && q.N > 0 && q.K > 0 ? plan_bytes(plan_gemm(q, SIZE_MAX)) : 0; }

int balanced_gemm(const GemmProblem& q, const void* A, const void* B, const void* addend, void* D, void* scratch, size_t scratch_bytes,
                  bool b_early, cudaStream_t st) {
  SRT_REQUIRE(q.M > 0 && q.N > 0 && q.K > 0 && (q.b_mn || !q.a_mn) && a_pitch(q) >= (q.a_mn ? q.M : q.K) && b_pitch(q) >= (q.b_mn ? q.N : q.K),
              "balanced_gemm: empty problem or an operand order that has no kernel");
  const GemmPlan g = plan_gemm(q, scratch && ((uintptr_t)scratch & 15) == 0 ? scratch_bytes : 0);
  GemmParams p = {};
  p.M = q.M;
  p.N = q.N;
  p.k_blocks = ceil_div(q.K, 64);
  p.n = g.n;
  p.m_units = g.m_units;
  p.n_tiles = g.n_tiles;
  p.band = 8;
  p.tiles = g.tiles;
  p.units = g.units;
  p.rounds = g.rounds;
  p.rest = g.rest;
  p.sharers = g.sharers;
  p.cols = 64;
  while (p.cols < 2 * g.n) p.cols *= 2;
  const int nc = g.pair ? g.n / 2 : g.n;
  const int a_rows = !q.a_mn && q.M < BM ? (q.M + 7) / 8 * 8 : BM;
  const int b_bytes = q.b_mn ? ceil_div(nc, 64) * 8192 : nc * 128;
  p.a_bytes = (uint32_t)a_rows * 128;
  p.load_bytes = p.a_bytes + (uint32_t)b_bytes;
  p.stage_bytes = (int)p.load_bytes;  // multiples of 1024: eight rows of 128 bytes
  p.f32_out = q.out_dtype == SRT_F32;
  p.b_early = b_early;
  p.addend = (const bf16*)addend;
  p.D = D;
  p.slots = (const float*)scratch;
  p.status = tc_status_device_ptr();
  SRT_REQUIRE(p.status != nullptr, "tcgen05 status word unavailable");
  CUtensorMap tm[4];
  int rc;
  if ((rc = q.a_mn ? tmap_rows(&tm[0], A, q.K, q.M, a_pitch(q), 2, 64, 64) : tmap_rows(&tm[0], A, q.M, q.K, a_pitch(q), 2, 64, a_rows)) ||
      (rc = q.b_mn ? tmap_rows(&tm[1], B, q.K, q.N, b_pitch(q), 2, 64, 64) : tmap_rows(&tm[1], B, q.N, q.K, b_pitch(q), 2, 64, nc)) ||
      (rc = tmap_rows(&tm[2], D, q.M, q.N, q.N, p.f32_out ? 4 : 2, p.f32_out ? 16 : 32, a_rows)))
    return rc;
  tm[3] = tm[2];
  if (g.split) {
    SplitParams s = {};
    s.M = q.M;
    s.N = q.N;
    s.n = g.n;
    s.c = g.split;
    s.m_units = g.m_units;
    s.steps = ceil_div(q.K, 128);
    s.cols = 32;
    while (s.cols < g.n) s.cols *= 2;
    s.a_bytes = p.a_bytes;
    s.b_bytes = (uint32_t)b_bytes;
    s.f32_out = p.f32_out;
    s.b_early = b_early;
    s.addend = p.addend;
    s.D = D;
    s.status = p.status;
    return q.b_mn ? launch_split<true>(s, tm, st) : launch_split<false>(s, tm, st);
  }
  if (g.rest && (rc = tmap_rows(&tm[3], scratch, (uint64_t)2 * g.sharers * (g.pair ? 2 * BM : BM), g.n, g.n, 4, 16, a_rows))) return rc;
  if (q.a_mn) return g.pair ? launch_gemm<true, true, true>(p, g, tm, st) : launch_gemm<false, true, true>(p, g, tm, st);
  if (q.b_mn) return g.pair ? launch_gemm<true, false, true>(p, g, tm, st) : launch_gemm<false, false, true>(p, g, tm, st);
  return g.pair ? launch_gemm<true, false, false>(p, g, tm, st) : launch_gemm<false, false, false>(p, g, tm, st);
}

}  // namespace srt
