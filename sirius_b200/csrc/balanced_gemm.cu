// Products whose work is dealt evenly to all SMs: D = A B (+ addend) with either operand stored along or across the reduction.
//
// The output is cut into tiles; a unit (a CTA, or a CTA pair with cta_group::2) takes whole tiles while there are enough for
// all, and what is left over, fewer tiles than units, is cut along the reduction into as many equal ranges as there are units.
// A unit that has only a part of a tile's reduction leaves fp32 sums in a slot of its own, and a second, small launch adds the
// slots of every such tile in the order of the reduction. So 152 tiles on 74 pairs take 2.05 rounds and not three, a few rows
// against a long reduction occupy the device, no CTA waits for another, and the sums have a fixed order.
//
// Warps as in the gated kernels: 0 TMA, 1 MMA, 2-9 two epilogue groups that take the 32-column slabs of a tile in turn. The
// accumulator is double-buffered in tensor memory, so the epilogue of a tile runs beside the products of the next.
#include <cuda.h>

#include "balanced_gemm.cuh"
#include "ptx.cuh"

namespace srt {

int* tc_status_device_ptr();  // igemm_tcgen05.cu
int tmap_rows(CUtensorMap* tm, const void* base, uint64_t rows, uint64_t cols, uint64_t pitch, int elem_bytes, uint32_t box_cols, uint32_t box_rows);

namespace {

using namespace ptx;
using bf16 = __nv_bfloat16;

constexpr int BM = 128;
constexpr int G_THREADS = 320;
constexpr int G_MAX_STAGES = 8;
constexpr int A_BYTES = BM * 128;
constexpr int SLAB_BYTES = BM * 128;  // 128 rows x 32 fp32 (or 32 bf16)
enum { W_GEMM_LOAD = 0x41, W_GEMM_FULL = 0x42, W_GEMM_ACC = 0x43, W_GEMM_EPI = 0x44, W_GEMM_DRAIN = 0x45 };

struct GemmParams {
  int M, N, k_blocks, n;       // n: columns of a tile, a multiple of 32
  int m_units, n_tiles, band;  // tiles are walked in bands of `band` columns of tiles
  int tiles, units, rounds;    // a unit has up to `rounds` whole tiles ...
  int rest, sharers;           // ... and the first `sharers` units share the `rest` tiles beyond those
  int cols;                    // tensor-memory columns
  int stages, stage_bytes;
  uint32_t load_bytes;         // of one CTA a k-block
  int f32_out;
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
__device__ __forceinline__ void tile_at(const GemmParams& p, int t, int& m, int& n) {
  const int b = t / (p.band * p.m_units), first = b * p.band;
  const int size = min(p.band, p.n_tiles - first), r = t - first * p.m_units;
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
  uint64_t* bars = (uint64_t*)(sOut + 2 * SLAB_BYTES);
  const uint32_t full = smem_u32(bars), empty = full + 8 * G_MAX_STAGES, acc_full = empty + 8 * G_MAX_STAGES, acc_empty = acc_full + 16;
  uint32_t* tmem_ptr = (uint32_t*)(bars + 2 * G_MAX_STAGES + 4);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = PAIR ? cluster_ctarank() : 0u;
  const int unit = (int)blockIdx.x / NCTA;
  const int n_cta = p.n / NCTA;  // columns of B that this CTA stages
  const uint32_t s0 = smem_u32(base);

  if (tid == 0) {
    for (int s = 0; s < NS; ++s) { mbar_init(full + 8 * s, 1); mbar_init(empty + 8 * s, 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(acc_full + 8 * b, 1); mbar_init(acc_empty + 8 * b, 8 * NCTA); }
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
  const uint32_t tmem = *tmem_ptr;
  pdl_enter();

  if (warp == 0) {
    if (lane == 0) {
      int it = 0, s = 0;
      uint32_t ph = 1;
      bool ok = true;
      Walk w = walk_begin(p, unit);
      Piece o;
      while (ok && walk_next(p, unit, w, o)) {
        int m, n;
        tile_at(p, o.tile, m, n);
        const int m0 = (m * NCTA + (int)rank) * BM, n0 = n * p.n + (int)rank * n_cta;
        for (int kb = o.k0; kb < o.k1; ++kb) {
          ok = mbar_wait(empty + 8 * s, ph, p.status, W_GEMM_LOAD);
          if (!ok) break;
          if (rank == 0) mbar_arrive_expect_tx(full + 8 * s, p.load_bytes * NCTA);
          const uint32_t bar = PAIR ? map_to_cta(full + 8 * s, 0u) : full + 8 * s;
          const uint32_t a = s0 + (uint32_t)s * p.stage_bytes, b = a + A_BYTES;
          auto load = [&](uint32_t dst, const CUtensorMap* tm, int x, int y) {
            if (PAIR) tma_load_2d_pair(dst, tm, bar, x, y);
            else tma_load_2d(dst, tm, bar, x, y);
          };
          if (A_MN) {
            load(a, &ta, m0, kb * 64);
            load(a + 8192u, &ta, m0 + 64, kb * 64);
          } else {
            load(a, &ta, kb * 64, m0);
          }
          if (B_MN) {
            for (int c = 0; c < n_cta; c += 64) load(b + (uint32_t)c * 128u, &tb, n0 + c, kb * 64);
          } else {
            load(b, &tb, kb * 64, n0);
          }
          ++it;
          if (++s == NS) { s = 0; ph ^= 1u; }
        }
      }
      // a wait that gave up: the copies in flight land before the CTA's memory is given back
      if (!ok && rank == 0)
        for (int k = it > NS ? it - NS : 0; k < it; ++k) mbar_wait(full + 8 * (k % NS), (uint32_t)(k / NS) & 1u, p.status, W_GEMM_DRAIN);
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      const uint32_t idesc = make_idesc_bf16(BM * NCTA, p.n, A_MN, B_MN);
      int s = 0, i = 0;
      uint32_t ph = 0;
      bool ok = true;
      auto wait = [&](uint32_t bar, uint32_t parity, int code) {
        ok = ok && (PAIR ? mbar_wait_cluster(bar, parity, p.status, code) : mbar_wait(bar, parity, p.status, code));
        if (ok) tc_fence_after_sync();
        return ok;
      };
      Walk w = walk_begin(p, unit);
      Piece o;
      for (; ok && walk_next(p, unit, w, o); ++i) {
        const uint32_t b2 = (uint32_t)i & 1u, acc = tmem + b2 * (uint32_t)(p.cols / 2);
        if (!wait(acc_empty + 8 * b2, ((uint32_t)(i >> 1) & 1u) ^ 1u, W_GEMM_ACC)) break;
        for (int kb = o.k0; kb < o.k1; ++kb) {
          if (!wait(full + 8 * s, ph, W_GEMM_FULL)) break;
          const uint32_t a = s0 + (uint32_t)s * p.stage_bytes, b = a + A_BYTES;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint64_t ad = A_MN ? make_smem_desc_sw128(a + k * 2048, 8192, 1024) : make_smem_desc_sw128(a + k * 32, 0, 1024);
            const uint64_t bd = B_MN ? make_smem_desc_sw128(b + k * 2048, 8192, 1024) : make_smem_desc_sw128(b + k * 32, 0, 1024);
            const uint32_t add = (kb != o.k0 || k != 0) ? 1u : 0u;
            if (PAIR) umma_bf16_pair(acc, ad, bd, idesc, add);
            else umma_bf16(acc, ad, bd, idesc, add);
          }
          if (PAIR) umma_commit_pair(empty + 8 * s, (uint16_t)3);
          else umma_commit(empty + 8 * s);
          if (++s == NS) { s = 0; ph ^= 1u; }
        }
        if (!ok) break;
        if (PAIR) umma_commit_pair(acc_full + 8 * b2, (uint16_t)3);
        else umma_commit(acc_full + 8 * b2);
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
      for (int c = grp * 32; c < p.n; c += 64) {
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
          fetch(c + 64);
        }
        if (issuer) bulk_wait_group_read<0>();  // the store before has read the slab
        named_bar_sync(1 + grp, 128);
        if (wide) {
#pragma unroll
          for (int v = 0; v < 8; ++v)
            st_shared_v4(slab + (uint32_t)row * 128u + (uint32_t)((v ^ (row & 7)) << 4), f[v * 4], f[v * 4 + 1], f[v * 4 + 2], f[v * 4 + 3]);
        } else {
          uint32_t h[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            __nv_bfloat162 v = __floats2bfloat162_rn(__uint_as_float(f[2 * e]), __uint_as_float(f[2 * e + 1]));
            h[e] = *reinterpret_cast<uint32_t*>(&v);
          }
#pragma unroll
          for (int v = 0; v < 4; ++v)  // 64-byte rows, 64-byte swizzle
            st_shared_v4(slab + (uint32_t)row * 64u + (uint32_t)((v ^ ((row >> 1) & 3)) << 4), h[v * 4], h[v * 4 + 1], h[v * 4 + 2], h[v * 4 + 3]);
        }
        fence_proxy_async_smem();
        named_bar_sync(1 + grp, 128);
        if (issuer) {
          if (whole) tma_store_2d(&td, slab, n0 + c, m0);
          else tma_store_2d(&tslot, slab, c, (o.slot * NCTA + (int)rank) * BM);
          bulk_commit_group();
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

// The tiles whose reduction was shared: block (u, y) looks at the border between the shares of units u and u + 1; the first
// border inside a tile stands for the tile. Sixteen rows a block.
constexpr int JOIN_ROWS = 16, JOIN_THREADS = 256;
__global__ void __launch_bounds__(JOIN_THREADS)
balanced_gemm_join_kernel(const GemmParams p, int unit_rows) {
  pdl_enter();
  const long long work = (long long)p.rest * p.k_blocks;
  const int u = (int)blockIdx.x + 1;
  const long long border = share_begin(work, u, p.sharers);
  const int t = (int)(border / p.k_blocks);
  const long long first = (long long)t * p.k_blocks;
  if (border == first || border >= work || share_begin(work, u - 1, p.sharers) > first) return;
  const int u0 = u - 1, u1 = (int)(((first + p.k_blocks) * p.sharers - 1) / work);  // units with a part of the tile
  int m, n;
  tile_at(p, p.rounds * p.units + t, m, n);
  const int per_row = p.n / 8;
  for (int i = threadIdx.x; i < JOIN_ROWS * per_row; i += JOIN_THREADS) {
    const int r = (int)blockIdx.y * JOIN_ROWS + i / per_row, c = (i % per_row) * 8;
    const int row = m * unit_rows + r, col = n * p.n + c;
    if (row >= p.M || col >= p.N) continue;  // N is a multiple of eight
    float s[8];
    const float* f = p.slots + ((size_t)(2 * u0 + 1) * unit_rows + r) * p.n + c;
    *reinterpret_cast<float4*>(s) = *reinterpret_cast<const float4*>(f);
    *reinterpret_cast<float4*>(s + 4) = *reinterpret_cast<const float4*>(f + 4);
#pragma unroll 4
    for (int k = u0 + 1; k <= u1; ++k) {
      const float* g = p.slots + ((size_t)(2 * k) * unit_rows + r) * p.n + c;
      const float4 a = *reinterpret_cast<const float4*>(g), b = *reinterpret_cast<const float4*>(g + 4);
      s[0] += a.x; s[1] += a.y; s[2] += a.z; s[3] += a.w;
      s[4] += b.x; s[5] += b.y; s[6] += b.z; s[7] += b.w;
    }
    const size_t at = (size_t)row * p.N + col;
    if (p.addend) {
      Vec16<bf16> v;
      float a[8];
      v.load(p.addend + at);
      v.unpack(a);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] += a[e];
    }
    if (p.f32_out) {
      *reinterpret_cast<float4*>((float*)p.D + at) = *reinterpret_cast<float4*>(s);
      *reinterpret_cast<float4*>((float*)p.D + at + 4) = *reinterpret_cast<float4*>(s + 4);
    } else {
      Vec16<bf16> v;
      v.pack(s);
      v.store((bf16*)p.D + at);
    }
  }
}

// How a problem is cut. Clocks a k-block of a unit: its products (a 128 x n x 64 product takes 2 n clocks an SM) or its
// operand stream out of L2 (about 50 bytes a clock and SM), whichever is longer; an epilogue takes about 12 clocks a column,
// twice that in fp32.
struct GemmPlan {
  bool pair;
  int n, m_units, n_tiles, tiles, units, rounds, rest, sharers;
};
size_t plan_bytes(const GemmPlan& g) { return g.rest ? (size_t)2 * g.sharers * (g.pair ? 2 * BM : BM) * g.n * sizeof(float) : 0; }
// Plans that need more than `room` bytes of slots are left out; one without any is always there.
GemmPlan plan_gemm(const GemmProblem& q, size_t room) {
  constexpr int LEAST = 4;  // k-blocks of a share: less is not worth a slot
  const int sms = sm_count(), kb = ceil_div(q.K, 64);
  const int a_rows = !q.a_mn && q.M < BM ? (q.M + 7) / 8 * 8 : BM;
  GemmPlan best = {};
  double best_cost = 1e30;
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
      const double bytes = 128.0 * a_rows + (q.b_mn ? 8192.0 * ceil_div(nc, 64) : 128.0 * nc);
      const double kclk = bytes / 50 > 2.0 * n ? bytes / 50 : 2.0 * n;
      const double eclk = 12.0 * n * (q.out_dtype == SRT_F32 ? 2 : 1);
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
        double cost = g.rounds * (kb * kclk > eclk ? kb * kclk : eclk) + eclk;
        if (g.rest > 0) cost += (double)g.rest * kb / g.sharers * kclk + 24.0 * n + 4000;  // a slot, and the joining launch
        if (cost < best_cost) { best_cost = cost; best = g; }
      }
    }
  }
  return best;
}

template <bool PAIR, bool A_MN, bool B_MN>
int launch_gemm(GemmParams& p, const GemmPlan& g, const CUtensorMap (&tm)[4], cudaStream_t st) {
  constexpr size_t fixed = 1024 + 2 * SLAB_BYTES + (2 * G_MAX_STAGES + 4) * 8 + 16;
  p.stages = (int)((232448 - fixed) / p.stage_bytes);
  if (p.stages > G_MAX_STAGES) p.stages = G_MAX_STAGES;
  SRT_CHECK_CUDA(cudaFuncSetAttribute(balanced_gemm_kernel<PAIR, A_MN, B_MN>, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448));
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
  const int rows = PAIR ? 2 * BM : BM, live = p.M < rows ? p.M : rows;
  SRT_CHECK_CUDA(launch_pdl(balanced_gemm_join_kernel, dim3(g.sharers - 1, ceil_div(live, JOIN_ROWS)), dim3(JOIN_THREADS), 0, st, p, rows));
  SRT_LAUNCH_CHECK();
  return SRT_OK;
}

}  // namespace

size_t balanced_gemm_scratch_bytes(const GemmProblem& q) { return q.M > 0 && q.N > 0 && q.K > 0 ? plan_bytes(plan_gemm(q, SIZE_MAX)) : 0; }

int balanced_gemm(const GemmProblem& q, const void* A, const void* B, const void* addend, void* D, void* scratch, size_t scratch_bytes,
                  cudaStream_t st) {
  SRT_REQUIRE(q.M > 0 && q.N > 0 && q.K > 0 && (q.b_mn || !q.a_mn), "balanced_gemm: empty problem or an operand order that has no kernel");
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
  p.load_bytes = (uint32_t)(q.a_mn ? A_BYTES : a_rows * 128) + (uint32_t)b_bytes;
  p.stage_bytes = A_BYTES + (b_bytes + 1023) / 1024 * 1024;
  p.f32_out = q.out_dtype == SRT_F32;
  p.addend = (const bf16*)addend;
  p.D = D;
  p.slots = (const float*)scratch;
  p.status = tc_status_device_ptr();
  SRT_REQUIRE(p.status != nullptr, "tcgen05 status word unavailable");
  CUtensorMap tm[4];
  int rc;
  if ((rc = q.a_mn ? tmap_rows(&tm[0], A, q.K, q.M, q.M, 2, 64, 64) : tmap_rows(&tm[0], A, q.M, q.K, q.K, 2, 64, a_rows)) ||
      (rc = q.b_mn ? tmap_rows(&tm[1], B, q.K, q.N, q.N, 2, 64, 64) : tmap_rows(&tm[1], B, q.N, q.K, q.K, 2, 64, nc)) ||
      (rc = tmap_rows(&tm[2], D, q.M, q.N, q.N, p.f32_out ? 4 : 2, 32, BM)))
    return rc;
  tm[3] = tm[2];
  if (g.rest && (rc = tmap_rows(&tm[3], scratch, (uint64_t)2 * g.sharers * (g.pair ? 2 * BM : BM), g.n, g.n, 4, 32, BM))) return rc;
  if (q.a_mn) return g.pair ? launch_gemm<true, true, true>(p, g, tm, st) : launch_gemm<false, true, true>(p, g, tm, st);
  if (q.b_mn) return g.pair ? launch_gemm<true, false, true>(p, g, tm, st) : launch_gemm<false, false, true>(p, g, tm, st);
  return g.pair ? launch_gemm<true, false, false>(p, g, tm, st) : launch_gemm<false, false, false>(p, g, tm, st);
}

}  // namespace srt
