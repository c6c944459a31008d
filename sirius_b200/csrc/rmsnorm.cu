// Root-mean-square norm with the residual's addition, its 8-bit output, its backward pass, and rows quantised as they are.
//
//   forward    h = x + residual,  rstd = 1 / sqrt(mean(h^2) + eps),  y = gamma h rstd
//   8 bits     scale = max(max |y| / 448, 2^-126) of a row, q = e4m3(y (1 / scale)): a product with the rounded reciprocal, so a
//              quotient within 2^-23 of itself of a rounding border may go to the other neighbour
//   backward   xhat = h rstd,  g = gamma dy:  dx = dh + rstd (g - xhat mean(g xhat)),  dgamma = sum over rows of dy xhat
//
// bf16 or fp32 rows, fp32 parameters and statistics, the root by rsqrtf. y comes from the fp32 sum, not from the rounded h that
// is stored: one rounding on the way to y instead of two.
//
// All of it is bound by memory: a row is read once, sits in the registers of one to sixteen warps (16 elements a lane, 32 in
// the longest rows) until its statistics are known, and is written once; the next row's loads are in flight meanwhile.
// Blocks walk over rows, so gamma is loaded once a block and, in backward, dgamma adds up in registers over the rows of a
// warp; blocks leave one partial row each, which a second launch adds in a fixed order. No atomics: a call repeats bit for bit.
#include <cuda_fp8.h>

#include "common.cuh"
#include "ops.cuh"

namespace srt {
namespace {

using bf16 = __nv_bfloat16;
constexpr int RN_MAX_BLOCKS = 160;   // partial rows of dgamma: one block an SM
constexpr int RN_MAX_ROW_BYTES = 32768;
constexpr float E4M3_MAX = 448.f;

// The larger of two values, NaN if either is (fmaxf would drop it, and with it the row's only sign of trouble).
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
template <bool MAX>
__device__ __forceinline__ float warp_all(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float w = __shfl_xor_sync(0xffffffffu, v, o);
    v = MAX ? max_nan(v, w) : v + w;
  }
  return v;
}
// Over the W warps of a row group, which meet on a barrier of their own; `red` has a slot per warp of the block, and `turn`
// alternates its halves so that one barrier a reduction is enough.
template <bool MAX>
__device__ __forceinline__ float group_all(float v, int W, float (*red)[32], int& turn) {
  v = warp_all<MAX>(v);
  if (W == 1) return v;
  const int warp = threadIdx.x >> 5, first = warp & ~(W - 1);
  if ((threadIdx.x & 31) == 0) red[turn][warp] = v;
  asm volatile("bar.sync %0, %1;" ::"r"(1 + first / W), "r"(W * 32) : "memory");
  v = red[turn][first];
  for (int w = 1; w < W; ++w) v = MAX ? max_nan(v, red[turn][first + w]) : v + red[turn][first + w];
  turn ^= 1;
  return v;
}
__device__ __forceinline__ uint32_t four_e4m3(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | hi << 16;
}

template <typename V>
__device__ __forceinline__ void clear(V& v) { v.raw = {}; }

struct RowShape {
  int64_t rows;
  int C, W;     // W warps a row, a power of two
  float inv_c;  // 1 / C
};

// NORM false: y = x, only quantised. OUT8: q and scale instead of y.
template <typename T, int NV, bool NORM, bool OUT8>
__global__ void __maxnreg__((NV * Vec16<T>::N > 16) ? 128 : 80)
rmsnorm_fwd_kernel(const RowShape s, const T* x, const T* residual, const float* __restrict__ gamma, T* h_out, T* __restrict__ y,
                   uint8_t* __restrict__ q, float* __restrict__ scale, float* __restrict__ rstd, float eps) {
  constexpr int V = Vec16<T>::N;
  constexpr bool AHEAD = NV * V <= 16;  // the next row's vectors beside the current one's
  __shared__ float red[2][32];
  pdl_enter();
  const int W = s.W, groups = (int)(blockDim.x >> 5) / W, grp = (int)(threadIdx.x >> 5) / W;
  const int lane = (int)threadIdx.x - grp * W * 32, nv = s.C / V;
  const int64_t step = (int64_t)gridDim.x * groups;
  int turn = 0;
  float gm[NORM ? NV : 1][V];
  if constexpr (NORM) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = lane + i * W * 32;
#pragma unroll
      for (int e = 0; e < V; ++e) gm[i][e] = v < nv ? gamma[v * V + e] : 0.f;
    }
  }
  Vec16<T> xv[NV], rv[NV];
  auto fetch = [&](int64_t row, int64_t at) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      clear(xv[i]);
      clear(rv[i]);
      if (row < s.rows && lane + i * W * 32 < nv) {
        xv[i].load(x + at + i * W * 32 * V);
        if (residual) rv[i].load(residual + at + i * W * 32 * V);
      }
    }
  };
  int64_t row = (int64_t)blockIdx.x * groups + grp;
  int64_t at = row * s.C + lane * V;  // of this lane's first vector
  const int64_t step_at = step * s.C;
  if (AHEAD) fetch(row, at);
  for (; row < s.rows; row += step, at += step_at) {
    if (!AHEAD) fetch(row, at);
    float f[NV][V], sq = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float r[V];
      xv[i].unpack(f[i]);
      rv[i].unpack(r);
      if (residual) {
#pragma unroll
        for (int e = 0; e < V; ++e) f[i][e] += r[e];
      }
#pragma unroll
      for (int e = 0; e < V; ++e) sq = fmaf(f[i][e], f[i][e], sq);
    }
    if (AHEAD) fetch(row + step, at + step_at);
    if (h_out) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = lane + i * W * 32;
        if (v >= nv) continue;
        Vec16<T> o;
        o.pack(f[i]);
        o.store(h_out + at + i * W * 32 * V);
      }
    }
    if constexpr (NORM) {
      const float rs = rsqrtf(group_all<false>(sq, W, red, turn) * s.inv_c + eps);
      if (rstd && lane == 0) rstd[row] = rs;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) f[i][e] = f[i][e] * rs * gm[i][e];
    }
    if constexpr (OUT8) {
      float mx = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) mx = max_nan(mx, fabsf(f[i][e]));
      mx = group_all<true>(mx, W, red, turn);
      const float sc = max_nan(mx / E4M3_MAX, 1.17549435e-38f), inv = 1.f / sc;
      if (lane == 0) scale[row] = sc;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = lane + i * W * 32;
        if (v >= nv) continue;
        uint32_t w[V / 4];
#pragma unroll
        for (int e = 0; e < V; e += 4) w[e / 4] = four_e4m3(f[i][e] * inv, f[i][e + 1] * inv, f[i][e + 2] * inv, f[i][e + 3] * inv);
        if constexpr (V == 8) *reinterpret_cast<uint2*>(q + at + i * W * 32 * V) = make_uint2(w[0], w[1]);
        else *reinterpret_cast<uint32_t*>(q + at + i * W * 32 * V) = w[0];
      }
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = lane + i * W * 32;
        if (v >= nv) continue;
        Vec16<T> o;
        o.pack(f[i]);
        o.store(y + at + i * W * 32 * V);
      }
    }
  }
}

template <typename T, int NV>
__global__ void __launch_bounds__(512, 1)
rmsnorm_bwd_kernel(const RowShape s, const T* dy, const T* __restrict__ h, const float* __restrict__ gamma,
                   const float* __restrict__ rstd, const T* dh, T* dx, float* __restrict__ partial) {
  constexpr int V = Vec16<T>::N;
  constexpr bool AHEAD = NV * V <= 16;
  extern __shared__ float cols[];  // [row groups of the block][C]
  __shared__ float red[2][32];
  pdl_enter();
  const int W = s.W, groups = (int)(blockDim.x >> 5) / W, grp = (int)(threadIdx.x >> 5) / W;
  const int lane = (int)threadIdx.x - grp * W * 32, nv = s.C / V;
  const int64_t step = (int64_t)gridDim.x * groups;
  int turn = 0;
  float gm[NV][V], dg[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = lane + i * W * 32;
#pragma unroll
    for (int e = 0; e < V; ++e) { gm[i][e] = v < nv ? gamma[v * V + e] : 0.f; dg[i][e] = 0.f; }
  }
  Vec16<T> gv[NV], hv[NV], av[NV];
  float rs_next = 0.f;
  auto fetch = [&](int64_t row, int64_t at) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      clear(gv[i]);
      clear(hv[i]);
      clear(av[i]);
      if (row < s.rows && lane + i * W * 32 < nv) {
        gv[i].load(dy + at + i * W * 32 * V);
        hv[i].load(h + at + i * W * 32 * V);
        if (dh) av[i].load(dh + at + i * W * 32 * V);
      }
    }
    rs_next = row < s.rows ? rstd[row] : 0.f;
  };
  int64_t row = (int64_t)blockIdx.x * groups + grp;
  int64_t at = row * s.C + lane * V;  // of this lane's first vector
  const int64_t step_at = step * s.C;
  if (AHEAD) fetch(row, at);
  for (; row < s.rows; row += step, at += step_at) {
    if (!AHEAD) fetch(row, at);
    const float rs = rs_next;
    Vec16<T> g0[NV], h0[NV], a0[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) { g0[i] = gv[i]; h0[i] = hv[i]; a0[i] = av[i]; }
    if (AHEAD) fetch(row + step, at + step_at);
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float g[V], f[V];
      g0[i].unpack(g);
      h0[i].unpack(f);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float p = g[e] * (f[e] * rs);
        dg[i][e] += p;
        dot = fmaf(p, gm[i][e], dot);
      }
    }
    dot = group_all<false>(dot, W, red, turn) * s.inv_c;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = lane + i * W * 32;
      if (v >= nv) continue;
      float g[V], f[V], a[V];
      g0[i].unpack(g);
      h0[i].unpack(f);
      a0[i].unpack(a);
#pragma unroll
      for (int e = 0; e < V; ++e) a[e] += rs * (g[e] * gm[i][e] - f[e] * rs * dot);
      Vec16<T> o;
      o.pack(a);
      o.store(dx + at + i * W * 32 * V);
    }
  }
  // the groups of the block in order
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = lane + i * W * 32;
    if (v >= nv) continue;
#pragma unroll
    for (int e = 0; e < V; e += 4)
      *reinterpret_cast<float4*>(cols + (size_t)grp * s.C + v * V + e) = make_float4(dg[i][e], dg[i][e + 1], dg[i][e + 2], dg[i][e + 3]);
  }
  __syncthreads();
  for (int c = threadIdx.x; c < s.C; c += blockDim.x) {
    float t = cols[c];
    for (int k = 1; k < groups; ++k) t += cols[(size_t)k * s.C + c];
    partial[(size_t)blockIdx.x * s.C + c] = t;
  }
}
// dgamma[c] = sum of the blocks' partial rows: 16 columns x 16 lanes a block, lane l adds rows l, l + 16, ... and the lanes
// are added in order.
__global__ void __launch_bounds__(256)
rmsnorm_dgamma_kernel(const float* __restrict__ partial, int blocks, int C, float* __restrict__ dgamma) {
  __shared__ float sh[16][17];
  pdl_enter();
  const int cl = threadIdx.x & 15, l = threadIdx.x >> 4, c = blockIdx.x * 16 + cl;
  float t = 0.f;
  if (c < C) {
    float v[RN_MAX_BLOCKS / 16];
#pragma unroll
    for (int k = 0; k < RN_MAX_BLOCKS / 16; ++k) v[k] = l + 16 * k < blocks ? partial[(size_t)(l + 16 * k) * C + c] : 0.f;
#pragma unroll
    for (int k = 0; k < RN_MAX_BLOCKS / 16; ++k) t += v[k];
  }
  sh[l][cl] = t;
  __syncthreads();
  if (l == 0 && c < C) {
#pragma unroll
    for (int k = 1; k < 16; ++k) t += sh[k][cl];
    dgamma[c] = t;
  }
}

// Warps a row: as few as hold it in 16 elements a lane, and more where the rows are too few to occupy the device; only bf16
// rows beyond 8192 have more elements a lane. Three blocks of eight warps an SM in forward (80 registers a thread), one of
// sixteen in backward.
// 8192 rows of 896 in bf16, out of memory: forward 12.3 us, 4.8 TB/s (13.7 with one warp and four vectors a lane, without the
// next row in flight; 14.6 through a ring of bulk copies in shared memory; 13.3 with 32 bytes a lane and load), backward 15.9
// (28.6; 19.2; 18.5). 777 fp32 rows of 2056 5.1 us. Both keep the issue slots 63 % busy at 36 % (25 % in backward) of the
// warps an SM can hold, waiting for arithmetic as much as for memory: unpacking, summing and packing take 22 instructions an
// element and lane, and more warps would need the registers that hold the rows.
struct RowLaunch {
  RowShape s;
  int nv, threads;
  unsigned blocks;
};
RowLaunch row_launch(int64_t rows, int C, int vec, int warps, int per_sm) {
  RowLaunch l;
  int W = 1;
  while (W < 16 && C > W * 32 * 16) W *= 2;
  const int sms = sm_count();
  while (W < 16 && rows * W < 8ll * sms && ceil_div(C, W * 32 * vec) > 1) W *= 2;
  l.s = {rows, C, W, 1.f / (float)C};
  l.nv = ceil_div(C, W * 32 * vec);
  if (warps < W) warps = W;
  while (warps > W && rows * W < (int64_t)warps * sms) warps /= 2;  // one row a block before a second one
  l.threads = warps * 32;
  const int64_t want = (rows + warps / W - 1) / (warps / W);
  const int64_t room = (int64_t)(warps > 8 ? 1 : per_sm) * sms;
  l.blocks = (unsigned)(want < room ? want : room);
  return l;
}

int check_rows(const char* what, int dtype, int64_t rows, int C) {
  SRT_REQUIRE(dtype == SRT_F32 || dtype == SRT_BF16, "%s: bad dtype %d", what, dtype);
  SRT_REQUIRE(rows >= 0 && C > 0 && C % 8 == 0, "%s: C (%d) must be a positive multiple of 8, rows not negative", what, C);
  SRT_REQUIRE((int64_t)C * (dtype == SRT_F32 ? 4 : 2) <= RN_MAX_ROW_BYTES, "%s: rows of %d elements are longer than %d bytes", what, C, RN_MAX_ROW_BYTES);
  SRT_REQUIRE(rows < (1ll << 31), "%s: more than 2^31 rows", what);
  return SRT_OK;
}
int check_ptrs(const char* what, std::initializer_list<const void*> ps, std::initializer_list<const void*> floats) {
  for (const void* p : ps) SRT_REQUIRE(((uintptr_t)p & 15) == 0, "%s: operands must be 16-byte aligned", what);
  for (const void* p : floats) SRT_REQUIRE(((uintptr_t)p & 3) == 0, "%s: parameters and statistics must be aligned to 4 bytes", what);
  return SRT_OK;
}

template <typename T, bool NORM, bool OUT8>
int fwd_launch(int64_t rows, int C, const void* x, const void* residual, const float* gamma, void* h, void* y, void* q, float* scale,
               float* rstd, float eps, cudaStream_t st) {
  const RowLaunch l = row_launch(rows, C, Vec16<T>::N, 8, 3);
  auto go = [&](auto kernel) -> int {
    SRT_CHECK_CUDA(launch_pdl(kernel, dim3(l.blocks), dim3(l.threads), 0, st, l.s, (const T*)x, (const T*)residual, gamma, (T*)h, (T*)y,
                              (uint8_t*)q, scale, rstd, eps));
    SRT_LAUNCH_CHECK();
    return SRT_OK;
  };
  switch (l.nv) {
    case 1: return go(rmsnorm_fwd_kernel<T, 1, NORM, OUT8>);
    case 2: return go(rmsnorm_fwd_kernel<T, 2, NORM, OUT8>);
    case 3: return go(rmsnorm_fwd_kernel<T, 3, NORM, OUT8>);
    default: return go(rmsnorm_fwd_kernel<T, 4, NORM, OUT8>);
  }
}
// The columns of dgamma that a block adds up, one set a row group: at most 32 KB, and 64 where sixteen warps share a row. They come on
// top of the kernel's static shared memory, so the limit is raised for every instance and not where they alone pass 48 KB.
constexpr int RN_BWD_SMEM = 64 * 1024;
template <typename T, int NV>
int bwd_instance(const RowLaunch& l, int C, const void* dy, const void* h, const float* gamma, const float* rstd, const void* dh, void* dx,
                 float* dgamma, float* partial, cudaStream_t st) {
  const size_t smem = (size_t)(l.threads / 32 / l.s.W) * C * sizeof(float);
  static SmemOptIn opt_in;
  SRT_CHECK_CUDA(opt_in.set(rmsnorm_bwd_kernel<T, NV>, RN_BWD_SMEM));
  SRT_CHECK_CUDA(launch_pdl(rmsnorm_bwd_kernel<T, NV>, dim3(l.blocks), dim3(l.threads), smem, st, l.s, (const T*)dy, (const T*)h, gamma, rstd,
                            (const T*)dh, (T*)dx, partial));
  SRT_LAUNCH_CHECK();
  SRT_CHECK_CUDA(launch_pdl(rmsnorm_dgamma_kernel, dim3(ceil_div(C, 16)), dim3(256), 0, st, (const float*)partial, (int)l.blocks, C, dgamma));
  SRT_LAUNCH_CHECK();
  return SRT_OK;
}
template <typename T>
int bwd_launch(int64_t rows, int C, const void* dy, const void* h, const float* gamma, const float* rstd, const void* dh, void* dx,
               float* dgamma, float* partial, cudaStream_t st) {
  const RowLaunch l = row_launch(rows, C, Vec16<T>::N, 16, 1);
  SRT_REQUIRE(l.blocks <= RN_MAX_BLOCKS, "rmsnorm_bwd: %u partial rows", l.blocks);
  switch (l.nv) {
    case 1: return bwd_instance<T, 1>(l, C, dy, h, gamma, rstd, dh, dx, dgamma, partial, st);
    case 2: return bwd_instance<T, 2>(l, C, dy, h, gamma, rstd, dh, dx, dgamma, partial, st);
    case 3: return bwd_instance<T, 3>(l, C, dy, h, gamma, rstd, dh, dx, dgamma, partial, st);
    default: return bwd_instance<T, 4>(l, C, dy, h, gamma, rstd, dh, dx, dgamma, partial, st);
  }
}

}  // namespace
}  // namespace srt

using namespace srt;

extern "C" {

int srt_rmsnorm_fwd(int dtype, const void* x, const void* residual, const float* gamma, void* h, void* y, float* rstd, int64_t rows,
                    int C, float eps, void* stream) {
  int rc = check_rows("rmsnorm_fwd", dtype, rows, C);
  if (rc || rows == 0) return rc;
  SRT_REQUIRE(x && gamma && y, "rmsnorm_fwd: null operand");
  if ((rc = check_ptrs("rmsnorm_fwd", {x, residual, h, y}, {gamma, rstd}))) return rc;
  return dtype == SRT_F32 ? fwd_launch<float, true, false>(rows, C, x, residual, gamma, h, y, nullptr, nullptr, rstd, eps, (cudaStream_t)stream)
                          : fwd_launch<bf16, true, false>(rows, C, x, residual, gamma, h, y, nullptr, nullptr, rstd, eps, (cudaStream_t)stream);
}

int srt_rmsnorm_fwd_e4m3(int dtype, const void* x, const void* residual, const float* gamma, void* h, void* q, float* scale, float* rstd,
                         int64_t rows, int C, float eps, void* stream) {
  int rc = check_rows("rmsnorm_fwd_e4m3", dtype, rows, C);
  if (rc || rows == 0) return rc;
  SRT_REQUIRE(x && gamma && q && scale, "rmsnorm_fwd_e4m3: null operand");
  if ((rc = check_ptrs("rmsnorm_fwd_e4m3", {x, residual, h, q}, {gamma, scale, rstd}))) return rc;
  return dtype == SRT_F32 ? fwd_launch<float, true, true>(rows, C, x, residual, gamma, h, nullptr, q, scale, rstd, eps, (cudaStream_t)stream)
                          : fwd_launch<bf16, true, true>(rows, C, x, residual, gamma, h, nullptr, q, scale, rstd, eps, (cudaStream_t)stream);
}

int srt_quantize_rows_e4m3(int dtype, const void* x, void* q, float* scale, int64_t rows, int C, void* stream) {
  int rc = check_rows("quantize_rows_e4m3", dtype, rows, C);
  if (rc || rows == 0) return rc;
  SRT_REQUIRE(x && q && scale, "quantize_rows_e4m3: null operand");
  if ((rc = check_ptrs("quantize_rows_e4m3", {x, q}, {scale}))) return rc;
  return dtype == SRT_F32 ? fwd_launch<float, false, true>(rows, C, x, nullptr, nullptr, nullptr, nullptr, q, scale, nullptr, 0.f, (cudaStream_t)stream)
                          : fwd_launch<bf16, false, true>(rows, C, x, nullptr, nullptr, nullptr, nullptr, q, scale, nullptr, 0.f, (cudaStream_t)stream);
}

size_t srt_rmsnorm_bwd_scratch_bytes(int C) { return C > 0 ? (size_t)RN_MAX_BLOCKS * C * sizeof(float) : 0; }

int srt_rmsnorm_bwd(int dtype, const void* dy, const void* h, const float* gamma, const float* rstd, const void* dh, void* dx,
                    float* dgamma, int64_t rows, int C, void* scratch, size_t scratch_bytes, void* stream) {
  int rc = check_rows("rmsnorm_bwd", dtype, rows, C);
  if (rc) return rc;
  SRT_REQUIRE(dgamma, "rmsnorm_bwd: null operand");
  if (rows == 0) {
    SRT_CHECK_CUDA(cudaMemsetAsync(dgamma, 0, (size_t)C * sizeof(float), (cudaStream_t)stream));
    return SRT_OK;
  }
  SRT_REQUIRE(dy && h && gamma && rstd && dx, "rmsnorm_bwd: null operand");
  SRT_REQUIRE(scratch && scratch_bytes >= srt_rmsnorm_bwd_scratch_bytes(C), "rmsnorm_bwd: scratch too small (%zu < %zu)", scratch_bytes,
              srt_rmsnorm_bwd_scratch_bytes(C));
  if ((rc = check_ptrs("rmsnorm_bwd", {dy, h, dh, dx}, {gamma, rstd, dgamma, scratch}))) return rc;
  return dtype == SRT_F32 ? bwd_launch<float>(rows, C, dy, h, gamma, rstd, dh, dx, dgamma, (float*)scratch, (cudaStream_t)stream)
                          : bwd_launch<bf16>(rows, C, dy, h, gamma, rstd, dh, dx, dgamma, (float*)scratch, (cudaStream_t)stream);
}

}  // extern "C"
