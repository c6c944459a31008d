// Global gradient norm over many tensors, and clipping by it.
//
//   norm = sqrt(sum over all tensors of g^2),   coefficient = min(1, max_norm / (norm + 1e-6))
//
// The squares are formed and added in 64 bits: no gradient that fp32 can hold overflows its square, and the result does not
// depend on how the sum is cut beyond its last bits. A NaN anywhere makes norm and coefficient NaN, an infinity a coefficient
// of zero; nothing is skipped on the way.
//
// The list of tensors travels in the kernel's parameters (nothing to copy, so a call can be captured), cut into chunks of which
// every block takes an equal share. Bound by memory: one read for the norm; clipping in place reads and writes once more. The
// second launch walks each share backwards, so that what the first one read last comes out of L2, and every block adds the
// partial sums for itself instead of waiting for a launch between.
#include <algorithm>
#include <new>
#include <vector>

#include "common.cuh"
#include "grad_clip.cuh"

namespace srt {
namespace {

using bf16 = __nv_bfloat16;
constexpr int GC_THREADS = 512;
// Elements of a chunk: one turn of a block's loop over fp32. Every block takes the same number of chunks, one after the other:
// the norm of 508 M fp32 in 169 tensors takes 344 us (5.9 TB/s), scaling them 657 (6.2 TB/s); with chunks of 32768 dealt in
// turn 353 and 675. The conversions to 64 bits are what keeps the norm from the memory's rate: with squares added in fp32 16 at
// a time it reads 498 MB in 91 us instead of 100, but then its last bit is no longer the sum's.
constexpr int GC_CHUNK = 8192;
constexpr int GC_MAX_BLOCKS = 1024;   // partial sums of a launch
// Tensors in the parameters of a launch. They are copied whole, 0.6 or 20 KB: 30 tensors take 7.0 us of the host with the short
// list and 9.5 with the long one; a hundred would take four launches a pass with the short one.
constexpr int GC_FEW = 32, GC_MANY = 1024;

template <int MAXT>
struct TensorList {
  void* ptr[MAXT];
  int64_t n[MAXT];
  int first[MAXT + 1];  // first chunk of every tensor, and the number of chunks
  int tensors;
};

__device__ __forceinline__ double block_sum(double v, double* sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0;
#pragma unroll
  for (int w = 0; w < GC_THREADS / 32; ++w) v += sh[w];
  return v;
}

// A block's share: as many chunks as any other's or one more, one after the other. f(tensor, first element, elements) for every tensor that
// the share meets, in order or (BACK) in the opposite order.
template <bool BACK, int MAXT, typename F>
__device__ __forceinline__ void share_of_block(const TensorList<MAXT>& l, F&& f) {
  constexpr int MOST = (1 << 28) / GC_CHUNK;  // chunks at a time, so that elements count in 32 bits
  const int all = l.first[l.tensors], b = (int)blockIdx.x, each = all / (int)gridDim.x, over = all - each * (int)gridDim.x;
  const int c0 = b * each + min(b, over), c1 = c0 + each + (b < over ? 1 : 0);  // the first `over` blocks have one more
  if (c0 >= c1) return;
  const int begin = BACK ? c1 - 1 : c0;
  int lo = 0, hi = l.tensors - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (l.first[mid] <= begin) lo = mid;
    else hi = mid - 1;
  }
  for (int t = lo, c = BACK ? c1 : c0; BACK ? c > c0 : c < c1;) {
    int from, to;  // chunks of tensor t
    if (BACK) {
      while (c <= l.first[t]) --t;
      to = c;
      from = max(max(c0, l.first[t]), c - MOST);
      c = from;
    } else {
      while (c >= l.first[t + 1]) ++t;
      from = c;
      to = min(min(c1, l.first[t + 1]), c + MOST);
      c = to;
    }
    const int64_t at = (int64_t)(from - l.first[t]) * GC_CHUNK, end = (int64_t)(to - l.first[t]) * GC_CHUNK;
    f(t, at, (int)((end < l.n[t] ? end : l.n[t]) - at));
  }
}
// Elements before the first 16-byte boundary.
template <typename T>
__device__ __forceinline__ int head_of(const T* p, int n) {
  const int h = (int)(((16 - ((uintptr_t)p & 15)) & 15) / sizeof(T));
  return h < n ? h : n;
}

template <typename T, int MAXT>
__global__ void __launch_bounds__(GC_THREADS)
grad_norm_partial_kernel(const __grid_constant__ TensorList<MAXT> l, double* __restrict__ partial) {
  constexpr int V = Vec16<T>::N, U = 4;
  __shared__ double sh[GC_THREADS / 32];
  pdl_enter();
  double acc = 0.0;
  share_of_block<false>(l, [&](int t, int64_t begin, int n) {
    const T* p = (const T*)l.ptr[t] + begin;
    const int head = head_of(p, n), nv = (n - head) / V;
    const T* pv = p + head;
    auto one = [&](float f) { acc = fma((double)f, (double)f, acc); };
    for (int v = threadIdx.x; v < nv; v += U * GC_THREADS) {
      Vec16<T> a[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        a[u].raw = {};
        if (v + u * GC_THREADS < nv) a[u].load(pv + (int64_t)(v + u * GC_THREADS) * V);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float f[V];
        a[u].unpack(f);
#pragma unroll
        for (int e = 0; e < V; ++e) one(f[e]);
      }
    }
    if ((int)threadIdx.x < head) one(ElemTraits<T>::to_f(p[threadIdx.x]));
    const int tail = head + nv * V + (int)threadIdx.x;
    if (tail < n) one(ElemTraits<T>::to_f(p[tail]));
  });
  acc = block_sum(acc, sh);
  if (threadIdx.x == 0) partial[blockIdx.x] = acc;
}

// Every block adds all partial sums in the same order and so has the same coefficient.
__device__ __forceinline__ float coefficient_of(const double* __restrict__ partial, int count, float max_norm, double* sh, float* __restrict__ clip) {
  double s = 0.0;
  for (int i = threadIdx.x; i < count; i += GC_THREADS) s += partial[i];
  const double norm = sqrt(block_sum(s, sh));
  const double c = (double)max_norm / (norm + 1e-6);
  const float k = c > 1.0 ? 1.f : (float)c;  // NaN stays
  if (blockIdx.x == 0 && threadIdx.x == 0 && clip) { clip[0] = (float)norm; clip[1] = k; }
  return k;
}
__global__ void __launch_bounds__(GC_THREADS)
grad_norm_final_kernel(const double* __restrict__ partial, int count, float max_norm, float* __restrict__ clip) {
  __shared__ double sh[GC_THREADS / 32];
  pdl_enter();
  coefficient_of(partial, count, max_norm, sh, clip);
}
template <typename T, int MAXT>
__global__ void __launch_bounds__(GC_THREADS)
grad_scale_kernel(const __grid_constant__ TensorList<MAXT> l, const double* __restrict__ partial, int count, float max_norm,
                  float* __restrict__ clip) {
  constexpr int V = Vec16<T>::N, U = 4;
  __shared__ double sh[GC_THREADS / 32];
  pdl_enter();
  const float k = coefficient_of(partial, count, max_norm, sh, clip);
  share_of_block<true>(l, [&](int t, int64_t begin, int n) {
    T* p = (T*)l.ptr[t] + begin;
    const int head = head_of(p, n), nv = (n - head) / V;
    T* pv = p + head;
    for (int v = (nv - 1) / (U * GC_THREADS) * (U * GC_THREADS) + (int)threadIdx.x; v >= 0; v -= U * GC_THREADS) {
      Vec16<T> a[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (v + u * GC_THREADS < nv) a[u].load(pv + (int64_t)(v + u * GC_THREADS) * V);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (v + u * GC_THREADS >= nv) break;
        float f[V];
        a[u].unpack(f);
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] *= k;
        a[u].pack(f);
        a[u].store(pv + (int64_t)(v + u * GC_THREADS) * V);
      }
    }
    if ((int)threadIdx.x < head) p[threadIdx.x] = ElemTraits<T>::from_f(ElemTraits<T>::to_f(p[threadIdx.x]) * k);
    const int tail = head + nv * V + (int)threadIdx.x;
    if (tail < n) p[tail] = ElemTraits<T>::from_f(ElemTraits<T>::to_f(p[tail]) * k);
  });
}

template <int MAXT>
void fill(TensorList<MAXT>& l, int tensors, void* const* grads, const int64_t* counts) {
  l.tensors = tensors;
  int chunk = 0;
  for (int i = 0; i < tensors; ++i) {
    l.ptr[i] = grads[i];
    l.n[i] = counts[i];
    l.first[i] = chunk;
    chunk += (int)((counts[i] + GC_CHUNK - 1) / GC_CHUNK);
  }
  l.first[tensors] = chunk;
}
inline unsigned blocks_for(int chunks) {
  const int room = 4 * sm_count() < GC_MAX_BLOCKS ? 4 * sm_count() : GC_MAX_BLOCKS;
  return (unsigned)(chunks < room ? chunks : room);
}

// Up to MAXT tensors a launch.
template <typename T, int MAXT>
int run(int tensors, void* const* grads, const int64_t* counts, float max_norm, int scale, float* clip, double* partial, cudaStream_t st) {
  TensorList<MAXT> l;
  int count = 0;
  for (int i = 0; i < tensors; i += MAXT) {
    fill(l, tensors - i < MAXT ? tensors - i : MAXT, grads + i, counts + i);
    const unsigned blocks = blocks_for(l.first[l.tensors]);
    if (blocks == 0) continue;
    SRT_CHECK_CUDA(launch_pdl(grad_norm_partial_kernel<T, MAXT>, dim3(blocks), dim3(GC_THREADS), 0, st, l, partial + count));
    SRT_LAUNCH_CHECK();
    count += (int)blocks;
  }
  if (!scale || count == 0) {
    SRT_CHECK_CUDA(launch_pdl(grad_norm_final_kernel, dim3(1), dim3(GC_THREADS), 0, st, (const double*)partial, count, max_norm, clip));
    SRT_LAUNCH_CHECK();
    return SRT_OK;
  }
  for (int i = tensors > 0 ? (tensors - 1) / MAXT * MAXT : -1; i >= 0; i -= MAXT) {
    if (tensors > MAXT) fill(l, tensors - i < MAXT ? tensors - i : MAXT, grads + i, counts + i);
    const unsigned blocks = blocks_for(l.first[l.tensors]);
    if (blocks == 0) continue;
    SRT_CHECK_CUDA(launch_pdl(grad_scale_kernel<T, MAXT>, dim3(blocks), dim3(GC_THREADS), 0, st, l, (const double*)partial, count, max_norm, clip));
    SRT_LAUNCH_CHECK();
  }
  return SRT_OK;
}

// A tensor that shares memory with another one, or -1. Lists that ascend in memory, as an executor lays its gradients out, need
// one look; others are put in order. -2: no memory for that.
int first_overlap(int esz, int tensors, void* const* grads, const int64_t* counts) {
  auto begin = [&](int i) { return (uintptr_t)grads[i]; };
  auto end = [&](int i) { return (uintptr_t)grads[i] + (uintptr_t)counts[i] * esz; };
  uintptr_t reached = 0;
  bool ascending = true;
  for (int i = 0; i < tensors && ascending; ++i) {
    if (counts[i] == 0) continue;
    ascending = begin(i) >= reached;
    reached = end(i);
  }
  if (ascending) return -1;
  std::vector<int> order;
  try {
    order.reserve((size_t)tensors);
  } catch (const std::bad_alloc&) {
    return -2;
  }
  for (int i = 0; i < tensors; ++i)
    if (counts[i] > 0) order.push_back(i);
  std::sort(order.begin(), order.end(), [&](int a, int b) { return begin(a) < begin(b); });
  for (size_t k = 1; k < order.size(); ++k)
    if (begin(order[k]) < end(order[k - 1])) return order[k];
  return -1;
}

}  // namespace

size_t grad_norm_scratch_bytes(int tensors) {
  return (size_t)(tensors > 0 ? (tensors + GC_MANY - 1) / GC_MANY : 1) * GC_MAX_BLOCKS * sizeof(double);
}

int grad_norm(int dtype, int tensors, void* const* grads, const int64_t* counts, float max_norm, int scale, float* clip, void* scratch,
              size_t scratch_bytes, cudaStream_t st) {
  SRT_REQUIRE(dtype == SRT_F32 || dtype == SRT_BF16, "grad_norm: bad dtype %d", dtype);
  SRT_REQUIRE(tensors >= 0 && (tensors == 0 || (grads && counts)) && clip, "grad_norm: null argument");
  SRT_REQUIRE(((uintptr_t)clip & 3) == 0, "grad_norm: clip is not aligned to its elements");
  SRT_REQUIRE(max_norm > 0.f, "grad_norm: max_norm (%g) must be positive", (double)max_norm);
  int64_t chunks = 0;
  for (int i = 0; i < tensors; ++i) {
    SRT_REQUIRE(counts[i] >= 0 && (counts[i] == 0 || grads[i]), "grad_norm: tensor %d has no memory or a negative count", i);
    SRT_REQUIRE(((uintptr_t)grads[i] & (dtype == SRT_F32 ? 3 : 1)) == 0, "grad_norm: tensor %d is not aligned to its elements", i);
    chunks += counts[i] / GC_CHUNK + 1;
    SRT_REQUIRE(chunks < (1ll << 30), "grad_norm: more than 2^43 elements");
  }
  if (scale) {
    const int twice = first_overlap(dtype == SRT_F32 ? 4 : 2, tensors, grads, counts);
    if (twice == -2) {
      set_error("clip_grad_norm: no host memory for a list of %d tensors", tensors);
      return SRT_ERR_NOMEM;
    }
    SRT_REQUIRE(twice < 0, "clip_grad_norm: tensor %d shares memory with another and would be scaled twice", twice);
  }
  SRT_REQUIRE(scratch && ((uintptr_t)scratch & 7) == 0 && scratch_bytes >= grad_norm_scratch_bytes(tensors),
              "grad_norm: scratch missing, unaligned or too small (%zu < %zu)", scratch_bytes, grad_norm_scratch_bytes(tensors));
  if (dtype == SRT_F32)
    return tensors <= GC_FEW ? run<float, GC_FEW>(tensors, grads, counts, max_norm, scale, clip, (double*)scratch, st)
                             : run<float, GC_MANY>(tensors, grads, counts, max_norm, scale, clip, (double*)scratch, st);
  return tensors <= GC_FEW ? run<bf16, GC_FEW>(tensors, grads, counts, max_norm, scale, clip, (double*)scratch, st)
                           : run<bf16, GC_MANY>(tensors, grads, counts, max_norm, scale, clip, (double*)scratch, st);
}

}  // namespace srt

using namespace srt;

extern "C" {

size_t srt_grad_norm_scratch_bytes(int tensors) { return grad_norm_scratch_bytes(tensors); }

int srt_grad_norm(int dtype, int tensors, const void* const* grads, const int64_t* counts, float max_norm, float* clip, void* scratch,
                  size_t scratch_bytes, void* stream) {
  return grad_norm(dtype, tensors, const_cast<void* const*>(grads), counts, max_norm, 0, clip, scratch, scratch_bytes, (cudaStream_t)stream);
}

int srt_clip_grad_norm(int dtype, int tensors, void* const* grads, const int64_t* counts, float max_norm, float* clip, void* scratch,
                       size_t scratch_bytes, void* stream) {
  return grad_norm(dtype, tensors, grads, counts, max_norm, 1, clip, scratch, scratch_bytes, (cudaStream_t)stream);
}

}  // extern "C"
