// Global gradient norm and clipping for the executors (grad_clip.cu).
#pragma once
#include "common.cuh"

namespace srt {

size_t grad_norm_scratch_bytes(int tensors);
// clip[0] = norm of all tensors together, clip[1] = min(1, max_norm / (norm + 1e-6)); scale = 1 also multiplies the tensors
// by clip[1] in place.
int grad_norm(int dtype, int tensors, void* const* grads, const int64_t* counts, float max_norm, int scale, float* clip, void* scratch,
              size_t scratch_bytes, cudaStream_t st);

// What an executor keeps for it: the two results, the partial sums, and whether the next optimizer step takes the coefficient.
struct GradClip {
  float* clip = nullptr;
  void* scratch = nullptr;
  bool armed = false, ran = false;
  ~GradClip() { cudaFree(clip); }
  GradClip() = default;
  GradClip(const GradClip&) = delete;
  GradClip& operator=(const GradClip&) = delete;
  // With the step's other buffers: a step that runs takes no memory.
  int prepare() {
    SRT_CHECK_CUDA(cudaMalloc((void**)&clip, 256 + grad_norm_scratch_bytes(1)));
    scratch = (char*)clip + 256;
    return SRT_OK;
  }
  int measure(float* grad, int64_t n, float max_norm, cudaStream_t st) {
    SRT_REQUIRE(max_norm > 0.f, "clip_grad_norm: max_norm (%g) must be positive", (double)max_norm);
    void* g = grad;
    int rc = grad_norm(SRT_F32, 1, &g, &n, max_norm, 0, clip, scratch, grad_norm_scratch_bytes(1), st);
    if (rc) return rc;
    armed = ran = true;
    return SRT_OK;
  }
  // the coefficient of the next optimizer step, once
  const float* take() {
    const float* c = armed ? clip + 1 : nullptr;
    armed = false;
    return c;
  }
  int read(float* host_norm, cudaStream_t st) {
    SRT_REQUIRE(host_norm && ran, "grad_norm: clip_grad_norm has not run");
    SRT_CHECK_CUDA(cudaMemcpyAsync(host_norm, clip, sizeof(float), cudaMemcpyDeviceToHost, st));
    SRT_CHECK_CUDA(cudaStreamSynchronize(st));
    return SRT_OK;
  }
};

}  // namespace srt
