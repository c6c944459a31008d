// Gated feed-forward block for the executors (gated_ffn.cu); the C entry points forward to these.
#pragma once
#include "common.cuh"

namespace srt {

// x_scale and w_scale with e4m3 operands, null with bf16 ones. The scratch takes act and the slots of shared tiles.
size_t gated_ffn_fwd_scratch_bytes(const srt_gated_ffn_desc& d);
int gated_ffn_fwd(const srt_gated_ffn_desc* d, const void* x, const float* x_scale, const void* w_gu, const float* w_scale,
                  const void* w_down, const void* residual, void* y, void* scratch, size_t scratch_bytes, bool e4m3, cudaStream_t st);
// Byte offsets into the scratch of a backward call: act at 0, dgu, the slots of shared tiles.
struct GatedFfnScratch { size_t dgu, slots, total; };
GatedFfnScratch gated_ffn_scratch(const srt_gated_ffn_desc& d, int grad_dtype);
int gated_ffn_bwd(const srt_gated_ffn_desc* d, const void* dy, const void* x, const void* w_gu, const void* w_down, int grad_dtype,
                  void* dx, void* dw_gu, void* dw_down, void* scratch, size_t scratch_bytes, cudaStream_t st);

}  // namespace srt
