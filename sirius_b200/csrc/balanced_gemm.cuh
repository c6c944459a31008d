// Plain bf16 products whose work is dealt evenly to all SMs (balanced_gemm.cu): the products around the gated kernels of the
// feed-forward block.
#pragma once
#include "common.cuh"

namespace srt {

// D[m][n] = sum_k A(m, k) B(n, k) (+ addend[m][n]), bf16 operands, fp32 accumulation, D bf16 or fp32. A is stored [M][K]
// (a_mn = 0) or [K][M] (1), B likewise [N][K] or [K][N], their rows a_pitch and b_pitch elements apart (0: dense). b_mn = 0 needs a_mn = 0. The stored widths and pitches are
// multiples of 8 and the pointers 16-byte aligned. scratch, 16-byte aligned: with less than
// balanced_gemm_scratch_bytes (a launch in a smaller SM partition may want another amount) the work is dealt less evenly.
// b_early: B may be fetched while the launch in front on the stream still runs: that launch does not write it, and is one that
// waits for its own predecessor before it lets this one start (every kernel here is).
struct GemmProblem {
  int M, N, K;
  bool a_mn, b_mn;
  int out_dtype;  // SRT_BF16 or SRT_F32
  int a_pitch = 0, b_pitch = 0;
};
size_t balanced_gemm_scratch_bytes(const GemmProblem& p);
int balanced_gemm(const GemmProblem& p, const void* A, const void* B, const void* addend, void* D, void* scratch, size_t scratch_bytes,
                  bool b_early, cudaStream_t st);

}  // namespace srt
