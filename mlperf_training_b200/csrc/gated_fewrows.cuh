// Gated projections, and the down projection behind them, of few activation rows (gated_fewrows.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>

namespace fewrows {

constexpr int MAX_ROWS = 64;

struct GatedArgs {
  const __nv_bfloat16* x; const __nv_bfloat16* w;     // [M, K], [2F, K]
  __nv_bfloat16* a; void* gu;                         // [M, F], [M, 2F] (bf16 or fp32) or null
  int M, F, K;
  long long ldx, ldw, lda, ldgu;
  int act;
  int gu_f32;
};
int run_gated(const GatedArgs& p, cudaStream_t stream);

struct DownArgs {
  const __nv_bfloat16* a; const __nv_bfloat16* w;     // [M, K], [N, K]
  const __nv_bfloat16* res; __nv_bfloat16* y;         // [M, N] or null, [M, N]
  int M, N, K;
  long long lda, ldw, ldr, ldy;
};
int run_down(const DownArgs& p, cudaStream_t stream);

}  // namespace fewrows
