// Gated projections of few activation rows (gated_fewrows.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>

namespace fewrows {

constexpr int MAX_ROWS = 64;

struct GatedArgs {
  const __nv_bfloat16* x; const __nv_bfloat16* w;     // [M, K], [2F, K]
  __nv_bfloat16* a; __nv_bfloat16* gu;                // [M, F], [M, 2F] or null
  int M, F, K;
  long long ldx, ldw, lda, ldgu;
  int act;
};
int run_gated(const GatedArgs& p, cudaStream_t stream);

}  // namespace fewrows
