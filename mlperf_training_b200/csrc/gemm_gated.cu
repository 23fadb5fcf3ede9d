// Gated feed-forward block in bf16, on the CTA-pair mainloop of gemm_core.cuh:
//
//   b200_gemm_gated       a = act(x Wg^T) * (x Wu^T), optionally with the projections themselves (gu, kept for the backward), in one launch
//   b200_gated_down       y = a Wd^T (+ residual) of up to 64 rows (more are a plain GEMM)
//   b200_gemm_gated_grad  da = dy Wd, then d gate = da u act'(g), d up = da act(g) and a again, in one launch
//
// W = [Wg; Wu] is the stacked [2F, D] weight of the two projections as the model keeps it.  A 256-row tile of 128 output columns runs as one
// 256 x 256 tile: the leader CTA stages the 128 gate rows, its partner the 128 up rows of the same columns, so that the gate lands in the
// accumulator's first half and the up projection in its second, and an epilogue warp has both at hand.  Against a GEMM and a SwiGLU kernel the
// projections are not read again by the forward, and one without a backward writes 2 bytes of T F instead of 6.
//
// Roundings: a once from fp32, da not at all.  gate and up are kept for the backward in fp32 where the caller asks for it (functional.py:
// GatedMLPFn does), else rounded once to bf16, half the bytes; then d gate and d up have two or three roundings of 2^-9 in them and the gradients
// of 4096 x 4096 x 14336 are 0.0030 off in norm, 0.0034 that of Wd, instead of 0.0023 (0.0017 the results' own rounding).
// Measured (4096 tokens, 4096 x 2 x 14336, caches cold): forward 648 us (1.48 PFLOP/s; 622 with projections in bf16, 600 without), gradient
// 411 us (1.17 PFLOP/s; 378 from projections in bf16, the GEMM of that size alone 293): bound by the tensor pipe under the power cap, the
// gradient by its epilogue (two operands in, three results out) where a tile's mainloop of 64 stages does not cover it.
// Up to 64 rows: gated_fewrows.cu.
#include "common.cuh"
#include "gemm_core.cuh"
#include "gated_fewrows.cuh"
#include "runtime.h"

namespace {
constexpr int GU_F32 = 2;
int check(const char* what, const void* p, long long ld) {
  return (((uintptr_t)p & 15) != 0 || ld % 8 != 0) ? b200::fail(861, "%s: operands must be 16-byte aligned, pitches multiples of 8", what) : 0;
}
}  // namespace

// x [M, K], w [2F, K], a [M, F], gu [M, 2F] or null; pitches in elements, multiples of 8; F and K multiples of 8.  act: 0 SiLU, 1 GELU (tanh),
// + 2 (GU_F32) where gu is fp32, else bf16.
B200_API int b200_gemm_gated(const void* x, const void* w, void* a, void* gu, int M, int F, int K, long long ldx, long long ldw,
                             long long lda, long long ldgu, int act, void* stream) {
  using namespace gemmcore;
  if (M <= 0 || F <= 0 || K <= 0) return b200::fail(860, "gemm_gated: empty problem %d x 2 x %d x %d", M, F, K);
  if (F % 8 != 0 || K % 8 != 0) return b200::fail(862, "gemm_gated: F=%d and K=%d must be multiples of 8", F, K);
  int r;
  if ((r = check("gemm_gated", x, ldx)) || (r = check("gemm_gated", w, ldw)) || (r = check("gemm_gated", a, lda)) ||
      (gu != nullptr && (r = check("gemm_gated", gu, ldgu))))
    return r;
  if (M <= fewrows::MAX_ROWS) {
    const fewrows::GatedArgs p = {(const __nv_bfloat16*)x, (const __nv_bfloat16*)w, (__nv_bfloat16*)a, gu, M, F, K, ldx, ldw, lda, ldgu,
                                  act & 1, (act & GU_F32) != 0};
    return fewrows::run_gated(p, (cudaStream_t)stream);
  }
  CUtensorMap tmX, tmW, tmA, tmG, tmU;
  if ((r = b200::make_tmap_2d(&tmX, b200::DT_BF16, x, K, M, ldx * 2, 64, a_box_rows(M), b200::SWZ_128))) return r;
  if ((r = b200::make_tmap_2d(&tmW, b200::DT_BF16, w, K, 2LL * F, ldw * 2, 64, 128, b200::SWZ_128))) return r;
  if ((r = b200::make_tmap_2d(&tmA, b200::DT_BF16, a, F, M, lda * 2, 32, 32, b200::SWZ_64))) return r;
  tmG = tmU = tmA;
  if (gu != nullptr) {
    const bool f32 = act & GU_F32;
    const auto type = f32 ? b200::DT_F32 : b200::DT_BF16;
    const auto swizzle = f32 ? b200::SWZ_128 : b200::SWZ_64;
    const long long es = f32 ? 4 : 2;
    if ((r = b200::make_tmap_2d(&tmG, type, gu, F, M, ldgu * es, 32, 32, swizzle))) return r;
    if ((r = b200::make_tmap_2d(&tmU, type, (uint8_t*)gu + es * F, F, M, ldgu * es, 32, 32, swizzle))) return r;
  }
  PairParams p = {};
  p.M = M; p.N = F; p.K = K;
  p.group_m = raster_group_m() > 1 ? raster_group_m() / 2 : 1;
  p.gate.act = act & 1; p.gate.gu_f32 = (act & GU_F32) != 0; p.gate.F = F; p.gate.want_gu = gu != nullptr;
  p.a_rows = a_box_rows(M);
  p.status = b200::status_ptr();
  return launch_pair<KIND_BF16, 256, 1, 1, 1>(tmX, tmW, tmG, tmU, tmA, tmA, p, (cudaStream_t)stream, "gemm_gated");
}

// a [M, K], w [N, K], res [M, N] or null, y [M, N]; M up to 64, N and K multiples of 8; pitches as above (any for res and y, which need 2-byte alignment).
B200_API int b200_gated_down(const void* a, const void* w, const void* res, void* y, int M, int N, int K, long long lda, long long ldw,
                             long long ldr, long long ldy, void* stream) {
  if (M <= 0 || M > fewrows::MAX_ROWS || N <= 0 || K <= 0) return b200::fail(865, "gated_down: %d x %d x %d is not a product of 1 to 64 rows", M, N, K);
  if (N % 8 != 0 || K % 8 != 0) return b200::fail(866, "gated_down: N=%d and K=%d must be multiples of 8", N, K);
  int r;
  if ((r = check("gated_down", a, lda)) || (r = check("gated_down", w, ldw))) return r;
  const fewrows::DownArgs p = {(const __nv_bfloat16*)a, (const __nv_bfloat16*)w, (const __nv_bfloat16*)res, (__nv_bfloat16*)y, M, N, K, lda, ldw, ldr, ldy};
  return fewrows::run_down(p, (cudaStream_t)stream);
}

// dy [M, K], wd [K, F] (the down projection's weight as it is), gu [M, 2F]; dgu [M, 2F] and a [M, F] (or null) bf16; act as above.
B200_API int b200_gemm_gated_grad(const void* dy, const void* wd, const void* gu, void* dgu, void* a, int M, int F, int K, long long lddy,
                                  long long ldwd, long long ldgu, long long lddgu, long long lda, int act, void* stream) {
  using namespace gemmcore;
  if (M <= 0 || F <= 0 || K <= 0) return b200::fail(863, "gemm_gated_grad: empty problem %d x %d x %d", M, F, K);
  if (F % 8 != 0 || K % 8 != 0) return b200::fail(864, "gemm_gated_grad: F=%d and K=%d must be multiples of 8", F, K);
  int r;
  if ((r = check("gemm_gated_grad", dy, lddy)) || (r = check("gemm_gated_grad", wd, ldwd)) || (r = check("gemm_gated_grad", gu, ldgu)) ||
      (r = check("gemm_gated_grad", dgu, lddgu)) || (a != nullptr && (r = check("gemm_gated_grad", a, lda))))
    return r;
  CUtensorMap tmY, tmW, tmA, tmG, tmU;
  if ((r = b200::make_tmap_2d(&tmY, b200::DT_BF16, dy, K, M, lddy * 2, 64, a_box_rows(M), b200::SWZ_128))) return r;
  if ((r = b200::make_tmap_2d(&tmW, b200::DT_BF16, wd, F, K, ldwd * 2, 64, 64, b200::SWZ_128))) return r;
  if ((r = b200::make_tmap_2d(&tmG, b200::DT_BF16, dgu, F, M, lddgu * 2, 32, 32, b200::SWZ_64))) return r;
  if ((r = b200::make_tmap_2d(&tmU, b200::DT_BF16, (uint8_t*)dgu + 2LL * F, F, M, lddgu * 2, 32, 32, b200::SWZ_64))) return r;
  tmA = tmG;
  if (a != nullptr && (r = b200::make_tmap_2d(&tmA, b200::DT_BF16, a, F, M, lda * 2, 32, 32, b200::SWZ_64))) return r;
  PairParams p = {};
  p.M = M; p.N = F; p.K = K;
  p.b_mn_major = 1;
  p.group_m = raster_group_m() > 1 ? raster_group_m() / 2 : 1;
  p.gate.act = act & 1; p.gate.gu_f32 = (act & GU_F32) != 0; p.gate.F = F; p.gate.want_a = a != nullptr;
  p.gate.gu = gu; p.gate.ldgu = ldgu;
  p.a_rows = a_box_rows(M);
  p.status = b200::status_ptr();
  return launch_pair<KIND_BF16, 256, 1, 1, 2>(tmY, tmW, tmG, tmU, tmA, tmA, p, (cudaStream_t)stream, "gemm_gated_grad");
}
