// MXFP4 block-scaled GEMM for sm_100a:
//
//   D[M,N] (=|+=) alpha * (A_q * 2^sfa)[M,K] * (B_q * 2^sfb)[N,K]^T (+ bias[N]) (+ residual[M,N])
//
// A_q / B_q are e2m1 codes, two per byte (the even element in the low half), K-major; sfa / sfb hold one UE8M0 scale per 32
// contraction elements in the atom layout of quant_mxfp8.cu (tile rows = 128 for A, = b200_gemm_mxfp4_bn(N) for B).
//
// gemmcore::gemm_pair_kernel<KIND_MXFP4> (gemm_core.cuh): CTA pairs on 256 x BN tiles with
// tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X, 64 elements an instruction, 256 elements of K (128 bytes) per
// pipeline stage; the scale sets of a stage reach tensor memory through the four forwarding warps.
//
// BN = 192: 2 x 192 accumulator columns leave 128 of tensor memory: six scale sets of 20 columns, so six stages (190 KB) in flight, beside one
// 4 KB staging buffer for each of the eight epilogue warps.
#include "common.cuh"
#include "gemm_core.cuh"
#include "runtime.h"

namespace {

template <int BN>
int run(const void* a_q, const void* sfa, const void* b_q, const void* sfb, void* d, int M, int N, int K, long long lda, long long ldb,
        long long ldd, const gemmcore::EpiArgs& epi, void* ws, long long ws_bytes, cudaStream_t stream) {
  using namespace gemmcore;
  CUtensorMap tmA, tmB, tmSFA, tmSFB, tmD, tmDt;
  int r;
  // (operands as bytes; what a box reaches past K, M or N arrives as zeros)
  if ((r = b200::make_tmap_2d(&tmA, b200::DT_U8, a_q, K / 2, M, lda, 128, 128, b200::SWZ_128))) return r;
  if ((r = b200::make_tmap_2d(&tmB, b200::DT_U8, b_q, K / 2, N, ldb, 128, BN / 2, b200::SWZ_128))) return r;
  const int kg = (K + 127) / 128, atoms = (BN + 127) / 128;
  const long long a_rows = (long long)((M + 127) / 128) * kg, b_rows = (long long)((N + BN - 1) / BN) * kg * atoms;
  if ((r = b200::make_tmap_2d(&tmSFA, b200::DT_I32, sfa, 128, a_rows, 512, 128, 2, b200::SWZ_NONE))) return r;
  if ((r = b200::make_tmap_2d(&tmSFB, b200::DT_I32, sfb, 128, b_rows, 512, 128, 2 * atoms, b200::SWZ_NONE))) return r;
  if ((r = make_out_tmap<BN>(&tmD, &tmDt, d, M, N, ldd, epi.out_f32))) return r;
  PairParams p = {};
  p.M = M; p.N = N; p.K = K;
  p.group_m = raster_group_m();    // (rows of half the bytes: groups twice as tall as the 8-bit kernels', 16384 x 28672 x 4096 829 -> 815 us)
  p.epi = epi;
  p.status = b200::status_ptr();
  return launch_pair<KIND_MXFP4, BN, 1, 1>(tmA, tmB, tmSFA, tmSFB, tmD, tmDt, p, stream, "gemm_mxfp4", nullptr, (float*)ws, ws_bytes, d, ldd);
}

}  // namespace

// N tile of the kernel for an output width N: the B operand's scales are laid out for it.
B200_API int b200_gemm_mxfp4_bn(int N) { return N <= 128 ? 128 : 192; }

// Workspace (bytes, 16-byte aligned) with which b200_gemm_mxfp4 splits the last wave along K; 0 where that does not pay.
B200_API long long b200_gemm_mxfp4_workspace(int M, int N, int K) {
  using namespace gemmcore;
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  int rc = 0;
  return b200_gemm_mxfp4_bn(N) == 192 ? split_bytes<192>(pair_split<KIND_MXFP4, 192, 1>(M, N, K, rc))
                                      : split_bytes<128>(pair_split<KIND_MXFP4, 128, 1>(M, N, K, rc));
}

// a_q [M, K / 2], b_q [N, K / 2] bytes with row pitches lda / ldb (multiples of 16).  K is a multiple of 32.  workspace: null, or
// b200_gemm_mxfp4_workspace(M, N, K) bytes that nothing else uses until this call's work is done.
B200_API int b200_gemm_mxfp4(const void* a_q, const void* sfa, const void* b_q, const void* sfb, void* d, int M, int N, int K,
                             long long lda, long long ldb, long long ldd, int out_f32, int accumulate, const void* bias,
                             const void* residual, long long ldr, float alpha, void* workspace, long long workspace_bytes, void* stream) {
  if (M <= 0 || N <= 0 || K <= 0) return b200::fail(850, "gemm_mxfp4: empty problem %d x %d x %d", M, N, K);
  if (K % 32 != 0) return b200::fail(851, "gemm_mxfp4: K=%d must be a multiple of 32", K);
  gemmcore::EpiArgs epi = {};
  epi.M = M; epi.N = N;
  epi.out_f32 = out_f32 ? 1 : 0; epi.accumulate = accumulate ? 1 : 0;
  epi.bias = (const __nv_bfloat16*)bias;
  epi.residual = (const __nv_bfloat16*)residual;
  epi.ldr = ldr;
  epi.alpha = alpha;
  if (b200_gemm_mxfp4_bn(N) == 192)
    return run<192>(a_q, sfa, b_q, sfb, d, M, N, K, lda, ldb, ldd, epi, workspace, workspace_bytes, (cudaStream_t)stream);
  return run<128>(a_q, sfa, b_q, sfb, d, M, N, K, lda, ldb, ldd, epi, workspace, workspace_bytes, (cudaStream_t)stream);
}
