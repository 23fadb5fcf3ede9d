// MXFP4 quantisation: bf16 [R, C] -> e2m1 codes (two per byte) + one UE8M0 scale per 32 elements along the contraction, in the layouts that
// the block-scaled GEMM reads (gemm_mxfp4.cu), and the way back from codes to values.
//
//   q_row [R, C / 2]    scaled along the columns;     sf_row: atoms of `row_tile`
//   q_col [C, Rp / 2]   scaled along the rows, transposed, Rp = R filled up with zeros to a multiple of 32;   sf_col: atoms of `col_tile`
//
// Rounding to nearest even, or stochastically from a given byte per element (mx_quant.cuh).  With `hadamard` the column copy is that of
// H x, H the orthonormal 16 x 16 Hadamard matrix along the (filled up) rows: (H a)^T (H b) = a^T b, while a column's outlier is spread over
// sixteen values before they share a scale.
#include "mx_quant.cuh"
#include "runtime.h"

namespace {

// Codes to values: a thread holds eight neighbouring elements.  out_f32: 0 bf16, 1 fp32.
template <int FMT>
__global__ void __launch_bounds__(256)
mx_dequant_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ sf, void* __restrict__ out, long long R, int K, int tile_rows,
                  int out_f32) {
  b200::begin_kernel();
  const int vecs = K >> 3;
  const long long n = R * vecs;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
    const long long r = i / vecs;
    const int v = (int)(i - r * vecs);
    const uint32_t e = sf[mxq::sf_offset(r, v >> 2, tile_rows, (tile_rows + 127) >> 7, (K + 127) >> 7)];
    const float s = e == 255u ? __uint_as_float(0x7fffffffu) : e == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(e << 23);
    float f[8];
    if constexpr (FMT == mxq::E4M3) {
      const uint2 c = *reinterpret_cast<const uint2*>(q + i * 8);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)((j < 2 ? c.x : c.y) >> (16 * (j & 1))), __NV_E4M3);
        const float2 g = __half22float2(*reinterpret_cast<const __half2*>(&h));
        f[2 * j] = g.x * s;
        f[2 * j + 1] = g.y * s;
      }
    } else {
      const uint32_t c = *reinterpret_cast<const uint32_t*>(q + i * 4);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        // magnitudes 0, 0.5, 1, 1.5, 2, 3, 4, 6: code m >= 2 is (1 + (m & 1) / 2) * 2^(m / 2 - 1)
        const uint32_t m = (c >> (4 * j)) & 7u, sign = ((c >> (4 * j)) & 8u) << 28;
        const uint32_t b = m >= 2u ? ((126u + (m >> 1)) << 23 | (m & 1u) << 22) : m * 0x3f000000u;
        f[j] = __uint_as_float(b | sign) * s;
      }
    }
    if (out_f32) {
      float4* o = reinterpret_cast<float4*>((float*)out + i * 8);
      o[0] = make_float4(f[0], f[1], f[2], f[3]);
      o[1] = make_float4(f[4], f[5], f[6], f[7]);
    } else {
      reinterpret_cast<uint4*>(out)[i] = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
    }
  }
}

}  // namespace

// x: bf16 [R, C], row pitch ldx (elements), 16-byte aligned; C a multiple of 32.  Either copy may be null.  noise: null, or bytes [R, C]
// (dense, 8-byte aligned); rows past R count as 128.
B200_API int b200_quant_mxfp4(const void* x, long long ldx, int R, int C, const void* noise, int hadamard, void* q_row, void* sf_row,
                              int row_tile, void* q_col, void* sf_col, int col_tile, void* stream) {
  if (R <= 0 || C <= 0 || C % 32 != 0) return b200::fail(720, "quant_mxfp4: R=%d must be positive and C=%d a positive multiple of 32", R, C);
  if (ldx % 8 != 0 || ((uintptr_t)x & 15) != 0) return b200::fail(721, "quant_mxfp4: input must be 16-byte aligned");
  if (((uintptr_t)noise & 7) != 0) return b200::fail(722, "quant_mxfp4: noise must be 8-byte aligned");
  if ((q_row && (row_tile <= 0 || row_tile % 16 != 0)) || (q_col && (col_tile <= 0 || col_tile % 16 != 0)))
    return b200::fail(723, "quant_mxfp4: tile rows must be positive multiples of 16");
  if (R > 65535 * mxq::TILE) return b200::fail(724, "quant_mxfp4: R=%d rows are more than a launch covers", R);
  mxq::TileArgs p = {};
  p.x = (const __nv_bfloat16*)x; p.ldx = ldx; p.R = R; p.C = C;
  p.noise = (const uint8_t*)noise; p.hadamard = hadamard;
  p.q_row = (uint8_t*)q_row; p.sf_row = (uint8_t*)sf_row; p.row_tile = row_tile;
  p.q_col = (uint8_t*)q_col; p.sf_col = (uint8_t*)sf_col; p.col_tile = col_tile;
  p.Rp = (R + 31) / 32 * 32;
  const dim3 grid((C + mxq::TILE - 1) / mxq::TILE, (R + mxq::TILE - 1) / mxq::TILE);
  if (noise != nullptr) {
    // (the tile of bytes comes on top of 36 KB of static shared memory: more than a launch gets unasked)
    static bool configured[64] = {false};
    int dev = 0;
    cudaGetDevice(&dev);
    if (!configured[dev & 63]) {
      const cudaError_t e = cudaFuncSetAttribute(mxq::mx_tile_kernel<mxq::E2M1, false, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, mxq::NOISE_WORDS * 4);
      if (e != cudaSuccess) {
        cudaGetLastError();
        return b200::fail(728, "quant_mxfp4: cannot set %d bytes of shared memory: %s", mxq::NOISE_WORDS * 4, cudaGetErrorString(e));
      }
      configured[dev & 63] = true;
    }
    b200::launch(mxq::mx_tile_kernel<mxq::E2M1, false, true>, grid, 256, mxq::NOISE_WORDS * 4, (cudaStream_t)stream, p);
  }
  else b200::launch(mxq::mx_tile_kernel<mxq::E2M1, false, false>, grid, 256, 0, (cudaStream_t)stream, p);
  b200::count_launch();
  return b200::check_launch("quant_mxfp4");
}

// Values of an operand: q [R, K] e4m3 (fmt 0) or [R, K / 2] e2m1 (fmt 1) codes, dense; out [R, K] bf16 or fp32, dense.
B200_API int b200_dequant_mx(const void* q, const void* sf, void* out, long long R, int K, int tile_rows, int fmt, int out_f32, void* stream) {
  if (R <= 0 || K <= 0 || K % 32 != 0) return b200::fail(725, "dequant_mx: R=%lld must be positive and K=%d a positive multiple of 32", R, K);
  if (tile_rows <= 0 || tile_rows % 16 != 0) return b200::fail(726, "dequant_mx: tile rows must be positive multiples of 16");
  if ((((uintptr_t)q | (uintptr_t)out) & 15) != 0) return b200::fail(727, "dequant_mx: codes and output must be 16-byte aligned");
  const long long blocks = (R * (K / 8) + 255) / 256, most = b200::sm_count() * 32ll;
  const dim3 grid((unsigned)(blocks < most ? blocks : most));
  if (fmt == mxq::E4M3) b200::launch(mx_dequant_kernel<mxq::E4M3>, grid, 256, 0, (cudaStream_t)stream, (const uint8_t*)q, (const uint8_t*)sf, out, R, K, tile_rows, out_f32);
  else b200::launch(mx_dequant_kernel<mxq::E2M1>, grid, 256, 0, (cudaStream_t)stream, (const uint8_t*)q, (const uint8_t*)sf, out, R, K, tile_rows, out_f32);
  b200::count_launch();
  return b200::check_launch("dequant_mx");
}
