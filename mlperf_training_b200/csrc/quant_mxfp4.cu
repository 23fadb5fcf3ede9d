// MXFP4 quantisation: bf16 [R, C] -> e2m1 codes (two per byte) + one UE8M0 scale per 32 elements along the contraction, in the layouts that
// the block-scaled GEMM reads (gemm_mxfp4.cu), and the way back from codes to values.
//
//   q_row [R, C / 2]    scaled along the columns;     sf_row: atoms of `row_tile`
//   q_col [C, Rp / 2]   scaled along the rows, transposed, Rp = R filled up with zeros to a multiple of 32;   sf_col: atoms of `col_tile`
//
// Rounding to nearest even, or stochastically from a given byte per element (mx_quant.cuh).  With `hadamard` the column copy is that of
// H x, H the orthonormal 16 x 16 Hadamard matrix along the (filled up) rows: (H a)^T (H b) = a^T b, while a column's outlier is spread over
// sixteen values before they share a scale.
//
// Measured (caches cold): 14336 x 4096, both copies 38 us (181 MB: 4.8 TB/s), the row copy of 16384 x 4096 29 us (5.9 TB/s); 4011 x 14336, both
// copies, with bytes and transform 68 us (236 MB).  Back to bf16: 58.7 M values of e2m1 31 us (4.8 TB/s), 67 M of e4m3 36 us (5.7 TB/s).
#include "mx_quant.cuh"
#include "runtime.h"

namespace {

// Codes to values, written to bf16 or fp32.  A lane has eight neighbouring elements, a warp eight (e4m3: four) consecutive rows: their
// scale bytes are 16 bytes apart in one atom (tile rows are multiples of 16), so one division places all of them, and as many loads of each
// kind are in flight (e4m3 with eight 43 us for 67 M values, with four 39; e2m1 with four 37 for 59 M, with eight 35).
// An e2m1 code becomes a bf16 by two table look-ups of its bytes (prmt) and its sign; the product with the scale, a power of two, is exact.

B200_DEVICE uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }
// elements 0, 1 and 2, 3 of four codes in the low half of c, as bf16 pairs
B200_DEVICE void e2m1x4_bf16(uint32_t c, uint32_t& w01, uint32_t& w23) {
  const uint32_t m = c & 0x7777u;
  const uint32_t lo = prmt(0xc0800000u, 0xc0804000u, m), hi = prmt(0x3f3f3f00u, 0x40404040u, m);   // 0 .5 1 1.5 | 2 3 4 6
  w01 = prmt(lo, hi, 0x5140u) | (c << 12 & 0x8000u) | (c << 24 & 0x80000000u);
  w23 = prmt(lo, hi, 0x7362u) | (c << 4 & 0x8000u) | (c << 16 & 0x80000000u);
}
B200_DEVICE uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

template <int FMT>
constexpr int DQ_ROWS = FMT == mxq::E4M3 ? 4 : 8;

template <int FMT, bool F32>
__global__ void __launch_bounds__(256)
mx_dequant_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ sf, void* __restrict__ out, int R, int K, int tile_rows) {
  b200::begin_kernel();
  constexpr int ROWS = DQ_ROWS<FMT>;
  const int vecs = K >> 3;
  const int v = blockIdx.x * 32 + (threadIdx.x & 31);
  if (v >= vecs) return;
  for (long long r0 = ((long long)blockIdx.y * 8 + (threadIdx.x >> 5)) * ROWS; r0 < R; r0 += (long long)gridDim.y * 8 * ROWS) {
    const uint8_t* s0 = sf + mxq::sf_offset(r0, v >> 2, tile_rows, (tile_rows + 127) >> 7, (K + 127) >> 7);
    uint32_t e[ROWS];
    uint2 c[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const bool in = r0 + i < R;
      e[i] = in ? s0[i * 16] : 0u;
      c[i] = make_uint2(0u, 0u);
      if (in) {
        if constexpr (FMT == mxq::E4M3) c[i] = *reinterpret_cast<const uint2*>(q + (r0 + i) * K + v * 8);
        else c[i].x = *reinterpret_cast<const uint32_t*>(q + (((r0 + i) * K) >> 1) + v * 4);
      }
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      if (r0 + i >= R) break;
      // 2^(e - 127) as bf16: 0 is 2^-127, below the normal numbers; 255 is a NaN
      const uint32_t sb = e[i] == 255u ? 0x7fc0u : e[i] == 0u ? 0x0040u : e[i] << 7;
      const float s = __uint_as_float(sb << 16);
      const long long at = (r0 + i) * K + v * 8;
      float f[8];
      uint32_t w[4];
      if constexpr (FMT == mxq::E4M3) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)((j < 2 ? c[i].x : c[i].y) >> (16 * (j & 1))), __NV_E4M3);
          const float2 g = __half22float2(*reinterpret_cast<const __half2*>(&h));
          f[2 * j] = g.x * s;
          f[2 * j + 1] = g.y * s;
          if constexpr (!F32) w[j] = pack_bf16x2(f[2 * j], f[2 * j + 1]);
        }
      } else {
        e2m1x4_bf16(c[i].x, w[0], w[1]);
        e2m1x4_bf16(c[i].x >> 16, w[2], w[3]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (F32) {
            const float2 g = unpack_bf16x2(w[j]);
            f[2 * j] = g.x * s;
            f[2 * j + 1] = g.y * s;
          } else {
            w[j] = mul_bf16x2(w[j], sb | sb << 16);
          }
        }
      }
      if constexpr (F32) {
        float4* o = reinterpret_cast<float4*>((float*)out + at);
        o[0] = make_float4(f[0], f[1], f[2], f[3]);
        o[1] = make_float4(f[4], f[5], f[6], f[7]);
      } else {
        *reinterpret_cast<uint4*>((__nv_bfloat16*)out + at) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
}

template <int FMT>
void launch_dequant(dim3 grid, cudaStream_t st, const void* q, const void* sf, void* out, int R, int K, int tile_rows, int out_f32) {
  if (out_f32) b200::launch(mx_dequant_kernel<FMT, true>, grid, 256, 0, st, (const uint8_t*)q, (const uint8_t*)sf, out, R, K, tile_rows);
  else b200::launch(mx_dequant_kernel<FMT, false>, grid, 256, 0, st, (const uint8_t*)q, (const uint8_t*)sf, out, R, K, tile_rows);
}

template <bool NOISE, bool HAD>
int launch_tile(dim3 grid, cudaStream_t st, const mxq::TileArgs& p) {
  const auto kern = mxq::mx_tile_kernel<NOISE, HAD>;
  const int dyn = NOISE ? mxq::NOISE_WORDS * 4 : 0;
  if (NOISE) {
    // (the tile of bytes comes on top of 36 KB of static shared memory: more than a launch gets unasked)
    static bool configured[64] = {false};
    int dev = 0;
    cudaGetDevice(&dev);
    if (!configured[dev & 63]) {
      const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, dyn);
      if (e != cudaSuccess) {
        cudaGetLastError();
        return b200::fail(728, "quant_mxfp4: cannot set %d bytes of shared memory: %s", dyn, cudaGetErrorString(e));
      }
      configured[dev & 63] = true;
    }
  }
  b200::launch(kern, grid, 256, dyn, st, p);
  return 0;
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
  p.noise = (const uint8_t*)noise;
  p.q_row = (uint8_t*)q_row; p.sf_row = (uint8_t*)sf_row; p.row_tile = row_tile;
  p.q_col = (uint8_t*)q_col; p.sf_col = (uint8_t*)sf_col; p.col_tile = col_tile;
  p.Rp = (R + 31) / 32 * 32;
  const dim3 grid((C + mxq::TILE - 1) / mxq::TILE, (R + mxq::TILE - 1) / mxq::TILE);
  int r;
  if (noise != nullptr) r = hadamard ? launch_tile<true, true>(grid, (cudaStream_t)stream, p) : launch_tile<true, false>(grid, (cudaStream_t)stream, p);
  else r = hadamard && q_col != nullptr ? launch_tile<false, true>(grid, (cudaStream_t)stream, p) : launch_tile<false, false>(grid, (cudaStream_t)stream, p);
  if (r) return r;
  b200::count_launch();
  return b200::check_launch("quant_mxfp4");
}

// Values of an operand: q [R, K] e4m3 (fmt 0) or [R, K / 2] e2m1 (fmt 1) codes, dense; out [R, K] bf16 or fp32, dense.
B200_API int b200_dequant_mx(const void* q, const void* sf, void* out, int R, int K, int tile_rows, int fmt, int out_f32, void* stream) {
  if (R <= 0 || K <= 0 || K % 32 != 0) return b200::fail(725, "dequant_mx: R=%d must be positive and K=%d a positive multiple of 32", R, K);
  if (tile_rows <= 0 || tile_rows % 16 != 0) return b200::fail(726, "dequant_mx: tile rows must be positive multiples of 16");
  if ((((uintptr_t)q | (uintptr_t)out) & 15) != 0) return b200::fail(727, "dequant_mx: codes and output must be 16-byte aligned");
  const int per = 8 * (fmt == mxq::E4M3 ? DQ_ROWS<mxq::E4M3> : DQ_ROWS<mxq::E2M1>), rows = (R - 1) / per + 1;
  const dim3 grid((K / 8 + 31) / 32, rows < 65535 ? rows : 65535);
  if (fmt == mxq::E4M3) launch_dequant<mxq::E4M3>(grid, (cudaStream_t)stream, q, sf, out, R, K, tile_rows, out_f32);
  else launch_dequant<mxq::E2M1>(grid, (cudaStream_t)stream, q, sf, out, R, K, tile_rows, out_f32);
  b200::count_launch();
  return b200::check_launch("dequant_mx");
}
