// RMS norm with a micro-scaled output:
//
//   h = bf16(x + residual) (or x),  rstd = rsqrt(mean(h^2) + eps),  n = h * rstd * w
//
// and n leaves as e4m3 codes with one UE8M0 scale per 32 values: along the columns (the A operand of the linear that follows), along the
// rows and transposed (the B operand of that linear's weight gradient), or both.  n itself, rounded to nothing in between, is never written:
// against the norm and the quantiser by themselves a pass writes 2 and reads 2 bytes a value less.
#include "mx_quant.cuh"
#include "runtime.h"

namespace {

constexpr int MAX_D = 8192;

struct NormMxArgs {
  const __nv_bfloat16* x;
  const __nv_bfloat16* res;       // or null
  const __nv_bfloat16* w;
  __nv_bfloat16* h;               // written when there is a residual
  float* rstd;
  int T, D;
  float eps;
  uint8_t* q_row; uint8_t* sf_row; int row_tile;      // or null
};

// NT threads hold a row, four 16-byte vectors each; a CTA of 256 threads has 256 / NT rows.
template <int NT>
__global__ void __launch_bounds__(256)
norm_mx_rows_kernel(const NormMxArgs p) {
  b200::begin_kernel();
  __shared__ float red[8];
  const int t = threadIdx.x % NT, team = threadIdx.x / NT, warp = threadIdx.x >> 5;
  const long long row = (long long)blockIdx.x * (256 / NT) + team;
  const bool live = row < p.T;
  uint4 v[4];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = (t + i * NT) * 8;
    v[i] = make_uint4(0u, 0u, 0u, 0u);
    if (live && c < p.D) v[i] = *reinterpret_cast<const uint4*>(p.x + row * p.D + c);
  }
  if (p.res != nullptr) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = (t + i * NT) * 8;
      if (live && c < p.D) {
        const uint4 u = *reinterpret_cast<const uint4*>(p.res + row * p.D + c);
        const float2 a0 = unpack_bf16x2(v[i].x), a1 = unpack_bf16x2(v[i].y), a2 = unpack_bf16x2(v[i].z), a3 = unpack_bf16x2(v[i].w);
        const float2 b0 = unpack_bf16x2(u.x), b1 = unpack_bf16x2(u.y), b2 = unpack_bf16x2(u.z), b3 = unpack_bf16x2(u.w);
        v[i] = make_uint4(pack_bf16x2(a0.x + b0.x, a0.y + b0.y), pack_bf16x2(a1.x + b1.x, a1.y + b1.y),
                          pack_bf16x2(a2.x + b2.x, a2.y + b2.y), pack_bf16x2(a3.x + b3.x, a3.y + b3.y));
        *reinterpret_cast<uint4*>(p.h + row * p.D + c) = v[i];      // what is normalised is the stored (rounded) sum
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 a0 = unpack_bf16x2(v[i].x), a1 = unpack_bf16x2(v[i].y), a2 = unpack_bf16x2(v[i].z), a3 = unpack_bf16x2(v[i].w);
    ss += a0.x * a0.x + a0.y * a0.y + a1.x * a1.x + a1.y * a1.y + a2.x * a2.x + a2.y * a2.y + a3.x * a3.x + a3.y * a3.y;
  }
  ss = warp_sum(ss);
  if constexpr (NT > 32) {
    if ((threadIdx.x & 31) == 0) red[warp] = ss;
    __syncthreads();
    ss = 0.f;
#pragma unroll
    for (int i = 0; i < NT / 32; ++i) ss += red[team * (NT / 32) + i];
  }
  const float rstd = rsqrtf(ss / p.D + p.eps);
  if (t == 0 && live) p.rstd[row] = rstd;
  if (p.q_row == nullptr) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int vi = t + i * NT, c = vi * 8;
    const uint4 u = c < p.D ? *reinterpret_cast<const uint4*>(p.w + c) : make_uint4(0u, 0u, 0u, 0u);
    const float2 a0 = unpack_bf16x2(v[i].x), a1 = unpack_bf16x2(v[i].y), a2 = unpack_bf16x2(v[i].z), a3 = unpack_bf16x2(v[i].w);
    const float2 b0 = unpack_bf16x2(u.x), b1 = unpack_bf16x2(u.y), b2 = unpack_bf16x2(u.z), b3 = unpack_bf16x2(u.w);
    float n[8] = {a0.x * rstd * b0.x, a0.y * rstd * b0.y, a1.x * rstd * b1.x, a1.y * rstd * b1.y,
                  a2.x * rstd * b2.x, a2.y * rstd * b2.y, a3.x * rstd * b3.x, a3.y * rstd * b3.y};
    if (c >= p.D) {
#pragma unroll
      for (int j = 0; j < 8; ++j) n[j] = 0.f;        // (an infinite rstd does not reach the padding)
    }
    uint2 q;
    uint32_t e = mxq::quant_row8<mxq::E4M3>(n, nullptr, q);
    if (live && c < p.D) *reinterpret_cast<uint2*>(p.q_row + row * p.D + c) = q;
    // the four scale bytes of a 128-column group, from lanes 0, 4, 8, 12 of its sixteen
    const int base = threadIdx.x & 16;
    uint32_t word = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) word |= __shfl_sync(0xffffffffu, e, base + 4 * j) << (8 * j);
    if (live && (vi & 15) == 0 && c < p.D) {
      const long long o = mxq::sf_offset(row, vi >> 2, p.row_tile, (p.row_tile + 127) >> 7, (p.D + 127) >> 7);
      *reinterpret_cast<uint32_t*>(p.sf_row + o) = word;
    }
  }
}

}  // namespace

// x, residual (or null), w: bf16, dense [T, D] / [D], 16-byte aligned; D a multiple of 32 up to 8192.  h [T, D]: written when there is a
// residual.  rstd [T].  Copies: q_row [T, D] with scales in atoms of row_tile, q_col [D, Tp] (Tp = T filled up with zeros to a multiple of
// 128) with scales in atoms of col_tile; either may be null.
B200_API int b200_norm_mx(const void* x, const void* residual, const void* w, void* h, void* rstd, int T, int D, float eps, void* q_row,
                          void* sf_row, int row_tile, void* q_col, void* sf_col, int col_tile, void* stream) {
  if (T <= 0 || D <= 0 || D % 32 != 0 || D > MAX_D)
    return b200::fail(730, "norm_mx: T=%d must be positive and D=%d a multiple of 32 up to %d", T, D, MAX_D);
  if ((((uintptr_t)x | (uintptr_t)residual | (uintptr_t)w | (uintptr_t)h) & 15) != 0)
    return b200::fail(731, "norm_mx: operands must be 16-byte aligned");
  if ((q_row && (row_tile <= 0 || row_tile % 16 != 0)) || (q_col && (col_tile <= 0 || col_tile % 16 != 0)))
    return b200::fail(732, "norm_mx: tile rows must be positive multiples of 16");
  if (residual != nullptr && h == nullptr) return b200::fail(733, "norm_mx: a residual needs a place for the sum");
  if (T > 65535 * mxq::TILE) return b200::fail(734, "norm_mx: T=%d rows are more than a launch covers", T);
  NormMxArgs p = {(const __nv_bfloat16*)x, (const __nv_bfloat16*)residual, (const __nv_bfloat16*)w, (__nv_bfloat16*)h, (float*)rstd, T, D, eps,
                  (uint8_t*)q_row, (uint8_t*)sf_row, row_tile};
  cudaStream_t st = (cudaStream_t)stream;
  if (D <= 1024) b200::launch(norm_mx_rows_kernel<32>, dim3((T + 7) / 8), 256, 0, st, p);
  else if (D <= 2048) b200::launch(norm_mx_rows_kernel<64>, dim3((T + 3) / 4), 256, 0, st, p);
  else if (D <= 4096) b200::launch(norm_mx_rows_kernel<128>, dim3((T + 1) / 2), 256, 0, st, p);
  else b200::launch(norm_mx_rows_kernel<256>, dim3(T), 256, 0, st, p);
  b200::count_launch();
  int r = b200::check_launch("norm_mx");
  if (r || q_col == nullptr) return r;
  mxq::TileArgs q = {};
  q.x = residual != nullptr ? (const __nv_bfloat16*)h : (const __nv_bfloat16*)x;
  q.ldx = D; q.R = T; q.C = D;
  q.rstd = (const float*)rstd; q.w = (const __nv_bfloat16*)w;
  q.q_col = (uint8_t*)q_col; q.sf_col = (uint8_t*)sf_col; q.col_tile = col_tile;
  q.Rp = (T + 127) / 128 * 128;
  b200::launch(mxq::mx_tile_kernel<mxq::E4M3, true, false, false>, dim3((D + 127) / 128, (T + 127) / 128), 256, 0, st, q);
  b200::count_launch();
  return b200::check_launch("norm_mx(columns)");
}
