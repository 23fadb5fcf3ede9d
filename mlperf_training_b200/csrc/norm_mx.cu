// RMS norm with a micro-scaled output:
//
//   h = bf16(x + residual) (or x),  rstd = rsqrt(mean(h^2) + eps),  n = (h * w) * rstd
//
// and n leaves as e4m3 codes with one UE8M0 scale per 32 values: along the columns (the A operand of the linear that follows), along the
// rows and transposed (the B operand of that linear's weight gradient), or both.  n itself, rounded once to fp32 in between, is never written:
// against the norm and the quantiser by themselves a pass writes 2 and reads 2 bytes a value less.
//
// Measured (caches cold): 16384 x 4096 with a residual, both copies 100 us (541 MB: 5.4 TB/s); a row of 4096 4.6 us, 1337 rows of 2880 8 us.
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

// Sums of bf16 pairs, rounded once; what is normalised is the stored (rounded) sum.
B200_DEVICE uint32_t add2(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hadd2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
B200_DEVICE uint4 add8(const uint4& a, const uint4& b) { return make_uint4(add2(a.x, b.x), add2(a.y, b.y), add2(a.z, b.z), add2(a.w, b.w)); }
B200_DEVICE float2 sumsq8(const uint4& u, float2 s) {
  const float2 a = unpack_bf16x2(u.x), b = unpack_bf16x2(u.y), c = unpack_bf16x2(u.z), d = unpack_bf16x2(u.w);
  return ffma2(d, d, ffma2(c, c, ffma2(b, b, ffma2(a, a, s))));
}
// h * w of eight values: exact in fp32 (two factors of eight bits), so n = (h w) rstd is rounded once
B200_DEVICE void mul8(const uint4& h, const uint4& w, float2 (&z)[4]) {
  z[0] = fmul2(unpack_bf16x2(h.x), unpack_bf16x2(w.x));
  z[1] = fmul2(unpack_bf16x2(h.y), unpack_bf16x2(w.y));
  z[2] = fmul2(unpack_bf16x2(h.z), unpack_bf16x2(w.z));
  z[3] = fmul2(unpack_bf16x2(h.w), unpack_bf16x2(w.w));
}

// The row copy alone.  A warp holds 512 columns of a row, two 16-byte vectors a lane: NT = 32, 64, .. 512 threads a row, 256 / NT rows a CTA.
// The squares are added up in the order of the kernel below (lane, warp, then 512-column pieces in order), so a row has the same codes
// whether the column copy is made with it or not.
template <int NT>
__global__ void __launch_bounds__(NT > 256 ? NT : 256)
norm_mx_rows_kernel(const NormMxArgs p) {
  b200::begin_kernel();
  constexpr int CTA = NT > 256 ? NT : 256;
  __shared__ float red[CTA / 32];
  const int t = threadIdx.x % NT, team = threadIdx.x / NT, lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * (CTA / NT) + team;
  const bool live = row < p.T;
  const int c0 = (t >> 5) * 512 + lane * 8;
  const long long at = row * p.D + c0;
  const bool in[2] = {c0 < p.D, c0 + 256 < p.D};
  uint4 v[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) v[j] = live && in[j] ? *reinterpret_cast<const uint4*>(p.x + at + j * 256) : make_uint4(0u, 0u, 0u, 0u);
  if (p.res != nullptr) {
    uint4 u[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) u[j] = live && in[j] ? *reinterpret_cast<const uint4*>(p.res + at + j * 256) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      v[j] = add8(v[j], u[j]);
      if (live && in[j]) *reinterpret_cast<uint4*>(p.h + at + j * 256) = v[j];
    }
  }
  const float2 s2 = sumsq8(v[1], sumsq8(v[0], make_float2(0.f, 0.f)));
  float ss = warp_sum(s2.x + s2.y);
  if constexpr (NT > 32) {
    if (lane == 0) red[threadIdx.x >> 5] = ss;
    __syncthreads();
    ss = 0.f;
#pragma unroll
    for (int i = 0; i < NT / 32; ++i) ss += red[team * (NT / 32) + i];
  }
  const float rstd = __frsqrt_rn(ss / p.D + p.eps);
  if (t == 0 && live) p.rstd[row] = rstd;
  if (p.q_row == nullptr) return;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int c = c0 + j * 256;
    float2 z[4];
    mul8(v[j], in[j] ? *reinterpret_cast<const uint4*>(p.w + c) : make_uint4(0u, 0u, 0u, 0u), z);
    uint2 q;
    uint32_t e = mxq::quant_row8_e4m3(z, rstd, q);
    if (!in[j]) e = 0u;                              // (an infinite rstd does not reach the padding)
    if (live && in[j]) *reinterpret_cast<uint2*>(p.q_row + at + j * 256) = q;
    // the four scale bytes of a 128-column group, from lanes 0, 4, 8, 12 of its sixteen
    uint32_t word = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) word |= __shfl_sync(0xffffffffu, e, (lane & 16) + 4 * k) << (8 * k);
    if (live && (lane & 15) == 0 && in[j]) {
      const long long o = mxq::sf_offset(row, c >> 5, p.row_tile, (p.row_tile + 127) >> 7, (p.D + 127) >> 7);
      *reinterpret_cast<uint32_t*>(p.sf_row + o) = word;
    }
  }
}

// Both copies (or the column copy) in one pass over the input.  A cluster of CTAs owns 32 rows, each CTA COLS columns of them: 32 rows are one
// block of the column copy's scales, and rows as wide as 8192 stay on chip as one piece.
//   * a warp loads four rows x 512 columns, two at a time, adds the residual and puts the sums into shared memory;
//   * the CTAs' partial sums of squares meet over distributed shared memory, in rank order: every CTA has the same rstd, and runs are
//     bit-reproducible;
//   * h and the row copy leave as the rows were loaded; for the column copy two lanes walk two columns, 16 rows each, and write 16 codes of
//     either.
// 33 KB a CTA (512 columns), so that several CTAs of an SM cover one another's barrier.  With 128-row tiles the columns' codes would leave as
// whole 128-byte lines, but a CTA would hold 130 KB and its load, barrier and compute phases would stand alone; the 32-byte pieces of four
// neighbouring clusters meet in L2.
struct NormMxCols {
  uint8_t* q_col; uint8_t* sf_col; int col_tile;
  int Tp;
};

template <int COLS>
struct ClusterCfg {
  static constexpr int PITCH_W = COLS / 2 + 4;                   // words; 16 more from row 16 on: the two lanes of a column lie 16 banks apart
  static constexpr int SMEM = (32 * PITCH_W + 16) * 4;
};
B200_DEVICE float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

template <int COLS>
__global__ void __launch_bounds__(COLS / 2, 2048 / COLS)
norm_mx_cluster_kernel(const NormMxArgs p, const NormMxCols o) {
  b200::begin_kernel();
  using C = ClusterCfg<COLS>;
  constexpr int HALVES = COLS / 512, MAX_CTAS = 8;
  extern __shared__ __align__(16) uint32_t tile[];
  __shared__ float part[HALVES][32];
  __shared__ float rstd_s[32];
  __shared__ __align__(4) uint8_t sfs[32][COLS / 32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = (int)cluster_ctarank(), ctas = gridDim.y;     // (the cluster spans the grid's y)
  const long long r0 = (long long)blockIdx.x * 32;
  const int c_cta = rank * COLS, rr0 = (warp & 7) * 4, cc = (warp >> 3) * 512 + lane * 8;
  const int rows = (int)min(32ll, p.T - r0), live = rows - rr0;              // (a warp's rows past T: live <= 0)
  const bool in0 = c_cta + cc < p.D, in1 = c_cta + cc + 256 < p.D;
  const long long at = (r0 + rr0) * p.D + c_cta + cc;
  uint32_t* const tw = tile + rr0 * C::PITCH_W + (rr0 >> 4) * 16 + cc / 2;      // (a warp's four rows are on one side of row 16)
#pragma unroll 1
  for (int i = 0; i < 4; i += 2) {
    uint4 v[2][2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const __nv_bfloat16* src = p.x + at + (i + k) * (long long)p.D;
      v[k][0] = i + k < live && in0 ? *reinterpret_cast<const uint4*>(src) : make_uint4(0u, 0u, 0u, 0u);
      v[k][1] = i + k < live && in1 ? *reinterpret_cast<const uint4*>(src + 256) : make_uint4(0u, 0u, 0u, 0u);
    }
    if (p.res != nullptr) {
      uint4 u[2][2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const __nv_bfloat16* src = p.res + at + (i + k) * (long long)p.D;
        u[k][0] = i + k < live && in0 ? *reinterpret_cast<const uint4*>(src) : make_uint4(0u, 0u, 0u, 0u);
        u[k][1] = i + k < live && in1 ? *reinterpret_cast<const uint4*>(src + 256) : make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) { v[k][0] = add8(v[k][0], u[k][0]); v[k][1] = add8(v[k][1], u[k][1]); }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      *reinterpret_cast<uint4*>(tw + (i + k) * C::PITCH_W) = v[k][0];
      *reinterpret_cast<uint4*>(tw + (i + k) * C::PITCH_W + 128) = v[k][1];
      const float2 s2 = sumsq8(v[k][1], sumsq8(v[k][0], make_float2(0.f, 0.f)));
      const float ss = warp_sum(s2.x + s2.y);
      if (lane == 0) part[warp >> 3][rr0 + i + k] = ss;
    }
  }
  cluster_sync_all();
  if (tid < 32) {
    float f[MAX_CTAS][HALVES];
#pragma unroll
    for (int q = 0; q < MAX_CTAS; ++q)
#pragma unroll
      for (int h = 0; h < HALVES; ++h) f[q][h] = q < ctas ? ld_cluster_f32(mapa_u32(smem_u32(&part[h][tid]), q)) : 0.f;
    float ss = 0.f;
#pragma unroll
    for (int q = 0; q < MAX_CTAS; ++q)
#pragma unroll
      for (int h = 0; h < HALVES; ++h) ss += f[q][h];
    const bool live = r0 + tid < p.T;
    const float rstd = live ? __frsqrt_rn(ss / p.D + p.eps) : 0.f;
    rstd_s[tid] = rstd;
    if (live && rank == 0) p.rstd[r0 + tid] = rstd;
  }
  __syncthreads();
  // (this CTA has read its peers' sums; they may leave once all have)
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  // h and the row copy, from the warp's own part of the tile (h leaves only now: a release waits for the stores before it)
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const bool in = j ? in1 : in0;
    const uint4 w = in ? *reinterpret_cast<const uint4*>(p.w + c_cta + cc + j * 256) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll 2
    for (int i = 0; i < 4; ++i) {
      const uint4 v = *reinterpret_cast<const uint4*>(tw + i * C::PITCH_W + j * 128);
      const long long to = at + i * (long long)p.D + j * 256;
      if (p.res != nullptr && i < live && in) *reinterpret_cast<uint4*>(p.h + to) = v;
      if (p.q_row == nullptr) continue;
      float2 z[4];
      mul8(v, w, z);
      uint2 q;
      uint32_t e = mxq::quant_row8_e4m3(z, rstd_s[rr0 + i], q);
      if (!in) e = 0u;                               // (an infinite rstd does not reach the padding)
      if (i < live && in) *reinterpret_cast<uint2*>(p.q_row + to) = q;
      if ((lane & 3) == 0) sfs[rr0 + i][(cc + j * 256) >> 5] = (uint8_t)e;
    }
  }
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    const int sub = lane & 1, cw = pass * (COLS / 4) + warp * 16 + (lane >> 1), c = c_cta + 2 * cw;
    const bool in = c < p.D;
    const uint32_t* t = tile + sub * (16 * C::PITCH_W + 16) + cw;
    const float2 w = in ? unpack_bf16x2(*reinterpret_cast<const uint32_t*>(p.w + c)) : make_float2(0.f, 0.f);
    float2 n[16];
    float ma = 0.f, mb = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float s = rstd_s[sub * 16 + i];
      n[i] = fmul2(fmul2(unpack_bf16x2(t[i * C::PITCH_W]), w), make_float2(s, s));       // (the row copy's product, in its order)
    }
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      ma = mxq::fmax3_nan(ma, n[i].x, n[i + 1].x);
      mb = mxq::fmax3_nan(mb, n[i].y, n[i + 1].y);
    }
    uint4 qa, qb;
    uint32_t ea, eb;
    mxq::quant_col16<mxq::E4M3>(n, mxq::abs_bits(ma), mxq::abs_bits(mb), nullptr, nullptr, qa, qb, ea, eb);
    if (in) {
      uint8_t* dst = o.q_col + (long long)c * o.Tp + r0 + sub * 16;
      *reinterpret_cast<uint4*>(dst) = qa;
      *reinterpret_cast<uint4*>(dst + o.Tp) = qb;
      o.sf_col[mxq::sf_offset(c + sub, (int)(r0 >> 5), o.col_tile, (o.col_tile + 127) >> 7, o.Tp >> 7)] = (uint8_t)(sub ? eb : ea);
    }
  }
  if (p.q_row != nullptr) {
    __syncthreads();
    for (int i = tid; i < 32 * (COLS / 128); i += COLS / 2) {
      const int r = i / (COLS / 128), g = i - r * (COLS / 128);
      if (r < rows && c_cta + g * 128 < p.D) {
        const long long to = mxq::sf_offset(r0 + r, (c_cta >> 5) + g * 4, p.row_tile, (p.row_tile + 127) >> 7, (p.D + 127) >> 7);
        *reinterpret_cast<uint32_t*>(p.sf_row + to) = *reinterpret_cast<const uint32_t*>(&sfs[r][g * 4]);
      }
    }
  }
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <int COLS>
int launch_cluster(const NormMxArgs& p, const NormMxCols& o, cudaStream_t stream) {
  using C = ClusterCfg<COLS>;
  const auto kern = norm_mx_cluster_kernel<COLS>;
  if (C::SMEM > 40 * 1024) {
    static bool configured[64] = {false};
    int dev = 0;
    cudaGetDevice(&dev);
    if (!configured[dev & 63]) {
      const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
      if (e != cudaSuccess) {
        cudaGetLastError();
        return b200::fail(735, "norm_mx: cannot set %d bytes of shared memory: %s", C::SMEM, cudaGetErrorString(e));
      }
      configured[dev & 63] = true;
    }
  }
  const int ctas = (p.D + COLS - 1) / COLS;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(o.Tp / 32, ctas, 1);
  cfg.blockDim = dim3(COLS / 2, 1, 1);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1; attr[0].val.clusterDim.y = ctas; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaLaunchKernelEx(&cfg, kern, p, o);
  b200::count_launch();
  return b200::check_launch("norm_mx(cluster)");
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
  if (T > 0x7fffff00) return b200::fail(734, "norm_mx: T=%d rows cannot be filled up to a multiple of 128", T);
  NormMxArgs p = {(const __nv_bfloat16*)x, (const __nv_bfloat16*)residual, (const __nv_bfloat16*)w, (__nv_bfloat16*)h, (float*)rstd, T, D, eps,
                  (uint8_t*)q_row, (uint8_t*)sf_row, row_tile};
  cudaStream_t st = (cudaStream_t)stream;
  if (q_col != nullptr) {
    const NormMxCols o = {(uint8_t*)q_col, (uint8_t*)sf_col, col_tile, (T + 127) / 128 * 128};
    // (clusters of more than eight CTAs are not portable: wider rows take CTAs of 1024 columns)
    return D <= 4096 ? launch_cluster<512>(p, o, st) : launch_cluster<1024>(p, o, st);
  }
  if (D <= 512) b200::launch(norm_mx_rows_kernel<32>, dim3((T + 7) / 8), 256, 0, st, p);
  else if (D <= 1024) b200::launch(norm_mx_rows_kernel<64>, dim3((T + 3) / 4), 256, 0, st, p);
  else if (D <= 2048) b200::launch(norm_mx_rows_kernel<128>, dim3((T + 1) / 2), 256, 0, st, p);
  else if (D <= 4096) b200::launch(norm_mx_rows_kernel<256>, dim3(T), 256, 0, st, p);
  else b200::launch(norm_mx_rows_kernel<512>, dim3(T), 512, 0, st, p);
  b200::count_launch();
  return b200::check_launch("norm_mx");
}
