// MXFP4 block-scaled GEMM for sm_100a:
//
//   D[M,N] (=|+=) alpha * (A_q * 2^sfa)[M,K] * (B_q * 2^sfb)[N,K]^T (+ bias[N]) (+ residual[M,N])
//
// A_q / B_q are e2m1 codes, two per byte (the even element in the low half), K-major; sfa / sfb hold one UE8M0 scale per 32
// contraction elements in the atom layout of quant_mxfp8.cu (tile rows = 128 for A, = b200_gemm_mxfp4_bn(N) for B).
//
// gemmcore::gemm_pair_kernel<KIND_MXFP4> (gemm_core.cuh): CTA pairs on 256 x BN tiles with
// tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X, 64 elements an instruction, two sub-blocks of 256 elements of K (128
// bytes) per pipeline stage; the scale sets of a stage reach tensor memory through the four forwarding warps.
//
// BN = 192: 2 x 192 accumulator columns leave 128 of tensor memory: six scale sets of 20 columns, so three stages of two sub-blocks (190 KB) in
// flight, beside one 4 KB staging buffer for each of the eight epilogue warps.  With six stages of one sub-block a stage's hand-overs (barriers,
// commit) took as long as its four instructions: 4096 x 14336 x 8192 196 -> 172 us (5.6 PFLOP/s), 16384 x 28672 x 4096 818 -> 740 us.  The
// tensor pipe is busy three quarters of the time at the clock the power limit leaves; L2 and shared memory are at half their rates.
//
// One row of A (a single token) runs without tensor cores: gemv_mxfp4_kernel below.
#include "common.cuh"
#include "gemm_core.cuh"
#include "runtime.h"

namespace {

constexpr int KSUB = 2;           // 256-element sub-blocks per stage

template <int BN>
int run(const void* a_q, const void* sfa, const void* b_q, const void* sfb, void* d, int M, int N, int K, long long lda, long long ldb,
        long long ldd, const gemmcore::EpiArgs& epi, void* ws, long long ws_bytes, cudaStream_t stream) {
  using namespace gemmcore;
  CUtensorMap tmA, tmB, tmSFA, tmSFB, tmD, tmDt;
  int r;
  // (operands as bytes; what a box reaches past K, M or N arrives as zeros)
  if ((r = b200::make_tmap_2d(&tmA, b200::DT_U8, a_q, K / 2, M, lda, 128, a_box_rows(M), b200::SWZ_128))) return r;
  if ((r = b200::make_tmap_2d(&tmB, b200::DT_U8, b_q, K / 2, N, ldb, 128, BN / 2, b200::SWZ_128))) return r;
  const int kg = (K + 127) / 128, atoms = (BN + 127) / 128;
  const long long a_rows = (long long)((M + 127) / 128) * kg, b_rows = (long long)((N + BN - 1) / BN) * kg * atoms;
  if ((r = b200::make_tmap_2d(&tmSFA, b200::DT_I32, sfa, 128, a_rows, 512, 128, 2 * KSUB, b200::SWZ_NONE))) return r;
  if ((r = b200::make_tmap_2d(&tmSFB, b200::DT_I32, sfb, 128, b_rows, 512, 128, 2 * KSUB * atoms, b200::SWZ_NONE))) return r;
  if ((r = make_out_tmap<BN>(&tmD, &tmDt, d, M, N, ldd, epi.out_f32))) return r;
  PairParams p = {};
  p.M = M; p.N = N; p.K = K;
  p.group_m = raster_group_m();    // (rows of half the bytes: groups twice as tall as the 8-bit kernels', 16384 x 28672 x 4096 829 -> 815 us)
  p.epi = epi;
  p.a_rows = a_box_rows(M);
  p.status = b200::status_ptr();
  return launch_pair<KIND_MXFP4, BN, KSUB, 1>(tmA, tmB, tmSFA, tmSFB, tmD, tmDt, p, stream, "gemm_mxfp4", nullptr, (float*)ws, ws_bytes, d, ldd);
}

// One row of A: D is bound by reading B once, and a tensor-core tile would be 1/256 full (and its 150 tiles of 192 columns make three rounds on
// 74 CTA pairs).  Products of two e2m1 values are multiples of 1/4 up to 36: a sum of eight of them is exact in f16 (11 bits), so the codes
// become f16 pairs, two HFMA2 chains of eight make a 32-block's sum, which goes on in fp32, scaled by both blocks' powers of two.
// A warp owns the rows of B whose scales share 16 bytes of an atom (rows r, r + 32, r + 64, r + 96 of it), a lane a block of each at a time.
// Measured (caches cold, tensor cores -> this): 4096 x 4096 15 -> 8.5 us, 4096 x 14336 22 -> 16.5, 28672 x 4096 26 -> 23 (2.7 TB/s); two rows
// took 34 us there, so it is taken for one.  Bound by how the rows lie on the SMs first, by instructions second (counted, caches cold): 3.4
// instructions an element of B for conversion, product and scale keep the issue slots of a working SM 64 % busy, but 28672 rows are 9600 units on
// 2368 warps, whose fifth round runs on a few SMs (an SM works 69 % of the time), and 4096 rows are 88 CTAs: 60 SMs have nothing to do (45 %).
struct GemvArgs {
  const uint8_t* a_q; const uint8_t* sfa;
  const uint8_t* b_q; const uint8_t* sfb;
  void* d;
  int N, K, bn;
  long long ldb;
  gemmcore::EpiArgs epi;
};
constexpr int GEMV_ELEMS = 28672;                // most elements of A (60 KB of shared memory beside the ring)

// eight codes to f16 pairs
B200_DEVICE void e2m1x8_f16(uint32_t c, __half2 (&h)[4]) {
  uint32_t r[4];
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "mov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(c));
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = *reinterpret_cast<const __half2*>(&r[i]);
}
// 2^(e - 127); 0 is 2^-127, below the normal numbers, 255 a NaN
B200_DEVICE float pow2_of(uint32_t e) { return e == 255u ? __uint_as_float(0x7fffffffu) : __uint_as_float(max(e << 23, 0x00400000u)); }

// A step of a warp: a 32-block of each of its rows of B per lane, and the sixteen scale bytes with theirs among them, copied asynchronously into
// the lane's own places of a ring in shared memory (so a lane waits for its own copies only).  Four steps a warp, 160 KB an SM, are in
// flight: with loads into registers, one step ahead, 7 MB were on the way on the whole GPU, a third of what the latency asks for.
constexpr int GEMV_WARPS = 16, GEMV_DEPTH = 4;
constexpr int GEMV_RING = GEMV_WARPS * GEMV_DEPTH * 5 * 32 * 16;
B200_DEVICE void copy16_async(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
B200_DEVICE void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
B200_DEVICE void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Place of a warp in B: the unit's rows, and what of them exists.
struct GemvUnit {
  const uint8_t* src;             // first row
  const uint8_t* sf;
  long long n0;
  int rows;                       // how many of the rows n0, n0 + 32, n0 + 64, n0 + 96 exist (0: none)
};
B200_DEVICE GemvUnit gemv_unit(const GemvArgs& p, int u, int kg, int atoms) {
  // (192-column tiles: the first atom has four rows of a place, the second two; they alternate, also from one of a warp's units to the next)
  const int tile = u / (32 * atoms), ua = u - tile * 32 * atoms;
  const int atom = atoms == 2 ? (ua ^ tile) & 1 : 0, r = atoms == 2 ? ua >> 1 : ua, in_tile = atom * 128 + r;
  GemvUnit g;
  g.n0 = (long long)tile * p.bn + in_tile;
  const int left = (int)min((long long)(p.bn - in_tile), p.N - g.n0);          // rows of the tile and of B from here on
  g.rows = left <= 0 ? 0 : min(4, (left + 31) >> 5);
  g.src = p.b_q + g.n0 * p.ldb;
  g.sf = p.sfb + (((long long)tile * kg * atoms) + atom) * 512 + r * 16;
  return g;
}
// Walk of a warp over its units and their steps.
struct GemvWalk {
  int u, step;
  GemvUnit g;
  B200_DEVICE void next(const GemvArgs& p, int units, int stride, int steps, int kg, int atoms) {
    if (++step < steps) return;
    step = 0;
    u += stride;
    if (u < units) g = gemv_unit(p, u, kg, atoms);
  }
};

// One step of a lane: NR rows' 32-blocks times A's.
template <int NR>
B200_DEVICE void gemv_step(const uint4* cur, const uint4* xs, const float* xf, int kb, int nb, float (&acc)[4]) {
  const uint4 sc = cur[128];
  const uint32_t sw[4] = {sc.x, sc.y, sc.z, sc.w};
  float sum[NR];
#pragma unroll
  for (int j = 0; j < 4; j += 2) {               // sixteen elements: eight products to either half of an f16 pair
    __half2 x[8];
    *reinterpret_cast<uint4*>(&x[0]) = xs[j * nb + kb];
    *reinterpret_cast<uint4*>(&x[4]) = xs[(j + 1) * nb + kb];
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      __half2 a[4], b[4];
      const uint2 c = *(reinterpret_cast<const uint2*>(cur + i * 32) + j / 2);
      e2m1x8_f16(c.x, a);
      e2m1x8_f16(c.y, b);
      __half2 t = __hmul2(a[0], x[0]);
#pragma unroll
      for (int k = 1; k < 4; ++k) t = __hfma2(a[k], x[k], t);
#pragma unroll
      for (int k = 0; k < 4; ++k) t = __hfma2(b[k], x[4 + k], t);
      const float2 f = __half22float2(t);
      sum[i] = j == 0 ? f.x + f.y : sum[i] + (f.x + f.y);
    }
  }
#pragma unroll
  for (int i = 0; i < NR; ++i)
    // (a row past the end has whatever codes and scale byte the ring held: its sum is not stored)
    acc[i] = fmaf(sum[i], pow2_of((sw[i] >> (8 * (kb & 3))) & 0xffu) * xf[kb], acc[i]);
}

__global__ void __launch_bounds__(GEMV_WARPS * 32)
gemv_mxfp4_kernel(const GemvArgs p) {
  b200::begin_kernel();
  extern __shared__ __align__(16) uint8_t smem[];
  const int nb = p.K / 32, kg = (p.K + 127) / 128, atoms = (p.bn + 127) / 128, steps = (nb + 31) / 32;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint4* ring = reinterpret_cast<uint4*>(smem) + warp * GEMV_DEPTH * 160 + lane;       // [depth][5][32 lanes]
  uint4* xs = reinterpret_cast<uint4*>(smem + GEMV_RING);                              // [4][nb]: eight f16 each
  float* xf = reinterpret_cast<float*>(smem + GEMV_RING + (size_t)nb * 64);            // [nb] scales
  const int units = ((p.N + p.bn - 1) / p.bn) * 32 * atoms, stride = gridDim.x * GEMV_WARPS;
  const uint32_t row32 = (uint32_t)(32 * p.ldb);       // (places inside a unit fit 32 bits: 96 rows' pitches of at most 28 KB)
  GemvWalk it;
  it.u = blockIdx.x * GEMV_WARPS + warp;
  it.step = 0;
  it.g = gemv_unit(p, min(it.u, units - 1), kg, atoms);
  GemvWalk ahead = it;
  const auto fetch = [&](int slot) {             // the copies of the step that `ahead` is at, as one group (empty past the end)
    const int kb = ahead.step * 32 + lane;
    if (ahead.u < units && kb < nb) {
      uint4* dst = ring + slot * 160;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < ahead.g.rows) copy16_async(dst + i * 32, ahead.g.src + (i * row32 + (uint32_t)kb * 16));
      if (ahead.g.rows > 0) copy16_async(dst + 128, ahead.g.sf + (uint32_t)(kb >> 2) * (uint32_t)(atoms * 512));
    }
    copy_commit();
    ahead.next(p, units, stride, steps, kg, atoms);
  };
#pragma unroll
  for (int i = 0; i < GEMV_DEPTH - 1; ++i) fetch(i);
  // A to f16 while they are under way
  for (int kb = tid; kb < nb; kb += GEMV_WARPS * 32) {
    const uint4 c = *reinterpret_cast<const uint4*>(p.a_q + kb * 16);
    const uint32_t cw[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      __half2 h[4];
      e2m1x8_f16(cw[j], h);
      xs[j * nb + kb] = *reinterpret_cast<const uint4*>(h);
    }
    xf[kb] = pow2_of(p.sfa[(kb >> 2) * 512 + (kb & 3)]);                        // (row 0 of the first atom)
  }
  __syncthreads();
  float acc[4];
  int slot = 0;
  while (it.u < units) {
    fetch((slot + GEMV_DEPTH - 1) % GEMV_DEPTH);
    copy_wait<GEMV_DEPTH - 1>();
    const int kb = it.step * 32 + lane;
    if (it.step == 0) acc[0] = acc[1] = acc[2] = acc[3] = 0.f;
    if (kb < nb) {
      if (it.g.rows > 2) gemv_step<4>(ring + slot * 160, xs, xf, kb, nb, acc);
      else gemv_step<2>(ring + slot * 160, xs, xf, kb, nb, acc);
    }
    if (it.step == steps - 1) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float v = warp_sum(acc[i]);
        if (lane != i || i >= it.g.rows) continue;
        const long long n = it.g.n0 + i * 32;
        v *= p.epi.alpha;
        if (p.epi.bias != nullptr) v += __bfloat162float(p.epi.bias[n]);
        if (p.epi.residual != nullptr) v += __bfloat162float(p.epi.residual[n]);
        if (p.epi.out_f32) {
          float* o = (float*)p.d + n;
          *o = p.epi.accumulate ? *o + v : v;
        } else {
          __nv_bfloat16* o = (__nv_bfloat16*)p.d + n;
          *o = __float2bfloat16_rn(p.epi.accumulate ? __bfloat162float(*o) + v : v);
        }
      }
    }
    it.next(p, units, stride, steps, kg, atoms);
    slot = slot + 1 == GEMV_DEPTH ? 0 : slot + 1;
  }
}

int run_gemv(const GemvArgs& p, cudaStream_t stream) {
  static bool configured[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!configured[dev & 63]) {
    constexpr int most = GEMV_RING + 2 * GEMV_ELEMS + GEMV_ELEMS / 8;
    static_assert(most <= 232448, "ring and A exceed shared memory");
    const cudaError_t e = cudaFuncSetAttribute(gemv_mxfp4_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    if (e != cudaSuccess) {
      cudaGetLastError();
      return b200::fail(852, "gemm_mxfp4: cannot set %d bytes of shared memory: %s", most, cudaGetErrorString(e));
    }
    configured[dev & 63] = true;
  }
  // one CTA per SM, each warp walks over its units
  const int units = ((p.N + p.bn - 1) / p.bn) * 32 * ((p.bn + 127) / 128), ctas = (units + GEMV_WARPS - 1) / GEMV_WARPS;
  b200::launch(gemv_mxfp4_kernel, dim3(ctas < b200::sm_count() ? ctas : b200::sm_count()), GEMV_WARPS * 32, GEMV_RING + 2 * p.K + p.K / 8, stream, p);
  b200::count_launch();
  return b200::check_launch("gemm_mxfp4(row)");
}
// Whether the kernel above is given the problem.
bool one_row(int M, int K, long long ldb) { return M == 1 && K <= GEMV_ELEMS && ldb <= GEMV_ELEMS; }

}  // namespace

// N tile of the kernel for an output width N: the B operand's scales are laid out for it.
B200_API int b200_gemm_mxfp4_bn(int N) { return N <= 128 ? 128 : 192; }

// Workspace (bytes, 16-byte aligned) with which b200_gemm_mxfp4 splits the last wave along K; 0 where that does not pay.
B200_API long long b200_gemm_mxfp4_workspace(int M, int N, int K) {
  using namespace gemmcore;
  if (M <= 0 || N <= 0 || K <= 0 || one_row(M, K, K / 2)) return 0;
  int rc = 0;
  return b200_gemm_mxfp4_bn(N) == 192 ? split_bytes<192>(pair_split<KIND_MXFP4, 192, KSUB>(M, N, K, rc))
                                      : split_bytes<128>(pair_split<KIND_MXFP4, 128, KSUB>(M, N, K, rc));
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
  if (one_row(M, K, ldb)) {
    if ((((uintptr_t)a_q | (uintptr_t)b_q | (uintptr_t)sfb | (uintptr_t)ldb) & 15) != 0)
      return b200::fail(853, "gemm_mxfp4: operands and their row pitches must be 16-byte aligned");
    const GemvArgs p = {(const uint8_t*)a_q, (const uint8_t*)sfa, (const uint8_t*)b_q, (const uint8_t*)sfb, d, N, K, b200_gemm_mxfp4_bn(N), ldb, epi};
    return run_gemv(p, (cudaStream_t)stream);
  }
  if (b200_gemm_mxfp4_bn(N) == 192)
    return run<192>(a_q, sfa, b_q, sfb, d, M, N, K, lda, ldb, ldd, epi, workspace, workspace_bytes, (cudaStream_t)stream);
  return run<128>(a_q, sfa, b_q, sfb, d, M, N, K, lda, ldb, ldd, epi, workspace, workspace_bytes, (cudaStream_t)stream);
}
