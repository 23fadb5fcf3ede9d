// Gated projections of up to 64 rows of activations (single tokens, small batches): a = act(x Wg^T) * (x Wu^T), optionally with the projections
// themselves.
//
// Such a product is bound by reading the weight once.  With the activations as the rows of the tensor-core tile an instruction works on 256 rows
// whatever their number is, and that time, not HBM, was the bound (7 x 2 x 14336 x 4096: 57 us for 235 MB).  Here the weight's rows are the
// tile's rows and the activations its columns, 16 to 64 of them: an instruction takes a quarter or less of the time in which its operand
// arrives, and every byte in flight is one of the weight (39 us, 6.0 TB/s).
//
// One CTA per 128 features, persistent, 192 threads: a TMA producer, an MMA issuer (tcgen05.mma.cta_group::1), four epilogue warps.  A stage is 64
// elements of K of 128 gate rows and of the 128 up rows of the same features, five stages of 40 KB; two accumulators of up to 64 columns, double
// buffered.  A lane of the epilogue has one feature of all tokens, so 32 lanes store 32 neighbouring features of a token.
// The rows and columns that no box reaches (the activations' box has as many rows as there are) hold what was there: they are rows and columns
// of the accumulators that nobody stores.
#include "common.cuh"
#include "gemm_core.cuh"
#include "gated_fewrows.cuh"
#include "runtime.h"

namespace {

using gemmcore::a_box_rows;
using gemmcore::gate_act;

constexpr int NUM_THREADS = 192;
constexpr int KB = 64;                                // elements of a stage
constexpr int A_STAGE = 256 * 128, B_STAGE = fewrows::MAX_ROWS * 128;
constexpr int STAGES = 5;
constexpr int SMEM = STAGES * (A_STAGE + B_STAGE) + 1024 + 256;
constexpr int ACC = fewrows::MAX_ROWS;                // columns of one accumulator
static_assert(SMEM <= 232448, "stages exceed shared memory");

struct Params {
  int M, F, K;
  int tiles;
  int a_rows;                                         // rows of the activations' box
  __nv_bfloat16* a;
  long long lda;
  __nv_bfloat16* gu;
  long long ldgu;
  int act;
  int* status;
};

__global__ void __launch_bounds__(NUM_THREADS, 1)
gated_fewrows_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const __grid_constant__ Params p) {
  b200::begin_kernel();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = sA + STAGES * A_STAGE;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sB + STAGES * B_STAGE);
  uint64_t* full = bars;
  uint64_t* empty = bars + STAGES;
  uint64_t* tfull = bars + 2 * STAGES;
  uint64_t* tempty = tfull + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(tempty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int num_kb = (p.K + KB - 1) / KB, cols = (p.M + 15) / 16 * 16;
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&tfull[i], 1); mbar_init(&tempty[i], 4); }
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_holder, 4 * ACC);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;

  if (warp == 0) {
    // ------------------------------ TMA producer ------------------------------
    if (lane == 0) {
      tma_prefetch_desc(&tmW); tma_prefetch_desc(&tmX);
      int stage = 0; uint32_t phase = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < p.tiles && ok; t += gridDim.x) {
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait_spin(&empty[stage], phase ^ 1, abort_flag, p.status, 810)) { ok = false; break; }
          mbar_expect_tx(&full[stage], A_STAGE + p.a_rows * 128);
          uint8_t* a = sA + stage * A_STAGE;
          tma_load_2d(a, &tmW, &full[stage], kb * KB, t * 128);
          tma_load_2d(a + 16384, &tmW, &full[stage], kb * KB, p.F + t * 128);
          tma_load_2d(sB + stage * B_STAGE, &tmX, &full[stage], kb * KB, 0);
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------ MMA issuer ------------------------------
    const uint32_t idesc = umma_idesc(1, 1, 0, 0, 128, cols);
    const uint64_t ad0 = umma_desc_sw128(smem_u32(sA), 16, 1024), bd0 = umma_desc_sw128(smem_u32(sB), 16, 1024);
    int stage = 0; uint32_t phase = 0;
    int it = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < p.tiles && ok; t += gridDim.x, ++it) {
      const int acc = it & 1;
      if (!warp_wait(&tempty[acc], ((it >> 1) & 1) ^ 1, abort_flag, p.status, 820)) { ok = false; break; }
      tc_fence_after();
      const uint32_t d = tmem_base + acc * 2 * ACC;
      for (int kb = 0; kb < num_kb; ++kb) {
        if (!warp_wait_spin(&full[stage], phase, abort_flag, p.status, 821)) { ok = false; break; }
        tc_fence_after();
        if (elect_one()) {
          const uint64_t ad = ad0 + (stage * A_STAGE >> 4), bd = bd0 + (stage * B_STAGE >> 4);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
#pragma unroll
            for (int h = 0; h < 2; ++h)               // gate, up
              tc_mma_f16_ss(d + h * ACC, ad + (h * 16384 >> 4) + kk * 2, bd + kk * 2, idesc, (kb > 0 || kk > 0) ? 1u : 0u);
          tc_commit(&empty[stage]);
          if (kb == num_kb - 1) tc_commit(&tfull[acc]);
        }
        __syncwarp();
        if (++stage == STAGES) { stage = 0; phase ^= 1; }
      }
    }
  } else {
    // ------------------------------ epilogue ------------------------------
    const int q = warp & 3;
    int it = 0;
    for (int t = blockIdx.x; t < p.tiles; t += gridDim.x, ++it) {
      const int acc = it & 1;
      if (!warp_wait(&tfull[acc], (it >> 1) & 1, abort_flag, p.status, 830)) break;
      tc_fence_after();
      const uint32_t row = tmem_base + (uint32_t(q * 32) << 16) + acc * 2 * ACC;
      const int f = t * 128 + q * 32 + lane;
      const bool live = f < p.F;
      __nv_bfloat16* out = p.a + f;
      __nv_bfloat16* gu = p.gu != nullptr ? p.gu + f : nullptr;
      for (int c = 0; c < cols; c += 16) {
        uint32_t g[16], u[16];
        tmem_ld_32x32b_x16(row + c, g);
        tmem_ld_32x32b_x16(row + ACC + c, u);
        tc_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if (live && c + i < p.M) {
            const float gv = __uint_as_float(g[i]), uv = __uint_as_float(u[i]);
            *out = __float2bfloat16_rn(gate_act(gv, p.act) * uv);
            if (gu != nullptr) { gu[0] = __float2bfloat16_rn(gv); gu[p.F] = __float2bfloat16_rn(uv); }
          }
          out += p.lda;
          if (gu != nullptr) gu += p.ldgu;
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty[acc]);
    }
  }
  if (*abort_flag) {
    // let copies that are still in flight land before shared memory is released
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 4 * ACC);
  }
}

}  // namespace

namespace fewrows {

int run_gated(const GatedArgs& a, cudaStream_t stream) {
  static bool configured[64] = {false};
  int dev = 0, r;
  cudaGetDevice(&dev);
  if (!configured[dev & 63]) {
    const cudaError_t e = cudaFuncSetAttribute(gated_fewrows_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
    if (e != cudaSuccess) {
      cudaGetLastError();
      return b200::fail(870, "gemm_gated: cannot set %d bytes of shared memory: %s", SMEM, cudaGetErrorString(e));
    }
    configured[dev & 63] = true;
  }
  CUtensorMap tmW, tmX;
  if ((r = b200::make_tmap_2d(&tmW, b200::DT_BF16, a.w, a.K, 2LL * a.F, a.ldw * 2, 64, 128, b200::SWZ_128))) return r;
  if ((r = b200::make_tmap_2d(&tmX, b200::DT_BF16, a.x, a.K, a.M, a.ldx * 2, 64, a_box_rows(a.M), b200::SWZ_128))) return r;
  const Params p = {a.M, a.F, a.K, (a.F + 127) / 128, a_box_rows(a.M), a.a, a.lda, a.gu, a.ldgu, a.act, b200::status_ptr()};
  b200::launch(gated_fewrows_kernel, dim3(p.tiles < b200::sm_count() ? p.tiles : b200::sm_count()), NUM_THREADS, SMEM, stream, tmW, tmX, p);
  b200::count_launch();
  return b200::check_launch("gemm_gated(few rows)");
}

}  // namespace fewrows
