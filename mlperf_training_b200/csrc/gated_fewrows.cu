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
  void* gu;
  long long ldgu;
  int act;
  int gu_f32;
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
      __nv_bfloat16* gu = p.gu != nullptr && !p.gu_f32 ? (__nv_bfloat16*)p.gu + f : nullptr;
      float* gu32 = p.gu != nullptr && p.gu_f32 ? (float*)p.gu + f : nullptr;
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
            if (gu32 != nullptr) { gu32[0] = gv; gu32[p.F] = uv; }
          }
          out += p.lda;
          if (gu != nullptr) gu += p.ldgu;
          if (gu32 != nullptr) gu32 += p.ldgu;
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

// ---------------------------------------------------------------------------------------------------------------------
// y = a W^T (+ residual) of the same few rows: the down projection.
//
// The weight is [N, K] with few rows and a long K, so that its 128-row tiles alone would leave most SMs idle (32 tiles of 4096 rows).  A cluster of
// 1, 2, 4 or 8 CTAs owns a tile, each CTA a run of K; they put their fp32 sums into their own shared memory (the operands are done with it) and
// each adds up every gridDim.y-th token of the tile, reading its neighbours' sums in the order of the ranks: one launch, no workspace, no atomics, the
// same result every time.  A stage is 128 elements of K of 128 weight rows, four stages of 48 KB
// (7 x 4096 x 14336: 24.5 us, 4.8 TB/s; the general GEMM and the sum of its parts 36).  The residual is brought into L2 meanwhile, and the
// tokens are finished eight at a time: one after the other each waited 0.5 us for its own loads (64 rows of 4096 x 1024: 33 -> 16 us).
constexpr int D_STAGES = 4;
constexpr int DA_STAGE = 2 * 128 * 128, DB_STAGE = 2 * fewrows::MAX_ROWS * 128;
constexpr int D_SMEM = D_STAGES * (DA_STAGE + DB_STAGE) + 1024 + 256;
static_assert(D_SMEM <= 232448, "stages exceed shared memory");
static_assert(fewrows::MAX_ROWS * 128 * 4 <= D_STAGES * DA_STAGE, "the sums take the operands' place");

struct DownParams {
  int M, N, K;
  int a_rows;
  const __nv_bfloat16* res;
  long long ldr;
  __nv_bfloat16* y;
  long long ldy;
  int* status;
};

B200_DEVICE float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));       // (between two cluster barriers, which order it)
  return v;
}

__global__ void __launch_bounds__(NUM_THREADS, 1)
down_fewrows_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmA, const __grid_constant__ DownParams p) {
  b200::begin_kernel();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = sA + D_STAGES * DA_STAGE;
  float* part = reinterpret_cast<float*>(smem);         // [tokens][128], once the products are done
  uint64_t* full = reinterpret_cast<uint64_t*>(sB + D_STAGES * DB_STAGE);
  uint64_t* empty = full + D_STAGES;
  uint64_t* tfull = empty + D_STAGES;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(tfull + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int split = gridDim.y, rank = blockIdx.y, n0 = blockIdx.x * 128;        // (the cluster spans the grid's y)
  const int num_kb = (p.K + 127) / 128, kb0 = num_kb * rank / split, kb1 = num_kb * (rank + 1) / split;
  const int cols = (p.M + 15) / 16 * 16;
  if (threadIdx.x == 0) {
    for (int i = 0; i < D_STAGES; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
    mbar_init(tfull, 1);
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_holder, ACC);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;

  if (warp == 0) {
    // ------------------------------ TMA producer ------------------------------
    if (lane == 0) {
      tma_prefetch_desc(&tmW); tma_prefetch_desc(&tmA);
      int stage = 0; uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait_spin(&empty[stage], phase ^ 1, abort_flag, p.status, 840)) break;
        // (a second half that begins past K is not fetched, nor multiplied)
        const int halves = kb * 128 + 64 < p.K ? 2 : 1;
        mbar_expect_tx(&full[stage], halves * (16384 + p.a_rows * 128));
        for (int h = 0; h < halves; ++h) {
          tma_load_2d(sA + stage * DA_STAGE + h * 16384, &tmW, &full[stage], kb * 128 + h * 64, n0);
          tma_load_2d(sB + stage * DB_STAGE + h * (DB_STAGE / 2), &tmA, &full[stage], kb * 128 + h * 64, 0);
        }
        if (++stage == D_STAGES) { stage = 0; phase ^= 1; }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------ MMA issuer ------------------------------
    const uint32_t idesc = umma_idesc(1, 1, 0, 0, 128, cols);
    const uint64_t ad0 = umma_desc_sw128(smem_u32(sA), 16, 1024), bd0 = umma_desc_sw128(smem_u32(sB), 16, 1024);
    int stage = 0; uint32_t phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!warp_wait_spin(&full[stage], phase, abort_flag, p.status, 841)) break;
      tc_fence_after();
      if (elect_one()) {
        const uint64_t ad = ad0 + (stage * DA_STAGE >> 4), bd = bd0 + (stage * DB_STAGE >> 4);
        const int halves = kb * 128 + 64 < p.K ? 2 : 1;
        for (int h = 0; h < halves; ++h)
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            tc_mma_f16_ss(tmem_base, ad + (h * 16384 >> 4) + kk * 2, bd + (h * (DB_STAGE / 2) >> 4) + kk * 2, idesc, (kb > kb0 || h > 0 || kk > 0) ? 1u : 0u);
        tc_commit(&empty[stage]);
        if (kb == kb1 - 1) tc_commit(tfull);
      }
      __syncwarp();
      if (++stage == D_STAGES) { stage = 0; phase ^= 1; }
    }
  } else {
    // ------------------------------ sums of this CTA ------------------------------
    if (p.res != nullptr) {
      // the residual on its way into L2 while the products run: 32 bytes a lane, eight lanes a token
      const int i = threadIdx.x - 64, n = n0 + (i & 7) * 16;
      if (n < p.N)
        for (int m = rank + (i >> 3) * split; m < p.M; m += 16 * split) asm volatile("prefetch.global.L2 [%0];" ::"l"(p.res + m * p.ldr + n));
    }
    if (warp_wait(tfull, 0, abort_flag, p.status, 842)) {
      tc_fence_after();
      const int q = warp & 3;
      const uint32_t row = tmem_base + (uint32_t(q * 32) << 16);
      for (int c = 0; c < cols; c += 16) {
        uint32_t v[16];
        tmem_ld_32x32b_x16(row + c, v);
        tc_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; ++i) part[(c + i) * 128 + q * 32 + lane] = __uint_as_float(v[i]);
      }
      tc_fence_before();
    }
  }
  // Every thread comes through here, after a wait that gave up too.
  __syncthreads();
  if (*abort_flag) {
    const uint64_t t0 = globaltimer_ns();               // let copies that are still in flight land
    while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
  __syncwarp();
  cluster_sync_all();
  if (warp >= 2) {
    const int f = (warp - 2) * 32 + lane;
    const long long n = n0 + f;
    if (n < p.N) {
      // eight tokens at a time, all their loads (past the last token: that token's) ahead of the first sum
      for (int m0 = rank; m0 < p.M; m0 += 8 * split) {
        float add[8], s[8];
        int at[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          at[i] = min(m0 + i * split, p.M - 1);
          add[i] = s[i] = 0.f;
        }
        if (p.res != nullptr) {
#pragma unroll
          for (int i = 0; i < 8; ++i) add[i] = __bfloat162float(p.res[at[i] * p.ldr + n]);
        }
        for (int r = 0; r < split; ++r) {
          const uint32_t base = mapa_u32(smem_u32(&part[f]), r);
          float v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = ld_cluster_f32(base + at[i] * 512);
#pragma unroll
          for (int i = 0; i < 8; ++i) s[i] += v[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (m0 + i * split < p.M) p.y[at[i] * p.ldy + n] = __float2bfloat16_rn(s[i] + add[i]);
      }
    }
  }
  __syncwarp();
  cluster_sync_all();                                   // nobody leaves while a neighbour reads its sums
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, ACC);
  }
}

}  // namespace

namespace fewrows {

static void down_config(cudaLaunchConfig_t& cfg, cudaLaunchAttribute* attr, int tiles, int split, cudaStream_t stream) {
  cfg = {};
  cfg.gridDim = dim3(tiles, split, 1);
  cfg.blockDim = dim3(NUM_THREADS, 1, 1);
  cfg.dynamicSmemBytes = D_SMEM;
  cfg.stream = stream;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1; attr[0].val.clusterDim.y = split; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
}

// CTAs of a tile: the most of 1, 2, 4 and 8 (the portable cluster) of which all tiles' clusters are on the GPU at the same time, while each has
// four stages to keep in flight.  A cluster lies in one GPC, so that fewer fit than the SMs would hold (at[]: of 2, 4 and 8 CTAs, asked once):
// 2048 x 5632 took two rounds of clusters of eight.
static int down_split(int tiles, int num_kb, const int* at) {
  int s = 1;
  for (int i = 0; i < 3 && tiles <= at[i] && num_kb >= 2 * s * D_STAGES; ++i) s *= 2;
  return s;
}

int run_down(const DownArgs& a, cudaStream_t stream) {
  static bool configured[64] = {false};
  static int fit[64][3];
  int dev = 0, r;
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attr[2];
  cudaGetDevice(&dev);
  if (!configured[dev & 63]) {
    const cudaError_t e = cudaFuncSetAttribute(down_fewrows_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, D_SMEM);
    if (e != cudaSuccess) {
      cudaGetLastError();
      return b200::fail(871, "gated_down: cannot set %d bytes of shared memory: %s", D_SMEM, cudaGetErrorString(e));
    }
    for (int i = 0; i < 3; ++i) {
      down_config(cfg, attr, 1, 2 << i, stream);
      int n = 0;
      if (cudaOccupancyMaxActiveClusters(&n, down_fewrows_kernel, &cfg) != cudaSuccess) {
        cudaGetLastError();
        n = 0;
      }
      fit[dev & 63][i] = n;
    }
    configured[dev & 63] = true;
  }
  CUtensorMap tmW, tmA;
  if ((r = b200::make_tmap_2d(&tmW, b200::DT_BF16, a.w, a.K, a.N, a.ldw * 2, 64, 128, b200::SWZ_128))) return r;
  if ((r = b200::make_tmap_2d(&tmA, b200::DT_BF16, a.a, a.K, a.M, a.lda * 2, 64, a_box_rows(a.M), b200::SWZ_128))) return r;
  const DownParams p = {a.M, a.N, a.K, a_box_rows(a.M), a.res, a.ldr, a.y, a.ldy, b200::status_ptr()};
  const int tiles = (a.N + 127) / 128, split = down_split(tiles, (a.K + 127) / 128, fit[dev & 63]);
  down_config(cfg, attr, tiles, split, stream);
  cudaLaunchKernelEx(&cfg, down_fewrows_kernel, tmW, tmA, p);
  b200::count_launch();
  return b200::check_launch("gated_down");
}

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
  const Params p = {a.M, a.F, a.K, (a.F + 127) / 128, a_box_rows(a.M), a.a, a.lda, a.gu, a.ldgu, a.act, a.gu_f32, b200::status_ptr()};
  b200::launch(gated_fewrows_kernel, dim3(p.tiles < b200::sm_count() ? p.tiles : b200::sm_count()), NUM_THREADS, SMEM, stream, tmW, tmX, p);
  b200::count_launch();
  return b200::check_launch("gemm_gated(few rows)");
}

}  // namespace fewrows
