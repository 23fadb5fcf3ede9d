// Backward of attention with the masks of attn_mask.cuh, capped scores and a distance bias: the engine of attention_bwd.cu (one CTA per
// batch, kv head and 128-key tile; transposed scores, P^T as a TMEM operand, dK and dV in TMEM, dQ by fp32 reduce-add) with
//
//   P = exp(s - lse)     dS = scale (1 - tanh^2) P (dP - delta)
//
//   * the query tiles of a key tile, and which of them hold anything to mask, from the mask's tables; key tiles of all sequences longest
//     first, over the kv heads of one after the other; a worker's key row sees one interval of queries;
//   * delta = rowsum(dO O) with the output as the forward had it: its bf16 value and what that lost;
//   * the factor of the cap is taken after P has gone to dV.
// 8192 tokens, 32 heads of 128 on 8, causal: 1.33 ms (1.04 PFLOP/s), 16 documents in them 0.23 (delta and a cleared dQ are 57 us of it).  Bound by the
// chain of a step (scores, P, dP, dS, their products), of which one CTA an SM has one under way.
#include "attn_masked.cuh"

namespace {

constexpr int BQ = 128;
constexpr int BKV = 128;
constexpr int NTHREADS = 512;  // warp 0 TMA, 1 MMA (2, 3 complete the warpgroup), 4-7 dQ drain, 8-15 P / dS workers
// 4 x 128 threads launch with 128 registers each: 88 + 88 + 2 x 168
constexpr int REGS_OTHER = 88, REGS_WORKER = 168;
constexpr int STG = 4096;  // dQ staging chunk: 32 rows x 32 fp32 (two per drain warp)

struct BwdParams {
  b200::MaskView mask;
  b200::ScoreParams score;
  int Hq, Hkv, Sq, Skv;
  float scale_log2;
  const float* lse;    // [B, Hq, Sq]
  const float* delta;  // [B, Hq, Sq]  rowsum(dO * O)
  int* status;
  int parts;           // CTAs that share a key tile's steps; above 1 their sums go to `partial`
  float* partial;      // fp32 [B * Hkv * key tiles][parts][dK | dV][128][HD]
};

template <int HD>
struct Smem {
  static constexpr int T_BYTES = 128 * HD * 2;        // K, V, Q (two stages), dO tiles
  static constexpr int DS_BYTES = BQ * BKV * 2;       // dS^T tile
  static constexpr int STG_BYTES = 8 * STG;
  static constexpr int LD_BYTES = 2 * 2 * BQ * 4;     // log-sum-exp and delta of two query tiles
  // The base of dynamic shared memory is 1024-byte aligned when a kernel has no static shared memory; checked at entry
  // (at head dim 128 there is no room to align it).
  static constexpr int TOTAL = 5 * T_BYTES + DS_BYTES + STG_BYTES + LD_BYTES + 256;
};

template <int HD, int SCORE>
__global__ void __launch_bounds__(NTHREADS, 1)
attn_masked_bwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmdO,
                const __grid_constant__ CUtensorMap tmdQ, const __grid_constant__ CUtensorMap tmdK,
                const __grid_constant__ CUtensorMap tmdV, const __grid_constant__ BwdParams p) {
  b200::begin_kernel();
  using SM = Smem<HD>;
  constexpr int NB = HD / 64;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* sK = smem;
  uint8_t* sV = sK + SM::T_BYTES;
  uint8_t* sQ = sV + SM::T_BYTES;           // two stages
  uint8_t* sdO = sQ + 2 * SM::T_BYTES;
  uint8_t* sdS = sdO + SM::T_BYTES;
  uint8_t* sStg = sdS + SM::DS_BYTES;
  float* sLD = reinterpret_cast<float*>(sStg + SM::STG_BYTES);   // [stage][lse2 | delta * scale][128]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sLD + 4 * BQ);
  uint64_t* kv_full = bars + 0;     // K and V landed
  uint64_t* q_full = bars + 1;      // 2: Q_i landed
  uint64_t* q_empty = bars + 3;     // 2: MMAs reading Q_i finished
  uint64_t* do_full = bars + 5;     // dO_i landed
  uint64_t* do_empty = bars + 6;    // MMAs reading dO_i finished
  uint64_t* s_full = bars + 7;      // S^T complete in TMEM
  uint64_t* dp_full = bars + 8;     // dP^T complete in TMEM (and every MMA of the step before: dS^T is free)
  uint64_t* p_full = bars + 9;      // P^T written to TMEM (8 arrivals)
  uint64_t* ds_full = bars + 10;    // dS^T written to shared memory (8 arrivals)
  uint64_t* dq_full = bars + 11;    // dQ tile complete in TMEM
  uint64_t* dq_drained = bars + 12; // dQ tile copied out of TMEM (4 arrivals)
  uint64_t* ld_full = bars + 13;    // 2: the step's log-sum-exp / delta are in shared memory (8 arrivals)
  uint64_t* acc_done = bars + 15;   // every MMA of this CTA finished
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars + 16);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  if (smem_u32(smem) & 1023u) {             // (the same for every thread of the launch)
    if (threadIdx.x == 0) b200_report(p.status, B200_ERR_BOUNDS, 94);
    return;
  }

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int nk = p.mask.Kp / BKV, group = p.Hq / p.Hkv, off = p.Skv - p.Sq;
  const int part = (int)blockIdx.x % p.parts, hk = (int)blockIdx.x / p.parts % p.Hkv;
  const int id = p.mask.ok[(int)blockIdx.x / p.parts / p.Hkv];
  const int b = id / nk, jt = id - b * nk;
  const int kv0 = jt * BKV;
  // query tiles that see at least one key of this tile, and the queries that see all of it
  const int4 span = p.mask.kt[id];
  const int i_lo = span.x, i_hi = span.y - 1, n_q = span.y - span.x;
  // this CTA's steps of the tile's
  const int steps = n_q * group;
  const int it0 = (int)((long long)steps * part / p.parts), n_iter = (int)((long long)steps * (part + 1) / p.parts) - it0;

  if (threadIdx.x == 0) {
    mbar_init(kv_full, 1); mbar_init(do_full, 1); mbar_init(do_empty, 1); mbar_init(s_full, 1); mbar_init(dp_full, 1);
    mbar_init(p_full, 8); mbar_init(ds_full, 8); mbar_init(dq_full, 1); mbar_init(dq_drained, 4); mbar_init(acc_done, 1);
    for (int i = 0; i < 2; ++i) { mbar_init(&q_full[i], 1); mbar_init(&q_empty[i], 1); mbar_init(&ld_full[i], 8); }
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 1) { tmem_alloc(tmem_holder, 512); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  const uint32_t tm_S = tmem_base;          // S^T; P^T of queries 0-63 in columns 0-31, of 64-127 in 64-95
  const uint32_t tm_dP = tmem_base + 128;   // dP^T, later dQ
  const uint32_t tm_dK = tmem_base + 256;
  const uint32_t tm_dV = tmem_base + 384;

  if (warp < 8) reg_dealloc<REGS_OTHER>();
  if (warp == 0) {
    // ------------------------------ TMA producer ------------------------------
    // (a key tile that no query sees loads nothing: nobody would wait for it, and the CTA must not leave with copies in flight)
    if (lane == 0 && n_iter > 0) {
      tma_prefetch_desc(&tmQ); tma_prefetch_desc(&tmK); tma_prefetch_desc(&tmV); tma_prefetch_desc(&tmdO);
      mbar_expect_tx(kv_full, 2 * SM::T_BYTES);
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        b200::load_4d(sK + i * (BKV * 128), &tmK, kv_full, i * 64, hk, kv0, b);
        b200::load_4d(sV + i * (BKV * 128), &tmV, kv_full, i * 64, hk, kv0, b);
      }
      for (int it = 0; it < n_iter; ++it) {
        const int h = hk * group + (it0 + it) / n_q;
        const int q0 = (i_lo + (it0 + it) % n_q) * BQ;
        const int st = it & 1;
        if (!mbar_wait(&q_empty[st], ((it >> 1) & 1) ^ 1, abort_flag, p.status, 70)) break;
        mbar_expect_tx(&q_full[st], SM::T_BYTES);
#pragma unroll
        for (int i = 0; i < NB; ++i) b200::load_4d(sQ + st * SM::T_BYTES + i * (BQ * 128), &tmQ, &q_full[st], i * 64, h, q0, b);
        if (!mbar_wait(do_empty, (it & 1) ^ 1, abort_flag, p.status, 71)) break;
        mbar_expect_tx(do_full, SM::T_BYTES);
#pragma unroll
        for (int i = 0; i < NB; ++i) b200::load_4d(sdO + i * (BQ * 128), &tmdO, do_full, i * 64, h, q0, b);
      }
    }
  } else if (warp == 1) {
    // ------------------------------ MMA issuer ------------------------------
    // The warp stays converged and one elected lane issues: operands live in uniform registers and descriptors advance by
    // an addition (rebuilt by one lane of a divergent warp they cost more than the 64 cycles an instruction runs).
    if (n_iter > 0) {
      const uint32_t id_kk = umma_idesc(1, 1, 0, 0, 128, 128);   // S^T = K Q^T, dP^T = V dO^T (both K-major)
      const uint32_t id_dv = umma_idesc(1, 1, 0, 1, 128, HD);    // dV = P^T (TMEM) x dO (MN-major)
      const uint32_t id_dk = umma_idesc(1, 1, 0, 1, 128, HD);    // dK = dS^T (K-major) x Q (MN-major)
      const uint32_t id_dq = umma_idesc(1, 1, 1, 1, 128, HD);    // dQ = dS (the tile read MN-major) x K (MN-major)
      const uint64_t kK = umma_desc_sw128(smem_u32(sK), 16, 1024), kV = umma_desc_sw128(smem_u32(sV), 16, 1024);
      const uint64_t kQ = umma_desc_sw128(smem_u32(sQ), 16, 1024), kdO = umma_desc_sw128(smem_u32(sdO), 16, 1024);
      const uint64_t kdS = umma_desc_sw128(smem_u32(sdS), 16, 1024), mdS = umma_desc_sw128(smem_u32(sdS), 128 * 128, 1024);
      const uint64_t mK = umma_desc_sw128(smem_u32(sK), 128 * 128, 1024), mQ = umma_desc_sw128(smem_u32(sQ), 128 * 128, 1024);
      const uint64_t mdO = umma_desc_sw128(smem_u32(sdO), 128 * 128, 1024);
      auto issue_s = [&](int it) -> bool {
        const int st = it & 1;
        if (!warp_wait_spin(&q_full[st], (it >> 1) & 1, abort_flag, p.status, 81)) return false;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t bd = kQ + (st * SM::T_BYTES >> 4);
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk) {
            const uint32_t o = ((kk / 4) * (128 * 128) + (kk % 4) * 32) >> 4;
            tc_mma_f16_ss(tm_S, kK + o, bd + o, id_kk, kk > 0);
          }
          tc_commit(s_full);
        }
        __syncwarp();
        return true;
      };
      auto issue_dp = [&](int it) -> bool {
        if (!warp_wait_spin(do_full, it & 1, abort_flag, p.status, 82)) return false;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk) {
            const uint32_t o = ((kk / 4) * (128 * 128) + (kk % 4) * 32) >> 4;
            tc_mma_f16_ss(tm_dP, kV + o, kdO + o, id_kk, kk > 0);
          }
          tc_commit(dp_full);
        }
        __syncwarp();
        return true;
      };
      bool ok = warp_wait_spin(kv_full, 0, abort_flag, p.status, 80) && issue_s(0) && issue_dp(0);
      for (int it = 0; it < n_iter && ok; ++it) {
        const uint32_t ph = it & 1;
        const int st = it & 1;
        const bool last = it == n_iter - 1;
        if (!warp_wait_spin(p_full, ph, abort_flag, p.status, 83)) { ok = false; break; }
        tc_fence_after();
        if (elect_one()) {
          // dV += P^T dO : 16 queries = 8 TMEM columns per step, dO as 16 query rows of 128 bytes
#pragma unroll
          for (int kk = 0; kk < BQ / 16; ++kk)
            tc_mma_f16_ts(tm_dV, tm_S + (kk / 4) * 64 + (kk % 4) * 8, mdO + kk * 128, id_dv, (it > 0 || kk > 0));
          tc_commit(do_empty);
        }
        __syncwarp();
        if (!warp_wait_spin(ds_full, ph, abort_flag, p.status, 84)) { ok = false; break; }
        tc_fence_after();
        if (elect_one()) {
          // dQ = dS K : contraction over keys, 16 key rows of the dS^T tile and of K per step
#pragma unroll
          for (int kk = 0; kk < BKV / 16; ++kk) tc_mma_f16_ss(tm_dP, mdS + kk * 128, mK + kk * 128, id_dq, kk > 0);
          tc_commit(dq_full);
        }
        __syncwarp();
        if (!last && !issue_s(it + 1)) { ok = false; break; }     // (P^T(i) was read by dV(i), issued before)
        if (elect_one()) {
          // dK += dS^T Q : contraction over queries
          const uint64_t bd = mQ + (st * SM::T_BYTES >> 4);
#pragma unroll
          for (int kk = 0; kk < BQ / 16; ++kk) {
            const uint32_t ao = ((kk / 4) * (128 * 128) + (kk % 4) * 32) >> 4;
            tc_mma_f16_ss(tm_dK, kdS + ao, bd + kk * 128, id_dk, (it > 0 || kk > 0));
          }
          tc_commit(&q_empty[st]);
          if (last) tc_commit(acc_done);
        }
        __syncwarp();
        if (!last) ok = warp_wait_spin(dq_drained, ph, abort_flag, p.status, 85) && issue_dp(it + 1);
      }
    }
  } else if (warp >= 4 && warp < 8) {
    // ------------------------------ dQ drain ------------------------------
    const int q = warp & 3;                   // TMEM lane quarter: 32 query rows
    const uint32_t lane_base = uint32_t(q * 32) << 16;
    uint8_t* stg = sStg + q * 2 * STG;
    for (int it = 0; it < n_iter; ++it) {
      const int h = hk * group + (it0 + it) / n_q;
      const int q0 = (i_lo + (it0 + it) % n_q) * BQ;
      if (!warp_wait(dq_full, it & 1, abort_flag, p.status, 95)) break;
      tc_fence_after();
#pragma unroll
      for (int c2 = 0; c2 < HD / 64; ++c2) {       // 64 columns at a time: two staging buffers
        uint32_t v[64];
        tmem_ld_32x32b_x32(tm_dP + lane_base + c2 * 64, *reinterpret_cast<uint32_t(*)[32]>(&v[0]));
        tmem_ld_32x32b_x32(tm_dP + lane_base + c2 * 64 + 32, *reinterpret_cast<uint32_t(*)[32]>(&v[32]));
        tc_wait_ld();
        if (c2 == HD / 64 - 1) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(dq_drained);  // the accumulator may be overwritten by the next dP
        }
#pragma unroll
        for (int cc = 0; cc < 2; ++cc) {
          if (lane == 0) tma_store_wait_read<1>(); // the reduce before the last has read this buffer
          __syncwarp();
          uint8_t* sb = stg + cc * STG + lane * 128;
#pragma unroll
          for (int g = 0; g < 8; ++g)
            *reinterpret_cast<uint4*>(sb + ((g ^ (lane & 7)) << 4)) =
                make_uint4(v[cc * 32 + 4 * g], v[cc * 32 + 4 * g + 1], v[cc * 32 + 4 * g + 2], v[cc * 32 + 4 * g + 3]);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            if (q0 + q * 32 < p.Sq) b200::reduce_add_4d(&tmdQ, stg + cc * STG, c2 * 64 + cc * 32, h, q0 + q * 32, b);
            tma_store_commit();
          }
        }
      }
    }
    if (lane == 0) tma_store_wait_all<0>();
  } else if (warp >= 8) {
    // ------------------------------ workers: P / dS ------------------------------
    reg_alloc<REGS_WORKER>();
    const int q = warp & 3;                   // TMEM lane quarter
    const int half = (warp - 8) >> 2;         // which half of the query columns
    const int r = q * 32 + lane;              // key row of the tile
    const uint32_t lane_base = uint32_t(q * 32) << 16;
    const int key = kv0 + r;
    const int2 seen = p.mask.k_iv[(long long)b * p.mask.Kp + key];      // queries [x, y) see this key
    // of this warp's keys: queries that see all of them, and that see any
    const bool is_seen = seen.x < seen.y;
    const int all_lo = __reduce_max_sync(0xffffffffu, seen.x), all_hi = __reduce_min_sync(0xffffffffu, seen.y);
    const int any_lo = __reduce_min_sync(0xffffffffu, is_seen ? seen.x : 0x7fffffff), any_hi = __reduce_max_sync(0xffffffffu, is_seen ? seen.y : 0);
    // this thread stages one value per step: the log-sum-exp (half 0) or delta (half 1) of query r of the tile
    // (loaded a step ahead as it is and turned into what the columns need only when it is stored: used at once, it cost the
    // step a global-memory latency)
    auto fetch = [&](int h, int q_pos) -> float {
      if (q_pos >= p.Sq) return half == 0 ? -INFINITY : 0.f;
      const long long idx = ((long long)b * p.Hq + h) * p.Sq + q_pos;
      return half == 1 ? p.delta[idx] : p.lse[idx];
    };
    // a row that is not there or sees no key: P = exp2(s - inf) = 0
    auto staged = [&](float x) -> float {
      return half == 1 ? x * p.score.scale : (x == -INFINITY ? INFINITY : x * 1.4426950408889634f);
    };
    int h_next = hk * group + (n_iter > 0 ? it0 / n_q : 0), i_next = i_lo + (n_iter > 0 ? it0 % n_q : 0);
    bool ok = true;
    if (n_iter > 0) {
      sLD[half * BQ + r] = staged(fetch(h_next, i_next * BQ + r));
      __syncwarp();
      if (lane == 0) mbar_arrive(&ld_full[0]);
    }
    for (int it = 0; it < n_iter && ok; ++it) {
      const int q0 = i_next * BQ;
      const float slope2 = (SCORE & b200::SCORE_BIAS) ? p.score.slopes[h_next] * b200::LOG2E : 0.f;
      if (++i_next > i_hi) { i_next = i_lo; ++h_next; }
      const float next = it + 1 < n_iter ? fetch(h_next, i_next * BQ + r) : 0.f;
      const bool need_mask = q0 < span.z || q0 + BQ > span.w;
      const int c_lo = seen.x - q0, c_hi = seen.y - q0;                 // visible queries of this key: columns [c_lo, c_hi)
      if (!warp_wait(&ld_full[it & 1], (it >> 1) & 1, abort_flag, p.status, 89)) { ok = false; break; }
      const float* ld = sLD + (it & 1) * 2 * BQ + half * 64;
      if (!warp_wait(s_full, it & 1, abort_flag, p.status, 90)) { ok = false; break; }
      tc_fence_after();
      float pr[64];
      uint32_t s[64];                         // scores, then (with a cap) 1 - tanh^2
      tmem_ld_32x32b_x32(tm_S + lane_base + half * 64, *reinterpret_cast<uint32_t(*)[32]>(&s[0]));
      tmem_ld_32x32b_x32(tm_S + lane_base + half * 64 + 32, *reinterpret_cast<uint32_t(*)[32]>(&s[32]));
      tc_wait_ld();
      if (SCORE & b200::SCORE_CAP) {
        const float inv2 = -1.f / (p.score.back * p.score.back);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float big = 0.f;
#pragma unroll
          for (int i = 0; i < 32; ++i) big = fmaxf(big, fabsf(__uint_as_float(s[c * 32 + i])));
          if (__all_sync(0xffffffffu, big <= p.score.limit)) {
#pragma unroll
            for (int i = c * 32; i < c * 32 + 32; i += 2) {
              const float2 y = b200::capped_small2(make_float2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), p.score);
              pr[i] = y.x; pr[i + 1] = y.y;
            }
          } else {
#pragma unroll
            for (int i = c * 32; i < c * 32 + 32; i += 2) {
              const float2 y = b200::capped_any2(make_float2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), p.score);
              pr[i] = y.x; pr[i + 1] = y.y;
            }
          }
        }
#pragma unroll
        for (int i = 0; i < 64; i += 2) {
          const float2 y = make_float2(pr[i], pr[i + 1]), f = ffma2(fmul2(y, make_float2(inv2, inv2)), y, make_float2(1.f, 1.f));
          s[i] = __float_as_uint(f.x); s[i + 1] = __float_as_uint(f.y);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 64; ++i) pr[i] = __uint_as_float(s[i]);
      }
      if (SCORE & b200::SCORE_BIAS) {
        const float d0 = (float)(q0 + half * 64 + off - key);
#pragma unroll
        for (int i = 0; i < 64; ++i) {
          const float x = (SCORE & b200::SCORE_CAP) ? pr[i] : pr[i] * p.scale_log2;
          pr[i] = fmaf(-slope2, fabsf(d0 + (float)i), x);
        }
      }
      {
        const float scale2 = SCORE == b200::SCORE_PLAIN ? p.scale_log2 : 1.f;
        const float2 sc2 = make_float2(scale2, scale2);
        // 32 queries at a time: none that sees a key of the warp (no exponential then), all, or a comparison each.  (With a cap the branches
        // cost more registers than they save: 4 x 2048 in six documents 309 us without, 345 with them.)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int c0 = half * 64 + h * 32, g0 = q0 + c0;
          if (!(SCORE & b200::SCORE_CAP) && need_mask && (g0 >= any_hi || g0 + 32 <= any_lo)) {
#pragma unroll
            for (int i = 0; i < 32; ++i) pr[h * 32 + i] = 0.f;
            continue;
          }
#pragma unroll
          for (int i = h * 32; i < h * 32 + 32; i += 4) {
            const float4 l4 = *reinterpret_cast<const float4*>(ld + i);
            const float2 a = ffma2(make_float2(pr[i], pr[i + 1]), sc2, make_float2(-l4.x, -l4.y));
            const float2 c = ffma2(make_float2(pr[i + 2], pr[i + 3]), sc2, make_float2(-l4.z, -l4.w));
            pr[i] = ex2_approx(a.x); pr[i + 1] = ex2_approx(a.y); pr[i + 2] = ex2_approx(c.x); pr[i + 3] = ex2_approx(c.y);
          }
          if (need_mask && ((SCORE & b200::SCORE_CAP) || g0 < all_lo || g0 + 32 > all_hi)) {
            const int from = c_lo - c0, to = c_hi - c0;
            const bool out = from >= 32 || to <= 0 || from >= to;
            if (__all_sync(0xffffffffu, out || (from <= 0 && to >= 32))) {      // each key by all of them or by none
#pragma unroll
              for (int i = 0; i < 32; ++i) pr[h * 32 + i] = out ? 0.f : pr[h * 32 + i];
            } else {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (i < from || i >= to) pr[h * 32 + i] = 0.f;
            }
          }
        }
      }
      {
        uint32_t pk[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) pk[i] = pack_bf16x2(pr[2 * i], pr[2 * i + 1]);
        tmem_st_32x32b_x32(tm_S + lane_base + half * 64, pk);
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full);
      }
      if (SCORE & b200::SCORE_CAP) {
#pragma unroll
        for (int i = 0; i < 64; i += 2) {
          const float2 x = fmul2(make_float2(pr[i], pr[i + 1]), make_float2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])));
          pr[i] = x.x; pr[i + 1] = x.y;
        }
      }
      if (!warp_wait(dp_full, it & 1, abort_flag, p.status, 91)) { ok = false; break; }
      tc_fence_after();
      uint8_t* drow = sdS + half * (BKV * 128) + r * 128;       // 64 queries of key r
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t d[32];
        tmem_ld_32x32b_x32(tm_dP + lane_base + half * 64 + c * 32, d);
        tc_wait_ld();
        const float2 s2 = make_float2(p.score.scale, p.score.scale);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float4 d0 = *reinterpret_cast<const float4*>(ld + BQ + c * 32 + g * 8);
          const float4 d1 = *reinterpret_cast<const float4*>(ld + BQ + c * 32 + g * 8 + 4);
          const float dl[8] = {d0.x, d0.y, d0.z, d0.w, d1.x, d1.y, d1.z, d1.w};
          uint32_t w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int i = g * 8 + 2 * j;
            const float2 t2 = ffma2(make_float2(__uint_as_float(d[i]), __uint_as_float(d[i + 1])), s2, make_float2(-dl[2 * j], -dl[2 * j + 1]));
            const float2 g2 = fmul2(make_float2(pr[c * 32 + i], pr[c * 32 + i + 1]), t2);
            w[j] = pack_bf16x2(g2.x, g2.y);
          }
          *reinterpret_cast<uint4*>(drow + (((c * 4 + g) ^ (r & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
      tc_fence_before();
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(ds_full);
      // the next step's staged value, into the buffer of step it - 1: every worker has left that step, since dP(it) was issued
      // after all of them had written dS(it - 1)
      if (it + 1 < n_iter) {
        sLD[((it + 1) & 1) * 2 * BQ + half * BQ + r] = staged(next);
        __syncwarp();
        if (lane == 0) mbar_arrive(&ld_full[(it + 1) & 1]);
      }
    }
    // ------------------------------ dK / dV epilogue ------------------------------
    // workers of half 0 write dK (staged in the dS tile), those of half 1 write dV (staged in the first Q stage)
    if (ok && n_iter > 0) ok = warp_wait(acc_done, 0, abort_flag, p.status, 92);
    if (ok) {
      tc_fence_after();
      uint8_t* tile = (half == 0) ? sdS : sQ;
      uint8_t* dst = tile + r * 128;
      const uint32_t src = (half == 0 ? tm_dK : tm_dV) + lane_base;
#pragma unroll 1
      for (int c = 0; c < HD / 32; ++c) {
        uint32_t v[32];
        if (n_iter > 0) { tmem_ld_32x32b_x32(src + c * 32, v); tc_wait_ld(); }
        else {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = 0u;
        }
        if (p.parts > 1) {                      // fp32, as it is: attn_masked_finish_kernel adds the parts up
          float4* o = reinterpret_cast<float4*>(p.partial + ((((long long)id * p.Hkv + hk) * p.parts + part) * 2 + half) * BKV * HD + r * HD +
                                                c * 32);
#pragma unroll
          for (int g = 0; g < 8; ++g)
            o[g] = make_float4(__uint_as_float(v[4 * g]), __uint_as_float(v[4 * g + 1]), __uint_as_float(v[4 * g + 2]),
                               __uint_as_float(v[4 * g + 3]));
          continue;
        }
        uint8_t* blk = dst + (c / 2) * (BKV * 128);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int sw = (((c & 1) * 4 + g) ^ (r & 7)) << 4;
          *reinterpret_cast<uint4*>(blk + sw) = make_uint4(
              pack_bf16x2(__uint_as_float(v[8 * g]), __uint_as_float(v[8 * g + 1])),
              pack_bf16x2(__uint_as_float(v[8 * g + 2]), __uint_as_float(v[8 * g + 3])),
              pack_bf16x2(__uint_as_float(v[8 * g + 4]), __uint_as_float(v[8 * g + 5])),
              pack_bf16x2(__uint_as_float(v[8 * g + 6]), __uint_as_float(v[8 * g + 7])));
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0 && p.parts == 1 && kv0 + q * 32 < p.Skv) {
#pragma unroll
        for (int i = 0; i < NB; ++i)
          b200::store_4d(half == 0 ? &tmdK : &tmdV, tile + i * (BKV * 128) + q * 32 * 128, i * 64, hk, kv0 + q * 32, b);
        tma_store_commit();
      }
    }
    if (lane == 0) tma_store_wait_all<0>();
  }

  __syncwarp();
  if (*abort_flag) {
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) { tc_fence_after(); tmem_dealloc(tmem_base, 512); }
}

// dK and dV of key tile blockIdx.x / Hkv (b * tiles + tile), head blockIdx.x % Hkv, from its parts, added in their order.
template <int HD>
__global__ void __launch_bounds__(256)
attn_masked_finish_kernel(const float* __restrict__ partial, int parts, int Hkv, int Skv, int nk, __nv_bfloat16* dk, __nv_bfloat16* dv,
                          long long dk_row, long long dv_row, long long dk_batch, long long dv_batch) {
  b200::begin_kernel();
  constexpr int VPR = HD / 8;
  const int hk = (int)blockIdx.x % Hkv, id = (int)blockIdx.x / Hkv, b = id / nk, jt = id - b * nk;
  const float* src = partial + (long long)blockIdx.x * parts * 2 * BKV * HD;
  for (int i = blockIdx.y * 256 + threadIdx.x; i < 2 * BKV * VPR; i += gridDim.y * 256) {
    const int half = i / (BKV * VPR), r = i / VPR % BKV, c = i % VPR * 8, key = jt * BKV + r;
    if (key >= Skv) continue;
    float v[8] = {};
    for (int z = 0; z < parts; ++z) {
      const float* f = src + (long long)z * 2 * BKV * HD + i * 8;
      const float4 x = *reinterpret_cast<const float4*>(f), y = *reinterpret_cast<const float4*>(f + 4);
      v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w; v[4] += y.x; v[5] += y.y; v[6] += y.z; v[7] += y.w;
    }
    __nv_bfloat16* o = half == 0 ? dk + b * dk_batch + (long long)key * dk_row : dv + b * dv_batch + (long long)key * dv_row;
    *reinterpret_cast<uint4*>(o + hk * HD + c) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                                                            pack_bf16x2(v[6], v[7]));
  }
}

// delta[b, h, s] = sum_d (O + low)[b, s, h, d] dO[b, s, h, d], and dq = 0 for the sums that follow; HD / 8 lanes per (token, head), 16-byte loads, of
// DELTA_ROWS rows at once.  All are contiguous.  8192 x 32 x 128: 57 us (335 MB, 5.9 TB/s); one row at
// a time 40, and 19 for a launch that clears dq.
constexpr int DELTA_ROWS = 4;
template <int HD>
__global__ void __launch_bounds__(256)
attn_masked_delta_kernel(const __nv_bfloat16* __restrict__ o, const __nv_bfloat16* __restrict__ low, const __nv_bfloat16* __restrict__ dout,
                         float* __restrict__ delta, float* __restrict__ dq, long long rows, int S, int H) {
  b200::begin_kernel();
  constexpr int LANES = HD / 8, STEP = 256 / LANES;
  const long long w0 = (long long)blockIdx.x * (DELTA_ROWS * STEP) + threadIdx.x / LANES;
  const int l = threadIdx.x % LANES;
  uint4 a[DELTA_ROWS], c[DELTA_ROWS], d[DELTA_ROWS];
#pragma unroll
  for (int k = 0; k < DELTA_ROWS; ++k) {
    const long long w = w0 + k * STEP;
    a[k] = c[k] = d[k] = make_uint4(0u, 0u, 0u, 0u);
    if (w < rows) {
      a[k] = reinterpret_cast<const uint4*>(o)[w * LANES + l];
      c[k] = reinterpret_cast<const uint4*>(low)[w * LANES + l];
      d[k] = reinterpret_cast<const uint4*>(dout)[w * LANES + l];
    }
  }
#pragma unroll
  for (int k = 0; k < DELTA_ROWS; ++k) {
    const long long w = w0 + k * STEP;
    const uint32_t x[4] = {a[k].x, a[k].y, a[k].z, a[k].w}, y[4] = {c[k].x, c[k].y, c[k].z, c[k].w}, z[4] = {d[k].x, d[k].y, d[k].z, d[k].w};
    float acc = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 p = unpack_bf16x2(x[j]), q = unpack_bf16x2(y[j]), g = unpack_bf16x2(z[j]);
      acc += (p.x + q.x) * g.x + (p.y + q.y) * g.y;
    }
#pragma unroll
    for (int off = LANES / 2; off > 0; off >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, off);
    if (w < rows) {
      float4* row = reinterpret_cast<float4*>(dq) + w * (HD / 4) + l;
      row[0] = row[LANES] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (l == 0) {
        const long long h = w % H, t = w / H, s = t % S, b = t / S;
        delta[(b * H + h) * S + s] = acc;
      }
    }
  }
}

template <int HD, int SCORE>
int launch_bwd(const CUtensorMap* m, const BwdParams& p, long long grid, cudaStream_t stream) {
  using SM = Smem<HD>;
  static bool configured[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!configured[dev & 63]) {
    cudaError_t e = cudaFuncSetAttribute(attn_masked_bwd_kernel<HD, SCORE>, cudaFuncAttributeMaxDynamicSharedMemorySize, SM::TOTAL);
    if (e != cudaSuccess) {
      cudaGetLastError();  // clear the sticky error before reporting
      return b200::fail(961, "attn_masked_bwd: cannot set %d bytes of shared memory: %s", SM::TOTAL, cudaGetErrorString(e));
    }
    configured[dev & 63] = true;
  }
  b200::launch(attn_masked_bwd_kernel<HD, SCORE>, (unsigned)grid, NTHREADS, SM::TOTAL, stream, m[0], m[1], m[2], m[3], m[4], m[5], m[6], p);
  b200::count_launch();
  return b200::check_launch("attn_masked_bwd");
}
template <int HD>
int launch_bwd(int score, const CUtensorMap* m, const BwdParams& p, long long grid, cudaStream_t s) {
  switch (score) {
    case b200::SCORE_PLAIN: return launch_bwd<HD, b200::SCORE_PLAIN>(m, p, grid, s);
    case b200::SCORE_CAP: return launch_bwd<HD, b200::SCORE_CAP>(m, p, grid, s);
    case b200::SCORE_BIAS: return launch_bwd<HD, b200::SCORE_BIAS>(m, p, grid, s);
    default: return launch_bwd<HD, b200::SCORE_CAP | b200::SCORE_BIAS>(m, p, grid, s);
  }
}

// CTAs that share a key tile: two to an SM in all at most, of four steps or more each (their fill and the sums behind them cost about three).
// Causal, us with 1 / 2 / 4 / 8: 64 tiles of up to 256 steps 615 / 326 / 180 / 197, 64 of 64 133 / 78 / 56 / 72, 128 of 64 177 / 120 / 146 / 188, 32 of
// 16 48 / 36 / 28 / 37, 256 of 128 361 / 378 / 461 / 581.
int parts_of(int B, int Sq, int Skv, int Hq, int Hkv) {
  const long long tiles = (long long)B * Hkv * ((Skv + BKV - 1) / BKV), steps = (long long)(Hq / Hkv) * ((Sq + BQ - 1) / BQ);
  const long long n = 2ll * b200::sm_count() / tiles, most = steps / 4 < 8 ? steps / 4 : 8, parts = n < most ? n : most;
  return (int)(parts > 1 ? parts : 1);
}

}  // namespace

// bytes of the sums that CTAs sharing a key tile leave (0: every tile has one)
B200_API long long b200_attn_masked_bwd_workspace(int B, int Sq, int Skv, int Hq, int Hkv, int HD) {
  if (!b200::sizes_ok(B, Sq, Skv, Hq, Hkv)) return 0;
  const long long tiles = (long long)B * Hkv * ((Skv + BKV - 1) / BKV);
  const int parts = parts_of(B, Sq, Skv, Hq, Hkv);
  return parts > 1 ? tiles * parts * 2 * BKV * HD * 4 : 0;
}

// q, k, v as in b200_attn_masked_fwd; out, low, dout [B, Sq, Hq, HD] contiguous; delta: fp32 [B, Hq, Sq], written here; dq_acc: fp32
// [B, Sq, Hq, HD] contiguous, cleared here (reduce-add target); dk / dv: bf16 [B, Skv, Hkv, HD] with their own pitches.
B200_API int b200_attn_masked_bwd(const void* q, const void* k, const void* v, const void* out, const void* low, const void* dout, const float* lse,
                                  float* delta, float* dq_acc, void* dk, void* dv, const float* slopes, const int* mask, int B, int Sq, int Skv,
                                  int Hq, int Hkv, int HD, long long q_row, long long k_row, long long v_row, long long dk_row, long long dv_row,
                                  long long q_batch, long long k_batch, long long v_batch, long long dk_batch, long long dv_batch, float scale,
                                  float cap, void* workspace, long long workspace_bytes, void* stream) {
  if (HD != 64 && HD != 128) return b200::fail(960, "attn_masked_bwd: head dim %d not supported (64 or 128)", HD);
  if (!b200::sizes_ok(B, Sq, Skv, Hq, Hkv))
    return b200::fail(960, "attn_masked_bwd: B=%d, Sq=%d, Skv=%d, Hq=%d, Hkv=%d", B, Sq, Skv, Hq, Hkv);
  if (!(scale > 0.f) || !b200::cap_ok(cap)) return b200::fail(960, "attn_masked_bwd: scale %g, cap %g", scale, cap);
  CUtensorMap m[7];
  int r;
  const long long o_row = (long long)Hq * HD, o_batch = o_row * Sq;
  if ((r = b200::map_bshd(&m[0], q, HD, Hq, Sq, B, q_row, q_batch, BQ))) return r;
  if ((r = b200::map_bshd(&m[1], k, HD, Hkv, Skv, B, k_row, k_batch, BKV))) return r;
  if ((r = b200::map_bshd(&m[2], v, HD, Hkv, Skv, B, v_row, v_batch, BKV))) return r;
  if ((r = b200::map_bshd(&m[3], dout, HD, Hq, Sq, B, o_row, o_batch, BQ))) return r;
  if ((r = b200::make_tmap_4d(&m[4], b200::DT_F32, dq_acc, HD, Hq, Sq, B, (uint64_t)HD * 4, (uint64_t)o_row * 4, (uint64_t)o_batch * 4, 32, 1, 32, 1,
                              b200::SWZ_128)))
    return r;
  if ((r = b200::map_bshd(&m[5], dk, HD, Hkv, Skv, B, dk_row, dk_batch, 32))) return r;
  if ((r = b200::map_bshd(&m[6], dv, HD, Hkv, Skv, B, dv_row, dv_batch, 32))) return r;
  const b200::MaskLayout lay = b200::MaskLayout::of(B, Sq, Skv);
  const int nk = lay.Kp / BKV;
  const long long tiles = (long long)B * Hkv * nk;
  BwdParams p;
  p.mask = b200::MaskView::of(mask, lay);
  p.score = b200::ScoreParams::of(scale, cap, slopes);
  p.Hq = Hq; p.Hkv = Hkv; p.Sq = Sq; p.Skv = Skv;
  p.scale_log2 = scale * b200::LOG2E;
  p.lse = lse; p.delta = delta;
  p.status = b200::status_ptr();
  p.parts = parts_of(B, Sq, Skv, Hq, Hkv);
  p.partial = (float*)workspace;
  if (p.parts > 1 && (workspace == nullptr || workspace_bytes < b200_attn_masked_bwd_workspace(B, Sq, Skv, Hq, Hkv, HD)))
    return b200::fail(962, "attn_masked_bwd: a workspace of %lld bytes", workspace_bytes);
  if (tiles * p.parts > 0x7fffffff) return b200::fail(963, "attn_masked_bwd: %lld key tiles", tiles);
  const long long rows = (long long)B * Sq * Hq, blocks = (rows * (HD / 8) + 256 * DELTA_ROWS - 1) / (256 * DELTA_ROWS);
  if (blocks > 0x7fffffff) return b200::fail(963, "attn_masked_bwd: %lld rows", rows);
  cudaStream_t s = (cudaStream_t)stream;
  b200::launch(HD == 128 ? attn_masked_delta_kernel<128> : attn_masked_delta_kernel<64>, (unsigned)blocks, 256, 0, s, (const __nv_bfloat16*)out,
               (const __nv_bfloat16*)low, (const __nv_bfloat16*)dout, delta, dq_acc, rows, Sq, Hq);
  b200::count_launch();
  if ((r = b200::check_launch("attn_masked_delta"))) return r;
  const int score = (cap > 0.f ? b200::SCORE_CAP : 0) | (slopes != nullptr ? b200::SCORE_BIAS : 0);
  if ((r = HD == 128 ? launch_bwd<128>(score, m, p, tiles * p.parts, s) : launch_bwd<64>(score, m, p, tiles * p.parts, s)) || p.parts == 1) return r;
  b200::launch(HD == 128 ? attn_masked_finish_kernel<128> : attn_masked_finish_kernel<64>, dim3((unsigned)tiles, HD / 16), 256, 0, s,
               (const float*)p.partial, p.parts, Hkv, Skv, nk, (__nv_bfloat16*)dk, (__nv_bfloat16*)dv, dk_row, dv_row, dk_batch, dv_batch);
  b200::count_launch();
  return b200::check_launch("attn_masked_finish");
}
