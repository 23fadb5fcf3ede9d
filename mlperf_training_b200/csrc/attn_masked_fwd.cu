// Attention with the masks of attn_mask.cuh (documents, prefix, window, causal, padding), capped scores and a distance bias: the forward
// engine of attention_fwd.cu (two query tiles a CTA in ping-pong, S and O in TMEM, P as a TMEM operand, lazy rescaling) with
//
//   s = scale q k     s = cap tanh(s / cap)     s -= slope_h |p - j|     O = softmax over the visible j of s, times V
//
//   * the key tiles of an item, and which of them hold anything to mask, from the mask's tables; items of all sequences longest first;
//   * few pairs of query tiles over many keys: their key tiles in parts, joined by a second launch;
//   * rows that see nothing: output 0, log-sum-exp -inf, whatever their inputs; a value row that no query sees is cleared in shared memory before
//     the product (its probability is 0, but 0 times NaN is not);
//   * for a backward pass and in parts, the sum of a row is taken over the rounded probabilities that the second product multiplies.  The output
//     is then a mean with weights that sum to 1, and a row with one dominant key is as exact as any other (before: error of dQ and dK up
//     to 0.7 % with scores of standard deviation 4, now 0.26, with the next point).  Without a backward pass it is taken over the
//     probabilities before their rounding: weights sum to 1 within 2^-9, and an output is off by 0.0018 of its size instead of 0.0017
//     (the other sum took 494 -> 513 us for 8192 tokens of one document, 84 -> 89 for 16, 822 -> 910 with a cap);
//   * for a backward pass, what the output loses to bf16, as a second bf16 tensor (delta = rowsum(dO O) is formed from both), and the log-sum-exp
//     of the probabilities before their rounding (dQ's error at standard deviation 2.25 0.250 % with that of the rounded ones, 0.244 with it; of
//     that 0.235 are the two roundings to bf16 that no order of the sums avoids, of dS and of dQ itself);
//   * capped scores by a polynomial (attn_masked.cuh): 8192 tokens, 32 heads, cap 50 822 us, 867 for a backward pass.
// 8192 tokens, 32 heads of 128 on 8, causal: 504 us (1.09 PFLOP/s), 525 for a backward pass.  Bound by the softmax of the two tiles and its
// turns with the products (2.4 us a key tile of both, of which 1.1 are exponentials at 16 a clock and SM); with 16 documents in those tokens 100 us,
// 14.7 an item, of which 6 are its key tiles' and the others the first products and the output of each.
#include "attn_masked.cuh"

namespace {

constexpr int BQ = 128;   // query rows per tile (two tiles per CTA)
constexpr int BKV = 128;  // keys per tile
constexpr int NTHREADS = 384;  // warps 0-3 / 4-7: softmax of tile 0 / 1; warp 8: TMA; warp 9: MMA
constexpr int PV_EARLY = 96;   // keys of P the second GEMM starts on
// 3 x 128 threads launch with 168 registers each (504 per triple): 104 + 2 x 200 (56 or 72 for the other warps spilled)
constexpr int REGS_SOFTMAX = 200, REGS_OTHER = 104;

struct FwdParams {
  b200::MaskView mask;
  b200::ScoreParams score;
  int Hq, Hkv, Sq, Skv;
  float scale_log2;   // softmax scale * log2(e)
  const float* sink;  // [Hq] learned sink logits (natural-log domain, unscaled) or null
  float* lse;         // [B, Hq, Sq] natural-log log-sum-exp of the scores
  __nv_bfloat16* out; // [B, Sq, Hq, HD] (rows that see nothing are written from here)
  __nv_bfloat16* low; // the same: what `out` has lost to bf16; or null
  int* status;
  int items;
  int parts, per;     // SPLIT: items for a pair's key tiles, each of them for `per` tiles or more (a pair of no more than that has one)
  float* part;        // SPLIT: [rows][parts][HD], rows = (b * Sq + q) * Hq + h: sums of values on the part's maximum
  float4* part_ml;    // SPLIT: [rows][parts]: maximum (log2), sum of the rounded probabilities and of those before
};

// Work item u of the launch (items go by the mask's order, over the heads of one pair of query tiles after the other, SPLIT: and over the parts of its
// key tiles), and the key tiles its two query tiles look at.
struct Item {
  int b, h, q0, j_lo;
  int lo0, lo1, hi0, hi1;   // per query tile: key tiles j_lo + [lo, hi); every tile of [0, n_max) is in one of them
  int n_max;
  bool unseen;              // some keys are seen by no query
  int mlo0, mlo1, mhi0, mhi1;   // per query tile: keys in [mlo, mhi) are visible to all of its rows
  int part, parts;
  B200_DEVICE int lo(int t) const { return t ? lo1 : lo0; }
  B200_DEVICE int hi(int t) const { return t ? hi1 : hi0; }
};
// What the mask's tables say about item u.  The roles load it an item ahead: two loads in a row, more than a key tile's time.
// Parts of the key tiles [x, y) that either tile of a pair looks at.
struct Union { int x, y; };
B200_DEVICE Union union_of(int4 a, int4 c) {
  a.y &= ~b200::UNSEEN;
  c.y &= ~b200::UNSEEN;
  const int x = a.y > a.x ? (c.y > c.x ? min(a.x, c.x) : a.x) : c.x;
  return {x, max(max(a.y, c.y), x)};
}
B200_DEVICE int parts_of(Union u, const FwdParams& p) { return min(max((u.y - u.x + p.per - 1) / p.per, 1), p.parts); }
struct Entry {
  int id = 0;
  int4 a = {0, 0, 0, 0}, c = {0, 0, 0, 0};
};
template <bool SPLIT>
B200_DEVICE Entry load_entry(int u, const FwdParams& p) {
  Entry e;
  if (u >= p.items) return e;
  e.id = p.mask.oq[SPLIT ? u / (p.Hq * p.parts) : u / p.Hq];                            // b * pairs + pair: its query tiles are entries 2 id and 2 id + 1
  e.a = p.mask.qt[2ll * e.id];
  e.c = p.mask.qt[2ll * e.id + 1];
  return e;
}
template <bool SPLIT>
B200_DEVICE Item make_item(int u, const Entry& e, const FwdParams& p) {
  Item it;
  const int np = p.mask.Sp / 256;
  it.part = SPLIT ? u % p.parts : 0;
  it.h = (SPLIT ? u / p.parts : u) % p.Hq;
  it.b = e.id / np;
  const int pair = e.id - it.b * np;
  it.q0 = pair * 2 * BQ;
  int4 a = e.a, c = e.c;
  it.unseen = (a.y & b200::UNSEEN) != 0;
  a.y &= ~b200::UNSEEN;
  c.y &= ~b200::UNSEEN;
  it.parts = 1;
  if (SPLIT) {                                           // this part of the key tiles (none: behind the last)
    const Union w = union_of(a, c);
    it.parts = parts_of(w, p);
    const int n = w.y - w.x, z = min(it.part, it.parts), j0 = w.x + n * z / it.parts, j1 = w.x + n * min(z + 1, it.parts) / it.parts;
    a.x = max(a.x, j0); a.y = min(a.y, j1);
    c.x = max(c.x, j0); c.y = min(c.y, j1);
  }
  const bool has0 = a.y > a.x, has1 = c.y > c.x;
  it.j_lo = has0 ? a.x : c.x;
  it.lo0 = 0;
  it.hi0 = has0 ? a.y - a.x : 0;
  it.lo1 = has0 ? min(c.x - it.j_lo, it.hi0) : 0;       // (tiles between the two ranges are the second one's, all masked)
  it.hi1 = c.y - it.j_lo;
  if (!has1) it.lo1 = it.hi1 = 0;
  it.n_max = max(it.hi0, it.hi1);
  it.mlo0 = a.z; it.mhi0 = a.w; it.mlo1 = c.z; it.mhi1 = c.w;
  return it;
}
// Items of CTA blockIdx.x: one per round of gridDim.x items, in alternating direction.
B200_DEVICE int item_of_round(int r) {
  return r * (int)gridDim.x + ((r & 1) ? (int)(gridDim.x - 1 - blockIdx.x) : (int)blockIdx.x);
}

B200_DEVICE float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

template <int HD>
struct Smem {
  static constexpr int Q_TILE = BQ * HD * 2;
  static constexpr int KV_BYTES = BKV * HD * 2;
  static constexpr int STAGE_O = 32 * 128;            // per softmax warp: 32 rows x 64 output columns
  static constexpr int TOTAL = 2 * Q_TILE + 4 * KV_BYTES + 8 * STAGE_O + 1024 + 256;
};

// LOW: what the output loses to bf16 is written too, and row sums go over the rounded probabilities (a backward pass follows).  SPLIT (with
// LOW's sums): items are parts of pairs, and leave their sums for attn_masked_parts_kernel.
template <int HD, int SCORE, bool LOW, bool SPLIT>
__global__ void __launch_bounds__(NTHREADS, 1)
attn_masked_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmO,
                const __grid_constant__ CUtensorMap tmLow, const __grid_constant__ FwdParams p) {
  b200::begin_kernel();
  using SM = Smem<HD>;
  constexpr int NB = HD / 64;  // 64-column (128-byte) blocks per head row
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                       // two tiles
  uint8_t* sK = sQ + 2 * SM::Q_TILE;        // two stages
  uint8_t* sV = sK + 2 * SM::KV_BYTES;      // two stages
  uint8_t* sO = sV + 2 * SM::KV_BYTES;      // eight warps' output staging
  uint64_t* bars = reinterpret_cast<uint64_t*>(sO + 8 * SM::STAGE_O);
  uint64_t* q_full = bars;          // 1
  uint64_t* q_empty = bars + 1;     // 1: every S of the item has been computed
  uint64_t* k_full = bars + 2;      // 2
  uint64_t* k_empty = bars + 4;     // 2
  uint64_t* v_full = bars + 6;      // 2
  uint64_t* v_empty = bars + 8;     // 2
  uint64_t* s_full = bars + 10;     // 2 (per query tile): once per key tile
  uint64_t* p_early = bars + 12;    // 2 (4 arrivals): the first PV_EARLY keys of P are in TMEM
  uint64_t* p_full = bars + 14;     // 2 (4 arrivals): all of P
  uint64_t* o_done = bars + 16;     // 2: once per item, O complete
  uint64_t* o_free = bars + 18;     // 2 (4 arrivals): once per item, O read out of TMEM
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars + 20);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int off = p.Skv - p.Sq;
  const int rounds = (p.items + (int)gridDim.x - 1) / (int)gridDim.x;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1); mbar_init(q_empty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 1); mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1); mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1); mbar_init(&p_early[i], 4); mbar_init(&p_full[i], 4);
      mbar_init(&o_done[i], 1); mbar_init(&o_free[i], 4);
    }
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 9) { tmem_alloc(tmem_holder, 512); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;

  if (warp >= 8) {
    reg_dealloc<REGS_OTHER>();
    if (warp == 8 && lane == 0) {
      // ------------------------------ TMA producer ------------------------------
      tma_prefetch_desc(&tmQ); tma_prefetch_desc(&tmK); tma_prefetch_desc(&tmV);
      bool ok = true;
      int kv = 0, nq = 0;                    // key tiles and items so far: stage and phase of the barriers
      Entry next = load_entry<SPLIT>(item_of_round(0), p);
      for (int r = 0; r < rounds && ok; ++r) {
        const int u = item_of_round(r);
        if (u >= p.items) continue;
        const Item it = make_item<SPLIT>(u, next, p);
        next = load_entry<SPLIT>(item_of_round(r + 1), p);
        if (it.n_max == 0) continue;
        const int hk = it.h / (p.Hq / p.Hkv);
        if (!mbar_wait(q_empty, (nq & 1) ^ 1, abort_flag, p.status, 39)) { ok = false; break; }
        ++nq;
        mbar_expect_tx(q_full, 2 * SM::Q_TILE);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < NB; ++i)
            b200::load_4d(sQ + t * SM::Q_TILE + i * (BQ * 128), &tmQ, q_full, i * 64, it.h, it.q0 + t * BQ, it.b);
        for (int n = 0; n < it.n_max; ++n, ++kv) {
          const int j = it.j_lo + n, st = kv & 1;
          const uint32_t ph = (kv >> 1) & 1;
          if (!mbar_wait(&k_empty[st], ph ^ 1, abort_flag, p.status, 40)) { ok = false; break; }
          mbar_expect_tx(&k_full[st], SM::KV_BYTES);
#pragma unroll
          for (int i = 0; i < NB; ++i)
            b200::load_4d(sK + st * SM::KV_BYTES + i * (BKV * 128), &tmK, &k_full[st], i * 64, hk, j * BKV, it.b);
          if (!mbar_wait(&v_empty[st], ph ^ 1, abort_flag, p.status, 41)) { ok = false; break; }
          mbar_expect_tx(&v_full[st], SM::KV_BYTES);
#pragma unroll
          for (int i = 0; i < NB; ++i)
            b200::load_4d(sV + st * SM::KV_BYTES + i * (BKV * 128), &tmV, &v_full[st], i * 64, hk, j * BKV, it.b);
        }
      }
    } else if (warp == 9) {
      // ------------------------------ MMA issuer ------------------------------
      // The whole warp walks the schedule and one elected lane issues: the operands of the instructions then stay in
      // uniform registers (descriptors advance by an addition).
      const uint32_t idesc_s = umma_idesc(1, 1, 0, 0, BQ, BKV);  // Q (K-major) x K (K-major)
      const uint32_t idesc_o = umma_idesc(1, 1, 0, 1, BQ, HD);   // P (TMEM)    x V (MN-major)
      const uint64_t dQ = umma_desc_sw128(smem_u32(sQ), 16, 1024), dK = umma_desc_sw128(smem_u32(sK), 16, 1024);
      const uint64_t dV = umma_desc_sw128(smem_u32(sV), BKV * 128, 1024);
      bool ok = true;
      int kv = 0, nq = 0;
      int np[2] = {0, 0}, no[2] = {0, 0};    // P tiles consumed / items finished per query tile
      Entry next = load_entry<SPLIT>(item_of_round(0), p);
      for (int r = 0; r < rounds && ok; ++r) {
        const int u = item_of_round(r);
        if (u >= p.items) continue;
        const Item it = make_item<SPLIT>(u, next, p);
        next = load_entry<SPLIT>(item_of_round(r + 1), p);
        if (it.n_max == 0) continue;
        if (!warp_wait_spin(q_full, nq & 1, abort_flag, p.status, 50)) { ok = false; break; }
        ++nq;
        int k_ready = -1, v_ready = -1;      // last key tile of the item whose full barrier has been observed
        int s_left = (it.hi0 - it.lo0) + (it.hi1 - it.lo1);
        // S_t(n) = Q_t K(n)^T into the S columns of tile t
        auto issue_s = [&](int t, int n) -> bool {
          const int st = (kv + n) & 1;
          while (k_ready < n) {
            ++k_ready;
            if (!warp_wait_spin(&k_full[(kv + k_ready) & 1], ((kv + k_ready) >> 1) & 1, abort_flag, p.status, 51)) return false;
          }
          // the last S that reads K(n) frees its stage: S_t(n) is issued in step n - 1, tile 0 first; a tile's first one, of the two
          // key tiles that are there at the start, before step 0
          const int o = 1 - t;
          const bool both = n >= it.lo(o) && n < it.hi(o);
          const int mine = n == it.lo(t) && n <= 1 ? -1 : n - 1, theirs = n == it.lo(o) && n <= 1 ? -1 : n - 1;
          const bool free_k = !both || mine > theirs || (mine == theirs && t == 1);
          const bool free_q = --s_left == 0;
          tc_fence_after();
          if (elect_one()) {
            const uint64_t ad = dQ + (t * SM::Q_TILE >> 4), bd = dK + (st * SM::KV_BYTES >> 4);
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk) {
              const uint32_t o4 = ((kk / 4) * (BQ * 128) + (kk % 4) * 32) >> 4;
              tc_mma_f16_ss(tmem_base + t * 128, ad + o4, bd + o4, idesc_s, kk > 0 ? 1u : 0u);
            }
            tc_commit(&s_full[t]);
            if (free_k) tc_commit(&k_empty[st]);
            if (free_q) tc_commit(q_empty);
          }
          __syncwarp();
          return true;
        };
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if (ok && it.lo(t) <= 1 && it.hi(t) > it.lo(t)) ok = issue_s(t, it.lo(t));
        for (int n = 0; n < it.n_max && ok; ++n) {
          const int st = (kv + n) & 1;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (ok && n > 0 && n + 1 == it.lo(t) && it.hi(t) > it.lo(t)) ok = issue_s(t, n + 1);      // (K has two stages: not before)
            if (!ok || n < it.lo(t) || n >= it.hi(t)) continue;
            const bool first = n == it.lo(t), last = n == it.hi(t) - 1;
            // O of the previous item has left TMEM
            if (first && !warp_wait_spin(&o_free[t], (no[t] & 1) ^ 1, abort_flag, p.status, 52)) { ok = false; continue; }
            while (ok && v_ready < n) {
              ++v_ready;
              ok = warp_wait_spin(&v_full[(kv + v_ready) & 1], ((kv + v_ready) >> 1) & 1, abort_flag, p.status, 54);
            }
            ok = ok && warp_wait_spin(&p_early[t], np[t] & 1, abort_flag, p.status, 53);
            if (!ok) continue;
            tc_fence_after();
            // A = P_t in TMEM: 16 bf16 keys = 8 columns per step; B = V: 16 key rows of 128 bytes
            const uint64_t bd = dV + (st * SM::KV_BYTES >> 4);
            if (elect_one()) {
#pragma unroll
              for (int kk = 0; kk < PV_EARLY / 16; ++kk)
                tc_mma_f16_ts(tmem_base + 256 + t * 128, tmem_base + t * 128 + kk * 8, bd + (kk * (16 * 128) >> 4), idesc_o,
                              (!first || kk > 0) ? 1u : 0u);
            }
            __syncwarp();
            ok = warp_wait_spin(&p_full[t], np[t] & 1, abort_flag, p.status, 55);
            if (!ok) continue;
            tc_fence_after();
            const bool free_v = (t == 1) || !(n >= it.lo1 && n < it.hi1);
            if (elect_one()) {
#pragma unroll
              for (int kk = PV_EARLY / 16; kk < BKV / 16; ++kk)
                tc_mma_f16_ts(tmem_base + 256 + t * 128, tmem_base + t * 128 + kk * 8, bd + (kk * (16 * 128) >> 4), idesc_o, 1u);
              if (last) tc_commit(&o_done[t]);
              if (free_v) tc_commit(&v_empty[st]);
            }
            __syncwarp();
            ++np[t];
            if (last) ++no[t];
            else ok = issue_s(t, n + 1);
          }
        }
        kv += it.n_max;
      }
    }
  } else {
    // ------------------------------ softmax + epilogue (one warpgroup per query tile) --------------
    reg_alloc<REGS_SOFTMAX>();
    const int t = warp >> 2;
    const int q = warp & 3;
    const int r = q * 32 + lane;           // row inside the query tile
    const uint32_t lane_base = uint32_t(q * 32) << 16;
    const uint32_t ts = tmem_base + lane_base + t * 128;        // S / P columns of this tile
    const uint32_t to = tmem_base + lane_base + 256 + t * 128;  // O columns of this tile
    uint8_t* stage = sO + warp * SM::STAGE_O;
    int ns = 0, no = 0;                    // S tiles and items so far
    int kv = 0;                            // key tiles before this item: stages and phases of V
    bool ok = true;
    Entry next = load_entry<SPLIT>(item_of_round(0), p);
    // (row r of the pair's tile t: pairs are 256 rows of the padded queries in order)
    auto load_row = [&](const Entry& e) { return p.mask.q_iv[256ll * e.id + t * BQ + r]; };
    int2 row_next = load_row(next);
    for (int round = 0; round < rounds && ok; ++round) {
      const int u = item_of_round(round);
      if (u >= p.items) continue;
      const Item it = make_item<SPLIT>(u, next, p);
      const int qt0 = it.q0 + t * BQ;
      const int q_pos = qt0 + r;
      const int kv_item = kv;
      kv += it.n_max;
      if (it.hi(t) <= it.lo(t)) {            // no row of the tile sees anything
        if (SPLIT && (it.parts > 1 || it.part > 0)) {
          if (it.part < it.parts && q_pos < p.Sq)
            p.part_ml[(((long long)it.b * p.Sq + q_pos) * p.Hq + it.h) * p.parts + it.part] = make_float4(-INFINITY, 0.f, 0.f, 0.f);
        } else if (q_pos < p.Sq) {
          const long long at = (((long long)it.b * p.Sq + q_pos) * p.Hq + it.h) * HD;
#pragma unroll
          for (int i = 0; i < HD / 8; ++i) {
            *reinterpret_cast<uint4*>(p.out + at + 8 * i) = make_uint4(0u, 0u, 0u, 0u);
            if (LOW && (!SPLIT || p.low != nullptr)) *reinterpret_cast<uint4*>(p.low + at + 8 * i) = make_uint4(0u, 0u, 0u, 0u);
          }
          p.lse[((long long)it.b * p.Hq + it.h) * p.Sq + q_pos] = p.sink != nullptr ? p.sink[it.h] : -INFINITY;
        }
        next = load_entry<SPLIT>(item_of_round(round + 1), p);
        row_next = load_row(next);
        continue;
      }
      const int2 seen = row_next;            // keys [x, y) of this row
      const int mlo = t ? it.mlo1 : it.mlo0, mhi = t ? it.mhi1 : it.mhi0;
      const float slope2 = (SCORE & b200::SCORE_BIAS) ? p.score.slopes[it.h] * b200::LOG2E : 0.f;
      // no row of the warp sees a key behind itself: the distance needs no absolute value, and the bias is two sums a pair
      const bool behind = (SCORE & b200::SCORE_BIAS) && __all_sync(0xffffffffu, seen.y <= q_pos + off + 1);
      float m_ref = -INFINITY, l = 0.f;      // (l: of the probabilities that are multiplied)
      float lx = 0.f;                        // LOW: of the probabilities before their rounding, for the log-sum-exp
      for (int n = it.lo(t); n < it.hi(t); ++n, ++ns) {
        const int kv0 = (it.j_lo + n) * BKV;
        const bool need_mask = kv0 < mlo || kv0 + BKV > mhi;
        bool unseen = false;                 // key kv0 + r, by every query (such a key lies in masked tiles alone)
        if (need_mask && it.unseen) {
          const int2 by = p.mask.k_iv[(long long)it.b * p.mask.Kp + kv0 + r];
          unseen = by.x >= by.y && kv0 + r < p.Skv;
        }
        if (!warp_wait(&s_full[t], ns & 1, abort_flag, p.status, 60)) { ok = false; break; }
        tc_fence_after();
        if (__any_sync(0xffffffffu, unseen)) {
          // both warpgroups may clear the row: each before its own product reads it, and what is read is 0 either way
          if (!warp_wait(&v_full[(kv_item + n) & 1], ((kv_item + n) >> 1) & 1, abort_flag, p.status, 61)) { ok = false; break; }
          if (unseen) {
            uint8_t* vr = sV + ((kv_item + n) & 1) * SM::KV_BYTES + r * 128;
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
              for (int g = 0; g < 8; ++g) *reinterpret_cast<uint4*>(vr + i * (BKV * 128) + g * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
          fence_proxy_async_smem();
        }
        // the whole score row (128 fp32) comes into registers with one TMEM round trip
        uint32_t v[BKV];
#pragma unroll
        for (int c = 0; c < BKV / 32; ++c) tmem_ld_32x32b_x32(ts + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&v[c * 32]));
        tc_wait_ld();
        if (SCORE & b200::SCORE_CAP) {
          // cap * tanh(s / cap), in units of log2
#pragma unroll
          for (int c = 0; c < BKV / 32; ++c) {
            float big = 0.f;
#pragma unroll
            for (int i = 0; i < 32; i += 2)
              big = max3(big, fabsf(__uint_as_float(v[c * 32 + i])), fabsf(__uint_as_float(v[c * 32 + i + 1])));
            if (__all_sync(0xffffffffu, big <= p.score.limit)) {
#pragma unroll
              for (int i = c * 32; i < c * 32 + 32; i += 2) {
                const float2 y = b200::capped_small2(make_float2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), p.score);
                v[i] = __float_as_uint(y.x); v[i + 1] = __float_as_uint(y.y);
              }
            } else {
#pragma unroll
              for (int i = c * 32; i < c * 32 + 32; i += 2) {
                const float2 y = b200::capped_any2(make_float2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), p.score);
                v[i] = __float_as_uint(y.x); v[i + 1] = __float_as_uint(y.y);
              }
            }
          }
        }
        if (SCORE & b200::SCORE_BIAS) {
          const float d0 = (float)(kv0 - q_pos - off);
          if (behind) {
            // (slope d0 + slope i: what it rounds is 2^-24 of the bias, like the score's own rounding)
            const float base = slope2 * d0, sc = (SCORE & b200::SCORE_CAP) ? 1.f : p.scale_log2;
#pragma unroll
            for (int i = 0; i < BKV; i += 2) {
              const float2 y = ffma2(make_float2(slope2, slope2), make_float2((float)i, (float)(i + 1)), make_float2(base, base));
              const float2 x = ffma2(make_float2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), make_float2(sc, sc), y);
              v[i] = __float_as_uint(x.x); v[i + 1] = __float_as_uint(x.y);
            }
          } else {
#pragma unroll
            for (int i = 0; i < BKV; ++i) {
              const float x = (SCORE & b200::SCORE_CAP) ? __uint_as_float(v[i]) : __uint_as_float(v[i]) * p.scale_log2;
              v[i] = __float_as_uint(fmaf(-slope2, fabsf(d0 + (float)i), x));
            }
          }
        }
        // Where each row of the warp sees all of the tile or nothing of it (documents that begin among its rows), the rows that see nothing
        // are taken out as rows, below; else an element at a time.  (A last tile with two documents among its rows had comparisons in every
        // step: 8192 x 32 heads, one document 540 us, with 57 tokens of another behind it 710, now 540 too.)
        bool out = false;                    // this row sees nothing of the tile
        bool by_element = false;
        if (need_mask) {
          out = kv0 >= seen.y || kv0 + BKV <= seen.x;
          by_element = !__all_sync(0xffffffffu, (out && !it.unseen) || (kv0 >= seen.x && kv0 + BKV <= seen.y));
        }
        if (by_element) {
          // visible: |i - mid| < half (one comparison; whole and half numbers, exact)
          const float from = (float)max(seen.x - kv0, -1), to = (float)min(seen.y - kv0, BKV + 1);
          const float mid = 0.5f * (from + to) - 0.5f, half = seen.y > seen.x ? 0.5f * (to - from) : 0.f;
#pragma unroll
          for (int i = 0; i < BKV; ++i)
            if (!(fabsf((float)i - mid) < half)) v[i] = 0xff800000u;  // -inf
        }
        float mx4[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) mx4[c] = fmaxf(__uint_as_float(v[2 * c]), __uint_as_float(v[2 * c + 1]));
#pragma unroll
        for (int i = 8; i < BKV; i += 8)
#pragma unroll
          for (int c = 0; c < 4; ++c) mx4[c] = max3(mx4[c], __uint_as_float(v[i + 2 * c]), __uint_as_float(v[i + 2 * c + 1]));
        float mx = fmaxf(max3(mx4[0], mx4[1], mx4[2]), mx4[3]);
        if (SCORE == b200::SCORE_PLAIN) mx *= p.scale_log2;  // -inf stays -inf (scale > 0)
        if (out) mx = -INFINITY;
        // lazy rescale: move the reference maximum only when it grew by more than 2^8
        const bool grow = (mx > m_ref + 8.f) || (m_ref == -INFINITY && mx > -INFINITY);
        if (__any_sync(0xffffffffu, grow)) {
          const float m_new = fmaxf(m_ref, mx);
          const float alpha = (m_ref == -INFINITY) ? 0.f : ex2_approx(m_ref - m_new);
          m_ref = m_new;
          l *= alpha;
          lx *= alpha;
          if (n > it.lo(t)) {
            // (S of this key tile was issued after P V of the one before it and completes after it: O is complete)
#pragma unroll 1
            for (int c = 0; c < HD / 32; ++c) {
              uint32_t o[32];
              tmem_ld_32x32b_x32(to + c * 32, o);
              tc_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              tmem_st_32x32b_x32(to + c * 32, o);
            }
            tc_wait_st();
          }
        }
        const float m_use = (m_ref == -INFINITY) ? 0.f : m_ref;
        // P = exp2(S * scale - m) as bf16 pairs over the first half of the S columns; -inf gives 0.  (All by ex2.approx: with every fourth
        // pair by a polynomial, as in attention_fwd.cu, 8192 x 32 heads took 519 us instead of 504: the sums leave the FMA pipe no room.)
        const float scale2 = SCORE == b200::SCORE_PLAIN ? p.scale_log2 : 1.f;
        const float2 sc2 = make_float2(scale2, scale2);
        const float nm = out ? -INFINITY : -m_use;             // (a row that is out: 2^-inf throughout)
        const float2 nm2 = make_float2(nm, nm);
        float2 x2 = make_float2(0.f, 0.f);
#pragma unroll
        for (int c = 0; c < BKV / 32; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int e = c * 32 + 2 * i;
            const float2 a = ffma2(make_float2(__uint_as_float(v[e]), __uint_as_float(v[e + 1])), sc2, nm2);
            const float2 x = make_float2(ex2_approx(a.x), ex2_approx(a.y));
            pk[i] = pack_bf16x2(x.x, x.y);
            if (LOW) x2 = fadd2(x2, x);
            v[e] = LOW ? pk[i] << 16 : __float_as_uint(x.x);
            v[e + 1] = LOW ? pk[i] & 0xffff0000u : __float_as_uint(x.y);
          }
          tmem_st_32x32b_x16(ts + c * 16, pk);
          if (c == PV_EARLY / 32 - 1 || c == BKV / 32 - 1) {
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(c == BKV / 32 - 1 ? &p_full[t] : &p_early[t]);
          }
        }
        // the row sum, off the path of the MMAs
        float2 rs2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int i = 0; i < BKV / 2; ++i)
          rs2[i & 1] = fadd2(rs2[i & 1], make_float2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])));
        l += (rs2[0].x + rs2[0].y) + (rs2[1].x + rs2[1].y);
        lx += x2.x + x2.y;
      }
      // ------------------------------ epilogue ------------------------------
      next = load_entry<SPLIT>(item_of_round(round + 1), p);          // (not before: the scores take the registers)
      if (!ok || !warp_wait(&o_done[t], no & 1, abort_flag, p.status, 62)) { ok = false; break; }
      ++no;
      tc_fence_after();
      row_next = load_row(next);
      if (SPLIT && it.parts > 1) {
        const long long at = (((long long)it.b * p.Sq + q_pos) * p.Hq + it.h) * p.parts + it.part;
        if (q_pos < p.Sq) p.part_ml[at] = make_float4(m_ref, l, lx, 0.f);
#pragma unroll 1
        for (int i = 0; i < HD / 32; ++i) {
          uint32_t v[32];
          tmem_ld_32x32b_x32(to + i * 32, v);
          tc_wait_ld();
          if (i == HD / 32 - 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&o_free[t]);
          }
          if (q_pos < p.Sq)
#pragma unroll
            for (int g = 0; g < 8; ++g)
              *reinterpret_cast<uint4*>(p.part + at * HD + i * 32 + g * 4) = make_uint4(v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]);
        }
        continue;
      }
      const bool none = m_ref == -INFINITY;                   // a row that sees nothing
      if (p.sink != nullptr) {
        const float sk = p.sink[it.h] * 1.4426950408889634f;
        if (m_ref == -INFINITY) { m_ref = sk; l = lx = 1.f; }
        else { l += ex2_approx(sk - m_ref); lx += ex2_approx(sk - m_ref); }
      }
      const float inv = l > 0.f ? 1.f / l : 0.f;
      if (q_pos < p.Sq)
        p.lse[((long long)it.b * p.Hq + it.h) * p.Sq + q_pos] =
            (l > 0.f) ? (m_ref + log2f(LOW ? lx : l)) * 0.6931471805599453f : -INFINITY;
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        uint32_t v[64];
        tmem_ld_32x32b_x32(to + i * 64, *reinterpret_cast<uint32_t(*)[32]>(&v[0]));
        tmem_ld_32x32b_x32(to + i * 64 + 32, *reinterpret_cast<uint32_t(*)[32]>(&v[32]));
        tc_wait_ld();
        if (i == NB - 1) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&o_free[t]);
        }
#pragma unroll
        for (int c = 0; c < 64; ++c) v[c] = none ? 0u : __float_as_uint(__uint_as_float(v[c]) * inv);
#pragma unroll 1
        for (int part = 0; part < (LOW && (!SPLIT || p.low != nullptr) ? 2 : 1); ++part) {
          if (lane == 0) tma_store_wait_read<0>();     // the block before has left the staging buffer
          __syncwarp();
#pragma unroll
          for (int g = 0; g < 8; ++g) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              float x = __uint_as_float(v[8 * g + 2 * j]), y = __uint_as_float(v[8 * g + 2 * j + 1]);
              w[j] = pack_bf16x2(x, y);
              v[8 * g + 2 * j] = __float_as_uint(x - __uint_as_float(w[j] << 16));
              v[8 * g + 2 * j + 1] = __float_as_uint(y - __uint_as_float(w[j] & 0xffff0000u));
            }
            *reinterpret_cast<uint4*>(stage + lane * 128 + ((g ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            if (qt0 + q * 32 < p.Sq) b200::store_4d(part == 0 ? &tmO : &tmLow, stage, i * 64, it.h, qt0 + q * 32, it.b);
            tma_store_commit();
          }
        }
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
  if (warp == 9) { tc_fence_after(); tmem_dealloc(tmem_base, 512); }
}

// Joins the parts of 8 rows of a pair of query tiles and a head, a warp a row; LOW as above.
template <int HD, bool LOW>
__global__ void __launch_bounds__(256) attn_masked_parts_kernel(const __grid_constant__ FwdParams p) {
  b200::begin_kernel();
  const int lane = threadIdx.x & 31, h = (int)blockIdx.x % p.Hq, id = (int)blockIdx.x / p.Hq, np = p.mask.Sp / 256, b = id / np;
  const int parts = parts_of(union_of(p.mask.qt[2ll * id], p.mask.qt[2ll * id + 1]), p);
  if (parts == 1) return;                                // written by the item itself
  const int q = (id - b * np) * 256 + (int)blockIdx.y * 8 + (int)(threadIdx.x >> 5);
  if (q >= p.Sq) return;
  const long long at = ((long long)b * p.Sq + q) * p.Hq + h;
  const float4 ml = lane < parts ? p.part_ml[at * p.parts + lane] : make_float4(-INFINITY, 0.f, 0.f, 0.f);
  float m = warp_max(ml.x);
  const bool none = m == -INFINITY;
  const float f = ml.x == -INFINITY ? 0.f : ex2_approx(ml.x - m);
  // (a part that the row sees nothing of may hold what an infinity made of its sums)
  float l = warp_sum(f == 0.f ? 0.f : ml.y * f), lx = warp_sum(f == 0.f ? 0.f : ml.z * f), acc[HD / 32] = {};
  for (int z = 0; z < parts; ++z) {
    const float w = __shfl_sync(0xffffffffu, f, z);
    if (w == 0.f) continue;
#pragma unroll
    for (int c = 0; c < HD / 32; ++c) acc[c] += w * p.part[(at * p.parts + z) * HD + c * 32 + lane];
  }
  if (p.sink != nullptr) {
    const float sk = p.sink[h] * b200::LOG2E;
    if (none) { m = sk; l = lx = 1.f; }
    else { l += ex2_approx(sk - m); lx += ex2_approx(sk - m); }
  }
  const float inv = none ? 0.f : 1.f / l;
#pragma unroll
  for (int c = 0; c < HD / 32; ++c) {
    const float x = none ? 0.f : acc[c] * inv;
    const __nv_bfloat16 o = __float2bfloat16(x);
    p.out[at * HD + c * 32 + lane] = o;
    if (LOW) p.low[at * HD + c * 32 + lane] = __float2bfloat16(x - __bfloat162float(o));
  }
  if (lane == 0) p.lse[((long long)b * p.Hq + h) * p.Sq + q] = l > 0.f ? (m + log2f(lx)) * 0.6931471805599453f : -INFINITY;
}

// Items for a pair's key tiles: two to an SM in all at most, of four key tiles or more each, where what the longest pair could save (2.4 us a tile)
// is more than a join costs (10 us, and 3.5 TB/s for what the parts leave and it reads).  us without and with:
// 2 x 6437 tokens of a head of 128 155 and 75, 8192 of one 132 and 47, of four 133 and 106, 300 after 16084 of 32 heads 261 and 150; 8192 of four in sixteen
// documents 45 and 48, with a window of 512 21 and 30 (their few key tiles stay whole: what is left is the launch).
int fwd_parts(int B, int Sq, int Skv, int Hq, int HD) {
  const long long items = (long long)B * ((Sq + 255) / 256) * Hq, tiles = (Skv + BKV - 1) / BKV, n = 2ll * b200::sm_count() / items;
  const long long most = tiles / 4 < 8 ? tiles / 4 : 8, parts = n < most ? n : most;
  if (parts < 2) return 1;
  const float saved = 2.4f * tiles * (1.f - 1.f / parts), cost = 10.f + 5.7e-7f * (float)((long long)B * Sq * Hq) * parts * (HD * 4 + 16);
  return saved > cost ? (int)parts : 1;
}

template <int HD, int SCORE, bool LOW, bool SPLIT>
int launch_fwd(const CUtensorMap* m, const FwdParams& p, cudaStream_t stream) {
  using SM = Smem<HD>;
  static bool configured[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!configured[dev & 63]) {
    cudaError_t e = cudaFuncSetAttribute(attn_masked_fwd_kernel<HD, SCORE, LOW, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, SM::TOTAL);
    if (e != cudaSuccess) {
      cudaGetLastError();  // clear the sticky error before reporting
      return b200::fail(951, "attn_masked_fwd: cannot set %d bytes of shared memory: %s", SM::TOTAL, cudaGetErrorString(e));
    }
    configured[dev & 63] = true;
  }
  const int grid = p.items < b200::sm_count() ? p.items : b200::sm_count();
  b200::launch(attn_masked_fwd_kernel<HD, SCORE, LOW, SPLIT>, grid, NTHREADS, SM::TOTAL, stream, m[0], m[1], m[2], m[3], m[4], p);
  b200::count_launch();
  return b200::check_launch("attn_masked_fwd");
}
template <int HD, int SCORE>
int launch_fwd(const CUtensorMap* m, const FwdParams& p, cudaStream_t s) {
  if (p.parts == 1) return p.low != nullptr ? launch_fwd<HD, SCORE, true, false>(m, p, s) : launch_fwd<HD, SCORE, false, false>(m, p, s);
  if (int r = launch_fwd<HD, SCORE, true, true>(m, p, s)) return r;
  b200::launch(p.low != nullptr ? attn_masked_parts_kernel<HD, true> : attn_masked_parts_kernel<HD, false>, dim3((unsigned)(p.items / p.parts), 32), 256, 0, s, p);
  b200::count_launch();
  return b200::check_launch("attn_masked_parts");
}
template <int HD>
int launch_fwd(int score, const CUtensorMap* m, const FwdParams& p, cudaStream_t s) {
  switch (score) {
    case b200::SCORE_PLAIN: return launch_fwd<HD, b200::SCORE_PLAIN>(m, p, s);
    case b200::SCORE_CAP: return launch_fwd<HD, b200::SCORE_CAP>(m, p, s);
    case b200::SCORE_BIAS: return launch_fwd<HD, b200::SCORE_BIAS>(m, p, s);
    default: return launch_fwd<HD, b200::SCORE_CAP | b200::SCORE_BIAS>(m, p, s);
  }
}

}  // namespace

// bytes of the sums that parts of the key tiles leave (0: the key tiles are not parted)
B200_API long long b200_attn_masked_fwd_workspace(int B, int Sq, int Skv, int Hq, int HD) {
  const int parts = b200::sizes_ok(B, Sq, Skv, Hq, 1) ? fwd_parts(B, Sq, Skv, Hq, HD) : 1;
  return parts > 1 ? (long long)B * Sq * Hq * parts * (HD * 4 + 16) : 0;
}

// q: [B, Sq, Hq, HD], k/v: [B, Skv, Hkv, HD] bf16, each with its own row and batch pitch (elements), heads contiguous inside a token row;
// out [B, Sq, Hq, HD] contiguous, `low` like it or null; mask: b200_attn_mask's buffer for (B, Sq, Skv).
B200_API int b200_attn_masked_fwd(const void* q, const void* k, const void* v, void* out, void* low, float* lse, const float* sink,
                                  const float* slopes, const int* mask, int B, int Sq, int Skv, int Hq, int Hkv, int HD, long long q_row,
                                  long long k_row, long long v_row, long long q_batch, long long k_batch, long long v_batch, float scale,
                                  float cap, void* workspace, long long workspace_bytes, void* stream) {
  if (HD != 64 && HD != 128) return b200::fail(950, "attn_masked_fwd: head dim %d not supported (64 or 128)", HD);
  if (!b200::sizes_ok(B, Sq, Skv, Hq, Hkv))
    return b200::fail(950, "attn_masked_fwd: B=%d, Sq=%d, Skv=%d, Hq=%d, Hkv=%d", B, Sq, Skv, Hq, Hkv);
  if (!(scale > 0.f) || !b200::cap_ok(cap)) return b200::fail(950, "attn_masked_fwd: scale %g, cap %g", scale, cap);
  CUtensorMap m[5];
  int r;
  if ((r = b200::map_bshd(&m[0], q, HD, Hq, Sq, B, q_row, q_batch, BQ))) return r;
  if ((r = b200::map_bshd(&m[1], k, HD, Hkv, Skv, B, k_row, k_batch, BKV))) return r;
  if ((r = b200::map_bshd(&m[2], v, HD, Hkv, Skv, B, v_row, v_batch, BKV))) return r;
  const long long o_row = (long long)Hq * HD, o_batch = o_row * Sq;
  if ((r = b200::map_bshd(&m[3], out, HD, Hq, Sq, B, o_row, o_batch, 32))) return r;
  if ((r = b200::map_bshd(&m[4], low != nullptr ? low : out, HD, Hq, Sq, B, o_row, o_batch, 32))) return r;
  const b200::MaskLayout lay = b200::MaskLayout::of(B, Sq, Skv);
  FwdParams p;
  p.mask = b200::MaskView::of(mask, lay);
  p.score = b200::ScoreParams::of(scale, cap, slopes);
  p.Hq = Hq; p.Hkv = Hkv; p.Sq = Sq; p.Skv = Skv;
  p.scale_log2 = scale * b200::LOG2E;
  p.sink = sink; p.lse = lse;
  p.out = (__nv_bfloat16*)out; p.low = (__nv_bfloat16*)low;
  p.status = b200::status_ptr();
  p.parts = fwd_parts(B, Sq, Skv, Hq, HD);
  p.per = ((Skv + BKV - 1) / BKV + 2 * p.parts - 1) / (2 * p.parts);
  if (p.per < 4) p.per = 4;
  if (p.parts > 1 && (workspace == nullptr || (uintptr_t)workspace % 16 != 0 || workspace_bytes < b200_attn_masked_fwd_workspace(B, Sq, Skv, Hq, HD)))
    return b200::fail(952, "attn_masked_fwd: a workspace of %lld bytes", workspace_bytes);
  p.part_ml = (float4*)workspace;
  p.part = (float*)(p.part_ml + (long long)B * Sq * Hq * p.parts);
  const long long items = (long long)B * (lay.Sp / 256) * Hq * p.parts;
  if (items > 0x3fffffff) return b200::fail(950, "attn_masked_fwd: %lld query tile pairs", items);
  p.items = (int)items;
  const int score = (cap > 0.f ? b200::SCORE_CAP : 0) | (slopes != nullptr ? b200::SCORE_BIAS : 0);
  return HD == 128 ? launch_fwd<128>(score, m, p, (cudaStream_t)stream) : launch_fwd<64>(score, m, p, (cudaStream_t)stream);
}
