// What the kernels of masked attention share: 4-D TMA copies of [B][S][H][D] tensors and the scores' transform.
#pragma once
#include "attn_mask.cuh"
#include "runtime.h"

namespace b200 {

B200_DEVICE void load_4d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
B200_DEVICE void store_4d(const CUtensorMap* map, const void* src, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(map),
               "r"(smem_u32(src)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
               : "memory");
}
B200_DEVICE void reduce_add_4d(const CUtensorMap* map, const void* src, int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.reduce.async.bulk.tensor.4d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(map),
      "r"(smem_u32(src)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}

// [B][S][H][HD] bf16 with its own pitches (elements), heads contiguous inside a row; boxes of 64 columns and `rows` rows
inline int map_bshd(CUtensorMap* m, const void* ptr, int HD, int H, int S, int B, long long row, long long batch, int rows) {
  return make_tmap_4d(m, DT_BF16, ptr, HD, H, S, B, (uint64_t)HD * 2, (uint64_t)row * 2, (uint64_t)batch * 2, 64, 1, rows, 1, SWZ_128);
}

constexpr float LOG2E = 1.4426950408889634f;

// Scores: what of cap and distance bias a kernel has.
enum : int { SCORE_PLAIN = 0, SCORE_CAP = 1, SCORE_BIAS = 2 };

struct ScoreParams {
  float scale;              // of the products
  float cap;                // c of c tanh(s / c), or 0
  const float* slopes;      // [Hq]: what a key at distance d loses is slope * d, or null
  float into, back;         // with a cap: what takes a product into the tangent, c log2(e)
  float limit, k[5];        // products up to `limit` in size: back * tanh(into * s) = s * (k0 + k1 s^2 + .. + k4 s^8)

  // tanh(x) for |x| <= 1 is x times a polynomial in x^2, fitted to the smallest largest relative error there (7e-6); the coefficients take the
  // scales in.  A capped score would otherwise take an exponential and a reciprocal more, and the softmax warps are bound by the MUFU
  // unit as it is.  It serves scores of up to 64 (an error of 4.5e-4 there, a tenth of what P loses to bf16); larger ones, which only larger
  // caps let through, and those of scales whose powers fp32 does not hold go through capped_any2.
  static ScoreParams of(float scale, float cap, const float* slopes) {
    ScoreParams p = {scale, cap, slopes, 0.f, 0.f, 0.f, {0.f, 0.f, 0.f, 0.f, 0.f}};
    if (cap > 0.f) {
      const double c[5] = {0.99999309, -0.33298064, 0.13036807, -0.04481748, 0.00903639}, into = (double)scale / cap, back = cap * 1.4426950408889634;
      p.into = (float)(into < 1e38 ? into : 1e38);
      p.back = (float)back;
      const double x = cap < 64.f ? 1. : 64. / cap, limit = x / into;      // the largest |into * s| and |s|
      double w = back * into, share = 1.;                                  // of term i: its scales, and what it is of the first one at most
      bool held = limit < 1e15;                                            // (its square)
      for (int i = 0; i < 5; ++i, w *= into * into, share *= x * x) {
        const double k = c[i] * w, size = k < 0. ? -k : k;
        held &= size < 1e38 && (size > 1e-37 || share < 1e-9);
        p.k[i] = size > 1e-37 ? (float)k : 0.f;
      }
      p.limit = held ? (float)limit : -1.f;
    }
    return p;
  }
};

// Capped scores, in units of log2, of a pair of products: of at most `limit` in size, and of any.
B200_DEVICE float2 capped_small2(float2 s, const ScoreParams& p) {
  const float2 q = fmul2(s, s);
  float2 r = ffma2(q, make_float2(p.k[4], p.k[4]), make_float2(p.k[3], p.k[3]));
  r = ffma2(r, q, make_float2(p.k[2], p.k[2]));
  r = ffma2(r, q, make_float2(p.k[1], p.k[1]));
  r = ffma2(r, q, make_float2(p.k[0], p.k[0]));
  return fmul2(r, s);
}
// tanh(x) = 1 - 2 / (1 + e^2x) from 1/2 on, and below, where that difference cancels, x times a polynomial in x^2 (fitted like the other, 1.3e-8):
// relative error below 5e-7, so that a cap far above the scores leaves them what they are
B200_DEVICE float2 capped_any2(float2 s, const ScoreParams& p) {
  auto both = [](float v) { return make_float2(v, v); };
  const float2 x = fmul2(s, both(p.into)), q = fmul2(x, x), y = fmul2(x, both(2.f * LOG2E)), d = fadd2(make_float2(ex2_approx(y.x), ex2_approx(y.y)), both(1.f));
  float2 r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(d.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(d.y));
  float2 t = ffma2(q, both(0.017135007f), both(-0.052986074f));
  t = ffma2(t, q, both(0.13324779f));
  t = ffma2(t, q, both(-0.33333069f));
  t = fmul2(ffma2(t, q, both(1.f)), x);
  r = ffma2(r, both(-2.f), both(1.f));
  return fmul2(make_float2(fabsf(x.x) < 0.5f ? t.x : r.x, fabsf(x.y) < 0.5f ? t.y : r.y), both(p.back));
}
// Sizes that a kernel can have; what is computed from others (sums to divide by) may be 0.
inline bool sizes_ok(int B, int Sq, int Skv, int Hq, int Hkv) {
  return B >= 1 && Sq >= 1 && Skv >= Sq && Hkv >= 1 && Hq >= 1 && Hq % Hkv == 0;
}
// Caps that the scales above hold in fp32, with their squares (0: none)
inline bool cap_ok(float cap) { return cap == 0.f || (cap >= 1e-12f && cap <= 1e18f); }

}  // namespace b200
