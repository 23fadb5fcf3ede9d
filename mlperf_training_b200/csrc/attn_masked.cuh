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

  // tanh(x) for |x| <= 1 is x times a polynomial in x^2, fitted to the smallest largest relative error there (7e-6: 3.5e-4 of a score capped at
  // 50); the coefficients take the scales in.  A capped score would otherwise take an exponential and a reciprocal more, and the
  // softmax warps are bound by the MUFU unit as it is.
  static ScoreParams of(float scale, float cap, const float* slopes) {
    ScoreParams p = {scale, cap, slopes, 0.f, 0.f, 0.f, {0.f, 0.f, 0.f, 0.f, 0.f}};
    if (cap > 0.f) {
      const double c[5] = {0.99999309, -0.33298064, 0.13036807, -0.04481748, 0.00903639}, into = (double)scale / cap, back = cap * 1.4426950408889634;
      p.into = (float)into;
      p.back = (float)back;
      double w = back * into;
      for (int i = 0; i < 5; ++i, w *= into * into) p.k[i] = (float)(c[i] * w);
      p.limit = into > 1e-4 && into < 1e3 ? (float)(1. / into) : 0.f;      // (powers of the scales that fp32 does not hold: never)
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
// tanh(x) = 1 - 2 / (1 + e^2x), absolute error below 3e-7
B200_DEVICE float capped_any(float s, const ScoreParams& p) {
  const float e = ex2_approx(s * p.into * (2.f * LOG2E));
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return p.back * fmaf(-2.f, r, 1.f);
}

}  // namespace b200
