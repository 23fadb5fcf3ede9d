// Routing to experts with a choice of scores: softmax over all experts or sigmoid, a bias that only selects (load balance), experts in
// groups of which the best are kept, the k best experts, weights renormalised over them; its gradient; the step of the bias.
//
//   s_e = sigmoid(x_e) or softmax(x)_e        c_e = s_e + bias_e
//   value of a group = the sum of its two largest c (its only c if it has one); the `top` best groups stay
//   idx = the k largest c among them, largest first, ties to the lower index         w_j = scale * s_j / (sum_j s_j + 1e-20)
//
// What is compared is c in 64 bits: two experts whose c differ by less than fp32 resolves would otherwise change places with the way
// an exponential is rounded.  A warp takes a token.  A key of 32 bits holds c as 23 bits of fixed point between the smallest and largest
// c that the biases allow, and the expert's index below, so that one warp-wide maximum gives the next expert; every lane keeps its
// experts' keys sorted.  Where neighbours in the order (the best one left out and groups included) lie closer than the error
// of what was compared, the token goes through the same steps in fp64 (`choose_exact`; normal logits: 0.1 % of the tokens of 256 experts with
// sigmoid scores, 1 % with softmax; a finite bias that is large widens the fixed point's step, and with one expert of 65536 x 256 at -100 the pass
// takes 91 us instead of 71, at -1e4 286, when nearly every token does; at -inf, which is no part of the span, 71).  Without a bias the order is that of the logits: their upper 24 bits are the key, exact for bf16,
// and where neighbours (at the border of the choice: any that have its key) agree in them but not in the rest, the token goes to `choose_exact`.
// 65536 tokens, 256 experts in 8 groups, k 8, bf16: 67 us of kernel time (33 MB in); with a scan for the maximum over unsorted fp32 values, an owner's
// ballot and a shuffle a round 203.
#include "common.cuh"
#include "runtime.h"

namespace {

constexpr int MAX_E = 256, MAX_K = 32, MAX_G = 32;
constexpr int WARPS = 8, WAIT = 32;
constexpr float EPS = 1e-20f;
constexpr unsigned ALL = 0xffffffffu;

struct RouteParams {
  const void* logits;
  long long ld;
  const float* bias;        // [E] or null
  int T, E, k, sigmoid, G, top, renorm, vec;
  float scale;
  int* idx;                 // [T, k]
  float* w;                 // [T, k]
  int* counts;              // [E]
};

B200_DEVICE float to_float(float v) { return v; }
B200_DEVICE float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
B200_DEVICE void from_float(float& o, float v) { o = v; }
B200_DEVICE void from_float(__nv_bfloat16& o, float v) { o = __float2bfloat16(v); }

// N consecutive values; `vec`: the address is aligned to their size (16 bytes at most)
template <typename TL, int N>
struct alignas(N * sizeof(TL) < 16 ? N * sizeof(TL) : 16) Pack { TL v[N]; };

// Order-preserving unsigned key of a float (NaN: as -inf, -0: as 0).
B200_DEVICE unsigned key_of(float v) {
  const int u = __float_as_int(fmaxf(v, -INFINITY) + 0.f);
  return (unsigned)(u ^ ((u >> 31) | (int)0x80000000));          // -inf: 0x007fffff
}
B200_DEVICE float fma_sat(float a, float b, float c) {            // NaN: 0
  float d;
  asm("fma.rn.sat.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// 1 / (1 + e^-x) to 3e-7
B200_DEVICE float sigmoid_fast(float x) {
  const float d = 1.f + ex2_approx(x * -1.4426950408889634f);
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
  return r;
}

// Above the error of the difference of two fp32 c, |c| <= 1 + b: 3e-7 a score (exponential by ex2.approx, reciprocal) and half a unit
// of the sum each.  The values of two groups hold two c each and a sum's rounding: four times that.
B200_DEVICE float gap_bound(float b) { return 1.5e-6f + 5e-7f * b; }

// Descending order of a lane's keys.
template <int N>
B200_DEVICE void sort_down(unsigned (&k)[N]) {
  auto ce = [&](int a, int b) {
    const unsigned hi = max(k[a], k[b]), lo = min(k[a], k[b]);
    k[a] = hi;
    k[b] = lo;
  };
  if (N == 2) ce(0, 1);
  if (N >= 4) {
#pragma unroll
    for (int h = 0; h < N; h += 4) { ce(h, h + 1); ce(h + 2, h + 3); ce(h, h + 2); ce(h + 1, h + 3); ce(h + 1, h + 2); }
  }
  if (N == 8) {                            // merge of the two sorted fours
    ce(0, 4); ce(1, 5); ce(2, 6); ce(3, 7);
    ce(2, 4); ce(3, 5);
    ce(1, 2); ce(3, 4); ce(5, 6);
  }
}

// A lane's experts of a row, as they are in memory (those that are not there: 0) and as numbers (-inf).
template <typename TL, int NPL>
B200_DEVICE Pack<TL, NPL> fetch_row(const TL* row, int e0, int E, bool vec) {
  Pack<TL, NPL> r;
  if (vec && e0 + NPL <= E) return *reinterpret_cast<const Pack<TL, NPL>*>(row + e0);
#pragma unroll
  for (int i = 0; i < NPL; ++i) r.v[i] = e0 + i < E ? row[e0 + i] : (TL)0.f;
  return r;
}
template <typename TL, int NPL, bool FULL = false>
B200_DEVICE void row_values(const Pack<TL, NPL>& r, int e0, int E, float (&x)[NPL]) {
#pragma unroll
  for (int i = 0; i < NPL; ++i) x[i] = FULL || e0 + i < E ? to_float(r.v[i]) : -INFINITY;
}

// max and sum of a softmax over the row (sum 0: no finite logit)
template <int NPL>
B200_DEVICE void softmax_stats(const float (&x)[NPL], float& m, float& inv) {
  m = x[0];
#pragma unroll
  for (int i = 1; i < NPL; ++i) m = fmaxf(m, x[i]);
  m = warp_max(m);
  const float base = m == -INFINITY ? 0.f : m;
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < NPL; ++i) s += __expf(x[i] - base);
  s = warp_sum(s);
  m = base;
  inv = s > 0.f ? 1.f / s : (s != s ? s : 0.f);
}

// Two largest values so far.
template <typename R>
struct Two {
  R a = -INFINITY, b = -INFINITY;
  B200_DEVICE void add(R v) {
    const R lo = a < v ? a : v;
    a = a < v ? v : a;
    b = b < lo ? lo : b;
  }
  B200_DEVICE void join(int o) {           // with another lane's, of other experts
    const R a2 = __shfl_xor_sync(ALL, a, o), b2 = __shfl_xor_sync(ALL, b, o);
    add(a2);
    b = b < b2 ? b2 : b;
  }
  B200_DEVICE R value(int n) const {       // (an expert at +inf and one at -inf: as -inf)
    const R v = n > 1 ? a + b : a;
    return v == v ? v : -INFINITY;
  }
};
// Whether a group's two best in fixed point are what their sum does not hold: one at -inf, or the first at +inf (see route_kernel's u).
constexpr float OFF = 1.f + 0x1p-21f, ON = 2.f - 0x1p-20f;
B200_DEVICE bool infinite(const Two<float>& t, int n) { return n > 1 && (t.b <= OFF || t.a >= ON); }
B200_DEVICE bool infinite(const Two<double>&, int) { return false; }       // (64 bits hold them)

// Whether this lane's group stays.  Groups are `sub` lanes each, in order; `v` is the group's value in all of them.  gap: between the worst that
// stays and the best that does not.
template <typename R>
B200_DEVICE bool keep_group(R v, int G, int top, int sub, int lane, R& gap) {
  const int g = lane / sub;
  int rank = 0;
  for (int h = 0; h < G; ++h) {
    const R o = __shfl_sync(ALL, v, h * sub);
    rank += (o > v || (o == v && h < g)) ? 1 : 0;
  }
  const R in = __shfl_sync(ALL, v, __ffs(__ballot_sync(ALL, g < G && rank == top - 1)) - 1);
  const R out = __shfl_sync(ALL, v, __ffs(__ballot_sync(ALL, g < G && rank == top)) - 1);
  gap = in - out;
  return g < G && rank < top;
}
// The same for positive fp32 values below 4 in `g` < G, by warp-wide maxima of keys that hold the group below 27 bits of its value (what they cut, 31
// units of 2^-22, is in the gap).
B200_DEVICE bool keep_group(float v, int G, int top, int g, float& gap) {
  unsigned key = g < G ? (__float_as_uint(v) & ~31u) | (31u - (unsigned)g) : 0u;
  unsigned last = 0u;
  bool keep = false;
  for (int j = 0; j < top; ++j) {
    last = __reduce_max_sync(ALL, key);
    if (key == last) { keep = true; key = 0u; }
  }
  const unsigned next = __reduce_max_sync(ALL, key);
  gap = __uint_as_float(last & ~31u) - __uint_as_float(next & ~31u) - 0x1p-17f;
  return keep;
}
// The same from c in shared memory, for groups that are not whole lanes: bit g * sub of the result, group g stays.
template <typename R>
B200_DEVICE unsigned keep_groups(const R* c, int E, int G, int top, int lane, int& sub, R& gap, bool& odd) {
  int gp = 1;
  while (gp < G) gp *= 2;
  sub = 32 / gp;
  const int g = lane / sub, n = E / G;
  Two<R> t;
  if (g < G)
    for (int i = lane % sub; i < n; i += sub) t.add(c[g * n + i]);
  for (int o = sub / 2; o > 0; o >>= 1) t.join(o);
  odd = __any_sync(ALL, g < G && infinite(t, n));
  const bool keep = keep_group<R>(t.value(n), G, top, sub, lane, gap);
  return __ballot_sync(ALL, keep && lane % sub == 0);
}

// The choice of one token in 64 bits; lane j returns expert j.
template <typename TL>
__device__ __noinline__ int choose_exact(const TL* row, const RouteParams& p, double* c, int lane) {
  double m = -INFINITY, sum = 0.;
  if (!p.sigmoid) {
    for (int e = lane; e < p.E; e += 32) m = fmax(m, (double)to_float(row[e]));
    for (int o = 16; o > 0; o >>= 1) m = fmax(m, __shfl_xor_sync(ALL, m, o));
    for (int e = lane; e < p.E; e += 32) sum += exp((double)to_float(row[e]) - m);
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(ALL, sum, o);
  }
  for (int e = lane; e < p.E; e += 32) {
    const double x = to_float(row[e]);
    const double s = p.sigmoid ? 1. / (1. + exp(-x)) : (m == -INFINITY ? 0. : exp(x - m) / sum);
    const double v = p.bias != nullptr ? s + (double)p.bias[e] : s;
    c[e] = v == v ? v : -INFINITY;
  }
  __syncwarp();
  unsigned groups = ALL;
  int sub = 1;
  double gap;
  bool odd;
  if (p.top < p.G) groups = keep_groups<double>(c, p.E, p.G, p.top, lane, sub, gap, odd);
  if (p.bias == nullptr) {                 // the order of the experts is that of the logits
    __syncwarp();
    for (int e = lane; e < p.E; e += 32) {
      const float x = to_float(row[e]);
      c[e] = x == x ? (double)x : -INFINITY;
    }
    __syncwarp();
  }
  // Order-preserving keys of 64 bits, of experts lane + 32 i; 0: not there, not in a group that stays, or taken.  A round is the maximum of
  // their upper halves, of the lower halves among those, and the least index.
  const int n = p.E / p.G;
  unsigned long long key[MAX_E / 32];
#pragma unroll
  for (int i = 0; i < MAX_E / 32; ++i) {
    const int e = lane + 32 * i;
    const bool in = e < p.E && (p.top == p.G || (groups >> (e / n * sub) & 1));
    const long long u = in ? __double_as_longlong(c[e] + 0.) : 0;          // (-0 is 0)
    key[i] = in ? (unsigned long long)(u ^ ((u >> 63) | (long long)0x8000000000000000ull)) : 0ull;
  }
  int mine = 0;
  for (int j = 0; j < p.k; ++j) {
    unsigned long long best = key[0];
    int at = lane;
#pragma unroll
    for (int i = 1; i < MAX_E / 32; ++i)
      if (key[i] > best) { best = key[i]; at = lane + 32 * i; }
    const unsigned hi = (unsigned)(best >> 32), lo = (unsigned)best;
    const bool first = hi == __reduce_max_sync(ALL, hi);
    const unsigned least = __reduce_max_sync(ALL, first ? lo : 0u);
    at = (int)__reduce_min_sync(ALL, first && lo == least && best != 0ull ? (unsigned)at : (unsigned)MAX_E - 1);
#pragma unroll
    for (int i = 0; i < MAX_E / 32; ++i)
      if (at == lane + 32 * i) key[i] = 0ull;
    if (j == lane) mine = at;
  }
  return mine;
}

// Weights of the experts that lanes below k hold, and what the token adds to the counts.
template <typename TL>
B200_DEVICE void weigh(const TL* row, int t, int at, float m, float inv, const RouteParams& p, int* hist, int lane) {
  float s = 0.f;
  if (lane < p.k) {
    const float x = to_float(row[at]);
    s = p.sigmoid ? sigmoid(x) : __expf(x - m) * inv;
  }
  const float total = p.renorm ? warp_sum(s) + EPS : 1.f;
  if (lane < p.k) {
    p.idx[(long long)t * p.k + lane] = at;
    p.w[(long long)t * p.k + lane] = p.scale * (s / total);
    atomicAdd(&hist[at], 1);
  }
}

// A warp takes a token; lane l holds experts l * NPL .. + NPL - 1.
// FULL: E is 32 * NPL.
template <typename TL, int NPL, bool FULL>
__global__ void __launch_bounds__(WARPS * 32, 4) route_kernel(const __grid_constant__ RouteParams p) {
  b200::begin_kernel();
  __shared__ double s_c[WARPS][MAX_E];
  __shared__ int s_hist[MAX_E];
  __shared__ int s_wait[WARPS * WAIT], s_waiting;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, e0 = lane * NPL, n = p.E / p.G;
  for (int e = threadIdx.x; e < p.E; e += WARPS * 32) s_hist[e] = 0;
  if (threadIdx.x == 0) s_waiting = 0;
  const bool biased = p.bias != nullptr, grouped = p.top < p.G;
  // Groups of whole lanes, a power of two of them, are reduced in registers.
  const int lanes = n / NPL;
  const bool by_lanes = n % NPL == 0 && (lanes & (lanes - 1)) == 0;
  // u = a c + b lies in [2^-20, 1 - 2^-20], and is 0 or 1 for an infinite c; t = 1 + 2^-22 + u (1 - 2^-20) in [1, 2): the fixed point is its mantissa
  float bias[NPL];
  float least = INFINITY, most = -INFINITY, largest = 0.f;       // of the finite biases
#pragma unroll
  for (int i = 0; i < NPL; ++i) {
    bias[i] = biased && e0 + i < p.E ? p.bias[e0 + i] : 0.f;
    if (fabsf(bias[i]) < INFINITY && e0 + i < p.E) {
      least = fminf(least, bias[i]);
      most = fmaxf(most, bias[i]);
      largest = fmaxf(largest, fabsf(bias[i]));
    }
  }
  least = -warp_max(-least);
  most = warp_max(most);
  if (!(least <= most)) least = most = 0.f;
  const float a = (1.f - 0x1p-19f) / (1.f + most - least), base = 0x1p-20f - a * least;
  const float near = a * gap_bound(1.f + warp_max(largest)) + 0x1p-21f;      // in units of t
  // (in shared memory: registers are what limits the warps of an SM)
  __shared__ __align__(16) float s_bias[32 * NPL];
  if (warp == 0)
#pragma unroll
    for (int i = 0; i < NPL; ++i) s_bias[e0 + i] = fmaf(bias[i], a, base);
  __syncthreads();
  float* sc = reinterpret_cast<float*>(s_c[warp]);
  unsigned* sk = reinterpret_cast<unsigned*>(s_c[warp]) + lane * NPL;        // (not while sc is in use)
  const unsigned T = (unsigned)p.T, step = gridDim.x * WARPS;     // (no sum below reaches 2^32)
  unsigned t = blockIdx.x * WARPS + warp;
  Pack<TL, NPL> ahead;                                           // the next token's logits are on their way meanwhile
  if (t < T) ahead = fetch_row<TL, NPL>(reinterpret_cast<const TL*>(p.logits) + t * p.ld, e0, p.E, p.vec);
  // Tokens for choose_exact wait until WAIT tokens of each warp are through and are then shared by the block's warps: a call inside the loop costs
  // its registers, and a warp that does its own two or three is waited for by the launch (90 us at 65536 tokens instead of 75).
  for (unsigned t0 = blockIdx.x * WARPS; t0 < T; t0 += WAIT * step) {
  for (const unsigned end = min(T, t0 + WAIT * step); t < end; t += step) {
    const TL* row = reinterpret_cast<const TL*>(p.logits) + t * p.ld;
    float x[NPL];
    row_values<TL, NPL, FULL>(ahead, e0, p.E, x);
    if (T - t > step) ahead = fetch_row<TL, NPL>(row + (long long)step * p.ld, e0, p.E, p.vec);
    float m = 0.f, inv = 1.f;
    if (!p.sigmoid) softmax_stats<NPL>(x, m, inv);
    unsigned key[NPL];
    bool exact = false;
    float c[NPL];                                                // t of each expert
    if (biased || grouped) {
#pragma unroll
      for (int i = 0; i < NPL; ++i) {
        const float s = p.sigmoid ? sigmoid_fast(x[i]) : __expf(x[i] - m) * inv;
        c[i] = fmaf(fma_sat(s, a, s_bias[e0 + i]), 1.f - 0x1p-20f, 1.f + 0x1p-22f);      // (NaN and -inf: the smallest)
      }
    }
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
      const unsigned inverse = 255u - (unsigned)(e0 + i);
      // (the exponent of t leaves the word at the top: 0x3f8 << 28 is 2^31, taken off again)
      key[i] = biased ? (__float_as_uint(c[i]) << 8) - 0x80000000u + inverse : (key_of(x[i]) & 0xffffff00u) | inverse;
      if (!FULL && e0 + i >= p.E) key[i] = 0u;
    }
    if (grouped) {
      float gap;
      bool odd;
      if (by_lanes) {
        Two<float> two;
#pragma unroll
        for (int i = 0; i < NPL; ++i) two.add(c[i]);
        for (int o = lanes / 2; o > 0; o >>= 1) two.join(o);
        odd = __any_sync(ALL, lane / lanes < p.G && infinite(two, n));
        const bool keep = keep_group(two.value(n), p.G, p.top, lane / lanes, gap);
#pragma unroll
        for (int i = 0; i < NPL; ++i) key[i] = keep ? key[i] : 0u;
      } else {
#pragma unroll
        for (int i = 0; i < NPL; ++i)
          if (e0 + i < p.E) sc[e0 + i] = c[i];
        __syncwarp();
        int sub;
        const unsigned groups = keep_groups<float>(sc, p.E, p.G, p.top, lane, sub, gap, odd);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < NPL; ++i)
          if (e0 + i < p.E && !(groups >> ((e0 + i) / n * sub) & 1)) key[i] = 0u;
      }
      exact = odd || gap < 4.f * near;
    }
    sort_down<NPL>(key);
    // the k largest keys of the warp, and the next one for the gap to it; lane j keeps the j-th.  A lane's keys behind its first wait in
    // shared memory (moving them up in registers took as many instructions as all else in a round).
    unsigned head = key[0];
    if (NPL > 1) {
#pragma unroll
      for (int i = 1; i < NPL; ++i) sk[i - 1] = key[i];
      sk[NPL - 1] = 0u;
    }
    const unsigned* next_key = sk;
    unsigned mine = 0u, top = 0u;
    for (int j = 0; j <= p.k; ++j) {
      top = __reduce_max_sync(ALL, head);
      if (lane == j) mine = top;
      if (head == top) head = NPL > 1 ? *next_key++ : 0u;          // (a lane whose keys are out stays at the 0 behind them)
    }
    int at = 255 - (int)(mine & 255u);
    {
      unsigned next = __shfl_down_sync(ALL, mine, 1);
      if (lane == p.k - 1) next = top;                           // the best one left out
      const bool pair = lane < p.k && (next >> 8) != 0u;
      const unsigned units = (mine >> 8) - (next >> 8);
      bool close = pair && (biased ? (float)units < near * 0x1p23f : units == 0u);
      if (__any_sync(ALL, close) && !biased) {
        // equal in 24 bits: equal logits are in order as they are
        const float mv = to_float(row[min(at, p.E - 1)]), nv = to_float(row[min(255 - (int)(next & 255u), p.E - 1)]);
        close = close && !(mv == nv || (mv != mv && nv != nv));
        if (sizeof(TL) == 4 && (__shfl_sync(ALL, mine, p.k - 1) ^ top) < 256u) {
          // the last of the choice and the best one left out agree in 24 bits: so may others that are left out, and be larger
          const float v = to_float(row[255 - (int)(top & 255u)]);
          for (int i = 0; i < NPL && e0 + i < p.E; ++i) {
            const float u = to_float(row[e0 + i]);
            close |= ((key_of(u) ^ top) & 0xffffff00u) == 0u && !(u == v || (u != u && v != v));
          }
        }
      }
      exact |= __any_sync(ALL, close);
    }
    if (exact) {
      if (lane == 0) s_wait[atomicAdd(&s_waiting, 1)] = t;
    } else {
      weigh<TL>(row, t, at, m, inv, p, s_hist, lane);
    }
  }
  __syncthreads();
  const int waiting = s_waiting;
  for (int i = warp; i < waiting; i += WARPS) {
    __syncwarp();
    const int tt = s_wait[i];
    const TL* row = reinterpret_cast<const TL*>(p.logits) + tt * p.ld;
    const int at = choose_exact<TL>(row, p, s_c[warp], lane);
    float m = 0.f, inv = 1.f;
    if (!p.sigmoid) {
      float x[NPL];
      row_values<TL, NPL>(fetch_row<TL, NPL>(row, e0, p.E, p.vec), e0, p.E, x);
      softmax_stats<NPL>(x, m, inv);
    }
    weigh<TL>(row, tt, at, m, inv, p, s_hist, lane);
  }
  __syncthreads();
  if (threadIdx.x == 0) s_waiting = 0;
  if (T - t0 > WAIT * step) __syncthreads();         // (the last time nothing is added any more)
  }
  for (int e = threadIdx.x; e < p.E; e += WARPS * 32) {
    if (gridDim.x == 1) p.counts[e] = s_hist[e];
    else if (s_hist[e] != 0) atomicAdd(&p.counts[e], s_hist[e]);         // (whole numbers: the order does not matter)
  }
}

struct RouteBwdParams {
  const void* logits;
  long long ld;
  const int* idx;
  const float* gw;
  int T, E, k, sigmoid, renorm, vec;
  float scale;
  void* dx;                 // [T, E], contiguous, of the logits' type
  int vec_out;
};

// dL/ds_j = (g_j - sum_i g_i s_i / S) / S with S = sum s + 1e-20 (renormalised; else g_j), g = scale * dL/dw, and through the score:
//   sigmoid  dx_j = dL/ds_j s_j (1 - s_j)
//   softmax  dx_e = s_e (dL/ds_e - r),  r = sum_j dL/ds_j s_j  (renormalised: sum_i g_i s_i / S * 1e-20 / S, the same without its cancellation)
template <typename TL, int NPL>
__global__ void __launch_bounds__(WARPS * 32) route_bwd_kernel(const RouteBwdParams p) {
  b200::begin_kernel();
  __shared__ __align__(16) float s_row[WARPS][32 * NPL];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, e0 = lane * NPL;
  float* sr = s_row[warp];
  for (long long t = (long long)blockIdx.x * WARPS + warp; t < p.T; t += (long long)gridDim.x * WARPS) {
    const TL* row = reinterpret_cast<const TL*>(p.logits) + t * p.ld;
    float x[NPL], m = 0.f, inv = 1.f;
    if (!p.sigmoid) {
      row_values<TL, NPL>(fetch_row<TL, NPL>(row, e0, p.E, p.vec), e0, p.E, x);
      softmax_stats<NPL>(x, m, inv);
    }
    const bool live = lane < p.k;
    const int e = live ? p.idx[t * p.k + lane] : 0;
    const float xj = live ? to_float(row[e]) : 0.f, g = live ? p.scale * p.gw[t * p.k + lane] : 0.f;
    const float s = live ? (p.sigmoid ? sigmoid(xj) : __expf(xj - m) * inv) : 0.f;
    float d = g, r;
    const float gs = warp_sum(g * s);
    if (p.renorm) {
      const float total = warp_sum(s) + EPS;
      d = (g - gs / total) / total;
      r = gs / total * (EPS / total);
    } else {
      r = gs;
    }
#pragma unroll
    for (int i = 0; i < NPL; ++i) sr[e0 + i] = p.sigmoid ? 0.f : -r * (__expf(x[i] - m) * inv);
    __syncwarp();
    if (live) sr[e] = p.sigmoid ? d * s * sigmoid(-xj) : s * (d - r);
    __syncwarp();
    TL* out = reinterpret_cast<TL*>(p.dx) + t * p.E;
    if (p.vec_out && e0 + NPL <= p.E) {
      Pack<TL, NPL> o;
#pragma unroll
      for (int i = 0; i < NPL; ++i) from_float(o.v[i], sr[e0 + i]);
      *reinterpret_cast<Pack<TL, NPL>*>(out + e0) = o;
    } else {
#pragma unroll
      for (int i = 0; i < NPL; ++i)
        if (e0 + i < p.E) from_float(out[e0 + i], sr[e0 + i]);
    }
    __syncwarp();
  }
}

// bias + rate * sign(mean load - load)
__global__ void balance_bias_kernel(const float* __restrict__ bias, const int* __restrict__ counts, int E, float rate, float* __restrict__ out) {
  b200::begin_kernel();
  __shared__ long long part[32];
  long long sum = 0;
  for (int e = threadIdx.x; e < E; e += blockDim.x) sum += counts[e];
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(ALL, sum, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sum;
  __syncthreads();
  sum = 0;
  for (int i = 0; i < (int)(blockDim.x >> 5); ++i) sum += part[i];
  for (int e = threadIdx.x; e < E; e += blockDim.x) {
    const long long d = sum - (long long)E * counts[e];
    out[e] = d == 0 ? bias[e] : bias[e] + (d > 0 ? rate : -rate);
  }
}

template <typename TL>
int row_pack(int E) {                    // bytes of a lane's experts, as they are loaded
  const int npl = E <= 32 ? 1 : E <= 64 ? 2 : E <= 128 ? 4 : 8;
  return npl * (int)sizeof(TL) < 16 ? npl * (int)sizeof(TL) : 16;
}
template <typename TL>
bool packable(const void* p, long long ld, int E) {
  const int b = row_pack<TL>(E);
  return ((uintptr_t)p % b) == 0 && (ld * (long long)sizeof(TL)) % b == 0;
}

// As many blocks as run at once (a second wave, of half as many, took 15 us of 76 at 65536 tokens).
template <auto KERNEL, typename P>
void launch_rows(const P& p, cudaStream_t s) {
  static const int at_once = [] {
    int n = 0;
    return cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, KERNEL, WARPS * 32, 0) == cudaSuccess && n > 0 ? n : 1;
  }();
  const long long blocks = ((long long)p.T + WARPS - 1) / WARPS, most = (long long)at_once * b200::sm_count();
  b200::launch(KERNEL, (unsigned)(blocks < most ? blocks : most), WARPS * 32, 0, s, p);
}

template <typename TL, int NPL>
void launch_of(const RouteParams& p, cudaStream_t s) {
  if (p.E == 32 * NPL) launch_rows<route_kernel<TL, NPL, true>>(p, s);
  else launch_rows<route_kernel<TL, NPL, false>>(p, s);
}
template <typename TL, int NPL>
void launch_of(const RouteBwdParams& p, cudaStream_t s) { launch_rows<route_bwd_kernel<TL, NPL>>(p, s); }
template <typename TL, typename P>
void launch_route(const P& p, cudaStream_t s) {
  if (p.E <= 32) launch_of<TL, 1>(p, s);
  else if (p.E <= 64) launch_of<TL, 2>(p, s);
  else if (p.E <= 128) launch_of<TL, 4>(p, s);
  else launch_of<TL, 8>(p, s);
}

int check_route(const char* what, int T, int E, int k) {
  if (T < 0 || E < 1 || E > MAX_E || k < 1 || k > MAX_K || k > E)
    return b200::fail(920, "%s: T=%d, E=%d (1 to %d), k=%d (1 to %d, at most E)", what, T, E, MAX_E, k, MAX_K);
  return 0;
}

}  // namespace

B200_API int b200_route(const void* logits, int is_bf16, long long ld, const float* bias, int T, int E, int k, int sigmoid, int groups,
                        int top_groups, int renorm, float scale, int* idx, float* w, int* counts, void* stream) {
  if (int r = check_route("route", T, E, k)) return r;
  if (groups < 1 || groups > MAX_G || E % groups != 0 || top_groups < 1 || top_groups > groups || top_groups * (E / groups) < k)
    return b200::fail(921, "route: %d experts in %d groups (at most %d) of which %d stay, for k=%d", E, groups, MAX_G, top_groups, k);
  if (T == 0) return 0;
  if (T > WARPS) {                 // (one block stores its counts, several add to them)
    const cudaError_t e = cudaMemsetAsync(counts, 0, sizeof(int) * E, (cudaStream_t)stream);
    if (e != cudaSuccess) return b200::fail(923, "route: clearing the counts: %s", cudaGetErrorString(e));
  }
  RouteParams p = {logits, ld, bias, T, E, k, sigmoid, groups, top_groups, renorm, 0, scale, idx, w, counts};
  p.vec = is_bf16 ? packable<__nv_bfloat16>(logits, ld, E) : packable<float>(logits, ld, E);
  if (is_bf16) launch_route<__nv_bfloat16>(p, (cudaStream_t)stream);
  else launch_route<float>(p, (cudaStream_t)stream);
  b200::count_launch();
  return b200::check_launch("route");
}

B200_API int b200_route_bwd(const void* logits, int is_bf16, long long ld, const int* idx, const float* gw, int T, int E, int k, int sigmoid,
                            int renorm, float scale, void* dx, void* stream) {
  if (int r = check_route("route_bwd", T, E, k)) return r;
  if (T == 0) return 0;
  RouteBwdParams p = {logits, ld, idx, gw, T, E, k, sigmoid, renorm, 0, scale, dx, 0};
  p.vec = is_bf16 ? packable<__nv_bfloat16>(logits, ld, E) : packable<float>(logits, ld, E);
  p.vec_out = is_bf16 ? packable<__nv_bfloat16>(dx, E, E) : packable<float>(dx, E, E);
  if (is_bf16) launch_route<__nv_bfloat16>(p, (cudaStream_t)stream);
  else launch_route<float>(p, (cudaStream_t)stream);
  b200::count_launch();
  return b200::check_launch("route_bwd");
}

B200_API int b200_balance_bias(const float* bias, const int* counts, int E, float rate, float* out, void* stream) {
  if (E < 1) return b200::fail(922, "balance_bias: E=%d", E);
  b200::launch(balance_bias_kernel, 1, 256, 0, (cudaStream_t)stream, bias, counts, E, rate, out);
  b200::count_launch();
  return b200::check_launch("balance_bias");
}
