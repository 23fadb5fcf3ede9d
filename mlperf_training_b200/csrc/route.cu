// Routing to experts with a choice of scores: softmax over all experts or sigmoid, a bias that only selects (load balance), experts in
// groups of which the best are kept, the k best experts, weights renormalised over them; its gradient; the step of the bias.
//
//   s_e = sigmoid(x_e) or softmax(x)_e        c_e = s_e + bias_e
//   value of a group = the sum of its two largest c (its only c if it has one); the `top` best groups stay
//   idx = the k largest c among them, largest first, ties to the lower index         w_j = scale * s_j / (sum_j s_j + 1e-20)
//
// What is compared is c in 64 bits: two experts whose c differ by less than fp32 resolves would otherwise change places with the way
// an exponential is rounded.  A warp takes a token in fp32 and keeps an eye on the gaps between neighbours (chosen experts, the best
// one left out, groups kept and left out); a gap below the error bound of the fp32 values sends the token through the
// same steps in fp64 (`choose_exact`; normal logits: 0.04 % of the tokens of 256 experts with sigmoid scores, 0.6 % with softmax).
// Without a bias and without groups the order of c is that of the logits, which are compared as they are.
#include "common.cuh"
#include "runtime.h"

namespace {

constexpr int MAX_E = 256, MAX_K = 32, MAX_G = 32;
constexpr int WARPS = 8;
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

// Order-preserving unsigned keys: 0 is nothing, NaN is below -inf.
B200_DEVICE unsigned key_of(float v) {
  const unsigned u = __float_as_uint(v);
  if (v != v) return 1u;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);        // -inf: 0x007fffff
}
B200_DEVICE float value_of(unsigned key) { return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key); }

// Above the error of the difference of two fp32 c, |c| <= 1 + b: 3e-7 a score (exponential by ex2.approx, reciprocal) and half a unit
// of the sum each.  The values of two groups hold two c each and a sum's rounding: four times that.
B200_DEVICE float gap_bound(float b) { return 1.5e-6f + 5e-7f * b; }

template <typename TL, int NPL>
B200_DEVICE void load_row(const TL* row, int e0, int E, bool vec, float (&x)[NPL]) {
  if (vec && e0 + NPL <= E) {
    const Pack<TL, NPL> p = *reinterpret_cast<const Pack<TL, NPL>*>(row + e0);
#pragma unroll
    for (int i = 0; i < NPL; ++i) x[i] = to_float(p.v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < NPL; ++i) x[i] = e0 + i < E ? to_float(row[e0 + i]) : -INFINITY;
  }
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

// Two largest of a warp's share of a group, merged over its `sub` lanes; value of the group.
template <typename R>
B200_DEVICE R group_value(const R* c, int n, int sub, int part, bool live) {
  R a = -INFINITY, b = -INFINITY;
  if (live)
    for (int i = part; i < n; i += sub) {
      const R v = c[i];
      if (v > a) { b = a; a = v; } else if (v > b) b = v;
    }
  for (int o = sub / 2; o > 0; o >>= 1) {
    const R a2 = __shfl_xor_sync(ALL, a, o), b2 = __shfl_xor_sync(ALL, b, o);
    const R lo = a < a2 ? a : a2, hi = a < a2 ? a2 : a, m = b < b2 ? b2 : b;
    a = hi;
    b = lo < m ? m : lo;
  }
  return n > 1 ? a + b : a;
}

// Bit g * sub of the result: group g stays.  gap: between the worst that stays and the best that does not.
template <typename R>
B200_DEVICE unsigned keep_groups(const R* c, int E, int G, int top, int lane, int& sub, R& gap) {
  int gp = 1;
  while (gp < G) gp *= 2;
  sub = 32 / gp;
  const int g = lane / sub, n = E / G;
  const R v = group_value(c + g * n, n, sub, lane % sub, g < G);
  int rank = 0;
  for (int h = 0; h < G; ++h) {
    const R o = __shfl_sync(ALL, v, h * sub);
    rank += (o > v || (o == v && h < g)) ? 1 : 0;
  }
  const bool keep = g < G && rank < top;
  // (the values at ranks top - 1 and top; lanes of one group agree)
  R in = __shfl_sync(ALL, v, __ffs(__ballot_sync(ALL, g < G && rank == top - 1)) - 1);
  R out = __shfl_sync(ALL, v, __ffs(__ballot_sync(ALL, g < G && rank == top)) - 1);
  gap = in - out;
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
  if (p.top < p.G) groups = keep_groups<double>(c, p.E, p.G, p.top, lane, sub, gap);
  const int n = p.E / p.G;
  unsigned taken = 0;                     // of this lane's experts lane + 32 i
  int mine = 0;
  for (int j = 0; j < p.k; ++j) {
    double best = -INFINITY;
    int at = MAX_E;                       // nothing yet: -inf at an index above all
    for (int i = 0, e = lane; e < p.E; ++i, e += 32)
      if (!(taken >> i & 1) && (p.top == p.G || (groups >> (e / n * sub) & 1)) && (c[e] > best || at == MAX_E)) { best = c[e]; at = e; }
    for (int o = 16; o > 0; o >>= 1) {
      const double b = __shfl_xor_sync(ALL, best, o);
      const int a = __shfl_xor_sync(ALL, at, o);
      if (a != MAX_E && (at == MAX_E || b > best || (b == best && a < at))) { best = b; at = a; }
    }
    if (at % 32 == lane) taken |= 1u << (at / 32);
    if (j == lane) mine = at;
  }
  return mine;
}

// A warp takes a token; lane l holds experts l * NPL .. + NPL - 1.
template <typename TL, int NPL>
__global__ void __launch_bounds__(WARPS * 32) route_kernel(const RouteParams p) {
  b200::begin_kernel();
  __shared__ double s_c[WARPS][MAX_E];
  __shared__ int s_hist[MAX_E];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, e0 = lane * NPL, n = p.E / p.G;
  for (int e = threadIdx.x; e < p.E; e += WARPS * 32) s_hist[e] = 0;
  __syncthreads();
  const bool by_logit = p.bias == nullptr && p.top == p.G;
  float bias[NPL];
  float largest = 0.f;                    // of the finite biases
#pragma unroll
  for (int i = 0; i < NPL; ++i) {
    bias[i] = p.bias != nullptr && e0 + i < p.E ? p.bias[e0 + i] : 0.f;
    if (fabsf(bias[i]) < INFINITY) largest = fmaxf(largest, fabsf(bias[i]));
  }
  const float near = gap_bound(1.f + warp_max(largest));
  float* sc = reinterpret_cast<float*>(s_c[warp]);
  for (long long t = (long long)blockIdx.x * WARPS + warp; t < p.T; t += (long long)gridDim.x * WARPS) {
    const TL* row = reinterpret_cast<const TL*>(p.logits) + t * p.ld;
    float x[NPL];
    load_row<TL, NPL>(row, e0, p.E, p.vec, x);
    float m = 0.f, inv = 1.f;
    if (!p.sigmoid) softmax_stats<NPL>(x, m, inv);
    unsigned key[NPL];
    unsigned groups = ALL;
    int sub = 1;
    bool exact = false;
    if (by_logit) {
#pragma unroll
      for (int i = 0; i < NPL; ++i) key[i] = e0 + i < p.E ? key_of(x[i]) : 0u;
    } else {
      float c[NPL];
#pragma unroll
      for (int i = 0; i < NPL; ++i) {
        c[i] = (p.sigmoid ? sigmoid(x[i]) : __expf(x[i] - m) * inv) + bias[i];
        if (c[i] != c[i]) c[i] = -INFINITY;
        key[i] = e0 + i < p.E ? key_of(c[i]) : 0u;
      }
      if (p.top < p.G) {
#pragma unroll
        for (int i = 0; i < NPL; ++i)
          if (e0 + i < p.E) sc[e0 + i] = c[i];
        __syncwarp();
        float gap;
        groups = keep_groups<float>(sc, p.E, p.G, p.top, lane, sub, gap);
        __syncwarp();
        exact = gap < 4.f * near;
#pragma unroll
        for (int i = 0; i < NPL; ++i)
          if (e0 + i < p.E && !(groups >> ((e0 + i) / n * sub) & 1)) key[i] = 0u;
      }
    }
    // k rounds of: the largest key of the warp; one more for the gap to the best one left out
    int mine = 0;
    float before = INFINITY;
    const int rounds = by_logit ? p.k : p.k + 1;
    for (int j = 0; j < rounds; ++j) {
      unsigned best = key[0];
#pragma unroll
      for (int i = 1; i < NPL; ++i) best = max(best, key[i]);
      const unsigned top = __reduce_max_sync(ALL, best);
      if (!by_logit) {
        const float v = value_of(top);
        exact |= top > 1u && before - v < near;
        before = v;
        if (j == p.k) break;
      }
      const int owner = __ffs(__ballot_sync(ALL, best == top)) - 1;
      int at = 0;
      if (lane == owner) {
        bool found = false;
#pragma unroll
        for (int i = 0; i < NPL; ++i)
          if (!found && key[i] == top) { found = true; at = e0 + i; key[i] = 0u; }
      }
      at = __shfl_sync(ALL, at, owner);
      if (lane == j) mine = at;
    }
    if (exact) {
      mine = choose_exact<TL>(row, p, s_c[warp], lane);
      __syncwarp();
    }
    // weights of the chosen
    float s = 0.f;
    if (lane < p.k) {
      const float xj = to_float(row[mine]);
      s = p.sigmoid ? sigmoid(xj) : __expf(xj - m) * inv;
    }
    const float total = p.renorm ? warp_sum(s) + EPS : 1.f;
    if (lane < p.k) {
      p.idx[t * p.k + lane] = mine;
      p.w[t * p.k + lane] = p.scale * (s / total);
      atomicAdd(&s_hist[mine], 1);
    }
  }
  __syncthreads();
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
      load_row<TL, NPL>(row, e0, p.E, p.vec, x);
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

unsigned route_grid(int T) {
  const long long blocks = ((long long)T + WARPS - 1) / WARPS, most = 6ll * b200::sm_count();
  return (unsigned)(blocks < most ? blocks : most);
}

template <typename TL>
void launch_route(const RouteParams& p, cudaStream_t s) {
  auto k = p.E <= 32 ? route_kernel<TL, 1> : p.E <= 64 ? route_kernel<TL, 2> : p.E <= 128 ? route_kernel<TL, 4> : route_kernel<TL, 8>;
  b200::launch(k, route_grid(p.T), WARPS * 32, 0, s, p);
}
template <typename TL>
void launch_route_bwd(const RouteBwdParams& p, cudaStream_t s) {
  auto k = p.E <= 32 ? route_bwd_kernel<TL, 1> : p.E <= 64 ? route_bwd_kernel<TL, 2> : p.E <= 128 ? route_bwd_kernel<TL, 4> : route_bwd_kernel<TL, 8>;
  b200::launch(k, route_grid(p.T), WARPS * 32, 0, s, p);
}

int check_route(const char* what, int T, int E, int k) {
  if (T < 0 || E < 1 || E > MAX_E || k < 1 || k > MAX_K || k > E)
    return b200::fail(920, "%s: T=%d, E=%d (1 to %d), k=%d (1 to %d, at most E)", what, T, E, MAX_E, k, MAX_K);
  return 0;
}

}  // namespace

// 1 if the counts of this call are stored whole (they need no clearing), else they are added to what is there
B200_API int b200_route_stores_counts(int T) { return T > 0 && T <= WARPS ? 1 : 0; }

B200_API int b200_route(const void* logits, int is_bf16, long long ld, const float* bias, int T, int E, int k, int sigmoid, int groups,
                        int top_groups, int renorm, float scale, int* idx, float* w, int* counts, void* stream) {
  if (int r = check_route("route", T, E, k)) return r;
  if (groups < 1 || groups > MAX_G || E % groups != 0 || top_groups < 1 || top_groups > groups || top_groups * (E / groups) < k)
    return b200::fail(921, "route: %d experts in %d groups (at most %d) of which %d stay, for k=%d", E, groups, MAX_G, top_groups, k);
  if (T == 0) return 0;
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
  if (is_bf16) launch_route_bwd<__nv_bfloat16>(p, (cudaStream_t)stream);
  else launch_route_bwd<float>(p, (cudaStream_t)stream);
  b200::count_launch();
  return b200::check_launch("route_bwd");
}

B200_API int b200_balance_bias(const float* bias, const int* counts, int E, float rate, float* out, void* stream) {
  if (E < 1) return b200::fail(922, "balance_bias: E=%d", E);
  b200::launch(balance_bias_kernel, 1, 256, 0, (cudaStream_t)stream, bias, counts, E, rate, out);
  b200::count_launch();
  return b200::check_launch("balance_bias");
}
