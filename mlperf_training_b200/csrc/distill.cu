// Distillation from a teacher's largest logits, mixed with cross-entropy, per token of student logits z [V]:
//
//   loss = a tau^2 KL + (1 - a) CE            u = z / tau, q = softmax(u), q1 = softmax(z)
//   KL   = sum_j p_j (log p_j - log q[id_j])  over the teacher's K entries (id_j, t_j)
//          plain: p = softmax(t / tau) over the entries that are there
//          rest:  p_j = exp(t_j); what they leave, r = 1 - sum p, is one further event "any other id": r (log r - log R),
//                 R = the student's mass outside the ids
//   dz   = gy (a tau (c q_v - p_v - [v not among the ids] (r / R) q_v) + (1 - a) (q1_v - [v = label])),  c = sum p + r
// q_v / R, a softmax over the ids that are left out, is formed on their own log-sum-exp: R may be far smaller than fp32 holds.
//
// An entry whose id is outside the vocabulary or whose value is -inf is not there.  Tokens labelled `ignore` have loss and gradient 0; so has
// the cross-entropy of another label outside the vocabulary.
//
// Forward: one pass over the row for the log-sum-exp of u and of z on one running maximum.  Where both are wanted and tau is 2, 4 or 8, the
// term of z is that of u squared once, twice or three times; another tau takes a second exponential (16 a clock and SM: 8192 rows of
// 128256 in bf16 with two 626 us, 336 with one).  With `rest` the ids are marked in a bitmap and left out of the sum, which is then that
// of the others without cancellation, and the ids' own terms join it at the end.  One warp forms the teacher's sums meanwhile, in fp64
// (r = 1 - sum p cancels); what they need of the student is its log-sum-exp alone.
// Backward: the row again from the saved log-sum-exps, written as it is read; the elements of the ids and the label are then written once
// more by a thread each, from logits read before any was overwritten, so the gradient may take the logits' place.
// Both are bound by memory (one read; one read and one write) with four 16-byte loads a thread under way: 8192 x 128256 bf16
// 336 and 640 us (6.25 and 6.56 TB/s).
#include "common.cuh"
#include "runtime.h"

namespace {

constexpr int MAX_K = 1024;
constexpr int MAX_T = 0x7fff0000;  // (a row's number and the next of its block's stay in 32 bits)
constexpr int AHEAD = 4;           // 16-byte loads of a thread under way
constexpr int MAX_SMEM = 225 * 1024;         // marks of 921600 ids, two rows of them
constexpr int SHORT_BYTES = 100 * 1024;      // of a row, up to which it is short
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

enum { F32 = 0, BF16 = 1 };

struct DistillParams {
  const void* logits;       // [T, ld]
  long long ld;
  const long long* labels;  // [T] or null
  const void* ids;          // [T, K], int32 or int64
  const void* values;       // [T, K], fp32 or bf16
  int ids64, values_bf16, T, K, V, rest;
  float alpha, tau;
  long long ignore;
  float* loss;              // [T]
  float* stats;             // [T, 4]: log-sum-exp of u and of z (log2 units), c, log-sum-exp of u outside the ids (rest)
  double* teacher;          // [T]: log-sum-exp of t / tau (plain), r (rest; 0 where no id is left out)
  // backward
  const float* gy;          // [T]
  void* grad;               // [T, ld_grad], may be the logits
  long long ld_grad;
};

template <typename TL> struct Vec { static constexpr int N = 16 / sizeof(TL); };

B200_DEVICE float load1(const float* p) { return *p; }
B200_DEVICE float load1(const __nv_bfloat16* p) { return __bfloat162float(*p); }
B200_DEVICE void store1(float* p, float v) { *p = v; }
B200_DEVICE void store1(__nv_bfloat16* p, float v) { *p = __float2bfloat16(v); }
B200_DEVICE void store_vec(float* p, const float (&x)[4]) { *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]); }
B200_DEVICE void store_vec(__nv_bfloat16* p, const float (&x)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
}

B200_DEVICE long long id_at(const DistillParams& p, long long i) {
  return p.ids64 ? reinterpret_cast<const long long*>(p.ids)[i] : (long long)reinterpret_cast<const int*>(p.ids)[i];
}
B200_DEVICE float value_at(const DistillParams& p, long long i) {
  return p.values_bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.values)[i]) : reinterpret_cast<const float*>(p.values)[i];
}

// The aligned part of columns [lo, hi) of a row: vectors [first, first + n * N), scalars before and after.
struct Span { int lo, hi, first, n; };
template <typename TL>
B200_DEVICE Span span_of(const TL* row, int lo, int hi) {
  constexpr int N = Vec<TL>::N;
  const int off = (int)(((uintptr_t)(row + lo) & 15) / sizeof(TL));
  Span s = {lo, hi, lo + (off ? N - off : 0), 0};
  if (s.first > hi) s.first = hi;
  s.n = (hi - s.first) / N;
  return s;
}

// Sums of 2^(x - m) and (Z) of its tau-th power, for the largest m so far.
template <bool Z>
struct Lse {
  float m = -INFINITY, s = 0.f, z = 0.f;
  B200_DEVICE void join(float m2, float s2, float z2, float tau) {
    const float n = fmax_nan(m, m2);
    const float f = m == -INFINITY ? 0.f : ex2_approx(m - n), g = m2 == -INFINITY ? 0.f : ex2_approx(m2 - n);
    s = s * f + s2 * g;
    if (Z) z = z * (m == -INFINITY ? 0.f : ex2_approx((m - n) * tau)) + z2 * (m2 == -INFINITY ? 0.f : ex2_approx((m2 - n) * tau));
    m = n;
  }
  B200_DEVICE void join_lane(int o, float tau) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o), z2 = Z ? __shfl_xor_sync(0xffffffffu, z, o) : 0.f;
    join(m2, s2, z2, tau);
  }
  B200_DEVICE float log2_s() const { return m == -INFINITY ? -INFINITY : m + log2f(s); }
  B200_DEVICE float log2_z(float tau) const { return m == -INFINITY ? -INFINITY : m * tau + log2f(z); }
};
B200_DEVICE double warp_sum64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
B200_DEVICE double warp_max64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// What one warp finds out about a token's teacher.
struct Teacher {
  double log_sum = 0.;      // of t / tau (plain)
  double mass = 0.;         // sum of p
  double own = 0.;          // sum of p log p
  double cross = 0.;        // sum of p u[id]
};

// The largest of N elements as floats (bf16: pairs at a time).
B200_DEVICE float largest(const float4& v) { return fmax_nan(fmax_nan(v.x, v.y), fmax_nan(v.z, v.w)); }
B200_DEVICE float largest(const uint4& v) {
  auto h = [](uint32_t x) { return *reinterpret_cast<const __nv_bfloat162*>(&x); };
  const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(h(v.x), h(v.y)), __hmax2_nan(h(v.z), h(v.w)));
  return fmax_nan(__low2float(m), __high2float(m));
}
B200_DEVICE void pairs(const float4& v, float2 (&x)[2]) { x[0] = make_float2(v.x, v.y); x[1] = make_float2(v.z, v.w); }
B200_DEVICE float2 pair(uint32_t u) { return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)); }
B200_DEVICE void pairs(const uint4& v, float2 (&x)[4]) { x[0] = pair(v.x); x[1] = pair(v.y); x[2] = pair(v.z); x[3] = pair(v.w); }
template <typename TL> struct Raw;
template <> struct Raw<float> { using T = float4; };
template <> struct Raw<__nv_bfloat16> { using T = uint4; };

// A CTA takes every gridDim.x-th row.  POWER: -1 the log-sum-exp of u alone; 1, 2, 3 that of z too, from u's terms squared so many times; 0
// from an exponential of its own.  REST: ids are left out of the pass.
// The last warp takes the teacher, whose chain of loads and sums is about as long as a third of a row (a warp that did both held the row
// back: 8192 x 128256 bf16 484 us, 410 with a warp for each), and the end of each row, while the others are at the next one already: their
// first loads of it are under way before they join their sums (336 us).  One barrier a row: sums and marks have two copies.
// NT threads for a row's elements: 512, or 64 in more CTAs where rows are short (see launch_fwd).
template <typename TL, int POWER, bool REST, int NT>
__global__ void __launch_bounds__(NT + 32, NT == 512 ? 2 : 10) distill_fwd_kernel(const DistillParams p) {
  b200::begin_kernel();
  constexpr bool BOTH = POWER >= 0;
  constexpr int N = Vec<TL>::N;
  using RawT = typename Raw<TL>::T;
  extern __shared__ unsigned s_mark[];                 // REST: a bit for each id, of two rows
  __shared__ Lse<BOTH> red[2][NT / 32];
  const int lane = threadIdx.x & 31, words = (p.V + 31) / 32, step = gridDim.x;
  const float cu = LOG2E / p.tau;
  const bool teaches = threadIdx.x >= NT;
  auto row_of = [&](long long t) { return reinterpret_cast<const TL*>(p.logits) + t * p.ld; };
  auto label_of = [&](long long t) { return p.labels != nullptr ? p.labels[t] : 0ll; };
  auto ignored = [&](long long label) { return p.labels != nullptr && label == p.ignore; };
  // entry j of token t: its id, or -1 where it is not there
  auto entry = [&](long long t, int j, float& val) -> int {
    const long long v = id_at(p, t * p.K + j);
    val = value_at(p, t * p.K + j);
    return v >= 0 && v < p.V && val != -INFINITY ? (int)v : -1;
  };
  // (REST, the teacher) marks the ids of token t; bit i of the result: entry lane + 32 i is the first of its id
  auto mark = [&](long long t, unsigned* marks) -> unsigned {
    unsigned first = 0u;
    float val;
    if (t < p.T && p.alpha > 0.f && !ignored(label_of(t)))
      for (int j = lane; j < p.K; j += 32) {
        const int v = entry(t, j, val);
        if (v >= 0 && !(atomicOr(&marks[v >> 5], 1u << (v & 31)) >> (v & 31) & 1u)) first |= 1u << (j >> 5);
      }
    return first;
  };
  unsigned first = 0u;
  if (REST) {
    for (int i = threadIdx.x; i < 2 * words; i += NT + 32) s_mark[i] = 0u;
    __syncthreads();
    if (teaches) first = mark(blockIdx.x, s_mark);
    __syncthreads();
  }

  if (teaches) {
    for (int t = blockIdx.x, n = 0; t < p.T; t += step, ++n) {
      const long long label = label_of(t);
      const bool live = !ignored(label);
      const TL* row = row_of(t);
      unsigned* marks = s_mark + (n & 1) * words;
      Teacher te;
      Lse<BOTH> ids;                                   // (REST) terms of the ids, each once
      float zlabel = 0.f;
      if (live && p.alpha < 1.f && label >= 0 && label < p.V) zlabel = load1(row + label);
      if (live && p.alpha > 0.f) {
        if (!p.rest) {
          double m = -INFINITY, s = 0.;
          float val;
          for (int j = lane; j < p.K; j += 32)
            if (entry(t, j, val) >= 0) m = fmax(m, (double)val / p.tau);
          m = warp_max64(m);
          for (int j = lane; j < p.K; j += 32)
            if (entry(t, j, val) >= 0) s += exp((double)val / p.tau - m);
          s = warp_sum64(s);
          te.log_sum = s != 0. ? m + log(s) : 0.;      // (no entry: s = 0)
        }
        for (int j = lane; j < p.K; j += 32) {
          float val;
          const int id = entry(t, j, val);
          if (id < 0) continue;
          const float zid = load1(row + id);
          if (REST && (first >> (j >> 5) & 1u)) ids.join(zid * cu, 1.f, 1.f, p.tau);
          const double logp = p.rest ? (double)val : (double)val / p.tau - te.log_sum, pj = exp(logp);
          te.mass += pj;
          if (pj != 0.) { te.own += pj * logp; te.cross += pj * ((double)zid / p.tau); }
        }
        te.mass = warp_sum64(te.mass);
        te.own = warp_sum64(te.own);
        te.cross = warp_sum64(te.cross);
        if (REST)
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) ids.join_lane(o, p.tau);
      }
      unsigned next = 0u;
      if (REST) next = mark((long long)t + step, s_mark + (1 - (n & 1)) * words);
      __syncthreads();                                 // the row's sums are there, its marks are no longer read
      if (REST && first) {
        float val;
        for (int j = lane; j < p.K; j += 32)
          if (first >> (j >> 5) & 1u) marks[entry(t, j, val) >> 5] = 0u;
      }
      __syncwarp();
      first = next;
      Lse<BOTH> acc = red[n & 1][lane % (NT / 32)];
#pragma unroll
      for (int o = NT / 64; o > 0; o >>= 1) acc.join_lane(o, p.tau);
      if (lane != 0) continue;
      float* st = p.stats + (long long)t * 4;
      if (!live) {
        p.loss[t] = 0.f;
        st[0] = st[1] = st[2] = st[3] = 0.f;
        p.teacher[t] = 0.;
        continue;
      }
      // with REST the sums are those of the others, and the ids join them
      const float others = acc.log2_s();
      if (REST) acc.join(ids.m, ids.s, ids.z, p.tau);
      const float lse_u = acc.log2_s(), lse_z = BOTH ? acc.log2_z(p.tau) : lse_u;
      double loss = 0., c = te.mass, left = 0.;
      if (p.alpha > 0.f) {
        const double ln2 = 0.6931471805599453094, lse = (double)lse_u * ln2;
        double kl = te.own - te.cross + (te.mass != 0. ? te.mass * lse : 0.);
        if (REST) {
          const double r = 1. - c;
          if (r > 0. && others > -INFINITY) {          // (no id left outside: nothing for the rest to be)
            const double lr = (double)(others - lse_u) * ln2;
            kl += r * (log(r) - lr);
            left = r;
            c += r;
          }
        }
        loss = (double)p.alpha * p.tau * p.tau * kl;
      }
      if (p.alpha < 1.f && label >= 0 && label < p.V) loss += (1. - (double)p.alpha) * (double)(lse_z * LN2 - zlabel);
      p.loss[t] = (float)loss;
      st[0] = lse_u;
      st[1] = lse_z;
      st[2] = (float)c;
      st[3] = others;
      p.teacher[t] = REST ? left : te.log_sum;
    }
    return;
  }

  // ------------------------------ the rows ------------------------------
  RawT raw[AHEAD];
  long long label = 0;
  auto begin = [&](int t) {                            // its label and first loads
    if (t >= p.T) return;
    label = label_of(t);
    const TL* row = row_of(t);
    const Span sp = span_of(row, 0, p.V);
    const RawT* vecs = reinterpret_cast<const RawT*>(row + sp.first);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (i * NT + (int)threadIdx.x < sp.n) raw[i] = vecs[i * NT + (int)threadIdx.x];
  };
  begin(blockIdx.x);
  for (int t = blockIdx.x, n = 0; t < p.T; t += step, ++n) {
    const TL* row = row_of(t);
    const unsigned* marks = s_mark + (n & 1) * words;
    Lse<BOTH> acc;                                     // in units of log2
    if (!ignored(label)) {
      float2 s2 = make_float2(0.f, 0.f), z2 = make_float2(0.f, 0.f);       // sums on acc.m
      auto raise = [&](float mx) {                     // the maximum seen so far; a NaN goes on to the sums
        const float m = mx * cu;
        if (!(m <= acc.m)) {
          if (acc.m > -INFINITY) {
            // (sums that are too large become infinite, and stay so)
            const float d = s2.x + s2.y + (BOTH ? z2.x + z2.y : 0.f) < 0x1p60f ? acc.m - m : INFINITY, f = ex2_approx(d);
            s2 = fmul2(s2, make_float2(f, f));
            if (BOTH) {
              const float g = ex2_approx(d * p.tau);
              z2 = fmul2(z2, make_float2(g, g));
            }
          }
          acc.m = m;
        }
      };
      auto add = [&](float2 x) {
        const float2 a = ffma2(x, make_float2(cu, cu), make_float2(-acc.m, -acc.m));
        float2 e = make_float2(ex2_approx(a.x), ex2_approx(a.y));
        s2 = fadd2(s2, e);
        if (POWER >= 1) {
#pragma unroll
          for (int i = 1; i < POWER; ++i) e = fmul2(e, e);
          z2 = ffma2(e, e, z2);
        }
        if (POWER == 0) z2 = fadd2(z2, make_float2(ex2_approx(a.x * p.tau), ex2_approx(a.y * p.tau)));
      };
      auto take1 = [&](int c) {                        // one element
        if (REST && (marks[c >> 5] >> (c & 31) & 1u)) return;
        const float x = load1(row + c);
        raise(x);
        if (acc.m != -INFINITY) add(make_float2(x, -INFINITY));
      };
      const Span sp = span_of(row, 0, p.V);
      const RawT* vecs = reinterpret_cast<const RawT*>(row + sp.first);
      const int head = sp.first - sp.lo, edge = head + (sp.hi - sp.first - sp.n * N);        // fewer than 2 N elements
      auto take_edge = [&]() {
        if ((int)threadIdx.x < edge) take1((int)threadIdx.x < head ? sp.lo + (int)threadIdx.x : sp.first + sp.n * N + (int)threadIdx.x - head);
      };
      // The sums go over the largest of the thread's first elements, without a look at the others: 36 instead of 83 instructions for 8
      // elements.  Where that was no measure, the thread goes over its part once more, on its largest element.  It was one where both sums
      // lie within 2^-60 .. 2^60, here and whenever the maximum was raised: then the 512 of a row do not overflow together, what a factor of
      // a larger maximum flushes to 0 (below 2^-126) is less than 2^-66 of what has that maximum, and so is what the exponential has
      // flushed here (an id, which REST leaves out, may lie far above all others).
      if ((int)threadIdx.x < sp.n) acc.m = fmax_nan(largest(raw[0]) * cu, -1e30f);
      for (int v0 = threadIdx.x; v0 < sp.n; v0 += NT * AHEAD) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
          const int v = v0 + i * NT, later = v + AHEAD * NT;
          const RawT now = raw[i];
          if (later < sp.n) raw[i] = vecs[later];
          if (v >= sp.n) continue;
          if (REST) {
            // N bits from bit c on
            const int c = sp.first + v * N;
            const unsigned lo = marks[c >> 5], hi = (c & 31) + N > 32 ? marks[(c >> 5) + 1] : 0u;
            if (__funnelshift_r(lo, hi, c & 31) & ((1u << N) - 1u)) {
              for (int k = 0; k < N; ++k) take1(c + k);
              continue;
            }
          }
          float2 x[N / 2];
          pairs(now, x);
#pragma unroll
          for (int k = 0; k < N / 2; ++k) add(x[k]);
        }
      }
      take_edge();
      acc.s = s2.x + s2.y;
      acc.z = z2.x + z2.y;
      auto measured = [](float v) { return v > 0x1p-60f && v < 0x1p60f; };
      if (!measured(acc.s) || (BOTH && !measured(acc.z))) {
        acc.m = -INFINITY;
        s2 = z2 = make_float2(0.f, 0.f);
        for (int v = threadIdx.x; v < sp.n; v += NT)
          for (int k = 0; k < N; ++k) take1(sp.first + v * N + k);
        take_edge();
        acc.s = s2.x + s2.y;
        acc.z = z2.x + z2.y;
      }
    }
    if (p.T - t > step) begin(t + step);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc.join_lane(o, p.tau);
    if (lane == 0) red[n & 1][threadIdx.x >> 5] = acc;
    __syncthreads();
  }
}

// CTA (t, part): columns [part, part + 1) * V / parts of row t.
template <typename TL, int POWER, int NT>
__global__ void __launch_bounds__(NT, 1024 / NT) distill_bwd_kernel(const DistillParams p) {
  b200::begin_kernel();
  __shared__ int s_id[MAX_K];
  __shared__ float s_p[MAX_K];
  constexpr int N = Vec<TL>::N, SLOTS = MAX_K / NT;
  const long long t = blockIdx.x;
  const int lo = (int)((long long)p.V * blockIdx.y / gridDim.y), hi = (int)((long long)p.V * (blockIdx.y + 1) / gridDim.y);
  const TL* row = reinterpret_cast<const TL*>(p.logits) + t * p.ld;
  TL* out = reinterpret_cast<TL*>(p.grad) + t * p.ld_grad;
  const long long label = p.labels != nullptr ? p.labels[t] : 0;
  const bool live = p.labels == nullptr || label != p.ignore, labelled = live && p.alpha < 1.f && label >= 0 && label < p.V;
  const float gy = live ? p.gy[t] : 0.f;
  const float lse_u = p.stats[t * 4], lse_z = p.stats[t * 4 + 1], c = p.stats[t * 4 + 2], others = p.stats[t * 4 + 3];
  const float left = p.rest ? (float)p.teacher[t] : 0.f;
  const float gu = gy * p.alpha * p.tau, gz = labelled ? gy * (1.f - p.alpha) : 0.f;
  const float cu = LOG2E / p.tau;
  // the elements that a thread each writes at the end
  float zid[SLOTS], zlabel = 0.f;
  int id[SLOTS];
  if (live) {
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
      const int j = threadIdx.x + i * NT;
      id[i] = -1;
      zid[i] = 0.f;
      if (j < p.K && p.alpha > 0.f) {
        const long long v = id_at(p, t * p.K + j);
        const float val = value_at(p, t * p.K + j);
        const bool there = v >= 0 && v < p.V && val != -INFINITY;
        s_id[j] = there ? (int)v : -1;
        s_p[j] = there ? (float)exp(p.rest ? (double)val : (double)val / p.tau - p.teacher[t]) : 0.f;
        if (there && v >= lo && v < hi) { id[i] = (int)v; zid[i] = load1(row + v); }
      }
    }
    if (threadIdx.x == 0 && labelled && label >= lo && label < hi) zlabel = load1(row + label);
    __syncthreads();
  }
  // One exponential e = 2^(u - shift) of an element that is not among the ids (what it is of an id does not matter: that is written again), at
  // most 1 on each of these: the log-sum-exp of u, or of u outside the ids (rest: q = e 2^(shift - lse_u), q / R = e), or (POWER above 0)
  // lse_z / tau, whose e is the tau-th root of q1, unless that lies so far above all others that e would flush to 0.  (q1 is then below
  // 2^-120 of e, and `left`, which e has beside it, 2^-53 or more: q1 is not added.  A branch for it took 7 % of the pass.)
  const float root = POWER >= 1 ? lse_z / p.tau : 0.f;
  const bool by_root = POWER >= 1 && !(left > 0.f && root - others > 60.f);
  const float shift = by_root ? root : left > 0.f ? others : lse_u, gr = by_root ? gz : 0.f;
  const float fq = ex2_approx(shift - lse_u), fe = gu * (c * fq - (left > 0.f ? left * ex2_approx(shift - others) : 0.f));
  auto other = [&](float2 x) -> float2 {
    const float2 a = ffma2(x, make_float2(cu, cu), make_float2(-shift, -shift));
    float2 e = make_float2(ex2_approx(a.x), ex2_approx(a.y));
    if (POWER < 0) return fmul2(e, make_float2(fe + gz * fq, fe + gz * fq));
    float2 z;
    if (POWER >= 1) {
      z = fmul2(e, e);
#pragma unroll
      for (int i = 1; i < POWER; ++i) z = fmul2(z, z);
      z = fmul2(z, make_float2(gr, gr));
    } else {
      const float2 b = ffma2(x, make_float2(LOG2E, LOG2E), make_float2(-lse_z, -lse_z));
      z = fmul2(make_float2(ex2_approx(b.x), ex2_approx(b.y)), make_float2(gz, gz));
    }
    return ffma2(e, make_float2(fe, fe), z);
  };
  const Span sp = span_of(out, lo, hi);
  const bool vec = (((uintptr_t)row ^ (uintptr_t)out) & 15) == 0;     // both rows are aligned at the same columns
  const int head = sp.first - sp.lo, body = sp.n * N;
  if (!live) {
    float zero[N] = {};
    for (int v = threadIdx.x; v < sp.n; v += NT) store_vec(out + sp.first + v * N, zero);
    for (int i = threadIdx.x; i < hi - lo - body; i += NT) store1(out + (i < head ? lo + i : lo + i + body), 0.f);
    return;
  }
  if (vec) {
    const typename Raw<TL>::T* src = reinterpret_cast<const typename Raw<TL>::T*>(row + sp.first);
    for (int v0 = 0; v0 < sp.n; v0 += NT * AHEAD) {
      typename Raw<TL>::T raw[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int v = v0 + i * NT + (int)threadIdx.x;
        if (v < sp.n) raw[i] = src[v];
      }
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int v = v0 + i * NT + (int)threadIdx.x;
        if (v >= sp.n) continue;
        float2 x[N / 2];
        pairs(raw[i], x);
        float y[N];
#pragma unroll
        for (int k = 0; k < N / 2; ++k) {
          const float2 g = other(x[k]);
          y[2 * k] = g.x;
          y[2 * k + 1] = g.y;
        }
        store_vec(out + sp.first + v * N, y);
      }
    }
  } else {
    for (int i = sp.first + (int)threadIdx.x; i < sp.first + body; i += NT) store1(out + i, other(make_float2(load1(row + i), 0.f)).x);
  }
  for (int i = threadIdx.x; i < hi - lo - body; i += NT) {
    const int col = i < head ? lo + i : lo + i + body;
    store1(out + col, other(make_float2(load1(row + col), 0.f)).x);
  }
  __syncthreads();
  auto special = [&](int v, float z) {
    float pv = 0.f;
    bool among = false;
    if (p.alpha > 0.f)
      for (int j = 0; j < p.K; ++j)
        if (s_id[j] == v) { pv += s_p[j]; among = true; }
    float g = gu * (c * ex2_approx(fmaf(z, cu, -lse_u)) - (among || !(left > 0.f) ? pv : left * ex2_approx(fmaf(z, cu, -others))));
    if (labelled) g += gz * (ex2_approx(fmaf(z, LOG2E, -lse_z)) - ((long long)v == label ? 1.f : 0.f));
    store1(out + v, g);
  };
  // (equal ids write equal values)
#pragma unroll
  for (int i = 0; i < SLOTS; ++i)
    if (id[i] >= 0) special(id[i], zid[i]);
  if (threadIdx.x == 0 && labelled && label >= lo && label < hi) special((int)label, zlabel);
}

int check_distill(const char* what, const DistillParams& p) {
  if (p.T < 0 || p.T > MAX_T || p.V < 1 || p.V > (1 << 30) || p.K < 1 || p.K > MAX_K)
    return b200::fail(930, "%s: T=%d, V=%d, K=%d (1 to %d)", what, p.T, p.V, p.K, MAX_K);
  if (!(p.tau > 0.f) || !(p.alpha >= 0.f && p.alpha <= 1.f)) return b200::fail(931, "%s: temperature %g, alpha %g", what, p.tau, p.alpha);
  if (p.alpha < 1.f && p.labels == nullptr) return b200::fail(932, "%s: the cross-entropy wants labels", what);
  return 0;
}

int set_smem(const void* fn, size_t bytes) {
  if (bytes <= 40 * 1024) return 0;                    // (what a launch has without asking, 48 KB, is for the kernel's own variables too)
  if (bytes > MAX_SMEM) return b200::fail(933, "distill: marks of %zu bytes, %d at most", bytes, MAX_SMEM);
  // (always the most of all vocabularies: a call of another thread with a smaller one may come between this and the launch)
  const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_SMEM);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return b200::fail(933, "distill: cannot set %d bytes of shared memory: %s", MAX_SMEM, cudaGetErrorString(e));
  }
  return 0;
}

// How the terms of z come from those of u (see distill_fwd_kernel).
int power_of(const DistillParams& p) {
  if (p.alpha >= 1.f || p.tau == 1.f) return -1;
  return p.tau == 2.f ? 1 : p.tau == 4.f ? 2 : p.tau == 8.f ? 3 : 0;
}

// Many short rows: what counts is how many are under way, not how fast one is.  us, forward and backward, 512 threads against 64 and 128:
// 16384 x 1000 fp32 213 + 261, 46 + 80; 8192 x 4096 bf16 91 + 143, 24 + 51; 4096 x 50304 bf16 91 + 172, 76 + 152; 4096 x 32000 fp32 78 + 181, 90 + 178.
template <typename TL>
bool short_rows(const DistillParams& p) { return p.T > 2 * b200::sm_count() && (long long)p.V * (int)sizeof(TL) <= SHORT_BYTES; }

template <typename TL, int POWER, int NT>
int launch_fwd(const DistillParams& p, cudaStream_t s) {
  auto k = p.rest ? distill_fwd_kernel<TL, POWER, true, NT> : distill_fwd_kernel<TL, POWER, false, NT>;
  const size_t smem = p.rest ? ((size_t)p.V + 31) / 32 * 8 : 0;
  if (int r = set_smem((const void*)k, smem)) return r;
  const int most = (NT == 512 ? 2 : 10) * b200::sm_count();
  b200::launch(k, p.T < most ? p.T : most, NT + 32, smem, s, p);
  b200::count_launch();
  return b200::check_launch("distill_fwd");
}
template <typename TL, int POWER>
int launch_fwd(const DistillParams& p, cudaStream_t s) {
  return short_rows<TL>(p) ? launch_fwd<TL, POWER, 64>(p, s) : launch_fwd<TL, POWER, 512>(p, s);
}
template <typename TL, int POWER>
int launch_bwd(const DistillParams& p, cudaStream_t s) {
  // few rows: several CTAs a row, of 4096 columns or more
  int parts = 1;
  while (parts < 32 && (long long)p.T * parts < 2 * b200::sm_count() && p.V / (2 * parts) >= 4096) parts *= 2;
  const dim3 grid((unsigned)p.T, (unsigned)parts);
  if (short_rows<TL>(p)) b200::launch(distill_bwd_kernel<TL, POWER, 128>, grid, 128, 0, s, p);
  else b200::launch(distill_bwd_kernel<TL, POWER, 512>, grid, 512, 0, s, p);
  b200::count_launch();
  return b200::check_launch("distill_bwd");
}
template <typename TL>
int dispatch(const DistillParams& p, bool backward, cudaStream_t s) {
  switch (power_of(p)) {
    case -1: return backward ? launch_bwd<TL, -1>(p, s) : launch_fwd<TL, -1>(p, s);
    case 0: return backward ? launch_bwd<TL, 0>(p, s) : launch_fwd<TL, 0>(p, s);
    case 1: return backward ? launch_bwd<TL, 1>(p, s) : launch_fwd<TL, 1>(p, s);
    case 2: return backward ? launch_bwd<TL, 2>(p, s) : launch_fwd<TL, 2>(p, s);
    default: return backward ? launch_bwd<TL, 3>(p, s) : launch_fwd<TL, 3>(p, s);
  }
}

}  // namespace

// logits [T, V] (fp32 or bf16, rows ld apart); loss [T], stats [T, 4], teacher [T] are kept for the backward pass.
B200_API int b200_distill_fwd(const void* logits, int is_bf16, long long ld, const long long* labels, const void* ids, int ids64, const void* values,
                              int values_bf16, int T, int K, int V, int rest, float alpha, float tau, long long ignore, float* loss, float* stats,
                              double* teacher, void* stream) {
  DistillParams p = {logits, ld, labels, ids, values, ids64, values_bf16, T, K, V, rest, alpha, tau, ignore, loss, stats, teacher, nullptr, nullptr, 0};
  if (int r = check_distill("distill_fwd", p)) return r;
  if (T == 0) return 0;
  return is_bf16 ? dispatch<__nv_bfloat16>(p, false, (cudaStream_t)stream) : dispatch<float>(p, false, (cudaStream_t)stream);
}

// grad [T, V] (the logits' type, rows ld_grad apart; may be the logits themselves) = gy[t] * dloss[t] / dlogits
B200_API int b200_distill_bwd(const void* logits, int is_bf16, long long ld, const long long* labels, const void* ids, int ids64, const void* values,
                              int values_bf16, int T, int K, int V, int rest, float alpha, float tau, long long ignore, const float* stats,
                              const double* teacher, const float* gy, void* grad, long long ld_grad, void* stream) {
  DistillParams p = {logits, ld, labels, ids, values, ids64, values_bf16, T, K, V, rest, alpha, tau, ignore, nullptr,
                     const_cast<float*>(stats), const_cast<double*>(teacher), gy, grad, ld_grad};
  if (int r = check_distill("distill_bwd", p)) return r;
  if (T == 0) return 0;
  return is_bf16 ? dispatch<__nv_bfloat16>(p, true, (cudaStream_t)stream) : dispatch<float>(p, true, (cudaStream_t)stream);
}
