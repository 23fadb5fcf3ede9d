// Distillation from a teacher's largest logits, mixed with cross-entropy, per token of student logits z [V]:
//
//   loss = a tau^2 KL + (1 - a) CE            u = z / tau, q = softmax(u), q1 = softmax(z)
//   KL   = sum_j p_j (log p_j - log q[id_j])  over the teacher's K entries (id_j, t_j)
//          plain: p = softmax(t / tau) over the entries that are there
//          rest:  p_j = exp(t_j); what they leave, r = 1 - sum p, is one further event "any other id": r (log r - log R),
//                 R = the student's mass outside the ids
//   dz   = gy (a tau (c q_v - p_v - [v not among the ids] (r / R) q_v) + (1 - a) (q1_v - [v = label])),  c = sum p + r
//
// An entry whose id is outside the vocabulary or whose value is -inf is not there.  Tokens labelled `ignore` have loss and gradient 0; so has
// the cross-entropy of another label outside the vocabulary.
//
// Forward: one pass over the row for the log-sum-exp of u and of z (the same pass; one exponential where tau is 1 or a is 1) on a running
// maximum; with `rest` the ids are marked in a bitmap and left out of the sum, which is then that of the others without cancellation, and
// the ids' own terms join it at the end.  Backward: the row again from the saved log-sum-exps, written as it is read; the elements of
// the ids and the label are then written once more by a thread each, from logits read before any was overwritten, so the gradient may take
// the logits' place.  p, r and their logarithms are in fp64 (r = 1 - sum p cancels), all else in fp32.
#include "common.cuh"
#include "runtime.h"

namespace {

constexpr int NT = 512, MAX_K = 1024, SLOTS = MAX_K / NT;
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
  float* stats;             // [T, 4]: log-sum-exp of u and of z (log2 units), c, r / R
  double* teacher;          // [T]: log-sum-exp of t / tau (plain)
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
B200_DEVICE void load_vec(const float* p, float (&x)[4]) {
  const float4 v = *reinterpret_cast<const float4*>(p);
  x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
}
B200_DEVICE void load_vec(const __nv_bfloat16* p, float (&x)[8]) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const float2 a = unpack_bf16x2(u.x), b = unpack_bf16x2(u.y), c = unpack_bf16x2(u.z), d = unpack_bf16x2(u.w);
  x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y; x[4] = c.x; x[5] = c.y; x[6] = d.x; x[7] = d.y;
}
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

// A sum of 2^(x - m) for the largest m so far.
struct Lse {
  float m, s;
  B200_DEVICE void join(float m2, float s2) {
    const float n = fmax_nan(m, m2);
    s = (m == -INFINITY ? 0.f : s * ex2_approx(m - n)) + (m2 == -INFINITY ? 0.f : s2 * ex2_approx(m2 - n));
    m = n;
  }
  B200_DEVICE float log2() const { return m == -INFINITY ? -INFINITY : m + log2f(s); }
};
B200_DEVICE Lse block_join(Lse v, Lse* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v.join(__shfl_xor_sync(0xffffffffu, v.m, o), __shfl_xor_sync(0xffffffffu, v.s, o));
  const int w = threadIdx.x >> 5, l = threadIdx.x & 31;
  __syncthreads();
  if (l == 0) red[w] = v;
  __syncthreads();
  v = red[l % (NT / 32)];
#pragma unroll
  for (int o = NT / 64; o > 0; o >>= 1) v.join(__shfl_xor_sync(0xffffffffu, v.m, o), __shfl_xor_sync(0xffffffffu, v.s, o));
  return v;
}
B200_DEVICE double block_sum(double v, double* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.;
  for (int i = 0; i < NT / 32; ++i) v += red[i];
  return v;
}
B200_DEVICE double block_max(double v, double* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
  for (int i = 1; i < NT / 32; ++i) v = fmax(v, red[i]);
  return v;
}

// One CTA a row.  BOTH: the log-sum-exp of z beside that of u.  REST: ids are left out of the pass.
template <typename TL, bool BOTH, bool REST>
__global__ void __launch_bounds__(NT) distill_fwd_kernel(const DistillParams p) {
  b200::begin_kernel();
  extern __shared__ unsigned s_mark[];                 // REST: a bit for each id
  __shared__ Lse red[NT / 32];
  __shared__ double redd[NT / 32];
  const long long t = blockIdx.x;
  const long long label = p.labels != nullptr ? p.labels[t] : 0;
  float* st = p.stats + t * 4;
  if (p.labels != nullptr && label == p.ignore) {      // (the whole CTA)
    if (threadIdx.x == 0) {
      p.loss[t] = 0.f;
      st[0] = st[1] = st[2] = st[3] = 0.f;
      p.teacher[t] = 0.;
    }
    return;
  }
  const TL* row = reinterpret_cast<const TL*>(p.logits) + t * p.ld;
  // this thread's entries
  int id[SLOTS];
  float val[SLOTS], zid[SLOTS];
  bool own[SLOTS];                                     // the first of equal ids
#pragma unroll
  for (int i = 0; i < SLOTS; ++i) {
    const int j = threadIdx.x + i * NT;
    id[i] = -1;
    val[i] = -INFINITY;
    zid[i] = 0.f;
    own[i] = false;
    if (j < p.K && p.alpha > 0.f) {
      const long long v = id_at(p, t * p.K + j);
      val[i] = value_at(p, t * p.K + j);
      if (v >= 0 && v < p.V && val[i] != -INFINITY) {
        id[i] = (int)v;
        zid[i] = load1(row + v);
      }
    }
  }
  if (REST) {
    for (int i = threadIdx.x; i < (p.V + 31) / 32; i += NT) s_mark[i] = 0u;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < SLOTS; ++i)
      if (id[i] >= 0) own[i] = !(atomicOr(&s_mark[id[i] >> 5], 1u << (id[i] & 31)) >> (id[i] & 31) & 1u);
    __syncthreads();
  }
  // the pass: u and z in units of log2
  const float cz = LOG2E, cu = LOG2E / p.tau;
  Lse lu = {-INFINITY, 0.f};
  float sz = 0.f, mz = -INFINITY;                      // (BOTH) sum for z on the same element's maximum
  constexpr int N = Vec<TL>::N;
  auto take = [&](const auto& x, const int n, const unsigned skip) {
    float mx = -INFINITY;
    for (int i = 0; i < n; ++i)
      if (!REST || !(skip >> i & 1u)) mx = fmax_nan(mx, x[i]);
    if (!(mx * cu <= lu.m)) {                          // (a NaN goes on to the sums)
      const float nu = mx * cu, nz = mx * cz;
      if (lu.m > -INFINITY) {
        lu.s *= ex2_approx(lu.m - nu);
        if (BOTH) sz *= ex2_approx(mz - nz);
      }
      lu.m = nu;
      if (BOTH) mz = nz;
    }
    if (lu.m == -INFINITY) return;
    for (int i = 0; i < n; ++i) {
      if (REST && (skip >> i & 1u)) continue;
      lu.s += ex2_approx(fmaf(x[i], cu, -lu.m));
      if (BOTH) sz += ex2_approx(fmaf(x[i], cz, -mz));
    }
  };
  const Span sp = span_of(row, 0, p.V);
  for (int v = threadIdx.x; v < sp.n; v += NT) {
    const int c = sp.first + v * N;
    float x[N];
    load_vec(row + c, x);
    unsigned skip = 0u;
    if (REST) {
      // N bits from bit c on
      const unsigned lo = s_mark[c >> 5], hi = (c & 31) + N > 32 ? s_mark[(c >> 5) + 1] : 0u;
      skip = __funnelshift_r(lo, hi, c & 31) & ((1u << N) - 1u);
    }
    take(x, N, skip);
  }
  {
    const int edge = (sp.first - sp.lo) + (sp.hi - sp.first - sp.n * N);        // fewer than 2 N elements
    if ((int)threadIdx.x < edge) {
      const int c = (int)threadIdx.x < sp.first - sp.lo ? sp.lo + (int)threadIdx.x : sp.first + sp.n * N + (int)threadIdx.x - (sp.first - sp.lo);
      const float x[1] = {load1(row + c)};
      take(x, 1, REST ? s_mark[c >> 5] >> (c & 31) & 1u : 0u);
    }
  }
  lu = block_join(lu, red);
  // logarithms (base 2) of the sums; with REST those of the others first, then the ids' own terms
  const float others = lu.log2();
  if (REST) {
    Lse mine = {-INFINITY, 0.f};
#pragma unroll
    for (int i = 0; i < SLOTS; ++i)
      if (own[i]) mine.join(zid[i] * cu, 1.f);
    mine = block_join(mine, red);
    lu.join(mine.m, mine.s);
  }
  const float lse_u = lu.log2();
  float lse_z = lse_u;
  if (BOTH) {
    Lse lz = {mz, sz};
    lz = block_join(lz, red);
    if (REST) {
      Lse mine = {-INFINITY, 0.f};
#pragma unroll
      for (int i = 0; i < SLOTS; ++i)
        if (own[i]) mine.join(zid[i] * cz, 1.f);
      mine = block_join(mine, red);
      lz.join(mine.m, mine.s);
    }
    lse_z = lz.log2();
  }
  // the teacher
  double kl = 0., lt = 0., c = 0., ratio = 0.;
  if (p.alpha > 0.f) {
    double mass = 0.;
    if (!p.rest) {
      double m = -INFINITY, s = 0.;
#pragma unroll
      for (int i = 0; i < SLOTS; ++i)
        if (id[i] >= 0) m = fmax(m, (double)val[i] / p.tau);
      m = block_max(m, redd);
#pragma unroll
      for (int i = 0; i < SLOTS; ++i)
        if (id[i] >= 0) s += exp((double)val[i] / p.tau - m);
      s = block_sum(s, redd);
      lt = s > 0. ? m + log(s) : 0.;
    }
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
      if (id[i] < 0) continue;
      const double logp = p.rest ? (double)val[i] : (double)val[i] / p.tau - lt, pj = exp(logp);
      mass += pj;
      if (pj != 0.) kl += pj * (logp - (double)(zid[i] * cu - lse_u) * 0.6931471805599453094);
    }
    kl = block_sum(kl, redd);
    c = block_sum(mass, redd);
    if (REST) {
      const double r = 1. - c;
      if (r > 0. && others > -INFINITY) {              // (no id left outside: nothing for the rest to be)
        const double lr = (double)(others - lse_u) * 0.6931471805599453094;
        kl += r * (log(r) - lr);
        ratio = r / exp(lr);
        c += r;
      }
    }
  }
  if (threadIdx.x == 0) {
    double loss = p.alpha > 0.f ? (double)p.alpha * p.tau * p.tau * kl : 0.;
    if (p.alpha < 1.f && label >= 0 && label < p.V) loss += (1. - (double)p.alpha) * (double)(lse_z * LN2 - load1(row + label));
    p.loss[t] = (float)loss;
    st[0] = lse_u;
    st[1] = lse_z;
    st[2] = (float)c;
    st[3] = (float)ratio;
    p.teacher[t] = lt;
  }
}

// CTA (t, part): columns [part, part + 1) * V / parts of row t.
template <typename TL, bool BOTH>
__global__ void __launch_bounds__(NT) distill_bwd_kernel(const DistillParams p) {
  b200::begin_kernel();
  __shared__ int s_id[MAX_K];
  __shared__ float s_p[MAX_K];
  constexpr int N = Vec<TL>::N;
  const long long t = blockIdx.x;
  const int lo = (int)((long long)p.V * blockIdx.y / gridDim.y), hi = (int)((long long)p.V * (blockIdx.y + 1) / gridDim.y);
  const TL* row = reinterpret_cast<const TL*>(p.logits) + t * p.ld;
  TL* out = reinterpret_cast<TL*>(p.grad) + t * p.ld_grad;
  const long long label = p.labels != nullptr ? p.labels[t] : 0;
  const bool live = p.labels == nullptr || label != p.ignore, labelled = live && p.alpha < 1.f && label >= 0 && label < p.V;
  const float gy = live ? p.gy[t] : 0.f;
  const float lse_u = p.stats[t * 4], lse_z = p.stats[t * 4 + 1], c = p.stats[t * 4 + 2], ratio = p.stats[t * 4 + 3];
  const float gu = gy * p.alpha * p.tau, gz = labelled ? gy * (1.f - p.alpha) : 0.f;
  const float cu = LOG2E / p.tau;
  const float fu = gu * (c - ratio);                   // of q, outside the ids
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
  auto other = [&](float x) -> float {
    if (!BOTH) return (fu + gz) * ex2_approx(fmaf(x, cu, -lse_u));
    return fu * ex2_approx(fmaf(x, cu, -lse_u)) + gz * ex2_approx(fmaf(x, LOG2E, -lse_z));
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
  for (int v = threadIdx.x; v < sp.n; v += NT) {
    const int col = sp.first + v * N;
    float x[N];
    if (vec) load_vec(row + col, x);
    else
      for (int i = 0; i < N; ++i) x[i] = load1(row + col + i);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = other(x[i]);
    store_vec(out + col, x);
  }
  for (int i = threadIdx.x; i < hi - lo - body; i += NT) {
    const int col = i < head ? lo + i : lo + i + body;
    store1(out + col, other(load1(row + col)));
  }
  __syncthreads();
  auto special = [&](int v, float z) {
    float pv = 0.f;
    bool among = false;
    if (p.alpha > 0.f)
      for (int j = 0; j < p.K; ++j)
        if (s_id[j] == v) { pv += s_p[j]; among = true; }
    float g = gu * ((among ? c : c - ratio) * ex2_approx(fmaf(z, cu, -lse_u)) - pv);
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
  if (p.T < 0 || p.V < 1 || p.V > (1 << 30) || p.K < 1 || p.K > MAX_K)
    return b200::fail(930, "%s: T=%d, V=%d, K=%d (1 to %d)", what, p.T, p.V, p.K, MAX_K);
  if (!(p.tau > 0.f) || !(p.alpha >= 0.f && p.alpha <= 1.f)) return b200::fail(931, "%s: temperature %g, alpha %g", what, p.tau, p.alpha);
  if (p.alpha < 1.f && p.labels == nullptr) return b200::fail(932, "%s: the cross-entropy wants labels", what);
  return 0;
}

int set_smem(const void* fn, size_t bytes) {
  if (bytes <= 48 * 1024) return 0;
  const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return b200::fail(933, "distill: cannot set %zu bytes of shared memory: %s", bytes, cudaGetErrorString(e));
  }
  return 0;
}

template <typename TL>
int launch_fwd(const DistillParams& p, cudaStream_t s) {
  const bool both = p.alpha < 1.f && p.tau != 1.f;
  auto k = p.rest ? (both ? distill_fwd_kernel<TL, true, true> : distill_fwd_kernel<TL, false, true>)
                  : (both ? distill_fwd_kernel<TL, true, false> : distill_fwd_kernel<TL, false, false>);
  const size_t smem = p.rest ? ((size_t)p.V + 31) / 32 * 4 : 0;
  if (int r = set_smem((const void*)k, smem)) return r;
  b200::launch(k, p.T, NT, smem, s, p);
  b200::count_launch();
  return b200::check_launch("distill_fwd");
}

}  // namespace

// logits [T, V] (fp32 or bf16, rows ld apart); loss [T], stats [T, 4], teacher [T] are kept for the backward pass.
B200_API int b200_distill_fwd(const void* logits, int is_bf16, long long ld, const long long* labels, const void* ids, int ids64, const void* values,
                              int values_bf16, int T, int K, int V, int rest, float alpha, float tau, long long ignore, float* loss, float* stats,
                              double* teacher, void* stream) {
  DistillParams p = {logits, ld, labels, ids, values, ids64, values_bf16, T, K, V, rest, alpha, tau, ignore, loss, stats, teacher, nullptr, nullptr, 0};
  if (int r = check_distill("distill_fwd", p)) return r;
  if (T == 0) return 0;
  return is_bf16 ? launch_fwd<__nv_bfloat16>(p, (cudaStream_t)stream) : launch_fwd<float>(p, (cudaStream_t)stream);
}

// grad [T, V] (the logits' type, rows ld_grad apart; may be the logits themselves) = gy[t] * dloss[t] / dlogits
B200_API int b200_distill_bwd(const void* logits, int is_bf16, long long ld, const long long* labels, const void* ids, int ids64, const void* values,
                              int values_bf16, int T, int K, int V, int rest, float alpha, float tau, long long ignore, const float* stats,
                              const double* teacher, const float* gy, void* grad, long long ld_grad, void* stream) {
  DistillParams p = {logits, ld, labels, ids, values, ids64, values_bf16, T, K, V, rest, alpha, tau, ignore, nullptr,
                     const_cast<float*>(stats), const_cast<double*>(teacher), gy, grad, ld_grad};
  if (int r = check_distill("distill_bwd", p)) return r;
  if (T == 0) return 0;
  const bool both = alpha < 1.f && tau != 1.f;
  auto k = is_bf16 ? (both ? distill_bwd_kernel<__nv_bfloat16, true> : distill_bwd_kernel<__nv_bfloat16, false>)
                   : (both ? distill_bwd_kernel<float, true> : distill_bwd_kernel<float, false>);
  // few rows: several CTAs a row, of 4096 columns or more
  int parts = 1;
  while (parts < 32 && (long long)T * parts < 2 * b200::sm_count() && V / (2 * parts) >= 4096) parts *= 2;
  b200::launch(k, dim3((unsigned)T, (unsigned)parts), NT, 0, (cudaStream_t)stream, p);
  b200::count_launch();
  return b200::check_launch("distill_bwd");
}
