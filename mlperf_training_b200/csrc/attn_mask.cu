// Masks of attention as intervals (attn_mask.cuh) from document ids and prefix flags.
//
// A CTA per sequence scans its positions twice, 4096 at a time: from the end for the next start of a document and the next position without a
// flag, then from the front for the start of the document, after which both intervals of a position are known.  Then a warp per tile of
// 128 rows or keys gathers the range of tiles that it meets and the bounds within which all of it is visible.  A second launch
// sorts the tiles of all sequences by that range, longest first, for the schedules of the attention kernels.
#include "attn_mask.cuh"
#include "runtime.h"

namespace {

using b200::MaskLayout;

constexpr int NT = 1024, PER = 4, CHUNK = NT * PER;
constexpr int BINS = 2048;
constexpr unsigned ALL = 0xffffffffu;

struct MaskParams {
  MaskLayout m;
  const void* ids;             // [B, Skv], int32 or int64, or null: one document
  const uint8_t* flags;        // [B, Skv] or null
  int ids64, causal, window;
  int* buf;
};

B200_DEVICE long long id_at(const MaskParams& p, long long i) {
  return p.ids64 ? reinterpret_cast<const long long*>(p.ids)[i] : (long long)reinterpret_cast<const int*>(p.ids)[i];
}

// Inclusive scan over the CTA's chunk (thread-major) in index order, from `carry`; MAXOP: running maximum, else running minimum from the end.
template <bool MAXOP>
B200_DEVICE void block_scan(int (&v)[PER], int carry, int* red) {
  auto op = [](int a, int b) { return MAXOP ? max(a, b) : min(a, b); };
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (MAXOP) {
#pragma unroll
    for (int i = 1; i < PER; ++i) v[i] = op(v[i], v[i - 1]);
  } else {
#pragma unroll
    for (int i = PER - 2; i >= 0; --i) v[i] = op(v[i], v[i + 1]);
  }
  int t = MAXOP ? v[PER - 1] : v[0];
  const int none = MAXOP ? -1 : 0x7fffffff;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = MAXOP ? __shfl_up_sync(ALL, t, o) : __shfl_down_sync(ALL, t, o);
    if (MAXOP ? lane >= o : lane + o < 32) t = op(t, u);
  }
  __syncthreads();
  if (lane == (MAXOP ? 31 : 0)) red[warp] = t;
  __syncthreads();
  int before = MAXOP ? __shfl_up_sync(ALL, t, 1) : __shfl_down_sync(ALL, t, 1);
  if (lane == (MAXOP ? 0 : 31)) before = none;
  before = op(before, carry);
  if (MAXOP) { for (int w = 0; w < warp; ++w) before = op(before, red[w]); }
  else { for (int w = warp + 1; w < NT / 32; ++w) before = op(before, red[w]); }
#pragma unroll
  for (int i = 0; i < PER; ++i) v[i] = op(v[i], before);
}

__global__ void __launch_bounds__(NT) attn_mask_kernel(const __grid_constant__ MaskParams p) {
  b200::begin_kernel();
  __shared__ int red[NT / 32];
  __shared__ int s_carry[2];
  const MaskLayout& m = p.m;
  const int b = blockIdx.x, S = m.Skv, off = m.Skv - m.Sq;
  const long long base = (long long)b * S;
  int2* q_iv = reinterpret_cast<int2*>(p.buf + m.q_iv) + (long long)b * m.Sp;
  int2* k_iv = reinterpret_cast<int2*>(p.buf + m.k_iv) + (long long)b * m.Kp;
  int2* next = reinterpret_cast<int2*>(p.buf + m.scratch) + base;     // (end of the document, next position without a flag)
  auto starts = [&](int i) { return i == 0 || (p.ids != nullptr && id_at(p, base + i) != id_at(p, base + i - 1)); };
  const int chunks = (S + CHUNK - 1) / CHUNK;

  int end_carry = S, bare_carry = S;
  for (int c = chunks - 1; c >= 0; --c) {
    const int i0 = c * CHUNK + (int)threadIdx.x * PER;
    int e[PER], f[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int i = i0 + k;
      e[k] = i + 1 < S && starts(i + 1) ? i + 1 : S;
      f[k] = i < S && !(p.flags != nullptr && p.flags[base + i]) ? i : S;
    }
    block_scan<false>(e, end_carry, red);
    block_scan<false>(f, bare_carry, red);
#pragma unroll
    for (int k = 0; k < PER; ++k)
      if (i0 + k < S) next[i0 + k] = make_int2(e[k], f[k]);
    if (threadIdx.x == 0) { s_carry[0] = e[0]; s_carry[1] = f[0]; }
    __syncthreads();
    end_carry = s_carry[0];
    bare_carry = s_carry[1];
  }
  __syncthreads();

  int start_carry = 0;
  for (int c = 0; c < chunks; ++c) {
    const int i0 = c * CHUNK + (int)threadIdx.x * PER;
    int s[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) s[k] = i0 + k < S && starts(i0 + k) ? i0 + k : -1;
    block_scan<true>(s, start_carry, red);
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int i = i0 + k;
      if (i >= S) continue;
      const int ds = s[k], de = next[i].x;
      int lo = i, hi = i, first = i, end = i;                         // a negative id: nothing
      if (p.ids == nullptr || id_at(p, base + i) >= 0) {
        const int pe = p.flags != nullptr ? min(next[ds].y, de) : ds;
        lo = p.window > 0 ? max(ds, i - p.window + 1) : ds;
        hi = p.causal ? max(i + 1, pe) : de;
        first = (!p.causal || i < pe) ? ds : i;
        end = p.window > 0 && i < de - p.window ? i + p.window : de;
      }
      first = max(first - off, 0);                                    // as queries
      end = max(end - off, 0);
      k_iv[i] = first < end ? make_int2(first, end) : make_int2(max(i - off, 0), max(i - off, 0));
      if (i >= off) q_iv[i - off] = make_int2(lo, hi);
    }
    if (threadIdx.x == NT - 1) s_carry[0] = s[PER - 1];
    __syncthreads();
    start_carry = s_carry[0];
  }
  for (int i = S + (int)threadIdx.x; i < m.Kp; i += NT) k_iv[i] = make_int2(0, 0);
  for (int i = m.Sq + (int)threadIdx.x; i < m.Sp; i += NT) q_iv[i] = make_int2(0, 0);
  __syncthreads();

  // tiles: rows that are there, of either side
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nq = m.Sp / 128, nk = m.Kp / 128;
  for (int t = warp; t < nq + nk; t += NT / 32) {
    const bool of_q = t < nq;
    const int tile = of_q ? t : t - nq, rows = of_q ? m.Sq : S;
    const int2* iv = (of_q ? q_iv : k_iv) + tile * 128;
    int lo_min = 0x7fffffff, hi_max = 0, lo_max = 0, hi_min = 0x7fffffff;
    for (int r = lane; r < 128 && tile * 128 + r < rows; r += 32) {
      const int2 v = iv[r];
      if (v.x < v.y) { lo_min = min(lo_min, v.x); hi_max = max(hi_max, v.y); }
      lo_max = max(lo_max, v.x);
      hi_min = min(hi_min, v.x < v.y ? v.y : v.x);
    }
    lo_min = __reduce_min_sync(ALL, lo_min);
    hi_max = __reduce_max_sync(ALL, hi_max);
    lo_max = __reduce_max_sync(ALL, lo_max);
    hi_min = __reduce_min_sync(ALL, hi_min);
    if (lane == 0) {
      int4 o = make_int4(0, 0, lo_max, hi_min);
      if (lo_min < hi_max) { o.x = lo_min / 128; o.y = (hi_max + 127) / 128; }
      if (!of_q && tile * 128 + 128 > S) o.w = 0;                     // keys behind the last: always masked
      (reinterpret_cast<int4*>(p.buf + (of_q ? m.qt : m.kt)) + (long long)b * (of_q ? nq : nk))[tile] = o;
    }
  }
}

// CTA 0: pairs of query tiles, CTA 1: key tiles, by their number of tiles on the other side, most first (numbers above BINS - 1 alike).
__global__ void __launch_bounds__(NT) attn_mask_order_kernel(const MaskLayout m, int* buf) {
  b200::begin_kernel();
  __shared__ int bins[BINS];
  __shared__ int red[NT / 32];
  const bool of_q = blockIdx.x == 0;
  const int n = of_q ? m.B * (m.Sp / 256) : m.B * (m.Kp / 128);
  const int4* t = reinterpret_cast<const int4*>(buf + (of_q ? m.qt : m.kt));
  int* out = buf + (of_q ? m.oq : m.ok);
  auto bin = [&](int i) {
    const int cost = of_q ? t[2 * i].y - t[2 * i].x + t[2 * i + 1].y - t[2 * i + 1].x : t[i].y - t[i].x;
    return BINS - 1 - min(max(cost, 0), BINS - 1);
  };
  for (int i = threadIdx.x; i < BINS; i += NT) bins[i] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += NT) atomicAdd(&bins[bin(i)], 1);
  __syncthreads();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int a = bins[2 * threadIdx.x], c = bins[2 * threadIdx.x + 1];
  int x = a + c;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(ALL, x, o);
    if (lane >= o) x += u;
  }
  if (lane == 31) red[warp] = x;
  __syncthreads();
  int at = x - a - c;
  for (int w = 0; w < warp; ++w) at += red[w];
  bins[2 * threadIdx.x] = at;
  bins[2 * threadIdx.x + 1] = at + a;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += NT) out[atomicAdd(&bins[bin(i)], 1)] = i;      // (order within a bin: the schedule's alone)
}
static_assert(BINS == 2 * NT, "a thread scans two bins");

}  // namespace

// ints of a mask's buffer (16-byte aligned), or -1
B200_API long long b200_attn_mask_ints(int B, int Sq, int Skv) {
  if (B < 1 || Sq < 1 || Skv < Sq || Skv > (1 << 30)) return -1;
  return MaskLayout::of(B, Sq, Skv).total;
}

// Queries are the last Sq of Skv positions.  ids [B, Skv] (int32 or int64) or null, flags [B, Skv] bytes or null.
B200_API int b200_attn_mask(const void* ids, int ids64, const uint8_t* flags, int B, int Sq, int Skv, int causal, int window, int* buf, void* stream) {
  if (B < 1 || Sq < 1 || Skv < Sq || Skv > (1 << 30)) return b200::fail(940, "attn_mask: B=%d, Sq=%d, Skv=%d", B, Sq, Skv);
  if (window < 0 || (flags != nullptr && !causal)) return b200::fail(941, "attn_mask: window %d, a prefix wants a causal mask", window);
  MaskParams p = {MaskLayout::of(B, Sq, Skv), ids, flags, ids64, causal, window, buf};
  if ((long long)B * (p.m.Kp / 128) > 0x3fffffff) return b200::fail(942, "attn_mask: %d sequences of %d keys", B, Skv);
  b200::launch(attn_mask_kernel, B, NT, 0, (cudaStream_t)stream, p);
  b200::launch(attn_mask_order_kernel, 2, NT, 0, (cudaStream_t)stream, p.m, buf);
  b200::count_launch(2);
  return b200::check_launch("attn_mask");
}
