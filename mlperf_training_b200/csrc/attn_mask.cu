// Masks of attention as intervals (attn_mask.cuh) from document ids and prefix flags.
//
// A CTA per sequence; a thread takes 16 neighbouring positions as bit masks (a document starts here, padding, flagged), so that the ends of
// a document inside them are bit searches.  What lies outside comes from two scans over the threads: from the end, the next start and the next
// position without a flag; from the front, the last start with the end of its prefix.  16384 positions go at a time; longer sequences are
// walked once from the end before for what each such chunk has behind it.  Then the warps take tiles of 128 positions, write their
// intervals and reduce the tables of the key tiles (and of the query tiles, where these lie on the same positions).  Then the tiles of all sequences
// are sorted by their range, longest first, for the schedules of the attention kernels: by the same launch where a cluster holds all sequences, else
// by a second one.  Above 4096 positions the tiles of a sequence are shared by the CTAs of a cluster, each of which makes the scans.
// One sequence of 61 positions 6.2 us (7.8 with bins for few tiles), of 8192 9.8 (12.5 by one CTA), of 32768 21 (35); 8 of 16384 12.0 (16.7).
#include "attn_mask.cuh"
#include "runtime.h"

namespace {

using b200::MaskLayout;

constexpr int NT = 1024, PER = 16, CHUNK = NT * PER;
constexpr int BINS = 2048;
constexpr unsigned ALL = 0xffffffffu;

struct MaskParams {
  MaskLayout m;
  const void* ids;             // [B, Skv], int32 or int64, or null: one document
  const uint8_t* flags;        // [B, Skv] or null
  int ids64, causal, window;
  int* buf;
  int parts;                   // CTAs a sequence, neighbours in a cluster: each makes the scans and writes its share of the tiles
  int whole;                   // the cluster holds all sequences, and sorts
};

B200_DEVICE long long id_at(const MaskParams& p, long long i) {
  return p.ids64 ? reinterpret_cast<const long long*>(p.ids)[i] : (long long)reinterpret_cast<const int*>(p.ids)[i];
}

// Bits of positions i0 + k: `start` of a document, `pad`, `flag`.  Positions that are not there: a start, padding, no flag.
struct Bits { unsigned start, pad, flag; };
B200_DEVICE Bits load_bits(const MaskParams& p, long long base, int i0, int S) {
  Bits r = {0u, 0u, 0u};
  const int n = max(min(S - i0, PER), 0);
  if (p.ids != nullptr) {
    long long id[PER];
    const long long at = base + i0;
    if (n == PER && !p.ids64 && ((uintptr_t)(reinterpret_cast<const int*>(p.ids) + at) & 15) == 0) {
#pragma unroll
      for (int k = 0; k < PER; k += 4) {
        const int4 v = *reinterpret_cast<const int4*>(reinterpret_cast<const int*>(p.ids) + at + k);
        id[k] = v.x; id[k + 1] = v.y; id[k + 2] = v.z; id[k + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int k = 0; k < PER; ++k) id[k] = k < n ? id_at(p, at + k) : 0;
    }
    const int lane = threadIdx.x & 31;
    long long before = __shfl_up_sync(ALL, id[PER - 1], 1);
    if (lane == 0 && i0 > 0 && i0 <= S) before = id_at(p, at - 1);
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      if ((k == 0 ? before : id[k - 1]) != id[k]) r.start |= 1u << k;
      if (id[k] < 0) r.pad |= 1u << k;
    }
  }
  if (p.flags != nullptr) {
    const uint8_t* f = p.flags + base + i0;
    if (n == PER && ((uintptr_t)f & 15) == 0) {
      const uint4 v = *reinterpret_cast<const uint4*>(f);
      const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int k = 0; k < PER; ++k)
        if ((w[k / 4] >> (k % 4 * 8)) & 0xffu) r.flag |= 1u << k;
    } else {
      for (int k = 0; k < n; ++k)
        if (f[k]) r.flag |= 1u << k;
    }
  }
  if (i0 == 0) r.start |= 1u;
  const unsigned gone = n < PER ? ~0u << n : 0u;               // positions behind the last
  r.start |= gone;
  r.pad |= gone;
  r.flag &= ~gone;
  return r;
}

// First position at or behind i0 + k that starts a document / that has no flag, within the thread's, else what lies behind.
B200_DEVICE int next_start(const Bits& b, int i0, int k, int behind) {
  const unsigned m = b.start & ((1u << PER) - 1u) & (~0u << k);
  return k < PER && m ? i0 + __ffs(m) - 1 : behind;
}
B200_DEVICE int next_bare(const Bits& b, int i0, int k, int behind) {
  const unsigned m = ~b.flag & ((1u << PER) - 1u) & (~0u << k);
  return m ? i0 + __ffs(m) - 1 : behind;
}

// (start << 32 | end of its prefix) for the start at i0 + k of a thread with `end` and `bare` behind it
B200_DEVICE long long prefix_key(const Bits& b, int i0, int k, int end, int bare) {
  return (long long)(i0 + k) << 32 | (long long)min(next_bare(b, i0, k, bare), next_start(b, i0, k + 1, end));
}

// Exclusive scans over the threads: running minimum from the end (two at once), running maximum from the front.  `carry` is what lies beyond
// the chunk, and becomes what lies beyond the next one.
B200_DEVICE void scan_back(int& a, int& b, int (&carry)[2], int (*red)[NT / 32]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int v[2] = {a, b};
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_down_sync(ALL, v[k], o);
      if (lane + o < 32) v[k] = min(v[k], u);
    }
  __syncthreads();
  if (lane == 0) { red[0][warp] = v[0]; red[1][warp] = v[1]; }
  __syncthreads();
  int out[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    int w = red[k][lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_down_sync(ALL, w, o);
      if (lane + o < 32) w = min(w, u);
    }
    const int whole = __shfl_sync(ALL, w, 0);
    int behind = __shfl_sync(ALL, w, min(warp + 1, 31));
    if (warp == 31) behind = 0x7fffffff;
    int mine = __shfl_down_sync(ALL, v[k], 1);
    if (lane == 31) mine = 0x7fffffff;
    out[k] = min(min(mine, behind), carry[k]);
    carry[k] = min(whole, carry[k]);
  }
  a = out[0];
  b = out[1];
}
B200_DEVICE long long scan_front(long long v, long long& carry, long long* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(ALL, v, o);
    if (lane >= o) v = max(v, u);
  }
  __syncthreads();
  if (lane == 31) red[warp] = v;
  __syncthreads();
  long long w = red[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(ALL, w, o);
    if (lane >= o) w = max(w, u);
  }
  const long long whole = __shfl_sync(ALL, w, 31);
  long long before = __shfl_sync(ALL, w, max(warp - 1, 0));
  if (warp == 0) before = -1;
  long long mine = __shfl_up_sync(ALL, v, 1);
  if (lane == 0) mine = -1;
  const long long out = max(max(mine, before), carry);
  carry = max(whole, carry);
  return out;
}
static_assert(NT == 1024, "a lane for each warp");

// What a tile of rows sees: of those that see something the first and last, and the bounds within which all see all.
struct Tile {
  int lo_min = 0x7fffffff, hi_max = 0, lo_max = 0, hi_min = 0x7fffffff;
  B200_DEVICE void add(int lo, int hi) {
    if (lo < hi) { lo_min = min(lo_min, lo); hi_max = max(hi_max, hi); }
    lo_max = max(lo_max, lo);
    hi_min = min(hi_min, lo < hi ? hi : lo);
  }
  B200_DEVICE void join() {                                   // over the warp
    lo_min = __reduce_min_sync(ALL, lo_min);
    hi_max = __reduce_max_sync(ALL, hi_max);
    lo_max = __reduce_max_sync(ALL, lo_max);
    hi_min = __reduce_min_sync(ALL, hi_min);
  }
  B200_DEVICE int4 entry(bool cut) const {                     // cut: rows of the tile are not there (keys behind the last: always masked)
    int4 o = make_int4(0, 0, lo_max, cut ? 0 : hi_min);
    if (lo_min < hi_max) { o.x = lo_min / 128; o.y = (hi_max + 127) / 128; }
    return o;
  }
};

// Pairs of query tiles or key tiles by what they cost, most first.  A key tile: its query tiles.  A pair: four for each key tile that
// either of its query tiles looks at and one more where both do (128 heads x 8192 keys of 128, a step of one tile 2.05 us and of two 2.63).
// (By the sum of their steps, pairs of one long and one short tile came too late: 8192 x 32 heads, 128 tokens of another document at the end,
// 531 us without them, 634 with.)
B200_DEVICE void order_tiles(const MaskLayout& m, int* buf, bool of_q, int* bins, int* red) {
  const int n = of_q ? m.B * (m.Sp / 256) : m.B * (m.Kp / 128);
  const int4* t = reinterpret_cast<const int4*>(buf + (of_q ? m.qt : m.kt));
  int* out = buf + (of_q ? m.oq : m.ok);
  const int unit = (of_q ? m.Kp : m.Sp) / 16 / BINS + 1;            // (costs reach eight a tile of the other side)
  auto bin = [&](int i) {
    if (!of_q) return BINS - 1 - (t[i].y - t[i].x) / unit;
    const int a0 = t[2 * i].x, e0 = t[2 * i].y & ~b200::UNSEEN, a1 = t[2 * i + 1].x, e1 = t[2 * i + 1].y & ~b200::UNSEEN;
    const int shared = max(min(e0, e1) - max(a0, a1), 0);
    return BINS - 1 - (4 * (e0 - a0 + e1 - a1 - shared) + shared) / unit;
  };
  if (n <= 32) {                                               // a warp: each lane's place is the number of tiles before it
    if (threadIdx.x < 32) {
      const int mine = (int)threadIdx.x < n ? bin((int)threadIdx.x) : BINS;
      int place = 0;
      for (int i = 0; i < n; ++i) {
        const int other = __shfl_sync(ALL, mine, i);
        place += other < mine || (other == mine && i < (int)threadIdx.x) ? 1 : 0;
      }
      if ((int)threadIdx.x < n) out[place] = (int)threadIdx.x;
    }
    return;
  }
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
  int w = red[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(ALL, w, o);
    if (lane >= o) w += u;
  }
  const int before = __shfl_sync(ALL, w, max(warp - 1, 0));
  const int at = x - a - c + (warp > 0 ? before : 0);
  bins[2 * threadIdx.x] = at;
  bins[2 * threadIdx.x + 1] = at + a;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += NT) out[atomicAdd(&bins[bin(i)], 1)] = i;      // (order within a bin: the schedule's alone)
  __syncthreads();
}
static_assert(BINS == 2 * NT, "a thread scans two bins");

__global__ void __launch_bounds__(NT) attn_mask_kernel(const __grid_constant__ MaskParams p) {
  b200::begin_kernel();
  __shared__ int red[2][NT / 32];
  __shared__ int s_any[8];
  __shared__ long long red64[NT / 32];
  __shared__ union {
    int bins[BINS];
    struct { long long cur[NT]; int2 behind[NT]; uint2 bits[NT]; } own;
  } sh;
  long long* s_cur = sh.own.cur;                                      // of each thread: start and prefix before it, what lies behind, its bits
  int2* s_behind = sh.own.behind;
  uint2* s_bits = sh.own.bits;
  const MaskLayout& m = p.m;
  const int part = (int)blockIdx.x % p.parts, b = (int)blockIdx.x / p.parts, S = m.Skv, off = m.Skv - m.Sq, nq = m.Sp / 128, nk = m.Kp / 128;
  const long long base = (long long)b * S;
  int2* q_iv = reinterpret_cast<int2*>(p.buf + m.q_iv) + (long long)b * m.Sp;
  int2* k_iv = reinterpret_cast<int2*>(p.buf + m.k_iv) + (long long)b * m.Kp;
  int4* qt = reinterpret_cast<int4*>(p.buf + m.qt) + (long long)b * nq;
  int4* kt = reinterpret_cast<int4*>(p.buf + m.kt) + (long long)b * nk;
  int2* behind = reinterpret_cast<int2*>(p.buf + m.scratch) + (long long)b * ((S + CHUNK - 1) / CHUNK);   // of chunk c: next start and next position without a flag
  const int chunks = (S + CHUNK - 1) / CHUNK, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool same = off % 128 == 0;                                   // query tiles are key tiles

  if (chunks > 1) {
    int carry[2] = {S, S};
    for (int c = chunks - 1; c >= 0; --c) {
      if (threadIdx.x == 0) behind[c] = make_int2(carry[0], carry[1]);
      const int i0 = c * CHUNK + (int)threadIdx.x * PER;
      const Bits t = load_bits(p, base, i0, S);
      int a = next_start(t, i0, 0, 0x7fffffff), e = next_bare(t, i0, 0, 0x7fffffff);
      scan_back(a, e, carry, red);
    }
    __syncthreads();
  }
  bool unseen = false;                                                // a key of this thread's
  long long front = 0;                                                // (start << 32 | end of its prefix)
  for (int c = 0; c < chunks; ++c) {
    const int i0 = c * CHUNK + (int)threadIdx.x * PER;
    const Bits t = load_bits(p, base, i0, S);
    int carry[2] = {S, S};
    if (chunks > 1) { const int2 v = behind[c]; carry[0] = v.x; carry[1] = v.y; }
    int end = next_start(t, i0, 0, 0x7fffffff), bare = next_bare(t, i0, 0, 0x7fffffff);
    scan_back(end, bare, carry, red);                                 // behind this thread
    end = min(end, S);
    bare = min(bare, S);
    const unsigned starts = t.start & (i0 < S ? (1u << PER) - 1u : 0u);
    const int top = starts ? 31 - __clz(starts) : 0;
    const long long cur = scan_front(starts ? prefix_key(t, i0, top, end, bare) : -1, front, red64);
    // positions to warps: a tile of 128 at a time, so that neighbouring lanes write neighbouring intervals (each thread its own 16 would
    // touch 32 lines a store, which took longer than all else: 7 us more for 16384 positions)
    s_cur[threadIdx.x] = cur;
    s_behind[threadIdx.x] = make_int2(end, bare);
    s_bits[threadIdx.x] = make_uint2((t.start & 0xffffu) | t.pad << 16, t.flag);
    __syncthreads();
    for (int j = (part * (NT / 32) + warp) * 128; j < CHUNK && c * CHUNK + j < S; j += p.parts * (NT / 32) * 128) {
      Tile tk, tq;
#pragma unroll
      for (int part = 0; part < 4; ++part) {
        const int at = j + part * 32 + lane, i = c * CHUNK + at, owner = at / PER, k = at % PER, o0 = i - k;
        if (i >= S) continue;
        const uint2 w = s_bits[owner];
        const int2 next = s_behind[owner];
        const Bits u = {w.x & 0xffffu, w.x >> 16, w.y};
        const unsigned mine = u.start & ((2u << k) - 1u);             // starts at or before this position
        const long long key = mine ? prefix_key(u, o0, 31 - __clz(mine), next.x, next.y) : s_cur[owner];
        const int ds = (int)(key >> 32), de = next_start(u, o0, k + 1, next.x);
        int lo = i, hi = i, first = i, last = i;                      // padding: nothing
        if (!(u.pad >> k & 1u)) {
          const int pe = p.flags != nullptr ? (int)key : ds;
          lo = p.window > 0 ? max(ds, i - p.window + 1) : ds;
          hi = p.causal ? max(i + 1, pe) : de;
          first = (!p.causal || i < pe) ? ds : i;
          last = p.window > 0 && i < de - p.window ? i + p.window : de;
        }
        first = max(first - off, 0);                                  // as queries
        last = max(last - off, 0);
        if (first >= last) first = last = max(i - off, 0);
        k_iv[i] = make_int2(first, last);
        unseen |= first >= last;
        tk.add(first, last);
        if (i >= off) {
          q_iv[i - off] = make_int2(lo, hi);
          tq.add(lo, hi);
        }
      }
      tk.join();
      if (same) tq.join();
      const int i = c * CHUNK + j;
      if (lane == 0) {
        kt[i / 128] = tk.entry(i + 128 > S);
        if (same && i >= off) qt[(i - off) / 128] = tq.entry(false);
      }
    }
    __syncthreads();
  }
  if (part == 0) {
    for (int i = S + (int)threadIdx.x; i < m.Kp; i += NT) k_iv[i] = make_int2(0, 0);
    for (int i = m.Sq + (int)threadIdx.x; i < m.Sp; i += NT) q_iv[i] = make_int2(0, 0);
  }
  const int any = __syncthreads_or(unseen);
  if (p.parts > 1) {
    cluster_sync_all();
    const uint32_t first = cluster_ctarank() - part;           // the sequence's first CTA
    if (threadIdx.x == 0) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(mapa_u32(smem_u32(&s_any[part]), first)), "r"(any) : "memory");
  }
  // query tiles on other positions than key tiles, and behind the last query
  for (int t = (same ? (m.Sq + 127) / 128 : 0) + part * (NT / 32) + warp; t < nq; t += p.parts * (NT / 32)) {
    Tile v;
    for (int r = t * 128 + lane; r < (t + 1) * 128 && r < m.Sq; r += 32) v.add(q_iv[r].x, q_iv[r].y);
    v.join();
    if (lane == 0) qt[t] = v.entry(false);
  }
  bool some = any != 0;
  if (p.parts > 1) {
    cluster_sync_all();
    if (part == 0)
      for (int i = 0; i < p.parts; ++i) some |= s_any[i] != 0;
  } else {
    __syncthreads();
  }
  if (part == 0 && some)
    for (int t = threadIdx.x; t < nq; t += NT) qt[t].y |= b200::UNSEEN;
  if (p.whole) {
    const int ctas = m.B * p.parts;
    if (m.B > 1) cluster_sync_all();
    else __syncthreads();
    if (blockIdx.x == 0) order_tiles(m, p.buf, true, sh.bins, red[0]);
    if ((int)blockIdx.x == (ctas > 1 ? 1 : 0)) order_tiles(m, p.buf, false, sh.bins, red[0]);
  }
}

__global__ void __launch_bounds__(NT) attn_mask_order_kernel(const __grid_constant__ MaskLayout m, int* buf) {
  b200::begin_kernel();
  __shared__ int bins[BINS];
  __shared__ int red[NT / 32];
  order_tiles(m, buf, blockIdx.x == 0, bins, red);
}

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
  MaskParams p = {MaskLayout::of(B, Sq, Skv), ids, flags, ids64, causal, window, buf, 1, 0};
  if ((long long)B * (p.m.Kp / 128) > 0x3fffffff) return b200::fail(942, "attn_mask: %d sequences of %d keys", B, Skv);
  // (a CTA has 32 warps, a tile each; one CTA for 16384 positions 8.9 us in its tiles)
  if (Skv > NT / 32 * 128)
    while (p.parts < 8 && 2ll * p.parts * B <= b200::sm_count()) p.parts *= 2;
  p.whole = (long long)B * p.parts <= 8;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)B * p.parts);
  cfg.blockDim = dim3(NT);
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = p.whole ? B * p.parts : p.parts;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = attr[1].val.clusterDim.x > 1 ? 2 : 1;
  cudaLaunchKernelEx(&cfg, attn_mask_kernel, p);               // (a failure is seen by check_launch)
  b200::count_launch();
  if (!p.whole) {
    b200::launch(attn_mask_order_kernel, 2, NT, 0, (cudaStream_t)stream, p.m, buf);
    b200::count_launch();
  }
  return b200::check_launch("attn_mask");
}
