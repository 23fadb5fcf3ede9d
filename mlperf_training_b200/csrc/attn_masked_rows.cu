// Masked attention of few queries over many keys (the next tokens of a batch of sequences): what counts is reading K and V once.
//
// The query rows of one key head (its group of heads x the queries, 16 at a time) share a CTA's tiles.  A CTA takes a share of the keys that
// any of its rows sees, its four warps take its tiles of 16 keys in turn, each with a ring of its own (TMA, one lane), online softmax
// in registers and m16n8k16 products (padded rows cost nothing that matters beside the loads: 16 keys are 8 KB and 32 instructions at head
// dim 128); they join in shared memory, and where a head's keys are split over several CTAs these join as a cluster or by a second launch.
// Probabilities are exactly 0 where a row does not see a key, their sum is of the rounded ones that are multiplied, and value rows
// that no row sees are cleared before the product.
// 8 tokens over 7400 to 16384 keys each, 8 key heads of 128: 372 MB in 61 us (6.1 TB/s), the join 7.
#include "attn_masked.cuh"

namespace {

constexpr int WARPS = 4, KT = 16, STAGES = 3, ROWS = 16, CLUSTER = 8;

struct RowsParams {
  b200::MaskView mask;
  b200::ScoreParams score;
  const __nv_bfloat16* q;
  long long q_row, q_batch;
  int B, Hq, Hkv, Sq, Skv, splits;
  const float* sink;
  float* lse;               // [B, Hq, Sq]
  __nv_bfloat16* out;       // [B, Sq, Hq, HD]
  int cluster;              // the CTAs of a head's shares are a cluster, and join in its shared memory
  float* part;              // else, splits > 1: [rows][splits][HD], rows = (b * Sq + q) * Hq + h
  float2* part_ml;          // [rows][splits]: maximum (log2) and sum
  int* status;
};

template <int HD>
struct Smem {
  static constexpr int TILE = KT * HD * 2;                     // K or V of a stage
  static constexpr int RING = WARPS * STAGES * 2 * TILE;
  static constexpr int TOTAL = RING + WARPS * STAGES * 8 + 64 + ROWS * 8 + WARPS * ROWS * 8 + 1024;
};

B200_DEVICE void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
B200_DEVICE void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
B200_DEVICE void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 16-byte chunk `ch` of row r of a tile of 64-column blocks, 128-byte swizzle
B200_DEVICE uint32_t chunk(uint32_t tile, int r, int ch) { return tile + (ch >> 3) * (KT * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4); }

B200_DEVICE float2 ld_cluster_f32x2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}
B200_DEVICE float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// A warp's row `at` = (b * Sq + q) * Hq + h from its sum of values, maximum and sum of probabilities (mw, lw).
template <int HD>
B200_DEVICE void finish_row(const RowsParams& p, long long at, float (&acc)[HD / 32], float mw, float lw, int lane) {
  const int h = (int)(at % p.Hq);
  const long long bq = at / p.Hq;
  const bool none = mw == -INFINITY;
  if (p.sink != nullptr) {
    const float sk = p.sink[h] * b200::LOG2E;
    if (none) { mw = sk; lw = 1.f; } else lw += ex2_approx(sk - mw);
  }
  const float inv = none ? 0.f : 1.f / lw;
#pragma unroll
  for (int c = 0; c < HD / 32; ++c) p.out[at * HD + c * 32 + lane] = __float2bfloat16(none ? 0.f : acc[c] * inv);
  if (lane == 0) p.lse[((bq / p.Sq) * p.Hq + h) * p.Sq + bq % p.Sq] = lw > 0.f ? (mw + log2f(lw)) * 0.6931471805599453f : -INFINITY;
}

template <int HD>
__global__ void __launch_bounds__(WARPS * 32, 2)
attn_masked_rows_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ RowsParams p) {
  b200::begin_kernel();
  using SM = Smem<HD>;
  constexpr int NB = HD / 64, KS = HD / 16, ND = HD / 8;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + SM::RING);
  int* abort_flag_ = reinterpret_cast<int*>(bars + WARPS * STAGES);
  volatile int* abort_flag = abort_flag_;
  int2* s_iv = reinterpret_cast<int2*>(abort_flag_ + 16);      // keys of each row
  float2* s_ml = reinterpret_cast<float2*>(s_iv + ROWS);       // [warp][row]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = p.Hq / p.Hkv, rows = group * p.Sq, blocks = (rows + ROWS - 1) / ROWS;
  const int split = blockIdx.x, hk = (int)blockIdx.y / blocks, row0 = ((int)blockIdx.y - hk * blocks) * ROWS, b = blockIdx.z;
  const int off = p.Skv - p.Sq;
  uint64_t* bar = bars + warp * STAGES;
  if (lane == 0) {
    for (int i = 0; i < STAGES; ++i) mbar_init(&bar[i], 1);
    if (warp == 0) *abort_flag = 0;
    mbar_fence_init();
  }
  if (threadIdx.x < ROWS) {
    const int r = row0 + threadIdx.x;
    s_iv[threadIdx.x] = r < rows ? p.mask.q_iv[(long long)b * p.mask.Sp + r / group] : make_int2(0, 0);
  }
  __syncthreads();
  // keys that some row sees, and those that every row sees
  int k_lo = 0x7fffffff, k_hi = 0, all_lo = 0, all_hi = 0x7fffffff;
  {
    const int2 v = s_iv[lane & 15];
    if (v.x < v.y) { k_lo = v.x; k_hi = v.y; }
    k_lo = __reduce_min_sync(0xffffffffu, k_lo);
    k_hi = __reduce_max_sync(0xffffffffu, k_hi);
    const bool there = row0 + (lane & 15) < rows;
    all_lo = __reduce_max_sync(0xffffffffu, there ? v.x : 0);
    all_hi = __reduce_min_sync(0xffffffffu, there ? v.y : 0x7fffffff);
  }
  k_lo = k_lo / KT * KT;
  const int tiles = k_hi > k_lo ? (k_hi - k_lo + KT - 1) / KT : 0;
  const int t0 = (int)((long long)tiles * split / p.splits), t1 = (int)((long long)tiles * (split + 1) / p.splits);
  const int n = t1 - t0 > warp ? (t1 - t0 - warp + WARPS - 1) / WARPS : 0;      // this warp's tiles t0 + warp + i * WARPS

  uint8_t* ring = smem + warp * STAGES * 2 * SM::TILE;
  auto fetch = [&](int i) {                                    // one lane
    uint8_t* dst = ring + (i % STAGES) * 2 * SM::TILE;
    uint64_t* br = &bar[i % STAGES];
    const int key = k_lo + (t0 + warp + i * WARPS) * KT;
    mbar_expect_tx(br, 2 * SM::TILE);
#pragma unroll
    for (int c = 0; c < NB; ++c) {
      b200::load_4d(dst + c * (KT * 128), &tmK, br, c * 64, hk, key, b);
      b200::load_4d(dst + SM::TILE + c * (KT * 128), &tmV, br, c * 64, hk, key, b);
    }
  };
  if (lane == 0)
    for (int i = 0; i < STAGES && i < n; ++i) fetch(i);

  // this lane's rows: lane / 4 and lane / 4 + 8; its query fragments, all of the head dim
  const int ra = lane >> 2, rb = ra + 8;
  uint32_t qf[KS][4];
  float slope[2] = {0.f, 0.f};
  int pos[2] = {0, 0};
  const int2 iv[2] = {s_iv[ra], s_iv[rb]};
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = row0 + (e ? rb : ra);
    const bool there = r < rows;
    const int h = hk * group + (there ? r % group : 0), qi = there ? r / group : 0;
    const __nv_bfloat16* src = p.q + b * p.q_batch + (long long)qi * p.q_row + h * HD + (lane & 3) * 2;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      qf[k][e] = there ? *reinterpret_cast<const uint32_t*>(src + k * 16) : 0u;
      qf[k][e + 2] = there ? *reinterpret_cast<const uint32_t*>(src + k * 16 + 8) : 0u;
    }
    if (p.score.slopes != nullptr && there) slope[e] = p.score.slopes[h] * b200::LOG2E;
    pos[e] = qi + off;
  }

  float o[ND][4];
#pragma unroll
  for (int d = 0; d < ND; ++d) o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  const float scale2 = p.score.scale * b200::LOG2E;
  const bool capped = p.score.cap > 0.f, biased = p.score.slopes != nullptr;
  bool ok = true;
  for (int i = 0; i < n; ++i) {
    const int key = k_lo + (t0 + warp + i * WARPS) * KT;
    const uint32_t tk = smem_u32(ring + (i % STAGES) * 2 * SM::TILE), tv = tk + SM::TILE;
    if (!warp_wait_spin(&bar[i % STAGES], (i / STAGES) & 1, abort_flag, p.status, 110)) { ok = false; break; }
    const bool masked = key < all_lo || key + KT > all_hi;
    if (masked) {
      // value rows that no row of this block sees (behind the keys of any, of another document, padding)
      const int kk = key + (lane & 15);
      bool seen = false;
      for (int r = 0; r < ROWS; ++r) seen |= kk >= s_iv[r].x && kk < s_iv[r].y;
      if (!seen) {
        uint8_t* vr = ring + (i % STAGES) * 2 * SM::TILE + SM::TILE + (lane & 15) * 128 + (lane >> 4) * 64;
#pragma unroll
        for (int c = 0; c < NB; ++c)
#pragma unroll
          for (int g = 0; g < 4; ++g) *reinterpret_cast<uint4*>(vr + c * (KT * 128) + g * 16) = make_uint4(0u, 0u, 0u, 0u);
      }
      __syncwarp();
    }
    // S: rows x 16 keys (two tiles of 8)
    float s[2][4] = {};
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      uint32_t kf[4];                                          // keys 0-7 | 8-15, columns k * 16 + 0-7 | 8-15
      ldsm4(kf, chunk(tk, (lane & 7) + ((lane >> 4) & 1) * 8, k * 2 + ((lane >> 3) & 1)));
      mma(s[0], qf[k], kf[0], kf[1]);
      mma(s[1], qf[k], kf[2], kf[3]);
    }
    float mx[2] = {-INFINITY, -INFINITY};
    if (capped)
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const float2 y = b200::capped_any2(make_float2(s[t][e], s[t][e + 1]), p.score);
          s[t][e] = y.x; s[t][e + 1] = y.y;
        }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int kk = key + t * 8 + (lane & 3) * 2 + (e & 1), w = e >> 1;
        float x = capped ? s[t][e] : s[t][e] * scale2;
        if (biased) x = fmaf(-slope[w], fabsf((float)(kk - pos[w])), x);
        if (masked && (kk < iv[w].x || kk >= iv[w].y)) x = -INFINITY;
        s[t][e] = x;
        mx[w] = fmaxf(mx[w], x);
      }
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      mx[w] = fmaxf(mx[w], __shfl_xor_sync(0xffffffffu, mx[w], 1));
      mx[w] = fmaxf(mx[w], __shfl_xor_sync(0xffffffffu, mx[w], 2));
    }
    if (__any_sync(0xffffffffu, mx[0] > m[0] || mx[1] > m[1])) {
      float f[2];
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const float nm = fmaxf(m[w], mx[w]);
        f[w] = m[w] == -INFINITY ? 0.f : ex2_approx(m[w] - nm);
        m[w] = nm;
        l[w] *= f[w];
      }
#pragma unroll
      for (int d = 0; d < ND; ++d) { o[d][0] *= f[0]; o[d][1] *= f[0]; o[d][2] *= f[1]; o[d][3] *= f[1]; }
    }
    const float base[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};
    uint32_t pf[4];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const uint32_t u = pack_bf16x2(ex2_approx(s[t][2 * w] - base[w]), ex2_approx(s[t][2 * w + 1] - base[w]));
        pf[t * 2 + w] = u;
        l[w] += __uint_as_float(u << 16) + __uint_as_float(u & 0xffff0000u);
      }
#pragma unroll
    for (int d = 0; d < ND / 2; ++d) {
      uint32_t vf[4];                                          // keys 0-7 | 8-15 of columns d * 16 + 0-7, then of 8-15
      ldsm4t(vf, chunk(tv, lane & 15, d * 2 + (lane >> 4)));
      mma(o[2 * d], pf, vf[0], vf[1]);
      mma(o[2 * d + 1], pf, vf[2], vf[3]);
    }
    if (masked) fence_proxy_async_smem();                      // (the cleared rows before the copy that overwrites them)
    __syncwarp();
    if (lane == 0 && i + STAGES < n) fetch(i + STAGES);
  }
  if (!ok) {                                                   // copies that are still in flight
    const uint64_t t = globaltimer_ns();
    while (globaltimer_ns() - t < 200000ull) __nanosleep(1000);
  }
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    l[w] += __shfl_xor_sync(0xffffffffu, l[w], 1);
    l[w] += __shfl_xor_sync(0xffffffffu, l[w], 2);
  }
  // join the warps: each leaves its rows in its own part of shared memory
  float* mine = reinterpret_cast<float*>(ring);                // [ROWS][HD + 4]
  static_assert(ROWS * (HD + 4) * 4 <= STAGES * 2 * SM::TILE, "a warp's ring holds its output rows");
  __syncwarp();
#pragma unroll
  for (int d = 0; d < ND; ++d) {
    const int c = d * 8 + (lane & 3) * 2;
    *reinterpret_cast<float2*>(mine + ra * (HD + 4) + c) = make_float2(o[d][0], o[d][1]);
    *reinterpret_cast<float2*>(mine + rb * (HD + 4) + c) = make_float2(o[d][2], o[d][3]);
  }
  if ((lane & 3) == 0) {
    s_ml[warp * ROWS + ra] = make_float2(m[0], l[0]);
    s_ml[warp * ROWS + rb] = make_float2(m[1], l[1]);
  }
  __syncthreads();
  // a warp a row at a time
  for (int rr = warp; rr < ROWS && row0 + rr < rows; rr += WARPS) {
    float mw = -INFINITY;
    for (int w = 0; w < WARPS; ++w) mw = fmaxf(mw, s_ml[w * ROWS + rr].x);
    float f[WARPS], lw = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float2 v = s_ml[w * ROWS + rr];
      f[w] = v.x == -INFINITY ? 0.f : ex2_approx(v.x - mw);
      lw += v.y * f[w];
    }
    const int r = row0 + rr, h = hk * group + r % group, qi = r / group;
    const long long at = ((long long)b * p.Sq + qi) * p.Hq + h;
    float acc[HD / 32];
#pragma unroll
    for (int c = 0; c < HD / 32; ++c) {
      acc[c] = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w)
        if (f[w] != 0.f) acc[c] += f[w] * reinterpret_cast<const float*>(smem + w * STAGES * 2 * SM::TILE)[rr * (HD + 4) + c * 32 + lane];
    }
    if (p.splits == 1) {
      finish_row<HD>(p, at, acc, mw, lw, lane);
    } else if (p.cluster) {                                    // (in the first warp's part: the row is this warp's alone)
      __syncwarp();                                            // its sums have been read by all lanes
#pragma unroll
      for (int c = 0; c < HD / 32; ++c) reinterpret_cast<float*>(smem)[rr * (HD + 4) + c * 32 + lane] = acc[c];
      if (lane == 0) s_ml[rr] = make_float2(mw, lw);
      __syncwarp();
    } else {
#pragma unroll
      for (int c = 0; c < HD / 32; ++c) p.part[(at * p.splits + split) * HD + c * 32 + lane] = acc[c];
      if (lane == 0) p.part_ml[at * p.splits + split] = make_float2(mw, lw);
    }
  }
  if (p.splits > 1 && p.cluster) {
    cluster_sync_all();
    // the rows in turn to the warps of the cluster
    for (int rr = split * WARPS + warp; rr < ROWS && row0 + rr < rows; rr += p.splits * WARPS) {
      const int r = row0 + rr;
      const float2 ml = lane < p.splits ? ld_cluster_f32x2(mapa_u32(smem_u32(&s_ml[rr]), lane)) : make_float2(-INFINITY, 0.f);
      const float mw = warp_max(ml.x), f = ml.x == -INFINITY ? 0.f : ex2_approx(ml.x - mw), lw = warp_sum(ml.y * f);
      float acc[HD / 32] = {};
      for (int z = 0; z < p.splits; ++z) {
        const float w = __shfl_sync(0xffffffffu, f, z);
        const uint32_t from = mapa_u32(smem_u32(smem) + (rr * (HD + 4) + lane) * 4, z);
#pragma unroll
        for (int c = 0; c < HD / 32; ++c) acc[c] += w * ld_cluster_f32(from + c * 128);
      }
      finish_row<HD>(p, ((long long)b * p.Sq + r / group) * p.Hq + hk * group + r % group, acc, mw, lw, lane);
    }
    cluster_sync_all();                                        // (shared memory stays until it has been read)
  }
}

// A warp joins the parts of a row.
template <int HD>
__global__ void __launch_bounds__(128) attn_masked_join_kernel(const __grid_constant__ RowsParams p) {
  b200::begin_kernel();
  const long long at = (blockIdx.x * 128ll + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (at >= (long long)p.B * p.Sq * p.Hq) return;
  // a lane a part for the weights, then all lanes over the parts' rows (empty ones are 0)
  const float2 ml = lane < p.splits ? p.part_ml[at * p.splits + lane] : make_float2(-INFINITY, 0.f);
  const float mw = warp_max(ml.x);
  const float f = ml.x == -INFINITY ? 0.f : ex2_approx(ml.x - mw);
  const float lw = warp_sum(ml.y * f);
  float acc[HD / 32] = {};
#pragma unroll 8
  for (int z = 0; z < p.splits; ++z) {
    const float w = __shfl_sync(0xffffffffu, f, z);
#pragma unroll
    for (int c = 0; c < HD / 32; ++c) acc[c] += w * p.part[(at * p.splits + z) * HD + c * 32 + lane];
  }
  finish_row<HD>(p, at, acc, mw, lw, lane);
}

// Shares of a head's keys: four CTAs an SM in all at most (two run at once; 8 sequences of 7400 to 16384 keys x 8 key heads at head dim 128: 60.8 us
// with 9 shares, 576 CTAs, and 70 with 10, 640), of 256 keys or more each.
// Where their CTAs all run at once and a head's are at most CLUSTER, these are a cluster that joins them (3000 keys of 8 heads 11.5 -> 10.8 us, and a launch
// less for the host); with more CTAs than that clusters wait for each other's places (2000 keys of 64 heads 18.3 -> 20.2, 32768 of 128 306 -> 323).
struct Splits { int n; bool cluster; };
Splits splits_of(int B, int Sq, int Skv, int Hq, int Hkv) {
  const long long heads = (long long)B * Hkv * (((long long)Hq / Hkv * Sq + ROWS - 1) / ROWS), at_once = b200::sm_count() * 3ll / 2;
  const long long n = 4ll * b200::sm_count() / heads, most = (Skv + 255) / 256;
  Splits s = {(int)(n < most ? n : most), false};
  if (s.n > CLUSTER && s.n < 2 * CLUSTER && heads * CLUSTER <= at_once) s.n = CLUSTER;
  if (s.n < 1) s.n = 1;
  if (s.n > 32) s.n = 32;                            // (a lane of the joining warp for each)
  s.cluster = s.n > 1 && s.n <= CLUSTER && heads * s.n <= at_once;
  return s;
}

template <int HD>
int launch_rows(const CUtensorMap& tk, const CUtensorMap& tv, const RowsParams& p, cudaStream_t stream) {
  using SM = Smem<HD>;
  static bool configured[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!configured[dev & 63]) {
    cudaError_t e = cudaFuncSetAttribute(attn_masked_rows_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, SM::TOTAL);
    if (e != cudaSuccess) {
      cudaGetLastError();  // clear the sticky error before reporting
      return b200::fail(971, "attn_masked_rows: cannot set %d bytes of shared memory: %s", SM::TOTAL, cudaGetErrorString(e));
    }
    configured[dev & 63] = true;
  }
  const int blocks = (p.Hq / p.Hkv * p.Sq + ROWS - 1) / ROWS;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)p.splits, (unsigned)(p.Hkv * blocks), (unsigned)p.B);
  cfg.blockDim = dim3(WARPS * 32);
  cfg.dynamicSmemBytes = SM::TOTAL;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = p.splits;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.cluster ? 2 : 1;
  cudaLaunchKernelEx(&cfg, attn_masked_rows_kernel<HD>, tk, tv, p);      // (a failure is seen by check_launch)
  b200::count_launch();
  int r = b200::check_launch("attn_masked_rows");
  if (r || p.splits == 1 || p.cluster) return r;
  const long long rows = (long long)p.B * p.Sq * p.Hq;
  b200::launch(attn_masked_join_kernel<HD>, (unsigned)((rows * 32 + 127) / 128), 128, 0, stream, p);
  b200::count_launch();
  return b200::check_launch("attn_masked_join");
}

}  // namespace

// Whether a forward pass without a backward one takes the kernel of few rows: up to 64 of them a key head.
B200_API int b200_attn_masked_few_rows(int B, int Sq, int Hq, int Hkv) {
  return b200::sizes_ok(B, Sq, Sq, Hq, Hkv) && B <= 65535 && (long long)(Hq / Hkv) * Sq <= 64 && (long long)Hkv * 4 <= 65535 ? 1 : 0;
}
// bytes of workspace (0: none)
B200_API long long b200_attn_masked_rows_workspace(int B, int Sq, int Skv, int Hq, int Hkv, int HD) {
  if (!b200::sizes_ok(B, Sq, Skv, Hq, Hkv)) return 0;
  const Splits s = splits_of(B, Sq, Skv, Hq, Hkv);
  return s.n > 1 && !s.cluster ? (long long)B * Sq * Hq * s.n * (HD * 4 + 8) : 0;
}

// As b200_attn_masked_fwd, for the calls that b200_attn_masked_few_rows names.
B200_API int b200_attn_masked_rows(const void* q, const void* k, const void* v, void* out, float* lse, const float* sink, const float* slopes,
                                   const int* mask, int B, int Sq, int Skv, int Hq, int Hkv, int HD, long long q_row, long long k_row,
                                   long long v_row, long long q_batch, long long k_batch, long long v_batch, float scale, float cap,
                                   void* workspace, long long workspace_bytes, void* stream) {
  if (HD != 64 && HD != 128) return b200::fail(970, "attn_masked_rows: head dim %d not supported (64 or 128)", HD);
  if (!b200::sizes_ok(B, Sq, Skv, Hq, Hkv) || !b200_attn_masked_few_rows(B, Sq, Hq, Hkv))
    return b200::fail(970, "attn_masked_rows: B=%d, Sq=%d, Skv=%d, Hq=%d, Hkv=%d", B, Sq, Skv, Hq, Hkv);
  if (!(scale > 0.f) || !b200::cap_ok(cap)) return b200::fail(970, "attn_masked_rows: scale %g, cap %g", scale, cap);
  CUtensorMap tk, tv;
  int r;
  if ((r = b200::map_bshd(&tk, k, HD, Hkv, Skv, B, k_row, k_batch, KT))) return r;
  if ((r = b200::map_bshd(&tv, v, HD, Hkv, Skv, B, v_row, v_batch, KT))) return r;
  RowsParams p;
  p.mask = b200::MaskView::of(mask, b200::MaskLayout::of(B, Sq, Skv));
  p.score = b200::ScoreParams::of(scale, cap, slopes);
  p.q = (const __nv_bfloat16*)q; p.q_row = q_row; p.q_batch = q_batch;
  p.B = B; p.Hq = Hq; p.Hkv = Hkv; p.Sq = Sq; p.Skv = Skv;
  const Splits sp = splits_of(B, Sq, Skv, Hq, Hkv);
  p.splits = sp.n;
  p.cluster = sp.cluster;
  p.sink = sink; p.lse = lse; p.out = (__nv_bfloat16*)out;
  p.status = b200::status_ptr();
  const long long rows = (long long)B * Sq * Hq;
  if (p.splits > 1 && !p.cluster && (workspace == nullptr || workspace_bytes < rows * p.splits * (HD * 4 + 8)))
    return b200::fail(972, "attn_masked_rows: a workspace of %lld bytes", workspace_bytes);
  p.part = (float*)workspace;
  p.part_ml = reinterpret_cast<float2*>(p.part + rows * p.splits * HD);
  return HD == 128 ? launch_rows<128>(tk, tv, p, (cudaStream_t)stream) : launch_rows<64>(tk, tv, p, (cudaStream_t)stream);
}
