// Micro-scaled quantisation of values in registers: blocks of 32 values with one UE8M0 scale, elements e4m3 (8 bits) or e2m1 (4 bits,
// two per byte, the even element in the low half).
//
// Scale: the smallest power of two s with amax / s <= vmax (448 = 1.75 * 2^8, 6 = 1.5 * 2^2), biased by 127; at least 1 (2^-126) where amax
// is not zero, 0 where it is.  255 (NaN) for a block that holds an infinity or a NaN: e2m1 has neither, and with any other scale the value
// would come back as an ordinary number.  No element saturates: amax / s <= vmax.
// Magnitudes are compared by the maximum that hands a NaN on, and as integers (a NaN's bits are above infinity's, both above every number's).
#pragma once
#include <cuda_fp8.h>

#include "common.cuh"

namespace mxq {

enum Fmt : int { E4M3 = 0, E2M1 = 1 };

template <int FMT>
B200_DEVICE uint32_t e8m0(uint32_t amax_bits) {
  // exponent of amax less that of vmax, one more where the fraction exceeds vmax's (the addition carries)
  const int e = (int)((amax_bits + (FMT == E2M1 ? 0x3fffffu : 0x1fffffu)) >> 23) - (FMT == E2M1 ? 2 : 8);
  return amax_bits >= 0x7f800000u ? 255u : amax_bits == 0u ? 0u : (uint32_t)max(e, 1);
}
// 2^(127 - e) for e <= 253 (no finite block has more)
B200_DEVICE float inv_scale(uint32_t e) { return __uint_as_float((254u - min(e, 254u)) << 23); }
B200_DEVICE uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

B200_DEVICE uint32_t pack4_e4m3(float a, float b, float c, float d) {
  const __nv_fp8x2_storage_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const __nv_fp8x2_storage_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return (uint32_t)lo | ((uint32_t)hi << 16);
}
// eight values to eight e2m1 codes, round to nearest even
B200_DEVICE uint32_t pack8_e2m1(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}
// y (|y| <= 6) to a value of e2m1: |y| / quantum + (u + 1/2) / 256 rounded down, u a random byte.  The expectation over u is y to within
// 1/512 of a quantum, and a value of the format stays as it is.
// y comes times 2^-126, which puts the smallest normal number of the format, 1, on the smallest one of fp32: e2m1's quantum is then the upper
// bit of the fraction in both formats' normal and subnormal numbers alike, and the rounding is an integer addition below that bit and a mask (a
// carry out of the fraction is the next power of two).  Seven instructions an element less than with floor, whose conversions run at a
// quarter of the rate.  Returns the value times 2^-126.  `u` is the word that holds the byte, `at` the byte's place in it.
constexpr float STOCH_DOWN = 1.17549435e-38f, STOCH_UP = 8.50705917e37f;      // 2^-126, 2^126
B200_DEVICE float round_stochastic(float y, uint32_t u, int at) {
  const uint32_t n = __byte_perm(u, 0x80u, 0x5504 | at << 4);                  // 256 u + 128
  return __uint_as_float((__float_as_uint(y) + n * 64u) & 0x81c00000u);
}
// eight of them to codes
B200_DEVICE uint32_t pack8_e2m1_stochastic(const float2 (&y)[4], uint32_t u0, uint32_t u1) {
  const float2 dn = make_float2(STOCH_DOWN, STOCH_DOWN), up = make_float2(STOCH_UP, STOCH_UP);
  float v[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 d = fmul2(y[i], dn);
    const uint32_t u = i < 2 ? u0 : u1;
    const float2 r = fmul2(make_float2(round_stochastic(d.x, u, 2 * (i & 1)), round_stochastic(d.y, u, 2 * (i & 1) + 1)), up);
    v[2 * i] = r.x;
    v[2 * i + 1] = r.y;
  }
  return pack8_e2m1(v);
}

// byte offset of scale (row r of the operand, scale column kc) in the atom layout the block-scaled GEMMs read (quant_mxfp8.cu)
B200_DEVICE long long sf_offset(long long r, int kc, int tile_rows, int atoms_per_tile, long long k_groups) {
  const long long tile = r / tile_rows;
  const int rr = (int)(r - tile * tile_rows);
  const int atom = rr >> 7, ra = rr & 127;
  return ((tile * k_groups + (kc >> 2)) * atoms_per_tile + atom) * 512 + (ra & 31) * 16 + (ra >> 5) * 4 + (kc & 3);
}

// max(m, |a|, |b|), a NaN handed on
B200_DEVICE float fmax3_nan(float m, float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(m), "f"(fabsf(a)), "f"(fabsf(b)));
  return y;
}
// Largest magnitude of bf16 pairs, halves by themselves; a NaN is handed on.
B200_DEVICE uint32_t amax2(uint32_t m, uint32_t pair) {
  const __nv_bfloat162 r = __hmax2_nan(*reinterpret_cast<__nv_bfloat162*>(&m), __habs2(*reinterpret_cast<__nv_bfloat162*>(&pair)));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// Eight values of a 32-block whose other values are in the three neighbouring lanes (lane / 4 is the block): codes in q, returns the scale
// byte.  From fp32 values to e4m3, and from bf16 as they are (magnitudes compared and values scaled in pairs) to e2m1; noise: eight random
// bytes, null for round to nearest.
// (e4m3: the values are z * s, s the same for the block.  s and the scale are not multiplied into one factor: that overflows for small blocks.)
B200_DEVICE uint32_t quant_row8_e4m3(const float2 (&z)[4], float s, uint2& q) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) m = fmax3_nan(m, z[i].x, z[i].y);
  m = fmax_nan(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = fmax_nan(m, __shfl_xor_sync(0xffffffffu, m, 2));
  const uint32_t e = e8m0<E4M3>(abs_bits(m * s));
  const float inv = inv_scale(e);
  const float2 s2 = make_float2(s, s), i2 = make_float2(inv, inv);
  const float2 a = fmul2(fmul2(z[0], s2), i2), b = fmul2(fmul2(z[1], s2), i2), c = fmul2(fmul2(z[2], s2), i2), d = fmul2(fmul2(z[3], s2), i2);
  q = make_uint2(pack4_e4m3(a.x, a.y, b.x, b.y), pack4_e4m3(c.x, c.y, d.x, d.y));
  return e;
}
B200_DEVICE uint32_t quant_row8_e2m1(const uint4& v, const uint2* noise, uint32_t& q) {
  uint32_t m = amax2(amax2(amax2(amax2(0u, v.x), v.y), v.z), v.w);
  m = amax2(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = amax2(m, __shfl_xor_sync(0xffffffffu, m, 2));
  const uint32_t e = e8m0<E2M1>(max(m << 16, m & 0xffff0000u));
  const float inv = inv_scale(e);
  const float2 i2 = make_float2(inv, inv);
  const float2 y[4] = {fmul2(unpack_bf16x2(v.x), i2), fmul2(unpack_bf16x2(v.y), i2), fmul2(unpack_bf16x2(v.z), i2),
                       fmul2(unpack_bf16x2(v.w), i2)};
  if (noise != nullptr) {
    q = pack8_e2m1_stochastic(y, noise->x, noise->y);
  } else {
    const float f[8] = {y[0].x, y[0].y, y[1].x, y[1].y, y[2].x, y[2].y, y[3].x, y[3].y};
    q = pack8_e2m1(f);
  }
  return e;
}

// v <- H v / 4, H[i][j] = (-1)^popcount(i & j), of two columns at a time: four steps of sums and differences in fp32 (divided first, so that
// no sum overflows that would not in the end).
B200_DEVICE void hadamard16(float2 (&v)[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = fmul2(v[i], make_float2(0.25f, 0.25f));
#pragma unroll
  for (int s = 1; s < 16; s <<= 1)
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if ((i & s) == 0) {
        const float2 a = v[i], b = v[i | s];
        v[i] = fadd2(a, b);
        v[i | s] = ffma2(b, make_float2(-1.f, -1.f), a);
      }
}

// Sixteen rows of two columns; the other halves of the 32-blocks are in the neighbouring lane.  `m`: the bits of the largest magnitudes of the
// two (this lane's rows).  noise: word i holds the bytes of rows 4 i .. 4 i + 3 (na: first column, nb: second), null for nearest.  Codes in
// qa, qb (e4m3: 16 bytes, e2m1: two words), scale bytes in ea, eb.
template <int FMT>
B200_DEVICE void quant_col16(float2 (&v)[16], uint32_t ma, uint32_t mb, const uint32_t* na, const uint32_t* nb, uint4& qa, uint4& qb,
                             uint32_t& ea, uint32_t& eb) {
  ma = max(ma, __shfl_xor_sync(0xffffffffu, ma, 1));
  mb = max(mb, __shfl_xor_sync(0xffffffffu, mb, 1));
  ea = e8m0<FMT>(ma);
  eb = e8m0<FMT>(mb);
  const float2 inv = make_float2(inv_scale(ea), inv_scale(eb));
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = fmul2(v[i], inv);
  uint32_t a[4], b[4];
  if constexpr (FMT == E4M3) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[i] = pack4_e4m3(v[4 * i].x, v[4 * i + 1].x, v[4 * i + 2].x, v[4 * i + 3].x);
      b[i] = pack4_e4m3(v[4 * i].y, v[4 * i + 1].y, v[4 * i + 2].y, v[4 * i + 3].y);
    }
  } else {
    a[2] = a[3] = b[2] = b[3] = 0u;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float2* w = v + 8 * h;
      if (na != nullptr) {
        const float2 x[4] = {make_float2(w[0].x, w[1].x), make_float2(w[2].x, w[3].x), make_float2(w[4].x, w[5].x), make_float2(w[6].x, w[7].x)};
        const float2 y[4] = {make_float2(w[0].y, w[1].y), make_float2(w[2].y, w[3].y), make_float2(w[4].y, w[5].y), make_float2(w[6].y, w[7].y)};
        a[h] = pack8_e2m1_stochastic(x, na[2 * h], na[2 * h + 1]);
        b[h] = pack8_e2m1_stochastic(y, nb[2 * h], nb[2 * h + 1]);
      } else {
        const float x[8] = {w[0].x, w[1].x, w[2].x, w[3].x, w[4].x, w[5].x, w[6].x, w[7].x};
        const float y[8] = {w[0].y, w[1].y, w[2].y, w[3].y, w[4].y, w[5].y, w[6].y, w[7].y};
        a[h] = pack8_e2m1(x);
        b[h] = pack8_e2m1(y);
      }
    }
  }
  qa = make_uint4(a[0], a[1], a[2], a[3]);
  qb = make_uint4(b[0], b[1], b[2], b[3]);
}

// ----------------------------------------------------------------------------------
// 128 x 128 tile to e2m1: rows pass and columns pass
// ----------------------------------------------------------------------------------
struct TileArgs {
  const __nv_bfloat16* x;         // [R, C], pitch ldx
  long long ldx;
  int R, C;
  const uint8_t* noise;           // [R, C] dense, or null
  uint8_t* q_row; uint8_t* sf_row; int row_tile;
  uint8_t* q_col; uint8_t* sf_col; int col_tile;
  int Rp;                         // rows of the column copy's contraction: R filled up with zeros
};

constexpr int TILE = 128;
// Shared tile of bf16 pairs: rows at a pitch of 68 words, 4 words more every 16 rows, so that the eight lanes of a column, 16 rows apart, lie
// 4 banks apart (quant_mxfp8.cu).  Bytes of noise: rows at a pitch of 34 words, 2 more every 16 rows.
constexpr int PITCH_W = 68, TILE_WORDS = TILE * PITCH_W + 8 * 4;
constexpr int NPITCH_W = 34, NOISE_WORDS = TILE * NPITCH_W + 8 * 2;
B200_DEVICE int tile_off(int r) { return r * PITCH_W + (r >> 4) * 4; }
B200_DEVICE int noise_off(int r) { return r * NPITCH_W + (r >> 4) * 2; }

// The tile goes through shared memory once, so that both copies come from one reading.  Bound by instructions where both are made (about nine
// an element and copy: comparing, scaling, converting, packing; stochastic rounding six more, the transform three), by memory for the row copy alone.
//
// grid (ceil(C / 128), ceil(R / 128)), 256 threads.  C is a multiple of 32; rows past R and columns past C read as zero and are not written,
// but for the zero codes and scale bytes that fill the copies' last 32 rows and last scale word: an operand read by a GEMM holds no byte
// inside its contraction that was not written here.
template <bool NOISE, bool HAD>
__global__ void __launch_bounds__(256)
mx_tile_kernel(const TileArgs p) {
  b200::begin_kernel();
  __shared__ __align__(16) uint32_t tile[TILE_WORDS];
  extern __shared__ __align__(16) uint32_t noise_s[];     // NOISE: NOISE_WORDS
  __shared__ __align__(4) uint8_t sfs[2][TILE][4];
  const int c0 = blockIdx.x * TILE;
  const long long r0 = (long long)blockIdx.y * TILE;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int sub_row = lane >> 4, chunk = lane & 15;
  const bool col_live = c0 + chunk * 8 < p.C;
  const bool rows = p.q_row != nullptr, cols = p.q_col != nullptr;
  const int row_lim = (int)min((long long)TILE, p.R - r0);            // rows of this tile
  // (addresses advance by sixteen rows; a multiplication and a 64-bit comparison a vector were a fifth of the instructions)
  const int t0 = warp * 2 + sub_row;
  const __nv_bfloat16* src = p.x + (r0 + t0) * p.ldx + c0 + chunk * 8;
  const uint8_t* nsrc = NOISE ? p.noise + (r0 + t0) * p.C + c0 + chunk * 8 : nullptr;
  uint8_t* qdst = rows ? p.q_row + (((r0 + t0) * p.C + c0) >> 1) + chunk * 4 : nullptr;
  const long long step = 16 * p.ldx, nstep = 16ll * p.C, qstep = 8ll * p.C;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint4 xv[4];
    uint2 nv[NOISE ? 4 : 1];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool live = col_live && (h * 4 + i) * 16 + t0 < row_lim;
      xv[i] = live ? *reinterpret_cast<const uint4*>(src) : make_uint4(0u, 0u, 0u, 0u);
      src += step;
      if constexpr (NOISE) {
        nv[i] = live ? *reinterpret_cast<const uint2*>(nsrc) : make_uint2(0x80808080u, 0x80808080u);
        nsrc += nstep;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = (h * 4 + i) * 16 + warp * 2 + sub_row;
      if (rows) {
        uint32_t q;
        const uint32_t e = quant_row8_e2m1(xv[i], NOISE ? &nv[NOISE ? i : 0] : nullptr, q);
        if (col_live && r < row_lim) *reinterpret_cast<uint32_t*>(qdst) = q;
        qdst += qstep;
        if ((chunk & 3) == 0) sfs[0][r][chunk >> 2] = (uint8_t)e;
      }
      if (cols) {
        *reinterpret_cast<uint4*>(tile + tile_off(r) + chunk * 4) = xv[i];
        if constexpr (NOISE) *reinterpret_cast<uint2*>(noise_s + noise_off(r) + chunk * 2) = nv[i];
      }
    }
  }
  __syncthreads();
  if (rows && tid < row_lim) {
    const long long o = sf_offset(r0 + tid, c0 >> 5, p.row_tile, (p.row_tile + 127) >> 7, (p.C + 127) >> 7);
    *reinterpret_cast<uint32_t*>(p.sf_row + o) = *reinterpret_cast<const uint32_t*>(&sfs[0][tid][0]);
  }
  if (!cols) return;
  const int sub = lane & 7;                      // rows sub * 16 .. + 15 of two columns
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    const int cw = pass * 32 + warp * 4 + (lane >> 3), c = 2 * cw;
    uint32_t na[NOISE ? 4 : 1], nb[NOISE ? 4 : 1];
    if constexpr (NOISE) {
      // bytes of the two columns, row by row, turned into words of four rows each
      const uint16_t* n = reinterpret_cast<const uint16_t*>(noise_s + noise_off(sub * 16)) + cw;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t u01 = __byte_perm(n[(4 * i) * NPITCH_W * 2], n[(4 * i + 1) * NPITCH_W * 2], 0x5140);
        const uint32_t u23 = __byte_perm(n[(4 * i + 2) * NPITCH_W * 2], n[(4 * i + 3) * NPITCH_W * 2], 0x5140);
        na[i] = __byte_perm(u01, u23, 0x5410);
        nb[i] = __byte_perm(u01, u23, 0x7632);
      }
    }
    float2 v[16];
    uint32_t ma = 0u, mb = 0u;
    const uint32_t* t = tile + tile_off(sub * 16) + cw;
    if constexpr (!HAD) {
      uint32_t m = 0u;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint32_t u = t[i * PITCH_W];
        m = amax2(m, u);
        v[i] = unpack_bf16x2(u);
      }
      ma = m << 16;
      mb = m & 0xffff0000u;
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = unpack_bf16x2(t[i * PITCH_W]);
      hadamard16(v);
      float fa = 0.f, fb = 0.f;
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        fa = fmax3_nan(fa, v[i].x, v[i + 1].x);
        fb = fmax3_nan(fb, v[i].y, v[i + 1].y);
      }
      ma = abs_bits(fa);
      mb = abs_bits(fb);
    }
    uint4 qa, qb;
    uint32_t ea, eb;
    quant_col16<E2M1>(v, ma, mb, NOISE ? na : nullptr, NOISE ? nb : nullptr, qa, qb, ea, eb);
    if (c0 + c < p.C && r0 + sub * 16 < p.Rp) {
      uint8_t* dst = p.q_col + (((long long)(c0 + c) * p.Rp + r0) >> 1) + sub * 8;
      *reinterpret_cast<uint2*>(dst) = make_uint2(qa.x, qa.y);
      *reinterpret_cast<uint2*>(dst + (p.Rp >> 1)) = make_uint2(qb.x, qb.y);
    }
    if ((sub & 1) == 0) { sfs[1][c][sub >> 1] = (uint8_t)ea; sfs[1][c + 1][sub >> 1] = (uint8_t)eb; }
  }
  __syncthreads();
  if (tid < TILE && c0 + tid < p.C) {
    const long long o = sf_offset(c0 + tid, (int)(r0 >> 5), p.col_tile, (p.col_tile + 127) >> 7, (p.Rp + 127) >> 7);
    *reinterpret_cast<uint32_t*>(p.sf_col + o) = *reinterpret_cast<const uint32_t*>(&sfs[1][tid][0]);
  }
}

}  // namespace mxq
