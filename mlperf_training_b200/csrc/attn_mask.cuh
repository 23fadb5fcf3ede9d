// What a mask of attention is to the kernels: an interval of keys for each query and an interval of queries for each key.
//
// Causal, window, document and prefix masks are all of that form.  With p = q + Skv - Sq the position of query q, a document the run of
// equal ids around a position, [ds, de) its ends, and pe the end of its leading run of flagged positions (ds without flags):
//   keys of query at p     [max(ds, p - window + 1), causal ? max(p + 1, pe) : de)
//   positions that see k   [k < pe or not causal ? ds : k, min(de, k + window))
// and an empty interval at p for a negative id.  Both ends of either never fall as p or k grows, so a tile of rows sees one range of tiles.
#pragma once
#include "common.cuh"

namespace b200 {

// Bit of a query tile's end tile: some key of the sequence is seen by no query.
constexpr int UNSEEN = 1 << 30;

// Offsets, in ints, of the parts of a mask's buffer.
struct MaskLayout {
  int B, Sq, Skv, Sp, Kp;                  // Sp: rows rounded up to a pair of tiles, Kp: keys to a tile
  long long q_iv, k_iv, qt, kt, oq, ok, scratch, total;
  __host__ __device__ static MaskLayout of(int B, int Sq, int Skv) {
    MaskLayout m;
    m.B = B; m.Sq = Sq; m.Skv = Skv;
    m.Sp = (Sq + 255) / 256 * 256;
    m.Kp = (Skv + 127) / 128 * 128;
    const long long b = B;
    m.qt = 0;                              // int4 [B][Sp / 128]: first and end key tile (with UNSEEN), largest first key, smallest end of a row's keys
    m.kt = m.qt + b * (m.Sp / 128) * 4;    // int4 [B][Kp / 128]: the same of a key tile over its queries
    m.q_iv = m.kt + b * (m.Kp / 128) * 4;  // int2 [B][Sp]; empty behind the last query
    m.k_iv = m.q_iv + b * m.Sp * 2;        // int2 [B][Kp]; empty behind the last key
    m.oq = m.k_iv + b * m.Kp * 2;          // int [B * Sp / 256]: b * (Sp / 256) + pair of query tiles, most key tiles first
    m.ok = m.oq + b * (m.Sp / 256);        // int [B * Kp / 128]: b * (Kp / 128) + key tile, most query tiles first
    m.scratch = (m.ok + b * (m.Kp / 128) + 1) / 2 * 2;   // int2 [B][Skv / 16384]: what lies behind each chunk
    m.total = m.scratch + b * ((Skv + 16383) / 16384) * 2;
    return m;
  }
};

// The parts that the attention kernels read.
struct MaskView {
  const int4 *qt, *kt;
  const int2 *q_iv, *k_iv;
  const int *oq, *ok;
  int Sp, Kp;
  static MaskView of(const int* buf, const MaskLayout& m) {
    MaskView v;
    v.qt = reinterpret_cast<const int4*>(buf + m.qt); v.kt = reinterpret_cast<const int4*>(buf + m.kt);
    v.q_iv = reinterpret_cast<const int2*>(buf + m.q_iv); v.k_iv = reinterpret_cast<const int2*>(buf + m.k_iv);
    v.oq = buf + m.oq; v.ok = buf + m.ok;
    v.Sp = m.Sp; v.Kp = m.Kp;
    return v;
  }
};

}  // namespace b200
