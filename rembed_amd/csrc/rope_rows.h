// rope_rows.h — rows of heads normed and turned by a workgroup: the body of rope.hip's kernel,
// and of the workgroups of the rotary append (cache.hip) that write q's rows.
#pragma once

#include "rowops.h"

#include <algorithm>
#include <type_traits>

namespace rh {

constexpr int kRopeThreads = 256;
constexpr int kRopeItems = 4;    // the most heads of a thread, whose loads are in flight together
// Cosines and sines that a workgroup holds, of heads of dh: sixteen rows', so that few large heads
// (a row of 4 heads of 256 is 16 threads) leave no threads without a row.
__host__ __device__ constexpr int rope_pairs(int dh) { return 8 * dh; }
// Floats of LDS: those, and q's and k's norm weights.
__host__ __device__ constexpr int rope_lds(int dh) { return 2 * rope_pairs(dh) + 2 * dh; }

__device__ __forceinline__ int rope_used(const RopeArgs& p) {
  return p.used ? min(*p.used, p.rows) : p.rows;
}

// Head h of a row, over q's, k's and the copied v's: its columns, and which of the three it is.
struct RopeHead {
  int in, out, part;
  __device__ __forceinline__ RopeHead(const RopeArgs& p, int h, int dh) {
    part = h < p.heads ? 0 : h < p.heads + p.kv_heads ? 1 : 2;
    const int i = part == 0 ? h : part == 1 ? h - p.heads : h - p.heads - p.kv_heads;
    in = (part == 0 ? p.q_off : part == 1 ? p.k_off : p.v_off) + i * dh;
    out = (part == 0 ? p.q_out : part == 1 ? p.k_out : p.v_out) + i * dh;
  }
};

// How rows are given to workgroups: `sets` threads' heads a row, kRopeItems or one each; a workgroup
// has `group` rows, of each one of `slices` ranges of `each` sets.
struct RopeShare {
  int many, sets, each, slices, group;
  int first;  // row of the first workgroup
  long long blocks(int rows) const { return (rows + (group - 1LL)) / group * slices; }
};
// Four heads a thread, whose cosines it then reads once and whose loads are in flight together, where
// two workgroups a CU remain (16384 rows of 24 heads of 128: 36.8 µs, with one head a thread 42.2;
// begun at half as many rows, 2000 take 7.5 for 6.0, at twice as many 3000 take 9.0 for 9.2 and 1500
// in fp32 8.5 for 8.1), counted with the lanes that hold no values (heads of 80 have some in five of
// eight, so they begin at five eighths of the work); as many rows as fill the workgroup's threads and as far as their cosines
// fit, and slices of one size where a row is more than a workgroup.
inline RopeShare rope_share(const RopeArgs& a, int lanes, int most_dh, int threads) {
  const long long nh = std::max(1LL, (long long)a.heads + a.kv_heads + a.v_heads);
  RopeShare s;
  s.many = nh * lanes * a.rows >= kRopeItems * 512LL * kRopeThreads;
  s.sets = (int)(s.many ? (nh + kRopeItems - 1) / kRopeItems : nh);
  s.slices = (s.sets - 1) / (threads / lanes) + 1;
  s.each = (s.sets - 1) / s.slices + 1;  // slices of one size
  s.group = std::max(1, std::min(threads / (s.each * lanes), rope_pairs(most_dh) / a.turn.pairs));
  s.group = std::min(s.group, a.rows / 512 + 1);
  s.first = 0;
  return s;
}

// What lane l of a head has: two runs of P values, beside the other lanes' (so that a store takes
// whole lines), and the cosines of their pairs.
//   halves: P pairs (a + i, b + i), with P cosines from l P; behind the pairs that turn, the
//           first and the second half of the rest;
//   pairs:  the first and the second half of the head, P / 2 pairs each, with P / 2 cosines.
template <int P>
struct RopeLane {
  int a, b;
  bool turns, second;  // the first run (and with it b's of halves), b's pairs
  __device__ __forceinline__ RopeLane(const RopeTurn& t, int l, int dh) {
    if (t.halves) {
      const int chunks = t.pairs / P, rest = (dh - 2 * t.pairs) / 2;
      turns = l < chunks;
      second = false;
      a = turns ? l * P : 2 * t.pairs + (l - chunks) * P;
      b = a + (turns ? t.pairs : rest);
    } else {
      a = l * P;
      b = a + dh / 2;
      turns = a < 2 * t.pairs;
      second = b < 2 * t.pairs;
    }
  }
};

// P values of a row as loaded. ANY: of any alignment, else 16 bytes.
template <int P, bool BF16, bool ANY>
struct RopeRun {
  using S = std::conditional_t<BF16, __bf16, float>;
  typedef S W __attribute__((ext_vector_type(P), aligned(ANY ? sizeof(S) : 16)));
  W raw;
  __device__ __forceinline__ void load(const S* p) { raw = *reinterpret_cast<const W*>(p); }
  __device__ __forceinline__ void widen(float (&v)[P]) const {
#pragma unroll
    for (int i = 0; i < P; i++) v[i] = (float)raw[i];
  }
};
template <int P, bool BF16, bool ANY>
__device__ __forceinline__ void store_run(void* base, size_t at, const float (&v)[P]) {
  if constexpr (!ANY) {
    store_values<P, BF16>(base, at, v);
  } else {
    using S = std::conditional_t<BF16, __bf16, float>;
    typedef S W __attribute__((ext_vector_type(P), aligned(sizeof(S))));
    W x;
#pragma unroll
    for (int i = 0; i < P; i++) x[i] = (S)v[i];
    __builtin_nontemporal_store(x, reinterpret_cast<W*>(static_cast<S*>(base) + at));
  }
}

// A lane takes P pairs of a head, LPH lanes a head; a thread ITEMS heads of a row. The rows'
// cosines and sines are in LDS once for all heads. ANY: heads of up to LPH * 2 P values and rows of
// any alignment; else heads of so many, and a lane's halves are 16 bytes each. lds:
// rope_lds(LPH * 2 * P) floats, 16-byte aligned.
template <int LPH, int P, bool XB, bool OB, int ITEMS, bool ANY = false, int THREADS = kRopeThreads>
__device__ __forceinline__ void rope_rows(const RopeArgs& p, const RopeShare& share, unsigned block,
                                          float* lds) {
  static_assert(ANY || P == (XB ? 8 : 4), "16 bytes");
  const int DH = ANY ? p.dh : LPH * 2 * P;
  constexpr int kPairs = rope_pairs(LPH * 2 * P);
  float *s_cos = lds, *s_sin = lds + kPairs, *s_w = lds + 2 * kPairs;
  const int tid = threadIdx.x, l = tid % LPH;
  const int nh = p.heads + p.kv_heads + p.v_heads, pairs = p.turn.pairs;
  const int used = rope_used(p);
  const int r0 = share.first + (int)(block / share.slices) * share.group;
  const int nr = min(share.group, used - r0);
  if (nr <= 0) return;
  const bool in = !ANY || l * 2 * P < DH;
  const RopeLane<P> at(p.turn, in ? l : 0, DH);
  // the thread's row of these, and its heads set, set + sets, ..
  const int unit = tid / LPH, row = unit / share.each;
  const int set = (int)(block % share.slices) * share.each + unit - row * share.each;
  const bool mine = row < nr && set < share.sets;
  using S = std::conditional_t<XB, __bf16, float>;
  const S* x = static_cast<const S*>(p.x) + (size_t)(r0 + min(row, nr - 1)) * p.ldx;
  RopeRun<P, XB, ANY> a[ITEMS], b[ITEMS];
#pragma unroll
  for (int k = 0; k < ITEMS; k++) {  // behind the last head: that one, not used
    const int from = RopeHead(p, min(set + k * share.sets, nh - 1), DH).in;
    a[k].load(x + from + at.a);
    b[k].load(x + from + at.b);
  }
  if (p.q_norm.on || p.k_norm.on)
    for (int i = tid; i < 2 * DH; i += THREADS) {
      const bool q = i < DH;
      const float* w = q ? p.q_norm.weight : p.k_norm.weight;
      s_w[i] = w ? w[q ? i : i - DH] : 1.0f;
    }
  for (int i = tid; i < nr * pairs; i += THREADS) {
    const int t = i / pairs;
    turn_cos_sin(turn_at(p.turn.freq[i - t * pairs], p.pos[r0 + t]), p.turn.amp, s_cos[i], s_sin[i]);
  }
  __syncthreads();
  if (!mine) return;
  float c[P], s[P];
  const float *cos = s_cos + row * pairs, *sin = s_sin + row * pairs;
  if (p.turn.halves) {
    if (at.turns) {
      load_floats<P>(cos + at.a, c);
      load_floats<P>(sin + at.a, s);
    }
  } else {
    if (at.turns) {
      load_floats<P / 2>(cos + at.a / 2, c);
      load_floats<P / 2>(sin + at.a / 2, s);
    }
    if (at.second) {
      load_floats<P / 2>(cos + at.b / 2, c + P / 2);
      load_floats<P / 2>(sin + at.b / 2, s + P / 2);
    }
  }
#pragma unroll
  for (int k = 0; k < ITEMS; k++) {
    const int h = set + k * share.sets;
    if (h >= nh) return;
    const RopeHead head(p, h, DH);
    const HeadNorm& norm = head.part == 0 ? p.q_norm : p.k_norm;
    float y[P], z[P];
    a[k].widen(y);
    b[k].widen(z);
    if (head.part < 2 && norm.on) {
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < P; i++) ss = __builtin_fmaf(y[i], y[i], __builtin_fmaf(z[i], z[i], ss));
      if (!in) ss = 0.0f;
      const float inv = inverse_root(group_sum<LPH>(ss) / (float)DH + norm.eps);
      float w[P];
      load_floats<P>(s_w + (head.part ? DH : 0) + at.a, w);
#pragma unroll
      for (int i = 0; i < P; i++) y[i] = y[i] * inv * w[i];
      load_floats<P>(s_w + (head.part ? DH : 0) + at.b, w);
#pragma unroll
      for (int i = 0; i < P; i++) z[i] = z[i] * inv * w[i];
    }
    if (head.part < 2 && at.turns) {
      if (p.turn.halves) {
        turn_halves<P>(y, z, c, s);
      } else {
        turn_pairs<P>(y, c, s);
        if (at.second) turn_pairs<P>(z, c + P / 2, s + P / 2);
      }
    }
    if (in) {
      const size_t to = (size_t)(r0 + row) * p.ldout + head.out;
      store_run<P, OB, ANY>(p.out, to + at.a, y);
      store_run<P, OB, ANY>(p.out, to + at.b, z);
    }
  }
}

}  // namespace rh
