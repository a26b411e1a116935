// rope_rows.h — rows of heads normed and turned by a workgroup: the body of rope.hip's kernel,
// and of the workgroups of the rotary append (cache.hip) that write q's rows.
#pragma once

#include "rowops.h"

#include <algorithm>

namespace rh {

constexpr int kRopeThreads = 256;
constexpr int kRopeItems = 4;    // heads' chunks of a thread whose loads are in flight together
constexpr int kRopePairs = 512;  // cosines and sines that a workgroup holds

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

// Rows of a workgroup: kRopeItems chunks for each thread where there are rows enough for two
// workgroups a CU, as far as their cosines fit.
inline int rope_group(const RopeArgs& a, int lanes) {
  const long long nh = (long long)a.heads + a.kv_heads + a.v_heads;
  long long g = kRopeThreads * kRopeItems / std::max(1LL, nh * lanes);
  g = std::min(g, (long long)kRopePairs / a.turn.pairs);
  g = std::min(g, ((long long)a.rows + 511) / 512);
  return (int)std::max(1LL, g);
}

// A lane takes P pairs of a head, LPH lanes a head; a workgroup `group` rows at a time, whose
// cosines and sines it puts into LDS once for all heads. lds: 2 * kRopePairs + 4 * LPH * P floats.
template <int LPH, int P, bool XB, bool OB>
__device__ __forceinline__ void rope_rows(const RopeArgs& p, int group, unsigned block,
                                          unsigned blocks, float* lds) {
  constexpr int DH = LPH * 2 * P;
  float *s_cos = lds, *s_sin = lds + kRopePairs, *s_w = lds + 2 * kRopePairs;
  const int tid = threadIdx.x, l = tid % LPH;
  const int nh = p.heads + p.kv_heads + p.v_heads, pairs = p.turn.pairs;
  const int used = rope_used(p);
  const RopePlace<P> at(p.turn, l);
  for (int i = tid; i < 2 * DH; i += kRopeThreads) {
    const float* w = i < DH ? p.q_norm.weight : p.k_norm.weight;
    s_w[i] = w ? w[i % DH] : 1.0f;
  }
  for (long long r0 = (long long)block * group; r0 < used; r0 += (long long)blocks * group) {
    const int nr = min(group, used - (int)r0);
    const unsigned slots = (unsigned)nr * nh;  // heads of these rows
    float a[kRopeItems][P], b[kRopeItems][P];
    auto load = [&](unsigned base) {
#pragma unroll
      for (int k = 0; k < kRopeItems; k++) {
        const unsigned slot = base + (tid + k * kRopeThreads) / LPH;
#pragma unroll
        for (int i = 0; i < P; i++) a[k][i] = b[k][i] = 0.0f;
        if (slot < slots) {
          const unsigned row = slot / (unsigned)nh;
          const RopeHead h(p, (int)(slot - row * nh), DH);
          const size_t from = (size_t)(r0 + row) * p.ldx + h.in;
          load_values<P, XB>(p.x, from + at.a, a[k]);
          load_values<P, XB>(p.x, from + at.b, b[k]);
        }
      }
    };
    load(0);
    for (int i = tid; i < nr * pairs; i += kRopeThreads) {
      const int row = i / pairs;
      turn_cos_sin(turn_at(p.turn.freq[i - row * pairs], p.pos[r0 + row]), p.turn.amp, s_cos[i],
                   s_sin[i]);
    }
    __syncthreads();
    for (unsigned base = 0; base < slots; base += kRopeThreads / LPH * kRopeItems) {
      if (base) load(base);
#pragma unroll
      for (int k = 0; k < kRopeItems; k++) {
        const unsigned slot = base + (tid + k * kRopeThreads) / LPH;
        const unsigned row = slot / (unsigned)nh;
        const RopeHead h(p, (int)(slot - row * nh), DH);
        const HeadNorm& norm = h.part == 0 ? p.q_norm : p.k_norm;
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < P; i++) ss += a[k][i] * a[k][i] + b[k][i] * b[k][i];
        ss = group_sum<LPH>(ss);
        if (slot >= slots) continue;
        if (h.part < 2 && norm.on) {
          const float inv = 1.0f / sqrtf(ss / (float)DH + norm.eps);
          const float* w = s_w + (h.part ? DH : 0);
#pragma unroll
          for (int i = 0; i < P; i++) {
            a[k][i] = a[k][i] * inv * w[at.a + i];
            b[k][i] = b[k][i] * inv * w[at.b + i];
          }
        }
        if (h.part < 2 && at.turns) {
          float c[P], s[P];
#pragma unroll
          for (int i = 0; i < P; i++) {
            c[i] = s_cos[row * pairs + l * P + i];
            s[i] = s_sin[row * pairs + l * P + i];
          }
          rope_turn<P>(a[k], b[k], c, s, p.turn.halves);
        }
        const size_t to = (size_t)(r0 + row) * p.ldout + h.out;
        store_values<P, OB>(p.out, to + at.a, a[k]);
        store_values<P, OB>(p.out, to + at.b, b[k]);
      }
    }
    __syncthreads();
  }
}

}  // namespace rh
