// rope.hip — RMS norm of each q and k head and its rotary turn at the row's position.
//
// For each pair: y = x * w / sqrt(mean(x^2) + eps) where a head norm is given, then
// rowops.h's turn; one rounding, at the end. The reference keeps a table of
// cosines and turns fp32 rows in place (applyRoPE, modernbert.go:130-143; qwen3.go:319-390); the
// model forwards here have a pass of their own for that (kernels_dec.hip).
#include "rope_rows.h"

#include <algorithm>

namespace rh {

template <int LPH, int P, bool XB, bool OB, int ITEMS>
__global__ __launch_bounds__(kRopeThreads) void rope_rows_kernel(RopeArgs p, RopeShare share) {
  __shared__ __attribute__((aligned(16))) float lds[2 * kRopePairs + 4 * LPH * P];
  rope_rows<LPH, P, XB, OB, ITEMS>(p, share, blockIdx.x, lds);
}

// Heads of any even size, rows of any alignment: a wave takes a head at a time, a lane the pairs
// lane and lane + 64.
template <bool XB, bool OB>
__global__ __launch_bounds__(256) void rope_any_kernel(RopeArgs p) {
  const int lane = threadIdx.x & 63;
  const int nh = p.heads + p.kv_heads + p.v_heads;
  const long long items = (long long)rope_used(p) * nh, step = (long long)gridDim.x * 4;
  for (long long it = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); it < items; it += step) {
    const int row = (int)(it / nh), h = (int)(it - (long long)row * nh);
    const RopeHead at(p, h, p.dh);
    const size_t in = (size_t)row * p.ldx + at.in, out = (size_t)row * p.ldout + at.out;
    float a[2], b[2], ss = 0.0f;
    int ia[2], ib[2];
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const int j = lane + 64 * e;
      const bool apart = p.turn.halves && j < p.turn.pairs;
      ia[e] = apart ? j : 2 * j;
      ib[e] = apart ? j + p.turn.pairs : 2 * j + 1;
      a[e] = b[e] = 0.0f;
      if (j < p.dh / 2) {
        if constexpr (XB) {
          a[e] = (float)static_cast<const __bf16*>(p.x)[in + ia[e]];
          b[e] = (float)static_cast<const __bf16*>(p.x)[in + ib[e]];
        } else {
          a[e] = static_cast<const float*>(p.x)[in + ia[e]];
          b[e] = static_cast<const float*>(p.x)[in + ib[e]];
        }
      }
      ss += a[e] * a[e] + b[e] * b[e];
    }
    const HeadNorm norm = at.part == 0 ? p.q_norm : p.k_norm;
    const bool normed = at.part < 2 && norm.on;
    const float inv = inverse_root(group_sum<64>(ss) / (float)p.dh + norm.eps);
    const int t = p.pos[row];
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const int j = lane + 64 * e;
      if (j >= p.dh / 2) continue;
      if (normed) {
        a[e] = a[e] * inv * (norm.weight ? norm.weight[ia[e]] : 1.0f);
        b[e] = b[e] * inv * (norm.weight ? norm.weight[ib[e]] : 1.0f);
      }
      if (at.part < 2 && j < p.turn.pairs) {
        float c, s;
        turn_cos_sin(turn_at(p.turn.freq[j], t), p.turn.amp, c, s);
        const float x = a[e], y = b[e];
        a[e] = __builtin_fmaf(x, c, -(y * s));
        b[e] = __builtin_fmaf(y, c, x * s);
      }
      if constexpr (OB) {
        static_cast<__bf16*>(p.out)[out + ia[e]] = (__bf16)a[e];
        static_cast<__bf16*>(p.out)[out + ib[e]] = (__bf16)b[e];
      } else {
        static_cast<float*>(p.out)[out + ia[e]] = a[e];
        static_cast<float*>(p.out)[out + ib[e]] = b[e];
      }
    }
  }
}

// Whether rope_rows may take these rows: P pairs a lane (8 of bf16 rows, 4 of fp32 ones), 16-byte
// loads, 16-byte stores (8 from fp32 to bf16).
static bool rope_by_lanes(const RopeArgs& a) {
  const int P = a.x_bf16 ? 8 : 4, to = a.out_bf16 ? P * 2 : 16, in = a.x_bf16 ? 8 : 4;
  const int out = to / (a.out_bf16 ? 2 : 4);
  if (a.dh != 32 && a.dh != 64 && a.dh != 128 && a.dh != 256) return false;
  if (a.turn.pairs % P) return false;
  if ((uintptr_t)a.x % 16 || (uintptr_t)a.out % to || a.ldx % in || a.ldout % out) return false;
  if (a.heads && (a.q_off % in || a.q_out % out)) return false;
  if (a.kv_heads && (a.k_off % in || a.k_out % out)) return false;
  return !a.v_heads || (a.v_off % in == 0 && a.v_out % out == 0);
}

hipError_t launch_rope_rows(const RopeArgs& a, hipStream_t s) {
  const long long nh = (long long)a.heads + a.kv_heads + a.v_heads;
  if (a.rows <= 0 || nh == 0) return hipSuccess;
  if (!rope_by_lanes(a)) {
    const unsigned wgs = (unsigned)std::min((nh * a.rows + 3) / 4, 1LL << 20);
#define RH_ANY(X, O) hipLaunchKernelGGL((rope_any_kernel<X, O>), dim3(wgs), dim3(256), 0, s, a)
    if (a.x_bf16) {
      if (a.out_bf16) RH_ANY(true, true);
      else RH_ANY(true, false);
    } else {
      if (a.out_bf16) RH_ANY(false, true);
      else RH_ANY(false, false);
    }
#undef RH_ANY
    return hipGetLastError();
  }
  const int lanes = a.dh / (a.x_bf16 ? 16 : 8);
  RopeShare share = rope_share(a, lanes);
  // a launch holds fewer than 2^32 threads
  const int most = std::max(1, (1 << 23) / share.slices) * share.group;
  for (; share.first < a.rows; share.first += std::min(most, a.rows - share.first)) {
    const dim3 grid((unsigned)share.blocks(std::min(most, a.rows - share.first)));
#define RH_ROPE(L, P, X, O, I) \
  hipLaunchKernelGGL((rope_rows_kernel<L, P, X, O, I>), grid, dim3(kRopeThreads), 0, s, a, share)
#define RH_MANY(L, P, X, O)                              \
  {                                                      \
    if (share.many) RH_ROPE(L, P, X, O, kRopeItems);     \
    else RH_ROPE(L, P, X, O, 1);                         \
  }
#define RH_LANES(D)                                       \
  if (a.dh == D) {                                        \
    if (a.x_bf16) {                                       \
      if (a.out_bf16) RH_MANY(D / 16, 8, true, true)      \
      else RH_MANY(D / 16, 8, true, false)                \
    } else {                                              \
      if (a.out_bf16) RH_MANY(D / 8, 4, false, true)      \
      else RH_MANY(D / 8, 4, false, false)                \
    }                                                     \
  }
    RH_LANES(32)
    RH_LANES(64)
    RH_LANES(128)
    RH_LANES(256)
#undef RH_LANES
#undef RH_MANY
#undef RH_ROPE
  }
  return hipGetLastError();
}

}  // namespace rh
