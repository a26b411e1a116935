// rope.hip — RMS norm of each q and k head and its rotary turn at the row's position.
//
// For each pair: y = x * w / sqrt(mean(x^2) + eps) where a head norm is given, then
// rowops.h's turn; one rounding, at the end. The reference keeps a table of
// cosines and turns fp32 rows in place (ropeTable, applyRoPE, modernbert.go:108-143); the
// model forwards here have a pass of their own for that (kernels_dec.hip).
//
// Every value is read and written once, and that bounds it: 16384 rows of 16 + 8 heads of 128, 201
// MB of bf16, take 37 µs, 5.4 TB/s (vector units 45 % busy); 48 rows 4.5, a launch.
#include "rope_rows.h"

#include <algorithm>
#include <type_traits>

namespace rh {

template <int LPH, int P, bool XB, bool OB, int ITEMS, bool ANY>
__global__ __launch_bounds__(kRopeThreads) void rope_rows_kernel(RopeArgs p, RopeShare share) {
  __shared__ __attribute__((aligned(16))) float lds[rope_lds(LPH * 2 * P)];
  rope_rows<LPH, P, XB, OB, ITEMS, ANY>(p, share, blockIdx.x, lds);
}

// An odd number of pairs of halves, or a head size that is no multiple of 4: a wave takes ITEMS
// heads of a row, a lane the pairs lane and (E = 2) lane + 64 of them, one value a load, and their
// cosines once.
template <bool XB, bool OB, int E, int ITEMS>
__global__ __launch_bounds__(256) void rope_any_kernel(RopeArgs p, int sets) {
  using X = std::conditional_t<XB, __bf16, float>;
  using Y = std::conditional_t<OB, __bf16, float>;
  const int lane = threadIdx.x & 63;
  const int nh = p.heads + p.kv_heads + p.v_heads, used = rope_used(p);
  const long long units = (long long)used * sets, step = (long long)gridDim.x * 4;
  int ia[E], ib[E];
  bool in[E];
#pragma unroll
  for (int e = 0; e < E; e++) {
    const int j = lane + 64 * e;
    const bool apart = p.turn.halves && j < p.turn.pairs;
    in[e] = j < p.dh / 2;
    ia[e] = !in[e] ? 0 : apart ? j : 2 * j;
    ib[e] = !in[e] ? 0 : apart ? j + p.turn.pairs : 2 * j + 1;
  }
  for (long long u = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); u < units; u += step) {
    const int row = (int)(u / sets), set = (int)(u - (long long)row * sets);
    const X* x = static_cast<const X*>(p.x) + (size_t)row * p.ldx;
    Y* y = static_cast<Y*>(p.out) + (size_t)row * p.ldout;
    float a[ITEMS][E], b[ITEMS][E];
#pragma unroll
    for (int k = 0; k < ITEMS; k++) {  // behind the last head: that one, not used
      const int from = RopeHead(p, min(set + k * sets, nh - 1), p.dh).in;
#pragma unroll
      for (int e = 0; e < E; e++) {
        a[k][e] = (float)x[from + ia[e]];
        b[k][e] = (float)x[from + ib[e]];
      }
    }
    const int t = p.pos[row];
    float c[E], s[E];
#pragma unroll
    for (int e = 0; e < E; e++) {
      const int j = lane + 64 * e;
      c[e] = 1.0f;
      s[e] = 0.0f;
      if (j < p.turn.pairs) turn_cos_sin(turn_at(p.turn.freq[j], t), p.turn.amp, c[e], s[e]);
    }
#pragma unroll
    for (int k = 0; k < ITEMS; k++) {
      if (set + k * sets >= nh) break;
      const RopeHead at(p, set + k * sets, p.dh);
      const HeadNorm& norm = at.part == 0 ? p.q_norm : p.k_norm;
      if (at.part < 2 && norm.on) {
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < E; e++)
          if (in[e]) ss = __builtin_fmaf(a[k][e], a[k][e], __builtin_fmaf(b[k][e], b[k][e], ss));
        const float inv = inverse_root(group_sum<64>(ss) / (float)p.dh + norm.eps);
#pragma unroll
        for (int e = 0; e < E; e++) {
          a[k][e] = a[k][e] * inv * (norm.weight ? norm.weight[ia[e]] : 1.0f);
          b[k][e] = b[k][e] * inv * (norm.weight ? norm.weight[ib[e]] : 1.0f);
        }
      }
#pragma unroll
      for (int e = 0; e < E; e++) {
        if (!in[e]) continue;
        float v = a[k][e], w = b[k][e];
        if (at.part < 2 && lane + 64 * e < p.turn.pairs) {
          v = __builtin_fmaf(a[k][e], c[e], -(b[k][e] * s[e]));
          w = __builtin_fmaf(b[k][e], c[e], a[k][e] * s[e]);
        }
        y[at.out + ia[e]] = (Y)v;
        y[at.out + ib[e]] = (Y)w;
      }
    }
  }
}

// Whether the pairs that turn are whole runs of `run` values.
static bool runs_fit(const RopeArgs& a, int run) {
  return (a.turn.halves ? a.turn.pairs : 2 * a.turn.pairs) % run == 0;
}

// Whether rope_rows may take these rows: P pairs a lane (8 of bf16 rows, 4 of fp32 ones), 16-byte
// loads, 16-byte stores (8 from fp32 to bf16).
static bool rope_by_lanes(const RopeArgs& a) {
  const int P = a.x_bf16 ? 8 : 4, to = a.out_bf16 ? P * 2 : 16, in = a.x_bf16 ? 8 : 4;
  const int out = to / (a.out_bf16 ? 2 : 4);
  if (a.dh != 32 && a.dh != 64 && a.dh != 128 && a.dh != 256) return false;
  if (!runs_fit(a, P)) return false;
  if ((uintptr_t)a.x % 16 || (uintptr_t)a.out % to || a.ldx % in || a.ldout % out) return false;
  if (a.heads && (a.q_off % in || a.q_out % out)) return false;
  if (a.kv_heads && (a.k_off % in || a.k_out % out)) return false;
  return !a.v_heads || (a.v_off % in == 0 && a.v_out % out == 0);
}

template <int LPH, int P, bool XB, bool OB, bool ANY>
static void launch_lanes(const RopeArgs& a, hipStream_t s) {
  RopeShare share = rope_share(a, LPH, LPH * 2 * P, kRopeThreads);
  // a launch holds fewer than 2^32 threads
  const int most = std::max(1, (1 << 23) / share.slices) * share.group;
  for (; share.first < a.rows; share.first += std::min(most, a.rows - share.first)) {
    const dim3 grid((unsigned)share.blocks(std::min(most, a.rows - share.first)));
    if (share.many)
      hipLaunchKernelGGL((rope_rows_kernel<LPH, P, XB, OB, kRopeItems, ANY>), grid,
                         dim3(kRopeThreads), 0, s, a, share);
    else
      hipLaunchKernelGGL((rope_rows_kernel<LPH, P, XB, OB, 1, ANY>), grid, dim3(kRopeThreads), 0, s,
                         a, share);
  }
}

template <int E, bool XB, bool OB>
static void launch_any(const RopeArgs& a, hipStream_t s) {
  const long long nh = (long long)a.heads + a.kv_heads + a.v_heads;
  const bool many = nh * a.rows >= kRopeItems * 2048LL;  // waves: as rope_share
  const int sets = (int)(many ? (nh + kRopeItems - 1) / kRopeItems : nh);
  const dim3 grid((unsigned)std::min(((long long)sets * a.rows + 3) / 4, 1LL << 20));
  if (many)
    hipLaunchKernelGGL((rope_any_kernel<XB, OB, E, kRopeItems>), grid, dim3(256), 0, s, a, sets);
  else
    hipLaunchKernelGGL((rope_any_kernel<XB, OB, E, 1>), grid, dim3(256), 0, s, a, sets);
}

// The widest run of values that both the pairs and the head are whole numbers of: 16 bytes (8 or 4
// values), half or a quarter of that. 4096 rows of 16 + 4 heads of 80, bf16, normed: 22.7 µs a value
// at a time, 9.0 in runs of 8; heads of 128 whose leading 20 turn, not normed: 18.5, 12.1 in runs of 2.
template <bool XB, bool OB>
static void launch_types(const RopeArgs& a, hipStream_t s) {
  constexpr int P = XB ? 8 : 4;
  if (rope_by_lanes(a)) {
    if (a.dh == 32) launch_lanes<16 / P, P, XB, OB, false>(a, s);
    else if (a.dh == 64) launch_lanes<32 / P, P, XB, OB, false>(a, s);
    else if (a.dh == 128) launch_lanes<64 / P, P, XB, OB, false>(a, s);
    else launch_lanes<128 / P, P, XB, OB, false>(a, s);
    return;
  }
  auto whole = [&](int run) { return runs_fit(a, run) && a.dh / 2 % run == 0; };
  if (whole(P)) {
    if (a.dh <= 64) launch_lanes<32 / P, P, XB, OB, true>(a, s);
    else if (a.dh <= 128) launch_lanes<64 / P, P, XB, OB, true>(a, s);
    else launch_lanes<128 / P, P, XB, OB, true>(a, s);
  } else if (XB && whole(4)) {
    if (a.dh <= 128) launch_lanes<16, 4, XB, OB, true>(a, s);
    else launch_lanes<32, 4, XB, OB, true>(a, s);
  } else if (whole(2)) {
    if (a.dh <= 128) launch_lanes<32, 2, XB, OB, true>(a, s);
    else launch_lanes<64, 2, XB, OB, true>(a, s);
  } else if (a.dh <= 128) {
    launch_any<1, XB, OB>(a, s);
  } else {
    launch_any<2, XB, OB>(a, s);
  }
}

hipError_t launch_rope_rows(const RopeArgs& a, hipStream_t s) {
  if (a.rows <= 0 || (long long)a.heads + a.kv_heads + a.v_heads == 0) return hipSuccess;
  if (a.x_bf16) {
    if (a.out_bf16) launch_types<true, true>(a, s);
    else launch_types<true, false>(a, s);
  } else {
    if (a.out_bf16) launch_types<false, true>(a, s);
    else launch_types<false, false>(a, s);
  }
  return hipGetLastError();
}

}  // namespace rh
