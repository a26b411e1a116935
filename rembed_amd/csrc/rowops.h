// rowops.h — the row operators between a layer's products: residual norms, rotary turns of
// heads, the paged cache read back; and what the kernels that turn heads share.
//
// A pair (a, b) of a head's values at position t turns by t times its frequency f:
//   a' = m (a cos(t f) - b sin(t f)),   b' = m (b cos(t f) + a sin(t f)).
// Positions are whole numbers, so whole turns of f drop out: f is kept as a 64-bit fraction of a
// turn, t f mod 1 is a product mod 2^64, exact but for f's own rounding (2^-65 of a turn a
// position, 2^-34 at 2^31, whatever f's size; a computed f, at most 1, is off by as much again) and
// the 32 bits that are kept, and no table limits how long a text is.
// fp32 angles would be off by 2^-24 of the angle itself: 0.004 rad at position 65536.
#pragma once

#include "fp8.h"

namespace rh {

// Sums over groups of L consecutive lanes, every lane of a group getting its sum. All lanes of
// the wave have to be active.
template <int L>
__device__ __forceinline__ float group_sum(float v) {
#if defined(__HIP_DEVICE_COMPILE__)
#define RH_DPP(ctrl) \
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), ctrl, 0xF, 0xF, true))
  if constexpr (L >= 2) RH_DPP(0xB1);   // quad_perm [1, 0, 3, 2]
  if constexpr (L >= 4) RH_DPP(0x4E);   // quad_perm [2, 3, 0, 1]
  if constexpr (L >= 8) RH_DPP(0x141);  // row_half_mirror: the other quad, whose lanes are equal
  if constexpr (L >= 16) RH_DPP(0x128);  // row_ror:8
#undef RH_DPP
  typedef unsigned v2u __attribute__((ext_vector_type(2)));
  if constexpr (L >= 32) {
    const unsigned u = __float_as_uint(v);
    const v2u r = __builtin_bit_cast(v2u, __builtin_amdgcn_permlane16_swap(u, u, false, false));
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if constexpr (L >= 64) {
    const unsigned u = __float_as_uint(v);
    const v2u r = __builtin_bit_cast(v2u, __builtin_amdgcn_permlane32_swap(u, u, false, false));
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
#endif
  return v;
}

// Eight (N) consecutive values of fp32 or bf16 rows, 16-byte aligned, and back.
template <int N, bool BF16>
__device__ __forceinline__ void load_values(const void* base, size_t at, float (&v)[N]) {
  static_assert(BF16 ? N % 8 == 0 : N % 4 == 0, "whole 16-byte loads");
  if constexpr (BF16) {
#pragma unroll
    for (int j = 0; j < N; j += 8) {
      const v8bf x = *reinterpret_cast<const v8bf*>(static_cast<const __bf16*>(base) + at + j);
#pragma unroll
      for (int e = 0; e < 8; e++) v[j + e] = (float)x[e];
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; j += 4) {
      const v4f x = *reinterpret_cast<const v4f*>(static_cast<const float*>(base) + at + j);
#pragma unroll
      for (int e = 0; e < 4; e++) v[j + e] = x[e];
    }
  }
}
template <int N, bool BF16>
__device__ __forceinline__ void store_values(void* base, size_t at, const float (&v)[N]) {
  if constexpr (BF16) {
    constexpr int W = N < 8 ? N : 8;
    typedef __bf16 T __attribute__((ext_vector_type(W)));
#pragma unroll
    for (int j = 0; j < N; j += W) {
      T x;
#pragma unroll
      for (int e = 0; e < W; e++) x[e] = (__bf16)v[j + e];
      __builtin_nontemporal_store(x, reinterpret_cast<T*>(static_cast<__bf16*>(base) + at + j));
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; j += 4)
      __builtin_nontemporal_store((v4f){v[j], v[j + 1], v[j + 2], v[j + 3]},
                                  reinterpret_cast<v4f*>(static_cast<float*>(base) + at + j));
  }
}

// 16 bytes of a row as values, and N aligned floats of LDS.
template <bool BF16, int N>
__device__ __forceinline__ void widen(const v4i& raw, float (&v)[N], int at = 0) {
  if constexpr (BF16) {
    const v8bf x = __builtin_bit_cast(v8bf, raw);
#pragma unroll
    for (int e = 0; e < 8; e++) v[at + e] = (float)x[e];
  } else {
    const v4f x = __builtin_bit_cast(v4f, raw);
#pragma unroll
    for (int e = 0; e < 4; e++) v[at + e] = x[e];
  }
}
template <int N>
__device__ __forceinline__ void load_floats(const float* lds, float* v) {
  constexpr int W = N < 4 ? N : 4;
  typedef float T __attribute__((ext_vector_type(W)));
#pragma unroll
  for (int j = 0; j < N; j += W) {
    const T x = *reinterpret_cast<const T*>(lds + j);
#pragma unroll
    for (int e = 0; e < W; e++) v[j + e] = x[e];
  }
}

// 1 / sqrt(a), within 0.6 steps: the hardware's (within one) and a correction with the product's
// own rounding taken along, where that neither under- nor overflows.
__device__ __forceinline__ float inverse_root(float a) {
  if (!(a >= 0x1p-100f && a <= 0x1p100f)) return 1.0f / sqrtf(a);
  const float r = __builtin_amdgcn_rsqf(a);
  const float h = a * r, low = __builtin_fmaf(a, r, -h);
  const float e = __builtin_fmaf(-low, r, __builtin_fmaf(-h, r, 1.0f));  // 1 - a r r
  return __builtin_fmaf(0.5f * r, e, r);
}

// ---- the turn ---------------------------------------------------------------------------
// A pair's turns a position: t -> t * high + (t * low >> 32) is the 32-bit fraction of a turn at
// position t. low is signed, what it lacks is in high.
struct RopeFreq {
  int32_t low, high;
};
struct RopeTurn {
  const RopeFreq* freq;  // [pairs]
  int pairs;             // rot / 2: the head's leading 2 * pairs values turn
  int halves;            // pair i is (i, i + pairs); else (2i, 2i + 1)
  float amp;             // cos and sin are multiplied by it
};
__device__ __forceinline__ uint32_t turn_at(const RopeFreq& f, int t) {
  return (uint32_t)__mulhi(t, f.low) + (uint32_t)t * (uint32_t)f.high;
}
// cos and sin of a fraction of a turn: of its distance t from the nearest quarter, at most 1/8
// turn, by polynomials in t whose largest error is least (found by exchange; sin 1.8e-9, cos
// 5.4e-11; 2 pi in two parts, so that the angle itself is not rounded again), then the quarter's
// exchange and signs. Over all fractions of a turn the cosine is off by at most 7.6e-8 before amp, the
// sine by 6.1e-8, both by 1.4e-8 in the mean: K's codes flip between two values no more often than
// those of cosines in 64 bits, rounded.
__device__ __forceinline__ void turn_cos_sin(uint32_t turn, float amp, float& c, float& s) {
  const uint32_t u = turn + 0x20000000u;  // its upper two bits: the quarter
  const float t = (float)(int)(turn << 2) * 0x1p-34f;
  const float t2 = t * t;
  float p = __builtin_fmaf(t2, -75.36964857f, 81.59198349f);
  p = __builtin_fmaf(t2, p, -41.34166256f);
  p = __builtin_fmaf(t2, p, -1.74845553e-7f);
  const float sn = __builtin_fmaf(t, 6.2831854820251465f, t * p);
  float q = __builtin_fmaf(t2, 59.24596417f, -85.44374173f);
  q = __builtin_fmaf(t2, q, 64.93932647f);
  q = __builtin_fmaf(t2, q, -19.73920869f);
  const float cs = __builtin_fmaf(t2, q, 1.0f);
  // quarters 0..3: (c, s), (-s, c), (-c, -s), (s, -c)
  const bool odd = u & 0x40000000u;
  const uint32_t a = __float_as_uint(odd ? sn : cs), b = __float_as_uint(odd ? cs : sn);
  c = __uint_as_float(a ^ ((u + 0x40000000u) & 0x80000000u)) * amp;
  s = __uint_as_float(b ^ (u & 0x80000000u)) * amp;
}

// Pairs (a[i], b[i]) turned by c and s, and pairs (v[2 i], v[2 i + 1]).
template <int P>
__device__ __forceinline__ void turn_halves(float* a, float* b, const float* c, const float* s) {
#pragma unroll
  for (int i = 0; i < P; i++) {
    const float x = a[i], y = b[i];
    a[i] = __builtin_fmaf(x, c[i], -(y * s[i]));
    b[i] = __builtin_fmaf(y, c[i], x * s[i]);
  }
}
template <int P>
__device__ __forceinline__ void turn_pairs(float* v, const float* c, const float* s) {
#pragma unroll
  for (int i = 0; i < P / 2; i++) {
    const float x = v[2 * i], y = v[2 * i + 1];
    v[2 * i] = __builtin_fmaf(x, c[i], -(y * s[i]));
    v[2 * i + 1] = __builtin_fmaf(y, c[i], x * s[i]);
  }
}

// ---- launchers ----------------------------------------------------------------------------
struct HeadNorm {  // RMS norm of a head's values
  int on;
  float eps;
  const float* weight;  // [dh] or null: ones
};
struct RopeArgs {
  RopeTurn turn;
  const void* x;
  void* out;
  int x_bf16, ldx, out_bf16, ldout;
  int q_off, k_off, v_off;     // columns in x
  int q_out, k_out, v_out;     // and in out
  int heads, kv_heads, v_heads, dh;  // v_heads: kv heads that are copied, or 0
  HeadNorm q_norm, k_norm;
  const int32_t* pos;
  const int32_t* used;  // null: all rows
  int rows;
};
hipError_t launch_rope_rows(const RopeArgs& a, hipStream_t s);
// The append with K's heads normed and turned on the way (append.kv: the q|k|v rows), and q's heads
// as rows (rope: x, q_off, heads; rows behind cu[batch] are left as they are).
hipError_t launch_rope_append(const CacheAppendArgs& append, const RopeArgs& rope, hipStream_t s);
// Its workgroups, of 512 threads at most.
long long rope_append_grid(const CacheAppendArgs& append, const RopeArgs& rope);

struct CacheReadArgs {
  rh_kv_cache cache;
  const int32_t* table;
  int ldt;
  const int32_t *cu, *first;  // first may be null: zeros
  int batch, rows;
  void* out;
  int out_bf16, ldout, k_off, v_off;
};
hipError_t launch_cache_read(const CacheReadArgs& a, hipStream_t s);

struct ResidualArgs {
  const void* x;
  const void* y;    // null: x alone
  void* sum;        // x's type; null: not stored
  void* out;        // null: not stored
  int x_bf16, ldx, y_bf16, ldy, ldsum, out_bf16, ldout;
  uint8_t* qa;      // e4m3 codes of out; null: none
  uint8_t* sa;
  int ldq;
  rh_norm post, pre;
  const float* gate;  // null: ones
  int ldg;            // 0: one row for all
  float x_scale, y_scale;
  const int32_t* used;
  int m, n;
};
hipError_t launch_residual_norm(const ResidualArgs& a, hipStream_t s);

}  // namespace rh
