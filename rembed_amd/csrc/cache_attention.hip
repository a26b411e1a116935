// cache_attention.hip — softmax attention of new tokens over the paged e4m3
// cache, on v_mfma_scale_f32_32x32x64_f8f6f4.
//
// A wave takes 32 query columns (token, head of the kv head's group) and walks
// pages. It computes S^T = K.Q^T, so that lane l owns column l % 32 and half of a
// page's 64 keys; P^T then already lies in the B operand of O^T = V^T.P^T, with
// V's tokens stored in that order. K and V go from memory to the matrix cores as
// they are: codes as operands, the block's scale byte as the instruction's scale.
// A query row (bf16, or fp32 rounded to 8 bits) is the sum of two e4m3 codes,
//   q = 2^x (hi + lo / 16),
// the residue of rounding 8 significant bits to 4 having at most 4: exactly, down to
// 2^-13 of the row's largest value, and off by at most 2^-21 of that below. P is split the
// same way, so two products of the double-rate fp8 instruction take the place of one
// bf16 product and no key or value is ever converted. A column's weights of a page are
// taken against the page's own largest, what that lies above or below other pages' being
// left to the instruction's scale: each is off by at most 2^-9 of itself or 2^-21 of the
// page's largest. (One reference for all pages made weights 12 nats under a single key's, as a
// text's first token draws them, wrong by their own size.)
#include "fp8.h"

#include <algorithm>
#include <cfloat>
#include <type_traits>

namespace rh {

constexpr int kPageT = RH_CACHE_BLOCK;
constexpr int kCols = 32;    // query columns per tile
constexpr int kWaves = 4;    // per workgroup
// P^T is taken against a reference of its page: the first whole number that no score of it,
// times cs, passes, less kHead, so that codes are about 2^8 at most, of 448.
constexpr float kHead = 8.0f;
// Powers of two that a page's reference may lie from the running one.
constexpr float kFar = 64.0f;

// Visible keys [klo, khi] of a query at position i of n; none: klo = khi = 2^31 - 1, behind
// any. A window may be as long as an int, a query lie before every key.
__device__ __forceinline__ void cache_key_range(const CacheAttnArgs& p, int i, int n, int& klo,
                                                int& khi) {
  khi = n - 1;
  klo = 0;
  if (p.causal) khi = min(khi, i);
  if (p.window > 0) {
    khi = (int)min((long long)khi, (long long)i + p.window - 1);
    klo = (int)max((long long)klo, (long long)i - p.window + 1);
  }
  if (khi < klo) klo = khi = 0x7FFFFFFF;
}

// The larger of a lane's value and that of lane ^ 32, in both.
__device__ __forceinline__ float max_halves(float v) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef unsigned v2u __attribute__((ext_vector_type(2)));
  const unsigned u = __float_as_uint(v);
  const v2u r = __builtin_bit_cast(v2u, __builtin_amdgcn_permlane32_swap(u, u, false, false));
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
#else
  return v;
#endif
}

// The columns' codes and scale bytes: lane (column, half) holds values
// 64 s + 32 half .. + 31 of step s, as K's pieces do. A wave does this once, in line, so its
// instructions count (9 a value took 4.9 µs of dh 256's 29 at 8 pages): conversions that
// scale by themselves, 4.5 a value. Columns with infinities or NaN, and those below 2^-103,
// whose unit's reciprocal conversions take other ways, go by the plain one.
template <int KS, bool BF16>
__device__ __forceinline__ void cache_load_q(const void* q, size_t at, int half, v8i (&hi)[KS],
                                             v8i (&lo)[KS], int& xh, int& xl) {
#if defined(__HIP_DEVICE_COMPILE__)
  using S = std::conditional_t<BF16, __bf16, float>;
  using T = std::conditional_t<BF16, v8bf, v4f>;
  constexpr int E = BF16 ? 8 : 4;
  T v[KS][32 / E];
  uint32_t m = 0;
#pragma unroll
  for (int s = 0; s < KS; s++)
#pragma unroll
    for (int i = 0; i < 32 / E; i++)
      v[s][i] =
          *reinterpret_cast<const T*>(static_cast<const S*>(q) + at + s * 64 + half * 32 + i * E);
  if constexpr (BF16) {
    typedef uint16_t v2u16 __attribute__((ext_vector_type(2)));
    v2u16 top = {0, 0};
#pragma unroll
    for (int s = 0; s < KS; s++)
#pragma unroll
      for (int i = 0; i < 32 / E; i++) {
        const v4i w = __builtin_bit_cast(v4i, v[s][i]);
#pragma unroll
        for (int e = 0; e < 4; e++)
          top = __builtin_elementwise_max(top, __builtin_bit_cast(v2u16, w[e] & 0x7FFF7FFF));
      }
    m = (uint32_t)max(top[0], top[1]) << 16;
  } else {
#pragma unroll
    for (int s = 0; s < KS; s++)
#pragma unroll
      for (int i = 0; i < 32 / E; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) m = max(m, __float_as_uint(v[s][i][e]) & 0x7FFFFFFFu);
  }
  m = max(m, (uint32_t)__shfl_xor((int)m, 32, 64));
  xh = fp8_exponent(m);
  auto value = [&](int s, int i) { return (float)v[s][i / E][i % E]; };
  if (__builtin_expect(__any(m >= 0x7F800000u || xh < 16), 0)) {
    m = 0;
    for (int s = 0; s < KS; s++)
      for (int i = 0; i < 32; i++) m = max(m, finite_abs_bits(value(s, i)));
    m = max(m, (uint32_t)__shfl_xor((int)m, 32, 64));
    xh = fp8_exponent(m);
    xl = max(xh - 4, 0);
    const float f = fp8_inverse(xh);
#pragma unroll
    for (int s = 0; s < KS; s++)
#pragma unroll
      for (int w = 0; w < 8; w++) {
        const float a = value(s, 4 * w) * f, b = value(s, 4 * w + 1) * f,
                    c = value(s, 4 * w + 2) * f, d = value(s, 4 * w + 3) * f;
        hi[s][w] = fp8_pack4(a, b, c, d);
        lo[s][w] = xh >= 4 ? fp8_rest4(hi[s][w], a, b, c, d) : 0;
      }
    return;
  }
  xl = xh - 4;
  const float unit = __uint_as_float((uint32_t)xh << 23), rest = unit * 0.0625f;
  typedef short v2s __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int s = 0; s < KS; s++)
#pragma unroll
    for (int w = 0; w < 8; w++) {
      const float a = value(s, 4 * w), b = value(s, 4 * w + 1), c = value(s, 4 * w + 2),
                  d = value(s, 4 * w + 3);
      v2s h, l;
      asm("" : "=v"(h) : "v"(a));  // any word: both halves get written
      h = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(h, a, b, unit, false);
      h = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(h, c, d, unit, true);
      const int codes = __builtin_bit_cast(int, h);
      const v2f x = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes, unit, false);
      const v2f y = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes, unit, true);
      asm("" : "=v"(l) : "v"(a));
      l = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(l, a - x[0], b - x[1], rest, false);
      l = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(l, c - y[0], d - y[1], rest, true);
      hi[s][w] = codes;
      lo[s][w] = __builtin_bit_cast(int, l);
    }
#endif
}

// V's codes behind the last token to zero: nothing was written there, and no NaN code may
// meet a zero P.
template <int DH>
__device__ __forceinline__ void cache_clean_v(v8i (&vf)[DH / 32], int key0, int n, int half) {
#pragma unroll
  for (int w = 0; w < 8; w++) {
    const int left = n - (key0 + w / 4 * 32 + w % 4 * 8 + half * 4);
    const int keep = left >= 4 ? -1 : left <= 0 ? 0 : (1 << (8 * left)) - 1;
#pragma unroll
    for (int t = 0; t < DH / 32; t++) vf[t][w] &= keep;
  }
}

// One wave's running state of its 32 columns, and a page's step, for scores of any size: O and
// the sum in units of the largest reference so far (mref).
template <int DH>
struct CacheTile {
  static constexpr int KS = DH / 64, DT = DH / 32;
  v8i qh[KS], ql[KS];
  int xh, xl;
  v16f o[DT];
  float mref, lrun;
  int klo, khi;

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int t = 0; t < DT; t++) o[t] = v16f{};
    mref = -INFINITY;
    lrun = 0.0f;
  }

  // kf[s][t]: keys 32t.., step s; vf[t]: values' columns 32t.., all 64 tokens.
  // key0: the page's first position; n: tokens in the cache.
  __device__ __forceinline__ void page(const v8i (&kf)[KS][2], v8i (&vf)[DT], int xk, int xv,
                                       int key0, int n, float cs, int half) {
    v16f sc[2] = {v16f{}, v16f{}};
#pragma unroll
    for (int s = 0; s < KS; s++)
#pragma unroll
      for (int t = 0; t < 2; t++) {
        sc[t] = mfma_fp8_32(kf[s][t], qh[s], sc[t], xk, xh);
        sc[t] = mfma_fp8_32(kf[s][t], ql[s], sc[t], xk, xl);
      }
    if (__any(key0 < klo || key0 + kPageT - 1 > khi)) {
      const unsigned span = (unsigned)(khi - klo);
      const int base = key0 + half * 4 - klo;
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int e = 0; e < 16; e++) {
          const unsigned off = (unsigned)(base + t * 32 + e / 4 * 8 + e % 4);
          sc[t][e] = off > span ? -INFINITY : sc[t][e];
        }
    }
    if (key0 + kPageT > n) cache_clean_v<DH>(vf, key0, n, half);
    float smax = -INFINITY;
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int e = 0; e < 16; e++) smax = fmaxf(smax, sc[t][e]);
    smax = max_halves(smax);
    const float mloc = smax * cs, to = __builtin_ceilf(mloc) - kHead;
    const bool up = to > mref;
    if (__any(up)) {
      float alpha = 1.0f;
      if (up) {
        alpha = __builtin_amdgcn_exp2f(mref - to);
        mref = to;
      }
      lrun *= alpha;
#pragma unroll
      for (int t = 0; t < DT; t++) o[t] *= alpha;
    }
    // the page's reference in units of the running one; against its largest score first, as a
    // difference of large products is no number near 0. No visible key: every p = 2^(-inf) = 0
    const float near = smax == -INFINITY ? 0.0f : smax;
    const float head = smax == -INFINITY ? 0.0f : kHead - (__builtin_ceilf(mloc) - mloc);
    const int unit = 127 + (smax == -INFINITY ? 0 : (int)fmaxf(to - mref, -kFar));
    float sum = 0.0f;
    v8i ph, pl;
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int w = 0; w < 4; w++) {
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
          x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][4 * w + e] - near, cs, head));
          sum += x[e];
        }
        ph[4 * t + w] = fp8_pack4(x[0], x[1], x[2], x[3]);
        pl[4 * t + w] = fp8_rest4(ph[4 * t + w], x[0], x[1], x[2], x[3]);
      }
    lrun = __builtin_fmaf(sum, __uint_as_float((uint32_t)unit << 23), lrun);
#pragma unroll
    for (int t = 0; t < DT; t++) {
      o[t] = mfma_fp8_32(vf[t], ph, o[t], xv, unit);
      o[t] = mfma_fp8_32(vf[t], pl, o[t], xv, unit - 4);
    }
  }
};

// A page's fragments of one head: 1 KiB pieces, 16 bytes a lane. STREAM: read by nobody else,
// so they need not stay in the L2.
template <bool STREAM>
__device__ __forceinline__ v8i cache_fetch(const v4i* at) {
  if constexpr (STREAM)
    return join8(__builtin_nontemporal_load(at), __builtin_nontemporal_load(at + 64));
  return join8(at[0], at[64]);
}
template <int DH, bool STREAM>
__device__ __forceinline__ void cache_fetch_k(const uint8_t* k, int lane, v8i (&kf)[DH / 64][2]) {
  const v4i* at = reinterpret_cast<const v4i*>(k) + lane;
#pragma unroll
  for (int s = 0; s < DH / 64; s++)
#pragma unroll
    for (int t = 0; t < 2; t++) kf[s][t] = cache_fetch<STREAM>(at + (s * 2 + t) * 128);
}
template <int DH, bool STREAM>
__device__ __forceinline__ void cache_fetch_v(const uint8_t* v, int lane, v8i (&vf)[DH / 32]) {
  const v4i* at = reinterpret_cast<const v4i*>(v) + lane;
#pragma unroll
  for (int t = 0; t < DH / 32; t++) vf[t] = cache_fetch<STREAM>(at + t * 128);
}

// The same with accumulators that products alone touch. O and the sum are kept in units of
// the first page's reference (`base`); what a page's lies above or below it, always a whole
// power of two, goes into P's scale byte. Pages more than 2^64 below weigh nothing in fp32 and
// count from there. A column with one more than 2^64 above, or with scores of 2^24 and more, whose
// rounding reaches the references, makes its wave go over its pages once more with CacheTile:
// its rescale inside the loops cost the compiler a second copy of O and 8 to 30 spilled registers.
template <int DH>
struct CacheFast {
  static constexpr int KS = DH / 64, DT = DH / 32;
  v8i qh[KS], ql[KS];
  int xh, xl;
  v16f o[DT], sc[2];
  v8i ph, pl;  // P of a page,
  int eh, el;  // its scale bytes
  float ref, base, lrun;  // the page's reference, the first one's (-inf: none), the sum of P
  unsigned long long far;  // lanes whose column is
  int klo, khi;

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int t = 0; t < DT; t++) o[t] = v16f{};
    ph = v8i{};
    pl = v8i{};
    eh = el = 127;
    ref = 0.0f;
    base = -INFINITY;
    lrun = 0.0f;
    far = 0;
  }
  // With more than 256 registers in use (dh 256) the compiler may move a scale word to an
  // accumulation register, which the instruction does not take: held in a VGPR here.
  static __device__ __forceinline__ v16f mul(const v8i& a, const v8i& b, const v16f& c, int ea,
                                             int eb) {
    if constexpr (DH == 256) asm("" : "+v"(ea), "+v"(eb));
    return mfma_fp8_32(a, b, c, ea, eb);
  }
  // Scores of a page (first position key0) to its reference. `none`: the page holds no keys
  // at all.
  __device__ __forceinline__ void refer(int key0, bool none, float cs, int half) {
    if (__builtin_expect(none || __any(key0 < klo || key0 + kPageT - 1 > khi), 0)) {
      const unsigned span = (unsigned)(khi - klo);
      const int at = key0 + half * 4 - klo;
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int e = 0; e < 16; e++) {
          const unsigned off = (unsigned)(at + t * 32 + e / 4 * 8 + e % 4);
          sc[t][e] = none || off > span ? -INFINITY : sc[t][e];
        }
    }
    float smax = -INFINITY;
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int e = 0; e < 16; e++) smax = fmaxf(smax, sc[t][e]);
    const float to = __builtin_ceilf(max_halves(smax) * cs) - kHead;
    // a column with no visible key yet: any finite number, every p = 2^(-inf) = 0
    ref = fmaxf(fmaxf(to, base - kFar), -FLT_MAX);
    base = base == -INFINITY ? to : base;
  }
  // P's scale bytes; the page's weights into the sum
  __device__ __forceinline__ void scales(float sum) {
    const float moved = base == -INFINITY ? 0.0f : ref - base;
    far |= __ballot(moved > kFar) |
           __ballot((base > -INFINITY) & (__builtin_fabsf(ref) >= 0x1p24f));
    eh = 127 + (int)fminf(moved, kFar);
    el = eh - 4;
    lrun = __builtin_fmaf(sum, __uint_as_float((uint32_t)eh << 23), lrun);
  }
  // one page, its fragments in registers (CacheTile::page)
  __device__ __forceinline__ void page(const v8i (&kf)[KS][2], v8i (&vf)[DT], int xk, int xv,
                                       int key0, int n, float cs, int half) {
    sc[0] = v16f{};
    sc[1] = v16f{};
#pragma unroll
    for (int s = 0; s < KS; s++)
#pragma unroll
      for (int u = 0; u < 4; u++)
        sc[u % 2] = mul(kf[s][u % 2], u < 2 ? qh[s] : ql[s], sc[u % 2], xk, u < 2 ? xh : xl);
    refer(key0, false, cs, half);
    if (key0 + kPageT > n) cache_clean_v<DH>(vf, key0, n, half);
    float sum = 0.0f;
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int w = 0; w < 4; w++) {
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
          x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][4 * w + e], cs, -ref));
          sum += x[e];
        }
        ph[4 * t + w] = fp8_pack4(x[0], x[1], x[2], x[3]);
        pl[4 * t + w] = fp8_rest4(ph[4 * t + w], x[0], x[1], x[2], x[3]);
      }
    scales(sum);
#pragma unroll
    for (int t = 0; t < DT; t++) o[t] = mul(vf[t], ph, o[t], xv, eh);
#pragma unroll
    for (int t = 0; t < DT; t++) o[t] = mul(vf[t], pl, o[t], xv, el);
  }
};

// Page ids and scale bytes of 64 consecutive pages of a request, one a lane: read once, then
// taken lane by lane, so that no page waits for its table entry and scales.
struct PageWindow {
  int page, xk, xv;  // page: -1, scales 1, where the entry is no page of the cache
  // pages g0 .. g0 + 63, none from `end` on
  __device__ __forceinline__ void load(const CacheAttnArgs& p, int b, int h, int g0, int end,
                                       int lane) {
    const int g = g0 + lane;
    page = g < end ? p.table[(size_t)b * p.ldt + g] : -1;
    if (page < 0 || page >= p.cache.pages) page = -1;
    const size_t unit = (size_t)max(page, 0) * p.cache.kv_heads + h;
    // no scale of page 0 for what is none: nobody may have written it, 255 is NaN there, and a
    // product of zeros under it NaN too
    xk = page < 0 ? 127 : p.cache.k_exp[unit];
    xv = page < 0 ? 127 : p.cache.v_exp[unit];
    // waited for here: at their uses, in every turn, the wait would cover younger loads
    asm("" : "+v"(page), "+v"(xk), "+v"(xv));
  }
  static __device__ __forceinline__ int at(int v, int i) {
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_amdgcn_readlane(v, i);
#else
    return v;
#endif
  }
};

// Many columns, up to so many workgroups of a unit (one request and kv head): the grid is
// units x workgroups x key ranges, so that those that short requests leave empty come last and
// not between the others (32 queries of 9 to 70 rows: 22.9 µs, so 22.3).
constexpr int kFewTiles = 4;

// Workgroup -> (request, kv head, tile of columns, key range). A unit's workgroups (one
// request and kv head) read the same pages: where eight units are left their workgroups are
// dealt to an XCD each (workgroup w runs on XCD w % 8) and share its L2, the last ones are
// spread over all XCDs.
__device__ __forceinline__ void cache_unit(const CacheAttnArgs& p, int tiles, int splits, int& b,
                                           int& h, int& tile, int& split) {
  const int units = p.batch * p.cache.kv_heads, nv = tiles * splits;
  const int whole = units / 8 * 8, w = blockIdx.x;
  int u, v;
  if (w < whole * nv) {
    const int t = w >> 3;
    v = t % nv;
    u = (t / nv) * 8 + (w & 7);
  } else {
    const int left = units - whole, t = w - whole * nv;
    v = t / left;
    u = whole + t % left;
  }
  b = u / p.cache.kv_heads;
  h = u % p.cache.kv_heads;
  tile = v / splits;
  split = v % splits;
}

// Pages [lo, hi) that columns c0 .. c1 - 1 of a request see.
__device__ __forceinline__ void cache_page_range(const CacheAttnArgs& p, int pos0, int n, int G,
                                                 int c0, int c1, int& lo, int& hi) {
  lo = 0;
  hi = (n + kPageT - 1) / kPageT;
  const int i0 = pos0 + c0 / G, i1 = pos0 + (c1 - 1) / G;
  if (p.causal) hi = min(hi, i1 < 0 ? 0 : i1 / kPageT + 1);
  if (p.window > 0) {
    lo = (int)(max(0LL, (long long)i0 - p.window + 1) / kPageT);
    const long long last = (long long)i1 + p.window - 1;
    if (last < n) hi = min(hi, last < 0 ? 0 : (int)(last / kPageT) + 1);
  }
}

__device__ __forceinline__ void cache_store4(const CacheAttnArgs& p, size_t to, const v4f& x) {
  if (p.out_bf16) {
    typedef __bf16 v4bf __attribute__((ext_vector_type(4)));
    *reinterpret_cast<v4bf*>(static_cast<__bf16*>(p.out) + to) =
        (v4bf){(__bf16)x[0], (__bf16)x[1], (__bf16)x[2], (__bf16)x[3]};
  } else {
    *reinterpret_cast<v4f*>(static_cast<float*>(p.out) + to) = x;
  }
}

// A wave's pages first, first + each, .. once more, by CacheTile; O, reference and sum to w.
template <int DH>
__device__ __forceinline__ void cache_again(CacheFast<DH>& w, const CacheAttnArgs& p, int b, int h,
                                            int first, int end, int each, int n, float cs,
                                            int lane) {
  constexpr int KS = DH / 64, DT = DH / 32, kHalf = kPageT * DH;
  CacheTile<DH> r;
#pragma unroll
  for (int s = 0; s < KS; s++) {
    r.qh[s] = w.qh[s];
    r.ql[s] = w.ql[s];
  }
  r.xh = w.xh;
  r.xl = w.xl;
  r.klo = w.klo;
  r.khi = w.khi;
  r.clear();
  for (int g = first; g < end; g += each) {
    const int page = p.table[(size_t)b * p.ldt + g];
    if (page < 0 || page >= p.cache.pages) continue;
    const size_t u = (size_t)page * p.cache.kv_heads + h;
    v8i kf[KS][2], vf[DT];
    cache_fetch_k<DH, false>(p.cache.k + u * kHalf, lane, kf);
    cache_fetch_v<DH, false>(p.cache.v + u * kHalf, lane, vf);
    r.page(kf, vf, p.cache.k_exp[u], p.cache.v_exp[u], g * kPageT, n, cs, lane >> 5);
  }
#pragma unroll
  for (int t = 0; t < DT; t++) w.o[t] = r.o[t];
  w.base = r.mref;
  w.lrun = r.lrun;
}

// A row of a partial result: DH values, the reference and the sum, 16-byte aligned.
template <int DH>
constexpr int kPartRow = DH + 4;

// ---- few columns -----------------------------------------------------------------------
// Four waves share a tile of columns and take its pages in turn, straight to registers: what
// bounds it is the cache's bytes, each read once: 48 single tokens over 500 to 8191 (463 MB,
// 16 heads over 8 of dh 128) take 80 µs, 5.8 TB/s, where a large copy reaches 4.9 and pages kept in
// the L2 94 µs (cache_streams). Two workgroups
// to a CU hide each other's waits; the next page's K asked for a page ahead did not gain and
// cost registers. The waves' results are joined in LDS, eight columns at a time.
template <int DH, bool BF16, bool STREAM>
__global__ __launch_bounds__(64 * kWaves, DH == 256 ? 1 : 2) void cache_attention_kernel(
    CacheAttnArgs p, int tiles, int splits, int max_cols) {
  constexpr int KS = DH / 64, DT = DH / 32, kStride = DH + 4, kHalf = kPageT * DH;
  constexpr int kJoin = 8;  // columns joined at a time
  __shared__ __attribute__((aligned(16))) float s_o[kWaves][kJoin][kStride];
  __shared__ float s_m[kWaves][kCols], s_l[kWaves][kCols];
  int b, h, tile, split;
  cache_unit(p, tiles, splits, b, h, tile, split);
  const int G = p.heads / p.cache.kv_heads;
  const int r0 = p.cu[b], nq = p.cu[b + 1] - r0;
  const int cols = min(nq * G, max_cols), c0 = tile * kCols;
  if (c0 >= cols) return;
  const int n = max(0, min(p.lens[b], p.ldt * kPageT));
  const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = min(c0 + col, cols - 1), ct = c / G;
  const int pos0 = n - nq;  // position of the first new token
  const float cs = p.scale * 1.44269504088896341f;

  // the tile's pages, this split's share of them
  int lo, hi;
  cache_page_range(p, pos0, n, G, c0, min(c0 + kCols, cols), lo, hi);
  if (p.cache.pages < 1) hi = lo;
  const int each = (max(0, hi - lo) + splits - 1) / splits;
  const int first = lo + split * each, end = min(hi, first + each);
  PageWindow win;
  if (first < end) win.load(p, b, h, first, end, lane);

  CacheFast<DH> w;
  cache_load_q<KS, BF16>(p.q, (size_t)(r0 + ct) * p.ldq + p.q_off + (h * G + c - ct * G) * DH, half,
                         w.qh, w.ql, w.xh, w.xl);
  w.clear();
  cache_key_range(p, pos0 + ct, n, w.klo, w.khi);

  for (int g0 = first; g0 < end; g0 += 64) {
    if (g0 > first) win.load(p, b, h, g0, end, lane);
    const int count = min(64, end - g0);
    for (int i = wave; i < count; i += kWaves) {
      const int page = win.at(win.page, i);
      if (page < 0) continue;  // no such page: no keys
      const size_t at = ((size_t)page * p.cache.kv_heads + h) * kHalf;
      v8i kf[KS][2], vf[DT];
      cache_fetch_k<DH, STREAM>(p.cache.k + at, lane, kf);
      cache_fetch_v<DH, STREAM>(p.cache.v + at, lane, vf);
      w.page(kf, vf, win.at(win.xk, i), win.at(win.xv, i), (g0 + i) * kPageT, n, cs, half);
    }
  }

  if (__builtin_expect(w.far != 0, 0))
    cache_again<DH>(w, p, b, h, first + wave, end, kWaves, n, cs, lane);

  // join the waves: the columns' references and sums, then O in wave order
  {
    const float l = w.lrun + __shfl_xor(w.lrun, 32, 64);
    if (half == 0) {
      s_m[wave][col] = w.base;
      s_l[wave][col] = l;
    }
  }
  const int here = min(kCols, cols - c0);
  constexpr int LPR = DH / 4, kRows = 64 * kWaves / LPR;
  for (int j0 = 0; j0 < here; j0 += kJoin) {
    if (col >= j0 && col < j0 + kJoin && c0 + col < cols) {
#pragma unroll
      for (int t = 0; t < DT; t++)
#pragma unroll
        for (int q4 = 0; q4 < 4; q4++) {
          v4f x;
#pragma unroll
          for (int e = 0; e < 4; e++) x[e] = w.o[t][q4 * 4 + e];
          *reinterpret_cast<v4f*>(&s_o[wave][col - j0][t * 32 + q4 * 8 + half * 4]) = x;
        }
    }
    __syncthreads();
    const int d = threadIdx.x % LPR * 4;
    for (int r = threadIdx.x / LPR; r < min(kJoin, here - j0); r += kRows) {
      float m = -INFINITY, l = 0.0f;
#pragma unroll
      for (int k = 0; k < kWaves; k++) m = fmaxf(m, s_m[k][j0 + r]);
      v4f x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < kWaves; k++) {
        // a wave with no visible key has zeros (or, with a NaN, that)
        const float mk = s_m[k][j0 + r];
        const float f = mk == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mk - m);
        l += s_l[k][j0 + r] * f;
        const v4f y = *reinterpret_cast<const v4f*>(&s_o[k][r][d]);
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] += y[e] * f;
      }
      const int cc = c0 + j0 + r;
      if (splits > 1) {
        const size_t u = ((size_t)b * p.cache.kv_heads + h) * tiles + tile;
        float* to =
            p.part + ((u * splits + split) * min(kCols, max_cols) + j0 + r) * kPartRow<DH>;
        *reinterpret_cast<v4f*>(to + d) = x;
        if (d == 0) {
          to[DH] = m;
          to[DH + 1] = l;
        }
      } else {
        x *= l == 0.0f ? 0.0f : 1.0f / l;
        const int tt = cc / G;
        cache_store4(p, (size_t)(r0 + tt) * p.ldout + (h * G + cc - tt * G) * DH + d, x);
      }
    }
    __syncthreads();
  }
}

// ---- many columns --------------------------------------------------------------------
// CW waves of 32 columns each walk the same pages, PG such groups a part of them each. What
// bounds it: a page's products take the matrix cores 64 cycles each (dh 128: 16 of them, 1024
// cycles) and its softmax the VALU 1390, and a wave issues in order, so one after the other they
// cost their sum even with two waves per SIMD. The loop is a pipeline over pages whose body has no
// branch: while page g's scores become P, two at a time, the products between them are
// page g + 1's scores and page g - 1's values. K and V come to LDS by global_load_lds in
// fragment order (1 KiB pieces, read back without bank conflicts), two turns before they are
// used (one turn where LDS has room for two pages only), with one barrier per turn. Where few
// workgroups come together, a CU has one of them and a wave's own chain bounds a turn: then
// two waves take two tiles, and two more the second half of the pages, joined in LDS.
// 4096 rows over 8192 of 16 heads over 8 of dh 128 take 305 µs, 1.13 PFLOP/s of attention and
// twice that of e4m3 products, with the VALU busy 70% of the time and the matrix cores 50%.
template <int DH>
struct CachePipe : CacheFast<DH> {  // ph, pl, eh, el: P of the page before
  using Base = CacheFast<DH>;
  using Base::qh, Base::ql, Base::xh, Base::xl, Base::o, Base::sc, Base::ph, Base::pl, Base::eh,
      Base::el, Base::ref, Base::mul, Base::KS, Base::DT;
  static constexpr int NF = 2 * KS + DT;  // fragments of a page

  // fragment f of a page at its lane's place in LDS
  static __device__ __forceinline__ v8i frag(const uint8_t* at, int f) {
    return join8(*reinterpret_cast<const v4i*>(at + 2 * f * 1024),
                 *reinterpret_cast<const v4i*>(at + 2 * f * 1024 + 1024));
  }
  __device__ __forceinline__ void scores(const uint8_t* k, int xk) {
    v16f s[2] = {v16f{}, v16f{}};
#pragma unroll
    for (int f = 0; f < 2 * KS; f++) {
      const v8i a = frag(k, f);
      s[f & 1] = mul(a, qh[f / 2], s[f & 1], xk, xh);
      s[f & 1] = mul(a, ql[f / 2], s[f & 1], xk, xl);
    }
    sc[0] = s[0];
    sc[1] = s[1];
  }
  __device__ __forceinline__ void values(const uint8_t* v, int xv) {
#pragma unroll
    for (int t = 0; t < DT; t++) {
      const v8i a = frag(v, t);
      o[t] = mul(a, ph, o[t], xv, eh);
      o[t] = mul(a, pl, o[t], xv, el);
    }
  }
  // P of page g, between the values of page g - 1 (v, xv) and the scores of g + 1 (k, xk).
  // `fetch` asks for the next pages, a 1 KiB piece of kFetch at a time: all at once they hold
  // the wave up while their addresses go out (32 queries of 9 to 70 rows: 24.8 µs, so 23.6).
  template <int kFetch, typename Fetch>
  __device__ __forceinline__ void turn(const uint8_t* k, int xk, const uint8_t* v, int xv,
                                       float cs, Fetch&& fetch) {
    v16f s[2] = {v16f{}, v16f{}};
    v8i nh, nl;
    float sum = 0.0f;
    constexpr int kPairs = 16;
    // Two scores at a time, 68 cycles of VALU beside a product's 64. Each step waits
    // on the one before it, so three pairs are under way: the exponentials of pair j, the
    // codes of j - 1, what those leave over of j - 2.
    float x[3], y[3];
    v2f rest[3];
    auto pair = [&](int j) {
#if defined(__HIP_DEVICE_COMPILE__)
      if (j >= 2) {
        const int i = j - 2, w = i / 2, q = i % 3;
        const float u = __builtin_fmaf(x[q], 16.0f, -rest[q][0]);
        const float t = __builtin_fmaf(y[q], 16.0f, -rest[q][1]);
        int l = nl[w];
        if (i % 2 == 0) {
          asm("" : "=v"(l) : "v"(u));  // any word: both halves get written
          l = __builtin_amdgcn_cvt_pk_fp8_f32(u, t, l, false);
        } else {
          l = __builtin_amdgcn_cvt_pk_fp8_f32(u, t, l, true);
        }
        nl[w] = l;
      }
      if (j >= 1 && j <= kPairs) {
        const int i = j - 1, w = i / 2, q = i % 3;
        sum += x[q];
        sum += y[q];
        int h = nh[w];
        if (i % 2 == 0) {
          asm("" : "=v"(h) : "v"(x[q]));
          h = __builtin_amdgcn_cvt_pk_fp8_f32(x[q], y[q], h, false);
          rest[q] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(h, 16.0f, false);
        } else {
          h = __builtin_amdgcn_cvt_pk_fp8_f32(x[q], y[q], h, true);
          rest[q] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(h, 16.0f, true);
        }
        nh[w] = h;
      }
      if (j < kPairs) {
        const int e = 2 * j % 16, q = j % 3;
        x[q] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[j / 8][e], cs, -ref));
        y[q] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[j / 8][e + 1], cs, -ref));
      }
#endif
    };
    // Products in fours: two fragments by hi, then by lo, so that no product waits for
    // the one before it; values first, whose P then makes room for the scores. Three
    // fragments at a time are in registers.
    constexpr int NM = 2 * NF;
    auto piece = [&](int f) { return f < DT ? frag(v, f) : frag(k, f - DT); };
    v8i a0 = piece(0), a1 = piece(1);
#pragma unroll
    for (int f = 0; f < NF; f += 2) {
      v8i b0 = a0, b1 = a1;
#pragma unroll
      for (int u = 0; u < 4; u++) {
        const v8i& a = u % 2 ? a1 : a0;
        const int g = f + u % 2, st = (f - DT) / 2;
        if (f < DT) o[g] = mul(a, u < 2 ? ph : pl, o[g], xv, u < 2 ? eh : el);
        else s[u % 2] = mul(a, u < 2 ? qh[st] : ql[st], s[u % 2], xk, u < 2 ? xh : xl);
        if (u == 0 && f + 2 < NF) b0 = piece(f + 2);
        if (u == 2 && f + 2 < NF) b1 = piece(f + 3);
        const int at = 2 * f + u;  // of NM
#pragma unroll
        for (int j = at * kFetch / NM; j < (at + 1) * kFetch / NM; j++) fetch(j);
#pragma unroll
        for (int j = at * kPairs / NM; j < (at + 1) * kPairs / NM; j++) pair(j);
      }
      a0 = b0;
      a1 = b1;
    }
    pair(kPairs);
    pair(kPairs + 1);
    ph = nh;
    pl = nl;
    Base::scales(sum);
    sc[0] = s[0];
    sc[1] = s[1];
  }
};

template <int DH, bool BF16, int CW, int PG, int SLOTS>
__global__ __launch_bounds__(64 * CW * PG, DH == 256 ? 1 : 2) void cache_attention_cols_kernel(
    CacheAttnArgs p, int tiles, int splits, int max_cols) {
  constexpr int KS = DH / 64, DT = DH / 32, kHalf = kPageT * DH;  // bytes of K or V of a page
  constexpr int kRing = 2 * SLOTS * kHalf;  // a group's K pages, then its V pages
  constexpr int kJoin = PG > 1 ? CW * kCols * (DH + 2) * 4 : 0;
  constexpr int kLds = PG * kRing > kJoin ? PG * kRing : kJoin;
  constexpr int kPieces = kHalf / 1024 / CW;  // 1 KiB pieces per wave, of K and of V
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kLds];
  const int wgs = (tiles + CW - 1) / CW;
  int b, h, wg, split;
  if (wgs <= kFewTiles) {
    b = blockIdx.x / p.cache.kv_heads;
    h = blockIdx.x % p.cache.kv_heads;
    wg = blockIdx.y;
    split = blockIdx.z;
  } else {
    cache_unit(p, wgs, splits, b, h, wg, split);
  }
  if (p.causal && wgs > kFewTiles) {
    // later columns see more pages: each XCD's 32 CUs get the long ones first, then
    // the next 32 in the other order, so that long and short ones share a CU
    const int k = wg / 32, size = min(32, wgs - 32 * k);
    wg = wgs - 1 - (32 * k + (k & 1 ? size - 1 - wg % 32 : wg % 32));
  }
  const int G = p.heads / p.cache.kv_heads;
  const int r0 = p.cu[b], nq = p.cu[b + 1] - r0;
  const int cols = min(nq * G, max_cols);
  if (wg * CW * kCols >= cols) return;
  const int n = max(0, min(p.lens[b], p.ldt * kPageT));
  const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = PG > 1 ? wave / CW : 0, part_of = PG > 1 ? wave % CW : wave;
  const int tile = wg * CW + part_of, c0 = tile * kCols;
  const int c = min(c0 + col, cols - 1), ct = c / G;
  const int pos0 = n - nq;
  const float cs = p.scale * 1.44269504088896341f;

  int lo, hi;
  cache_page_range(p, pos0, n, G, wg * CW * kCols, min((wg + 1) * CW * kCols, cols), lo, hi);
  if (p.cache.pages < 1) hi = lo;
  const int each = (max(0, hi - lo) + splits - 1) / splits;
  // the group's pages; the last group's may end behind the range, with pages that are none
  const int limit = min(hi, lo + (split + 1) * each);
  const int turns = (max(0, limit - lo - split * each) + PG - 1) / PG;
  const int first = lo + split * each + group * turns, end = first + turns;
  const bool active = c0 < cols;

  // A page that is none is read as page 0 and holds no keys.
  PageWindow win;
  int base = first;  // the window's first page
  auto source = [&](const uint8_t* src, int page) {
    const size_t unit = (size_t)max(page, 0) * p.cache.kv_heads + h;
    return src + unit * kHalf + part_of * kPieces * 1024 + lane * 16;
  };
  auto dma = [&](const uint8_t* src, int page, uint8_t* dst) {
    const uint8_t* at = source(src, page);
#pragma unroll
    for (int i = 0; i < kPieces; i++)
      lds_dma16(at + i * 1024, dst + (part_of * kPieces + i) * 1024);
  };
  uint8_t* const ldsk = lds + group * kRing;
  uint8_t* const ldsv = ldsk + SLOTS * kHalf;
  // V behind the last token is zeroed: no NaN code may meet a zero P. A wave does it to the
  // pieces it fetched, before the barrier that gives them to the others.
  auto clean = [&](int g, bool none, uint8_t* v) {
    if (!none && (g + 1) * kPageT <= n) return;
    for (int i = part_of * kPieces * 1024 + lane * 4; i < (part_of + 1) * kPieces * 1024; i += 256) {
      // four tokens of one column: 32 * part + 8 * (byte / 4) + 4 * half
      const int t = (i / 1024 & 1) * 32 + (i % 16) / 4 * 8 + (i % 1024) / 512 * 4;
      const int left = none ? 0 : n - (g * kPageT + t);
      const int keep = left >= 4 ? -1 : left <= 0 ? 0 : (1 << (8 * left)) - 1;
      *reinterpret_cast<int*>(v + i) &= keep;
    }
  };

  CachePipe<DH> w;
  if (turns > 0) {
    win.load(p, b, h, first, limit, lane);
    dma(p.cache.k, win.at(win.page, 0), ldsk);
    dma(p.cache.k, win.at(win.page, 1), ldsk + kHalf);
    if (SLOTS > 2) {
      dma(p.cache.v, win.at(win.page, 0), ldsv + kHalf);
      dma(p.cache.k, win.at(win.page, 2), ldsk + 2 * kHalf);
    }
  }
  cache_load_q<KS, BF16>(p.q, (size_t)(r0 + ct) * p.ldq + p.q_off + (h * G + c - ct * G) * DH, half,
                         w.qh, w.ql, w.xh, w.xl);
  w.clear();
  cache_key_range(p, pos0 + ct, n, w.klo, w.khi);
  // turn g: K of g + 1 in slot ks of ldsk, V of g - 1 in slot vs of ldsv
  int ks = 1, vs = 0;
  bool nonep = false, none = false;  // page g - 1, g is none
  auto after = [](int slot) { return slot == SLOTS - 1 ? 0 : slot + 1; };
  const uint8_t *vfrom = nullptr, *kfrom = nullptr;
  uint8_t *vplace = nullptr, *kplace = nullptr;
  constexpr int kAhead = SLOTS;  // K of g + kAhead, V of g + kAhead - 2 are asked for in turn g
  auto stage = [&](int g) {
    if (SLOTS > 2) wait_vmcnt<2 * kPieces>();  // all but the last turn's
    else wait_vmcnt<0>();
    if (g > first) clean(g - 1, nonep, ldsv + vs * kHalf);
    wait_lgkmcnt0();
    stage_barrier();
    if (g + kAhead >= base + 64) {
      win.load(p, b, h, g, limit, lane);
      base = g;
    }
    none = win.at(win.page, g - base) < 0;
    // Three slots: V of g + 1 and K of g + 3 go where V of g - 2 and K of g were.
    // Two: V of g and K of g + 2.
    const int vto = SLOTS > 2 ? after(after(vs)) : after(vs);
    const int kto = SLOTS > 2 ? after(after(ks)) : after(ks);
    vfrom = source(p.cache.v, win.at(win.page, g + kAhead - 2 - base));
    kfrom = source(p.cache.k, win.at(win.page, g + kAhead - base));
    vplace = ldsv + vto * kHalf + part_of * kPieces * 1024;
    kplace = ldsk + kto * kHalf + part_of * kPieces * 1024;
  };
  auto fetch = [&](int i) {
    if (i < kPieces) lds_dma16(vfrom + i * 1024, vplace + i * 1024);
    else lds_dma16(kfrom + (i - kPieces) * 1024, kplace + (i - kPieces) * 1024);
  };
  auto done = [&] {
    nonep = none;
    ks = after(ks);
    vs = after(vs);
  };
  auto last = [&] {
    wait_vmcnt<0>();
    clean(end - 1, nonep, ldsv + vs * kHalf);
    wait_lgkmcnt0();
    stage_barrier();
  };
  if (turns > 0) {
    // V of page `first - 1` is multiplied by P = 0: any finite codes
    for (int i = part_of * 1024 + lane * 16; i < kHalf; i += CW * 1024)
      *reinterpret_cast<v4i*>(ldsv + i) = v4i{0, 0, 0, 0};
    __syncthreads();  // waits for the DMA too
    if (!active) {  // a wave without columns stages its pieces
      for (int g = first; g < end; g++) {
        stage(g);
#pragma unroll
        for (int i = 0; i < 2 * kPieces; i++) fetch(i);
        done();
      }
      last();
    } else {
      w.scores(ldsk + lane * 16, win.at(win.xk, 0));
      int xvp = 127;  // scale of V of page g - 1
      for (int g = first; g < end; g++) {
        stage(g);
        const uint8_t* kn = ldsk + ks * kHalf + lane * 16;
        const uint8_t* vp = ldsv + vs * kHalf + lane * 16;
        w.refer(g * kPageT, none, cs, half);
        // of a SIMD's two waves the one that has products to feed goes first (3%)
        if (DH < 256) __builtin_amdgcn_s_setprio(2);
        w.template turn<2 * kPieces>(kn, win.at(win.xk, g + 1 - base), vp, xvp, cs, fetch);
        if (DH < 256) __builtin_amdgcn_s_setprio(0);
        xvp = win.at(win.xv, g - base);
        done();
      }
      last();
      w.values(ldsv + vs * kHalf + lane * 16, xvp);
    }
  }
  __syncthreads();
  if (__builtin_expect(active && w.far != 0, 0))
    cache_again<DH>(w, p, b, h, first, min(end, limit), 1, n, cs, lane);
  float l = w.lrun + __shfl_xor(w.lrun, 32, 64);
  if constexpr (PG > 1) {
    // the second group's results to the first, lane by lane
    float* at = reinterpret_cast<float*>(lds) + part_of * kCols * (DH + 2);
    float* mine = at + lane * 4;
    float* top = at + kCols * DH;
    if (group == 1 && active) {
#pragma unroll
      for (int t = 0; t < DT; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          v4f x;
#pragma unroll
          for (int e = 0; e < 4; e++) x[e] = w.o[t][i * 4 + e];
          *reinterpret_cast<v4f*>(mine + (t * 4 + i) * 256) = x;
        }
      top[col] = w.base;
      top[kCols + col] = l;
    }
    __syncthreads();
    if (group == 1) return;
    if (active) {
      const float m2 = top[col], l2 = top[kCols + col], to = fmaxf(w.base, m2);
      const float f = w.base == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(w.base - to);
      const float f2 = m2 == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m2 - to);
      l = l * f + l2 * f2;
#pragma unroll
      for (int t = 0; t < DT; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const v4f x = *reinterpret_cast<const v4f*>(mine + (t * 4 + i) * 256);
#pragma unroll
          for (int e = 0; e < 4; e++)
            w.o[t][i * 4 + e] = w.o[t][i * 4 + e] * f + x[e] * f2;
        }
      w.base = to;
    }
  }
  if (!active) return;

  const float inv = splits > 1 ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
  const size_t to = (size_t)(r0 + ct) * p.ldout + (h * G + c - ct * G) * DH;
  if (splits == 1 && p.out_bf16) {
    // A lane holds four consecutive values of its column at a time, its other half the next
    // four: written as they are, 64 pieces of 8 bytes a store. Whole rows instead, through LDS
    // (16-byte pieces at places that the row turns, so that a column of them meets all banks).
    uint8_t* own = lds + part_of * (PG > 1 ? kCols * (DH + 2) * 4 : kCols * (DH * 2 + 8));
    int64_t* dest = reinterpret_cast<int64_t*>(own + kCols * DH * 2);
    auto place = [&](int row, int piece) {
      return own + row * (DH * 2) + (piece ^ (DH == 64 ? row / 2 % 8 : row % 16)) * 16;
    };
    if (half == 0) dest[col] = c0 + col < cols ? (int64_t)to : -1;
#pragma unroll
    for (int t = 0; t < DT; t++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        typedef __bf16 v4bf __attribute__((ext_vector_type(4)));
        const v4bf x = {(__bf16)(w.o[t][i * 4] * inv), (__bf16)(w.o[t][i * 4 + 1] * inv),
                        (__bf16)(w.o[t][i * 4 + 2] * inv), (__bf16)(w.o[t][i * 4 + 3] * inv)};
        *reinterpret_cast<v4bf*>(place(col, t * 4 + i) + half * 8) = x;
      }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    constexpr int kLanes = DH / 8;  // of a row
    typedef v8bf Out __attribute__((aligned(8)));
#pragma unroll
    for (int r = 0; r < kCols; r += 64 / kLanes) {
      const int row = r + lane / kLanes;
      const v8bf x = *reinterpret_cast<const v8bf*>(place(row, lane % kLanes));
      const int64_t at = dest[row];
      // past the L2, whose lines would be written back at the kernel's end (dh 256, windowed:
      // 30.1 -> 29.2 µs)
      if (at >= 0)
        __builtin_nontemporal_store(
            (Out)x, reinterpret_cast<Out*>(static_cast<__bf16*>(p.out) + at + lane % kLanes * 8));
    }
    return;
  }
  if (c0 + col >= cols) return;
  float* part = nullptr;
  if (splits > 1) {
    const size_t u = ((size_t)b * p.cache.kv_heads + h) * tiles + tile;
    part = p.part + ((u * splits + split) * kCols + col) * kPartRow<DH>;
    if (half == 0) {
      part[DH] = w.base;
      part[DH + 1] = l;
    }
  } else {
    part = static_cast<float*>(p.out) + to;
  }
#pragma unroll
  for (int t = 0; t < DT; t++)
#pragma unroll
    for (int i = 0; i < 4; i++) {
      v4f x;
#pragma unroll
      for (int e = 0; e < 4; e++) x[e] = w.o[t][i * 4 + e] * inv;
      *reinterpret_cast<v4f*>(part + t * 32 + i * 8 + half * 4) = x;
    }
}

// Partial results of a tile's key ranges to its output rows, in range order.
template <int DH>
__global__ __launch_bounds__(256) void cache_join_kernel(CacheAttnArgs p, int tiles, int splits,
                                                         int max_cols) {
  constexpr int LPR = DH / 4;
  const int G = p.heads / p.cache.kv_heads;
  const int u = blockIdx.x;
  const int tile = u % tiles, h = u / tiles % p.cache.kv_heads, b = u / tiles / p.cache.kv_heads;
  const int r0 = p.cu[b], nq = p.cu[b + 1] - r0;
  const int cols = min(nq * G, max_cols), c0 = tile * kCols;
  const int d = threadIdx.x % LPR * 4;
  const int part_cols = min(kCols, max_cols);
  const size_t step = (size_t)part_cols * kPartRow<DH>;
  for (int rr = threadIdx.x / LPR; rr < min(kCols, cols - c0); rr += 256 / LPR) {
    const float* at = p.part + ((size_t)u * splits * part_cols + rr) * kPartRow<DH>;
    float m = -INFINITY, l = 0.0f;
    v4f x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int s = 0; s < splits; s++) {
      const float ms = at[s * step + DH], ls = at[s * step + DH + 1];
      const v4f y = *reinterpret_cast<const v4f*>(at + s * step + d);
      const float to = fmaxf(m, ms);
      const float f = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - to);
      const float g = ms == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(ms - to);
      l = l * f + ls * g;
#pragma unroll
      for (int e = 0; e < 4; e++) x[e] = x[e] * f + y[e] * g;
      m = to;
    }
    x *= l == 0.0f ? 0.0f : 1.0f / l;
    const int cc = c0 + rr, tt = cc / G;
    cache_store4(p, (size_t)(r0 + tt) * p.ldout + (h * G + cc - tt * G) * DH + d, x);
  }
}

static int cache_tiles(int max_q, int heads, int kv_heads) {
  return (int)(((long long)max_q * (heads / kv_heads) + kCols - 1) / kCols);
}
static int cache_part_cols(int max_q, int heads, int kv_heads) {
  return (int)std::min((long long)kCols, (long long)max_q * (heads / kv_heads));
}

// Columns of one kv head that a request may have at most. Up to 32: a workgroup's waves share
// a tile and take pages in turn; more: each wave takes a tile.
static bool cache_by_cols(int max_q, int heads, int kv_heads) {
  return (long long)max_q * (heads / kv_heads) > kCols;
}

static long long cache_pages(int max_q, int max_len, int window, int cols) {
  const long long pages = ((long long)max_len + kPageT - 1) / kPageT;
  if (window <= 0) return pages;
  return std::min(pages, (2LL * window + std::min(max_q, cols)) / kPageT + 2);
}

// Many columns: two tiles or four per workgroup. A page then takes a CU with one workgroup
// 0.62 µs (two tiles) or 1.1 (four), with two of them 1.11 or 2.05 (dh 128), so two tiles are
// faster while they fill the chip at most one and a half times (32 requests of 9 to 70
// rows: 24.9 µs against 28.3), four are by 8% behind that (4096 rows). dh 256 has room for
// one workgroup per CU, 1.0 or 1.6 µs a page, and where enough key ranges of four tiles can be
// made, they fill the chip (2000 rows over 4000: 56 µs against 69).
static bool cache_two_tiles(int batch, int max_q, int heads, int kv_heads, int dh,
                            long long pages) {
  const long long tiles = cache_tiles(max_q, heads, kv_heads), units = (long long)batch * kv_heads;
  if (dh == 256) return units * ((tiles + 3) / 4) * std::max(1LL, pages / 8) <= 128;
  return units * ((tiles + 1) / 2) <= 768;
}

// Key ranges: as many as give the chip's 256 CUs six workgroups each (many columns: one),
// where a range still has a page for every wave (many columns: 16 pages, dh 256: 8). A window
// leaves a tile few pages, and no range of its own for each.
static int cache_ranges(int batch, int max_q, int heads, int kv_heads, int dh, int per_wg,
                        long long pages) {
  const bool cols = cache_by_cols(max_q, heads, kv_heads);
  const long long tiles = cache_tiles(max_q, heads, kv_heads);
  const long long wgs = (long long)batch * kv_heads * ((tiles + per_wg - 1) / per_wg);
  const long long want = cols ? 256 : 1536;
  const bool one = cols && dh == 256;  // a CU has room for one: no second round
  const long long s = wgs > 0 ? (one ? want : want + wgs - 1) / wgs : 1;
  return (int)std::max(1LL, std::min(s, pages / (!cols ? kWaves : one ? 8 : 16)));
}

// Tiles per workgroup and key ranges per tile.
static void cache_split(int batch, int max_q, int max_len, int heads, int kv_heads, int dh,
                        int window, int* per_wg, int* splits) {
  const bool cols = cache_by_cols(max_q, heads, kv_heads);
  const long long pages = cache_pages(max_q, max_len, window, cols ? 4 * kCols : kCols);
  *per_wg = !cols ? 1 : cache_two_tiles(batch, max_q, heads, kv_heads, dh, pages) ? 2 : 4;
  *splits = cache_ranges(batch, max_q, heads, kv_heads, dh, *per_wg, pages);
}

// Few columns: pages past the L2 where those of all requests, of which a cache of `pool` pages
// has no more, could not stay in the memory's own 256 MiB cache. Below, texts that share pages
// find them (512 queries of 4 tokens behind a shared 640: 71 µs, past the L2 80). An upper
// estimate: texts that share, or are shorter than the longest, may read less from a large pool.
bool cache_streams(long long pages, int batch, int pool, int kv_heads, int dh) {
  return std::min(pages * batch, (long long)pool) * kPageT * kv_heads * dh * 2 > 256LL << 20;
}

// For any window: all pages, and four tiles, which never make fewer ranges than two.
size_t cache_attention_floats(int batch, int max_q, int max_len, int heads, int kv_heads, int dh) {
  const int per_wg = cache_by_cols(max_q, heads, kv_heads) ? 4 : 1;
  const int splits = cache_ranges(batch, max_q, heads, kv_heads, dh, per_wg,
                                  cache_pages(max_q, max_len, 0, 0));
  if (splits < 2) return 0;
  return (size_t)batch * kv_heads * cache_tiles(max_q, heads, kv_heads) * splits *
         cache_part_cols(max_q, heads, kv_heads) * (dh + 4);
}

template <int DH>
static hipError_t launch_dh(const CacheAttnArgs& a, hipStream_t s) {
  int per_wg, splits;
  cache_split(a.batch, a.max_q, a.max_len, a.heads, a.cache.kv_heads, DH, a.window, &per_wg,
              &splits);
  const int tiles = cache_tiles(a.max_q, a.heads, a.cache.kv_heads);
  const int max_cols =
      (int)std::min(0x7FFFFFFFLL, (long long)a.max_q * (a.heads / a.cache.kv_heads));
  const int units = a.batch * a.cache.kv_heads;
  const int wgs = (tiles + per_wg - 1) / per_wg;  // of a unit and key range
  const bool few = per_wg > 1 && wgs <= kFewTiles;
  const dim3 grid = few ? dim3((unsigned)units, (unsigned)wgs, (unsigned)splits)
                        : dim3((unsigned)(units * wgs * splits));
  const dim3 block(64 * kWaves);
  const long long pages = cache_pages(a.max_q, a.max_len, a.window, kCols);
#define RH_ATTN(B)                                                                             \
  if (per_wg == 4)                                                                             \
    hipLaunchKernelGGL((cache_attention_cols_kernel<DH, B, 4, 1, 3>), grid, block, 0, s, a,    \
                       tiles, splits, max_cols);                                               \
  else if (per_wg == 2)                                                                        \
    hipLaunchKernelGGL((cache_attention_cols_kernel<DH, B, 2, 2, DH == 64 ? 3 : 2>), grid,     \
                       block, 0, s, a, tiles, splits, max_cols);                               \
  else if (cache_streams(pages, a.batch, a.cache.pages, a.cache.kv_heads, DH))                 \
    hipLaunchKernelGGL((cache_attention_kernel<DH, B, true>), grid, block, 0, s, a, tiles,     \
                       splits, max_cols);                                                      \
  else                                                                                         \
    hipLaunchKernelGGL((cache_attention_kernel<DH, B, false>), grid, block, 0, s, a, tiles,    \
                       splits, max_cols)
  if (a.in_bf16) {
    RH_ATTN(true);
  } else {
    RH_ATTN(false);
  }
#undef RH_ATTN
  if (splits > 1)
    hipLaunchKernelGGL((cache_join_kernel<DH>), dim3(units * tiles), dim3(256), 0, s, a, tiles,
                       splits, max_cols);
  return hipGetLastError();
}

hipError_t launch_cache_attention(const CacheAttnArgs& a, hipStream_t s) {
  switch (a.cache.dh) {
    case 64: return launch_dh<64>(a, s);
    case 128: return launch_dh<128>(a, s);
    case 256: return launch_dh<256>(a, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace rh
