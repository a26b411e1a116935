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
// exactly: the residue of rounding 8 significant bits to 4 has at most 4. P is
// split the same way (off by 2^-8 of itself, as bf16 is), so two products of the
// double-rate fp8 instruction take the place of one bf16 product and no key or
// value is ever converted.
#include "fp8.h"

#include <algorithm>

namespace rh {

constexpr int kPageT = RH_CACHE_BLOCK;
constexpr int kCols = 32;    // query columns per tile
constexpr int kWaves = 4;    // per workgroup
// P^T is 2^4 * exp(score - reference): the reference moves when a score passes it
// by more than 2^4, so codes stay within 2^8 < 448.
constexpr float kHead = 4.0f;

// Visible keys [klo, khi] of a query at position i of n; none: klo = khi = 2^30.
__device__ __forceinline__ void cache_key_range(const CacheAttnArgs& p, int i, int n, int& klo,
                                                int& khi) {
  khi = n - 1;
  klo = 0;
  if (p.causal) khi = min(khi, i);
  if (p.window > 0) {
    khi = min(khi, i + p.window - 1);
    klo = max(klo, i - p.window + 1);
  }
  if (khi < klo) klo = khi = 1 << 30;
}

// The columns' codes and scale bytes: lane (column, half) holds values
// 64 s + 32 half .. + 31 of step s, as K's pieces do.
template <int KS, bool BF16>
__device__ __forceinline__ void cache_load_q(const void* q, size_t at, int half, v8i (&hi)[KS],
                                             v8i (&lo)[KS], int& xh, int& xl) {
  float v[KS][32];
  uint32_t m = 0;
#pragma unroll
  for (int s = 0; s < KS; s++)
#pragma unroll
    for (int e = 0; e < 32; e += 8) {
      const size_t o = at + s * 64 + half * 32 + e;
      if constexpr (BF16) {
        const v8bf x = *reinterpret_cast<const v8bf*>(static_cast<const __bf16*>(q) + o);
#pragma unroll
        for (int i = 0; i < 8; i++) v[s][e + i] = (float)x[i];
      } else {
        const v4f a = *reinterpret_cast<const v4f*>(static_cast<const float*>(q) + o);
        const v4f b = *reinterpret_cast<const v4f*>(static_cast<const float*>(q) + o + 4);
#pragma unroll
        for (int i = 0; i < 8; i++) v[s][e + i] = i < 4 ? a[i] : b[i - 4];
      }
#pragma unroll
      for (int i = 0; i < 8; i++) m = max(m, finite_abs_bits(v[s][e + i]));
    }
  m = max(m, (uint32_t)__shfl_xor((int)m, 32, 64));
  xh = fp8_exponent(m);
  xl = max(xh - 4, 0);
  const float f = fp8_inverse(xh);
#pragma unroll
  for (int s = 0; s < KS; s++)
#pragma unroll
    for (int w = 0; w < 8; w++) {
      const float a = v[s][4 * w] * f, b = v[s][4 * w + 1] * f, c = v[s][4 * w + 2] * f,
                  d = v[s][4 * w + 3] * f;
      hi[s][w] = fp8_pack4(a, b, c, d);
      lo[s][w] = xh >= 4 ? fp8_rest4(hi[s][w], a, b, c, d) : 0;
    }
}

// One wave's running state of its 32 columns, and a page's step.
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
    for (int t = 0; t < DT; t++)
#pragma unroll
      for (int e = 0; e < 16; e++) o[t][e] = 0.0f;
    mref = -INFINITY;
    lrun = 0.0f;
  }

  // kf[s][t]: keys 32t.., step s; vf[t]: values' columns 32t.., all 64 tokens.
  // key0: the page's first position; n: tokens in the cache.
  __device__ __forceinline__ void page(const v8i (&kf)[KS][2], v8i (&vf)[DT], int xk, int xv,
                                       int key0, int n, float cs, int half) {
    v16f sc[2];
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int e = 0; e < 16; e++) sc[t][e] = 0.0f;
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
    if (key0 + kPageT > n) {
      // nothing was written behind the last token: no NaN code may meet a zero P
#pragma unroll
      for (int w = 0; w < 8; w++) {
        const int left = n - (key0 + w / 4 * 32 + w % 4 * 8 + half * 4);
        const int keep = left >= 4 ? -1 : left <= 0 ? 0 : (1 << (8 * left)) - 1;
#pragma unroll
        for (int t = 0; t < DT; t++) vf[t][w] &= keep;
      }
    }
    float smax = -INFINITY;
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int e = 0; e < 16; e++) smax = fmaxf(smax, sc[t][e]);
    smax = fmaxf(smax, __shfl_xor(smax, 32, 64));
    const float mloc = smax * cs;
    const bool up = mloc > mref + kHead;  // -inf + 4 = -inf: the first visible key moves it
    if (__any(up)) {
      float alpha = 1.0f;
      if (up) {
        alpha = __builtin_amdgcn_exp2f(mref - mloc);
        mref = mloc;
      }
      lrun *= alpha;
#pragma unroll
      for (int t = 0; t < DT; t++)
#pragma unroll
        for (int e = 0; e < 16; e++) o[t][e] *= alpha;
    }
    // a column with no visible key yet: every p = 2^(-inf) = 0
    const float m = mref == -INFINITY ? 0.0f : mref - kHead;
    v8i ph, pl;
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int w = 0; w < 4; w++) {
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
          x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][4 * w + e], cs, -m));
          lrun += x[e];
        }
        ph[4 * t + w] = fp8_pack4(x[0], x[1], x[2], x[3]);
        pl[4 * t + w] = fp8_rest4(ph[4 * t + w], x[0], x[1], x[2], x[3]);
      }
#pragma unroll
    for (int t = 0; t < DT; t++) {
      o[t] = mfma_fp8_32(vf[t], ph, o[t], xv, 127);
      o[t] = mfma_fp8_32(vf[t], pl, o[t], xv, 123);
    }
  }
};

// A page's fragments of one head: 1 KiB pieces, 16 bytes a lane.
template <int DH>
__device__ __forceinline__ void cache_fetch(const uint8_t* k, const uint8_t* v, int lane,
                                            v8i (&kf)[DH / 64][2], v8i (&vf)[DH / 32]) {
  const v4i* kp = reinterpret_cast<const v4i*>(k) + lane;
  const v4i* vp = reinterpret_cast<const v4i*>(v) + lane;
#pragma unroll
  for (int s = 0; s < DH / 64; s++)
#pragma unroll
    for (int t = 0; t < 2; t++)
      kf[s][t] = join8(kp[((s * 2 + t) * 2) * 64], kp[((s * 2 + t) * 2 + 1) * 64]);
#pragma unroll
  for (int t = 0; t < DH / 32; t++) vf[t] = join8(vp[t * 2 * 64], vp[(t * 2 + 1) * 64]);
}

// Workgroup -> (request, kv head, tile of columns, key range). Units of one (request,
// kv head) read the same pages: their workgroups are dealt to one XCD (workgroup w
// runs on XCD w % 8) and share its L2.
__device__ __forceinline__ bool cache_unit(const CacheAttnArgs& p, int tiles, int splits, int& b,
                                           int& h, int& tile, int& split) {
  const int w = blockIdx.x, nv = tiles * splits;
  const int t = w >> 3, v = t % nv, u = (t / nv) * 8 + (w & 7);
  if (u >= p.batch * p.cache.kv_heads) return false;
  b = u / p.cache.kv_heads;
  h = u % p.cache.kv_heads;
  tile = v / splits;
  split = v % splits;
  return true;
}

template <int DH, bool BF16>
__global__ __launch_bounds__(64 * kWaves) void cache_attention_kernel(CacheAttnArgs p, int tiles,
                                                                      int splits, int part_cols) {
  constexpr int KS = DH / 64, DT = DH / 32, kStride = DH + 4;
  __shared__ __attribute__((aligned(16))) float s_o[kCols * kStride];
  __shared__ float s_m[kWaves][kCols], s_l[kWaves][kCols];
  int b, h, tile, split;
  if (!cache_unit(p, tiles, splits, b, h, tile, split)) return;
  const int G = p.heads / p.cache.kv_heads;
  const int r0 = p.cu[b], nq = p.cu[b + 1] - r0;
  const int cols = nq * G, c0 = tile * kCols;
  if (c0 >= cols) return;
  const int n = max(0, min(p.lens[b], p.ldt * kPageT));
  const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = min(c0 + col, cols - 1);
  const int pos0 = n - nq;  // position of the first new token
  const float cs = p.scale * 1.44269504088896341f;

  CacheTile<DH> w;
  cache_load_q<KS, BF16>(p.q, (size_t)(r0 + c / G) * p.ldq + p.q_off + (h * G + c % G) * DH, half,
                         w.qh, w.ql, w.xh, w.xl);
  w.clear();
  cache_key_range(p, pos0 + c / G, n, w.klo, w.khi);

  // the tile's pages, this split's share of them
  int lo = 0, hi = (n + kPageT - 1) / kPageT;
  {
    const int i0 = pos0 + c0 / G, i1 = pos0 + (min(c0 + kCols, cols) - 1) / G;
    if (p.causal) hi = min(hi, i1 < 0 ? 0 : i1 / kPageT + 1);
    if (p.window > 0) {
      lo = max(0, i0 - p.window + 1) / kPageT;
      const long long last = (long long)i1 + p.window - 1;
      if (last < n) hi = min(hi, last < 0 ? 0 : (int)(last / kPageT) + 1);
    }
  }
  const int each = (max(0, hi - lo) + splits - 1) / splits;
  const int first = lo + split * each, end = min(hi, first + each);
  for (int g = first + wave; g < end; g += kWaves) {
    const int pg = p.table[(size_t)b * p.ldt + g];
    if (pg < 0 || pg >= p.cache.pages) continue;  // no such page: no keys
    const size_t unit = (size_t)pg * p.cache.kv_heads + h;
    v8i kf[KS][2], vf[DT];
    cache_fetch<DH>(p.cache.k + unit * (kPageT * DH), p.cache.v + unit * (kPageT * DH), lane, kf,
                    vf);
    w.page(kf, vf, p.cache.k_exp[unit], p.cache.v_exp[unit], g * kPageT, n, cs, half);
  }

  // join the waves: columns' references and sums, then O in wave order
  float l = w.lrun + __shfl_xor(w.lrun, 32, 64);
  if (half == 0) {
    s_m[wave][col] = w.mref;
    s_l[wave][col] = l;
  }
  __syncthreads();
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < kWaves; i++) m = fmaxf(m, s_m[i][col]);
  const float mine = w.mref == -INFINITY ? (l == 0.0f ? 0.0f : l) : __builtin_amdgcn_exp2f(w.mref - m);
  for (int i = 0; i < kWaves; i++) {
    if (wave == i) {
#pragma unroll
      for (int t = 0; t < DT; t++)
#pragma unroll
        for (int q4 = 0; q4 < 4; q4++) {
          v4f* at = reinterpret_cast<v4f*>(s_o + col * kStride + t * 32 + q4 * 8 + half * 4);
          v4f x = i == 0 ? v4f{0.0f, 0.0f, 0.0f, 0.0f} : *at;
#pragma unroll
          for (int e = 0; e < 4; e++) x[e] += w.o[t][q4 * 4 + e] * mine;
          *at = x;
        }
    }
    __syncthreads();
  }
  // a row of the tile per LPR threads, 4 values each
  constexpr int LPR = DH / 4, RPP = 64 * kWaves / LPR;
  const int d = threadIdx.x % LPR * 4;
  for (int rr = threadIdx.x / LPR; rr < min(kCols, cols - c0); rr += RPP) {
    float mm = -INFINITY, ll = 0.0f;
#pragma unroll
    for (int i = 0; i < kWaves; i++) mm = fmaxf(mm, s_m[i][rr]);
#pragma unroll
    for (int i = 0; i < kWaves; i++) {
      const float f = s_m[i][rr] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(s_m[i][rr] - mm);
      ll += s_l[i][rr] * f;  // a wave with no visible key has a sum of 0 (or NaN)
    }
    v4f x = *reinterpret_cast<const v4f*>(s_o + rr * kStride + d);
    const int cc = c0 + rr;
    if (splits > 1) {
      const size_t u = ((size_t)b * p.cache.kv_heads + h) * tiles + tile;
      float* at = p.part + (u * splits + split) * (size_t)part_cols * (DH + 2) +
                  (size_t)rr * (DH + 2);
      typedef float v2 __attribute__((ext_vector_type(2)));
      *reinterpret_cast<v2*>(at + d) = (v2){x[0], x[1]};
      *reinterpret_cast<v2*>(at + d + 2) = (v2){x[2], x[3]};
      if (d == 0) {
        at[DH] = mm;
        at[DH + 1] = ll;
      }
      continue;
    }
    const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
    x *= inv;
    const size_t to = (size_t)(r0 + cc / G) * p.ldout + (h * G + cc % G) * DH + d;
    if (p.out_bf16) {
      typedef __bf16 v4bf __attribute__((ext_vector_type(4)));
      *reinterpret_cast<v4bf*>(static_cast<__bf16*>(p.out) + to) =
          (v4bf){(__bf16)x[0], (__bf16)x[1], (__bf16)x[2], (__bf16)x[3]};
    } else {
      *reinterpret_cast<v4f*>(static_cast<float*>(p.out) + to) = x;
    }
  }
}

// Partial results of a tile's key ranges to its output rows, in range order.
template <int DH>
__global__ __launch_bounds__(256) void cache_join_kernel(CacheAttnArgs p, int tiles, int splits,
                                                         int part_cols) {
  constexpr int LPR = DH / 2;
  const int G = p.heads / p.cache.kv_heads;
  const int u = blockIdx.x;
  const int tile = u % tiles, h = u / tiles % p.cache.kv_heads, b = u / tiles / p.cache.kv_heads;
  const int r0 = p.cu[b], nq = p.cu[b + 1] - r0;
  const int cols = nq * G, c0 = tile * kCols;
  const int d = threadIdx.x % LPR * 2;
  typedef float v2 __attribute__((ext_vector_type(2)));
  for (int rr = threadIdx.x / LPR; rr < min(kCols, cols - c0); rr += 256 / LPR) {
    const float* at = p.part + ((size_t)u * splits * part_cols + rr) * (DH + 2);
    const size_t step = (size_t)part_cols * (DH + 2);
    float m = -INFINITY, l = 0.0f;
    for (int s = 0; s < splits; s++) m = fmaxf(m, at[s * step + DH]);
    v2 x = {0.0f, 0.0f};
    for (int s = 0; s < splits; s++) {
      const float ms = at[s * step + DH];
      const float f = ms == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(ms - m);
      l += at[s * step + DH + 1] * f;
      const v2 y = *reinterpret_cast<const v2*>(at + s * step + d);
      x[0] += y[0] * f;
      x[1] += y[1] * f;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const int cc = c0 + rr;
    const size_t to = (size_t)(r0 + cc / G) * p.ldout + (h * G + cc % G) * DH + d;
    if (p.out_bf16) {
      typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
      *reinterpret_cast<v2bf*>(static_cast<__bf16*>(p.out) + to) =
          (v2bf){(__bf16)(x[0] * inv), (__bf16)(x[1] * inv)};
    } else {
      *reinterpret_cast<v2*>(static_cast<float*>(p.out) + to) = (v2){x[0] * inv, x[1] * inv};
    }
  }
}

static int cache_tiles(int max_q, int heads, int kv_heads) {
  return (int)(((long long)max_q * (heads / kv_heads) + kCols - 1) / kCols);
}
static int cache_part_cols(int max_q, int heads, int kv_heads) {
  return (int)std::min((long long)kCols, (long long)max_q * (heads / kv_heads));
}

// Key ranges: as many as give the chip's 256 CUs four workgroups each, where a range
// still has a page for every wave.
void cache_attention_plan(int batch, int max_q, int max_len, int heads, int kv_heads, int dh,
                          int* splits, size_t* part_floats) {
  const long long tiles = cache_tiles(max_q, heads, kv_heads);
  const long long units = (long long)batch * kv_heads * tiles;
  const long long pages = ((long long)max_len + kPageT - 1) / kPageT;
  long long s = units > 0 ? (1024 + units - 1) / units : 1;
  s = std::max(1LL, std::min(s, pages / kWaves));
  *splits = (int)s;
  *part_floats = s > 1 ? (size_t)units * s * cache_part_cols(max_q, heads, kv_heads) * (dh + 2) : 0;
}

template <int DH>
static hipError_t launch_dh(const CacheAttnArgs& a, hipStream_t s) {
  int splits;
  size_t part;
  cache_attention_plan(a.batch, a.max_q, a.max_len, a.heads, a.cache.kv_heads, DH, &splits, &part);
  const int tiles = cache_tiles(a.max_q, a.heads, a.cache.kv_heads);
  const int pc = cache_part_cols(a.max_q, a.heads, a.cache.kv_heads);
  const int units = a.batch * a.cache.kv_heads;
  const dim3 grid((unsigned)((units + 7) / 8 * 8 * tiles * splits)), block(64 * kWaves);
  if (a.in_bf16)
    hipLaunchKernelGGL((cache_attention_kernel<DH, true>), grid, block, 0, s, a, tiles, splits, pc);
  else
    hipLaunchKernelGGL((cache_attention_kernel<DH, false>), grid, block, 0, s, a, tiles, splits, pc);
  if (splits > 1)
    hipLaunchKernelGGL((cache_join_kernel<DH>), dim3(units * tiles), dim3(256), 0, s, a, tiles,
                       splits, pc);
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
