// residual_norm.hip — what stands between two blocks of a layer, in one pass over the rows:
//   s = x_scale x + y_scale gate * post(y),   out = pre(s),
// post and pre each an RMS norm, a layer norm or nothing; s is the residual stream, out the next
// block's input, as fp32 or bf16 rows and/or as e4m3 codes with a scale byte for each 128 values.
//   rms:   v * w / sqrt(mean(v^2) + eps)
//   layer: (v - mean(v)) * w / sqrt(mean((v - mean(v))^2) + eps) + b
// Statistics are fp32 sums over values in registers, the layer norm's variance around its mean; s
// reaches `pre` unrounded, whatever type it is stored in, and codes are those of fp32 values.
// Every row is read and written once: 8192 rows of 4096, 235 MB, take 48 µs, 4.9 TB/s; 2111 of 768
// 4.9, of which a launch is 4.0; odd rows (1213 of 1001) 6.1. Rows of over 8192 values have two chunks
// a thread, whose registers (86 to 113) leave a CU one workgroup: nothing else is loaded while a row is
// summed, and 2048 rows of 16384 (235 MB, e4m3 out) take 56 µs, 4.2 TB/s, 1024 fp32 rows of 12288 with a
// norm on both sides (201 MB) 50, 4.0 TB/s.
// Covers what the model forwards do in passes of their own (Add and the norms, tensor.go:383-387,
// 433-471; Gemma's post-norms, gemma3.go:357,376).
#include "rowops.h"

#include <algorithm>
#include <type_traits>

namespace rh {

// T threads a row (a wave, or the workgroup), V chunks of eight consecutive values each: chunk e of
// thread t is values 8 (t + T e) .. + 7, so 16 lanes have a block of 128. Rows and weights are
// all asked for at once, before anything is summed: a row's time is one latency of the memory, its
// reductions (at most four, a barrier each where a row has several waves) and its stores, and
// whole lines leave past the L2.
template <int T>
struct RowSum {
  static constexpr int kWaves = T / 64;
  float (*slot)[kWaves];  // of the workgroup: a place for each wave, for each sum of a row
  int k = 0;
  __device__ __forceinline__ float operator()(float v) {
    v = group_sum<64>(v);
    if constexpr (T == 64) return v;
    if ((threadIdx.x & 63) == 0) slot[k][threadIdx.x >> 6] = v;
    __syncthreads();
    if constexpr (kWaves & (kWaves - 1)) {
      v = slot[k][0];
#pragma unroll
      for (int w = 1; w < kWaves; w++) v += slot[k][w];
    } else {
      v = group_sum<kWaves>(slot[k][threadIdx.x % kWaves]);
    }
    k++;
    return v;
  }
};

enum Type : int { kNone, kF32, kBF16 };

// A thread's eight values: WHOLE: from column c on, 16-byte aligned. Else rows of any length and
// alignment (memory takes 16 bytes at any address): the row's last chunk begins `twice` columns
// early, so that it ends with the row; what it shares with the chunk before is computed and stored
// by both, alike, and summed by that one. Threads behind the row (not `here`) read the row's last
// values as well, and neither sum nor store them. Rows of under eight values are taken one by one.
template <bool WHOLE>
struct Chunk {
  int from, twice, n;
  bool here;
  Chunk() = default;
  __device__ __forceinline__ Chunk(int c, int n) : from(min(c, max(n - 8, 0))), n(n), here(c < n) {
    twice = here ? c - from : 8;
  }
  __device__ __forceinline__ bool counts(int i) const { return i >= twice && i < n; }
  // a sum over the values that count, of x(value)
  template <class F>
  __device__ __forceinline__ float over(const float (&v)[8], float s, F&& add) const {
    if constexpr (WHOLE) {
      float own = s;
#pragma unroll
      for (int i = 0; i < 8; i++) own = add(own, v[i]);
      return here ? own : s;
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) s = add(s, counts(i) ? v[i] : 0.0f);
      return s;
    }
  }
  template <Type K>
  __device__ __forceinline__ void load(const void* base, size_t at, float (&v)[8]) const {
    if constexpr (WHOLE) {
      load_values<8, K == kBF16>(base, at + from, v);
    } else {
      using S = std::conditional_t<K == kBF16, __bf16, float>;
      constexpr int kW = 16 / sizeof(S);
      typedef S W __attribute__((ext_vector_type(kW), aligned(sizeof(S))));
      const S* p = static_cast<const S*>(base) + at + from;
      if (n >= 8) {
#pragma unroll
        for (int j = 0; j < 8; j += kW) {
          const W x = *reinterpret_cast<const W*>(p + j);
#pragma unroll
          for (int i = 0; i < kW; i++) v[j + i] = (float)x[i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = i < n ? (float)p[i < n ? i : 0] : 0.0f;
      }
    }
  }
  template <Type K>
  __device__ __forceinline__ void store(void* base, size_t at, const float (&v)[8]) const {
    if (!here) return;
    if constexpr (WHOLE) {
      store_values<8, K == kBF16>(base, at + from, v);
    } else {
      using S = std::conditional_t<K == kBF16, __bf16, float>;
      constexpr int kW = 16 / sizeof(S);
      typedef S W __attribute__((ext_vector_type(kW), aligned(sizeof(S))));
      S* p = static_cast<S*>(base) + at + from;
      if (n >= 8) {
#pragma unroll
        for (int j = 0; j < 8; j += kW) {
          W x;
#pragma unroll
          for (int i = 0; i < kW; i++) x[i] = (S)v[j + i];
          __builtin_nontemporal_store(x, reinterpret_cast<W*>(p + j));
        }
      } else {
#pragma unroll
        for (int i = 0; i < 7; i++)
          if (i < n) p[i] = (S)v[i];
      }
    }
  }
};

// A norm's weights, as the row's chunks.
template <int V, bool WHOLE>
struct NormWeights {
  float w[V][8], b[V][8];
  __device__ __forceinline__ void load(const rh_norm& norm, const Chunk<WHOLE>* at) {
    if (norm.weight) {
#pragma unroll
      for (int e = 0; e < V; e++) at[e].template load<kF32>(norm.weight, 0, w[e]);
    }
    if (norm.bias) {
#pragma unroll
      for (int e = 0; e < V; e++) at[e].template load<kF32>(norm.bias, 0, b[e]);
    }
  }
};

// v normed in place.
template <int V, int T, bool WHOLE>
__device__ __forceinline__ void norm_row(float (&v)[V][8], const rh_norm& norm,
                                         const NormWeights<V, WHOLE>& by, const Chunk<WHOLE>* at,
                                         int n, RowSum<T>& sum) {
  if (norm.kind == RH_NORM_LAYER) {
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < V; e++) s = at[e].over(v[e], s, [](float a, float x) { return a + x; });
    const float mean = sum(s) / (float)n;
#pragma unroll
    for (int e = 0; e < V; e++)
#pragma unroll
      for (int i = 0; i < 8; i++) v[e][i] -= mean;
  }
  float ss = 0.0f;
#pragma unroll
  for (int e = 0; e < V; e++)
    ss = at[e].over(v[e], ss, [](float a, float x) { return __builtin_fmaf(x, x, a); });
  const float inv = inverse_root(sum(ss) / (float)n + norm.eps);
#pragma unroll
  for (int e = 0; e < V; e++)
#pragma unroll
    for (int i = 0; i < 8; i++) v[e][i] *= inv;
  if (norm.weight) {
#pragma unroll
    for (int e = 0; e < V; e++)
#pragma unroll
      for (int i = 0; i < 8; i++) v[e][i] *= by.w[e][i];
  }
  if (norm.bias) {
#pragma unroll
    for (int e = 0; e < V; e++)
#pragma unroll
      for (int i = 0; i < 8; i++) v[e][i] += by.b[e][i];
  }
}

template <int V, int T, bool WHOLE, Type X, Type Y>
__global__ __launch_bounds__(T == 64 ? 256 : T) void residual_norm_kernel(ResidualArgs p, int r0) {
  constexpr int kRows = T == 64 ? 4 : 1;
  __shared__ float s_sum[4][RowSum<T>::kWaves];
  const int t = threadIdx.x % T;
  // of the wave, and so a scalar; unsigned: behind the last row it may pass 2^31
  const unsigned row = (unsigned)r0 + blockIdx.x * kRows +
                       (T == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x / 64) : 0);
  const int used = p.used ? min(*p.used, p.m) : p.m;
  if (row >= (unsigned)max(used, 0)) return;  // whole waves; a workgroup of one row as a whole
  const int n = p.n;
  RowSum<T> sum{s_sum};
  Chunk<WHOLE> at[V];
#pragma unroll
  for (int e = 0; e < V; e++) at[e] = Chunk<WHOLE>((t + T * e) * 8, n);
  float v[V][8], w[V][8], g[V][8];
  NormWeights<V, WHOLE> post, pre;
#pragma unroll
  for (int e = 0; e < V; e++) at[e].template load<X>(p.x, (size_t)row * p.ldx, v[e]);
  if constexpr (Y != kNone) {
#pragma unroll
    for (int e = 0; e < V; e++) at[e].template load<Y>(p.y, (size_t)row * p.ldy, w[e]);
    if (p.gate) {
#pragma unroll
      for (int e = 0; e < V; e++) at[e].template load<kF32>(p.gate, (size_t)row * p.ldg, g[e]);
    }
    post.load(p.post, at);
  }
  if constexpr (V == 1) pre.load(p.pre, at);
  // a chunk's shared values may be another wave's to store, where an output lies on its input
  if constexpr (!WHOLE && T > 64) __syncthreads();
  if constexpr (Y != kNone) {
    if (p.post.kind != RH_NORM_NONE) norm_row<V, T, WHOLE>(w, p.post, post, at, n, sum);
    if (p.gate) {
#pragma unroll
      for (int e = 0; e < V; e++)
#pragma unroll
        for (int i = 0; i < 8; i++) w[e][i] *= g[e][i];
    }
  }
  if constexpr (Y != kNone) {
    if (p.y_scale != 1.0f) {
#pragma unroll
      for (int e = 0; e < V; e++)
#pragma unroll
        for (int i = 0; i < 8; i++) w[e][i] *= p.y_scale;
    }
  }
#pragma unroll
  for (int e = 0; e < V; e++) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      if constexpr (Y != kNone) v[e][i] = __builtin_fmaf(v[e][i], p.x_scale, w[e][i]);
      else v[e][i] *= p.x_scale;
    }
    if (p.sum) at[e].template store<X>(p.sum, (size_t)row * p.ldsum, v[e]);
  }
  if constexpr (V > 1) pre.load(p.pre, at);  // registers: late
  if (p.pre.kind != RH_NORM_NONE) norm_row<V, T, WHOLE>(v, p.pre, pre, at, n, sum);
#pragma unroll
  for (int e = 0; e < V; e++) {
    const int c = (t + T * e) * 8;
    if (p.out) {
      if (p.out_bf16) at[e].template store<kBF16>(p.out, (size_t)row * p.ldout, v[e]);
      else at[e].template store<kF32>(p.out, (size_t)row * p.ldout, v[e]);
    }
    if (p.qa) {
      uint32_t u = 0;
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (WHOLE || at[e].counts(i)) u = max(u, __float_as_uint(v[e][i]) & 0x7FFFFFFFu);
      if (u >= 0x7F800000u) {  // infinities and NaN set no scale
        u = 0;
#pragma unroll
        for (int i = 0; i < 8; i++)
          if (WHOLE || at[e].counts(i)) u = max(u, finite_abs_bits(v[e][i]));
      }
      if (!at[e].here) u = 0;
#if defined(__HIP_DEVICE_COMPILE__)
#define RH_ROR(n) u = max(u, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, 0x120 + n, 0xF, 0xF, true))
      RH_ROR(8);
      RH_ROR(4);
      RH_ROR(2);
      RH_ROR(1);
#undef RH_ROR
#endif
      if (c < p.ldq) {  // a multiple of 128: whole groups of 16 lanes
        const int x = fp8_exponent(u);
        const float f = fp8_inverse(x);
        uint64_t q = (uint32_t)fp8_pack4(v[e][4] * f, v[e][5] * f, v[e][6] * f, v[e][7] * f);
        q = q << 32 | (uint32_t)fp8_pack4(v[e][0] * f, v[e][1] * f, v[e][2] * f, v[e][3] * f);
        if constexpr (!WHOLE) {  // and zeros behind the row
          q >>= 8 * (at[e].twice & 7);
          if (n < 8) q &= (1ull << 8 * n) - 1;
        }
        if (!at[e].here) q = 0;
        __builtin_nontemporal_store(q, reinterpret_cast<uint64_t*>(p.qa + (size_t)row * p.ldq + c));
        if (t % 16 == 0)
          p.sa[fp8_scale_at((int)row, c / kFp8Block, (p.m - 1) / 128 + 1)] = (uint8_t)x;
      }
    }
  }
}

// 16-byte loads of every row and weight, and stores as wide.
static bool by_chunks(const ResidualArgs& a) {
  if (a.n % 8) return false;
  auto fits = [](const void* q, int ld, int bf16) {
    return !q || ((uintptr_t)q % 16 == 0 && ld % (bf16 ? 8 : 4) == 0);
  };
  return fits(a.x, a.ldx, a.x_bf16) && fits(a.y, a.ldy, a.y_bf16) &&
         fits(a.sum, a.ldsum, a.x_bf16) && fits(a.out, a.ldout, a.out_bf16) &&
         fits(a.gate, a.ldg, 0) && fits(a.post.weight, 0, 0) && fits(a.post.bias, 0, 0) &&
         fits(a.pre.weight, 0, 0) && fits(a.pre.bias, 0, 0);
}

template <int V, int T, bool WHOLE>
static void launch_rows(const ResidualArgs& a, int r0, int rows, hipStream_t s) {
  constexpr int kThreads = T == 64 ? 256 : T;
  const dim3 grid(ceil_div(rows, kThreads / T)), block(kThreads);
#define RH_RN(X, Y) \
  hipLaunchKernelGGL((residual_norm_kernel<V, T, WHOLE, X, Y>), grid, block, 0, s, a, r0)
  if (a.x_bf16) {
    if (!a.y) RH_RN(kBF16, kNone);
    else if (a.y_bf16) RH_RN(kBF16, kBF16);
    else RH_RN(kBF16, kF32);
  } else {
    if (!a.y) RH_RN(kF32, kNone);
    else if (a.y_bf16) RH_RN(kF32, kBF16);
    else RH_RN(kF32, kF32);
  }
#undef RH_RN
}

// The fewest threads of these that have eight values each: waves that sit out a row's end cost
// their share (2272 rows of 5520 values: 32.5 µs with 1024 threads, 26.8 with 768; 8192 of 2560:
// 37.6 with 512, 35.0 with 384).
template <bool WHOLE>
static void launch_part(const ResidualArgs& a, int r0, int rows, hipStream_t s) {
  const int waves = (a.n + 511) / 512;
  if (waves <= 1) launch_rows<1, 64, WHOLE>(a, r0, rows, s);
  else if (waves <= 2) launch_rows<1, 128, WHOLE>(a, r0, rows, s);
  else if (waves <= 3) launch_rows<1, 192, WHOLE>(a, r0, rows, s);
  else if (waves <= 4) launch_rows<1, 256, WHOLE>(a, r0, rows, s);
  else if (waves <= 6) launch_rows<1, 384, WHOLE>(a, r0, rows, s);
  else if (waves <= 8) launch_rows<1, 512, WHOLE>(a, r0, rows, s);
  else if (waves <= 12) launch_rows<1, 768, WHOLE>(a, r0, rows, s);
  else if (waves <= 16) launch_rows<1, 1024, WHOLE>(a, r0, rows, s);
  else launch_rows<2, 1024, WHOLE>(a, r0, rows, s);
}

hipError_t launch_residual_norm(const ResidualArgs& a, hipStream_t s) {
  const bool whole = by_chunks(a);
  constexpr int kMost = 1 << 21;  // a launch holds fewer than 2^32 threads
  for (int r0 = 0; r0 < a.m; r0 += std::min(kMost, a.m - r0)) {
    const int rows = std::min(kMost, a.m - r0);
    if (whole) launch_part<true>(a, r0, rows, s);
    else launch_part<false>(a, r0, rows, s);
  }
  return hipGetLastError();
}

}  // namespace rh
