// residual_norm.hip — what stands between two blocks of a layer, in one pass over the rows:
//   s = x_scale x + y_scale gate * post(y),   out = pre(s),
// post and pre each an RMS norm, a layer norm or nothing; s is the residual stream, out the next
// block's input, as fp32 or bf16 rows and/or as e4m3 codes with a scale byte for each 128 values.
//   rms:   v * w / sqrt(mean(v^2) + eps)
//   layer: (v - mean(v)) * w / sqrt(mean((v - mean(v))^2) + eps) + b
// Statistics are fp32 sums over values in registers, the layer norm's variance around its mean; s
// reaches `pre` unrounded, whatever type it is stored in, and codes are those of fp32 values.
// Covers what the model forwards do in passes of their own (Add and the norms, tensor.go:383-389,
// 430-471; Gemma's post-norms, gemma3.go:357,376).
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
    v = slot[k][threadIdx.x % kWaves];
    k++;
    return group_sum<kWaves>(v);
  }
};

enum Type : int { kNone, kF32, kBF16 };

// Eight values; WHOLE: 16-byte aligned, in the row or behind it; else of any alignment (memory
// takes 16 bytes at any address), the row's last ones by themselves.
template <bool WHOLE, Type K>
__device__ __forceinline__ void load_chunk(const void* base, size_t at, int c, int n, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] = 0.0f;
  if constexpr (WHOLE) {
    if (c < n) load_values<8, K == kBF16>(base, at + c, v);
  } else {
    using S = std::conditional_t<K == kBF16, __bf16, float>;
    typedef S W __attribute__((ext_vector_type(16 / sizeof(S)), aligned(sizeof(S))));
    constexpr int kW = 16 / sizeof(S);
    const S* p = static_cast<const S*>(base) + at + c;
    if (c + 8 <= n) {
#pragma unroll
      for (int j = 0; j < 8; j += kW) {
        const W x = *reinterpret_cast<const W*>(p + j);
#pragma unroll
        for (int i = 0; i < kW; i++) v[j + i] = (float)x[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (c + i < n) v[i] = (float)p[i];
    }
  }
}
template <bool WHOLE, Type K>
__device__ __forceinline__ void store_chunk(void* base, size_t at, int c, int n, const float (&v)[8]) {
  if constexpr (WHOLE) {
    if (c < n) store_values<8, K == kBF16>(base, at + c, v);
  } else {
    using S = std::conditional_t<K == kBF16, __bf16, float>;
    typedef S W __attribute__((ext_vector_type(16 / sizeof(S)), aligned(sizeof(S))));
    constexpr int kW = 16 / sizeof(S);
    S* p = static_cast<S*>(base) + at + c;
    if (c + 8 <= n) {
#pragma unroll
      for (int j = 0; j < 8; j += kW) {
        W x;
#pragma unroll
        for (int i = 0; i < kW; i++) x[i] = (S)v[j + i];
        *reinterpret_cast<W*>(p + j) = x;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (c + i < n) p[i] = (S)v[i];
    }
  }
}

// A norm's weights, as the row's chunks.
template <int V, int T, bool WHOLE>
struct NormWeights {
  float w[V][8], b[V][8];
  __device__ __forceinline__ void load(const rh_norm& norm, int n, int t) {
    if (norm.weight) {
#pragma unroll
      for (int e = 0; e < V; e++) load_chunk<WHOLE, kF32>(norm.weight, 0, (t + T * e) * 8, n, w[e]);
    }
    if (norm.bias) {
#pragma unroll
      for (int e = 0; e < V; e++) load_chunk<WHOLE, kF32>(norm.bias, 0, (t + T * e) * 8, n, b[e]);
    }
  }
};

// v normed in place; values past n are zeros before, and anything after.
template <int V, int T, bool WHOLE>
__device__ __forceinline__ void norm_row(float (&v)[V][8], const rh_norm& norm,
                                         const NormWeights<V, T, WHOLE>& by, int n, int t,
                                         RowSum<T>& sum) {
  if (norm.kind == RH_NORM_LAYER) {
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < V; e++)
#pragma unroll
      for (int i = 0; i < 8; i++) s += v[e][i];
    const float mean = sum(s) / (float)n;
#pragma unroll
    for (int e = 0; e < V; e++)
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const int c = (t + T * e) * 8;
        v[e][i] = (WHOLE ? c < n : c + i < n) ? v[e][i] - mean : 0.0f;
      }
  }
  float ss = 0.0f;
#pragma unroll
  for (int e = 0; e < V; e++)
#pragma unroll
    for (int i = 0; i < 8; i++) ss = __builtin_fmaf(v[e][i], v[e][i], ss);
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
  const long long row = r0 + (long long)blockIdx.x * kRows + threadIdx.x / T;
  const int used = p.used ? min(*p.used, p.m) : p.m;
  if (row >= used) return;  // whole waves; a workgroup of one row as a whole
  const int n = p.n;
  RowSum<T> sum{s_sum};
  float v[V][8], w[V][8], g[V][8];
  NormWeights<V, T, WHOLE> post, pre;
#pragma unroll
  for (int e = 0; e < V; e++)
    load_chunk<WHOLE, X>(p.x, (size_t)row * p.ldx, (t + T * e) * 8, n, v[e]);
  if constexpr (Y != kNone) {
#pragma unroll
    for (int e = 0; e < V; e++)
      load_chunk<WHOLE, Y>(p.y, (size_t)row * p.ldy, (t + T * e) * 8, n, w[e]);
    if (p.gate) {
#pragma unroll
      for (int e = 0; e < V; e++)
        load_chunk<WHOLE, kF32>(p.gate, (size_t)row * p.ldg, (t + T * e) * 8, n, g[e]);
    }
    post.load(p.post, n, t);
  }
  if constexpr (V == 1) pre.load(p.pre, n, t);
  if constexpr (Y != kNone) {
    if (p.post.kind != RH_NORM_NONE) norm_row<V, T, WHOLE>(w, p.post, post, n, t, sum);
    if (p.gate) {
#pragma unroll
      for (int e = 0; e < V; e++)
#pragma unroll
        for (int i = 0; i < 8; i++) w[e][i] *= g[e][i];
    }
  }
#pragma unroll
  for (int e = 0; e < V; e++) {
    const int c = (t + T * e) * 8;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      if constexpr (Y != kNone) v[e][i] = __builtin_fmaf(v[e][i], p.x_scale, w[e][i] * p.y_scale);
      else v[e][i] *= p.x_scale;
      if (WHOLE ? c >= n : c + i >= n) v[e][i] = 0.0f;  // what a norm left past the row
    }
    if (p.sum) store_chunk<WHOLE, X>(p.sum, (size_t)row * p.ldsum, c, n, v[e]);
  }
  if constexpr (V > 1) pre.load(p.pre, n, t);  // registers: late
  if (p.pre.kind != RH_NORM_NONE) norm_row<V, T, WHOLE>(v, p.pre, pre, n, t, sum);
#pragma unroll
  for (int e = 0; e < V; e++) {
    const int c = (t + T * e) * 8;
    if (p.out) {
      if (p.out_bf16) store_chunk<WHOLE, kBF16>(p.out, (size_t)row * p.ldout, c, n, v[e]);
      else store_chunk<WHOLE, kF32>(p.out, (size_t)row * p.ldout, c, n, v[e]);
    }
    if (p.qa) {
      uint32_t u = 0;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        if (WHOLE ? c >= n : c + i >= n) v[e][i] = 0.0f;
        u = max(u, finite_abs_bits(v[e][i]));
      }
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
        typedef int v2i __attribute__((ext_vector_type(2)));
        v2i q;
        q[0] = fp8_pack4(v[e][0] * f, v[e][1] * f, v[e][2] * f, v[e][3] * f);
        q[1] = fp8_pack4(v[e][4] * f, v[e][5] * f, v[e][6] * f, v[e][7] * f);
        __builtin_nontemporal_store(q, reinterpret_cast<v2i*>(p.qa + (size_t)row * p.ldq + c));
        if (t % 16 == 0)
          p.sa[fp8_scale_at((int)row, c / kFp8Block, (p.m + 127) / 128)] = (uint8_t)x;
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

template <bool WHOLE>
static void launch_part(const ResidualArgs& a, int r0, int rows, hipStream_t s) {
  if (a.n <= 512) launch_rows<1, 64, WHOLE>(a, r0, rows, s);
  else if (a.n <= 1024) launch_rows<1, 128, WHOLE>(a, r0, rows, s);
  else if (a.n <= 2048) launch_rows<1, 256, WHOLE>(a, r0, rows, s);
  else if (a.n <= 4096) launch_rows<1, 512, WHOLE>(a, r0, rows, s);
  else if (a.n <= 8192) launch_rows<1, 1024, WHOLE>(a, r0, rows, s);
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
