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

namespace rh {

// T threads a row (a wave, or the workgroup's four), V chunks of eight consecutive values each:
// chunk e of thread t is values 8 (t + T e) .. + 7, so 16 lanes have a block of 128.
template <int T>
struct RowSum {
  float (*slot)[4];  // of the workgroup: a place for each wave, for each sum of a row
  int k = 0;
  __device__ __forceinline__ float operator()(float v) {
    v = group_sum<64>(v);
    if constexpr (T == 64) return v;
    if ((threadIdx.x & 63) == 0) slot[k][threadIdx.x >> 6] = v;
    __syncthreads();
    v = (slot[k][0] + slot[k][1]) + (slot[k][2] + slot[k][3]);
    k++;
    return v;
  }
};

template <bool VEC, bool BF16>
__device__ __forceinline__ void load_chunk(const void* base, size_t at, int c, int n, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] = 0.0f;
  if constexpr (VEC) {
    if (c < n) load_values<8, BF16>(base, at + c, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (c + i < n)
        v[i] = BF16 ? (float)static_cast<const __bf16*>(base)[at + c + i]
                    : static_cast<const float*>(base)[at + c + i];
  }
}
template <bool VEC, bool BF16>
__device__ __forceinline__ void store_chunk(void* base, size_t at, int c, int n, const float (&v)[8]) {
  if constexpr (VEC) {
    if (c < n) store_values<8, BF16>(base, at + c, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (c + i < n) {
        if constexpr (BF16) static_cast<__bf16*>(base)[at + c + i] = (__bf16)v[i];
        else static_cast<float*>(base)[at + c + i] = v[i];
      }
  }
}

// v normed in place; values past n are zeros before, and anything after.
template <int V, int T, bool VEC>
__device__ __forceinline__ void norm_row(float (&v)[V][8], const rh_norm& norm, int n, int t,
                                         RowSum<T>& sum) {
  float mean = 0.0f, ss = 0.0f;
  if (norm.kind == RH_NORM_LAYER) {
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < V; e++)
#pragma unroll
      for (int i = 0; i < 8; i++) s += v[e][i];
    mean = sum(s) / (float)n;
  }
#pragma unroll
  for (int e = 0; e < V; e++)
#pragma unroll
    for (int i = 0; i < 8; i++) {
      v[e][i] -= mean;
      const bool in = VEC ? (t + T * e) * 8 < n : (t + T * e) * 8 + i < n;
      ss += in ? v[e][i] * v[e][i] : 0.0f;
    }
  const float inv = inverse_root(sum(ss) / (float)n + norm.eps);
#pragma unroll
  for (int e = 0; e < V; e++) {
    const int c = (t + T * e) * 8;
    float w[8], b[8];
    if (norm.weight) load_chunk<VEC, false>(norm.weight, 0, c, n, w);
    if (norm.bias) load_chunk<VEC, false>(norm.bias, 0, c, n, b);
#pragma unroll
    for (int i = 0; i < 8; i++) {
      v[e][i] *= inv;
      if (norm.weight) v[e][i] *= w[i];
      if (norm.bias) v[e][i] += b[i];
    }
  }
}

template <int V, int T, bool VEC>
__global__ __launch_bounds__(256) void residual_norm_kernel(ResidualArgs p, int r0) {
  __shared__ float s_sum[4][4];
  const int t = threadIdx.x % T;
  const long long row = r0 + (long long)blockIdx.x * (256 / T) + threadIdx.x / T;
  const int used = p.used ? min(*p.used, p.m) : p.m;
  if (row >= used) return;  // whole waves; with T = 256 the whole workgroup
  const int n = p.n;
  RowSum<T> sum{s_sum};
  float v[V][8], w[V][8];
#pragma unroll
  for (int e = 0; e < V; e++) {
    const int c = (t + T * e) * 8;
    if (p.x_bf16) load_chunk<VEC, true>(p.x, (size_t)row * p.ldx, c, n, v[e]);
    else load_chunk<VEC, false>(p.x, (size_t)row * p.ldx, c, n, v[e]);
  }
  if (p.y) {
#pragma unroll
    for (int e = 0; e < V; e++) {
      const int c = (t + T * e) * 8;
      if (p.y_bf16) load_chunk<VEC, true>(p.y, (size_t)row * p.ldy, c, n, w[e]);
      else load_chunk<VEC, false>(p.y, (size_t)row * p.ldy, c, n, w[e]);
    }
    if (p.post.kind != RH_NORM_NONE) norm_row<V, T, VEC>(w, p.post, n, t, sum);
#pragma unroll
    for (int e = 0; e < V; e++) {
      float g[8];
      if (p.gate)
        load_chunk<VEC, false>(p.gate, (size_t)row * p.ldg, (t + T * e) * 8, n, g);
#pragma unroll
      for (int i = 0; i < 8; i++) {
        if (p.gate) w[e][i] *= g[i];
        v[e][i] = __builtin_fmaf(v[e][i], p.x_scale, w[e][i] * p.y_scale);
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; e++)
#pragma unroll
      for (int i = 0; i < 8; i++) v[e][i] *= p.x_scale;
  }
#pragma unroll
  for (int e = 0; e < V; e++) {
    const int c = (t + T * e) * 8;
#pragma unroll
    for (int i = 0; i < 8; i++)  // post's bias reaches past the row
      if (VEC ? c >= n : c + i >= n) v[e][i] = 0.0f;
    if (p.sum) {
      if (p.x_bf16) store_chunk<VEC, true>(p.sum, (size_t)row * p.ldsum, c, n, v[e]);
      else store_chunk<VEC, false>(p.sum, (size_t)row * p.ldsum, c, n, v[e]);
    }
  }
  if (p.pre.kind != RH_NORM_NONE) norm_row<V, T, VEC>(v, p.pre, n, t, sum);
#pragma unroll
  for (int e = 0; e < V; e++) {
    const int c = (t + T * e) * 8;
    if (p.out) {
      if (p.out_bf16) store_chunk<VEC, true>(p.out, (size_t)row * p.ldout, c, n, v[e]);
      else store_chunk<VEC, false>(p.out, (size_t)row * p.ldout, c, n, v[e]);
    }
    if (p.qa) {
      uint32_t u = 0;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        if (VEC ? c >= n : c + i >= n) v[e][i] = 0.0f;
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

hipError_t launch_residual_norm(const ResidualArgs& a, hipStream_t s) {
  if (a.m <= 0) return hipSuccess;
  const bool vec = by_chunks(a);
  const bool wide = a.n > 1024 || (a.n > 512 && a.m < 1024);  // a workgroup for a row
  const int chunks = ceil_div(a.n, wide ? 2048 : 512);
  const int per = wide ? 1 : 4, most = 1 << 23;  // a launch holds fewer than 2^32 threads
  for (int r0 = 0; r0 < a.m; r0 += std::min(most * per, a.m - r0)) {
    const int rows = std::min(most * per, a.m - r0);
    const dim3 grid(ceil_div(rows, per)), block(256);
#define RH_RN(V, T)                                                                              \
  {                                                                                              \
    if (vec) hipLaunchKernelGGL((residual_norm_kernel<V, T, true>), grid, block, 0, s, a, r0);   \
    else hipLaunchKernelGGL((residual_norm_kernel<V, T, false>), grid, block, 0, s, a, r0);      \
  }
    if (wide) {
      if (chunks <= 1) RH_RN(1, 256)
      else if (chunks <= 2) RH_RN(2, 256)
      else if (chunks <= 4) RH_RN(4, 256)
      else RH_RN(8, 256)
    } else {
      if (chunks <= 1) RH_RN(1, 64)
      else RH_RN(2, 64)
    }
#undef RH_RN
  }
  return hipGetLastError();
}

}  // namespace rh
