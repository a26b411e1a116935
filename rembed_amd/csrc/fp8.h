// fp8.h — e4m3 values with power-of-two scales, shared by the 8-bit linears
// and the 8-bit cache.
//
// A block of values (128 of an activation row, 128 x 128 of a weight, 64
// tokens of a cached head) is held as e4m3 codes times 2^(x - 127) for one
// byte x, the smallest with which the block's largest magnitude is at most 448,
// e4m3's largest. Multiplying by a power of two is exact, so every code is the
// e4m3 value nearest to its input and no scale is ever rounded; against a scale
// of max / 448 a power of two costs nothing but up to one bit of the range below
// the block's maximum (2^-13 of it is still a normal number). CDNA4's
// v_mfma_scale_* takes these bytes as they are (E8M0), one for each row and 32 k.
#pragma once

#include "context.h"
#include "gemm_common.h"

namespace rh {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v2f __attribute__((ext_vector_type(2)));

// The byte x of the smallest 2^(x - 127) with |max| <= 448 * 2^(x - 127), from
// the bits of a finite |max|: 448 = 1.75 * 2^8. 0 for magnitudes below.
__host__ __device__ __forceinline__ int fp8_exponent(uint32_t absmax_bits) {
  const int e = (int)(absmax_bits >> 23) - 8 + ((absmax_bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return e < 0 ? 0 : e;
}
// 2^(127 - x) for x = 0..253: what a value is multiplied by to get its code.
__device__ __forceinline__ float fp8_inverse(int x) {
  return __uint_as_float((uint32_t)(254 - x) << 23);
}
// |v|'s bits, 0 for infinities and NaN (they set no scale).
__device__ __forceinline__ uint32_t finite_abs_bits(float v) {
  const uint32_t u = __float_as_uint(v) & 0x7FFFFFFFu;
  return u < 0x7F800000u ? u : 0u;
}

// Four values to four e4m3 codes, rounded to nearest even; |v| <= 448, and
// infinities and NaN become NaN codes.
__device__ __forceinline__ int fp8_pack4(float a, float b, float c, float d) {
#if defined(__HIP_DEVICE_COMPILE__)
  // the first conversion keeps half of a word that the second one writes: any word
  int w;
  asm("" : "=v"(w) : "v"(a));
  w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, w, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
#else
  return 0;
#endif
}
__device__ __forceinline__ void fp8_unpack4(int w, float (&v)[4]) {
#if defined(__HIP_DEVICE_COMPILE__)
  const v2f lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false);
  const v2f hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
  v[0] = lo[0];
  v[1] = lo[1];
  v[2] = hi[0];
  v[3] = hi[1];
#endif
}
// What four values (|v| <= 448) leave over after rounding to `codes`, times 16
// and as e4m3 again: codes + 2^-4 * rest is v to 8 bits (exactly, where v has
// no more than bf16's 8) from 2^-6 on, off by up to 2^-14 below. 16 v - 16 code is exact, fused or not.
__device__ __forceinline__ int fp8_rest4(int codes, float a, float b, float c, float d) {
#if defined(__HIP_DEVICE_COMPILE__)
  const v2f lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes, 16.0f, false);
  const v2f hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes, 16.0f, true);
  return fp8_pack4(__builtin_fmaf(a, 16.0f, -lo[0]), __builtin_fmaf(b, 16.0f, -lo[1]),
                   __builtin_fmaf(c, 16.0f, -hi[0]), __builtin_fmaf(d, 16.0f, -hi[1]));
#else
  return 0;
#endif
}

// D += A.B over 64 (128) e4m3 k of 32 x 32 (16 x 16) rows; ea / eb: the scale
// bytes at byte SA / SB of each lane's word. Checked on the GPU: k = 0..31 are
// bytes 0..15 of the lanes of both halves (32x32x64), scaled by the words of
// lanes 0..31, k = 32..63 bytes 16..31, scaled by lanes 32..63. Here a row's
// scale is the same for all k of an instruction, so every lane passes its row's
// byte and any order of k that A and B share will do. A sum's products keep 13
// bits below the largest of their group, whatever is done afterwards: 1.5e-5 of
// the result on normal values, far inside bf16's 2^-8 but not fp32's 2^-24.
template <int SA = 0, int SB = 0>
__device__ __forceinline__ v16f mfma_fp8_32(const v8i& a, const v8i& b, const v16f& c, int ea,
                                            int eb) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, SA, ea, SB, eb);
#else
  return c;
#endif
}
template <int SA = 0, int SB = 0>
__device__ __forceinline__ v4f mfma_fp8_16(const v8i& a, const v8i& b, const v4f& c, int ea,
                                           int eb) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, SA, ea, SB, eb);
#else
  return c;
#endif
}
__device__ __forceinline__ v8i join8(const v4i& a, const v4i& b) {
  return (v8i){a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}

// Scale bytes of rows (activations or packed weight rows) for the GEMM: block kb
// of row r lies at byte ((kb * groups + r / 128) * 32 + r % 32) * 4 + r % 128 / 32,
// groups = ceil(rows / 128), so one word serves a lane's row in each of the four
// 32-row tiles of a group.
__host__ __device__ __forceinline__ size_t fp8_scale_at(int r, int kb, int groups) {
  return (((size_t)kb * groups + r / 128) * 32 + r % 32) * 4 + r % 128 / 32;
}

// ---- launchers (gemm_fp8.hip) -------------------------------------------------------
// a: fp32 (a_bf16 0) or bf16 rows [m][lda] -> codes [m][ldq] (ldq = round_up(k, 128),
// zeros past k) and their scale bytes (fp8_scale_at)
hipError_t launch_quantize_rows_fp8(const void* a, int a_bf16, int lda, int m, int k, uint8_t* qa,
                                    int ldq, uint8_t* sa, hipStream_t s);
// w [n][k] on the device -> codes [..][kp] and scale bytes of blocks of 128 x 128; half: -1, or
// 0 / 1 for the gate / up rows of an interleaved pair. *bad becomes the place of the first value
// that is not finite (its block is then left out); the caller sets it to all ones.
hipError_t launch_pack_fp8(const float* w, int k, int n, uint8_t* img, int kp, uint8_t* exps,
                           int groups, int half, unsigned long long* bad, hipStream_t s);
struct GemmFp8Args {
  const uint8_t* A;   // codes [M][lda]
  int lda;            // bytes, round_up(K, 128)
  const uint8_t* sa;  // scale bytes of A's rows
  const uint8_t* B;   // codes [Np][ldb], zero outside [N][K]
  int ldb;            // bytes, a multiple of 128
  const uint8_t* sb;  // scale bytes of B's rows, Np / 128 groups
  int M, N, K, Np;
  const float* bias;  // [N] or null
  void* out;          // f32 or bf16 [M][ldo]; gated: N / 2 columns
  int ldo;            // elements, a multiple of 4
  int out_bf16;
  int act;
  int tile_group;
};
// src: fp32 or bf16 rows to make e4m3 on the way (A and sa unused), where
// gemm_fp8_takes_rows; null: A and sa.
bool gemm_fp8_takes_rows(int M, int N, int K, const void* a, int a_bf16, int lda);
hipError_t launch_gemm_fp8(const GemmFp8Args& a, const void* src, int src_bf16, int ld_src,
                           hipStream_t s);

// ---- shared checks (capi_fp8.cpp) ------------------------------------------------------
int check_cache(const rh_kv_cache* c);
// Whether m rows of `wa` bytes, `sa` apart, share bytes with m rows of `wb`, `sb` apart.
bool rows_overlap(const void* a, size_t wa, size_t sa, const void* b, size_t wb, size_t sb, int m);

// ---- launchers (cache.hip, cache_attention.hip) ----------------------------------------
struct CachePlanArgs {
  const int32_t *past, *fresh;
  int batch;
  const int32_t* free_pages;
  int n_free;
  int32_t* table;
  int ldt;
  int32_t *cu, *blocks, *lens;
  int64_t* slots;
  int32_t* pos;
  int rows;
  int32_t* status;
};
hipError_t launch_cache_plan(const CachePlanArgs& a, hipStream_t s);
struct CacheAppendArgs {
  rh_kv_cache cache;
  const void* kv;
  int in_bf16, ldkv, k_off, v_off;
  const int32_t *cu, *blocks;
  const int64_t* slots;
  int batch, rows;
};
hipError_t launch_cache_append(const CacheAppendArgs& a, hipStream_t s);
struct CacheAttnArgs {
  const void* q;
  int in_bf16, ldq, q_off;
  rh_kv_cache cache;
  const int32_t* table;
  int ldt;
  const int32_t *cu, *lens;
  int batch, max_q, max_len, heads;
  float scale;
  int causal, window;
  void* out;
  int out_bf16, ldout;
  float* part;  // partial results of split key ranges (cache_attention_floats)
};
// Floats that the partial results of split key ranges take.
size_t cache_attention_floats(int batch, int max_q, int max_len, int heads, int kv_heads, int dh);
hipError_t launch_cache_attention(const CacheAttnArgs& a, hipStream_t s);

}  // namespace rh
