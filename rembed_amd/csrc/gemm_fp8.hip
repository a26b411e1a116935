// gemm_fp8.hip — e4m3 activations x e4m3 weights for gfx950, a power-of-two scale
// for each 128 values of an activation row and each 128 x 128 block of the weight:
//   y[r][n] = act(sum_b 2^(ea[r][b] + ew[n][b]) sum_{k in b} qa[r][k] qw[n][k] + bias[n]).
//
// The fourth mode beside the fp32, weight-only int8 and full-int8 linears
// (applyDense, internal/model/bert.go:282-301); no counterpart in the reference.
// The scale bytes are the matrix instruction's own (fp8.h), so the main loop is
// loads and v_mfma_scale_f32_32x32x64_f8f6f4 alone, one accumulation over all of K.
#include "fp8.h"

#include <algorithm>
#include <type_traits>

namespace rh {

// ---- rows to e4m3 -----------------------------------------------------------------
// A wave takes 512 values of a row, 16 lanes a block of 128: eight values a lane,
// their maximum over the 16 lanes by row rotations, codes as one 8-byte store. One
// read and one write of every value bound it: 8192 x 4096 of bf16, 101 MB, take 21 µs, the
// 4.9 TB/s of a large copy.
template <bool BF16, bool VEC>
__global__ __launch_bounds__(256) void quantize_rows_fp8_kernel(const void* a, int lda, int m,
                                                                int k, uint8_t* qa, int ldq,
                                                                uint8_t* sa, int per_row,
                                                                int r0) {
  const int wave = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int row = wave / per_row;
  if (row >= m - r0) return;
  const int r = r0 + row;
  const int c = (wave - row * per_row) * 512 + lane * 8;
  float v[8];
  const size_t at = (size_t)r * lda + c;
  if constexpr (VEC) {  // k % 8 == 0, rows 16-byte aligned
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = 0.0f;
    if (c < k) {
      if constexpr (BF16) {
        const v8bf x = *reinterpret_cast<const v8bf*>(static_cast<const __bf16*>(a) + at);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = (float)x[e];
      } else {
        const v4f x = *reinterpret_cast<const v4f*>(static_cast<const float*>(a) + at);
        const v4f y = *reinterpret_cast<const v4f*>(static_cast<const float*>(a) + at + 4);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = e < 4 ? x[e] : y[e - 4];
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) {
      v[e] = 0.0f;
      if (c + e < k)
        v[e] = BF16 ? (float)static_cast<const __bf16*>(a)[at + e]
                    : static_cast<const float*>(a)[at + e];
    }
  }
  uint32_t u = 0;
#pragma unroll
  for (int e = 0; e < 8; e++) u = max(u, finite_abs_bits(v[e]));
#if defined(__HIP_DEVICE_COMPILE__)
#define RH_ROR(n) u = max(u, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, 0x120 + n, 0xF, 0xF, true))
  RH_ROR(8);
  RH_ROR(4);
  RH_ROR(2);
  RH_ROR(1);
#undef RH_ROR
#endif
  if (c >= ldq) return;  // ldq is a multiple of 128: whole groups of 16 lanes
  const int x = fp8_exponent(u);
  const float f = fp8_inverse(x);
  typedef int v2i __attribute__((ext_vector_type(2)));
  v2i w;
  w[0] = fp8_pack4(v[0] * f, v[1] * f, v[2] * f, v[3] * f);
  w[1] = fp8_pack4(v[4] * f, v[5] * f, v[6] * f, v[7] * f);
  *reinterpret_cast<v2i*>(qa + (size_t)r * ldq + c) = w;
  if (lane % 16 == 0) sa[fp8_scale_at(r, c / kFp8Block, (m + 127) / 128)] = (uint8_t)x;
}

hipError_t launch_quantize_rows_fp8(const void* a, int a_bf16, int lda, int m, int k, uint8_t* qa,
                                    int ldq, uint8_t* sa, hipStream_t s) {
  if (m <= 0) return hipSuccess;
  const int per_row = (ldq - 1) / 512 + 1;  // ldq may be the last multiple of 128 below 2^31
  const bool vec = k % 8 == 0 && lda % 8 == 0 && ((uintptr_t)a & 15) == 0;
  // a launch holds fewer than 2^32 threads
  const int each = std::max(1, (1 << 25) / per_row);
  for (int r0 = 0; r0 < m; r0 += std::min(each, m - r0)) {
    const int rows = std::min(each, m - r0);
    const dim3 grid((unsigned)(((long long)rows * per_row + 3) / 4)), block(256);
#define RH_Q(B, V)                                                                              \
  hipLaunchKernelGGL((quantize_rows_fp8_kernel<B, V>), grid, block, 0, s, a, lda, m, k, qa, ldq, \
                     sa, per_row, r0)
    if (a_bf16) {
      if (vec) RH_Q(true, true);
      else RH_Q(true, false);
    } else {
      if (vec) RH_Q(false, true);
      else RH_Q(false, false);
    }
  }
#undef RH_Q
  return hipGetLastError();
}

// ---- weights to e4m3 ----------------------------------------------------------------
// A workgroup takes one 128 x 128 block, 16 words of four consecutive values a thread. half: -1,
// or which of a gated pair's matrices this is, whose rows interleave in groups of kGluGroup.
// bad: the first value that is not finite, by its place in the matrix.
__global__ __launch_bounds__(256) void pack_fp8_kernel(const float* w, int k, int n, uint8_t* img,
                                                       int kp, uint8_t* exps, int groups, int half,
                                                       unsigned long long* bad) {
  constexpr int kWords = kFp8Block * kFp8Block / 4 / 256;
  __shared__ uint32_t s_top[4];
  const int tid = threadIdx.x, kb = blockIdx.x;
  const int c = kb * kFp8Block + tid % 32 * 4, r0 = blockIdx.y * kFp8Block + tid / 32;
  float v[kWords][4];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kWords; i++) {
    const int r = r0 + i * 8;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const size_t at = (size_t)r * k + c + e;
      v[i][e] = r < n && c + e < k ? w[at] : 0.0f;
      const uint32_t u = __float_as_uint(v[i][e]) & 0x7FFFFFFFu;
      if (u >= 0x7F800000u) atomicMin(bad, (unsigned long long)at);
      top = max(top, u);
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
  if (tid % 64 == 0) s_top[tid / 64] = top;
  __syncthreads();
  top = max(max(s_top[0], s_top[1]), max(s_top[2], s_top[3]));
  if (top >= 0x7F800000u) return;  // refused
  const int x = fp8_exponent(top);
  const float f = fp8_inverse(x);
#pragma unroll
  for (int i = 0; i < kWords; i++) {
    const int r = r0 + i * 8;
    if (r >= n) break;
    const int to = half < 0 ? r : (r / kGluGroup * 2 + half) * kGluGroup + r % kGluGroup;
    *reinterpret_cast<int*>(img + (size_t)to * kp + c) =
        fp8_pack4(v[i][0] * f, v[i][1] * f, v[i][2] * f, v[i][3] * f);
    if (tid % 32 == 0) exps[fp8_scale_at(to, kb, groups)] = (uint8_t)x;
  }
}

hipError_t launch_pack_fp8(const float* w, int k, int n, uint8_t* img, int kp, uint8_t* exps,
                           int groups, int half, unsigned long long* bad, hipStream_t s) {
  hipLaunchKernelGGL(pack_fp8_kernel,
                     dim3((unsigned)ceil_div(k, kFp8Block), (unsigned)ceil_div(n, kFp8Block)),
                     dim3(256), 0, s, w, k, n, img, kp, exps, groups, half, bad);
  return hipGetLastError();
}

// act(gate) * up. SiLU and the tanh GELU, x / (1 + e^-z), on the hardware's exponential and
// reciprocal, each within an ulp: about 2^-22 of the value where the products before them
// are off by 2^-16 and a bf16 result rounds at 2^-8; expf and a division take 50
// instructions a value, a third of a short-K tile's time.
__device__ __forceinline__ float fp8_glu(float g, float u, int act) {
  if (act == ACT_GEGLU_ERF) return gelu_avx2(g) * u;
  const float z = act == ACT_SWIGLU
                      ? g
                      : 1.5957691216057308f * __builtin_fmaf(0.044715f * g * g, g, g);
  return g * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * z)) * u;
}

__device__ __forceinline__ void fp8_store4(const GemmFp8Args& p, int row, int col, const v4f& v) {
  typedef __bf16 v4bf __attribute__((ext_vector_type(4)));
  const size_t at = (size_t)row * p.ldo + col;
  if (p.out_bf16)
    *reinterpret_cast<v4bf*>(static_cast<__bf16*>(p.out) + at) =
        (v4bf){(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
  else
    *reinterpret_cast<v4f*>(static_cast<float*>(p.out) + at) = v;
}

// ---- GEMM ---------------------------------------------------------------------------
// The weights are the products' rows and the activations their columns, so a lane holds four
// consecutive outputs of one row at a time (gated: gates in lanes 0..31, their ups in
// 32..63, which one exchange of halves brings together). Per 32 rows a wave finishes them in
// registers, parks them in LDS as they will be stored and writes whole rows, 16 bytes a lane.
template <int WM, int WN, int TM, int TN, bool GLU, bool BF16>
__device__ __forceinline__ void fp8_rows_out(const GemmFp8Args& p, v16f (&acc)[TM][TN],
                                             uint8_t* own, int row0, int col0, int lane) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int kCols = GLU ? WN / 2 : WN, kEach = BF16 ? 2 : 4;
  constexpr int kRow = kCols * kEach + 16;  // bytes; 16 rows apart by 4 mod 64 banks
  typedef __bf16 v4bf __attribute__((ext_vector_type(4)));
  const int fr = lane & 31, fg = lane >> 5;
#pragma unroll
  for (int i = 0; i < TM; i++) {
    uint8_t* mine = own + fr * kRow;
    auto park = [&](int at, const v4f& v) {
      if constexpr (BF16)
        *reinterpret_cast<v4bf*>(mine + at * 2) =
            (v4bf){(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
      else
        *reinterpret_cast<v4f*>(mine + at * 4) = v;
    };
#pragma unroll
    for (int j = 0; j < TN; j++)
#pragma unroll
      for (int q = 0; q < 4; q += GLU ? 2 : 1) {
        v4f v;
        if constexpr (GLU) {
          typedef unsigned v2u __attribute__((ext_vector_type(2)));
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const v2u x = __builtin_bit_cast(
                v2u, __builtin_amdgcn_permlane32_swap(__float_as_uint(acc[i][j][q * 4 + e]),
                                                      __float_as_uint(acc[i][j][q * 4 + 4 + e]),
                                                      false, false));
            v[e] = fp8_glu(__uint_as_float(x[0]), __uint_as_float(x[1]), p.act);
          }
          park(j * 16 + q * 4 + fg * 4, v);
        } else {
          const int col = j * 32 + q * 8 + fg * 4;
          v4f bs = {0.0f, 0.0f, 0.0f, 0.0f};
          if (p.bias && col0 + col < p.N) bs = *reinterpret_cast<const v4f*>(p.bias + col0 + col);
#pragma unroll
          for (int e = 0; e < 4; e++) v[e] = acc[i][j][q * 4 + e] + bs[e];
          if (p.act == ACT_GELU) {
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = gelu_avx2(v[e]);
          }
          park(col, v);
        }
      }
    wait_lgkmcnt0();
    __builtin_amdgcn_wave_barrier();
    constexpr int kL = kCols * kEach / 16, kR = 64 / kL;  // lanes of a row, rows at once
    const int l = lane % kL, to = (GLU ? col0 / 2 : col0) + l * (16 / kEach);
#pragma unroll
    for (int k = 0; k < 32; k += kR) {
      const int r = k + lane / kL, row = row0 + i * 32 + r;
      const v4i x = *reinterpret_cast<const v4i*>(own + r * kRow + l * 16);
      typedef v4i Out __attribute__((aligned(8)));
      if (row >= p.M || to >= (GLU ? p.N / 2 : p.N)) continue;
      Out* at = reinterpret_cast<Out*>(static_cast<uint8_t*>(p.out) +
                                       ((size_t)row * p.ldo + to) * kEach);
      // past the L2, whose lines would be written back at the kernel's end (8192 x 4096 x 4096
      // with its quantizer 136.8 -> 132.7 µs); the small tile's pieces of lines stay in it
      // (300 x 640 x 640 6.5 µs, past it 7.0)
      if constexpr (WN >= 64) __builtin_nontemporal_store((Out)x, at);
      else *at = x;
    }
    __builtin_amdgcn_wave_barrier();
  }
#endif
}

template <int WM, int WN, int TM, int TN>
__device__ __forceinline__ void fp8_epilogue(const GemmFp8Args& p, v16f (&acc)[TM][TN],
                                             uint8_t* lds, int row0, int col0, int wave, int wm,
                                             int wn, int lane) {
  uint8_t* own = lds + wave * 32 * (WN + 4) * 4;
  const int r = row0 + wm * WM, c = col0 + wn * WN;
  if (is_glu(p.act)) {
    if (p.out_bf16) fp8_rows_out<WM, WN, TM, TN, true, true>(p, acc, own, r, c, lane);
    else fp8_rows_out<WM, WN, TM, TN, true, false>(p, acc, own, r, c, lane);
  } else {
    if (p.out_bf16) fp8_rows_out<WM, WN, TM, TN, false, true>(p, acc, own, r, c, lane);
    else fp8_rows_out<WM, WN, TM, TN, false, false>(p, acc, own, r, c, lane);
  }
}

// One row tile's products with all column tiles; the scale bytes' places are constants of the
// instruction.
template <int I, int TN, int J = 0>
__device__ __forceinline__ void fp8_cols(v16f (&acc)[TN], const v8i& a, const v8i (&b)[TN], int ea,
                                         int eb) {
  acc[J] = mfma_fp8_32<J, I>(b[J], a, acc[J], eb, ea);
  if constexpr (J + 1 < TN) fp8_cols<I, TN, J + 1>(acc, a, b, ea, eb);
}
template <int TM, int TN>
__device__ __forceinline__ void fp8_row(v16f (&acc)[TM][TN], const v8i& a, const v8i (&b)[TN],
                                        int i, int ea, int eb) {
  if (i == 0) fp8_cols<0>(acc[0], a, b, ea, eb);
  if constexpr (TM > 1)
    if (i == 1) fp8_cols<1>(acc[1], a, b, ea, eb);
  if constexpr (TM > 2)
    if (i == 2) fp8_cols<2>(acc[2], a, b, ea, eb);
  if constexpr (TM > 3)
    if (i == 3) fp8_cols<3>(acc[3], a, b, ea, eb);
}

// BM x BN tile of 2 x WGN waves, K in stages of 128 bytes (one scale block), an
// NS-slot ring filled by global_load_lds; the stage's scale words come the same
// way, behind its codes. What bounds it are LDS and the matrix cores alike: a stage of 256 x 256
// reads 192 KB of fragments and takes in 64 KB, 2048 cycles at 128 bytes each, as its products
// do (128 x 256: 1400 and 1024). 8192 x 4096 x 4096 takes 112 µs, 2.45 PFLOP/s, where the card's
// library product takes 110; four waves of 128 x 128, which read a third less, 19 more than this,
// because one wave a SIMD hides less than two.
template <int BM, int BN, int NS, int WGN>
__global__ __launch_bounds__(128 * WGN) void gemm_fp8_kernel(GemmFp8Args p) {
  constexpr int NT = 128 * WGN, BK = 128, CPR = BK / 16;
  constexpr int WM = BM / 2, WN = BN / WGN, TM = WM / 32, TN = WN / 32;
  constexpr int kA = BM * BK, kB = BN * BK, kScale = 256, kStage = kA + kB + 2 * kScale;
  constexpr int LA = kA / (NT * 16), LB = kB / (NT * 16), kLoads = LA + LB + 1;
  constexpr int kEpi = 2 * WGN * 32 * (WN + 4) * 4;
  static_assert(BM >= 64 && BN >= 64 && BM <= 256 && BN <= 256, "scale words");
  static_assert(WM % 32 == 0 && WN % 32 == 0 && (WM <= 128 && WN <= 128), "a wave's scale words");
  static_assert(NS * kStage <= 160 * 1024 && NS * kStage >= kEpi, "LDS");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[NS * kStage];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WGN, wn = wave % WGN;
  const int tiles_n = (p.N + BN - 1) / BN;
  int rb, cb;
  tile_origin(xcd_remap(blockIdx.x, gridDim.x), (p.M + BM - 1) / BM, tiles_n, p.tile_group, rb,
              cb);
  const int row0 = rb * BM, col0 = cb * BN;
  const int nk = (p.K + BK - 1) / BK;

  // rows past M read row M - 1 (their outputs are not stored); B's rows are
  // padded to a multiple of 256
  const uint8_t* asrc[LA];
#pragma unroll
  for (int j = 0; j < LA; j++) {
    const int slot = (wave * LA + j) * 64 + lane, r = slot / CPR, gr = row0 + r;
    asrc[j] = p.A + (size_t)(gr < p.M ? gr : p.M - 1) * p.lda + stage_slot_chunk<BK>(r, slot % CPR) * 16;
  }
  const uint8_t* bsrc[LB];
#pragma unroll
  for (int j = 0; j < LB; j++) {
    const int slot = (wave * LB + j) * 64 + lane, r = slot / CPR;
    bsrc[j] = p.B + (size_t)(col0 + r) * p.ldb + stage_slot_chunk<BK>(r, slot % CPR) * 16;
  }
  // scale words: even waves bring A's, odd waves B's; a lane's word is row
  // group lane / 32, clamped to the last one
  const int ga = (p.M + 127) / 128, gb = p.Np / 128;
  const bool odd = wave & 1;
  const int groups = odd ? gb : ga, g0 = (odd ? col0 : row0) / 128;
  const uint8_t* ssrc = (odd ? p.sb : p.sa) + (size_t)(min(g0 + lane / 32, groups - 1) * 128 + lane % 32 * 4);
  const size_t sstep = (size_t)groups * 128;
  const int wrow = row0 % 128 + wm * WM, wcol = col0 % 128 + wn * WN;  // within the words

  auto issue = [&](int kt, int slot) {
    uint8_t* s = lds + slot * kStage;
#pragma unroll
    for (int j = 0; j < LA; j++) lds_dma16(asrc[j] + kt * BK, s + (wave * LA + j) * 1024);
#pragma unroll
    for (int j = 0; j < LB; j++) lds_dma16(bsrc[j] + kt * BK, s + kA + (wave * LB + j) * 1024);
#if defined(__HIP_DEVICE_COMPILE__)
    __builtin_amdgcn_global_load_lds(ssrc + kt * sstep, s + kA + kB + (odd ? kScale : 0), 4, 0, 0);
#endif
  };
  // Fragment addresses: chunk 4 step + 2 part + fg of a row lies at slot chunk ^ (r ^ r >> 3) % 8,
  // and a row tile further (32 rows) that mask changes by 4, as a step further does. So four
  // addresses serve every fragment of an operand, the rest is offsets.
  const int fr = lane & 31, fg = lane >> 5;
  int fa[2][2], fb[2][2];
#pragma unroll
  for (int st = 0; st < 2; st++)
#pragma unroll
    for (int pt = 0; pt < 2; pt++) {
      fa[st][pt] = lds_off(wm * WM + fr, 4 * st + 2 * pt + fg);
      fb[st][pt] = kA + lds_off(wn * WN + fr, 4 * st + 2 * pt + fg);
    }
  auto frag = [&](int slot, const int (&f)[2][2], int i, int st) {
    const uint8_t* at = lds + slot * kStage + i * 4096;
    return join8(*reinterpret_cast<const v4i*>(at + f[st ^ (i & 1)][0]),
                 *reinterpret_cast<const v4i*>(at + f[st ^ (i & 1)][1]));
  };
  // a wave's 32-row tiles are consecutive bytes of its group's scale words
  const int at_ea = kA + kB + (wrow / 128) * 128 + fr * 4;
  const int at_eb = kA + kB + kScale + (wcol / 128) * 128 + fr * 4;
  auto words = [&](int slot, int& ea, int& eb) {
    ea = (int)(*reinterpret_cast<const uint32_t*>(lds + slot * kStage + at_ea) >> (wrow % 128 / 32 * 8));
    eb = (int)(*reinterpret_cast<const uint32_t*>(lds + slot * kStage + at_eb) >> (wcol % 128 / 32 * 8));
  };

  v16f acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; i++)
#pragma unroll
    for (int j = 0; j < TN; j++) acc[i][j] = v16f{};

#pragma unroll
  for (int st = 0; st < NS; st++) issue(min(st, nk - 1), st);
  wait_vmcnt<(NS - 1) * kLoads>();
  stage_barrier();
  v8i b[TN], a;
  int ea, eb;
#pragma unroll
  for (int j = 0; j < TN; j++) b[j] = frag(0, fb, j, 0);
  a = frag(0, fa, 0, 0);
  words(0, ea, eb);

  // A stage is 2 TM row tiles' turns. Each reads the next one's row fragment (and, at the
  // step's end, the next step's columns) before its products. Before the last two turns' products
  // every fragment of the stage is in registers: the slot is given back, the next stage's
  // first fragments are asked for, and their latency and the barrier's pass behind the
  // products that are left.
  // The body has no branch (stages past the last are asked for again and read by nobody), so
  // that the accumulators stay where they are.
  constexpr int U = 2 * TM, kGive = U - 2 > TM ? U - 2 : TM;
  int slot = 0;
  for (int kt = 0; kt < nk; kt++) {
    const int next = slot + 1 == NS ? 0 : slot + 1;
    v8i bn[TN];
    int ean, ebn;
#pragma unroll
    for (int u = 0; u < U; u++) {
      v8i an;
      if (u + 1 < U) an = frag(slot, fa, (u + 1) % TM, (u + 1) / TM);
      if (u + 1 == TM) {
#pragma unroll
        for (int j = 0; j < TN; j++) bn[j] = frag(slot, fb, j, 1);
      }
      if (u == kGive) {
        wait_lgkmcnt0();
        wait_vmcnt<(NS - 2) * kLoads>();
        stage_barrier();
        issue(min(kt + NS, nk - 1), slot);
#pragma unroll
        for (int j = 0; j < TN; j++) bn[j] = frag(next, fb, j, 0);
        words(next, ean, ebn);
      }
      if (u + 1 == U) an = frag(next, fa, 0, 0);
      fp8_row<TM, TN>(acc, a, b, u % TM, ea, eb);
      a = an;
      if (u + 1 == TM || u + 1 == U) {
#pragma unroll
        for (int j = 0; j < TN; j++) b[j] = bn[j];
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    ea = ean;
    eb = ebn;
    slot = next;
  }
  wait_vmcnt<0>();
  __syncthreads();
  fp8_epilogue<WM, WN, TM, TN>(p, acc, lds, row0, col0, wave, wm, wn, lane);
}

// ---- few rows -------------------------------------------------------------------------
template <bool BF16>
struct Fp8RowBlock {
  using S = std::conditional_t<BF16, __bf16, float>;
  using T = std::conditional_t<BF16, v8bf, v4f>;
  static constexpr int E = BF16 ? 8 : 4;
  T v[32 / E];  // 32 values of a row's block, the others 16, 32 and 48 lanes further

  __device__ __forceinline__ void load(const void* src, size_t row, int c, int K, bool vec) {
    const S* at = static_cast<const S*>(src) + row + c;
    if (vec && c + 32 <= K) {
#pragma unroll
      for (int i = 0; i < 32 / E; i++) v[i] = *reinterpret_cast<const T*>(at + i * E);
    } else {
#pragma unroll
      for (int e = 0; e < 32; e++) v[e / E][e % E] = c + e < K ? at[e] : (S)0.0f;
    }
  }
  // Its codes; ex: the block's byte. Conversions that scale by themselves, 2.5 instructions a
  // value of bf16 for 6.5; blocks with infinities or NaN, and below 2^-103, go the quantizer's
  // way.
  __device__ __forceinline__ v8i codes(int& ex) const {
    v8i x = {};
#if defined(__HIP_DEVICE_COMPILE__)
    auto value = [&](int e) { return (float)v[e / E][e % E]; };
    auto block = [](uint32_t top) {
      top = max(top, (uint32_t)__shfl_xor((int)top, 16, 64));
      return max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
    };
    uint32_t top = 0;
    if constexpr (BF16) {
      typedef uint16_t v2u16 __attribute__((ext_vector_type(2)));
      v2u16 m = {0, 0};
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const v4i w = __builtin_bit_cast(v4i, v[i]);
#pragma unroll
        for (int e = 0; e < 4; e++)
          m = __builtin_elementwise_max(m, __builtin_bit_cast(v2u16, w[e] & 0x7FFF7FFF));
      }
      top = (uint32_t)max(m[0], m[1]) << 16;
    } else {
#pragma unroll
      for (int e = 0; e < 32; e++) top = max(top, __float_as_uint(value(e)) & 0x7FFFFFFFu);
    }
    top = block(top);
    ex = fp8_exponent(top);
    if (__builtin_expect(__any(top >= 0x7F800000u || ex < 16), 0)) {
      top = 0;
#pragma unroll
      for (int e = 0; e < 32; e++) top = max(top, finite_abs_bits(value(e)));
      ex = fp8_exponent(block(top));
      const float f = fp8_inverse(ex);
#pragma unroll
      for (int e = 0; e < 8; e++)
        x[e] = fp8_pack4(value(4 * e) * f, value(4 * e + 1) * f, value(4 * e + 2) * f,
                         value(4 * e + 3) * f);
      return x;
    }
    const float unit = __uint_as_float((uint32_t)ex << 23);
#pragma unroll
    for (int e = 0; e < 8; e++) {
      typedef short v2s __attribute__((ext_vector_type(2)));
      v2s h;
      asm("" : "=v"(h) : "v"(unit));  // any word: both halves get written
      h = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(h, value(4 * e), value(4 * e + 1), unit, false);
      h = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(h, value(4 * e + 2), value(4 * e + 3), unit,
                                                   true);
      x[e] = __builtin_bit_cast(int, h);
    }
#endif
    return x;
  }
};

// A query's rows: the weights' bytes are all there is to move, so 16 of their rows go to
// a workgroup (4096 outputs: 256 workgroups), whose NW waves hold different 128-blocks
// of K and read them straight to registers as the A operand of 16x16x128 products (32
// consecutive bytes a lane, four lanes a row's block). The activations are the columns, 16 MT of
// them. The waves' sums are joined in LDS in wave order, and a thread finishes four
// consecutive outputs of a row.
// SRC 0: rows are e4m3 already; 1 / 2: fp32 / bf16 rows are made so here, to the same codes as
// quantize_rows_fp8_kernel's (a launch less, but every workgroup does it: gemm_fp8_takes_rows).
// 37 rows of bf16 by 2560 x 1024 take 6.2 µs, 2.2 over a launch; the next block's rows asked for a
// block ahead did not gain (6.5).
template <int MT, int NW, int SRC>
__global__ __launch_bounds__(64 * NW) void gemm_fp8_rows_kernel(GemmFp8Args p, const void* src,
                                                                int lds_src) {
  __shared__ __attribute__((aligned(16))) float red[NW][MT][64][4];
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * MT;
  const int nk = (p.K + kFp8Block - 1) / kFp8Block;
  const int ga = (p.M + 127) / 128, gb = p.Np / 128;
  const uint8_t* wrow = p.B + (size_t)(n0 + r) * p.ldb + g * 32;
  const uint8_t* wexp = p.sb + fp8_scale_at(n0 + r, 0, gb);
  int mrow[MT];
#pragma unroll
  for (int t = 0; t < MT; t++) mrow[t] = min(m0 + t * 16 + r, p.M - 1);

  v4f acc[MT];
#pragma unroll
  for (int t = 0; t < MT; t++) acc[t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  if constexpr (SRC == 0) {
#pragma unroll 4
    for (int kb = wave; kb < nk; kb += NW) {
      const v4i* at = reinterpret_cast<const v4i*>(wrow + (size_t)kb * kFp8Block);
      const v8i w = join8(at[0], at[1]);
      const int ew = wexp[(size_t)kb * gb * 128];
#pragma unroll
      for (int t = 0; t < MT; t++) {
        const v4i* xt = reinterpret_cast<const v4i*>(p.A + (size_t)mrow[t] * p.lda +
                                                     (size_t)kb * kFp8Block + g * 32);
        const int ex = p.sa[fp8_scale_at(mrow[t], kb, ga)];
        acc[t] = mfma_fp8_16(w, join8(xt[0], xt[1]), acc[t], ew, ex);
      }
    }
  } else {
    static_assert(MT == 1, "one column tile");
    const bool vec = lds_src % 8 == 0 && ((uintptr_t)src & 15) == 0;
#pragma unroll 4
    for (int kb = wave; kb < nk; kb += NW) {
      const v4i* at = reinterpret_cast<const v4i*>(wrow + (size_t)kb * kFp8Block);
      const v8i w = join8(at[0], at[1]);
      const int ew = wexp[(size_t)kb * gb * 128];
      Fp8RowBlock<SRC == 2> rows;
      rows.load(src, (size_t)mrow[0] * lds_src, kb * kFp8Block + g * 32, p.K, vec);
      int ex;
      const v8i x = rows.codes(ex);
      acc[0] = mfma_fp8_16(w, x, acc[0], ew, ex);
    }
  }
#pragma unroll
  for (int t = 0; t < MT; t++) *reinterpret_cast<v4f*>(red[wave][t][lane]) = acc[t];
  __syncthreads();
  // thread -> column tile t, lane l of it: row m0 + 16 t + l % 16, outputs n0 + 4 (l / 16) ..
  const bool glu = is_glu(p.act);
  const int t = threadIdx.x >> 6, l = threadIdx.x & 63;
  if (t >= MT) return;
  const int row = m0 + t * 16 + (l & 15), q = l >> 4, col = n0 + 4 * q;
  if (row >= p.M || (glu && (q & 1))) return;
  auto sum = [&](int at) {
    v4f x = *reinterpret_cast<const v4f*>(red[0][t][at]);
#pragma unroll
    for (int w = 1; w < NW; w++) x += *reinterpret_cast<const v4f*>(red[w][t][at]);
    return x;
  };
  v4f x = sum(l);
  if (glu) {  // groups of four rows: gate, then up
    const v4f u = sum(l + 16);
#pragma unroll
    for (int e = 0; e < 4; e++) x[e] = fp8_glu(x[e], u[e], p.act);
  } else {
#pragma unroll
    for (int e = 0; e < 4; e++) x[e] = apply_act(x[e] + (p.bias ? p.bias[col + e] : 0.0f), p.act);
  }
  fp8_store4(p, row, glu ? col / 2 : col, x);
}

template <int BM, int BN, int NS, int WGN>
static void launch_tile(const GemmFp8Args& a, hipStream_t s) {
  const dim3 grid((unsigned)(ceil_div(a.M, BM) * ceil_div(a.N, BN)));
  timed_launch(gemm_fp8_kernel<BM, BN, NS, WGN>, grid, dim3(128 * WGN), 0, s, a);
}

template <int MT, int NW, int SRC>
static void launch_rows(const GemmFp8Args& a, const void* src, int ld, hipStream_t s) {
  const dim3 grid((unsigned)(a.N / 16), (unsigned)ceil_div(a.M, 16 * MT));
  timed_launch(gemm_fp8_rows_kernel<MT, NW, SRC>, grid, dim3(64 * NW), 0, s, a, src, ld);
}

// The kernel of few rows where it makes at most a workgroup per CU (of up to 16 rows: two).
// µs, K 4096, bf16 out, against the 64 x 64 tiles: N 1024, M 64: 6.1 / 9.7, M 128: 8.3 / 9.9;
// N 4096, M 16: 6.4 / 10.0, M 32: 9.1 / 9.9, M 48: 12.9 / 9.9; N 8192, M 16: 10.0 / 10.1.
// One column tile a workgroup where that fits, else two (four were never ahead).
static int rows_tiles(int M, int N) {
  const long long wgs = N / 16;
  if (wgs * ceil_div(M, 16) <= (M <= 16 ? 512 : 256)) return 1;
  if (wgs * ceil_div(M, 32) <= 256) return 2;
  return 0;
}

// fp32 / bf16 rows go straight into it where its workgroups' work on them, up to 16 rows of K
// each, is less than a launch. µs against quantizing first, rows in 16-byte pieces: bf16, N 1024:
// M 16 K 1024 4.5 / 7.1, M 64 K 2560 6.6 / 7.6, M 16 K 4096 8.3 / 8.7; fp32, N 1024: M 64 K 1024
// 5.3 / 7.2, M 5 K 3584 7.2 / 7.2, M 16 K 2560 8.4 / 7.3; M 1 K 4096 6.9 / 6.9, K 8192 10.8 / 9.4;
// two workgroups to a CU, N 8192 K 1024 M 16: bf16 5.9 / 6.9, fp32 7.7 / 6.8. Rows read value by
// value: M 16 K 301 5.7 / 6.8, K 516 5.8 / 7.1, K 1001 8.2 / 7.1, K 3500 22 / 8.7.
bool gemm_fp8_takes_rows(int M, int N, int K, const void* a, int a_bf16, int lda) {
  if (rows_tiles(M, N) != 1) return false;
  const bool two = (long long)(N / 16) * ceil_div(M, 16) > 256;
  if (lda % 8 || ((uintptr_t)a & 15)) return !two && K <= 512;
  const long long bytes = (long long)std::min(M, 16) * K * (a_bf16 ? 2 : 4);
  return K <= 3584 && bytes * (two ? 2 : 1) <= 80 * 1024;
}

// A tile's time by rounds of the chip's 256 CUs: µs per started round at K 4096 (about a
// third of it at K 1024), from M 400 .. 12000, N 1024 .. 4096. The tile with the least is
// taken: M 400 64 x 64 (N 4096: 16.5 µs, next 19.5), M 1500 128 x 256 (33.6, 36.0), M 3000
// 256 x 256 (53.6, 59.0), M 6000 128 x 256 (98.3, 106.6), M 8192 256 x 256 (108 of the
// 110 that this card's fp8 library product takes for its share).
static long long tile_cost(int M, int N, int bm, int bn, int each) {
  return (long long)ceil_div(ceil_div(M, bm) * ceil_div(N, bn), 256) * each;
}

hipError_t launch_gemm_fp8(const GemmFp8Args& a, const void* src, int src_bf16, int ld_src,
                           hipStream_t s) {
  if (a.M <= 0) return hipSuccess;
  if (src) {
    if (src_bf16) launch_rows<1, 8, 2>(a, src, ld_src, s);
    else launch_rows<1, 8, 1>(a, src, ld_src, s);
    return hipGetLastError();
  }
  const int rows = rows_tiles(a.M, a.N);
  if (rows == 1) launch_rows<1, 8, 0>(a, nullptr, 0, s);
  else if (rows == 2) launch_rows<2, 8, 0>(a, nullptr, 0, s);
  if (rows) return hipGetLastError();
  const long long c64 = tile_cost(a.M, a.N, 64, 64, 76), c128 = tile_cost(a.M, a.N, 128, 128, 185),
                  cwide = tile_cost(a.M, a.N, 128, 256, 325),
                  c256 = tile_cost(a.M, a.N, 256, 256, 540);
  const long long best = std::min(std::min(c64, c128), std::min(cwide, c256));
  if (best == c64) launch_tile<64, 64, 4, 2>(a, s);
  else if (best == c128) launch_tile<128, 128, 2, 2>(a, s);
  else if (best == cwide) launch_tile<128, 256, 3, 4>(a, s);
  else launch_tile<256, 256, 2, 4>(a, s);
  return hipGetLastError();
}

}  // namespace rh
