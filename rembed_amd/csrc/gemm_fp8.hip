// gemm_fp8.hip — e4m3 activations x e4m3 weights for gfx950, a power-of-two scale
// for each 128 values of an activation row and each 128 x 128 block of the weight:
//   y[r][n] = act(sum_b 2^(ea[r][b] + ew[n][b]) sum_{k in b} qa[r][k] qw[n][k] + bias[n]).
//
// The fourth mode beside the fp32, weight-only int8 and full-int8 linears
// (applyDense, internal/model/bert.go:282-301); no counterpart in the reference.
// The scale bytes are the matrix instruction's own (fp8.h), so the main loop is
// loads and v_mfma_scale_f32_32x32x64_f8f6f4 alone, one accumulation over all of K.
#include "fp8.h"
#include <cstdlib>

namespace rh {

// ---- rows to e4m3 -----------------------------------------------------------------
// A wave takes 512 values of a row, 16 lanes a block of 128: eight values a lane,
// their maximum over the 16 lanes by row rotations, codes as one 8-byte store. One
// read and one write of every value.
template <bool BF16, bool VEC>
__global__ __launch_bounds__(256) void quantize_rows_fp8_kernel(const void* a, int lda, int m,
                                                                int k, uint8_t* qa, int ldq,
                                                                uint8_t* sa, int per_row) {
  const int wave = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int r = wave / per_row;
  if (r >= m) return;
  const int c = (wave - r * per_row) * 512 + lane * 8;
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
  const int per_row = ceil_div(ldq, 512);
  const dim3 grid((unsigned)(((long long)m * per_row + 3) / 4)), block(256);
  const bool vec = k % 8 == 0 && lda % 8 == 0 && ((uintptr_t)a & 15) == 0;
#define RH_Q(B, V)                                                                              \
  hipLaunchKernelGGL((quantize_rows_fp8_kernel<B, V>), grid, block, 0, s, a, lda, m, k, qa, ldq, \
                     sa, per_row)
  if (a_bf16) {
    if (vec) RH_Q(true, true);
    else RH_Q(true, false);
  } else {
    if (vec) RH_Q(false, true);
    else RH_Q(false, false);
  }
#undef RH_Q
  return hipGetLastError();
}

// ---- GEMM ---------------------------------------------------------------------------
// Epilogue: per 32-row band a wave parks its accumulators in LDS and reads rows
// back 4 (gated: 8) columns a lane, so outputs leave as vectors of 4.
template <int BM, int WM, int WN, int TM, int TN>
__device__ __forceinline__ void fp8_epilogue(const GemmFp8Args& p, v16f (&acc)[TM][TN],
                                             uint8_t* lds, int row0, int col0, int wave, int wm,
                                             int wn, int lane) {
  constexpr int kStride = WN + 4;
  typedef __bf16 v4bf __attribute__((ext_vector_type(4)));
  const int fr = lane & 31, fg = lane >> 5;
  float* ep = reinterpret_cast<float*>(lds) + wave * 32 * kStride;
  const bool glu = is_glu(p.act);
  auto store = [&](int row, int col, const v4f& v) {
    const size_t at = (size_t)row * p.ldo + col;
    if (p.out_bf16)
      *reinterpret_cast<v4bf*>(static_cast<__bf16*>(p.out) + at) =
          (v4bf){(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
    else
      *reinterpret_cast<v4f*>(static_cast<float*>(p.out) + at) = v;
  };
#pragma unroll
  for (int i = 0; i < TM; i++) {
#pragma unroll
    for (int j = 0; j < TN; j++)
#pragma unroll
      for (int r = 0; r < 16; r++)
        ep[((r >> 2) * 8 + fg * 4 + (r & 3)) * kStride + j * 32 + fr] = acc[i][j][r];
    wait_lgkmcnt0();
    __builtin_amdgcn_wave_barrier();
    const int rows = row0 + wm * WM + i * 32;
    if (glu) {  // columns 8t..8t+3 gate, 8t+4..8t+7 up
      constexpr int kL = WN / 8, kR = 64 / kL;
      const int c8 = lane % kL * 8, col = col0 + wn * WN + c8;
      for (int rr = lane / kL; rr < 32; rr += kR) {
        const v4f g = *reinterpret_cast<const v4f*>(ep + rr * kStride + c8);
        const v4f u = *reinterpret_cast<const v4f*>(ep + rr * kStride + c8 + 4);
        if (rows + rr < p.M && col < p.N) {
          v4f o;
#pragma unroll
          for (int e = 0; e < 4; e++) o[e] = glu_act(g[e], u[e], p.act);
          store(rows + rr, col / 2, o);
        }
      }
    } else {
      constexpr int kL = WN / 4, kR = 64 / kL;
      const int c4 = lane % kL * 4, col = col0 + wn * WN + c4;
      v4f bs = {0.0f, 0.0f, 0.0f, 0.0f};
      if (p.bias && col < p.N) bs = *reinterpret_cast<const v4f*>(p.bias + col);
      for (int rr = lane / kL; rr < 32; rr += kR) {
        v4f v = *reinterpret_cast<const v4f*>(ep + rr * kStride + c4);
        if (rows + rr < p.M && col < p.N) {
#pragma unroll
          for (int e = 0; e < 4; e++) v[e] = apply_act(v[e] + bs[e], p.act);
          store(rows + rr, col, v);
        }
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// BM x BN tile of 2 x WGN waves, K in stages of 128 bytes (one scale block), an
// NS-slot ring filled by global_load_lds; the stage's scale words come the same
// way, behind its codes.
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
  auto wait_stage = [&](int later) {
    if (later >= NS - 2) wait_vmcnt<(NS - 2) * kLoads>();
    else if (NS > 3 && later == 1) wait_vmcnt<kLoads>();
    else wait_vmcnt<0>();
  };

  v16f acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; i++)
#pragma unroll
    for (int j = 0; j < TN; j++)
#pragma unroll
      for (int e = 0; e < 16; e++) acc[i][j][e] = 0.0f;

#pragma unroll
  for (int st = 0; st < NS - 1; st++)
    if (st < nk) issue(st, st);

  const int fr = lane & 31, fg = lane >> 5;
  int slot = 0;
  for (int kt = 0; kt < nk; kt++) {
    wait_stage(min(NS - 2, nk - 1 - kt));
    wait_lgkmcnt0();  // this wave has read the slot that is refilled below
    stage_barrier();
    if (kt + NS - 1 < nk) issue(kt + NS - 1, slot == 0 ? NS - 1 : slot - 1);
    const uint8_t* sA = lds + slot * kStage;
    const uint8_t* sB = sA + kA;
    // a wave's 32-row tiles are consecutive bytes of its group's words
    int ea = *reinterpret_cast<const int*>(sA + kA + kB + (wrow / 128) * 128 + fr * 4);
    int eb = *reinterpret_cast<const int*>(sA + kA + kB + kScale + (wcol / 128) * 128 + fr * 4);
    ea = (int)((uint32_t)ea >> (wrow % 128 / 32 * 8));
    eb = (int)((uint32_t)eb >> (wcol % 128 / 32 * 8));
#pragma unroll
    for (int s = 0; s < 2; s++) {
      v8i a[TM], b[TN];
#pragma unroll
      for (int i = 0; i < TM; i++) {
        const int r = wm * WM + i * 32 + fr;
        a[i] = join8(*reinterpret_cast<const v4i*>(sA + lds_off(r, 4 * s + fg)),
                     *reinterpret_cast<const v4i*>(sA + lds_off(r, 4 * s + 2 + fg)));
      }
#pragma unroll
      for (int j = 0; j < TN; j++) {
        const int r = wn * WN + j * 32 + fr;
        b[j] = join8(*reinterpret_cast<const v4i*>(sB + lds_off(r, 4 * s + fg)),
                     *reinterpret_cast<const v4i*>(sB + lds_off(r, 4 * s + 2 + fg)));
      }
#define RH_MM(i, j)                                                                    \
  if constexpr ((i) < TM && (j) < TN)                                                  \
    acc[i][j] = mfma_fp8_32<(i), (j)>(a[i], b[j], acc[i][j], ea, eb);
#define RH_ROW(i) RH_MM(i, 0) RH_MM(i, 1) RH_MM(i, 2) RH_MM(i, 3)
      RH_ROW(0) RH_ROW(1) RH_ROW(2) RH_ROW(3)
#undef RH_ROW
#undef RH_MM
    }
    slot = slot + 1 == NS ? 0 : slot + 1;
  }
  __syncthreads();
  fp8_epilogue<BM, WM, WN, TM, TN>(p, acc, lds, row0, col0, wave, wm, wn, lane);
}

template <int BM, int BN, int NS, int WGN>
static void launch_tile(const GemmFp8Args& a, hipStream_t s) {
  const dim3 grid((unsigned)(ceil_div(a.M, BM) * ceil_div(a.N, BN)));
  timed_launch(gemm_fp8_kernel<BM, BN, NS, WGN>, grid, dim3(128 * WGN), 0, s, a);
}

hipError_t launch_gemm_fp8(const GemmFp8Args& a, hipStream_t s) {
  if (a.M <= 0) return hipSuccess;
  int t = 0;
  if (const char* e = getenv("RH_TILE")) t = atoi(e);
  switch (t) {
    case 1: launch_tile<128, 128, 3, 2>(a, s); break;
    case 2: launch_tile<128, 128, 4, 2>(a, s); break;
    case 3: launch_tile<256, 256, 2, 4>(a, s); break;
    case 4: launch_tile<128, 256, 2, 4>(a, s); break;
    case 5: launch_tile<128, 256, 3, 4>(a, s); break;
    case 6: launch_tile<256, 128, 2, 2>(a, s); break;
    case 7: launch_tile<64, 64, 4, 2>(a, s); break;
    case 8: launch_tile<64, 128, 3, 2>(a, s); break;
    case 9: launch_tile<256, 256, 2, 2>(a, s); break;
    case 10: launch_tile<64, 128, 2, 2>(a, s); break;
    default: launch_tile<128, 128, 2, 2>(a, s); break;
  }
  return hipGetLastError();
}

}  // namespace rh
