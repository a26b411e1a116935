// cache.hip — the paged 8-bit key/value cache of the decoder embedders: block
// tables and slot maps built on the device, and new rows appended to it.
//
// No counterpart in the reference, which recomputes an instruction's prefix for
// every query (qwen3.go:395-548). A page holds the 64 tokens of one block for all
// kv heads; per head its K and V are 64 x dh e4m3 codes with one scale byte each
// (fp8.h), laid out as the attention's MFMA fragments read them:
//   K: value d of token t at ((d/64 * 2 + t/32) * 2 + d%32/16) * 1024
//      + (d%64/32 * 32 + t%32) * 16 + d%16
//   V: value d of token t at (d/32 * 2 + t/32) * 1024
//      + (t%8/4 * 32 + d%32) * 16 + t%32/8 * 4 + t%4
// so a wave's fragment load is 1 KiB of consecutive bytes, and V's tokens come in
// the order in which the score tiles leave the matrix cores.
#include "fp8.h"

#include <algorithm>

namespace rh {

constexpr int kPage = RH_CACHE_BLOCK;

__host__ __device__ __forceinline__ int k_at(int t, int d) {
  return ((d / 64 * 2 + t / 32) * 2 + d % 32 / 16) * 1024 + (d % 64 / 32 * 32 + t % 32) * 16 +
         d % 16;
}
__host__ __device__ __forceinline__ int v_at(int t, int d) {
  return (d / 32 * 2 + t / 32) * 1024 + (t % 8 / 4 * 32 + d % 32) * 16 + t % 32 / 8 * 4 + t % 4;
}

// ---- block tables and slot maps ---------------------------------------------------------
// Request b has past[b] tokens in the cache and fresh[b] new ones:
//   need = ceil((past + fresh) / 64) - ceil(past / 64) pages, taken from the free
//   list in request order (first = the sum of need over the requests before it);
//   its row t lies at row cu[b] + t, position past + t, slot page * 64 + position % 64.
// Every workgroup scans the lengths itself (they are a few KiB from L2) and then
// fills its share of rows and table entries, so one launch serves: prefix sums in
// a kernel of their own would cost a second launch's gap, more than the scan.
constexpr int kPlanThreads = 256;
constexpr int kPlanChunk = 1024;  // requests whose prefix sums are in LDS at once

struct PlanSums {
  long long rows, need, touched;
};

__global__ __launch_bounds__(kPlanThreads) void cache_plan_kernel(CachePlanArgs p) {
  __shared__ int s_past[kPlanChunk];
  __shared__ int s_cu[kPlanChunk + 1], s_first[kPlanChunk + 1], s_blk[kPlanChunk + 1];
  __shared__ int s_wave[3][kPlanThreads / 64];
  __shared__ long long s_tot[3];
  __shared__ int s_err;
  const int tid = threadIdx.x;
  const int lane = tid & 63, wave = tid >> 6;
  const bool writer = blockIdx.x == 0;

  // Totals and faults first: a plan that does not fit changes nothing.
  if (tid < 3) s_tot[tid] = 0;
  if (tid == 0) s_err = 0;
  __syncthreads();
  {
    long long rows = 0, need = 0;
    int err = 0;
    for (int b = tid; b < p.batch; b += kPlanThreads) {
      const long long pa = p.past[b], fr = p.fresh[b];
      if (pa < 0 || fr < 0) {
        err |= 1;
        continue;
      }
      const long long blk = (pa + fr + kPage - 1) / kPage;
      if (blk > p.ldt || pa + fr > 0x7FFFFF00) err |= 2;
      rows += fr;
      need += blk - (pa + kPage - 1) / kPage;
    }
    for (int o = 32; o; o >>= 1) {
      rows += __shfl_xor(rows, o, 64);
      need += __shfl_xor(need, o, 64);
      err |= __shfl_xor(err, o, 64);
    }
    if (lane == 0) {
      // integer sums: the order of the atomics does not show
      atomicAdd(reinterpret_cast<unsigned long long*>(&s_tot[0]), (unsigned long long)rows);
      atomicAdd(reinterpret_cast<unsigned long long*>(&s_tot[1]), (unsigned long long)need);
      atomicOr(&s_err, err);
    }
  }
  __syncthreads();
  int err = s_err;
  if (s_tot[0] > p.rows) err |= 4;
  if (s_tot[1] > p.n_free) err |= 8;
  const int stride = gridDim.x * kPlanThreads, at0 = blockIdx.x * kPlanThreads + tid;
  if (err) {
    for (int r = at0; r < p.rows; r += stride) {
      p.slots[r] = -1;
      p.pos[r] = 0;
    }
    for (int b = at0; b <= p.batch; b += stride) {
      p.cu[b] = 0;
      p.blocks[b] = 0;
      if (b < p.batch) p.lens[b] = p.past[b];
    }
    if (writer && tid < 4) p.status[tid] = tid == 0 ? err : 0;
    return;
  }

  int c_rows = 0, c_need = 0, c_touch = 0;  // sums over the chunks before
  for (int b0 = 0; b0 < p.batch; b0 += kPlanChunk) {
    const int n = min(kPlanChunk, p.batch - b0);
    // four consecutive requests per thread, then a scan over the threads
    int past[4], fresh[4], need[4], touch[4], sum[3] = {0, 0, 0};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int b = tid * 4 + i;
      past[i] = b < n ? p.past[b0 + b] : 0;
      fresh[i] = b < n ? p.fresh[b0 + b] : 0;
      need[i] = (past[i] + fresh[i] + kPage - 1) / kPage - (past[i] + kPage - 1) / kPage;
      touch[i] = fresh[i] > 0 ? (past[i] + fresh[i] - 1) / kPage - past[i] / kPage + 1 : 0;
      sum[0] += fresh[i];
      sum[1] += need[i];
      sum[2] += touch[i];
    }
    int before[3];
#pragma unroll
    for (int k = 0; k < 3; k++) {
      int v = sum[k];
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(v, o, 64);
        if (lane >= o) v += u;
      }
      before[k] = v - sum[k];
      if (lane == 63) s_wave[k][wave] = v;
    }
    __syncthreads();
    int all[3] = {0, 0, 0};
#pragma unroll
    for (int k = 0; k < 3; k++)
#pragma unroll
      for (int w = 0; w < kPlanThreads / 64; w++) {
        if (w < wave) before[k] += s_wave[k][w];
        all[k] += s_wave[k][w];
      }
    int at[3] = {c_rows + before[0], c_need + before[1], c_touch + before[2]};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int b = tid * 4 + i;
      if (b < n) {
        s_past[b] = past[i];
        s_cu[b] = at[0];
        s_first[b] = at[1];
        s_blk[b] = at[2];
        if (writer) p.lens[b0 + b] = past[i] + fresh[i];
      }
      at[0] += fresh[i];
      at[1] += need[i];
      at[2] += touch[i];
    }
    if (tid == 0) {
      s_cu[n] = c_rows + all[0];
      s_first[n] = c_need + all[1];
      s_blk[n] = c_touch + all[2];
    }
    __syncthreads();
    // the last request of the chunk with start[b] <= x
    auto find = [&](const int* start, int x) {
      int lo = 0, hi = n - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (start[mid] <= x) lo = mid;
        else hi = mid - 1;
      }
      return lo;
    };
    if (writer)
      for (int b = tid; b < n; b += kPlanThreads) {
        p.cu[b0 + b] = s_cu[b];
        p.blocks[b0 + b] = s_blk[b];
      }
    // table entries behind the past's blocks are written here and read nowhere
    // in this launch (rows take new pages from the free list)
    for (int e = c_need + at0; e < c_need + all[1]; e += stride) {
      const int b = find(s_first, e);
      const int have = (s_past[b] + kPage - 1) / kPage;
      p.table[(size_t)(b0 + b) * p.ldt + have + e - s_first[b]] = p.free_pages[e];
    }
    for (int r = c_rows + at0; r < c_rows + all[0]; r += stride) {
      const int b = find(s_cu, r);
      const int pos = s_past[b] + r - s_cu[b];
      const int have = (s_past[b] + kPage - 1) / kPage, blk = pos / kPage;
      const int page = blk >= have ? p.free_pages[s_first[b] + blk - have]
                                   : p.table[(size_t)(b0 + b) * p.ldt + blk];
      p.slots[r] = page < 0 ? -1 : (int64_t)page * kPage + pos % kPage;
      p.pos[r] = pos;
    }
    c_rows += all[0];
    c_need += all[1];
    c_touch += all[2];
    __syncthreads();
  }
  for (int r = c_rows + at0; r < p.rows; r += stride) {  // rows behind the last request
    p.slots[r] = -1;
    p.pos[r] = 0;
  }
  if (writer && tid == 0) {
    p.cu[p.batch] = c_rows;
    p.blocks[p.batch] = c_touch;
    p.status[0] = 0;
    p.status[1] = c_rows;
    p.status[2] = c_need;
    p.status[3] = c_touch;
  }
}

hipError_t launch_cache_plan(const CachePlanArgs& a, hipStream_t s) {
  const int wgs = std::max(1, std::min(512, ceil_div(a.rows, 2 * kPlanThreads)));
  hipLaunchKernelGGL(cache_plan_kernel, dim3(wgs), dim3(kPlanThreads), 0, s, a);
  return hipGetLastError();
}

// ---- append ----------------------------------------------------------------------------
// One workgroup per (block touched, kv head), K and V together, four threads per
// token: the new rows stay in registers, the block's codes are put together in
// LDS and written whole. With e the byte of the new tokens' largest magnitude:
//   x' = max(e, x of the codes kept),  kept codes * 2^(x - x'),  new value * 2^(127 - x').
// A block whose first token is new keeps nothing: zeros behind the new tokens.
// A token whose K or V has an infinity or NaN in a head is stored as K = NaN,
// V = 0: whoever sees the token gets NaN, and nobody else does (0 * NaN would
// reach queries that must not see it through V). It sets no scale.
constexpr int kAppendThreads = 256;

template <int DH, bool BF16>
__global__ __launch_bounds__(kAppendThreads) void cache_append_kernel(CacheAppendArgs p) {
  constexpr int kBytes = kPage * DH, E = DH / 4;  // a head's block; values per thread
  __shared__ __attribute__((aligned(16))) uint8_t s_k[kBytes], s_v[kBytes];
  __shared__ uint32_t s_max[2];
  const int tid = threadIdx.x;
  const int heads = p.cache.kv_heads;
  const int seg = blockIdx.x / heads, h = blockIdx.x % heads;
  if (seg >= p.blocks[p.batch]) return;
  int lo = 0, hi = p.batch - 1;  // the last request with blocks[b] <= seg
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (p.blocks[mid] <= seg) lo = mid;
    else hi = mid - 1;
  }
  const int j = seg - p.blocks[lo];
  const int r0 = p.cu[lo], fresh = p.cu[lo + 1] - r0;
  if (r0 < 0 || fresh <= 0 || r0 + fresh > p.rows) return;
  const int64_t slot0 = p.slots[r0];
  if (slot0 < 0) return;
  const int off0 = (int)(slot0 % kPage);
  const int first = j == 0 ? 0 : j * kPage - off0;  // first new token of this block
  const int off = j == 0 ? off0 : 0;
  const int cnt = min(kPage - off, fresh - first);
  if (cnt <= 0) return;
  const int64_t slot = p.slots[r0 + first];
  if (slot < 0 || slot / kPage >= p.cache.pages) return;
  const size_t unit = (size_t)(slot / kPage) * heads + h;
  uint8_t* gk = p.cache.k + unit * kBytes;
  uint8_t* gv = p.cache.v + unit * kBytes;

  if (tid < 2) s_max[tid] = 0;
  // this thread's quarter of its token's K and V
  const int tok = tid >> 2, quarter = tid & 3;
  float k[E], v[E];
  uint32_t mk = 0, mv = 0;
  bool bad = false;
  if (tok < cnt) {
    const size_t at = (size_t)(r0 + first + tok) * p.ldkv + h * DH + quarter * E;
#pragma unroll
    for (int e = 0; e < E; e++) {
      if constexpr (BF16) {
        k[e] = (float)(static_cast<const __bf16*>(p.kv) + p.k_off)[at + e];
        v[e] = (float)(static_cast<const __bf16*>(p.kv) + p.v_off)[at + e];
      } else {
        k[e] = (static_cast<const float*>(p.kv) + p.k_off)[at + e];
        v[e] = (static_cast<const float*>(p.kv) + p.v_off)[at + e];
      }
      const uint32_t uk = __float_as_uint(k[e]) & 0x7FFFFFFFu;
      const uint32_t uv = __float_as_uint(v[e]) & 0x7FFFFFFFu;
      bad |= uk >= 0x7F800000u || uv >= 0x7F800000u;
      mk = max(mk, uk);
      mv = max(mv, uv);
    }
  }
  int any = bad;
  any |= __shfl_xor(any, 1, 64);
  any |= __shfl_xor(any, 2, 64);
  if (any) mk = mv = 0;
  for (int o = 32; o; o >>= 1) {
    mk = max(mk, (uint32_t)__shfl_xor((int)mk, o, 64));
    mv = max(mv, (uint32_t)__shfl_xor((int)mv, o, 64));
  }
  __syncthreads();
  if ((tid & 63) == 0) {
    atomicMax(&s_max[0], mk);
    atomicMax(&s_max[1], mv);
  }
  __syncthreads();
  int xk = fp8_exponent(s_max[0]), xv = fp8_exponent(s_max[1]);
  // the codes kept, four at a time
  if (off == 0) {
    for (int i = tid * 4; i < kBytes; i += kAppendThreads * 4) {
      *reinterpret_cast<int*>(s_k + i) = 0;
      *reinterpret_cast<int*>(s_v + i) = 0;
    }
  } else {
    const int ok = p.cache.k_exp[unit], ov = p.cache.v_exp[unit];
    xk = max(xk, ok);
    xv = max(xv, ov);
    auto scaled = [](int w, int down) {
      if (down == 0) return w;
      const float f = __uint_as_float((uint32_t)(127 - min(down, 126)) << 23);
      float c[4] = {};
      fp8_unpack4(w, c);
      return fp8_pack4(c[0] * f, c[1] * f, c[2] * f, c[3] * f);
    };
    for (int i = tid * 4; i < kBytes; i += kAppendThreads * 4) {
      *reinterpret_cast<int*>(s_k + i) = scaled(*reinterpret_cast<const int*>(gk + i), xk - ok);
      *reinterpret_cast<int*>(s_v + i) = scaled(*reinterpret_cast<const int*>(gv + i), xv - ov);
    }
  }
  __syncthreads();
  if (tok < cnt) {
    const float fk = fp8_inverse(xk), fv = fp8_inverse(xv);
#pragma unroll
    for (int e = 0; e < E; e += 4) {
      int wk = 0x7F7F7F7F, wv = 0;
      if (!any) {
        wk = fp8_pack4(k[e] * fk, k[e + 1] * fk, k[e + 2] * fk, k[e + 3] * fk);
        wv = fp8_pack4(v[e] * fv, v[e + 1] * fv, v[e + 2] * fv, v[e + 3] * fv);
      }
      const int d = quarter * E + e;
      *reinterpret_cast<int*>(s_k + k_at(off + tok, d)) = wk;
#pragma unroll
      for (int i = 0; i < 4; i++) s_v[v_at(off + tok, d + i)] = (uint8_t)(wv >> (8 * i));
    }
  }
  __syncthreads();
  for (int i = tid * 16; i < kBytes; i += kAppendThreads * 16) {
    *reinterpret_cast<v4i*>(gk + i) = *reinterpret_cast<const v4i*>(s_k + i);
    *reinterpret_cast<v4i*>(gv + i) = *reinterpret_cast<const v4i*>(s_v + i);
  }
  if (tid == 0) {
    p.cache.k_exp[unit] = (uint8_t)xk;
    p.cache.v_exp[unit] = (uint8_t)xv;
  }
}

hipError_t launch_cache_append(const CacheAppendArgs& a, hipStream_t s) {
  // every touched block holds a new row, and each request has at most two
  // partly new blocks
  const long long segs = std::min((long long)a.rows, (long long)a.rows / kPage + 2LL * a.batch);
  const dim3 grid((unsigned)(segs * a.cache.kv_heads)), block(kAppendThreads);
#define RH_APPEND(D)                                                                          \
  if (a.cache.dh == D) {                                                                      \
    if (a.in_bf16) hipLaunchKernelGGL((cache_append_kernel<D, true>), grid, block, 0, s, a);  \
    else hipLaunchKernelGGL((cache_append_kernel<D, false>), grid, block, 0, s, a);           \
  }
  RH_APPEND(64)
  RH_APPEND(128)
  RH_APPEND(256)
#undef RH_APPEND
  return hipGetLastError();
}

}  // namespace rh
