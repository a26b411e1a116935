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
#include <type_traits>

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
// a kernel of their own would cost a second launch's gap, more than the scan. What bounds
// it is latency: the lengths are loaded once (batches of up to 1024), and a thread
// takes four consecutive rows to one search for their request (512 texts, up to 700 new
// tokens each: 8.0 -> 7.0 µs; 48 single tokens 5.5, where an empty launch takes 4.0).
constexpr int kPlanThreads = 256;
constexpr int kPlanChunk = 1024;  // requests whose prefix sums are in LDS at once
constexpr int kPlanRows = 4;      // consecutive rows of a thread

// What a request adds: new tokens (high enough for any batch's sum), pages and blocks.
struct PlanSum {
  long long rows;
  unsigned long long both;  // pages << 32 | blocks touched
};
__device__ __forceinline__ int plan_add(PlanSum& s, long long past, long long fresh, int ldt) {
  if (past < 0 || fresh < 0) return 1;
  const long long blk = (past + fresh + kPage - 1) / kPage;
  const long long need = blk - (past + kPage - 1) / kPage;
  const long long touch = fresh > 0 ? (past + fresh - 1) / kPage - past / kPage + 1 : 0;
  s.rows += fresh;
  s.both += (unsigned long long)need << 32 | (unsigned long long)touch;
  return blk > ldt || past + fresh > 0x7FFFFF00 ? 2 : 0;
}

__global__ __launch_bounds__(kPlanThreads) void cache_plan_kernel(CachePlanArgs p) {
  __shared__ int s_past[kPlanChunk];
  __shared__ int s_cu[kPlanChunk + 1], s_first[kPlanChunk + 1], s_blk[kPlanChunk + 1];
  __shared__ PlanSum s_wave[kPlanThreads / 64];
  __shared__ int s_err[kPlanThreads / 64];
  const int tid = threadIdx.x;
  const int lane = tid & 63, wave = tid >> 6;
  const bool writer = blockIdx.x == 0;
  // unsigned: a loop's last step may pass 2^31
  const unsigned stride = gridDim.x * kPlanThreads, at0 = blockIdx.x * kPlanThreads + tid;

  // The chunk's lengths, four consecutive requests a thread, and the sums before each
  // thread's (`before`) and over the chunk (`all`).
  int past[4], fresh[4], err = 0;
  PlanSum mine, before, all;
  auto chunk = [&](int b0, int n) {
    mine = PlanSum{0, 0};
    int e = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int b = tid * 4 + i;
      past[i] = b < n ? p.past[b0 + b] : 0;
      fresh[i] = b < n ? p.fresh[b0 + b] : 0;
      e |= plan_add(mine, past[i], fresh[i], p.ldt);
    }
    PlanSum v = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const long long r = __shfl_up(v.rows, o, 64);
      const unsigned long long t = __shfl_up(v.both, o, 64);
      if (lane >= o) {
        v.rows += r;
        v.both += t;
      }
    }
    const unsigned long long any1 = __ballot(e & 1), any2 = __ballot(e & 2);
    if (lane == 63) {
      s_wave[wave] = v;
      s_err[wave] = (any1 ? 1 : 0) | (any2 ? 2 : 0);
    }
    __syncthreads();
    before = PlanSum{v.rows - mine.rows, v.both - mine.both};
    all = PlanSum{0, 0};
#pragma unroll
    for (int w = 0; w < kPlanThreads / 64; w++) {
      if (w < wave) {
        before.rows += s_wave[w].rows;
        before.both += s_wave[w].both;
      }
      all.rows += s_wave[w].rows;
      all.both += s_wave[w].both;
      err |= s_err[w];
    }
  };

  // Totals and faults first: a plan that does not fit changes nothing.
  const bool one = p.batch <= kPlanChunk;
  long long rows = 0, need = 0;
  for (int b0 = 0; b0 < p.batch; b0 += kPlanChunk) {
    chunk(b0, min(kPlanChunk, p.batch - b0));
    rows += all.rows;
    need += (long long)(all.both >> 32);
    if (!one) __syncthreads();
  }
  if (rows > p.rows) err |= 4;
  if (need > p.n_free) err |= 8;
  if (err) {
    for (unsigned r = at0; r < (unsigned)p.rows; r += stride) {
      p.slots[r] = -1;
      p.pos[r] = 0;
    }
    for (unsigned b = at0; b <= (unsigned)p.batch; b += stride) {
      p.cu[b] = 0;
      p.blocks[b] = 0;
      if (b < (unsigned)p.batch) p.lens[b] = p.past[b];
    }
    if (writer && tid < 4) p.status[tid] = tid == 0 ? err : 0;
    return;
  }

  int c_rows = 0, c_need = 0, c_touch = 0;  // sums over the chunks before
  for (int b0 = 0; b0 < p.batch; b0 += kPlanChunk) {
    const int n = min(kPlanChunk, p.batch - b0);
    if (!one) chunk(b0, n);
    int at[3] = {c_rows + (int)before.rows, c_need + (int)(before.both >> 32),
                 c_touch + (int)(uint32_t)before.both};
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
      PlanSum d{0, 0};
      plan_add(d, past[i], fresh[i], p.ldt);
      at[0] += (int)d.rows;
      at[1] += (int)(d.both >> 32);
      at[2] += (int)(uint32_t)d.both;
    }
    const int end_rows = c_rows + (int)all.rows, end_need = c_need + (int)(all.both >> 32),
              end_touch = c_touch + (int)(uint32_t)all.both;
    if (tid == 0) {
      s_cu[n] = end_rows;
      s_first[n] = end_need;
      s_blk[n] = end_touch;
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
    for (unsigned e = c_need + at0; e < (unsigned)end_need; e += stride) {
      const int b = find(s_first, e);
      const int have = (s_past[b] + kPage - 1) / kPage;
      p.table[(size_t)(b0 + b) * p.ldt + have + ((int)e - s_first[b])] = p.free_pages[e];
    }
    for (unsigned u = c_rows + at0 * kPlanRows; u < (unsigned)end_rows; u += stride * kPlanRows) {
      const int r0 = (int)u;
      int b = find(s_cu, r0), page = -1, page_of = -1;  // page_of: block of `page`, of request b
#pragma unroll
      for (int i = 0; i < kPlanRows; i++) {
        if (u + i >= (unsigned)end_rows) break;
        const int r = r0 + i;
        while (r >= s_cu[b + 1]) {
          b++;
          page_of = -1;
        }
        const int pos = s_past[b] + (r - s_cu[b]), blk = pos / kPage;
        if (blk != page_of) {
          const int have = (s_past[b] + kPage - 1) / kPage;
          page = blk >= have ? p.free_pages[s_first[b] + blk - have]
                             : p.table[(size_t)(b0 + b) * p.ldt + blk];
          page_of = blk;
        }
        p.slots[r] = page < 0 ? -1 : (int64_t)page * kPage + pos % kPage;
        p.pos[r] = pos;
      }
    }
    c_rows = end_rows;
    c_need = end_need;
    c_touch = end_touch;
    if (!one) __syncthreads();
  }
  for (unsigned r = c_rows + at0; r < (unsigned)p.rows; r += stride) {  // rows behind the last request
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
  constexpr int kEach = kPlanRows * kPlanThreads;
  const int wgs = std::max(1, std::min(512, a.rows / kEach + (a.rows % kEach != 0)));
  hipLaunchKernelGGL(cache_plan_kernel, dim3(wgs), dim3(kPlanThreads), 0, s, a);
  return hipGetLastError();
}

// ---- append ----------------------------------------------------------------------------
// One workgroup per (block touched, kv head), K and V together, four threads per
// token: the new rows stay in registers, the block's codes are put together in
// LDS and written whole. With e the byte of the new tokens' largest magnitude:
//   x' = max(e, x of the codes kept),  kept codes * 2^(x - x'),  new value * 2^(127 - x').
// A block whose first token is new keeps nothing: zeros behind the new tokens. One
// whose scale stays (most single tokens) is not read at all: only the new codes are written.
// A token whose K or V has an infinity or NaN in a head is stored as K = NaN,
// V = 0: whoever sees the token gets NaN, and nobody else does (0 * NaN would
// reach queries that must not see it through V). It sets no scale.
// Single tokens are bound by latency, so a request is found by a 64-way search (one load of
// a wave per level; a binary search took 3 µs of 7.6 for 48 requests) and its rows are
// asked for before their page is known: 48 single tokens of 8 heads of 128 take 5.5 µs. Many
// tokens are bound by their bytes: 22k tokens, 140 MB, take 28.6 µs, 4.9 TB/s, what a large copy
// reaches (a thread's loads one after the other in a row instead of 64 bytes by four threads:
// 30.7; stores that stay in the L2: 36.2).
constexpr int kAppendThreads = 256;

// The last request b with blocks[b] <= seg: every level looks at 64 evenly spaced ones.
__device__ __forceinline__ int append_request(const int32_t* blocks, int batch, int seg, int lane) {
  int lo = 0, n = batch;  // it is among lo .. lo + n - 1
  while (n > 1) {
    const int step = (n + 63) / 64;
    const int at = lo + lane * step;
    const bool le = lane * step < n && blocks[at] <= seg;
    const int k = __popcll(__ballot(le)) - 1;  // blocks do not fall: the first k + 1 of them
    lo += max(k, 0) * step;
    n = min(step, n - max(k, 0) * step);
  }
  return lo;
}

// Where a byte of V lies in LDS: 16-byte pieces change places within their 256 bytes, so
// that the words a wave writes at once (tokens 4 apart among them) meet all banks.
__device__ __forceinline__ int spread(int at) {
  return at ^ (at >> 9 & 1) << 6;
}

template <int DH, bool BF16>
__global__ __launch_bounds__(kAppendThreads) void cache_append_kernel(CacheAppendArgs p) {
  constexpr int kBytes = kPage * DH, E = DH / 4;  // a head's block; values per thread
  __shared__ __attribute__((aligned(16))) uint8_t s_k[kBytes], s_v[kBytes];
  __shared__ uint32_t s_max[kAppendThreads / 64][2];
  const int tid = threadIdx.x;
  const int heads = p.cache.kv_heads;
  const int seg = blockIdx.x / heads, h = blockIdx.x % heads;
  const int b = append_request(p.blocks, p.batch, seg, tid & 63);
  if (seg >= p.blocks[p.batch]) return;
  const int j = seg - p.blocks[b];
  const int r0 = p.cu[b], fresh = p.cu[b + 1] - r0;
  if (r0 < 0 || fresh <= 0 || r0 + (long long)fresh > p.rows) return;
  // a row of this block, wherever in its first block the request starts
  const int probe = j > (fresh - 1) / kPage ? fresh - 1 : j * kPage;
  int64_t start = p.slots[r0];
  const int64_t slot = p.slots[r0 + probe];
  if (__builtin_expect(start < 0, 0)) start = slot - probe;  // the first block has no page
  const int off0 = (int)(start & (kPage - 1));
  const int first = j == 0 ? 0 : j * kPage - off0;  // first new token of this block
  const int off = j == 0 ? off0 : 0;
  const int cnt = min(kPage - off, fresh - first);
  if (cnt <= 0) return;

  // every fourth 16 bytes of its token's K and V to a thread (so a load of a token's four takes 64
  // bytes at a time); four lanes beside each other have the four tokens of one word of V
  const int tok = tid / 16 * 4 + tid % 4, quarter = tid / 4 % 4;
  const bool mine = tok >= off && tok < off + cnt;
  using T = std::conditional_t<BF16, v8bf, v4f>;  // 16 bytes of a row, widened when used
  constexpr int kStep = BF16 ? 8 : 4;
  T k[E / kStep], v[E / kStep];
  uint32_t mk = 0, mv = 0;
  if (mine) {
    const size_t at = (size_t)(r0 + first + tok - off) * p.ldkv + h * DH + quarter * kStep;
    using S = std::conditional_t<BF16, __bf16, float>;
    const S* row = static_cast<const S*>(p.kv) + at;
#pragma unroll
    for (int e = 0; e < E / kStep; e++) {
      k[e] = *reinterpret_cast<const T*>(row + p.k_off + e * 4 * kStep);
      v[e] = *reinterpret_cast<const T*>(row + p.v_off + e * 4 * kStep);
    }
  }
  const bool here = slot >= 0 && slot / kPage < p.cache.pages;
  const size_t unit = here ? (size_t)(slot / kPage) * heads + h : 0;
  uint8_t* gk = p.cache.k + unit * kBytes;
  uint8_t* gv = p.cache.v + unit * kBytes;
  const int ok = p.cache.k_exp[unit], ov = p.cache.v_exp[unit];
  if (mine) {
#pragma unroll
    for (int e = 0; e < E; e++) {
      mk = max(mk, __float_as_uint((float)k[e / kStep][e % kStep]) & 0x7FFFFFFFu);
      mv = max(mv, __float_as_uint((float)v[e / kStep][e % kStep]) & 0x7FFFFFFFu);
    }
  }
  int bad = mk >= 0x7F800000u || mv >= 0x7F800000u;
  bad |= __shfl_xor(bad, 4, 64);
  bad |= __shfl_xor(bad, 8, 64);
  if (bad) mk = mv = 0;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    mk = max(mk, (uint32_t)__shfl_xor((int)mk, o, 64));
    mv = max(mv, (uint32_t)__shfl_xor((int)mv, o, 64));
  }
  if ((tid & 63) == 0) {
    s_max[tid >> 6][0] = mk;
    s_max[tid >> 6][1] = mv;
  }
  if (!here) return;  // the whole workgroup
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kAppendThreads / 64; w++) {
    mk = max(mk, s_max[w][0]);
    mv = max(mv, s_max[w][1]);
  }
  int xk = fp8_exponent(mk), xv = fp8_exponent(mv);
  bool whole_k = true, whole_v = true;  // the block's bytes are all written
  auto scaled = [](int w, int down) {
    const float f = __uint_as_float((uint32_t)(127 - min(down, 126)) << 23);
    float c[4] = {};
    fp8_unpack4(w, c);
    return fp8_pack4(c[0] * f, c[1] * f, c[2] * f, c[3] * f);
  };
  if (off == 0) {
    if (cnt < kPage) {
      for (int i = tid * 16; i < kBytes; i += kAppendThreads * 16) {
        *reinterpret_cast<v4i*>(s_k + i) = v4i{0, 0, 0, 0};
        *reinterpret_cast<v4i*>(s_v + i) = v4i{0, 0, 0, 0};
      }
      __syncthreads();
    }
  } else {
    whole_k = xk > ok;
    whole_v = xv > ov;
    xk = max(xk, ok);
    xv = max(xv, ov);
    for (int i = tid * 16; i < kBytes && (whole_k || whole_v); i += kAppendThreads * 16) {
      v4i a, c;
      if (whole_k) a = *reinterpret_cast<const v4i*>(gk + i);
      if (whole_v) c = *reinterpret_cast<const v4i*>(gv + i);
#pragma unroll
      for (int e = 0; e < 4; e++) {
        if (whole_k) a[e] = scaled(a[e], xk - ok);
        if (whole_v) c[e] = scaled(c[e], xv - ov);
      }
      if (whole_k) *reinterpret_cast<v4i*>(s_k + i) = a;
      if (whole_v) *reinterpret_cast<v4i*>(s_v + spread(i)) = c;
    }
    if (whole_k || whole_v) __syncthreads();
  }
  // single tokens' values of V, a byte to a place, from all threads by way of LDS
  const bool few = !whole_v && cnt < 4;
  if (mine) {
    const float fk = fp8_inverse(xk), fv = fp8_inverse(xv);
    int wk[E / 4], wv[E / 4];
#pragma unroll
    for (int e = 0; e < E; e += 4) {
      const T x = k[e / kStep], y = v[e / kStep];
      const int i = e % kStep;
      wk[e / 4] = fp8_pack4((float)x[i] * fk, (float)x[i + 1] * fk, (float)x[i + 2] * fk,
                            (float)x[i + 3] * fk);
      wv[e / 4] = fp8_pack4((float)y[i] * fv, (float)y[i + 1] * fv, (float)y[i + 2] * fv,
                            (float)y[i + 3] * fv);
      if (bad) {
        wk[e / 4] = 0x7F7F7F7F;
        wv[e / 4] = 0;
      }
    }
    // value e of the thread lies at this one of the row
    auto place = [&](int e) { return (e / kStep * 4 + quarter) * kStep + e % kStep; };
    typedef int W __attribute__((ext_vector_type(kStep / 4)));
#pragma unroll
    for (int e = 0; e < E; e += kStep) {
      W w;
#pragma unroll
      for (int i = 0; i < kStep / 4; i++) w[i] = wk[e / 4 + i];
      *reinterpret_cast<W*>((whole_k ? s_k : gk) + k_at(tok, place(e))) = w;
    }
    if (few) {
#pragma unroll
      for (int e = 0; e < E; e += 4)
        *reinterpret_cast<int*>(s_v + (tok - off) * DH + place(e)) = wv[e / 4];
    } else if (tok - tid % 4 >= off && tok - tid % 4 + 3 < off + cnt) {
      // all four tokens are new: four values of one token each become four tokens'
      // value d + tid % 4 (bytes change places with the neighbour's, pairs with the pair's)
      const int odd = tid & 1, high = tid & 2;
#pragma unroll
      for (int e = 0; e < E; e += 4) {
        int w = wv[e / 4];
        int o = __builtin_amdgcn_mov_dpp(w, 0xB1, 0xF, 0xF, true);  // lanes 1 0 3 2
        w = __builtin_amdgcn_perm(o, w, odd ? 0x03070105 : 0x06020400);
        o = __builtin_amdgcn_mov_dpp(w, 0x4E, 0xF, 0xF, true);  // lanes 2 3 0 1
        w = __builtin_amdgcn_perm(o, w, high ? 0x03020706 : 0x05040100);
        const int at = v_at(tok - tid % 4, place(e) + tid % 4);
        if (whole_v) *reinterpret_cast<int*>(s_v + spread(at)) = w;
        else *reinterpret_cast<int*>(gv + at) = w;
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; e++) {
        const int at = v_at(tok, place(e));
        const uint8_t c = (uint8_t)(wv[e / 4] >> (e % 4 * 8));
        if (whole_v) s_v[spread(at)] = c;
        else gv[at] = c;
      }
    }
  }
  if (few) {
    __syncthreads();
    for (int i = tid; i < cnt * DH; i += kAppendThreads) gv[v_at(off + i / DH, i % DH)] = s_v[i];
  }
  if (!whole_k && !whole_v) return;  // the scales stay as well
  __syncthreads();
  for (int i = tid * 16; i < kBytes; i += kAppendThreads * 16) {
    // whole lines, past the L2, whose own would be written back at the kernel's end
    if (whole_k)
      __builtin_nontemporal_store(*reinterpret_cast<const v4i*>(s_k + i),
                                  reinterpret_cast<v4i*>(gk + i));
    if (whole_v)
      __builtin_nontemporal_store(*reinterpret_cast<const v4i*>(s_v + spread(i)),
                                  reinterpret_cast<v4i*>(gv + i));
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
