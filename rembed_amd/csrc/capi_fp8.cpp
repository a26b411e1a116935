// capi_fp8.cpp — C ABI of the 8-bit floating-point operators: e4m3 weights and
// linears, and the paged e4m3 key/value cache (block tables, append, attention).
//
// Like the rest of the ABI every entry point checks its arguments, returns an
// RH_* status and enqueues on the context's stream. None of these calls allocates
// (rh_linear's workspace apart) or waits, so they can be captured into a HIP graph.
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <memory>
#include <vector>

#include "fp8.h"

namespace rh {

// Device memory of one call.
struct Staging {
  void* p = nullptr;
  ~Staging() {
    if (p) (void)hipFree(p);
  }
};

// The matrices [n][k] of a weight (gate and up, or one alone) to codes and scale bytes, on the
// device: a 4096 x 4096 matrix took the host 42 ms.
static int pack_fp8(Context* ctx, const float* const* mats, int count, const float* bias, int k,
                    int n, rh_weight** out) {
  std::unique_ptr<rh_weight, void (*)(rh_weight*)> w(new rh_weight(), destroy_weight);
  w->ctx = ctx;
  w->mode = RH_MODE_FP8;
  w->k = k;
  w->n = n * count;
  w->glu = count == 2;
  w->kp = (int)round_up(k, kWeightKPad);
  w->np = (int)round_up(w->n, kWeightRowPad);
  const int groups = w->np / kFp8Block;
  const size_t codes = (size_t)w->np * w->kp, exps = (size_t)w->np * (w->kp / kFp8Block);
  const size_t bytes = (size_t)n * k * sizeof(float), flag = round_up(bytes, 8);
  Staging stage;
  RH_HIP(hipMalloc(&stage.p, flag + 8));
  RH_HIP(hipMalloc(&w->d_data, codes));
  RH_HIP(hipMalloc((void**)&w->d_exp, exps));
  RH_HIP(hipMemsetAsync(w->d_data, 0, codes, ctx->stream));
  RH_HIP(hipMemsetAsync(w->d_exp, 0, exps, ctx->stream));
  auto* bad = reinterpret_cast<unsigned long long*>(static_cast<uint8_t*>(stage.p) + flag);
  for (int h = 0; h < count; h++) {
    unsigned long long at = ~0ull;
    RH_HIP(hipMemcpyAsync(bad, &at, 8, hipMemcpyHostToDevice, ctx->stream));
    RH_HIP(hipMemcpyAsync(stage.p, mats[h], bytes, hipMemcpyHostToDevice, ctx->stream));
    RH_HIP(launch_pack_fp8(static_cast<const float*>(stage.p), k, n,
                           static_cast<uint8_t*>(w->d_data), w->kp, w->d_exp, groups,
                           count == 2 ? h : -1, bad, ctx->stream));
    RH_HIP(hipMemcpyAsync(&at, bad, 8, hipMemcpyDeviceToHost, ctx->stream));
    RH_HIP(hipStreamSynchronize(ctx->stream));
    if (at != ~0ull) {
      char buf[160];
      snprintf(buf, sizeof buf, "PackFP8: weight [%llu,%llu] is not finite", at / k, at % k);
      return fail(RH_ERR_NONFINITE, buf);
    }
  }
  if (bias) {
    RH_HIP(hipMalloc((void**)&w->d_bias, n * sizeof(float)));
    RH_HIP(hipMemcpy(w->d_bias, bias, n * sizeof(float), hipMemcpyHostToDevice));
  }
  ctx_retain(ctx);
  *out = w.release();
  return RH_OK;
}

int pack_weight_fp8(Context* ctx, const float* bT, const float* bias, int k, int n,
                    rh_weight** out) {
  return pack_fp8(ctx, &bT, 1, bias, k, n, out);
}

// gate and up keep blocks of their own; rows interleave in groups of kGluGroup.
int pack_weight_fp8_gated(Context* ctx, const float* gate, const float* up, int k, int i,
                          rh_weight** out) {
  const float* mats[2] = {gate, up};
  return pack_fp8(ctx, mats, 2, nullptr, k, i, out);
}

int export_fp8_scales(const rh_weight* w, float* scales, int32_t* colsum) {
  if (colsum) return fail(RH_ERR_INVALID, "weight has no colsum");
  const int kb = w->kp / kFp8Block, groups = w->np / kFp8Block;
  std::vector<uint8_t> exps((size_t)w->np * kb);
  RH_HIP(hipMemcpy(exps.data(), w->d_exp, exps.size(), hipMemcpyDeviceToHost));
  for (int j = 0; j < w->n; j++)
    for (int b = 0; b < kb; b++)
      scales[(size_t)j * kb + b] = ldexpf(1.0f, (int)exps[fp8_scale_at(j, b, groups)] - 127);
  return RH_OK;
}

// Whether m rows of `wa` bytes, `sa` apart, share bytes with m rows of `wb`, `sb` apart. Rows of
// one stride beside each other (columns of one buffer) do not; other strides go by their ranges.
bool rows_overlap(const void* a, size_t wa, size_t sa, const void* b, size_t wb, size_t sb, int m) {
  const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
  const size_t above = (size_t)(m - 1);
  if (m <= 0 || x + above * sa + wa <= y || y + above * sb + wb <= x) return false;
  if (sa != sb) return true;
  const size_t off = y >= x ? (y - x) % sa : (sa - (x - y) % sa) % sa;  // b's rows in a's
  return off < wa || off + wb > sa;
}

int run_linear_fp8(Context* ctx, const rh_weight* w, const void* a, int a_bf16, int lda, int m,
                   void* dst, int dst_bf16, int ldd, int act, const float* bias, uint8_t* qa,
                   int ldq, uint8_t* sa) {
  if (m <= 0) return RH_OK;
  const double M = m, K = w->k, N = w->n;
  // Rows made e4m3 by the product's own workgroups are read while others of them store theirs:
  // not where dst lies on them.
  const size_t ea = a_bf16 ? 2 : 4, ed = dst_bf16 ? 2 : 4, cols = w->glu ? w->n / 2 : w->n;
  const bool direct = a && gemm_fp8_takes_rows(m, w->n, w->k, a, a_bf16, lda) &&
                      !rows_overlap(a, w->k * ea, lda * ea, dst, cols * ed, ldd * ed, m);
  if (a && !direct)
    RH_HIP(launch_quantize_rows_fp8(a, a_bf16, lda, m, w->k, qa, ldq, sa, ctx->stream));
  GemmFp8Args g{};
  g.A = qa;
  g.lda = ldq;
  g.sa = sa;
  g.B = static_cast<const uint8_t*>(w->d_data);
  g.ldb = w->kp;
  g.sb = w->d_exp;
  g.M = m;
  g.N = w->n;
  g.K = w->k;
  g.Np = w->np;
  g.bias = bias;
  g.out = dst;
  g.ldo = ldd;
  g.out_bf16 = dst_bf16;
  g.act = act;
  g.tile_group = ctx->tile_group;
  const double out_b = (dst_bf16 ? 2.0 : 4.0) * (w->glu ? N / 2 : N);
  int slot = -1;
  RH_HIP(ctx->prof_begin(6, 2.0 * M * K * N, M * K + K * N + M * out_b, &slot));
  RH_HIP(launch_gemm_fp8(g, direct ? a : nullptr, a_bf16, lda, ctx->stream));
  RH_HIP(ctx->prof_end(slot));
  return RH_OK;
}

static bool aligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// What rh_linear_fp8 and rh_matmul_fp8 share.
static int check_fp8(const rh_context* ctx, const rh_weight* w, const void* dst, int dst_bf16,
                     int ldd, int m, int act, const void* qa, int ldq, const void* sa) {
  if (!ctx) return fail(RH_ERR_INVALID, "null context");
  if (!w) return fail(RH_ERR_INVALID, "null weight");
  if (w->ctx != ctx) return fail(RH_ERR_INVALID, "weight belongs to another context");
  if (w->mode != RH_MODE_FP8) return fail(RH_ERR_INVALID, "weight must be RH_MODE_FP8");
  if (m < 0) return fail(RH_ERR_INVALID, "negative m");
  if (act < RH_ACT_NONE || act > RH_ACT_GEGLU_ERF) return fail(RH_ERR_INVALID, "unknown act");
  if (w->glu != is_glu(act))
    return fail(RH_ERR_INVALID, "gated acts need a gated weight and vice versa");
  if (m > 0 && (!dst || !qa || !sa)) return fail(RH_ERR_INVALID, "null argument");
  if (ldq != (int)round_up(w->k, kFp8Block))
    return fail(RH_ERR_SHAPE, "ldq must be k rounded up to 128");
  if (ldd < (w->glu ? w->n / 2 : w->n) || ldd % 4)
    return fail(RH_ERR_SHAPE, "ldd must cover the columns and be a multiple of 4");
  if (!aligned(dst, dst_bf16 ? 8 : 16) || !aligned(qa, 16) || !aligned(sa, 4))
    return fail(RH_ERR_INVALID, "dst and qa must be 16-byte (bf16 dst: 8-byte), sa 4-byte aligned");
  return RH_OK;
}

static int check_cache(const rh_kv_cache* c) {
  if (!c) return fail(RH_ERR_INVALID, "null cache");
  if (c->dh != 64 && c->dh != 128 && c->dh != 256)
    return fail(RH_ERR_SHAPE, "cache head dim must be 64, 128 or 256");
  if (c->kv_heads < 1 || c->pages < 0) return fail(RH_ERR_SHAPE, "bad cache shape");
  if (c->pages > 0 && (!c->k || !c->v || !c->k_exp || !c->v_exp))
    return fail(RH_ERR_INVALID, "null cache buffer");
  if (!aligned(c->k, 16) || !aligned(c->v, 16))
    return fail(RH_ERR_INVALID, "cache buffers must be 16-byte aligned");
  return RH_OK;
}

}  // namespace rh

using namespace rh;

extern "C" {

size_t rh_fp8_scale_bytes(int m, int k) {
  if (m <= 0 || k <= 0) return 0;
  return round_up((size_t)m, 128) * ((size_t)(k - 1) / kFp8Block + 1);
}

int rh_quantize_rows_fp8(rh_context* ctx, const void* a, int a_bf16, int lda, int m, int k,
                         uint8_t* qa, int ldq, uint8_t* sa) {
  return api_call([&]() -> int {
    if (m < 0 || k < 1 || k > 0x7FFFFF00) return fail(RH_ERR_INVALID, "bad m/k");
    if (lda < k) return fail(RH_ERR_SHAPE, "lda must be >= k");
    if (ldq != (int)round_up((size_t)k, kFp8Block))
      return fail(RH_ERR_SHAPE, "ldq must be k rounded up to 128");
    if (m > 0 && (!a || !qa || !sa)) return fail(RH_ERR_INVALID, "null argument");
    if (!aligned(a, a_bf16 ? 2 : 4) || !aligned(qa, 16) || !aligned(sa, 4))
      return fail(RH_ERR_INVALID, "misaligned buffer");
    CTX_GUARD(ctx);
    RH_HIP(launch_quantize_rows_fp8(a, a_bf16 ? 1 : 0, lda, m, k, qa, ldq, sa, ctx->stream));
    return RH_OK;
  });
}

int rh_matmul_fp8(rh_context* ctx, void* dst, int dst_bf16, int ldd, const uint8_t* qa, int ldq,
                  const uint8_t* sa, const rh_weight* w, int m, int act) {
  return api_call([&]() -> int {
    int st = check_fp8(ctx, w, dst, dst_bf16, ldd, m, act, qa, ldq, sa);
    if (st) return st;
    CTX_GUARD(ctx);
    return run_linear_fp8(ctx, w, nullptr, 0, 0, m, dst, dst_bf16 ? 1 : 0, ldd, act, w->d_bias,
                          const_cast<uint8_t*>(qa), ldq, const_cast<uint8_t*>(sa));
  });
}

int rh_linear_fp8(rh_context* ctx, void* dst, int dst_bf16, int ldd, const void* a, int a_bf16,
                  int lda, const rh_weight* w, int m, int act, uint8_t* qa, int ldq,
                  uint8_t* sa) {
  return api_call([&]() -> int {
    int st = check_fp8(ctx, w, dst, dst_bf16, ldd, m, act, qa, ldq, sa);
    if (st) return st;
    if (m > 0 && !a) return fail(RH_ERR_INVALID, "null argument");
    if (lda < w->k) return fail(RH_ERR_SHAPE, "lda must be >= k");
    if (!aligned(a, a_bf16 ? 2 : 4)) return fail(RH_ERR_INVALID, "misaligned buffer");
    CTX_GUARD(ctx);
    return run_linear_fp8(ctx, w, a, a_bf16 ? 1 : 0, lda, m, dst, dst_bf16 ? 1 : 0, ldd, act,
                          w->d_bias, qa, ldq, sa);
  });
}

int rh_cache_plan(rh_context* ctx, const int32_t* past, const int32_t* fresh, int batch,
                  const int32_t* free_pages, int n_free, int32_t* table, int ldt, int32_t* cu,
                  int32_t* blocks, int32_t* lens, int64_t* slots, int32_t* pos, int rows,
                  int32_t* status) {
  return api_call([&]() -> int {
    if (batch < 0 || n_free < 0 || rows < 0) return fail(RH_ERR_INVALID, "negative size");
    if (ldt < 1) return fail(RH_ERR_SHAPE, "a table row holds at least one block");
    if (!cu || !blocks || !status) return fail(RH_ERR_INVALID, "null argument");
    if (batch > 0 && (!past || !fresh || !table || !lens))
      return fail(RH_ERR_INVALID, "null argument");
    if ((n_free > 0 && !free_pages) || (rows > 0 && (!slots || !pos)))
      return fail(RH_ERR_INVALID, "null argument");
    if (batch > 0 && (lens == past || lens == fresh))
      return fail(RH_ERR_INVALID, "lens must not be past or fresh: workgroups read those");
    if (!aligned(slots, 8)) return fail(RH_ERR_INVALID, "slots must be 8-byte aligned");
    CTX_GUARD(ctx);
    CachePlanArgs a{past, fresh, batch, free_pages, n_free, table, ldt,
                    cu,   blocks, lens, slots, pos, rows, status};
    RH_HIP(launch_cache_plan(a, ctx->stream));
    return RH_OK;
  });
}

int rh_cache_append(rh_context* ctx, const rh_kv_cache* cache, const void* kv, int kv_bf16,
                    int ldkv, int k_off, int v_off, const int32_t* cu, const int32_t* blocks,
                    const int64_t* slots, int batch, int rows) {
  return api_call([&]() -> int {
    if (int st = check_cache(cache)) return st;
    if (batch < 0 || rows < 0) return fail(RH_ERR_INVALID, "negative size");
    if (batch > 0 && rows > 0 && (!kv || !cu || !blocks || !slots))
      return fail(RH_ERR_INVALID, "null argument");
    const long long width = (long long)cache->kv_heads * cache->dh;
    if (k_off < 0 || v_off < 0 || k_off + width > ldkv || v_off + width > ldkv)
      return fail(RH_ERR_SHAPE, "K and V columns must lie inside the rows");
    if (ldkv % 8 || k_off % 8 || v_off % 8 || !aligned(kv, 16))
      return fail(RH_ERR_SHAPE, "rows and offsets must be multiples of 8 values, kv 16-byte aligned");
    const long long segs = std::min((long long)rows, (long long)rows / RH_CACHE_BLOCK + 2LL * batch);
    if (segs * cache->kv_heads > 0x7FFFFFFF) return fail(RH_ERR_SHAPE, "too many blocks for one call");
    CTX_GUARD(ctx);
    if (batch == 0 || rows == 0 || cache->pages == 0) return RH_OK;
    CacheAppendArgs a{*cache, kv, kv_bf16 ? 1 : 0, ldkv, k_off, v_off, cu, blocks, slots, batch, rows};
    RH_HIP(launch_cache_append(a, ctx->stream));
    return RH_OK;
  });
}

size_t rh_cache_attention_scratch(int batch, int max_q, int max_len, int heads, int kv_heads,
                                  int dh) {
  if (batch <= 0 || max_q <= 0 || max_len < 0 || kv_heads < 1 || heads < kv_heads ||
      heads % kv_heads || dh < 1)
    return 0;
  return cache_attention_floats(batch, max_q, max_len, heads, kv_heads, dh) * sizeof(float);
}

int rh_cache_attention(rh_context* ctx, const void* q, int q_bf16, int ldq, int q_off,
                       const rh_kv_cache* cache, const int32_t* table, int ldt, const int32_t* cu,
                       const int32_t* lens, int batch, int max_q, int max_len, int heads,
                       float scale, int causal, int window, void* out, int out_bf16, int ldout,
                       void* scratch, size_t scratch_bytes) {
  return api_call([&]() -> int {
    if (int st = check_cache(cache)) return st;
    if (batch < 0 || max_q < 0 || max_len < 0 || window < 0)
      return fail(RH_ERR_INVALID, "negative size");
    if (heads < 1 || heads % cache->kv_heads)
      return fail(RH_ERR_SHAPE, "heads must be a positive multiple of kv_heads");
    if (!(scale > 0.0f) || !std::isfinite(scale))
      return fail(RH_ERR_INVALID, "scale must be positive and finite");
    if (ldt < 1 || ldt > 0x7FFFFFFF / RH_CACHE_BLOCK)
      return fail(RH_ERR_SHAPE, "a table row holds at least one block, and positions fit 31 bits");
    const long long width = (long long)heads * cache->dh;
    if (q_off < 0 || q_off + width > ldq || width > ldout)
      return fail(RH_ERR_SHAPE, "the heads' columns must lie inside the rows");
    if (ldq % 8 || q_off % 8 || ldout % 4 || !aligned(q, 16) || !aligned(out, out_bf16 ? 8 : 16))
      return fail(RH_ERR_SHAPE,
                  "q rows and offsets must be multiples of 8 values, q 16-byte, out 16-byte (bf16: "
                  "8-byte) aligned, ldout a multiple of 4");
    const long long tiles = ((long long)max_q * (heads / cache->kv_heads) + 31) / 32;
    if (batch * tiles > 0x3FFFFFFF / cache->kv_heads)
      return fail(RH_ERR_SHAPE, "too many queries for one call");
    if (batch > 0 && max_q > 0 && (!q || !table || !cu || !lens || !out))
      return fail(RH_ERR_INVALID, "null argument");
    const size_t need =
        rh_cache_attention_scratch(batch, max_q, max_len, heads, cache->kv_heads, cache->dh);
    if (need > scratch_bytes || (need && !scratch))
      return fail(RH_ERR_INVALID, "scratch is smaller than rh_cache_attention_scratch says");
    if (!aligned(scratch, 16)) return fail(RH_ERR_INVALID, "scratch must be 16-byte aligned");
    CTX_GUARD(ctx);
    if (batch == 0 || max_q == 0) return RH_OK;
    CacheAttnArgs a{};
    a.q = q;
    a.in_bf16 = q_bf16 ? 1 : 0;
    a.ldq = ldq;
    a.q_off = q_off;
    a.cache = *cache;
    a.table = table;
    a.ldt = ldt;
    a.cu = cu;
    a.lens = lens;
    a.batch = batch;
    a.max_q = max_q;
    a.max_len = max_len;
    a.heads = heads;
    a.scale = scale;
    a.causal = causal ? 1 : 0;
    a.window = window;
    a.out = out;
    a.out_bf16 = out_bf16 ? 1 : 0;
    a.ldout = ldout;
    a.part = static_cast<float*>(scratch);
    RH_HIP(launch_cache_attention(a, ctx->stream));
    return RH_OK;
  });
}

}  // extern "C"
