// capi_rows.cpp — C ABI of the row operators between a layer's products: residual norms, rotary
// positions, the rotary append to the cache and reading it back.
//
// Like the rest of the ABI every entry point checks its arguments, returns an RH_* status and
// enqueues on the context's stream. None but rh_rope_create allocates or waits.
#include <algorithm>
#include <array>
#include <cmath>
#include <initializer_list>
#include <memory>
#include <vector>

#include "rowops.h"

// The frequencies of a turn in HBM.
struct rh_rope {
  rh_context* ctx = nullptr;
  rh::RopeFreq* d_freq = nullptr;
  int pairs = 0, halves = 0;
  float amp = 1.0f;
};

namespace rh {

static bool aligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// Radians a position of each pair, in long double, and amp.
static int rope_frequencies(const rh_rope_config* c, std::vector<long double>& f, double& amp) {
  if (!c) return fail(RH_ERR_INVALID, "null rope config");
  if (c->layout != RH_ROPE_HALVES && c->layout != RH_ROPE_PAIRS)
    return fail(RH_ERR_INVALID, "unknown rope layout");
  if (c->rot < 2 || c->rot > 256 || c->rot % 2)
    return fail(RH_ERR_SHAPE, "rot must be even, 2 to 256");
  if (c->scaling < RH_ROPE_PLAIN || c->scaling > RH_ROPE_GIVEN)
    return fail(RH_ERR_INVALID, "unknown rope scaling");
  if (!std::isfinite((float)c->amp) || c->amp < 0)
    return fail(RH_ERR_INVALID, "amp must be finite in fp32, >= 0");
  const int pairs = c->rot / 2;
  f.resize(pairs);
  amp = 1.0;
  if (c->scaling == RH_ROPE_GIVEN) {
    if (!c->freq) return fail(RH_ERR_INVALID, "RH_ROPE_GIVEN needs freq");
    for (int i = 0; i < pairs; i++) {
      if (!std::isfinite(c->freq[i])) return fail(RH_ERR_NONFINITE, "freq is not finite");
      f[i] = c->freq[i];
    }
    if (c->amp > 0) amp = c->amp;
    return RH_OK;
  }
  if (!std::isfinite(c->theta) || !(c->theta > 1))
    return fail(RH_ERR_INVALID, "theta must be finite and > 1");
  if (!std::isfinite(c->factor) || !(c->factor >= 1))
    return fail(RH_ERR_INVALID, "factor must be finite and >= 1");
  const long double s = c->factor, rot = c->rot, pi2 = 2 * acosl(-1.0L);
  long double theta = c->theta;
  if (c->scaling == RH_ROPE_NTK) {
    if (c->rot < 4) return fail(RH_ERR_SHAPE, "RH_ROPE_NTK needs rot > 2");
    theta *= powl(s, rot / (rot - 2));
  }
  for (int i = 0; i < pairs; i++) f[i] = powl(theta, -2 * i / rot);
  if (c->scaling == RH_ROPE_LINEAR)
    for (auto& x : f) x /= s;
  if (c->scaling == RH_ROPE_YARN || c->scaling == RH_ROPE_WAVELENGTH) {
    const bool yarn = c->scaling == RH_ROPE_YARN;
    const double fast = c->fast == 0 ? (yarn ? 32 : 4) : c->fast, slow = c->slow == 0 ? 1 : c->slow;
    if (c->original < 1) return fail(RH_ERR_INVALID, "the scaling needs original >= 1");
    if (!std::isfinite(fast) || !(slow > 0) || !(fast > slow))
      return fail(RH_ERR_INVALID, "the scaling needs fast > slow > 0");
    const long double n = c->original;
    // i of the pair that turns `turns` times in n positions
    auto pair_of = [&](double turns) { return rot * logl(n / (turns * pi2)) / (2 * logl(theta)); };
    long double lo = std::max(floorl(pair_of(fast)), 0.0L);
    long double hi = std::min(ceill(pair_of(slow)), rot - 1);
    if (lo == hi) hi += 0.001L;
    for (int i = 0; i < pairs; i++) {
      long double stay = yarn ? 1 - (i - lo) / (hi - lo) : (n * f[i] / pi2 - slow) / (fast - slow);
      if (yarn && hi < lo) stay = hi < 0 ? 0 : 1;  // every pair turns under `slow` or over `fast` times
      const long double w = std::min(std::max(stay, 0.0L), 1.0L);
      f[i] = f[i] / s * (1 - w) + f[i] * w;
    }
    if (yarn) amp = 0.1 * log(c->factor) + 1.0;
  }
  if (c->amp > 0) amp = c->amp;
  return RH_OK;
}

// 1 / (2 pi) in binary, 64 bits a word: behind the point as many as the largest double's fraction of
// a turn takes.
static const uint64_t kInvTwoPi[18] = {
    0x28BE60DB9391054A, 0x7F09D5F47D4D3770, 0x36D8A5664F10E410, 0x7F9458EAF7AEF158, 0x6DC91B8E909374B8,
    0x01924BBA82746487, 0x3F877AC72C4A69CF, 0xBA208D7D4BAED121, 0x3A671C09AD17DF90, 0x4E64758E60D4CE7D,
    0x272117E2EF7E4A0E, 0xC7FE25FFF7816603, 0xFBCBC462D6829B47, 0xDB4D9FB3C9F2C26D, 0xD3D18FD9A797FA8B,
    0x5D49EEB1FAF97C5E, 0xCF41CE7DE294A4BA, 0x9AFED7EC47E35742};

// f radians in turns, mod 1, rounded to 64 bits: |f| = m 2^e with m whole, and only the bits of
// 1 / (2 pi) from 2^(-e - 1) on give m 2^e / (2 pi) a fraction, of which the first 192 leave out under
// 2^-128 of a turn. A quotient of long doubles instead would be off by up to 2^-64 of its own size:
// at f = 50 and position 2^31 by 2^-30 of a turn, and by whole turns from f = 2^67 on.
static uint64_t turns_of(long double f) {
  int e;
  const uint64_t m = (uint64_t)ldexpl(frexpl(fabsl(f), &e), 64);
  e -= 64;
  auto bits = [](int from) -> uint64_t {  // 64 of 1 / (2 pi), behind the first `from`
    if (from <= -64) return 0;
    if (from < 0) return kInvTwoPi[0] >> -from;
    auto word = [](int i) -> uint64_t { return i < 18 ? kInvTwoPi[i] : 0; };
    const int i = from / 64, s = from % 64;
    return s ? word(i) << s | word(i + 1) >> (64 - s) : word(i);
  };
  using u128 = unsigned __int128;
  const u128 low = (u128)m * bits(e + 64) + (uint64_t)((u128)m * bits(e + 128) >> 64);
  const uint64_t u = m * bits(e) + (uint64_t)(low >> 64) + ((uint64_t)low >> 63);
  return f < 0 ? 0 - u : u;
}

static void destroy_rope(rh_rope* r) {
  if (r->d_freq) (void)hipFree(r->d_freq);
  delete r;
}

// Rows of `wide` values, `ld` apart, of a buffer.
struct Rows {
  const void* p;
  size_t each, wide, ld;  // bytes
};
static Rows rows_of(const void* p, int bf16, long long wide, int ld) {
  const size_t each = bf16 ? 2 : 4;
  return {p, each, (size_t)wide * each, (size_t)ld * each};
}
// Whether writing `out` may change `in` before it is read: they share bytes and are not the same
// values in the same places.
static bool clash(const Rows& out, const Rows& in, int m) {
  if (!out.p || !in.p || m <= 0) return false;
  if (out.p == in.p && out.each == in.each && out.ld == in.ld) return false;
  return rows_overlap(out.p, out.wide, out.ld, in.p, in.wide, in.ld, m);
}
static bool share(const Rows& a, const Rows& b, int m) {
  return a.p && b.p && m > 0 && rows_overlap(a.p, a.wide, a.ld, b.p, b.wide, b.ld, m);
}

// A stretch of memory that a call reads, or writes as a whole.
struct Bytes {
  const void* p;
  size_t n;
};
static bool meet(const Bytes& a, const Bytes& b) {
  const uintptr_t x = (uintptr_t)a.p, y = (uintptr_t)b.p;
  return a.p && b.p && a.n && b.n && x < y + b.n && y < x + a.n;
}
// Whether a stretch shares bytes with m rows; what lies between two rows is none of theirs.
static bool meet(const Rows& r, int m, const Bytes& a) {
  if (!r.p || !a.p || m <= 0 || !r.wide || !a.n) return false;
  const uintptr_t x = (uintptr_t)r.p, y = (uintptr_t)a.p;
  size_t i = 0;  // the first row that ends behind a's beginning
  if (y >= x + r.wide) {
    if (!r.ld) return false;  // one row for all
    i = (y - x - r.wide) / r.ld + 1;
  }
  return i < (size_t)m && x + i * r.ld < y + a.n;
}
// Whether an output's rows lie on one of the stretches.
static bool on_any(const Rows& out, int m, std::initializer_list<Bytes> all) {
  return std::any_of(all.begin(), all.end(), [&](const Bytes& a) { return meet(out, m, a); });
}
static Bytes ints(const int32_t* p, long long n) { return {p, (size_t)n * sizeof(int32_t)}; }
static Bytes floats(const float* p, int n) { return {p, (size_t)n * sizeof(float)}; }
// What a cache holds: K, V and their scale bytes.
static std::array<Bytes, 4> buffers_of(const rh_kv_cache& c) {
  const size_t heads = (size_t)c.pages * c.kv_heads, codes = heads * RH_CACHE_BLOCK * c.dh;
  return {Bytes{c.k, codes}, Bytes{c.v, codes}, Bytes{c.k_exp, heads}, Bytes{c.v_exp, heads}};
}

// Checks a norm. One of RH_NORM_NONE names no memory: what its other fields hold is not looked at.
static int take_norm(const rh_norm& n, rh_norm& to) {
  to = rh_norm{};
  if (n.kind < RH_NORM_NONE || n.kind > RH_NORM_LAYER) return fail(RH_ERR_INVALID, "unknown norm");
  if (n.kind == RH_NORM_NONE) return RH_OK;
  if (!std::isfinite(n.eps) || n.eps < 0) return fail(RH_ERR_INVALID, "eps must be finite, >= 0");
  if (n.bias && n.kind != RH_NORM_LAYER) return fail(RH_ERR_INVALID, "only a layer norm has a bias");
  if (!aligned(n.weight, 4) || !aligned(n.bias, 4))
    return fail(RH_ERR_INVALID, "misaligned norm weight");
  to = n;
  return RH_OK;
}

static int check_head_norm(const rh_norm* n, HeadNorm& to) {
  to = HeadNorm{};
  rh_norm own{};
  if (!n) return RH_OK;
  if (int st = take_norm(*n, own)) return st;
  if (own.kind == RH_NORM_NONE) return RH_OK;
  if (own.kind != RH_NORM_RMS) return fail(RH_ERR_INVALID, "heads take an RMS norm");
  to = HeadNorm{1, own.eps, own.weight};
  return RH_OK;
}

static int check_rope(const rh_context* ctx, const rh_rope* rope, int dh) {
  if (!ctx) return fail(RH_ERR_INVALID, "null context");
  if (!rope) return fail(RH_ERR_INVALID, "null rope");
  if (rope->ctx != ctx) return fail(RH_ERR_INVALID, "rope belongs to another context");
  if (2 * rope->pairs > dh) return fail(RH_ERR_SHAPE, "rot is more than the head dim");
  return RH_OK;
}

static RopeTurn turn_of(const rh_rope* r) { return {r->d_freq, r->pairs, r->halves, r->amp}; }

// Two ranges of columns.
static bool columns_meet(long long a, long long wa, long long b, long long wb) {
  return wa > 0 && wb > 0 && a < b + wb && b < a + wa;
}

}  // namespace rh

using namespace rh;

extern "C" {

int rh_residual_norm(rh_context* ctx, const rh_residual* r, const void* x, int x_bf16, int ldx,
                     const void* y, int y_bf16, int ldy, void* sum, int ldsum, void* out,
                     int out_bf16, int ldout, uint8_t* qa, int ldq, uint8_t* sa, int m, int n,
                     const int32_t* used) {
  return api_call([&]() -> int {
    if (!r) return fail(RH_ERR_INVALID, "null residual");
    if (m < 0 || n < 1) return fail(RH_ERR_INVALID, "bad m/n");
    if (n > 16384) return fail(RH_ERR_SHAPE, "n must be at most 16384");
    rh_norm post, pre;
    if (int st = take_norm(r->post, post)) return st;
    if (int st = take_norm(r->pre, pre)) return st;
    if (!std::isfinite(r->x_scale) || !std::isfinite(r->y_scale))
      return fail(RH_ERR_INVALID, "scales must be finite");
    if (!y && (post.kind != RH_NORM_NONE || r->gate))
      return fail(RH_ERR_INVALID, "a post norm or gate needs y");
    if (r->gate && r->ldg != 0 && r->ldg < n)
      return fail(RH_ERR_SHAPE, "ldg must be 0 or cover the columns");
    if (!sum && !out && !qa) return fail(RH_ERR_INVALID, "no output");
    if (!qa != !sa) return fail(RH_ERR_INVALID, "codes need their scales, and scales codes");
    if (m > 0 && !x) return fail(RH_ERR_INVALID, "null argument");
    if (ldx < n || (y && ldy < n) || (sum && ldsum < n) || (out && ldout < n))
      return fail(RH_ERR_SHAPE, "rows must cover the columns");
    if (qa && ldq != (int)round_up((size_t)n, kFp8Block))
      return fail(RH_ERR_SHAPE, "ldq must be n rounded up to 128");
    if (!aligned(x, x_bf16 ? 2 : 4) || !aligned(y, y_bf16 ? 2 : 4) ||
        !aligned(sum, x_bf16 ? 2 : 4) || !aligned(out, out_bf16 ? 2 : 4) || !aligned(qa, 16) ||
        !aligned(sa, 4) || !aligned(r->gate, 4) || !aligned(used, 4))
      return fail(RH_ERR_INVALID, "misaligned buffer");
    const Rows rx = rows_of(x, x_bf16, n, ldx), ry = rows_of(y, y_bf16, n, ldy);
    const Rows rs = rows_of(sum, x_bf16, n, ldsum), ro = rows_of(out, out_bf16, n, ldout);
    const Rows rg = rows_of(r->gate, 0, n, r->ldg);
    const Rows rq{qa, 1, (size_t)ldq, (size_t)ldq};
    const Bytes scales{sa, rh_fp8_scale_bytes(m, n)};
    if (clash(rs, rx, m) || clash(rs, ry, m) || share(rs, rg, m) || clash(ro, rx, m) ||
        clash(ro, ry, m) || share(ro, rg, m) || share(rs, ro, m) || share(rq, rx, m) ||
        share(rq, ry, m) || share(rq, rg, m) || share(rq, rs, m) || share(rq, ro, m))
      return fail(RH_ERR_INVALID, "an output overlaps another buffer");
    for (const Rows& rows : {rx, ry, rg, rs, ro, rq})
      if (meet(rows, m, scales)) return fail(RH_ERR_INVALID, "an output overlaps another buffer");
    for (const Bytes& b : {floats(post.weight, n), floats(post.bias, n), floats(pre.weight, n),
                           floats(pre.bias, n), ints(used, 1)})
      if (meet(rs, m, b) || meet(ro, m, b) || meet(rq, m, b) || meet(scales, b))
        return fail(RH_ERR_INVALID, "an output overlaps a norm's weights or used");
    CTX_GUARD(ctx);
    ResidualArgs a{};
    a.x = x;
    a.y = y;
    a.sum = sum;
    a.out = out;
    a.x_bf16 = x_bf16 ? 1 : 0;
    a.ldx = ldx;
    a.y_bf16 = y_bf16 ? 1 : 0;
    a.ldy = ldy;
    a.ldsum = ldsum;
    a.out_bf16 = out_bf16 ? 1 : 0;
    a.ldout = ldout;
    a.qa = qa;
    a.sa = sa;
    a.ldq = ldq;
    a.post = post;
    a.pre = pre;
    a.gate = r->gate;
    a.ldg = r->ldg;
    a.x_scale = r->x_scale;
    a.y_scale = r->y_scale;
    a.used = used;
    a.m = m;
    a.n = n;
    RH_HIP(launch_residual_norm(a, ctx->stream));
    return RH_OK;
  });
}

int rh_rope_frequencies(const rh_rope_config* cfg, double* freq, double* amp) {
  return api_call([&]() -> int {
    std::vector<long double> f;
    double a = 1.0;
    if (int st = rope_frequencies(cfg, f, a)) return st;
    if (freq)
      for (size_t i = 0; i < f.size(); i++) freq[i] = (double)f[i];
    if (amp) *amp = a;
    return RH_OK;
  });
}

int rh_rope_create(rh_context* ctx, const rh_rope_config* cfg, rh_rope** out) {
  return api_call([&]() -> int {
    if (!out) return fail(RH_ERR_INVALID, "null argument");
    std::vector<long double> f;
    double amp = 1.0;
    if (int st = rope_frequencies(cfg, f, amp)) return st;
    // whole turns a position change nothing: positions are whole numbers
    std::vector<RopeFreq> turns(f.size());
    for (size_t i = 0; i < f.size(); i++) {
      const uint64_t u = turns_of(f[i]);
      turns[i] = RopeFreq{(int32_t)(uint32_t)u, (int32_t)(uint32_t)((u + 0x80000000u) >> 32)};
    }
    CTX_GUARD(ctx);
    std::unique_ptr<rh_rope, void (*)(rh_rope*)> r(new rh_rope(), destroy_rope);
    r->ctx = ctx;
    r->pairs = (int)f.size();
    r->halves = cfg->layout == RH_ROPE_HALVES;
    r->amp = (float)amp;
    RH_HIP(hipMalloc((void**)&r->d_freq, turns.size() * sizeof(RopeFreq)));
    RH_HIP(hipMemcpy(r->d_freq, turns.data(), turns.size() * sizeof(RopeFreq),
                     hipMemcpyHostToDevice));
    ctx_retain(ctx);
    *out = r.release();
    return RH_OK;
  });
}

void rh_rope_destroy(rh_rope* rope) {
  api_void([&] {
    if (!rope) return;
    rh_context* ctx = rope->ctx;
    {
      std::lock_guard<std::mutex> lk(ctx->mu);
      (void)hipSetDevice(ctx->device);
      (void)hipStreamSynchronize(ctx->stream);
      destroy_rope(rope);
    }
    ctx_release(ctx);
  });
}

int rh_rope_rows(rh_context* ctx, const rh_rope* rope, const void* x, int x_bf16, int ldx,
                 void* out, int out_bf16, int ldout, int q_off, int k_off, int v_off, int heads,
                 int kv_heads, int dh, const int32_t* pos, int rows, const rh_norm* q_norm,
                 const rh_norm* k_norm, const int32_t* used) {
  return api_call([&]() -> int {
    if (rows < 0 || heads < 0 || kv_heads < 0) return fail(RH_ERR_INVALID, "negative size");
    if (dh < 2 || dh > 256 || dh % 2) return fail(RH_ERR_SHAPE, "dh must be even, 2 to 256");
    if (int st = check_rope(ctx, rope, dh)) return st;
    RopeArgs a{};
    if (int st = check_head_norm(q_norm, a.q_norm)) return st;
    if (int st = check_head_norm(k_norm, a.k_norm)) return st;
    if (v_off < -1) return fail(RH_ERR_SHAPE, "v_off must be a column, or -1");
    if (heads == 0) q_off = 0;  // columns of no head are not looked at
    if (kv_heads == 0) k_off = 0, v_off = -1;
    const bool on_x = out == x && !x_bf16 == !out_bf16 && ldout == ldx;
    const long long wq = (long long)heads * dh, wk = (long long)kv_heads * dh;
    const long long wv = v_off >= 0 ? wk : 0;
    const long long end = std::max({q_off + wq, k_off + wk, wv ? v_off + wv : 0LL});
    if (q_off < 0 || k_off < 0 || end > ldx || end > ldout)
      return fail(RH_ERR_SHAPE, "the heads' columns must lie inside the rows");
    if (columns_meet(q_off, wq, k_off, wk) || columns_meet(q_off, wq, v_off, wv) ||
        columns_meet(k_off, wk, v_off, wv))
      return fail(RH_ERR_SHAPE, "heads share columns");
    if (rows > 0 && wq + wk > 0 && (!x || !out || !pos))
      return fail(RH_ERR_INVALID, "null argument");
    if (!aligned(x, x_bf16 ? 2 : 4) || !aligned(out, out_bf16 ? 2 : 4) || !aligned(pos, 4) ||
        !aligned(used, 4))
      return fail(RH_ERR_INVALID, "misaligned buffer");
    if (!on_x && share(rows_of(out, out_bf16, end, ldout), rows_of(x, x_bf16, end, ldx), rows))
      return fail(RH_ERR_INVALID, "out overlaps x without being it");
    a.v_heads = wv && !on_x ? kv_heads : 0;
    auto written = [&](int off, long long wide) {
      return rows_of(static_cast<char*>(out) + (size_t)off * (out_bf16 ? 2 : 4), out_bf16, wide, ldout);
    };
    for (const Rows& r : {written(q_off, wq), written(k_off, wk), written(v_off, a.v_heads ? wv : 0)})
      if (on_any(r, rows, {floats(a.q_norm.weight, dh), floats(a.k_norm.weight, dh), ints(pos, rows),
                           ints(used, 1)}))
        return fail(RH_ERR_INVALID, "out overlaps a norm's weights, pos or used");
    CTX_GUARD(ctx);
    a.turn = turn_of(rope);
    a.x = x;
    a.out = out;
    a.x_bf16 = x_bf16 ? 1 : 0;
    a.ldx = ldx;
    a.out_bf16 = out_bf16 ? 1 : 0;
    a.ldout = ldout;
    a.q_off = a.q_out = q_off;
    a.k_off = a.k_out = k_off;
    a.v_off = a.v_out = v_off;
    a.heads = heads;
    a.kv_heads = kv_heads;
    a.dh = dh;
    a.pos = pos;
    a.used = used;
    a.rows = rows;
    RH_HIP(launch_rope_rows(a, ctx->stream));
    return RH_OK;
  });
}

int rh_rope_append(rh_context* ctx, const rh_rope* rope, const rh_kv_cache* cache, const void* x,
                   int x_bf16, int ldx, int q_off, int k_off, int v_off, void* q, int q_bf16,
                   int ldq, int heads, const int32_t* pos, const int32_t* cu,
                   const int32_t* blocks, const int64_t* slots, int batch, int rows,
                   const rh_norm* q_norm, const rh_norm* k_norm) {
  return api_call([&]() -> int {
    if (int st = check_cache(cache)) return st;
    if (batch < 0 || rows < 0 || heads < 0) return fail(RH_ERR_INVALID, "negative size");
    if (int st = check_rope(ctx, rope, cache->dh)) return st;
    if (rope->pairs % 8) return fail(RH_ERR_SHAPE, "rot must be a multiple of 16");
    RopeArgs a{};
    if (int st = check_head_norm(q_norm, a.q_norm)) return st;
    if (int st = check_head_norm(k_norm, a.k_norm)) return st;
    if (batch > 0 && rows > 0 && (!x || !pos || !cu || !blocks || !slots || (heads && !q)))
      return fail(RH_ERR_INVALID, "null argument");
    if (heads == 0) q_off = 0;
    const long long wk = (long long)cache->kv_heads * cache->dh, wq = (long long)heads * cache->dh;
    const long long end = std::max({q_off + wq, k_off + wk, v_off + wk});
    if (q_off < 0 || k_off < 0 || v_off < 0 || end > ldx || (heads && wq > ldq))
      return fail(RH_ERR_SHAPE, "the heads' columns must lie inside the rows");
    if (ldx % 8 || q_off % 8 || k_off % 8 || v_off % 8 || !aligned(x, 16) ||
        (heads && (ldq % 8 || !aligned(q, 16))))
      return fail(RH_ERR_SHAPE, "rows and offsets must be multiples of 8 values, x and q 16-byte aligned");
    if (!aligned(pos, 4) || !aligned(slots, 8) || !aligned(cu, 4) || !aligned(blocks, 4))
      return fail(RH_ERR_INVALID, "misaligned buffer");
    // q may lie on its own columns of x, and nowhere else among the rows
    const size_t each = x_bf16 ? 2 : 4;
    const bool on_x = x && q == static_cast<const char*>(x) + q_off * each && !x_bf16 == !q_bf16 && ldq == ldx;
    const Rows out = rows_of(heads ? q : nullptr, q_bf16, wq, ldq);
    if (on_x ? columns_meet(q_off, wq, k_off, wk) || columns_meet(q_off, wq, v_off, wk)
             : share(out, rows_of(x, x_bf16, end, ldx), rows))
      return fail(RH_ERR_INVALID, "q overlaps x without being its own columns");
    CacheAppendArgs c{*cache, x, x_bf16 ? 1 : 0, ldx, k_off, v_off, cu, blocks, slots, batch,
                      cache->pages ? rows : 0};
    a.turn = turn_of(rope);
    a.x = x;
    a.out = q;
    a.x_bf16 = x_bf16 ? 1 : 0;
    a.ldx = ldx;
    a.out_bf16 = q_bf16 ? 1 : 0;
    a.ldout = ldq;
    a.q_off = q_off;
    a.heads = heads;
    a.dh = cache->dh;
    a.pos = pos;
    a.used = cu + batch;
    a.rows = rows;
    if (batch > 0 && rope_append_grid(c, a) >= 1 << 23)
      return fail(RH_ERR_SHAPE, "too many rows for one call");
    if (batch > 0 && rows > 0) {
      const auto read = {ints(pos, rows), ints(cu, batch + 1LL), ints(blocks, batch + 1LL),
                         Bytes{slots, (size_t)rows * sizeof(int64_t)},
                         floats(a.q_norm.weight, cache->dh), floats(a.k_norm.weight, cache->dh)};
      if (on_any(out, rows, read)) return fail(RH_ERR_INVALID, "q overlaps what the call reads");
      const Rows in = rows_of(x, x_bf16, end, ldx);
      for (const Bytes& held : buffers_of(*cache)) {
        if (meet(out, rows, held)) return fail(RH_ERR_INVALID, "q overlaps the cache");
        if (meet(in, rows, held) || std::any_of(read.begin(), read.end(), [&](const Bytes& b) {
              return meet(held, b);
            }))
          return fail(RH_ERR_INVALID, "the cache overlaps what the call reads");
      }
    }
    CTX_GUARD(ctx);
    if (batch == 0 || rows == 0) return RH_OK;
    RH_HIP(launch_rope_append(c, a, ctx->stream));
    return RH_OK;
  });
}

int rh_cache_read(rh_context* ctx, const rh_kv_cache* cache, const int32_t* table, int ldt,
                  const int32_t* cu, const int32_t* first, int batch, int rows, void* out,
                  int out_bf16, int ldout, int k_off, int v_off) {
  return api_call([&]() -> int {
    if (int st = check_cache(cache)) return st;
    if (batch < 0 || rows < 0) return fail(RH_ERR_INVALID, "negative size");
    if (ldt < 1) return fail(RH_ERR_SHAPE, "a table row holds at least one block");
    if (batch > 0 && rows > 0 && (!table || !cu || !out)) return fail(RH_ERR_INVALID, "null argument");
    const long long width = (long long)cache->kv_heads * cache->dh;
    if (k_off < 0 || v_off < 0 || k_off + width > ldout || v_off + width > ldout)
      return fail(RH_ERR_SHAPE, "K and V columns must lie inside the rows");
    if (columns_meet(k_off, width, v_off, width)) return fail(RH_ERR_SHAPE, "K and V share columns");
    if (ldout % 8 || k_off % 8 || v_off % 8 || !aligned(out, 16))
      return fail(RH_ERR_SHAPE, "rows and offsets must be multiples of 8 values, out 16-byte aligned");
    if (!aligned(table, 4) || !aligned(cu, 4) || !aligned(first, 4))
      return fail(RH_ERR_INVALID, "misaligned buffer");
    if (((long long)rows / RH_CACHE_BLOCK + 2LL * batch) * cache->kv_heads >= 1 << 24)
      return fail(RH_ERR_SHAPE, "too many blocks for one call");  // 2^32 threads
    if (batch > 0 && rows > 0) {
      const size_t each = out_bf16 ? 2 : 4;
      for (int off : {k_off, v_off}) {
        const Rows r = rows_of(static_cast<char*>(out) + off * each, out_bf16, width, ldout);
        if (on_any(r, rows, {ints(table, (long long)batch * ldt), ints(cu, batch + 1LL),
                             ints(first, batch)}))
          return fail(RH_ERR_INVALID, "out overlaps what the call reads");
        for (const Bytes& held : buffers_of(*cache))
          if (meet(r, rows, held)) return fail(RH_ERR_INVALID, "out overlaps the cache");
      }
    }
    CTX_GUARD(ctx);
    if (batch == 0 || rows == 0) return RH_OK;
    CacheReadArgs a{*cache, table, ldt, cu, first, batch, rows, out, out_bf16 ? 1 : 0, ldout,
                    k_off, v_off};
    RH_HIP(launch_cache_read(a, ctx->stream));
    return RH_OK;
  });
}

}  // extern "C"
