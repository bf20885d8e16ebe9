// The extern "C" entry points of the paged key/value cache: rotation plans, the cache handle, the append and the
// attention that reads it. Argument checks on the host, before the context is used; then the kernel hosts.
#include <math.h>
#include <stdlib.h>

#include <new>

#include "dc_internal.h"

int ops_rope(dc_ctx *, const dc_rope_plan *, const void *, long, const int *, void *, long, int, int, int);
int ops_kv_append(dc_ctx *, const dc_kv_cache *, const dc_rope_plan *, const void *, long, const void *, const void *,
                  float, int, const int *, const int *, void *, long, int, int);
int attn_cache_maps(dc_kv_cache *);
size_t attn_paged_ws(dc_ctx *, const dc_kv_cache *, int, int);
int attn_paged_launch(dc_ctx *, const dc_kv_cache *, const void *, long, const int *, int, const int *, const int *,
                      int, const int *, int, const int *, const int *, int, void *, long, int, int, float, void *);

static bool aln(const void *p, unsigned a) { return ((uintptr_t)p & (a - 1)) == 0; }
static bool al16(const void *p) { return aln(p, 16); }

// Whether n rows of aw halves, as apart, from A and of bw halves, bs apart, from B share no byte.
static bool apart(const void *A, long as, long aw, const void *B, long bs, long bw, long n) {
  const uintptr_t a = (uintptr_t)A, b = (uintptr_t)B;
  const uintptr_t ae = a + 2 * (uintptr_t)((n - 1) * as + aw), be = b + 2 * (uintptr_t)((n - 1) * bs + bw);
  if (ae <= b || be <= a) return true;
  if (as != bs) return false;
  long d = ((long)(b - a) / 2) % as;  // B's first column in A's rows
  if (d < 0) d += as;
  return d >= aw && d + bw <= as;
}

// Whether n rows of aw halves, as apart, from A lie outside `size` bytes from B.
static bool outside(const void *A, long as, long aw, long n, const void *B, uintptr_t size) {
  const uintptr_t a = (uintptr_t)A, ae = a + 2 * (uintptr_t)((n - 1) * as + aw), b = (uintptr_t)B;
  return ae <= b || b + size <= a;
}

static uintptr_t cache_bytes(const dc_kv_cache *c) { return 2 * (uintptr_t)c->pages * c->kv * c->page * c->D; }
static bool clear_of(const void *A, long as, long aw, long n, const dc_kv_cache *c) {
  return outside(A, as, aw, n, c->K, cache_bytes(c)) && outside(A, as, aw, n, c->V, cache_bytes(c));
}

extern "C" int dc_rope_frequencies(int rot, double theta, int scaling, double factor, double trained, double a,
                                   double b, double *h_freq, double *h_factor) {
  DC_CHECK(h_freq && h_factor && rot >= 2 && rot <= 512 && rot % 2 == 0, DC_EINVAL,
           "decision.js: rope_frequencies: rot=%d must be even, 2 to 512", rot);
  DC_CHECK(theta > 1 && isfinite(theta), DC_EINVAL, "decision.js: rope_frequencies: theta must be above 1");
  DC_CHECK(scaling >= DC_ROPE_PLAIN && scaling <= DC_ROPE_BANDS, DC_EINVAL,
           "decision.js: rope_frequencies: unknown scaling %d", scaling);
  DC_CHECK(scaling == DC_ROPE_PLAIN || (factor >= 1 && isfinite(factor)), DC_EINVAL,
           "decision.js: rope_frequencies: factor must be at least 1");
  const bool ramp = scaling == DC_ROPE_YARN || scaling == DC_ROPE_BANDS;
  DC_CHECK(!ramp || (trained > 0 && isfinite(trained) && a > b && b > 0 && isfinite(a)), DC_EINVAL,
           "decision.js: rope_frequencies: the trained context must be positive and a > b > 0");
  DC_CHECK(scaling != DC_ROPE_NTK || rot > 2, DC_EINVAL, "decision.js: rope_frequencies: NTK needs rot above 2");
  const double two_pi = 6.283185307179586476925286766559;
  if (scaling == DC_ROPE_NTK) theta *= pow(factor, rot / (rot - 2.0));
  // YARN ramps over the pair index, between the (whole) indices that make `a` and `b` turns in the trained context
  double lo = 0, hi = 0;
  if (scaling == DC_ROPE_YARN) {
    lo = fmax(floor(rot * log(trained / (a * two_pi)) / (2 * log(theta))), 0);
    hi = fmin(ceil(rot * log(trained / (b * two_pi)) / (2 * log(theta))), rot - 1);
  }
  for (int i = 0; i < rot / 2; i++) {
    const double w = pow(theta, -2.0 * i / rot);
    double keep = 1;  // the share of the plain frequency
    if (scaling == DC_ROPE_LINEAR) keep = 0;
    if (scaling == DC_ROPE_YARN) keep = 1 - fmin(fmax((i - lo) / fmax(hi - lo, 1e-3), 0), 1);
    if (scaling == DC_ROPE_BANDS) keep = fmin(fmax((trained * w / two_pi - b) / (a - b), 0), 1);
    h_freq[i] = keep >= 1 ? w : w * keep + w / factor * (1 - keep);
  }
  *h_factor = scaling == DC_ROPE_YARN ? 0.1 * log(factor) + 1 : 1;
  return DC_OK;
}

extern "C" int dc_rope_plan_create(dc_ctx *ctx, int rot, int layout, const double *h_freq, double factor,
                                   dc_rope_plan **out) {
  DC_CHECK(out && h_freq, DC_EINVAL, "decision.js: rope_plan: null pointer");
  *out = nullptr;
  DC_CHECK(rot >= 16 && rot <= 512 && rot % 16 == 0, DC_EINVAL,
           "decision.js: rope_plan: rot=%d must be a multiple of 16, at most 512", rot);
  DC_CHECK(layout == DC_ROPE_HALF || layout == DC_ROPE_INTERLEAVED, DC_EINVAL,
           "decision.js: rope_plan: unknown layout %d", layout);
  DC_CHECK(isfinite(factor), DC_EINVAL, "decision.js: rope_plan: the factor is not finite");
  uint64_t turns[256];
  for (int i = 0; i < rot / 2; i++) {
    DC_CHECK(isfinite(h_freq[i]), DC_EINVAL, "decision.js: rope_plan: frequency %d is not finite", i);
    const double t = h_freq[i] * 0.15915494309189533576888376337251;  // turns per position
    const double f = t - floor(t);                                      // [0, 1]: 1 when t is a hair below a whole
    turns[i] = f >= 1 ? 0 : (uint64_t)ldexp(f, 64);
  }
  int rc = dc_use(ctx);
  if (rc) return rc;
  dc_rope_plan *p = new (std::nothrow) dc_rope_plan();
  DC_CHECK(p, DC_ENOMEM, "decision.js: rope_plan: out of memory");
  p->device = ctx->device, p->rot = rot, p->layout = layout, p->factor = (float)factor;
  cudaError_t e = cudaMalloc((void **)&p->d_freq, (size_t)rot / 2 * 8);
  if (e != cudaSuccess) {
    cudaGetLastError();
    delete p;
    return dc_fail(DC_ENOMEM, "decision.js: rope_plan: %s", cudaGetErrorString(e));
  }
  e = cudaMemcpyAsync(p->d_freq, turns, (size_t)rot / 2 * 8, cudaMemcpyHostToDevice, ctx->stream);
  if (e == cudaSuccess) e = cudaStreamSynchronize(ctx->stream);
  if (e != cudaSuccess) {
    cudaFree(p->d_freq);
    delete p;
    return dc_fail(DC_ECUDA, "decision.js: rope_plan: %s", cudaGetErrorString(e));
  }
  *out = p;
  return DC_OK;
}

extern "C" int dc_rope_plan_free(dc_rope_plan *plan) {
  if (!plan) return DC_OK;
  cudaSetDevice(plan->device);
  cudaError_t e = cudaFree(plan->d_freq);
  delete plan;
  DC_CHECK(e == cudaSuccess, DC_ECUDA, "decision.js: rope_plan_free: %s", cudaGetErrorString(e));
  return DC_OK;
}

extern "C" int dc_rope(dc_ctx *ctx, const dc_rope_plan *plan, const void *X, long xs, const int32_t *pos, void *Y,
                       long ys, int T, int heads, int D) {
  DC_CHECK(plan && X && pos && Y, DC_EINVAL, "decision.js: rope: null pointer");
  DC_CHECK(T >= 0 && heads > 0 && D > 0 && D % 16 == 0 && D <= 512 && plan->rot <= D, DC_EINVAL,
           "decision.js: rope: D=%d must be a multiple of 16, at most 512, and hold the plan's %d dims", D, plan->rot);
  const long w = (long)heads * D;
  DC_CHECK(xs >= w && ys >= w && xs % 8 == 0 && ys % 8 == 0, DC_EINVAL,
           "decision.js: rope: row strides %ld and %ld must hold %d heads of %d and be multiples of 8", xs, ys, heads, D);
  DC_CHECK(al16(X) && al16(Y) && aln(pos, 4), DC_EINVAL,
           "decision.js: rope: X and Y must be 16-byte aligned, pos 4-byte");
  if (T > 0)
    DC_CHECK((X == Y && xs == ys) || apart(X, xs, w, Y, ys, w, T), DC_EINVAL,
             "decision.js: rope: Y overlaps X without being X");
  int rc = dc_use(ctx);
  if (rc) return rc;
  DC_CHECK(plan->device == ctx->device, DC_EINVAL, "decision.js: rope: the plan is on device %d, the context on %d",
           plan->device, ctx->device);
  if (T == 0) return DC_OK;
  dc_prof_begin(ctx, DC_K_OTHER, 0, 4.0 * T * w);
  rc = ops_rope(ctx, plan, X, xs, pos, Y, ys, T, heads, D);
  dc_prof_end(ctx);
  return rc;
}

extern "C" int dc_kv_cache_create(dc_ctx *ctx, void *K, void *V, int pages, int page, int kv, int D,
                                  dc_kv_cache **out) {
  DC_CHECK(out && K && V, DC_EINVAL, "decision.js: kv_cache: null pointer");
  *out = nullptr;
  DC_CHECK(page == 16 || page == 32 || page == 64 || page == 128, DC_EINVAL,
           "decision.js: kv_cache: a page of %d tokens (16, 32, 64 or 128)", page);
  DC_CHECK(D == 64 || D == 128 || D == 256, DC_EINVAL, "decision.js: kv_cache: head dim %d (64, 128 or 256)", D);
  DC_CHECK(pages > 0 && kv > 0 && (double)pages * kv * page < 2147483648.0, DC_EINVAL,
           "decision.js: kv_cache: %d pages of %d kv heads: pages * kv * page must be below 2^31", pages, kv);
  DC_CHECK(al16(K) && al16(V), DC_EINVAL, "decision.js: kv_cache: K and V must be 16-byte aligned");
  const uintptr_t size = 2 * (uintptr_t)pages * kv * page * D;
  DC_CHECK((uintptr_t)K + size <= (uintptr_t)V || (uintptr_t)V + size <= (uintptr_t)K, DC_EINVAL,
           "decision.js: kv_cache: K and V overlap");
  int rc = dc_use(ctx);
  if (rc) return rc;
  for (void *p : {K, V}) {
    cudaPointerAttributes at;
    DC_CUDA(cudaPointerGetAttributes(&at, p));
    DC_CHECK(at.type == cudaMemoryTypeDevice && at.device == ctx->device, DC_EINVAL,
             "decision.js: kv_cache: %s is not memory of device %d", p == K ? "K" : "V", ctx->device);
  }
  dc_kv_cache *c = new (std::nothrow) dc_kv_cache();
  DC_CHECK(c, DC_ENOMEM, "decision.js: kv_cache: out of memory");
  c->device = ctx->device, c->pages = pages, c->page = page, c->kv = kv, c->D = D;
  c->K = K, c->V = V;
  rc = attn_cache_maps(c);
  if (rc) {
    delete c;
    return rc;
  }
  *out = c;
  return DC_OK;
}

extern "C" int dc_kv_cache_free(dc_kv_cache *cache) {
  delete cache;
  return DC_OK;
}

extern "C" int dc_kv_append(dc_ctx *ctx, const dc_kv_cache *cache, const dc_rope_plan *plan, const void *Z, long zs,
                            const void *qn, const void *kn, float eps, int vnorm, const int32_t *pos,
                            const int32_t *slots, void *Q, long qs, int T, int heads) {
  DC_CHECK(cache && Z && slots && Q && (!plan || pos), DC_EINVAL, "decision.js: kv_append: null pointer");
  DC_CHECK(T >= 0 && heads > 0 && heads % cache->kv == 0, DC_EINVAL,
           "decision.js: kv_append: heads=%d must be a multiple of kv=%d", heads, cache->kv);
  DC_CHECK(!plan || plan->rot <= cache->D, DC_EINVAL, "decision.js: kv_append: the plan turns %d dims of %d-wide heads",
           plan ? plan->rot : 0, cache->D);
  const long zw = ((long)heads + 2L * cache->kv) * cache->D, qw = (long)heads * cache->D;
  DC_CHECK(zs >= zw && qs >= qw && zs % 8 == 0 && qs % 8 == 0, DC_EINVAL,
           "decision.js: kv_append: row strides %ld (q | k | v) and %ld (q) must hold the heads and be multiples of 8",
           zs, qs);
  DC_CHECK(al16(Z) && al16(Q) && al16(qn) && al16(kn) && aln(pos, 4) && aln(slots, 4), DC_EINVAL,
           "decision.js: kv_append: Z, Q and the norm weights must be 16-byte aligned, pos and slots 4-byte");
  if (T > 0)
    DC_CHECK(((Q == Z && qs == zs) || apart(Z, zs, zw, Q, qs, qw, T)) && clear_of(Z, zs, zw, T, cache) &&
                 clear_of(Q, qs, qw, T, cache),
             DC_EINVAL, "decision.js: kv_append: Z, Q and the cache overlap");
  int rc = dc_use(ctx);
  if (rc) return rc;
  DC_CHECK(cache->device == ctx->device && (!plan || plan->device == ctx->device), DC_EINVAL,
           "decision.js: kv_append: the cache or the plan is on another device than the context (%d)", ctx->device);
  if (T == 0) return DC_OK;
  dc_prof_begin(ctx, DC_K_NORM, 0, 4.0 * T * zw);
  rc = ops_kv_append(ctx, cache, plan, Z, zs, qn, kn, eps, vnorm, pos, slots, Q, qs, T, heads);
  dc_prof_end(ctx);
  return rc;
}

static int check_paged(const dc_kv_cache *c, int T, int heads, int S, int G) {
  DC_CHECK(c, DC_EINVAL, "decision.js: attention_paged: null cache");
  DC_CHECK(T >= 0 && S >= 0 && G >= 0, DC_EINVAL, "decision.js: attention_paged: bad sizes T=%d S=%d G=%d", T, S, G);
  DC_CHECK(heads > 0 && heads % c->kv == 0 && heads / c->kv <= 64, DC_EINVAL,
           "decision.js: attention_paged: heads=%d must be a multiple of kv=%d, at most 64 times it", heads, c->kv);
  return DC_OK;
}

extern "C" int dc_attention_paged_workspace(dc_ctx *ctx, const dc_kv_cache *cache, int T, int heads, int S, int G,
                                            size_t *out) {
  DC_CHECK(out, DC_EINVAL, "decision.js: attention_paged: null output");
  int rc = check_paged(cache, T, heads, S, G);
  if (rc) return rc;
  DC_CHECK(ctx, DC_EINVAL, "decision.js: null context");
  *out = attn_paged_ws(ctx, cache, T, heads);
  return DC_OK;
}

extern "C" int dc_attention_paged(dc_ctx *ctx, const dc_kv_cache *cache, const void *Q, long qs, const int32_t *table,
                                  int tstride, const int32_t *lens, const int32_t *qoff, int S, const int32_t *ptable,
                                  int pstride, const int32_t *plens, const int32_t *goff, int G, void *Y, long ys,
                                  int T, int heads, float scale, void *ws, size_t ws_bytes) {
  int rc = check_paged(cache, T, heads, S, G);
  if (rc) return rc;
  DC_CHECK(Q && Y && ws && table && lens && qoff && (G == 0 || (ptable && plens && goff)), DC_EINVAL,
           "decision.js: attention_paged: null pointer");
  const long w = (long)heads * cache->D;
  DC_CHECK(qs >= w && ys >= w && qs % 8 == 0 && ys % 8 == 0, DC_EINVAL,
           "decision.js: attention_paged: row strides %ld and %ld must hold %d heads of %d and be multiples of 8", qs, ys,
           heads, cache->D);
  DC_CHECK(tstride >= 0 && pstride >= 0, DC_EINVAL, "decision.js: attention_paged: negative table stride");
  DC_CHECK(al16(Q) && al16(Y) && al16(ws) && aln(table, 4) && aln(lens, 4) && aln(qoff, 4) && aln(ptable, 4) &&
               aln(plens, 4) && aln(goff, 4),
           DC_EINVAL, "decision.js: attention_paged: Q, Y and the workspace must be 16-byte aligned, the arrays 4-byte");
  if (T > 0)
    DC_CHECK(((Q == Y && qs == ys) || apart(Q, qs, w, Y, ys, w, T)) && clear_of(Y, ys, w, T, cache), DC_EINVAL,
             "decision.js: attention_paged: Y overlaps Q without being Q, or the cache");
  rc = dc_use(ctx);
  if (rc) return rc;
  DC_CHECK(cache->device == ctx->device, DC_EINVAL,
           "decision.js: attention_paged: the cache is on device %d, the context on %d", cache->device, ctx->device);
  const size_t need = attn_paged_ws(ctx, cache, T, heads);
  DC_CHECK(ws_bytes >= need, DC_EINVAL, "decision.js: attention_paged: a workspace of %zu bytes, %zu are needed",
           ws_bytes, need);
  if (T > 0)
    DC_CHECK(outside(Q, qs, w, T, ws, need) && outside(Y, ys, w, T, ws, need) &&
                 clear_of(ws, (long)need, (long)((need + 1) / 2), 1, cache),
             DC_EINVAL, "decision.js: attention_paged: the workspace overlaps Q, Y or the cache");
  if (T == 0 || S == 0) return DC_OK;
  dc_prof_begin(ctx, DC_K_ATTN, 0, 0);
  rc = attn_paged_launch(ctx, cache, Q, qs, table, tstride, lens, qoff, S, ptable, pstride, plens, goff, G, Y, ys, T,
                         heads, scale, ws);
  dc_prof_end(ctx);
  return rc;
}
