// Rotary positions with any frequencies, and appending keys and values to a paged cache with the rotation on the way.
//
// Rotation: pair i of a head (dims i and i + rot/2, or 2i and 2i + 1) at position p turns by the angle p w_i:
//   (a, b) -> f (a cos - b sin, b cos + a sin).
// The angle is kept as a fraction of a turn in 64-bit fixed point: a plan holds w_i / 2 pi as a 64-bit fraction (53 bits of
// it, as it comes from a double), and p times it modulo 2^64 is the fraction of a turn left after the whole ones, with no
// further rounding. A 32-bit product p w_i would be off by 2^-24 of itself: 0.06 rad at a million radians. The nearest
// quarter turns are taken out in the same fixed point, and cos and sin of what is left, at most pi/4, are their Taylor
// series (cos_sin): off by 3.2 steps of 2^-24 of themselves at most (and 2^-54), however small, so that each term of a pair is
// good to f32. The hardware's sine is off by 2^-21 of 1, which shows in results that are small beside their pair, by
// hundreds of f16 steps. The series costs more instructions, so the lanes of a warp that need the same angles work
// out a share each and exchange them (4,099 x 10 heads of 256, 64 dims, from the host: 9.2 us with the hardware's sine, 10.0
// with the series in every lane, 9.3 shared; 2,332 rows of 32 + 2 x 8 heads of 64 appended 6.7, 7.6 and 6.6).
//
// Both kernels read and write each row once and are bound by memory (many tokens) or by the launch (few): the rotation of
// 16,384 x 32 heads of 128 takes 42.2 us, 97% of the measured copy rate, the append of 16 x 1,024 tokens of 24 + 2 x 8 heads
// 56.6 us, 91% of it; one token takes 1.6 and 2.5 us (all within a graph).
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>

#include <algorithm>

#include "dc_internal.h"

namespace {

__device__ __forceinline__ uint4 ld16(const __half *p) { return *reinterpret_cast<const uint4 *>(p); }
__device__ __forceinline__ void st16(__half *p, const uint4 &u) { *reinterpret_cast<uint4 *>(p) = u; }

__device__ __forceinline__ void unpack8(const uint4 &u, float (&f)[8]) {
  const __half2 *h = reinterpret_cast<const __half2 *>(&u);
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const float2 v = __half22float2(h[j]);
    f[2 * j] = v.x, f[2 * j + 1] = v.y;
  }
}

__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  uint4 u;
  __half2 *h = reinterpret_cast<__half2 *>(&u);
#pragma unroll
  for (int j = 0; j < 4; j++) h[j] = __floats2half2_rn(f[2 * j], f[2 * j + 1]);
  return u;
}

// cos and sin of `turn` / 2^64 turns. On |x| <= pi/4 the series' next terms, x^11 / 11! and x^12 / 12!, are below 2^-28 of sin
// and 2^-32 of cos.
__device__ __forceinline__ void cos_sin(uint64_t turn, float &cs, float &sn) {
  const uint32_t hi = (uint32_t)(turn >> 32), quarter = (hi + (1u << 29)) >> 30;  // the nearest, modulo 4
  const float x = fmaf((float)(int)(hi - (quarter << 30)), 1.4629180792671596e-9f,  // 2 pi 2^-32
                       (float)(uint32_t)turn * 3.4061215800865545e-19f);            // 2 pi 2^-64
  const float x2 = x * x;
  const float p = fmaf(fmaf(fmaf(1.0f / 362880, x2, -1.0f / 5040), x2, 1.0f / 120), x2, -1.0f / 6);
  const float q = fmaf(fmaf(fmaf(fmaf(-1.0f / 3628800, x2, 1.0f / 40320), x2, -1.0f / 720), x2, 1.0f / 24), x2, -0.5f);
  const float s = fmaf(x * x2, p, x), c = fmaf(x2, q, 1.0f);
  const float a = quarter & 1 ? s : c, b = quarter & 1 ? c : s;
  cs = __uint_as_float(__float_as_uint(a) ^ (((quarter + 1) & 2) << 30));
  sn = __uint_as_float(__float_as_uint(b) ^ ((quarter & 2) << 30));
}

// The eight pairs of a unit, two 16-byte chunks: dims 8c.. and 8c + rot/2.. (half layout), or 16 dims in a row.
template <bool INTER>
__device__ __forceinline__ void rotate(float (&a)[8], float (&b)[8], const float (&cs)[8], const float (&sn)[8]) {
  if (INTER) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float x = a[2 * i], y = a[2 * i + 1], z = b[2 * i], w = b[2 * i + 1];
      a[2 * i] = x * cs[i] - y * sn[i], a[2 * i + 1] = y * cs[i] + x * sn[i];
      b[2 * i] = z * cs[4 + i] - w * sn[4 + i], b[2 * i + 1] = w * cs[4 + i] + z * sn[4 + i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float x = a[i], y = b[i];
      a[i] = x * cs[i] - y * sn[i], b[i] = y * cs[i] + x * sn[i];
    }
  }
}

// The two 16-byte chunks of unit u of a head (D / 16 units): the first rot / 16 units hold the pairs, the others what
// is not rotated.
template <bool INTER>
__device__ __forceinline__ int2 unit_chunks(int u, int rot) {
  const int nr = rot / 16;
  if (INTER || u >= nr) return make_int2(2 * u, 2 * u + 1);
  return make_int2(u, u + nr);
}

// factor * cos and factor * sin of unit u's eight pairs at position p, for SH lanes of a warp, U apart, that need the same:
// each works out 8 / SH of them (this one the sub-th). The whole warp calls it.
template <int SH>
__device__ __forceinline__ void angles8(const uint64_t *freq, bool turn, int u, int U, int sub, int p, float factor,
                                        float (&cs)[8], float (&sn)[8]) {
  constexpr int N = 8 / SH;
  float c[N], s[N];
#pragma unroll
  for (int j = 0; j < N; j++) {
    cos_sin(turn ? (uint64_t)(int64_t)p * freq[8 * u + N * sub + j] : 0, c[j], s[j]);  // modulo one turn
    c[j] *= factor, s[j] *= factor;
  }
  const int first = (threadIdx.x & 31) - U * sub;
#pragma unroll
  for (int e = 0; e < 8; e++) {
    cs[e] = SH == 1 ? c[e % N] : __shfl_sync(0xffffffffu, c[e % N], first + U * (e / N));
    sn[e] = SH == 1 ? s[e % N] : __shfl_sync(0xffffffffu, s[e % N], first + U * (e / N));
  }
}

// A thread takes one unit of one token for every HS-th head, so that its angles serve all of them; consecutive
// threads take the units of a head, then HS heads, then the next token. SH lanes of a warp have the same unit and token.
template <bool INTER, int SH>
__global__ void __launch_bounds__(256) rope_kernel(const __half *X, long xs, const int *pos, __half *Y, long ys, int T,
                                                   int heads, int D, int rot, const uint64_t *freq, float factor,
                                                   int HS, int tpb) {
  dc_pdl_begin();
  const int U = D / 16;
  const int u = threadIdx.x % U, rest = threadIdx.x / U, hs = rest % HS, tok = rest / HS;
  const long t = (long)blockIdx.x * tpb + tok;
  const int2 ch = unit_chunks<INTER>(u, rot);
  const __half *x = X + t * xs;
  __half *y = Y + t * ys;
  const bool turn = u < rot / 16 && tok < tpb && t < T;
  const bool live = tok < tpb && t < T && (turn || X != Y);
  float cs[8], sn[8];
  constexpr int NB = 4;  // heads in flight
  for (int h0 = hs; h0 == hs || (live && h0 < heads); h0 += NB * HS) {
    uint4 ra[NB], rb[NB];
#pragma unroll
    for (int i = 0; i < NB; i++) {
      const int h = h0 + i * HS;
      if (live && h < heads) ra[i] = ld16(x + (long)h * D + 8 * ch.x), rb[i] = ld16(x + (long)h * D + 8 * ch.y);
    }
    // while the first heads are on their way
    if (h0 == hs) angles8<SH>(freq, turn, u, U, hs % SH, turn ? pos[t] : 0, factor, cs, sn);
    if (!live) return;
#pragma unroll
    for (int i = 0; i < NB; i++) {
      const int h = h0 + i * HS;
      if (h >= heads) continue;
      if (turn) {
        float a[8], b[8];
        unpack8(ra[i], a), unpack8(rb[i], b);
        rotate<INTER>(a, b, cs, sn);
        ra[i] = pack8(a), rb[i] = pack8(b);
      }
      st16(y + (long)h * D + 8 * ch.x, ra[i]);
      st16(y + (long)h * D + 8 * ch.y, rb[i]);
    }
  }
}

struct AppendArgs {
  const __half *Z, *qn, *kn;
  const int *pos, *slots;
  __half *Q, *K, *V;
  const uint64_t *freq;
  uint32_t *err;
  long zs, qs;
  int T, heads, kv, rot, page, pshift, nslots, vnorm, W;
  float eps, factor;
};

// W warps per token; a pass of a warp covers 32 / (D/16) of the token's q, k and v heads, U = D/16 lanes to a head
// (one unit each). NP passes are loaded at a time, the next NP while these are worked on: 16 x 1,024 tokens take 57 us with
// two passes at three blocks an SM, 67 with four at two blocks, 62 with two at four, 69 with three at three.
template <int D, bool INTER>
__global__ void __launch_bounds__(256, 3) kv_append_kernel(const AppendArgs a) {
  dc_pdl_begin();
  constexpr int U = D / 16, HPP = 32 / U, NP = 2;
  __shared__ __align__(16) float weights[2][D];  // the norms', in f32: converted once, not in every pass
  const long wid = (long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const long t = wid / a.W;
  const bool live = t < a.T;  // the whole warp
  const int wsub = (int)(wid - t * a.W);
  const int lane = threadIdx.x & 31, u = lane % U, sub = lane / U;
  const int per = a.heads + 2 * a.kv, npass = (per + HPP - 1) / HPP;
  const int2 ch = unit_chunks<INTER>(u, a.rot);
  const __half *z = a.Z + t * a.zs;
  const int slot = live ? a.slots[t] : -1, pos = live && a.pos ? a.pos[t] : 0;
  uint4 ra[NP], rb[NP];
  // q heads are always loaded, k and v heads with them: the slot is not known yet
  auto load = [&](int p0) {
#pragma unroll
    for (int i = 0; i < NP; i++) {
      const int h = (p0 + i * a.W) * HPP + sub;
      ra[i] = rb[i] = make_uint4(0, 0, 0, 0);
      if (live && h < per) ra[i] = ld16(z + (long)h * D + 8 * ch.x), rb[i] = ld16(z + (long)h * D + 8 * ch.y);
    }
  };
  load(wsub);
  if (a.qn || a.kn) {
    for (int d = threadIdx.x; d < D; d += 256) {
      if (a.qn) weights[0][d] = __half2float(a.qn[d]);
      if (a.kn) weights[1][d] = __half2float(a.kn[d]);
    }
    __syncthreads();
  }
  if (!live) return;
  const bool turn = u < a.rot / 16, stored = slot >= 0 && slot < a.nslots;
  if (slot >= a.nslots && lane == 0) atomicOr(a.err, (uint32_t)DC_DEVERR_BOUNDS);
  const int pg = slot >> a.pshift, off = slot & (a.page - 1);
  float cs[8], sn[8];
  if (a.rot) angles8<HPP>(a.freq, turn, u, U, sub, pos, a.factor, cs, sn);
  for (int p0 = wsub; p0 < npass; p0 += NP * a.W) {
    uint4 xa[NP], xb[NP];
#pragma unroll
    for (int i = 0; i < NP; i++) xa[i] = ra[i], xb[i] = rb[i];
    if (p0 + NP * a.W < npass) load(p0 + NP * a.W);
#pragma unroll
    for (int i = 0; i < NP; i++) {
      const int h = (p0 + i * a.W) * HPP + sub;
      const bool isq = h < a.heads, isk = !isq && h < a.heads + a.kv;
      const bool normed = isq ? a.qn != nullptr : isk ? a.kn != nullptr : a.vnorm != 0;
      float x[8], y[8];
      unpack8(xa[i], x), unpack8(xb[i], y);
      if (a.qn || a.kn || a.vnorm) {
        float s0 = 0.f, s1 = 0.f;
#pragma unroll
        for (int e = 0; e < 8; e++) s0 = fmaf(x[e], x[e], s0), s1 = fmaf(y[e], y[e], s1);
        float ss = s0 + s1;
#pragma unroll
        for (int o = U / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);  // every lane of the warp
        if (normed) {
          const float inv = rsqrtf(ss * (1.0f / D) + a.eps);
          const float *w = weights[isq ? 0 : 1];
#pragma unroll
          for (int e = 0; e < 8; e += 4) {
            float4 wx = make_float4(inv, inv, inv, inv), wy = wx;
            if (isq || isk) {
              const float4 px = *reinterpret_cast<const float4 *>(w + 8 * ch.x + e);
              const float4 py = *reinterpret_cast<const float4 *>(w + 8 * ch.y + e);
              wx = make_float4(px.x * inv, px.y * inv, px.z * inv, px.w * inv);
              wy = make_float4(py.x * inv, py.y * inv, py.z * inv, py.w * inv);
            }
            x[e] *= wx.x, x[e + 1] *= wx.y, x[e + 2] *= wx.z, x[e + 3] *= wx.w;
            y[e] *= wy.x, y[e + 1] *= wy.y, y[e + 2] *= wy.z, y[e + 3] *= wy.w;
          }
        }
      }
      if (h >= per) continue;
      if (turn && (isq || isk)) rotate<INTER>(x, y, cs, sn);
      __half *dst;
      if (isq) {
        dst = a.Q + t * a.qs + (long)h * D;
      } else {
        if (!stored) continue;
        const int hk = h - a.heads - (isk ? 0 : a.kv);
        dst = (isk ? a.K : a.V) + ((((long)pg * a.kv + hk) << a.pshift) + off) * D;
      }
      st16(dst + 8 * ch.x, pack8(x));
      st16(dst + 8 * ch.y, pack8(y));
    }
  }
}

}  // namespace

int ops_rope(dc_ctx *ctx, const dc_rope_plan *p, const void *X, long xs, const int *pos, void *Y, long ys, int T,
             int heads, int D) {
  const int U = D / 16;
  // Heads apart: 4 (a warp's threads cover 64 U halves in a row) unless that leaves the card without threads. 16,384 x 32
  // heads: 42.2 us with 4, 57.6 with 1 (whose lanes share no angles), 68.6 with as many as fit (each thread has its angles for
  // fewer heads); one token of 32 heads 2.4 us with 4, 1.6 with as many as fit.
  const long want = (1024L * ctx->sms + (long)T * U - 1) / ((long)T * U);
  const int most = std::max(1, std::min(heads, 256 / U));
  const int HS = (int)std::min<long>(most, std::max<long>(want, std::min(4, most)));
  const int tpb = std::max(1, 256 / (U * HS));
  const dim3 grid((unsigned)((T + (long)tpb - 1) / tpb));
  // Lanes of a warp with one unit and token, which share the angles' work: 4,099 x 10 heads of 256 9.3 us with two, 10.0 with
  // one.
  const int SH = 32 % U ? 1 : 32 / U >= 4 && HS % 4 == 0 ? 4 : 32 / U >= 2 && HS % 2 == 0 ? 2 : 1;
  const bool inter = p->layout == DC_ROPE_INTERLEAVED;
  auto *kernel = SH == 4   ? (inter ? rope_kernel<true, 4> : rope_kernel<false, 4>)
                 : SH == 2 ? (inter ? rope_kernel<true, 2> : rope_kernel<false, 2>)
                           : (inter ? rope_kernel<true, 1> : rope_kernel<false, 1>);
  DC_CUDA(dc_launch_pdl(ctx->stream, kernel, grid, dim3(256), 0, (const __half *)X, xs, pos, (__half *)Y, ys, T, heads, D, p->rot,
                        p->d_freq, p->factor, HS, tpb));
  return dc_launch_check("rope");
}

int ops_kv_append(dc_ctx *ctx, const dc_kv_cache *c, const dc_rope_plan *p, const void *Z, long zs, const void *qn,
                  const void *kn, float eps, int vnorm, const int *pos, const int *slots, void *Q, long qs, int T,
                  int heads) {
  AppendArgs a;
  a.Z = (const __half *)Z, a.qn = (const __half *)qn, a.kn = (const __half *)kn;
  a.pos = pos, a.slots = slots;
  a.Q = (__half *)Q, a.K = (__half *)c->K, a.V = (__half *)c->V;
  a.freq = p ? p->d_freq : nullptr, a.factor = p ? p->factor : 1.0f, a.rot = p ? p->rot : 0;
  a.err = ctx->d_err;
  a.zs = zs, a.qs = qs;
  a.T = T, a.heads = heads, a.kv = c->kv, a.page = c->page, a.nslots = c->pages * c->page;
  a.pshift = c->page == 16 ? 4 : c->page == 32 ? 5 : c->page == 64 ? 6 : 7;
  a.vnorm = vnorm, a.eps = eps;
  const int npass = (heads + 2 * c->kv + 512 / c->D - 1) / (512 / c->D);
  // Warps per token: one, which works the angles out once for all heads, unless that leaves the card without warps.
  // 16 x 1,024 tokens of 24 + 2 x 8 heads: 57 us with one, 125 with a warp to every pass; one token 6.6 us with one, 2.5
  // with a warp to every pass.
  a.W = (int)std::max<long>(1, std::min<long>(npass, (32L * ctx->sms + T - 1) / T));
  const dim3 grid((unsigned)(((long)T * a.W + 7) / 8));
  const bool inter = p && p->layout == DC_ROPE_INTERLEAVED;
#define APPEND(DD)                                                                                               \
  if (c->D == DD)                                                                                                \
    DC_CUDA(dc_launch_pdl(ctx->stream, inter ? kv_append_kernel<DD, true> : kv_append_kernel<DD, false>, grid,   \
                          dim3(256), 0, a));
  APPEND(64) APPEND(128) APPEND(256)
#undef APPEND
  return dc_launch_check("kv_append");
}
