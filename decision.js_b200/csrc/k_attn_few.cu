// The attention over the paged cache for groups of few rows (a decode step: some sequences at one token each). The line
// of blocks, its cutting and the join are those of the wide kernel (k_attn_paged.cu), as are the tiles of 128 rows; here
// most rows of a tile are empty and what has to flow is the cache. What a block costs then is the latency of its chain
// (scores, maximum, weights, product), so two CTAs share an SM and within each two warps share a row:
//   warps 0-7  softmax: two warps per TMEM lane quadrant, thread = row, each half of a block's keys; the halves' maxima
//              meet in shared memory. Quadrants without rows only keep step.
//   warp 8     walks the line, loads K and Q; warp 9 walks it and loads V; warp 10 Q K^T and P V (and TMEM); warp 11 looks
//              values over
// Blocks are 64 keys with two scores' buffers, which leaves each warp 32 scores: they stay in registers from the maximum
// to the weights. The weights are scaled by 2^7 as in the wide kernel.
// Bound by the chain of a block at D = 64 (0.9 us for 64 keys, two CTAs at a time: 218 sequences of one token over 24
// prefixes of up to 6,000 tokens, 32 heads over 8, 90 us where the bytes need 44.5), by memory while it streams at D = 128
// (35 sequences of one token over a shared prefix of 18,000 tokens, 16 heads over 8: 36 us where the bytes need 18.6; 22 us
// of streaming, 4 for the line, 4 until the first keys are there, 5 for the last CTAs and the join). 32 groups of 3
// questions of 40 tokens over 512 tokens take 58 us, of which the way from one tile to the next is the most. Kept steps: two
// CTAs an SM with halves of rows 45 -> 40 us on the second; one code for both producers, Q after the keys, Q K^T from a loop
// 73 -> 61 on the third (see the instruction caches in the wide kernel). Measured and not taken: blocks of 128 keys in one
// scores' buffer at D = 64, one pass with the weights kept in registers, products by warps' own matrix instructions, waits
// that poll (but for the halves' exchange of maxima: 24 prefixes, D = 64, 99.7 -> 95.1 us), rows of an SM's second CTA on
// the other two quadrants.
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <float.h>

#include "dc_internal.h"
#include "dc_paged.cuh"
#include "dc_ptx.cuh"

using namespace dcx;

namespace {

constexpr int FS = 8;  // softmax warps
constexpr int FW_K = FS, FW_V = FS + 1, FW_M = FS + 2, FW_C = FS + 3;
constexpr int F_THREADS = (FS + 4) * 32;

template <int D>
struct FewCfg {
  static constexpr int KB = 64, SB = 2;  // keys of a block; scores' buffers
  static constexpr int NA = D / 64, Q_ROWS = 128, THREADS = F_THREADS;
  static constexpr int KST = D == 64 ? 4 : 2, VST = KST;
  static constexpr int Q_BYTES = Q_ROWS * D * 2, KV_BYTES = KB * D * 2;
  static constexpr int K_OFF = Q_BYTES, V_OFF = K_OFF + KST * KV_BYTES;
  static constexpr int BAR_OFF = V_OFF + VST * KV_BYTES;
  static constexpr int B_QF = 0, B_QE = 1, B_OD = 2, B_OE = 3, B_OR = 4, B_SF = 5, B_PF = B_SF + SB,
                       B_KF = B_PF + SB, B_KE = B_KF + KST, B_VF = B_KE + KST, B_VE = B_VF + VST, B_VS = B_VE + VST,
                       B_IF = B_VS + VST, B_IE = B_IF + PA_RING, B_END = B_IE + PA_RING, NBARS = B_END + 2;
  static constexpr int MISC_OFF = BAR_OFF + ((NBARS * 8 + 15) & ~15), LOADED_OFF = MISC_OFF + 20;
  static constexpr int POISON_OFF = MISC_OFF + 32, SCAN_OFF = POISON_OFF + PA_MARK_BYTES,
                       RUN_OFF = SCAN_OFF + ((F_THREADS / 32 * 8 + 15) & ~15), GOFF_OFF = RUN_OFF + PA_RING * (int)sizeof(Run),
                       XCH_OFF = GOFF_OFF + PA_META;  // (turn, value), 64 bits [2 turns][2 halves][128 rows]
  static constexpr int SMEM = XCH_OFF + 2 * 2 * 128 * 8 + 1024;
  static constexpr int S_COL = 0, O_COL = SB * KB, TCOLS = 256;
  static_assert(O_COL + D <= TCOLS, "tensor memory");
  static_assert(XCH_OFF % 8 == 0, "64-bit accesses");
  static_assert(2 * (SMEM + 1024) <= 228 * 1024, "shared memory");  // (1 KB of each CTA's is the system's)
};

template <int D>
__global__ void __launch_bounds__(F_THREADS, 2)
    attention_paged_few_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                               const __grid_constant__ CUtensorMap tmV, const PArgs a) {
  using C = FewCfg<D>;
  constexpr int KB = C::KB, SB = C::SB, KST = C::KST, VST = C::VST, COLS = KB / 2;
  extern __shared__ uint8_t smem_raw[];
  const Cta<C> k(a, smem_raw);
  const int tid = k.tid, warp = k.warp, lane = k.lane;
  if (tid == 0) {
    for (int i = 0; i < C::NBARS; i++) {
      const int n = i == C::B_OE || (i >= C::B_PF && i < C::B_PF + SB) ? FS
                    : i >= C::B_VE && i < C::B_VE + VST                ? 2
                    : i >= C::B_IE && i < C::B_END                     ? FS + 2
                                                                       : 1;
      mbar_init(k.bar(i), n);
    }
    *k.abort() = 0;
    mbar_init_fence();
  }
  k.clear_marks();
  for (int i = tid; i < 512; i += F_THREADS) reinterpret_cast<int2 *>(k.smem + C::XCH_OFF)[i] = make_int2(0, 0);
  if (warp == FW_K && lane == 0) tma_prefetch_desc(&tmQ), tma_prefetch_desc(&tmK);
  if (warp == FW_V && lane == 0) tma_prefetch_desc(&tmV);
  // (tensor memory after the kernels before, and before the next is let in: see the wide kernel)
  dc_pdl_wait();
  if (warp == FW_M) tmem_alloc(smem_u32(k.tmem_slot()), C::TCOLS);
  Groups gs;
  Stretch st;
  const bool fine = line_start(k, gs, st);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *k.tmem_slot();

  if (!fine || st.p0 >= st.p1) {
  } else if (warp == FW_K || warp == FW_V) {
    walk_line(k, gs, st, warp == FW_V, &tmQ, warp == FW_V ? &tmV : &tmK);
  } else if (warp == FW_C) {
    look_over(k);
  } else if (warp == FW_M) {
    constexpr uint32_t idesc_qk = idesc_f16_f32(128, KB);
    constexpr uint32_t idesc_pv = idesc_f16_f32(128, D) | (1u << 16);  // V MN-major
    const uint64_t q0 = desc_sw128(k.base), k0 = desc_sw128(k.base + C::K_OFF), v0 = desc_mn(k.base + C::V_OFF, KB * 128);
    Run r = {};
    int g = 0;
    bool ok = true, pend = false, begins = true;  // begins: the tile has had no block yet
    int looked = 0;
    bool look = false;     // whether the pending product's (block g - 1) values are looked over first,
    int steps = 0;         // its steps of 16 keys,
    uint32_t off[4] = {};  // and the rows that it leaves alone
    auto pv = [&](int x) -> bool {
      const int vs = x % VST;
      if (!k.wait_warp(C::B_VF + vs, x / VST)) return false;
      if (look) {
        if (!k.wait_warp(C::B_VS + looked % VST, looked / VST)) return false;
        looked++;
      }
      if (!k.wait_warp(C::B_PF + x % SB, x / SB)) return false;
      tc_fence_after();
      // the weights of keys [0, COLS) begin the scores' buffer, those of [COLS, KB) its second half
      const uint32_t p = tmem + (uint32_t)(C::S_COL + x % SB * KB);
      const uint64_t v = v0 + (uint32_t)(vs * C::KV_BYTES >> 4);
      if (elect_one()) {
#pragma unroll 1
        for (int kk = 0; kk < steps; kk++)
          mma_f16_ts_rows(tmem + C::O_COL, p + (kk * 16 < COLS ? 8 * kk : COLS + 8 * kk - COLS / 2), v + kk * (2048 >> 4),
                            idesc_pv, off);
        mma_commit(k.bar(C::B_VE + vs));
        mma_commit(k.bar(C::B_OR));
      }
      __syncwarp();
      return true;
    };
    for (int n = 0; ok && k.next_run(n, r); n++) {
      if (r.flags & RUN_FIRST) ok = k.wait_warp(C::B_QF, r.item), begins = true;
      // each turn a block's scores and the product before them; the tile's last run has one more for its last product
      const bool last = (r.flags & RUN_LAST) != 0;
      for (int b = 0; ok && b < r.nb + last; b++) {
        const int key0 = (r.kb + b) * KB;
        const bool more = b < r.nb;
        if (more) {
          const int ks = g % KST;
          if (!(ok = k.wait_warp(C::B_KF + ks, g / KST))) break;
          tc_fence_after();
          if (elect_one()) {
            const uint32_t sc = tmem + (uint32_t)(C::S_COL + g % SB * KB);
            const uint64_t kd0 = k0 + (uint32_t)(ks * C::KV_BYTES >> 4);
#pragma unroll 1
            for (int kd = 0; kd < D / 16; kd++)
              mma_f16(sc, q0 + (((kd >> 2) * 128 * 128 + (kd & 3) * 32) >> 4),
                      kd0 + (((kd >> 2) * KB * 128 + (kd & 3) * 32) >> 4), idesc_qk, kd > 0);
            mma_commit(k.bar(C::B_SF + g % SB));
            mma_commit(k.bar(C::B_KE + ks));
          }
          __syncwarp();
        }
        if (last && b == max(r.nb - 1, 0)) {
          if (elect_one()) mma_commit(k.bar(C::B_QE));
          __syncwarp();
        }
        if (pend && !(ok = pv(g - 1))) break;
        pend = more;
        if (!more) break;
        begins = false, g++;
        look = to_look_over<KB>(r, key0);
        steps = (min(KB, r.kend - key0) + 15) >> 4;
        // own blocks: the rows of the sequence that see a key of it
        const int lo = r.seg < 0 ? 0 : (max(max(r.tok0, r.qb), key0 - r.len + r.qe) - r.tok0) * a.r;
        const int hi = r.seg < 0 ? 128 : (min(r.qe, r.tok0 + r.ntok) - r.tok0) * a.r;
#pragma unroll
        for (int w = 0; w < 4; w++) off[w] = ~mask_word(lo, hi, w);
      }
      if (ok && last) {
        // a tile without keys: the last tile's end has to be past before this one's is announced
        if (begins) ok = k.wait_warp(C::B_OE, r.item + 1);
        if (ok && elect_one()) mma_commit(k.bar(C::B_OD));
        __syncwarp();
      }
      if (ok) k.done_run(n);
    }
  } else {
    const int q = warp & 3, hf = warp >> 2;
    const int row = 32 * q + lane, irow = row / a.r, jrow = row - irow * a.r;
    const uint32_t lrow = tmem + ((uint32_t)(32 * q) << 16), ocol = lrow + (uint32_t)(C::O_COL + hf * (D / 2));
    const uint32_t xch = k.base + C::XCH_OFF + 8 * row;
    int g = 0, meets = 0;
    bool ok = true;
    // the tile's state
    bool valid = false, anyv = false, seen = false, tfirst = false;  // seen: the row has seen a key
    int t = 0;
    float ref = -FLT_MAX, l = 0.f;
    // Gives this half's value of the row and takes the other's: both write theirs with the number of the turn, in one
    // 64-bit store (a vector of two would be two, in any order), and look for the other's (a half writes to a place again
    // only when the other has read it: it has then seen the other's value of the turn between).
    auto meet = [&](float mine, float &theirs) -> bool {
      const uint32_t at = xch + (meets & 1) * 2048, mark = ++meets;
      const uint64_t put = (uint64_t)mark << 32 | __float_as_uint(mine);
      asm volatile("st.volatile.shared.b64 [%0], %1;" ::"r"(at + 1024 * hf), "l"(put) : "memory");
      uint64_t t0 = 0;
#pragma unroll 1
      for (uint32_t i = 1;; i++) {
        uint64_t got;
        asm volatile("ld.volatile.shared.b64 %0, [%1];" : "=l"(got) : "r"(at + 1024 * (hf ^ 1)) : "memory");
        const uint32_t seen = (uint32_t)(got >> 32);
        theirs = __uint_as_float((uint32_t)got);
        if (__all_sync(0xffffffffu, seen == mark)) return true;
        if ((i & 1023) == 0) {
          const uint64_t now = globaltimer();
          t0 = t0 ? t0 : now;
          if (now - t0 > 2000000000ull) *k.abort() = 1, atomicOr(a.err, (uint32_t)DC_DEVERR_ATTN_WAIT);
          if (__any_sync(0xffffffffu, *k.abort() != 0)) return false;
        }
      }
    };
    for (int n = 0; ok && k.wait_warp(C::B_IF + n % PA_RING, n / PA_RING); n++) {
      const Run &r = k.runs()[n % PA_RING];  // (stays as it is until done_run)
      if (r.flags & RUN_END) break;
      if (r.flags & RUN_FIRST) {
        t = r.tok0 + irow;
        valid = irow < r.ntok && irow < a.tpt;
        anyv = __any_sync(0xffffffffu, valid);
        seen = false, tfirst = (r.flags & RUN_TFIRST) != 0;
        ref = -FLT_MAX, l = 0.f;
        if (anyv) {  // the accumulator to zero; the last tile's was read by this very warp
          const uint32_t z[16] = {};
          __syncwarp();
#pragma unroll 1
          for (int c = 0; c < D / 2; c += 16) tmem_st16(ocol + c, z);
          tmem_st_wait();
          tc_fence_before();
        }
      }
      // the run's keys that the row sees
      const int rlim = !valid ? 0 : r.seg < 0 ? r.kend : t >= r.qb && t < r.qe ? own_limit(t, r.qe, r.len) : 0;
      const int nb = r.nb, kb = r.kb;
      seen = seen || (nb > 0 && rlim > kb * KB);
      // the run's first blocks that every row here sees whole (lanes without a row have no say)
      const int full = __reduce_min_sync(0xffffffffu, valid ? rlim : 0x7fffffff) / KB - kb;
      for (int b = 0; b < nb; b++, g++) {
        const int sb = g % SB;
        if (!(ok = k.wait_warp(C::B_SF + sb, g / SB))) break;
        const int nv = rlim - (kb + b) * KB;  // its keys that the row sees (or fewer than none, or more than there are)
        const bool part = b >= full;
        if (part ? __any_sync(0xffffffffu, nv > 0) : anyv) {
          tc_fence_after();
          const uint32_t scol = lrow + (uint32_t)(C::S_COL + sb * KB + hf * COLS);
          float sc = a.scale_log2;
          uint32_t x[32];
          __syncwarp();
          tmem_ld32(scol, x);
          tmem_ld_wait(x);
          if (sc <= 0.f) {  // the largest score is not the largest product: scale first
#pragma unroll
            for (int e = 0; e < 32; e++) x[e] = __float_as_uint(__uint_as_float(x[e]) * sc);
            sc = 1.f;
          }
          if (part)  // minus infinity where the row does not see the key
#pragma unroll
            for (int e = 0; e < 32; e++) x[e] = hf * COLS + e < nv ? x[e] : 0xff800000u;
          float m2[2] = {MINUS_INF, MINUS_INF};
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            m2[0] = max3(m2[0], __uint_as_float(x[e]), __uint_as_float(x[e + 1]));
            m2[1] = max3(m2[1], __uint_as_float(x[e + 2]), __uint_as_float(x[e + 3]));
          }
          const float pmx = fmaxf(m2[0], m2[1]) * sc;
          float omx;
          if (!(ok = meet(pmx, omx))) break;
          const float mx = fmaxf(pmx, omx);
          const bool grow = mx > ref + 8.0f;
          const bool resc = grow && ref > -FLT_MAX;
          if (__any_sync(0xffffffffu, resc)) {
            if (!(ok = k.wait_warp(C::B_OR, g - 1))) break;  // the products so far
            tc_fence_after();
            const float f = resc ? ex2_approx(ref - mx) : 1.0f;
            l *= f;
#pragma unroll 1
            for (int c = 0; c < D / 2; c += 16) {
              uint32_t o[16];
              __syncwarp();
              tmem_ld16(ocol + c, o);
              tmem_ld_wait(o);
#pragma unroll
              for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              __syncwarp();
              tmem_st16(ocol + c, o);
            }
            tmem_st_wait();
          }
          if (grow) ref = mx;
          const uint64_t ref2 = f32x2(7.0f - ref, 7.0f - ref), sc2 = f32x2(sc, sc);
          uint64_t sum[2] = {0, 0};
          uint32_t w[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float2 v = f32x2_split(fma_f32x2(f32x2(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), sc2, ref2));
            const float p0 = ex2_approx(v.x), p1 = ex2_approx(v.y);
            sum[(e >> 1) & 1] = add_f32x2(sum[(e >> 1) & 1], f32x2(p0, p1));
            const __half2 hp = __floats2half2_rn(p0, p1);
            w[e / 2] = *reinterpret_cast<const uint32_t *>(&hp);
          }
          // 32 weights over 16 of this warp's own scores, all done with
          __syncwarp();
          tmem_st16(scol, w);
          const float2 add = f32x2_split(add_f32x2(sum[0], sum[1]));
          l += add.x + add.y;
          tmem_st_wait();
        }  // none of these rows sees the block: the product leaves them alone
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(k.bar(C::B_PF + sb));
      }
      if (!ok) break;
      if (r.flags & RUN_LAST) {
        const bool tlast = (r.flags & RUN_TLAST) != 0, direct = tfirst && tlast;
        if (!direct && !a.by_row && tid == 0) {
          if (tlast) a.head[blockIdx.x] = make_int4(r.tok0, r.ntok, r.kvh, 0);
          if (tfirst) a.tail[blockIdx.x] = 1;
        }
        float lt = 0.f;
        if (anyv) {  // the sums meet while the last product runs
          float ol;
          if (!(ok = meet(l, ol))) break;
          lt = l + ol;
        }
        if (!(ok = k.wait_warp(C::B_OD, r.item))) break;
        tc_fence_after();
        if (anyv) {
          if (seen && ((k.poison(r.item)[irow >> 5] >> (irow & 31)) & 1u)) lt = __int_as_float(0x7fc00000);
          if (seen && lt == 0.f) ref = MINUS_INF, lt = direct ? __int_as_float(0x7fc00000) : 0.f;  // all keys minus infinity
          const long prow = ((long)r.kvh * a.T + r.tok0) * a.r + 128L * blockIdx.x + row;
          if (a.by_row && valid && jrow == 0 && hf == 0) {
            if (tfirst) a.first[(long)r.kvh * a.T + t] = direct ? -1 : (int)blockIdx.x;
            if (tlast) a.last[(long)r.kvh * a.T + t] = (int)blockIdx.x;
          }
          if (!direct && valid && hf == 0) a.ml[prow] = make_float2(ref, lt);
          const float inv = lt == 0.f ? 0.f : 1.0f / lt;
          __half *y = a.Y + (long)t * a.ystride + (long)(r.kvh * a.r + jrow) * D + hf * (D / 2);
          float *po = a.O + prow * D + hf * (D / 2);
#pragma unroll 1
          for (int c = 0; c < D / 2; c += 16) {
            uint32_t o[16];
            __syncwarp();
            tmem_ld16(ocol + c, o);
            tmem_ld_wait(o);
            if (!valid) continue;
            if (direct) {
#pragma unroll
              for (int e = 0; e < 8; e++) {
                const __half2 hv = __floats2half2_rn(__uint_as_float(o[2 * e]) * inv, __uint_as_float(o[2 * e + 1]) * inv);
                o[e] = *reinterpret_cast<const uint32_t *>(&hv);
              }
              store_row16(y + c, o, a.y32);
            } else if (lt != 0.f) {
              st_global_v8(po + c, o), st_global_v8(po + c + 8, o + 8);
            }
          }
          __syncwarp();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(k.bar(C::B_OE));
      }
      k.done_run(n);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (*k.abort()) {  // a wait ran out
    if (tid == 0) a.hdr[0] = 1;  // the records may be missing
    settle<C>(k.smem, FW_M, FW_M);
  }
  if (warp == FW_M) {
    tc_fence_after();
    tmem_dealloc(tmem, C::TCOLS);
  }
}

template <int D>
int launch(dc_ctx *ctx, const CUtensorMap &tq, const CUtensorMap &tk, const CUtensorMap &tv, const PArgs &a) {
  using C = FewCfg<D>;
  static uint64_t attr_done = 0;
  if (!(attr_done & (1ull << ctx->device))) {
    DC_CUDA(cudaFuncSetAttribute(attention_paged_few_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    attr_done |= 1ull << ctx->device;
  }
  DC_CUDA(dc_launch_pdl(ctx->stream, attention_paged_few_kernel<D>, dim3(2 * ctx->sms), dim3(F_THREADS), C::SMEM, tq, tk, tv,
                        a));
  return dc_launch_check("attention_paged (few rows)");
}

}  // namespace

// D = 64 or 128; two CTAs an SM. The caller launches the join.
int attn_few_launch(dc_ctx *ctx, int D, const CUtensorMap &tq, const CUtensorMap &tk, const CUtensorMap &tv, const PArgs &a) {
  return D == 64 ? launch<64>(ctx, tq, tk, tv, a) : launch<128>(ctx, tq, tk, tv, a);
}
