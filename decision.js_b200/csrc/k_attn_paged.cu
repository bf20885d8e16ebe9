// Attention of a batch of sequences over a paged cache, with a prefix that a group of sequences shares.
//
// For a query row, o = sum_j p_j v_j / sum_j p_j with p_j = exp(scale q . k_j), j over its group's prefix and its own
// keys up to its own. A tile is 128 rows of one kv head: TPT = 128 / r consecutive tokens of a group (r query heads to
// a kv head), so tokens of several sequences share the tile and the prefix passes through the tensor cores once for
// all of them. The keys of a tile are a list of blocks: the prefix's, then, sequence by sequence, the own blocks of the
// sequences that the tile's tokens belong to, seen by that sequence's rows alone (the product leaves the other rows'
// accumulators as they are).
//
// The blocks of all tiles of all kv heads in a row make one line of units (a sequence piece without keys counts as
// one unit, so that every tile is visited). Each CTA of a resident grid takes an equal stretch of it, whatever the
// lengths: a long prefix is cut over many CTAs, short tiles are walked one after the other. Every CTA works the line
// out for itself from the offsets and lengths (one scan over the sequences), so nothing is planned on the host and a
// captured call follows new contents. A tile inside one stretch is written straight to Y; a tile that was cut leaves
// f32 parts (value sums, row maximum and weight sum) that a second kernel joins in order of the stretches, so results
// do not depend on timing.
//
// This file holds the kernel for many rows, the join and the host side; k_attn_few.cu the kernel for few rows; the line
// and what both kernels' producers do with it are in dc_paged.cuh. Within a CTA here, one to an SM:
//   warps 0-11 softmax, three warpgroups that take the blocks (128 keys; 64 at D = 256) in turn, thread = row. A row's
//              reference (what its weights are relative to) goes from block to block through shared memory: a warp waits
//              for its turn only between its own maximum and its weights. The reference moves when a maximum is more than
//              2^8 above it, and weights are scaled by 2^7: they stay under 2^15, and small ones out of f16's subnormals.
//              The rounding of a weight to f16, half a step of itself, is the matrix unit's operand type; sums are f32.
//   warp 12    looks over V blocks that some row of the tile does not see: rows past the last key are zeroed, and
//              values that are not finite too (a weight of 0 times them would be NaN in every row), with a mark on
//              the rows that see them
//   warp 13    walks the line and loads V
//   warp 14    Q K^T (and TMEM), warp 15 P V: two threads, as one would be busy issuing for longer than the products take
//   warp 16    walks the line, hands runs of blocks to the others through a ring of descriptors, loads K and Q
// All roles run ahead across tiles; Q (single buffer) and the accumulator wait for a tile's end, which the warpgroup of the
// tile's last block sees to while the other two go on.
//
// What bounds it. Many rows over a long prefix (49 sequences of up to 50 tokens, 12,800 keys, 24 heads over 8, D = 128):
// 208 to 224 us with the power clock, 810 to 870 TFLOP/s, half the measured matrix rate; without the softmax it still takes
// 167, as every tile of 128 rows brings all its keys from L2 (about 39 bytes a clock and SM): only tiles of 256 rows would
// change that, for which the tensor memory of one SM has no room (scores next to two accumulators), that of two would. Short tiles (a few blocks each):
// the chain from a tile's last product over its stores to the next tile's first product, and the instruction caches, which
// the roles' code (70 KB) does not fit: a look-up in four missed, and every loop that was rolled and every path that two
// roles share has shortened such calls. Steps measured: two softmax warpgroups in turn 264 -> 245 us, three with 128-key
// blocks 232, the tile's end by one warpgroup instead of all three 2% (8% at D = 64).
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <float.h>

#include <algorithm>

#include "dc_internal.h"
#include "dc_paged.cuh"
#include "dc_ptx.cuh"

using namespace dcx;

int attn_few_launch(dc_ctx *, int, const CUtensorMap &, const CUtensorMap &, const CUtensorMap &, const PArgs &);

namespace {

constexpr int PA_WG = 3, PA_SOFT = 4 * PA_WG;  // softmax warpgroups, warps
constexpr int PA_WC = PA_SOFT, PA_WV = PA_SOFT + 1, PA_WM = PA_SOFT + 2, PA_WP = PA_SOFT + 3, PA_WK = PA_SOFT + 4;
constexpr int PA_THREADS = (PA_SOFT + 5) * 32;

template <int D>
struct WideCfg {
  // keys per block; 64 at D = 256, whose tiles and accumulator leave room for no more
  static constexpr int KB = D == 256 ? 64 : 128, NA = D / 64, Q_ROWS = 128, THREADS = PA_THREADS;
  static constexpr int KST = D == 64 ? 4 : 2, VST = D == 64 ? 4 : D == 128 ? 3 : 2;  // stages of the K and of the V ring
  static constexpr int Q_BYTES = 128 * D * 2, KV_BYTES = KB * D * 2;
  static constexpr int K_OFF = Q_BYTES, V_OFF = K_OFF + KST * KV_BYTES;
  static constexpr int BAR_OFF = V_OFF + VST * KV_BYTES;
  static constexpr int B_QF = 0, B_QE = 1, B_OE = 2, B_OD = 3, B_XB = 7, B_SF = 23, B_PF = B_SF + PA_WG,
                       B_SE = B_PF + PA_WG, B_CH = B_SE + PA_WG, B_KF = B_CH + 4 * PA_WG, B_KE = B_KF + KST, B_VF = B_KE + KST,
                       B_VE = B_VF + VST, B_VS = B_VE + VST, B_IF = B_VS + VST, B_IE = B_IF + PA_RING,
                       B_END = B_IE + PA_RING, NBARS = B_END + 2;
  static constexpr int MISC_OFF = BAR_OFF + ((NBARS * 8 + 15) & ~15), LOADED_OFF = MISC_OFF + 20;
  // misc: tmem slot, abort, start (s, offset), loaded; poison; scan; runs; groups; references and sums
  static constexpr int POISON_OFF = MISC_OFF + 32, SCAN_OFF = POISON_OFF + PA_MARK_BYTES,
                       RUN_OFF = SCAN_OFF + ((PA_THREADS / 32 * 8 + 15) & ~15), GOFF_OFF = RUN_OFF + PA_RING * (int)sizeof(Run),
                       XCH_OFF = GOFF_OFF + PA_META;
  static constexpr int SMEM = XCH_OFF + 128 * 4 + 4 * PA_WG * 128 * 8 + 1024;
  static constexpr int S_COL = 0, O_COL = PA_WG * KB;  // tensor memory: a scores' buffer per warpgroup, the accumulator
  static constexpr int TCOLS = 512;
  static_assert(O_COL + D <= TCOLS, "tensor memory");
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

template <int D>
__global__ void __launch_bounds__(PA_THREADS, 1)
    attention_paged_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                           const __grid_constant__ CUtensorMap tmV, const PArgs a) {
  using C = WideCfg<D>;
  constexpr int KB = C::KB, KST = C::KST, VST = C::VST;
  extern __shared__ uint8_t smem_raw[];
  const Cta<C> k(a, smem_raw);
  uint8_t *smem = k.smem;
  const uint32_t sbase = k.base;
  auto bar = [&](int i) { return k.bar(i); };
  const int tid = k.tid, warp = k.warp, lane = k.lane;
  const Run *runs = k.runs();

  if (tid == 0) {
    for (int i = 0; i < C::NBARS; i++) {
      const int n = i == C::B_OE || (i >= C::B_PF && i < C::B_PF + PA_WG) ? 4
                    : i >= C::B_XB && i < C::B_XB + 16                     ? PA_WG - 1
                    : i >= C::B_VE && i < C::B_VE + VST                    ? 2
                    : i >= C::B_IE && i < C::B_END                         ? PA_SOFT + 3
                                                                           : 1;
      mbar_init(bar(i), n);
    }
    *k.abort() = 0;
    mbar_init_fence();
  }
  k.clear_marks();
  if (warp == PA_WK && lane == 0) tma_prefetch_desc(&tmQ), tma_prefetch_desc(&tmK);
  if (warp == PA_WV && lane == 0) tma_prefetch_desc(&tmV);
  // Tensor memory is taken only when the kernels before are done, and the next kernel is let in only when every CTA
  // here has its own: of two kernels on an SM, neither can hold columns while it waits for the other.
  dc_pdl_wait();
  if (warp == PA_WM) tmem_alloc(smem_u32(k.tmem_slot()), C::TCOLS);

  Groups gs;
  Stretch st;
  const bool fine = line_start(k, gs, st);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *k.tmem_slot();

  auto wait_warp = [&](int i, int parity) { return k.wait_warp(i, parity); };
  auto wait1 = [&](int i, int parity) { return k.wait1(i, parity); };
  if (!fine || st.p0 >= st.p1) {
  } else if (warp == PA_WK || warp == PA_WV) {
    walk_line(k, gs, st, warp == PA_WV, &tmQ, warp == PA_WV ? &tmV : &tmK);
  } else if (warp == PA_WC) {
    look_over(k);
  } else if (warp == PA_WM) {
    // Q K^T, one thread: a block's scores go to the buffer of the warpgroup that takes it, free since the P V of the
    // block PA_WG before
    constexpr uint32_t idesc_qk = idesc_f16_f32(128, KB);
    if (elect_one()) {
      const uint64_t q0 = desc_sw128(sbase), k0 = desc_sw128(sbase + C::K_OFF);
      int g = 0;
      bool ok = true;
      for (int n = 0; ok && wait1(C::B_IF + n % PA_RING, n / PA_RING); n++) {
        const int flags = runs[n % PA_RING].flags, nb = runs[n % PA_RING].nb, item = runs[n % PA_RING].item;
        if (flags & RUN_END) break;
        if (flags & RUN_FIRST) ok = wait1(C::B_QF, item);
#pragma unroll 1
        for (int b = 0; ok && b < nb; b++, g++) {
          const int st = g % KST, sb = g % PA_WG;
          if (!(ok = wait1(C::B_KF + st, g / KST) && wait1(C::B_SE + sb, g / PA_WG + 1))) break;
          tc_fence_after();
          const uint32_t sc = tmem + (uint32_t)(C::S_COL + sb * KB);
          const uint64_t k = k0 + (uint32_t)(st * C::KV_BYTES >> 4);
#pragma unroll
          for (int kd = 0; kd < D / 16; kd++)
            mma_f16(sc, q0 + (((kd >> 2) * 128 * 128 + (kd & 3) * 32) >> 4),
                    k + (((kd >> 2) * KB * 128 + (kd & 3) * 32) >> 4), idesc_qk, kd > 0);
          mma_commit(bar(C::B_SF + sb));
          mma_commit(bar(C::B_KE + st));
        }
        if (ok && (flags & RUN_LAST)) mma_commit(bar(C::B_QE));
        if (ok) mbar_arrive(bar(C::B_IE + n % PA_RING));
      }
    }
    __syncwarp();
  } else if (warp == PA_WP) {
    // P V, one thread
    constexpr uint32_t idesc_pv = idesc_f16_f32(128, D) | (1u << 16);  // V MN-major
    if (elect_one()) {
      const uint64_t v0 = desc_mn(sbase + C::V_OFF, KB * 128);
      int g = 0, looked = 0;
      bool ok = true;
      for (int n = 0; ok && wait1(C::B_IF + n % PA_RING, n / PA_RING); n++) {
        const Run r = runs[n % PA_RING];
        if (r.flags & RUN_END) break;
        if (r.flags & RUN_FIRST) ok = wait1(C::B_OE, r.item);  // the accumulator is zero
#pragma unroll 1
        for (int b = 0; ok && b < r.nb; b++, g++) {
          const int st = g % VST, sb = g % PA_WG, key0 = (r.kb + b) * KB;
          const int steps = (min(KB, r.kend - key0) + 15) >> 4;  // of 16 keys
          uint32_t off[4] = {0, 0, 0, 0};                        // rows that it leaves alone
          if (r.seg >= 0) {                                      // own blocks: but the sequence's that see a key of it
            const int lo = (max(max(r.tok0, r.qb), key0 - r.len + r.qe) - r.tok0) * a.r;
            const int hi = (min(r.qe, r.tok0 + r.ntok) - r.tok0) * a.r;
#pragma unroll
            for (int w = 0; w < 4; w++) off[w] = ~mask_word(lo, hi, w);
          }
          if (!(ok = wait1(C::B_VF + st, g / VST))) break;
          if (to_look_over<KB>(r, key0)) {
            if (!(ok = wait1(C::B_VS + looked % VST, looked / VST))) break;
            looked++;
          }
          if (!(ok = wait1(C::B_PF + sb, g / PA_WG))) break;
          tc_fence_after();
          const uint32_t p = tmem + (uint32_t)(C::S_COL + sb * KB);
          const uint64_t v = v0 + (uint32_t)(st * C::KV_BYTES >> 4);
#pragma unroll
          for (int kk = 0; kk < KB / 16; kk++)
            if (kk < steps) mma_f16_ts_rows(tmem + C::O_COL, p + 8 * kk, v + kk * (2048 >> 4), idesc_pv, off);
          mma_commit(bar(C::B_SE + sb));
          mma_commit(bar(C::B_VE + st));
        }
        if (ok && (r.flags & RUN_LAST)) mma_commit(bar(C::B_OD + (r.item & 3)));
        if (ok) mbar_arrive(bar(C::B_IE + n % PA_RING));
      }
    }
    __syncwarp();
  } else {
    const int q = warp & 3, wg = warp >> 2;
    const int row = 32 * q + lane, irow = row / a.r, jrow = row - irow * a.r;
    const uint32_t lrow = tmem + ((uint32_t)(32 * q) << 16), ocol = lrow + (uint32_t)C::O_COL;
    const uint32_t scol = lrow + (uint32_t)(C::S_COL + wg * KB);
    float *s_ref = reinterpret_cast<float *>(smem + C::XCH_OFF);
    float2 *s_sum = reinterpret_cast<float2 *>(s_ref + 128);  // [tile % 4][PA_WG][128]
    int g = 0, turn = 0;  // blocks before the run, this warpgroup's blocks before this one
    const int prev = wg == 0 ? PA_WG - 1 : wg - 1;
    bool ok = true;
    // the tile's state
    bool valid = false, anyv = false, had = false, seen = false, tfirst = false;  // seen: the row has seen a key
    int t = 0;
    float ref = -FLT_MAX, l = 0.f;  // l: the sum of this thread's weights, in units of 2^(ref - 7)
    auto zero = [&]() {             // its rows' accumulators, for the next tile
      const uint32_t z[16] = {};
      __syncwarp();
#pragma unroll 1
      for (int c = 0; c < D; c += 16) tmem_st16(ocol + c, z);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(C::B_OE));
    };
    if (wg == 0) zero();
    for (int n = 0; ok && wait_warp(C::B_IF + n % PA_RING, n / PA_RING); n++) {
      const Run &r = runs[n % PA_RING];  // (stays as it is until done_run)
      if (r.flags & RUN_END) break;
      if (r.flags & RUN_FIRST) {
        t = r.tok0 + irow;
        valid = irow < r.ntok && irow < a.tpt;
        anyv = __any_sync(0xffffffffu, valid);
        had = seen = false, tfirst = (r.flags & RUN_TFIRST) != 0;
        ref = -FLT_MAX, l = 0.f;
      }
      // the run's keys that the row sees
      const int rlim = !valid ? 0 : r.seg < 0 ? r.kend : t >= r.qb && t < r.qe ? own_limit(t, r.qe, r.len) : 0;
      const int nb = r.nb, kb = r.kb, kend = r.kend;
      seen = seen || (nb > 0 && rlim > kb * KB);
      // the run's first blocks that every row here sees whole (lanes without a row have no say)
      const int full = __reduce_min_sync(0xffffffffu, valid ? rlim : 0x7fffffff) / KB - kb;
      for (int b = (wg + PA_WG - g % PA_WG) % PA_WG; b < nb; b += PA_WG, turn++) {
        const bool opens = b == 0 && !had;  // the tile's first block
        if (!(ok = wait_warp(C::B_SF + wg, turn))) break;
        const int nv = rlim - (kb + b) * KB;  // its keys that the row sees (or fewer than none, or more than there are)
        const bool part = b >= full;
        const bool sees = part ? __any_sync(0xffffffffu, nv > 0) : anyv;
        const int cols = part ? min(KB, (kend - (kb + b) * KB + 31) & ~31) : KB;  // the others' weights are not read
        float sc = a.scale_log2, pmx = -FLT_MAX;
        if (sees) {
          tc_fence_after();
          if (sc <= 0.f) {  // the largest score is not the largest product: scale first
#pragma unroll 1
            for (int c = 0; c < cols; c += 16) {
              uint32_t x[16];
              __syncwarp();
              tmem_ld16(scol + c, x);
              tmem_ld_wait(x);
#pragma unroll
              for (int e = 0; e < 16; e++) x[e] = __float_as_uint(__uint_as_float(x[e]) * sc);
              __syncwarp();
              tmem_st16(scol + c, x);
            }
            tmem_st_wait();
            sc = 1.f;
          }
          float m2[2] = {MINUS_INF, MINUS_INF};
#pragma unroll 1
          for (int c = 0; c < cols; c += 32) {
            uint32_t x[32];
            __syncwarp();
            tmem_ld32(scol + c, x);
            tmem_ld_wait(x);
            if (part)
#pragma unroll
              for (int e = 0; e < 32; e++) x[e] = c + e < nv ? x[e] : 0xff800000u;
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              m2[0] = max3(m2[0], __uint_as_float(x[e]), __uint_as_float(x[e + 1]));
              m2[1] = max3(m2[1], __uint_as_float(x[e + 2]), __uint_as_float(x[e + 3]));
            }
          }
          pmx = fmaxf(m2[0], m2[1]) * sc;
        }
        // the row's reference goes from block to block through shared memory, with the turn to move it
        if (g + b > 0 && !(ok = wait_warp(C::B_CH + PA_WG * q + prev, wg == 0 ? turn - 1 : turn))) break;
        if (anyv) {
          const float cur = opens ? -FLT_MAX : s_ref[row];
          const bool grow = pmx > cur + 8.0f;
          const float now = grow ? pmx : cur;
          const bool resc = grow && cur > -FLT_MAX;
          if (__any_sync(0xffffffffu, resc)) {
            if (!(ok = wait_warp(C::B_SE + prev, wg == 0 ? turn - 1 : turn))) break;  // the products so far
            tc_fence_after();
            const float f = resc ? ex2_approx(cur - now) : 1.0f;
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
              uint32_t o[16];
              __syncwarp();
              tmem_ld16(lrow + (uint32_t)(C::O_COL + c), o);
              tmem_ld_wait(o);
#pragma unroll
              for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              __syncwarp();
              tmem_st16(lrow + (uint32_t)(C::O_COL + c), o);
            }
            tmem_st_wait();
          }
          if (grow || opens) s_ref[row] = now;
          if (__any_sync(0xffffffffu, now != ref)) {
            l *= ex2_approx(ref - now);  // 0 * 0 where there was none
            ref = now;
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(C::B_CH + PA_WG * q + wg));
        if (sees) {
          const uint64_t ref2 = f32x2(7.0f - ref, 7.0f - ref), sc2 = f32x2(sc, sc);
          uint64_t sum[2] = {0, 0};
#pragma unroll 1
          for (int c = 0; c < cols; c += 32) {  // 32 weights go where 16 of the scores were that are done with
            uint32_t x[32];
            __syncwarp();
            tmem_ld32(scol + c, x);
            tmem_ld_wait(x);
            if (part)
#pragma unroll
              for (int e = 0; e < 32; e++) x[e] = c + e < nv ? x[e] : 0xff800000u;
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              const float2 v = f32x2_split(fma_f32x2(f32x2(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), sc2, ref2));
              const float p0 = ex2_approx(v.x), p1 = ex2_approx(v.y);
              sum[(e >> 1) & 1] = add_f32x2(sum[(e >> 1) & 1], f32x2(p0, p1));
              const __half2 hp = __floats2half2_rn(p0, p1);
              x[e / 2] = *reinterpret_cast<const uint32_t *>(&hp);
            }
            __syncwarp();
            tmem_st16(scol + c / 2, *reinterpret_cast<const uint32_t (*)[16]>(&x[0]));
          }
          const float2 add = f32x2_split(add_f32x2(sum[0], sum[1]));
          l += add.x + add.y;
          tmem_st_wait();
        }  // none of these rows sees the block: the product leaves them alone
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(C::B_PF + wg));
      }
      if (!ok) break;
      g += nb, had = had || nb > 0;
      // The tile's end is the work of the warpgroup that took its last block: the others leave their sums and go on to the
      // next tile, whose first product waits for the accumulator.
      if (r.flags & RUN_LAST) {
        const int four = r.item & 3, turn4 = r.item >> 2;
        float2 *sums = s_sum + four * PA_WG * 128 + row;
        if (wg != (g + PA_WG - 1) % PA_WG) {
          sums[wg * 128] = make_float2(l, ref);
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(C::B_XB + 4 * q + four));
        } else {
          if (!(ok = wait_warp(C::B_XB + 4 * q + four, turn4) && wait_warp(C::B_OD + four, turn4))) break;
          tc_fence_after();
          const bool tlast = (r.flags & RUN_TLAST) != 0, direct = tfirst && tlast;
          if (!direct && !a.by_row && q == 0 && lane == 0) {
            if (tlast) a.head[blockIdx.x] = make_int4(r.tok0, r.ntok, r.kvh, 0);
            if (tfirst) a.tail[blockIdx.x] = 1;
          }
          if (anyv) {
            float lt = l;  // at the row's last reference, which the last block's warpgroup has
#pragma unroll
            for (int w = 1; w < PA_WG; w++) {
              const float2 x = sums[(wg + w) % PA_WG * 128];
              lt += x.x * ex2_approx(x.y - ref);
            }
            if (seen && ((k.poison(r.item)[irow >> 5] >> (irow & 31)) & 1u)) lt = __int_as_float(0x7fc00000);
            if (seen && lt == 0.f) ref = MINUS_INF, lt = direct ? __int_as_float(0x7fc00000) : 0.f;  // all keys minus infinity
            const long prow = ((long)r.kvh * a.T + r.tok0) * a.r + 128L * blockIdx.x + row;
            if (!direct && valid) a.ml[prow] = make_float2(ref, lt);
            if (a.by_row && valid && jrow == 0) {
              if (tfirst) a.first[(long)r.kvh * a.T + t] = direct ? -1 : (int)blockIdx.x;
              if (tlast) a.last[(long)r.kvh * a.T + t] = (int)blockIdx.x;
            }
            const float inv = lt == 0.f ? 0.f : 1.0f / lt;
            __half *y = a.Y + (long)t * a.ystride + (long)(r.kvh * a.r + jrow) * D;
            float *po = a.O + prow * D;
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              uint32_t o[32];
              __syncwarp();
              tmem_ld32(ocol + c, o);
              tmem_ld_wait(o);
              if (!valid) continue;
              if (direct) {
#pragma unroll
                for (int e = 0; e < 16; e++) {
                  const __half2 hv =
                      __floats2half2_rn(__uint_as_float(o[2 * e]) * inv, __uint_as_float(o[2 * e + 1]) * inv);
                  o[e] = *reinterpret_cast<const uint32_t *>(&hv);
                }
                store_row16(y + c, o, a.y32), store_row16(y + c + 16, o + 8, a.y32);
              } else if (lt != 0.f) {
#pragma unroll
                for (int e = 0; e < 32; e += 8) st_global_v8(po + c + e, o + e);
              }
            }
          }
          zero();
        }
      }
      k.done_run(n);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (*k.abort()) {  // a wait ran out
    if (tid == 0) a.hdr[0] = 1;  // the records may be missing
    settle<C>(k.smem, PA_WM, PA_WP);
  }
  if (warp == PA_WM) {
    tc_fence_after();
    tmem_dealloc(tmem, C::TCOLS);
  }
}

template <int D>
struct JoinRows {  // rows of a warp in the join by tile
  static constexpr int R = D == 256 ? 2 : 4;
};

// Joins the parts of the tiles that were cut: y = sum_c 2^(m_c - M) O_c / sum_c 2^(m_c - M) l_c over the CTAs c from the
// tile's first to its last; NaN, as the formula has it, where all keys that the row sees score minus infinity (parts of
// weight 0 with that maximum). For few rows in many parts: a block to a (row, head), each of its W warps every W-th part,
// joined in order of the warps.
template <int D>
__global__ void __launch_bounds__(128) attention_join_kernel(const PArgs a) {
  dc_pdl_begin();
  constexpr int N = D / 32, W = 4;  // a lane's values; warps
  __shared__ float s_o[W][D], s_m[W], s_l[W];
  const int part = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long t = blockIdx.x / a.heads;
  const int h = blockIdx.x - (int)t * a.heads, kvh = h / a.r;
  const int t0 = a.qoff[0], t1 = a.qoff[a.S];
  const int c0 = a.first[(long)kvh * a.T + t], c1 = a.last[(long)kvh * a.T + t];
  // (a refused call, or one whose waits ran out, has no records)
  if (a.hdr[0] || t < t0 || t >= t1 || c0 < 0 || c1 < c0 || c1 >= a.ctas) return;
  const long base = ((long)kvh * a.T + t) * a.r + h - kvh * a.r;  // part c of the row: row base + 128 c
  auto fetch = [&](float (&v)[N], int c) {
    const float *p = a.O + (base + 128L * c) * D + N * lane;
    if (N == 2) {
      *reinterpret_cast<float2 *>(v) = *reinterpret_cast<const float2 *>(p);
    } else {
#pragma unroll
      for (int e = 0; e < N; e += 4) *reinterpret_cast<float4 *>(v + e) = *reinterpret_cast<const float4 *>(p + e);
    }
  };
  // the first parts' values are on their way with their weights, whether those turn out 0 (and nothing was stored) or not
  float v[4][N];
#pragma unroll
  for (int k = 0; k < 4; k++)
    if (c0 + part + W * k <= c1) fetch(v[k], c0 + part + W * k);
  float M = -FLT_MAX, L = 0.f, o[N] = {};
  bool low = false;  // a part that saw nothing but minus infinity
  for (int cb = c0 + part; cb <= c1; cb += 32 * W) {  // 32 parts at a time, usually all
    const int c = cb + W * lane;
    const float2 x = c <= c1 ? a.ml[base + 128L * c] : make_float2(-FLT_MAX, 0.f);
    low = low || (x.y == 0.f && x.x == MINUS_INF);
    float m = x.y == 0.f ? -FLT_MAX : x.x;  // a part of weight 0 stored no values
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, s));
    m = fmaxf(m, M);
    const float f = ex2_approx(M - m);  // what is there goes to the new maximum
    M = m;
    const float w = x.y == 0.f ? 0.f : ex2_approx(x.x - M);
    L = L * f + (x.y == 0.f ? 0.f : w * x.y);
#pragma unroll
    for (int e = 0; e < N; e++) o[e] *= f;
    uint32_t have = __ballot_sync(0xffffffffu, x.y != 0.f);
    if (cb == c0 + part) {
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const float wk = __shfl_sync(0xffffffffu, w, k);
        if ((have >> k) & 1u)
#pragma unroll
          for (int e = 0; e < N; e++) o[e] = fmaf(wk, v[k][e], o[e]);
      }
      have &= ~15u;
    }
    while (have) {  // four parts' values on their way
      float wk[4];
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const int at = have ? __ffs(have) - 1 : 0;
        wk[k] = __shfl_sync(0xffffffffu, w, at);
#pragma unroll
        for (int e = 0; e < N; e++) v[k][e] = 0.f;
        if (have)
          fetch(v[k], cb + W * at);
        else
          wk[k] = 0.f;
        have &= have - 1;
      }
#pragma unroll
      for (int k = 0; k < 4; k++)
#pragma unroll
        for (int e = 0; e < N; e++) o[e] = fmaf(wk[k], v[k][e], o[e]);
    }
  }
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) L += __shfl_xor_sync(0xffffffffu, L, s);
  low = __any_sync(0xffffffffu, low);
  if (lane == 0) s_m[part] = low && L == 0.f ? MINUS_INF : M, s_l[part] = L;
  __syncthreads();
  float all = -FLT_MAX;
#pragma unroll
  for (int w = 0; w < W; w++) all = s_l[w] != 0.f ? fmaxf(all, s_m[w]) : all;
  const float f = s_l[part] != 0.f ? ex2_approx(M - all) : 0.f;
#pragma unroll
  for (int e = 0; e < N; e++) s_o[part][N * lane + e] = s_l[part] != 0.f ? o[e] * f : 0.f;
  L = 0.f;
#pragma unroll
  for (int w = 0; w < W; w++)
    if (s_l[w] != 0.f) L += s_l[w] * ex2_approx(s_m[w] - all);
  __syncthreads();
  if (part) return;
#pragma unroll
  for (int e = 0; e < N; e++) {
    o[e] = 0.f;
#pragma unroll
    for (int w = 0; w < W; w++) o[e] += s_o[w][N * lane + e];
  }
  if (L == 0.f)
#pragma unroll
    for (int w = 0; w < W; w++) L = s_m[w] == MINUS_INF ? __int_as_float(0x7fc00000) : L;
  const float inv = L == 0.f ? 0.f : 1.0f / L;
  __half *y = a.Y + t * a.ystride + (long)h * D + N * lane;
#pragma unroll
  for (int e = 0; e < N; e += 2)
    *reinterpret_cast<__half2 *>(y + e) = __floats2half2_rn(o[e] * inv, o[e + 1] * inv);
}

// The same for many rows, most of them whole or cut once: blockIdx.y is the CTA that ends a cut tile. A warp takes R rows
// of it, two parts of each at a time, all on their way together, as what a row costs is the way to memory and back. 64
// groups of 2 x 20 tokens over 500, D = 64: 40.2 us with a row to a warp, 35.2 with four rows and four parts at a time,
// 34.0 with two parts (fewer registers, more warps), 35.4 with two rows.
template <int D>
__global__ void __launch_bounds__(128) attention_join_tiles_kernel(const PArgs a) {
  dc_pdl_begin();
  constexpr int N = D / 32, R = JoinRows<D>::R, P = 2;  // a lane's values; rows; parts
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c1 = blockIdx.y, row0 = (blockIdx.x * 4 + warp) * R;
  const int refused = a.hdr[0];
  const int4 tile = a.head[c1];
  bool begins = c1 > lane && a.tail[c1 - 1 - lane] != 0;
  const int rows = min(R, tile.y * a.r - row0);
  if (refused || rows <= 0) return;
  int c0 = c1;  // the last CTA before that begins a tile and does not end it
  for (uint32_t at; (at = __ballot_sync(0xffffffffu, begins)) == 0;) {
    c0 -= 32;
    if (c0 <= 0) return;
    begins = c0 > lane && a.tail[c0 - 1 - lane] != 0;
  }
  c0 -= __ffs(__ballot_sync(0xffffffffu, begins));
  const long base = ((long)tile.z * a.T + tile.x) * a.r + row0;  // part c of a row: 128 c rows on
  float M[R], L[R], o[R][N];
  uint32_t low = 0;  // rows with a part that saw nothing but minus infinity
#pragma unroll
  for (int i = 0; i < R; i++) {
    M[i] = -FLT_MAX, L[i] = 0.f;
#pragma unroll
    for (int e = 0; e < N; e++) o[i][e] = 0.f;
  }
#pragma unroll 1
  for (int cb = c0; cb <= c1; cb += P) {
    float2 x[R][P];
    float v[R][P][N];  // (where a part's weight is 0, nothing was stored and nothing is used)
#pragma unroll
    for (int i = 0; i < R; i++)
#pragma unroll
      for (int k = 0; k < P; k++) {
        x[i][k] = make_float2(-FLT_MAX, 0.f);
#pragma unroll
        for (int e = 0; e < N; e++) v[i][k][e] = 0.f;
        if (i >= rows || cb + k > c1) continue;
        const long at = base + i + 128L * (cb + k);
        x[i][k] = a.ml[at];
        const float *p = a.O + at * D + N * lane;
        if (N == 2) {
          *reinterpret_cast<float2 *>(v[i][k]) = *reinterpret_cast<const float2 *>(p);
        } else {
#pragma unroll
          for (int e = 0; e < N; e += 4)
            *reinterpret_cast<float4 *>(v[i][k] + e) = *reinterpret_cast<const float4 *>(p + e);
        }
      }
#pragma unroll
    for (int i = 0; i < R; i++) {
      float m = M[i];
#pragma unroll
      for (int k = 0; k < P; k++) m = x[i][k].y != 0.f ? fmaxf(m, x[i][k].x) : m;
      const float f = ex2_approx(M[i] - m);  // what is there goes to the new maximum
      M[i] = m, L[i] *= f;
#pragma unroll
      for (int e = 0; e < N; e++) o[i][e] *= f;
#pragma unroll
      for (int k = 0; k < P; k++)
        if (x[i][k].y != 0.f) {
          const float w = ex2_approx(x[i][k].x - m);
          L[i] = fmaf(w, x[i][k].y, L[i]);
#pragma unroll
          for (int e = 0; e < N; e++) o[i][e] = fmaf(w, v[i][k][e], o[i][e]);
        } else {
          low |= (x[i][k].x == MINUS_INF ? 1u : 0u) << i;
        }
    }
  }
#pragma unroll
  for (int i = 0; i < R; i++) {
    if (i >= rows) break;
    const int tok = (row0 + i) / a.r, h = tile.z * a.r + row0 + i - tok * a.r;
    const float inv = L[i] != 0.f ? 1.0f / L[i] : (low >> i) & 1u ? __int_as_float(0x7fc00000) : 0.f;
    __half *y = a.Y + (long)(tile.x + tok) * a.ystride + (long)h * D + N * lane;
#pragma unroll
    for (int e = 0; e < N; e += 2)
      *reinterpret_cast<__half2 *>(y + e) = __floats2half2_rn(o[i][e] * inv, o[i][e + 1] * inv);
  }
}

typedef CUresult (*EncodeTiledP)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                 const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

int encode(CUtensorMap *m, const void *p, int rank, const cuuint64_t *dims, const cuuint64_t *strides,
           const cuuint32_t *box) {
  static EncodeTiledP enc = nullptr;
  if (!enc) {
    void *f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      enc = reinterpret_cast<EncodeTiledP>(f);
  }
  DC_CHECK(enc, DC_ECUDA, "decision.js: cuTensorMapEncodeTiled is unavailable");
  const cuuint32_t es[3] = {1, 1, 1};
  const CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank, const_cast<void *>(p), dims, strides, box, es,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  DC_CHECK(r == CUDA_SUCCESS, DC_ECUDA, "decision.js: attention_paged: tensor map encode failed (%d)", (int)r);
  return DC_OK;
}

size_t up(size_t x) { return (x + 255) & ~(size_t)255; }  // (WS_ALIGN)

// The workspace: a status word, the join's records, parts' maxima and sums, parts' sums of values. Part c of a tile
// starts at row (kvh T + first row) r + 128 c: along the line either the tile moves on, by at least its rows, or c does,
// so no two parts meet. The caller's address is a multiple of 16; the layout starts at the next multiple of WS_ALIGN (parts
// are stored in 32-byte pieces, records of 16 and 8 bytes).
constexpr size_t WS_ALIGN = 256;
struct Ws {
  size_t first, last, head, tail, ml, O, bytes;
};
Ws ws_layout(int T, int heads, int kv, int D, int ctas) {
  Ws w;
  const size_t rows = (size_t)T * heads + 128 * (size_t)(ctas + 1);
  w.first = 256;
  w.last = w.first + up((size_t)T * kv * 4);
  w.head = w.last + up((size_t)T * kv * 4);
  w.tail = w.head + up((size_t)ctas * 16);
  w.ml = w.tail + up((size_t)ctas * 4);
  w.O = w.ml + up(rows * 8);
  w.bytes = w.O + up(rows * (size_t)D * 4) + WS_ALIGN - 16;
  return w;
}

// The kernel for few rows where a group has four tiles or less. Measured, few against many rows' kernel, us: decode of 218
// sequences over 24 prefixes, D = 64, 90 against 94; about 300 rows over 16,000 keys 35 against 40, D = 128 39 against 42; 32
// groups of 3 questions of 40 tokens over 512 tokens 58 against 60; 64 of 2 x 20 tokens over 500 tokens 34 against 44, D = 128
// 43 against 53. 1,100 rows over 16,000 keys 62 against 56, D = 128 74 against 61; 4,500 rows 176 against 159, D = 128 260
// against 206. (Over 4,000 tokens 64 groups of 2 x 20 would gain by the other, 171 against 157; how long a prefix is the host
// does not know.) At D = 256 the accumulators of two CTAs do not fit.
bool paged_few(int D, int T, int r, int G) { return D <= 128 && (long)T * r <= 512L * std::max(G, 1); }

template <int D>
int launch(dc_ctx *ctx, const dc_kv_cache *c, const void *Q, long qs, PArgs a, bool few) {
  using C = WideCfg<D>;
  CUtensorMap tq;
  const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)a.heads, (cuuint64_t)a.T};
  const cuuint64_t strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)qs * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)a.r, (cuuint32_t)a.tpt};
  int rc = encode(&tq, Q, 3, dims, strides, box);
  if (rc) return rc;
  if (few) {  // (D <= 128)
    rc = attn_few_launch(ctx, D, tq, c->mapK, c->mapV, a);
  } else {
    static uint64_t attr_done = 0;
    if (!(attr_done & (1ull << ctx->device))) {
      DC_CUDA(cudaFuncSetAttribute(attention_paged_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
      attr_done |= 1ull << ctx->device;
    }
    DC_CUDA(dc_launch_pdl(ctx->stream, attention_paged_kernel<D>, dim3(ctx->sms), dim3(PA_THREADS), C::SMEM, tq, c->mapK,
                          c->mapV, a));
    rc = dc_launch_check("attention_paged");
  }
  if (rc) return rc;
  if (a.by_row) {
    const dim3 grid((unsigned)((long)a.T * a.heads));
    DC_CUDA(dc_launch_pdl(ctx->stream, attention_join_kernel<D>, grid, dim3(128), 0, a));
    return dc_launch_check("attention_paged (join)");
  }
  constexpr int R = 4 * JoinRows<D>::R;  // of a block
  const dim3 grid((unsigned)((std::min((long)a.T * a.r, 128L) + R - 1) / R), a.ctas);
  DC_CUDA(dc_launch_pdl(ctx->stream, attention_join_tiles_kernel<D>, grid, dim3(128), 0, a));
  return dc_launch_check("attention_paged (join)");
}

}  // namespace

int attn_cache_maps(dc_kv_cache *c) {
  const cuuint64_t dims[2] = {(cuuint64_t)c->D, (cuuint64_t)c->pages * c->kv * c->page};
  const cuuint64_t strides[1] = {(cuuint64_t)c->D * 2};
  const cuuint32_t box[2] = {64, (cuuint32_t)std::min(c->page, 64)};
  int rc = encode(&c->mapK, c->K, 2, dims, strides, box);
  return rc ? rc : encode(&c->mapV, c->V, 2, dims, strides, box);
}

size_t attn_paged_ws(dc_ctx *ctx, const dc_kv_cache *c, int T, int heads) {
  return ws_layout(T, heads, c->kv, c->D, 2 * ctx->sms).bytes;
}

int attn_paged_launch(dc_ctx *ctx, const dc_kv_cache *c, const void *Q, long qs, const int *table, int tstride,
                      const int *lens, const int *qoff, int S, const int *ptable, int pstride, const int *plens,
                      const int *goff, int G, void *Y, long ys, int T, int heads, float scale, void *ws) {
  const Ws w = ws_layout(T, heads, c->kv, c->D, 2 * ctx->sms);
  char *p = reinterpret_cast<char *>((reinterpret_cast<uintptr_t>(ws) + WS_ALIGN - 1) & ~(uintptr_t)(WS_ALIGN - 1));
  PArgs a;
  a.Y = static_cast<__half *>(Y), a.ystride = ys;
  a.table = table, a.lens = lens, a.qoff = qoff, a.ptable = ptable, a.plens = plens, a.goff = goff;
  a.first = reinterpret_cast<int *>(p + w.first), a.last = reinterpret_cast<int *>(p + w.last);
  a.hdr = reinterpret_cast<int *>(p), a.head = reinterpret_cast<int4 *>(p + w.head);
  a.tail = reinterpret_cast<int *>(p + w.tail), a.ml = reinterpret_cast<float2 *>(p + w.ml);
  a.O = reinterpret_cast<float *>(p + w.O);
  a.err = ctx->d_err;
  a.tstride = tstride, a.pstride = pstride, a.S = S, a.G = G, a.T = T, a.heads = heads, a.kv = c->kv;
  a.r = heads / c->kv;
  const bool few = paged_few(c->D, T, a.r, G);
  const int ctas = few ? 2 * ctx->sms : ctx->sms;
  a.tpt = 128 / a.r, a.page = c->page, a.pages = c->pages;
  a.pshift = c->page == 16 ? 4 : c->page == 32 ? 5 : c->page == 64 ? 6 : 7, a.rows = c->pages * c->kv * c->page;
  a.chunk_min = 2;  // no stretch is shorter, so that short calls have few parts (1 and 4 measured the same)
  a.ctas = ctas;
  // Few tiles are cut into many parts each, and a join by row takes them up in four warps (one sequence over 30,000 keys 26
  // us against 48 by tile, 35 over a shared prefix 36 against 67, 8 groups of 4 x 16 tokens 20 against 23). Many tiles are
  // whole or in two or three parts, and blocks for rows that were not cut would cost more than the tiles' search (24 groups
  // of 12 tokens 95 us by row, 91 by tile; 16 groups of 8 x 8 tokens 34 and 31; 32 of 3 questions 54 and 41). At D = 256
  // fewer such blocks fit an SM: 4,000 rows 43 us by row, 41 by tile; 400 rows 35 and 36; one 25 and 40.
  const long groups = std::max(G, 1), tiles = c->kv * groups * (((long)T * a.r + 128 * groups - 1) / (128 * groups));
  a.by_row = 3 * tiles <= ctas && (c->D < 256 || (long)T * heads <= 2048);
  a.y32 = (reinterpret_cast<uintptr_t>(Y) & 31) == 0 && ys % 16 == 0;
  a.scale_log2 = scale * 1.4426950408889634f;
  if (c->D == 64) return launch<64>(ctx, c, Q, qs, a, few);
  if (c->D == 128) return launch<128>(ctx, c, Q, qs, a, few);
  return launch<256>(ctx, c, Q, qs, a, few);
}
