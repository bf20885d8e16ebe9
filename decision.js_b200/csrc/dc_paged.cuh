// What the kernels over the paged cache share: the line of blocks and how a CTA finds and walks its stretch of it, the
// producers of K and V, and the warp that looks values over. A kernel's layout C names its shared memory, barriers and
// threads.
#pragma once
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <float.h>

#include "dc_internal.h"
#include "dc_ptx.cuh"

namespace dcx {

constexpr int PA_RING = 4;    // runs handed out ahead
// Tiles whose rows' marks (128 bits each) are held at a time. A tile's are cleared PA_RING tiles ahead (look_over), while
// those of up to PA_RING tiles before may still be read.
constexpr int PA_MARKS = 2 * PA_RING, PA_MARK_BYTES = PA_MARKS * 16;
constexpr int PA_GOFF = 512;  // groups and sequences whose offsets and lengths are kept in shared memory
constexpr int PA_META = 4 * (PA_GOFF + 4) * 4;  // bytes

#define MINUS_INF __uint_as_float(0xff800000u)

enum { RUN_FIRST = 1, RUN_LAST = 2, RUN_TFIRST = 4, RUN_TLAST = 8, RUN_END = 16 };

// A run of blocks of one segment (the prefix or one sequence's own keys) for one tile.
struct Run {
  const int *tab;          // its page row
  int tok0, ntok, kvh;     // the tile
  int flags, item;
  int seg;                 // sequence, or -1: the prefix
  int kb, nb, kend;        // first block, blocks, keys of the segment that the tile's last row in it sees
  int qb, qe, len;         // own runs: the sequence's rows and own keys
};

struct PArgs {
  __half *Y;
  const int *table, *lens, *qoff, *ptable, *plens, *goff;
  int *hdr;
  // what the join goes by: with by_row, first and last CTA of each (kv head, row)'s tile, first -1 where it was not cut;
  // else by CTA the tile that it ends and did not begin (first row, rows, kv head; no rows: none), and whether it begins
  // a tile that it does not end
  int *first, *last;
  int4 *head;
  int *tail;
  float2 *ml;  // a part's (maximum, sum of weights) by row; (minus infinity, 0): keys were seen and all scored that
  float *O;
  uint32_t *err;
  long ystride;
  int tstride, pstride, S, G, T, heads, kv, r, tpt, page, pshift, pages, rows, chunk_min, ctas, by_row, y32;
  float scale_log2;
};

__device__ __forceinline__ uint64_t desc_mn(uint32_t saddr, uint32_t lbo) {
  // MN-major operand in 128-byte-swizzled {64, rows} boxes: 8-row groups 1024 bytes apart, 64-wide chunks `lbo` apart
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (uint64_t)((lbo >> 4) & 0x3FFFu) << 16 | (uint64_t)(1024 >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

__device__ __forceinline__ void st_global_v8(void *p, const uint32_t *r) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

// 16 values of a row of Y: whole 32-byte sectors where Y's rows begin at them (y32).
__device__ __forceinline__ void store_row16(__half *y, const uint32_t *w, int y32) {
  if (y32) {
    st_global_v8(y, w);
  } else {
    reinterpret_cast<uint4 *>(y)[0] = make_uint4(w[0], w[1], w[2], w[3]);
    reinterpret_cast<uint4 *>(y)[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
}

// own keys that query row `t` of a sequence [.., qe) with `len` own tokens sees
__device__ __forceinline__ int own_limit(int t, int qe, int len) { return max(len - (qe - 1 - t), 0); }
template <int KB>
__device__ __forceinline__ int blocks_of(int keys) { return (keys + KB - 1) / KB; }

struct Groups {  // offsets and lengths of groups and sequences, from shared memory when they fit
  const int *goff, *plens, *qoff, *lens;
  int G, S;
  __device__ __forceinline__ int of(int s) const {  // the last g with goff[g] <= s
    int lo = 0, hi = G;
#pragma unroll 1
    while (hi - lo > 1) {
      const int m = (lo + hi) >> 1;
      if (goff[m] <= s) lo = m; else hi = m;
    }
    return lo;
  }
};

struct Group {
  int tg, te, pb;  // its rows, its prefix's blocks
};
template <int KB>
__device__ __forceinline__ Group group_of(const Groups &gs, int g) {
  if (gs.G == 0) return Group{gs.qoff[0], gs.qoff[gs.S], 0};
  return Group{gs.qoff[min(max(gs.goff[g], 0), gs.S)], gs.qoff[min(max(gs.goff[g + 1], 0), gs.S)], blocks_of<KB>(gs.plens[g])};
}

// The units of a sequence: for each tile its rows touch, the prefix's blocks if the tile starts in it, and its own.
template <int KB>
static __device__ __forceinline__ long seq_cost(int tpt, Group g, int qb, int qe, int len) {
  long c = 0;
  const int lo = qb - g.tg, hi = qe - g.tg;
  if (hi <= lo) return 0;
#pragma unroll 1
  for (int ts = lo / tpt * tpt; ts < hi; ts += tpt) {
    if (ts >= lo) c += g.pb;
    c += max(1, blocks_of<KB>(own_limit(g.tg + min(hi, ts + tpt) - 1, qe, len)));
  }
  return c;
}

// The page ids of a sequence's first 32 pages (`len` tokens), read while the run before it is loaded (lanes past them: 0;
// the table's row may end there, and the tensor with it).
__device__ __forceinline__ int read_ahead(const PArgs &a, int s, int len, int lane) {
  return s < a.S && lane < (len + a.page - 1) >> a.pshift ? a.table[(long)s * a.tstride + lane] : 0;
}

static __device__ __noinline__ void bad_page(uint32_t *err) { atomicOr(err, (uint32_t)DC_DEVERR_BOUNDS); }

// A run's blocks for a producer warp: page ids are read 32 at a time, the next 32 on their way, and turned into rows of
// the cache as tensor-map coordinates before the stage is waited for.
template <class C>
struct Blocks {
  static constexpr int NA = C::NA, KB = C::KB, NB = KB / 16;
  const int *tab;
  int base, count, cur, nxt, kend, kvh;
  __device__ __forceinline__ int row_of(const PArgs &a, int id) const {
    if ((unsigned)id < (unsigned)a.pages) return (id * a.kv + kvh) << a.pshift;
    bad_page(a.err);
    return a.rows;  // past the cache: zeros
  }
  __device__ __forceinline__ int ld(const PArgs &a, int i) const { return i < count ? row_of(a, tab[i]) : a.rows; }
  // `ahead`: the ids of the first 32 pages of sequence ahead_seq, if they were read already. The ids are on their way
  // until settle() looks at them.
  __device__ __forceinline__ void start(const PArgs &a, const Run &r, int lane, int ahead_seq, int ahead) {
    tab = r.tab, kend = r.kend, kvh = r.kvh, count = (kend + a.page - 1) >> a.pshift, base = (r.kb * KB) >> a.pshift;
    const bool have = r.seg >= 0 && r.seg == ahead_seq && base == 0;
    cur = have ? ahead : base + lane < count ? tab[base + lane] : 0;
    nxt = base + 32 + lane < count ? tab[base + 32 + lane] : 0;
  }
  __device__ __forceinline__ void settle(const PArgs &a, int lane) {
    cur = base + lane < count ? row_of(a, cur) : a.rows;
    nxt = base + 32 + lane < count ? row_of(a, nxt) : a.rows;
  }
  // The whole warp: block `kb`'s rows, one per box of min(page, 64) rows (boxes that hold none of the run's keys are
  // left out).
  struct Rows {
    int row[NB], n, prow;
  };
  __device__ __forceinline__ Rows rows(const PArgs &a, int kb, int lane) {
    Rows x;
    const int pr = min(a.pshift, 6), key0 = kb * KB, i = key0 >> a.pshift, sub = a.pshift - pr;
    x.prow = 1 << pr;
    if (i - base >= 32) base += 32, cur = nxt, nxt = ld(a, base + 32 + lane);
    x.n = min(KB >> pr, (kend - key0 + x.prow - 1) >> pr);
    const int first = (key0 & (a.page - 1)) >> pr;  // the first box within its page
#pragma unroll
    for (int p = 0; p < NB; p++) {
      const int at = first + p, v = __shfl_sync(0xffffffffu, cur, (i - base + (at >> sub)) & 31);
      x.row[p] = v == a.rows ? v : v + ((at & ((1 << sub) - 1)) << pr);
    }
    return x;
  }
  // One thread.
  __device__ __forceinline__ static void load(const CUtensorMap *map, const Rows &x, uint32_t dst, uint32_t full) {
    mbar_expect_tx(full, (uint32_t)(x.n * NA * x.prow * 128));
#pragma unroll
    for (int p = 0; p < NB; p++) {
      if (p >= x.n) break;
#pragma unroll
      for (int j = 0; j < NA; j++) tma_load_2d(dst + j * (KB * 128) + p * x.prow * 128, map, 64 * j, x.row[p], full);
    }
  }
};

// A CTA's view of its shared memory, with the waits of its roles.
template <class C>
struct Cta {
  const PArgs &a;
  uint8_t *smem;
  uint32_t base;
  int tid, warp, lane;
  __device__ __forceinline__ Cta(const PArgs &args, uint8_t *raw) : a(args) {
    smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    base = smem_u32(smem);
    tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  }
  __device__ __forceinline__ uint32_t bar(int i) const { return base + C::BAR_OFF + 8u * (uint32_t)i; }
  __device__ __forceinline__ uint32_t *tmem_slot() const { return reinterpret_cast<uint32_t *>(smem + C::MISC_OFF); }
  __device__ __forceinline__ volatile int *abort() const { return reinterpret_cast<volatile int *>(smem + C::MISC_OFF + 4); }
  __device__ __forceinline__ int *start() const { return reinterpret_cast<int *>(smem + C::MISC_OFF + 8); }
  __device__ __forceinline__ volatile uint32_t *poison(int item) const {  // marked rows of a tile, 128 bits
    return reinterpret_cast<volatile uint32_t *>(smem + C::POISON_OFF) + 4 * (item % PA_MARKS);
  }
  // every thread, before the first barrier: no marks
  __device__ __forceinline__ void clear_marks() const {
    if (tid < PA_MARK_BYTES / 4) reinterpret_cast<uint32_t *>(smem + C::POISON_OFF)[tid] = 0;
  }
  __device__ __forceinline__ Run *runs() const { return reinterpret_cast<Run *>(smem + C::RUN_OFF); }
  __device__ __forceinline__ bool wait(int i, int parity) const {
    return mbar_wait_asleep(bar(i), (uint32_t)parity & 1u, abort(), a.err, DC_DEVERR_ATTN_WAIT);
  }
  // the whole warp waits, and goes on or gives up together
  __device__ __forceinline__ bool wait_warp(int i, int parity) const {
    return __all_sync(0xffffffffu, wait(i, parity)) != 0;
  }
  // one thread that issues products
  __device__ __forceinline__ bool wait1(int i, int parity) const {
    return mbar_wait_alert(bar(i), (uint32_t)parity & 1u, abort(), a.err, DC_DEVERR_ATTN_WAIT);
  }
  // a consumer's n-th run: false at the end (or on abort)
  __device__ __forceinline__ bool next_run(int n, Run &r) const {
    if (!wait_warp(C::B_IF + n % PA_RING, n / PA_RING)) return false;
    r = runs()[n % PA_RING];
    return !(r.flags & RUN_END);
  }
  __device__ __forceinline__ void done_run(int n) const {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(C::B_IE + n % PA_RING));
  }
};

// A CTA's stretch [p0, p1) of the line; it begins at kv head kvh (the sequence and the place in it are left in start()).
struct Stretch {
  long p0, p1;
  int kvh;
};

// The line: units per sequence, their sum, this CTA's stretch. Every thread calls it; false: the arrays are refused, in
// every CTA alike. A barrier has to follow before the stretch is walked.
template <class C>
__device__ __forceinline__ bool line_start(const Cta<C> &k, Groups &gs, Stretch &st) {
  constexpr int KB = C::KB;
  const PArgs &a = k.a;
  const int tid = k.tid, warp = k.warp, lane = k.lane;
  int *s_start = k.start(), *s_goff = reinterpret_cast<int *>(k.smem + C::GOFF_OFF);
  long *s_scan = reinterpret_cast<long *>(k.smem + C::SCAN_OFF);
  bool bad = false;
  gs = Groups{a.goff, a.plens, a.qoff, a.lens, a.G, a.S};
  // into shared memory, all in one round of loads
  int *s_plens = s_goff + PA_GOFF + 4, *s_qoff = s_plens + PA_GOFF + 4, *s_lens = s_qoff + PA_GOFF + 4;
  if (a.S <= PA_GOFF) {
#pragma unroll 1
    for (int i = tid; i <= a.S; i += C::THREADS) {
      s_qoff[i] = a.qoff[i];
      if (i < a.S) s_lens[i] = a.lens[i];
    }
    gs.qoff = s_qoff, gs.lens = s_lens;
  }
  if (a.G > 0 && a.G <= PA_GOFF) {
#pragma unroll 1
    for (int i = tid; i <= a.G; i += C::THREADS) {
      s_goff[i] = a.goff[i];
      if (i < a.G) s_plens[i] = a.plens[i];
    }
    gs.goff = s_goff, gs.plens = s_plens;
  }
  const int per = (a.S + C::THREADS - 1) / C::THREADS;
  const int sb = min(tid * per, a.S), se = min(sb + per, a.S);
  __syncthreads();
  dc_pdl_launch_dependents();
  if (a.G > 0) {
#pragma unroll 1
    for (int i = tid; i < a.G; i += C::THREADS) {
      const int x = gs.goff[i], y = gs.goff[i + 1], n = gs.plens[i];
      bad |= x < 0 || y < x || y > a.S || n < 0 || n > (long)a.pstride * a.page || n > (1 << 30);
    }
    if (tid == 0) bad |= gs.goff[0] != 0 || gs.goff[a.G] != a.S;
  }
  // a sequence's units; nothing for offsets that are refused below (the sum is then not used)
  auto units = [&](int s, int qb, int qe, int len) -> long {
    if (qb < 0 || qe <= qb || qe > a.T || len < 0) return 0;
    const Group g = group_of<KB>(gs, a.G ? gs.of(s) : 0);
    return g.tg < 0 || g.tg > qb ? 0 : seq_cost<KB>(a.tpt, g, qb, qe, len);
  };
  long mine = 0;
#pragma unroll 1
  for (int s = sb; s < se; s++) {
    const int x = gs.qoff[s], y = gs.qoff[s + 1], n = gs.lens[s];
    bad |= x < 0 || y < x || y > a.T || n < 0 || n > (long)a.tstride * a.page || n > (1 << 30);
    mine += units(s, x, y, n);
  }
  long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) s_scan[warp] = incl;
  if (__syncthreads_or(bad)) {  // the same in every CTA
    if (blockIdx.x == 0 && tid == 0) a.hdr[0] = 1, atomicOr(a.err, (uint32_t)DC_DEVERR_BOUNDS);
    return false;
  }
  if (tid == 0) {
    if (blockIdx.x == 0) a.hdr[0] = 0;
    a.head[blockIdx.x] = make_int4(0, 0, 0, 0), a.tail[blockIdx.x] = 0;
  }
  long before = incl - mine, line = 0;
#pragma unroll
  for (int w = 0; w < C::THREADS / 32; w++) {
    const long v = s_scan[w];
    if (w < warp) before += v;
    line += v;
  }
  const long B = line * a.kv;
  long chunk;
  st.kvh = 0;
  const int sh = B < 0x7fff0000 ? 0 : 16;  // (64-bit divisions take a microsecond)
  chunk = max((long)a.chunk_min, (long)(((unsigned)(B >> sh) + gridDim.x - (sh ? 0 : 1)) / gridDim.x) << sh);
  st.p0 = chunk * blockIdx.x;
  if (st.p0 < B) {
    if (sh == 0)
      st.kvh = (unsigned)st.p0 / (unsigned)line;
    else
#pragma unroll 1
      while (line * (st.kvh + 1) <= st.p0) st.kvh++;
  }
  st.p1 = min(st.p0 + chunk, B);
  if (st.p0 < st.p1 && mine > 0) {
    long off = st.p0 - st.kvh * line - before;
    if (off >= 0 && off < mine) {
      int s = sb;
#pragma unroll 1
      for (; s < se - 1; s++) {
        const long c = units(s, gs.qoff[s], gs.qoff[s + 1], gs.lens[s]);
        if (off < c) break;
        off -= c;
      }
      s_start[0] = s, s_start[1] = (int)(uint32_t)off, s_start[2] = (int)(off >> 32);
    }
  }
  return true;
}

// The producers of K and of V, a warp each, in the same code (which the instruction caches then hold once). Both walk the
// line; K's hands out the runs and loads Q.
template <class C>
__device__ __forceinline__ void walk_line(const Cta<C> &k, const Groups &gs, const Stretch &st, const bool values,
                                          const CUtensorMap *tmQ, const CUtensorMap *map) {
  constexpr int KB = C::KB, NA = C::NA;
  const int stages = values ? C::VST : C::KST, filled = values ? C::B_VF : C::B_KF, empty = values ? C::B_VE : C::B_KE;
  const uint32_t ring = k.base + (values ? C::V_OFF : C::K_OFF);
  int stage = 0, turn = 1;
  const PArgs &a = k.a;
  const int lane = k.lane;
  const int *s_start = k.start();
  int item = -1, n = 0;  // tiles, runs
  bool ok = true, first = true;
  long pos = st.p0, off = (long)(uint32_t)s_start[1] | (long)s_start[2] << 32;  // on the line; in the sequence's pieces
  int s = s_start[0], kvh = st.kvh, gi = a.G ? gs.of(s) : 0;
  Group gr = group_of<KB>(gs, gi);
  int qb = gs.qoff[s], qe = gs.qoff[s + 1], len = gs.lens[s];
  int lo = qb - gr.tg, hi = qe - gr.tg, ts = lo / a.tpt * a.tpt;  // from the group's first row; ts: the piece's tile
  // the next sequence's offset, length and first pages, on their way while this one's blocks are loaded
  int nqe = s + 1 < a.S ? gs.qoff[s + 2] : 0, nlen = s + 1 < a.S ? gs.lens[s + 1] : 0;
  int ahead_seq = -1, ahead = 0, coming = read_ahead(a, s + 1, nlen, lane);
  auto advance = [&]() {
    do {
      if (++s == a.S) {
        s = 0, kvh++, gi = 0;
        qb = gs.qoff[0], qe = gs.qoff[1], len = gs.lens[0];
        ahead_seq = -1;
      } else {
        qb = qe, qe = nqe, len = nlen;
        ahead_seq = s, ahead = coming;
      }
      if (s + 1 < a.S) nqe = gs.qoff[s + 2], nlen = gs.lens[s + 1];
      coming = read_ahead(a, s + 1, nlen, lane);
    } while (qe <= qb && kvh < a.kv);
    while (gi + 1 < a.G && gs.goff[gi + 1] <= s) gi++;
    gr = group_of<KB>(gs, gi);
    lo = qb - gr.tg, hi = qe - gr.tg, ts = lo / a.tpt * a.tpt;
  };
  while (pos < st.p1 && kvh < a.kv) {
    const int rows = gr.te - gr.tg, pe = min(hi, ts + a.tpt);
    const bool starts = ts >= lo, ends = pe == min(rows, ts + a.tpt);
    const int pc = starts ? gr.pb : 0, lim = own_limit(gr.tg + pe - 1, qe, len), all = pc + max(1, blocks_of<KB>(lim));
    if (off >= all) {  // the next piece
      off -= all, ts += a.tpt;
      if (ts >= hi) advance();
      continue;
    }
    const bool prefix = off < pc;
    const int units = (int)min((prefix ? pc : all) - off, st.p1 - pos);
    const bool done = off + units == all && ends;
    Run r;
    r.qb = qb, r.qe = qe, r.len = len;
    r.tok0 = gr.tg + ts, r.ntok = min(rows - ts, a.tpt), r.kvh = kvh;
    r.tab = prefix ? a.ptable + (long)gi * a.pstride : a.table + (long)s * a.tstride;
    r.seg = prefix ? -1 : s, r.kend = prefix ? gs.plens[gi] : lim;
    r.kb = (int)(prefix ? off : off - pc), r.nb = r.kend > 0 ? units : 0;
    r.flags = (first ? RUN_FIRST : 0) | (off == 0 && starts ? RUN_TFIRST : 0) |
              (done || pos + units == st.p1 ? RUN_LAST : 0) | (done ? RUN_TLAST : 0);
    pos += units, off += units;
    if (r.nb == 0 && !(r.flags & (RUN_FIRST | RUN_LAST))) continue;  // (a run in a tile's midst always has blocks)
    if (first) item++;
    r.item = item;
    Blocks<C> bl;
    bl.start(a, r, lane, ahead_seq, ahead);
    if (!values) {
      if (!(ok = k.wait_warp(C::B_IE + n % PA_RING, n / PA_RING + 1))) break;
      if (lane == 0) {
        k.runs()[n % PA_RING] = r;
        mbar_arrive(k.bar(C::B_IF + n % PA_RING));
      }
      n++;
      __syncwarp();
    }
    bl.settle(a, lane);
    // Q comes after as many blocks as the ring takes without it: its buffer is free only when the tile before is done
    const int q_at = !first || values ? -1 : item == 0 ? 0 : min(r.nb, C::KST);
#pragma unroll 1
    for (int b = 0;; b++) {
      if (b == q_at) {
        if (!(ok = k.wait_warp(C::B_QE, item + 1))) break;
        if (elect_one()) {
          mbar_expect_tx(k.bar(C::B_QF), (uint32_t)(a.r * a.tpt * 128 * NA));
#pragma unroll 1
          for (int j = 0; j < NA; j++)
            tma_load_3d(k.base + j * C::Q_ROWS * 128, tmQ, 64 * j, r.kvh * a.r, r.tok0, k.bar(C::B_QF));
        }
        __syncwarp();
      }
      if (b == r.nb) break;
      const typename Blocks<C>::Rows x = bl.rows(a, r.kb + b, lane);
      if (!(ok = k.wait_warp(empty + stage, turn))) break;
      if (elect_one()) bl.load(map, x, ring + stage * C::KV_BYTES, k.bar(filled + stage));
      __syncwarp();
      if (++stage == stages) stage = 0, turn ^= 1;
    }
    if (!ok) break;
    first = (r.flags & RUN_LAST) != 0;
  }
  if (!values && ok && k.wait_warp(C::B_IE + n % PA_RING, n / PA_RING + 1) && lane == 0) {
    k.runs()[n % PA_RING].flags = RUN_END;
    mbar_arrive(k.bar(C::B_IF + n % PA_RING));
  }
  int *loaded = reinterpret_cast<int *>(k.smem + C::LOADED_OFF);  // for settle
  if (lane == 0) loaded[values] = stage | turn << 8 | item << 9;
}

// After a wait ran out and every role has stopped (the whole CTA calls it): the loads and products still in flight. Of a ring
// the stages below `stage` hold the loads of the last time around, the others those of the time before (or none, which passes).
// Warps mma0 and mma1 issued the products, from the thread that elect_one names.
template <class C>
static __device__ __noinline__ void settle(uint8_t *smem, int mma0, int mma1) {
  const uint32_t bars = smem_u32(smem) + C::BAR_OFF;
  const int tid = threadIdx.x, warp = tid >> 5;
  if (tid < 2) {
    const int x = reinterpret_cast<int *>(smem + C::LOADED_OFF)[tid], stage = x & 255, turn = x >> 8 & 1, item = x >> 9;
    for (int s = 0; s < (tid ? C::VST : C::KST); s++)
      mbar_settle(bars + 8 * ((tid ? C::B_VF : C::B_KF) + s), s < stage ? turn ^ 1 : turn);
    if (tid == 0) mbar_settle(bars + 8 * C::B_QF, item & 1);  // (the last tile's Q, if it was asked for)
  }
  __syncwarp();
  if ((warp == mma0 || warp == mma1) && elect_one()) {
    const uint32_t end = bars + 8 * (warp == mma0 ? C::B_END : C::B_END + 1);
    mma_commit(end);
    mbar_settle(end, 0);
  }
  __syncthreads();
}

// Whether `n` 16-byte chunks of f16, `step` bytes apart, are finite: 0 x summed is 0 then and else NaN.
__device__ __forceinline__ bool all_finite(const uint8_t *p, int step, int n) {
  __half2 sum[4];
#pragma unroll
  for (int e = 0; e < 4; e++) sum[e] = __half2half2(__ushort_as_half(0));
#pragma unroll 4
  for (int i = 0; i < n; i++) {
    const uint4 x = *reinterpret_cast<const uint4 *>(p + i * step);
    const __half2 *h = reinterpret_cast<const __half2 *>(&x);
#pragma unroll
    for (int e = 0; e < 4; e++) sum[e] = __hfma2(h[e], __half2half2(__ushort_as_half(0)), sum[e]);
  }
  const __half2 all = __hadd2(__hadd2(sum[0], sum[1]), __hadd2(sum[2], sum[3]));
  return !(__hisnan(__low2half(all)) || __hisnan(__high2half(all)));
}
// Zeroes the chunks at rows row, row + step, ... < end of a column of chunks (rows 128 bytes apart) that hold a value that
// is not finite, and gives the first such row (1 << 20: none).
static __device__ __noinline__ int clear_not_finite(uint8_t *p, int row, int step, int end) {
  int first = 1 << 20;
  for (; row < end; row += step)
    if (!all_finite(p + row * 128, 0, 1)) {
      *reinterpret_cast<uint4 *>(p + row * 128) = make_uint4(0, 0, 0, 0);
      first = min(first, row);
    }
  return first;
}
// The rows [from, to) of a tile's 128 as the four words of a bit mask: word w.
__device__ __forceinline__ uint32_t mask_word(int from, int to, int w) {
  const int x = min(max(from - 32 * w, 0), 32), y = min(max(to - 32 * w, 0), 32);
  const uint32_t upto = y >= 32 ? ~0u : (1u << y) - 1u, under = x >= 32 ? ~0u : (1u << x) - 1u;
  return upto & ~under;
}
// Marks the tokens of a run's sequence in the tile that see key `key` of it (four lanes, a word each).
__device__ __forceinline__ void mark_rows(volatile uint32_t *mark, const Run &r, int key, int lane) {
  const int from = max(max(r.tok0, r.qb), key - r.len + r.qe) - r.tok0, to = min(r.qe, r.tok0 + r.ntok) - r.tok0;
  const uint32_t m = lane < 4 ? mask_word(from, to, lane) : 0u;
  if (m) atomicOr(const_cast<uint32_t *>(mark) + lane, m);
}

// Whether the block of a run at key0 has to be looked over before its product: the 16 keys of a product step reach past
// the last key, or a row of the tile that sees the block does not see all its keys (its first such row sees the fewest).
template <int KB>
__device__ __forceinline__ bool partly_seen(const Run &r, int key0) {
  const int t = max(max(r.tok0, r.qb), key0 - r.len + r.qe);
  return r.seg >= 0 && own_limit(t, r.qe, r.len) < min(key0 + KB, r.kend);
}
template <int KB>
__device__ __forceinline__ bool to_look_over(const Run &r, int key0) {
  return (min(KB, r.kend - key0) & 15) != 0 || partly_seen<KB>(r, key0);
}

// Looks those blocks over, one warp: the rows past the last key are zeroed, and values that are not finite too where some
// row would multiply them by a weight of 0, with a mark on the rows that see them. The product of the c-th of them waits
// for barrier B_VS + c % VST; the others go straight from V's arrival, so a tile without such a block can end, and its marks
// be read, before this warp has come to it. Its marks are therefore cleared earlier, and the ring of runs gives the order:
// at the start of tile i this warp clears those of tile i + PA_RING, whose runs are handed out only after its done_run of a
// run of tile i or later (a tile has at least one run, the ring PA_RING); the place was last that of tile i - PA_RING, whose
// last run every reader has given back before tile i's first is handed out. The first PA_RING tiles: clear_marks.
template <class C>
__device__ __forceinline__ void look_over(const Cta<C> &k) {
  constexpr int KB = C::KB, VST = C::VST, NA = C::NA;
  const int lane = k.lane;
  Run r;
  int g = 0, looked = 0;
  bool ok = true;
  for (int n = 0; ok && k.next_run(n, r); n++) {
    volatile uint32_t *mark = k.poison(r.item);
    if ((r.flags & RUN_FIRST) && lane < 4) k.poison(r.item + PA_RING)[lane] = 0;
    __syncwarp();
    for (int b = 0; b < r.nb; b++, g++) {
      const int st = g % VST, key0 = (r.kb + b) * KB;
      if (!(ok = k.wait_warp(C::B_VF + st, g / VST))) break;
      // every block counts this warp among those that give its stage back, or it could fall a phase behind
      if (!to_look_over<KB>(r, key0)) {
        if (lane == 0) mbar_arrive(k.bar(C::B_VE + st));
        continue;
      }
      const int valid = min(KB, r.kend - key0), pad = (valid + 15) & ~15;
      uint8_t *v = k.smem + C::V_OFF + st * C::KV_BYTES + (lane & 7) * 16;
      for (int row = valid + lane / 8; row < pad; row += 4)
#pragma unroll
        for (int at = 0; at < NA; at++) *reinterpret_cast<uint4 *>(v + at * (KB * 128) + row * 128) = make_uint4(0, 0, 0, 0);
      if (partly_seen<KB>(r, key0)) {
        int worst = KB;  // the first row with a value that is not finite
#pragma unroll 1
        for (int at = 0; at < NA; at++) {
          if (__any_sync(0xffffffffu, !all_finite(v + at * (KB * 128) + (lane / 8) * 128, 512, (valid - lane / 8 + 3) / 4)))
            worst = min(worst, clear_not_finite(v + at * (KB * 128), lane / 8, 4, valid));
        }
        worst = __reduce_min_sync(0xffffffffu, worst);
        if (worst < KB) mark_rows(mark, r, key0 + worst, lane);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(k.bar(C::B_VS + looked % VST));
        mbar_arrive(k.bar(C::B_VE + st));
      }
      looked++;
    }
    if (ok) k.done_run(n);
  }
}

}  // namespace dcx
