// The paged KV cache's step plan and its attention for batches with shared
// prefixes, for sm_100a:
//   * plan:             request lengths -> row starts, positions, slot map; pages
//                       popped from a free stack into the block tables
//   * prefix_attention: causal GQA attention of each sequence's newest tokens over
//                       its paged history; the keys that a group of sequences
//                       shares are read and scored once for all their rows
//
// Measured on one B200 (bf16, D = 128, 40 query and 8 kv heads; device times, from replays
// of a CUDA graph; a call outside one adds 2 to 9 us of host side):
//   plan, 64 x 1 rows: 5 us; 510k rows of 256 prompts: 14 us. prefix_attention, 8 groups x
//   8 sequences, prefixes of 512 to 1024 and own keys of 432 to 6912 tokens: 132 us = 4.7
//   TB/s of the keys read once; one group of 256 on 16,384 shared tokens: 224 us = 391
//   TFLOP/s; 4 sequences of 260 tokens: 15 us.
// Groups cost a second unit and the join. Beside attention that reads every sequence's own
// history (paged_attention in decode_sm100.cu, whose repeated pages come from L2), one token
// a sequence: 8 groups x 8 on 1024 / 4096 / 8192 shared tokens and up to 500 own ones take
// 52 / 65 / 87 us against 28 / 72 / 140, one group of 64 on 4096 50 against 80; on short
// prefixes they lose. Several tokens a sequence are for this kernel with or without groups:
// 64 new tokens behind 1,024 shared ones, 64 sequences, 0.6 ms (0.2 without groups) against 11.7.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <algorithm>
#include <cmath>
#include <numeric>
#include <tuple>

#include "common.cuh"
#include "tma_host.h"

namespace kore {
namespace paged {

// ------------------------------------------------------------------- plan
struct PlanParams {
  const int *ctx, *new_toks, *held;     // held may be null: the pages that ctx tokens fill
  int* table;                           // plain loads: the rows read what the sequences' threads wrote
  long ld_table;
  int M, page_size;
  long B, rows;
  const int *free_stack, *free_count;   // free_count null: no pool (an empty stack has no address either)
  long nfree;
  int *q_start, *lens, *pos, *slots, *held_out, *count_out;
  bool* ok;
};

constexpr int kPlanThreads = 1024;
constexpr int kPlanRows = 4096;         // rows that the planning block maps itself: a launch less (2.5 us) for four rows a thread

// Inclusive sum over the block; `total` is the sum of all.
KORE_DEV long warp_scan(long v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long y = __shfl_up_sync(0xffffffff, v, o);
    if (lane >= o) v += y;
  }
  return v;
}
KORE_DEV long block_scan(long v, long* part, long& total) {
  static_assert(kPlanThreads == 32 * 32, "one warp adds the warps' sums");
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  v = warp_scan(v);
  __syncthreads();
  if (lane == 31) part[w] = v;
  __syncthreads();
  const long sums = warp_scan(part[lane]);
  total = __shfl_sync(0xffffffff, sums, 31);
  const long before = __shfl_sync(0xffffffff, sums, max(w - 1, 0));
  return v + (w ? before : 0);
}

// Positions and slots of rows t .. t + N - 1; q_start in global or shared memory.
template <int N>
KORE_DEV void plan_rows(const PlanParams& p, const int* q_start, long t) {
  int b = 0, hi = (int)p.B;             // the sequence with q_start[b] <= t < q_start[b + 1]
  while (b < hi) {
    const int mid = (int)(((unsigned)b + (unsigned)hi) >> 1);
    if (q_start[mid + 1] <= t) b = mid + 1; else hi = mid;
  }
  int pos[N], slot[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    while (b < p.B && q_start[b + 1] <= t + i) ++b;
    pos[i] = 0;                         // behind the last sequence
    slot[i] = -1;
    if (b == p.B || t + i >= p.rows) continue;
    pos[i] = max(p.ctx[b], 0) + (int)(t + i - q_start[b]);
    if (!p.ok[b]) continue;
    const int at = (unsigned)pos[i] / (unsigned)p.page_size, page = p.table[b * p.ld_table + at];
    const long s = (long)page * p.page_size + (pos[i] - at * p.page_size);
    if (page >= 0 && s <= 0x7fffffffL) slot[i] = (int)s;
  }
  if (N == 4 && t + 4 <= p.rows) {
    *reinterpret_cast<int4*>(p.pos + t) = make_int4(pos[0], pos[N / 4], pos[N / 2], pos[N - 1]);
    *reinterpret_cast<int4*>(p.slots + t) = make_int4(slot[0], slot[N / 4], slot[N / 2], slot[N - 1]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (t + i < p.rows) {
        p.pos[t + i] = pos[i];
        p.slots[t + i] = slot[i];
      }
  }
}

// One block: rows' starts and granted pages are running sums over the sequences. With
// `map_rows` (B <= 1024) it goes on to the rows.
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(PlanParams p, bool map_rows) {
  __shared__ long part[32];
  __shared__ int starts[kPlanThreads + 1], granted, asks[kPlanThreads], holds[kPlanThreads];
  pdl_trigger();
  const int count = p.free_count ? (int)min((long)max(*p.free_count, 0), p.nfree) : 0;
  long rows = 0, asked = 0, total;
  if (threadIdx.x == 0) {
    p.q_start[0] = starts[0] = 0;
    granted = 0;
  }
  for (long b0 = 0; b0 < p.B; b0 += kPlanThreads) {
    const long b = b0 + threadIdx.x;
    const bool in = b < p.B;
    const int want = in ? max(p.new_toks[b], 0) : 0, ctx = in ? max(p.ctx[b], 0) : 0;
    const int have = in && p.held ? min(max(p.held[b], 0), p.M) : 0;
    const long to = block_scan(want, part, total) + rows;
    rows += total;
    const long n = min(to, p.rows) - min(to - want, p.rows);   // a batch has p.rows rows: what is behind them is cut
    const long ps = p.page_size, need = (ctx + n + ps - 1) / ps, held = p.held ? have : (ctx + ps - 1) / ps;
    const bool fits = need <= p.M;
    const long take = p.free_count && fits ? max(need - held, 0L) : 0;
    long upto = 0;
    if (p.free_count) {
      upto = block_scan(take, part, total) + asked;
      asked += total;
    }
    const bool ok = fits && upto <= count;
    const int got = ok ? (int)take : 0;
    if (in) {
      if (got) atomicMax(&granted, (int)upto);       // granted sequences are a prefix of those that ask
      const int end = (int)min(to, p.rows);
      p.q_start[b + 1] = end;
      if (b0 == 0) starts[b + 1] = end;
      p.lens[b] = ok ? (int)(ctx + n) : ctx;
      p.ok[b] = ok;
      p.held_out[b] = (int)held + got;
    }
    if (p.free_count) {
      // pages to threads, not sequences to threads: a long prompt alone may ask for hundreds
      const long before = asked - total;
      asks[threadIdx.x] = (int)min(upto - before, (long)count + 1);
      holds[threadIdx.x] = (int)held;
      __syncthreads();
      const int most = (int)min(total, count - before);
      for (int k = threadIdx.x; k < most; k += kPlanThreads) {
        int lo = 0, hi = kPlanThreads - 1;           // whose page k of this round is
        while (lo < hi) {
          const int mid = (lo + hi) >> 1;
          if (asks[mid] <= k) lo = mid + 1; else hi = mid;
        }
        if (before + asks[lo] > count) continue;     // not granted
        const int j = k - (lo ? asks[lo - 1] : 0);
        p.table[(b0 + lo) * p.ld_table + holds[lo] + j] = p.free_stack[count - 1 - before - k];
      }
    }
  }
  __syncthreads();
  if (threadIdx.x == 0 && p.count_out) *p.count_out = count - granted;
  if (map_rows)
    for (long t = threadIdx.x; t < p.rows; t += kPlanThreads) plan_rows<1>(p, starts, t);
}

__global__ void __launch_bounds__(256) plan_rows_kernel(PlanParams p) {
  pdl_wait();
  const long t = 4 * ((long)blockIdx.x * blockDim.x + threadIdx.x);      // four rows to a search
  if (t < p.rows) plan_rows<4>(p, p.q_start, t);
}

// -------------------------------------------------------- prefix attention
// A unit of work is the prefix of a group (all query rows of its sequences against
// the shared keys) or a sequence's own keys (its rows against what follows the
// prefix). A unit is cut into items, one for each kv head and each block of query
// rows (row = token x query head of the kv head), and an item into tiles of 64 keys.
// All tiles, in one order, are dealt to the blocks in equal runs, so that a long
// prefix is split over as many blocks as it needs and no host value depends on the
// lengths. An item that one block has whole, and that no other unit's part joins, is
// written as the result; all else goes to fp32 partials (reference exponent, sum and
// unnormalised output), which a second kernel joins in a fixed order:
//   m = max m_i, l = sum l_i 2^(m_i - m), o = sum o_i 2^(m_i - m) / l.
//
// Items come in two forms, each with its own runs:
//   wide   S[128 rows x 64 keys] = Q K^T, O[128 x 128] += P V: prefixes, and own keys
//          when a sequence has more than 32 rows. One softmax thread owns a row.
//   narrow S^T[64 keys x N rows] = K Q^T, O^T[128 x N] += V^T P^T with N = 16 or 32:
//          own keys under few rows. A tile's exponentials are spread over its keys,
//          where the wide form would have one thread to a row do all of them.
// Every block has a run of each form, the narrow one first. (Half of them the other way
// round, so that one form's products overlap the other's loads, was slower by a third:
// the code of both does not fit the instruction cache.)
constexpr int D = 128;
constexpr int BK = 64;                            // keys of a tile
constexpr int kStages = 2;
constexpr int kTileBytes = BK * D * 2;            // 16 KB: 64 keys as two 8 KB swizzle atoms
constexpr int kQBytes = 128 * D * 2;
constexpr int kAttnThreads = 256;                 // producer, S products, O products, one more, four softmax warps
constexpr int kTmemCols = 256;                    // wide: two S / P buffers of 64 columns, O of 128; narrow: the same S buffers, two O
constexpr uint32_t kTmemO = 128;
constexpr int kMaxSeqs = 512;
constexpr float kLn2 = 0.6931471805599453f;

struct AttnParams {
  const int *table, *lens, *q_start;
  long ld_table;
  int M, page_size, B, T, Hq, Hkv, G;
  int tokens_prefix, tokens_own;                  // tokens of a row block, for a group's prefix and a sequence's own keys
  int nwide;                                      // units in wide form: the first nwide
  int box;                                        // keys of one TMA box: gcd(64, page_size)
  const int *group_start, *prefix;                // null: no groups
  int ngroups;
  float scale_log2;
  __nv_bfloat16* out;
  float* lse;
  // Partial rows: o, then m and l. Items that one block had whole, by their result's
  // row; what the runs cut, two items (a run's first and last) for each run.
  float *whole_prefix, *whole_own, *split_wide, *split_narrow;
  int4* where;                                    // [T][2] for the join: where the token's parts begin
  int* runs;                                      // wide tiles, narrow tiles
};
constexpr int kPart = D + 4;                      // floats of a partial row (16-byte aligned)

// mbar_wait without its limit's clock on the way in.
KORE_DEV bool wait_on(uint64_t* bar, uint32_t phase) { return mbar_try_wait(smem_u32(bar), phase) || mbar_wait(bar, phase); }
// A whole warp's wait: the lanes go on together or give up together.
KORE_DEV bool warp_wait(uint64_t* bar, uint32_t phase) { return __all_sync(0xffffffff, wait_on(bar, phase)); }

struct AttnSmem {
  static constexpr int Q_OFF = 0;                                    // wide: Q; narrow: two Q, then two P buffers
  static constexpr int K_OFF = kQBytes;
  static constexpr int V_OFF = K_OFF + kStages * kTileBytes;
  static constexpr int BAR_OFF = V_OFF + kStages * kTileBytes;
  static constexpr int X_OFF = BAR_OFF + 256;                        // NarrowSmem
  static constexpr int UNITS_OFF = X_OFF + 6 * 32 * 4;               // Units
  static constexpr int TOTAL = UNITS_OFF + 4 * 7 * kMaxSeqs + 1024;
};
static_assert(2 * (AttnSmem::TOTAL + 1024) <= 228 * 1024, "two blocks share an SM");

// Shared-memory layouts, all of 64-column (128-byte) swizzled atoms: Q 128 x 128 in two
// atoms of 16 KB; K and V 64 x 128 in two of 8 KB (V as an MN-major operand: rows = K);
// narrow Q N x 128 in two of N * 128 bytes and P^T N x 64 in one.
KORE_DEV void tma_load_4d(void* dst, const CUtensorMap* d, uint64_t* bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(d)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}
KORE_DEV void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  tmem_st16(taddr, *reinterpret_cast<const uint32_t(*)[16]>(&r[0]));
  tmem_st16(taddr + 16, *reinterpret_cast<const uint32_t(*)[16]>(&r[16]));
}
// Warp-wide maximum (NaN is passed over) and a vote and a barrier of the four softmax warps.
KORE_DEV float warp_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
KORE_DEV bool softmax_any(bool v) {
  uint32_t r;
  asm volatile(
      "{\n.reg .pred P, Q;\nsetp.ne.u32 P, %1, 0;\n"
      "barrier.cta.red.or.pred Q, 1, 128, P;\n"
      "selp.u32 %0, 1, 0, Q;\n}\n"
      : "=r"(r) : "r"((uint32_t)v) : "memory");
  return r != 0;
}
KORE_DEV void softmax_sync() { asm volatile("barrier.cta.sync 1, 128;" ::: "memory"); }

// The units as every block sees them, in shared memory: unit u < ngroups is a prefix,
// unit ngroups + b sequence b.
struct Units {
  const AttnParams& p;
  int *qs, *gs, *cum;     // [B + 1] rows, [ngroups + 1] sequences (both clamped to what exists), [units + 1] tiles before the unit
  int *len, *prefix;      // [B], [ngroups] keys, clamped to the table
  short* grp;             // [B] group, -1: none
  KORE_DEV Units(const AttnParams& p_, uint8_t* at) : p(p_) {
    qs = reinterpret_cast<int*>(at);
    gs = qs + kMaxSeqs + 4;
    cum = gs + kMaxSeqs + 4;
    len = cum + 2 * kMaxSeqs + 4;
    prefix = len + kMaxSeqs;
    grp = reinterpret_cast<short*>(prefix + kMaxSeqs);
    static_assert(3 * (kMaxSeqs + 4) + 3 * kMaxSeqs + kMaxSeqs / 2 <= 7 * kMaxSeqs, "the units fit");
  }
  KORE_DEV int seq_of(int t, int lo, int hi) const {  // the sequence in [lo, hi] that holds row t
#pragma unroll 1
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (qs[mid + 1] <= t) lo = mid + 1; else hi = mid;
    }
    return lo;
  }
  KORE_DEV int row0(int u) const { return u < p.ngroups ? qs[gs[u]] : qs[u - p.ngroups]; }
  KORE_DEV int tokens(int u) const {
    return u < p.ngroups ? qs[gs[u + 1]] - qs[gs[u]] : qs[u - p.ngroups + 1] - qs[u - p.ngroups];
  }
  KORE_DEV int block_tokens(int u) const { return u < p.ngroups ? p.tokens_prefix : p.tokens_own; }
  KORE_DEV int blocks(int u) const {
    const int tb = block_tokens(u), n = tokens(u);
    return n <= tb ? 1 : (n + tb - 1) / tb;
  }
  KORE_DEV void keys(int u, int& lo, int& hi) const {      // the unit's keys
    if (u < p.ngroups) {
      lo = 0;
      hi = prefix[u];
    } else {
      const int g = grp[u - p.ngroups];
      lo = g < 0 ? 0 : prefix[g];
      hi = len[u - p.ngroups];
    }
  }
  KORE_DEV int item_tiles(int u) const {
    int lo, hi;
    keys(u, lo, hi);
    return hi > lo ? (hi + BK - 1) / BK - lo / BK : 0;
  }
  KORE_DEV int tiles(int u) const { return tokens(u) > 0 ? item_tiles(u) * blocks(u) * p.Hkv : 0; }
  KORE_DEV bool shared(int b) const {                      // sequence b has a part that a group's unit computes
    const int g = grp[b];
    return g >= 0 && cum[g + 1] > cum[g];
  }
};

struct Item {
  int u, h, rb, n, j0, j1;       // unit, kv head, row block, tiles of the item, this run's tiles of it
};
struct Walk {                    // what is left of a run: tiles [x, end), x in unit u or behind it
  int x, end, u;
};
// The run's next item; false at its end.
KORE_DEV bool next_item(const Units& w, Walk& r, Item& it) {
  if (r.x >= r.end) return false;
#pragma unroll 1
  while (w.cum[r.u + 1] <= r.x) ++r.u;
  const int nb = w.blocks(r.u), d = r.x - w.cum[r.u];
  it.u = r.u;
  it.n = w.item_tiles(r.u);
  const int i = d / it.n;
  it.h = nb == 1 ? i : i / nb;
  it.rb = i - it.h * nb;
  it.j0 = d - i * it.n;
  it.j1 = min(it.n, it.j0 + r.end - r.x);
  r.x += it.j1 - it.j0;
  return true;
}
// W tiles dealt to C runs: run c is [start(c), start(c + 1)), start(c) = floor(c W / C).
struct Runs {
  int W, C, q, r;                // q = W / C, r = W % C
  KORE_DEV Runs(int W_, int grid) : W(W_), C(min(W_, grid)) {
    q = C ? W / C : 0;
    r = W - q * C;
  }
  KORE_DEV int start(int c) const { return c * q + (r ? (unsigned)(c * r) / (unsigned)C : 0); }
  KORE_DEV int of(int x) const { // whose run holds tile x
    int c = min((int)((float)x * (float)C / (float)W), C - 1);     // within one of it
    if (start(c) > x) --c;
    else if (start(c + 1) <= x) ++c;
    return c;
  }
};
KORE_DEV Walk make_walk(const int* cum, int nu, int base, const Runs& runs, int c) {
  Walk w = {0, 0, 0};
  if (c < runs.C) {
    w.x = base + runs.start(c);
    w.end = base + runs.start(c + 1);
    int lo = 0, hi = nu;         // the unit that holds w.x
#pragma unroll 1
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (cum[mid + 1] <= w.x) lo = mid + 1; else hi = mid;
    }
    w.u = lo;
  }
  return w;
}

// Narrow form: Q buffers (by the item's number) and, behind them, two P buffers (by the tile's parity).
constexpr int p_off(int N) { return AttnSmem::Q_OFF + 2 * N * 256; }
static_assert(kStages == 2 && p_off(32) + 2 * 32 * 128 <= AttnSmem::K_OFF, "narrow Q and P");

struct Bars {
  uint64_t *k_full, *k_empty, *v_full, *v_empty;     // [kStages]
  uint64_t *s_full, *p_full;                         // [2]
  uint64_t *o_done, *o_final;                        // [2] by the tile's parity; one phase per item
  uint64_t *q_full, *q_empty, *o_free;               // wide: one buffer each
  uint64_t *qn_full, *qn_empty, *on_free;            // narrow: by the Q or O buffer
  uint64_t* drained;                                 // [2] after an abort: S products, O products
  volatile int* aborted;
};
// The producer's loads by full barrier: how many phases it has begun there (parity) and whether any.
struct Sent {
  unsigned parity, any;
  KORE_DEV void add(int bar) {
    parity ^= 1u << bar;
    any |= 1u << bar;
  }
};
constexpr int kSentK = 0, kSentV = 2, kSentQ = 4, kSentQn = 5;

// ---- producer warp: Q of each item, K and V of each tile
template <int N>
KORE_DEV bool produce(const bool wide, const AttnParams& p, const Units& w, Walk r, uint8_t* smem, const Bars& bar, int& cnt, Sent& sent,
                      const CUtensorMap* tmQp, const CUtensorMap* tmQo, const CUtensorMap* tmK, const CUtensorMap* tmV) {
  using S = AttnSmem;
  constexpr int QB = 2;
  const int lane = threadIdx.x & 31, nbox = BK / p.box;
  Item it;
#pragma unroll 1
  for (int k = 0; next_item(w, r, it); ++k) {
    const bool pre = it.u < p.ngroups;
    const int tb = w.block_tokens(it.u), t0 = w.row0(it.u) + it.rb * tb;
    int klo, khi;
    w.keys(it.u, klo, khi);
    const int* bt = p.table + (pre ? (long)w.gs[it.u] : (long)(it.u - p.ngroups)) * p.ld_table;
    const int tile0 = klo / BK;
    auto slot_of = [&](int key) {               // the cache slot where the box at `key` begins
      const int page = (unsigned)key / (unsigned)p.page_size;
      return key + p.box > klo && key < khi ? (int)((unsigned)bt[page] * (unsigned)p.page_size + (unsigned)(key - page * p.page_size)) : 0;
    };
    int slot = slot_of((tile0 + it.j0) * BK + lane * p.box), window = 0;     // lane i: of the item's box window + i
    bool ok = true;
    if (lane == 0) {
      const int nq = wide ? 1 : QB, qi = wide ? 0 : k % QB, ph = wide ? k : k / QB;
      uint64_t* full = (wide ? bar.q_full : bar.qn_full) + qi;
      ok = !*bar.aborted && (k < nq || wait_on((wide ? bar.q_empty : bar.qn_empty) + qi, (ph - 1) & 1));
      if (ok) {
        const CUtensorMap* tm = pre ? tmQp : tmQo;
        uint8_t* q = smem + S::Q_OFF + qi * N * 256;
        mbar_arrive_expect_tx(full, 2 * 128 * p.G * tb);
        sent.add(wide ? kSentQ : kSentQn + qi);
        tma_load_3d(q, tm, full, 0, it.h * p.G, t0);
        tma_load_3d(q + (wide ? 16384 : N * 128), tm, full, 64, it.h * p.G, t0);
      }
    }
    int first = 0;                              // the tile's first box, from the item's first on
#pragma unroll 1
    for (int j = it.j0; j < it.j1; ++j, ++cnt, first += nbox) {
      const int st = cnt % kStages, key0 = (tile0 + j) * BK;
      const uint32_t ph = (cnt / kStages) & 1;
      if (first == window + 32) {               // 32 is a multiple of nbox: a tile's boxes lie in one window
        window = first;
        slot = slot_of(key0 + lane * p.box);
      }
      // boxes that hold keys of the unit; the others are not loaded
      const unsigned held = __ballot_sync(0xffffffff, key0 + lane * p.box < khi && key0 + (lane + 1) * p.box > klo && lane < nbox);
#pragma unroll 1
      for (int kv = 0; kv < 2; ++kv) {
        const CUtensorMap* tm = kv ? tmV : tmK;
        uint64_t* full = (kv ? bar.v_full : bar.k_full) + st;
        uint8_t* dst = smem + (kv ? S::V_OFF : S::K_OFF) + st * kTileBytes;
        if (lane == 0 && ok) {
          ok = wait_on((kv ? bar.v_empty : bar.k_empty) + st, ph ^ 1);
          if (ok) {
            mbar_arrive_expect_tx(full, __popc(held) * p.box * 256);
            sent.add((kv ? kSentV : kSentK) + st);
          }
        }
        if (nbox == 1) {                        // one box of 64 keys x two 64-column halves
          const int z = __shfl_sync(0xffffffff, slot, first - window);
          if (lane == 0 && ok) tma_load_4d(dst, tm, full, 0, z, 0, it.h);
        } else {
#pragma unroll 1
          for (int b = 0; b < nbox; ++b) {
            const int z = __shfl_sync(0xffffffff, slot, first - window + b);
            if (lane == 0 && ok && (held >> b & 1)) {
              tma_load_4d(dst + b * p.box * 128, tm, full, 0, z, 0, it.h);
              tma_load_4d(dst + 8192 + b * p.box * 128, tm, full, 0, z, 1, it.h);
            }
          }
        }
      }
      ok = __shfl_sync(0xffffffff, ok && !*bar.aborted, 0);
      if (!ok) return false;
    }
  }
  return true;
}

// ---- the products, one thread of a warp each for S and for O. A product of this size
// takes about 98 cycles in its chain (measured; 32 to 64 at full rate), and the issuing
// thread goes along with it: the eight products of an S and the four of an O, issued by
// one thread, were 1,100 of a tile's 2,200 cycles. From two threads they overlap.
constexpr uint64_t step16(int kk, int half) { return (uint64_t)(((kk >> 2) * half + (kk & 3) * 32) >> 4); }   // K-step kk of K-major atoms `half` bytes apart

template <bool WIDE, int N>
KORE_DEV bool multiply_s(const Units& w, Walk r, uint8_t* smem, const Bars& bar, uint32_t tmem, int& cnt) {
  using S = AttnSmem;
  constexpr uint32_t idesc = WIDE ? make_idesc_bf16(128, BK, false, false) : make_idesc_bf16(128, N, false, false);
  constexpr int QB = WIDE ? 1 : 2;
  const uint64_t q0 = make_sw128_desc(smem_u32(smem + S::Q_OFF), 16, 1024), k0 = make_sw128_desc(smem_u32(smem + S::K_OFF), 16, 1024);
  Item it;
#pragma unroll 1
  for (int k = 0; next_item(w, r, it); ++k) {
    const int qi = k % QB, last = cnt + it.j1 - it.j0 - 1;
    const uint64_t qd = q0 + (uint64_t)(qi * N * 16);
    if (!wait_on(WIDE ? bar.q_full : bar.qn_full + qi, (k / QB) & 1)) return false;
#pragma unroll 1
    for (; cnt <= last; ++cnt) {
      const int st = cnt & 1;
      if (!wait_on(&bar.k_full[st], (cnt >> 1) & 1)) return false;
      if (cnt >= 2 && !wait_on(&bar.o_done[st], ((cnt >> 1) - 1) & 1)) return false;   // this S buffer's last tile is through
      tc_fence_after();
      const uint64_t kd = k0 + (uint64_t)(st * (kTileBytes >> 4));
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        // narrow: K is the left operand; its rows 64..127 are whatever lies behind the 64 of the tile, and nobody reads their result
        if (WIDE) umma_f16_ss(tmem + st * 64, qd + step16(kk, 16384), kd + step16(kk, 8192), idesc, kk > 0);
        else umma_f16_ss(tmem + st * 64, kd + step16(kk, 8192), qd + step16(kk, N * 128), idesc, kk > 0);
      }
      umma_commit(&bar.k_empty[st]);
      umma_commit(&bar.s_full[st]);
    }
    if (!WIDE) umma_commit(bar.qn_empty + qi);
  }
  return true;
}

template <bool WIDE, int N>
KORE_DEV bool multiply_o(const Units& w, Walk r, uint8_t* smem, const Bars& bar, uint32_t tmem, int& cnt) {
  constexpr uint32_t idesc = WIDE ? make_idesc_bf16(128, D, false, true) : make_idesc_bf16(128, N, true, false);
  const uint64_t v0 = make_sw128_desc(smem_u32(smem + AttnSmem::V_OFF), 8192, 1024), p0 = make_sw128_desc(smem_u32(smem + p_off(N)), 16, 1024);
  Item it;
#pragma unroll 1
  for (int k = 0; next_item(w, r, it); ++k) {
    const int first = cnt, last = cnt + it.j1 - it.j0 - 1, ob = WIDE ? 1 : 2;
    const uint32_t to = tmem + kTmemO + (WIDE ? 0 : (k & 1) * 64);
    // the last item in this O has been read
    if (k >= ob && !wait_on(WIDE ? bar.o_free : bar.on_free + (k & 1), (WIDE ? k - 1 : (k >> 1) - 1) & 1)) return false;
#pragma unroll 1
    for (; cnt <= last; ++cnt) {
      const int st = cnt & 1;
      if (!wait_on(&bar.v_full[st], (cnt >> 1) & 1) || !wait_on(&bar.p_full[st], (cnt >> 1) & 1)) return false;
      tc_fence_after();
      const uint64_t vd = v0 + (uint64_t)(st * (kTileBytes >> 4)), pd = p0 + (uint64_t)(st * N * 8);
#pragma unroll
      for (int kk = 0; kk < BK / 16; ++kk) {
        if (WIDE) umma_f16_ts(to, tmem + st * 64 + kk * 8, vd + kk * 128, idesc, (cnt > first || kk > 0) ? 1u : 0u);
        else umma_f16_ss(to, vd + kk * 128, pd + step16(kk, 0), idesc, (cnt > first || kk > 0) ? 1u : 0u);
      }
      umma_commit(&bar.v_empty[st]);
      umma_commit(&bar.o_done[st]);
    }
    umma_commit(bar.o_final);
  }
  return true;
}

// What lies outside a unit's keys in the cache may be anything, NaN included, and
// 0 x NaN is not 0: those rows of a V tile are cleared before the product reads them.
KORE_DEV bool clear_v(uint8_t* smem, const Bars& bar, int cnt, int kv0, int klo, int khi) {
  const int lane = threadIdx.x & 31, vs = cnt % kStages, r = (threadIdx.x / 32 & 3) * 16 + (lane >> 1);
  if (!warp_wait(&bar.v_full[vs], (cnt / kStages) & 1)) return false;
  if (kv0 + r < klo || kv0 + r >= khi) {
    uint4* dst = reinterpret_cast<uint4*>(smem + AttnSmem::V_OFF + vs * kTileBytes + (lane & 1) * 8192 + r * 128);
#pragma unroll
    for (int i = 0; i < 8; ++i) dst[i] = make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async_smem();
  return true;
}

// ---- four warps, wide form: a thread owns a row
KORE_DEV bool softmax_wide(const AttnParams& p, const Units& w, Walk r, uint8_t* smem, const Bars& bar, uint32_t tmem, int& cnt, int& items, int run) {
  const int lane = threadIdx.x & 31, q4 = threadIdx.x / 32 & 3, row = q4 * 32 + lane;
  const uint32_t lane_base = (uint32_t)(q4 * 32) << 16;
  Item it;
  int tile = cnt;
#pragma unroll 1
  for (int k = 0; next_item(w, r, it); ++k) {
    const bool pre = it.u < p.ngroups;
    const int tb = w.block_tokens(it.u), rt = it.rb * tb + row / p.G;      // token within the unit
    const bool live = row < tb * p.G && rt < w.tokens(it.u);
    const bool warp_live = __any_sync(0xffffffff, live);
    const int t = w.row0(it.u) + rt, h = it.h * p.G + row % p.G;
    int klo, khi, limit = 0;                    // the row sees keys [klo, limit)
    w.keys(it.u, klo, khi);
    bool joined = pre;                          // another part of the row's keys is another unit's
    if (live) {
      const int b = pre ? w.seq_of(t, w.gs[it.u], w.gs[it.u + 1] - 1) : it.u - p.ngroups;
      if (!pre) joined = w.shared(b);
      limit = min(w.len[b] - (w.qs[b + 1] - t) + 1, khi);
    }
    const int tile0 = klo / BK;
    float m = -INFINITY, l = 0.f, sv[BK];
#pragma unroll 1
    for (int j = it.j0; j < it.j1; ++j, ++tile) {
      const int st = tile & 1, kv0 = (tile0 + j) * BK;
      if (!warp_wait(&bar.s_full[st], (tile >> 1) & 1)) return false;
      if ((kv0 < klo || kv0 + BK > khi) && !clear_v(smem, bar, tile, kv0, klo, khi)) return false;
      if (warp_live) {
        tc_fence_after();
        {
          uint32_t x[2][32];
          tmem_ld32(tmem + lane_base + st * 64, x[0]);
          tmem_ld32(tmem + lane_base + st * 64 + 32, x[1]);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < BK; ++i) sv[i] = __uint_as_float(x[i / 32][i % 32]);
        }
        if (kv0 + BK > limit || kv0 < klo) {
#pragma unroll
          for (int i = 0; i < BK; ++i)
            if (kv0 + i >= limit || kv0 + i < klo) sv[i] = -INFINITY;
        }
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < BK; i += 8) {
          mx4[0] = fmax3f(mx4[0], sv[i], sv[i + 1]);
          mx4[1] = fmax3f(mx4[1], sv[i + 2], sv[i + 3]);
          mx4[2] = fmax3f(mx4[2], sv[i + 4], sv[i + 5]);
          mx4[3] = fmax3f(mx4[3], sv[i + 6], sv[i + 7]);
        }
        const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * p.scale_log2;
        const float m_new = fmaxf(m, mx);
        // O follows the running maximum only when that grew by more than 2^8 (fp32 has the room)
        const bool need = m == -INFINITY || m_new > m + 8.f;
        if (j > it.j0) {
          const float alpha = need && m != -INFINITY ? exp2f(m - m_new) : 1.f;
          if (__any_sync(0xffffffff, need && m != -INFINITY)) {
            if (!warp_wait(&bar.o_done[(tile - 1) & 1], ((tile - 1) >> 1) & 1)) return false;
            tc_fence_after();
#pragma unroll
            for (int i4 = 0; i4 < 4; ++i4) {
              uint32_t x[32];
              const uint32_t a = tmem + lane_base + kTmemO + i4 * 32;
              tmem_ld32(a, x);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) * alpha);
              tmem_st32(a, x);
            }
            tmem_wait_st();
          }
          l *= alpha;
        }
        if (need) m = m_new;
        const float mref = m == -INFINITY ? 0.f : m;
        const uint64_t sc2 = f2_pack(p.scale_log2, p.scale_log2), nm2 = f2_pack(-mref, -mref);
        uint64_t rs2[2] = {f2_pack(0.f, 0.f), f2_pack(0.f, 0.f)};
#pragma unroll
        for (int i = 0; i < BK; i += 2) {
          float a, b;
          f2_unpack(f2_fma(f2_pack(sv[i], sv[i + 1]), sc2, nm2), a, b);
          sv[i] = exp2f(a);
          sv[i + 1] = exp2f(b);
          rs2[(i >> 1) & 1] = f2_add(rs2[(i >> 1) & 1], f2_pack(sv[i], sv[i + 1]));
        }
        float a0, b0, a1, b1;
        f2_unpack(rs2[0], a0, b0);
        f2_unpack(rs2[1], a1, b1);
        l += (a0 + b0) + (a1 + b1);
        // P in bf16 (the operand type of V): a probability is off by up to 2^-8 of itself, the sum l is not rounded
        uint32_t pk[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) pk[i] = pack_bf16(sv[2 * i], sv[2 * i + 1]);
        tmem_st32(tmem + lane_base + st * 64, pk);
        tmem_wait_st();
        tc_fence_before();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.p_full[st]);
    }
    if (!warp_wait(bar.o_final, items++ & 1)) return false;
    if (warp_live) {
      // Rows go out through this warp's 8 KB of the Q buffer, which the item needs no
      // more, 64 columns at a time (16-byte pieces swizzled by the row): a store
      // instruction then covers two whole row halves, not 16 bytes of 32 rows.
      tc_fence_after();
      const bool whole = it.j0 == 0 && it.j1 == it.n, direct = whole && !joined;
      const int at = t * p.Hq + h, dst = whole ? at : (2 * run + (it.j0 == 0 ? 1 : 0)) * 128 + row;
      float* const part = whole ? (pre ? p.whole_prefix : p.whole_own) : p.split_wide;
      const float inv = !direct ? 1.f : l == 0.f ? 0.f : 1.f / l;
      const unsigned rows = __ballot_sync(0xffffffff, live), joins = __ballot_sync(0xffffffff, !direct);
      uint8_t* const stage = smem + AttnSmem::Q_OFF + q4 * 8192;
#pragma unroll 1
      for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t x[32];
          tmem_ld32(tmem + lane_base + kTmemO + half * 64 + c * 32, x);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 8; ++i)
            *reinterpret_cast<float4*>(stage + lane * 256 + (((c * 8 + i) ^ (lane & 7)) << 4)) =
                make_float4(__uint_as_float(x[4 * i]) * inv, __uint_as_float(x[4 * i + 1]) * inv, __uint_as_float(x[4 * i + 2]) * inv,
                            __uint_as_float(x[4 * i + 3]) * inv);
        }
        __syncwarp();
#pragma unroll 4
        for (int i = 0; i < 16; ++i) {
          const int rr = 2 * i + (lane >> 4), c = lane & 15;
          const float4 v = *reinterpret_cast<const float4*>(stage + rr * 256 + ((c ^ (rr & 7)) << 4));
          const int to = __shfl_sync(0xffffffff, dst, rr);
          if (!(rows >> rr & 1)) continue;
          if (joins >> rr & 1)
            *reinterpret_cast<float4*>(part + (size_t)to * kPart + half * 64 + c * 4) = v;
          else
            *reinterpret_cast<uint2*>(p.out + (size_t)to * D + half * 64 + c * 4) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
        }
        __syncwarp();
      }
      if (live && direct && p.lse) p.lse[at] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
      if (live && !direct) *reinterpret_cast<float2*>(part + (size_t)dst * kPart + D) = make_float2(m, l);
      tc_fence_before();
      fence_proxy_async_smem();                 // the next Q is written by the TMA unit
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(bar.q_empty);
    if (lane == 0) mbar_arrive(bar.o_free);
  }
  cnt = tile;
  return true;
}

// ---- four warps, narrow form, NL >= the block's rows: threads of the first two own a
// key of S^T, all own a column of O^T. The rows' reference exponents are common to
// the keys and kept in shared memory; they move only when some score passes its row's
// by more than 2^8.
template <int NL>
KORE_DEV void tmem_ld(uint32_t taddr, float (&v)[NL]) {
  uint32_t x[NL];
  if constexpr (NL == 8) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]), "=r"(x[4]), "=r"(x[5]), "=r"(x[6]), "=r"(x[7]) : "r"(taddr));
  } else if constexpr (NL == 16) {
    tmem_ld16(taddr, x);
  } else {
#pragma unroll
    for (int i = 0; i < NL; i += 32) tmem_ld32(taddr + i, *reinterpret_cast<uint32_t(*)[32]>(&x[i]));
  }
  tmem_wait_ld();
#pragma unroll
  for (int i = 0; i < NL; ++i) v[i] = __uint_as_float(x[i]);
}
template <int NL>
KORE_DEV void tmem_st(uint32_t taddr, const float (&v)[NL]) {
  uint32_t x[NL];
#pragma unroll
  for (int i = 0; i < NL; ++i) x[i] = __float_as_uint(v[i]);
  if constexpr (NL == 8) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr),
                 "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(x[4]), "r"(x[5]), "r"(x[6]), "r"(x[7]));
  } else {
#pragma unroll
    for (int i = 0; i < NL; i += 16) tmem_st16(taddr + i, *reinterpret_cast<const uint32_t(*)[16]>(&x[i]));
  }
  tmem_wait_st();
}
// Sums of v[i] over the warp's lanes, by halving: a lane ends with that of column
// lane / (32 / NL), in v[0].
template <int NL>
KORE_DEV void warp_sums(float (&v)[NL]) {
  const int lane = threadIdx.x & 31;
  int n = NL;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    if (n > 1) {
      n >>= 1;
#pragma unroll
      for (int i = 0; i < NL / 2; ++i)
        if (i < n) {
          const float keep = lane & o ? v[i + n] : v[i], give = lane & o ? v[i] : v[i + n];
          v[i] = keep + __shfl_xor_sync(0xffffffff, give, o);
        }
    } else {
      v[0] += __shfl_xor_sync(0xffffffff, v[0], o);
    }
  }
}

struct NarrowSmem {               // per row of the block
  float ref[32], factor[32], mine[2][32];       // reference exponent; factor when it moves, later 1 / sum; the two key warps' values
  int limit[32], at[32];                        // the row sees keys [klo, limit); row of the result
};

template <int N, int NL>
KORE_DEV bool softmax_narrow(const AttnParams& p, const Units& w, Walk r, uint8_t* smem, const Bars& bar, uint32_t tmem, int& cnt, int& items, int run) {
  const int lane = threadIdx.x & 31, q4 = threadIdx.x / 32 & 3, tid = q4 * 32 + lane;
  const uint32_t lane_base = (uint32_t)(q4 * 32) << 16;
  NarrowSmem& x = *reinterpret_cast<NarrowSmem*>(smem + AttnSmem::X_OFF);
  // The four warps meet at named barriers, whose waits have no limit: one whose wait on an
  // mbarrier ran out goes through the rest of the run without waiting, so that all meet.
  bool ok = true;
  Item it;
  int tile = cnt;
#pragma unroll 1
  for (int k = 0; next_item(w, r, it); ++k) {
    const int b = it.u - p.ngroups, tb = p.tokens_own, rt0 = it.rb * tb, t0 = w.row0(it.u) + rt0;
    const int rows = min(tb, w.tokens(it.u) - rt0) * p.G;                  // live rows of the block
    int klo, khi;
    w.keys(it.u, klo, khi);
    const bool joined = w.shared(b);
    if (tid < NL) {
      const int i = tid / p.G;
      x.limit[tid] = tid < rows ? min(w.len[b] - (w.qs[b + 1] - t0 - i) + 1, khi) : -1;    // behind the block's rows Q is not defined
      x.at[tid] = (t0 + i) * p.Hq + it.h * p.G + tid % p.G;
    }
    softmax_sync();
    const int tile0 = klo / BK;
    const uint32_t to = tmem + lane_base + kTmemO + (k & 1) * 64;
    float l[NL];
#pragma unroll
    for (int i = 0; i < NL; ++i) l[i] = 0.f;
#pragma unroll 1
    for (int j = it.j0; j < it.j1; ++j, ++tile) {
      const int st = tile & 1, kv0 = (tile0 + j) * BK;
      ok = ok && warp_wait(&bar.s_full[st], (tile >> 1) & 1);
      if (kv0 < klo || kv0 + BK > khi) ok = ok && clear_v(smem, bar, tile, kv0, klo, khi);
      float s[NL];
      bool over = false;
      if (q4 < 2) {
        tc_fence_after();
        tmem_ld<NL>(tmem + lane_base + st * 64, s);
        const int key = kv0 + tid >= klo ? kv0 + tid : 0x7fffffff;
#pragma unroll
        for (int i = 0; i < NL; ++i) {
          s[i] = key < x.limit[i] ? s[i] * p.scale_log2 : -INFINITY;
          over = over || s[i] > x.ref[i] + 8.f;
        }
      }
      if (softmax_any(over || j == it.j0)) {
        if (q4 < 2) {
          float top = -INFINITY;
#pragma unroll
          for (int i = 0; i < NL; ++i) {
            const float v = warp_max(s[i]);
            if (lane == i) top = v;
          }
          if (lane < NL) x.mine[q4][lane] = top;
        }
        softmax_sync();
        if (tid < NL) {
          const float old = j == it.j0 ? -INFINITY : x.ref[tid], v = fmaxf(x.mine[0][tid], x.mine[1][tid]);
          const bool need = v > old + 8.f || old == -INFINITY;
          const float now = need ? fmaxf(v, old) : old;
          x.factor[tid] = need && old != -INFINITY ? exp2f(old - now) : 1.f;
          x.ref[tid] = now;
        }
        softmax_sync();
        if (j > it.j0) {
          ok = ok && warp_wait(&bar.o_done[(tile - 1) & 1], ((tile - 1) >> 1) & 1);
          tc_fence_after();
          constexpr int step = NL < 16 ? NL : 16;
#pragma unroll
          for (int i0 = 0; i0 < NL; i0 += step) {
            float o[step];
            tmem_ld<step>(to + i0, o);
#pragma unroll
            for (int i = 0; i < step; ++i) {
              l[i0 + i] *= x.factor[i0 + i];
              o[i] *= x.factor[i0 + i];
            }
            tmem_st<step>(to + i0, o);
          }
        }
      }
      if (q4 < 2) {
        // P^T as the right operand: row i of the block is 64 keys, 128 bytes, swizzled in 16-byte pieces by the row
        uint8_t* pt = smem + p_off(N) + st * N * 128 + (tid & 7) * 2;
#pragma unroll
        for (int i = 0; i < NL; ++i) {
          const float m = x.ref[i], e = exp2f(s[i] - (m == -INFINITY ? 0.f : m));
          l[i] += e;
          *reinterpret_cast<__nv_bfloat16*>(pt + i * 128 + (((tid >> 3) ^ (i & 7)) << 4)) = __float2bfloat16(e);
        }
        fence_proxy_async_smem();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.p_full[st]);
    }
    if (q4 < 2) {
      warp_sums<NL>(l);
      if (lane % (32 / NL) == 0) x.mine[q4][lane / (32 / NL)] = l[0];
    }
    ok = ok && warp_wait(bar.o_final, items++ & 1);
    tc_fence_after();
    float o[NL];
    tmem_ld<NL>(to, o);
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar.on_free + (k & 1));
    softmax_sync();                             // `mine` is there
    const bool whole = it.j0 == 0 && it.j1 == it.n, direct = whole && !joined;
    float* split = p.split_narrow + (size_t)(2 * run + (it.j0 == 0 ? 1 : 0)) * 32 * kPart;
    if (tid < rows) {
      const float sum = x.mine[0][tid] + x.mine[1][tid], m = x.ref[tid];
      if (direct) {
        if (p.lse) p.lse[x.at[tid]] = sum == 0.f ? -INFINITY : (m + log2f(sum)) * kLn2;
        x.factor[tid] = sum == 0.f ? 0.f : 1.f / sum;
      } else {
        float* part = whole ? p.whole_own + (size_t)x.at[tid] * kPart : split + tid * kPart;
        part[D] = m;
        part[D + 1] = sum;
      }
    }
    softmax_sync();
    if (direct) {
#pragma unroll
      for (int i = 0; i < NL; ++i)
        if (i < rows) p.out[(size_t)x.at[i] * D + tid] = __float2bfloat16(x.factor[i] == 0.f ? 0.f : o[i] * x.factor[i]);
    } else {
      float* part = (whole ? p.whole_own : split) + tid;
#pragma unroll
      for (int i = 0; i < NL; ++i)
        if (i < rows) part[(size_t)(whole ? x.at[i] : i) * kPart] = o[i];
    }
    softmax_sync();                             // the rows' values have been read
  }
  cnt = tile;
  return ok;
}

template <int NL>
__global__ void __launch_bounds__(kAttnThreads, 2)
    attn_kernel(const __grid_constant__ CUtensorMap tmQp, const __grid_constant__ CUtensorMap tmQo,
                const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ AttnParams p) {
  using S = AttnSmem;
  constexpr int N = NL < 16 ? 16 : NL;           // the narrow products' width: rows in multiples of 16
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::BAR_OFF);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 24);
  int* warp_sum = reinterpret_cast<int*>(tmem_slot + 2);             // [8]
  const Bars bar = {bars, bars + 2, bars + 4, bars + 6, bars + 8, bars + 10, bars + 12, bars + 14, bars + 15,
                    bars + 16, bars + 17, bars + 18, bars + 20, bars + 22, bars + 29, reinterpret_cast<volatile int*>(tmem_slot + 1)};
  static_assert(kStages == 2 && 31 * 8 <= S::X_OFF - S::BAR_OFF, "barrier layout: 24, the two words and eight sums, 2");
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  const Units w(p, smem + S::UNITS_OFF);
  int* const cum = w.cum;

  pdl_trigger();
  // ---- the units' tiles, summed
  {
    constexpr int R = (kMaxSeqs + kAttnThreads) / kAttnThreads;      // all loads in flight together
    int q[R], n[R], g[R], x[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int i = threadIdx.x + r * kAttnThreads;
      q[r] = i <= p.B ? p.q_start[i] : 0;
      n[r] = i < p.B ? p.lens[i] : 0;
      g[r] = p.ngroups && i <= p.ngroups ? p.group_start[i] : 0;
      x[r] = i < p.ngroups ? p.prefix[i] : 0;
    }
    const int cap = p.M * p.page_size;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int i = threadIdx.x + r * kAttnThreads;
      if (i <= p.B) w.qs[i] = min(max(q[r], 0), p.T);
      if (i < p.B) w.len[i] = min(max(n[r], 0), cap);
      if (i <= p.ngroups) w.gs[i] = min(max(g[r], 0), p.B);
      if (i < p.ngroups) w.prefix[i] = min(max(x[r], 0), cap);
    }
  }
  if (threadIdx.x == 0) {
#pragma unroll 1
    for (int i = 0; i < 24; ++i)     // p_full, wide q_empty, o_free, on_free: a lane of each softmax warp
      mbar_init(bars + i, i == 10 || i == 11 || i == 16 || i == 17 || i >= 22 ? 4 : 1);
    mbar_init(bar.drained, 1);
    mbar_init(bar.drained + 1, 1);
    *bar.aborted = 0;
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc(tmem_slot, kTmemCols);
  __syncthreads();
  const int nu = p.ngroups + p.B, per = (nu + kAttnThreads - 1) / kAttnThreads;
#pragma unroll 1
  for (int b = threadIdx.x; b < p.B; b += kAttnThreads) {
    int lo = 0, hi = p.ngroups;      // the first group that starts behind b
#pragma unroll 1
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (w.gs[mid] <= b) lo = mid + 1; else hi = mid;
    }
    w.grp[b] = (short)(lo > 0 && b < w.gs[lo] ? lo - 1 : -1);
  }
  // Starts that decrease would give rows or sequences to several units, whose tiles are more
  // than the host allowed for: such a call has no tiles (its rows get zeros) and sets the error word.
  bool falls = false;
#pragma unroll 1
  for (int i = threadIdx.x; i < p.B; i += kAttnThreads) falls = falls || w.qs[i] > w.qs[i + 1] || (i < p.ngroups && w.gs[i] > w.gs[i + 1]);
  const bool refused = __syncthreads_or(falls);
  if (refused && blockIdx.x == 0 && threadIdx.x == 0) atomicExch(&g_error, 3);
  {
    const int u0 = min((int)threadIdx.x * per, nu), u1 = min(u0 + per, nu);
    int mine = 0;
#pragma unroll 1
    for (int u = u0; u < u1; ++u) {
      cum[u] = mine;
      mine += refused ? 0 : w.tiles(u);
    }
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffff, upto, o);
      if (lane >= o) upto += y;
    }
    if (lane == 31) warp_sum[warp] = upto;
    __syncthreads();
    int at = upto - mine;
#pragma unroll 1
    for (int i = 0; i < warp; ++i) at += warp_sum[i];
#pragma unroll 1
    for (int u = u0; u < u1; ++u) cum[u] += at;
    if (u1 == nu) cum[nu] = at + mine;      // the same from every thread that ends there
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const int Ww = cum[p.nwide];
  const Runs wides(Ww, gridDim.x), narrows(cum[nu] - Ww, gridDim.x);
  const uint32_t tmem = *tmem_slot;
  const int cw = blockIdx.x, cn = gridDim.x - 1 - blockIdx.x;       // few runs of both forms land on different blocks
  const Walk wide = make_walk(cum, nu, 0, wides, cw), narrow = make_walk(cum, nu, Ww, narrows, cn);
  // The end of a turn: both forms use the same buffers. True: give up, once `drain` has seen
  // to what the warp has in flight.
  auto turned = [&](bool ok, auto drain) {
    if (!ok) *bar.aborted = 1;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const bool stop = *bar.aborted;
    if (stop) drain();
    __syncthreads();
    return stop;
  };
  int cnt = 0;                     // tiles so far, in both turns
  // 56 and 200 registers for four warps each: together the 256 x 128 of the launch (the
  // host checks that it has these: an increase beyond them would wait for good).
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    const bool lead = elect_one();
    Sent sent = {0, 0};
    auto drain = [&] {               // waits, up to their limit, for this thread's loads or products
      if (warp == 0 && lane == 0) {
        uint64_t* const full[7] = {bar.k_full, bar.k_full + 1, bar.v_full, bar.v_full + 1, bar.q_full, bar.qn_full, bar.qn_full + 1};
#pragma unroll
        for (int i = 0; i < 7; ++i)
          if (sent.any >> i & 1) mbar_wait(full[i], (sent.parity >> i & 1) ^ 1);
      } else if ((warp == 1 || warp == 2) && lead) {
        umma_commit(bar.drained + (warp - 1));
        mbar_wait(bar.drained + (warp - 1), 0);
      }
    };
    if (warp == 3) {
      // ---- for the join: first tile (of head 0) of the token's prefix and own items, tiles of an item, tiles to the next head, row in the block
      const int id = blockIdx.x * 32 + lane;
      if (id == 0) *reinterpret_cast<int2*>(p.runs) = make_int2(Ww, narrows.W);
#pragma unroll 1
      for (int i = 2 * w.qs[0] + id; i < 2 * w.qs[p.B]; i += gridDim.x * 32) {
        const int t = i >> 1, b = w.seq_of(t, 0, p.B - 1), u = i & 1 ? p.ngroups + b : w.grp[b];
        int4 e = make_int4(0, 0, 0, 0);
        if (u >= 0 && cum[u + 1] > cum[u]) {
          const int tb = w.block_tokens(u), d = t - w.row0(u), rb = d / tb;
          e.y = w.item_tiles(u);
          e.x = cum[u] - (u < p.nwide ? 0 : Ww) + rb * e.y;
          e.z = w.blocks(u) * e.y;
          e.w = (d - rb * tb) * p.G;
        }
        p.where[i] = e;
      }
    }
#pragma unroll 1
    for (int turn = 0; turn < 2; ++turn) {
      const bool is_wide = turn == 1;
      bool ok = true;
      if (warp == 0) {
        ok = produce<N>(is_wide, p, w, is_wide ? wide : narrow, smem, bar, cnt, sent, &tmQp, &tmQo, &tmK, &tmV);
      } else if (warp == 1) {
        if (lead) ok = is_wide ? multiply_s<true, N>(w, wide, smem, bar, tmem, cnt) : multiply_s<false, N>(w, narrow, smem, bar, tmem, cnt);
      } else if (warp == 2) {
        if (lead) ok = is_wide ? multiply_o<true, N>(w, wide, smem, bar, tmem, cnt) : multiply_o<false, N>(w, narrow, smem, bar, tmem, cnt);
      }
      __syncwarp();
      if (turned(ok, drain)) break;
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    int items = 0;                 // items so far
#pragma unroll 1
    for (int turn = 0; turn < 2; ++turn) {
      const bool is_wide = turn == 1;
      const bool ok = is_wide ? softmax_wide(p, w, wide, smem, bar, tmem, cnt, items, cw) : softmax_narrow<N, NL>(p, w, narrow, smem, bar, tmem, cnt, items, cn);
      if (turned(ok, [] {})) break;
    }
  }
  if (warp == 1) tmem_dealloc(tmem, kTmemCols);
}

// Joins the partials of a (token, head), WPR warps for each: their every WPR-th part, four
// at a time. Parts are the prefix's and the own keys' runs, in the order of their tiles.
template <int WPR>
__global__ void __launch_bounds__(128) join_kernel(AttnParams p, int grid) {
  pdl_wait();
  __shared__ float4 acc[4][32];
  __shared__ float2 ml[4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32, sub = warp % WPR;
  const int at = blockIdx.x * (4 / WPR) + warp / WPR, t = at / p.Hq, h = at - t * p.Hq;
  if (t >= p.T) return;                              // whole warps, and whole blocks where they meet
  const int2 tiles = *reinterpret_cast<const int2*>(p.runs);
  const int4 e0 = p.where[2 * t], e1 = p.where[2 * t + 1];
  if (t < p.q_start[0] || t >= p.q_start[p.B]) return;       // a row of no sequence: it has no entry, and its result stays
  const bool own_wide = p.nwide > p.ngroups;
  const int kvh = h / p.G, g = h - kvh * p.G;
  int first0 = 0, first1 = 0, n0 = 0, n1 = 0;
  const Runs wides(tiles.x, grid), narrows(tiles.y, grid);
  if (e0.y) {
    const int x = e0.x + kvh * e0.z;
    first0 = wides.of(x);
    n0 = wides.of(x + e0.y - 1) - first0 + 1;
  }
  if (e1.y) {
    const Runs& r = own_wide ? wides : narrows;
    const int x = e1.x + kvh * e1.z;
    first1 = r.of(x);
    n1 = r.of(x + e1.y - 1) - first1 + 1;
  }
  if (n0 == 0 && n1 == 1) return;                    // written by the block that had it all
  auto part = [&](int j) -> const float* {           // part j of n0 + n1
    const bool own = j >= n0;
    j -= own ? n0 : 0;
    if ((own ? n1 : n0) == 1) return (own ? p.whole_own : p.whole_prefix) + (size_t)at * kPart;
    const size_t slot = 2 * ((own ? first1 : first0) + j) + (j == 0 ? 1 : 0);
    return own && !own_wide ? p.split_narrow + (slot * 32 + e1.w + g) * kPart
                            : p.split_wide + (slot * 128 + (own ? e1.w : e0.w) + g) * kPart;
  };
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](float mj, float lj, float4 v) {
    if (mj == -INFINITY) return;                     // no key of this part was visible
    const float now = fmaxf(m, mj), a = exp2f(m - now), b = exp2f(mj - now);     // m = -inf: a = 0
    l = l * a + lj * b;
    o.x = o.x * a + v.x * b; o.y = o.y * a + v.y * b; o.z = o.z * a + v.z * b; o.w = o.w * a + v.w * b;
    m = now;
  };
#pragma unroll 1
  for (int j = sub; j < n0 + n1; j += 4 * WPR) {
    float2 s[4];
    float4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[i] = make_float2(-INFINITY, 0.f);
      if (j + WPR * i < n0 + n1) {
        const float* r = part(j + WPR * i);
        s[i] = *reinterpret_cast<const float2*>(r + D);
        v[i] = *reinterpret_cast<const float4*>(r + lane * 4);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) add(s[i].x, s[i].y, v[i]);
  }
  if constexpr (WPR > 1) {
    acc[warp][lane] = o;
    if (lane == 0) ml[warp] = make_float2(m, l);
    __syncthreads();
    if (sub) return;
    for (int i = 1; i < WPR; ++i) add(ml[i].x, ml[i].y, acc[i][lane]);
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  *reinterpret_cast<uint2*>(p.out + (size_t)at * D + lane * 4) = make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
  if (p.lse && lane == 0) p.lse[at] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

// A cache as [64 columns, slots, 2 halves, heads]: a box of 64 keys holds both halves of a
// head, one of fewer keys (small pages) a half of it.
CUtensorMap cache_map(const at::Tensor& c, int box) {
  CUtensorMap m;
  const cuuint64_t dims[4] = {64, (cuuint64_t)c.size(0), 2, (cuuint64_t)c.size(1)};
  const cuuint64_t strides[3] = {(cuuint64_t)c.stride(0) * 2, 128, (cuuint64_t)c.stride(1) * 2};
  const cuuint32_t b[4] = {64, (cuuint32_t)box, box == BK ? 2u : 1u, 1}, unit[4] = {1, 1, 1, 1};
  const CUresult r = get_encode_tiled()(&m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, c.data_ptr(), dims, strides, b, unit,
                                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(r == CUDA_SUCCESS, "prefix_attention: the cache's strides cannot be described to the TMA unit (code ", std::to_string((int)r), ")");
  return m;
}

void check_ints(const at::Tensor& t, const at::Tensor& like, int64_t n, const char* name) {
  TORCH_CHECK(t.device() == like.device() && t.scalar_type() == at::kInt && t.dim() == 1 && t.is_contiguous() &&
                  (n < 0 || t.numel() == n),
              "paged: ", name, " must be a contiguous int32 vector", n < 0 ? std::string() : " of " + std::to_string(n),
              " on the other arguments' device");
}

void check_table(const at::Tensor& table, const at::Tensor& like, int64_t B, int64_t page_size) {
  TORCH_CHECK(table.device() == like.device() && table.scalar_type() == at::kInt && table.dim() == 2 &&
                  table.size(0) == B && (table.size(1) <= 1 || table.stride(1) == 1),
              "paged: table must be int32 [sequences, pages] with contiguous rows");
  TORCH_CHECK(page_size > 0 && page_size <= 1 << 20, "paged: page_size out of range");
  TORCH_CHECK(table.size(1) * page_size <= 0x7fffffff, "paged: a table row spans more than 2^31 positions");
}

}  // namespace paged

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, c10::optional<at::Tensor>>
paged_plan(const at::Tensor& ctx, const at::Tensor& new_toks, at::Tensor& table, int64_t page_size, int64_t rows,
           const c10::optional<at::Tensor>& held, const c10::optional<at::Tensor>& free_stack,
           const c10::optional<at::Tensor>& free_count) {
  using namespace paged;
  TORCH_CHECK(ctx.is_cuda(), "paged: expected CUDA tensors");
  const int64_t B = ctx.numel();
  check_ints(ctx, ctx, B, "ctx");
  check_ints(new_toks, ctx, B, "new");
  check_table(table, ctx, B, page_size);
  TORCH_CHECK(rows >= 0 && rows <= 0x7fffffff && B < (int64_t)1 << 31, "paged: rows out of range");
  if (held) check_ints(*held, ctx, B, "held");
  TORCH_CHECK(free_stack.has_value() == free_count.has_value(), "paged: give free and free_count, or neither");
  if (free_stack) {
    check_ints(*free_stack, ctx, -1, "free");
    check_ints(*free_count, ctx, 1, "free_count");
    TORCH_CHECK(B <= 1 || table.stride(0) >= table.size(1), "paged: rows of a table that pages are written to must not overlap");
  }
  c10::cuda::CUDAGuard g(ctx.device());
  const auto i32 = ctx.options();
  at::Tensor q_start = at::empty({B + 1}, i32), lens = at::empty({B}, i32), pos = at::empty({rows}, i32),
             slots = at::empty({rows}, i32), ok = at::empty({B}, i32.dtype(at::kBool)), held_out = at::empty({B}, i32);
  c10::optional<at::Tensor> count_out;
  if (free_count) count_out = at::empty({1}, i32);
  PlanParams p;
  p.ctx = ctx.data_ptr<int>();
  p.new_toks = new_toks.data_ptr<int>();
  p.held = held ? held->data_ptr<int>() : nullptr;
  p.table = table.data_ptr<int>();
  p.ld_table = table.stride(0);
  p.M = (int)table.size(1);
  p.page_size = (int)page_size;
  p.B = B;
  p.rows = rows;
  p.free_stack = free_stack ? free_stack->data_ptr<int>() : nullptr;
  p.free_count = free_count ? free_count->data_ptr<int>() : nullptr;
  p.nfree = free_stack ? free_stack->numel() : 0;
  p.q_start = q_start.data_ptr<int>();
  p.lens = lens.data_ptr<int>();
  p.pos = pos.data_ptr<int>();
  p.slots = slots.data_ptr<int>();
  p.held_out = held_out.data_ptr<int>();
  p.count_out = count_out ? count_out->data_ptr<int>() : nullptr;
  p.ok = ok.data_ptr<bool>();
  auto st = at::cuda::getCurrentCUDAStream();
  const bool map_rows = B <= kPlanThreads && rows <= kPlanRows;
  plan_kernel<<<1, kPlanThreads, 0, st>>>(p, map_rows);
  check_cuda(cudaGetLastError(), "paged_plan");
  if (!map_rows && rows > 0) launch_after("paged_plan rows", plan_rows_kernel, dim3((unsigned)((rows + 1023) / 1024)), dim3(256), 0, st, p);
  return {q_start, lens, pos, slots, ok, held_out, count_out};
}

void paged_prefix_attention(const at::Tensor& q, const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& table,
                            const at::Tensor& lens, const at::Tensor& q_start, int64_t page_size, int64_t max_q,
                            double scale, const c10::optional<at::Tensor>& group_start,
                            const c10::optional<at::Tensor>& prefix_len, at::Tensor& out,
                            const c10::optional<at::Tensor>& lse) {
  using namespace paged;
  TORCH_CHECK(q.is_cuda() && q.scalar_type() == at::kBFloat16 && q.dim() == 3 && q.size(2) == D && q.stride(2) == 1 &&
                  (q.size(1) <= 1 || q.stride(1) == D) && q.stride(0) % 8 == 0 && (uintptr_t)q.data_ptr() % 16 == 0,
              "prefix_attention: q must be bf16 [T, Hq, 128] with contiguous heads and 16-byte aligned rows");
  for (const at::Tensor* c : {&kc, &vc})
    TORCH_CHECK(c->device() == q.device() && c->scalar_type() == at::kBFloat16 && c->dim() == 3 && c->size(2) == D &&
                    c->stride(2) == 1 && c->stride(1) % 8 == 0 && c->stride(0) % 8 == 0 &&
                    (uintptr_t)c->data_ptr() % 16 == 0 && c->sizes() == kc.sizes(),
                "prefix_attention: caches must be bf16 [slots, Hkv, 128] with 16-byte aligned heads, of one shape");
  const int64_t T = q.size(0), Hq = q.size(1), Hkv = kc.size(1), B = lens.numel();
  TORCH_CHECK(Hkv > 0 && Hq % Hkv == 0 && Hq / Hkv <= 128, "prefix_attention: Hq must be a multiple (up to 128) of Hkv");
  static_assert(kMaxSeqs == 512, "the message below");
  TORCH_CHECK(B <= kMaxSeqs, "prefix_attention: at most 512 sequences a call");
  TORCH_CHECK(page_size % 8 == 0, "prefix_attention: page_size must be a multiple of 8");
  TORCH_CHECK(max_q >= 1, "prefix_attention: max_q must be positive");
  check_ints(lens, q, B, "lens");
  check_ints(q_start, q, B + 1, "q_start");
  check_table(table, q, B, page_size);
  TORCH_CHECK(group_start.has_value() == prefix_len.has_value(), "prefix_attention: give group_start and prefix_len, or neither");
  if (group_start) {
    check_ints(*prefix_len, q, -1, "prefix_len");
    check_ints(*group_start, q, prefix_len->numel() + 1, "group_start");
    TORCH_CHECK(prefix_len->numel() <= B, "prefix_attention: more groups than sequences");
  }
  TORCH_CHECK(out.device() == q.device() && out.scalar_type() == at::kBFloat16 && out.is_contiguous() && out.sizes() == q.sizes(),
              "prefix_attention: out must be contiguous bf16 of q's shape");
  if (lse)
    TORCH_CHECK(lse->device() == q.device() && lse->scalar_type() == at::kFloat && lse->is_contiguous() &&
                    lse->dim() == 2 && lse->size(0) == T && lse->size(1) == Hq,
                "prefix_attention: lse must be contiguous fp32 [T, Hq]");
  // a factor that underflows makes NaN of a masked score
  const float scale_log2 = (float)(scale * 1.4426950408889634);
  TORCH_CHECK(scale_log2 > 0 && std::isnormal(scale_log2), "prefix_attention: scale must be a positive normal fp32 number");
  if (T == 0 || B == 0 || Hq == 0) return;
  // Blocks read q while others write results.
  const uintptr_t q0 = (uintptr_t)q.data_ptr(), q1 = q0 + 2 * ((T - 1) * q.stride(0) + Hq * D), o0 = (uintptr_t)out.data_ptr();
  TORCH_CHECK(o0 + 2 * T * Hq * D <= q0 || o0 >= q1, "prefix_attention: out must not overlap q");
  c10::cuda::CUDAGuard g(q.device());
  const int G = (int)(Hq / Hkv), ngroups = prefix_len ? (int)prefix_len->numel() : 0;
  AttnParams p;
  p.table = table.data_ptr<int>();
  p.lens = lens.data_ptr<int>();
  p.q_start = q_start.data_ptr<int>();
  p.ld_table = table.stride(0);
  p.M = (int)table.size(1);
  p.page_size = (int)page_size;
  p.B = (int)B;
  p.T = (int)T;
  p.Hq = (int)Hq;
  p.Hkv = (int)Hkv;
  p.G = G;
  p.tokens_prefix = 128 / G;
  // The narrow form up to 32 rows of a sequence; what max_q leaves out is further row blocks.
  const bool narrow = max_q * G <= 32;
  p.tokens_own = (int)std::min<int64_t>(128 / G, max_q);
  p.nwide = narrow ? ngroups : ngroups + (int)B;
  p.box = (int)std::gcd<int64_t, int64_t>(page_size, BK);
  p.group_start = group_start ? group_start->data_ptr<int>() : nullptr;
  p.prefix = prefix_len ? prefix_len->data_ptr<int>() : nullptr;
  p.ngroups = ngroups;
  p.scale_log2 = scale_log2;
  p.out = (__nv_bfloat16*)out.data_ptr();
  p.lse = lse ? lse->data_ptr<float>() : nullptr;
  const int64_t tiles = (table.size(1) * page_size + BK - 1) / BK + 1;
  TORCH_CHECK(T * Hq < (int64_t)1 << 31, "prefix_attention: too many rows");
  TORCH_CHECK(tiles * Hkv * (T / p.tokens_prefix + ngroups + T / p.tokens_own + B) < (int64_t)1 << 30,
              "prefix_attention: rows x table length out of range");
  const int grid = 2 * num_sms(q.get_device());
  const int64_t rows = ngroups ? T * Hq * kPart : 0, wide = (int64_t)2 * grid * 128 * kPart, thin = wide / 4;
  at::Tensor ws = at::empty({8 * T + 4 + 2 * rows + wide + thin}, q.options().dtype(at::kFloat));
  p.where = reinterpret_cast<int4*>(ws.data_ptr<float>());
  p.runs = reinterpret_cast<int*>(p.where + 2 * T);
  p.whole_prefix = reinterpret_cast<float*>(p.runs + 4);
  p.whole_own = p.whole_prefix + rows;
  p.split_wide = p.whole_own + rows;
  p.split_narrow = p.split_wide + wide;
  const auto bf = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const CUtensorMap tq = make_tmap_3d(q.data_ptr(), bf, 2, D, Hq, T, D, q.stride(0), 64, G, p.tokens_prefix);
  const CUtensorMap to = make_tmap_3d(q.data_ptr(), bf, 2, D, Hq, T, D, q.stride(0), 64, G, p.tokens_own);
  const CUtensorMap tk = cache_map(kc, p.box), tv = cache_map(vc, p.box);
  const int form = !narrow || p.tokens_own * G <= 8 ? 0 : p.tokens_own * G <= 16 ? 1 : 2;
  void (*const kernels[])(CUtensorMap, CUtensorMap, CUtensorMap, CUtensorMap, AttnParams) = {attn_kernel<8>, attn_kernel<16>, attn_kernel<32>};
  static bool attr[64][3] = {};
  const int dev = q.get_device();
  if (!attr[dev][form]) {
    cudaFuncAttributes fa;
    check_cuda(cudaFuncGetAttributes(&fa, kernels[form]), "prefix_attention attributes");
    TORCH_CHECK(fa.numRegs == 128, "prefix_attention: built with another register count than its warps share out");
    check_cuda(cudaFuncSetAttribute(kernels[form], cudaFuncAttributeMaxDynamicSharedMemorySize, AttnSmem::TOTAL), "prefix_attention smem");
    attr[dev][form] = true;
  }
  auto st = at::cuda::getCurrentCUDAStream();
  kernels[form]<<<grid, kAttnThreads, AttnSmem::TOTAL, st>>>(tq, to, tk, tv, p);
  check_cuda(cudaGetLastError(), "prefix_attention");
  // A row to a warp when the rows fill the SMs by themselves (64 warps each), else to four:
  // few rows may have their parts on all blocks.
  const int64_t all = T * Hq;
  if (all >= 32 * grid)
    launch_after("prefix_attention join", join_kernel<1>, dim3((unsigned)((all + 3) / 4)), dim3(128), 0, st, p, grid);
  else
    launch_after("prefix_attention join", join_kernel<4>, dim3((unsigned)all), dim3(128), 0, st, p, grid);
}

}  // namespace kore
