// The paged KV cache's step plan and its attention for batches with shared
// prefixes, for sm_100a:
//   * plan:             request lengths -> row starts, positions, slot map; pages
//                       popped from a free stack into the block tables
//   * prefix_attention: causal GQA attention of each sequence's newest tokens over
//                       its paged history; the keys that a group of sequences
//                       shares are read and scored once for all their rows
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <algorithm>
#include <numeric>
#include <tuple>

#include "common.cuh"
#include "tma_host.h"

namespace kore {
namespace paged {

// ------------------------------------------------------------------- plan
struct PlanParams {
  const int *ctx, *new_toks, *held;     // held may be null: the pages that ctx tokens fill
  int* table;
  long ld_table;
  int M, page_size;
  long B, rows;
  const int *free_stack, *free_count;   // null: no pool
  long nfree;
  int *q_start, *lens, *pos, *slots, *held_out, *count_out;
  bool* ok;
};

constexpr int kPlanThreads = 1024;

// Inclusive sum over the block; `total` is the sum of all.
KORE_DEV long block_scan(long v, long* part, long& total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long y = __shfl_up_sync(0xffffffff, v, o);
    if (lane >= o) v += y;
  }
  __syncthreads();
  if (lane == 31) part[w] = v;
  __syncthreads();
  long before = 0;
  total = 0;
  for (int i = 0; i < kPlanThreads / 32; ++i) {
    if (i < w) before += part[i];
    total += part[i];
  }
  return v + before;
}

KORE_DEV void plan_row(const PlanParams& p, long t) {
  long lo = 0, hi = p.B;                // the sequence with q_start[b] <= t < q_start[b + 1]
  while (lo < hi) {
    const long mid = (lo + hi) >> 1;
    if (p.q_start[mid + 1] <= t) lo = mid + 1; else hi = mid;
  }
  if (lo == p.B) {                      // behind the last sequence
    p.pos[t] = 0;
    p.slots[t] = -1;
    return;
  }
  const int pos = max(p.ctx[lo], 0) + (int)(t - p.q_start[lo]);
  p.pos[t] = pos;
  long slot = -1;
  if (p.ok[lo]) {
    const int page = p.table[lo * p.ld_table + pos / p.page_size];
    slot = (long)page * p.page_size + pos % p.page_size;
    if (page < 0 || slot > 0x7fffffffL) slot = -1;
  }
  p.slots[t] = (int)slot;
}

// One block: rows' starts and granted pages are running sums over the sequences.
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(PlanParams p) {
  __shared__ long part[kPlanThreads / 32];
  const long count = p.free_stack ? min((long)max(*p.free_count, 0), p.nfree) : 0;
  long rows = 0, asked = 0, granted = 0, total;
  if (threadIdx.x == 0) p.q_start[0] = 0;
  for (long b0 = 0; b0 < p.B; b0 += kPlanThreads) {
    const long b = b0 + threadIdx.x;
    const bool in = b < p.B;
    const long want = in ? max(p.new_toks[b], 0) : 0;
    const long to = block_scan(want, part, total) + rows;
    rows += total;
    const long n = min(to, p.rows) - min(to - want, p.rows);   // a batch has p.rows rows: what is behind them is cut
    const long ctx = in ? max(p.ctx[b], 0) : 0;
    const long full = (ctx + p.page_size - 1) / p.page_size, need = (ctx + n + p.page_size - 1) / p.page_size;
    const long held = in && p.held ? min(max(p.held[b], 0), p.M) : full;
    const bool fits = need <= p.M;
    const long take = p.free_stack && fits ? max(need - held, 0L) : 0;
    const long upto = block_scan(take, part, total) + asked;
    asked += total;
    const bool ok = fits && (!p.free_stack || upto <= count);
    const long got = ok ? take : 0;
    block_scan(got, part, total);
    granted += total;
    if (!in) continue;
    for (long j = 0; j < got; ++j)
      p.table[b * p.ld_table + held + j] = p.free_stack[count - 1 - (upto - take) - j];
    p.q_start[b + 1] = (int)min(to, p.rows);
    p.lens[b] = (int)(ok ? ctx + n : ctx);
    p.ok[b] = ok;
    if (p.held_out) p.held_out[b] = (int)(held + got);
  }
  if (threadIdx.x == 0 && p.count_out) *p.count_out = (int)(count - granted);
}

__global__ void plan_rows_kernel(PlanParams p) {
  const long t = (long)blockIdx.x * blockDim.x + threadIdx.x;
  if (t < p.rows) plan_row(p, t);
}

// -------------------------------------------------------- prefix attention
// A unit of work is the prefix of a group (all query rows of its sequences against
// the shared keys) or a sequence's own keys (its rows against what follows the
// prefix). A unit is cut into items, one for each kv head and each block of at most
// 128 rows (row = token x query head of the kv head), and an item into tiles of 64
// keys. All tiles of a call, in one order, are dealt to the blocks in equal runs, so
// that a long prefix is split over as many blocks as it needs and no host value
// depends on the lengths. A block that has an item's every tile and no other part to
// join it with writes the result; all else goes to fp32 partials (running maximum,
// sum and unnormalised output), which a second kernel joins in a fixed order:
//   m = max m_i, l = sum l_i 2^(m_i - m), o = sum o_i 2^(m_i - m) / l.
constexpr int D = 128;
constexpr int BK = 64;                            // keys of a tile
constexpr int kStages = 2;
constexpr int kTileBytes = BK * D * 2;            // 16 KB: 64 keys as two 8 KB swizzle atoms
constexpr int kQBytes = 128 * D * 2;
constexpr int kAttnThreads = 192;                 // producer, MMA, four softmax warps
constexpr int kTmemCols = 256;                    // two S / P buffers of 64 columns, O of 128
constexpr int kMaxSeqs = 1024;
constexpr int kMinTiles = 4;                      // of a block: fewer cost more in partials than they save
constexpr float kLn2 = 0.6931471805599453f;

struct AttnParams {
  const int *table, *lens, *q_start;
  long ld_table;
  int M, page_size, B, T, Hq, Hkv, G;
  int tokens_prefix, tokens_own;                  // tokens of a row block, for a group's prefix and a sequence's own keys
  int box;                                        // keys of one TMA box: gcd(64, page_size)
  const int *group_start, *prefix;                // null: no groups
  int ngroups;
  float scale_log2;
  __nv_bfloat16* out;
  float* lse;
  float *whole_prefix, *whole_own;                // [T * Hq][D + 2]: o, then m and l, of items that one block had whole
  float* split;                                   // [2 * blocks][128][D + 2]: a block's first and last, part-done items
  int* meta;                                      // [units + 1] running sum of tiles
};
constexpr int kPart = D + 4;                      // floats of a partial row (16-byte aligned)

// A whole warp's wait: the lanes go on together or give up together.
KORE_DEV bool warp_wait(uint64_t* bar, uint32_t phase) { return __all_sync(0xffffffff, mbar_wait(bar, phase)); }

struct AttnSmem {
  static constexpr int Q_OFF = 0;
  static constexpr int K_OFF = kQBytes;
  static constexpr int V_OFF = K_OFF + kStages * kTileBytes;
  static constexpr int BAR_OFF = V_OFF + kStages * kTileBytes;
  static constexpr int QS_OFF = BAR_OFF + 256;                       // int [kMaxSeqs + 1]
  static constexpr int CUM_OFF = QS_OFF + 4 * (kMaxSeqs + 2);        // int [2 * kMaxSeqs + 1]
  static constexpr int GS_OFF = CUM_OFF + 4 * (2 * kMaxSeqs + 2);    // uint16 [kMaxSeqs + 1]
  static constexpr int TOTAL = GS_OFF + 2 * (kMaxSeqs + 2) + 1024;
};
static_assert(2 * (AttnSmem::TOTAL + 1024) <= 228 * 1024, "two blocks share an SM");

// 128 x 128 tile as two K-major 64-column atoms of 16 KB, at K-step kk; 64 x 128 tile
// (two atoms of 8 KB) K-major and MN-major (rows = K) at K-step kk.
KORE_DEV uint64_t q_desc(uint32_t base, int kk) { return make_sw128_desc(base + (kk >> 2) * 16384 + (kk & 3) * 32, 16, 1024); }
KORE_DEV uint64_t k_desc(uint32_t base, int kk) { return make_sw128_desc(base + (kk >> 2) * 8192 + (kk & 3) * 32, 16, 1024); }
KORE_DEV uint64_t v_desc(uint32_t base, int kk) { return make_sw128_desc(base + kk * 2048, 8192, 1024); }
KORE_DEV void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  tmem_st16(taddr, *reinterpret_cast<const uint32_t(*)[16]>(&r[0]));
  tmem_st16(taddr + 16, *reinterpret_cast<const uint32_t(*)[16]>(&r[16]));
}

// The units as every block sees them: unit u < ngroups is a prefix, unit ngroups + b sequence b.
struct Units {
  const AttnParams& p;
  const int* qs;          // [B + 1] clamped to [0, T]
  const int* cum;         // [units + 1] tiles before the unit
  const uint16_t* gs;     // [ngroups + 1] clamped to [0, B]
  KORE_DEV int cap() const { return p.M * p.page_size; }
  KORE_DEV int group_of(int b) const {              // -1: none
    int lo = 0, hi = p.ngroups;                     // first group that starts behind b
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (gs[mid] <= b) lo = mid + 1; else hi = mid;
    }
    return lo > 0 && b < gs[lo] ? lo - 1 : -1;
  }
  KORE_DEV int prefix_of(int g) const { return min(max(p.prefix[g], 0), cap()); }
  KORE_DEV int row0(int u) const { return u < p.ngroups ? qs[gs[u]] : qs[u - p.ngroups]; }
  KORE_DEV int tokens(int u) const {
    return u < p.ngroups ? qs[gs[u + 1]] - qs[gs[u]] : qs[u - p.ngroups + 1] - qs[u - p.ngroups];
  }
  KORE_DEV int block_tokens(int u) const { return u < p.ngroups ? p.tokens_prefix : p.tokens_own; }
  KORE_DEV int blocks(int u) const { return (tokens(u) + block_tokens(u) - 1) / block_tokens(u); }
  KORE_DEV void keys(int u, int& lo, int& hi) const {      // the unit's keys
    if (u < p.ngroups) {
      lo = 0;
      hi = prefix_of(u);
    } else {
      const int g = p.ngroups ? group_of(u - p.ngroups) : -1;
      lo = g < 0 ? 0 : prefix_of(g);
      hi = min(max(p.lens[u - p.ngroups], 0), cap());
    }
  }
  KORE_DEV int tiles(int u) const {
    if (tokens(u) <= 0) return 0;
    int lo, hi;
    keys(u, lo, hi);
    return hi > lo ? ((hi + BK - 1) / BK - lo / BK) * blocks(u) * p.Hkv : 0;
  }
};

struct Item {
  int u, h, rb, n, j0, j1;       // unit, kv head, row block, tiles of the item, this block's tiles of it
};
// The item at tile x of [x, hi); advances x past this block's part of it. False at the end.
KORE_DEV bool next_item(const Units& w, int& x, int hi, int& u, Item& it) {
  if (x >= hi) return false;
  while (w.cum[u + 1] <= x) ++u;
  const int nb = w.blocks(u);
  it.u = u;
  it.n = (w.cum[u + 1] - w.cum[u]) / (nb * w.p.Hkv);
  const int r = x - w.cum[u], i = r / it.n;
  it.h = i / nb;
  it.rb = i % nb;
  it.j0 = r % it.n;
  it.j1 = min(it.n, it.j0 + hi - x);
  x += it.j1 - it.j0;
  return true;
}
KORE_DEV int run_start(long c, long W, long C) { return (int)(c * W / C); }
KORE_DEV int block_of(long x, long W, long C) { return (int)(((x + 1) * C - 1) / W); }   // whose run holds tile x
KORE_DEV int used_blocks(int W, int grid) { return max(1, min(grid, (W + kMinTiles - 1) / kMinTiles)); }

__global__ void __launch_bounds__(kAttnThreads, 2)
    attn_kernel(const __grid_constant__ CUtensorMap tmQp, const __grid_constant__ CUtensorMap tmQo,
                const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, AttnParams p) {
  using S = AttnSmem;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::BAR_OFF);
  uint64_t *q_full = bars, *q_empty = bars + 1, *o_done = bars + 2, *o_final = bars + 3, *o_free = bars + 4;
  uint64_t *k_full = bars + 5, *k_empty = k_full + kStages, *v_full = k_empty + kStages, *v_empty = v_full + kStages;
  uint64_t *s_full = v_empty + kStages, *p_full = s_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(p_full + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* warp_sum = reinterpret_cast<int*>(tmem_slot + 2);             // [6]
  int* qs = reinterpret_cast<int*>(smem + S::QS_OFF);
  int* cum = reinterpret_cast<int*>(smem + S::CUM_OFF);
  uint16_t* gs = reinterpret_cast<uint16_t*>(smem + S::GS_OFF);
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  const Units w{p, qs, cum, gs};

  pdl_trigger();
  // ---- the units' tiles, summed
  for (int i = threadIdx.x; i <= p.B; i += kAttnThreads) qs[i] = min(max(p.q_start[i], 0), p.T);
  for (int i = threadIdx.x; i <= p.ngroups; i += kAttnThreads)
    gs[i] = (uint16_t)(p.ngroups ? min(max(p.group_start[i], 0), p.B) : 0);
  if (threadIdx.x == 0) {
    for (uint64_t* b : {q_full, q_empty, o_done, o_final}) mbar_init(b, 1);
    mbar_init(o_free, 4);
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  __syncthreads();
  const int nu = p.ngroups + p.B, per = (nu + kAttnThreads - 1) / kAttnThreads;
  {
    const int u0 = min((int)threadIdx.x * per, nu), u1 = min(u0 + per, nu);
    int mine = 0;
    for (int u = u0; u < u1; ++u) mine += w.tiles(u);
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffff, upto, o);
      if (lane >= o) upto += y;
    }
    if (lane == 31) warp_sum[warp] = upto;
    __syncthreads();
    int at = upto - mine;
    for (int i = 0; i < warp; ++i) at += warp_sum[i];
    for (int u = u0; u < u1; ++u) {
      cum[u] = at;
      at += w.tiles(u);
    }
    if (u1 == nu) cum[nu] = at;      // the same from every thread that ends there
  }
  __syncthreads();
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i <= nu; i += kAttnThreads) p.meta[i] = cum[i];
  const int W = cum[nu], C = used_blocks(W, gridDim.x), c = blockIdx.x;
  if (W == 0 || c >= C) return;
  const int x0 = run_start(c, W, C), x1 = run_start(c + 1, W, C);
  int u_first = 0;
  {
    int lo = 0, hi = nu;             // the last unit that starts at or before x0
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (cum[mid + 1] <= x0) lo = mid + 1; else hi = mid;
    }
    u_first = lo;
  }
  if (warp == 1) tmem_alloc(tmem_slot, kTmemCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  constexpr uint32_t T_O = 128;
  int x = x0, u = u_first, k = 0, cnt = 0;        // tile, unit, items done, tiles done
  Item it;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    while (next_item(w, x, x1, u, it)) {
      const bool pre = it.u < p.ngroups;
      const int tb = w.block_tokens(it.u), t0 = w.row0(it.u) + it.rb * tb;
      int klo, khi;
      w.keys(it.u, klo, khi);
      const int* bt = p.table + (pre ? (long)gs[it.u] : (long)(it.u - p.ngroups)) * p.ld_table;
      bool ok = true;
      if (lane == 0) {
        ok = !*abort_flag && (k == 0 || mbar_wait(q_empty, (k - 1) & 1));
        if (ok) {
          const CUtensorMap* tm = pre ? &tmQp : &tmQo;
          mbar_arrive_expect_tx(q_full, 2 * 128 * p.G * tb);
          tma_load_3d(smem + S::Q_OFF, tm, q_full, 0, it.h * p.G, t0);
          tma_load_3d(smem + S::Q_OFF + 16384, tm, q_full, 64, it.h * p.G, t0);
        }
      }
      const int tile0 = klo / BK, nbox = BK / p.box;
      int page = 0, window = -32;                 // lane i holds the page of the item's box window + i
      for (int j = it.j0; j < it.j1; ++j, ++cnt) {
        const int st = cnt % kStages;
        const uint32_t ph = (cnt / kStages) & 1;
        const int key0 = (tile0 + j) * BK;
        const int b0 = min(max((klo - key0) / p.box, 0), nbox), b1 = min((khi - key0 + p.box - 1) / p.box, nbox);  // boxes with keys of the unit
        const int first = (j - it.j0) * nbox;
        if (first >= window + 32) {               // 32 is a multiple of nbox: a tile's boxes lie in one window
          window = first;
          const int key = key0 + lane * p.box;
          page = key >= klo - (klo % p.box) && key < khi ? bt[key / p.page_size] : 0;
        }
        if (lane == 0 && ok) ok = mbar_wait(&k_empty[st], ph ^ 1);
        uint8_t* kt = smem + S::K_OFF + st * kTileBytes;
        uint8_t* vt = smem + S::V_OFF + st * kTileBytes;
        const uint32_t bytes = (uint32_t)(b1 - b0) * p.box * 256;
        if (lane == 0 && ok) mbar_arrive_expect_tx(&k_full[st], bytes);
        for (int b = b0; b < b1; ++b) {
          const int key = key0 + b * p.box;
          const int z = (int)((unsigned)__shfl_sync(0xffffffff, page, first - window + b) * (unsigned)p.page_size + key % p.page_size);
          if (lane == 0 && ok) {
            tma_load_3d(kt + b * p.box * 128, &tmK, &k_full[st], 0, it.h, z);
            tma_load_3d(kt + 8192 + b * p.box * 128, &tmK, &k_full[st], 64, it.h, z);
          }
        }
        if (lane == 0 && ok) ok = mbar_wait(&v_empty[st], ph ^ 1);
        if (lane == 0 && ok) mbar_arrive_expect_tx(&v_full[st], bytes);
        for (int b = b0; b < b1; ++b) {
          const int key = key0 + b * p.box;
          const int z = (int)((unsigned)__shfl_sync(0xffffffff, page, first - window + b) * (unsigned)p.page_size + key % p.page_size);
          if (lane == 0 && ok) {
            tma_load_3d(vt + b * p.box * 128, &tmV, &v_full[st], 0, it.h, z);
            tma_load_3d(vt + 8192 + b * p.box * 128, &tmV, &v_full[st], 64, it.h, z);
          }
        }
        ok = __shfl_sync(0xffffffff, ok && !*abort_flag, 0);
        if (!ok) break;
      }
      if (!ok) { *abort_flag = 1; break; }
      ++k;
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA
    constexpr uint32_t idesc_qk = make_idesc_bf16(128, BK, false, false);
    constexpr uint32_t idesc_pv = make_idesc_bf16(128, D, false, true);
    if (elect_one()) {
      const uint32_t qa = smem_u32(smem + S::Q_OFF);
      bool ok = true;
      auto issue_s = [&](int i) -> bool {         // i: tile of this block
        const int st = i % kStages;
        if (!mbar_wait(&k_full[st], (i / kStages) & 1)) return false;
        tc_fence_after();
        const uint32_t ka = smem_u32(smem + S::K_OFF + st * kTileBytes);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          umma_f16_ss(tmem + (i & 1) * BK, q_desc(qa, kk), k_desc(ka, kk), idesc_qk, kk > 0);
        umma_commit(&k_empty[st]);
        umma_commit(&s_full[i & 1]);
        return true;
      };
      while (ok && next_item(w, x, x1, u, it)) {
        const int n = it.j1 - it.j0;
        ok = mbar_wait(q_full, k & 1);
        if (ok) ok = issue_s(cnt);
        for (int j = 0; j < n && ok; ++j) {
          const int i = cnt + j;
          // the buffer of S_{i+1} held P_{i-1}, which PV_{i-1}, issued before, has read by then (one in-order pipe)
          if (j + 1 < n) ok = issue_s(i + 1);
          if (ok && j + 1 == n) umma_commit(q_empty);              // the item's last S is issued
          const int st = i % kStages;
          if (ok && j == 0 && k > 0) ok = mbar_wait(o_free, (k - 1) & 1);   // the last item's O has been read
          if (ok) ok = mbar_wait(&p_full[i & 1], (i >> 1) & 1);
          if (ok) ok = mbar_wait(&v_full[st], (i / kStages) & 1);
          if (!ok) break;
          tc_fence_after();
          const uint32_t va = smem_u32(smem + S::V_OFF + st * kTileBytes);
#pragma unroll
          for (int kk = 0; kk < BK / 16; ++kk)
            umma_f16_ts(tmem + T_O, tmem + (i & 1) * BK + kk * 8, v_desc(va, kk), idesc_pv, (j > 0 || kk > 0) ? 1u : 0u);
          umma_commit(&v_empty[st]);
          umma_commit(o_done);
        }
        if (ok) umma_commit(o_final);
        cnt += n;
        ++k;
      }
      if (!ok) *abort_flag = 1;
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ softmax
    const int q4 = warp & 3, row = q4 * 32 + lane;
    const uint32_t lane_base = (uint32_t)(q4 * 32) << 16;
    bool ok = true;
    while (ok && next_item(w, x, x1, u, it)) {
      const bool pre = it.u < p.ngroups;
      const int tb = w.block_tokens(it.u), rt = it.rb * tb + row / p.G;      // token within the unit
      const bool live = row < tb * p.G && rt < w.tokens(it.u);
      const bool warp_live = __any_sync(0xffffffff, live);
      const int t = w.row0(it.u) + rt, h = it.h * p.G + row % p.G;
      int klo, khi, limit = 0;                    // the row sees keys [klo, limit)
      w.keys(it.u, klo, khi);
      bool joined = pre;                          // another part of the row's keys is another unit's
      if (live) {
        int b = it.u - p.ngroups;
        if (pre) {
          int lo = gs[it.u], hi = gs[it.u + 1] - 1;
          while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (qs[mid + 1] <= t) lo = mid + 1; else hi = mid;
          }
          b = lo;
        } else if (p.ngroups) {
          const int g = w.group_of(b);
          joined = g >= 0 && cum[g + 1] > cum[g];
        }
        limit = min(p.lens[b] - (qs[b + 1] - t) + 1, khi);
      }
      const int tile0 = klo / BK;
      float m = -INFINITY, l = 0.f, sv[BK];
      for (int j = it.j0; j < it.j1; ++j, ++cnt) {
        const int st = cnt & 1, kv0 = (tile0 + j) * BK;
        if (!warp_wait(&s_full[st], (cnt >> 1) & 1)) { ok = false; break; }
        if (kv0 < klo || kv0 + BK > khi) {
          // What lies outside the unit's keys may be anything, NaN included, and
          // 0 x NaN is not 0: these rows of V are cleared before the product reads them.
          const int vs = cnt % kStages;
          if (!warp_wait(&v_full[vs], (cnt / kStages) & 1)) { ok = false; break; }
          const int r = q4 * 16 + (lane >> 1);
          if (kv0 + r < klo || kv0 + r >= khi) {
            uint4* dst = reinterpret_cast<uint4*>(smem + S::V_OFF + vs * kTileBytes + (lane & 1) * 8192 + r * 128);
#pragma unroll
            for (int i = 0; i < 8; ++i) dst[i] = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        }
        if (warp_live) {
          tc_fence_after();
          {
            uint32_t r[2][32];
            tmem_ld32(tmem + lane_base + st * BK, r[0]);
            tmem_ld32(tmem + lane_base + st * BK + 32, r[1]);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < BK; ++i) sv[i] = __uint_as_float(r[i / 32][i % 32]);
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
              if (!warp_wait(o_done, (cnt - 1) & 1)) { ok = false; break; }
              tc_fence_after();
#pragma unroll
              for (int i4 = 0; i4 < 4; ++i4) {
                uint32_t r[32];
                const uint32_t a = tmem + lane_base + T_O + i4 * 32;
                tmem_ld32(a, r);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * alpha);
                tmem_st32(a, r);
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
          // P in bf16 (the operand type of V): each probability is off by 2^-9 of itself, the sum l is not rounded
          uint32_t pk[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) pk[i] = pack_bf16(sv[2 * i], sv[2 * i + 1]);
          tmem_st32(tmem + lane_base + st * BK, pk);
          tmem_wait_st();
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[st]);
      }
      if (!ok || !warp_wait(o_final, k & 1)) { ok = false; break; }
      if (warp_live) {
        tc_fence_after();
        const bool whole = it.j0 == 0 && it.j1 == it.n, direct = whole && !joined;
        const size_t at = (size_t)t * p.Hq + h;
        const float inv = l == 0.f ? 0.f : 1.f / l;
        float* part = whole ? (pre ? p.whole_prefix : p.whole_own) + at * kPart
                            : p.split + ((size_t)(2 * c + (it.j0 == 0 ? 1 : 0)) * 128 + row) * kPart;
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
          uint32_t r[32];
          tmem_ld32(tmem + lane_base + T_O + i4 * 32, r);
          tmem_wait_ld();
          if (live && direct) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint4 v;
              v.x = pack_bf16(__uint_as_float(r[8 * i + 0]) * inv, __uint_as_float(r[8 * i + 1]) * inv);
              v.y = pack_bf16(__uint_as_float(r[8 * i + 2]) * inv, __uint_as_float(r[8 * i + 3]) * inv);
              v.z = pack_bf16(__uint_as_float(r[8 * i + 4]) * inv, __uint_as_float(r[8 * i + 5]) * inv);
              v.w = pack_bf16(__uint_as_float(r[8 * i + 6]) * inv, __uint_as_float(r[8 * i + 7]) * inv);
              *reinterpret_cast<uint4*>(p.out + at * D + i4 * 32 + 8 * i) = v;
            }
          } else if (live) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              *reinterpret_cast<uint4*>(part + i4 * 32 + 4 * i) = make_uint4(r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
          }
        }
        if (live && direct && p.lse) p.lse[at] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
        if (live && !direct) {
          part[D] = m;
          part[D + 1] = l;
        }
        tc_fence_before();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(o_free);
      ++k;
    }
    if (!ok) *abort_flag = 1;
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// Joins the partials of a token's rows: one block per token, one warp per head.
// Parts are added in the order prefix, own keys, ascending tiles.
__global__ void __launch_bounds__(256) join_kernel(AttnParams p, int grid) {
  pdl_wait();
  const int t = blockIdx.x, lane = threadIdx.x & 31;
  if (t >= min(p.q_start[p.B], p.T)) return;
  // the last i in [0, n] with v[i] <= key (v[0] <= key), 32 probes at a time
  auto last_at_most = [&](const int* v, int n, int key) {
    int lo = 0, hi = n;
    while (hi > lo) {
      const int step = (hi - lo + 31) / 32, i = lo + (lane + 1) * step;
      const unsigned m = __ballot_sync(0xffffffff, i <= hi && v[i] <= key);
      const int k = __popc(m);       // probes are ascending: the first k hold
      lo += k * step;
      hi = min(hi, lo + step - 1);
    }
    return lo;
  };
  auto start = [&](int i) { return min(max(p.q_start[i], 0), p.T); };
  auto group = [&](int i) { return min(max(p.group_start[i], 0), p.B); };
  const int b = min(last_at_most(p.q_start, p.B, t), p.B - 1);
  const int nu = p.ngroups + p.B, W = p.meta[nu], C = used_blocks(W, grid);
  int g = -1;
  if (p.ngroups && p.group_start[0] <= b) {
    g = last_at_most(p.group_start, p.ngroups, b);
    if (g >= p.ngroups || p.meta[g + 1] == p.meta[g]) g = -1;          // in no group, or nothing shared
  }
  for (int h = threadIdx.x / 32; h < p.Hq; h += blockDim.x / 32) {
    const size_t at = (size_t)t * p.Hq + h;
    // up to two units: first partial row and the distance to the next
    const float* first[2] = {nullptr, nullptr};
    int count[2] = {0, 0}, c0[2] = {0, 0}, row[2] = {0, 0};
    bool whole_own = false;
    for (int i = 0; i < 2; ++i) {
      const int u = i == 0 ? g : p.ngroups + b;
      if (u < 0) continue;
      const int tiles = p.meta[u + 1] - p.meta[u];
      if (tiles == 0) continue;
      const int s0 = i == 0 ? group(g) : b, s1 = i == 0 ? group(g + 1) : b + 1;
      const int tb = i == 0 ? p.tokens_prefix : p.tokens_own, q0 = start(s0);
      const int nb = (start(s1) - q0 + tb - 1) / tb, rb = (t - q0) / tb;
      if (nb <= 0 || t < q0 || rb >= nb) continue;   // starts that do not ascend: nothing is read out of range
      const int n = tiles / (nb * p.Hkv), x = p.meta[u] + ((h / p.G) * nb + rb) * n;
      const int ca = block_of(x, W, C), cb = block_of(x + n - 1, W, C);
      row[i] = (t - q0 - rb * tb) * p.G + h % p.G;
      c0[i] = ca;
      count[i] = cb - ca + 1;
      if (count[i] == 1) {
        first[i] = (i == 0 ? p.whole_prefix : p.whole_own) + at * kPart;
        whole_own = whole_own || i == 1;
      }
    }
    if (whole_own && count[0] == 0) continue;        // written by the block that had it all
    auto part = [&](int i, int j) -> const float* {
      if (first[i]) return first[i];
      return p.split + ((size_t)(2 * (c0[i] + j) + (j == 0 ? 1 : 0)) * 128 + row[i]) * kPart;
    };
    float m = -INFINITY;
    for (int i = 0; i < 2; ++i)
      for (int j = 0; j < count[i]; ++j) m = fmaxf(m, part(i, j)[D]);
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = 0; i < 2; ++i)
      for (int j = 0; j < count[i]; ++j) {
        const float* r = part(i, j);
        if (r[D] == -INFINITY) continue;             // no key of this part was visible
        const float f = exp2f(r[D] - m);
        const float4 v = *reinterpret_cast<const float4*>(r + lane * 4);
        l += r[D + 1] * f;
        o.x += v.x * f; o.y += v.y * f; o.z += v.z * f; o.w += v.w * f;
      }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    *reinterpret_cast<uint2*>(p.out + at * D + lane * 4) = make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
    if (p.lse && lane == 0) p.lse[at] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
  }
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
  TORCH_CHECK(rows >= 0 && rows <= 0x7fffffff, "paged: rows out of range");
  if (held) check_ints(*held, ctx, B, "held");
  TORCH_CHECK(free_stack.has_value() == free_count.has_value(), "paged: give free and free_count, or neither");
  if (free_stack) {
    check_ints(*free_stack, ctx, -1, "free");
    check_ints(*free_count, ctx, 1, "free_count");
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
  plan_kernel<<<1, kPlanThreads, 0, st>>>(p);
  check_cuda(cudaGetLastError(), "paged_plan");
  if (rows) {
    plan_rows_kernel<<<(unsigned)((rows + 255) / 256), 256, 0, st>>>(p);
    check_cuda(cudaGetLastError(), "paged_plan rows");
  }
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
  TORCH_CHECK(B <= 1024, "prefix_attention: at most 1024 sequences a call");
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
  TORCH_CHECK(scale > 0, "prefix_attention: scale must be positive");
  if (T == 0 || B == 0) return;
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
  p.tokens_own = (int)std::min<int64_t>(128 / G, max_q);
  p.box = (int)std::gcd<int64_t, int64_t>(page_size, BK);
  p.group_start = group_start ? group_start->data_ptr<int>() : nullptr;
  p.prefix = prefix_len ? prefix_len->data_ptr<int>() : nullptr;
  p.ngroups = ngroups;
  p.scale_log2 = (float)(scale * 1.4426950408889634);
  p.out = (__nv_bfloat16*)out.data_ptr();
  p.lse = lse ? lse->data_ptr<float>() : nullptr;
  const int64_t tiles = (table.size(1) * page_size + BK - 1) / BK + 1;
  TORCH_CHECK(tiles * Hkv * (T / p.tokens_prefix + ngroups + T / p.tokens_own + B) < (int64_t)1 << 30,
              "prefix_attention: rows x table length out of range");
  // Partials: whole items of rows that have a shared prefix, one row each; what the
  // blocks' runs cut, two row blocks for each of them.
  const int grid = 2 * num_sms(q.get_device());
  const int64_t rows = ngroups ? T * Hq * kPart : 0, split = (int64_t)2 * grid * 128 * kPart;
  at::Tensor ws = at::empty({2 * rows + split + ngroups + B + 1}, q.options().dtype(at::kFloat));
  p.whole_prefix = ws.data_ptr<float>();
  p.whole_own = p.whole_prefix + rows;
  p.split = p.whole_own + rows;
  p.meta = reinterpret_cast<int*>(p.split + split);
  const auto bf = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const CUtensorMap tq = make_tmap_3d(q.data_ptr(), bf, 2, D, Hq, T, D, q.stride(0), 64, G, p.tokens_prefix);
  const CUtensorMap to = make_tmap_3d(q.data_ptr(), bf, 2, D, Hq, T, D, q.stride(0), 64, G, p.tokens_own);
  const CUtensorMap tk = make_tmap_3d(kc.data_ptr(), bf, 2, D, Hkv, kc.size(0), kc.stride(1), kc.stride(0), 64, 1, p.box);
  const CUtensorMap tv = make_tmap_3d(vc.data_ptr(), bf, 2, D, Hkv, vc.size(0), vc.stride(1), vc.stride(0), 64, 1, p.box);
  static bool attr[64] = {};
  const int dev = q.get_device();
  if (!attr[dev]) {
    check_cuda(cudaFuncSetAttribute(attn_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, AttnSmem::TOTAL), "prefix_attention smem");
    attr[dev] = true;
  }
  auto st = at::cuda::getCurrentCUDAStream();
  attn_kernel<<<grid, kAttnThreads, AttnSmem::TOTAL, st>>>(tq, to, tk, tv, p);
  check_cuda(cudaGetLastError(), "prefix_attention");
  launch_after("prefix_attention join", join_kernel, dim3((unsigned)T), dim3(256), 0, st, p, grid);
}

}  // namespace kore
