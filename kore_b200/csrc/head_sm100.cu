// Language-model head in pieces of the vocabulary, without keeping logits.
//
//   z_tj  = (x_t . W_j) / tau                       x [T, H], W [V, H] bf16
//   lse_t = log sum_j e^{z_tj},  logp_t = z_{t,y_t} - lse_t
//   ent_t = lse_t - sum_j p_tj z_tj,  p_tj = e^{z_tj - lse_t}
//   L = sum_t c_t logp_t:  dz_tj = (c_t / tau) (1[j = y_t] - p_tj)
//                          dx = dz W,  dW = dz^T x
//
// Forward: a 2-CTA tcgen05 GEMM whose epilogue never writes z. Each thread owns
// half a row of a tile in TMEM and turns its columns into a triple (m = max,
// s = sum e^{z-m}, u = sum (z-m) e^{z-m}; ent = log s - u / s, which does not
// cancel when the logits are large); the triples go to a workspace, and a second
// kernel joins those of a row. The logit of the label is written by the one tile
// that holds it. Logits stay fp32 from the accumulator on.
// Backward: per piece of the vocabulary the same GEMM runs again and its
// epilogue turns z into dz (bf16, the operand type of the two products that
// follow; few rows: two bf16 terms); then one launch computes dW[piece] = dz^T x
// and dx += dz W[piece]: the tiles of both products fill each other's last wave.
// dW rows are final after their piece (one rounding); dx sums its pieces in fp32
// and is rounded once.
// Rows with coefficient 0 have dz = 0 whatever x or the statistics hold there,
// and dW reads such rows of x as zeros, so an inf or NaN in them stays out.
//
// Bound by the tensor cores: at T = 8192, V = 151936, H = 5120 the forward takes 9.1 ms
// in a short run (1.40 PFLOP/s) and 10.0 ms under the power cap (1.28; a library
// GEMM sustains 1.38), forward and gradients 40 ms over four products of 2 T V H.
// One row is bound by W (255 us, 6.1 TB/s); small H by the latency of the epilogue,
// which reads 256 columns a row from TMEM and takes as many exponentials with two
// warps per scheduler (T = 1065, V = 124357, H = 136: 117 us, 3.6 us a tile; issue
// slots 35% busy, the exponential unit 34%, the tensor pipe 26%).
//
// Reference parity: kore/policy/grpo.py:2728-2743 (log-softmax and gather over
// the full vocabulary), kore/policy/sft.py:346-399 (mean cross-entropy).
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "common.cuh"
#include "tma_host.h"

namespace kore {

namespace head {

constexpr int BM = 128;        // rows per CTA (256 per pair)
constexpr int BK = 64;
constexpr int kMaxBN = 256;    // columns of a pair's tile
constexpr int kEpiWarps = 8;   // two per TMEM lane quadrant, each takes half of the columns
constexpr int kThreads = 64 + 32 * kEpiWarps;  // TMA producer, MMA issuer, epilogue
constexpr int kABytes = BM * BK * 2;
constexpr int kBBytes = (kMaxBN / 2) * BK * 2;
constexpr int kStageBytes = kABytes + kBBytes;
constexpr int kStoreBytes = 32 * 128;  // one store box: 32 rows x 128 bytes
// The tensor cores truncate the fp32 accumulator at every 16 products, which
// biases a long sum towards zero: log-probs were off by 2.6e-6 of themselves at
// H = 5120, against 0.7e-6 for an fp32 matrix product. The forward therefore
// reads the accumulator out after each part of K and adds the parts in registers
// with rounding. A read-out stalls the MMAs by about 1100 clocks (a k-block takes
// 720). With parts of 8, 12, 16 k-blocks the error was 2.2e-7, 3.3e-7, 4.7e-7 and
// the time 11.8, 11.0, 10.3 ms (T = 8192, V = 151936); unsplit 10.3 ms. Short
// sums take a few parts too: 8.6e-7 with one at H = 1024.
// The gradient's logits are summed in the same parts. Where the label is well
// predicted, its entry c (p - 1) is what is left of the difference of its logit and
// the forward's lse: summed over all of K at once the logit is off by 1e-4 at H = 5120,
// always to one side, which was half of such a row's dx at 1 - p = 2e-4 (0.6% with the
// parts). All of head_bwd, ms, one part / parts: T = 8192, H = 2048 11.9 / 12.4; H = 5120
// about 2% more. With one or two rows the forward's sums are exact and the parts' error
// (3e-7 of the logit) is left.
__host__ __device__ constexpr int k_parts(int kblocks) {
  return kblocks <= 8 ? 1 : kblocks <= 16 ? 2 : kblocks <= 48 ? 3 : (kblocks + 15) / 16;
}
// dz is rounded to bf16 for the products that follow: at most 2^-8 of a value,
// which the sums over many rows and entries average out. With few rows a single
// rounding shows in a whole row of dW (2.9e-3 of it, against 1.6e-3 from the
// rounding of the output), and the products are bound by W and dW: up to this
// many rows dz is kept as the sum of two bf16 terms, which fill otherwise idle
// rows and k-blocks of the same tiles.
constexpr int kTwoTerms = 128;
constexpr int kRowBlock = 32768;  // rows per forward launch: bounds the statistics workspace
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// What a launch does with its tiles of A B^T:
//   STATS  A = x, B = W piece: row statistics      (columns: vocabulary, K = H)
//   GRAD   A = x, B = W piece: dz, bf16            (columns: vocabulary, K = H in one part)
//   GRADK  the same where K has several parts
//   PRODS  first A = dz, B = W piece^T: fp32 parts of dx   (columns: H, K = vocabulary, split)
//          then  A = dz^T, B = x^T: dW of the piece        (rows: vocabulary, columns: H, K = dz's rows)
enum Mode { STATS, GRAD, GRADK, PRODS };

template <Mode M>
struct Layout {
  static constexpr int kStages = M == STATS ? 7 : 6;
  static constexpr int kEpiOff = kStages * kStageBytes;
  static constexpr int kBarOff = kEpiOff + (M == STATS ? 0 : kEpiWarps * kStoreBytes);
  static constexpr int kSmem = kBarOff + 256 + 1024;
};

struct Params {
  int rows, cols, K;    // A rows, B rows (columns of the product), contraction
  int bn;               // columns per tile (multiple of 16, <= 256)
  const long* targets;  // STATS, GRAD(K); may be null
  int v0;               // vocabulary id of column 0
  float scale;          // log2(e) / tau: the epilogue works in powers of two
  float inv_temp;
  // STATS
  float* stats;         // [planes][2 num_n][rows]: m, s, (u)
  float* zt;            // [rows] label logit in units of log2
  int entropy;
  // GRAD, GRADK
  const float* lse;
  const float* coef;
  __nv_bfloat16* low;   // not null: what bf16 leaves of dz goes here, row stride low_ld
  long low_ld;
  // PRODS
  int splits;           // parts of dx's K; part i is stored at row i * split_rows
  int split_rows;
  int add;              // add to the dx parts of earlier pieces
  void* dw;             // the piece's rows of dW, contiguous
  int dw_f32, dw_add;   // fp32 (else bf16); add to what is there
};

// The tensor maps of a launch: A, B and the output; PRODS: those of dx, then of dW.
struct Maps {
  CUtensorMap a, b, d, a2, b2, d2;
};

KORE_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

KORE_DEV void tma_reduce_add_2d(const CUtensorMap* d, const void* smem_src, int x, int y) {
  asm volatile(
      "cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
          reinterpret_cast<uint64_t>(d)),
      "r"(smem_u32(smem_src)), "r"(x), "r"(y)
      : "memory");
}

// 64 accumulator columns of this lane's row, both loads in flight
KORE_DEV void load64(float (&f)[64], uint32_t from) {
  uint32_t a[32], b[32];
  tmem_ld32(from, a);
  tmem_ld32(from + 32, b);
  tmem_wait_ld();
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    f[i] = __uint_as_float(a[i]);
    f[32 + i] = __uint_as_float(b[i]);
  }
}

// groups of 8 row blocks walk the columns together, so a B tile is read
// from HBM once per 2048 rows and the group's A rows stay in L2
KORE_DEV void tile_coords(int t, int num_m, int num_n, int& tm, int& tn) {
  constexpr int G = 8;
  const int per_group = G * num_n;
  const int g = t / per_group;
  const int first_m = g * G;
  const int gsize = min(num_m - first_m, G);
  const int r = t - g * per_group;
  tm = first_m + r % gsize;
  tn = r / gsize;
}

template <Mode M>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    head_kernel(const __grid_constant__ Maps maps, const Params p) {
  using L = Layout<M>;
  constexpr int kStages = L::kStages;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + L::kBarOff);
  uint64_t* empty_bar = full_bar + kStages;
  uint64_t* tfull_bar = empty_bar + kStages;  // [2]
  uint64_t* tempty_bar = tfull_bar + 2;       // [2] (leader: both CTAs' epilogue warps arrive)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty_bar + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int pair = blockIdx.x / 2, npairs = gridDim.x / 2;
  const int bn = p.bn;
  const int num_m = (p.rows + 2 * BM - 1) / (2 * BM);
  const int num_n = (p.cols + bn - 1) / bn;
  const int num_mn = num_m * num_n;
  const int kblocks = (p.K + BK - 1) / BK;
  const int part = (kblocks + k_parts(kblocks) - 1) / k_parts(kblocks);  // k-blocks per part of a logit's sum
  const int dw_m = M == PRODS ? (p.K + 2 * BM - 1) / (2 * BM) : 0;
  const int first_dw = M == PRODS ? num_mn * p.splits : num_mn;          // work items before dW's
  const int num_items = first_dw + dw_m * num_n;
  // work item t: is it a tile of dW, its first row and column, its k-blocks [k0, k1)
  struct Item {
    bool dw;
    int m0, n0, tn, k0, k1, rows, split;
  };
  auto item = [&](int t) {
    Item w;
    int tm;
    w.dw = M == PRODS && t >= first_dw;
    w.k0 = 0;
    w.k1 = kblocks;
    w.split = 0;
    w.rows = p.rows;
    if (w.dw) {
      tile_coords(t - first_dw, dw_m, num_n, tm, w.tn);
      w.k1 = (p.rows + BK - 1) / BK;
      w.rows = p.K;
    } else {
      tile_coords(M == PRODS ? t % num_mn : t, num_m, num_n, tm, w.tn);
      if (M == PRODS) {
        w.split = t / num_mn;
        w.k0 = (int)((long)w.split * kblocks / p.splits);
        w.k1 = (int)((long)(w.split + 1) * kblocks / p.splits);
      }
    }
    w.m0 = tm * 2 * BM;
    w.n0 = w.tn * bn;
    return w;
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull_bar[b], 1);
      mbar_init(&tempty_bar[b], 2 * kEpiWarps);
    }
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&maps.a);
    tma_prefetch_desc(&maps.b);
    if (M != STATS) tma_prefetch_desc(&maps.d);
    if (M == PRODS) {
      tma_prefetch_desc(&maps.a2);
      tma_prefetch_desc(&maps.b2);
      tma_prefetch_desc(&maps.d2);
    }
  }
  if (warp == 1) tmem_alloc_pair(tmem_slot, 2 * kMaxBN);
  tc_fence_before();
  cluster_sync();  // both CTAs' barriers initialised and TMEM allocated
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();
  pdl_trigger();

  if (warp == 0) {
    // ------------------------------------------------------------ producer (both CTAs)
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      for (int t = pair; t < num_items && !*abort_flag; t += npairs) {
        const Item w = item(t);
        // a box that lies wholly past the rows or the columns is not loaded
        // (its part of the accumulator is never used)
        auto a_bytes = [&](int r) -> uint32_t {
          const int m = w.m0 + r * BM;
          if (!w.dw) return m < w.rows ? kABytes : 0u;
          return (m < w.rows ? 8192u : 0u) + (m + 64 < w.rows ? 8192u : 0u);
        };
        auto b_bytes = [&](int r) -> uint32_t {
          const int n = w.n0 + r * (bn / 2);
          if (M != PRODS) return n < p.cols ? (uint32_t)(bn / 2) * BK * 2 : 0u;
          return (n < p.cols ? 8192u : 0u) + (n + 64 < p.cols ? 8192u : 0u);
        };
        const uint32_t bytes = a_bytes(0) + a_bytes(1) + b_bytes(0) + b_bytes(1);
        const int m = w.m0 + (int)rank * BM, n = w.n0 + (int)rank * (bn / 2);
        for (int kb = w.k0; kb < w.k1; ++kb) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1)) { *abort_flag = 1; break; }
          uint8_t* sA = smem + stage * kStageBytes;
          uint8_t* sB = sA + kABytes;
          const uint32_t fb = mapa_shared(smem_u32(&full_bar[stage]), 0);
          const int k = kb * BK;
          if (rank == 0) mbar_arrive_expect_tx(&full_bar[stage], bytes);
          if (!w.dw) {
            if (m < w.rows) tma_load_2d_pair(sA, &maps.a, fb, k, m);
          } else {  // dz is [K, rows]: two 64-column boxes
            if (m < w.rows) tma_load_2d_pair(sA, &maps.a2, fb, m, k);
            if (m + 64 < w.rows) tma_load_2d_pair(sA + 8192, &maps.a2, fb, m + 64, k);
          }
          if (M != PRODS) {
            if (n < p.cols) tma_load_2d_pair(sB, &maps.b, fb, k, n);
          } else {  // W piece and x are [K, columns]
            const CUtensorMap* mb = w.dw ? &maps.b2 : &maps.b;
            if (n < p.cols) tma_load_2d_pair(sB, mb, fb, n, k);
            if (n + 64 < p.cols) tma_load_2d_pair(sB + 8192, mb, fb, n + 64, k);
          }
          if (++stage == kStages) { stage = 0; phase ^= 1; }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (leader)
    if (rank == 0 && elect_one()) {
      const uint32_t idesc_x = make_idesc_bf16(2 * BM, bn, false, M == PRODS);
      const uint32_t idesc_w = make_idesc_bf16(2 * BM, bn, true, true);
      int stage = 0, it = 0;
      uint32_t phase = 0;
      for (int t = pair; t < num_items && !*abort_flag; t += npairs) {
        const Item w = item(t);
        const uint32_t idesc = w.dw ? idesc_w : idesc_x;
        for (int c0 = w.k0; c0 < w.k1; ++it) {
          const int c1 = M == STATS || M == GRADK ? min(c0 + part, w.k1) : w.k1;
          const int acc = it & 1;
          if (!mbar_wait(&tempty_bar[acc], ((it >> 1) & 1) ^ 1)) { *abort_flag = 1; break; }
          tc_fence_after();
          const uint32_t d_tmem = tmem_base + acc * kMaxBN;
          bool ok = true;
          for (int kb = c0; kb < c1; ++kb) {
            if (!mbar_wait(&full_bar[stage], phase)) { ok = false; break; }
            tc_fence_after();
            const uint32_t a_addr = smem_u32(smem + stage * kStageBytes);
            const uint32_t b_addr = a_addr + kABytes;
#pragma unroll
            for (int k = 0; k < BK / 16; ++k)
              umma_f16_ss_pair(d_tmem,
                               w.dw ? make_sw128_desc(a_addr + k * 2048, 8192, 1024)
                                    : make_sw128_desc(a_addr + k * 32, 16, 1024),
                               M == PRODS ? make_sw128_desc(b_addr + k * 2048, 8192, 1024)
                                          : make_sw128_desc(b_addr + k * 32, 16, 1024),
                               idesc, kb != c0 || k != 0);
            umma_commit_pair(&empty_bar[stage], 0x3);
            if (++stage == kStages) { stage = 0; phase ^= 1; }
          }
          if (!ok) { *abort_flag = 1; break; }
          umma_commit_pair(&tfull_bar[acc], 0x3);
          c0 = c1;
        }
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ epilogue (both CTAs)
    const int q = warp & 3;            // TMEM lane quadrant this warp may access
    const int half = (warp - 2) / 4;   // and its half of the columns
    const int width = (bn + 63) / 64 * 32, h0 = half * width;
    uint8_t* stage_buf = smem + L::kEpiOff + (warp - 2) * kStoreBytes;
    const uint32_t tempty_leader[2] = {mapa_shared(smem_u32(&tempty_bar[0]), 0),
                                       mapa_shared(smem_u32(&tempty_bar[1]), 0)};
    int it = 0;
    for (int t = pair; t < num_items && !*abort_flag; t += npairs) {
      const Item w = item(t);
      if (w.k0 >= w.k1) continue;  // a narrow last piece leaves some parts of K empty: nothing was issued
      const int n0 = w.n0 + h0;
      const int row0 = w.m0 + (int)rank * BM + q * 32;
      const int row = row0 + lane;
      const int cols = row0 < w.rows ? min(min(width, bn - h0), p.cols - n0) : 0;  // this warp's columns
      const bool live = row < w.rows;
      // column of the label among them (negative: not here)
      int tc = -1;
      float lse2 = 0.f, c = 0.f;
      if (M != PRODS && live && p.targets != nullptr) {
        const long y = p.targets[row] - p.v0 - n0;
        if (y >= 0 && y < cols) tc = (int)y;
      }
      if ((M == GRAD || M == GRADK) && live) {
        lse2 = p.lse[row] * kLog2e;
        c = p.coef[row] * p.inv_temp;
      }
      const uint32_t t_row = tmem_base + ((uint32_t)(q * 32) << 16) + h0;
      // hands the accumulator back to the MMA warp
      auto release = [&](int acc) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(tempty_leader[acc]);
      };
      // sends a box of the warp's 32 rows x 128 bytes, a lane's row in eight vectors, to
      // column x and row y; add: into what is there
      auto store_begin = [&]() {
        if (lane == 0) tma_store_wait_read<0>();  // the last store has read the buffer
        __syncwarp();
      };
      auto store_put = [&](int j, const uint4& u) {
        *reinterpret_cast<uint4*>(stage_buf + lane * 128 + ((j ^ (lane & 7)) * 16)) = u;
      };
      auto store_end = [&](const CUtensorMap* map, int x, int y, bool add) {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          if (add) tma_reduce_add_2d(map, stage_buf, x, y);
          else tma_store_2d(map, stage_buf, x, y);
          tma_store_commit();
        }
      };
      auto store = [&](const CUtensorMap* map, const uint4 (&out)[8], int x, int y, bool add) {
        store_begin();
#pragma unroll
        for (int j = 0; j < 8; ++j) store_put(j, out[j]);
        store_end(map, x, y, add);
      };
      // 64 logits of the row, from the warp's column c0 on: dz is made in place and sent
      auto send_dz = [&](float (&f)[64], int c0) {
#pragma unroll
        for (int i = 0; i < 64; ++i) f[i] = -c * ex2(fmaf(f[i], p.scale, -lse2));
        if (c == 0.f || c0 + 64 > cols) {
          // coefficient 0, or past the piece's last column: 0
#pragma unroll
          for (int i = 0; i < 64; ++i)
            if (c == 0.f || c0 + i >= cols) f[i] = 0.f;
        }
        const int ti = tc - c0;
        if (ti >= 0 && ti < 64) {
#pragma unroll
          for (int i = 0; i < 64; ++i)
            if (i == ti) f[i] += c;
        }
        store_begin();
#pragma unroll
        for (int j = 0; j < 8; ++j)
          store_put(j, make_uint4(pack_bf16(f[8 * j], f[8 * j + 1]), pack_bf16(f[8 * j + 2], f[8 * j + 3]),
                                  pack_bf16(f[8 * j + 4], f[8 * j + 5]), pack_bf16(f[8 * j + 6], f[8 * j + 7])));
        store_end(&maps.d, n0 + c0, row0, false);
        if (p.low != nullptr && live) {
          __nv_bfloat16* low = p.low + row * p.low_ld + n0 + c0;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            uint32_t l[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float a = f[8 * j + 2 * e], b = f[8 * j + 2 * e + 1];
              const uint32_t hi = pack_bf16(a, b);
              l[e] = pack_bf16(a - __uint_as_float(hi << 16), b - __uint_as_float(hi & 0xffff0000u));
            }
            if (c0 + 8 * j < cols) *reinterpret_cast<uint4*>(low + 8 * j) = make_uint4(l[0], l[1], l[2], l[3]);
          }
        }
      };
      if (M == STATS) {
        // the row's columns stay in registers: first the maximum, then the sums
        // against it, each in four independent chains (two warps per scheduler
        // cannot hide a serial one)
        constexpr int kCols = kMaxBN / 2;
        uint32_t v[kCols];
        bool ok = true;
        for (int c0 = w.k0; c0 < w.k1; c0 += part, ++it) {
          const int acc = it & 1;
          if (!mbar_wait(&tfull_bar[acc], (it >> 1) & 1)) { ok = false; break; }
          tc_fence_after();
          const uint32_t from = t_row + acc * kMaxBN;
          if (c0 == w.k0) {
#pragma unroll
            for (int j = 0; j < kCols / 32; ++j)
              if (32 * j < cols) tmem_ld32(from + 32 * j, *reinterpret_cast<uint32_t(*)[32]>(v + 32 * j));
            tmem_wait_ld();
          } else {
#pragma unroll
            for (int j = 0; j < kCols / 32; ++j)
              if (32 * j < cols) {
                uint32_t r[32];
                tmem_ld32(from + 32 * j, r);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  v[32 * j + i] = __float_as_uint(__uint_as_float(v[32 * j + i]) + __uint_as_float(r[i]));
              }
          }
          release(acc);
        }
        if (!ok) { *abort_flag = 1; break; }
        if (cols < kCols) {
#pragma unroll
          for (int i = 0; i < kCols; ++i)
            if (i >= cols) v[i] = 0xff800000u;  // -inf: not a column of the vocabulary
        }
        if (tc >= 0) {
          uint32_t z = 0;
#pragma unroll
          for (int i = 0; i < kCols; ++i)
            if (i == tc) z = v[i];
          p.zt[row] = __uint_as_float(z) * p.scale;
        }
        float top[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) top[i] = __uint_as_float(v[i]);
#pragma unroll
        for (int i = 4; i + 8 <= kCols; i += 8)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            top[e] = fmax3f(top[e], __uint_as_float(v[i + 2 * e]), __uint_as_float(v[i + 2 * e + 1]));
#pragma unroll
        for (int e = 0; e < 4; ++e) top[e] = fmaxf(top[e], __uint_as_float(v[kCols - 4 + e]));
        const float m = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * p.scale;
        const float base = m == -INFINITY ? 0.f : m;  // all columns -inf: their terms are 0
        const uint64_t scale2 = f2_pack(p.scale, p.scale), base2 = f2_pack(-base, -base);
        uint64_t s2[4] = {0, 0, 0, 0}, u2[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < kCols; i += 2) {
          float z0, z1;
          f2_unpack(f2_fma(f2_pack(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), scale2, base2), z0, z1);
          const uint64_t e = f2_pack(ex2(z0), ex2(z1));
          s2[(i / 2) & 3] = f2_add(s2[(i / 2) & 3], e);
          // (0 times -inf is 0 here)
          if (p.entropy) u2[(i / 2) & 3] = f2_fma(e, f2_pack(fmaxf(z0, -1e30f), fmaxf(z1, -1e30f)), u2[(i / 2) & 3]);
        }
        float lo, hi;
        f2_unpack(f2_add(f2_add(s2[0], s2[1]), f2_add(s2[2], s2[3])), lo, hi);
        const float s = lo + hi;
        f2_unpack(f2_add(f2_add(u2[0], u2[1]), f2_add(u2[2], u2[3])), lo, hi);
        const float u = lo + hi;
        if (live) {
          const size_t o = (size_t)(2 * w.tn + half) * p.rows + row, plane = (size_t)2 * num_n * p.rows;
          p.stats[o] = m;
          p.stats[o + plane] = s;
          if (p.entropy) p.stats[o + 2 * plane] = u;
        }
      } else if (M == GRADK) {
        // the sum of the parts, as the forward sums them; the row's logits stay in registers
        float v[2][64];
        bool ok = true;
        for (int k = w.k0; k < w.k1; k += part, ++it) {
          const int acc = it & 1;
          if (!mbar_wait(&tfull_bar[acc], (it >> 1) & 1)) { ok = false; break; }
          tc_fence_after();
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (32 * j < cols) {
              uint32_t r[32];
              tmem_ld32(t_row + acc * kMaxBN + 32 * j, r);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                float& z = v[j / 2][32 * (j & 1) + i];
                z = k == w.k0 ? __uint_as_float(r[i]) : z + __uint_as_float(r[i]);
              }
            }
          release(acc);
        }
        if (!ok) { *abort_flag = 1; break; }
        if (cols > 0) send_dz(v[0], 0);
        // the second half's arithmetic stays behind the first half's stores (registers)
#pragma unroll
        for (int i = 0; i < 64; ++i) asm volatile("" : "+f"(v[1][i]));
        if (cols > 64) send_dz(v[1], 64);
      } else if (M == GRAD) {
        const int acc = it & 1;
        if (!mbar_wait(&tfull_bar[acc], (it >> 1) & 1)) { *abort_flag = 1; break; }
        ++it;
        tc_fence_after();
        for (int c0 = 0; c0 < cols; c0 += 64) {
          float f[64];
          load64(f, t_row + acc * kMaxBN + c0);
          send_dz(f, c0);
        }
        release(acc);
      } else {
        const int acc = it & 1;
        if (!mbar_wait(&tfull_bar[acc], (it >> 1) & 1)) { *abort_flag = 1; break; }
        ++it;
        tc_fence_after();
        const int box = w.dw && !p.dw_f32 ? 64 : 32;  // columns of 128 bytes
        for (int c0 = 0; c0 < cols; c0 += box) {
          uint4 out[8];
          if (w.dw && !p.dw_f32) {
            float f[64];
            load64(f, t_row + acc * kMaxBN + c0);
            if (p.dw_add && live) {  // one rounding of the sum: no bf16 reduction of a rounded tile
              const __nv_bfloat16* old = (const __nv_bfloat16*)p.dw + (size_t)row * p.cols + n0 + c0;
#pragma unroll
              for (int j = 0; j < 8; ++j)
                if (c0 + 8 * j < cols) {
                  const uint4 u = *reinterpret_cast<const uint4*>(old + 8 * j);
                  const __nv_bfloat162* o2 = reinterpret_cast<const __nv_bfloat162*>(&u);
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    const float2 o = __bfloat1622float2(o2[e]);
                    f[8 * j + 2 * e] += o.x;
                    f[8 * j + 2 * e + 1] += o.y;
                  }
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j)
              out[j] = make_uint4(pack_bf16(f[8 * j], f[8 * j + 1]), pack_bf16(f[8 * j + 2], f[8 * j + 3]),
                                  pack_bf16(f[8 * j + 4], f[8 * j + 5]), pack_bf16(f[8 * j + 6], f[8 * j + 7]));
            store(&maps.d2, out, n0 + c0, row0, false);
          } else {
            uint32_t r[32];
            tmem_ld32(t_row + acc * kMaxBN + c0, r);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 8; ++j) out[j] = make_uint4(r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
            if (w.dw) store(&maps.d2, out, n0 + c0, row0, p.dw_add != 0);
            else store(&maps.d, out, n0 + c0, w.split * p.split_rows + row0, p.add != 0);
          }
        }
        release(acc);
      }
    }
    if (M != STATS && lane == 0) tma_store_wait_all<0>();
    __syncwarp();
  }

  tc_fence_before();
  cluster_sync();  // the peer's shared memory is no longer read by the leader's MMAs
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 2 * kMaxBN);
  }
}

// ---------------------------------------------------------------- few rows
// One or two rows are bound by reading W once. Fused multiply-adds keep up with
// that, and start and finish sooner than the tensor-core pipeline (a pass, us, this
// kernel / the 256-row tiles: T = 1, V = 151936, H = 5120: 255 / 300; T = 2: 310 / 300;
// T = 1, V = 32000, H = 256: 13.5 / 24; T = 2: 17.6 / 24; four rows here: 338 at H = 5120).
// A warp takes 4 vocabulary entries at a time, lanes stride H, x stays in
// shared memory; products and sums are fp32 (two per instruction).
constexpr int kFew = 2;
constexpr int kFewThreads = 512;
constexpr int kFewMaxH = 8192;

KORE_DEV void fold(float& m, float& s, float& u, float m2, float s2, float u2) {
  // parts (m, s, u); one whose logits are all -inf has m = -inf and s = u = 0 (or NaN)
  const float nm = fmaxf(m, m2);
  const float base = nm == -INFINITY ? 0.f : nm;
  const float d1 = m == -INFINITY ? 0.f : m - base, d2 = m2 == -INFINITY ? 0.f : m2 - base;
  const float c1 = ex2(d1), c2 = ex2(d2);
  u = c1 * (u + d1 * s) + c2 * (u2 + d2 * s2);
  s = c1 * s + c2 * s2;
  m = nm;
}

KORE_DEV uint64_t bf2_to_f2(uint32_t v) {
  return f2_pack(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}

template <int NT>
__global__ void __launch_bounds__(kFewThreads) few_rows_kernel(const __nv_bfloat16* x, long ldx,
                                                               const __nv_bfloat16* w, long ldw,
                                                               const Params p) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  uint4* sx = reinterpret_cast<uint4*>(smem_raw);  // [NT][H / 8]
  __shared__ float s_part[kFewThreads / 32][4][NT][3];
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  const int T = p.rows, V = p.cols, nvec = p.K / 8;
  pdl_wait();
  pdl_trigger();
  for (int i = threadIdx.x; i < NT * nvec; i += kFewThreads) {
    const int t = i / nvec, j = i - t * nvec;
    sx[i] = t < T ? reinterpret_cast<const uint4*>(x + t * ldx)[j] : make_uint4(0, 0, 0, 0);
  }
  int tgt[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const long y = p.targets != nullptr && t < T ? p.targets[t] : -1;
    tgt[t] = y >= 0 && y < V ? (int)y : -1;
  }
  float m[NT], s[NT], u[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    m[t] = -INFINITY;
    s[t] = u[t] = 0.f;
  }
  __syncthreads();
  const int warps = kFewThreads / 32;
  const int mine = (lane >> 4) + 2 * ((lane >> 3) & 1);  // the entry whose sum this lane ends up with
  for (int r0 = ((int)blockIdx.x * warps + warp) * 4; r0 < V; r0 += (int)gridDim.x * warps * 4) {
    uint64_t acc[4][NT];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[r][t] = 0;
#pragma unroll 2
    for (int j = lane; j < nvec; j += 32) {
      uint4 wv[4];
#pragma unroll
      for (int r = 0; r < 4; ++r)
        wv[r] = r0 + r < V ? load_once(reinterpret_cast<const uint4*>(w + (r0 + r) * ldw) + j) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const uint4 xv = sx[t * nvec + j];
        const uint64_t x0 = bf2_to_f2(xv.x), x1 = bf2_to_f2(xv.y), x2 = bf2_to_f2(xv.z), x3 = bf2_to_f2(xv.w);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          acc[r][t] = f2_fma(bf2_to_f2(wv[r].x), x0, acc[r][t]);
          acc[r][t] = f2_fma(bf2_to_f2(wv[r].y), x1, acc[r][t]);
          acc[r][t] = f2_fma(bf2_to_f2(wv[r].z), x2, acc[r][t]);
          acc[r][t] = f2_fma(bf2_to_f2(wv[r].w), x3, acc[r][t]);
        }
      }
    }
    const int v = r0 + mine;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float z[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float hi;
        f2_unpack(acc[r][t], z[r], hi);
        z[r] += hi;
      }
      // four sums over 32 lanes: halve the number of sums, then of lanes
      float a = (lane & 16) ? z[1] : z[0], b = (lane & 16) ? z[3] : z[2];
      a += __shfl_xor_sync(0xffffffff, (lane & 16) ? z[0] : z[1], 16);
      b += __shfl_xor_sync(0xffffffff, (lane & 16) ? z[2] : z[3], 16);
      float c = (lane & 8) ? b : a;
      c += __shfl_xor_sync(0xffffffff, (lane & 8) ? a : b, 8);
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) c += __shfl_xor_sync(0xffffffff, c, o);
      if (v < V) {
        c *= p.scale;
        if (v == tgt[t] && (lane & 7) == 0) p.zt[t] = c;
        // one more logit: m is its own maximum, s = 1, u = 0 (of a NaN: s = NaN)
        if (c == -INFINITY) continue;
        fold(m[t], s[t], u[t], c, c == c ? 1.f : c, 0.f);
      }
    }
  }
  // the 4 streams of each warp, then the warps
  if ((lane & 7) == 0)
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      s_part[warp][mine][t][0] = m[t];
      s_part[warp][mine][t][1] = s[t];
      s_part[warp][mine][t][2] = u[t];
    }
  __syncthreads();
  if (warp < NT && warp < T) {  // warp t joins row t: lanes over the 4 * warps streams
    float fm = -INFINITY, fs = 0.f, fu = 0.f;
    for (int i = lane; i < 4 * warps; i += 32) {
      const float* q = s_part[i >> 2][i & 3][warp];
      fold(fm, fs, fu, q[0], q[1], q[2]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float m2 = __shfl_xor_sync(0xffffffff, fm, o);
      const float s2 = __shfl_xor_sync(0xffffffff, fs, o);
      const float u2 = __shfl_xor_sync(0xffffffff, fu, o);
      fold(fm, fs, fu, m2, s2, u2);
    }
    if (lane == 0) {
      const size_t o = (size_t)blockIdx.x * T + warp, plane = (size_t)gridDim.x * T;
      p.stats[o] = fm;
      p.stats[o + plane] = fs;
      if (p.entropy) p.stats[o + 2 * plane] = fu;
    }
  }
}

// Joins the parts (half tiles, or blocks of few_rows_kernel) of each row: 32 rows per block, 32 threads per row.
__global__ void __launch_bounds__(1024) head_join_kernel(
    const float* stats, const float* zt, const long* targets, int parts,
    int T, int V, float* __restrict__ logp, float* __restrict__ ent, float* __restrict__ lse) {
  __shared__ float sm[32][33], ss[32][33], su[32][33];
  pdl_wait();
  const int r = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int row = blockIdx.x * 32 + r;
  const size_t plane = (size_t)parts * T;
  float m = -INFINITY, s = 0.f, u = 0.f;
  if (row < T)
    for (int i = g; i < parts; i += 32) {
      const size_t o = (size_t)i * T + row;
      fold(m, s, u, stats[o], stats[o + plane], ent != nullptr ? stats[o + 2 * plane] : 0.f);
    }
  sm[g][r] = m;
  ss[g][r] = s;
  su[g][r] = u;
  __syncthreads();
  // warp g finishes row g: lane r holds part r
  m = sm[r][g];
  s = ss[r][g];
  u = su[r][g];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffff, m, o);
    const float s2 = __shfl_xor_sync(0xffffffff, s, o);
    const float u2 = __shfl_xor_sync(0xffffffff, u, o);
    fold(m, s, u, m2, s2, u2);
  }
  const int out = blockIdx.x * 32 + g;
  if (r == 0 && out < T) {
    const float ls = log2f(s), l = (m + ls) * kLn2;
    lse[out] = l;
    if (ent != nullptr) ent[out] = (ls - u / s) * kLn2;
    if (logp != nullptr) {
      const long y = targets[out];
      logp[out] = y >= 0 && y < V ? zt[out] * kLn2 - l : 0.f;
    }
  }
}

// out = x with the rows of coefficient 0 set to zero, once or twice (8 elements per thread)
__global__ void mask_rows_kernel(const __nv_bfloat16* x, long ldx, const float* coef,
                                 __nv_bfloat16* __restrict__ out, int T, int H, int copies) {
  pdl_wait();
  pdl_trigger();
  const int nvec = H / 8;
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < (long)T * nvec; i += (long)gridDim.x * blockDim.x) {
    const long t = i / nvec;
    const int j = (int)(i - t * nvec) * 8;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (coef[t] != 0.f) v = *reinterpret_cast<const uint4*>(x + t * ldx + j);
    *reinterpret_cast<uint4*>(out + t * H + j) = v;
    if (copies == 2) *reinterpret_cast<uint4*>(out + (T + t) * H + j) = v;
  }
}

// dx = the sum of the K parts (and of dz's two terms, T rows apart), rounded once
__global__ void sum_parts_kernel(const float* src, int parts, int copies, long part_stride,
                                 __nv_bfloat16* __restrict__ dst, long ld, int T, int H) {
  pdl_wait();
  pdl_trigger();
  const int nvec = H / 8;
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < (long)T * nvec; i += (long)gridDim.x * blockDim.x) {
    const long t = i / nvec;
    const int j = (int)(i - t * nvec) * 8;
    float f[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int s = 0; s < parts * copies; ++s) {
      const float* r = src + (s / copies) * part_stride + (s % copies) * (long)T * H + i * 8;
      const float4 a = *reinterpret_cast<const float4*>(r), b = *reinterpret_cast<const float4*>(r + 4);
      f[0] += a.x; f[1] += a.y; f[2] += a.z; f[3] += a.w;
      f[4] += b.x; f[5] += b.y; f[6] += b.z; f[7] += b.w;
    }
    *reinterpret_cast<uint4*>(dst + t * ld + j) =
        make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
  }
}

template <Mode M>
void launch(const Maps& maps, const Params& p, int dev, cudaStream_t st) {
  static bool attr_set[64] = {};
  TORCH_CHECK(dev >= 0 && dev < 64, "head: device index");
  auto k = head_kernel<M>;
  constexpr int smem = Layout<M>::kSmem;
  if (!attr_set[dev]) {
    check_cuda(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem),
               "cudaFuncSetAttribute(head smem)");
    attr_set[dev] = true;
  }
  const long num_n = (p.cols + p.bn - 1) / p.bn;
  long items = (long)((p.rows + 2 * BM - 1) / (2 * BM)) * num_n * p.splits;
  if (M == PRODS) items += (long)((p.K + 2 * BM - 1) / (2 * BM)) * num_n;
  const int grid = (int)std::min<long>(2 * items, num_sms(dev) & ~1);
  launch_after("head launch", k, dim3(grid), dim3(kThreads), (size_t)smem, st, maps, p);
}

template <int NT>
void launch_few(const __nv_bfloat16* x, long ldx, const __nv_bfloat16* w, long ldw, const Params& p, int blocks,
                int dev, cudaStream_t st) {
  static bool attr_set[64] = {};
  TORCH_CHECK(dev >= 0 && dev < 64, "head: device index");
  auto k = few_rows_kernel<NT>;
  if (!attr_set[dev]) {
    check_cuda(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, NT * kFewMaxH * 2),
               "cudaFuncSetAttribute(head few rows smem)");
    attr_set[dev] = true;
  }
  launch_after("head few rows", k, dim3(blocks), dim3(kFewThreads), (size_t)NT * p.K * 2, st, x, ldx, w, ldw, p);
}

// Parts of dx's contraction (the piece's vocabulary): as many as fill the pairs
// when T x H has few tiles; each part costs a pass over [T, H] in fp32. In units
// of one k-block of a tile (0.27 us at the nominal rate, 0.37 at the 720 clocks it
// takes): 1.5 MB of HBM traffic.
int pick_splits(long tiles, long kblocks, long dx_elems, int pairs) {
  int best = 1;
  double best_cost = -1;
  for (int s = 1; s <= 32 && s <= (kblocks + 3) / 4; ++s) {
    const double cost = (double)((tiles * s + pairs - 1) / pairs) * ((kblocks + s - 1) / s) + dx_elems * 8e-6 / 1.5 * s;
    if (best_cost < 0 || cost < best_cost) { best_cost = cost; best = s; }
  }
  return best;
}

// Tile width of the forward. The pairs of a wave stop together, so a narrower
// tile can leave less idle in the last wave, but reads x from shared memory and
// the accumulator out more often: about 68 columns' time per tile (T = 1003,
// V = 151936, H = 5120: 33 waves of 256 columns 1.33 ms, 40 of 208 1.37 ms; T = 8192:
// 257 of 256 10.6 ms, 411 of 160 12.0 ms).
int pick_bn(long num_m, long V, int pairs) {
  int best = 256;
  long best_cost = -1;
  for (int bn = 256; bn >= 128; bn -= 16) {
    const long tiles = num_m * ((V + bn - 1) / bn);
    const long cost = ((tiles + pairs - 1) / pairs) * (bn + 68);
    if (best_cost < 0 || cost < best_cost) { best_cost = cost; best = bn; }
  }
  return best;
}

void check_operands(const at::Tensor& x, const at::Tensor& w, const c10::optional<at::Tensor>& targets,
                    double inv_temp) {
  TORCH_CHECK(x.is_cuda() && w.is_cuda() && x.device() == w.device(), "head: x and w must be on one CUDA device");
  TORCH_CHECK(x.dim() == 2 && w.dim() == 2 && x.scalar_type() == at::kBFloat16 && w.scalar_type() == at::kBFloat16,
              "head: x [T, H] and w [V, H] must be bf16");
  TORCH_CHECK(x.size(1) == w.size(1), "head: x and w differ in H");
  TORCH_CHECK(w.size(0) >= 1 && x.size(1) >= 8 && x.size(1) % 8 == 0, "head: V >= 1 and H a positive multiple of 8");
  TORCH_CHECK(x.size(0) < (1 << 30) && w.size(0) < (1 << 30), "head: T and V must be below 2^30");
  TORCH_CHECK(x.stride(1) == 1 && w.stride(1) == 1 && (x.size(0) <= 1 || x.stride(0) % 8 == 0) &&
                  (w.size(0) <= 1 || w.stride(0) % 8 == 0),
              "head: rows must be contiguous and 16-byte aligned");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0 && reinterpret_cast<uintptr_t>(w.data_ptr()) % 16 == 0,
              "head: x and w must start on 16 bytes");
  TORCH_CHECK(std::isfinite(inv_temp) && inv_temp > 0, "head: temperature must be positive and finite");
  if (targets)
    TORCH_CHECK(targets->device() == x.device() && targets->scalar_type() == at::kLong && targets->dim() == 1 &&
                    targets->size(0) == x.size(0) && targets->is_contiguous(),
                "head: targets must be int64 [T]");
}

void check_rows(const at::Tensor& t, const at::Tensor& x, const char* name) {
  TORCH_CHECK(t.device() == x.device() && t.scalar_type() == at::kFloat && t.dim() == 1 && t.size(0) == x.size(0) &&
                  t.is_contiguous(),
              "head: ", name, " must be fp32 [T]");
}

int64_t row_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

}  // namespace head

// Returns (logp if there are targets, entropy if wanted, lse).
std::tuple<c10::optional<at::Tensor>, c10::optional<at::Tensor>, at::Tensor> head_fwd(
    const at::Tensor& x, const at::Tensor& w, const c10::optional<at::Tensor>& targets, double inv_temp,
    bool want_entropy) {
  using namespace head;
  check_operands(x, w, targets, inv_temp);
  const int T = x.size(0), V = w.size(0), H = x.size(1);
  c10::cuda::CUDAGuard g(x.device());
  const auto f32 = x.options().dtype(at::kFloat);
  at::Tensor lse = at::empty({T}, f32);
  c10::optional<at::Tensor> logp, entropy;
  if (targets) logp = at::empty({T}, f32);
  if (want_entropy) entropy = at::empty({T}, f32);
  if (T == 0) return {logp, entropy, lse};
  const int dev = x.get_device();
  auto st = at::cuda::getCurrentCUDAStream();
  Params p = {};
  p.cols = V; p.K = H; p.splits = 1;
  p.scale = (float)(inv_temp * 1.4426950408889634);
  p.inv_temp = (float)inv_temp;
  p.entropy = entropy.has_value();
  const int block = std::min(T, kRowBlock), sms = num_sms(dev);
  const bool few = T <= kFew && H <= kFewMaxH;
  p.bn = pick_bn((block + 2 * BM - 1) / (2 * BM), V, sms / 2);
  const int few_blocks = std::min((V + kFewThreads / 8 - 1) / (kFewThreads / 8), 2 * sms);
  const int parts = few ? few_blocks : 2 * ((V + p.bn - 1) / p.bn);
  at::Tensor ws = at::empty({((int64_t)parts * (p.entropy ? 3 : 2) + 1) * block}, f32);
  auto bf = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  for (int t0 = 0; t0 < T; t0 += kRowBlock) {
    p.rows = std::min(T - t0, kRowBlock);
    p.zt = ws.data_ptr<float>();
    p.stats = p.zt + p.rows;
    p.targets = logp ? targets->data_ptr<long>() + t0 : nullptr;
    const __nv_bfloat16* xp = (const __nv_bfloat16*)x.data_ptr() + t0 * row_stride(x);
    if (few) {
      const __nv_bfloat16* wp = (const __nv_bfloat16*)w.data_ptr();
      if (T == 1) launch_few<1>(xp, row_stride(x), wp, row_stride(w), p, few_blocks, dev, st);
      else launch_few<2>(xp, row_stride(x), wp, row_stride(w), p, few_blocks, dev, st);
    } else {
      Maps maps = {};
      maps.a = make_tmap_2d(xp, bf, 2, H, p.rows, row_stride(x), BK, BM);
      maps.b = make_tmap_2d(w.data_ptr(), bf, 2, H, V, row_stride(w), BK, p.bn / 2);
      launch<STATS>(maps, p, dev, st);
    }
    launch_after("head join", head_join_kernel, dim3((p.rows + 31) / 32), dim3(1024), 0, st, p.stats, p.zt, p.targets,
                 parts, p.rows, V, logp ? logp->data_ptr<float>() + t0 : nullptr,
                 entropy ? entropy->data_ptr<float>() + t0 : nullptr, lse.data_ptr<float>() + t0);
  }
  return {logp, entropy, lse};
}

// Returns dx (into `into` when it is given).
at::Tensor head_bwd(const at::Tensor& x, const at::Tensor& w, const c10::optional<at::Tensor>& targets,
                    const at::Tensor& lse, const at::Tensor& coef, double inv_temp,
                    const c10::optional<at::Tensor>& into, at::Tensor& dw, bool accumulate, int64_t piece) {
  using namespace head;
  check_operands(x, w, targets, inv_temp);
  check_rows(lse, x, "lse");
  check_rows(coef, x, "coef");
  const int T = x.size(0), V = w.size(0), H = x.size(1);
  if (into)
    TORCH_CHECK(into->device() == x.device() && into->scalar_type() == at::kBFloat16 && into->dim() == 2 &&
                    into->size(0) == T && into->size(1) == H && into->stride(1) == 1 &&
                    (T <= 1 || into->stride(0) % 8 == 0) && reinterpret_cast<uintptr_t>(into->data_ptr()) % 16 == 0,
                "head: dx must be bf16 [T, H] with contiguous, 16-byte aligned rows");
  const bool f32 = dw.scalar_type() == at::kFloat;
  TORCH_CHECK(dw.device() == x.device() && (f32 || dw.scalar_type() == at::kBFloat16) && dw.dim() == 2 &&
                  dw.size(0) == V && dw.size(1) == H && dw.is_contiguous() &&
                  reinterpret_cast<uintptr_t>(dw.data_ptr()) % 16 == 0,
              "head: dw must be contiguous bf16 or fp32 [V, H] on 16 bytes");
  TORCH_CHECK(piece >= 0, "head: piece must not be negative");
  c10::cuda::CUDAGuard g(x.device());
  at::Tensor dx = into ? *into : at::empty({T, H}, x.options());
  if (T == 0) {
    if (!accumulate) dw.zero_();
    return dx;
  }
  const int dev = x.get_device(), sms = num_sms(dev);
  auto st = at::cuda::getCurrentCUDAStream();
  // dz of one piece is the only workspace as wide as the vocabulary: about 256 MB
  // by default, in equal pieces of whole tiles
  int64_t width = piece;
  if (width == 0) width = std::max<int64_t>(4096, (int64_t(128) << 20) / T);
  const int64_t n_pieces = (V + width - 1) / width;
  if (piece == 0) width = ((V + n_pieces - 1) / n_pieces + kMaxBN - 1) / kMaxBN * kMaxBN;
  width = std::min<int64_t>((width + 7) / 8 * 8, ((int64_t)V + 7) / 8 * 8);
  // up to kTwoTerms rows dz is held as two bf16 terms, 2 T rows in all
  const int copies = T <= kTwoTerms ? 2 : 1, R = T * copies, r32 = (R + 31) / 32 * 32;
  const int splits = pick_splits((long)((R + 2 * BM - 1) / (2 * BM)) * ((H + kMaxBN - 1) / kMaxBN),
                                 (std::min<int64_t>(width, V) + BK - 1) / BK, (long)R * H, sms / 2);
  // workspace: dx parts fp32 [splits r32, H], dz bf16 [R, width], masked x bf16 [R, H]
  const int64_t acc_bytes = (int64_t)splits * r32 * H * 4, dz_bytes = ((int64_t)R * width * 2 + 127) / 128 * 128;
  at::Tensor ws = at::empty({acc_bytes + dz_bytes + (int64_t)R * H * 2}, x.options().dtype(at::kByte));
  float* acc = reinterpret_cast<float*>(ws.data_ptr());
  __nv_bfloat16* dz = reinterpret_cast<__nv_bfloat16*>((uint8_t*)ws.data_ptr() + acc_bytes);
  __nv_bfloat16* xm = reinterpret_cast<__nv_bfloat16*>((uint8_t*)ws.data_ptr() + acc_bytes + dz_bytes);
  const long nvec = (long)T * H / 8;
  const int grid = (int)std::min<long>((nvec + 255) / 256, (long)sms * 8);
  launch_after("head mask rows", mask_rows_kernel, dim3(grid), dim3(256), 0, st, (const __nv_bfloat16*)x.data_ptr(),
               row_stride(x), coef.data_ptr<float>(), xm, T, H, copies);
  const auto bf = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, ff = CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
  Maps grad = {}, prods = {};
  grad.a = make_tmap_2d(x.data_ptr(), bf, 2, H, T, row_stride(x), BK, BM);
  prods.d = make_tmap_2d(acc, ff, 4, H, (uint64_t)splits * r32, H, 32, 32);
  prods.b2 = make_tmap_2d(xm, bf, 2, H, R, H, 64, BK);
  Params p = {};
  p.rows = T; p.K = H;
  p.bn = kMaxBN;
  p.splits = 1;
  p.scale = (float)(inv_temp * 1.4426950408889634);
  p.inv_temp = (float)inv_temp;
  p.targets = targets ? targets->data_ptr<long>() : nullptr;
  p.lse = lse.data_ptr<float>();
  p.coef = coef.data_ptr<float>();
  p.low = copies == 2 ? dz + (long)T * width : nullptr;
  p.low_ld = width;
  Params d = {};
  d.rows = R; d.cols = H;
  d.bn = kMaxBN;
  d.splits = splits;
  d.split_rows = r32;
  d.dw_f32 = f32;
  d.dw_add = accumulate;
  for (int64_t v0 = 0; v0 < V; v0 += width) {
    const int n = (int)std::min<int64_t>(width, V - v0);
    const __nv_bfloat16* wp = (const __nv_bfloat16*)w.data_ptr() + v0 * row_stride(w);
    p.cols = n;
    p.v0 = (int)v0;
    grad.b = make_tmap_2d(wp, bf, 2, H, n, row_stride(w), BK, kMaxBN / 2);
    grad.d = make_tmap_2d(dz, bf, 2, (n + 7) / 8 * 8, T, width, 64, 32);
    if (k_parts((H + BK - 1) / BK) == 1) launch<GRAD>(grad, p, dev, st);
    else launch<GRADK>(grad, p, dev, st);
    d.K = n;
    d.add = v0 > 0;
    d.dw = (uint8_t*)dw.data_ptr() + v0 * H * (f32 ? 4 : 2);
    prods.a = make_tmap_2d(dz, bf, 2, n, R, width, BK, BM);
    prods.b = make_tmap_2d(wp, bf, 2, H, n, row_stride(w), 64, BK);
    prods.a2 = make_tmap_2d(dz, bf, 2, n, R, width, 64, BK);
    prods.d2 = f32 ? make_tmap_2d(d.dw, ff, 4, H, n, H, 32, 32) : make_tmap_2d(d.dw, bf, 2, H, n, H, 64, 32);
    launch<PRODS>(prods, d, dev, st);
  }
  launch_after("head sum parts", sum_parts_kernel, dim3(grid), dim3(256), 0, st, (const float*)acc, splits, copies,
               (long)r32 * H, (__nv_bfloat16*)dx.data_ptr(), row_stride(dx), T, H);
  return dx;
}

}  // namespace kore
