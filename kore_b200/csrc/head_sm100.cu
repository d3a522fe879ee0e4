// Language-model head in pieces of the vocabulary, without keeping logits.
//
//   z_tj  = (x_t . W_j) / tau                       x [T, H], W [V, H] bf16
//   lse_t = log sum_j e^{z_tj},  logp_t = z_{t,y_t} - lse_t
//   ent_t = lse_t - sum_j p_tj z_tj,  p_tj = e^{z_tj - lse_t}
//   L = sum_t c_t logp_t:  dz_tj = (c_t / tau) (1[j = y_t] - p_tj)
//                          dx = dz W,  dW = dz^T x
//
// Forward: a 2-CTA tcgen05 GEMM whose epilogue never writes z. Each thread owns
// one row of a tile in TMEM and folds its columns into a running triple
// (m = max, s = sum e^{z-m}, u = sum (z-m) e^{z-m}; ent = log s - u / s, which
// does not cancel when the logits are large); one triple per (tile, row) goes
// to a workspace, and a second kernel joins the tiles of a row. The logit of
// the label is written by the one tile that holds it. Logits stay fp32 from
// the accumulator on.
// Backward: per piece of the vocabulary the same GEMM runs again and its
// epilogue turns z into dz (bf16, the operand type of the two products that
// follow: its rounding, at most 2^-8 of a value, is of the size of the rounding
// of dx and dW themselves); then dW[piece] = dz^T x and dx += dz W[piece] run on the
// plain GEMM. dW rows are final after their piece (one rounding); dx sums its
// pieces in fp32 and is rounded once.
// Rows with coefficient 0 have dz = 0 whatever x or the statistics hold there,
// and dW reads such rows of x as zeros, so an inf or NaN in them stays out.
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

void gemm_bf16(const at::Tensor& a, const at::Tensor& b, at::Tensor& out, bool a_mn, bool b_mn,
               double alpha, bool accumulate, const c10::optional<at::Tensor>& residual,
               int64_t max_ctas);

namespace head {

constexpr int BM = 128;        // rows per CTA (256 per pair)
constexpr int BK = 64;
constexpr int kMaxBN = 256;    // vocabulary columns of a pair's tile
constexpr int kThreads = 192;  // TMA producer, MMA issuer, 4 epilogue warps
constexpr int kEpiWarps = 4;
constexpr int kStages = 6;
constexpr int kABytes = BM * BK * 2;
constexpr int kBBytes = (kMaxBN / 2) * BK * 2;
constexpr int kStageBytes = kABytes + kBBytes;
constexpr int kStoreBytes = 32 * 128;  // one store box: 32 rows x 64 bf16
constexpr int kEpiOff = kStages * kStageBytes;
constexpr int kBarOff = kEpiOff + kEpiWarps * 2 * kStoreBytes;
constexpr int kSmem = kBarOff + 256 + 1024;
constexpr int kRowBlock = 32768;       // rows per forward launch: bounds the statistics workspace
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct Params {
  int T, V, H;          // rows, columns of this launch's W, contraction
  int bn;               // columns per tile (multiple of 16, <= 256)
  int v0;               // vocabulary id of column 0
  float scale;          // log2(e) / tau: epilogue works in powers of two
  float inv_temp;
  const long* targets;  // may be null
  // statistics
  float* stats;         // [planes][num_n][T]: m, s, (u)
  float* zt;            // [T] label logit in units of log2
  int entropy;
  // gradient
  const float* lse;
  const float* coef;
};

KORE_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// groups of 8 row blocks walk the vocabulary together, so a W tile is read
// from HBM once per 2048 rows and the group's x rows stay in L2
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

template <bool GRAD>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    head_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW,
                const __grid_constant__ CUtensorMap tmD, const Params p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + kBarOff);
  uint64_t* empty_bar = full_bar + kStages;
  uint64_t* tfull_bar = empty_bar + kStages;  // [2]
  uint64_t* tempty_bar = tfull_bar + 2;       // [2] (leader: both CTAs' epilogue warps arrive)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty_bar + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int pair = blockIdx.x / 2, npairs = gridDim.x / 2;
  const int bn = p.bn;
  const int num_m = (p.T + 2 * BM - 1) / (2 * BM);
  const int num_n = (p.V + bn - 1) / bn;
  const int num_tiles = num_m * num_n;
  const int kblocks = (p.H + BK - 1) / BK;

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
    tma_prefetch_desc(&tmX);
    tma_prefetch_desc(&tmW);
    if (GRAD) tma_prefetch_desc(&tmD);
  }
  if (warp == 1) tmem_alloc_pair(tmem_slot, 2 * kMaxBN);
  tc_fence_before();
  cluster_sync();  // both CTAs' barriers initialised and TMEM allocated
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    // ------------------------------------------------------------ producer (both CTAs)
    if (elect_one()) {
      const uint32_t b_box = (uint32_t)(bn / 2) * BK * 2;
      int stage = 0;
      uint32_t phase = 0;
      for (int t = pair; t < num_tiles && !*abort_flag; t += npairs) {
        int tm, tn;
        tile_coords(t, num_m, num_n, tm, tn);
        const int m0 = tm * 2 * BM, n0 = tn * bn;
        // a box that lies wholly past the rows or the vocabulary is not loaded
        // (its part of the accumulator is never used)
        const bool a1 = m0 + BM < p.T, b1 = n0 + bn / 2 < p.V;
        const uint32_t bytes = kABytes * (a1 ? 2 : 1) + b_box * (b1 ? 2 : 1);
        const bool load_a = rank == 0 || a1, load_b = rank == 0 || b1;
        for (int kb = 0; kb < kblocks; ++kb) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1)) { *abort_flag = 1; break; }
          uint8_t* sA = smem + stage * kStageBytes;
          const uint32_t fb = mapa_shared(smem_u32(&full_bar[stage]), 0);
          if (rank == 0) mbar_arrive_expect_tx(&full_bar[stage], bytes);
          if (load_a) tma_load_2d_pair(sA, &tmX, fb, kb * BK, m0 + (int)rank * BM);
          if (load_b) tma_load_2d_pair(sA + kABytes, &tmW, fb, kb * BK, n0 + (int)rank * (bn / 2));
          if (++stage == kStages) { stage = 0; phase ^= 1; }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (leader)
    if (rank == 0 && elect_one()) {
      const uint32_t idesc = make_idesc_bf16(2 * BM, bn, false, false);
      int stage = 0, it = 0;
      uint32_t phase = 0;
      for (int t = pair; t < num_tiles && !*abort_flag; t += npairs, ++it) {
        const int acc = it & 1;
        if (!mbar_wait(&tempty_bar[acc], ((it >> 1) & 1) ^ 1)) { *abort_flag = 1; break; }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * kMaxBN;
        bool ok = true;
        for (int kb = 0; kb < kblocks; ++kb) {
          if (!mbar_wait(&full_bar[stage], phase)) { ok = false; break; }
          tc_fence_after();
          const uint32_t a_addr = smem_u32(smem + stage * kStageBytes);
#pragma unroll
          for (int k = 0; k < BK / 16; ++k)
            umma_f16_ss_pair(d_tmem, make_sw128_desc(a_addr + k * 32, 16, 1024),
                             make_sw128_desc(a_addr + kABytes + k * 32, 16, 1024), idesc, (kb | k) != 0);
          umma_commit_pair(&empty_bar[stage], 0x3);
          if (++stage == kStages) { stage = 0; phase ^= 1; }
        }
        if (!ok) { *abort_flag = 1; break; }
        umma_commit_pair(&tfull_bar[acc], 0x3);
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ epilogue (both CTAs)
    const int q = warp & 3;  // TMEM lane quadrant this warp may access
    uint8_t* stage_buf = smem + kEpiOff + (warp - 2) * 2 * kStoreBytes;
    const uint32_t tempty_leader[2] = {mapa_shared(smem_u32(&tempty_bar[0]), 0),
                                       mapa_shared(smem_u32(&tempty_bar[1]), 0)};
    int buf = 0, it = 0;
    for (int t = pair; t < num_tiles && !*abort_flag; t += npairs, ++it) {
      int tm, tn;
      tile_coords(t, num_m, num_n, tm, tn);
      const int n0 = tn * bn;
      const int row0 = tm * 2 * BM + (int)rank * BM + q * 32;
      const int row = row0 + lane;
      const int cols = min(bn, p.V - n0);
      const int acc = it & 1;
      const bool live = row < p.T;
      // column of the label in this tile (outside [0, cols): not here)
      int tc = -1;
      float lse2 = 0.f, c = 0.f;
      if (live && p.targets != nullptr) {
        const long y = p.targets[row] - p.v0 - n0;
        if (y >= 0 && y < cols) tc = (int)y;
      }
      if (GRAD && live) {
        lse2 = p.lse[row] * kLog2e;
        c = p.coef[row] * p.inv_temp;
      }
      if (!mbar_wait(&tfull_bar[acc], (it >> 1) & 1)) { *abort_flag = 1; break; }
      tc_fence_after();
      const uint32_t t_row = tmem_base + ((uint32_t)(q * 32) << 16) + acc * kMaxBN;
      if (!GRAD) {
        float m = -INFINITY, s = 0.f, u = 0.f;
        if (row0 < p.T)
        for (int c0 = 0; c0 < cols; c0 += 32) {
          uint32_t r[32];
          tmem_ld32(t_row + c0, r);
          tmem_wait_ld();
          if (c0 + 32 > cols) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (c0 + i >= cols) r[i] = 0xff800000u;  // -inf: not a column of the vocabulary
          }
          const int ti = tc - c0;
          if (ti >= 0 && ti < 32) {
            float z = 0.f;
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (i == ti) z = __uint_as_float(r[i]);
            p.zt[row] = z * p.scale;
          }
          float cm = __uint_as_float(r[0]);
#pragma unroll
          for (int i = 1; i < 32; ++i) cm = fmaxf(cm, __uint_as_float(r[i]));
          const float nm = fmaxf(m, cm * p.scale);
          const float base = nm == -INFINITY ? 0.f : nm;  // all columns so far -inf: keep their terms 0
          const float d = m == -INFINITY ? 0.f : m - base;
          const float corr = ex2(d);
          u = corr * (u + d * s);
          s *= corr;
          m = nm;
          if (p.entropy) {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const float zr = fmaf(__uint_as_float(r[i]), p.scale, -base);
              const float e = ex2(zr);
              s += e;
              u += e == 0.f ? 0.f : e * zr;
            }
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) s += ex2(fmaf(__uint_as_float(r[i]), p.scale, -base));
          }
        }
        if (live) {
          const size_t o = (size_t)tn * p.T + row, plane = (size_t)num_n * p.T;
          p.stats[o] = m;
          p.stats[o + plane] = s;
          if (p.entropy) p.stats[o + 2 * plane] = u;
        }
      } else {
        if (row0 < p.T)
        for (int c0 = 0; c0 < cols; c0 += 64) {
          float v[64];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t r[32];
            tmem_ld32(t_row + c0 + 32 * h, r);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const float e = ex2(fmaf(__uint_as_float(r[i]), p.scale, -lse2));
              // coefficient 0, or past the piece's last column: 0
              v[32 * h + i] = c == 0.f || c0 + 32 * h + i >= cols ? 0.f : -c * e;
            }
          }
          const int ti = tc - c0;
          if (ti >= 0 && ti < 64) {
#pragma unroll
            for (int i = 0; i < 64; ++i)
              if (i == ti) v[i] += c;
          }
          if (lane == 0) tma_store_wait_read<1>();
          __syncwarp();
          uint8_t* sb = stage_buf + buf * kStoreBytes + lane * 128;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            *reinterpret_cast<uint4*>(sb + ((j ^ (lane & 7)) * 16)) =
                make_uint4(pack_bf16(v[8 * j], v[8 * j + 1]), pack_bf16(v[8 * j + 2], v[8 * j + 3]),
                           pack_bf16(v[8 * j + 4], v[8 * j + 5]), pack_bf16(v[8 * j + 6], v[8 * j + 7]));
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&tmD, stage_buf + buf * kStoreBytes, n0 + c0, row0);
            tma_store_commit();
          }
          buf ^= 1;
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(tempty_leader[acc]);
    }
    if (GRAD && lane == 0) tma_store_wait_all<0>();
    __syncwarp();
  }

  tc_fence_before();
  cluster_sync();  // the peer's shared memory is no longer read by the leader's MMAs
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 2 * kMaxBN);
  }
}

// Joins the tiles' triples of each row: 32 rows per block, 32 threads per row.
__global__ void __launch_bounds__(1024) head_join_kernel(
    const float* __restrict__ stats, const float* __restrict__ zt, const long* __restrict__ targets, int num_n,
    int T, int V, float* __restrict__ logp, float* __restrict__ ent, float* __restrict__ lse) {
  __shared__ float sm[32][33], ss[32][33], su[32][33];
  const int r = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int row = blockIdx.x * 32 + r;
  const size_t plane = (size_t)num_n * T;
  float m = -INFINITY, s = 0.f, u = 0.f;
  // a part whose logits are all -inf has m = -inf and s = u = 0 (or NaN)
  auto fold = [&](float m2, float s2, float u2) {
    const float nm = fmaxf(m, m2);
    const float base = nm == -INFINITY ? 0.f : nm;
    const float d1 = m == -INFINITY ? 0.f : m - base, d2 = m2 == -INFINITY ? 0.f : m2 - base;
    const float c1 = ex2(d1), c2 = ex2(d2);
    u = c1 * (u + d1 * s) + c2 * (u2 + d2 * s2);
    s = c1 * s + c2 * s2;
    m = nm;
  };
  if (row < T)
    for (int i = g; i < num_n; i += 32) {
      const size_t o = (size_t)i * T + row;
      fold(stats[o], stats[o + plane], ent != nullptr ? stats[o + 2 * plane] : 0.f);
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
    fold(m2, s2, u2);
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

// out = x with the rows of coefficient 0 set to zero (8 elements per thread)
__global__ void mask_rows_kernel(const __nv_bfloat16* __restrict__ x, long ldx, const float* __restrict__ coef,
                                 __nv_bfloat16* __restrict__ out, int T, int H) {
  const int nvec = H / 8;
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < (long)T * nvec; i += (long)gridDim.x * blockDim.x) {
    const long t = i / nvec;
    const int j = (int)(i - t * nvec) * 8;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (coef[t] != 0.f) v = *reinterpret_cast<const uint4*>(x + t * ldx + j);
    *reinterpret_cast<uint4*>(out + t * H + j) = v;
  }
}

__global__ void round_kernel(const float* __restrict__ src, __nv_bfloat16* __restrict__ dst, long ld, int T, int H) {
  const int nvec = H / 8;
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < (long)T * nvec; i += (long)gridDim.x * blockDim.x) {
    const long t = i / nvec;
    const int j = (int)(i - t * nvec) * 8;
    const float4 a = *reinterpret_cast<const float4*>(src + t * H + j);
    const float4 b = *reinterpret_cast<const float4*>(src + t * H + j + 4);
    *reinterpret_cast<uint4*>(dst + t * ld + j) =
        make_uint4(pack_bf16(a.x, a.y), pack_bf16(a.z, a.w), pack_bf16(b.x, b.y), pack_bf16(b.z, b.w));
  }
}

template <bool GRAD>
void launch(const CUtensorMap& tx, const CUtensorMap& tw, const CUtensorMap& td, const Params& p, int dev,
            cudaStream_t st) {
  static bool attr_set[64] = {};
  TORCH_CHECK(dev >= 0 && dev < 64, "head: device index");
  auto k = head_kernel<GRAD>;
  if (!attr_set[dev]) {
    check_cuda(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem),
               "cudaFuncSetAttribute(head smem)");
    attr_set[dev] = true;
  }
  const long tiles = (long)((p.T + 2 * BM - 1) / (2 * BM)) * ((p.V + p.bn - 1) / p.bn);
  const int grid = (int)std::min<long>(2 * tiles, num_sms(dev) & ~1);
  k<<<grid, kThreads, kSmem, st>>>(tx, tw, td, p);
  check_cuda(cudaGetLastError(), "head launch");
}

// Tile width of the forward: the pairs of a wave stop together, so the width is
// the multiple of 16 that leaves the least work in the last wave (ties: wider,
// which reads x from shared memory less often).
int pick_bn(long num_m, long V, int pairs) {
  int best = 256;
  long best_cost = -1;
  for (int bn = 256; bn >= 128; bn -= 16) {
    const long tiles = num_m * ((V + bn - 1) / bn);
    const long cost = ((tiles + pairs - 1) / pairs) * bn;
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

void head_fwd(const at::Tensor& x, const at::Tensor& w, const c10::optional<at::Tensor>& targets, double inv_temp,
              const c10::optional<at::Tensor>& logp, const c10::optional<at::Tensor>& entropy, at::Tensor& lse) {
  using namespace head;
  check_operands(x, w, targets, inv_temp);
  check_rows(lse, x, "lse");
  if (logp) {
    check_rows(*logp, x, "logp");
    TORCH_CHECK(targets.has_value(), "head: logp needs targets");
  }
  if (entropy) check_rows(*entropy, x, "entropy");
  const int T = x.size(0), V = w.size(0), H = x.size(1);
  if (T == 0) return;
  c10::cuda::CUDAGuard g(x.device());
  const int dev = x.get_device();
  auto st = at::cuda::getCurrentCUDAStream();
  Params p = {};
  p.V = V; p.H = H;
  p.bn = pick_bn((std::min(T, kRowBlock) + 2 * BM - 1) / (2 * BM), V, num_sms(dev) / 2);
  p.scale = (float)(inv_temp * 1.4426950408889634);
  p.inv_temp = (float)inv_temp;
  p.entropy = entropy.has_value();
  const int num_n = (V + p.bn - 1) / p.bn;
  auto bf = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  CUtensorMap tw = make_tmap_2d(w.data_ptr(), bf, 2, H, V, row_stride(w), BK, p.bn / 2);
  at::Tensor ws = at::empty({((int64_t)num_n * (p.entropy ? 3 : 2) + 1) * std::min(T, kRowBlock)},
                            x.options().dtype(at::kFloat));
  for (int t0 = 0; t0 < T; t0 += kRowBlock) {
    p.T = std::min(T - t0, kRowBlock);
    p.zt = ws.data_ptr<float>();
    p.stats = p.zt + p.T;
    p.targets = logp ? targets->data_ptr<long>() + t0 : nullptr;
    CUtensorMap tx = make_tmap_2d((const __nv_bfloat16*)x.data_ptr() + t0 * row_stride(x), bf, 2, H, p.T,
                                  row_stride(x), BK, BM);
    launch<false>(tx, tw, tx, p, dev, st);
    head_join_kernel<<<(p.T + 31) / 32, 1024, 0, st>>>(
        p.stats, p.zt, p.targets, num_n, p.T, V, logp ? logp->data_ptr<float>() + t0 : nullptr,
        entropy ? entropy->data_ptr<float>() + t0 : nullptr, lse.data_ptr<float>() + t0);
    check_cuda(cudaGetLastError(), "head join");
  }
}

void head_bwd(const at::Tensor& x, const at::Tensor& w, const c10::optional<at::Tensor>& targets,
              const at::Tensor& lse, const at::Tensor& coef, double inv_temp, at::Tensor& dx, at::Tensor& dw,
              bool accumulate, int64_t piece) {
  using namespace head;
  check_operands(x, w, targets, inv_temp);
  check_rows(lse, x, "lse");
  check_rows(coef, x, "coef");
  const int T = x.size(0), V = w.size(0), H = x.size(1);
  TORCH_CHECK(dx.device() == x.device() && dx.scalar_type() == at::kBFloat16 && dx.dim() == 2 && dx.size(0) == T &&
                  dx.size(1) == H && dx.stride(1) == 1 && (T <= 1 || dx.stride(0) % 8 == 0) &&
                  reinterpret_cast<uintptr_t>(dx.data_ptr()) % 16 == 0,
              "head: dx must be bf16 [T, H] with contiguous, 16-byte aligned rows");
  TORCH_CHECK(dw.device() == x.device() && (dw.scalar_type() == at::kBFloat16 || dw.scalar_type() == at::kFloat) &&
                  dw.dim() == 2 && dw.size(0) == V && dw.size(1) == H && dw.is_contiguous() &&
                  reinterpret_cast<uintptr_t>(dw.data_ptr()) % 16 == 0,
              "head: dw must be contiguous bf16 or fp32 [V, H] on 16 bytes");
  TORCH_CHECK(piece >= 0, "head: piece must not be negative");
  if (T == 0) {
    if (!accumulate) dw.zero_();
    return;
  }
  c10::cuda::CUDAGuard g(x.device());
  const int dev = x.get_device();
  auto st = at::cuda::getCurrentCUDAStream();
  // dz of one piece is the only [T, .] workspace: about 256 MB by default, in
  // equal pieces of whole tiles
  int64_t width = piece;
  if (width == 0) width = std::max<int64_t>(4096, (int64_t(128) << 20) / T);
  const int64_t n_pieces = (V + width - 1) / width;
  if (piece == 0) width = ((V + n_pieces - 1) / n_pieces + kMaxBN - 1) / kMaxBN * kMaxBN;
  width = std::min<int64_t>((width + 7) / 8 * 8, ((int64_t)V + 7) / 8 * 8);
  const bool one = width >= V;
  at::Tensor dz = at::empty({T, width}, x.options());
  at::Tensor xm = at::empty({T, H}, x.options());
  at::Tensor acc = one ? dx : at::empty({T, H}, x.options().dtype(at::kFloat));
  const long nvec = (long)T * H / 8;
  const int grid = (int)std::min<long>((nvec + 255) / 256, (long)num_sms(dev) * 8);
  mask_rows_kernel<<<grid, 256, 0, st>>>((const __nv_bfloat16*)x.data_ptr(), row_stride(x), coef.data_ptr<float>(),
                                         (__nv_bfloat16*)xm.data_ptr(), T, H);
  check_cuda(cudaGetLastError(), "head mask rows");
  auto bf = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  CUtensorMap tx = make_tmap_2d(x.data_ptr(), bf, 2, H, T, row_stride(x), BK, BM);
  Params p = {};
  p.T = T; p.H = H;
  p.bn = kMaxBN;
  p.scale = (float)(inv_temp * 1.4426950408889634);
  p.inv_temp = (float)inv_temp;
  p.targets = targets ? targets->data_ptr<long>() : nullptr;
  p.lse = lse.data_ptr<float>();
  p.coef = coef.data_ptr<float>();
  for (int64_t v0 = 0; v0 < V; v0 += width) {
    const int n = (int)std::min<int64_t>(width, V - v0);
    at::Tensor wp = w.narrow(0, v0, n);
    at::Tensor dwp = dw.narrow(0, v0, n);
    at::Tensor dzp = dz.narrow(1, 0, n);
    p.V = n;
    p.v0 = (int)v0;
    CUtensorMap tw = make_tmap_2d(wp.data_ptr(), bf, 2, H, n, row_stride(w), BK, kMaxBN / 2);
    CUtensorMap td = make_tmap_2d(dz.data_ptr(), bf, 2, (n + 7) / 8 * 8, T, width, 64, 32);
    launch<true>(tx, tw, td, p, dev, st);
    gemm_bf16(dzp, xm, dwp, true, true, 1.0, accumulate, c10::nullopt, 0);
    gemm_bf16(dzp, wp, acc, false, true, 1.0, !one && v0 > 0, c10::nullopt, 0);
  }
  if (!one) {
    round_kernel<<<grid, 256, 0, st>>>(acc.data_ptr<float>(), (__nv_bfloat16*)dx.data_ptr(), row_stride(dx), T, H);
    check_cuda(cudaGetLastError(), "head round");
  }
}

}  // namespace kore
