// Activation checkpoints in 8 bits, and the backward-pass kernels that read them.
//
// A row is held in blocks of 128 columns (the last may be shorter):
//   a = max |x|,  scale = a * (1/127),  q = rint(x * ((1/a) * 127)) (ties to even)
// and stands for q * scale: the error of a value is at most a / 254. A block
// with a < 1e-30 is held as zeros (1/a would overflow); a block with an inf
// or a NaN reads back as NaN everywhere, so an overflow in the forward pass is
// still seen in the backward. Reciprocal and products are IEEE fp32, so the held
// bytes do not depend on how the kernel is built.
//
// All kernels are one pass over HBM: 16 lanes hold a block (8 values each, one
// 16-byte bf16 vector), its maximum is an integer maximum over the values'
// magnitude bits. They are bound by HBM (copy rate 6.5 TB/s), measured at
//   16384 x 5120   RMSNorm + save 69 us, 6.1 TB/s; load + RMSNorm 66 us, 6.4 TB/s
//                  save 42 us, 6.0 TB/s; load 44 us, 5.8 TB/s
//   8192 x 17408   SwiGLU + save 194 us, 5.9 TB/s; SwiGLU backward 237 us, 6.1 TB/s
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "common.cuh"
#include "tma_host.h"

namespace kore {
namespace act8 {

constexpr int kBlock = 128;
constexpr int kMaxNorm = 8192;  // columns of an RMSNorm row

// 8 values of a 16-byte vector as 4 pairs (packed fp32 instructions: the kernels
// are near the issue limit with single ones)
KORE_DEV void unpack8(const uint4& u, uint64_t (&f)[4]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = f2_pack(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
}
KORE_DEV uint4 pack8(const uint64_t (&f)[4]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float lo, hi;
    f2_unpack(f[i], lo, hi);
    w[i] = pack_bf16(lo, hi);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
KORE_DEV float sum_pair(uint64_t v) {
  float lo, hi;
  f2_unpack(v, lo, hi);
  return lo + hi;
}

// The largest magnitude of 8 values, as bf16 bits in both halves (NaN > inf > finite)
KORE_DEV uint32_t magnitude2(const uint4& raw) {
  return __vmaxu2(__vmaxu2(raw.x & 0x7fff7fffu, raw.y & 0x7fff7fffu),
                  __vmaxu2(raw.z & 0x7fff7fffu, raw.w & 0x7fff7fffu));
}

// Quantises 8 values of a block whose largest magnitude has the bf16 bits `top`.
KORE_DEV uint2 quantise_by(const uint4& raw, uint32_t top, float& scale) {
  const float a = __uint_as_float(top << 16);
  float inv = 0.f;
  scale = 0.f;
  if (top >= 0x7f80u) {
    scale = __uint_as_float(0x7fffffffu);
  } else if (a >= 1e-30f) {
    // above 2^126 the reciprocal would be flushed to zero: take it of a scaled by
    // a power of two (127 / a itself is a normal number up to the largest bf16)
    const float p = a > 1e37f ? 0x1p-64f : 1.f;
    inv = __fmul_rn(__frcp_rn(a * p), 127.f) * p;
    scale = __fmul_rn(a, 1.f / 127.f);
  }
  uint64_t f[4];
  unpack8(raw, f);
  const uint64_t magic = f2_pack(12582912.f, 12582912.f);
  uint32_t b[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // adding 1.5 * 2^23 rounds to the nearest integer and leaves its low byte
    // in the low byte of the sum; the product is rounded first (a packed product
    // would be fused with the addition)
    float lo, hi;
    f2_unpack(f[i], lo, hi);
    f2_unpack(f2_add(f2_pack(__fmul_rn(lo, inv), __fmul_rn(hi, inv)), magic), lo, hi);
    b[2 * i] = __float_as_uint(lo);
    b[2 * i + 1] = __float_as_uint(hi);
  }
  if (top >= 0x7f80u) return make_uint2(0, 0);
  const uint32_t lo0 = __byte_perm(b[0], b[1], 0x0040), lo1 = __byte_perm(b[2], b[3], 0x0040);
  const uint32_t hi0 = __byte_perm(b[4], b[5], 0x0040), hi1 = __byte_perm(b[6], b[7], 0x0040);
  return make_uint2(__byte_perm(lo0, lo1, 0x5410), __byte_perm(hi0, hi1, 0x5410));
}

// Quantises the 8 values of this lane; the 16 lanes of a half warp share a
// block. All lanes of the warp take part. Returns the bytes, sets the scale.
KORE_DEV uint2 quantise(const uint4& raw, float& scale) {
  uint32_t m = magnitude2(raw);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffff, m, o));
  return quantise_by(raw, max(m & 0xffffu, m >> 16), scale);
}

// The 8 values that the bytes stand for. 0x4B000000 | (q + 128) is the float
// 2^23 + 128 + q.
KORE_DEV void restore(const uint2& q, float scale, uint64_t (&f)[4]) {
  const uint32_t w[2] = {q.x ^ 0x80808080u, q.y ^ 0x80808080u};
  const uint64_t off = f2_pack(-8388736.f, -8388736.f), s2 = f2_pack(scale, scale);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int e = 2 * i;
    const uint32_t lo = __byte_perm(w[e / 4], 0x4B000000u, 0x7440 | (e & 3));
    const uint32_t hi = __byte_perm(w[e / 4], 0x4B000000u, 0x7440 | ((e + 1) & 3));
    f[i] = f2_mul(f2_add(f2_pack(__uint_as_float(lo), __uint_as_float(hi)), off), s2);
  }
}

struct Held {
  int8_t* q;      // [T, H]
  float* s;       // [T, nb]
  int H, nb;
};

// Element-wise kernels: a thread owns one 8-column vector j and walks rows with
// the grid's y; the loads of a few rows are issued before the first is used.
// More rows cost registers and so resident warps (us, L2 flushed, with 1, 2, 4 rows:
// 16384 x 5120 save -, 49, 57; load -, 49, 49; 8192 x 17408 SwiGLU save 217, 197, -;
// its backward, when it was tried, 229, 246, -).
constexpr int kSaveRows = 2;
constexpr int kLoadRows = 4;

// ---------------------------------------------------------------- save / load
__global__ void __launch_bounds__(256) save_kernel(const __nv_bfloat16* x, long ldx, Held h, long T) {
  const int j = blockIdx.x * blockDim.x + threadIdx.x;
  const bool live = j * 8 < h.H;
  pdl_wait();
  pdl_trigger();
  for (long t0 = (long)blockIdx.y * kSaveRows; t0 < T; t0 += (long)gridDim.y * kSaveRows) {
    uint4 raw[kSaveRows];
#pragma unroll
    for (int r = 0; r < kSaveRows; ++r) {
      raw[r] = make_uint4(0, 0, 0, 0);
      if (live && t0 + r < T) raw[r] = reinterpret_cast<const uint4*>(x + (t0 + r) * ldx)[j];
    }
#pragma unroll
    for (int r = 0; r < kSaveRows; ++r) {
      float scale;
      const uint2 q = quantise(raw[r], scale);
      if (live && t0 + r < T) {
        reinterpret_cast<uint2*>(h.q + (t0 + r) * h.H)[j] = q;
        if ((j & 15) == 0) h.s[(t0 + r) * h.nb + j / 16] = scale;
      }
    }
  }
}

__global__ void __launch_bounds__(256) load_kernel(Held h, __nv_bfloat16* __restrict__ out, long ldo, long T) {
  const int j = blockIdx.x * blockDim.x + threadIdx.x;
  pdl_wait();
  pdl_trigger();
  if (j * 8 >= h.H) return;
  for (long t0 = (long)blockIdx.y * kLoadRows; t0 < T; t0 += (long)gridDim.y * kLoadRows) {
    uint2 q[kLoadRows];
    float s[kLoadRows];
#pragma unroll
    for (int r = 0; r < kLoadRows; ++r)
      if (t0 + r < T) {
        q[r] = reinterpret_cast<const uint2*>(h.q + (t0 + r) * h.H)[j];
        s[r] = h.s[(t0 + r) * h.nb + j / 16];
      }
#pragma unroll
    for (int r = 0; r < kLoadRows; ++r)
      if (t0 + r < T) {
        uint64_t f[4];
        restore(q[r], s[r], f);
        reinterpret_cast<uint4*>(out + (t0 + r) * ldo)[j] = pack8(f);
      }
  }
}

// ------------------------------------------------------------------- RMSNorm
// One block per row, blockDim.x * VPT vectors (H <= 8192); the row stays in registers.
KORE_DEV float block_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffff, v, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x / 32] = v;
  __syncthreads();
  float t = 0.f;
  for (int i = 0; i < (int)blockDim.x / 32; ++i) t += red[i];
  return t;
}

// hn = x rstd w and the 8-bit copy of x, one read of x
// (5 blocks of 256 threads: 48 registers; 16384 x 5120: 69 us, 74 with 62 registers)
template <int VPT>
__global__ void __launch_bounds__(256, 5) norm_save_kernel(const __nv_bfloat16* x, long ldx, const __nv_bfloat16* w,
                                                        __nv_bfloat16* __restrict__ hn, float* __restrict__ rstd,
                                                        Held h, float eps) {
  __shared__ float red[8];
  const int nvec = h.H / 8;
  const long t = blockIdx.x;
  pdl_wait();
  pdl_trigger();
  uint4 raw[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int j = threadIdx.x + i * blockDim.x;
    raw[i] = make_uint4(0, 0, 0, 0);
    if (j < nvec) raw[i] = reinterpret_cast<const uint4*>(x + t * ldx)[j];
  }
  uint64_t ss = 0;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    uint64_t f[4];
    unpack8(raw[i], f);
#pragma unroll
    for (int e = 0; e < 4; ++e) ss = f2_fma(f[e], f[e], ss);
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int j = threadIdx.x + i * blockDim.x;
    float scale;
    const uint2 q = quantise(raw[i], scale);
    if (j < nvec) {
      reinterpret_cast<uint2*>(h.q + t * h.H)[j] = q;
      if ((j & 15) == 0) h.s[t * h.nb + j / 16] = scale;
    }
  }
  const float rs = rsqrtf(block_sum(sum_pair(ss), red) / h.H + eps);
  const uint64_t rs2 = f2_pack(rs, rs);
  if (threadIdx.x == 0) rstd[t] = rs;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int j = threadIdx.x + i * blockDim.x;
    if (j < nvec) {
      uint64_t f[4], g[4];
      unpack8(raw[i], f);
      unpack8(reinterpret_cast<const uint4*>(w)[j], g);
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = f2_mul(f2_mul(f[e], rs2), g[e]);
      reinterpret_cast<uint4*>(hn + t * h.H)[j] = pack8(f);
    }
  }
}

// x back from 8 bits (bf16), and its RMSNorm from the unrounded values
template <int VPT>
__global__ void __launch_bounds__(256) norm_load_kernel(Held h, const __nv_bfloat16* w,
                                                        __nv_bfloat16* __restrict__ x,
                                                        __nv_bfloat16* __restrict__ hn, float* __restrict__ rstd,
                                                        float eps) {
  __shared__ float red[8];
  const int nvec = h.H / 8;
  const long t = blockIdx.x;
  pdl_wait();
  pdl_trigger();
  uint2 q[VPT];
  float s[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int j = threadIdx.x + i * blockDim.x;
    q[i] = make_uint2(0, 0);
    s[i] = 0.f;
    if (j < nvec) {
      q[i] = reinterpret_cast<const uint2*>(h.q + t * h.H)[j];
      s[i] = h.s[t * h.nb + j / 16];
    }
  }
  uint64_t ss = 0;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int j = threadIdx.x + i * blockDim.x;
    uint64_t f[4];
    restore(q[i], s[i], f);
#pragma unroll
    for (int e = 0; e < 4; ++e) ss = f2_fma(f[e], f[e], ss);
    if (j < nvec) reinterpret_cast<uint4*>(x + t * h.H)[j] = pack8(f);
  }
  const float rs = rsqrtf(block_sum(sum_pair(ss), red) / h.H + eps);
  const uint64_t rs2 = f2_pack(rs, rs);
  if (threadIdx.x == 0) rstd[t] = rs;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int j = threadIdx.x + i * blockDim.x;
    if (j < nvec) {
      uint64_t f[4], g[4];
      restore(q[i], s[i], f);
      unpack8(reinterpret_cast<const uint4*>(w)[j], g);
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = f2_mul(f2_mul(f[e], rs2), g[e]);
      reinterpret_cast<uint4*>(hn + t * h.H)[j] = pack8(f);
    }
  }
}

// -------------------------------------------------------------------- SwiGLU
//   a = silu(gate) up;  dgate = d up sg (1 + gate (1 - sg)),  dup = d gate sg,  sg = sigmoid(gate)
constexpr int kGluRows = 2;   // forward; the backward takes one row at a time

KORE_DEV uint64_t sigmoid(uint64_t x) {
  float lo, hi;
  f2_unpack(x, lo, hi);
  return f2_pack(1.f / (1.f + __expf(-lo)), 1.f / (1.f + __expf(-hi)));
}

// HOLD (F % 128 == 0, so that a block lies wholly in gate or in up): also
// writes the 8-bit copy (4 blocks of 256 threads per SM: 194 us at 8192 x 17408, 211 without)
template <bool HOLD>
__global__ void __launch_bounds__(256, 4) swiglu_kernel(const __nv_bfloat16* gu, long ldg,
                                                     __nv_bfloat16* __restrict__ a, Held h, long T) {
  const int F = h.H / 2;
  const int j = blockIdx.x * blockDim.x + threadIdx.x;
  const bool live = j * 8 < F;
  pdl_wait();
  pdl_trigger();
  for (long t0 = (long)blockIdx.y * kGluRows; t0 < T; t0 += (long)gridDim.y * kGluRows) {
    uint4 g[kGluRows], u[kGluRows];
#pragma unroll
    for (int r = 0; r < kGluRows; ++r) {
      g[r] = u[r] = make_uint4(0, 0, 0, 0);
      if (live && t0 + r < T) {
        g[r] = reinterpret_cast<const uint4*>(gu + (t0 + r) * ldg)[j];
        u[r] = reinterpret_cast<const uint4*>(gu + (t0 + r) * ldg + F)[j];
      }
    }
#pragma unroll
    for (int r = 0; r < kGluRows; ++r) {
      const long t = t0 + r;
      const bool ok = live && t < T;
      uint64_t gf[4], uf[4];
      unpack8(g[r], gf);
      unpack8(u[r], uf);
#pragma unroll
      for (int e = 0; e < 4; ++e) gf[e] = f2_mul(f2_mul(gf[e], sigmoid(gf[e])), uf[e]);
      if (ok) reinterpret_cast<uint4*>(a + t * F)[j] = pack8(gf);
      if (HOLD) {
        float sg, su;
        const uint2 qg = quantise(g[r], sg), qu = quantise(u[r], su);
        if (ok) {
          reinterpret_cast<uint2*>(h.q + t * h.H)[j] = qg;
          reinterpret_cast<uint2*>(h.q + t * h.H + F)[j] = qu;
          if ((j & 15) == 0) {
            h.s[t * h.nb + j / 16] = sg;
            h.s[t * h.nb + (F / 8 + j) / 16] = su;
          }
        }
      }
    }
  }
}

// Any F: the blocks of up are not aligned to those of gate, and one block may
// hold columns of both. One block of threads per row; a block's maximum is joined
// in shared memory from the lanes that hold a part of it (at most three groups of
// neighbouring lanes per warp). 8192 x 17400: 255 us, 4.5 TB/s (rows wait for the
// slowest warp at each of the two barriers); 4877 x 4048: 34 us.
constexpr int kRowThreads = 512;
constexpr int kMaxRowF = 5 * kRowThreads * 8;

KORE_DEV void join_block_max(uint32_t* s_top, uint32_t mine, int blk, bool live) {
  // lanes with the same block are neighbours: the first of them and their mask
  const int lane = threadIdx.x & 31;
  const int prev = __shfl_up_sync(0xffffffff, blk, 1), next = __shfl_down_sync(0xffffffff, blk, 1);
  const uint32_t starts = __ballot_sync(0xffffffff, lane == 0 || prev != blk);
  const uint32_t ends = __ballot_sync(0xffffffff, lane == 31 || next != blk);
  const int lo = 31 - __clz(starts & (0xffffffffu >> (31 - lane)));
  const int hi = __ffs(ends & (0xffffffffu << lane)) - 1;
  const uint32_t group = (0xffffffffu >> (31 - hi)) & (0xffffffffu << lo);
  const uint32_t top = __reduce_max_sync(group, live ? max(mine & 0xffffu, mine >> 16) : 0u);
  if (lane == lo && top != 0) atomicMax(s_top + blk, top);
}

template <int VPT>
__global__ void __launch_bounds__(kRowThreads) swiglu_row_kernel(const __nv_bfloat16* gu, long ldg,
                                                                 __nv_bfloat16* __restrict__ a, Held h) {
  __shared__ uint32_t s_top[2 * kMaxRowF / kBlock + 2];
  const int F = h.H / 2, nvec = F / 8;
  const long t = blockIdx.x;
  pdl_wait();
  pdl_trigger();
  uint4 g[VPT], u[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int j = threadIdx.x + i * blockDim.x;
    g[i] = u[i] = make_uint4(0, 0, 0, 0);
    if (j < nvec) {
      g[i] = reinterpret_cast<const uint4*>(gu + t * ldg)[j];
      u[i] = reinterpret_cast<const uint4*>(gu + t * ldg + F)[j];
    }
  }
  for (int b = threadIdx.x; b < h.nb; b += blockDim.x) s_top[b] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int j = threadIdx.x + i * blockDim.x;
    const bool live = j < nvec;
    join_block_max(s_top, magnitude2(g[i]), live ? j / 16 : h.nb, live);
    join_block_max(s_top, magnitude2(u[i]), live ? (nvec + j) / 16 : h.nb, live);
  }
  __syncthreads();
  for (int b = threadIdx.x; b < h.nb; b += blockDim.x) {
    float scale;
    quantise_by(make_uint4(0, 0, 0, 0), s_top[b], scale);
    h.s[t * h.nb + b] = scale;
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int j = threadIdx.x + i * blockDim.x;
    if (j < nvec) {
      float scale;
      reinterpret_cast<uint2*>(h.q + t * h.H)[j] = quantise_by(g[i], s_top[j / 16], scale);
      reinterpret_cast<uint2*>(h.q + t * h.H + F)[j] = quantise_by(u[i], s_top[(nvec + j) / 16], scale);
      uint64_t gf[4], uf[4];
      unpack8(g[i], gf);
      unpack8(u[i], uf);
#pragma unroll
      for (int e = 0; e < 4; ++e) gf[e] = f2_mul(f2_mul(gf[e], sigmoid(gf[e])), uf[e]);
      reinterpret_cast<uint4*>(a + t * F)[j] = pack8(gf);
    }
  }
}

__global__ void __launch_bounds__(256) swiglu_bwd_kernel(Held h, const __nv_bfloat16* dout, long ldd,
                                                         __nv_bfloat16* __restrict__ dgu,
                                                         __nv_bfloat16* __restrict__ a, long T) {
  const int F = h.H / 2;
  const int j = blockIdx.x * blockDim.x + threadIdx.x;
  pdl_wait();
  pdl_trigger();
  if (j * 8 >= F) return;
  for (long t = blockIdx.y; t < T; t += gridDim.y) {
    const uint2 qg = load_once(reinterpret_cast<const uint2*>(h.q + t * h.H) + j);
    const uint2 qu = load_once(reinterpret_cast<const uint2*>(h.q + t * h.H + F) + j);
    const uint4 dv = load_once(reinterpret_cast<const uint4*>(dout + t * ldd) + j);
    const float sg = h.s[t * h.nb + j / 16], su = h.s[t * h.nb + (F / 8 + j) / 16];
    uint64_t g[4], u[4], d[4], dg[4];
    restore(qg, sg, g);
    restore(qu, su, u);
    unpack8(dv, d);
    const uint64_t one = f2_pack(1.f, 1.f), neg = f2_pack(-1.f, -1.f);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint64_t s = sigmoid(g[e]), act = f2_mul(g[e], s);
      dg[e] = f2_mul(f2_mul(d[e], u[e]), f2_fma(act, f2_fma(s, neg, one), s));
      u[e] = f2_mul(act, u[e]);   // the activation again
      d[e] = f2_mul(d[e], act);   // dup
    }
    reinterpret_cast<uint4*>(dgu + t * h.H)[j] = pack8(dg);
    reinterpret_cast<uint4*>(dgu + t * h.H + F)[j] = pack8(d);
    reinterpret_cast<uint4*>(a + t * F)[j] = pack8(u);
  }
}

// ---------------------------------------------------------------- host side
void check_bf16(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.scalar_type() == at::kBFloat16 && t.dim() == 2 && t.stride(1) == 1 &&
                  (t.size(0) <= 1 || t.stride(0) % 8 == 0) && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0,
              "act8: ", name, " must be a 2-D bf16 CUDA tensor with contiguous 16-byte aligned rows");
  TORCH_CHECK(t.size(1) >= 8 && t.size(1) % 8 == 0, "act8: the width of ", name, " must be a positive multiple of 8");
}

Held held_of(const at::Tensor& q, const at::Tensor& s) {
  Held h;
  h.q = q.data_ptr<int8_t>();
  h.s = s.data_ptr<float>();
  h.H = (int)q.size(1);
  h.nb = (int)s.size(1);
  return h;
}

Held check_held(const at::Tensor& q, const at::Tensor& s) {
  TORCH_CHECK(q.is_cuda() && q.scalar_type() == at::kChar && q.dim() == 2 && q.is_contiguous() &&
                  q.size(1) >= 8 && q.size(1) % 8 == 0 && reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0,
              "act8: q must be contiguous int8 [T, H], H a multiple of 8");
  TORCH_CHECK(s.device() == q.device() && s.scalar_type() == at::kFloat && s.dim() == 2 && s.is_contiguous() &&
                  s.size(0) == q.size(0) && s.size(1) == (q.size(1) + kBlock - 1) / kBlock,
              "act8: scales must be contiguous fp32 [T, ceil(H / 128)]");
  return held_of(q, s);
}

void check_weight(const at::Tensor& w, const at::Tensor& like, int64_t H) {
  TORCH_CHECK(H <= kMaxNorm, "act8: RMSNorm rows hold at most 8192 columns");
  TORCH_CHECK(w.device() == like.device() && w.scalar_type() == at::kBFloat16 && w.dim() == 1 && w.is_contiguous() &&
                  w.size(0) == H && reinterpret_cast<uintptr_t>(w.data_ptr()) % 16 == 0,
              "act8: w must be contiguous bf16 [H] on 16 bytes");
}

std::pair<at::Tensor, at::Tensor> new_held(int64_t T, int64_t H, const at::Tensor& like) {
  return {at::empty({T, H}, like.options().dtype(at::kChar)),
          at::empty({T, (H + kBlock - 1) / kBlock}, like.options().dtype(at::kFloat))};
}

long stride_of(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

// Element-wise launch over nvec vectors by T rows, `rows` rows per thread and
// step: the block width that leaves the fewest idle lanes at the row's end, and
// about 8 blocks of 256 threads per SM in all.
struct Shape {
  dim3 grid;
  int threads;
};
Shape shape_for(int nvec, long T, int rows, int dev) {
  int best = 32, idle = -1;
  for (int th = 256; th >= 64; th -= 32) {
    const int waste = (nvec + th - 1) / th * th - nvec;
    if (idle < 0 || waste < idle) { idle = waste; best = th; }
  }
  if (nvec <= 32) best = 32;
  const int gx = (nvec + best - 1) / best;
  const long resident = (long)num_sms(dev) * (2048 / best);
  const long gy = std::min<long>((T + rows - 1) / rows, std::max<long>(1, resident / gx));
  return {dim3(gx, (unsigned)std::min<long>(gy, 65535)), best};
}

// vectors per thread: 4 for wide rows (a row in 64 to 256 threads), else 1
int norm_vpt(int nvec) { return nvec > 128 ? 4 : 1; }

}  // namespace act8

// Returns (q, scales): the given ones (both or none), or new ones.
std::tuple<at::Tensor, at::Tensor> act8_save(const at::Tensor& x, const c10::optional<at::Tensor>& q_into,
                                             const c10::optional<at::Tensor>& s_into) {
  using namespace act8;
  check_bf16(x, "x");
  const long T = x.size(0);
  TORCH_CHECK(q_into.has_value() == s_into.has_value(), "act8: give q and scales, or neither");
  c10::cuda::CUDAGuard g(x.device());
  at::Tensor q, s;
  if (q_into) {
    q = *q_into;
    s = *s_into;
    check_held(q, s);
    TORCH_CHECK(q.device() == x.device() && q.size(0) == T && q.size(1) == x.size(1), "act8: q must match x");
  } else {
    std::tie(q, s) = new_held(T, x.size(1), x);
  }
  if (T == 0) return {q, s};
  const Held h = held_of(q, s);
  const Shape sh = shape_for(h.H / 8, T, kSaveRows, x.get_device());
  launch_after("act8_save", save_kernel, sh.grid, dim3(sh.threads), 0, at::cuda::getCurrentCUDAStream(),
               (const __nv_bfloat16*)x.data_ptr(), stride_of(x), h, T);
  return {q, s};
}

// Returns the values as bf16, in `into` when it is given.
at::Tensor act8_load(const at::Tensor& q, const at::Tensor& s, const c10::optional<at::Tensor>& into) {
  using namespace act8;
  Held h = check_held(q, s);
  const long T = q.size(0);
  if (into) {
    check_bf16(*into, "out");
    TORCH_CHECK(q.device() == into->device() && q.size(0) == into->size(0) && q.size(1) == into->size(1),
                "act8: out must match the held shape");
  }
  c10::cuda::CUDAGuard g(q.device());
  at::Tensor out = into ? *into : at::empty({T, h.H}, s.options().dtype(at::kBFloat16));
  if (T == 0) return out;
  const Shape sh = shape_for(h.H / 8, T, kLoadRows, q.get_device());
  launch_after("act8_load", load_kernel, sh.grid, dim3(sh.threads), 0, at::cuda::getCurrentCUDAStream(), h,
               (__nv_bfloat16*)out.data_ptr(), stride_of(out), T);
  return out;
}

// Returns (hn, rstd, q, scales).
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> act8_rmsnorm_save(const at::Tensor& x,
                                                                             const at::Tensor& w, double eps) {
  using namespace act8;
  check_bf16(x, "x");
  const long T = x.size(0);
  const int64_t H = x.size(1);
  check_weight(w, x, H);
  c10::cuda::CUDAGuard g(x.device());
  at::Tensor hn = at::empty({T, H}, x.options()), rstd = at::empty({T}, x.options().dtype(at::kFloat));
  auto [q, s] = new_held(T, H, x);
  if (T == 0) return {hn, rstd, q, s};
  const int nvec = H / 8;
  auto st = at::cuda::getCurrentCUDAStream();
  const int vpt = norm_vpt(nvec);
  launch_after("act8_rmsnorm_save", vpt == 4 ? norm_save_kernel<4> : norm_save_kernel<1>, dim3((unsigned)T),
               dim3(((nvec + vpt - 1) / vpt + 31) / 32 * 32), 0, st, (const __nv_bfloat16*)x.data_ptr(), stride_of(x),
               (const __nv_bfloat16*)w.data_ptr(), (__nv_bfloat16*)hn.data_ptr(), rstd.data_ptr<float>(),
               held_of(q, s), (float)eps);
  return {hn, rstd, q, s};
}

// Returns (x, hn, rstd).
std::tuple<at::Tensor, at::Tensor, at::Tensor> act8_rmsnorm_load(const at::Tensor& q, const at::Tensor& s,
                                                                 const at::Tensor& w, double eps) {
  using namespace act8;
  Held h = check_held(q, s);
  const long T = q.size(0);
  check_weight(w, q, h.H);
  c10::cuda::CUDAGuard g(q.device());
  at::Tensor x = at::empty({T, h.H}, w.options()), hn = at::empty({T, h.H}, w.options());
  at::Tensor rstd = at::empty({T}, s.options());
  if (T == 0) return {x, hn, rstd};
  const int nvec = h.H / 8;
  auto st = at::cuda::getCurrentCUDAStream();
  const int vpt = norm_vpt(nvec);
  launch_after("act8_rmsnorm_load", vpt == 4 ? norm_load_kernel<4> : norm_load_kernel<1>, dim3((unsigned)T),
               dim3(((nvec + vpt - 1) / vpt + 31) / 32 * 32), 0, st, h, (const __nv_bfloat16*)w.data_ptr(),
               (__nv_bfloat16*)x.data_ptr(), (__nv_bfloat16*)hn.data_ptr(), rstd.data_ptr<float>(), (float)eps);
  return {x, hn, rstd};
}

// Returns (a, q, scales).
std::tuple<at::Tensor, at::Tensor, at::Tensor> act8_swiglu_save(const at::Tensor& gu) {
  using namespace act8;
  check_bf16(gu, "gate|up");
  const long T = gu.size(0);
  const int64_t H = gu.size(1);
  TORCH_CHECK(H % 16 == 0, "act8: the width of gate|up must be a multiple of 16");
  const int F = H / 2;
  c10::cuda::CUDAGuard g(gu.device());
  at::Tensor a = at::empty({T, F}, gu.options());
  auto [q, s] = new_held(T, H, gu);
  if (T == 0) return {a, q, s};
  auto st = at::cuda::getCurrentCUDAStream();
  const int dev = gu.get_device();
  const Held h = held_of(q, s);
  const __nv_bfloat16* gp = (const __nv_bfloat16*)gu.data_ptr();
  __nv_bfloat16* ap = (__nv_bfloat16*)a.data_ptr();
  const Shape sh = shape_for(F / 8, T, kGluRows, dev);
  if (F % kBlock == 0) {
    launch_after("act8_swiglu_save", swiglu_kernel<true>, sh.grid, dim3(sh.threads), 0, st, gp, stride_of(gu), ap, h, T);
  } else if (F <= kMaxRowF) {
    const int nvec = F / 8, vpt = (nvec + kRowThreads - 1) / kRowThreads;
    auto k = vpt == 1 ? swiglu_row_kernel<1> : vpt == 2 ? swiglu_row_kernel<2> : vpt == 3 ? swiglu_row_kernel<3>
                                                                                         : swiglu_row_kernel<5>;
    const int per = vpt == 4 ? 5 : vpt;
    launch_after("act8_swiglu_save", k, dim3((unsigned)T), dim3(((nvec + per - 1) / per + 31) / 32 * 32), 0, st, gp,
                 stride_of(gu), ap, h);
  } else {
    const Shape ss = shape_for(h.H / 8, T, kSaveRows, dev);
    launch_after("act8_swiglu_save", save_kernel, ss.grid, dim3(ss.threads), 0, st, gp, stride_of(gu), h, T);
    launch_after("act8_swiglu_save", swiglu_kernel<false>, sh.grid, dim3(sh.threads), 0, st, gp, stride_of(gu), ap, h, T);
  }
  return {a, q, s};
}

// Returns (dgate|dup, a).
std::tuple<at::Tensor, at::Tensor> act8_swiglu_bwd(const at::Tensor& dout, const at::Tensor& q, const at::Tensor& s) {
  using namespace act8;
  check_bf16(dout, "dout");
  Held h = check_held(q, s);
  const long T = q.size(0);
  TORCH_CHECK(h.H % 16 == 0, "act8: the width of gate|up must be a multiple of 16");
  const int F = h.H / 2;
  TORCH_CHECK(dout.device() == q.device() && dout.size(0) == T && dout.size(1) == F, "act8: dout must be [T, F]");
  c10::cuda::CUDAGuard g(q.device());
  at::Tensor dgu = at::empty({T, h.H}, dout.options()), a = at::empty({T, F}, dout.options());
  if (T == 0) return {dgu, a};
  const Shape sh = shape_for(F / 8, T, 1, q.get_device());
  launch_after("act8_swiglu_bwd", swiglu_bwd_kernel, sh.grid, dim3(sh.threads), 0, at::cuda::getCurrentCUDAStream(), h,
               (const __nv_bfloat16*)dout.data_ptr(), stride_of(dout), (__nv_bfloat16*)dgu.data_ptr(),
               (__nv_bfloat16*)a.data_ptr(), T);
  return {dgu, a};
}

}  // namespace kore
