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
// magnitude bits. They are bound by HBM.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "common.cuh"
#include "tma_host.h"

namespace kore {
namespace act8 {

constexpr int kBlock = 128;
constexpr int kNormVecs = 1024;  // RMSNorm rows: H <= 8192

KORE_DEV void unpack8(const uint4& u, float (&f)[8]) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = __bfloat1622float2(h[i]);
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}
KORE_DEV uint4 pack8(const float (&f)[8]) {
  return make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
}

// Quantises the 8 values of this lane; the 16 lanes of a half warp share a
// block. All lanes of the warp take part. Returns the bytes, sets the scale.
KORE_DEV uint2 quantise(const uint4& raw, float& scale) {
  // the largest magnitude, as bf16 bits in both halves (NaN > inf > finite)
  uint32_t m = __vmaxu2(__vmaxu2(raw.x & 0x7fff7fffu, raw.y & 0x7fff7fffu),
                        __vmaxu2(raw.z & 0x7fff7fffu, raw.w & 0x7fff7fffu));
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffff, m, o));
  const uint32_t top = max(m & 0xffffu, m >> 16);
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
  float f[8];
  unpack8(raw, f);
  uint32_t b[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    // adding 1.5 * 2^23 rounds to the nearest integer and leaves its low byte
    // in the low byte of the sum
    b[e] = __float_as_uint(__fadd_rn(__fmul_rn(f[e], inv), 12582912.f));
  }
  if (top >= 0x7f80u) return make_uint2(0, 0);
  const uint32_t lo0 = __byte_perm(b[0], b[1], 0x0040), lo1 = __byte_perm(b[2], b[3], 0x0040);
  const uint32_t hi0 = __byte_perm(b[4], b[5], 0x0040), hi1 = __byte_perm(b[6], b[7], 0x0040);
  return make_uint2(__byte_perm(lo0, lo1, 0x5410), __byte_perm(hi0, hi1, 0x5410));
}

// The 8 values that the bytes stand for. 0x4B000000 | (q + 128) is the float
// 2^23 + 128 + q.
KORE_DEV void restore(const uint2& q, float scale, float (&f)[8]) {
  const uint32_t w[2] = {q.x ^ 0x80808080u, q.y ^ 0x80808080u};
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t bits = __byte_perm(w[e / 4], 0x4B000000u, 0x7440 | (e & 3));
    f[e] = __fmul_rn(__fadd_rn(__uint_as_float(bits), -8388736.f), scale);
  }
}

struct Held {
  int8_t* q;      // [T, H]
  float* s;       // [T, nb]
  int H, nb;
};

// ---------------------------------------------------------------- save / load
__global__ void save_kernel(const __nv_bfloat16* __restrict__ x, long ldx, Held h, long T) {
  const long total = T * h.nb;
  const int sub = threadIdx.x & 15;
  // whole half warps step together; the warp's two halves may be in different rows
  for (long i = ((long)blockIdx.x * blockDim.x + threadIdx.x) / 16; i - ((threadIdx.x >> 4) & 1) < total;
       i += (long)gridDim.x * blockDim.x / 16) {
    const long t = i / h.nb;
    const int b = (int)(i - t * h.nb);
    const int col = b * kBlock + sub * 8;
    const bool live = i < total && col < h.H;
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (live) raw = *reinterpret_cast<const uint4*>(x + t * ldx + col);
    float scale;
    const uint2 q = quantise(raw, scale);
    if (live) *reinterpret_cast<uint2*>(h.q + t * h.H + col) = q;
    if (live && sub == 0) h.s[i] = scale;
  }
}

__global__ void load_kernel(Held h, __nv_bfloat16* __restrict__ out, long ldo, long T) {
  const int nvec = h.H / 8;
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < T * nvec; i += (long)gridDim.x * blockDim.x) {
    const long t = i / nvec;
    const int j = (int)(i - t * nvec);
    float f[8];
    restore(*reinterpret_cast<const uint2*>(h.q + i * 8), h.s[t * h.nb + j / 16], f);
    *reinterpret_cast<uint4*>(out + t * ldo + j * 8) = pack8(f);
  }
}

// ------------------------------------------------------------------- RMSNorm
template <int THREADS>
KORE_DEV float block_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffff, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x / 32] = v;
  __syncthreads();
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) t += red[i];
  return t;
}

// hn = x rstd w and the 8-bit copy of x, one read of x
template <int THREADS, int VPT>
__global__ void __launch_bounds__(THREADS) norm_save_kernel(const __nv_bfloat16* __restrict__ x, long ldx,
                                                            const __nv_bfloat16* __restrict__ w,
                                                            __nv_bfloat16* __restrict__ hn, float* __restrict__ rstd,
                                                            Held h, long T, float eps) {
  __shared__ float red[THREADS / 32];
  const int nvec = h.H / 8;
  for (long t = blockIdx.x; t < T; t += gridDim.x) {
    uint4 raw[VPT];
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int j = threadIdx.x + i * THREADS;
      raw[i] = make_uint4(0, 0, 0, 0);
      if (j < nvec) raw[i] = *reinterpret_cast<const uint4*>(x + t * ldx + j * 8);
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int j = threadIdx.x + i * THREADS;
      float f[8], scale;
      unpack8(raw[i], f);
#pragma unroll
      for (int e = 0; e < 8; ++e) ss += f[e] * f[e];
      const uint2 q = quantise(raw[i], scale);
      if (j < nvec) *reinterpret_cast<uint2*>(h.q + t * h.H + j * 8) = q;
      if (j < nvec && (j & 15) == 0) h.s[t * h.nb + j / 16] = scale;
    }
    const float rs = rsqrtf(block_sum<THREADS>(ss, red) / h.H + eps);
    if (threadIdx.x == 0) rstd[t] = rs;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int j = threadIdx.x + i * THREADS;
      if (j < nvec) {
        float f[8], g[8];
        unpack8(raw[i], f);
        unpack8(__ldg(reinterpret_cast<const uint4*>(w) + j), g);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = f[e] * rs * g[e];
        *reinterpret_cast<uint4*>(hn + t * h.H + j * 8) = pack8(f);
      }
    }
  }
}

// x back from 8 bits (bf16), and its RMSNorm from the unrounded values
template <int THREADS, int VPT>
__global__ void __launch_bounds__(THREADS) norm_load_kernel(Held h, const __nv_bfloat16* __restrict__ w,
                                                            __nv_bfloat16* __restrict__ x,
                                                            __nv_bfloat16* __restrict__ hn, float* __restrict__ rstd,
                                                            long T, float eps) {
  __shared__ float red[THREADS / 32];
  const int nvec = h.H / 8;
  for (long t = blockIdx.x; t < T; t += gridDim.x) {
    float f[VPT][8];
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int j = threadIdx.x + i * THREADS;
      if (j < nvec) {
        restore(*reinterpret_cast<const uint2*>(h.q + t * h.H + j * 8), h.s[t * h.nb + j / 16], f[i]);
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += f[i][e] * f[i][e];
        *reinterpret_cast<uint4*>(x + t * h.H + j * 8) = pack8(f[i]);
      }
    }
    const float rs = rsqrtf(block_sum<THREADS>(ss, red) / h.H + eps);
    if (threadIdx.x == 0) rstd[t] = rs;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int j = threadIdx.x + i * THREADS;
      if (j < nvec) {
        float g[8];
        unpack8(__ldg(reinterpret_cast<const uint4*>(w) + j), g);
#pragma unroll
        for (int e = 0; e < 8; ++e) g[e] = f[i][e] * rs * g[e];
        *reinterpret_cast<uint4*>(hn + t * h.H + j * 8) = pack8(g);
      }
    }
  }
}

// -------------------------------------------------------------------- SwiGLU
//   a = silu(gate) up;  dgate = d up sg (1 + gate (1 - sg)),  dup = d gate sg,  sg = sigmoid(gate)
KORE_DEV float sigmoid(float x) { return 1.f / (1.f + __expf(-x)); }

// F % 128 == 0: a block lies wholly in gate or in up, and one half warp takes
// the block of gate and the block of up of the same columns
__global__ void swiglu_save_kernel(const __nv_bfloat16* __restrict__ gu, long ldg, __nv_bfloat16* __restrict__ a,
                                   Held h, long T) {
  const int F = h.H / 2, fb = F / kBlock;
  const long total = T * fb;
  const int sub = threadIdx.x & 15;
  for (long i = ((long)blockIdx.x * blockDim.x + threadIdx.x) / 16; i - ((threadIdx.x >> 4) & 1) < total;
       i += (long)gridDim.x * blockDim.x / 16) {
    const long t = i / fb;
    const int b = (int)(i - t * fb);
    const int col = b * kBlock + sub * 8;
    const bool live = i < total;
    uint4 g = make_uint4(0, 0, 0, 0), u = g;
    if (live) {
      g = *reinterpret_cast<const uint4*>(gu + t * ldg + col);
      u = *reinterpret_cast<const uint4*>(gu + t * ldg + F + col);
    }
    float sg, su;
    const uint2 qg = quantise(g, sg), qu = quantise(u, su);
    float gf[8], uf[8];
    unpack8(g, gf);
    unpack8(u, uf);
#pragma unroll
    for (int e = 0; e < 8; ++e) gf[e] = gf[e] * sigmoid(gf[e]) * uf[e];
    if (live) {
      *reinterpret_cast<uint4*>(a + t * F + col) = pack8(gf);
      *reinterpret_cast<uint2*>(h.q + t * h.H + col) = qg;
      *reinterpret_cast<uint2*>(h.q + t * h.H + F + col) = qu;
      if (sub == 0) {
        h.s[t * h.nb + b] = sg;
        h.s[t * h.nb + fb + b] = su;
      }
    }
  }
}

__global__ void swiglu_kernel(const __nv_bfloat16* __restrict__ gu, long ldg, __nv_bfloat16* __restrict__ a, int F,
                              long T) {
  const int nvec = F / 8;
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < T * nvec; i += (long)gridDim.x * blockDim.x) {
    const long t = i / nvec;
    const int j = (int)(i - t * nvec) * 8;
    float gf[8], uf[8];
    unpack8(*reinterpret_cast<const uint4*>(gu + t * ldg + j), gf);
    unpack8(*reinterpret_cast<const uint4*>(gu + t * ldg + F + j), uf);
#pragma unroll
    for (int e = 0; e < 8; ++e) gf[e] = gf[e] * sigmoid(gf[e]) * uf[e];
    *reinterpret_cast<uint4*>(a + t * F + j) = pack8(gf);
  }
}

__global__ void swiglu_bwd_kernel(Held h, const __nv_bfloat16* __restrict__ dout, long ldd,
                                  __nv_bfloat16* __restrict__ dgu, __nv_bfloat16* __restrict__ a, long T) {
  const int F = h.H / 2, nvec = F / 8;
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < T * nvec; i += (long)gridDim.x * blockDim.x) {
    const long t = i / nvec;
    const int j = (int)(i - t * nvec) * 8;
    float g[8], u[8], d[8], dg[8];
    restore(*reinterpret_cast<const uint2*>(h.q + t * h.H + j), h.s[t * h.nb + j / kBlock], g);
    restore(*reinterpret_cast<const uint2*>(h.q + t * h.H + F + j), h.s[t * h.nb + (F + j) / kBlock], u);
    unpack8(*reinterpret_cast<const uint4*>(dout + t * ldd + j), d);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float sg = sigmoid(g[e]), act = g[e] * sg;
      dg[e] = d[e] * u[e] * (sg + act * (1.f - sg));
      u[e] = act * u[e];   // the activation again
      d[e] = d[e] * act;   // dup
    }
    *reinterpret_cast<uint4*>(dgu + t * h.H + j) = pack8(dg);
    *reinterpret_cast<uint4*>(dgu + t * h.H + F + j) = pack8(d);
    *reinterpret_cast<uint4*>(a + t * F + j) = pack8(u);
  }
}

// ---------------------------------------------------------------- host side
void check_bf16(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.scalar_type() == at::kBFloat16 && t.dim() == 2 && t.stride(1) == 1 &&
                  (t.size(0) <= 1 || t.stride(0) % 8 == 0) && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0,
              "act8: ", name, " must be a 2-D bf16 CUDA tensor with contiguous 16-byte aligned rows");
}

void check_out(const at::Tensor& t, const at::Tensor& like, int64_t T, int64_t H, const char* name) {
  check_bf16(t, name);
  TORCH_CHECK(t.device() == like.device() && t.size(0) == T && t.size(1) == H && t.is_contiguous(), "act8: ", name,
              " must be contiguous [T, H]");
}

Held check_held(const at::Tensor& q, const at::Tensor& s) {
  TORCH_CHECK(q.is_cuda() && q.scalar_type() == at::kChar && q.dim() == 2 && q.is_contiguous() &&
                  q.size(1) >= 8 && q.size(1) % 8 == 0 && reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0,
              "act8: q must be contiguous int8 [T, H], H a multiple of 8");
  const int64_t nb = (q.size(1) + kBlock - 1) / kBlock;
  TORCH_CHECK(s.device() == q.device() && s.scalar_type() == at::kFloat && s.dim() == 2 && s.is_contiguous() &&
                  s.size(0) == q.size(0) && s.size(1) == nb,
              "act8: scales must be contiguous fp32 [T, ceil(H / 128)]");
  Held h;
  h.q = q.data_ptr<int8_t>();
  h.s = s.data_ptr<float>();
  h.H = (int)q.size(1);
  h.nb = (int)nb;
  return h;
}

void check_vec(const at::Tensor& t, const at::Tensor& like, int64_t n, at::ScalarType dt, const char* name) {
  TORCH_CHECK(t.device() == like.device() && t.scalar_type() == dt && t.dim() == 1 && t.is_contiguous() &&
                  t.size(0) == n && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0,
              "act8: ", name, " has the wrong type or length");
}

long stride_of(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

int grid_for(long threads, int dev) {
  return (int)std::max<long>(1, std::min<long>((threads + 255) / 256, (long)num_sms(dev) * 8));
}

}  // namespace act8

void act8_save(const at::Tensor& x, at::Tensor& q, at::Tensor& s) {
  using namespace act8;
  check_bf16(x, "x");
  Held h = check_held(q, s);
  TORCH_CHECK(q.device() == x.device() && q.size(0) == x.size(0) && q.size(1) == x.size(1), "act8: q must match x");
  const long T = x.size(0);
  if (T == 0) return;
  c10::cuda::CUDAGuard g(x.device());
  save_kernel<<<grid_for(T * h.nb * 16, x.get_device()), 256, 0, at::cuda::getCurrentCUDAStream()>>>(
      (const __nv_bfloat16*)x.data_ptr(), stride_of(x), h, T);
  check_cuda(cudaGetLastError(), "act8_save");
}

void act8_load(const at::Tensor& q, const at::Tensor& s, at::Tensor& out) {
  using namespace act8;
  Held h = check_held(q, s);
  check_bf16(out, "out");
  TORCH_CHECK(q.device() == out.device() && q.size(0) == out.size(0) && q.size(1) == out.size(1),
              "act8: out must match the held shape");
  const long T = q.size(0);
  if (T == 0) return;
  c10::cuda::CUDAGuard g(q.device());
  load_kernel<<<grid_for(T * h.H / 8, q.get_device()), 256, 0, at::cuda::getCurrentCUDAStream()>>>(
      h, (__nv_bfloat16*)out.data_ptr(), stride_of(out), T);
  check_cuda(cudaGetLastError(), "act8_load");
}

#define KORE_ACT8_NORM(LAUNCH)                \
  if (nvec <= 128) { LAUNCH(128, 1); }        \
  else if (nvec <= 256) { LAUNCH(256, 1); }   \
  else if (nvec <= 512) { LAUNCH(256, 2); }   \
  else if (nvec <= 768) { LAUNCH(256, 3); }   \
  else { LAUNCH(256, 4); }

void act8_rmsnorm_save(const at::Tensor& x, const at::Tensor& w, at::Tensor& hn, at::Tensor& rstd, at::Tensor& q,
                       at::Tensor& s, double eps) {
  using namespace act8;
  check_bf16(x, "x");
  Held h = check_held(q, s);
  const long T = x.size(0);
  TORCH_CHECK(q.device() == x.device() && q.size(0) == T && q.size(1) == x.size(1), "act8: q must match x");
  TORCH_CHECK(h.H <= kNormVecs * 8, "act8: RMSNorm rows hold at most 8192 columns");
  check_out(hn, x, T, h.H, "hn");
  check_vec(w, x, h.H, at::kBFloat16, "w");
  check_vec(rstd, x, T, at::kFloat, "rstd");
  if (T == 0) return;
  c10::cuda::CUDAGuard g(x.device());
  const int nvec = h.H / 8;
  auto st = at::cuda::getCurrentCUDAStream();
  const int sms = num_sms(x.get_device());
#define KORE_LAUNCH(TH, VP)                                                                                  \
  norm_save_kernel<TH, VP><<<(int)std::min<long>(T, (long)sms * (2048 / TH)), TH, 0, st>>>(                  \
      (const __nv_bfloat16*)x.data_ptr(), stride_of(x), (const __nv_bfloat16*)w.data_ptr(),                  \
      (__nv_bfloat16*)hn.data_ptr(), rstd.data_ptr<float>(), h, T, (float)eps)
  KORE_ACT8_NORM(KORE_LAUNCH)
#undef KORE_LAUNCH
  check_cuda(cudaGetLastError(), "act8_rmsnorm_save");
}

void act8_rmsnorm_load(const at::Tensor& q, const at::Tensor& s, const at::Tensor& w, at::Tensor& x, at::Tensor& hn,
                       at::Tensor& rstd, double eps) {
  using namespace act8;
  Held h = check_held(q, s);
  const long T = q.size(0);
  TORCH_CHECK(h.H <= kNormVecs * 8, "act8: RMSNorm rows hold at most 8192 columns");
  check_out(x, q, T, h.H, "x");
  check_out(hn, q, T, h.H, "hn");
  check_vec(w, q, h.H, at::kBFloat16, "w");
  check_vec(rstd, q, T, at::kFloat, "rstd");
  if (T == 0) return;
  c10::cuda::CUDAGuard g(q.device());
  const int nvec = h.H / 8;
  auto st = at::cuda::getCurrentCUDAStream();
  const int sms = num_sms(q.get_device());
#define KORE_LAUNCH(TH, VP)                                                                                  \
  norm_load_kernel<TH, VP><<<(int)std::min<long>(T, (long)sms * (2048 / TH)), TH, 0, st>>>(                  \
      h, (const __nv_bfloat16*)w.data_ptr(), (__nv_bfloat16*)x.data_ptr(), (__nv_bfloat16*)hn.data_ptr(),    \
      rstd.data_ptr<float>(), T, (float)eps)
  KORE_ACT8_NORM(KORE_LAUNCH)
#undef KORE_LAUNCH
  check_cuda(cudaGetLastError(), "act8_rmsnorm_load");
}

void act8_swiglu_save(const at::Tensor& gu, at::Tensor& a, at::Tensor& q, at::Tensor& s) {
  using namespace act8;
  check_bf16(gu, "gate|up");
  Held h = check_held(q, s);
  const long T = gu.size(0);
  TORCH_CHECK(q.device() == gu.device() && q.size(0) == T && q.size(1) == gu.size(1), "act8: q must match gate|up");
  TORCH_CHECK(h.H % 16 == 0, "act8: SwiGLU's width must be a multiple of 8");
  const int F = h.H / 2;
  check_out(a, gu, T, F, "a");
  if (T == 0) return;
  c10::cuda::CUDAGuard g(gu.device());
  auto st = at::cuda::getCurrentCUDAStream();
  const int dev = gu.get_device();
  const __nv_bfloat16* gp = (const __nv_bfloat16*)gu.data_ptr();
  __nv_bfloat16* ap = (__nv_bfloat16*)a.data_ptr();
  if (F % kBlock == 0) {
    swiglu_save_kernel<<<grid_for(T * (F / 8), dev), 256, 0, st>>>(gp, stride_of(gu), ap, h, T);
  } else {
    // the block at the border holds columns of gate and of up: two passes
    save_kernel<<<grid_for(T * h.nb * 16, dev), 256, 0, st>>>(gp, stride_of(gu), h, T);
    swiglu_kernel<<<grid_for(T * (F / 8), dev), 256, 0, st>>>(gp, stride_of(gu), ap, F, T);
  }
  check_cuda(cudaGetLastError(), "act8_swiglu_save");
}

void act8_swiglu_bwd(const at::Tensor& dout, const at::Tensor& q, const at::Tensor& s, at::Tensor& dgu,
                     at::Tensor& a) {
  using namespace act8;
  check_bf16(dout, "dout");
  Held h = check_held(q, s);
  const long T = q.size(0);
  TORCH_CHECK(h.H % 16 == 0, "act8: SwiGLU's width must be a multiple of 8");
  const int F = h.H / 2;
  TORCH_CHECK(dout.device() == q.device() && dout.size(0) == T && dout.size(1) == F, "act8: dout must be [T, F]");
  check_out(dgu, q, T, h.H, "dgu");
  check_out(a, q, T, F, "a");
  if (T == 0) return;
  c10::cuda::CUDAGuard g(q.device());
  swiglu_bwd_kernel<<<grid_for(T * (F / 8), q.get_device()), 256, 0, at::cuda::getCurrentCUDAStream()>>>(
      h, (const __nv_bfloat16*)dout.data_ptr(), stride_of(dout), (__nv_bfloat16*)dgu.data_ptr(),
      (__nv_bfloat16*)a.data_ptr(), T);
  check_cuda(cudaGetLastError(), "act8_swiglu_bwd");
}

}  // namespace kore
