// Verification of drafted tokens for sm_100a: a sequence's drafts are accepted
// one after the other against the target's probabilities from given uniform
// numbers, and the next token is drawn from what the first rejected draft left
// over (or from the last row's distribution, when all are accepted).
//
// With p = softmax(z / tau) of a row and q the draft's probabilities (1 at the
// draft where it has none): accept while u0 q(x) < p(x); the next token is the
// lowest v with sum_{w <= v} r(w) > u1 sum r, r = max(0, p - q) (p itself when
// nothing was rejected). The emitted tokens are then distributed as p for every q.
//
// The statistics of all rows are sums in fp32: an accept decision is one
// comparison, which a relative error of 1e-7 moves with probability 1e-7. The
// draw compares against every border of a running sum over the vocabulary, where
// such an error moves a token in up to 1% of the draws of a flat distribution, so
// the one row that is drawn from is summed again in fp64.
//
// Measured on one B200 (device times, from replays of a CUDA graph), V = 151,936: 64
// sequences with 0 to 4 drafts (240 rows, 73 MB in bf16) 52 us, half of it the statistics;
// 48 with 0 to 7 drafts and their probabilities (310 rows) 90 us; greedy, 200 with at most
// one (294 rows of 50,257 in fp32) 19 us. The statistics issue in 73% of their cycles, with
// the exponentials' unit busy for 49% and HBM for 34%; the draw issues in 49%, its fp64
// pipe is busy for 24%, and it waits mostly at barriers and for its own results (ncu).
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <algorithm>
#include <cmath>
#include <limits>
#include <tuple>

#include "common.cuh"
#include "tma_host.h"

namespace kore {
namespace verify {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxBlocks = 8;     // of a sequence: a cluster, each with a part of the vocabulary
constexpr int kStatThreads = 256;
constexpr int kMaxParts = 16;     // of a row's statistics
constexpr int kMaxSteps = 257;    // vectors of a thread in the drawing pass, by one block alone

struct Stat;
struct Params {
  const void* logits;
  long ld, V;
  const long* tokens;
  const int* q_start;
  const float* u;                 // [T, 2]
  const float* probs;             // [T, V] or null
  long ld_probs;
  long B, T;
  int blocks, parts;              // blocks of a sequence in the draw, of a row in the statistics
  double inv_tau;                 // 1 when greedy
  float c;                        // inv_tau log2 e, kept a normal number: 0 x inf is NaN at the maximum and at masked tokens
  bool greedy;
  int* accepted;
  long* next;
  float* logp;
  Stat* stats;             // [T, parts]
};

// A row as vectors of VE elements that start on 16-byte boundaries: the first
// and the last may be part-filled, elements outside the row read as -inf.
template <typename T>
struct RowView {
  static constexpr int VE = 16 / sizeof(T);
  const T* base;                  // 16-byte aligned, at or before the row
  int off;                        // elements between base and the row
  long V, nvec;
  KORE_DEV RowView(const T* row, long V_) : V(V_) {
    off = (int)(((uintptr_t)row & 15) / sizeof(T));
    base = row - off;
    nvec = (V + off + VE - 1) / VE;
  }
  KORE_DEV long elem(long j) const { return j * VE - off; }
  KORE_DEV bool whole(long j) const { return elem(j) >= 0 && elem(j) + VE <= V; }
  KORE_DEV uint4 raw(long j) const;
};
template <>
KORE_DEV uint4 RowView<__nv_bfloat16>::raw(long j) const {
  if (whole(j)) return *reinterpret_cast<const uint4*>(base + j * 8);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t h[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const long e = elem(j) + 2 * i + k;
      h[k] = e >= 0 && e < V ? *reinterpret_cast<const uint16_t*>(base + j * 8 + 2 * i + k) : 0xff80u;
    }
    w[i] = h[0] | h[1] << 16;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <>
KORE_DEV uint4 RowView<float>::raw(long j) const {
  if (whole(j)) return *reinterpret_cast<const uint4*>(base + j * 4);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const long e = elem(j) + i;
    w[i] = e >= 0 && e < V ? __float_as_uint(base[j * 4 + i]) : 0xff800000u;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
KORE_DEV void unpack(const uint4& u, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
KORE_DEV void unpack(const uint4& u, float (&f)[4]) {
  f[0] = __uint_as_float(u.x);
  f[1] = __uint_as_float(u.y);
  f[2] = __uint_as_float(u.z);
  f[3] = __uint_as_float(u.w);
}
KORE_DEV float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
KORE_DEV float to_float(float x) { return x; }

struct Stat {                     // running maximum, sum of exp2((z - m) c), lowest index of the maximum
  float m, s;
  int at;
};
KORE_DEV void join(Stat& a, const Stat& b, float c) {
  if (b.m > a.m) {
    a.s = (a.m == -INFINITY ? a.s : a.s * exp2f((a.m - b.m) * c)) + b.s;
    a.m = b.m;
    a.at = b.at;
  } else {
    a.s += b.m == -INFINITY ? b.s : b.s * exp2f((b.m - a.m) * c);
    if (b.m == a.m) a.at = min(a.at, b.at);
  }
}

// Another block's shared memory (the variable at the same place there).
KORE_DEV double peer_f64(const double* p, uint32_t rank) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(mapa_shared(smem_u32(p), rank)) : "memory");
  return v;
}

// 2^(i / 32), i < 32, and exp(x) for x <= 0 from it: x = (32 k + i) ln2 / 32 + r with
// |r| <= ln2 / 64, exp(r) by its series up to r^4 / 24 (off by r^5 / 120 < 2e-12: a draw
// from 152k tokens moves with probability 3e-7). Nine fp64 operations, where the
// library's exp takes more than twice as many.
struct Exp {
  const double* tab;
  KORE_DEV double operator()(double x) const {
    if (!(x > -700.0)) return 0.0;                       // NaN does not come here
    const double t = fma(x, 32 * 1.4426950408889634, 6755399441055744.0);   // 1.5 * 2^52: the integer is in the low bits
    const int n = __double2loint(t);
    const double r = fma(t - 6755399441055744.0, -0.6931471805599453 / 32, x);
    const double e = fma(fma(fma(fma(r, 1.0 / 24, 1.0 / 6), r, 0.5), r, 1.0), r, 1.0) * tab[n & 31];
    return __hiloint2double(__double2hiint(e) + (int)((unsigned)(n & ~31) << 15), __double2loint(e));
  }
};

// Statistics of the rows, p.parts blocks to each (all rows at once: a pass over the logits
// that fills the SMs whatever the shape of the batch).
template <typename T>
__global__ void __launch_bounds__(kStatThreads) stats_kernel(Params p) {
  constexpr int VE = RowView<T>::VE;
  constexpr int U = sizeof(T) == 2 ? 4 : 8;     // loads of a thread in flight
  __shared__ Stat part[kStatThreads / 32];
  pdl_trigger();
  const long row = blockIdx.x / p.parts;
  const int own = blockIdx.x - (int)(row * p.parts), warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  const float c = p.c;
  const RowView<T> v(static_cast<const T*>(p.logits) + row * p.ld, p.V);
  const long step = (long)p.parts * kStatThreads;
  const uint32_t none = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;      // -inf
  Stat a = {-INFINITY, 0.f, 0x7fffffff};
#pragma unroll 1
  for (long j0 = own * kStatThreads + threadIdx.x; j0 < v.nvec; j0 += U * step) {
    uint4 x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = j0 + u * step < v.nvec ? v.raw(j0 + u * step) : make_uint4(none, none, none, none);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float f[VE];
      unpack(x[u], f);
      float mx = f[0];
#pragma unroll
      for (int e = 1; e < VE; ++e) mx = fmaxf(mx, f[e]);
      if (mx > a.m) {             // rare after the first vectors
        int at = 0;
#pragma unroll
        for (int e = VE - 1; e >= 0; --e)
          if (f[e] == mx) at = e;
        a.s = a.m == -INFINITY ? a.s : a.s * exp2f((a.m - mx) * c);
        a.m = mx;
        a.at = (int)v.elem(j0 + u * step) + at;
      }
      const float mref = a.m == -INFINITY ? 0.f : a.m;
      float add[2] = {0.f, 0.f};
#pragma unroll
      for (int e = 0; e < VE; ++e) add[e & 1] += exp2f((f[e] - mref) * c);   // a NaN or +inf makes the sum NaN
      a.s += add[0] + add[1];
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Stat x = {__shfl_xor_sync(0xffffffff, a.m, o), __shfl_xor_sync(0xffffffff, a.s, o), __shfl_xor_sync(0xffffffff, a.at, o)};
    join(a, x, c);
  }
  if (lane == 0) part[warp] = a;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kStatThreads / 32; ++w) join(a, part[w], c);
    p.stats[blockIdx.x] = a;
  }
}

// One cluster of p.blocks blocks per sequence: accepts, then draws.
template <typename T>
__global__ void __launch_bounds__(kThreads, 2) verify_kernel(Params p) {
  constexpr int VE = RowView<T>::VE;
  __shared__ Stat s_stat;
  __shared__ double red[kWarps], group[kMaxSteps * kWarps], total_of[3], tab[32];
  __shared__ long s_row;
  const int nblk = p.blocks;
  const long b = blockIdx.x / nblk;
  const uint32_t rank = cluster_ctarank();
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  if (threadIdx.x < 32) tab[threadIdx.x] = exp2((double)threadIdx.x / 32);
  pdl_wait();
  const long t0 = min(max((long)p.q_start[b], 0L), p.T), t1 = min(max((long)p.q_start[b + 1], t0), p.T);
  const T* logits = static_cast<const T*>(p.logits);
  const float c = p.c;
  const bool first = rank == 0;   // the block that writes what all know
  if (b == 0 && first)            // rows before the first sequence
    for (long t = threadIdx.x; t < t0; t += kThreads) p.logp[t] = 0.f;
  if (b == p.B - 1 && first)      // rows behind the last one
    for (long t = t1 + threadIdx.x; t < p.T; t += kThreads) p.logp[t] = 0.f;
  if (t0 == t1) {                 // the whole cluster
    if (first && threadIdx.x == 0) {
      p.accepted[b] = 0;
      p.next[b] = -1;
    }
    return;
  }
  if (warp == 0) {                // a row to a lane, 32 rows at a time, until one stops
    long row = -1;
    for (long r0 = t0; r0 < t1 && row < 0; r0 += 32) {
      const long t = r0 + lane;
      Stat a = {-INFINITY, 0.f, 0x7fffffff};
      bool stop = t < t1;
      float logp = 0.f;
      if (t < t1) {
        for (int k = 0; k < p.parts; ++k) join(a, p.stats[t * p.parts + k], c);
        const bool fine = a.s > 0.f && a.s < INFINITY;     // a distribution: neither empty nor NaN nor +inf
        if (fine && t + 1 < t1) {
          const long x = p.tokens[t + 1];
          if (x >= 0 && x < p.V) {
            const double zx = ((double)to_float(logits[t * p.ld + x]) - (double)a.m) * p.inv_tau;
            const double px = exp(zx) / (double)a.s;
            const double qx = p.probs ? (double)p.probs[t * p.ld_probs + x] : 1.0;
            if (p.greedy ? x == a.at : (double)p.u[2 * t] * qx < px) {
              stop = false;
              logp = (float)(zx - log((double)a.s));
            }
          }
        }
      }
      const unsigned bad = __ballot_sync(0xffffffff, stop);
      const int end = bad ? __ffs(bad) - 1 : 32;
      if (first && lane < end && t < t1) p.logp[t] = logp;
      if (bad) {
        row = r0 + end;
        if (lane == end) s_stat = a;
      }
    }
    if (lane == 0) s_row = row;
  }
  __syncthreads();
  const long row = s_row;         // the row that gives the next token
  const Stat rs = s_stat;
  const bool good = rs.s > 0.f && rs.s < INFINITY;
  for (long t = row + 1 + threadIdx.x; t < t1; t += kThreads) p.logp[t] = 0.f;
  const bool over = row + 1 < t1;                          // a draft was rejected
  const long x = over ? p.tokens[row + 1] : -1;
  if (!good || p.greedy) {
    if (first && threadIdx.x == 0) {
      p.accepted[b] = (int)(row - t0);
      p.next[b] = good ? rs.at : -1;
      p.logp[row] = good ? (float)-log((double)rs.s) : NAN;
    }
    return;
  }
  // ---- the draw: weights in fp64, summed in the order of the vocabulary, a part to a block
  const RowView<T> v(logits + row * p.ld, p.V);
  const long per = (v.nvec + nblk - 1) / nblk, lo = min(rank * per, v.nvec), hi = min(lo + per, v.nvec);
  const float* qrow = p.probs && over ? p.probs + row * p.ld_probs : nullptr;
  // Exponents are (z - m) / tau with the difference taken first: 0 at the maximum for every
  // tau. (z / tau - m / tau in one fma saves an operation, but has the rounding of m / tau,
  // which passes 1 from tau = 1e-15 on and leaves no weight at all from 1e-18.)
  const double m = rs.m;
  const Exp ex = {tab};
  const uint32_t none = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;      // -inf
  // Weights of a vector's tokens: p s (mode 0), without the draft (1), max(0, p - q) (2).
  auto weights = [&](long j, const uint4& z, const float (&q)[VE], int mode, double inv_s, double (&w)[VE]) {
    float f[VE];
    unpack(z, f);
    if (mode == 1 && x >= v.elem(j) && x < v.elem(j) + VE) {
#pragma unroll
      for (int e = 0; e < VE; ++e)
        if (v.elem(j) + e == x) f[e] = -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < VE; ++e) w[e] = ex(((double)f[e] - m) * p.inv_tau);   // 0 at -inf
    if (mode == 2) {
#pragma unroll
      for (int e = 0; e < VE; ++e) w[e] = fmax(__dmul_rn(w[e], inv_s) - (double)q[e], 0.0);
    }
  };
  auto draft = [&](long j, float (&q)[VE]) {               // the draft's probabilities of vector j
    const float* at = qrow + v.elem(j);
    if (v.whole(j) && ((uintptr_t)at & 15) == 0) {
#pragma unroll
      for (int e = 0; e < VE; e += 4) *reinterpret_cast<float4*>(&q[e]) = *reinterpret_cast<const float4*>(at + e);
    } else {
#pragma unroll
      for (int e = 0; e < VE; ++e) q[e] = v.elem(j) + e >= 0 && v.elem(j) + e < p.V ? at[e] : 0.f;
    }
  };
  // The cluster's total and the sum of the blocks before this one; group[] gets each warp's part of each step.
  auto sums = [&](int mode, double inv_s, int slot, double& before) -> double {
    double own = 0;
    int step = 0;
    constexpr int U = 2;          // vectors of a thread in flight
#pragma unroll 1
    for (long j0 = lo; j0 < hi; j0 += U * kThreads, step += U) {
      uint4 z[U];
      float q[U][VE];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const long j = j0 + u * kThreads + threadIdx.x;
        z[u] = make_uint4(none, none, none, none);
        if (j < hi) z[u] = v.raw(j);
        if (mode != 2) continue;
        if (j < hi) {
          draft(j, q[u]);
        } else {
#pragma unroll
          for (int e = 0; e < VE; ++e) q[u][e] = 0.f;
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        double w[VE];
        weights(j0 + u * kThreads + threadIdx.x, z[u], q[u], mode, inv_s, w);
        double sum = 0;
#pragma unroll
        for (int e = 0; e < VE; ++e) sum += w[e];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffff, sum, o);
        if (lane == 0 && j0 + u * kThreads < hi) {
          group[(step + u) * kWarps + warp] = sum;
          own += sum;
        }
      }
    }
    if (lane == 0) red[warp] = own;
    __syncthreads();
    if (threadIdx.x == 0) {
      double t = 0;
      for (int i = 0; i < kWarps; ++i) t += red[i];
      total_of[slot] = t;
    }
    __syncthreads();
    cluster_sync();
    double total = 0;
#pragma unroll 1
    for (int k = 0; k < nblk; ++k) {
      if (k == (int)rank) before = total;
      total += peer_f64(&total_of[slot], k);
    }
    return total;
  };
  int mode = over && !qrow ? 1 : 0, slot = 0;
  double before, total = sums(mode, 1.0, slot, before), s64 = total;
  if (mode == 1 && x >= 0 && x < p.V) s64 += ex(((double)to_float(logits[row * p.ld + x]) - m) * p.inv_tau);
  const double inv_s = 1.0 / s64;
  if (qrow) {
    mode = 2;
    total = sums(mode, inv_s, ++slot, before);
  }
  if (!(total > 0.0)) {                                    // nothing is left over: the target's own distribution
    mode = 0;
    total = sums(mode, inv_s, ++slot, before);
  }
  const double want = (double)p.u[2 * row + 1] * total;
  // the block whose part holds `want`: the first whose sum passes it, else (rounding) the last that has weight
  int owner = -1, last = 0;
  double upto = 0;
  for (int k = 0; k < nblk; ++k) {
    const double w = peer_f64(&total_of[slot], k);
    upto += w;
    if (w > 0) {
      last = k;
      if (owner < 0 && upto > want) owner = k;
    }
  }
  if (owner < 0) owner = last;
  if (owner == (int)rank && warp == 0) {
    // the group (32 vectors of one step) that holds it, in the same way
    const int ngroups = (int)((hi - lo + kThreads - 1) / kThreads) * kWarps;
    int found = -1, lastpos = 0;
    double at = before, last_at = before;
#pragma unroll 1
    for (int i0 = 0; i0 < ngroups && found < 0; i0 += 32) {
      const double w = i0 + lane < ngroups ? group[i0 + lane] : 0.0;
      double cum = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(0xffffffff, cum, o);
        if (lane >= o) cum += y;
      }
      const unsigned pos = __ballot_sync(0xffffffff, w > 0), past = __ballot_sync(0xffffffff, w > 0 && at + cum > want);
      if (pos) {
        const int k = past ? __ffs(past) - 1 : 31 - __clz(pos);
        const double start = at + __shfl_sync(0xffffffff, cum - w, k);
        if (past) { found = i0 + k; last_at = start; }
        else { lastpos = i0 + k; last_at = start; }
      }
      at += __shfl_sync(0xffffffff, cum, 31);
    }
    if (found < 0) found = lastpos;
    const long j = lo + (long)(found / kWarps) * kThreads + (found % kWarps) * 32 + lane;
    double w[VE], own = 0;
    float q[VE] = {};
    if (mode == 2 && j < hi) draft(j, q);
    weights(j, j < hi ? v.raw(j) : make_uint4(none, none, none, none), q, mode, inv_s, w);
#pragma unroll
    for (int e = 0; e < VE; ++e) own += w[e];
    double cum = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xffffffff, cum, o);
      if (lane >= o) cum += y;
    }
    cum += last_at - own;
    int hit = 0x7fffffff, any = -1;                        // first element past `want`; last one with weight
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      cum += w[e];
      const int at_e = (int)(v.elem(j) + e);
      if (w[e] > 0) {
        any = at_e;
        if (cum > want) hit = min(hit, at_e);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      hit = min(hit, __shfl_xor_sync(0xffffffff, hit, o));
      any = max(any, __shfl_xor_sync(0xffffffff, any, o));
    }
    if (lane == 0) {
      const int y = hit != 0x7fffffff ? hit : any;
      p.accepted[b] = (int)(row - t0);
      p.next[b] = y;
      p.logp[row] = (float)(((double)to_float(logits[row * p.ld + y]) - m) * p.inv_tau - log(s64));
    }
  }
  cluster_sync();                                          // peers have read this block's sums
}

}  // namespace verify

std::tuple<at::Tensor, at::Tensor, at::Tensor> spec_verify(const at::Tensor& logits, const at::Tensor& tokens,
                                                           const at::Tensor& q_start, const at::Tensor& u,
                                                           double temperature, const c10::optional<at::Tensor>& probs) {
  using namespace verify;
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && (logits.scalar_type() == at::kBFloat16 || logits.scalar_type() == at::kFloat) &&
                  (logits.size(1) <= 1 || logits.stride(1) == 1),
              "verify: logits must be bf16 or fp32 [T, V] with contiguous rows");
  const int64_t T = logits.size(0), V = logits.size(1), B = q_start.numel() - 1;
  TORCH_CHECK(B < (int64_t)1 << 27, "verify: too many sequences");
  TORCH_CHECK(V >= 1 && V <= (kMaxSteps - 1L) * kThreads * (logits.scalar_type() == at::kFloat ? 4 : 8) - 8,
              "verify: a vocabulary holds at most 1,048,568 (bf16) or 524,280 (fp32) tokens");
  TORCH_CHECK(tokens.device() == logits.device() && tokens.scalar_type() == at::kLong && tokens.dim() == 1 &&
                  tokens.is_contiguous() && tokens.numel() == T, "verify: tokens must be contiguous int64 [T]");
  TORCH_CHECK(q_start.device() == logits.device() && q_start.scalar_type() == at::kInt && q_start.dim() == 1 &&
                  q_start.is_contiguous() && B >= 0, "verify: q_start must be contiguous int32 [sequences + 1]");
  TORCH_CHECK(u.device() == logits.device() && u.scalar_type() == at::kFloat && u.dim() == 2 && u.is_contiguous() &&
                  u.size(0) == T && u.size(1) == 2, "verify: u must be contiguous fp32 [T, 2]");
  TORCH_CHECK(temperature >= 0 && std::isfinite(temperature), "verify: temperature must be finite and not negative");
  if (probs)
    TORCH_CHECK(probs->device() == logits.device() && probs->scalar_type() == at::kFloat && probs->dim() == 2 &&
                    probs->size(0) == T && probs->size(1) == V && (V <= 1 || probs->stride(1) == 1),
                "verify: draft_probs must be fp32 [T, V] with contiguous rows");
  c10::cuda::CUDAGuard g(logits.device());
  at::Tensor accepted = at::empty({B}, q_start.options()), next = at::empty({B}, tokens.options()),
             logp = at::empty({T}, u.options());
  if (B == 0) return {accepted, next, logp.zero_()};
  if (T == 0) return {accepted.zero_(), next.fill_(-1), logp};
  TORCH_CHECK(T < (int64_t)1 << 27, "verify: too many rows");
  Params p;
  p.logits = logits.data_ptr();
  p.ld = logits.stride(0);
  p.V = V;
  p.tokens = tokens.data_ptr<int64_t>();
  p.q_start = q_start.data_ptr<int>();
  p.u = u.data_ptr<float>();
  p.probs = probs ? probs->data_ptr<float>() : nullptr;
  p.ld_probs = probs ? probs->stride(0) : 0;
  p.B = B;
  p.T = T;
  p.greedy = temperature == 0;
  p.inv_tau = p.greedy ? 1.0 : std::min(1.0 / temperature, std::numeric_limits<double>::max());
  p.c = (float)std::clamp(p.inv_tau * 1.4426950408889634, (double)std::numeric_limits<float>::min(), (double)std::numeric_limits<float>::max());
  p.accepted = accepted.data_ptr<int>();
  p.next = next.data_ptr<int64_t>();
  p.logp = logp.data_ptr<float>();
  // As many blocks to a sequence as two on each SM leave room for, at most a portable
  // cluster. (Eight for all took 57 us for 200 sequences x 2 rows x 50,257 in several
  // waves of blocks, one each 27, with the statistics still in this kernel.)
  const int room = 2 * num_sms(logits.get_device());
  p.blocks = 1;
  while (p.blocks < kMaxBlocks && B * p.blocks * 2 <= room) p.blocks *= 2;
  // Statistics: blocks for eight to an SM, each thread with a vector at least. (Six of the
  // bf16 form fit by its registers, four of the fp32 form: the rest are a second wave.)
  p.parts = (int)std::min<int64_t>(kMaxParts, std::max<int64_t>(1, std::min<int64_t>(4 * room / T, V / (8 * kStatThreads))));
  at::Tensor stats = at::empty({T * p.parts, 3}, u.options());
  p.stats = reinterpret_cast<Stat*>(stats.data_ptr<float>());
  const bool f32 = logits.scalar_type() == at::kFloat;
  auto st = at::cuda::getCurrentCUDAStream();
  (f32 ? stats_kernel<float> : stats_kernel<__nv_bfloat16>)<<<(unsigned)(T * p.parts), kStatThreads, 0, st>>>(p);
  check_cuda(cudaGetLastError(), "verify statistics");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(B * p.blocks));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.blocks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  check_cuda(cudaLaunchKernelEx(&cfg, f32 ? verify_kernel<float> : verify_kernel<__nv_bfloat16>, p), "verify");
  return {accepted, next, logp};
}

}  // namespace kore
