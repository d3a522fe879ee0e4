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
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <tuple>

#include "common.cuh"
#include "tma_host.h"

namespace kore {
namespace verify {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kRows = 8;          // rows whose statistics are taken together
constexpr int kMaxSteps = 128;    // vectors of a thread in the drawing pass
constexpr long kMaxV = 1L << 20;

struct Params {
  const void* logits;
  long ld, V;
  const long* tokens;
  const int* q_start;
  const float* u;                 // [T, 2]
  const float* probs;             // [T, V] or null
  long ld_probs;
  long B, T;
  double inv_tau;                 // 1 when greedy
  bool greedy;
  int* accepted;
  long* next;
  float* logp;
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
  KORE_DEV void load(long j, float (&f)[VE]) const;
};
template <>
KORE_DEV void RowView<__nv_bfloat16>::load(long j, float (&f)[8]) const {
  const long e0 = elem(j);
  if (e0 >= 0 && e0 + 8 <= V) {
    const uint4 u = *reinterpret_cast<const uint4*>(base + j * 8);
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 x = __bfloat1622float2(h[i]);
      f[2 * i] = x.x;
      f[2 * i + 1] = x.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = e0 + i >= 0 && e0 + i < V ? __bfloat162float(base[j * 8 + i]) : -INFINITY;
  }
}
template <>
KORE_DEV void RowView<float>::load(long j, float (&f)[4]) const {
  const long e0 = elem(j);
  if (e0 >= 0 && e0 + 4 <= V) {
    const float4 u = *reinterpret_cast<const float4*>(base + j * 4);
    f[0] = u.x; f[1] = u.y; f[2] = u.z; f[3] = u.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = e0 + i >= 0 && e0 + i < V ? base[j * 4 + i] : -INFINITY;
  }
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

// Sum over the block; every thread gets it.
KORE_DEV double block_sum(double v, double* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffff, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x / 32] = v;
  __syncthreads();
  double t = 0;
  for (int i = 0; i < kWarps; ++i) t += red[i];
  return t;
}

// One block per sequence.
template <typename T>
__global__ void __launch_bounds__(kThreads) verify_kernel(Params p) {
  constexpr int VE = RowView<T>::VE;
  __shared__ Stat part[kRows][kWarps], stat[kRows];
  __shared__ double red[kWarps], group[kMaxSteps * kWarps];
  __shared__ int s_stop;
  __shared__ long s_next;
  const long b = blockIdx.x;
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  const long t0 = min(max((long)p.q_start[b], 0L), p.T), t1 = min(max((long)p.q_start[b + 1], t0), p.T);
  const T* logits = static_cast<const T*>(p.logits);
  const float c = (float)(p.inv_tau * 1.4426950408889634);
  if (b == p.B - 1)               // rows behind the last sequence
    for (long t = t1 + threadIdx.x; t < p.T; t += kThreads) p.logp[t] = 0.f;
  if (t0 == t1) {
    if (threadIdx.x == 0) {
      p.accepted[b] = 0;
      p.next[b] = -1;
    }
    return;
  }
  long row = t1;                  // the row that gives the next token
  Stat rs = {-INFINITY, 0.f, 0};
  bool good = false;
  for (long r0 = t0; r0 < t1; r0 += kRows) {
    const int n = (int)min((long)kRows, t1 - r0);
    for (int i = 0; i < n; ++i) {
      const RowView<T> v(logits + (r0 + i) * p.ld, p.V);
      Stat a = {-INFINITY, 0.f, 0x7fffffff};
      for (long j = threadIdx.x; j < v.nvec; j += kThreads) {
        float f[VE];
        v.load(j, f);
        float mx = f[0];
        int at = 0;
#pragma unroll
        for (int e = 1; e < VE; ++e)
          if (f[e] > mx) { mx = f[e]; at = e; }
        if (mx > a.m) {
          a.s = a.m == -INFINITY ? a.s : a.s * exp2f((a.m - mx) * c);
          a.m = mx;
          a.at = (int)v.elem(j) + at;
        }
        const float mref = a.m == -INFINITY ? 0.f : a.m;
#pragma unroll
        for (int e = 0; e < VE; ++e) a.s += exp2f((f[e] - mref) * c);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        Stat x = {__shfl_xor_sync(0xffffffff, a.m, o), __shfl_xor_sync(0xffffffff, a.s, o), __shfl_xor_sync(0xffffffff, a.at, o)};
        join(a, x, c);
      }
      if (lane == 0) part[i][warp] = a;
    }
    __syncthreads();
    if (threadIdx.x < 32) {
      bool stop = false;
      if (lane < n) {
        Stat a = part[lane][0];
        for (int w = 1; w < kWarps; ++w) join(a, part[lane][w], c);
        stat[lane] = a;
        const long t = r0 + lane;
        const bool fine = a.s > 0.f && a.s < INFINITY;     // a distribution: neither empty nor NaN nor +inf
        stop = true;
        if (fine && t + 1 < t1) {
          const long x = p.tokens[t + 1];
          if (x >= 0 && x < p.V) {
            const double zx = ((double)to_float(logits[t * p.ld + x]) - (double)a.m) * p.inv_tau;
            const double px = exp(zx) / (double)a.s;
            const double qx = p.probs ? (double)p.probs[t * p.ld_probs + x] : 1.0;
            if (p.greedy ? x == a.at : (double)p.u[2 * t] * qx < px) {
              stop = false;
              p.logp[t] = (float)(zx - log((double)a.s));
            }
          }
        }
      }
      const unsigned bad = __ballot_sync(0xffffffff, stop);
      if (lane == 0) s_stop = bad ? __ffs(bad) - 1 : -1;
    }
    __syncthreads();
    if (s_stop >= 0) {
      row = r0 + s_stop;
      rs = stat[s_stop];
      good = rs.s > 0.f && rs.s < INFINITY;
      break;
    }
  }
  for (long t = row + 1 + threadIdx.x; t < t1; t += kThreads) p.logp[t] = 0.f;
  const bool over = row + 1 < t1;                          // a draft was rejected
  const long x = over ? p.tokens[row + 1] : -1;
  if (!good || p.greedy) {
    if (threadIdx.x == 0) {
      p.accepted[b] = (int)(row - t0);
      p.next[b] = good ? rs.at : -1;
      p.logp[row] = good ? (float)-log((double)rs.s) : NAN;
    }
    return;
  }
  // ---- the draw: weights in fp64, summed in the order of the vocabulary
  const RowView<T> v(logits + row * p.ld, p.V);
  const float* qrow = p.probs && over ? p.probs + row * p.ld_probs : nullptr;
  const double m = rs.m;
  auto weight = [&](float z, long e, int mode, double inv_s) -> double {  // mode 0: p s, 1: without the draft, 2: max(0, p - q)
    double w = exp(((double)z - m) * p.inv_tau);
    if (mode == 1 && e == x) w = 0.0;
    if (mode == 2) w = z == -INFINITY ? 0.0 : fmax(w * inv_s - (double)qrow[e], 0.0);
    return w;
  };
  auto sums = [&](int mode, double inv_s) -> double {      // the block's total; group[] gets each warp's part of each step
    double mine = 0;
    int step = 0;
    for (long j0 = 0; j0 < v.nvec; j0 += kThreads, ++step) {
      const long j = j0 + threadIdx.x;
      double w = 0;
      if (j < v.nvec) {
        float f[VE];
        v.load(j, f);
#pragma unroll
        for (int e = 0; e < VE; ++e)
          if (f[e] != -INFINITY) w += weight(f[e], v.elem(j) + e, mode, inv_s);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffff, w, o);
      if (lane == 0) {
        group[step * kWarps + warp] = w;
        mine += w;
      }
    }
    return block_sum(mine, red);
  };
  int mode = over && !qrow ? 1 : 0;
  double total = sums(mode, 1.0), s64 = total;
  if (mode == 1 && x >= 0 && x < p.V) s64 += exp(((double)to_float(logits[row * p.ld + x]) - m) * p.inv_tau);
  const double inv_s = 1.0 / s64;
  if (qrow) {
    mode = 2;
    total = sums(mode, inv_s);
  }
  if (!(total > 0.0)) {                                    // nothing is left over: the target's own distribution
    mode = 0;
    total = sums(mode, inv_s);
  }
  const double want = (double)p.u[2 * row + 1] * total;
  if (warp == 0) {
    const int ngroups = (int)((v.nvec + kThreads - 1) / kThreads) * kWarps;
    int found = -1, lastpos = 0;
    double before = 0, last_before = 0;
    for (int i = 0; i < ngroups && found < 0; ++i) {       // uniform over the warp
      const double w = group[i];
      if (w > 0) { lastpos = i; last_before = before; }
      if (w > 0 && before + w > want) found = i; else before += w;
    }
    if (found < 0) { found = lastpos; before = last_before; }
    const long j = (long)(found / kWarps) * kThreads + (found % kWarps) * 32 + lane;
    double w[VE], mine = 0;
#pragma unroll
    for (int e = 0; e < VE; ++e) w[e] = 0;
    if (j < v.nvec) {
      float f[VE];
      v.load(j, f);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        w[e] = f[e] != -INFINITY ? weight(f[e], v.elem(j) + e, mode, inv_s) : 0.0;
        mine += w[e];
      }
    }
    double upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xffffffff, upto, o);
      if (lane >= o) upto += y;
    }
    double cum = before + upto - mine;
    int hit = 0x7fffffff, any = -1;                        // first element past `want`; last one with weight
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      cum += w[e];
      const int at = (int)(v.elem(j) + e);
      if (w[e] > 0) {
        any = at;
        if (cum > want) hit = min(hit, at);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      hit = min(hit, __shfl_xor_sync(0xffffffff, hit, o));
      any = max(any, __shfl_xor_sync(0xffffffff, any, o));
    }
    if (lane == 0) s_next = hit != 0x7fffffff ? hit : any;
    if (lane == 0) {
      p.accepted[b] = (int)(row - t0);
      p.next[b] = s_next;
      p.logp[row] = (float)(((double)to_float(logits[row * p.ld + s_next]) - m) * p.inv_tau - log(s64));
    }
  }
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
  TORCH_CHECK(V >= 1 && V <= kMaxV / (logits.scalar_type() == at::kFloat ? 4 : 2) - 8, "verify: vocabulary size out of range");
  TORCH_CHECK(tokens.device() == logits.device() && tokens.scalar_type() == at::kLong && tokens.dim() == 1 &&
                  tokens.is_contiguous() && tokens.numel() == T, "verify: tokens must be contiguous int64 [T]");
  TORCH_CHECK(q_start.device() == logits.device() && q_start.scalar_type() == at::kInt && q_start.dim() == 1 &&
                  q_start.is_contiguous() && B >= 0, "verify: q_start must be contiguous int32 [sequences + 1]");
  TORCH_CHECK(u.device() == logits.device() && u.scalar_type() == at::kFloat && u.dim() == 2 && u.is_contiguous() &&
                  u.size(0) == T && u.size(1) == 2, "verify: u must be contiguous fp32 [T, 2]");
  TORCH_CHECK(temperature >= 0, "verify: temperature must not be negative");
  if (probs)
    TORCH_CHECK(probs->device() == logits.device() && probs->scalar_type() == at::kFloat && probs->dim() == 2 &&
                    probs->size(0) == T && probs->size(1) == V && (V <= 1 || probs->stride(1) == 1),
                "verify: draft_probs must be fp32 [T, V] with contiguous rows");
  c10::cuda::CUDAGuard g(logits.device());
  at::Tensor accepted = at::empty({B}, q_start.options()), next = at::empty({B}, tokens.options()),
             logp = at::empty({T}, u.options());
  if (B == 0) return {accepted, next, logp.zero_()};
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
  p.inv_tau = p.greedy ? 1.0 : 1.0 / temperature;
  p.accepted = accepted.data_ptr<int>();
  p.next = next.data_ptr<int64_t>();
  p.logp = logp.data_ptr<float>();
  auto st = at::cuda::getCurrentCUDAStream();
  if (logits.scalar_type() == at::kFloat)
    verify_kernel<float><<<(unsigned)B, kThreads, 0, st>>>(p);
  else
    verify_kernel<__nv_bfloat16><<<(unsigned)B, kThreads, 0, st>>>(p);
  check_cuda(cudaGetLastError(), "verify");
  return {accepted, next, logp};
}

}  // namespace kore
