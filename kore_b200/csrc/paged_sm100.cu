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
#include <torch/extension.h>

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
constexpr int D = 128;
constexpr float kLn2 = 0.6931471805599453f, kLog2e = 1.4426950408889634f;

struct AttnParams {
  const __nv_bfloat16 *q, *kc, *vc;
  long ldq, ldk_slot, ldk_head, ldv_slot, ldv_head, nslots;
  const int *table, *lens, *q_start;
  long ld_table;
  int M, page_size, B, T, Hq, Hkv;
  const int *group_start, *prefix;      // null: no groups
  int ngroups;
  float scale_log2;
  __nv_bfloat16* out;
  float* lse;
};

// One warp per (row, head), four columns a lane.
__global__ void __launch_bounds__(256) attn_kernel(AttnParams p) {
  const long w = (long)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
  const int lane = threadIdx.x & 31;
  const long t = w / p.Hq;
  const int h = (int)(w % p.Hq), kvh = h / (p.Hq / p.Hkv);
  if (t >= min((long)p.q_start[p.B], (long)p.T)) return;
  int lo = 0, hi = p.B - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (p.q_start[mid + 1] <= t) lo = mid + 1; else hi = mid;
  }
  const int b = lo, first = p.q_start[b], n = p.q_start[b + 1] - first;
  const long cap = (long)p.M * p.page_size;
  const int keys = (int)min((long)p.lens[b] - n + (t - first) + 1, cap);
  int shared = 0, lead = b;
  for (int g = 0; g < p.ngroups; ++g)
    if (b >= p.group_start[g] && b < p.group_start[g + 1]) { shared = p.prefix[g]; lead = p.group_start[g]; }
  float q[4], acc[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
  for (int e = 0; e < 4; ++e) q[e] = __bfloat162float(p.q[t * p.ldq + h * D + lane * 4 + e]) * p.scale_log2;
  for (int k = 0; k < keys; ++k) {
    const int page = p.table[(k < shared ? lead : b) * p.ld_table + k / p.page_size];
    const long slot = (long)page * p.page_size + k % p.page_size;
    float kv[4] = {0.f, 0.f, 0.f, 0.f}, vv[4] = {0.f, 0.f, 0.f, 0.f}, s = 0.f;
    if (slot >= 0 && slot < p.nslots)
      for (int e = 0; e < 4; ++e) {
        kv[e] = __bfloat162float(p.kc[slot * p.ldk_slot + kvh * p.ldk_head + lane * 4 + e]);
        vv[e] = __bfloat162float(p.vc[slot * p.ldv_slot + kvh * p.ldv_head + lane * 4 + e]);
      }
    for (int e = 0; e < 4; ++e) s += q[e] * kv[e];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffff, s, o);
    const float mn = fmaxf(m, s), mref = mn == -INFINITY ? 0.f : mn;
    const float c = exp2f(m - mref), x = exp2f(s - mref);
    l = l * c + x;
    for (int e = 0; e < 4; ++e) acc[e] = acc[e] * c + x * vv[e];
    m = mn;
  }
  for (int e = 0; e < 4; ++e)
    p.out[(t * p.Hq + h) * D + lane * 4 + e] = __float2bfloat16(l == 0.f ? 0.f : acc[e] / l);
  if (p.lse && lane == 0) p.lse[t * p.Hq + h] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
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
  if (T == 0 || B == 0) return;
  c10::cuda::CUDAGuard g(q.device());
  AttnParams p;
  p.q = (const __nv_bfloat16*)q.data_ptr();
  p.kc = (const __nv_bfloat16*)kc.data_ptr();
  p.vc = (const __nv_bfloat16*)vc.data_ptr();
  p.ldq = q.stride(0);
  p.ldk_slot = kc.stride(0);
  p.ldk_head = kc.stride(1);
  p.ldv_slot = vc.stride(0);
  p.ldv_head = vc.stride(1);
  p.nslots = kc.size(0);
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
  p.group_start = group_start ? group_start->data_ptr<int>() : nullptr;
  p.prefix = prefix_len ? prefix_len->data_ptr<int>() : nullptr;
  p.ngroups = prefix_len ? (int)prefix_len->numel() : 0;
  p.scale_log2 = (float)(scale * 1.4426950408889634);
  p.out = (__nv_bfloat16*)out.data_ptr();
  p.lse = lse ? lse->data_ptr<float>() : nullptr;
  attn_kernel<<<(unsigned)((T * Hq + 7) / 8), 256, 0, at::cuda::getCurrentCUDAStream()>>>(p);
  check_cuda(cudaGetLastError(), "prefix_attention");
}

}  // namespace kore
