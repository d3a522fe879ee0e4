// Token embedding with scaling, and its gradient by sorted tokens.
//
//   out_t = s E[id_t]                          dE_v (+)= s sum_{t: id_t = v} dy_t
//
// The sum runs over a token's positions in ascending order in fp32 and is
// rounded once when the row is written, so the gradient does not depend on the
// order in which blocks run and a frequent token loses nothing to repeated
// bf16 additions. ids outside [0, V) read a zero row and receive no gradient.
//
// Gradient: the keys (id, position) are sorted (they are distinct, so any sort
// is stable); tiles of kTile keys are sorted in shared memory and an element's
// place among all tiles is its place in its own tile plus, by binary search,
// the number of smaller keys in each of the others. The sorted positions are
// cut in chunks of kChunk; a block sums its chunk's rows segment by segment.
// A segment inside a chunk goes straight to its row; what crosses a chunk's
// border goes to a workspace and is joined by the chunk where it begins, in
// chunk order. A token with thousands of positions is thus summed by many
// blocks.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "common.cuh"
#include "tma_host.h"

namespace kore {
namespace embed {

typedef unsigned long long u64;

constexpr int kTile = 4096;
constexpr int kSortThreads = 1024;
constexpr int kChunk = 32;

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

__global__ void lookup_kernel(const long* __restrict__ ids, const __nv_bfloat16* __restrict__ table, long ldt,
                              __nv_bfloat16* __restrict__ out, float scale, long T, int V, int H) {
  const int nvec = H / 8;
  for (long t = blockIdx.x; t < T; t += gridDim.x) {
    const long id = ids[t];
    const bool ok = id >= 0 && id < V;
    for (int j = threadIdx.x; j < nvec; j += blockDim.x) {
      uint4 u = make_uint4(0, 0, 0, 0);
      if (ok) {
        u = __ldg(reinterpret_cast<const uint4*>(table + id * ldt) + j);
        if (scale != 1.f) {
          float f[8];
          unpack8(u, f);
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] *= scale;
          u = pack8(f);
        }
      }
      reinterpret_cast<uint4*>(out + t * (long)H)[j] = u;
    }
  }
}

// Sorts tile blockIdx.x of the keys (id << 32 | position); ids outside the
// table sort behind all others as V. Bitonic network over the next power of two.
__global__ void __launch_bounds__(kSortThreads) sort_tiles_kernel(const long* __restrict__ ids, u64* __restrict__ keys,
                                                                  int T, int V) {
  __shared__ u64 k[kTile];
  const int base = blockIdx.x * kTile;
  const int n = min(kTile, T - base);
  int size = 32;
  while (size < n) size <<= 1;
  for (int i = threadIdx.x; i < size; i += kSortThreads) {
    u64 key = ~0ull;
    if (i < n) {
      const long id = ids[base + i];
      key = ((u64)(uint32_t)(id >= 0 && id < V ? (int)id : V) << 32) | (uint32_t)(base + i);
    }
    k[i] = key;
  }
  for (int w = 2; w <= size; w <<= 1)
    for (int d = w >> 1; d > 0; d >>= 1) {
      __syncthreads();
      for (int i = threadIdx.x; i < size / 2; i += kSortThreads) {
        const int a = 2 * i - (i & (d - 1)), b = a + d;
        const u64 x = k[a], y = k[b];
        if ((x > y) == ((a & w) == 0)) {
          k[a] = y;
          k[b] = x;
        }
      }
    }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kSortThreads) keys[base + i] = k[i];
}

__global__ void rank_kernel(const u64* __restrict__ tiles, u64* __restrict__ keys, int T) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= T) return;
  const u64 key = tiles[i];
  const int own = i / kTile;
  int rank = i - own * kTile;
  for (int j = 0; j * kTile < T; ++j) {
    if (j == own) continue;
    const u64* t = tiles + (size_t)j * kTile;
    int lo = 0, hi = min(kTile, T - j * kTile);
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (t[mid] < key) lo = mid + 1; else hi = mid;
    }
    rank += lo;
  }
  keys[rank] = key;
}

template <typename G>
KORE_DEV void write_row(G* row, int j, const float (&sum)[8], float scale, bool add);
template <>
KORE_DEV void write_row<float>(float* row, int j, const float (&sum)[8], float scale, bool add) {
  float4* p = reinterpret_cast<float4*>(row) + 2 * j;
  float4 a = make_float4(sum[0] * scale, sum[1] * scale, sum[2] * scale, sum[3] * scale);
  float4 b = make_float4(sum[4] * scale, sum[5] * scale, sum[6] * scale, sum[7] * scale);
  if (add) {
    const float4 c = p[0], d = p[1];
    a.x += c.x; a.y += c.y; a.z += c.z; a.w += c.w;
    b.x += d.x; b.y += d.y; b.z += d.z; b.w += d.w;
  }
  p[0] = a;
  p[1] = b;
}
template <>
KORE_DEV void write_row<__nv_bfloat16>(__nv_bfloat16* row, int j, const float (&sum)[8], float scale, bool add) {
  uint4* p = reinterpret_cast<uint4*>(row) + j;
  float f[8];
  if (add) {
    unpack8(*p, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = fmaf(sum[e], scale, f[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = sum[e] * scale;
  }
  *p = pack8(f);
}

KORE_DEV int key_id(u64 k) { return (int)(k >> 32); }

// grid (chunks, slabs of blockDim.x 8-column vectors)
template <typename G>
__global__ void segments_kernel(const u64* __restrict__ keys, const __nv_bfloat16* __restrict__ dy, long ldy,
                                G* __restrict__ dtable, float* __restrict__ part, float scale, int add, int T, int V,
                                int H) {
  __shared__ int s_id[kChunk + 2];
  __shared__ int s_pos[kChunk];
  const int first = blockIdx.x * kChunk;
  const int n = min(kChunk, T - first);
  for (int i = threadIdx.x; i < n + 2; i += blockDim.x) {
    const int at = first + i - 1;
    const bool in = at >= 0 && at < T;
    const u64 k = in ? keys[at] : 0;
    s_id[i] = in ? key_id(k) : -1;
    if (i >= 1 && i <= n) s_pos[i - 1] = (int)(uint32_t)k;
  }
  __syncthreads();
  const int j = blockIdx.y * blockDim.x + threadIdx.x;
  if (j * 8 >= H) return;
  const uint4* src = reinterpret_cast<const uint4*>(dy) + j;
  const long ld = ldy / 8;
  float sum[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  bool begins = s_id[0] != s_id[1];
  for (int i0 = 0; i0 < n; i0 += 8) {
    uint4 v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (i0 + u < n && s_id[i0 + u + 1] < V) v[u] = __ldg(src + s_pos[i0 + u] * ld);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int i = i0 + u;
      if (i >= n) break;
      const int id = s_id[i + 1];
      if (id >= V) break;  // ids outside the table are last
      float f[8];
      unpack8(v[u], f);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] += f[e];
      const bool ends = s_id[i + 2] != id;
      if (!ends && i + 1 < n) continue;
      if (begins && ends) {
        write_row<G>(dtable + (size_t)id * H, j, sum, scale, add != 0);
      } else {
        float4* p = reinterpret_cast<float4*>(part + ((size_t)blockIdx.x * 2 + (begins ? 1 : 0)) * H) + 2 * j;
        p[0] = make_float4(sum[0], sum[1], sum[2], sum[3]);
        p[1] = make_float4(sum[4], sum[5], sum[6], sum[7]);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] = 0.f;
      begins = true;
    }
  }
}

// The chunk in which a border-crossing segment begins joins its parts.
template <typename G>
__global__ void join_kernel(const u64* __restrict__ keys, const float* __restrict__ part, G* __restrict__ dtable,
                            float scale, int add, int T, int V, int H) {
  const int c = blockIdx.x;
  const int first = c * kChunk, next = first + kChunk;
  if (next >= T) return;
  const int id = key_id(keys[next - 1]);
  if (id >= V || key_id(keys[next]) != id) return;                                    // nothing crosses this border
  if (key_id(keys[first]) == id && first > 0 && key_id(keys[first - 1]) == id) return;  // it began earlier
  const int j = blockIdx.y * blockDim.x + threadIdx.x;
  if (j * 8 >= H) return;
  float sum[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  size_t slot = (size_t)c * 2 + 1;
  for (int d = c;;) {
    const float4* p = reinterpret_cast<const float4*>(part + slot * H) + 2 * j;
    const float4 a = p[0], b = p[1];
    sum[0] += a.x; sum[1] += a.y; sum[2] += a.z; sum[3] += a.w;
    sum[4] += b.x; sum[5] += b.y; sum[6] += b.z; sum[7] += b.w;
    ++d;
    if (d * kChunk >= T || key_id(keys[d * kChunk]) != id) break;
    slot = (size_t)d * 2;
  }
  write_row<G>(dtable + (size_t)id * H, j, sum, scale, add != 0);
}

int slab_threads(int H) { return std::min(128, (H / 8 + 31) / 32 * 32); }

template <typename G>
void grad(const u64* keys, const at::Tensor& dy, long ldy, at::Tensor& dtable, float* part, float scale, bool add,
          int T, int V, int H, cudaStream_t st) {
  const int threads = slab_threads(H);
  const dim3 grid((T + kChunk - 1) / kChunk, (H / 8 + threads - 1) / threads);
  G* out = reinterpret_cast<G*>(dtable.data_ptr());
  segments_kernel<G><<<grid, threads, 0, st>>>(keys, (const __nv_bfloat16*)dy.data_ptr(), ldy, out, part, scale,
                                               add ? 1 : 0, T, V, H);
  check_cuda(cudaGetLastError(), "embed segments");
  if (grid.x > 1) {
    join_kernel<G><<<grid, threads, 0, st>>>(keys, part, out, scale, add ? 1 : 0, T, V, H);
    check_cuda(cudaGetLastError(), "embed join");
  }
}

void check_ids(const at::Tensor& ids, const at::Tensor& like) {
  TORCH_CHECK(ids.device() == like.device() && ids.scalar_type() == at::kLong && ids.dim() == 1 && ids.is_contiguous(),
              "embed: ids must be a contiguous int64 vector on the table's device");
  TORCH_CHECK(ids.numel() < (int64_t(1) << 30), "embed: at most 2^30 tokens");
}

void check_rows(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.scalar_type() == at::kBFloat16 && t.dim() == 2 && t.stride(1) == 1 &&
                  (t.size(0) <= 1 || t.stride(0) % 8 == 0) && t.size(1) >= 8 && t.size(1) % 8 == 0 &&
                  reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0,
              "embed: ", name, " must be bf16 with contiguous 16-byte aligned rows, H a multiple of 8");
}

}  // namespace embed

void embed_scaled(const at::Tensor& ids, const at::Tensor& table, at::Tensor& out, double scale) {
  using namespace embed;
  check_rows(table, "table");
  check_rows(out, "out");
  check_ids(ids, table);
  const long T = ids.numel();
  const int H = table.size(1);
  TORCH_CHECK(table.size(0) < (int64_t(1) << 30), "embed: at most 2^30 table rows");
  TORCH_CHECK(out.device() == table.device() && out.size(0) == T && out.size(1) == H && out.is_contiguous(),
              "embed: out must be contiguous [T, H]");
  if (T == 0) return;
  c10::cuda::CUDAGuard g(table.device());
  const int threads = std::min(256, (H / 8 + 31) / 32 * 32);
  lookup_kernel<<<(int)std::min<long>(T, 1 << 20), threads, 0, at::cuda::getCurrentCUDAStream()>>>(
      ids.data_ptr<long>(), (const __nv_bfloat16*)table.data_ptr(), table.stride(0), (__nv_bfloat16*)out.data_ptr(),
      (float)scale, T, (int)table.size(0), H);
  check_cuda(cudaGetLastError(), "embed_scaled");
}

void embed_grad_sorted(const at::Tensor& ids, const at::Tensor& dy, at::Tensor& dtable, double scale,
                       bool accumulate) {
  using namespace embed;
  check_rows(dy, "dy");
  check_ids(ids, dy);
  const bool f32 = dtable.scalar_type() == at::kFloat;
  TORCH_CHECK(dtable.device() == dy.device() && (f32 || dtable.scalar_type() == at::kBFloat16) && dtable.dim() == 2 &&
                  dtable.is_contiguous() && reinterpret_cast<uintptr_t>(dtable.data_ptr()) % 16 == 0,
              "embed: dtable must be a contiguous bf16 or fp32 table on 16 bytes");
  const int T = ids.numel(), H = dy.size(1);
  TORCH_CHECK(dy.size(0) == T && dtable.size(1) == H, "embed: dy [T, H] and dtable [V, H] do not fit the ids");
  TORCH_CHECK(dtable.size(0) < (int64_t(1) << 30), "embed: at most 2^30 table rows");
  const int V = dtable.size(0);
  c10::cuda::CUDAGuard g(dy.device());
  auto st = at::cuda::getCurrentCUDAStream();
  if (!accumulate)
    check_cuda(cudaMemsetAsync(dtable.data_ptr(), 0, (size_t)dtable.numel() * dtable.element_size(), st),
               "embed zero rows");
  if (T == 0) return;
  const int tiles = (T + kTile - 1) / kTile, chunks = (T + kChunk - 1) / kChunk;
  at::Tensor keys = at::empty({(int64_t)T * (tiles > 1 ? 2 : 1)}, ids.options());
  at::Tensor part = at::empty({chunks > 1 ? (int64_t)chunks * 2 * H : 0}, dy.options().dtype(at::kFloat));
  u64* k = reinterpret_cast<u64*>(keys.data_ptr<long>());
  sort_tiles_kernel<<<tiles, kSortThreads, 0, st>>>(ids.data_ptr<long>(), k, T, V);
  check_cuda(cudaGetLastError(), "embed sort");
  if (tiles > 1) {
    rank_kernel<<<(T + 255) / 256, 256, 0, st>>>(k, k + T, T);
    check_cuda(cudaGetLastError(), "embed rank");
    k += T;
  }
  const long ldy = T > 1 ? dy.stride(0) : H;
  if (f32) grad<float>(k, dy, ldy, dtable, part.data_ptr<float>(), (float)scale, accumulate, T, V, H, st);
  else grad<__nv_bfloat16>(k, dy, ldy, dtable, part.data_ptr<float>(), (float)scale, accumulate, T, V, H, st);
}

}  // namespace kore
