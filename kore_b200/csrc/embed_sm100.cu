// Token embedding with scaling, and its gradient by sorted tokens.
//
//   out_t = s E[id_t]                          dE_v (+)= s sum_{t: id_t = v} dy_t
//
// The sum runs over a token's positions in ascending order in fp32 and is
// rounded once when the row is written, so the gradient does not depend on the
// order in which blocks run and a frequent token loses nothing to repeated
// bf16 additions. ids outside [0, V) read a zero row and receive no gradient.
//
// Gradient: the keys (id, position) are distinct, so a key's place in the sorted
// order is the number of smaller keys. Within a tile of kTile tokens the ids are
// compared one by one; the places in the other tiles are found by binary search.
// The sorted positions are cut in chunks of kChunk; a block sums its chunk's
// rows segment by segment. A segment inside a chunk goes straight to its row;
// what crosses a chunk's border goes to a workspace and is joined by the chunk
// where it begins, in chunk order. A token with thousands of positions is thus
// summed by many blocks. When the table is overwritten, further blocks of the
// same launch write zeros to the rows that no token has.
//
// Bound by HBM, mostly by writing the table: at T = 16384, V = 151936, H = 5120
// (bf16 table) the gradient takes 325 us, 5.3 TB/s over its 1.72 GB (launched one
// by one: places 28, rows and zeros 270, joins 10); zeros by bulk copies from shared memory
// because they need no registers (a plain fill of the table alone: 395 us). The
// lookup takes 40 us (8.3 TB/s: a frequent token's row comes from L2).
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "common.cuh"
#include "tma_host.h"

namespace kore {
namespace embed {

typedef unsigned long long u64;

constexpr int kTile = 1024;      // tokens whose ids are compared one by one
constexpr int kRankThreads = 256;
constexpr int kChunk = 32;       // sorted positions per block
// Up to this many tokens a block walks the segments that begin in its 4 positions
// to their ends: no workspace and one launch less (T = 129: 5 us; the longest walk,
// one id everywhere, is 64 steps). Beyond it long segments are split over blocks.
constexpr int kWalk = 256;
constexpr int kZeroRows = 128;   // table rows per zero-writing block
constexpr int kZeroBytes = 4096;

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

// blockDim.x * VPT 8-column vectors cover a row: all loads are issued before the
// first store (rows of 1024 columns and more: four per thread, 40 us at 16384 x 5120,
// 65 us with one)
template <int VPT>
__global__ void lookup_kernel(const long* ids, const __nv_bfloat16* table, long ldt,
                              __nv_bfloat16* __restrict__ out, float scale, int V, int H) {
  const int nvec = H / 8;
  const long t = blockIdx.x;
  pdl_wait();
  pdl_trigger();
  const long id = ids[t];
  const bool ok = id >= 0 && id < V;
  for (int j0 = threadIdx.x; j0 < nvec; j0 += VPT * blockDim.x) {
    uint4 u[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int j = j0 + i * blockDim.x;
      u[i] = make_uint4(0, 0, 0, 0);
      if (ok && j < nvec) u[i] = reinterpret_cast<const uint4*>(table + id * ldt)[j];
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int j = j0 + i * blockDim.x;
      if (scale != 1.f) {
        float f[8];
        unpack8(u[i], f);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] *= scale;
        u[i] = pack8(f);
      }
      if (j < nvec) reinterpret_cast<uint4*>(out + t * (long)H)[j] = u[i];
    }
  }
}

// Places of kRankThreads tokens within their tile of kTile: the key (id << 32 |
// position) goes to that place. ids outside the table count as V, behind all others.
__global__ void __launch_bounds__(kRankThreads) rank_in_tile_kernel(const long* ids, u64* __restrict__ keys, int T,
                                                                    int V) {
  __shared__ __align__(16) int s_id[kTile];
  const int i = blockIdx.x * kRankThreads + threadIdx.x;
  const int base = i / kTile * kTile;            // the same for all threads of the block
  const int n = min(kTile, T - base);
  pdl_wait();
  pdl_trigger();
  {
    long id[kTile / kRankThreads];
#pragma unroll
    for (int r = 0; r < kTile / kRankThreads; ++r) {
      const int j = threadIdx.x + r * kRankThreads;
      id[r] = j < n ? ids[base + j] : V;
    }
#pragma unroll
    for (int r = 0; r < kTile / kRankThreads; ++r)
      s_id[threadIdx.x + r * kRankThreads] = id[r] >= 0 && id[r] < V ? (int)id[r] : V;
  }
  __syncthreads();
  if (i >= T) return;
  const int own = i - base, id = s_id[own];
  const int4* s4 = reinterpret_cast<const int4*>(s_id);
  int rank = 0;
  // before this token: keys with an id up to its own are smaller; after it: with a smaller id
  const int cut = own / 4;
#pragma unroll 4
  for (int j = 0; j < cut; ++j) {
    const int4 v = s4[j];
    rank += (v.x <= id) + (v.y <= id) + (v.z <= id) + (v.w <= id);
  }
  for (int j = cut * 4; j < own; ++j) rank += s_id[j] <= id;
  for (int j = own + 1; j < min(cut * 4 + 4, n); ++j) rank += s_id[j] < id;
  const int full = n / 4;
#pragma unroll 4
  for (int j = cut + 1; j < full; ++j) {
    const int4 v = s4[j];
    rank += (v.x < id) + (v.y < id) + (v.z < id) + (v.w < id);
  }
  for (int j = max(full, cut + 1) * 4; j < n; ++j) rank += s_id[j] < id;
  keys[base + rank] = ((u64)(uint32_t)id << 32) | (uint32_t)i;
}

// Places among all tiles: 8 tiles are searched at once, without branches, so
// that their loads overlap.
__global__ void rank_kernel(const u64* tiles, u64* __restrict__ keys, int T) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  pdl_wait();
  pdl_trigger();
  if (i >= T) return;
  const u64 key = tiles[i];
  const int num = (T + kTile - 1) / kTile;
  int rank = 0;
  for (int j0 = 0; j0 < num; j0 += 8) {
    int pos[8], n[8];   // keys known to be smaller, keys of the tile
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      pos[u] = 0;
      n[u] = j0 + u < num ? min(kTile, T - (j0 + u) * kTile) : 0;
    }
#pragma unroll
    for (int s = kTile; s > 0; s >>= 1) {
      u64 k[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) k[u] = pos[u] + s <= n[u] ? tiles[(size_t)(j0 + u) * kTile + pos[u] + s - 1] : ~0ull;
#pragma unroll
      for (int u = 0; u < 8; ++u) pos[u] += k[u] < key ? s : 0;
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) rank += pos[u];
  }
  keys[rank] = key;
}

KORE_DEV int key_id(u64 k) { return (int)(k >> 32); }

// Zeros in the rows [r0, r0 + kZeroRows) of the table that no sorted key names:
// a thread per row sends copies of a zeroed piece of shared memory.
template <typename G>
KORE_DEV void zero_rows(const u64* keys, G* __restrict__ dtable, int r0, int T, int V, int H) {
  __shared__ __align__(128) uint4 s_zero[kZeroBytes / 16];
  for (int i = threadIdx.x; i < kZeroBytes / 16; i += blockDim.x) s_zero[i] = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  __syncthreads();
  const int bytes = H * (int)sizeof(G);
  for (int r = r0 + threadIdx.x; r < min(r0 + kZeroRows, V); r += blockDim.x) {
    int lo = 0, hi = T;
    const u64 key = (u64)(uint32_t)r << 32;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (keys[mid] < key) lo = mid + 1; else hi = mid;
    }
    if (lo < T && key_id(keys[lo]) == r) continue;
    uint8_t* row = reinterpret_cast<uint8_t*>(dtable + (size_t)r * H);
    for (int b = 0; b < bytes; b += kZeroBytes)
      asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(row + b),
                   "r"(smem_u32(s_zero)), "r"(min(kZeroBytes, bytes - b))
                   : "memory");
  }
  tma_store_commit();
  tma_store_wait_all<0>();
}

// a row's 8 columns before the sum is added
template <typename G>
struct Old;
template <>
struct Old<float> { float4 a, b; };
template <>
struct Old<__nv_bfloat16> { uint4 a; };

KORE_DEV void read_old(Old<float>& o, const float* row, int j) {
  o.a = reinterpret_cast<const float4*>(row)[2 * j];
  o.b = reinterpret_cast<const float4*>(row)[2 * j + 1];
}
KORE_DEV void read_old(Old<__nv_bfloat16>& o, const __nv_bfloat16* row, int j) {
  o.a = reinterpret_cast<const uint4*>(row)[j];
}
KORE_DEV void write_row(float* row, int j, const float (&sum)[8], float scale, bool add, const Old<float>& o) {
  float4 a = make_float4(sum[0] * scale, sum[1] * scale, sum[2] * scale, sum[3] * scale);
  float4 b = make_float4(sum[4] * scale, sum[5] * scale, sum[6] * scale, sum[7] * scale);
  if (add) {
    a.x += o.a.x; a.y += o.a.y; a.z += o.a.z; a.w += o.a.w;
    b.x += o.b.x; b.y += o.b.y; b.z += o.b.z; b.w += o.b.w;
  }
  reinterpret_cast<float4*>(row)[2 * j] = a;
  reinterpret_cast<float4*>(row)[2 * j + 1] = b;
}
KORE_DEV void write_row(__nv_bfloat16* row, int j, const float (&sum)[8], float scale, bool add,
                        const Old<__nv_bfloat16>& o) {
  float f[8];
  if (add) {
    unpack8(o.a, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = fmaf(sum[e], scale, f[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = sum[e] * scale;
  }
  reinterpret_cast<uint4*>(row)[j] = pack8(f);
}

// grid: `chunks` blocks of `chunk` sorted positions, then the zero-writing
// blocks (overwriting launches); y: slabs of blockDim.x 8-column vectors.
// walk: a block sums the segments that begin in its chunk to their ends and
// passes over what began before (no workspace, no second launch).
template <typename G>
__global__ void segments_kernel(const u64* keys, const __nv_bfloat16* dy, long ldy,
                                G* __restrict__ dtable, float* __restrict__ part, float scale, int add, int chunk,
                                int chunks, int walk, int T, int V, int H) {
  __shared__ int s_id[kChunk + 2];
  __shared__ int s_pos[kChunk];
  pdl_wait();
  pdl_trigger();
  if ((int)blockIdx.x >= chunks) {
    if (blockIdx.y == 0) zero_rows<G>(keys, dtable, ((int)blockIdx.x - chunks) * kZeroRows, T, V, H);
    return;
  }
  const int first = blockIdx.x * chunk;
  const int j = blockIdx.y * blockDim.x + threadIdx.x;
  const bool mine = j * 8 < H;
  const uint4* src = reinterpret_cast<const uint4*>(dy) + j;
  const long ld = ldy / 8;
  float sum[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  bool begins = false;
  for (int at = first, n; at < T; at += n) {
    n = min(chunk, T - at);
    __syncthreads();
    for (int i = threadIdx.x; i < n + 2; i += blockDim.x) {
      const int k = at + i - 1;
      const bool in = k >= 0 && k < T;
      const u64 key = in ? keys[k] : 0;
      s_id[i] = in ? key_id(key) : -1;
      if (i >= 1 && i <= n) s_pos[i - 1] = (int)(uint32_t)key;
    }
    __syncthreads();
    const bool beyond = at > first;     // (walk) only the segment that is still open
    if (!beyond) begins = s_id[0] != s_id[1];
    if (beyond && s_id[0] != s_id[1]) break;
    bool done = false, open = begins;   // open: the segment being summed begins in this chunk
    for (int i0 = 0; i0 < n && !done && mine; i0 += 8) {
      uint4 v[8];
      Old<G> old[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int i = i0 + u;
        if (i < n && s_id[i + 1] < V) {
          v[u] = src[s_pos[i] * ld];
          if (add && s_id[i + 2] != s_id[i + 1]) read_old(old[u], dtable + (size_t)s_id[i + 1] * H, j);
        }
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int i = i0 + u;
        if (i >= n || done) break;
        const int id = s_id[i + 1];
        if (id >= V) { done = true; break; }  // ids outside the table are last
        float f[8];
        unpack8(v[u], f);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += f[e];
        const bool ends = s_id[i + 2] != id;
        if (!ends && (walk || i + 1 < n)) continue;
        if (open && ends) {
          write_row(dtable + (size_t)id * H, j, sum, scale, add != 0, old[u]);
        } else if (!walk) {
          float4* p = reinterpret_cast<float4*>(part + ((size_t)blockIdx.x * 2 + (open ? 1 : 0)) * H) + 2 * j;
          p[0] = make_float4(sum[0], sum[1], sum[2], sum[3]);
          p[1] = make_float4(sum[4], sum[5], sum[6], sum[7]);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] = 0.f;
        open = true;
        if (beyond) done = true;
      }
    }
    // walk on while the last segment is open and began in this block's chunk; every test
    // here is the same for all threads, those without columns load keys for the others
    begins = begins || s_id[1] != s_id[n];
    if (!walk || s_id[n + 1] != s_id[n] || s_id[n] >= V) break;
    if (beyond && s_id[n] != s_id[0]) break;   // it has ended; what is open now began later
    if (!begins) break;
  }
}

// The chunk in which a border-crossing segment begins joins its parts.
template <typename G>
__global__ void join_kernel(const u64* keys, const float* part, G* __restrict__ dtable,
                            float scale, int add, int T, int V, int H) {
  __shared__ int s_last;
  const int c = blockIdx.x;
  const int first = c * kChunk, next = first + kChunk;
  pdl_wait();
  pdl_trigger();
  if (next >= T) return;
  const int id = key_id(keys[next - 1]);
  if (id >= V || key_id(keys[next]) != id) return;                                    // nothing crosses this border
  if (key_id(keys[first]) == id && first > 0 && key_id(keys[first - 1]) == id) return;  // it began earlier
  // the first chunk after c whose first key is another's: all threads look at once
  const int chunks = (T + kChunk - 1) / kChunk;
  if (threadIdx.x == 0) s_last = chunks;
  __syncthreads();
  int last;
  for (int d0 = c + 1;; d0 += blockDim.x) {
    const int d = d0 + threadIdx.x;
    if (d < chunks && key_id(keys[d * kChunk]) != id) atomicMin(&s_last, d);
    __syncthreads();
    last = s_last;
    if (last < chunks || d0 + (int)blockDim.x >= chunks) break;
    __syncthreads();   // all have read it before the next turn lowers it
  }
  const int j = blockIdx.y * blockDim.x + threadIdx.x;
  if (j * 8 >= H) return;
  float sum[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  for (int d0 = c; d0 < last; d0 += 8) {
    float4 a[8], b[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int d = d0 + u;
      if (d < last) {
        const float4* p = reinterpret_cast<const float4*>(part + ((size_t)d * 2 + (d == c ? 1 : 0)) * H) + 2 * j;
        a[u] = p[0];
        b[u] = p[1];
      }
    }
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (d0 + u < last) {
        sum[0] += a[u].x; sum[1] += a[u].y; sum[2] += a[u].z; sum[3] += a[u].w;
        sum[4] += b[u].x; sum[5] += b[u].y; sum[6] += b[u].z; sum[7] += b[u].w;
      }
  }
  Old<G> old;
  G* row = dtable + (size_t)id * H;
  if (add) read_old(old, row, j);
  write_row(row, j, sum, scale, add != 0, old);
}

template <typename G>
void grad(const u64* keys, const at::Tensor& dy, long ldy, at::Tensor& dtable, float* part, float scale, bool add,
          int T, int V, int H, cudaStream_t st) {
  const int threads = std::min(128, (H / 8 + 31) / 32 * 32), slabs = (H / 8 + threads - 1) / threads;
  const bool walk = T <= kWalk;
  const int chunk = walk ? 4 : kChunk, chunks = (T + chunk - 1) / chunk;
  const int zero = add ? 0 : (V + kZeroRows - 1) / kZeroRows;
  G* out = reinterpret_cast<G*>(dtable.data_ptr());
  launch_after("embed segments", segments_kernel<G>, dim3(chunks + zero, slabs), dim3(threads), 0, st, keys,
               (const __nv_bfloat16*)dy.data_ptr(), ldy, out, part, scale, add ? 1 : 0, chunk, chunks, walk ? 1 : 0, T, V,
               H);
  if (!walk)
    launch_after("embed join", join_kernel<G>, dim3(chunks, slabs), dim3(threads), 0, st, keys, part, out, scale,
                 add ? 1 : 0, T, V, H);
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

at::Tensor embed_scaled(const at::Tensor& ids, const at::Tensor& table, const c10::optional<at::Tensor>& into,
                        double scale) {
  using namespace embed;
  check_rows(table, "table");
  check_ids(ids, table);
  const long T = ids.numel();
  const int H = table.size(1);
  TORCH_CHECK(table.size(0) < (int64_t(1) << 30), "embed: at most 2^30 table rows");
  if (into) {
    check_rows(*into, "out");
    TORCH_CHECK(into->device() == table.device() && into->size(0) == T && into->size(1) == H && into->is_contiguous(),
                "embed: out must be contiguous [T, H]");
  }
  c10::cuda::CUDAGuard g(table.device());
  at::Tensor out = into ? *into : at::empty({T, H}, table.options());
  if (T == 0) return out;
  const int nvec = H / 8;
  auto st = at::cuda::getCurrentCUDAStream();
  const int vpt = nvec >= 128 ? 4 : 1;
  launch_after("embed_scaled", vpt == 4 ? lookup_kernel<4> : lookup_kernel<1>, dim3((unsigned)T),
               dim3(std::min(256, ((nvec + vpt - 1) / vpt + 31) / 32 * 32)), 0, st, ids.data_ptr<long>(),
               (const __nv_bfloat16*)table.data_ptr(), table.stride(0), (__nv_bfloat16*)out.data_ptr(), (float)scale,
               (int)table.size(0), H);
  return out;
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
  if (T == 0) {
    if (!accumulate) dtable.zero_();
    return;
  }
  const int tiles = (T + kTile - 1) / kTile, chunks = (T + kChunk - 1) / kChunk;
  at::Tensor keys = at::empty({(int64_t)T * (tiles > 1 ? 2 : 1)}, ids.options());
  at::Tensor part;
  if (T > kWalk) part = at::empty({(int64_t)chunks * 2 * H}, dy.options().dtype(at::kFloat));
  u64* k = reinterpret_cast<u64*>(keys.data_ptr<long>());
  launch_after("embed rank in tile", rank_in_tile_kernel, dim3((T + kRankThreads - 1) / kRankThreads),
               dim3(kRankThreads), 0, st, ids.data_ptr<long>(), k, T, V);
  if (tiles > 1) {
    launch_after("embed rank", rank_kernel, dim3((T + 127) / 128), dim3(128), 0, st, k, k + T, T);
    k += T;
  }
  float* pp = T > kWalk ? part.data_ptr<float>() : nullptr;
  const long ldy = T > 1 ? dy.stride(0) : H;
  if (f32) grad<float>(k, dy, ldy, dtable, pp, (float)scale, accumulate, T, V, H, st);
  else grad<__nv_bfloat16>(k, dy, ldy, dtable, pp, (float)scale, accumulate, T, V, H, st);
}

}  // namespace kore
