// Page operators: forking sequences that share pages, and compacting the pages a
// table refers to into another arena.
//
// Both move whole page records, byte for byte, and rewrite table entries on the
// device; neither looks at the values.  They are bound by HBM: a page is read
// once and written once (a compacted page that several entries share moves
// once), and the tables are 8 bytes a page beside 16 to 64 KB of payload.
#include <algorithm>
#include <atomic>

#include "akv_common.cuh"

namespace akv {

// Bytes of a page (all its heads) by mode; 0 for a skip entry.
struct PageBytes {
  int64_t of[4];
  __host__ __device__ int64_t operator()(int mode) const {
    return mode == AKV_MODE_INT4 ? of[1] : (mode == AKV_MODE_INT8 ? of[2] : (mode == AKV_MODE_FP16 ? of[3] : 0));
  }
};
static PageBytes page_bytes(int heads, int head_dim, int group) {
  PageBytes b;
  for (int mode = 0; mode < 4; ++mode) b.of[mode] = heads * record_bytes(head_dim, group, mode);
  return b;
}

constexpr int kCopyThreads = 256;

// Copy 16-byte units [lo, hi) of a page by one CTA, U loads of a thread in flight
// before the first is stored.
template <int U>
__device__ __forceinline__ void copy_units(const uint8_t *src, uint8_t *dst, int lo, int hi) {
  const uint4 *s = reinterpret_cast<const uint4 *>(src);
  uint4 *d = reinterpret_cast<uint4 *>(dst);
  for (int i = lo + (int)threadIdx.x; i < hi; i += U * kCopyThreads) {
    uint4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + u * kCopyThreads < hi) v[u] = __ldg(s + i + u * kCopyThreads);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + u * kCopyThreads < hi) d[i + u * kCopyThreads] = v[u];
  }
}

// ==================================================================== fork
struct ForkParams {
  const int64_t *table;
  int64_t layer_stride, seq_stride;
  int32_t batch, children, columns, uniform_tokens, parts;
  const int32_t *tokens;
  const int64_t *parents, *fresh;
  int64_t *out;
  uint8_t *arena;
  int64_t arena_bytes;
  PageBytes bytes;
  int32_t *status;
};

// One CTA per (layer, child, part): it writes its share of the child's table row
// and copies its share of the page that the child's next token goes to, when
// that page is half filled and the child was given a fresh slot.
__global__ void __launch_bounds__(kCopyThreads) fork_pages_kernel(const ForkParams p) {
  grid_dependency_wait();
  allow_dependents_launch();
  const int part = blockIdx.x % p.parts;
  const int64_t row = blockIdx.x / p.parts;  // layer * children + child
  const int child = (int)(row % p.children);
  const int64_t layer = row / p.children;
  int64_t *out = p.out + row * p.columns;
  const int64_t fresh = p.fresh ? p.fresh[row] : 0;
  const int c0 = (int)((int64_t)p.columns * part / p.parts), c1 = (int)((int64_t)p.columns * (part + 1) / p.parts);
  const int64_t parent = p.parents[child];
  if (parent < 0 || parent >= p.batch) {  // no such sequence: an empty row
    if (threadIdx.x == 0 && part == 0) set_status(p.status, AKV_DEV_BAD_PARENT);
    for (int c = c0 + threadIdx.x; c < c1; c += kCopyThreads) out[c] = 0;
    return;
  }
  const int64_t *src_row = p.table + layer * p.layer_stride + parent * p.seq_stride;
  const int tokens = p.tokens ? p.tokens[parent] : p.uniform_tokens;
  int copied = -1;  // the column whose page is copied
  int64_t old = 0;
  if (fresh != 0 && tokens > 0 && tokens % kBlock != 0 && tokens / kBlock < p.columns) {
    old = src_row[tokens / kBlock];
    const int mode = desc_mode(old);
    if (mode != AKV_MODE_SKIP) {
      if (mode == desc_mode(fresh) && page_in_arena(old, p.bytes(mode), p.arena_bytes) &&
          page_in_arena(fresh, p.bytes(mode), p.arena_bytes))
        copied = tokens / kBlock;
      else if (threadIdx.x == 0 && part == 0)  // the child goes on sharing the parent's page
        set_status(p.status, AKV_DEV_BAD_DESCRIPTOR);
    }
  }
  for (int c = c0 + threadIdx.x; c < c1; c += kCopyThreads)
    out[c] = c == copied ? (fresh & ~(int64_t)255) | (old & 255) : src_row[c];
  if (copied < 0) return;
  const int64_t units = p.bytes(desc_mode(old)) / 16;
  copy_units<8>(p.arena + desc_offset(old), p.arena + desc_offset(fresh), (int)(units * part / p.parts),
             (int)(units * (part + 1) / p.parts));
}

// ================================================================= compact
// The pages that a table names move to another arena, each once, in the order
// in which the table first names them within their precision:
//   mark   owner[key] = the first entry naming the page (a key per page: two pages
//          of one arena start at least the smallest page apart);
//   count  owners of each precision per block of 1024 entries;
//   rank   an owner's rank is the owners before it; place[key] = its new offset;
//   move   owners copy their page, every entry is rewritten through place[key].
constexpr int kRankThreads = 1024;
// Entries and keys that one CTA plans, in shared memory: it takes about 8 us, the launches
// of the four kernels of a larger plan cost more.  A call for 3700 entries that name 87 MB
// of pages: 26 us (27 with the owners in global memory), 13 of them the copy's floor.
constexpr int kOnePlan = 8192, kOnePlanKeys = 48 << 10;

struct CompactParams {
  const int64_t *table;
  int64_t n;
  int64_t *out;
  const uint8_t *arena;
  int64_t arena_bytes;
  uint8_t *into;
  int64_t base[4], capacity[4];  // of the target's slots, by mode
  PageBytes bytes;
  int64_t unit;  // bytes of the smallest page
  uint32_t *owner;
  int64_t *place;
  int32_t *counts;  // [blocks][4]
  int32_t blocks;
  int32_t *status;
};

__device__ __forceinline__ bool movable(const CompactParams &p, int64_t d) {
  const int mode = desc_mode(d);
  return mode != AKV_MODE_SKIP && page_in_arena(d, p.bytes(mode), p.arena_bytes);
}

__global__ void __launch_bounds__(256) compact_mark_kernel(const CompactParams p) {
  allow_dependents_launch();
  for (int64_t e = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; e < p.n; e += (int64_t)gridDim.x * blockDim.x) {
    const int64_t d = p.table[e];
    if (movable(p, d)) atomicMin(p.owner + desc_offset(d) / p.unit, (uint32_t)e);
    else if (desc_mode(d) != AKV_MODE_SKIP) set_status(p.status, AKV_DEV_BAD_DESCRIPTOR);
  }
}

// The rank of this thread's entry among the owners of its precision within the CTA
// (mode 0: none), and how many each precision has there.
__device__ __forceinline__ int block_rank(int mode, int (&warps)[4][32], int (&all)[4]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int rank = 0;
#pragma unroll
  for (int m = 1; m < 4; ++m) {
    const uint32_t mask = __ballot_sync(0xffffffffu, mode == m);
    if (mode == m) rank = __popc(mask & ((1u << lane) - 1u));
    if (lane == 0) warps[m][warp] = __popc(mask);
  }
  __syncthreads();
#pragma unroll
  for (int m = 1; m < 4; ++m) {
    const int n = warps[m][lane];
    const int before = __reduce_add_sync(0xffffffffu, lane < warp ? n : 0);
    all[m] = __reduce_add_sync(0xffffffffu, n);
    if (mode == m) rank += before;
  }
  __syncthreads();
  return rank;
}
__device__ __forceinline__ void set_place(const CompactParams &p, int64_t d, int rank) {
  const int mode = desc_mode(d);
  const bool fits = rank < p.capacity[mode];  // else: more pages than the target holds, skip entries
  if (!fits) set_status(p.status, AKV_DEV_BAD_DESCRIPTOR);
  p.place[desc_offset(d) / p.unit] = fits ? p.base[mode] + rank * p.bytes(mode) : -1;
}

// The mode of entry e when it is the first to name its page, else 0.
__device__ __forceinline__ int owner_mode(const CompactParams &p, int64_t e, int64_t &d) {
  d = e < p.n ? p.table[e] : 0;
  return movable(p, d) && __ldcg(p.owner + desc_offset(d) / p.unit) == (uint32_t)e ? desc_mode(d) : 0;
}

__global__ void __launch_bounds__(kRankThreads) compact_count_kernel(const CompactParams p) {
  grid_dependency_wait();
  allow_dependents_launch();
  int64_t d;
  const int mode = owner_mode(p, blockIdx.x * (int64_t)kRankThreads + threadIdx.x, d);
#pragma unroll
  for (int m = 1; m < 4; ++m) {
    const int n = __syncthreads_count(mode == m);
    if (threadIdx.x == 0) p.counts[4 * blockIdx.x + m] = n;
  }
}

__global__ void __launch_bounds__(kRankThreads) compact_rank_kernel(const CompactParams p) {
  __shared__ int before[4], warps[4][32];
  grid_dependency_wait();
  allow_dependents_launch();
  if (threadIdx.x < 4) before[threadIdx.x] = 0;
  __syncthreads();
  // owners of each precision in the blocks before this one
  int sum[4] = {0, 0, 0, 0};
  for (int b = threadIdx.x; b < (int)blockIdx.x; b += kRankThreads)
#pragma unroll
    for (int m = 1; m < 4; ++m) sum[m] += __ldcg(p.counts + 4 * b + m);
#pragma unroll
  for (int m = 1; m < 4; ++m) {
    const int s = __reduce_add_sync(0xffffffffu, sum[m]);
    if ((threadIdx.x & 31) == 0 && s) atomicAdd(&before[m], s);  // integers: any order gives the same sum
  }
  int64_t d;
  const int mode = owner_mode(p, blockIdx.x * (int64_t)kRankThreads + threadIdx.x, d);
  int all[4];
  const int rank = block_rank(mode, warps, all);
  if (mode != 0) set_place(p, d, before[mode] + rank);
}

// Small tables: all of the plan in one CTA, which saves three launches.
__global__ void __launch_bounds__(kRankThreads) compact_plan_kernel(const CompactParams p, int keys) {
  __shared__ int warps[4][32];
  grid_dependency_wait();
  allow_dependents_launch();
  extern __shared__ __align__(16) uint32_t owner[];
  for (int k = threadIdx.x; k < (keys + 3) / 4; k += kRankThreads)
    reinterpret_cast<uint4 *>(owner)[k] = make_uint4(~0u, ~0u, ~0u, ~0u);
  __syncthreads();
  constexpr int N = kOnePlan / kRankThreads;  // entries of a thread, their loads in flight together
  int64_t d[N];
  int64_t key[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int e = i * kRankThreads + threadIdx.x;
    d[i] = e < (int)p.n ? p.table[e] : 0;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    key[i] = -1;
    if (movable(p, d[i])) {
      key[i] = desc_offset(d[i]) / p.unit;
      atomicMin(owner + key[i], (uint32_t)(i * kRankThreads + threadIdx.x));
    } else if (desc_mode(d[i]) != AKV_MODE_SKIP) {
      set_status(p.status, AKV_DEV_BAD_DESCRIPTOR);
    }
  }
  __syncthreads();
  uint32_t first[N];
#pragma unroll
  for (int i = 0; i < N; ++i) first[i] = key[i] >= 0 ? owner[key[i]] : ~0u;
  int before[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (i * kRankThreads >= (int)p.n) break;
    const int mode = first[i] == (uint32_t)(i * kRankThreads + threadIdx.x) ? desc_mode(d[i]) : 0;
    int all[4];
    const int rank = block_rank(mode, warps, all);
    if (mode != 0) {
      p.owner[key[i]] = first[i];
      set_place(p, d[i], before[mode] + rank);
    }
#pragma unroll
    for (int m = 1; m < 4; ++m) before[m] += all[m];
  }
}

// One CTA per table entry.
__global__ void __launch_bounds__(kCopyThreads) compact_move_kernel(const CompactParams p) {
  const int64_t e = blockIdx.x;
  grid_dependency_wait();
  allow_dependents_launch();
  const int64_t d = p.table[e];
  if (!movable(p, d)) {
    if (threadIdx.x == 0) p.out[e] = 0;
    return;
  }
  const int64_t key = desc_offset(d) / p.unit;
  const uint32_t owner = __ldcg(p.owner + key);
  const int64_t place = __ldcg(p.place + key);
  // An entry that overlaps another page without being it cannot move.
  const bool same = owner == (uint32_t)e || ((p.table[owner] ^ d) & ~(int64_t)0xfc) == 0;
  if (threadIdx.x == 0) {
    if (!same) set_status(p.status, AKV_DEV_BAD_DESCRIPTOR);
    p.out[e] = !same || place < 0 ? 0 : (place << 8) | (d & 255);
  }
  if (owner != (uint32_t)e || place < 0) return;
  copy_units<4>(p.arena + desc_offset(d), p.into + place, 0, (int)(p.bytes(desc_mode(d)) / 16));
}

static int check_page_geometry(int heads, int head_dim, int group) {
  if (heads <= 0) return AKV_ERR_INVALID;
  if (head_dim != 64 && head_dim != 128) return AKV_ERR_UNSUPPORTED;
  if (group != 32 && group != 64 && group != 128 && group != 16 * head_dim) return AKV_ERR_UNSUPPORTED;
  return AKV_OK;
}
static bool overlap(const void *a, int64_t a_bytes, const void *b, int64_t b_bytes) {
  return (const uint8_t *)a < (const uint8_t *)b + b_bytes && (const uint8_t *)b < (const uint8_t *)a + a_bytes;
}
// Raise the small plan's shared-memory limit, once per device.
static cudaError_t plan_ready() {
  static std::atomic<bool> ready[256];
  int dev = 0;
  if (cudaError_t err = cudaGetDevice(&dev)) return err;
  if (dev < 256 && ready[dev].load(std::memory_order_acquire)) return cudaSuccess;
  if (cudaError_t err = cudaFuncSetAttribute(compact_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 4 * kOnePlanKeys))
    return err;
  if (dev < 256) ready[dev].store(true, std::memory_order_release);
  return cudaSuccess;
}
static int64_t round16(int64_t n) { return (n + 15) & ~(int64_t)15; }

struct CompactSizes {
  int64_t keys, blocks, place_at, owner_at, counts_at, bytes;
};
static CompactSizes compact_sizes(int64_t entries, int64_t arena_bytes, int64_t unit) {
  CompactSizes z;
  z.keys = arena_bytes / unit + 1;
  z.blocks = (entries + kRankThreads - 1) / kRankThreads;
  z.place_at = 0;
  z.owner_at = round16(8 * z.keys);
  z.counts_at = z.owner_at + round16(4 * z.keys);
  z.bytes = z.counts_at + round16(16 * z.blocks);
  return z;
}

}  // namespace akv

using namespace akv;

extern "C" int akv_fork_pages(const int64_t *table, int64_t layer_stride, int64_t seq_stride, int32_t layers,
                              int32_t batch, int32_t columns, const int32_t *tokens, int32_t uniform_tokens,
                              const int64_t *parents, int32_t children, const int64_t *fresh, int64_t *out_table,
                              void *arena, int64_t arena_bytes, int heads, int head_dim, int group,
                              int32_t *dev_status, void *stream) {
  if (int st = check_page_geometry(heads, head_dim, group)) return st;
  if (layers <= 0 || batch <= 0 || children < 0 || columns < 0 || arena_bytes < 0) return AKV_ERR_INVALID;
  if (!table || !parents || !out_table || !arena || ((uintptr_t)arena & 15)) return AKV_ERR_INVALID;
  if (seq_stride < columns || (layers > 1 && layer_stride < 0) || (!tokens && uniform_tokens < 0)) return AKV_ERR_INVALID;
  const int64_t rows = (int64_t)layers * children;
  if (rows == 0 || columns == 0) return AKV_OK;
  const int64_t span = (layers - 1) * layer_stride + (int64_t)(batch - 1) * seq_stride + columns;
  if (overlap(table, 8 * span, out_table, 8 * rows * columns)) return AKV_ERR_INVALID;
  // A page is cut into 32 KB parts; finer, down to 8 KB, where the rows alone do not
  // fill the device.
  const int64_t page = page_bytes(heads, head_dim, group)(AKV_MODE_FP16);
  const int64_t most = std::max<int64_t>(1, page >> 13), least = std::max<int64_t>(1, page >> 15);
  const int parts = (int)std::max(least, std::min(most, 8 * 148 / rows));
  if (rows * parts >= (1ll << 31)) return AKV_ERR_UNSUPPORTED;
  const ForkParams p{table, layer_stride, seq_stride, batch, children, columns, uniform_tokens, parts, tokens, parents,
                     fresh, out_table, (uint8_t *)arena, arena_bytes, page_bytes(heads, head_dim, group), dev_status};
  const cudaError_t err =
      launch_dependent(fork_pages_kernel, (unsigned)(rows * parts), kCopyThreads, 0, (cudaStream_t)stream, p);
  return err == cudaSuccess ? AKV_OK : AKV_ERR_CUDA;
}

extern "C" int64_t akv_compact_workspace_bytes(int64_t entries, int64_t arena_bytes, int heads, int head_dim,
                                               int group) {
  if (check_page_geometry(heads, head_dim, group) != AKV_OK || entries < 0 || entries >= (1ll << 31) || arena_bytes < 0)
    return -1;
  return compact_sizes(entries, arena_bytes, page_bytes(heads, head_dim, group)(AKV_MODE_INT4)).bytes;
}

extern "C" int akv_compact_pages(const int64_t *table, int64_t entries, int64_t *out_table, const void *arena,
                                 int64_t arena_bytes, void *into, int64_t into_bytes, const int64_t *slots, int heads,
                                 int head_dim, int group, void *workspace, int64_t workspace_bytes,
                                 int32_t *dev_status, void *stream) {
  if (int st = check_page_geometry(heads, head_dim, group)) return st;
  if (!table || !out_table || !arena || !into || !slots || !workspace || entries < 0 || entries >= (1ll << 31))
    return AKV_ERR_INVALID;
  if (arena_bytes < 0 || into_bytes < 0 || ((uintptr_t)arena & 15) || ((uintptr_t)into & 15) || ((uintptr_t)workspace & 15))
    return AKV_ERR_INVALID;
  if (overlap(arena, arena_bytes, into, into_bytes) || overlap(table, 8 * entries, out_table, 8 * entries))
    return AKV_ERR_INVALID;  // pages and entries are read while others are written
  CompactParams p = {};
  p.bytes = page_bytes(heads, head_dim, group);
  for (int m = 1; m < 4; ++m) {
    p.base[m] = slots[2 * (m - 1)], p.capacity[m] = slots[2 * (m - 1) + 1];
    if (p.base[m] < 0 || p.base[m] % 16 || p.capacity[m] < 0 || p.base[m] > into_bytes ||
        p.capacity[m] > (into_bytes - p.base[m]) / p.bytes.of[m])
      return AKV_ERR_INVALID;
  }
  p.unit = p.bytes.of[AKV_MODE_INT4];
  const CompactSizes z = compact_sizes(entries, arena_bytes, p.unit);
  if (workspace_bytes < z.bytes) return AKV_ERR_INVALID;
  if (entries == 0) return AKV_OK;
  p.table = table, p.n = entries, p.out = out_table;
  p.arena = (const uint8_t *)arena, p.arena_bytes = arena_bytes, p.into = (uint8_t *)into;
  uint8_t *ws = (uint8_t *)workspace;
  p.place = (int64_t *)(ws + z.place_at), p.owner = (uint32_t *)(ws + z.owner_at);
  p.counts = (int32_t *)(ws + z.counts_at), p.blocks = (int32_t)z.blocks;
  p.status = dev_status;
  cudaStream_t s = (cudaStream_t)stream;
  cudaError_t err;
  if (entries <= kOnePlan && z.keys <= kOnePlanKeys) {
    if (plan_ready() != cudaSuccess) return AKV_ERR_CUDA;
    err = launch_dependent(compact_plan_kernel, 1, kRankThreads, (int)round16(4 * z.keys), s, p, (int)z.keys);
  } else {
    if (cudaMemsetAsync(p.owner, 0xff, 4 * z.keys, s) != cudaSuccess) return AKV_ERR_CUDA;
    compact_mark_kernel<<<(unsigned)std::min<int64_t>((entries + 255) / 256, 4 * 148), 256, 0, s>>>(p);
    err = launch_dependent(compact_count_kernel, (unsigned)z.blocks, kRankThreads, 0, s, p);
    if (err == cudaSuccess) err = launch_dependent(compact_rank_kernel, (unsigned)z.blocks, kRankThreads, 0, s, p);
  }
  if (err == cudaSuccess) err = launch_dependent(compact_move_kernel, (unsigned)entries, kCopyThreads, 0, s, p);
  return err == cudaSuccess ? AKV_OK : AKV_ERR_CUDA;
}
