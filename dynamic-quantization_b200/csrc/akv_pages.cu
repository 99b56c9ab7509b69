// Page operators: forking sequences that share pages, and compacting the pages a
// table refers to into another arena.
//
// Both move whole page records, byte for byte, and rewrite table entries on the
// device; neither looks at the values.  They are bound by HBM: a page is read
// once and written once (a compacted page that several entries share moves
// once), and the tables are 8 bytes a page beside 16 to 64 KB of payload.
#include <algorithm>

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

// Copy 16-byte units [lo, hi) of a page by one CTA; four loads of a thread are in
// flight before the first is stored.
__device__ __forceinline__ void copy_units(const uint8_t *src, uint8_t *dst, int64_t lo, int64_t hi) {
  const uint4 *s = reinterpret_cast<const uint4 *>(src);
  uint4 *d = reinterpret_cast<uint4 *>(dst);
  constexpr int U = 4;
  for (int64_t i = lo + threadIdx.x; i < hi; i += U * kCopyThreads) {
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
  const int part = blockIdx.x % p.parts;
  const int64_t row = blockIdx.x / p.parts;  // layer * children + child
  const int child = (int)(row % p.children);
  const int64_t layer = row / p.children;
  int64_t *out = p.out + row * p.columns;
  const int c0 = (int)((int64_t)p.columns * part / p.parts), c1 = (int)((int64_t)p.columns * (part + 1) / p.parts);
  const int64_t parent = p.parents[child];
  if (parent < 0 || parent >= p.batch) {  // no such sequence: an empty row
    if (threadIdx.x == 0 && part == 0) set_status(p.status, AKV_DEV_BAD_PARENT);
    for (int c = c0 + threadIdx.x; c < c1; c += kCopyThreads) out[c] = 0;
    return;
  }
  const int64_t *src_row = p.table + layer * p.layer_stride + parent * p.seq_stride;
  const int tokens = p.tokens ? p.tokens[parent] : p.uniform_tokens;
  const int64_t fresh = p.fresh ? p.fresh[row] : 0;
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
  copy_units(p.arena + desc_offset(old), p.arena + desc_offset(fresh), units * part / p.parts,
             units * (part + 1) / p.parts);
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
  for (int64_t e = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; e < p.n; e += (int64_t)gridDim.x * blockDim.x) {
    const int64_t d = p.table[e];
    if (movable(p, d)) atomicMin(p.owner + desc_offset(d) / p.unit, (uint32_t)e);
    else if (desc_mode(d) != AKV_MODE_SKIP) set_status(p.status, AKV_DEV_BAD_DESCRIPTOR);
  }
}

// The mode of entry e when it is the first to name its page, else 0.
__device__ __forceinline__ int owner_mode(const CompactParams &p, int64_t e, int64_t &d) {
  d = e < p.n ? p.table[e] : 0;
  return movable(p, d) && p.owner[desc_offset(d) / p.unit] == (uint32_t)e ? desc_mode(d) : 0;
}

__global__ void __launch_bounds__(kRankThreads) compact_count_kernel(const CompactParams p) {
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
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x < 4) before[threadIdx.x] = 0;
  __syncthreads();
  // owners of each precision in the blocks before this one
  int sum[4] = {0, 0, 0, 0};
  for (int b = threadIdx.x; b < (int)blockIdx.x; b += kRankThreads)
#pragma unroll
    for (int m = 1; m < 4; ++m) sum[m] += p.counts[4 * b + m];
#pragma unroll
  for (int m = 1; m < 4; ++m) {
    const int s = __reduce_add_sync(0xffffffffu, sum[m]);
    if (lane == 0 && s) atomicAdd(&before[m], s);  // integers: any order gives the same sum
  }
  int64_t d;
  const int mode = owner_mode(p, blockIdx.x * (int64_t)kRankThreads + threadIdx.x, d);
  int rank = 0;
#pragma unroll
  for (int m = 1; m < 4; ++m) {
    const uint32_t mask = __ballot_sync(0xffffffffu, mode == m);
    if (mode == m) rank = __popc(mask & ((1u << lane) - 1u));
    if (lane == 0) warps[m][warp] = __popc(mask);
  }
  __syncthreads();
  if (mode == 0) return;
  for (int w = 0; w < warp; ++w) rank += warps[mode][w];
  rank += before[mode];
  const int64_t key = desc_offset(d) / p.unit;
  if (rank >= p.capacity[mode]) {  // more pages than the target holds: the entries become skip entries
    set_status(p.status, AKV_DEV_BAD_DESCRIPTOR);
    p.place[key] = -1;
  } else {
    p.place[key] = p.base[mode] + rank * p.bytes(mode);
  }
}

// One CTA per table entry.
__global__ void __launch_bounds__(kCopyThreads) compact_move_kernel(const CompactParams p) {
  const int64_t e = blockIdx.x;
  const int64_t d = p.table[e];
  if (!movable(p, d)) {
    if (threadIdx.x == 0) p.out[e] = 0;
    return;
  }
  const int64_t key = desc_offset(d) / p.unit;
  const uint32_t owner = p.owner[key];
  const int64_t place = p.place[key];
  // An entry that overlaps another page without being it cannot move.
  const bool same = owner == (uint32_t)e || ((p.table[owner] ^ d) & ~(int64_t)0xfc) == 0;
  if (threadIdx.x == 0) {
    if (!same) set_status(p.status, AKV_DEV_BAD_DESCRIPTOR);
    p.out[e] = !same || place < 0 ? 0 : (place << 8) | (d & 255);
  }
  if (owner != (uint32_t)e || place < 0) return;
  copy_units(p.arena + desc_offset(d), p.into + place, 0, p.bytes(desc_mode(d)) / 16);
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
  const int parts = std::max(1, std::min(heads, 8));  // 8 KB of an 8-head FP16 page of head_dim 128 a CTA
  if (rows * parts >= (1ll << 31)) return AKV_ERR_UNSUPPORTED;
  const ForkParams p{table, layer_stride, seq_stride, batch, children, columns, uniform_tokens, parts, tokens, parents,
                     fresh, out_table, (uint8_t *)arena, arena_bytes, page_bytes(heads, head_dim, group), dev_status};
  fork_pages_kernel<<<(unsigned)(rows * parts), kCopyThreads, 0, (cudaStream_t)stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? AKV_OK : AKV_ERR_CUDA;
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
  if (cudaMemsetAsync(p.owner, 0xff, 4 * z.keys, s) != cudaSuccess) return AKV_ERR_CUDA;
  compact_mark_kernel<<<(unsigned)std::min<int64_t>((entries + 255) / 256, 4 * 148), 256, 0, s>>>(p);
  compact_count_kernel<<<(unsigned)z.blocks, kRankThreads, 0, s>>>(p);
  compact_rank_kernel<<<(unsigned)z.blocks, kRankThreads, 0, s>>>(p);
  compact_move_kernel<<<(unsigned)entries, kCopyThreads, 0, s>>>(p);
  return cudaGetLastError() == cudaSuccess ? AKV_OK : AKV_ERR_CUDA;
}
