// Chunk attention on the 5th-generation tensor cores (tcgen05, TMEM).
//
// The rows of a KV head are its (query token, query head) pairs, token-major; 128 of
// them form a row tile.  The pages that the rows can see are walked in tiles of
// 128 tokens (8 resident pages; evicted pages take no place in a tile):
//
//   S = Q K^T          tcgen05.mma, both operands in shared memory, S in TMEM
//   P = 2^(c S - m)    two threads per row: running max m and sum l in fp32
//   O = O + P V        tcgen05.mma, P (fp16) in TMEM over S's columns, O in TMEM
//
// P is rounded to fp16 because the MMA takes both operands in one 16-bit type and
// V's values are fp16.  m is the max less 7 when it moves, and moves only when a tile
// exceeds it by 15 (then O is rescaled), so P <= 2^15 and the row's largest is at least
// 2^7: a weight is off by 2^-11 of itself down to 2^-21 of the largest, by 2^-32 of the
// largest below that (with m at the max by 2^-25: small weights behind one large one
// would be lost, 2^-7 of it over 262144 tokens).
//
// A page would be dequantised once per pair of row tiles; chunk_unpack_kernel does it
// once per call instead, into operand tiles in the workspace, and the attention
// kernel copies whole tiles.  It runs one CTA per SM, each with two row tiles that
// share every K and V tile; the work (row tiles x tiles of tokens) is cut into equal
// contiguous ranges, one per CTA, whose partial (O, m, l) a merge kernel joins.
// Waits on mbarriers are bounded: a role whose wait runs out reports AKV_DEV_TIMEOUT and
// leaves.  The named barrier of a row's two warps is not; a leaving warp arrives there
// once, which is enough: its partner meets it at most once more before it waits on an
// mbarrier that this warp's missing arrival (p_full or q_full) keeps from completing,
// and leaves in turn.  A form in which a warp passes two exchanges without such a wait
// between them would need more.
//
// What bounds it, measured on a B200 with clocks read in the kernel: a tile of tokens
// takes about 3500 to 3700 clocks.  Of these a row tile's warps spend 150 on reading S,
// 250 on the max, 200 on agreeing on it, 1350 on the exponentials (1024 if the
// special-function unit did nothing else) and 150 on handing P over; its next S is
// there 1300 (head_dim 64) to 1700 clocks (128) later, behind O += P V, while the other
// row tile is at its exponentials.  A 2048-token chunk of 32768 (32 heads over 8, 128)
// takes 905 us by itself, 1.1 PFLOP/s, and 1066 to 1097 in long runs, where the power
// cap lowers the clock; 1000 tokens through a window of 2048
// (4 sequences, 24 heads over 8, 64) 150 us, of which the tiles take 115.
// Slower or no faster were: tiles of 64 tokens with S twice; S a tile ahead of P where
// head_dim 64 leaves TMEM for it (149 to 157 us against 154); a thread per row tile
// issuing the MMAs (1296 against 905); exponentials of some pairs by a polynomial
// (993 against 963 for one of 16); weights tried against the old max before a new one
// is looked for (171 against 154); one thread a row.
#include <math.h>
#include <stddef.h>

#include <algorithm>
#include <atomic>

#include "akv_chunk.cuh"

namespace akv {

// ------------------------------------------------------------ PTX: tcgen05
__device__ __forceinline__ void tmem_alloc(uint32_t smem_dst, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_dst), "r"(cols)
               : "memory");
}
__device__ __forceinline__ void tmem_release_permit() {
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t base, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// D[128 x N] (+)= A[128 x 16] B[16 x N], f16 operands, f32 accumulation.
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
// 32 consecutive columns of this thread's TMEM lane.
__device__ __forceinline__ void tc_ld32(uint32_t addr, float *v) {
  uint32_t *r = reinterpret_cast<uint32_t *>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tc_st16(uint32_t addr, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tc_st8(uint32_t addr, const uint32_t *r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(addr)
               : "memory");
}
__device__ __forceinline__ void tc_ld16(uint32_t addr, float *v) {
  uint32_t *r = reinterpret_cast<uint32_t *>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}
template <int N>
__device__ __forceinline__ void set_registers_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void set_registers_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// ----------------------------------------------------------- operand tiles
// Q, K and V tiles are 128 rows (query rows or tokens) of head_dim fp16 values,
// stored as head_dim / 64 panels of [128 rows][128 bytes], the 16-byte units of a
// row XORed with its index mod 8 (the 128-byte swizzle).  Read along head_dim (Q,
// K) such a tile is K-major, read along the rows (V) it is MN-major.
constexpr int kPanel = 128 * 128;  // bytes of one panel
__device__ __forceinline__ uint32_t panel_offset(int row, int unit) {  // 16-byte unit of a row
  return (uint32_t)((unit >> 3) * kPanel + row * 128 + (((unit & 7) ^ (row & 7)) << 4));
}
// Shared-memory descriptor, 128-byte swizzle: start address, leading and stride
// byte offsets in 16-byte units, version 1 (bit 46), swizzle mode 2 (bits 61-63).
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, uint32_t lead_bytes, uint32_t stride_bytes) {
  return (uint64_t)((addr & 0x3ffff) >> 4) | ((uint64_t)(lead_bytes >> 4) << 16) | ((uint64_t)(stride_bytes >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}
// Instruction descriptor: f32 accumulator, f16 operands, M = 128; bit 16: B is MN-major.
constexpr uint32_t mma_idesc(int n, bool b_mn_major) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24) | (b_mn_major ? 1u << 16 : 0u);
}

constexpr int kTilePages = 8;
constexpr int kTileTokens = kTilePages * kBlock;
constexpr int kMaxSlots = 8;  // operand tiles: K0 V0 K1 V1 ...
constexpr int kTmemCols = 512;
constexpr uint32_t kTmemS = 0, kTmemO = 256;  // S/P of stream x at 128 x, O at 256 + 128 x

// What the roles have to know about a tile of tokens.
struct __align__(16) TileMeta {
  int32_t col[kTilePages];
  uint32_t page[kTilePages];  // mode | valid tokens << 2; 0: no page
  uint32_t last;              // no tile of this segment follows
  uint32_t whole;             // every row of the CTA sees every token
  uint32_t none;              // not a tile: the segment has none
  uint32_t pad;
};
struct __align__(16) PageList {  // a tile's part that chunk_plan_kernel writes
  int32_t col[kTilePages];
  uint32_t page[kTilePages];
};

struct ChunkBars {
  uint64_t kv_full[kMaxSlots], kv_empty[kMaxSlots], q_full[2], s_full[2], p_full[2], o_full[2];
};
// Where a CTA's range of the work begins.
struct Place {
  int32_t b, kvh, m, pos;  // sequence, KV head, row block, tile within the unit
  int64_t left;            // tiles of the range
};
template <int D>
struct ChunkShared {
  // The loader is at most as many metas ahead as there are slots.
  static constexpr int kSlots = D == 128 ? 5 : 8, kMetas = D == 128 ? 8 : 16;
  ChunkBars bars;
  TileMeta meta[kMetas];
  Place place;
  uint32_t tmem;
  float shared_rows[2][2][128];  // [stream][half][row]: what the two threads of a row exchange
};
static_assert(sizeof(ChunkBars) % 16 == 0 && sizeof(TileMeta) % 16 == 0, "lists move 16 bytes at a time");

// What the tiles kernel reads from the workspace.
struct ChunkSpace {
  int32_t *counts;   // [batch]: resident pages that the call's rows may see
  int64_t *lists;    // [batch][tiles_max * 8]: their descriptors, in order
  PageList *metas;   // [batch][tiles_max]: their columns and valid tokens
  int4 *ranges;      // [batch][blocks]: sink tiles, first window tile, tiles
  int32_t *prefix;   // [batch][blocks + 1]: tiles of the row blocks before
  int4 *cuts;        // [CTAs]: what its range cut (see chunk_merge_kernel)
  uint8_t *tiles;    // [batch][kv head][tiles_max]: K tile, V tile
  int32_t tiles_max;
};
struct ChunkParams {
  ChunkArgs a;
  int32_t heads_per_kv, rows_kv, blocks, q_sign, vector_out, ctas;
  FastDiv fd_hpk;  // heads_per_kv
  float scale_log2;
  float *partials;  // rows of D + 4: O, m, l
  ChunkSpace w;
};

// What a block of rows sees: rows row0 .. row0 + n - 1 of a KV head.
struct ChunkView {
  int at_first, row0, n, at_lo, at_hi, window, sinks;
  int lead, first, total;  // virtual page columns: 0 .. lead - 1, then first ..; `total` of them
  __device__ __forceinline__ int column(int v) const { return v < lead ? v : first + (v - lead); }
  __device__ __forceinline__ bool whole_page(int col) const {
    const int p0 = kBlock * col, p1 = p0 + kBlock - 1;
    return p1 <= at_lo && (p0 > at_hi - window || p1 < sinks);
  }
  __device__ __forceinline__ bool any(int pos) const {
    return pos <= at_hi && (pos > at_lo - window || pos < sinks);
  }
};
__device__ __forceinline__ ChunkView chunk_view(const ChunkParams &p, int b, int row0, int nrows) {
  const ChunkArgs &a = p.a;
  ChunkView v;
  const int held = a.seq_blocks ? max(0, min(__ldg(a.seq_blocks + b), a.columns)) : a.columns;
  const int tokens = max(0, min(a.tokens ? __ldg(a.tokens + b) : a.uniform_tokens, kBlock * held));
  v.at_first = tokens - a.rows;
  v.row0 = row0, v.n = nrows;
  v.at_lo = v.at_first + fdiv(row0, p.fd_hpk);
  v.at_hi = v.at_first + fdiv(row0 + nrows - 1, p.fd_hpk);
  v.window = a.window, v.sinks = a.sinks, v.lead = a.lead;
  v.first = max(a.lead, max(v.at_lo - a.window + 1, 0) / kBlock);
  const int end = v.at_hi < 0 ? 0 : min(v.at_hi / kBlock + 1, held);  // columns up to the newest row's
  v.total = end <= v.lead ? end : v.lead + max(0, end - v.first);
  return v;
}

// ------------------------------------------------------------ work of a CTA
// Units are (sequence, KV head, row block), the row block fastest; a unit's cost is
// its tiles of tokens, at least 1 (its rows are written all the same).  The costs
// laid end to end are cut into equal ranges.
struct TileWork {  // as chunk_plan_kernel found it
  const ChunkParams &p;
  __device__ __forceinline__ int before(int b, int m) const {
    return __ldcg(p.w.prefix + (int64_t)b * (p.blocks + 1) + m);
  }
  __device__ __forceinline__ int cost(int b, int m) const { return before(b, m + 1) - before(b, m); }
  __device__ __forceinline__ int total(int b) const { return before(b, p.blocks); }
};
__device__ __forceinline__ int64_t warp_sum(int64_t v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}
// All of the work, by a whole warp.
__device__ __forceinline__ int64_t work_total(const TileWork &work) {
  const ChunkArgs &a = work.p.a;
  int64_t all = 0;
  for (int b = threadIdx.x & 31; b < a.batch; b += 32) all += (int64_t)work.total(b) * a.kv_heads;
  return warp_sum(all);
}
// A range of fewer tiles than this costs more to set up than it saves.
constexpr int kMinTiles = 2;
__device__ __forceinline__ int work_ctas(const ChunkParams &p, int64_t all) {
  return (int)max((int64_t)1, min((int64_t)p.ctas, (all + kMinTiles - 1) / kMinTiles));
}
__device__ __forceinline__ int64_t range_start(int64_t all, int ctas, int c) { return all * c / ctas; }
__device__ __forceinline__ Place find_place(const TileWork &work, int cta) {  // a whole warp
  const ChunkArgs &a = work.p.a;
  const int lane = threadIdx.x & 31;
  const int64_t all = work_total(work);
  const int ctas = work_ctas(work.p, all);
  Place at{0, 0, 0, 0, 0};
  if (cta >= ctas) return at;
  int64_t start = range_start(all, ctas, cta);
  at.left = range_start(all, ctas, cta + 1) - start;
  for (int b0 = 0;; b0 += 32) {  // the sequence
    const int64_t t = b0 + lane < a.batch ? (int64_t)work.total(b0 + lane) * a.kv_heads : 0;
    int64_t upto = t;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t o = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += o;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, start < upto);
    if (hit) {
      const int k = __ffs(hit) - 1;
      at.b = b0 + k;
      start -= __shfl_sync(0xffffffffu, upto - t, k);
      break;
    }
    start -= __shfl_sync(0xffffffffu, upto, 31);
  }
  const int per_head = work.total(at.b);
  at.kvh = (int)(start / per_head);
  const int rest = (int)(start - (int64_t)at.kvh * per_head);
  int m = 0;  // the row block: the last whose `before` is at most rest
  for (int m0 = 0; m0 < work.p.blocks; m0 += 32) {
    const bool upto = m0 + lane < work.p.blocks && work.before(at.b, m0 + lane) <= rest;
    const uint32_t hit = __ballot_sync(0xffffffffu, upto);
    if (hit) m = m0 + 31 - __clz(hit);
    if (hit != 0xffffffffu) break;
  }
  at.m = m, at.pos = rest - work.before(at.b, m);
  return at;
}
// The units of a CTA's range, one after the other.
struct Segments {
  const TileWork &work;
  Place at;
  int t0, t1, cost;
  __device__ __forceinline__ Segments(const TileWork &w, const Place &start) : work(w), at(start) { load(); }
  __device__ __forceinline__ void load() {
    if (at.left <= 0) return;
    cost = work.cost(at.b, at.m);
    t0 = at.pos;
    t1 = (int)min((int64_t)cost, t0 + at.left);
  }
  __device__ __forceinline__ bool valid() const { return at.left > 0; }
  __device__ __forceinline__ bool whole() const { return t0 == 0 && t1 == cost; }
  __device__ __forceinline__ int rows() const { return min(256, work.p.rows_kv - 256 * at.m); }
  __device__ __forceinline__ ChunkView view() const { return chunk_view(work.p, at.b, 256 * at.m, rows()); }
  __device__ __forceinline__ void next() {
    at.left -= t1 - t0;
    at.pos = 0;
    if (++at.m == work.p.blocks) {
      at.m = 0;
      if (++at.kvh == work.p.a.kv_heads) at.kvh = 0, ++at.b;
    }
    load();
  }
};

// ------------------------------------------------------------ loader of tiles
// Lists of the next tile are read while the slots of this one are awaited.
template <int D>
__device__ __forceinline__ void chunk_load_tiles(const TileWork &work, ChunkShared<D> &sh, uint8_t *tiles, int lane) {
  using Shared = ChunkShared<D>;
  constexpr int kOperand = 128 * D * 2, kSlots = Shared::kSlots;
  const ChunkParams &p = work.p;
  const ChunkSpace &w = p.w;
  int n = 0, metas = 0;
  bool ok = true;
  for (Segments seg(work, sh.place); seg.valid() && ok; seg.next()) {
    const int b = seg.at.b;
    const ChunkView view = seg.view();
    const int4 range = __ldcg(w.ranges + (int64_t)b * p.blocks + seg.at.m);
    const uint32_t *lists = reinterpret_cast<const uint32_t *>(w.metas + (int64_t)b * w.tiles_max);
    const uint8_t *src = w.tiles + ((int64_t)b * p.a.kv_heads + seg.at.kvh) * w.tiles_max * 2 * kOperand;
    if (range.z == 0) {  // no tile: the slot only carries the news
      const int slot = n % kSlots;
      ok = mbar_wait_bounded(smem_u32(&sh.bars.kv_empty[slot]), ((n / kSlots) & 1) ^ 1);
      if (!ok) break;
      if (lane == 0) {
        sh.meta[metas % Shared::kMetas].none = 1;
        mbar_arrive(smem_u32(&sh.bars.kv_full[slot]));
      }
      ++n, ++metas;
      continue;
    }
    auto tile_at = [&](int t) { return t < range.x ? t : range.y + (t - range.x); };
    uint32_t next = __ldcg(lists + 16ll * tile_at(seg.t0) + (lane & 15));
    for (int t = seg.t0; t < seg.t1 && ok; ++t) {
      const uint32_t word = next;
      if (t + 1 < seg.t1) next = __ldcg(lists + 16ll * tile_at(t + 1) + (lane & 15));
      const uint32_t page = __shfl_sync(0xffffffffu, word, 8 + (lane & 7));
      const int col = (int)__shfl_sync(0xffffffffu, word, lane & 7);
      const bool whole = __all_sync(0xffffffffu, (page & 3u) != 0 && (page >> 2) == kBlock && view.whole_page(col));
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const int slot = n % kSlots;
        ok = mbar_wait_bounded(smem_u32(&sh.bars.kv_empty[slot]), ((n / kSlots) & 1) ^ 1);
        if (!ok) break;
        ++n;
        if (kv == 0) {  // the slot being free, the meta's last user is past it too
          TileMeta &m = sh.meta[metas++ % Shared::kMetas];
          if (lane < 16) reinterpret_cast<uint32_t *>(&m)[lane] = word;
          if (lane == 0) m.last = t + 1 == seg.t1, m.whole = whole, m.none = 0;
          __syncwarp();
        }
        if (lane == 0) {
          const uint32_t bar = smem_u32(&sh.bars.kv_full[slot]);
          mbar_expect_tx(bar, kOperand);
          bulk_g2s(smem_u32(tiles + slot * kOperand), src + ((int64_t)tile_at(t) * 2 + kv) * kOperand, kOperand, bar);
        }
      }
    }
  }
  if (!ok) {
    if (lane == 0) set_status(p.a.status, AKV_DEV_TIMEOUT);
    for (int i = max(0, n - kSlots); i < n; ++i)  // let the copies in flight land (bounded)
      if (!mbar_wait_bounded(smem_u32(&sh.bars.kv_full[i % kSlots]), (i / kSlots) & 1)) break;
  }
}

// ---------------------------------------------------------------- MMA issue
// One thread issues every MMA; they execute in the order of issue, so a stream's S
// may overwrite the P that the MMA before it read.
template <int D>
struct MmaIssuer {
  static constexpr int kOperand = 128 * D * 2, kSlots = ChunkShared<D>::kSlots;
  static constexpr uint32_t kQk = mma_idesc(kTileTokens, false), kPv = mma_idesc(D, true);
  ChunkBars &bar;
  uint32_t q0, kv0, tmem;
  int n = 0;               // fills taken, in order K0 V0 K1 V1 ...
  int weights[2] = {0, 0}; // P tiles taken of each stream

  __device__ __forceinline__ MmaIssuer(ChunkBars &b, uint32_t tm, const uint8_t *q, const uint8_t *kv)
      : bar(b), q0(smem_u32(q)), kv0(smem_u32(kv)), tmem(tm) {}
  __device__ __forceinline__ bool wait(uint64_t &b, int phase) const { return mbar_wait_bounded(smem_u32(&b), phase & 1); }
  __device__ __forceinline__ bool filled(int fill) const {
    const bool ok = wait(bar.kv_full[fill % kSlots], fill / kSlots);
    tc_fence_after();
    return ok;
  }
  __device__ __forceinline__ void release(int fill) const { tc_commit(smem_u32(&bar.kv_empty[fill % kSlots])); }
  // Descriptors differ in the start address alone, in 16-byte units of its low word.
  __device__ __forceinline__ static uint64_t at(uint64_t desc, uint32_t bytes) { return desc + (bytes >> 4); }
  // S of stream x from Q tile `q` and K in `fill`.
  __device__ __forceinline__ void scores(int x, int q, int fill) const {
    const uint64_t qd = at(operand_desc(q0, 16, 1024), q * kOperand), kd = at(operand_desc(kv0, 16, 1024), fill % kSlots * kOperand);
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      const uint32_t off = (k >> 2) * kPanel + (k & 3) * 32;
      tc_mma_ss(tmem + kTmemS + 128 * x, at(qd, off), at(kd, off), kQk, k > 0);
    }
    tc_commit(smem_u32(&bar.s_full[x]));
  }
  // O of stream x; P's first 64 tokens lie at S's columns 0-31, the others at 64-95.
  __device__ __forceinline__ bool values(int x, int fill, bool accumulate) {
    const uint64_t vd = at(operand_desc(kv0, kPanel, 1024), fill % kSlots * kOperand);
    if (!wait(bar.p_full[x], weights[x]++)) return false;
    tc_fence_after();
#pragma unroll
    for (int k = 0; k < kTileTokens / 16; ++k)
      tc_mma_ts(tmem + kTmemO + 128 * x, tmem + kTmemS + 128 * x + 8 * k + (k >= 4 ? 32 : 0), at(vd, k * 2048), kPv,
                accumulate || k > 0);
    return true;
  }
  __device__ __forceinline__ void outputs(int streams) const {
    for (int x = 0; x < streams; ++x) tc_commit(smem_u32(&bar.o_full[x]));
  }
};

// Two row tiles (one where the block has no more rows) share every tile of tokens.
template <int D>
__device__ __forceinline__ void chunk_mma(const TileWork &work, ChunkShared<D> &sh, const uint8_t *q_tiles,
                                          const uint8_t *tiles) {
  using Shared = ChunkShared<D>;
  MmaIssuer<D> mma(sh.bars, sh.tmem, q_tiles, tiles);
  int metas = 0, loads[2] = {0, 0};
  bool ok = true;
  for (Segments seg(work, sh.place); seg.valid() && ok; seg.next()) {
    const int streams = seg.rows() > 128 ? 2 : 1;
    ok = mma.wait(mma.bar.q_full[0], loads[0]++) && (streams == 1 || mma.wait(mma.bar.q_full[1], loads[1]++)) &&
         mma.filled(mma.n);
    if (!ok) break;
    if (sh.meta[metas % Shared::kMetas].none) {  // nothing to attend: the softmax only has to know
      mbar_arrive(smem_u32(&mma.bar.kv_empty[mma.n % Shared::kSlots]));
      ++mma.n, ++metas;
      for (int x = 0; x < streams; ++x) mbar_arrive(smem_u32(&mma.bar.s_full[x]));
      mma.outputs(streams);
      continue;
    }
    int k_fill = mma.n++;
    mma.scores(0, 0, k_fill);
    if (streams == 2) mma.scores(1, 1, k_fill);
    mma.release(k_fill);
    for (bool first = true;; first = false) {
      const bool last = sh.meta[metas++ % Shared::kMetas].last;
      const int v_fill = mma.n++;
      if (!last) k_fill = mma.n++;
      ok = mma.filled(v_fill) && (last || mma.filled(k_fill));  // before the weights, not behind them
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (!ok || x >= streams) break;
        ok = mma.values(x, v_fill, !first);
        if (x == streams - 1) mma.release(v_fill);
        if (!ok || last) continue;
        mma.scores(x, x, k_fill);
        if (x == streams - 1) mma.release(k_fill);
      }
      if (!ok || last) break;
    }
    if (ok) mma.outputs(streams);
  }
  if (!ok) set_status(work.p.a.status, AKV_DEV_TIMEOUT);
}

// ----------------------------------------------------------------- softmax
// Load row tile x of Q into its operand tile, 16 rows a warp: two rows of head_dim
// 128 (four of 64) at a time, 16 bytes a lane, all of them in flight.  A negative softmax scale is
// folded into Q's sign (exact), so that the row max is the max of the products.
template <int D>
__device__ __forceinline__ void load_rows(const ChunkParams &p, const ChunkView &view, int b, int kvh, int x, int warp,
                                          int lane, uint8_t *tile) {
  constexpr int kUnits = D / 8, kPer = 32 / kUnits;
  const ChunkArgs &a = p.a;
  const uint32_t flip = p.q_sign < 0 ? 0x80008000u : 0u, keep = p.q_sign == 0 ? 0u : 0xffffffffu;
  const int unit = lane % kUnits;
#pragma unroll
  for (int i = 0; i < 16; i += kPer) {
    const int row = 16 * warp + i + lane / kUnits, r = 128 * x + row;
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (r < view.n) {
      const int rho = view.row0 + r, t = fdiv(rho, p.fd_hpk), h = kvh * p.heads_per_kv + (rho - t * p.heads_per_kv);
      v = __ldg(reinterpret_cast<const uint4 *>(a.q + (int64_t)b * a.q_bs + (int64_t)h * a.q_hs + (int64_t)t * a.q_ts) + unit);
      v.x = (v.x ^ flip) & keep, v.y = (v.y ^ flip) & keep, v.z = (v.z ^ flip) & keep, v.w = (v.w ^ flip) & keep;
    }
    *reinterpret_cast<uint4 *>(tile + panel_offset(row, unit)) = v;
  }
}

__device__ __forceinline__ uint32_t bits_below(int n) {  // the n lowest of 16 bits, n clamped
  return n <= 0 ? 0u : (n >= 16 ? 0xffffu : (1u << n) - 1u);
}

// The larger of three, NaN if one is NaN.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// 32 normalised outputs of a row.
__device__ __forceinline__ void store_out32(__half *out, const float (&o)[32], float inv, bool vector) {
  uint32_t w[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) w[k] = pack_f16x2(o[2 * k] * inv, o[2 * k + 1] * inv);
  if (vector) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      reinterpret_cast<uint4 *>(out)[k] = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
  } else {
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      out[2 * k] = __ushort_as_half((unsigned short)(w[k] & 0xffff));
      out[2 * k + 1] = __ushort_as_half((unsigned short)(w[k] >> 16));
    }
  }
}

// The softmax of row tile x over one CTA's segments: 8 warps, two threads a row, one
// for tokens 0-63 of a tile and one for 64-127 (a warp reaches the TMEM lanes of its
// number mod 4).  They agree on the row's max through shared memory.  One thread a row
// would leave a scheduler one warp of this row tile, which waits for its own
// instructions most of the time.
template <int D>
__device__ __forceinline__ void chunk_softmax(const TileWork &work, ChunkShared<D> &sh, uint8_t *q_tile, int x, int warp,
                                              int lane) {
  using Shared = ChunkShared<D>;
  constexpr int kRowStride = D + 4, kOut = D / 2;
  constexpr float kNegInf = -INFINITY, kSlack = 15.f, kLift = 7.f;
  const ChunkParams &p = work.p;
  const ChunkArgs &a = p.a;
  const int quarter = warp & 3, half = warp >> 2;
  const uint32_t base = sh.tmem + ((uint32_t)(32 * quarter) << 16);
  const uint32_t ts = base + kTmemS + 128 * x + 64 * half, to = base + kTmemO + 128 * x + kOut * half;
  const float c = p.scale_log2;
  const int tile_row = 32 * quarter + lane, r = 128 * x + tile_row;  // row of the tile, of the block
  const int pair = 1 + 4 * x + quarter;                              // the named barrier of the row's two warps
  float *mine = &sh.shared_rows[x][half][tile_row], *theirs = &sh.shared_rows[x][half ^ 1][tile_row];
  // The partner read the last value before the scores that this one is about came.
  auto exchange = [&](float v) {
    *mine = v;
    asm volatile("bar.sync %0, 64;" ::"r"(pair) : "memory");
    return *theirs;
  };
  int tiles = 0, metas = 0, segments = 0;
  int4 cut = make_int4(0, 0, 0, 0);
  bool ok = true;
  for (Segments seg(work, sh.place); seg.valid() && ok; seg.next()) {
    const ChunkView view = seg.view();
    const int b = seg.at.b, kvh = seg.at.kvh;
    if (seg.t0 > 0) cut.x = seg.t1 == seg.cost ? 2 : 1;
    else if (seg.t1 < seg.cost) cut.y = b, cut.z = kvh, cut.w = seg.at.m + 1;
    if (128 * x >= view.n) {  // the block has one row tile: its tiles are only counted
      const int4 range = __ldcg(p.w.ranges + (int64_t)b * p.blocks + seg.at.m);
      metas += range.z == 0 ? 1 : seg.t1 - seg.t0;
      continue;
    }
    load_rows<D>(p, view, b, kvh, x, warp, lane, q_tile);
    fence_proxy_async_smem();
    tc_fence_before();  // the reads of the last segment's O come before this segment's MMAs
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&sh.bars.q_full[x]));
    const bool active = r - lane < view.n;  // a warp without rows only keeps the barriers going
    const int at = view.at_first + fdiv(view.row0 + min(r, view.n - 1), p.fd_hpk);
    float m = kNegInf, l = 0.f;
    bool first = true;
    while (true) {
      ok = mbar_wait_bounded(smem_u32(&sh.bars.s_full[x]), tiles & 1);
      if (!ok) break;
      ++tiles;
      tc_fence_after();
      const TileMeta &meta = sh.meta[metas++ % Shared::kMetas];
      if (meta.none) break;
      const bool last = meta.last;
      if (active) {
        float s[64];
        tc_ld32(ts, s);
        tc_ld32(ts + 32, s + 32);
        tc_wait_ld();
        if (!meta.whole) {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int pos0 = kBlock * meta.col[4 * half + g], ntok = (int)(meta.page[4 * half + g] >> 2);
            const uint32_t bits = bits_below(min(ntok, at - pos0 + 1)) &
                                  (~bits_below(at - view.window - pos0 + 1) | bits_below(view.sinks - pos0));
#pragma unroll
            for (int i = 0; i < kBlock; ++i)
              if (!((bits >> i) & 1u)) s[kBlock * g + i] = kNegInf;
          }
        }
        float tops[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int i = 4; i < 60; i += 8)
#pragma unroll
          for (int k = 0; k < 4; ++k) tops[k] = max3(tops[k], s[i + k], s[i + 4 + k]);
        float top = max3(max3(tops[0], tops[1], s[60]), max3(tops[2], tops[3], s[61]), max3(s[62], s[63], s[63]));
        top = c * max3(top, exchange(top), top);
        // S of this tile came after O of the row tile's tile before it, so O is at rest
        // here.  A NaN score makes the row's max, and with it the row, NaN.
        if (__any_sync(0xffffffffu, !(top <= m + kSlack))) {
          const float low = top - kLift, n = max3(m, low, low);
          const float w = n == kNegInf ? 1.f : ex2(m - n);
          l *= w, m = n;
          if (!first) {
#pragma unroll 1
            for (int i = 0; i < kOut / 16; ++i) {
              float o[16];
              tc_ld16(to + 16 * i, o);
              tc_wait_ld();
#pragma unroll
              for (int k = 0; k < 16; ++k) o[k] *= w;
              tc_st16(to + 16 * i, reinterpret_cast<const uint32_t *>(o));
            }
          }
        }
        const float neg = m == kNegInf ? 0.f : -m;
        const uint64_t c2 = f2_pack(c, c), neg2 = f2_pack(neg, neg);
        uint64_t sum[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // 16 tokens at a time; P replaces the thread's own scores
          uint32_t pk[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const uint64_t x2 = f2_fma(f2_pack(s[16 * i + 2 * k], s[16 * i + 2 * k + 1]), c2, neg2);
            const uint64_t p2 = f2_pack(ex2(f2_lo(x2)), ex2(f2_hi(x2)));
            sum[k & 1] = f2_add(sum[k & 1], p2);
            pk[k] = pack_f16x2(f2_lo(p2), f2_hi(p2));
          }
          tc_st8(ts + 8 * i, pk);
        }
        const uint64_t both = f2_add(sum[0], sum[1]);
        l += f2_lo(both) + f2_hi(both);
        tc_wait_st();
        tc_fence_before();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sh.bars.p_full[x]));
      first = false;
      if (last) break;
    }
    ok = ok && mbar_wait_bounded(smem_u32(&sh.bars.o_full[x]), segments++ & 1);
    if (!ok) break;
    tc_fence_after();
    if (!active) continue;
    l += exchange(l);
    // The block's rows, or this range's share of them.
    const bool direct = seg.whole();
    float *part = p.partials + ((2ll * blockIdx.x + (seg.t0 > 0 ? 0 : 1)) * 256 + r) * kRowStride;
    const int rho = view.row0 + r, tok = fdiv(rho, p.fd_hpk), h = kvh * p.heads_per_kv + (rho - tok * p.heads_per_kv);
    __half *out = a.out + (int64_t)b * a.o_bs + (int64_t)h * a.o_hs + (int64_t)tok * a.o_ts + kOut * half;
    const float inv = l > 0.f ? 1.f / l : l;  // a row that saw nothing is 0, a NaN stays one
#pragma unroll
    for (int i = 0; i < kOut / 32; ++i) {
      float o[32];
      tc_ld32(to + 32 * i, o);
      tc_wait_ld();
      if (first) {  // O was never written
#pragma unroll
        for (int k = 0; k < 32; ++k) o[k] = 0.f;
      }
      if (r >= view.n) continue;
      if (direct) {
        store_out32(out + 32 * i, o, inv, p.vector_out);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          reinterpret_cast<float4 *>(part + kOut * half + 32 * i)[k] =
              make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
      }
    }
    if (!direct && half == 0 && r < view.n) *reinterpret_cast<float2 *>(part + D) = make_float2(m, l);
  }
  if (x == 0 && warp == 0 && lane == 0) p.w.cuts[blockIdx.x] = cut;
  if (!ok) {  // release a partner that may be waiting for this warp
    asm volatile("bar.arrive %0, 64;" ::"r"(pair) : "memory");
    if (lane == 0) set_status(a.status, AKV_DEV_TIMEOUT);
  }
}

// ---------------------------------------------------------- CTA set-up
template <int D>
__device__ __forceinline__ void chunk_begin(const TileWork &work, ChunkShared<D> &sh, int alloc_warp) {
  if (threadIdx.x == 0) {
    ChunkBars &bar = sh.bars;
    for (int i = 0; i < kMaxSlots; ++i) mbar_init(smem_u32(&bar.kv_full[i]), 1), mbar_init(smem_u32(&bar.kv_empty[i]), 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&bar.q_full[i]), 8);
      mbar_init(smem_u32(&bar.s_full[i]), 1);
      mbar_init(smem_u32(&bar.p_full[i]), 8);
      mbar_init(smem_u32(&bar.o_full[i]), 1);
    }
    fence_mbar_init();
  }
  if ((int)(threadIdx.x >> 5) == alloc_warp) {
    tmem_alloc(smem_u32(&sh.tmem), kTmemCols);
    tmem_release_permit();
  }
  grid_dependency_wait();
  allow_dependents_launch();
  if (threadIdx.x < 32) {
    const Place at = find_place(work, blockIdx.x);
    if (threadIdx.x == 0) sh.place = at;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
}
template <int D>
__device__ __forceinline__ void chunk_end(ChunkShared<D> &sh, int alloc_warp) {
  tc_fence_before();
  __syncthreads();
  if ((int)(threadIdx.x >> 5) == alloc_warp) {
    tc_fence_after();
    tmem_dealloc(sh.tmem, kTmemCols);
  }
}

// ------------------------------------------------------------ plan and unpack
// One CTA per sequence: the resident pages in column order, and the tiles that each
// block of 256 rows sees of them.
__global__ void __launch_bounds__(1024) chunk_plan_kernel(const __grid_constant__ ChunkParams p) {
  constexpr int kNear = 8192;  // columns kept for the searches below (2^17 tokens)
  __shared__ int warps[32], near[kNear];
  grid_dependency_wait();
  allow_dependents_launch();
  const ChunkArgs &a = p.a;
  const ChunkSpace &w = p.w;
  const int b = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const ChunkView view = chunk_view(p, b, 0, p.rows_kv);
  const int64_t *table = a.table + (int64_t)b * a.table_stride;
  int64_t *list = w.lists + (int64_t)b * w.tiles_max * kTilePages;
  PageList *metas = w.metas + (int64_t)b * w.tiles_max;
  int n = 0;
  const int threads = blockDim.x, all_warps = threads / 32;
  for (int base = 0; base < view.total; base += threads) {
    const int v = base + (int)threadIdx.x;
    int64_t d = 0;
    int col = 0;
    if (v < view.total) {
      col = view.column(v);
      d = __ldg(table + col);
    }
    const int mode = desc_mode(d);
    bool ok = mode != AKV_MODE_SKIP;
    if (ok && !page_in_arena(d, a.page_heads * record_bytes(a.head_dim, 1 << a.log2_group, mode), a.arena_bytes)) {
      set_status(a.status, AKV_DEV_BAD_DESCRIPTOR);
      ok = false;
    }
    const uint32_t mask = __ballot_sync(0xffffffffu, ok);
    if (lane == 0) warps[warp] = __popc(mask);
    __syncthreads();
    int before = 0, all = 0;
    for (int i = 0; i < all_warps; ++i) {
      if (i == warp) before = all;
      all += warps[i];
    }
    __syncthreads();
    if (ok) {
      const int rank = n + before + __popc(mask & ((1u << lane) - 1u));
      list[rank] = d;
      if (rank < kNear) near[rank] = col;
      metas[rank / kTilePages].col[rank % kTilePages] = col;
      metas[rank / kTilePages].page[rank % kTilePages] = (uint32_t)mode | ((uint32_t)desc_ntok(d) << 2);
    }
    n += all;
  }
  if (threadIdx.x < kTilePages && (int)threadIdx.x >= n % kTilePages && n % kTilePages) {
    const int rank = n / kTilePages * kTilePages + (int)threadIdx.x;
    list[rank] = 0;
    metas[rank / kTilePages].col[threadIdx.x] = 0, metas[rank / kTilePages].page[threadIdx.x] = 0;
  }
  if (threadIdx.x == 0) w.counts[b] = n;
  __syncthreads();
  // Pages of the list below a column.
  auto below = [&](int column) {
    int lo = 0, hi = n;
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if ((mid < kNear ? near[mid] : metas[mid / kTilePages].col[mid % kTilePages]) < column) lo = mid + 1;
      else hi = mid;
    }
    return lo;
  };
  int4 *ranges = w.ranges + (int64_t)b * p.blocks;
  int *prefix = w.prefix + (int64_t)b * (p.blocks + 1);
  int sum = 0;
  for (int base = 0; base < p.blocks; base += threads) {
    const int m = base + (int)threadIdx.x;
    int cost = 0;
    if (m < p.blocks) {
      const ChunkView v = chunk_view(p, b, 256 * m, min(256, p.rows_kv - 256 * m));
      const int end = v.at_hi < 0 ? 0 : (below(v.at_hi / kBlock + 1) + kTilePages - 1) / kTilePages;
      const int sinks = min(end, (below(v.lead) + kTilePages - 1) / kTilePages);
      const int first = max(sinks, min(end, below(v.first) / kTilePages));
      const int tiles = sinks + (end - first);
      ranges[m] = make_int4(sinks, first, tiles, 0);
      cost = max(1, tiles);
    }
    int upto = cost;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += o;
    }
    if (lane == 31) warps[warp] = upto;
    __syncthreads();
    int before = 0, all = 0;
    for (int i = 0; i < all_warps; ++i) {
      if (i == warp) before = all;
      all += warps[i];
    }
    __syncthreads();
    if (m < p.blocks) prefix[m] = sum + before + upto - cost;
    sum += all;
  }
  if (threadIdx.x == 0) prefix[p.blocks] = sum;
}

// One warp per (KV head, page, K or V) of a tile: 8 elements a lane and step, all
// loads of a page issued before the first is converted.
template <int D, bool SLAB>
__global__ void __launch_bounds__(256) chunk_unpack_kernel(const __grid_constant__ ChunkParams p) {
  constexpr int kOperand = 128 * D * 2, NC = D / 16, kUnits = D / 8, kRows = 32 / kUnits;
  grid_dependency_wait();
  allow_dependents_launch();
  const ChunkArgs &a = p.a;
  const ChunkSpace &w = p.w;
  const int tile = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & 31;
  if (tile * kTilePages >= __ldcg(w.counts + b)) return;
  const ChunkView view = chunk_view(p, b, 0, p.rows_kv);
  const int64_t *list = w.lists + ((int64_t)b * w.tiles_max + tile) * kTilePages;
  const int row0 = lane / kUnits, unit = lane % kUnits;
  for (int job = blockIdx.z * 8 + (threadIdx.x >> 5); job < 2 * kTilePages * a.kv_heads; job += 8 * gridDim.z) {
    const int kv = job & 1, i = (job >> 1) % kTilePages, kvh = (job >> 1) / kTilePages;
    const int64_t d = __ldcg(list + i);
    const int mode = desc_mode(d), ntok = desc_ntok(d);
    const int pos0 = kBlock * __ldcg(&w.metas[(int64_t)b * w.tiles_max + tile].col[i]);
    uint8_t *out = w.tiles + ((((int64_t)b * a.kv_heads + kvh) * w.tiles_max + tile) * 2 + kv) * kOperand;
    const uint8_t *rec = a.arena + desc_offset(d) + (a.kv_first + kvh) * record_bytes(D, 1 << a.log2_group, mode);
    const int64_t pb = payload_bytes(D, mode);
    const __half *sc = reinterpret_cast<const __half *>(rec + 2 * pb) + (kv ? (kBlock * D) >> a.log2_group : 0);
    uint4 raw[NC];
    float s[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) raw[c] = make_uint4(0u, 0u, 0u, 0u), s[c] = 0.f;
    if (mode != AKV_MODE_SKIP) {
      if (kv) slab_raw<D, NC, true>(mode, rec + pb, lane, raw);
      else slab_raw<D, NC, false>(mode, rec, lane, raw);
      if (mode != AKV_MODE_FP16) {
#pragma unroll
        for (int c = 0; c < NC; ++c) s[c] = __half2float(sc[SLAB ? 0 : (256 * c + 8 * lane) >> a.log2_group]);
      }
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int row = kRows * c + row0;
      uint4 v = mode == AKV_MODE_SKIP ? raw[c] : raw8_to_f16(mode, raw[c], s[c]);
      if (kv && (row >= ntok || !view.any(pos0 + row))) v = make_uint4(0u, 0u, 0u, 0u);
      *reinterpret_cast<uint4 *>(out + panel_offset(kBlock * i + row, unit)) = v;
    }
  }
}

// Warps 0-15 softmax, 16 loader, 17 MMA issue (18 and 19 make up the warpgroup).
// Registers a thread: at launch, and after the split.
constexpr int kTileThreads = 640;
constexpr int kTileRegs = 96, kSoftmaxRegs = 104, kIssueRegs = 64;
static_assert(4 * kSoftmaxRegs + kIssueRegs <= 5 * kTileRegs, "a warpgroup would wait for registers");

template <int D>
__global__ void __launch_bounds__(kTileThreads, 1) chunk_tiles_kernel(const __grid_constant__ ChunkParams p) {
  constexpr int kOperand = 128 * D * 2;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t *q_tiles = smem, *tiles = smem + 2 * kOperand;
  ChunkShared<D> &sh = *reinterpret_cast<ChunkShared<D> *>(tiles + ChunkShared<D>::kSlots * kOperand);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const TileWork work{p};
  chunk_begin(work, sh, 17);
  if (warp < 16) {
    set_registers_up<kSoftmaxRegs>();
    const int x = warp >> 3;
    chunk_softmax<D>(work, sh, q_tiles + x * kOperand, x, warp & 7, lane);
  } else {
    set_registers_down<kIssueRegs>();
    if (warp == 16) chunk_load_tiles<D>(work, sh, tiles, lane);
    if (warp == 17 && lane == 0) chunk_mma<D>(work, sh, q_tiles, tiles);
    __syncwarp();
  }
  chunk_end(sh, 17);
}

// ------------------------------------------------------------------- merge
// Join the partial (O, m, l) rows of the units that the ranges cut, a warp for four
// rows; a share that saw nothing (m = -inf) weighs 0.  CTA c's entry of `cuts`: y, z, w - 1
// the unit (sequence, KV head, row block) that its range begins and does not end (w 0:
// none); x: it goes on with a unit begun before (1), and ends it (2).  Block c joins
// the unit that range c begins.
constexpr int kMergeRows = 4;  // of a warp, whose loads are in flight together
template <int D>
__global__ void __launch_bounds__(256) chunk_merge_kernel(const __grid_constant__ ChunkParams p) {
  constexpr int VEC = D / 32, kRowStride = D + 4, R = kMergeRows, CB = 2;  // CB shares of each row at a time
  grid_dependency_wait();
  allow_dependents_launch();
  const ChunkArgs &a = p.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c0 = blockIdx.x;
  const int4 cut = __ldcg(p.w.cuts + c0);
  const int b = cut.y, kvh = cut.z, row0 = 256 * (cut.w - 1), r0 = blockIdx.y * 8 * R + warp;
  const int rows = min(256, p.rows_kv - row0);
  if (cut.w == 0 || r0 >= rows) return;
  int c1 = c0 + 1;
  while (c1 < p.ctas - 1 && __ldcg(&p.w.cuts[c1].x) == 1) ++c1;
  float m[R], l[R], acc[R][VEC];
#pragma unroll
  for (int k = 0; k < R; ++k) {
    m[k] = -INFINITY, l[k] = 0.f;
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[k][i] = 0.f;
  }
  for (int c = c0; c <= c1; c += CB) {
    float2 ml[R][CB];
    float o[R][CB][VEC];
#pragma unroll
    for (int k = 0; k < R; ++k)
#pragma unroll
      for (int j = 0; j < CB; ++j) {
        ml[k][j].x = -INFINITY;
        if (c + j <= c1 && r0 + 8 * k < rows) {
          const float *part = p.partials + ((2ll * (c + j) + (c + j == c0 ? 1 : 0)) * 256 + r0 + 8 * k) * kRowStride;
          ml[k][j] = __ldcg(reinterpret_cast<const float2 *>(part + D));
#pragma unroll
          for (int i = 0; i < VEC; i += 2) {
            const float2 v = __ldcg(reinterpret_cast<const float2 *>(part + VEC * lane + i));
            o[k][j][i] = v.x, o[k][j][i + 1] = v.y;
          }
        }
      }
#pragma unroll
    for (int k = 0; k < R; ++k)
#pragma unroll
      for (int j = 0; j < CB; ++j) {
        if (ml[k][j].x == -INFINITY) continue;
        const float top = fmaxf(m[k], ml[k][j].x), x = ex2(m[k] - top), y = ex2(ml[k][j].x - top);
        l[k] = l[k] * x + ml[k][j].y * y;
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[k][i] = acc[k][i] * x + o[k][j][i] * y;
        m[k] = isnan(ml[k][j].x) ? ml[k][j].x : top;
      }
  }
#pragma unroll
  for (int k = 0; k < R; ++k) {
    const int r = r0 + 8 * k;
    if (r >= rows) break;
    const int rho = row0 + r, tok = fdiv(rho, p.fd_hpk), h = kvh * p.heads_per_kv + (rho - tok * p.heads_per_kv);
    __half *out = a.out + (int64_t)b * a.o_bs + (int64_t)h * a.o_hs + (int64_t)tok * a.o_ts + VEC * lane;
    const float inv = l[k] > 0.f ? 1.f / l[k] : l[k];
#pragma unroll
    for (int i = 0; i < VEC; ++i) out[i] = __float2half_rn(acc[k][i] * inv);
  }
}

// ------------------------------------------------------------------- host
// SMs of the current device (one CTA each), 0 on error.
static int device_sms() {
  static std::atomic<int> cached[256];
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  if (dev < 256 && (sms = cached[dev].load(std::memory_order_relaxed)) > 0) return sms;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  if (dev < 256) cached[dev].store(sms, std::memory_order_relaxed);
  return sms;
}

// Raise a kernel's shared-memory limit, once per device, and check that it starts
// with the registers its warpgroups then share out: with fewer, setmaxnreg would wait
// for ever.  A compiler that gives it another number makes every large chunk fail here
// (AKV_ERR_CUDA) until kTileRegs and the split are set to its number.
template <typename Kernel>
static cudaError_t chunk_ready(Kernel kernel, int smem, int regs, std::atomic<bool> (&ready)[256]) {
  int dev = 0;
  if (cudaError_t err = cudaGetDevice(&dev)) return err;
  if (dev < 256 && ready[dev].load(std::memory_order_acquire)) return cudaSuccess;
  cudaFuncAttributes attr;
  if (cudaError_t err = cudaFuncGetAttributes(&attr, kernel)) return err;
  if (attr.numRegs != regs) return cudaErrorLaunchOutOfResources;
  if (cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) return err;
  if (dev < 256) ready[dev].store(true, std::memory_order_release);
  return cudaSuccess;
}

template <int D, bool SLAB>
static cudaError_t launch_tiles(const ChunkParams &p) {
  constexpr int smem = (2 + ChunkShared<D>::kSlots) * 128 * D * 2 + (int)sizeof(ChunkShared<D>);
  static_assert(smem <= 232448, "one CTA's shared memory");
  static std::atomic<bool> ready[256];
  if (cudaError_t err = chunk_ready(chunk_tiles_kernel<D>, smem, kTileRegs, ready)) return err;
  cudaStream_t s = p.a.stream;
  // few columns: fewer warps meet at the barriers of the one step they take
  const int planners = p.w.tiles_max * kTilePages <= 512 ? 256 : 1024;
  if (cudaError_t err = launch_dependent(chunk_plan_kernel, p.a.batch, planners, 0, s, p)) return err;
  // 16 KV-head-pages a warp where there are tiles enough for the device, down to one
  const int64_t tiles = (int64_t)p.w.tiles_max * p.a.batch;
  const int jobs = std::min(2 * kTilePages * p.a.kv_heads / 8, 65535);  // of a tile, per warp of a CTA
  const int parts = (int)std::max<int64_t>(1, std::min<int64_t>(jobs, std::max<int64_t>(jobs / 16, 8 * p.ctas / std::max<int64_t>(tiles, 1))));
  if (p.w.tiles_max > 0)
    if (cudaError_t err =
            launch_dependent(chunk_unpack_kernel<D, SLAB>, dim3(p.w.tiles_max, p.a.batch, parts), 256, 0, s, p))
      return err;
  if (cudaError_t err = launch_dependent(chunk_tiles_kernel<D>, p.ctas, kTileThreads, smem, s, p)) return err;
  return launch_dependent(chunk_merge_kernel<D>, dim3(p.ctas, std::min(256, p.rows_kv + 8 * kMergeRows - 1) / (8 * kMergeRows)), 256, 0, s, p);
}

static int64_t align256(int64_t n) { return (n + 255) & ~(int64_t)255; }
// The workspace of a call, and where its parts lie (p: nullable).
static int64_t chunk_layout(const ChunkArgs &a, int sms, uint8_t *base, ChunkParams *p) {
  const int hpk = a.q_heads / a.kv_heads;
  const int64_t rows_kv = (int64_t)a.rows * hpk, pairs = (int64_t)a.batch * a.kv_heads;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += align256(bytes);
    return base + here;
  };
  const int64_t blocks = (rows_kv + 255) / 256;
  int64_t columns = a.columns;  // that some row may see
  if (a.window < (1 << 30))
    columns = std::min<int64_t>(columns, a.lead + ((int64_t)a.window + a.rows + 2 * kBlock - 3) / kBlock);
  const int64_t tiles = (columns + kTilePages - 1) / kTilePages;
  ChunkSpace w;
  w.counts = (int32_t *)take(4ll * a.batch);
  w.lists = (int64_t *)take(8ll * kTilePages * tiles * a.batch);
  w.metas = (PageList *)take((int64_t)sizeof(PageList) * tiles * a.batch);
  w.ranges = (int4 *)take(16ll * blocks * a.batch);
  w.prefix = (int32_t *)take(4ll * (blocks + 1) * a.batch);
  w.cuts = (int4 *)take(16ll * sms);
  float *parts = (float *)take(2ll * sms * 256 * (a.head_dim + 4) * 4);
  w.tiles = take(tiles * pairs * 2 * 128 * a.head_dim * 2);
  w.tiles_max = (int32_t)tiles;
  if (p) p->w = w, p->partials = parts, p->blocks = (int32_t)blocks;
  return at;
}

// Operand tiles are four times the bytes of INT4 pages and more, so a large call goes
// in slices that share a workspace of at most about this size (unless one KV head of one
// sequence needs more): slices of whole sequences, or of a sequence's KV heads where
// even one sequence is too large.
constexpr int64_t kSpaceBytes = 2ll << 30;
static ChunkArgs sized(ChunkArgs a, int batch, int kv_heads) {
  a.q_heads = a.q_heads / a.kv_heads * kv_heads, a.kv_heads = kv_heads, a.batch = batch;
  return a;
}
static ChunkArgs slice_of(const ChunkArgs &all, int first, int count, int kv_first, int kv_heads) {
  ChunkArgs a = sized(all, count, kv_heads);
  const int64_t head = (int64_t)kv_first * (all.q_heads / all.kv_heads);
  a.table += first * a.table_stride;
  if (a.seq_blocks) a.seq_blocks += first;
  if (a.tokens) a.tokens += first;
  a.q += first * a.q_bs + head * a.q_hs, a.out += first * a.o_bs + head * a.o_hs;
  a.kv_first = kv_first, a.page_heads = all.kv_heads;
  return a;
}
struct Slice {
  int batch, kv_heads;
};
static Slice slice_size(const ChunkArgs &a, int sms) {
  auto bytes = [&](int batch, int kv_heads) { return chunk_layout(sized(a, batch, kv_heads), sms, nullptr, nullptr); };
  auto fit = [](int64_t one, int64_t two) {  // how many, the first of them `one` with what they share
    return 1 + std::max<int64_t>(0, kSpaceBytes - one) / std::max<int64_t>(1, two - one);
  };
  if (bytes(1, a.kv_heads) > kSpaceBytes && a.kv_heads > 1)
    return Slice{1, (int)std::min<int64_t>(a.kv_heads, fit(bytes(1, 1), bytes(1, 2)))};
  const int64_t sequences = fit(bytes(1, a.kv_heads), bytes(2, a.kv_heads));
  return Slice{(int)std::min<int64_t>({sequences, a.batch, 65535}), a.kv_heads};  // a grid's second dimension
}

// Tiles of a KV head's row blocks are counted in 32 bits.
static bool countable(const ChunkArgs &a) {
  const int64_t blocks = ((int64_t)a.rows * (a.q_heads / a.kv_heads) + 255) / 256;
  return blocks * (a.columns / kTilePages + 2) < (1ll << 31);
}

int64_t chunk_tiles_bytes(const ChunkArgs &a) {
  const int sms = device_sms();
  if (sms <= 0 || !countable(a)) return -1;
  const Slice slice = slice_size(a, sms);
  return chunk_layout(sized(a, slice.batch, slice.kv_heads), sms, nullptr, nullptr);
}

int chunk_tiles_launch(const ChunkArgs &all, void *workspace, int64_t workspace_bytes) {
  const int sms = device_sms();
  if (sms <= 0) return AKV_ERR_CUDA;
  if (!countable(all)) return AKV_ERR_UNSUPPORTED;
  if (workspace_bytes < chunk_tiles_bytes(all)) return AKV_ERR_INVALID;
  const Slice slice = slice_size(all, sms);
  auto launch = [&](const ChunkArgs &a) {
    ChunkParams p = {};
    p.a = a;
    p.heads_per_kv = a.q_heads / a.kv_heads;
    p.rows_kv = a.rows * p.heads_per_kv;
    p.fd_hpk = fast_div((uint32_t)p.heads_per_kv);
    p.ctas = sms;
    // scale 0 weighs every token alike: Q counts as zero
    p.q_sign = a.scale > 0.f ? 1 : (a.scale < 0.f ? -1 : 0);
    p.scale_log2 = p.q_sign == 0 ? 1.f : fabsf(a.scale) * 1.4426950408889634f;
    p.vector_out = ((uintptr_t)a.out & 15) == 0 && a.o_bs % 8 == 0 && a.o_hs % 8 == 0 && a.o_ts % 8 == 0;
    chunk_layout(a, sms, (uint8_t *)workspace, &p);
    const bool slab = (1 << a.log2_group) == 16 * a.head_dim;
    return a.head_dim == 64 ? (slab ? launch_tiles<64, true>(p) : launch_tiles<64, false>(p))
                            : (slab ? launch_tiles<128, true>(p) : launch_tiles<128, false>(p));
  };
  for (int first = 0; first < all.batch; first += slice.batch)
    for (int head = 0; head < all.kv_heads; head += slice.kv_heads)
      if (launch(slice_of(all, first, std::min(slice.batch, all.batch - first), head,
                          std::min(slice.kv_heads, all.kv_heads - head))) != cudaSuccess)
        return AKV_ERR_CUDA;
  return AKV_OK;
}

}  // namespace akv
