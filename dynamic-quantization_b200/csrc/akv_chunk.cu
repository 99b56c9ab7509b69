// Chunk attention on the 5th-generation tensor cores (tcgen05, TMEM).
//
// The rows of a KV head are its (query token, query head) pairs, token-major.  A
// CTA holds one or two tiles of 128 rows and walks the pages they can see in
// tiles of 128 tokens (8 resident pages; evicted pages take no place in a tile):
//
//   S = Q K^T          tcgen05.mma, both operands in shared memory, S in TMEM
//   P = 2^(c S - m)    one thread per row: running max m and sum l in fp32
//   O = O + P V        tcgen05.mma, P (fp16) in TMEM over S's columns, O in TMEM
//
// P is rounded to fp16 because the MMA takes both operands in one 16-bit type and
// V's values are fp16; m moves only when a tile exceeds it by 2^8 (then O is
// rescaled), so P <= 2^8 and its rounding is relative, 2^-11 a term.
//
// Roles (warps): 0-3 and 4-7 softmax of the two row tiles; 8-11 dequantise pages
// into operand tiles; 12 loads records (bulk copies into a byte ring); 13 issues
// the MMAs.  K and V are dequantised to the values the reference attends over,
// fp16(int * float(scale)), once per CTA and tile.  Waits are bounded: a role whose
// wait runs out reports AKV_DEV_TIMEOUT and leaves its loop.
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
__device__ __forceinline__ void tc_st32(uint32_t addr, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,"
      "%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
      "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
      "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(addr)
      : "memory");
}
// Shared memory by 32-bit address.
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void lds64(uint32_t a, uint32_t (&v)[2]) {
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(a) : "memory");
}
__device__ __forceinline__ void lds128(uint32_t a, uint32_t (&v)[4]) {
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
               : "r"(a)
               : "memory");
}
__device__ __forceinline__ void sts128(uint32_t a, const uint32_t (&v)[4]) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
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
constexpr int kMaxSlots = 8;    // operand tiles: K0 V0 K1 V1 ...
constexpr int kItems = 8;       // half tiles of raw records in flight
constexpr int kMetas = 8;       // the loader runs at most 5 tiles ahead of the softmax
constexpr int kRawRing = 32768;
constexpr int kTmemCols = 512;
constexpr uint32_t kTmemS = 0, kTmemO = 256;  // S/P of row tile x at 128 x, O at 256 + 128 x

struct __align__(16) TileMeta {
  int32_t col[kTilePages];
  uint32_t page[kTilePages];  // mode | valid tokens << 2; 0: no page
  int64_t src[kTilePages];    // byte offset of the KV head's record (page kernel)
  uint32_t last, whole, none;  // no tile follows; every row of the CTA sees every token; there is no tile at all
};

struct ChunkBars {
  uint64_t raw_full[kItems], raw_empty[kItems], kv_full[kMaxSlots], kv_empty[kMaxSlots], q_full, s_full[2], p_full[2],
      o_full[2];
};

struct ChunkShared {
  ChunkBars bars;
  TileMeta meta[kMetas];
  uint32_t raw_at[kItems][4];  // ring offset of each page of an item
  uint32_t tmem;
};


static_assert(offsetof(ChunkShared, meta) % 16 == 0 && sizeof(TileMeta) % 16 == 0, "lists move 16 bytes at a time");

struct ChunkParams {
  ChunkArgs a;
  int32_t heads_per_kv, rows_kv, q_sign, vector_out;
  float scale_log2;
};

// What a CTA's rows see: rows row0 .. row0 + n - 1 of a KV head.
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
  const int tokens = min(a.tokens ? __ldg(a.tokens + b) : a.uniform_tokens, kBlock * held);
  v.at_first = tokens - a.rows;
  v.row0 = row0, v.n = nrows;
  v.at_lo = v.at_first + row0 / p.heads_per_kv;
  v.at_hi = v.at_first + (row0 + nrows - 1) / p.heads_per_kv;
  v.window = a.window, v.sinks = a.sinks, v.lead = a.lead;
  v.first = max(a.lead, max(v.at_lo - a.window + 1, 0) / kBlock);
  const int end = v.at_hi < 0 ? 0 : min(v.at_hi / kBlock + 1, held);  // columns up to the newest row's
  v.total = end <= v.lead ? end : v.lead + max(0, end - v.first);
  return v;
}

// ------------------------------------------------------------------ loader
// Descriptors are read 32 columns at a time, one per lane, a window ahead; the
// resident pages of a window fill tiles in order.
template <int D>
__device__ __forceinline__ void chunk_load(const ChunkParams &p, ChunkShared &sh, uint8_t *ring, const ChunkView &view,
                                           int b, int kvh, int lane) {
  const ChunkArgs &a = p.a;
  const uint32_t scale_bytes = 2u * (uint32_t)((kBlock * D) >> a.log2_group);  // K's (or V's) scales of a record
  const int64_t *table = a.table + (int64_t)b * a.table_stride;
  auto fetch = [&](int w0, int64_t &raw, int &col) {
    const int v = w0 + lane;
    raw = 0, col = 0;
    if (v < view.total) {
      col = view.column(v);
      raw = __ldg(table + col);
    }
  };
  int64_t src = 0;
  uint32_t page = 0, mask = 0;
  int col = 0;
  auto prepare = [&](int64_t raw, int c) {
    const int mode = desc_mode(raw);
    bool ok = mode != AKV_MODE_SKIP;
    int64_t rb = 2 * payload_bytes(D, mode) + (mode == AKV_MODE_FP16 ? 0 : 2 * (int64_t)scale_bytes);
    rb = (rb + 15) & ~(int64_t)15;
    if (ok && !page_in_arena(raw, rb * a.kv_heads, a.arena_bytes)) {
      set_status(a.status, AKV_DEV_BAD_DESCRIPTOR);
      ok = false;
    }
    src = desc_offset(raw) + kvh * rb;
    page = (uint32_t)mode | ((uint32_t)desc_ntok(raw) << 2);
    col = c;
    mask = __ballot_sync(0xffffffffu, ok);
  };
  int win0 = 0, next_col;
  int64_t next_raw;
  {
    int64_t raw;
    int c;
    fetch(0, raw, c);
    fetch(32, next_raw, next_col);
    prepare(raw, c);
  }
  auto advance = [&]() {
    win0 += 32;
    const int64_t raw = next_raw;
    const int c = next_col;
    fetch(win0 + 32, next_raw, next_col);
    prepare(raw, c);
  };

  uint32_t head = 0, head_p = 0, tail = 0;  // byte ring: virtual positions and the physical write position
  uint32_t starts = 0;                      // lane i: virtual start of the item in slot i
  int issued = 0, freed = 0;
  bool dead = false;
  for (int tile = 0; !dead; ++tile) {
    TileMeta &m = sh.meta[tile % kMetas];
    int have = 0;
    while (have < kTilePages) {
      if (mask == 0) {
        if (win0 + 32 >= view.total) break;
        advance();
        continue;
      }
      const int rank = have + __popc(mask & ((1u << lane) - 1u));
      const bool take = ((mask >> lane) & 1u) && rank < kTilePages;
      if (take) m.col[rank] = col, m.page[rank] = page, m.src[rank] = src;
      const uint32_t taken = __ballot_sync(0xffffffffu, take);
      mask &= ~taken;
      have += __popc(taken);
    }
    if (lane >= have && lane < kTilePages) m.col[lane] = 0, m.page[lane] = 0, m.src[lane] = 0;
    while (mask == 0 && win0 + 32 < view.total) advance();
    const bool last = mask == 0;
    __syncwarp();
    bool whole = true;
    if (lane < kTilePages) whole = (m.page[lane] >> 2) == kBlock && view.whole_page(m.col[lane]);
    whole = __all_sync(0xffffffffu, whole);
    if (lane == 0) m.last = last, m.whole = whole, m.none = 0;
    __syncwarp();
    for (int part = 0; part < 4; ++part) {  // K of pages 0-3, of 4-7, then V
      const int kv = part >> 1, i = 4 * (part & 1) + (lane & 3);
      const int mode = lane < 4 ? (int)(m.page[i] & 3) : 0;
      const uint32_t pay = mode ? (uint32_t)payload_bytes(D, mode) : 0u;
      // K and V scales lie one after the other; both of a slab record share one 16-byte unit
      const uint32_t sc = mode == 0 || mode == AKV_MODE_FP16 ? 0u : max(16u, scale_bytes);
      uint32_t off = pay + sc;
#pragma unroll
      for (int d = 1; d < 4; d <<= 1) {
        const uint32_t o = __shfl_up_sync(0xffffffffu, off, d);
        if (lane >= d) off += o;
      }
      const uint32_t total = __shfl_sync(0xffffffffu, off, 3);
      off -= pay + sc;
      const int slot = issued % kItems;
      uint32_t start, start_p;
      while (true) {
        start = head, start_p = head_p;
        if (issued == freed && start_p != 0) {  // empty ring: restart at a lap boundary
          start += kRawRing - start_p;
          start_p = 0;
          tail = start;
        } else if (start_p + total > (uint32_t)kRawRing) {
          start += kRawRing - start_p;
          start_p = 0;
        }
        if (issued - freed < kItems && start + total - tail <= (uint32_t)kRawRing) break;
        if (!mbar_wait_bounded(smem_u32(&sh.bars.raw_empty[freed % kItems]), (freed / kItems) & 1)) {
          dead = true;
          break;
        }
        ++freed;
        tail = freed == issued ? head : __shfl_sync(0xffffffffu, starts, freed % kItems);
      }
      if (dead) break;
      if (lane == slot) starts = start;
      if (lane < 4) sh.raw_at[slot][lane] = start_p + off;
      __syncwarp();
      const uint32_t bar = smem_u32(&sh.bars.raw_full[slot]);
      if (lane == 0) mbar_expect_tx(bar, total);
      __syncwarp();
      if (mode) {
        const uint8_t *rec = a.arena + m.src[i];
        const uint32_t dst = smem_u32(ring + start_p + off);
        bulk_g2s(dst, rec + kv * pay, pay, bar);
        if (sc) bulk_g2s(dst + pay, rec + 2 * pay + (kv && scale_bytes >= 16 ? scale_bytes : 0), sc, bar);
      }
      head = start + total, head_p = start_p + total;
      ++issued;
    }
    if (last) break;
  }
  if (dead) {
    if (lane == 0) set_status(a.status, AKV_DEV_TIMEOUT);
    for (int i = freed; i < issued; ++i)  // let the copies in flight land (bounded)
      if (!mbar_wait_bounded(smem_u32(&sh.bars.raw_full[i % kItems]), (i / kItems) & 1)) break;
  }
}

// ------------------------------------------------------------ dequantisation
// One page's K or V payload (at raw, scales behind it) into tokens token0 .. + 15
// of an operand tile, by one warp: 8 elements (one 16-byte unit of the tile) a
// lane and step.  `seen(row)`: V rows that no row sees become zero, so that a
// weight of 0 never meets what their memory holds.
template <int D, int MODE, bool VPAY, bool SLAB, typename Seen>
__device__ __forceinline__ void dequant_page(const uint8_t *raw, const __half *scales, int log2_group, uint8_t *tile,
                                             int token0, int lane, bool check, Seen seen) {
  constexpr int NC = D / 16;
  constexpr int BYTES = MODE == AKV_MODE_FP16 ? 16 : (MODE == AKV_MODE_INT8 ? 8 : 4);  // of 8 elements
  // Chunk c holds elements 256 c + 8 lane + [0, 8): row kRows c + row0, unit `unit`.
  // Both swizzles are XORs of bits that c alone (or c and the lane apart) sets, so
  // an address is a lane constant, one XOR with a constant and an immediate.
  constexpr int kUnits = D / 8, kRows = 32 / kUnits;
  const int row0 = lane / kUnits, unit = lane % kUnits;
  const uint32_t dst0 = smem_u32(tile) + (uint32_t)((unit >> 3) * kPanel + (token0 + row0) * 128 + (((unit & 7) ^ row0) << 4));
  const uint32_t src0 = smem_u32(raw);
  const __half *sc = SLAB ? scales : scales + ((8 * lane) >> log2_group);
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const uint32_t src = src0 + (uint32_t)((BYTES * lane) ^ (VPAY ? v_chunk_xor<D>(MODE, c, lane) : 0)) + 32 * BYTES * c;
    uint32_t h[4];
    if constexpr (MODE == AKV_MODE_FP16) {
      lds128(src, h);
    } else {
      const uint32_t s1 = __half_as_ushort(sc[SLAB ? 0 : (256 * c) >> log2_group]), s = s1 | (s1 << 16);
      if constexpr (MODE == AKV_MODE_INT8) {
        uint32_t w[2];
        lds64(src, w);
        h[0] = hmul2(int8_to_f16x2(prmt(w[0], 0, 0x1100)), s), h[1] = hmul2(int8_to_f16x2(prmt(w[0], 0, 0x3322)), s);
        h[2] = hmul2(int8_to_f16x2(prmt(w[1], 0, 0x1100)), s), h[3] = hmul2(int8_to_f16x2(prmt(w[1], 0, 0x3322)), s);
      } else {
        const uint32_t w = lds32(src);
        const uint32_t e04 = hmul2(int4_lo_to_f16x2(w), s), e15 = hmul2(int4_hi_to_f16x2(w), s);
        const uint32_t e26 = hmul2(int4_lo_to_f16x2(w >> 8), s), e37 = hmul2(int4_hi_to_f16x2(w >> 8), s);
        h[0] = prmt(e04, e15, 0x5410), h[1] = prmt(e26, e37, 0x5410);
        h[2] = prmt(e04, e15, 0x7632), h[3] = prmt(e26, e37, 0x7632);
      }
    }
    if (VPAY && check && !seen(kRows * c + row0)) h[0] = h[1] = h[2] = h[3] = 0u;
    sts128((dst0 ^ (((kRows * c) & 7) << 4)) + kRows * 128 * c, h);
  }
}

template <int D, bool SLAB>
__device__ __forceinline__ void chunk_dequant(const ChunkParams &p, ChunkShared &sh, const uint8_t *ring, uint8_t *tiles,
                                              const ChunkView &view, int warp, int lane) {
  constexpr int kOperand = 128 * D * 2;
  constexpr int kSlots = 4;
  const int lg = p.a.log2_group;
  bool dead = false;
  for (int n = 0; !dead; ++n) {
    const int slot = n % kSlots, kv = n & 1;
    const TileMeta &m = sh.meta[(n >> 1) % kMetas];
    uint8_t *tile = tiles + slot * kOperand;
    if (!mbar_wait_bounded(smem_u32(&sh.bars.kv_empty[slot]), ((n / kSlots) & 1) ^ 1)) {
      dead = true;
      break;
    }
    for (int half = 0; half < 2; ++half) {
      const int item = 2 * n + half, rs = item % kItems, i = 4 * half + warp;
      if (!mbar_wait_bounded(smem_u32(&sh.bars.raw_full[rs]), (item / kItems) & 1)) {
        dead = true;
        break;
      }
      const uint32_t page = m.page[i];
      const int mode = (int)(page & 3), ntok = (int)(page >> 2), pos0 = kBlock * m.col[i], token0 = kBlock * i;
      const bool check = !m.whole;
      const uint8_t *raw = ring + sh.raw_at[rs][warp];
      auto seen = [&](int row) { return row < ntok && view.any(pos0 + row); };
      // a slab record's two scales share the unit behind the payload
      auto scales = [&](int md) {
        return reinterpret_cast<const __half *>(raw + payload_bytes(D, md)) + (SLAB ? kv : 0);
      };
      if (mode == AKV_MODE_INT4) {
        if (kv) dequant_page<D, AKV_MODE_INT4, true, SLAB>(raw, scales(mode), lg, tile, token0, lane, check, seen);
        else dequant_page<D, AKV_MODE_INT4, false, SLAB>(raw, scales(mode), lg, tile, token0, lane, check, seen);
      } else if (mode == AKV_MODE_INT8) {
        if (kv) dequant_page<D, AKV_MODE_INT8, true, SLAB>(raw, scales(mode), lg, tile, token0, lane, check, seen);
        else dequant_page<D, AKV_MODE_INT8, false, SLAB>(raw, scales(mode), lg, tile, token0, lane, check, seen);
      } else if (mode == AKV_MODE_FP16) {
        if (kv) dequant_page<D, AKV_MODE_FP16, true, SLAB>(raw, nullptr, lg, tile, token0, lane, check, seen);
        else dequant_page<D, AKV_MODE_FP16, false, SLAB>(raw, nullptr, lg, tile, token0, lane, check, seen);
      } else if (kv) {  // no page: its tokens are masked, and V is finite
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          const int e = 256 * c + 8 * lane;
          *reinterpret_cast<uint4 *>(tile + panel_offset(token0 + e / D, (e % D) / 8)) = make_uint4(0u, 0u, 0u, 0u);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sh.bars.raw_empty[rs]));
    }
    if (dead) break;
    const bool last = m.last;
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&sh.bars.kv_full[slot]));
    if (kv && last) break;
  }
  if (dead && lane == 0) set_status(p.a.status, AKV_DEV_TIMEOUT);
}

// ---------------------------------------------------------------- MMA issue
// One thread issues every MMA; they execute in the order of issue, so a row
// tile's S may overwrite the P that the MMA before it read.
template <int D, int NT, int kSlots>
__device__ __forceinline__ void chunk_mma(const ChunkParams &p, ChunkShared &sh, const uint8_t *q_tiles,
                                          const uint8_t *tiles, uint32_t tmem) {
  constexpr int kOperand = 128 * D * 2;
  constexpr uint32_t kQk = mma_idesc(kTileTokens, false), kPv = mma_idesc(D, true);
  const uint32_t q0 = smem_u32(q_tiles), kv0 = smem_u32(tiles);
  ChunkBars &bar = sh.bars;
  auto wait = [&](uint64_t &b, int phase) { return mbar_wait_bounded(smem_u32(&b), phase & 1); };
  auto scores = [&](int x, int slot) {
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      const uint32_t at = (k >> 2) * kPanel + (k & 3) * 32;
      tc_mma_ss(tmem + kTmemS + 128 * x, operand_desc(q0 + x * kOperand + at, 16, 1024),
                operand_desc(kv0 + slot * kOperand + at, 16, 1024), kQk, k > 0);
    }
  };
  auto values = [&](int x, int slot, bool accumulate) {
#pragma unroll
    for (int k = 0; k < kTileTokens / 16; ++k)
      tc_mma_ts(tmem + kTmemO + 128 * x, tmem + kTmemS + 128 * x + 8 * k,
                operand_desc(kv0 + slot * kOperand + k * 2048, kPanel, 1024), kPv, accumulate || k > 0);
  };
  bool ok = wait(bar.q_full, 0) && wait(bar.kv_full[0], 0);
  if (ok && sh.meta[0].none) {  // nothing to attend: the softmax only has to know
    for (int x = 0; x < NT; ++x) mbar_arrive(smem_u32(&bar.s_full[x]));
    return;
  }
  if (ok) {
    tc_fence_after();
#pragma unroll
    for (int x = 0; x < NT; ++x) {
      scores(x, 0);
      tc_commit(smem_u32(&bar.s_full[x]));
    }
    tc_commit(smem_u32(&bar.kv_empty[0]));
  }
  for (int j = 0; ok; ++j) {
    const bool last = sh.meta[j % kMetas].last;
    const int vn = 2 * j + 1, kn = 2 * j + 2, vs = vn % kSlots, ks = kn % kSlots;
#pragma unroll
    for (int x = 0; x < NT; ++x) {
      ok = ok && wait(bar.p_full[x], j) && (x > 0 || wait(bar.kv_full[vs], vn / kSlots));
      if (!ok) break;
      tc_fence_after();
      values(x, vs, j > 0);
      if (x == NT - 1) tc_commit(smem_u32(&bar.kv_empty[vs]));
      if (last) {
        tc_commit(smem_u32(&bar.o_full[x]));
        continue;
      }
      ok = x > 0 || wait(bar.kv_full[ks], kn / kSlots);
      if (!ok) break;
      tc_fence_after();
      scores(x, ks);
      tc_commit(smem_u32(&bar.s_full[x]));
      if (x == NT - 1) tc_commit(smem_u32(&bar.kv_empty[ks]));
    }
    if (last) break;
  }
  if (!ok) set_status(p.a.status, AKV_DEV_TIMEOUT);
}

// ----------------------------------------------------------------- softmax
// Load row tile x of Q into its operand tile: a warp takes two rows of head_dim
// 128 (four of 64) at a time, 16 bytes a lane.  A negative softmax scale is
// folded into Q's sign (exact), so that the row max is the max of the products.
template <int D>
__device__ __forceinline__ void load_rows(const ChunkParams &p, const ChunkView &view, int b, int kvh, int x, int warp,
                                          int lane, uint8_t *tile) {
  constexpr int kUnits = D / 8, kPer = 32 / kUnits;
  const ChunkArgs &a = p.a;
  const uint32_t flip = p.q_sign < 0 ? 0x80008000u : 0u, keep = p.q_sign == 0 ? 0u : 0xffffffffu;
  const int unit = lane % kUnits;
#pragma unroll 4
  for (int i = 0; i < 32; i += kPer) {
    const int row = 32 * warp + i + lane / kUnits, r = 128 * x + row;
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (r < view.n) {
      const int rho = view.row0 + r, t = rho / p.heads_per_kv, h = kvh * p.heads_per_kv + (rho - t * p.heads_per_kv);
      v = __ldg(reinterpret_cast<const uint4 *>(a.q + (int64_t)b * a.q_bs + (int64_t)h * a.q_hs + (int64_t)t * a.q_ts) + unit);
      v.x = (v.x ^ flip) & keep, v.y = (v.y ^ flip) & keep, v.z = (v.z ^ flip) & keep, v.w = (v.w ^ flip) & keep;
    }
    *reinterpret_cast<uint4 *>(tile + panel_offset(row, unit)) = v;
  }
}

__device__ __forceinline__ uint32_t bits_below(int n) {  // the n lowest of 16 bits, n clamped
  return n <= 0 ? 0u : (n >= 16 ? 0xffffu : (1u << n) - 1u);
}

template <int D>
__device__ __forceinline__ void chunk_softmax(const ChunkParams &p, ChunkShared &sh, const ChunkView &view, int b,
                                              int kvh, int x, int warp, int lane, uint32_t tmem) {
  const uint32_t lane_base = (uint32_t)(32 * warp) << 16;
  const uint32_t ts = tmem + lane_base + kTmemS + 128 * x, to = tmem + lane_base + kTmemO + 128 * x;
  const int r = 128 * x + 32 * warp + lane;
  const int at = view.at_first + (view.row0 + min(r, view.n - 1)) / p.heads_per_kv;
  const float c = p.scale_log2;
  constexpr float kNegInf = -INFINITY, kSlack = 8.f;
  float m = kNegInf, l = 0.f;
  bool dead = false;
  for (int j = 0;; ++j) {
    if (!mbar_wait_bounded(smem_u32(&sh.bars.s_full[x]), j & 1)) {
      dead = true;
      break;
    }
    tc_fence_after();
    const TileMeta &meta = sh.meta[j % kMetas];
    const bool last = meta.last;
    if (meta.none) break;
    float s[128];
#pragma unroll
    for (int i = 0; i < 4; ++i) tc_ld32(ts + 32 * i, s + 32 * i);
    tc_wait_ld();
    if (!meta.whole) {
#pragma unroll
      for (int g = 0; g < kTilePages; ++g) {
        const int pos0 = kBlock * meta.col[g], ntok = (int)(meta.page[g] >> 2);
        const uint32_t bits = bits_below(min(ntok, at - pos0 + 1)) &
                              (~bits_below(at - view.window - pos0 + 1) | bits_below(view.sinks - pos0));
#pragma unroll
        for (int i = 0; i < kBlock; ++i)
          if (!((bits >> i) & 1u)) s[kBlock * g + i] = kNegInf;
      }
    }
    float tops[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) tops[i] = s[i];
#pragma unroll
    for (int i = 8; i < 128; ++i) tops[i % 8] = fmaxf(tops[i % 8], s[i]);
    const float top = c * fmaxf(fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])),
                                fmaxf(fmaxf(tops[4], tops[5]), fmaxf(tops[6], tops[7])));
    // S of this tile came after O of the tile before it, so O is at rest here.
    if (__any_sync(0xffffffffu, top > m + kSlack)) {
      const float n = fmaxf(m, top);
      const float w = n == kNegInf ? 1.f : ex2(m - n);
      l *= w, m = n;
      if (j > 0) {
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          float o[32];
          tc_ld32(to + 32 * i, o);
          tc_wait_ld();
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] *= w;
          tc_st32(to + 32 * i, reinterpret_cast<const uint32_t *>(o));
        }
      }
    }
    const float neg = m == kNegInf ? 0.f : -m;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t pk[32];
#pragma unroll
      for (int k = 0; k < 32; ++k) {
        const float p0 = ex2(fmaf(s[64 * i + 2 * k], c, neg)), p1 = ex2(fmaf(s[64 * i + 2 * k + 1], c, neg));
        sum[2 * (k & 1)] += p0, sum[2 * (k & 1) + 1] += p1;
        pk[k] = pack_f16x2(p0, p1);
      }
      tc_st32(ts + 32 * i, pk);
    }
    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
    tc_wait_st();
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&sh.bars.p_full[x]));
    if (last) break;
  }
  const bool none = sh.meta[0].none;  // set once, for a CTA without a tile
  if (!dead && !none && !mbar_wait_bounded(smem_u32(&sh.bars.o_full[x]), 0)) dead = true;
  if (dead) {
    if (lane == 0) set_status(p.a.status, AKV_DEV_TIMEOUT);
    return;
  }
  tc_fence_after();
  const ChunkArgs &a = p.a;
  const int rho = view.row0 + r, t = rho / p.heads_per_kv, h = kvh * p.heads_per_kv + (rho - t * p.heads_per_kv);
  __half *out = a.out + (int64_t)b * a.o_bs + (int64_t)h * a.o_hs + (int64_t)t * a.o_ts;
  const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    float o[32];
    tc_ld32(to + 32 * i, o);
    tc_wait_ld();
    if (r >= view.n) continue;
    uint32_t w[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) w[k] = pack_f16x2(l > 0.f ? o[2 * k] * inv : l, l > 0.f ? o[2 * k + 1] * inv : l);
    if (p.vector_out) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        reinterpret_cast<uint4 *>(out + 32 * i)[k] = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
    } else {
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        out[32 * i + 2 * k] = __ushort_as_half((unsigned short)(w[k] & 0xffff));
        out[32 * i + 2 * k + 1] = __ushort_as_half((unsigned short)(w[k] >> 16));
      }
    }
  }
}

// ---------------------------------------------------------- CTA set-up
__device__ __forceinline__ void chunk_begin(ChunkShared &sh, int nt, int kv_arrivals, int alloc_warp) {
  if (threadIdx.x == 0) {
    ChunkBars &bar = sh.bars;
    for (int i = 0; i < kItems; ++i) mbar_init(smem_u32(&bar.raw_full[i]), 1), mbar_init(smem_u32(&bar.raw_empty[i]), 4);
    for (int i = 0; i < kMaxSlots; ++i)
      mbar_init(smem_u32(&bar.kv_full[i]), kv_arrivals), mbar_init(smem_u32(&bar.kv_empty[i]), 1);
    mbar_init(smem_u32(&bar.q_full), 4 * nt);
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&bar.s_full[i]), 1);
      mbar_init(smem_u32(&bar.p_full[i]), 4);
      mbar_init(smem_u32(&bar.o_full[i]), 1);
    }
    fence_mbar_init();
    sh.meta[0].none = 0;
  }
  if ((int)(threadIdx.x >> 5) == alloc_warp) {
    tmem_alloc(smem_u32(&sh.tmem), kTmemCols);
    tmem_release_permit();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
}
__device__ __forceinline__ void chunk_end(uint32_t tmem, int alloc_warp) {
  tc_fence_before();
  __syncthreads();
  if ((int)(threadIdx.x >> 5) == alloc_warp) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}
template <int D>
__device__ __forceinline__ void chunk_rows_role(const ChunkParams &p, ChunkShared &sh, const ChunkView &view, int b,
                                                int kvh, int x, int w, int lane, uint8_t *q_tile, uint32_t tmem) {
  load_rows<D>(p, view, b, kvh, x, w, lane, q_tile);
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) mbar_arrive(smem_u32(&sh.bars.q_full));
  chunk_softmax<D>(p, sh, view, b, kvh, x, w, lane, tmem);
}

// ============================================== pages dequantised in the kernel
constexpr int kPageSlots = 4;
// Registers a thread: at launch, and after the split (softmax, dequantisation, loader and MMA warpgroups).
constexpr int kPageThreads = 512;
constexpr int kPageRegs = 128, kSoftmaxRegs = 192, kDequantRegs = 80, kIssueRegs = 48;
static_assert(2 * kSoftmaxRegs + kDequantRegs + kIssueRegs <= 4 * kPageRegs, "a warpgroup would wait for registers");

template <int D, bool SLAB, int NT>
__global__ void __launch_bounds__(kPageThreads, 1) chunk_pages_kernel(const __grid_constant__ ChunkParams p) {
  constexpr int kOperand = 128 * D * 2;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t *q_tiles = smem, *tiles = smem + NT * kOperand, *ring = tiles + kPageSlots * kOperand;
  ChunkShared &sh = *reinterpret_cast<ChunkShared *>(ring + kRawRing);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  chunk_begin(sh, NT, 4, 13);
  const uint32_t tmem = sh.tmem;
  grid_dependency_wait();
  allow_dependents_launch();
  const int kvh = blockIdx.y, b = blockIdx.z;
  const int row0 = (int)blockIdx.x * (128 * NT);
  const ChunkView view = chunk_view(p, b, row0, min(128 * NT, p.rows_kv - row0));
  if (warp < 8) {
    const int x = warp >> 2, w = warp & 3;
    set_registers_up<kSoftmaxRegs>();
    if (x < NT) chunk_rows_role<D>(p, sh, view, b, kvh, x, w, lane, q_tiles + x * kOperand, tmem);
  } else if (warp < 12) {
    set_registers_down<kDequantRegs>();
    chunk_dequant<D, SLAB>(p, sh, ring, tiles, view, warp - 8, lane);
  } else {
    set_registers_down<kIssueRegs>();
    if (warp == 12) chunk_load<D>(p, sh, ring, view, b, kvh, lane);
    if (warp == 13 && lane == 0) chunk_mma<D, NT, kPageSlots>(p, sh, q_tiles, tiles, tmem);
    __syncwarp();
  }
  chunk_end(tmem, 13);
}

// ==================================================== pages dequantised before
// Where many row tiles share the pages, each page is dequantised once per call
// into operand tiles in the workspace (plan, then unpack), and the attention
// kernel copies whole tiles:
//   counts [batch]                resident pages the call's rows may see
//   lists  [batch][tiles * 8]     their descriptors, in order
//   metas  [batch][tiles]         their columns and valid tokens
//   tiles  [batch][kv head][tile] K tile, V tile
struct __align__(16) PageList {  // of one tile, as the kernels read it: 64 bytes
  int32_t col[kTilePages];
  uint32_t page[kTilePages];
};
struct ChunkSpace {
  int32_t *counts;
  int64_t *lists;
  PageList *metas;
  uint8_t *tiles;
  int32_t tiles_max;
};

// One CTA per sequence: the resident pages in column order.
__global__ void __launch_bounds__(1024) chunk_plan_kernel(const __grid_constant__ ChunkParams p, const ChunkSpace w) {
  __shared__ int warps[32];
  grid_dependency_wait();
  allow_dependents_launch();
  const ChunkArgs &a = p.a;
  const int b = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const ChunkView view = chunk_view(p, b, 0, p.rows_kv);
  const int64_t *table = a.table + (int64_t)b * a.table_stride;
  int64_t *list = w.lists + (int64_t)b * w.tiles_max * kTilePages;
  PageList *metas = w.metas + (int64_t)b * w.tiles_max;
  int n = 0;
  for (int base = 0; base < view.total; base += 1024) {
    const int v = base + (int)threadIdx.x;
    int64_t d = 0;
    int col = 0;
    if (v < view.total) {
      col = view.column(v);
      d = __ldg(table + col);
    }
    const int mode = desc_mode(d);
    bool ok = mode != AKV_MODE_SKIP;
    if (ok && !page_in_arena(d, a.kv_heads * record_bytes(a.head_dim, 1 << a.log2_group, mode), a.arena_bytes)) {
      set_status(a.status, AKV_DEV_BAD_DESCRIPTOR);
      ok = false;
    }
    const uint32_t mask = __ballot_sync(0xffffffffu, ok);
    if (lane == 0) warps[warp] = __popc(mask);
    __syncthreads();
    int before = 0, all = 0;
    for (int i = 0; i < 32; ++i) {
      if (i == warp) before = all;
      all += warps[i];
    }
    __syncthreads();
    if (ok) {
      const int rank = n + before + __popc(mask & ((1u << lane) - 1u));
      list[rank] = d;
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
}

// One warp per (KV head, page, K or V) of a tile: 8 elements a lane and step, all
// loads of a page issued before the first is converted.
template <int D, bool SLAB>
__global__ void __launch_bounds__(256) chunk_unpack_kernel(const __grid_constant__ ChunkParams p, const ChunkSpace w) {
  constexpr int kOperand = 128 * D * 2, NC = D / 16, kUnits = D / 8, kRows = 32 / kUnits;
  grid_dependency_wait();
  allow_dependents_launch();
  const ChunkArgs &a = p.a;
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
    const uint8_t *rec = a.arena + desc_offset(d) + kvh * record_bytes(D, 1 << a.log2_group, mode);
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

// The loader of whole tiles: 32 tiles' lists at a time, one per lane, a window
// ahead; tiles that no row of the CTA sees are passed over.
template <int D, int kSlots>
__device__ __forceinline__ void chunk_load_tiles(const ChunkParams &p, const ChunkSpace &w, ChunkShared &sh,
                                                 uint8_t *tiles, const ChunkView &view, int b, int kvh, int lane) {
  constexpr int kOperand = 128 * D * 2;
  const int pages = __ldcg(w.counts + b), count = (pages + kTilePages - 1) / kTilePages;
  const PageList *metas = w.metas + (int64_t)b * w.tiles_max;
  const uint8_t *src = w.tiles + ((int64_t)b * p.a.kv_heads + kvh) * w.tiles_max * 2 * kOperand;
  uint4 next[4], cur[4];
  auto fetch = [&](int w0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) next[i] = make_uint4(0u, 0u, 0u, 0u);
    if (w0 + lane < count) {
#pragma unroll
      for (int i = 0; i < 4; ++i) next[i] = __ldcg(reinterpret_cast<const uint4 *>(metas + w0 + lane) + i);
    }
  };
  uint32_t mask = 0, wholes = 0;
  int win0 = 0;
  auto prepare = [&]() {
#pragma unroll
    for (int i = 0; i < 4; ++i) cur[i] = next[i];
    const uint32_t c[8] = {cur[0].x, cur[0].y, cur[0].z, cur[0].w, cur[1].x, cur[1].y, cur[1].z, cur[1].w};
    const uint32_t g[8] = {cur[2].x, cur[2].y, cur[2].z, cur[2].w, cur[3].x, cur[3].y, cur[3].z, cur[3].w};
    bool some = false, whole = true;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int col = (int)c[i], p0 = kBlock * col;
      const bool here = (g[i] & 3u) != 0;
      some |= here && p0 <= view.at_hi && (p0 + kBlock - 1 > view.at_lo - view.window || p0 < view.sinks);
      whole &= here && (g[i] >> 2) == kBlock && view.whole_page(col);
    }
    mask = __ballot_sync(0xffffffffu, some);
    wholes = __ballot_sync(0xffffffffu, whole);
  };
  fetch(0);
  prepare();
  fetch(32);
  auto seek = [&]() {  // to the next window with a visible tile
    while (mask == 0 && win0 + 32 < count) {
      win0 += 32;
      prepare();
      fetch(win0 + 32);
    }
  };
  seek();
  if (mask == 0) {
    if (lane == 0) {
      sh.meta[0].last = 1, sh.meta[0].none = 1;
      mbar_arrive(smem_u32(&sh.bars.kv_full[0]));
    }
    return;
  }
  for (int t = 0, n = 0;; ++t) {
    const int k = __ffs(mask) - 1, tile = win0 + k;
    TileMeta &m = sh.meta[t % kMetas];
    // The first of this tile's slots is free only after the tile that last used
    // its meta has been attended, so the wait comes before the writes.
    const int slot = n % kSlots;
    if (!mbar_wait_bounded(smem_u32(&sh.bars.kv_empty[slot]), ((n / kSlots) & 1) ^ 1)) break;
    if (lane == k) {
#pragma unroll
      for (int i = 0; i < 4; ++i) reinterpret_cast<uint4 *>(&m)[i] = cur[i];
      m.whole = (wholes >> k) & 1u;
    }
    mask &= mask - 1u;
    seek();
    const bool last = mask == 0;
    if (lane == 0) m.last = last, m.none = 0;
    __syncwarp();
    bool ok = true;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv, ++n) {
      const int s = n % kSlots;
      if (kv == 1) ok = mbar_wait_bounded(smem_u32(&sh.bars.kv_empty[s]), ((n / kSlots) & 1) ^ 1);
      if (!ok) break;
      if (lane == 0) {
        const uint32_t bar = smem_u32(&sh.bars.kv_full[s]);
        mbar_expect_tx(bar, kOperand);
        bulk_g2s(smem_u32(tiles + s * kOperand), src + ((int64_t)tile * 2 + kv) * kOperand, kOperand, bar);
      }
    }
    if (!ok) {  // the copies in flight end before the CTA does: its K tile's, at most
      mbar_wait_bounded(smem_u32(&sh.bars.kv_full[slot]), ((n - 1) / kSlots) & 1);
      break;
    }
    if (last) return;
  }
  if (lane == 0) set_status(p.a.status, AKV_DEV_TIMEOUT);
}

constexpr int kTileThreads = 384;
// At launch, and after the split (softmax warpgroups; loader and MMA warpgroup).
constexpr int kTileRegs = 168, kTileSoftmaxRegs = 216, kTileIssueRegs = 72;
static_assert(2 * kTileSoftmaxRegs + kTileIssueRegs <= 3 * kTileRegs, "a warpgroup would wait for registers");
template <int D>
constexpr int tile_slots() {
  return D == 128 ? 5 : 8;
}

template <int D>
__global__ void __launch_bounds__(kTileThreads, 1)
    chunk_tiles_kernel(const __grid_constant__ ChunkParams p, const ChunkSpace w) {
  constexpr int kOperand = 128 * D * 2, kSlots = tile_slots<D>();
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t *q_tiles = smem, *tiles = smem + 2 * kOperand;
  ChunkShared &sh = *reinterpret_cast<ChunkShared *>(tiles + kSlots * kOperand);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  chunk_begin(sh, 2, 1, 9);
  const uint32_t tmem = sh.tmem;
  grid_dependency_wait();
  allow_dependents_launch();
  const int kvh = blockIdx.y, b = blockIdx.z;
  const int row0 = (int)blockIdx.x * 256;
  const ChunkView view = chunk_view(p, b, row0, min(256, p.rows_kv - row0));
  if (warp < 8) {
    set_registers_up<kTileSoftmaxRegs>();
    const int x = warp >> 2;
    chunk_rows_role<D>(p, sh, view, b, kvh, x, warp & 3, lane, q_tiles + x * kOperand, tmem);
  } else {
    set_registers_down<kTileIssueRegs>();
    if (warp == 8) chunk_load_tiles<D, kSlots>(p, w, sh, tiles, view, b, kvh, lane);
    if (warp == 9 && lane == 0) chunk_mma<D, 2, kSlots>(p, sh, q_tiles, tiles, tmem);
    __syncwarp();
  }
  chunk_end(tmem, 9);
}

// ------------------------------------------------------------------- host
// Raise a kernel's shared-memory limit, once per device, and check that it starts
// with the registers its warpgroups then share out.
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

template <int D, bool SLAB, int NT>
static cudaError_t launch_pages(const ChunkParams &p) {
  constexpr int smem = (NT + kPageSlots) * 128 * D * 2 + kRawRing + (int)sizeof(ChunkShared);
  static_assert(smem <= 232448, "one CTA's shared memory");
  static std::atomic<bool> ready[256];
  if (cudaError_t err = chunk_ready(chunk_pages_kernel<D, SLAB, NT>, smem, kPageRegs, ready)) return err;
  const dim3 grid((p.rows_kv + 128 * NT - 1) / (128 * NT), p.a.kv_heads, p.a.batch);
  return launch_dependent(chunk_pages_kernel<D, SLAB, NT>, grid, kPageThreads, smem, p.a.stream, p);
}

template <int D, bool SLAB>
static cudaError_t launch_tiles(const ChunkParams &p, const ChunkSpace &w) {
  constexpr int smem = (2 + tile_slots<D>()) * 128 * D * 2 + (int)sizeof(ChunkShared);
  static_assert(smem <= 232448, "one CTA's shared memory");
  static std::atomic<bool> ready[256];
  if (cudaError_t err = chunk_ready(chunk_tiles_kernel<D>, smem, kTileRegs, ready)) return err;
  cudaStream_t s = p.a.stream;
  if (cudaError_t err = launch_dependent(chunk_plan_kernel, p.a.batch, 1024, 0, s, p, w)) return err;
  if (w.tiles_max > 0)
    if (cudaError_t err = launch_dependent(chunk_unpack_kernel<D, SLAB>, dim3(w.tiles_max, p.a.batch, 2), 256, 0, s, p, w))
      return err;
  const dim3 grid((p.rows_kv + 255) / 256, p.a.kv_heads, p.a.batch);
  return launch_dependent(chunk_tiles_kernel<D>, grid, kTileThreads, smem, s, p, w);
}

// Tiles the rows of a call may see, at most.
static int64_t space_tiles(const ChunkArgs &a) {
  int64_t columns = a.columns;
  if (a.window < (1 << 30)) columns = std::min<int64_t>(columns, a.lead + ((int64_t)a.window + a.rows + 2 * kBlock - 3) / kBlock);
  return (columns + kTilePages - 1) / kTilePages;
}
static int64_t align256(int64_t n) { return (n + 255) & ~(int64_t)255; }
static int64_t space_layout(const ChunkArgs &a, int64_t tiles, uint8_t *base, ChunkSpace *w) {
  const int64_t counts = 0, lists = align256(4ll * a.batch);
  const int64_t metas = lists + align256(8ll * kTilePages * tiles * a.batch);
  const int64_t data = (metas + align256((int64_t)sizeof(PageList) * tiles * a.batch) + 1023) & ~(int64_t)1023;
  if (w) {
    w->counts = (int32_t *)(base + counts), w->lists = (int64_t *)(base + lists);
    w->metas = (PageList *)(base + metas), w->tiles = base + data, w->tiles_max = (int32_t)tiles;
  }
  return data + tiles * a.batch * a.kv_heads * 2 * 128 * a.head_dim * 2;
}

int64_t chunk_tiles_bytes(const ChunkArgs &a) {
  return a.rows * (a.q_heads / a.kv_heads) > 128 ? space_layout(a, space_tiles(a), nullptr, nullptr) : 0;
}

int chunk_tiles_launch(const ChunkArgs &a, void *workspace, int64_t workspace_bytes) {
  ChunkParams p;
  p.a = a;
  p.heads_per_kv = a.q_heads / a.kv_heads;
  p.rows_kv = a.rows * p.heads_per_kv;
  // scale 0 weighs every token alike: Q counts as zero
  p.q_sign = a.scale > 0.f ? 1 : (a.scale < 0.f ? -1 : 0);
  p.scale_log2 = p.q_sign == 0 ? 1.f : fabsf(a.scale) * 1.4426950408889634f;
  p.vector_out = ((uintptr_t)a.out & 15) == 0 && a.o_bs % 8 == 0 && a.o_hs % 8 == 0 && a.o_ts % 8 == 0;
  const bool slab = (1 << a.log2_group) == 16 * a.head_dim;
  const int64_t need = chunk_tiles_bytes(a);
  cudaError_t err;
  if (need > 0) {
    if (workspace_bytes < need) return AKV_ERR_INVALID;
    ChunkSpace w;
    space_layout(a, space_tiles(a), (uint8_t *)workspace, &w);
    if (a.head_dim == 64) err = slab ? launch_tiles<64, true>(p, w) : launch_tiles<64, false>(p, w);
    else err = slab ? launch_tiles<128, true>(p, w) : launch_tiles<128, false>(p, w);
  } else {
    if (a.head_dim == 64) err = slab ? launch_pages<64, true, 1>(p) : launch_pages<64, false, 1>(p);
    else err = slab ? launch_pages<128, true, 1>(p) : launch_pages<128, false, 1>(p);
  }
  return err == cudaSuccess ? AKV_OK : AKV_ERR_CUDA;
}

}  // namespace akv
