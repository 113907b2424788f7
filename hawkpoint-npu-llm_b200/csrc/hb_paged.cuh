// hb_paged.cuh -- what the paged-cache operators share: the page layout, the
// view of a call's rows, and the division of an attention call's work.
//
// A page holds 64 positions of every layer and kv head:
// [layer][kv head][K | V][head_dim / 64][64 positions][64 dims], two-byte
// elements, the eight 16-byte blocks of a position's 64 dims stored at
// block ^ (position & 7).  A [64][64] block is thus 8 KB whose rows of 128
// bytes are swizzled as a 128-byte-swizzled shared-memory operand wants them:
// a plain bulk copy of a page's K or V is an MMA operand tile, and its first
// r positions are its first 128 r bytes.
#pragma once

#include <cuda_fp16.h>

#include "hawkb200.h"
#include "hb_attn.cuh"

namespace hb {
namespace paged {

constexpr int kPage = 64;             // positions a page
constexpr int kBlockBytes = 8192;     // [64 positions][64 dims]
constexpr int kMaxEntries = 1024;     // batch entries a call

// The workspace's first bytes: the waits' control block and the operators'
// sticky status, then what a page operator's first kernel leaves for its
// second one.
struct Control {
  Ctrl ctrl;
  int status;    // HB_PAGED_* bits, cleared by hb_paged_status
  int copies;    // entries of the copy list
  int refused;   // a reserve or fork changed nothing since the status was read
  int began;     // pair_arrive, zero between calls
  int pad[4];
};
static_assert(sizeof(Control) == 64, "control block");

// A pool as the kernels see it.
struct Pool {
  uint8_t *pages;
  int64_t page_stride;   // bytes from page to page
  int n_pages, kv_heads, width, n_slots;
  int *table, *refs, *lengths;
  Control *control;
};

// A call's rows: entry b is slot slots[b] with rows row_start[b] ..
// row_start[b + 1].
struct Batch {
  const int *slots, *row_start;
  int entries, rows;
};

struct Entry {
  int row0, n, length, slot;   // n < 0: the row starts descend; slot -1: none (its rows see nothing)
};

// What an earlier kernel may have written.  The attention kernels read it past
// L1 (PAST): a block needs each once.
template <bool PAST, class T>
__device__ __forceinline__ T read(const T *p) {
  return PAST ? __ldcg(p) : *p;
}

// Entry b with every index held inside its array.
template <bool PAST = false>
__device__ __forceinline__ Entry entry_of(const Pool &P, const Batch &B, int b) {
  Entry e;
  e.row0 = min(max(read<PAST>(B.row_start + b), 0), B.rows);
  e.n = min(max(read<PAST>(B.row_start + b + 1), 0), B.rows) - e.row0;
  e.slot = read<PAST>(B.slots + b);
  if (e.slot < 0 || e.slot >= P.n_slots) e.slot = -1;
  e.length = e.slot < 0 ? 0 : max(read<PAST>(P.lengths + e.slot), 0);
  return e;
}

// Every kernel here is launched early (programmatic launch): its blocks take
// their places while the kernel before it ends, wait for it and what it wrote,
// and let the next one do the same.  Waiting comes first, so that at most two
// kernels of a stream are under way.
__device__ __forceinline__ void grid_begin() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// A call of two kernels, the second launched early and beside the first, whose
// results it does not need, only what the first one's wait made visible.  A
// wait of its own would last until the first one ends (7 to 11 us more in a
// step of 96 streams of which 12 or 24 have chunks).  So the first's first block
// counts kFirst up when it has waited, before it lets the second begin, and
// the second's blocks count one up each: a block that finds the first one's
// count has what came before it (release and acquire, cumulative), one that
// does not (it cannot happen, but nothing here depends on that) waits in full.
// Whoever completes the count sets it to zero.  True: kFirst was there.
constexpr int kFirst = 1 << 16;   // more than the second kernel has blocks
__device__ __forceinline__ bool pair_arrive(Control *c, int n, int blocks) {
  int old;
  asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], %2;" : "=r"(old) : "l"(&c->began), "r"(n) : "memory");
  if (old + n == kFirst + blocks) atomicExch(&c->began, 0);
  return old >= kFirst;
}
__device__ __forceinline__ void first_begin(Control *c, int blocks) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (blockIdx.x == 0 && threadIdx.x == 0) pair_arrive(c, kFirst, blocks);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
// `seen`: a word of shared memory.  The second kernel lets none begin early,
// and waits for the first one before it ends (grid_end), so that whoever waits
// for it has waited for both.
__device__ __forceinline__ void second_begin(Control *c, int *seen) {
  if (threadIdx.x == 0) *seen = pair_arrive(c, 1, gridDim.x);
  __syncthreads();
  if (*seen == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("fence.proxy.async;" ::: "memory");   // the bulk copies of pages, which earlier kernels wrote
}
__device__ __forceinline__ void grid_end() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ---- division of an attention call --------------------------------------------
// The rows of an entry and the q heads of a kv head's group are packed into
// tiles of `tile` rows: packed row r is row r / group, head r % group.  A
// tile's work is the blocks of `block` positions that any of its rows sees
// (one at least, so that a tile without any is still written), and `extra`
// units for its start and end.  The units of all tiles, entry by entry, head
// by head, are one line that the thread blocks cut into equal pieces, so ragged
// lengths leave none idle; a tile cut by a border is joined from its parts, in
// the pieces' order, so that results do not depend on who joins.
struct Shape {
  int group, width, window, tile, block, extra;
  uint32_t group_inv;   // 2^32 / group, rounded down (at most 2^32 - 1)
  // r / group for r >= 0: the product is at most one too low
  __device__ __forceinline__ int row_of(int r) const {
    const int q = static_cast<int>(__umulhi(static_cast<uint32_t>(r), group_inv));
    return r - q * group >= group ? q + 1 : q;
  }
  // The first position that a row at position p sees.  Compared before it is
  // subtracted: windows go up to 2^31 - 1, and p is negative for rows before
  // their sequence.
  __device__ __forceinline__ int first_seen(int p) const { return window > 0 && p >= window ? p - window + 1 : 0; }
};

struct Span {
  int lo, hi;   // blocks [lo, hi) of positions; hi <= lo: none
};

__device__ __forceinline__ Span tile_span(const Shape &S, const Entry &e, int t) {
  const int packed = e.n * S.group;
  const int i0 = S.row_of(t * S.tile), i1 = S.row_of(min(packed, (t + 1) * S.tile) - 1);
  const int last = e.length - e.n + i1, first = e.length - e.n + i0;
  // blocks are 64 or 128 positions: shifts
  const int shift = S.block == 128 ? 7 : 6;
  Span s;
  s.hi = last < 0 ? 0 : min(last >> shift, (S.width * kPage - 1) >> shift) + 1;
  s.lo = S.first_seen(first) >> shift;
  return s;
}
__device__ __forceinline__ int tile_units(const Shape &S, const Entry &e, int t) {
  const Span s = tile_span(S, e, t);
  return max(1, s.hi - s.lo) + S.extra;
}
__device__ __forceinline__ int tiles_of(const Shape &S, const Entry &e) { return (e.n * S.group + S.tile - 1) / S.tile; }

// The line of a call: its entries and prefix[b], the units before entry b, in
// shared memory.
struct Line {
  int *prefix;       // [entries + 1]; the host has checked that the total fits
  Entry *entry;      // [entries]
};
__host__ __device__ inline size_t line_bytes(int entries) {
  return (static_cast<size_t>(entries) * (4 + sizeof(Entry)) + 4 + 15) / 16 * 16;
}
__device__ __forceinline__ Line line_at(uint8_t *smem, int entries) {
  return Line{reinterpret_cast<int *>(smem + entries * sizeof(Entry)), reinterpret_cast<Entry *>(smem)};
}

// Fills the line, by all threads of the block: a thread an entry, so that the
// entries' reads are in flight together; the tiles of a long entry are
// counted by its warp.  `take(entry)`: whether this kernel takes its rows.
// False when row starts descend: entries would share rows, the host's bound
// on the total would not hold, and a total that wraps leads a walk out of the
// line.  Starts that ascend are disjoint ranges of the call's rows.
template <class Take>
__device__ __forceinline__ bool fill_line(const Pool &P, const Batch &B, const Shape &S, const Line &line,
                                          const Take &take) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  bool descends = false;
#pragma unroll 1
  for (int b0 = warp * 32; b0 < B.entries; b0 += blockDim.x) {
    const int b = b0 + lane;
    Entry e{0, 0, 0, -1};
    if (b < B.entries) line.entry[b] = e = entry_of<true>(P, B, b);
    descends |= e.n < 0;
    const int tiles = b < B.entries && take(e) ? tiles_of(S, e) : 0;
    int u = 0;
    if (tiles <= 4)
#pragma unroll 1
      for (int t = 0; t < tiles; ++t) u += tile_units(S, e, t);
    for (unsigned many = __ballot_sync(0xffffffffu, tiles > 4); many; many &= many - 1) {
      const int x = __ffs(many) - 1, n = __shfl_sync(0xffffffffu, tiles, x);
      const Entry y{0, __shfl_sync(0xffffffffu, e.n, x), __shfl_sync(0xffffffffu, e.length, x), 0};
      int v = 0;
#pragma unroll 1
      for (int t = lane; t < n; t += 32) v += tile_units(S, y, t);
      v = __reduce_add_sync(0xffffffffu, v);
      if (lane == x) u = v;
    }
    if (b < B.entries) line.prefix[b + 1] = u * P.kv_heads;
  }
  if (__syncthreads_or(descends)) {
    if (threadIdx.x == 0 && blockIdx.x == 0) atomicOr(&P.control->status, HB_PAGED_BAD_INDEX);
    return false;
  }
  if (warp == 0) {
    int base = 0;
#pragma unroll 1
    for (int b0 = 0; b0 < B.entries; b0 += 32) {
      const int b = b0 + lane;
      int v = b < B.entries ? line.prefix[b + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int w = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += w;
      }
      if (b < B.entries) line.prefix[b + 1] = base + v;
      base += __shfl_sync(0xffffffffu, v, 31);
    }
    if (lane == 0) line.prefix[0] = 0;
  }
  __syncthreads();
  return true;
}

// A walk over the tiles of one piece [u, end) of the line, the same in every
// lane of the warps that make it.
struct Walk {
  int u, end;            // units left
  int tile_u;            // first unit of the current tile, its extra ones included
  int b, head, t, units, tiles, blocks_before;
  Entry e;
  Span span;

  __device__ __forceinline__ void at(const Shape &S, int tile) {
    t = tile;
    span = tile_span(S, e, t);
    units = max(1, span.hi - span.lo) + S.extra;
    // where the piece enters the tile's blocks
    blocks_before = max(0, u - tile_u - S.extra);
  }
  // On the tile that holds unit u; false when the piece is done.
  __device__ __forceinline__ bool start(const Pool &P, const Batch &B, const Shape &S, const Line &line) {
    if (u >= end) return false;
    const int *prefix = line.prefix;
    int lo = 0, hi = B.entries - 1;
    while (lo < hi) {  // the entry that holds unit u
      const int mid = (lo + hi) >> 1;
      if (prefix[mid + 1] > u) hi = mid; else lo = mid + 1;
    }
    b = lo;
    e = line.entry[b];
    tiles = tiles_of(S, e);
    int rem = u - prefix[b];
    head = 0;
    if (P.kv_heads > 1) {
      const int per = (prefix[b + 1] - prefix[b]) / P.kv_heads;
      head = rem / per;
      rem -= head * per;
    }
    tile_u = u - rem;
    int tile = 0;
    const int lane = threadIdx.x & 31;
    for (int t0 = 0; tiles > 1; t0 += 32) {   // a lane a tile: the one that holds the unit
      const int mine = t0 + lane < tiles ? tile_units(S, e, t0 + lane) : 0;
      int sum = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += x;
      }
      const unsigned past = __ballot_sync(0xffffffffu, sum > rem);
      if (past) {
        const int x = __ffs(past) - 1;
        tile = t0 + x;
        tile_u += __shfl_sync(0xffffffffu, sum - mine, x);
        break;
      }
      const int all = __shfl_sync(0xffffffffu, sum, 31);
      rem -= all;
      tile_u += all;
    }
    at(S, tile);
    return end > tile_u + S.extra;   // else the piece ends before the tile's first block
  }
  // the piece's blocks of the tile: [first, first + count)
  __device__ __forceinline__ int first() const { return span.lo + blocks_before; }
  __device__ __forceinline__ int count(const Shape &S) const {
    return min(end, tile_u + units) - tile_u - S.extra - blocks_before;
  }
  __device__ __forceinline__ bool opens() const { return blocks_before == 0; }
  __device__ __forceinline__ bool whole() const { return opens() && tile_u + units <= end; }
  __device__ __forceinline__ bool next(const Pool &P, const Batch &B, const Shape &S, const Line &line) {
    u = tile_u + units;
    if (u + S.extra >= end) return false;
    if (t + 1 < tiles) {
      tile_u = u;
      at(S, t + 1);
      return true;
    }
    if (head + 1 < P.kv_heads) {
      ++head;
      tile_u = u;
      at(S, 0);
      return true;
    }
    // the next entry that has units
    do ++b; while (line.prefix[b + 1] == u);
    e = line.entry[b];
    tiles = tiles_of(S, e);
    head = 0;
    tile_u = u;
    at(S, 0);
    return true;
  }
};

// The line cut into `pieces` pieces, the first `longer` of them a unit longer.
struct Cut {
  int pieces, size, longer;
  __device__ __forceinline__ Cut(int total, int most, int least) {
    pieces = min(most, (total + least - 1) / least);
    size = pieces ? total / pieces : 0;
    longer = total - size * pieces;
  }
  __device__ __forceinline__ int begin(int c) const { return size * c + min(c, longer); }
  // the piece that holds unit u
  __device__ __forceinline__ int of(int u) const {
    const int border = (size + 1) * longer;
    return u < border ? u / (size + 1) : longer + (u - border) / size;
  }
};

// Counts one up and returns what was there, ordered after what the block's
// threads wrote before the barrier above it and before what they read after
// the one below it.
__device__ __forceinline__ int arrive_acq_rel(int *p) {
  int v;
  asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(v) : "l"(p) : "memory");
  return v;
}

// Another thread's count, ordered before what is read after it.
__device__ __forceinline__ int load_acquire(const int *p) {
  int v;
  asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}

// ---- elements -------------------------------------------------------------------
template <class T>
struct Elem;
template <>
struct Elem<__nv_bfloat16> {
  static constexpr uint32_t kInfinity = 0x7f80;
  static __device__ __forceinline__ float lo(uint32_t u) { return bf_lo(u); }
  static __device__ __forceinline__ float hi(uint32_t u) { return bf_hi(u); }
  static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
  }
};
template <>
struct Elem<__half> {
  static constexpr uint32_t kInfinity = 0x7c00;
  static __device__ __forceinline__ float lo(uint32_t u) { return __half2float(__ushort_as_half(u & 0xffffu)); }
  static __device__ __forceinline__ float hi(uint32_t u) { return __half2float(__ushort_as_half(u >> 16)); }
  static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
  }
};

// 8 elements; VEC: the address is 16-byte aligned.
template <bool VEC>
__device__ __forceinline__ uint4 load8(const uint16_t *p) {
  if constexpr (VEC) {
    return *reinterpret_cast<const uint4 *>(p);   // not as read-only data: nothing goes ahead of grid_begin
  } else {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      w[k] = static_cast<uint32_t>(__ldcg(p + 2 * k)) | static_cast<uint32_t>(__ldcg(p + 2 * k + 1)) << 16;
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}
template <bool VEC>
__device__ __forceinline__ void store8(uint16_t *p, const uint4 &v) {
  if constexpr (VEC) {
    *reinterpret_cast<uint4 *>(p) = v;
  } else {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      p[2 * k] = static_cast<uint16_t>(w[k]);
      p[2 * k + 1] = static_cast<uint16_t>(w[k] >> 16);
    }
  }
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// What an attention kernel gets.
struct Attend {
  Pool pool;
  Batch batch;
  int64_t layer_off, head_bytes;   // bytes: of the layer in a page, of a kv head's K and V
  const void *q;
  int64_t q_row, q_head;           // strides in elements
  void *out;
  int64_t o_row, o_head;
  float *lse;                      // [rows][q_heads], or NULL
  int q_heads;
  Shape shape;
  float scale, scale_log2;         // of the scores; times log2(e)
  int q_vec, o_vec;                // q rows / out rows are 16-byte aligned
  int o_wide;                      // 32-byte aligned
  int beside;                      // blocks of the tiles kernel that runs beside the rows kernel, 0: one has all entries
  int few;                         // entries of up to this many packed rows are the rows kernel's, others the tiles'
  float *parts;                    // joined tiles: per piece two parts
  int *arrived;                    // per piece, zero between launches
  float *parts2;                   // the tiles kernel's
  int *arrived2;
  uint64_t limit_ns;
};

__device__ __forceinline__ const uint8_t *kv_block(const Attend &A, int page, int head) {
  return A.pool.pages + static_cast<int64_t>(page) * A.pool.page_stride + A.layer_off + head * A.head_bytes;
}

// Page `j` of a slot, -1 where none is mapped.
template <bool PAST = false>
__device__ __forceinline__ int page_of(const Pool &P, int slot, int j) {
  if (slot < 0 || j < 0 || j >= P.width) return -1;
  const int pg = read<PAST>(P.table + static_cast<int64_t>(slot) * P.width + j);
  return pg >= 0 && pg < P.n_pages ? pg : -1;
}

// The call's rows but [from, to), which see nothing, by all threads of the
// grid: 0 and -infinity.
template <int D>
__device__ __noinline__ void rows_unseen(const Attend &A, int from, int to) {
  const int64_t parts = static_cast<int64_t>(A.q_heads) * (D / 8);
  const int64_t n = static_cast<int64_t>(A.batch.rows - (to - from)) * parts;
  for (int64_t x = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; x < n;
       x += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    int64_t row = x / parts;
    if (row >= from) row += to - from;
    const int part = static_cast<int>(x % parts), head = part / (D / 8), d = part % (D / 8) * 8;
    uint16_t *out = static_cast<uint16_t *>(A.out) + row * A.o_row + head * A.o_head + d;
    if (A.o_vec) store8<true>(out, make_uint4(0, 0, 0, 0)); else store8<false>(out, make_uint4(0, 0, 0, 0));
    if (A.lse != nullptr && d == 0) A.lse[row * A.q_heads + head] = -INFINITY;
  }
}

// The rows of a filled line's entries, all of the call's but before the first
// and after the last.
template <int D>
__device__ __forceinline__ void rows_of_no_entry(const Attend &A, const Line &line) {
  const Entry &last = line.entry[A.batch.entries - 1];
  const int from = line.entry[0].row0, to = last.row0 + last.n;
  if (to - from < A.batch.rows) rows_unseen<D>(A, from, to);
}

// ---- rows that did not come out finite ------------------------------------------
// The tiled kernels multiply the V of positions that a row does not see by
// weight zero, and infinity or NaN among them makes that NaN; the rows kernel
// multiplies V by two halves of a weight, which makes an infinity NaN.  So a
// row whose sum of weights is finite and whose output is not is looked at
// again, by its warp, after the block's last tile: no wait with a limit is
// open then, however long that takes.  A row whose sum is not finite saw the
// NaN itself (scores are masked, so nothing hidden gets there): it is NaN.

// Positions of [from, to) whose V holds an infinity or NaN.
struct Odd {
  int first, last;   // of either; last < first: none
  bool infinity;
};
template <int D, class T>
__device__ __forceinline__ Odd odd_values(const Attend &A, const Entry &e, int head, int from, int to) {
  constexpr uint32_t kInf = Elem<T>::kInfinity;
  const int lane = threadIdx.x & 31;
  int first = INT32_MAX, last = -1;
  bool infinity = false;
  to = min(to, e.length);
  for (int j = from + lane; j < to; j += 32) {
    const int pg = page_of<true>(A.pool, e.slot, j >> 6);
    if (pg < 0) continue;
    const uint8_t *vb = kv_block(A, pg, head) + D / 64 * kBlockBytes;
    bool odd = false;
#pragma unroll
    for (int c = 0; c < D / 8; ++c) {
      const uint4 v = __ldcg(reinterpret_cast<const uint4 *>(vb + (c >> 3) * kBlockBytes + kv_off(j & 63, c & 7)));
      const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const uint32_t lo = u[x] & 0x7fffu, hi = u[x] >> 16 & 0x7fffu;
        odd |= lo >= kInf || hi >= kInf;
        infinity |= lo == kInf || hi == kInf;
      }
    }
    if (odd) {
      first = min(first, j);
      last = j;
    }
  }
  return Odd{__reduce_min_sync(0xffffffffu, first), __reduce_max_sync(0xffffffffu, last),
             __any_sync(0xffffffffu, infinity) != 0};
}

// One output row by one warp from the positions it sees alone, in FP32: 32 of
// them a step, a score a lane, the newest first (a row that is NaN by its own
// K or V ends there).
template <int D, class T>
__device__ __forceinline__ void row_alone(const Attend &A, const Entry &e, int head, int i, int g) {
  using E = Elem<T>;
  const int lane = threadIdx.x & 31;
  const int qh = head * A.shape.group + g, row = e.row0 + i, p = e.length - e.n + i;
  const uint16_t *q = static_cast<const uint16_t *>(A.q) + row * A.q_row + qh * A.q_head;
  const int lo = A.shape.first_seen(p);
  float m = -INFINITY, l = 0.f, o[D / 32];   // l: this lane's part; dims 64 k + 2 lane, 64 k + 2 lane + 1
#pragma unroll
  for (int k = 0; k < D / 32; ++k) o[k] = 0.f;
  bool nan = false;
  for (int top = min(p, A.shape.width * kPage - 1); top >= lo && !nan; top -= 32) {
    const int j = top - lane, pg = j >= lo ? page_of<true>(A.pool, e.slot, j >> 6) : -1;
    float s = -INFINITY;
    if (pg >= 0) {
      const uint8_t *kb = kv_block(A, pg, head);
      s = 0.f;
#pragma unroll 4
      for (int c = 0; c < D / 8; ++c) {
        const uint4 k = __ldcg(reinterpret_cast<const uint4 *>(kb + (c >> 3) * kBlockBytes + kv_off(j & 63, c & 7)));
        const uint4 x = load8<false>(q + c * 8);
        const uint32_t a[4] = {k.x, k.y, k.z, k.w}, b[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int y = 0; y < 4; ++y) s = fmaf(E::lo(a[y]), E::lo(b[y]), fmaf(E::hi(a[y]), E::hi(b[y]), s));
      }
    }
    float mx = s;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
    nan = __any_sync(0xffffffffu, !(s < INFINITY)) != 0;   // NaN, or infinity less infinity
    const float nm = fmaxf(m, mx), use = nm == -INFINITY ? 0.f : nm;
    const float a = exp2_approx((m - use) * A.scale_log2), w = exp2_approx((s - use) * A.scale_log2);
    m = nm;
    l = fmaf(l, a, w);
#pragma unroll
    for (int k = 0; k < D / 32; ++k) o[k] *= a;
#pragma unroll 8
    for (int x = 0; x < 32; ++x) {
      const int px = __shfl_sync(0xffffffffu, pg, x);
      const float wx = __shfl_sync(0xffffffffu, w, x);
      if (px < 0) continue;
      const uint8_t *vb = kv_block(A, px, head) + D / 64 * kBlockBytes + kv_off((top - x) & 63, lane >> 2) + (lane & 3) * 4;
#pragma unroll
      for (int k = 0; k < D / 64; ++k) {
        const uint32_t v = __ldcg(reinterpret_cast<const uint32_t *>(vb + k * kBlockBytes));
        o[2 * k] = fmaf(wx, E::lo(v), o[2 * k]);
        o[2 * k + 1] = fmaf(wx, E::hi(v), o[2 * k + 1]);
      }
    }
    bool gone = true;   // every dim is NaN, and stays it
#pragma unroll
    for (int k = 0; k < D / 32; ++k) gone &= o[k] != o[k];
    nan |= __all_sync(0xffffffffu, gone) && __any_sync(0xffffffffu, l > 0.f);
  }
  l = warp_sum(l);
  T *out = static_cast<T *>(A.out) + row * A.o_row + qh * A.o_head + 2 * lane;
#pragma unroll
  for (int k = 0; k < D / 32; ++k)
    out[(k >> 1) * 64 + (k & 1)] = E::put(nan ? NAN : l == 0.f ? 0.f : o[k] / l);
}

// A warp's rows, `first` .. first + count - 1 of each tile of the block's piece,
// that are not finite.  done: bit 0 and bit 1 say that this block finished the
// cut tile that it entered and the one that it opened.  (The line is cut again:
// the kernels' loops have no registers to keep that for this.)
template <int D, class T>
__device__ __noinline__ void rows_again(const Attend &A, const Line line, int least, int first, int count,
                                        unsigned done) {
  const Shape &S = A.shape;
  const int lane = threadIdx.x & 31;
  const Cut cut(line.prefix[A.batch.entries], gridDim.x, least);
  Walk w;
  w.u = cut.begin(blockIdx.x);
  w.end = cut.begin(blockIdx.x + 1);
  __syncwarp();   // its lanes' stores of the rows
  for (bool more = w.start(A.pool, A.batch, S, line); more; more = w.next(A.pool, A.batch, S, line)) {
    if (!w.whole() && !(done >> (w.opens() ? 1 : 0) & 1u)) continue;
    Odd odd{0, -1, false};
    bool known = false;
    const int base = w.t * S.tile + first, end = min(w.e.n * S.group, base + count);
    for (int r = base; r < end; ++r) {
      const int i = S.row_of(r), g = r - i * S.group, p = w.e.length - w.e.n + i;
      const uint16_t *out =
          static_cast<const uint16_t *>(A.out) + (w.e.row0 + i) * A.o_row + (w.head * S.group + g) * A.o_head + lane;
      bool bad = false;
#pragma unroll
      for (int k = 0; k < D / 32; ++k) bad |= (__ldcg(out + 32 * k) & 0x7fffu) >= Elem<T>::kInfinity;
      if (!__any_sync(0xffffffffu, bad)) continue;
      if (!known) odd = odd_values<D, T>(A, w.e, w.head, w.span.lo * S.block, w.span.hi * S.block);
      known = true;
      // NaN that the row sees, and nothing else in its tile: it stays
      const bool stays = odd.first <= odd.last && !odd.infinity && odd.first >= S.first_seen(p) && odd.last <= p;
      if (!stays) row_alone<D, T>(A, w.e, w.head, i, g);
    }
  }
}

}  // namespace paged
}  // namespace hb
