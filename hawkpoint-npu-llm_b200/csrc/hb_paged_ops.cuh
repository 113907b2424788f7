// hb_paged_ops.cuh -- the paged cache's writers: RoPE and append of new K / V
// rows, and the page operators (reserve, fork, free, compact, copy).
//
// append moves each byte once: HBM bounds it from a few thousand rows on,
// the launch below.  A block takes a few rows, finds each row's entry,
// position and page once (one thread a row), then its threads take 16 bytes
// of the low and the high half of a head each, so that the rotation's two
// results are two 16-byte stores into the page's blocks; the next row's reads
// are in flight under them.  RoPE is FP32 with unfused products, rounded once.
// Measured, 14 q heads on 2 of 64, BF16: 24 prompts, 29,000 rows, 27 us,
// 4.9 TB/s, three quarters of a plain copy's rate: four rows in flight a
// thread instead of two need registers that halve the threads (52 us and
// more).  One row 2.4 us on the device, a launch.
//
// The page operators keep the pool's books on the device, so that a serving
// loop neither waits for them nor uploads tables, and can be captured: one
// thread block does the books of a call (a few thousand integers; its
// latency, a handful of block scans, is the cost) and leaves a copy list that
// a second kernel, launched early, works off with the whole GPU at HBM rate.
// A new page is always the lowest free one, so results do not depend on the
// order threads run in.  Measured: a fork of one stream 7.4 us (two launches
// and the books' four phases); of 64, 49 MB of partial pages copied, 18 us;
// compaction of 1.1 GB 191 us, 5.9 TB/s of 6.5; free and reserve for 32
// slots 8.4 us.  Books and copies as one launch, the blocks waiting for a
// flag, cost 1.3 us less of the host and 3.1 us more on the device.
#pragma once

#include "hb_paged.cuh"

namespace hb {
namespace paged {

// ---- append -------------------------------------------------------------------------
struct Append {
  Pool pool;
  Batch batch;
  int64_t layer_off, head_bytes;
  const void *qkv;
  int64_t qkv_row;               // elements
  void *q;
  int64_t q_row, q_head;
  const float *cos, *sin;        // [rope_positions][head_dim / 2]
  int rope_positions, q_heads;
  int block_rows;                // rows a block
};
constexpr int kAppendThreads = 256, kAppendRows = 64;   // the most of a block

template <class T>
__device__ __forceinline__ void rope8(const uint4 &x0, const uint4 &x1, const float *c, const float *s, uint4 &lo,
                                      uint4 &hi) {
  using E = Elem<T>;
  const uint32_t a[4] = {x0.x, x0.y, x0.z, x0.w}, b[4] = {x1.x, x1.y, x1.z, x1.w};
  uint32_t l[4], h[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    // unfused products, as the persistent decoder's rope_vals
    const float a0 = E::lo(a[k]), a1 = E::hi(a[k]), b0 = E::lo(b[k]), b1 = E::hi(b[k]);
    const float c0 = c[2 * k], c1 = c[2 * k + 1], s0 = s[2 * k], s1 = s[2 * k + 1];
    l[k] = E::pack(__fsub_rn(__fmul_rn(a0, c0), __fmul_rn(b0, s0)), __fsub_rn(__fmul_rn(a1, c1), __fmul_rn(b1, s1)));
    h[k] = E::pack(__fadd_rn(__fmul_rn(b0, c0), __fmul_rn(a0, s0)), __fadd_rn(__fmul_rn(b1, c1), __fmul_rn(a1, s1)));
  }
  lo = make_uint4(l[0], l[1], l[2], l[3]);
  hi = make_uint4(h[0], h[1], h[2], h[3]);
}

template <int D, class T, bool VEC>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(const __grid_constant__ Append A) {
  __shared__ int s_pos[kAppendRows], s_page[kAppendRows];
  grid_begin();
  const int row0 = blockIdx.x * A.block_rows, rows = min(A.block_rows, A.batch.rows - row0);
  // a thread keeps its part of a head (8 dims of either half) and takes every
  // `step`-th row, the next one's reads ahead
  constexpr int kPer = D / 16;
  const int kvh = A.pool.kv_heads, parts = (A.q_heads + 2 * kvh) * kPer;
  const int step = max(1, static_cast<int>(blockDim.x) / parts);
  const int lanes = step * parts;   // threads at work; a row with more parts than threads takes turns
  const uint16_t *qkv = static_cast<const uint16_t *>(A.qkv) + row0 * A.qkv_row;
  int x = threadIdx.x, r = x / parts;
  uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
  const auto part_of = [&](int i) { return i % parts / kPer * D + i % parts % kPer * 8; };
  if (x < lanes && r < rows) {   // does not wait for the positions
    lo = load8<VEC>(qkv + r * A.qkv_row + part_of(x));
    hi = load8<VEC>(qkv + r * A.qkv_row + part_of(x) + D / 2);
  }
  if (threadIdx.x < 32) {
    // the entry of the block's first row by 32-way search, a lane's own from there
    const int lane = threadIdx.x;
    int first = 0, n = A.batch.entries;
    while (n > 1) {
      const int stride = (n + 31) / 32, i = first + lane * stride;
      const bool in = lane * stride < n && A.batch.row_start[i] <= row0;
      const int k = max(0, 31 - __clz(__ballot_sync(0xffffffffu, in)));   // the last that starts at or before the row
      first += k * stride;
      n = min(stride, n - k * stride);
    }
    for (int i = lane; i < rows; i += 32) {
      const int row = row0 + i;
      int b = first;
      while (b + 1 < A.batch.entries && A.batch.row_start[b + 1] <= row) ++b;
      const Entry e = entry_of(A.pool, A.batch, b);
      int pos = e.length - e.n + row - e.row0, pg = -1, bad = 0;
      if (row < e.row0 || row >= e.row0 + e.n || e.slot < 0 || pos < 0) {
        pos = -1;            // no entry's row, or before its sequence: nothing to append, no position to turn to
      } else {
        pg = page_of(A.pool, e.slot, pos >> 6);
        if (pg < 0) bad = HB_PAGED_UNMAPPED;
        if (pos >= A.rope_positions) {
          bad |= HB_PAGED_BAD_INDEX;
          pos = pg = -1;
        }
      }
      if (bad) atomicOr(&A.pool.control->status, bad);
      // a reserve or fork that was refused left lengths and pages as they were: these are not this row's places
      if (ld_volatile_int(&A.pool.control->refused)) pg = -1;
      s_pos[i] = pos;
      s_page[i] = pg;
    }
  }
  __syncthreads();
  for (; x < lanes; x += blockDim.x, r = x / parts) {
    const int part = x % parts, c = part % kPer, head = part / kPer;
    const bool is_v = head >= A.q_heads + kvh, is_q = head < A.q_heads;
    const int h = is_v ? head - A.q_heads - kvh : head - A.q_heads;
    uint8_t *kv = A.pool.pages + A.layer_off + h * A.head_bytes + (is_v ? D / 64 * kBlockBytes : 0);
    uint16_t *q = static_cast<uint16_t *>(A.q) + row0 * A.q_row + head * A.q_head + c * 8;
    const uint16_t *src = qkv + part_of(x);
    const int d0 = c * 8, d1 = D / 2 + c * 8;
    if (x != static_cast<int>(threadIdx.x) && r < rows) {
      lo = load8<VEC>(src + r * A.qkv_row);
      hi = load8<VEC>(src + r * A.qkv_row + D / 2);
    }
    for (; r < rows; r += step) {
      const int pos = s_pos[r], pg = s_page[r];
      uint4 a = lo, b = hi;
      if (r + step < rows) {
        lo = load8<VEC>(src + (r + step) * A.qkv_row);
        hi = load8<VEC>(src + (r + step) * A.qkv_row + D / 2);
      }
      if (!is_v) {
        if (pos >= 0) {
          const int64_t off = static_cast<int64_t>(pos) * (D / 2) + c * 8;
          // plain loads, as load8's: the heads of a row share them in L1
          const float4 c0 = *reinterpret_cast<const float4 *>(A.cos + off), c1 = *(reinterpret_cast<const float4 *>(A.cos + off) + 1);
          const float4 s0 = *reinterpret_cast<const float4 *>(A.sin + off), s1 = *(reinterpret_cast<const float4 *>(A.sin + off) + 1);
          const float cv[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
          const float sv[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
          rope8<T>(a, b, cv, sv, a, b);
        } else {
          a = b = make_uint4(0, 0, 0, 0);
        }
      }
      if (is_q) {
        store8<VEC>(q + r * A.q_row, a);
        store8<VEC>(q + r * A.q_row + D / 2, b);
      } else if (pg >= 0) {
        uint8_t *dst = kv + pg * A.pool.page_stride;
        *reinterpret_cast<uint4 *>(dst + (d0 >> 6) * kBlockBytes + kv_off(pos & 63, (d0 & 63) >> 3)) = a;
        *reinterpret_cast<uint4 *>(dst + (d1 >> 6) * kBlockBytes + kv_off(pos & 63, (d1 & 63) >> 3)) = b;
      }
    }
  }
}

// ---- page operators ------------------------------------------------------------------
constexpr int kBookThreads = 1024;

// A call's scratch in the workspace.
struct Scratch {
  int *mark;     // [n_slots]: zero between calls
  int *need;     // [max(n_slots, ..)] pages an entry needs
  int *off;      // exclusive sum of need
  int *fresh;    // [n_pages] the lowest free pages
  int *from, *to, *held;   // the copy list: page, page, positions
  int *stage;    // [n_slots][width]: rows in the making
};

// Exclusive sum over the block of v, by thread; `sum` gets the total.
__device__ __forceinline__ int block_scan(int v, int *warp_sums, int &sum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  int s = warp_sums[lane];   // kBookThreads / 32 = 32 warps
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += y;
  }
  sum = __shfl_sync(0xffffffffu, s, 31);
  const int before = __shfl_sync(0xffffffffu, s, (warp + 31) & 31);
  __syncthreads();           // warp_sums may be written again
  return x - v + (warp ? before : 0);
}

// The `want` lowest pages that nobody holds, ascending, into fresh[];
// returns how many there are (at most want).
__device__ __forceinline__ int lowest_free(const int *refs, int n_pages, int want, int *fresh, int *warp_sums) {
  int found = 0;
  for (int base = 0; base < n_pages && found < want; base += 4 * kBookThreads) {
    const int p = base + 4 * threadIdx.x;
    int n = 0;
    bool f[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      f[k] = p + k < n_pages && refs[p + k] == 0;
      n += f[k] ? 1 : 0;
    }
    int sum, at = found + block_scan(n, warp_sums, sum);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (f[k]) {
        if (at < want) fresh[at] = p + k;
        ++at;
      }
    found += sum;
  }
  return min(found, want);
}

// off[b] = pages that entries before b need; returns all of them.
__device__ __forceinline__ int scan_needs(const int *need, int *off, int n, int *warp_sums) {
  int total = 0;
  for (int b0 = 0; b0 < n; b0 += kBookThreads) {
    const int b = b0 + threadIdx.x;
    int sum;
    const int x = block_scan(b < n ? need[b] : 0, warp_sums, sum);
    if (b < n) off[b] = total + x;
    total += sum;
  }
  return total;
}

// One entry of the copy list: the first `held` positions of a page.
__device__ __forceinline__ void push_copy(const Pool &P, const Scratch &X, int from, int to, int held) {
  const int k = atomicAdd(&P.control->copies, 1);
  X.from[k] = from;
  X.to[k] = to;
  X.held[k] = held;
}

constexpr int kKeep = -2;   // stage: the page stays

// hb_pages_reserve: every entry's pages [old / 64, ceil(new / 64)) that are
// missing, or shared and about to be written, get the lowest free pages in
// entry order; the written part of a shared page is copied first.
__global__ void __launch_bounds__(kBookThreads) reserve_kernel(Pool P, Scratch X, const int *slots, const int *counts,
                                                               int n) {
  grid_begin();
  __shared__ int s_sums[32], s_bad;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    s_bad = 0;
    P.control->copies = 0;
  }
  __syncthreads();
  for (int b = warp; b < n; b += 32) {   // a warp an entry, lanes over its pages
    const int slot = slots[b], count = counts[b];
    int bad = 0, need = 0;
    if (slot < 0 || slot >= P.n_slots || count < 0) {
      bad = HB_PAGED_BAD_INDEX;
    } else {
      if (lane == 0 && atomicExch(&X.mark[slot], 1) != 0) bad = HB_PAGED_BAD_INDEX;   // twice in one call
      const int old = max(P.lengths[slot], 0);
      const int64_t len = static_cast<int64_t>(old) + count;
      if (len > static_cast<int64_t>(P.width) * kPage) {
        bad = HB_PAGED_BAD_INDEX;
      } else if (count > 0) {
        const int64_t row = static_cast<int64_t>(slot) * P.width;
        const int end = static_cast<int>((len + kPage - 1) / kPage);
        for (int i = old / kPage + lane; i < end; i += 32) {
          const int pg = page_of(P, slot, i);
          const bool take = pg < 0 || P.refs[pg] > 1;
          X.stage[row + i] = take ? pg : kKeep;   // the decision: counts change from the next phase on
          need += take ? 1 : 0;
        }
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) need += __shfl_xor_sync(0xffffffffu, need, o);
    if (lane == 0) X.need[b] = need;
    if (bad) atomicOr(&s_bad, bad);
  }
  __syncthreads();
  const int total = scan_needs(X.need, X.off, n, s_sums);
  if (s_bad == 0 && total > 0 && (total > P.n_pages || lowest_free(P.refs, P.n_pages, total, X.fresh, s_sums) < total)) {
    __syncthreads();
    if (threadIdx.x == 0) s_bad = HB_PAGED_EXHAUSTED;
  }
  for (int b = threadIdx.x; b < n; b += kBookThreads)
    if (slots[b] >= 0 && slots[b] < P.n_slots) X.mark[slots[b]] = 0;
  __syncthreads();
  if (s_bad) {   // all or nothing
    if (threadIdx.x == 0) {
      atomicOr(&P.control->status, s_bad);
      P.control->refused = 1;
    }
    return;
  }
  for (int b = warp; b < n; b += 32) {
    const int slot = slots[b], count = counts[b];
    if (count <= 0) continue;
    const int old = max(P.lengths[slot], 0), len = old + count;
    const int64_t row = static_cast<int64_t>(slot) * P.width;
    const int end = (len + kPage - 1) / kPage;
    int at = X.off[b];
    for (int i0 = old / kPage; i0 < end; i0 += 32) {
      const int i = i0 + lane;
      const int was = i < end ? X.stage[row + i] : kKeep;
      const unsigned mask = __ballot_sync(0xffffffffu, was != kKeep);
      if (was != kKeep) {
        const int fresh = X.fresh[at + __popc(mask & ((1u << lane) - 1u))];
        P.table[row + i] = fresh;
        P.refs[fresh] = 1;
        if (was >= 0) {
          atomicSub(&P.refs[was], 1);
          if (i == old / kPage && old % kPage != 0) push_copy(P, X, was, fresh, old % kPage);
        }
      }
      at += __popc(mask);
    }
    __syncwarp();
    if (lane == 0) P.lengths[slot] = len;
  }
}

// The rows of a call that fit, being made in shared memory.
constexpr int kStageInts = 8192;

// hb_pages_fork: dst[b] becomes the first counts[b] positions of src[b], all
// sources as they were before the call (so a permutation of slots, as a beam
// search's, is one call).  Whole pages are shared; the positions of a partial
// last page go to the lowest pages that were free before the call.
__global__ void __launch_bounds__(kBookThreads) fork_kernel(Pool P, Scratch X, const int *src, const int *dst,
                                                            const int *counts, int n) {
  grid_begin();
  __shared__ int s_sums[32], s_bad, s_stage[kStageInts];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    s_bad = 0;
    P.control->copies = 0;
  }
  // at most a page an entry: looked for while the entries are read
  const int free = lowest_free(P.refs, P.n_pages, n, X.fresh, s_sums);
  __syncthreads();
  for (int b = threadIdx.x; b < n; b += kBookThreads) {
    const int from = src[b], to = dst[b], count = counts[b];
    int need = 0;
    if (from < 0 || from >= P.n_slots || to < 0 || to >= P.n_slots || count < 0 || count > P.width * kPage) {
      atomicOr(&s_bad, HB_PAGED_BAD_INDEX);
    } else {
      const int length = P.lengths[from], page = page_of(P, from, count / kPage);
      if (atomicExch(&X.mark[to], 1) != 0 || count > length) atomicOr(&s_bad, HB_PAGED_BAD_INDEX);
      need = count % kPage != 0 && page >= 0 ? 1 : 0;
    }
    X.need[b] = need;
  }
  __syncthreads();
  const int total = scan_needs(X.need, X.off, n, s_sums);
  for (int b = threadIdx.x; b < n; b += kBookThreads)
    if (dst[b] >= 0 && dst[b] < P.n_slots) X.mark[dst[b]] = 0;
  if (s_bad || total > free) {   // all or nothing
    if (threadIdx.x == 0) {
      atomicOr(&P.control->status, s_bad ? s_bad : HB_PAGED_EXHAUSTED);
      P.control->refused = 1;
    }
    return;
  }
  __syncthreads();
  // the new rows beside the old ones, and the counts: what the sources share,
  // what the destinations give up (additions, so in any order)
  int *stage = static_cast<int64_t>(n) * P.width <= kStageInts ? s_stage : X.stage;
  for (int b = warp; b < n; b += 32) {
    const int from = src[b], to = dst[b], count = counts[b], whole = count / kPage, need = X.need[b];
    const int fresh = need ? X.fresh[X.off[b]] : -1;
    for (int i = lane; i < P.width; i += 32) {
      const int gone = page_of(P, to, i);
      int now = i <= whole ? page_of(P, from, i) : -1;
      if (i == whole) {
        if (need) push_copy(P, X, now, fresh, count % kPage);
        now = fresh;
      }
      stage[static_cast<int64_t>(b) * P.width + i] = now;
      if (now >= 0) atomicAdd(&P.refs[now], 1);
      if (gone >= 0) atomicSub(&P.refs[gone], 1);
    }
  }
  __syncthreads();
  for (int b = warp; b < n; b += 32) {
    const int64_t row = static_cast<int64_t>(dst[b]) * P.width;
    for (int i = lane; i < P.width; i += 32) P.table[row + i] = stage[static_cast<int64_t>(b) * P.width + i];
    if (lane == 0) P.lengths[dst[b]] = counts[b];
  }
}

// hb_pages_free: a warp a slot.  A slot named twice is freed once.
__global__ void __launch_bounds__(128) free_kernel(Pool P, const int *slots, int n) {
  grid_begin();
  const int b = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (b >= n) return;
  const int slot = slots[b];
  if (slot < 0 || slot >= P.n_slots) {
    if (lane == 0) atomicOr(&P.control->status, HB_PAGED_BAD_INDEX);
    return;
  }
  for (int i = lane; i < P.width; i += 32) {
    int *at = P.table + static_cast<int64_t>(slot) * P.width + i;
    if (*at < 0) continue;
    const int pg = atomicExch(at, -1);
    if (pg >= 0 && pg < P.n_pages) atomicSub(&P.refs[pg], 1);
  }
  if (lane == 0) P.lengths[slot] = 0;
}

// hb_pages_compact: of L live pages the k-th with an index of L or more goes
// to the k-th free index below L.  map[page] = its new index, -1 for a free one.
__global__ void __launch_bounds__(kBookThreads) compact_kernel(Pool P, Scratch X, int *map) {
  grid_begin();
  __shared__ int s_sums[32];
  int live = 0;
  for (int base = 0; base < P.n_pages; base += 4 * kBookThreads) {
    int n = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int p = base + k * kBookThreads + threadIdx.x;
      n += p < P.n_pages && P.refs[p] > 0 ? 1 : 0;
    }
    int sum;
    block_scan(n, s_sums, sum);
    live += sum;
  }
  int holes = 0, movers = 0;   // as many of one as of the other in the end
  for (int base = 0; base < P.n_pages; base += 4 * kBookThreads) {
    const int p = base + 4 * threadIdx.x;
    bool hole[4], mover[4];
    int nh = 0, nm = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool in = p + k < P.n_pages, held = in && P.refs[p + k] > 0;
      hole[k] = in && !held && p + k < live;
      mover[k] = held && p + k >= live;
      nh += hole[k] ? 1 : 0;
      nm += mover[k] ? 1 : 0;
      if (in) map[p + k] = held ? p + k : -1;
    }
    int sum_h, sum_m;
    int ah = holes + block_scan(nh, s_sums, sum_h), am = movers + block_scan(nm, s_sums, sum_m);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (hole[k]) X.to[ah++] = p + k;
      if (mover[k]) {
        X.from[am] = p + k;
        X.held[am++] = kPage;
      }
    }
    holes += sum_h;
    movers += sum_m;
  }
  __syncthreads();
  for (int k = threadIdx.x; k < movers; k += kBookThreads) {
    const int from = X.from[k], to = X.to[k];
    map[from] = to;
    P.refs[to] = P.refs[from];
    P.refs[from] = 0;
  }
  if (threadIdx.x == 0) P.control->copies = movers;
}

// The copy list's pages, and for a compaction the table's entries: a warp an
// 8 KB block of positions.  `copies` NULL: n copies.
__global__ void __launch_bounds__(256) copy_kernel(Pool P, uint8_t *to_pages, int to_n, const int *from, const int *to,
                                                   const int *held, const int *copies, int n, int blocks,
                                                   const int *map) {
  grid_begin();   // the copy list is complete
  if (map != nullptr) {
    const int64_t entries = static_cast<int64_t>(P.n_slots) * P.width;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < entries; i += gridDim.x * 256ll) {
      const int pg = P.table[i];
      if (pg >= 0 && pg < P.n_pages && map[pg] != pg) P.table[i] = map[pg];
    }
  }
  const int count = copies != nullptr ? *copies : n, lane = threadIdx.x & 31;
  const int64_t units = static_cast<int64_t>(count) * blocks;
  for (int64_t u = blockIdx.x * 8ll + (threadIdx.x >> 5); u < units; u += gridDim.x * 8ll) {
    const int k = static_cast<int>(u / blocks);
    const int64_t off = (u - static_cast<int64_t>(k) * blocks) * kBlockBytes;
    const int a = from[k], b = to[k], words = (held != nullptr ? held[k] : kPage) * 8;   // 16-byte words
    if (a < 0 || a >= P.n_pages || b < 0 || b >= to_n) {
      if (lane == 0) atomicOr(&P.control->status, HB_PAGED_BAD_INDEX);
      continue;
    }
    const uint4 *src = reinterpret_cast<const uint4 *>(P.pages + a * P.page_stride + off);
    uint4 *dst = reinterpret_cast<uint4 *>(to_pages + b * P.page_stride + off);
#pragma unroll
    for (int h = 0; h < 2; ++h) {   // eight loads in flight a lane
      uint4 v[8];
#pragma unroll
      for (int x = 0; x < 8; ++x)
        if (lane + 32 * (x + 8 * h) < words) v[x] = __ldcs(src + lane + 32 * (x + 8 * h));
#pragma unroll
      for (int x = 0; x < 8; ++x)
        if (lane + 32 * (x + 8 * h) < words) __stcs(dst + lane + 32 * (x + 8 * h), v[x]);
    }
  }
}

}  // namespace paged
}  // namespace hb
