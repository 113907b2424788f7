// hb_paged_tiles.cuh -- attention over a paged cache for chunks and prompts, on
// the 5th-generation tensor cores.
//
// o_i = sum_j softmax_j(scale q_i . k_j) v_j.  A tile is 256 packed rows (the q
// heads of a kv head's group times consecutive rows), as two halves of 128,
// the M of tcgen05.mma; a step is a block of 128 positions, two pages.  Per
// half and step: S = Q K^T (128 x 128 x D) into TMEM; one thread a row reads
// its 128 scores, keeps the running maximum and sum in FP32, and writes the
// weights exp2(c s - c m) back to TMEM as 16-bit; O += P V with P from TMEM.
// A page's K and V are operand tiles as they lie in the pool (128-byte
// swizzled rows; V is the MN-major B), fetched by plain bulk copies.
//
// What bounds it: with heads of 64 a step's 2 x 2.1 MFLOP take the tensor
// pipe 512 cycles a half, its 16,384 exponentials the 16-a-cycle special
// function units 1,024: the softmax is the bound, and the two halves take
// turns so that one's MMAs run under the other's exponentials (when first
// tried, 193 us without turns, 175 with).  With heads of 128 both take 1,024 cycles.  O is rescaled
// only when a row's maximum has grown by more than 2^8 (the sum and O share
// the stale maximum, so the result is the same), which after the first blocks
// is almost never.
//
// Measured, BF16, in replays of a CUDA graph: four prompts of 3000 to 4096
// positions, 14 q heads on 2 of 64: 164 us, 581 TFLOP/s, 2.0 times the
// exponentials' 83 us; a step of both halves takes 3,300 cycles, 2,050 of them the exponentials themselves, the
// rest scores on their way from the MMA, their maximum, and the hand-over of
// the turn.  Chunks of 200 to 512 rows of four prompts, 32 q heads on 8 of 128,
// window 1024: 55 us, 476 TFLOP/s; a multiprocessor has some 12 steps of 3,900
// cycles there (P lies over S, so a half's next S waits for its P V), and the
// start (7 us to the first scores) and the joins weigh as much as they do.
//
// Warps 0-3 and 4-7: the softmax of either half; warp 8: MMA issue; warp 9:
// K and V; warps 10 and 11: the halves' q, a tile ahead with heads of 64, with
// heads of 128 (one buffer) once the tile's last scores are issued.  One block a
// multiprocessor; the line of blocks is cut evenly (hb_paged.cuh), a tile cut
// by a border is joined by the last of its pieces to get to its end, which
// keeps its own part in TMEM (all parts through memory: chunks 65 us instead
// of 58, prompts 172 instead of 165).
//
// The weights are rounded once to the element type for the product with V, whose
// operands have one type; their sum is of what they were before, in FP32.  The
// output's error against 64 bits is 0.0020 to 0.0023 of its norm in BF16 and
// 0.00025 to 0.00028 in FP16, where its own rounding alone gives 0.0016 and
// 0.0002.  A low half beside the high one, as the rows kernel has it, would
// come to those, at half as many MMAs more, 128 subtractions and 64 conversions
// of pairs more a row and step in the softmax warps that bound the kernel, and
// with heads of 64 no TMEM is left for it (S 256 columns, O 128, P 128).
#pragma once

#include "hb_paged_rows.cuh"

namespace hb {
namespace paged {

constexpr int kTilesTile = 256, kTilesHalf = 128, kTilesBlock = 128;
// A tile's start and end, in blocks (0: whole prompts 190 us, chunks 58; 1:
// 164.7, 55; 2: 162, 54; 3: 166, 54).
constexpr int kTilesExtra = 2;
// Units a piece has at least: fewer pieces for small calls, whose joins would
// cost more than the blocks (2, 3 and 5 the same on calls that fill the GPU).
constexpr int kTilesLeast = 3;
// The quarter of its exponentials after which a half passes its turn on (1:
// 166.5 us, 2: 164.7, 3: 167.8).
constexpr int kTurnAt = 2;
constexpr int kTilesThreads = 384;
constexpr int kTilesPieces = 160;   // blocks of a launch at most

// Registers a thread after the split: 256 softmax threads x 216 + 128 others x
// 72 = 384 x 168, what the block is launched with.
constexpr int kTilesRegs = 216, kOtherRegs = 72;

template <int D>
struct TilesSize {
  static constexpr bool kEarly = D == 64;   // TMEM has room for P beside S: the next S starts before this P V
  static constexpr int kOperand = (D / 64) * 16384;              // 128 rows or positions
  static constexpr int kStages = D == 64 ? 8 : 4;
  static constexpr int kQ = D == 64 ? 2 : 1;                     // q buffers of either half
  static constexpr int kSmem = (2 * kQ + kStages) * kOperand + 1024;
  static constexpr uint32_t kS = 0, kO = 256, kP = D == 64 ? 384 : 0;   // TMEM columns; P of half h: + h * (64 or 128)
  static constexpr uint32_t kPHalf = D == 64 ? 64 : 128;
  static constexpr int kPartFloats = kTilesHalf * (D + 2);
};

// ---- PTX -------------------------------------------------------------------------------
__device__ __forceinline__ void t_alloc(uint32_t *dst, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst)), "r"(ncols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void t_dealloc(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
__device__ __forceinline__ void t_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void t_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// The MMA warp's instructions are issued by one lane (`leader` nonzero in
// one) as predicated instructions in code that all lanes run: their operands
// live in uniform registers, and a branch of one lane would have each of them
// moved there anew (eight MMAs took 650 cycles to issue).
__device__ __forceinline__ uint32_t t_leader() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r;
}
__device__ __forceinline__ void t_commit(uint32_t bar, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
      ::"r"(bar), "r"(leader) : "memory");
}
// D[tmem] (+)= A[smem] B[smem], and A[tmem] B[smem]
__device__ __forceinline__ void t_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc,
                                         uint32_t leader) {
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
               "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
               ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(leader) : "memory");
}
__device__ __forceinline__ void t_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc,
                                         uint32_t leader) {
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
               "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
               ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(leader) : "memory");
}
// 32 consecutive 32-bit columns of this thread's TMEM lane.
__device__ __forceinline__ void t_ld32(uint32_t taddr, float *r) {
  uint32_t *u = reinterpret_cast<uint32_t *>(r);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
        "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]),
        "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]),
        "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
      : "r"(taddr));
}
__device__ __forceinline__ void t_st32(uint32_t taddr, const uint32_t *u) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
      ::"r"(taddr), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]),
        "r"(u[8]), "r"(u[9]), "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15]), "r"(u[16]),
        "r"(u[17]), "r"(u[18]), "r"(u[19]), "r"(u[20]), "r"(u[21]), "r"(u[22]), "r"(u[23]), "r"(u[24]), "r"(u[25]),
        "r"(u[26]), "r"(u[27]), "r"(u[28]), "r"(u[29]), "r"(u[30]), "r"(u[31])
      : "memory");
}
__device__ __forceinline__ void t_st16(uint32_t taddr, const uint32_t *u) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      ::"r"(taddr), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]),
        "r"(u[8]), "r"(u[9]), "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15])
      : "memory");
}
// This thread's TMEM loads are done; names 32 registers that they fill, so
// that nothing reads those before.
__device__ __forceinline__ void t_ld_wait(float *r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
      : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]),
        "+f"(r[8]), "+f"(r[9]), "+f"(r[10]), "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]), "+f"(r[15]),
        "+f"(r[16]), "+f"(r[17]), "+f"(r[18]), "+f"(r[19]), "+f"(r[20]), "+f"(r[21]), "+f"(r[22]), "+f"(r[23]),
        "+f"(r[24]), "+f"(r[25]), "+f"(r[26]), "+f"(r[27]), "+f"(r[28]), "+f"(r[29]), "+f"(r[30]), "+f"(r[31])
      ::"memory");
}
__device__ __forceinline__ void t_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Two FP32 operations an instruction.
__device__ __forceinline__ uint64_t f2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void f2_split(uint64_t v, float &a, float &b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float log2_approx(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 32 bytes at a 32-byte-aligned address.
__device__ __forceinline__ void store32(void *p, const uint32_t *u) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(u[0]), "r"(u[1]), "r"(u[2]),
               "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]) : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// A 128-byte-swizzled shared-memory operand (rows of 128 bytes, groups of
// eight rows 1 KB apart) as the low word of its descriptor, to which 16-byte
// steps are added; `lead`: bytes between the 64-column parts of an MN-major
// operand (a K-major one is addressed part by part).
__device__ __forceinline__ uint32_t swizzled_lo(uint32_t saddr, uint32_t lead) {
  return (saddr >> 4) | ((lead >> 4) << 16);
}
__device__ __forceinline__ uint64_t swizzled_desc(uint32_t lo) {
  constexpr uint32_t kHi = (1024 >> 4) | (1u << 14) | (2u << 29);   // 8-row step, version, 128-byte swizzle
  return static_cast<uint64_t>(kHi) << 32 | lo;
}
// kind::f16, FP32 accumulator, M = 128, N = n; `mn`: B is MN-major.
template <class T>
__host__ __device__ constexpr uint32_t tiles_idesc(int n, bool mn) {
  return (1u << 4) | (std::is_same<T, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u) | (mn ? 1u << 16 : 0u) |
         (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(128 >> 4) << 24);
}

// mbar_wait without a call: the softmax threads wait with a row of scores in
// registers, which a call would move to memory.
__device__ __forceinline__ bool t_wait(uint64_t *bar, uint32_t parity, Ctrl *ctrl, uint64_t limit_ns, int where) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t start = globaltimer_ns();
  while (!mbar_try_wait_suspend(bar, parity, 20000u)) {
    if (ld_volatile_int(&ctrl->abort)) return false;
    if (globaltimer_ns() - start > limit_ns) {
      if (atomicCAS(&ctrl->err, 0, kErrTimeout) == 0) atomicExch(&ctrl->err_where, where);
      atomicExch(&ctrl->abort, 1);
      return false;
    }
  }
  return true;
}

// A tile as the q warps tell it to the MMA and softmax warps.
struct TileInfo {
  int count;             // blocks; 0: there are no more tiles
  int first;             // first block
  int base, packed;      // the half's first packed row; the entry's rows
  int row0, n, length, slot, head;
  int two;               // both halves have rows
  int whole, opens;      // the piece has all its blocks; the first of them
  int hole;              // a page of the blocks is missing
  int c0, c1;            // not whole: the pieces that share it
};
// A slot is written again four tiles later, when the q buffers' barriers say
// that the softmax is past its tile.
constexpr int kInfoSlots = 4;

struct TilesBars {
  uint64_t full[8], empty[8];                              // the ring of K and V blocks
  uint64_t q_full[2][2], q_empty[2][2];                    // [half][buffer]
  uint64_t s_full[2], s_read[2], p_full[2], o_done[2];
  uint64_t i_full[2][kInfoSlots];                          // a tile is told: what the softmax, which MMAs of
                                                           // short tiles may run ahead of, waits for
  uint64_t turn[2][4];                                     // the exponentials are free for a half's warp
  uint64_t half[2];                                        // a half's four softmax warps
  uint64_t done;
};

template <int D, class T>
__global__ void __launch_bounds__(kTilesThreads, 1) paged_tiles_kernel(const __grid_constant__ Attend A, int least) {
  using E = Elem<T>;
  using Z = TilesSize<D>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ TilesBars bars;
  __shared__ uint32_t s_tmem;
  __shared__ TileInfo s_info[2][kInfoSlots];
  __shared__ int s_last[2], s_seen[2];
  __shared__ unsigned s_done[8];
  uint8_t *smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint8_t *ring = smem + 2 * Z::kQ * Z::kOperand;   // behind the q of either half, kQ tiles
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Shape S = A.shape;
  const Line line = line_at(smem + (2 * Z::kQ + Z::kStages) * Z::kOperand, A.batch.entries);
  Ctrl *ctrl = &A.pool.control->ctrl;

  if (threadIdx.x == 0) {
    for (int i = 0; i < Z::kStages; ++i) {
      mbar_init(&bars.full[i], 1);
      mbar_init(&bars.empty[i], 1);
    }
    for (int h = 0; h < 2; ++h) {
      for (int x = 0; x < 2; ++x) {
        mbar_init(&bars.q_full[h][x], 1);
        mbar_init(&bars.q_empty[h][x], 1);
      }
      mbar_init(&bars.s_full[h], 1);
      mbar_init(&bars.s_read[h], 4);
      mbar_init(&bars.p_full[h], 4);
      mbar_init(&bars.o_done[h], 1);
      mbar_init(&bars.half[h], 4);
      for (int x = 0; x < 4; ++x) mbar_init(&bars.turn[h][x], 1);
      for (int x = 0; x < kInfoSlots; ++x) mbar_init(&bars.i_full[h][x], 1);
    }
    mbar_init(&bars.done, 1);
    fence_mbar_init();
  }
  if (A.beside) second_begin(A.pool.control, s_seen); else grid_begin();
  const bool ascends = fill_line(A.pool, A.batch, S, line, [&](const Entry &e) { return e.n * S.group > A.few; });
  if (A.few == 0) {   // else the rows kernel does these
    if (ascends) rows_of_no_entry<D>(A, line); else rows_unseen<D>(A, 0, 0);
  }
  const Cut cut(ascends ? line.prefix[A.batch.entries] : 0, gridDim.x, least);
  if (static_cast<int>(blockIdx.x) >= cut.pieces) {
    grid_end();
    return;
  }
  if (warp == 0) t_alloc(&s_tmem, 512);
  t_before();
  __syncthreads();
  t_after();
  // 512 columns are all of them: the allocation starts at column 0

  Walk w;
  w.u = cut.begin(blockIdx.x);
  w.end = cut.begin(blockIdx.x + 1);
  bool more = w.start(A.pool, A.batch, S, line);
  auto halves = [&]() { return w.e.n * S.group - w.t * kTilesTile > kTilesHalf ? 2 : 1; };

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == 9) {
      // ---- loads: K(0), then K(j + 1), V(j), the order the MMAs use them in
      int it = 0;
      bool ok = true;
      auto load = [&](bool is_v, int block, int pg0, int pg1) {
        const int s = it % Z::kStages;
        const uint32_t ph = static_cast<uint32_t>(it / Z::kStages) & 1u;
        ok = __all_sync(0xffffffffu, mbar_wait(&bars.empty[s], ph ^ 1u, ctrl, A.limit_ns, kWhereEmpty)) != 0;
        if (!ok) return;
        uint8_t *dst = ring + s * Z::kOperand;
        int held[2];
        uint32_t bytes = 0;
        bool wrote = false;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          held[x] = (x ? pg1 : pg0) < 0 ? 0 : max(0, min(kPage, w.e.length - (2 * block + x) * kPage));
          bytes += (D / 64) * held[x] * 128;
          if (is_v && held[x] < kPage) {   // V where there is no position: zero, so that weight zero times it is zero
            for (int h = 0; h < D / 64; ++h)
              for (int y = held[x] * 128 + lane * 16; y < kBlockBytes; y += 512)
                *reinterpret_cast<uint4 *>(dst + h * 16384 + x * kBlockBytes + y) = make_uint4(0, 0, 0, 0);
            wrote = true;
          }
        }
        if (wrote) {
          fence_proxy_async_smem();
          __syncwarp();
        }
        if (lane == 0) {
          if (bytes) mbar_arrive_expect_tx(&bars.full[s], bytes); else mbar_arrive_count(&bars.full[s], 1);
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            if (!held[x]) continue;
            const uint8_t *src = kv_block(A, x ? pg1 : pg0, w.head) + (is_v ? D / 64 * kBlockBytes : 0);
            for (int h = 0; h < D / 64; ++h)
              bulk_g2s(dst + h * 16384 + x * kBlockBytes, src + h * kBlockBytes, held[x] * 128, &bars.full[s]);
          }
        }
        __syncwarp();
        ++it;
      };
      for (; more && ok; more = w.next(A.pool, A.batch, S, line)) {
        const int first = w.first(), count = w.count(S);
        int mine = -1, k0 = -1, k1 = -1, v0 = -1, v1 = -1;
        // K(0), then K(j), V(j - 1) in turn, at last V(count - 1).  One place for
        // all loads: the warps' loops share the instruction cache.
#pragma unroll 1
        for (int x = 0; x < 2 * count && ok; ++x) {
          const bool last = x == 2 * count - 1, is_v = last || (x != 0 && (x & 1) == 0);
          int block = last ? count - 1 : (x >> 1) - 1, p0 = last ? k0 : v0, p1 = last ? k1 : v1;
          if (!is_v) {
            block = (x + 1) >> 1;
            if ((block & 15) == 0) mine = page_of<true>(A.pool, w.e.slot, 2 * (first + block) + lane);
            v0 = k0;
            v1 = k1;
            p0 = k0 = __shfl_sync(0xffffffffu, mine, 2 * (block & 15));
            p1 = k1 = __shfl_sync(0xffffffffu, mine, 2 * (block & 15) + 1);
          }
          load(is_v, first + block, p0, p1);
        }
      }
      for (int i = max(0, it - Z::kStages); i < it; ++i)   // nothing in flight when the block ends
        mbar_wait_quiet(&bars.full[i % Z::kStages], static_cast<uint32_t>(i / Z::kStages) & 1u, A.limit_ns);
    } else if (warp == 8) {
      // ---- MMA issue
      constexpr uint32_t kIdescS = tiles_idesc<T>(kTilesBlock, false), kIdescO = tiles_idesc<T>(D, true);
      constexpr uint32_t kStep = Z::kOperand >> 4;
      const uint32_t leader = t_leader();
      const uint32_t q_lo = swizzled_lo(smem_u32(smem), 16), k_lo = swizzled_lo(smem_u32(ring), 16),
                     v_lo = swizzled_lo(smem_u32(ring), 16384);
      uint32_t it = 0;                // ring stages consumed
      uint32_t n_q0 = 0, n_q1 = 0, n_s[2] = {0, 0};   // tiles and steps of either half so far
      bool ok = true;
      auto wait = [&](uint64_t *bar, uint32_t phase) {
        ok = __all_sync(0xffffffffu, ok && t_wait(bar, phase & 1u, ctrl, A.limit_ns, kWhereFull)) != 0;
        return ok;
      };
      auto stage = [&](uint32_t i) { return i % Z::kStages; };
      auto wait_ring = [&](uint32_t i) { return wait(&bars.full[stage(i)], i / Z::kStages); };
      auto commit = [&](uint64_t *bar) { t_commit(smem_u32(bar), leader); };
      // S of half h from its q buffer and the K in ring use i
      auto mma_s = [&](int h, uint32_t buf, uint32_t i) {
        t_after();
        const uint32_t a = q_lo + (buf * 2 + h) * kStep, b = k_lo + stage(i) * kStep;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t off = ((k >> 2) * 16384 + (k & 3) * 32) >> 4;
          t_mma_ss(Z::kS + h * 128, swizzled_desc(a + off), swizzled_desc(b + off), kIdescS, k != 0, leader);
        }
        commit(&bars.s_full[h]);
      };
      // O of half h from its P and the V in ring use i
      auto mma_o = [&](int h, uint32_t i, uint32_t acc) {
        t_after();
        const uint32_t b = v_lo + stage(i) * kStep;
#pragma unroll
        for (int k = 0; k < kTilesBlock / 16; ++k)
          t_mma_ts(Z::kO + h * D, Z::kP + h * Z::kPHalf + k * 8, swizzled_desc(b + k * (2048 >> 4)), kIdescO, k ? 1 : acc,
                   leader);
        commit(&bars.o_done[h]);
      };
      while (ok) {
        const uint32_t buf0 = n_q0 % Z::kQ;
        if (!wait(&bars.q_full[0][buf0], n_q0 / Z::kQ)) break;
        const TileInfo &info = s_info[0][n_q0 % kInfoSlots];
        // reductions over the warp, for results in uniform registers
        const uint32_t count = __reduce_max_sync(0xffffffffu, static_cast<unsigned>(info.count));
        const bool two = __reduce_max_sync(0xffffffffu, static_cast<unsigned>(info.two)) != 0;
        if (count == 0) break;
        // S is free: the last step's P of either half, which was waited for,
        // was written after its S was read
        ++n_q0;
        const uint32_t buf1 = n_q1 % Z::kQ;
        if (two) {
          wait(&bars.q_full[1][buf1], n_q1 / Z::kQ);
          ++n_q1;
        }
        // steps -1 (the first S alone), 0 .. count - 1: the next step's S, this
        // one's O; one place for either, the warps' loops share the instruction cache
#pragma unroll 1
        for (int j = -1; ok && j < static_cast<int>(count); ++j) {
          const bool next = j + 1 < static_cast<int>(count);
          const uint32_t ik = it + (j < 0 ? 0 : 2 * j + 1), iv = next ? ik + 1 : ik;
          if (!next) {   // every S of the tile is issued
            commit(&bars.q_empty[0][buf0]);
            if (two) commit(&bars.q_empty[1][buf1]);
          }
          if (next && !wait_ring(ik)) break;
          if (Z::kEarly && next) {
#pragma unroll 1
            for (int h = 0; h < (two ? 2 : 1); ++h)
              if (j < 0 || wait(&bars.s_read[h], n_s[h])) mma_s(h, h ? buf1 : buf0, ik);
            commit(&bars.empty[stage(ik)]);
          }
          if (j >= 0 && !wait_ring(iv)) break;
#pragma unroll 1
          for (int h = 0; h < (two ? 2 : 1); ++h) {
            if (j >= 0 && wait(&bars.p_full[h], n_s[h]++)) mma_o(h, iv, j != 0);
            if (!Z::kEarly && next && ok) mma_s(h, h ? buf1 : buf0, ik);   // over the P just used: MMAs run in order
          }
          if (!Z::kEarly && next) commit(&bars.empty[stage(ik)]);
          if (j >= 0) commit(&bars.empty[stage(iv)]);
        }
        it += 2 * count;
      }
      commit(&bars.done);   // after a give-up too: nothing in flight when TMEM is freed
    } else {
      // ---- warps 10, 11: the q rows of half h, a tile ahead of its softmax
      const int h = warp - 10;
      uint32_t n = 0;
      bool ok = true;
      while (ok) {
        while (more && h >= halves()) more = w.next(A.pool, A.batch, S, line);
        const int buf = n % Z::kQ;
        ok = __all_sync(0xffffffffu, n < Z::kQ || mbar_wait(&bars.q_empty[h][buf], (n / Z::kQ - 1) & 1u, ctrl, A.limit_ns,
                                                            kWhereEmpty)) != 0;
        TileInfo &info = s_info[h][n % kInfoSlots];
        if (!more || !ok) {
          if (lane == 0) {
            info.count = 0;
            mbar_arrive_count(&bars.q_full[h][buf], 1);
            mbar_arrive_count(&bars.i_full[h][n % kInfoSlots], 1);
          }
          break;
        }
        const int packed = w.e.n * S.group, base = w.t * kTilesTile + h * kTilesHalf;
        uint8_t *dst = smem + (buf * 2 + h) * Z::kOperand;
        // two lanes a row, 16 bytes of it each a step: a warp alone pays for every
        // instruction, and a row is found once (a lane a row reads half sectors:
        // prompts 169 us; four lanes a row 167; two 165)
        constexpr int kLanes = 2, kRows = 32 / kLanes;
        const int part = lane % kLanes;
#pragma unroll 1
        for (int x = 0; x < kTilesHalf; x += kRows) {
          const int r = x + lane / kLanes, row = base + r, i = S.row_of(row), g = row - i * S.group;
          const bool there = row < packed;   // else no bytes are read and zeros written
          const uint16_t *from = static_cast<const uint16_t *>(A.q) + part * 8 +
                                 (there ? (w.e.row0 + i) * A.q_row + (w.head * S.group + g) * A.q_head : 0);
          uint8_t *to = dst + r * 128;
          const int at = (part ^ (r & 7)) << 4;
          if (A.q_vec) {
#pragma unroll
            for (int c = 0; c < D / 8; c += kLanes)
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                               smem_u32(to) + ((c >> 3) * 16384 + (at ^ (c & 7) << 4))),
                           "l"(from + c * 8), "r"(there ? 16 : 0)
                           : "memory");
          } else {
#pragma unroll 1
            for (int c = 0; c < D / 8; c += kLanes)
              *reinterpret_cast<uint4 *>(to + (c >> 3) * 16384 + (at ^ (c & 7) << 4)) =
                  there ? load8<false>(from + c * 8) : make_uint4(0, 0, 0, 0);
          }
        }
        cp_async_commit();
        const int first = w.first(), count = w.count(S);
        bool hole = false;   // whether a page of the piece's blocks is missing
        for (int p = 2 * first + lane; p < 2 * (first + count); p += 32)
          hole |= p * kPage < w.e.length && page_of<true>(A.pool, w.e.slot, p) < 0;
        hole = __any_sync(0xffffffffu, hole) != 0;
        if (lane == 0) {
          info.count = count;
          info.first = first;
          info.base = base;
          info.packed = packed;
          info.row0 = w.e.row0;
          info.n = w.e.n;
          info.length = w.e.length;
          info.slot = w.e.slot;
          info.head = w.head;
          info.two = halves() == 2;
          info.whole = w.whole();
          info.opens = w.opens();
          info.hole = hole;
          if (!w.whole()) {
            info.c0 = cut.of(w.tile_u + S.extra);
            info.c1 = cut.of(w.tile_u + w.units - 1);
          }
        }
        cp_async_wait_all();
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive_count(&bars.q_full[h][buf], 1);
          mbar_arrive_count(&bars.i_full[h][n % kInfoSlots], 1);
        }
        ++n;
        more = w.next(A.pool, A.batch, S, line);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kTilesRegs));
    // ---- softmax of half h, a thread a row
    const int h = warp >> 2, r = threadIdx.x & 127;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t t_s = Z::kS + h * 128 + lanes, t_o = Z::kO + h * D + lanes,
                   t_p = Z::kP + h * Z::kPHalf + lanes;
    const float c = A.scale_log2;
    uint32_t steps = 0, n_tiles = 0;   // of this half so far
    uint32_t turns = 0;                // steps of tiles with two halves
    bool ok = true;
    unsigned &done = s_done[warp];     // of rows_again; bit 2: there is a row to look at.  Not in a register
    if (lane == 0) done = 0;
    auto wait = [&](uint64_t *bar, uint32_t phase) {
      ok = __all_sync(0xffffffffu, ok && t_wait(bar, phase & 1u, ctrl, A.limit_ns, kWhereFull)) != 0;
      return ok;
    };
    uint32_t n_syncs = 0;
    auto half_sync = [&]() {   // with a limit, as every wait here
      __syncwarp();
      if (lane == 0) mbar_arrive_count(&bars.half[h], 1);
      return wait(&bars.half[h], n_syncs++);
    };
    while (true) {
      if (!wait(&bars.i_full[h][n_tiles % kInfoSlots], n_tiles / kInfoSlots)) break;
      const TileInfo &info = s_info[h][n_tiles % kInfoSlots];
      const int first = info.first, count = info.count;
      if (count == 0) break;
      ++n_tiles;
      const bool two = info.two != 0;
      const int row = info.base + r, i = S.row_of(row), before = info.length - info.n;   // positions before the rows
      const bool in = row < info.packed, hole = info.hole != 0;
      const int pos = in ? before + i : -1;
      // positions that every row of the half sees need no mask
      const int all_hi = before + S.row_of(info.base);
      const int all_lo = S.first_seen(before + S.row_of(min(info.packed, info.base + kTilesHalf) - 1));

      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < count; ++j, ++steps) {
        if (!wait(&bars.s_full[h], steps)) break;
        t_after();
        float s[128];
#pragma unroll
        for (int x = 0; x < 4; ++x) t_ld32(t_s + x * 32, s + x * 32);
#pragma unroll
        for (int x = 0; x < 4; ++x) t_ld_wait(s + x * 32);
        if constexpr (Z::kEarly) {
          t_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_count(&bars.s_read[h], 1);
        }
        const int j0 = (first + j) * kTilesBlock;
        if (hole || j0 + kTilesBlock - 1 > all_hi || j0 < all_lo) {
          // sees lo < x <= hi: a bit a position, which predicates are made from
          // eight at a time (comparisons took twice the instructions)
          const int hi = pos - j0, lo = S.first_seen(pos) - 1 - j0;
          bool gone[2] = {false, false};
          if (hole) {
            gone[0] = page_of<true>(A.pool, info.slot, 2 * (first + j)) < 0;
            gone[1] = page_of<true>(A.pool, info.slot, 2 * (first + j) + 1) < 0;
          }
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int top = hi - 32 * x, under = lo - 32 * x;
            uint32_t sees = top >= 31 ? ~0u : top < 0 ? 0u : (2u << top) - 1u;
            if (under >= 0) sees &= under >= 31 ? 0u : ~1u << under;
            if (gone[x >> 1]) sees = 0;
#pragma unroll
            for (int y = 0; y < 32; ++y)
              if (!(sees >> y & 1u)) s[32 * x + y] = -INFINITY;
          }
        }
        float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int x = 4; x < 124; x += 8) {
#pragma unroll
          for (int y = 0; y < 4; ++y) mx[y] = max3(mx[y], s[x + y], s[x + 4 + y]);
        }
        const float top = max3(max3(mx[0], s[124], s[125]), max3(mx[1], s[126], s[127]), fmaxf(mx[2], mx[3]));
        if (__any_sync(0xffffffffu, (top - m) * c > 8.f)) {   // also from m = -inf; both -inf: NaN, no
          const float nm = fmaxf(m, top), a = nm == -INFINITY ? 1.f : exp2_approx((m - nm) * c);
          m = nm;
          l *= a;
          if (j > 0) {
            if (!wait(&bars.o_done[h], steps - 1)) break;
            t_after();
#pragma unroll
            for (int x = 0; x < D / 32; ++x) {
              float o[32];
              t_ld32(t_o + x * 32, o);
              t_ld_wait(o);
#pragma unroll
              for (int y = 0; y < 32; ++y) o[y] *= a;
              t_st32(t_o + x * 32, reinterpret_cast<const uint32_t *>(o));
            }
          }
        }
        if constexpr (Z::kEarly) {   // P is free when the last step's P V has read it
          if (j > 0 && !wait(&bars.o_done[h], steps - 1)) break;
        }
        // The halves take turns at the exponentials: left alone they run them at
        // the same time, at half speed each, and then both wait at the same time.
        if (two && !wait(&bars.turn[h][warp & 3], turns - (h == 0 ? 1 : 0))) break;
        const float mc = m == -INFINITY ? 0.f : m * c;
        const uint64_t c2 = f2(c, c), mc2 = f2(-mc, -mc);
        uint64_t sum[4] = {0, 0, 0, 0};
#pragma unroll
        for (int x = 0; x < 4; ++x) {   // 32 at a time; the stores hold their order
          uint32_t p[16];
#pragma unroll
          for (int y = 0; y < 16; ++y) {
            float a, b;
            f2_split(f2_fma(f2(s[x * 32 + 2 * y], s[x * 32 + 2 * y + 1]), c2, mc2), a, b);
            a = exp2_approx(a);
            b = exp2_approx(b);
            sum[y & 3] = f2_add(sum[y & 3], f2(a, b));
            p[y] = E::pack(a, b);
          }
          t_st16(t_p + x * 16, p);
          if (x == kTurnAt && two && lane == 0) mbar_arrive_count(&bars.turn[h ^ 1][warp & 3], 1);
        }
        turns += two ? 1 : 0;
        float l0, l1;
        f2_split(f2_add(f2_add(sum[0], sum[1]), f2_add(sum[2], sum[3])), l0, l1);
        l += l0 + l1;
        t_st_wait();
        t_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_count(&bars.p_full[h], 1);
      }
      if (!wait(&bars.o_done[h], steps - 1)) break;   // or a wait above gave up: the control block says which
      t_after();
      const bool whole = info.whole != 0;
      constexpr int64_t kTwo = 2 * Z::kPartFloats;   // a part has two halves
      int c0 = 0, c1 = -1, own = 0;
      float own_m = 0.f;   // before the parts are joined
      if (!whole) {
        // A tile that other pieces share.  All but the last of them to get here
        // leave their parts ([D / 4][128] of 4 floats) and say so; that one
        // waits for the parts and joins them with its own, which stays in TMEM,
        // in the pieces' order.
        c0 = info.c0;
        c1 = info.c1;
        own = blockIdx.x;
        int *arrived = A.arrived + 2 * c0 + h, *left = arrived + 2 * kTilesPieces;
        if (r == 0) s_last[h] = atomicAdd(arrived, 1) == c1 - c0;
        if (!half_sync()) break;
        if (s_last[h] == 0) {
          float *part = A.parts + (static_cast<int64_t>(own) * 2 + (info.opens ? 1 : 0)) * kTwo + h * Z::kPartFloats;
#pragma unroll
          for (int x = 0; x < D / 32; ++x) {
            float o[32];
            t_ld32(t_o + x * 32, o);
            t_ld_wait(o);
#pragma unroll
            for (int y = 0; y < 8; ++y)
              __stcg(reinterpret_cast<float4 *>(part) + (x * 8 + y) * 128 + r,
                     make_float4(o[4 * y], o[4 * y + 1], o[4 * y + 2], o[4 * y + 3]));
          }
          __stcg(part + 128 * D + r, m);
          __stcg(part + 128 * (D + 1) + r, l);
          if (!half_sync()) break;   // the half's part is written
          if (r == 0) arrive_acq_rel(left);
          t_before();   // as below
          continue;
        }
        if (r == 0) {
          const uint64_t start = globaltimer_ns();
          bool seen = true;
          while (seen && load_acquire(left) < c1 - c0) {   // they are being written
            if (ld_volatile_int(&ctrl->abort)) {
              seen = false;
            } else if (globaltimer_ns() - start > A.limit_ns) {
              if (atomicCAS(&ctrl->err, 0, kErrTimeout) == 0) atomicExch(&ctrl->err_where, kWhereFull);
              atomicExch(&ctrl->abort, 1);
              seen = false;
            }
          }
          if (seen) {
            *arrived = 0;
            *left = 0;
          }
          s_seen[h] = seen;
        }
        if (!half_sync()) break;
        ok = s_seen[h] != 0;
        if (!ok) break;
        if (lane == 0) done |= info.opens ? 2u : 1u;
        const float *p = A.parts + h * Z::kPartFloats + 128 * D + r;
        const float om = m, ol = l;
        m = -INFINITY;
        l = 0.f;
#pragma unroll 4
        for (int k = c0; k <= c1; ++k) {
          const float *pk = p + (k * 2 + (k == c0 ? 1 : 0)) * kTwo;
          const float pm = k == own ? om : __ldcg(pk), pl = k == own ? ol : __ldcg(pk + 128);
          const float nm = fmaxf(m, pm), use = nm == -INFINITY ? 0.f : nm;
          l = l * exp2_approx((m - use) * c) + pl * exp2_approx((pm - use) * c);
          m = nm;
        }
        own_m = om;
      }
      const int g = row - i * S.group, qh = info.head * S.group + g;
      const int64_t orow = info.row0 + i;
      if (in && A.lse != nullptr)
        A.lse[orow * A.q_heads + qh] = l == 0.f ? -INFINITY : fmaf(m, A.scale, log2_approx(l) * 0.6931471805599453f);
      const float inv = l == 0.f ? 0.f : 1.f / l;
      T *out = static_cast<T *>(A.out) + orow * A.o_row + qh * A.o_head;
      uint64_t wrong = 0;   // NaN as soon as a value is not finite
#pragma unroll
      for (int x = 0; x < D / 64; ++x) {   // 64 dims at a time
        float o[64];
        if (whole) {
          t_ld32(t_o + x * 64, o);
          t_ld32(t_o + x * 64 + 32, o + 32);
          t_ld_wait(o);
          t_ld_wait(o + 32);
        } else {
          const float *p = A.parts + h * Z::kPartFloats;
          const float use = m == -INFINITY ? 0.f : m;
#pragma unroll
          for (int y = 0; y < 64; ++y) o[y] = 0.f;
          // parts [c0, own), this one, the others
#pragma unroll 1
          for (int side = 0; side < 2; ++side) {
            if (side == 1) {
              const float f = exp2_approx((own_m - use) * c);
#pragma unroll
              for (int z = 0; z < 64; z += 32) {
                float v[32];
                t_ld32(t_o + x * 64 + z, v);
                t_ld_wait(v);
#pragma unroll
                for (int y = 0; y < 32; ++y) o[z + y] = fmaf(v[y], f, o[z + y]);
              }
            }
#pragma unroll 2
            for (int k = side ? own + 1 : c0; k < (side ? c1 + 1 : own); ++k) {
              const float *pk = p + (k * 2 + (k == c0 ? 1 : 0)) * kTwo;
              const float f = exp2_approx((__ldcg(pk + 128 * D + r) - use) * c);
              float4 v[16];
#pragma unroll
              for (int y = 0; y < 16; ++y) v[y] = __ldcg(reinterpret_cast<const float4 *>(pk) + (x * 16 + y) * 128 + r);
#pragma unroll
              for (int y = 0; y < 16; ++y) {
                o[4 * y] = fmaf(v[y].x, f, o[4 * y]);
                o[4 * y + 1] = fmaf(v[y].y, f, o[4 * y + 1]);
                o[4 * y + 2] = fmaf(v[y].z, f, o[4 * y + 2]);
                o[4 * y + 3] = fmaf(v[y].w, f, o[4 * y + 3]);
              }
            }
          }
        }
        if (in) {
          uint32_t u[32];
#pragma unroll
          for (int y = 0; y < 32; ++y) {
            const uint64_t v = f2_mul(f2(o[2 * y], o[2 * y + 1]), f2(inv, inv));
            wrong = f2_fma(v, 0, wrong);
            float a, b;
            f2_split(v, a, b);
            u[y] = E::pack(a, b);
          }
          uint16_t *dst = reinterpret_cast<uint16_t *>(out) + x * 64;
          if (A.o_wide) {
#pragma unroll
            for (int y = 0; y < 4; ++y) store32(dst + y * 16, u + y * 8);
          } else {
#pragma unroll
            for (int y = 0; y < 8; ++y) {
              const uint4 v = make_uint4(u[4 * y], u[4 * y + 1], u[4 * y + 2], u[4 * y + 3]);
              if (A.o_vec) store8<true>(dst + y * 8, v); else store8<false>(dst + y * 8, v);
            }
          }
        }
      }
      t_before();   // this half's O is read: its next p arrival says so
      float w0, w1;
      f2_split(wrong, w0, w1);
      if (__any_sync(0xffffffffu, w0 + w1 != 0.f && l <= 3.4e38f) && lane == 0) done |= 4u;
    }
  }
  __syncwarp();
  // every MMA has completed before TMEM is freed
  mbar_wait_quiet(&bars.done, 0, A.limit_ns);
  t_before();
  __syncthreads();
  t_after();
  if (warp == 0) t_dealloc(s_tmem, 512);
  // here, not in the softmax branch: a call there costs its loops registers (whole prompts 170 us instead of 165)
  if (warp < 8 && s_done[warp] & 4u)
    rows_again<D, T>(A, line_at(smem + (2 * Z::kQ + Z::kStages) * Z::kOperand, A.batch.entries), least, warp * 32, 32,
                     s_done[warp]);
  grid_end();
}

}  // namespace paged
}  // namespace hb
