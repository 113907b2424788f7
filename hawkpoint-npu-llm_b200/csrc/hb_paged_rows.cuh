// hb_paged_rows.cuh -- attention over a paged cache for few rows per kv head:
// decoded tokens and short chunks.
//
// o_i = sum_j softmax_j(scale q_i . k_j) v_j over the positions j that row i
// sees.  With a row or a few per sequence every K and V byte is used for at
// most 16 rows, 16 FLOP a byte and less, far below the ~250 of this GPU: HBM
// bounds it, so the kernel is a stream of pages.  A tile is 16 packed rows
// (the MMA's M: the q heads that share a kv head read its pages once), a
// stage is one page of one kv head, K and V, which the pool's layout makes
// one bulk copy.  A producer warp keeps the ring of stages full; four
// consumer warps take 16 positions of each page each (mma.sync m16n8k16: a
// tcgen05 tile would be 128 rows for 16), with a running maximum and sum of
// their own that are joined once a tile.  The weights are multiplied as a
// high and a low half, to 16 bits in BF16 and 22 in FP16 (there down to 2^-25 of a
// warp's largest, where the low half and then the weight leave the type's
// range), because these calls have the cycles: HBM bounds them.
//
// Measured in replays of a CUDA graph over three sets of inputs (of the largest,
// 2 GB a call, some pages are then still in L2): 48 streams of 4000 to 16,000
// positions, 32 q heads on 8 of 128, FP16: 286 us; call by call, inputs anew,
// 323 us, 6.1 TB/s, 93 % of a plain copy's rate.  128 streams of 200 to 4096,
// 14 heads on 2 of 64, BF16: 33 us, 4.4 TB/s; 5 us to the first page's scores,
// 22 of pages at a copy's rate, 2.7 of joins, the rest not accounted for.
// One such stream of 4032: 9.9 us, all of it latency.
#pragma once

#include "hb_paged.cuh"

namespace hb {
namespace paged {

constexpr int kRowsTile = 16;
// A tile's start and end, in pages (2: 128 streams 36.2 us, a step that mixes
// chunks and decoding 42; 4: 34.4, 37; 8: 34.4, 39).
constexpr int kRowsExtra = 4;
// Units a piece has at least: more and shorter pieces read a lone stream's pages
// sooner and have more parts to join (3 and 5: 10.2 us, 8: 12.1).
constexpr int kRowsLeast = 5;
constexpr int kRowsWarps = 4;                       // consumer warps
constexpr int kRowsThreads = 32 * (kRowsWarps + 1);
template <int D>
struct RowsSize {
  static constexpr int kStageBytes = 2 * (D / 64) * kBlockBytes;
  // 128 KB in flight a multiprocessor and more: two blocks of 4 x 16 KB (3, 4
  // or 5 stages: 33.8, 33.6, 34.4 us for 128 streams), one of 5 x 32 KB (3, 4, 5:
  // 303, 293, 291 us for 64 streams of 32,768)
  static constexpr int kStages = D == 64 ? 4 : 5;
  static constexpr int kPitch = D + 4;              // floats a row of the joined tile
  static constexpr int kJoinBytes = kRowsWarps * kRowsTile * kPitch * 4;
  static constexpr int kSmem = kStages * kStageBytes + kJoinBytes;
  static constexpr int kPartFloats = kRowsTile * (D + 2);   // o, m, l
};

template <class T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

// Barrier 1 over the consumer warps; the second form also ORs a predicate.
__device__ __forceinline__ void rows_sync() { consumer_sync(32 * kRowsWarps); }
__device__ __forceinline__ bool rows_any(bool pred) {
  uint32_t out;
  asm volatile(
      "{\n\t.reg .pred p, r;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "bar.red.or.pred r, 1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, r;\n\t}"
      : "=r"(out) : "r"(pred ? 1u : 0u), "r"(32 * kRowsWarps) : "memory");
  return out != 0;
}

// Two neighbouring elements of packed row r of a tile, as they lie in memory:
// not as read-only data, which they are not while the kernel before this one
// still writes them.  Plain loads: the four warps share a tile's q in L1 (past L1:
// 96 streams with heads of 128, 12 of them with 8 rows, 105 us instead of 94).
template <class T>
__device__ __forceinline__ uint32_t q_pair(const Attend &A, const T *row, int col, bool ok) {
  if (!ok) return 0u;
  if (A.q_vec) return *reinterpret_cast<const uint32_t *>(row + col);
  const uint16_t *h = reinterpret_cast<const uint16_t *>(row + col);
  return static_cast<uint32_t>(h[0]) | static_cast<uint32_t>(h[1]) << 16;
}

// Row r's kPer values v[] (dims d0 ..) of a finished tile, and its lse by the
// thread that holds dim 0.  False when a value is not finite though l is.
template <int D, class T, int kPer>
__device__ __forceinline__ bool store_row(const Attend &A, const Entry &e, int head, int r, int d0, const float *o,
                                          float m, float l) {
  using E = Elem<T>;
  const int i = A.shape.row_of(r), g = r - i * A.shape.group;
  const int64_t row = e.row0 + i;
  const int qh = head * A.shape.group + g;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T *out = static_cast<T *>(A.out) + row * A.o_row + qh * A.o_head + d0;
  float v[kPer];
  bool fine = true;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    v[k] = l == 0.f ? 0.f : o[k] * inv;
    fine &= fabsf(v[k]) <= 3.4e38f;
  }
  if (A.o_vec) {
#pragma unroll
    for (int k = 0; k < kPer; k += 8)
      *reinterpret_cast<uint4 *>(out + k) = make_uint4(E::pack(v[k], v[k + 1]), E::pack(v[k + 2], v[k + 3]),
                                                       E::pack(v[k + 4], v[k + 5]), E::pack(v[k + 6], v[k + 7]));
  } else {
#pragma unroll
    for (int k = 0; k < kPer; ++k) out[k] = E::put(v[k]);
  }
  if (A.lse != nullptr && d0 == 0) A.lse[row * A.q_heads + qh] = l == 0.f ? -INFINITY : m * A.scale + logf(l);
  return fine || !(l <= 3.4e38f);
}

// Two blocks a multiprocessor with heads of 64 (three would have to keep parts
// of O in memory), one with heads of 128, whose ring has the same bytes.
template <int D, class T>
__global__ void __launch_bounds__(kRowsThreads, D == 64 ? 2 : 1) paged_rows_kernel(const __grid_constant__ Attend A, int least) {
  using E = Elem<T>;
  using Z = RowsSize<D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ __align__(8) uint64_t s_full[Z::kStages], s_empty[Z::kStages];
  __shared__ int s_valid[Z::kStages];
  __shared__ float s_m[kRowsWarps][kRowsTile], s_l[kRowsWarps][kRowsTile];
  __shared__ int s_last;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Shape S = A.shape;
  const Line line = line_at(smem + Z::kSmem, A.batch.entries);
  Ctrl *ctrl = &A.pool.control->ctrl;

  if (threadIdx.x == 0) {
    for (int i = 0; i < Z::kStages; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_empty[i], kRowsWarps);
    }
    fence_mbar_init();
  }
  if (A.beside) first_begin(A.pool.control, A.beside); else grid_begin();
  if (!fill_line(A.pool, A.batch, S, line, [&](const Entry &e) { return e.n * S.group <= A.few; })) {
    rows_unseen<D>(A, 0, 0);
    return;
  }
  rows_of_no_entry<D>(A, line);
  const Cut cut(line.prefix[A.batch.entries], gridDim.x, least);
  if (static_cast<int>(blockIdx.x) >= cut.pieces) return;
  Walk w;
  w.u = cut.begin(blockIdx.x);
  w.end = cut.begin(blockIdx.x + 1);
  bool more = w.start(A.pool, A.batch, S, line);
  int it = 0;  // stages used so far

  if (warp == kRowsWarps) {
    bool ok = true;
    for (; more && ok; more = w.next(A.pool, A.batch, S, line)) {
      const int first = w.first(), count = w.count(S);
      for (int k0 = 0; k0 < count && ok; k0 += 32) {
        const int mine = k0 + lane < count ? page_of<true>(A.pool, w.e.slot, first + k0 + lane) : -1;
        for (int k = k0; k < min(count, k0 + 32); ++k, ++it) {
          const int s = it % Z::kStages;
          const uint32_t ph = static_cast<uint32_t>(it / Z::kStages) & 1u;
          ok = __all_sync(0xffffffffu, mbar_wait(&s_empty[s], ph ^ 1u, ctrl, A.limit_ns, kWhereEmpty)) != 0;
          if (!ok) break;
          const int pg = __shfl_sync(0xffffffffu, mine, k - k0);
          const int held = min(kPage, w.e.length - (first + k) * kPage);   // positions of the page that exist
          uint8_t *dst = smem + s * Z::kStageBytes;
          const bool valid = pg >= 0 && held > 0;
          if (valid && held < kPage) {
            // V past the last position: zero, so that weight zero times it is zero
            for (int h = 0; h < D / 64; ++h)
              for (int x = held * 128 + lane * 16; x < kBlockBytes; x += 512)
                *reinterpret_cast<uint4 *>(dst + (D / 64 + h) * kBlockBytes + x) = make_uint4(0, 0, 0, 0);
            fence_proxy_async_smem();
            __syncwarp();
          }
          if (lane == 0) {
            s_valid[s] = valid ? 1 : 0;
            const uint8_t *src = valid ? kv_block(A, pg, w.head) : nullptr;
            if (!valid) {
              mbar_arrive_count(&s_full[s], 1);
            } else if (held == kPage) {
              mbar_arrive_expect_tx(&s_full[s], Z::kStageBytes);
              bulk_g2s(dst, src, Z::kStageBytes, &s_full[s]);
            } else {
              mbar_arrive_expect_tx(&s_full[s], 2 * (D / 64) * held * 128);
              for (int h = 0; h < 2 * (D / 64); ++h)
                bulk_g2s(dst + h * kBlockBytes, src + h * kBlockBytes, held * 128, &s_full[s]);
            }
          }
          __syncwarp();
        }
      }
    }
    // nothing in flight when the block ends
    for (int i = max(0, it - Z::kStages); i < it; ++i)
      mbar_wait_quiet(&s_full[i % Z::kStages], static_cast<uint32_t>(i / Z::kStages) & 1u, A.limit_ns);
    return;
  }

  float *join = reinterpret_cast<float *>(smem + Z::kStages * Z::kStageBytes);
  const int mat = lane >> 3, mrow = lane & 7;
  bool ok = true;
  unsigned done = 0;   // of rows_again; bit 2: there is a row to look at
  for (; more; more = w.next(A.pool, A.batch, S, line)) {
    const int packed = w.e.n * S.group;
    // this thread's rows of the tile: r, r + 8
    const int r0 = w.t * kRowsTile + (lane >> 2);
    int pos[2];
    const T *qrow[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = r0 + 8 * h, i = S.row_of(r), g = r - i * S.group;
      const bool in = r < packed;
      pos[h] = in ? w.e.length - w.e.n + i : -1;
      qrow[h] = static_cast<const T *>(A.q) +
                (in ? (w.e.row0 + i) * A.q_row + (w.head * S.group + g) * A.q_head : 0);
    }
    uint32_t qa[D / 16][4];
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
      for (int x = 0; x < 4; ++x)
        qa[ks][x] = q_pair<T>(A, qrow[x & 1], ks * 16 + (x >> 1) * 8 + (lane & 3) * 2, r0 + 8 * (x & 1) < packed);
    // positions that every row of the tile sees need no mask
    const int tail = min(packed, (w.t + 1) * kRowsTile) - 1;
    const int all_hi = w.e.length - w.e.n + S.row_of(w.t * kRowsTile);
    const int all_lo = S.first_seen(w.e.length - w.e.n + S.row_of(tail));

    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    float o[D / 8][4];
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
      for (int x = 0; x < 4; ++x) o[n][x] = 0.f;

    const int first = w.first(), count = w.count(S);
    for (int k = 0; k < count; ++k, ++it) {
      const int s = it % Z::kStages;
      const uint32_t ph = static_cast<uint32_t>(it / Z::kStages) & 1u;
      ok = ok && mbar_wait(&s_full[s], ph, ctrl, A.limit_ns, kWhereFull);
      if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
      const int j0 = (first + k) * kPage + warp * 16;
      if (s_valid[s] && j0 < w.e.length) {
        const uint32_t kb = smem_u32(smem + s * Z::kStageBytes), vb = kb + D / 64 * kBlockBytes;
        float sc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
        const int key = warp * 16 + (mat >> 1) * 8 + mrow;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          const int c = ks * 2 + (mat & 1);
          uint32_t b[4];
          ldsm4(b, kb + (c >> 3) * kBlockBytes + key * 128 + (((c & 7) ^ (key & 7)) << 4));
          mma16816<T>(sc[0], qa[ks], b[0], b[1]);
          mma16816<T>(sc[1], qa[ks], b[2], b[3]);
        }
        if (j0 + 15 > all_hi || j0 < all_lo) {
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int j = j0 + n * 8 + (lane & 3) * 2 + (x & 1), p = pos[x >> 1];
              if (j > p || j < S.first_seen(p)) sc[n][x] = -INFINITY;
            }
        }
        uint32_t ph_[4], pl_[4];   // the weights' high and low halves
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float mx = fmaxf(fmaxf(sc[0][2 * h], sc[0][2 * h + 1]), fmaxf(sc[1][2 * h], sc[1][2 * h + 1]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          const float nm = fmaxf(m[h], mx), use = nm == -INFINITY ? 0.f : nm;
          const float a = exp2_approx((m[h] - use) * A.scale_log2);
          m[h] = nm;
          float p[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) p[x] = exp2_approx((sc[x >> 1][2 * h + (x & 1)] - use) * A.scale_log2);
          l[h] = fmaf(l[h], a, (p[0] + p[1]) + (p[2] + p[3]));
#pragma unroll
          for (int n = 0; n < D / 8; ++n) {
            o[n][2 * h] *= a;
            o[n][2 * h + 1] *= a;
          }
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const uint32_t hi = E::pack(p[2 * n], p[2 * n + 1]);
            ph_[2 * n + h] = hi;
            pl_[2 * n + h] = E::pack(p[2 * n] - E::lo(hi), p[2 * n + 1] - E::hi(hi));
          }
        }
        const int vkey = warp * 16 + (mat & 1) * 8 + mrow;
#pragma unroll
        for (int n = 0; n < D / 16; ++n) {
          const int c = n * 2 + (mat >> 1);
          uint32_t b[4];
          ldsm4_t(b, vb + (c >> 3) * kBlockBytes + vkey * 128 + (((c & 7) ^ (vkey & 7)) << 4));
          mma16816<T>(o[2 * n], ph_, b[0], b[1]);
          mma16816<T>(o[2 * n + 1], ph_, b[2], b[3]);
          mma16816<T>(o[2 * n], pl_, b[0], b[1]);
          mma16816<T>(o[2 * n + 1], pl_, b[2], b[3]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive_count(&s_empty[s], 1);
    }
    if (rows_any(!ok)) return;   // a wait gave up: the control block says which

    // join the warps' halves of the tile
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
      if ((lane & 3) == 0) {
        s_m[warp][(lane >> 2) + 8 * h] = m[h];
        s_l[warp][(lane >> 2) + 8 * h] = l[h];
      }
      float *dst = join + (warp * kRowsTile + (lane >> 2) + 8 * h) * Z::kPitch + (lane & 3) * 2;
#pragma unroll
      for (int n = 0; n < D / 8; ++n) *reinterpret_cast<float2 *>(dst + n * 8) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
    }
    rows_sync();
    constexpr int kPer = D / 8;
    const int r = threadIdx.x >> 3, d0 = (threadIdx.x & 7) * kPer;   // this thread's row and dims
    float tm = -INFINITY, tl = 0.f, v[kPer];
#pragma unroll
    for (int x = 0; x < kRowsWarps; ++x) tm = fmaxf(tm, s_m[x][r]);
#pragma unroll
    for (int d = 0; d < kPer; ++d) v[d] = 0.f;
#pragma unroll
    for (int x = 0; x < kRowsWarps; ++x) {
      const float f = exp2_approx((s_m[x][r] - (tm == -INFINITY ? 0.f : tm)) * A.scale_log2);
      tl = fmaf(s_l[x][r], f, tl);
#pragma unroll
      for (int d = 0; d < kPer; d += 4) {
        const float4 y = *reinterpret_cast<const float4 *>(join + (x * kRowsTile + r) * Z::kPitch + d0 + d);
        v[d] = fmaf(y.x, f, v[d]);
        v[d + 1] = fmaf(y.y, f, v[d + 1]);
        v[d + 2] = fmaf(y.z, f, v[d + 2]);
        v[d + 3] = fmaf(y.w, f, v[d + 3]);
      }
    }
    const int row = w.t * kRowsTile + r;
    const bool whole = w.whole();
    bool write = row < packed;
    if (!whole) {
      // a tile that other pieces share: leave this part, and the last of
      // them to arrive joins all parts in order
      float *part = A.parts + (static_cast<int64_t>(blockIdx.x) * 2 + (w.opens() ? 1 : 0)) * Z::kPartFloats;
      if (write) {
#pragma unroll
        for (int d = 0; d < kPer; d += 4)
          __stcg(reinterpret_cast<float4 *>(part + r * D + d0 + d), make_float4(v[d], v[d + 1], v[d + 2], v[d + 3]));
        if (d0 == 0) {
          __stcg(part + kRowsTile * D + r, tm);
          __stcg(part + kRowsTile * (D + 1) + r, tl);
        }
      }
      rows_sync();
      const int c0 = cut.of(w.tile_u + S.extra), parts = cut.of(w.tile_u + w.units - 1) - c0 + 1;
      if (threadIdx.x == 0) {
        s_last = arrive_acq_rel(&A.arrived[c0]) == parts - 1;   // the barriers make it all threads'
        if (s_last) A.arrived[c0] = 0;
      }
      rows_sync();
      write = write && s_last != 0;
      if (s_last != 0) {
        done |= w.opens() ? 2u : 1u;
        // part k: the second slot of the first piece, the first of the others
        const float *base = A.parts + static_cast<int64_t>(c0) * 2 * Z::kPartFloats;
        auto part_at = [&](int k) { return base + (static_cast<int64_t>(k) * 2 + (k == 0 ? 1 : 0)) * Z::kPartFloats; };
        // eight parts a round, all their reads in flight; of the eight threads
        // of a row each weighs one part
        const int mine = threadIdx.x & 7;
        tm = -INFINITY;
        tl = 0.f;
#pragma unroll
        for (int d = 0; d < kPer; ++d) v[d] = 0.f;
#pragma unroll 2
        for (int k0 = 0; k0 < parts; k0 += 8) {
          const float *own = part_at(min(k0 + mine, parts - 1)) + kRowsTile * D + r;
          float pm = __ldcg(own), pl = __ldcg(own + kRowsTile);
          float4 y[8][kPer / 4];
#pragma unroll
          for (int x = 0; x < 8; ++x)
#pragma unroll
            for (int d = 0; d < kPer / 4; ++d)
              y[x][d] = k0 + x < parts ? __ldcg(reinterpret_cast<const float4 *>(part_at(k0 + x) + r * D + d0) + d)
                                       : make_float4(0.f, 0.f, 0.f, 0.f);
          if (k0 + mine >= parts) pm = -INFINITY;
          float top = pm;
#pragma unroll
          for (int x = 1; x < 8; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
          top = fmaxf(top, tm);
          const float use = top == -INFINITY ? 0.f : top;
          const float old = exp2_approx((tm - use) * A.scale_log2), f = exp2_approx((pm - use) * A.scale_log2);
          tm = top;
          float sum = f * pl;
          if (k0 + mine >= parts) sum = 0.f;
#pragma unroll
          for (int x = 1; x < 8; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
          tl = fmaf(tl, old, sum);
#pragma unroll
          for (int d = 0; d < kPer; ++d) v[d] *= old;
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            const float g = __shfl_sync(0xffffffffu, f, (lane & 24) + x);
#pragma unroll
            for (int d = 0; d < kPer / 4; ++d) {
              v[4 * d] = fmaf(y[x][d].x, g, v[4 * d]);
              v[4 * d + 1] = fmaf(y[x][d].y, g, v[4 * d + 1]);
              v[4 * d + 2] = fmaf(y[x][d].z, g, v[4 * d + 2]);
              v[4 * d + 3] = fmaf(y[x][d].w, g, v[4 * d + 3]);
            }
          }
        }
      }
    }
    if (write && !store_row<D, T, kPer>(A, w.e, w.head, row, d0, v, tm, tl)) done |= 4u;
  }
  if (__any_sync(0xffffffffu, done & 4u)) rows_again<D, T>(A, line, least, warp * (kRowsTile / kRowsWarps), kRowsTile / kRowsWarps, done);
}

}  // namespace paged
}  // namespace hb
