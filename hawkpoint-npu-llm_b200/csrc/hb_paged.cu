// hb_paged.cu -- the paged K/V cache operators of the C ABI: argument checks,
// workspace and launches around hb_paged_rows.cuh and hb_paged_tiles.cuh
// (attention) and hb_paged_ops.cuh (append and the page operators).
#include <atomic>

#include "hb_engine_impl.h"
#include "hb_paged_ops.cuh"
#include "hb_paged_tiles.cuh"

using namespace hbi;
namespace pg = hb::paged;

namespace {

constexpr int kMaxDevices = 64;
constexpr int kMaxHeads = 1 << 16;   // q heads: products with them are 32-bit
constexpr int kAppendMost = pg::kAppendRows;
constexpr int kAppendBlocks = 8;   // blocks a multiprocessor, at most (4: 27.4 us for 24 prompts, 8: 27.5, 16: 29.7)

// What a device's calls need to know, looked up on the first of them.
struct DeviceInfo {
  std::atomic<int> ready{0};
  int sms = 0;
};
DeviceInfo g_devices[kMaxDevices];

template <int D, class T>
cudaError_t opt_in() {
  const cudaError_t err = cudaFuncSetAttribute(pg::paged_rows_kernel<D, T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               static_cast<int>(pg::RowsSize<D>::kSmem + pg::line_bytes(pg::kMaxEntries)));
  if (err != cudaSuccess) return err;
  return cudaFuncSetAttribute(pg::paged_tiles_kernel<D, T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              static_cast<int>(pg::TilesSize<D>::kSmem + pg::line_bytes(pg::kMaxEntries)));
}

// The current device's multiprocessors; the first call on a device also opts
// the kernels into their shared memory there.
int device_info(const char *who, int *sms) {
  int dev = 0;
  HB_CUDA(nullptr, cudaGetDevice(&dev));
  if (dev < 0 || dev >= kMaxDevices) return fail(nullptr, HB_ERR_UNSUPPORTED, "%s: device %d", who, dev);
  DeviceInfo &d = g_devices[dev];
  if (!d.ready.load(std::memory_order_acquire)) {
    int major = 0, n = 0;
    HB_CUDA(nullptr, cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev));
    if (major != 10) return fail(nullptr, HB_ERR_UNSUPPORTED, "%s: needs an sm_100 GPU", who);
    HB_CUDA(nullptr, cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
    HB_CUDA(nullptr, (opt_in<64, __nv_bfloat16>()));
    HB_CUDA(nullptr, (opt_in<64, __half>()));
    HB_CUDA(nullptr, (opt_in<128, __nv_bfloat16>()));
    HB_CUDA(nullptr, (opt_in<128, __half>()));
    d.sms = n;
    d.ready.store(1, std::memory_order_release);
  }
  *sms = d.sms;
  return HB_OK;
}

// The pieces an attention call is cut into at most: resident blocks.
constexpr int kMaxSms = pg::kTilesPieces;
int rows_pieces(int head_dim, int sms) { return head_dim == 64 ? 2 * sms : sms; }

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

// Byte offsets of the workspace's regions.
struct Regions {
  size_t mark, need, off, fresh, from, to, held, stage, arrived, arrived2, parts, parts2, total;
};
Regions regions(const hb_page_pool &p) {
  Regions r{};
  const size_t slots = static_cast<size_t>(p.n_slots), pages = static_cast<size_t>(p.n_pages);
  const size_t list = std::max(pages, slots) * 4;
  size_t at = 256;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += align256(bytes);
    return here;
  };
  r.mark = take(slots * 4);
  r.arrived = take(2 * kMaxSms * 4);
  r.arrived2 = take(2 * 2 * pg::kTilesPieces * 4);
  r.need = take(slots * 4);
  r.off = take(slots * 4);
  r.fresh = take(pages * 4);
  r.from = take(list);
  r.to = take(list);
  r.held = take(list);
  r.stage = take(slots * static_cast<size_t>(p.table_width) * 4);
  const size_t rows = p.head_dim == 64 ? pg::RowsSize<64>::kPartFloats : pg::RowsSize<128>::kPartFloats;
  r.parts = take(static_cast<size_t>(rows_pieces(p.head_dim, kMaxSms)) * 2 * rows * 4);
  const size_t tiles = p.head_dim == 64 ? pg::TilesSize<64>::kPartFloats : pg::TilesSize<128>::kPartFloats;
  r.parts2 = take(static_cast<size_t>(kMaxSms) * 2 * 2 * tiles * 4);
  r.total = at;
  return r;
}

int64_t layer_bytes(const hb_page_pool &p) {
  return static_cast<int64_t>(p.kv_heads) * 2 * (p.head_dim / 64) * pg::kBlockBytes;
}

// The checks of a pool that need no device.
int check_shape(const char *who, const hb_page_pool *p) {
  if (!p) return fail(nullptr, HB_ERR_INVALID_ARG, "%s: pool is NULL", who);
  if (p->head_dim != 64 && p->head_dim != 128)
    return fail(nullptr, HB_ERR_UNSUPPORTED, "%s: head_dim must be 64 or 128", who);
  if (p->element != HB_ELEM_BF16 && p->element != HB_ELEM_FP16)
    return fail(nullptr, HB_ERR_UNSUPPORTED, "%s: elements must be BF16 or FP16", who);
  if (p->n_pages < 1 || p->layers < 1 || p->kv_heads < 1 || p->n_slots < 1 || p->table_width < 1 ||
      p->table_width > (1 << 24) || p->kv_heads > 1024 || p->layers > 4096)
    return fail(nullptr, HB_ERR_INVALID_ARG, "%s: pages, layers, kv heads, slots and table width must be positive", who);
  if (static_cast<int64_t>(p->n_slots) * p->table_width > INT32_MAX)   // what a reserve's page counts can add up to
    return fail(nullptr, HB_ERR_UNSUPPORTED, "%s: the table must have fewer than 2^31 entries", who);
  if (p->page_stride < layer_bytes(*p) * p->layers || p->page_stride % 128)
    return fail(nullptr, HB_ERR_INVALID_ARG, "%s: page_stride must be a multiple of 128 and hold a page", who);
  return HB_OK;
}

int check_pool(const char *who, const hb_page_pool *p) {
  int rc = check_shape(who, p);
  if (rc) return rc;
  if (!p->pages_dev || !p->table_dev || !p->refs_dev || !p->lengths_dev || !p->workspace_dev)
    return fail(nullptr, HB_ERR_INVALID_ARG, "%s: null pool pointer", who);
  if ((reinterpret_cast<uintptr_t>(p->pages_dev) & 127) || (reinterpret_cast<uintptr_t>(p->workspace_dev) & 255))
    return fail(nullptr, HB_ERR_INVALID_ARG, "%s: pages must be 128-byte and the workspace 256-byte aligned", who);
  const size_t need = regions(*p).total;
  if (p->workspace_bytes < need)
    return fail(nullptr, HB_ERR_INVALID_ARG, "%s: the workspace needs %zu bytes", who, need);
  return HB_OK;
}

int check_rows(const char *who, const hb_page_pool &p, int layer, const hb_paged_rows *r) {
  if (!r) return fail(nullptr, HB_ERR_INVALID_ARG, "%s: rows is NULL", who);
  if (layer < 0 || layer >= p.layers) return fail(nullptr, HB_ERR_INVALID_ARG, "%s: layer %d outside [0, %d)", who, layer, p.layers);
  if (r->entries < 0 || r->rows < 0 || r->max_rows < 0)
    return fail(nullptr, HB_ERR_INVALID_ARG, "%s: negative entries or rows", who);
  if (r->entries > pg::kMaxEntries)
    return fail(nullptr, HB_ERR_UNSUPPORTED, "%s: at most %d entries a call", who, pg::kMaxEntries);
  if (r->entries > 0 && (!r->slots_dev || !r->row_start_dev))
    return fail(nullptr, HB_ERR_INVALID_ARG, "%s: null rows pointer", who);
  return HB_OK;
}

pg::Pool pool_view(const hb_page_pool &p) {
  pg::Pool v{};
  v.pages = static_cast<uint8_t *>(p.pages_dev);
  v.page_stride = p.page_stride;
  v.n_pages = p.n_pages;
  v.kv_heads = p.kv_heads;
  v.width = p.table_width;
  v.n_slots = p.n_slots;
  v.table = p.table_dev;
  v.refs = p.refs_dev;
  v.lengths = p.lengths_dev;
  v.control = static_cast<pg::Control *>(p.workspace_dev);
  return v;
}

pg::Scratch scratch_view(const hb_page_pool &p, const Regions &r) {
  auto at = [&](size_t off) { return reinterpret_cast<int *>(static_cast<uint8_t *>(p.workspace_dev) + off); };
  return pg::Scratch{at(r.mark), at(r.need), at(r.off), at(r.fresh), at(r.from), at(r.to), at(r.held), at(r.stage)};
}

// Rows at a base and with strides (elements) that all are multiples of `bytes`.
bool vec_ok(const void *base, int64_t a, int64_t b, unsigned bytes = 16) {
  return ((reinterpret_cast<uintptr_t>(base) | static_cast<uintptr_t>(a * 2) | static_cast<uintptr_t>(b * 2)) & (bytes - 1)) == 0;
}

// A launch that may begin while the kernel before it on the stream ends (every
// kernel here waits for that one first).
template <class... P, class... X>
cudaError_t launch(void (*kernel)(P...), int grid, int block, size_t smem, cudaStream_t st, const X &...args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}

int launch_copy(const hb_page_pool &p, void *to_pages, int to_n, const int *from, const int *to, const int *held,
                const int *copies, int n, const int *map, int grid, cudaStream_t st) {
  const int blocks = static_cast<int>(layer_bytes(p) * p.layers / pg::kBlockBytes);
  HB_CUDA(nullptr, launch(pg::copy_kernel, grid, 256, 0, st, pool_view(p), static_cast<uint8_t *>(to_pages), to_n, from, to, held,
                          copies, n, blocks, map));
  return HB_OK;
}

// Which kernels an attention call launches: the rows kernel for entries of up
// to 16 packed rows (its tile), the tiles kernel for the others, one of them
// where the host's numbers say that it may have them all.  The tiles kernel
// costs a prologue and steps of 256 rows however few there are; the rows kernel
// reads an entry's pages again for every 16 rows of it, which heads of 64 can
// afford twice on average and heads of 128 hardly at all.  So the rows kernel
// has the call alone if no entry has more than 8 of its tiles and the average
// is at most 32 packed rows (heads of 64) or 8 (heads of 128).  Measured, rows
// kernel alone / otherwise, us: heads of 64, 64 streams of 1024 with 21 packed
// rows each 19.9 / 23.6, with 63 30.0 / 23.9; 96 streams of 200 to 2000 of which
// 12 have 126 packed rows (21.9 on average) 25.3 / 35.8.  Heads of 128: 64 streams
// with 24 packed rows 98 / 69; 96 streams, 12 with 32 (7.5 on average) 94 / 100,
// 12 with 64 (11.5) 112 / 104.  All entries alike above that are the tiles
// kernel's alone.  A bound on an entry's rows that is wrong costs time, not
// rows: a kernel launched alone takes every entry.
template <int D, class T>
cudaError_t launch_attend(pg::Attend A, int max_rows, int sms, cudaStream_t st) {
  const pg::Batch &b = A.batch;
  const int64_t most = static_cast<int64_t>(max_rows) * A.shape.group;
  constexpr int kMean = D == 64 ? 2 * pg::kRowsTile : pg::kRowsTile / 2;
  const bool rows_only =
      most <= pg::kRowsTile || (most <= 8 * pg::kRowsTile &&
                                static_cast<int64_t>(b.rows) * A.shape.group <= static_cast<int64_t>(b.entries) * kMean);
  const bool tiles_only = !rows_only && static_cast<int64_t>(b.entries) * max_rows == b.rows;
  const size_t line = pg::line_bytes(b.entries);
  A.few = rows_only ? INT32_MAX : tiles_only ? 0 : pg::kRowsTile;
  A.beside = !rows_only && !tiles_only ? sms : 0;
  if (!tiles_only) {
    A.shape.tile = pg::kRowsTile;
    A.shape.block = pg::kPage;
    A.shape.extra = pg::kRowsExtra;
    const cudaError_t err = launch(pg::paged_rows_kernel<D, T>, rows_pieces(D, sms), pg::kRowsThreads,
                                   pg::RowsSize<D>::kSmem + line, st, A, pg::kRowsLeast);
    if (err != cudaSuccess || rows_only) return err;
  }
  A.shape.tile = pg::kTilesTile;
  A.shape.block = pg::kTilesBlock;
  A.shape.extra = pg::kTilesExtra;
  A.arrived = A.arrived2;
  A.parts = A.parts2;
  const cudaError_t err =
      launch(pg::paged_tiles_kernel<D, T>, sms, pg::kTilesThreads, pg::TilesSize<D>::kSmem + line, st, A, pg::kTilesLeast);
  // the rows kernel's count would be taken for the next call's
  if (err != cudaSuccess && A.beside) cudaMemsetAsync(&A.pool.control->began, 0, sizeof(int), st);
  return err;
}

template <int D, class T>
cudaError_t launch_append(const pg::Append &A, bool vec, int grid, cudaStream_t st) {
  // whole rows a block: as many as fit, a row's part a thread
  const int parts = (A.q_heads + 2 * A.pool.kv_heads) * (D / 16);
  const int threads = parts >= pg::kAppendThreads ? pg::kAppendThreads
                                                  : (pg::kAppendThreads / parts * parts + 31) / 32 * 32;
  return vec ? launch(pg::paged_append_kernel<D, T, true>, grid, threads, 0, st, A)
             : launch(pg::paged_append_kernel<D, T, false>, grid, threads, 0, st, A);
}

}  // namespace

extern "C" {

size_t hb_paged_workspace_bytes(const hb_page_pool *pool) {
  return check_shape("hb_paged_workspace_bytes", pool) == HB_OK ? regions(*pool).total : 0;
}

int hb_paged_status(const hb_page_pool *pool, int32_t *status, void *stream) {
  int rc = check_pool("hb_paged_status", pool);
  if (rc) return rc;
  pg::Control c{};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  HB_CUDA(nullptr, cudaMemcpyAsync(&c, pool->workspace_dev, sizeof(c), cudaMemcpyDeviceToHost, st));
  HB_CUDA(nullptr, cudaStreamSynchronize(st));
  if (status) *status = c.status;
  if (c.ctrl.err || c.status) {
    HB_CUDA(nullptr, cudaMemsetAsync(pool->workspace_dev, 0, sizeof(c), st));
    if (c.ctrl.err) {   // a call that gave up may have left tiles half joined
      const Regions r = regions(*pool);
      HB_CUDA(nullptr, cudaMemsetAsync(static_cast<uint8_t *>(pool->workspace_dev) + r.arrived, 0, r.need - r.arrived, st));
    }
    HB_CUDA(nullptr, cudaStreamSynchronize(st));
  }
  if (c.ctrl.err)
    return fail(nullptr, HB_ERR_DEVICE_TIMEOUT, "paged attention: a device wait gave up (where %d)", c.ctrl.err_where);
  if (c.status & HB_PAGED_EXHAUSTED)
    return fail(nullptr, HB_ERR_STATE, "page pool exhausted: a reserve or fork changed nothing");
  if (c.status & HB_PAGED_BAD_INDEX)
    return fail(nullptr, HB_ERR_STATE, "a slot, page, position or length was out of range: the call skipped it");
  if (c.status & HB_PAGED_UNMAPPED)
    return fail(nullptr, HB_ERR_STATE, "a row was appended where no page is mapped: it was dropped");
  return HB_OK;
}

int hb_paged_attend(const hb_page_pool *pool, int layer, const hb_paged_rows *rows, const hb_paged_query *q,
                    void *stream) {
  int rc = check_pool("hb_paged_attend", pool);
  if (rc || (rc = check_rows("hb_paged_attend", *pool, layer, rows))) return rc;
  if (!q) return fail(nullptr, HB_ERR_INVALID_ARG, "hb_paged_attend: query is NULL");
  if (q->q_heads < 1 || q->q_heads % pool->kv_heads)
    return fail(nullptr, HB_ERR_INVALID_ARG, "hb_paged_attend: q_heads must be a positive multiple of kv_heads");
  if (q->q_heads > kMaxHeads) return fail(nullptr, HB_ERR_UNSUPPORTED, "hb_paged_attend: at most %d q heads", kMaxHeads);
  if (!(q->scale > 0.f) || q->scale > 1e30f || q->window < 0)
    return fail(nullptr, HB_ERR_INVALID_ARG, "hb_paged_attend: scale must be positive, window not negative");
  if (rows->rows == 0 || rows->entries == 0) return HB_OK;
  // the most units the call's line can have (16-row tiles), counted in 32 bits
  const double units = (static_cast<double>(rows->rows) * q->q_heads / pg::kRowsTile + pool->kv_heads * rows->entries) *
                       (pool->table_width + pg::kRowsExtra);
  if (units >= 2e9 || static_cast<double>(rows->rows) * q->q_heads >= 2e9)   // nor more packed rows
    return fail(nullptr, HB_ERR_UNSUPPORTED, "hb_paged_attend: too many rows for the table's width in one call");
  if (!q->q_dev || !q->out_dev) return fail(nullptr, HB_ERR_INVALID_ARG, "hb_paged_attend: null pointer");
  if ((reinterpret_cast<uintptr_t>(q->q_dev) | reinterpret_cast<uintptr_t>(q->out_dev)) & 1)
    return fail(nullptr, HB_ERR_INVALID_ARG, "hb_paged_attend: q and out must be element aligned");
  int sms = 0;
  if ((rc = device_info("hb_paged_attend", &sms))) return rc;
  sms = std::min(sms, kMaxSms);
  const Regions r = regions(*pool);
  pg::Attend A{};
  A.pool = pool_view(*pool);
  A.batch = pg::Batch{rows->slots_dev, rows->row_start_dev, rows->entries, rows->rows};
  A.layer_off = layer_bytes(*pool) * layer;
  A.head_bytes = 2 * (pool->head_dim / 64) * pg::kBlockBytes;
  A.q = q->q_dev;
  A.q_row = q->q_row_stride;
  A.q_head = q->q_head_stride;
  A.out = q->out_dev;
  A.o_row = q->out_row_stride;
  A.o_head = q->out_head_stride;
  A.lse = q->lse_dev;
  A.q_heads = q->q_heads;
  A.scale = q->scale;
  A.scale_log2 = q->scale * 1.4426950408889634f;
  A.q_vec = vec_ok(q->q_dev, q->q_row_stride, q->q_head_stride);
  A.o_vec = vec_ok(q->out_dev, q->out_row_stride, q->out_head_stride);
  A.o_wide = vec_ok(q->out_dev, q->out_row_stride, q->out_head_stride, 32);
  A.arrived = reinterpret_cast<int *>(static_cast<uint8_t *>(pool->workspace_dev) + r.arrived);
  A.parts = reinterpret_cast<float *>(static_cast<uint8_t *>(pool->workspace_dev) + r.parts);
  A.limit_ns = kDefaultLimitNs;
  A.arrived2 = reinterpret_cast<int *>(static_cast<uint8_t *>(pool->workspace_dev) + r.arrived2);
  A.parts2 = reinterpret_cast<float *>(static_cast<uint8_t *>(pool->workspace_dev) + r.parts2);
  A.shape.group = q->q_heads / pool->kv_heads;
  A.shape.width = pool->table_width;
  A.shape.window = q->window;
  A.shape.group_inv = static_cast<uint32_t>(0xFFFFFFFFull / static_cast<uint32_t>(A.shape.group));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool bf = pool->element == HB_ELEM_BF16;
  const int most = rows->max_rows;
  if (pool->head_dim == 64)
    HB_CUDA(nullptr, bf ? (launch_attend<64, __nv_bfloat16>(A, most, sms, st)) : (launch_attend<64, __half>(A, most, sms, st)));
  else
    HB_CUDA(nullptr, bf ? (launch_attend<128, __nv_bfloat16>(A, most, sms, st)) : (launch_attend<128, __half>(A, most, sms, st)));
  return HB_OK;
}

int hb_paged_append(const hb_page_pool *pool, int layer, const hb_paged_rows *rows, const hb_paged_new *n,
                    void *stream) {
  int rc = check_pool("hb_paged_append", pool);
  if (rc || (rc = check_rows("hb_paged_append", *pool, layer, rows))) return rc;
  if (!n) return fail(nullptr, HB_ERR_INVALID_ARG, "hb_paged_append: new rows are NULL");
  if (n->q_heads < 0 || n->rope_positions < 1)
    return fail(nullptr, HB_ERR_INVALID_ARG, "hb_paged_append: q_heads must not be negative, rope_positions positive");
  if (n->q_heads > kMaxHeads) return fail(nullptr, HB_ERR_UNSUPPORTED, "hb_paged_append: at most %d q heads", kMaxHeads);
  if (rows->rows == 0 || rows->entries == 0) return HB_OK;
  if (!n->qkv_dev || !n->cos_dev || !n->sin_dev || (n->q_heads > 0 && !n->q_dev))
    return fail(nullptr, HB_ERR_INVALID_ARG, "hb_paged_append: null pointer");
  if ((reinterpret_cast<uintptr_t>(n->cos_dev) | reinterpret_cast<uintptr_t>(n->sin_dev)) & 15)
    return fail(nullptr, HB_ERR_INVALID_ARG, "hb_paged_append: cos and sin must be 16-byte aligned");
  if ((reinterpret_cast<uintptr_t>(n->qkv_dev) | reinterpret_cast<uintptr_t>(n->q_dev)) & 1)
    return fail(nullptr, HB_ERR_INVALID_ARG, "hb_paged_append: qkv and q must be element aligned");
  int sms = 0;
  if ((rc = device_info("hb_paged_append", &sms))) return rc;
  pg::Append A{};
  A.pool = pool_view(*pool);
  A.batch = pg::Batch{rows->slots_dev, rows->row_start_dev, rows->entries, rows->rows};
  A.layer_off = layer_bytes(*pool) * layer;
  A.head_bytes = 2 * (pool->head_dim / 64) * pg::kBlockBytes;
  A.qkv = n->qkv_dev;
  A.qkv_row = n->qkv_row_stride;
  A.q = n->q_dev;
  A.q_row = n->q_row_stride;
  A.q_head = n->q_head_stride;
  A.cos = n->cos_dev;
  A.sin = n->sin_dev;
  A.rope_positions = n->rope_positions;
  A.q_heads = n->q_heads;
  // few rows: a block each; many: enough blocks for every multiprocessor
  A.block_rows = std::max(1, std::min(kAppendMost, (rows->rows + kAppendBlocks * sms - 1) / (kAppendBlocks * sms)));
  const bool vec = vec_ok(n->qkv_dev, n->qkv_row_stride, 0) && vec_ok(n->q_dev, n->q_row_stride, n->q_head_stride);
  const int grid = (rows->rows + A.block_rows - 1) / A.block_rows;
  const bool bf = pool->element == HB_ELEM_BF16;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (pool->head_dim == 64)
    HB_CUDA(nullptr, bf ? (launch_append<64, __nv_bfloat16>(A, vec, grid, st)) : (launch_append<64, __half>(A, vec, grid, st)));
  else
    HB_CUDA(nullptr, bf ? (launch_append<128, __nv_bfloat16>(A, vec, grid, st)) : (launch_append<128, __half>(A, vec, grid, st)));
  return HB_OK;
}

int hb_pages_reserve(const hb_page_pool *pool, int n, const int32_t *slots_dev, const int32_t *counts_dev,
                     void *stream) {
  int rc = check_pool("hb_pages_reserve", pool);
  if (rc) return rc;
  if (n < 0 || n > pool->n_slots) return fail(nullptr, HB_ERR_INVALID_ARG, "hb_pages_reserve: n outside [0, n_slots]");
  if (n == 0) return HB_OK;
  if (!slots_dev || !counts_dev) return fail(nullptr, HB_ERR_INVALID_ARG, "hb_pages_reserve: null pointer");
  int sms = 0;
  if ((rc = device_info("hb_pages_reserve", &sms))) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const Regions r = regions(*pool);
  const pg::Scratch x = scratch_view(*pool, r);
  const pg::Pool v = pool_view(*pool);
  HB_CUDA(nullptr, launch(pg::reserve_kernel, 1, pg::kBookThreads, 0, st, v, x, slots_dev, counts_dev, n));
  return launch_copy(*pool, pool->pages_dev, pool->n_pages, x.from, x.to, x.held, &v.control->copies, 0, nullptr, sms, st);
}

int hb_pages_fork(const hb_page_pool *pool, int n, const int32_t *src_dev, const int32_t *dst_dev,
                  const int32_t *counts_dev, void *stream) {
  int rc = check_pool("hb_pages_fork", pool);
  if (rc) return rc;
  if (n < 0 || n > pool->n_slots) return fail(nullptr, HB_ERR_INVALID_ARG, "hb_pages_fork: n outside [0, n_slots]");
  if (n == 0) return HB_OK;
  if (!src_dev || !dst_dev || !counts_dev) return fail(nullptr, HB_ERR_INVALID_ARG, "hb_pages_fork: null pointer");
  int sms = 0;
  if ((rc = device_info("hb_pages_fork", &sms))) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const Regions r = regions(*pool);
  const pg::Scratch x = scratch_view(*pool, r);
  const pg::Pool v = pool_view(*pool);
  HB_CUDA(nullptr, launch(pg::fork_kernel, 1, pg::kBookThreads, 0, st, v, x, src_dev, dst_dev, counts_dev, n));
  // a warp an 8 KB block to copy, as far as the GPU holds them at once
  const int64_t most = (static_cast<int64_t>(n) * (layer_bytes(*pool) * pool->layers / pg::kBlockBytes) + 7) / 8;
  return launch_copy(*pool, pool->pages_dev, pool->n_pages, x.from, x.to, x.held, &v.control->copies, 0, nullptr,
                     static_cast<int>(std::min<int64_t>(most, 8 * sms)), st);
}

int hb_pages_free(const hb_page_pool *pool, int n, const int32_t *slots_dev, void *stream) {
  int rc = check_pool("hb_pages_free", pool);
  if (rc) return rc;
  if (n < 0) return fail(nullptr, HB_ERR_INVALID_ARG, "hb_pages_free: n is negative");
  if (n == 0) return HB_OK;
  if (!slots_dev) return fail(nullptr, HB_ERR_INVALID_ARG, "hb_pages_free: null pointer");
  int sms = 0;
  if ((rc = device_info("hb_pages_free", &sms))) return rc;
  HB_CUDA(nullptr, launch(pg::free_kernel, n / 4 + (n % 4 ? 1 : 0), 128, 0, static_cast<cudaStream_t>(stream), pool_view(*pool), slots_dev, n));
  return HB_OK;
}

int hb_pages_compact(const hb_page_pool *pool, int32_t *map_dev, void *stream) {
  int rc = check_pool("hb_pages_compact", pool);
  if (rc) return rc;
  if (!map_dev) return fail(nullptr, HB_ERR_INVALID_ARG, "hb_pages_compact: null pointer");
  int sms = 0;
  if ((rc = device_info("hb_pages_compact", &sms))) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const Regions r = regions(*pool);
  const pg::Scratch x = scratch_view(*pool, r);
  const pg::Pool v = pool_view(*pool);
  HB_CUDA(nullptr, launch(pg::compact_kernel, 1, pg::kBookThreads, 0, st, v, x, map_dev));
  return launch_copy(*pool, pool->pages_dev, pool->n_pages, x.from, x.to, x.held, &v.control->copies, 0, map_dev, 8 * sms, st);
}

int hb_pages_copy(const hb_page_pool *pool, int n, const int32_t *src_dev, const int32_t *dst_dev, void *dst_pages_dev,
                  int dst_n_pages, void *stream) {
  int rc = check_pool("hb_pages_copy", pool);
  if (rc) return rc;
  if (n < 0) return fail(nullptr, HB_ERR_INVALID_ARG, "hb_pages_copy: n is negative");
  if (dst_pages_dev && dst_n_pages < 1)
    return fail(nullptr, HB_ERR_INVALID_ARG, "hb_pages_copy: the destination has no pages");
  if (n == 0) return HB_OK;
  if (!src_dev || !dst_dev) return fail(nullptr, HB_ERR_INVALID_ARG, "hb_pages_copy: null pointer");
  if (reinterpret_cast<uintptr_t>(dst_pages_dev) & 127)
    return fail(nullptr, HB_ERR_INVALID_ARG, "hb_pages_copy: destination pages must be 128-byte aligned");
  int sms = 0;
  if ((rc = device_info("hb_pages_copy", &sms))) return rc;
  return launch_copy(*pool, dst_pages_dev ? dst_pages_dev : pool->pages_dev, dst_pages_dev ? dst_n_pages : pool->n_pages,
                     src_dev, dst_dev, nullptr, nullptr, n, nullptr, 8 * sms, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
