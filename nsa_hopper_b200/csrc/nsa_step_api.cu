// Host side of what comes before attention: pages and packing of a batch (nsa_cache_reserve), block selection from the 4-bit
// cache (nsa_cache_select) and rotary positions (nsa_rotary) of include/nsa_sel.h: checks and launches.
#include <cuda_runtime.h>
#include <algorithm>
#include <mutex>
#include <string.h>

#include "nsa_sel.h"
#include "nsa_cache_host.h"
#include "nsa_cache_select_kernel.cuh"
#include "nsa_reserve_kernel.cuh"
#include "nsa_rotary_kernel.cuh"

namespace {

namespace cache = nsa::cache;
namespace reserve = nsa::reserve;
namespace rotary = nsa::rotary;
namespace select = nsa::cache_select;
using nsa::cache::done;
using nsa::cache::kMaxIndex;
using nsa::cache::launch;
using nsa::cache::misaligned;
using nsa::host::cuda_fail;
using nsa::host::fail;

std::mutex g_mu;
uint32_t g_attr_done[nsa::host::kMaxDevices] = {};  // one bit for each kernel that needs much shared memory

// Once for each device: lets `kernel` have up to `bytes` of dynamic shared memory.
int allow_smem(const void* kernel, int bytes, int dev, uint32_t bit) {
  std::lock_guard<std::mutex> lk(g_mu);
  if ((g_attr_done[dev] & bit) != 0) return NSA_OK;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(shared memory)");
  g_attr_done[dev] |= bit;
  return NSA_OK;
}

// ------------------------------------------------------------------ pages
int check_reserve(const nsa_cache_reserve_desc* d) {
  if (d == nullptr) return fail(NSA_ERR_INVALID_ARG, "desc is NULL");
  if (d->n_seqs < 0 || d->width < 0 || d->pool_size < 0 || d->n_rows < 0)
    return fail(NSA_ERR_INVALID_ARG, "n_seqs, width, pool_size and n_rows must not be negative");
  if (d->cu_seqlens == nullptr && d->n_rows != d->n_seqs)
    return fail(NSA_ERR_INVALID_ARG, "without cu_seqlens there is one row a sequence: n_rows %d, n_seqs %d", d->n_rows, d->n_seqs);
  if (d->n_seqs > reserve::kMaxSeqs)
    return fail(NSA_ERR_UNSUPPORTED, "n_seqs must be at most %d", reserve::kMaxSeqs);
  if ((int64_t)d->n_seqs * d->width > kMaxIndex) return fail(NSA_ERR_UNSUPPORTED, "n_seqs * width must be below 2^31");
  if (d->pages_stride != 0 && d->pages_stride < d->width)
    return fail(NSA_ERR_INVALID_ARG, "pages_stride must not be below width");
  if (d->n_free == nullptr || d->n_free_out == nullptr || (d->pool_size > 0 && d->pool == nullptr))
    return fail(NSA_ERR_INVALID_ARG, "pool, n_free and n_free_out must be non-NULL");
  if (d->n_seqs > 0 && (d->held == nullptr || d->rows == nullptr || d->held_out == nullptr || d->lens == nullptr ||
                        (d->width > 0 && d->pages == nullptr)))
    return fail(NSA_ERR_INVALID_ARG, "pages, held, rows, held_out and lens must be non-NULL");
  for (const void* p : {(const void*)d->pages, (const void*)d->held, (const void*)d->rows, (const void*)d->pool,
                        (const void*)d->n_free, (const void*)d->held_out, (const void*)d->n_free_out, (const void*)d->lens,
                        (const void*)d->cu_seqlens})
    if (misaligned(p, 4)) return fail(NSA_ERR_INVALID_ARG, "all arrays must be aligned to their element size");
  if (misaligned(d->positions, 16) || misaligned(d->slots, 16))
    return fail(NSA_ERR_INVALID_ARG, "positions and slots must be 16-byte aligned");
  return NSA_OK;
}

int run_reserve(const nsa_cache_reserve_desc* d, cudaStream_t st) {
  int rc = check_reserve(d);
  if (rc != NSA_OK) return rc;
  int sm = 0, dev = 0;
  rc = nsa::host::current_sm_count(&sm, &dev);
  if (rc != NSA_OK) return rc;
  rc = allow_smem(reinterpret_cast<const void*>(&reserve::reserve_kernel), reserve::smem_bytes(reserve::kMaxSeqs), dev, 1u);
  if (rc != NSA_OK) return rc;
  reserve::Args a;
  memset(&a, 0, sizeof(a));
  a.pages = d->pages, a.held = d->held, a.rows = d->rows, a.pool = d->pool, a.n_free = d->n_free;
  a.held_out = d->held_out, a.n_free_out = d->n_free_out, a.lens = d->lens, a.cu = d->cu_seqlens;
  a.positions = d->positions, a.slots = d->slots;
  a.page_row = d->pages_stride ? d->pages_stride : d->width;
  a.n_seqs = d->n_seqs, a.width = d->width, a.pool_size = d->pool_size, a.n_rows = d->n_rows;
  a.rows_apart = d->cu_seqlens != nullptr && (d->positions != nullptr || d->slots != nullptr) && d->n_rows > reserve::kRowsInside;
  // One block where there is little to share out, else a cluster; threads for all sequences at once, or many.
  const int inside = a.rows_apart ? 0 : d->n_rows;
  const int blocks = std::max(d->n_seqs, inside / 8) <= 64 ? 1 : reserve::kCluster;
  const int threads = blocks == 1 ? 256 : reserve::kMaxThreads;
  cudaError_t e = launch(&reserve::reserve_kernel, dim3((unsigned)blocks), threads, reserve::smem_bytes(d->n_seqs), blocks, st, a);
  if (e == cudaSuccess && a.rows_apart)
    e = launch(&reserve::rows_kernel, dim3((unsigned)(((int64_t)d->n_rows + 255) / 256)), 256, 0, 1, st, a);
  return done(e, "cache reserve launch");
}

// ------------------------------------------------------------------ block selection
int shift_of(int32_t block_size) { return block_size == 64 ? 6 : block_size == 128 ? 7 : 8; }
// Tokens and blocks of a row, at most.
int32_t most_tokens(const nsa_cache_select_desc* d) { return select::most_tokens(d->batch.width, d->cmp_block, d->cmp_stride); }
int32_t most_blocks(const nsa_cache_select_desc* d) { return std::max(1, select::blocks_of(most_tokens(d), shift_of(d->block_size))); }
// Blocks of a warp's unit: those of about 64 keys.
int32_t unit_of(const nsa_cache_select_desc* d) {
  const int64_t blocks = (int64_t)select::kUnitKeys * d->cmp_stride / d->block_size;
  return (int32_t)std::min<int64_t>(std::max<int64_t>(blocks, 1), select::kUnitBlocks);
}
// Units of a row and KV head, at most.
int64_t units_of(const nsa_cache_select_desc* d) { return ((int64_t)most_blocks(d) + unit_of(d) - 1) / unit_of(d); }
// Rows of a launch, at most: their units have numbers of 31 bits.
int64_t rows_of_launch(const nsa_cache_select_desc* d) {
  return std::max<int64_t>(1, std::min<int64_t>(select::kMaxRows, kMaxIndex / (units_of(d) * d->batch.heads_kv)));
}

int check_select(const nsa_cache_select_desc* d) {
  if (d == nullptr) return fail(NSA_ERR_INVALID_ARG, "desc is NULL");
  const int rc = cache::check_batch(&d->batch);
  if (rc != NSA_OK) return rc;
  const nsa_cache_batch& b = d->batch;
  if (d->heads_q <= 0 || d->heads_q % b.heads_kv != 0)
    return fail(NSA_ERR_INVALID_ARG, "heads_q (%d) must be a positive multiple of heads_kv (%d)", d->heads_q, b.heads_kv);
  if (d->heads_q / b.heads_kv > select::kMaxGroup)
    return fail(NSA_ERR_UNSUPPORTED, "heads_q / heads_kv must be at most %d", select::kMaxGroup);
  if (d->q_dtype != NSA_DTYPE_BF16 && d->q_dtype != NSA_DTYPE_F16)
    return fail(NSA_ERR_INVALID_ARG, "q_dtype must be NSA_DTYPE_BF16 or NSA_DTYPE_F16");
  if (d->n_sel <= 0) return fail(NSA_ERR_INVALID_ARG, "n_sel must be positive");
  if (d->n_sel > select::kMaxSel) return fail(NSA_ERR_UNSUPPORTED, "n_sel must be at most %d", select::kMaxSel);
  if (d->block_size != 64 && d->block_size != 128 && d->block_size != 256)
    return fail(NSA_ERR_UNSUPPORTED, "block_size must be 64, 128 or 256");
  if (d->cmp_block <= 0 || d->cmp_stride <= 0) return fail(NSA_ERR_INVALID_ARG, "cmp_block and cmp_stride must be positive");
  if (units_of(d) * b.heads_kv > kMaxIndex)
    return fail(NSA_ERR_UNSUPPORTED, "heads_kv * (blocks of the longest sequence that the table holds) is too large");
  if (b.n_rows == 0) return NSA_OK;
  if (d->q == nullptr || d->sel == nullptr) return fail(NSA_ERR_INVALID_ARG, "q and sel must be non-NULL");
  if (misaligned(d->q, 16) || d->q_row_stride % 8 != 0 || d->q_head_stride % 8 != 0)
    return fail(NSA_ERR_INVALID_ARG, "q must be 16-byte aligned and its strides multiples of 8");
  if (misaligned(d->sel, 4)) return fail(NSA_ERR_INVALID_ARG, "sel must be aligned to its element size");
  return NSA_OK;
}

template <int D, int THREADS, int PER_SM>
int launch_pick(const select::Args& a, int dev, uint32_t bit, cudaStream_t st) {
  const auto kernel = &select::pick_kernel<D, THREADS, PER_SM>;
  const int rc = allow_smem(reinterpret_cast<const void*>(kernel), select::list_bytes(select::kMaxSel), dev, bit);
  if (rc != NSA_OK) return rc;
  const cudaError_t e = launch(kernel, dim3((unsigned)(a.rows * a.hkv)), THREADS, select::list_bytes(a.n_sel), 1, st, a);
  return e == cudaSuccess ? NSA_OK : done(e, "cache selection launch");
}

template <int D>
int launch_select(select::Args a, int32_t n_rows, int64_t most, int sm, int dev, cudaStream_t st) {
  const int fixed = (int)sizeof(select::ScoreWarp<D>) * select::warps_of(D);
  const uint32_t bit = D == 64 ? 2u : D == 128 ? 16u : 128u;  // (three kernels each)
  int rc = allow_smem(reinterpret_cast<const void*>(&select::score_kernel<D>), fixed + select::kMaxRows * 12 + 4, dev, bit);
  if (rc != NSA_OK) return rc;
  const int64_t units = (a.blocks + a.unit - 1) / a.unit;  // of a row and KV head
  for (int64_t row0 = 0; row0 < n_rows; row0 += most) {
    a.row0 = (int32_t)row0;
    a.rows = (int32_t)std::min(most, n_rows - row0);
    // (two units for a block at least, so that where there are few some SMs are left for pick_kernel, which begins before this
    // one has ended: one sequence of 65536 tokens 11.8 us, and 9.4 so)
    const int64_t grid = std::min<int64_t>(sm, (units * a.hkv * a.rows + 1) / 2);
    cudaError_t e = launch(&select::score_kernel<D>, dim3((unsigned)grid), select::warps_of(D) * 32, fixed + a.rows * 12 + 4, 1, st, a);
    if (e != cudaSuccess) return done(e, "cache selection's score launch");
    // A block's chain of steps takes longer with 128 threads than with 256, but less of it is spent in waiting for one another: where
    // the blocks are more than fit at once, 8 small ones an SM win (256 sequences of up to 65536 tokens, 4 heads: 56 us
    // against 64; 400 of up to 8192: 34 against 41), else 3 large ones (64 of up to 32768: 17 against 23).  They are even at
    // 4 to 6 an SM.  The small ones look at 1024 of a row's blocks at a time, and a second look costs more than they gain (200
    // sequences of up to 131072: 84 against 75).  The host sees the table's width, not the lengths: where short sequences
    // have a table for more than 1024 blocks the large ones are taken.
    const int32_t covered = (a.most - a.cmp_block + 1) >> a.shift;  // (by whole pages of keys; a.blocks may be one or a few more)
    const bool many = (int64_t)a.rows * a.hkv > 5 * (int64_t)sm && covered <= select::checked(128);
    rc = many ? launch_pick<D, 128, 8>(a, dev, 4 * bit, st) : launch_pick<D, 256, 3>(a, dev, 2 * bit, st);
    if (rc != NSA_OK) return rc;
  }
  return done(cudaSuccess, "");
}

int run_select(const nsa_cache_select_desc* d, cudaStream_t st) {
  int rc = check_select(d);
  if (rc != NSA_OK) return rc;
  const nsa_cache_batch& b = d->batch;
  if (b.n_rows == 0) return done(cudaSuccess, "");
  if (d->workspace == nullptr || misaligned(d->workspace, 16))
    return fail(NSA_ERR_INVALID_ARG, "workspace must be non-NULL and 16-byte aligned");
  int sm = 0, dev = 0;
  rc = nsa::host::current_sm_count(&sm, &dev);
  if (rc != NSA_OK) return rc;
  select::Args a;
  memset(&a, 0, sizeof(a));
  a.b = cache::device_batch(&b);
  a.q = d->q;
  a.q_row = d->q_row_stride ? d->q_row_stride : (int64_t)d->heads_q * b.d_qk;
  a.q_head = d->q_head_stride ? d->q_head_stride : b.d_qk;
  a.cache = static_cast<const uint8_t*>(b.cache);
  a.page_stride = cache::page_stride_of(&b);
  a.bounds = static_cast<float2*>(d->workspace);
  a.sel = d->sel;
  a.hkv = b.heads_kv, a.group = d->heads_q / b.heads_kv, a.n_sel = d->n_sel;
  a.shift = shift_of(d->block_size);
  a.blocks = most_blocks(d);
  a.unit = unit_of(d);
  a.most = most_tokens(d);
  a.cmp_block = d->cmp_block, a.cmp_stride = d->cmp_stride;
  a.record = cache::record_bytes(b.d_qk, b.d_v);
  a.q_half = d->q_dtype == NSA_DTYPE_F16;
  a.bits = 44;  // (the sum of the heads, below 2^46, in six signed bytes; a value's whole part is below 2^22)
  while ((1 << (46 - a.bits)) < a.group) --a.bits;
  a.keys = d->block_size / d->cmp_stride + 2;  // (keys are at least cmp_stride apart, but for a rounding; at most 258)
  a.per_key = ((1u << 20) + a.keys - 1) / a.keys;
  a.at_once = select::kKeys / a.keys;
  const int64_t most = rows_of_launch(d);
  if (b.d_qk == 64) return launch_select<64>(a, b.n_rows, most, sm, dev, st);
  if (b.d_qk == 128) return launch_select<128>(a, b.n_rows, most, sm, dev, st);
  return launch_select<192>(a, b.n_rows, most, sm, dev, st);
}

// ------------------------------------------------------------------ rotary positions
int check_rotary(const nsa_rotary_desc* d) {
  if (d == nullptr) return fail(NSA_ERR_INVALID_ARG, "desc is NULL");
  if (d->batch < 0 || d->tokens < 0) return fail(NSA_ERR_INVALID_ARG, "batch and tokens must not be negative");
  if (d->dtype != NSA_DTYPE_BF16 && d->dtype != NSA_DTYPE_F16 && d->dtype != NSA_DTYPE_F32)
    return fail(NSA_ERR_INVALID_ARG, "dtype must be NSA_DTYPE_BF16, NSA_DTYPE_F16 or NSA_DTYPE_F32");
  if (d->pairs <= 0 || d->offset < 0 || (int64_t)d->offset + 2 * (int64_t)d->pairs > d->d)
    return fail(NSA_ERR_INVALID_ARG, "the rotary part, %d pairs from value %d on, must lie in the head's %d values", d->pairs,
                d->offset, d->d);
  if (d->d > 2 * rotary::kMaxPairs) return fail(NSA_ERR_UNSUPPORTED, "d must be at most %d", 2 * rotary::kMaxPairs);
  if (d->axes < 1 || d->axes > 4) return fail(NSA_ERR_UNSUPPORTED, "there must be one to four axes");
  if (d->turns == nullptr) return fail(NSA_ERR_INVALID_ARG, "turns must be non-NULL");
  for (int i = 0; d->axis != nullptr && i < d->pairs; ++i)
    if (d->axis[i] >= d->axes) return fail(NSA_ERR_INVALID_ARG, "axis[%d] = %d, of %d axes", i, d->axis[i], d->axes);
  const int size = d->dtype == NSA_DTYPE_F32 ? 4 : 2;
  int64_t heads = 0;
  for (int i = 0; i < 2; ++i) {
    const nsa_rotary_tensor& t = d->t[i];
    if (t.heads < 0) return fail(NSA_ERR_INVALID_ARG, "heads must not be negative");
    if (t.x == nullptr) {
      if (i == 0 && t.heads > 0 && (int64_t)d->batch * d->tokens > 0) return fail(NSA_ERR_INVALID_ARG, "x must be non-NULL");
      continue;
    }
    heads += t.heads;
    if (t.y == nullptr) return fail(NSA_ERR_INVALID_ARG, "y must be non-NULL");
    if (misaligned(t.x, size) || misaligned(t.y, size))
      return fail(NSA_ERR_INVALID_ARG, "x and y must be aligned to their element size");
  }
  if (heads > 65535) return fail(NSA_ERR_UNSUPPORTED, "there must be at most 65535 heads");
  if ((int64_t)d->batch * d->tokens > kMaxIndex) return fail(NSA_ERR_UNSUPPORTED, "batch * tokens must be below 2^31");
  if ((int64_t)d->batch * d->tokens > 0 && (d->positions == nullptr || misaligned(d->positions, 4)))
    return fail(NSA_ERR_INVALID_ARG, "positions must be non-NULL and aligned to its element size");
  return NSA_OK;
}

template <class T, int VEC>
cudaError_t launch_rotary(const rotary::Args& a, dim3 grid, int threads, int smem, cudaStream_t st) {
  if (a.tokens_block > 1) return launch(&rotary::rotary_kernel<T, VEC, true>, grid, threads, smem, 1, st, a);
  return launch(&rotary::rotary_kernel<T, VEC, false>, grid, threads, smem, 1, st, a);
}

int run_rotary(const nsa_rotary_desc* d, cudaStream_t st) {
  int rc = check_rotary(d);
  if (rc != NSA_OK) return rc;
  rotary::Args a;
  memset(&a, 0, sizeof(a));
  a.first = d->t[0].x != nullptr ? d->t[0].heads : 0;
  a.heads = a.first + (d->t[1].x != nullptr ? d->t[1].heads : 0);
  const int64_t total = (int64_t)d->batch * d->tokens;
  if (total == 0 || a.heads == 0) return done(cudaSuccess, "");
  int sm = 0, dev = 0;
  rc = nsa::host::current_sm_count(&sm, &dev);
  if (rc != NSA_OK) return rc;
  // Words of 16 bytes where everything is a multiple of them, else of fewer.
  const int size = d->dtype == NSA_DTYPE_F32 ? 4 : 2;
  uint64_t all = (uint64_t)d->offset | (uint64_t)d->pairs | (uint64_t)d->d | (uint64_t)(16 / size);
  for (int i = 0; i < 2; ++i) {
    const nsa_rotary_tensor& t = d->t[i];
    if (t.x == nullptr) continue;
    a.t[i].x = t.x, a.t[i].y = t.y;
    for (int j = 0; j < 3; ++j) {
      a.t[i].xs[j] = t.x_stride[j], a.t[i].ys[j] = t.y_stride[j];
      all |= (uint64_t)t.x_stride[j] | (uint64_t)t.y_stride[j];
    }
    all |= (uint64_t)((reinterpret_cast<uintptr_t>(t.x) | reinterpret_cast<uintptr_t>(t.y)) / (uintptr_t)size);
  }
  const int vec = (int)(all & (~all + 1));  // the largest power of two that divides all of them
  a.pos = d->positions;
  for (int j = 0; j < 3; ++j) a.ps[j] = d->pos_stride[j];
  a.batch = d->batch, a.tokens = d->tokens;
  a.offset = d->offset, a.pairs = d->pairs, a.rest = d->d - 2 * d->pairs;
  a.interleaved = d->interleaved != 0;
  a.flip = d->inverse ? 0x80000000u : 0u;
  memcpy(a.turn, d->turns, sizeof(uint64_t) * d->pairs);
  if (d->axis != nullptr) memcpy(a.axis, d->axis, d->pairs);
  // A block has a token; where tokens are few, its heads are shared out among blocks.  Where they are more than are turned at once,
  // a block has as many threads as its turns need (16384 tokens of 32 + 8 heads of 128 in bf16: 56 us, and 61 with 256), and as
  // many tokens as they have room for (10 heads of 64: 12 us, and 24 with one; 2 of 128 and 65536 tokens: 28 and 90).  Where all
  // are turned at once more threads are faster (1024 tokens of 68 heads: 7.4 us with 256, 8.2 with the 192 that they need).
  const int items = a.pairs / vec + (a.rest + 2 * vec - 1) / (2 * vec);
  const int64_t most = ((int64_t)a.heads * items + rotary::kThreads - 1) / rotary::kThreads;
  const int64_t parts = std::min<int64_t>(std::max<int64_t>(1, 2 * sm / total), most);
  a.heads_block = (int32_t)((a.heads + parts - 1) / parts);
  a.total = (int32_t)total;
  const int64_t work = (int64_t)a.heads_block * items, turns = (work + rotary::kThreads - 1) / rotary::kThreads;
  const bool many = total > 8 * sm;
  a.tokens_block = (int32_t)std::max<int64_t>(1, std::min({rotary::kThreads / work, rotary::kAngles / (int64_t)a.pairs, total / (2 * sm)}));
  const int64_t needed = std::max<int64_t>((work * a.tokens_block + turns - 1) / turns, a.pairs);
  const int threads = many || a.tokens_block > 1 ? (int)((needed + 31) / 32 * 32) : rotary::kThreads;
  const int smem = a.tokens_block * a.pairs * (int)sizeof(float2);
  const dim3 grid((unsigned)((total + a.tokens_block - 1) / a.tokens_block), (unsigned)((a.heads + a.heads_block - 1) / a.heads_block));
  cudaError_t e;
  if (d->dtype == NSA_DTYPE_F32) {
    e = vec == 4   ? launch_rotary<float, 4>(a, grid, threads, smem, st)
        : vec == 2 ? launch_rotary<float, 2>(a, grid, threads, smem, st)
                   : launch_rotary<float, 1>(a, grid, threads, smem, st);
  } else if (d->dtype == NSA_DTYPE_F16) {
    e = vec == 8   ? launch_rotary<__half, 8>(a, grid, threads, smem, st)
        : vec == 4 ? launch_rotary<__half, 4>(a, grid, threads, smem, st)
        : vec == 2 ? launch_rotary<__half, 2>(a, grid, threads, smem, st)
                   : launch_rotary<__half, 1>(a, grid, threads, smem, st);
  } else {
    e = vec == 8   ? launch_rotary<__nv_bfloat16, 8>(a, grid, threads, smem, st)
        : vec == 4 ? launch_rotary<__nv_bfloat16, 4>(a, grid, threads, smem, st)
        : vec == 2 ? launch_rotary<__nv_bfloat16, 2>(a, grid, threads, smem, st)
                   : launch_rotary<__nv_bfloat16, 1>(a, grid, threads, smem, st);
  }
  return done(e, "rotary launch");
}

}  // namespace

extern "C" {

int nsa_cache_reserve(const nsa_cache_reserve_desc* desc, nsa_stream_t stream) {
  return run_reserve(desc, reinterpret_cast<cudaStream_t>(stream));
}

int64_t nsa_cache_select_workspace_bytes(const nsa_cache_select_desc* desc) {
  if (check_select(desc) != NSA_OK) return -1;
  done(cudaSuccess, "");
  // (the rows of one launch: the next one's bounds are written when the last one's have been read)
  const int64_t rows = std::min<int64_t>(desc->batch.n_rows, rows_of_launch(desc));
  return std::max<int64_t>(16, rows * desc->batch.heads_kv * most_blocks(desc) * 8);
}
int nsa_cache_select(const nsa_cache_select_desc* desc, nsa_stream_t stream) {
  return run_select(desc, reinterpret_cast<cudaStream_t>(stream));
}

int nsa_rotary(const nsa_rotary_desc* desc, nsa_stream_t stream) { return run_rotary(desc, reinterpret_cast<cudaStream_t>(stream)); }

}  // extern "C"
