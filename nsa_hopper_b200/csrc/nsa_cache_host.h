// Host helpers that the cache's translation units share: the checks of a batch, its form on the device, programmatic
// launches.
#pragma once
#include <cuda_runtime.h>
#include <algorithm>
#include <string.h>
#include <type_traits>

#include "nsa_cache_index.h"
#include "nsa_host.h"
#include "nsa_sel.h"

namespace nsa {
namespace cache {

using host::cuda_fail;
using host::fail;

constexpr int64_t kMaxIndex = 0x7FFFFFFF;

inline bool misaligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

inline bool dims_built(int32_t d_qk, int32_t d_v) {
  return (d_qk == 64 && d_v == 64) || (d_qk == 128 && (d_v == 128 || d_v == 64)) || (d_qk == 192 && d_v == 128);
}

inline int check_batch(const nsa_cache_batch* b) {
  if (b == nullptr) return fail(NSA_ERR_INVALID_ARG, "batch is NULL");
  if (b->n_rows < 0 || b->n_seqs < 0 || b->width < 0 || b->num_pages < 0 || b->heads_kv <= 0)
    return fail(NSA_ERR_INVALID_ARG, "n_rows, n_seqs, width and num_pages must not be negative, heads_kv must be positive");
  if (!dims_built(b->d_qk, b->d_v))
    return fail(NSA_ERR_UNSUPPORTED, "(d_qk, d_v) = (%d, %d) is not one of (64, 64), (128, 128), (192, 128), (128, 64)", b->d_qk,
                b->d_v);
  if (b->cu_seqlens == nullptr && b->n_rows != b->n_seqs)
    return fail(NSA_ERR_INVALID_ARG, "without cu_seqlens there is one row a sequence: n_rows %d, n_seqs %d", b->n_rows, b->n_seqs);
  if (b->n_rows == 0) return NSA_OK;
  if (b->n_seqs > 0 && (b->lens == nullptr || (b->width > 0 && b->pages == nullptr)))
    return fail(NSA_ERR_INVALID_ARG, "pages and lens must be non-NULL");
  if (b->num_pages > 0 && b->cache == nullptr) return fail(NSA_ERR_INVALID_ARG, "cache must be non-NULL");
  if (misaligned(b->cache, 16)) return fail(NSA_ERR_INVALID_ARG, "cache must be 16-byte aligned");
  if (misaligned(b->pages, 4) || misaligned(b->lens, 4) || misaligned(b->cu_seqlens, 4))
    return fail(NSA_ERR_INVALID_ARG, "pages, lens and cu_seqlens must be aligned to their element size");
  const int64_t page = (int64_t)b->heads_kv * record_bytes(b->d_qk, b->d_v);
  if (b->page_stride != 0 && (b->page_stride < page || b->page_stride % 16 != 0))
    return fail(NSA_ERR_INVALID_ARG, "page_stride must be a multiple of 16 and not below %lld", (long long)page);
  if (b->pages_stride != 0 && b->pages_stride < b->width)
    return fail(NSA_ERR_INVALID_ARG, "pages_stride must not be below width");
  if ((int64_t)b->n_rows * b->heads_kv > kMaxIndex / (b->d_qk / kGroup))
    return fail(NSA_ERR_UNSUPPORTED, "n_rows * heads_kv * d_qk / 16 must be below 2^31");
  return NSA_OK;
}

inline Batch device_batch(const nsa_cache_batch* b) {
  return {b->pages, b->lens, b->cu_seqlens, b->pages_stride ? b->pages_stride : b->width, b->n_seqs, b->width, b->num_pages,
          b->n_rows};
}
inline int64_t page_stride_of(const nsa_cache_batch* b) {
  return b->page_stride ? b->page_stride : (int64_t)b->heads_kv * record_bytes(b->d_qk, b->d_v);
}

// Calls f with the head dims as types' constants.
template <class F>
inline int for_dims(int32_t d_qk, int32_t d_v, F&& f) {
  using std::integral_constant;
  if (d_qk == 64) return f(integral_constant<int, 64>(), integral_constant<int, 64>());
  if (d_qk == 192) return f(integral_constant<int, 192>(), integral_constant<int, 128>());
  if (d_v == 128) return f(integral_constant<int, 128>(), integral_constant<int, 128>());
  return f(integral_constant<int, 128>(), integral_constant<int, 64>());
}

inline int done(cudaError_t e, const char* what) {
  if (e != cudaSuccess) return cuda_fail(e, what);
  return fail(NSA_OK, "%s", "");
}

// A programmatic launch (see start_in_order), in clusters of `cluster` blocks.
template <class Args>
inline cudaError_t launch(void (*kernel)(Args), dim3 grid, int threads, int smem, int cluster, cudaStream_t st, const Args& a) {
  cudaLaunchAttribute attr[2];
  memset(attr, 0, sizeof(attr));
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

}  // namespace cache
}  // namespace nsa
