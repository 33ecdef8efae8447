// Host side of the 4-bit paged KV cache (nsa_cache_* in include/nsa_sel.h): checks, the attention's plan and
// the launches.
#include <cuda_runtime.h>
#include <math.h>
#include <algorithm>
#include <mutex>
#include <string.h>

#include "nsa_sel.h"
#include "nsa_cache_host.h"
#include "nsa_cache_kernel.cuh"

namespace {

using nsa::cache::AttendArgs;
using nsa::cache::CfgFor;
using nsa::cache::check_batch;
using nsa::cache::device_batch;
using nsa::cache::dims_built;
using nsa::cache::done;
using nsa::cache::for_dims;
using nsa::cache::kMaxIndex;
using nsa::cache::launch;
using nsa::cache::misaligned;
using nsa::cache::page_stride_of;
using nsa::host::cuda_fail;
using nsa::host::fail;

// ------------------------------------------------------------------ attention
// A KV head's G query heads: one tile of 8, or tiles of 16.
int tiles_of(int group) { return group <= 8 ? 1 : (group + 15) / 16; }

// Calls f with the attention's configuration for a checked description.
template <class F>
int for_config(const nsa_cache_attend_desc* d, F&& f) {
  return for_dims(d->batch.d_qk, d->batch.d_v, [&](auto dqk, auto dv) {
    constexpr int kQk = decltype(dqk)::value, kV = decltype(dv)::value;
    return d->heads_q / d->batch.heads_kv <= 8 ? f(CfgFor<kQk, kV, 1>()) : f(CfgFor<kQk, kV, 2>());
  });
}

// Slots (64-key sub-blocks) of a row and KV head, at most.
int64_t most_slots(const nsa_cache_attend_desc* d) {
  if (d->sel != nullptr) return (int64_t)d->n_sel * (d->block_size / 64);
  const int64_t all = std::max(d->batch.width, 1);
  return d->window > 0 ? std::min<int64_t>(all, ((int64_t)d->window + 62) / 64 + 1) : all;
}

int check_attend(const nsa_cache_attend_desc* d) {
  if (d == nullptr) return fail(NSA_ERR_INVALID_ARG, "desc is NULL");
  int rc = check_batch(&d->batch);
  if (rc != NSA_OK) return rc;
  const nsa_cache_batch& b = d->batch;
  if (d->heads_q <= 0 || d->heads_q % b.heads_kv != 0)
    return fail(NSA_ERR_INVALID_ARG, "heads_q (%d) must be a positive multiple of heads_kv (%d)", d->heads_q, b.heads_kv);
  if (d->q_dtype != NSA_DTYPE_BF16 && d->q_dtype != NSA_DTYPE_F16)
    return fail(NSA_ERR_INVALID_ARG, "q_dtype must be NSA_DTYPE_BF16 or NSA_DTYPE_F16");
  if (d->o_dtype != d->q_dtype && d->o_dtype != NSA_DTYPE_F32)
    return fail(NSA_ERR_INVALID_ARG, "o_dtype must be q_dtype or NSA_DTYPE_F32");
  if (d->o_accumulate && d->o_dtype != NSA_DTYPE_F32) return fail(NSA_ERR_INVALID_ARG, "o_accumulate needs an fp32 O");
  if (d->window < 0) return fail(NSA_ERR_INVALID_ARG, "window must not be negative");
  if (d->sel != nullptr) {
    if (d->n_sel <= 0) return fail(NSA_ERR_INVALID_ARG, "n_sel must be positive");
    if (d->block_size != 64 && d->block_size != 128 && d->block_size != 256)
      return fail(NSA_ERR_UNSUPPORTED, "block_size must be 64, 128 or 256");
    if (d->n_sel > 1024) return fail(NSA_ERR_UNSUPPORTED, "n_sel must be at most 1024");
  }
  if (b.n_rows == 0) return NSA_OK;
  const int64_t rows = (int64_t)b.n_rows * b.heads_kv * tiles_of(d->heads_q / b.heads_kv);
  if (rows > kMaxIndex / 2 || rows * most_slots(d) > kMaxIndex)
    return fail(NSA_ERR_UNSUPPORTED, "n_rows * heads_kv * (pages that a row can see) must be below 2^31");
  if (d->q == nullptr || d->o == nullptr) return fail(NSA_ERR_INVALID_ARG, "q and o must be non-NULL");
  if (misaligned(d->q, 16) || misaligned(d->o, 16) || d->q_row_stride % 8 != 0 || d->q_head_stride % 8 != 0)
    return fail(NSA_ERR_INVALID_ARG, "q and o must be 16-byte aligned and q's strides multiples of 8");
  if (misaligned(d->sel, 4) || misaligned(d->lse, 4) || misaligned(d->o_weight, 4) || misaligned(d->err, 4))
    return fail(NSA_ERR_INVALID_ARG, "sel, lse, o_weight and err must be aligned to their element size");
  return NSA_OK;
}

// Splits the call's slots (checked description, n_rows > 0).
template <class C>
int plan_attend(const nsa_cache_attend_desc* d, int sm_count, nsa_cache_attend_plan_info* p) {
  const nsa_cache_batch& b = d->batch;
  const int group = d->heads_q / b.heads_kv;
  p->tiles = tiles_of(group);
  const uint32_t most = (uint32_t)most_slots(d), rows = (uint32_t)b.n_rows * b.heads_kv * p->tiles;
  const uint32_t warps = (uint32_t)sm_count * C::NW;
  p->cluster = (int32_t)nsa::cache::cluster_of(rows, most, warps);
  // The ragged line is for rows that may have to be cut by their real lengths.
  const bool ragged = d->sel == nullptr && d->window == 0 && b.n_rows <= C::kMaxRagged && p->cluster == 1 &&
                      nsa::cache::may_cut(rows, most, warps);
  const nsa::cache::Split s = nsa::cache::split_line(rows, rows * most, most, warps);
  p->slots = ragged ? 0 : (int32_t)most;
  bool cut = ragged;
  uint32_t teams;  // with a share of their own, at most
  if (ragged) {
    teams = (uint32_t)std::min<uint64_t>(warps, (uint64_t)rows * most);
  } else if (p->cluster > 1) {
    p->team = nsa::cache::kTeam;
    p->share = 1;
    teams = rows;
  } else {
    cut = s.cut != 0;
    p->team = (int32_t)s.team;
    p->share = (int32_t)s.share;
    teams = nsa::cache::ceil_div(cut ? rows * most : rows, s.share);
  }
  p->grid = p->cluster > 1 ? (int32_t)(rows * p->cluster) : (int32_t)std::min<uint32_t>(sm_count, teams);
  p->threads = C::NW * 32;
  p->smem_bytes = C::kSmem;
  // Eight warps for each query head while the device has room for them at once (8 blocks an SM), else one: rows that are
  // few have many parts.
  p->merge = !cut ? 0 : (int64_t)b.n_rows * d->heads_q <= 8ll * sm_count ? 8 : 1;
  p->workspace_bytes = cut ? ((int64_t)(b.n_rows + 2) * 4 + 15) / 16 * 16 + (int64_t)teams * 2 * C::kPart * 4 : 16;
  return NSA_OK;
}

int plan(const nsa_cache_attend_desc* d, int sm_count, nsa_cache_attend_plan_info* p) {
  memset(p, 0, sizeof(*p));
  int rc = check_attend(d);
  if (rc != NSA_OK) return rc;
  if (d->batch.n_rows == 0) {
    p->workspace_bytes = 16;
    return NSA_OK;
  }
  return for_config(d, [&](auto cfg) { return plan_attend<decltype(cfg)>(d, sm_count, p); });
}

std::mutex g_mu;
uint32_t g_attr_done[nsa::host::kMaxDevices] = {};  // one bit for each attention kernel

template <class C>
int launch_attend(const AttendArgs& a, const nsa_cache_attend_plan_info& p, int dev, cudaStream_t st) {
  {
    std::lock_guard<std::mutex> lk(g_mu);
    const uint32_t bit = 1u << ((C::DQK + C::DV) / 64 * 2 + C::NH);
    if ((g_attr_done[dev] & bit) == 0) {
      const cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(&nsa::cache::attend_kernel<C>),
                                                 cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
      if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(cache attention smem)");
      g_attr_done[dev] |= bit;
    }
  }
  cudaError_t e = launch(&nsa::cache::attend_kernel<C>, dim3((unsigned)p.grid), p.threads, C::kSmem, p.cluster, st, a);
  if (e != cudaSuccess || p.merge == 0) return done(e, "cache attention launch");
  const int64_t units = (int64_t)a.b.n_rows * a.hq;
  e = p.merge == 1 ? launch(&nsa::cache::merge_kernel<C, 1>, dim3((unsigned)((units + 7) / 8)), 256, 0, 1, st, a)
                   : launch(&nsa::cache::merge_kernel<C, 8>, dim3((unsigned)units), 256, 0, 1, st, a);
  return done(e, "cache attention's merge launch");
}

int attend(const nsa_cache_attend_desc* d, cudaStream_t st) {
  int rc = check_attend(d);
  if (rc != NSA_OK) return rc;
  if (d->batch.n_rows == 0) return done(cudaSuccess, "");
  int sm = 0, dev = 0;
  rc = nsa::host::current_sm_count(&sm, &dev);
  if (rc != NSA_OK) return rc;
  nsa_cache_attend_plan_info p;
  rc = plan(d, sm, &p);
  if (rc != NSA_OK) return rc;
  if (p.merge != 0 && (d->workspace == nullptr || misaligned(d->workspace, 16)))
    return fail(NSA_ERR_INVALID_ARG, "workspace must be non-NULL and 16-byte aligned");
  const nsa_cache_batch& b = d->batch;
  AttendArgs a;
  memset(&a, 0, sizeof(a));
  a.b = device_batch(&b);
  a.q = d->q;
  a.q_row = d->q_row_stride ? d->q_row_stride : (int64_t)d->heads_q * b.d_qk;
  a.q_head = d->q_head_stride ? d->q_head_stride : b.d_qk;
  a.cache = static_cast<const uint8_t*>(b.cache);
  a.page_stride = page_stride_of(&b);
  a.sel = d->sel;
  a.o = d->o;
  a.lse = d->lse;
  a.weight = d->o_weight;
  a.starts = static_cast<uint32_t*>(d->workspace);
  a.part = p.merge == 0 ? nullptr
                        : reinterpret_cast<float*>(static_cast<uint8_t*>(d->workspace) + ((int64_t)(b.n_rows + 2) * 4 + 15) / 16 * 16);
  a.hq = d->heads_q;
  a.hkv = b.heads_kv;
  a.group = d->heads_q / b.heads_kv;
  a.tiles = p.tiles;
  a.n_sel = d->n_sel;
  a.per = d->sel != nullptr ? d->block_size / 64 : 1;
  a.window = d->window;
  a.slots = p.slots;
  a.warps = (uint32_t)sm * (uint32_t)(p.threads / 32);
  a.split = {(uint32_t)p.team, (uint32_t)p.share, p.merge != 0};
  a.cluster = (uint32_t)p.cluster;
  a.q_half = d->q_dtype == NSA_DTYPE_F16;
  a.o_dtype = d->o_dtype;
  a.accumulate = d->o_accumulate != 0;
  a.fill = d->keep_rows == 0;
  a.scale_log2 = (float)((d->scale > 0.0f ? (double)d->scale : 1.0 / sqrt((double)b.d_qk)) * 1.4426950408889634074);
  a.err = d->err;
  a.wait_ns = (uint64_t)(d->timeout_ms > 0 ? d->timeout_ms : 2000) * 1000000u;
  a.stall = (d->debug_flags & NSA_DEBUG_STALL) != 0;
  return for_config(d, [&](auto cfg) { return launch_attend<decltype(cfg)>(a, p, dev, st); });
}

}  // namespace

extern "C" {

int64_t nsa_cache_record_bytes(int32_t d_qk, int32_t d_v) {
  if (!dims_built(d_qk, d_v)) return -1;
  return nsa::cache::record_bytes(d_qk, d_v);
}

int nsa_cache_write(const nsa_cache_batch* b, const void* k, const void* v, int64_t k_row_stride, int64_t k_head_stride,
                    int64_t v_row_stride, int64_t v_head_stride, int32_t in_dtype, nsa_stream_t stream) {
  int rc = check_batch(b);
  if (rc != NSA_OK) return rc;
  if (in_dtype != NSA_DTYPE_BF16 && in_dtype != NSA_DTYPE_F16)
    return fail(NSA_ERR_INVALID_ARG, "in_dtype must be NSA_DTYPE_BF16 or NSA_DTYPE_F16");
  if (b->n_rows == 0) return done(cudaSuccess, "");
  if (k == nullptr || v == nullptr) return fail(NSA_ERR_INVALID_ARG, "k and v must be non-NULL");
  if (misaligned(k, 16) || misaligned(v, 16) || ((k_row_stride | k_head_stride | v_row_stride | v_head_stride) & 7) != 0)
    return fail(NSA_ERR_INVALID_ARG, "k and v must be 16-byte aligned and their strides multiples of 8");
  int sm = 0, dev = 0;
  rc = nsa::host::current_sm_count(&sm, &dev);
  if (rc != NSA_OK) return rc;
  const nsa::cache::WriteArgs a = {device_batch(b), {k, v}, {k_row_stride, v_row_stride}, {k_head_stride, v_head_stride},
                                   static_cast<uint8_t*>(b->cache), page_stride_of(b), b->heads_kv, in_dtype == NSA_DTYPE_F16};
  const int64_t threads = (int64_t)b->n_rows * b->heads_kv * std::max(b->d_qk, b->d_v) / (2 * nsa::cache::kGroup);
  return for_dims(b->d_qk, b->d_v, [&](auto dqk, auto dv) {
    return done(launch(&nsa::cache::write_kernel<decltype(dqk)::value, decltype(dv)::value>, dim3((unsigned)((threads + 255) / 256), 2),
                       256, 0, 1, reinterpret_cast<cudaStream_t>(stream), a),
                "cache write launch");
  });
}

int nsa_cache_read(const nsa_cache_batch* b, void* k, void* v, int32_t out_dtype, nsa_stream_t stream) {
  int rc = check_batch(b);
  if (rc != NSA_OK) return rc;
  if (out_dtype != NSA_DTYPE_BF16 && out_dtype != NSA_DTYPE_F16 && out_dtype != NSA_DTYPE_F32)
    return fail(NSA_ERR_INVALID_ARG, "out_dtype must be NSA_DTYPE_BF16, NSA_DTYPE_F16 or NSA_DTYPE_F32");
  if (b->n_rows == 0) return done(cudaSuccess, "");
  if (k == nullptr || v == nullptr) return fail(NSA_ERR_INVALID_ARG, "k and v must be non-NULL");
  if (misaligned(k, 32) || misaligned(v, 32)) return fail(NSA_ERR_INVALID_ARG, "k and v must be 32-byte aligned");
  int sm = 0, dev = 0;
  rc = nsa::host::current_sm_count(&sm, &dev);
  if (rc != NSA_OK) return rc;
  const nsa::cache::ReadArgs a = {device_batch(b), static_cast<const uint8_t*>(b->cache), page_stride_of(b), {k, v}, b->heads_kv,
                                  out_dtype};
  const int64_t groups = (int64_t)b->n_rows * b->heads_kv * std::max(b->d_qk, b->d_v) / nsa::cache::kGroup;
  return for_dims(b->d_qk, b->d_v, [&](auto dqk, auto dv) {
    constexpr int kQk = decltype(dqk)::value, kV = decltype(dv)::value;
    const int items = groups > 32ll * 256 * sm ? 2 : 1;  // (the border: 32 blocks an SM)
    return done(launch(items == 2 ? &nsa::cache::read_kernel<kQk, kV, 2> : &nsa::cache::read_kernel<kQk, kV, 1>,
                       dim3((unsigned)((groups + 256 * items - 1) / (256 * items)), 2), 256, 0, 1,
                       reinterpret_cast<cudaStream_t>(stream), a),
                "cache read launch");
  });
}

int nsa_cache_attend_plan(const nsa_cache_attend_desc* desc, int32_t sm_count, nsa_cache_attend_plan_info* out) {
  if (out == nullptr) return fail(NSA_ERR_INVALID_ARG, "out is NULL");
  int sm = sm_count, dev = 0;
  if (sm <= 0) {
    const int rc = nsa::host::current_sm_count(&sm, &dev);
    if (rc != NSA_OK) return rc;
  }
  const int rc = plan(desc, sm, out);
  return rc != NSA_OK ? rc : done(cudaSuccess, "");
}

int64_t nsa_cache_attend_workspace_bytes(const nsa_cache_attend_desc* desc) {
  nsa_cache_attend_plan_info p;
  return nsa_cache_attend_plan(desc, 0, &p) == NSA_OK ? p.workspace_bytes : -1;
}

int nsa_cache_attend(const nsa_cache_attend_desc* desc, nsa_stream_t stream) {
  return attend(desc, reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
