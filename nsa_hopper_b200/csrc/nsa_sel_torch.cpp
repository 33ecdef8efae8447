// PyTorch extension with the reference's op signature, over the C ABI of libnsa_sel.so.
//
//   forward(Q, K, V, sel, l_prime, BQ, cyc) -> O (fp32)
//       same arguments, meaning and errors as the reference's pybind op
//       (nsa_v2.cu:147-170, nsa_v1.cu:125-147, nsa_v0.cu:118-146): Q [B,Hq,S,D] bf16,
//       K/V [B,Hkv,S,D] bf16, sel int32 [B,Hkv,NQB,KSEL], cyc int64 [NQB*B*Hkv*2] or empty.
//       Unsupported shapes raise RuntimeError (TORCH_CHECK), as in the reference.
//   forward_lse(Q, K, V, sel, l_prime, BQ, cu_seqlens=None, scale=0, out_f32=False)
//       -> (O bf16 (or fp32), LSE fp32 [B,Hq,T]); d_qk may differ from d_v; optional varlen.
//
// The translation unit holds no device code, so it also builds when a harness compiles it
// with the reference's flags (e.g. `-arch=sm_90a`).  libnsa_sel.so is opened at first use
// from the directory of this extension, or from the package directory next to this source.
#include <dlfcn.h>
#include <torch/extension.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <limits>
#include <mutex>
#include <string>

#include "../../include/nsa_sel.h"

namespace {

// Error text is formatted into a per-thread buffer and raised through the `const char*` form
// of TORCH_CHECK: no std::string crosses into libtorch, so the message survives translation
// units that a harness compiles with its own flags (e.g. nvcc host code in a JIT build).
thread_local char g_msg[768];

const char* format_msg(const char* f, ...) {
  va_list ap;
  va_start(ap, f);
  vsnprintf(g_msg, sizeof(g_msg), f, ap);
  va_end(ap);
  return g_msg;
}

struct Api {
  decltype(&nsa_sel_forward) forward = nullptr;
  decltype(&nsa_sel_run) run = nullptr;
  decltype(&nsa_sel_last_error) last_error = nullptr;
  decltype(&nsa_sel_version) version = nullptr;
  decltype(&nsa_sel_select) select = nullptr;
  decltype(&nsa_sel_select_workspace_bytes) select_ws = nullptr;
  decltype(&nsa_cache_record_bytes) cache_record = nullptr;
  decltype(&nsa_cache_write) cache_write = nullptr;
  decltype(&nsa_cache_read) cache_read = nullptr;
  decltype(&nsa_cache_attend) cache_attend = nullptr;
  decltype(&nsa_cache_attend_workspace_bytes) cache_attend_ws = nullptr;
  decltype(&nsa_cache_reserve) cache_reserve = nullptr;
  decltype(&nsa_cache_select) cache_select = nullptr;
  decltype(&nsa_cache_select_workspace_bytes) cache_select_ws = nullptr;
  decltype(&nsa_rotary) rotary = nullptr;
};

std::string dir_of(const std::string& path) {
  const size_t p = path.find_last_of('/');
  return p == std::string::npos ? std::string(".") : path.substr(0, p);
}

const Api& api() {
  static Api a;
  static std::once_flag once;
  static std::string error;
  std::call_once(once, [] {
    std::string candidates[3];
    Dl_info info;
    if (dladdr(reinterpret_cast<void*>(&dir_of), &info) != 0 && info.dli_fname != nullptr)
      candidates[0] = dir_of(info.dli_fname) + "/libnsa_sel.so";
    candidates[1] = dir_of(dir_of(__FILE__)) + "/libnsa_sel.so";  // <pkg>/csrc/.. = <pkg>
    if (const char* env = getenv("NSA_SEL_LIBRARY")) candidates[2] = env;
    void* h = nullptr;
    for (const std::string& c : candidates) {
      if (c.empty()) continue;
      h = dlopen(c.c_str(), RTLD_NOW | RTLD_LOCAL);
      if (h != nullptr) break;
      error += c + ": " + dlerror() + "; ";
    }
    if (h == nullptr) return;
    a.forward = reinterpret_cast<decltype(a.forward)>(dlsym(h, "nsa_sel_forward"));
    a.run = reinterpret_cast<decltype(a.run)>(dlsym(h, "nsa_sel_run"));
    a.last_error = reinterpret_cast<decltype(a.last_error)>(dlsym(h, "nsa_sel_last_error"));
    a.version = reinterpret_cast<decltype(a.version)>(dlsym(h, "nsa_sel_version"));
    a.select = reinterpret_cast<decltype(a.select)>(dlsym(h, "nsa_sel_select"));
    a.select_ws = reinterpret_cast<decltype(a.select_ws)>(dlsym(h, "nsa_sel_select_workspace_bytes"));
    a.cache_record = reinterpret_cast<decltype(a.cache_record)>(dlsym(h, "nsa_cache_record_bytes"));
    a.cache_write = reinterpret_cast<decltype(a.cache_write)>(dlsym(h, "nsa_cache_write"));
    a.cache_read = reinterpret_cast<decltype(a.cache_read)>(dlsym(h, "nsa_cache_read"));
    a.cache_attend = reinterpret_cast<decltype(a.cache_attend)>(dlsym(h, "nsa_cache_attend"));
    a.cache_attend_ws = reinterpret_cast<decltype(a.cache_attend_ws)>(dlsym(h, "nsa_cache_attend_workspace_bytes"));
    a.cache_reserve = reinterpret_cast<decltype(a.cache_reserve)>(dlsym(h, "nsa_cache_reserve"));
    a.cache_select = reinterpret_cast<decltype(a.cache_select)>(dlsym(h, "nsa_cache_select"));
    a.cache_select_ws = reinterpret_cast<decltype(a.cache_select_ws)>(dlsym(h, "nsa_cache_select_workspace_bytes"));
    a.rotary = reinterpret_cast<decltype(a.rotary)>(dlsym(h, "nsa_rotary"));
  });
  if (!(a.forward && a.run && a.last_error && a.version && a.select && a.select_ws && a.cache_record && a.cache_write &&
        a.cache_read && a.cache_attend && a.cache_attend_ws && a.cache_reserve && a.cache_select && a.cache_select_ws && a.rotary))
    TORCH_CHECK(false, format_msg("libnsa_sel.so could not be loaded (build it first): %s", error.c_str()));
  return a;
}

void check_inputs(const torch::Tensor& Q, const torch::Tensor& K, const torch::Tensor& V, const torch::Tensor& sel) {
  TORCH_CHECK(Q.is_cuda() && K.is_cuda() && V.is_cuda() && sel.is_cuda(), "Q, K, V and sel must be CUDA tensors");
  TORCH_CHECK(Q.scalar_type() == at::kBFloat16 && K.scalar_type() == at::kBFloat16 &&
                  V.scalar_type() == at::kBFloat16,
              "Q, K and V must be bfloat16");
  TORCH_CHECK(sel.scalar_type() == at::kInt, "sel must be int32");
  TORCH_CHECK(Q.dim() == 4 && K.dim() == 4 && V.dim() == 4 && sel.dim() == 4,
              "expected Q/K/V [B,H,S,D] and sel [B,Hkv,NQB,KSEL]");
  TORCH_CHECK(Q.is_contiguous() && K.is_contiguous() && V.is_contiguous() && sel.is_contiguous(),
              "Q, K, V and sel must be contiguous");
  TORCH_CHECK(K.size(0) == Q.size(0) && V.size(0) == Q.size(0) && sel.size(0) == Q.size(0), "batch mismatch");
  TORCH_CHECK(K.size(2) == Q.size(2) && V.size(2) == Q.size(2), "sequence length mismatch");
  TORCH_CHECK(V.size(1) == K.size(1) && sel.size(1) == K.size(1), "KV head count mismatch");
  TORCH_CHECK(K.size(3) == Q.size(3), "Q and K head dims differ");
  TORCH_CHECK(K.get_device() == Q.get_device() && V.get_device() == Q.get_device() &&
                  sel.get_device() == Q.get_device(),
              "all tensors must be on one device");
}

int32_t i32(int64_t x, const char* what) {
  if (!(x >= 0 && x < (int64_t(1) << 31))) TORCH_CHECK(false, format_msg("%s out of int32 range", what));
  return static_cast<int32_t>(x);
}

torch::Tensor forward(torch::Tensor Q, torch::Tensor K, torch::Tensor V, torch::Tensor sel, int64_t l_prime,
                      int64_t BQ, torch::Tensor cyc) {
  check_inputs(Q, K, V, sel);
  TORCH_CHECK(V.size(3) == Q.size(3), "forward() needs d_v == d_qk (use forward_lse for d_qk != d_v)");
  const Api& a = api();
  const c10::cuda::CUDAGuard guard(Q.device());
  auto O = torch::empty({Q.size(0), Q.size(1), Q.size(2), V.size(3)}, Q.options().dtype(torch::kFloat32));
  int64_t* cyc_ptr = nullptr;
  if (cyc.defined() && cyc.numel() > 0) {
    TORCH_CHECK(cyc.is_cuda() && cyc.scalar_type() == at::kLong && cyc.is_contiguous(), "cyc must be CUDA int64");
    TORCH_CHECK(cyc.numel() >= sel.size(2) * sel.size(0) * sel.size(1) * 2, "cyc must hold NQB*B*Hkv*2 entries");
    cyc_ptr = cyc.data_ptr<int64_t>();
  }
  const int rc = a.forward(Q.data_ptr(), K.data_ptr(), V.data_ptr(), sel.data_ptr<int32_t>(), O.data_ptr<float>(),
                           cyc_ptr, i32(Q.size(0), "B"), i32(Q.size(1), "Hq"), i32(K.size(1), "Hkv"),
                           i32(Q.size(2), "S"), i32(Q.size(3), "D"), i32(sel.size(2), "NQB"),
                           i32(sel.size(3), "KSEL"), i32(l_prime, "l_prime"), i32(BQ, "BQ"),
                           reinterpret_cast<nsa_stream_t>(c10::cuda::getCurrentCUDAStream().stream()));
  if (rc != NSA_OK) TORCH_CHECK(false, format_msg("nsa_sel_forward failed (%d): %s", rc, a.last_error()));
  return O;
}

std::vector<torch::Tensor> forward_lse(torch::Tensor Q, torch::Tensor K, torch::Tensor V, torch::Tensor sel,
                                       int64_t l_prime, int64_t BQ, c10::optional<torch::Tensor> cu_seqlens,
                                       double scale, bool out_f32) {
  check_inputs(Q, K, V, sel);
  const Api& a = api();
  const c10::cuda::CUDAGuard guard(Q.device());
  auto O = torch::empty({Q.size(0), Q.size(1), Q.size(2), V.size(3)},
                        Q.options().dtype(out_f32 ? torch::kFloat32 : torch::kBFloat16));
  auto L = torch::empty({Q.size(0), Q.size(1), Q.size(2)}, Q.options().dtype(torch::kFloat32));
  nsa_sel_desc d;
  memset(&d, 0, sizeof(d));
  d.q = Q.data_ptr();
  d.k = K.data_ptr();
  d.v = V.data_ptr();
  d.sel = sel.data_ptr<int32_t>();
  if (cu_seqlens.has_value() && cu_seqlens->defined()) {
    const auto& cu = *cu_seqlens;
    TORCH_CHECK(cu.is_cuda() && cu.scalar_type() == at::kInt && cu.dim() == 1 && cu.is_contiguous(),
                "cu_seqlens must be a contiguous CUDA int32 vector");
    d.cu_seqlens = cu.data_ptr<int32_t>();
    d.n_seqs = i32(cu.numel() - 1, "n_seqs");
  }
  d.o = O.data_ptr();
  d.lse = L.data_ptr<float>();
  d.batch = i32(Q.size(0), "B");
  d.heads_q = i32(Q.size(1), "Hq");
  d.heads_kv = i32(K.size(1), "Hkv");
  d.seq_len = i32(Q.size(2), "T");
  d.d_qk = i32(Q.size(3), "d_qk");
  d.d_v = i32(V.size(3), "d_v");
  d.n_qblocks = i32(sel.size(2), "NQB");
  d.n_sel = i32(sel.size(3), "KSEL");
  d.block_size = i32(l_prime, "l_prime");
  d.q_block = i32(BQ, "BQ");
  d.o_dtype = out_f32 ? NSA_DTYPE_F32 : NSA_DTYPE_BF16;
  d.scale = static_cast<float>(scale);
  const int rc = a.run(&d, reinterpret_cast<nsa_stream_t>(c10::cuda::getCurrentCUDAStream().stream()));
  if (rc != NSA_OK) TORCH_CHECK(false, format_msg("nsa_sel_run failed (%d): %s", rc, a.last_error()));
  return {O, L};
}

// Forward with the extended key visibility of nsa_sel_desc (window, compressed key map; K/V may
// have kv_len != T rows with the compressed map): returns [O (fp32), LSE].
std::vector<torch::Tensor> forward_ext(torch::Tensor Q, torch::Tensor K, torch::Tensor V, torch::Tensor sel,
                                       int64_t l_prime, int64_t BQ, int64_t window, int64_t key_map, double scale,
                                       c10::optional<torch::Tensor> out, c10::optional<torch::Tensor> weight,
                                       bool accumulate, bool with_lse) {
  TORCH_CHECK(Q.is_cuda() && K.is_cuda() && V.is_cuda() && sel.is_cuda(), "Q, K, V and sel must be CUDA tensors");
  TORCH_CHECK(Q.scalar_type() == at::kBFloat16 && K.scalar_type() == at::kBFloat16 &&
                  V.scalar_type() == at::kBFloat16,
              "Q, K and V must be bfloat16");
  TORCH_CHECK(sel.scalar_type() == at::kInt, "sel must be int32");
  TORCH_CHECK(Q.dim() == 4 && K.dim() == 4 && V.dim() == 4 && sel.dim() == 4,
              "expected Q [B,Hq,T,d], K/V [B,Hkv,kv_len,d] and sel [B,Hkv,NQB,KSEL]");
  TORCH_CHECK(Q.is_contiguous() && K.is_contiguous() && V.is_contiguous() && sel.is_contiguous(),
              "Q, K, V and sel must be contiguous");
  TORCH_CHECK(K.size(0) == Q.size(0) && V.size(0) == Q.size(0) && sel.size(0) == Q.size(0), "batch mismatch");
  TORCH_CHECK(V.size(2) == K.size(2) && V.size(1) == K.size(1) && sel.size(1) == K.size(1), "K/V shape mismatch");
  TORCH_CHECK(K.size(3) == Q.size(3), "Q and K head dims differ");
  const Api& a = api();
  const c10::cuda::CUDAGuard guard(Q.device());
  torch::Tensor O;
  if (out.has_value()) {
    O = *out;
    TORCH_CHECK(O.is_cuda() && O.scalar_type() == at::kFloat && O.is_contiguous() && O.get_device() == Q.get_device(),
                "out must be a contiguous fp32 CUDA tensor on Q's device");
    TORCH_CHECK(O.dim() == 4 && O.size(0) == Q.size(0) && O.size(1) == Q.size(1) && O.size(2) == Q.size(2) &&
                    O.size(3) == V.size(3),
                "out must be [B, Hq, T, d_v]");
  } else {
    TORCH_CHECK(!accumulate, "accumulate needs an out tensor");
    O = torch::empty({Q.size(0), Q.size(1), Q.size(2), V.size(3)}, Q.options().dtype(torch::kFloat32));
  }
  if (weight.has_value())
    TORCH_CHECK(weight->is_cuda() && weight->scalar_type() == at::kFloat && weight->numel() >= 1 &&
                    weight->get_device() == Q.get_device(),
                "weight must be an fp32 CUDA tensor (its first element is used) on Q's device");
  torch::Tensor L = with_lse ? torch::empty({Q.size(0), Q.size(1), Q.size(2)}, Q.options().dtype(torch::kFloat32))
                             : torch::empty({0}, Q.options().dtype(torch::kFloat32));
  nsa_sel_desc d;
  memset(&d, 0, sizeof(d));
  d.q = Q.data_ptr();
  d.k = K.data_ptr();
  d.v = V.data_ptr();
  d.sel = sel.data_ptr<int32_t>();
  d.o = O.data_ptr();
  d.lse = with_lse ? L.data_ptr<float>() : nullptr;
  d.o_accumulate = accumulate ? 1 : 0;
  d.o_weight = weight.has_value() ? weight->data_ptr<float>() : nullptr;
  d.batch = i32(Q.size(0), "B");
  d.heads_q = i32(Q.size(1), "Hq");
  d.heads_kv = i32(K.size(1), "Hkv");
  d.seq_len = i32(Q.size(2), "T");
  d.kv_len = i32(K.size(2), "kv_len");
  d.d_qk = i32(Q.size(3), "d_qk");
  d.d_v = i32(V.size(3), "d_v");
  d.n_qblocks = i32(sel.size(2), "NQB");
  d.n_sel = i32(sel.size(3), "KSEL");
  d.block_size = i32(l_prime, "l_prime");
  d.q_block = i32(BQ, "BQ");
  d.window = i32(window, "window");
  d.key_map = i32(key_map, "key_map");
  d.o_dtype = NSA_DTYPE_F32;
  d.scale = static_cast<float>(scale);
  const int rc = a.run(&d, reinterpret_cast<nsa_stream_t>(c10::cuda::getCurrentCUDAStream().stream()));
  if (rc != NSA_OK) TORCH_CHECK(false, format_msg("nsa_sel_run failed (%d): %s", rc, a.last_error()));
  return {O, L};
}

// Block selection (nsa_sel_select): sel int32 [B, Hkv, T, min(n_sel, ceil(T/l_prime))].
torch::Tensor select_blocks(torch::Tensor Q, torch::Tensor K, int64_t n_sel, int64_t l_prime, int64_t cmp_block,
                            int64_t cmp_stride) {
  TORCH_CHECK(Q.is_cuda() && K.is_cuda(), "Q and K must be CUDA tensors");
  TORCH_CHECK(Q.scalar_type() == at::kBFloat16 && K.scalar_type() == at::kBFloat16, "Q and K must be bfloat16");
  TORCH_CHECK(Q.dim() == 4 && K.dim() == 4, "expected Q [B,Hq,T,d] and K [B,Hkv,T,d]");
  TORCH_CHECK(Q.is_contiguous() && K.is_contiguous(), "Q and K must be contiguous");
  TORCH_CHECK(K.size(0) == Q.size(0) && K.size(2) == Q.size(2) && K.size(3) == Q.size(3), "Q/K shape mismatch");
  const Api& a = api();
  const c10::cuda::CUDAGuard guard(Q.device());
  const int32_t B = i32(Q.size(0), "B"), Hq = i32(Q.size(1), "Hq"), Hkv = i32(K.size(1), "Hkv");
  const int32_t T = i32(Q.size(2), "T"), d = i32(Q.size(3), "d"), lp = i32(l_prime, "l_prime");
  const int64_t ws = a.select_ws(B, Hkv, T, d, lp);
  if (ws < 0) TORCH_CHECK(false, "invalid selection shape");
  const int64_t n_blk = (T + lp - 1) / lp;
  const int64_t k = std::min<int64_t>(n_sel, n_blk);
  auto work = torch::empty({std::max<int64_t>(ws / 4, 1)}, Q.options().dtype(torch::kFloat32));
  auto sel = torch::empty({Q.size(0), K.size(1), Q.size(2), std::max<int64_t>(k, 1)}, Q.options().dtype(torch::kInt));
  const int rc = a.select(Q.data_ptr(), K.data_ptr(), work.data_ptr<float>(), sel.data_ptr<int32_t>(), B, Hq, Hkv, T, d,
                          lp, i32(n_sel, "n_sel"), i32(cmp_block, "cmp_block"), i32(cmp_stride, "cmp_stride"),
                          reinterpret_cast<nsa_stream_t>(c10::cuda::getCurrentCUDAStream().stream()));
  if (rc != NSA_OK) TORCH_CHECK(false, format_msg("nsa_sel_select failed (%d): %s", rc, a.last_error()));
  return sel;
}

// ------------------------------------------------------------------ the 4-bit paged KV cache
using OptTensor = c10::optional<torch::Tensor>;

nsa_stream_t current_stream() { return reinterpret_cast<nsa_stream_t>(c10::cuda::getCurrentCUDAStream().stream()); }

int32_t dtype_code(const torch::Tensor& t, const char* name) {
  if (t.scalar_type() == at::kBFloat16) return NSA_DTYPE_BF16;
  if (t.scalar_type() != at::kHalf) TORCH_CHECK(false, format_msg("%s must be bfloat16 or float16", name));
  return NSA_DTYPE_F16;
}

// Strides as the kernels take them: unit along the last dim; a dim of one element has none that counts.
int64_t stride_of(const torch::Tensor& t, int64_t dim) { return t.size(dim) > 1 ? t.stride(dim) : 0; }

void check_rows(const torch::Tensor& t, const char* name) {
  if (!(t.stride(2) == 1 && stride_of(t, 0) % 8 == 0 && stride_of(t, 1) % 8 == 0 &&
        reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0))
    TORCH_CHECK(false, format_msg("%s must have unit stride along its last dim, other strides that are multiples of 8, and be "
                                  "16-byte aligned", name));
}

// Checks what the three calls share and fills the batch; d_qk and d_v are the heads' dims.
nsa_cache_batch cache_batch(const torch::Tensor& cache, const torch::Tensor& pages, const torch::Tensor& lens,
                            const OptTensor& cu_seqlens, int64_t n_rows, int64_t d_qk, int64_t d_v) {
  TORCH_CHECK(cache.is_cuda(), "cache must be a CUDA tensor");
  TORCH_CHECK(cache.scalar_type() == at::kByte && cache.dim() == 3, "cache must be uint8 [num_pages, Hkv, record bytes]");
  TORCH_CHECK(pages.is_cuda() && lens.is_cuda() && pages.get_device() == cache.get_device() &&
                  lens.get_device() == cache.get_device(),
              "pages and lens must be on the cache's device");
  TORCH_CHECK(pages.scalar_type() == at::kInt && pages.dim() == 2 && lens.scalar_type() == at::kInt && lens.dim() == 1,
              "pages must be int32 [n_seqs, width] and lens int32 [n_seqs]");
  TORCH_CHECK(pages.size(0) == lens.size(0), "pages and lens must have one row for each sequence");
  TORCH_CHECK((pages.size(1) <= 1 || pages.stride(1) == 1) && (pages.size(0) <= 1 || pages.stride(0) >= pages.size(1)) &&
                  lens.is_contiguous(),
              "pages' rows and lens must be contiguous");
  const int64_t record = api().cache_record(i32(d_qk, "d_qk"), i32(d_v, "d_v"));
  if (record < 0)
    TORCH_CHECK(false, format_msg("(d_qk, d_v) = (%lld, %lld) is not one of (64, 64), (128, 128), (192, 128), (128, 64)",
                                  (long long)d_qk, (long long)d_v));
  if (cache.size(2) != record)
    TORCH_CHECK(false, format_msg("a record of the cache has %lld bytes, (d_qk, d_v) = (%lld, %lld) needs %lld",
                                  (long long)cache.size(2), (long long)d_qk, (long long)d_v, (long long)record));
  TORCH_CHECK(cache.size(1) >= 1 && cache.stride(2) == 1 && (cache.size(1) == 1 || cache.stride(1) == record) &&
                  (cache.size(0) <= 1 || (cache.stride(0) >= cache.size(1) * record && cache.stride(0) % 16 == 0)) &&
                  reinterpret_cast<uintptr_t>(cache.data_ptr()) % 16 == 0,
              "cache must be 16-byte aligned, its pages contiguous and their stride a multiple of 16");
  nsa_cache_batch b;
  memset(&b, 0, sizeof(b));
  b.cache = cache.data_ptr();
  b.pages = pages.data_ptr<int32_t>();
  b.lens = lens.data_ptr<int32_t>();
  if (cu_seqlens.has_value() && cu_seqlens->defined()) {
    const auto& cu = *cu_seqlens;
    TORCH_CHECK(cu.is_cuda() && cu.get_device() == cache.get_device() && cu.scalar_type() == at::kInt && cu.dim() == 1 &&
                    cu.is_contiguous(),
                "cu_seqlens must be a contiguous int32 vector on the cache's device");
    TORCH_CHECK(cu.numel() == lens.size(0) + 1, "cu_seqlens must have one entry more than there are sequences");
    b.cu_seqlens = cu.data_ptr<int32_t>();
  } else {
    TORCH_CHECK(n_rows == lens.size(0), "without cu_seqlens there must be one row for each sequence");
  }
  b.page_stride = cache.size(0) > 1 ? cache.stride(0) : 0;
  b.pages_stride = pages.size(0) > 1 ? pages.stride(0) : 0;
  b.num_pages = i32(cache.size(0), "num_pages");
  b.n_seqs = i32(lens.size(0), "n_seqs");
  b.width = i32(pages.size(1), "width");
  b.n_rows = i32(n_rows, "n_rows");
  b.heads_kv = i32(cache.size(1), "Hkv");
  b.d_qk = i32(d_qk, "d_qk");
  b.d_v = i32(d_v, "d_v");
  return b;
}

void cache_write(torch::Tensor cache, torch::Tensor K, torch::Tensor V, torch::Tensor pages, torch::Tensor lens,
                 OptTensor cu_seqlens) {
  TORCH_CHECK(K.dim() == 3 && V.dim() == 3 && K.size(0) == V.size(0) && K.size(1) == V.size(1),
              "K must be [N, Hkv, d_qk] and V [N, Hkv, d_v]");
  TORCH_CHECK(K.scalar_type() == V.scalar_type(), "K and V must have one dtype");
  const int32_t dtype = dtype_code(K, "K and V");
  const nsa_cache_batch b = cache_batch(cache, pages, lens, cu_seqlens, K.size(0), K.size(2), V.size(2));
  TORCH_CHECK(K.is_cuda() && V.is_cuda() && K.get_device() == cache.get_device() && V.get_device() == cache.get_device(),
              "all tensors must be on one device");
  TORCH_CHECK(K.size(1) == cache.size(1), "K, V and the cache must have the same heads");
  if (K.size(0) == 0) return;
  check_rows(K, "K");
  check_rows(V, "V");
  const c10::cuda::CUDAGuard guard(cache.device());
  const int rc = api().cache_write(&b, K.data_ptr(), V.data_ptr(), stride_of(K, 0), stride_of(K, 1), stride_of(V, 0),
                                   stride_of(V, 1), dtype, current_stream());
  if (rc != NSA_OK) TORCH_CHECK(false, format_msg("nsa_cache_write failed (%d): %s", rc, api().last_error()));
}

std::vector<torch::Tensor> cache_read(torch::Tensor cache, int64_t d_qk, torch::Tensor pages, torch::Tensor lens,
                                      OptTensor cu_seqlens, int64_t n_tokens, at::ScalarType dtype) {
  TORCH_CHECK(dtype == at::kBFloat16 || dtype == at::kHalf || dtype == at::kFloat, "dtype must be bfloat16, float16 or float32");
  TORCH_CHECK(cache.dim() == 3, "cache must be uint8 [num_pages, Hkv, record bytes]");
  TORCH_CHECK(n_tokens >= 0, "n_tokens must not be negative");
  const int64_t d_v = cache.size(2) / 36 - d_qk;
  const nsa_cache_batch b = cache_batch(cache, pages, lens, cu_seqlens, n_tokens, d_qk, std::max<int64_t>(d_v, 0));
  const c10::cuda::CUDAGuard guard(cache.device());
  auto K = torch::empty({1, cache.size(1), n_tokens, d_qk}, cache.options().dtype(dtype));
  auto V = torch::empty({1, cache.size(1), n_tokens, d_v}, cache.options().dtype(dtype));
  if (n_tokens == 0) return {K, V};
  const int32_t code = dtype == at::kBFloat16 ? NSA_DTYPE_BF16 : dtype == at::kHalf ? NSA_DTYPE_F16 : NSA_DTYPE_F32;
  const int rc = api().cache_read(&b, K.data_ptr(), V.data_ptr(), code, current_stream());
  if (rc != NSA_OK) TORCH_CHECK(false, format_msg("nsa_cache_read failed (%d): %s", rc, api().last_error()));
  return {K, V};
}

std::vector<torch::Tensor> cache_attend(torch::Tensor Q, torch::Tensor cache, torch::Tensor pages, torch::Tensor lens,
                                        OptTensor sel, int64_t l_prime, int64_t window, OptTensor cu_seqlens, double scale,
                                        OptTensor out, OptTensor weight, bool accumulate, bool with_lse, OptTensor err,
                                        int64_t timeout_ms, int64_t debug_flags) {
  TORCH_CHECK(Q.dim() == 3, "Q must be [N, Hq, d_qk]");
  const int32_t dtype = dtype_code(Q, "Q");
  TORCH_CHECK(cache.dim() == 3, "cache must be uint8 [num_pages, Hkv, record bytes]");
  const int64_t d_qk = Q.size(2), d_v = cache.size(2) / 36 - d_qk;
  nsa_cache_attend_desc d;
  memset(&d, 0, sizeof(d));
  d.batch = cache_batch(cache, pages, lens, cu_seqlens, Q.size(0), d_qk, std::max<int64_t>(d_v, 0));
  TORCH_CHECK(Q.is_cuda() && Q.get_device() == cache.get_device(), "all tensors must be on one device");
  TORCH_CHECK(Q.size(1) > 0 && Q.size(1) % cache.size(1) == 0, "Hq must be a multiple of Hkv");
  TORCH_CHECK(window >= 0, "window must not be negative");
  if (sel.has_value()) {
    TORCH_CHECK(sel->is_cuda() && sel->get_device() == cache.get_device() && sel->scalar_type() == at::kInt &&
                    sel->dim() == 3 && sel->is_contiguous(),
                "sel must be a contiguous int32 [N, Hkv, KSEL] on the cache's device");
    TORCH_CHECK(sel->size(0) == Q.size(0) && sel->size(1) == cache.size(1) && sel->size(2) >= 1,
                "sel must be [N, Hkv, KSEL] with the rows of Q and the heads of the cache");
    d.sel = sel->data_ptr<int32_t>();
    d.n_sel = i32(sel->size(2), "KSEL");
    d.block_size = i32(l_prime, "l_prime");
  }
  if (weight.has_value()) {
    TORCH_CHECK(weight->is_cuda() && weight->scalar_type() == at::kFloat && weight->numel() >= 1 &&
                    weight->get_device() == cache.get_device(),
                "weight must be an fp32 CUDA tensor (its first element is used) on Q's device");
    d.o_weight = weight->data_ptr<float>();
  }
  if (err.has_value()) {
    TORCH_CHECK(err->is_cuda() && err->scalar_type() == at::kInt && err->numel() >= 1 && err->get_device() == cache.get_device(),
                "err must be an int32 CUDA tensor (its first element is used) on Q's device");
    d.err = err->data_ptr<int32_t>();
  }
  const c10::cuda::CUDAGuard guard(cache.device());
  torch::Tensor O, L;
  if (out.has_value()) {
    O = *out;
    TORCH_CHECK(O.is_cuda() && O.get_device() == cache.get_device() && O.is_contiguous() && O.dim() == 3 &&
                    O.size(0) == Q.size(0) && O.size(1) == Q.size(1) && O.size(2) == d_v &&
                    (O.scalar_type() == at::kFloat || O.scalar_type() == Q.scalar_type()) &&
                    reinterpret_cast<uintptr_t>(O.data_ptr()) % 16 == 0,
                "out must be a contiguous, 16-byte aligned [N, Hq, d_v] on Q's device, fp32 or of Q's dtype");
    TORCH_CHECK(!accumulate || O.scalar_type() == at::kFloat, "accumulate needs an fp32 out");
  } else {
    TORCH_CHECK(!accumulate, "accumulate needs an out tensor");
    O = torch::empty({Q.size(0), Q.size(1), d_v}, Q.options());
  }
  const bool keep = out.has_value();
  const auto f32 = Q.options().dtype(torch::kFloat32);
  if (with_lse && keep && d.batch.cu_seqlens != nullptr)
    L = torch::full({Q.size(0), Q.size(1)}, -INFINITY, f32);  // rows of no sequence, which the call leaves
  else
    L = torch::empty({with_lse ? Q.size(0) : 0, Q.size(1)}, f32);
  if (Q.size(0) == 0) return {O, L};
  if ((Q.size(0) > 1 && Q.stride(0) == 0) || (Q.size(1) > 1 && Q.stride(1) == 0)) Q = Q.contiguous();  // (0 means the default)
  check_rows(Q, "Q");
  d.q = Q.data_ptr();
  d.o = O.data_ptr();
  d.lse = with_lse ? L.data_ptr<float>() : nullptr;
  d.q_row_stride = stride_of(Q, 0);
  d.q_head_stride = stride_of(Q, 1);
  d.heads_q = i32(Q.size(1), "Hq");
  d.window = i32(window, "window");
  d.q_dtype = dtype;
  d.o_dtype = O.scalar_type() == at::kFloat ? NSA_DTYPE_F32 : dtype;
  d.o_accumulate = accumulate ? 1 : 0;
  d.keep_rows = keep ? 1 : 0;
  d.scale = static_cast<float>(scale);
  d.timeout_ms = i32(timeout_ms, "timeout_ms");
  d.debug_flags = i32(debug_flags, "debug_flags");
  const Api& a = api();
  const int64_t ws = a.cache_attend_ws(&d);
  if (ws < 0) TORCH_CHECK(false, format_msg("nsa_cache_attend failed: %s", a.last_error()));
  torch::Tensor work;
  if (ws > 16) {  // (16: no row is cut, nothing is kept)
    work = torch::empty({ws}, Q.options().dtype(torch::kByte));
    d.workspace = work.data_ptr();
  }
  const int rc = a.cache_attend(&d, current_stream());
  if (rc != NSA_OK) TORCH_CHECK(false, format_msg("nsa_cache_attend failed (%d): %s", rc, a.last_error()));
  return {O, L};
}

int64_t cache_record_bytes(int64_t d_qk, int64_t d_v) {
  const int64_t n = api().cache_record(i32(d_qk, "d_qk"), i32(d_v, "d_v"));
  if (n < 0)
    TORCH_CHECK(false, format_msg("(d_qk, d_v) = (%lld, %lld) is not one of (64, 64), (128, 128), (192, 128), (128, 64)",
                                  (long long)d_qk, (long long)d_v));
  return n;
}

// ------------------------------------------------------------------ pages, selection and positions of a step
// torch::empty on the current device without its dispatch: a step's small calls take less time than that.
torch::Tensor empty_like_on(const torch::Tensor& t, c10::IntArrayRef sizes, at::ScalarType dtype) {
  return at::detail::empty_cuda(sizes, dtype, t.device(), c10::nullopt);
}
// `n` elements of a buffer, from byte `at` on, as a tensor of its own.
torch::Tensor part_of(const torch::Tensor& buffer, at::ScalarType dtype, int64_t at, int64_t n) {
  auto t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(buffer.storage()), c10::DispatchKeySet(c10::DispatchKey::CUDA),
                                                    c10::scalarTypeToTypeMeta(dtype));
  t.unsafeGetTensorImpl()->set_storage_offset(at / static_cast<int64_t>(c10::elementSize(dtype)));
  t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
  return t;
}

// [lens, cu_seqlens (empty without n_tokens), positions, slots, held, n_free]
std::vector<torch::Tensor> cache_reserve(torch::Tensor pages, torch::Tensor held, torch::Tensor rows, torch::Tensor pool,
                                         torch::Tensor n_free, c10::optional<int64_t> n_tokens, bool update) {
  TORCH_CHECK(pages.is_cuda() && pages.scalar_type() == at::kInt && pages.dim() == 2, "pages must be an int32 CUDA tensor [S, W]");
  const int64_t n = pages.size(0);
  for (const torch::Tensor* t : {&held, &rows, &pool, &n_free})
    TORCH_CHECK(t->is_cuda() && t->get_device() == pages.get_device() && t->scalar_type() == at::kInt && t->dim() == 1 &&
                    t->is_contiguous(),
                "held, rows, pool and n_free must be contiguous int32 vectors on the device of pages");
  TORCH_CHECK(held.size(0) == n && rows.size(0) == n, "held and rows must have one entry for each sequence of pages");
  TORCH_CHECK(n_free.size(0) == 1, "n_free must have one element");
  TORCH_CHECK((pages.size(1) <= 1 || pages.stride(1) == 1) && (n <= 1 || pages.stride(0) >= pages.size(1)),
              "the rows of pages must be contiguous and must not overlap");
  TORCH_CHECK(!n_tokens.has_value() || *n_tokens >= 0, "n_tokens must not be negative");
  const c10::cuda::CUDAGuard guard(pages.device());
  const int64_t n_rows = n_tokens.value_or(n);
  // one buffer for all results, each at a multiple of 16 bytes
  int64_t bytes = 0;
  const auto place = [&](int64_t size) {
    const int64_t at = bytes;
    bytes += (size + 15) / 16 * 16;
    return at;
  };
  const int64_t n_cu = n_tokens.has_value() ? n + 1 : 0;
  TORCH_CHECK(n_rows <= std::numeric_limits<int32_t>::max(), "n_tokens out of int32 range");
  const int64_t at_slots = place(8 * n_rows), at_positions = place(4 * n_rows), at_lens = place(4 * n), at_cu = place(4 * n_cu);
  const int64_t at_held = place(update ? 0 : 4 * n), at_free = place(update ? 0 : 4);
  const auto buffer = empty_like_on(pages, {std::max<int64_t>(bytes, 16)}, at::kByte);
  const auto lens = part_of(buffer, at::kInt, at_lens, n), cu = part_of(buffer, at::kInt, at_cu, n_cu);
  const auto positions = part_of(buffer, at::kInt, at_positions, n_rows), slots = part_of(buffer, at::kLong, at_slots, n_rows);
  const auto held_out = update ? held : part_of(buffer, at::kInt, at_held, n);
  const auto n_free_out = update ? n_free : part_of(buffer, at::kInt, at_free, 1);
  nsa_cache_reserve_desc d;
  memset(&d, 0, sizeof(d));
  d.pages = pages.data_ptr<int32_t>();
  d.held = held.data_ptr<int32_t>();
  d.rows = rows.data_ptr<int32_t>();
  d.pool = pool.data_ptr<int32_t>();
  d.n_free = n_free.data_ptr<int32_t>();
  d.held_out = held_out.data_ptr<int32_t>();
  d.n_free_out = n_free_out.data_ptr<int32_t>();
  d.lens = lens.data_ptr<int32_t>();
  d.cu_seqlens = n_tokens.has_value() ? cu.data_ptr<int32_t>() : nullptr;
  d.positions = n_rows > 0 ? positions.data_ptr<int32_t>() : nullptr;
  d.slots = n_rows > 0 ? slots.data_ptr<int64_t>() : nullptr;
  d.pages_stride = n > 1 ? pages.stride(0) : 0;
  d.n_seqs = i32(n, "n_seqs");
  d.width = i32(pages.size(1), "width");
  d.pool_size = i32(pool.size(0), "pool_size");
  d.n_rows = i32(n_rows, "n_tokens");
  const int rc = api().cache_reserve(&d, current_stream());
  if (rc != NSA_OK) TORCH_CHECK(false, format_msg("nsa_cache_reserve failed (%d): %s", rc, api().last_error()));
  return {lens, cu, positions, slots, held_out, n_free_out};
}

torch::Tensor cache_select(torch::Tensor Q, torch::Tensor cache, torch::Tensor pages, torch::Tensor lens, int64_t n_sel,
                           int64_t l_prime, int64_t cmp_block, int64_t cmp_stride, OptTensor cu_seqlens) {
  TORCH_CHECK(Q.dim() == 3, "Q must be [N, Hq, d_qk]");
  const int32_t dtype = dtype_code(Q, "Q");
  TORCH_CHECK(cache.dim() == 3, "cache must be uint8 [num_pages, Hkv, record bytes]");
  const int64_t d_qk = Q.size(2), d_v = cache.size(2) / 36 - d_qk;
  nsa_cache_select_desc d;
  memset(&d, 0, sizeof(d));
  d.batch = cache_batch(cache, pages, lens, cu_seqlens, Q.size(0), d_qk, std::max<int64_t>(d_v, 0));
  TORCH_CHECK(Q.is_cuda() && Q.get_device() == cache.get_device(), "all tensors must be on one device");
  TORCH_CHECK(Q.size(1) > 0 && Q.size(1) % cache.size(1) == 0, "Hq must be a multiple of Hkv");
  TORCH_CHECK(n_sel >= 1 && cmp_block >= 1 && cmp_stride >= 1, "n_sel, cmp_block and cmp_stride must be positive");
  const c10::cuda::CUDAGuard guard(cache.device());
  auto sel = empty_like_on(Q, {Q.size(0), cache.size(1), n_sel}, at::kInt);
  if ((Q.size(0) > 1 && Q.stride(0) == 0) || (Q.size(1) > 1 && Q.stride(1) == 0)) Q = Q.contiguous();  // (0 means the default)
  if (Q.size(0) > 0) {
    check_rows(Q, "Q");
    d.q = Q.data_ptr();
    d.sel = sel.data_ptr<int32_t>();
  }
  d.q_row_stride = stride_of(Q, 0);
  d.q_head_stride = stride_of(Q, 1);
  d.heads_q = i32(Q.size(1), "Hq");
  d.n_sel = i32(n_sel, "n_sel");
  d.block_size = i32(l_prime, "l_prime");
  d.cmp_block = i32(cmp_block, "cmp_block");
  d.cmp_stride = i32(cmp_stride, "cmp_stride");
  d.q_dtype = dtype;
  const int64_t ws = api().cache_select_ws(&d);
  if (ws < 0) TORCH_CHECK(false, format_msg("nsa_cache_select failed: %s", api().last_error()));
  const auto work = empty_like_on(Q, {ws}, at::kByte);
  d.workspace = work.data_ptr();
  const int rc = api().cache_select(&d, current_stream());
  if (rc != NSA_OK) TORCH_CHECK(false, format_msg("nsa_cache_select failed (%d): %s", rc, api().last_error()));
  return sel;
}

// X [N, H, d] or [B, H, T, d]: strides of batch, head, token.
void rotary_strides(const torch::Tensor& x, int64_t (&s)[3]) {
  const bool rows = x.dim() == 3;
  s[0] = rows ? 0 : stride_of(x, 0);
  s[1] = stride_of(x, 1);
  s[2] = stride_of(x, rows ? 0 : 2);
}

// [Q', K'] (K' undefined without K).  `token_major` says of each whether [B, H, T, d] is laid out as [B, T, H, d].
std::vector<torch::Tensor> turned(torch::Tensor Q, OptTensor K, const torch::Tensor& positions, const torch::Tensor& turns,
                                  const torch::Tensor& axis, int64_t axes, int64_t d_head, int64_t offset, bool interleaved,
                                  bool inverse, bool q_token_major, bool k_token_major) {
  TORCH_CHECK(Q.is_cuda() && (Q.dim() == 3 || Q.dim() == 4), "Q must be a CUDA tensor [N, H, d] or [B, H, T, d]");
  TORCH_CHECK(Q.scalar_type() == at::kBFloat16 || Q.scalar_type() == at::kHalf || Q.scalar_type() == at::kFloat,
              "Q must be bfloat16, float16 or float32");
  const bool rows = Q.dim() == 3;
  const int64_t B = rows ? 1 : Q.size(0), T = Q.size(rows ? 0 : 2);
  TORCH_CHECK(Q.size(-1) == d_head, "the plan is for heads of another size");
  if (K.has_value()) {
    TORCH_CHECK(K->is_cuda() && K->get_device() == Q.get_device() && K->scalar_type() == Q.scalar_type() && K->dim() == Q.dim(),
                "K must be of Q's dtype and dims, on its device");
    TORCH_CHECK((rows ? 1 : K->size(0)) == B && K->size(rows ? 0 : 2) == T && K->size(-1) == d_head,
                "K must have Q's tokens and head size");
  }
  TORCH_CHECK(positions.is_cuda() && positions.get_device() == Q.get_device() && positions.scalar_type() == at::kInt,
              "positions must be int32 on Q's device");
  const int64_t lead = axes > 1 ? 1 : 0;
  TORCH_CHECK(positions.dim() == lead + (rows ? 1 : 2) && (!lead || positions.size(0) == axes) &&
                  (rows || positions.size(lead) == B) && positions.size(-1) == T,
              "positions must be [N] or [B, T], one for each token of Q, with the axes before them if there are several");
  TORCH_CHECK(!turns.is_cuda() && turns.scalar_type() == at::kLong && turns.is_contiguous() && !axis.is_cuda() &&
                  axis.scalar_type() == at::kByte && axis.is_contiguous() && axis.numel() == turns.numel(),
              "a plan's turns and axis are int64 and uint8 host vectors of one length");
  const c10::cuda::CUDAGuard guard(Q.device());
  nsa_rotary_desc d;
  memset(&d, 0, sizeof(d));
  torch::Tensor out[2];
  for (int i = 0; i < 2; ++i) {
    if (i == 1 && !K.has_value()) {
      continue;
    }
    torch::Tensor x = i == 0 ? Q : *K;
    if (x.size(-1) > 1 && x.stride(-1) != 1) x = x.contiguous();
    if (!rows && (i == 0 ? q_token_major : k_token_major))
      out[i] = empty_like_on(x, {B, T, x.size(1), d_head}, x.scalar_type()).transpose(1, 2);
    else
      out[i] = empty_like_on(x, x.sizes(), x.scalar_type());
    if (x.numel() == 0) continue;
    d.t[i].x = x.data_ptr();
    d.t[i].y = out[i].data_ptr();
    rotary_strides(x, d.t[i].x_stride);
    rotary_strides(out[i], d.t[i].y_stride);
    d.t[i].heads = i32(x.size(1), "heads");
    (i == 0 ? Q : *K) = x;  // (a copy lives until the launch)
  }
  if (B * T > 0) d.positions = positions.data_ptr<int32_t>();
  d.pos_stride[0] = lead ? positions.stride(0) : 0;
  d.pos_stride[1] = rows ? 0 : positions.stride(lead);
  d.pos_stride[2] = positions.stride(-1);
  d.turns = reinterpret_cast<const uint64_t*>(turns.data_ptr<int64_t>());
  d.axis = axis.data_ptr<uint8_t>();
  d.batch = i32(B, "batch");
  d.tokens = i32(T, "tokens");
  d.d = i32(d_head, "d");
  d.offset = i32(offset, "offset");
  d.pairs = i32(turns.numel(), "pairs");
  d.axes = i32(axes, "axes");
  d.interleaved = interleaved ? 1 : 0;
  d.inverse = inverse ? 1 : 0;
  d.dtype = Q.scalar_type() == at::kBFloat16 ? NSA_DTYPE_BF16 : Q.scalar_type() == at::kHalf ? NSA_DTYPE_F16 : NSA_DTYPE_F32;
  const int rc = api().rotary(&d, current_stream());
  if (rc != NSA_OK) TORCH_CHECK(false, format_msg("nsa_rotary failed (%d): %s", rc, api().last_error()));
  return {out[0], out[1]};
}

std::vector<torch::Tensor> rotary(torch::Tensor Q, OptTensor K, torch::Tensor positions, torch::Tensor turns, torch::Tensor axis,
                                  int64_t axes, int64_t d_head, int64_t offset, bool interleaved, bool inverse,
                                  bool q_token_major, bool k_token_major);

// The turn is linear and its transpose the turn back, so the gradient is a call of the same kind, and has gradients too.
struct RotaryFunction : torch::autograd::Function<RotaryFunction> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, torch::Tensor Q, OptTensor K,
                                                torch::Tensor positions, torch::Tensor turns, torch::Tensor axis, int64_t axes,
                                                int64_t d_head, int64_t offset, bool interleaved, bool inverse, bool q_token_major,
                                                bool k_token_major) {
    const bool both = K.has_value();
    ctx->save_for_backward({positions, turns, axis});
    ctx->set_materialize_grads(false);
    // gradients come back as the inputs lie: [B, H, T, d] may be a view of [B, T, H, d], or of a part of a fused projection
    const auto as_view = [](const torch::Tensor& x) {
      return x.dim() == 4 && x.size(1) > 1 && x.size(2) > 1 && x.stride(1) > 0 && x.stride(1) < x.stride(2);
    };
    const int64_t flags = (both ? 1 : 0) | (interleaved ? 2 : 0) | (inverse ? 4 : 0) | (as_view(Q) ? 8 : 0) |
                          (both && as_view(*K) ? 16 : 0);
    ctx->saved_data["flags"] = flags;
    ctx->saved_data["axes"] = axes;
    ctx->saved_data["d"] = d_head;
    ctx->saved_data["offset"] = offset;
    auto out = turned(Q, K, positions, turns, axis, axes, d_head, offset, interleaved, inverse,
                      q_token_major, k_token_major);
    if (!both) out.pop_back();
    return out;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const int64_t flags = ctx->saved_data["flags"].toInt();
    const auto back = [&](const torch::Tensor& q, const OptTensor& k, bool q_major, bool k_major) {
      return rotary(q, k, saved[0], saved[1], saved[2], ctx->saved_data["axes"].toInt(), ctx->saved_data["d"].toInt(),
                    ctx->saved_data["offset"].toInt(), (flags & 2) != 0, (flags & 4) == 0, q_major, k_major);
    };
    torch::autograd::variable_list result(12);
    const bool q = grads[0].defined() && ctx->needs_input_grad(0);
    const bool k = (flags & 1) != 0 && grads[1].defined() && ctx->needs_input_grad(1);
    if (q) {
      const auto d = back(grads[0], k ? OptTensor(grads[1]) : OptTensor(), (flags & 8) != 0, (flags & 16) != 0);
      result[0] = d[0];
      if (k) result[1] = d[1];
    } else if (k) {
      result[1] = back(grads[1], OptTensor(), (flags & 16) != 0, false)[0];
    }
    return result;
  }
};

// Whether forward mode has a tangent for x that is not zero.
bool has_tangent(const torch::Tensor& x) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return false;
  const torch::Tensor& t = x._fw_grad(0);
  return t.defined() && !t._is_zerotensor();
}

std::vector<torch::Tensor> rotary(torch::Tensor Q, OptTensor K, torch::Tensor positions, torch::Tensor turns, torch::Tensor axis,
                                  int64_t axes, int64_t d_head, int64_t offset, bool interleaved, bool inverse,
                                  bool q_token_major, bool k_token_major) {
  const bool q_moves = has_tangent(Q), k_moves = K.has_value() && has_tangent(*K);
  if (q_moves || k_moves) {
    // forward mode: an output's tangent is the turned tangent of its input
    const auto turn = [&](const torch::Tensor& q, const OptTensor& k, bool q_major) {
      return rotary(q, k, positions, turns, axis, axes, d_head, offset, interleaved, inverse, q_major, k_token_major);
    };
    const auto primal = [](const torch::Tensor& x) { return std::get<0>(at::_unpack_dual(x, 0)); };
    auto out = turn(primal(Q), K.has_value() ? OptTensor(primal(*K)) : OptTensor(), q_token_major);
    torch::Tensor dq, dk;
    if (q_moves) {
      const auto d = turn(Q._fw_grad(0), k_moves ? OptTensor(K->_fw_grad(0)) : OptTensor(), q_token_major);
      dq = d[0], dk = d[1];
    } else {
      dk = turn(K->_fw_grad(0), OptTensor(), k_token_major)[0];
    }
    if (q_moves) out[0] = at::_make_dual(out[0], dq, 0);
    if (k_moves) out[1] = at::_make_dual(out[1], dk, 0);
    return out;
  }
  if (torch::GradMode::is_enabled() && (Q.requires_grad() || (K.has_value() && K->requires_grad()))) {
    auto out = RotaryFunction::apply(Q, K, positions, turns, axis, axes, d_head, offset,
                                     interleaved, inverse, q_token_major, k_token_major);
    if (!K.has_value()) out.push_back(torch::Tensor());
    return out;
  }
  return turned(Q, K, positions, turns, axis, axes, d_head, offset, interleaved, inverse, q_token_major, k_token_major);
}

int64_t library_version() { return api().version(); }

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "B200 NSA selected-branch forward (sm_100a) with the nsa-hopper op signature";
  m.def("forward", &forward, "forward(Q, K, V, sel, l_prime, BQ, cyc) -> O (fp32)");
  m.def("forward_lse", &forward_lse, "forward_lse(Q, K, V, sel, l_prime, BQ, cu_seqlens, scale, out_f32) -> [O, LSE]",
        py::arg("Q"), py::arg("K"), py::arg("V"), py::arg("sel"), py::arg("l_prime"), py::arg("BQ"),
        py::arg("cu_seqlens") = py::none(), py::arg("scale") = 0.0, py::arg("out_f32") = false);
  m.def("forward_ext", &forward_ext,
        "forward_ext(Q, K, V, sel, l_prime, BQ, window, key_map, scale, out, weight, accumulate, with_lse) -> "
        "[O fp32, LSE]",
        py::arg("Q"), py::arg("K"), py::arg("V"), py::arg("sel"), py::arg("l_prime"), py::arg("BQ"),
        py::arg("window") = 0, py::arg("key_map") = 0, py::arg("scale") = 0.0, py::arg("out") = py::none(),
        py::arg("weight") = py::none(), py::arg("accumulate") = false, py::arg("with_lse") = true);
  m.def("select_blocks", &select_blocks, "select_blocks(Q, K, n_sel, l_prime, cmp_block, cmp_stride) -> sel int32",
        py::arg("Q"), py::arg("K"), py::arg("n_sel"), py::arg("l_prime"), py::arg("cmp_block") = 32,
        py::arg("cmp_stride") = 16);
  m.def("cache_record_bytes", &cache_record_bytes, py::arg("d_qk"), py::arg("d_v"));
  m.def("cache_write", &cache_write, "cache_write(cache, K, V, pages, lens, cu_seqlens): quantises rows into the cache",
        py::arg("cache"), py::arg("K"), py::arg("V"), py::arg("pages"), py::arg("lens"), py::arg("cu_seqlens") = py::none());
  m.def("cache_read",
        [](torch::Tensor cache, int64_t d_qk, torch::Tensor pages, torch::Tensor lens, OptTensor cu_seqlens, int64_t n_tokens,
           py::object dtype) {
          return cache_read(cache, d_qk, pages, lens, cu_seqlens, n_tokens, torch::python::detail::py_object_to_dtype(dtype));
        },
        "cache_read(cache, d_qk, pages, lens, cu_seqlens, n_tokens, dtype) -> [K, V]", py::arg("cache"), py::arg("d_qk"),
        py::arg("pages"), py::arg("lens"), py::arg("cu_seqlens"), py::arg("n_tokens"), py::arg("dtype"));
  m.def("cache_attend", &cache_attend,
        "cache_attend(Q, cache, pages, lens, sel, l_prime, window, cu_seqlens, scale, out, weight, accumulate, with_lse, err, "
        "timeout_ms, debug_flags) -> [O, LSE]",
        py::arg("Q"), py::arg("cache"), py::arg("pages"), py::arg("lens"), py::arg("sel") = py::none(),
        py::arg("l_prime") = 64, py::arg("window") = 0, py::arg("cu_seqlens") = py::none(), py::arg("scale") = 0.0,
        py::arg("out") = py::none(), py::arg("weight") = py::none(), py::arg("accumulate") = false,
        py::arg("with_lse") = true, py::arg("err") = py::none(), py::arg("timeout_ms") = 0, py::arg("debug_flags") = 0);
  m.def("cache_reserve", &cache_reserve,
        "cache_reserve(pages, held, rows, pool, n_free, n_tokens, update) -> [lens, cu_seqlens, positions, slots, held, n_free]",
        py::arg("pages"), py::arg("held"), py::arg("rows"), py::arg("pool"), py::arg("n_free"), py::arg("n_tokens") = py::none(),
        py::arg("update") = true);
  m.def("cache_select", &cache_select,
        "cache_select(Q, cache, pages, lens, n_sel, l_prime, cmp_block, cmp_stride, cu_seqlens) -> sel int32", py::arg("Q"),
        py::arg("cache"), py::arg("pages"), py::arg("lens"), py::arg("n_sel"), py::arg("l_prime") = 64,
        py::arg("cmp_block") = 32, py::arg("cmp_stride") = 16, py::arg("cu_seqlens") = py::none());
  m.def("rotary", &rotary,
        "rotary(Q, K, positions, turns, axis, axes, d, offset, interleaved, inverse, q_token_major, k_token_major) -> [Q', K']",
        py::arg("Q"), py::arg("K"), py::arg("positions"), py::arg("turns"), py::arg("axis"), py::arg("axes"), py::arg("d"),
        py::arg("offset"), py::arg("interleaved"), py::arg("inverse") = false, py::arg("q_token_major") = false,
        py::arg("k_token_major") = false);
  m.def("library_version", &library_version);
}
