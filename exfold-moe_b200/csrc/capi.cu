// extern "C" entry points of libexfold_b200.so: argument checks, error reporting, dispatch.
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include <atomic>
#include <map>
#include <mutex>
#include <tuple>

#include "exf_adapters.h"
#include "exf_balance.h"
#include "exf_common.cuh"
#include "exf_gated.h"
#include "exf_kernels.h"
#include "exf_launch.h"
#include "exf_moe.h"
#include "exf_mxfp4.h"
#include "exf_mxmoe.h"
#include "exf_norm.h"

namespace exf {



// ---- launch helpers -----------------------------------------------------------------------
static std::mutex g_grid_mu;
static std::map<std::tuple<const void*, int, size_t, int>, int> g_grid_cache;

int sm_count() {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  int n = 0;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  return n;
}

int persistent_grid(const void* kernel, int threads, size_t smem) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  const auto key = std::make_tuple(kernel, threads, smem, dev);
  {
    std::lock_guard<std::mutex> lk(g_grid_mu);
    auto it = g_grid_cache.find(key);
    if (it != g_grid_cache.end()) return it->second;
  }
  int per_sm = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, smem) != cudaSuccess)
    return 0;
  const int grid = per_sm * sm_count();
  std::lock_guard<std::mutex> lk(g_grid_mu);
  g_grid_cache[key] = grid;
  return grid;
}

}  // namespace exf

using namespace exf;

// ---- error reporting ------------------------------------------------------------------------
static thread_local char g_err[512] = "";

static int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

static int cuda_status(cudaError_t e, const char* what) {
  if (e == cudaSuccess) {
    g_err[0] = 0;
    return EXF_OK;
  }
  if (e == cudaErrorNotSupported) return fail(EXF_ERR_UNSUPPORTED, "%s: shape not compiled", what);
  return fail(EXF_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

#define EXF_REQUIRE(cond, ...)                                 \
  do {                                                         \
    if (!(cond)) return fail(EXF_ERR_INVALID, __VA_ARGS__);    \
  } while (0)

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
static bool good_wdtype(int d) { return d == EXF_F32 || d == EXF_BF16 || d == EXF_F16; }
static bool good_idtype(int d) { return d == EXF_I32 || d == EXF_I64; }

// ---- entry points ---------------------------------------------------------------------------
extern "C" {

EXF_API int exf_abi_version(void) { return 3; }

EXF_API int64_t exf_router_tile_min_rows(int64_t rows) { return router_tile_min_rows(rows); }

EXF_API const char* exf_last_error(void) { return g_err; }

static int router_common(const char* name, const void* logits, int logit_dtype, int64_t tokens,
                         int layers, int experts, int top_k, int scoring, const float* out_w,
                         const int32_t* out_ids) {
  EXF_REQUIRE(good_wdtype(logit_dtype), "%s: logits must be EXF_F32, EXF_BF16 or EXF_F16", name);
  EXF_REQUIRE(tokens >= 0 && layers >= 1, "%s: tokens must be >= 0 and layers >= 1", name);
  EXF_REQUIRE(top_k >= 1 && top_k <= 8, "%s: top_k must be in [1, 8], got %d", name, top_k);
  EXF_REQUIRE(experts >= top_k, "%s: experts (%d) < top_k (%d)", name, experts, top_k);
  EXF_REQUIRE(scoring == EXF_SOFTMAX || scoring == EXF_SIGMOID || scoring == EXF_SQRTSOFTPLUS,
              "%s: unknown scoring %d", name, scoring);
  if (experts != 64 && experts != 128 && experts != 256 && experts != 512)
    return fail(EXF_ERR_UNSUPPORTED, "%s: experts must be one of 64, 128, 256, 512 (got %d)", name,
                experts);
  if (tokens > 0) {
    EXF_REQUIRE(logits && out_w && out_ids, "%s: null pointer", name);
    EXF_REQUIRE(aligned16(logits), "%s: logits must be 16-byte aligned", name);
  }
  return EXF_OK;
}

EXF_API int exf_router_topk(const void* logits, int logit_dtype, int64_t tokens, int experts,
                            int top_k, int scoring, const float* bias, int renormalize,
                            float scaling, float* out_w, int32_t* out_ids, exf_stream_t stream) {
  int rc = router_common("exf_router_topk", logits, logit_dtype, tokens, 1, experts, top_k,
                         scoring, out_w, out_ids);
  if (rc != EXF_OK) return rc;
  if (tokens == 0) return EXF_OK;
  EXF_REQUIRE(!bias || aligned16(bias), "exf_router_topk: bias must be 16-byte aligned");
  RouterParams p{logits, tokens, 1, top_k, bias, renormalize, scaling, top_k, 0,
                 nullptr, nullptr, nullptr, out_w, out_ids, logit_dtype};
  return cuda_status(launch_router(experts, scoring, 0, p, (cudaStream_t)stream), "exf_router_topk");
}

EXF_API int exf_router_hash(const void* logits, int logit_dtype, int64_t tokens, int experts,
                            int top_k, int scoring, const void* token_ids, int id_dtype,
                            const int32_t* table, int64_t table_rows, int renormalize,
                            float scaling, float* out_w, int32_t* out_ids, exf_stream_t stream) {
  const char* name = "exf_router_hash";
  EXF_REQUIRE(tokens >= 0, "%s: tokens must be >= 0", name);
  EXF_REQUIRE(top_k >= 1 && top_k <= 8, "%s: top_k must be in [1, 8], got %d", name, top_k);
  EXF_REQUIRE(experts >= 1, "%s: experts must be >= 1", name);
  EXF_REQUIRE(good_idtype(id_dtype), "%s: unsupported token id dtype", name);
  EXF_REQUIRE(good_wdtype(logit_dtype), "%s: logits must be EXF_F32, EXF_BF16 or EXF_F16", name);
  EXF_REQUIRE(table_rows >= 1, "%s: the hash table needs at least one row", name);
  if (scoring == EXF_SOFTMAX)
    return fail(EXF_ERR_UNSUPPORTED, "%s: hash routing takes sigmoid or sqrtsoftplus scores", name);
  EXF_REQUIRE(scoring == EXF_SIGMOID || scoring == EXF_SQRTSOFTPLUS, "%s: unknown scoring %d",
              name, scoring);
  if (tokens == 0) return EXF_OK;
  EXF_REQUIRE(logits && token_ids && table && out_w && out_ids, "%s: null pointer", name);
  return cuda_status(launch_router_hash(logits, logit_dtype, tokens, experts, top_k, scoring,
                                        token_ids,
                                        id_dtype, table, table_rows, renormalize, scaling, out_w,
                                        out_ids, (cudaStream_t)stream),
                     name);
}

EXF_API int exf_router_fold_prefill(const void* logits, int logit_dtype, int64_t tokens,
                                    int layers, int experts, int top_k, int scoring,
                                    const float* bias, int renormalize,
                                    float scaling, int target_k, int variant, int renorm_mode,
                                    const float* coeff, const float* sel_loss,
                                    const float* conf_loss, float* out_w, int32_t* out_ids,
                                    exf_stream_t stream) {
  const char* name = "exf_router_fold_prefill";
  int rc = router_common(name, logits, logit_dtype, tokens, layers, experts, top_k, scoring,
                         out_w, out_ids);
  if (rc != EXF_OK) return rc;
  EXF_REQUIRE(variant == EXF_QWEN3 || variant == EXF_DSV4, "%s: unknown variant %d", name, variant);
  EXF_REQUIRE(target_k >= 1 && target_k <= top_k, "%s: target_k must be in [1, top_k]", name);
  EXF_REQUIRE(renorm_mode >= 0 && renorm_mode <= 2, "%s: renorm_mode must be 0, 1 or 2", name);
  EXF_REQUIRE(variant == EXF_DSV4 || renorm_mode == 0, "%s: renorm_mode needs EXF_DSV4", name);
  if (tokens == 0) return EXF_OK;
  EXF_REQUIRE(coeff && sel_loss, "%s: null calibration table", name);
  EXF_REQUIRE(renorm_mode != 2 || conf_loss, "%s: similarity_blend needs conf_loss", name);
  EXF_REQUIRE(!bias || aligned16(bias), "%s: bias must be 16-byte aligned", name);
  RouterParams p{logits, tokens, layers, top_k, bias, renormalize, scaling, target_k, renorm_mode,
                 coeff, sel_loss, conf_loss, out_w, out_ids, logit_dtype};
  return cuda_status(launch_router(experts, scoring, variant == EXF_QWEN3 ? 1 : 2, p,
                                   (cudaStream_t)stream),
                     name);
}

EXF_API int exf_fold_prefill(const void* w, int w_dtype, const void* ids, int id_dtype,
                             int64_t tokens, int top_k, int target_k, int experts, int variant,
                             int renorm_mode, const float* coeff, const float* sel_loss,
                             const float* conf_loss, void* out_w, void* out_ids,
                             exf_stream_t stream) {
  const char* name = "exf_fold_prefill";
  EXF_REQUIRE(good_wdtype(w_dtype) && good_idtype(id_dtype), "%s: unsupported dtype", name);
  EXF_REQUIRE(tokens >= 0, "%s: tokens must be >= 0", name);
  EXF_REQUIRE(top_k >= 1 && top_k <= 8, "%s: top_k must be in [1, 8], got %d", name, top_k);
  EXF_REQUIRE(target_k >= 1 && target_k <= top_k, "%s: target_k must be in [1, top_k]", name);
  EXF_REQUIRE(experts >= 1, "%s: experts must be >= 1", name);
  EXF_REQUIRE(variant == EXF_QWEN3 || variant == EXF_DSV4, "%s: unknown variant %d", name, variant);
  EXF_REQUIRE(renorm_mode >= 0 && renorm_mode <= 2, "%s: renorm_mode must be 0, 1 or 2", name);
  if (tokens == 0) return EXF_OK;
  EXF_REQUIRE(w && ids && out_w && out_ids && coeff && sel_loss, "%s: null pointer", name);
  EXF_REQUIRE(variant != EXF_DSV4 || renorm_mode != 2 || conf_loss,
              "%s: similarity_blend needs conf_loss", name);
  FoldParams p{w, ids, tokens, top_k, target_k, experts, variant == EXF_DSV4 ? renorm_mode : 0,
               coeff, sel_loss, conf_loss, out_w, out_ids};
  return cuda_status(launch_fold(w_dtype, id_dtype, variant, p, (cudaStream_t)stream), name);
}

static int decode_checks(const char* name, int w_dtype, int id_dtype, int64_t batch, int top_k,
                         int experts, int budget, int variant) {
  EXF_REQUIRE(good_wdtype(w_dtype) && good_idtype(id_dtype), "%s: unsupported dtype", name);
  EXF_REQUIRE(batch >= 0 && top_k >= 1, "%s: bad routing shape", name);
  EXF_REQUIRE(experts >= 1 && experts <= 1024, "%s: experts must be in [1, 1024]", name);
  EXF_REQUIRE(budget >= 1 && budget <= experts, "%s: budget must be in [1, experts]", name);
  EXF_REQUIRE(variant == EXF_QWEN3 || variant == EXF_DSV4, "%s: unknown variant %d", name, variant);
  return EXF_OK;
}

EXF_API int exf_decode(const void* w, int w_dtype, const void* ids, int id_dtype, int64_t batch,
                       int top_k, int experts, int budget, int variant, const float* norms,
                       const float* coeff, const float* loss, void* out_w, void* out_ids,
                       int32_t* out_subset, exf_stream_t stream) {
  const char* name = "exf_decode";
  int rc = decode_checks(name, w_dtype, id_dtype, batch, top_k, experts, budget, variant);
  if (rc != EXF_OK) return rc;
  EXF_REQUIRE(norms && coeff && loss, "%s: null calibration table", name);
  EXF_REQUIRE(batch == 0 || (w && ids && out_w && out_ids), "%s: null routing pointer", name);
  DecodeParams p{w, ids, batch * top_k, experts, budget, variant, 0 /*from routes*/, norms,
                 nullptr, nullptr, coeff, loss, out_w, out_ids, out_subset};
  return cuda_status(launch_decode(w_dtype, id_dtype, p, (cudaStream_t)stream), name);
}

EXF_API int exf_decode_importance(const void* w, int w_dtype, const void* ids, int id_dtype,
                                  int64_t routes, int experts, const float* norms,
                                  int64_t* importance, exf_stream_t stream) {
  const char* name = "exf_decode_importance";
  EXF_REQUIRE(good_wdtype(w_dtype) && good_idtype(id_dtype), "%s: unsupported dtype", name);
  EXF_REQUIRE(routes >= 0 && experts >= 1 && experts <= 1024, "%s: bad shape", name);
  EXF_REQUIRE(norms && importance, "%s: null pointer", name);
  if (routes == 0) return EXF_OK;
  EXF_REQUIRE(w && ids, "%s: null routing pointer", name);
  return cuda_status(launch_importance(w_dtype, id_dtype, w, ids, routes, experts, norms,
                                       importance, (cudaStream_t)stream),
                     name);
}

EXF_API int exf_decode_apply(const int64_t* importance, const void* w, int w_dtype,
                             const void* ids, int id_dtype, int64_t batch, int top_k,
                             int experts, int budget, int variant, const float* coeff,
                             const float* loss, void* out_w, void* out_ids, int32_t* out_subset,
                             exf_stream_t stream) {
  const char* name = "exf_decode_apply";
  int rc = decode_checks(name, w_dtype, id_dtype, batch, top_k, experts, budget, variant);
  if (rc != EXF_OK) return rc;
  EXF_REQUIRE(importance && coeff && loss, "%s: null pointer", name);
  EXF_REQUIRE(batch == 0 || (w && ids && out_w && out_ids), "%s: null routing pointer", name);
  DecodeParams p{w, ids, batch * top_k, experts, budget, variant, 1 /*importance given*/,
                 nullptr, importance, nullptr, coeff, loss, out_w, out_ids, out_subset};
  return cuda_status(launch_decode(w_dtype, id_dtype, p, (cudaStream_t)stream), name);
}

// ---- sharded decode with the importance exchanged over peer memory ---------------------------
EXF_API int64_t exf_decode_exchange_bytes(int experts, int world) {
  if (experts < 1 || experts > 1024 || world < 1 || world > kMaxPeers) return -1;
  return exchange_longs(experts, world) * (int64_t)sizeof(int64_t);
}

// cuMemGetAddressRange through the runtime's driver entry point (no link against libcuda)
typedef int (*exf_get_range_fn)(unsigned long long*, size_t*, unsigned long long);

static cudaError_t allocation_base(const void* ptr, uintptr_t* base) {
  static exf_get_range_fn fn = nullptr;
  static std::once_flag once;
  static cudaError_t lookup = cudaSuccess;
  std::call_once(once, [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    lookup = cudaGetDriverEntryPoint("cuMemGetAddressRange", &f, cudaEnableDefault, &q);
    if (lookup == cudaSuccess && (q != cudaDriverEntryPointSuccess || f == nullptr))
      lookup = cudaErrorSymbolNotFound;
    fn = reinterpret_cast<exf_get_range_fn>(f);
  });
  if (lookup != cudaSuccess) return lookup;
  unsigned long long b = 0;
  size_t size = 0;
  if (fn(&b, &size, reinterpret_cast<unsigned long long>(ptr)) != 0)
    return cudaErrorInvalidDevicePointer;
  *base = static_cast<uintptr_t>(b);
  return cudaSuccess;
}

EXF_API int exf_ipc_export(const void* ptr, void* handle, int64_t* offset) {
  const char* name = "exf_ipc_export";
  EXF_REQUIRE(ptr && handle && offset, "%s: null pointer", name);
  uintptr_t base = 0;
  cudaError_t e = allocation_base(ptr, &base);
  if (e != cudaSuccess) return cuda_status(e, name);
  cudaIpcMemHandle_t h;
  e = cudaIpcGetMemHandle(&h, reinterpret_cast<void*>(base));
  if (e != cudaSuccess) return cuda_status(e, name);
  memcpy(handle, &h, sizeof(h));
  *offset = static_cast<int64_t>(reinterpret_cast<uintptr_t>(ptr) - base);
  return EXF_OK;
}

EXF_API int exf_ipc_import(const void* handle, int64_t offset, void** ptr) {
  const char* name = "exf_ipc_import";
  EXF_REQUIRE(handle && ptr && offset >= 0, "%s: bad argument", name);
  cudaIpcMemHandle_t h;
  memcpy(&h, handle, sizeof(h));
  void* base = nullptr;
  const cudaError_t e = cudaIpcOpenMemHandle(&base, h, cudaIpcMemLazyEnablePeerAccess);
  if (e != cudaSuccess) return cuda_status(e, name);
  *ptr = static_cast<uint8_t*>(base) + offset;
  return EXF_OK;
}

EXF_API int exf_ipc_release(void* ptr, int64_t offset) {
  const char* name = "exf_ipc_release";
  EXF_REQUIRE(ptr && offset >= 0, "%s: bad argument", name);
  return cuda_status(cudaIpcCloseMemHandle(static_cast<uint8_t*>(ptr) - offset), name);
}

EXF_API int exf_decode_sharded(const void* w, int w_dtype, const void* ids, int id_dtype,
                               int64_t batch, int top_k, int experts, int budget, int variant,
                               const float* norms, const float* coeff, const float* loss,
                               int world, int rank, void* const* peers, uint64_t wait_ns,
                               void* out_w, void* out_ids, int32_t* out_subset, int32_t* status,
                               exf_stream_t stream) {
  const char* name = "exf_decode_sharded";
  int rc = decode_checks(name, w_dtype, id_dtype, batch, top_k, experts, budget, variant);
  if (rc != EXF_OK) return rc;
  EXF_REQUIRE(world >= 1 && world <= kMaxPeers && rank >= 0 && rank < world,
              "%s: world must be in [1, %d] and 0 <= rank < world", name, kMaxPeers);
  EXF_REQUIRE(norms && coeff && loss && peers, "%s: null pointer", name);
  EXF_REQUIRE(batch == 0 || (w && ids && out_w && out_ids), "%s: null routing pointer", name);
  DecodeParams p{w, ids, batch * top_k, experts, budget, variant, kImportanceExchanged, norms,
                 nullptr, nullptr, coeff, loss, out_w, out_ids, out_subset};
  p.world = world;
  p.rank = rank;
  for (int r = 0; r < world; ++r) {
    EXF_REQUIRE(peers[r] && (reinterpret_cast<uintptr_t>(peers[r]) & 63u) == 0,
                "%s: exchange buffer of rank %d is null or not 64-byte aligned", name, r);
    p.peers[r] = static_cast<int64_t*>(peers[r]);
  }
  p.status = status;
  p.wait_ns = wait_ns;
  return cuda_status(launch_decode(w_dtype, id_dtype, p, (cudaStream_t)stream), name);
}

EXF_API int exf_reroute_subset(const void* w, int w_dtype, const void* ids, int id_dtype,
                               int64_t batch, int top_k, int experts, const int32_t* subset,
                               int subset_size, const float* coeff, const float* loss,
                               void* out_w, void* out_ids, exf_stream_t stream) {
  const char* name = "exf_reroute_subset";
  EXF_REQUIRE(subset_size >= 1 && subset_size <= experts, "%s: subset_size must be in [1, experts]",
              name);
  int rc = decode_checks(name, w_dtype, id_dtype, batch, top_k, experts, subset_size, EXF_QWEN3);
  if (rc != EXF_OK) return rc;
  EXF_REQUIRE(subset && coeff && loss, "%s: null pointer", name);
  if (batch == 0) return EXF_OK;
  EXF_REQUIRE(w && ids && out_w && out_ids, "%s: null routing pointer", name);
  DecodeParams p{w, ids, batch * top_k, experts, subset_size, EXF_QWEN3, 2 /*subset given*/,
                 nullptr, nullptr, subset, coeff, loss, out_w, out_ids, nullptr};
  return cuda_status(launch_decode(w_dtype, id_dtype, p, (cudaStream_t)stream), name);
}

EXF_API int exf_static_table(const float* norms, const float* coeff, const float* loss,
                             int experts, int budget, int32_t* target, float* scale,
                             exf_stream_t stream) {
  const char* name = "exf_static_table";
  EXF_REQUIRE(experts >= 1 && experts <= 1024, "%s: experts must be in [1, 1024]", name);
  EXF_REQUIRE(budget >= 1 && budget <= experts, "%s: budget must be in [1, experts]", name);
  EXF_REQUIRE(norms && coeff && loss && target && scale, "%s: null pointer", name);
  return cuda_status(launch_static_table(norms, coeff, loss, experts, budget, target, scale,
                                         (cudaStream_t)stream),
                     name);
}

EXF_API int exf_static_remap(void* w, int w_dtype, void* ids, int id_dtype, int64_t routes,
                             int experts, const int32_t* target, const float* scale,
                             exf_stream_t stream) {
  const char* name = "exf_static_remap";
  EXF_REQUIRE(good_wdtype(w_dtype) && good_idtype(id_dtype), "%s: unsupported dtype", name);
  EXF_REQUIRE(routes >= 0 && experts >= 1, "%s: bad shape", name);
  if (routes == 0) return EXF_OK;
  EXF_REQUIRE(w && ids && target && scale, "%s: null pointer", name);
  return cuda_status(launch_static_remap(w_dtype, id_dtype, w, ids, routes, experts, target, scale,
                                         (cudaStream_t)stream),
                     name);
}

EXF_API int64_t exf_moe_align_capacity(int64_t numel, int experts, int block_size, int pad_sorted) {
  if (numel < 0 || experts < 1 || block_size < 1) return -1;
  int64_t cap = numel + (int64_t)experts * (block_size - 1);
  if (pad_sorted) cap = (cap + block_size - 1) / block_size * block_size;
  if (numel < experts && numel * block_size < cap) cap = numel * block_size;
  return cap;
}

EXF_API int64_t exf_moe_align_workspace_bytes(int64_t numel, int experts) {
  if (numel < 0 || experts < 1) return -1;
  return align_workspace_bytes(numel, experts);
}

// Checks shared by the two moe_align entry points.  The kernels keep expert offsets, the padded
// total and block starts in int32, so the padded total (at most the capacity formula) and the
// capacity must stay below 2^31.
static int align_checks(const char* name, const void* ids, int id_dtype, int64_t numel,
                        int experts, int block_size, int64_t capacity, const int32_t* sorted_ids,
                        const int32_t* expert_ids, const int32_t* num_post_pad) {
  EXF_REQUIRE(good_idtype(id_dtype), "%s: unsupported id dtype", name);
  EXF_REQUIRE(numel >= 0 && numel < (int64_t)1 << 31, "%s: numel out of range", name);
  EXF_REQUIRE(block_size >= 1, "%s: block_size must be >= 1", name);
  if (experts < 1 || experts > align_max_experts())
    return fail(EXF_ERR_UNSUPPORTED, "%s: experts must be in [1, %d]", name, align_max_experts());
  const int64_t padded = exf_moe_align_capacity(numel, experts, block_size, 0);
  EXF_REQUIRE(padded < ((int64_t)1 << 31) && capacity < ((int64_t)1 << 31),
              "%s: %lld routes over %d experts in blocks of %d (capacity %lld) exceed the int32 "
              "offsets: the padded total and the capacity must be below 2^31",
              name, (long long)numel, experts, block_size, (long long)capacity);
  EXF_REQUIRE(capacity >= padded || capacity >= numel * (int64_t)block_size,
              "%s: capacity too small", name);
  EXF_REQUIRE(num_post_pad && (capacity == 0 || (sorted_ids && expert_ids)), "%s: null output",
              name);
  EXF_REQUIRE(numel == 0 || ids, "%s: null ids", name);
  return EXF_OK;
}

EXF_API int exf_moe_align(const void* ids, int id_dtype, int64_t numel, int experts,
                          int block_size, int64_t capacity, int32_t* sorted_ids,
                          int32_t* expert_ids, int32_t* num_post_pad, void* workspace,
                          int64_t workspace_bytes, exf_stream_t stream) {
  const char* name = "exf_moe_align";
  const int rc = align_checks(name, ids, id_dtype, numel, experts, block_size, capacity,
                              sorted_ids, expert_ids, num_post_pad);
  if (rc != EXF_OK) return rc;
  const int64_t need = align_workspace_bytes(numel, experts);
  EXF_REQUIRE(need == 0 || (workspace && workspace_bytes >= need),
              "%s: workspace of %lld bytes required", name, (long long)need);
  AlignParams p{ids, numel, experts, block_size, capacity, sorted_ids, expert_ids, num_post_pad,
                static_cast<int32_t*>(workspace), 0};
  return cuda_status(launch_align(id_dtype, p, (cudaStream_t)stream), name);
}

EXF_API int64_t exf_fused_experts_workspace_bytes(int64_t tokens, int top_k, int experts,
                                                  int hidden, int inter) {
  if (tokens < 0 || top_k < 1 || experts < 1 || hidden < 1 || inter < 1) return -1;
  return moe_workspace(tokens, top_k, experts, hidden, inter, nullptr).bytes;
}

EXF_API int exf_fused_experts(const void* x, const float* topk_w, const int32_t* topk_ids,
                              int64_t tokens, int top_k, const void* w13, const void* w2,
                              int experts, int hidden, int inter, void* y, void* workspace,
                              int64_t workspace_bytes, int32_t* status, exf_stream_t stream) {
  const char* name = "exf_fused_experts";
  EXF_REQUIRE(tokens >= 0 && top_k >= 1 &&
                  tokens * top_k + (int64_t)experts * 127 < ((int64_t)1 << 31),
              "%s: bad routing shape (routes plus block padding must stay below 2^31)", name);
  if (top_k > 8) return fail(EXF_ERR_UNSUPPORTED, "%s: top_k must be at most 8, got %d", name, top_k);
  if (experts < 1 || experts > align_max_experts())
    return fail(EXF_ERR_UNSUPPORTED, "%s: experts must be in [1, %d]", name, align_max_experts());
  if (hidden % 256 != 0 || inter % 128 != 0)
    return fail(EXF_ERR_UNSUPPORTED,
                "%s: hidden must be a multiple of 256 and intermediate a multiple of 128", name);
  if (tokens == 0) return EXF_OK;
  EXF_REQUIRE(x && topk_w && topk_ids && w13 && w2 && y && workspace, "%s: null pointer", name);
  EXF_REQUIRE(aligned16(x) && aligned16(w13) && aligned16(w2) && aligned16(y) &&
                  aligned16(workspace),
              "%s: tensors must be 16-byte aligned", name);
  MoeWorkspace ws = moe_workspace(tokens, top_k, experts, hidden, inter, workspace);
  EXF_REQUIRE(workspace_bytes >= ws.bytes, "%s: workspace of %lld bytes required", name,
              (long long)ws.bytes);
  MoeArgs a{x, topk_w, topk_ids, tokens, top_k, w13, w2, experts, hidden, inter, y, status};
  return cuda_status(launch_moe_experts(a, ws, (cudaStream_t)stream), name);
}

EXF_API int64_t exf_decode_fused_experts_workspace_bytes(int64_t batch, int top_k, int experts,
                                                        int hidden, int inter) {
  if (batch < 0 || top_k < 1 || experts < 1) return -1;
  return decode_moe_workspace_bytes(batch, top_k, experts, hidden, inter);
}

EXF_API int exf_decode_fused_experts(const void* x, const float* w, const int32_t* ids,
                                     int64_t batch, int top_k, int experts, int budget,
                                     int variant, const float* norms, const float* coeff,
                                     const float* loss, const void* w13, const void* w2,
                                     int hidden, int inter, float* out_w, int32_t* out_ids,
                                     void* y, void* workspace, int64_t workspace_bytes,
                                     int32_t* status, exf_stream_t stream) {
  const char* name = "exf_decode_fused_experts";
  int rc = decode_checks(name, EXF_F32, EXF_I32, batch, top_k, experts, budget, variant);
  if (rc != EXF_OK) return rc;
  if (experts > kDecodeAlignMaxExperts || top_k > 8 ||
      batch * top_k > (int64_t)kDecodeAlignMaxRoutes)
    return fail(EXF_ERR_UNSUPPORTED,
                "%s: at most %d experts, top_k <= 8 and %d routes (batch * top_k)", name,
                kDecodeAlignMaxExperts, kDecodeAlignMaxRoutes);
  if (hidden % 256 != 0 || inter % 128 != 0)
    return fail(EXF_ERR_UNSUPPORTED,
                "%s: hidden must be a multiple of 256 and intermediate a multiple of 128", name);
  if (batch == 0) return EXF_OK;
  EXF_REQUIRE(norms && coeff && loss, "%s: null calibration table", name);
  EXF_REQUIRE(x && w && ids && w13 && w2 && out_w && out_ids && y && workspace,
              "%s: null pointer", name);
  EXF_REQUIRE(aligned16(x) && aligned16(w13) && aligned16(w2) && aligned16(y) &&
                  aligned16(workspace),
              "%s: tensors must be 16-byte aligned", name);
  const int64_t need = decode_moe_workspace_bytes(batch, top_k, experts, hidden, inter);
  EXF_REQUIRE(workspace_bytes >= need, "%s: workspace of %lld bytes required", name,
              (long long)need);
  DecodeParams d{w, ids, batch * top_k, experts, budget, variant, 0 /*from routes*/, norms,
                 nullptr, nullptr, coeff, loss, out_w, out_ids, nullptr};
  MoeArgs a{x, out_w, out_ids, batch, top_k, w13, w2, experts, hidden, inter, y, status};
  return cuda_status(launch_decode_moe_experts(d, a, workspace, (cudaStream_t)stream), name);
}

// ---- microscaled 4-bit floating point ----------------------------------------------------------
EXF_API int exf_mxfp4_quantize(const void* x, int dtype, int64_t rows, int64_t cols,
                               int64_t row_stride, uint8_t* codes, uint8_t* scales,
                               exf_stream_t stream) {
  const char* name = "exf_mxfp4_quantize";
  EXF_REQUIRE(good_wdtype(dtype), "%s: dtype must be EXF_F32, EXF_BF16 or EXF_F16", name);
  EXF_REQUIRE(rows >= 0 && cols >= 0 && cols < ((int64_t)1 << 40) &&
                  rows <= ((int64_t)1 << 50) / (cols + 64),
              "%s: bad shape", name);
  EXF_REQUIRE(rows <= 1 || row_stride >= cols, "%s: row_stride is below cols", name);
  if (rows == 0 || cols == 0) return EXF_OK;
  EXF_REQUIRE(x && codes && scales, "%s: null pointer", name);
  EXF_REQUIRE(aligned16(codes), "%s: codes must be 16-byte aligned", name);
  EXF_REQUIRE(reinterpret_cast<uintptr_t>(x) % (dtype == EXF_F32 ? 4 : 2) == 0,
              "%s: x is not aligned to its elements", name);
  return cuda_status(
      launch_mxfp4_quantize(x, dtype, rows, cols, row_stride, codes, scales, (cudaStream_t)stream),
      name);
}

EXF_API int exf_mxfp4_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t rows,
                                 int64_t cols, void* out, int dtype, exf_stream_t stream) {
  const char* name = "exf_mxfp4_dequantize";
  EXF_REQUIRE(good_wdtype(dtype), "%s: dtype must be EXF_F32, EXF_BF16 or EXF_F16", name);
  EXF_REQUIRE(rows >= 0 && cols >= 0 && cols < ((int64_t)1 << 40) &&
                  rows <= ((int64_t)1 << 50) / (cols + 64),
              "%s: bad shape", name);
  if (rows == 0 || cols == 0) return EXF_OK;
  EXF_REQUIRE(codes && scales && out, "%s: null pointer", name);
  EXF_REQUIRE(aligned16(codes) && aligned16(out), "%s: codes and out must be 16-byte aligned",
              name);
  return cuda_status(
      launch_mxfp4_dequantize(codes, scales, rows, cols, out, dtype, (cudaStream_t)stream), name);
}

EXF_API int64_t exf_fused_experts_mxfp4_workspace_bytes(int64_t tokens, int top_k, int experts,
                                                        int hidden, int inter) {
  if (tokens < 0 || top_k < 1 || experts < 1 || hidden < 1 || inter < 1) return -1;
  return mx_workspace(tokens, top_k, experts, hidden, inter, nullptr).bytes;
}

EXF_API int exf_fused_experts_mxfp4(const void* x, const float* topk_w, const int32_t* topk_ids,
                                    int64_t tokens, int top_k, const uint8_t* w13,
                                    const uint8_t* s13, const uint8_t* w2, const uint8_t* s2,
                                    int experts, int hidden, int inter, void* y, void* workspace,
                                    int64_t workspace_bytes, int32_t* status,
                                    exf_stream_t stream) {
  const char* name = "exf_fused_experts_mxfp4";
  EXF_REQUIRE(tokens >= 0 && top_k >= 1 && hidden >= 1 && inter >= 1 && tokens < (1 << 30),
              "%s: bad shape", name);
  EXF_REQUIRE(tokens * top_k + (int64_t)experts * 127 < ((int64_t)1 << 30),
              "%s: bad routing shape (routes plus block padding must stay below 2^30)", name);
  if (top_k > 8) return fail(EXF_ERR_UNSUPPORTED, "%s: top_k must be at most 8, got %d", name, top_k);
  if (experts < 1 || experts > align_max_experts())
    return fail(EXF_ERR_UNSUPPORTED, "%s: experts must be in [1, %d]", name, align_max_experts());
  if (hidden % 256 != 0 || inter % 128 != 0)
    return fail(EXF_ERR_UNSUPPORTED,
                "%s: hidden must be a multiple of 256 and intermediate a multiple of 128", name);
  if (hidden >= (1 << 23) || inter >= (1 << 23) ||
      (int64_t)experts * 2 * inter >= ((int64_t)1 << 31) ||
      (int64_t)experts * hidden >= ((int64_t)1 << 31))
    return fail(EXF_ERR_UNSUPPORTED, "%s: shape too large", name);
  if (tokens == 0) return EXF_OK;
  EXF_REQUIRE(x && topk_w && topk_ids && w13 && s13 && w2 && s2 && y && workspace,
              "%s: null pointer", name);
  EXF_REQUIRE(aligned16(x) && aligned16(y) && aligned16(s13) && aligned16(s2),
              "%s: tensors must be 16-byte aligned", name);
  EXF_REQUIRE(reinterpret_cast<uintptr_t>(w13) % 32 == 0 &&
                  reinterpret_cast<uintptr_t>(w2) % 32 == 0 &&
                  reinterpret_cast<uintptr_t>(workspace) % 32 == 0,
              "%s: weight codes and the workspace must be 32-byte aligned", name);
  const MxWorkspace ws = mx_workspace(tokens, top_k, experts, hidden, inter, workspace);
  EXF_REQUIRE(workspace_bytes >= ws.bytes, "%s: workspace of %lld bytes required", name,
              (long long)ws.bytes);
  MxArgs a{x,       topk_w, topk_ids, tokens, top_k, w13, s13, w2, s2,
           experts, hidden, inter,    y,      status};
  return cuda_status(launch_mx_experts(a, ws, (cudaStream_t)stream), name);
}

// ---- gated feed-forward block --------------------------------------------------------------------
// (a reduction of 2^24 stays far inside the kernels' bounded waits)
static bool gated_too_large(int64_t tokens, int hidden, int inter) {
  return tokens >= (1 << 24) || hidden >= (1 << 23) || inter >= (1 << 23) ||
         ((tokens + 127) / 128) * (((int64_t)inter + 31) / 32) >= ((int64_t)1 << 31) ||
         ((tokens + 127) / 128) * (((int64_t)hidden + 31) / 32) >= ((int64_t)1 << 31) ||
         (((int64_t)inter + 63) / 64) * (((int64_t)hidden + 31) / 32) >= ((int64_t)1 << 31);
}

static int gated_checks(const char* name, int dtype, int64_t tokens, int hidden, int inter,
                        int activation) {
  if (dtype != EXF_BF16 && dtype != EXF_F16)
    return fail(EXF_ERR_UNSUPPORTED, "%s: dtype must be EXF_BF16 or EXF_F16", name);
  EXF_REQUIRE(activation == EXF_SILU || activation == EXF_GELU_TANH, "%s: unknown activation %d",
              name, activation);
  EXF_REQUIRE(tokens >= 0 && hidden >= 1 && inter >= 1, "%s: bad shape", name);
  if (hidden % 8 != 0 || inter % 8 != 0)
    return fail(EXF_ERR_UNSUPPORTED, "%s: hidden and intermediate must be multiples of 8", name);
  if (gated_too_large(tokens, hidden, inter))
    return fail(EXF_ERR_UNSUPPORTED, "%s: shape too large", name);
  return EXF_OK;
}

EXF_API int64_t exf_gated_mlp_workspace_bytes(int64_t tokens, int hidden, int inter) {
  if (tokens < 0 || hidden < 1 || inter < 1 || gated_too_large(tokens, hidden, inter)) return -1;
  return gated_forward_workspace(tokens, hidden, inter);
}

EXF_API int exf_gated_mlp(const void* x, const void* w13, int dtype, int64_t tokens, int hidden,
                          int inter, int activation, void* h, float* pre, void* workspace,
                          int64_t workspace_bytes, int32_t* status, exf_stream_t stream) {
  const char* name = "exf_gated_mlp";
  const int rc = gated_checks(name, dtype, tokens, hidden, inter, activation);
  if (rc != EXF_OK) return rc;
  if (tokens == 0) return EXF_OK;
  EXF_REQUIRE(x && w13 && h, "%s: null pointer", name);
  EXF_REQUIRE(aligned16(x) && aligned16(w13) && aligned16(h) && aligned16(pre) &&
                  aligned16(workspace),
              "%s: tensors must be 16-byte aligned", name);
  EXF_REQUIRE(reinterpret_cast<uintptr_t>(pre) % 32 == 0 &&
                  reinterpret_cast<uintptr_t>(workspace) % 32 == 0,
              "%s: pre and the workspace must be 32-byte aligned", name);
  const int64_t need = gated_forward_workspace(tokens, hidden, inter);
  EXF_REQUIRE(need == 0 || (workspace && workspace_bytes >= need),
              "%s: workspace of %lld bytes required", name, (long long)need);
  GatedArgs a{x, w13, dtype == EXF_BF16, tokens, hidden, inter, activation, status};
  return cuda_status(launch_gated_forward(a, h, pre, workspace, (cudaStream_t)stream), name);
}

EXF_API int64_t exf_gated_mlp_backward_workspace_bytes(int64_t tokens, int hidden, int inter) {
  if (tokens < 0 || hidden < 1 || inter < 1 || gated_too_large(tokens, hidden, inter)) return -1;
  return gated_backward_workspace(tokens, hidden, inter);
}

EXF_API int exf_gated_mlp_backward(const void* dh, const float* pre, const void* x,
                                   const void* w13, int dtype, int64_t tokens, int hidden,
                                   int inter, int activation, void* dx, void* dw13,
                                   void* workspace, int64_t workspace_bytes, int32_t* status,
                                   exf_stream_t stream) {
  const char* name = "exf_gated_mlp_backward";
  const int rc = gated_checks(name, dtype, tokens, hidden, inter, activation);
  if (rc != EXF_OK) return rc;
  if (!dx && !dw13) return EXF_OK;
  if (tokens == 0) {
    if (!dw13) return EXF_OK;
    return cuda_status(
        cudaMemsetAsync(dw13, 0, (size_t)inter * 2 * hidden * 2, (cudaStream_t)stream), name);
  }
  EXF_REQUIRE(dh && pre && workspace && (w13 || !dx) && (x || !dw13), "%s: null pointer", name);
  EXF_REQUIRE(aligned16(dh) && aligned16(pre) && aligned16(x) && aligned16(w13) &&
                  aligned16(dx) && aligned16(dw13) && aligned16(workspace),
              "%s: tensors must be 16-byte aligned", name);
  EXF_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 32 == 0,
              "%s: the workspace must be 32-byte aligned", name);
  const int64_t need = exf_gated_mlp_backward_workspace_bytes(tokens, hidden, inter);
  EXF_REQUIRE(workspace_bytes >= need, "%s: workspace of %lld bytes required", name,
              (long long)need);
  GatedArgs a{x, w13, dtype == EXF_BF16, tokens, hidden, inter, activation, status};
  return cuda_status(
      launch_gated_backward(a, dh, pre, workspace, dx, dw13, (cudaStream_t)stream), name);
}

// ---- root-mean-square norm ------------------------------------------------------------------------
static int norm_checks(const char* name, int dtype, int weight_dtype, int64_t rows, int64_t cols,
                       int64_t x_stride, float eps) {
  EXF_REQUIRE(good_wdtype(dtype), "%s: dtype must be EXF_F32, EXF_BF16 or EXF_F16", name);
  EXF_REQUIRE(weight_dtype == EXF_F32 || weight_dtype == dtype,
              "%s: the weight's dtype must be EXF_F32 or dtype", name);
  EXF_REQUIRE(rows >= 0 && cols >= 1, "%s: bad shape", name);
  if (rows >= ((int64_t)1 << 31) || cols >= (1 << 24))
    return fail(EXF_ERR_UNSUPPORTED, "%s: at most 2^31 - 1 rows and 2^24 - 1 columns", name);
  EXF_REQUIRE(rows <= 1 || x_stride >= cols, "%s: row stride below the row's length", name);
  EXF_REQUIRE(eps >= 0.0f, "%s: eps must not be negative", name);
  return EXF_OK;
}
static bool aligned_to(const void* p, int dtype) {
  return reinterpret_cast<uintptr_t>(p) % (dtype == EXF_F32 ? 4 : 2) == 0;
}

EXF_API int exf_rms_norm(const void* x, int64_t x_stride, const void* residual, int64_t r_stride,
                         const void* weight, int dtype, int weight_dtype, int64_t rows, int64_t cols,
                         float eps, void* sum, void* y, exf_stream_t stream) {
  const char* name = "exf_rms_norm";
  const int rc = norm_checks(name, dtype, weight_dtype, rows, cols, x_stride, eps);
  if (rc != EXF_OK) return rc;
  EXF_REQUIRE(!residual || rows <= 1 || r_stride >= cols, "%s: row stride below the row's length",
              name);
  if (rows == 0) return EXF_OK;
  EXF_REQUIRE(x && weight && y && (!residual || sum), "%s: null pointer", name);
  EXF_REQUIRE(aligned_to(x, dtype) && aligned_to(residual, dtype) && aligned_to(sum, dtype) &&
                  aligned_to(y, dtype) && aligned_to(weight, weight_dtype),
              "%s: a tensor is not aligned to its type", name);
  NormArgs a{x,    x_stride, residual, r_stride, weight, dtype, weight_dtype == EXF_F32,
             rows, (int)cols, eps,     sum};
  return cuda_status(launch_rms_norm(a, y, (cudaStream_t)stream), name);
}

static int code_checks(const char* name, int code, int64_t cols, int group) {
  EXF_REQUIRE(code == EXF_E4M3 || code == EXF_I8, "%s: code must be EXF_E4M3 or EXF_I8", name);
  EXF_REQUIRE(group == 0 || group == 32 || group == 64 || group == 128,
              "%s: group must be 0 (a row), 32, 64 or 128", name);
  if (cols > (1 << 17))
    return fail(EXF_ERR_UNSUPPORTED, "%s: at most 2^17 columns", name);
  return EXF_OK;
}

EXF_API int exf_rms_norm_8bit(const void* x, int64_t x_stride, const void* residual,
                              int64_t r_stride, const void* weight, int dtype, int weight_dtype,
                              int64_t rows, int64_t cols, float eps, int code, int group, void* sum,
                              void* codes, float* scales, exf_stream_t stream) {
  const char* name = "exf_rms_norm_8bit";
  int rc = norm_checks(name, dtype, weight_dtype, rows, cols, x_stride, eps);
  if (rc == EXF_OK) rc = code_checks(name, code, cols, group);
  if (rc != EXF_OK) return rc;
  EXF_REQUIRE(!residual || rows <= 1 || r_stride >= cols, "%s: row stride below the row's length",
              name);
  if (rows == 0) return EXF_OK;
  EXF_REQUIRE(x && weight && codes && scales && (!residual || sum), "%s: null pointer", name);
  EXF_REQUIRE(aligned_to(x, dtype) && aligned_to(residual, dtype) && aligned_to(sum, dtype) &&
                  aligned_to(scales, EXF_F32) && aligned_to(weight, weight_dtype),
              "%s: a tensor is not aligned to its type", name);
  NormArgs a{x,    x_stride, residual, r_stride, weight, dtype, weight_dtype == EXF_F32,
             rows, (int)cols, eps,     sum};
  return cuda_status(launch_rms_norm_8bit(a, code == EXF_I8, group, static_cast<uint8_t*>(codes),
                                          scales, (cudaStream_t)stream),
                     name);
}

EXF_API int exf_dequantize_8bit(const void* codes, int code, const float* scales, int64_t rows,
                                int64_t cols, int group, void* out, int dtype,
                                exf_stream_t stream) {
  const char* name = "exf_dequantize_8bit";
  EXF_REQUIRE(good_wdtype(dtype), "%s: dtype must be EXF_F32, EXF_BF16 or EXF_F16", name);
  EXF_REQUIRE(rows >= 0 && cols >= 1 && rows < ((int64_t)1 << 31), "%s: bad shape", name);
  const int rc = code_checks(name, code, cols, group);
  if (rc != EXF_OK) return rc;
  if (rows == 0) return EXF_OK;
  EXF_REQUIRE(codes && scales && out, "%s: null pointer", name);
  EXF_REQUIRE(aligned16(codes) && aligned16(out) && aligned_to(scales, EXF_F32),
              "%s: codes and out must be 16-byte aligned", name);
  return cuda_status(launch_dequantize_8bit(static_cast<const uint8_t*>(codes), code == EXF_I8,
                                            scales, rows, (int)cols, group, out, dtype,
                                            (cudaStream_t)stream),
                     name);
}

EXF_API int64_t exf_rms_norm_backward_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows < 0 || cols < 1 || rows >= ((int64_t)1 << 31) || cols >= (1 << 24)) return -1;
  return norm_backward_workspace(rows, (int)cols);
}

EXF_API int exf_rms_norm_backward(const void* dy, const void* dsum, const void* x, int64_t x_stride,
                                  const void* weight, int dtype, int weight_dtype, int64_t rows,
                                  int64_t cols, float eps, void* dx, void* dweight, void* workspace,
                                  int64_t workspace_bytes, exf_stream_t stream) {
  const char* name = "exf_rms_norm_backward";
  const int rc = norm_checks(name, dtype, weight_dtype, rows, cols, x_stride, eps);
  if (rc != EXF_OK) return rc;
  if (!dx && !dweight) return EXF_OK;
  if (rows == 0) {
    if (!dweight) return EXF_OK;
    return cuda_status(cudaMemsetAsync(dweight, 0, (size_t)cols * (weight_dtype == EXF_F32 ? 4 : 2),
                                       (cudaStream_t)stream),
                       name);
  }
  EXF_REQUIRE(dy && x && weight && (workspace || !dweight), "%s: null pointer", name);
  EXF_REQUIRE(aligned_to(dy, dtype) && aligned_to(dsum, dtype) && aligned_to(x, dtype) &&
                  aligned_to(dx, dtype) && aligned_to(weight, weight_dtype) &&
                  aligned_to(dweight, weight_dtype) && aligned_to(workspace, EXF_F32),
              "%s: a tensor is not aligned to its type", name);
  const int64_t need = norm_backward_workspace(rows, (int)cols);
  EXF_REQUIRE(!dweight || workspace_bytes >= need, "%s: workspace of %lld bytes required", name,
              (long long)need);
  NormArgs a{x,    x_stride,  nullptr, 0,      weight, dtype, weight_dtype == EXF_F32,
             rows, (int)cols, eps,     nullptr};
  return cuda_status(
      launch_rms_norm_backward(a, dy, dsum, dx, dweight, workspace, (cudaStream_t)stream), name);
}

// ---- balance loss -----------------------------------------------------------------------------------
static int balance_checks(const char* name, int dtype, int groups, int64_t tokens, int experts,
                          int top_k, int scoring) {
  EXF_REQUIRE(good_wdtype(dtype), "%s: logits must be EXF_F32, EXF_BF16 or EXF_F16", name);
  EXF_REQUIRE(scoring == EXF_SOFTMAX || scoring == EXF_SIGMOID,
              "%s: scoring must be EXF_SOFTMAX or EXF_SIGMOID", name);
  EXF_REQUIRE(groups >= 0 && tokens >= 0 && experts >= 1 && top_k >= 1, "%s: bad shape", name);
  if (experts > 1024 || groups > 65535)
    return fail(EXF_ERR_UNSUPPORTED, "%s: at most 1024 experts and 65535 groups", name);
  if (tokens >= ((int64_t)1 << 31) / top_k)
    return fail(EXF_ERR_UNSUPPORTED, "%s: a group's routes must be below 2^31", name);
  return EXF_OK;
}

EXF_API int64_t exf_balance_loss_workspace_bytes(int groups, int64_t tokens, int experts) {
  if (groups < 0 || groups > 65535 || tokens < 0 || tokens >= ((int64_t)1 << 31) || experts < 1 ||
      experts > 1024)
    return -1;
  return groups == 0 ? 0 : balance_workspace(groups, tokens, experts);
}

EXF_API int exf_balance_loss(const void* logits, int dtype, const void* ids, int id_dtype,
                             const uint8_t* mask, int groups, int64_t tokens, int experts, int top_k,
                             int scoring, float* loss, int32_t* counts, int32_t* valid,
                             void* workspace, int64_t workspace_bytes, exf_stream_t stream) {
  const char* name = "exf_balance_loss";
  const int rc = balance_checks(name, dtype, groups, tokens, experts, top_k, scoring);
  if (rc != EXF_OK) return rc;
  EXF_REQUIRE(good_idtype(id_dtype), "%s: ids must be EXF_I32 or EXF_I64", name);
  if (groups == 0) return EXF_OK;
  EXF_REQUIRE(loss && counts && valid, "%s: null pointer", name);
  EXF_REQUIRE(tokens == 0 || (logits && ids && workspace), "%s: null pointer", name);
  EXF_REQUIRE(aligned_to(logits, dtype) && reinterpret_cast<uintptr_t>(workspace) % 8 == 0 &&
                  reinterpret_cast<uintptr_t>(ids) % (id_dtype == EXF_I64 ? 8 : 4) == 0,
              "%s: a tensor is not aligned to its type", name);
  const int64_t need = balance_workspace(groups, tokens, experts);
  EXF_REQUIRE(workspace_bytes >= need, "%s: workspace of %lld bytes required", name,
              (long long)need);
  BalanceArgs a{logits, dtype, mask, groups, tokens, experts, top_k, scoring == EXF_SIGMOID};
  return cuda_status(launch_balance_loss(a, ids, id_dtype == EXF_I64, workspace, loss, counts, valid,
                                         (cudaStream_t)stream),
                     name);
}

EXF_API int exf_balance_loss_backward(const float* dloss, const void* logits, int dtype,
                                      const uint8_t* mask, const int32_t* counts,
                                      const int32_t* valid, int groups, int64_t tokens, int experts,
                                      int top_k, int scoring, void* dlogits, exf_stream_t stream) {
  const char* name = "exf_balance_loss_backward";
  const int rc = balance_checks(name, dtype, groups, tokens, experts, top_k, scoring);
  if (rc != EXF_OK) return rc;
  if (groups == 0 || tokens == 0) return EXF_OK;
  EXF_REQUIRE(dloss && logits && counts && valid && dlogits, "%s: null pointer", name);
  EXF_REQUIRE(aligned_to(logits, dtype) && aligned_to(dlogits, dtype),
              "%s: a tensor is not aligned to its type", name);
  BalanceArgs a{logits, dtype, mask, groups, tokens, experts, top_k, scoring == EXF_SIGMOID};
  return cuda_status(
      launch_balance_loss_backward(a, dloss, counts, valid, dlogits, (cudaStream_t)stream), name);
}

// ---- projection with adapters ----------------------------------------------------------------------
static bool adapted_too_large(int64_t tokens, int64_t inner, int64_t outer, int64_t adapters) {
  return tokens >= (1 << 24) || inner >= (1 << 23) || outer >= (1 << 23) ||
         adapters >= (1 << 24) ||
         ((tokens + 127) / 128) * ((outer + 63) / 64) >= ((int64_t)1 << 31);
}

EXF_API int64_t exf_adapted_linear_workspace_bytes(int64_t tokens, int inner, int outer, int rank) {
  if (tokens < 0 || inner < 1 || outer < 1 || rank < 1 || rank > 128 ||
      adapted_too_large(tokens, inner, outer, 0))
    return -1;
  return adapters_workspace(tokens, rank);
}

EXF_API int exf_adapted_linear(const void* x, const void* w, const void* a, const void* b,
                               const int32_t* ids, const float* scaling, int dtype, int64_t tokens,
                               int inner, int outer, int adapters, int rank, void* y,
                               void* workspace, int64_t workspace_bytes, int32_t* status,
                               exf_stream_t stream) {
  const char* name = "exf_adapted_linear";
  if (dtype != EXF_BF16 && dtype != EXF_F16)
    return fail(EXF_ERR_UNSUPPORTED, "%s: dtype must be EXF_BF16 or EXF_F16", name);
  EXF_REQUIRE(tokens >= 0 && inner >= 1 && outer >= 1 && adapters >= 0 && rank >= 1,
              "%s: bad shape", name);
  if (inner % 8 != 0 || outer % 8 != 0 || rank % 8 != 0)
    return fail(EXF_ERR_UNSUPPORTED, "%s: inner, outer and rank must be multiples of 8", name);
  if (rank > 128) return fail(EXF_ERR_UNSUPPORTED, "%s: rank must be at most 128", name);
  if (adapted_too_large(tokens, inner, outer, adapters))
    return fail(EXF_ERR_UNSUPPORTED, "%s: shape too large", name);
  if (tokens == 0) return EXF_OK;
  EXF_REQUIRE(x && w && ids && y && workspace && (adapters == 0 || (a && b)), "%s: null pointer",
              name);
  EXF_REQUIRE(aligned16(x) && aligned16(w) && aligned16(a) && aligned16(b) && aligned16(y),
              "%s: tensors must be 16-byte aligned", name);
  EXF_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 32 == 0,
              "%s: the workspace must be 32-byte aligned", name);
  EXF_REQUIRE(reinterpret_cast<uintptr_t>(ids) % 4 == 0 && aligned_to(scaling, EXF_F32),
              "%s: a tensor is not aligned to its type", name);
  const int64_t need = adapters_workspace(tokens, rank);
  EXF_REQUIRE(workspace_bytes >= need, "%s: workspace of %lld bytes required", name,
              (long long)need);
  AdapterArgs p{x,     w,     a,     b,        ids,  scaling, dtype == EXF_BF16,
                tokens, inner, outer, adapters, rank, y,       status};
  return cuda_status(launch_adapters(p, workspace, (cudaStream_t)stream), name);
}

// moe_align without any device allocation: the chunk-count table lives in the library's fixed
// scratch array (exf::g_align_static_table) instead of a caller workspace.
EXF_API int exf_moe_align_noalloc(const void* ids, int id_dtype, int64_t numel, int experts,
                                  int block_size, int64_t capacity, int32_t* sorted_ids,
                                  int32_t* expert_ids, int32_t* num_post_pad,
                                  exf_stream_t stream) {
  const char* name = "exf_moe_align_noalloc";
  const int rc = align_checks(name, ids, id_dtype, numel, experts, block_size, capacity,
                              sorted_ids, expert_ids, num_post_pad);
  if (rc != EXF_OK) return rc;
  const int64_t entries = align_workspace_bytes(numel, experts) / (int64_t)sizeof(int32_t);
  const int64_t limit = align_static_table_ints();
  if (entries > limit) {
    const int64_t max_numel = (limit / experts) * 2048;
    return fail(EXF_ERR_INVALID,
                "%s: %lld routes over %d experts need %lld scratch entries but the fixed scratch "
                "holds %lld; at most %lld routes for %d experts (use exf_moe_align with a "
                "workspace for larger inputs)",
                name, (long long)numel, experts, (long long)entries, (long long)limit,
                (long long)max_numel, experts);
  }
  AlignParams p{ids, numel, experts, block_size, capacity, sorted_ids, expert_ids, num_post_pad,
                nullptr, 0};
  return cuda_status(launch_align_static(id_dtype, p, (cudaStream_t)stream), name);
}

// ---- calibration statistics (offline) ------------------------------------------------------
EXF_API int exf_calibration_update(const void* outputs, int out_dtype, const void* ids,
                                   int id_dtype, int64_t tokens, int top_k, int hidden,
                                   int experts, double* dot, double* target_sq,
                                   double* source_sq, double* norm_sum, double* norm_count,
                                   exf_stream_t stream) {
  const char* name = "exf_calibration_update";
  EXF_REQUIRE(good_wdtype(out_dtype) && good_idtype(id_dtype), "%s: unsupported dtype", name);
  EXF_REQUIRE(tokens >= 0, "%s: tokens must be >= 0", name);
  EXF_REQUIRE(top_k >= 1 && top_k <= 8, "%s: top_k must be in [1, 8], got %d", name, top_k);
  EXF_REQUIRE(hidden >= 8 && hidden % 8 == 0, "%s: hidden must be a positive multiple of 8", name);
  EXF_REQUIRE(experts >= 2 && experts <= 1024, "%s: experts must be in [2, 1024]", name);
  if (tokens == 0) return EXF_OK;
  EXF_REQUIRE(outputs && ids && dot && target_sq && source_sq && norm_sum && norm_count,
              "%s: null pointer", name);
  EXF_REQUIRE(aligned16(outputs), "%s: outputs must be 16-byte aligned", name);
  return cuda_status(launch_calib_update(out_dtype, id_dtype, outputs, ids, tokens, top_k, hidden,
                                         experts, dot, target_sq, source_sq, norm_sum, norm_count,
                                         (cudaStream_t)stream),
                     name);
}

EXF_API int exf_calibration_finalize(const double* dot, const double* target_sq,
                                     const double* source_sq, int experts, double ridge,
                                     double clip_min, double clip_max, float* coeff, float* loss,
                                     int32_t* nonfinite, exf_stream_t stream) {
  const char* name = "exf_calibration_finalize";
  EXF_REQUIRE(experts >= 2 && experts <= 1024, "%s: experts must be in [2, 1024]", name);
  EXF_REQUIRE(ridge > 0, "%s: ridge must be positive", name);
  EXF_REQUIRE(clip_min < clip_max, "%s: clip_min must be smaller than clip_max", name);
  EXF_REQUIRE(dot && target_sq && source_sq && coeff && loss, "%s: null pointer", name);
  return cuda_status(launch_calib_finalize(dot, target_sq, source_sq, experts, ridge, clip_min,
                                           clip_max, coeff, loss, nonfinite, (cudaStream_t)stream),
                     name);
}

EXF_API int exf_calibration_norms(const double* norm_sum, const double* norm_count, int experts,
                                  float* norms, exf_stream_t stream) {
  const char* name = "exf_calibration_norms";
  EXF_REQUIRE(experts >= 2 && experts <= 1024, "%s: experts must be in [2, 1024]", name);
  EXF_REQUIRE(norm_sum && norm_count && norms, "%s: null pointer", name);
  return cuda_status(launch_calib_norms(norm_sum, norm_count, experts, norms, (cudaStream_t)stream),
                     name);
}

}  // extern "C"
