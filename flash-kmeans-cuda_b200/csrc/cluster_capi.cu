// extern "C" entry points of the operators on clustered rows: grouping, lookup and
// its gradient, selection and attention (declared in include/fkc_capi.h). Every
// argument is checked here, on the host, before anything is launched.
#include "cluster_attention.cuh"
#include "fkc_internal.h"

namespace fkc {
namespace {

constexpr int64_t kMaxRows = (1ll << 31) - (1ll << 16);  // room for the last step's overshoot

int check_workspace(const char* what, const void* ws, size_t bytes, size_t need) {
  if (need == 0) return FKC_OK;
  if (ws == nullptr || bytes < need)
    return set_error(FKC_EWORKSPACE, "%s workspace needs %zu bytes (got %zu)", what, need, bytes);
  FKC_REQUIRE((reinterpret_cast<uintptr_t>(ws) & 255u) == 0, "workspace must be 256-byte aligned");
  return FKC_OK;
}

int check_group(int64_t B, int64_t N, int64_t K) {
  FKC_REQUIRE(B >= 1 && N >= 1 && K >= 1, "B, N and K must be >= 1 (got %lld, %lld, %lld)",
              static_cast<long long>(B), static_cast<long long>(N), static_cast<long long>(K));
  FKC_REQUIRE(N <= kMaxRows && K < kMaxRows && B <= kMaxRows, "B, N and K must fit int32");
  // the grids: a CTA per chunk of at least 1024 positions, or per 32 counters
  FKC_REQUIRE(B <= (1 << 20) && B * N <= (1ll << 40) && B * K <= (1ll << 40),
              "B must be at most 2^20, B * N and B * K at most 2^40");
  return FKC_OK;
}

bool ids_aligned(const void* ids, int ids_64) {
  return (reinterpret_cast<uintptr_t>(ids) & (ids_64 ? 7u : 3u)) == 0;
}

int check_table(int64_t B, int64_t N, int64_t K, int64_t D, int dtype) {
  FKC_TRY(check_group(B, N, K));
  FKC_REQUIRE(dtype_valid(dtype), "dtype must be FKC_DTYPE_F16, BF16 or F32 (got %d)", dtype);
  FKC_REQUIRE(D >= 1 && D <= (1 << 20), "D must be between 1 and 2^20");
  return FKC_OK;
}

// The checks that selection and attention share; fills the kernels' arguments.
int fill_args(const fkc_attention_desc* d, bool attention, attn::Args* out) {
  FKC_REQUIRE(d != nullptr, "descriptor must be non-null");
  const int64_t big = kMaxRows;
  FKC_REQUIRE(d->batch >= 1 && d->q_heads >= 1 && d->kv_heads >= 1 && d->n_queries >= 1 &&
                  d->n_keys >= 1 && d->n_clusters >= 1 && d->top_k >= 1 && d->head_dim >= 1,
              "every size of the descriptor must be >= 1");
  FKC_REQUIRE(d->q_heads % d->kv_heads == 0, "q_heads must be a multiple of kv_heads");
  FKC_REQUIRE(d->q_heads <= (1 << 16), "q_heads must be at most 2^16");
  FKC_REQUIRE(d->dtype == FKC_DTYPE_F16 || d->dtype == FKC_DTYPE_BF16,
              "dtype must be FKC_DTYPE_F16 or FKC_DTYPE_BF16 (got %d)", d->dtype);
  FKC_REQUIRE(d->head_dim % 8 == 0 && d->head_dim <= 128,
              "head_dim must be a multiple of 8, at most 128 (got %lld)",
              static_cast<long long>(d->head_dim));
  FKC_REQUIRE(d->batch <= big && d->n_queries <= big && d->n_keys <= big && d->n_clusters <= big,
              "sizes must fit int32");
  FKC_REQUIRE(d->batch * d->kv_heads <= (1 << 20), "batch * kv_heads must be at most 2^20");
  FKC_REQUIRE(d->batch * d->q_heads <= big / d->n_queries, "batch * q_heads * n_queries must fit int32");
  FKC_REQUIRE(d->top_k <= 1024, "top_k must be at most 1024");
  FKC_REQUIRE(d->n_queries <= big / d->top_k, "n_queries * top_k must fit int32");
  FKC_REQUIRE(d->q != nullptr && d->offsets != nullptr, "q and offsets must be non-null");
  auto rows_ok = [](const void* p, const int64_t* s) {
    return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && s[0] % 8 == 0 && s[1] % 8 == 0 &&
           s[2] % 8 == 0;
  };
  FKC_REQUIRE(rows_ok(d->q, d->q_stride), "rows of q must be 16-byte aligned");
  attn::Args a{};
  if (attention) {
    FKC_REQUIRE(d->k != nullptr && d->v != nullptr && d->sel != nullptr && d->order != nullptr,
                "k, v, sel and order must be non-null");
    FKC_REQUIRE(rows_ok(d->k, d->k_stride) && rows_ok(d->v, d->v_stride),
                "rows of k and v must be 16-byte aligned");
    FKC_REQUIRE(d->top_k * d->n_keys <= (1ll << 30), "top_k * n_keys must be at most 2^30");
  } else {
    FKC_REQUIRE(d->n_clusters <= 16384, "selection takes at most 16384 clusters");
    FKC_REQUIRE(d->q_pos == nullptr || d->order != nullptr, "q_pos needs order");
  }
  a.q = d->q;
  a.k = d->k;
  a.v = d->v;
  a.qs = {d->q_stride[0], d->q_stride[1], d->q_stride[2]};
  a.ks = {d->k_stride[0], d->k_stride[1], d->k_stride[2]};
  a.vs = {d->v_stride[0], d->v_stride[1], d->v_stride[2]};
  a.sel = d->sel;
  a.order = d->order;
  a.offsets = d->offsets;
  a.q_pos = d->q_pos;
  a.batch = static_cast<int>(d->batch);
  a.Hq = static_cast<int>(d->q_heads);
  a.Hkv = static_cast<int>(d->kv_heads);
  a.G = a.Hq / a.Hkv;
  a.Nq = static_cast<int>(d->n_queries);
  a.N = static_cast<int>(d->n_keys);
  a.K = static_cast<int>(d->n_clusters);
  a.top = static_cast<int>(d->top_k);
  a.D = static_cast<int>(d->head_dim);
  a.scale = static_cast<float>(d->scale);
  *out = a;
  return FKC_OK;
}

cudaStream_t as_stream(fkc_stream_t s) { return reinterpret_cast<cudaStream_t>(s); }

int check_device() {
  const DeviceInfo* di = nullptr;
  FKC_TRY(current_device_info(&di));
  if (di->cc_major != 10)
    return set_error(FKC_EUNSUPPORTED, "device is sm_%d%d, this library is built for sm_100a",
                     di->cc_major, di->cc_minor);
  return FKC_OK;
}

}  // namespace
}  // namespace fkc

using namespace fkc;

extern "C" {

FKC_CAPI_EXPORT size_t fkc_cluster_order_workspace_size(int64_t B, int64_t N, int64_t K) {
  if (check_group(B, N, K) != FKC_OK) return 0;
  return group_workspace_bytes(B, N, K);
}

FKC_CAPI_EXPORT int fkc_cluster_order(const void* ids, int ids_64, int32_t* order,
                                      int32_t* offsets, int64_t B, int64_t N, int64_t K,
                                      void* workspace, size_t workspace_bytes,
                                      fkc_stream_t stream) {
  clear_error();
  FKC_TRY(check_group(B, N, K));
  FKC_REQUIRE(ids != nullptr && order != nullptr && offsets != nullptr,
              "ids, order and offsets must be non-null");
  FKC_REQUIRE(ids_aligned(ids, ids_64), "ids must be aligned to their type");
  FKC_TRY(check_workspace("order", workspace, workspace_bytes, group_workspace_bytes(B, N, K)));
  FKC_TRY(check_device());
  return launch_group(ids, ids_64 != 0, N, order, offsets, B, N, K, workspace, as_stream(stream));
}

FKC_CAPI_EXPORT int fkc_cluster_lookup(const void* table, const void* ids, int ids_64, void* y,
                                       int64_t B, int64_t N, int64_t K, int64_t D, int dtype,
                                       float scale, fkc_stream_t stream) {
  clear_error();
  FKC_TRY(check_table(B, N, K, D, dtype));
  FKC_REQUIRE(table != nullptr && ids != nullptr && y != nullptr,
              "table, ids and y must be non-null");
  FKC_REQUIRE(ids_aligned(ids, ids_64), "ids must be aligned to their type");
  FKC_TRY(check_device());
  return launch_lookup(table, ids, ids_64 != 0, y, B, N, K, D, dtype, scale, as_stream(stream));
}

FKC_CAPI_EXPORT size_t fkc_cluster_lookup_grad_workspace_size(int64_t B, int64_t N, int64_t K,
                                                              int64_t D) {
  if (check_table(B, N, K, D, FKC_DTYPE_F32) != FKC_OK) return 0;
  return lookup_grad_workspace_bytes(B, N, K, D);
}

FKC_CAPI_EXPORT int fkc_cluster_lookup_grad(const void* dy, const void* ids, int ids_64,
                                            void* dtable, int64_t B, int64_t N, int64_t K,
                                            int64_t D, int dtype, float scale, void* workspace,
                                            size_t workspace_bytes, fkc_stream_t stream) {
  clear_error();
  FKC_TRY(check_table(B, N, K, D, dtype));
  FKC_REQUIRE(dy != nullptr && ids != nullptr && dtable != nullptr,
              "dy, ids and dtable must be non-null");
  FKC_REQUIRE(ids_aligned(ids, ids_64), "ids must be aligned to their type");
  FKC_TRY(check_workspace("lookup gradient", workspace, workspace_bytes,
                          lookup_grad_workspace_bytes(B, N, K, D)));
  FKC_TRY(check_device());
  return launch_lookup_grad(dy, ids, ids_64 != 0, dtable, B, N, K, D, dtype, scale, workspace,
                            as_stream(stream));
}

FKC_CAPI_EXPORT size_t fkc_cluster_select_workspace_size(const fkc_attention_desc* desc) {
  attn::Args a;
  if (fill_args(desc, false, &a) != FKC_OK) return 0;
  return attn::select_workspace_bytes(static_cast<int64_t>(a.batch) * a.Hkv, a.Nq, a.K);
}

FKC_CAPI_EXPORT int fkc_cluster_select(const fkc_attention_desc* desc, const void* centroids,
                                       const float* bias, int32_t* sel, void* workspace,
                                       size_t workspace_bytes, fkc_stream_t stream) {
  clear_error();
  attn::Args a;
  FKC_TRY(fill_args(desc, false, &a));
  FKC_REQUIRE(centroids != nullptr && sel != nullptr, "centroids and sel must be non-null");
  FKC_REQUIRE((reinterpret_cast<uintptr_t>(centroids) & 15u) == 0,
              "rows of centroids must be 16-byte aligned");
  FKC_TRY(check_workspace("select", workspace, workspace_bytes,
                          attn::select_workspace_bytes(static_cast<int64_t>(a.batch) * a.Hkv, a.Nq,
                                                       a.K)));
  FKC_TRY(check_device());
  return attn::launch_select(a, centroids, bias, desc->scale, desc->dtype, sel, workspace,
                             as_stream(stream));
}

FKC_CAPI_EXPORT size_t fkc_cluster_attention_workspace_size(const fkc_attention_desc* desc) {
  attn::Args a;
  if (fill_args(desc, true, &a) != FKC_OK) return 0;
  return attn::forward_workspace_bytes(a);
}

FKC_CAPI_EXPORT int fkc_cluster_attention(const fkc_attention_desc* desc, void* out, float* lse,
                                          void* workspace, size_t workspace_bytes,
                                          fkc_stream_t stream) {
  clear_error();
  attn::Args a;
  FKC_TRY(fill_args(desc, true, &a));
  FKC_REQUIRE(out != nullptr && lse != nullptr, "out and lse must be non-null");
  FKC_REQUIRE((reinterpret_cast<uintptr_t>(out) & 15u) == 0, "out must be 16-byte aligned");
  FKC_TRY(check_workspace("attention", workspace, workspace_bytes,
                          attn::forward_workspace_bytes(a)));
  FKC_TRY(check_device());
  return attn::launch_forward(a, desc->dtype, out, lse, workspace, as_stream(stream));
}

FKC_CAPI_EXPORT size_t fkc_cluster_attention_grad_workspace_size(const fkc_attention_desc* desc) {
  attn::Args a;
  if (fill_args(desc, true, &a) != FKC_OK) return 0;
  return attn::backward_workspace_bytes(a);
}

FKC_CAPI_EXPORT int fkc_cluster_attention_grad(const fkc_attention_desc* desc, const void* out,
                                               const float* lse, const void* dout, void* dq,
                                               void* dk, void* dv, void* workspace,
                                               size_t workspace_bytes, fkc_stream_t stream) {
  clear_error();
  attn::Args a;
  FKC_TRY(fill_args(desc, true, &a));
  FKC_REQUIRE(lse != nullptr && dout != nullptr, "lse and dout must be non-null");
  FKC_REQUIRE((dk == nullptr) == (dv == nullptr), "dk and dv go together");
  for (const void* p : {out, dout, static_cast<const void*>(dq), static_cast<const void*>(dk),
                        static_cast<const void*>(dv)})
    FKC_REQUIRE((reinterpret_cast<uintptr_t>(p) & 15u) == 0,
                "out, dout and the gradients must be 16-byte aligned");
  FKC_TRY(check_workspace("attention gradient", workspace, workspace_bytes,
                          attn::backward_workspace_bytes(a)));
  FKC_TRY(check_device());
  return attn::launch_backward(a, desc->dtype, lse, dout, dq, dk, dv, workspace, as_stream(stream));
}

}  // extern "C"
