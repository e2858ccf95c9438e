// The operators on clustered rows in flash_kmeans_cuda._C: argument checks, autograd
// and scratch memory over the C-ABI. flash_kmeans_cuda/clusters.py documents them.
//
// Calls run on the current stream of the inputs' device. Tensors that are not laid
// out as the C-ABI wants them (dense last dimension, 16-byte aligned rows) are copied.
#include <cmath>
#include <optional>

#include "py_common.h"

namespace fkc_py {
namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void need(bool ok, const char* msg) {
  if (!ok) throw std::runtime_error(msg);
}
// The same about a named tensor.
void need(bool ok, const char* name, const char* msg) {
  if (!ok) throw std::runtime_error(std::string(name) + msg);
}

// The error of the package's ops for a tensor elsewhere.
void need_cuda(const Tensor& t, const char* name) {
  if (!t.is_cuda())
    throw py::value_error(std::string(name) + " must be a CUDA tensor (got " + t.device().str() +
                          ")");
}

void need_on(const Tensor& t, const char* name, const Tensor& first) {
  need_cuda(t, name);
  if (t.device() != first.device())
    throw std::runtime_error(std::string(name) + " must be on " + first.device().str());
}

Tensor workspace(size_t bytes, const Tensor& like) {
  return at::empty({static_cast<int64_t>(bytes > 0 ? bytes : 1)}, like.options().dtype(at::kByte));
}

bool is_64(const Tensor& ids) {
  need(ids.scalar_type() == at::kInt || ids.scalar_type() == at::kLong,
       "ids must be int32 or int64");
  return ids.scalar_type() == at::kLong;
}

Tensor int32_of(const Tensor& t, const char* name, const Tensor& first) {
  need_on(t, name, first);
  need(t.scalar_type() == at::kInt, name, " must be int32");
  return t.contiguous();
}

// Contiguous, in 16-byte aligned memory.
Tensor dense(const Tensor& t) {
  Tensor c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0 ? c : c.clone();
}

// ---------------------------------------------------------------------------
std::tuple<Tensor, Tensor> cluster_order(const Tensor& ids, int64_t n_clusters) {
  need_cuda(ids, "ids");
  need(ids.dim() == 2, "ids must be (B, N)");
  const bool wide = is_64(ids);
  const int64_t B = ids.size(0), N = ids.size(1), K = n_clusters;
  need(K >= 1, "n_clusters must be at least 1");
  const c10::cuda::CUDAGuard guard(ids.device());
  const auto opt = ids.options().dtype(at::kInt);
  if (B == 0 || N == 0) return {at::empty({B, N}, opt), at::zeros({B, K + 1}, opt)};
  const Tensor in = ids.contiguous();
  Tensor order = at::empty({B, N}, opt), offsets = at::empty({B, K + 1}, opt);
  const size_t bytes = fkc_cluster_order_workspace_size(B, N, K);
  const Tensor ws = workspace(bytes, in);
  check_status(fkc_cluster_order(in.data_ptr(), wide, order.data_ptr<int32_t>(),
                                 offsets.data_ptr<int32_t>(), B, N, K, ws.data_ptr(), bytes,
                                 stream_of(in)),
               "cluster_order");
  return {order, offsets};
}

// ---------------------------------------------------------------------------
struct Table {
  int64_t B, N, K, D;
};

Table table_sizes(const Tensor& table, const Tensor& ids) {
  if (table.dim() == 2) return {1, ids.numel(), table.size(0), table.size(1)};
  return {table.size(0), ids.size(1), table.size(1), table.size(2)};
}

Tensor lookup_forward(const Tensor& table, const Tensor& ids, double scale) {
  const Table s = table_sizes(table, ids);
  auto shape = ids.sizes().vec();
  shape.push_back(s.D);
  if (s.B * s.N * s.D == 0 || s.K == 0) return at::zeros(shape, table.options());
  const Tensor t = table.contiguous(), i = ids.contiguous();
  const c10::cuda::CUDAGuard guard(t.device());
  Tensor y = at::empty(shape, t.options());
  check_status(fkc_cluster_lookup(t.data_ptr(), i.data_ptr(), is_64(i), y.data_ptr(), s.B, s.N, s.K,
                                  s.D, dtype_code(t), static_cast<float>(scale), stream_of(t)),
               "cluster_lookup");
  return y;
}

// Gradients are given as they are, not as functions of the inputs.
void need_first_order(const char* what) {
  need(!at::GradMode::is_enabled(), what,
       " is differentiable once: its gradient has no graph (create_graph)");
}

// A tangent of torch.autograd.forward_ad would be dropped here without a word, which reads as a
// derivative of zero.
void need_no_tangent(const Tensor& t, const char* what) {
  need(!t._fw_grad(/*level=*/0).defined(), what,
       " has no forward-mode derivative: an input carries a tangent");
}

class Lookup : public torch::autograd::Function<Lookup> {
 public:
  static Tensor forward(AutogradContext* ctx, const Tensor& table, const Tensor& ids,
                        double scale) {
    ctx->save_for_backward({ids});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["shape"] = table.sizes().vec();
    return lookup_forward(table, ids, scale);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor()};
    need_first_order("cluster_lookup");
    const Tensor ids = ctx->get_saved_variables()[0].contiguous();
    const auto shape = ctx->saved_data["shape"].toIntVector();
    const Tensor dy = grads[0].contiguous();
    const c10::cuda::CUDAGuard guard(dy.device());
    const bool flat = shape.size() == 2;
    const Table s = flat ? Table{1, ids.numel(), shape[0], shape[1]}
                         : Table{shape[0], ids.size(1), shape[1], shape[2]};
    if (s.B * s.N * s.D == 0 || s.K == 0)
      return {at::zeros(shape, dy.options()), Tensor(), Tensor()};
    Tensor dt = at::empty(shape, dy.options());
    const size_t bytes = fkc_cluster_lookup_grad_workspace_size(s.B, s.N, s.K, s.D);
    const Tensor ws = workspace(bytes, dy);
    check_status(fkc_cluster_lookup_grad(
                     dy.data_ptr(), ids.data_ptr(), is_64(ids), dt.data_ptr(), s.B, s.N, s.K, s.D,
                     dtype_code(dy), static_cast<float>(ctx->saved_data["scale"].toDouble()),
                     ws.data_ptr(), bytes, stream_of(dy)),
                 "cluster_lookup");
    return {dt, Tensor(), Tensor()};
  }
};

Tensor cluster_lookup(const Tensor& table, const Tensor& ids, double scale) {
  need_no_tangent(table, "cluster_lookup");
  need_cuda(table, "table");
  need_on(ids, "ids", table);
  dtype_code(table);
  is_64(ids);
  need(table.dim() == 2 || table.dim() == 3, "table must be (K, D) or (B, K, D)");
  if (table.dim() == 3)
    need(ids.dim() == 2 && ids.size(0) == table.size(0), "ids must be (B, N) matching table");
  if (at::GradMode::is_enabled() && table.requires_grad()) return Lookup::apply(table, ids, scale);
  return lookup_forward(table, ids, scale);
}

// ---------------------------------------------------------------------------
// A 4-D tensor as the kernels read it: dense last dimension, rows on 16 bytes.
Tensor gathered(const Tensor& t) {
  bool ok = t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int d = 0; d < 3; ++d) ok = ok && (t.size(d) == 1 || t.stride(d) % 8 == 0);
  return ok ? t : dense(t);
}

void put_strides(const Tensor& t, int64_t* s) {
  for (int d = 0; d < 3; ++d) s[d] = t.size(d) == 1 ? 0 : t.stride(d);
}

void check_q(const Tensor& q) {
  need_cuda(q, "q");
  need(q.dim() == 4, "q must be (batch, q_heads, n_queries, head_dim)");
  if (q.scalar_type() != at::kHalf && q.scalar_type() != at::kBFloat16)
    throw std::runtime_error(std::string("q must be float16 or bfloat16 (got ") +
                             c10::toString(q.scalar_type()) + ")");
  if (q.size(3) % 8 != 0 || q.size(3) < 8 || q.size(3) > 128)
    throw std::runtime_error("head_dim must be a multiple of 8 between 8 and 128 (got " +
                             std::to_string(q.size(3)) + ")");
}

// Sizes that come with q and the clusters: rows = batch * kv_heads.
fkc_attention_desc describe(const Tensor& q, int64_t rows, int64_t n_keys, int64_t n_clusters,
                            int64_t top_k, double scale) {
  const int64_t batch = q.size(0);
  if (batch == 0 ? rows != 0 : rows % batch != 0 || rows == 0 || q.size(1) % (rows / batch) != 0)
    throw std::runtime_error("the clusters have " + std::to_string(rows) + " rows: they must be "
                             "batch * kv_heads, and q_heads a multiple of kv_heads (q is " +
                             std::to_string(batch) + " x " + std::to_string(q.size(1)) + " heads)");
  fkc_attention_desc d{};
  d.q = q.data_ptr();
  put_strides(q, d.q_stride);
  d.batch = batch;
  d.q_heads = q.size(1);
  d.kv_heads = batch == 0 ? 1 : rows / batch;
  d.n_queries = q.size(2);
  d.n_keys = n_keys;
  d.n_clusters = n_clusters;
  d.top_k = top_k;
  d.head_dim = q.size(3);
  d.dtype = dtype_code(q);
  d.scale = scale;
  return d;
}

double scale_of(const Tensor& q, std::optional<double> scale) {
  return scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(q.size(3)));
}

void check_pos(const Tensor& q_pos, const Tensor& q) {
  need(q_pos.dim() == 2 && q_pos.size(0) == q.size(0) && q_pos.size(1) == q.size(2),
       "q_pos must be (batch, n_queries)");
}

Tensor cluster_select(const Tensor& q_in, const Tensor& centroids_in, const Tensor& offsets_in,
                      int64_t top_k, std::optional<Tensor> order, std::optional<Tensor> q_pos,
                      std::optional<Tensor> bias, std::optional<double> scale) {
  check_q(q_in);
  need_on(centroids_in, "centroids", q_in);
  need(centroids_in.dim() == 3 && centroids_in.size(2) == q_in.size(3),
       "centroids must be (batch * kv_heads, n_clusters, head_dim)");
  need(centroids_in.scalar_type() == q_in.scalar_type(), "q and centroids must share dtype");
  const Tensor offsets = int32_of(offsets_in, "offsets", q_in);
  const int64_t rows = centroids_in.size(0), K = centroids_in.size(1);
  need(offsets.dim() == 2 && offsets.size(0) == rows && offsets.size(1) == K + 1,
       "offsets must be (batch * kv_heads, n_clusters + 1)");
  need(top_k >= 0, "top_k must not be negative");
  need(!q_pos.has_value() || order.has_value(), "q_pos needs order");
  const c10::cuda::CUDAGuard guard(q_in.device());
  const Tensor q = gathered(q_in), centroids = dense(centroids_in);
  Tensor ord, pos, bs;
  int64_t N = 1;
  if (order.has_value()) {
    ord = int32_of(*order, "order", q_in);
    need(ord.dim() == 2 && ord.size(0) == rows, "order must be (batch * kv_heads, n_keys)");
    N = ord.size(1);
  } else {
    N = (1ll << 31) - (1ll << 16);  // not read: any position an offset may hold
  }
  fkc_attention_desc d = describe(q, rows, N, K, top_k, scale_of(q, scale));
  if (q_pos.has_value()) {
    pos = int32_of(*q_pos, "q_pos", q_in);
    check_pos(pos, q);
  }
  if (bias.has_value()) {
    need_on(*bias, "bias", q_in);
    need(bias->scalar_type() == at::kFloat && bias->dim() == 2 && bias->size(0) == rows &&
             bias->size(1) == K,
         "bias must be (batch * kv_heads, n_clusters) float32");
    bs = bias->contiguous();
  }
  const auto opt = q.options().dtype(at::kInt);
  if (rows * d.n_queries * top_k == 0) return at::empty({rows, d.n_queries, top_k}, opt);
  if (K == 0 || N == 0) return at::full({rows, d.n_queries, top_k}, -1, opt);
  d.offsets = offsets.data_ptr<int32_t>();
  d.order = ord.defined() ? ord.data_ptr<int32_t>() : nullptr;
  d.q_pos = pos.defined() ? pos.data_ptr<int32_t>() : nullptr;
  Tensor sel = at::empty({rows, d.n_queries, top_k}, opt);
  const size_t bytes = fkc_cluster_select_workspace_size(&d);
  const Tensor ws = workspace(bytes, q);
  check_status(fkc_cluster_select(&d, centroids.data_ptr(),
                                  bs.defined() ? bs.data_ptr<float>() : nullptr,
                                  sel.data_ptr<int32_t>(), ws.data_ptr(), bytes, stream_of(q)),
               "cluster_select");
  return sel;
}

// ---------------------------------------------------------------------------
// The tensors of an attention call, checked and laid out.
struct Attention {
  Tensor q, k, v, sel, order, offsets, q_pos;
  fkc_attention_desc d;
  bool nothing;  // no query, no key or no selection
};

Attention attention_of(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& sel,
                       const Tensor& order, const Tensor& offsets, const Tensor& q_pos,
                       double scale) {
  Attention a;
  check_q(q);
  for (const Tensor* t : {&k, &v}) {
    const char* name = t == &k ? "k" : "v";
    need_on(*t, name, q);
    need(t->scalar_type() == q.scalar_type(), "q, k and v must share dtype");
    need(t->dim() == 4 && t->size(0) == q.size(0) && t->size(3) == q.size(3),
         name, " must be (batch, kv_heads, n_keys, head_dim)");
  }
  need(k.size(1) == v.size(1) && k.size(2) == v.size(2), "k and v must have the same sizes");
  const int64_t rows = k.size(0) * k.size(1), N = k.size(2);
  a.sel = int32_of(sel, "sel", q);
  a.order = int32_of(order, "order", q);
  a.offsets = int32_of(offsets, "offsets", q);
  need(a.sel.dim() == 3 && a.sel.size(0) == rows && a.sel.size(1) == q.size(2),
       "sel must be (batch * kv_heads, n_queries, top_k)");
  need(a.order.dim() == 2 && a.order.size(0) == rows && a.order.size(1) == N,
       "order must be (batch * kv_heads, n_keys)");
  need(a.offsets.dim() == 2 && a.offsets.size(0) == rows && a.offsets.size(1) >= 1,
       "offsets must be (batch * kv_heads, n_clusters + 1)");
  a.q = gathered(q);
  a.k = gathered(k);
  a.v = gathered(v);
  a.d = describe(a.q, rows, N, a.offsets.size(1) - 1, a.sel.size(2), scale);
  if (q_pos.defined()) {
    a.q_pos = int32_of(q_pos, "q_pos", q);
    check_pos(a.q_pos, q);
    a.d.q_pos = a.q_pos.data_ptr<int32_t>();
  }
  a.d.k = a.k.data_ptr();
  a.d.v = a.v.data_ptr();
  put_strides(a.k, a.d.k_stride);
  put_strides(a.v, a.d.v_stride);
  a.d.sel = a.sel.data_ptr<int32_t>();
  a.d.order = a.order.data_ptr<int32_t>();
  a.d.offsets = a.offsets.data_ptr<int32_t>();
  a.nothing = q.numel() == 0 || rows * N * a.d.n_clusters * a.d.top_k == 0;
  return a;
}

std::tuple<Tensor, Tensor> attention_forward(const Attention& a) {
  const auto sizes = a.q.sizes();
  const auto fl = a.q.options().dtype(at::kFloat);
  if (a.nothing)
    return {at::zeros(sizes, a.q.options()),
            at::full(sizes.slice(0, 3), -std::numeric_limits<double>::infinity(), fl)};
  Tensor out = at::empty(sizes, a.q.options()), lse = at::empty(sizes.slice(0, 3), fl);
  const size_t bytes = fkc_cluster_attention_workspace_size(&a.d);
  const Tensor ws = bytes > 0 ? workspace(bytes, a.q) : Tensor();
  check_status(fkc_cluster_attention(&a.d, out.data_ptr(), lse.data_ptr<float>(),
                                     bytes > 0 ? ws.data_ptr() : nullptr, bytes, stream_of(a.q)),
               "cluster_attention");
  return {out, lse};
}

class Attend : public torch::autograd::Function<Attend> {
 public:
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k,
                               const Tensor& v, const Tensor& sel, const Tensor& order,
                               const Tensor& offsets, const std::optional<Tensor>& q_pos,
                               double scale) {
    const c10::cuda::CUDAGuard guard(q.device());
    const Attention a =
        attention_of(q, k, v, sel, order, offsets, q_pos.value_or(Tensor()), scale);
    auto [out, lse] = attention_forward(a);
    ctx->save_for_backward({q, k, v, a.sel, a.order, a.offsets, a.q_pos, lse});
    ctx->saved_data["scale"] = scale;
    ctx->mark_non_differentiable({lse});
    return {out, lse};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list none(8);
    if (!grads[0].defined()) return none;
    need_first_order("cluster_attention");
    const auto s = ctx->get_saved_variables();
    const c10::cuda::CUDAGuard guard(s[0].device());
    Attention a = attention_of(s[0], s[1], s[2], s[3], s[4], s[5], s[6],
                               ctx->saved_data["scale"].toDouble());
    const Tensor& lse = s[7];
    const Tensor dout = dense(grads[0]);
    const bool want_q = ctx->needs_input_grad(0);
    const bool want_kv = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);
    Tensor dq, dk, dv;
    auto like = [&](const Tensor& t) {
      return a.nothing ? at::zeros(t.sizes(), t.options()) : at::empty(t.sizes(), t.options());
    };
    if (want_q) dq = like(a.q);
    if (want_kv) dk = like(a.k), dv = like(a.v);
    if (!a.nothing && (want_q || want_kv)) {
      const size_t bytes = fkc_cluster_attention_grad_workspace_size(&a.d);
      const Tensor ws = workspace(bytes, dout);
      check_status(fkc_cluster_attention_grad(
                       &a.d, nullptr, lse.data_ptr<float>(), dout.data_ptr(),
                       want_q ? dq.data_ptr() : nullptr, want_kv ? dk.data_ptr() : nullptr,
                       want_kv ? dv.data_ptr() : nullptr, ws.data_ptr(), bytes, stream_of(dout)),
                   "cluster_attention");
    }
    none[0] = dq;
    if (ctx->needs_input_grad(1)) none[1] = dk;
    if (ctx->needs_input_grad(2)) none[2] = dv;
    return none;
  }
};

std::tuple<Tensor, Tensor> cluster_attention(const Tensor& q, const Tensor& k, const Tensor& v,
                                             const Tensor& sel, const Tensor& order,
                                             const Tensor& offsets, std::optional<Tensor> q_pos,
                                             std::optional<double> scale) {
  for (const Tensor* t : {&q, &k, &v}) need_no_tangent(*t, "cluster_attention");
  check_q(q);
  const double sc = scale_of(q, scale);
  if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad())) {
    const auto r = Attend::apply(q, k, v, sel, order, offsets, q_pos, sc);
    return {r[0], r[1]};
  }
  const c10::cuda::CUDAGuard guard(q.device());
  return attention_forward(
      attention_of(q, k, v, sel, order, offsets, q_pos.value_or(Tensor()), sc));
}

}  // namespace

void bind_clusters(py::module_& m) {
  m.def("cluster_order", &cluster_order, py::arg("ids"), py::arg("n_clusters"),
        "positions grouped by id: (order, offsets)");
  m.def("cluster_lookup", &cluster_lookup, py::arg("table"), py::arg("ids"), py::arg("scale"),
        "scale * table[ids], differentiable in table");
  m.def("cluster_select", &cluster_select, py::arg("q"), py::arg("centroids"), py::arg("offsets"),
        py::arg("top_k"), py::arg("order"), py::arg("q_pos"), py::arg("bias"), py::arg("scale"),
        "the top_k clusters for each query");
  m.def("cluster_attention", &cluster_attention, py::arg("q"), py::arg("k"), py::arg("v"),
        py::arg("sel"), py::arg("order"), py::arg("offsets"), py::arg("q_pos"), py::arg("scale"),
        "attention over the keys of the selected clusters: (out, lse)");
}

}  // namespace fkc_py
