// Host path of rotary positions, the 4-bit key / value cache and attention over it.
#include <ATen/ops/empty_like.h>
#include <cmath>

#include "host.h"

namespace {

using namespace bsp_host;

// ---- rotary positions --------------------------------------------------------------------------
struct RotaryOp : torch::CustomClassHolder {
  Tensor table;                            // [2, pairs] int64 on one device: turns, axes
  int64_t head_dim, axes;
  bool interleaved;
};

struct Positions {
  const void* at = nullptr;
  int bytes = 0;
  int64_t sa = 0, sz = 0, sl = 0;
};

// [L], [axes, L] or [axes, Z, L] whole numbers; dimensions of size 1 are shared by the batch.
Positions positions_of(const OptTensor& pos, const RotaryOp& p, const Tensor& q) {
  Positions r;
  const int64_t Z = q.size(0), L = q.size(2);
  if (!pos) {
    TORCH_CHECK_VALUE(p.axes == 1, "rotary: positions are needed for ", p.axes, " axes");
    return r;
  }
  TORCH_CHECK(pos->device() == q.device(), "rotary: the positions are on ", pos->device(), ", the call runs on ", q.device());
  TORCH_CHECK_VALUE(pos->scalar_type() == at::kInt || pos->scalar_type() == at::kLong,
                    "rotary: positions must be int32 or int64 (got ", pos->scalar_type(), ")");
  const int64_t d = pos->dim();
  TORCH_CHECK_VALUE(d >= 1 && d <= 3 && pos->size(d - 1) == L && (d < 2 ? p.axes == 1 : pos->size(0) == p.axes) &&
                        (d < 3 || pos->size(1) == Z || pos->size(1) == 1),
                    "rotary: positions must be [", p.axes, ", ", Z, ", ", L, "], [", p.axes, ", ", L, "]",
                    p.axes == 1 ? " or, for one axis, [L]" : "", " (got ", pos->sizes(), ")");
  r.at = pos->const_data_ptr();
  r.bytes = static_cast<int>(pos->element_size());
  r.sl = pos->stride(d - 1);
  if (d > 1) r.sa = pos->stride(0);
  if (d == 3 && pos->size(1) > 1) r.sz = pos->stride(1);
  return r;
}

// Rows with a unit stride; where they are read in pairs, also on a boundary of a pair's size.
Tensor even_rows(const Tensor& x, bool pairs) {
  const int64_t even = pairs ? 2 : 1;
  bool ok = x.stride(3) == 1 && reinterpret_cast<uintptr_t>(x.const_data_ptr()) % (even * x.element_size()) == 0;
  for (int i = 0; i < 3; ++i) ok = ok && (x.size(i) == 1 || x.stride(i) % even == 0);
  return ok ? x : x.clone(at::MemoryFormat::Contiguous);
}
// The result, in the memory order of x.
Tensor rotary_out(const Tensor& x) {
  Tensor y = at::empty_like(x);
  return y.stride(3) == 1 ? y : at::empty(x.sizes(), x.options());
}

std::pair<Tensor, Tensor> rotary(const RotaryOp& p, const OptTensor& q0, const OptTensor& k0, const OptTensor& pos, bool inverse) {
  const Tensor& any = q0 ? *q0 : *k0;
  const c10::cuda::CUDAGuard guard(any.device());
  const Positions at = positions_of(pos, p, any);
  Tensor x[2], y[2];
  int64_t s[2][6] = {};
  for (int i = 0; i < 2; ++i) {
    const OptTensor& t = i ? k0 : q0;
    if (!t) continue;
    x[i] = even_rows(*t, p.interleaved);
    y[i] = rotary_out(x[i]);
    for (int j = 0; j < 3; ++j) {
      s[i][j] = x[i].stride(j);
      s[i][3 + j] = y[i].stride(j);
    }
  }
  auto in = [&](int i) { return x[i].defined() ? x[i].const_data_ptr() : nullptr; };
  auto out = [&](int i) { return y[i].defined() ? y[i].mutable_data_ptr() : nullptr; };
  auto heads = [&](int i) { return x[i].defined() ? x[i].size(1) : 0; };
  check(bsp_rotary(in(0), out(0), heads(0), s[0][0], s[0][1], s[0][2], s[0][3], s[0][4], s[0][5], in(1), out(1), heads(1), s[1][0],
                   s[1][1], s[1][2], s[1][3], s[1][4], s[1][5], dtype_code(any), any.size(0), any.size(2), any.size(3),
                   p.table.size(1), p.interleaved, p.table.const_data_ptr<int64_t>(), p.axes, at.at, at.bytes, at.sa, at.sz, at.sl,
                   inverse, stream_of(any)));
  return {y[0], y[1]};
}

std::pair<Tensor, Tensor> rotary_recorded(const c10::intrusive_ptr<RotaryOp>& p, const OptTensor& q, const OptTensor& k,
                                          const OptTensor& pos, bool inverse);

struct RotaryFn : torch::autograd::Function<RotaryFn> {
  static variable_list forward(AutogradContext* ctx, const c10::intrusive_ptr<RotaryOp>& p, const OptTensor& q, const OptTensor& k,
                               const OptTensor& pos, bool inverse) {
    ctx->set_materialize_grads(false);
    ctx->saved_data["p"] = c10::IValue::make_capsule(p);
    ctx->saved_data["inverse"] = inverse;
    ctx->saved_data["q"] = q.has_value();
    if (pos) ctx->save_for_backward({*pos});
    auto [yq, yk] = rotary(*p, q, k, pos, inverse);
    // (an operand that needs no gradient: its result needs none either, and the backward does not turn one for it)
    if (q && k && needs_grad(*q) != needs_grad(*k)) ctx->mark_non_differentiable({needs_grad(*q) ? yk : yq});
    if (!q) return {yk};
    return k ? variable_list{yq, yk} : variable_list{yq};
  }
  // The turn back; a gradient of its own, so that it can be differentiated again.
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const auto p = c10::static_intrusive_pointer_cast<RotaryOp>(ctx->saved_data["p"].toCapsule());
    const variable_list saved = ctx->get_saved_variables();
    const OptTensor pos = saved.empty() ? OptTensor() : OptTensor(saved[0]);
    const bool has_q = ctx->saved_data["q"].toBool();
    OptTensor dq, dk;
    if (has_q && grads[0].defined()) dq = grads[0];
    const size_t at = has_q ? 1 : 0;
    if (grads.size() > at && grads[at].defined()) dk = grads[at];
    variable_list out(5);
    if (!dq && !dk) return out;
    auto [q, k] = rotary_recorded(p, dq, dk, pos, !ctx->saved_data["inverse"].toBool());
    out[1] = q;
    out[2] = k;
    return out;
  }
};

std::pair<Tensor, Tensor> rotary_recorded(const c10::intrusive_ptr<RotaryOp>& p, const OptTensor& q, const OptTensor& k,
                                          const OptTensor& pos, bool inverse) {
  auto is = [](const OptTensor& t) { return t && recorded(*t); };
  if (!is(q) && !is(k)) return rotary(*p, q, k, pos, inverse);
  const variable_list y = RotaryFn::apply(p, q, k, pos, inverse);
  if (!q) return {Tensor(), y[0]};
  return {y[0], k ? y[1] : Tensor()};
}

void check_rotary(const RotaryOp& p, const Tensor& x, const char* what) {
  TORCH_CHECK_VALUE(x.dim() == 4 && x.size(3) == p.head_dim, "rotary: ", what, " must be [Z, H, L, ", p.head_dim, "] (got ", x.sizes(), ")");
  require_cuda(x);
  dtype_code(x);
  TORCH_CHECK_NOT_IMPLEMENTED(x.size(0) <= INT32_MAX && x.size(1) <= INT32_MAX && x.size(2) <= INT32_MAX, "rotary: too many tokens ", x.sizes());
  TORCH_CHECK(x.device() == p.table.device(), "rotary: ", what, " is on ", x.device(), ", the call runs on ", p.table.device());
}

void check_rotary_call(const c10::intrusive_ptr<RotaryOp>& p, const Tensor& q, const OptTensor& k) {
  check_rotary(*p, q, "the query");
  if (k) {
    check_rotary(*p, *k, "the key");
    require_same(*k, q, "rotary: the key");
    TORCH_CHECK_VALUE(k->size(0) == q.size(0) && k->size(2) == q.size(2), "rotary: query ", q.sizes(), " and key ", k->sizes(),
                      " differ in batch or length");
  }
}

std::pair<Tensor, OptTensor> rotary_call(const c10::intrusive_ptr<RotaryOp>& p, const Tensor& q, const OptTensor& k,
                                         const OptTensor& pos) {
  check_rotary_call(p, q, k);
  auto [yq, yk] = rotary_recorded(p, q, k, pos, false);
  return {yq, yk.defined() ? OptTensor(yk) : OptTensor()};
}

// ---- the 4-bit cache ---------------------------------------------------------------------------
struct CacheOp : torch::CustomClassHolder {
  Tensor data;                             // [pages, heads, page bytes] uint8
  int64_t page, head_dim;
  int64_t pages() const { return data.size(0); }
  int64_t heads() const { return data.size(1); }
};

// int32 [Z] on the cache's device, without gaps.
const int32_t* per_sequence(const OptTensor& t, int64_t Z, const CacheOp& c, const char* what) {
  if (!t) return nullptr;
  TORCH_CHECK(t->device() == c.data.device(), what, " is on ", t->device(), ", the cache on ", c.data.device());
  TORCH_CHECK_VALUE(t->scalar_type() == at::kInt && t->dim() == 1 && t->size(0) == Z && (Z < 2 || t->stride(0) == 1), what,
                    " must be int32 [", Z, "] without gaps (got ", t->scalar_type(), " ", t->sizes(), ")");
  return t->const_data_ptr<int32_t>();
}
struct PageTable {
  const int32_t* at;
  int64_t stride, slots;
};
PageTable page_table(const Tensor& t, int64_t Z, const CacheOp& c) {
  TORCH_CHECK_NOT_IMPLEMENTED(t.dim() != 2 || t.size(1) * c.page <= INT32_MAX, "sequences of up to 2^31 tokens (got a table of ", t.sizes(), " pages)");
  TORCH_CHECK(t.device() == c.data.device(), "the page table is on ", t.device(), ", the cache on ", c.data.device());
  TORCH_CHECK_VALUE(t.scalar_type() == at::kInt && t.dim() == 2 && t.size(0) == Z && (t.size(1) < 2 || t.stride(1) == 1),
                    "pages must be int32 [", Z, ", slots] with unit stride on the slots (got ", t.scalar_type(), " ", t.sizes(), ")");
  return {t.const_data_ptr<int32_t>(), t.stride(0), t.size(1)};
}
// Nothing in a cache is differentiable: an operand that wants a gradient would lose it silently.
void no_gradient(const Tensor& t, const char* what) {
  TORCH_CHECK_NOT_IMPLEMENTED(!recorded(t), what, " needs a gradient, which the cache does not give; call under torch.no_grad()");
}
Tensor unit_rows(const Tensor& x) { return x.stride(3) == 1 ? x : x.clone(at::MemoryFormat::Contiguous); }

void cache_write(const c10::intrusive_ptr<CacheOp>& c, const Tensor& k0, const Tensor& v0, const Tensor& pages, const Tensor& start,
                 const OptTensor& count) {
  TORCH_CHECK_VALUE(k0.dim() == 4 && k0.size(1) == c->heads() && k0.size(3) == c->head_dim && v0.sizes() == k0.sizes(),
                    "key and value must be [Z, ", c->heads(), ", T, ", c->head_dim, "] (got ", k0.sizes(), ", ", v0.sizes(), ")");
  require_cuda(k0);
  TORCH_CHECK(k0.device() == c->data.device(), "the key is on ", k0.device(), ", the cache on ", c->data.device());
  require_same(v0, k0, "the value");
  // (rows of a tensor may share memory, so that there can be more than an int counts)
  TORCH_CHECK_NOT_IMPLEMENTED(k0.size(0) <= INT32_MAX && k0.size(2) <= INT32_MAX, "cannot write ", k0.sizes(), " tokens at once");
  const int code = dtype_code(k0);
  no_gradient(k0, "the key");
  no_gradient(v0, "the value");
  const c10::cuda::CUDAGuard guard(k0.device());
  const Tensor k = unit_rows(k0), v = unit_rows(v0);
  const int64_t Z = k.size(0);
  const PageTable t = page_table(pages, Z, *c);
  check(bsp_cache_write(k.const_data_ptr(), v.const_data_ptr(), code, Z, c->heads(), k.size(2), c->head_dim, k.stride(0), k.stride(1),
                        k.stride(2), v.stride(0), v.stride(1), v.stride(2), c->data.mutable_data_ptr(), c->pages(), c->page, t.at,
                        t.stride, t.slots, per_sequence(start, Z, *c, "start"), per_sequence(count, Z, *c, "count"), stream_of(k)));
}

std::pair<Tensor, Tensor> cache_read(const c10::intrusive_ptr<CacheOp>& c, const Tensor& pages, const Tensor& start, int64_t length,
                                     const OptTensor& count, at::ScalarType type) {
  TORCH_CHECK_VALUE(start.dim() == 1 && length >= 0 && length <= INT32_MAX, "cannot read ", length, " tokens from ", start.sizes());
  const c10::cuda::CUDAGuard guard(c->data.device());
  const int64_t Z = start.size(0);
  const PageTable t = page_table(pages, Z, *c);
  const auto options = c->data.options().dtype(type);
  const Tensor k = at::empty({Z, c->heads(), length, c->head_dim}, options), v = at::empty(k.sizes(), options);
  check(bsp_cache_read(k.mutable_data_ptr(), v.mutable_data_ptr(), dtype_code(k), Z, c->heads(), length, c->head_dim, k.stride(0), k.stride(1),
                       k.stride(2), v.stride(0), v.stride(1), v.stride(2), c->data.const_data_ptr(), c->pages(), c->page, t.at, t.stride,
                       t.slots, per_sequence(start, Z, *c, "start"), per_sequence(count, Z, *c, "count"), stream_of(k)));
  return {k, v};
}

// ---- attention over the cache --------------------------------------------------------------------
struct CacheAttentionOp : torch::CustomClassHolder {
  Tensor hdr, meta;                        // header (host) and tables (device) of the layout
  int64_t block, rows;                     // rows: those of the layout that count
};

Tensor cache_attention(const c10::intrusive_ptr<CacheAttentionOp>& p, const Tensor& q0, const c10::intrusive_ptr<CacheOp>& c,
                       const Tensor& pages, const Tensor& lengths, std::optional<double> scale) {
  TORCH_CHECK_VALUE(q0.dim() == 4 && q0.size(3) == c->head_dim && q0.size(1) % c->heads() == 0, "query must be [Z, n * ", c->heads(),
                    ", T, ", c->head_dim, "] for this cache (got ", q0.sizes(), ")");
  require_cuda(q0);
  TORCH_CHECK(q0.device() == c->data.device(), "the query is on ", q0.device(), ", the cache on ", c->data.device());
  const int code = dtype_code(q0);
  no_gradient(q0, "the query");
  const c10::cuda::CUDAGuard guard(q0.device());
  const Tensor q = even_rows(q0, true), o = at::empty(q.sizes(), q.options());
  const int64_t Z = q.size(0);
  const PageTable t = page_table(pages, Z, *c);
  check(bsp_cache_attn_rows(q.const_data_ptr(), o.mutable_data_ptr(), code, Z, q.size(1), c->heads(), q.size(2), c->head_dim, q.stride(0),
                       q.stride(1), q.stride(2), o.stride(0), o.stride(1), o.stride(2), c->data.const_data_ptr(), c->pages(), c->page,
                       t.at, t.stride, t.slots, per_sequence(lengths, Z, *c, "lengths"), p->block, p->hdr.const_data_ptr<int32_t>(),
                       p->meta.const_data_ptr<int32_t>(), static_cast<int>(p->rows), static_cast<float>(scale ? *scale : 1.0 / std::sqrt(static_cast<double>(c->head_dim))), stream_of(q)));
  return o;
}

}  // namespace

void bind_serving(pybind11::module_& m) {
  namespace py = pybind11;
  py::class_<RotaryOp, c10::intrusive_ptr<RotaryOp>>(m, "RotaryOp")
      .def(py::init([](Tensor table, int64_t head_dim, int64_t axes, bool interleaved) {
        auto p = c10::make_intrusive<RotaryOp>();
        p->table = table; p->head_dim = head_dim; p->axes = axes; p->interleaved = interleaved;
        return p;
      }))
      .def("__call__", &rotary_call, py::call_guard<py::gil_scoped_release>())
      .def("check", &check_rotary_call, py::call_guard<py::gil_scoped_release>())
      .def("one", [](const c10::intrusive_ptr<RotaryOp>& p, const Tensor& x, const OptTensor& pos) { return rotary_call(p, x, {}, pos).first; },
           py::call_guard<py::gil_scoped_release>());
  py::class_<CacheOp, c10::intrusive_ptr<CacheOp>>(m, "CacheOp")
      .def(py::init([](Tensor data, int64_t page, int64_t head_dim) {
        auto c = c10::make_intrusive<CacheOp>();
        c->data = data; c->page = page; c->head_dim = head_dim;
        return c;
      }))
      .def_property_readonly("heads", &CacheOp::heads)
      .def("write", &cache_write, py::call_guard<py::gil_scoped_release>())
      .def("read", &cache_read, py::call_guard<py::gil_scoped_release>());
  py::class_<CacheAttentionOp, c10::intrusive_ptr<CacheAttentionOp>>(m, "CacheAttentionOp")
      .def(py::init([](Tensor hdr, Tensor meta, int64_t block, int64_t rows) {
        auto p = c10::make_intrusive<CacheAttentionOp>();
        p->hdr = hdr; p->meta = meta; p->block = block; p->rows = rows;
        return p;
      }))
      .def("__call__", &cache_attention, py::call_guard<py::gil_scoped_release>());
}
