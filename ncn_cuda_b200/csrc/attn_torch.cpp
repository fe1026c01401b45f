// PyTorch autograd nodes of the attention operators (part of the extension module _ncn_torch): norms of queries and keys with
// the position rotation, windowed attention, and its form over a cache.  As with the NCN nodes, one node per call over the C ABI,
// because at small sizes the host is the bound; a call that a node cannot take goes to the Python Function (attention.py).
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/extension.h>

#include <optional>
#include <string>

#include "../../include/ncn_b200.h"
#include "ncn_torch.h"

namespace py = pybind11;
using at::Tensor;
using ncn_ext::check_status;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

namespace {

int dtype_code(const Tensor& t) { return t.scalar_type() == at::kBFloat16 ? NCN_BF16 : NCN_F32; }
void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

void check_tensors(const char* names, const Tensor& first, std::initializer_list<const Tensor*> rest) {
  if (!first.is_cuda()) throw std::runtime_error("NCN kernels run on CUDA tensors only; there is no CPU path in this package");
  if (first.scalar_type() != at::kFloat && first.scalar_type() != at::kBFloat16)
    throw py::type_error(std::string("NCN kernels take float32 or bfloat16 tensors, got ") + c10::toString(first.scalar_type()));
  if (first.dim() != 3) throw py::value_error("expected [B, N, E] tensors");
  for (const Tensor* t : rest) {
    if (t->dim() != 3) throw py::value_error("expected [B, N, E] tensors");
    if (t->size(0) != first.size(0) || t->scalar_type() != first.scalar_type() || t->device() != first.device())
      throw py::value_error(std::string(names) + " must agree in batch size, dtype and device");
  }
}

// Features per head; the head counts have to divide.
int64_t head_size(const Tensor& q, const Tensor& k, int64_t n_head) {
  const int64_t E = q.size(2);
  if (n_head < 1 || E < 1 || E % n_head != 0)
    throw py::value_error("n_head = " + std::to_string(n_head) + " does not divide the " + std::to_string(E) + " features of the queries");
  const int64_t d = E / n_head;
  if (k.defined() && (k.size(2) < 1 || k.size(2) % d != 0))
    throw py::value_error("the keys' " + std::to_string(k.size(2)) + " features are no whole number of heads of " + std::to_string(d));
  return d;
}

// The tensor as the kernels can read it: features of a position next to each other.
Tensor rows_of(const Tensor& t) { return t.numel() > 0 && t.stride(2) == 1 ? t : t.contiguous(); }
// The tensor as the kernels read it fast: rows on 16-byte boundaries too.  Views of a wider tensor (a joint projection, a cache) stay as they
// are; what does not fit is copied, unless a row's width is no multiple of 16 bytes, which a copy would not change.
Tensor readable(const Tensor& t) {
  const int64_t per = 16 / t.element_size();
  if (t.size(2) % per != 0) return rows_of(t);
  const bool fine = t.stride(2) == 1 && reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0 &&
                    (t.size(1) == 1 || (t.stride(1) >= t.size(2) && t.stride(1) % per == 0)) &&
                    (t.size(0) == 1 || (t.stride(0) >= t.size(2) && t.stride(0) % per == 0));
  if (t.numel() == 0) return t.contiguous();
  if (fine) return t;
  if (!t.is_contiguous()) return t.contiguous();
  return reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0 ? t : t.clone();
}
// its strides of rows and positions; those of a dimension of one are free, and made plain here
void strides_of(const Tensor& t, int64_t* s) {
  s[1] = t.size(1) == 1 ? t.size(2) : t.stride(1);
  s[0] = t.size(0) == 1 ? t.size(1) * s[1] : t.stride(0);
}

Tensor per_row(const std::optional<Tensor>& t, const char* name, int64_t B, const at::Device& dev) {
  if (!t) return Tensor();
  if (t->numel() != B)
    throw py::value_error(std::string(name) + " has " + std::to_string(t->numel()) + " entries for " + std::to_string(B) + " batch rows");
  if (t->is_floating_point() || t->is_complex() || t->scalar_type() == at::kBool) throw py::type_error(std::string(name) + " holds whole numbers");
  if (t->scalar_type() == at::kLong) return t->clamp(INT32_MIN, INT32_MAX).to(dev, at::kInt).contiguous();  // ("no limit" stays one)
  return t->to(dev, at::kInt).contiguous();
}
const int* int_ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr<int>() : nullptr; }

bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
bool needs_function(std::initializer_list<const Tensor*> ts) {
  if (ncn_ext::under_transform()) return true;
  for (const Tensor* t : ts)
    if (t->defined() && !ncn_ext::plain(*t)) return true;
  return false;
}

// There is no second derivative: what a pass with create_graph gets leads back to the inputs through an error, not to a silent zero.
variable_list once(variable_list&& grads, Node& node, bool graph) {
  if (!graph) return std::move(grads);
  std::shared_ptr<Node> error(new torch::autograd::Error(node.name() + " has no derivative of its own", torch::autograd::edge_list(node.next_edges())),
                              torch::autograd::deleteNode);
  for (Tensor& t : grads)
    if (t.defined()) torch::autograd::set_history(t, error);
  return std::move(grads);
}

// ---------------------------------------------------------------- windowed attention
struct WindowCfg {
  int64_t n_head, window, n_sink, start;
  double scale;
};

struct WindowNode : public Node {
  WindowCfg c{};
  SavedVariable q, k, v, y, state, ctxlen, q_start;
  bool has_ctx = false, has_start = false;

  std::string name() const override { return "NCNWindowAttentionBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* s : {&q, &k, &v, &y, &state, &ctxlen, &q_start}) s->reset_data();
  }
  variable_list apply(variable_list&& g) override {
    std::lock_guard<std::mutex> lock(mutex_);
    const bool graph = at::GradMode::is_enabled();
    at::NoGradGuard no_grad;
    if (!g[0].defined()) return variable_list(3);
    const Tensor Q = q.unpack(), K = k.unpack(), V = v.unpack(), Y = y.unpack(shared_from_this()), L = state.unpack();
    const Tensor ctx = has_ctx ? ctxlen.unpack() : Tensor(), st = has_start ? q_start.unpack() : Tensor();
    const c10::cuda::OptionalCUDAGuard guard(Q.device());
    const Tensor dy = readable(g[0]), y_c = Y.contiguous();
    const Tensor qr = readable(Q), kr = readable(K), vr = readable(V);
    const int64_t B = Q.size(0), Nq = Q.size(1), Nk = K.size(1), E = Q.size(2), Ek = K.size(2);
    const bool none = B == 0 || Nq == 0;
    Tensor dq = at::empty(Q.sizes(), qr.options()), dk = none ? at::zeros(K.sizes(), kr.options()) : at::empty(K.sizes(), kr.options()),
           dv = none ? at::zeros(V.sizes(), vr.options()) : at::empty(V.sizes(), vr.options());
    const int dt = dtype_code(Q);
    const size_t bytes = ncn_window_bwd_workspace_bytes(B, Nq, Nk, E, Ek, (int)c.n_head, c.window, c.n_sink, dt);
    const Tensor ws = at::empty({(int64_t)bytes}, qr.options().dtype(at::kByte));
    int64_t s[8];
    strides_of(qr, s), strides_of(kr, s + 2), strides_of(vr, s + 4), strides_of(dy, s + 6);
    check_status("ncn_window_bwd",
                 ncn_window_bwd(qr.const_data_ptr(), kr.const_data_ptr(), vr.const_data_ptr(), y_c.const_data_ptr(), dy.const_data_ptr(),
                                L.const_data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), int_ptr(ctx), int_ptr(st), s,
                                ws.data_ptr(), bytes, B, Nq, Nk, E, Ek, (int)c.n_head, c.window, c.n_sink, c.start, c.scale, dt,
                                stream_of(Q)));
    return once({dq, dk, dv}, *this, graph);
  }
};

std::optional<Tensor> py_window(const Tensor& q, const Tensor& k, const Tensor& v, int64_t n_head, int64_t window, int64_t n_sink,
                                double scale, const std::optional<Tensor>& ctxlen, const std::optional<Tensor>& q_start, int64_t start) {
  if (needs_function({&q, &k, &v})) return std::nullopt;
  check_tensors("q, k and v", q, {&k, &v});
  if (k.sizes() != v.sizes()) throw py::value_error("k and v must agree in shape");
  head_size(q, k, n_head);
  py::gil_scoped_release nogil;
  const bool grad = wants_grad({&q, &k, &v});
  const c10::cuda::OptionalCUDAGuard guard(q.device());
  std::shared_ptr<WindowNode> node;
  if (grad) {
    node = std::shared_ptr<WindowNode>(new WindowNode(), torch::autograd::deleteNode);
    node->set_next_edges({torch::autograd::impl::gradient_edge(q), torch::autograd::impl::gradient_edge(k), torch::autograd::impl::gradient_edge(v)});
    node->c = WindowCfg{n_head, window, n_sink, start, scale};
  }
  Tensor y;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    const int64_t B = q.size(0), Nq = q.size(1), Nk = k.size(1), E = q.size(2), Ek = k.size(2);
    const Tensor ctx = per_row(ctxlen, "ctxlen", B, q.device()), st = per_row(q_start, "q_start", B, q.device());
    const Tensor qr = readable(q), kr = readable(k), vr = readable(v);
    y = at::empty(q.sizes(), qr.options());
    Tensor state;
    if (grad) state = at::empty({(int64_t)ncn_window_state_bytes(B, Nq, E, (int)n_head, dtype_code(q))}, qr.options().dtype(at::kByte));
    int64_t s[6];
    strides_of(qr, s), strides_of(kr, s + 2), strides_of(vr, s + 4);
    check_status("ncn_window_fwd",
                 ncn_window_fwd(qr.const_data_ptr(), kr.const_data_ptr(), vr.const_data_ptr(), y.data_ptr(),
                                grad ? state.data_ptr() : nullptr, int_ptr(ctx), int_ptr(st), s, B, Nq, Nk, E, Ek, (int)n_head,
                                window, n_sink, start, scale, dtype_code(q), stream_of(q)));
    if (grad) {
      node->q = SavedVariable(q, false), node->k = SavedVariable(k, false), node->v = SavedVariable(v, false);
      node->state = SavedVariable(state, false);
      if (ctx.defined()) node->ctxlen = SavedVariable(ctx, false), node->has_ctx = true;
      if (st.defined()) node->q_start = SavedVariable(st, false), node->has_start = true;
    }
  }
  if (grad) {
    torch::autograd::set_history(y, node);
    node->y = SavedVariable(y, true);
  }
  return y;
}

std::optional<Tensor> py_decode(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& ctxlen, int64_t n_head, int64_t window,
                                int64_t n_sink, double scale) {
  if (needs_function({&q, &k, &v}) || wants_grad({&q, &k, &v})) return std::nullopt;  // (the Function's backward is an error)
  check_tensors("q and the caches of keys and values", q, {&k, &v});
  if (k.sizes() != v.sizes()) throw py::value_error("k and v must agree in shape");
  head_size(q, k, n_head);
  py::gil_scoped_release nogil;
  const c10::cuda::OptionalCUDAGuard guard(q.device());
  at::NoGradGuard no_grad;
  const int64_t B = q.size(0), Nq = q.size(1), S = k.size(1), E = q.size(2), Ek = k.size(2);
  const Tensor ctx = per_row(ctxlen, "ctxlen", B, q.device());
  // The caches as they lie: a step needs no memory but its result, and reads what is seen.  (8 rows of 8192 places, 32 on 8 heads of 128, bf16,
  // rows off the 16-byte boundary: windows of 1024 65 us, 335 with copies; all places seen 649, 369 with copies.)
  const Tensor qr = readable(q), kr = rows_of(k), vr = rows_of(v);
  Tensor y = at::empty(q.sizes(), qr.options());
  int64_t s[6];
  strides_of(qr, s), strides_of(kr, s + 2), strides_of(vr, s + 4);
  check_status("ncn_window_decode",
               ncn_window_decode(qr.const_data_ptr(), kr.const_data_ptr(), vr.const_data_ptr(), y.data_ptr(), int_ptr(ctx), s, B, Nq, S, E,
                                 Ek, (int)n_head, window, n_sink, scale, dtype_code(q), stream_of(q)));
  return y;
}

// ---------------------------------------------------------------- norms of queries and keys, rotation
struct RotaryCfg {
  int64_t n_head, start;
  bool interleaved;
  double eps, magnitude;
};
struct Positions {
  Tensor t;  // int64, or undefined: start, start + 1, ...
  int64_t stride = 0;
  const int64_t* ptr() const { return t.defined() ? t.const_data_ptr<int64_t>() : nullptr; }
};
Positions positions_of(const std::optional<Tensor>& t, const Tensor& q) {
  Positions p;
  if (!t) return p;
  const int64_t B = q.size(0), N = q.size(1);
  if (t->is_floating_point() || t->is_complex() || t->scalar_type() == at::kBool) throw py::type_error("positions are whole numbers");
  const bool shared = t->dim() == 1 || (t->dim() == 2 && t->size(0) == 1);
  if (t->dim() < 1 || t->dim() > 2 || t->size(-1) != N || (!shared && t->size(0) != B))
    throw py::value_error("positions must be [N] or [B, N] for tensors [B, N, E]");
  p.t = t->to(q.device(), at::kLong).contiguous();
  p.stride = shared ? 0 : N;
  return p;
}
Tensor freqs_of(const Tensor& f, const at::Device& dev, int64_t d) {
  if (f.dim() != 1 || 2 * f.numel() > d)
    throw py::value_error("freqs must hold one frequency for each rotated pair, at most " + std::to_string(d / 2) + " for heads of " + std::to_string(d));
  return f.detach().to(dev, at::kDouble).contiguous();
}
Tensor norm_weight(const Tensor& w, int64_t d, const at::Device& dev) {
  if (w.numel() != d) throw py::value_error("weight has " + std::to_string(w.numel()) + " elements, expected " + std::to_string(d));
  if (w.scalar_type() == at::kFloat && w.is_contiguous() && w.device() == dev) return w;
  return w.detach().to(dev, at::kFloat).contiguous();
}
const void* ptr_or_null(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
const float* float_or_null(const Tensor& t) { return t.defined() ? t.const_data_ptr<float>() : nullptr; }

// forward, and the backward of a rotation without a norm (inverse)
void rotate(const Tensor& q, const Tensor& k, const Tensor& wq, const Tensor& wk, const Tensor& freqs, const Positions& pos, const RotaryCfg& c,
            bool inverse, Tensor& yq, Tensor& yk) {
  const Tensor qr = readable(q), kr = k.defined() ? readable(k) : Tensor();
  yq = at::empty(q.sizes(), qr.options());
  if (k.defined()) yk = at::empty(k.sizes(), kr.options());
  int64_t s[4] = {0, 0, 0, 0};
  strides_of(qr, s);
  if (k.defined()) strides_of(kr, s + 2);
  check_status("ncn_qk_rotary",
               ncn_qk_rotary(qr.const_data_ptr(), ptr_or_null(kr), float_or_null(wq), float_or_null(wk), freqs.const_data_ptr<double>(),
                             pos.ptr(), pos.stride, c.start, yq.data_ptr(), k.defined() ? yk.data_ptr() : nullptr, s, q.size(0), q.size(1),
                             q.size(2), k.defined() ? k.size(2) : 0, (int)c.n_head, 2 * freqs.numel(), c.interleaved, c.eps, c.magnitude,
                             inverse, dtype_code(q), stream_of(q)));
}

struct RotaryNode : public Node {
  RotaryCfg c{};
  bool norm = false, has_k = false, has_pos = false;
  int64_t pos_stride = 0;
  SavedVariable q, k, wq, wk, freqs, pos;
  at::TensorOptions opt_q, opt_k, opt_wq, opt_wk;
  std::vector<int64_t> size_q, size_k, size_wq, size_wk;

  std::string name() const override { return norm ? "NCNQKNormRotaryBackward" : "NCNRotaryBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* s : {&q, &k, &wq, &wk, &freqs, &pos}) s->reset_data();
  }
  variable_list apply(variable_list&& g) override {
    std::lock_guard<std::mutex> lock(mutex_);
    const bool graph = at::GradMode::is_enabled();
    at::NoGradGuard no_grad;
    if (!g[0].defined() && !(g.size() > 1 && g[1].defined())) return variable_list(4);
    const Tensor& any = g[0].defined() ? g[0] : g[1];
    const c10::cuda::OptionalCUDAGuard guard(any.device());
    const Tensor gq = g[0].defined() ? g[0] : at::zeros(size_q, opt_q);
    const Tensor gk = !has_k ? Tensor() : g[1].defined() ? g[1] : at::zeros(size_k, opt_k);
    Positions p;
    if (has_pos) p.t = pos.unpack(), p.stride = pos_stride;
    const Tensor f = freqs.unpack();
    variable_list out(4);
    if (!norm) {
      rotate(gq, gk, Tensor(), Tensor(), f, p, c, true, out[0], out[1]);
      return once(std::move(out), *this, graph);
    }
    const Tensor Q = q.unpack(), K = has_k ? k.unpack() : Tensor();
    const int64_t B = Q.size(0), N = Q.size(1), E = Q.size(2), Ek = has_k ? K.size(2) : 0, d = E / c.n_head;
    const Tensor wqf = norm_weight(wq.unpack(), d, Q.device()), wkf = has_k ? norm_weight(wk.unpack(), d, Q.device()) : Tensor();
    const at::TensorOptions f32 = opt_q.dtype(at::kFloat);
    Tensor dwq = at::empty(size_wq, f32), dwk = has_k ? at::empty(size_wk, f32) : Tensor();
    out[0] = at::empty(size_q, opt_q);
    if (has_k) out[1] = at::empty(size_k, opt_k);
    if (B == 0 || N == 0) {
      dwq.zero_();
      if (has_k) dwk.zero_();
    } else {
      const Tensor qr = readable(Q), kr = has_k ? readable(K) : Tensor(), gqr = readable(gq), gkr = has_k ? readable(gk) : Tensor();
      int64_t s[8] = {};
      strides_of(qr, s), strides_of(gqr, s + 4);
      if (has_k) strides_of(kr, s + 2), strides_of(gkr, s + 6);
      const size_t bytes = ncn_qk_norm_rotary_workspace_bytes(B, N, E, (int)c.n_head);
      const Tensor ws = at::empty({(int64_t)bytes}, f32.dtype(at::kByte));
      check_status("ncn_qk_norm_rotary_bwd",
                   ncn_qk_norm_rotary_bwd(qr.const_data_ptr(), ptr_or_null(kr), wqf.const_data_ptr<float>(), float_or_null(wkf),
                                          f.const_data_ptr<double>(), p.ptr(), p.stride, c.start, gqr.const_data_ptr(), ptr_or_null(gkr),
                                          out[0].data_ptr(), has_k ? out[1].data_ptr() : nullptr, dwq.mutable_data_ptr<float>(),
                                          has_k ? dwk.mutable_data_ptr<float>() : nullptr, s, ws.data_ptr(), bytes, B, N, E, Ek,
                                          (int)c.n_head, 2 * f.numel(), c.interleaved, c.eps, c.magnitude, dtype_code(Q), stream_of(Q)));
    }
    out[2] = dwq.to(opt_wq.device(), c10::typeMetaToScalarType(opt_wq.dtype()));
    if (has_k) out[3] = dwk.to(opt_wk.device(), c10::typeMetaToScalarType(opt_wk.dtype()));
    return once(std::move(out), *this, graph);
  }
};

using Pair = std::tuple<Tensor, std::optional<Tensor>>;
std::optional<Pair> py_rotary(const Tensor& q, const std::optional<Tensor>& k_in, const std::optional<Tensor>& wq_in, const std::optional<Tensor>& wk_in,
                              const Tensor& freqs_in, const std::optional<Tensor>& pos_in, int64_t n_head, int64_t start, bool interleaved,
                              double eps, double magnitude) {
  const Tensor k = k_in.value_or(Tensor()), wq = wq_in.value_or(Tensor()), wk = wk_in.value_or(Tensor());
  if (needs_function({&q, &k, &wq, &wk, &freqs_in})) return std::nullopt;
  check_tensors("q and k", q, {});
  if (k.defined()) {
    check_tensors("q and k", q, {&k});
    if (k.size(1) != q.size(1)) throw py::value_error("q and k must agree in the number of positions");
  }
  const int64_t d = head_size(q, k, n_head);
  if (k.defined() && wq.defined() != wk.defined()) throw py::value_error("both weights or none");
  py::gil_scoped_release nogil;
  const bool grad = wants_grad({&q, &k, &wq, &wk});
  const c10::cuda::OptionalCUDAGuard guard(q.device());
  const RotaryCfg c{n_head, start, interleaved, eps, magnitude};
  std::shared_ptr<RotaryNode> node;
  if (grad) {
    node = std::shared_ptr<RotaryNode>(new RotaryNode(), torch::autograd::deleteNode);
    torch::autograd::edge_list edges;
    for (const Tensor* t : {&q, &k, &wq, &wk}) edges.push_back(t->defined() ? torch::autograd::impl::gradient_edge(*t) : torch::autograd::Edge());
    node->set_next_edges(std::move(edges));
    node->c = c;
    node->norm = wq.defined();
    node->has_k = k.defined();
    node->opt_q = q.options(), node->size_q = q.sizes().vec();
    if (k.defined()) node->opt_k = k.options(), node->size_k = k.sizes().vec();
    if (wq.defined()) node->opt_wq = wq.options(), node->size_wq = wq.sizes().vec();
    if (wk.defined()) node->opt_wk = wk.options(), node->size_wk = wk.sizes().vec();
  }
  Tensor yq, yk;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    const Positions pos = positions_of(pos_in, q);
    const Tensor freqs = freqs_of(freqs_in, q.device(), d);
    const Tensor wqf = wq.defined() ? norm_weight(wq, d, q.device()) : Tensor(), wkf = wk.defined() ? norm_weight(wk, d, q.device()) : Tensor();
    rotate(q, k, wqf, k.defined() ? wkf : Tensor(), freqs, pos, c, false, yq, yk);
    if (grad) {
      node->freqs = SavedVariable(freqs, false);
      if (pos.t.defined()) node->pos = SavedVariable(pos.t, false), node->has_pos = true, node->pos_stride = pos.stride;
      if (wq.defined()) {
        node->q = SavedVariable(q, false), node->wq = SavedVariable(wq, false);
        if (k.defined()) node->k = SavedVariable(k, false), node->wk = SavedVariable(wk, false);
      }
    }
  }
  if (grad) {
    torch::autograd::set_history(yq, node);
    if (yk.defined()) torch::autograd::set_history(yk, node);
  }
  return Pair{yq, yk.defined() ? std::optional<Tensor>(yk) : std::nullopt};
}

}  // namespace

void ncn_ext::bind_attention(py::module_& m) {
  m.def("window", &py_window);
  m.def("window_decode", &py_decode);
  m.def("rotary", &py_rotary);
}
