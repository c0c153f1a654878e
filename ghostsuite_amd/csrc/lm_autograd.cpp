// Host side of the language-model operators: argument checks, allocation and automatic
// differentiation around gs_embedding_lookup*, gs_qk_rotary* and gs_distill_*
// (include/ghost_hip.h), as a Python extension module.
//
// C++ because a training step calls these in every layer: a Python autograd function costs the host
// 50 to 100 us a forward and backward pass (its backward pass runs on the autograd engine's thread,
// where the interpreter's state has to move to another core), this one 34 to 53, of which an empty
// node's share is 22 to 37 (MI355X host, embedding of 16 tokens, fast and slow thread placement).
//
// Everything runs on the current stream of the tensors' device; nothing synchronises.  Backward passes
// read what autograd saved, so they see a tensor that was changed in place since as an error, and are
// not differentiable themselves.
#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/custom_class.h>

#include <optional>
#include <sstream>
#include <string>
#include <vector>

#include "ghost_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

// Becomes the package's GhostHipError.
struct GhostError : std::runtime_error {
  using std::runtime_error::runtime_error;
};

template <class... A>
[[noreturn]] void refuse(const A&... a) {
  std::ostringstream s;
  (s << ... << a);
  throw GhostError(s.str());
}
template <class... A>
void require(bool ok, const A&... a) {
  if (!ok) refuse(a...);
}
void check(int rc, const char* what) {
  if (rc != GS_OK) refuse(what, " failed (", rc, "): ", gs_last_error());
}

int gs_dtype_of(const Tensor& t, const char* what) {
  if (t.scalar_type() == at::kBFloat16) return GS_DTYPE_BF16;
  if (t.scalar_type() == at::kFloat) return GS_DTYPE_F32;
  refuse(what, ": bf16 or fp32, got ", t.scalar_type());
}

// A tensor that is its memory: no wrapper of a function transform or subclass, no compressed layout, no
// sign or zeros that are only marked.
bool in_memory(const Tensor& t) {
  return t.layout() == at::kStrided && t.has_storage() && !t.is_nested() && !t.is_neg() &&
         !t._is_zerotensor() && !t.unsafeGetTensorImpl()->is_python_dispatch() &&
         !t.key_set().has(c10::DispatchKey::Functionalize);
}

// The operators are no operators of torch's dispatcher: what it does around those (forward-mode
// differentiation, function transforms, tracing) would pass them by unseen, so it is refused.
void check_plain(std::initializer_list<const Tensor*> ts) {
  require(!torch::jit::tracer::isTracing(), "the language-model operators cannot be traced");
  for (const Tensor* t : ts) {
    if (!t->defined()) continue;
    require(in_memory(*t), "the language-model operators take plain strided tensors (no sparse or nested "
            "ones, no subclasses, no lazily negated views, no function transforms)");
    require(!t->_fw_grad(0).defined(),
            "the language-model operators have no forward-mode differentiation");
  }
}

// An output gradient in memory: marked zeros and signs are written.
Tensor gradient_in_memory(const Tensor& g) {
  if (in_memory(g)) return g;
  if (g._is_zerotensor())
    return at::zeros(g.sizes(), at::TensorOptions().dtype(g.dtype()).device(g.device()));
  const Tensor r = g.is_neg() ? g.resolve_neg() : g;
  require(in_memory(r), "an output gradient that is no plain strided tensor");
  return r;
}

// All tensors (undefined ones aside) on one GPU.
c10::Device device_of(std::initializer_list<const Tensor*> ts) {
  std::optional<c10::Device> dev;
  for (const Tensor* t : ts) {
    if (!t->defined()) continue;
    require(t->is_cuda(), "ghostsuite_amd kernels need tensors on a ROCm GPU device; got a tensor on ",
            t->device(), " (there is no CPU path)");
    if (!dev) dev = t->device();
    require(t->device() == *dev, "tensors on different devices: ", *dev, " and ", t->device());
  }
  return *dev;
}

void* stream_on(c10::Device dev) { return c10::hip::getCurrentHIPStream(dev.index()).stream(); }

Tensor given(const OptTensor& t) { return t ? *t : Tensor(); }
OptTensor some(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }
const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* mut(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }

// The last dimension contiguous.
Tensor features_contiguous(const Tensor& t) {
  return t.size(-1) == 1 || t.stride(-1) == 1 ? t : t.contiguous();
}

Tensor scratch(size_t bytes, const Tensor& like) {
  return at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte).requires_grad(false));
}

bool recorded(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// Gradients of a backward pass that is itself recorded: differentiating them raises.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list defined;
  for (Tensor& g : grads)
    if (g.defined()) defined.push_back(g.detach().requires_grad_());
  auto node = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function whose backward pass is not differentiable",
      static_cast<int64_t>(defined.size()));
  defined = (*node)(std::move(defined));
  size_t k = 0;
  for (Tensor& g : grads)
    if (g.defined()) g = defined[k++];
  return grads;
}

// A plain struct kept by an autograd node.
template <class T>
struct Kept : torch::CustomClassHolder {
  T value;
  explicit Kept(T v) : value(std::move(v)) {}
};
template <class T>
void keep(AutogradContext* ctx, T value) {
  ctx->saved_data["kept"] = c10::IValue::make_capsule(c10::make_intrusive<Kept<T>>(std::move(value)));
}
template <class T>
T& kept(AutogradContext* ctx) {
  return static_cast<Kept<T>*>(ctx->saved_data["kept"].toCapsule().get())->value;
}

// ------------------------------------------------------------------------------ embedding lookup

struct LookupHow {
  double scale;
  int64_t padding;   // -1: none
  std::vector<int64_t> table;
  at::ScalarType dtype;
};

// scale * weight[ids]; with grad_ids the ids as the gradient takes them.
Tensor lookup(const Tensor& ids_in, const Tensor& weight_in, const LookupHow& how, Tensor* grad_ids) {
  const c10::Device dev = device_of({&ids_in, &weight_in});
  const int dt = gs_dtype_of(weight_in, "embedding weight");
  const bool wide = ids_in.scalar_type() == at::kLong;
  require(wide || ids_in.scalar_type() == at::kInt, "token ids of dtype ", ids_in.scalar_type(),
          ": int32 or int64 expected");
  require(weight_in.dim() == 2 && weight_in.numel() > 0, "embedding weight ", weight_in.sizes(),
          ": [vocab, d] expected");
  const Tensor ids = ids_in.contiguous(), weight = weight_in.contiguous();
  const int64_t vocab = weight.size(0), d = weight.size(1);
  std::vector<int64_t> shape = ids.sizes().vec();
  shape.push_back(d);
  const Tensor out = at::empty(shape, weight.options().requires_grad(false));
  Tensor written;
  if (grad_ids != nullptr) {
    if (!wide || how.padding >= 0) written = at::empty(ids.sizes(), ids.options().dtype(at::kLong));
    *grad_ids = written.defined() ? written : ids;
  }
  if (ids.numel() > 0) {
    c10::DeviceGuard guard(dev);
    check(gs_embedding_lookup(ptr(ids), wide ? 64 : 32, ids.numel(), ptr(weight), dt, vocab, d,
                              static_cast<float>(how.scale), how.padding, mut(out),
                              static_cast<int64_t*>(mut(written)), stream_on(dev)),
          "gs_embedding_lookup");
  }
  return out;
}

Tensor lookup_grad(const Tensor& ids, const Tensor& g_given, const LookupHow& how) {
  const Tensor g_in = gradient_in_memory(g_given);
  const c10::Device dev = device_of({&ids, &g_in});
  const auto options = g_in.options().dtype(how.dtype).requires_grad(false);
  const int64_t n = ids.numel(), vocab = how.table[0], d = how.table[1];
  if (n == 0) return at::zeros(how.table, options);
  require(g_in.scalar_type() == how.dtype, "output gradient of dtype ", g_in.scalar_type(), ", table of ",
          how.dtype);
  const Tensor g = g_in.contiguous(), out = at::empty(how.table, options);
  const size_t bytes = gs_embedding_lookup_grad_workspace(n, vocab, d);
  Tensor ws;
  if (bytes > 0) ws = scratch(bytes, g);
  c10::DeviceGuard guard(dev);
  check(gs_embedding_lookup_grad(static_cast<const int64_t*>(ptr(ids)), ptr(g),
                                 gs_dtype_of(g, "output gradient"), n, vocab, d,
                                 static_cast<float>(how.scale), mut(out), mut(ws), bytes, stream_on(dev)),
        "gs_embedding_lookup_grad");
  return out;
}

struct Lookup : torch::autograd::Function<Lookup> {
  static Tensor forward(AutogradContext* ctx, const Tensor& ids, const Tensor& weight, LookupHow how) {
    how.table = weight.sizes().vec();
    how.dtype = weight.scalar_type();
    Tensor grad_ids;
    Tensor out = lookup(ids, weight, how, &grad_ids);
    ctx->save_for_backward({grad_ids});
    keep(ctx, std::move(how));
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const variable_list saved = ctx->get_saved_variables();
    return once({Tensor(), lookup_grad(saved[0], g[0], kept<LookupHow>(ctx)), Tensor()});
  }
};

Tensor embedding_lookup(const Tensor& ids, const Tensor& weight, double scale,
                        std::optional<int64_t> padding_idx) {
  check_plain({&ids, &weight});
  LookupHow how{scale, padding_idx.value_or(-1), {}, weight.scalar_type()};
  if (recorded({&weight})) return Lookup::apply(ids, weight, std::move(how));
  return lookup(ids, weight, how, nullptr);
}

// ------------------------------------------------- norms of queries and keys with their rotation

struct QkHow {
  int64_t heads[3];
  bool norm, interleaved;
  double eps;
  Tensor samples;   // where the backward pass writes each sample's weight gradients, or undefined;
                    // its version counts the passes
  int edge[4];      // each input's place among the node's edges, or -1
};

// The arguments of a gs_qk_rotary* call.  `a`: one packed tensor (b undefined), or queries a, keys b.
struct QkCall {
  c10::Device dev;
  gs_qk_shape shape{};
  gs_qk_rows x[3]{};
  int64_t B, T, D;
  Tensor held[4];   // what the pointers are into

  QkCall(const Tensor& a_in, const Tensor& b_in, const Tensor& qw, const Tensor& kw,
         const Tensor& table, const Tensor& positions, const QkHow& how)
      : dev(device_of({&a_in, &b_in, &qw, &kw, &table, &positions})) {
    const Tensor a = held[0] = features_contiguous(a_in);
    const int64_t total = how.heads[0] + how.heads[1] + how.heads[2];
    require(how.heads[0] > 0 && how.heads[1] > 0, how.heads[0], " query and ", how.heads[1],
            " key heads");
    if (b_in.defined()) {
      held[1] = features_contiguous(b_in);
      require(a.size(0) == b_in.size(0) && a.size(1) == b_in.size(1) && a.size(3) == b_in.size(3) &&
                  a.scalar_type() == b_in.scalar_type(),
              "queries ", a.sizes(), " ", a.scalar_type(), " and keys ", b_in.sizes(), " ",
              b_in.scalar_type(), " disagree");
    } else {
      require((a.dim() == 3 && a.size(2) % total == 0) || (a.dim() == 4 && a.size(2) == total), "qkv ",
              a.sizes(), " does not hold ", total, " heads");
    }
    B = a.size(0), T = a.size(1), D = a.dim() == 4 ? a.size(3) : a.size(2) / total;
    require(D > 0, "heads without features");
    shape.dtype = gs_dtype_of(a, "queries and keys");
    require(table.dim() == 3 && table.size(1) == 2 && table.scalar_type() == at::kFloat &&
                table.is_contiguous() && 2 * table.size(2) <= D,
            "table ", table.sizes(), " ", table.scalar_type(),
            ": contiguous fp32 [positions, 2, n_rot / 2] with n_rot up to ", D, " expected");
    shape.B = B, shape.T = T, shape.D = D, shape.n_rot = 2 * table.size(2);
    require(total <= INT32_MAX, total, " heads");
    for (int k = 0; k < 3; ++k) shape.heads[k] = static_cast<int32_t>(how.heads[k]);
    shape.norm = how.norm, shape.interleaved = how.interleaved;
    shape.eps = static_cast<float>(how.eps);
    for (int k = 0; k < 2; ++k) {
      const Tensor& w = k == 0 ? qw : kw;
      shape.weight_dtype[k] = shape.dtype;
      if (!w.defined()) continue;
      require(w.dim() == 1 && w.size(0) == D, "norm weight ", w.sizes(), ": [", D, "] expected");
      shape.weight_dtype[k] = gs_dtype_of(w, "norm weights");
      held[2 + k] = w.contiguous();
      shape.weight[k] = ptr(held[2 + k]);
    }
    if (shape.n_rot > 0) {
      shape.table = static_cast<const float*>(ptr(table));
      shape.n_positions = table.size(0);
      if (positions.defined()) {
        const bool wide = positions.scalar_type() == at::kLong;
        const int64_t n = positions.dim();
        require((wide || positions.scalar_type() == at::kInt) && (n == 1 || n == 2) &&
                    positions.size(-1) == T &&
                    (n == 1 || positions.size(0) == 1 || positions.size(0) == B),
                "positions ", positions.sizes(), " ", positions.scalar_type(), ": int32 or int64 [", T,
                "] or [", B, ", ", T, "] expected");
        shape.positions = ptr(positions);
        shape.position_bits = wide ? 64 : 32;
        shape.position_stride_t = positions.stride(-1);
        shape.position_stride_b = n == 2 && positions.size(0) > 1 ? positions.stride(0) : 0;
      }
    }
    rows(held[0], held[1], x);
  }

  // The rows of the parts of input-shaped tensors.
  void rows(const Tensor& a, const Tensor& b, gs_qk_rows (&out)[3]) const {
    const int64_t esz = a.element_size(), sh = a.dim() == 4 ? a.stride(2) : D;
    char* p = static_cast<char*>(const_cast<void*>(a.const_data_ptr()));
    out[0] = {p, a.stride(0), a.stride(1), sh};
    if (b.defined()) {
      out[1] = {const_cast<void*>(b.const_data_ptr()), b.stride(0), b.stride(1), b.stride(2)};
      return;
    }
    out[1] = {p + shape.heads[0] * sh * esz, a.stride(0), a.stride(1), sh};
    out[2] = {p + (shape.heads[0] + shape.heads[1]) * sh * esz, a.stride(0), a.stride(1), sh};
  }
  bool empty() const { return B == 0 || T == 0; }
};

// The rows of heads-first tensors [B, heads, T, D] (undefined: none).
void heads_first(const variable_list& ts, gs_qk_rows (&out)[3]) {
  for (size_t k = 0; k < ts.size() && k < 3; ++k)
    if (ts[k].defined())
      out[k] = {const_cast<void*>(ts[k].const_data_ptr()), ts[k].stride(0), ts[k].stride(2),
                ts[k].stride(1)};
}

// Output gradients as the kernels take them.
variable_list output_gradients(const QkCall& c, const variable_list& given_grads) {
  variable_list grads;
  for (size_t k = 0; k < given_grads.size() && k < 3; ++k) {
    Tensor g = given_grads[k];
    if (g.defined()) {
      g = gradient_in_memory(g);
      device_of({&c.held[0], &g});
      require(g.dim() == 4 && g.size(0) == c.B && g.size(1) == c.shape.heads[k] && g.size(2) == c.T &&
                  g.size(3) == c.D && g.scalar_type() == c.held[0].scalar_type(),
              "output gradient ", g.sizes(), " ", g.scalar_type());
      g = features_contiguous(g);
    }
    grads.push_back(g);
  }
  return grads;
}

variable_list qk_forward(const Tensor& a, const Tensor& b, const Tensor& qw, const Tensor& kw,
                         const Tensor& table, const Tensor& positions, const QkHow& how) {
  const QkCall c(a, b, qw, kw, table, positions, how);
  variable_list out;
  for (int k = 0; k < 3; ++k)
    if (how.heads[k] > 0)
      out.push_back(at::empty({c.B, how.heads[k], c.T, c.D}, a.options().requires_grad(false)));
  if (!c.empty()) {
    gs_qk_rows y[3]{};
    heads_first(out, y);
    c10::DeviceGuard guard(c.dev);
    check(gs_qk_rotary(&c.shape, c.x, y, stream_on(c.dev)), "gs_qk_rotary");
  }
  return out;
}

struct QkNormRotary : torch::autograd::Function<QkNormRotary> {
  static variable_list forward(AutogradContext* ctx, const Tensor& a, const OptTensor& b,
                               const OptTensor& qw, const OptTensor& kw, const Tensor& table,
                               const OptTensor& positions, QkHow how) {
    ctx->set_materialize_grads(false);
    int edges = 0;
    how.edge[0] = edges++;
    how.edge[1] = b ? edges++ : -1;
    how.edge[2] = qw ? edges++ : -1;
    how.edge[3] = kw ? edges++ : -1;
    ctx->save_for_backward({a, given(b), given(qw), given(kw), table, given(positions)});
    variable_list out = qk_forward(a, given(b), given(qw), given(kw), table, given(positions), how);
    keep(ctx, how);
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list given_grads) {
    const variable_list s = ctx->get_saved_variables();
    const QkHow& how = kept<QkHow>(ctx);
    const auto needs = [&](int k) {
      return how.edge[k] >= 0 && ctx->needs_input_grad(static_cast<size_t>(how.edge[k]));
    };
    const QkCall c(s[0], s[1], s[2], s[3], s[4], s[5], how);
    const variable_list grads = output_gradients(c, given_grads);
    Tensor da, db, dw[2];
    const bool want_x = needs(0) || needs(1);
    if (want_x) {
      da = at::empty(s[0].sizes(), s[0].options().requires_grad(false));
      if (s[1].defined()) db = at::empty(s[1].sizes(), s[1].options().requires_grad(false));
    }
    for (int k = 0; k < 2; ++k)
      if (needs(2 + k)) dw[k] = at::empty({c.D}, s[2 + k].options().requires_grad(false));
    if (c.empty()) {
      for (Tensor& w : dw)
        if (w.defined()) w.zero_();
      if (how.samples.defined()) how.samples.zero_();
    } else if (want_x || dw[0].defined() || dw[1].defined() || how.samples.defined()) {
      gs_qk_rows dy[3]{}, dx[3]{};
      heads_first(grads, dy);
      if (want_x) c.rows(da, db, dx);
      Tensor ws;
      size_t bytes = 0;
      if (dw[0].defined() || dw[1].defined() || how.samples.defined()) {
        bytes = gs_qk_rotary_grad_workspace(&c.shape, how.samples.defined());
        ws = scratch(bytes, s[0]);
      }
      c10::DeviceGuard guard(c.dev);
      check(gs_qk_rotary_grad(&c.shape, c.x, dy, want_x ? dx : nullptr, mut(dw[0]), mut(dw[1]),
                              static_cast<float*>(mut(how.samples)), mut(ws), bytes,
                              stream_on(c.dev)),
            "gs_qk_rotary_grad");
    }
    if (how.samples.defined()) how.samples.unsafeGetTensorImpl()->bump_version();   // written
    return once({da, db, dw[0], dw[1], Tensor(), Tensor(), Tensor()});
  }
};

QkHow qk_how(const std::vector<int64_t>& heads, bool norm, double eps, bool interleaved) {
  return QkHow{{heads.at(0), heads.at(1), heads.at(2)}, norm, interleaved, eps, Tensor(),
               {-1, -1, -1, -1}};
}

// (queries, keys[, values]) of a packed tensor a, or of queries a and keys b; the backward pass fills
// `samples`.
variable_list qk_norm_rotary(const Tensor& a, const OptTensor& b, const std::vector<int64_t>& heads,
                             const Tensor& table, const OptTensor& positions, const OptTensor& qw,
                             const OptTensor& kw, bool norm, double eps, bool interleaved,
                             const OptTensor& samples) {
  const Tensor bt = given(b), q = given(qw), k = given(kw), pos = given(positions);
  QkHow how = qk_how(heads, norm, eps, interleaved);
  how.samples = given(samples);
  check_plain({&a, &bt, &q, &k, &table, &pos, &how.samples});
  if (how.samples.defined())
    require(norm && how.samples.is_cuda() && how.samples.device() == a.device() &&
                how.samples.scalar_type() == at::kFloat && how.samples.is_contiguous() &&
                how.samples.dim() == 3 && how.samples.size(0) == 2 &&
                how.samples.size(1) == a.size(0) &&
                how.samples.size(2) * (heads[0] + heads[1] + heads[2]) * a.size(1) * a.size(0) ==
                    a.numel(),
            "sample gradients ", how.samples.sizes(), ": fp32 [2, B, D] for a packed input expected");
  if (recorded({&a, &bt, &q, &k}))
    return QkNormRotary::apply(a, b, qw, kw, table, positions, how);
  return qk_forward(a, bt, q, k, table, pos, how);
}

// (dot_q, dot_k, train gradient of q's weight, of k's; the gradients undefined without a scale).
std::vector<OptTensor> qk_norm_rotary_dots(const Tensor& a, const OptTensor& b,
                                           const std::vector<int64_t>& heads, const Tensor& table,
                                           const OptTensor& positions, const OptTensor& qw,
                                           const OptTensor& kw, double eps, bool interleaved,
                                           const std::vector<OptTensor>& given_grads, int64_t n_val,
                                           std::optional<int64_t> val_start,
                                           std::optional<double> grad_scale) {
  const Tensor bt = given(b), q = given(qw), k = given(kw), pos = given(positions);
  check_plain({&a, &bt, &q, &k, &table, &pos});
  const QkCall c(a, bt, q, k, table, pos, qk_how(heads, true, eps, interleaved));
  require(!c.empty(), "qk_norm_rotary_dots: no tokens");
  const int64_t n_train = c.B - n_val;
  require(n_train > 0, "qk_norm_rotary_dots: ", n_val, " validation samples of ", c.B);
  variable_list grads;
  for (const OptTensor& g : given_grads) grads.push_back(given(g));
  grads = output_gradients(c, grads);
  gs_qk_rows dy[3]{};
  heads_first(grads, dy);
  const auto fp32 = a.options().dtype(at::kFloat).requires_grad(false);
  const Tensor dots[2] = {at::empty({n_train}, fp32), at::empty({n_train}, fp32)};
  Tensor dw[2];
  if (grad_scale)
    for (int k = 0; k < 2; ++k)
      dw[k] = at::empty({c.D}, (c.held[2 + k].defined() ? c.held[2 + k] : a).options().requires_grad(false));
  const size_t bytes = gs_qk_rotary_dots_workspace(&c.shape);
  const Tensor ws = scratch(bytes, a);
  c10::DeviceGuard guard(c.dev);
  check(gs_qk_rotary_dots(&c.shape, c.x, dy, n_val, val_start.value_or(n_train),
                          static_cast<float*>(mut(dots[0])), static_cast<float*>(mut(dots[1])),
                          mut(dw[0]), mut(dw[1]), static_cast<float>(grad_scale.value_or(0.0)), mut(ws),
                          bytes, stream_on(c.dev)),
        "gs_qk_rotary_dots");
  return {dots[0], dots[1], some(dw[0]), some(dw[1])};
}

std::vector<OptTensor> qk_sample_dots(const Tensor& samples, const Tensor& qw, const Tensor& kw,
                                      int64_t n_val, std::optional<int64_t> val_start,
                                      std::optional<double> grad_scale) {
  check_plain({&samples, &qw, &kw});
  const c10::Device dev = device_of({&samples, &qw, &kw});
  require(samples.dim() == 3 && samples.size(0) == 2 && samples.scalar_type() == at::kFloat &&
              samples.is_contiguous(),
          "sample gradients ", samples.sizes(), ": fp32 [2, B, D] expected");
  const int64_t B = samples.size(1), D = samples.size(2), n_train = B - n_val;
  require(n_train > 0, "qk_sample_dots: ", n_val, " validation samples of ", B);
  const auto fp32 = samples.options().requires_grad(false);
  const Tensor dots[2] = {at::empty({n_train}, fp32), at::empty({n_train}, fp32)};
  const int dt[2] = {gs_dtype_of(qw, "norm weights"), gs_dtype_of(kw, "norm weights")};
  Tensor dw[2];
  if (grad_scale) {
    dw[0] = at::empty({D}, qw.options().requires_grad(false));
    dw[1] = at::empty({D}, kw.options().requires_grad(false));
  }
  const size_t bytes = gs_qk_sample_dots_workspace(B, D);
  Tensor ws;
  if (bytes > 0) ws = scratch(bytes, samples);
  c10::DeviceGuard guard(dev);
  check(gs_qk_sample_dots(static_cast<const float*>(ptr(samples)), B, D, n_val,
                          val_start.value_or(n_train), static_cast<float*>(mut(dots[0])),
                          static_cast<float*>(mut(dots[1])), mut(dw[0]), dt[0], mut(dw[1]), dt[1],
                          static_cast<float>(grad_scale.value_or(0.0)), mut(ws), bytes, stream_on(dev)),
        "gs_qk_sample_dots");
  return {dots[0], dots[1], some(dw[0]), some(dw[1])};
}

// ------------------------------------------------------------------------------ distillation

struct DistillHow {
  double temperature, alpha;
  int64_t ignore_index;
  int reduction;
  Tensor unit, ws;   // the gradient for an upstream of one, and the scratch of the call that wrote it
};

// Elements from a tensor's first to its last.
int64_t span_of(const Tensor& x) {
  int64_t span = 1;
  for (int64_t k = 0; k < x.dim(); ++k) span += (x.size(k) - 1) * x.stride(k);
  return span;
}

// Logits as [N, V] or [B, T, V] with contiguous rows that do not overlap; a copy where the strides do
// not allow that, or where the rows are less than half of what they lie in: their gradient has the same
// strides, and would take its memory.
Tensor rows_of_logits(const Tensor& logits) {
  const int64_t V = logits.size(-1);
  const Tensor z = logits.dim() == 3 ? logits : logits.reshape({-1, V});
  const int64_t T = z.size(-2);
  bool ok = (V == 1 || z.stride(-1) == 1) && (T == 1 || z.stride(-2) >= V);
  if (z.dim() == 3 && z.size(0) > 1) ok = ok && z.stride(0) >= (T - 1) * z.stride(1) + V;
  return ok && span_of(z) <= 2 * z.numel() ? z : z.contiguous();
}

struct DistillCall {
  c10::Device dev;
  gs_distill d{};
  Tensor z, ids, t, labels;   // what the pointers are into

  DistillCall(const Tensor& logits, const Tensor& ids_in, const Tensor& t_in, const Tensor& labels_in,
              const DistillHow& how)
      : dev(device_of({&logits, &ids_in, &t_in, &labels_in})) {
    const bool ok = logits.dim() >= 1 && ids_in.dim() == logits.dim() && ids_in.sizes() == t_in.sizes() &&
                    logits.size(-1) > 0 && ids_in.size(-1) > 0 &&
                    ids_in.sizes().slice(0, ids_in.dim() - 1) ==
                        logits.sizes().slice(0, logits.dim() - 1) &&
                    (!labels_in.defined() ||
                     labels_in.sizes() == logits.sizes().slice(0, logits.dim() - 1));
    if (!ok) {
      std::ostringstream y;
      if (labels_in.defined()) y << labels_in.sizes(); else y << "none";
      refuse("logits ", logits.sizes(), ", teacher ids ", ids_in.sizes(), ", teacher logits ",
             t_in.sizes(), ", labels ", y.str(), ": [..., V], [..., K] twice and [...] expected");
    }
    const auto whole = [](const Tensor& x) {
      return !x.defined() || at::isIntegralType(x.scalar_type(), false);
    };
    require(whole(ids_in) && whole(labels_in), "teacher ids and labels have to be integers");
    require(at::isFloatingType(t_in.scalar_type()), "teacher logits of dtype ", t_in.scalar_type());
    d.dtype = gs_dtype_of(logits, "logits");
    z = rows_of_logits(logits);
    t = t_in.scalar_type() == at::kBFloat16 ? t_in.contiguous() : t_in.to(at::kFloat).contiguous();
    ids = ids_in.to(at::kLong).contiguous();
    if (labels_in.defined()) labels = labels_in.to(at::kLong).contiguous();
    d.N = ids.numel() / ids.size(-1), d.V = z.size(-1), d.K = ids.size(-1);
    d.inner = d.N, d.stride_inner = d.N == 1 ? d.V : z.stride(-2);
    if (z.dim() == 3) d.inner = z.size(1), d.stride_outer = z.stride(0), d.stride_inner = z.stride(1);
    d.Z = ptr(z);
    d.teacher_ids = static_cast<const int64_t*>(ptr(ids));
    d.teacher = ptr(t);
    d.teacher_dtype = gs_dtype_of(t, "teacher logits");
    d.labels = static_cast<const int64_t*>(ptr(labels));
    d.ignore_index = how.ignore_index;
    d.temperature = static_cast<float>(how.temperature), d.alpha = static_cast<float>(how.alpha);
    d.reduction = how.reduction;
  }

  // Elements past a 16-byte boundary: the kernels read and write the same pieces of rows and gradient.
  int64_t offset(const Tensor& x) const {
    return static_cast<int64_t>(reinterpret_cast<uintptr_t>(ptr(x)) % 16) / x.element_size();
  }
  Tensor empty_gradient() const {
    const auto options = z.options().requires_grad(false);
    const int64_t span = span_of(z), off = offset(z);
    if (off == 0 && span == z.numel()) return at::empty(z.sizes(), options);
    return at::empty({off + span}, options).as_strided(z.sizes(), z.strides(), off);
  }
  bool fits(const Tensor& grad) const {
    return grad.sizes() == z.sizes() && grad.strides() == z.strides() && offset(grad) == offset(z);
  }
  Tensor workspace() const { return scratch(gs_distill_workspace(&d), z); }
};

// The loss; with `unit` also the gradient for an upstream of one, and the call's scratch.
Tensor distill_loss(const Tensor& logits, const Tensor& ids, const Tensor& t, const Tensor& labels,
                    const DistillHow& how, Tensor* unit, Tensor* ws_kept) {
  const DistillCall c(logits, ids, t, labels, how);
  const auto fp32 = logits.options().dtype(at::kFloat).requires_grad(false);
  const at::IntArrayRef shape = how.reduction == GS_REDUCE_NONE
                                    ? logits.sizes().slice(0, logits.dim() - 1) : at::IntArrayRef();
  if (c.d.N == 0)
    return at::full(shape, how.reduction == GS_REDUCE_MEAN ? std::nan("") : 0.0, fp32);
  const Tensor loss = at::empty(shape, fp32), ws = c.workspace();
  if (unit != nullptr) {
    *unit = c.empty_gradient();
    *ws_kept = ws;
  }
  c10::DeviceGuard guard(c.dev);
  check(gs_distill_loss(&c.d, static_cast<float*>(mut(loss)), unit != nullptr ? mut(*unit) : nullptr,
                        mut(ws), static_cast<size_t>(ws.numel()), stream_on(c.dev)),
        "gs_distill_loss");
  return loss;
}

struct Distillation : torch::autograd::Function<Distillation> {
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& ids, const Tensor& t,
                        const OptTensor& labels, DistillHow how) {
    // A mean's or sum's gradient is written in the loss's own pass, for an upstream gradient of one;
    // the backward pass keeps it or, for another upstream, forms it again.
    const bool fused = how.reduction != GS_REDUCE_NONE;
    Tensor loss = distill_loss(logits, ids, t, given(labels), how, fused ? &how.unit : nullptr, &how.ws);
    ctx->save_for_backward({logits, ids, t, given(labels)});
    keep(ctx, std::move(how));
    return loss;
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const variable_list s = ctx->get_saved_variables();
    DistillHow& how = kept<DistillHow>(ctx);
    Tensor grad = std::move(how.unit), ws = std::move(how.ws);   // handed out once
    how.unit = how.ws = Tensor();
    const DistillCall c(s[0], s[1], s[2], s[3], how);
    if (c.d.N == 0) return once({at::empty_like(s[0]), Tensor(), Tensor(), Tensor(), Tensor()});
    const Tensor up = gradient_in_memory(g[0]).to(at::kFloat).contiguous();
    const bool filled = grad.defined() && c.fits(grad);   // autograd may have moved the logits
    if (!filled) grad = c.empty_gradient(), ws = c.workspace();
    {
      c10::DeviceGuard guard(c.dev);
      check(gs_distill_grad(&c.d, static_cast<const float*>(ptr(up)), filled, mut(grad), mut(ws),
                            static_cast<size_t>(ws.numel()), stream_on(c.dev)),
            "gs_distill_grad");
    }
    return once({grad.sizes() == s[0].sizes() ? grad : grad.view(s[0].sizes()), Tensor(), Tensor(),
                 Tensor(), Tensor()});
  }
};

Tensor distillation_loss(const Tensor& logits, const Tensor& ids, const Tensor& t,
                         const OptTensor& labels, double temperature, double alpha,
                         int64_t ignore_index, int reduction) {
  const Tensor y = given(labels);
  check_plain({&logits, &ids, &t, &y});
  DistillHow how{temperature, alpha, ignore_index, reduction, {}, {}};
  if (recorded({&logits}))
    return Distillation::apply(logits, ids.detach(), t.detach(), labels, std::move(how));
  return distill_loss(logits, ids, t, y, how, nullptr, nullptr);
}

}  // namespace

PYBIND11_MODULE(_lm_autograd, m) {
  static PyObject* error = nullptr;   // lives as long as the process
  m.def("raise_as", [](py::object type) { error = type.release().ptr(); },
        "The exception class for refused arguments and failed calls.");
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const GhostError& e) {
      PyErr_SetString(error != nullptr ? error : PyExc_RuntimeError, e.what());
    }
  });
  m.def("embedding_lookup", &embedding_lookup);
  m.def("qk_norm_rotary", &qk_norm_rotary);
  m.def("qk_norm_rotary_dots", &qk_norm_rotary_dots);
  m.def("qk_sample_dots", &qk_sample_dots);
  m.def("distillation_loss", &distillation_loss);
}
