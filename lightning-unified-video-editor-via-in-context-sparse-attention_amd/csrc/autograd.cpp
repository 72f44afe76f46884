// Autograd nodes of the training operators (icsa_hip/train.py) over the C ABI of libicsa.so.
//
// A Python autograd function runs its backward on a thread of autograd's own, which waits for the interpreter and finds its objects
// in another core's cache: a layer norm of six rows, forward and backward, took 130 us in Python and 63 here, where the
// backward never enters the interpreter.
//
// Arguments have been checked in Python.  The library is the one that the package has loaded, found by its path.  What the
// backward reads is taken from the saved tensors, not remembered by address: hooks may have moved it.
#include <torch/extension.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <dlfcn.h>
#include <algorithm>

#include "../../include/icsa.h"

namespace {

using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
typedef c10::optional<Tensor> MaybeTensor;

struct Api {
  decltype(&icsa_last_error) last_error = nullptr;
  decltype(&icsa_cross_attn_workspace_size) attn_workspace;
  decltype(&icsa_cross_attn_fwd) attn_fwd;
  decltype(&icsa_cross_attn_wants_rest) attn_wants_rest;
  decltype(&icsa_cross_attn_bwd_workspace_size) attn_bwd_workspace;
  decltype(&icsa_cross_attn_bwd) attn_bwd;
  decltype(&icsa_norm_fwd) norm_fwd;
  decltype(&icsa_norm_bwd_workspace_size) norm_workspace;
  decltype(&icsa_norm_bwd) norm_bwd;
  decltype(&icsa_rotary) rotary;
} api;
PyObject* g_error = nullptr;                          // icsa_hip._lib.IcsaError

void bind(const std::string& path, py::object error) {
  void* h = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);
  TORCH_CHECK(h, "cannot open ", path, ": ", dlerror());
  auto get = [&](auto& f, const char* name) {
    f = reinterpret_cast<std::decay_t<decltype(f)>>(dlsym(h, name));
    TORCH_CHECK(f, path, " lacks ", name);
  };
  get(api.attn_workspace, "icsa_cross_attn_workspace_size");
  get(api.attn_fwd, "icsa_cross_attn_fwd");
  get(api.attn_wants_rest, "icsa_cross_attn_wants_rest");
  get(api.attn_bwd_workspace, "icsa_cross_attn_bwd_workspace_size");
  get(api.attn_bwd, "icsa_cross_attn_bwd");
  get(api.norm_fwd, "icsa_norm_fwd");
  get(api.norm_workspace, "icsa_norm_bwd_workspace_size");
  get(api.norm_bwd, "icsa_norm_bwd");
  get(api.rotary, "icsa_rotary");
  get(api.last_error, "icsa_last_error");
  g_error = error.release().ptr();
}

struct Failure : public torch::PyTorchError {
  explicit Failure(const std::string& what) : PyTorchError(what) {}
  PyObject* python_type() override { return g_error; }
};

void check(const char* fn, int64_t code) {
  if (code < 0) throw Failure(std::string(fn) + " failed with status " + std::to_string(code) + ": " + api.last_error());
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

// Inputs with memory of their own, in a call that is not traced.  A batched, lifted or functional tensor has none; a null address (of a
// wrapper, or a tensor of zeros that is none) would read as an operand that is not given; and a trace would hold the results'
// allocation without what fills it.
void require_plain(std::initializer_list<const Tensor*> ts) {
  bool plain = !torch::jit::tracer::isTracing();
  for (const Tensor* t : ts)
    plain = plain && (!t->defined() || (t->has_storage() && !t->key_set().has(c10::DispatchKey::Functionalize) &&
                                        (t->numel() == 0 || t->data_ptr() != nullptr)));
  TORCH_CHECK_NOT_IMPLEMENTED(plain, "icsa_hip's training operators take tensors with memory of their own: not under vmap, torch.func, "
                                     "batched gradients or tracing");
}

// constants: inputs without a gradient, which may have no tangent either
bool wants_grad(std::initializer_list<const Tensor*> ts, std::initializer_list<const Tensor*> constants = {}) {
  auto no_tangent = [](const Tensor& t) {
    TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), "icsa_hip's training operators have no forward-mode derivative");
  };
  bool some = false;
  for (const Tensor* t : ts)
    if (t->defined()) {
      no_tangent(*t);
      some = some || t->requires_grad();
    }
  for (const Tensor* t : constants) no_tangent(*t);
  return some && c10::GradMode::is_enabled();
}

template <class N, class... T> std::shared_ptr<N> make_node(const T&... inputs) {
  std::shared_ptr<N> node(new N(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(inputs...));
  return node;
}

// A captured backward must not meet a node that an eager graph has made on another stream, a leaf's accumulation among them, as
// long as that graph lives: the engine would have the one wait for the other, which a capture does not allow, and the process
// ends.  Refused while nothing of it is captured.
void refuse_capture(std::initializer_list<const Tensor*> ts) {
  auto capturing = [](hipStream_t s) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    return s != nullptr && hipStreamIsCapturing(s, &status) == hipSuccess && status == hipStreamCaptureStatusActive;
  };
  const auto now = c10::hip::getCurrentHIPStream((*ts.begin())->device().index());
  if (!capturing(now.stream())) return;
  for (const Tensor* t : ts) {
    if (!t->defined() || !t->requires_grad()) continue;
    const std::shared_ptr<torch::autograd::Node> node = t->grad_fn() ? t->grad_fn() : torch::autograd::impl::try_get_grad_accumulator(*t);
    const auto of = node ? node->stream() : std::nullopt;
    if (!of || of->id() == now.id()) continue;
    if (!capturing(c10::hip::HIPStream(c10::hip::HIPStream::UNCHECKED, *of).stream()))
      throw Failure("under capture an input has a node of an eager graph: drop that graph, or detach the input, before a backward is captured "
                    "(torch.no_grad() for a forward alone)");
  }
}

Tensor get(const MaybeTensor& t) { return t.has_value() ? *t : Tensor(); }
void* at_or_null(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
int code_of(at::ScalarType t) { return t == at::kBFloat16 ? ICSA_BF16 : ICSA_F32; }

Tensor workspace(int64_t bytes, const Tensor& like) {
  return bytes > 0 ? at::empty({bytes}, like.options().dtype(at::kByte)) : Tensor();
}

// Gradients have none themselves: where a graph of them is asked for they raise when it is used.
variable_list once(variable_list grads) {
  if (!c10::GradMode::is_enabled()) return grads;
  variable_list in;
  for (const Tensor& g : grads) in.push_back(g.defined() ? g.detach().set_requires_grad(true) : g);
  torch::autograd::DelayedError error("icsa_hip's training operators have no second derivative", (int64_t)in.size());
  return error.apply(std::move(in));
}

// t [B, S, H, D] with a unit stride in each row and rows on 16 bytes (itself where they are), its address and strides.  group: of
// heads (1 for k, v) where 64 rows with a group's heads have to lie within 2 GiB, as the backward reads them; 0: they need not.
struct Rows {
  Tensor t;
  void* p;
  int64_t sb, ss, sh;
};
Rows rows16(const Tensor& t, int64_t group) {
  auto of = [](const Tensor& x) {
    Rows r{x, x.data_ptr(), x.size(0) > 1 ? x.stride(0) : 0, x.size(1) > 1 ? x.stride(1) : 0, x.size(2) > 1 ? x.stride(2) : 0};
    return r;
  };
  auto ok = [group](const Rows& r) {
    const int64_t most = 0x3fffffff;
    return r.t.stride(3) == 1 && ((reinterpret_cast<uintptr_t>(r.p) | (uintptr_t)((r.sb | r.ss | r.sh) * 2)) & 15) == 0 &&
           (group == 0 || (r.ss <= most / 65 && (group == 1 || r.sh <= (most - 65 * r.ss) / group)));
  };
  Rows r = of(t);
  if (ok(r)) return r;
  r = of(t.contiguous());
  return ok(r) || !t.is_contiguous() ? r : of(t.clone(at::MemoryFormat::Contiguous));
}

// ------------------------------------------------------------------------------------------ cross attention
// a saved tensor, contiguous as it was (hooks may have changed its strides), or none
Tensor whole(SavedVariable& s) {
  const Tensor t = s.unpack();
  return t.defined() ? t.contiguous() : t;
}

struct AttnSizes {
  int B, Sq, Sk, H, Hk, D;
};
AttnSizes attn_sizes(const Tensor& q, const Tensor& k) {
  return {(int)q.size(0), (int)q.size(1), (int)k.size(1), (int)q.size(2), (int)k.size(2), (int)q.size(3)};
}

// out, and with them the state of the backward: lse and rest
Tensor attn_forward(const Rows& q, const Rows& k, const Rows& v, const Tensor& qs, const Tensor& ks, int64_t docs, double scale,
                    Tensor* lse, Tensor* rest) {
  c10::DeviceGuard guard(q.t.device());
  const AttnSizes z = attn_sizes(q.t, k.t);
  Tensor out = at::empty({z.B, z.Sq, z.H, z.D}, q.t.options());
  if (lse != nullptr) {
    *lse = at::empty({z.B, z.Hk, z.Sq, z.H / z.Hk}, q.t.options().dtype(at::kFloat));
    if (api.attn_wants_rest(z.Sq, z.Sk, z.H, z.Hk, z.D, qs.defined())) *rest = at::empty({z.B, z.Sq, z.H, z.D}, q.t.options().dtype(at::kByte));
  }
  const int64_t bytes = api.attn_workspace(z.B, z.Sq, z.Sk, z.H, z.Hk, z.D, (int)docs);
  check("icsa_cross_attn_workspace_size", bytes);
  const Tensor ws = workspace(bytes, out);
  check("icsa_cross_attn_fwd",
        api.attn_fwd(q.p, q.sb, q.ss, q.sh, k.p, k.sb, k.ss, k.sh, v.p, v.sb, v.ss, v.sh, z.B, z.Sq, z.Sk, z.H, z.Hk, z.D,
                     (const int32_t*)at_or_null(qs), (const int32_t*)at_or_null(ks), (int)docs, (float)scale, out.data_ptr(),
                     (int64_t)z.Sq * z.H * z.D, (int64_t)z.H * z.D, z.D, lse ? (float*)lse->data_ptr() : nullptr,
                     rest ? at_or_null(*rest) : nullptr, at_or_null(ws), bytes, stream_of(out)));
  return out;
}

struct CrossAttnBackward : public torch::autograd::Node {
  SavedVariable q, k, v, qs, ks, out, lse, rest;
  int docs = 1;
  double scale = 1.;
  std::string name() const override { return "CrossAttnBackward"; }

  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* s : {&q, &k, &v, &qs, &ks, &out, &lse, &rest}) s->reset_data();
  }

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list res(3);
    if (!grads[0].defined()) return res;
    require_plain({&grads[0]});
    const Tensor sq = q.unpack(), sk = k.unpack(), sv = v.unpack(), so = out.unpack(shared_from_this());
    {
      at::AutoDispatchBelowADInplaceOrView below;
      c10::DeviceGuard guard(grads[0].device());
      const int64_t G = sq.size(2) / sk.size(2);
      const Rows g = rows16(grads[0], G), q = rows16(sq, G), k = rows16(sk, 1), v = rows16(sv, 1), o = rows16(so, 0);
      const Tensor lse = whole(this->lse), rest = whole(this->rest), qs = whole(this->qs), ks = whole(this->ks);
      const AttnSizes z = attn_sizes(q.t, k.t);
      const auto opt = q.t.options();
      if (task_should_compute_output(0)) res[0] = at::empty({z.B, z.Sq, z.H, z.D}, opt);
      if (task_should_compute_output(1)) res[1] = at::empty({z.B, z.Sk, z.Hk, z.D}, opt);
      if (task_should_compute_output(2)) res[2] = at::empty({z.B, z.Sk, z.Hk, z.D}, opt);
      const int64_t bytes = api.attn_bwd_workspace(z.B, z.Sq, z.Sk, z.H, z.Hk, z.D, docs);
      check("icsa_cross_attn_bwd_workspace_size", bytes);
      const Tensor ws = workspace(bytes, q.t);
      const int64_t qss = (int64_t)z.H * z.D, kss = (int64_t)z.Hk * z.D;
      check("icsa_cross_attn_bwd",
            api.attn_bwd(g.p, g.sb, g.ss, g.sh, q.p, q.sb, q.ss, q.sh, k.p, k.sb, k.ss, k.sh, v.p, v.sb, v.ss, v.sh, o.p, o.sb, o.ss, o.sh,
                         (const float*)lse.data_ptr(), at_or_null(rest), z.B, z.Sq, z.Sk, z.H, z.Hk, z.D,
                         (const int32_t*)at_or_null(qs), (const int32_t*)at_or_null(ks), docs, (float)scale, ICSA_BF16,
                         at_or_null(res[0]), z.Sq * qss, qss, z.D, at_or_null(res[1]), z.Sk * kss, kss, z.D,
                         at_or_null(res[2]), z.Sk * kss, kss, z.D, at_or_null(ws), bytes, stream_of(q.t)));
    }
    return once(std::move(res));
  }
};

Tensor cross_attn(const Tensor& q_, const Tensor& k_, const Tensor& v_, const MaybeTensor& qs_, const MaybeTensor& ks_, int64_t docs,
                  double scale) {
  const Tensor qs = get(qs_), ks = get(ks_);
  require_plain({&q_, &k_, &v_, &qs, &ks});
  std::shared_ptr<CrossAttnBackward> node;
  if (wants_grad({&q_, &k_, &v_})) {
    refuse_capture({&q_, &k_, &v_});
    node = make_node<CrossAttnBackward>(q_, k_, v_);
  }
  Tensor out, lse, rest;
  Rows q, k, v;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    q = rows16(q_, node ? q_.size(2) / k_.size(2) : 0);
    k = rows16(k_, node ? 1 : 0);
    v = rows16(v_, node ? 1 : 0);
    out = attn_forward(q, k, v, qs, ks, docs, scale, node ? &lse : nullptr, node ? &rest : nullptr);
  }
  if (node) {
    torch::autograd::set_history(out, node);
    node->q = SavedVariable(q.t, false);
    node->k = SavedVariable(k.t, false);
    node->v = SavedVariable(v.t, false);
    node->qs = SavedVariable(qs, false);
    node->ks = SavedVariable(ks, false);
    node->out = SavedVariable(out, true);
    node->lse = SavedVariable(lse, false);
    node->rest = SavedVariable(rest, false);
    node->docs = (int)docs;
    node->scale = scale;
  }
  return out;
}

// ------------------------------------------------------------------------------------------ layer norm, RMS norm
// t [..., dim] as [rows, dim] with a unit stride in each row
Tensor rows(const Tensor& t) {
  const Tensor x = t.size(-1) != 1 && t.stride(-1) != 1 ? t.contiguous() : t.resolve_neg();
  return x.dim() == 2 ? x : x.reshape({-1, x.size(-1)});
}
int64_t row_stride(const Tensor& x) { return x.size(0) > 1 ? x.stride(0) : x.size(1); }

// gain and shift as [groups, dim] with one group stride
struct Params {
  Tensor gain, shift;
  int groups = 1, code = ICSA_F32;
  int64_t stride = 0;
};
Params params(const Tensor& gain, const Tensor& shift) {
  Params p;
  if (!gain.defined()) return p;
  p.gain = rows(gain);
  if (shift.defined()) p.shift = rows(shift);
  if (p.gain.size(0) > 1 && p.shift.defined() && p.gain.stride(0) != p.shift.stride(0)) {
    p.gain = p.gain.contiguous();
    p.shift = p.shift.contiguous();
  }
  p.groups = std::max(1, (int)p.gain.size(0));          // without batch rows there are no rows either
  p.code = code_of(gain.scalar_type());
  p.stride = p.gain.stride(0);
  return p;
}

Tensor norm_forward(const Tensor& x, const Tensor& r, const Tensor& gain, const Tensor& shift, bool plus_one, bool rms, double eps,
                    at::ScalarType out, Tensor* stats) {
  c10::DeviceGuard guard(x.device());
  const Params p = params(gain, shift);
  const int64_t n = r.size(0), dim = r.size(1);
  Tensor y = at::empty(x.sizes(), x.options().dtype(out));
  float* rstd = nullptr;
  if (stats != nullptr) {                              // [1 / deviation, mean] of each row
    *stats = at::empty({rms ? 1 : 2, n}, x.options().dtype(at::kFloat));
    rstd = (float*)stats->data_ptr();
  }
  check("icsa_norm_fwd", api.norm_fwd(r.data_ptr(), code_of(r.scalar_type()), row_stride(r), n / p.groups, p.groups, (int)dim,
                                      at_or_null(p.gain), at_or_null(p.shift), p.code, p.stride, plus_one, rms, (float)eps, y.data_ptr(),
                                      code_of(out), dim, rstd && !rms ? rstd + n : nullptr, rstd, stream_of(x)));
  return y;
}

struct NormBackward : public torch::autograd::Node {
  SavedVariable x, gain, stats;
  std::vector<int64_t> x_sizes, shift_sizes;
  bool plus_one = false, rms = false, shifted = false;
  std::string name() const override { return rms ? "RmsNormBackward" : "LayerNormBackward"; }

  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* s : {&x, &gain, &stats}) s->reset_data();
  }

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list res(3);
    if (!grads[0].defined()) return res;
    require_plain({&grads[0]});
    const Tensor sx = x.unpack(), sg = gain.unpack();
    {
      at::AutoDispatchBelowADInplaceOrView below;
      c10::DeviceGuard guard(grads[0].device());
      const Tensor d = rows(grads[0]), r = rows(sx), stats = whole(this->stats);
      const Params p = params(sg, Tensor());
      const int64_t n = r.size(0), dim = r.size(1);
      const bool need_gain = sg.defined() && task_should_compute_output(1), need_shift = shifted && task_should_compute_output(2);
      if (task_should_compute_output(0)) res[0] = at::empty(x_sizes, r.options());
      auto make = [&](at::IntArrayRef size) { return n > 0 ? at::empty(size, sg.options()) : at::zeros(size, sg.options()); };
      if (need_gain) res[1] = make(sg.sizes());
      if (need_shift) res[2] = make(shift_sizes);
      if (n > 0) {
        const int64_t bytes = need_gain || need_shift ? api.norm_workspace(n / p.groups, p.groups, (int)dim) : 0;
        check("icsa_norm_bwd_workspace_size", bytes);
        const Tensor ws = workspace(bytes, r);
        check("icsa_norm_bwd", api.norm_bwd(d.data_ptr(), code_of(d.scalar_type()), row_stride(d), r.data_ptr(), code_of(r.scalar_type()),
                                            row_stride(r), n / p.groups, p.groups, (int)dim, at_or_null(p.gain), p.code, p.stride, plus_one,
                                            rms, rms ? nullptr : (const float*)stats.data_ptr() + n, (const float*)stats.data_ptr(),
                                            at_or_null(res[0]), dim, at_or_null(res[1]), at_or_null(res[2]), at_or_null(ws), bytes, stream_of(r)));
      }
    }
    return once(std::move(res));
  }
};

Tensor norm(const Tensor& x, const MaybeTensor& gain_, const MaybeTensor& shift_, bool plus_one, bool rms, double eps, at::ScalarType out) {
  const Tensor gain = get(gain_), shift = get(shift_);
  require_plain({&x, &gain, &shift});
  std::shared_ptr<NormBackward> node;
  if (wants_grad({&x, &gain, &shift})) {
    refuse_capture({&x, &gain, &shift});
    node = make_node<NormBackward>(x, gain, shift);
  }
  Tensor r, y, stats;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    r = rows(x);
    y = norm_forward(x, r, gain, shift, plus_one, rms, eps, out, node ? &stats : nullptr);
  }
  if (node) {
    torch::autograd::set_history(y, node);
    node->x = SavedVariable(r.is_alias_of(x) ? x : r, false);            // x itself: its changes in place are seen
    node->gain = SavedVariable(gain, false);
    node->stats = SavedVariable(stats, false);
    node->x_sizes = x.sizes().vec();
    node->plus_one = plus_one;
    node->rms = rms;
    node->shifted = shift.defined();
    if (shift.defined()) node->shift_sizes = shift.sizes().vec();
  }
  return y;
}

// ------------------------------------------------------------------------------------------ rotary positions
Tensor unit_last(const Tensor& t) { return !t.defined() ? t : t.size(-1) == 1 || t.stride(-1) == 1 ? t.resolve_neg() : t.contiguous(); }

// Both turned (either may be undefined), new and contiguous.  axes 0: one axis without sections.
std::pair<Tensor, Tensor> rotate(const Tensor& q_, const Tensor& k_, const Tensor& cos, const Tensor& sin, const Tensor& pos,
                                 const std::vector<int64_t>& sections, bool interleaved, bool back) {
  const Tensor x[2] = {unit_last(q_), unit_last(k_)};
  const Tensor& any = x[0].defined() ? x[0] : x[1];
  c10::DeviceGuard guard(any.device());
  Tensor y[2];
  void *xp[2] = {}, *yp[2] = {};
  int64_t st[2][3] = {};
  int H[2] = {};
  for (int i = 0; i < 2; ++i) {
    if (!x[i].defined()) continue;
    y[i] = at::empty(x[i].sizes(), x[i].options());
    xp[i] = x[i].data_ptr();
    yp[i] = y[i].data_ptr();
    H[i] = (int)x[i].size(2);
    for (int d = 0; d < 3; ++d) st[i][d] = x[i].stride(d);
  }
  int32_t sec[4] = {};
  for (size_t i = 0; i < sections.size() && i < 4; ++i) sec[i] = (int32_t)sections[i];
  const int axes = sections.empty() ? 1 : (int)sections.size();
  const bool each = pos.dim() == (sections.empty() ? 2 : 3);
  check("icsa_rotary",
        api.rotary(xp[0], st[0][0], st[0][1], st[0][2], H[0], yp[0], xp[1], st[1][0], st[1][1], st[1][2], H[1], yp[1],
                   code_of(any.scalar_type()), (int)any.size(0), (int)any.size(1), (int)any.size(3), 2 * (int)cos.size(1), interleaved,
                   back, (const int32_t*)pos.data_ptr(), each ? pos.stride(0) : 0, axes, sections.empty() ? nullptr : sec,
                   (const float*)cos.data_ptr(), (const float*)sin.data_ptr(), (int)cos.size(0), stream_of(any)));
  return {y[0], y[1]};
}

struct RotaryBackward : public torch::autograd::Node {
  SavedVariable cos, sin, pos;
  std::vector<int64_t> sections;
  bool interleaved = true;
  std::string name() const override { return "RotaryBackward"; }

  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* s : {&cos, &sin, &pos}) s->reset_data();
  }

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list res(2);
    {
      at::AutoDispatchBelowADInplaceOrView below;
      const Tensor c = whole(cos), s = whole(sin), p = whole(pos);
      const Tensor dq = task_should_compute_output(0) ? grads[0] : Tensor();
      const Tensor dk = grads.size() > 1 && task_should_compute_output(1) ? grads[1] : Tensor();
      require_plain({&dq, &dk});
      if (dq.defined() || dk.defined()) std::tie(res[0], res[1]) = rotate(dq, dk, c, s, p, sections, interleaved, true);
    }
    return once(std::move(res));
  }
};

variable_list rotary(const Tensor& q, const MaybeTensor& k_, const Tensor& cos, const Tensor& sin, const Tensor& pos,
                     std::vector<int64_t> sections, bool interleaved) {
  const Tensor k = get(k_);
  require_plain({&q, &k, &cos, &sin, &pos});
  const bool grad = wants_grad({&q, &k}, {&cos, &sin});
  const Tensor c = cos.contiguous().resolve_neg(), s = sin.contiguous().resolve_neg(), p = pos.contiguous();
  std::shared_ptr<RotaryBackward> node;
  if (grad) {
    refuse_capture({&q, &k});
    node = make_node<RotaryBackward>(q, k);
  }
  variable_list out;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    auto y = rotate(q, k, c, s, p, sections, interleaved, false);
    out.push_back(y.first);
    if (k.defined()) out.push_back(y.second);
  }
  if (node) {
    torch::autograd::set_history(out, node);
    node->cos = SavedVariable(c, false);
    node->sin = SavedVariable(s, false);
    node->pos = SavedVariable(p, false);
    node->sections = std::move(sections);
    node->interleaved = interleaved;
  }
  return out;
}

}  // namespace

// Without the interpreter's lock, as torch's own operators and the package's calls of the library: allocations and launches may wait.
PYBIND11_MODULE(_autograd, m) {
  m.def("bind", torch::wrap_pybind_function(bind));
  m.def("cross_attn", torch::wrap_pybind_function_no_gil(cross_attn));
  m.def("norm", torch::wrap_pybind_function_no_gil(norm));
  m.def("rotary", torch::wrap_pybind_function_no_gil(rotary));
}
