// The host side of the PyTorch entry points in native code: argument checks, output and workspace allocation and the
// autograd chain around the C ABI of libfhog_hip.so (include/fhog_hip.h). A call that is anything but well formed is declined
// (None, or no tensors), and the Python wrappers then find out what is wrong with it and say so; they also take what needs
// the workspace afterwards (row statistics, single passes).
//
// Why native: on short sequences the GPU finishes before Python has prepared the next launch. Host time per call, the Python
// wrappers -> here (same machine): flash_bwdbwd 56 -> 14 us; attention() differentiated twice 208 -> 154 us, of which some 100 are
// torch's own two calls of autograd.grad. On fresh tensors, where the Python nodes also hand the interpreter lock back and forth
// between the caller's and autograd's threads, that program went from 393 to 149 us on 2 x 256 bf16 rows.
#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <cmath>
#include <optional>
#include <tuple>

#include "fhog_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::tensor_list;

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return FHOG_DTYPE_BF16;
    case at::kHalf: return FHOG_DTYPE_FP16;
    case at::kFloat: return FHOG_DTYPE_FP32;
    default: return -1;
  }
}

// False where the storage holds no memory: fake tensors and wrappers of other tensors, and storages that were resized to nothing. A view of one that starts behind its first
// element has an address all the same, and it is no one's.
bool in_memory(const Tensor& t) { return !t.has_storage() || t.numel() == 0 || t.storage().data() != nullptr; }

// (batch, N, d) or (B, H, N, d) as the library sees it: batch = B * H slices sb elements apart, rows sn elements apart
struct Layout {
  int64_t batch = 0, n = 0, d = 0, sb = 0, sn = 0;
  bool direct = false;   // usable where it lies: contiguous rows, 16-byte multiples, slices that do not overlap
  bool rows = false;     // contiguous rows, and (B, H) is one dimension of evenly spaced slices
};

Layout layout_of(const Tensor& t) {
  Layout l;
  const auto s = t.sizes(), st = t.strides();
  const int64_t dim = t.dim();
  if (dim != 3 && dim != 4) return l;
  l.n = s[dim - 2], l.d = s[dim - 1], l.sn = st[dim - 2];
  l.batch = dim == 3 ? s[0] : s[0] * s[1];
  const int64_t vec = 16 / t.element_size();
  l.rows = st[dim - 1] == 1;
  if (dim == 3 || s[1] == 1) l.sb = st[0];
  else l.sb = st[1], l.rows = l.rows && (s[0] == 1 || st[0] == s[1] * st[1]);
  if (l.batch == 1) l.sb = l.n * l.sn;   // never used to address anything
  l.direct = l.rows && l.sn >= l.d && l.sn % vec == 0 && l.sb % vec == 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && (l.batch == 1 || l.sb >= l.n * l.sn);
  return l;
}

// Tensors of one group share shape, type, device, batch stride and row stride; copied into contiguous ones if they do not.
// strict: rows that are contiguous but not 16-byte multiples apart are declined instead (the first-order entry points
// have always left those to their callers).
template <size_t N>
struct Group {
  std::array<Tensor, N> t;
  Layout l;
  // shapes, types and devices have to agree with the first tensor
  bool set(const std::array<const Tensor*, N>& in, bool strict) {
    bool same = true;
    for (size_t i = 0; i < N; i++) {
      if (!in[i]->defined() || !in_memory(*in[i]) || !in[i]->is_cuda() || in[i]->scalar_type() != in[0]->scalar_type() || in[i]->device() != in[0]->device())
        return false;
      t[i] = *in[i];
      Layout x = layout_of(t[i]);
      if (strict && !x.direct) {
        if (x.rows) return false;
        t[i] = t[i].contiguous();
        x = layout_of(t[i]);
      }
      if (i == 0) l = x;
      if (x.n != l.n || x.d != l.d || x.batch != l.batch || x.batch == 0) return false;
      same = same && x.direct && x.sb == l.sb && x.sn == l.sn;
    }
    if (!same) {
      for (auto& x : t) x = x.contiguous();
      l = layout_of(t[0]);
      for (auto& x : t)
        if (!layout_of(x).direct) return false;
    }
    return true;
  }
  void* ptr(size_t i) const { return t[i].data_ptr(); }
  Tensor like() const { return at::empty_strided(t[0].sizes(), t[0].strides(), t[0].options()); }
};

// What autograd hands over, packed. contiguous() passes over the stride of a dimension of one (a single query that came back
// through (B, 1, H, d)) and over the address, both of which the kernels look at.
Tensor packed(const Tensor& t) {
  const Tensor c = t.contiguous();
  return layout_of(c).direct ? c : c.clone(at::MemoryFormat::Contiguous);
}

// What a saved-tensor hook gave back may lie anywhere; where it lies as it was saved nothing is copied.
Tensor unpacked(const Tensor& t) { return layout_of(t).direct ? t : packed(t); }
Tensor unpacked_lse(const Tensor& L) {
  return reinterpret_cast<uintptr_t>(L.data_ptr()) % 16 == 0 ? L : L.clone(at::MemoryFormat::Contiguous);
}

Tensor as_lse(const Tensor& L) { return L.scalar_type() == at::kFloat && L.is_contiguous() ? L : L.to(at::kFloat).contiguous(); }
Tensor workspace(int64_t bytes, const Tensor& like) { return at::empty({(bytes + 3) / 4}, like.options().dtype(at::kFloat)); }
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

struct Mask {
  int32_t causal;
  int64_t window, sinks;
};

bool mask_applies(const Mask& m, int64_t n_q, int64_t n_k) {
  if (m.causal < FHOG_MASK_NONE || m.causal > FHOG_MASK_BOTTOM_RIGHT || m.window < 0 || m.window > INT32_MAX || m.sinks < 0) return false;
  if (m.causal == FHOG_MASK_NONE) return m.window == 0;
  return m.causal == FHOG_MASK_TOP_LEFT ? n_q == n_k : n_k >= n_q;
}

template <size_t NQ, size_t NK>
bool attn_args(fhog_attn_args& a, const Group<NQ>& q, const Group<NK>& k, double scale, const Mask& m) {
  if (k.l.batch != q.l.batch || k.l.d != q.l.d || k.t[0].scalar_type() != q.t[0].scalar_type() || k.t[0].device() != q.t[0].device() ||
      !mask_applies(m, q.l.n, k.l.n))
    return false;
  a = {};
  a.q = q.ptr(0), a.k = k.ptr(0), a.v = k.ptr(1);
  a.batch = q.l.batch, a.n_q = q.l.n, a.n_k = k.l.n, a.d = q.l.d;
  a.stride_qb = q.l.sb, a.stride_qn = q.l.sn, a.stride_kb = k.l.sb, a.stride_kn = k.l.sn;
  a.scale = (float)scale, a.dtype = dtype_code(q.t[0].scalar_type()), a.causal = m.causal, a.window = (int32_t)m.window;
  return a.dtype >= 0;
}

using Forward = std::optional<std::tuple<Tensor, Tensor>>;
Forward forward(const Tensor& q_, const Tensor& k_, const Tensor& v_, double scale, const Mask& m) {
  Group<1> q;
  Group<2> k;
  fhog_attn_args a;
  if (!q.set({&q_}, true) || !k.set({&k_, &v_}, true) || !attn_args(a, q, k, scale, m)) return std::nullopt;
  const c10::DeviceGuard guard(q_.device());
  Tensor o = q.like();
  Tensor lse = at::empty(q_.sizes().slice(0, q_.dim() - 1), q_.options().dtype(at::kFloat));
  a.o = o.data_ptr(), a.lse = (float*)lse.data_ptr();
  if (fhog_attn_validate(&a, 0) != FHOG_OK) return std::nullopt;
  if (m.sinks == 0) {
    TORCH_CHECK(fhog_attn_fwd(&a, stream_of(q_)) == FHOG_OK, "fhog_attn_fwd: ", fhog_last_error());
  } else {
    const int64_t bytes = (int64_t)fhog_attn_sinks_workspace_bytes(&a, m.sinks, 0);
    const Tensor ws = workspace(bytes, q_);
    TORCH_CHECK(fhog_attn_fwd_sinks(&a, m.sinks, ws.data_ptr(), bytes, stream_of(q_)) == FHOG_OK, "fhog_attn_fwd_sinks: ", fhog_last_error());
  }
  return std::make_tuple(o, lse);
}

using Backward = std::optional<std::tuple<Tensor, Tensor, Tensor>>;
Backward backward(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& o_, const Tensor& do_, const Tensor& L, double scale,
                  const Mask& m, bool strict) {
  Group<3> q;
  Group<2> k;
  fhog_attn_args a;
  if (!q.set({&q_, &o_, &do_}, strict) || !k.set({&k_, &v_}, strict) || !attn_args(a, q, k, scale, m)) return std::nullopt;
  if (!in_memory(L) || !L.is_cuda() || L.device() != q_.device() || L.numel() != a.batch * a.n_q) return std::nullopt;
  const c10::DeviceGuard guard(q_.device());
  const Tensor lse = as_lse(L);
  Tensor dq = q.like(), dk = k.like(), dv = k.like();
  a.o = q.ptr(1), a.dO = q.ptr(2), a.lse = (float*)lse.data_ptr();
  a.dq = dq.data_ptr(), a.dk = dk.data_ptr(), a.dv = dv.data_ptr();
  int64_t bytes = a.batch * a.n_q * 4;
  if (m.sinks > 0) bytes = std::max(bytes, (int64_t)fhog_attn_sinks_workspace_bytes(&a, m.sinks, 1));
  const Tensor ws = workspace(bytes, q_);
  a.ws = (float*)ws.data_ptr();
  if (fhog_attn_validate(&a, 1) != FHOG_OK) return std::nullopt;
  const int rc = m.sinks > 0 ? fhog_attn_bwd_sinks(&a, m.sinks, bytes, stream_of(q_)) : fhog_attn_bwd(&a, stream_of(q_));
  TORCH_CHECK(rc == FHOG_OK, m.sinks > 0 ? "fhog_attn_bwd_sinks: " : "fhog_attn_bwd: ", fhog_last_error());
  return std::make_tuple(dq, dk, dv);
}

using DoubleBackward = std::optional<std::tuple<Tensor, Tensor, Tensor, Tensor>>;
DoubleBackward double_backward(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& o_, const Tensor& do_, const Tensor& ddq_,
                               const Tensor& ddk_, const Tensor& ddv_, const Tensor& L, double scale, const Mask& m, int impl, int schedule,
                               bool split) {
  Group<4> q, k;
  if (!q.set({&q_, &o_, &do_, &ddq_}, false) || !k.set({&k_, &v_, &ddk_, &ddv_}, false)) return std::nullopt;
  if (k.l.batch != q.l.batch || k.l.d != q.l.d || k_.scalar_type() != q_.scalar_type() || k_.device() != q_.device() ||
      !mask_applies(m, q.l.n, k.l.n) || !in_memory(L) || !L.is_cuda() || L.device() != q_.device() || L.numel() != q.l.batch * q.l.n)
    return std::nullopt;
  fhog_bwdbwd_args a = {};
  a.dtype = dtype_code(q_.scalar_type());
  if (a.dtype < 0) return std::nullopt;
  const c10::DeviceGuard guard(q_.device());
  const Tensor lse = as_lse(L);
  Tensor dq2 = q.like(), ddo = q.like(), dk2 = k.like(), dv2 = k.like();
  a.q = q.ptr(0), a.o = q.ptr(1), a.dO = q.ptr(2), a.ddq = q.ptr(3);
  a.k = k.ptr(0), a.v = k.ptr(1), a.ddk = k.ptr(2), a.ddv = k.ptr(3);
  a.lse = (const float*)lse.data_ptr();
  a.dq2 = dq2.data_ptr(), a.dk2 = dk2.data_ptr(), a.dv2 = dv2.data_ptr(), a.ddo = ddo.data_ptr();
  a.batch = q.l.batch, a.n_q = q.l.n, a.n_k = k.l.n, a.d = q.l.d;
  a.stride_qb = q.l.sb, a.stride_qn = q.l.sn, a.stride_kb = k.l.sb, a.stride_kn = k.l.sn;
  a.scale = (float)scale, a.causal = m.causal, a.window = m.window, a.impl = impl, a.schedule = schedule;
  a.ws = (float*)q.ptr(0);   // any valid pointer: the hint is computed on the host
  if (m.sinks > 0 && schedule != FHOG_SCHEDULE_FUSED_STATS) return std::nullopt;
  const size_t hint = m.sinks > 0 ? fhog_bwdbwd_sinks_workspace_bytes(&a, m.sinks) : fhog_bwdbwd_workspace_hint(&a);
  if (hint == 0) return std::nullopt;   // not valid
  const int64_t bytes = split || m.sinks > 0 ? (int64_t)hint : 3 * a.batch * a.n_q * 4;
  const Tensor ws = workspace(bytes, q_);
  a.ws = (float*)ws.data_ptr(), a.ws_bytes = bytes;
  const int rc = m.sinks > 0 ? fhog_bwdbwd_sinks(&a, m.sinks, stream_of(q_)) : fhog_bwdbwd(&a, stream_of(q_));
  TORCH_CHECK(rc == FHOG_OK, m.sinks > 0 ? "fhog_bwdbwd_sinks: " : "fhog_bwdbwd: ", fhog_last_error());
  return std::make_tuple(dq2, dk2, dv2, ddo);
}

// ---- autograd: attention -> first backward -> double-backward (the chain of the Python classes in attention.py) ------
double scale_of(const Tensor& q) { return 1.0 / std::sqrt((double)q.size(-1)); }

struct FirstBackward : torch::autograd::Function<FirstBackward> {
  static tensor_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& o, const Tensor& grad,
                             const Tensor& L, int64_t causal, int64_t window, int64_t schedule, int64_t sinks) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({q, k, v, o, grad, L});
    ctx->saved_data["arg"] = std::vector<int64_t>{causal, window, schedule, sinks};
    const auto r = backward_(q, k, v, o, grad, L, causal, window, sinks);
    return {std::get<0>(r), std::get<1>(r), std::get<2>(r)};
  }
  static std::tuple<Tensor, Tensor, Tensor> backward_(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& o, const Tensor& grad,
                                                      const Tensor& L, int64_t causal, int64_t window, int64_t sinks) {
    const auto r = ::backward(unpacked(q), unpacked(k), unpacked(v), unpacked(o), grad, unpacked_lse(L), scale_of(q), Mask{(int32_t)causal, window, sinks}, false);
    TORCH_CHECK(r, "fhog: first-order backward: ", fhog_last_error());
    return *r;
  }
  static tensor_list backward(AutogradContext* ctx, tensor_list g) {
    tensor_list out(10);
    if (!g[0].defined() && !g[1].defined() && !g[2].defined()) return out;
    const auto s = ctx->get_saved_variables();
    const auto arg = ctx->saved_data["arg"].toIntVector();
    const bool differentiable = at::GradMode::is_enabled() && ((g[0].defined() && g[0].requires_grad()) || (g[1].defined() && g[1].requires_grad()) ||
                                                               (g[2].defined() && g[2].requires_grad()));
    {
      const at::NoGradGuard no_grad;
      const auto dir = [&](size_t i) { return g[i].defined() ? packed(g[i]) : at::zeros_like(s[i]); };
      const auto r = double_backward(unpacked(s[0]), unpacked(s[1]), unpacked(s[2]), unpacked(s[3]), unpacked(s[4]), dir(0), dir(1), dir(2),
                                     unpacked_lse(s[5]), scale_of(s[0]), Mask{(int32_t)arg[0], arg[1], arg[3]}, FHOG_IMPL_AUTO, (int)arg[2], true);
      TORCH_CHECK(r, "fhog: double-backward: ", fhog_last_error());
      // O and L are caches of (q, k, v): the four results are already total derivatives
      out[0] = std::get<0>(*r), out[1] = std::get<1>(*r), out[2] = std::get<2>(*r), out[4] = std::get<3>(*r);
    }
    if (differentiable) {   // third derivatives do not exist: say so when they are asked for
      tensor_list v = {out[0].detach().requires_grad_(), out[1].detach().requires_grad_(), out[2].detach().requires_grad_(), out[4].detach().requires_grad_()};
      const auto err = std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice the double-backward of fhog.attention", 4);
      v = err->apply(std::move(v));
      out[0] = v[0], out[1] = v[1], out[2] = v[2], out[4] = v[3];
    }
    return out;
  }
};

struct Attention : torch::autograd::Function<Attention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, int64_t causal, int64_t window, int64_t schedule,
                        int64_t sinks) {
    // The graph of the first backward reaches this node a second time through the saved O, whose gradient FirstBackward
    // does not have: without work to do, and not to be filled in with zeros
    ctx->set_materialize_grads(false);
    const auto r = ::forward(q, k, v, scale_of(q), Mask{(int32_t)causal, window, sinks});
    TORCH_CHECK(r, "fhog: forward: ", fhog_last_error());
    ctx->save_for_backward({q, k, v, std::get<0>(*r), std::get<1>(*r)});
    ctx->saved_data["arg"] = std::vector<int64_t>{causal, window, schedule, sinks};
    return std::get<0>(*r);
  }
  static tensor_list backward(AutogradContext* ctx, tensor_list g) {
    tensor_list out(7);
    if (!g[0].defined()) return out;
    const auto s = ctx->get_saved_variables();
    const auto arg = ctx->saved_data["arg"].toIntVector();
    const auto r = FirstBackward::apply(s[0], s[1], s[2], s[3], packed(g[0]), s[4], arg[0], arg[1], arg[2], arg[3]);
    out[0] = r[0], out[1] = r[1], out[2] = r[2];
    return out;
  }
};

// What attention() takes here: what ::forward takes, checked before a node of the graph exists
std::optional<Tensor> attention(const Tensor& q, const Tensor& k, const Tensor& v, int64_t causal, int64_t window, int64_t schedule, int64_t sinks) {
  // torch.jit.trace records a Python node as a call of it; of a native one it would record the allocations and miss the launches
  if (at::tracer::impl::is_dispatch_enabled()) return std::nullopt;
  // torch.func transforms: the Python nodes say that they have no rule for them
  if (c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode)) return std::nullopt;
  for (const Tensor* t : {&q, &k, &v}) {
    const int64_t dim = t->dim();
    if (t->unsafeGetTensorImpl()->is_python_dispatch() || !in_memory(*t)) return std::nullopt;
    if (!t->is_cuda() || t->device() != q.device() || t->scalar_type() != q.scalar_type() || (dim != 3 && dim != 4) || dim != q.dim()) return std::nullopt;
    for (int64_t i = 0; i < dim; i++)
      if (i != dim - 2 && t->size(i) != q.size(i)) return std::nullopt;
    const Layout l = layout_of(*t);
    if (l.rows && !l.direct) return std::nullopt;
  }
  const int64_t d = q.size(-1), n_q = q.size(-2), n_k = k.size(-2);
  if (dtype_code(q.scalar_type()) < 0 || (d != 32 && d != 64 && d != 128) || v.size(-2) != n_k || q.numel() == 0 || k.numel() == 0 ||
      q.numel() / d >= INT32_MAX || q.numel() / d / n_q > 65535 || n_q > (1 << 24) || n_k > (1 << 24) ||
      !mask_applies(Mask{(int32_t)causal, window, sinks}, n_q, n_k) || schedule < FHOG_SCHEDULE_FOUR_PASS || schedule > FHOG_SCHEDULE_THREE_SWEEP ||
      (sinks > 0 && schedule != FHOG_SCHEDULE_FUSED_STATS))
    return std::nullopt;
  return Attention::apply(q, k, v, causal, window, schedule, sinks);
}

// ---- rotary positions -----------------------------------------------------------------------------------------------
// What a call turns by, apart from the positions
struct Turn {
  double theta;
  int64_t rotary_dim;
  bool interleaved, inverse;
  std::vector<int64_t> sections;
};

// positions as (axes, batch, n) strides; false where they are no such thing for a (batch, .., n, d) tensor
bool positions_of(const Tensor& p, const Tensor& q, size_t axes, fhog_rotary_args& a) {
  switch (p.scalar_type()) {
    case at::kInt: a.position_type = FHOG_POSITIONS_INT32; break;
    case at::kLong: a.position_type = FHOG_POSITIONS_INT64; break;
    case at::kFloat: a.position_type = FHOG_POSITIONS_FP32; break;
    default: return false;
  }
  if (!p.is_cuda() || p.device() != q.device()) return false;
  const int64_t lead = axes > 1 ? 1 : 0, dim = p.dim();   // one axis has no dimension of its own
  if (dim != lead + 1 && dim != lead + 2) return false;
  if (lead && p.size(0) != (int64_t)axes) return false;
  if (p.size(dim - 1) != a.n || (dim == lead + 2 && p.size(lead) != a.batch && p.size(lead) != 1)) return false;
  a.stride_pa = lead ? p.stride(0) : 0;
  a.stride_pb = dim == lead + 2 && p.size(lead) != 1 ? p.stride(lead) : 0;
  a.stride_pn = p.stride(dim - 1);
  a.positions = p.data_ptr();
  return true;
}

// The arguments of a call, outputs packed; false where they are not well formed. (batch, N, d) tensors have one head. What is not known yet, the
// addresses of the outputs, is filled in with those of the inputs.
bool rotary_args(const Tensor& q, const Tensor& k, const Tensor& positions, const Turn& turn, fhog_rotary_args& a) {
  const int64_t dim = q.dim();
  if (!in_memory(q) || !in_memory(positions) || (k.defined() && !in_memory(k))) return false;
  if (!q.is_cuda() || (dim != 3 && dim != 4) || turn.sections.empty() || turn.sections.size() > FHOG_ROTARY_MAX_AXES) return false;
  if (k.defined() && (!k.is_cuda() || k.device() != q.device() || k.scalar_type() != q.scalar_type() || k.dim() != dim || k.size(0) != q.size(0) ||
                      k.size(-1) != q.size(-1) || k.size(-2) != q.size(-2)))
    return false;
  a = {};
  a.dtype = dtype_code(q.scalar_type());
  if (a.dtype < 0) return false;
  a.batch = q.size(0), a.n = q.size(-2), a.d = q.size(-1), a.rotary_dim = turn.rotary_dim;
  a.heads_q = dim == 4 ? q.size(1) : 1, a.heads_k = !k.defined() ? 0 : dim == 4 ? k.size(1) : 1;
  if (k.defined() && a.heads_k == 0) return false;
  a.theta = turn.theta, a.interleaved = turn.interleaved, a.inverse = turn.inverse, a.axes = (int32_t)turn.sections.size();
  for (size_t i = 0; i < turn.sections.size(); i++) {
    if (turn.sections[i] < 0 || turn.sections[i] > FHOG_ROTARY_MAX_D) return false;
    a.sections[i] = (int32_t)turn.sections[i];
  }
  if (!positions_of(positions, q, turn.sections.size(), a)) return false;
  const auto strides = [&](const Tensor& t, int64_t& b, int64_t& h, int64_t& n) { b = t.stride(0), h = dim == 4 ? t.stride(1) : 0, n = t.stride(dim - 2); };
  strides(q, a.stride_qb, a.stride_qh, a.stride_qn);
  a.q = q.data_ptr(), a.q_out = const_cast<void*>(a.q);
  a.stride_qon = a.d, a.stride_qoh = a.n * a.d, a.stride_qob = a.heads_q * a.stride_qoh;
  if (k.defined()) {
    strides(k, a.stride_kb, a.stride_kh, a.stride_kn);
    a.k = k.data_ptr(), a.k_out = const_cast<void*>(a.k);
    a.stride_kon = a.d, a.stride_koh = a.n * a.d, a.stride_kob = a.heads_k * a.stride_koh;
  }
  return fhog_rotary_validate(&a) == FHOG_OK;
}

// The turned q and, where k is defined, k, packed; nothing where the arguments are not well formed
std::optional<tensor_list> rotary_call(const Tensor& q_, const Tensor& k_, const Tensor& positions, const Turn& turn) {
  fhog_rotary_args a;
  if (!rotary_args(q_, k_, positions, turn, a)) return std::nullopt;
  const c10::DeviceGuard guard(q_.device());
  const auto rows = [](const Tensor& t) { return !t.defined() || t.stride(-1) == 1 ? t : t.contiguous(); };   // channels side by side
  const Tensor q = rows(q_), k = rows(k_);
  rotary_args(q, k, positions, turn, a);
  tensor_list out = {at::empty(q.sizes(), q.options())};
  a.q_out = out[0].data_ptr();
  if (k.defined()) out.push_back(at::empty(k.sizes(), k.options())), a.k_out = out[1].data_ptr();
  TORCH_CHECK(fhog_rotary(&a, stream_of(q)) == FHOG_OK, "fhog_rotary: ", fhog_last_error());
  return out;
}

// The rotation of one or two tensors as a node; its gradient is the rotation back, as a node again, so derivatives of every order exist
struct RotaryNode : torch::autograd::Function<RotaryNode> {
  static tensor_list forward(AutogradContext* ctx, const Tensor& q, const std::optional<Tensor>& k, const Tensor& positions, const Turn& turn) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({positions});
    ctx->saved_data["sections"] = turn.sections;
    ctx->saved_data["theta"] = turn.theta;
    ctx->saved_data["how"] = std::vector<int64_t>{turn.rotary_dim, turn.interleaved, turn.inverse};
    auto r = rotary_call(q, k ? *k : Tensor(), positions, turn);
    TORCH_CHECK(r, "fhog: rotary: ", fhog_last_error());
    return *r;
  }
  static tensor_list backward(AutogradContext* ctx, tensor_list g) {
    tensor_list out(4);
    const auto how = ctx->saved_data["how"].toIntVector();
    const Turn back{ctx->saved_data["theta"].toDouble(), how[0], how[1] != 0, how[2] == 0, ctx->saved_data["sections"].toIntVector()};
    const bool both = g.size() == 2 && g[0].defined() && g[1].defined();
    const size_t one = g[0].defined() ? 0 : 1;
    if (!both && (one >= g.size() || !g[one].defined())) return out;
    const Tensor positions = ctx->get_saved_variables()[0];
    const tensor_list r = both ? RotaryNode::apply(g[0], std::optional<Tensor>(g[1]), positions, back) : RotaryNode::apply(g[one], std::optional<Tensor>(), positions, back);
    if (both) out[0] = r[0], out[1] = r[1];
    else out[one] = r[0];
    return out;
  }
};

// What rotary() takes here: what rotary_call takes, checked before a node of the graph exists
std::optional<tensor_list> rotary(const Tensor& q, const std::optional<Tensor>& k, const Tensor& positions, std::vector<int64_t> sections, double theta,
                                  int64_t rotary_dim, bool interleaved) {
  if (at::tracer::impl::is_dispatch_enabled()) return std::nullopt;   // as in attention()
  if (c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode)) return std::nullopt;
  for (const Tensor* t : {&q, k ? &*k : &q, &positions})
    if (t->unsafeGetTensorImpl()->is_python_dispatch()) return std::nullopt;
  const Turn turn{theta, rotary_dim, interleaved, false, std::move(sections)};
  // Who asks for a derivative, backwards or forwards, gets the node, which refuses what it does not have: a tangent (dual tensors require no gradient)
  // and, by the caller, a gradient of the positions
  bool reverse = false, dual = false;
  for (const Tensor* t : {&q, k ? &*k : &q, &positions}) reverse = reverse || t->requires_grad(), dual = dual || t->_fw_grad(0).defined();
  reverse = reverse && at::GradMode::is_enabled();
  if (!reverse && !dual) {
    const at::NoGradGuard no_grad;
    return rotary_call(q, k ? *k : Tensor(), positions, turn);
  }
  fhog_rotary_args a;
  if ((reverse && positions.requires_grad()) || !rotary_args(q, k ? *k : Tensor(), positions, turn, a)) return std::nullopt;
  return RotaryNode::apply(q, k, positions, turn);
}

}  // namespace

PYBIND11_MODULE(_fhog_torch, m) {
  namespace py = pybind11;
  const auto free_lock = py::call_guard<py::gil_scoped_release>();
  m.def("forward", [](const Tensor& q, const Tensor& k, const Tensor& v, double scale, int causal, int64_t window, int64_t sinks) {
    const at::NoGradGuard no_grad;
    return forward(q, k, v, scale, Mask{causal, window, sinks});
  }, free_lock);
  m.def("backward", [](const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& o, const Tensor& g, const Tensor& L, double scale, int causal,
                       int64_t window, int64_t sinks) {
    const at::NoGradGuard no_grad;
    return backward(q, k, v, o, g, L, scale, Mask{causal, window, sinks}, true);
  }, free_lock);
  m.def("double_backward", [](const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& o, const Tensor& g, const Tensor& ddq, const Tensor& ddk,
                              const Tensor& ddv, const Tensor& L, double scale, int causal, int64_t window, int impl, int schedule, bool split, int64_t sinks) {
    const at::NoGradGuard no_grad;
    return double_backward(q, k, v, o, g, ddq, ddk, ddv, L, scale, Mask{causal, window, sinks}, impl, schedule, split);
  }, free_lock);
  m.def("in_memory", &in_memory, free_lock);
  m.def("dispatches_to_python", [](const Tensor& t) { return t.unsafeGetTensorImpl()->is_python_dispatch(); }, free_lock);
  m.def("attention", &attention, free_lock);
  m.def("rotary", &rotary, free_lock);
}
