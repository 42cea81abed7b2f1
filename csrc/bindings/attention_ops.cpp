// Rotary positions, normalised queries and keys, and attention over another sequence: argument rules, autograd functions and launches in one call, since a step
// of small tensors is bound by the host. Each entry returns nothing for a call that its kernels do not take; the caller then explains or falls back.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_runtime.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <cfloat>
#include <cmath>
#include <optional>
#include <vector>

#include "device_word.h"
#include "flodl_b200.h"

torch::Tensor& status_word(int device);       // ops.cpp

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;
using Found = std::optional<std::vector<Tensor>>;

void* stream_of(const Tensor& t) { return at::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

void check(int rc, const char* what) {
  if (rc == 0) return;
  if (rc > 0) TORCH_CHECK(false, what, ": CUDA error ", rc, " (", cudaGetErrorString(static_cast<cudaError_t>(rc)), ")");
  TORCH_CHECK(false, what, ": rejected arguments (code ", rc, ")");
}

bool records(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
// Whether a tensor is its memory and nothing else: no transform's wrapper, subclass, tangent or sign that a reader has to apply. The plain forms take the others.
bool plain_memory(const Tensor& t) {
  constexpr c10::DispatchKeySet wrapped({c10::DispatchKey::Python, c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper});
  return t.has_storage() && !t.key_set().has_any(wrapped) && !t.is_neg() && !t._fw_grad(/*level=*/0).defined();
}
// ... of all that are there; and no trace, which would keep a result of these functions as a constant.
bool plain_call(std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    if (t->defined() && !plain_memory(*t)) return false;
  return !torch::jit::tracer::isTracing();
}
void first_derivative_only() { TORCH_CHECK(!at::GradMode::is_enabled(), "the native kernels have no second derivative: use ops.set_native(False)"); }

Tensor value(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
OptTensor given(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }      // an autograd function takes no undefined tensors

// ------------------------------------------------------------------------------------------ positions
struct Turn {
  int64_t offset;
  bool interleaved;
  double amplitude;
  bool norm;
  double eps;
};

// Values of an access that the halves of the rotary part and what is behind it allow.
int64_t width(const Tensor& t, int64_t pairs) {
  int64_t v = 16 / t.element_size();
  while (v > 1 && (pairs % v || (t.size(-1) - 2 * pairs) % (2 * v))) v /= 2;
  return v;
}

// `t` as the kernel can address it: a unit inner stride; with the norm, whose rows have to fit a warp, accesses of the full width too.
Tensor rows_of(const Tensor& t, int64_t pairs, bool norm) {
  if (t.stride(-1) != 1 && t.size(-1) > 1) return t.contiguous();
  if (norm) {
    const int64_t v = width(t, pairs);
    bool whole = reinterpret_cast<uintptr_t>(t.data_ptr()) % (v * t.element_size()) == 0;
    for (int64_t d = 0; d + 1 < t.dim(); ++d) whole = whole && (t.size(d) <= 1 || t.stride(d) % v == 0);
    if (!whole) return t.clone(at::MemoryFormat::Contiguous);
  }
  return t;
}

// x: queries (or a packed projection) and keys; dy: their results' gradients, for the backward pass. The results in the layouts given, then dwq and dwk.
std::vector<Tensor> launch_turn(const Tensor x_in[2], const Tensor dy_in[2], const Tensor& freqs, const Tensor& positions, const Turn& c, const Tensor w[2], bool want_dw) {
  const bool backward = dy_in != nullptr;
  const int64_t pairs = freqs.numel();
  Tensor x[2], dy[2];
  for (int i = 0; i < 2; ++i) {
    if (x_in && x_in[i].defined()) x[i] = rows_of(x_in[i], pairs, c.norm);
    if (backward && dy_in[i].defined()) dy[i] = rows_of(dy_in[i], pairs, c.norm);
  }
  const Tensor* of = backward ? dy : x;
  const Tensor& lead = of[0];
  c10::cuda::CUDAGuard guard(lead.device());
  const bool packed = lead.dim() == 5;
  fb_rotary_args a = {};
  a.B = static_cast<int>(lead.size(0));
  a.S = static_cast<int>(lead.size(1));
  a.D = static_cast<int>(lead.size(-1));
  a.rot = static_cast<int>(pairs) * 2;
  const auto kind = lead.scalar_type();
  a.dtype = kind == at::kFloat ? FLODL_FLOAT32 : kind == at::kHalf ? FLODL_FLOAT16 : FLODL_BFLOAT16;
  a.interleaved = c.interleaved;
  a.norm = c.norm;
  a.backward = backward;
  a.amplitude = static_cast<float>(c.amplitude);
  a.eps = static_cast<float>(c.eps);
  a.freqs = freqs.data_ptr<double>();
  a.offset = c.offset;
  if (positions.defined()) {
    a.positions = reinterpret_cast<const long long*>(positions.data_ptr<int64_t>());
    a.pos_strides[0] = positions.stride(0);
    a.pos_strides[1] = positions.stride(1);
  }
  // one row of heads as the kernel addresses it (the stride of a dimension of one is never used, whatever it is)
  const auto slice = [&](const Tensor& t, int seg, const void** at, long long* strides) {
    const int64_t h = t.dim() - 2;
    TORCH_CHECK(t.sizes().slice(0, 2) == lead.sizes().slice(0, 2) && t.size(-1) == a.D && t.scalar_type() == kind && t.dim() == lead.dim());
    *at = static_cast<const char*>(t.data_ptr()) + (packed ? seg * t.stride(2) * t.element_size() : 0);
    strides[0] = t.size(0) == 1 ? 0 : t.stride(0);
    strides[1] = t.size(1) == 1 ? 0 : t.stride(1);
    strides[2] = t.size(h) == 1 ? 0 : t.stride(h);
    if (a.heads[seg] == 0) a.heads[seg] = static_cast<int>(t.size(h));
    TORCH_CHECK(a.heads[seg] == t.size(h), "heads differ");
  };
  std::vector<Tensor> out;
  out.reserve(4);
  for (int seg = 0; seg < (packed ? 3 : 2); ++seg) {
    const int i = packed ? 0 : seg;
    if (!of[i].defined()) continue;
    if (x[i].defined()) slice(x[i], seg, &a.x[seg], a.x_strides[seg]);
    if (backward) slice(dy[i], seg, &a.dy[seg], a.dy_strides[seg]);
    if (!packed || seg == 0) out.push_back(at::empty(of[i].sizes(), of[i].options().requires_grad(false)));
    const void* y = nullptr;
    slice(out.back(), seg, &y, a.y_strides[seg]);
    a.y[seg] = const_cast<void*>(y);
  }
  Tensor w32[2], partial;
  for (int i = 0; i < 2; ++i) {
    if (!w[i].defined()) continue;
    w32[i] = w[i].scalar_type() == at::kFloat && w[i].is_contiguous() ? w[i] : w[i].detach().to(at::kFloat).contiguous();
    a.weight[i] = w32[i].data_ptr<float>();
  }
  if (c.norm && backward) {
    const auto f32 = at::TensorOptions().dtype(at::kFloat).device(lead.device());
    partial = at::empty({fb_rotary_partial_rows(), 2, a.D}, f32);
    a.partial = partial.data_ptr<float>();
    if (want_dw) {
      for (int i = 0; i < 2; ++i) {
        out.push_back(lead.numel() == 0 ? at::zeros({a.D}, f32) : at::empty({a.D}, f32));
        a.dw[i] = out.back().data_ptr<float>();
      }
    }
  }
  check(fb_rotary(&a, stream_of(lead)), "fb_rotary");
  return out;
}

void keep(AutogradContext* ctx, const Turn& c) {       // one entry: each is a look-up by name
  ctx->saved_data["turn"] = std::vector<double>{static_cast<double>(c.offset), static_cast<double>(c.interleaved), c.amplitude, static_cast<double>(c.norm), c.eps};
}
Turn kept(AutogradContext* ctx) {
  const auto v = ctx->saved_data["turn"].toDoubleVector();
  return {static_cast<int64_t>(v[0]), v[1] != 0, v[2], v[3] != 0, v[4]};
}

struct TurnFn : public torch::autograd::Function<TurnFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const OptTensor& k_in, const OptTensor& wq_in, const OptTensor& wk_in, const Tensor& freqs,
                               const OptTensor& positions_in, Turn c) {
    const Tensor k = value(k_in), wq = value(wq_in), wk = value(wk_in), positions = value(positions_in);
    const Tensor x[2] = {q, k}, w[2] = {wq, wk};
    auto out = launch_turn(x, nullptr, freqs, positions, c, w, false);
    keep(ctx, c);
    if (c.norm) ctx->save_for_backward({freqs, positions, q, k, wq, wk});
    else ctx->save_for_backward({freqs, positions});
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list dys) {
    first_derivative_only();
    const Turn c = kept(ctx);
    const auto saved = ctx->get_saved_variables();
    variable_list grads(7);
    const bool pair = dys.size() > 1;
    bool want_w[2] = {false, false};
    for (int i = 0, at = pair ? 2 : 1; c.norm && i < 2; ++i)
      if (saved[4 + i].defined()) want_w[i] = ctx->needs_input_grad(at++);
    // of a pair, the one or both that anything is wanted of
    int of[2] = {0, 1}, n = 0;
    for (int i = 0; i < (pair ? 2 : 1); ++i)
      if (ctx->needs_input_grad(i) || want_w[i] || (!pair && want_w[1])) of[n++] = i;
    if (n == 0) return grads;
    Tensor dy[2], x[2], w[2];
    for (int i = 0; i < n; ++i) {
      dy[i] = dys[of[i]];
      if (c.norm) x[i] = saved[2 + of[i]];
    }
    if (c.norm)
      for (int i = 0; i < (pair ? n : 2); ++i) w[i] = saved[4 + (pair ? of[i] : i)];
    const bool want_dw = want_w[0] || want_w[1];
    auto out = launch_turn(c.norm ? x : nullptr, dy, saved[0], saved[1], c, w, want_dw);
    for (int i = 0; i < n; ++i) grads[of[i]] = out[i];
    for (int i = 0; want_dw && i < (pair ? n : 2); ++i) {
      const int j = pair ? of[i] : i;
      if (want_w[j]) grads[2 + j] = out[n + i].to(w[i].scalar_type());
    }
    return grads;
  }
};

// The rules of a call to `ops.rotary` (norm: `ops.qk_norm_rotary`), and the call.
Found turn(const Tensor& q, const OptTensor& k_in, const Tensor& freqs_in, const OptTensor& positions_in, int64_t offset, bool interleaved, double amplitude, bool norm,
           const OptTensor& wq_in, const OptTensor& wk_in, double eps) {
  const Tensor k = value(k_in), wq = value(wq_in), wk = value(wk_in);
  const bool packed = q.dim() == 5;
  const auto kind = q.scalar_type();
  if (!q.is_cuda() || (kind != at::kFloat && kind != at::kBFloat16 && kind != at::kHalf)) return std::nullopt;
  if (packed ? (q.size(2) != 3 || k.defined()) : q.dim() != 4) return std::nullopt;
  const int64_t B = q.size(0), S = q.size(1), D = q.size(-1);
  if (k.defined() && (k.dim() != 4 || k.size(0) != B || k.size(1) != S || k.size(3) != D || k.scalar_type() != kind || k.device() != q.device())) return std::nullopt;
  if (freqs_in.dim() != 1 || freqs_in.scalar_type() != at::kDouble || freqs_in.device() != q.device()) return std::nullopt;
  if (!plain_call({&q, &k, &freqs_in, &wq, &wk}) || records({&freqs_in})) return std::nullopt;       // the kernel knows no gradient of frequencies
  const int64_t pairs = freqs_in.numel();
  if (D < 2 || D % 2 || 2 * pairs > D || B >= 1 << 30 || S >= 1 << 30 || B * S >= 1ll << 31 || q.size(-2) < 1 || q.size(-2) >= 1 << 14) return std::nullopt;
  if (k.defined() && (k.size(2) < 1 || k.size(2) >= 1 << 14)) return std::nullopt;
  if (!std::isfinite(amplitude) || !std::isfinite(eps) || eps < 0) return std::nullopt;
  if (norm && (D > 64 * width(q, pairs) || D > 512)) return std::nullopt;
  if (D > 8192 || (q.size(-2) * (packed ? 3 : 1) + (k.defined() ? k.size(2) : 0)) * D > 1 << 24) return std::nullopt;       // of a tile's items and its angles
  Tensor positions;
  if (positions_in.has_value()) {
    positions = *positions_in;
    if (!c10::isIntegralType(positions.scalar_type(), false) || !plain_memory(positions) || positions.device() != q.device()) return std::nullopt;
    if ((positions.dim() != 1 && positions.dim() != 2) || positions.size(-1) != S || (positions.dim() == 2 && positions.size(0) != 1 && positions.size(0) != B)) return std::nullopt;
    if (positions.scalar_type() != at::kLong) positions = positions.to(at::kLong);
    positions = positions.expand({B, S});
  }
  for (const Tensor* w : {&wq, &wk})
    if (w->defined() && (w->dim() != 1 || w->size(0) != D || w->device() != q.device() || !w->is_floating_point())) return std::nullopt;
  if (wk.defined() && !packed && !k.defined()) return std::nullopt;
  if (offset > (1ll << 52) || offset < -(1ll << 52)) return std::nullopt;       // kept as a double
  const Turn c = {offset, interleaved, amplitude, norm, eps};
  const Tensor freqs = freqs_in.contiguous();
  if (records({&q, &k, &wq, &wk})) return TurnFn::apply(q, given(k), given(wq), given(wk), freqs, given(positions), c);
  const Tensor x[2] = {q, k}, w[2] = {wq, wk};
  return launch_turn(x, nullptr, freqs, positions, c, w, false);
}

// ------------------------------------------------------------------------- attention over another sequence
void strides_of(const Tensor& t, long long* s) {
  for (int d = 0; d < 3; ++d) s[d] = t.size(d) > 1 ? t.stride(d) : 8;
}
// `t` as a tensor map can address it: 16-byte rows, no stride of zero.
Tensor mapped(const Tensor& t) {
  bool ok = t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int d = 0; d < 3; ++d) ok = ok && (t.size(d) <= 1 || (t.stride(d) % 8 == 0 && t.stride(d) > 0));
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

fb_cross_args cross_args(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& mask, double scale) {
  fb_cross_args a = {};
  a.q = q.data_ptr();
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  strides_of(q, a.q_strides);
  strides_of(k, a.k_strides);
  strides_of(v, a.v_strides);
  a.B = static_cast<int>(q.size(0));
  a.Sq = static_cast<int>(q.size(1));
  a.H = static_cast<int>(q.size(2));
  a.D = static_cast<int>(q.size(3));
  a.Sk = static_cast<int>(k.size(1));
  a.Hk = static_cast<int>(k.size(2));
  if (mask.defined()) {
    a.mask = mask.data_ptr();
    a.mask_stride = mask.size(0) == 1 ? 0 : mask.stride(0);
    a.mask_bool = mask.scalar_type() == at::kBool;
  }
  a.scale = static_cast<float>(scale);
  a.status = status_word(q.get_device()).data_ptr<int>();
  return a;
}
Tensor space_for(fb_cross_args& a, bool backward, const Tensor& like) {
  const long long n = fb_cross_workspace(&a, backward);
  TORCH_CHECK(n >= 0, "fb_cross_workspace: rejected arguments");
  if (n == 0) return Tensor();
  Tensor t = at::empty({n}, at::TensorOptions().dtype(at::kFloat).device(like.device()));
  a.workspace = t.data_ptr<float>();
  return t;
}

Tensor launch_cross(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, const Tensor& mask, double scale, Tensor* stats, Tensor* info) {
  const Tensor q = mapped(q_in), k = mapped(k_in), v = mapped(v_in);
  c10::cuda::CUDAGuard guard(q.device());
  Tensor o = at::empty(q.sizes(), at::TensorOptions().dtype(at::kBFloat16).device(q.device()));
  fb_cross_args a = cross_args(q, k, v, mask, scale);
  a.o = o.data_ptr();
  strides_of(o, a.o_strides);
  if (stats) {
    *stats = at::empty({q.size(0) * q.size(2) * q.size(1)}, at::TensorOptions().dtype(at::kFloat).device(q.device()));
    a.stats = stats->data_ptr<float>();
  }
  if (mask.defined()) {
    const long long n = fb_cross_mask_info(&a);
    TORCH_CHECK(n > 0, "fb_cross_mask_info: rejected arguments");
    *info = at::empty({n}, at::TensorOptions().dtype(at::kInt).device(q.device()));
    a.mask_info = info->data_ptr<int>();
  }
  const Tensor space = space_for(a, false, q);
  check(fb_cross_attn_fwd(&a, stream_of(q)), "fb_cross_attn_fwd");
  return o;
}

// The gradients by way of the plain form, for those that are differentiated again or are more than memory themselves (a batch of them).
variable_list plain_gradients(const Tensor (&given)[3], const Tensor& mask, const Tensor& d_o, double scale) {
  const bool again = at::GradMode::is_enabled();
  at::AutoGradMode record(true);
  Tensor x[3], o;        // each by a name of its own: one tensor may be queries, keys and values
  for (int i = 0; i < 3; ++i) x[i] = given[i].view_as(given[i]);
  {
    py::gil_scoped_acquire gil;
    o = py::module_::import("flodl_b200.ops.cross").attr("_plain")(x[0], x[1], x[2], mask.defined() ? py::cast(mask) : py::none(), scale).cast<Tensor>();
  }
  variable_list of, out(6);
  for (const Tensor& t : x)
    if (t.requires_grad()) of.push_back(t);
  const auto grads = torch::autograd::grad({o}, of, {d_o}, /*retain_graph=*/again, /*create_graph=*/again);
  for (size_t i = 0, at = 0; i < 3; ++i)
    if (x[i].requires_grad()) out[i] = grads[at++];
  return out;
}

struct CrossFn : public torch::autograd::Function<CrossFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& mask_in, double scale, bool twice) {
    const Tensor mask = value(mask_in);
    Tensor stats, info, o = launch_cross(q, k, v, mask, scale, &stats, &info);
    ctx->save_for_backward({q, k, v, mask, o, stats, info});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["twice"] = twice;
    return o;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!ctx->saved_data["twice"].toBool()) first_derivative_only();
    const auto saved = ctx->get_saved_variables();
    if (at::GradMode::is_enabled() || !plain_memory(grads[0]))
      return plain_gradients({saved[0], saved[1], saved[2]}, saved[3], grads[0], ctx->saved_data["scale"].toDouble());
    const Tensor q = mapped(saved[0]), k = mapped(saved[1]), v = mapped(saved[2]), d_o = mapped(grads[0]);
    const Tensor &mask = saved[3], &o = saved[4], &stats = saved[5];
    c10::cuda::CUDAGuard guard(q.device());
    const auto bf16 = at::TensorOptions().dtype(at::kBFloat16).device(q.device());
    const bool for_k = ctx->needs_input_grad(1), for_v = ctx->needs_input_grad(2);
    Tensor dq, dk, dv;
    if (ctx->needs_input_grad(0)) dq = at::empty(q.sizes(), bf16);
    if (for_k || for_v) dk = at::empty(k.sizes(), bf16), dv = at::empty(v.sizes(), bf16);       // one pass gives both
    if (!dq.defined() && !dk.defined()) return variable_list(6);
    fb_cross_args a = cross_args(q, k, v, mask, ctx->saved_data["scale"].toDouble());
    a.o = o.data_ptr();
    strides_of(o, a.o_strides);
    a.d_o = d_o.data_ptr();
    strides_of(d_o, a.do_strides);
    if (dq.defined()) {
      a.dq = dq.data_ptr();
      strides_of(dq, a.dq_strides);
    }
    if (dk.defined()) {
      a.dk = dk.data_ptr();
      a.dv = dv.data_ptr();
      strides_of(dk, a.dk_strides);
    }
    a.stats = stats.data_ptr<float>();
    if (mask.defined()) a.mask_info = saved[6].data_ptr<int>();
    const Tensor space = space_for(a, true, q);
    check(fb_cross_attn_bwd(&a, stream_of(q)), "fb_cross_attn_bwd");
    return {dq, for_k ? dk : Tensor(), for_v ? dv : Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

// A 64-bit mask for the kernel, relative to each row's largest before it is rounded to 32 bits; finite values stay finite. A largest beyond 2^100 leaves nothing of the scores, nor of keys
// that are any further away: it is told from the others by one that is as large in 32 bits.
Tensor narrowed(const Tensor& mask) {
  const Tensor top = mask.amax(-1, true), rest = mask - top.masked_fill(top.isinf(), 0.0);
  const Tensor far = at::where(rest == 0, top.clamp(-0x1p101, 0x1p101), -FLT_MAX);
  return at::where(mask.isinf(), mask, at::where(top.abs() >= 0x1p100, far, rest.clamp(-FLT_MAX, FLT_MAX)));
}

// The rules of a call to `ops.cross_attention`, and the call; with `twice` its gradients can be differentiated again. `mask`: bool or floating point [B or 1, Sk], or with two dimensions of one between.
std::optional<Tensor> cross_attention(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& mask_in, double scale, bool twice) {
  if (!q.is_cuda() || q.dim() != 4 || k.dim() != 4 || v.dim() != 4) return std::nullopt;
  for (const Tensor* t : {&q, &k, &v})
    if (t->scalar_type() != at::kBFloat16 || t->device() != q.device()) return std::nullopt;
  const int64_t B = q.size(0), D = q.size(3), H = q.size(2), Hk = k.size(2), Sk = k.size(1);
  if ((D != 64 && D != 128) || k.sizes() != v.sizes() || k.size(0) != B || k.size(3) != D || !std::isfinite(scale)) return std::nullopt;
  if (B < 1 || H < 1 || Hk < 1 || H % Hk || q.size(1) < 1 || Sk < 1 || q.size(1) > 1 << 26 || Sk > 1 << 28 || B > 1 << 20 || H > 1 << 16) return std::nullopt;
  Tensor mask;
  if (!plain_call({&q, &k, &v})) return std::nullopt;
  if (mask_in.has_value()) {
    mask = *mask_in;
    if (!plain_memory(mask)) return std::nullopt;
    if (mask.requires_grad() && at::GradMode::is_enabled()) return std::nullopt;
    if (mask.device() != q.device() || (mask.scalar_type() != at::kBool && !mask.is_floating_point())) return std::nullopt;
    if (mask.dim() == 4 && mask.size(1) == 1 && mask.size(2) == 1) mask = mask.select(1, 0).select(1, 0);
    if (mask.dim() != 2 || mask.size(1) != Sk || (mask.size(0) != 1 && mask.size(0) != B)) return std::nullopt;
    if (mask.scalar_type() == at::kDouble) mask = narrowed(mask);
    if (mask.scalar_type() != at::kBool) mask = mask.to(at::kFloat);
    if (Sk > 1 && mask.stride(1) != 1) mask = mask.contiguous();
  }
  if (records({&q, &k, &v})) return CrossFn::apply(q, k, v, given(mask), scale, twice);
  Tensor info;
  return launch_cross(q, k, v, mask, scale, nullptr, &info);
}

}  // namespace

void bind_attention_ops(py::module_& m) {
  m.def("turn", &turn);
  m.def("cross_attention", &cross_attention);
}
