// ggd_blocks.cpp -- the decoder-block operators' calls from Python (the _blocks module of blocks.py): argument checks, outputs and
// workspaces from torch's allocator, and their nodes in torch's autograd graph, around the C entries of include/ggd_train.h.
//
// In C++ because a small call's time is the host's: with ctypes and torch.autograd.Function a training pass of cross attention
// over 64 clips of 40 frames took 143 us of which its kernels are 34.  The entries come as addresses from native.py, so that
// they are those of the library it loaded.
#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPCachingAllocator.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstring>
#include <optional>
#include <sstream>
#include <string>

#include "../../include/ggd_train.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

struct Entries {
  decltype(&ggd_tr_battn_fwd) battn_fwd;
  decltype(&ggd_tr_battn_bwd) battn_bwd;
  decltype(&ggd_tr_battn_ws) battn_ws;
  decltype(&ggd_tr_resnorm_fwd) resnorm_fwd;
  decltype(&ggd_tr_resnorm_bwd) resnorm_bwd;
  decltype(&ggd_tr_resnorm_ws) resnorm_ws;
  decltype(&ggd_tr_gate_sum) gate_sum;
  decltype(&ggd_tr_gate_sum_ws) gate_sum_ws;
} entries;

// ValueError of what does not hold
template <typename... A>
[[noreturn]] void refuse(const char* what, const A&... parts) {
  std::ostringstream s;
  s << what << ": ";
  (s << ... << parts);
  throw py::value_error(s.str());
}

void check_status(int rc, const char* what) {
  if (rc == -2) refuse(what, "unsupported shape");
  TORCH_CHECK(rc == 0, what, " failed (ggd_train status ", rc, ")");
}

int dtype_of(const Tensor& t) { return t.scalar_type() == at::kFloat ? GGD_TR_F32 : t.scalar_type() == at::kBFloat16 ? GGD_TR_BF16 : -1; }

void on_gpu(const char* what, const Tensor& first) {
  if (!first.is_cuda()) refuse(what, "the inputs have to be on a GPU device (no CPU fallback)");
  if (first.layout() != at::kStrided) refuse(what, "the inputs have to be dense tensors");
}
void beside(const char* what, const char* name, const OptTensor& t, const Tensor& first) {
  if (t && t->device() != first.device()) refuse(what, name, " has to be on ", first.device().str());
  if (t && t->layout() != at::kStrided) refuse(what, name, " has to be a dense tensor");
}

template <typename T = void>
T* at_of(const Tensor& t) { return t.defined() ? (T*)t.data_ptr() : nullptr; }
Tensor or_none(const OptTensor& t) { return t ? *t : Tensor(); }
OptTensor given(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }

// the workspace of one call, which the allocator hands on in stream order
Tensor workspace(int64_t bytes, const Tensor& like) { return bytes ? at::empty({bytes}, like.options().dtype(at::kByte)) : Tensor(); }

void* stream_of(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

// In a captured call: a leaf whose gradient accumulator another stream made -- an eager graph of it is alive -- would draw that stream
// into the capture when its gradient arrives, past any error that could be caught.
void check_capture(const char* what, std::initializer_list<Tensor> inputs) {
  for (const Tensor& t : inputs) {
    if (!t.defined() || !t.requires_grad()) continue;
    const at::TensorBase& leaf = t.is_view() ? t._base() : t;
    if (!leaf.requires_grad() || !leaf.is_leaf()) continue;
    const auto accumulator = torch::autograd::impl::try_get_grad_accumulator(leaf);
    if (!accumulator) continue;
    const auto made = accumulator->stream();
    const auto stream = c10::hip::getCurrentHIPStream(t.device().index());
    if (!made || made->id() == stream.id()) continue;
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(stream.stream(), &status) == hipSuccess && status == hipStreamCaptureStatusActive)
      refuse(what, "captured while an eager graph of an input is alive; let go of that graph's outputs first");
  }
}

// Calls that would be answered wrongly without an error.  A tracer sees the allocation of an output and not the kernels that fill it, and a
// tensor that only stands for another has no memory to give them; and the kernels know no tangents, neither of inputs nor (in a backward
// pass) of incoming gradients.
const Tensor* there(const Tensor& t) { return t.defined() ? &t : nullptr; }
const Tensor* there(const OptTensor& t) { return t && t->defined() ? &*t : nullptr; }
template <typename... T>
void check_plain(const char* what, const T&... inputs) {
  using Modes = c10::impl::TorchDispatchModeTLS;
  using Key = c10::impl::TorchDispatchModeKey;
  bool traced = torch::jit::tracer::isTracing() || c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch) ||
                (Modes::stack_len() && (Modes::get_mode(Key::PROXY) || Modes::get_mode(Key::FAKE) || Modes::get_mode(Key::FUNCTIONAL)));
  const bool forward_mode = c10::AutogradState::get_tls_state().get_fw_grad_mode();
  bool tangent = false;
  auto look = [&](const Tensor* t) {
    if (!t) return;
    traced = traced || t->unsafeGetTensorImpl()->is_python_dispatch();
    tangent = tangent || (forward_mode && t->_fw_grad(0).defined());
  };
  (look(there(inputs)), ...);
  TORCH_CHECK_NOT_IMPLEMENTED(!traced, what, " cannot be traced, nor called with fake tensors");
  TORCH_CHECK_NOT_IMPLEMENTED(!tangent, what, " has no forward-mode derivative");
}

// (n, L, W) with contiguous rows: the tensor where its rows are, whatever their strides, else a copy (as of one whose values are negated
// when they are read, by torch's operations alone)
Tensor plain(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }
Tensor rows(const Tensor& t) { return t.dim() == 0 || t.stride(-1) == 1 || t.size(-1) == 1 ? plain(t) : t.contiguous(); }

// Saved tensors may come back through hooks that move them about.  The kernels read them by the types and sizes they had: a tensor of
// another one, or on another device, is an error, and one laid out anew is read where it is now.
// (The forms -- type and contiguity, then the sizes -- as bytes: a list's elements would be boxed one by one.)
void save(AutogradContext* ctx, const variable_list& tensors) {
  std::string forms;
  forms.reserve(512);
  auto add = [&](int64_t x) { forms.append((const char*)&x, sizeof(x)); };
  for (const Tensor& t : tensors) {
    add(t.defined() ? (int64_t)t.scalar_type() * 2 + t.is_contiguous() : -1);
    if (t.defined()) forms.append((const char*)t.sizes().data(), t.dim() * sizeof(int64_t));
  }
  ctx->saved_data["forms"] = std::move(forms);
  ctx->save_for_backward(tensors);
}
variable_list saved_by(AutogradContext* ctx, const char* what, const Tensor& like) {
  variable_list tensors = ctx->get_saved_variables();
  const std::string& forms = ctx->saved_data["forms"].toStringRef();
  const char* at = forms.data();
  for (Tensor& t : tensors) {
    int64_t form;
    std::memcpy(&form, at, sizeof(form));
    at += sizeof(form);
    bool same = t.defined() == (form >= 0);
    if (same && t.defined()) {
      const size_t bytes = t.dim() * sizeof(int64_t);
      same = t.device() == like.device() && t.layout() == at::kStrided && (int64_t)t.scalar_type() == form / 2 &&
             at + bytes <= forms.data() + forms.size() && std::memcmp(at, t.sizes().data(), bytes) == 0;
      at += bytes;
    }
    TORCH_CHECK(same, what, " backward: a saved tensor came back on another device or of another type or shape");
    if (t.defined() && !t.is_contiguous()) t = form & 1 ? t.contiguous() : rows(t);
  }
  return tensors;
}

// Gradients come once: where a graph of them is asked for, one that raises when it is used.
variable_list once(variable_list grads, const char* what) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list real;
  for (Tensor& g : grads)
    if (g.defined()) real.push_back(g.detach().requires_grad_());
  auto error = std::make_shared<torch::autograd::DelayedError>(std::string(what) + " has no second derivative", (int64_t)real.size());
  real = (*error)(std::move(real));
  size_t at = 0;
  for (Tensor& g : grads)
    if (g.defined()) g = real[at++];
  return grads;
}

// ------------------------------------------------------------------------------------------
// attention
// ------------------------------------------------------------------------------------------
struct Inputs {
  Tensor q, k, v, table, mask, q_mask, buckets;
  int64_t heads, kv_heads, offset;
  double scale;
};

ggd_tr_battn_args args_of(const Inputs& in) {
  ggd_tr_battn_args a{};
  const int64_t lq = in.q.size(1), width = in.q.size(2);
  a.n = (int32_t)in.q.size(0), a.heads = (int32_t)in.heads, a.kv_heads = (int32_t)in.kv_heads, a.lq = (int32_t)lq, a.lk = (int32_t)in.k.size(1);
  a.dk = (int32_t)(width / in.heads), a.dtype = dtype_of(in.q), a.scale = (float)in.scale;
  a.q = in.q.data_ptr(), a.k = in.k.data_ptr(), a.v = in.v.data_ptr();
  a.ldq = in.q.stride(1), a.bq = in.q.stride(0), a.ldk = in.k.stride(1), a.bk = in.k.stride(0), a.ldv = in.v.stride(1), a.bv = in.v.stride(0);
  a.ldo = width, a.bo = lq * width;
  if (in.mask.defined()) a.mask = at_of<const uint8_t>(in.mask), a.bmask = in.mask.stride(0);
  if (in.q_mask.defined()) a.q_mask = at_of<const uint8_t>(in.q_mask), a.bq_mask = in.q_mask.stride(0);
  if (in.table.defined()) {
    a.table = at_of<const float>(in.table), a.buckets = at_of<const int32_t>(in.buckets);
    a.n_buckets = (int32_t)in.table.size(0), a.distance = (int32_t)(in.buckets.size(0) / 2), a.offset = in.offset;
  }
  return a;
}

// o; with keep also what the backward pass needs (undefined where there is no query or no key: o is zeros then)
Tensor attend(const Inputs& in, bool keep, Tensor& stat, Tensor& o32) {
  Tensor o = at::empty({in.q.size(0), in.q.size(1), in.q.size(2)}, in.q.options());
  if (o.numel() == 0 || in.k.size(1) == 0) return o.zero_();
  const c10::DeviceGuard guard(in.q.device());
  ggd_tr_battn_args a = args_of(in);
  a.o = o.data_ptr();
  if (keep) {
    const auto f32 = in.q.options().dtype(at::kFloat);
    stat = at::empty({in.q.size(0), in.heads, in.q.size(1), 2}, f32);
    o32 = a.dtype == GGD_TR_F32 ? o : at::empty(o.sizes(), f32);
    a.stat = at_of<float>(stat), a.o32 = at_of<float>(o32);
  }
  a.ws_bytes = entries.battn_ws(&a, 0);
  const Tensor ws = workspace(a.ws_bytes, in.q);
  a.ws = at_of(ws);
  check_status(entries.battn_fwd(&a, stream_of(in.q)), "attention");
  return o;
}

struct Attention : torch::autograd::Function<Attention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& table, const OptTensor& mask,
                        const OptTensor& q_mask, const OptTensor& buckets, int64_t heads, int64_t kv_heads, double scale, int64_t offset) {
    Tensor stat, o32;
    const Inputs in{q, k, v, or_none(table), or_none(mask), or_none(q_mask), or_none(buckets), heads, kv_heads, offset, scale};
    Tensor o = attend(in, true, stat, o32);
    save(ctx, {q, k, v, in.table, in.mask, in.q_mask, in.buckets, stat, o32});
    ctx->saved_data["heads"] = heads, ctx->saved_data["kv_heads"] = kv_heads, ctx->saved_data["scale"] = scale, ctx->saved_data["offset"] = offset;
    return o;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_plain("attention backward", grads[0]);
    const variable_list saved = saved_by(ctx, "attention", grads[0]);
    const Inputs in{saved[0], saved[1], saved[2], saved[3], saved[4], saved[5], saved[6], ctx->saved_data["heads"].toInt(),
                    ctx->saved_data["kv_heads"].toInt(), ctx->saved_data["offset"].toInt(), ctx->saved_data["scale"].toDouble()};
    variable_list out(11);
    {
      const at::NoGradGuard no_grad;
      const Tensor &stat = saved[7], &o32 = saved[8];
      // dq's kernel also forms delta; dk and dv have one of their own, which a frozen memory does not need
      const bool memory = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);
      for (int i = 0; i < (memory ? 3 : 1); ++i) out[i] = at::empty(saved[i].sizes(), saved[i].options());
      if (in.table.defined() && ctx->needs_input_grad(3)) out[3] = at::empty(in.table.sizes(), in.table.options());
      if (!stat.defined()) {
        for (Tensor& t : out)
          if (t.defined()) t.zero_();
      } else {
        const c10::DeviceGuard guard(in.q.device());
        const Tensor dout = grads[0].contiguous();
        ggd_tr_battn_args a = args_of(in);
        a.stat = at_of<float>(stat), a.o32 = at_of<float>(o32), a.dout = dout.data_ptr();
        a.dq = out[0].data_ptr(), a.dk_out = at_of(out[1]), a.dv = at_of(out[2]), a.dtable = at_of<float>(out[3]);
        a.ws_bytes = entries.battn_ws(&a, 1);
        const Tensor ws = workspace(a.ws_bytes, in.q);
        a.ws = at_of(ws);
        const int rc = entries.battn_bwd(&a, stream_of(in.q));
        TORCH_CHECK(rc == 0, "attention backward failed (ggd_train status ", rc, ")");
      }
    }
    return once(std::move(out), "attention");
  }
};

Tensor mask_rows(const char* what, const char* name, const OptTensor& m, int64_t n, int64_t length) {
  if (!m) return Tensor();
  if (m->scalar_type() != at::kBool || m->dim() != 2 || m->size(0) != n || m->size(1) != length)
    refuse(what, name, " has to be (", n, ", ", length, ") truth values");
  return rows(*m);
}

Tensor attention(const char* what, const Tensor& q, const Tensor& k, const Tensor& v, int64_t heads, std::optional<int64_t> kv, std::optional<double> sc,
                 const OptTensor& mask, const OptTensor& q_mask, const OptTensor& buckets, const OptTensor& table, int64_t offset) {
  check_plain(what, q, k, v, mask, q_mask, table);
  on_gpu(what, q);
  beside(what, "k", k, q), beside(what, "v", v, q), beside(what, "mask", mask, q), beside(what, "q_mask", q_mask, q), beside(what, "table", table, q);
  beside(what, "the plan", buckets, q);
  const int64_t kv_heads = kv.value_or(heads);
  if (heads < 1 || kv_heads < 1 || heads % kv_heads) refuse(what, heads, " heads over ", kv_heads, " kv heads");
  if (q.dim() != 3 || k.dim() != 3 || v.dim() != 3) refuse(what, "q, k and v have to be (n, L, heads dk)");
  const int64_t n = q.size(0), width = q.size(2), dk = width / heads;
  if (width % heads || dk < 1 || dk > 128) refuse(what, "q rows of ", width, " elements are not ", heads, " heads of 1 to 128");
  if (k.size(0) != n || k.size(2) != kv_heads * dk || v.sizes() != k.sizes())
    refuse(what, "k ", k.sizes(), " and v ", v.sizes(), " have to be (", n, ", Lk, ", kv_heads * dk, ")");
  if (dtype_of(q) < 0 || k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type())
    refuse(what, "q, k and v have to be of one type, float32 or bfloat16");
  if (q.size(1) > 1 << 28 || k.size(1) > 1 << 28 || n > INT32_MAX || heads > INT32_MAX) refuse(what, "unsupported shape");
  const double scale = sc.value_or(1.0 / std::sqrt((double)dk));
  if (!((float)scale > 0.f && scale <= 1e30)) refuse(what, "scale ", scale, " has to be positive");
  Inputs in{rows(q), rows(k), rows(v), Tensor(), mask_rows(what, "mask", mask, n, k.size(1)), mask_rows(what, "q_mask", q_mask, n, q.size(1)),
            or_none(buckets), heads, kv_heads, offset, scale};
  if (table) in.table = plain(*table).contiguous();
  // (the plan's own memory, which no caller sees: let go while this stream works on it, it must not be handed on)
  if (buckets) c10::hip::HIPCachingAllocator::recordStream(buckets->storage().data_ptr(), c10::hip::getCurrentHIPStream(q.device().index()));
  const bool grad = at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad() || (table && table->requires_grad()));
  if (grad) check_capture(what, {q, k, v, or_none(table)});
  if (grad) return Attention::apply(in.q, in.k, in.v, given(in.table), given(in.mask), given(in.q_mask), given(in.buckets), heads, kv_heads, scale, offset);
  Tensor stat, o32;
  return attend(in, false, stat, o32);
}

// ------------------------------------------------------------------------------------------
// the norms around a block
// ------------------------------------------------------------------------------------------
struct Shape {
  int64_t rows, d, gate_rows, kind;
  double scale, eps;
  bool expanded;   // the gate is read expanded to h's shape
};

// the gate as the kernels read it
Tensor whole_gate(const Tensor& gate, const Tensor& h, bool expanded) { return expanded ? gate.expand(h.sizes()).contiguous() : gate; }

// an expanded gate's gradient, of h's shape in f32, -> that of the gate
void sum_gate(const Tensor& whole, const Tensor& gate, Tensor& out) {
  const int64_t dims = whole.dim(), less = dims - gate.dim();
  c10::SmallVector<uint8_t, 8> kept;
  for (int64_t i = 0; i < dims; ++i) kept.push_back(i >= less && gate.size(i - less) == whole.size(i));
  const int64_t bytes = entries.gate_sum_ws((int)dims, whole.sizes().data(), kept.data());
  const Tensor ws = workspace(bytes, whole);
  const int rc = entries.gate_sum((int)dims, whole.sizes().data(), kept.data(), at_of<const float>(whole), dtype_of(out), at_of(out), at_of(ws), bytes,
                                  stream_of(whole));
  TORCH_CHECK(rc == 0, "residual_norm backward failed (ggd_train status ", rc, ")");
}

variable_list norm_forward(const Tensor& h, const Tensor& y, const Tensor& gate, const variable_list& w, const Shape& g, bool keep, Tensor& stats) {
  Tensor h_out = at::empty_like(h), u = at::empty_like(h);
  if (g.rows) {
    const c10::DeviceGuard guard(h.device());
    if (keep) stats = at::empty({4, g.rows}, h.options().dtype(at::kFloat));
    check_status(entries.resnorm_fwd(g.rows, (int)g.d, dtype_of(h), (int)g.kind, (float)g.scale, (float)g.eps, at_of(h), at_of(y), at_of(gate), g.gate_rows,
                                     at_of<float>(w[0]), at_of<float>(w[1]), at_of<float>(w[2]), at_of<float>(w[3]), at_of(h_out), at_of(u),
                                     at_of<float>(stats), stream_of(h)),
                 "residual_norm");
  }
  return {h_out, u};
}

struct ResidualNorm : torch::autograd::Function<ResidualNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& h, const Tensor& y, const OptTensor& gate, const OptTensor& post_g,
                               const OptTensor& post_b, const OptTensor& pre_g, const OptTensor& pre_b, int64_t rows, int64_t d, int64_t gate_rows, int64_t kind, double scale, double eps,
                               bool expanded) {
    Tensor stats;
    const variable_list w{or_none(post_g), or_none(post_b), or_none(pre_g), or_none(pre_b)};
    const Tensor whole = whole_gate(or_none(gate), h, expanded);
    variable_list out = norm_forward(h, y, whole, w, {rows, d, gate_rows, kind, scale, eps, expanded}, true, stats);
    save(ctx, {h, y, or_none(gate), w[0], w[1], w[2], w[3], stats, expanded ? whole : Tensor()});
    ctx->saved_data["rows"] = rows, ctx->saved_data["d"] = d, ctx->saved_data["gate_rows"] = gate_rows, ctx->saved_data["kind"] = kind;
    ctx->saved_data["scale"] = scale, ctx->saved_data["eps"] = eps;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_plain("residual_norm backward", grads[0], grads[1]);
    const variable_list saved = saved_by(ctx, "residual_norm", grads[0]);
    auto whole = [&](const char* name) { return ctx->saved_data[name].toInt(); };
    const int64_t rows = whole("rows"), d = whole("d"), gate_rows = whole("gate_rows"), kind = whole("kind");
    const float scale = (float)ctx->saved_data["scale"].toDouble(), eps = (float)ctx->saved_data["eps"].toDouble();
    variable_list out(14);
    {
      const at::NoGradGuard no_grad;
      const bool expanded = saved[8].defined(), sum = expanded && ctx->needs_input_grad(2);
      const Tensor &h = saved[0], &y = saved[1], &gate = expanded ? saved[8] : saved[2], &stats = saved[7];
      for (int i = 0; i < 7; ++i)
        if (saved[i].defined()) out[i] = at::empty(saved[i].sizes(), saved[i].options());
      if (rows == 0) {
        for (Tensor& t : out)
          if (t.defined()) t.zero_();
      } else {
        const c10::DeviceGuard guard(h.device());
        const Tensor dh_out = grads[0].contiguous(), du = grads[1].contiguous();
        const int64_t bytes = entries.resnorm_ws(rows, (int)d, gate_rows, gate.defined());
        const Tensor ws = workspace(bytes, h);
        const Tensor dgate = expanded ? at::empty(h.sizes(), sum ? h.options().dtype(at::kFloat) : h.options()) : out[2];
        const int rc = entries.resnorm_bwd(rows, (int)d, dtype_of(h), (int)kind | (sum ? GGD_TR_GATE_F32 : 0), scale, eps, at_of(h), at_of(y), at_of(gate), gate_rows, at_of<float>(saved[3]),
                                           at_of<float>(saved[4]), at_of<float>(saved[5]), at_of<float>(saved[6]), at_of<float>(stats), at_of(dh_out),
                                           at_of(du), at_of(out[0]), at_of(out[1]), at_of(dgate), at_of<float>(out[3]), at_of<float>(out[4]),
                                           at_of<float>(out[5]), at_of<float>(out[6]), at_of(ws), bytes, stream_of(h));
        TORCH_CHECK(rc == 0, "residual_norm backward failed (ggd_train status ", rc, ")");
        if (sum) sum_gate(dgate, saved[2], out[2]);
        else if (expanded) out[2] = Tensor();
      }
    }
    return once(std::move(out), "residual_norm");
  }
};

// Rows of h that share a row of the gate, which is read as it is: leading dimensions of h, then ones, then d.  Any other shape
// that broadcasts is read expanded (0).
int64_t gate_rows_of(const char* what, Tensor& gate, const Tensor& h) {
  const int64_t dims = h.dim(), less = dims - gate.dim();
  bool fits = gate.dim() >= 1 && less >= 0;
  for (int64_t i = 0; fits && i < gate.dim(); ++i) fits = gate.size(i) == 1 || gate.size(i) == h.size(i + less);
  if (!fits) refuse(what, "gate ", gate.sizes(), " does not broadcast to ", h.sizes());
  auto size = [&](int64_t i) { return i < less ? 1 : gate.size(i - less); };
  int64_t ones = dims - 1, shared = 1;
  while (ones > 0 && size(ones - 1) == 1) --ones;
  bool direct = size(dims - 1) == h.size(dims - 1);
  for (int64_t i = 0; i < ones; ++i) direct = direct && size(i) == h.size(i);
  if (!direct) return 0;
  for (int64_t i = ones; i < dims - 1; ++i) shared *= h.size(i);
  gate = gate.contiguous();
  return std::max<int64_t>(1, shared);
}

std::pair<Tensor, Tensor> residual_norm(Tensor h, Tensor y, const OptTensor& pre_g, const OptTensor& pre_b, const OptTensor& post_g, const OptTensor& post_b,
                                        const OptTensor& gate_in, double scale, int64_t kind, double eps) {
  const char* what = "residual_norm";
  check_plain(what, h, y, gate_in, pre_g, pre_b, post_g, post_b);
  on_gpu(what, h);
  if (!pre_g || (!post_g && post_b)) refuse(what, "a norm needs a weight");
  beside(what, "y", y, h), beside(what, "gate", gate_in, h);
  if (h.dim() < 1 || h.sizes() != y.sizes()) refuse(what, "h ", h.sizes(), " and y ", y.sizes(), " have to be of one shape");
  if (dtype_of(h) < 0 || y.scalar_type() != h.scalar_type() || (gate_in && gate_in->scalar_type() != h.scalar_type()))
    refuse(what, "h, y and gate have to be of one type, float32 or bfloat16");
  const int64_t d = h.size(-1);
  if (d < 1 || d > 8192) refuse(what, "rows of ", d, " elements: 1 to 8192");
  variable_list w{or_none(post_g), or_none(post_b), or_none(pre_g), or_none(pre_b)};
  bool grad = h.requires_grad() || y.requires_grad() || (gate_in && gate_in->requires_grad());
  if (at::GradMode::is_enabled()) check_capture(what, {h, y, or_none(gate_in), w[0], w[1], w[2], w[3]});
  for (Tensor& t : w)
    if (t.defined()) {
      beside(what, "a weight or bias", t, h);
      if (t.scalar_type() != at::kFloat || t.dim() != 1 || t.size(0) != d) refuse(what, "weights and biases have to be (", d, ",) in float32");
      grad = grad || t.requires_grad();
      t = plain(t).contiguous();
    }
  if (!std::isfinite((float)scale) || !std::isfinite((float)eps) || !((float)eps > 0.f)) refuse(what, "scale ", scale, " has to be finite, eps ", eps, " positive");
  Shape g{h.numel() / d, d, 1, kind, scale, eps, false};
  Tensor gate = or_none(gate_in);
  if (gate.defined()) {
    gate = plain(gate);
    g.gate_rows = gate_rows_of(what, gate, h);
    g.expanded = g.gate_rows == 0;
    if (g.expanded && h.dim() > 16) refuse(what, "a gate along other axes than whole trailing rows has to have at most 16");
    g.gate_rows = std::max<int64_t>(1, g.gate_rows);
  }
  h = plain(h).contiguous(), y = plain(y).contiguous();
  variable_list out;
  if (grad && at::GradMode::is_enabled()) {
    out = ResidualNorm::apply(h, y, given(gate), given(w[0]), given(w[1]), given(w[2]), given(w[3]), g.rows, g.d, g.gate_rows, g.kind, g.scale, g.eps, g.expanded);
  } else {
    Tensor stats;
    out = norm_forward(h, y, whole_gate(gate, h, g.expanded), w, g, false, stats);
  }
  return {out[0], out[1]};
}

void bind(const std::vector<uintptr_t>& at) {
  if (at.size() != 8) throw py::value_error("eight entries are wanted");
  entries = {(decltype(entries.battn_fwd))at[0],   (decltype(entries.battn_bwd))at[1],   (decltype(entries.battn_ws))at[2],
             (decltype(entries.resnorm_fwd))at[3], (decltype(entries.resnorm_bwd))at[4], (decltype(entries.resnorm_ws))at[5],
             (decltype(entries.gate_sum))at[6],    (decltype(entries.gate_sum_ws))at[7]};
}

}  // namespace

PYBIND11_MODULE(_blocks, m) {
  m.attr("torch_version") = GGD_TORCH;
  m.def("bind", &bind);
  m.def("attention", &attention, py::call_guard<py::gil_scoped_release>());
  m.def("residual_norm", &residual_norm, py::call_guard<py::gil_scoped_release>());
}
