// The torch-side host path in C++: what ops.py and attention_op.py do around a C-ABI call (checks, strides, allocation,
// the stream, the autograd node), for the inputs that need nothing unusual.  Every function returns None for any other
// input -- another dtype, a CPU tensor, a shape the kernels refuse -- and the Python path beside the call takes over and
// raises or converts as it always did; nothing is computed here that the kernels do not compute.  A backward call that a kernel
// refuses (a gradient at an unaligned address) raises the MdattnError that the Python nodes raise.
//
// Why native: a call of the smallest size is host time (4 heads x 126 tokens: 10 us of kernels).  The Python path took
// 36.7 us for prologue + attention (ctypes' conversion of twenty arguments, four stride structs, the checks), this one
// 16.5; a training step's backward runs in autograd's own thread without the interpreter: 255-465 us of host time per
// step become 91-108.
#include <ATen/ATen.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <pybind11/stl.h>
#include <torch/csrc/utils/pybind.h>

#include <array>
#include <cmath>
#include <cstring>
#include <optional>

#include "mdattn.h"
#include "mdattn_host.h"
#include "mdlayers.h"
#include "mdpacked.h"

namespace {

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// the current stream of the device of a tensor that the call has checked (`beside`)
void* stream(const Tensor& on) { return c10::hip::getCurrentHIPStream(on.get_device()).stream(); }
const void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* mut(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* f32(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }

Tensor value(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
// autograd's apply() takes an argument that may be missing as an optional, never as an undefined tensor
OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }
// a tensor that carries a tangent (forward-mode differentiation): left to the Python path, which refuses it
bool dual(const Tensor& t) { return t._fw_grad(0).defined(); }
// ref is the call's first tensor, on the device whose current stream the call takes
bool beside(const Tensor& t, const Tensor& ref) { return t.get_device() == (&t == &ref ? c10::hip::current_device() : ref.get_device()); }
bool bf16_on(const Tensor& t, const Tensor& ref) {
  return t.is_cuda() && t.scalar_type() == at::kBFloat16 && beside(t, ref) && !t.is_neg() && !dual(t);
}
bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
// A leaf's node in the autograd graph belongs to the stream on which it was made and lives as long as any graph that leads to it.  A backward pass
// captured on another stream makes that stream wait inside the capture: a stream of a program's own joins it, the default stream cannot be captured,
// and the failure ends the process.  A forward call that would lead there is refused.
void no_older_graph(std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts) {
    if (!t->defined() || !t->is_cuda() || !t->requires_grad() || t->grad_fn()) continue;
    const auto leaf = torch::autograd::impl::try_get_grad_accumulator(*t);
    const auto on = leaf ? leaf->stream() : std::nullopt;
    if (!on || on->id() != c10::hip::getDefaultHIPStream(t->get_device()).id()) continue;
    TORCH_CHECK(c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None,
                "cannot capture a call that is to be differentiated: one of its inputs is still part of an autograd graph from another stream, the default "
                "stream, which a capture cannot wait for; drop the outputs that hold that graph, or build it on a stream of its own");
  }
}
// A node's plain values as one entry of its saved_data (an entry each, boxed, cost a small backward call a few us)
template <class T>
void keep(AutogradContext* ctx, const T& values) {
  static_assert(std::is_trivially_copyable_v<T>);
  ctx->saved_data["values"] = std::string(reinterpret_cast<const char*>(&values), sizeof values);
}
template <class T>
T kept(AutogradContext* ctx) {
  T values;
  const std::string& s = ctx->saved_data["values"].toStringRef();
  TORCH_INTERNAL_ASSERT(s.size() == sizeof values);
  std::memcpy(&values, s.data(), sizeof values);
  return values;
}
// a tensor's shape of up to eight axes
struct Shape8 {
  int64_t dim = 0, size[8];
  explicit Shape8(const Tensor& t = Tensor()) {
    if (!t.defined()) return;
    dim = t.dim();
    for (int64_t i = 0; i < dim && i < 8; ++i) size[i] = t.size(i);
  }
  at::IntArrayRef get() const { return {size, (size_t)dim}; }
};

// what a saved-tensor hook hands back is read with the form that the forward checked, or refused
void unpacked(bool ok) { TORCH_CHECK_VALUE(ok, "a tensor saved for the backward pass came back from its hook with another dtype, shape or layout"); }
// a backward call: _lib.check(rc, where), whose MdattnError autograd's engine carries back to the thread that waits for it
void must(int rc, const char* where) {
  if (rc == MDATTN_OK) return;
  py::gil_scoped_acquire gil;
  try {
    py::module_::import("maxdiffusion_amd._lib").attr("check")(rc, where);
  } catch (py::error_already_set& e) {
    e.restore();
  }
  python_error err;
  err.persist();
  throw err;
}
// thrown by a node's forward when a kernel refuses the request, before anything was saved: the Python path takes the call
struct Refused {};
template <class F>
auto unless_refused(F&& apply) -> std::optional<decltype(apply())> {
  try {
    return apply();
  } catch (const Refused&) {
    return std::nullopt;
  }
}

// Gradients have none of their own.  Where autograd records a backward pass (create_graph), its results hang on a node that leads to what the
// differentiated node led to, and to the gradients that came in, so that a second derivative reaches it and is refused, not left out.
struct NoSecondDerivative : torch::autograd::Node {
  using Node::Node;
  variable_list apply(variable_list&&) override {
    TORCH_CHECK_NOT_IMPLEMENTED(false, "the gradients of this package's operators cannot be differentiated again: second derivatives are not implemented");
  }
};
variable_list first_order(const variable_list& grads, variable_list results) {
  const auto node = torch::autograd::get_current_node();
  if (!node) return results;
  torch::autograd::edge_list to;
  for (const auto& e : node->next_edges())
    if (e.is_valid()) to.push_back(e);
  for (const Tensor& g : grads)
    if (g.defined() && g.requires_grad()) to.push_back(torch::autograd::impl::gradient_edge(g));
  const std::shared_ptr<torch::autograd::Node> refuses(new NoSecondDerivative(std::move(to)), torch::autograd::deleteNode);
  for (Tensor& r : results) {
    if (!r.defined()) continue;
    r = r.detach();
    torch::autograd::create_gradient_edge(r, refuses);
  }
  return results;
}
// A node that makes its gradients in F::gradients
template <class F>
struct FirstOrder : torch::autograd::Function<F> {
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!at::GradMode::is_enabled()) return F::gradients(ctx, std::move(grads));
    variable_list results;
    {
      at::NoGradGuard guard;
      results = F::gradients(ctx, grads);
    }
    return first_order(grads, std::move(results));
  }
};

// [B,S,H,D] as the kernels walk it, over a rank-3 [B,S,H*D] or a rank-4 [B,H,S,D] tensor (attention_op._as_bshd)
struct View {
  int64_t b = 0, s = 0, h = 0, d = 0;
  mdattn_strides st{0, 0, 0};
};
std::optional<View> as_view(const Tensor& t, int64_t heads) {
  View v;
  if (t.dim() == 3) {
    const int64_t n = t.size(2);
    if (t.stride(2) != 1 || heads <= 0 || n % heads) return std::nullopt;
    v.b = t.size(0); v.s = t.size(1); v.h = heads; v.d = n / heads;
    v.st = {t.stride(0), t.stride(1), v.d};
  } else if (t.dim() == 4) {
    if (t.stride(3) != 1) return std::nullopt;
    v.b = t.size(0); v.h = t.size(1); v.s = t.size(2); v.d = t.size(3);
    v.st = {t.stride(0), t.stride(2), t.stride(1)};
  } else {
    return std::nullopt;
  }
  return v;
}
bool aligned(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }
// Whether the kernels read this place and these strides (their own checks refuse the others): the padding of a head dim makes
// a copy, and with it takes views at any address, so head dims walked unpadded have to fall back to it before a node exists.
bool walkable(const Tensor& t, const View& v) {
  const int64_t m = v.st.batch | v.st.seq | v.st.head;
  return aligned(t) && m % 8 == 0 && v.st.seq >= v.d && v.st.seq < (1 << 23) && v.st.head > 0;
}
// a logical [B,S,H,D] tensor
mdattn_strides strides4(const Tensor& t) { return {t.stride(0), t.stride(1), t.stride(2)}; }

Tensor alloc_bshd(const Tensor& like, int64_t b, int64_t s, int64_t h, int64_t d, bool bhsd) {
  return bhsd ? at::empty({b, h, s, d}, like.options().dtype(at::kBFloat16)).permute({0, 2, 1, 3})
              : at::empty({b, s, h, d}, like.options().dtype(at::kBFloat16));
}
// A gradient as the kernels read it: bf16, last axis contiguous, with the strides of `like` when given.
Tensor grad_like(const Tensor& g, const Tensor& like) {
  Tensor x = g.scalar_type() == at::kBFloat16 ? g : g.to(at::kBFloat16);
  if (like.defined()) return x.strides() == like.strides() ? x : at::empty_strided(like.sizes(), like.strides(), x.options()).copy_(x);
  return x.stride(-1) == 1 ? x : x.contiguous();
}
// The gradients of a prologue's outputs, all with the strides of the first: the kernels walk them with one set.  A first one
// that is expanded (stride 0, as the sum over an axis hands it back) is read in place only when the others are too: nothing
// can be copied into its layout.
bool repeats(const Tensor& t) {
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.size(i) > 1 && t.stride(i) == 0) return true;
  return false;
}
void grads_alike(std::initializer_list<Tensor*> gs) {
  Tensor& first = **gs.begin();
  first = grad_like(first, Tensor());
  if (repeats(first))
    for (const Tensor* g : gs)
      if (g->defined() && (g->strides() != first.strides() || !aligned(*g) || g->scalar_type() != at::kBFloat16)) {
        first = first.contiguous();
        break;
      }
  for (Tensor* g : gs)
    if (g->defined() && g != &first) *g = grad_like(*g, first);
}

// ------------------------------------------------------------------------------------------------ attention
// A key mask as the kernels take it, in one buffer: the additive bias f32 [B, ceil32(Skv)], then the tile lists
struct Mask {
  float* bias = nullptr;
  int* tiles = nullptr;
  int64_t stride = 0;
  static int64_t cols(int64_t skv) { return (skv + 31) / 32 * 32; }
  static int64_t floats(const View& vk) { return vk.b * cols(vk.s) + mdattn_host_key_tiles_ints((int)vk.b, (int)vk.s); }
  Mask(const Tensor& m, const View& vk) {
    if (!m.defined()) return;
    stride = cols(vk.s);
    bias = m.data_ptr<float>();
    tiles = reinterpret_cast<int*>(bias + vk.b * stride);
  }
};

int fwd(const Tensor& q, const Tensor& k, const Tensor& v, const View& vq, const View& vk, const View& vv, const Tensor& out, const Tensor& lse,
        const Tensor& mask, double scale) {
  const Mask m(mask, vk);
  const mdattn_strides so{out.stride(0), out.stride(1), vq.d};
  const int64_t nws = m.bias ? 0 : mdattn_host_fwd_workspace_floats((int)vq.b, (int)vq.h, (int)vq.s, (int)vk.s, (int)vq.d);
  const Tensor ws = nws ? at::empty({nws}, q.options().dtype(at::kFloat)) : Tensor();
  return mdattn_host_fwd_bf16(stream(q), ptr(q), ptr(k), ptr(v), mut(out), f32(lse), (int)vq.b, (int)vq.h, (int)vq.s, (int)vk.s, (int)vq.d, &vq.st, &vk.st,
                              &vv.st, &so, (float)scale, m.bias, m.stride, m.tiles, f32(ws), nws);
}

bool operands(const Tensor& q, const Tensor& k, const Tensor& v, int64_t heads, View& vq, View& vk, View& vv) {
  if (!q.is_cuda() || !bf16_on(q, q) || !bf16_on(k, q) || !bf16_on(v, q)) return false;
  const auto a = as_view(q, heads), b = as_view(k, heads), c = as_view(v, heads);
  if (!a || !b || !c || a->b != b->b || a->b != c->b || a->h != b->h || a->h != c->h || a->d != b->d || a->d != c->d || b->s != c->s) return false;
  vq = *a; vk = *b; vv = *c;
  return true;
}

// q, k, v in the caller's own rank; out [B,Sq,H*D]
struct FlashFn : FirstOrder<FlashFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& mask_, int64_t heads, double scale) {
    const Tensor mask = value(mask_);
    const View vq = *as_view(q, heads), vk = *as_view(k, heads), vv = *as_view(v, heads);
    Tensor out = at::empty({vq.b, vq.s, vq.h * vq.d}, q.options());
    Tensor lse = at::empty({vq.b, vq.h, vq.s}, q.options().dtype(at::kFloat));
    if (fwd(q, k, v, vq, vk, vv, out, lse, mask, scale) != MDATTN_OK) throw Refused{};
    ctx->save_for_backward({q, k, v, out, lse});
    ctx->saved_data["mask"] = mask;  // not for hooks: its tile lists are indices
    ctx->saved_data["heads"] = heads;
    ctx->saved_data["scale"] = scale;
    return out;
  }
  static variable_list gradients(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &out = saved[3], &lse = saved[4];
    const Tensor mask = ctx->saved_data["mask"].toTensor();
    const int64_t heads = ctx->saved_data["heads"].toInt();
    const double scale = ctx->saved_data["scale"].toDouble();
    View vq, vk, vv;
    unpacked(operands(q, k, v, heads, vq, vk, vv) && q.is_non_overlapping_and_dense() && k.is_non_overlapping_and_dense() &&
             v.is_non_overlapping_and_dense() && bf16_on(out, q) && out.is_contiguous() && out.sizes() == grads[0].sizes() && out.dim() == 3 &&
             out.size(0) == vq.b && out.size(1) == vq.s && out.size(2) == vq.h * vq.d && lse.is_cuda() && lse.scalar_type() == at::kFloat &&
             lse.is_contiguous() && lse.numel() == vq.b * vq.h * vq.s && (!mask.defined() || mask.numel() == Mask::floats(vk)));
    const Mask m(mask, vk);
    Tensor dout = grad_like(grads[0], out);
    if (vq.d != 64 && vq.d != 128 && !aligned(dout)) dout = dout.clone();  // (a padded call's backward copies it as well)
    Tensor dq = at::empty_like(q), dk = at::empty_like(k), dv = at::empty_like(v);
    const int B = (int)vq.b, H = (int)vq.h, Sq = (int)vq.s, Skv = (int)vk.s, D = (int)vq.d;
    mdattn_host_bwd_plan plan;
    const int64_t nws = mdattn_host_bwd_plan_floats(B, H, Sq, Skv, D, m.bias != nullptr, -1, &plan);
    Tensor ws = at::empty({nws}, lse.options());
    const mdattn_strides so{out.stride(0), out.stride(1), vq.d};
    const int rc = mdattn_host_bwd_bf16(stream(q), ptr(q), ptr(k), ptr(v), ptr(out), ptr(dout), f32(lse), mut(dq), mut(dk), mut(dv), f32(ws), nws, B, H, Sq,
                                        Skv, D, &vq.st, &vk.st, &vv.st, &so, (float)scale, m.bias, m.stride, m.tiles, &plan);
    must(rc, "mdattn_bwd_bf16");
    return {dq, dk, dv, Tensor(), Tensor(), Tensor()};
  }
};

// [B,Skv] keep-mask (bool or uint8) -> Mask, or undefined when it needs the Python path
Tensor make_mask(const Tensor& keep, const View& vk, const Tensor& ref) {
  if (!keep.is_cuda() || keep.get_device() != ref.get_device() || (keep.scalar_type() != at::kBool && keep.scalar_type() != at::kByte) ||
      keep.dim() != 2 || keep.size(0) != vk.b || keep.size(1) != vk.s || !keep.is_contiguous())
    return Tensor();
  const int B = (int)vk.b, S = (int)vk.s;
  Tensor m = at::empty({Mask::floats(vk)}, keep.options().dtype(at::kFloat));
  const Mask v(m, vk);
  return mdattn_host_key_tiles(stream(keep), ptr(keep), v.bias, v.tiles, B, S, v.stride) == MDATTN_OK ? m : Tensor();
}

// The registry entry's operands, checked: false when the Python path has to take over
bool flash_args(const Tensor& q, const Tensor& k, const Tensor& v, int64_t heads, double scale, const OptTensor& keep, View& vq, View& vk, View& vv,
                Tensor& mask) {
  if (!operands(q, k, v, heads, vq, vk, vv) || !(scale > 0)) return false;
  if (!mdattn_host_head_dim((int)vq.d)) return false;  // padded first
  if (q.numel() == 0 || k.numel() == 0 || std::max(vq.s, vk.s) >= ((int64_t)1 << 31)) return false;
  return !keep.has_value() || (mask = make_mask(*keep, vk, q)).defined();
}

// The registry entry `hip_flash`: [B,S,H*D] or [B,H,S,D] operands -> [B,Sq,H*D]; q_mul is rounded into q first.
OptTensor flash(const Tensor& q, const Tensor& k, const Tensor& v, int64_t heads, double scale, const OptTensor& keep, double q_mul) {
  View vq, vk, vv;
  Tensor mask;
  if (!flash_args(q, k, v, heads, scale, keep, vq, vk, vv, mask)) return std::nullopt;
  at::NoGradGuard guard;
  Tensor qf = q;
  if (q_mul != 1.0) {
    qf = q.mul(q_mul);
    const auto w = as_view(qf, heads);
    if (!w) return std::nullopt;
    vq = *w;
  }
  Tensor out = at::empty({vq.b, vq.s, vq.h * vq.d}, q.options());
  if (fwd(qf, k, v, vq, vk, vv, out, Tensor(), mask, scale) != MDATTN_OK) return std::nullopt;
  return out;
}

OptTensor flash_autograd(const Tensor& q, const Tensor& k, const Tensor& v, int64_t heads, double scale, const OptTensor& keep) {
  View vq, vk, vv;
  Tensor mask;
  for (const Tensor* t : {&q, &k, &v})
    if (!t->is_non_overlapping_and_dense()) return std::nullopt;  // their gradients take the same strides
  if (!operands(q, k, v, heads, vq, vk, vv) || !walkable(q, vq) || !walkable(k, vk) || !walkable(v, vv)) return std::nullopt;
  if (!flash_args(q, k, v, heads, scale, keep, vq, vk, vv, mask)) return std::nullopt;
  return unless_refused([&] { return FlashFn::apply(q, k, v, opt(mask), heads, scale); });
}

// The registry entry `hip_flash_fp8`: dense bf16 operands of either rank -> [B,Sq,H*D]
OptTensor flash_fp8(const Tensor& q, const Tensor& k, const Tensor& v, int64_t heads, double scale, const OptTensor& keep) {
  View vq, vk, vv;
  Tensor mask;
  for (const Tensor* t : {&q, &k, &v})  // the quantised copies are dense [B,S,H,D]
    if (t->dim() == 4 ? !t->permute({0, 2, 1, 3}).is_contiguous() : !t->is_contiguous()) return std::nullopt;
  if (!flash_args(q, k, v, heads, scale, keep, vq, vk, vv, mask) || (vq.d != 64 && vq.d != 128)) return std::nullopt;
  at::NoGradGuard guard;
  const auto bytes = q.options().dtype(at::kByte);
  Tensor q8 = at::empty({q.numel()}, bytes), k8 = at::empty({k.numel()}, bytes), v8 = at::empty({v.numel()}, bytes);
  Tensor ws = at::empty({mdattn_host_quant3_floats()}, q.options().dtype(at::kFloat));
  if (mdattn_host_quant3_e4m3(stream(q), ptr(q), ptr(k), ptr(v), mut(q8), mut(k8), mut(v8), f32(ws), q.numel(), k.numel(),
                              (float)(scale * 1.4426950408889634)) != MDATTN_OK)
    return std::nullopt;
  Tensor out = at::empty({vq.b, vq.s, vq.h * vq.d}, q.options());
  auto dense = [](const View& x) { return mdattn_strides{x.s * x.h * x.d, x.h * x.d, x.d}; };
  const mdattn_strides sq = dense(vq), skv = dense(vk);
  const float *s = f32(ws), scale8 = (float)0.6931471805599453;  // q's quantisation carries scale * log2(e)
  const int B = (int)vq.b, H = (int)vq.h, Sq = (int)vq.s, Skv = (int)vk.s, D = (int)vq.d;
  const Mask m(mask, vk);
  const int rc = m.bias ? mdattn_fwd_fp8_bias(stream(q8), ptr(q8), ptr(k8), ptr(v8), mut(out), nullptr, B, H, Sq, Skv, D, &sq, &skv, &skv, &sq, scale8, s,
                                              s + 2, s + 4, m.bias, m.stride)
                        : mdattn_fwd_fp8(stream(q8), ptr(q8), ptr(k8), ptr(v8), mut(out), nullptr, B, H, Sq, Skv, D, &sq, &skv, &skv, &sq, scale8, s, s + 2,
                                         s + 4, MDATTN_FP8_SOFTMAX_BYTE_GRID);
  if (rc != MDATTN_OK) return std::nullopt;
  return out;
}

// One ring step (ops.flash_attention_merge) on logical [B,S,H,D] views; false: the Python path takes it
bool flash_merge(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& o_run, const Tensor& lse_run, double scale) {
  if (!q.is_cuda() || !bf16_on(q, q) || !bf16_on(k, q) || !bf16_on(v, q) || q.dim() != 4 || k.dim() != 4 || v.dim() != 4 || o_run.dim() != 4)
    return false;
  if (q.stride(3) != 1 || k.stride(3) != 1 || v.stride(3) != 1 || o_run.stride(3) != 1 || k.sizes() != v.sizes() || k.size(0) != q.size(0) ||
      k.size(2) != q.size(2) || k.size(3) != q.size(3) || o_run.sizes() != q.sizes() || o_run.scalar_type() != at::kFloat || !o_run.is_cuda() ||
      !beside(o_run, q) || !beside(lse_run, q) ||
      lse_run.scalar_type() != at::kFloat || !lse_run.is_cuda() || !lse_run.is_contiguous() || lse_run.dim() != 3 || lse_run.size(0) != q.size(0) ||
      lse_run.size(1) != q.size(2) || lse_run.size(2) != q.size(1))
    return false;
  const mdattn_strides sq = strides4(q), sk = strides4(k), sv = strides4(v), so = strides4(o_run);
  return mdattn_fwd_bf16_merge(stream(q), ptr(q), ptr(k), ptr(v), f32(o_run), f32(lse_run), (int)q.size(0), (int)q.size(2), (int)q.size(1),
                               (int)k.size(1), (int)q.size(3), &sq, &sk, &sv, &so, (float)scale) == MDATTN_OK;
}

// ------------------------------------------------------------------------------------------------ attention over packed sequences
// q [Tq,H,D], k, v [Tk,Hkv,D] as the kernels walk them (ops._packed_rows); an axis of one element may have any stride
mdattn_strides row_strides(const Tensor& t) { return {0, t.size(0) > 1 ? t.stride(0) : 0, t.size(1) > 1 ? t.stride(1) : 0}; }
bool packed_rows(const Tensor& t, const Tensor& ref, int64_t group) {
  if (!bf16_on(t, ref) || t.dim() != 3 || t.numel() == 0 || t.stride(2) != 1 || !aligned(t)) return false;
  const mdattn_strides s = row_strides(t);
  return (s.seq | s.head) % 8 == 0 && s.seq < (1 << 23) && group * s.head < (1 << 29);
}
bool index_ok(const Tensor& t, int64_t n, const Tensor& ref) {
  return t.is_cuda() && t.get_device() == ref.get_device() && t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == n && t.is_contiguous();
}
// false: the Python path takes the call (and says what is wrong with it)
bool packed_args(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& qo, const Tensor& ko, const Tensor& kl, bool causal, int64_t max_q,
                 int64_t max_k, mdattn_packed& p) {
  if (!q.is_cuda() || q.dim() != 3 || k.dim() != 3 || k.sizes() != v.sizes() || k.numel() == 0 || q.size(1) % k.size(1) || q.size(2) != k.size(2) ||
      std::max(q.size(0), k.size(0)) >= (int64_t)1 << 31 || !packed_rows(q, q, q.size(1) / k.size(1)) || !packed_rows(k, q, 0) || !packed_rows(v, q, 0))
    return false;
  const int64_t n = qo.numel();
  if (n < 1 || n >= (int64_t)1 << 31 || !index_ok(qo, n, q) || !index_ok(ko, n, q) || (kl.defined() && !index_ok(kl, n - 1, q))) return false;
  auto hint = [](int64_t x) { return (int)std::min<int64_t>(std::max<int64_t>(x, 0), INT32_MAX); };
  p = {static_cast<const int*>(ptr(qo)), static_cast<const int*>(ptr(ko)), static_cast<const int*>(ptr(kl)), (int)(n - 1), (int)q.size(0),
       (int)k.size(0), (int)q.size(1), (int)k.size(1), (int)q.size(2), causal, hint(max_q), hint(max_k)};
  return true;
}
int packed_fwd(const Tensor& q, const Tensor& k, const Tensor& v, const mdattn_packed& p, double scale, const Tensor& out, const Tensor& rest,
               const Tensor& lse) {
  const int64_t nws = mdattn_fwd_bf16_packed_workspace_floats(&p);
  const Tensor ws = nws ? at::empty({nws}, q.options().dtype(at::kFloat)) : Tensor();
  const mdattn_strides sq = row_strides(q), sk = row_strides(k), sv = row_strides(v), so = row_strides(out);
  return mdattn_fwd_bf16_packed(stream(q), &p, ptr(q), ptr(k), ptr(v), mut(out), mut(rest), f32(lse), &sq, &sk, &sv, &so, (float)scale, f32(ws), nws);
}
bool dense_like(const Tensor& t, const Tensor& q) { return bf16_on(t, q) && t.is_contiguous() && t.sizes() == q.sizes() && aligned(t); }
struct PackedFn : FirstOrder<PackedFn> {
  struct Values {
    double scale;
    bool causal;
    int64_t max_q, max_k;
    Shape8 q, k;
    int64_t offsets;
  };
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& qo, const Tensor& ko, bool causal,
                        double scale, int64_t max_q, int64_t max_k) {
    mdattn_packed p;
    packed_args(q, k, v, qo, ko, Tensor(), causal, max_q, max_k, p);
    Tensor out = at::empty(q.sizes(), q.options()), rest = at::empty(q.sizes(), q.options()),
           lse = at::empty({q.size(1), q.size(0)}, q.options().dtype(at::kFloat));
    if (packed_fwd(q, k, v, p, scale, out, rest, lse) != MDATTN_OK) throw Refused{};
    ctx->save_for_backward({q, k, v, qo, ko, out, lse, rest});
    keep(ctx, Values{scale, causal, max_q, max_k, Shape8(q), Shape8(k), qo.size(0)});
    return out;
  }
  static variable_list gradients(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Values c = kept<Values>(ctx);
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &qo = saved[3], &ko = saved[4], &out = saved[5], &lse = saved[6], &rest = saved[7];
    mdattn_packed p;
    unpacked(packed_args(q, k, v, qo, ko, Tensor(), c.causal, c.max_q, c.max_k, p) && q.sizes() == c.q.get() && k.sizes() == c.k.get() && qo.size(0) == c.offsets &&
             dense_like(out, q) && dense_like(rest, q) && lse.is_cuda() && lse.get_device() == q.get_device() && lse.scalar_type() == at::kFloat && lse.is_contiguous() &&
             lse.numel() == q.size(0) * q.size(1));
    Tensor dout = grads[0];
    if (dout.scalar_type() != at::kBFloat16) dout = dout.to(at::kBFloat16);
    if (dout.is_neg()) dout = dout.resolve_neg();
    dout = dout.contiguous();
    if (!aligned(dout)) dout = dout.clone();
    Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()), dv = at::empty(k.sizes(), k.options());
    const int64_t nws = mdattn_bwd_bf16_packed_workspace_floats(&p);
    const Tensor ws = at::empty({nws}, lse.options());
    const mdattn_strides sq = row_strides(q), sk = row_strides(k), sv = row_strides(v), so = row_strides(out), dqs = row_strides(dq), dks = row_strides(dk);
    must(mdattn_bwd_bf16_packed(stream(q), &p, ptr(q), ptr(k), ptr(v), ptr(out), ptr(rest), ptr(dout), f32(lse), mut(dq), mut(dk), mut(dv), &sq, &sk, &sv, &so, &dqs, &dks,
                                &dks, (float)c.scale, f32(ws), nws),
         "mdattn_bwd_bf16_packed");
    return {dq, dk, dv, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};
OptTensor flash_packed(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& qo, const OptTensor& ko_, const OptTensor& kl_, bool causal,
                       double scale, int64_t max_q, int64_t max_k) {
  const Tensor ko = ko_.has_value() ? *ko_ : qo, kl = value(kl_);
  const bool grad = wants_grad({&q, &k, &v});
  if (grad) no_older_graph({&q, &k, &v});
  mdattn_packed p;
  if (!packed_args(q, k, v, qo, ko, kl, causal, max_q, max_k, p)) return std::nullopt;
  if (grad) {
    if (kl.defined() || !(scale >= 1e-30)) return std::nullopt;  // (which the backward pass would refuse)
    return unless_refused([&] { return PackedFn::apply(q, k, v, qo, ko, causal, scale, max_q, max_k); });
  }
  at::NoGradGuard guard;
  Tensor out = at::empty(q.sizes(), q.options());
  if (packed_fwd(q, k, v, p, scale, out, Tensor(), Tensor()) != MDATTN_OK) return std::nullopt;
  return out;
}

// ------------------------------------------------------------------------------------------------ prologues
// A rotary table in one of the layouts that the kernels read in place (attention_op._rope_table)
struct Table {
  Tensor cos, sin;
  int64_t kind = MDATTN_TABLE_PLANES;
};
bool in_place(const Tensor& t, at::ScalarType dtype, int64_t numel, const Tensor& ref) {
  return t.is_cuda() && t.get_device() == ref.get_device() && t.scalar_type() == dtype && t.is_contiguous() && t.numel() == numel &&
         !t.is_conj() && !t.is_neg() && !dual(t) && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0;
}
std::optional<Table> as_table(const OptTensor& a, const OptTensor& b, int64_t s, int64_t d, bool per_head, const Tensor& ref) {
  Table t;
  if (!a.has_value()) return t;
  if (b.has_value()) {  // a (cos, sin) tuple
    if (per_head && in_place(*a, at::kFloat, s * d, ref) && in_place(*b, at::kFloat, s * d, ref)) t.kind = MDATTN_TABLE_REPEATED;
    else if (in_place(*a, at::kFloat, s * d / 2, ref) && in_place(*b, at::kFloat, s * d / 2, ref)) t.kind = MDATTN_TABLE_PLANES;
    else return std::nullopt;
    t.sin = *b;
  } else if (in_place(*a, at::kComplexFloat, s * d / 2, ref)) {
    t.kind = MDATTN_TABLE_COMPLEX;
  } else if (per_head && in_place(*a, at::kFloat, s * d * 2, ref)) {
    t.kind = MDATTN_TABLE_MATRIX;
  } else {
    return std::nullopt;
  }
  t.cos = *a;
  return t;
}
// Replaces a tensor that in_place has accepted, or two of one size (b may be undefined), by copies, in one launch.  False, and nothing
// replaced, for a size that is no multiple of 16 bytes: no kernel takes such rows either.
bool own(Tensor& a, Tensor& b) {
  const Tensor x = at::empty(a.sizes(), a.options()), y = b.defined() ? at::empty(b.sizes(), b.options()) : Tensor();
  if (mdattn_host_copy(stream(a), ptr(a), mut(x), ptr(b), mut(y), (int64_t)a.nbytes()) != MDATTN_OK) return false;
  a = x;
  b = y;
  return true;
}
// The table as a node keeps it.  One that is read in place belongs to the caller, who may have made it in inference mode (autograd
// refuses to save such a tensor) or may rewrite it before the backward: a dense copy of it, one launch.  Half planes [S, D/2] were
// always saved as they are.
bool own_table(Table& t) { return !t.cos.defined() || t.kind == MDATTN_TABLE_PLANES || own(t.cos, t.sin); }
const float* table_ptr(const Tensor& t) { return t.defined() ? static_cast<const float*>(t.data_ptr()) : nullptr; }
bool weight_ok(const Tensor& w, int64_t n, const Tensor& ref) { return bf16_on(w, ref) && w.is_contiguous() && w.numel() == n; }

// a saved q (or fused q|k|v), the k beside it, their weights and table in the form that the forward took
bool rows_back(const Tensor& q, const Tensor& k, int64_t dim, bool dense) {
  return bf16_on(q, q) && q.dim() == dim && q.stride(-1) == 1 && (!dense || q.is_non_overlapping_and_dense()) &&
         (!k.defined() || (bf16_on(k, q) && k.sizes() == q.sizes() && k.strides() == q.strides()));
}
bool weights_back(std::initializer_list<const Tensor*> ws, int64_t n, const Tensor& ref) {
  for (const Tensor* w : ws)
    if (w->defined() && !weight_ok(*w, n, ref)) return false;
  return true;
}
bool table_back(const Tensor& cos, const Tensor& sin, int64_t kind, int64_t s, int64_t d, const Tensor& ref) {
  if (!cos.defined()) return true;
  if (kind == MDATTN_TABLE_COMPLEX) return in_place(cos, at::kComplexFloat, s * d / 2, ref);
  if (kind == MDATTN_TABLE_MATRIX) return in_place(cos, at::kFloat, s * d * 2, ref);
  const int64_t n = kind == MDATTN_TABLE_REPEATED ? s * d : s * d / 2;
  return in_place(cos, at::kFloat, n, ref) && in_place(sin, at::kFloat, n, ref);
}

struct Prologue {
  int64_t heads, kind, n_txt = 0;
  double eps, q_mul;
  bool bhsd;
  void save(AutogradContext* ctx) const {
    ctx->saved_data["i"] = c10::List<int64_t>({heads, kind, n_txt});
    ctx->saved_data["f"] = c10::List<double>({eps, q_mul});
  }
  static Prologue saved(AutogradContext* ctx) {
    const auto i = ctx->saved_data["i"].toIntVector();
    const auto f = ctx->saved_data["f"].toDoubleVector();
    return {i[0], i[1], i[2], f[0], f[1], false};
  }
};

// Wan: q, k [B,S,H*D] (k may be undefined) -> {q_out(, k_out)} or empty when a kernel refuses the request
variable_list fullrow_run(const Tensor& q, const Tensor& k, const Tensor& wq, const Tensor& wk, const Tensor& cos, const Tensor& sin, const Prologue& p) {
  const int64_t b = q.size(0), s = q.size(1), d = q.size(2) / p.heads;
  Tensor qo = alloc_bshd(q, b, s, p.heads, d, p.bhsd), ko = k.defined() ? alloc_bshd(q, b, s, p.heads, d, p.bhsd) : Tensor();
  const mdattn_strides so = strides4(qo);
  const int rc = mdattn_host_norm_rope_fullrow(stream(q), ptr(q), ptr(k), mut(qo), mut(ko), ptr(wq), ptr(wk), table_ptr(cos), table_ptr(sin), (int)p.kind,
                                               (int)b, (int)s, (int)p.heads, (int)d, (float)p.eps, (float)p.q_mul, q.stride(0), q.stride(1), &so);
  if (rc != MDATTN_OK) return {};
  return k.defined() ? variable_list{qo, ko} : variable_list{qo};
}
struct FullrowFn : FirstOrder<FullrowFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const OptTensor& k_, const Tensor& wq, const OptTensor& wk_,
                               const OptTensor& cos_, const OptTensor& sin_, const Prologue& p) {
    const Tensor k = value(k_), wk = value(wk_), cos = value(cos_), sin = value(sin_);
    variable_list out = fullrow_run(q, k, wq, wk, cos, sin, p);
    if (out.empty()) throw Refused{};
    ctx->save_for_backward({q, k, wq, wk, cos, sin});
    p.save(ctx);
    return out;
  }
  static variable_list gradients(AutogradContext* ctx, variable_list g) {
    const auto sv = ctx->get_saved_variables();
    const Tensor &q = sv[0], &k = sv[1], &wq = sv[2], &wk = sv[3];
    const Prologue p = Prologue::saved(ctx);
    unpacked(rows_back(q, k, 3, true) && q.numel() == g[0].numel());
    const int64_t b = q.size(0), s = q.size(1), n = q.size(2), d = n / p.heads;
    unpacked(weights_back({&wq, &wk}, n, q) && table_back(sv[4], sv[5], p.kind, s, d, q) && g[0].sizes() == at::IntArrayRef({b, s, p.heads, d}));
    const bool has_k = k.defined();
    Tensor gq = g[0], gk = has_k ? g[1] : Tensor();
    grads_alike({&gq, &gk});
    Tensor dq = at::empty_strided(q.sizes(), q.strides(), q.options()), dk = has_k ? at::empty_strided(q.sizes(), q.strides(), q.options()) : Tensor();
    Tensor dwq = at::empty({n}, q.options()), dwk = has_k ? at::empty({n}, q.options()) : Tensor();
    const int64_t nws = mdattn_norm_rope_bwd_workspace_floats(b * s, (has_k ? 2 : 1) * n);
    Tensor ws = at::empty({nws}, q.options().dtype(at::kFloat));
    const mdattn_strides sg = strides4(gq);
    must(mdattn_host_norm_rope_fullrow_bwd(stream(q), ptr(q), ptr(k), nullptr, ptr(gq), ptr(gk), mut(dq), mut(dk), ptr(wq), ptr(wk), mut(dwq), mut(dwk),
                                           nullptr, 1, nullptr, nullptr, table_ptr(sv[4]), table_ptr(sv[5]), (int)p.kind, (int)b, (int)s, (int)p.heads, (int)d, (float)p.eps,
                                           (float)p.q_mul, q.stride(0), q.stride(1), dq.stride(0), dq.stride(1), &sg, f32(ws), nws),
         "mdattn_norm_rope_fullrow_bwd");
    return {dq, dk, dwq, dwk, Tensor(), Tensor(), Tensor()};
  }
};

std::optional<variable_list> norm_rope(const Tensor& q, const OptTensor& k_, const Tensor& wq, const OptTensor& wk_, const OptTensor& fa, const OptTensor& fb,
                                       int64_t heads, double eps, double q_mul, bool bhsd) {
  const Tensor k = value(k_), wk = value(wk_);
  if (!q.is_cuda() || !bf16_on(q, q) || q.dim() != 3 || q.numel() == 0 || q.stride(2) != 1 || heads <= 0 || q.size(2) % heads) return std::nullopt;
  const int64_t n = q.size(2);
  if (!weight_ok(wq, n, q)) return std::nullopt;
  if (k.defined() && (!bf16_on(k, q) || k.sizes() != q.sizes() || k.strides() != q.strides() || !wk.defined() || !weight_ok(wk, n, q))) return std::nullopt;
  auto t = as_table(fa, fb, q.size(1), n / heads, false, q);
  if (!t) return std::nullopt;
  const Prologue p{heads, t->kind, 0, eps, q_mul, bhsd};
  if (wants_grad({&q, &k, &wq, &wk})) {
    if (!q.is_non_overlapping_and_dense()) return std::nullopt;
    if (!own_table(*t)) return std::nullopt;
    return unless_refused([&] { return FullrowFn::apply(q, opt(k), wq, k.defined() ? opt(wk) : std::nullopt, opt(t->cos), opt(t->sin), p); });
  }
  variable_list out = fullrow_run(q, k, wq, wk, t->cos, t->sin, p);
  if (out.empty()) return std::nullopt;
  return out;
}

// Flux: q, k logical [B,S,H,D]
variable_list perhead_run(const Tensor& q, const Tensor& k, const Tensor& wq, const Tensor& wk, const Tensor& wqt, const Tensor& wkt, const Tensor& cos,
                          const Tensor& sin, const Prologue& p) {
  const int64_t b = q.size(0), s = q.size(1), h = q.size(2), d = q.size(3);
  Tensor qo = alloc_bshd(q, b, s, h, d, p.bhsd), ko = k.defined() ? alloc_bshd(q, b, s, h, d, p.bhsd) : Tensor();
  const mdattn_strides si = strides4(q), so = strides4(qo);
  const int rc = mdattn_host_norm_rope_perhead(stream(q), ptr(q), ptr(k), mut(qo), mut(ko), ptr(wq), ptr(wk), ptr(wqt), ptr(wkt), (int)p.n_txt,
                                               table_ptr(cos), table_ptr(sin), (int)p.kind, (int)b, (int)s, (int)h, (int)d, (float)p.eps, (float)p.q_mul,
                                               &si, &so);
  if (rc != MDATTN_OK) return {};
  return k.defined() ? variable_list{qo, ko} : variable_list{qo};
}
struct PerheadFn : FirstOrder<PerheadFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const OptTensor& k_, const Tensor& wq, const OptTensor& wk_, const OptTensor& wqt_,
                               const OptTensor& wkt_, const OptTensor& cos_, const OptTensor& sin_, const Prologue& p) {
    const Tensor k = value(k_), wk = value(wk_), wqt = value(wqt_), wkt = value(wkt_), cos = value(cos_), sin = value(sin_);
    variable_list out = perhead_run(q, k, wq, wk, wqt, wkt, cos, sin, p);
    if (out.empty()) throw Refused{};
    ctx->save_for_backward({q, k, wq, wk, wqt, wkt, cos, sin});
    p.save(ctx);
    return out;
  }
  static variable_list gradients(AutogradContext* ctx, variable_list g) {
    const auto sv = ctx->get_saved_variables();
    const Tensor &q = sv[0], &k = sv[1], &wq = sv[2], &wk = sv[3], &wqt = sv[4], &wkt = sv[5];
    const Prologue p = Prologue::saved(ctx);
    unpacked(rows_back(q, k, 4, true) && q.sizes() == g[0].sizes());
    const int64_t b = q.size(0), s = q.size(1), h = q.size(2), d = q.size(3);
    unpacked(weights_back({&wq, &wk, &wqt, &wkt}, d, q) && table_back(sv[6], sv[7], p.kind, s, d, q));
    const bool has_k = k.defined();
    Tensor gq = g[0], gk = has_k ? g[1] : Tensor();
    grads_alike({&gq, &gk});
    Tensor dq = at::empty_strided(q.sizes(), q.strides(), q.options()), dk = has_k ? at::empty_strided(q.sizes(), q.strides(), q.options()) : Tensor();
    auto dw = [&](bool want) { return want ? at::empty({d}, q.options()) : Tensor(); };
    Tensor dwq = dw(true), dwk = dw(has_k), dwqt = dw(wqt.defined()), dwkt = dw(wkt.defined() && has_k);
    const int64_t nws = mdattn_norm_rope_bwd_workspace_floats(b * s * h, 4 * d);
    Tensor ws = at::empty({nws}, q.options().dtype(at::kFloat));
    const mdattn_strides si = strides4(q), sd = strides4(dq), sg = strides4(gq);
    must(mdattn_host_norm_rope_perhead_bwd(stream(q), ptr(q), ptr(k), ptr(gq), ptr(gk), mut(dq), mut(dk), ptr(wq), ptr(wk), ptr(wqt),
                                           has_k ? ptr(wkt) : nullptr, (int)p.n_txt, mut(dwq), mut(dwk), mut(dwqt), mut(dwkt), 1, table_ptr(sv[6]),
                                           table_ptr(sv[7]), (int)p.kind, (int)b, (int)s, (int)h, (int)d, (float)p.eps, (float)p.q_mul, &si, &sd, &sg,
                                           f32(ws), nws),
         "mdattn_norm_rope_perhead_bwd");
    return {dq, dk, dwq, dwk, dwqt, dwkt, Tensor(), Tensor(), Tensor()};
  }
};

std::optional<variable_list> norm_rope_perhead(const Tensor& q, const OptTensor& k_, const Tensor& wq, const OptTensor& wk_, const OptTensor& wqt_,
                                               const OptTensor& wkt_, int64_t n_txt, const OptTensor& fa, const OptTensor& fb, double eps, double q_mul,
                                               bool bhsd) {
  const Tensor k = value(k_), wk = value(wk_), wqt = value(wqt_), wkt = value(wkt_);
  if (!q.is_cuda() || !bf16_on(q, q) || q.dim() != 4 || q.numel() == 0 || q.stride(3) != 1) return std::nullopt;
  const int64_t d = q.size(3);
  if (!weight_ok(wq, d, q) || (wqt.defined() && !weight_ok(wqt, d, q)) || (wkt.defined() && !weight_ok(wkt, d, q))) return std::nullopt;
  if (k.defined() ? (!bf16_on(k, q) || k.sizes() != q.sizes() || k.strides() != q.strides() || !wk.defined() || !weight_ok(wk, d, q)) : wkt.defined())
    return std::nullopt;
  auto t = as_table(fa, fb, q.size(1), d, true, q);
  if (!t) return std::nullopt;
  const Prologue p{q.size(2), t->kind, n_txt, eps, q_mul, bhsd};
  if (wants_grad({&q, &k, &wq, &wk, &wqt, &wkt})) {
    if (!q.is_non_overlapping_and_dense()) return std::nullopt;
    if (!own_table(*t)) return std::nullopt;
    return unless_refused([&] { return PerheadFn::apply(q, opt(k), wq, k.defined() ? opt(wk) : std::nullopt, opt(wqt), opt(wkt), opt(t->cos), opt(t->sin), p); });
  }
  variable_list out = perhead_run(q, k, wq, wk, wqt, wkt, t->cos, t->sin, p);
  if (out.empty()) return std::nullopt;
  return out;
}

// Wan over one fused q|k|v projection output with its biases
variable_list qkv_run(const Tensor& x, const Tensor& bias, const Tensor& wq, const Tensor& wk, const Tensor& cos, const Tensor& sin, const Prologue& p) {
  const int64_t b = x.size(0), s = x.size(1), d = x.size(2) / 3 / p.heads;
  Tensor o[3];
  for (Tensor& t : o) t = alloc_bshd(x, b, s, p.heads, d, p.bhsd);
  const mdattn_strides so = strides4(o[0]);
  const int rc = mdattn_host_norm_rope_qkv(stream(x), ptr(x), ptr(bias), mut(o[0]), mut(o[1]), mut(o[2]), ptr(wq), ptr(wk), table_ptr(cos), table_ptr(sin),
                                           (int)p.kind, (int)b, (int)s, (int)p.heads, (int)d, (float)p.eps, (float)p.q_mul, x.stride(0), x.stride(1), &so);
  if (rc != MDATTN_OK) return {};
  return {o[0], o[1], o[2]};
}
struct QkvFn : FirstOrder<QkvFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& bias, const Tensor& wq, const Tensor& wk, const OptTensor& cos_,
                               const OptTensor& sin_, const Prologue& p) {
    const Tensor cos = value(cos_), sin = value(sin_);
    variable_list out = qkv_run(x, bias, wq, wk, cos, sin, p);
    if (out.empty()) throw Refused{};
    ctx->save_for_backward({x, bias, wq, wk, cos, sin});
    p.save(ctx);
    return out;
  }
  static variable_list gradients(AutogradContext* ctx, variable_list g) {
    const auto sv = ctx->get_saved_variables();
    const Tensor &x = sv[0], &bias = sv[1], &wq = sv[2], &wk = sv[3];
    const Prologue p = Prologue::saved(ctx);
    unpacked(rows_back(x, Tensor(), 3, false));
    const int64_t b = x.size(0), s = x.size(1), n = x.size(2) / 3, d = n / p.heads;
    unpacked(weights_back({&wq, &wk}, n, x) && weight_ok(bias, 3 * n, x) && table_back(sv[4], sv[5], p.kind, s, d, x) &&
             g[0].sizes() == at::IntArrayRef({b, s, p.heads, d}));
    Tensor gq = g[0], gk = g[1], gv = g[2];
    grads_alike({&gq, &gk, &gv});
    // the value block took a view at any address; the copy has gq's strides also where these leave gaps (a clone would close them)
    if (!aligned(gv)) gv = at::empty_strided(gq.sizes(), gq.strides(), gq.options()).copy_(gv);
    Tensor dx = at::empty({b, s, 3 * n}, x.options());
    Tensor dwq = at::empty({n}, x.options()), dwk = at::empty({n}, x.options()), db = at::empty({3 * n}, x.options());
    const int64_t nws = mdattn_norm_rope_bwd_workspace_floats(b * s, 5 * n);
    Tensor ws = at::empty({nws}, x.options().dtype(at::kFloat));
    const mdattn_strides sg = strides4(gq);
    const char* xp = static_cast<const char*>(ptr(x));
    char* dp = static_cast<char*>(mut(dx));
    must(mdattn_host_norm_rope_fullrow_bwd(stream(x), xp, xp + 2 * n, ptr(bias), ptr(gq), ptr(gk), dp, dp + 2 * n, ptr(wq), ptr(wk), mut(dwq), mut(dwk),
                                           mut(db), 1, ptr(gv), dp + 4 * n, table_ptr(sv[4]), table_ptr(sv[5]), (int)p.kind, (int)b, (int)s, (int)p.heads, (int)d, (float)p.eps,
                                           (float)p.q_mul, x.stride(0), x.stride(1), dx.stride(0), dx.stride(1), &sg, f32(ws), nws),
         "mdattn_norm_rope_fullrow_bwd");
    return {dx, db, dwq, dwk, Tensor(), Tensor(), Tensor()};
  }
};

std::optional<variable_list> norm_rope_qkv(const Tensor& x, const Tensor& bias, const Tensor& wq, const Tensor& wk, const OptTensor& fa, const OptTensor& fb,
                                           int64_t heads, double eps, double q_mul, bool bhsd) {
  if (!x.is_cuda() || !bf16_on(x, x) || x.dim() != 3 || x.numel() == 0 || x.stride(2) != 1 || heads <= 0 || x.size(2) % (3 * heads)) return std::nullopt;
  const int64_t n = x.size(2) / 3;
  if (!weight_ok(wq, n, x) || !weight_ok(wk, n, x) || !weight_ok(bias, 3 * n, x)) return std::nullopt;
  auto t = as_table(fa, fb, x.size(1), n / heads, false, x);
  if (!t) return std::nullopt;
  const Prologue p{heads, t->kind, 0, eps, q_mul, bhsd};
  if (wants_grad({&x, &bias, &wq, &wk})) {
    if (!own_table(*t)) return std::nullopt;
    return unless_refused([&] { return QkvFn::apply(x, bias, wq, wk, opt(t->cos), opt(t->sin), p); });
  }
  variable_list out = qkv_run(x, bias, wq, wk, t->cos, t->sin, p);
  if (out.empty()) return std::nullopt;
  return out;
}

// LTX-2: q, or q and k with one table; f32 weights; tables of the tensors' own size (mode 1) or [B,H,S,D/2] (mode 2)
struct Rows {
  int64_t heads, mode;
  double eps, w_mul;
};
variable_list rows_run(const Tensor& q, const Tensor& k, const Tensor& wq, const Tensor& wk, const Tensor& cos, const Tensor& sin, const Rows& p) {
  const int64_t b = q.size(0), s = q.size(1), d = q.size(2) / p.heads;
  Tensor qo = alloc_bshd(q, b, s, p.heads, d, false), ko = k.defined() ? alloc_bshd(q, b, s, p.heads, d, false) : Tensor();
  const mdattn_strides so = strides4(qo);
  const int rc = mdattn_host_norm_rope_rows(stream(q), ptr(q), ptr(k), q.scalar_type() == at::kFloat, mut(qo), mut(ko), f32(wq), f32(wk), f32(cos), f32(sin),
                                            (int)p.mode, (int)b, (int)s, (int)p.heads, (int)d, (float)p.eps, (float)p.w_mul, q.stride(0), q.stride(1), &so);
  if (rc != MDATTN_OK) return {};
  return k.defined() ? variable_list{qo, ko} : variable_list{qo};
}
struct RowsFn : FirstOrder<RowsFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const OptTensor& k_, const Tensor& wq, const OptTensor& wk_, const OptTensor& cos_,
                               const OptTensor& sin_, const Rows& p) {
    const Tensor k = value(k_), wk = value(wk_), cos = value(cos_), sin = value(sin_);
    variable_list out = rows_run(q, k, wq, wk, cos, sin, p);
    if (out.empty()) throw Refused{};
    // a weight with a factor is saved as a copy, as its product with the factor was: the caller's may be an inference tensor, or
    // be updated before the backward
    Tensor kept_wq = wq, none;
    if (p.w_mul != 1.0 && !own(kept_wq, none)) throw Refused{};
    ctx->save_for_backward({q, k, kept_wq, wk, cos, sin});
    ctx->saved_data["i"] = c10::List<int64_t>({p.heads, p.mode, (int64_t)q.scalar_type()});
    ctx->saved_data["f"] = c10::List<double>({p.eps, p.w_mul});
    ctx->set_materialize_grads(false);  // an output that the loss does not reach: no gradient for its input and weight
    return out;
  }
  // A backward through one output frees what both have saved; the other output's is kept beside, with its versions, so that a
  // second backward through that one runs as it would through a node of its own.
  static void leave(AutogradContext* ctx, const variable_list& sv, int64_t which) {
    variable_list left(6);
    for (const int64_t i : {which, 2 + which, (int64_t)4, (int64_t)5}) left[i] = sv[i];
    c10::List<int64_t> versions;
    for (const Tensor& t : left) versions.push_back(!t.defined() || t.is_inference() ? 0 : t._version());
    ctx->saved_data["left"] = left;
    ctx->saved_data["versions"] = versions;
  }
  static variable_list saved(AutogradContext* ctx, int64_t one, bool pair) {
    try {
      return ctx->get_saved_variables();
    } catch (const c10::Error&) {
      const auto at = ctx->saved_data.find("left");
      if (pair || at == ctx->saved_data.end()) throw;
      const variable_list left = at->second.toTensorVector();
      const auto versions = ctx->saved_data["versions"].toIntVector();
      if (!left[one].defined()) throw;
      for (size_t i = 0; i < left.size(); ++i)
        TORCH_CHECK(!left[i].defined() || left[i].is_inference() || left[i]._version() == versions[i],
                    "one of the variables needed for gradient computation has been modified by an inplace operation");
      ctx->saved_data.erase(at);
      return left;
    }
  }
  static variable_list gradients(AutogradContext* ctx, variable_list grads) {
    const bool has[2] = {grads[0].defined(), grads.size() > 1 && grads[1].defined()};
    if (!has[0] && !has[1]) return variable_list(7);
    const bool pair = has[0] && has[1];
    const int one = has[0] ? 0 : 1;  // the tensor of a backward of one
    const variable_list sv = saved(ctx, one, pair);
    if (!pair && sv[1 - one].defined()) leave(ctx, sv, 1 - one);
    const Tensor q = sv[one], k = pair ? sv[1] : Tensor(), wq = sv[2 + one], wk = pair ? sv[3] : Tensor();
    const auto iv = ctx->saved_data["i"].toIntVector();
    const auto fv = ctx->saved_data["f"].toDoubleVector();
    const int64_t heads = iv[0], mode = iv[1];
    unpacked(q.is_cuda() && (int64_t)q.scalar_type() == iv[2] && q.dim() == 3 && q.stride(2) == 1 && q.is_non_overlapping_and_dense() &&
             (!pair || (k.get_device() == q.get_device() && k.scalar_type() == q.scalar_type() && k.sizes() == q.sizes() && k.strides() == q.strides())));
    const int64_t b = q.size(0), s = q.size(1), n = q.size(2);
    unpacked(grads[one].sizes() == at::IntArrayRef({b, s, heads, n / heads}) && in_place(wq, at::kFloat, n, q) && (!pair || in_place(wk, at::kFloat, n, q)));
    for (const Tensor& t : {sv[4], sv[5]}) unpacked(!mode || in_place(t, at::kFloat, mode == 1 ? q.numel() : q.numel() / 2, q));
    Tensor gq = grads[one], gk = pair ? grads[1] : Tensor();
    grads_alike({&gq, &gk});
    Tensor dq = at::empty_strided(q.sizes(), q.strides(), q.options()), dk = pair ? at::empty_strided(q.sizes(), q.strides(), q.options()) : Tensor();
    Tensor dwq = at::empty({n}, wq.options()), dwk = pair ? at::empty({n}, wq.options()) : Tensor();
    const int64_t nws = mdattn_norm_rope_bwd_workspace_floats(b * s, (pair ? 2 : 1) * n);
    Tensor ws = at::empty({nws}, wq.options());
    const mdattn_strides sg = strides4(gq);
    must(mdattn_host_norm_rope_rows_bwd(stream(q), ptr(q), ptr(k), q.scalar_type() == at::kFloat, ptr(gq), ptr(gk), mut(dq), mut(dk), f32(wq), f32(wk),
                                        f32(dwq), f32(dwk), f32(sv[4]), f32(sv[5]), (int)mode, (int)b, (int)s, (int)heads, (int)(n / heads), (float)fv[0],
                                        one ? 1.0f : (float)fv[1], q.stride(0), q.stride(1), dq.stride(0), dq.stride(1), &sg, f32(ws), nws),
         "mdattn_norm_rope_rows_bwd");
    if (one) return {Tensor(), dq, Tensor(), dwq, Tensor(), Tensor(), Tensor()};
    return {dq, dk, dwq, dwk, Tensor(), Tensor(), Tensor()};
  }
};

std::optional<variable_list> norm_rope_rows(const Tensor& q, const OptTensor& k_, const Tensor& wq, const OptTensor& wk_, const OptTensor& cos_,
                                            const OptTensor& sin_, int64_t heads, int64_t mode, double eps, double w_mul) {
  const Tensor k = value(k_), wk = value(wk_), cos = value(cos_), sin = value(sin_);
  if (!q.is_cuda() || !beside(q, q) || (q.scalar_type() != at::kFloat && q.scalar_type() != at::kBFloat16) || q.is_neg() || dual(q) || q.dim() != 3 || q.numel() == 0 ||
      q.stride(2) != 1 || heads <= 0 || q.size(2) % heads)
    return std::nullopt;
  const int64_t b = q.size(0), s = q.size(1), n = q.size(2);
  if (!in_place(wq, at::kFloat, n, q)) return std::nullopt;
  if (k.defined() && (n > 4096 || k.scalar_type() != q.scalar_type() || !k.is_cuda() || k.get_device() != q.get_device() || k.is_neg() || dual(k) ||
                      k.sizes() != q.sizes() || k.strides() != q.strides() || !wk.defined() || !in_place(wk, at::kFloat, n, q)))
    return std::nullopt;
  if (mode) {
    const std::array<int64_t, 3> full{b, s, n};
    const std::array<int64_t, 4> half{b, heads, s, n / heads / 2};
    const at::IntArrayRef want = mode == 1 ? at::IntArrayRef(full) : at::IntArrayRef(half);
    for (const Tensor* t : {&cos, &sin})
      if (!t->defined() || t->sizes() != want || !in_place(*t, at::kFloat, t->numel(), q)) return std::nullopt;
  }
  const Rows p{heads, mode, eps, w_mul};
  const Tensor c = mode ? cos : Tensor(), sn = mode ? sin : Tensor();
  const bool grad_q = wants_grad({&q, &wq}), grad_k = k.defined() ? wants_grad({&k, &wk}) : grad_q;
  if (grad_q != grad_k) return std::nullopt;  // one call each: the other output needs no gradient
  if (grad_q) {
    if (!q.is_non_overlapping_and_dense()) return std::nullopt;
    return unless_refused([&] { return RowsFn::apply(q, opt(k), wq, k.defined() ? opt(wk) : std::nullopt, opt(c), opt(sn), p); });
  }
  variable_list out = rows_run(q, k, wq, wk, c, sn, p);
  if (out.empty()) return std::nullopt;
  return out;
}

// ------------------------------------------------------------------------------------------------ the layers beside attention
// (layer_op.py, ops.py.)  An undefined tensor is a missing one.
bool float_on(const Tensor& t, const Tensor& ref) {
  return t.is_cuda() && (t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat) && beside(t, ref) && !t.is_neg() &&
         !dual(t);
}
int is_f32(const Tensor& t) { return t.defined() && t.scalar_type() == at::kFloat; }

// x [..., C] as the norm walks it: the first axis, and the ones between it and the last, which have to be dense (an axis of one element
// may have any stride)
struct Rows3 {
  int64_t groups = 0, rows = 0, c = 0, sg = 0, sr = 0;
  int64_t all() const { return groups * rows; }
};
std::optional<Rows3> as_rows(const Tensor& x) {
  const int64_t n = x.dim();
  if (n < 2 || x.numel() == 0 || (x.stride(n - 1) != 1 && x.size(n - 1) > 1)) return std::nullopt;
  Rows3 r;
  r.c = x.size(n - 1);
  r.sr = n == 2 ? x.stride(0) : r.c;
  int64_t next = -1;  // the stride that the next axis outwards has to have
  for (int64_t i = n - 2; i > 0 && n > 2; --i) {
    if (x.size(i) == 1) continue;
    if (next < 0) r.sr = x.stride(i);
    else if (x.stride(i) != next) return std::nullopt;
    next = x.stride(i) * x.size(i);
  }
  r.groups = n == 2 ? 1 : x.size(0);
  r.sg = n == 2 ? 0 : x.stride(0);
  r.rows = x.numel() / r.c / r.groups;
  if (r.c > 16384) return std::nullopt;
  return r;
}
// elements between the groups' vectors of w and b, which have to agree; false: the Python path says what is wrong
bool norm_vectors(const Tensor& x, const Rows3& r, const Tensor& w, const Tensor& b, int64_t& stride, int& f32) {
  stride = -1;
  f32 = 0;
  for (const Tensor* t : {&w, &b}) {
    if (!t->defined()) continue;
    if (!float_on(*t, x) || !t->is_contiguous() || t->numel() == 0 || t->dim() == 0 || t->size(t->dim() - 1) != r.c) return false;
    const bool per_group = (t->dim() == 2 && t->size(0) == r.groups) || (t->dim() == 3 && t->size(0) == r.groups && t->size(1) == 1);
    if (!per_group && t->dim() != 1) return false;
    const int64_t mine = per_group ? r.c : 0;
    if (stride >= 0 && (stride != mine || f32 != is_f32(*t))) return false;
    stride = mine;
    f32 = is_f32(*t);
  }
  if (stride < 0) stride = 0;
  return true;
}

Tensor norm_run(const Tensor& x, const Rows3& r, const Tensor& w, const Tensor& b, int64_t stride, int f32, double eps, double offset) {
  Tensor y = at::empty(x.sizes(), x.options());
  const int rc = mdattn_layer_norm(stream(x), ptr(x), is_f32(x), mut(y), is_f32(x), ptr(w), ptr(b), f32, r.groups, r.rows, (int)r.c, r.sg, r.sr, r.rows * r.c,
                                   r.c, stride, (float)eps, (float)offset);
  return rc == MDATTN_OK ? y : Tensor();
}
// Saved for the backward: x and w; of b only its shape and type.
struct NormFn : FirstOrder<NormFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& w_, const OptTensor& b_, double eps, double offset) {
    const Tensor w = value(w_), b = value(b_);
    const Rows3 r = *as_rows(x);
    int64_t stride;
    int f32;
    norm_vectors(x, r, w, b, stride, f32);
    Tensor y = norm_run(x, r, w, b, stride, f32, eps, offset);
    if (!y.defined()) throw Refused{};
    ctx->save_for_backward({x, w});
    ctx->saved_data["f"] = c10::List<double>({eps, offset});
    ctx->saved_data["i"] = c10::List<int64_t>({stride, f32, w.defined(), b.defined(), (w.defined() && w.requires_grad()) || (b.defined() && b.requires_grad()), is_f32(x)});
    ctx->saved_data["wshape"] = w.defined() ? w.sizes().vec() : std::vector<int64_t>{};
    ctx->saved_data["bshape"] = b.defined() ? b.sizes().vec() : std::vector<int64_t>{};
    return y;
  }
  static variable_list gradients(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const auto f = ctx->saved_data["f"].toDoubleVector();
    const auto i = ctx->saved_data["i"].toIntVector();
    const Tensor &x = saved[0], &w = saved[1];
    Tensor g = grads[0];
    const auto r = as_rows(x);
    unpacked(r && float_on(x, x) && is_f32(x) == (int)i[5] && x.sizes() == g.sizes() && w.defined() == (bool)i[2] &&
             (!w.defined() || (float_on(w, x) && is_f32(w) == (int)i[1] && w.is_contiguous() && w.sizes() == at::IntArrayRef(ctx->saved_data["wshape"].toIntVector()))));
    if (g.scalar_type() != x.scalar_type()) g = g.to(x.scalar_type());
    auto rg = as_rows(g);
    if (!rg || g.is_neg()) {
      g = g.contiguous();
      rg = as_rows(g);
    }
    const bool vectors = i[4];
    const auto vec = x.options().dtype(i[1] ? at::kFloat : at::kBFloat16);
    Tensor dx = at::empty(x.sizes(), x.options());
    Tensor dw = vectors && i[2] ? at::empty(ctx->saved_data["wshape"].toIntVector(), vec) : Tensor();
    Tensor db = vectors && i[3] ? at::empty(ctx->saved_data["bshape"].toIntVector(), vec) : Tensor();
    const int64_t nws = dw.defined() || db.defined() ? mdattn_layer_norm_bwd_workspace_floats(r->groups, r->rows, (int)r->c) : 0;
    const Tensor ws = nws ? at::empty({nws}, x.options().dtype(at::kFloat)) : Tensor();
    must(mdattn_layer_norm_bwd(stream(x), ptr(x), is_f32(x), ptr(g), mut(dx), ptr(w), mut(dw), mut(db), (int)i[1], r->groups, r->rows, (int)r->c, r->sg, r->sr,
                               rg->sg, rg->sr, r->rows * r->c, r->c, i[0], (float)f[0], (float)f[1], f32(ws), nws),
         "mdattn_layer_norm_bwd");
    return {dx, dw, db, Tensor(), Tensor()};
  }
};
OptTensor layer_norm(const Tensor& x, const OptTensor& w_, const OptTensor& b_, double eps, double offset) {
  const Tensor w = value(w_), b = value(b_);
  int64_t stride;
  int f32;
  if (!x.is_cuda() || !float_on(x, x)) return std::nullopt;
  const auto r = as_rows(x);
  if (!r || !norm_vectors(x, *r, w, b, stride, f32)) return std::nullopt;
  if (wants_grad({&x, &w, &b})) return unless_refused([&] { return NormFn::apply(x, w_, b_, eps, offset); });
  at::NoGradGuard guard;
  const Tensor y = norm_run(x, *r, w, b, stride, f32, eps, offset);
  return opt(y);
}

// The residual beside x: its rows, or none; false: the Python path says what is wrong
bool residual_rows(const Tensor& x, const Tensor& res, Rows3& r) {
  if (!res.defined()) return true;
  if (!float_on(res, x) || res.sizes() != x.sizes() || is_f32(res) < is_f32(x)) return false;
  const auto rows = as_rows(res);
  if (!rows) return false;
  r = *rows;
  return true;
}
// {y} or {y, s}, or empty where a kernel refuses the request
variable_list rms_run(const Tensor& x, const Rows3& r, const Tensor& w, const Tensor& b, const Tensor& res, const Rows3& rr, int64_t stride, int f32, double eps,
                      double offset) {
  Tensor y = at::empty(x.sizes(), x.options()), s = res.defined() ? at::empty(x.sizes(), res.options()) : Tensor();
  const int64_t sg = r.rows * r.c;
  if (mdattn_rms_norm(stream(x), ptr(x), is_f32(x), ptr(res), is_f32(res), mut(y), mut(s), ptr(w), ptr(b), f32, r.groups, r.rows, (int)r.c, r.sg, r.sr, rr.sg,
                      rr.sr, sg, r.c, sg, r.c, stride, (float)eps, (float)offset) != MDATTN_OK)
    return {};
  return s.defined() ? variable_list{y, s} : variable_list{y};
}
// Saved for the backward: s (x, without a residual) and w; of b only its shape and type.  Where the gradient of an f32 w is wanted beside an s in bf16,
// whose rounding it would show: x and the residual in place of s.
struct RmsFn : FirstOrder<RmsFn> {
  struct Values {
    double eps, offset;
    int64_t stride;
    int vectors_f32, s_f32, x_f32;
    bool w, b, vectors, residual, again;  // which there are; whether the vectors' gradients are wanted; whether s is added up again
    Shape8 x, w_shape, b_shape;
  };
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& w_, const OptTensor& b_, const OptTensor& res_, double eps, double offset) {
    const Tensor w = value(w_), b = value(b_), res = value(res_);
    const Rows3 r = *as_rows(x);
    Rows3 rr;
    int64_t stride;
    int f32;
    residual_rows(x, res, rr);
    norm_vectors(x, r, w, b, stride, f32);
    variable_list out = rms_run(x, r, w, b, res, rr, stride, f32, eps, offset);
    if (out.empty()) throw Refused{};
    ctx->set_materialize_grads(false);
    const bool again = res.defined() && !is_f32(res) && w.defined() && is_f32(w) && w.requires_grad();
    ctx->save_for_backward({res.defined() && !again ? out[1] : x, w, again ? res : Tensor()});
    keep(ctx, Values{eps, offset, stride, f32, is_f32(res.defined() ? res : x), is_f32(x), w.defined(), b.defined(),
                     (w.defined() && w.requires_grad()) || (b.defined() && b.requires_grad()), res.defined(), again, Shape8(x), Shape8(w), Shape8(b)});
    return out;
  }
  // a gradient as rows of the wanted type
  static Rows3 as_gradient(Tensor& g, at::ScalarType type) {
    if (g.scalar_type() != type) g = g.to(type);
    auto r = as_rows(g);
    if (!r || g.is_neg()) {
      g = g.resolve_neg().contiguous();
      r = as_rows(g);
    }
    return *r;
  }
  static variable_list gradients(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Values c = kept<Values>(ctx);
    const Tensor &s = saved[0], &w = saved[1], &res = saved[2];
    const auto r = as_rows(s);
    Rows3 rr{};
    unpacked(r && res.defined() == c.again && residual_rows(s, res, rr) && (!c.again || !is_f32(res)) && float_on(s, s) && is_f32(s) == c.s_f32 && s.sizes() == c.x.get() && w.defined() == c.w &&
             (!c.w || (float_on(w, s) && is_f32(w) == c.vectors_f32 && w.is_contiguous() && w.sizes() == c.w_shape.get())));
    const auto g_type = c.x_f32 ? at::kFloat : at::kBFloat16;
    Tensor g = grads[0].defined() ? grads[0] : at::zeros(s.sizes(), s.options().dtype(g_type)), gs = c.residual ? grads[1] : Tensor();
    const Rows3 rg = as_gradient(g, g_type), rs = gs.defined() ? as_gradient(gs, s.scalar_type()) : Rows3{};
    const bool narrow = c.s_f32 != c.x_f32;
    const auto vec = s.options().dtype(c.vectors_f32 ? at::kFloat : at::kBFloat16);
    Tensor ds = at::empty(s.sizes(), s.options()), dx = narrow ? at::empty(s.sizes(), s.options().dtype(at::kBFloat16)) : Tensor();
    Tensor dw = c.vectors && c.w ? at::empty(c.w_shape.get(), vec) : Tensor(), db = c.vectors && c.b ? at::empty(c.b_shape.get(), vec) : Tensor();
    const int64_t nws = dw.defined() || db.defined() ? mdattn_rms_norm_bwd_workspace_floats(r->groups, r->rows, (int)r->c) : 0;
    const Tensor ws = nws ? at::empty({nws}, s.options().dtype(at::kFloat)) : Tensor();
    must(mdattn_rms_norm_bwd(stream(s), ptr(s), is_f32(s), ptr(res), ptr(g), is_f32(g), ptr(gs), mut(ds), mut(dx), ptr(w), mut(dw), mut(db), c.vectors_f32, r->groups,
                             r->rows, (int)r->c, r->sg, r->sr, rr.sg, rr.sr, rg.sg, rg.sr, rs.sg, rs.sr, c.stride, (float)c.eps, (float)c.offset, f32(ws), nws),
         "mdattn_rms_norm_bwd");
    return {narrow ? dx : ds, dw, db, c.residual ? ds : Tensor(), Tensor(), Tensor()};
  }
};
std::optional<variable_list> rms_norm(const Tensor& x, const OptTensor& w_, const OptTensor& b_, const OptTensor& res_, double eps, double offset) {
  const Tensor w = value(w_), b = value(b_), res = value(res_);
  int64_t stride;
  int f32;
  Rows3 rr;
  const bool grad = wants_grad({&x, &w, &b, &res});
  if (grad) no_older_graph({&x, &w, &b, &res});
  if (!x.is_cuda() || !float_on(x, x)) return std::nullopt;
  const auto r = as_rows(x);
  if (!r || !norm_vectors(x, *r, w, b, stride, f32) || !residual_rows(x, res, rr)) return std::nullopt;
  if (grad) {
    if (x.dim() > 8) return std::nullopt;
    return unless_refused([&] { return RmsFn::apply(x, w_, b_, res_, eps, offset); });
  }
  at::NoGradGuard guard;
  variable_list out = rms_run(x, *r, w, b, res, rr, stride, f32, eps, offset);
  if (out.empty()) return std::nullopt;
  return out;
}

// [rows, cols] in blocks of e4m3 (ops.BlockQuant), in one buffer: the values, then the scales
struct Blocks {
  Tensor buf;
  int64_t rows, cols, block_rows;
  static int64_t values_bytes(int64_t rows, int64_t cols) { return rows * ((cols + 127) / 128 * 128); }
  static int64_t bytes(int64_t rows, int64_t cols, int64_t block_rows) {
    return values_bytes(rows, cols) + (rows + block_rows - 1) / block_rows * ((cols + 511) / 512 * 4);
  }
  Blocks(const Tensor& like, int64_t r, int64_t c, int64_t br) : buf(at::empty({bytes(r, c, br)}, like.options().dtype(at::kByte))), rows(r), cols(c), block_rows(br) {}
  Blocks(const Tensor& saved, int64_t r, int64_t c, int64_t br, const Tensor& ref) : buf(saved), rows(r), cols(c), block_rows(br) {
    unpacked(buf.is_cuda() && buf.get_device() == ref.get_device() && buf.scalar_type() == at::kByte && buf.is_contiguous() && buf.numel() == bytes(r, c, br) && aligned(buf));
  }
  uint8_t* values() const { return static_cast<uint8_t*>(buf.data_ptr()); }
  uint8_t* scales() const { return values() + values_bytes(rows, cols); }
};
// x [..., K] as a matrix of contiguous rows with one stride, or undefined
Tensor as_matrix(const Tensor& x) {
  const int64_t k = x.size(-1);
  if (x.is_contiguous()) return x.view({x.numel() / k, k});
  if (x.dim() == 2 && x.stride(1) == 1) return x;
  return Tensor();
}
int quant(const Tensor& x, int64_t block_rows, const Blocks* q, const Blocks* qt, const Tensor& sums) {
  return mdattn_quant_block_e4m3(stream(x), ptr(x), is_f32(x), x.size(0), x.size(1), x.stride(0), (int)block_rows, q ? q->values() : nullptr,
                                 q ? q->scales() : nullptr, qt ? qt->values() : nullptr, qt ? qt->scales() : nullptr, f32(sums));
}
// into out, dense, of m x n elements in whatever shape the caller wants: a view of it would be one that autograd forbids to change in place
int product(const uint8_t* a, const uint8_t* sa, const uint8_t* b, const uint8_t* sb, int64_t b_block_rows, const Tensor& bias, const Tensor& out, int64_t m,
            int64_t n, int64_t k) {
  const int64_t nws = mdattn_matmul_fp8_block_workspace_floats(m, n, k);
  const Tensor ws = nws ? at::empty({nws}, out.options().dtype(at::kFloat)) : Tensor();
  return mdattn_matmul_fp8_block(stream(out), a, sa, b, sb, (int)b_block_rows, ptr(bias), is_f32(bias), mut(out), n, m, n, k, f32(ws), nws);
}
std::vector<int64_t> with_last(const Tensor& x, int64_t n) {
  auto v = x.sizes().vec();
  v.back() = n;
  return v;
}
bool bias_ok(const Tensor& b, int64_t n, const Tensor& ref) { return !b.defined() || (float_on(b, ref) && b.dim() == 1 && b.size(0) == n && b.is_contiguous()); }

// From a weight that the program keeps quantised; with a norm in front where `norm` says so (rows by `r`)
OptTensor linear_quantized(const Tensor& x, const Tensor& values, const Tensor& scales, int64_t n, int64_t k, int64_t block_rows, const OptTensor& bias_, bool norm,
                           const OptTensor& w_, const OptTensor& b_, double eps, double offset) {
  const Tensor bias = value(bias_), w = value(w_), b = value(b_);
  if (!x.is_cuda() || !float_on(x, x) || x.dim() < 1 || x.size(-1) != k || x.numel() == 0 || k <= 0 || n <= 0 || !values.is_cuda() ||
      values.get_device() != x.get_device() || scales.get_device() != x.get_device() || !bias_ok(bias, n, x) || wants_grad({&x, &bias, &w, &b}))
    return std::nullopt;
  at::NoGradGuard guard;
  std::optional<Rows3> r;
  Tensor rows;
  int64_t stride = 0;
  int f32 = 0;
  if (norm) {
    r = as_rows(x);
    if (!r || !norm_vectors(x, *r, w, b, stride, f32)) return std::nullopt;
  } else {
    rows = as_matrix(x);
    if (!rows.defined()) return std::nullopt;
  }
  const int64_t m = norm ? r->all() : rows.size(0);
  const Blocks q(x, m, k, 1);
  const int rc = norm ? mdattn_layer_norm_e4m3(stream(x), ptr(x), is_f32(x), q.values(), q.scales(), ptr(w), ptr(b), f32, r->groups, r->rows, (int)r->c, r->sg, r->sr,
                                               stride, (float)eps, (float)offset)
                      : quant(rows, 1, &q, nullptr, Tensor());
  if (rc != MDATTN_OK) return std::nullopt;
  Tensor y = at::empty(with_last(x, n), x.options().dtype(at::kBFloat16));
  if (product(q.values(), q.scales(), static_cast<const uint8_t*>(ptr(values)), static_cast<const uint8_t*>(ptr(scales)), block_rows, bias, y, m, n, k) !=
      MDATTN_OK)
    return std::nullopt;
  return y;
}

// RMS norm, with the residual's addition, and the product with a weight that the program keeps quantised: {product} or {product, s}
std::optional<variable_list> rms_norm_linear(const Tensor& x, const Tensor& values, const Tensor& scales, int64_t n, int64_t k, int64_t block_rows,
                                             const OptTensor& bias_, const OptTensor& w_, const OptTensor& b_, const OptTensor& res_, double eps, double offset) {
  const Tensor bias = value(bias_), w = value(w_), b = value(b_), res = value(res_);
  if (!x.is_cuda() || !float_on(x, x) || x.dim() < 1 || x.size(-1) != k || x.numel() == 0 || k <= 0 || n <= 0 || !values.is_cuda() ||
      values.get_device() != x.get_device() || scales.get_device() != x.get_device() || !bias_ok(bias, n, x) || wants_grad({&x, &bias, &w, &b, &res}))
    return std::nullopt;
  at::NoGradGuard guard;
  int64_t stride;
  int f32;
  Rows3 rr;
  const auto r = as_rows(x);
  if (!r || !norm_vectors(x, *r, w, b, stride, f32) || !residual_rows(x, res, rr)) return std::nullopt;
  const int64_t m = r->all(), sg = r->rows * r->c;
  const Blocks q(x, m, k, 1);
  Tensor s = res.defined() ? at::empty(x.sizes(), res.options()) : Tensor();
  if (mdattn_rms_norm_e4m3(stream(x), ptr(x), is_f32(x), ptr(res), is_f32(res), q.values(), q.scales(), mut(s), ptr(w), ptr(b), f32, r->groups, r->rows, (int)r->c,
                           r->sg, r->sr, rr.sg, rr.sr, sg, r->c, stride, (float)eps, (float)offset) != MDATTN_OK)
    return std::nullopt;
  Tensor y = at::empty(with_last(x, n), x.options().dtype(at::kBFloat16));
  if (product(q.values(), q.scales(), static_cast<const uint8_t*>(ptr(values)), static_cast<const uint8_t*>(ptr(scales)), block_rows, bias, y, m, n, k) !=
      MDATTN_OK)
    return std::nullopt;
  return s.defined() ? variable_list{y, s} : variable_list{y};
}

// y = x8 w8^T + b, dx = dy8 w8, dw = dy8'^T x8', ' quantised along the tokens.  Saved: x and w in e4m3, transposed, from one read of each.
struct LinearFn : FirstOrder<LinearFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& bias_) {
    const Tensor bias = value(bias_), rows = as_matrix(x);
    const bool need_dx = x.requires_grad(), need_dw = w.requires_grad(), need_db = bias.defined() && bias.requires_grad();
    const int64_t m = rows.size(0), k = rows.size(1), n = w.size(0);
    const Blocks xq(x, m, k, 1), wq(x, n, k, 128);
    std::optional<Blocks> xt, wt;
    if (need_dw) xt.emplace(x, k, m, 1);
    if (need_dx) wt.emplace(x, k, n, 128);
    if (quant(rows, 1, &xq, xt ? &*xt : nullptr, Tensor()) != MDATTN_OK || quant(w, 128, &wq, wt ? &*wt : nullptr, Tensor()) != MDATTN_OK) throw Refused{};
    Tensor y = at::empty(with_last(x, n), x.options());
    if (product(xq.values(), xq.scales(), wq.values(), wq.scales(), 128, bias, y, m, n, k) != MDATTN_OK) throw Refused{};
    ctx->save_for_backward({xt ? xt->buf : Tensor(), wt ? wt->buf : Tensor()});
    ctx->saved_data["i"] = c10::List<int64_t>({m, n, k, need_dx, need_dw, need_db, is_f32(bias)});
    ctx->saved_data["shape"] = x.sizes().vec();
    return y;
  }
  static variable_list gradients(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const auto i = ctx->saved_data["i"].toIntVector();
    const auto shape = ctx->saved_data["shape"].toIntVector();
    const int64_t m = i[0], n = i[1], k = i[2];
    Tensor g = grads[0];
    if (g.scalar_type() != at::kBFloat16) g = g.to(at::kBFloat16);
    if (g.is_neg()) g = g.resolve_neg();
    Tensor rows = as_matrix(g);
    if (!rows.defined()) rows = as_matrix(g = g.contiguous());
    std::optional<Blocks> xt, wt, gq, gt;
    if (i[4]) xt.emplace(saved[0], k, m, 1, rows);
    if (i[3]) wt.emplace(saved[1], k, n, 128, rows);
    if (i[3] || !i[4]) gq.emplace(rows, m, n, 1);
    if (i[4]) gt.emplace(rows, n, m, 1);
    const Tensor sums = i[5] ? at::empty({(m + 127) / 128, n}, rows.options().dtype(at::kFloat)) : Tensor();
    must(quant(rows, 1, gq ? &*gq : nullptr, gt ? &*gt : nullptr, sums), "mdattn_quant_block_e4m3");
    Tensor dx, dw, db;
    if (i[3]) {
      dx = at::empty(shape, rows.options());
      must(product(gq->values(), gq->scales(), wt->values(), wt->scales(), 128, Tensor(), dx, m, k, n), "mdattn_matmul_fp8_block");
    }
    if (i[4]) {
      dw = at::empty({n, k}, rows.options());
      must(product(gt->values(), gt->scales(), xt->values(), xt->scales(), 1, Tensor(), dw, n, k, m), "mdattn_matmul_fp8_block");
    }
    if (i[5]) {
      db = at::empty({n}, rows.options().dtype(i[6] ? at::kFloat : at::kBFloat16));
      must(mdattn_sum_rows(stream(sums), f32(sums), sums.size(0), n, mut(db), (int)i[6]), "mdattn_sum_rows");
    }
    return {dx, dw, db};
  }
};
OptTensor linear_autograd(const Tensor& x, const Tensor& w, const OptTensor& bias_) {
  const Tensor bias = value(bias_);
  if (!x.is_cuda() || !bf16_on(x, x) || !bf16_on(w, x) || x.dim() < 1 || w.dim() != 2 || x.numel() == 0 || w.numel() == 0 || x.size(-1) != w.size(1) || w.stride(1) != 1 ||
      !bias_ok(bias, w.size(0), x) || !as_matrix(x).defined())
    return std::nullopt;
  return unless_refused([&] { return LinearFn::apply(x, w, bias_); });
}

// the id of the sources, behind the marker that build.py finds in the file (as in libmdattn.so)
const char kBuildIdRecord[] = "mdattn-build-id:" MDATTN_BUILD_ID;

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("build_id", [] { return std::string(kBuildIdRecord + 16); });
  // Other Python threads run meanwhile, as they do during a call through ctypes: a launch may wait for room in its queue, an
  // allocation for memory.
  using Unlocked = py::call_guard<py::gil_scoped_release>;
  m.def("flash", &flash, Unlocked());
  m.def("flash_autograd", &flash_autograd, Unlocked());
  m.def("flash_fp8", &flash_fp8, Unlocked());
  m.def("flash_merge", &flash_merge, Unlocked());
  m.def("flash_packed", &flash_packed, Unlocked());
  m.def("norm_rope", &norm_rope, Unlocked());
  m.def("norm_rope_perhead", &norm_rope_perhead, Unlocked());
  m.def("norm_rope_qkv", &norm_rope_qkv, Unlocked());
  m.def("norm_rope_rows", &norm_rope_rows, Unlocked());
  m.def("layer_norm", &layer_norm, Unlocked());
  m.def("linear_quantized", &linear_quantized, Unlocked());
  m.def("rms_norm", &rms_norm, Unlocked());
  m.def("rms_norm_linear", &rms_norm_linear, Unlocked());
  m.def("first_order", [](const std::vector<OptTensor>& grads, const std::vector<OptTensor>& results) {
    variable_list g, r;
    for (const auto& t : grads) g.push_back(value(t));
    for (const auto& t : results) r.push_back(value(t));
    std::vector<OptTensor> out;
    for (const Tensor& t : first_order(g, std::move(r))) out.push_back(opt(t));
    return out;
  });
  m.def("linear_autograd", &linear_autograd, Unlocked());
}
