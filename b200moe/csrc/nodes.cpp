// Autograd nodes of the training step in C++: embedding, norm, the attention half of a block, the routed layer on one rank, the
// LM head with its loss, routing, the gated residual norm and the linear layer in 8 bits.  They do what the nodes of the same name in b200moe/ops do from Python, with the same kernels in
// the same order: what they save is the host's time, 20-30 us per launch and 30 per node of the backward pass (from Python's
// second thread), which is what a small layer costs.  A step of two blocks of width 512 took 4.7 ms for 1.5 ms of kernels.
//
// The functions at the end answer None where an operand is not what the node takes (type, layout, alignment, device); the
// caller then goes the general way.  Kernels come from the library that b200moe.ops.native has loaded (``bind``).
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/extension.h>

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cmath>

#include "entries.h"

using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;
using Tensor = at::Tensor;
using Optional = std::optional<Tensor>;

namespace {

std::atomic<long long> launches{0};

struct Library {
  decltype(&b2_layers_refused) layers_refused;
  decltype(&b2_attn_half_fwd) attn_half_fwd;
  decltype(&b2_attn_half_bwd) attn_half_bwd;
  decltype(&b2_moe_layer_fwd) moe_layer_fwd;
  decltype(&b2_moe_experts_bwd) moe_experts_bwd;
  decltype(&b2_moe_router_bwd) moe_router_bwd;
  decltype(&b2_moe_aux) moe_aux;
  decltype(&b2_rmsnorm_fwd) rmsnorm_fwd;
  decltype(&b2_rmsnorm_bwd) rmsnorm_bwd;
  decltype(&b2_rmsnorm_bwd_parts) rmsnorm_bwd_parts;
  decltype(&b2_swiglu_bwd_in_product) swiglu_bwd_in_product;
  decltype(&b2_head_chunk) head_chunk;
  decltype(&b2_scale_bf16) scale_bf16;
  decltype(&b2_embedding_fwd) embedding_fwd;
  decltype(&b2_embedding_bwd) embedding_bwd;
  decltype(&b2_gemm_tn) gemm_tn;
  decltype(&b2_route_topk) route_topk;
  decltype(&b2_route_topk_bwd) route_topk_bwd;
  decltype(&b2_gated_norm_fwd) gated_norm_fwd;
  decltype(&b2_gated_norm_bwd) gated_norm_bwd;
  decltype(&b2_gated_norm_bwd_floats) gated_norm_bwd_floats;
  decltype(&b2_quantize_fp8) quantize_fp8;
  decltype(&b2_gemm_fp8) gemm_fp8;
} lib;

void bind(const std::string& path) {
  void* const handle = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);
  TORCH_CHECK(handle, "cannot load ", path, ": ", dlerror());
  auto resolve = [&](auto& entry, const char* name) {
    void* const symbol = dlsym(handle, name);
    TORCH_CHECK(symbol, path, " has no ", name);
    entry = reinterpret_cast<std::remove_reference_t<decltype(entry)>>(symbol);
  };
  resolve(lib.layers_refused, "b2_layers_refused");
  resolve(lib.attn_half_fwd, "b2_attn_half_fwd");
  resolve(lib.attn_half_bwd, "b2_attn_half_bwd");
  resolve(lib.moe_layer_fwd, "b2_moe_layer_fwd");
  resolve(lib.moe_experts_bwd, "b2_moe_experts_bwd");
  resolve(lib.moe_router_bwd, "b2_moe_router_bwd");
  resolve(lib.moe_aux, "b2_moe_aux");
  resolve(lib.rmsnorm_fwd, "b2_rmsnorm_fwd");
  resolve(lib.rmsnorm_bwd, "b2_rmsnorm_bwd");
  resolve(lib.rmsnorm_bwd_parts, "b2_rmsnorm_bwd_parts");
  resolve(lib.swiglu_bwd_in_product, "b2_swiglu_bwd_in_product");
  resolve(lib.head_chunk, "b2_head_chunk");
  resolve(lib.scale_bf16, "b2_scale_bf16");
  resolve(lib.embedding_fwd, "b2_embedding_fwd");
  resolve(lib.embedding_bwd, "b2_embedding_bwd");
  resolve(lib.gemm_tn, "b2_gemm_tn");
  resolve(lib.route_topk, "b2_route_topk");
  resolve(lib.route_topk_bwd, "b2_route_topk_bwd");
  resolve(lib.gated_norm_fwd, "b2_gated_norm_fwd");
  resolve(lib.gated_norm_bwd, "b2_gated_norm_bwd");
  resolve(lib.gated_norm_bwd_floats, "b2_gated_norm_bwd_floats");
  resolve(lib.quantize_fp8, "b2_quantize_fp8");
  resolve(lib.gemm_fp8, "b2_gemm_fp8");
}

cudaStream_t stream() { return c10::cuda::getCurrentCUDAStream().stream(); }
// Raises what b200moe.ops.native raises for a refused launch; ``name``: its entry point, null for a sequence of layers.cu.
void check(int code, const char* name, int count) {
  if (code != 0) {
    if (!name) name = lib.layers_refused();
    std::string detail;
    try {
      pybind11::gil_scoped_acquire gil;
      detail = pybind11::module_::import("b200moe.ops.native").attr("_failure_detail")(name, code).cast<std::string>();
    } catch (pybind11::error_already_set&) {      // the code alone, then
    }
    TORCH_CHECK(false, name, " failed with code ", code, detail);
  }
  launches += count;
}
// Addresses as the entry points type them; the tensors' types have been looked at by then.
struct Const {
  const void* at;
  template <typename T> operator const T*() const { return static_cast<const T*>(at); }
};
struct Mutable {
  void* at;
  template <typename T> operator T*() const { return static_cast<T*>(at); }
};
Const ptr(const Tensor& t) { return {t.defined() ? t.const_data_ptr() : nullptr}; }
Mutable mut(const Tensor& t) { return {t.defined() ? t.data_ptr() : nullptr}; }
Tensor fp32(at::IntArrayRef sizes, const Tensor& like) { return at::empty(sizes, like.options().dtype(at::kFloat)); }
Tensor bf16(at::IntArrayRef sizes, const Tensor& like) { return at::empty(sizes, like.options().dtype(at::kBFloat16)); }
Tensor int32(at::IntArrayRef sizes, const Tensor& like) { return at::empty(sizes, like.options().dtype(at::kInt)); }

bool aligned(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0; }
bool plain(const Tensor& t, at::ScalarType type, const Tensor& beside) {
  return t.scalar_type() == type && t.is_contiguous() && t.device() == beside.device() && aligned(t);
}
// A bf16 weight and the buffer that its gradient is added to.
bool trained(const Tensor& weight, const Tensor& grad, const Tensor& beside) {
  return plain(weight, at::kBFloat16, beside) && plain(grad, at::kFloat, beside) && grad.sizes() == weight.sizes();
}
bool follows(std::initializer_list<Tensor> inputs) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor& t : inputs)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}
// Scratch of one call, ``bytes`` per buffer (0: null).  Small calls take it as one allocation (1.3 us each); large ones buffer by
// buffer, as blocks that the allocator has use for elsewhere.
class Scratch {
 public:
  static constexpr int64_t TOGETHER = 16 << 20;
  Scratch(const Tensor& like, std::initializer_list<int64_t> bytes) {
    int64_t total = 0;
    for (int64_t b : bytes) total += (b + 255) / 256 * 256;
    const bool together = total <= TOGETHER;
    const auto options = like.options().dtype(at::kByte);
    if (together) held_.push_back(at::empty({total}, options));
    char* next = together ? static_cast<char*>(held_[0].data_ptr()) : nullptr;
    for (int64_t b : bytes) {
      if (together) {
        at_.push_back(b ? next : nullptr);
        next += (b + 255) / 256 * 256;
      } else {
        held_.push_back(b ? at::empty({b}, options) : Tensor());
        at_.push_back(mut(held_.back()).at);
      }
    }
  }
  Mutable operator[](size_t i) const { return {at_[i]}; }

 private:
  std::vector<Tensor> held_;
  std::vector<void*> at_;
};

// Where the gradient of a weight goes in a backward pass: the buffer that the weight carries then (its ``main_grad``; as in the
// Python nodes, one that took the place of the forward pass's is followed).  A buffer that the kernels do not take, or none,
// gets the sum afterwards.
class Gradient {
 public:
  Gradient(const Tensor& weight, const Tensor& buffer, at::ScalarType kind) : weight_(weight), buffer_(buffer) {
    const bool direct = buffer_.defined() && plain(buffer_, kind, weight) && buffer_.sizes() == weight.sizes();
    sum_ = direct ? buffer_ : at::zeros(weight.sizes(), weight.options().dtype(kind).requires_grad(false));
  }
  Mutable operator*() const { return {sum_.data_ptr()}; }
  // What autograd is told: nothing where there is a buffer.
  Tensor given() {
    if (buffer_.is_same(sum_)) return Tensor();
    if (buffer_.defined()) {
      buffer_.add_(sum_);
      return Tensor();
    }
    return weight_.requires_grad() ? sum_.to(weight_.scalar_type()) : Tensor();
  }
  // The buffers that ``count`` weights carry.
  static std::vector<Tensor> of(const std::vector<Tensor>& weights, size_t count) {
    std::vector<Tensor> buffers(count);
    pybind11::gil_scoped_acquire gil;
    static PyObject* const name = PyUnicode_InternFromString("main_grad");
    for (size_t i = 0; i < count; ++i) {
      const auto object = pybind11::reinterpret_steal<pybind11::object>(THPVariable_Wrap(weights[i]));
      const auto buffer = pybind11::reinterpret_steal<pybind11::object>(PyObject_GetAttr(object.ptr(), name));
      if (!buffer) PyErr_Clear();
      else if (THPVariable_Check(buffer.ptr())) buffers[i] = THPVariable_Unpack(buffer.ptr());
    }
    return buffers;
  }

 private:
  Tensor weight_, buffer_, sum_;
};

// What a node keeps beside the saved tensors: weights, as the Python nodes keep them.
void keep(AutogradContext* ctx, std::vector<Tensor> tensors) { ctx->saved_data["kept"] = std::move(tensors); }
std::vector<Tensor> kept(AutogradContext* ctx) { return ctx->saved_data["kept"].toTensorVector(); }

struct Embedding : public Function<Embedding> {
  static Tensor forward(AutogradContext* ctx, const Tensor& ids, const Tensor& table) {
    ctx->save_for_backward({ids});
    keep(ctx, {table});
    std::vector<int64_t> sizes = ids.sizes().vec();
    sizes.push_back(table.size(1));
    Tensor out = bf16(sizes, table);
    check(lib.embedding_fwd(ptr(ids), ptr(table), mut(out), ids.numel(), table.size(1), stream()), "b2_embedding_fwd", 1);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor ids = ctx->get_saved_variables()[0], dy = grads[0].contiguous();
    const std::vector<Tensor> w = kept(ctx);
    TORCH_CHECK(dy.scalar_type() == at::kBFloat16, "expected bfloat16, got ", dy.scalar_type());
    Gradient grad(w[0], Gradient::of(w, 1)[0], at::kFloat);
    check(lib.embedding_bwd(ptr(ids), ptr(dy), *grad, ids.numel(), w[0].size(1), stream()), "b2_embedding_bwd", 1);
    return {Tensor(), grad.given()};
  }
};

struct RMSNorm : public Function<RMSNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, double eps, const Tensor& status) {
    const int D = x.size(-1), rows = x.numel() / D;
    Tensor y = at::empty_like(x), rstd = fp32({rows}, x);
    check(lib.rmsnorm_fwd(ptr(x), nullptr, ptr(weight), nullptr, mut(y), mut(rstd), rows, D, eps, mut(status), stream()),
          "b2_rmsnorm_fwd", 1);
    ctx->save_for_backward({x, weight, rstd});
    keep(ctx, {status});
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1], &rstd = saved[2];
    const Tensor dy = grads[0].contiguous(), status = kept(ctx)[0];
    const int D = x.size(-1), rows = x.numel() / D;
    TORCH_CHECK(dy.scalar_type() == at::kBFloat16, "expected bfloat16, got ", dy.scalar_type());
    Tensor dx = at::empty_like(x), dw = fp32({D}, x), partial = fp32({lib.rmsnorm_bwd_parts(rows, D), D}, x);
    check(lib.rmsnorm_bwd(ptr(dy), ptr(x), ptr(weight), ptr(rstd), nullptr, mut(dx), mut(partial), mut(dw), rows, D, mut(status),
                          stream()), "b2_rmsnorm_bwd", 2);
    return {dx, dw, Tensor(), Tensor()};
  }
};

struct AttnHalf : public Function<AttnHalf> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& ln1, const Tensor& wqkv,
                               const Tensor& cos, const Tensor& sin, const Tensor& wo, const Tensor& ln2, const Tensor& status,
                               int64_t hq, int64_t hkv, double eps1, double eps2) {
    const int B = x.size(0), S = x.size(1);
    const int64_t T = x.size(0) * x.size(1);
    Tensor n1 = at::empty_like(x), a = at::empty_like(x), proj = at::empty_like(x), sum = at::empty_like(x), n2 = at::empty_like(x);
    Tensor qkv = bf16({T, 128 * (hq + 2 * hkv)}, x), stats = fp32({T * (2 + hq)}, x);
    check(lib.attn_half_fwd(ptr(x), ptr(ln1), ptr(wqkv), ptr(cos), ptr(sin), ptr(wo), ptr(ln2), mut(n1), mut(qkv), mut(a),
                            mut(proj), mut(sum), mut(n2), mut(stats), B, S, hq, hkv, eps1, eps2, mut(status), stream()),
          nullptr, 5);
    ctx->save_for_backward({x, ln1, ln2, cos, sin, n1, qkv, a, sum, stats});
    keep(ctx, {wqkv, wo, status});
    ctx->saved_data["heads"] = hq * 4096 + hkv;
    return {sum, n2};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &ln1 = saved[1], &ln2 = saved[2], &cos = saved[3], &sin = saved[4], &n1 = saved[5],
                 &qkv = saved[6], &a = saved[7], &sum = saved[8], &stats = saved[9];
    const std::vector<Tensor> w = kept(ctx);
    const int64_t heads = ctx->saved_data["heads"].toInt(), hq = heads / 4096, hkv = heads % 4096;
    const int B = x.size(0), S = x.size(1), D = x.size(2);
    const int64_t T = x.size(0) * x.size(1);
    const Tensor dsum = grads[0].contiguous(), dn2 = grads[1].contiguous();
    TORCH_CHECK(dsum.scalar_type() == at::kBFloat16 && dn2.scalar_type() == at::kBFloat16, "expected bfloat16 gradients");
    // The gradient of the first norm's output takes the place of the attention output's, which is used up by then, and dx that
    // of the sum's, which the first norm's kernel adds row by row before it stores the row: as much as the separate nodes hold.
    Tensor dx = at::empty_like(x), dln1 = fp32({D}, x), dln2 = fp32({D}, x);
    // da, dqkv, the norms' partial sums, the attention's row statistics
    const Scratch tmp(x, {2 * T * D, 2 * qkv.numel(), int64_t{4} * lib.rmsnorm_bwd_parts(T, D) * D, 8 * T * hq});
    const std::vector<Tensor> buffers = Gradient::of(w, 2);
    Gradient gqkv(w[0], buffers[0], at::kFloat), go(w[1], buffers[1], at::kFloat);
    check(lib.attn_half_bwd(ptr(dsum), ptr(dn2), ptr(x), ptr(ln1), ptr(w[0]), ptr(cos), ptr(sin), ptr(w[1]), ptr(ln2), ptr(n1),
                            ptr(qkv), ptr(a), ptr(sum), ptr(stats), *gqkv, *go, mut(dln1), mut(dln2), mut(dx), mut(dx), tmp[0],
                            tmp[0], tmp[1], tmp[2], tmp[3], B, S, hq, hkv, mut(w[2]), stream()),
          nullptr, 11);
    const Tensor none;
    return {dx, dln1, gqkv.given(), none, none, go.given(), dln2, none, none, none, none, none};
  }
};

struct MoELayer : public Function<MoELayer> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& router, const Tensor& w1, const Tensor& w3,
                               const Tensor& w2, const Optional& residual, const Tensor& status, int64_t cap, bool keeps,
                               bool balance) {
    ctx->set_materialize_grads(false);
    const int64_t D = x.size(-1), T = x.numel() / D, E = w1.size(0), F = w1.size(1);
    Tensor weights = fp32({T, 2}, x), probs = fp32({T, E}, x), idx = at::empty({T, 2}, x.options().dtype(at::kLong));
    Tensor tables = int32({2 * T + cap + 2 * E + cap / 128 + 4}, x);
    Tensor x_perm = bf16({cap, D}, x), y_perm = bf16({cap, D}, x), h = bf16({cap, F}, x), out = at::empty_like(x), gate, up;
    if (keeps) gate = at::empty_like(h), up = at::empty_like(h);
    check(lib.moe_layer_fwd(ptr(x), ptr(router), ptr(w1), ptr(w3), ptr(w2), ptr(residual ? *residual : Tensor()), mut(weights),
                            mut(idx), mut(probs), mut(tables), mut(x_perm), mut(h), mut(gate), mut(up), mut(y_perm), mut(out), T, D,
                            F, E, cap, mut(status), stream()), nullptr, 6);
    variable_list saved = {x, weights, idx, probs, tables, x_perm, y_perm};
    if (keeps) saved.insert(saved.end(), {gate, up});
    ctx->save_for_backward(std::move(saved));
    keep(ctx, {router, w1, w3, w2, status});
    ctx->saved_data["residual"] = residual.has_value();
    if (!balance) return {out};
    Tensor aux = fp32({}, x);
    check(lib.moe_aux(ptr(probs), tables.const_data_ptr<int>() + tables.numel() - E, mut(aux), T, E, stream()), "b2_moe_aux", 1);
    return {out, aux};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weights = saved[1], &idx = saved[2], &probs = saved[3], &tables = saved[4], &x_perm = saved[5],
                 &y_perm = saved[6];
    const std::vector<Tensor> w = kept(ctx);
    const int64_t D = x.size(-1), T = x.numel() / D, E = w[1].size(0), F = w[1].size(1), cap = x_perm.size(0);
    const bool rebuild = saved.size() < 9;
    const Tensor dout = grads[0].defined() ? grads[0].contiguous() : at::zeros_like(x);
    TORCH_CHECK(dout.scalar_type() == at::kBFloat16, "expected bfloat16, got ", dout.scalar_type());
    Tensor daux = grads.size() > 1 && grads[1].defined() ? grads[1].to(x.device(), at::kFloat) : Tensor();
    const int64_t row = 2 * cap * D, wide = 2 * cap * F;
    const bool own = !lib.swiglu_bwd_in_product(cap, F, D);      // the SwiGLU backward is a kernel of its own
    const std::vector<Tensor> buffers = Gradient::of(w, 4);
    const at::ScalarType kind = buffers[1].defined() && buffers[1].scalar_type() == at::kBFloat16 ? at::kBFloat16 : at::kFloat;
    Gradient grouter(w[0], buffers[0], at::kFloat), g1(w[1], buffers[1], kind), g3(w[2], buffers[2], kind), g2(w[3], buffers[3], kind);
    // dx_perm takes the place of what is used up by then: dh, and gate and up where they are formed again.  dweights, dlogits.
    // Behind them dy_perm, dgu and h, which large calls hold no longer than the experts need them.
    const int64_t used_bytes = std::max(row, (own + 2 * rebuild) * wide);
    const int64_t few = used_bytes + row + 3 * wide <= Scratch::TOGETHER;
    const Scratch tmp(x, {used_bytes, 8 * T, 4 * T * E, few * row, few * 2 * wide, few * wide});
    char* const used = tmp[0];
    char* const formed = used + own * wide;
    {
      std::optional<Scratch> large;
      if (!few) large.emplace(x, std::initializer_list<int64_t>{row, 2 * wide, wide});
      const auto inner = [&](size_t i) { return few ? tmp[3 + i] : (*large)[i]; };
      check(lib.moe_experts_bwd(ptr(dout), ptr(w[1]), ptr(w[2]), ptr(w[3]), ptr(weights), mut(tables), ptr(x_perm), ptr(y_perm),
                                rebuild ? formed : mut(saved[7]).at, rebuild ? formed + wide : mut(saved[8]).at, rebuild, *g1, *g3,
                                *g2, kind == at::kFloat ? 1 : 2, inner(0), inner(1), inner(2), own ? used : nullptr, used, tmp[1],
                                T, D, F, E, cap, mut(w[4]), stream()), nullptr, 5 + own + rebuild);
    }
    Tensor dx = at::empty_like(x);
    check(lib.moe_router_bwd(ptr(x), ptr(w[0]), ptr(weights), ptr(idx), ptr(probs), mut(tables), ptr(daux), *grouter, used, tmp[1],
                             tmp[2], mut(dx), T, D, E, cap, stream()), nullptr, 2);
    const Tensor none;
    return {dx, grouter.given(), g1.given(), g3.given(), g2.given(), ctx->saved_data["residual"].toBool() ? grads[0] : none,
            none, none, none, none};
  }
};

// The head where the factor that will be back-propagated into the loss is known: b200moe/ops/loss.py.
struct Head : public Function<Head> {
  static Tensor forward(AutogradContext* ctx, const Tensor& hidden, const Tensor& weight, const Tensor& targets, const Tensor& grad,
                        double scale, int64_t chunk, const Tensor& status) {
    const int64_t V = weight.size(0), D = weight.size(1), T = hidden.numel() / D;
    Tensor loss = at::zeros({}, hidden.options().dtype(at::kDouble)), dh = at::empty_like(hidden);
    for (int64_t lo = 0; lo < T; lo += chunk) {
      const int64_t n = std::min(chunk, T - lo);
      Tensor logits = bf16({n, V}, hidden);
      check(lib.head_chunk(static_cast<const char*>(ptr(hidden).at) + 2 * lo * D, ptr(weight),
                           static_cast<const long long*>(ptr(targets)) + lo, mut(logits), mut(loss),
                           static_cast<char*>(mut(dh).at) + 2 * lo * D, mut(grad), n, V, D, 1.0 / T, scale / T, mut(status),
                           stream()),
            nullptr, 4);
    }
    ctx->save_for_backward({dh});
    ctx->saved_data["scale"] = scale;
    return loss.to(at::kFloat);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    Tensor dh = ctx->get_saved_variables()[0];
    if (torch::autograd::get_current_graph_task_keep_graph()) dh = dh.clone();
    const Tensor factor = (grads[0] / ctx->saved_data["scale"].toDouble()).to(dh.device(), at::kFloat);
    check(lib.scale_bf16(mut(dh), ptr(factor), dh.numel(), stream()), "b2_scale_bf16", 1);
    const Tensor none;
    return {dh, none, none, none, none, none, none};
  }
};

// Type of the kernels that take fp32, bf16 and fp16; -1 for others.
int float_type(const Tensor& t) {
  return t.scalar_type() == at::kFloat ? 0 : t.scalar_type() == at::kBFloat16 ? 1 : t.scalar_type() == at::kHalf ? 2 : -1;
}
// Gradients that cannot be differentiated again: where a graph of them is asked for, using it raises (as once_differentiable does for
// the nodes in Python).
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list defined;
  for (const Tensor& g : grads)
    if (g.defined()) defined.push_back(g.detach().requires_grad_(true));
  auto refuse = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that was marked with @once_differentiable", static_cast<int64_t>(defined.size()));
  defined = (*refuse)(std::move(defined));
  size_t i = 0;
  for (Tensor& g : grads)
    if (g.defined()) g = defined[i++];
  return grads;
}

struct RouteTopk : public Function<RouteTopk> {
  // weights and idx
  static variable_list run(const Tensor& logits, const Optional& bias, int64_t k, bool sigmoid, int64_t groups, int64_t top_groups,
                           bool two_best, bool renormalize, double scale) {
    const c10::cuda::CUDAGuard guard(logits.device());
    const int64_t T = logits.size(0), E = logits.size(1);
    Tensor weights = fp32({T, k}, logits), idx = at::empty({T, k}, logits.options().dtype(at::kLong));
    check(lib.route_topk(ptr(logits), ptr(bias ? *bias : Tensor()), mut(weights), mut(idx), T, E, k, float_type(logits), sigmoid,
                         groups, top_groups, two_best, renormalize, scale, stream()), "b2_route_topk", 1);
    return {weights, idx};
  }
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Optional& bias, int64_t k, bool sigmoid,
                               int64_t groups, int64_t top_groups, bool two_best, bool renormalize, double scale) {
    ctx->set_materialize_grads(false);
    variable_list out = run(logits, bias, k, sigmoid, groups, top_groups, two_best, renormalize, scale);
    ctx->mark_non_differentiable({out[1]});
    ctx->save_for_backward({logits, out[0], out[1]});
    ctx->saved_data["how"] = int64_t{sigmoid} + 2 * renormalize;
    ctx->saved_data["scale"] = scale;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(9);
    if (!grads[0].defined()) return out;
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &logits = saved[0], &weights = saved[1], &idx = saved[2], dweights = grads[0].contiguous();
    const c10::cuda::CUDAGuard guard(logits.device());
    const int64_t how = ctx->saved_data["how"].toInt();
    out[0] = at::empty_like(logits);
    check(lib.route_topk_bwd(ptr(logits), ptr(weights), ptr(idx), ptr(dweights), mut(out[0]), logits.size(0), logits.size(1),
                             idx.size(1), float_type(logits), how & 1, how >> 1, ctx->saved_data["scale"].toDouble(), stream()),
          "b2_route_topk_bwd", 1);
    return once(std::move(out));
  }
};

struct GatedNorm : public Function<GatedNorm> {
  // the sum, its norm, and 1 / rms of delta and of the sum
  static variable_list run(const Tensor& x, const Tensor& delta, const Tensor& wd, const Tensor& w, const Optional& gate,
                           int64_t kind, int64_t seq, double scale, double eps, const Tensor& status) {
    const c10::cuda::CUDAGuard guard(x.device());
    const int64_t D = x.size(-1), rows = x.numel() / D;
    Tensor summed = at::empty_like(x), normed = at::empty_like(x), stats = fp32({2 * rows}, x);
    float* const rstd = mut(stats);
    check(lib.gated_norm_fwd(ptr(x), ptr(delta), ptr(wd), ptr(w), ptr(gate ? *gate : Tensor()), mut(summed), mut(normed), rstd,
                             rstd + rows, rows, D, seq, float_type(x), kind, gate && gate->scalar_type() == at::kFloat, scale, eps,
                             mut(status), stream()), "b2_gated_norm_fwd", 1);
    return {summed, normed, stats};
  }
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& delta, const Tensor& wd, const Tensor& w,
                               const Optional& gate, int64_t kind, int64_t seq, double scale, double eps, const Tensor& status) {
    ctx->set_materialize_grads(false);
    variable_list out = run(x, delta, wd, w, gate, kind, seq, scale, eps, status);
    ctx->save_for_backward({x, delta, wd, w, gate ? *gate : Tensor(), out[2]});
    keep(ctx, {status});
    ctx->saved_data["kind"] = kind;
    ctx->saved_data["seq"] = seq;
    ctx->saved_data["scale"] = scale;
    out.pop_back();
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(10);
    if (!grads[0].defined() && !grads[1].defined()) return out;
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &delta = saved[1], &wd = saved[2], &w = saved[3], &gate = saved[4], &stats = saved[5];
    const c10::cuda::CUDAGuard guard(x.device());
    const int64_t D = x.size(-1), rows = x.numel() / D, kind = ctx->saved_data["kind"].toInt(), seq = ctx->saved_data["seq"].toInt();
    const Tensor ds = grads[0].defined() ? grads[0].contiguous() : Tensor(), dy = grads[1].defined() ? grads[1].contiguous() : Tensor();
    const Tensor status = kept(ctx)[0];
    Tensor dx = at::empty_like(x), ddelta = at::empty_like(x), dwd = fp32({D}, x), dw = fp32({D}, x), dgate;
    if (gate.defined()) dgate = at::empty_like(gate);
    const Tensor partial = fp32({lib.gated_norm_bwd_floats(rows, D, seq, kind)}, x);
    const float* const rstd = ptr(stats);
    check(lib.gated_norm_bwd(ptr(ds), ptr(dy), ptr(x), ptr(delta), ptr(wd), ptr(w), ptr(gate), rstd, rstd + rows, mut(dx),
                             mut(ddelta), mut(dwd), mut(dw), mut(dgate), mut(partial), rows, D, seq, float_type(x), kind,
                             gate.defined() && gate.scalar_type() == at::kFloat, ctx->saved_data["scale"].toDouble(), mut(status),
                             stream()), "b2_gated_norm_bwd", 2);
    out[0] = dx, out[1] = ddelta, out[2] = dwd, out[3] = dw, out[4] = dgate;
    return once(std::move(out));
  }
};

// e4m3 values by rows of 128 and their scales, in scratch memory of the call.
struct Rows8 {
  Rows8(const Tensor& x, int64_t rows, int64_t cols)
      : rows(rows), cols(cols), pitch((cols + 15) / 16 * 16), held(x, {rows * pitch, 4 * rows * ((cols + 127) / 128)}) {
    check(lib.quantize_fp8(ptr(x), float_type(x), held[0], held[1], rows, cols, cols, pitch, rows, 1, stream()), "b2_quantize_fp8", 1);
  }
  // times w [N, K] transposed, or (nn) times w [K, N]
  void times(const Tensor& w, const Tensor& scales, bool nn, const Tensor& out, const Tensor& status) const {
    check(lib.gemm_fp8(held[0], held[1], ptr(w), ptr(scales), mut(out), rows, nn ? w.size(1) : w.size(0), cols, pitch, w.stride(0), 1,
                       rows, scales.stride(nn), scales.stride(!nn), nn, mut(status), stream()), "b2_gemm_fp8", 1);
  }
  int64_t rows, cols, pitch;
  Scratch held;
};

struct LinearFp8 : public Function<LinearFp8> {
  static Tensor run(const Tensor& x, const Tensor& weight, const Tensor& values, const Tensor& scales, const Tensor& status) {
    const c10::cuda::CUDAGuard guard(x.device());
    const int64_t K = weight.size(1), N = weight.size(0), rows = x.numel() / K;
    std::vector<int64_t> sizes = x.sizes().vec();
    sizes.back() = N;
    Tensor y = bf16(sizes, x);
    Rows8(x, rows, K).times(values, scales, false, y, status);
    return y;
  }
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Tensor& values, const Tensor& scales,
                        const Tensor& status) {
    Tensor y = run(x, weight, values, scales, status);
    ctx->save_for_backward({x, values, scales});
    keep(ctx, {weight, status});
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &values = saved[1], &scales = saved[2], dy = grads[0].contiguous();
    const std::vector<Tensor> w = kept(ctx);
    const c10::cuda::CUDAGuard guard(x.device());
    const int64_t K = w[0].size(1), N = w[0].size(0), rows = x.numel() / K;
    TORCH_CHECK(dy.scalar_type() == at::kBFloat16, "expected bfloat16, got ", dy.scalar_type());
    const Tensor dy16 = aligned(dy) ? dy : dy.clone();
    Tensor dx, dw;
    if (ctx->needs_input_grad(0)) {
      dx = at::empty_like(x);
      Rows8(dy16, rows, N).times(values, scales, true, dx, w[1]);
    }
    const Tensor buffer = Gradient::of(w, 1)[0];
    if (buffer.defined() || w[0].requires_grad()) {
      const bool direct = buffer.defined() && plain(buffer, at::kFloat, x) && buffer.sizes() == w[0].sizes();
      Tensor sum = direct ? buffer : at::empty(w[0].sizes(), w[0].options().requires_grad(false).dtype(buffer.defined() ? at::kFloat : w[0].scalar_type()));
      check(lib.gemm_tn(ptr(dy16), ptr(x), mut(sum), nullptr, 0, N, K, rows, N, K, K, 1, nullptr, nullptr,
                        sum.scalar_type() == at::kFloat ? 1 : 2, direct ? 1.f : 0.f, nullptr, mut(w[1]), stream()), "b2_gemm_tn", 1);
      if (!buffer.defined()) dw = sum;
      else if (!direct) buffer.add_(sum);
    }
    return once({dx, dw, Tensor(), Tensor(), Tensor()});
  }
};

// ------------------------------------------------------------------ entry points
Optional embedding(const Tensor& ids, const Tensor& table, const Tensor& grad) {
  if (!(ids.scalar_type() == at::kLong && ids.is_contiguous() && ids.numel() > 0 && ids.numel() < INT_MAX && table.dim() == 2 &&
        table.size(1) % 8 == 0 && table.is_cuda() && ids.device() == table.device() && trained(table, grad, table)))
    return std::nullopt;
  return Embedding::apply(ids, table);
}

Optional rmsnorm(const Tensor& x, const Tensor& weight, double eps, const Tensor& status) {
  if (!(x.is_cuda() && x.dim() > 0 && x.numel() > 0 && plain(x, at::kBFloat16, x) && weight.dim() == 1 &&
        weight.size(0) == x.size(-1) && plain(weight, at::kFloat, x) && x.size(-1) % 8 == 0 && x.size(-1) <= 8192 &&
        x.numel() / x.size(-1) < INT_MAX))
    return std::nullopt;
  return RMSNorm::apply(x, weight, eps, status);
}

std::optional<variable_list> attn_half(const Tensor& x, const Tensor& ln1, const Tensor& wqkv, const Tensor& gqkv, const Tensor& cos,
                                       const Tensor& sin, const Tensor& wo, const Tensor& go, const Tensor& ln2,
                                       const Tensor& status, int64_t hq, int64_t hkv, double eps1, double eps2) {
  if (!(x.is_cuda() && x.dim() == 3 && x.numel() > 0 && plain(x, at::kBFloat16, x))) return std::nullopt;
  const int64_t S = x.size(1), D = x.size(2);
  if (!(S % 128 == 0 && D == 128 * hq && D <= 8192 && hkv > 0 && hq % hkv == 0 && x.size(0) * S * (hq + 2 * hkv) < INT_MAX / 128 &&
        wqkv.dim() == 2 && wqkv.size(0) == 128 * (hq + 2 * hkv) && wqkv.size(1) == D && trained(wqkv, gqkv, x) && wo.dim() == 2 &&
        wo.size(0) == D && wo.size(1) == D && trained(wo, go, x)))
    return std::nullopt;
  for (const Tensor& gain : {ln1, ln2})
    if (!(gain.dim() == 1 && gain.size(0) == D && plain(gain, at::kFloat, x))) return std::nullopt;
  for (const Tensor& table : {cos, sin})
    if (!(table.dim() == 2 && table.size(1) == 64 && table.size(0) >= S && plain(table, at::kFloat, x))) return std::nullopt;
  return AttnHalf::apply(x, ln1, wqkv, cos, sin, wo, ln2, status, hq, hkv, eps1, eps2);
}

std::optional<variable_list> moe_layer(const Tensor& x, const Tensor& router, const Tensor& w1, const Tensor& w3, const Tensor& w2,
                                       const Optional& residual, const Tensor& grouter, const Tensor& g1, const Tensor& g3,
                                       const Tensor& g2, const Tensor& status, int64_t align, bool recompute, bool balance) {
  if (!(x.is_cuda() && x.dim() >= 2 && x.numel() > 0 && plain(x, at::kBFloat16, x) && router.dim() == 2 && w1.dim() == 3))
    return std::nullopt;
  const int64_t E = w1.size(0), F = w1.size(1), D = x.size(-1), T = x.numel() / D;
  if (!(E >= 2 && E <= 16 && D % 64 == 0 && F % 128 == 0 && router.size(0) == E && router.size(1) == D && w1.size(2) == D &&
        w3.sizes() == w1.sizes() && w2.dim() == 3 && w2.size(0) == E && w2.size(1) == D && w2.size(2) == F &&
        E * D * 2 <= 200 * 1024 && T < (1 << 28) && trained(router, grouter, x)))
    return std::nullopt;
  const at::ScalarType kind = g1.scalar_type();
  if (kind != at::kFloat && kind != at::kBFloat16) return std::nullopt;
  const std::pair<const Tensor&, const Tensor&> experts[] = {{w1, g1}, {w3, g3}, {w2, g2}};
  for (const auto& [weight, grad] : experts)
    if (!(plain(weight, at::kBFloat16, x) && plain(grad, kind, x) && grad.sizes() == weight.sizes())) return std::nullopt;
  if (residual && !(plain(*residual, at::kBFloat16, x) && residual->sizes() == x.sizes())) return std::nullopt;
  const bool keeps = !recompute && follows({x, router, w1, w3, w2, residual ? *residual : Tensor()});
  const int64_t cap = (2 * T + E * (align - 1) + align - 1) / align * align;      // moe_fused.capacity_rows
  return MoELayer::apply(x, router, w1, w3, w2, residual, status, cap, keeps, balance);
}

Optional head(const Tensor& hidden, const Tensor& weight, const Tensor& targets, const Tensor& grad, double scale, int64_t chunk,
              const Tensor& status) {
  if (!(hidden.is_cuda() && hidden.dim() > 0 && hidden.numel() > 0 && plain(hidden, at::kBFloat16, hidden) && weight.dim() == 2 &&
        hidden.size(-1) == weight.size(1) && weight.size(1) % 64 == 0 && weight.size(0) % 64 == 0 && weight.size(0) > 16 &&
        weight.size(0) <= 32768 && trained(weight, grad, hidden) && targets.scalar_type() == at::kLong && targets.is_contiguous() &&
        targets.device() == hidden.device() && targets.numel() == hidden.numel() / weight.size(1) && scale != 0.0))
    return std::nullopt;
  if (!(at::GradMode::is_enabled() && hidden.requires_grad())) return std::nullopt;
  return Head::apply(hidden, weight, targets, grad, scale, chunk, status);
}

// ``score``: 0 softmax, 1 sigmoid, -1 what the caller refuses.
std::optional<variable_list> route_topk(const Tensor& logits, const Optional& bias, int64_t k, int64_t score, int64_t groups,
                                        int64_t top_groups, int64_t group_score, bool renormalize, double scale) {
  if (!(logits.is_cuda() && logits.dim() == 2 && logits.size(0) > 0 && float_type(logits) >= 0 && logits.is_contiguous() && score >= 0))
    return std::nullopt;
  const int64_t E = logits.size(1);
  if (!(E >= 1 && E <= 1024 && groups >= 1 && groups <= 32 && E % groups == 0 && top_groups >= 1 && top_groups <= groups && k >= 1 &&
        k <= 32 && k <= E / groups * top_groups && (group_score == 1 || (group_score == 2 && E / groups >= 2)) &&
        std::fabs(scale) >= FLT_MIN && std::fabs(scale) <= FLT_MAX))
    return std::nullopt;
  if (bias && !(bias->dim() == 1 && bias->size(0) == E && bias->scalar_type() == at::kFloat && bias->is_contiguous() &&
                bias->device() == logits.device() && !bias->requires_grad()))
    return std::nullopt;
  if (!follows({logits})) return RouteTopk::run(logits, bias, k, score == 1, groups, top_groups, group_score == 2, renormalize, scale);
  return RouteTopk::apply(logits, bias, k, score == 1, groups, top_groups, group_score == 2, renormalize, scale);
}

std::optional<variable_list> gated_norm(const Tensor& x, const Tensor& delta, const Tensor& wd, const Tensor& w, const Optional& gate,
                                        double scale, double eps, const Tensor& status) {
  const int64_t dims = x.dim();
  if (!(x.is_cuda() && dims >= 1 && x.numel() > 0 && float_type(x) >= 0 && x.is_contiguous() && delta.sizes() == x.sizes() &&
        delta.scalar_type() == x.scalar_type() && delta.is_contiguous() && delta.device() == x.device() && std::fabs(scale) <= FLT_MAX &&
        eps >= FLT_MIN && eps <= FLT_MAX))
    return std::nullopt;
  const int64_t D = x.size(-1);
  if (!(D <= 8192 && x.numel() / D <= INT_MAX - 0xffff)) return std::nullopt;
  for (const Tensor& t : {wd, w})
    if (!(t.dim() == 1 && t.size(0) == D && t.scalar_type() == at::kFloat && t.is_contiguous() && t.device() == x.device()))
      return std::nullopt;
  int64_t kind = 0, seq = 1;                       // as _gate_kind in dense.py
  if (gate) {
    if (!((gate->scalar_type() == x.scalar_type() || gate->scalar_type() == at::kFloat) && gate->is_contiguous() &&
          gate->device() == x.device()))
      return std::nullopt;
    std::vector<int64_t> token = x.sizes().vec(), sequence(dims, 1);
    token.back() = 1;
    sequence[0] = x.size(0);
    sequence.back() = D;
    if (gate->sizes() == x.sizes()) kind = 4;
    else if (gate->dim() == 1 && gate->size(0) == D) kind = 1;
    else if (gate->sizes() == at::IntArrayRef(token)) kind = 3;
    else if (dims >= 3 && gate->sizes() == at::IntArrayRef(sequence)) kind = 2, seq = x.numel() / (x.size(0) * D);
    else return std::nullopt;
  }
  if (!follows({x, delta, wd, w, gate ? *gate : Tensor()})) {
    variable_list out = GatedNorm::run(x, delta, wd, w, gate, kind, seq, scale, eps, status);
    out.pop_back();
    return out;
  }
  return GatedNorm::apply(x, delta, wd, w, gate, kind, seq, scale, eps, status);
}

// Operands of a product that a tensor map takes: e4m3 rows of unit stride that start at multiples of 16 bytes, with fp32 scales.
bool rows8(const Tensor& t, const Tensor& scales, int64_t block_rows, const Tensor& beside) {
  return t.dim() == 2 && t.scalar_type() == at::kFloat8_e4m3fn && t.device() == beside.device() && t.size(0) > 0 && t.size(1) > 0 &&
         t.stride(1) == 1 && t.stride(0) % 16 == 0 && t.stride(0) >= t.size(1) && aligned(t) && scales.dim() == 2 &&
         scales.scalar_type() == at::kFloat && scales.device() == beside.device() &&
         scales.size(0) == (t.size(0) + block_rows - 1) / block_rows && scales.size(1) == (t.size(1) + 127) / 128;
}

Optional matmul_fp8(const Tensor& a, const Tensor& sa, const Tensor& b, const Tensor& sb, const Tensor& status) {
  if (!(a.is_cuda() && rows8(a, sa, 1, a) && rows8(b, sb, 128, a) && a.size(1) == b.size(1) &&
        std::max({a.size(0), a.size(1), b.size(0)}) <= INT_MAX - 255))
    return std::nullopt;
  const c10::cuda::CUDAGuard guard(a.device());
  Tensor out = bf16({a.size(0), b.size(0)}, a);
  check(lib.gemm_fp8(ptr(a), ptr(sa), ptr(b), ptr(sb), mut(out), a.size(0), b.size(0), a.size(1), a.stride(0), b.stride(0),
                     sa.stride(0), sa.stride(1), sb.stride(0), sb.stride(1), 0, mut(status), stream()), "b2_gemm_fp8", 1);
  return out;
}

Optional linear_fp8(const Tensor& x, const Tensor& weight, const Optional& values, const Optional& scales, const Tensor& status) {
  if (!(x.is_cuda() && x.dim() >= 1 && x.numel() > 0 && plain(x, at::kBFloat16, x) && weight.dim() == 2 && weight.size(0) > 0 &&
        x.size(-1) == weight.size(1) && weight.device() == x.device() &&
        std::max({x.numel() / x.size(-1), weight.size(0), weight.size(1)}) <= INT_MAX - 255))
    return std::nullopt;
  const int64_t N = weight.size(0), K = weight.size(1);
  if (N % 8 || K % 32 || !(weight.scalar_type() == at::kBFloat16 || weight.scalar_type() == at::kFloat)) return std::nullopt;
  if (values) {
    if (!(scales && rows8(*values, *scales, 128, x) && values->sizes() == weight.sizes())) return std::nullopt;
    return follows({x, weight}) ? LinearFp8::apply(x, weight, *values, *scales, status) : LinearFp8::run(x, weight, *values, *scales, status);
  }
  if (!weight.is_contiguous()) return std::nullopt;
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor q = at::empty({N, K}, weight.options().dtype(at::kFloat8_e4m3fn).requires_grad(false));      // K is a multiple of 16
  const Tensor s = at::empty({(N + 127) / 128, (K + 127) / 128}, weight.options().dtype(at::kFloat).requires_grad(false));
  check(lib.quantize_fp8(ptr(weight), float_type(weight), mut(q), mut(s), N, K, K, K, N, 128, stream()), "b2_quantize_fp8", 1);
  return follows({x, weight}) ? LinearFp8::apply(x, weight, q, s, status) : LinearFp8::run(x, weight, q, s, status);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  using Release = pybind11::call_guard<pybind11::gil_scoped_release>;
  m.def("bind", &bind);
  m.def("check", &check, Release());
  m.def("launches", [] { return launches.load(); });
  m.def("embedding", &embedding, Release());
  m.def("rmsnorm", &rmsnorm, Release());
  m.def("attn_half", &attn_half, Release());
  m.def("moe_layer", &moe_layer, Release());
  m.def("head", &head, Release());
  m.def("route_topk", &route_topk, Release());
  m.def("gated_norm", &gated_norm, Release());
  m.def("matmul_fp8", &matmul_fp8, Release());
  m.def("linear_fp8", &linear_fp8, Release());
}
