// dtk_torch.cpp — the view-token operators (dtk_*, include/dsplat_hip.h) as torch functions with their
// autograd nodes: argument checks, allocation on torch's allocator, torch's current stream of the tensors' device.
//
// Why not ctypes and Python autograd functions, as the other operators have: a pass over a few MB takes the GPU
// 5 - 60 us, and the Python layers took 90 - 120 us of host time forward and backward (11 us forward alone) against
// torch's own 45 us for any node (its engine's thread). From here it is that and the launches.
//
// Errors: ValueError for arguments, NotImplementedError for forward-mode derivatives, DsplatError (my_depthsplat_amd._lib) for
// tensors that are not on a GPU and for a status of the C ABI.
#include <torch/extension.h>

#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <cmath>

#include "../../include/dsplat_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<Tensor>;

struct DsplatError : std::runtime_error {
  using std::runtime_error::runtime_error;
};

// The library's functions, bound by address: whichever build of it is loaded.
struct Api {
  decltype(&dtk_dropout) dropout;
  decltype(&dtk_layer_norm_fwd) layer_norm_fwd;
  decltype(&dtk_layer_norm_bwd_workspace_size) layer_norm_bwd_workspace_size;
  decltype(&dtk_layer_norm_bwd) layer_norm_bwd;
  decltype(&dtk_rotary) rotary;
  decltype(&dtk_select_blocks_workspace_size) select_blocks_workspace_size;
  decltype(&dtk_select_blocks) select_blocks;
  decltype(&dtk_block_sparse_attention_fwd_workspace_size) attention_fwd_workspace_size;
  decltype(&dtk_block_sparse_attention_fwd) attention_fwd;
  decltype(&dtk_block_sparse_attention_bwd_workspace_size) attention_bwd_workspace_size;
  decltype(&dtk_block_sparse_attention_bwd) attention_bwd;
  decltype(&dsplat_last_error) last_error;
} api;

// fn(args..., stream) on the current stream of the device of `on`.
template <typename F, typename... A>
void launch(const char* what, const Tensor& on, F fn, A... args) {
  const c10::DeviceGuard guard(on.device());
  if (fn(args..., (void*)c10::hip::getCurrentHIPStream(on.device().index()).stream()) != 0)
    throw DsplatError(std::string(what) + ": " + api.last_error());
}

void on_gpu(const Tensor& t) {
  if (!t.is_cuda())
    throw DsplatError(
        "my_depthsplat_amd ops need device (HIP) tensors; got a CPU tensor. There is no CPU fallback (the CPU restatement in "
        "oracle/ is test-only).");
}
void same_device(const Tensor& x, std::initializer_list<std::pair<const char*, const Tensor*>> others) {
  on_gpu(x);
  for (const auto& [name, t] : others)
    if (t->defined()) {
      on_gpu(*t);
      TORCH_CHECK_VALUE(t->device() == x.device(), name, " is on ", t->device(), ", the rows on ", x.device());
    }
}

int row_type(const Tensor& x, const char* name = "x") {
  switch (x.scalar_type()) {
    case at::kFloat: return DTK_F32;
    case at::kBFloat16: return DTK_BF16;
    case at::kHalf: return DTK_F16;
    default: break;
  }
  TORCH_CHECK_VALUE(false, name, " must be float32, bfloat16 or float16, got ", x.scalar_type());
}

Tensor or_none(const MaybeTensor& t) { return t.has_value() ? *t : Tensor(); }
// (an autograd node's optional tensors: one that is undefined is no argument of its graph)
MaybeTensor maybe(const Tensor& t) { return t.defined() ? MaybeTensor(t) : std::nullopt; }
Tensor contiguous(const Tensor& t) { return t.defined() ? t.contiguous() : t; }
const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* out(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
Tensor empty_as(const Tensor& x) { return at::empty(x.sizes(), x.options()); }
Tensor bytes(const Tensor& on, size_t n) { return n ? at::empty({(int64_t)n}, on.options().dtype(at::kByte)) : Tensor(); }

bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// A forward-mode derivative would be lost on the way to the result, which is a derivative of 0: refused. (A look at the
// tensors' own data; no dispatch.)
void no_tangent(std::initializer_list<const Tensor*> ts) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor* t : ts)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(/*level=*/0).defined(),
                                "the view-token operators have no forward-mode derivatives: take the tangent off (unpack_dual)");
}

// A backward's gradients. Where a graph of the backward is being made, differentiating them is an error, not zeros.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list real;
  for (auto& g : grads)
    if (g.defined()) real.push_back(g.detach().requires_grad_(true));
  if (real.empty()) return grads;
  auto node = std::make_shared<torch::autograd::DelayedError>("the view-token operators are not differentiable twice",
                                                              (int)real.size());
  real = (*node)(std::move(real));
  size_t k = 0;
  for (auto& g : grads)
    if (g.defined()) g = real[k++];
  return grads;
}

// Which gradients are asked for: of the arguments that are tensors, in order (none where an optional one is missing).
struct Needs {
  AutogradContext* ctx;
  size_t edge = 0;
  bool operator()(bool given) { return given && ctx->needs_input_grad(edge++); }
};

// ---- dropout ------------------------------------------------------------------------------------------------------

void check_drop(double p, const Tensor& rng, int64_t call) {
  TORCH_CHECK_VALUE(p >= 0.0 && p <= 1.0, "p must be in [0, 1], got ", p);
  TORCH_CHECK_VALUE(p == 0.0 || (rng.defined() && rng.scalar_type() == at::kLong && rng.numel() == 2 && rng.is_contiguous()),
                    "dropout needs rng, a contiguous int64 tensor (seed, step): dropout_rng()");
  TORCH_CHECK_VALUE(call >= 0 && call < (1LL << 32), "call must be in [0, 2^32), got ", call);
}

Tensor run_dropout(const Tensor& x, const Tensor& residual, double p, const Tensor& rng, int64_t call) {
  Tensor y = empty_as(x);
  launch("dtk_dropout", x, api.dropout, x.numel(), row_type(x), ptr(x), ptr(residual), p, (const int64_t*)ptr(rng), (uint32_t)call,
         out(y));
  return y;
}

struct Dropout : torch::autograd::Function<Dropout> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const MaybeTensor& residual_, double p, const MaybeTensor& rng_,
                        int64_t call) {
    const Tensor residual = or_none(residual_), rng = or_none(rng_);
    ctx->save_for_backward({rng});
    ctx->saved_data["p"] = p;
    ctx->saved_data["call"] = call;
    ctx->saved_data["residual"] = residual.defined();
    return run_dropout(x, residual, p, rng, call);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    Needs need{ctx};
    const bool x = need(true), residual = need(ctx->saved_data["residual"].toBool());
    Tensor dx;
    if (x)
      dx = run_dropout(grads[0].contiguous(), Tensor(), ctx->saved_data["p"].toDouble(), ctx->get_saved_variables()[0],
                       ctx->saved_data["call"].toInt());
    return once({dx, residual ? grads[0] : Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

Tensor dropout(const Tensor& x, double p, const MaybeTensor& rng_, int64_t call, const MaybeTensor& residual_) {
  Tensor rng = or_none(rng_), residual = or_none(residual_);
  check_drop(p, rng, call);
  row_type(x);
  TORCH_CHECK_VALUE(!residual.defined() || (residual.sizes() == x.sizes() && residual.scalar_type() == x.scalar_type()),
                    "residual does not match x: ", x.scalar_type(), " ", x.sizes());
  if (p == 0.0) rng = Tensor();
  if (p > 0.0 || residual.defined()) no_tangent({&x, &residual});  // (else x is returned with all it has)
  same_device(x, {{"residual", &residual}, {"rng", &rng}});
  if (p == 0.0 && !residual.defined()) return x;
  residual = contiguous(residual);
  if (wants_grad({&x, &residual})) return Dropout::apply(x.contiguous(), maybe(residual), p, maybe(rng), call);
  return run_dropout(x.contiguous(), residual, p, rng, call);
}

// ---- layer norm ---------------------------------------------------------------------------------------------------

struct Normed {
  Tensor s, y, mean, rstd;
};
Normed run_norm(const Tensor& x, const Tensor& residual, const Tensor& weight, const Tensor& bias, double eps, double p,
                const Tensor& rng, int64_t call, bool stats) {
  const int64_t width = x.size(-1), rows = x.numel() / width;
  Normed n;
  if (residual.defined()) n.s = empty_as(x);
  n.y = empty_as(x);
  if (stats) {
    const Tensor both = at::empty({2, rows}, x.options().dtype(at::kFloat));
    n.mean = both[0];
    n.rstd = both[1];
  }
  const Tensor& w = weight.defined() ? weight : bias;
  launch("dtk_layer_norm_fwd", x, api.layer_norm_fwd, rows, (int)width, row_type(x), w.defined() ? row_type(w) : row_type(x), ptr(x),
         ptr(residual), ptr(weight), ptr(bias), (float)eps, p, (const int64_t*)ptr(rng), (uint32_t)call, out(n.s), out(n.y),
         (float*)out(n.mean), (float*)out(n.rstd));
  return n;
}

struct NormGrads {
  Tensor dx, dresidual, dweight, dbias;
};
NormGrads run_norm_bwd(const Tensor& z, const Tensor& dy, const Tensor& ds, const Tensor& weight, const Tensor& bias, const Tensor& mean,
                       const Tensor& rstd, bool add, double p, const Tensor& rng, int64_t call, bool nx, bool nr, bool nw, bool nb) {
  const int64_t width = z.size(-1), rows = z.numel() / width;
  NormGrads g;
  const bool shared = add && p == 0.0 && nx && nr;  // without dropout x's gradient is the residual's
  if (nx && !shared) g.dx = empty_as(z);
  if (nr) g.dresidual = empty_as(z);
  if (nw) g.dweight = empty_as(weight);
  if (nb) g.dbias = empty_as(bias);
  Tensor ws;
  if (nw || nb) ws = bytes(z, api.layer_norm_bwd_workspace_size(rows, (int)width, row_type(z)));
  const Tensor& w = weight.defined() ? weight : bias;
  launch("dtk_layer_norm_bwd", z, api.layer_norm_bwd, rows, (int)width, row_type(z), w.defined() ? row_type(w) : row_type(z), ptr(z),
         ptr(dy), ptr(ds), ptr(weight), (const float*)ptr(mean), (const float*)ptr(rstd), (int)add, p, (const int64_t*)ptr(rng),
         (uint32_t)call, out(g.dx), out(g.dresidual), out(g.dweight), out(g.dbias), out(ws));
  if (shared) g.dx = g.dresidual;
  return g;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const MaybeTensor& weight_, const MaybeTensor& bias_, double eps) {
    const Tensor weight = or_none(weight_), bias = or_none(bias_);
    Normed n = run_norm(x, Tensor(), weight, bias, eps, 0.0, Tensor(), 0, true);
    ctx->save_for_backward({x, weight, bias, n.mean, n.rstd});
    return n.y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto v = ctx->get_saved_variables();
    Needs need{ctx};
    const bool nx = need(true), nw = need(v[1].defined()), nb = need(v[2].defined());
    NormGrads g = run_norm_bwd(v[0], grads[0].contiguous(), Tensor(), v[1], v[2], v[3], v[4], false, 0.0, Tensor(), 0, nx, false, nw, nb);
    return once({g.dx, g.dweight, g.dbias, Tensor()});
  }
};

struct AddLayerNorm : torch::autograd::Function<AddLayerNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& residual, const MaybeTensor& weight_,
                               const MaybeTensor& bias_, double eps, double p, const MaybeTensor& rng_, int64_t call) {
    const Tensor weight = or_none(weight_), bias = or_none(bias_), rng = or_none(rng_);
    Normed n = run_norm(x, residual, weight, bias, eps, p, rng, call, true);
    ctx->save_for_backward({n.s, weight, bias, n.mean, n.rstd, rng});
    ctx->saved_data["p"] = p;
    ctx->saved_data["call"] = call;
    ctx->set_materialize_grads(false);
    return {n.s, n.y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list none(8);
    if (!grads[0].defined() && !grads[1].defined()) return none;
    const auto v = ctx->get_saved_variables();
    Needs need{ctx};
    const bool nx = need(true), nr = need(true), nw = need(v[1].defined()), nb = need(v[2].defined());
    NormGrads g = run_norm_bwd(v[0], contiguous(grads[1]), contiguous(grads[0]), v[1], v[2], v[3], v[4], true,
                               ctx->saved_data["p"].toDouble(), v[5], ctx->saved_data["call"].toInt(), nx, nr, nw, nb);
    none[0] = g.dx;
    none[1] = g.dresidual;
    none[2] = g.dweight;
    none[3] = g.dbias;
    return once(std::move(none));
  }
};

void check_norm(const Tensor& x, const Tensor& weight, const Tensor& bias, double eps) {
  row_type(x);
  TORCH_CHECK_VALUE(x.dim() > 0 && x.size(-1) > 0, "layer norm needs rows [..., width > 0], got ", x.sizes());
  TORCH_CHECK_VALUE(x.size(-1) <= (1LL << 28) && x.numel() / x.size(-1) < (1LL << 31), "x is too large: ", x.sizes());
  TORCH_CHECK_VALUE(eps >= 0.0, "eps must not be negative, got ", eps);
  for (const auto& [name, w] : {std::pair<const char*, const Tensor*>{"weight", &weight}, {"bias", &bias}})
    if (w->defined()) {
      TORCH_CHECK_VALUE(w->dim() == 1 && w->size(0) == x.size(-1), name, " must be [", x.size(-1), "], got ", w->sizes());
      TORCH_CHECK_VALUE(w->scalar_type() == x.scalar_type() || w->scalar_type() == at::kFloat, name, " must be ", x.scalar_type(),
                        " or float32, got ", w->scalar_type());
    }
  TORCH_CHECK_VALUE(!weight.defined() || !bias.defined() || weight.scalar_type() == bias.scalar_type(),
                    "weight and bias must have one type");
}

Tensor layer_norm(const Tensor& x, const MaybeTensor& weight_, const MaybeTensor& bias_, double eps) {
  Tensor weight = or_none(weight_), bias = or_none(bias_);
  check_norm(x, weight, bias, eps);
  no_tangent({&x, &weight, &bias});
  same_device(x, {{"weight", &weight}, {"bias", &bias}});
  weight = contiguous(weight);
  bias = contiguous(bias);
  if (wants_grad({&x, &weight, &bias})) return LayerNorm::apply(x.contiguous(), maybe(weight), maybe(bias), eps);
  return run_norm(x.contiguous(), Tensor(), weight, bias, eps, 0.0, Tensor(), 0, false).y;
}

std::pair<Tensor, Tensor> dropout_add_layer_norm(const Tensor& x, const Tensor& residual, const MaybeTensor& weight_,
                                                 const MaybeTensor& bias_, double p, const MaybeTensor& rng_, int64_t call, double eps) {
  Tensor weight = or_none(weight_), bias = or_none(bias_), rng = or_none(rng_);
  check_drop(p, rng, call);
  check_norm(x, weight, bias, eps);
  TORCH_CHECK_VALUE(residual.sizes() == x.sizes() && residual.scalar_type() == x.scalar_type(),
                    "residual does not match x: ", x.scalar_type(), " ", x.sizes());
  if (p == 0.0) rng = Tensor();
  no_tangent({&x, &residual, &weight, &bias});
  same_device(x, {{"residual", &residual}, {"weight", &weight}, {"bias", &bias}, {"rng", &rng}});
  weight = contiguous(weight);
  bias = contiguous(bias);
  if (wants_grad({&x, &residual, &weight, &bias})) {
    const auto r = AddLayerNorm::apply(x.contiguous(), residual.contiguous(), maybe(weight), maybe(bias), eps, p, maybe(rng), call);
    return {r[0], r[1]};
  }
  Normed n = run_norm(x.contiguous(), residual.contiguous(), weight, bias, eps, p, rng, call, false);
  return {n.s, n.y};
}

// ---- rotary positions ---------------------------------------------------------------------------------------------

// the token stride: of a single token it may be any number, and is not used
int64_t token_stride(const Tensor& t) { return t.size(1) > 1 ? t.stride(1) : 0; }
// rows whose channels are dense, and whose token stride the kernels take
Tensor dense_rows(const Tensor& t) { return t.stride(-1) == 1 && token_stride(t) < (1LL << 24) ? t : t.contiguous(); }

struct Strides {
  int64_t s[3];
  explicit Strides(const Tensor& t) : s{t.stride(0), token_stride(t), t.stride(2)} {}
};

// Sizes that the C ABI takes as 32-bit numbers.
void check_sizes(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.size(0) < 65536 && t.size(1) <= (1LL << 31) - 256 && t.size(2) < 65536 && t.size(3) < (1LL << 20), name,
                    " is too large: ", t.sizes());
}

std::pair<Tensor, Tensor> run_rotary(const Tensor& q, const Tensor& k, const Tensor& positions, const Tensor& freqs, bool interleaved,
                                     double factor, bool backward) {
  const Tensor& any = q.defined() ? q : k;
  Tensor oq, ok;
  if (q.defined()) oq = empty_as(q);
  if (k.defined()) ok = empty_as(k);
  const int64_t ps[3] = {positions.dim() == 2 ? 0 : positions.stride(0), positions.stride(-2), positions.stride(-1)};
  const int ptype = positions.scalar_type() == at::kLong ? DTK_I64 : positions.scalar_type() == at::kInt ? DTK_I32 : DTK_F32;
  const Strides sq(any), sk(k.defined() ? k : any);
  launch("dtk_rotary", any, api.rotary, any.size(0), any.size(1), q.defined() ? (int)q.size(2) : 0, k.defined() ? (int)k.size(2) : 0,
         (int)any.size(3), (int)freqs.numel(), (int)positions.size(-1), (int)interleaved, (int)backward, row_type(any), ptype, ptr(q), sq.s,
         ptr(k), sk.s, ptr(positions), ps, (const double*)ptr(freqs), (float)factor, out(oq), out(ok));
  return {oq, ok};
}

struct Rotary : torch::autograd::Function<Rotary> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const MaybeTensor& k_, const Tensor& positions, const Tensor& freqs,
                               bool interleaved, double factor) {
    const Tensor k = or_none(k_);
    ctx->save_for_backward({positions, freqs});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["factor"] = factor;
    ctx->set_materialize_grads(false);
    auto [oq, ok] = run_rotary(q, k, positions, freqs, interleaved, factor, false);
    return k.defined() ? variable_list{oq, ok} : variable_list{oq};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list none(6);
    Needs need{ctx};
    const Tensor dq = need(true) ? grads[0] : Tensor(), dk = need(grads.size() > 1) ? grads[1] : Tensor();
    if (!dq.defined() && !dk.defined()) return none;
    const auto v = ctx->get_saved_variables();
    std::tie(none[0], none[1]) = run_rotary(dq.defined() ? dense_rows(dq) : dq, dk.defined() ? dense_rows(dk) : dk, v[0], v[1],
                                            ctx->saved_data["interleaved"].toBool(), ctx->saved_data["factor"].toDouble(), true);
    return once(std::move(none));
  }
};

std::pair<Tensor, MaybeTensor> rotary(const Tensor& q_, const MaybeTensor& k_, Tensor positions, const Tensor& freqs, bool interleaved,
                                      double factor) {
  Tensor q = q_, k = or_none(k_);
  TORCH_CHECK_VALUE(q.dim() == 4, "q must be [B,L,Hq,D], got ", q.sizes());
  TORCH_CHECK_VALUE(!k.defined() || (k.dim() == 4 && k.size(0) == q.size(0) && k.size(1) == q.size(1) && k.size(3) == q.size(3)),
                    "k must be [B,L,Hk,D] beside q ", q.sizes(), ", got ", k.defined() ? k.sizes() : q.sizes());
  for (const Tensor* t : {&q, &k})  // (any number of sequences)
    TORCH_CHECK_VALUE(!t->defined() || (t->size(0) <= INT32_MAX && t->size(1) <= INT32_MAX && t->size(0) * t->size(1) <= INT32_MAX &&
                                        t->size(2) < 65536 && t->size(3) < (1LL << 20)),
                      "too many tokens, heads or channels: ", t->sizes());
  row_type(q, "q");
  TORCH_CHECK_VALUE(!k.defined() || k.scalar_type() == q.scalar_type(), "q and k must have one type");
  const int64_t B = q.size(0), L = q.size(1), D = q.size(3);
  if (positions.dim() == 1) positions = positions.unsqueeze(1);
  TORCH_CHECK_VALUE((positions.dim() == 2 || (positions.dim() == 3 && positions.size(0) == B)) && positions.size(-2) == L,
                    "positions must be [L=", L, "], [L,axes] or [B=", B, ",L,axes], got ", positions.sizes());
  TORCH_CHECK_VALUE(positions.scalar_type() == at::kLong || positions.scalar_type() == at::kInt || positions.scalar_type() == at::kFloat,
                    "positions must be int64, int32 or float32, got ", positions.scalar_type());
  const int64_t F = freqs.numel(), axes = positions.size(-1);
  TORCH_CHECK_VALUE(freqs.scalar_type() == at::kDouble && freqs.dim() == 1 && 2 * F <= D && axes > 0 && F % axes == 0,
                    "freqs must be float64 [F], 2 F <= ", D, ", F a multiple of the ", axes, " axes, got ", freqs.scalar_type(), " ",
                    freqs.sizes());
  TORCH_CHECK_VALUE(!wants_grad({&positions, &freqs}), "positions and freqs have no gradient: detach them");
  no_tangent({&q, &k, &positions, &freqs});
  same_device(q, {{"k", &k}, {"positions", &positions}, {"freqs", &freqs}});
  q = dense_rows(q);
  if (k.defined()) k = dense_rows(k);
  if (wants_grad({&q, &k})) {
    const auto r = Rotary::apply(q, maybe(k), positions, freqs.contiguous(), interleaved, factor);
    return {r[0], k.defined() ? MaybeTensor(r[1]) : std::nullopt};
  }
  auto [oq, ok] = run_rotary(q, k, positions, freqs.contiguous(), interleaved, factor, false);
  return {oq, k.defined() ? MaybeTensor(ok) : std::nullopt};
}

// ---- block choice and attention -----------------------------------------------------------------------------------

void check_heads(const Tensor& q, const Tensor& k, int64_t block) {
  TORCH_CHECK_VALUE(block == 32 || block == 64 || block == 128, "block must be 32, 64 or 128, got ", block);
  TORCH_CHECK_VALUE(q.dim() == 4 && k.dim() == 4 && k.size(0) == q.size(0) && k.size(3) == q.size(3),
                    "q must be [B,Lq,Hq,D] and k [B,Lk,Hkv,D], got ", q.sizes(), " and ", k.sizes());
  TORCH_CHECK_VALUE(k.size(2) > 0 && q.size(2) > 0 && q.size(2) % k.size(2) == 0, "the ", q.size(2),
                    " query heads must be a multiple of the ", k.size(2), " key heads");
  check_sizes(q, "q");
  check_sizes(k, "k");
  row_type(q, "q");
  TORCH_CHECK_VALUE(k.scalar_type() == q.scalar_type(), "q, k and v must have one type");
}
void check_lengths(const Tensor& t, const char* name, int64_t B) {
  TORCH_CHECK_VALUE(!t.defined() || (t.dim() == 1 && t.size(0) == B && (t.scalar_type() == at::kInt || t.scalar_type() == at::kLong)),
                    name, " must be int32 or int64 [B=", B, "]");
}
// Lengths as the kernels take them: 64 bits are cut to what 32 hold (all of a sequence, or nothing), not to their lower half.
Tensor int32(const Tensor& t) {
  if (!t.defined()) return t;
  return (t.scalar_type() == at::kLong ? t.clamp(0, INT32_MAX).to(at::kInt) : t).contiguous();
}
int64_t tiles_of(int64_t n, int64_t block) { return (n + block - 1) / block; }

Tensor select_blocks(const Tensor& q_, const Tensor& k_, int64_t top, int64_t block, const MaybeTensor& q_lengths_,
                     const MaybeTensor& kv_lengths_, const MaybeTensor& allowed_) {
  Tensor q_lengths = or_none(q_lengths_), kv_lengths = or_none(kv_lengths_), allowed = or_none(allowed_);
  check_heads(q_, k_, block);
  const int64_t B = q_.size(0), Lq = q_.size(1), Lk = k_.size(1), Hkv = k_.size(2), D = q_.size(3);
  TORCH_CHECK_VALUE(D > 0 && D <= 256, "the head size must be in [1, 256], got ", D);
  TORCH_CHECK_VALUE(top > 0 && top < (1LL << 31), "top must be positive, got ", top);
  check_lengths(q_lengths, "q_lengths", B);
  check_lengths(kv_lengths, "kv_lengths", B);
  const int64_t Tq = tiles_of(Lq, block), Tk = tiles_of(Lk, block);
  TORCH_CHECK_VALUE(!allowed.defined() ||
                        (allowed.scalar_type() == at::kBool && allowed.dim() == 2 && allowed.size(0) == Tq && allowed.size(1) == Tk),
                    "allowed must be bool [", Tq, ", ", Tk, "]");
  same_device(q_, {{"k", &k_}, {"q_lengths", &q_lengths}, {"kv_lengths", &kv_lengths}, {"allowed", &allowed}});
  const at::NoGradGuard no_grad;
  const Tensor q = dense_rows(q_), k = dense_rows(k_);
  q_lengths = int32(q_lengths);
  kv_lengths = int32(kv_lengths);
  allowed = contiguous(allowed);
  Tensor index = at::empty({B, Hkv, Tq, top}, q.options().dtype(at::kInt));
  const Tensor ws = bytes(q, api.select_blocks_workspace_size((int)B, Lq, Lk, (int)Hkv, (int)D, (int)block));
  const Strides sq(q), sk(k);
  launch("dtk_select_blocks", q, api.select_blocks, (int)B, Lq, Lk, (int)q.size(2), (int)Hkv, (int)D, (int)block, (int)top, row_type(q),
         ptr(q), sq.s, ptr(k), sk.s, (const int32_t*)ptr(q_lengths), (const int32_t*)ptr(kv_lengths), (const uint8_t*)ptr(allowed),
         (int32_t*)out(index), out(ws));
  return index;
}

dtk_attention attention_of(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& index, int64_t block, const Tensor& q_lengths,
                           const Tensor& kv_lengths, double scale, const Tensor& o, const Tensor& lse, const Tensor& rest) {
  dtk_attention a = {};
  a.Lq = q.size(1);
  a.Lk = k.size(1);
  a.B = (int32_t)q.size(0);
  a.Hq = (int32_t)q.size(2);
  a.Hkv = (int32_t)k.size(2);
  a.D = (int32_t)q.size(3);
  a.block = (int32_t)block;
  a.top = (int32_t)index.size(3);
  a.dtype = row_type(q);
  a.scale = (float)scale;
  a.q = ptr(q);
  a.k = ptr(k);
  a.v = ptr(v);
  const Strides sq(q), sk(k), sv(v);
  for (int i = 0; i < 3; ++i) {
    a.q_strides[i] = sq.s[i];
    a.k_strides[i] = sk.s[i];
    a.v_strides[i] = sv.s[i];
  }
  a.index = (const int32_t*)ptr(index);
  a.q_lengths = (const int32_t*)ptr(q_lengths);
  a.kv_lengths = (const int32_t*)ptr(kv_lengths);
  a.o = out(o);
  a.lse = (float*)out(lse);
  a.o_rest = out(rest);
  return a;
}

struct Attended {
  Tensor o, lse, rest;
};
Attended run_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& index, int64_t block,
                                        const Tensor& q_lengths, const Tensor& kv_lengths, double scale, bool stats) {
  Attended r;
  r.o = empty_as(q);
  if (stats) {
    r.lse = at::empty({q.size(0), q.size(2), q.size(1)}, q.options().dtype(at::kFloat));
    if (q.scalar_type() != at::kFloat) r.rest = empty_as(q);
  }
  const dtk_attention a = attention_of(q, k, v, index, block, q_lengths, kv_lengths, scale, r.o, r.lse, r.rest);
  const Tensor ws = bytes(q, api.attention_fwd_workspace_size(&a));
  launch("dtk_block_sparse_attention_fwd", q, api.attention_fwd, &a, out(ws));
  return r;
}

struct Attention : torch::autograd::Function<Attention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& index, int64_t block,
                        const MaybeTensor& q_lengths_, const MaybeTensor& kv_lengths_, double scale) {
    const Tensor q_lengths = or_none(q_lengths_), kv_lengths = or_none(kv_lengths_);
    Attended r = run_attention(q, k, v, index, block, q_lengths, kv_lengths, scale, true);
    ctx->save_for_backward({q, k, v, index, q_lengths, kv_lengths, r.o, r.lse, r.rest});
    ctx->saved_data["block"] = block;
    ctx->saved_data["scale"] = scale;
    return r.o;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor g = dense_rows(grads[0]);
    Needs need{ctx};
    const bool nq = need(true), nk = need(true), nv = need(true), keys = nk || nv;
    // (dq's kernel finds the lists that dk's reads; dk and dv are one kernel's)
    Tensor dq = empty_as(s[0]), dk = keys ? empty_as(s[1]) : Tensor(), dv = keys ? empty_as(s[2]) : Tensor();
    const dtk_attention a = attention_of(s[0], s[1], s[2], s[3], ctx->saved_data["block"].toInt(), s[4], s[5],
                                         ctx->saved_data["scale"].toDouble(), s[6], s[7], s[8]);
    const Tensor ws = bytes(g, api.attention_bwd_workspace_size(&a));
    const Strides sg(g);
    launch("dtk_block_sparse_attention_bwd", g, api.attention_bwd, &a, ptr(g), sg.s, out(dq), out(dk), out(dv), out(ws));
    variable_list none(8);
    if (nq) none[0] = dq;
    if (nk) none[1] = dk;
    if (nv) none[2] = dv;
    return once(std::move(none));
  }
};

Tensor block_sparse_attention(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& index_, int64_t block,
                              const MaybeTensor& q_lengths_, const MaybeTensor& kv_lengths_, const std::optional<double>& scale_) {
  Tensor q_lengths = or_none(q_lengths_), kv_lengths = or_none(kv_lengths_);
  check_heads(q_, k_, block);
  TORCH_CHECK_VALUE(v_.sizes() == k_.sizes(), "v ", v_.sizes(), " does not match k ", k_.sizes());
  TORCH_CHECK_VALUE(v_.scalar_type() == q_.scalar_type(), "q, k and v must have one type");
  const int64_t B = q_.size(0), Lq = q_.size(1), D = q_.size(3), Hkv = k_.size(2), Tq = tiles_of(Lq, block);
  TORCH_CHECK_VALUE(D > 0 && D % 8 == 0 && D <= 128, "the head size must be a multiple of 8 up to 128, got ", D);
  TORCH_CHECK_VALUE(q_.size(2) / Hkv <= 1024, "at most 1024 query heads may share a key head, got ", q_.size(2) / Hkv);
  TORCH_CHECK_VALUE(index_.scalar_type() == at::kInt && index_.dim() == 4 && index_.size(0) == B && index_.size(1) == Hkv &&
                        index_.size(2) == Tq && index_.size(3) >= 1 && index_.size(3) <= 1024,
                    "index must be int32 [", B, ", ", Hkv, ", ", Tq, ", 1..1024], got ", index_.scalar_type(), " ", index_.sizes());
  check_lengths(q_lengths, "q_lengths", B);
  check_lengths(kv_lengths, "kv_lengths", B);
  const double scale = scale_.has_value() ? *scale_ : 1.0 / std::sqrt((double)D);
  TORCH_CHECK_VALUE(std::isfinite((float)scale), "scale must be a finite 32-bit number, got ", scale);
  no_tangent({&q_, &k_, &v_});
  same_device(q_, {{"k", &k_}, {"v", &v_}, {"index", &index_}, {"q_lengths", &q_lengths}, {"kv_lengths", &kv_lengths}});
  const Tensor q = dense_rows(q_), k = dense_rows(k_), v = dense_rows(v_), index = index_.contiguous();
  q_lengths = int32(q_lengths);
  kv_lengths = int32(kv_lengths);
  if (wants_grad({&q, &k, &v})) return Attention::apply(q, k, v, index, block, maybe(q_lengths), maybe(kv_lengths), scale);
  return run_attention(q, k, v, index, block, q_lengths, kv_lengths, scale, false).o;
}

void bind(const std::map<std::string, uintptr_t>& fn) {
  const auto set = [&](auto& f, const char* name) { f = (std::decay_t<decltype(f)>)fn.at(name); };
  set(api.dropout, "dtk_dropout");
  set(api.layer_norm_fwd, "dtk_layer_norm_fwd");
  set(api.layer_norm_bwd_workspace_size, "dtk_layer_norm_bwd_workspace_size");
  set(api.layer_norm_bwd, "dtk_layer_norm_bwd");
  set(api.rotary, "dtk_rotary");
  set(api.select_blocks_workspace_size, "dtk_select_blocks_workspace_size");
  set(api.select_blocks, "dtk_select_blocks");
  set(api.attention_fwd_workspace_size, "dtk_block_sparse_attention_fwd_workspace_size");
  set(api.attention_fwd, "dtk_block_sparse_attention_fwd");
  set(api.attention_bwd_workspace_size, "dtk_block_sparse_attention_bwd_workspace_size");
  set(api.attention_bwd, "dtk_block_sparse_attention_bwd");
  set(api.last_error, "dsplat_last_error");
}

}  // namespace

PYBIND11_MODULE(dsplat_torch, m) {
  static py::object error;
  error = py::module_::import("my_depthsplat_amd._lib").attr("DsplatError");
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const DsplatError& e) {
      PyErr_SetString(error.ptr(), e.what());
    }
  });
  m.def("bind", &bind);
  using release = py::call_guard<py::gil_scoped_release>;
  m.def("dropout", &dropout, release());
  m.def("layer_norm", &layer_norm, release());
  m.def("dropout_add_layer_norm", &dropout_add_layer_norm, release());
  m.def("rotary", &rotary, release());
  m.def("select_blocks", &select_blocks, release());
  m.def("block_sparse_attention", &block_sparse_attention, release());
}
