// Host side of the MoC calls that a program makes per step: the layer and the
// functional op as autograd nodes, the forward with a state, and the decode
// step, each one call from Python.  What they launch and return is what the
// Python functions of moc/api.py and moc/ops.py do (which stay for every call
// that one of these hands back as not its own: other dtypes and shapes, tensor
// subclasses, tracing, function transforms, forward-mode differentiation).
//
// Why: a step of a small layer spent most of its time in the interpreter: checks,
// argument conversion and allocations in Python, and a backward that waits for
// the interpreter lock on autograd's own thread.  Us a call, Python functions ->
// here: training step B 3 T 1021 D 1130 138 to 165 (by box) -> 92 (53 of it
// kernels), fp32 B 2 T 512 D 256 170 -> 95; 777-token prefill 31 -> 17.6; decode step
// 10.5 -> 7.6, fp32 25.6 -> 11.4.
#include <ATen/autocast_mode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_cpp_function.h>
#include <torch/extension.h>

#include "../../include/moc_hip.h"

namespace {

using at::Tensor;
using c10::DispatchKey;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

int dtype_code(at::ScalarType t) { return t == at::kFloat ? 0 : (t == at::kBFloat16 ? 1 : -1); }

// A dense GPU tensor of its own: no wrapper or transform of one, no dual number.
bool plain(const Tensor& t) {
  if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || t.is_neg() || t.is_conj()) return false;
  static const c10::DispatchKeySet wrapped({DispatchKey::Python, DispatchKey::PythonTLSSnapshot,
                                            DispatchKey::FuncTorchBatched, DispatchKey::FuncTorchGradWrapper,
                                            DispatchKey::Batched, DispatchKey::Functionalize});
  return !t.key_set().has_any(wrapped) && t.has_storage() && !t._fw_grad(0).defined();
}

// No tracer, dispatch mode or function transform is watching this thread.
bool unwatched() {
  using c10::impl::tls_is_dispatch_key_included;
  return !tls_is_dispatch_key_included(DispatchKey::Python) &&
         !tls_is_dispatch_key_included(DispatchKey::Tracer) &&
         !tls_is_dispatch_key_included(DispatchKey::Functionalize) &&
         !tls_is_dispatch_key_included(DispatchKey::FuncTorchDynamicLayerFrontMode);
}

bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t != nullptr && t->defined() && t->requires_grad()) return true;
  return false;
}

void check(int rc, const char* what) {
  if (rc != 0) TORCH_CHECK(false, what, " failed (status ", rc, "): ", moc_last_error());
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

Tensor bytes(size_t n, const Tensor& like) {
  return at::empty({static_cast<int64_t>(n > 0 ? n : 1)}, like.options().dtype(at::kByte));
}

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// A layer call's sizes and codes.  Fixed-length x [B, T, D] or packed x [N, D]
// with cu.
struct Call {
  int act, route;  // route: 1 softmax, 2 exp (layer); 0 weights given (func)
  int dt;
  int64_t N, T, D, K, S, Z;
  Tensor cu;       // undefined: fixed length
  const void* cu_ptr() const { return ptr(cu); }
  int cu64() const { return cu.defined() && cu.scalar_type() == at::kLong; }
  int64_t n_seqs() const { return cu.defined() ? cu.numel() - 1 : 0; }
  int64_t seq_len() const { return cu.defined() ? 0 : T; }
};

// Fills the sizes that x, the basis and the packed offsets give; false where
// the call is not one of these (the Python path then names what is wrong).
bool sizes(Call& c, const Tensor& x, const Tensor& basis, const OptTensor& cu) {
  c.dt = dtype_code(x.scalar_type());
  if (c.dt < 0 || basis.scalar_type() != x.scalar_type() || basis.dim() != 3) return false;
  c.K = basis.size(0), c.S = basis.size(1), c.D = basis.size(2);
  if (x.dim() != (cu.has_value() ? 2 : 3) || x.size(-1) != c.D) return false;
  if (x.numel() == 0 || basis.numel() == 0) return false;
  c.N = x.numel() / c.D;
  c.T = cu.has_value() ? 0 : x.size(1);
  if (cu.has_value()) {
    if (!plain(*cu) || cu->device() != x.device() || cu->dim() != 1 || cu->numel() < 2) return false;
    if (cu->scalar_type() != at::kInt && cu->scalar_type() != at::kLong) return false;
    c.cu = cu->contiguous();
  }
  return basis.device() == x.device();
}

// The router's sizes; whether its kernels take them (as ops.router_supported and
// ops.router_f32_supported say).
bool router_ok(Call& c, const Tensor& x, const Tensor& z, const Tensor& router) {
  if (z.scalar_type() != x.scalar_type() || router.scalar_type() != x.scalar_type()) return false;
  if (z.device() != x.device() || router.device() != x.device()) return false;
  if (router.dim() != 2 || router.size(0) != c.K || z.dim() != x.dim()) return false;
  c.Z = router.size(1);
  if (z.size(-1) != c.Z || z.numel() == 0) return false;
  for (int64_t i = 0; i + 1 < z.dim(); ++i)
    if (z.size(i) != x.size(i)) return false;
  if (c.K > 32) return false;
  if (c.dt == 1) return moc_router_supported(c.N, c.Z, c.K, 1) != 0;
  return !at::autocast::is_autocast_enabled(at::kCUDA) && moc_router_f32_supported(c.N, c.Z, c.K) != 0;
}

// softmax / exp (or the logits: route 0) of z . router^T
Tensor run_router(const Call& c, const Tensor& z, const Tensor& router, int route) {
  auto shape = z.sizes().vec();
  shape.back() = c.K;
  Tensor out = at::empty(shape, z.options());
  if (c.dt == 0)
    check(moc_router_f32_forward(ptr(z), ptr(router), ptr(out), c.N, c.Z, c.K, route, stream_of(z)),
          "moc_router_f32_forward");
  else if (route == 0)
    check(moc_router_forward(ptr(z), ptr(router), ptr(out), c.N, c.Z, c.K, 1, stream_of(z)),
          "moc_router_forward");
  else
    check(moc_router_forward_routed(ptr(z), ptr(router), ptr(out), c.N, c.Z, c.K, 1, route, stream_of(z)),
          "moc_router_forward");
  return out;
}

// moc_forward on weights of the given routing code
Tensor run_forward(const Call& c, const Tensor& x, const Tensor& a, const Tensor& basis, int routing) {
  Tensor y = at::empty_like(x);
  Tensor ws = bytes(moc_forward_workspace_bytes(c.N, c.D, c.K, c.S, c.dt, routing), x);
  check(moc_forward(ptr(x), ptr(a), ptr(basis), ptr(y), c.cu_ptr(), c.cu64(), c.n_seqs(), c.N, c.seq_len(),
                    c.D, c.K, c.S, c.dt, c.dt, c.dt, c.act, routing, ptr(ws), ws.numel(), stream_of(x)),
        "moc_forward");
  return y;
}

// dy as the kernels take it (ops.dy_operand): rows D apart, one broadcast row (0)
// or one broadcast element (-1)
Tensor dy_operand(const Tensor& dy, at::ScalarType dt, int64_t& stride) {
  const auto st = dy.strides();
  const int64_t D = dy.size(-1);
  bool lead0 = true;
  for (size_t i = 0; i + 1 < st.size(); ++i) lead0 = lead0 && st[i] == 0;
  if (dy.numel() > 1 && lead0 && st.back() == 0) {
    stride = -1;
    return dy.as_strided({1}, {1}, dy.storage_offset()).to(dt);
  }
  if (dy.dim() >= 2 && dy.numel() > D && lead0) {
    stride = 0;
    return dy.as_strided({D}, {st.back()}, dy.storage_offset()).to(dt).contiguous();
  }
  stride = D;
  return dy.contiguous().to(dt);
}

struct Grads {
  Tensor dx, da, db;
};
Grads run_backward(const Call& c, const Tensor& x, const Tensor& a, const Tensor& basis, const Tensor& dy,
                   bool need_x, int routing) {
  int64_t stride;
  const Tensor dyo = dy_operand(dy, x.scalar_type(), stride);
  Grads g{need_x ? at::empty_like(x) : Tensor(), at::empty_like(a), at::empty_like(basis)};
  Tensor ws = bytes(moc_backward_workspace_bytes(c.N, c.D, c.K, c.S, c.dt, routing), x);
  check(moc_backward(ptr(x), ptr(a), ptr(basis), ptr(dyo), stride, ptr(g.dx), ptr(g.da), ptr(g.db), c.cu_ptr(),
                     c.cu64(), c.n_seqs(), c.N, c.seq_len(), c.D, c.K, c.S, c.dt, c.dt, c.dt, c.act, routing,
                     ptr(ws), ws.numel(), stream_of(x)),
        "moc_backward");
  return g;
}

// The nodes are differentiable once: with a graph asked for, their results
// raise when they are differentiated again.
variable_list once(variable_list out, const variable_list& grads) {
  bool any = false;
  for (const auto& g : grads) any = any || (g.defined() && g.requires_grad());
  if (!any) return out;
  variable_list defined;
  for (auto& t : out)
    if (t.defined()) defined.push_back(t.detach().set_requires_grad(true));
  auto err = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that was marked with @once_differentiable",
      static_cast<int64_t>(defined.size()));
  variable_list wrapped = (*err)(std::move(defined));
  size_t i = 0;
  for (auto& t : out)
    if (t.defined()) t = wrapped[i++];
  return out;
}

void keep(AutogradContext* ctx, const Call& c) {
  ctx->saved_data["c"] = std::vector<int64_t>{c.act, c.route, c.dt, c.N, c.T, c.D, c.K, c.S, c.Z};
}
Call kept(AutogradContext* ctx, const Tensor& cu) {
  const auto v = ctx->saved_data["c"].toIntVector();
  return Call{static_cast<int>(v[0]), static_cast<int>(v[1]), static_cast<int>(v[2]), v[3], v[4], v[5], v[6],
              v[7], v[8], cu};
}

// MoC.forward as one node (api._MoCLayerFunction)
struct LayerFn : public torch::autograd::Function<LayerFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x0, const Tensor& z0, const Tensor& r0,
                        const Tensor& b0, const Call* c) {
    const Tensor x = x0.contiguous(), z = z0.contiguous(), r = r0.contiguous(), b = b0.contiguous();
    const Tensor w = run_router(*c, z, r, c->route);
    Tensor y = run_forward(*c, x, w, b, c->route + 2);
    ctx->save_for_backward({x, w, b, z0, r0, c->cu});
    keep(ctx, *c);
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &b = saved[2];
    const Call c = kept(ctx, saved[5]);
    const bool need[3] = {ctx->needs_input_grad(0), ctx->needs_input_grad(1), ctx->needs_input_grad(2)};
    variable_list out(5);
    {
      at::NoGradGuard ng;
      const c10::DeviceGuard dg(x.device());
      const Grads g = run_backward(c, x, w, b, grads[0], need[0], c.route + 2);
      out[0] = g.dx;
      out[3] = g.db;
      if (need[1] || need[2]) {
        const Tensor z = saved[3].contiguous(), r = saved[4].contiguous();
        if (need[1]) out[1] = at::empty_like(z);
        if (need[2]) out[2] = at::empty_like(r);
        const bool f32 = c.dt == 0;
        const size_t n = !need[2] ? 0
                         : f32    ? moc_router_f32_backward_workspace_bytes(c.N, c.Z, c.K)
                                  : moc_router_backward_workspace_bytes(c.N, c.Z, c.K, 1);
        Tensor ws = n > 0 ? bytes(n, x) : Tensor();
        check(f32 ? moc_router_f32_backward(ptr(z), ptr(r), ptr(g.da), ptr(out[1]), ptr(out[2]), c.N, c.Z, c.K,
                                            ptr(ws), n, stream_of(x))
                  : moc_router_backward(ptr(z), ptr(r), ptr(g.da), ptr(out[1]), ptr(out[2]), c.N, c.Z, c.K, 1,
                                        ptr(ws), n, stream_of(x)),
              "moc_router_backward");
      }
    }
    return at::GradMode::is_enabled() ? once(std::move(out), grads) : out;
  }
};

// moc_triton on routing weights as one node (api._MoCFunction)
struct FuncFn : public torch::autograd::Function<FuncFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x0, const Tensor& a0, const Tensor& b0,
                        const Call* c) {
    const Tensor x = x0.contiguous(), a = a0.contiguous(), b = b0.contiguous();
    Tensor y = run_forward(*c, x, a, b, 0);
    ctx->save_for_backward({x, a, b, c->cu});
    keep(ctx, *c);
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Call c = kept(ctx, saved[3]);
    variable_list out(4);
    const bool need_x = ctx->needs_input_grad(0);
    {
      at::NoGradGuard ng;
      const c10::DeviceGuard dg(saved[0].device());
      const Grads g = run_backward(c, saved[0], saved[1], saved[2], grads[0], need_x, 0);
      out[0] = g.dx;
      out[1] = g.da;
      out[2] = g.db;
    }
    return at::GradMode::is_enabled() ? once(std::move(out), grads) : out;
  }
};

// y of MoC.forward without a cache, or nothing: not a call of this path
OptTensor layer(const Tensor& x, const Tensor& z, const Tensor& router, const Tensor& basis, int act, int route,
                const OptTensor& cu) {
  if (!unwatched() || !plain(x) || !plain(z) || !plain(router) || !plain(basis)) return std::nullopt;
  Call c{act, route};
  const c10::DeviceGuard dg(x.device());
  if (!sizes(c, x, basis, cu) || !router_ok(c, x, z, router)) return std::nullopt;
  if (wants_grad({&x, &z, &router, &basis})) return LayerFn::apply(x, z, router, basis, &c);
  at::NoGradGuard ng;
  return run_forward(c, x.contiguous(), run_router(c, z.contiguous(), router.contiguous(), route),
                     basis.contiguous(), route + 2);
}

// y of moc_triton without a cache, or nothing
OptTensor func(const Tensor& x, const Tensor& alpha, const Tensor& basis, int act, const OptTensor& cu) {
  if (!unwatched() || !plain(x) || !plain(alpha) || !plain(basis)) return std::nullopt;
  Call c{act, 0};
  const c10::DeviceGuard dg(x.device());
  if (!sizes(c, x, basis, cu) || alpha.scalar_type() != x.scalar_type() || alpha.device() != x.device() ||
      alpha.dim() != x.dim() || alpha.size(-1) != c.K || alpha.numel() != c.N * c.K)
    return std::nullopt;
  for (int64_t i = 0; i + 1 < x.dim(); ++i)
    if (alpha.size(i) != x.size(i)) return std::nullopt;
  if (wants_grad({&x, &alpha, &basis})) return FuncFn::apply(x, alpha, basis, &c);
  at::NoGradGuard ng;
  return run_forward(c, x.contiguous(), alpha.contiguous(), basis.contiguous(), 0);
}

// Whether a prompt's state is cheaper written by the forward launch than as a copy of
// its last rows after the plain forward.  It saves a launch and a slow transposed copy
// (bf16, 8 x 1024 tokens, D 2048, 16 routes, 4 taps: 27 -> 22 us), but the kernel with
// a cache to read walks a sequence's first S - 1 rows one tap at a time (8 taps, 8 x 3
// tokens: 6.3 us plain, 18.9), and in fp32 its larger tile costs more than the copy
// from about 2^22 elements on with more than 3 taps or 16 routes (8 x 2048 tokens, D
// 4096, 4 taps, 16 routes 126 -> 141; 6 taps, 32 routes 256 -> 309; 3 x 300 tokens, D
// 1544, 4 taps 12 -> 10).
bool state_in_forward(const Call& c) {
  if (c.T < c.S - 1) return false;
  return c.dt == 1 || c.N * c.D <= (int64_t(1) << 22) || (c.S <= 3 && c.K <= 16);
}

// (y, state or None) of MoC.forward with a cache or a final state, fixed length:
// one token per sequence and a cache: the decode step, in place on the cache
// (not differentiable); else without gradients only.  Nothing: not a call of
// this path
std::optional<std::tuple<Tensor, OptTensor>> stateful(const Tensor& x, const Tensor& z, const Tensor& router,
                                                      const Tensor& basis, const OptTensor& cache, int act,
                                                      int route, bool want) {
  if (!unwatched() || !plain(x) || !plain(z) || !plain(router) || !plain(basis)) return std::nullopt;
  Call c{act, route};
  const c10::DeviceGuard dg(x.device());
  if (!sizes(c, x, basis, std::nullopt) || z.dim() != 3) return std::nullopt;
  const int64_t B = x.size(0);
  if (cache.has_value()) {
    if (!plain(*cache) || cache->device() != x.device() || cache->scalar_type() != x.scalar_type() ||
        cache->dim() != 3 || cache->size(0) != B || cache->size(1) != c.D || cache->size(2) != c.S)
      return std::nullopt;
  }
  if (!router_ok(c, x, z, router)) return std::nullopt;
  if (cache.has_value() && c.T == 1) {
    const bool one = c.dt == 1 && cache->is_contiguous() && moc_decode_step_supported(B, c.Z, c.D, c.K, c.S);
    if (!one && c.dt == 1) return std::nullopt;
    at::NoGradGuard ng;
    const Tensor xc = x.contiguous(), zc = z.contiguous(), rc = router.contiguous(), bc = basis.contiguous();
    Tensor y = at::empty_like(xc);
    if (one) {
      check(moc_decode_step(ptr(zc), ptr(rc), ptr(xc), ptr(bc), ptr(*cache), ptr(y), B, c.Z, c.D, c.K, c.S, act,
                            route, stream_of(x)),
            "moc_decode_step");
    } else {
      const Tensor lg = run_router(c, zc, rc, 0);
      check(moc_update(ptr(xc), ptr(lg), ptr(bc), ptr(*cache), cache->stride(0), cache->stride(1),
                       cache->stride(2), ptr(y), B, c.D, c.K, c.S, c.dt, c.dt, c.dt, act, route, stream_of(x)),
            "moc_update");
    }
    return std::make_tuple(y, want ? cache : OptTensor());
  }
  if (wants_grad({&x, &z, &router, &basis, cache.has_value() ? &*cache : nullptr})) return std::nullopt;
  if (!moc_prefill_supported(B, c.T, c.D, c.K, c.S, c.dt, cache.has_value())) return std::nullopt;
  if (!cache.has_value() && !state_in_forward(c)) return std::nullopt;
  at::NoGradGuard ng;
  const Tensor xc = x.contiguous(), bc = basis.contiguous();
  const Tensor w = run_router(c, z.contiguous(), router.contiguous(), route);
  const Tensor hist = cache.has_value() ? cache->contiguous() : Tensor();
  Tensor y = at::empty_like(xc), fin;
  if (want) fin = at::empty({B, c.D, c.S}, x.options());
  Tensor ws = bytes(moc_forward_workspace_bytes(c.N, c.D, c.K, c.S, c.dt, route + 2), x);
  check(moc_forward_prefill(ptr(xc), ptr(w), ptr(bc), ptr(y), ptr(hist), ptr(fin), B, c.T, c.D, c.K, c.S, c.dt,
                            c.dt, c.dt, act, route + 2, ptr(ws), ws.numel(), stream_of(x)),
        "moc_forward_prefill");
  return std::make_tuple(y, want ? OptTensor(fin) : OptTensor());
}

// ---------------------------------------------------------------------------
// The operators next to the layers (moc/blocks.py), each as one call: with gradients
// as a node, else straight.  Us a call of small sizes, Python functions -> here: layer norm
// 10.9 -> 4.3, a step of the convolution 15.8 -> 5.1 and of the scan 23.8 -> 4.7; forward and
// gradients of the norm 112 -> 65, the convolution 108 -> 60, the scan 196 -> 100.

// a parameter's storage code (any floating dtype that the kernels read), or -1
int param_code(const Tensor& t) {
  if (!t.defined()) return 0;
  return t.scalar_type() == at::kHalf ? 2 : dtype_code(t.scalar_type());
}

// A parameter of the operators: absent, or plain, on x's device, of the shape and readable.
bool param_ok(const Tensor& t, const Tensor& x, at::IntArrayRef shape) {
  return !t.defined() || (plain(t) && t.device() == x.device() && t.sizes() == shape && param_code(t) >= 0);
}

Tensor like(const Tensor& t) { return t.defined() ? at::empty(t.sizes(), t.options()) : Tensor(); }
Tensor f32(at::IntArrayRef shape, const Tensor& x) { return at::empty(shape, x.options().dtype(at::kFloat)); }
Tensor dense(const Tensor& t) { return t.defined() ? t.contiguous() : t; }
// (a node takes what may be absent as an optional: an undefined tensor is no input of it)
OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }
Tensor dense(const OptTensor& t) { return t.has_value() ? t->contiguous() : Tensor(); }

// Which of a node's tensor inputs need a gradient; edges are counted over those present.
struct Needs {
  AutogradContext* ctx;
  size_t edge = 0;
  bool operator()(bool present) { return present && ctx->needs_input_grad(edge++); }
};

void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// The packed offsets, as the library takes them; false where they are not ones it takes.
bool offsets_ok(const OptTensor& cu, const Tensor& x) {
  return !cu.has_value() ||
         (plain(*cu) && cu->device() == x.device() && cu->dim() == 1 && cu->numel() >= 2 &&
          (cu->scalar_type() == at::kInt || cu->scalar_type() == at::kLong));
}

struct Packing {
  Tensor cu;
  int64_t tokens, seq_len;
  const void* p() const { return ptr(cu); }
  int i64() const { return cu.defined() && cu.scalar_type() == at::kLong; }
  int64_t n_seqs() const { return cu.defined() ? cu.numel() - 1 : 0; }
};

// --- layer norm

struct NormFn : public torch::autograd::Function<NormFn> {
  static Tensor run(const Tensor& x, const Tensor& w, const Tensor& b, double eps, Tensor* mean, Tensor* rstd) {
    const int64_t D = x.size(-1), rows = x.numel() / D;
    Tensor y = at::empty_like(x);
    if (mean != nullptr) {
      const Tensor both = f32({2, rows}, x);
      *mean = both.select(0, 0);
      *rstd = both.select(0, 1);
    }
    check(moc_norm_forward(ptr(x), ptr(w), ptr(b), ptr(y), static_cast<float*>(mean ? ptr(*mean) : nullptr),
                           static_cast<float*>(rstd ? ptr(*rstd) : nullptr), rows, D, dtype_code(x.scalar_type()),
                           param_code(w), param_code(b), static_cast<float>(eps), stream_of(x)),
          "moc_norm_forward");
    return y;
  }
  static Tensor forward(AutogradContext* ctx, const Tensor& x0, const OptTensor& w0, const OptTensor& b0, double eps) {
    const Tensor x = x0.contiguous(), w = dense(w0), b = dense(b0);
    Tensor mean, rstd;
    Tensor y = run(x, w, b, eps, &mean, &rstd);
    ctx->save_for_backward({x, w, b, mean, rstd});
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &b = saved[2];
    variable_list out(4);
    {
      at::NoGradGuard ng;
      const c10::DeviceGuard dg(x.device());
      const Tensor dy = grads[0].to(x.scalar_type()).contiguous();
      const int64_t D = x.size(-1), rows = x.numel() / D;
      Needs need{ctx};
      if (need(true)) out[0] = at::empty_like(x);
      if (need(w.defined())) out[1] = like(w);
      if (need(b.defined())) out[2] = like(b);
      const bool sums = out[1].defined() || out[2].defined();
      const size_t n = sums ? moc_norm_backward_workspace_bytes(rows, D) : 0;
      const Tensor ws = sums ? bytes(n, x) : Tensor();
      check(moc_norm_backward(ptr(x), ptr(w), ptr(dy), static_cast<float*>(ptr(saved[3])),
                              static_cast<float*>(ptr(saved[4])), ptr(out[0]), ptr(out[1]), ptr(out[2]), rows, D,
                              dtype_code(x.scalar_type()), param_code(w), param_code(b), ptr(ws), n, stream_of(x)),
            "moc_norm_backward");
    }
    return at::GradMode::is_enabled() ? once(std::move(out), grads) : out;
  }
};

OptTensor norm(const Tensor& x, const Tensor& w, const Tensor& b, double eps) {
  if (!unwatched() || !plain(x) || dtype_code(x.scalar_type()) < 0 || x.dim() < 1 || x.numel() == 0)
    return std::nullopt;
  if (!param_ok(w, x, {x.size(-1)}) || !param_ok(b, x, {x.size(-1)})) return std::nullopt;
  const c10::DeviceGuard dg(x.device());
  if (wants_grad({&x, &w, &b})) return NormFn::apply(x, opt(w), opt(b), eps);
  at::NoGradGuard ng;
  return NormFn::run(x.contiguous(), dense(w), dense(b), eps, nullptr, nullptr);
}

// --- causal convolution

struct ConvFn : public torch::autograd::Function<ConvFn> {
  static Tensor run(const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& cache, Tensor* fin, int act,
                    const Packing& k) {
    Tensor y = at::empty_like(x);
    check(moc_conv_forward(ptr(x), ptr(w), ptr(b), ptr(cache), ptr(y), fin ? ptr(*fin) : nullptr, k.p(), k.i64(),
                           k.n_seqs(), k.tokens, k.seq_len, w.size(1), w.size(0), dtype_code(x.scalar_type()),
                           param_code(w), param_code(b), act, stream_of(x)),
          "moc_conv_forward");
    return y;
  }
  static Tensor forward(AutogradContext* ctx, const Tensor& x0, const Tensor& w0, const OptTensor& b0, int64_t act,
                        const Packing* k) {
    const Tensor x = x0.contiguous(), w = dense(w0), b = dense(b0);
    Tensor y = run(x, w, b, Tensor(), nullptr, static_cast<int>(act), *k);
    ctx->save_for_backward({x, w, b, k->cu});
    ctx->saved_data["k"] = std::vector<int64_t>{act, k->tokens, k->seq_len};
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &b = saved[2];
    const auto v = ctx->saved_data["k"].toIntVector();
    const Packing k{saved[3], v[1], v[2]};
    variable_list out(5);
    {
      at::NoGradGuard ng;
      const c10::DeviceGuard dg(x.device());
      const Tensor dy = grads[0].to(x.scalar_type()).contiguous();
      Needs need{ctx};
      if (need(true)) out[0] = at::empty_like(x);
      if (need(true)) out[1] = like(w);
      if (need(b.defined())) out[2] = like(b);
      const bool sums = out[1].defined() || out[2].defined();
      const size_t n = sums ? moc_conv_backward_workspace_bytes(k.tokens, w.size(1), w.size(0), dtype_code(x.scalar_type())) : 0;
      const Tensor ws = sums ? bytes(n, x) : Tensor();
      check(moc_conv_backward(ptr(x), ptr(w), ptr(b), ptr(dy), ptr(out[0]), ptr(out[1]), ptr(out[2]), k.p(), k.i64(),
                              k.n_seqs(), k.tokens, k.seq_len, w.size(1), w.size(0), dtype_code(x.scalar_type()),
                              param_code(w), param_code(b), static_cast<int>(v[0]), ptr(ws), n, stream_of(x)),
            "moc_conv_backward");
    }
    return at::GradMode::is_enabled() ? once(std::move(out), grads) : out;
  }
};

// (y, state or None) of a fixed-length [B, T, D] or packed [N, D] x.  Nothing also where
// gradients flow with a cache or a final state (blocks.py puts those together).
std::optional<std::tuple<Tensor, OptTensor>> conv(const Tensor& x, const Tensor& w, const Tensor& b,
                                                  const OptTensor& cache, int act, bool want, const OptTensor& cu) {
  if (!unwatched() || !plain(x) || dtype_code(x.scalar_type()) < 0 || !w.defined() || w.dim() != 2) return std::nullopt;
  const int64_t S = w.size(0), D = w.size(1);
  if (x.dim() != (cu.has_value() ? 2 : 3) || x.size(-1) != D || x.numel() == 0 || S < 1 || S > 16) return std::nullopt;
  if (!param_ok(w, x, {S, D}) || !param_ok(b, x, {D}) || !offsets_ok(cu, x)) return std::nullopt;
  if (cu.has_value() && (cache.has_value() || want)) return std::nullopt;
  if (cache.has_value() && (!plain(*cache) || cache->device() != x.device() || cache->scalar_type() != x.scalar_type() ||
                            cache->sizes() != at::IntArrayRef({x.size(0), D, S})))
    return std::nullopt;
  const c10::DeviceGuard dg(x.device());
  const Packing k{cu.has_value() ? cu->contiguous() : Tensor(), x.numel() / D, cu.has_value() ? 0 : x.size(1)};
  if (cache.has_value() && x.size(1) == 1) {
    for (int64_t i = 0; i < 3; ++i)
      if (cache->size(i) > 1 && cache->stride(i) == 0) return std::nullopt;
    at::NoGradGuard ng;
    const Tensor xc = x.contiguous(), wc = dense(w), bc = dense(b);
    Tensor y = at::empty_like(xc);
    check(moc_conv_update(ptr(xc), ptr(wc), ptr(bc), ptr(*cache), cache->stride(0), cache->stride(1), cache->stride(2),
                          ptr(y), x.size(0), D, S, dtype_code(x.scalar_type()), param_code(w), param_code(b), act,
                          stream_of(x)),
          "moc_conv_update");
    written(*cache);
    return std::make_tuple(y, want ? cache : OptTensor());
  }
  if (wants_grad({&x, &w, &b, cache.has_value() ? &*cache : nullptr})) {
    if (cache.has_value() || want) return std::nullopt;
    return std::make_tuple(ConvFn::apply(x, w, opt(b), static_cast<int64_t>(act), &k), OptTensor());
  }
  at::NoGradGuard ng;
  Tensor fin = want ? at::empty({x.size(0), D, S}, x.options()) : Tensor();
  Tensor y = ConvFn::run(x.contiguous(), dense(w), dense(b), cache.has_value() ? cache->contiguous() : Tensor(),
                         want ? &fin : nullptr, act, k);
  return std::make_tuple(y, want ? OptTensor(fin) : OptTensor());
}

// --- selective scan

// ops.token_rows: t itself where a token's `inner` dimensions are contiguous and tokens
// evenly apart (below 2^31 elements), a copy otherwise
Tensor token_rows(const Tensor& t, int64_t inner, int64_t& step) {
  const int64_t lead = t.dim() - inner;
  int64_t n = 1;
  bool ok = true;
  for (int64_t i = t.dim() - 1; i >= lead; --i) {
    ok = ok && (t.size(i) == 1 || t.stride(i) == n);
    n *= t.size(i);
  }
  step = n;
  bool any = false;
  for (int64_t i = lead - 1; i >= 0; --i) {
    if (t.size(i) == 1) continue;
    if (!any) step = t.stride(i);
    else ok = ok && t.stride(i) == t.size(lead - 1) * step;
    any = true;
  }
  if (ok && step >= n && step < int64_t(1) << 31) return t;
  step = n;
  return t.contiguous();
}

// The inputs of a scan and the library's table of them.
struct ScanCall {
  Tensor x, dt, A, B, C, D, bias;
  Packing k;
  int softplus;
  MocScan table() {
    MocScan t{};
    x = token_rows(x, 2, t.x_stride);
    dt = token_rows(dt, 1, t.dt_stride);
    B = token_rows(B, 2, t.b_stride);
    C = token_rows(C, 2, t.c_stride);
    A = dense(A), D = dense(D), bias = dense(bias);
    t.x = ptr(x), t.dt = ptr(dt), t.a = ptr(A), t.b = ptr(B), t.c = ptr(C), t.d = ptr(D), t.dt_bias = ptr(bias);
    t.cu_seqlens = k.p(), t.cu_seqlens_i64 = k.i64(), t.n_seqs = k.n_seqs();
    t.n_tokens = k.tokens, t.seq_len = k.seq_len;
    t.heads = x.size(-2), t.head_dim = x.size(-1), t.groups = B.size(-2), t.state_dim = B.size(-1);
    t.x_dtype = dtype_code(x.scalar_type()), t.a_dtype = param_code(A), t.d_dtype = param_code(D);
    t.bias_dtype = param_code(bias), t.dt_softplus = softplus;
    return t;
  }
  // (y, final state); saved: what the backward reads
  Tensor run(const Tensor& init, Tensor* fin, Tensor* saved) {
    const MocScan t = table();
    Tensor y = at::empty(x.sizes(), x.options());
    const auto size = [](size_t n) {
      TORCH_CHECK(n > 0 || moc_last_error()[0] == 0, "moc_scan_forward: ", moc_last_error());
      return n;
    };
    if (fin != nullptr) *fin = f32({x.size(0), t.heads, t.head_dim, t.state_dim}, x);
    if (saved != nullptr) *saved = bytes(size(moc_scan_saved_bytes(&t)), x);
    const Tensor ws = bytes(size(moc_scan_forward_workspace_bytes(&t, saved != nullptr)), x);
    check(moc_scan_forward(&t, ptr(y), static_cast<float*>(ptr(init)), static_cast<float*>(fin ? ptr(*fin) : nullptr),
                           saved ? ptr(*saved) : nullptr, saved ? saved->numel() : 0, ptr(ws), ws.numel(),
                           stream_of(x)),
          "moc_scan_forward");
    return y;
  }
};

struct ScanFn : public torch::autograd::Function<ScanFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B,
                               const Tensor& C, const OptTensor& D, const OptTensor& bias, const OptTensor& cache,
                               int64_t softplus, bool want, const Packing* k) {
    ScanCall c{x, dt, A, B, C, dense(D), dense(bias), *k, static_cast<int>(softplus)};
    Tensor fin, saved;
    const Tensor init = dense(cache);
    Tensor y = c.run(init, want ? &fin : nullptr, &saved);
    ctx->save_for_backward({c.x, c.dt, c.A, c.B, c.C, c.D, c.bias, saved, k->cu});
    ctx->saved_data["k"] = std::vector<int64_t>{softplus, init.defined(), k->tokens, k->seq_len};
    ctx->set_materialize_grads(false);
    if (want) return {y, fin};
    return {y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const auto v = ctx->saved_data["k"].toIntVector();
    ScanCall c{saved[0], saved[1], saved[2], saved[3], saved[4], saved[5], saved[6], Packing{saved[8], v[2], v[3]},
               static_cast<int>(v[0])};
    variable_list out(11);
    const Tensor &dy0 = grads[0], dfin0 = grads.size() > 1 ? grads[1] : Tensor();
    if (!dy0.defined() && !dfin0.defined()) return out;
    {
      at::NoGradGuard ng;
      const c10::DeviceGuard dg(c.x.device());
      const MocScan t = c.table();
      const Tensor dy = dy0.defined() ? dy0.to(c.x.scalar_type()).contiguous() : at::zeros(c.x.sizes(), c.x.options());
      const Tensor dfin = dfin0.defined() ? dfin0.to(at::kFloat).contiguous() : Tensor();
      const Tensor ins[7] = {c.x, c.dt, c.A, c.B, c.C, c.D, c.bias};
      Needs need{ctx};
      bool needs[7];
      for (int i = 0; i < 7; ++i) {
        out[i] = like(ins[i]);
        needs[i] = need(ins[i].defined());
      }
      if (need(v[1] != 0)) out[7] = f32({c.x.size(0), t.heads, t.head_dim, t.state_dim}, c.x);
      const MocScanGrads g{ptr(out[0]), ptr(out[1]), ptr(out[2]), ptr(out[3]), ptr(out[4]), ptr(out[5]), ptr(out[6]),
                           static_cast<float*>(ptr(out[7]))};
      const Tensor ws = bytes(moc_scan_backward_workspace_bytes(&t), c.x);
      check(moc_scan_backward(&t, ptr(dy), v[1] != 0, static_cast<float*>(ptr(dfin)), ptr(saved[7]), saved[7].numel(),
                              &g, ptr(ws), ws.numel(), stream_of(c.x)),
            "moc_scan_backward");
      for (int i = 0; i < 7; ++i)
        if (!needs[i]) out[i] = Tensor();
    }
    return at::GradMode::is_enabled() ? once(std::move(out), grads) : out;
  }
};

// (y, state or None) of fixed-length [B, T, ..] or packed [N, ..] inputs
std::optional<std::tuple<Tensor, OptTensor>> scan(const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B,
                                                  const Tensor& C, const Tensor& D, const Tensor& bias,
                                                  const OptTensor& cache, bool softplus, bool want, const OptTensor& cu) {
  const int64_t lead = cu.has_value() ? 1 : 2;
  if (!unwatched() || dtype_code(x.scalar_type()) < 0 || x.dim() != lead + 2 || dt.dim() != lead + 1 ||
      B.dim() != lead + 2 || C.sizes() != B.sizes())
    return std::nullopt;
  for (const Tensor* t : {&x, &dt, &B, &C})
    if (!plain(*t) || t->device() != x.device() || t->scalar_type() != x.scalar_type() || t->numel() == 0 ||
        t->sizes().slice(0, lead) != x.sizes().slice(0, lead))
      return std::nullopt;
  const int64_t H = x.size(-2), P = x.size(-1), G = B.size(-2), N = B.size(-1);
  if (dt.size(-1) != H || H % G != 0 || P > 128 || N > 256 || !A.defined()) return std::nullopt;
  if (!param_ok(A, x, {H}) || !param_ok(D, x, {H}) || !param_ok(bias, x, {H}) || !offsets_ok(cu, x)) return std::nullopt;
  if (cu.has_value() && (cache.has_value() || want)) return std::nullopt;
  if (cache.has_value() && (!plain(*cache) || cache->device() != x.device() || cache->scalar_type() != at::kFloat ||
                            cache->sizes() != at::IntArrayRef({x.size(0), H, P, N})))
    return std::nullopt;
  const c10::DeviceGuard dg(x.device());
  const Packing k{cu.has_value() ? cu->contiguous() : Tensor(), x.numel() / (H * P), cu.has_value() ? 0 : x.size(1)};
  if (cache.has_value() && x.size(1) == 1) {
    if (!cache->is_contiguous()) return std::nullopt;
    at::NoGradGuard ng;
    ScanCall c{x, dt, A, B, C, D, bias, k, softplus};
    const MocScan t = c.table();
    Tensor y = at::empty(x.sizes(), x.options());
    check(moc_scan_update(&t, static_cast<float*>(ptr(*cache)), ptr(y), stream_of(x)), "moc_scan_update");
    written(*cache);
    return std::make_tuple(y, want ? cache : OptTensor());
  }
  if (wants_grad({&x, &dt, &A, &B, &C, &D, &bias, cache.has_value() ? &*cache : nullptr})) {
    const auto out = ScanFn::apply(x, dt, A, B, C, opt(D), opt(bias), cache, static_cast<int64_t>(softplus), want, &k);
    return std::make_tuple(out[0], want ? OptTensor(out[1]) : OptTensor());
  }
  at::NoGradGuard ng;
  ScanCall c{x, dt, A, B, C, D, bias, k, softplus};
  Tensor fin;
  Tensor y = c.run(cache.has_value() ? cache->contiguous() : Tensor(), want ? &fin : nullptr, nullptr);
  return std::make_tuple(y, want ? OptTensor(fin) : OptTensor());
}

// the nodes' Python type, under the name of the Python function they stand for
template <typename F>
void name_node(const char* name) {
  static PyTypeObject type{};
  torch::autograd::_initFunctionPyTypeObject(type, name, nullptr, nullptr);
  torch::autograd::registerCppFunction(typeid(torch::autograd::CppNode<F>), &type);
}

// A call's tensor arguments as Python hands them over.  Only torch.Tensor and
// torch.nn.Parameter themselves are taken: a subclass, with or without a dispatch
// key of its own, keeps its result type and its __torch_function__ in the Python
// functions, and what is no tensor its error there.  The calls then run without the
// interpreter lock: an allocation may wait for the device and a launch for space in
// the queue, and other threads' work goes on meanwhile (saved-tensor hooks take the
// lock themselves).
struct Args {
  bool own = true;
  Tensor operator()(py::handle h) {
    own = own && THPVariable_CheckExact(h.ptr());
    return own ? THPVariable_Unpack(h.ptr()) : Tensor();
  }
  OptTensor opt(py::handle h) { return h.is_none() ? OptTensor() : OptTensor((*this)(h)); }
  Tensor or_none(py::handle h) { return h.is_none() ? Tensor() : (*this)(h); }
};

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  name_node<LayerFn>("_MoCLayerFunctionBackward");
  name_node<FuncFn>("_MoCFunctionBackward");
  name_node<NormFn>("_LayerNormFunctionBackward");
  name_node<ConvFn>("_CausalConvFunctionBackward");
  name_node<ScanFn>("_SelectiveScanFunctionBackward");
  m.def("norm", [](py::handle x, py::handle w, py::handle b, double eps) -> OptTensor {
    Args a;
    const Tensor tx = a(x), tw = a.or_none(w), tb = a.or_none(b);
    if (!a.own) return std::nullopt;
    const py::gil_scoped_release unlocked;
    return norm(tx, tw, tb, eps);
  });
  m.def("conv", [](py::handle x, py::handle w, py::handle b, py::handle cache, int act, bool want,
                   py::handle cu) -> std::optional<std::tuple<Tensor, OptTensor>> {
    Args a;
    const Tensor tx = a(x), tw = a(w), tb = a.or_none(b);
    const OptTensor tc = a.opt(cache), tu = a.opt(cu);
    if (!a.own) return std::nullopt;
    const py::gil_scoped_release unlocked;
    return conv(tx, tw, tb, tc, act, want, tu);
  });
  m.def("scan", [](py::handle x, py::handle dt, py::handle A, py::handle B, py::handle C, py::handle D, py::handle bias,
                   py::handle cache, bool softplus, bool want,
                   py::handle cu) -> std::optional<std::tuple<Tensor, OptTensor>> {
    Args a;
    const Tensor tx = a(x), tdt = a(dt), tA = a(A), tB = a(B), tC = a(C), tD = a.or_none(D), tb = a.or_none(bias);
    const OptTensor tc = a.opt(cache), tu = a.opt(cu);
    if (!a.own) return std::nullopt;
    const py::gil_scoped_release unlocked;
    return scan(tx, tdt, tA, tB, tC, tD, tb, tc, softplus, want, tu);
  });
  m.def("layer", [](py::handle x, py::handle z, py::handle router, py::handle basis, int act, int route,
                    py::handle cu) -> OptTensor {
    Args a;
    const Tensor tx = a(x), tz = a(z), tr = a(router), tb = a(basis);
    const OptTensor tc = a.opt(cu);
    if (!a.own) return std::nullopt;
    const py::gil_scoped_release unlocked;
    return layer(tx, tz, tr, tb, act, route, tc);
  });
  m.def("func", [](py::handle x, py::handle alpha, py::handle basis, int act, py::handle cu) -> OptTensor {
    Args a;
    const Tensor tx = a(x), ta = a(alpha), tb = a(basis);
    const OptTensor tc = a.opt(cu);
    if (!a.own) return std::nullopt;
    const py::gil_scoped_release unlocked;
    return func(tx, ta, tb, act, tc);
  });
  m.def("stateful", [](py::handle x, py::handle z, py::handle router, py::handle basis, py::handle cache, int act,
                       int route, bool want) -> std::optional<std::tuple<Tensor, OptTensor>> {
    Args a;
    const Tensor tx = a(x), tz = a(z), tr = a(router), tb = a(basis);
    const OptTensor tc = a.opt(cache);
    if (!a.own) return std::nullopt;
    const py::gil_scoped_release unlocked;
    return stateful(tx, tz, tr, tb, tc, act, route, want);
  });
}
