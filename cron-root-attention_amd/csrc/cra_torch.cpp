// Torch operator binding of libcra_hip.so (include/cra.h) with its autograd
// in C++: torch.ops.cra.attention(q, k, v, window, relay, top_k, scale), and
// layer_attention, the same over [B, S, H, D] buffers.
//
// It serves the common call of cron_root_attention_v14 (reference
// core.py:3767-3797) -- GPU tensors, head dim 32/64/128/256, no
// relay_log_scale, the tiled forward -- with the
// same launches as the Python autograd Function (cra_build_global + cra_fwd,
// then cra_bwd) but without the Python autograd and ctypes layers, which at
// small S cost more host time than the kernels take on the GPU. Layouts the
// kernels cannot take are copied to contiguous ones here, as the Python path
// does. Everything else (padded head dims, relay scale, the persistent kernel,
// varlen, CPU tensors) stays on the Python path; both reach the same C ABI.
//
// Beside them: rotary (rotary positions and head norms of q and k, with their
// autograd), cache_write, cache_append and paged_attention (a paged cache and the
// attention of new tokens over it), for the same reason: at a few rows a call's host time is what
// it costs.
//
// The library is bound at run time (cra::bind(path)) so that the op uses the
// very library the Python binding loaded.
#include <dlfcn.h>

#include <atomic>
#include <cmath>
#include <mutex>
#include <string>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/autograd.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include "cra.h"

namespace {

struct Api {
  decltype(&cra_global_rows) global_rows = nullptr;
  decltype(&cra_reads_global_rows) reads_global = nullptr;
  decltype(&cra_build_global) build_global = nullptr;
  decltype(&cra_fwd) fwd = nullptr;
  decltype(&cra_fwd_inplace) fwd_inplace = nullptr;
  decltype(&cra_bwd_workspace_bytes) ws_bytes = nullptr;
  decltype(&cra_bwd) bwd = nullptr;
  decltype(&cra_bwd_inplace) bwd_inplace = nullptr;
  decltype(&cra_rotary) rotary = nullptr;
  decltype(&cra_rotary_bwd_workspace_bytes) rotary_ws = nullptr;
  decltype(&cra_norm_rotary_bwd) norm_rotary_bwd = nullptr;
  decltype(&cra_cache_write) cache_write = nullptr;
  decltype(&cra_cache_append) cache_append = nullptr;
  decltype(&cra_fwd_paged_workspace_bytes) paged_ws = nullptr;
  decltype(&cra_fwd_paged) fwd_paged = nullptr;
  decltype(&cra_fwd_paged_shared_workspace_bytes) shared_ws = nullptr;
  decltype(&cra_fwd_paged_shared) fwd_shared = nullptr;
  decltype(&cra_linear_e4m3_workspace_bytes) linear_ws = nullptr;
  decltype(&cra_linear_e4m3) linear_e4m3 = nullptr;
  decltype(&cra_strerror) strerror_ = nullptr;
  decltype(&cra_last_error) last_error = nullptr;
  decltype(&cra_abi_version) abi_version = nullptr;
};

// Written once under g_mu by bind(); g_bound is published last (release) and
// read with acquire, so a reader that sees it set sees the whole table.
std::mutex g_mu;
Api g_api;
std::atomic<bool> g_bound{false};

template <typename F>
void resolve(void* h, const std::string& path, const char* name, F& out) {
  void* f = dlsym(h, name);
  TORCH_CHECK(f != nullptr, path, " does not export ", name);
  out = reinterpret_cast<F>(f);
}

void bind(std::string path) {
  std::lock_guard<std::mutex> lk(g_mu);
  void* h = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);
  TORCH_CHECK(h != nullptr, "cannot load ", path, ": ", dlerror());
  Api api;
  resolve(h, path, "cra_global_rows", api.global_rows);
  resolve(h, path, "cra_reads_global_rows", api.reads_global);
  resolve(h, path, "cra_build_global", api.build_global);
  resolve(h, path, "cra_fwd", api.fwd);
  resolve(h, path, "cra_fwd_inplace", api.fwd_inplace);
  resolve(h, path, "cra_bwd_workspace_bytes", api.ws_bytes);
  resolve(h, path, "cra_bwd", api.bwd);
  resolve(h, path, "cra_bwd_inplace", api.bwd_inplace);
  resolve(h, path, "cra_rotary", api.rotary);
  resolve(h, path, "cra_rotary_bwd_workspace_bytes", api.rotary_ws);
  resolve(h, path, "cra_norm_rotary_bwd", api.norm_rotary_bwd);
  resolve(h, path, "cra_cache_write", api.cache_write);
  resolve(h, path, "cra_cache_append", api.cache_append);
  resolve(h, path, "cra_fwd_paged_workspace_bytes", api.paged_ws);
  resolve(h, path, "cra_fwd_paged", api.fwd_paged);
  resolve(h, path, "cra_fwd_paged_shared_workspace_bytes", api.shared_ws);
  resolve(h, path, "cra_fwd_paged_shared", api.fwd_shared);
  resolve(h, path, "cra_linear_e4m3_workspace_bytes", api.linear_ws);
  resolve(h, path, "cra_linear_e4m3", api.linear_e4m3);
  resolve(h, path, "cra_strerror", api.strerror_);
  resolve(h, path, "cra_last_error", api.last_error);
  resolve(h, path, "cra_abi_version", api.abi_version);
  TORCH_CHECK(api.abi_version() == CRA_ABI_VERSION, path, ": ABI ", api.abi_version(),
              " != ", CRA_ABI_VERSION);
  if (g_bound.load(std::memory_order_acquire)) {
    // already bound (a second bind is a no-op unless it names another library)
    TORCH_CHECK(api.fwd == g_api.fwd, "cra::bind: already bound to another library");
    return;
  }
  g_api = api;
  g_bound.store(true, std::memory_order_release);
}

const Api& api() {
  TORCH_CHECK(g_bound.load(std::memory_order_acquire),
              "cra::attention: library not bound (call torch.ops.cra.bind first)");
  return g_api;
}

void check(int code, const char* func) {
  if (code == CRA_OK) return;
  const char* msg = api().last_error();
  TORCH_CHECK(false, func, ": ", (msg && *msg) ? msg : api().strerror_(code), " (code ", code,
              ")");
}

int32_t dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kHalf: return CRA_F16;
    case at::kBFloat16: return CRA_BF16;
    case at::kFloat: return CRA_F32;
    default: TORCH_CHECK(false, "cra::attention: unsupported dtype ", t);
  }
  return -1;
}

cra_tensor targ(const at::Tensor& t) {
  return cra_tensor{t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)};
}

// D contiguous, 16-byte aligned rows, one head within 2 GiB: what the kernels
// address.
bool kernel_ready(const at::Tensor& t) {
  const int64_t es = t.element_size(), vec = 16 / es;
  const int64_t span = ((t.size(2) - 1) * t.stride(2) + t.size(3)) * es;
  return t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 &&
         span < (int64_t(1) << 31) && t.stride(0) % vec == 0 && t.stride(1) % vec == 0 &&
         t.stride(2) % vec == 0;
}

cra_problem make_problem(const at::Tensor& q, const at::Tensor& k, int64_t window, bool relay,
                         int64_t top_k, double scale) {
  cra_problem p;
  p.B = (int32_t)q.size(0);
  p.H_q = (int32_t)q.size(1);
  p.H_kv = (int32_t)k.size(1);
  p.S = (int32_t)q.size(2);
  p.D = (int32_t)q.size(3);
  p.W = (int32_t)window;
  p.relay = relay ? 1 : 0;
  p.top_k = relay ? (int32_t)top_k : 0;
  p.dtype = dtype_code(q.scalar_type());
  p.scale = (float)scale;
  return p;
}

void* stream_of(const at::Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

// Addresses of the packed K and V rows.
std::pair<char*, char*> glob_ptrs(const at::Tensor& gkv) {
  char* p = static_cast<char*>(gkv.data_ptr());
  return {p, p + gkv.numel() / 2 * gkv.element_size()};
}

// A [B, H, S, D] tensor like t: contiguous, or with bshd a view of a
// contiguous [B, S, H, D] one, the layout a projection takes and gives. A layer
// that asks for it saves the copies between the two: at B=1 S=16000 H=16/4
// D=128 one of the output (50 us) and one of each of dq, dk, dv (50 + 2 x 17).
at::Tensor empty_bhsd(const at::Tensor& t, bool bshd) {
  if (!bshd) return at::empty(t.sizes(), t.options());
  return at::empty({t.size(0), t.size(2), t.size(1), t.size(3)}, t.options()).transpose(1, 2);
}

// Forward launches: packed global rows (one allocation for K and V rows) and
// relay source rows where the call needs them, then the three-phase forward.
// Returns o, lse, the packed rows and the relay source rows (either may be
// undefined). At S = 512 the packing was 3 of the call's 12 us on the GPU.
std::array<at::Tensor, 4> run_forward(const cra_problem& p, const at::Tensor& q,
                                      const at::Tensor& k, const at::Tensor& v, bool bshd) {
  const Api& a = api();
  void* st = stream_of(q);
  const int reads = a.reads_global(&p, targ(k), targ(v));
  TORCH_CHECK(reads >= 0, "cra_reads_global_rows: invalid problem");
  at::Tensor gkv, src;
  if (reads) {
    const int64_t G = a.global_rows(&p);
    TORCH_CHECK(G >= 0, "cra_global_rows: invalid problem");
    gkv = at::empty({2, p.B, p.H_kv, G, p.D}, k.options());
    if (p.relay) {
      const int64_t nb = (p.S + p.W - 1) / p.W;
      src = at::empty({p.B, p.H_kv, nb * p.top_k}, k.options().dtype(at::kInt));
    }
    const auto [gk, gv] = glob_ptrs(gkv);
    check(a.build_global(&p, targ(k), targ(v), gk, gv, p.relay ? src.data_ptr<int32_t>() : nullptr,
                         nullptr, st),
          "cra_build_global");
  }
  at::Tensor o = empty_bhsd(q, bshd);
  at::Tensor lse = at::empty({p.B, p.H_q, p.S}, q.options().dtype(at::kFloat));
  if (reads) {
    const auto [gk, gv] = glob_ptrs(gkv);
    check(a.fwd(&p, targ(q), targ(k), targ(v), gk, gv, targ(o), lse.data_ptr<float>(), st),
          "cra_fwd");
  } else {
    check(a.fwd_inplace(&p, targ(q), targ(k), targ(v), targ(o), lse.data_ptr<float>(), st),
          "cra_fwd_inplace");
  }
  return {o, lse, gkv, src};
}

void check_inputs(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v) {
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && v.dim() == 4, "q, k, v must be [B, H, S, D]");
  TORCH_CHECK(q.is_cuda() && k.device() == q.device() && v.device() == q.device(),
              "cra::attention: q, k, v must be on one GPU");
  TORCH_CHECK(k.sizes() == v.sizes() && k.size(0) == q.size(0) && k.size(2) == q.size(2) &&
                  k.size(3) == q.size(3) && q.size(1) % k.size(1) == 0,
              "cra::attention: shapes do not match");
  TORCH_CHECK(q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type(),
              "cra::attention: q, k, v dtypes differ");
  const int64_t D = q.size(3);
  TORCH_CHECK(D == 32 || D == 64 || D == 128 || D == 256,
              "cra::attention: head dim must be 32, 64, 128 or 256");
}

// The tensor itself when the kernels take its layout, else a contiguous copy
// (what the Python path does).
at::Tensor ready(const at::Tensor& t) { return kernel_ready(t) ? t : t.contiguous(); }

class CraAttention : public torch::autograd::Function<CraAttention> {
 public:
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& q_in,
                            const at::Tensor& k_in, const at::Tensor& v_in, int64_t window,
                            bool relay, int64_t top_k, double scale, bool bshd) {
    check_inputs(q_in, k_in, v_in);
    const at::Tensor q = ready(q_in), k = ready(k_in), v = ready(v_in);
    const cra_problem p = make_problem(q, k, window, relay, top_k, scale);
    auto r = run_forward(p, q, k, v, bshd);
    ctx->save_for_backward({q, k, v, r[0], r[1], r[2], r[3]});
    ctx->saved_data["window"] = window;
    ctx->saved_data["relay"] = relay;
    ctx->saved_data["top_k"] = top_k;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["bshd"] = bshd;
    return r[0];
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const at::Tensor &q = s[0], &o = s[3], &lse = s[4], &gkv = s[5], &src = s[6];
    at::Tensor k = s[1], v = s[2];
    const cra_problem p =
        make_problem(q, k, ctx->saved_data["window"].toInt(), ctx->saved_data["relay"].toBool(),
                     ctx->saved_data["top_k"].toInt(), ctx->saved_data["scale"].toDouble());
    at::Tensor dout = grads[0].to(q.scalar_type());
    if (!kernel_ready(dout)) dout = dout.contiguous();
    const Api& a = api();
    void* st = stream_of(q);
    if (!gkv.defined() && a.reads_global(&p, targ(k), targ(v)) != 0) {
      // nothing was packed, and a saved-tensor hook gave k and v back in
      // layouts that would need it
      k = k.contiguous();
      v = v.contiguous();
    }
    const bool bshd = ctx->saved_data["bshd"].toBool();
    at::Tensor dq = empty_bhsd(q, bshd), dk = empty_bhsd(k, bshd), dv = empty_bhsd(v, bshd);
    const size_t nws = a.ws_bytes(&p);
    at::Tensor ws = at::empty({(int64_t)std::max<size_t>(nws, 256)}, q.options().dtype(at::kByte));
    if (gkv.defined()) {
      const auto [gk, gv] = glob_ptrs(gkv);
      check(a.bwd(&p, targ(q), targ(k), targ(v), targ(o), targ(dout), lse.data_ptr<float>(), gk, gv,
                  p.relay ? src.data_ptr<int32_t>() : nullptr, nullptr, targ(dq), targ(dk),
                  targ(dv), nullptr, ws.data_ptr(), (size_t)ws.numel(), st),
            "cra_bwd");
    } else {
      check(a.bwd_inplace(&p, targ(q), targ(k), targ(v), targ(o), targ(dout),
                          lse.data_ptr<float>(), targ(dq), targ(dk), targ(dv), ws.data_ptr(),
                          (size_t)ws.numel(), st),
            "cra_bwd_inplace");
    }
    return {dq, dk, dv, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

template <bool BSHD>
at::Tensor attention_autograd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                              int64_t window, bool relay, int64_t top_k, double scale) {
  return CraAttention::apply(q, k, v, window, relay, top_k, scale, BSHD);
}

// Below autograd (inference mode, or tensors without autograd keys): the
// forward launches alone.
template <bool BSHD>
at::Tensor attention_forward(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                             int64_t window, bool relay, int64_t top_k, double scale) {
  check_inputs(q, k, v);
  const at::Tensor qr = ready(q), kr = ready(k), vr = ready(v);
  return run_forward(make_problem(qr, kr, window, relay, top_k, scale), qr, kr, vr, BSHD)[0];
}

// ---------------------------------------------------------------------------
// Rotary positions and head norms, the paged cache and the attention over it. An
// argument that the calls below do not take (and any invalid one) makes them
// return nothing; the Python layer then serves the call its own way, or raises.
// ---------------------------------------------------------------------------
using OptTensor = std::optional<at::Tensor>;

at::Tensor get(const OptTensor& t) { return t.has_value() ? *t : at::Tensor(); }

bool float_type(at::ScalarType t) { return t == at::kHalf || t == at::kBFloat16 || t == at::kFloat; }

// As targ, the stride of a dimension of one element (which is never taken) as 0.
cra_tensor row_arg(const at::Tensor& t) {
  if (!t.defined()) return cra_tensor{nullptr, 0, 0, 0};
  auto st = [&](int d) { return t.size(d) > 1 ? t.stride(d) : 0; };
  return cra_tensor{t.data_ptr(), st(0), st(1), st(2)};
}

void* ptr_of(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

at::Tensor rows_of(const at::Tensor& t) {
  return !t.defined() || t.stride(3) == 1 || t.size(3) == 1 ? t : t.contiguous();
}

// Whether the sizes fit the C ABI's 32-bit ones.
bool sizes_fit(const at::Tensor& t) {
  for (int64_t n : t.sizes())
    if (n > INT32_MAX) return false;
  return true;
}

// Gradients that are not differentiated again: under create_graph they carry a node
// that raises when they are.
torch::autograd::variable_list once(torch::autograd::variable_list out, const char* name) {
  if (!at::GradMode::is_enabled()) return out;
  auto node = std::make_shared<torch::autograd::DelayedError>(
      std::string(name) + " has no second derivative", (int64_t)out.size());
  for (at::Tensor& t : out)
    if (t.defined()) t = t.detach().set_requires_grad(true);
  return (*node)(std::move(out));
}

struct Turn {
  bool norm, interleaved;
  double eps;
  at::Tensor table, pos;  // either may be undefined
};

cra_turn make_turn(const Turn& t, const at::Tensor& q, const at::Tensor& k, bool norm,
                   const at::Tensor& w) {
  cra_turn p{};
  p.B = (int32_t)q.size(0);
  p.H_q = (int32_t)q.size(1);
  p.H_kv = k.defined() ? (int32_t)k.size(1) : 0;
  p.S = (int32_t)q.size(2);
  p.D = (int32_t)q.size(3);
  p.dtype = dtype_code(q.scalar_type());
  p.weight_dtype = w.defined() ? dtype_code(w.scalar_type()) : p.dtype;
  p.norm = norm;
  p.eps = (float)t.eps;
  if (t.table.defined() && t.table.size(1) > 0) {
    p.rot = (int32_t)t.table.size(1);
    p.interleaved = t.interleaved;
    p.table = t.table.data_ptr<float>();
    p.table_rows = t.table.size(0);
    if (t.pos.defined()) {
      const int s = (int)t.pos.dim() - 1;  // [S] or [B or 1, S]
      p.positions = t.pos.data_ptr();
      p.positions_64 = t.pos.scalar_type() == at::kLong;
      p.psb = s == 1 && t.pos.size(0) > 1 ? t.pos.stride(0) : 0;
      p.pss = t.pos.stride(s);
    }
  }
  return p;
}

std::array<at::Tensor, 2> run_rotary(const Turn& t, const at::Tensor& q, const at::Tensor& k,
                                     const at::Tensor& wq, const at::Tensor& wk, bool norm,
                                     bool transpose) {
  c10::DeviceGuard guard(q.device());
  at::Tensor yq = at::empty_like(q), yk;
  if (k.defined()) yk = at::empty_like(k);
  const cra_turn p = make_turn(t, q, k, norm, wq.defined() ? wq : wk);
  check(api().rotary(&p, row_arg(q), row_arg(k), ptr_of(wq), ptr_of(wk), row_arg(yq), row_arg(yk),
                     transpose, stream_of(q)),
        "cra_rotary");
  return {yq, yk};
}

class CraRotary : public torch::autograd::Function<CraRotary> {
 public:
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx,
                                                const at::Tensor& q_in, const OptTensor& k_in,
                                                const OptTensor& wq_in, const OptTensor& wk_in,
                                                const OptTensor& table_in, const OptTensor& pos_in,
                                                bool interleaved, bool norm, double eps) {
    const at::Tensor q = rows_of(q_in), k = rows_of(get(k_in));
    const at::Tensor wq = get(wq_in), wk = get(wk_in), table = get(table_in), pos = get(pos_in);
    const Turn t{norm, interleaved, eps, table, pos};
    ctx->set_materialize_grads(false);
    if (norm)
      ctx->save_for_backward({q, k, wq, wk, table, pos});
    else  // the rotation's backward needs none of its inputs
      ctx->save_for_backward({at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), table, pos});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["norm"] = norm;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["dtype"] = q.scalar_type();
    const auto y = run_rotary(t, q, k, wq, wk, norm, false);
    if (k.defined()) return {y[0], y[1]};
    return {y[0]};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    torch::autograd::variable_list out(9);
    const at::Tensor dyq = grads[0], dyk = grads.size() > 1 ? grads[1] : at::Tensor();
    if (!dyq.defined() && !dyk.defined()) return out;
    const auto s = ctx->get_saved_variables();
    const bool norm = ctx->saved_data["norm"].toBool();
    const Turn t{norm, ctx->saved_data["interleaved"].toBool(), ctx->saved_data["eps"].toDouble(), s[4],
                 s[5]};
    const auto dtype = ctx->saved_data["dtype"].toScalarType();
    auto grad = [&](const at::Tensor& g) { return g.defined() ? rows_of(g.to(dtype)) : g; };
    if (!norm) {
      // one call over the gradients that are there
      const at::Tensor a = grad(dyq.defined() ? dyq : dyk);
      const at::Tensor b = dyq.defined() ? grad(dyk) : at::Tensor();
      const auto y = run_rotary(t, a, b, at::Tensor(), at::Tensor(), false, true);
      if (dyq.defined()) {
        out[0] = y[0];
        out[1] = y[1];
      } else {
        out[1] = y[0];
      }
      return once(std::move(out), "rotary_embedding");
    }
    const at::Tensor q = rows_of(s[0]), k = rows_of(s[1]);  // layouts that a saved-tensor hook changed
    const at::Tensor &wq = s[2], &wk = s[3];
    const at::Tensor gq = dyq.defined() ? grad(dyq) : at::zeros_like(q);
    const at::Tensor gk = !k.defined() ? at::Tensor() : dyk.defined() ? grad(dyk) : at::zeros_like(k);
    c10::DeviceGuard guard(q.device());
    at::Tensor dq = at::empty_like(q), dk, dwq, dwk, ws;
    if (k.defined()) dk = at::empty_like(k);
    // needs_input_grad counts edges: an absent tensor before the weights has none
    const size_t eq = 1 + k.defined(), ek = eq + wq.defined();
    if (wq.defined() && ctx->needs_input_grad(eq)) dwq = at::empty_like(wq);
    if (wk.defined() && ctx->needs_input_grad(ek)) dwk = at::empty_like(wk);
    const cra_turn p = make_turn(t, q, k, true, wq.defined() ? wq : wk);
    size_t nws = 0;
    if (dwq.defined() || dwk.defined()) {
      nws = api().rotary_ws(&p);
      ws = at::empty({(int64_t)nws}, q.options().dtype(at::kByte));
    }
    check(api().norm_rotary_bwd(&p, row_arg(q), row_arg(k), ptr_of(wq), ptr_of(wk), row_arg(gq),
                                row_arg(gk), row_arg(dq), row_arg(dk), ptr_of(dwq), ptr_of(dwk),
                                ptr_of(ws), nws, stream_of(q)),
          "cra_norm_rotary_bwd");
    out[0] = dq;
    out[1] = dk;
    out[2] = dwq;
    out[3] = dwk;
    return once(std::move(out), "qk_norm_rotary");
  }
};

// Positions [S], [1, S] or [B, S] of rows q [B, H, S, D].
bool positions_fit(const at::Tensor& pos, const at::Tensor& q) {
  if (pos.device() != q.device() || (pos.scalar_type() != at::kInt && pos.scalar_type() != at::kLong))
    return false;
  const int64_t n = pos.dim();
  return n >= 1 && n <= 2 && pos.size(n - 1) == q.size(2) &&
         (n == 1 || pos.size(0) == 1 || pos.size(0) == q.size(0));
}

bool weights_fit(const at::Tensor& wq, const at::Tensor& wk, const at::Tensor& q) {
  for (const at::Tensor& w : {wq, wk})
    if (w.defined() && (w.dim() != 1 || w.size(0) != q.size(3) || w.device() != q.device() || !w.is_contiguous() ||
                        (w.scalar_type() != q.scalar_type() && w.scalar_type() != at::kFloat)))
      return false;
  return !wq.defined() || !wk.defined() || wq.scalar_type() == wk.scalar_type();
}

bool rotary_takes(const at::Tensor& q, const at::Tensor& k, const at::Tensor& wq, const at::Tensor& wk,
                  const at::Tensor& table, const at::Tensor& pos, bool norm, double eps) {
  if (q.dim() != 4 || !q.is_cuda() || !float_type(q.scalar_type()) || q.numel() == 0) return false;
  const int64_t B = q.size(0), S = q.size(2), D = q.size(3);
  if (D > 256 || !sizes_fit(q)) return false;
  if (k.defined() && (!sizes_fit(k) || k.dim() != 4 || k.size(0) != B || k.size(2) != S || k.size(3) != D ||
                      k.size(1) < 1 || k.scalar_type() != q.scalar_type() || k.device() != q.device()))
    return false;
  if (!table.defined() && (pos.defined() || !norm)) return false;
  if (table.defined() && (table.device() != q.device() || table.dim() != 2 || table.size(1) > D ||
                          table.scalar_type() != at::kFloat || !table.is_contiguous() ||
                          (at::GradMode::is_enabled() && table.requires_grad()) || table._fw_grad(0).defined()))
    return false;
  if (pos.defined()) {
    if (!positions_fit(pos, q)) return false;
  } else if (table.defined() && S > table.size(0)) {
    return false;
  }
  if (!weights_fit(wq, wk, q)) return false;
  if (wk.defined() && !k.defined()) return false;
  return !norm || eps >= 0;
}

std::vector<at::Tensor> rotary_autograd(const at::Tensor& q, const OptTensor& k, const OptTensor& wq,
                                        const OptTensor& wk, const OptTensor& table,
                                        const OptTensor& pos, bool interleaved, bool norm, double eps) {
  const at::Tensor k_ = get(k), wq_ = get(wq), wk_ = get(wk), table_ = get(table), pos_ = get(pos);
  if (!rotary_takes(q, k_, wq_, wk_, table_, pos_, norm, eps)) return {};
  auto wants = [](const at::Tensor& t) {
    return t.defined() && ((at::GradMode::is_enabled() && t.requires_grad()) || t._fw_grad(0).defined());
  };
  if (wants(q) || wants(k_) || wants(wq_) || wants(wk_))  // (a tangent raises in there)
    return CraRotary::apply(q, k, wq, wk, table, pos, interleaved, norm, eps);
  at::AutoDispatchBelowADInplaceOrView below;
  const at::Tensor qr = rows_of(q), kr = rows_of(k_);
  const auto y = run_rotary(Turn{norm, interleaved, eps, table_, pos_}, qr, kr, wq_, wk_, norm, false);
  if (kr.defined()) return {y[0], y[1]};
  return {y[0]};
}

// Rows that the paged calls can address as they are.
bool paged_rows(const at::Tensor& t) {
  const int64_t vec = 16 / t.element_size();
  auto st = [&](int d) { return t.size(d) == 1 || t.stride(d) % vec == 0; };
  return t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && st(0) && st(1) && st(2);
}

// The structures of a call over a cache whose own tensors were checked when it was
// made; false where a tensor of the call is not what the plain path takes.
bool paged_call(const at::Tensor& x, const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& norm,
                const OptTensor& ks, const OptTensor& vs, const at::Tensor& table, const at::Tensor& lens,
                const OptTensor& cu, int64_t head_dim, cra_cache& c, cra_batch& b) {
  if (x.dim() != 4 || x.device() != kc.device() || !float_type(x.scalar_type()) || x.numel() == 0 ||
      x.size(3) != head_dim || head_dim % 8 || !paged_rows(x) || !sizes_fit(x) || !sizes_fit(table) ||
      x._fw_grad(0).defined())
    return false;
  if (table.scalar_type() != at::kInt || lens.scalar_type() != at::kInt || table.dim() != 2 ||
      lens.dim() != 1 || table.device() != kc.device() || lens.device() != kc.device() ||
      !lens.is_contiguous() || lens.size(0) != table.size(0) || table.size(0) < 1 || table.size(1) < 1 ||
      (table.size(1) > 1 && table.stride(1) != 1))
    return false;
  const int64_t N = table.size(0);
  if (cu.has_value()) {
    if (cu->scalar_type() != at::kInt || cu->device() != kc.device() || cu->dim() != 1 ||
        cu->size(0) != N + 1 || !cu->is_contiguous() || x.size(0) != 1)
      return false;
  } else if (x.size(0) != N) {
    return false;
  }
  const auto st = kc.scalar_type();
  const bool same = st == x.scalar_type();
  if (!same && (!ks.has_value() || !vs.has_value())) return false;  // another dtype than the cache's
  c = cra_cache{kc.data_ptr(), vc.data_ptr(), norm.data_ptr<float>(),
                same ? nullptr : ks->data_ptr<float>(), same ? nullptr : vs->data_ptr<float>(),
                (int32_t)kc.size(0), (int32_t)kc.size(1), (int32_t)kc.size(2), (int32_t)kc.size(3),
                dtype_code(x.scalar_type()),
                same ? CRA_STORE_SAME : st == at::kChar ? CRA_STORE_INT8 : CRA_STORE_E4M3};
  b = cra_batch{table.data_ptr<int32_t>(), table.stride(0), lens.data_ptr<int32_t>(),
                cu.has_value() ? cu->data_ptr<int32_t>() : nullptr, (int32_t)N, (int32_t)table.size(1),
                cu.has_value() ? (int32_t)x.size(2) : 0, cu.has_value() ? 0 : (int32_t)x.size(2)};
  return true;
}

bool cache_write(const at::Tensor& k, const at::Tensor& v, const at::Tensor& kc, const at::Tensor& vc,
                 const at::Tensor& norm, const OptTensor& ks, const OptTensor& vs,
                 const at::Tensor& table, const at::Tensor& lens, const OptTensor& cu, int64_t head_dim) {
  cra_cache c;
  cra_batch b;
  if (!paged_call(k, kc, vc, norm, ks, vs, table, lens, cu, head_dim, c, b) || v.sizes() != k.sizes() ||
      v.scalar_type() != k.scalar_type() || v.device() != k.device() || !paged_rows(v) ||
      v._fw_grad(0).defined() || k.size(1) != kc.size(1))
    return false;
  c10::DeviceGuard guard(k.device());
  check(api().cache_write(&c, &b, row_arg(k), row_arg(v), (int32_t)head_dim, stream_of(k)),
        "cra_cache_write");
  return true;
}

// q normed and turned, with k and v stored; nothing where the plain path does not take
// the call.
std::vector<at::Tensor> cache_append(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                     const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& norm,
                                     const OptTensor& ks, const OptTensor& vs, const at::Tensor& table,
                                     const at::Tensor& lens, const OptTensor& cu, int64_t head_dim,
                                     const OptTensor& wq_in, const OptTensor& wk_in,
                                     const OptTensor& angles_in, const OptTensor& pos_in,
                                     bool interleaved, bool normed, double eps) {
  const at::Tensor wq = get(wq_in), wk = get(wk_in), angles = get(angles_in), pos = get(pos_in);
  cra_cache c;
  cra_batch b;
  if (!paged_call(k, kc, vc, norm, ks, vs, table, lens, cu, head_dim, c, b) || v.sizes() != k.sizes() ||
      v.scalar_type() != k.scalar_type() || v.device() != k.device() || !paged_rows(v) ||
      v._fw_grad(0).defined() || k.size(1) != kc.size(1) || q.dim() != 4 || q.numel() == 0 ||
      (!angles.defined() && !normed) || (angles.defined() && angles.size(0) < 1) ||
      (pos.defined() && !angles.defined()))
    return {};
  if (q.size(0) != k.size(0) || q.size(2) != k.size(2) || q.size(3) != head_dim ||
      q.scalar_type() != k.scalar_type() || q.device() != k.device() || !sizes_fit(q) || !paged_rows(q) ||
      q._fw_grad(0).defined())
    return {};
  if (angles.defined() &&
      (angles.device() != q.device() || angles.dim() != 2 || angles.size(1) > head_dim || angles.size(1) % 2 ||
       angles.scalar_type() != at::kFloat || !angles.is_contiguous() || angles._fw_grad(0).defined()))
    return {};
  if (pos.defined() && !positions_fit(pos, q)) return {};
  if (!weights_fit(wq, wk, q) || (normed && !(eps >= 0)) || (!normed && (wq.defined() || wk.defined())))
    return {};
  for (const at::Tensor& w : {wq, wk})
    if (w.defined() && w._fw_grad(0).defined()) return {};
  c10::DeviceGuard guard(q.device());
  at::Tensor y = at::empty_like(q);
  if (!paged_rows(y)) return {};
  const cra_turn p = make_turn(Turn{normed, interleaved, eps, angles, pos}, q, k, normed, wq.defined() ? wq : wk);
  const int code = api().cache_append(&c, &b, &p, row_arg(q), row_arg(k), row_arg(v), ptr_of(wq),
                                      ptr_of(wk), row_arg(y), stream_of(q));
  if (code == CRA_E_UNSUPPORTED) return {};
  check(code, "cra_cache_append");
  return {y};
}

std::vector<at::Tensor> paged_attention(const at::Tensor& q, const at::Tensor& kc, const at::Tensor& vc,
                                        const at::Tensor& norm, const OptTensor& ks, const OptTensor& vs,
                                        const at::Tensor& table, const at::Tensor& lens,
                                        const OptTensor& cu, int64_t head_dim, int64_t max_query_len,
                                        int64_t max_seqlen, int64_t window, int64_t relay,
                                        int64_t top_k, const OptTensor& prefix_table,
                                        const OptTensor& prefix_len) {
  cra_cache c;
  cra_batch b;
  if (prefix_table.has_value() != prefix_len.has_value()) return {};
  if (prefix_table.has_value() &&
      (window < 1 || prefix_table->scalar_type() != at::kInt || prefix_len->scalar_type() != at::kInt ||
       prefix_table->device() != kc.device() || prefix_len->device() != kc.device() || prefix_table->dim() != 1 ||
       !prefix_table->is_contiguous() || !sizes_fit(*prefix_table) || prefix_table->numel() < 1 ||
       prefix_len->dim() != 1 || prefix_len->size(0) != 1 ||
       prefix_table->numel() * kc.size(2) > 0x7fff0000))
    return {};
  if (!paged_call(q, kc, vc, norm, ks, vs, table, lens, cu, head_dim, c, b) || q.size(1) % kc.size(1) ||
      window < 0 || (relay != 0 && (top_k < 1 || top_k > 4)) || max_query_len < 0 || max_seqlen < 0)
    return {};
  c10::DeviceGuard guard(q.device());
  const int64_t held = std::min<int64_t>(table.size(1) * kc.size(2), INT32_MAX), M = q.size(2);
  cra_paged_plan p{(int32_t)q.size(1), (int32_t)head_dim, (int32_t)std::min<int64_t>(window, INT32_MAX),
                   (int32_t)relay, (int32_t)top_k,
                   (int32_t)std::min<int64_t>(M, max_query_len ? max_query_len : M),
                   (int32_t)std::min<int64_t>(held, max_seqlen ? max_seqlen : held), 1,
                   (float)(1.0 / std::sqrt((double)head_dim))};
  at::Tensor o = at::empty_like(q), ws;
  auto space = [&](size_t n) {
    if (n) ws = at::empty({(int64_t)n}, q.options().dtype(at::kByte));
    return n;
  };
  if (prefix_table.has_value()) {
    const cra_prefix x{prefix_table->data_ptr<int32_t>(), prefix_len->data_ptr<int32_t>(),
                       (int32_t)prefix_table->numel()};
    const size_t n = space(api().shared_ws(&c, &b, &p, &x));
    check(api().fwd_shared(&c, &b, &p, &x, row_arg(q), row_arg(o), ptr_of(ws), n, stream_of(q)),
          "cra_fwd_paged_shared");
    return {o};
  }
  const size_t n = space(api().paged_ws(&c, &b, &p));
  check(api().fwd_paged(&c, &b, &p, row_arg(q), row_arg(o), ptr_of(ws), n, stream_of(q)), "cra_fwd_paged");
  return {o};
}

// x [.., K] times the transpose of an 8-bit weight; nothing where the plain path does not
// take the call.
std::vector<at::Tensor> linear_e4m3(const at::Tensor& x, const at::Tensor& codes, const at::Tensor& exps,
                                    const OptTensor& bias_in, int64_t N, int64_t K) {
  const at::Tensor bias = get(bias_in);
  const int64_t d = x.dim();
  if (d < 1 || x.size(d - 1) != K || !float_type(x.scalar_type()) || x.device() != codes.device() ||
      x.numel() == 0 || (K > 1 && x.stride(d - 1) != 1) || x._fw_grad(0).defined())
    return {};
  int64_t M = 1, ld = K;
  if (d == 2) {
    M = x.size(0);
    ld = M > 1 ? x.stride(0) : K;
  } else {
    if (!x.is_contiguous()) return {};
    M = x.numel() / K;
  }
  if (bias.defined() && (bias.dim() != 1 || bias.size(0) != N || bias.scalar_type() != x.scalar_type() ||
                         bias.device() != x.device() || !bias.is_contiguous() || bias._fw_grad(0).defined()))
    return {};
  c10::DeviceGuard guard(x.device());
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = N;
  at::Tensor y = at::empty(shape, x.options()), ws;
  const cra_linear p{M, (int32_t)N, (int32_t)K, dtype_code(x.scalar_type())};
  const size_t n = api().linear_ws(&p);
  if (n) ws = at::empty({(int64_t)n}, x.options().dtype(at::kByte));
  check(api().linear_e4m3(&p, x.data_ptr(), ld, codes.data_ptr(), exps.data_ptr(), ptr_of(bias), y.data_ptr(),
                          N, ptr_of(ws), n, stream_of(x)),
        "cra_linear_e4m3");
  return {y};
}

}  // namespace

TORCH_LIBRARY(cra, m) {
  m.def("bind(str path) -> ()", &bind);
  m.def(
      "attention(Tensor q, Tensor k, Tensor v, int window, bool relay, int top_k, float scale)"
      " -> Tensor");
  // the output and the gradients as [B, H, S, D] views of [B, S, H, D] buffers
  m.def(
      "layer_attention(Tensor q, Tensor k, Tensor v, int window, bool relay, int top_k,"
      " float scale) -> Tensor");
  // rotary positions (and head norms): y of q and of k, or nothing
  m.def(
      "rotary(Tensor q, Tensor? k, Tensor? wq, Tensor? wk, Tensor? table, Tensor? positions,"
      " bool interleaved, bool norm, float eps) -> Tensor[]");
  m.def(
      "cache_write(Tensor k, Tensor v, Tensor(a!) k_pages, Tensor(b!) v_pages, Tensor(c!) k_norm,"
      " Tensor(d!)? k_scale, Tensor(e!)? v_scale, Tensor page_table, Tensor seq_lens,"
      " Tensor? cu_seqlens, int head_dim) -> bool");
  m.def(
      "cache_append(Tensor q, Tensor k, Tensor v, Tensor(a!) k_pages, Tensor(b!) v_pages,"
      " Tensor(c!) k_norm, Tensor(d!)? k_scale, Tensor(e!)? v_scale, Tensor page_table,"
      " Tensor seq_lens, Tensor? cu_seqlens, int head_dim, Tensor? wq, Tensor? wk, Tensor? table,"
      " Tensor? positions, bool interleaved, bool norm, float eps) -> Tensor[]");
  m.def(
      "paged_attention(Tensor q, Tensor k_pages, Tensor v_pages, Tensor k_norm, Tensor? k_scale,"
      " Tensor? v_scale, Tensor page_table, Tensor seq_lens, Tensor? cu_seqlens, int head_dim,"
      " int max_query_len, int max_seqlen, int window, int relay, int top_k, Tensor? prefix_table,"
      " Tensor? prefix_len) -> Tensor[]");
  m.def(
      "linear_e4m3(Tensor x, Tensor codes, Tensor exponents, Tensor? bias, int out_features,"
      " int in_features) -> Tensor[]");
}

TORCH_LIBRARY_IMPL(cra, Autograd, m) {
  m.impl("attention", &attention_autograd<false>);
  m.impl("layer_attention", &attention_autograd<true>);
  m.impl("rotary", &rotary_autograd);
}

TORCH_LIBRARY_IMPL(cra, CUDA, m) {
  m.impl("attention", &attention_forward<false>);
  m.impl("layer_attention", &attention_forward<true>);
  m.impl("rotary", &rotary_autograd);
  m.impl("cache_write", &cache_write);
  m.impl("cache_append", &cache_append);
  m.impl("paged_attention", &paged_attention);
  m.impl("linear_e4m3", &linear_e4m3);
}
