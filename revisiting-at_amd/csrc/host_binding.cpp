// host_binding.cpp — the host side of ops.mha, ops.qk_norm_rope and ops.attention_rope (autograd nodes and launches) and of optim.FusedAdamW
// (its look at the parameters and gradients), as a Python module.
//
// A small attention is a few 10 us kernels; in Python the same node costs the host more than that - twice over in the backward, which the
// autograd engine runs in a thread of its own.  (Forward and backward of 4 x 197 tokens: 133 us in Python, 65 here, 58 of them the engine's.)
// Arguments have been checked by ops.py.  The kernels are reached through the C ABI of the library that ops.py has loaded (bind()).
#include <dlfcn.h>

#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/extension.h>

#include "apgd_hip.h"
#include "convnext_hip.h"

namespace {

using at::Tensor;
using torch::autograd::collect_next_edges;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
using Maybe = std::optional<Tensor>;

struct Library {
  decltype(&apgd_hip_strerror) strerror;
  decltype(&cnx_mha_ws_floats) mha_ws_floats;
  decltype(&cnx_mha_bwd_ws_floats) mha_bwd_ws_floats;
  decltype(&cnx_mha_fwd) mha_fwd;
  decltype(&cnx_mha_bwd) mha_bwd;
  decltype(&cnx_qk_norm_rope_ws_floats) rope_ws_floats;
  decltype(&cnx_qk_norm_rope_fwd) rope_fwd;
  decltype(&cnx_qk_norm_rope_bwd) rope_bwd;
  decltype(&cnx_attention_rope_fwd) layer_fwd;
  decltype(&cnx_attention_rope_bwd_ws_floats) layer_bwd_ws_floats;
  decltype(&cnx_attention_rope_bwd) layer_bwd;
} lib = {};
const volatile int32_t* input_grad_only = nullptr;                     // ops.py's flag: no weight gradients

void bind(uintptr_t handle, uintptr_t flag) {
  void* h = reinterpret_cast<void*>(handle);
  auto find = [&](auto& f, const char* name) {
    f = reinterpret_cast<std::decay_t<decltype(f)>>(dlsym(h, name));
    TORCH_CHECK(f, "the library does not export ", name);
  };
  find(lib.strerror, "apgd_hip_strerror");
  find(lib.mha_ws_floats, "cnx_mha_ws_floats");
  find(lib.mha_bwd_ws_floats, "cnx_mha_bwd_ws_floats");
  find(lib.mha_fwd, "cnx_mha_fwd");
  find(lib.mha_bwd, "cnx_mha_bwd");
  find(lib.rope_ws_floats, "cnx_qk_norm_rope_ws_floats");
  find(lib.rope_fwd, "cnx_qk_norm_rope_fwd");
  find(lib.rope_bwd, "cnx_qk_norm_rope_bwd");
  find(lib.layer_fwd, "cnx_attention_rope_fwd");
  find(lib.layer_bwd_ws_floats, "cnx_attention_rope_bwd_ws_floats");
  find(lib.layer_bwd, "cnx_attention_rope_bwd");
  input_grad_only = reinterpret_cast<const volatile int32_t*>(flag);
}
void check(int code, const char* what) { TORCH_CHECK(code == APGD_OK, what, " failed: ", code, " (", lib.strerror(code), ")"); }

int code_of(const Tensor& t) { return t.scalar_type() == at::kFloat ? APGD_F32 : t.scalar_type() == at::kBFloat16 ? APGD_BF16 : APGD_F16; }
void* current() { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream(); }
template <typename T> T* ptr(const Tensor& t) { return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr; }
Tensor fresh(const Tensor& like) { return at::empty(like.sizes(), like.options()); }
Tensor floats(int64_t n, const Tensor& like) { return n ? at::empty({n}, like.options().dtype(at::kFloat)) : Tensor(); }
Tensor of(const Maybe& t) { return t ? *t : Tensor(); }

// t [B, N, H, d] itself where the kernels can read it in place (contiguous heads that begin at 16 bytes, any other strides up to 2^22 elements
// between tokens and 2^28 over the heads that share a key head, zero included), else a contiguous copy
Tensor head_rows(const Tensor& t, int64_t share = 1) {
  const int64_t piece = 16 / t.element_size();
  const auto s = t.strides();
  if (s[3] == 1 && s[0] % piece == 0 && s[1] % piece == 0 && s[2] % piece == 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 &&
      s[1] < 1 << 22 && s[2] * share < 1 << 28)
    return t;
  return fresh(t).copy_(t);
}
// (sample, token, head) strides of the tensors in turn
template <typename... Ts>
std::array<int64_t, 3 * sizeof...(Ts)> strides(const Ts&... ts) {
  std::array<int64_t, 3 * sizeof...(Ts)> r;
  int64_t* p = r.data();
  ((p[0] = ts.stride(0), p[1] = ts.stride(1), p[2] = ts.stride(2), p += 3), ...);
  return r;
}

struct Rotation {
  Tensor positions, inv_freq;
  std::vector<int32_t> sections;
  int pos_dtype;
  int64_t batch_stride;
  float eps;
  int32_t norm, interleaved;
  bool turns() const { return norm || positions.defined(); }
};
// what a node saves of a rotation's tensors, so that a change in place raises as any other input's does (one made in inference mode has no version
// to tell a change by, and is copied)
Tensor kept(const Tensor& t) { return t.defined() && t.is_inference() ? t.clone() : t; }
// weights of one type: where one is float32 and the other is not, both are
std::pair<Tensor, Tensor> head_weights(Tensor wq, Tensor wk) {
  if (wq.defined() && wk.defined() && wq.scalar_type() != wk.scalar_type()) {
    wq = wq.to(at::kFloat);
    wk = wk.to(at::kFloat);
  }
  return {wq.defined() ? wq.contiguous() : wq, wk.defined() ? wk.contiguous() : wk};
}
int weight_code(const Tensor& wq, const Tensor& wk) { return wq.defined() ? code_of(wq) : wk.defined() ? code_of(wk) : APGD_F32; }

void rope_forward(const Tensor& q, const Tensor& k, const Tensor& yq, const Tensor& yk, const Tensor& wq, const Tensor& wk, const Rotation& r) {
  check(lib.rope_fwd(q.data_ptr(), k.data_ptr(), yq.data_ptr(), yk.data_ptr(), code_of(q), strides(q, k, yq, yk).data(), ptr<void>(wq), ptr<void>(wk),
                     weight_code(wq, wk), ptr<void>(r.positions), r.pos_dtype, r.batch_stride, static_cast<int32_t>(r.sections.size()), r.sections.data(),
                     ptr<float>(r.inv_freq), q.size(0), q.size(1), q.size(2), k.size(2), q.size(3), r.eps, r.norm, r.interleaved, current()),
        "cnx_qk_norm_rope_fwd");
}
// gradients into dq, dk and, where wanted, those of the weights (fp32)
void rope_backward(const Tensor& dyq, const Tensor& dyk, const Tensor& q, const Tensor& k, const Tensor& dq, const Tensor& dk, const Tensor& wq,
                   const Tensor& wk, const Rotation& r, bool want_q, bool want_k, Tensor& dwq, Tensor& dwk) {
  const int32_t d = dyq.size(3);
  if (want_q) dwq = floats(d, dyq);
  if (want_k) dwk = floats(d, dyq);
  const Tensor ws = want_q || want_k ? floats(lib.rope_ws_floats(d), dyq) : Tensor();
  const Tensor &xq = r.norm ? q : dyq, &xk = r.norm ? k : dyk;          // without norm q and k are not read
  check(lib.rope_bwd(dyq.data_ptr(), dyk.data_ptr(), xq.data_ptr(), xk.data_ptr(), dq.data_ptr(), dk.data_ptr(), ptr<float>(dwq), ptr<float>(dwk),
                     ptr<float>(ws), code_of(dyq), strides(dyq, dyk, xq, xk, dq, dk).data(), ptr<void>(wq), ptr<void>(wk), weight_code(wq, wk),
                     ptr<void>(r.positions), r.pos_dtype, r.batch_stride, static_cast<int32_t>(r.sections.size()), r.sections.data(), ptr<float>(r.inv_freq),
                     dyq.size(0), dyq.size(1), dyq.size(2), dyk.size(2), d, r.eps, r.norm, r.interleaved, current()),
        "cnx_qk_norm_rope_bwd");
}
Tensor mha_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& out, double scale, bool causal, const Tensor& q_lens,
                   const Tensor& kv_lens, bool want_lse) {
  const int64_t B = q.size(0);
  const int32_t Nq = q.size(1), H = q.size(2), d = q.size(3), Nk = k.size(1), Hkv = k.size(2);
  const Tensor lse = want_lse ? at::empty({B, H, Nq}, q.options().dtype(at::kFloat)) : Tensor();
  const Tensor ws = floats(lib.mha_ws_floats(B, Nq, Nk, H, Hkv, d), q);
  check(lib.mha_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), ptr<float>(lse), ptr<int32_t>(q_lens), ptr<int32_t>(kv_lens), ptr<float>(ws),
                    strides(q, k, v, out).data(), code_of(q), B, Nq, Nk, H, Hkv, d, causal, static_cast<float>(scale), current()),
        "cnx_mha_fwd");
  return lse;
}
void mha_backward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& out, const Tensor& dout, const Tensor& lse, const Tensor& dq,
                  const Tensor& dk, const Tensor& dv, double scale, bool causal, const Tensor& q_lens, const Tensor& kv_lens) {
  const int64_t B = q.size(0);
  const int32_t Nq = q.size(1), H = q.size(2), d = q.size(3), Nk = k.size(1), Hkv = k.size(2);
  const Tensor dvec = at::empty({B, H, Nq}, lse.options()), ws = floats(lib.mha_bwd_ws_floats(B, Nq, Nk, H, Hkv, d, causal), q);
  check(lib.mha_bwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), dout.data_ptr(), ptr<float>(lse), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                    ptr<float>(dvec), ptr<int32_t>(q_lens), ptr<int32_t>(kv_lens), ptr<float>(ws), strides(q, k, v, out, dout, dq, dk, dv).data(), code_of(q),
                    B, Nq, Nk, H, Hkv, d, causal, static_cast<float>(scale), current()),
        "cnx_mha_bwd");
}

// ------------------------------------------------------------------------------------------------------------------ autograd
struct Node : torch::autograd::Node {
  std::vector<SavedVariable> saved;
  void save(std::initializer_list<Tensor> ts) {
    for (const Tensor& t : ts) saved.emplace_back(t, false);
  }
  Tensor at(size_t i) { return saved[i].unpack(); }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (auto& s : saved) s.reset_data();
    released = true;
  }
  bool wants(size_t i) const { return task_should_compute_output(i); }
  // Gradients have no derivative of their own: where a graph of them is recorded, going back through them - to the incoming gradients or to
  // this node's inputs - raises.
  variable_list once(variable_list&& grads, const variable_list& in) {
    if (!at::GradMode::is_enabled()) return std::move(grads);
    torch::autograd::edge_list edges = collect_next_edges(in);
    for (const auto& e : next_edges()) edges.push_back(e);
    const std::shared_ptr<torch::autograd::Node> error(new torch::autograd::Error(name() + " is differentiable once", std::move(edges)),
                                                       torch::autograd::deleteNode);
    for (const Tensor& g : grads)
      if (g.defined()) torch::autograd::set_history(g, error);
    return std::move(grads);
  }
  variable_list apply(variable_list&& in) final {
    std::lock_guard<std::mutex> lock(mutex_);
    TORCH_CHECK(!released, torch::autograd::ERR_BACKWARD_TWICE);
    variable_list grads;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      grads = gradients(in);
    }
    return once(std::move(grads), in);
  }
  virtual variable_list gradients(const variable_list& in) = 0;
  bool released = false;
};
template <typename N, typename... Ts>
std::shared_ptr<N> node_of(const Ts&... inputs) {
  std::shared_ptr<N> n(new N(), torch::autograd::deleteNode);
  n->set_next_edges(collect_next_edges(inputs...));
  return n;
}
template <typename... Ts>
bool wants_grad(const Ts&... ts) { return at::GradMode::is_enabled() && ((ts.defined() && ts.requires_grad()) || ...); }
// Dual tensors are refused: their tangents would be lost without a word, which reads as a derivative of zero.
template <typename... Ts>
void no_tangents(const char* what, const Ts&... ts) {
  TORCH_CHECK_NOT_IMPLEMENTED(!((ts.defined() && ts._fw_grad(0).defined()) || ...), what, " has no forward-mode derivative");
}

struct MhaBackward : Node {
  double scale;
  bool causal;
  std::string name() const override { return "mha"; }
  variable_list gradients(const variable_list& in) override {
    if (!in[0].defined()) return {Tensor(), Tensor(), Tensor()};
    const Tensor q = at(0), k = at(1), v = at(2), lse = at(3);
    const c10::DeviceGuard guard(q.device());
    const Tensor dout = head_rows(in[0], q.size(2) / k.size(2)), dq = fresh(q), dk = fresh(k), dv = fresh(v);
    mha_backward(q, k, v, saved[4].unpack(shared_from_this()), dout, lse, dq, dk, dv, scale, causal, at(5), at(6));
    return {dq, dk, dv};
  }
};

Tensor mha(const Tensor& q0, const Tensor& k0, const Tensor& v0, double scale, bool causal, const Maybe& q_lens, const Maybe& kv_lens) {
  no_tangents("mha", q0, k0, v0);
  const c10::DeviceGuard guard(q0.device());
  const bool grad = wants_grad(q0, k0, v0);
  Tensor q, k, v, out, lse;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    q = head_rows(q0, q0.size(2) / k0.size(2)); k = head_rows(k0); v = head_rows(v0);
    out = fresh(q);
    lse = mha_forward(q, k, v, out, scale, causal, of(q_lens), of(kv_lens), grad);
  }
  if (grad) {
    auto n = node_of<MhaBackward>(q0, k0, v0);
    n->scale = scale; n->causal = causal;
    torch::autograd::set_history(out, n);
    n->save({q, k, v, lse});
    n->saved.emplace_back(out, true);
    n->save({of(q_lens), of(kv_lens)});
  }
  return out;
}

struct QkNormRopeBackward : Node {
  Rotation rot;
  at::ScalarType wq_type, wk_type;
  std::vector<int64_t> q_size, k_size;
  at::TensorOptions options;
  std::string name() const override { return "qk_norm_rope"; }
  variable_list gradients(const variable_list& in) override {
    if (!in[0].defined() && !in[1].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const c10::DeviceGuard guard(options.device());
    const Tensor q = at(0), k = at(1), wq = at(2), wk = at(3);
    Rotation turn = rot;
    turn.positions = at(4); turn.inv_freq = at(5);
    const Tensor dyq = head_rows(in[0].defined() ? in[0] : at::zeros(q_size, options)), dyk = head_rows(in[1].defined() ? in[1] : at::zeros(k_size, options));
    const Tensor dq = fresh(dyq), dk = fresh(dyk);
    Tensor dwq, dwk;
    rope_backward(dyq, dyk, q, k, dq, dk, wq, wk, turn, wants(2) && !*input_grad_only, wants(3) && !*input_grad_only, dwq, dwk);
    return {dq, dk, dwq.defined() ? dwq.to(wq_type) : dwq, dwk.defined() ? dwk.to(wk_type) : dwk};
  }
};

Rotation rotation(const Maybe& positions, const Maybe& inv_freq, std::vector<int32_t> sections, int pos_dtype, int64_t batch_stride, double eps,
                  bool norm, bool interleaved) {
  return Rotation{of(positions), of(inv_freq), std::move(sections), pos_dtype, batch_stride, static_cast<float>(eps), norm, interleaved};
}

std::tuple<Tensor, Tensor> qk_norm_rope(const Tensor& q0, const Tensor& k0, const Maybe& wq0, const Maybe& wk0, const Maybe& positions,
                                        const Maybe& inv_freq, std::vector<int32_t> sections, int pos_dtype, int64_t batch_stride, double eps,
                                        bool norm, bool interleaved) {
  const c10::DeviceGuard guard(q0.device());
  Rotation rot = rotation(positions, inv_freq, std::move(sections), pos_dtype, batch_stride, eps, norm, interleaved);
  const Tensor w0 = of(wq0), w1 = of(wk0);
  no_tangents("qk_norm_rope", q0, k0, w0, w1, rot.positions, rot.inv_freq);
  const bool grad = wants_grad(q0, k0, w0, w1);
  Tensor q, k, wq, wk, yq, yk;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    q = head_rows(q0); k = head_rows(k0);
    std::tie(wq, wk) = head_weights(w0, w1);
    yq = fresh(q); yk = fresh(k);
    rope_forward(q, k, yq, yk, wq, wk, rot);
  }
  if (grad) {
    auto n = node_of<QkNormRopeBackward>(q0, k0, w0, w1);
    if (w0.defined()) n->wq_type = w0.scalar_type();
    if (w1.defined()) n->wk_type = w1.scalar_type();
    n->q_size = q.sizes().vec(); n->k_size = k.sizes().vec(); n->options = q.options();
    torch::autograd::set_history({yq, yk}, n);
    n->save({norm ? q : Tensor(), norm ? k : Tensor(), wq, wk, kept(rot.positions), kept(rot.inv_freq)});
    rot.positions = rot.inv_freq = Tensor();
    n->rot = std::move(rot);
  }
  return {yq, yk};
}

std::array<Tensor, 3> parts(const Tensor& packed, int64_t heads) {     // q, k, v slices [B, N, H, d] of [B, N, 3 H d]
  const int64_t B = packed.size(0), N = packed.size(1), C = packed.size(2) / 3, d = C / heads;
  std::array<Tensor, 3> r;
  for (int i = 0; i < 3; ++i) r[i] = packed.as_strided({B, N, heads, d}, {N * 3 * C, 3 * C, d, 1}, packed.storage_offset() + i * C);
  return r;
}

// qk_norm_rope and mha on a packed projection: q, k, v and their gradients stay slices of it, no copies between the two
struct AttentionRopeBackward : Node {
  Rotation rot;
  at::ScalarType wq_type, wk_type;
  int64_t heads;
  double scale;
  std::string name() const override { return "attention_rope"; }
  variable_list gradients(const variable_list& in) override {
    if (!in[0].defined()) return {Tensor(), Tensor(), Tensor()};
    const Tensor qkv = at(0), yq = at(1), yk = at(2), wq = at(3), wk = at(4), lse = at(5);
    Rotation turn = rot;
    turn.positions = at(6); turn.inv_freq = at(7);
    const c10::DeviceGuard guard(qkv.device());
    const int64_t B = qkv.size(0), N = qkv.size(1), C = qkv.size(2) / 3, d = C / heads;
    const Tensor out = saved[8].unpack(shared_from_this()).view({B, N, heads, d}), dout = head_rows(in[0].reshape({B, N, heads, d})), dqkv = fresh(qkv);
    const bool want_q = wants(1) && !*input_grad_only, want_k = wants(2) && !*input_grad_only;
    Tensor dwq, dwk;
    if (turn.turns()) {
      const Tensor ws = floats(lib.layer_bwd_ws_floats(B, N, heads, d, turn.batch_stride != 0), qkv);
      const Tensor fq = wq.defined() ? wq.to(at::kFloat) : wq, fk = wk.defined() ? wk.to(at::kFloat) : wk;
      if (want_q) dwq = floats(d, qkv);
      if (want_k) dwk = floats(d, qkv);
      check(lib.layer_bwd(qkv.data_ptr(), yq.data_ptr(), yk.data_ptr(), out.data_ptr(), dout.data_ptr(), ptr<float>(lse), dqkv.data_ptr(), ptr<float>(dwq),
                          ptr<float>(dwk), ptr<float>(ws), strides(dout).data(), code_of(qkv), ptr<float>(fq), ptr<float>(fk), ptr<void>(turn.positions),
                          turn.pos_dtype, turn.batch_stride, static_cast<int32_t>(turn.sections.size()), turn.sections.data(), ptr<float>(turn.inv_freq), B, N,
                          heads, d, turn.eps, turn.norm, turn.interleaved, static_cast<float>(scale), current()),
            "cnx_attention_rope_bwd");
    } else {
      const auto x = parts(qkv, heads), g = parts(dqkv, heads);
      mha_backward(x[0], x[1], x[2], out, dout, lse, g[0], g[1], g[2], scale, false, Tensor(), Tensor());
    }
    return {dqkv, dwq.defined() ? dwq.to(wq_type) : dwq, dwk.defined() ? dwk.to(wk_type) : dwk};
  }
};

Tensor attention_rope(const Tensor& qkv0, int64_t heads, double scale, const Maybe& wq0, const Maybe& wk0, const Maybe& positions, const Maybe& inv_freq,
                      std::vector<int32_t> sections, int pos_dtype, int64_t batch_stride, double eps, bool norm, bool interleaved) {
  const c10::DeviceGuard guard(qkv0.device());
  Rotation rot = rotation(positions, inv_freq, std::move(sections), pos_dtype, batch_stride, eps, norm, interleaved);
  const Tensor w0 = of(wq0), w1 = of(wk0);
  no_tangents("attention_rope", qkv0, w0, w1, rot.positions, rot.inv_freq);
  const bool grad = wants_grad(qkv0, w0, w1);
  Tensor qkv, wq, wk, yq, yk, out, lse;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    qkv = qkv0.contiguous();
    if (reinterpret_cast<uintptr_t>(qkv.data_ptr()) % 16) qkv = qkv.clone();
    std::tie(wq, wk) = head_weights(w0, w1);
    const int64_t B = qkv.size(0), N = qkv.size(1), C = qkv.size(2) / 3, d = C / heads;
    out = at::empty({B, N, C}, qkv.options());
    if (rot.turns()) {                           // (16 bits, of either type)
      yq = fresh(out);
      yk = fresh(out);
    }
    if (grad) lse = at::empty({B, heads, N}, qkv.options().dtype(at::kFloat));
    const Tensor ws = floats(lib.mha_ws_floats(B, N, N, heads, heads, d), qkv);
    check(lib.layer_fwd(qkv.data_ptr(), ptr<void>(yq), ptr<void>(yk), out.data_ptr(), ptr<float>(lse), ptr<float>(ws), code_of(qkv), ptr<void>(wq),
                        ptr<void>(wk), weight_code(wq, wk), ptr<void>(rot.positions), rot.pos_dtype, rot.batch_stride,
                        static_cast<int32_t>(rot.sections.size()), rot.sections.data(), ptr<float>(rot.inv_freq), B, N, heads, d, rot.eps, rot.norm,
                        rot.interleaved, static_cast<float>(scale), current()),
          "cnx_attention_rope_fwd");
  }
  if (grad) {
    auto n = node_of<AttentionRopeBackward>(qkv0, w0, w1);
    if (w0.defined()) n->wq_type = w0.scalar_type();
    if (w1.defined()) n->wk_type = w1.scalar_type();
    n->heads = heads; n->scale = scale;
    torch::autograd::set_history(out, n);
    n->save({qkv, yq, yk, wq, wk, lse, kept(rot.positions), kept(rot.inv_freq)});
    n->saved.emplace_back(out, true);
    rot.positions = rot.inv_freq = Tensor();
    n->rot = std::move(rot);
  }
  return out;
}

// ------------------------------------------------------------------------------------------------------------------ optimizer
// Parameters as the optimizer's tables describe them.  (The address alone does not tell: memory that was given back comes again for other
// sizes and types.)
class Layout {
 public:
  explicit Layout(const std::vector<Tensor>& params) {
    for (const Tensor& p : params) all_.push_back({p.data_ptr(), p.scalar_type(), p.sizes().vec(), p.strides().vec()});
  }
  bool matches(const std::vector<Tensor>& params) const {
    if (params.size() != all_.size()) return false;
    for (size_t i = 0; i < all_.size(); ++i) {
      const Tensor& p = params[i];
      const One& o = all_[i];
      if (p.data_ptr() != o.at || p.scalar_type() != o.type || p.sizes() != at::IntArrayRef(o.sizes) || p.strides() != at::IntArrayRef(o.strides)) return false;
    }
    return true;
  }
  // Addresses of the gradients (0: none) into `to`; those of another type or order of elements are copied, and the copies returned.
  std::vector<Tensor> gradients(const std::vector<Tensor>& params, uintptr_t to) const {
    const at::NoGradGuard no_grad;
    std::vector<Tensor> kept;
    void** out = reinterpret_cast<void**>(to);
    for (size_t i = 0; i < all_.size(); ++i) {
      Tensor g = params[i].grad();
      if (!g.defined()) { out[i] = nullptr; continue; }
      TORCH_CHECK(g.layout() == at::kStrided, "FusedAdamW does not take sparse gradients");
      if (g.scalar_type() != all_[i].type || g.strides() != at::IntArrayRef(all_[i].strides)) {
        g = at::empty_like(params[i]).copy_(g);
        kept.push_back(g);
      }
      out[i] = g.data_ptr();
    }
    return kept;
  }

 private:
  struct One {
    void* at;
    at::ScalarType type;
    std::vector<int64_t> sizes, strides;
  };
  std::vector<One> all_;
};

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("bind", &bind);
  m.def("mha", &mha);
  m.def("qk_norm_rope", &qk_norm_rope);
  m.def("attention_rope", &attention_rope);
  py::class_<Layout>(m, "Layout")
      .def(py::init<const std::vector<Tensor>&>())
      .def("matches", &Layout::matches)
      .def("gradients", &Layout::gradients);
}
