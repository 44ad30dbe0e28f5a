// Host side of the operators as a CPython extension: argument checks, output and workspace allocation, launches through
// the C ABI of libfla_hip.so, and the autograd nodes, without a Python frame between a model's call and its launches.
//
// A decode step or a short training step is a handful of launches of a few microseconds each; with ctypes and Python
// autograd functions the host needed 20 us for the former and 170 us for the latter, several times the device.
//
// Every entry takes the operands as a model holds them and returns None where a call needs a conversion first (head-first
// layout, head dims to be padded, fp32 q/k/v, a gradient through a step that has none here): the Python wrappers then take
// their general route.  Sequence-first layout, as in include/fla_hip.h.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/python_variable.h>

#include <map>
#include <mutex>
#include <optional>
#include <unordered_set>
#include <vector>

#include "../../include/fla_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int64_t BT = 64;

// ---------------------------------------------------------------------------------------------------- helpers
void check(int code, const char* what) {
  TORCH_CHECK(code == 0, what, " failed with code ", code, ": ", fla_error_string(code));
}

bool is16(const Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf; }
int dt(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return FLA_F32;
    case at::kBFloat16: return FLA_BF16;
    case at::kHalf: return FLA_F16;
    default: TORCH_CHECK_TYPE(false, "fla_amd: unsupported dtype ", t.scalar_type());
  }
}
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* fptr(const Tensor& t) { return (float*)ptr(t); }
fla_stream_t stream_of(const Tensor& t) { return (fla_stream_t)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
Tensor fresh(at::IntArrayRef sizes, const Tensor& like, at::ScalarType type) { return at::empty(sizes, like.options().dtype(type)); }
Tensor fresh_like(const Tensor& x) { return at::empty(x.sizes(), x.options()); }
Tensor f32(const Tensor& x) {
  if (!x.defined()) return x;
  return (x.scalar_type() == at::kFloat ? x : x.to(at::kFloat)).contiguous();
}
// Whether a call has to go through its autograd node.  An operand with a tangent does too, also where nothing requires a
// gradient: the nodes have no forward-mode derivative and say so, a launch beside them would drop the tangent.
bool has_tangent(std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    if (t->defined() && t->_fw_grad(0).defined()) return true;
  return false;
}
bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (has_tangent(ts)) return true;
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
// A leaf's accumulation node stays on the stream that was current when it was made, for as long as a graph holds it.  One of the default stream, which
// cannot be captured, makes a captured backward pass end the process: the call is refused while it is only a call.  Leaves are looked for through the
// whole graph behind the operands (a cast of autocast, the layers ahead), in a call under capture alone.
void refuse_eager_leaves(std::initializer_list<const Tensor*> ts, const char* who) {
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  std::vector<std::shared_ptr<torch::autograd::Node>> open;
  std::unordered_set<const torch::autograd::Node*> seen;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) open.push_back(t->is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(*t) : t->grad_fn());
  while (!open.empty()) {
    const auto node = std::move(open.back());
    open.pop_back();
    if (!node || !seen.insert(node.get()).second) continue;
    if (dynamic_cast<const torch::autograd::AccumulateGrad*>(node.get())) {
      const auto stream = node->stream();
      TORCH_CHECK(!stream || stream->id() != 0, "fla_amd ", who, ": an eager graph of the default stream still holds these leaves, or some behind them, and a "
                  "backward pass of theirs cannot be captured: drop its results ahead of the capture, or call this under torch.no_grad()");
    }
    for (const auto& edge : node->next_edges()) open.push_back(edge.function);
  }
}
bool on_gpu(std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    if (t->defined() && !t->is_cuda()) return false;
  return true;
}
// grads in the dtype of the operand they belong to
Tensor as(const Tensor& g, at::ScalarType type) { return g.scalar_type() == type ? g : g.to(type); }

// Whether an operand of a node has a gradient: those of frozen weights are not formed
bool asks(const Tensor& t) { return t.defined() && t.requires_grad(); }

// An operand that may be absent, as a node takes it
using Maybe = std::optional<Tensor>;
Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : std::nullopt; }
Tensor given(const Maybe& t) { return t ? *t : Tensor(); }

// Anything a node keeps beside tensors
template <typename X>
struct Held : torch::CustomClassHolder {
  X x;
  explicit Held(X v) : x(std::move(v)) {}
};
template <typename X>
void hold(AutogradContext* ctx, X v) {
  ctx->saved_data["s"] = c10::IValue::make_capsule(c10::make_intrusive<Held<X>>(std::move(v)));
}
template <typename X>
const X& held(AutogradContext* ctx) {
  return static_cast<Held<X>*>(ctx->saved_data["s"].toCapsule().get())->x;
}

// ---------------------------------------------------------------------------------------------------- packed batches
// A pinned host tensor as a device tensor that any stream may read from now on.  The copy goes through a stream of its own
// and is waited for there: the streams that compute go on (a blocking copy would wait for everything queued on its stream:
// a whole forward, where it is a backward's tables).  The memory belongs to that stream: readers call record_stream.
Tensor upload(const Tensor& host, at::Device device) {
  static std::mutex mu;
  static std::map<int, hipStream_t> streams;   // one per device, never destroyed
  c10::DeviceGuard on_device(device);
  std::lock_guard<std::mutex> lock(mu);
  hipStream_t& raw = streams[device.index()];
  if (!raw) TORCH_CHECK(hipStreamCreateWithFlags(&raw, hipStreamNonBlocking) == hipSuccess, "fla_amd: no stream for uploads");
  const auto own = c10::hip::getStreamFromExternal(raw, device.index());
  struct Current {
    c10::hip::HIPStream before;
    ~Current() { c10::hip::setCurrentHIPStream(before); }
  } current{c10::hip::getCurrentHIPStream(device.index())};
  c10::hip::setCurrentHIPStream(own);
  Tensor out = at::empty(host.sizes(), host.options().device(device).pinned_memory(false));
  out.copy_(host, /*non_blocking=*/true);
  own.synchronize();
  return out;
}

struct SplitTables {
  bool cut = false;
  fla_split ints{};
  Tensor tables;   // seg_table, sub_table and sub_base, one behind the other
};
// The device tables of a packed batch, made once per offsets tensor by fla_amd.utils.VarlenPlan, `offsets` a copy among them.  (A node
// saves the caller's own tensor beside them, so that a backward after it has been written to is refused.)
struct Plan : torch::CustomClassHolder {
  Tensor offsets, indices, chunk_offsets, seq_order;
  std::vector<int64_t> host;
  int64_t N = 0, NT = 0;
  std::mutex mu;
  std::map<std::tuple<int64_t, int, bool, int>, SplitTables> splits;

  bool covers(int64_t begin, int64_t end) const { return !host.empty() && host.front() == begin && host.back() == end; }

  // The boundaries and tables share one allocation; it belongs to the stream that uploaded it.  (Tensors of this build call
  // their device CUDA.)
  void used() const {
    const auto stream = c10::hip::getCurrentHIPStream(offsets.device().index());
    offsets.record_stream(c10::Stream(c10::Stream::UNSAFE, offsets.device(), stream.id()));
  }

  // The tables of a cut are used by later calls on any stream.  A stream that is being captured takes no copy: a call whose
  // tables are not there yet runs uncut under it.
  SplitTables split(int64_t H, int slabs, bool reverse, int kind) {
    std::lock_guard<std::mutex> lock(mu);
    const auto stream = c10::hip::getCurrentHIPStream(offsets.device().index());
    if (!splits.count({H, slabs, reverse, kind}) &&
        c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None)
      return {};
    auto [it, fresh] = splits.try_emplace({H, slabs, reverse, kind});
    SplitTables& s = it->second;
    if (fresh && N > 0) {
      fla_split sp{};
      auto plan = [&](int32_t* a, int32_t* b, int32_t* c) {
        return fla_scan_split(host.data(), N, 0, H, slabs, reverse, kind, &sp, a, b, c);
      };
      if (plan(nullptr, nullptr, nullptr)) {
        const int64_t sub = 2 * (int64_t)sp.nseg, base = sub + 2 * (int64_t)sp.nsub;
        const Tensor host_tables = at::empty({base + N + 1}, at::TensorOptions().dtype(at::kInt).pinned_memory(true));
        int32_t* h = host_tables.data_ptr<int32_t>();
        plan(h, h + sub, h + base);
        s.tables = upload(host_tables, offsets.device());
        const int32_t* d = s.tables.data_ptr<int32_t>();
        sp.seg_table = d;
        sp.sub_table = d + sub;
        sp.sub_base = d + base;
        s.ints = sp;
        s.cut = true;
      }
    }
    // the plan may be dropped while this stream still reads its tables (tensors of this build call their device CUDA)
    if (s.cut) s.tables.record_stream(c10::Stream(c10::Stream::UNSAFE, offsets.device(), stream.id()));
    return s;
  }
};
using PlanPtr = c10::intrusive_ptr<Plan>;

// Every launch that reads a plan takes its boundaries from here: the plan may be dropped while this stream still reads it.
const int64_t* offs(const PlanPtr& p) {
  if (!p) return nullptr;
  p->used();
  return (const int64_t*)p->offsets.data_ptr();
}
const int64_t* idx(const PlanPtr& p) { return p ? (const int64_t*)p->indices.data_ptr() : nullptr; }
const int64_t* coff(const PlanPtr& p) { return p ? (const int64_t*)p->chunk_offsets.data_ptr() : nullptr; }
const int64_t* order(const PlanPtr& p) { return p ? (const int64_t*)p->seq_order.data_ptr() : nullptr; }

// One call's cut: the integers (and tables) of fla_scan_split and the two workspaces.
struct Cut {
  SplitTables tables;   // keeps a packed batch's tables alive
  fla_split s{};
  Tensor states, transitions;
};
std::optional<Cut> cut_scan(const PlanPtr& plan, int64_t N, int64_t T, int64_t H, int slabs, bool reverse, const Tensor& like,
                            int64_t state_elems, int64_t transition_elems, int kind = FLA_SCAN_GLA) {
  Cut c;
  if (plan) {
    c.tables = plan->split(H, slabs, reverse, kind);
    if (!c.tables.cut) return std::nullopt;
    c.s = c.tables.ints;
  } else if (!fla_scan_split(nullptr, N, T, H, slabs, reverse, kind, &c.s, nullptr, nullptr, nullptr)) {
    return std::nullopt;
  }
  c.states = fresh({c.s.slots * H * state_elems}, like, at::kFloat);
  c.transitions = fresh({c.s.slots * H * transition_elems}, like, at::kFloat);
  c.s.states = fptr(c.states);
  c.s.decays = fptr(c.transitions);
  return c;
}

struct Dims {
  int64_t B, T, H, K, V, N, NT, chunks;
};
// q, k [B,T,H,K], v [B,T,H,V] of one 16-bit dtype on one GPU, head dims 64 or 128
bool chunk_operands(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& h0, const PlanPtr& plan, Dims* d) {
  if (!q.defined() || !k.defined() || !v.defined()) return false;
  if (q.dim() != 4 || v.dim() != 4 || q.sizes() != k.sizes() || q.numel() == 0) return false;
  if (!is16(q) || k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type()) return false;
  if (!on_gpu({&q, &k, &v, &h0})) return false;
  d->B = q.size(0), d->T = q.size(1), d->H = q.size(2), d->K = q.size(3), d->V = v.size(3);
  if (v.size(0) != d->B || v.size(1) != d->T || v.size(2) != d->H) return false;
  if ((d->K != 64 && d->K != 128) || (d->V != 64 && d->V != 128)) return false;
  if (plan && d->B != 1) return false;
  TORCH_CHECK_VALUE(!plan || plan->offsets.device() == q.device(), "fla_amd: offsets on ", plan->offsets.device(), ", the operands on ", q.device());
  d->N = plan ? plan->N : d->B;
  const int64_t per = (d->T + BT - 1) / BT;
  d->NT = plan ? plan->NT : 0;
  d->chunks = plan ? plan->NT : d->B * per;
  if (h0.defined() && (h0.scalar_type() != at::kFloat || h0.dim() != 4 || h0.size(0) != d->N || h0.size(1) != d->H ||
                       h0.size(2) != d->K || h0.size(3) != d->V))
    return false;
  return true;
}

// ---------------------------------------------------------------------------------------------------- GLA
struct GlaArgs {
  Dims d;
  PlanPtr plan;
  double scale;
  bool want_ht, head_gates;
  int gate_form = 0;
  double normalizer = 1.0;
  std::optional<double> clamp;
};
struct GlaKept {
  Tensor wide, hT, qg, decay;
};

Tensor gla_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& h0, const GlaArgs& a,
                   Tensor* ht, GlaKept* kept) {
  const Dims& d = a.d;
  Tensor o = fresh_like(v);
  if (a.want_ht) *ht = fresh({d.N, d.H, d.K, d.V}, q, at::kFloat);
  // the range guard's flags and the states it hands over for flagged chunks
  Tensor wide = fresh({d.chunks, d.H}, q, at::kInt), hwide = fresh({d.chunks, d.H, d.K * d.V}, q, q.scalar_type());
  GlaKept none, &x = kept ? *kept : none;
  if (kept) {
    x.wide = wide;
    x.hT = fresh({d.chunks, d.H, d.K, d.V}, q, q.scalar_type());
    x.qg = fresh_like(q);
    x.decay = fresh({d.chunks, d.H, d.K}, q, at::kFloat);
  }
  const fla_stream_t st = stream_of(q);
  const int form = a.head_gates ? 1 : a.gate_form;
  if (auto c = cut_scan(a.plan, d.N, d.T, d.H, (int)(d.V / 64), false, q, d.K * d.V, d.K)) {
    check(fla_chunk_gla_fwd_fused_split(ptr(q), ptr(k), ptr(v), ptr(g), fptr(h0), ptr(o), fptr(*ht), (int*)ptr(wide),
                                        ptr(hwide), ptr(x.hT), ptr(x.qg), fptr(x.decay), nullptr, nullptr, offs(a.plan),
                                        idx(a.plan), coff(a.plan), &c->s, d.NT, dt(q), dt(g), d.B, d.T, d.H, d.K, d.V, d.N,
                                        (float)a.scale, form, (float)a.normalizer, a.clamp.has_value(),
                                        (float)a.clamp.value_or(0.0), st),
          "fla_chunk_gla_fwd_fused_split");
  } else if (form == 1) {
    check(fla_chunk_simple_gla_fwd_fused(ptr(q), ptr(k), ptr(v), fptr(g), fptr(h0), ptr(o), fptr(*ht), (int*)ptr(wide),
                                         ptr(hwide), ptr(x.hT), ptr(x.qg), fptr(x.decay), nullptr, nullptr, offs(a.plan),
                                         idx(a.plan), coff(a.plan), order(a.plan), d.NT, dt(q), d.B, d.T, d.H, d.K, d.V,
                                         d.N, (float)a.scale, st),
          "fla_chunk_simple_gla_fwd_fused");
  } else if (form == 2) {
    check(fla_chunk_gla_fwd_fused_logits(ptr(q), ptr(k), ptr(v), ptr(g), fptr(h0), ptr(o), fptr(*ht), (int*)ptr(wide),
                                         ptr(hwide), offs(a.plan), idx(a.plan), coff(a.plan), order(a.plan), d.NT, dt(q),
                                         dt(g), d.B, d.T, d.H, d.K, d.V, d.N, (float)a.scale, (float)a.normalizer,
                                         a.clamp.has_value(), (float)a.clamp.value_or(0.0), st),
          "fla_chunk_gla_fwd_fused_logits");
  } else if (kept) {
    check(fla_chunk_gla_fwd_fused_kept(ptr(q), ptr(k), ptr(v), ptr(g), fptr(h0), ptr(o), fptr(*ht), (int*)ptr(wide),
                                       ptr(hwide), ptr(x.hT), ptr(x.qg), fptr(x.decay), nullptr, nullptr, offs(a.plan),
                                       idx(a.plan), coff(a.plan), order(a.plan), d.NT, dt(q), dt(g), d.B, d.T, d.H, d.K,
                                       d.V, d.N, (float)a.scale, st),
          "fla_chunk_gla_fwd_fused_kept");
  } else {
    check(fla_chunk_gla_fwd_fused(ptr(q), ptr(k), ptr(v), ptr(g), fptr(h0), ptr(o), fptr(*ht), (int*)ptr(wide), ptr(hwide),
                                  offs(a.plan), idx(a.plan), coff(a.plan), order(a.plan), d.NT, dt(q), dt(g), d.B, d.T, d.H,
                                  d.K, d.V, d.N, (float)a.scale, st),
          "fla_chunk_gla_fwd_fused");
  }
  return o;
}

struct GlaNode : torch::autograd::Function<GlaNode> {
  struct Rest {
    GlaArgs a;
    at::ScalarType g_type;
    bool has_h0;
  };
  static variable_list forward(AutogradContext* ctx, const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& g_,
                               const Maybe& h0_, const Maybe& offsets, const GlaArgs& a) {
    at::AutoDispatchBelowADInplaceOrView guard;
    const Tensor q = q_.contiguous(), k = k_.contiguous(), v = v_.contiguous();
    const Tensor g = (a.head_gates ? f32(g_) : g_.contiguous());
    const Tensor h0 = h0_ ? h0_->contiguous() : Tensor();
    Tensor ht;
    GlaKept x;
    Tensor o = gla_forward(q, k, v, g, h0, a, &ht, &x);
    ctx->save_for_backward({q, k, v, g, x.wide, x.hT, x.qg, x.decay, given(offsets)});
    ctx->set_materialize_grads(false);
    hold(ctx, Rest{a, g_.scalar_type(), h0.defined()});
    return a.want_ht ? variable_list{o, ht} : variable_list{o};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    at::AutoDispatchBelowADInplaceOrView guard;
    const auto saved = ctx->get_saved_variables();
    const Rest& rest = held<Rest>(ctx);
    const GlaArgs& a = rest.a;
    const Dims& d = a.d;
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &g = saved[3], &wide = saved[4], &hT = saved[5], &qg = saved[6],
                 &decay = saved[7];
    const Tensor dout = grads[0].defined() ? as(grads[0], q.scalar_type()).contiguous() : at::zeros(v.sizes(), v.options());
    const Tensor dht = a.want_ht ? f32(grads[1]) : Tensor();
    Tensor dhtf = fresh_like(hT), dq = fresh_like(q), dk = fresh_like(k), dv = fresh_like(v);
    // per-head gates: rows of a packed batch that belong to no sequence have a gradient of zero
    Tensor dg = !a.head_gates                       ? fresh(q.sizes(), q, at::kFloat)
                : !a.plan || a.plan->covers(0, d.T) ? fresh({d.B, d.T, d.H}, q, at::kFloat)
                                                    : at::zeros({d.B, d.T, d.H}, g.options());
    Tensor dh0 = rest.has_h0 ? fresh({d.N, d.H, d.K, d.V}, q, at::kFloat) : Tensor();
    const fla_stream_t st = stream_of(q);
    // (the reverse scan's workgroups hold 64 x 64 tiles of a state)
    auto c = cut_scan(a.plan, d.N, d.T, d.H, (int)(d.K / 64 * (d.V / 64)), true, q, d.K * d.V, d.K,
                      FLA_SCAN_GLA_GRADIENT);
    if (c) {
      check(fla_chunk_gla_bwd_split(ptr(q), ptr(k), ptr(v), ptr(g), ptr(dout), fptr(dht), ptr(hT), ptr(qg), fptr(decay),
                                    nullptr, nullptr, ptr(dhtf), ptr(dq), ptr(dk), ptr(dv), fptr(dg), fptr(dh0),
                                    (const int*)ptr(wide), offs(a.plan), idx(a.plan), coff(a.plan), &c->s, d.NT, dt(q), dt(g),
                                    d.B, d.T, d.H, d.K, d.V, d.N, (float)a.scale, a.head_gates, st),
            "fla_chunk_gla_bwd_split");
    } else if (a.head_gates) {
      check(fla_chunk_simple_gla_bwd(ptr(q), ptr(k), ptr(v), fptr(g), ptr(dout), fptr(dht), ptr(hT), ptr(qg), fptr(decay),
                                     nullptr, nullptr, ptr(dhtf), ptr(dq), ptr(dk), ptr(dv), fptr(dg), fptr(dh0),
                                     (const int*)ptr(wide), offs(a.plan), idx(a.plan), coff(a.plan), d.NT, dt(q), d.B, d.T,
                                     d.H, d.K, d.V, d.N, (float)a.scale, st),
            "fla_chunk_simple_gla_bwd");
    } else {
      check(fla_chunk_gla_bwd_kept(ptr(q), ptr(k), ptr(v), ptr(g), ptr(dout), fptr(dht), ptr(hT), ptr(qg), fptr(decay),
                                   nullptr, nullptr, ptr(dhtf), ptr(dq), ptr(dk), ptr(dv), fptr(dg), fptr(dh0),
                                   (const int*)ptr(wide), offs(a.plan), idx(a.plan), coff(a.plan), d.NT, dt(q), dt(g), d.B,
                                   d.T, d.H, d.K, d.V, d.N, (float)a.scale, st),
            "fla_chunk_gla_bwd_kept");
    }
    return {dq, dk, dv, as(dg, rest.g_type), dh0, Tensor(), Tensor()};
  }
};

// The forward of chunk_simple_gla that is not differentiated
Tensor simple_gla_scan(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& h0, const GlaArgs& a,
                       Tensor* ht) {
  const Dims& d = a.d;
  Tensor o = fresh_like(v);
  if (a.want_ht) *ht = fresh({d.N, d.H, d.K, d.V}, q, at::kFloat);
  if (auto c = cut_scan(a.plan, d.N, d.T, d.H, (int)(d.V / 64), false, q, d.K * d.V, d.K,
                        FLA_SCAN_SIMPLE)) {
    check(fla_chunk_gated_delta_rule_fwd_scan_split(ptr(q), ptr(k), ptr(v), nullptr, fptr(g), nullptr, fptr(h0), ptr(o),
                                                    fptr(*ht), nullptr, nullptr, nullptr, offs(a.plan), coff(a.plan), &c->s,
                                                    dt(q), d.B, d.T, d.H, d.K, d.V, d.N, (float)a.scale, 0.f, stream_of(q)),
          "fla_chunk_gated_delta_rule_fwd_scan_split");
    return o;
  }
  check(fla_chunk_simple_gla_fwd_scan(ptr(q), ptr(k), ptr(v), fptr(g), fptr(h0), ptr(o), fptr(*ht), offs(a.plan),
                                      coff(a.plan), order(a.plan), dt(q), d.B, d.T, d.H, d.K, d.V, d.N, (float)a.scale,
                                      stream_of(q)),
        "fla_chunk_simple_gla_fwd_scan");
  return o;
}

// ---------------------------------------------------------------------------------------------------- delta rule
struct GdrArgs {
  Dims d;
  PlanPtr plan;
  double scale;
  bool want_ht;
  std::optional<double> l2norm_eps;
};
struct GdrKept {
  Tensor gc, AT, Aw, v_new, hT, Aqk, Mt;   // Mt: the segments' transposed transitions where the forward was cut
};

// the kind of a delta-rule scan as fla_scan_split takes it: the same for a forward that keeps its intermediates and its backward
int delta_scan(const Dims& d, bool kept) {
  return (kept ? FLA_SCAN_DELTA_KEPT : FLA_SCAN_DELTA) | (d.K == 64 ? FLA_SCAN_KEYS_64 : 0);
}

Tensor gdr_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta, const Tensor& h0,
                   const GdrArgs& a, Tensor* ht, GdrKept* kept) {
  const Dims& d = a.d;
  const fla_stream_t st = stream_of(q);
  Tensor AT = fresh({d.chunks, d.H, 10, 16, 16}, q, q.scalar_type());
  Tensor gc = g.defined() ? fresh_like(g) : Tensor();
  Tensor o = fresh_like(v);
  if (a.want_ht) *ht = fresh({d.N, d.H, d.K, d.V}, q, at::kFloat);
  // sequences cut into segments: their K x K transitions take the place of the decays
  auto cut = cut_scan(a.plan, d.N, d.T, d.H, (int)(d.V / 64), false, q, d.K * d.V, d.K * d.K,
                      delta_scan(d, kept));
  auto scan_cut = [&](const Tensor& rstd, const GdrKept& x) {
    check(fla_chunk_gated_delta_rule_fwd_scan_split(ptr(q), ptr(k), ptr(v), ptr(AT), fptr(gc), fptr(rstd), fptr(h0), ptr(o),
                                                    fptr(*ht), ptr(x.v_new), ptr(x.hT), ptr(x.Aqk), offs(a.plan), coff(a.plan),
                                                    &cut->s, dt(q), d.B, d.T, d.H, d.K, d.V, d.N, (float)a.scale,
                                                    (float)a.l2norm_eps.value_or(0.0), st),
          "fla_chunk_gated_delta_rule_fwd_scan_split");
  };
  if (a.l2norm_eps) {
    Tensor rstd = fresh({d.B, d.T, d.H}, q, at::kFloat);
    check(fla_gdr_fwd_prep_l2norm(ptr(k), fptr(beta), fptr(g), 0, fptr(gc), ptr(AT), fptr(rstd), offs(a.plan), idx(a.plan),
                                  d.NT, dt(q), d.B, d.T, d.H, d.K, (float)*a.l2norm_eps, st),
          "fla_gdr_fwd_prep_l2norm");
    if (cut) {
      scan_cut(rstd, {});
      return o;
    }
    check(fla_chunk_gated_delta_rule_fwd_scan_l2norm(ptr(q), ptr(k), ptr(v), ptr(AT), fptr(gc), fptr(rstd), fptr(h0), ptr(o),
                                                     fptr(*ht), offs(a.plan), coff(a.plan), order(a.plan), dt(q), d.B, d.T,
                                                     d.H, d.K, d.V, d.N, (float)a.scale, (float)*a.l2norm_eps, st),
          "fla_chunk_gated_delta_rule_fwd_scan_l2norm");
    return o;
  }
  GdrKept none, &x = kept ? *kept : none;
  if (kept) {
    x.gc = gc;
    x.AT = AT;
    x.Aw = fresh({d.B, d.T, d.H, BT}, q, q.scalar_type());
    x.v_new = fresh_like(v);
    x.hT = fresh({d.chunks, d.H, d.K, d.V}, q, q.scalar_type());
    x.Aqk = fresh_like(AT);
    if (cut) {
      x.Mt = fresh_like(cut->transitions);
      cut->s.transitions_t = fptr(x.Mt);
    }
  }
  if (kept)
    check(fla_gdr_fwd_prep_kept(ptr(k), fptr(beta), fptr(g), 0, fptr(gc), ptr(AT), ptr(x.Aw), offs(a.plan), idx(a.plan),
                                d.NT, dt(q), d.B, d.T, d.H, d.K, st),
          "fla_gdr_fwd_prep_kept");
  else
    check(fla_gdr_fwd_prep(ptr(k), fptr(beta), fptr(g), 0, fptr(gc), ptr(AT), nullptr, nullptr, offs(a.plan), idx(a.plan),
                           d.NT, dt(q), d.B, d.T, d.H, d.K, st),
          "fla_gdr_fwd_prep");
  if (cut) {
    scan_cut({}, x);
    return o;
  }
  check(fla_chunk_gated_delta_rule_fwd_scan(ptr(q), ptr(k), ptr(v), ptr(AT), fptr(gc), fptr(h0), ptr(o), fptr(*ht),
                                            ptr(x.v_new), ptr(x.hT), ptr(x.Aqk), offs(a.plan), coff(a.plan), order(a.plan),
                                            dt(q), d.B, d.T, d.H, d.K, d.V, d.N, (float)a.scale, st),
        "fla_chunk_gated_delta_rule_fwd_scan");
  return o;
}

struct GdrNode : torch::autograd::Function<GdrNode> {
  struct Rest {
    GdrArgs a;
    std::optional<at::ScalarType> g_type;
    at::ScalarType beta_type;
    bool has_h0;
  };
  static variable_list forward(AutogradContext* ctx, const Tensor& q_, const Tensor& k_, const Tensor& v_, const Maybe& g_,
                               const Tensor& beta_, const Maybe& h0_, const Maybe& offsets, const GdrArgs& a) {
    at::AutoDispatchBelowADInplaceOrView guard;
    const Tensor q = q_.contiguous(), k = k_.contiguous(), v = v_.contiguous(), g = f32(given(g_)), beta = f32(beta_);
    const Tensor h0 = h0_ ? h0_->contiguous() : Tensor();
    Tensor ht;
    GdrKept x;
    Tensor o = gdr_forward(q, k, v, g, beta, h0, a, &ht, &x);
    ctx->save_for_backward({q, k, v, beta, x.gc, x.AT, x.Aw, x.v_new, x.hT, x.Aqk, x.Mt, given(offsets)});
    ctx->set_materialize_grads(false);
    Rest r{a, std::nullopt, beta_.scalar_type(), h0.defined()};
    if (g_) r.g_type = g_->scalar_type();
    hold(ctx, std::move(r));
    return a.want_ht ? variable_list{o, ht} : variable_list{o};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    at::AutoDispatchBelowADInplaceOrView guard;
    const auto saved = ctx->get_saved_variables();
    const Rest& r = held<Rest>(ctx);
    const GdrArgs& a = r.a;
    const Dims& d = a.d;
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &beta = saved[3], &gc = saved[4], &AT = saved[5], &Aw = saved[6],
                 &v_new = saved[7], &hT = saved[8], &Aqk = saved[9],
                 &Mt = saved[10];
    const Tensor dout = grads[0].defined() ? as(grads[0], q.scalar_type()).contiguous() : at::zeros(v.sizes(), v.options());
    const Tensor dht = a.want_ht ? f32(grads[1]) : Tensor();
    Tensor dv2 = fresh_like(v), dh = fresh_like(hT);
    Tensor dq = fresh_like(q), dk = fresh_like(k), dv = fresh_like(v);
    Tensor dbeta = fresh({d.B, d.T, d.H}, q, at::kFloat), dg = fresh({d.B, d.T, d.H}, q, at::kFloat);
    Tensor dh0 = r.has_h0 ? fresh({d.N, d.H, d.K, d.V}, q, at::kFloat) : Tensor();
    std::optional<Cut> cut;
    if (Mt.defined())
      cut = cut_scan(a.plan, d.N, d.T, d.H, (int)(d.V / 64), true, q, d.K * d.V, 0, delta_scan(d, true));
    if (cut) cut->s.decays = fptr(Mt);
    check(fla_chunk_gated_delta_rule_bwd_tiles(
              ptr(q), ptr(k), ptr(v), ptr(AT), ptr(v_new), fptr(beta), fptr(gc), ptr(Aw), ptr(dout), fptr(dht), ptr(hT),
              ptr(Aqk), ptr(dv2), ptr(dh), ptr(dq), ptr(dk), ptr(dv), fptr(dbeta), fptr(dg), fptr(dh0), offs(a.plan),
              idx(a.plan), coff(a.plan), cut ? &cut->s : nullptr, d.NT, dt(q), d.B, d.T, d.H, d.K, d.V, d.N, (float)a.scale,
              stream_of(q)),
          "fla_chunk_gated_delta_rule_bwd_tiles");
    return {dq, dk, dv, r.g_type ? as(dg, *r.g_type) : Tensor(), as(dbeta, r.beta_type), dh0, Tensor(), Tensor()};
  }
};

// ---------------------------------------------------------------------------------------------------- layer steps
bool rows_ok(const Tensor& x) {
  return x.defined() && x.is_cuda() && x.dim() >= 1 && x.numel() > 0 && x.size(-1) % 8 == 0 && x.size(-1) <= 2048 &&
         (is16(x) || x.scalar_type() == at::kFloat);
}

// The column sums of per-workgroup partial sums [parts, ...], in the dtype and shape of the weight they belong to
Tensor sum_partials(const Tensor& part, at::IntArrayRef shape, at::ScalarType type) {
  const bool direct = type == at::kFloat || type == at::kBFloat16 || type == at::kHalf;
  Tensor out = fresh(shape, part, direct ? type : at::kFloat);
  check(fla_sum_partials(fptr(part), ptr(out), part.size(0), part.numel() / part.size(0), dt(out), stream_of(part)),
        "fla_sum_partials");
  return as(out, type);
}

// Two weights' partial sums side by side [parts, 2, n], added in one launch where both are of one type.  Either may be unwanted.
struct PartialPair {
  Tensor both, a, b;      // (both: where they are of one type)
  int64_t n, ld;
  at::ScalarType at_, bt_;
  PartialPair(bool want_a, bool want_b, at::ScalarType ta, at::ScalarType tb, int64_t parts, int64_t n_, const Tensor& like) : n(n_), ld(n_), at_(ta), bt_(tb) {
    if (want_a && want_b && ta == tb) {
      both = fresh({parts, 2, n}, like, at::kFloat), ld = 2 * n;
    } else {
      if (want_a) a = fresh({parts, n}, like, at::kFloat);
      if (want_b) b = fresh({parts, n}, like, at::kFloat);
    }
  }
  float* first() const { return both.defined() ? fptr(both) : fptr(a); }
  float* second() const { return both.defined() ? fptr(both) + n : fptr(b); }
  void sums(Tensor* x, Tensor* y) const {
    if (both.defined()) {
      const Tensor s = sum_partials(both, {2, n}, at_);
      *x = s.select(0, 0), *y = s.select(0, 1);
    } else {
      if (a.defined()) *x = sum_partials(a, {n}, at_);
      if (b.defined()) *y = sum_partials(b, {n}, bt_);
    }
  }
};

struct L2NormNode : torch::autograd::Function<L2NormNode> {
  static Tensor run(const Tensor& x, double eps) {
    Tensor y = fresh_like(x);
    const int64_t D = x.size(-1);
    check(fla_l2norm_fwd(ptr(x), ptr(y), x.numel() / D, D, (float)eps, dt(x), dt(y), stream_of(x)), "fla_l2norm_fwd");
    return y;
  }
  static Tensor forward(AutogradContext* ctx, const Tensor& x_, double eps) {
    at::AutoDispatchBelowADInplaceOrView guard;
    const Tensor x = x_.contiguous();
    ctx->save_for_backward({x});
    hold(ctx, eps);
    return run(x, eps);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    at::AutoDispatchBelowADInplaceOrView guard;
    const Tensor x = ctx->get_saved_variables()[0], dy = grads[0].contiguous();
    Tensor dx = fresh_like(x);
    const int64_t D = x.size(-1);
    check(fla_l2norm_bwd(ptr(x), ptr(dy), ptr(dx), x.numel() / D, D, (float)held<double>(ctx), dt(x), dt(dy), stream_of(x)),
          "fla_l2norm_bwd");
    return {dx, Tensor()};
  }
};

struct ConvNode : torch::autograd::Function<ConvNode> {
  struct Rest {
    int silu;
    std::vector<int64_t> w_shape;
    at::ScalarType w_type;
    std::optional<at::ScalarType> b_type;
  };
  static Tensor run(const Tensor& x, const Tensor& w, const Tensor& b, int silu) {
    Tensor y = fresh_like(x);
    check(fla_causal_conv1d_fwd(ptr(x), fptr(w), fptr(b), ptr(y), x.size(0), x.size(1), x.size(2), w.size(-1), silu, dt(x),
                                stream_of(x)),
          "fla_causal_conv1d_fwd");
    return y;
  }
  static Tensor forward(AutogradContext* ctx, const Tensor& x_, const Tensor& w_, const Maybe& b_, int silu) {
    at::AutoDispatchBelowADInplaceOrView guard;
    const Tensor x = x_.contiguous(), w = f32(w_), b = f32(given(b_));
    ctx->save_for_backward({x, w, b});
    Rest r{silu, w_.sizes().vec(), w_.scalar_type(), std::nullopt};
    if (b_) r.b_type = b_->scalar_type();
    hold(ctx, std::move(r));
    return run(x, w, b, silu);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    at::AutoDispatchBelowADInplaceOrView guard;
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &b = saved[2];
    const Rest& r = held<Rest>(ctx);
    const int64_t B = x.size(0), T = x.size(1), D = x.size(2), W = w.size(-1);
    const Tensor dy = as(grads[0], x.scalar_type()).contiguous();
    Tensor dx = fresh_like(x);
    const int64_t parts = fla_causal_conv1d_bwd_partials(B, T);
    Tensor dw = fresh({parts, D, W}, x, at::kFloat), db = b.defined() ? fresh({parts, D}, x, at::kFloat) : Tensor();
    check(fla_causal_conv1d_bwd(ptr(x), fptr(w), fptr(b), ptr(dy), ptr(dx), fptr(dw), fptr(db), B, T, D, W, r.silu, dt(x),
                                stream_of(x)),
          "fla_causal_conv1d_bwd");
    return {dx, sum_partials(dw, r.w_shape, r.w_type), b.defined() ? sum_partials(db, {D}, *r.b_type) : Tensor(), Tensor()};
  }
};

struct NormGateNode : torch::autograd::Function<NormGateNode> {
  struct Rest {
    double eps;
    bool rms;
  };
  static Tensor run(const Tensor& x, const Tensor& o, const Tensor& w, const Tensor& b, double eps, bool rms, Tensor* mean,
                    Tensor* rstd) {
    const int64_t D = x.size(-1), M = x.numel() / D;
    Tensor y = fresh_like(x);
    if (!rms) *mean = fresh({M}, x, at::kFloat);
    *rstd = fresh({M}, x, at::kFloat);
    check(fla_norm_swish_gate_fwd(ptr(x), ptr(o), fptr(w), fptr(b), ptr(y), fptr(*mean), fptr(*rstd), M, D, (float)eps, rms,
                                  dt(x), stream_of(x)),
          "fla_norm_swish_gate_fwd");
    return y;
  }
  static Tensor forward(AutogradContext* ctx, const Tensor& x_, const Tensor& o_, const Maybe& w_, const Maybe& b_,
                        double eps, bool rms) {
    at::AutoDispatchBelowADInplaceOrView guard;
    const Tensor w = given(w_), b = given(b_);
    const Tensor x = x_.contiguous(), o = o_.contiguous();
    Tensor mean, rstd;
    Tensor y = run(x, o, f32(w), f32(b), eps, rms, &mean, &rstd);
    ctx->save_for_backward({x, o, w, b, mean, rstd});
    hold(ctx, Rest{eps, rms});
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    at::AutoDispatchBelowADInplaceOrView guard;
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &o = saved[1], &w = saved[2], &b = saved[3], &mean = saved[4], &rstd = saved[5];
    const Rest& r = held<Rest>(ctx);
    const int64_t D = x.size(-1), M = x.numel() / D;
    const Tensor dy = as(grads[0], x.scalar_type()).contiguous();
    Tensor dx = fresh_like(x), dgate = fresh_like(o);
    const int64_t parts = fla_norm_swish_gate_workgroups(M, D);
    Tensor dw = w.defined() ? fresh({parts, D}, x, at::kFloat) : Tensor();
    Tensor db = b.defined() ? fresh({parts, D}, x, at::kFloat) : Tensor();
    const Tensor w32 = f32(w), b32 = f32(b);
    check(fla_norm_swish_gate_bwd(ptr(dy), ptr(x), ptr(o), fptr(w32), fptr(b32), fptr(mean), fptr(rstd), ptr(dx), ptr(dgate),
                                  fptr(dw), fptr(db), M, D, (float)r.eps, r.rms, dt(x), stream_of(x)),
          "fla_norm_swish_gate_bwd");
    return {dx, dgate, w.defined() ? sum_partials(dw, w.sizes(), w.scalar_type()) : Tensor(),
            b.defined() ? sum_partials(db, b.sizes(), b.scalar_type()) : Tensor(), Tensor(), Tensor()};
  }
};

// ---------------------------------------------------------------------------------------------------- elementwise recurrence
// Rows of a [B,T,D] operand as the kernels take them: elements next to each other, all rows one pitch apart (a slice of a wider
// projection is such a one).  Anything else is copied first.
Tensor pitched(const Tensor& x, int64_t* ld) {
  const int64_t B = x.size(0), T = x.size(1), D = x.size(2);
  const int64_t pitch = T > 1 ? x.stride(1) : B > 1 ? x.stride(0) : D;
  const bool fits = (D == 1 || x.stride(2) == 1) && pitch >= D && pitch <= FLA_HGRN_MAX_PITCH && (T == 1 || B == 1 || x.stride(0) == T * x.stride(1));
  *ld = fits ? pitch : D;
  return fits ? x : x.contiguous();
}

struct HgrnArgs {
  PlanPtr plan;           // chunks of `segment` tokens
  int64_t B, T, D, N, segment;
  bool gates, want_ht;
  // whether some sequence has more than one segment
  bool cut() const {
    if (!plan) return T > segment;
    int64_t used = 0;
    for (int64_t i = 0; i < plan->N; ++i) used += plan->host[i + 1] > plan->host[i];
    return plan->NT > used;
  }
  int64_t segments() const { return plan ? plan->NT : B * ((T + segment - 1) / segment); }
  Tensor maps(const Tensor& like) const { return cut() ? fresh({segments(), 2, D}, like, at::kFloat) : Tensor(); }
  // rows of a packed batch that belong to no sequence are zeros
  Tensor rows(const Tensor& like) const {
    return !plan || plan->covers(0, T) ? at::empty({B, T, D}, like.options()) : at::zeros({B, T, D}, like.options());
  }
};

Tensor hgrn_forward(const Tensor& x_, const Tensor& g_, const Tensor& lb, const Tensor& h0, const HgrnArgs& a, Tensor* ht, Tensor* states) {
  int64_t ldx, ldg;
  const Tensor x = pitched(x_, &ldx), g = pitched(g_, &ldg);
  Tensor o = a.rows(x), maps = a.maps(x);
  if (a.want_ht && !ht->defined()) *ht = fresh({a.N, a.D}, x, at::kFloat);
  if (states) *states = fresh({a.B * a.T / FLA_HGRN_STATE_ROWS + a.N + 1, a.D}, x, at::kFloat);
  if (a.T == 1 && !a.plan && !states)
    check(fla_hgrn_step(ptr(x), ptr(g), fptr(lb), fptr(h0), ptr(o), fptr(*ht), a.gates, dt(x), dt(g), a.N, a.D, ldx, ldg, stream_of(x)),
          "fla_hgrn_step");
  else
    check(fla_hgrn_fwd(ptr(x), ptr(g), fptr(lb), fptr(h0), ptr(o), fptr(*ht), states ? fptr(*states) : nullptr, fptr(maps), offs(a.plan),
                       idx(a.plan), coff(a.plan), a.plan ? a.plan->NT : 0, a.segment, a.gates, dt(x), dt(g), a.B, a.T, a.D, a.N, ldx, ldg,
                       stream_of(x)),
          "fla_hgrn_fwd");
  return o;
}

struct HgrnNode : torch::autograd::Function<HgrnNode> {
  struct Rest {
    HgrnArgs a;
    bool lb, h0;     // whether they have a gradient
  };
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& g, const Maybe& lb_, const Maybe& h0_,
                               const Maybe& offsets, const HgrnArgs& a) {
    at::AutoDispatchBelowADInplaceOrView guard;
    const Tensor lb = given(lb_), h0 = given(h0_);
    Tensor ht, states;
    Tensor o = hgrn_forward(x, g, lb, h0, a, &ht, &states);
    ctx->save_for_backward({x, g, lb, states, given(offsets)});
    ctx->set_materialize_grads(false);
    hold(ctx, Rest{a, asks(lb), asks(h0)});
    return a.want_ht ? variable_list{o, ht} : variable_list{o};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    at::AutoDispatchBelowADInplaceOrView guard;
    const auto saved = ctx->get_saved_variables();
    const Rest& r = held<Rest>(ctx);
    const HgrnArgs& a = r.a;
    int64_t ldx, ldg;
    const Tensor x = pitched(saved[0], &ldx), g = pitched(saved[1], &ldg);
    const Tensor &lb = saved[2], &states = saved[3];
    c10::DeviceGuard on_device(x.device());
    const Tensor dout = grads[0].defined() ? as(grads[0], x.scalar_type()).contiguous() : Tensor();
    const Tensor dht = a.want_ht ? f32(grads[1]) : Tensor();
    Tensor dx = a.rows(x), dg = a.rows(g), maps = a.maps(x);
    Tensor dh0 = r.h0 ? fresh({a.N, a.D}, x, at::kFloat) : Tensor();
    const int64_t segments = a.segments();
    Tensor part = r.lb && segments > 0 ? fresh({segments, a.D}, x, at::kFloat) : Tensor();
    check(fla_hgrn_bwd(ptr(x), ptr(g), fptr(lb), fptr(states), ptr(dout), fptr(dht), ptr(dx), ptr(dg), fptr(dh0), fptr(part), fptr(maps),
                       offs(a.plan), idx(a.plan), coff(a.plan), a.plan ? a.plan->NT : 0, a.segment, a.gates, dt(x), dt(g), a.B, a.T, a.D,
                       a.N, ldx, ldg, stream_of(x)),
          "fla_hgrn_bwd");
    Tensor dlb;
    if (part.defined()) dlb = sum_partials(part, {a.D}, at::kFloat);
    else if (r.lb) dlb = at::zeros({a.D}, x.options().dtype(at::kFloat));
    return {dx, dg, dlb, dh0, Tensor(), Tensor()};
  }
};

// ---------------------------------------------------------------------------------------------------- RMS norm, layer norm
enum NormKind { kRowsOnly, kRms, kLayer };
struct NormArgs {
  double eps;
  std::optional<at::ScalarType> kept_type;   // of the sum x + residual; none: nothing is added and x itself is what is normalised
  long rows8;                                // FLA_ROWS_*
  NormKind kind;
};
struct NormOut {
  Tensor y, scale, kept, mean, rstd;
};
// Any shape [..., N], contiguous operands
NormOut norm_forward(const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& res, const NormArgs& a, bool want_rstd) {
  const int64_t N = x.size(-1), M = x.numel() / N;
  NormOut o;
  o.y = a.rows8 ? fresh(x.sizes(), x, a.rows8 == FLA_ROWS_INT8 ? at::kChar : at::kFloat8_e4m3fn) : fresh_like(x);
  if (a.rows8) o.scale = fresh(x.sizes().slice(0, x.dim() - 1), x, at::kFloat);
  if (a.kept_type) o.kept = fresh(x.sizes(), x, *a.kept_type);
  if (want_rstd) o.rstd = fresh({M}, x, at::kFloat);
  if (want_rstd && a.kind == kLayer) o.mean = fresh({M}, x, at::kFloat);
  if (M == 0) return o;
  const Tensor& any_w = w.defined() ? w : b;
  const int rt = res.defined() ? dt(res) : dt(x), wt = any_w.defined() ? dt(any_w) : dt(x), kt = o.kept.defined() ? dt(o.kept) : dt(x);
  if (a.kind == kLayer)
    check(fla_layer_norm_fwd(ptr(x), ptr(res), rt, ptr(w), ptr(b), wt, ptr(o.y), fptr(o.scale), ptr(o.kept), kt, fptr(o.mean), fptr(o.rstd), M,
                             N, (float)a.eps, (int)a.rows8, dt(x), stream_of(x)),
          "fla_layer_norm_fwd");
  else if (a.rows8)
    check(fla_rms_norm_rows8_fwd(ptr(x), ptr(res), rt, ptr(w), ptr(b), wt, ptr(o.y), fptr(o.scale), ptr(o.kept), kt, M, N, (float)a.eps,
                                 a.kind == kRms, (int)a.rows8, dt(x), stream_of(x)),
          "fla_rms_norm_rows8_fwd");
  else
    check(fla_rms_norm_fwd(ptr(x), ptr(res), rt, ptr(w), ptr(b), wt, ptr(o.y), nullptr, ptr(o.kept), kt, fptr(o.rstd), M, N, (float)a.eps, 1,
                           dt(x), stream_of(x)),
          "fla_rms_norm_fwd");
  return o;
}

struct NormNode : torch::autograd::Function<NormNode> {
  struct Rest {
    bool w, b, res;  // whether they have a gradient
    at::ScalarType type;
  };
  static variable_list forward(AutogradContext* ctx, const Tensor& x_, const Maybe& w_, const Maybe& b_, const Maybe& res_, const NormArgs& a) {
    at::AutoDispatchBelowADInplaceOrView guard;
    const Tensor x = x_.contiguous(), w = given(w_), b = given(b_), res = res_ ? res_->contiguous() : Tensor();
    NormOut o = norm_forward(x, w, b, res, a, true);
    ctx->save_for_backward({o.kept.defined() ? o.kept : x, w, b, o.rstd, o.mean});
    ctx->set_materialize_grads(false);
    hold(ctx, Rest{asks(w), asks(b), res_ && asks(*res_), x.scalar_type()});
    return o.kept.defined() ? variable_list{o.y, o.kept} : variable_list{o.y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    at::AutoDispatchBelowADInplaceOrView guard;
    const auto saved = ctx->get_saved_variables();
    const Tensor &kept = saved[0], &w = saved[1], &b = saved[2], &rstd = saved[3], &mean = saved[4];
    const Rest& r = held<Rest>(ctx);
    c10::DeviceGuard on_device(kept.device());
    const int64_t N = kept.size(-1), M = kept.numel() / N;
    const Tensor dy = grads[0].defined() ? as(grads[0], r.type).contiguous() : at::zeros(kept.sizes(), kept.options().dtype(r.type));
    const Tensor dres = grads.size() > 1 && grads[1].defined() ? as(grads[1], kept.scalar_type()).contiguous() : Tensor();
    Tensor dx = fresh(kept.sizes(), kept, r.type);
    Tensor dres_in = r.res && kept.scalar_type() != r.type ? fresh_like(kept) : Tensor();
    if (M == 0)
      return {dx, r.w ? at::zeros_like(w) : Tensor(), r.b ? at::zeros_like(b) : Tensor(), r.res ? (dres_in.defined() ? dres_in : dx) : Tensor(),
              Tensor()};
    const int64_t parts = mean.defined() ? fla_layer_norm_workgroups(M, N) : fla_rms_norm_workgroups(M, N);
    const int wt = w.defined() ? dt(w) : dt(kept);
    if (mean.defined()) {
      const PartialPair part(r.w, r.b, w.defined() ? w.scalar_type() : at::kFloat, b.defined() ? b.scalar_type() : at::kFloat, parts, N, kept);
      check(fla_layer_norm_bwd(ptr(dy), ptr(kept), dt(kept), ptr(w), wt, fptr(mean), fptr(rstd), ptr(dres), ptr(dx), ptr(dres_in), part.first(),
                               part.second(), part.ld, M, N, dt(dx), stream_of(kept)),
            "fla_layer_norm_bwd");
      Tensor gw, gb;
      part.sums(&gw, &gb);
      return {dx, gw, gb, r.res ? (dres_in.defined() ? dres_in : dx) : Tensor(), Tensor()};
    }
    Tensor dw = r.w ? fresh({parts, N}, kept, at::kFloat) : Tensor(), db = r.b ? fresh({parts, N}, kept, at::kFloat) : Tensor();
    check(fla_rms_norm_bwd(ptr(dy), ptr(kept), dt(kept), ptr(w), wt, fptr(rstd), ptr(dres), ptr(dx), ptr(dres_in), fptr(dw), fptr(db), M, N,
                           dt(dx), stream_of(kept)),
          "fla_rms_norm_bwd");
    return {dx, r.w ? sum_partials(dw, w.sizes(), w.scalar_type()) : Tensor(), r.b ? sum_partials(db, b.sizes(), b.scalar_type()) : Tensor(),
            r.res ? (dres_in.defined() ? dres_in : dx) : Tensor(), Tensor()};
  }
};

// ---------------------------------------------------------------------------------------------------- gated product
// Rows at 16-byte addresses; with `pieces`, of a multiple of so many elements: zeros are added behind them
Tensor whole_rows(const Tensor& t, int64_t pieces = 1) {
  const int64_t K = t.size(-1), more = (pieces - K % pieces) % pieces;
  Tensor c = more ? at::constant_pad_nd(t, {0, more}) : t.contiguous();
  return (uintptr_t)c.data_ptr() % 16 == 0 ? c : c.clone();
}

// A bias, or none, at an address of whole words
Tensor whole_bias(const Tensor& b) {
  if (!b.defined()) return b;
  const Tensor c = b.contiguous();
  return (uintptr_t)c.data_ptr() % 4 == 0 ? c : c.clone();
}

struct GatedNode : torch::autograd::Function<GatedNode> {
  struct Rest {
    bool x, wg, wu, bg, bu;  // whether they have a gradient
    at::ScalarType type, bg_type, bu_type;
    int64_t F;
    long act;
  };
  // kept: g and u [2, M, ld] in fp32 for a backward, and the operands as the kernels took them; or NULL
  struct Kept {
    Tensor gu, x, wg, wu;
  };
  static Tensor run(const Tensor& x_, const Tensor& wg_, const Tensor& wu_, const Tensor& bg_, const Tensor& bu_, long act, Kept* kept) {
    const int64_t F = wg_.size(0), K0 = x_.size(-1), M = x_.numel() / K0, ld = (F + 7) / 8 * 8;
    auto shape = x_.sizes().vec();
    shape.back() = F;
    Tensor h = fresh(shape, x_, x_.scalar_type());
    if (kept) kept->gu = fresh({2, M, ld}, x_, at::kFloat);
    if (M == 0) return h;
    const Tensor x = whole_rows(x_, 8), wg = whole_rows(wg_, 8), wu = whole_rows(wu_, 8);
    if (kept) kept->x = x, kept->wg = wg, kept->wu = wu;
    const bool same = (!bg_.defined() || bg_.scalar_type() == x.scalar_type()) && (!bu_.defined() || bu_.scalar_type() == x.scalar_type());
    const Tensor bg = whole_bias(same ? bg_ : f32(bg_)), bu = whole_bias(same ? bu_ : f32(bu_));
    const int64_t K = x.size(-1);
    const int splits = fla_gated_linear_splits(M, F, K, 2);
    const Tensor sums = splits > 1 ? fresh({splits, M, 2, F}, x, at::kFloat) : Tensor();
    float* keep = kept ? fptr(kept->gu) : nullptr;
    check(fla_gated_linear_fwd(ptr(x), ptr(wg), ptr(wu), ptr(bg), ptr(bu), same ? dt(x) : FLA_F32, ptr(h), keep,
                               keep ? keep + M * ld : nullptr, ld, M, F, K, (int)act, dt(x), ptr(sums), stream_of(x)),
          "fla_gated_linear_fwd");
    return h;
  }
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& wg, const Tensor& wu, const Maybe& bg_, const Maybe& bu_, long act) {
    at::AutoDispatchBelowADInplaceOrView guard;
    const Tensor bg = given(bg_), bu = given(bu_);
    Kept kept;
    Tensor h = run(x, wg, wu, bg, bu, act, &kept);
    const Rest r{asks(x), asks(wg), asks(wu), asks(bg), asks(bu), x.scalar_type(), bg.defined() ? bg.scalar_type() : at::kFloat, bu.defined() ? bu.scalar_type() : at::kFloat,
                 wg.size(0), act};
    // (x for the weights' gradients, the weights for x's)
    // The operands themselves are saved, so that a backward after they were written to is refused, and beside them what they were copied into, if they were.
    auto copy = [](bool wanted, const Tensor& k, const Tensor& t) { return wanted && k.defined() && !k.is_same(t) && k.data_ptr() != t.data_ptr() ? k : Tensor(); };
    const bool w = r.wg || r.wu;
    ctx->save_for_backward({w ? x : Tensor(), r.x ? wg : Tensor(), r.x ? wu : Tensor(), kept.gu, copy(w, kept.x, x), copy(r.x, kept.wg, wg), copy(r.x, kept.wu, wu)});
    ctx->saved_data["shape"] = x.sizes().vec();
    hold(ctx, r);
    return h;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    at::AutoDispatchBelowADInplaceOrView guard;
    const auto saved = ctx->get_saved_variables();
    const Tensor& kept = saved[3];
    const Rest& r = held<Rest>(ctx);
    const auto shape = ctx->saved_data["shape"].toIntVector();
    c10::DeviceGuard on_device(kept.device());
    const int64_t M = kept.size(1), ld = kept.size(2), F = r.F, K0 = shape.back(), K = (K0 + 7) / 8 * 8;
    const auto type = r.type;
    Tensor dx, dwg, dwu, dbg, dbu;
    if (M == 0) {
      auto zeros = [&](bool wanted, at::IntArrayRef sizes, at::ScalarType t) { return wanted ? at::zeros(sizes, kept.options().dtype(t)) : Tensor(); };
      return {zeros(r.x, shape, type), zeros(r.wg, {F, K0}, type), zeros(r.wu, {F, K0}, type), zeros(r.bg, {F}, r.bg_type), zeros(r.bu, {F}, r.bu_type),
              Tensor()};
    }
    const Tensor dh = as(grads[0], type).contiguous();
    const Tensor d = fresh(kept.sizes(), kept, type);
    const int64_t rows = fla_gated_linear_bwd_rows(M), parts = (M + rows - 1) / rows, half = M * ld * 2;
    const PartialPair part(r.bg, r.bu, r.bg_type, r.bu_type, parts, F, kept);
    const fla_stream_t stream = stream_of(kept);
    const float* g = fptr(kept);
    char* dg = (char*)d.data_ptr();
    check(fla_gated_linear_bwd_gate(ptr(dh), g, g + M * ld, dg, dg + half, part.first(), part.second(), part.ld, ld, M, F, (int)r.act, dt(d), stream),
          "fla_gated_linear_bwd_gate");
    part.sums(&dbg, &dbu);
    if (r.x) {
      const Tensor wg = saved[5].defined() ? saved[5] : whole_rows(saved[1], 8), wu = saved[6].defined() ? saved[6] : whole_rows(saved[2], 8);
      dx = fresh(shape, kept, type);
      const int splits = fla_gated_linear_bwd_dx_splits(M, F, K);
      const Tensor sums = splits > 1 ? fresh({splits, M, K}, kept, at::kFloat) : Tensor();
      check(fla_gated_linear_bwd_dx(dg, dg + half, ptr(wg), ptr(wu), ptr(dx), ld, K0, M, F, K, dt(d), fptr(sums), stream), "fla_gated_linear_bwd_dx");
    }
    if (r.wg || r.wu) {
      const Tensor x = saved[4].defined() ? saved[4] : whole_rows(saved[0], 8);
      if (r.wg) dwg = fresh({F, K0}, kept, type);
      if (r.wu) dwu = fresh({F, K0}, kept, type);
      const int splits = fla_gated_linear_bwd_dw_splits(M, F, K, r.wg && r.wu);
      const Tensor sums = splits > 1 ? fresh({r.wg && r.wu ? 2 : 1, splits, F, K}, kept, at::kFloat) : Tensor();
      check(fla_gated_linear_bwd_dw(dg, dg + half, ptr(x), ptr(dwg), ptr(dwu), ld, K0, M, F, K, dt(d), fptr(sums), stream), "fla_gated_linear_bwd_dw");
    }
    return {dx, dwg, dwu, dbg, dbu, Tensor()};
  }
};

// ---------------------------------------------------------------------------------------------------- Python entries
Tensor arg_tensor(PyObject* o) {
  if (o == Py_None) return Tensor();
  TORCH_CHECK_TYPE(THPVariable_Check(o), "fla_amd: expected a tensor, got ", Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}
bool arg_bool(PyObject* o) {
  const int r = PyObject_IsTrue(o);
  if (r < 0) throw python_error();
  return r != 0;
}
long arg_long(PyObject* o) {
  const long r = PyLong_AsLong(o);
  if (r == -1 && PyErr_Occurred()) throw python_error();
  return r;
}
double arg_double(PyObject* o) {
  const double r = PyFloat_AsDouble(o);
  if (r == -1.0 && PyErr_Occurred()) throw python_error();
  return r;
}
std::optional<double> arg_opt_double(PyObject* o) {
  if (o == Py_None) return std::nullopt;
  return arg_double(o);
}
constexpr const char* kPlanName = "fla_amd.plan";
PlanPtr arg_plan(PyObject* o) {
  if (o == Py_None) return PlanPtr();
  auto* p = (Plan*)PyCapsule_GetPointer(o, kPlanName);
  if (!p) throw python_error();
  return PlanPtr::reclaim_copy(p);
}
void expect(Py_ssize_t n, Py_ssize_t want) { TORCH_CHECK_TYPE(n == want, "fla_amd: expected ", want, " arguments, got ", n); }
PyObject* none() { Py_RETURN_NONE; }
PyObject* pair(const Tensor& o, const Tensor& ht) {
  PyObject* t = PyTuple_New(2);
  if (!t) throw python_error();
  PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(o));
  if (ht.defined()) {
    PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(ht));
  } else {
    Py_INCREF(Py_None);
    PyTuple_SET_ITEM(t, 1, Py_None);
  }
  return t;
}

void plan_free(PyObject* cap) { PlanPtr::reclaim((Plan*)PyCapsule_GetPointer(cap, kPlanName)); }

// plan(offsets, indices, chunk_offsets, seq_order, host offsets as a CPU int64 tensor)
PyObject* py_plan(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 5);
  auto p = c10::make_intrusive<Plan>();
  p->offsets = arg_tensor(a[0]);
  p->indices = arg_tensor(a[1]);
  p->chunk_offsets = arg_tensor(a[2]);
  p->seq_order = arg_tensor(a[3]);
  const Tensor host = arg_tensor(a[4]).contiguous();
  const int64_t* h = host.data_ptr<int64_t>();
  p->host.assign(h, h + host.numel());
  p->N = host.numel() - 1;
  p->NT = p->indices.size(0);
  return PyCapsule_New(p.release(), kPlanName, plan_free);
  END_HANDLE_TH_ERRORS
}

// chunk_gla(q, k, v, g, scale, h0, want_ht, plan, may_differentiate, normalizer, clamp, offsets)
//   normalizer None: g holds log-gates
PyObject* py_chunk_gla(PyObject*, PyObject* const* p, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 12);
  Tensor q = arg_tensor(p[0]), k = arg_tensor(p[1]), v = arg_tensor(p[2]), g = arg_tensor(p[3]), h0 = arg_tensor(p[5]),
         offsets = arg_tensor(p[11]);
  GlaArgs a{};
  a.plan = arg_plan(p[7]);
  if (!chunk_operands(q, k, v, h0, a.plan, &a.d) || !g.defined() || !g.is_cuda() || g.sizes() != q.sizes()) return none();
  if (g.scalar_type() != at::kFloat && g.scalar_type() != q.scalar_type()) return none();
  const bool grad = wants_grad({&q, &k, &v, &g, &h0});
  const auto normalizer = arg_opt_double(p[9]);
  if (grad && (normalizer || !arg_bool(p[8]))) return none();
  a.scale = p[4] == Py_None ? 1.0 / std::sqrt((double)a.d.K) : arg_double(p[4]);
  if (grad && a.scale == 0.0) return none();
  a.want_ht = arg_bool(p[6]);
  if (normalizer) {
    a.gate_form = 2;
    a.normalizer = *normalizer;
    a.clamp = arg_opt_double(p[10]);
  }
  if (grad) {
    auto out = GlaNode::apply(q, k, v, g, maybe(h0), maybe(offsets), a);
    return pair(out[0], a.want_ht ? out[1] : Tensor());
  }
  at::AutoDispatchBelowADInplaceOrView guard;
  Tensor ht;
  Tensor o = gla_forward(q.contiguous(), k.contiguous(), v.contiguous(), g.contiguous(), h0.defined() ? h0.contiguous() : h0, a,
                         &ht, nullptr);
  return pair(o, ht);
  END_HANDLE_TH_ERRORS
}

// chunk_simple_gla(q, k, v, g, scale, h0, want_ht, plan, may_differentiate, offsets)
PyObject* py_chunk_simple_gla(PyObject*, PyObject* const* p, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 10);
  Tensor q = arg_tensor(p[0]), k = arg_tensor(p[1]), v = arg_tensor(p[2]), g = arg_tensor(p[3]), h0 = arg_tensor(p[5]),
         offsets = arg_tensor(p[9]);
  GlaArgs a{};
  a.plan = arg_plan(p[7]);
  if (!chunk_operands(q, k, v, h0, a.plan, &a.d) || !g.defined() || !g.is_cuda() || g.dim() != 3 || g.size(0) != a.d.B ||
      g.size(1) != a.d.T || g.size(2) != a.d.H || !g.is_floating_point())
    return none();
  const bool grad = wants_grad({&q, &k, &v, &g, &h0});
  if (grad && !arg_bool(p[8])) return none();
  a.scale = p[4] == Py_None ? 1.0 / std::sqrt((double)a.d.K) : arg_double(p[4]);
  if (grad && a.scale == 0.0) return none();
  a.want_ht = arg_bool(p[6]);
  a.head_gates = true;
  if (grad) {
    auto out = GlaNode::apply(q, k, v, g, maybe(h0), maybe(offsets), a);
    return pair(out[0], a.want_ht ? out[1] : Tensor());
  }
  at::AutoDispatchBelowADInplaceOrView guard;
  Tensor ht;
  Tensor o = simple_gla_scan(q.contiguous(), k.contiguous(), v.contiguous(), f32(g), h0.defined() ? h0.contiguous() : h0, a, &ht);
  return pair(o, ht);
  END_HANDLE_TH_ERRORS
}

// chunk_gdr(q, k, v, g | None, beta, scale, h0, want_ht, plan, may_differentiate, l2norm_eps | None, offsets)
PyObject* py_chunk_gdr(PyObject*, PyObject* const* p, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 12);
  Tensor q = arg_tensor(p[0]), k = arg_tensor(p[1]), v = arg_tensor(p[2]), g = arg_tensor(p[3]), beta = arg_tensor(p[4]),
         h0 = arg_tensor(p[6]), offsets = arg_tensor(p[11]);
  GdrArgs a{};
  a.plan = arg_plan(p[8]);
  if (!chunk_operands(q, k, v, h0, a.plan, &a.d) || !beta.defined() || !on_gpu({&g, &beta})) return none();
  auto per_head = [&](const Tensor& t) {
    return t.dim() == 3 && t.size(0) == a.d.B && t.size(1) == a.d.T && t.size(2) == a.d.H && t.is_floating_point();
  };
  if (!per_head(beta) || (g.defined() && !per_head(g))) return none();
  const bool grad = wants_grad({&q, &k, &v, &g, &beta, &h0});
  if (grad && !arg_bool(p[9])) return none();
  a.scale = arg_double(p[5]);
  a.want_ht = arg_bool(p[7]);
  a.l2norm_eps = arg_opt_double(p[10]);
  if (grad) {
    if (a.l2norm_eps) {
      q = L2NormNode::apply(q, *a.l2norm_eps);
      k = L2NormNode::apply(k, *a.l2norm_eps);
      a.l2norm_eps.reset();
    }
    auto out = GdrNode::apply(q, k, v, maybe(g), beta, maybe(h0), maybe(offsets), a);
    return pair(out[0], a.want_ht ? out[1] : Tensor());
  }
  at::AutoDispatchBelowADInplaceOrView guard;
  Tensor ht;
  Tensor o = gdr_forward(q.contiguous(), k.contiguous(), v.contiguous(), f32(g), f32(beta), h0.defined() ? h0.contiguous() : h0, a,
                         &ht, nullptr);
  return pair(o, ht);
  END_HANDLE_TH_ERRORS
}

// The recurrences on equal-length sequences, without gradients.  State in fp32, contiguous where it is updated in place.
bool recurrent_operands(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& h0, bool inplace, Dims* d) {
  if (!q.defined() || !k.defined() || !v.defined() || q.dim() != 4 || v.dim() != 4 || q.sizes() != k.sizes() || q.numel() == 0)
    return false;
  if (!(is16(q) || q.scalar_type() == at::kFloat) || k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type())
    return false;
  d->B = d->N = q.size(0), d->T = q.size(1), d->H = q.size(2), d->K = q.size(3), d->V = v.size(3);
  if (v.size(0) != d->B || v.size(1) != d->T || v.size(2) != d->H || d->K > 256 || d->V % 4 != 0 || d->V == 0) return false;
  if (inplace && (!h0.defined() || !h0.is_contiguous())) return false;
  return !h0.defined() || (h0.scalar_type() == at::kFloat && h0.dim() == 4 && h0.size(0) == d->N && h0.size(1) == d->H &&
                           h0.size(2) == d->K && h0.size(3) == d->V);
}
Tensor cont(const Tensor& x) { return x.defined() && !x.is_contiguous() ? x.contiguous() : x; }

// recurrent_gla(q, k, v, g | None, gk | None, gv | None, scale, h0, want_ht, reverse, inplace)
PyObject* py_recurrent_gla(PyObject*, PyObject* const* p, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 11);
  Tensor q = arg_tensor(p[0]), k = arg_tensor(p[1]), v = arg_tensor(p[2]), g = arg_tensor(p[3]), gk = arg_tensor(p[4]),
         gv = arg_tensor(p[5]), h0 = arg_tensor(p[7]);
  Dims d{};
  const bool want = arg_bool(p[8]), inplace = arg_bool(p[10]);
  if (wants_grad({&q, &k, &v, &g, &gk, &gv, &h0}) || !on_gpu({&q, &k, &v, &g, &gk, &gv, &h0}) ||
      !recurrent_operands(q, k, v, h0, inplace && want, &d))
    return none();
  at::ScalarType gt = at::kFloat;
  bool have = false;
  for (const Tensor* t : {&g, &gk, &gv}) {
    if (!t->defined()) continue;
    if (have && t->scalar_type() != gt) return none();
    gt = t->scalar_type();
    have = true;
  }
  if (gt != at::kFloat && gt != q.scalar_type()) return none();
  if ((g.defined() && g.numel() != d.B * d.T * d.H) || (gk.defined() && gk.sizes() != k.sizes()) ||
      (gv.defined() && gv.sizes() != v.sizes()))
    return none();
  at::AutoDispatchBelowADInplaceOrView guard;
  q = cont(q), k = cont(k), v = cont(v), g = cont(g), gk = cont(gk), gv = cont(gv), h0 = cont(h0);
  Tensor o = fresh_like(v), ht;
  if (want) ht = inplace ? h0 : fresh({d.N, d.H, d.K, d.V}, q, at::kFloat);
  check(fla_fused_recurrent_fwd(ptr(q), ptr(k), ptr(v), ptr(g), ptr(gk), ptr(gv), ptr(o), fptr(h0), fptr(ht), nullptr, dt(q),
                                gt == at::kFloat ? FLA_F32 : dt(q), dt(o), d.B, d.T, d.H, d.K, d.V, d.N,
                                (float)arg_double(p[6]), arg_bool(p[9]), stream_of(q)),
        "fla_fused_recurrent_fwd");
  return pair(o, ht);
  END_HANDLE_TH_ERRORS
}

// recurrent_gdr(q, k, v, g | None, beta, scale, h0, want_ht, inplace, l2norm_eps | None)
PyObject* py_recurrent_gdr(PyObject*, PyObject* const* p, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 10);
  Tensor q = arg_tensor(p[0]), k = arg_tensor(p[1]), v = arg_tensor(p[2]), g = arg_tensor(p[3]), beta = arg_tensor(p[4]),
         h0 = arg_tensor(p[6]);
  Dims d{};
  const bool want = arg_bool(p[7]), inplace = arg_bool(p[8]);
  if (wants_grad({&q, &k, &v, &g, &beta, &h0}) || !beta.defined() || !on_gpu({&q, &k, &v, &g, &beta, &h0}) ||
      !recurrent_operands(q, k, v, h0, inplace && want, &d))
    return none();
  const bool per_value = beta.dim() == 4;
  if (per_value ? beta.sizes() != v.sizes() : beta.numel() != d.B * d.T * d.H) return none();
  if (g.defined() && g.numel() != d.B * d.T * d.H) return none();
  at::AutoDispatchBelowADInplaceOrView guard;
  q = cont(q), k = cont(k), v = cont(v), h0 = cont(h0), g = f32(g), beta = f32(beta);
  Tensor o = fresh_like(v), ht;
  if (want) ht = inplace ? h0 : fresh({d.N, d.H, d.K, d.V}, q, at::kFloat);
  const float scale = (float)arg_double(p[5]);
  if (const auto eps = arg_opt_double(p[9]))
    check(fla_fused_recurrent_gated_delta_rule_fwd_l2norm(ptr(q), ptr(k), ptr(v), ptr(g), ptr(beta), ptr(o), fptr(h0), fptr(ht),
                                                          nullptr, dt(q), FLA_F32, dt(o), per_value, d.B, d.T, d.H, d.K, d.V,
                                                          d.N, scale, (float)*eps, stream_of(q)),
          "fla_fused_recurrent_gated_delta_rule_fwd_l2norm");
  else
    check(fla_fused_recurrent_gated_delta_rule_fwd(ptr(q), ptr(k), ptr(v), ptr(g), ptr(beta), ptr(o), fptr(h0), fptr(ht),
                                                   nullptr, dt(q), FLA_F32, dt(o), per_value, d.B, d.T, d.H, d.K, d.V, d.N,
                                                   scale, stream_of(q)),
          "fla_fused_recurrent_gated_delta_rule_fwd");
  return pair(o, ht);
  END_HANDLE_TH_ERRORS
}

// l2_norm(x, eps)
PyObject* py_l2_norm(PyObject*, PyObject* const* p, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 2);
  const Tensor x = arg_tensor(p[0]);
  if (!rows_ok(x)) return none();
  const double eps = arg_double(p[1]);
  if (wants_grad({&x})) return THPVariable_Wrap(L2NormNode::apply(x, eps));
  at::AutoDispatchBelowADInplaceOrView guard;
  return THPVariable_Wrap(L2NormNode::run(x.contiguous(), eps));
  END_HANDLE_TH_ERRORS
}

bool conv_weights_ok(const Tensor& w, const Tensor& b, int64_t D) {
  return w.defined() && w.is_cuda() && w.dim() >= 2 && w.size(0) == D && w.size(-1) >= 2 && w.size(-1) <= 4 &&
         w.numel() == D * w.size(-1) && w.is_floating_point() &&
         (!b.defined() || (b.is_cuda() && b.numel() == D && b.is_floating_point()));
}

// causal_conv1d(x [B,T,D], weight, bias | None, silu)
PyObject* py_conv(PyObject*, PyObject* const* p, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 4);
  const Tensor x = arg_tensor(p[0]), w = arg_tensor(p[1]), b = arg_tensor(p[2]);
  if (!x.defined() || !x.is_cuda() || x.dim() != 3 || x.numel() == 0 || x.size(2) % 8 != 0 ||
      !(is16(x) || x.scalar_type() == at::kFloat) || !conv_weights_ok(w, b, x.size(2)))
    return none();
  const int silu = arg_bool(p[3]);
  if (wants_grad({&x, &w, &b})) return THPVariable_Wrap(ConvNode::apply(x, w, maybe(b), silu));
  at::AutoDispatchBelowADInplaceOrView guard;
  return THPVariable_Wrap(ConvNode::run(x.contiguous(), f32(w), f32(b), silu));
  END_HANDLE_TH_ERRORS
}

// causal_conv1d_update(x [B,D], cache [B,D,W], weight, bias | None, silu): the cache is updated in place
// short_conv_step: the same for x [B,1,D], as the module gets it (a squeeze and an unsqueeze around a launch of 2.5 us cost the
// host 2 us)
template <bool STEP>
PyObject* py_conv_update(PyObject*, PyObject* const* p, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 5);
  const Tensor x = arg_tensor(p[0]), cache = arg_tensor(p[1]), w = arg_tensor(p[2]), b = arg_tensor(p[3]);
  if (!x.defined() || !cache.defined() || !x.is_cuda() || !cache.is_cuda() || x.dim() != (STEP ? 3 : 2) || x.numel() == 0 ||
      (STEP && x.size(1) != 1) || !(is16(x) || x.scalar_type() == at::kFloat) || !conv_weights_ok(w, b, x.size(-1)))
    return none();
  if (has_tangent({&x, &cache, &w, &b})) return none();   // (the wrapper refuses it)
  const int64_t B = x.size(0), D = x.size(-1), W = w.size(-1);
  if (cache.dim() != 3 || cache.size(0) != B || cache.size(1) != D || cache.size(2) != W || !cache.is_contiguous() ||
      cache.scalar_type() != x.scalar_type())
    return none();
  at::AutoDispatchBelowADInplaceOrView guard;
  const Tensor xc = x.contiguous(), b32 = f32(b);
  const Tensor wc = w.scalar_type() == x.scalar_type() ? w.contiguous() : f32(w);
  Tensor y = fresh_like(xc);
  check(fla_causal_conv1d_update(ptr(xc), ptr(cache), ptr(wc), fptr(b32), ptr(y), B, D, W, arg_bool(p[4]), dt(xc), dt(wc),
                                 stream_of(xc)),
        "fla_causal_conv1d_update");
  return THPVariable_Wrap(y);
  END_HANDLE_TH_ERRORS
}

// norm_swish_gate(x, gate, weight | None, bias | None, eps, is_rms_norm)
PyObject* py_norm_gate(PyObject*, PyObject* const* p, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 6);
  const Tensor x = arg_tensor(p[0]), o = arg_tensor(p[1]), w = arg_tensor(p[2]), b = arg_tensor(p[3]);
  if (!rows_ok(x) || !o.defined() || !o.is_cuda() || o.sizes() != x.sizes() || o.scalar_type() != x.scalar_type()) return none();
  for (const Tensor* t : {&w, &b})
    if (t->defined() && (!t->is_cuda() || t->numel() != x.size(-1) || !t->is_floating_point())) return none();
  const double eps = arg_double(p[4]);
  const bool rms = arg_bool(p[5]);
  if (wants_grad({&x, &o, &w, &b})) return THPVariable_Wrap(NormGateNode::apply(x, o, maybe(w), maybe(b), eps, rms));
  at::AutoDispatchBelowADInplaceOrView guard;
  Tensor mean, rstd;
  return THPVariable_Wrap(NormGateNode::run(x.contiguous(), o.contiguous(), f32(w), f32(b), eps, rms, &mean, &rstd));
  END_HANDLE_TH_ERRORS
}

bool floating(const Tensor& x) { return is16(x) || x.scalar_type() == at::kFloat; }
void need_gpu(std::initializer_list<const Tensor*> ts) {
  const Tensor* first = nullptr;
  for (const Tensor* t : ts) {
    if (!t->defined()) continue;
    TORCH_CHECK(t->is_cuda(), "fla_amd: the HIP kernels need tensors on a GPU device; there is no CPU fallback");
    if (!first) first = t;
    TORCH_CHECK_VALUE(t->device() == first->device(), "fla_amd: operands on ", first->device(), " and ", t->device());
  }
}

// hgrn(x, g, lower_bound | None, h0 | None, want_ht, plan, segment, gates, inplace, offsets)
PyObject* py_hgrn(PyObject*, PyObject* const* p, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 10);
  const Tensor x = arg_tensor(p[0]), offsets = arg_tensor(p[9]);
  Tensor g = arg_tensor(p[1]), lb = arg_tensor(p[2]), h0 = arg_tensor(p[3]);
  HgrnArgs a{};
  a.want_ht = arg_bool(p[4]);
  a.plan = arg_plan(p[5]);
  a.gates = arg_bool(p[7]);
  const bool inplace = arg_bool(p[8]);
  TORCH_CHECK_VALUE(x.defined() && g.defined() && x.dim() == 3 && g.sizes() == x.sizes(),
                    "fla_amd hgrn: x and g are [B, T, D] of one shape");
  TORCH_CHECK_TYPE(floating(x) && g.is_floating_point() && (!lb.defined() || lb.is_floating_point()) &&
                       (!h0.defined() || h0.is_floating_point()),
                   "fla_amd hgrn: x in bf16, fp16 or fp32, the other operands in a floating type");
  TORCH_CHECK_VALUE(!lb.defined() || a.gates, "fla_amd hgrn: a lower bound goes with use_gate_in_kernel=True");
  a.B = x.size(0), a.T = x.size(1), a.D = x.size(2);
  a.N = a.plan ? a.plan->N : a.B;
  TORCH_CHECK_VALUE(!lb.defined() || lb.numel() == a.D, "fla_amd hgrn: lower_bound holds one value per channel, ", a.D);
  TORCH_CHECK_VALUE(!h0.defined() || (h0.dim() == 2 && h0.size(0) == a.N && h0.size(1) == a.D), "fla_amd hgrn: initial_state is [", a.N, ", ",
                    a.D, "]");
  TORCH_CHECK_VALUE(!a.plan || (a.plan->host.front() >= 0 && a.plan->host.back() <= a.T), "fla_amd hgrn: offsets leave the ", a.T, " rows");
  need_gpu({&x, &g, &lb, &h0});
  TORCH_CHECK_VALUE(!a.plan || a.plan->offsets.device() == x.device(), "fla_amd: offsets on ", a.plan->offsets.device(),
                    ", the operands on ", x.device());
  const bool grad = wants_grad({&x, &g, &lb, &h0});
  if (inplace) {
    TORCH_CHECK_VALUE(h0.defined() && a.want_ht && h0.scalar_type() == at::kFloat && h0.is_contiguous(),
                      "fla_amd hgrn: inplace_state needs a contiguous fp32 initial_state and output_final_state=True");
    TORCH_CHECK_VALUE(!grad, "fla_amd hgrn: inplace_state where a gradient is wanted");
  }
  c10::DeviceGuard on_device(x.device());
  if (g.scalar_type() != at::kFloat && g.scalar_type() != x.scalar_type()) g = g.to(at::kFloat);
  if (lb.defined()) lb = f32(lb).reshape({a.D});
  if (h0.defined()) h0 = f32(h0);
  if (x.numel() == 0 || a.N == 0) {   // no token: the states stay
    Tensor o = grad && x.numel() == 0 ? (lb.defined() ? x * g * lb : x * g).to(x.scalar_type())   // (empty, of their graph)
                                      : at::zeros(x.sizes(), x.options());
    Tensor ht;
    if (a.want_ht) ht = inplace ? h0 : h0.defined() ? h0.clone() : at::zeros({a.N, a.D}, x.options().dtype(at::kFloat));
    return pair(o, ht);
  }
  if (p[6] == Py_None) {
    a.segment = fla_hgrn_segment(a.B, a.B * a.T, a.T, a.D);
  } else {
    a.segment = PyLong_AsLongLong(p[6]);
    if (a.segment == -1 && PyErr_Occurred()) throw python_error();
  }
  if (grad) {
    auto out = HgrnNode::apply(x, g, maybe(lb), maybe(h0), maybe(offsets), a);
    return pair(out[0], a.want_ht ? out[1] : Tensor());
  }
  at::AutoDispatchBelowADInplaceOrView guard;
  Tensor ht;
  // A step writes each state where it read it; a scan's workgroups may still read the initial one when the final one is there
  const bool direct = inplace && a.T == 1 && !a.plan;
  if (direct) ht = h0;
  Tensor o = hgrn_forward(x, g, lb, h0, a, &ht, nullptr);
  if (inplace && !direct) ht = h0.copy_(ht);
  // written to: a node that saved the state before refuses its backward (inference tensors have no version)
  if (inplace && !h0.is_inference()) h0.unsafeGetTensorImpl()->bump_version();
  return pair(o, ht);
  END_HANDLE_TH_ERRORS
}

// norm(x, weight | None, bias | None, residual | None, eps, prenorm, residual_in_fp32, rows8, kind): rows8 FLA_ROWS_*, kind a NormKind
//   -> y, (y, residual_out), (q, scale) or ((q, scale), residual_out)
PyObject* py_norm(PyObject*, PyObject* const* p, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 9);
  Tensor x = arg_tensor(p[0]), w = arg_tensor(p[1]), b = arg_tensor(p[2]), res = arg_tensor(p[3]);
  NormArgs a{};
  a.eps = arg_double(p[4]);
  const bool prenorm = arg_bool(p[5]), in_f32 = arg_bool(p[6]);
  a.rows8 = arg_long(p[7]);
  a.kind = (NormKind)arg_long(p[8]);
  const char* who = a.kind == kLayer ? "fla_amd layer_norm" : a.kind == kRms ? "fla_amd rms_norm" : "fla_amd quantize_rows";
  TORCH_CHECK_VALUE(x.defined() && x.dim() >= 1 && x.size(-1) > 0, who, ": x is [..., N], N at least 1");
  TORCH_CHECK_TYPE(floating(x), who, ": x in bf16, fp16 or fp32, not ", x.scalar_type());
  const int64_t N = x.size(-1);
  for (const Tensor* t : {&w, &b}) {
    if (!t->defined()) continue;
    TORCH_CHECK_TYPE(t->is_floating_point(), who, ": weight and bias in a floating type");
    TORCH_CHECK_VALUE(t->numel() == N && t->dim() == 1, who, ": weight and bias hold ", N, " values");
  }
  if (res.defined()) {
    TORCH_CHECK_VALUE(res.sizes() == x.sizes(), who, ": the residual has x's shape");
    TORCH_CHECK_TYPE(res.scalar_type() == x.scalar_type() || res.scalar_type() == at::kFloat,
                     who, ": the residual is in x's type or in fp32");
  }
  const int64_t most = a.kind != kRowsOnly ? 16384 : 1 << 23;
  TORCH_CHECK_NOT_IMPLEMENTED(N <= most, who, ": rows of at most ", most, " elements, not ", N);
  need_gpu({&x, &w, &b, &res});
  const bool grad = wants_grad({&x, &w, &b, &res});
  TORCH_CHECK(!(grad && a.rows8), "fla_amd: rows in 8 bits have no gradient; call it under torch.no_grad()");
  c10::DeviceGuard on_device(x.device());
  if (grad && a.kind == kLayer) refuse_eager_leaves({&x, &w, &b, &res}, "layer_norm");
  // one type for both, x's or fp32
  auto fits = [&](const Tensor& t) { return !t.defined() || t.scalar_type() == x.scalar_type(); };
  if (!fits(w) || !fits(b)) w = f32(w), b = f32(b);
  if (w.defined()) w = w.contiguous();
  if (b.defined()) b = b.contiguous();
  if (res.defined()) a.kept_type = res.scalar_type();
  else if (in_f32 && prenorm && x.scalar_type() != at::kFloat) a.kept_type = at::kFloat;
  if (!prenorm && !grad) a.kept_type.reset();   // nobody asks for the sum
  Tensor y, scale, kept;
  if (grad) {
    auto out = NormNode::apply(x, maybe(w), maybe(b), maybe(res), a);
    y = out[0];
    if (out.size() > 1) kept = out[1];
  } else {
    at::AutoDispatchBelowADInplaceOrView guard;
    NormOut o = norm_forward(x.contiguous(), w, b, res.defined() ? res.contiguous() : res, a, false);
    y = o.y, scale = o.scale, kept = o.kept;
  }
  PyObject* first = a.rows8 ? pair(y, scale) : THPVariable_Wrap(y);
  if (!prenorm) return first;
  PyObject* t = PyTuple_New(2);
  if (!first || !t) throw python_error();
  PyTuple_SET_ITEM(t, 0, first);
  PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(kept.defined() ? kept : x));
  return t;
  END_HANDLE_TH_ERRORS
}

// The type of results, as a number of fla_dtype
at::ScalarType result_type(PyObject* o) {
  const long t = arg_long(o);
  return t == FLA_F32 ? at::kFloat : t == FLA_BF16 ? at::kBFloat16 : at::kHalf;
}
// Whether pairs of rows in 8 bits and their scales are of one type and of the shapes of a product; whether it is integers
bool int8_rows(const char* who, const Tensor& x, const Tensor& sx, std::initializer_list<const Tensor*> ws, std::initializer_list<const Tensor*> sws) {
  const bool known = x.defined() && (x.scalar_type() == at::kFloat8_e4m3fn || x.scalar_type() == at::kChar);
  bool one = known && sx.defined() && sx.scalar_type() == at::kFloat;
  for (const Tensor* w : ws) one = one && w->defined() && w->scalar_type() == x.scalar_type();
  for (const Tensor* s : sws) one = one && s->defined() && s->scalar_type() == at::kFloat;
  TORCH_CHECK_TYPE(one, who, ": x and weight are pairs of rows in torch.float8_e4m3fn, or in torch.int8, and their fp32 scales");
  const Tensor& first = **ws.begin();
  for (const Tensor* w : ws)
    TORCH_CHECK_VALUE(x.dim() >= 1 && w->dim() == 2 && w->size(1) == x.size(-1) && w->size(0) > 0 && w->sizes() == first.sizes(), who,
                      ": x is [..., K], weight [N, K]");
  TORCH_CHECK_VALUE(sx.sizes() == x.sizes().slice(0, x.dim() - 1), who, ": one scale for every row of x and of weight");
  for (const Tensor* s : sws)
    TORCH_CHECK_VALUE(s->dim() == 1 && s->size(0) == first.size(0), who, ": one scale for every row of x and of weight");
  const bool ints = x.scalar_type() == at::kChar;
  const int64_t K = x.size(-1), most = ints ? FLA_INT8_MAX_K : 1 << 23;
  TORCH_CHECK_NOT_IMPLEMENTED(K > 0 && K % 16 == 0 && K <= most, who, ": rows of a multiple of 16 elements, at most ", most, ", not ", K);
  return ints;
}

// quant_linear(x, x_scale, weight, weight_scale, bias | None, residual | None, activation, type)
PyObject* py_quant_linear(PyObject*, PyObject* const* p, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 8);
  Tensor x = arg_tensor(p[0]), sx = arg_tensor(p[1]), w = arg_tensor(p[2]), sw = arg_tensor(p[3]), bias = arg_tensor(p[4]),
         res = arg_tensor(p[5]);
  const long act = arg_long(p[6]);
  const auto type = result_type(p[7]);
  const bool ints = int8_rows("fla_amd quant_linear", x, sx, {&w}, {&sw});
  const int64_t K = x.size(-1), N = w.size(0);
  TORCH_CHECK_NOT_IMPLEMENTED(ints || type != at::kFloat, "fla_amd quant_linear: results of torch.float8_e4m3fn rows in bf16 or fp16");
  TORCH_CHECK_NOT_IMPLEMENTED(!ints || N <= 1 << 22, "fla_amd quant_linear: integer weights of at most 2^22 rows");
  if (bias.defined()) {
    TORCH_CHECK_VALUE(bias.dim() == 1 && bias.size(0) == N, "fla_amd quant_linear: bias holds ", N, " values");
    TORCH_CHECK_TYPE(bias.is_floating_point(), "fla_amd quant_linear: bias in a floating type");
  }
  auto shape = x.sizes().vec();
  shape.back() = N;
  if (res.defined()) {
    TORCH_CHECK_VALUE(res.sizes() == at::IntArrayRef(shape), "fla_amd quant_linear: residual is [..., N]");
    TORCH_CHECK_TYPE(res.scalar_type() == type || res.scalar_type() == at::kFloat,
                     "fla_amd quant_linear: the residual is in the output's type or in fp32");
  }
  need_gpu({&x, &sx, &w, &sw, &bias, &res});
  TORCH_CHECK(!wants_grad({&x, &sx, &w, &sw, &bias, &res}),
              "fla_amd: products of 8-bit rows have no gradient; call them under torch.no_grad()");
  c10::DeviceGuard on_device(x.device());
  at::AutoDispatchBelowADInplaceOrView guard;
  Tensor y = at::empty(shape, x.options().dtype(type));
  if (y.numel() == 0) return THPVariable_Wrap(y);
  x = whole_rows(x), w = whole_rows(w), sx = sx.contiguous(), sw = sw.contiguous();
  if (bias.defined()) bias = whole_bias(bias.scalar_type() == type ? bias : f32(bias));
  if (res.defined()) res = res.contiguous();
  const int64_t M = x.numel() / K;
  const int splits = ints ? fla_int8_linear_splits(M, N, K, dt(y)) : fla_quant_linear_splits(M, N, K);
  const Tensor sums = splits > 1 ? fresh({splits, M, N}, x, ints ? at::kInt : at::kFloat) : Tensor();
  const int bt = bias.defined() ? dt(bias) : FLA_F32, rt = res.defined() ? dt(res) : FLA_F32;
  if (ints)
    check(fla_int8_linear(ptr(x), fptr(sx), ptr(w), fptr(sw), ptr(bias), bt, ptr(res), rt, ptr(y), M, N, K, (int)act, dt(y), ptr(sums), stream_of(x)),
          "fla_int8_linear");
  else
    check(fla_quant_linear(ptr(x), fptr(sx), ptr(w), fptr(sw), ptr(bias), bt, ptr(res), rt, ptr(y), M, N, K, (int)act, dt(y), fptr(sums), stream_of(x)),
          "fla_quant_linear");
  return THPVariable_Wrap(y);
  END_HANDLE_TH_ERRORS
}

// quant_gated_linear(x, x_scale, gate_weight, gate_scale, up_weight, up_scale, gate_bias | None, up_bias | None, activation, type)
PyObject* py_quant_gated_linear(PyObject*, PyObject* const* p, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 10);
  Tensor x = arg_tensor(p[0]), sx = arg_tensor(p[1]), wg = arg_tensor(p[2]), sg = arg_tensor(p[3]), wu = arg_tensor(p[4]), su = arg_tensor(p[5]),
         bg = arg_tensor(p[6]), bu = arg_tensor(p[7]);
  const long act = arg_long(p[8]);
  const auto type = result_type(p[9]);
  const bool ints = int8_rows("fla_amd quant_gated_linear", x, sx, {&wg, &wu}, {&sg, &su});
  TORCH_CHECK_NOT_IMPLEMENTED(ints, "fla_amd quant_gated_linear: rows in torch.int8");
  const int64_t K = x.size(-1), F = wg.size(0), M = x.numel() / K;
  TORCH_CHECK_NOT_IMPLEMENTED(F <= 1 << 22, "fla_amd quant_gated_linear: weights of at most 2^22 rows");
  for (const Tensor* t : {&bg, &bu}) {
    if (!t->defined()) continue;
    TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == F, "fla_amd quant_gated_linear: biases hold ", F, " values");
    TORCH_CHECK_TYPE(t->is_floating_point(), "fla_amd quant_gated_linear: biases in a floating type");
  }
  need_gpu({&x, &sx, &wg, &sg, &wu, &su, &bg, &bu});
  TORCH_CHECK(!wants_grad({&sx, &sg, &su, &bg, &bu}), "fla_amd: products of 8-bit rows have no gradient; call them under torch.no_grad()");
  c10::DeviceGuard on_device(x.device());
  at::AutoDispatchBelowADInplaceOrView guard;
  auto shape = x.sizes().vec();
  shape.back() = F;
  Tensor h = at::empty(shape, x.options().dtype(type));
  if (h.numel() == 0) return THPVariable_Wrap(h);
  x = whole_rows(x), wg = whole_rows(wg), wu = whole_rows(wu), sx = sx.contiguous(), sg = sg.contiguous(), su = su.contiguous();
  auto fits = [&](const Tensor& t) { return !t.defined() || t.scalar_type() == type; };
  const bool same = fits(bg) && fits(bu);
  if (!same) bg = f32(bg), bu = f32(bu);
  bg = whole_bias(bg), bu = whole_bias(bu);
  const int splits = fla_gated_linear_splits(M, F, K, 1);
  const Tensor sums = splits > 1 ? fresh({splits, M, 2, F}, x, at::kInt) : Tensor();
  check(fla_int8_gated_linear_fwd(ptr(x), fptr(sx), ptr(wg), fptr(sg), ptr(wu), fptr(su), ptr(bg), ptr(bu), same ? dt(h) : FLA_F32, ptr(h), M, F, K,
                                  (int)act, dt(h), ptr(sums), stream_of(x)),
        "fla_int8_gated_linear_fwd");
  return THPVariable_Wrap(h);
  END_HANDLE_TH_ERRORS
}

// gated_linear(x, gate_weight, up_weight, gate_bias | None, up_bias | None, activation)
PyObject* py_gated_linear(PyObject*, PyObject* const* p, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 6);
  const Tensor x = arg_tensor(p[0]), wg = arg_tensor(p[1]), wu = arg_tensor(p[2]), bg = arg_tensor(p[3]), bu = arg_tensor(p[4]);
  const long act = arg_long(p[5]);
  TORCH_CHECK_VALUE(x.defined() && wg.defined() && wu.defined() && x.dim() >= 1 && wg.dim() == 2 && wg.sizes() == wu.sizes() &&
                        wg.size(1) == x.size(-1) && wg.size(0) > 0 && wg.size(1) > 0,
                    "fla_amd gated_linear: x is [..., K], both weights [F, K], neither empty");
  TORCH_CHECK_TYPE(is16(x) && wg.scalar_type() == x.scalar_type() && wu.scalar_type() == x.scalar_type(),
                   "fla_amd gated_linear: x and both weights in bf16 or in fp16, not ", x.scalar_type(), ", ", wg.scalar_type(), " and ",
                   wu.scalar_type());
  const int64_t F = wg.size(0), K = wg.size(1);
  for (const Tensor* t : {&bg, &bu}) {
    if (!t->defined()) continue;
    TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == F, "fla_amd gated_linear: biases hold ", F, " values");
    TORCH_CHECK_TYPE(t->is_floating_point(), "fla_amd gated_linear: biases in a floating type");
  }
  TORCH_CHECK_NOT_IMPLEMENTED(F <= 1 << 22 && K <= 1 << 22 && x.numel() / K <= 0x7fffffff,
                              "fla_amd gated_linear: weights of at most 2^22 rows and columns, x of less than 2^31 rows");
  need_gpu({&x, &wg, &wu, &bg, &bu});
  c10::DeviceGuard on_device(x.device());
  const bool grad = wants_grad({&x, &wg, &wu, &bg, &bu});
  if (grad) refuse_eager_leaves({&x, &wg, &wu, &bg, &bu}, "gated_linear");
  if (grad) return THPVariable_Wrap(GatedNode::apply(x, wg, wu, maybe(bg), maybe(bu), act));
  at::AutoDispatchBelowADInplaceOrView guard;
  return THPVariable_Wrap(GatedNode::run(x, wg, wu, bg, bu, act, nullptr));
  END_HANDLE_TH_ERRORS
}

#define ENTRY(name, fn) {name, (PyCFunction)(void (*)(void))fn, METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {
    ENTRY("plan", py_plan),
    ENTRY("chunk_gla", py_chunk_gla),
    ENTRY("chunk_simple_gla", py_chunk_simple_gla),
    ENTRY("chunk_gdr", py_chunk_gdr),
    ENTRY("recurrent_gla", py_recurrent_gla),
    ENTRY("recurrent_gdr", py_recurrent_gdr),
    ENTRY("l2_norm", py_l2_norm),
    ENTRY("causal_conv1d", py_conv),
    ENTRY("causal_conv1d_update", py_conv_update<false>),
    ENTRY("short_conv_step", py_conv_update<true>),
    ENTRY("norm_swish_gate", py_norm_gate),
    ENTRY("hgrn", py_hgrn),
    ENTRY("norm", py_norm),
    ENTRY("quant_linear", py_quant_linear),
    ENTRY("gated_linear", py_gated_linear),
    ENTRY("quant_gated_linear", py_quant_gated_linear),
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_fla_host", nullptr, -1, kMethods};

}  // namespace

PyMODINIT_FUNC PyInit__fla_host(void) {
  PyObject* m = PyModule_Create(&kModule);
  if (m) PyModule_AddIntConstant(m, "ABI_VERSION", FLA_ABI_VERSION);
  return m;
}
