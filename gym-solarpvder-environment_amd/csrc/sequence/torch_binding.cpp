// torch_binding.cpp -- the sequence operators as torch sees them (gym_PVDER_amd/agents/sequence_ops.py documents them): checks of the
// arguments, outputs and workspaces from torch's allocator, the current stream, and the autograd nodes.  The mathematics is behind the
// C ABI of include/pvder_sequence.h.  In C++ because a call from Python with ctypes costs more than the kernels of a small batch: a step
// of one env took 19 us from call to call, 5 here; a training pass over 64 windows of 160 steps 160 us, 60 here, which is its kernels' time.
#include <torch/extension.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <cmath>
#include <initializer_list>
#include <optional>

#include "pvder_sequence.h"

namespace {

using at::Tensor;
using std::optional;
typedef const optional<Tensor> &Maybe;

// what is refused raises ValueError or TypeError, as everywhere in the package
#define NEED(cond, ...) TORCH_CHECK_VALUE(cond, __VA_ARGS__)
#define NEED_TYPE(cond, ...) TORCH_CHECK_TYPE(cond, __VA_ARGS__)

void checked(int64_t rc, const char *what) {
    if (rc >= 0) return;
    TORCH_CHECK_VALUE(rc != -10001, what, ": invalid argument (PVDER_EINVAL)");
    TORCH_CHECK(false, what, ": HIP error ", -rc);
}

void *stream_of(const Tensor &t) { return (void *)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream(); }

bool has(Maybe t) { return t.has_value() && t->defined(); }
const void *ptr(Maybe t) { return has(t) ? t->data_ptr() : nullptr; }

int dtype_of(const Tensor &t) { return t.scalar_type() == at::kFloat ? PVDER_SEQ_F32 : PVDER_SEQ_BF16; }
bool dtype_ok(const Tensor &t) { return t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16; }

void same_device(const Tensor &q, Maybe t, const char *name) {
    if (has(t)) NEED(t->device() == q.device(), name, " is on ", t->device(), ", the call on ", q.device());
}
void on_gpu(const Tensor &t, const char *name) {
    NEED(t.is_cuda(), name, " is on ", t.device(), ": the kernels need a GPU, there is no CPU path");
}
// The kernels take memory, past torch's dispatcher: what it would do to a call besides computing it does not happen.  A tangent would be
// lost, which torch reads as a derivative of zero; a trace would record outputs that nothing writes.  Both are refused, and so are
// tensors that stand for others (torch.func, tensor subclasses).  A null is an argument that was not given.
void plain(std::initializer_list<const Tensor *> all) {
    NEED(!torch::jit::tracer::isTracing(), "the sequence operators cannot be traced (torch.jit.trace)");
    typedef c10::impl::TorchDispatchModeKey Mode;
    for (const Mode m : {Mode::FAKE, Mode::PROXY, Mode::FUNCTIONAL})
        NEED(!c10::impl::TorchDispatchModeTLS::get_mode(m).has_value(), "the sequence operators cannot be traced (make_fx, fake tensors)");
    for (const Tensor *t : all) {
        if (!t || !t->defined()) continue;
        NEED(t->has_storage() && !t->key_set().has(c10::DispatchKey::Python) && !t->key_set().has(c10::DispatchKey::Functionalize),
             "the sequence operators take plain tensors, not wrappers of them (torch.func, tensor subclasses with __torch_dispatch__)");
        NEED(!t->_fw_grad(0).defined(), "the sequence operators have no forward-mode gradient: an argument has a tangent");
    }
}
const Tensor *given(Maybe t) { return has(t) ? &*t : nullptr; }

bool wants_grad(const Tensor &t) { return t.requires_grad(); }
bool wants_grad(Maybe t) { return has(t) && t->requires_grad(); }

// unit stride in the last dimension (a copy only where it has another)
Tensor rows(const Tensor &t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }
// and tokens that lie behind each other (not on each other, as in an expanded tensor) and near enough for 32-bit offsets within a chunk
Tensor tokens(const Tensor &t) {
    const Tensor r = rows(t);
    const int64_t st = r.stride(1);
    return r.size(1) <= 1 || (st >= r.size(3) && st * (int64_t)r.element_size() <= PVDER_SEQ_MAX_TOKEN_STRIDE) ? r : r.contiguous();
}

struct Heads { int64_t H, DK, DV; };

Heads check_qkv(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &log_decay, int64_t dims, const char *form) {
    same_device(q, k, "k");
    same_device(q, v, "v");
    same_device(q, log_decay, "log_decay");
    NEED_TYPE(dtype_ok(q) && k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
              "q, k and v must be float32 or bfloat16, all three alike: got ", q.scalar_type(), ", ", k.scalar_type(), ", ", v.scalar_type());
    NEED(q.dim() == dims && k.dim() == dims && v.dim() == dims, "q, k and v must be ", form);
    NEED(k.sizes() == q.sizes(), "q and k differ in shape: ", q.sizes(), ", ", k.sizes());
    NEED(v.sizes().slice(0, dims - 1) == q.sizes().slice(0, dims - 1), "v must be ", form, " beside q: got ", v.sizes(), ", ", q.sizes());
    const Heads d = {q.size(-2), q.size(-1), v.size(-1)};
    NEED(d.H >= 1 && d.DK >= 1 && d.DK <= PVDER_SEQ_MAX_HEAD && d.DV >= 1 && d.DV <= PVDER_SEQ_MAX_HEAD,
         "there must be a head, and heads must be 1 .. ", (int)PVDER_SEQ_MAX_HEAD, " wide: got ", d.H, " heads of ", d.DK, " and ", d.DV);
    for (int64_t i = 0; i + 2 < dims; ++i) NEED(q.size(i) < (1ll << 31), "too many rows");
    NEED(d.H < (1ll << 31), "too many heads");
    NEED_TYPE(log_decay.scalar_type() == at::kFloat, "log_decay must be float32");
    NEED(log_decay.dim() == 1 && log_decay.size(0) == d.H && log_decay.is_contiguous(), "log_decay must be a contiguous [", d.H, "], one for each head");
    NEED(!(log_decay.requires_grad() && at::GradMode::is_enabled()),
         "log_decay is a constant of the heads: the kernels give it no gradient; detach it");
    return d;
}

float scale_of(optional<double> scale, int64_t dk) {
    if (!scale) return (float)(1.0 / std::sqrt((double)dk));
    NEED(std::isfinite(*scale) && std::isfinite((float)*scale), "scale must be a finite number");
    return (float)*scale;
}

void check_flags(Maybe t, at::IntArrayRef shape) {
    if (!has(t)) return;
    NEED_TYPE(t->scalar_type() == at::kBool || t->scalar_type() == at::kByte, "starts must be bool or uint8");
    NEED(t->sizes() == shape, "starts must be ", shape, ": got ", t->sizes());
}

// ---- decay attention over windows -------------------------------------------------------------------------------------------
// a state whose matrices are dense (rows or columns first)
Tensor dense(const Tensor &s) {
    const int64_t k = s.size(2), v = s.size(3);
    return (s.stride(3) == 1 && s.stride(2) == v) || (s.stride(2) == 1 && s.stride(3) == k) ? s : s.contiguous();
}
struct State { int64_t b, h, k, v; };
State state_strides(Maybe t, const Heads &d) {
    if (has(t)) return {t->stride(0), t->stride(1), t->stride(2), t->stride(3)};
    return {d.H * d.DK * d.DV, d.DK * d.DV, d.DV, 1};
}

pvder_seq_scan scan_of(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &o, const void *s_in, void *s_out, const State &s, float a_read,
                       float a_write, float a_intra, bool reverse) {
    pvder_seq_scan c = {};
    c.q = q.data_ptr(); c.k = k.data_ptr(); c.v = v.data_ptr(); c.o = o.data_ptr();
    const bool many = q.size(1) > 1;                       // (the stride of a single token says nothing: a row's length)
    c.q_b = q.stride(0); c.q_t = many ? q.stride(1) : q.size(3); c.q_h = q.stride(2);
    c.k_b = k.stride(0); c.k_t = many ? k.stride(1) : k.size(3); c.k_h = k.stride(2);
    c.v_b = v.stride(0); c.v_t = many ? v.stride(1) : v.size(3); c.v_h = v.stride(2);
    c.o_b = o.stride(0); c.o_t = many ? o.stride(1) : o.size(3); c.o_h = o.stride(2);
    c.s_in = (const float *)s_in; c.s_out = (float *)s_out;
    c.s_b = s.b; c.s_h = s.h; c.s_k = s.k; c.s_v = s.v;
    c.a_read = a_read; c.a_write = a_write; c.a_intra = a_intra;
    c.dk = (int32_t)q.size(3); c.dv = (int32_t)v.size(3); c.reverse = reverse;
    return c;
}

// `a.scan` and `a.n_scans` are set (and a.segments, where they have states of an earlier run); the rest comes from q's sizes and the options.
// Returns the workspace, undefined where T is one piece.
Tensor run_scans(pvder_seq_attn &a, const Tensor &q, const Tensor &log_decay, Maybe starts, Maybe lengths) {
    a.log_decay = log_decay.data_ptr<float>();
    a.starts = (const uint8_t *)ptr(starts);
    a.starts_b = has(starts) ? starts->stride(0) : 0;
    a.starts_t = has(starts) ? starts->stride(1) : 0;
    a.lengths = (const int32_t *)ptr(lengths);
    a.B = (int32_t)q.size(0); a.T = (int32_t)q.size(1); a.H = (int32_t)q.size(2);
    a.dtype = dtype_of(q);
    a.workspace = nullptr;
    const int64_t floats = pvder_seq_attn_plan(&a);
    checked(floats, "pvder_seq_attn_plan");
    Tensor work;
    if (floats > 0) {
        work = at::empty({floats}, log_decay.options());
        a.workspace = work.data_ptr<float>();
    }
    checked(pvder_seq_attn_run(&a, stream_of(q)), "pvder_seq_attn_run");
    return work;
}

// The states of the pieces of T as the forward pass left them, for the backward pass (at most 2048 strips of 16 KB)
struct Kept {
    Tensor states;
    int32_t segments = 1;
};

std::tuple<Tensor, Tensor> attention_forward(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &log_decay, Maybe initial, Maybe starts,
                                             Maybe lengths, float scale, bool want_state, Kept *kept = nullptr) {
    const Heads d = {q.size(2), q.size(3), v.size(3)};
    const c10::DeviceGuard guard(q.device());
    Tensor out = at::empty({q.size(0), q.size(1), d.H, d.DV}, q.options()), final;
    optional<Tensor> in = initial;
    if (want_state) {
        final = at::empty({q.size(0), d.H, d.DK, d.DV}, log_decay.options());
        if (has(in) && !in->is_contiguous()) in = in->contiguous();      // (one set of strides for the state in and out)
    }
    pvder_seq_attn a;
    a.n_scans = 1;
    a.scan[0] = scan_of(q, k, v, out, ptr(in), want_state ? final.data_ptr() : nullptr, state_strides(in, d), scale, 1.f, scale, false);
    const Tensor work = run_scans(a, q, log_decay, starts, lengths);
    if (kept && work.defined()) *kept = {work, a.segments};
    return {out, final};
}

// A leaf's gradient accumulator belongs to the stream on which its first graph was recorded, and lives as long as a graph does.  A
// backward pass that is captured while such a graph of another stream lives would have to wait for that stream, which a capture cannot:
// torch's engine throws in a thread of its own, and the process ends.  So the forward pass is refused, for arguments that are leaves and
// for views of leaves.  (A leaf behind other operations meets them first: torch's own captures have the same limit.)
void capturable(const Tensor &arg, const char *name) {
    if (!arg.defined() || !arg.requires_grad()) return;
    Tensor t = arg;
    if (arg.grad_fn() && arg.is_view()) t = arg._base();
    if (!t.requires_grad() || t.grad_fn()) return;
    const auto acc = torch::autograd::impl::try_get_grad_accumulator(t);
    if (!acc) return;
    const auto own = acc->stream();
    const c10::Stream now = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).unwrap();
    TORCH_CHECK(!own || *own == now, name, " is a leaf, or a view of one, of a graph that lives on another stream: its backward pass cannot be captured. Delete what "
                "holds that graph (its outputs, its losses) before the capture.");
}
bool capturing() { return c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None; }

void once() {
    TORCH_CHECK(!at::GradMode::is_enabled(), "the sequence operators are differentiable once: create_graph=True is not supported");
}

struct DecayAttention : torch::autograd::Function<DecayAttention> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v,
                                                  const Tensor &log_decay, Maybe initial, Maybe starts, Maybe lengths, double scale, bool want_state) {
        ctx->set_materialize_grads(false);
        const Tensor none;
        Kept kept;
        auto [out, final] = attention_forward(q, k, v, log_decay, initial, starts, lengths, (float)scale, want_state, q.requires_grad() ? &kept : nullptr);
        ctx->save_for_backward({q, k, v, log_decay, has(initial) ? *initial : none, has(starts) ? *starts : none, has(lengths) ? *lengths : none, kept.states});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["segments"] = (int64_t)kept.segments;
        if (want_state) return {out, final};
        return {out};
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
        once();
        torch::autograd::variable_list res(9);
        const bool has_state = grads.size() > 1;
        Tensor dout = grads[0], dfinal = has_state ? grads[1] : Tensor();
        if (!dout.defined() && !dfinal.defined()) return res;
        const auto saved = ctx->get_saved_variables();
        const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &log_decay = saved[3];
        const optional<Tensor> initial = saved[4], starts = saved[5], lengths = saved[6];
        const float scale = (float)ctx->saved_data["scale"].toDouble();
        const Heads d = {q.size(2), q.size(3), v.size(3)};
        const c10::DeviceGuard guard(q.device());
        dout = dout.defined() ? tokens(dout) : at::zeros({q.size(0), q.size(1), d.H, d.DV}, q.options());
        if (dfinal.defined()) dfinal = dfinal.contiguous();
        const void *ds_in = dfinal.defined() ? dfinal.data_ptr() : nullptr;
        const State plain = state_strides(optional<Tensor>(), d);
        pvder_seq_attn a;
        a.n_scans = 0;
        a.segments = (int32_t)ctx->saved_data["segments"].toInt();
        const bool need_v = ctx->needs_input_grad(2), need_s = has(initial) && ctx->needs_input_grad(4);
        if (need_v || need_s) {
            const Tensor dv = at::empty({q.size(0), q.size(1), d.H, d.DV}, q.options());
            if (need_s) res[4] = at::empty({q.size(0), d.H, d.DK, d.DV}, log_decay.options());
            a.scan[a.n_scans++] = scan_of(k, q, dout, dv, ds_in, need_s ? res[4].data_ptr() : nullptr, plain, 1.f, scale, scale, true);
            res[2] = dv;
        }
        if (ctx->needs_input_grad(1)) {
            res[1] = at::empty({q.size(0), q.size(1), d.H, d.DK}, q.options());
            a.scan[a.n_scans] = scan_of(v, dout, q, res[1], ds_in, nullptr, {plain.b, plain.h, plain.v, plain.k}, 1.f, scale, scale, true);
            a.scan[a.n_scans].transpose_of = a.n_scans;    // (dv's, if that is there)
            ++a.n_scans;
        }
        if (ctx->needs_input_grad(0)) {
            // dq_t = scale S_t do_t: the attention of do over (v, k), its state the transpose of S
            const State s = state_strides(initial, d);
            res[0] = at::empty({q.size(0), q.size(1), d.H, d.DK}, q.options());
            a.scan[a.n_scans] = scan_of(dout, v, k, res[0], ptr(initial), nullptr, {s.b, s.h, s.v, s.k}, scale, 1.f, scale, false);
            if (saved[7].defined()) a.scan[a.n_scans].kept = saved[7].data_ptr<float>();
            ++a.n_scans;
        }
        if (a.n_scans) run_scans(a, q, log_decay, starts, lengths);
        if (!need_v) res[2] = Tensor();
        return res;
    }
};

py::object decay_attention(const Tensor &q_, const Tensor &k_, const Tensor &v_, const Tensor &log_decay, optional<double> scale_, Maybe initial_,
                           Maybe starts, Maybe lengths, bool want_state) {
    plain({&q_, &k_, &v_, &log_decay, given(initial_), given(starts), given(lengths)});
    const Heads d = check_qkv(q_, k_, v_, log_decay, 4, "[B, T, H, D]");
    const int64_t B = q_.size(0), T = q_.size(1);
    same_device(q_, initial_, "initial_state");
    same_device(q_, starts, "starts");
    same_device(q_, lengths, "lengths");
    if (has(initial_)) {
        NEED_TYPE(initial_->scalar_type() == at::kFloat, "initial_state must be float32");
        const at::IntArrayRef is = initial_->sizes();
        NEED(is.size() == 4 && is[0] == B && is[1] == d.H && is[2] == d.DK && is[3] == d.DV, "initial_state must be [", B, ", ", d.H, ", ", d.DK, ", ", d.DV, "]: got ", is);
    }
    check_flags(starts, {B, T});
    if (has(lengths)) {
        NEED_TYPE(lengths->scalar_type() == at::kInt, "lengths must be int32");
        NEED(lengths->dim() == 1 && lengths->size(0) == B && lengths->is_contiguous(), "lengths must be a contiguous [", B, "]");
    }
    const float scale = scale_of(scale_, d.DK);
    on_gpu(q_, "q");
    const c10::DeviceGuard guard(q_.device());
    if (at::GradMode::is_enabled() && capturing()) {       // (before anything is made of the arguments)
        capturable(q_, "q");
        capturable(k_, "k");
        capturable(v_, "v");
        if (has(initial_)) capturable(*initial_, "initial_state");
    }
    const int64_t least = 16 / (int64_t)q_.element_size();
    if (d.DK < least || d.DV < least) {
        // heads of less than 16 bytes: with zeros behind them, and without them again
        const int64_t k0 = d.DK < least ? least - d.DK : 0, v0 = d.DV < least ? least - d.DV : 0;
        optional<Tensor> s0;
        if (has(initial_)) s0 = at::constant_pad_nd(*initial_, {0, v0, 0, k0});
        const py::object r = decay_attention(at::constant_pad_nd(q_, {0, k0}), at::constant_pad_nd(k_, {0, k0}), at::constant_pad_nd(v_, {0, v0}), log_decay,
                                             (double)scale, s0, starts, lengths, want_state);
        auto cut = [&](const py::handle &o) { return o.cast<Tensor>().narrow(-1, 0, d.DV); };
        if (!want_state) return py::cast(cut(r));
        const py::tuple both = r.cast<py::tuple>();
        return py::make_tuple(cut(both[0]), cut(both[1]).narrow(2, 0, d.DK).contiguous());      // (as the step form wants it)
    }
    const Tensor q = tokens(q_), k = tokens(k_), v = tokens(v_);
    const optional<Tensor> initial = has(initial_) ? optional<Tensor>(dense(*initial_)) : optional<Tensor>();
    Tensor out, final;
    if (at::GradMode::is_enabled() && (wants_grad(q) || wants_grad(k) || wants_grad(v) || wants_grad(initial))) {
        const auto r = DecayAttention::apply(q, k, v, log_decay, initial, starts, lengths, (double)scale, want_state);
        out = r[0];
        if (want_state) final = r[1];
    } else {
        std::tie(out, final) = attention_forward(q, k, v, log_decay, initial, starts, lengths, scale, want_state);
    }
    if (want_state) return py::make_tuple(out, final);
    return py::cast(out);
}

Tensor decay_attention_step(const Tensor &q_, const Tensor &k_, const Tensor &v_, const Tensor &log_decay, const Tensor &state, optional<double> scale_,
                            Maybe starts) {
    plain({&q_, &k_, &v_, &log_decay, &state, given(starts)});
    const Heads d = check_qkv(q_, k_, v_, log_decay, 3, "[N, H, D]");
    const int64_t N = q_.size(0);
    same_device(q_, state, "state");
    same_device(q_, starts, "starts");
    NEED_TYPE(state.scalar_type() == at::kFloat, "state must be float32");
    const at::IntArrayRef ss = state.sizes();
    NEED(ss.size() == 4 && ss[0] == N && ss[1] == d.H && ss[2] == d.DK && ss[3] == d.DV && state.is_contiguous(), "state must be a contiguous [", N, ", ", d.H,
         ", ", d.DK, ", ", d.DV, "]: got ", ss);
    check_flags(starts, {N});
    NEED(!(at::GradMode::is_enabled() && (wants_grad(q_) || wants_grad(k_) || wants_grad(v_) || wants_grad(state))),
         "the step form has no gradient: call it under torch.no_grad(), or train on windows with decay_attention");
    const float scale = scale_of(scale_, d.DK);
    on_gpu(q_, "q");
    const c10::DeviceGuard guard(q_.device());
    const Tensor q = rows(q_), k = rows(k_), v = rows(v_);
    Tensor out = at::empty({N, d.H, d.DV}, q.options());
    pvder_seq_step a;
    a.q = q.data_ptr(); a.k = k.data_ptr(); a.v = v.data_ptr(); a.o = out.data_ptr();
    a.q_n = q.stride(0); a.q_h = q.stride(1); a.k_n = k.stride(0); a.k_h = k.stride(1); a.v_n = v.stride(0); a.v_h = v.stride(1);
    a.o_n = out.stride(0); a.o_h = out.stride(1);
    a.state = state.data_ptr<float>();
    a.log_decay = log_decay.data_ptr<float>();
    a.starts = (const uint8_t *)ptr(starts);
    a.starts_n = has(starts) ? starts->stride(0) : 0;
    a.N = (int32_t)N; a.H = (int32_t)d.H; a.dk = (int32_t)d.DK; a.dv = (int32_t)d.DV; a.dtype = dtype_of(q);
    a.scale = scale;
    checked(pvder_seq_step_run(&a, stream_of(q)), "pvder_seq_step_run");
    if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();     // a graph that saved it has to see the change
    return out;
}

// ---- gated residual norm ----------------------------------------------------------------------------------------------------
// [rows, width] with dense rows (a view wherever the strides allow one)
Tensor two(const Tensor &t, int64_t width) { return rows(t.dim() == 2 ? t : t.reshape({-1, width})); }
optional<Tensor> two(Maybe t, int64_t width) { return has(t) ? optional<Tensor>(two(*t, width)) : optional<Tensor>(); }

pvder_seq_norm norm_arg(const Tensor &h, const Tensor &y, Maybe gate, const Tensor &post, const Tensor &pre, Maybe scale, double eps) {
    pvder_seq_norm a = {};
    a.h = h.data_ptr(); a.y = y.data_ptr(); a.gate = ptr(gate);
    a.h_r = h.stride(0); a.y_r = y.stride(0); a.gate_r = has(gate) ? gate->stride(0) : 0;
    a.post = post.data_ptr<float>(); a.pre = pre.data_ptr<float>(); a.scale = (const float *)ptr(scale);
    a.rows = h.size(0); a.width = (int32_t)h.size(1); a.dtype = dtype_of(h); a.eps = (float)eps;
    return a;
}

std::tuple<Tensor, Tensor, Tensor> norm_forward(const Tensor &h, const Tensor &y, const Tensor &post, const Tensor &pre, Maybe gate, Maybe scale, double eps,
                                                bool want_stats) {
    const int64_t D = h.size(-1);
    const c10::DeviceGuard guard(h.device());
    const Tensor h2 = two(h, D), y2 = two(y, D);
    const optional<Tensor> g2 = two(gate, D);
    Tensor h_out = at::empty(h.sizes(), h.options()), x_out = at::empty(h.sizes(), h.options()), stats;
    pvder_seq_norm a = norm_arg(h2, y2, g2, post, pre, scale, eps);
    a.h_out = h_out.data_ptr(); a.x_out = x_out.data_ptr();
    if (want_stats) {
        stats = at::empty({h2.size(0), 2}, post.options());
        a.stats = stats.data_ptr<float>();
    }
    checked(pvder_seq_norm_forward(&a, stream_of(h)), "pvder_seq_norm_forward");
    return {h_out, x_out, stats};
}

struct GatedResidualNorm : torch::autograd::Function<GatedResidualNorm> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext *ctx, const Tensor &h, const Tensor &y, const Tensor &post,
                                                  const Tensor &pre, Maybe gate, Maybe scale, double eps) {
        ctx->set_materialize_grads(false);
        auto [h_out, x_out, stats] = norm_forward(h, y, post, pre, gate, scale, eps, true);
        const Tensor none;
        ctx->save_for_backward({h, y, post, pre, has(gate) ? *gate : none, has(scale) ? *scale : none, stats});
        ctx->saved_data["eps"] = eps;
        return {h_out, x_out};
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
        once();
        torch::autograd::variable_list res(7);
        if (!grads[0].defined() && !grads[1].defined()) return res;
        const auto saved = ctx->get_saved_variables();
        const Tensor &h = saved[0], &y = saved[1], &post = saved[2], &pre = saved[3], &stats = saved[6];
        const optional<Tensor> gate = saved[4], scale = saved[5];
        const int64_t D = h.size(-1);
        const c10::DeviceGuard guard(h.device());
        const Tensor h2 = two(h, D), y2 = two(y, D);
        const optional<Tensor> g2 = two(gate, D), dh = two(optional<Tensor>(grads[0]), D), dx = two(optional<Tensor>(grads[1]), D);
        const int at_scale = has(gate) ? 5 : 4;            // (needs_input_grad counts the tensors that were given)
        const bool need_scale = has(scale) && ctx->needs_input_grad(at_scale);
        auto like = [&]() { return at::empty(h.sizes(), h.options()); };
        Tensor dh_out = like(), dy_out = like(), dgate, dparam, work;
        pvder_seq_norm a = norm_arg(h2, y2, g2, post, pre, scale, ctx->saved_data["eps"].toDouble());
        a.stats = stats.data_ptr<float>();
        a.dh = ptr(dh); a.dx = ptr(dx);
        a.dh_r = has(dh) ? dh->stride(0) : 0; a.dx_r = has(dx) ? dx->stride(0) : 0;
        a.dh_out = dh_out.data_ptr(); a.dy_out = dy_out.data_ptr();
        if (has(gate)) { dgate = like(); a.dgate_out = dgate.data_ptr(); }
        if (ctx->needs_input_grad(2) || ctx->needs_input_grad(3) || need_scale) {
            dparam = h.numel() ? at::empty({3, D}, post.options()) : at::zeros({3, D}, post.options());
            a.dparam = dparam.data_ptr<float>();
            const int64_t floats = pvder_seq_norm_workspace(&a);
            checked(floats, "pvder_seq_norm_workspace");
            if (floats > 0) {
                work = at::empty({floats}, post.options());
                a.workspace = work.data_ptr<float>();
            }
        }
        checked(pvder_seq_norm_backward(&a, stream_of(h)), "pvder_seq_norm_backward");
        if (ctx->needs_input_grad(0)) res[0] = dh_out;
        if (ctx->needs_input_grad(1)) res[1] = dy_out;
        if (ctx->needs_input_grad(2)) res[2] = dparam[0];
        if (ctx->needs_input_grad(3)) res[3] = dparam[1];
        if (has(gate) && ctx->needs_input_grad(4)) res[4] = dgate;
        if (need_scale) res[5] = dparam[2];
        return res;
    }
};

std::tuple<Tensor, Tensor> gated_residual_norm(const Tensor &h, const Tensor &y, const Tensor &post, const Tensor &pre, Maybe gate, Maybe scale, double eps) {
    plain({&h, &y, &post, &pre, given(gate), given(scale)});
    same_device(h, y, "y");
    same_device(h, post, "post_weight");
    same_device(h, pre, "pre_weight");
    same_device(h, gate, "gate");
    same_device(h, scale, "scale");
    NEED_TYPE(dtype_ok(h) && y.scalar_type() == h.scalar_type() && (!has(gate) || gate->scalar_type() == h.scalar_type()),
              "residual, y and gate must be float32 or bfloat16, all alike");
    NEED(h.dim() >= 1 && h.size(-1) >= 1 && h.size(-1) <= PVDER_SEQ_MAX_WIDTH, "the last dimension must be 1 .. ", (int)PVDER_SEQ_MAX_WIDTH, " wide");
    const int64_t D = h.size(-1);
    NEED(y.sizes() == h.sizes(), "y must have the shape of residual, ", h.sizes());
    if (has(gate)) NEED(gate->sizes() == h.sizes(), "gate must have the shape of residual, ", h.sizes());
    auto weight = [&](const Tensor &t, const char *name) {
        NEED_TYPE(t.scalar_type() == at::kFloat, name, " must be float32");
        NEED(t.dim() == 1 && t.size(0) == D && t.is_contiguous(), name, " must be a contiguous [", D, "]");
    };
    weight(post, "post_weight");
    weight(pre, "pre_weight");
    if (has(scale)) weight(*scale, "scale");
    NEED(std::isfinite((float)eps) && eps >= 0.0, "eps must be a finite number >= 0");
    on_gpu(h, "residual");
    const c10::DeviceGuard guard(h.device());
    if (at::GradMode::is_enabled() && (wants_grad(h) || wants_grad(y) || wants_grad(post) || wants_grad(pre) || wants_grad(gate) || wants_grad(scale))) {
        if (capturing()) {
            const Tensor *all[] = {&h, &y, &post, &pre, has(gate) ? &*gate : nullptr, has(scale) ? &*scale : nullptr};
            const char *names[] = {"residual", "y", "post_weight", "pre_weight", "gate", "scale"};
            for (int i = 0; i < 6; ++i)
                if (all[i]) capturable(*all[i], names[i]);
        }
        const auto r = GatedResidualNorm::apply(h, y, post, pre, gate, scale, eps);
        return {r[0], r[1]};
    }
    auto [h_out, x_out, stats] = norm_forward(h, y, post, pre, gate, scale, eps, false);
    return {h_out, x_out};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("decay_attention", &decay_attention, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("log_decay"), py::arg("scale"), py::arg("initial_state"),
          py::arg("starts"), py::arg("lengths"), py::arg("output_final_state"));
    m.def("decay_attention_step", &decay_attention_step, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("log_decay"), py::arg("state"), py::arg("scale"),
          py::arg("starts"));
    m.def("gated_residual_norm", &gated_residual_norm, py::arg("residual"), py::arg("y"), py::arg("post_weight"), py::arg("pre_weight"), py::arg("gate"),
          py::arg("scale"), py::arg("eps"));
}
