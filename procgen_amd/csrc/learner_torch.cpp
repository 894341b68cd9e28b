// learner_torch.cpp -- the learner operators as functions of torch tensors: allocation of outputs and workspaces, the argument structs of
// include/procgen_amd_learner.h, and the autograd nodes.  learner_ops.py checks the arguments and calls these; no arithmetic is done here.
//
// In C++ and not in Python because an operator's kernels take less time than a Python backward function: of the 110 us that a small loss and its gradient
// took, 50 are torch's engine and some 50 were Python's.
#include <ATen/core/grad_mode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include "../../include/procgen_amd_learner.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef c10::optional<Tensor> Maybe;

void *data(const Tensor &x) { return x.defined() ? x.data_ptr() : nullptr; }
template <class T>
T *data_as(const Tensor &x) {
    return (T *)data(x);
}
Tensor grad_of(const Tensor &x) { return x.defined() ? x.resolve_neg() : x; }  // a gradient coming in may be a view that is negated when it is read
Tensor or_none(const Maybe &x) { return x.has_value() ? *x : Tensor(); }
Maybe contiguous(const Maybe &x) { return x.has_value() ? Maybe(x->contiguous()) : x; }
bool wants_grad(const Tensor &x) { return at::GradMode::is_enabled() && x.requires_grad(); }
Tensor floats(at::IntArrayRef shape, const Tensor &like) { return at::empty(shape, like.options().dtype(at::kFloat)); }
Tensor bytes(long long n, const Tensor &like) { return n > 0 ? at::empty({n}, like.options().dtype(at::kByte)) : Tensor(); }
void *stream_of(const Tensor &x) { return c10::hip::getCurrentHIPStream(x.get_device()).stream(); }
int dtype_of(const Tensor &x) { return x.scalar_type() == at::kFloat ? PROCGEN_AMD_F32 : x.scalar_type() == at::kHalf ? PROCGEN_AMD_F16 : PROCGEN_AMD_BF16; }
void check(int rc, const char *name) {
    if (rc) throw std::runtime_error(std::string(name) + (rc < 0 ? ": the library refused the arguments" : ": HIP error " + std::to_string(rc)));
}

// What torch would have to carry on beside the values is refused: no formula of a tangent is here, and a trace would hold the allocations alone
void values_only(std::initializer_list<const Tensor *> all) {
    typedef c10::impl::TorchDispatchModeTLS Modes;
    bool traced = torch::jit::tracer::isTracing();
    if (Modes::any_modes_set())
        for (auto key : {c10::impl::TorchDispatchModeKey::FAKE, c10::impl::TorchDispatchModeKey::PROXY, c10::impl::TorchDispatchModeKey::FUNCTIONAL})
            traced = traced || Modes::get_mode(key).has_value();
    if (traced) throw std::invalid_argument("the learner operators cannot be traced");
    for (const Tensor *x : all)
        if (x->defined() && x->_fw_grad(0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode())
            throw std::invalid_argument("the learner operators have no forward-mode derivatives: an input has a tangent");
}
const Tensor *in(const Maybe &x) {
    static const Tensor none;
    return x.has_value() ? &*x : &none;
}

// gradients of a backward pass that is itself recorded (create_graph): they are right, and differentiating them is an error
variable_list once(variable_list out) {
    if (!at::GradMode::is_enabled()) return out;
    for (Tensor &x : out)
        if (x.defined()) {
            variable_list one{x.detach()};
            one[0].set_requires_grad(true);
            x = (*std::make_shared<torch::autograd::DelayedError>("the learner operators can be differentiated once", 1))(std::move(one))[0];
        }
    return out;
}

// what else a node keeps for its backward pass: one object, since entries of saved_data of their own are copied list by list
template <class T>
T &keep(AutogradContext *ctx, c10::intrusive_ptr<T> x) {
    T &kept = *x;
    ctx->saved_data["kept"] = c10::IValue::make_capsule(std::move(x));
    return kept;
}
template <class T>
T &kept(AutogradContext *ctx) {
    return static_cast<T &>(*ctx->saved_data["kept"].toCapsule());
}

// What a backward pass got back of the tensors that were saved.  Hooks (torch.autograd.graph.saved_tensors_hooks) may have kept them elsewhere meanwhile:
// other strides are taken, anything else would be read as what it is not.
void came_back(const Tensor &x, at::IntArrayRef sizes, at::ScalarType type, at::Device device) {
    if (!x.defined() || x.sizes() != sizes || x.scalar_type() != type || x.device() != device || x.layout() != at::kStrided || x.is_neg())
        throw std::runtime_error("a saved tensor came back from its hooks with another shape, type or device than it was saved with");
}
// one that was contiguous, or undefined
Tensor dense(const Tensor &x, at::IntArrayRef sizes, at::ScalarType type, at::Device device) {
    if (!x.defined()) return x;
    came_back(x, sizes, type, device);
    return x.contiguous();
}

// ---- the recurrence -------------------------------------------------------------------------------------------------------------------------

procgen_amd_array3 array3(const Tensor &x) {
    if (!x.defined()) return {nullptr, 0, 0, 0};
    return {x.data_ptr(), x.stride(0), x.stride(1), x.stride(2)};
}
procgen_amd_recurrence recurrence(const Tensor &gate, const Tensor &update, const Tensor &first, const Tensor &state, const Tensor &checkpoints, const Tensor &work) {
    procgen_amd_recurrence a = {};
    a.dtype = dtype_of(gate);
    a.T = (int)gate.size(0), a.N = (int)gate.size(1), a.D = (int)gate.size(2);
    a.gate = array3(gate), a.update = array3(update);
    if (first.defined()) a.first = data_as<uint8_t>(first), a.first_t_stride = first.stride(0), a.first_n_stride = first.stride(1);
    a.state = data_as<float>(state);
    a.checkpoints = data_as<float>(checkpoints);
    a.workspace = data(work);
    return a;
}
Tensor recurrence_workspace(const Tensor &gate) { return bytes(procgen_amd_recurrence_workspace((int)gate.size(0), (int)gate.size(1), (int)gate.size(2)), gate); }

std::pair<Tensor, Tensor> recurrence_forward(const Tensor &gate, const Tensor &update, const Tensor &first, const Tensor &state, const Tensor &state_out, const Tensor &checkpoints) {
    if (state_out.defined()) torch::autograd::impl::bump_version(state_out);  // a graph that had saved it must not go on with the new values
    Tensor h = at::empty_like(update), last = state_out.defined() ? state_out : floats({gate.size(1), gate.size(2)}, gate), work = recurrence_workspace(gate);
    procgen_amd_recurrence a = recurrence(gate, update, first, state, checkpoints, work);
    a.h = array3(h);
    a.state_out = data_as<float>(last);
    check(procgen_amd_recurrence_forward(&a, gate.get_device(), stream_of(gate)), "gated_recurrence");
    return {h, last};
}

struct RecurrenceKept : torch::CustomClassHolder {
    const std::array<int64_t, 3> shape;
    const at::ScalarType type, first_type;
    const at::Device device;
    RecurrenceKept(const Tensor &gate, const Tensor &first)
        : shape{gate.size(0), gate.size(1), gate.size(2)}, type(gate.scalar_type()), first_type(first.defined() ? first.scalar_type() : at::kByte), device(gate.device()) {}
};

struct GatedRecurrence : torch::autograd::Function<GatedRecurrence> {
    static variable_list forward(AutogradContext *ctx, const Tensor &gate, const Tensor &update, const Maybe &first_, const Maybe &state_) {
        const Tensor first = or_none(first_), state = or_none(state_);
        Tensor checkpoints = floats({procgen_amd_recurrence_checkpoints((int)gate.size(0)), gate.size(1), gate.size(2)}, gate);
        auto [h, last] = recurrence_forward(gate, update, first, state, Tensor(), checkpoints);
        ctx->save_for_backward({gate, update, first, state, checkpoints});
        keep(ctx, c10::make_intrusive<RecurrenceKept>(gate, first));
        ctx->set_materialize_grads(false);
        return {h, last};
    }
    static variable_list backward(AutogradContext *ctx, variable_list d) {
        const variable_list saved = ctx->get_saved_variables();
        const RecurrenceKept &k = kept<RecurrenceKept>(ctx);
        const auto [T, N, D] = k.shape;
        const Tensor &gate = saved[0], &update = saved[1], &first = saved[2];
        came_back(gate, k.shape, k.type, k.device);
        came_back(update, k.shape, k.type, k.device);
        if (first.defined()) came_back(first, {T, N}, k.first_type, k.device);
        const Tensor state = dense(saved[3], {N, D}, at::kFloat, k.device), checkpoints = dense(saved[4], {procgen_amd_recurrence_checkpoints((int)T), N, D}, at::kFloat, k.device);
        Tensor work = recurrence_workspace(gate), d_h = grad_of(d[0]), d_last = d[1].defined() ? grad_of(d[1]).contiguous() : Tensor();
        Tensor d_gate = ctx->needs_input_grad(0) ? at::empty_like(gate) : Tensor(), d_update = ctx->needs_input_grad(1) ? at::empty_like(update) : Tensor();
        Tensor d_state = state.defined() && ctx->needs_input_grad(first.defined() ? 3 : 2) ? at::empty_like(state) : Tensor();
        procgen_amd_recurrence a = recurrence(gate, update, first, state, checkpoints, work);
        a.d_h = array3(d_h), a.d_gate = array3(d_gate), a.d_update = array3(d_update);
        a.d_state_out = data_as<float>(d_last);
        a.d_state = data_as<float>(d_state);
        check(procgen_amd_recurrence_backward(&a, gate.get_device(), stream_of(gate)), "gated_recurrence");
        return once({d_gate, d_update, Tensor(), d_state});
    }
};

std::pair<Tensor, Tensor> gated_recurrence(const Tensor &gate, const Tensor &update, const Maybe &first_, const Maybe &state_, const Maybe &state_out_) {
    values_only({&gate, &update, in(state_), in(state_out_)});
    const Maybe state = contiguous(state_);
    if (!wants_grad(gate) && !wants_grad(update) && !(state && wants_grad(*state)))
        return recurrence_forward(gate, update, or_none(first_), or_none(state), or_none(state_out_), Tensor());
    const variable_list out = GatedRecurrence::apply(gate, update, first_, state);
    return {out[0], out[1]};
}

std::pair<Tensor, Tensor> advantages(const Tensor &rew, const Tensor &values, const Tensor &first, double gamma, double lam) {
    values_only({&rew, &values});
    const int T = (int)rew.size(0), N = (int)rew.size(1);
    Tensor adv = floats({T, N}, rew), ret = floats({T, N}, rew), work = bytes(procgen_amd_recurrence_workspace(T, N, 1), rew);
    procgen_amd_advantage a = {};
    a.dtype = dtype_of(values), a.T = T, a.N = N;
    a.rew = data_as<float>(rew), a.rew_t_stride = rew.stride(0), a.rew_n_stride = rew.stride(1);
    a.values = data(values), a.values_t_stride = values.stride(0), a.values_n_stride = values.stride(1);
    a.first = data_as<uint8_t>(first), a.first_t_stride = first.stride(0), a.first_n_stride = first.stride(1);
    a.gamma = (float)gamma, a.lam = (float)lam;
    a.adv = data_as<float>(adv), a.ret = data_as<float>(ret);
    a.workspace = data(work);
    check(procgen_amd_advantages(&a, rew.get_device(), stream_of(rew)), "advantages");
    return {adv, ret};
}

// ---- rows of logits -------------------------------------------------------------------------------------------------------------------------

// where the rows of a [..., columns] tensor are: the leading dimensions as at most two strided ones (worked out by learner_ops.py)
struct Layout {
    int64_t inner, outer_stride, inner_stride;
    static Layout contiguous(const Tensor &x) { return {1, x.size(-1), 0}; }
};
procgen_amd_rows rows_of(const Tensor &logits, const Layout &at, const Tensor &actions, const Tensor &d_logits, const Tensor &work) {
    procgen_amd_rows a = {};
    a.dtype = dtype_of(logits);
    a.columns = logits.size(-1), a.rows = logits.numel() / a.columns, a.inner = at.inner;
    a.logits = data(logits), a.outer_stride = at.outer_stride, a.inner_stride = at.inner_stride;
    a.actions = data(actions), a.actions_are_64_bit = actions.scalar_type() == at::kLong;
    a.d_logits = data(d_logits);
    a.workspace = data(work);
    return a;
}
struct PolicyArgs {
    Layout at, ref_at;
    double clip_low, clip_high, kl_coef, entropy_coef;
};
struct RowsKept : torch::CustomClassHolder {
    const at::DimVector sizes, strides;
    const at::ScalarType type, action_type;
    const at::Device device;
    const PolicyArgs p;  // of log-probabilities the first layout alone
    at::DimVector ref_strides;
    at::ScalarType valid_type = at::kByte;
    Tensor work, d_logits;
    int64_t capture = 0;
    RowsKept(const Tensor &logits, const Tensor &actions, const PolicyArgs &args)
        : sizes(logits.sizes()), strides(logits.strides()), type(logits.scalar_type()), action_type(actions.scalar_type()), device(logits.device()), p(args) {}
    Tensor per_row(const Tensor &x, at::ScalarType t) const { return dense(x, at::IntArrayRef(sizes).slice(0, sizes.size() - 1), t, device); }
};

void logprobs_forward(const Tensor &logits, const Layout &at, const Tensor &actions, const Tensor &logp, const Tensor &entropy, const Tensor &lse) {
    const procgen_amd_rows a = rows_of(logits, at, actions, Tensor(), Tensor());
    check(procgen_amd_action_logprobs(&a, data_as<float>(logp), data_as<float>(entropy), data_as<procgen_amd_lse>(lse), logits.get_device(), stream_of(logits)), "action_logprobs");
}

struct ActionLogprobs : torch::autograd::Function<ActionLogprobs> {
    static variable_list forward(AutogradContext *ctx, const Tensor &logits, const Tensor &actions, Layout at) {
        Tensor logp = floats(actions.sizes(), logits), entropy = floats(actions.sizes(), logits), lse = floats({actions.numel(), 2}, logits);
        logprobs_forward(logits, at, actions, logp, entropy, lse);
        ctx->save_for_backward({logits, actions, lse, entropy});
        keep(ctx, c10::make_intrusive<RowsKept>(logits, actions, PolicyArgs{at, {}, 0, 0, 0, 0}));
        ctx->set_materialize_grads(false);
        return {logp, entropy};
    }
    static variable_list backward(AutogradContext *ctx, variable_list d) {
        const variable_list saved = ctx->get_saved_variables();
        const RowsKept &k = kept<RowsKept>(ctx);
        came_back(saved[0], k.sizes, k.type, k.device);
        const bool moved = saved[0].strides() != at::IntArrayRef(k.strides);
        const Tensor logits = moved ? saved[0].contiguous() : saved[0], actions = k.per_row(saved[1], k.action_type);
        const Layout at = moved ? Layout::contiguous(logits) : k.p.at;
        const Tensor lse = dense(saved[2], {actions.numel(), 2}, at::kFloat, k.device), entropy = k.per_row(saved[3], at::kFloat);
        Tensor d_logits = at::empty(logits.sizes(), logits.options().memory_format(at::MemoryFormat::Contiguous));
        Tensor d_logp = d[0].defined() ? grad_of(d[0]).contiguous() : Tensor(), d_entropy = d[1].defined() ? grad_of(d[1]).contiguous() : Tensor();
        const procgen_amd_rows a = rows_of(logits, at, actions, d_logits, Tensor());
        check(procgen_amd_action_logprobs_backward(&a, data_as<procgen_amd_lse>(lse), data_as<float>(entropy), data_as<float>(d_logp), data_as<float>(d_entropy), logits.get_device(),
                                                   stream_of(logits)),
              "action_logprobs");
        return once({d_logits, Tensor(), Tensor()});
    }
};

std::pair<Tensor, Tensor> action_logprobs(const Tensor &logits, const Tensor &actions_, int64_t inner, int64_t outer_stride, int64_t inner_stride) {
    values_only({&logits});
    const Layout at{inner, outer_stride, inner_stride};
    const Tensor actions = actions_.contiguous();
    if (wants_grad(logits)) {
        const variable_list out = ActionLogprobs::apply(logits, actions, at);
        return {out[0], out[1]};
    }
    Tensor logp = floats(actions.sizes(), logits), entropy = floats(actions.sizes(), logits);
    logprobs_forward(logits, at, actions, logp, entropy, Tensor());
    return {logp, entropy};
}

procgen_amd_policy policy_of(const PolicyArgs &p, const Tensor &old, const Tensor &adv, const Tensor &valid, const Tensor &ref_logits, const Tensor &ref_logp) {
    procgen_amd_policy q = {};
    q.old_logprobs = data_as<float>(old), q.adv = data_as<float>(adv), q.valid = data_as<uint8_t>(valid);
    q.ref_logits = data(ref_logits), q.ref_outer_stride = p.ref_at.outer_stride, q.ref_inner_stride = p.ref_at.inner_stride;
    q.ref_logprobs = data_as<float>(ref_logp);
    q.clip_low = (float)p.clip_low, q.clip_high = (float)p.clip_high, q.kl_coef = (float)p.kl_coef, q.entropy_coef = (float)p.entropy_coef;
    return q;
}
struct PolicyOut {
    Tensor loss, stats, work;
};
PolicyOut policy_forward(const PolicyArgs &p, const Tensor &d_logits, const Tensor &logits, const Tensor &actions, const Tensor &old, const Tensor &adv, const Tensor &valid,
                         const Tensor &ref_logits, const Tensor &ref_logp) {
    PolicyOut out{floats({}, logits), floats({4}, logits), bytes(procgen_amd_rows_workspace(logits.numel() / logits.size(-1), logits.size(-1)), logits)};
    const procgen_amd_rows a = rows_of(logits, p.at, actions, d_logits, out.work);
    procgen_amd_policy q = policy_of(p, old, adv, valid, ref_logits, ref_logp);
    q.loss = data_as<float>(out.loss), q.stats = data_as<float>(out.stats);
    check(procgen_amd_policy_loss(&a, &q, logits.get_device(), stream_of(logits)), "policy_loss");
    return out;
}

// The forward call writes the gradient too, from the row that it has in registers.  The first backward pass hands it out, after a kernel that goes over
// the rows again only where the loss's own gradient is not 1; each further one (retain_graph) computes its own, and so does a backward pass that is
// captured apart from its forward call.
struct PolicyLoss : torch::autograd::Function<PolicyLoss> {
    static variable_list forward(AutogradContext *ctx, const Tensor &logits, const Tensor &actions, const Tensor &old, const Tensor &adv, const Maybe &valid_,
                                 const Maybe &ref_logits_, const Maybe &ref_logp_, PolicyArgs p) {
        const Tensor valid = or_none(valid_), ref_logits = or_none(ref_logits_), ref_logp = or_none(ref_logp_);
        Tensor d_logits = at::empty(logits.sizes(), logits.options().memory_format(at::MemoryFormat::Contiguous));
        const PolicyOut out = policy_forward(p, d_logits, logits, actions, old, adv, valid, ref_logits, ref_logp);
        ctx->save_for_backward({logits, actions, old, adv, valid, ref_logits, ref_logp});
        RowsKept &k = keep(ctx, c10::make_intrusive<RowsKept>(logits, actions, p));
        if (ref_logits.defined()) k.ref_strides = at::DimVector(ref_logits.strides());
        if (valid.defined()) k.valid_type = valid.scalar_type();
        k.work = out.work, k.d_logits = d_logits;
        k.capture = procgen_amd_capture_id(stream_of(logits));
        ctx->mark_non_differentiable({out.stats});
        return {out.loss, out.stats};
    }
    static variable_list backward(AutogradContext *ctx, variable_list d) {
        const variable_list saved = ctx->get_saved_variables();
        RowsKept &k = kept<RowsKept>(ctx);
        PolicyArgs p = k.p;
        Tensor logits = saved[0], ref_logits = saved[5];
        came_back(logits, k.sizes, k.type, k.device);
        if (ref_logits.defined()) came_back(ref_logits, k.sizes, k.type, k.device);
        if (logits.strides() != at::IntArrayRef(k.strides) || (ref_logits.defined() && ref_logits.strides() != at::IntArrayRef(k.ref_strides))) {  // the two share one split of their rows
            logits = logits.contiguous();
            p.at = Layout::contiguous(logits);
            if (ref_logits.defined()) ref_logits = ref_logits.contiguous(), p.ref_at = Layout::contiguous(ref_logits);
        }
        const Tensor actions = k.per_row(saved[1], k.action_type), old = k.per_row(saved[2], at::kFloat), adv = k.per_row(saved[3], at::kFloat);
        const Tensor valid = k.per_row(saved[4], k.valid_type), ref_logp = k.per_row(saved[6], at::kFloat), scale = grad_of(d[0]).contiguous();
        Tensor d_logits = std::move(k.d_logits);
        const bool held = d_logits.defined() && k.capture >= 0 && k.capture == procgen_amd_capture_id(stream_of(logits));
        if (!held) d_logits = at::empty(logits.sizes(), logits.options().memory_format(at::MemoryFormat::Contiguous));
        const procgen_amd_rows a = rows_of(logits, p.at, actions, d_logits, k.work);
        procgen_amd_policy q = policy_of(p, old, adv, valid, ref_logits, ref_logp);
        q.scale = data_as<float>(scale);
        q.resume = held ? 3 : 1;
        check(procgen_amd_policy_loss(&a, &q, logits.get_device(), stream_of(logits)), "policy_loss");
        return once({d_logits, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()});
    }
};

std::pair<Tensor, Tensor> policy_loss(const Tensor &logits, const Tensor &actions_, const Tensor &old_, const Tensor &adv_, const Maybe &valid_, const Maybe &ref_logits_,
                                      const Maybe &ref_logp_, double clip_low, double clip_high, double kl_coef, double entropy_coef, int64_t inner, int64_t outer_stride,
                                      int64_t inner_stride, int64_t ref_outer_stride, int64_t ref_inner_stride) {
    values_only({&logits, &old_, &adv_, in(ref_logits_), in(ref_logp_)});
    const PolicyArgs p{{inner, outer_stride, inner_stride}, {inner, ref_outer_stride, ref_inner_stride}, clip_low, clip_high, kl_coef, entropy_coef};
    const Tensor actions = actions_.contiguous(), old = old_.contiguous(), adv = adv_.contiguous();
    const Maybe valid = contiguous(valid_), ref_logp = contiguous(ref_logp_);
    if (wants_grad(logits)) {
        const variable_list out = PolicyLoss::apply(logits, actions, old, adv, valid, ref_logits_, ref_logp, p);
        return {out[0], out[1]};
    }
    const PolicyOut out = policy_forward(p, Tensor(), logits, actions, old, adv, or_none(valid), or_none(ref_logits_), or_none(ref_logp));
    return {out.loss, out.stats};
}

}  // namespace

PYBIND11_MODULE(learner_torch, m) {
    m.def("gated_recurrence", &gated_recurrence);
    m.def("advantages", &advantages);
    m.def("action_logprobs", &action_logprobs);
    m.def("policy_loss", &policy_loss);
}
