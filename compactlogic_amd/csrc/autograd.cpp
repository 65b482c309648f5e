// The autograd side of the losses on chosen log-probabilities, of dropout and of the recurrence: what
// their calls allocate, launch and save, and their backwards, over the entry points of
// libcompactlogic_hip.so; and the walk over an optimizer's tensors.
//
// A small call's kernels take 6 to 15 us.  As Functions in Python such calls took 76 to 97 us, here
// 45 to 62: autograd runs a backward on a thread of its own, and an interpreter on either side of
// that hand-over costs 30 us more (torch's own negation, forward and backward, takes 45).
// Most arguments are checked in policy.py, dropout_layer.py and drafts.py; nothing here is a public
// interface.
#include <torch/extension.h>

#include <c10/hip/HIPStream.h>

#include <stdexcept>
#include <string>
#include <tuple>
#include <utility>
#include <vector>

#include "../../include/compactlogic_hip.h"
#include "timed_hook.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

namespace {

// A failure status of the library as the Python package's exception.  It is raised as one here, on
// any thread: of a C++ exception that leaves a backward, autograd hands on the text alone.
[[noreturn]] void fail(const char* name, int status) {
    const std::string text = std::string(name) + " failed (status " + std::to_string(status) +
                             "): " + cl_last_error();
    py::gil_scoped_acquire gil;
    const py::object type =
        status == CL_ERR_VALUE
            ? py::reinterpret_borrow<py::object>(PyExc_ValueError)
            : py::module_::import("compactlogic_amd._capi").attr("CompactLogicError");
    PyErr_SetString(type.ptr(), text.c_str());
    throw py::error_already_set();
}

cl::TimedHook g_timed;

// One entry point on the current stream of the current device.
template <typename F>
void launch(const char* name, int device, F&& f) {
    void* stream = c10::hip::getCurrentHIPStream(c10::DeviceIndex(device)).stream();
    g_timed.run(name, [&] {
        if (const int rc = f(stream)) fail(name, rc);
    });
}

int code_of(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return CL_DTYPE_F32;
        case at::kDouble: return CL_DTYPE_F64;
        case at::kHalf: return CL_DTYPE_F16;
        case at::kBFloat16: return CL_DTYPE_BF16;
        default: throw std::runtime_error("unsupported dtype");
    }
}

at::TensorOptions wide_of(const Tensor& t) {
    return t.options().dtype(t.scalar_type() == at::kDouble ? at::kDouble : at::kFloat);
}

void sized(const char* name, int rc) {
    if (rc) fail(name, rc);
}

const int64_t* ints(const Tensor& t) { return static_cast<const int64_t*>(t.data_ptr()); }

// Contiguous rows, any distance apart.
Tensor rows_of(const Tensor& x) {
    return x.stride(1) != 1 && x.size(1) > 1 ? x.contiguous() : x;
}

// What a call keeps to itself: one allocation, its parts on 32 bytes each.
struct Parts {
    int64_t total = 0;
    int64_t add(int64_t bytes) {
        const int64_t at = total;
        total += (bytes + 31) & ~int64_t(31);
        return at;
    }
    Tensor allocate(const Tensor& like) const {
        return at::empty({total < 32 ? 32 : total}, like.options().dtype(at::kByte));
    }
};

int64_t rows_workspace(int code, int64_t rows, int64_t cols) {
    int64_t need = 0;
    sized("cl_token_loss_workspace", cl_token_loss_workspace(code, rows, cols, &need));
    return need;
}

// GroupSum's k classes and tau; k = 0 where the logits are the input itself.
struct Group {
    int64_t k = 0;
    double tau = 1;
    int64_t batch = 0, features = 0;
    bool batch_major = false;
};

// What a forward leaves for its backward beside the saved tensors.
struct Plan : torch::CustomClassHolder {
    Group group;
    int reduction = 0;
    int64_t pairs = 0;
    int64_t count = 0, row_seq = 0, seq_slope = 0;  // places in the buffer
    Tensor grad;           // formed in the forward, for an upstream gradient of 1
    uint64_t capture = 0;  // the graph capture it was formed in
};

void keep(AutogradContext* ctx, c10::intrusive_ptr<Plan> plan, const Tensor& logits,
          const Tensor& actions, const Tensor& aux) {
    ctx->save_for_backward({logits, actions, aux});
    ctx->saved_data["plan"] = c10::IValue::make_capsule(std::move(plan));
}

// The logits, actions and buffer that a forward saved, wherever they lie now (hooks on saved
// tensors may have moved them), and its plan.
struct Saved {
    Tensor logits, actions, aux;
    c10::intrusive_ptr<torch::CustomClassHolder> holder;
    char* at;

    explicit Saved(AutogradContext* ctx) {
        // the backwards are kernels without a derivative of their own: under create_graph a
        // second derivative would silently lack its part
        if (at::GradMode::is_enabled())
            throw std::runtime_error(
                "the losses on chosen log-probabilities cannot be differentiated twice");
        variable_list v = ctx->get_saved_variables();
        logits = rows_of(v[0]);
        actions = v[1];
        aux = v[2];
        at = static_cast<char*>(aux.data_ptr());
        holder = ctx->saved_data["plan"].toCapsule();
    }
    Plan& plan() const { return *static_cast<Plan*>(holder.get()); }
};

// The rows of logits to work on: x itself, or GroupSum's scores of the activations x [batch,
// features], less each sample's largest one (which no loss here depends on), so that they are not
// rounded at the size of a class sum.
Tensor logits_of(const Tensor& input, Group& g) {
    if (!g.k) return rows_of(input);
    Tensor x = input;
    g.batch = x.size(0);
    g.features = x.size(1);
    if (g.batch > 1 && g.features > 1 && (x.stride(0) == 0 || x.stride(1) == 0))
        x = x.contiguous();
    const int64_t sb = x.stride(0), sf = x.stride(1);
    g.batch_major = sb == 1 && sf != 1;
    const int code = code_of(x);
    int64_t need = 0;
    sized("cl_group_sum_centered_workspace_size",
          cl_group_sum_centered_workspace_size(code, g.batch, g.features, sb, g.k, &need));
    Tensor scores = at::empty({g.batch, g.k}, x.options()), ws;
    if (need > 0) ws = at::empty({need}, x.options().dtype(at::kByte));
    launch("cl_group_sum_centered_forward", x.get_device(), [&](void* stream) {
        return cl_group_sum_centered_forward(code, x.data_ptr(), g.batch, g.features, sb, sf, g.k,
                                             g.tau, scores.data_ptr(),
                                             need > 0 ? ws.data_ptr() : nullptr, need, stream);
    });
    return scores;
}

// The upstream gradient of the scores of GroupSum, see cl_group_sum_chosen_backward.
struct ScoreUpstream {
    const void *row_grad = nullptr, *loss_grad = nullptr, *count = nullptr;
    const int32_t* row_seq = nullptr;
    const void *seq_slope = nullptr, *pair_grad = nullptr;
    int64_t pairs = 0;
};

// The gradient of GroupSum's input in its layout, formed from the scores where it is spread over
// the features.
Tensor group_grad(const Saved& s, const Group& g, const ScoreUpstream& up) {
    Tensor grad;
    if (g.batch_major)
        grad = at::empty_strided({g.batch, g.features}, {1, g.batch}, s.logits.options());
    else
        grad = at::empty({g.batch, g.features}, s.logits.options());
    const int64_t sb = g.batch_major ? 1 : g.features, sf = g.batch_major ? g.batch : 1;
    launch("cl_group_sum_chosen_backward", grad.get_device(), [&](void* stream) {
        return cl_group_sum_chosen_backward(code_of(grad), s.logits.data_ptr(), g.batch,
                                            g.features, g.k, g.tau, ints(s.actions), s.at,
                                            up.row_grad, up.loss_grad, up.count, up.row_seq,
                                            up.seq_slope, up.pair_grad, up.pairs, grad.data_ptr(),
                                            sb, sf, stream);
    });
    return grad;
}

uint64_t capture_id(const Tensor& t) {
    uint64_t id = 0;
    void* stream = c10::hip::getCurrentHIPStream(t.get_device()).stream();
    sized("cl_stream_capture_id", cl_stream_capture_id(stream, &id));
    return id;
}

int64_t state_bytes(const Tensor& logits) {
    return 4 * (logits.scalar_type() == at::kDouble ? 8 : 4) * logits.size(0);
}

// ---- lp[n] = log_softmax(logits[n])[actions[n]] in one pass over the logits; the backward makes
// the probabilities again from the row's maximum and sum.
struct LogProbArgs {
    Tensor actions;
    int64_t ignore;
    Group group;
};

struct LogProbs : Function<LogProbs> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const LogProbArgs& a) {
        auto plan = c10::make_intrusive<Plan>();
        plan->group = a.group;
        const Tensor logits = logits_of(x, plan->group);
        const int code = code_of(logits);
        const int64_t rows = logits.size(0), cols = logits.size(1);
        const int64_t need = rows_workspace(code, rows, cols);
        Parts parts;
        parts.add(state_bytes(logits));
        const int64_t ws = parts.add(need);
        const Tensor aux = parts.allocate(logits);
        char* at = static_cast<char*>(aux.data_ptr());
        Tensor lp = at::empty({rows}, wide_of(logits));
        launch("cl_selected_log_prob_forward", x.get_device(), [&](void* stream) {
            return cl_selected_log_prob_forward(code, logits.data_ptr(), logits.stride(0), rows,
                                                cols, ints(a.actions), a.ignore, lp.data_ptr(), at,
                                                at + ws, need, stream);
        });
        keep(ctx, std::move(plan), logits, a.actions, aux);
        return lp;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const Saved s(ctx);
        const c10::DeviceGuard guard(s.logits.device());
        const Tensor up = grads[0].contiguous();
        if (s.plan().group.k) {
            ScoreUpstream u;
            u.row_grad = up.data_ptr();
            return {group_grad(s, s.plan().group, u), Tensor()};
        }
        const int64_t rows = s.logits.size(0), cols = s.logits.size(1);
        Tensor grad = at::empty({rows, cols}, s.logits.options());
        launch("cl_selected_log_prob_backward", grad.get_device(), [&](void* stream) {
            return cl_selected_log_prob_backward(code_of(grad), s.logits.data_ptr(),
                                                 s.logits.stride(0), rows, cols, ints(s.actions),
                                                 s.at, up.data_ptr(), grad.data_ptr(), stream);
        });
        return {grad, Tensor()};
    }
};

// ---- the clipped policy loss with a KL term: (loss, log_probs), the second not differentiable.
struct PolicyArgs {
    Tensor actions, old, adv;
    c10::optional<Tensor> ref;
    double low, high, kl;
    int64_t ignore;
    int reduction;
    bool prefill;  // the logits' gradient along with the loss
    Group group;
};

struct PolicyLoss : Function<PolicyLoss> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const PolicyArgs& a) {
        auto plan = c10::make_intrusive<Plan>();
        plan->group = a.group;
        plan->reduction = a.reduction;
        const Tensor logits = logits_of(x, plan->group);
        const int code = code_of(logits);
        const int64_t rows = logits.size(0), cols = logits.size(1);
        const at::TensorOptions wide = wide_of(logits);
        const int64_t size = logits.scalar_type() == at::kDouble ? 8 : 4;
        const int64_t need = rows_workspace(code, rows, cols);
        const bool scalar = a.reduction != CL_REDUCE_NONE;
        Parts parts;
        parts.add(state_bytes(logits));
        plan->count = parts.add(size);
        const int64_t terms = parts.add(scalar ? size * rows : 0), ws = parts.add(need);
        const Tensor aux = parts.allocate(logits);
        char* at = static_cast<char*>(aux.data_ptr());
        Tensor lp = at::empty({rows}, wide);
        Tensor loss = scalar ? at::empty({}, wide) : at::empty({rows}, wide);
        if (a.prefill) {
            plan->grad = at::empty({rows, cols}, logits.options());
            plan->capture = capture_id(logits);
        }
        launch("cl_policy_loss_forward", x.get_device(), [&](void* stream) {
            return cl_policy_loss_forward(
                code, logits.data_ptr(), logits.stride(0), rows, cols, ints(a.actions), a.ignore,
                a.old.data_ptr(), a.adv.data_ptr(), a.ref ? a.ref->data_ptr() : nullptr, a.low,
                a.high, a.kl, a.reduction, lp.data_ptr(), at,
                scalar ? static_cast<void*>(at + terms) : loss.data_ptr(), loss.data_ptr(),
                at + plan->count, a.prefill ? plan->grad.data_ptr() : nullptr, at + ws, need,
                stream);
        });
        keep(ctx, std::move(plan), logits, a.actions, aux);
        ctx->mark_non_differentiable({lp});
        ctx->set_materialize_grads(false);
        return {loss, lp};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        if (!grads[0].defined()) return {Tensor(), Tensor()};
        const Saved s(ctx);
        const c10::DeviceGuard guard(s.logits.device());
        Plan& plan = s.plan();
        const Tensor up = grads[0].contiguous();
        if (plan.group.k) {
            ScoreUpstream u;
            (plan.reduction == CL_REDUCE_NONE ? u.row_grad : u.loss_grad) = up.data_ptr();
            if (plan.reduction == CL_REDUCE_MEAN) u.count = s.at + plan.count;
            return {group_grad(s, plan.group, u), Tensor()};
        }
        const int64_t rows = s.logits.size(0), cols = s.logits.size(1);
        // the forward's gradient is handed out once, and only in the capture (or outside of any)
        // that it was written in: a replay of the backward alone would find it used
        Tensor grad = std::move(plan.grad);
        plan.grad = Tensor();
        const bool prefilled = grad.defined() && plan.capture == capture_id(s.logits);
        if (!prefilled) grad = at::empty({rows, cols}, s.logits.options());
        launch("cl_policy_loss_backward", grad.get_device(), [&](void* stream) {
            return cl_policy_loss_backward(code_of(grad), s.logits.data_ptr(), s.logits.stride(0),
                                           rows, cols, ints(s.actions), s.at, plan.reduction,
                                           up.data_ptr(), s.at + plan.count, prefilled,
                                           grad.data_ptr(), stream);
        });
        return {grad, Tensor()};
    }
};

// ---- the preference loss of paired sequences: (loss, margins), the second not differentiable.
struct PreferenceArgs {
    Tensor actions, offsets;
    c10::optional<Tensor> ref;
    double beta, smoothing;
    int64_t ignore;
    int reduction;
    Group group;
};

struct PreferenceLoss : Function<PreferenceLoss> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const PreferenceArgs& a) {
        auto plan = c10::make_intrusive<Plan>();
        plan->group = a.group;
        plan->reduction = a.reduction;
        const Tensor logits = logits_of(x, plan->group);
        const int code = code_of(logits);
        const int64_t rows = logits.size(0), cols = logits.size(1);
        const int64_t pairs = plan->pairs = (a.offsets.numel() - 1) / 2;
        const at::TensorOptions wide = wide_of(logits);
        const int64_t size = logits.scalar_type() == at::kDouble ? 8 : 4;
        const int64_t need = rows_workspace(code, rows, cols);
        const bool scalar = a.reduction != CL_REDUCE_NONE;
        Parts parts;
        parts.add(state_bytes(logits));
        plan->count = parts.add(size);
        plan->row_seq = parts.add(4 * rows);
        plan->seq_slope = parts.add(2 * pairs * size);
        const int64_t gaps = parts.add(8 * rows), lp = parts.add(size * rows);
        const int64_t terms = parts.add(scalar ? size * pairs : 0), ws = parts.add(need);
        const Tensor aux = parts.allocate(logits);
        char* at = static_cast<char*>(aux.data_ptr());
        Tensor margins = at::empty({pairs}, wide);
        Tensor loss = scalar ? at::empty({}, wide) : at::empty({pairs}, wide);
        launch("cl_preference_loss_forward", x.get_device(), [&](void* stream) {
            return cl_preference_loss_forward(
                code, logits.data_ptr(), logits.stride(0), rows, cols, ints(a.actions), a.ignore,
                a.ref ? a.ref->data_ptr() : nullptr, ints(a.offsets), pairs, a.beta, a.smoothing,
                a.reduction, at + lp, at, reinterpret_cast<double*>(at + gaps),
                reinterpret_cast<int32_t*>(at + plan->row_seq), at + plan->seq_slope,
                margins.data_ptr(), scalar ? static_cast<void*>(at + terms) : loss.data_ptr(),
                loss.data_ptr(), at + plan->count, at + ws, need, stream);
        });
        keep(ctx, std::move(plan), logits, a.actions, aux);
        ctx->mark_non_differentiable({margins});
        ctx->set_materialize_grads(false);
        return {loss, margins};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        if (!grads[0].defined()) return {Tensor(), Tensor()};
        const Saved s(ctx);
        const c10::DeviceGuard guard(s.logits.device());
        const Plan& plan = s.plan();
        const Tensor up = grads[0].contiguous();
        const auto* row_seq = reinterpret_cast<const int32_t*>(s.at + plan.row_seq);
        if (plan.group.k) {
            ScoreUpstream u;
            (plan.reduction == CL_REDUCE_NONE ? u.pair_grad : u.loss_grad) = up.data_ptr();
            if (plan.reduction == CL_REDUCE_MEAN) u.count = s.at + plan.count;
            u.row_seq = row_seq;
            u.seq_slope = s.at + plan.seq_slope;
            u.pairs = plan.pairs;
            return {group_grad(s, plan.group, u), Tensor()};
        }
        const int64_t rows = s.logits.size(0), cols = s.logits.size(1);
        Tensor grad = at::empty({rows, cols}, s.logits.options());
        launch("cl_preference_loss_backward", grad.get_device(), [&](void* stream) {
            return cl_preference_loss_backward(
                code_of(grad), s.logits.data_ptr(), s.logits.stride(0), rows, cols,
                ints(s.actions), s.at, row_seq, s.at + plan.seq_slope, plan.pairs, plan.reduction,
                up.data_ptr(), s.at + plan.count, grad.data_ptr(), stream);
        });
        return {grad, Tensor()};
    }
};

// ---- dropout of a 2-D tensor; the gradient passes the same mask, made again from the seed (and
// is itself a dropout, so it can be differentiated as often as one likes).
struct DropArgs {
    int64_t threshold;
    c10::optional<double> fill;
    uint64_t seed, offset;
    c10::optional<Tensor> rng;
};

// The result lies as the tensor does.
Tensor dropped(const Tensor& input, const DropArgs& a, bool rescale, double fill,
               const Tensor& rng) {
    Tensor x = input;
    const int64_t rows = x.size(0), cols = x.size(1);
    if (!(x.stride(1) == 1 || cols == 1 || x.stride(0) == 1 || rows == 1)) x = x.contiguous();
    const bool by_rows = x.stride(1) == 1 || cols == 1;
    Tensor y = by_rows ? at::empty({rows, cols}, x.options())
                       : at::empty_strided({rows, cols}, {1, rows}, x.options());
    const int64_t yr = by_rows ? cols : 1, yc = by_rows ? 1 : rows;
    launch("cl_dropout", x.get_device(), [&](void* stream) {
        return cl_dropout(code_of(x), x.data_ptr(), x.stride(0), x.stride(1), y.data_ptr(), yr, yc,
                          rows, cols, a.threshold, rescale, fill, a.seed, a.offset,
                          rng.defined() ? ints(rng) : nullptr, stream);
    });
    return y;
}

struct DropPlan : torch::CustomClassHolder {
    DropArgs args;
};

struct Drop : Function<Drop> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const DropArgs& a) {
        auto plan = c10::make_intrusive<DropPlan>();
        plan->args = a;
        plan->args.rng.reset();
        if (a.rng) ctx->save_for_backward({*a.rng});
        ctx->saved_data["plan"] = c10::IValue::make_capsule(std::move(plan));
        return dropped(x, a, !a.fill, a.fill.value_or(0.0), a.rng ? *a.rng : Tensor());
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto holder = ctx->saved_data["plan"].toCapsule();
        DropArgs a = static_cast<DropPlan*>(holder.get())->args;
        const variable_list saved = ctx->get_saved_variables();
        const Tensor rng = saved.empty() ? Tensor() : saved[0];
        const c10::DeviceGuard guard(grads[0].device());
        if (!at::GradMode::is_enabled())
            return {dropped(grads[0], a, !a.fill, 0.0, rng), Tensor()};
        if (a.fill) a.fill = 0.0;
        if (rng.defined()) a.rng = rng;
        return {Drop::apply(grads[0], a), Tensor()};
    }
};

// ---- the gated linear recurrence of [batch, time, features]: (y, last state).

// What is contiguous in x, and the order of the rest (CL_RECURRENCE_*); -1: nothing that a kernel takes.
int order_of(const Tensor& x) {
    const int64_t batch = x.size(0), time = x.size(1), features = x.size(2);
    if (features > 1 && x.stride(2) == 1) return CL_RECURRENCE_FEATURES;
    if (time > 1)
        return x.stride(1) != 1 ? -1
               : x.stride(0) >= x.stride(2) ? CL_RECURRENCE_TIME_BATCH
                                            : CL_RECURRENCE_TIME_FEATURES;
    if (batch > 1) return x.stride(0) == 1 ? CL_RECURRENCE_BATCH : -1;
    return features > 1 ? -1 : CL_RECURRENCE_FEATURES;
}

bool ordered(const Tensor& t, int order) {
    const int d = order == CL_RECURRENCE_FEATURES ? 2 : order == CL_RECURRENCE_BATCH ? 0 : 1;
    return t.size(d) <= 1 || t.stride(d) == 1;
}

bool features_outermost(int order) {
    return order == CL_RECURRENCE_TIME_FEATURES || order == CL_RECURRENCE_BATCH;
}

Tensor sequence_like(const Tensor& x, int order) {
    const int64_t batch = x.size(0), time = x.size(1), features = x.size(2);
    if (order == CL_RECURRENCE_FEATURES) return at::empty({batch, time, features}, x.options());
    if (order == CL_RECURRENCE_TIME_BATCH)
        return at::empty_strided({batch, time, features}, {features * time, 1, time}, x.options());
    return at::empty_strided({batch, time, features}, {time, 1, batch * time}, x.options());
}

Tensor state_like(const Tensor& x, int order) {
    const int64_t batch = x.size(0), features = x.size(2);
    if (!features_outermost(order)) return at::empty({batch, features}, wide_of(x));
    return at::empty_strided({batch, features}, {1, batch}, wide_of(x));
}

Tensor in_order(const Tensor& t, int order) {
    if (ordered(t, order)) return t;
    return sequence_like(t, order).copy_(t);
}

const int64_t* strides_of(const Tensor& t) { return t.defined() ? t.strides().data() : nullptr; }
void* data_of(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

struct Sizes {
    int64_t starts = 0, workspace = 0;
    Sizes(const Tensor& x, int order) {
        sized("cl_recurrence_sizes", cl_recurrence_sizes(code_of(x), order, x.size(0), x.size(1),
                                                         x.size(2), &starts, &workspace));
    }
    Tensor allocate(const Tensor& x) const {
        return workspace ? at::empty({workspace}, x.options().dtype(at::kByte)) : Tensor();
    }
};

struct Swept {
    Tensor x, gate, y, last, starts;
    int order;
};

Swept swept(const Tensor& input, const Tensor& gates, const Tensor& state, int form, bool keep) {
    Swept r;
    r.order = order_of(input);
    r.x = input;
    if (r.order < 0) {
        r.x = input.contiguous();
        r.order = order_of(r.x);
    }
    r.gate = in_order(gates, r.order);
    r.y = sequence_like(r.x, r.order);
    r.last = state_like(r.x, r.order);
    const Sizes sizes(r.x, r.order);
    if (keep && sizes.starts) r.starts = at::empty({sizes.starts}, r.last.options());
    const Tensor ws = sizes.allocate(r.x);
    launch("cl_recurrence_forward", r.x.get_device(), [&](void* stream) {
        return cl_recurrence_forward(
            code_of(r.x), r.order, form, r.x.data_ptr(), strides_of(r.x), r.gate.data_ptr(),
            strides_of(r.gate), data_of(state), strides_of(state), r.x.size(0), r.x.size(1),
            r.x.size(2), r.y.data_ptr(), strides_of(r.y), r.last.data_ptr(), strides_of(r.last),
            data_of(r.starts), data_of(ws), sizes.workspace, stream);
    });
    return r;
}

struct Recurrence : Function<Recurrence> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& gate,
                                 const c10::optional<Tensor>& given, int64_t form) {
        const Tensor state = given.value_or(Tensor());
        Swept r = swept(x, gate, state, int(form), true);
        ctx->save_for_backward({r.x, r.gate, state, r.starts});
        ctx->saved_data["form"] = form;
        ctx->saved_data["order"] = int64_t(r.order);
        ctx->set_materialize_grads(false);
        return {r.y, r.last};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        if (at::GradMode::is_enabled())
            throw std::runtime_error("the gated recurrence cannot be differentiated twice");
        if (!grads[0].defined() && !grads[1].defined())
            return {Tensor(), Tensor(), Tensor(), Tensor()};
        const int form = int(ctx->saved_data["form"].toInt());
        const int order = int(ctx->saved_data["order"].toInt());
        const variable_list v = ctx->get_saved_variables();
        const c10::DeviceGuard guard(v[0].device());
        // (hooks on saved tensors may have moved them)
        const Tensor x = in_order(v[0], order), gate = in_order(v[1], order), state = v[2];
        const Tensor starts = v[3].defined() ? v[3].contiguous() : v[3];
        const Tensor gy = grads[0].defined() ? in_order(grads[0], order) : grads[0];
        const Tensor gl = grads[1];
        Tensor gx, gg, gs;
        if (ctx->needs_input_grad(0)) gx = sequence_like(x, order);
        if (ctx->needs_input_grad(1)) gg = sequence_like(x, order);
        if (state.defined() && ctx->needs_input_grad(2)) gs = state_like(x, order);
        const Sizes sizes(x, order);
        const Tensor ws = sizes.allocate(x);
        launch("cl_recurrence_backward", x.get_device(), [&](void* stream) {
            return cl_recurrence_backward(
                code_of(x), order, form, x.data_ptr(), strides_of(x), gate.data_ptr(),
                strides_of(gate), data_of(state), strides_of(state), data_of(starts), data_of(gy),
                strides_of(gy), data_of(gl), strides_of(gl), x.size(0), x.size(1), x.size(2),
                data_of(gx), strides_of(gx), data_of(gg), strides_of(gg), data_of(gs),
                strides_of(gs), data_of(ws), sizes.workspace, stream);
        });
        return {gx, gg, gs, Tensor()};
    }
};

// ---- what Python calls, with the arguments checked

// (Its arguments are checked here: for one step of a sequence the checks in Python took 1.5 of 7 us.)
std::string said(const Tensor& t) {
    std::string s = "[";
    for (const int64_t n : t.sizes()) s += (s.size() > 1 ? ", " : "") + std::to_string(n);
    return s + "] " + c10::toString(t.scalar_type());
}

std::pair<Tensor, Tensor> gated_recurrence(const Tensor& x, const Tensor& gate,
                                           const c10::optional<Tensor>& given, int64_t form) {
    const auto require = [](bool good, auto&& text) {
        if (!good) throw std::runtime_error(text());
    };
    require(x.is_cuda() && gate.device() == x.device(),
            [] { return std::string("x and gate must be on the same HIP device"); });
    const at::ScalarType type = x.scalar_type();
    require(type == at::kFloat || type == at::kDouble || type == at::kHalf || type == at::kBFloat16, [&] {
        return std::string("unsupported floating dtype ") + c10::toString(type) +
               "; the kernels take float16, bfloat16, float32 and float64";
    });
    require(x.dim() == 3 && gate.sizes() == x.sizes() && gate.scalar_type() == type, [&] {
        return "x and gate must be [batch, time, features] of one shape and dtype, got " + said(x) +
               " and " + said(gate);
    });
    require(x.layout() == at::kStrided && gate.layout() == at::kStrided,
            [] { return std::string("x and gate must be dense"); });
    const c10::DeviceGuard guard(x.device());
    const at::ScalarType wide = type == at::kDouble ? at::kDouble : at::kFloat;
    c10::optional<Tensor> state = given;
    if (given) {
        const Tensor& h = *given;
        require(h.device() == x.device() && h.dim() == 2 && h.size(0) == x.size(0) &&
                    h.size(1) == x.size(2) && at::isFloatingType(h.scalar_type()) &&
                    h.layout() == at::kStrided,
                [&] {
                    return "state must be a floating-point tensor of shape [" +
                           std::to_string(x.size(0)) + ", " + std::to_string(x.size(2)) +
                           "] on x's device, got " + said(h);
                });
        if (h.scalar_type() != wide) state = h.to(wide);
    }
    if (x.size(1) == 0)
        return {x.clone(),
                state ? state->clone() : at::zeros({x.size(0), x.size(2)}, x.options().dtype(wide))};
    const Tensor h0 = state.value_or(Tensor());
    // (a tensor with a tangent, which torch refuses there, need not require a gradient)
    const auto traced = [](const Tensor& t) {
        return t.defined() && ((at::GradMode::is_enabled() && t.requires_grad()) ||
                               t._fw_grad(0).defined());
    };
    if (traced(x) || traced(gate) || traced(h0)) {
        variable_list r = Recurrence::apply(x, gate, state, form);
        return {r[0], r[1]};
    }
    Swept r = swept(x, gate, h0, int(form), false);
    return {r.y, r.last};
}

Tensor selected_log_probs(const Tensor& x, const Tensor& actions, int64_t ignore, int64_t k,
                          double tau) {
    const c10::DeviceGuard guard(x.device());
    return LogProbs::apply(x, LogProbArgs{actions, ignore, Group{k, tau}});
}

std::pair<Tensor, Tensor> policy_loss(const Tensor& x, const Tensor& actions, const Tensor& old,
                                      const Tensor& adv, const c10::optional<Tensor>& ref,
                                      double low, double high, double kl, int64_t ignore,
                                      int reduction, bool prefill, int64_t k, double tau) {
    const c10::DeviceGuard guard(x.device());
    variable_list r = PolicyLoss::apply(x, PolicyArgs{actions, old, adv, ref, low, high, kl, ignore,
                                                      reduction, prefill, Group{k, tau}});
    return {r[0], r[1]};
}

std::pair<Tensor, Tensor> preference_loss(const Tensor& x, const Tensor& actions,
                                          const Tensor& offsets, const c10::optional<Tensor>& ref,
                                          double beta, double smoothing, int64_t ignore,
                                          int reduction, int64_t k, double tau) {
    const c10::DeviceGuard guard(x.device());
    variable_list r = PreferenceLoss::apply(x, PreferenceArgs{actions, offsets, ref, beta,
                                                              smoothing, ignore, reduction,
                                                              Group{k, tau}});
    return {r[0], r[1]};
}

Tensor dropout(const Tensor& x, int64_t threshold, c10::optional<double> fill, uint64_t seed,
               uint64_t offset, const c10::optional<Tensor>& rng) {
    const c10::DeviceGuard guard(x.device());
    return Drop::apply(x, DropArgs{threshold, fill, seed, offset, rng});
}

// The (seed, offset) of a module's next mask.
Tensor dropout_next(const Tensor& rng) {
    const c10::DeviceGuard guard(rng.device());
    Tensor used = at::empty({2}, rng.options());
    launch("cl_dropout_next", rng.get_device(), [&](void* stream) {
        return cl_dropout_next(static_cast<int64_t*>(rng.data_ptr()),
                               static_cast<int64_t*>(used.data_ptr()), stream);
    });
    return used;
}

// (tokens, accepted, log_probs) of logits [sequences, drafts + 1, cols]
std::tuple<Tensor, Tensor, Tensor> verify_drafts(const Tensor& logits, const Tensor& drafted,
                                                 const c10::optional<Tensor>& draft,
                                                 const Tensor& uniforms, int64_t ignore) {
    const c10::DeviceGuard guard(logits.device());
    const at::NoGradGuard no_grad;
    const int code = code_of(logits);
    const int64_t seqs = logits.size(0), drafts = drafted.size(1), cols = logits.size(2);
    auto rows = [&](const Tensor& t) {
        return cols > 1 && t.stride(2) != 1 ? t.contiguous() : t;
    };
    const Tensor p = rows(logits), q = draft ? rows(*draft) : Tensor();
    Tensor tokens = at::empty({seqs, drafts + 1}, drafted.options());
    Tensor accepted = at::empty({seqs}, drafted.options());
    Tensor lp = at::empty({seqs, drafts + 1}, wide_of(logits));
    int64_t need = 0;
    sized("cl_verify_drafts_workspace",
          cl_verify_drafts_workspace(code, seqs, drafts, cols, &need));
    const Tensor ws = need ? at::empty({need}, logits.options().dtype(at::kByte)) : Tensor();
    launch("cl_verify_drafts", logits.get_device(), [&](void* stream) {
        return cl_verify_drafts(
            code, p.data_ptr(), p.stride(0), p.stride(1), data_of(q), q.defined() ? q.stride(0) : 0,
            q.defined() ? q.stride(1) : 0, ints(drafted), ignore, uniforms.data_ptr(),
            code_of(uniforms), seqs, drafts, cols, static_cast<int64_t*>(tokens.data_ptr()),
            static_cast<int64_t*>(accepted.data_ptr()), lp.data_ptr(), data_of(ws), need, stream);
    });
    return {tokens, accepted, lp};
}

// ---- one AdamW step over the parameters of an optimizer.  The walk over its groups and states is here
// because a Python loop costs some 2 us a tensor, a small tensor's share of the kernels 0.1.

[[noreturn]] void refuse(const std::string& text) { throw std::runtime_error("FusedAdamW " + text); }

py::handle item_of(PyObject* dict, const char* name) {
    PyObject* v = PyDict_GetItemString(dict, name);
    return v ? v : Py_None;
}

// The state's tensor of that name as a kernel can take it (contiguous on the device, of the type and
// shape), else null.
const Tensor* held(PyObject* state, const char* name, const Tensor& p, at::ScalarType type,
                   bool shaped) {
    PyObject* v = PyDict_GetItemString(state, name);
    if (!v || !THPVariable_Check(v)) return nullptr;
    const Tensor& t = THPVariable_Unpack(v);
    if (t.scalar_type() != type || t.device() != p.device() || !t.is_contiguous() ||
        (shaped ? t.sizes() != p.sizes() : t.numel() != 2 * ((p.numel() + 255) / 256)))
        return nullptr;
    return &t;
}

// The parameter's moments in `out`; false where the state has none that fit.
bool moments_of(const Tensor& p, PyObject* state, int bits, cl_adamw_tensor& out) {
    const bool small = bits == 8;
    const at::ScalarType wide = p.scalar_type() == at::kDouble ? at::kDouble : at::kFloat;
    const Tensor* m = held(state, "exp_avg", p, small ? at::kFloat8_e4m3fn : wide, true);
    const Tensor* v = held(state, "exp_avg_sq", p, small ? at::kByte : wide, true);
    const Tensor* e = small ? held(state, "exponents", p, at::kByte, false) : nullptr;
    if (!m || !v || (small && !e)) return false;
    out.exp_avg = m->data_ptr();
    out.exp_avg_sq = v->data_ptr();
    out.powers = small ? static_cast<uint8_t*>(e->data_ptr()) : nullptr;
    out.numel = p.numel();
    out.bits = bits;
    return true;
}

int rounding_of(py::handle name) {
    const auto text = py::cast<std::string>(name);
    if (text == "nearest") return CL_ADAMW_NEAREST;
    if (text != "random") refuse("rounds moments to the \"nearest\" or at \"random\", not by \"" + text + "\"");
    return CL_ADAMW_AT_RANDOM;
}

// False, with nothing done, where a parameter with a gradient has no moments yet.
bool adamw_step(const py::list& param_groups, const py::dict& states, const Tensor& step,
                double max_norm) {
    const at::NoGradGuard no_grad;
    const c10::Device device = step.device();
    std::vector<cl_adamw_tensor> tensors;
    std::vector<cl_adamw_group> groups;
    std::vector<Tensor> copies;  // of gradients that are not contiguous
    std::vector<at::TensorImpl*> stepped;
    for (const py::handle group : param_groups) {
        const auto betas = py::cast<py::sequence>(item_of(group.ptr(), "betas"));
        const int bits = py::cast<int>(item_of(group.ptr(), "state_bits"));
        const int rounding = rounding_of(item_of(group.ptr(), "rounding"));
        const int64_t first = int64_t(tensors.size());
        for (const py::handle item : py::cast<py::list>(item_of(group.ptr(), "params"))) {
            const Tensor& p = THPVariable_Unpack(item.ptr());
            const Tensor& grad = p.grad();
            if (!grad.defined()) continue;
            if (grad.layout() != at::kStrided) refuse("does not support sparse gradients");
            if (p.device() != device) refuse("needs all parameters on one HIP device");
            if (!p.is_contiguous()) refuse("needs contiguous parameters");
            if (grad.scalar_type() != p.scalar_type() || grad.device() != device ||
                grad.sizes() != p.sizes())
                refuse("needs gradients of the parameters' dtype, shape and device");
            PyObject* state = PyDict_GetItem(states.ptr(), item.ptr());
            cl_adamw_tensor t{};
            if (!state || !moments_of(p, state, bits, t)) return false;
            t.param = p.data_ptr();
            if (grad.is_contiguous()) {
                t.grad = grad.data_ptr();
            } else {
                copies.push_back(grad.contiguous());
                t.grad = copies.back().data_ptr();
            }
            t.dtype = code_of(p);
            t.group = int(groups.size());
            t.rounding = rounding;
            tensors.push_back(t);
            stepped.push_back(p.unsafeGetTensorImpl());
        }
        if (int64_t(tensors.size()) == first) continue;
        groups.push_back({py::cast<double>(item_of(group.ptr(), "lr")), py::cast<double>(betas[0]),
                          py::cast<double>(betas[1]), py::cast<double>(item_of(group.ptr(), "eps")),
                          py::cast<double>(item_of(group.ptr(), "weight_decay"))});
    }
    if (tensors.empty()) return true;
    const c10::DeviceGuard guard(device);
    int64_t need = 0;
    sized("cl_adamw_workspace", cl_adamw_workspace(int64_t(tensors.size()), &need));
    const Tensor ws = at::empty({need}, step.options().dtype(at::kByte));
    launch("cl_adamw_step", device.index(), [&](void* stream) {
        return cl_adamw_step(int64_t(tensors.size()), tensors.data(), int64_t(groups.size()),
                             groups.data(), max_norm, static_cast<double*>(step.data_ptr()),
                             ws.data_ptr(), need, stream);
    });
    for (at::TensorImpl* p : stepped)
        if (!p->is_inference()) p->bump_version();  // autograd: what it saved of them is another now
    return true;
}

// 8-bit moments of the parameters, each with its state, taken in from fp32 tensors (write) or given
// back into bf16 ones.
void moments_between(const std::vector<Tensor>& params, const py::list& states,
                     const std::vector<Tensor>& first, const std::vector<Tensor>& second, bool write) {
    std::vector<cl_adamw_tensor> tensors;
    for (size_t i = 0; i < params.size(); ++i) {
        cl_adamw_tensor t{};
        if (params[i].device() != params[0].device() ||
            !moments_of(params[i], states[i].ptr(), 8, t))
            refuse("has no moments in 8 bits for a parameter");
        t.param = first[i].data_ptr();
        t.grad = second[i].data_ptr();
        tensors.push_back(t);
    }
    const c10::DeviceGuard guard(params[0].device());
    launch(write ? "cl_adamw_moments_write" : "cl_adamw_moments_read", params[0].get_device(),
           [&](void* stream) {
               return (write ? cl_adamw_moments_write : cl_adamw_moments_read)(
                   int64_t(tensors.size()), tensors.data(), stream);
           });
}

void adamw_hold(const Tensor& param, const py::dict& state, const Tensor& first, const Tensor& second) {
    py::list states;
    states.append(state);
    moments_between({param}, states, {first}, {second}, true);
}

std::pair<std::vector<Tensor>, std::vector<Tensor>> adamw_held(const std::vector<Tensor>& params,
                                                               const py::list& states) {
    std::vector<Tensor> first, second;
    if (params.empty()) return {first, second};
    for (const Tensor& p : params) {
        first.push_back(at::empty(p.sizes(), p.options().dtype(at::kBFloat16)));
        second.push_back(at::empty(p.sizes(), p.options().dtype(at::kBFloat16)));
    }
    moments_between(params, states, first, second, false);
    return {first, second};
}

void set_timed(py::object timed) { g_timed.set(std::move(timed)); }

}  // namespace

PYBIND11_MODULE(_autograd, m) {
    using unlocked = py::call_guard<py::gil_scoped_release>;
    m.def("selected_log_probs", &selected_log_probs, unlocked());
    m.def("policy_loss", &policy_loss, unlocked());
    m.def("preference_loss", &preference_loss, unlocked());
    m.def("gated_recurrence", &gated_recurrence, unlocked(), py::arg("x"), py::arg("gate"),
          py::arg("state"), py::arg("form"));
    m.def("verify_drafts", &verify_drafts, unlocked());
    m.def("dropout", &dropout, unlocked());
    m.def("dropout_next", &dropout_next, unlocked());
    m.def("adamw_step", &adamw_step);
    m.def("adamw_hold", &adamw_hold);
    m.def("adamw_held", &adamw_held);
    m.def("set_timed", &set_timed);
    m.attr("torch_version") = TORCH_VERSION;
}
