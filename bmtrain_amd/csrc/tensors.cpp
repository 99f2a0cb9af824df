// The operators between logits and optimizer as calls on tensors: argument checks, memory, autograd nodes and the C entries
// of include/bmt_hip.h behind them.  Small batches are bound by the host, and a backward pass runs on autograd's own thread,
// where Python costs twice what it does on the caller's.  With checks and nodes in Python / here: policy loss 8 x 512
// forward and backward 107 / 51 us (37 of them a native operation's), log-probabilities of 16 tokens 12.2 / 5.9 (the kernel
// bounds it now), 36 tensors clipped 26.5 / 17.7.
//
// Module bmtrain_amd._tensors.  Wrong arguments raise AssertionError or ValueError, a refused or failed launch
// RuntimeError.  Nothing here holds the interpreter's lock.
#include "../../include/bmt_hip.h"

#include <ATen/ATen.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <string>
#include <tuple>
#include <vector>

namespace {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
typedef std::optional<Tensor> MaybeTensor;

struct Assertion : torch::PyTorchError {
    using PyTorchError::PyTorchError;
    PyObject *python_type() override { return PyExc_AssertionError; }
};
struct Value : torch::PyTorchError {
    using PyTorchError::PyTorchError;
    PyObject *python_type() override { return PyExc_ValueError; }
};
void expect(bool holds, const char *text) {
    if (!holds) throw Assertion(text);
}
void expect(bool holds, const char *name, const char *text) {
    if (!holds) throw Assertion(std::string(name) + text);
}

const char *name_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return "torch.float32";
        case at::kHalf: return "torch.float16";
        case at::kBFloat16: return "torch.bfloat16";
        case at::kDouble: return "torch.float64";
        case at::kInt: return "torch.int32";
        case at::kLong: return "torch.int64";
        default: return c10::toString(t);
    }
}
// The type codes of the C entries; -1: none of them.
int32_t code_of(at::ScalarType t) { return t == at::kFloat ? 0 : t == at::kHalf ? 1 : t == at::kBFloat16 ? 2 : -1; }
int32_t type_code(const char *op, at::ScalarType t) {
    const int32_t code = code_of(t);
    if (code < 0) throw Value(std::string(op) + " not supported for dtype " + name_of(t));
    return code;
}

void *stream_of(const Tensor &t) { return (void *)c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
void launched(const char *who, int status) {
    TORCH_CHECK(status == 0, who, " failed with status ", status, ": ", bmt_hip_last_error());
}
Tensor floats(at::IntArrayRef shape, const Tensor &like) { return at::empty(shape, like.options().dtype(at::kFloat)); }
void *pointer(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

// Forward-mode derivatives would be lost without a word.
void no_tangent(const Tensor &t) {
    TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(), "forward-mode differentiation is not supported");
}

// `t` with its last dimension's elements next to each other (a copy where they are not).
Tensor tokens_adjacent(const Tensor &t) {
    if (t.is_neg()) return t.resolve_neg().contiguous();
    return t.dim() == 0 || t.is_contiguous() || t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous();
}
Tensor tokens_adjacent(const MaybeTensor &t) { return t ? tokens_adjacent(*t) : Tensor(); }
// An upstream gradient as the kernels read it: its numbers in memory, in order.  Complex arithmetic behind an operator hands
// back lazily negated ones, which contiguous() leaves negated.  The result has to live until its launch.
Tensor upstream_of(const Tensor &grad) {
    if (!grad.defined()) return Tensor();
    return grad.is_neg() ? grad.resolve_neg().contiguous() : grad.contiguous();
}
// A bool / uint8 mask as it is; anything else as mask != 0.
Tensor as_mask(const MaybeTensor &mask) {
    if (!mask) return Tensor();
    return tokens_adjacent(mask->scalar_type() == at::kBool || mask->scalar_type() == at::kByte ? *mask : mask->ne(0));
}

// Gradients that were computed outside of any graph: differentiating them again is an error, not a wrong result.
variable_list once_differentiable(variable_list &&out, const variable_list &grads) {
    if (!at::GradMode::is_enabled() ||
        std::none_of(grads.begin(), grads.end(), [](const Tensor &g) { return g.defined() && g.requires_grad(); }))
        return std::move(out);
    for (Tensor &t : out)
        if (t.defined()) t = t.detach().set_requires_grad(true);
    auto error = std::make_shared<torch::autograd::DelayedError>(
        "trying to differentiate twice a function that is differentiable once", (int)out.size());
    return (*error)(std::move(out));
}

bool wants_grad(const Tensor &t) { return at::GradMode::is_enabled() && t.defined() && t.requires_grad(); }

template <typename N>
std::shared_ptr<N> node_behind(const Tensor &a, const Tensor &b = Tensor()) {
    std::shared_ptr<N> node(new N(), torch::autograd::deleteNode);
    if (b.defined()) node->set_next_edges(torch::autograd::collect_next_edges(a, b));
    else node->set_next_edges(torch::autograd::collect_next_edges(a));
    return node;
}

// ---- token log-probabilities -------------------------------------------------------------------------------------------

// Logits [..., n]: at most two strides lead from row to row and the classes lie next to each other; a tensor laid out
// otherwise is copied first.
struct Rows {
    Tensor logits;
    int64_t rows, n, inner, outer_stride, inner_stride;
};
Rows rows_of(const Tensor &logits) {
    const int64_t dims = logits.dim(), n = logits.size(-1);
    if (dims > 3 || (n > 1 && logits.stride(-1) != 1) || logits.is_neg()) {
        const Tensor copy = logits.resolve_neg().contiguous();
        const int64_t rows = n ? copy.numel() / n : 0;
        return {copy, rows, n, std::max<int64_t>(rows, 1), 0, n};
    }
    if (dims == 1) return {logits, 1, n, 1, 0, n};
    if (dims == 2) return {logits, logits.size(0), n, std::max<int64_t>(logits.size(0), 1), 0, logits.stride(0)};
    return {logits, logits.size(0) * logits.size(1), n, std::max<int64_t>(logits.size(1), 1), logits.stride(0), logits.stride(1)};
}

struct TokenLogProbsBackward : Node {
    SavedVariable logits_, target_, stats_;
    int64_t ignore_index;
    float temperature;

    variable_list apply(variable_list &&grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        variable_list out(1);
        const bool of_entropy = grads.size() > 1 && grads[1].defined();
        if (!task_should_compute_output(0) || !(grads[0].defined() || of_entropy)) return out;
        const Tensor logits = logits_.unpack(), target = target_.unpack(), stats = stats_.unpack();
        {
            const at::NoGradGuard no_graph;
            const c10::DeviceGuard device(logits.device());
            const Rows r = rows_of(logits);
            const Tensor grad_logprob = upstream_of(grads[0]), grad_entropy = of_entropy ? upstream_of(grads[1]) : Tensor();
            out[0] = at::empty(logits.sizes(), logits.options().memory_format(at::MemoryFormat::Contiguous));
            launched("token_logprobs_backward_launcher",
                     token_logprobs_backward_launcher(r.rows, r.n, r.inner, r.outer_stride, r.inner_stride, r.logits.data_ptr(),
                                                      code_of(logits.scalar_type()), target.data_ptr(),
                                                      target.scalar_type() == at::kInt ? 32 : 64, ignore_index, temperature,
                                                      stats.data_ptr(), pointer(grad_logprob), pointer(grad_entropy),
                                                      out[0].data_ptr(), stream_of(logits)));
        }
        return once_differentiable(std::move(out), grads);
    }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        logits_.reset_data(), target_.reset_data(), stats_.reset_data();
    }
    std::string name() const override { return "TokenLogProbsBackward"; }
};

// (log-probabilities, entropies or None) of the tokens `target`.  Where a gradient is wanted the logits and four numbers
// per token are kept for it.
std::tuple<Tensor, MaybeTensor> token_logprobs(const Tensor &logits, const Tensor &target_in, int64_t ignore_index,
                                               double temperature, bool entropy) {
    expect(logits.dim() >= 1 && logits.sizes().slice(0, logits.dim() - 1) == target_in.sizes(),
           "target must have the shape of logits without its last dimension");
    expect(logits.is_cuda(), "logits must be on cuda");
    no_tangent(logits);
    const int32_t code = type_code("token_logprobs", logits.scalar_type());
    expect(target_in.device() == logits.device(), "target must be on the same cuda device as the logits");
    expect(target_in.scalar_type() == at::kInt || target_in.scalar_type() == at::kLong, "target must be an int or long tensor");
    const bool keep = wants_grad(logits);
    Tensor logprob, entropies, stats, target;
    {
        const at::NoGradGuard no_graph;
        const c10::DeviceGuard device(logits.device());
        const Rows r = rows_of(logits);
        expect(r.n > 0 || r.rows == 0, "logits must have at least one class");
        target = target_in.contiguous();
        logprob = floats(target.sizes(), logits);
        if (entropy) entropies = floats(target.sizes(), logits);
        if (keep) stats = floats({r.rows, 4}, logits);
        launched("token_logprobs_forward_launcher",
                 token_logprobs_forward_launcher(r.rows, r.n, r.inner, r.outer_stride, r.inner_stride, r.logits.data_ptr(), code,
                                                 target.data_ptr(), target.scalar_type() == at::kInt ? 32 : 64, ignore_index,
                                                 (float)temperature, logprob.data_ptr(), pointer(entropies), pointer(stats),
                                                 stream_of(logits)));
    }
    if (keep) {
        auto node = node_behind<TokenLogProbsBackward>(logits);
        node->logits_ = SavedVariable(logits, false);
        node->target_ = SavedVariable(target, false);
        node->stats_ = SavedVariable(stats, false);
        node->ignore_index = ignore_index, node->temperature = (float)temperature;
        torch::autograd::set_history(logprob, node);
        if (entropy) torch::autograd::set_history(entropies, node);
    }
    return {logprob, entropy ? MaybeTensor(entropies) : std::nullopt};
}

// ---- policy and preference losses -----------------------------------------------------------------------------------------

// Pointer and row stride of a [rows, time] tensor whose tokens lie next to each other; null and 0 for an undefined one.
struct Strided {
    const void *data = nullptr;
    int64_t row = 0;
    Strided(const char *name, const Tensor &t, const Tensor &like, at::ScalarType type) {
        if (!t.defined()) return;
        expect(t.device() == like.device(), name, " must be on the same cuda device as the other tensors");
        expect(t.sizes() == like.sizes(), name, " must have the shape of logprob");
        if (t.scalar_type() != type) throw Value(std::string(name) + " must have the dtype of logprob, " + name_of(type));
        data = t.data_ptr(), row = t.stride(0);
    }
};

struct PolicyLossBackward : Node {
    SavedVariable scratch_, mask_;
    int64_t rows, time, weights_at, saved_at;
    int32_t reduction;
    float entropy_coef;
    at::ScalarType type;
    bool masked;

    variable_list apply(variable_list &&grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        variable_list out(num_outputs());
        if (!grads[0].defined()) return out;
        const Tensor scratch = scratch_.unpack(), mask = masked ? mask_.unpack() : Tensor();
        {
            const at::NoGradGuard no_graph;
            const c10::DeviceGuard device(scratch.device());
            const Tensor upstream = upstream_of(grads[0]);
            for (size_t k = 0; k < out.size(); k++)
                if (task_should_compute_output(k)) out[k] = at::empty({rows, time}, scratch.options().dtype(type));
            const float *base = (const float *)scratch.data_ptr();
            launched("policy_loss_backward_launcher",
                     policy_loss_backward_launcher(rows, time, code_of(type), reduction, saved_at >= 0 ? base + saved_at : nullptr,
                                                   base + weights_at, upstream.data_ptr(), pointer(mask), masked ? mask.stride(0) : 0,
                                                   entropy_coef, pointer(out[0]), out.size() > 1 ? pointer(out[1]) : nullptr,
                                                   stream_of(scratch)));
        }
        return once_differentiable(std::move(out), grads);
    }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        scratch_.reset_data(), mask_.reset_data();
    }
    std::string name() const override { return "PolicyLossBackward"; }
};

// (loss, the five statistics).  The scratch of one call is one allocation: the workspace's doubles, the weights, and, where
// the log-probabilities' gradient is wanted, the derivative of every token.
std::tuple<Tensor, Tensor> policy_loss(const Tensor &logprob_in, const Tensor &old_in, const Tensor &advantages_in,
                                       const MaybeTensor &mask_in, const MaybeTensor &ref_in, const MaybeTensor &entropy_in,
                                       double clip_low, double clip_high, double dual_clip, double kl_coef, double entropy_coef,
                                       int32_t reduction) {
    expect(logprob_in.dim() == 2, "logprob must be [sequences, tokens]");
    Tensor advantages = advantages_in.detach();
    if (advantages.dim() == 2 && advantages.size(1) && (advantages.sizes() != logprob_in.sizes() || advantages.stride(1) == 0)) {
        expect(advantages.size(1) == 1 || advantages.sizes() == logprob_in.sizes(),
               "advantages must be one to a sequence or one to a token");
        advantages = advantages.select(1, 0);          // one to a sequence: [sequences, 1], or an expanded view
    }
    expect(logprob_in.is_cuda(), "tensors must be on cuda");
    const Tensor logprob = tokens_adjacent(logprob_in), entropy = tokens_adjacent(entropy_in);      // with their gradients
    no_tangent(logprob), no_tangent(entropy);
    const bool keep = wants_grad(logprob), entropy_grad = wants_grad(entropy);
    const at::ScalarType type = logprob.scalar_type();
    const int32_t code = type_code("policy_loss", type);
    const int64_t rows = logprob.size(0), time = logprob.size(1);
    Tensor loss, stats, scratch, mask;
    int64_t weights_at, saved_at = -1;
    {
        const at::NoGradGuard no_graph;
        const c10::DeviceGuard device(logprob.device());
        const Tensor old = tokens_adjacent(old_in), ref = tokens_adjacent(ref_in);
        mask = as_mask(mask_in);
        if (advantages.scalar_type() != at::kFloat) advantages = advantages.to(at::kFloat);
        advantages = advantages.dim() == 2 ? tokens_adjacent(advantages) : advantages.resolve_neg();
        const bool per_token = advantages.dim() == 2;
        expect(per_token ? advantages.sizes() == logprob.sizes() : advantages.dim() == 1 && advantages.size(0) == rows,
               "advantages must be one to a sequence or one to a token");
        expect(advantages.device() == logprob.device(), "advantages must be on the same cuda device as the other tensors");
        const Strided l("logprob", logprob, logprob, type), o("old_logprob", old, logprob, type), f("ref_logprob", ref, logprob, type),
            e("entropy", entropy, logprob, type), m("mask", mask, logprob, mask.defined() ? mask.scalar_type() : at::kBool);
        weights_at = 2 * policy_loss_workspace_doubles(rows, time);
        int64_t size = weights_at + (reduction == 1 ? 1 + rows : 1);
        if (keep) {
            saved_at = (size + 3) / 4 * 4;
            size = saved_at + rows * time;
        }
        loss = floats({}, logprob), stats = floats({5}, logprob), scratch = floats({size}, logprob);
        float *base = (float *)scratch.data_ptr();
        launched("policy_loss_forward_launcher",
                 policy_loss_forward_launcher(rows, time, code, l.data, l.row, o.data, o.row, f.data, f.row, e.data, e.row,
                                              advantages.data_ptr(), advantages.stride(0), per_token, m.data, m.row, clip_low,
                                              clip_high, dual_clip, (float)kl_coef, (float)entropy_coef, reduction,
                                              keep ? base + saved_at : nullptr, base + weights_at, base, loss.data_ptr(),
                                              stats.data_ptr(), stream_of(logprob)));
    }
    if (keep || entropy_grad) {
        auto node = node_behind<PolicyLossBackward>(logprob, entropy);
        node->scratch_ = SavedVariable(scratch, false);
        node->masked = mask.defined();
        if (node->masked) node->mask_ = SavedVariable(mask, false);
        node->rows = rows, node->time = time, node->weights_at = weights_at, node->saved_at = saved_at;
        node->reduction = reduction, node->entropy_coef = (float)entropy_coef, node->type = type;
        torch::autograd::set_history(loss, node);
    }
    return {loss, stats};
}

struct PreferenceLossBackward : Node {
    SavedVariable scratch_, mask_;
    int64_t pairs, time, slope_at;
    at::ScalarType type;
    bool masked;

    variable_list apply(variable_list &&grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        variable_list out(1);
        if (!grads[0].defined() || !task_should_compute_output(0)) return out;
        const Tensor scratch = scratch_.unpack(), mask = masked ? mask_.unpack() : Tensor();
        {
            const at::NoGradGuard no_graph;
            const c10::DeviceGuard device(scratch.device());
            const Tensor upstream = upstream_of(grads[0]);
            out[0] = at::empty({2 * pairs, time}, scratch.options().dtype(type));
            launched("preference_loss_backward_launcher",
                     preference_loss_backward_launcher(pairs, time, code_of(type), (const float *)scratch.data_ptr() + slope_at,
                                                       upstream.data_ptr(), pointer(mask), masked ? mask.stride(0) : 0,
                                                       out[0].data_ptr(), stream_of(scratch)));
        }
        return once_differentiable(std::move(out), grads);
    }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        scratch_.reset_data(), mask_.reset_data();
    }
    std::string name() const override { return "PreferenceLossBackward"; }
};

// (loss, rewards of the chosen answers, rewards of the rejected ones).  Scratch: the workspace's doubles, then one slope per
// row behind their common factor.
std::tuple<Tensor, Tensor, Tensor> preference_loss(const Tensor &logprob_in, const MaybeTensor &ref_in, const MaybeTensor &mask_in,
                                                   int32_t kind, bool average, double beta, double label_smoothing) {
    const bool sums = logprob_in.dim() == 1;           // sums per row: one token each
    auto column = [&](const MaybeTensor &t) { return t && sums && t->dim() == 1 ? MaybeTensor(t->unsqueeze(1)) : t; };
    const Tensor logprob = tokens_adjacent(sums ? logprob_in.unsqueeze(1) : logprob_in);             // with its gradient
    expect(logprob.dim() == 2 && logprob.size(0) % 2 == 0, "logprob must be [2 * pairs, tokens]");
    expect(logprob.is_cuda(), "tensors must be on cuda");
    no_tangent(logprob);
    const at::ScalarType type = logprob.scalar_type();
    const int32_t code = type_code("preference_loss", type);
    const int64_t pairs = logprob.size(0) / 2, time = logprob.size(1);
    const bool keep = wants_grad(logprob);
    Tensor loss, chosen, rejected, scratch, mask;
    int64_t slope_at;
    {
        const at::NoGradGuard no_graph;
        const c10::DeviceGuard device(logprob.device());
        const Tensor ref = tokens_adjacent(column(ref_in));
        mask = as_mask(column(mask_in));
        const Strided l("logprob", logprob, logprob, type), f("ref_logprob", ref, logprob, type),
            m("mask", mask, logprob, mask.defined() ? mask.scalar_type() : at::kBool);
        slope_at = 2 * preference_loss_workspace_doubles(pairs, time);
        loss = floats({}, logprob), chosen = floats({pairs}, logprob), rejected = floats({pairs}, logprob);
        scratch = floats({slope_at + 1 + 2 * pairs}, logprob);
        float *base = (float *)scratch.data_ptr();
        launched("preference_loss_forward_launcher",
                 preference_loss_forward_launcher(pairs, time, code, l.data, l.row, f.data, f.row, m.data, m.row, kind, average, beta,
                                                  label_smoothing, base, loss.data_ptr(), chosen.data_ptr(), rejected.data_ptr(),
                                                  base + slope_at, stream_of(logprob)));
    }
    if (keep) {
        auto node = node_behind<PreferenceLossBackward>(logprob);
        node->scratch_ = SavedVariable(scratch, false);
        node->masked = mask.defined();
        if (node->masked) node->mask_ = SavedVariable(mask, false);
        node->pairs = pairs, node->time = time, node->slope_at = slope_at, node->type = type;
        torch::autograd::set_history(loss, node);
    }
    return {loss, chosen, rejected};
}

// ---- lists of gradients ----------------------------------------------------------------------------------------------------

// True if the elements fill one run of memory without gaps, in whatever order of dimensions.
bool is_dense(const Tensor &t) { return t.numel() == 0 || t.is_non_overlapping_and_dense(); }

// SIGNS: a lazily negated gradient or output is refused.
template <bool SIGNS>
std::vector<bmt_clip_tensor> clip_table(const std::vector<Tensor> &grads, const std::vector<Tensor> &outs) {
    std::vector<bmt_clip_tensor> table(grads.size());
    auto type = [](const Tensor &t) {
        const int32_t code = code_of(t.scalar_type());
        if (code < 0) throw Value(std::string("gradients must be fp32, fp16 or bf16, not ") + name_of(t.scalar_type()));
        return code;
    };
    for (size_t k = 0; k < grads.size(); k++) {
        const Tensor &g = grads[k], &o = outs[k];
        bmt_clip_tensor &row = table[k];
        row.src_type = type(g), row.dst_type = type(o);
        expect(g.is_cuda() && g.device() == grads[0].device() && o.device() == g.device(), "gradients must be on one cuda device");
        expect(o.numel() == g.numel(), "outputs must have their gradients' numbers of elements");
        expect(!SIGNS || (!g.is_neg() && !o.is_neg()), "gradients must not be lazily negated");
        expect(is_dense(g), "gradients must not have gaps nor elements that share memory");
        expect((g.is_contiguous() && o.is_contiguous()) || (g.sizes() == o.sizes() && g.strides() == o.strides()),
               "outputs must have their gradients' strides");
        row.src = g.data_ptr(), row.dst = o.data_ptr(), row.n = g.numel();
    }
    return table;
}

// What an in-place operation refuses where a graph is recorded: a write into a leaf or a view of one would be no part of it.
void may_be_written(const Tensor &t) {
    TORCH_CHECK(!t.requires_grad() || (!t.is_leaf() && !(t.is_view() && t._base().is_leaf())),
                "a leaf that requires a gradient, or a view of one, is written under torch.no_grad() only");
}

// Clips `grads` into `outs` (None: in place) and returns their norm.
Tensor clip_grads(const std::vector<Tensor> &grads, const std::optional<std::vector<Tensor>> &outs_in, double max_norm, bool use_max,
                  double eps, double scale) {
    const std::vector<Tensor> &outs = outs_in ? *outs_in : grads;
    expect(!grads.empty() && outs.size() == grads.size(), "as many outputs as gradients, at least one");
    if (at::GradMode::is_enabled())
        for (const Tensor &o : outs) may_be_written(o);
    const std::vector<bmt_clip_tensor> table = clip_table<true>(grads, outs);
    const int32_t count = (int32_t)table.size();
    const c10::DeviceGuard device(grads[0].device());
    const Tensor result = floats({2}, grads[0]);
    const Tensor work = at::empty({grad_norm_workspace_doubles(count, table.data())}, grads[0].options().dtype(at::kDouble));
    float *norm_and_factor = (float *)result.data_ptr();
    void *stream = stream_of(grads[0]);
    launched("grad_norm_multi_launcher",
             grad_norm_multi_launcher(count, table.data(), use_max, max_norm, eps, scale, work.data_ptr(), norm_and_factor, stream));
    launched("grad_scale_multi_launcher", grad_scale_multi_launcher(count, table.data(), norm_and_factor + 1, 0, stream));
    for (const Tensor &o : outs)                       // autograd is to notice the write, as with any in-place operation
        if (!o.is_inference()) o.unsafeGetTensorImpl()->bump_version();
    return result.select(0, 0);
}

// Every gradient times the factor rounded to its type, if the factor (one float on the GPU) is below one.  In place the
// product rounds alike under either sign, so a lazily negated gradient is scaled in memory as it is.
void scale_grads(const std::vector<Tensor> &grads, const Tensor &coef) {
    expect(coef.is_cuda() && coef.scalar_type() == at::kFloat && coef.numel() == 1, "coef must be one float on cuda");
    if (grads.empty()) return;
    const std::vector<bmt_clip_tensor> table = clip_table<false>(grads, grads);
    expect(grads[0].device() == coef.device(), "gradients and coef must be on one cuda device");
    const c10::DeviceGuard device(coef.device());
    launched("grad_scale_multi_launcher",
             grad_scale_multi_launcher((int32_t)table.size(), table.data(), coef.data_ptr(), 1, stream_of(coef)));
}

}  // namespace

PYBIND11_MODULE(_tensors, m) {
    namespace py = pybind11;
    using torch::wrap_pybind_function_no_gil;
    m.def("token_logprobs", wrap_pybind_function_no_gil(token_logprobs), py::arg("logits"), py::arg("target"), py::arg("ignore_index"),
          py::arg("temperature"), py::arg("entropy"));
    // for callers of the C entries: (logits or their copy, rows, n, inner, outer_stride, inner_stride)
    m.def("row_layout", wrap_pybind_function_no_gil([](const Tensor &logits) {
              const Rows r = rows_of(logits);
              return std::make_tuple(r.logits, r.rows, r.n, r.inner, r.outer_stride, r.inner_stride);
          }));
    m.def("policy_loss", wrap_pybind_function_no_gil(policy_loss), py::arg("logprob"), py::arg("old_logprob"), py::arg("advantages"),
          py::arg("mask"), py::arg("ref_logprob"), py::arg("entropy"), py::arg("clip_low"), py::arg("clip_high"), py::arg("dual_clip"),
          py::arg("kl_coef"), py::arg("entropy_coef"), py::arg("reduction"));
    m.def("preference_loss", wrap_pybind_function_no_gil(preference_loss), py::arg("logprob"), py::arg("ref_logprob"), py::arg("mask"),
          py::arg("kind"), py::arg("average"), py::arg("beta"), py::arg("label_smoothing"));
    m.def("is_dense", wrap_pybind_function_no_gil(is_dense));
    m.def("clip_grads", wrap_pybind_function_no_gil(clip_grads), py::arg("grads"), py::arg("outs"), py::arg("max_norm"),
          py::arg("use_max"), py::arg("eps"), py::arg("scale"));
    m.def("scale_grads", wrap_pybind_function_no_gil(scale_grads), py::arg("grads"), py::arg("coef"));
}
