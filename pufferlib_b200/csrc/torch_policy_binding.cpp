// PyTorch operators of the policy update, with their gradients.
//
// Adds to the `pufferlib` operator library of torch_binding.cpp what follows the advantages in the trainer: the
// log-probability and entropy of chosen actions (sample_logits of pufferlib/pytorch.py), the clipped policy loss
// (pufferl.py:390-411, 422) and the gated linear recurrence along the horizon.  No arithmetic here: tensors are
// checked, buffers allocated, and the C ABI of include/puff_advantage.h is called on the current stream of the
// tensors' device.
//
// Each differentiable operator has an autograd kernel whose node keeps what the backward operator needs and calls it (nodes
// of their own rather than torch::autograd::Function, whose context costs several microseconds a pass at the host).  A
// node unpacks what it kept before it goes below autograd: saved-tensor hooks run then, and those of activation
// checkpointing compute a whole region again.
// The *_forward and *_backward operators can be called without autograd (for a program that captures a whole update
// into a CUDA graph); their results are not differentiable, and a second derivative raises.  So does a forward-mode
// derivative: a node like these has none, and its tangent would be lost.
#include <ATen/cuda/CUDAContext.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/all.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/library.h>

#include <optional>
#include <string>
#include <tuple>

#include "../../include/puff_advantage.h"

namespace pufferlib_b200 {
namespace {

using torch::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

void check_rc(int rc, const char* what)
{
    TORCH_CHECK(rc == PUFF_OK, what, ": ", puff_advantage_sm100_strerror(rc), " (code ", rc, ")");
}

int dtype_code(const Tensor& t, const char* name)
{
    switch (t.scalar_type()) {
        case torch::kFloat32: return PUFF_DTYPE_F32;
        case torch::kFloat16: return PUFF_DTYPE_F16;
        case torch::kBFloat16: return PUFF_DTYPE_BF16;
        default: TORCH_CHECK(false, name, " must be float32, float16 or bfloat16, got ", t.scalar_type());
    }
}

// A tensor's sizes as numbers, for the CUDA kernels, or as what may be symbols, for the Meta kernels, which also run while a
// program is traced for sizes that change.
template <typename I> struct Dims;
template <> struct Dims<int64_t> {
    using Ref = at::IntArrayRef;
    static Ref sizes(const Tensor& t) { return t.sizes(); }
    static Ref strides(const Tensor& t) { return t.strides(); }
    static int64_t numel(const Tensor& t) { return t.numel(); }
    static Tensor empty(Ref sizes, const at::TensorOptions& o) { return torch::empty(sizes, o); }
};
template <> struct Dims<c10::SymInt> {
    using Ref = c10::SymIntArrayRef;
    static Ref sizes(const Tensor& t) { return t.sym_sizes(); }
    static Ref strides(const Tensor& t) { return t.sym_strides(); }
    static c10::SymInt numel(const Tensor& t) { return t.sym_numel(); }
    static Tensor empty(Ref sizes, const at::TensorOptions& o) { return at::empty_symint(sizes, o); }
};

template <typename I>
void check_f32(const Tensor& t, const Tensor& like, typename Dims<I>::Ref sizes, const char* name)
{
    TORCH_CHECK(t.device() == like.device(), "All tensors must be on same device");
    TORCH_CHECK(t.scalar_type() == torch::kFloat32, name, " must be float32");
    TORCH_CHECK(Dims<I>::sizes(t) == sizes, name, " must have shape ", sizes, ", got ", Dims<I>::sizes(t));
    TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}
void check_f32(const Tensor& t, const Tensor& like, at::IntArrayRef sizes, const char* name) { check_f32<int64_t>(t, like, sizes, name); }

template <typename T> T* ptr(const Tensor& t) { return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr; }
template <typename T> const T* ptr(const OptTensor& t) { return t.has_value() && t->defined() ? static_cast<const T*>(t->data_ptr()) : nullptr; }
bool present(const OptTensor& t) { return t.has_value() && t->defined(); }
OptTensor optional(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }
cudaStream_t current_stream() { return at::cuda::getCurrentCUDAStream().stream(); }

template <typename N> std::shared_ptr<N> new_node(torch::autograd::edge_list&& edges)
{
    std::shared_ptr<N> node(new N(), torch::autograd::deleteNode);
    node->set_next_edges(std::move(edges));
    return node;
}
// Where a backward pass builds a graph, its results hang on this node, with every input of the operator and every incoming
// gradient behind it: whichever of them a second derivative is asked for, it raises.
struct NoSecondDerivative : public Node {
    const char* what = "";
    std::string name() const override { return "PuffNoSecondDerivative"; }
    variable_list apply(variable_list&&) override { TORCH_CHECK(false, what, " has no second derivative"); }
};
variable_list refuse_second_derivatives(const char* what, const Node& node, const variable_list& grads, variable_list&& results)
{
    if (!at::GradMode::is_enabled()) return std::move(results);
    torch::autograd::edge_list edges = node.next_edges();
    for (const Tensor& g : grads)
        if (g.defined() && g.requires_grad()) edges.push_back(torch::autograd::impl::gradient_edge(g));
    auto refuse = new_node<NoSecondDerivative>(std::move(edges));
    refuse->what = what;
    for (const Tensor& r : results)
        if (r.defined()) torch::autograd::set_history(r, refuse);
    return std::move(results);
}
bool dual(const Tensor& t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }
bool dual(const OptTensor& t) { return t.has_value() && dual(*t); }
template <typename... Tensors> void refuse_forward_mode(const char* what, const Tensors&... tensors)
{
    TORCH_CHECK(!((dual(tensors) || ...) && c10::AutogradState::get_tls_state().get_fw_grad_mode()), what,
                " has no forward-mode derivative");
}
SavedVariable saved(const OptTensor& t) { return present(t) ? SavedVariable(*t, false) : SavedVariable(); }

// ---- log-probabilities ------------------------------------------------------------------------------------------

// The leading sizes of a tensor as rows [outer, inner] with one stride each
template <typename I> struct Rows {
    I outer = 1, inner = 1, outer_stride = 0, inner_stride = 0;
};
template <typename I> Rows<I> rows_of(const Tensor& t, int64_t lead, const char* name)
{
    Rows<I> r;
    const auto sizes = Dims<I>::sizes(t), strides = Dims<I>::strides(t);
    bool second = false;
    // from the innermost leading dimension outwards: one that continues the run so far is folded into it
    for (int64_t d = lead - 1; d >= 0; --d) {
        const I &n = sizes[d], &s = strides[d];
        if (n == 1) continue;
        if (!second && (r.inner == 1 || s == r.inner * r.inner_stride)) {
            if (r.inner == 1) r.inner_stride = s;
            r.inner *= n;
        } else if (r.outer == 1 || s == r.outer * r.outer_stride) {
            if (r.outer == 1) r.outer_stride = s;
            r.outer *= n;
            second = true;
        } else {
            TORCH_CHECK(false, name, " has more than two runs of rows that a stride separates; make it contiguous");
        }
    }
    return r;
}
// logits and actions must be cut into [outer, inner] alike
template <typename I> void rows_alike(Rows<I>& a, Rows<I>& b, const char* what)
{
    if (a.inner == b.inner) return;
    Rows<I>& coarse = a.inner > b.inner ? a : b;
    const Rows<I>& fine = a.inner > b.inner ? b : a;
    TORCH_CHECK(coarse.outer == 1 && fine.inner > 0 && coarse.inner % fine.inner == 0, what,
                " must be cut into rows alike; make one of them contiguous");
    coarse.outer = coarse.inner / fine.inner;
    coarse.outer_stride = coarse.inner_stride * fine.inner;
    coarse.inner = fine.inner;
}

template <typename I> struct LogprobArgs {
    int dtype;
    I vocab, rows;
    Rows<I> l, a;
};
template <typename I> LogprobArgs<I> logprob_args(const Tensor& logits, const Tensor& actions)
{
    LogprobArgs<I> g;
    g.dtype = dtype_code(logits, "logits");
    TORCH_CHECK(logits.dim() >= 1, "logits must have at least one dimension");
    TORCH_CHECK(actions.scalar_type() == torch::kInt64, "actions must be int64");
    TORCH_CHECK(actions.device() == logits.device(), "All tensors must be on same device");
    const int64_t lead = logits.dim() - 1;
    const auto sizes = Dims<I>::sizes(logits);
    TORCH_CHECK(Dims<I>::sizes(actions) == sizes.slice(0, lead), "actions must have the shape of logits without its last dimension");
    g.vocab = sizes[lead];
    g.rows = Dims<I>::numel(actions);
    TORCH_CHECK(g.vocab > 0 || g.rows == 0, "logits must have at least one entry per row");
    TORCH_CHECK(g.vocab <= 1 || Dims<I>::strides(logits)[lead] == 1, "the last dimension of logits must be contiguous");
    if (g.rows > 0) {
        g.l = rows_of<I>(logits, lead, "logits");
        g.a = rows_of<I>(actions, lead, "actions");
        rows_alike<I>(g.l, g.a, "logits and actions");
    }
    return g;
}

// (logprobs, entropy or an empty tensor, row_stats or an empty tensor; undefined tensors for those with `bare`)
template <typename I>
bool stats_saved(const I& vocab) { return vocab > PUFF_LOGPROBS_STATS_ABOVE; }
template <typename I>
std::tuple<Tensor, Tensor, Tensor> logprobs_buffers(const Tensor& logits, const Tensor& actions, double temperature,
                                                    bool want_entropy, bool save, bool bare)
{
    TORCH_CHECK(temperature > 0, "temperature must be positive");
    const auto opts = logits.options().dtype(torch::kFloat32);
    const auto sizes = Dims<I>::sizes(actions);
    return {Dims<I>::empty(sizes, opts), want_entropy ? Dims<I>::empty(sizes, opts) : bare ? Tensor() : torch::empty({0}, opts),
            save && stats_saved<I>(Dims<I>::sizes(logits)[logits.dim() - 1]) ? Dims<I>::empty({Dims<I>::numel(actions), 2}, opts)
            : bare                                                           ? Tensor()
                                                                             : torch::empty({0, 2}, opts)};
}
std::tuple<Tensor, Tensor, Tensor> logprobs_forward_meta(const Tensor& logits, const Tensor& actions, double temperature,
                                                         bool want_entropy, bool save)
{
    logprob_args<c10::SymInt>(logits, actions);
    return logprobs_buffers<c10::SymInt>(logits, actions, temperature, want_entropy, save, false);
}
std::tuple<Tensor, Tensor, Tensor> logprobs_run(const Tensor& logits, const Tensor& actions, double temperature,
                                                bool want_entropy, bool save, bool bare)
{
    const auto g = logprob_args<int64_t>(logits, actions);
    const c10::cuda::CUDAGuard guard(logits.device());
    auto out = logprobs_buffers<int64_t>(logits, actions, temperature, want_entropy, save, bare);
    if (g.rows == 0) return out;
    check_rc(puff_policy_sm100_logprobs(logits.data_ptr(), g.dtype, ptr<const long long>(actions), g.l.outer, g.l.inner,
                                        g.vocab, g.l.outer_stride, g.l.inner_stride, g.a.outer_stride, g.a.inner_stride,
                                        static_cast<float>(temperature), ptr<float>(std::get<0>(out)),
                                        want_entropy ? ptr<float>(std::get<1>(out)) : nullptr,
                                        save && stats_saved(g.vocab) ? ptr<float>(std::get<2>(out)) : nullptr, current_stream()),
             "puff_action_logprobs");
    return out;
}
std::tuple<Tensor, Tensor, Tensor> logprobs_forward_cuda(const Tensor& logits, const Tensor& actions, double temperature,
                                                         bool want_entropy, bool save)
{
    return logprobs_run(logits, actions, temperature, want_entropy, save, false);
}
std::tuple<Tensor, Tensor, Tensor> logprobs_forward(const Tensor& logits, const Tensor& actions, double temperature,
                                                    bool want_entropy, bool save)
{
    static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("pufferlib::puff_action_logprobs_forward", "")
                         .typed<decltype(logprobs_forward_meta)>();
    return op.call(logits, actions, temperature, want_entropy, save);
}
std::tuple<Tensor, Tensor> action_logprobs_cuda(const Tensor& logits, const Tensor& actions, double temperature, bool want_entropy)
{
    // without entropy an undefined tensor, None in Python, here and below: an empty one would cost a tenth of a small call
    auto [logprobs, entropy, stats] = logprobs_run(logits, actions, temperature, want_entropy, false, true);
    return {logprobs, entropy};
}
std::tuple<Tensor, Tensor> action_logprobs_meta(const Tensor& logits, const Tensor& actions, double temperature, bool want_entropy)
{
    auto out = logprobs_forward_meta(logits, actions, temperature, want_entropy, false);
    return {std::get<0>(out), want_entropy ? std::get<1>(out) : Tensor()};
}
std::tuple<Tensor, Tensor> action_logprobs(const Tensor& logits, const Tensor& actions, double temperature, bool want_entropy)
{
    static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("pufferlib::puff_action_logprobs", "")
                         .typed<decltype(action_logprobs_meta)>();
    return op.call(logits, actions, temperature, want_entropy);
}

Tensor logprobs_backward_meta(const Tensor& logits, const Tensor& actions, double, const Tensor&, const OptTensor&,
                              const Tensor&, const OptTensor&)
{
    logprob_args<c10::SymInt>(logits, actions);
    return at::empty_symint(logits.sym_sizes(), logits.options());
}
Tensor logprobs_backward_cuda(const Tensor& logits, const Tensor& actions, double temperature, const Tensor& row_stats,
                              const OptTensor& entropy, const Tensor& dlogprobs, const OptTensor& dentropy)
{
    const auto g = logprob_args<int64_t>(logits, actions);
    check_f32(row_stats, logits, {stats_saved(g.vocab) ? g.rows : 0, 2}, "row_stats");
    // where they are not read, some address that is none of the output's
    const float* stats = stats_saved(g.vocab) ? ptr<const float>(row_stats) : ptr<const float>(actions);
    check_f32(dlogprobs, logits, actions.sizes(), "dlogprobs");
    if (present(dentropy)) {
        TORCH_CHECK(present(entropy), "dentropy needs the entropy of the forward pass");
        check_f32(*dentropy, logits, actions.sizes(), "dentropy");
        check_f32(*entropy, logits, actions.sizes(), "entropy");
    }
    const c10::cuda::CUDAGuard guard(logits.device());
    Tensor dlogits = torch::empty(logits.sizes(), logits.options());
    if (g.rows == 0) return dlogits;
    check_rc(puff_policy_sm100_logprobs_backward(
                 logits.data_ptr(), g.dtype, ptr<const long long>(actions), g.l.outer, g.l.inner, g.vocab,
                 g.l.outer_stride, g.l.inner_stride, g.a.outer_stride, g.a.inner_stride, static_cast<float>(temperature),
                 stats, present(dentropy) ? ptr<float>(entropy) : nullptr,
                 ptr<const float>(dlogprobs), ptr<float>(dentropy), dlogits.data_ptr(), current_stream()),
             "puff_action_logprobs_backward");
    return dlogits;
}
Tensor logprobs_backward(const Tensor& logits, const Tensor& actions, double temperature, const Tensor& row_stats,
                         const OptTensor& entropy, const Tensor& dlogprobs, const OptTensor& dentropy)
{
    static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("pufferlib::puff_action_logprobs_backward", "")
                         .typed<decltype(logprobs_backward_meta)>();
    return op.call(logits, actions, temperature, row_stats, entropy, dlogprobs, dentropy);
}

struct LogprobsNode : public Node {
    SavedVariable logits, actions, row_stats, entropy;
    double temperature = 1.0;
    std::string name() const override { return "PuffActionLogprobsBackward"; }
    void release_variables() override
    {
        std::lock_guard<std::mutex> lock(mutex_);
        for (SavedVariable* v : {&logits, &actions, &row_stats, &entropy}) v->reset_data();
    }
    variable_list apply(variable_list&& grads) override
    {
        std::lock_guard<std::mutex> lock(mutex_);
        if ((!grads[0].defined() && !grads[1].defined()) || !task_should_compute_output(0)) return {Tensor()};
        refuse_forward_mode("the backward pass of puff_action_logprobs", grads[0], grads[1]);
        const Tensor z = logits.unpack(), a = actions.unpack(), stats = row_stats.unpack();
        const OptTensor h = optional(entropy.unpack(shared_from_this()));
        Tensor dlogits;
        {
            at::AutoDispatchBelowADInplaceOrView below;
            const Tensor dlp = grads[0].defined() ? grads[0].contiguous() : torch::zeros_like(grads[1], at::MemoryFormat::Contiguous);
            const OptTensor dh = grads[1].defined() ? OptTensor(grads[1].contiguous()) : std::nullopt;
            dlogits = logprobs_backward(z, a, temperature, stats, h, dlp, dh);
        }
        return refuse_second_derivatives("puff_action_logprobs", *this, grads, {dlogits});
    }
};
std::tuple<Tensor, Tensor> action_logprobs_autograd(const Tensor& logits, const Tensor& actions, double temperature,
                                                    bool want_entropy)
{
    refuse_forward_mode("puff_action_logprobs", logits);
    if (!(at::GradMode::is_enabled() && logits.requires_grad())) {
        at::AutoDispatchBelowADInplaceOrView below;
        return action_logprobs(logits, actions, temperature, want_entropy);
    }
    auto node = new_node<LogprobsNode>(torch::autograd::collect_next_edges(logits));
    Tensor logprobs, entropy, stats;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        std::tie(logprobs, entropy, stats) = logprobs_forward(logits, actions, temperature, want_entropy, true);
    }
    torch::autograd::set_history(logprobs, node);
    if (want_entropy) torch::autograd::set_history(entropy, node);
    else node->add_input_metadata(Node::undefined_input());
    node->logits = SavedVariable(logits, false);
    node->actions = SavedVariable(actions, false);
    node->row_stats = SavedVariable(stats, false);
    if (want_entropy) node->entropy = SavedVariable(entropy, true);
    node->temperature = temperature;
    return {logprobs, want_entropy ? entropy : Tensor()};
}

// ---- policy loss -------------------------------------------------------------------------------------------------

int reduction_code(c10::string_view reduction)
{
    TORCH_CHECK(reduction == "token" || reduction == "sequence", "reduction must be \"token\" or \"sequence\"");
    return reduction == "token" ? PUFF_MEAN_TOKENS : PUFF_MEAN_SEQUENCES;
}
// one advantage per row?
template <typename I>
bool loss_args(const Tensor& logprobs, const Tensor& old_logprobs, const Tensor& advantages, const OptTensor& ref_logprobs,
               const OptTensor& entropy, const OptTensor& mask, double clip_low, double clip_high, double denominator)
{
    TORCH_CHECK(logprobs.dim() == 2, "logprobs must be 2D [rows, steps]");
    const auto sizes = Dims<I>::sizes(logprobs);
    check_f32<I>(logprobs, logprobs, sizes, "logprobs");
    check_f32<I>(old_logprobs, logprobs, sizes, "old_logprobs");
    const I &rows = sizes[0], &steps = sizes[1];
    const bool per_row = advantages.dim() == 1 || (advantages.dim() == 2 && Dims<I>::sizes(advantages)[1] == 1 && steps != 1);
    if (per_row && advantages.dim() == 2) check_f32<I>(advantages, logprobs, {rows, 1}, "advantages");
    else if (per_row) check_f32<I>(advantages, logprobs, {rows}, "advantages");
    else check_f32<I>(advantages, logprobs, sizes, "advantages");
    if (present(ref_logprobs)) check_f32<I>(*ref_logprobs, logprobs, sizes, "ref_logprobs");
    if (present(entropy)) check_f32<I>(*entropy, logprobs, sizes, "entropy");
    if (present(mask)) {
        TORCH_CHECK(mask->device() == logprobs.device(), "All tensors must be on same device");
        TORCH_CHECK(mask->scalar_type() == torch::kBool, "mask must be bool");
        TORCH_CHECK(Dims<I>::sizes(*mask) == sizes, "mask must have the shape of logprobs");
        TORCH_CHECK(mask->is_contiguous(), "mask must be contiguous");
    }
    TORCH_CHECK(clip_low >= 0 && clip_high >= 0, "clip_low and clip_high must not be negative");
    TORCH_CHECK(denominator >= 0, "denominator must be positive");
    return per_row;
}

using LossOut = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor>;
// (loss, ratio, stats, slope, row_scale, weight); the last three hold nothing unless `save` (undefined with `bare`)
template <typename I>
LossOut loss_buffers(const Tensor& logprobs, bool sequence, bool save, bool bare)
{
    const auto opts = logprobs.options();
    const auto sizes = Dims<I>::sizes(logprobs);
    auto kept = [&](bool there, typename Dims<I>::Ref of) {
        return there ? Dims<I>::empty(of, opts) : bare ? Tensor() : torch::empty({0}, opts);
    };
    return {torch::empty({}, opts), Dims<I>::empty(sizes, opts), torch::empty({6}, opts), kept(save, sizes),
            kept(save && sequence, sizes.slice(0, 1)), kept(save, {1})};
}
LossOut loss_forward_meta(const Tensor& logprobs, const Tensor& old_logprobs, const Tensor& advantages, double clip_low,
                          double clip_high, const OptTensor& ref_logprobs, double, const OptTensor& entropy, double,
                          const OptTensor& mask, c10::string_view reduction, double denominator, bool save)
{
    loss_args<c10::SymInt>(logprobs, old_logprobs, advantages, ref_logprobs, entropy, mask, clip_low, clip_high, denominator);
    return loss_buffers<c10::SymInt>(logprobs, reduction_code(reduction) == PUFF_MEAN_SEQUENCES, save, false);
}
LossOut loss_run(const Tensor& logprobs, const Tensor& old_logprobs, const Tensor& advantages, double clip_low,
                          double clip_high, const OptTensor& ref_logprobs, double kl_coef, const OptTensor& entropy,
                 double ent_coef, const OptTensor& mask, c10::string_view reduction, double denominator, bool save, bool bare)
{
    const bool per_row =
        loss_args<int64_t>(logprobs, old_logprobs, advantages, ref_logprobs, entropy, mask, clip_low, clip_high, denominator);
    const c10::cuda::CUDAGuard guard(logprobs.device());
    const bool sequence = reduction_code(reduction) == PUFF_MEAN_SEQUENCES;
    LossOut out = loss_buffers<int64_t>(logprobs, sequence, save, bare);
    auto& [loss, ratio, stats, slope, row_scale, weight] = out;
    const int64_t rows = logprobs.size(0), steps = logprobs.size(1);
    const size_t sbytes = puff_policy_sm100_loss_scratch_bytes(rows, steps);
    Tensor scratch = torch::empty({static_cast<int64_t>((sbytes + 7) / 8)}, logprobs.options().dtype(torch::kFloat64));
    check_rc(puff_policy_sm100_loss(ptr<const float>(logprobs), ptr<const float>(old_logprobs), ptr<const float>(advantages),
                                    per_row, ptr<float>(ref_logprobs), ptr<float>(entropy), ptr<unsigned char>(mask),
                                    clip_low, clip_high, static_cast<float>(kl_coef), static_cast<float>(ent_coef),
                                    sequence ? PUFF_MEAN_SEQUENCES : PUFF_MEAN_TOKENS, denominator, rows, steps,
                                    ptr<float>(loss), ptr<float>(ratio), ptr<float>(stats),
                                    save ? ptr<float>(slope) : nullptr, save && sequence ? ptr<float>(row_scale) : nullptr,
                                    save ? ptr<float>(weight) : nullptr, scratch.data_ptr(), sbytes, current_stream()),
             "puff_policy_loss");
    return out;
}
LossOut loss_forward_cuda(const Tensor& logprobs, const Tensor& old_logprobs, const Tensor& advantages, double clip_low,
                          double clip_high, const OptTensor& ref_logprobs, double kl_coef, const OptTensor& entropy,
                          double ent_coef, const OptTensor& mask, c10::string_view reduction, double denominator, bool save)
{
    return loss_run(logprobs, old_logprobs, advantages, clip_low, clip_high, ref_logprobs, kl_coef, entropy, ent_coef, mask,
                    reduction, denominator, save, false);
}
LossOut loss_forward(const Tensor& logprobs, const Tensor& old_logprobs, const Tensor& advantages, double clip_low,
                     double clip_high, const OptTensor& ref_logprobs, double kl_coef, const OptTensor& entropy,
                     double ent_coef, const OptTensor& mask, c10::string_view reduction, double denominator, bool save)
{
    static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("pufferlib::puff_policy_loss_forward", "")
                         .typed<decltype(loss_forward_meta)>();
    return op.call(logprobs, old_logprobs, advantages, clip_low, clip_high, ref_logprobs, kl_coef, entropy, ent_coef, mask,
                   reduction, denominator, save);
}
std::tuple<Tensor, Tensor, Tensor> policy_loss_cuda(const Tensor& logprobs, const Tensor& old_logprobs, const Tensor& advantages,
                                                    double clip_low, double clip_high, const OptTensor& ref_logprobs,
                                                    double kl_coef, const OptTensor& entropy, double ent_coef,
                                                    const OptTensor& mask, c10::string_view reduction, double denominator)
{
    LossOut out = loss_run(logprobs, old_logprobs, advantages, clip_low, clip_high, ref_logprobs, kl_coef, entropy, ent_coef,
                           mask, reduction, denominator, false, true);
    return {std::get<0>(out), std::get<1>(out), std::get<2>(out)};
}
std::tuple<Tensor, Tensor, Tensor> policy_loss_meta(const Tensor& logprobs, const Tensor& old_logprobs, const Tensor& advantages,
                                                    double clip_low, double clip_high, const OptTensor& ref_logprobs,
                                                    double kl_coef, const OptTensor& entropy, double ent_coef,
                                                    const OptTensor& mask, c10::string_view reduction, double denominator)
{
    LossOut out = loss_forward_meta(logprobs, old_logprobs, advantages, clip_low, clip_high, ref_logprobs, kl_coef, entropy,
                                    ent_coef, mask, reduction, denominator, false);
    return {std::get<0>(out), std::get<1>(out), std::get<2>(out)};
}
std::tuple<Tensor, Tensor, Tensor> policy_loss(const Tensor& logprobs, const Tensor& old_logprobs, const Tensor& advantages,
                                               double clip_low, double clip_high, const OptTensor& ref_logprobs,
                                               double kl_coef, const OptTensor& entropy, double ent_coef,
                                               const OptTensor& mask, c10::string_view reduction, double denominator)
{
    static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("pufferlib::puff_policy_loss", "")
                         .typed<decltype(policy_loss_meta)>();
    return op.call(logprobs, old_logprobs, advantages, clip_low, clip_high, ref_logprobs, kl_coef, entropy, ent_coef, mask,
                   reduction, denominator);
}

// (dlogprobs, dentropy or an empty tensor)
std::tuple<Tensor, Tensor> loss_backward_meta(const Tensor& slope, const Tensor&, const Tensor&, const Tensor&,
                                              const OptTensor&, double, bool want_dentropy)
{
    return {torch::empty_like(slope), want_dentropy ? torch::empty_like(slope) : torch::empty({0}, slope.options())};
}
std::tuple<Tensor, Tensor> loss_backward_cuda(const Tensor& slope, const Tensor& row_scale, const Tensor& weight,
                                              const Tensor& dloss, const OptTensor& mask, double ent_coef,
                                              bool want_dentropy)
{
    TORCH_CHECK(slope.dim() == 2, "slope must be 2D [rows, steps]");
    check_f32(slope, slope, slope.sizes(), "slope");
    check_f32(weight, slope, {1}, "weight");
    check_f32(dloss, slope, {}, "dloss");
    TORCH_CHECK(row_scale.numel() == 0 || row_scale.numel() == slope.size(0), "row_scale must be [rows] or empty");
    check_f32(row_scale, slope, row_scale.sizes(), "row_scale");
    if (present(mask))
        TORCH_CHECK(mask->scalar_type() == torch::kBool && mask->sizes() == slope.sizes() && mask->is_contiguous() &&
                        mask->device() == slope.device(),
                    "mask must be a contiguous bool tensor of the shape of slope on the same device");
    const c10::cuda::CUDAGuard guard(slope.device());
    auto out = loss_backward_meta(slope, row_scale, weight, dloss, mask, ent_coef, want_dentropy);
    check_rc(puff_policy_sm100_loss_backward(ptr<const float>(slope), row_scale.numel() > 0 ? ptr<const float>(row_scale) : nullptr,
                                             ptr<const float>(weight), ptr<const float>(dloss), ptr<unsigned char>(mask),
                                             static_cast<float>(ent_coef), slope.size(0), slope.size(1),
                                             ptr<float>(std::get<0>(out)),
                                             want_dentropy ? ptr<float>(std::get<1>(out)) : nullptr, current_stream()),
             "puff_policy_loss_backward");
    return out;
}
std::tuple<Tensor, Tensor> loss_backward(const Tensor& slope, const Tensor& row_scale, const Tensor& weight,
                                         const Tensor& dloss, const OptTensor& mask, double ent_coef, bool want_dentropy)
{
    static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("pufferlib::puff_policy_loss_backward", "")
                         .typed<decltype(loss_backward_meta)>();
    return op.call(slope, row_scale, weight, dloss, mask, ent_coef, want_dentropy);
}

struct PolicyLossNode : public Node {
    SavedVariable slope, row_scale, weight, mask;
    double ent_coef = 0.0;
    std::string name() const override { return "PuffPolicyLossBackward"; }
    void release_variables() override
    {
        std::lock_guard<std::mutex> lock(mutex_);
        for (SavedVariable* v : {&slope, &row_scale, &weight, &mask}) v->reset_data();
    }
    variable_list apply(variable_list&& grads) override
    {
        std::lock_guard<std::mutex> lock(mutex_);
        if (!grads[0].defined()) return {Tensor(), Tensor()};
        refuse_forward_mode("the backward pass of puff_policy_loss", grads[0]);
        const bool want_dentropy = task_should_compute_output(1);
        const Tensor s = slope.unpack(), scale = row_scale.unpack(), w = weight.unpack();
        const OptTensor kept = optional(mask.unpack());
        Tensor dlogprobs, dentropy;
        {
            at::AutoDispatchBelowADInplaceOrView below;
            std::tie(dlogprobs, dentropy) = loss_backward(s, scale, w, grads[0], kept, ent_coef, want_dentropy);
        }
        return refuse_second_derivatives("puff_policy_loss", *this, grads, {dlogprobs, want_dentropy ? dentropy : Tensor()});
    }
};
bool wants_grad(const OptTensor& t) { return present(t) && t->requires_grad(); }
std::tuple<Tensor, Tensor, Tensor> policy_loss_autograd(const Tensor& logprobs, const Tensor& old_logprobs,
                                                        const Tensor& advantages, double clip_low, double clip_high,
                                                        const OptTensor& ref_logprobs, double kl_coef,
                                                        const OptTensor& entropy, double ent_coef, const OptTensor& mask,
                                                        c10::string_view reduction, double denominator)
{
    refuse_forward_mode("puff_policy_loss", logprobs, old_logprobs, advantages, ref_logprobs, entropy);
    if (at::GradMode::is_enabled())
        TORCH_CHECK(!old_logprobs.requires_grad() && !advantages.requires_grad() && !wants_grad(ref_logprobs),
                    "old_logprobs, advantages and ref_logprobs are constants of the loss; detach them");
    if (!(at::GradMode::is_enabled() && (logprobs.requires_grad() || wants_grad(entropy)))) {
        at::AutoDispatchBelowADInplaceOrView below;
        return policy_loss(logprobs, old_logprobs, advantages, clip_low, clip_high, ref_logprobs, kl_coef, entropy,
                           ent_coef, mask, reduction, denominator);
    }
    auto node = new_node<PolicyLossNode>(torch::autograd::collect_next_edges(logprobs, entropy.value_or(Tensor())));
    LossOut out;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        out = loss_forward(logprobs, old_logprobs, advantages, clip_low, clip_high, ref_logprobs, kl_coef, entropy, ent_coef,
                           mask, reduction, denominator, true);
    }
    auto& [loss, ratio, stats, slope, row_scale, weight] = out;
    torch::autograd::set_history(loss, node);
    node->slope = SavedVariable(slope, false);
    node->row_scale = SavedVariable(row_scale, false);
    node->weight = SavedVariable(weight, false);
    node->mask = saved(mask);
    node->ent_coef = ent_coef;
    return {loss, ratio, stats};
}

// ---- gated recurrence --------------------------------------------------------------------------------------------

template <typename I>
int check_resets(const OptTensor& resets, const Tensor& like, typename Dims<I>::Ref sizes)
{
    if (!present(resets)) return 0;
    const auto t = resets->scalar_type();
    TORCH_CHECK(resets->device() == like.device(), "All tensors must be on same device");
    TORCH_CHECK(t == torch::kFloat32 || t == torch::kBool || t == torch::kUInt8, "resets must be float32 or bool");
    TORCH_CHECK(Dims<I>::sizes(*resets) == sizes, "resets must have shape ", sizes, ", got ", Dims<I>::sizes(*resets));
    TORCH_CHECK(resets->is_contiguous(), "resets must be contiguous");
    return t == torch::kFloat32 ? 4 : 1;
}
// the size of an element of `resets`, 0 without
template <typename I>
int recurrence_args(const Tensor& gates, const Tensor& inputs, const OptTensor& resets, int64_t dims)
{
    dtype_code(gates, "gates");
    TORCH_CHECK(gates.dim() == dims, "gates must be ", dims == 3 ? "3D [batch, steps, channels]" : "2D [batch, channels]");
    const auto sizes = Dims<I>::sizes(gates);
    TORCH_CHECK(Dims<I>::sizes(inputs) == sizes && inputs.scalar_type() == gates.scalar_type(),
                "gates and inputs must have one shape and one type");
    TORCH_CHECK(inputs.device() == gates.device(), "All tensors must be on same device");
    if (Dims<I>::numel(gates) > 0 && sizes[dims - 1] > 1)
        TORCH_CHECK(Dims<I>::strides(gates)[dims - 1] == 1 && Dims<I>::strides(inputs)[dims - 1] == 1, "the last dimension of gates and inputs must be contiguous");
    return check_resets<I>(resets, gates, sizes.slice(0, dims - 1));
}

// the workspace of one call, or an undefined tensor where it needs none
Tensor recurrence_scratch(const Tensor& gates, size_t* bytes)
{
    *bytes = puff_policy_sm100_recurrence_scratch_bytes(gates.size(0), gates.size(1), gates.size(2));
    return *bytes == 0 ? Tensor() : torch::empty({static_cast<int64_t>((*bytes + 7) / 8)}, gates.options().dtype(torch::kFloat64));
}

using RecOut = std::tuple<Tensor, Tensor, Tensor>;
// (outputs, final state, saved states or an empty tensor)
template <typename I>
RecOut recurrence_buffers(const Tensor& gates, const Tensor& inputs, const OptTensor& resets, const OptTensor& state, bool save,
                          int* reset_bytes)
{
    *reset_bytes = recurrence_args<I>(gates, inputs, resets, 3);
    const auto sizes = Dims<I>::sizes(gates);
    const I &B = sizes[0], &T = sizes[1], &C = sizes[2];
    if (present(state)) check_f32<I>(*state, gates, {B, C}, "state");
    const auto f32 = gates.options().dtype(torch::kFloat32);
    const I states = (T + (PUFF_RECURRENCE_SAVED_STEPS - 1)) / PUFF_RECURRENCE_SAVED_STEPS;
    return {Dims<I>::empty(sizes, gates.options()), Dims<I>::empty({B, C}, f32), Dims<I>::empty({save ? B * states * C : I(0)}, f32)};
}
RecOut recurrence_forward_meta(const Tensor& gates, const Tensor& inputs, const OptTensor& resets, const OptTensor& state,
                               bool save)
{
    int reset_bytes;
    return recurrence_buffers<c10::SymInt>(gates, inputs, resets, state, save, &reset_bytes);
}
RecOut recurrence_forward_cuda(const Tensor& gates, const Tensor& inputs, const OptTensor& resets, const OptTensor& state,
                               bool save)
{
    const c10::cuda::CUDAGuard guard(gates.device());
    int reset_bytes;
    RecOut out = recurrence_buffers<int64_t>(gates, inputs, resets, state, save, &reset_bytes);
    auto& [outputs, final_state, saved] = out;
    size_t sbytes;
    const Tensor scratch = recurrence_scratch(gates, &sbytes);
    check_rc(puff_policy_sm100_recurrence(gates.data_ptr(), inputs.data_ptr(), dtype_code(gates, "gates"), ptr<void>(resets),
                                          reset_bytes, ptr<float>(state),
                                          gates.size(0), gates.size(1), gates.size(2), gates.stride(0), gates.stride(1),
                                          inputs.stride(0), inputs.stride(1), outputs.data_ptr(), ptr<float>(final_state),
                                          save && saved.numel() > 0 ? ptr<float>(saved) : nullptr, ptr<void>(scratch), sbytes,
                                          current_stream()),
             "puff_gated_recurrence");
    return out;
}
RecOut recurrence_forward(const Tensor& gates, const Tensor& inputs, const OptTensor& resets, const OptTensor& state, bool save)
{
    static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("pufferlib::puff_gated_recurrence_forward", "")
                         .typed<decltype(recurrence_forward_meta)>();
    return op.call(gates, inputs, resets, state, save);
}
std::tuple<Tensor, Tensor> gated_recurrence(const Tensor& gates, const Tensor& inputs, const OptTensor& resets, const OptTensor& state)
{
    RecOut out = recurrence_forward(gates, inputs, resets, state, false);
    return {std::get<0>(out), std::get<1>(out)};
}

// (dgates, dinputs, dstate)
template <typename I>
RecOut recurrence_gradients(const Tensor& gates, const Tensor& inputs, const OptTensor& resets, int* reset_bytes)
{
    *reset_bytes = recurrence_args<I>(gates, inputs, resets, 3);
    const auto sizes = Dims<I>::sizes(gates);
    return {Dims<I>::empty(sizes, gates.options()), Dims<I>::empty(sizes, gates.options()),
            Dims<I>::empty({sizes[0], sizes[2]}, gates.options().dtype(torch::kFloat32))};
}
RecOut recurrence_backward_meta(const Tensor& gates, const Tensor& inputs, const OptTensor& resets, const Tensor&,
                                const OptTensor&, const OptTensor&)
{
    int reset_bytes;
    return recurrence_gradients<c10::SymInt>(gates, inputs, resets, &reset_bytes);
}
RecOut recurrence_backward_cuda(const Tensor& gates, const Tensor& inputs, const OptTensor& resets, const Tensor& saved,
                                const OptTensor& doutputs, const OptTensor& dfinal)
{
    const c10::cuda::CUDAGuard guard(gates.device());
    int reset_bytes;
    RecOut out = recurrence_gradients<int64_t>(gates, inputs, resets, &reset_bytes);
    const int64_t B = gates.size(0), T = gates.size(1), C = gates.size(2);
    check_f32(saved, gates, {puff_policy_sm100_recurrence_saved_floats(B, T, C)}, "saved");
    if (present(doutputs))
        TORCH_CHECK(doutputs->sizes() == gates.sizes() && doutputs->scalar_type() == gates.scalar_type() &&
                        doutputs->is_contiguous() && doutputs->device() == gates.device(),
                    "doutputs must be contiguous, of the shape and type of gates, on the same device");
    if (present(dfinal)) check_f32(*dfinal, gates, {B, C}, "dfinal");
    auto& [dgates, dinputs, dstate] = out;
    size_t sbytes;
    const Tensor scratch = recurrence_scratch(gates, &sbytes);
    check_rc(puff_policy_sm100_recurrence_backward(
                 gates.data_ptr(), inputs.data_ptr(), dtype_code(gates, "gates"), ptr<void>(resets), reset_bytes,
                 ptr<const float>(saved), B, T, C, gates.stride(0),
                 gates.stride(1), inputs.stride(0), inputs.stride(1), ptr<void>(doutputs), ptr<float>(dfinal),
                 dgates.data_ptr(), dinputs.data_ptr(), ptr<float>(dstate), ptr<void>(scratch), sbytes, current_stream()),
             "puff_gated_recurrence_backward");
    return out;
}
RecOut recurrence_backward(const Tensor& gates, const Tensor& inputs, const OptTensor& resets, const Tensor& saved,
                           const OptTensor& doutputs, const OptTensor& dfinal)
{
    static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("pufferlib::puff_gated_recurrence_backward", "")
                         .typed<decltype(recurrence_backward_meta)>();
    return op.call(gates, inputs, resets, saved, doutputs, dfinal);
}

struct RecurrenceNode : public Node {
    SavedVariable gates, inputs, resets, states;
    std::string name() const override { return "PuffGatedRecurrenceBackward"; }
    void release_variables() override
    {
        std::lock_guard<std::mutex> lock(mutex_);
        for (SavedVariable* v : {&gates, &inputs, &resets, &states}) v->reset_data();
    }
    variable_list apply(variable_list&& grads) override
    {
        std::lock_guard<std::mutex> lock(mutex_);
        if (!grads[0].defined() && !grads[1].defined()) return {Tensor(), Tensor(), Tensor()};
        refuse_forward_mode("the backward pass of puff_gated_recurrence", grads[0], grads[1]);
        const Tensor g = gates.unpack(), x = inputs.unpack(), kept = states.unpack();
        const OptTensor cut = optional(resets.unpack());
        Tensor dgates, dinputs, dstate;
        {
            at::AutoDispatchBelowADInplaceOrView below;
            const OptTensor dout = grads[0].defined() ? OptTensor(grads[0].contiguous()) : std::nullopt;
            const OptTensor dfinal = grads[1].defined() ? OptTensor(grads[1].contiguous()) : std::nullopt;
            std::tie(dgates, dinputs, dstate) = recurrence_backward(g, x, cut, kept, dout, dfinal);
        }
        return refuse_second_derivatives("puff_gated_recurrence", *this, grads, {dgates, dinputs, dstate});
    }
};
std::tuple<Tensor, Tensor> gated_recurrence_autograd(const Tensor& gates, const Tensor& inputs, const OptTensor& resets,
                                                     const OptTensor& state)
{
    refuse_forward_mode("puff_gated_recurrence", gates, inputs, state);
    if (!(at::GradMode::is_enabled() && (gates.requires_grad() || inputs.requires_grad() || wants_grad(state)))) {
        at::AutoDispatchBelowADInplaceOrView below;
        return gated_recurrence(gates, inputs, resets, state);
    }
    auto node = new_node<RecurrenceNode>(torch::autograd::collect_next_edges(gates, inputs, state.value_or(Tensor())));
    Tensor outputs, final_state, states;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        std::tie(outputs, final_state, states) = recurrence_forward(gates, inputs, resets, state, true);
    }
    torch::autograd::set_history(outputs, node);
    torch::autograd::set_history(final_state, node);
    node->gates = SavedVariable(gates, false);
    node->inputs = SavedVariable(inputs, false);
    node->resets = saved(resets);
    node->states = SavedVariable(states, false);
    return {outputs, final_state};
}

template <typename I>
int step_args(const Tensor& gates, const Tensor& inputs, const Tensor& state, const OptTensor& resets, const Tensor& new_state)
{
    check_f32<I>(state, gates, Dims<I>::sizes(gates), "state");
    check_f32<I>(new_state, gates, Dims<I>::sizes(gates), "new_state");
    return recurrence_args<I>(gates, inputs, resets, 2);
}
Tensor recurrence_step_meta(const Tensor& gates, const Tensor& inputs, const Tensor& state, const OptTensor& resets, Tensor new_state)
{
    step_args<c10::SymInt>(gates, inputs, state, resets, new_state);
    return at::empty_symint(gates.sym_sizes(), gates.options());
}
Tensor recurrence_step_cuda(const Tensor& gates, const Tensor& inputs, const Tensor& state, const OptTensor& resets, Tensor new_state)
{
    const int reset_bytes = step_args<int64_t>(gates, inputs, state, resets, new_state);
    const c10::cuda::CUDAGuard guard(gates.device());
    Tensor outputs = torch::empty(gates.sizes(), gates.options());
    check_rc(puff_policy_sm100_recurrence_step(gates.data_ptr(), inputs.data_ptr(), dtype_code(gates, "gates"), ptr<void>(resets),
                                               reset_bytes, ptr<const float>(state),
                                               gates.size(0), gates.size(1), gates.stride(0), inputs.stride(0),
                                               outputs.data_ptr(), ptr<float>(new_state), current_stream()),
             "puff_gated_recurrence_step");
    return outputs;
}
// the single step is for acting, not for training
Tensor recurrence_step_autograd(const Tensor& gates, const Tensor& inputs, const Tensor& state, const OptTensor& resets, Tensor new_state)
{
    refuse_forward_mode("puff_gated_recurrence_step", gates, inputs, state, new_state);
    TORCH_CHECK(!(at::GradMode::is_enabled() && (gates.requires_grad() || inputs.requires_grad() || state.requires_grad() ||
                                                 new_state.requires_grad())),
                "the single step has no gradient; call it under torch.no_grad() or use puff_gated_recurrence");
    at::AutoDispatchBelowADInplaceOrView below;
    static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("pufferlib::puff_gated_recurrence_step", "")
                         .typed<decltype(recurrence_step_meta)>();
    Tensor outputs = op.call(gates, inputs, state, resets, new_state);
    new_state.unsafeGetTensorImpl()->bump_version();
    return outputs;
}
}  // namespace

TORCH_LIBRARY_FRAGMENT(pufferlib, m)
{
    m.def("puff_action_logprobs(Tensor logits, Tensor actions, float temperature=1.0, bool entropy=True) -> (Tensor, Tensor)");
    m.def("puff_action_logprobs_forward(Tensor logits, Tensor actions, float temperature, bool entropy, bool save) -> (Tensor, Tensor, Tensor)");
    m.def("puff_action_logprobs_backward(Tensor logits, Tensor actions, float temperature, Tensor row_stats, Tensor? entropy, Tensor dlogprobs, Tensor? dentropy) -> Tensor");
    m.def("puff_policy_loss(Tensor logprobs, Tensor old_logprobs, Tensor advantages, float clip_low, float clip_high, Tensor? ref_logprobs, float kl_coef, Tensor? entropy, float ent_coef, Tensor? mask, str reduction, float denominator) -> (Tensor, Tensor, Tensor)");
    m.def("puff_policy_loss_forward(Tensor logprobs, Tensor old_logprobs, Tensor advantages, float clip_low, float clip_high, Tensor? ref_logprobs, float kl_coef, Tensor? entropy, float ent_coef, Tensor? mask, str reduction, float denominator, bool save) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
    m.def("puff_policy_loss_backward(Tensor slope, Tensor row_scale, Tensor weight, Tensor dloss, Tensor? mask, float ent_coef, bool want_dentropy) -> (Tensor, Tensor)");
    m.def("puff_gated_recurrence(Tensor gates, Tensor inputs, Tensor? resets, Tensor? state) -> (Tensor, Tensor)");
    m.def("puff_gated_recurrence_forward(Tensor gates, Tensor inputs, Tensor? resets, Tensor? state, bool save) -> (Tensor, Tensor, Tensor)");
    m.def("puff_gated_recurrence_backward(Tensor gates, Tensor inputs, Tensor? resets, Tensor saved, Tensor? doutputs, Tensor? dfinal) -> (Tensor, Tensor, Tensor)");
    m.def("puff_gated_recurrence_step(Tensor gates, Tensor inputs, Tensor state, Tensor? resets, Tensor(a!) new_state) -> Tensor");
}

TORCH_LIBRARY_IMPL(pufferlib, CUDA, m)
{
    m.impl("puff_action_logprobs", &action_logprobs_cuda);
    m.impl("puff_action_logprobs_forward", &logprobs_forward_cuda);
    m.impl("puff_action_logprobs_backward", &logprobs_backward_cuda);
    m.impl("puff_policy_loss", &policy_loss_cuda);
    m.impl("puff_policy_loss_forward", &loss_forward_cuda);
    m.impl("puff_policy_loss_backward", &loss_backward_cuda);
    m.impl("puff_gated_recurrence", &gated_recurrence);
    m.impl("puff_gated_recurrence_forward", &recurrence_forward_cuda);
    m.impl("puff_gated_recurrence_backward", &recurrence_backward_cuda);
    m.impl("puff_gated_recurrence_step", &recurrence_step_cuda);
}

TORCH_LIBRARY_IMPL(pufferlib, Meta, m)
{
    m.impl("puff_action_logprobs", &action_logprobs_meta);
    m.impl("puff_action_logprobs_forward", &logprobs_forward_meta);
    m.impl("puff_action_logprobs_backward", &logprobs_backward_meta);
    m.impl("puff_policy_loss", &policy_loss_meta);
    m.impl("puff_policy_loss_forward", &loss_forward_meta);
    m.impl("puff_policy_loss_backward", &loss_backward_meta);
    m.impl("puff_gated_recurrence", &gated_recurrence);
    m.impl("puff_gated_recurrence_forward", &recurrence_forward_meta);
    m.impl("puff_gated_recurrence_backward", &recurrence_backward_meta);
    m.impl("puff_gated_recurrence_step", &recurrence_step_meta);
}

TORCH_LIBRARY_IMPL(pufferlib, Autograd, m)
{
    m.impl("puff_action_logprobs", &action_logprobs_autograd);
    m.impl("puff_policy_loss", &policy_loss_autograd);
    m.impl("puff_gated_recurrence", &gated_recurrence_autograd);
    m.impl("puff_gated_recurrence_step", &recurrence_step_autograd);
    for (const char* name : {"puff_action_logprobs_forward", "puff_action_logprobs_backward", "puff_policy_loss_forward",
                             "puff_policy_loss_backward", "puff_gated_recurrence_forward", "puff_gated_recurrence_backward"})
        m.impl(name, torch::autograd::autogradNotImplementedFallback());
}

}  // namespace pufferlib_b200
