// framewise_torch.cpp -- torch extension `framewise_core`: the operators of framewise training over the C ABI of
// include/framewise_b200.h, as autograd nodes.  Input errors are RuntimeErrors; work is enqueued on torch's current
// stream of the inputs' device under a device guard; scratch comes from torch's caching allocator.
#include <torch/extension.h>

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>

#include <algorithm>
#include <cmath>
#include <memory>
#include <string>
#include <tuple>
#include <vector>

#include "framewise_b200.h"

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

void check_status(int status) {
    if (status == FRAMEWISE_B200_OK) return;
    if (status == FRAMEWISE_B200_CUDA_ERROR)
        TORCH_CHECK(false, "framewise: CUDA error: ", cudaGetErrorString(cudaGetLastError()));
    TORCH_CHECK(false, "framewise: ", framewise_b200_status_string(status));
}

framewise_b200_stream_t stream_of() {
    return reinterpret_cast<framewise_b200_stream_t>(at::cuda::getCurrentCUDAStream().stream());
}

Tensor bytes(size_t n, const Tensor& like) {
    return torch::empty({(int64_t)(n > 0 ? n : 1)}, like.options().dtype(torch::kUInt8));
}

int dtype_of(const Tensor& x, const char* name) {
    TORCH_CHECK(x.is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(x.scalar_type() == torch::kFloat32 || x.scalar_type() == torch::kBFloat16, name, " must have dtype float32 or bfloat16");
    return x.scalar_type() == torch::kFloat32 ? FRAMEWISE_B200_F32 : FRAMEWISE_B200_BF16;
}

// values where they are: a view that holds them negated or conjugated is copied
Tensor plain(const Tensor& x) { return x.is_neg() ? x.resolve_neg() : x; }

// There are no forward-mode derivatives: a tensor that carries one is refused, for its tangent would be lost.
void check_no_tangent(const Tensor& x, const char* name) {
    TORCH_CHECK(!x.defined() || !x._fw_grad(/*level=*/0).defined(), "framewise: there are no forward-mode derivatives (of ", name, ")");
}

// (B,T) labels and (B,) lengths of a call; labels of one dimension are a batch of one
struct Positions {
    int64_t B, T;
    Tensor  labels, lens;
    bool    wide;
    Positions(const Tensor& labels_in, const OptTensor& lens_in, const Tensor& on) {
        TORCH_CHECK(labels_in.is_cuda() && labels_in.device() == on.device(), "labels must be on the device of the other tensors");
        TORCH_CHECK(labels_in.scalar_type() == torch::kInt32 || labels_in.scalar_type() == torch::kInt64, "labels must have dtype int32 or int64");
        TORCH_CHECK(labels_in.dim() == 1 || labels_in.dim() == 2, "labels must have shape (N,) or (B, T)");
        wide = labels_in.scalar_type() == torch::kInt64;
        B = labels_in.dim() == 2 ? labels_in.size(0) : 1;
        T = labels_in.size(-1);
        labels = labels_in.contiguous();
        if (lens_in.has_value()) {
            lens = *lens_in;
            TORCH_CHECK(labels_in.dim() == 2, "seq_lens needs labels of shape (B, T)");
            TORCH_CHECK(lens.is_cuda() && lens.device() == on.device(), "seq_lens must be on the device of the other tensors");
            TORCH_CHECK(lens.scalar_type() == torch::kInt32, "seq_lens must have dtype int32");
            TORCH_CHECK(lens.dim() == 1 && lens.size(0) == B, "seq_lens must have shape (B,)");
            lens = lens.contiguous();
        }
    }
    const int32_t* lens_ptr() const { return lens.defined() ? lens.data_ptr<int32_t>() : nullptr; }
};

// ------------------------------------------------------------------------------------------ cross entropy

struct CeCall {
    framewise_b200_ce_shape shape = {};
    size_t saved = 0, forward = 0, backward = 0;
};

struct CeInputs {
    Tensor hidden, weight, bias;
    Positions at;
    CeCall call;
};

CeInputs ce_inputs(const Tensor& hidden_in, const Tensor& weight_in, const OptTensor& bias_in, const Tensor& targets,
                   const OptTensor& seq_lens, int64_t ignore_index, bool train) {
    const int dtype = dtype_of(hidden_in, "hidden");
    TORCH_CHECK(weight_in.device() == hidden_in.device() && weight_in.scalar_type() == hidden_in.scalar_type(),
                "weight must have the device and dtype of hidden");
    TORCH_CHECK(hidden_in.dim() == targets.dim() + 1, "hidden must have one dimension more than targets");
    for (int64_t d = 0; d < targets.dim(); ++d)
        TORCH_CHECK(hidden_in.size(d) == targets.size(d), "hidden must have shape (*targets.shape, D)");
    const int64_t D = hidden_in.size(-1);
    TORCH_CHECK(weight_in.dim() == 2 && weight_in.size(1) == D, "weight must have shape (V, D)");
    TORCH_CHECK(D > 0 && weight_in.size(0) > 0, "weight must not be empty");
    CeInputs in{plain(hidden_in), plain(weight_in).contiguous(), Tensor(), Positions(targets, seq_lens, hidden_in), CeCall()};
    if (in.hidden.stride(-1) != 1) in.hidden = in.hidden.contiguous();
    if (bias_in.has_value()) {
        TORCH_CHECK(bias_in->device() == hidden_in.device() && bias_in->scalar_type() == hidden_in.scalar_type(),
                    "bias must have the device and dtype of hidden");
        TORCH_CHECK(bias_in->dim() == 1 && bias_in->size(0) == weight_in.size(0), "bias must have shape (V,)");
        in.bias = plain(*bias_in).contiguous();
    }
    auto& s = in.call.shape;
    s.B = in.at.B, s.T = in.at.T, s.V = weight_in.size(0), s.D = D;
    s.hidden_stride_b = targets.dim() == 2 ? in.hidden.stride(0) : 0;
    s.hidden_stride_t = in.hidden.stride(-2);
    s.ignore_index = ignore_index;
    s.dtype = dtype, s.labels64 = in.at.wide, s.has_bias = in.bias.defined(), s.train = train;
    s.copy_weight = dtype == FRAMEWISE_B200_BF16 && (D % 8 != 0 || reinterpret_cast<uintptr_t>(in.weight.data_ptr()) % 16 != 0);
    check_status(framewise_b200_ce_bytes(&s, &in.call.saved, &in.call.forward, &in.call.backward));
    return in;
}

// (loss, what the backward pass needs: that alone, for the graph holds it, and hooks may carry it elsewhere and back)
std::pair<Tensor, Tensor> ce_forward(const CeInputs& in, const Tensor& targets) {
    const bool   apart = in.call.shape.train;  // without gradients scratch follows in the same buffer
    const size_t kept  = (in.call.saved + 255) / 256 * 256;
    Tensor loss  = torch::empty(targets.sizes(), in.hidden.options().dtype(torch::kFloat32));
    Tensor saved = bytes(apart ? in.call.saved : kept + in.call.forward, in.hidden);
    Tensor work  = apart ? bytes(in.call.forward, in.hidden) : Tensor();
    char* const at = static_cast<char*>(saved.data_ptr());
    check_status(framewise_b200_ce_forward(&in.call.shape, in.hidden.data_ptr(), in.weight.data_ptr(),
                                           in.bias.defined() ? in.bias.data_ptr() : nullptr, in.at.labels.data_ptr(), in.at.lens_ptr(),
                                           loss.data_ptr<float>(), at, in.call.saved, apart ? work.data_ptr() : at + kept, in.call.forward,
                                           stream_of()));
    return {loss, saved};
}

// The node of the graph that a call leaves behind.  (A node of its own, rather than torch::autograd::Function: that packs
// sizes into a dictionary, some ten microseconds a step.)
struct LinearCrossEntropyBackward : public torch::autograd::Node {
    torch::autograd::SavedVariable weight, saved;  // a change of the weight before the backward pass is noticed
    CeCall  call;
    bool    flat = false;

    std::string name() const override { return "LinearCrossEntropyBackward"; }
    void release_variables() override {
        weight.reset_data();
        saved.reset_data();
    }
    torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
        TORCH_CHECK(!torch::GradMode::is_enabled(), "framewise: there are no gradients of these gradients");
        check_no_tangent(grads[0], "gradients");
        if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor()};
        const Tensor w = weight.unpack(), kept = saved.unpack();
        const auto& s = call.shape;
        TORCH_CHECK(w.is_cuda() && w.device() == kept.device() && w.is_contiguous() && w.dim() == 2 && w.size(0) == s.V && w.size(1) == s.D &&
                        w.scalar_type() == (s.dtype == FRAMEWISE_B200_F32 ? torch::kFloat32 : torch::kBFloat16) && kept.is_contiguous() &&
                        kept.scalar_type() == torch::kUInt8 && (size_t)kept.numel() >= call.saved,
                    "framewise: saved-tensor hooks must give back what they were given");
        c10::cuda::CUDAGuard guard(w.device());
        Tensor g = plain(grads[0]);
        if (g.scalar_type() != torch::kFloat32) g = g.to(torch::kFloat32);
        Tensor dh, dw, db, work = bytes(call.backward, w);
        const auto options = w.options().requires_grad(false);
        if (task_should_compute_output(0)) dh = flat ? torch::empty({s.T, s.D}, options) : torch::empty({s.B, s.T, s.D}, options);
        if (task_should_compute_output(1)) dw = torch::empty({s.V, s.D}, options);
        if (s.has_bias && task_should_compute_output(2)) db = torch::empty({s.V}, options);
        auto ptr = [](const Tensor& x) { return x.defined() ? x.data_ptr() : nullptr; };
        check_status(framewise_b200_ce_backward(&s, w.data_ptr(), g.data_ptr<float>(), flat ? 0 : g.stride(0), g.stride(-1), ptr(dh), ptr(dw),
                                                ptr(db), kept.data_ptr(), call.saved, work.data_ptr(), call.backward,
                                                stream_of()));
        return {dh, dw, db};
    }
};

Tensor linear_cross_entropy(const Tensor& hidden, const Tensor& weight, const Tensor& targets, const OptTensor& bias,
                            const OptTensor& seq_lens, int64_t ignore_index) {
    dtype_of(hidden, "hidden");
    check_no_tangent(hidden, "hidden");
    check_no_tangent(weight, "weight");
    if (bias.has_value()) check_no_tangent(*bias, "bias");
    const bool train = torch::GradMode::is_enabled() &&
                       (hidden.requires_grad() || weight.requires_grad() || (bias.has_value() && bias->requires_grad()));
    c10::cuda::CUDAGuard guard(hidden.device());
    if (!train) return ce_forward(ce_inputs(hidden, weight, bias, targets, seq_lens, ignore_index, false), targets).first;
    Tensor loss, w, saved;
    std::shared_ptr<LinearCrossEntropyBackward> node(new LinearCrossEntropyBackward(), torch::autograd::deleteNode);
    {
        at::AutoDispatchBelowADInplaceOrView below;
        const CeInputs in = ce_inputs(hidden, weight, bias, targets, seq_lens, ignore_index, true);
        std::tie(loss, saved) = ce_forward(in, targets);
        w          = in.weight;
        node->call = in.call;
        node->flat = targets.dim() == 1;
    }
    node->weight = torch::autograd::SavedVariable(w, false);  // outside of the guard: hooks may run
    node->saved  = torch::autograd::SavedVariable(saved, false);
    node->set_next_edges(torch::autograd::collect_next_edges(hidden, weight, bias.has_value() ? *bias : Tensor()));
    torch::autograd::set_history(loss, node);
    return loss;
}

// ------------------------------------------------------------------------------------------ embedding

Tensor embed_forward(const Tensor& weight, const Tensor& labels, const Positions& at, double scale, int64_t ignore_index) {
    const int dtype = dtype_of(weight, "weight");
    TORCH_CHECK(weight.dim() == 2 && weight.size(0) > 0 && weight.size(1) > 0, "weight must have shape (V, D)");
    auto shape = labels.sizes().vec();
    shape.push_back(weight.size(1));
    const Tensor w   = plain(weight).contiguous();
    Tensor       out = torch::empty(shape, w.options());
    check_status(framewise_b200_embed_forward(at.B, at.T, w.size(0), w.size(1), dtype, at.wide, ignore_index, (float)scale, w.data_ptr(),
                                              at.labels.data_ptr(), at.lens_ptr(), out.data_ptr(), stream_of()));
    return out;
}

struct LabelEmbeddingBackward : public torch::autograd::Node {
    torch::autograd::SavedVariable labels, lens;
    bool    has_lens = false, flat = false;
    int64_t B = 0, T = 0, V = 0, D = 0, ignore_index = 0;
    double  scale = 1.0;

    std::string name() const override { return "LabelEmbeddingBackward"; }
    void release_variables() override {
        labels.reset_data();
        lens.reset_data();
    }
    torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
        TORCH_CHECK(!torch::GradMode::is_enabled(), "framewise: there are no gradients of these gradients");
        check_no_tangent(grads[0], "gradients");
        if (!grads[0].defined()) return {Tensor()};
        const Tensor t = labels.unpack(), n = has_lens ? lens.unpack() : Tensor();
        TORCH_CHECK(t.is_cuda() && t.is_contiguous() && t.numel() == B * T && (t.scalar_type() == torch::kInt32 || t.scalar_type() == torch::kInt64) &&
                        t.device() == grads[0].device() &&
                        (!has_lens || (n.device() == t.device() && n.is_contiguous() && n.numel() == B && n.scalar_type() == torch::kInt32)),
                    "framewise: saved-tensor hooks must give back what they were given");
        c10::cuda::CUDAGuard guard(t.device());
        Tensor g = plain(grads[0]);
        if (g.stride(-1) != 1) g = g.contiguous();
        Tensor dw = torch::empty({V, D}, g.options());
        const size_t need = framewise_b200_embed_bytes(B, T, V, D);
        Tensor work = bytes(need, g);
        check_status(framewise_b200_embed_backward(B, T, V, D, dtype_of(g, "the gradient"), t.scalar_type() == torch::kInt64, ignore_index,
                                                   (float)scale, g.data_ptr(), flat ? 0 : g.stride(0), g.stride(-2), t.data_ptr(),
                                                   n.defined() ? n.data_ptr<int32_t>() : nullptr, dw.data_ptr(), work.data_ptr(), need, stream_of()));
        return {dw};
    }
};

Tensor label_embedding(const Tensor& labels, const Tensor& weight, double scale, const OptTensor& seq_lens, int64_t ignore_index) {
    dtype_of(weight, "weight");
    check_no_tangent(weight, "weight");
    c10::cuda::CUDAGuard guard(weight.device());
    if (!torch::GradMode::is_enabled() || !weight.requires_grad())
        return embed_forward(weight, labels, Positions(labels, seq_lens, weight), scale, ignore_index);
    Tensor out, t, n;
    std::shared_ptr<LabelEmbeddingBackward> node(new LabelEmbeddingBackward(), torch::autograd::deleteNode);
    {
        at::AutoDispatchBelowADInplaceOrView below;
        const Positions at(labels, seq_lens, weight);
        out = embed_forward(weight, labels, at, scale, ignore_index);
        t = at.labels, n = at.lens;
        node->flat = labels.dim() == 1, node->B = at.B, node->T = at.T, node->V = weight.size(0), node->D = weight.size(1);
        node->ignore_index = ignore_index, node->scale = scale;
    }
    node->labels = torch::autograd::SavedVariable(t, false);
    if ((node->has_lens = n.defined())) node->lens = torch::autograd::SavedVariable(n, false);
    node->set_next_edges(torch::autograd::collect_next_edges(weight));
    torch::autograd::set_history(out, node);
    return out;
}

// ------------------------------------------------------------------------------------------ label scores

using Tensors = std::vector<Tensor>;

struct ScoresInputs {
    Tensor    logits;
    Positions at;
    framewise_b200_scores_shape shape = {};
};

ScoresInputs scores_inputs(const Tensor& logits_in, const Tensor& labels, int64_t top, const OptTensor& seq_lens, int64_t ignore_index) {
    const int dtype = dtype_of(logits_in, "logits");
    TORCH_CHECK(logits_in.dim() == labels.dim() + 1, "logits must have one dimension more than labels");
    for (int64_t d = 0; d < labels.dim(); ++d) TORCH_CHECK(logits_in.size(d) == labels.size(d), "logits must have shape (*labels.shape, V)");
    const int64_t V = logits_in.size(-1);
    TORCH_CHECK(V > 0, "logits must have classes");
    TORCH_CHECK(top >= 0 && top <= std::min<int64_t>(V, 32), "top must be in 0..min(V, 32)");
    ScoresInputs in{plain(logits_in), Positions(labels, seq_lens, logits_in)};
    if (V > 1 && in.logits.stride(-1) != 1) in.logits = in.logits.contiguous();
    auto& s = in.shape;
    s.B = in.at.B, s.T = in.at.T, s.V = V, s.top = (int32_t)top, s.ignore_index = ignore_index, s.dtype = dtype, s.labels64 = in.at.wide;
    s.logits_stride_b = labels.dim() == 2 ? in.logits.stride(0) : 0;
    s.logits_stride_t = in.logits.stride(-2);
    return in;
}

// log probabilities, entropies, the alternatives' log probabilities and labels; `kept` (undefined: not kept) for the backward pass
Tensors scores_forward(const ScoresInputs& in, const Tensor& labels, Tensor* kept) {
    const auto options = in.logits.options().dtype(torch::kFloat32);
    auto shape = labels.sizes().vec();
    Tensor log_probs = torch::empty(shape, options), entropy = torch::empty(shape, options);
    shape.push_back(in.shape.top);
    Tensor top_log_probs = torch::empty(shape, options), top_labels = torch::empty(shape, labels.options());
    if (kept) *kept = bytes((size_t)(in.at.B * in.at.T) * 16, in.logits);
    check_status(framewise_b200_scores_forward(&in.shape, in.logits.data_ptr(), in.at.labels.data_ptr(), in.at.lens_ptr(), log_probs.data_ptr<float>(),
                                               entropy.data_ptr<float>(), top_log_probs.data_ptr<float>(), top_labels.data_ptr(),
                                               kept ? kept->data_ptr() : nullptr, stream_of()));
    return {log_probs, entropy, top_log_probs, top_labels};
}

struct LabelScoresBackward : public torch::autograd::Node {
    torch::autograd::SavedVariable logits, labels, lens, top_labels, kept;  // a change of the logits in between is noticed
    framewise_b200_scores_shape shape = {};
    bool has_lens = false, flat = false;

    std::string name() const override { return "LabelScoresBackward"; }
    void release_variables() override {
        for (auto* x : {&logits, &labels, &lens, &top_labels, &kept}) x->reset_data();
    }
    torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
        TORCH_CHECK(!torch::GradMode::is_enabled(), "framewise: there are no gradients of these gradients");
        for (const Tensor& g : grads) check_no_tangent(g, "gradients");
        if (!grads[0].defined() && !grads[1].defined() && !grads[2].defined()) return {Tensor()};
        const Tensor z = logits.unpack(), t = labels.unpack(), n = has_lens ? lens.unpack() : Tensor(), best = top_labels.unpack(), k = kept.unpack();
        const auto&  s = shape;
        const auto   label_type = s.labels64 ? torch::kInt64 : torch::kInt32;
        TORCH_CHECK(z.is_cuda() && z.scalar_type() == (s.dtype == FRAMEWISE_B200_F32 ? torch::kFloat32 : torch::kBFloat16) && z.numel() == s.B * s.T * s.V &&
                        z.dim() == (flat ? 2 : 3) && z.size(-1) == s.V && (s.V == 1 || z.stride(-1) == 1) && t.device() == z.device() && t.is_contiguous() &&
                        t.numel() == s.B * s.T && t.scalar_type() == label_type && best.device() == z.device() && best.is_contiguous() &&
                        best.numel() == s.B * s.T * s.top && best.scalar_type() == label_type && k.device() == z.device() && k.is_contiguous() &&
                        k.scalar_type() == torch::kUInt8 && k.numel() >= 16 * s.B * s.T &&
                        (!has_lens || (n.device() == z.device() && n.is_contiguous() && n.numel() == s.B && n.scalar_type() == torch::kInt32)),
                    "framewise: saved-tensor hooks must give back what they were given");
        c10::cuda::CUDAGuard guard(z.device());
        framewise_b200_scores_shape with = s;
        with.logits_stride_b = flat ? 0 : z.stride(0), with.logits_stride_t = z.stride(-2);  // hooks may have laid them out anew
        Tensor g[3];
        for (int i = 0; i < 3; ++i) {
            if (!grads[i].defined()) continue;
            g[i] = plain(grads[i]);
            if (g[i].scalar_type() != torch::kFloat32) g[i] = g[i].to(torch::kFloat32);
        }
        framewise_b200_scores_grads in = {};
        auto strides = [&](const Tensor& x, int64_t& b, int64_t& t) { b = flat ? 0 : x.stride(0), t = x.stride(flat ? 0 : 1); };
        if (g[0].defined()) in.log_probs = g[0].data_ptr<float>(), strides(g[0], in.log_probs_stride_b, in.log_probs_stride_t);
        if (g[1].defined()) in.entropy = g[1].data_ptr<float>(), strides(g[1], in.entropy_stride_b, in.entropy_stride_t);
        if (g[2].defined() && s.top > 0) {
            in.top_log_probs = g[2].data_ptr<float>(), strides(g[2], in.top_stride_b, in.top_stride_t);
            in.top_stride_k = g[2].stride(-1);
        }
        Tensor dz = torch::empty(z.sizes(), z.options().requires_grad(false).memory_format(torch::MemoryFormat::Contiguous));
        check_status(framewise_b200_scores_backward(&with, z.data_ptr(), t.data_ptr(), n.defined() ? n.data_ptr<int32_t>() : nullptr, best.data_ptr(),
                                                    k.data_ptr(), &in, dz.data_ptr(), stream_of()));
        return {dz};
    }
};

std::tuple<Tensor, Tensor, Tensor, Tensor> label_scores(const Tensor& logits, const Tensor& labels, int64_t top, const OptTensor& seq_lens,
                                                        int64_t ignore_index) {
    dtype_of(logits, "logits");
    check_no_tangent(logits, "logits");
    c10::cuda::CUDAGuard guard(logits.device());
    Tensors out;
    if (!torch::GradMode::is_enabled() || !logits.requires_grad()) {
        out = scores_forward(scores_inputs(logits, labels, top, seq_lens, ignore_index), labels, nullptr);
        return {out[0], out[1], out[2], out[3]};
    }
    Tensor z, t, n, kept;
    std::shared_ptr<LabelScoresBackward> node(new LabelScoresBackward(), torch::autograd::deleteNode);
    {
        at::AutoDispatchBelowADInplaceOrView below;
        const ScoresInputs in = scores_inputs(logits, labels, top, seq_lens, ignore_index);
        out = scores_forward(in, labels, &kept);
        z = in.logits, t = in.at.labels, n = in.at.lens;
        node->shape = in.shape, node->flat = labels.dim() == 1;
    }
    node->logits     = torch::autograd::SavedVariable(z, false);  // outside of the guard: hooks may run
    node->labels     = torch::autograd::SavedVariable(t, false);
    node->top_labels = torch::autograd::SavedVariable(out[3], false);
    node->kept       = torch::autograd::SavedVariable(kept, false);
    if ((node->has_lens = n.defined())) node->lens = torch::autograd::SavedVariable(n, false);
    node->set_next_edges(torch::autograd::collect_next_edges(logits));
    torch::autograd::set_history(torch::autograd::variable_list{out[0], out[1], out[2]}, node);
    return {out[0], out[1], out[2], out[3]};
}

// ------------------------------------------------------------------------------------------ AdamW

void check_state(const Tensor& x, const Tensor& p, torch::ScalarType dtype, const char* name) {
    TORCH_CHECK(x.device() == p.device() && x.scalar_type() == dtype && x.is_contiguous() && x.sizes() == p.sizes(), name,
                " must be contiguous ", dtype, " of the shape and device of its parameter");
}
void check_steps(const Tensor& x, const Tensor& codes, const char* name) {
    const int64_t n = (codes.numel() + FRAMEWISE_B200_STATE_BLOCK - 1) / FRAMEWISE_B200_STATE_BLOCK;
    static_assert(FRAMEWISE_B200_STATE_BLOCK == 256, "the message says so");
    TORCH_CHECK(x.device() == codes.device() && x.scalar_type() == torch::kFloat32 && x.is_contiguous() && x.numel() == n, "the steps of ", name,
                " must be contiguous float32, one per 256 values in a row");
}

// Autograd learns that a tensor has been written: a graph that needs its former values refuses to go on.
void written(const Tensors& list) {
    for (const Tensor& x : list)
        if (!x.is_inference()) x.unsafeGetTensorImpl()->bump_version();
}

// exp_avg_steps, exp_avg_sq_steps: empty (states of 32 bits), or one per parameter.  master: empty, or one per parameter;
// follow: the copies take over what has been changed in the parameters.
void adamw_step(const Tensors& params, const Tensors& grads, const Tensors& master, const Tensors& exp_avg, const Tensors& exp_avg_sq,
                const Tensors& exp_avg_steps, const Tensors& exp_avg_sq_steps, double lr, double beta1, double beta2, double eps,
                double weight_decay, int64_t step, bool follow) {
    const size_t n = params.size();
    TORCH_CHECK(grads.size() == n && exp_avg.size() == n && exp_avg_sq.size() == n && (master.empty() || master.size() == n) &&
                    exp_avg_steps.size() == exp_avg_sq_steps.size() && (exp_avg_steps.empty() || exp_avg_steps.size() == n),
                "AdamW: the lists must have one entry per parameter");
    TORCH_CHECK(step >= 1, "AdamW: step counts from 1");
    TORCH_CHECK(lr >= 0 && eps >= 0 && weight_decay >= 0 && beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1,
                "AdamW: lr, eps and weight_decay must not be negative, betas must be in [0, 1)");
    if (n == 0) return;
    const bool eight = !exp_avg_steps.empty();
    const int  dtype = dtype_of(params[0], "parameters");
    c10::cuda::CUDAGuard guard(params[0].device());
    Tensors kept;  // gradients that had to be copied
    std::vector<framewise_b200_tensor> list(n);
    for (size_t i = 0; i < n; ++i) {
        const Tensor& p = params[i];
        TORCH_CHECK(p.device() == params[0].device() && p.scalar_type() == params[0].scalar_type(), "AdamW: parameters of one call must share device and dtype");
        TORCH_CHECK(p.is_contiguous() && !p.is_neg(), "AdamW: parameters must be contiguous");
        TORCH_CHECK(grads[i].layout() == torch::kStrided && grads[i].device() == p.device() && grads[i].scalar_type() == p.scalar_type() && grads[i].sizes() == p.sizes(),
                    "AdamW: a gradient must be dense, with the shape, device and dtype of its parameter");
        Tensor g = grads[i];
        if (!g.is_contiguous() || g.is_neg()) {
            g = plain(g).contiguous();
            kept.push_back(g);
        }
        check_state(exp_avg[i], p, eight ? torch::kInt8 : torch::kFloat32, "exp_avg");
        check_state(exp_avg_sq[i], p, eight ? torch::kUInt8 : torch::kFloat32, "exp_avg_sq");
        auto& t = list[i];
        t.param = p.data_ptr(), t.grad = g.data_ptr(), t.exp_avg = exp_avg[i].data_ptr(), t.exp_avg_sq = exp_avg_sq[i].data_ptr();
        t.n = p.numel(), t.master = nullptr, t.exp_avg_steps = t.exp_avg_sq_steps = nullptr;
        if (!master.empty()) {
            check_state(master[i], p, torch::kFloat32, "master");
            t.master = master[i].data_ptr<float>();
        }
        if (eight) {
            check_steps(exp_avg_steps[i], exp_avg[i], "exp_avg");
            check_steps(exp_avg_sq_steps[i], exp_avg_sq[i], "exp_avg_sq");
            t.exp_avg_steps = exp_avg_steps[i].data_ptr<float>(), t.exp_avg_sq_steps = exp_avg_sq_steps[i].data_ptr<float>();
        }
    }
    const auto run = follow ? framewise_b200_adamw_follow : framewise_b200_adamw;
    check_status(run(list.data(), (int64_t)n, dtype, eight ? 8 : 32, lr, beta1, beta2, eps, weight_decay, step, stream_of()));
    for (const Tensors* const x : {&params, &master, &exp_avg, &exp_avg_sq, &exp_avg_steps, &exp_avg_sq_steps}) written(*x);
}

// What 8-bit states stand for: (first moments, second moments), f32.
std::pair<Tensors, Tensors> adamw_values(const Tensors& exp_avg, const Tensors& exp_avg_steps, const Tensors& exp_avg_sq, const Tensors& exp_avg_sq_steps) {
    const size_t n = exp_avg.size();
    TORCH_CHECK(exp_avg_sq.size() == n && exp_avg_steps.size() == n && exp_avg_sq_steps.size() == n, "the lists must have one entry per parameter");
    Tensors m, v;
    if (n == 0) return {m, v};
    TORCH_CHECK(exp_avg[0].is_cuda(), "exp_avg must be a CUDA tensor");
    c10::cuda::CUDAGuard guard(exp_avg[0].device());
    std::vector<framewise_b200_tensor> list(n);
    for (size_t i = 0; i < n; ++i) {
        check_state(exp_avg[i], exp_avg[0].sizes() == exp_avg[i].sizes() ? exp_avg[0] : exp_avg[i], torch::kInt8, "exp_avg");
        TORCH_CHECK(exp_avg[i].device() == exp_avg[0].device(), "the states must be on one device");
        check_state(exp_avg_sq[i], exp_avg[i], torch::kUInt8, "exp_avg_sq");
        check_steps(exp_avg_steps[i], exp_avg[i], "exp_avg");
        check_steps(exp_avg_sq_steps[i], exp_avg_sq[i], "exp_avg_sq");
        m.push_back(torch::empty(exp_avg[i].sizes(), exp_avg[i].options().dtype(torch::kFloat32)));
        v.push_back(torch::empty(exp_avg[i].sizes(), exp_avg[i].options().dtype(torch::kFloat32)));
        auto& t = list[i];
        t = {m[i].data_ptr(), nullptr, v[i].data_ptr<float>(), exp_avg[i].data_ptr(), exp_avg_sq[i].data_ptr(), exp_avg_steps[i].data_ptr<float>(),
             exp_avg_sq_steps[i].data_ptr<float>(), exp_avg[i].numel()};
    }
    check_status(framewise_b200_adamw_decode(list.data(), (int64_t)n, stream_of()));
    return {m, v};
}

// ------------------------------------------------------------------------------------------ Muon

// coefficients: three per step
void check_coefficients(const std::vector<double>& coefficients) {
    TORCH_CHECK(!coefficients.empty() && coefficients.size() % 3 == 0 && coefficients.size() <= 300, "steps must be in 1..100, of three coefficients each");
    for (double c : coefficients) TORCH_CHECK(std::isfinite(c), "coefficients must be finite");
}

void check_muon_status(int status, const char* sizes) {
    TORCH_CHECK(status != FRAMEWISE_B200_BAD_ARGUMENT, "coefficients must keep singular values below 10^6, and ", sizes);
    check_status(status);
}

Tensor orthogonalize(const Tensor& x_in, const std::vector<double>& coefficients, double eps) {
    const int dtype = dtype_of(x_in, "x");
    check_no_tangent(x_in, "x");
    TORCH_CHECK(!torch::GradMode::is_enabled() || !x_in.requires_grad(), "framewise: orthogonalize has no gradient: detach x");
    TORCH_CHECK(x_in.dim() >= 2, "x must have shape (..., rows, cols)");
    TORCH_CHECK(eps >= 1e-37, "eps must be positive");
    check_coefficients(coefficients);
    c10::cuda::CUDAGuard guard(x_in.device());
    const Tensor  x = plain(x_in).contiguous();
    Tensor        out = torch::empty(x.sizes(), x.options().requires_grad(false).memory_format(torch::MemoryFormat::Contiguous));
    const int64_t rows = x.size(-2), cols = x.size(-1), count = x.numel() > 0 ? x.numel() / (rows * cols) : 0;
    const size_t  need = framewise_b200_orthogonalize_bytes(count, rows, cols, dtype);
    TORCH_CHECK(need > 0, "x is too large");
    Tensor work = bytes(need, x);
    check_muon_status(framewise_b200_orthogonalize(count, rows, cols, dtype, x.data_ptr(), out.data_ptr(), coefficients.data(),
                                                   (int32_t)(coefficients.size() / 3), eps, work.data_ptr(), need, stream_of()),
                      "x must not be too large");
    return out;
}

// master: empty, or one per parameter; follow: the copies take over what has been changed in the parameters.
void muon_step(const Tensors& params, const Tensors& grads, const Tensors& momentum, const Tensors& master, double lr, double beta, bool nesterov,
               double weight_decay, bool match_rms, const std::vector<double>& coefficients, double eps, bool follow) {
    const size_t n = params.size();
    TORCH_CHECK(grads.size() == n && momentum.size() == n && (master.empty() || master.size() == n), "Muon: the lists must have one entry per parameter");
    TORCH_CHECK(lr >= 0 && weight_decay >= 0 && beta >= 0 && beta < 1 && eps >= 1e-37,
                "Muon: lr and weight_decay must not be negative, beta must be in [0, 1), eps positive");
    check_coefficients(coefficients);
    if (n == 0) return;
    const int dtype = dtype_of(params[0], "parameters");
    TORCH_CHECK(master.empty() || dtype != FRAMEWISE_B200_F32, "Muon: float32 parameters need no copies");
    c10::cuda::CUDAGuard guard(params[0].device());
    Tensors kept;  // gradients that had to be copied
    std::vector<framewise_b200_matrix> list(n);
    for (size_t i = 0; i < n; ++i) {
        const Tensor& p = params[i];
        TORCH_CHECK(p.device() == params[0].device() && p.scalar_type() == params[0].scalar_type(), "Muon: parameters of one call must share device and dtype");
        TORCH_CHECK(p.dim() == 2, "Muon: parameters must be matrices");
        TORCH_CHECK(p.is_contiguous() && !p.is_neg(), "Muon: parameters must be contiguous");
        TORCH_CHECK(grads[i].layout() == torch::kStrided && grads[i].device() == p.device() && grads[i].scalar_type() == p.scalar_type() && grads[i].sizes() == p.sizes(),
                    "Muon: a gradient must be dense, with the shape, device and dtype of its parameter");
        Tensor g = grads[i];
        if (!g.is_contiguous() || g.is_neg()) {
            g = plain(g).contiguous();
            kept.push_back(g);
        }
        check_state(momentum[i], p, torch::kFloat32, "momentum");
        if (!master.empty()) check_state(master[i], p, torch::kFloat32, "master");
        list[i] = {p.data_ptr(), g.data_ptr(), momentum[i].data_ptr<float>(), master.empty() ? nullptr : master[i].data_ptr<float>(), p.size(0), p.size(1)};
    }
    const size_t need = framewise_b200_muon_bytes(list.data(), (int64_t)n, dtype);
    TORCH_CHECK(need > 0, "Muon: a parameter is too large");
    Tensor work = bytes(need, params[0]);
    check_muon_status(framewise_b200_muon(list.data(), (int64_t)n, dtype, lr, beta, nesterov, weight_decay, match_rms, coefficients.data(),
                                          (int32_t)(coefficients.size() / 3), eps, follow, work.data_ptr(), need, stream_of()),
                      "parameters must not be too large");
    for (const Tensors* const x : {&params, &master, &momentum}) written(*x);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("linear_cross_entropy", &linear_cross_entropy);
    m.def("label_embedding", &label_embedding);
    m.def("label_scores", &label_scores);
    m.def("adamw_step", &adamw_step);
    m.def("adamw_values", &adamw_values);
    m.def("orthogonalize", &orthogonalize);
    m.def("muon_step", &muon_step);
    m.attr("state_block") = FRAMEWISE_B200_STATE_BLOCK;
    m.def("launch_count", []() { return framewise_b200_launch_count(); });
}
