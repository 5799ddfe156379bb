// gm_tape.cpp -- the tape nodes of the fine-tuning operators (graphmaker_amd.autograd: token_embedding, layer_norm,
// class_log_prob, policy_loss, preference_loss) as torch::autograd::Function, over the C ABI of libgraphmaker_hip.so.
//
// Host code only.  A short call of these operators costs what its host side costs: the kernels of a sequence of a few
// thousand items take 5 to 20 us, forward and backward of a Python tape node 85 to 110 us, of which the engine's own round
// trip is some 35; as nodes that never take the interpreter's lock they take 45 to 60 us.  Checks of arguments are here too;
// the meaning of the arguments is documented at the Python functions.
//
// Every tensor a call needs besides its inputs comes from torch's allocator, on the current stream of the input's device; a
// workspace belongs to one call.  Nothing is read back to the host.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>
#include <optional>
#include <sstream>
#include <string>
#include <unordered_set>
#include <vector>

#include "graphmaker_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct HipError : std::runtime_error {
    using std::runtime_error::runtime_error;
};

template <class... Args> std::string say(const Args&... args) {
    std::ostringstream s;
    (s << ... << args);
    return s.str();
}

void call(int rc, const char* what) {
    if (rc != GM_OK) throw HipError(say(what, " failed (rc=", rc, "): ", gm_last_error()));
}

gm_stream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

int row_dtype(const Tensor& t, const char* what) {
    switch (t.scalar_type()) {
        case at::kFloat: return GM_DTYPE_F32;
        case at::kBFloat16: return GM_DTYPE_BF16;
        case at::kHalf: return GM_DTYPE_F16;
        default: throw py::type_error(say(what, ": expected float32, bfloat16 or float16, got ", t.scalar_type()));
    }
}

void on_gpu(const Tensor& t, const char* what) {
    if (!t.is_cuda()) throw HipError(say(what, ": graphmaker_amd runs on a ROCm device only (tensor is on ", t.device(), ")"));
}

void same_device(const Tensor& t, const char* what, const Tensor& like) {
    if (t.device() != like.device()) throw py::value_error(say(what, ": on ", t.device(), ", expected ", like.device()));
}

// A dual number (torch.autograd.forward_ad) is refused: these operators have no forward-mode derivative, and an output without a
// tangent would count as a derivative of zero.
void no_tangent(const Tensor& t, const char* what) {
    if (t.defined() && t._fw_grad(0).defined())
        C10_THROW_ERROR(NotImplementedError, say(what, " has a tangent: this graphmaker_amd operator has no forward-mode derivative"));
}

// an index argument, contiguous, int32 or int64
Tensor index_of(const Tensor& t, const char* what, const Tensor& like) {
    if (t.scalar_type() != at::kLong && t.scalar_type() != at::kInt)
        throw py::type_error(say(what, ": expected int32 or int64, got ", t.scalar_type()));
    same_device(t, what, like);
    return t.contiguous();
}
int is_i64(const Tensor& t) { return t.scalar_type() == at::kLong; }

// t as rows of `width` elements `ld` apart at its address; a copy only where its strides need one
struct Rows {
    Tensor t;
    int64_t ld;
};
Rows rows_of(const Tensor& t, int64_t width) {
    if (t.is_contiguous()) return {t, width};
    Tensor r = t.reshape({-1, width});
    if (r.size(0) == 0 || (r.size(0) == 1 && (width == 1 || r.stride(1) == 1))) return {r, width};
    if ((width > 1 && r.stride(1) != 1) || r.stride(0) < width) r = r.contiguous();
    return {r, r.stride(0)};
}

const void* at_of(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
template <class T> T* out_of(const Tensor& t) { return t.defined() ? static_cast<T*>(t.mutable_data_ptr()) : nullptr; }
const float* floats(const Tensor& t) { return static_cast<const float*>(at_of(t)); }
const uint8_t* bytes(const Tensor& t) { return static_cast<const uint8_t*>(at_of(t)); }

Tensor empty(at::IntArrayRef shape, at::ScalarType type, const Tensor& like) { return at::empty(shape, like.options().dtype(type).requires_grad(false)); }
Tensor workspace(int64_t size, const Tensor& like) { return size > 0 ? empty({size}, at::kByte, like) : Tensor(); }

// Whether a call on t is recorded.  A captured call over a leaf whose gradient is accumulated on another stream is refused, also
// where casts, views or other operators lie between: torch ties a leaf's accumulation to the stream of the first graph that is
// alive, a backward pass inside the capture would run it there, and that ends the process.
void refuse_foreign(const c10::hip::HIPStream now, const std::shared_ptr<torch::autograd::Node>& accumulator) {
    if (accumulator && accumulator->stream() && accumulator->stream()->id() != now.id())
        throw HipError("captured while a graph recorded on another stream over the same leaf tensor is alive: drop that graph first");
}
bool records(const Tensor& t) {
    if (!t.defined() || !t.requires_grad() || !at::GradMode::is_enabled()) return false;
    if (!t.is_cuda()) return true;
    const c10::hip::HIPStream now = c10::hip::getCurrentHIPStream(t.device().index());
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(now.stream(), &status) != hipSuccess) {
        (void)hipGetLastError();                         // or the next launch would report it as its own
    } else if (status != hipStreamCaptureStatusNone) {
        if (t.is_leaf()) {
            refuse_foreign(now, torch::autograd::impl::try_get_grad_accumulator(t));
        } else {
            std::vector<std::shared_ptr<torch::autograd::Node>> todo{t.grad_fn()};
            std::unordered_set<torch::autograd::Node*> seen{todo[0].get()};
            while (!todo.empty()) {
                const auto node = std::move(todo.back());
                todo.pop_back();
                if (dynamic_cast<torch::autograd::AccumulateGrad*>(node.get())) refuse_foreign(now, node);
                for (const auto& edge : node->next_edges())
                    if (edge.function && seen.insert(edge.function.get()).second) todo.push_back(edge.function);
            }
        }
    }
    return true;
}

// Gradients of an operator without a second derivative: who differentiates them (create_graph) gets an error, not zeros.  They
// depend on the operator's inputs and on the upstream gradient, so that every way from them to either meets the error.
variable_list once(variable_list grads, const Tensor& upstream) {
    if (!at::GradMode::is_enabled()) return grads;
    torch::autograd::edge_list edges;
    for (const torch::autograd::Edge& edge : torch::autograd::get_current_node()->next_edges())
        if (edge.is_valid()) edges.push_back(edge);
    if (upstream.requires_grad()) edges.push_back(torch::autograd::impl::gradient_edge(upstream));
    const auto error = std::make_shared<torch::autograd::Error>("this graphmaker_amd operator has no second derivative", std::move(edges));
    for (Tensor& t : grads)
        if (t.defined()) torch::autograd::set_history(t, error);
    return grads;
}

// A saved tensor as the backward pass may use it.  Hooks on saved tensors (torch.autograd.graph) can hand it back with other
// strides, or as something else altogether, so nothing is taken over from the forward but what it has to be.
void saved_is(const Tensor& t, const char* what, at::ScalarType type, int64_t numel, const Tensor& like) {
    if (t.scalar_type() != type || t.numel() != numel || t.device() != like.device())
        throw HipError(say("the saved ", what, " came back as ", t.scalar_type(), " ", t.sizes(), " on ", t.device(), ", saved were ", numel, " of ", type,
                           " on ", like.device()));
}
Tensor saved_packed(const Tensor& t, const char* what, at::ScalarType type, int64_t numel, const Tensor& like) {
    if (!t.defined()) return t;
    saved_is(t, what, type, numel, like);
    return t.contiguous();
}
int64_t type_code(const Tensor& t) { return t.defined() ? (int64_t)t.scalar_type() : (int64_t)at::kByte; }

// ------------------------------------------------------------------ token_embedding
struct EmbeddingArgs {
    double scale;
    int64_t padding;
};

Tensor embedding_fwd(const Tensor& weight, const Tensor& tokens, const EmbeddingArgs& a) {
    const c10::DeviceGuard guard(weight.device());
    const int64_t C = weight.size(0), w = weight.size(1);
    std::vector<int64_t> shape(tokens.sizes().begin(), tokens.sizes().end());
    shape.push_back(w);
    Tensor out = empty(shape, weight.scalar_type(), weight);
    const Rows table = rows_of(weight, w);
    call(gm_token_embedding_fwd(tokens.numel(), C, w, at_of(tokens), is_i64(tokens), at_of(table.t), table.ld, row_dtype(weight, "weight"),
                                (float)a.scale, out_of<void>(out), w, stream_of(weight)),
         "gm_token_embedding_fwd");
    return out;
}

struct TokenEmbedding : torch::autograd::Function<TokenEmbedding> {
    static Tensor forward(AutogradContext* ctx, const Tensor& weight, const Tensor& tokens, const EmbeddingArgs& a) {
        ctx->save_for_backward({tokens});
        ctx->saved_data["C"] = weight.size(0);
        ctx->saved_data["type"] = type_code(tokens);
        ctx->saved_data["scale"] = a.scale;
        ctx->saved_data["padding"] = a.padding;
        return embedding_fwd(weight, tokens, a);
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        const Tensor& g = grads[0];
        const c10::DeviceGuard guard(g.device());
        const int64_t C = ctx->saved_data["C"].toInt(), w = g.size(-1), n = g.numel() / w;
        const Tensor tokens = saved_packed(ctx->get_saved_variables()[0], "tokens", (at::ScalarType)ctx->saved_data["type"].toInt(), n, g);
        const Rows r = rows_of(g, w);
        Tensor dW = empty({C, w}, g.scalar_type(), g);
        const int64_t need = gm_token_embedding_bwd_workspace_bytes(n, C, w);
        const Tensor ws = workspace(need, g);
        call(gm_token_embedding_bwd(n, C, w, at_of(tokens), is_i64(tokens), ctx->saved_data["padding"].toInt(), at_of(r.t), r.ld,
                                    row_dtype(g, "gradient"), (float)ctx->saved_data["scale"].toDouble(), out_of<void>(dW), w,
                                    out_of<void>(ws), need, stream_of(g)),
             "gm_token_embedding_bwd");
        return once({dW, Tensor(), Tensor()}, g);
    }
};

Tensor token_embedding(const Tensor& weight, const Tensor& tokens, double scale, std::optional<int64_t> padding_idx) {
    if (weight.dim() != 2 || weight.numel() == 0)
        throw py::value_error(say("token_embedding: weight must be (C, w) with C, w > 0, got ", weight.sizes()));
    row_dtype(weight, "weight");
    no_tangent(weight, "weight");
    const Tensor tok = index_of(tokens, "tokens", weight);
    const int64_t C = weight.size(0);
    if (!std::isfinite((float)scale)) throw py::value_error(say("token_embedding: scale must be finite in float32, got ", scale));
    EmbeddingArgs a{scale, -1};
    if (padding_idx) {
        if (*padding_idx < -C || *padding_idx >= C)
            throw py::value_error(say("token_embedding: padding_idx ", *padding_idx, " is outside the ", C, " rows of weight"));
        a.padding = *padding_idx < 0 ? *padding_idx + C : *padding_idx;
    }
    on_gpu(weight, "weight");
    return records(weight) ? TokenEmbedding::apply(weight, tok, a) : embedding_fwd(weight, tok, a);
}

// ------------------------------------------------------------------ layer_norm
int weight_dtype(const Tensor& x, const Tensor& gamma, const Tensor& beta) {
    const Tensor& t = gamma.defined() ? gamma : beta;
    return row_dtype(t.defined() ? t : x, "gamma");
}

Tensor norm_fwd(const Tensor& x, const Rows& r, const Tensor& gamma, const Tensor& beta, double eps, const Tensor& stats) {
    const int64_t N = x.size(-1), M = x.numel() / N;
    Tensor y = empty(x.sizes(), x.scalar_type(), x);
    float* mean = out_of<float>(stats);
    call(gm_layer_norm_fwd(M, N, at_of(r.t), r.ld, row_dtype(x, "x"), at_of(gamma), at_of(beta), weight_dtype(x, gamma, beta), (float)eps,
                           out_of<void>(y), N, mean, mean ? mean + M : nullptr, stream_of(x)),
         "gm_layer_norm_fwd");
    return y;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
    // absent weights are absent optionals: the tape takes no undefined input
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& gamma_, const std::optional<Tensor>& beta_, double eps) {
        const c10::DeviceGuard guard(x.device());
        const Tensor gamma = gamma_.value_or(Tensor()), beta = beta_.value_or(Tensor());
        const int64_t N = x.size(-1);
        const Rows r = rows_of(x, N);
        const Tensor stats = empty({2 * (x.numel() / N)}, at::kFloat, x);
        ctx->save_for_backward({r.t, stats, gamma});
        ctx->saved_data["gamma"] = type_code(gamma);
        ctx->saved_data["beta"] = beta.defined() ? (int64_t)beta.scalar_type() : -1;
        return norm_fwd(x, r, gamma, beta, eps, stats);
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        const Tensor& g = grads[0];
        const variable_list saved = ctx->get_saved_variables();
        const c10::DeviceGuard guard(g.device());
        const int64_t N = g.size(-1), M = g.numel() / N;
        saved_is(saved[0], "x", g.scalar_type(), M * N, g);
        const Rows x = rows_of(saved[0], N);
        const Tensor stats = saved_packed(saved[1], "statistics", at::kFloat, 2 * M, g);
        const Tensor gamma = saved_packed(saved[2], "gamma", (at::ScalarType)ctx->saved_data["gamma"].toInt(), N, g);
        const int64_t beta_type = ctx->saved_data["beta"].toInt();
        const bool has_gamma = gamma.defined(), has_beta = beta_type >= 0;      // edges are numbered over the present inputs
        const Rows r = rows_of(g, N);
        const Tensor dx = ctx->needs_input_grad(0) ? empty(g.sizes(), g.scalar_type(), g) : Tensor();
        const Tensor dgamma = has_gamma && ctx->needs_input_grad(1) ? empty({N}, gamma.scalar_type(), g) : Tensor();
        const Tensor dbeta = has_beta && ctx->needs_input_grad(1 + has_gamma) ? empty({N}, (at::ScalarType)beta_type, g) : Tensor();
        const int64_t need = dgamma.defined() || dbeta.defined() ? gm_layer_norm_bwd_workspace_bytes(M, N) : 0;
        const Tensor ws = workspace(need, g);
        const Tensor& wt = gamma.defined() ? gamma : dbeta;
        call(gm_layer_norm_bwd(M, N, at_of(r.t), r.ld, at_of(x.t), x.ld, row_dtype(g, "gradient"), floats(stats), M ? floats(stats) + M : nullptr,
                               at_of(gamma), row_dtype(wt.defined() ? wt : g, "gamma"), out_of<void>(dx), N, out_of<void>(dgamma),
                               out_of<void>(dbeta), out_of<void>(ws), need, stream_of(g)),
             "gm_layer_norm_bwd");
        return once({dx, dgamma, dbeta, Tensor()}, g);
    }
};

Tensor layer_norm(const Tensor& x, const std::optional<Tensor>& gamma_, const std::optional<Tensor>& beta_, double eps) {
    const int64_t N = x.dim() ? x.size(-1) : 0;
    if (N == 0) throw py::value_error(say("layer_norm: x must have a last dimension of at least 1, got ", x.sizes()));
    row_dtype(x, "x");
    no_tangent(x, "x");
    Tensor weights[2] = {gamma_.value_or(Tensor()), beta_.value_or(Tensor())};
    for (int k = 0; k < 2; ++k) {
        const Tensor& t = weights[k];
        const char* what = k ? "beta" : "gamma";
        if (!t.defined()) continue;
        if (t.dim() != 1 || t.numel() != N) throw py::value_error(say("layer_norm: ", what, " is ", t.sizes(), ", x's rows have ", N, " columns"));
        if (t.scalar_type() != x.scalar_type() && t.scalar_type() != at::kFloat)
            throw py::type_error(say("layer_norm: ", what, " is ", t.scalar_type(), ", expected ", x.scalar_type(), " or float32"));
        same_device(t, what, x);
        no_tangent(t, what);
    }
    if (weights[0].defined() && weights[1].defined() && weights[0].scalar_type() != weights[1].scalar_type())
        throw py::type_error(say("layer_norm: gamma is ", weights[0].scalar_type(), " and beta is ", weights[1].scalar_type()));
    if (!(eps >= 0.0)) throw py::value_error(say("layer_norm: eps must not be negative, got ", eps));
    on_gpu(x, "x");
    for (Tensor& t : weights)
        if (t.defined()) t = t.contiguous();
    if (records(x) | records(weights[0]) | records(weights[1])) {        // each of them is looked at
        auto given = [](const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; };
        return LayerNorm::apply(x, given(weights[0]), given(weights[1]), eps);
    }
    const c10::DeviceGuard guard(x.device());
    return norm_fwd(x, rows_of(x, N), weights[0], weights[1], eps, Tensor());
}

// ------------------------------------------------------------------ class_log_prob
Tensor log_prob_fwd(const Tensor& logits, const Rows& r, const Tensor& classes, int64_t ignore_index, const Tensor& stats) {
    const int64_t V = logits.size(-1), M = classes.numel();
    const int code = row_dtype(logits, "logits");
    Tensor lp = empty(classes.sizes(), at::kFloat, logits);
    const int64_t need = gm_class_log_prob_workspace_bytes(M, V, code);
    const Tensor ws = workspace(need, logits);
    call(gm_class_log_prob_fwd(M, V, at_of(r.t), r.ld, code, at_of(classes), is_i64(classes), ignore_index, out_of<float>(lp),
                               out_of<float>(stats), out_of<void>(ws), need, stream_of(logits)),
         "gm_class_log_prob_fwd");
    return lp;
}

struct ClassLogProb : torch::autograd::Function<ClassLogProb> {
    static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& classes, int64_t ignore_index) {
        const c10::DeviceGuard guard(logits.device());
        const Rows r = rows_of(logits, logits.size(-1));
        const int64_t need = gm_class_log_prob_stats_floats(classes.numel(), logits.size(-1), row_dtype(logits, "logits"));
        const Tensor stats = need > 0 ? empty({need}, at::kFloat, logits) : Tensor();
        ctx->save_for_backward({r.t, classes, stats});
        ctx->saved_data["type"] = type_code(logits);
        ctx->saved_data["classes"] = type_code(classes);
        ctx->saved_data["shape"] = logits.sizes().vec();
        ctx->saved_data["ignore"] = ignore_index;
        return log_prob_fwd(logits, r, classes, ignore_index, stats);
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        const Tensor g = grads[0].contiguous();
        const variable_list saved = ctx->get_saved_variables();
        const c10::DeviceGuard guard(g.device());
        const std::vector<int64_t> shape = ctx->saved_data["shape"].toIntVector();
        const auto type = (at::ScalarType)ctx->saved_data["type"].toInt();
        const int64_t V = shape.back(), M = g.numel();
        Tensor dx = empty(shape, type, g);
        const int code = row_dtype(dx, "logits");
        saved_is(saved[0], "logits", type, M * V, g);
        const Rows x = rows_of(saved[0], V);
        const Tensor classes = saved_packed(saved[1], "classes", (at::ScalarType)ctx->saved_data["classes"].toInt(), M, g);
        const Tensor stats = saved_packed(saved[2], "statistics", at::kFloat, gm_class_log_prob_stats_floats(M, V, code), g);
        call(gm_class_log_prob_bwd(M, V, floats(g), at_of(x.t), x.ld, code, at_of(classes),
                                   is_i64(classes), ctx->saved_data["ignore"].toInt(), floats(stats), out_of<void>(dx), V, stream_of(g)),
             "gm_class_log_prob_bwd");
        return once({dx, Tensor(), Tensor()}, g);
    }
};

Tensor class_log_prob(const Tensor& logits, const Tensor& classes, int64_t ignore_index) {
    const int64_t V = logits.dim() ? logits.size(-1) : 0;
    if (V == 0) throw py::value_error(say("class_log_prob: logits must have a last dimension of at least 1, got ", logits.sizes()));
    if (classes.sizes() != logits.sizes().slice(0, logits.dim() - 1))
        throw py::value_error(say("class_log_prob: classes is ", classes.sizes(), ", logits is ", logits.sizes()));
    row_dtype(logits, "logits");
    no_tangent(logits, "logits");
    const Tensor cls = index_of(classes, "classes", logits);
    on_gpu(logits, "logits");
    if (records(logits)) return ClassLogProb::apply(logits, cls, ignore_index);
    const c10::DeviceGuard guard(logits.device());
    return log_prob_fwd(logits, rows_of(logits, V), cls, ignore_index, Tensor());
}

// ------------------------------------------------------------------ losses over sequences
void constant(const Tensor& t, const char* what) {
    if (t.requires_grad()) throw py::value_error(say(what, " is a constant of the loss and gets no gradient: pass ", what, ".detach()"));
    no_tangent(t, what);
}
Tensor items(const Tensor& t, const char* what) {
    if (t.scalar_type() != at::kFloat) throw py::type_error(say(what, ": expected float32, got ", t.scalar_type()));
    return t;
}
// a per-item argument that takes no gradient
Tensor items_like(const Tensor& t, const char* what, const Tensor& like) {
    items(t, what);
    if (t.sizes() != like.sizes()) throw py::value_error(say(what, " is ", t.sizes(), ", log_prob is ", like.sizes()));
    constant(t, what);
    same_device(t, what, like);
    return t.contiguous();
}
Tensor mask_like(const std::optional<Tensor>& mask, const Tensor& like) {
    if (!mask || !mask->defined()) return Tensor();
    if (mask->scalar_type() != at::kBool && mask->scalar_type() != at::kByte)
        throw py::type_error(say("mask: expected bool or uint8, got ", mask->scalar_type()));
    if (mask->sizes() != like.sizes()) throw py::value_error(say("mask is ", mask->sizes(), ", log_prob is ", like.sizes()));
    same_device(*mask, "mask", like);
    return mask->contiguous();
}
Tensor offsets_of(const Tensor& t, const Tensor& like) {
    if (t.dim() != 1 || t.numel() < 2)
        throw py::value_error(say("offsets: expected the S + 1 borders of S > 0 sequences, got ", t.sizes()));
    return index_of(t, "offsets", like);
}

struct LossArgs {
    Tensor old, adv, ref, mask, offsets;
    int64_t S;
    double clip_low, clip_high, kl_coef, beta, smoothing;
    int by_sequence, average;
};

// what a loss keeps for its backward: the S weights, then the slopes
struct Kept {
    Tensor t;
    float *weight, *slope;
};
Kept kept_floats(int64_t S, int64_t slopes, const Tensor& like) {
    Kept k{empty({S + slopes}, at::kFloat, like), nullptr, nullptr};
    k.weight = out_of<float>(k.t);
    k.slope = slopes ? k.weight + S : nullptr;
    return k;
}
int64_t loss_workspace(int64_t M, int64_t S) {
    const int64_t need = gm_sequence_loss_workspace_bytes(M, S);
    if (need < 0) throw HipError("gm_sequence_loss_workspace_bytes: too many items or sequences");
    return need;
}

variable_list policy_fwd(const Tensor& lp, const LossArgs& a, bool grad, Tensor* kept) {
    const c10::DeviceGuard guard(lp.device());
    const Tensor l = lp.contiguous();
    const int64_t M = l.numel();
    Tensor loss = empty({}, at::kFloat, lp), stats = empty({4}, at::kFloat, lp);
    const int64_t need = loss_workspace(M, a.S);
    const Tensor ws = workspace(need, lp);
    const Kept k = kept_floats(a.S, grad ? M : 0, lp);
    call(gm_policy_loss_fwd(M, a.S, floats(l), floats(a.old), floats(a.adv), floats(a.ref), bytes(a.mask), at_of(a.offsets),
                            a.offsets.defined() && is_i64(a.offsets), (float)a.clip_low, (float)a.clip_high, (float)a.kl_coef, a.by_sequence,
                            out_of<float>(loss), out_of<float>(stats), k.slope, k.weight, out_of<void>(ws), need, stream_of(lp)),
         "gm_policy_loss_fwd");
    if (kept) *kept = k.t;
    return {loss, stats};
}
variable_list preference_fwd(const Tensor& lp, const LossArgs& a, Tensor* kept) {
    const c10::DeviceGuard guard(lp.device());
    const Tensor l = lp.contiguous();
    const int64_t M = l.numel();
    Tensor loss = empty({}, at::kFloat, lp), rewards = empty({a.S}, at::kFloat, lp);
    const int64_t need = loss_workspace(M, a.S);
    const Tensor ws = workspace(need, lp);
    const Kept k = kept_floats(a.S, 0, lp);
    call(gm_preference_loss_fwd(M, a.S / 2, floats(l), floats(a.ref), bytes(a.mask), at_of(a.offsets), is_i64(a.offsets), (float)a.beta,
                                (float)a.smoothing, a.average, out_of<float>(loss), out_of<float>(rewards), k.weight, out_of<void>(ws), need,
                                stream_of(lp)),
         "gm_preference_loss_fwd");
    if (kept) *kept = k.t;
    return {loss, rewards};
}

template <bool POLICY> struct SequenceLoss : torch::autograd::Function<SequenceLoss<POLICY>> {
    static variable_list forward(AutogradContext* ctx, const Tensor& lp, const LossArgs& a) {
        Tensor kept;
        variable_list out = POLICY ? policy_fwd(lp, a, true, &kept) : preference_fwd(lp, a, &kept);
        ctx->save_for_backward({kept, a.mask, a.offsets});
        ctx->saved_data["S"] = a.S;
        ctx->saved_data["shape"] = lp.sizes().vec();
        ctx->saved_data["mask"] = type_code(a.mask);
        ctx->saved_data["offsets"] = type_code(a.offsets);
        ctx->mark_non_differentiable({out[1]});
        ctx->set_materialize_grads(false);
        return out;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        if (!grads[0].defined()) return {Tensor(), Tensor()};
        const Tensor& g = grads[0];
        const variable_list saved = ctx->get_saved_variables();
        const c10::DeviceGuard guard(g.device());
        const int64_t S = ctx->saved_data["S"].toInt();
        Tensor dl = empty(ctx->saved_data["shape"].toIntVector(), at::kFloat, g);
        const int64_t M = dl.numel();
        const Tensor kept = saved_packed(saved[0], "weights", at::kFloat, POLICY ? S + M : S, g);
        const Tensor mask = saved_packed(saved[1], "mask", (at::ScalarType)ctx->saved_data["mask"].toInt(), M, g);
        const Tensor offsets = saved_packed(saved[2], "offsets", (at::ScalarType)ctx->saved_data["offsets"].toInt(), S + 1, g);
        const float* weight = floats(kept);
        call(gm_sequence_loss_bwd(M, S, POLICY ? weight + S : nullptr, bytes(mask), at_of(offsets), offsets.defined() && is_i64(offsets),
                                  weight, floats(g), out_of<float>(dl), stream_of(g)),
             "gm_sequence_loss_bwd");
        return once({dl, Tensor()}, g);
    }
};

std::pair<Tensor, Tensor> policy_loss(const Tensor& log_prob, const Tensor& old_log_prob, const Tensor& advantage,
                                      const std::optional<Tensor>& offsets, const std::optional<Tensor>& mask,
                                      const std::optional<Tensor>& ref_log_prob, double clip_low, double clip_high, double kl_coef,
                                      const std::string& reduction) {
    LossArgs a{};
    a.S = 1;
    items(log_prob, "log_prob");
    no_tangent(log_prob, "log_prob");
    a.old = items_like(old_log_prob, "old_log_prob", log_prob);
    if (ref_log_prob && ref_log_prob->defined()) a.ref = items_like(*ref_log_prob, "ref_log_prob", log_prob);
    a.mask = mask_like(mask, log_prob);
    if (offsets && offsets->defined()) {
        a.offsets = offsets_of(*offsets, log_prob);
        a.S = a.offsets.numel() - 1;
        items(advantage, "advantage");
        same_device(advantage, "advantage", log_prob);
        constant(advantage, "advantage");
        if (advantage.dim() != 1 || advantage.numel() != a.S)
            throw py::value_error(say("advantage is ", advantage.sizes(), ", offsets border ", a.S, " sequences"));
        a.adv = advantage.contiguous();
    } else {
        a.adv = items_like(advantage, "advantage", log_prob);
    }
    if (reduction != "token" && reduction != "sequence")
        throw py::value_error(say("reduction: expected 'token' or 'sequence', got '", reduction, "'"));
    a.by_sequence = reduction == "sequence";
    if (a.by_sequence && !a.offsets.defined()) throw py::value_error("reduction 'sequence' needs offsets");
    if (!(clip_low >= 0.0 && clip_low <= 1.0 && clip_high >= 0.0 && std::isfinite(clip_high)))
        throw py::value_error(say("clip range: 0 <= clip_low <= 1 and 0 <= clip_high, got ", clip_low, ", ", clip_high));
    if (!std::isfinite(kl_coef)) throw py::value_error(say("kl_coef must be finite, got ", kl_coef));
    if (kl_coef != 0.0 && !a.ref.defined()) throw py::value_error("kl_coef needs ref_log_prob");
    on_gpu(log_prob, "log_prob");
    a.clip_low = clip_low;
    a.clip_high = clip_high;
    a.kl_coef = kl_coef;
    const variable_list out = records(log_prob) ? SequenceLoss<true>::apply(log_prob, a) : policy_fwd(log_prob, a, false, nullptr);
    return {out[0], out[1]};
}

std::pair<Tensor, Tensor> preference_loss(const Tensor& log_prob, const Tensor& ref_log_prob, const Tensor& offsets,
                                          const std::optional<Tensor>& mask, double beta, double label_smoothing, bool average) {
    LossArgs a{};
    items(log_prob, "log_prob");
    no_tangent(log_prob, "log_prob");
    a.ref = items_like(ref_log_prob, "ref_log_prob", log_prob);
    a.mask = mask_like(mask, log_prob);
    a.offsets = offsets_of(offsets, log_prob);
    a.S = a.offsets.numel() - 1;
    if (a.S % 2) throw py::value_error(say("offsets border ", a.S, " sequences: an even number makes pairs"));
    if (!(beta > 0.0 && std::isfinite(beta) && label_smoothing >= 0.0 && label_smoothing <= 0.5))
        throw py::value_error(say("0 < beta and 0 <= label_smoothing <= 0.5, got ", beta, ", ", label_smoothing));
    on_gpu(log_prob, "log_prob");
    a.beta = beta;
    a.smoothing = label_smoothing;
    a.average = average;
    const variable_list out = records(log_prob) ? SequenceLoss<false>::apply(log_prob, a) : preference_fwd(log_prob, a, nullptr);
    return {out[0], out[1]};
}

}  // namespace

PYBIND11_MODULE(gm_tape, m) {
    static py::handle error_class;          // graphmaker_amd._lib.GraphMakerHipError, held for the life of the process
    m.def("set_error_class", [](py::object cls) { error_class = cls.release(); });
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const HipError& e) {
            PyErr_SetString(error_class ? error_class.ptr() : PyExc_RuntimeError, e.what());
        } catch (const c10::Error&) {                  // torch's own, such as running out of memory
            torch::translate_exception_to_python(p);
        }
    });
    const py::call_guard<py::gil_scoped_release> no_lock;
    m.def("token_embedding", &token_embedding, no_lock);
    m.def("layer_norm", &layer_norm, no_lock);
    m.def("class_log_prob", &class_log_prob, no_lock);
    m.def("policy_loss", &policy_loss, no_lock);
    m.def("preference_loss", &preference_loss, no_lock);
}
