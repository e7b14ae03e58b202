// Operators either side of the experts' products and of the head's, over libtorch's C++ API as in
// torch_ext.cpp: the router of a mixture-of-experts layer, its balance loss, rows sorted by expert and back
// (moe_router, moe_balance_loss, moe_dispatch, moe_combine, with their gradients) and the rules on a
// generation step's logits (logit_rules).
#include <ATen/MemoryOverlap.h>
#include <c10/util/ScopeExit.h>

#include <mutex>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/dynamo/compiled_autograd.h>

#include "torch_ext.h"

namespace {

using namespace tgo_ext;

int type_code(const Tensor& logits) {
    switch (logits.scalar_type()) {
        case at::kBFloat16: return TGO_BF16;
        case at::kHalf: return TGO_FP16;
        case at::kFloat: return TGO_FP32;
        default: TORCH_CHECK(false, "logits must have dtype torch.bfloat16, torch.float16 or torch.float32; got ", logits.scalar_type());
    }
}
// [..., width] as rows: a matrix whose rows may lie apart, or anything contiguous
struct Rows {
    int64_t rows, width, stride;
};
Rows as_rows(const Tensor& t, const char* name) {
    TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(t.dim() >= 1, name, " must have at least one dimension");
    const int64_t width = t.size(-1);
    TORCH_CHECK(width > 0, name, " must not be empty in its last dimension");
    const int64_t rows = t.numel() / width;
    if (t.is_contiguous()) return {rows, width, width};
    TORCH_CHECK(t.dim() == 2 && (width == 1 || t.stride(1) == 1) && t.stride(0) >= width, name,
                " must be contiguous, or a matrix whose rows lie apart; torch_ggml_ops will not insert a hidden copy");
    return {rows, width, t.stride(0)};
}
void check_plain(const Tensor& t, const Tensor& like, at::ScalarType type, const char* name) {
    TORCH_CHECK(t.device() == like.device() && t.scalar_type() == type && t.is_contiguous(), name, " must be a contiguous ", type,
                " tensor on the other inputs' device; torch_ggml_ops will not insert a hidden copy");
}
std::vector<int64_t> with_last(at::IntArrayRef sizes, int64_t last) {
    std::vector<int64_t> v = sizes.vec();
    v.back() = last;
    return v;
}

// ------------------------------------------------------------------ formulas
// As nodes of the graph themselves and not by way of Function, whose context costs some 4 us of a forward and backward pass of 58.
using torch::autograd::SavedVariable;
struct Formula : public torch::autograd::Node {
    using Node::Node;
    std::vector<SavedVariable> kept;
    SavedVariable result;             // the node's own, where a formula needs it
    int64_t scoring = 0;
    bool norm = true;
    c10::SymInt rows = 0;             // a size that a formula needs of an input that it does not keep
    void keep(std::initializer_list<Tensor> inputs) {
        for (const Tensor& t : inputs) kept.emplace_back(t, false);
    }
    variable_list apply(variable_list&& g) override {
        const std::lock_guard<std::mutex> lock(mutex_);
        variable_list d(num_outputs());
        if (g[0].defined()) gradients(g[0], d);
        return d;
    }
    void release_variables() override {
        const std::lock_guard<std::mutex> lock(mutex_);
        for (SavedVariable& v : kept) v.reset_data();
        result.reset_data();
    }
    // for compiled autograd: what is kept, what a traced graph is specialised on, and the formula with traced tensors in the place of the kept ones
    void compiled_args(torch::dynamo::autograd::CompiledNodeArgs& args) const override {
        args.collect(kept, false);
        args.collect(result, true);
        args.collect(scoring);
        args.collect(norm);
        args.collect(rows);
    }
    variable_list apply_with_saved(const variable_list& inputs, torch::dynamo::autograd::SwapSavedVariables& saved) override {
        saved.before(kept);
        saved.before(result);
        saved.before(rows);
        const auto back = c10::make_scope_exit([&] {
            saved.after(kept);
            saved.after(result);
            saved.after(rows);
        });
        return apply(variable_list(inputs));
    }
    virtual void gradients(const Tensor& g, variable_list& d) = 0;
};
// a node whose inputs are `inputs`; an undefined one has no edge
template <typename N>
std::shared_ptr<N> formula(std::initializer_list<Tensor> inputs) {
    torch::autograd::edge_list next;
    for (const Tensor& t : inputs) next.push_back(t.defined() ? torch::autograd::impl::gradient_edge(t) : torch::autograd::Edge());
    return std::shared_ptr<N>(new N(std::move(next)), torch::autograd::deleteNode);
}

// ------------------------------------------------------------------ moe_router
void check_router(const Rows& r, int64_t top_k, int64_t scoring) {
    TORCH_CHECK(r.width <= 1024, "the router takes up to 1024 experts; got ", r.width);
    TORCH_CHECK(top_k >= 1 && top_k <= 32 && top_k <= r.width, "top_k must be in 1..32 and at most the number of experts; got ", top_k);
    TORCH_CHECK(scoring == TGO_SCORING_SOFTMAX || scoring == TGO_SCORING_SIGMOID, "unknown scoring");
}
std::tuple<Tensor, Tensor> router_cuda(const Tensor& logits, int64_t top_k, int64_t scoring, bool normalize, const std::optional<Tensor>& mask) {
    const int code = type_code(logits);
    const Rows r = as_rows(logits, "logits");
    check_router(r, top_k, scoring);
    if (mask.has_value()) {
        check_plain(*mask, logits, at::kBool, "token_mask");
        TORCH_CHECK(mask->sizes() == logits.sizes().slice(0, logits.dim() - 1), "token_mask must have one entry per token");
    }
    const c10::cuda::CUDAGuard guard(logits.device());
    const auto sizes = with_last(logits.sizes(), top_k);
    Tensor w = new_cuda(sizes, at::kFloat, logits), ids = new_cuda(sizes, at::kInt, logits);
    if (r.rows > 0)
        check_rc(tgo_moe_router(logits.const_data_ptr(), code, r.rows, r.width, r.stride, top_k, static_cast<int>(scoring), normalize,
                                mask.has_value() ? reinterpret_cast<const uint8_t*>(mask->const_data_ptr<bool>()) : nullptr,
                                w.mutable_data_ptr<float>(), ids.mutable_data_ptr<int32_t>(), stream_of(logits)),
                 "moe_router");
    return {w, ids};
}
Tensor router_grad_cuda(const Tensor& grad, const Tensor& logits, const Tensor& ids, const Tensor& w, int64_t scoring, bool normalize) {
    const int code = type_code(logits);
    const Rows r = as_rows(logits, "logits");
    check_plain(ids, logits, at::kInt, "expert_ids");
    check_plain(w, logits, at::kFloat, "weights");
    TORCH_CHECK(grad.sizes() == w.sizes() && grad.scalar_type() == at::kFloat && grad.device() == w.device() && ids.sizes() == w.sizes() &&
                    w.dim() == logits.dim() && w.sizes().slice(0, w.dim() - 1) == logits.sizes().slice(0, w.dim() - 1),
                "grad, expert_ids and weights must be tensors of one shape, one row per token");
    check_router(r, w.size(-1), scoring);
    const c10::cuda::CUDAGuard guard(logits.device());
    const Tensor d = grad.contiguous();
    Tensor dx = new_cuda(logits.sizes(), logits.scalar_type(), logits);
    if (r.rows > 0)
        check_rc(tgo_moe_router_grad(logits.const_data_ptr(), code, r.rows, r.width, r.stride, ids.const_data_ptr<int32_t>(),
                                     w.const_data_ptr<float>(), d.const_data_ptr<float>(), w.size(-1), static_cast<int>(scoring), normalize,
                                     dx.mutable_data_ptr(), stream_of(logits)),
                 "moe_router_grad");
    return dx;
}
std::tuple<Tensor, Tensor> call_router(const Tensor& x, int64_t k, int64_t scoring, bool norm, const std::optional<Tensor>& mask) {
    static const auto h = op<std::tuple<Tensor, Tensor>(const Tensor&, int64_t, int64_t, bool, const std::optional<Tensor>&)>(
        "torch_ggml_ops_b200::moe_router");
    return h.call(x, k, scoring, norm, mask);
}
Tensor call_router_grad(const Tensor& g, const Tensor& x, const Tensor& ids, const Tensor& w, int64_t scoring, bool norm) {
    static const auto h = op<Tensor(const Tensor&, const Tensor&, const Tensor&, const Tensor&, int64_t, bool)>(
        "torch_ggml_ops_b200::moe_router_grad");
    return h.call(g, x, ids, w, scoring, norm);
}
[[noreturn]] void once_only(const char* name) {
    TORCH_CHECK(false, "torch_ggml_ops_b200::", name, " does not support higher-order gradients");
}
struct RouterFormula : public Formula {
    using Formula::Formula;
    void gradients(const Tensor& g, variable_list& d) override {
        if (task_should_compute_output(0))
            d[0] = call_router_grad(g, kept[0].unpack(), kept[1].unpack(), result.unpack(shared_from_this()), scoring, norm);
    }
    std::string name() const override { return "MoeRouterBackward"; }
};
std::tuple<Tensor, Tensor> router_autograd(const Tensor& x, int64_t k, int64_t scoring, bool norm, const std::optional<Tensor>& mask) {
    if (!wants_grad(x)) {
        at::AutoDispatchBelowADInplaceOrView guard;
        return call_router(x, k, scoring, norm, mask);
    }
    const auto node = formula<RouterFormula>({x});
    Tensor w, ids;
    {
        at::AutoDispatchBelowADInplaceOrView guard;
        std::tie(w, ids) = call_router(x, k, scoring, norm, mask);
    }
    torch::autograd::set_history(w, node);
    node->keep({x, ids});
    node->result = SavedVariable(w, true);
    node->scoring = scoring;
    node->norm = norm;
    return {std::move(w), std::move(ids)};
}
struct RouterGradFn : public Function<RouterGradFn> {
    static Tensor forward(AutogradContext*, const Tensor& g, const Tensor& x, const Tensor& ids, const Tensor& w, int64_t scoring, bool norm) {
        at::AutoDispatchBelowADInplaceOrView guard;
        return call_router_grad(g, x, ids, w, scoring, norm);
    }
    static tensor_list backward(AutogradContext*, tensor_list) { once_only("moe_router_grad"); }
};
Tensor router_grad_autograd(const Tensor& g, const Tensor& x, const Tensor& ids, const Tensor& w, int64_t scoring, bool norm) {
    if (wants_grad(g, x, w)) return RouterGradFn::apply(g, x, ids, w, scoring, norm);
    at::AutoDispatchBelowADInplaceOrView guard;
    return call_router_grad(g, x, ids, w, scoring, norm);
}

// ------------------------------------------------------------------ moe_balance_loss
void check_ids(const Tensor& ids, const Tensor& tokens, const char* of) {
    check_plain(ids, tokens, at::kInt, "expert_ids");
    TORCH_CHECK(ids.dim() == tokens.dim() && ids.sizes().slice(0, ids.dim() - 1) == tokens.sizes().slice(0, ids.dim() - 1),
                "expert_ids must have one row per row of ", of);
}
std::tuple<Tensor, Tensor, Tensor> balance_cuda(const Tensor& logits, const Tensor& ids, int64_t scoring) {
    const int code = type_code(logits);
    const Rows r = as_rows(logits, "logits");
    check_ids(ids, logits, "logits");
    check_router(r, ids.size(-1), scoring);
    const c10::cuda::CUDAGuard guard(logits.device());
    const auto f32 = logits.options().dtype(at::kFloat);
    if (r.rows == 0) return {at::zeros({}, f32), at::zeros({r.width}, f32.dtype(at::kInt)), at::zeros({r.width}, f32)};
    Tensor loss = new_cuda({}, at::kFloat, logits), counts = new_cuda({r.width}, at::kInt, logits), coef = new_cuda({r.width}, at::kFloat, logits);
    const int64_t bytes = tgo_moe_balance_workspace_bytes(r.rows, r.width);
    TORCH_CHECK(bytes >= 0, "unsupported sizes");
    Tensor ws = new_cuda({bytes}, at::kByte, logits);
    check_rc(tgo_moe_balance_loss(logits.const_data_ptr(), code, r.rows, r.width, r.stride, ids.const_data_ptr<int32_t>(), ids.size(-1),
                                  static_cast<int>(scoring), loss.mutable_data_ptr<float>(), counts.mutable_data_ptr<int32_t>(),
                                  coef.mutable_data_ptr<float>(), ws.mutable_data_ptr(), bytes, stream_of(logits)),
             "moe_balance_loss");
    return {loss, counts, coef};
}
Tensor balance_grad_cuda(const Tensor& grad, const Tensor& logits, const Tensor& ids, const Tensor& coef, int64_t scoring) {
    const int code = type_code(logits);
    const Rows r = as_rows(logits, "logits");
    check_ids(ids, logits, "logits");
    check_router(r, ids.size(-1), scoring);
    check_plain(coef, logits, at::kFloat, "coef");
    TORCH_CHECK(coef.numel() == r.width, "coef must have one entry per expert");
    check_plain(grad, logits, at::kFloat, "grad");
    TORCH_CHECK(grad.numel() == 1, "grad must be one number");
    const c10::cuda::CUDAGuard guard(logits.device());
    Tensor dx = new_cuda(logits.sizes(), logits.scalar_type(), logits);
    if (r.rows > 0)
        check_rc(tgo_moe_balance_grad(logits.const_data_ptr(), code, r.rows, r.width, r.stride, ids.const_data_ptr<int32_t>(), ids.size(-1),
                                      static_cast<int>(scoring), coef.const_data_ptr<float>(), grad.const_data_ptr<float>(),
                                      dx.mutable_data_ptr(), stream_of(logits)),
                 "moe_balance_grad");
    return dx;
}
std::tuple<Tensor, Tensor, Tensor> call_balance(const Tensor& x, const Tensor& ids, int64_t scoring) {
    static const auto h = op<std::tuple<Tensor, Tensor, Tensor>(const Tensor&, const Tensor&, int64_t)>("torch_ggml_ops_b200::moe_balance_loss");
    return h.call(x, ids, scoring);
}
Tensor call_balance_grad(const Tensor& g, const Tensor& x, const Tensor& ids, const Tensor& coef, int64_t scoring) {
    static const auto h = op<Tensor(const Tensor&, const Tensor&, const Tensor&, const Tensor&, int64_t)>("torch_ggml_ops_b200::moe_balance_grad");
    return h.call(g, x, ids, coef, scoring);
}
struct BalanceFormula : public Formula {
    using Formula::Formula;
    void gradients(const Tensor& g, variable_list& d) override {
        if (task_should_compute_output(0)) d[0] = call_balance_grad(g, kept[0].unpack(), kept[1].unpack(), kept[2].unpack(), scoring);
    }
    std::string name() const override { return "MoeBalanceLossBackward"; }
};
std::tuple<Tensor, Tensor, Tensor> balance_autograd(const Tensor& x, const Tensor& ids, int64_t scoring) {
    if (!wants_grad(x)) {
        at::AutoDispatchBelowADInplaceOrView guard;
        return call_balance(x, ids, scoring);
    }
    const auto node = formula<BalanceFormula>({x});
    Tensor loss, counts, coef;
    {
        at::AutoDispatchBelowADInplaceOrView guard;
        std::tie(loss, counts, coef) = call_balance(x, ids, scoring);
    }
    torch::autograd::set_history(loss, node);
    node->keep({x, ids, coef});
    node->scoring = scoring;
    return {std::move(loss), std::move(counts), std::move(coef)};
}
struct BalanceGradFn : public Function<BalanceGradFn> {
    static Tensor forward(AutogradContext*, const Tensor& g, const Tensor& x, const Tensor& ids, const Tensor& coef, int64_t scoring) {
        at::AutoDispatchBelowADInplaceOrView guard;
        return call_balance_grad(g, x, ids, coef, scoring);
    }
    static tensor_list backward(AutogradContext*, tensor_list) { once_only("moe_balance_grad"); }
};
Tensor balance_grad_autograd(const Tensor& g, const Tensor& x, const Tensor& ids, const Tensor& coef, int64_t scoring) {
    if (wants_grad(g, x, coef)) return BalanceGradFn::apply(g, x, ids, coef, scoring);
    at::AutoDispatchBelowADInplaceOrView guard;
    return call_balance_grad(g, x, ids, coef, scoring);
}

// ------------------------------------------------------------------ moe_dispatch and moe_combine
void check_moved(const Tensor& t, const char* name) {
    TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(t.scalar_type() == at::kBFloat16 && t.is_contiguous() && reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0, name,
                " must be a contiguous torch.bfloat16 tensor that starts at a multiple of 16 bytes; torch_ggml_ops will not insert a hidden copy");
    TORCH_CHECK(t.dim() >= 1 && t.size(-1) > 0 && t.size(-1) % 8 == 0, name, " must have rows whose length is a positive multiple of 8");
}
void check_pairs(int64_t pairs, int64_t top_k) {
    TORCH_CHECK(top_k >= 1 && top_k <= 1024, "top_k must be in 1..1024; got ", top_k);
    TORCH_CHECK(pairs <= INT32_MAX, "tokens * top_k must be below 2^31; got ", pairs);
}
std::tuple<Tensor, Tensor, Tensor, Tensor> dispatch_cuda(const Tensor& x, const Tensor& ids, int64_t experts) {
    check_moved(x, "input");
    TORCH_CHECK(ids.dim() >= 1, "expert_ids must have one row per row of input");
    check_ids(ids, x, "input");
    const int64_t h = x.size(-1), tokens = x.numel() / h, k = ids.size(-1), pairs = ids.numel();
    check_pairs(pairs, k);
    TORCH_CHECK(experts >= 1 && experts <= 4096, "num_experts must be in 1..4096; got ", experts);
    const c10::cuda::CUDAGuard guard(x.device());
    const auto i32 = ids.options(), i64 = i32.dtype(at::kLong);
    Tensor rows = new_cuda({pairs, h}, at::kBFloat16, x), at_row = new_cuda(ids.sizes(), at::kInt, x);
    if (pairs == 0) return {rows, at_row, at::arange(experts, i64), at::zeros({experts}, i32)};
    Tensor indices = new_cuda({experts}, at::kLong, x), offsets = new_cuda({experts}, at::kInt, x);
    const int64_t bytes = tgo_moe_dispatch_workspace_bytes(pairs, experts);
    TORCH_CHECK(bytes >= 0, "unsupported sizes");
    const Tensor ws = bytes > 0 ? new_cuda({bytes}, at::kByte, x) : Tensor();
    check_rc(tgo_moe_dispatch(x.const_data_ptr(), ids.const_data_ptr<int32_t>(), tokens, k, experts, h, rows.mutable_data_ptr(),
                              at_row.mutable_data_ptr<int32_t>(), indices.mutable_data_ptr<int64_t>(), offsets.mutable_data_ptr<int32_t>(),
                              bytes > 0 ? ws.mutable_data_ptr() : nullptr, bytes, stream_of(x)),
             "moe_dispatch");
    return {rows, at_row, indices, offsets};
}
void check_map(const Tensor& at_row, const std::optional<Tensor>& w, const Tensor& like) {
    check_plain(at_row, like, at::kInt, "row_of_pair");
    TORCH_CHECK(at_row.dim() >= 1, "row_of_pair must have shape [..., top_k]");
    check_pairs(at_row.numel(), at_row.size(-1));
    if (w.has_value()) {
        check_plain(*w, like, at::kFloat, "weights");
        TORCH_CHECK(w->sizes() == at_row.sizes(), "weights must have one entry per pair");
    }
}
void check_combine(const Tensor& rows, const Tensor& at_row, const std::optional<Tensor>& w) {
    check_moved(rows, "rows");
    TORCH_CHECK(rows.dim() == 2, "rows must have shape [rows, width]");
    TORCH_CHECK(rows.size(0) <= INT32_MAX, "too many rows");
    check_map(at_row, w, rows);
}
Tensor combine_run(const Tensor& rows, const Tensor& at_row, const std::optional<Tensor>& w) {
    const int64_t h = rows.size(1), k = at_row.size(-1), tokens = at_row.numel() / k;
    const c10::cuda::CUDAGuard guard(rows.device());
    const auto sizes = with_last(at_row.sizes(), h);
    if (rows.size(0) == 0) return at::zeros(sizes, rows.options());
    Tensor out = new_cuda(sizes, at::kBFloat16, rows);
    if (tokens > 0)
        check_rc(tgo_moe_combine(rows.const_data_ptr(), rows.size(0), at_row.const_data_ptr<int32_t>(),
                                 w.has_value() ? w->const_data_ptr<float>() : nullptr, out.mutable_data_ptr(), tokens, k, h, stream_of(rows)),
                 "moe_combine");
    return out;
}
Tensor combine_cuda(const Tensor& rows, const Tensor& at_row, const std::optional<Tensor>& w) {
    check_combine(rows, at_row, w);
    return combine_run(rows, at_row, w);
}
// A cotangent is what autograd makes of it: a view of a larger tensor that starts anywhere, or no plain rows at all.
Tensor plain_rows(const Tensor& grad) {
    const Tensor d = grad.contiguous();
    return reinterpret_cast<uintptr_t>(d.const_data_ptr()) % 16 == 0 ? d : d.clone();
}
// the gradient of dispatch: a token's sum over its pairs' rows
Tensor dispatch_grad_cuda(const Tensor& grad, const Tensor& at_row) {
    TORCH_CHECK(grad.is_cuda() && grad.scalar_type() == at::kBFloat16 && grad.dim() == 2 && grad.size(1) > 0 && grad.size(1) % 8 == 0 && grad.size(0) <= INT32_MAX,
                "grad must be a torch.bfloat16 tensor like the rows");
    check_map(at_row, std::nullopt, grad);
    const c10::cuda::CUDAGuard guard(grad.device());
    return combine_run(plain_rows(grad), at_row, std::nullopt);
}
// The gradients of combine: of `rows` where n_rows is no less than 0, of the weights where `rows` are there.
std::tuple<Tensor, Tensor> combine_grads(const Tensor& grad, const std::optional<Tensor>& rows, int64_t n_rows, const Tensor& at_row,
                                         const std::optional<Tensor>& w) {
    const int64_t h = grad.size(-1), k = at_row.size(-1), tokens = at_row.numel() / k;
    const bool need_rows = n_rows >= 0, need_weights = rows.has_value();
    const Tensor d = plain_rows(grad);
    Tensor d_rows = new_cuda({need_rows ? n_rows : 0, h}, at::kBFloat16, grad);
    Tensor d_w = need_weights ? new_cuda(at_row.sizes(), at::kFloat, grad) : new_cuda({0}, at::kFloat, grad);
    if (!need_rows && !need_weights) return {d_rows, d_w};
    const int64_t existing = need_weights ? rows->size(0) : n_rows;
    if (existing == 0 || tokens == 0) return {d_rows.zero_(), d_w.zero_()};
    const int64_t bytes = need_rows ? tgo_moe_combine_grad_workspace_bytes(at_row.numel(), n_rows) : 0;
    const Tensor ws = bytes > 0 ? new_cuda({bytes}, at::kByte, grad) : Tensor();
    check_rc(tgo_moe_combine_grad(d.const_data_ptr(), need_weights ? rows->const_data_ptr() : nullptr, existing, at_row.const_data_ptr<int32_t>(),
                                  w.has_value() ? w->const_data_ptr<float>() : nullptr, need_rows ? d_rows.mutable_data_ptr() : nullptr,
                                  need_weights ? d_w.mutable_data_ptr<float>() : nullptr, tokens, k, h, bytes > 0 ? ws.mutable_data_ptr() : nullptr,
                                  bytes, stream_of(grad)),
             "moe_combine_grad");
    return {d_rows, d_w};
}
void check_result_grad(const Tensor& grad, const Tensor& at_row) {
    TORCH_CHECK(grad.is_cuda() && grad.device() == at_row.device() && grad.scalar_type() == at::kBFloat16 && grad.dim() == at_row.dim() &&
                    grad.sizes().slice(0, grad.dim() - 1) == at_row.sizes().slice(0, grad.dim() - 1),
                "grad must be a torch.bfloat16 tensor like the result");
}
// an empty tensor in the place of a gradient that is not wanted
std::tuple<Tensor, Tensor> combine_grad_cuda(const Tensor& grad, const Tensor& rows, const Tensor& at_row, const std::optional<Tensor>& w, bool need_rows,
                                             bool need_weights) {
    check_combine(rows, at_row, w);
    check_result_grad(grad, at_row);
    TORCH_CHECK(grad.size(-1) == rows.size(1), "grad must be a torch.bfloat16 tensor like the result");
    const c10::cuda::CUDAGuard guard(rows.device());
    return combine_grads(grad, need_weights ? std::optional<Tensor>(rows) : std::nullopt, need_rows ? rows.size(0) : -1, at_row, w);
}
// the gradient of the rows alone, for which the rows themselves are not needed
Tensor combine_rows_grad_cuda(const Tensor& grad, const Tensor& at_row, const std::optional<Tensor>& w, int64_t n_rows) {
    TORCH_CHECK(n_rows >= 0 && n_rows <= INT32_MAX, "the number of rows must be in 0..2^31-1; got ", n_rows);
    check_map(at_row, w, grad);
    check_result_grad(grad, at_row);
    TORCH_CHECK(grad.size(-1) > 0 && grad.size(-1) % 8 == 0, "grad must have rows whose length is a positive multiple of 8");
    const c10::cuda::CUDAGuard guard(grad.device());
    return std::get<0>(combine_grads(grad, std::nullopt, n_rows, at_row, w));
}
std::tuple<Tensor, Tensor, Tensor, Tensor> call_dispatch(const Tensor& x, const Tensor& ids, int64_t experts) {
    static const auto h = op<std::tuple<Tensor, Tensor, Tensor, Tensor>(const Tensor&, const Tensor&, int64_t)>("torch_ggml_ops_b200::moe_dispatch");
    return h.call(x, ids, experts);
}
Tensor call_combine(const Tensor& rows, const Tensor& at_row, const std::optional<Tensor>& w) {
    static const auto h = op<Tensor(const Tensor&, const Tensor&, const std::optional<Tensor>&)>("torch_ggml_ops_b200::moe_combine");
    return h.call(rows, at_row, w);
}
std::tuple<Tensor, Tensor> call_combine_grad(const Tensor& g, const Tensor& rows, const Tensor& at_row, const std::optional<Tensor>& w, bool need_rows,
                                             bool need_weights) {
    static const auto h = op<std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const std::optional<Tensor>&, bool, bool)>(
        "torch_ggml_ops_b200::moe_combine_grad");
    return h.call(g, rows, at_row, w, need_rows, need_weights);
}
Tensor call_combine_rows_grad(const Tensor& g, const Tensor& at_row, const std::optional<Tensor>& w, c10::SymInt n_rows) {
    static const auto h = op<Tensor(const Tensor&, const Tensor&, const std::optional<Tensor>&, c10::SymInt)>("torch_ggml_ops_b200::moe_combine_rows_grad");
    return h.call(g, at_row, w, std::move(n_rows));
}
Tensor call_dispatch_grad(const Tensor& g, const Tensor& at_row) {
    static const auto h = op<Tensor(const Tensor&, const Tensor&)>("torch_ggml_ops_b200::moe_dispatch_grad");
    return h.call(g, at_row);
}
struct DispatchFormula : public Formula {
    using Formula::Formula;
    void gradients(const Tensor& g, variable_list& d) override {
        if (task_should_compute_output(0)) d[0] = call_dispatch_grad(g, kept[0].unpack());
    }
    std::string name() const override { return "MoeDispatchBackward"; }
};
// dispatch is linear, its gradient, too
struct DispatchGradFormula : public Formula {
    using Formula::Formula;
    void gradients(const Tensor& g, variable_list& d) override {
        if (task_should_compute_output(0)) d[0] = call_combine_rows_grad(g, kept[0].unpack(), std::nullopt, rows);
    }
    std::string name() const override { return "MoeDispatchGradBackward"; }
};
Tensor dispatch_grad_autograd(const Tensor& g, const Tensor& at_row) {
    if (!wants_grad(g)) {
        at::AutoDispatchBelowADInplaceOrView guard;
        return call_dispatch_grad(g, at_row);
    }
    const auto node = formula<DispatchGradFormula>({g});
    Tensor d;
    {
        at::AutoDispatchBelowADInplaceOrView guard;
        d = call_dispatch_grad(g, at_row);
    }
    torch::autograd::set_history(d, node);
    node->keep({at_row});
    node->rows = g.sym_size(0);
    return d;
}
std::tuple<Tensor, Tensor, Tensor, Tensor> dispatch_autograd(const Tensor& x, const Tensor& ids, int64_t experts) {
    if (!wants_grad(x)) {
        at::AutoDispatchBelowADInplaceOrView guard;
        return call_dispatch(x, ids, experts);
    }
    const auto node = formula<DispatchFormula>({x});
    Tensor rows, at_row, indices, offsets;
    {
        at::AutoDispatchBelowADInplaceOrView guard;
        std::tie(rows, at_row, indices, offsets) = call_dispatch(x, ids, experts);
    }
    torch::autograd::set_history(rows, node);
    node->keep({at_row});
    return {std::move(rows), std::move(at_row), std::move(indices), std::move(offsets)};
}
// Keeps the map; the weights, where the rows want a gradient; the rows, where the weights do.  What is kept is handed on, needed for the gradients
// asked for or not: compiled autograd wants a use of all that it unpacks.
struct CombineFormula : public Formula {
    using Formula::Formula;
    void gradients(const Tensor& g, variable_list& d) override {
        const bool need_rows = task_should_compute_output(0), need_w = task_should_compute_output(1);
        if (!need_rows && !need_w) return;
        const Tensor at_row = kept[0].unpack(), kept_w = kept[1].unpack(), kept_rows = kept[2].unpack();
        const std::optional<Tensor> w = kept_w.defined() ? std::optional<Tensor>(kept_w) : std::nullopt;
        if (!kept_rows.defined()) {
            d[0] = call_combine_rows_grad(g, at_row, w, rows);
            return;
        }
        auto [a, b] = call_combine_grad(g, kept_rows, at_row, w, need_rows, need_w);
        if (need_rows) d[0] = a;
        if (need_w) d[1] = b;
    }
    std::string name() const override { return "MoeCombineBackward"; }
};
Tensor combine_autograd(const Tensor& rows, const Tensor& at_row, const std::optional<Tensor>& w) {
    if (!wants_grad(rows, w)) {
        at::AutoDispatchBelowADInplaceOrView guard;
        return call_combine(rows, at_row, w);
    }
    const bool of_weights = w.has_value() && w->requires_grad();
    const auto node = formula<CombineFormula>({rows, w.has_value() ? *w : Tensor()});
    Tensor y;
    {
        at::AutoDispatchBelowADInplaceOrView guard;
        y = call_combine(rows, at_row, w);
    }
    torch::autograd::set_history(y, node);
    node->keep({at_row, w.has_value() && rows.requires_grad() ? *w : Tensor(), of_weights ? rows : Tensor()});
    node->rows = rows.sym_size(0);
    return y;
}
struct CombineGradFn : public Function<CombineGradFn> {
    static variable_list forward(AutogradContext*, const Tensor& g, const Tensor& rows, const Tensor& at_row, const std::optional<Tensor>& w, bool need_rows,
                                 bool need_weights) {
        at::AutoDispatchBelowADInplaceOrView guard;
        auto [a, b] = call_combine_grad(g, rows, at_row, w, need_rows, need_weights);
        return {a, b};
    }
    static tensor_list backward(AutogradContext*, tensor_list) { once_only("moe_combine_grad"); }
};
std::tuple<Tensor, Tensor> combine_grad_autograd(const Tensor& g, const Tensor& rows, const Tensor& at_row, const std::optional<Tensor>& w, bool need_rows,
                                                 bool need_weights) {
    if (wants_grad(g, rows, w)) {
        const variable_list r = CombineGradFn::apply(g, rows, at_row, w, need_rows, need_weights);
        return {r[0], r[1]};
    }
    at::AutoDispatchBelowADInplaceOrView guard;
    return call_combine_grad(g, rows, at_row, w, need_rows, need_weights);
}

struct CombineRowsGradFn : public Function<CombineRowsGradFn> {
    static Tensor forward(AutogradContext*, const Tensor& g, const Tensor& at_row, const std::optional<Tensor>& w, c10::SymInt n_rows) {
        at::AutoDispatchBelowADInplaceOrView guard;
        return call_combine_rows_grad(g, at_row, w, std::move(n_rows));
    }
    static tensor_list backward(AutogradContext*, tensor_list) { once_only("moe_combine_rows_grad"); }
};
Tensor combine_rows_grad_autograd(const Tensor& g, const Tensor& at_row, const std::optional<Tensor>& w, c10::SymInt n_rows) {
    if (wants_grad(g, w)) return CombineRowsGradFn::apply(g, at_row, w, std::move(n_rows));
    at::AutoDispatchBelowADInplaceOrView guard;
    return call_combine_rows_grad(g, at_row, w, std::move(n_rows));
}

// ------------------------------------------------------------------ logit_rules
using MaybeTensor = std::optional<Tensor>;
bool is_id(const Tensor& t) { return t.scalar_type() == at::kInt || t.scalar_type() == at::kLong; }
// [rows, n] (rows may lie apart) or [n] for every row: the distance of its rows
int64_t row_stride(const Tensor& t, const Tensor& logits, int64_t rows, const char* name) {
    TORCH_CHECK(t.device() == logits.device(), name, " must be on the logits' device");
    TORCH_CHECK(t.dim() == 1 || (t.dim() == 2 && t.size(0) == rows), name, " must have one row per row of logits, or be one row for all of them");
    const int64_t n = t.size(-1);
    TORCH_CHECK(n <= 1 || t.stride(-1) == 1, name, " must be contiguous in its last dimension; torch_ggml_ops will not insert a hidden copy");
    return t.dim() == 2 ? t.stride(0) : 0;
}
const float* per_row(const MaybeTensor& t, const Tensor& logits, int64_t rows, const char* name) {
    if (!t.has_value()) return nullptr;
    check_plain(*t, logits, at::kFloat, name);
    TORCH_CHECK(t->dim() == 1 && t->size(0) == rows, name, " must be a number or have one entry per row of logits");
    return t->const_data_ptr<float>();
}
void rules_into(const Tensor& logits, const MaybeTensor& history, const MaybeTensor& lengths, const MaybeTensor& repetition, double repetition_all,
                const MaybeTensor& presence, double presence_all, const MaybeTensor& frequency, double frequency_all, const MaybeTensor& bias_ids,
                const MaybeTensor& bias_values, const MaybeTensor& allowed, const Tensor& out) {
    const int code = type_code(logits);
    const Rows r = as_rows(logits, "logits"), o = as_rows(out, "out");
    TORCH_CHECK(logits.dim() <= 2, "logits must have shape [rows, vocab] or [vocab]");
    TORCH_CHECK(out.sizes() == logits.sizes() && out.scalar_type() == logits.scalar_type() && out.device() == logits.device(),
                "out must be a tensor like logits");
    TORCH_CHECK(r.width <= INT32_MAX, "the vocabulary must be below 2^31; got ", r.width);
    TORCH_CHECK(repetition.has_value() || static_cast<float>(repetition_all) > 0, "repetition_penalty must be positive in fp32; got ", repetition_all);
    int64_t history_stride = 0, ids_stride = 0, values_stride = 0, allowed_stride = 0;
    if (history.has_value()) {
        TORCH_CHECK(is_id(*history), "history must have dtype torch.int32 or torch.int64");
        history_stride = row_stride(*history, logits, r.rows, "history");
    }
    if (lengths.has_value()) {
        TORCH_CHECK(history.has_value(), "history_lengths need a history");
        TORCH_CHECK(is_id(*lengths) && lengths->dim() == 1 && lengths->size(0) == r.rows && lengths->is_contiguous() && lengths->device() == logits.device(),
                    "history_lengths must be a contiguous torch.int32 or torch.int64 tensor with one entry per row of logits");
    }
    const float* rep = per_row(repetition, logits, r.rows, "repetition_penalty");
    const float* pres = per_row(presence, logits, r.rows, "presence_penalty");
    const float* freq = per_row(frequency, logits, r.rows, "frequency_penalty");
    TORCH_CHECK(bias_ids.has_value() == bias_values.has_value(), "bias_ids and bias_values come together");
    if (bias_ids.has_value()) {
        TORCH_CHECK(is_id(*bias_ids), "bias_ids must have dtype torch.int32 or torch.int64");
        TORCH_CHECK(bias_values->scalar_type() == at::kFloat, "bias_values must have dtype torch.float32");
        ids_stride = row_stride(*bias_ids, logits, r.rows, "bias_ids");
        values_stride = row_stride(*bias_values, logits, r.rows, "bias_values");
        TORCH_CHECK(bias_ids->size(-1) == bias_values->size(-1), "bias_ids and bias_values must have the same length");
    }
    if (allowed.has_value()) {
        TORCH_CHECK(allowed->scalar_type() == at::kInt, "allowed must have dtype torch.int32");
        allowed_stride = row_stride(*allowed, logits, r.rows, "allowed");
        TORCH_CHECK(allowed->size(-1) >= (r.width + 31) / 32, "allowed must have one bit per token: ", (r.width + 31) / 32, " words a row; got ",
                    allowed->size(-1));
    }
    if (r.rows == 0) return;
    const c10::cuda::CUDAGuard guard(logits.device());
    const bool some = history.has_value() && history->size(-1) > 0, biased = bias_ids.has_value() && bias_ids->size(-1) > 0;
    check_rc(tgo_logit_rules(logits.const_data_ptr(), out.mutable_data_ptr(), code, r.rows, r.width, r.stride, o.stride,
                             some ? history->const_data_ptr() : nullptr, some && lengths.has_value() ? lengths->const_data_ptr() : nullptr,
                             some ? history->size(-1) : 0, history_stride, some ? static_cast<int>(history->element_size()) : 8,
                             lengths.has_value() ? static_cast<int>(lengths->element_size()) : 8, rep, static_cast<float>(repetition_all), pres,
                             static_cast<float>(presence_all), freq, static_cast<float>(frequency_all), biased ? bias_ids->const_data_ptr() : nullptr,
                             biased ? bias_values->const_data_ptr<float>() : nullptr, biased ? bias_ids->size(-1) : 0, ids_stride, values_stride,
                             biased ? static_cast<int>(bias_ids->element_size()) : 8,
                             allowed.has_value() ? reinterpret_cast<const uint32_t*>(allowed->const_data_ptr<int32_t>()) : nullptr, allowed_stride,
                             stream_of(logits)),
             "logit_rules");
}
Tensor rules_cuda(const Tensor& logits, const MaybeTensor& history, const MaybeTensor& lengths, const MaybeTensor& repetition, double repetition_all,
                  const MaybeTensor& presence, double presence_all, const MaybeTensor& frequency, double frequency_all, const MaybeTensor& bias_ids,
                  const MaybeTensor& bias_values, const MaybeTensor& allowed) {
    type_code(logits);   // refused before anything is allocated
    TORCH_CHECK(logits.is_cuda(), "logits must be a CUDA tensor");
    const c10::cuda::CUDAGuard guard(logits.device());
    Tensor out = new_cuda(logits.sizes(), logits.scalar_type(), logits);
    rules_into(logits, history, lengths, repetition, repetition_all, presence, presence_all, frequency, frequency_all, bias_ids, bias_values, allowed, out);
    return out;
}
void rules_out_cuda(const Tensor& logits, const MaybeTensor& history, const MaybeTensor& lengths, const MaybeTensor& repetition, double repetition_all,
                    const MaybeTensor& presence, double presence_all, const MaybeTensor& frequency, double frequency_all, const MaybeTensor& bias_ids,
                    const MaybeTensor& bias_values, const MaybeTensor& allowed, Tensor& out) {
    at::assert_no_internal_overlap(out);
    for (const MaybeTensor* t : {&history, &lengths, &repetition, &presence, &frequency, &bias_ids, &bias_values, &allowed})
        if (t->has_value()) at::assert_no_overlap(out, **t);
    rules_into(logits, history, lengths, repetition, repetition_all, presence, presence_all, frequency, frequency_all, bias_ids, bias_values, allowed, out);
}
// Neither form has a gradient: what wants one is refused and not dropped.
template <typename... T>
void refuse_gradients(const T&... t) {
    TORCH_CHECK(!wants_grad(t...), "logit_rules has no gradient; call it under torch.no_grad() or on detached tensors");
}
Tensor rules_autograd(const Tensor& logits, const MaybeTensor& history, const MaybeTensor& lengths, const MaybeTensor& repetition, double repetition_all,
                      const MaybeTensor& presence, double presence_all, const MaybeTensor& frequency, double frequency_all, const MaybeTensor& bias_ids,
                      const MaybeTensor& bias_values, const MaybeTensor& allowed) {
    refuse_gradients(logits, repetition, presence, frequency, bias_values);
    static const auto h = op<decltype(rules_cuda)>("torch_ggml_ops_b200::logit_rules");
    at::AutoDispatchBelowADInplaceOrView guard;
    return h.call(logits, history, lengths, repetition, repetition_all, presence, presence_all, frequency, frequency_all, bias_ids, bias_values, allowed);
}
void call_rules_out(const Tensor& logits, const MaybeTensor& history, const MaybeTensor& lengths, const MaybeTensor& repetition, double repetition_all,
                    const MaybeTensor& presence, double presence_all, const MaybeTensor& frequency, double frequency_all, const MaybeTensor& bias_ids,
                    const MaybeTensor& bias_values, const MaybeTensor& allowed, Tensor& out) {
    static const auto h = op<decltype(rules_out_cuda)>("torch_ggml_ops_b200::logit_rules_out");
    h.call(logits, history, lengths, repetition, repetition_all, presence, presence_all, frequency, frequency_all, bias_ids, bias_values, allowed, out);
}
void rules_out_autograd(const Tensor& logits, const MaybeTensor& history, const MaybeTensor& lengths, const MaybeTensor& repetition, double repetition_all,
                        const MaybeTensor& presence, double presence_all, const MaybeTensor& frequency, double frequency_all, const MaybeTensor& bias_ids,
                        const MaybeTensor& bias_values, const MaybeTensor& allowed, Tensor& out) {
    refuse_gradients(logits, out, repetition, presence, frequency, bias_values);
    at::AutoDispatchBelowAutograd guard;
    call_rules_out(logits, history, lengths, repetition, repetition_all, presence, presence_all, frequency, frequency_all, bias_ids, bias_values, allowed, out);
}
// Whoever kept out for a backward pass learns from its version that it was written over.  (A tensor of inference mode has no
// version, as nothing keeps it.)
void rules_out_versioned(const Tensor& logits, const MaybeTensor& history, const MaybeTensor& lengths, const MaybeTensor& repetition, double repetition_all,
                         const MaybeTensor& presence, double presence_all, const MaybeTensor& frequency, double frequency_all, const MaybeTensor& bias_ids,
                         const MaybeTensor& bias_values, const MaybeTensor& allowed, Tensor& out) {
    {
        at::AutoDispatchBelowADInplaceOrView guard;
        call_rules_out(logits, history, lengths, repetition, repetition_all, presence, presence_all, frequency, frequency_all, bias_ids, bias_values, allowed, out);
    }
    if (!out.is_inference()) torch::autograd::impl::bump_version(out);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(torch_ggml_ops_b200, m) {
    m.def("moe_router(Tensor logits, int top_k, int scoring, bool normalize, Tensor? token_mask) -> (Tensor, Tensor)");
    m.def("moe_router_grad(Tensor grad, Tensor logits, Tensor expert_ids, Tensor weights, int scoring, bool normalize) -> Tensor");
    m.def("moe_balance_loss(Tensor logits, Tensor expert_ids, int scoring) -> (Tensor, Tensor, Tensor)");
    m.def("moe_balance_grad(Tensor grad, Tensor logits, Tensor expert_ids, Tensor coef, int scoring) -> Tensor");
    m.def("moe_dispatch(Tensor input, Tensor expert_ids, int num_experts) -> (Tensor, Tensor, Tensor, Tensor)");
    m.def("moe_dispatch_grad(Tensor grad, Tensor row_of_pair) -> Tensor");
    m.def("moe_combine(Tensor rows, Tensor row_of_pair, Tensor? weights) -> Tensor");
    m.def("moe_combine_grad(Tensor grad, Tensor rows, Tensor row_of_pair, Tensor? weights, bool need_rows, bool need_weights) -> (Tensor, Tensor)");
    m.def("moe_combine_rows_grad(Tensor grad, Tensor row_of_pair, Tensor? weights, SymInt n_rows) -> Tensor");
    m.def(
        "logit_rules(Tensor logits, Tensor? history, Tensor? history_lengths, Tensor? repetition, float repetition_all, Tensor? presence, "
        "float presence_all, Tensor? frequency, float frequency_all, Tensor? bias_ids, Tensor? bias_values, Tensor? allowed) -> Tensor");
    m.def(
        "logit_rules_out(Tensor logits, Tensor? history, Tensor? history_lengths, Tensor? repetition, float repetition_all, Tensor? presence, "
        "float presence_all, Tensor? frequency, float frequency_all, Tensor? bias_ids, Tensor? bias_values, Tensor? allowed, Tensor(a!) out) -> ()");
}
TORCH_LIBRARY_IMPL(torch_ggml_ops_b200, CUDA, m) {
    m.impl("moe_router", &router_cuda);
    m.impl("moe_router_grad", &router_grad_cuda);
    m.impl("moe_balance_loss", &balance_cuda);
    m.impl("moe_balance_grad", &balance_grad_cuda);
    m.impl("moe_dispatch", &dispatch_cuda);
    m.impl("moe_dispatch_grad", &dispatch_grad_cuda);
    m.impl("moe_combine", &combine_cuda);
    m.impl("moe_combine_grad", &combine_grad_cuda);
    m.impl("moe_combine_rows_grad", &combine_rows_grad_cuda);
    m.impl("logit_rules", &rules_cuda);
    m.impl("logit_rules_out", &rules_out_cuda);
}
TORCH_LIBRARY_IMPL(torch_ggml_ops_b200, Autograd, m) {
    m.impl("moe_router", &router_autograd);
    m.impl("moe_router_grad", &router_grad_autograd);
    m.impl("moe_balance_loss", &balance_autograd);
    m.impl("moe_balance_grad", &balance_grad_autograd);
    m.impl("moe_dispatch", &dispatch_autograd);
    m.impl("moe_dispatch_grad", &dispatch_grad_autograd);
    m.impl("moe_combine", &combine_autograd);
    m.impl("moe_combine_grad", &combine_grad_autograd);
    m.impl("moe_combine_rows_grad", &combine_rows_grad_autograd);
    m.impl("logit_rules", &rules_autograd);
    m.impl("logit_rules_out", &rules_out_autograd);
}
TORCH_LIBRARY_IMPL(torch_ggml_ops_b200, ADInplaceOrView, m) { m.impl("logit_rules_out", &rules_out_versioned); }
