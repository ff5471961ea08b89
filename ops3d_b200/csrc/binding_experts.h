// Binding of the operators around the linear layers: layer norm, routing to experts, rows sorted by expert and back.  Part of
// binding.cpp, behind its helpers.
#pragma once

void *ptr_of(const at::Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
cudaStream_t current_stream() { return at::cuda::getCurrentCUDAStream().stream(); }

void check_cuda(const at::Tensor &t, const char *name) {
    TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor (this operator has no CPU implementation)");
}
void check_device(const at::Tensor &t, const at::Tensor &like, const char *name, const char *like_name) {
    check_cuda(t, name);
    TORCH_CHECK(t.device() == like.device(), like_name, " and ", name, " must be on the same device");
}
// A tensor that may have a row tensor's dtype or be float32 beside it.
void check_dtype_or_f32(const at::Tensor &t, const at::Tensor &like, const char *name, const char *like_name) {
    TORCH_CHECK(t.scalar_type() == like.scalar_type() || t.scalar_type() == at::kFloat, name, " must have the dtype of ", like_name, ", ",
                like.scalar_type(), ", or float32, got ", t.scalar_type());
}

// ---- layer norm --------------------------------------------------------------------------------------------------------------
struct NormTensors {
    at::Tensor x, weight, bias, residual;  // dense; all but x may be undefined
    int64_t rows;
    int features, dtype, param_dtype, residual_dtype;
};

NormTensors check_norm(const at::Tensor &x, const at::Tensor &weight, const at::Tensor &bias, const at::Tensor &residual) {
    NormTensors n;
    check_cuda(x, "x");
    n.dtype = n.param_dtype = n.residual_dtype = dtype_code(x, "x");
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) > 0, "x must be [..., features] with at least one feature, got ", x.sizes());
    const int64_t features = x.size(-1), rows = x.numel() / features;
    TORCH_CHECK(features <= INT32_MAX && rows <= INT32_MAX, "layer_norm: too large dimension");
    const auto parameter = [&](const at::Tensor &t, const char *name) {
        if (!t.defined()) return at::Tensor();
        check_device(t, x, name, "x");
        check_dtype_or_f32(t, x, name, "x");
        TORCH_CHECK(t.dim() == 1 && t.size(0) == features, name, " must be [", features, "] like the last dimension of x, got ", t.sizes());
        n.param_dtype = dtype_code(t, name);
        return t.contiguous();
    };
    n.weight = parameter(weight, "weight");
    n.bias = parameter(bias, "bias");
    TORCH_CHECK(!weight.defined() || !bias.defined() || weight.scalar_type() == bias.scalar_type(), "weight and bias must have one dtype, got ",
                weight.scalar_type(), " and ", bias.scalar_type());
    if (residual.defined()) {
        check_device(residual, x, "residual", "x");
        check_dtype_or_f32(residual, x, "residual", "x");
        TORCH_CHECK(residual.sizes() == x.sizes(), "residual must have the shape of x, ", x.sizes(), ", got ", residual.sizes());
        n.residual_dtype = dtype_code(residual, "residual");
        n.residual = dense(residual);
    }
    n.x = dense(x);
    n.rows = rows;
    n.features = (int)features;
    return n;
}

// y, and the sum where it is wanted.
std::array<at::Tensor, 2> layer_norm_forward_impl(const at::Tensor &x, const at::Tensor &weight, const at::Tensor &bias, const at::Tensor &residual,
                                                  double eps, bool return_sum) {
    const NormTensors n = check_norm(x, weight, bias, residual);
    TORCH_CHECK(!return_sum || residual.defined(), "return_sum needs a residual");
    c10::cuda::CUDAGuard guard(x.device());
    std::array<at::Tensor, 2> out;
    out[0] = empty_on(x, x.sizes(), x.scalar_type());
    if (return_sum) out[1] = empty_on(x, x.sizes(), residual.scalar_type());
    raise_status(fda_layer_norm_forward(n.x.data_ptr(), ptr_of(n.weight), ptr_of(n.bias), ptr_of(n.residual), out[0].data_ptr(), ptr_of(out[1]),
                                        n.rows, n.features, (float)eps, n.dtype, n.param_dtype, n.residual_dtype, current_stream()),
                 "layer_norm_forward");
    return out;
}

// Gradients of x, weight, bias and residual; grad_sum may be undefined.
std::array<at::Tensor, 4> layer_norm_backward_impl(const at::Tensor &x, const at::Tensor &weight, const at::Tensor &bias, const at::Tensor &residual,
                                                   const at::Tensor &grad_y, const at::Tensor &grad_sum, double eps, bool need_x,
                                                   bool need_weight, bool need_bias, bool need_residual) {
    const NormTensors n = check_norm(x, weight, bias, residual);
    check_device(grad_y, x, "grad_output", "x");
    TORCH_CHECK(grad_y.scalar_type() == x.scalar_type() && grad_y.sizes() == x.sizes(), "grad_output must have the dtype and shape of x, ", x.sizes(),
                ", got ", grad_y.scalar_type(), " ", grad_y.sizes());
    if (grad_sum.defined()) {
        TORCH_CHECK(residual.defined(), "grad_sum needs a residual");
        check_device(grad_sum, x, "grad_sum", "x");
        TORCH_CHECK(grad_sum.scalar_type() == residual.scalar_type() && grad_sum.sizes() == x.sizes(),
                    "grad_sum must have the residual's dtype and shape");
    }
    c10::cuda::CUDAGuard guard(x.device());
    const at::Tensor dy = dense(grad_y), ds = grad_sum.defined() ? dense(grad_sum) : at::Tensor();
    need_residual = need_residual && residual.defined();
    const bool same = n.residual_dtype == n.dtype;  // one tensor for both
    std::array<at::Tensor, 4> out;
    if (need_x || (need_residual && same)) out[0] = empty_on(x, x.sizes(), x.scalar_type());
    if (need_weight && weight.defined()) out[1] = empty_on(weight, weight.sizes(), weight.scalar_type());
    if (need_bias && bias.defined()) out[2] = empty_on(bias, bias.sizes(), bias.scalar_type());
    if (need_residual && !same) out[3] = empty_on(x, x.sizes(), residual.scalar_type());
    const size_t bytes = fda_layer_norm_backward_workspace_bytes(n.rows, n.features, n.dtype);
    const at::Tensor ws = linear_workspace(x, bytes);
    raise_status(fda_layer_norm_backward(n.x.data_ptr(), ptr_of(n.weight), ptr_of(n.residual), dy.data_ptr(), ptr_of(ds), ptr_of(out[0]),
                                         ptr_of(out[3]), ptr_of(out[1]), ptr_of(out[2]), ptr_of(ws), bytes, n.rows, n.features, (float)eps, n.dtype,
                                         n.param_dtype, n.residual_dtype, current_stream()),
                 "layer_norm_backward");
    if (need_residual && same) out[3] = out[0];
    if (!need_x) out[0] = at::Tensor();
    return out;
}

std::array<OptionalTensor, 2> layer_norm_forward(const at::Tensor &x, const OptionalTensor &weight, const OptionalTensor &bias,
                                                 const OptionalTensor &residual, double eps, bool return_sum) {
    const auto r = layer_norm_forward_impl(x, or_undefined(weight), or_undefined(bias), or_undefined(residual), eps, return_sum);
    std::array<OptionalTensor, 2> out{r[0]};
    if (r[1].defined()) out[1] = r[1];
    return out;
}

std::array<OptionalTensor, 4> layer_norm_backward(const at::Tensor &x, const OptionalTensor &weight, const OptionalTensor &bias,
                                                  const OptionalTensor &residual, const at::Tensor &grad_y, const OptionalTensor &grad_sum,
                                                  double eps, bool need_x, bool need_weight, bool need_bias, bool need_residual) {
    const auto grads = layer_norm_backward_impl(x, or_undefined(weight), or_undefined(bias), or_undefined(residual), grad_y, or_undefined(grad_sum),
                                                eps, need_x, need_weight, need_bias, need_residual);
    std::array<OptionalTensor, 4> out;
    for (int i = 0; i < 4; ++i)
        if (grads[i].defined()) out[i] = grads[i];
    return out;
}

// LayerNormFunction.apply.
struct LayerNormBackward : public fda_nodes::SavedNode {
    double eps;
    std::string name() const override { return "LayerNormFunctionBackward"; }
    torch::autograd::variable_list apply(torch::autograd::variable_list &&grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        torch::autograd::variable_list results(4);
        const bool recording = at::GradMode::is_enabled();
        {
            at::NoGradGuard no_grad;
            const auto r = layer_norm_backward_impl(unpack(0), unpack(1), unpack(2), unpack(3), grad_output(grads),
                                                    grads.size() > 1 ? grads[1] : at::Tensor(), eps, task_should_compute_output(0),
                                                    task_should_compute_output(1), task_should_compute_output(2), task_should_compute_output(3));
            std::copy(r.begin(), r.end(), results.begin());
        }
        return fda_nodes::once_differentiable(std::move(results), recording);
    }
};

std::array<OptionalTensor, 2> layer_norm(const at::Tensor &x, const OptionalTensor &weight, const OptionalTensor &bias,
                                         const OptionalTensor &residual, double eps, bool return_sum) {
    const at::Tensor w = or_undefined(weight), b = or_undefined(bias), r = or_undefined(residual);
    std::array<at::Tensor, 2> y;
    {
        at::NoGradGuard no_grad;
        y = layer_norm_forward_impl(x, w, b, r, eps, return_sum);
    }
    if (fda_nodes::needs_node({x, w, b, r})) {
        auto node = std::make_shared<LayerNormBackward>();
        node->eps = eps;
        node->save(0, x);
        node->save(1, w);
        node->save(2, b);
        node->save(3, r);
        fda_nodes::connect(node, y[0], torch::autograd::collect_next_edges(x, w, b, r));
        if (return_sum) torch::autograd::set_history(y[1], node);
    }
    std::array<OptionalTensor, 2> out{y[0]};
    if (return_sum) out[1] = y[1];
    return out;
}

// ---- routing -----------------------------------------------------------------------------------------------------------------
struct RouteOptions {
    int top_k, score, n_groups, top_groups, group_score;
    bool renormalise;
    double scale;
};

int64_t check_logits(const at::Tensor &logits) {
    check_cuda(logits, "logits");
    dtype_code(logits, "logits");
    TORCH_CHECK(logits.dim() >= 1 && logits.size(-1) > 0, "logits must be [..., n_experts] with at least one expert, got ", logits.sizes());
    const int64_t tokens = logits.numel() / logits.size(-1);
    TORCH_CHECK(logits.size(-1) <= INT32_MAX && tokens <= INT32_MAX, "route_experts: too large dimension");
    return tokens;
}

// Weights (float32) and experts (int64), [..., top_k].
std::array<at::Tensor, 2> route_forward(const at::Tensor &logits, const OptionalTensor &bias, int top_k, int score, int n_groups, int top_groups,
                                        int group_score, bool renormalise, double scale) {
    const int64_t tokens = check_logits(logits), n_experts = logits.size(-1);
    TORCH_CHECK(n_groups >= 1 && n_experts % n_groups == 0, "n_groups must divide the ", n_experts, " experts, got ", n_groups);
    TORCH_CHECK(top_groups >= 1 && top_groups <= n_groups, "top_groups must be in 1 .. n_groups (", n_groups, "), got ", top_groups);
    TORCH_CHECK(top_k >= 1 && top_k <= n_experts / n_groups * top_groups, "top_k must be in 1 .. ", n_experts / n_groups * top_groups,
                " (the experts of top_groups groups), got ", top_k);
    at::Tensor b;
    if (bias.has_value()) {
        check_device(*bias, logits, "bias", "logits");
        TORCH_CHECK(bias->scalar_type() == at::kFloat, "bias must be float32, got ", bias->scalar_type());
        TORCH_CHECK(bias->dim() == 1 && bias->size(0) == n_experts, "bias must be [", n_experts, "], one for each expert, got ", bias->sizes());
        b = bias->contiguous();
    }
    c10::cuda::CUDAGuard guard(logits.device());
    const at::Tensor l = logits.contiguous();
    std::vector<int64_t> size = logits.sizes().vec();
    size.back() = top_k;
    std::array<at::Tensor, 2> out{empty_on(logits, size, at::kFloat), empty_on(logits, size, at::kLong)};
    raise_status(fda_route_forward(l.data_ptr(), static_cast<const float *>(ptr_of(b)), out[0].data_ptr<float>(), out[1].data_ptr<int64_t>(),
                                   tokens, (int)n_experts, top_k, score, n_groups, top_groups, group_score, renormalise, (float)scale,
                                   dtype_code(logits, "logits"), current_stream()),
                 "route_experts");
    return out;
}

at::Tensor route_backward(const at::Tensor &logits, const at::Tensor &experts, const at::Tensor &grad_weights, int score, bool renormalise,
                          double scale) {
    const int64_t tokens = check_logits(logits);
    check_device(experts, logits, "experts", "logits");
    check_device(grad_weights, logits, "grad_weights", "logits");
    TORCH_CHECK(experts.scalar_type() == at::kLong && grad_weights.scalar_type() == at::kFloat && experts.dim() == logits.dim() &&
                    grad_weights.sizes() == experts.sizes() && experts.sizes().slice(0, experts.dim() - 1) == logits.sizes().slice(0, logits.dim() - 1),
                "experts must be int64 and grad_weights float32, both [..., top_k] like logits");
    c10::cuda::CUDAGuard guard(logits.device());
    const at::Tensor l = logits.contiguous(), e = experts.contiguous(), g = grad_weights.contiguous();
    at::Tensor out = empty_on(logits, logits.sizes(), logits.scalar_type());
    raise_status(fda_route_backward(l.data_ptr(), e.data_ptr<int64_t>(), g.data_ptr<float>(), out.data_ptr(), tokens, (int)logits.size(-1),
                                    (int)experts.size(-1), score, renormalise, (float)scale, dtype_code(logits, "logits"), current_stream()),
                 "route_experts backward");
    return out;
}

// RouteExpertsFunction.apply.
struct RouteExpertsBackward : public fda_nodes::SavedNode {
    int score;
    bool renormalise;
    double scale;
    std::string name() const override { return "RouteExpertsFunctionBackward"; }
    torch::autograd::variable_list apply(torch::autograd::variable_list &&grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        torch::autograd::variable_list results(1);
        const bool recording = at::GradMode::is_enabled();
        {
            at::NoGradGuard no_grad;
            results[0] = route_backward(unpack(0), unpack(1), grad_output(grads), score, renormalise, scale);
        }
        return fda_nodes::once_differentiable(std::move(results), recording);
    }
};

std::array<at::Tensor, 2> route(const at::Tensor &logits, const OptionalTensor &bias, int top_k, int score, int n_groups, int top_groups,
                                int group_score, bool renormalise, double scale) {
    std::array<at::Tensor, 2> out;
    {
        at::NoGradGuard no_grad;
        out = route_forward(logits, bias, top_k, score, n_groups, top_groups, group_score, renormalise, scale);
    }
    if (fda_nodes::needs_node({logits})) {
        auto node = std::make_shared<RouteExpertsBackward>();
        node->score = score;
        node->renormalise = renormalise;
        node->scale = scale;
        node->save(0, logits);
        node->save(1, out[1]);
        fda_nodes::connect(node, out[0], torch::autograd::collect_next_edges(logits));
    }
    return out;
}

// ---- rows sorted by expert ---------------------------------------------------------------------------------------------------
// rows [tokens * top_k, features], group_start_index [n_experts + 1], position like experts.
std::array<at::Tensor, 3> dispatch_forward(const at::Tensor &x, const at::Tensor &experts, int64_t n_experts) {
    check_cuda(x, "x");
    const int dtype = dtype_code(x, "x");
    check_device(experts, x, "experts", "x");
    TORCH_CHECK(experts.scalar_type() == at::kLong, "experts must be int64, got ", experts.scalar_type());
    TORCH_CHECK(x.dim() >= 1 && experts.dim() == x.dim() && experts.sizes().slice(0, x.dim() - 1) == x.sizes().slice(0, x.dim() - 1),
                "experts must be [..., top_k] with the leading dimensions of x, ", x.sizes(), ", got ", experts.sizes());
    const int64_t features = x.size(-1), top_k = experts.size(-1);
    TORCH_CHECK(features > 0 && top_k > 0, "x must have at least one feature, experts at least one choice");
    const int64_t tokens = x.numel() / features;
    TORCH_CHECK(n_experts >= 1 && n_experts <= INT32_MAX, "n_experts must be positive, got ", n_experts);
    TORCH_CHECK(tokens <= INT32_MAX && features <= INT32_MAX && top_k <= INT32_MAX, "dispatch_rows: too large dimension");
    c10::cuda::CUDAGuard guard(x.device());
    const at::Tensor rows_in = dense(x), e = experts.contiguous();
    std::array<at::Tensor, 3> out{empty_on(x, {tokens * top_k, features}, x.scalar_type()), empty_on(x, {n_experts + 1}, at::kLong),
                                  empty_on(x, experts.sizes(), at::kLong)};
    const size_t bytes = fda_dispatch_workspace_bytes(tokens, (int)top_k, (int)n_experts);
    const at::Tensor ws = linear_workspace(x, bytes);
    raise_status(fda_dispatch_rows(rows_in.data_ptr(), e.data_ptr<int64_t>(), out[0].data_ptr(), out[1].data_ptr<int64_t>(),
                                   out[2].data_ptr<int64_t>(), ptr_of(ws), bytes, tokens, (int)top_k, (int)n_experts, (int)features, dtype,
                                   current_stream()),
                 "dispatch_rows");
    return out;
}

// DispatchRowsFunction.apply; the gradient of x is the sum of its rows' gradients.
at::Tensor combine_forward_impl(const at::Tensor &rows, const at::Tensor &position, const at::Tensor &weights, const at::Tensor &residual);

struct DispatchRowsBackward : public fda_nodes::SavedNode {
    std::string name() const override { return "DispatchRowsFunctionBackward"; }
    torch::autograd::variable_list apply(torch::autograd::variable_list &&grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        torch::autograd::variable_list results(1);
        const bool recording = at::GradMode::is_enabled();
        {
            at::NoGradGuard no_grad;
            results[0] = combine_forward_impl(grad_output(grads), unpack(0), at::Tensor(), at::Tensor());
        }
        return fda_nodes::once_differentiable(std::move(results), recording);
    }
};

std::array<at::Tensor, 3> dispatch(const at::Tensor &x, const at::Tensor &experts, int64_t n_experts) {
    std::array<at::Tensor, 3> out;
    {
        at::NoGradGuard no_grad;
        out = dispatch_forward(x, experts, n_experts);
    }
    if (fda_nodes::needs_node({x})) {
        auto node = std::make_shared<DispatchRowsBackward>();
        node->save(0, out[2]);
        fda_nodes::connect(node, out[0], torch::autograd::collect_next_edges(x));
    }
    return out;
}

struct CombineTensors {
    at::Tensor position, weights;
    int64_t tokens;
    int top_k, features, dtype, weight_dtype;
    std::vector<int64_t> out_size;
};

// position and weights beside `like`, a tensor with as many features as the rows and of their type.
CombineTensors check_combine(const at::Tensor &like, const char *name, const at::Tensor &position, const at::Tensor &weights) {
    CombineTensors c;
    check_cuda(like, name);
    c.dtype = c.weight_dtype = dtype_code(like, name);
    check_device(position, like, "position", name);
    TORCH_CHECK(position.scalar_type() == at::kLong && position.dim() >= 1 && position.size(-1) > 0, "position must be int64 [..., top_k]");
    TORCH_CHECK(like.dim() >= 1 && like.size(-1) > 0, name, " must have at least one feature, got ", like.sizes());
    if (weights.defined()) {
        check_device(weights, like, "weights", name);
        check_dtype_or_f32(weights, like, "weights", name);
        TORCH_CHECK(weights.sizes() == position.sizes(), "weights must have the shape of position, ", position.sizes(), ", got ", weights.sizes());
        c.weight_dtype = dtype_code(weights, "weights");
        c.weights = weights.contiguous();
    }
    const int64_t top_k = position.size(-1), features = like.size(-1);
    TORCH_CHECK(position.numel() <= INT32_MAX && features <= INT32_MAX && top_k <= INT32_MAX, "combine_rows: too large dimension");
    c.position = position.contiguous();
    c.tokens = position.numel() / top_k;
    c.top_k = (int)top_k;
    c.features = (int)features;
    c.out_size = position.sizes().vec();
    c.out_size.back() = features;
    return c;
}
void check_combined_rows(const at::Tensor &rows, const CombineTensors &c) {
    TORCH_CHECK(rows.dim() == 2 && rows.size(0) == c.position.numel() && rows.size(1) == c.features, "rows must be [", c.position.numel(),
                ", features], a row for each entry of position, got ", rows.sizes());
}

at::Tensor combine_forward_impl(const at::Tensor &rows, const at::Tensor &position, const at::Tensor &weights, const at::Tensor &residual) {
    const CombineTensors c = check_combine(rows, "rows", position, weights);
    check_combined_rows(rows, c);
    at::Tensor res;
    if (residual.defined()) {
        check_device(residual, rows, "residual", "rows");
        TORCH_CHECK(residual.scalar_type() == rows.scalar_type(), "residual must have the dtype of rows, ", rows.scalar_type(), ", got ",
                    residual.scalar_type());
        TORCH_CHECK(residual.sizes() == at::IntArrayRef(c.out_size), "residual must have the shape of the output, ", at::IntArrayRef(c.out_size),
                    ", got ", residual.sizes());
        res = dense(residual);
    }
    c10::cuda::CUDAGuard guard(rows.device());
    const at::Tensor r = dense(rows);
    at::Tensor y = empty_on(rows, c.out_size, rows.scalar_type());
    raise_status(fda_combine_rows(r.data_ptr(), c.position.data_ptr<int64_t>(), ptr_of(c.weights), ptr_of(res), y.data_ptr(), c.tokens, c.top_k,
                                  c.features, c.dtype, c.weight_dtype, current_stream()),
                 "combine_rows");
    return y;
}

// Gradients of rows and weights.  `rows` may be undefined where the weights need none.
std::array<at::Tensor, 2> combine_backward_impl(const at::Tensor &rows, const at::Tensor &position, const at::Tensor &weights,
                                                const at::Tensor &grad_y, bool need_rows, bool need_weights) {
    std::array<at::Tensor, 2> out;
    need_weights = need_weights && weights.defined();
    if (!need_rows && !need_weights) return out;
    const CombineTensors c = check_combine(grad_y, "grad_output", position, weights);
    TORCH_CHECK(grad_y.sizes() == at::IntArrayRef(c.out_size), "grad_output must have the shape of the output, ", at::IntArrayRef(c.out_size),
                ", got ", grad_y.sizes());
    c10::cuda::CUDAGuard guard(grad_y.device());
    at::Tensor r;
    if (need_weights) {
        TORCH_CHECK(rows.defined() && rows.scalar_type() == grad_y.scalar_type(), "grad_output must have the dtype of rows");
        check_device(rows, grad_y, "rows", "grad_output");
        check_combined_rows(rows, c);
        r = dense(rows);
    }
    const at::Tensor dy = dense(grad_y);
    if (need_rows) out[0] = empty_on(grad_y, {c.position.numel(), c.features}, grad_y.scalar_type());
    if (need_weights) out[1] = empty_on(grad_y, weights.sizes(), weights.scalar_type());
    const size_t bytes = need_rows ? fda_combine_rows_backward_workspace_bytes(c.tokens, c.top_k) : 0;
    const at::Tensor ws = linear_workspace(grad_y, bytes);
    raise_status(fda_combine_rows_backward(ptr_of(r), c.position.data_ptr<int64_t>(), ptr_of(c.weights), dy.data_ptr(), ptr_of(out[0]),
                                           ptr_of(out[1]), ptr_of(ws), bytes, c.tokens, c.top_k, c.features, c.dtype, c.weight_dtype,
                                           current_stream()),
                 "combine_rows backward");
    return out;
}

at::Tensor combine_forward(const at::Tensor &rows, const at::Tensor &position, const OptionalTensor &weights, const OptionalTensor &residual) {
    return combine_forward_impl(rows, position, or_undefined(weights), or_undefined(residual));
}

std::array<OptionalTensor, 2> combine_backward(const OptionalTensor &rows, const at::Tensor &position, const OptionalTensor &weights,
                                               const at::Tensor &grad_y, bool need_rows, bool need_weights) {
    const auto grads = combine_backward_impl(or_undefined(rows), position, or_undefined(weights), grad_y, need_rows, need_weights);
    std::array<OptionalTensor, 2> out;
    for (int i = 0; i < 2; ++i)
        if (grads[i].defined()) out[i] = grads[i];
    return out;
}

// CombineRowsFunction.apply; the residual's gradient is the output's.
struct CombineRowsBackward : public fda_nodes::SavedNode {
    std::string name() const override { return "CombineRowsFunctionBackward"; }
    torch::autograd::variable_list apply(torch::autograd::variable_list &&grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        torch::autograd::variable_list results(3);
        const bool recording = at::GradMode::is_enabled();
        {
            at::NoGradGuard no_grad;
            const at::Tensor g = grad_output(grads);
            const auto r = combine_backward_impl(unpack(0), unpack(1), unpack(2), g, task_should_compute_output(0), task_should_compute_output(1));
            results[0] = r[0];
            results[1] = r[1];
            if (task_should_compute_output(2)) results[2] = g;
        }
        return fda_nodes::once_differentiable(std::move(results), recording);
    }
};

at::Tensor combine(const at::Tensor &rows, const at::Tensor &position, const OptionalTensor &weights, const OptionalTensor &residual) {
    const at::Tensor w = or_undefined(weights), r = or_undefined(residual);
    at::Tensor y;
    {
        at::NoGradGuard no_grad;
        y = combine_forward_impl(rows, position, w, r);
    }
    if (fda_nodes::needs_node({rows, w, r})) {
        auto node = std::make_shared<CombineRowsBackward>();
        if (w.defined() && w.requires_grad()) node->save(0, rows);  // only the weights' gradient reads them
        node->save(1, position);
        node->save(2, w);
        fda_nodes::connect(node, y, torch::autograd::collect_next_edges(rows, w, r));
    }
    return y;
}
