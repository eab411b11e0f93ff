// torch_recurrent_layer.h -- the part of the PyTorch binding for the layer of the
// gated delta rule: the norms around it; included by torch_ext.cpp after
// torch_operators.h, whose helpers it uses.
#pragma once

namespace {

// ---- the norm with the residual's addition ----

void check_weight(ArgCheck& c, const c10::optional<at::Tensor>& weight, const at::Tensor& x, int64_t d) {
    if (!weight) return;
    const at::Tensor& w = *weight;
    c.on_gpu("weight", w).dtype_is("weight", w, true)
        .require(w.scalar_type() == at::kFloat || w.scalar_type() == x.scalar_type(), "weight",
                 "is neither float32 nor of x's dtype")
        .require(w.device() == x.device() && w.dim() == 1 && w.numel() == d, "weight",
                 [&] { return "must hold " + std::to_string(d) + " values on x's device"; });
}

int32_t weight_dtype_of(const c10::optional<at::Tensor>& weight, const at::Tensor& x) {
    return weight ? dtype_of(*weight) : dtype_of(x);
}

// x and residual as [rows, D].
race_add_norm_shape add_norm_shape(const char* entry, const at::Tensor& x, const c10::optional<at::Tensor>& residual,
                                   const c10::optional<at::Tensor>& weight, double eps, bool e4m3, int64_t group) {
    ArgCheck c(entry);
    check_rows(c, "x", x, 2, "[rows, D]");
    c.raise();
    const int64_t rows = x.size(0), D = x.size(1);
    c.require(D >= 1 && D <= 16384, "x", [&] { return "has rows of " + std::to_string(D) + " values; 1 .. 16384 are taken"; })
        .require(D < 1 || rows <= (int64_t(1) << 46) / D, "x", "has more than 2^46 values");
    if (residual) {
        check_rows(c, "residual", *residual, 2, "[rows, D]");
        c.matches("residual", *residual, "x", x)
            .require(residual->sizes() == x.sizes(), "residual", [&] { return "has shape " + dims(*residual) + ", x " + dims(x); });
    }
    check_weight(c, weight, x, D);
    c.require(eps >= 0 && eps < 1e30, "eps", "must be a number of at least 0")
        .require(group == 0 || group == 32 || group == 64 || group == 128, "group", "must be 0 (a scale a row), 32, 64 or 128")
        .require(group == 0 || D % 8 == 0, "group", [&] { return "needs rows of a multiple of 8 values, not " + std::to_string(D); })
        .raise();
    race_add_norm_shape sh{};
    sh.rows = rows, sh.width = static_cast<int32_t>(D);
    sh.dtype = dtype_of(x), sh.weight_dtype = weight_dtype_of(weight, x);
    sh.out = e4m3 ? RACE_ROWS_E4M3 : RACE_ROWS_SAME;
    sh.group = static_cast<int32_t>(group), sh.eps = static_cast<float>(eps);
    sh.x_row_stride = rows > 1 ? x.stride(0) : 0;
    sh.residual_row_stride = residual && rows > 1 ? residual->stride(0) : 0;
    return sh;
}

// (y, sum or None, scales or None) of rows [rows, D].
std::tuple<at::Tensor, c10::optional<at::Tensor>, c10::optional<at::Tensor>> add_norm_forward(
    const char* entry, const at::Tensor& x, const c10::optional<at::Tensor>& residual,
    const c10::optional<at::Tensor>& weight, double eps, bool e4m3, int64_t group) {
    const race_add_norm_shape sh = add_norm_shape(entry, x, residual, weight, eps, e4m3, group);
    const c10::DeviceGuard guard(x.device());
    const at::Tensor y = at::empty(x.sizes(), e4m3 ? x.options().dtype(at::kFloat8_e4m3fn) : x.options());
    c10::optional<at::Tensor> sum, scales;
    if (residual) sum = at::empty(x.sizes(), x.options());
    if (e4m3) scales = at::empty({sh.rows, group ? (sh.width + group - 1) / group : 1}, x.options().dtype(at::kFloat));
    check_status(race_add_norm_fwd(x.data_ptr(), data_of(residual), data_of(weight), y.data_ptr(), floats_of(scales),
                                   ptr_of(sum), &sh, current_stream()),
                 "race_add_norm_fwd");
    return {y, sum, scales};
}

// Gradients of the rows and the weight; `s` is what was normed.
std::tuple<c10::optional<at::Tensor>, c10::optional<at::Tensor>> add_norm_backward(
    const at::Tensor& s, const c10::optional<at::Tensor>& weight, const c10::optional<at::Tensor>& dy,
    const c10::optional<at::Tensor>& dsum, double eps, bool need_rows, bool need_weight) {
    const char* entry = "race_add_norm backward";
    const race_add_norm_shape sh = add_norm_shape(entry, s, c10::nullopt, weight, eps, false, 0);
    ArgCheck c(entry);
    for (const auto& [name, g] : {std::make_pair("dy", &dy), std::make_pair("dsum", &dsum)})
        if (*g)
            c.on_gpu(name, **g).matches(name, **g, "x", s)
                .require((*g)->sizes() == s.sizes(), name, [&, g = g] { return "has shape " + dims(**g); });
    c.raise();
    const c10::DeviceGuard guard(s.device());
    c10::optional<at::Tensor> dx, dw;
    if (need_rows) dx = at::empty(s.sizes(), s.options());
    if (need_weight && weight) dw = at::empty_like(*weight);
    size_t bytes = 0;
    at::Tensor ws;
    if (dw) {
        check_status(race_add_norm_bwd_workspace_bytes(&sh, &bytes), "race_add_norm_bwd_workspace_bytes");
        ws = workspace_of(bytes, s);
    }
    check_status(race_add_norm_bwd(s.data_ptr(), data_of(weight), data_of(dy), data_of(dsum), ptr_of(dx), ptr_of(dw), &sh,
                                   bytes > 0 ? ws.data_ptr() : nullptr, bytes, current_stream()),
                 "race_add_norm_bwd");
    return {dx, dw};
}

// ---- the gated norm of a recurrence's heads ----

race_gate_norm_shape gate_norm_shape(const char* entry, const at::Tensor& x, const at::Tensor& gate,
                                     const c10::optional<at::Tensor>& weight, double eps) {
    ArgCheck c(entry);
    check_rows(c, "x", x, 3, "[B * H, T, d]");
    check_rows(c, "gate", gate, 4, "[B, T, H, d]");
    c.matches("gate", gate, "x", x).raise();
    const int64_t B = gate.size(0), T = gate.size(1), H = gate.size(2), d = gate.size(3);
    c.require(x.size(0) == B * H && x.size(1) == T && x.size(2) == d, "x",
              [&] { return "has shape " + dims(x) + ", not [B * H, T, d] of gate's " + dims(gate); })
        .require(H >= 1 && H <= 65535 && d >= 1 && d <= 256, "gate",
                 [&] { return "has shape " + dims(gate) + "; rows of 1 .. 256 values in 1 .. 65535 heads are taken"; })
        .require(T == 0 || B <= (int64_t(1) << 30) / T, "gate", "has more than 2^30 tokens");
    check_weight(c, weight, x, d);
    c.require(eps >= 0 && eps < 1e30, "eps", "must be a number of at least 0").raise();
    auto stride = [](const at::Tensor& t, int64_t i) { return t.size(i) > 1 ? t.stride(i) : 0; };
    race_gate_norm_shape sh{};
    sh.batch = B, sh.seq_len = T, sh.heads = static_cast<int32_t>(H), sh.head_dim = static_cast<int32_t>(d);
    sh.dtype = dtype_of(x), sh.weight_dtype = weight_dtype_of(weight, x), sh.eps = static_cast<float>(eps);
    sh.x_stream_stride = stride(x, 0), sh.x_token_stride = stride(x, 1);
    sh.gate_batch_stride = stride(gate, 0), sh.gate_token_stride = stride(gate, 1), sh.gate_head_stride = stride(gate, 2);
    return sh;
}

at::Tensor gate_norm_forward(const at::Tensor& x, const at::Tensor& gate, const c10::optional<at::Tensor>& weight,
                             double eps) {
    const race_gate_norm_shape sh = gate_norm_shape("race_gate_norm", x, gate, weight, eps);
    const c10::DeviceGuard guard(x.device());
    const at::Tensor y = at::empty(gate.sizes(), gate.options());
    check_status(race_gate_norm_fwd(x.data_ptr(), gate.data_ptr(), data_of(weight), y.data_ptr(), &sh, current_stream()),
                 "race_gate_norm_fwd");
    return y;
}

std::tuple<c10::optional<at::Tensor>, c10::optional<at::Tensor>, c10::optional<at::Tensor>> gate_norm_backward(
    const at::Tensor& x, const at::Tensor& gate, const c10::optional<at::Tensor>& weight, const at::Tensor& dy, double eps,
    bool need_x, bool need_gate, bool need_weight) {
    const char* entry = "race_gate_norm backward";
    const race_gate_norm_shape sh = gate_norm_shape(entry, x, gate, weight, eps);
    ArgCheck(entry).on_gpu("dy", dy).matches("dy", dy, "x", x)
        .require(dy.sizes() == gate.sizes(), "dy", [&] { return "has shape " + dims(dy) + ", gate " + dims(gate); })
        .raise();
    const c10::DeviceGuard guard(x.device());
    c10::optional<at::Tensor> dx, dz, dw;
    if (need_x) dx = at::empty(x.sizes(), x.options());
    if (need_gate) dz = at::empty(gate.sizes(), gate.options());
    if (need_weight && weight) dw = at::empty_like(*weight);
    size_t bytes = 0;
    at::Tensor ws;
    if (dw) {
        check_status(race_gate_norm_bwd_workspace_bytes(&sh, &bytes), "race_gate_norm_bwd_workspace_bytes");
        ws = workspace_of(bytes, x);
    }
    check_status(race_gate_norm_bwd(x.data_ptr(), gate.data_ptr(), data_of(weight), dy.data_ptr(), ptr_of(dx), ptr_of(dz),
                                    ptr_of(dw), &sh, bytes > 0 ? ws.data_ptr() : nullptr, bytes, current_stream()),
                 "race_gate_norm_bwd");
    return {dx, dz, dw};
}

// ---- the operators with their gradients ----

struct AddNormNode : torch::autograd::Function<AddNormNode> {
    static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const c10::optional<at::Tensor>& residual,
                                 const c10::optional<at::Tensor>& weight, double eps) {
        const auto [y, sum, scales] = add_norm_forward("race_add_norm", x, residual, weight, eps, false, 0);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({sum ? *sum : x, or_undefined(weight)});
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["residual"] = residual.has_value();
        if (sum) return {y, *sum};
        return {y};
    }
    static variable_list backward(AutogradContext* ctx, variable_list up) {
        variable_list grads(4);
        const variable_list saved = ctx->get_saved_variables();
        const at::Tensor& s = saved[0];
        const auto weight = if_defined(saved[1]);
        check_capture("race_add_norm backward", {s, weight});
        const auto dy = dense_grad(up[0], s.scalar_type());
        const auto ds = up.size() > 1 ? dense_grad(up[1], s.scalar_type()) : c10::nullopt;
        if (dy || ds) {
            const auto need = needed(ctx, {true, ctx->saved_data["residual"].toBool(), weight.has_value()});
            const auto [dx, dw] = add_norm_backward(s, weight, dy, ds, ctx->saved_data["eps"].toDouble(),
                                                    need[0] || need[1], need[2]);
            grads = {need[0] ? or_undefined(dx) : at::Tensor(), need[1] ? or_undefined(dx) : at::Tensor(), or_undefined(dw),
                     at::Tensor()};
        }
        return differentiated_once("race_add_norm", up, std::move(grads));
    }
};

struct GateNormNode : torch::autograd::Function<GateNormNode> {
    static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& gate,
                                 const c10::optional<at::Tensor>& weight, double eps) {
        const at::Tensor y = gate_norm_forward(x, gate, weight, eps);
        ctx->save_for_backward({x, gate, or_undefined(weight)});
        ctx->saved_data["eps"] = eps;
        return {y};
    }
    static variable_list backward(AutogradContext* ctx, variable_list up) {
        const variable_list saved = ctx->get_saved_variables();
        const at::Tensor &x = saved[0], &gate = saved[1];
        const auto weight = if_defined(saved[2]);
        check_capture("race_gate_norm backward", {x, gate, weight});
        const auto need = needed(ctx, {true, true, weight.has_value()});
        const auto dy = dense_grad(up[0], x.scalar_type());
        const auto [a, b, c] = gate_norm_backward(x, gate, weight, *dy, ctx->saved_data["eps"].toDouble(), need[0], need[1],
                                                  need[2]);
        return differentiated_once("race_gate_norm", up, {or_undefined(a), or_undefined(b), or_undefined(c), at::Tensor()});
    }
};

// Rows of any leading dimensions as [rows, D]: a view where one row stride
// reaches them all, else a copy.
at::Tensor as_matrix(const char* entry, const char* name, const at::Tensor& t) {
    ArgCheck(entry).require(t.dim() >= 1, name, "is a scalar; rows [..., D] are taken").raise();
    return as_rows(t.dim() == 2 ? t : t.reshape({-1, t.size(-1)}));
}

// (y, sum or None); rows [..., D].
std::tuple<at::Tensor, c10::optional<at::Tensor>> add_norm(const at::Tensor& x_in, const c10::optional<at::Tensor>& residual_in,
                                                           const c10::optional<at::Tensor>& weight, double eps) {
    const char* entry = "race_add_norm";
    const bool node = wants_grad({x_in, residual_in, weight});
    if (node) check_capture(entry, {x_in, residual_in, weight});
    if (residual_in)
        ArgCheck(entry).require(residual_in->sizes() == x_in.sizes(), "residual",
                                [&] { return "has shape " + dims(*residual_in) + ", x " + dims(x_in); }).raise();
    const at::Tensor x = as_matrix(entry, "x", x_in);
    c10::optional<at::Tensor> residual;
    if (residual_in) residual = as_matrix(entry, "residual", *residual_in);
    c10::optional<at::Tensor> sum;
    at::Tensor y;
    if (node) {
        const variable_list outs = AddNormNode::apply(x, residual, weight, eps);
        y = outs[0];
        if (outs.size() > 1) sum = outs[1];
    } else {
        std::tie(y, sum, std::ignore) = add_norm_forward(entry, x, residual, weight, eps, false, 0);
    }
    if (x_in.dim() == 2) return {y, sum};
    if (sum) sum = sum->view(x_in.sizes());
    return {y.view(x_in.sizes()), sum};
}

// (y in e4m3, scales, sum or None); no gradients.
std::tuple<at::Tensor, at::Tensor, c10::optional<at::Tensor>> add_norm_e4m3(
    const at::Tensor& x_in, const c10::optional<at::Tensor>& residual_in, const c10::optional<at::Tensor>& weight, double eps,
    int64_t group) {
    const char* entry = "race_add_norm_e4m3";
    if (residual_in)
        ArgCheck(entry).require(residual_in->sizes() == x_in.sizes(), "residual",
                                [&] { return "has shape " + dims(*residual_in) + ", x " + dims(x_in); }).raise();
    auto rows = [&](const char* name, const at::Tensor& t) {
        const at::Tensor m = as_matrix(entry, name, t);
        return group != 0 && m.size(0) > 1 && m.stride(0) % 8 != 0 ? m.clone(at::MemoryFormat::Contiguous) : m;
    };
    const at::Tensor x = rows("x", x_in);
    c10::optional<at::Tensor> residual;
    if (residual_in) residual = rows("residual", *residual_in);
    auto [y, sum, scales] = add_norm_forward(entry, x, residual, weight, eps, true, group);
    if (x_in.dim() == 2) return {y, *scales, sum};
    std::vector<int64_t> per(x_in.sizes().begin(), x_in.sizes().end());
    per.back() = scales->size(1);
    if (sum) sum = sum->view(x_in.sizes());
    return {y.view(x_in.sizes()), scales->view(per), sum};
}

at::Tensor gate_norm(const at::Tensor& x_in, const at::Tensor& gate_in, const c10::optional<at::Tensor>& weight, double eps) {
    const bool node = wants_grad({x_in, gate_in, weight});
    if (node) check_capture("race_gate_norm", {x_in, gate_in, weight});
    const at::Tensor x = as_rows(x_in), gate = as_rows(gate_in);
    if (!node) return gate_norm_forward(x, gate, weight, eps);
    return GateNormNode::apply(x, gate, weight, eps)[0];
}

void bind_recurrent_layer(pybind11::module& m) {
    namespace py = pybind11;
    m.def("add_norm", &add_norm, "race_add_norm with its gradients -> (y, sum or None)", py::arg("x"), py::arg("residual"),
          py::arg("weight"), py::arg("eps"));
    m.def("add_norm_e4m3", &add_norm_e4m3, "race_add_norm with y in 8 bits -> (y, scales, sum or None)", py::arg("x"),
          py::arg("residual"), py::arg("weight"), py::arg("eps"), py::arg("group"));
    m.def("gate_norm", &gate_norm, "race_gate_norm with its gradients -> y", py::arg("x"), py::arg("gate"),
          py::arg("weight"), py::arg("eps"));
}

}  // namespace
