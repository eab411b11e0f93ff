// torch_recurrent_layer.h -- the part of the PyTorch binding for the layer of the
// gated delta rule: the recurrence and the norms around it; included by torch_ext.cpp after
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

// ---- the gated delta rule ----

race_delta_shape delta_shape(const char* entry, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                             const c10::optional<at::Tensor>& gate, const at::Tensor& beta,
                             const c10::optional<at::Tensor>& state, const c10::optional<at::Tensor>& lengths, int64_t form,
                             double scale) {
    ArgCheck c(entry);
    check_rows(c, "q", q, 3, "[N, T, dk]");
    check_rows(c, "k", k, 3, "[N, T, dk]");
    check_rows(c, "v", v, 3, "[N, T, dv]");
    c.matches("k", k, "q", q).matches("v", v, "q", q)
        .require(k.sizes() == q.sizes(), "k", [&] { return "has shape " + dims(k) + ", q " + dims(q); })
        .raise();
    const int64_t N = v.size(0), Nk = q.size(0), T = q.size(1), dk = q.size(2), dv = v.size(2);
    c.require(v.size(1) == T, "v", [&] { return "has shape " + dims(v) + ", not q's " + std::to_string(T) + " tokens"; })
        .require(Nk > 0 ? N >= Nk && N % Nk == 0 : N == 0, "v",
                 [&] { return "has " + std::to_string(N) + " streams, no multiple of the " + std::to_string(Nk) + " key streams"; })
        .require(dk >= 1 && dk <= 128 && dv >= 1 && dv <= 256, "q",
                 [&] { return "and v have rows of " + std::to_string(dk) + " and " + std::to_string(dv) +
                           " values; keys of 1 .. 128 and values of 1 .. 256 are taken"; })
        .require(N <= 65535 && T <= (int64_t(1) << 30) && (N == 0 || (T + 63) / 64 <= ((int64_t(1) << 24) - 1) / N), "v",
                 [&] { return "has shape " + dims(v) + "; up to 65535 streams and 2^30 tokens in all are taken"; });
    auto per_token = [&](const char* name, const at::Tensor& t) {
        c.on_gpu(name, t).dtype_is(name, t, true)
            .require(t.device() == q.device() && t.sizes() == at::IntArrayRef({N, T}), name,
                     [&] { return "has shape " + dims(t) + ", not v's [N, T] on its device"; })
            .require(t.scalar_type() == at::kFloat || t.scalar_type() == q.scalar_type(), name, "is neither float32 nor of q's dtype");
    };
    per_token("beta", beta);
    if (gate) {
        per_token("gate", *gate);
        c.require(gate->scalar_type() == beta.scalar_type(), "gate", "has another dtype than beta");
    }
    if (state)
        c.on_gpu("state", *state)
            .require(state->scalar_type() == at::kFloat && state->device() == q.device(), "state", "must be float32 on q's device")
            .require(state->sizes() == at::IntArrayRef({N, dk, dv}), "state",
                     [&] { return "has shape " + dims(*state) + ", not [N, dk, dv] of v's streams"; });
    const int64_t group = check_lengths(c, lengths, q, N);
    c.require(scale > -1e30 && scale < 1e30, "scale", "must be a finite number").raise();
    auto stride = [](const at::Tensor& t, int64_t i) { return t.size(i) > 1 ? t.stride(i) : 0; };
    race_delta_shape sh{};
    sh.value_streams = N, sh.key_streams = Nk, sh.seq_len = T;
    sh.key_dim = static_cast<int32_t>(dk), sh.value_dim = static_cast<int32_t>(dv);
    sh.dtype = dtype_of(q), sh.gate_dtype = dtype_of(beta), sh.gate_form = static_cast<int32_t>(form);
    sh.lengths_group = static_cast<int32_t>(group), sh.scale = static_cast<float>(scale);
    sh.q_stream_stride = stride(q, 0), sh.q_token_stride = stride(q, 1);
    sh.k_stream_stride = stride(k, 0), sh.k_token_stride = stride(k, 1);
    sh.v_stream_stride = stride(v, 0), sh.v_token_stride = stride(v, 1);
    return sh;
}

constexpr int64_t kDeltaFar = int64_t(1) << 22;  // the largest token stride; a copy past it

// q or k as rows [N, T, dk]: bucket probabilities [N, T, L, R] are rows of L R.
at::Tensor as_key_rows(const at::Tensor& t) { return as_rows(t.dim() == 4 ? t.flatten(2) : t, kDeltaFar); }

// Gates and strengths [N, T] are small: a copy where they are not dense.
at::Tensor as_per_token(const at::Tensor& t) {
    const at::Tensor d = t.contiguous();
    return d.numel() > 0 && !starts_aligned(d) ? d.clone() : d;
}
c10::optional<at::Tensor> as_per_token(const c10::optional<at::Tensor>& t) {
    if (!t) return c10::nullopt;
    return as_per_token(*t);
}

// (out, final state, records or None).
std::tuple<at::Tensor, at::Tensor, c10::optional<at::Tensor>> delta_forward(
    const char* entry, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const c10::optional<at::Tensor>& gate,
    const at::Tensor& beta, const c10::optional<at::Tensor>& state, const c10::optional<at::Tensor>& lengths, int64_t form,
    double scale, bool want_records, bool inplace) {
    const race_delta_shape sh = delta_shape(entry, q, k, v, gate, beta, state, lengths, form, scale);
    TORCH_CHECK(!inplace || state, entry, ": an in-place call needs a state");
    TORCH_CHECK(!inplace || !(at::GradMode::is_enabled() && state->requires_grad()), entry,
                ": a state that requires a gradient cannot be advanced in place");
    const c10::DeviceGuard guard(q.device());
    const at::Tensor out = at::empty(v.sizes(), v.options());
    const at::Tensor fin = inplace ? *state
                                   : at::empty({sh.value_streams, sh.key_dim, sh.value_dim}, v.options().dtype(at::kFloat));
    size_t bytes = 0, record_bytes = 0;
    check_status(race_delta_fwd_workspace_bytes(&sh, want_records, &bytes, &record_bytes), "race_delta_fwd_workspace_bytes");
    c10::optional<at::Tensor> records;
    if (want_records) records = workspace_of(record_bytes, q);
    const at::Tensor ws = bytes > 0 ? workspace_of(bytes, q) : at::Tensor();
    if (inplace) state->unsafeGetTensorImpl()->bump_version();  // a graph that saved it must notice
    check_status(race_delta_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), data_of(gate), beta.data_ptr(), floats_of(state),
                                lengths_of(lengths), out.data_ptr(), fin.data_ptr<float>(), ptr_of(records), &sh,
                                bytes > 0 ? ws.data_ptr() : nullptr, bytes, current_stream()),
                 "race_delta_fwd");
    return {out, fin, records};
}

struct DeltaBackward {
    c10::optional<at::Tensor> dq, dk, dv, dgate, dbeta, dstate;
};

// Gradients for those asked for, in the order q, k, v, gate, beta, state.
DeltaBackward delta_backward(const at::Tensor& q, const at::Tensor& k, const c10::optional<at::Tensor>& gate,
                             const at::Tensor& beta, const c10::optional<at::Tensor>& lengths, const at::Tensor& dout,
                             const c10::optional<at::Tensor>& dfinal, const at::Tensor& records, int64_t form, double scale,
                             const std::vector<bool>& need) {
    const char* entry = "race_delta_rule backward";
    const race_delta_shape sh = delta_shape(entry, q, k, dout, gate, beta, dfinal, lengths, form, scale);
    size_t bytes = 0, record_bytes = 0;
    check_status(race_delta_fwd_workspace_bytes(&sh, 1, &bytes, &record_bytes), "race_delta_fwd_workspace_bytes");
    check_status(race_delta_bwd_workspace_bytes(&sh, &bytes), "race_delta_bwd_workspace_bytes");
    ArgCheck(entry).on_gpu("dout", dout).on_gpu("records", records)
        .require(records.scalar_type() == at::kFloat && records.device() == q.device() &&
                     records.numel() == static_cast<int64_t>((record_bytes + 3) / 4),
                 "records", "are not those of the forward of these inputs")
        .raise();
    const c10::DeviceGuard guard(q.device());
    DeltaBackward g;
    if (need[0]) g.dq = at::empty(q.sizes(), q.options());
    if (need[1]) g.dk = at::empty(k.sizes(), k.options());
    if (need[2]) g.dv = at::empty(dout.sizes(), dout.options());
    if (need[3]) g.dgate = at::empty(beta.sizes(), beta.options());
    if (need[4]) g.dbeta = at::empty(beta.sizes(), beta.options());
    if (need[5]) g.dstate = at::empty({sh.value_streams, sh.key_dim, sh.value_dim}, q.options().dtype(at::kFloat));
    const at::Tensor ws = workspace_of(bytes, q);
    check_status(race_delta_bwd(q.data_ptr(), k.data_ptr(), data_of(gate), beta.data_ptr(), lengths_of(lengths),
                                dout.data_ptr(), floats_of(dfinal), records.data_ptr(), ptr_of(g.dq), ptr_of(g.dk),
                                ptr_of(g.dv), ptr_of(g.dgate), ptr_of(g.dbeta), floats_of(g.dstate), &sh, ws.data_ptr(), bytes,
                                current_stream()),
                 "race_delta_bwd");
    return g;
}

// ---- the operators with their gradients ----

struct DeltaHeld : torch::CustomClassHolder {
    c10::optional<at::Tensor> lengths;
    int64_t form;
    double scale;
    bool state;
    std::vector<int64_t> v_sizes;
};

struct DeltaNode : torch::autograd::Function<DeltaNode> {
    static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                 const c10::optional<at::Tensor>& gate, const at::Tensor& beta,
                                 const c10::optional<at::Tensor>& state, const c10::intrusive_ptr<DeltaHeld>& h) {
        const auto [out, fin, records] = delta_forward("race_delta_rule", q, k, v, gate, beta, state, h->lengths, h->form,
                                                       h->scale, true, false);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({q, k, or_undefined(gate), beta, or_undefined(h->lengths), *records});
        h->lengths = c10::nullopt;
        h->state = state.has_value();
        h->v_sizes.assign(v.sizes().begin(), v.sizes().end());
        ctx->saved_data["held"] = c10::IValue::make_capsule(h);
        return {out, fin};
    }
    static variable_list backward(AutogradContext* ctx, variable_list up) {
        variable_list grads(7);
        const variable_list saved = ctx->get_saved_variables();
        const DeltaHeld& h = held<DeltaHeld>(ctx);
        const at::Tensor &q = saved[0], &k = saved[1], &beta = saved[3];
        const auto gate = if_defined(saved[2]);
        check_capture("race_delta_rule backward", {q, k, gate, beta});
        if (up[0].defined() || up[1].defined()) {
            const auto need = needed(ctx, {true, true, true, gate.has_value(), true, h.state});
            const auto dout = dense_grad(up[0].defined() ? up[0] : at::zeros(h.v_sizes, q.options()), q.scalar_type());
            const DeltaBackward g = delta_backward(q, k, gate, beta, if_defined(saved[4]), *dout, dense_grad(up[1], at::kFloat),
                                                   saved[5], h.form, h.scale, need);
            grads = {or_undefined(g.dq),    or_undefined(g.dk),    or_undefined(g.dv), or_undefined(g.dgate),
                     or_undefined(g.dbeta), or_undefined(g.dstate), at::Tensor()};
        }
        return differentiated_once("race_delta_rule", up, std::move(grads));
    }
};

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

// The residual stream's gradient; the rows in 8 bits and their scales have none.
struct AddNormE4m3Node : torch::autograd::Function<AddNormE4m3Node> {
    static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& residual,
                                 const c10::optional<at::Tensor>& weight, double eps, int64_t group) {
        const auto [y, sum, scales] = add_norm_forward("race_add_norm_e4m3", x, residual, weight, eps, true, group);
        ctx->set_materialize_grads(false);
        ctx->mark_non_differentiable({y, *scales});
        return {y, *scales, *sum};
    }
    static variable_list backward(AutogradContext*, variable_list up) {
        return {up[2], up[2], at::Tensor(), at::Tensor(), at::Tensor()};
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

// For calls without derivatives.
void refuse_tangents(const char* entry, std::initializer_list<c10::optional<at::Tensor>> inputs) {
    for (const auto& t : inputs)
        TORCH_CHECK(!t || !t->_fw_grad(0).defined(), entry, ": an input has a forward-mode tangent; the call has no jvp");
}

// Rows of any leading dimensions as [rows, D]: a view where one row stride
// reaches them all, else a copy.
at::Tensor as_matrix(const char* entry, const char* name, const at::Tensor& t) {
    ArgCheck(entry).require(t.dim() >= 1, name, "is a scalar; rows [..., D] are taken").raise();
    return as_rows(t.dim() == 2 ? t : t.dim() == 1 ? t.unsqueeze(0) : t.flatten(0, -2));
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

// (y in e4m3, scales, sum or None); gradients through sum alone.
std::tuple<at::Tensor, at::Tensor, c10::optional<at::Tensor>> add_norm_e4m3(
    const at::Tensor& x_in, const c10::optional<at::Tensor>& residual_in, const c10::optional<at::Tensor>& weight, double eps,
    int64_t group) {
    const char* entry = "race_add_norm_e4m3";
    refuse_tangents(entry, {x_in, residual_in, weight});
    const bool node = residual_in && wants_grad({x_in, residual_in});
    if (node) check_capture(entry, {x_in, residual_in});
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
    at::Tensor y;
    c10::optional<at::Tensor> sum, scales;
    if (node) {
        const variable_list outs = AddNormE4m3Node::apply(x, *residual, weight, eps, group);
        y = outs[0], scales = outs[1], sum = outs[2];
    } else {
        std::tie(y, sum, scales) = add_norm_forward(entry, x, residual, weight, eps, true, group);
    }
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

std::tuple<at::Tensor, at::Tensor> delta_rule(const at::Tensor& q_in, const at::Tensor& k_in, const at::Tensor& v_in,
                                              const c10::optional<at::Tensor>& gate_in, const at::Tensor& beta_in,
                                              const c10::optional<at::Tensor>& state,
                                              const c10::optional<at::Tensor>& lengths_in, int64_t form, double scale) {
    const char* entry = "race_delta_rule";
    const bool node = wants_grad({q_in, k_in, v_in, gate_in, beta_in, state});
    if (node) check_capture(entry, {q_in, k_in, v_in, gate_in, beta_in, state});
    const at::Tensor q = as_key_rows(q_in), k = as_key_rows(k_in), v = as_rows(v_in, kDeltaFar), beta = as_per_token(beta_in);
    const auto gate = as_per_token(gate_in);
    const auto lengths = as_lengths(lengths_in);
    if (!node) {
        const auto r = delta_forward(entry, q, k, v, gate, beta, state, lengths, form, scale, false, false);
        return {std::get<0>(r), std::get<1>(r)};
    }
    auto h = c10::make_intrusive<DeltaHeld>();
    h->lengths = lengths, h->form = form, h->scale = scale;
    const variable_list outs = DeltaNode::apply(q, k, v, gate, beta, state, h);
    return {outs[0], outs[1]};
}

std::tuple<at::Tensor, at::Tensor> delta_rule_carry(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                                    const c10::optional<at::Tensor>& gate, const at::Tensor& beta,
                                                    const at::Tensor& state, const c10::optional<at::Tensor>& lengths,
                                                    int64_t form, double scale, bool inplace) {
    refuse_tangents("race_delta_rule_carry", {q, k, v, gate, beta, state});
    const auto r = delta_forward("race_delta_rule_carry", as_key_rows(q), as_key_rows(k), as_rows(v, kDeltaFar),
                                 as_per_token(gate), as_per_token(beta), state, as_lengths(lengths), form, scale, false, inplace);
    return {std::get<0>(r), std::get<1>(r)};
}

void bind_recurrent_layer(pybind11::module& m) {
    namespace py = pybind11;
    m.def("delta_rule", &delta_rule, "race_delta_rule with its gradients -> (out, final state)", py::arg("q"), py::arg("k"),
          py::arg("v"), py::arg("gate"), py::arg("beta"), py::arg("state"), py::arg("lengths"), py::arg("form"),
          py::arg("scale"));
    m.def("delta_rule_carry", &delta_rule_carry, "race_delta_rule from a carried state -> (out, state)", py::arg("q"),
          py::arg("k"), py::arg("v"), py::arg("gate"), py::arg("beta"), py::arg("state"), py::arg("lengths"), py::arg("form"),
          py::arg("scale"), py::arg("inplace"));
    m.def("add_norm", &add_norm, "race_add_norm with its gradients -> (y, sum or None)", py::arg("x"), py::arg("residual"),
          py::arg("weight"), py::arg("eps"));
    m.def("add_norm_e4m3", &add_norm_e4m3, "race_add_norm with y in 8 bits -> (y, scales, sum or None)", py::arg("x"),
          py::arg("residual"), py::arg("weight"), py::arg("eps"), py::arg("group"));
    m.def("gate_norm", &gate_norm, "race_gate_norm with its gradients -> y", py::arg("x"), py::arg("gate"),
          py::arg("weight"), py::arg("eps"));
}

}  // namespace
