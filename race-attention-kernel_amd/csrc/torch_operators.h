// torch_operators.h -- the part of the PyTorch binding for the operators beside
// the per-bucket op; included by torch_ext.cpp, whose helpers it uses.
#pragma once

namespace {

hipStream_t current_stream() { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream(); }

int32_t dtype_of(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 ? RACE_BF16 : RACE_F32; }

at::Tensor workspace_of(size_t bytes, const at::Tensor& like) {
    return at::empty({static_cast<int64_t>((bytes + 3) / 4)}, like.options().dtype(at::kFloat));
}

void* ptr_of(const c10::optional<at::Tensor>& t) { return t ? t->data_ptr() : nullptr; }
float* floats_of(const c10::optional<at::Tensor>& t) { return t ? t->data_ptr<float>() : nullptr; }

bool starts_aligned(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// Rows read by strides: on the GPU, aligned, the last dimension dense.
void check_rows(ArgCheck& c, const char* name, const at::Tensor& t, int64_t dim, const char* layout) {
    c.require(t.is_cuda(), name, "lives on the CPU; the library reads it on the GPU")
        .dtype_is(name, t, true)
        .require(t.dim() == dim, name, [&] { return "has shape " + dims(t) + ", not " + layout; })
        .require(t.dim() != dim || t.numel() == 0 || t.size(dim - 1) == 1 || t.stride(dim - 1) == 1, name,
                 "has a strided last dimension; its elements must be next to each other")
        .require(t.numel() == 0 || starts_aligned(t), name,
                 "starts at an address that is not a multiple of 16 bytes; pass a fresh copy");
}

// One int32 per `per` consecutive streams, on the rows' device.
int64_t check_lengths(ArgCheck& c, const c10::optional<at::Tensor>& lengths, const at::Tensor& rows, int64_t streams) {
    if (!lengths) return 1;
    const at::Tensor& l = *lengths;
    c.require(l.scalar_type() == at::kInt && l.device() == rows.device() && l.is_contiguous() && l.dim() == 1, "lengths",
              "must be a contiguous int32 vector on the rows' device")
        .require(l.numel() > 0 ? streams % l.numel() == 0 : streams == 0, "lengths",
                 [&] { return "has " + std::to_string(l.numel()) + " entries, which do not divide the " + std::to_string(streams) +
                     " streams"; });
    return l.dim() == 1 && l.numel() > 0 && streams >= l.numel() ? streams / l.numel() : 1;
}

// Refuses a differentiable call on a stream under capture whose leaf inputs are
// still held by a graph from the default stream: the backward would wait for
// that stream inside the capture, which ends the process.  Deleting the eager
// outputs (or detaching them) frees the leaves.  `inputs` are the caller's own:
// a copy as_rows makes of a leaf is none.
void check_capture(const char* entry, const std::vector<c10::optional<at::Tensor>>& inputs) {
    bool capturing = false, asked = false;
    for (const auto& t : inputs) {
        if (!t || !t->defined() || !t->is_cuda() || !t->requires_grad() || !t->is_leaf()) continue;
        if (!asked) {
            hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
            const hipStream_t stream = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t->device().index()).stream();
            TORCH_CHECK(hipStreamIsCapturing(stream, &status) == hipSuccess, entry, ": hipStreamIsCapturing failed");
            capturing = status == hipStreamCaptureStatusActive;
            asked = true;
        }
        if (!capturing) return;
        const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
        const auto stream = node ? node->stream() : c10::nullopt;
        TORCH_CHECK(!stream || stream->id() != 0, entry,
                    ": an input that requires a gradient belongs to a graph built on the default stream that is still "
                    "alive, so its backward cannot be captured; delete or detach that graph's outputs first");
    }
}

// ---- gated linear recurrence ----

race_scan_shape scan_shape(const char* entry, const at::Tensor& x, const at::Tensor& gate,
                           const c10::optional<at::Tensor>& state, const c10::optional<at::Tensor>& lengths,
                           int64_t form, bool complement) {
    ArgCheck c(entry);
    check_rows(c, "x", x, 3, "[N, T, D]");
    check_rows(c, "gate", gate, 3, "[N, T, D]");
    c.matches("gate", gate, "x", x)
        .require(gate.sizes() == x.sizes(), "gate", [&] { return "has shape " + dims(gate) + ", x " + dims(x); });
    c.raise();
    const int64_t N = x.size(0), D = x.size(2);
    if (state)
        c.on_gpu("state", *state)
            .require(state->scalar_type() == at::kFloat && state->device() == x.device(), "state",
                     "must be float32 on x's device")
            .require(state->sizes() == at::IntArrayRef({N, D}), "state", [&] { return "has shape " + dims(*state) + ", not [N, D]"; });
    const int64_t group = check_lengths(c, lengths, x, N);
    c.require(N <= 65535 && D >= 1 && D <= 65536, "x",
              [&] { return "has shape " + dims(x) + "; the scan takes up to 65535 streams of 1 .. 65536 channels"; })
        .raise();
    race_scan_shape sh{};
    sh.num_streams = N;
    sh.seq_len = x.size(1);
    sh.channels = D;
    // The stride of a dimension with one entry is never used.
    sh.x_stream_stride = N > 1 ? x.stride(0) : 0;
    sh.x_token_stride = sh.seq_len > 1 ? x.stride(1) : 0;
    sh.gate_stream_stride = N > 1 ? gate.stride(0) : 0;
    sh.gate_token_stride = sh.seq_len > 1 ? gate.stride(1) : 0;
    sh.dtype = dtype_of(x);
    sh.gate_form = static_cast<int32_t>(form);
    sh.complement = complement;
    sh.lengths_group = static_cast<int32_t>(group);
    return sh;
}

std::tuple<at::Tensor, at::Tensor, c10::optional<at::Tensor>> gated_scan_forward(
    const at::Tensor& x, const at::Tensor& gate, const c10::optional<at::Tensor>& state,
    const c10::optional<at::Tensor>& lengths, int64_t form, bool complement, bool want_records, bool inplace) {
    const race_scan_shape sh = scan_shape("race_gated_scan", x, gate, state, lengths, form, complement);
    TORCH_CHECK(!inplace || state, "race_gated_scan_carry: an in-place call needs a state");
    TORCH_CHECK(!inplace || !(at::GradMode::is_enabled() && state->requires_grad()),
                "race_gated_scan_carry: a state that requires a gradient cannot be advanced in place");
    const c10::DeviceGuard guard(x.device());
    const at::Tensor out = at::empty(x.sizes(), x.options());
    const auto fopt = x.options().dtype(at::kFloat);
    const at::Tensor fin = inplace ? *state : at::empty({sh.num_streams, sh.channels}, fopt);
    size_t bytes = 0;
    int64_t floats = 0;
    check_status(race_gated_scan_workspace_bytes(&sh, 0, &bytes, &floats), "race_gated_scan_workspace_bytes");
    c10::optional<at::Tensor> records;
    if (want_records) records = at::empty({floats}, fopt);
    const at::Tensor ws = bytes > 0 ? workspace_of(bytes, x) : at::Tensor();
    if (inplace) state->unsafeGetTensorImpl()->bump_version();  // a graph that saved it must notice
    check_status(race_gated_scan_fwd(x.data_ptr(), gate.data_ptr(), floats_of(state),
                                     lengths ? lengths->data_ptr<int32_t>() : nullptr, out.data_ptr(),
                                     fin.data_ptr<float>(), floats_of(records), &sh, bytes > 0 ? ws.data_ptr() : nullptr,
                                     bytes, current_stream()),
                 "race_gated_scan_fwd");
    return {out, fin, records};
}

std::tuple<c10::optional<at::Tensor>, c10::optional<at::Tensor>, c10::optional<at::Tensor>> gated_scan_backward(
    const at::Tensor& x, const at::Tensor& gate, const c10::optional<at::Tensor>& lengths, const at::Tensor& dout,
    const c10::optional<at::Tensor>& dfinal, const at::Tensor& records, int64_t form, bool complement, bool need_x,
    bool need_gate, bool need_state) {
    const char* entry = "race_gated_scan backward";
    const race_scan_shape sh = scan_shape(entry, x, gate, dfinal, lengths, form, complement);
    size_t bytes = 0;
    int64_t floats = 0;
    check_status(race_gated_scan_workspace_bytes(&sh, 1, &bytes, &floats), "race_gated_scan_workspace_bytes");
    ArgCheck(entry).on_gpu("dout", dout).matches("dout", dout, "x", x)
        .require(dout.sizes() == x.sizes(), "dout", [&] { return "has shape " + dims(dout) + ", x " + dims(x); })
        .on_gpu("records", records)
        .require(records.scalar_type() == at::kFloat && records.device() == x.device() && records.numel() == floats,
                 "records", "are not those of the forward of these inputs")
        .raise();
    const c10::DeviceGuard guard(x.device());
    c10::optional<at::Tensor> dx, dgate, dstate;
    if (need_x) dx = at::empty(x.sizes(), x.options());
    if (need_gate) dgate = at::empty(x.sizes(), x.options());
    if (need_state) dstate = at::empty({sh.num_streams, sh.channels}, x.options().dtype(at::kFloat));
    const at::Tensor ws = bytes > 0 ? workspace_of(bytes, x) : at::Tensor();
    check_status(race_gated_scan_bwd(x.data_ptr(), gate.data_ptr(), lengths ? lengths->data_ptr<int32_t>() : nullptr,
                                     dout.data_ptr(), floats_of(dfinal), records.data_ptr<float>(), ptr_of(dx),
                                     ptr_of(dgate), floats_of(dstate), &sh, bytes > 0 ? ws.data_ptr() : nullptr, bytes,
                                     current_stream()),
                 "race_gated_scan_bwd");
    return {dx, dgate, dstate};
}

// ---- norm and rotation of query and key heads ----

struct RopeCall {
    race_norm_rope_shape sh{};
    int64_t B = 0, T = 0, d = 0;
};

RopeCall rope_call(const char* entry, const at::Tensor& q, const c10::optional<at::Tensor>& k,
                   const c10::optional<at::Tensor>& positions, const c10::optional<at::Tensor>& inv_freq,
                   const c10::optional<at::Tensor>& q_weight, const c10::optional<at::Tensor>& k_weight, double eps,
                   bool norm, const std::vector<int64_t>& sections, bool interleaved) {
    ArgCheck c(entry);
    check_rows(c, "q", q, 4, "[B, T, H, d]");
    c.raise();
    RopeCall r;
    r.B = q.size(0), r.T = q.size(1), r.d = q.size(3);
    c.require(q.size(2) >= 1 && q.size(2) <= 65535 && r.d >= 1 && r.d <= 256, "q",
              [&] { return "has shape " + dims(q) + "; rows of 1 .. 256 values in 1 .. 65535 heads are taken"; })
        .require(r.T == 0 || r.B <= (int64_t(1) << 30) / r.T, "q", "has more than 2^30 tokens");
    if (k) {
        check_rows(c, "k", *k, 4, "[B, T, H, d]");
        c.matches("k", *k, "q", q)
            .require(k->dim() == 4 && k->size(0) == r.B && k->size(1) == r.T && k->size(3) == r.d && k->size(2) >= 1 &&
                         k->size(2) <= 65535,
                     "k", [&] { return "has shape " + dims(*k) + ", not q's batch, tokens and head width"; });
    }
    int64_t pairs = 0;
    const bool many = inv_freq && sections.size() > 1;  // without a rotation there are no axes
    if (inv_freq) {
        c.on_gpu("inv_freq", *inv_freq)
            .require(inv_freq->scalar_type() == at::kFloat && inv_freq->device() == q.device() && inv_freq->dim() == 1,
                     "inv_freq", "must be a float32 vector on q's device")
            .require(2 * inv_freq->numel() <= r.d, "inv_freq",
                     [&] { return "has " + std::to_string(inv_freq->numel()) + " pairs, more than half of d = " + std::to_string(r.d); });
        pairs = inv_freq->numel();
        c.require(positions.has_value(), "positions", "are needed for a rotation");
        if (positions) {
            const at::Tensor& p = *positions;
            c.require(p.device() == q.device() && (p.scalar_type() == at::kInt || p.scalar_type() == at::kLong),
                      "positions", "must be int32 or int64 on q's device")
                .require(p.dim() >= 1 && p.dim() <= 3 && p.size(p.dim() - 1) == r.T &&
                             (p.dim() < 2 || p.size(p.dim() - 2) == r.B),
                         "positions", [&] { return "have shape " + dims(p) + ", not [T], [B, T] or [axes, B, T]"; })
                .require(sections.size() <= 4 && (p.dim() == 3 ? p.size(0) == int64_t(many ? sections.size() : 1) : !many),
                         "positions", [&] { return "have shape " + dims(p) + " for " +
                                          std::to_string(sections.empty() ? 1 : sections.size()) +
                                          " sections; one axis each (at most 4)"; });
        }
        int64_t sum = 0;
        for (int64_t s : sections) {
            c.require(s >= 0 && s <= 256, "sections", "hold a count that is not 0 .. 256");
            sum += s;
        }
        c.require(sections.empty() || sum == pairs, "sections",
                  [&] { return "sum to " + std::to_string(sum) + ", not the " + std::to_string(pairs) + " pairs of inv_freq"; });
    }
    at::ScalarType wt = q.scalar_type();
    bool first = true;
    for (const auto& [name, w] : {std::make_pair("q_weight", &q_weight), std::make_pair("k_weight", &k_weight)}) {
        if (!*w) continue;
        const at::Tensor& t = **w;
        c.on_gpu(name, t).dtype_is(name, t, true)
            .require(t.device() == q.device() && t.dim() == 1 && t.numel() == r.d, name,
                     [&] { return "must hold d = " + std::to_string(r.d) + " values on q's device"; })
            .require(first || t.scalar_type() == wt, name, "has another dtype than q_weight")
            .require(norm, name, "is given without a norm (eps is None)");
        wt = t.scalar_type(), first = false;
    }
    c.require(!norm || (eps >= 0 && eps < 1e30), "eps", "must be a number of at least 0").raise();
    race_norm_rope_shape& sh = r.sh;
    sh.batch = r.B, sh.seq_len = r.T;
    sh.q_heads = static_cast<int32_t>(q.size(2)), sh.k_heads = k ? static_cast<int32_t>(k->size(2)) : 0;
    sh.head_dim = static_cast<int32_t>(r.d), sh.pairs = static_cast<int32_t>(pairs);
    auto stride = [](const at::Tensor& t, int64_t i) { return t.size(i) > 1 ? t.stride(i) : 0; };
    sh.q_batch_stride = stride(q, 0), sh.q_token_stride = stride(q, 1), sh.q_head_stride = stride(q, 2);
    if (k) sh.k_batch_stride = stride(*k, 0), sh.k_token_stride = stride(*k, 1), sh.k_head_stride = stride(*k, 2);
    sh.axes = many ? static_cast<int32_t>(sections.size()) : 1;
    for (int i = 0; i < sh.axes; ++i) sh.sections[i] = static_cast<int32_t>(many ? sections[i] : pairs);
    sh.pos_bits = 64;
    if (pairs > 0) {
        const at::Tensor& p = *positions;
        const int64_t n = p.dim();
        sh.pos_bits = p.scalar_type() == at::kLong ? 64 : 32;
        sh.pos_token_stride = stride(p, n - 1);
        sh.pos_batch_stride = n > 1 ? stride(p, n - 2) : 0;
        sh.pos_axis_stride = n > 2 ? stride(p, 0) : 0;
    }
    sh.interleaved = interleaved, sh.norm = norm, sh.eps = static_cast<float>(eps);
    sh.dtype = dtype_of(q), sh.weight_dtype = wt == at::kFloat ? RACE_F32 : RACE_BF16;
    return r;
}

const void* data_of(const c10::optional<at::Tensor>& t) { return t ? t->data_ptr() : nullptr; }

std::tuple<at::Tensor, c10::optional<at::Tensor>> norm_rope_forward(
    const at::Tensor& q, const c10::optional<at::Tensor>& k, const c10::optional<at::Tensor>& positions,
    const c10::optional<at::Tensor>& inv_freq, const c10::optional<at::Tensor>& q_weight,
    const c10::optional<at::Tensor>& k_weight, double eps, bool norm, const std::vector<int64_t>& sections,
    bool interleaved) {
    const RopeCall r = rope_call("race_norm_rope", q, k, positions, inv_freq, q_weight, k_weight, eps, norm, sections,
                                 interleaved);
    const c10::DeviceGuard guard(q.device());
    const at::Tensor q_out = at::empty({r.B * q.size(2), r.T, r.d}, q.options());
    c10::optional<at::Tensor> k_out;
    if (k) k_out = at::empty({r.B * k->size(2), r.T, r.d}, q.options());
    check_status(race_norm_rope_fwd(q.data_ptr(), data_of(k), data_of(positions),
                                    static_cast<const float*>(data_of(inv_freq)), data_of(q_weight), data_of(k_weight),
                                    q_out.data_ptr(), ptr_of(k_out), &r.sh, current_stream()),
                 "race_norm_rope_fwd");
    return {q_out, k_out};
}

// Gradients of q, k and the weights, for those asked for; dq_out or dk_out
// missing leaves that tensor's out.
std::tuple<c10::optional<at::Tensor>, c10::optional<at::Tensor>, c10::optional<at::Tensor>, c10::optional<at::Tensor>>
norm_rope_backward(const at::Tensor& q, const c10::optional<at::Tensor>& k, const c10::optional<at::Tensor>& positions,
                   const c10::optional<at::Tensor>& inv_freq, const c10::optional<at::Tensor>& q_weight,
                   const c10::optional<at::Tensor>& k_weight, const c10::optional<at::Tensor>& dq_out,
                   const c10::optional<at::Tensor>& dk_out, double eps, bool norm, const std::vector<int64_t>& sections,
                   bool interleaved, bool need_q, bool need_k, bool need_qw, bool need_kw) {
    const char* entry = "race_norm_rope backward";
    const RopeCall r = rope_call(entry, q, k, positions, inv_freq, q_weight, k_weight, eps, norm, sections, interleaved);
    ArgCheck c(entry);
    if (dq_out)
        c.on_gpu("dq_out", *dq_out).matches("dq_out", *dq_out, "q", q)
            .require(dq_out->sizes() == at::IntArrayRef({r.B * q.size(2), r.T, r.d}), "dq_out", [&] { return "has shape " + dims(*dq_out); });
    if (dk_out)
        c.require(k.has_value(), "dk_out", "is given without k")
            .on_gpu("dk_out", *dk_out).matches("dk_out", *dk_out, "q", q)
            .require(k && dk_out->sizes() == at::IntArrayRef({r.B * k->size(2), r.T, r.d}), "dk_out",
                     [&] { return "has shape " + dims(*dk_out); });
    c.raise();
    const c10::DeviceGuard guard(q.device());
    c10::optional<at::Tensor> dq, dk, dqw, dkw;
    if (need_q && dq_out) dq = at::empty(q.sizes(), q.options());
    if (need_k && dk_out) dk = at::empty(k->sizes(), k->options());
    if (need_qw && dq_out && q_weight) dqw = at::empty_like(*q_weight);
    if (need_kw && dk_out && k_weight) dkw = at::empty_like(*k_weight);
    if (r.B == 0 || r.T == 0) {  // empty tensors have no address to hand on
        if (dqw) dqw->zero_();
        if (dkw) dkw->zero_();
        return {dq, dk, dqw, dkw};
    }
    size_t bytes = 0;
    at::Tensor ws;
    if (dqw || dkw) {
        check_status(race_norm_rope_bwd_workspace_bytes(&r.sh, &bytes), "race_norm_rope_bwd_workspace_bytes");
        ws = workspace_of(bytes, q);
    }
    check_status(race_norm_rope_bwd(q.data_ptr(), data_of(k), data_of(positions),
                                    static_cast<const float*>(data_of(inv_freq)), data_of(q_weight), data_of(k_weight),
                                    data_of(dq_out), data_of(dk_out), ptr_of(dq), ptr_of(dk), ptr_of(dqw), ptr_of(dkw),
                                    &r.sh, bytes > 0 ? ws.data_ptr() : nullptr, bytes, current_stream()),
                 "race_norm_rope_bwd");
    return {dq, dk, dqw, dkw};
}

// ---- the non-causal op between two sequences ----

struct CrossCall {
    race_cross_shape sh{};
    int64_t S = 0, d = 0, Nq = 0, Tq = 0;
};

int64_t buckets_of(const at::Tensor& t) { return t.dim() == 4 ? t.size(2) * t.size(3) : t.size(2); }

// q (nullable): [Nq, Tq, L, R] or [Nq, Tq, S]; k likewise and V [Nk, Tk, d], or
// in their place a state [Nk, S*d + S].
CrossCall cross_call(const char* entry, const at::Tensor* q, const at::Tensor* k, const at::Tensor* v,
                     const at::Tensor* state, const c10::optional<at::Tensor>& lengths) {
    ArgCheck c(entry);
    CrossCall r;
    const at::Tensor& ref = q ? *q : *k;
    auto probs = [&](const char* name, const at::Tensor& t) {
        c.on_gpu(name, t).dtype_is(name, t, true)
            .require(t.dim() == 3 || t.dim() == 4, name, [&] { return "has shape " + dims(t) + ", not [N, T, L, R] or [N, T, S]"; });
    };
    if (q) probs("probsQ", *q);
    if (k) probs("probsK", *k);
    c.raise();
    r.S = buckets_of(ref);
    int64_t Nk = 0;
    if (k) {
        Nk = k->size(0);
        c.matches("probsK", *k, "probsQ", ref)
            .require(buckets_of(*k) == r.S, "probsK", [&] { return "has shape " + dims(*k) + ", another number of buckets than probsQ"; })
            .on_gpu("V", *v).matches("V", *v, "probsK", *k)
            .require(v->dim() == 3 && v->size(0) == Nk && v->size(1) == k->size(1), "V",
                     [&] { return "has shape " + dims(*v) + ", not [N, T, d] with probsK's N and T"; });
        if (v->dim() == 3) r.d = v->size(2);
        r.sh.kv_len = k->size(1);
    } else {
        c.on_gpu("state", *state)
            .require(state->scalar_type() == at::kFloat && state->device() == ref.device(), "state",
                     "must be float32 on probsQ's device")
            .require(state->dim() == 2 && r.S > 0 && state->size(1) % r.S == 0 && state->size(1) / r.S >= 2, "state",
                     [&] { return "has shape " + dims(*state) + ", not [N, S*d + S] with probsQ's S"; });
        c.raise();
        Nk = state->size(0);
        r.d = state->size(1) / r.S - 1;
    }
    r.Nq = q ? q->size(0) : Nk, r.Tq = q ? q->size(1) : 0;
    c.require(Nk > 0 ? r.Nq % Nk == 0 : r.Nq == 0, "probsQ",
              [&] { return "has " + std::to_string(r.Nq) + " streams, no multiple of the " + std::to_string(Nk) + " key streams"; });
    const int64_t group = check_lengths(c, lengths, ref, Nk);
    const int64_t heads = Nk > 0 ? std::max<int64_t>(r.Nq / Nk, 1) : 1;
    constexpr int64_t kMost = int64_t(1) << 30;
    c.require(Nk <= 65535 && r.S >= 1 && r.S <= 256 && r.d >= 1 && r.d <= 128 && heads <= kMost && r.Tq <= kMost / heads &&
                  r.sh.kv_len <= kMost,
              "probsQ", "has no kernel: up to 65535 key streams, S <= 256 buckets, d <= 128 columns and 2^30 tokens a "
                        "key stream are taken")
        .raise();
    r.sh.kv_streams = Nk, r.sh.q_len = r.Nq > 0 ? r.Tq * heads : 0;
    r.sh.num_tables = 1, r.sh.num_buckets = static_cast<int32_t>(r.S), r.sh.head_dim = static_cast<int32_t>(r.d);
    r.sh.dtype = dtype_of(ref), r.sh.lengths_group = static_cast<int32_t>(group);
    return r;
}

const int32_t* lengths_of(const c10::optional<at::Tensor>& t) { return t ? t->data_ptr<int32_t>() : nullptr; }

// (out or None, state or None).
std::tuple<c10::optional<at::Tensor>, c10::optional<at::Tensor>> cross_forward(
    const c10::optional<at::Tensor>& q, const at::Tensor& k, const at::Tensor& v,
    const c10::optional<at::Tensor>& lengths, bool want_state) {
    const CrossCall r = cross_call(q ? "race_cross_fwd" : "race_cross_state", q ? &*q : nullptr, &k, &v, nullptr, lengths);
    const c10::DeviceGuard guard(k.device());
    c10::optional<at::Tensor> out, state;
    if (q) out = at::empty({r.Nq, r.Tq, r.d}, v.options());
    if (want_state) state = at::empty({r.sh.kv_streams, r.S * r.d + r.S}, v.options().dtype(at::kFloat));
    size_t bytes = 0;
    check_status(race_cross_fwd_workspace_bytes(&r.sh, &bytes), "race_cross_fwd_workspace_bytes");
    const at::Tensor ws = workspace_of(bytes, k);
    check_status(race_cross_fwd(q ? q->data_ptr() : nullptr, k.data_ptr(), v.data_ptr(), lengths_of(lengths), ptr_of(out),
                                floats_of(state), &r.sh, ws.data_ptr(), bytes, current_stream()),
                 "race_cross_fwd");
    return {out, state};
}

at::Tensor cross_query(const at::Tensor& q, const at::Tensor& state) {
    const CrossCall r = cross_call("race_cross_query", &q, nullptr, nullptr, &state, c10::nullopt);
    const c10::DeviceGuard guard(q.device());
    const at::Tensor out = at::empty({r.Nq, r.Tq, r.d}, q.options());
    check_status(race_cross_query(q.data_ptr(), state.data_ptr<float>(), out.data_ptr(), &r.sh, current_stream()),
                 "race_cross_query");
    return out;
}

std::tuple<c10::optional<at::Tensor>, c10::optional<at::Tensor>, c10::optional<at::Tensor>> cross_backward(
    const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const c10::optional<at::Tensor>& lengths,
    const at::Tensor& dout, const at::Tensor& state, bool need_q, bool need_k, bool need_v) {
    const char* entry = "race_cross_fwd backward";
    const CrossCall r = cross_call(entry, &q, &k, &v, nullptr, lengths);
    ArgCheck(entry).on_gpu("dout", dout).matches("dout", dout, "V", v)
        .require(dout.sizes() == at::IntArrayRef({r.Nq, r.Tq, r.d}), "dout", [&] { return "has shape " + dims(dout); })
        .on_gpu("state", state)
        .require(state.scalar_type() == at::kFloat && state.device() == q.device() &&
                     state.sizes() == at::IntArrayRef({r.sh.kv_streams, r.S * r.d + r.S}),
                 "state", "is not the forward's float32 [N, S*d + S] state")
        .raise();
    const c10::DeviceGuard guard(q.device());
    c10::optional<at::Tensor> dq, dk, dv;
    if (need_q) dq = at::empty_like(q);
    if (need_k) dk = at::empty_like(k);
    if (need_v) dv = at::empty_like(v);
    size_t bytes = 0;
    check_status(race_cross_bwd_workspace_bytes(&r.sh, &bytes), "race_cross_bwd_workspace_bytes");
    const at::Tensor ws = workspace_of(bytes, q);
    check_status(race_cross_bwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), lengths_of(lengths), dout.data_ptr(),
                                state.data_ptr<float>(), ptr_of(dq), ptr_of(dk), ptr_of(dv), &r.sh, ws.data_ptr(), bytes,
                                current_stream()),
                 "race_cross_bwd");
    return {dq, dk, dv};
}

// ---- the operators with their gradients ----
// Autograd nodes in C++: a training step of small tensors is bound by the host,
// and nodes in Python cost it about 50 us more (forward and backward of a
// few rows through race_norm_rope: 93 us with one).

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Inputs the kernels read by strides; a copy where the last dimension is apart,
// the first value is not 16-byte aligned, or dimension 1 strides too far.
at::Tensor as_rows(const at::Tensor& t, int64_t far = int64_t(1) << 40) {
    const int64_t n = t.dim();
    if (t.numel() == 0 || n < 2) return t;
    const bool apart = t.size(n - 1) > 1 && t.stride(n - 1) != 1;
    if (!apart && starts_aligned(t) && !(t.size(1) > 1 && t.stride(1) > far)) return t;
    return t.clone(at::MemoryFormat::Contiguous);
}

c10::optional<at::Tensor> as_lengths(const c10::optional<at::Tensor>& lengths) {
    if (lengths && lengths->scalar_type() == at::kLong)
        return lengths->clamp(0, INT32_MAX).to(at::kInt).contiguous();
    return lengths;
}

// Whether a call takes its autograd node: for gradients, and for inputs with a
// forward-mode tangent, which a node without that mode refuses.
bool wants_grad(std::initializer_list<c10::optional<at::Tensor>> inputs) {
    for (const auto& t : inputs)
        if (t && t->_fw_grad(0).defined()) return true;
    if (!at::GradMode::is_enabled()) return false;
    for (const auto& t : inputs)
        if (t && t->requires_grad()) return true;
    return false;
}

// An upstream gradient as the kernels read it.
c10::optional<at::Tensor> dense_grad(const at::Tensor& g, at::ScalarType type) {
    if (!g.defined()) return c10::nullopt;
    at::Tensor t = g.detach().to(type).contiguous();
    return t.numel() > 0 && !starts_aligned(t) ? t.clone() : t;
}

c10::optional<at::Tensor> if_defined(const at::Tensor& t) {
    if (t.defined()) return t;
    return c10::nullopt;
}
at::Tensor or_undefined(const c10::optional<at::Tensor>& t) { return t ? *t : at::Tensor(); }

// Gradients of a node whose backward has none of its own: differentiating them
// raises, as once_differentiable does.
variable_list differentiated_once(const char* entry, const variable_list& upstream, variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    bool again = false;
    for (const at::Tensor& g : upstream) again = again || (g.defined() && g.requires_grad());
    if (!again) return grads;
    for (at::Tensor& g : grads)
        if (g.defined()) g = g.detach().requires_grad_(true);
    auto error = std::make_shared<torch::autograd::DelayedError>(
        std::string("trying to differentiate ") + entry + " twice, whose backward has no gradient",
        static_cast<int64_t>(grads.size()));
    return (*error)(std::move(grads));
}

// Which of the node's inputs need a gradient now (those that were given, in
// order, have the edges).
std::vector<bool> needed(AutogradContext* ctx, std::initializer_list<bool> given) {
    std::vector<bool> need;
    size_t edge = 0;
    for (bool there : given) need.push_back(there && ctx->needs_input_grad(edge++));
    return need;
}

// What a node keeps beside its saved tensors, and its tensors without gradients.
struct RopeHeld : torch::CustomClassHolder {
    c10::optional<at::Tensor> positions, inv_freq;  // for the forward
    double eps;
    bool norm, interleaved;
    std::vector<int64_t> sections;
};
struct ScanHeld : torch::CustomClassHolder {
    c10::optional<at::Tensor> lengths;
    int64_t form;
    bool complement;
};
struct CrossHeld : torch::CustomClassHolder {
    c10::optional<at::Tensor> lengths;
};

template <typename T>
const T& held(AutogradContext* ctx) {
    return static_cast<const T&>(*ctx->saved_data["held"].toCapsule());
}

struct NormRopeNode : torch::autograd::Function<NormRopeNode> {
    static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const c10::optional<at::Tensor>& k,
                                 const c10::optional<at::Tensor>& q_weight, const c10::optional<at::Tensor>& k_weight,
                                 const c10::intrusive_ptr<RopeHeld>& h) {
        const auto [q_out, k_out] = norm_rope_forward(q, k, h->positions, h->inv_freq, q_weight, k_weight, h->eps, h->norm,
                                                      h->sections, h->interleaved);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({q, or_undefined(k), or_undefined(q_weight), or_undefined(k_weight),
                                or_undefined(h->positions), or_undefined(h->inv_freq)});
        h->positions = h->inv_freq = c10::nullopt;
        ctx->saved_data["held"] = c10::IValue::make_capsule(h);
        if (k_out) return {q_out, *k_out};
        return {q_out};
    }
    static variable_list backward(AutogradContext* ctx, variable_list up) {
        variable_list grads(5);
        const variable_list saved = ctx->get_saved_variables();
        const RopeHeld& h = held<RopeHeld>(ctx);
        const at::Tensor& q = saved[0];
        const auto k = if_defined(saved[1]), qw = if_defined(saved[2]), kw = if_defined(saved[3]);
        check_capture("race_norm_rope backward", {q, k, qw, kw});
        const auto dq = dense_grad(up[0], q.scalar_type());
        const auto dk = up.size() > 1 ? dense_grad(up[1], q.scalar_type()) : c10::nullopt;
        if (dq || dk) {
            const auto need = needed(ctx, {true, k.has_value(), qw.has_value(), kw.has_value()});
            const auto [a, b, c, d] = norm_rope_backward(q, k, if_defined(saved[4]), if_defined(saved[5]), qw, kw, dq, dk,
                                                         h.eps, h.norm, h.sections, h.interleaved, need[0], need[1],
                                                         need[2], need[3]);
            grads = {or_undefined(a), or_undefined(b), or_undefined(c), or_undefined(d), at::Tensor()};
        }
        return differentiated_once("race_norm_rope", up, std::move(grads));
    }
};

struct GatedScanNode : torch::autograd::Function<GatedScanNode> {
    static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& gate,
                                 const c10::optional<at::Tensor>& state, const c10::intrusive_ptr<ScanHeld>& h) {
        const auto [out, fin, records] = gated_scan_forward(x, gate, state, h->lengths, h->form, h->complement, true, false);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({x, gate, or_undefined(h->lengths), *records});
        h->lengths = c10::nullopt;
        ctx->saved_data["held"] = c10::IValue::make_capsule(h);
        ctx->saved_data["state"] = state.has_value();
        return {out, fin};
    }
    static variable_list backward(AutogradContext* ctx, variable_list up) {
        variable_list grads(4);
        const variable_list saved = ctx->get_saved_variables();
        const ScanHeld& h = held<ScanHeld>(ctx);
        const at::Tensor &x = saved[0], &gate = saved[1];
        check_capture("race_gated_scan backward", {x, gate});
        if (up[0].defined() || up[1].defined()) {
            const auto need = needed(ctx, {true, true, ctx->saved_data["state"].toBool()});
            const auto dout = dense_grad(up[0].defined() ? up[0] : at::zeros(x.sizes(), x.options()), x.scalar_type());
            const auto [a, b, c] = gated_scan_backward(x, gate, if_defined(saved[2]), *dout, dense_grad(up[1], at::kFloat),
                                                       saved[3], h.form, h.complement, need[0], need[1], need[2]);
            grads = {or_undefined(a), or_undefined(b), or_undefined(c), at::Tensor()};
        }
        return differentiated_once("race_gated_scan", up, std::move(grads));
    }
};

struct CrossNode : torch::autograd::Function<CrossNode> {
    static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                 const c10::intrusive_ptr<CrossHeld>& h) {
        const auto [out, state] = cross_forward(q, k, v, h->lengths, true);
        ctx->save_for_backward({q, k, v, or_undefined(h->lengths), *state});
        return {*out};
    }
    static variable_list backward(AutogradContext* ctx, variable_list up) {
        const variable_list saved = ctx->get_saved_variables();
        check_capture("race_cross_fwd backward", {saved[0], saved[1], saved[2]});
        const auto need = needed(ctx, {true, true, true});
        const auto dout = dense_grad(up[0], saved[2].scalar_type());
        const auto [a, b, c] = cross_backward(saved[0], saved[1], saved[2], if_defined(saved[3]), *dout, saved[4], need[0],
                                              need[1], need[2]);
        return differentiated_once("race_cross_fwd", up, {or_undefined(a), or_undefined(b), or_undefined(c), at::Tensor()});
    }
};

std::tuple<at::Tensor, c10::optional<at::Tensor>> norm_rope(
    const at::Tensor& q_in, const c10::optional<at::Tensor>& k_in, const c10::optional<at::Tensor>& positions,
    const c10::optional<at::Tensor>& inv_freq, const c10::optional<at::Tensor>& q_weight,
    const c10::optional<at::Tensor>& k_weight, c10::optional<double> eps, const std::vector<int64_t>& sections,
    bool interleaved) {
    const bool node = wants_grad({q_in, k_in, q_weight, k_weight});
    if (node) check_capture("race_norm_rope", {q_in, k_in, q_weight, k_weight});
    const at::Tensor q = as_rows(q_in);
    c10::optional<at::Tensor> k;
    if (k_in) k = as_rows(*k_in);
    if (!node)
        return norm_rope_forward(q, k, positions, inv_freq, q_weight, k_weight, eps.value_or(0.0), eps.has_value(),
                                 sections, interleaved);
    auto h = c10::make_intrusive<RopeHeld>();
    h->positions = positions, h->inv_freq = inv_freq;
    h->eps = eps.value_or(0.0), h->norm = eps.has_value();
    h->sections = sections, h->interleaved = interleaved;
    const variable_list outs = NormRopeNode::apply(q, k, q_weight, k_weight, h);
    return {outs[0], outs.size() > 1 ? c10::optional<at::Tensor>(outs[1]) : c10::nullopt};
}

std::tuple<at::Tensor, at::Tensor> gated_scan(const at::Tensor& x_in, const at::Tensor& gate_in,
                                              const c10::optional<at::Tensor>& state,
                                              const c10::optional<at::Tensor>& lengths_in, int64_t form, bool complement) {
    const bool node = wants_grad({x_in, gate_in, state});
    if (node) check_capture("race_gated_scan", {x_in, gate_in, state});
    const at::Tensor x = as_rows(x_in, RACE_SCAN_MAX_TOKEN_STRIDE), gate = as_rows(gate_in, RACE_SCAN_MAX_TOKEN_STRIDE);
    const auto lengths = as_lengths(lengths_in);
    if (!node) {
        const auto r = gated_scan_forward(x, gate, state, lengths, form, complement, false, false);
        return {std::get<0>(r), std::get<1>(r)};
    }
    auto h = c10::make_intrusive<ScanHeld>();
    h->lengths = lengths, h->form = form, h->complement = complement;
    const variable_list outs = GatedScanNode::apply(x, gate, state, h);
    return {outs[0], outs[1]};
}

std::tuple<at::Tensor, at::Tensor> gated_scan_carry(const at::Tensor& x, const at::Tensor& gate, const at::Tensor& state,
                                                    const c10::optional<at::Tensor>& lengths, int64_t form,
                                                    bool complement, bool inplace) {
    const auto r = gated_scan_forward(as_rows(x, RACE_SCAN_MAX_TOKEN_STRIDE), as_rows(gate, RACE_SCAN_MAX_TOKEN_STRIDE),
                                      state, as_lengths(lengths), form, complement, false, inplace);
    return {std::get<0>(r), std::get<1>(r)};
}

at::Tensor cross(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const c10::optional<at::Tensor>& lengths) {
    if (!wants_grad({q, k, v})) return *std::get<0>(cross_forward(q, k, v, as_lengths(lengths), false));
    check_capture("race_cross_fwd", {q, k, v});
    auto h = c10::make_intrusive<CrossHeld>();
    h->lengths = as_lengths(lengths);
    return CrossNode::apply(q, k, v, h)[0];
}

at::Tensor cross_state(const at::Tensor& k, const at::Tensor& v, const c10::optional<at::Tensor>& lengths) {
    return *std::get<1>(cross_forward(c10::nullopt, k, v, as_lengths(lengths), true));
}

void bind_operators(pybind11::module& m) {
    namespace py = pybind11;
    m.def("norm_rope", &norm_rope, "race_norm_rope with its gradients -> (q, k or None)", py::arg("q"), py::arg("k"),
          py::arg("positions"), py::arg("inv_freq"), py::arg("q_weight"), py::arg("k_weight"), py::arg("eps"),
          py::arg("sections"), py::arg("interleaved"));
    m.def("gated_scan", &gated_scan, "race_gated_scan with its gradients -> (out, final state)", py::arg("x"),
          py::arg("gate"), py::arg("state"), py::arg("lengths"), py::arg("form"), py::arg("complement"));
    m.def("gated_scan_carry", &gated_scan_carry, "race_gated_scan from a carried state -> (out, state)", py::arg("x"),
          py::arg("gate"), py::arg("state"), py::arg("lengths"), py::arg("form"), py::arg("complement"),
          py::arg("inplace"));
    m.def("cross", &cross, "race_cross_fwd with its gradients -> out", py::arg("probsQ"), py::arg("probsK"), py::arg("V"),
          py::arg("lengths"));
    m.def("cross_state", &cross_state, "The sums race_cross_query reads", py::arg("probsK"), py::arg("V"),
          py::arg("lengths"));
    m.def("cross_query", &cross_query, "Queries against a kept state -> out", py::arg("probsQ"), py::arg("state"));
}

}  // namespace
