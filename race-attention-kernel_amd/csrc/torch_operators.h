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
        .require(t.dim() == dim, name, "has shape " + dims(t) + ", not " + layout)
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
                 "has " + std::to_string(l.numel()) + " entries, which do not divide the " + std::to_string(streams) +
                     " streams");
    return l.dim() == 1 && l.numel() > 0 && streams >= l.numel() ? streams / l.numel() : 1;
}

// ---- gated linear recurrence ----

race_scan_shape scan_shape(const char* entry, const at::Tensor& x, const at::Tensor& gate,
                           const c10::optional<at::Tensor>& state, const c10::optional<at::Tensor>& lengths,
                           int64_t form, bool complement) {
    ArgCheck c(entry);
    check_rows(c, "x", x, 3, "[N, T, D]");
    check_rows(c, "gate", gate, 3, "[N, T, D]");
    c.matches("gate", gate, "x", x)
        .require(gate.sizes() == x.sizes(), "gate", "has shape " + dims(gate) + ", x " + dims(x));
    c.raise();
    const int64_t N = x.size(0), D = x.size(2);
    if (state)
        c.on_gpu("state", *state)
            .require(state->scalar_type() == at::kFloat && state->device() == x.device(), "state",
                     "must be float32 on x's device")
            .require(state->sizes() == at::IntArrayRef({N, D}), "state", "has shape " + dims(*state) + ", not [N, D]");
    const int64_t group = check_lengths(c, lengths, x, N);
    c.require(N <= 65535 && D >= 1 && D <= 65536, "x",
              "has shape " + dims(x) + "; the scan takes up to 65535 streams of 1 .. 65536 channels")
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
    TORCH_CHECK(!inplace || state, "race_gated_scan: an in-place call needs a state");
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
        .require(dout.sizes() == x.sizes(), "dout", "has shape " + dims(dout) + ", x " + dims(x))
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

void bind_operators(pybind11::module& m) {
    namespace py = pybind11;
    m.def("gated_scan_forward", &gated_scan_forward,
          "h_t = a_t h_{t-1} + u_t -> (out, final state, records or None)", py::arg("x"), py::arg("gate"),
          py::arg("state"), py::arg("lengths"), py::arg("form"), py::arg("complement"), py::arg("want_records"),
          py::arg("inplace"));
    m.def("gated_scan_backward", &gated_scan_backward, "Gradients of gated_scan_forward -> (dx, dgate, dstate)",
          py::arg("x"), py::arg("gate"), py::arg("lengths"), py::arg("dout"), py::arg("dfinal"), py::arg("records"),
          py::arg("form"), py::arg("complement"), py::arg("need_x"), py::arg("need_gate"), py::arg("need_state"));
}

}  // namespace
