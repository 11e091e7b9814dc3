// gated_ffn_tk (extension) -- the gated projection pair of a feed-forward layer
// in one kernel, FP8 and bf16, and the gradients of the bf16 form. W [2F, K]:
// gate and up rows as halves or interleaved; activations by name.
#include "bind_common.h"

using namespace hkqbind;

namespace {

// A bf16 [rows, cols] operand; its pitch to *ld.
TensorView matrix(py::object t, const char* name, int64_t rows, int64_t cols, int64_t* ld) {
    auto v = view(t, name);
    expect_dtype(v, name, {kBF16});
    *ld = row_stride(v, name);
    expect(v.dim(0) == rows && v.dim(1) == cols,
           std::string(name) + " must be [" + std::to_string(rows) + ", " + std::to_string(cols) + "]");
    return v;
}

}  // namespace

void gated_ffn_a8w8(py::object X, py::object W, py::object x_scale, py::object w_scale, py::object H,
                    const std::string& act, float alpha, bool interleaved) {
    const OnDevice on({X, W, x_scale, w_scale, H});
    auto x = view(X, "X"), w = view(W, "W"), sx = view(x_scale, "x_scale"), sw = view(w_scale, "w_scale");
    expect_dtype(x, "X", {kFP8, kU8});
    expect_dtype(w, "W", {kFP8, kU8});
    expect_dtype(sx, "x_scale", {kF32});
    expect_dtype(sw, "w_scale", {kF32});
    const int64_t ldx = row_stride(x, "X"), ldw = row_stride(w, "W");
    const int64_t M = x.dim(0), K = x.dim(1), F = w.dim(0) / 2;
    expect(w.dim(0) % 2 == 0 && w.dim(1) == K, "W must be [2F, K]");
    expect(sx.numel() == M && sx.contiguous(), "x_scale must be contiguous with M elements");
    expect(sw.numel() == 2 * F && sw.contiguous(), "w_scale must be contiguous with 2F elements");
    int64_t ldh;
    auto h = matrix(H, "H", M, F, &ldh);
    check(hkq_gated_ffn_a8w8((const void*)x.ptr, (const void*)w.ptr, (const float*)sx.ptr, (const float*)sw.ptr,
                             (void*)h.ptr, M, F, K, ldx, ldw, ldh, activation(act), alpha, interleaved ? 1 : 0,
                             current_stream()),
          "gated_ffn_a8w8");
}

void gated_ffn_bf16(py::object X, py::object W, py::object H, py::object Y, const std::string& act, float alpha,
                    bool interleaved) {
    const OnDevice on({X, W, H, Y});
    auto x = view(X, "X"), w = view(W, "W");
    expect_dtype(x, "X", {kBF16});
    expect_dtype(w, "W", {kBF16});
    const int64_t ldx = row_stride(x, "X"), ldw = row_stride(w, "W");
    const int64_t M = x.dim(0), K = x.dim(1), F = w.dim(0) / 2;
    expect(w.dim(0) % 2 == 0 && w.dim(1) == K, "W must be [2F, K]");
    int64_t ldh, ldy = 0;
    auto h = matrix(H, "H", M, F, &ldh);
    void* py_ = nullptr;
    if (!Y.is_none()) py_ = (void*)matrix(Y, "Y", M, 2 * F, &ldy).ptr;
    check(hkq_gated_ffn_bf16((const void*)x.ptr, (const void*)w.ptr, (void*)h.ptr, py_, M, F, K, ldx, ldw, ldh, ldy,
                             activation(act), alpha, interleaved ? 1 : 0, current_stream()),
          "gated_ffn_bf16");
}

void gated_ffn_backward(py::object dH, py::object X, py::object W, py::object Y, py::object dX, py::object dW,
                        const std::string& act, float alpha, bool interleaved) {
    const OnDevice on({dH, X, W, Y, dX, dW});
    auto x = view(X, "X"), w = view(W, "W");
    expect_dtype(x, "X", {kBF16});
    expect_dtype(w, "W", {kBF16});
    const int64_t ldx = row_stride(x, "X"), ldw = row_stride(w, "W");
    const int64_t M = x.dim(0), K = x.dim(1), F = w.dim(0) / 2;
    expect(w.dim(0) % 2 == 0 && w.dim(1) == K, "W must be [2F, K]");
    int64_t lddh, ldy, lddx = 0, lddw = 0;
    auto dh = matrix(dH, "dH", M, F, &lddh), y = matrix(Y, "Y", M, 2 * F, &ldy);
    void *pdx = nullptr, *pdw = nullptr;
    if (!dX.is_none()) pdx = (void*)matrix(dX, "dX", M, K, &lddx).ptr;
    if (!dW.is_none()) pdw = (void*)matrix(dW, "dW", 2 * F, K, &lddw).ptr;
    const int id = activation(act);
    Workspace ws = workspace(pdx || pdw ? hkq_gated_ffn_backward_workspace(M, F, K) : 0, X);
    check(hkq_gated_ffn_backward((const void*)dh.ptr, (const void*)x.ptr, (const void*)w.ptr, (const void*)y.ptr, pdx, pdw,
                                 M, F, K, lddh, ldx, ldw, ldy, lddx, lddw, id, alpha, interleaved ? 1 : 0, ws.ptr, ws.bytes,
                                 current_stream()),
          "gated_ffn_backward");
}

PYBIND11_MODULE(gated_ffn_tk, m) {
    m.doc() = "Gated feed-forward projections, FP8 and bf16, and their backward pass (gfx950 MFMA)";
    m.def("gated_ffn_a8w8", &gated_ffn_a8w8, "H = act(X . Wg^T) * (X . Wu^T), E4M3FN codes and scales", py::arg("X"),
          py::arg("W"), py::arg("x_scale"), py::arg("w_scale"), py::arg("H"), py::arg("act") = "silu",
          py::arg("alpha") = 1.0f, py::arg("interleaved") = false);
    m.def("gated_ffn_bf16", &gated_ffn_bf16, "H = act(X . Wg^T) * (X . Wu^T); Y keeps both projections", py::arg("X"),
          py::arg("W"), py::arg("H"), py::arg("Y") = py::none(), py::arg("act") = "silu", py::arg("alpha") = 1.0f,
          py::arg("interleaved") = false);
    m.def("gated_ffn_backward", &gated_ffn_backward, "Gradients dX, dW of gated_ffn_bf16 from dH and the kept Y",
          py::arg("dH"), py::arg("X"), py::arg("W"), py::arg("Y"), py::arg("dX") = py::none(), py::arg("dW") = py::none(),
          py::arg("act") = "silu", py::arg("alpha") = 1.0f, py::arg("interleaved") = false);
}
