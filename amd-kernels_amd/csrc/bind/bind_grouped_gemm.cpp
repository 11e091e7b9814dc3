// grouped_gemm_tk (extension) -- bf16 products over ragged groups of rows (the experts
// of a mixture) and their gradients.
#include "group_bind.h"

using namespace hkqbind;

namespace {

struct Rows {
    void* ptr = nullptr;
    int64_t ld = 0;
};
Rows rows(py::object t, const char* name, int64_t n, int64_t cols) {
    auto v = view(t, name);
    expect_dtype(v, name, {kBF16});
    expect(v.shape.size() == 2, std::string(name) + " must be 2-D");
    const Groups g = groups(v, name);
    expect_groups(g, name, 1, n, cols);
    return Rows{(void*)v.ptr, g.ld};
}

}  // namespace

void grouped_gemm_bf16(py::object X, py::object W, py::object Y, py::object offs) {
    const OnDevice on({X, W, Y, offs});
    auto w = view(W, "W");
    expect_dtype(w, "W", {kBF16});
    expect(w.shape.size() == 3, "W must be [E, N, K]");
    const Groups g = groups(w, "W");
    const int64_t M = view(X, "X").dim(0);
    const Rows x = rows(X, "X", M, g.cols), y = rows(Y, "Y", M, g.N);
    check(hkq_grouped_gemm_bf16(x.ptr, (const void*)w.ptr, y.ptr, bounds(offs, g.E), M, g.E, g.N, g.cols, x.ld, g.ld, g.stride,
                                y.ld, current_stream()),
          "grouped_gemm_bf16");
}

void grouped_gemm_backward(py::object dY, py::object X, py::object W, py::object offs, py::object dX, py::object dW) {
    const OnDevice on({dY, X, W, offs, dX, dW});
    auto w = view(W, "W");
    expect_dtype(w, "W", {kBF16});
    expect(w.shape.size() == 3, "W must be [E, N, K]");
    const Groups g = groups(w, "W");
    const int64_t M = view(X, "X").dim(0);
    const Rows x = rows(X, "X", M, g.cols), dy = rows(dY, "dY", M, g.N);
    Rows dx;
    if (!dX.is_none()) dx = rows(dX, "dX", M, g.cols);
    Groups d{};
    void* dw = nullptr;
    if (!dW.is_none()) {
        auto v = view(dW, "dW");
        expect_dtype(v, "dW", {kBF16});
        expect(v.shape.size() == 3, "dW must be [E, N, K]");
        d = groups(v, "dW");
        expect_groups(d, "dW", g.E, g.N, g.cols);
        dw = (void*)v.ptr;
    }
    check(hkq_grouped_gemm_backward(dy.ptr, x.ptr, (const void*)w.ptr, dx.ptr, dw, bounds(offs, g.E), M, g.E, g.N, g.cols, dy.ld,
                                    x.ld, g.ld, g.stride, dx.ld, d.ld, d.stride, current_stream()),
          "grouped_gemm_backward");
}

PYBIND11_MODULE(grouped_gemm_tk, m) {
    m.doc() = "bf16 products over ragged groups of rows, and their gradients (gfx950 MFMA)";
    m.def("grouped_gemm_bf16", &grouped_gemm_bf16, "Y[r] = X[r] . W[e]^T for offs[e] <= r < offs[e + 1]", py::arg("X"),
          py::arg("W"), py::arg("Y"), py::arg("offs"));
    m.def("grouped_gemm_backward", &grouped_gemm_backward, "Gradients dX, dW of grouped_gemm_bf16 from dY", py::arg("dY"),
          py::arg("X"), py::arg("W"), py::arg("offs"), py::arg("dX") = py::none(), py::arg("dW") = py::none());
}
