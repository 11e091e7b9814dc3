// w4_tk (extension) -- 4-bit weights: quantizer, and products of bf16 rows with INT4
// (group scales, zero points) or MXFP4 weights, dense and over ragged groups of rows.
#include "group_bind.h"

using namespace hkqbind;

namespace {

struct Rows {
    void* ptr;
    int64_t n, cols, ld;
};
Rows rows(py::object t, const char* name, const char* dtype) {
    auto v = view(t, name);
    expect_dtype(v, name, {dtype});
    expect(v.shape.size() == 2, std::string(name) + " must be 2-D");
    const Groups g = groups(v, name);
    return Rows{(void*)v.ptr, g.N, g.cols, g.ld};
}

}  // namespace

void w4_quant(py::object w, py::object q, py::object s, py::object z) {
    const OnDevice on({w, q, s, z});
    const Rows a = rows(w, "w", kBF16), c = rows(q, "q", kU8), sc = rows(s, "s", kBF16);
    expect(c.n == a.n && c.cols * 2 == a.cols, "q must be [N, K / 2]");
    expect(sc.n == a.n && sc.cols > 0 && a.cols % sc.cols == 0, "s must be [N, K / group]");
    void* zp = nullptr;
    if (!z.is_none()) {
        const Rows v = rows(z, "z", kU8);
        expect(v.n == sc.n && v.cols == sc.cols && v.ld == sc.ld, "z must have the shape and pitch of s");
        zp = v.ptr;
    }
    check(hkq_w4_quant(a.ptr, c.ptr, sc.ptr, zp, a.n, a.cols, a.ld, c.ld, sc.ld, a.cols / sc.cols, current_stream()), "w4_quant");
}

void w4_dequant(py::object q, py::object s, py::object out, py::object z) {
    const OnDevice on({q, s, out, z});
    const W4 w = w4_weights(q, s, z, false);
    if (w.kind != HKQ_W4_INT4) throw py::type_error("s must be bf16 (MXFP4: upcast_from_mxfp)");
    const Rows o = rows(out, "out", kBF16);
    expect(o.n == w.q.N && o.cols == w.K, "out must be [N, K]");
    check(hkq_w4_dequant(w.codes, w.scales, w.zeros, o.ptr, o.n, o.cols, w.q.ld, w.s.ld, o.ld, w.group, current_stream()),
          "w4_dequant");
}

void gemm_w4a16(py::object X, py::object Q, py::object S, py::object C, py::object Z) {
    const OnDevice on({X, Q, S, C, Z});
    const W4 w = w4_weights(Q, S, Z, false);
    const Rows x = rows(X, "X", kBF16), c = rows(C, "C", kBF16);
    expect(x.cols == w.K, "X and the weights must have the same K");
    expect(c.n == x.n && c.cols == w.q.N, "C must be [M, N]");
    const Workspace ws = workspace(hkq_gemm_w4a16_workspace(x.n, w.q.N, w.K), X);
    check(hkq_gemm_w4a16(x.ptr, w.codes, w.scales, w.zeros, c.ptr, x.n, w.q.N, w.K, x.ld, w.q.ld, w.s.ld, c.ld, w.group, w.kind,
                         ws.ptr, ws.bytes, current_stream()),
          "gemm_w4a16");
}

void grouped_gemm_w4a16(py::object X, py::object Q, py::object S, py::object Y, py::object offs, py::object Z, py::object gather,
                        int64_t topk) {
    const OnDevice on({X, Q, S, Y, offs, Z, gather});
    const W4 w = w4_weights(Q, S, Z, true);
    const Rows x = rows(X, "X", kBF16), y = rows(Y, "Y", kBF16);
    expect(x.cols == w.K, "X and the weights must have the same K");
    const int32_t* g = nullptr;
    if (!gather.is_none()) {
        auto v = view(gather, "gather");
        expect_dtype(v, "gather", {kI32});
        expect(v.shape.size() == 1 && v.dim(0) == y.n && v.contiguous(), "gather must be contiguous with an element per row of Y");
        g = (const int32_t*)v.ptr;
    }
    expect(y.cols == w.q.N && (g || y.n == x.n), "Y must be [M, N]");
    const Workspace ws = workspace(hkq_grouped_gemm_w4a16_workspace(y.n, w.q.E, w.q.N, w.K), X);
    check(hkq_grouped_gemm_w4a16(x.ptr, w.codes, w.scales, w.zeros, y.ptr, bounds(offs, w.q.E), g, y.n, x.n, w.q.E, w.q.N, w.K, topk,
                                 x.ld, w.q.ld, w.q.stride, w.s.ld, w.s.stride, y.ld, w.group, w.kind, ws.ptr, ws.bytes,
                                 current_stream()),
          "grouped_gemm_w4a16");
}

PYBIND11_MODULE(w4_tk, m) {
    m.doc() = "4-bit weights (INT4 with group scales, MXFP4): quantizer, products with bf16 rows (gfx950 MFMA)";
    m.def("w4_quant", &w4_quant, "INT4 codes and scales (and zero points) of bf16 weights", py::arg("w"), py::arg("q"),
          py::arg("s"), py::arg("z") = py::none());
    m.def("w4_dequant", &w4_dequant, "bf16((code - zero) * scale)", py::arg("q"), py::arg("s"), py::arg("out"),
          py::arg("z") = py::none());
    m.def("gemm_w4a16", &gemm_w4a16, "C = X . W^T with 4-bit weights", py::arg("X"), py::arg("Q"), py::arg("S"), py::arg("C"),
          py::arg("Z") = py::none());
    m.def("grouped_gemm_w4a16", &grouped_gemm_w4a16, "Y[r] = X[x(r)] . W[e]^T with 4-bit weights, offs[e] <= r < offs[e + 1]",
          py::arg("X"), py::arg("Q"), py::arg("S"), py::arg("Y"), py::arg("offs"), py::arg("Z") = py::none(),
          py::arg("gather") = py::none(), py::arg("topk") = 1);
}
