// fused_gemm_a8w8_epilogue_tk (extension) -- the A8W8 GEMM with bias, activation
// and residual in its epilogue: dispatch(A, B, a_scale, b_scale, C, bias,
// residual, act, alpha).
#include "gemm_bind.h"

using namespace hkqbind;

void dispatch(py::object A, py::object B, py::object a_scale, py::object b_scale, py::object C, py::object bias,
              py::object residual, const std::string& act, float alpha) {
    gemm_epilogue(true, A, B, a_scale, b_scale, C, bias, residual, act, alpha, "fused_gemm_a8w8_epilogue");
}

PYBIND11_MODULE(fused_gemm_a8w8_epilogue_tk, m) {
    m.doc() = "A8W8 GEMM with bias, activation and residual (gfx950 FP8 MFMA)";
    m.def("dispatch", &dispatch, "C = act((A . B^T) * a_scale * b_scale + bias) + residual", py::arg("A"), py::arg("B"),
          py::arg("a_scale"), py::arg("b_scale"), py::arg("C"), py::arg("bias") = py::none(),
          py::arg("residual") = py::none(), py::arg("act") = "none", py::arg("alpha") = 1.0f);
}
