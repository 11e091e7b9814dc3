// fused_gemm_a16w16_epilogue_tk (extension) -- the bf16 GEMM with bias, activation
// and residual in its epilogue: dispatch(A, B, C, bias, residual, act, alpha).
#include "gemm_bind.h"

using namespace hkqbind;

void dispatch(py::object A, py::object B, py::object C, py::object bias, py::object residual, const std::string& act,
              float alpha) {
    gemm_epilogue(false, A, B, py::none(), py::none(), C, bias, residual, act, alpha, "fused_gemm_a16w16_epilogue");
}

PYBIND11_MODULE(fused_gemm_a16w16_epilogue_tk, m) {
    m.doc() = "bf16 GEMM with bias, activation and residual (gfx950 MFMA)";
    m.def("dispatch", &dispatch, "C = act(A . B^T + bias) + residual", py::arg("A"), py::arg("B"), py::arg("C"),
          py::arg("bias") = py::none(), py::arg("residual") = py::none(), py::arg("act") = "none", py::arg("alpha") = 1.0f);
}
