// fused_fp8_quant_tk -- the reference module of kernels/quantization/fused_fp8_quant/kernel.cpp:251-275:
// fused_rmsnorm_fp8_quant_fwd(input, weight, output, scales, eps). input bf16
// [M, D]; weight bf16 [D]; output [M, D] E4M3FN codes (float8_e4m3fn or
// uint8); scales fp32 [M, D/128]. D any multiple of 128 up to 8192 (the
// reference: 4096 or 8192). fused_add_rmsnorm_quant_fwd (extension): the same
// behind a residual addition, FP8 or INT8, per token or per 128 columns.
#include "bind_common.h"

using namespace hkqbind;

void fused_rmsnorm_fp8_quant_fwd(py::object input, py::object weight, py::object output, py::object scales,
                                 float eps) {
    auto x = view(input, "input"), w = view(weight, "weight"), q = view(output, "output"), s = view(scales, "scales");
    expect_dtype(x, "input", {kBF16});
    expect_dtype(w, "weight", {kBF16});
    expect_dtype(q, "output", {kFP8, kU8});
    expect_dtype(s, "scales", {kF32});
    const int64_t ldx = row_stride(x, "input"), ldq = row_stride(q, "output");
    const int64_t M = x.dim(0), D = x.dim(1);
    expect(D % 128 == 0 && D <= 8192, "D must be a multiple of 128, at most 8192");
    expect(w.numel() == D && w.contiguous(), "weight must be a contiguous [D] tensor");
    expect(q.dim(0) == M && q.dim(1) == D, "output must be [M, D]");
    expect(s.shape.size() == 2 && s.dim(0) == M && s.dim(1) == D / 128, "scales must be [M, D/128]");
    const int64_t lds = row_stride(s, "scales");
    check(hkq_rmsnorm_quant((const void*)x.ptr, (const void*)w.ptr, (void*)q.ptr, (void*)s.ptr, M, D, ldx, ldq, lds,
                            eps, 0, current_stream()),
          "fused_rmsnorm_fp8_quant_fwd");
}

// input, residual, hidden bf16 [M, D] (residual and hidden both None: no
// addition); weight bf16 [D]; output [M, D] E4M3FN codes or int8; scales fp32
// [M] / [M, 1] (group_size 0: per token) or [M, D/128] (128). hidden =
// bf16(input + residual); it may be either of them.
void fused_add_rmsnorm_quant_fwd(py::object input, py::object residual, py::object weight, py::object hidden,
                                 py::object output, py::object scales, float eps, int64_t group_size) {
    const OnDevice on({input, residual, weight, hidden, output, scales});
    auto x = view(input, "input"), w = view(weight, "weight"), q = view(output, "output"), s = view(scales, "scales");
    expect_dtype(x, "input", {kBF16});
    expect_dtype(w, "weight", {kBF16});
    expect_dtype(q, "output", {kI8, kFP8, kU8});
    expect_dtype(s, "scales", {kF32});
    const int64_t ldx = row_stride(x, "input"), ldq = row_stride(q, "output");
    const int64_t M = x.dim(0), D = x.dim(1);
    expect(group_size == 0 || group_size == 128, "group_size must be 0 (per token) or 128");
    expect(w.numel() == D && w.contiguous(), "weight must be a contiguous [D] tensor");
    expect(q.dim(0) == M && q.dim(1) == D, "output must be [M, D]");
    int64_t lds = 1, ldr = 0, ldh = 0;
    if (group_size == 0) {
        expect(s.numel() == M && s.contiguous(), "scales must be a contiguous [M] or [M, 1] tensor");
    } else {
        expect(s.shape.size() == 2 && s.dim(0) == M && s.dim(1) * 128 == D, "scales must be [M, D/128]");
        lds = row_stride(s, "scales");
    }
    expect(residual.is_none() == hidden.is_none(), "residual and hidden go together: both or neither");
    const void *res = nullptr;
    void* h = nullptr;
    if (!residual.is_none()) {
        auto r = view(residual, "residual"), o = view(hidden, "hidden");
        expect_dtype(r, "residual", {kBF16});
        expect_dtype(o, "hidden", {kBF16});
        ldr = row_stride(r, "residual");
        ldh = row_stride(o, "hidden");
        expect(r.dim(0) == M && r.dim(1) == D, "residual must be [M, D]");
        expect(o.dim(0) == M && o.dim(1) == D, "hidden must be [M, D]");
        res = (const void*)r.ptr;
        h = (void*)o.ptr;
    }
    check(hkq_add_rmsnorm_quant((const void*)x.ptr, res, (const void*)w.ptr, h, (void*)q.ptr, (float*)s.ptr, M, D, ldx,
                                ldr, ldh, ldq, lds, eps, (int)group_size, q.dtype == kI8 ? HKQ_KIND_INT8 : HKQ_KIND_FP8,
                                current_stream()),
          "fused_add_rmsnorm_quant_fwd");
}

PYBIND11_MODULE(fused_fp8_quant_tk, m) {
    m.doc() = "Fused RMSNorm + 1x128 FP8 (E4M3FN) quantization (gfx950)";
    m.def("fused_rmsnorm_fp8_quant_fwd", &fused_rmsnorm_fp8_quant_fwd, "Fused RMSNorm + FP8 quantization forward pass",
          py::arg("input"), py::arg("weight"), py::arg("output"), py::arg("scales"), py::arg("eps"));
    m.def("fused_add_rmsnorm_quant_fwd", &fused_add_rmsnorm_quant_fwd,
          "Residual addition + RMSNorm + FP8 / INT8 quantization forward pass", py::arg("input"), py::arg("residual"),
          py::arg("weight"), py::arg("hidden"), py::arg("output"), py::arg("scales"), py::arg("eps"),
          py::arg("group_size") = 0);
}
