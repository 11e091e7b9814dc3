// group_bind.h -- argument handling of the products over ragged groups of rows and of
// the 4-bit weights: [E, N, ..] operands, bounds, kinds.
#pragma once
#include "bind_common.h"

namespace hkqbind {

// Rows of an operand [N, ..] or groups of rows [E, N, ..], last dimension contiguous.
// What is not stepped over counts as contiguous.
struct Groups {
    int64_t E, N, cols, stride, ld;
};
inline Groups groups(const TensorView& v, const char* name) {
    const size_t nd = v.shape.size();
    expect(nd == 2 || nd == 3, std::string(name) + " must be 2-D or 3-D");
    Groups g{nd == 3 ? v.shape[0] : 1, v.dim(-2), v.dim(-1), 0, v.stride[nd - 2]};
    expect(v.stride[nd - 1] == 1 || g.cols <= 1, std::string(name) + " must have a contiguous last dimension");
    if (g.N <= 1 || v.numel() == 0) g.ld = g.cols;
    g.stride = nd == 3 && g.E > 1 && v.numel() > 0 ? v.stride[0] : g.N * g.ld;
    return g;
}
inline void expect_groups(const Groups& g, const char* name, int64_t E, int64_t N, int64_t cols) {
    expect(g.E == E && g.N == N && g.cols == cols, std::string(name) + " must be [" + (E > 1 ? std::to_string(E) + ", " : "") +
                                                       std::to_string(N) + ", " + std::to_string(cols) + "]");
}
inline const int32_t* bounds(const py::object& t, int64_t E) {
    auto v = view(t, "offs");
    expect_dtype(v, "offs", {kI32});
    expect(v.shape.size() == 1 && v.dim(0) == E + 1 && v.contiguous(), "offs must be contiguous with E + 1 elements");
    return (const int32_t*)v.ptr;
}

// 4-bit weights: codes, scales and (or None) zero points of one shape.
struct W4 {
    Groups q, s;
    const void *codes, *scales, *zeros = nullptr;
    int kind;
    int64_t K, group;
};
inline W4 w4_weights(py::object Q, py::object S, py::object Z, bool grouped) {
    auto q = view(Q, "Q"), s = view(S, "S");
    expect_dtype(q, "Q", {kU8});
    expect_dtype(s, "S", {kBF16, kU8});
    expect((q.shape.size() == 3) == grouped, std::string("Q must be ") + (grouped ? "[E, N, K / 2]" : "[N, K / 2]"));
    W4 w{groups(q, "Q"), groups(s, "S"), (const void*)q.ptr, (const void*)s.ptr};
    w.K = 2 * w.q.cols;
    w.kind = s.dtype == kU8 ? HKQ_W4_MXFP4 : HKQ_W4_INT4;
    w.group = w.kind == HKQ_W4_MXFP4 || w.K == 0 ? 32 : w.s.cols > 0 ? w.K / w.s.cols : 0;
    expect((w.group == 32 || w.group == 64 || w.group == 128) && w.s.cols * w.group == w.K,
           "S must hold a scale per 32, 64 or 128 values of K (MXFP4: 32)");
    expect(s.shape.size() == q.shape.size(), "Q and S must have the same dimensions");
    expect_groups(w.s, "S", w.q.E, w.q.N, w.K / w.group);
    if (!Z.is_none()) {
        expect(w.kind == HKQ_W4_INT4, "MXFP4 weights have no zero points");
        auto z = view(Z, "Z");
        expect_dtype(z, "Z", {kU8});
        const Groups g = groups(z, "Z");
        expect(z.shape.size() == q.shape.size(), "Q and Z must have the same dimensions");
        expect_groups(g, "Z", w.q.E, w.q.N, w.K / w.group);
        expect(g.ld == w.s.ld && (w.q.E <= 1 || g.stride == w.s.stride), "S and Z must have the same strides");
        w.zeros = (const void*)z.ptr;
    }
    return w;
}

}  // namespace hkqbind
