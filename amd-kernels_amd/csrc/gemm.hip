// gemm.hip -- dense scaled GEMMs on CDNA4 matrix cores.
//
//   hkq_gemm_a8w8        C = bf16((A . B^T) * sa[m] * sb[n]), A/B E4M3FN codes
//                        (gemm-basic/gemm_a8w8/kernel.cpp:46-160 and
//                        gemm_a8w8_per_token_scale/kernel.cpp:49-156; formula
//                        tests/test_gemm.py:116);
//   hkq_gemm_mxfp4       C = bf16(sum_k e2m1(a) 2^(sa-127) e2m1(b) 2^(sb-127)),
//                        e8m0 scales per 32 K-values fed to the MFMA scale
//                        operands (gemm-basic/gemm_afp4wfp4/kernel.cpp:1-12 for
//                        the data format; the reference kernel itself consumes
//                        pre-dequantized bf16);
//   hkq_gemm_bf16,       C = bf16(A . B^T (+ bias[n])), bf16 operands
//   hkq_batched_gemm_*   (gemm_a16w16, formula tests/test_gemm.py:21-42),
//                        batched over grid.y (gemm-batched/batched_gemm_a8w8/
//                        kernel.cpp:59-203, batched_gemm_bf16/kernel.cpp:53-187;
//                        formulas tests/test_gemm.py:316-390).
#include <mutex>

#include "gemm_dense.h"

using namespace hkq;

static int check_common(int64_t M, int64_t N, int64_t K, int64_t ldc, const void* C) {
    HKQ_CHECK_ARG(M >= 0 && N >= 0 && K > 0, "M, N must be >= 0 and K > 0");
    HKQ_CHECK_ARG(M < (1 << 30) && N < (1 << 30) && K < (1 << 30), "dimensions must be < 2^30");
    HKQ_CHECK_ARG(N % 4 == 0, "N must be a multiple of 4");
    HKQ_CHECK_ARG(ldc >= N && ldc % 4 == 0, "ldc must be >= N and a multiple of 4");
    HKQ_CHECK_ALIGN(C, 8);
    return 0;
}

// Shapes that the workspace queries answer with 0: M <= 16, and M <= 32 with
// fewer than two 16-column slices per CU and at most 32 K-steps of 128 values
// (`step` bytes each), whose rows hold whole K-steps.
static bool no_split(int64_t M, int64_t N, int64_t kbytes, int64_t step) {
    if (M > 32 || kbytes % step != 0 || 64 * kbytes >= (1ll << 31)) return false;
    const int64_t ncu = cu_count() > 0 ? cu_count() : 256;
    return M <= 16 || ((N + 15) / 16 < 2 * ncu && kbytes / step <= 32);
}

extern "C" {

size_t hkq_gemm_a8w8_workspace(int64_t M, int64_t N, int64_t K) {
    if (M <= 0 || N <= 0 || K <= 0 || K % 64 != 0 || no_split(M, N, K, 128)) return 0;
    return dense_plan(MODE_A8W8, M, N, K).ws_bytes;
}

int hkq_gemm_a8w8_ws(const void* A, const void* B, const float* sa, const float* sb, void* C, int64_t M, int64_t N,
                     int64_t K, int64_t lda, int64_t ldb, int64_t ldc, void* workspace, size_t workspace_bytes,
                     hipStream_t stream) {
    if (int e = check_common(M, N, K, ldc, C)) return e;
    HKQ_CHECK_ARG(K % 64 == 0, "K must be a multiple of 64");
    HKQ_CHECK_ARG(lda >= K && ldb >= K && lda % 16 == 0 && ldb % 16 == 0,
                  "lda/ldb must be >= K and multiples of 16");
    HKQ_CHECK_ALIGN(A, 16);
    HKQ_CHECK_ALIGN(B, 16);
    HKQ_CHECK_ALIGN(sb, 16);
    HKQ_CHECK_ALIGN(workspace, 16);
    DenseParams p{};
    p.A = static_cast<const uint8_t*>(A);
    p.B = static_cast<const uint8_t*>(B);
    p.C = static_cast<uint16_t*>(C);
    p.sa = sa;
    p.sb = sb;
    p.M = (int)M; p.N = (int)N; p.K = (int)K; p.kbytes = (int)K;
    p.lda = lda; p.ldb = ldb; p.ldc = ldc;
    return launch_dense<PlainOp, MODE_A8W8>(p, workspace, workspace_bytes, stream);
}

int hkq_gemm_a8w8(const void* A, const void* B, const float* sa, const float* sb, void* C, int64_t M, int64_t N,
                  int64_t K, int64_t lda, int64_t ldb, int64_t ldc, hipStream_t stream) {
    return hkq_gemm_a8w8_ws(A, B, sa, sb, C, M, N, K, lda, ldb, ldc, nullptr, 0, stream);
}

}  // extern "C"

// Split-K counters and partial sums of hkq_gemm_a8w8_noalloc: a library-owned
// workspace that each GPU holds from the library's load to the end of the
// process, so that the entry point allocates nothing. Its size bounds every
// split plan on 256 CUs (at most 1.5 * 256 tile splits of 128 x 128 fp32
// sums: 25.2 MB, after 4 KB of counters).
constexpr size_t HKQ_SCRATCH_BYTES = size_t(32) << 20;
static __device__ __align__(256) uint8_t scratch[HKQ_SCRATCH_BYTES];

// Device address of `scratch` on the current device, looked up once per device
// with that device current (the host-side name is only a stand-in for it).
static int scratch_address(void** out) {
    constexpr int MAXDEV = 64;
    static void* addr[MAXDEV] = {};
    static std::mutex mu;
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess || dev < 0 || dev >= MAXDEV) {
        set_error("hkq_gemm_a8w8_noalloc: no usable current device (%s)", hipGetErrorString(e));
        return e != hipSuccess ? (int)e : (int)hipErrorInvalidDevice;
    }
    std::lock_guard<std::mutex> lock(mu);
    if (!addr[dev]) {
        void* p = nullptr;
        e = hipGetSymbolAddress(&p, HIP_SYMBOL(scratch));
        if (e != hipSuccess || p == nullptr) {
            set_error("hkq_gemm_a8w8_noalloc: hipGetSymbolAddress(scratch) failed: %s", hipGetErrorString(e));
            return e != hipSuccess ? (int)e : (int)hipErrorInvalidSymbol;
        }
        addr[dev] = p;
    }
    *out = addr[dev];
    return 0;
}

extern "C" {

size_t hkq_gemm_a8w8_noalloc_max_workspace(void) { return HKQ_SCRATCH_BYTES; }

int hkq_gemm_a8w8_noalloc(const void* A, const void* B, const float* sa, const float* sb, void* C, int64_t M,
                          int64_t N, int64_t K, int64_t lda, int64_t ldb, int64_t ldc, hipStream_t stream) {
    // the same argument checks and plan as hkq_gemm_a8w8_ws, whose launches run
    // unchanged on the library's scratch workspace
    const size_t need = hkq_gemm_a8w8_workspace(M, N, K);
    if (need > HKQ_SCRATCH_BYTES) {
        set_error("hkq_gemm_a8w8_noalloc: the split plan of %lldx%lldx%lld needs %zu workspace bytes, more than the "
                  "%zu-byte library scratch; use hkq_gemm_a8w8_ws with a caller workspace",
                  (long long)M, (long long)N, (long long)K, need, HKQ_SCRATCH_BYTES);
        return (int)hipErrorInvalidValue;
    }
    void* ws = nullptr;
    if (need > 0)
        if (int e = scratch_address(&ws)) return e;
    return hkq_gemm_a8w8_ws(A, B, sa, sb, C, M, N, K, lda, ldb, ldc, ws, need, stream);
}

size_t hkq_gemm_mxfp4_workspace(int64_t M, int64_t N, int64_t K) {
    if (M <= 0 || N <= 0 || K <= 0 || K % 128 != 0 || no_split(M, N, K / 2, 64)) return 0;
    return dense_plan(MODE_MXFP4, M, N, K / 2).ws_bytes;
}

int hkq_gemm_mxfp4_ws(const void* A, const void* As, const void* B, const void* Bs, void* C, int64_t M, int64_t N,
                      int64_t K, int64_t lda, int64_t ldb, int64_t ldsa, int64_t ldsb, int64_t ldc, void* workspace,
                      size_t workspace_bytes, hipStream_t stream) {
    if (int e = check_common(M, N, K, ldc, C)) return e;
    HKQ_CHECK_ARG(K % 128 == 0, "K must be a multiple of 128");
    HKQ_CHECK_ARG(lda >= K / 2 && ldb >= K / 2 && lda % 16 == 0 && ldb % 16 == 0,
                  "lda/ldb (bytes) must be >= K/2 and multiples of 16");
    HKQ_CHECK_ARG(ldsa >= K / 32 && ldsb >= K / 32 && ldsa % 4 == 0 && ldsb % 4 == 0,
                  "scale row strides must be >= K/32 and multiples of 4");
    HKQ_CHECK_ALIGN(A, 16);
    HKQ_CHECK_ALIGN(B, 16);
    HKQ_CHECK_ALIGN(As, 4);
    HKQ_CHECK_ALIGN(Bs, 4);
    HKQ_CHECK_ALIGN(workspace, 16);
    DenseParams p{};
    p.A = static_cast<const uint8_t*>(A);
    p.B = static_cast<const uint8_t*>(B);
    p.C = static_cast<uint16_t*>(C);
    p.sa = As;
    p.sb = Bs;
    p.M = (int)M; p.N = (int)N; p.K = (int)K; p.kbytes = (int)(K / 2);
    p.lda = lda; p.ldb = ldb; p.ldc = ldc;
    p.lsa = ldsa; p.lsb = ldsb;
    return launch_dense<PlainOp, MODE_MXFP4>(p, workspace, workspace_bytes, stream);
}

int hkq_gemm_mxfp4(const void* A, const void* As, const void* B, const void* Bs, void* C, int64_t M, int64_t N,
                   int64_t K, int64_t lda, int64_t ldb, int64_t ldsa, int64_t ldsb, int64_t ldc, hipStream_t stream) {
    return hkq_gemm_mxfp4_ws(A, As, B, Bs, C, M, N, K, lda, ldb, ldsa, ldsb, ldc, nullptr, 0, stream);
}

int hkq_batched_gemm_a8w8(const void* A, const void* B, const float* sa, const float* sb, const void* bias, void* C,
                          int64_t batch, int64_t M, int64_t N, int64_t K, int64_t lda, int64_t ldb, int64_t ldc,
                          int64_t batch_stride_a, int64_t batch_stride_b, int64_t batch_stride_c,
                          int64_t batch_stride_sa, int64_t batch_stride_sb, int64_t batch_stride_bias,
                          hipStream_t stream) {
    if (int e = check_common(M, N, K, ldc, C)) return e;
    HKQ_CHECK_ARG(batch >= 0 && batch <= 65535, "batch must be in [0, 65535]");
    HKQ_CHECK_ARG(K % 64 == 0, "K must be a multiple of 64");
    HKQ_CHECK_ARG(lda >= K && ldb >= K && lda % 16 == 0 && ldb % 16 == 0,
                  "lda/ldb must be >= K and multiples of 16");
    HKQ_CHECK_ARG(batch <= 1 || (batch_stride_a % 16 == 0 && batch_stride_b % 16 == 0 && batch_stride_c % 8 == 0 &&
                                 batch_stride_sb % 4 == 0 && batch_stride_bias % 4 == 0),
                  "batch strides must keep every batch's operands aligned (A, B: 16 bytes; C: 8 elements; "
                  "b_scale, bias: 4 elements)");
    HKQ_CHECK_ALIGN(A, 16);
    HKQ_CHECK_ALIGN(B, 16);
    HKQ_CHECK_ALIGN(sb, 16);
    HKQ_CHECK_ALIGN(bias, 8);
    if (batch == 0) return 0;
    DenseParams p{};
    p.A = static_cast<const uint8_t*>(A);
    p.B = static_cast<const uint8_t*>(B);
    p.C = static_cast<uint16_t*>(C);
    p.sa = sa;
    p.sb = sb;
    p.M = (int)M; p.N = (int)N; p.K = (int)K; p.kbytes = (int)K;
    p.lda = lda; p.ldb = ldb; p.ldc = ldc;
    p.batch = (int)batch;
    p.bias = static_cast<const uint16_t*>(bias);
    p.bs_a = batch_stride_a; p.bs_b = batch_stride_b; p.bs_c = batch_stride_c;
    p.bs_sa = batch_stride_sa; p.bs_sb = batch_stride_sb; p.bs_bias = batch_stride_bias;
    return launch_dense<PlainOp, MODE_A8W8>(p, nullptr, 0, stream);
}

size_t hkq_gemm_bf16_workspace(int64_t M, int64_t N, int64_t K) {
    if (M <= 0 || N <= 0 || K <= 0 || K % 32 != 0) return 0;
    return dense_plan(MODE_BF16, M, N, 2 * K).ws_bytes;
}

int hkq_batched_gemm_bf16(const void* A, const void* B, const void* bias, void* C, int64_t batch, int64_t M, int64_t N,
                          int64_t K, int64_t lda, int64_t ldb, int64_t ldc, int64_t batch_stride_a,
                          int64_t batch_stride_b, int64_t batch_stride_c, int64_t batch_stride_bias, void* workspace,
                          size_t workspace_bytes, hipStream_t stream) {
    if (int e = check_common(M, N, K, ldc, C)) return e;
    HKQ_CHECK_ARG(batch >= 0 && batch <= 65535, "batch must be in [0, 65535]");
    HKQ_CHECK_ARG(K % 32 == 0, "K must be a multiple of 32");
    HKQ_CHECK_ARG(lda >= K && ldb >= K && lda % 8 == 0 && ldb % 8 == 0,
                  "lda/ldb (elements) must be >= K and multiples of 8");
    HKQ_CHECK_ARG(batch <= 1 || (batch_stride_a % 8 == 0 && batch_stride_b % 8 == 0 && batch_stride_c % 8 == 0 &&
                                 batch_stride_bias % 4 == 0),
                  "batch strides must keep every batch's operands aligned (A, B, C: 8 elements; bias: 4)");
    HKQ_CHECK_ALIGN(A, 16);
    HKQ_CHECK_ALIGN(B, 16);
    HKQ_CHECK_ALIGN(bias, 8);
    HKQ_CHECK_ALIGN(workspace, 16);
    if (batch == 0) return 0;
    DenseParams p{};
    p.A = static_cast<const uint8_t*>(A);
    p.B = static_cast<const uint8_t*>(B);
    p.C = static_cast<uint16_t*>(C);
    p.M = (int)M; p.N = (int)N; p.K = (int)K; p.kbytes = (int)(2 * K);
    p.lda = 2 * lda; p.ldb = 2 * ldb; p.ldc = ldc;
    p.batch = (int)batch;
    p.bias = static_cast<const uint16_t*>(bias);
    p.bs_a = 2 * batch_stride_a; p.bs_b = 2 * batch_stride_b; p.bs_c = batch_stride_c;
    p.bs_bias = batch_stride_bias;
    return launch_dense<PlainOp, MODE_BF16>(p, workspace, workspace_bytes, stream);
}

int hkq_gemm_bf16(const void* A, const void* B, void* C, int64_t M, int64_t N, int64_t K, int64_t lda, int64_t ldb,
                  int64_t ldc, hipStream_t stream) {
    return hkq_batched_gemm_bf16(A, B, nullptr, C, 1, M, N, K, lda, ldb, ldc, 0, 0, 0, 0, nullptr, 0, stream);
}

}  // extern "C"
