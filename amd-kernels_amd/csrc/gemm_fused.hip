// gemm_fused.hip -- the products of a feed-forward layer with what follows them:
//
//   hkq_gemm_*_epilogue      C = bf16(act(sums * scales + bias) + residual), FP8
//                            and bf16 operands;
//   hkq_gated_ffn_*          H = bf16(act(X Wg^T) * (X Wu^T)) in one kernel, FP8
//                            and bf16 operands (bf16 may keep both projections);
//   hkq_gated_ffn_backward   the gradients of X and W from those of H.
//
// The K loops, tile sizes and their choice are the dense GEMMs' (gemm_dense.h);
// this file adds the epilogues, the pairing of gate and up columns in a tile,
// and for the backward products bf16 operands whose K runs across memory rows.
//
// Few rows are bound by the weights' way from memory, many by the matrix cores;
// what a fused epilogue saves is the passes after the product (an activation of
// [M, 2F] alone reads 4 and writes 2 bytes per feature). us on MI355X, M x N x K
// (gated: M x F x K), inputs that rotate:
//   FP8 + residual      16x4096x14336 12.4 (the weights at 4.7 TB/s), 4096x4096x14336
//                       184 (2.61 PFLOP/s);
//   bf16, bias, GELU    601x14336x4096 87 (0.81 PFLOP/s: a fifth of the 192-row
//                       tiles' rows is padding, 224 of them on 256 CUs);
//   gated FP8           24x14336x4096 25.3 (4.6 TB/s), 4096x14336x4096 359 (2.68
//                       PFLOP/s);
//   gated bf16          301x2816x2048 12.7, 4096x14336x4096 with the projections
//                       kept 737 (1.30 PFLOP/s, and 352 MB written);
//   gated backward      1001x2816x2048 62.9, 4096x14336x4096 1484 (1.30 PFLOP/s
//                       and the gradients' pass over memory).
#include <limits>

#include "gemm_dense.h"

namespace hkq {

static bool make_act(int act, float alpha, ActParams& a) {
    constexpr float LOG2E = 1.44269504089f, TANH_C1 = 1.59576912161f;  // 2 sqrt(2 / pi)
    a = ActParams{0, -std::numeric_limits<float>::infinity(), 0.f, 0.f};
    switch (act) {
        case HKQ_ACT_NONE: return true;
        case HKQ_ACT_RELU: a.lo = 0.f; return true;
        case HKQ_ACT_SILU: a.form = 1; a.c1 = -LOG2E * alpha; return true;
        case HKQ_ACT_GELU_TANH: a.form = 2; a.c1 = -LOG2E * TANH_C1; a.c3 = a.c1 * 0.044715f; return true;
        case HKQ_ACT_GELU: a.form = 3; return true;
    }
    return false;
}

// --------------------------------------------------------------------------
// Gradients of the projections, from dH [M, F] and the kept Y [M, 2F]:
//   dgate = dH * up * act'(gate),  dup = dH * act(gate)
// in fp32, rounded to bf16 (they are operands of bf16 matrix products) into
// rows of P values in Y's column order; values 2F .. P - 1 are zeros, so that
// the products take whole K-tiles. HBM-bound: 6 bytes read and 4 written per
// feature; a thread owns 8 features. 4096x14336 91 us (6.4 TB/s), 1001x2816 8.0.
// A pass of its own, not the products' operand load: both products read dY, each
// of its values once per column of tiles, and the activation would be formed
// anew every time (16 times in either at 4096x14336x4096).
// --------------------------------------------------------------------------
__device__ __forceinline__ void act_grad(const ActParams& p, float v, float& f, float& df) {
    if (p.form == 0) {
        f = v < p.lo ? p.lo : v;
        df = p.lo == 0.0f && v <= 0.0f ? 0.0f : 1.0f;
    } else if (p.form <= 2) {  // SiLU: c3 = 0
        // v^2 is bounded only so that a c3 of zero, or the logistic function's
        // saturation, never meets an infinity
        const float q = min_num(v * v, 1e8f);
        const float s = logistic2(v * __builtin_fmaf(p.c3, q, p.c1));
        const float slope = -0.69314718056f * __builtin_fmaf(3.0f * p.c3, q, p.c1);
        f = v * s;
        df = __builtin_fmaf(f * (1.0f - s), slope, s);
    } else {
        float e;
        const float phi = normal_cdf(v, &e);
        f = v * phi;
        df = __builtin_fmaf(v * 0.3989422804f, e, phi);
    }
}

__device__ __forceinline__ void unpack_bf16x8(const v4i& v, float* f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = bf16_to_f32((uint32_t)v[i] & 0xFFFF);
        f[2 * i + 1] = bf16_to_f32((uint32_t)v[i] >> 16);
    }
}

__global__ __launch_bounds__(256) void gated_grad_kernel(const uint16_t* __restrict__ dh, const uint16_t* __restrict__ y,
                                                         uint16_t* __restrict__ dy, int64_t M, int F, int64_t lddh,
                                                         int64_t ldy, int64_t P, int segs, int interleaved, ActParams act) {
    for (int64_t b = blockIdx.x; b < M * segs; b += gridDim.x) {
        const int64_t row = b / segs;
        const int f = ((int)(b - row * segs) * 256 + (int)threadIdx.x) * 8;
        if (f >= F) continue;
        const uint16_t* yr = y + row * ldy;
        uint16_t* dr = dy + row * P;
        const v4i hv = *reinterpret_cast<const v4i*>(dh + row * lddh + f);
        const v4i y0 = *reinterpret_cast<const v4i*>(yr + (interleaved ? 2 * f : f));
        const v4i y1 = *reinterpret_cast<const v4i*>(yr + (interleaved ? 2 * f + 8 : F + f));
        float h[8], a[8], c[8], g[8], u[8];
        unpack_bf16x8(hv, h);
        unpack_bf16x8(y0, a);
        unpack_bf16x8(y1, c);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            g[j] = interleaved ? (j < 4 ? a[2 * j & 7] : c[2 * j & 7]) : a[j];
            u[j] = interleaved ? (j < 4 ? a[(2 * j & 7) + 1] : c[(2 * j & 7) + 1]) : c[j];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float v, dv;
            act_grad(act, g[j], v, dv);
            g[j] = h[j] * u[j] * dv;
            u[j] = h[j] * v;
        }
        v4i o0, o1;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            o0[j] = (int)(interleaved ? pk_bf16(g[j], u[j]) : pk_bf16(g[2 * j], g[2 * j + 1]));
            o1[j] = (int)(interleaved ? pk_bf16(g[j + 4], u[j + 4]) : pk_bf16(u[2 * j], u[2 * j + 1]));
        }
        *reinterpret_cast<v4i*>(dr + (interleaved ? 2 * f : f)) = o0;
        *reinterpret_cast<v4i*>(dr + (interleaved ? 2 * f + 8 : F + f)) = o1;
        if (f + 8 == F)
            for (int64_t t = 2 * (int64_t)F; t < P; t += 8) *reinterpret_cast<v4i*>(dr + t) = v4i{0, 0, 0, 0};
    }
}

// --------------------------------------------------------------------------
// dX of few tokens and a wide layer: 256 x 256 tiles whose K is split over
// workgroups, each writing its fp32 sums to the workspace in register order (per
// wave, float4 q of lane l at (q * 64 + l) * 16 bytes), and a second launch that
// adds a value's partial sums in split order. The tile that feeds the matrix
// cores best thus serves products of a quarter of the tiles that the CUs want;
// 128 x 128 tiles, which fill the CUs without a split, are bound by their LDS
// reads. A wave's 256 accumulators leave no room for a sum in the same launch.
// --------------------------------------------------------------------------
template <class Op>
__global__ __launch_bounds__(256, 1) void part_gemm_kernel(const DenseParams p) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem_raw[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tiles = p.tiles_m * p.tiles_n;
    const int tile = blockIdx.x % tiles, split = blockIdx.x / tiles;
    int tm, tn;
    tile_coords(tile, p.tiles_m, p.tiles_n, p.group_m, tm, tn);
    const int m0 = tm * DENSE_BM, n0 = tn * DENSE_BN;
    const int kt0 = split * p.kt_split, kt1 = min(p.kbytes / 128, kt0 + p.kt_split);
    v16f acc[DENSE_TN][DENSE_TM];
    dense_kloop<Op, MODE_BF16, DENSE_WAVES_M, DENSE_WAVES_N, DENSE_TM, DENSE_TN, 128>(p, m0, n0, kt0, kt1,
                                                                                      (HKQ_LDS uint8_t*)smem_raw, acc);
    const int rows = p.M - m0 - wave / DENSE_WAVES_N * 128;
    float4* out = reinterpret_cast<float4*>(p.ws) + ((int64_t)(split * tiles + tile) * 4 + wave) * (64 * 64) + lane;
#pragma unroll
    for (int j = 0; j < DENSE_TM; ++j) {
        if (j * 32 >= rows) continue;  // (uniform) rows past the last
#pragma unroll
        for (int i = 0; i < DENSE_TN; ++i) {
            float v[16];
            read_acc(acc[i][j], v, 0);
#pragma unroll
            for (int g = 0; g < 4; ++g)
                out[((i * DENSE_TM + j) * 4 + g) * 64] = make_float4(v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]);
        }
    }
}
// A wave per 32 x 32 values.
__global__ __launch_bounds__(256) void part_sum_kernel(const DenseParams p) {
    const int lane = threadIdx.x & 63;
    const int block = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    const int tiles = p.tiles_m * p.tiles_n, tile = block >> 6, w = block >> 4 & 3, i = block >> 2 & 3, j = block & 3;
    int tm, tn;
    tile_coords(tile, p.tiles_m, p.tiles_n, p.group_m, tm, tn);
    const int m = tm * DENSE_BM + w / DENSE_WAVES_N * 128 + j * 32, n = tn * DENSE_BN + w % DENSE_WAVES_N * 128 + i * 32;
    if (m >= p.M || n >= p.N) return;
    const float4* in = reinterpret_cast<const float4*>(p.ws) + ((int64_t)tile * 4 + w) * (64 * 64) +
                       (i * DENSE_TM + j) * 256 + lane;
    const int64_t stride = (int64_t)tiles * 4 * (64 * 64);
    float4 sum[4] = {in[0], in[64], in[128], in[192]};
#pragma unroll 3
    for (int s = 1; s < p.splits; ++s) {
        in += stride;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const float4 v = in[g * 64];
            sum[g].x += v.x, sum[g].y += v.y, sum[g].z += v.z, sum[g].w += v.w;
        }
    }
    const int row = m + (lane & 31);
    if (row >= p.M) return;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const int col = n + 8 * g + 4 * (lane >> 5);
        if (col < p.N)
            *reinterpret_cast<v2i*>(p.C + (int64_t)row * p.ldc + col) =
                v2i{(int)pk_bf16(sum[g].x, sum[g].y), (int)pk_bf16(sum[g].z, sum[g].w)};
    }
}
template <class Op>
static int launch_part(DenseParams& p, int splits, int kt_split, void* ws, hipStream_t stream) {
    constexpr int LDS = dense_ring_lds<MODE_BF16, 128>();
    auto kern = part_gemm_kernel<Op>;
    static bool attr_set = false;
    if (int e = set_lds(kern, LDS, attr_set)) return e;
    p.tiles_m = (p.M + DENSE_BM - 1) / DENSE_BM;
    p.tiles_n = (p.N + DENSE_BN - 1) / DENSE_BN;
    if (p.group_m <= 0) p.group_m = 8;
    p.splits = splits;
    p.kt_split = kt_split;
    p.ws = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + SPLIT_CNT_BYTES);
    const unsigned tiles = (unsigned)(p.tiles_m * p.tiles_n);
    kern<<<tiles * splits, 256, LDS, stream>>>(p);
    if (int e = hkq_launch_status()) return e;
    part_sum_kernel<<<tiles * 16, 256, 0, stream>>>(p);
    return hkq_launch_status();
}

// Plan of a backward product over `KT` K-tiles of 64: the least estimated time
// over the tile sizes, rounds over the CUs * (K-tiles * us + e), or K split over
// workgroups in one round of them, on 128 x 128 tiles (summed by the last one) or
// (`part`, dX) on 256 x 256 tiles with a second launch. us and e fitted to MI355X
// times of every size at 16 .. 4096 tokens of six layers (K-tiles of one size cost
// more the more of the weight comes from memory; the constants are those of a
// large one). Tokens x F x K, us: dX 4096x14336x4096 256 x 256 672, 128 x 256 784,
// 128 x 128 1047; 1024x14336x4096 256 x 256 in four parts 209, 128 x 128 280;
// 512x14336x4096 eight parts 121, 128 x 128 in two splits 155; 256x14336x4096
// twelve parts 86, four splits 83; 1001x2816x2048 128 x 64 31, 128 x 128 36, two
// splits 30, six parts 41; 64x2816x2048 21, 33, six splits 12.5. dW 1001x2816x2048
// 192 x 256 (one round only) 26, 256 x 256 29, 128 x 256 34, 128 x 128 34;
// 1001x1408x2048 21, 21, 18.5, 23.
struct TransPlan {
    int tile;  // a DenseTile
    int splits, kt_split;
    size_t ws_bytes;
};
static TransPlan trans_plan(int64_t M, int64_t N, int64_t KT, bool part) {
    const int64_t ncu = cu_count() > 0 ? cu_count() : 256;
    static const struct { int tile, bm, bn; TileCost c; } T[] = {
        {DT_256, 256, 256, {1.37f, 5.7f}}, {DT_128x256, 128, 256, {0.85f, 3.2f}}, {DT_128x128, 128, 128, {0.57f, 2.2f}},
        {DT_128x64, 128, 64, {0.40f, 2.0f}}, {DT_192x256, 192, 256, {1.06f, 5.0f}}};
    TransPlan p{DT_256, 1, (int)KT, 0};
    float best = 0.f;
    for (const auto& t : T) {
        const int64_t tiles = ((M + t.bm - 1) / t.bm) * ((N + t.bn - 1) / t.bn), rounds = (tiles + ncu - 1) / ncu;
        if (t.tile == DT_192x256 && rounds > 1) continue;
        float us = (float)rounds * ((float)KT * t.c.us + t.c.e);
        // few tiles run as M halves (launch_dense_whole)
        if (t.tile == DT_256 && 2 * tiles <= ncu && M > 128) us = (float)KT * 0.88f + 3.0f;
        if (best == 0.f || us < best) p.tile = t.tile, best = us;
    }
    const int64_t t128 = ((M + 127) / 128) * ((N + 127) / 128);
    const int64_t most = t128 <= SPLIT_MAX_TILES ? std::min<int64_t>(ncu / t128, KT / 4) : 0;
    for (int64_t s = 2; s <= most; ++s) {
        const int64_t per = (KT + s - 1) / s, n = (KT + per - 1) / per;
        const float us = (float)per * 0.62f + 6.5f + 1.2f * (float)n;
        if (us < best) {
            best = us;
            p = TransPlan{DT_SPLIT, (int)n, (int)per, SPLIT_CNT_BYTES + (size_t)(n * t128) * (128 * 128 * 4)};
        }
    }
    // the parts take 12 % less than the rest or stay out: the estimates are those of
    // a weight that comes from memory (1500x5632x2048, whose weight the caches hold,
    // estimated 97 and 102, measured 81 and 73)
    const int64_t t256 = ((M + 255) / 256) * ((N + 255) / 256);
    best *= 0.88f;
    for (int64_t s = 2; part && s <= std::min<int64_t>(ncu / t256, KT / 8); ++s) {
        const int64_t per = (KT + s - 1) / s, n = (KT + per - 1) / per;
        const float us = (float)per * 1.30f + 4.6f + (float)(n * t256) * 0.19f;
        if (us < best) {
            best = us;
            p = TransPlan{DT_PART, (int)n, (int)per, SPLIT_CNT_BYTES + (size_t)(n * t256) * (256 * 256 * 4)};
        }
    }
    return p;
}

// C [M, N] = A . B^T over K rows of memory (B, and A with AT), K-tiles of 64.
// Weights and activations stay as the forward has them: a transposed copy of W
// alone would read and write 235 MB each at 14336x4096 features, 90 us; the
// transposed LDS reads cost nothing against the plain product's (dX 693 us, dW
// 702, the forward's gate and up 735; 1.39 PFLOP/s).
template <bool AT>
static int launch_trans(DenseParams& p, void* ws, hipStream_t stream) {
    using Op = TransOp<AT, true>;
    p.c16 = p.ldc % 8 == 0 && reinterpret_cast<uintptr_t>(p.C) % 16 == 0;
    const TransPlan pl = trans_plan(p.M, p.N, p.kbytes / 128, !AT);
    switch (pl.tile) {
        case DT_128x64: return launch_dense_kgroup<Op, KgCfg<MODE_BF16, 4, 1, 2, 1, 2, 3>>(p, stream);
        case DT_128x128: return launch_dense_kgroup<Op, KgCfg<MODE_BF16, 4, 2, 1, 1, 2, 4>>(p, stream);
        case DT_128x256: return launch_dense_kgroup<Op, KgCfg<MODE_BF16, 2, 4, 1, 2, 2, 3>>(p, stream);
        case DT_192x256: return launch_dense_mid<Op, MODE_BF16>(p, stream);
        case DT_PART:
            if constexpr (!AT) return launch_part<Op>(p, pl.splits, pl.kt_split, ws, stream);
            break;
        case DT_SPLIT: return launch_dense_kgroup<Op, KgCfg<MODE_BF16, 4, 2, 1, 1, 2, 4>>(p, stream, pl.splits, pl.kt_split, ws);
    }
    return launch_dense_whole<Op, MODE_BF16, 128>(p, stream);
}

// rows x cols zeros (cols a multiple of 4) in rows ld apart: a gradient without
// tokens or features.
__global__ __launch_bounds__(256) void zero_rows_kernel(uint16_t* out, int64_t rows, int64_t cols, int64_t ld) {
    const int64_t quads = cols / 4;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * quads; i += (int64_t)gridDim.x * 256)
        *reinterpret_cast<v2i*>(out + i / quads * ld + i % quads * 4) = v2i{0, 0};
}
static int launch_zero_rows(void* out, int64_t rows, int64_t cols, int64_t ld, hipStream_t stream) {
    const int64_t blocks = (rows * (cols / 4) + 255) / 256;
    zero_rows_kernel<<<(unsigned)std::min<int64_t>(blocks, 1 << 16), 256, 0, stream>>>(static_cast<uint16_t*>(out), rows, cols, ld);
    return hkq_launch_status();
}

// Row pitch (values) of the projections' gradients, and their place in the
// backward's workspace after the split counters and partial sums of either
// product.
static int64_t grad_pitch(int64_t F) { return (2 * F + 63) / 64 * 64; }
static size_t grad_offset(int64_t M, int64_t F, int64_t K) {
    const size_t dx = trans_plan(M, K, grad_pitch(F) / 64, true).ws_bytes,
                 dw = trans_plan(2 * F, K, (M + 63) / 64, false).ws_bytes;
    return ((dx > dw ? dx : dw) + 255) / 256 * 256;
}

}  // namespace hkq

using namespace hkq;

static int check_act(int act, float alpha, ActParams& a) {
    HKQ_CHECK_ARG(make_act(act, alpha, a), "act must be one of HKQ_ACT_NONE, _RELU, _SILU, _GELU_TANH, _GELU");
    HKQ_CHECK_ARG(act != HKQ_ACT_SILU || (alpha >= -1e30f && alpha <= 1e30f), "alpha must be a number in [-1e30, 1e30]");
    return 0;
}

// The refusal of a call whose output shares memory with an operand; pitches that
// no kernel reaches are named as such.
template <int MODE>
static int check_overlap(const FusedParams& p, bool gated, const char* clash) {
    HKQ_CHECK_ARG(!clash || dense_tile_plan(MODE, p, 1, nullptr, gated, !gated) != DT_NONE, PITCH_REFUSAL);
    HKQ_CHECK_ARG(!clash, clash);
    return 0;
}

template <int MODE>
static int gemm_epilogue(const void* A, const void* B, const float* sa, const float* sb, const void* bias,
                         const void* residual, void* C, int64_t M, int64_t N, int64_t K, int64_t lda, int64_t ldb, int64_t ldr,
                         int64_t ldc, int act, float alpha, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    constexpr int ES = MODE == MODE_BF16 ? 2 : 1;  // bytes per value of A and B
    HKQ_CHECK_ARG(M >= 0 && N >= 0 && K > 0, "M, N must be >= 0 and K > 0");
    HKQ_CHECK_ARG(M < (1 << 30) && N < (1 << 30) && K < (1 << 30), "dimensions must be < 2^30");
    HKQ_CHECK_ARG(N % 4 == 0, "N must be a multiple of 4");
    HKQ_CHECK_ARG(ldc >= N && ldc % 4 == 0 && ldc < (1 << 24), "ldc must be >= N, a multiple of 4 and < 2^24");
    HKQ_CHECK_ARG(MODE == MODE_BF16 || K % 64 == 0, "K must be a multiple of 64");
    HKQ_CHECK_ARG(MODE != MODE_BF16 || K % 32 == 0, "K must be a multiple of 32");
    HKQ_CHECK_ARG(lda >= K && ldb >= K && lda * ES % 16 == 0 && ldb * ES % 16 == 0,
                  "lda/ldb must be >= K and keep rows 16-byte aligned");
    HKQ_CHECK_ARG(!residual || (ldr >= N && ldr % 4 == 0 && ldr < (1 << 24)), "ldr must be >= N, a multiple of 4 and < 2^24");
    FusedParams p{};
    if (int e = check_act(act, alpha, p.act)) return e;
    HKQ_CHECK_ARG(residual != C || ldr == ldc || !residual, "a residual in place of C must have its pitch");
    if (M == 0 || N == 0) return 0;
    HKQ_CHECK_ARG(A && B && C && (MODE == MODE_BF16 || (sa && sb)), "A, B, C and the scales are required");
    HKQ_CHECK_ALIGN(A, 16);
    HKQ_CHECK_ALIGN(B, 16);
    HKQ_CHECK_ALIGN(C, 8);
    HKQ_CHECK_ALIGN(sa, 4);
    HKQ_CHECK_ALIGN(sb, 16);
    HKQ_CHECK_ALIGN(bias, 8);
    HKQ_CHECK_ALIGN(residual, 8);
    HKQ_CHECK_ALIGN(workspace, 16);
    p.A = static_cast<const uint8_t*>(A);
    p.B = static_cast<const uint8_t*>(B);
    p.C = static_cast<uint16_t*>(C);
    p.sa = sa;
    p.sb = sb;
    p.bias = static_cast<const uint16_t*>(bias);
    p.M = (int)M; p.N = (int)N; p.K = (int)K; p.kbytes = (int)(K * ES);
    p.lda = lda * ES; p.ldb = ldb * ES; p.ldc = ldc;
    p.residual = static_cast<const uint16_t*>(residual);
    p.ldr = ldr;
    const MemRows mc{C, M, 2 * N, 2 * ldc};
    const size_t need = MODE == MODE_BF16 ? hkq_gemm_bf16_workspace(M, N, K) : hkq_gemm_a8w8_workspace(M, N, K);
    const MemRows mws{workspace_bytes >= need ? workspace : nullptr, 1, (int64_t)need, 0};
    const char* clash = nullptr;
    if (overlap(mc, {A, M, K * ES, lda * ES}) || overlap(mc, {B, N, K * ES, ldb * ES}) || overlap(mc, {sa, 1, 4 * M, 0}) ||
        overlap(mc, {sb, 1, 4 * N, 0}) || overlap(mc, {bias, 1, 2 * N, 0}))
        clash = "C must not overlap A, B, the scales or the bias";
    else if (residual != C && overlap(mc, {residual, M, 2 * N, 2 * ldr}))
        clash = "the residual must be C itself or not overlap it";
    else if (overlap(mws, mc) || overlap(mws, {residual, M, 2 * N, 2 * ldr}) || overlap(mws, {A, M, K * ES, lda * ES}) ||
             overlap(mws, {B, N, K * ES, ldb * ES}))
        clash = "the workspace must not overlap an operand";
    if (int e = check_overlap<MODE>(p, false, clash)) return e;
    return launch_dense<FusedOp, MODE>(p, workspace, workspace_bytes, stream);
}

template <int MODE>
static int gated_ffn(const void* X, const void* W, const float* sx, const float* sw, void* H, void* Y, int64_t M, int64_t F,
                     int64_t K, int64_t ldx, int64_t ldw, int64_t ldh, int64_t ldy, int act, float alpha, int interleaved,
                     hipStream_t stream) {
    constexpr int ES = MODE == MODE_BF16 ? 2 : 1;
    HKQ_CHECK_ARG(M >= 0 && F >= 0 && K > 0, "M, F must be >= 0 and K > 0");
    HKQ_CHECK_ARG(M < (1 << 30) && F < (1 << 28) && K < (1 << 30), "M and K must be < 2^30, F < 2^28");
    HKQ_CHECK_ARG(F % 8 == 0, "F must be a multiple of 8");
    HKQ_CHECK_ARG(MODE == MODE_BF16 || K % 64 == 0, "K must be a multiple of 64");
    HKQ_CHECK_ARG(MODE != MODE_BF16 || K % 32 == 0, "K must be a multiple of 32");
    HKQ_CHECK_ARG(ldx >= K && ldw >= K && ldx * ES % 16 == 0 && ldw * ES % 16 == 0,
                  "ldx/ldw must be >= K and keep rows 16-byte aligned");
    HKQ_CHECK_ARG(ldh >= F && ldh % 4 == 0 && ldh < (1 << 24), "ldh must be >= F, a multiple of 4 and < 2^24");
    HKQ_CHECK_ARG(!Y || (ldy >= 2 * F && ldy % 4 == 0 && ldy < (1 << 24)), "ldy must be >= 2F, a multiple of 4 and < 2^24");
    FusedParams p{};
    if (int e = check_act(act, alpha, p.act)) return e;
    if (M == 0 || F == 0) return 0;
    HKQ_CHECK_ARG(X && W && H && (MODE == MODE_BF16 || (sx && sw)), "X, W, H and the scales are required");
    HKQ_CHECK_ALIGN(X, 16);
    HKQ_CHECK_ALIGN(W, 16);
    HKQ_CHECK_ALIGN(sx, 4);
    HKQ_CHECK_ALIGN(sw, 16);
    HKQ_CHECK_ALIGN(H, 8);
    HKQ_CHECK_ALIGN(Y, 8);
    p.A = static_cast<const uint8_t*>(X);
    p.B = static_cast<const uint8_t*>(W);
    p.Bu = p.B + (interleaved ? ldw : F * ldw) * ES;
    p.C = static_cast<uint16_t*>(H);
    p.sa = sx;
    p.sb = sw;
    p.M = (int)M; p.N = (int)(2 * F); p.F = (int)F; p.K = (int)K; p.kbytes = (int)(K * ES);
    p.lda = ldx * ES; p.ldb = (interleaved ? 2 : 1) * ldw * ES; p.ldc = ldh;
    p.interleaved = interleaved != 0;
    p.Y = static_cast<uint16_t*>(Y);
    p.ldy = ldy;
    p.y16 = ldy % 8 == 0 && reinterpret_cast<uintptr_t>(Y) % 16 == 0;
    const MemRows mh{H, M, 2 * F, 2 * ldh}, my{Y, M, 4 * F, 2 * ldy}, mx{X, M, K * ES, ldx * ES}, mw{W, 2 * F, K * ES, ldw * ES};
    const char* clash = nullptr;
    if (overlap(mh, mx) || overlap(mh, mw) || overlap(mh, {sx, 1, 4 * M, 0}) || overlap(mh, {sw, 1, 8 * F, 0}))
        clash = "H must not overlap X, W or the scales";
    else if (overlap(my, mx) || overlap(my, mw) || overlap(my, mh))
        clash = "Y must not overlap X, W or H";
    if (int e = check_overlap<MODE>(p, true, clash)) return e;
    return launch_dense<GatedOp, MODE>(p, nullptr, 0, stream);
}

extern "C" {

int hkq_gemm_a8w8_epilogue(const void* A, const void* B, const float* sa, const float* sb, const void* bias,
                           const void* residual, void* C, int64_t M, int64_t N, int64_t K, int64_t lda, int64_t ldb,
                           int64_t ldr, int64_t ldc, int act, float alpha, void* workspace, size_t workspace_bytes,
                           hipStream_t stream) {
    return gemm_epilogue<MODE_A8W8>(A, B, sa, sb, bias, residual, C, M, N, K, lda, ldb, ldr, ldc, act, alpha, workspace,
                                    workspace_bytes, stream);
}

int hkq_gemm_bf16_epilogue(const void* A, const void* B, const void* bias, const void* residual, void* C, int64_t M,
                           int64_t N, int64_t K, int64_t lda, int64_t ldb, int64_t ldr, int64_t ldc, int act, float alpha,
                           void* workspace, size_t workspace_bytes, hipStream_t stream) {
    return gemm_epilogue<MODE_BF16>(A, B, nullptr, nullptr, bias, residual, C, M, N, K, lda, ldb, ldr, ldc, act, alpha,
                                    workspace, workspace_bytes, stream);
}

int hkq_gated_ffn_a8w8(const void* X, const void* W, const float* sx, const float* sw, void* H, int64_t M, int64_t F,
                       int64_t K, int64_t ldx, int64_t ldw, int64_t ldh, int act, float alpha, int interleaved,
                       hipStream_t stream) {
    return gated_ffn<MODE_A8W8>(X, W, sx, sw, H, nullptr, M, F, K, ldx, ldw, ldh, 0, act, alpha, interleaved, stream);
}

int hkq_gated_ffn_bf16(const void* X, const void* W, void* H, void* Y, int64_t M, int64_t F, int64_t K, int64_t ldx,
                       int64_t ldw, int64_t ldh, int64_t ldy, int act, float alpha, int interleaved, hipStream_t stream) {
    return gated_ffn<MODE_BF16>(X, W, nullptr, nullptr, H, Y, M, F, K, ldx, ldw, ldh, ldy, act, alpha, interleaved, stream);
}

size_t hkq_gated_ffn_backward_workspace(int64_t M, int64_t F, int64_t K) {
    if (M <= 0 || F <= 0 || K <= 0) return 0;
    return grad_offset(M, F, K) + (size_t)M * (size_t)grad_pitch(F) * 2;
}

int hkq_gated_ffn_backward(const void* dH, const void* X, const void* W, const void* Y, void* dX, void* dW, int64_t M,
                           int64_t F, int64_t K, int64_t lddh, int64_t ldx, int64_t ldw, int64_t ldy, int64_t lddx,
                           int64_t lddw, int act, float alpha, int interleaved, void* workspace, size_t workspace_bytes,
                           hipStream_t stream) {
    HKQ_CHECK_ARG(M >= 0 && F >= 0 && K > 0, "M, F must be >= 0 and K > 0");
    // tokens are dW's K: their bytes count in 32 bits
    HKQ_CHECK_ARG(M < (1 << 29) && F <= (1 << 20) && K < (1 << 30), "M must be < 2^29, K < 2^30, F <= 2^20");
    HKQ_CHECK_ARG(F % 8 == 0, "F must be a multiple of 8");
    HKQ_CHECK_ARG(K % 32 == 0, "K must be a multiple of 32");
    HKQ_CHECK_ARG(lddh >= F && lddh % 8 == 0, "lddh must be >= F and a multiple of 8");
    HKQ_CHECK_ARG(ldy >= 2 * F && ldy % 8 == 0, "ldy must be >= 2F and a multiple of 8");
    HKQ_CHECK_ARG(!dW || (ldx >= K && ldx % 8 == 0 && ldx < (1 << 24)), "ldx must be >= K, a multiple of 8 and < 2^24");
    HKQ_CHECK_ARG(!dX || (ldw >= K && ldw % 8 == 0 && ldw < (1 << 24)), "ldw must be >= K, a multiple of 8 and < 2^24");
    HKQ_CHECK_ARG(!dX || (lddx >= K && lddx % 4 == 0 && lddx < (1 << 23)), "lddx must be >= K, a multiple of 4 and < 2^23");
    HKQ_CHECK_ARG(!dW || (lddw >= K && lddw % 4 == 0 && lddw < (1 << 23)), "lddw must be >= K, a multiple of 4 and < 2^23");
    ActParams a;
    if (int e = check_act(act, alpha, a)) return e;
    if (!dX && !dW) return 0;
    if (F == 0 && (M == 0 || !dX)) return 0;
    HKQ_CHECK_ARG(M == 0 || F == 0 || (dH && Y), "dH and Y are required");
    HKQ_CHECK_ARG(M == 0 || F == 0 || ((!dW || X) && (!dX || W)), "X is required for dW, W for dX");
    HKQ_CHECK_ARG(workspace_bytes >= hkq_gated_ffn_backward_workspace(M, F, K) && (workspace || M == 0 || F == 0),
                  "the workspace is smaller than hkq_gated_ffn_backward_workspace(M, F, K)");
    HKQ_CHECK_ALIGN(dH, 16);
    HKQ_CHECK_ALIGN(X, 16);
    HKQ_CHECK_ALIGN(W, 16);
    HKQ_CHECK_ALIGN(Y, 16);
    HKQ_CHECK_ALIGN(dX, 8);
    HKQ_CHECK_ALIGN(dW, 8);
    HKQ_CHECK_ALIGN(workspace, 16);
    // The outputs over the operands of the products: dX = dY . W and dW = dY^T . X
    // run one after the other, dW first where dX takes X's memory.
    const MemRows mx{X, M, 2 * K, 2 * ldx}, mw{W, 2 * F, 2 * K, 2 * ldw}, mdx{dX, M, 2 * K, 2 * lddx},
        mdw{dW, 2 * F, 2 * K, 2 * lddw}, mws{workspace, 1, (int64_t)hkq_gated_ffn_backward_workspace(M, F, K), 0};
    HKQ_CHECK_ARG(!overlap(mdx, mw), "dX must not overlap W");
    HKQ_CHECK_ARG(!overlap(mdw, mx), "dW must not overlap X");
    HKQ_CHECK_ARG(!overlap(mdx, mdw), "dX and dW must not overlap");
    const bool dw_first = dW && overlap(mdx, mx);
    HKQ_CHECK_ARG(!dw_first || !overlap(mdw, mw), "dX over X and dW over W: one of the two at most");
    const MemRows mdh{dH, M, 2 * F, 2 * lddh}, my{Y, M, 4 * F, 2 * ldy};
    HKQ_CHECK_ARG(!overlap(mws, mdh) && !overlap(mws, my) && !(dW && overlap(mws, mx)) && !(dX && overlap(mws, mw)) &&
                      !overlap(mws, mdx) && !overlap(mws, mdw),
                  "the workspace must not overlap an operand");
    if (M == 0) return dW ? launch_zero_rows(dW, 2 * F, K, lddw, stream) : 0;
    if (F == 0) return launch_zero_rows(dX, M, K, lddx, stream);
    const int64_t P = grad_pitch(F);
    uint16_t* dy_rows = reinterpret_cast<uint16_t*>(static_cast<uint8_t*>(workspace) + grad_offset(M, F, K));
    const uint8_t* dy = reinterpret_cast<const uint8_t*>(dy_rows);
    const int segs = (int)((F / 8 + 255) / 256);
    gated_grad_kernel<<<(unsigned)std::min<int64_t>(M * segs, 1 << 20), 256, 0, stream>>>(
        static_cast<const uint16_t*>(dH), static_cast<const uint16_t*>(Y), dy_rows, M, (int)F, lddh, ldy, P, segs,
        interleaved != 0, a);
    if (int e = hkq_launch_status()) return e;
    auto product_dx = [&]() -> int {  // [M, K] = dY [M, 2F] . W [2F, K]
        DenseParams p{};
        p.A = dy; p.B = static_cast<const uint8_t*>(W); p.C = static_cast<uint16_t*>(dX);
        p.M = (int)M; p.N = (int)K; p.K = (int)(2 * F); p.kbytes = (int)(2 * P);
        p.lda = 2 * P; p.ldb = 2 * ldw; p.ldc = lddx;
        return launch_trans<false>(p, workspace, stream);
    };
    auto product_dw = [&]() -> int {  // [2F, K] = dY^T . X [M, K]
        DenseParams p{};
        p.A = dy; p.B = static_cast<const uint8_t*>(X); p.C = static_cast<uint16_t*>(dW);
        p.M = (int)(2 * F); p.N = (int)K; p.K = (int)M; p.kbytes = (int)((M + 63) / 64 * 128);
        p.lda = 2 * P; p.ldb = 2 * ldx; p.ldc = lddw;
        return launch_trans<true>(p, workspace, stream);
    };
    if (dw_first)
        if (int e = product_dw()) return e;
    if (dX)
        if (int e = product_dx()) return e;
    if (dW && !dw_first)
        if (int e = product_dw()) return e;
    return 0;
}

}  // extern "C"
