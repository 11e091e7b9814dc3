// gemm_dense.h -- kernels, tile plan and launchers of the dense GEMMs, over an
// operation `Op` that says what a workgroup does around the K loop:
//   PlainOp  C = bf16(sums x scales (+ bias)), one or a batch of GEMMs
//            (gemm.hip);
//   FusedOp  bias, activation and residual in the epilogue;
//   GatedOp  gate and up rows of one weight in one tile;
//   TransOp  bf16 operands with K across memory rows (these three:
//            gemm_fused.hip).
#pragma once
#include <algorithm>
#include <cstdlib>
#include <type_traits>

#include "gemm_kgroup.h"
#include "gemm_stream.h"
#include "hkq_host.h"

namespace hkq {

struct DenseParams {
    const uint8_t* A;
    const uint8_t* B;
    uint16_t* C;
    const void* sa;
    const void* sb;
    int M, N, K;          // K in elements
    int kbytes;           // K in bytes per row of A/B (a multiple of the K-tile)
    int64_t lda, ldb;     // bytes
    int64_t ldc;          // elements
    int64_t lsa, lsb;     // MXFP4 scale row strides (bytes)
    int tiles_m, tiles_n, group_m;
    int n_whole;          // workgroups [0, n_whole) compute whole tiles 0 .. n_whole-1
    int n_split;          // tiles n_whole .. n_whole+n_split-1 are computed as two M halves
    int c16;              // rows of C are 16-byte aligned (ldc % 8 == 0, C 16-byte aligned)
    int splits;           // K splits of the split path (1: none)
    int kt_split;         // K-tiles per split
    float* ws;            // split partials (splits > 1)
    uint64_t* split_cnt;  // splits > 1: per tile, the arrival counter of its splits
    // batched A8W8 GEMMs: grid.y walks the batch; the operands of batch z start
    // z * bs_* further (bytes for A/B, elements for the others); bias bf16 [N]
    // per batch (nullptr: none), added after the scales
    int batch;  // 0 or 1: one GEMM
    const uint16_t* bias;
    int64_t bs_a, bs_b, bs_c, bs_sa, bs_sb, bs_bias;
};

// The parameters of this workgroup's batch (blockIdx.y).
__device__ __forceinline__ DenseParams batch_slice(const DenseParams& p) {
    DenseParams q = p;
    if (gridDim.y > 1) {
        const int64_t z = blockIdx.y;
        q.A += z * p.bs_a;
        q.B += z * p.bs_b;
        q.C += z * p.bs_c;
        q.sa = static_cast<const float*>(p.sa) + z * p.bs_sa;
        q.sb = static_cast<const float*>(p.sb) + z * p.bs_sb;
        if (p.bias) q.bias += z * p.bs_bias;
    }
    return q;
}

// bias of columns n .. n+3 (zero when there is none or n is past N; N % 4 == 0)
__device__ __forceinline__ float4 bias4(const DenseParams& p, int n) {
    if (!p.bias || n >= p.N) return make_float4(0.f, 0.f, 0.f, 0.f);
    const uint2 b = *reinterpret_cast<const uint2*>(p.bias + n);
    return make_float4(bf16_to_f32(b.x & 0xFFFF), bf16_to_f32(b.x >> 16), bf16_to_f32(b.y & 0xFFFF),
                       bf16_to_f32(b.y >> 16));
}

// What a workgroup does besides the plain product, as a template argument of
// the kernels:
//   FUSED   bias, activation and residual in the epilogue (FusedParams);
//   GATED   the columns of a tile are gate and up rows of the same features of
//           one weight (gemm_mainloop); the epilogue forms act(gate) * up;
//   AT, BT  the operand lies with its rows contiguous and K across memory rows
//           (bf16; p.kbytes counts 2 bytes per value of K, rounded up to whole
//           K-tiles, p.K the rows that there are).
struct PlainOp {
    using Params = DenseParams;
    static constexpr bool FUSED = false, GATED = false, AT = false, BT = false;
};

// Activations: 0 max(v, lo) (lo -inf: none, 0: ReLU), 1 v * logistic(c1 v) (SiLU,
// c1 = alpha), 2 v * logistic(v (c1 + c3 v^2)) (tanh GELU, whose 0.5 (1 + tanh z)
// is the logistic function of 2z), 3 v * Phi(v), Phi the normal distribution
// function (GELU). c1 and c3 hold a factor -log2(e).
struct ActParams {
    int form;
    float lo, c1, c3;
};

// Phi(v) by Abramowitz & Stegun 7.1.26: erfc(z) = (a1 t + .. + a5 t^5) exp(-z^2),
// t = 1 / (1 + 0.3275911 z), z >= 0, absolute error at most 1.5e-7. *density:
// exp(-v^2 / 2).
__device__ __forceinline__ float normal_cdf(float v, float* density) {
    const float e = __builtin_amdgcn_exp2f(v * v * -0.72134752f);
    const float k = __builtin_amdgcn_rcpf(__builtin_fmaf(__builtin_fabsf(v), 0.23164189f, 1.0f));
    float a = __builtin_fmaf(k, 0.530702715f, -0.726576014f);
    a = __builtin_fmaf(k, a, 0.710706871f);
    a = __builtin_fmaf(k, a, -0.142248368f);
    a = __builtin_fmaf(k, a, 0.127414796f);
    const float tail = a * k * e;  // erfc(|v| / sqrt 2) / 2
    *density = e;
    return v < 0.0f ? tail : 1.0f - tail;
}

// 1 / (1 + 2^t)
__device__ __forceinline__ float logistic2(float t) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(t)); }

// The activation of N values: one uniform branch for all of them.
template <int N>
__device__ __forceinline__ void act_n(const ActParams& a, float (&v)[N]) {
    if (a.form == 0) {
        if (a.lo != 0.0f) return;
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = v[i] < 0.0f ? 0.0f : v[i];
    } else if (a.form == 1) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] *= logistic2(a.c1 * v[i]);
    } else if (a.form == 2) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] *= logistic2(v[i] * __builtin_fmaf(a.c3, v[i] * v[i], a.c1));
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float d;
            v[i] *= normal_cdf(v[i], &d);
        }
    }
}
__device__ __forceinline__ float4 act4(const ActParams& a, float4 v) {
    float x[4] = {v.x, v.y, v.z, v.w};
    act_n(a, x);
    return make_float4(x[0], x[1], x[2], x[3]);
}

// The activation of a wave's sub-tile.
template <int TN, int TM>
__device__ __forceinline__ void act_tile(const ActParams& a, v16f (&v)[TN][TM]) {
    float x[TN * TM * 16];
#pragma unroll
    for (int i = 0; i < TN * TM * 16; ++i) x[i] = v[i / 16 / TM][i / 16 % TM][i % 16];
    act_n(a, x);
#pragma unroll
    for (int i = 0; i < TN * TM * 16; ++i) v[i / 16 / TM][i / 16 % TM][i % 16] = x[i];
}

struct FusedParams : DenseParams {
    ActParams act;
    // FUSED: residual bf16 [M, N] (nullptr: none), rows ldr elements apart
    const uint16_t* residual;
    int64_t ldr;
    // GATED: B holds F gate and F up rows, the up rows from Bu, both p.ldb bytes
    // apart; N = 2F. C is [M, F]. Column scales (A8W8) in the weight's row order:
    // feature f's at f and F + f, or (interleaved) 2f and 2f + 1. Y: nullptr, or
    // bf16 [M, 2F] in that order, the scaled sums themselves; y16: its rows are
    // 16-byte aligned.
    const uint8_t* Bu;
    int F, interleaved, y16;
    uint16_t* Y;
    int64_t ldy;
};
__device__ __forceinline__ const FusedParams& batch_slice(const FusedParams& p) { return p; }

struct FusedOp {
    using Params = FusedParams;
    static constexpr bool FUSED = true, GATED = false, AT = false, BT = false;
};
struct GatedOp {
    using Params = FusedParams;
    static constexpr bool FUSED = false, GATED = true, AT = false, BT = false;
};
template <bool AT_, bool BT_>
struct TransOp {
    using Params = DenseParams;
    static constexpr bool FUSED = false, GATED = false, AT = AT_, BT = BT_;
};

// Tile geometry of the dense GEMMs: 256 x 256 tiles computed by 4 waves of
// 128 x 128 (whole tiles) or 64 x 128 (M halves of a tile, 128 x 256). K-tiles
// are 128 bytes per row (whole 128-byte lines per row and load: half the
// cache-line requests of 64-byte K-tiles) in a 2-stage ring when K allows,
// else 64 bytes in a 4-stage ring.
constexpr int DENSE_WAVES_M = 2, DENSE_WAVES_N = 2, DENSE_TM = 4, DENSE_TN = 4;
constexpr int DENSE_BM = DENSE_WAVES_M * DENSE_TM * 32, DENSE_BN = DENSE_WAVES_N * DENSE_TN * 32;
template <int KTB>
constexpr int dense_ns() { return KTB == 128 ? 2 : 4; }

// LDS of a dense workgroup: the K-tile ring / epilogue staging (the larger of
// the whole- and half-tile configurations), then (A8W8) the tile's row and
// column scales, 256 floats each, fetched at the start of the tile.
template <int MODE, int KTB>
constexpr int dense_ring_lds() {
    using Whole = DenseCfg<MODE, DENSE_WAVES_M, DENSE_WAVES_N, DENSE_TM, DENSE_TN, KTB>;
    using Half = DenseCfg<MODE, DENSE_WAVES_M, DENSE_WAVES_N, DENSE_TM / 2, DENSE_TN, KTB>;
    constexpr int NS = dense_ns<KTB>();
    return Whole::lds_bytes(NS) > Half::lds_bytes(NS) ? Whole::lds_bytes(NS) : Half::lds_bytes(NS);
}
template <class Op, int MODE, int KTB>
constexpr int dense_lds() {
    return dense_ring_lds<MODE, KTB>() + (MODE == MODE_A8W8 ? 2 * DENSE_BM * 4 : 0) + (Op::FUSED ? DENSE_BN * 2 : 0);
}

// K loop of one (WM*TM*32) x (WN*TN*32) block of C at (m0, n0) over K-tiles
// [kt0, kt1): the operand sources start kt0 K-tiles into the rows, so the
// loop (and its scale-block schedule) counts K-tiles from 0.
template <class Op, int MODE, int WM, int WN, int TM, int TN, int KTB, int NS = dense_ns<KTB>()>
__device__ __forceinline__ void dense_kloop(const typename Op::Params& p, int m0, int n0, int kt0, int kt1, HKQ_LDS uint8_t* smem,
                                            v16f (&acc)[TN][TM]) {
    using Cfg = DenseCfg<MODE, WM, WN, TM, TN, KTB>;
    constexpr int NW = Cfg::NW, BM = Cfg::BM, BN = Cfg::BN;
    constexpr bool FP4 = Cfg::FP4;
    constexpr int SCB_PER_KT = KTB / 16;  // FP4 scale bytes per row per K-tile
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int rows_a = min(p.M - m0, BM), rows_b = min(p.N - n0, BN);
    const int64_t kb0 = (int64_t)kt0 * KTB, ks0 = (int64_t)kt0 * SCB_PER_KT;

    LoopSrc src;
    src.a = p.A + (int64_t)m0 * p.lda + kb0;
    src.b = p.B + (int64_t)n0 * p.ldb + kb0;
    // extents end with the last row's K bytes: whatever the pitch, an offset past
    // the tile's rows that wraps at 32 bits stays inside the operand
    src.a_bytes = min((int64_t)(rows_a - 1) * p.lda + p.kbytes - kb0, (int64_t)0x7FFFFFFF);
    src.b_bytes = min((int64_t)(rows_b - 1) * p.ldb + p.kbytes - kb0, (int64_t)0x7FFFFFFF);
    src.as = FP4 ? static_cast<const uint8_t*>(p.sa) + (int64_t)m0 * p.lsa + ks0 : nullptr;
    src.bs = FP4 ? static_cast<const uint8_t*>(p.sb) + (int64_t)n0 * p.lsb + ks0 : nullptr;
    src.as_bytes = FP4 ? min((int64_t)(rows_a - 1) * p.lsa + p.K / 32 - ks0, (int64_t)0x7FFFFFFF) : 0;
    src.bs_bytes = FP4 ? min((int64_t)(rows_b - 1) * p.lsb + p.K / 32 - ks0, (int64_t)0x7FFFFFFF) : 0;
    src.lsa = p.lsa;
    src.lsb = p.lsb;
    src.KT = kt1 - kt0;
    auto a_off = dense_offs<NW, KTB, Cfg::LA>(wave, lane, p.lda);
    auto b_off = dense_offs<NW, KTB, Cfg::LB>(wave, lane, p.ldb);
    if constexpr (Op::GATED) {
        // the tile's features [n0 / 2, n0 / 2 + BN / 2): gate and up rows alike
        const int f0 = n0 / 2, rows_f = min(p.F - f0, BN / 2);
        src.b = p.B + (int64_t)f0 * p.ldb + kb0;
        src.b2 = p.Bu + (int64_t)f0 * p.ldb + kb0;
        src.b_bytes = min((int64_t)(rows_f - 1) * p.ldb + p.kbytes - kb0, (int64_t)0x7FFFFFFF);
        b_off = dense_offs_gated<NW, KTB, Cfg::LB, TN>(wave, lane, p.ldb);
    }
    // rows of K across memory: columns m0 / n0 of every row from kt0 K-tiles on
    if constexpr (Op::AT) {
        src.ta = T16Src::of(p.A + (int64_t)m0 * 2, p.lda, rows_a, kt0 * 64, p.K, kt1);
        a_off = dense_offs_t16<NW, Cfg::LA, BM>(wave, lane, p.lda);
    }
    if constexpr (Op::BT) {
        src.tb = T16Src::of(p.B + (int64_t)n0 * 2, p.ldb, rows_b, kt0 * 64, p.K, kt1);
        b_off = dense_offs_t16<NW, Cfg::LB, BN>(wave, lane, p.ldb);
    }
    gemm_mainloop<MODE, WM, WN, TM, TN, KTB, NS, Op::BT, Op::AT, Op::GATED>(src, a_off, b_off, smem, lane, wave, acc);
}

// A staged tile to C: the wave's TM*32 rows of COLS bf16 columns, PITCH bytes
// apart at ep, go to rows [mw, ..) and columns [nw, ..) of C inside M x N.
template <int TM, int COLS, int PITCH>
__device__ __forceinline__ void store_staged(const HKQ_LDS uint8_t* ep, int lane, uint16_t* C, int64_t ldc, int M, int N,
                                             int mw, int nw, bool c16) {
    constexpr int SEGS = COLS * 2 / 16, ROWS_PER_PASS = 64 / SEGS, PASSES = TM * 32 / ROWS_PER_PASS;
    constexpr int BATCH = PASSES < 8 ? PASSES : 8;
    int ln = lane;  // opaque copy: keeps rl / seg out of the kernel's prologue
    asm volatile("" : "+v"(ln));
    const int rl = ln / SEGS, seg = ln % SEGS;
    const int n = nw + seg * 8;
#pragma unroll
    for (int b = 0; b < PASSES; b += BATCH) {
        v4i v[BATCH];
#pragma unroll
        for (int k = 0; k < BATCH; ++k) v[k] = lds_read16(ep + ((b + k) * ROWS_PER_PASS + rl) * PITCH + seg * 16);
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            const int m = mw + (b + k) * ROWS_PER_PASS + rl;
            if (m < M) store_piece_bf16(C + (int64_t)m * ldc + n, v[k], N - n, c16);
        }
    }
}

// Residual of a wave's sub-tile, in registers from before the K loop, so that
// nothing waits on it after the sums (no residual: an empty buffer, whose loads
// give zeros). Sub-tiles of one row of accumulator blocks, or of two blocks, HOLD
// it in the accumulators' layout; larger ones as whole row pieces (16 bytes per lane, full
// lines), which reach that layout through the staging area: read straight, 32 rows
// x 8 bytes per load, they would cost a line request per row and load. FP8
// 128x5632x2048 with a residual 10.2 us, 10.6 with the pieces fetched after the
// sums.
template <class Op, int TM, int TN>
struct EpiResidual {
    static constexpr bool HELD = Op::FUSED && (TM == 1 || TM * TN <= 2);
    static constexpr int SEGS = TN * 4, ROWS_PER_PASS = 64 / SEGS, PASSES = TM * 32 / ROWS_PER_PASS;
    v2i v[HELD ? TN : 1][4][HELD ? TM : 1];
    v4i piece[Op::FUSED && !HELD ? PASSES : 1];
    __device__ __forceinline__ void load(const typename Op::Params& p, int lane, int mw, int nw) {
        if constexpr (HELD) {
            const auto rc = make_rsrc(p.residual + (int64_t)mw * p.ldr + nw, p.residual ? 0x7FFFFFFFu : 0u);
            const int khalf = lane >> 5;
#pragma unroll
            for (int i = 0; i < TN; ++i)
#pragma unroll
                for (int g = 0; g < 4; ++g)
#pragma unroll
                    for (int j = 0; j < TM; ++j) {
                        const int m = j * 32 + (lane & 31), n = i * 32 + 8 * g + 4 * khalf;
                        v[i][g][j] = __builtin_amdgcn_raw_buffer_load_b64(
                            rc, mw + m < p.M && nw + n < p.N ? (uint32_t)((m * p.ldr + n) * 2) : OOB, 0, 0);
                    }
        } else if constexpr (Op::FUSED) {
            // reads at or past the last row's end give zeros; what lies past the columns is not stored
            const int rows = min(p.M - mw, TM * 32), cols = min(p.N - nw, TN * 32);
            const auto rc = make_rsrc(p.residual + (int64_t)mw * p.ldr + nw,
                                      p.residual && rows > 0 && cols > 0 ? (uint32_t)(((rows - 1) * p.ldr + cols) * 2) : 0u);
#pragma unroll
            for (int k = 0; k < PASSES; ++k)
                piece[k] = __builtin_amdgcn_raw_buffer_load_b128(
                    rc, (uint32_t)(((k * ROWS_PER_PASS + lane / SEGS) * p.ldr + lane % SEGS * 8) * 2), 0, 0);
        }
    }
};
// Bias of a wave's columns, loaded before the K loop likewise.
template <class Op, int TN>
struct EpiBias {
    v2i v[Op::FUSED ? TN : 1][4];
    __device__ __forceinline__ void load(const typename Op::Params& p, int lane, int nw) {
        if constexpr (Op::FUSED) {
            const auto rc = make_rsrc(p.bias + nw, p.bias && nw < p.N ? (uint32_t)(p.N - nw) * 2u : 0u);
#pragma unroll
            for (int i = 0; i < TN; ++i)
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    v[i][g] = __builtin_amdgcn_raw_buffer_load_b64(rc, (uint32_t)(i * 32 + 8 * g + 4 * (lane >> 5)) * 2u, 0, 0);
        }
    }
};
__device__ __forceinline__ float4 add_bf16x4(float4 v, const v2i& r) {
    const uint32_t lo = (uint32_t)r[0], hi = (uint32_t)r[1];
    return make_float4(v.x + bf16_to_f32(lo & 0xFFFF), v.y + bf16_to_f32(lo >> 16), v.z + bf16_to_f32(hi & 0xFFFF),
                       v.w + bf16_to_f32(hi >> 16));
}

// FUSED epilogue: act(sums * scales + bias) + residual in fp32, one rounding,
// staged and stored as store_tile_bf16 does. A residual in row pieces is put where
// the results will go, and each lane replaces its own values. One branch on the
// activation for the whole sub-tile: one per four columns jumped over the other
// forms' code 8 to 16 times, each a fetch of instructions from L2 (FP8
// 1024x1024x1024 with bias 9.0 us, with one branch 8.0, the plain GEMM 7.0).
template <class Op, int TM, int TN, typename RowScale, typename ColScale4>
__device__ __forceinline__ void fused_store_tile(const FusedParams& p, v16f (&acc)[TN][TM], const EpiResidual<Op, TM, TN>& res,
                                                 const EpiBias<Op, TN>& bias, HKQ_LDS uint8_t* smem, int wave,
                                                 int lane, int mw, int nw, RowScale row_scale, ColScale4 col_scale4) {
    constexpr int PITCH = TN * 32 * 2 + 16;
    constexpr bool HELD = EpiResidual<Op, TM, TN>::HELD;
    HKQ_LDS uint8_t* ep = smem + wave * (TM * 32) * PITCH;
    const int khalf = lane >> 5;
    const bool staged = !HELD && p.residual != nullptr;
    if (staged) {
        using R = EpiResidual<Op, TM, TN>;
        int ln = lane;
        asm volatile("" : "+v"(ln));
        const int rl = ln / R::SEGS, seg = ln % R::SEGS;
#pragma unroll
        for (int k = 0; k < (HELD ? 0 : R::PASSES); ++k)
            *reinterpret_cast<HKQ_LDS v4i*>(ep + (k * R::ROWS_PER_PASS + rl) * PITCH + seg * 16) = res.piece[k];
    }
    float rs[TM];
#pragma unroll
    for (int j = 0; j < TM; ++j) rs[j] = row_scale(j);
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const float4 cs = col_scale4(i, g), cb = add_bf16x4(make_float4(0.f, 0.f, 0.f, 0.f), bias.v[i][g]);
#pragma unroll
            for (int j = 0; j < TM; ++j) {
                const float a = rs[j];
                v16f& v = acc[i][j];
                v[4 * g + 0] = v[4 * g + 0] * a * cs.x + cb.x;
                v[4 * g + 1] = v[4 * g + 1] * a * cs.y + cb.y;
                v[4 * g + 2] = v[4 * g + 2] * a * cs.z + cb.z;
                v[4 * g + 3] = v[4 * g + 3] * a * cs.w + cb.w;
            }
        }
    act_tile(p.act, acc);
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int nl = i * 32 + 8 * g + 4 * khalf;
#pragma unroll
            for (int j = 0; j < TM; ++j) {
                float4 v = make_float4(acc[i][j][4 * g + 0], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]);
                HKQ_LDS v2i* at = reinterpret_cast<HKQ_LDS v2i*>(ep + (j * 32 + (lane & 31)) * PITCH + nl * 2);
                if constexpr (HELD) {
                    if (p.residual) v = add_bf16x4(v, res.v[i][g][j]);
                } else {
                    if (staged) v = add_bf16x4(v, v2i(*at));
                }
                *at = v2i{(int)pk_bf16(v.x, v.y), (int)pk_bf16(v.z, v.w)};
            }
        }
    store_staged<TM, TN * 32, PITCH>(ep, lane, p.C, p.ldc, p.M, p.N, mw, nw, p.c16 != 0);
}

// GATED epilogue: n-tiles i and i + TN / 2 of a lane hold gate and up of the same
// features; C gets act(gate) * up, Y (if kept) both. fw: the wave's first
// feature. The halves of Y go out one after the other through the same staging
// area (a wave's LDS operations complete in order); interleaved, as pairs.
template <int TM, int TN, typename RowScale, typename ColScale4>
__device__ __forceinline__ void gated_store_tile(const FusedParams& p, v16f (&acc)[TN][TM], HKQ_LDS uint8_t* smem, int wave,
                                                 int lane, int mw, int fw, RowScale row_scale, ColScale4 col_scale4) {
    // one n-tile: its rows 0 .. 15 are the gate's, 16 .. 31 the up's, so groups g
    // and g + 2 of a lane's registers belong together
    constexpr int HN = TN == 1 ? 1 : TN / 2, HG = TN == 1 ? 2 : 4, UN = TN / 2, UG = 4 - HG;
    constexpr int PITCH = TN * 32 + 16, PITCH_Y = TN * 64 + 16;
    HKQ_LDS uint8_t* ep = smem + wave * (TM * 32) * PITCH_Y;
    const int khalf = lane >> 5;
    float rs[TM];
#pragma unroll
    for (int j = 0; j < TM; ++j) rs[j] = row_scale(j);
    auto value = [&](int i, int j, int g) {
        const float4 cs = col_scale4(i, g);
        const float a = rs[j];
        return make_float4(acc[i][j][4 * g + 0] * a * cs.x, acc[i][j][4 * g + 1] * a * cs.y, acc[i][j][4 * g + 2] * a * cs.z,
                           acc[i][j][4 * g + 3] * a * cs.w);
    };
    auto each = [&](auto put) {
#pragma unroll
        for (int i = 0; i < HN; ++i)
#pragma unroll
            for (int g = 0; g < HG; ++g)
#pragma unroll
                for (int j = 0; j < TM; ++j) put(i, g, j, j * 32 + (lane & 31), i * 32 + 8 * g + 4 * khalf);
    };
    v16f gate[HN][TM] = {};
    each([&](int i, int g, int j, int, int) {
        const float4 v = value(i, j, g);
        gate[i][j][4 * g + 0] = v.x, gate[i][j][4 * g + 1] = v.y, gate[i][j][4 * g + 2] = v.z, gate[i][j][4 * g + 3] = v.w;
    });
    act_tile(p.act, gate);
    each([&](int i, int g, int j, int r, int n) {
        const v16f& v = gate[i][j];
        const float4 u = value(i + UN, j, g + UG), a = make_float4(v[4 * g + 0], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]);
        *reinterpret_cast<HKQ_LDS v2i*>(ep + r * PITCH + n * 2) =
            v2i{(int)pk_bf16(a.x * u.x, a.y * u.y), (int)pk_bf16(a.z * u.z, a.w * u.w)};
    });
    store_staged<TM, TN * 16, PITCH>(ep, lane, p.C, p.ldc, p.M, p.F, mw, fw, p.c16 != 0);
    if (!p.Y) return;
    if (p.interleaved) {
        each([&](int i, int g, int j, int r, int n) {
            const float4 a = value(i, j, g), u = value(i + UN, j, g + UG);
            *reinterpret_cast<HKQ_LDS v4i*>(ep + r * PITCH_Y + n * 4) =
                v4i{(int)pk_bf16(a.x, u.x), (int)pk_bf16(a.y, u.y), (int)pk_bf16(a.z, u.z), (int)pk_bf16(a.w, u.w)};
        });
        store_staged<TM, TN * 32, PITCH_Y>(ep, lane, p.Y, p.ldy, p.M, 2 * p.F, mw, 2 * fw, p.y16 != 0);
        return;
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        each([&](int i, int g, int j, int r, int n) {
            const float4 v = value(i + half * UN, j, g + half * UG);
            *reinterpret_cast<HKQ_LDS v2i*>(ep + r * PITCH + n * 2) = v2i{(int)pk_bf16(v.x, v.y), (int)pk_bf16(v.z, v.w)};
        });
        store_staged<TM, TN * 16, PITCH>(ep, lane, p.Y + (half ? p.F : 0), p.ldy, p.M, p.F, mw, fw, p.y16 != 0);
    }
}

// Epilogue of the 256-column tiles with something to compute per element: as
// stream_store_tile, groups of 32 rows x 64 columns through the wave's staging
// area, but over loops instead of unrolled code. Unrolled over a wave's 256
// accumulators the activation's instructions alone (every form of it) passed the
// instruction cache and each tile fetched them anew: bf16 4096x28672x4096
// without any activation 772 us against the plain GEMM's 683. A group's
// accumulators are picked by a switch (register numbers cannot be computed), the
// rest is one copy of the code. Stores and residual loads are buffer operations
// that every lane issues, out of range where its row or column is: the stream
// counts them. tile: the tile's row scales, column scales (256 fp32 each, A8W8)
// and bias (256 bf16, FUSED) in LDS; wr / wc: the wave's first row / column of it.
template <int N>
__device__ __forceinline__ void read_acc(const v16f& a, float (&v)[N], int at) {
#pragma unroll
    for (int e = 0; e < 16; ++e) asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(v[at + e]) : "a"(a[e]));
}

// A group's staged 32 rows x 64 columns (row pitch STREAM_STG_PITCH) to rows
// [0, rows) and columns [0, cols) at `base`.
__device__ __forceinline__ void store_group(const HKQ_LDS uint8_t* stg, int lane, uint16_t* base, int64_t ld, int rows, int cols) {
    const auto rc = make_rsrc(base, 0x7FFFFFFFu);
    const int sr = lane >> 3, sc = (lane & 7) * 8;
    const bool ragged = cols < 64 && (cols & 7) != 0;
    v4i d[4];
#pragma unroll
    for (int q = 0; q < 4; ++q)
        d[q] = *reinterpret_cast<const HKQ_LDS v4i*>(stg + (q * 8 + sr) * STREAM_STG_PITCH + (lane & 7) * 16);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int m = q * 8 + sr;
        const uint32_t at = (uint32_t)((m * ld + sc) * 2);
        __builtin_amdgcn_raw_buffer_store_b128(d[q], rc, m < rows && sc + 8 <= cols ? at : OOB, 0, CPOL_NT);
        if (ragged)
            __builtin_amdgcn_raw_buffer_store_b64(v2i{d[q][0], d[q][1]}, rc, m < rows && sc + 4 == cols ? at : OOB, 0, CPOL_NT);
    }
}

template <int MODE>
constexpr int epi_bias_at() { return MODE == MODE_A8W8 ? 2 * DENSE_BM * 4 : 0; }  // LDS: bias after the scales
template <class Op, int MODE>
constexpr int epi_lds() { return epi_bias_at<MODE>() + (Op::FUSED ? DENSE_BN * 2 : 0); }

// The tile's scales and bias into LDS, 64 values of each per wave (rows past M
// and columns past N read zero); every wave issues the same loads.
template <class Op, int MODE>
__device__ __forceinline__ void load_tile_params(const typename Op::Params& p, HKQ_LDS uint8_t* to, int m0, int n0, int rows,
                                                 int cols, int wave, int lane) {
    const int c = wave * 64 + lane;
    if constexpr (MODE == MODE_A8W8) {
        lds_load4(static_cast<const float*>(p.sa) + m0, (uint32_t)rows * 4u, to + wave * 256, (uint32_t)c * 4u);
        if constexpr (Op::GATED) {
            // tile column c of wave column c / 128: a gate column where c % 128 < 64
            const int f = n0 / 2 + gated_row<DENSE_TN>(c), up = c % (DENSE_TN * 32) >= DENSE_TN * 16;
            lds_load4(p.sb, (uint32_t)p.F * 8u, to + DENSE_BM * 4 + wave * 256,
                      f < p.F ? (uint32_t)(p.interleaved ? 2 * f + up : f + up * p.F) * 4u : OOB);
        } else {
            lds_load4(static_cast<const float*>(p.sb) + n0, (uint32_t)cols * 4u, to + DENSE_BM * 4 + wave * 256, (uint32_t)c * 4u);
        }
    }
    // bias: two columns per dword, so 128 dwords (waves 2 and 3 load waves 0 and 1's again)
    if constexpr (Op::FUSED)
        lds_load4(p.bias + n0, p.bias ? (uint32_t)cols * 2u : 0u, to + epi_bias_at<MODE>() + (wave & 1) * 256,
                  (uint32_t)((wave & 1) * 64 + lane) * 4u);
}

template <class Op, int MODE, int TM, int TN>
__device__ __forceinline__ void rolled_store_tile(const FusedParams& p, v16f (&acc)[TN][TM], const HKQ_LDS uint8_t* tile,
                                                  HKQ_LDS uint8_t* stg, int lane, int mw, int nw, int wr, int wc) {
    static_assert(TN == 4, "two groups of columns per wave");
    constexpr bool A8 = MODE == MODE_A8W8;
    int ln = lane;  // opaque copy: the lane's offsets stay out of the tile loop's prologue
    asm volatile("" : "+v"(ln));
    const int khalf = ln >> 5, r = ln & 31;
    const HKQ_LDS float* rows_s = reinterpret_cast<const HKQ_LDS float*>(tile) + wr;
    const HKQ_LDS float* cols_s = reinterpret_cast<const HKQ_LDS float*>(tile) + DENSE_BM + wc + 4 * khalf;
    HKQ_LDS uint8_t* wr_at = stg + r * STREAM_STG_PITCH + 8 * khalf;
    // values of n-tile i of the group's column scales: 16 per lane
    auto scales = [&](int i, float (&s)[16]) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const v4f c = *reinterpret_cast<const HKQ_LDS v4f*>(cols_s + i * 32 + 8 * g);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[4 * g + e] = c[e];
        }
    };
    auto put = [&](int ii, const float (&v)[16]) {
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *reinterpret_cast<HKQ_LDS v2i*>(wr_at + (ii * 32 + 8 * g) * 2) =
                v2i{(int)pk_bf16(v[4 * g], v[4 * g + 1]), (int)pk_bf16(v[4 * g + 2], v[4 * g + 3])};
    };

    if constexpr (Op::FUSED) {
        const int sr = ln >> 3, sc = (ln & 7) * 8;
        const int rows = p.M - mw, cols = p.N - nw;
        // the residual's 32 x 64 values of a group: whole row pieces, one group ahead
        v4i res[4];
        auto load_res = [&](int ip, int j) {
            const int64_t first = (int64_t)(mw + j * 32) * p.ldr + nw + ip * 64;
            const int rr = min(rows - j * 32, 32);
            // reads at or past the last row's end give zeros; what lies past the columns is not stored
            const auto rs = make_rsrc(p.residual + first, rr > 0 && cols > ip * 64
                                                              ? (uint32_t)(((rr - 1) * p.ldr + min(cols - ip * 64, 64)) * 2) : 0u);
#pragma unroll
            for (int q = 0; q < 4; ++q)
                res[q] = __builtin_amdgcn_raw_buffer_load_b128(rs, (uint32_t)(((q * 8 + sr) * p.ldr + sc) * 2), 0, 0);
        };
        if (p.residual) load_res(0, 0);
#pragma unroll 1
        for (int ip = 0; ip < TN / 2; ++ip) {
            float cs[2][16];
            v2i cb[2][4];
#pragma unroll
            for (int ii = 0; ii < 2; ++ii) {
                if constexpr (A8) scales(2 * ip + ii, cs[ii]);
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    cb[ii][g] = *reinterpret_cast<const HKQ_LDS v2i*>(tile + epi_bias_at<MODE>() +
                                                                      (wc + ip * 64 + ii * 32 + 8 * g + 4 * khalf) * 2);
            }
#pragma unroll 1
            for (int j = 0; j < TM; ++j) {
                if (p.residual) {
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        *reinterpret_cast<HKQ_LDS v4i*>(stg + (q * 8 + sr) * STREAM_STG_PITCH + (ln & 7) * 16) = res[q];
                    if (j + 1 < TM) load_res(ip, j + 1);
                    else if (ip + 1 < TN / 2) load_res(ip + 1, 0);
                }
                float v[32];
                switch (ip * TM + j) {
#define HKQ_PICK(S)                                                          \
    case S:                                                                  \
        if constexpr (S < TM * TN / 2) {                                     \
            read_acc(acc[S / TM * 2][S % TM], v, 0);                         \
            read_acc(acc[S / TM * 2 + 1][S % TM], v, 16);                    \
        }                                                                    \
        break;
                    HKQ_PICK(0) HKQ_PICK(1) HKQ_PICK(2) HKQ_PICK(3) HKQ_PICK(4) HKQ_PICK(5) HKQ_PICK(6) HKQ_PICK(7)
#undef HKQ_PICK
                }
                const float a = A8 ? rows_s[j * 32 + r] : 1.0f;
#pragma unroll
                for (int ii = 0; ii < 2; ++ii)
#pragma unroll
                    for (int g = 0; g < 4; ++g)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float& x = v[16 * ii + 4 * g + e];
                            if constexpr (A8) x = x * a * cs[ii][4 * g + e];
                        }
                if (p.bias) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        const uint32_t w = (uint32_t)cb[e / 16][e / 4 % 4][e % 4 >> 1];
                        v[e] += bf16_to_f32(e & 1 ? w >> 16 : w & 0xFFFF);
                    }
                }
                act_n(p.act, v);
                if (p.residual) {
#pragma unroll
                    for (int ii = 0; ii < 2; ++ii)
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            const v2i rv = *reinterpret_cast<const HKQ_LDS v2i*>(wr_at + (ii * 32 + 8 * g) * 2);
                            float* x = v + 16 * ii + 4 * g;
                            const float4 o = add_bf16x4(make_float4(x[0], x[1], x[2], x[3]), rv);
                            x[0] = o.x, x[1] = o.y, x[2] = o.z, x[3] = o.w;
                        }
                }
                float lo[16], hi[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) lo[e] = v[e], hi[e] = v[16 + e];
                put(0, lo);
                put(1, hi);
                // a wave's LDS operations complete in order: the reads see the writes
                store_group(stg, ln, p.C + (int64_t)(mw + j * 32) * p.ldc + nw + ip * 64, p.ldc, rows - j * 32, cols - ip * 64);
            }
        }
    } else {
        const int fw = nw / 2, rows = p.M - mw, cols = p.F - fw;
        // out 0: act(gate) * up; 1, 2: gate and up themselves (interleaved: 1, 2
        // are the pairs of the group's first and second 32 features)
#pragma unroll 1
        for (int out = 0; out < (p.Y ? 3 : 1); ++out) {
#pragma unroll 1
            for (int j = 0; j < TM; ++j) {
                const float a = A8 ? rows_s[j * 32 + r] : 1.0f;
#pragma unroll 1
                for (int ii = 0; ii < 2; ++ii) {
                    float g[16], u[16];
                    switch (ii * TM + j) {
#define HKQ_PICK(S)                                            \
    case S:                                                    \
        if constexpr (S < TM * 2) {                            \
            read_acc(acc[S / TM][S % TM], g, 0);               \
            read_acc(acc[S / TM + 2][S % TM], u, 0);           \
        }                                                      \
        break;
                        HKQ_PICK(0) HKQ_PICK(1) HKQ_PICK(2) HKQ_PICK(3) HKQ_PICK(4) HKQ_PICK(5) HKQ_PICK(6) HKQ_PICK(7)
#undef HKQ_PICK
                    }
                    if constexpr (A8) {
                        float cg[16], cu[16];
                        scales(ii, cg);
                        scales(ii + 2, cu);
#pragma unroll
                        for (int e = 0; e < 16; ++e) g[e] *= a * cg[e], u[e] *= a * cu[e];
                    }
                    if (out == 0) {
                        act_n(p.act, g);
#pragma unroll
                        for (int e = 0; e < 16; ++e) g[e] *= u[e];
                        put(ii, g);
                    } else if (!p.interleaved) {
                        if (out == 1) put(ii, g);
                        else put(ii, u);
                    } else if (ii == out - 1) {
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            *reinterpret_cast<HKQ_LDS v4i*>(stg + r * STREAM_STG_PITCH + (8 * q + 4 * khalf) * 4) =
                                v4i{(int)pk_bf16(g[4 * q], u[4 * q]), (int)pk_bf16(g[4 * q + 1], u[4 * q + 1]),
                                    (int)pk_bf16(g[4 * q + 2], u[4 * q + 2]), (int)pk_bf16(g[4 * q + 3], u[4 * q + 3])};
                    }
                }
                uint16_t* base = out == 0 ? p.C : p.Y;
                const int64_t ld = out == 0 ? p.ldc : p.ldy;
                int col = fw, left = cols;
                if (out != 0 && p.interleaved) {
                    col = 2 * fw + (out - 1) * 64;
                    left = 2 * cols - (out - 1) * 64;
                } else if (out == 2) {
                    col += p.F;
                }
                store_group(stg, ln, base + (int64_t)(mw + j * 32) * ld + col, ld, rows - j * 32, left);
            }
        }
    }
}

// One (TM*64) x 256 block of C at (m0, n0) on an NS-stage K-tile ring; the tile's
// row and column scales (and bias) follow RING bytes of it.
template <class Op, int MODE, int TM, int KTB, int NS, int RING>
__device__ __forceinline__ void dense_rows(const typename Op::Params& p, int m0, int n0, HKQ_LDS uint8_t* smem) {
    constexpr int WAVES_M = DENSE_WAVES_M, WAVES_N = DENSE_WAVES_N, TN = DENSE_TN;
    using Cfg = DenseCfg<MODE, WAVES_M, WAVES_N, TM, TN, KTB>;
    constexpr int BM = Cfg::BM, BN = Cfg::BN;

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WAVES_N, wn = wave % WAVES_N;
    const int khalf = lane >> 5;

    const int rows_a = min(p.M - m0, BM), rows_b = min(p.N - n0, BN);
    if (rows_a <= 0) return;  // the M half below the last row (uniform per workgroup)

    // A8W8: the tile's row and column scales go to LDS while the K loop runs
    // (rows past M / columns past N read zero); each wave loads 64 of each.
    // These loads are older than the K-tile loads, so the loop's vmcnt waits
    // cover them, and its final vmcnt(0) barrier makes them visible.
    HKQ_LDS uint8_t* scl = smem + RING;
    load_tile_params<Op, MODE>(p, scl, m0, n0, rows_a, rows_b, wave, lane);

    v16f acc[TN][TM];
    dense_kloop<Op, MODE, WAVES_M, WAVES_N, TM, TN, KTB, NS>(p, m0, n0, 0, p.kbytes / KTB, smem, acc);

    // Epilogue (scales of A8W8 applied in registers; MXFP4 has none left)
    const int mw = m0 + wm * TM * 32, nw = n0 + wn * TN * 32;
    auto row_scale = [&](int j) {
        const int r = wm * TM * 32 + j * 32 + (lane & 31);
        return MODE == MODE_A8W8 ? *reinterpret_cast<const HKQ_LDS float*>(scl + r * 4) : 1.0f;
    };
    auto col_scale4 = [&](int i, int g) {
        const int n = wn * TN * 32 + i * 32 + 8 * g + 4 * khalf;
        if constexpr (MODE == MODE_A8W8) {
            const v4f c = *reinterpret_cast<const HKQ_LDS v4f*>(scl + DENSE_BM * 4 + n * 4);
            return make_float4(c[0], c[1], c[2], c[3]);
        }
        return make_float4(1.f, 1.f, 1.f, 1.f);
    };
    if constexpr (Op::FUSED || Op::GATED)
        rolled_store_tile<Op, MODE, TM, TN>(p, acc, scl, smem + wave * STREAM_STG, lane, mw, nw, wm * TM * 32, wn * TN * 32);
    else if (p.bias)
        store_tile_bf16<TM, TN>(acc, smem, wave, lane, p.C, p.ldc, p.M, p.N, mw, nw, p.c16 != 0, row_scale, col_scale4,
                                [&](int i, int g) { return bias4(p, nw + i * 32 + 8 * g + 4 * khalf); });
    else
        store_tile_bf16<TM, TN>(acc, smem, wave, lane, p.C, p.ldc, p.M, p.N, mw, nw, p.c16 != 0, row_scale, col_scale4,
                                NoBias{});
}

// Rows [m0, m0 + TM*64) of tile (tm, tn) of the 256 x 256 tile grid, starting
// `half` * 128 rows into the tile.
template <class Op, int MODE, int TM, int KTB, int NS = dense_ns<KTB>()>
__device__ __forceinline__ void dense_block(const typename Op::Params& p, int tm, int tn, int half, HKQ_LDS uint8_t* smem) {
    using Cfg = DenseCfg<MODE, DENSE_WAVES_M, DENSE_WAVES_N, TM, DENSE_TN, KTB>;
    constexpr int RING = NS == dense_ns<KTB>() ? dense_ring_lds<MODE, KTB>() : Cfg::lds_bytes(NS);
    dense_rows<Op, MODE, TM, KTB, NS, RING>(p, tm * DENSE_BM + half * Cfg::BM, tn * DENSE_BN, smem);
}

// Workgroup u < n_whole computes tile u. When the last round of tiles would
// leave at least half of the CUs idle, its tiles are instead computed as M
// halves by twice as many workgroups: unit v = u - n_whole (XCD v & 7, as the
// dispatcher assigns workgroups round-robin) computes half (v >> 3) & 1 of tile
// n_whole + 8 * (v >> 4) + (v & 7), so both halves of a tile run on one XCD.
// Tile ids then go through tile_coords' XCD-aware order.
template <class Op, int MODE, int KTB>
__global__ __launch_bounds__(64 * DENSE_WAVES_M * DENSE_WAVES_N, 1) void dense_gemm_kernel(const typename Op::Params pb) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem_raw[];
    HKQ_LDS uint8_t* smem = (HKQ_LDS uint8_t*)smem_raw;
    const typename Op::Params p = batch_slice(pb);
    const int u = blockIdx.x;
    int whole = -1, t = -1, half = 0;
    if (u < p.n_whole) {
        whole = u;
    } else {
        const int v = u - p.n_whole;
        t = 8 * (v >> 4) + (v & 7);
        half = (v >> 3) & 1;
        if (t >= p.n_split) return;
    }
    int tm, tn;
    if (whole >= 0) {
        tile_coords(whole, p.tiles_m, p.tiles_n, p.group_m, tm, tn);
        dense_block<Op, MODE, DENSE_TM, KTB>(p, tm, tn, 0, smem);
    } else {
        tile_coords(p.n_whole + t, p.tiles_m, p.tiles_n, p.group_m, tm, tn);
        dense_block<Op, MODE, DENSE_TM / 2, KTB>(p, tm, tn, half, smem);
    }
}

// 192 x 256 tiles (4 waves of 96 x 128), one per workgroup: where the rows fill
// them and leave the last 256-row tile mostly empty (601 rows: 4 tiles of 192
// on 224 of 256 CUs instead of 3 of 256 on 168).
constexpr int MID_TM = 3, MID_BM = DENSE_WAVES_M * MID_TM * 32;
template <class Op, int MODE>
constexpr int mid_lds() {
    return DenseCfg<MODE, DENSE_WAVES_M, DENSE_WAVES_N, MID_TM, DENSE_TN, 128>::lds_bytes(2) + epi_lds<Op, MODE>();
}
template <class Op, int MODE>
__global__ __launch_bounds__(64 * DENSE_WAVES_M * DENSE_WAVES_N, 1) void dense_mid_kernel(const typename Op::Params p) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem_raw[];
    int tm, tn;
    tile_coords(blockIdx.x, p.tiles_m, p.tiles_n, p.group_m, tm, tn);
    dense_rows<Op, MODE, MID_TM, 128, 2, DenseCfg<MODE, DENSE_WAVES_M, DENSE_WAVES_N, MID_TM, DENSE_TN, 128>::lds_bytes(2)>(
        p, tm * MID_BM, tn * DENSE_BN, (HKQ_LDS uint8_t*)smem_raw);
}

// ---------------------------------------------------------------------------
// Persistent streaming kernel (128-byte K-tiles, K-tiles per tile a multiple
// of 8, one 2-D GEMM without bias): workgroup b of G computes whole tiles
// b, b + G, ... < n_whole as one K-tile stream (gemm_stream.h) and, when the
// last round is split, the M half (b >> 3) & 1 of tile n_whole + 8*(b >> 4) +
// (b & 7) (before or after the whole tiles). Epilogues store C from registers
// through a per-wave LDS staging area (DirectEpi). A8W8 row/column scales of
// tile k are prefetched into LDS slot k & 1 when the tile starts.
//
// A half tile (128 x 256) runs on the one-tile K loop with a 3-stage ring:
// per K-tile it moves 48 KB through the LDS for half of a whole tile's MFMAs,
// and its K loop is bound by that traffic; the deeper ring gives the loads
// two K-tiles of lead (measured on MI355X, with the staged epilogue below:
// 4096 x 14336 x 4096 308.8K -> 293.7K cycles per workgroup, 179.4 -> 173.8 us).
constexpr int HALF_NS = 3;                    // ring stages of a half tile

template <int MODE>
constexpr int stream_ring_lds() {
    using Whole = DenseCfg<MODE, DENSE_WAVES_M, DENSE_WAVES_N, DENSE_TM, DENSE_TN, 128>;
    return 2 * Whole::STAGE + Whole::SB_BYTES;
}
// The staging areas follow the ring and (A8W8) the two scale slots.
template <class Op, int MODE>
constexpr int stream_stg_off() { return stream_ring_lds<MODE>() + 2 * epi_lds<Op, MODE>(); }
template <class Op, int MODE>
constexpr int stream_lds() {
    using Half = DenseCfg<MODE, DENSE_WAVES_M, DENSE_WAVES_N, DENSE_TM / 2, DENSE_TN, 128>;
    constexpr int whole = stream_stg_off<Op, MODE>() + DENSE_WAVES_M * DENSE_WAVES_N * STREAM_STG;
    constexpr int half = Half::lds_bytes(HALF_NS) + epi_lds<Op, MODE>();
    return whole > half ? whole : half;
}

// Tile k of the stream: tile id first + k * stride in tile_coords order,
// rows [tm*256 + half*BM, +BM) of it.
template <class Op, int BM>
struct DenseSeq {
    static constexpr bool GATHER = false;
    const typename Op::Params* p;
    int tiles, KT;
    uint32_t lsa, lsb;
    int first, stride, half;
    __device__ void coords(int k, int& m0, int& n0) const {
        int tm, tn;
        tile_coords(first + k * stride, p->tiles_m, p->tiles_n, p->group_m, tm, tn);
        m0 = tm * DENSE_BM + half * BM;
        n0 = tn * DENSE_BN;
    }
    __device__ StreamSrc src(int k) const {
        int m0, n0;
        coords(k, m0, n0);
        const int rows_a = min(p->M - m0, BM), rows_b = min(p->N - n0, DENSE_BN);
        StreamSrc s;
        s.a = p->A + (int64_t)m0 * p->lda;
        s.b = p->B + (int64_t)n0 * p->ldb;
        s.a_bytes = clamp_bytes((int64_t)(rows_a - 1) * p->lda + p->kbytes);
        s.b_bytes = clamp_bytes((int64_t)(rows_b - 1) * p->ldb + p->kbytes);
        if constexpr (Op::GATED) {
            const int f0 = n0 / 2;
            s.b = p->B + (int64_t)f0 * p->ldb;
            s.b2 = p->Bu + (int64_t)f0 * p->ldb;
            s.b_bytes = clamp_bytes((int64_t)(min(p->F - f0, DENSE_BN / 2) - 1) * p->ldb + p->kbytes);
        }
        if constexpr (Op::AT) s.ta = T16Src::of(p->A + (int64_t)m0 * 2, p->lda, rows_a, 0, p->K, KT);
        if constexpr (Op::BT) s.tb = T16Src::of(p->B + (int64_t)n0 * 2, p->ldb, rows_b, 0, p->K, KT);
        s.as = static_cast<const uint8_t*>(p->sa) + (int64_t)m0 * p->lsa;
        s.bs = static_cast<const uint8_t*>(p->sb) + (int64_t)n0 * p->lsb;
        s.as_bytes = (uint32_t)min((int64_t)rows_a * p->lsa, (int64_t)0x7FFFFFFF);
        s.bs_bytes = (uint32_t)min((int64_t)rows_b * p->lsb, (int64_t)0x7FFFFFFF);
        return s;
    }
};

template <class Op, int MODE, int TM, int BM>
struct DirectEpi {
    static constexpr int TN = DENSE_TN;
    // vector-memory instructions a wave issues in end() (at least: ragged
    // tiles add 8-byte stores, a residual its loads, kept projections their
    // stores) plus the next begin(); the stream's first barrier after an
    // epilogue leaves that many in flight
    static constexpr int VM_ISSUED = (Op::GATED ? TM * 4 : TN * TM * 2) + (MODE == MODE_A8W8 ? 2 : 0) + (Op::FUSED ? 1 : 0);
    const DenseSeq<Op, BM>* seq;
    const typename Op::Params* p;
    HKQ_LDS uint8_t* scl;  // 2 slots of epi_lds() bytes
    HKQ_LDS uint8_t* stg;  // this wave's STREAM_STG bytes of staging
    int lane, wave;
    __device__ void begin(int k) {
        int m0, n0;
        seq->coords(k, m0, n0);
        load_tile_params<Op, MODE>(*p, scl + (k & 1) * epi_lds<Op, MODE>(), m0, n0, min(p->M - m0, BM),
                                   min(p->N - n0, DENSE_BN), wave, lane);
    }
    // Stores through the wave's staging area (stream_store_tile), with the
    // tile's row and column scales from its LDS slot.
    __device__ void end(int k, v16f (&acc)[TN][TM]) {
        int m0, n0;
        seq->coords(k, m0, n0);
        const int wm = wave / DENSE_WAVES_N, wn = wave % DENSE_WAVES_N;
        const int khalf = lane >> 5, r = lane & 31;
        const HKQ_LDS uint8_t* slot = scl + (k & 1) * epi_lds<Op, MODE>();
        const HKQ_LDS float* sl = reinterpret_cast<const HKQ_LDS float*>(slot);
        const int mw0 = m0 + wm * TM * 32, nw0 = n0 + wn * TN * 32;
        if constexpr (Op::FUSED || Op::GATED) {
            rolled_store_tile<Op, MODE, TM, TN>(*p, acc, slot, stg, lane, mw0, nw0, wm * TM * 32, wn * TN * 32);
            return;
        } else {
            float rs[TM];
#pragma unroll
            for (int j = 0; j < TM; ++j) rs[j] = MODE == MODE_A8W8 ? sl[wm * TM * 32 + j * 32 + r] : 1.0f;
            stream_store_tile<TM, TN>(
                acc, stg, p->C + (int64_t)mw0 * p->ldc + nw0, p->ldc, p->M - mw0, p->N - nw0, rs,
                [&](int i, int g) {
                    return MODE == MODE_A8W8 ? *reinterpret_cast<const HKQ_LDS v4f*>(sl + DENSE_BM + wn * TN * 32 + i * 32 +
                                                                                     8 * g + 4 * khalf)
                                             : v4f{1.f, 1.f, 1.f, 1.f};
                },
                lane);
        }
    }
};

template <class Op, int MODE, int TM>
__device__ __forceinline__ void dense_stream(const typename Op::Params& p, int tiles, int first, int stride, int half,
                                             HKQ_LDS uint8_t* smem) {
    constexpr int WM = DENSE_WAVES_M, WN = DENSE_WAVES_N, TN = DENSE_TN;
    using Cfg = DenseCfg<MODE, WM, WN, TM, TN, 128>;
    constexpr int BM = Cfg::BM;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    DenseSeq<Op, BM> seq{&p, tiles, p.kbytes / 128, (uint32_t)p.lsa, (uint32_t)p.lsb, first, stride, half};
    DirectEpi<Op, MODE, TM, BM> epi{&seq, &p, smem + stream_ring_lds<MODE>(),
                                    smem + stream_stg_off<Op, MODE>() + wave * STREAM_STG, lane, wave};
    TableOff<Cfg::LA> a_off;
    TableOff<Cfg::LB> b_off;
    if constexpr (Op::AT) a_off = dense_offs_t16<Cfg::NW, Cfg::LA, BM>(wave, lane, p.lda);
    else a_off = dense_offs<Cfg::NW, 128, Cfg::LA>(wave, lane, p.lda);
    if constexpr (Op::GATED) b_off = dense_offs_gated<Cfg::NW, 128, Cfg::LB, TN>(wave, lane, p.ldb);
    else if constexpr (Op::BT) b_off = dense_offs_t16<Cfg::NW, Cfg::LB, Cfg::BN>(wave, lane, p.ldb);
    else b_off = dense_offs<Cfg::NW, 128, Cfg::LB>(wave, lane, p.ldb);
    v16f acc[TN][TM];
    gemm_stream<MODE, WM, WN, TM, TN, Op::BT, Op::AT, Op::GATED>(seq, a_off, b_off, smem, lane, wave, acc, epi);
}

template <class Op, int MODE>
__global__ __launch_bounds__(64 * DENSE_WAVES_M * DENSE_WAVES_N, 1) void dense_stream_kernel(const typename Op::Params p) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem_raw[];
    HKQ_LDS uint8_t* smem = (HKQ_LDS uint8_t*)smem_raw;
    const int b = blockIdx.x, G = gridDim.x;
    const int mine = b < p.n_whole ? (p.n_whole - 1 - b) / G + 1 : 0;
    const int t = 8 * (b >> 4) + (b & 7);
    // Half of the workgroups (half of each XCD's) take their half tile first:
    // their tile boundaries then fall between the others', so the epilogues'
    // bursts of C stores come in two waves (measured on MI355X: 4096 x 14336
    // x 4096, 190.3 -> 186.9 us)
    const bool half_first = (b >> 4) & 1;
    const bool has_half = t < p.n_split;
    int tm = 0, tn = 0;
    if (has_half) tile_coords(p.n_whole + t, p.tiles_m, p.tiles_n, p.group_m, tm, tn);
    if (half_first && has_half) {
        dense_block<Op, MODE, DENSE_TM / 2, 128, HALF_NS>(p, tm, tn, (b >> 3) & 1, smem);
        // the stream's first loads overwrite the half tile's staging: every
        // wave's LDS reads are done first (its C stores may still drain)
        lds_barrier();
    }
    if (mine > 0) dense_stream<Op, MODE, DENSE_TM>(p, mine, b, G, 0, smem);
    if (!half_first && has_half) dense_block<Op, MODE, DENSE_TM / 2, 128, HALF_NS>(p, tm, tn, (b >> 3) & 1, smem);
}

// ---------------------------------------------------------------------------
// 128 x 128 tiles (4 waves of 64 x 64; FP8 with M <= 128 and K <= 16384: 128 x
// 64 tiles, 4 waves of 32 x 64) with two workgroups per CU or with K split over
// the workgroups of one launch. A split's workgroup u computes tile
// u % tiles over K-tiles [s * kt_split, (s+1) * kt_split), s = u / tiles, and
// writes its fp32 sums to the workspace in register order (per wave, float4 q
// of lane l at (q * 64 + l) * 16 bytes: every store is a contiguous 1 KB).
// Then it counts itself in at the tile's arrival counter; the split that
// arrives last (ticket splits - 1) adds the partials of all splits in split
// order (s = 0, 1, ...: the same fp32 sums whichever split arrives last), runs
// the epilogue and puts the counter back to SPLIT_IDLE. Without a split the
// workgroup runs the epilogue itself.

// The scales of a wave's (TM*32) x (TN*32) block (A8W8: rows past M and
// columns past N read 1; other modes: 1), loaded into registers before the K
// loop so that the epilogue waits on none of them.
template <class Op, int MODE, int TM, int TN>
struct EpiScales {
    float r[TM];
    float4 c[TN][4];
    __device__ __forceinline__ void load(const typename Op::Params& p, int lane, int mw, int nw) {
        const int khalf = lane >> 5;
#pragma unroll
        for (int j = 0; j < TM; ++j) {
            const int m = mw + j * 32 + (lane & 31);
            r[j] = (MODE == MODE_A8W8 && m < p.M) ? static_cast<const float*>(p.sa)[m] : 1.0f;
        }
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                if constexpr (Op::GATED) {
                    c[i][g] = make_float4(1.f, 1.f, 1.f, 1.f);
                    const int f = nw / 2 + (TN == 1 ? 8 * (g & 1) : i % (TN / 2) * 32 + 8 * g) + 4 * khalf;
                    const bool up = TN == 1 ? g >= 2 : i >= TN / 2;
                    if (MODE == MODE_A8W8 && f < p.F) {
                        const float* s = static_cast<const float*>(p.sb) + (p.interleaved ? 2 * f : up ? p.F + f : f);
                        c[i][g] = *reinterpret_cast<const float4*>(s);
                        if (p.interleaved) {
                            const float4 d = *reinterpret_cast<const float4*>(s + 4);
                            c[i][g] = up ? make_float4(c[i][g].y, c[i][g].w, d.y, d.w)
                                         : make_float4(c[i][g].x, c[i][g].z, d.x, d.z);
                        }
                    }
                    continue;
                }
                const int n = nw + i * 32 + 8 * g + 4 * khalf;
                c[i][g] = (MODE == MODE_A8W8 && n < p.N)
                              ? *reinterpret_cast<const float4*>(static_cast<const float*>(p.sb) + n)
                              : make_float4(1.f, 1.f, 1.f, 1.f);
            }
    }
};

template <class Op, int MODE, int TM, int TN>
__device__ __forceinline__ void dense_epilogue_global(const typename Op::Params& p, v16f (&acc)[TN][TM],
                                                      const EpiScales<Op, MODE, TM, TN>& sc,
                                                      const EpiResidual<Op, TM, TN>& res, const EpiBias<Op, TN>& bias,
                                                      HKQ_LDS uint8_t* smem, int wave, int lane, int mw, int nw) {
    const int khalf = lane >> 5;
    auto row_scale = [&](int j) { return sc.r[j]; };
    auto col_scale4 = [&](int i, int g) { return sc.c[i][g]; };
    if constexpr (Op::FUSED)
        fused_store_tile<Op, TM, TN>(p, acc, res, bias, smem, wave, lane, mw, nw, row_scale, col_scale4);
    else if constexpr (Op::GATED)
        gated_store_tile<TM, TN>(p, acc, smem, wave, lane, mw, nw / 2, row_scale, col_scale4);
    else if (p.bias)
        store_tile_bf16<TM, TN>(acc, smem, wave, lane, p.C, p.ldc, p.M, p.N, mw, nw, p.c16 != 0, row_scale, col_scale4,
                                [&](int i, int g) { return bias4(p, nw + i * 32 + 8 * g + 4 * khalf); });
    else
        store_tile_bf16<TM, TN>(acc, smem, wave, lane, p.C, p.ldc, p.M, p.N, mw, nw, p.c16 != 0, row_scale, col_scale4,
                                NoBias{});
}

// Split partials cross XCDs, whose L2s are not coherent with each other: they
// are written and read with device-scope cache policy (sc1: the store writes
// through to the coherent level, the load does not hit a line another XCD may
// have changed), so no whole-L2 write-back or invalidate is needed; a wave's
// stores are complete (vmcnt 0) before its workgroup counts in.
constexpr int CPOL_SC1 = 16;

// Arrival counters of split tiles: bits 63..16 hold the SPLIT_MAGIC mark,
// 15..0 the number of splits counted in. An idle counter is SPLIT_MAGIC << 16
// (count 0), and the last split of a call leaves it so; one arrival then costs
// a single fetch-and-add. A counter without the mark (a workspace never used
// for a split plan, or memory another tensor held) is claimed by compare-and-
// swap: the arrival whose swap installs a count of 1 is counted by it, every
// other arrival that found the counter unmarked counts itself in again once it
// sees the mark. Exactly `splits` arrivals are counted, so exactly one draws
// the last ticket.
constexpr uint64_t SPLIT_MAGIC = 0x686B71535054ull;  // 48 bits
constexpr uint64_t SPLIT_IDLE = SPLIT_MAGIC << 16;
// Counters sit at the start of the split workspace, one per tile, for at most
// SPLIT_MAX_TILES tiles (every plan uses the same ones, so partial sums of
// another plan never overwrite them); the partial sums follow.
constexpr int SPLIT_MAX_TILES = 512;
constexpr size_t SPLIT_CNT_BYTES = SPLIT_MAX_TILES * 8;

__device__ __forceinline__ int split_ticket(uint64_t* cnt, int splits) {
    auto fresh = [&](uint64_t v) { return (v >> 16) == SPLIT_MAGIC && (int)(v & 0xFFFF) < splits; };
    const uint64_t old = __hip_atomic_fetch_add(cnt, 1ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (fresh(old)) return (int)(old & 0xFFFF);
    uint64_t cur = old + 1;
    for (;;) {  // ends: a swap fails only when another arrival changed the counter
        if (__hip_atomic_compare_exchange_strong(cnt, &cur, SPLIT_IDLE | 1ull, __ATOMIC_RELAXED, __ATOMIC_RELAXED,
                                                 __HIP_MEMORY_SCOPE_AGENT))
            return 0;
        if (fresh(cur)) {  // claimed by another arrival: this one's increment was dropped with the old value
            const uint64_t o = __hip_atomic_fetch_add(cnt, 1ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            return (int)(o & 0xFFFF);
        }
    }
}

// The partial sums of a split tile: this workgroup's go to the workspace, and the
// split that arrives last returns true with all of them added in `sum`
// (`summing` runs in it before the partial sums are read). WIDE: registers for
// three splits' float4 at a time. last_split: LDS past the epilogue's staging, in
// the (idle) K-tile ring.
template <int TM, int TN, int NW, bool WIDE, typename Summing>
__device__ __forceinline__ bool split_sum(const DenseParams& p, v16f (&acc)[TN][TM], v16f (&sum)[TN][TM], int split, int tile,
                                          int tiles, int wave, int lane, HKQ_LDS int& last_split, Summing summing) {
    constexpr int NQ = TN * TM * 4;  // float4 of accumulators per lane
    // this split's partial: float4 q of lane l of wave w at
    // ((s * tiles + tile) * NW + w) * NQ * 64 + q * 64 + l
    const uint32_t wave_slot = (uint32_t)(((int64_t)tile * NW + wave) * NQ * 64 + lane) * 16u;
    const uint32_t split_stride = (uint32_t)tiles * NW * NQ * 64 * 16u;
    const __amdgpu_buffer_rsrc_t ws =
        __builtin_amdgcn_make_buffer_rsrc(p.ws, 0, (int)(split_stride * (uint32_t)p.splits), 0x00020000);
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const v4f v = {acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4i, v), ws,
                                                       (uint32_t)split * split_stride + wave_slot +
                                                           (uint32_t)(((i * TM + j) * 4 + g) * 64 * 16),
                                                       0, CPOL_SC1);
            }
    __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, 0));
    // count this split in (one thread per workgroup)
    __syncthreads();
    if (threadIdx.x == 0) {
        const bool last = split_ticket(p.split_cnt + tile, p.splits) == p.splits - 1;
        if (last) __hip_atomic_store(p.split_cnt + tile, SPLIT_IDLE, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last_split = last;
    }
    __syncthreads();
    if (!last_split) return false;
    summing();
    // sum in split order; the other splits' float4 come in chunks of RCH
    // splits, all loads of a chunk in flight together (three splits' worth of
    // registers where the budget allows: 8 float4 per lane, or one workgroup
    // per CU)
    constexpr int RCH = (NQ <= 8 || WIDE) ? 3 : 1;
    for (int s0 = 0; s0 < p.splits; s0 += RCH) {
        v4f part[RCH][NQ] = {};
#pragma unroll
        for (int c = 0; c < RCH; ++c) {
            const int s = s0 + c;
            if (s < p.splits && s != split) {
#pragma unroll
                for (int q = 0; q < NQ; ++q)
                    part[c][q] = __builtin_bit_cast(
                        v4f, __builtin_amdgcn_raw_buffer_load_b128(ws, (uint32_t)s * split_stride + wave_slot +
                                                                           (uint32_t)(q * 64 * 16),
                                                                   0, CPOL_SC1));
            }
        }
#pragma unroll
        for (int c = 0; c < RCH; ++c) {
            const int s = s0 + c;
            if (s >= p.splits) break;
#pragma unroll
            for (int i = 0; i < TN; ++i)
#pragma unroll
                for (int j = 0; j < TM; ++j)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const int q = (i * TM + j) * 4 + g;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float x = s == split ? acc[i][j][4 * g + e] : part[c][q][e];
                            sum[i][j][4 * g + e] = s == 0 ? x : sum[i][j][4 * g + e] + x;
                        }
                    }
        }
    }
    return true;
}

template <class Op, int MODE, int WM, int WN, int TM, int TN, int KTB, int MINB, int NS>
__global__ __launch_bounds__(64 * WM * WN, MINB) void dense_tile_kernel(const typename Op::Params pb) {
    using Cfg = DenseCfg<MODE, WM, WN, TM, TN, KTB>;
    constexpr int BM = Cfg::BM, BN = Cfg::BN, NW = Cfg::NW;
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem_raw[];
    HKQ_LDS uint8_t* smem = (HKQ_LDS uint8_t*)smem_raw;
    const typename Op::Params p = batch_slice(pb);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tiles = p.tiles_m * p.tiles_n;
    const int tile = blockIdx.x % tiles, split = blockIdx.x / tiles;
    int tm, tn;
    tile_coords(tile, p.tiles_m, p.tiles_n, p.group_m, tm, tn);
    const int m0 = tm * BM, n0 = tn * BN;
    const int KT = p.kbytes / KTB;
    const int kt0 = split * p.kt_split, kt1 = min(KT, kt0 + p.kt_split);
    const int wm = wave / WN, wn = wave % WN;
    const int mw = m0 + wm * TM * 32, nw = n0 + wn * TN * 32;

    // older than the K-tile loads: the loop's vmcnt waits cover them
    EpiScales<Op, MODE, TM, TN> sc;
    sc.load(p, lane, mw, nw);
    EpiResidual<Op, TM, TN> res;
    constexpr bool EARLY = MINB == 1;  // two workgroups per CU: no registers for it (57 spilled)
    if (EARLY && p.splits == 1) res.load(p, lane, mw, nw);
    EpiBias<Op, TN> bias;
    bias.load(p, lane, nw);

    v16f acc[TN][TM];
    dense_kloop<Op, MODE, WM, WN, TM, TN, KTB, NS>(p, m0, n0, kt0, kt1, smem, acc);

    if (p.splits == 1) {
        if (!EARLY) res.load(p, lane, mw, nw);
        dense_epilogue_global<Op, MODE, TM, TN>(p, acc, sc, res, bias, smem, wave, lane, mw, nw);
        return;
    }
    v16f sum[TN][TM];
    static_assert(Cfg::EP_BYTES + 16 <= Cfg::lds_bytes(NS), "room for the split flag");
    HKQ_LDS int& flag = *reinterpret_cast<HKQ_LDS int*>(smem + Cfg::lds_bytes(NS) - 16);
    auto summing = [&] {
        if (EARLY) res.load(p, lane, mw, nw);
    };
    if (!split_sum<TM, TN, NW, MINB == 1>(p, acc, sum, split, tile, tiles, wave, lane, flag, summing)) return;
    if (!EARLY) res.load(p, lane, mw, nw);
    dense_epilogue_global<Op, MODE, TM, TN>(p, sum, sc, res, bias, smem, wave, lane, mw, nw);
}

// ---------------------------------------------------------------------------
// Narrow M (few rows and short K, where 16-column workgroups pay; FP8 and FP4):
// a streaming path on the 16x16x128 MFMA. Workgroup (u, z) owns the 16 columns
// [16u, 16u + 16) of C for rows [16z, 16z + 16); its 4 waves split K (wave w
// takes the 128-value K-steps [w*S/4, (w+1)*S/4) of S) and load their operand
// fragments from memory straight into registers, all steps at once. The waves'
// sums meet in LDS, and wave 0 adds them in wave order, applies the scales and
// writes C.
//
// Fragment layout of the 16x16x128 MFMA (verified on gfx950): lane l supplies
// row l % 16 and 32 K-values of the 128-deep slice (FP8: 32 bytes; FP4: 16 bytes
// in the low 4 VGPRs, scaled per lane by its 32-value block's e8m0); lane l,
// register i of the result holds D[4*(l/16) + i][l % 16]. The MFMA A operand is
// the weight rows (n), B the activation rows (m): a lane holds 4 consecutive n of
// one m. An FP8 sum over K does not depend on which lane supplies which K-value
// as long as both operands agree, so an FP8 lane takes bytes [16q, 16q+16) and
// [64+16q, 64+16q+16) of the step (q = l/16): each 16-byte load covers 64
// contiguous bytes of 16 rows.
//
// Bound by latency: one memory round trip for everything, then the sums'
// exchange. All of a wave's steps (at most 8) are in flight at once, the
// epilogue's scales before them, and no look-ahead load is issued past them:
// 4x4096x4096 5.75 -> 4.9 us against a loop of 8-step rings whose look-ahead
// read nothing and whose scales were fetched after the sums.
constexpr int NARROW_WAVES = 4, NARROW_ROWS = 16, NARROW_MAX_STEPS = 32;

// GATED: 16 features per workgroup, a gate and an up row of the weight per lane
// and step; PAIR: 8 features, rows 0 .. 7 of the operand the gate's and 8 .. 15
// the up's, as many workgroups as the plain product has and no more loads in
// each; a feature's sums then lie in lanes l and l + 32. One row of 4096x4096
// (F 2048): PAIR 5.4 us, 16 features 7.3, the plain product 5.3.
template <class Op, int MODE, bool PAIR = false>
__global__ __launch_bounds__(64 * NARROW_WAVES) void narrow_gemm_kernel(const typename Op::Params pb) {
    constexpr bool FP4 = MODE == MODE_MXFP4;
    constexpr int SB = FP4 ? 64 : 128;                      // bytes of a row per K-step
    constexpr int DEPTH = NARROW_MAX_STEPS / NARROW_WAVES;  // K-steps of a wave at most, all in flight together
    struct Frag {
        v4i b0, b1, a0, a1;  // weight row, activation row (b1, a1: FP8 only)
        uint32_t sb, sa;     // FP4: e8m0 scales of the step's 4 blocks (byte q is the lane's)
        v4i u0, u1;          // GATED (FP8): the up row
    };
    constexpr bool GATED = Op::GATED && !PAIR;
    constexpr int COLS = PAIR ? 8 : 16;
    static_assert(!Op::GATED || !FP4, "gated: FP8");
    __shared__ v4f red[GATED ? 2 : 1][NARROW_WAVES][64];
    const typename Op::Params p = batch_slice(pb);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, q = lane >> 4;
    const int n0 = blockIdx.x * COLS, m0 = blockIdx.z * NARROW_ROWS;
    const int S = p.kbytes / SB;
    const int s0 = wave * S / NARROW_WAVES, s1 = (wave + 1) * S / NARROW_WAVES;
    int cols = p.N;  // GATED: n counts features
    if constexpr (Op::GATED) cols = p.F;
    const int rows_a = min(NARROW_ROWS, p.M - m0), rows_b = min(COLS, cols - n0);
    uint32_t to_up = 0;  // PAIR (F % 8 == 0: all 8 features): from a gate row to its up row
    if constexpr (PAIR) to_up = (uint32_t)(p.Bu - p.B);
    const auto rb = make_rsrc(p.B + (int64_t)n0 * p.ldb, to_up + (uint32_t)(rows_b * p.ldb));
    const uint8_t* up = p.B;
    if constexpr (GATED) up = p.Bu;
    const auto ru = make_rsrc(up + (int64_t)n0 * p.ldb, (uint32_t)(rows_b * p.ldb));
    const auto ra = make_rsrc(p.A + (int64_t)m0 * p.lda, (uint32_t)(rows_a * p.lda));
    const uint32_t b_off = (uint32_t)((PAIR ? r & 7 : r) * p.ldb + 16 * q) + (PAIR && r >= 8 ? to_up : 0u);
    const uint32_t a_off = (uint32_t)(r * p.lda + 16 * q);
    const auto rsb = make_rsrc(FP4 ? static_cast<const uint8_t*>(p.sb) + (int64_t)n0 * p.lsb : p.B,
                               FP4 ? (uint32_t)((rows_b - 1) * p.lsb + 4 * S) : 0u);
    const auto rsa = make_rsrc(FP4 ? static_cast<const uint8_t*>(p.sa) + (int64_t)m0 * p.lsa : p.A,
                               FP4 ? (uint32_t)((rows_a - 1) * p.lsa + 4 * S) : 0u);

    // Steps at or past s1 read zeros (their MFMAs add nothing): offsets with
    // the OOB bit set are past every buffer's range.
    auto load = [&](int s, Frag& f) {
        const uint32_t kill = s < s1 ? 0u : OOB, kb = (uint32_t)s * SB | kill;
        f.b0 = __builtin_amdgcn_raw_buffer_load_b128(rb, b_off + kb, 0, 0);
        if constexpr (!FP4) f.b1 = __builtin_amdgcn_raw_buffer_load_b128(rb, b_off + kb + 64, 0, 0);
        if constexpr (GATED) {
            f.u0 = __builtin_amdgcn_raw_buffer_load_b128(ru, b_off + kb, 0, 0);
            f.u1 = __builtin_amdgcn_raw_buffer_load_b128(ru, b_off + kb + 64, 0, 0);
        }
        f.a0 = __builtin_amdgcn_raw_buffer_load_b128(ra, a_off + kb, 0, 0);
        if constexpr (!FP4) f.a1 = __builtin_amdgcn_raw_buffer_load_b128(ra, a_off + kb + 64, 0, 0);
        if constexpr (FP4) {
            f.sb = __builtin_amdgcn_raw_buffer_load_b32(rsb, (uint32_t)(r * p.lsb) + ((uint32_t)s * 4 | kill), 0, 0);
            f.sa = __builtin_amdgcn_raw_buffer_load_b32(rsa, (uint32_t)(r * p.lsa) + ((uint32_t)s * 4 | kill), 0, 0);
        }
    };
    v4f acc = v4f{0.f, 0.f, 0.f, 0.f}, acc_up = acc;
    auto mma = [&](const Frag& f) {
        if constexpr (FP4) {
            const v8i a = v8i{f.b0[0], f.b0[1], f.b0[2], f.b0[3], 0, 0, 0, 0};
            const v8i b = v8i{f.a0[0], f.a0[1], f.a0[2], f.a0[3], 0, 0, 0, 0};
            acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 4, 4, 0, (int)(f.sb >> (8 * q)), 0,
                                                                   (int)(f.sa >> (8 * q)));
        } else {
            const v8i a = v8i{f.b0[0], f.b0[1], f.b0[2], f.b0[3], f.b1[0], f.b1[1], f.b1[2], f.b1[3]};
            const v8i b = v8i{f.a0[0], f.a0[1], f.a0[2], f.a0[3], f.a1[0], f.a1[1], f.a1[2], f.a1[3]};
            acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 0, 0, 0, 127, 0, 127);
            if constexpr (GATED) {
                const v8i u = v8i{f.u0[0], f.u0[1], f.u0[2], f.u0[3], f.u1[0], f.u1[1], f.u1[2], f.u1[3]};
                acc_up = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(u, b, acc_up, 0, 0, 0, 127, 0, 127);
            }
        }
    };
    // the epilogue's scales go out before the operands: no memory latency
    // follows the K loop
    const int n = n0 + 4 * q, m = m0 + r;
    const bool in = n < cols && m < p.M && (!PAIR || q < 2);  // N % 4 == 0: n .. n+3 all in or all out
    float4 cs = make_float4(1.f, 1.f, 1.f, 1.f), cu = cs;
    float a = 1.f;
    v2i res = v2i{0, 0};
    if (!FP4 && in) {
        const float* sb = static_cast<const float*>(p.sb);
        a = static_cast<const float*>(p.sa)[m];
        if constexpr (Op::GATED) {
            cs = *reinterpret_cast<const float4*>(sb + (p.interleaved ? 2 * n : n));
            cu = *reinterpret_cast<const float4*>(sb + (p.interleaved ? 2 * n + 4 : p.F + n));
            if (p.interleaved) {
                const float4 x = cs, y = cu;
                cs = make_float4(x.x, x.z, y.x, y.z);
                cu = make_float4(x.y, x.w, y.y, y.w);
            }
        } else {
            cs = *reinterpret_cast<const float4*>(sb + n);
        }
        if constexpr (Op::FUSED)
            if (p.residual) res = *reinterpret_cast<const v2i*>(p.residual + (int64_t)m * p.ldr + n);
    }
    float4 c = make_float4(0.f, 0.f, 0.f, 0.f);
    if constexpr (!Op::GATED) c = bias4(p, n);
    Frag f[DEPTH];
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) load(s0 + d, f[d]);
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) mma(f[d]);
    red[0][wave][lane] = acc;
    if constexpr (GATED) red[1][wave][lane] = acc_up;
    __syncthreads();
    if (wave != 0 || !in) return;
    v4f v = red[0][0][lane];
#pragma unroll
    for (int w = 1; w < NARROW_WAVES; ++w) v += red[0][w][lane];
    if constexpr (Op::GATED) {
        const int at = PAIR ? lane + 32 : lane, h = PAIR ? 0 : 1;
        v4f u = red[h][0][at];
#pragma unroll
        for (int w = 1; w < NARROW_WAVES; ++w) u += red[h][w][at];
        const float4 g = act4(p.act, make_float4(v[0] * a * cs.x, v[1] * a * cs.y, v[2] * a * cs.z, v[3] * a * cs.w));
        *reinterpret_cast<v2i*>(p.C + (int64_t)m * p.ldc + n) =
            v2i{(int)pk_bf16(g.x * (u[0] * a * cu.x), g.y * (u[1] * a * cu.y)),
                (int)pk_bf16(g.z * (u[2] * a * cu.z), g.w * (u[3] * a * cu.w))};
        return;
    }
    if constexpr (Op::FUSED) {
        float4 o = act4(p.act, make_float4(v[0] * a * cs.x + c.x, v[1] * a * cs.y + c.y, v[2] * a * cs.z + c.z,
                                           v[3] * a * cs.w + c.w));
        if (p.residual) o = add_bf16x4(o, res);
        *reinterpret_cast<v2i*>(p.C + (int64_t)m * p.ldc + n) = v2i{(int)pk_bf16(o.x, o.y), (int)pk_bf16(o.z, o.w)};
        return;
    }
    *reinterpret_cast<v2i*>(p.C + (int64_t)m * p.ldc + n) =
        v2i{(int)pk_bf16(v[0] * a * cs.x + c.x, v[1] * a * cs.y + c.y),
            (int)pk_bf16(v[2] * a * cs.z + c.z, v[3] * a * cs.w + c.w)};
}

template <typename K>
static int set_lds(K kern, int lds, bool& done) {
    if (done) return 0;
    hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) {
        set_error("hipFuncSetAttribute(MaxDynamicSharedMemorySize=%d) failed: %s", lds, hipGetErrorString(e));
        return (int)e;
    }
    done = true;
    return 0;
}

// ---------------------------------------------------------------------------
// Small tiles with K split over the workgroup's waves (gemm_kgroup.h), chosen
// by dense_tile_plan below. Bound by the way into LDS: a CU takes 95-100 GB/s
// from the caches while it computes (125 GB/s when it only loads from L2), so
// a K-tile of a BM x BN tile costs about its (BM + BN) * 128 bytes at that
// rate. Measured on MI355X against the (32 or 64) x 256 tiles, split-K
// 128 x 64 tiles and streaming kernel that served these shapes before: A8W8
// 48x4096x4096 17.1 -> 6.6 us, 160x4096x4096 15.0 -> 9.9, 64x4096x14336
// 29.6 -> 13.6, 64x28672x4096 42 -> 26; MXFP4 64x8192x8192 19.9 -> 9.1,
// 1x8192x8192 11.9 -> 8.0; bf16 64x4096x4096 25.8 -> 9.0, 1x4096x4096
// 17.1 -> 7.9, 300x4096x4096 22.9 -> 19.1.
template <class Op, class Cfg>
__global__ __launch_bounds__(Cfg::THREADS, 1) void dense_kgroup_kernel(const typename Op::Params pb) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem_raw[];
    HKQ_LDS uint8_t* smem = (HKQ_LDS uint8_t*)smem_raw;
    constexpr int MODE = Cfg::MODE, BM = Cfg::BM, BN = Cfg::BN, TN = Cfg::TN, TM = Cfg::TM;
    const typename Op::Params p = batch_slice(pb);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wg = wave % Cfg::GW, kg = wave / Cfg::GW;
    int tm, tn;
    // BT, eight waves of one sub-tile row: K may be split over workgroups (this
    // one takes K-tiles [kt0, kt1) of its tile)
    constexpr bool SPLITS = Op::BT && Cfg::KG == 1 && TM * TN <= 2;
    int tile = blockIdx.x, split = 0, kt0 = 0, kt1 = (p.kbytes + 64) / 128;
    if constexpr (SPLITS)
        if (p.splits > 1) {
            const int tiles = p.tiles_m * p.tiles_n;
            split = tile / tiles;
            tile -= split * tiles;
            kt0 = split * p.kt_split;
            kt1 = min(kt1, kt0 + p.kt_split);
        }
    tile_coords(tile, p.tiles_m, p.tiles_n, p.group_m, tm, tn);
    const int m0 = tm * BM, n0 = tn * BN;
    const int rows_a = min(p.M - m0, BM), rows_b = min(p.N - n0, BN);

    KgSrc<Cfg> src;
    src.KT = kt1 - kt0;
    src.half_tail = p.kbytes % 128 != 0;
    src.a = buffer_desc(p.A + (int64_t)m0 * p.lda + kt0 * 128, clamp_bytes((int64_t)rows_a * p.lda - kt0 * 128));
    src.b = buffer_desc(p.B + (int64_t)n0 * p.ldb, clamp_bytes((int64_t)rows_b * p.ldb));
#pragma unroll
    for (int i = 0; i < Cfg::SWP; ++i) {
        const int r = kg_row<Cfg>(i, wg, lane);
        src.a_off[i] = (uint32_t)(r * p.lda) + kg_chunk<Cfg>(r, lane);
        src.b_off[i] = (uint32_t)(r * p.ldb) + kg_chunk<Cfg>(r, lane);
    }
    src.a_step = (uint32_t)(8 * Cfg::GW * Cfg::SWP * p.lda);
    src.b_step = (uint32_t)(8 * Cfg::GW * Cfg::SWP * p.ldb);
    src.bs_step = 0;
    src.sc_shift = 0;
    if constexpr (Op::GATED) {
        constexpr int GW = Cfg::GW;
        const int f0 = n0 / 2, rows_f = min(p.F - f0, BN / 2);
        src.b = buffer_desc(p.B + (int64_t)f0 * p.ldb, clamp_bytes((int64_t)(rows_f - 1) * p.ldb + p.kbytes));
        src.b2 = buffer_desc(p.Bu + (int64_t)f0 * p.ldb, clamp_bytes((int64_t)(rows_f - 1) * p.ldb + p.kbytes));
        if (GW == 8 && wg >= 4) src.b = src.b2;
#pragma unroll
        for (int i = 0; i < Cfg::SWP; ++i)
            src.b_off[i] = (uint32_t)(((i * GW + wg) * 8 % 32 + lane / 8) * p.ldb) + kg_chunk<Cfg>(kg_row<Cfg>(i, wg, lane), lane);
        src.b_step = (uint32_t)((GW == 8 ? 32 : 8 * GW * Cfg::SWP) * p.ldb);
    }
    if constexpr (Cfg::FP4) {
        src.as = buffer_desc(static_cast<const uint8_t*>(p.sa) + (int64_t)m0 * p.lsa,
                             clamp_bytes((int64_t)(rows_a - 1) * p.lsa + p.K / 32));
        src.bs = buffer_desc(static_cast<const uint8_t*>(p.sb) + (int64_t)n0 * p.lsb,
                             clamp_bytes((int64_t)(rows_b - 1) * p.lsb + p.K / 32));
#pragma unroll
        for (int i = 0; i < Cfg::PW; ++i) {
            const int q = i * Cfg::GW + wg;
            const int r = kg_piece_row<Cfg>(q < Cfg::PA ? q : q - Cfg::PA, lane);
            src.s_off[i] = (uint32_t)(r * (q < Cfg::PA ? p.lsa : p.lsb)) + kg_piece_half(lane);
        }
    }
    if constexpr (Op::AT) {
        using T = KTileT16<BM>;
        const int r = wg * T::ROWS_PER_LOAD + lane / (T::ROW / 16);
        src.ta = T16Src::of(p.A + (int64_t)m0 * 2, p.lda, rows_a, kt0 * 64, p.K, kt1);
        src.a_off[0] = (uint32_t)(r * p.lda) + (uint32_t)(T::phys(r, lane % (T::ROW / 16)) << 4);
        src.a_step = (uint32_t)(Cfg::GW * T::ROWS_PER_LOAD * p.lda);
    }
    if constexpr (Op::BT) {
        using T = KTileT16<BN>;
        const int r = wg * T::ROWS_PER_LOAD + lane / (T::ROW / 16);
        src.tb = T16Src::of(p.B + (int64_t)n0 * 2, p.ldb, rows_b, kt0 * 64, p.K, kt1);
        src.b_off[0] = (uint32_t)(r * p.ldb) + (uint32_t)(T::phys(r, lane % (T::ROW / 16)) << 4);
        src.b_step = (uint32_t)(Cfg::GW * T::ROWS_PER_LOAD * p.ldb);
    }
    const int mw = m0 + wg / Cfg::WN * TM * 32, nw = n0 + wg % Cfg::WN * TN * 32;
    EpiScales<Op, MODE, TM, TN> sc;
    sc.load(p, lane, mw, nw);
    EpiResidual<Op, TM, TN> res;
    constexpr bool EARLY = !(MODE == MODE_A8W8 && Cfg::GW == 8 && TM * TN == 4);  // no registers for it (48 spilled)
    if (EARLY && kg == 0) res.load(p, lane, mw, nw);
    EpiBias<Op, TN> bias;
    bias.load(p, lane, nw);

    v16f acc[TN][TM];
    kgroup_kloop<Cfg, false, Op::GATED, Op::AT, Op::BT>(src, smem, lane, wg, kg, acc);
    if constexpr (SPLITS)
        if (p.splits > 1) {
            v16f sum[TN][TM];
            static_assert(Cfg::EP + 16 <= Cfg::LDS, "room for the split flag");
            HKQ_LDS int& flag = *reinterpret_cast<HKQ_LDS int*>(smem + Cfg::LDS - 16);
            if (split_sum<TM, TN, Cfg::GW, true>(p, acc, sum, split, tile, p.tiles_m * p.tiles_n, wg, lane, flag, [] {}))
                dense_epilogue_global<Op, MODE, TM, TN>(p, sum, sc, res, bias, smem, wg, lane, mw, nw);
            return;
        }
    if (kg != 0) return;
    if (!EARLY) res.load(p, lane, mw, nw);
    dense_epilogue_global<Op, MODE, TM, TN>(p, acc, sc, res, bias, smem, wg, lane, mw, nw);
}

template <class Op, class Cfg>
static int launch_dense_kgroup(typename Op::Params& p, hipStream_t stream, int splits = 1, int kt_split = 0, void* ws = nullptr) {
    auto kern = dense_kgroup_kernel<Op, Cfg>;
    static bool attr_set = false;
    if (int e = set_lds(kern, Cfg::LDS, attr_set)) return e;
    p.tiles_m = (p.M + Cfg::BM - 1) / Cfg::BM;
    p.tiles_n = (p.N + Cfg::BN - 1) / Cfg::BN;
    if (p.group_m <= 0) p.group_m = 8;
    p.splits = splits;
    if (splits > 1) {  // the arrival counters, then the partial sums (one K group, BT)
        p.kt_split = kt_split;
        p.split_cnt = static_cast<uint64_t*>(ws);
        p.ws = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + SPLIT_CNT_BYTES);
    }
    const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
    kern<<<dim3((unsigned)(tiles * splits), (unsigned)std::max(1, p.batch)), Cfg::THREADS, Cfg::LDS, stream>>>(p);
    return hkq_launch_status();
}

// Split plan of a dense GEMM: the tile geometry, how many K splits, and the
// workspace the splits need (bytes). It answers the workspace queries for all
// shapes (GEO_SKINNY's included, which now run without one), so a caller's
// workspace always covers the launch; dense_tile_plan decides where a split
// runs.
enum DenseGeo { GEO_256 = 0, GEO_128 = 1, GEO_SKINNY = 2, GEO_128x64 = 3 };
struct DensePlan {
    int geo;
    int64_t tiles;
    int splits, kt_split;
    size_t ws_bytes;
};

static DensePlan dense_plan(int mode, int64_t M, int64_t N, int64_t kbytes) {
    DensePlan pl{};
    const int ktb = kbytes % 128 == 0 ? 128 : 64;
    const int64_t KT = kbytes / ktb;
    const int ncu = cu_count() > 0 ? cu_count() : 256;
    auto ntiles = [&](int64_t bm, int64_t bn) { return ((M + bm - 1) / bm) * ((N + bn - 1) / bn); };
    int64_t bm = DENSE_BM, bn = DENSE_BN;
    pl.geo = GEO_256;
    if (ktb == 128 && M <= 64) {
        pl.geo = GEO_SKINNY;
        bm = M <= 32 ? 32 : 64;
        bn = 256;
    } else if (ktb == 128 && 2 * ntiles(DENSE_BM, DENSE_BN) <= ncu) {
        pl.geo = GEO_128;
        bm = bn = 128;
        // FP8 with M <= 128 and K <= 16384: 128 x 64 tiles (4 waves of 32 x 64),
        // twice the workgroups for the same K split and a quarter of the
        // partial sums the last split reads
        if (mode == MODE_A8W8 && M <= 128 && KT <= 128) {
            pl.geo = GEO_128x64;
            bn = 64;
        }
    }
    pl.tiles = ntiles(bm, bn);
    pl.splits = 1;
    pl.kt_split = (int)KT;
    // split K when the tiles fill at most half of the CUs, keeping at least 4
    // K-tiles per split
    if (pl.geo != GEO_256 && pl.tiles > 0 && 2 * pl.tiles <= ncu && pl.tiles <= SPLIT_MAX_TILES && KT >= 8) {
        int64_t s = (ncu + pl.tiles - 1) / pl.tiles;
        s = std::min<int64_t>(s, KT / 4);
        if (s > 1) {
            const int64_t per = (KT + s - 1) / s;
            pl.splits = (int)((KT + per - 1) / per);
            pl.kt_split = (int)per;
        }
    }
    // the arrival counters, then the partial sums
    if (pl.splits > 1) pl.ws_bytes = SPLIT_CNT_BYTES + (size_t)pl.splits * (size_t)pl.tiles * (size_t)(bm * bn) * 4;
    return pl;
}

// Tile size of a dense GEMM: the least estimated time over the sizes below,
//   rounds of tiles over the CUs * (K-tiles * us + e) + 2.3 us,
// us and e per size and operand format fitted to MI355X times of every size at
// 1 .. 2048 rows of 17 weights (512 .. 57344 columns, K 128 .. 16384) and 25
// batches. 128 x 128 tiles on two workgroups per CU run their K-tiles faster
// while there are no more of them than CUs (`alone`: MXFP4 1024x4096x4096 12.9
// us, the eight-wave tile 15.4). 32 x 256 tiles are for up to 32 rows of a short
// K, where every other size takes more rounds (A8W8 batch of 128 1x512x128 4.1
// us, on 128 x 256 5.2; bf16 batch of 64 32x512x512 6.9, on 128 x 128 9.0); with
// a longer one their columns starve the CUs of rows in flight (A8W8
// 300x4096x14336 47 us, on 128 x 64 34). Split K (A8W8 and bf16, a workspace
// given): one round of its own plan, the partial sums' exchange in the constant.
// It is still the better one where half of the CUs' worth of tiles meets a long
// K: 400x4096x14336 31.7 us against 34.7, 128x4096x14336 17.7 against 18.4, bf16
// 512x4096x14336 64 against 72.
//
// The fused and gated products have two sizes more. 192 x 256 tiles in one round
// of them: epilogue bf16 601x14336x4096 86 us, 256 x 256 tiles 95, 128 x 256 103;
// 3000x4096x4096 85, 95, 110; over more rounds the streaming kernel is the better
// one (gated bf16 601x28672x4096 165, 149). 64 x 128: gated bf16 301x5632x2048
// 13.0, 128 x 128 15.9, 64 x 64 19.2; FP8 64x28672x4096 26.0, 28.3, 34.9; bf16
// with up to 64 rows is bound by the weights' way from memory, where 64 x 64
// tiles keep more of them in flight (33x28672x4096 58, 64 x 64 49).
// Their estimates rank the sizes and are no times: those of 256-row tiles were
// fitted where a last round runs as M halves, and 192 x 256 stands beside them, so
// whole tiles take about twice as long (epilogue bf16 601x14336x4096 with SiLU and
// a residual, estimated and measured: 192 x 256 44 and 89, 256 x 256 46 and 98,
// 128 x 256 82 and 106, 128 x 128 71 and 114). By these constants 192 x 256 comes
// before 256 x 256 where its own tiles are one round, and only where 128 x 256
// tiles take a second one, which is where it was measured to be the better one.
enum DenseTile {
    DT_32x32, DT_32x64, DT_32x128, DT_32x256, DT_64x64, DT_128x64, DT_128x128, DT_128x256,
    DT_128x128_PAIR,  // two workgroups per CU (dense_tile_kernel)
    DT_256, DT_SPLIT,
    DT_NONE,  // rows too far apart for every size
    // of the fused and gated products only
    DT_64x128, DT_192x256,
    DT_PART  // 256 x 256 tiles, K split over workgroups, the sums in a second launch (gemm_fused.hip)
};
struct TileCost { float us, e; };
struct TileCosts {
    TileCost tile[DT_256 + 1], alone;
    float split64_us, split64_e;           // 128 x 64 tiles: per K-tile, constant
    float split_us, split_e, split_parts;  // 128 x 128 tiles: per K-tile, constant, per split
    TileCost t64x128, t192x256;
};
static int dense_tile_plan(int mode, const DenseParams& p, int64_t batch, const DensePlan* split, bool gated = false,
                           bool fused = false) {
    const int64_t M = p.M, N = p.N, kbytes = p.kbytes;
    // Tile rows `ld` bytes apart that a 32-bit buffer offset reaches. The 256-row
    // kernels end their extents with the last live row, so only those count
    // there; the smaller ones form offsets for all of a tile's rows.
    auto reach = [](int64_t rows, int64_t ld) { return ld <= 0x7FFFFFFF / rows; };
    auto fits = [&](int64_t bm, int64_t bn) {
        return reach(bm, p.lda) && reach(bn, p.ldb) && reach(bm, p.lsa) && reach(bn, p.lsb);
    };
    static const int BM[] = {32, 32, 32, 32, 64, 128, 128, 128, 128, 256},
                     BN[] = {32, 64, 128, 256, 64, 64, 128, 256, 128, 256};
    static const TileCosts A8W8 = {{{0.082f, 1.8f}, {0.118f, 2.3f}, {0.198f, 3.4f}, {0.36f, 1.5f}, {0.145f, 3.5f},
                                    {0.245f, 2.5f}, {0.345f, 2.0f}, {0.54f, 3.0f}, {0.60f, 1.8f}, {0.716f, 4.5f}},
                                   {0.60f, 1.8f}, 0.345f, 5.7f, 0.4f, 4.2f, 1.3f, {0.26f, 2.5f}, {0.65f, 4.0f}};
    // MXFP4's 128 x 256 tile would cost more than the 256 x 256 one
    static const TileCosts FP4 = {{{0.091f, 1.8f}, {0.125f, 1.9f}, {0.233f, 2.7f}, {0.5f, 1.1f}, {0.188f, 2.9f},
                                   {0.431f, 2.2f}, {0.478f, 2.9f}, {-1.f, 0.f}, {0.717f, 1.2f}, {0.909f, 3.9f}},
                                  {0.611f, 0.0f}, 0.f, 0.f, 0.f, 0.f, 0.f, {}, {}};
    static const TileCosts BF16 = {{{0.098f, 1.0f}, {0.132f, 1.45f}, {0.216f, 1.7f}, {0.31f, 0.85f}, {0.162f, 2.2f},
                                    {0.278f, 1.7f}, {0.347f, 0.6f}, {0.606f, 1.2f}, {0.645f, 0.9f}, {0.647f, 2.1f}},
                                   {0.559f, 0.6f}, 0.f, 0.f, 0.494f, 5.5f, 1.2f, {0.29f, 2.0f}, {0.62f, 2.0f}};
    const TileCosts& T = mode == MODE_A8W8 ? A8W8 : mode == MODE_MXFP4 ? FP4 : BF16;
    const int64_t ncu = cu_count() > 0 ? cu_count() : 256;
    const float KT = (float)((kbytes + 64) / 128);
    int best = DT_NONE;
    float best_us = 0.f;
    for (int t = DT_256; t >= 0; --t) {
        if (T.tile[t].us < 0.f || (t == DT_128x128_PAIR && kbytes % 128 != 0) || (t == DT_32x256 && (M > 32 || KT > 8)))
            continue;
        if (!(t == DT_256 ? fits(std::min<int64_t>(M, 256), std::min<int64_t>(N, 256)) : fits(BM[t], BN[t]))) continue;
        const int64_t tiles = batch * ((M + BM[t] - 1) / BM[t]) * ((N + BN[t] - 1) / BN[t]);
        const int64_t slots = t == DT_128x128_PAIR ? 2 * ncu : ncu;
        const TileCost c = t == DT_128x128_PAIR && tiles <= ncu ? T.alone : T.tile[t];
        const float us = (float)((tiles + slots - 1) / slots) * (KT * c.us + c.e);
        if (best_us == 0.f || us < best_us) {
            best = t;
            best_us = us;
        }
    }
    if (gated || fused) {
        const struct { int t, bm, bn; TileCost c; } more[] = {{DT_64x128, 64, 128, T.t64x128}, {DT_192x256, 192, 256, T.t192x256}};
        for (const auto& o : more) {
            if (!fits(o.bm, o.bn)) continue;
            const int64_t tiles = batch * ((M + o.bm - 1) / o.bm) * ((N + o.bn - 1) / o.bn);
            if (o.t == DT_192x256 && (kbytes % 128 != 0 || tiles > ncu)) continue;
            if (o.t == DT_64x128 && mode == MODE_BF16 && M <= 64) continue;
            const float us = (float)((tiles + ncu - 1) / ncu) * (KT * o.c.us + o.c.e);
            if (best == DT_NONE || us < best_us) best = o.t, best_us = us;
        }
    }
    if (split != nullptr && fits(128, 128)) {
        const float kt = (float)split->kt_split;
        const float us = split->geo == GEO_128x64 ? kt * T.split64_us + T.split64_e
                                                  : kt * T.split_us + T.split_e + T.split_parts * (float)split->splits;
        if (best == DT_NONE || us < best_us) best = DT_SPLIT;
    }
    return best;
}

template <class Op, int MODE, int WM, int WN, int TM, int TN, int KTB, int MINB, int NS = dense_ns<KTB>()>
static int launch_dense_tiles(typename Op::Params& p, int splits, int kt_split, void* ws, hipStream_t stream) {
    using Cfg = DenseCfg<MODE, WM, WN, TM, TN, KTB>;
    constexpr int LDS = Cfg::lds_bytes(NS);
    static_assert(LDS * MINB <= 160 * 1024, "LDS budget of a CDNA4 CU");
    auto kern = dense_tile_kernel<Op, MODE, WM, WN, TM, TN, KTB, MINB, NS>;
    static bool attr_set = false;
    if (int e = set_lds(kern, LDS, attr_set)) return e;
    p.tiles_m = (p.M + Cfg::BM - 1) / Cfg::BM;
    p.tiles_n = (p.N + Cfg::BN - 1) / Cfg::BN;
    if (p.group_m <= 0) p.group_m = 8;
    p.splits = splits;
    p.kt_split = kt_split;
    const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
    if (p.splits > 1) {  // dense_plan's workspace: the arrival counters, then the partial sums
        p.split_cnt = static_cast<uint64_t*>(ws);
        p.ws = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + SPLIT_CNT_BYTES);
    }
    kern<<<dim3((unsigned)(tiles * p.splits), (unsigned)std::max(1, p.batch)), 64 * WM * WN, LDS, stream>>>(p);
    return hkq_launch_status();
}

template <class Op, int MODE>
static int launch_dense_mid(typename Op::Params& p, hipStream_t stream) {
    constexpr int LDS = mid_lds<Op, MODE>();
    static_assert(LDS <= 160 * 1024, "LDS budget of a CDNA4 CU");
    auto kern = dense_mid_kernel<Op, MODE>;
    static bool attr_set = false;
    if (int e = set_lds(kern, LDS, attr_set)) return e;
    p.tiles_m = (p.M + MID_BM - 1) / MID_BM;
    p.tiles_n = (p.N + DENSE_BN - 1) / DENSE_BN;
    if (p.group_m <= 0) p.group_m = 8;
    kern<<<dim3((unsigned)((int64_t)p.tiles_m * p.tiles_n)), 64 * DENSE_WAVES_M * DENSE_WAVES_N, LDS, stream>>>(p);
    return hkq_launch_status();
}

template <class Op, int MODE, int KTB>
static int launch_dense_whole(typename Op::Params& p, hipStream_t stream) {
    constexpr int LDS = dense_lds<Op, MODE, KTB>();
    static_assert(LDS <= 160 * 1024, "LDS budget of a CDNA4 CU");
    auto kern = dense_gemm_kernel<Op, MODE, KTB>;
    static bool attr_set = false;  // per instantiation; the attribute is per-process
    if (int e = set_lds(kern, LDS, attr_set)) return e;
    p.tiles_m = (p.M + DENSE_BM - 1) / DENSE_BM;
    p.tiles_n = (p.N + DENSE_BN - 1) / DENSE_BN;
    // tile rows per group of the walk (measured best: 8 for FP8, 4 for FP4)
    if (p.group_m <= 0) p.group_m = MODE == MODE_MXFP4 ? 4 : 8;
    const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
    if (tiles == 0) return 0;
    // Split the last round into M halves when it would fill at most half of the
    // CUs and the tiles have rows in both halves.
    const int ncu = cu_count();
    const int64_t last = ncu > 0 ? tiles % ncu : 0;
    const bool batched = p.batch > 1;  // a batch fills the GPU by itself: no half tiles
    const int64_t split = (!batched && last > 0 && 2 * last <= ncu && p.M > DENSE_BM / 2) ? last : 0;
    p.n_whole = (int)(tiles - split);
    p.n_split = (int)split;
    // MXFP4 stays on the one-tile kernel: its stream (the K loop below with
    // compile-time scale slots, C stored from registers since the ring and the
    // scale blocks fill the LDS) spills and measured 1.8x slower on MI355X.
    if constexpr (KTB == 128 && MODE != MODE_MXFP4) {
        // the persistent streaming kernel: one workgroup per CU, whole tiles as
        // a K-tile stream (needs K-tiles per tile % 8 == 0; one 2-D GEMM without
        // bias, C's rows 16-byte aligned); HKQ_DENSE_STREAM=0 selects the
        // one-tile-per-workgroup kernel
        static const bool stream_on = [] {
            const char* e = std::getenv("HKQ_DENSE_STREAM");
            return !(e && e[0] == '0');
        }();
        // Measured on MI355X against the one-tile-per-workgroup kernel: 1-3%
        // faster at 1.75-3.5 rounds of tiles, 1-2% at 7 and 14 rounds
        // (4096x28672, 8192x14336 and 8192x28672, K = 4096).
        // Half tile t belongs to workgroup b with t = 8 * (b >> 4) + (b & 7), so
        // the split needs 2 * roundup8(split) workgroups: grids that cannot hold
        // them within one per CU take the one-tile kernel.
        const int64_t g = std::min<int64_t>(ncu, std::max<int64_t>(p.n_whole, 2 * ((split + 7) / 8 * 8)));
        if (stream_on && ncu > 0 && !batched && (Op::FUSED || p.bias == nullptr) && (p.kbytes / 128) % 8 == 0 && p.c16 &&
            2 * ((split + 7) / 8 * 8) <= g) {
            constexpr int SLDS = stream_lds<Op, MODE>();
            static_assert(SLDS <= 160 * 1024, "LDS budget of a CDNA4 CU");
            auto skern = dense_stream_kernel<Op, MODE>;
            static bool sattr = false;
            if (int e = set_lds(skern, SLDS, sattr)) return e;
            skern<<<dim3((unsigned)g), 64 * DENSE_WAVES_M * DENSE_WAVES_N, SLDS, stream>>>(p);
            return hkq_launch_status();
        }
    }
    const int64_t nblk = p.n_whole + 2 * ((split + 7) / 8 * 8);
    kern<<<dim3((unsigned)nblk, (unsigned)std::max(1, p.batch)), 64 * DENSE_WAVES_M * DENSE_WAVES_N, LDS, stream>>>(p);
    return hkq_launch_status();
}

// The narrow path: FP8 and FP4 with at most 32 K-steps, up to 64 rows in groups
// of 16 while there is a CU for every 16-column workgroup of every group; the
// groups' activation loads grow with K, so FP4, whose small tiles are the
// cheaper ones, takes more than 16 steps to 8 rows only. Measured on MI355X
// against the small tiles, us: A8W8 1x4096x4096 4.0 and 5.3, 16x4096x4096 5.4
// both, 32x1000x256 3.7 and 4.1, 64x1000x4096 5.6 and 5.7; MXFP4 1x1000x256 3.7
// and 3.9, 32x1000x1024 3.7 and 4.2, 8x2048x4096 4.6 and 4.7, 16 rows of
// 24 steps 4.8 and 4.5. More workgroups start one after another, 0.9 us per round of them
// whatever K is (A8W8 1x28672x128 8.3 us, 4.0 on small tiles; 1x6144x4096 6.2,
// 5.4), which only a stream that is long by itself hides: A8W8 from 24 K-steps
// on, 1 row from two rounds (1x9216x4096 8.5, 8.9; 4 rows 9.4, 9.0) and 4 rows
// from three (4x12288x4096 9.6, 10.6; 4x28672x4096 19.8, 20.6; 8x28672x4096
// 22.0, 20.6; 4x28672x2048 14.6, 12.8). Its buffer offsets are 32-bit.
static bool use_narrow(int mode, const DenseParams& p, int64_t batch, int64_t cols, bool one_round = false) {
    const int64_t step = mode == MODE_MXFP4 ? 64 : 128, S = p.kbytes / step;
    if (p.M < 1 || p.kbytes % step != 0 || S > NARROW_MAX_STEPS) return false;
    const int64_t wide = (1ll << 31) / NARROW_ROWS;
    if (p.lda >= wide || p.ldb >= wide || p.lsa >= wide || p.lsb >= wide) return false;
    const int64_t ncu = cu_count() > 0 ? cu_count() : 256;
    const int64_t groups = (p.M + NARROW_ROWS - 1) / NARROW_ROWS, wgs = batch * ((cols + 15) / 16);
    if (groups <= 4 && groups * wgs <= ncu) return mode == MODE_A8W8 || S <= 16 || p.M <= 8;
    return !one_round && mode == MODE_A8W8 && S >= 24 && p.M <= (wgs >= 3 * ncu ? 4 : wgs >= 2 * ncu ? 1 : 0);
}

constexpr char PITCH_REFUSAL[] = "row pitches too large: 32 rows of each operand (or all of its rows) and of its scales "
                                 "must span less than 2^31 bytes";

template <class Op, int MODE>
static int launch_dense(typename Op::Params& p, void* ws, size_t ws_bytes, hipStream_t stream) {
    p.c16 = (p.ldc % 8 == 0) && (reinterpret_cast<uintptr_t>(p.C) % 16 == 0);
    if (p.M == 0 || p.N == 0) return 0;
    const int64_t batch = std::max(1, p.batch);
    if (p.M == 1) {  // a single row's pitch is never stepped over
        p.lda = p.kbytes;
        if (MODE == MODE_MXFP4) p.lsa = p.K / 32;
    }
    if constexpr (MODE != MODE_BF16) {
        if constexpr (Op::GATED) {  // 8 features per workgroup where that is one round, buffer offsets in 32 bits
            const int64_t span = (p.Bu - p.B) + 8 * p.ldb;
            if (span < (1ll << 31) && use_narrow(MODE, p, batch, p.N, true)) {
                const dim3 grid((unsigned)(p.F / 8), 1, (unsigned)((p.M + NARROW_ROWS - 1) / NARROW_ROWS));
                narrow_gemm_kernel<Op, MODE, true><<<grid, 64 * NARROW_WAVES, 0, stream>>>(p);
                return hkq_launch_status();
            }
        }
        // gated: a workgroup's 16 columns are 16 features, for up to 8 rows: us against small
        // tiles 8x5632x2048 (F 2816) 6.0, 6.0, 16 rows 6.3, 6.0; 24x4096x4096 8.6, 7.9
        const int cols = Op::GATED ? p.N / 2 : p.N;
        if ((!Op::GATED || p.M <= 8) && use_narrow(MODE, p, batch, cols)) {
            const dim3 grid((unsigned)((cols + 15) / 16), (unsigned)batch, (unsigned)((p.M + NARROW_ROWS - 1) / NARROW_ROWS));
            narrow_gemm_kernel<Op, MODE><<<grid, 64 * NARROW_WAVES, 0, stream>>>(p);
            return hkq_launch_status();
        }
    }
    // the split partials and their reduction are per 2-D GEMM without bias
    DensePlan pl{};
    bool split = false;
    if constexpr (MODE != MODE_MXFP4) {
        pl = dense_plan(MODE, p.M, p.N, p.kbytes);
        split = !Op::GATED && p.batch <= 1 && (Op::FUSED || p.bias == nullptr) && pl.geo != GEO_SKINNY && pl.splits > 1 &&
                ws != nullptr && ws_bytes >= pl.ws_bytes;
    }
    constexpr int M4 = MODE == MODE_MXFP4;  // the e8m0 blocks take LDS from the ring
    switch (dense_tile_plan(MODE, p, batch, split ? &pl : nullptr, Op::GATED, Op::FUSED)) {
        case DT_32x32: return launch_dense_kgroup<Op, KgCfg<MODE, 1, 1, 4, 1, 1, 4>>(p, stream);
        case DT_32x64: return launch_dense_kgroup<Op, KgCfg<MODE, 1, 1, 4, 1, 2, 3 - M4>>(p, stream);
        case DT_32x128: return launch_dense_kgroup<Op, KgCfg<MODE, 1, 1, 4 - M4, 1, 4, 2>>(p, stream);
        case DT_32x256: return launch_dense_kgroup<Op, KgCfg<MODE, 1, 4, 1, 1, 2, 3>>(p, stream);
        case DT_64x64: return launch_dense_kgroup<Op, KgCfg<MODE, 1, 1, 4, 2, 2, 2>>(p, stream);
        case DT_128x64: return launch_dense_kgroup<Op, KgCfg<MODE, 4, 1, 2, 1, 2, 3 - M4>>(p, stream);
        case DT_128x128: return launch_dense_kgroup<Op, KgCfg<MODE, 4, 2, 1, 1, 2, 4>>(p, stream);
        case DT_128x256:
            if constexpr (!M4) return launch_dense_kgroup<Op, KgCfg<MODE, 2, 4, 1, 2, 2, 3>>(p, stream);
            break;
        case DT_64x128:
            if constexpr (Op::FUSED || Op::GATED) return launch_dense_kgroup<Op, KgCfg<MODE, 2, 2, 2, 1, 2, 3>>(p, stream);
            break;
        case DT_192x256:
            if constexpr (Op::FUSED || Op::GATED) return launch_dense_mid<Op, MODE>(p, stream);
            break;
        case DT_128x128_PAIR:
            return launch_dense_tiles<Op, MODE, 2, 2, 2, 2, 128, 2>(p, 1, p.kbytes / 128, nullptr, stream);
        case DT_SPLIT:
            // one workgroup per CU where the splits allow, on a deeper ring
            // (two K-tiles of loads in flight or more)
            if constexpr (!M4 && !Op::GATED) {
                const int ncu = cu_count() > 0 ? cu_count() : 256;
                const bool one_round = pl.tiles * pl.splits <= ncu;
                const int S = pl.splits, kt = pl.kt_split;
                if constexpr (MODE == MODE_A8W8)
                    if (pl.geo == GEO_128x64) {
                        if (!one_round) return launch_dense_tiles<Op, MODE, 4, 1, 1, 2, 128, 2>(p, S, kt, ws, stream);
                        if (kt >= 6) return launch_dense_tiles<Op, MODE, 4, 1, 1, 2, 128, 1, 6>(p, S, kt, ws, stream);
                        return launch_dense_tiles<Op, MODE, 4, 1, 1, 2, 128, 1, 3>(p, S, kt, ws, stream);
                    }
                if (!one_round) return launch_dense_tiles<Op, MODE, 2, 2, 2, 2, 128, 2>(p, S, kt, ws, stream);
                return launch_dense_tiles<Op, MODE, 2, 2, 2, 2, 128, 1, 4>(p, S, kt, ws, stream);
            }
            break;
        case DT_NONE:
            HKQ_CHECK_ARG(false, PITCH_REFUSAL);
    }
    // 128-byte K-tiles of this kernel need whole ones in every row: a partial
    // last K-tile would read the next row's bytes instead of zeros
    return p.kbytes % 128 == 0 ? launch_dense_whole<Op, MODE, 128>(p, stream) : launch_dense_whole<Op, MODE, 64>(p, stream);
}

}  // namespace hkq
