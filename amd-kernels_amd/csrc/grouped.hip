// grouped.hip -- bf16 matrix products over ragged groups of rows (the experts of a
// mixture), and their gradients:
//
//   hkq_grouped_gemm_bf16      Y[r, :] = X[r, :] . W[e]^T  for offs[e] <= r < offs[e + 1]
//   hkq_grouped_gemm_backward  dX[r, :] = dY[r, :] . W[e],  dW[e] = sum over r of dY[r]^T X[r]
//
// The groups' bounds are on the GPU: a launch has a workgroup for every tile that
// M rows in E groups can need, and each finds its group from the bounds (ragged_tile).
// K loops and tiles are the dense GEMMs'; in dX and dW the operands whose K runs
// across memory rows are read transposed from LDS, so that nothing is copied.
#include <algorithm>

#include "gemm_dense.h"
#include "ragged.h"

namespace hkq {

struct GroupedParams {
    const uint8_t* A;  // rows of the groups
    const uint8_t* B;  // Y, dX: group e's weight; dW: rows of the groups
    uint16_t* C;
    const int32_t* offs;
    int M, E, N, K;  // C has N columns; K: the length of the sums (Y, dX), the columns of A (dW)
    int64_t lda, ldb, stride_e;  // bytes; stride_e: group to group, of B (Y, dX) or C (dW, values)
    int64_t ldc;                 // values
    int tiles_m, tiles_n, group_m, c16;  // tiles_m: Y, dX: the most there can be
};

struct NoScale {
    __device__ float operator()(int) const { return 1.0f; }
    __device__ float4 operator()(int, int) const { return make_float4(1.f, 1.f, 1.f, 1.f); }
};

// One tile of C = A . B^T on the small tiles' K loop: rows_a / rows_b live rows of
// the operands, kt K-tiles of 64 values, tail_chunk 16-byte chunks in the last one
// where an operand is K-contiguous.
template <bool AT, bool BT, class Cfg>
__device__ __forceinline__ void small_tile(const uint8_t* a, const uint8_t* b, int64_t lda, int64_t ldb, int rows_a, int rows_b,
                                           int K, HKQ_LDS uint8_t* smem, v16f (&acc)[Cfg::TN][Cfg::TM]) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wg = wave % Cfg::GW, kg = wave / Cfg::GW;
    KgSrc<Cfg> src;
    src.KT = (K + 63) / 64;
    src.half_tail = K % 64 != 0;
    src.tail_chunk = (K % 64 + 7) / 8;
    src.a = buffer_desc(a, clamp_bytes((int64_t)(rows_a - 1) * lda + K * 2));
    src.b = buffer_desc(b, clamp_bytes((int64_t)(rows_b - 1) * ldb + K * 2));
#pragma unroll
    for (int i = 0; i < Cfg::SWP; ++i) {
        const int r = kg_row<Cfg>(i, wg, lane);
        src.a_off[i] = (uint32_t)(r * lda) + kg_chunk<Cfg>(r, lane);
        src.b_off[i] = (uint32_t)(r * ldb) + kg_chunk<Cfg>(r, lane);
    }
    src.a_step = (uint32_t)(8 * Cfg::GW * Cfg::SWP * lda);
    src.b_step = (uint32_t)(8 * Cfg::GW * Cfg::SWP * ldb);
    src.bs_step = 0;
    src.sc_shift = 0;
    if constexpr (AT) {
        using T = KTileT16<Cfg::BM>;
        const int r = wg * T::ROWS_PER_LOAD + lane / (T::ROW / 16);
        src.ta = T16Src::of(a, lda, rows_a, 0, K, src.KT);
        src.a_off[0] = (uint32_t)(r * lda) + (uint32_t)(T::phys(r, lane % (T::ROW / 16)) << 4);
        src.a_step = (uint32_t)(Cfg::GW * T::ROWS_PER_LOAD * lda);
    }
    if constexpr (BT) {
        using T = KTileT16<Cfg::BN>;
        const int r = wg * T::ROWS_PER_LOAD + lane / (T::ROW / 16);
        src.tb = T16Src::of(b, ldb, rows_b, 0, K, src.KT);
        src.b_off[0] = (uint32_t)(r * ldb) + (uint32_t)(T::phys(r, lane % (T::ROW / 16)) << 4);
        src.b_step = (uint32_t)(Cfg::GW * T::ROWS_PER_LOAD * ldb);
    }
    kgroup_kloop<Cfg, false, false, AT, BT>(src, smem, lane, wg, kg, acc);
}

// The same for 256 x 256 tiles (4 waves of 128 x 128).
constexpr int WHOLE_LDS = DenseCfg<MODE_BF16, DENSE_WAVES_M, DENSE_WAVES_N, DENSE_TM, DENSE_TN, 128>::lds_bytes(2);
template <bool AT, bool BT>
__device__ __forceinline__ void whole_tile(const uint8_t* a, const uint8_t* b, int64_t lda, int64_t ldb, int rows_a, int rows_b,
                                           int K, HKQ_LDS uint8_t* smem, v16f (&acc)[DENSE_TN][DENSE_TM]) {
    using Cfg = DenseCfg<MODE_BF16, DENSE_WAVES_M, DENSE_WAVES_N, DENSE_TM, DENSE_TN, 128>;
    constexpr int NW = Cfg::NW;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    LoopSrc src{};
    src.KT = (K + 63) / 64;
    src.tail_chunk = K % 64 == 0 ? 8 : (K % 64 + 7) / 8;
    src.a = a;
    src.b = b;
    src.a_bytes = (int64_t)(rows_a - 1) * lda + K * 2;
    src.b_bytes = (int64_t)(rows_b - 1) * ldb + K * 2;
    auto a_off = dense_offs<NW, 128, Cfg::LA>(wave, lane, lda);
    auto b_off = dense_offs<NW, 128, Cfg::LB>(wave, lane, ldb);
    if constexpr (AT) {
        src.ta = T16Src::of(a, lda, rows_a, 0, K, src.KT);
        a_off = dense_offs_t16<NW, Cfg::LA, Cfg::BM>(wave, lane, lda);
    }
    if constexpr (BT) {
        src.tb = T16Src::of(b, ldb, rows_b, 0, K, src.KT);
        b_off = dense_offs_t16<NW, Cfg::LB, Cfg::BN>(wave, lane, ldb);
    }
    gemm_mainloop<MODE_BF16, DENSE_WAVES_M, DENSE_WAVES_N, DENSE_TM, DENSE_TN, 128, 2, BT, AT, false, !(AT && BT)>(
        src, a_off, b_off, smem, lane, wave, acc);
}

// Y and dX.
template <bool BT, class Cfg, int MINB>
__global__ __launch_bounds__(Cfg::THREADS, MINB) void grouped_small_kernel(const GroupedParams p) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem_raw[];
    HKQ_LDS uint8_t* smem = (HKQ_LDS uint8_t*)smem_raw;
    RaggedTile t;
    if (!ragged_tile<Cfg::BM>(p, t)) return;
    const int n0 = t.tn * Cfg::BN;
    const uint8_t* b = p.B + t.e * p.stride_e + (BT ? n0 * 2 : n0 * p.ldb);
    v16f acc[Cfg::TN][Cfg::TM];
    small_tile<false, BT, Cfg>(p.A + t.m0 * p.lda, b, p.lda, p.ldb, min(t.rows, Cfg::BM), min(p.N - n0, Cfg::BN), p.K, smem, acc);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wg = wave % Cfg::GW;
    if (wave >= Cfg::GW) return;
    store_tile_bf16<Cfg::TM, Cfg::TN>(acc, smem, wg, threadIdx.x & 63, p.C + t.m0 * p.ldc, p.ldc, t.rows, p.N,
                                      wg / Cfg::WN * Cfg::TM * 32, n0 + wg % Cfg::WN * Cfg::TN * 32, p.c16 != 0, NoScale{},
                                      NoScale{}, NoBias{});
}
template <bool BT>
__global__ __launch_bounds__(256, 1) void grouped_whole_kernel(const GroupedParams p) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem_raw[];
    HKQ_LDS uint8_t* smem = (HKQ_LDS uint8_t*)smem_raw;
    RaggedTile t;
    if (!ragged_tile<DENSE_BM>(p, t)) return;
    const int n0 = t.tn * DENSE_BN;
    const uint8_t* b = p.B + t.e * p.stride_e + (BT ? n0 * 2 : n0 * p.ldb);
    v16f acc[DENSE_TN][DENSE_TM];
    whole_tile<false, BT>(p.A + t.m0 * p.lda, b, p.lda, p.ldb, min(t.rows, DENSE_BM), min(p.N - n0, DENSE_BN), p.K, smem, acc);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    store_tile_bf16<DENSE_TM, DENSE_TN>(acc, smem, wave, threadIdx.x & 63, p.C + t.m0 * p.ldc, p.ldc, t.rows, p.N,
                                        wave / DENSE_WAVES_N * DENSE_TM * 32, n0 + wave % DENSE_WAVES_N * DENSE_TN * 32,
                                        p.c16 != 0, NoScale{}, NoScale{}, NoBias{});
}

// dW: tile (tm, tn) of group e's [K columns of dY] x [N columns of X], summed over
// the group's rows; zeros where it has none.
struct DwTile {
    int e, m0, n0, start, rows;
};
template <int BM, int BN>
__device__ __forceinline__ DwTile dw_tile(const GroupedParams& p) {
    const int per = p.tiles_m * p.tiles_n, id = xcd_order(blockIdx.x, per * p.E);
    DwTile t;
    t.e = id / per;
    const int in = id - t.e * per, group = p.group_m * p.tiles_n, first = in / group * p.group_m,
              size = min(p.tiles_m - first, p.group_m), at = in % group;
    t.m0 = (first + at % size) * BM;
    t.n0 = at / size * BN;
    const int2 r = group_rows(p, t.e);
    t.start = r.x;
    t.rows = r.y - r.x;
    return t;
}
template <class Cfg, int MINB>
__global__ __launch_bounds__(Cfg::THREADS, MINB) void grouped_dw_small_kernel(const GroupedParams p) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem_raw[];
    HKQ_LDS uint8_t* smem = (HKQ_LDS uint8_t*)smem_raw;
    const DwTile t = dw_tile<Cfg::BM, Cfg::BN>(p);
    v16f acc[Cfg::TN][Cfg::TM];
    small_tile<true, true, Cfg>(p.A + t.start * p.lda + t.m0 * 2, p.B + t.start * p.ldb + t.n0 * 2, p.lda, p.ldb,
                                min(p.K - t.m0, Cfg::BM), min(p.N - t.n0, Cfg::BN), t.rows, smem, acc);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wg = wave % Cfg::GW;
    if (wave >= Cfg::GW) return;
    store_tile_bf16<Cfg::TM, Cfg::TN>(acc, smem, wg, threadIdx.x & 63, p.C + t.e * p.stride_e, p.ldc, p.K, p.N,
                                      t.m0 + wg / Cfg::WN * Cfg::TM * 32, t.n0 + wg % Cfg::WN * Cfg::TN * 32, p.c16 != 0,
                                      NoScale{}, NoScale{}, NoBias{});
}
__global__ __launch_bounds__(256, 1) void grouped_dw_whole_kernel(const GroupedParams p) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem_raw[];
    HKQ_LDS uint8_t* smem = (HKQ_LDS uint8_t*)smem_raw;
    const DwTile t = dw_tile<DENSE_BM, DENSE_BN>(p);
    v16f acc[DENSE_TN][DENSE_TM];
    whole_tile<true, true>(p.A + t.start * p.lda + t.m0 * 2, p.B + t.start * p.ldb + t.n0 * 2, p.lda, p.ldb,
                           min(p.K - t.m0, DENSE_BM), min(p.N - t.n0, DENSE_BN), t.rows, smem, acc);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    store_tile_bf16<DENSE_TM, DENSE_TN>(acc, smem, wave, threadIdx.x & 63, p.C + t.e * p.stride_e, p.ldc, p.K, p.N,
                                        t.m0 + wave / DENSE_WAVES_N * DENSE_TM * 32, t.n0 + wave % DENSE_WAVES_N * DENSE_TN * 32,
                                        p.c16 != 0, NoScale{}, NoScale{}, NoBias{});
}

template <class Kern>
static int launch_grouped(Kern kern, bool& attr, int lds, int bm, int bn, int threads, GroupedParams& p, hipStream_t stream) {
    if (int e = set_lds(kern, lds, attr)) return e;
    p.tiles_m = (int)ragged_most(p.M, p.E, bm);
    p.tiles_n = (p.N + bn - 1) / bn;
    p.group_m = 8;
    const int64_t blocks = (int64_t)p.tiles_m * p.tiles_n;
    HKQ_CHECK_ARG(blocks < (1 << 23), "too many tiles for one launch");
    kern<<<(unsigned)blocks, threads, lds, stream>>>(p);
    return hkq_launch_status();
}
template <bool BT, class Cfg, int MINB = 1>
static int launch_small(GroupedParams& p, hipStream_t stream) {
    static_assert(Cfg::LDS * MINB <= 160 * 1024, "LDS budget of a CDNA4 CU");
    static bool attr = false;
    return launch_grouped(grouped_small_kernel<BT, Cfg, MINB>, attr, Cfg::LDS, Cfg::BM, Cfg::BN, Cfg::THREADS, p, stream);
}
template <bool BT>
static int launch_whole(GroupedParams& p, hipStream_t stream) {
    static bool attr = false;
    return launch_grouped(grouped_whole_kernel<BT>, attr, WHOLE_LDS, DENSE_BM, DENSE_BN, 256, p, stream);
}
template <class Kern>
static int launch_dw(Kern kern, bool& attr, int lds, int bm, int bn, int threads, GroupedParams& p, hipStream_t stream) {
    if (int e = set_lds(kern, lds, attr)) return e;
    p.tiles_m = (p.K + bm - 1) / bm;
    p.tiles_n = (p.N + bn - 1) / bn;
    p.group_m = 8;
    const int64_t blocks = (int64_t)p.tiles_m * p.tiles_n * p.E;
    HKQ_CHECK_ARG(blocks < (1 << 23), "too many tiles for one launch");
    kern<<<(unsigned)blocks, threads, lds, stream>>>(p);
    return hkq_launch_status();
}

// Tile size by the mean rows of a group: the least of rounds over the CUs * (K-tiles
// * us + e).
struct RaggedSize {
    int bm, bn, slots;  // slots: workgroups per CU
    float us, e;
};
template <bool BT>
static int run_ragged(GroupedParams& p, hipStream_t stream) {
    p.c16 = p.ldc % 8 == 0 && reinterpret_cast<uintptr_t>(p.C) % 16 == 0;
    static const RaggedSize S[] = {{256, 256, 1, 1.37f, 5.7f}, {128, 256, 1, 0.85f, 3.2f}, {128, 128, 1, 0.57f, 2.2f},
                                   {64, 128, 2, 0.60f, 2.0f}, {64, 64, 3, 0.55f, 2.0f}};
    const int64_t ncu = cu_count() > 0 ? cu_count() : 256;
    const double KT = (p.K + 63) / 64, live = (double)std::min(p.M, p.E), r = p.M / live;
    int best = 0;
    double best_us = 0;
    for (int i = 0; i < 5; ++i) {
        const double tiles = live * std::max(1.0, r / S[i].bm + 0.5) * ((p.N + S[i].bn - 1) / S[i].bn);
        const double rounds = std::max(1.0, tiles / (double)(ncu * S[i].slots));
        const double us = rounds * (KT * S[i].us + S[i].e);
        if (best_us == 0 || us < best_us) best = i, best_us = us;
    }
    switch (best) {
        case 0: return launch_whole<BT>(p, stream);
        case 1: return launch_small<BT, KgCfg<MODE_BF16, 2, 4, 1, 2, 2, 3>>(p, stream);
        case 2: return launch_small<BT, KgCfg<MODE_BF16, 4, 2, 1, 1, 2, 4>>(p, stream);
        case 3: return launch_small<BT, KgCfg<MODE_BF16, 2, 4, 1, 1, 1, 3>, 2>(p, stream);
    }
    return launch_small<BT, KgCfg<MODE_BF16, 2, 2, 1, 1, 1, 3>, 3>(p, stream);
}
static int run_dw(GroupedParams& p, hipStream_t stream) {
    p.c16 = p.ldc % 8 == 0 && p.stride_e % 8 == 0 && reinterpret_cast<uintptr_t>(p.C) % 16 == 0;
    const int64_t ncu = cu_count() > 0 ? cu_count() : 256;
    const int64_t tiles = (int64_t)((p.K + 255) / 256) * ((p.N + 255) / 256) * p.E;
    if (tiles >= ncu) {
        static bool attr = false;
        return launch_dw(grouped_dw_whole_kernel, attr, WHOLE_LDS, DENSE_BM, DENSE_BN, 256, p, stream);
    }
    using Cfg = KgCfg<MODE_BF16, 4, 2, 1, 1, 2, 4>;
    static bool attr = false;
    return launch_dw(grouped_dw_small_kernel<Cfg, 1>, attr, Cfg::LDS, Cfg::BM, Cfg::BN, Cfg::THREADS, p, stream);
}

}  // namespace hkq

using namespace hkq;

// Dimensions and pitches that every product here takes.
static int check_grouped(int64_t M, int64_t E, int64_t N, int64_t K) {
    HKQ_CHECK_ARG(M >= 0 && E >= 0 && N >= 0 && K >= 0, "M, E, N, K must be >= 0");
    HKQ_CHECK_ARG(M < (1 << 28) && E < (1 << 16) && N < (1 << 22) && K < (1 << 22), "M must be < 2^28, E < 2^16, N and K < 2^22");
    HKQ_CHECK_ARG(N % 8 == 0 && K % 8 == 0, "N and K must be multiples of 8");
    return 0;
}
#define HKQ_CHECK_PITCH(ld, n) \
    HKQ_CHECK_ARG((ld) >= (n) && (ld) % 8 == 0 && (ld) < (1 << 22), #ld " must be >= " #n ", a multiple of 8 and < 2^22")

extern "C" int hkq_grouped_gemm_bf16(const void* X, const void* W, void* Y, const int32_t* offs, int64_t M, int64_t E, int64_t N,
                                     int64_t K, int64_t ldx, int64_t ldw, int64_t stride_we, int64_t ldy, hipStream_t stream) {
    if (int e = check_grouped(M, E, N, K)) return e;
    HKQ_CHECK_PITCH(ldx, K);
    HKQ_CHECK_PITCH(ldw, K);
    HKQ_CHECK_PITCH(ldy, N);
    HKQ_CHECK_ARG(stride_we >= 0 && stride_we % 8 == 0 && stride_we < (1ll << 40), "stride_we must be >= 0, a multiple of 8 and < 2^40");
    if (M == 0 || E == 0 || N == 0) return 0;
    HKQ_CHECK_ARG(Y && offs && (K == 0 || (X && W)), "X, W, Y and offs are required");
    HKQ_CHECK_ALIGN(X, 16);
    HKQ_CHECK_ALIGN(W, 16);
    HKQ_CHECK_ALIGN(Y, 16);
    HKQ_CHECK_ALIGN(offs, 4);
    const MemRows my{Y, M, 2 * N, 2 * ldy};
    HKQ_CHECK_ARG(!overlap(my, {X, M, 2 * K, 2 * ldx}) && !overlap(my, grouped_mem(W, E, N, 2 * K, 2 * ldw, 2 * stride_we)) &&
                      !overlap(my, {offs, 1, 4 * (E + 1), 0}),
                  "Y must not overlap X, W or offs");
    GroupedParams p{};
    p.A = static_cast<const uint8_t*>(X);
    p.B = static_cast<const uint8_t*>(W);
    p.C = static_cast<uint16_t*>(Y);
    p.offs = offs;
    p.M = (int)M; p.E = (int)E; p.N = (int)N; p.K = (int)K;
    p.lda = 2 * ldx; p.ldb = 2 * ldw; p.stride_e = 2 * stride_we; p.ldc = ldy;
    return run_ragged<false>(p, stream);
}

extern "C" int hkq_grouped_gemm_backward(const void* dY, const void* X, const void* W, void* dX, void* dW, const int32_t* offs,
                                         int64_t M, int64_t E, int64_t N, int64_t K, int64_t lddy, int64_t ldx, int64_t ldw,
                                         int64_t stride_we, int64_t lddx, int64_t lddw, int64_t stride_dwe, hipStream_t stream) {
    if (int e = check_grouped(M, E, N, K)) return e;
    HKQ_CHECK_PITCH(lddy, N);
    if (dX) {
        HKQ_CHECK_PITCH(ldw, K);
        HKQ_CHECK_PITCH(lddx, K);
        HKQ_CHECK_ARG(stride_we >= 0 && stride_we % 8 == 0 && stride_we < (1ll << 40),
                      "stride_we must be >= 0, a multiple of 8 and < 2^40");
    }
    if (dW) {
        HKQ_CHECK_PITCH(ldx, K);
        HKQ_CHECK_PITCH(lddw, K);
        HKQ_CHECK_ARG(stride_dwe >= 0 && stride_dwe % 8 == 0 && stride_dwe < (1ll << 40),
                      "stride_dwe must be >= 0, a multiple of 8 and < 2^40");
        HKQ_CHECK_ARG(E <= 1 || N <= 0 || stride_dwe >= (N - 1) * lddw + K || (stride_dwe >= K && lddw >= (E - 1) * stride_dwe + K),
                      "the groups of dW must not overlap each other");
    }
    if (M == 0 || E == 0) dX = nullptr;  // nothing of it to write
    if (K == 0 || N == 0) dW = nullptr;
    if (K == 0 || E == 0 || (!dX && !dW)) return 0;
    HKQ_CHECK_ARG(offs, "offs is required");
    HKQ_CHECK_ARG(M == 0 || N == 0 || (dY && (!dX || W) && (!dW || X)), "dY, and W for dX, X for dW, are required");
    HKQ_CHECK_ALIGN(dY, 16);
    HKQ_CHECK_ALIGN(X, 16);
    HKQ_CHECK_ALIGN(W, 16);
    HKQ_CHECK_ALIGN(dX, 16);
    HKQ_CHECK_ALIGN(dW, 16);
    HKQ_CHECK_ALIGN(offs, 4);
    const MemRows mdx{dX, M, 2 * K, 2 * lddx}, mdw = grouped_mem(dW, E, N, 2 * K, 2 * lddw, 2 * stride_dwe),
                  mdy{dY, M, 2 * N, 2 * lddy}, mx{X, M, 2 * K, 2 * ldx}, mw = grouped_mem(W, E, N, 2 * K, 2 * ldw, 2 * stride_we),
                  mo{offs, 1, 4 * (E + 1), 0};
    if (dX) {
        HKQ_CHECK_ARG(!overlap(mdx, mdy) && !overlap(mdx, mw) && !overlap(mdx, mo) && !(dW && overlap(mdx, mx)),
                      "dX must not overlap dY, X, W or offs");
    }
    if (dW) {
        HKQ_CHECK_ARG(!overlap(mdw, mdy) && !overlap(mdw, mx) && !overlap(mdw, mo) && !(dX && (overlap(mdw, mw) || overlap(mdw, mdx))),
                      "dW must not overlap dY, X, W, dX or offs");
    }
    GroupedParams p{};
    p.offs = offs;
    p.M = (int)M; p.E = (int)E;
    p.A = static_cast<const uint8_t*>(dY);
    p.lda = 2 * lddy;
    if (dX) {
        p.B = static_cast<const uint8_t*>(W);
        p.C = static_cast<uint16_t*>(dX);
        p.N = (int)K; p.K = (int)N;
        p.ldb = 2 * ldw; p.stride_e = 2 * stride_we; p.ldc = lddx;
        if (int e = run_ragged<true>(p, stream)) return e;
    }
    if (dW) {
        p.B = static_cast<const uint8_t*>(X);
        p.C = static_cast<uint16_t*>(dW);
        p.N = (int)K; p.K = (int)N;
        p.ldb = 2 * ldx; p.stride_e = stride_dwe; p.ldc = lddw;
        return run_dw(p, stream);
    }
    return 0;
}
