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
//
// Few rows are bound by the weights' way from memory (48 rows of 8 groups 4096x14336: 175
// us, 5.3 TB/s; 6006 rows of 64 groups 2816x2048: 165 to 174 us, 4.6 TB/s), many by the
// matrix cores (8192 rows of 8 groups 28672x4096: 1550 to 1610 us, 1.2 PFLOP/s, dX 1760 to
// 1790, dW 1640; the dense product of one group 1340). Few outputs with long sums leave CUs
// idle, as a workgroup walks its whole sum (dX of 3 rows, N 8160, K 640: 37 us).
#include <algorithm>
#include <cmath>

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
    int64_t ldc;                 // values; 16-byte pieces of C are aligned (pitch, stride and base are checked)
    int tiles_m, tiles_n, group_m;  // tiles_m: Y, dX: the most there can be
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
                                      wg / Cfg::WN * Cfg::TM * 32, n0 + wg % Cfg::WN * Cfg::TN * 32, true, NoScale{},
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
                                        true, NoScale{}, NoScale{}, NoBias{});
}

// dW: tile (tm, tn) of group e's [K columns of dY] x [N columns of X], summed over
// the group's rows; zeros where it has none.
struct DwTile {
    int e, m0, n0, start, rows;
};
template <int BM, int BN, class Rows>
__device__ __forceinline__ DwTile dw_tile(const GroupedParams& p, int id, Rows group) {
    const int per = p.tiles_m * p.tiles_n;
    DwTile t;
    t.e = id / per;
    // every group's tiles over all XCDs: groups differ in rows
    tile_coords(id - t.e * per, p.tiles_m, p.tiles_n, p.group_m, t.m0, t.n0);
    t.m0 *= BM;
    t.n0 *= BN;
    const int2 r = group(t.e);
    t.start = __builtin_amdgcn_readfirstlane(r.x);
    t.rows = __builtin_amdgcn_readfirstlane(r.y) - t.start;
    return t;
}
template <class Cfg, int MINB>
__global__ __launch_bounds__(Cfg::THREADS, MINB) void grouped_dw_small_kernel(const GroupedParams p) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem_raw[];
    HKQ_LDS uint8_t* smem = (HKQ_LDS uint8_t*)smem_raw;
    const DwTile t = dw_tile<Cfg::BM, Cfg::BN>(p, blockIdx.x, [&](int e) { return group_rows(p, e); });
    v16f acc[Cfg::TN][Cfg::TM];
    small_tile<true, true, Cfg>(p.A + t.start * p.lda + t.m0 * 2, p.B + t.start * p.ldb + t.n0 * 2, p.lda, p.ldb,
                                min(p.K - t.m0, Cfg::BM), min(p.N - t.n0, Cfg::BN), t.rows, smem, acc);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wg = wave % Cfg::GW;
    if (wave >= Cfg::GW) return;
    store_tile_bf16<Cfg::TM, Cfg::TN>(acc, smem, wg, threadIdx.x & 63, p.C + t.e * p.stride_e, p.ldc, p.K, p.N,
                                      t.m0 + wg / Cfg::WN * Cfg::TM * 32, t.n0 + wg % Cfg::WN * Cfg::TN * 32, true,
                                      NoScale{}, NoScale{}, NoBias{});
}
__global__ __launch_bounds__(256, 1) void grouped_dw_whole_kernel(const GroupedParams p) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem_raw[];
    HKQ_LDS uint8_t* smem = (HKQ_LDS uint8_t*)smem_raw;
    const DwTile t = dw_tile<DENSE_BM, DENSE_BN>(p, blockIdx.x, [&](int e) { return group_rows(p, e); });
    v16f acc[DENSE_TN][DENSE_TM];
    whole_tile<true, true>(p.A + t.start * p.lda + t.m0 * 2, p.B + t.start * p.ldb + t.n0 * 2, p.lda, p.ldb,
                           min(p.K - t.m0, DENSE_BM), min(p.N - t.n0, DENSE_BN), t.rows, smem, acc);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    store_tile_bf16<DENSE_TM, DENSE_TN>(acc, smem, wave, threadIdx.x & 63, p.C + t.e * p.stride_e, p.ldc, p.K, p.N,
                                        t.m0 + wave / DENSE_WAVES_N * DENSE_TM * 32, t.n0 + wave % DENSE_WAVES_N * DENSE_TN * 32,
                                        true, NoScale{}, NoScale{}, NoBias{});
}

// ---------------------------------------------------------------------------
// Large groups: one workgroup per CU computes its 256 x 256 tiles as one stream of
// K-tiles (gemm_stream.h), so that a tile's stores run under the next one's loads (dW's,
// 128 KB from each CU after 16 K-tiles of a group of 1024 rows, in part only). The
// groups' tile counts go to LDS at the start, where each tile's group is looked up.
// ---------------------------------------------------------------------------
constexpr int STREAM_GROUPS = 512;  // groups that the LDS table holds
constexpr int STREAM_TABLE = stream_stg_off<PlainOp, MODE_BF16>() + DENSE_WAVES_M * DENSE_WAVES_N * STREAM_STG;
constexpr int STREAM_LDS = STREAM_TABLE + 3 * STREAM_GROUPS * 4 + 16;
static_assert(STREAM_LDS <= 160 * 1024, "LDS budget of a CDNA4 CU");
// a wave may load its half tile's K-tiles while another still looks its own up in the table
static_assert(DenseCfg<MODE_BF16, DENSE_WAVES_M, DENSE_WAVES_N, DENSE_TM / 2, DENSE_TN, 128>::lds_bytes(HALF_NS) <= STREAM_TABLE,
              "a half tile's ring ends before the table");

struct GroupTable {
    HKQ_LDS int *end, *row0, *row1;  // row tiles up to the group's end (512 x 2^20 at the most), its rows
    int E;
    // fills the table; the tiles of all groups (every wave; ends in a barrier)
    __device__ int fill(const GroupedParams& p, HKQ_LDS uint8_t* at) {
        end = reinterpret_cast<HKQ_LDS int*>(at);
        row0 = end + STREAM_GROUPS;
        row1 = row0 + STREAM_GROUPS;
        E = p.E;
        HKQ_LDS int* total = row1 + STREAM_GROUPS;
        if (threadIdx.x < 64) {
            const int lane = threadIdx.x;
            int before = 0;
            for (int e0 = 0; e0 < E; e0 += 64) {
                const int e = e0 + lane;
                int2 r = make_int2(0, 0);
                if (e < E) r = group_rows(p, e);
                int s = (r.y - r.x + DENSE_BM - 1) / DENSE_BM;
#pragma unroll
                for (int d = 1; d < 64; d *= 2) {
                    const int o = __shfl_up(s, d, 64);
                    if (lane >= d) s += o;
                }
                if (e < E) end[e] = before + s, row0[e] = r.x, row1[e] = r.y;
                before += __builtin_amdgcn_readlane(s, 63);
            }
            if (lane == 0) *total = min(before, p.tiles_m);  // bounds that count a row twice: the most there can be
        }
        __syncthreads();
        return __builtin_amdgcn_readfirstlane(*total);
    }
    // tile id of total * tiles_n: its group, first row and the group's rows from there on,
    // and its column tile
    __device__ __forceinline__ void find(const GroupedParams& p, int id, int total, int& e, int& m0, int& rows, int& tn) const {
        const int lane = threadIdx.x & 63;
        id = xcd_order(id, total * p.tiles_n);
        const int at = id / p.tiles_n;
        e = 0;
        for (int e0 = 0; e0 < E; e0 += 64) {
            const uint64_t past = __ballot(e0 + lane < E && end[min(e0 + lane, E - 1)] > at);
            if (past) {
                e = e0 + __builtin_ctzll(past);
                break;
            }
        }
        const int r0 = __builtin_amdgcn_readfirstlane(row0[e]), r1 = __builtin_amdgcn_readfirstlane(row1[e]);
        const int tiles = max(1, (r1 - r0 + DENSE_BM - 1) / DENSE_BM), first = __builtin_amdgcn_readfirstlane(end[e]) - tiles;
        int tm;
        group_tile(id - first * p.tiles_n, tiles, p.tiles_n, p.group_m, tm, tn);
        m0 = r0 + tm * DENSE_BM;
        rows = r1 - m0;
    }
};

template <bool BT>
struct RaggedSeq {
    static constexpr bool GATHER = false;
    const GroupedParams* p;
    GroupTable table;
    int tiles, KT;
    uint32_t lsa, lsb;
    int total, first, stride;
    __device__ void at(int k, int& e, int& m0, int& rows, int& n0) const {
        table.find(*p, first + k * stride, total, e, m0, rows, n0);
        n0 *= DENSE_BN;
    }
    __device__ StreamSrc src(int k) const {
        int e, m0, rows, n0;
        at(k, e, m0, rows, n0);
        const int cols = min(p->N - n0, DENSE_BN);
        StreamSrc s{};
        s.a = p->A + m0 * p->lda;
        s.a_bytes = clamp_bytes((int64_t)(min(rows, DENSE_BM) - 1) * p->lda + p->K * 2);
        s.b = p->B + e * p->stride_e + (BT ? n0 * 2 : n0 * p->ldb);
        s.b_bytes = clamp_bytes((int64_t)(cols - 1) * p->ldb + p->K * 2);
        if constexpr (BT) s.tb = T16Src::of(s.b, p->ldb, cols, 0, p->K, KT);
        return s;
    }
};
struct DwSeq {
    static constexpr bool GATHER = false, VARIES = true;
    const GroupedParams* p;
    GroupTable table;
    int tiles, KT;
    uint32_t lsa, lsb;
    int first, stride;
    __device__ DwTile at(int k) const {
        return dw_tile<DENSE_BM, DENSE_BN>(*p, first + k * stride, [&](int e) { return make_int2(table.row0[e], table.row1[e]); });
    }
    __device__ int kt_live(int k) const { return (at(k).rows + 63) / 64; }
    __device__ int kt(int k) const { return max(4, (kt_live(k) + 1) / 2 * 2); }
    __device__ StreamSrc src(int k) const {
        const DwTile t = at(k);
        const int n = (t.rows + 63) / 64;
        StreamSrc s{};
        s.ta = T16Src::of(p->A + t.start * p->lda + t.m0 * 2, p->lda, min(p->K - t.m0, DENSE_BM), 0, t.rows, n);
        s.tb = T16Src::of(p->B + t.start * p->ldb + t.n0 * 2, p->ldb, min(p->N - t.n0, DENSE_BN), 0, t.rows, n);
        return s;
    }
};
template <bool DW, class Seq>
struct GroupedEpi {
    static constexpr int TM = DENSE_TM, TN = DENSE_TN, VM_ISSUED = TN * TM * 2;
    const Seq* seq;
    HKQ_LDS uint8_t* stg;
    int lane, wave;
    __device__ void begin(int) {}
    __device__ void end(int k, v16f (&acc)[TN][TM]) {
        const GroupedParams& p = *seq->p;
        const int mw = wave / DENSE_WAVES_N * TM * 32, nw = wave % DENSE_WAVES_N * TN * 32;
        uint16_t* c;
        int rows, cols;
        if constexpr (DW) {
            const DwTile t = seq->at(k);
            c = p.C + t.e * p.stride_e + t.m0 * p.ldc + t.n0;
            rows = p.K - t.m0, cols = p.N - t.n0;
        } else {
            int e, m0, n0;
            seq->at(k, e, m0, rows, n0);
            c = p.C + m0 * p.ldc + n0;
            cols = p.N - n0;
        }
        float one[TM];
#pragma unroll
        for (int j = 0; j < TM; ++j) one[j] = 1.0f;
        stream_store_tile<TM, TN>(acc, stg, c + mw * p.ldc + nw, p.ldc, rows - mw, cols - nw, one,
                                  [](int, int) { return v4f{1.f, 1.f, 1.f, 1.f}; }, lane);
    }
};

// The M half `half` of row tile (e, m0), column tile n0.
template <bool BT>
__device__ __forceinline__ void grouped_half(const GroupedParams& p, int e, int m0, int rows, int n0, int half, HKQ_LDS uint8_t* smem) {
    using Op = TransOp<false, BT>;
    using Half = DenseCfg<MODE_BF16, DENSE_WAVES_M, DENSE_WAVES_N, DENSE_TM / 2, DENSE_TN, 128>;
    DenseParams d{};
    d.A = p.A + m0 * p.lda;
    d.B = p.B + e * p.stride_e;
    d.C = p.C + m0 * p.ldc;
    d.M = rows; d.N = p.N; d.K = p.K; d.kbytes = p.K * 2;
    d.lda = p.lda; d.ldb = p.ldb; d.ldc = p.ldc;
    d.c16 = 1;
    dense_rows<Op, MODE_BF16, DENSE_TM / 2, 128, HALF_NS, Half::lds_bytes(HALF_NS)>(d, half * Half::BM, n0, smem);
}

// Where the last round of tiles would leave half of the CUs idle or more, its tiles run
// as M halves, by workgroups b with b / 16 * 8 + b % 8 the tile and b / 8 % 2 the half
// (both on one XCD). All of them last: an XCD's workgroups stay side by side in K and
// share their rows and columns in its L2. With every second half first, so that the tiles'
// ends fall between the others', 8192 rows of 8 groups 28672x4096 took 1606 us (1555 in the
// same run) and their dX, 448 K-tiles a tile, 1960 with 7.7 GB fetched (1760 to 1790).
template <bool BT>
__global__ __launch_bounds__(256, 1) void grouped_stream_kernel(const GroupedParams p) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem_raw[];
    HKQ_LDS uint8_t* smem = (HKQ_LDS uint8_t*)smem_raw;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    GroupTable table;
    const int total = table.fill(p, smem + STREAM_TABLE);
    const int b = blockIdx.x, G = gridDim.x, tiles = total * p.tiles_n, last = tiles % G;
    const int split = last > 0 && (last + 7) / 8 * 16 <= G ? last : 0, whole = tiles - split;
    const int mine = b < whole ? (whole - 1 - b) / G + 1 : 0;
    const int t = 8 * (b >> 4) + (b & 7);
    if (mine > 0) {
        using Cfg = DenseCfg<MODE_BF16, DENSE_WAVES_M, DENSE_WAVES_N, DENSE_TM, DENSE_TN, 128>;
        RaggedSeq<BT> seq{&p, table, mine, p.K / 64, 0, 0, total, b, G};
        GroupedEpi<false, RaggedSeq<BT>> epi{&seq, smem + stream_stg_off<PlainOp, MODE_BF16>() + wave * STREAM_STG, lane, wave};
        auto a_off = dense_offs<Cfg::NW, 128, Cfg::LA>(wave, lane, p.lda);
        auto b_off = dense_offs<Cfg::NW, 128, Cfg::LB>(wave, lane, p.ldb);
        if constexpr (BT) b_off = dense_offs_t16<Cfg::NW, Cfg::LB, Cfg::BN>(wave, lane, p.ldb);
        v16f acc[DENSE_TN][DENSE_TM];
        gemm_stream<MODE_BF16, DENSE_WAVES_M, DENSE_WAVES_N, DENSE_TM, DENSE_TN, BT>(seq, a_off, b_off, smem, lane, wave, acc, epi);
    }
    if (t < split) {
        int e, m0, rows, tn;
        table.find(p, whole + t, total, e, m0, rows, tn);
        grouped_half<BT>(p, e, m0, rows, tn * DENSE_BN, (b >> 3) & 1, smem);
    }
}
__global__ __launch_bounds__(256, 1) void grouped_dw_stream_kernel(const GroupedParams p) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem_raw[];
    HKQ_LDS uint8_t* smem = (HKQ_LDS uint8_t*)smem_raw;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    using Cfg = DenseCfg<MODE_BF16, DENSE_WAVES_M, DENSE_WAVES_N, DENSE_TM, DENSE_TN, 128>;
    const int b = blockIdx.x, G = gridDim.x, tiles = p.tiles_m * p.tiles_n * p.E;
    GroupTable table;
    table.fill(p, smem + STREAM_TABLE);
    if (b >= tiles) return;
    DwSeq seq{&p, table, (tiles - 1 - b) / G + 1, 0, 0, 0, b, G};
    GroupedEpi<true, DwSeq> epi{&seq, smem + stream_stg_off<PlainOp, MODE_BF16>() + wave * STREAM_STG, lane, wave};
    auto a_off = dense_offs_t16<Cfg::NW, Cfg::LA, Cfg::BM>(wave, lane, p.lda);
    auto b_off = dense_offs_t16<Cfg::NW, Cfg::LB, Cfg::BN>(wave, lane, p.ldb);
    v16f acc[DENSE_TN][DENSE_TM];
    gemm_stream<MODE_BF16, DENSE_WAVES_M, DENSE_WAVES_N, DENSE_TM, DENSE_TN, true, true>(seq, a_off, b_off, smem, lane, wave, acc, epi);
}

template <bool BT, class Kern>
static int launch_grouped(Kern kern, std::atomic<uint64_t>& attr, int lds, int bm, int bn, int threads, GroupedParams& p,
                          hipStream_t stream) {
    if (int e = set_device_lds(kern, lds, attr)) return e;
    p.tiles_m = (int)ragged_most(p.M, p.E, bm);
    p.group_m = 8;
    return launch_columns(
        p, bn, threads, [](GroupedParams& q, int64_t n) { q.B += BT ? 2 * n : n * q.ldb, q.C += n; },
        [&](const GroupedParams& q, unsigned blocks) { kern<<<blocks, threads, lds, stream>>>(q); });
}
template <bool BT, class Cfg, int MINB = 1>
static int launch_small(GroupedParams& p, hipStream_t stream) {
    static_assert(Cfg::LDS * MINB <= 160 * 1024, "LDS budget of a CDNA4 CU");
    static std::atomic<uint64_t> attr{0};
    return launch_grouped<BT>(grouped_small_kernel<BT, Cfg, MINB>, attr, Cfg::LDS, Cfg::BM, Cfg::BN, Cfg::THREADS, p, stream);
}
template <bool BT>
static int launch_whole(GroupedParams& p, hipStream_t stream) {
    const int ncu = cu_count();
    if (ncu > 0 && p.E <= STREAM_GROUPS && p.K % 128 == 0 && p.K >= 256) {
        p.tiles_m = (int)ragged_most(p.M, p.E, DENSE_BM);
        p.tiles_n = (p.N + DENSE_BN - 1) / DENSE_BN;
        p.group_m = 8;
        if ((int64_t)p.tiles_m * p.tiles_n < (1 << 23)) {
            auto kern = grouped_stream_kernel<BT>;
            static std::atomic<uint64_t> attr{0};
            if (int e = set_device_lds(kern, STREAM_LDS, attr)) return e;
            kern<<<ncu, 256, STREAM_LDS, stream>>>(p);
            return hkq_launch_status();
        }
    }
    static std::atomic<uint64_t> attr{0};
    return launch_grouped<BT>(grouped_whole_kernel<BT>, attr, WHOLE_LDS, DENSE_BM, DENSE_BN, 256, p, stream);
}
// (a launch takes as many groups as keep it below 2^32 threads; one group's tiles do, as its
// gradient fits the memory)
template <class Kern>
static int launch_dw(Kern kern, std::atomic<uint64_t>& attr, int lds, int bm, int bn, int threads, const GroupedParams& p,
                     hipStream_t stream) {
    if (int e = set_device_lds(kern, lds, attr)) return e;
    GroupedParams q = p;
    q.tiles_m = (p.K + bm - 1) / bm;
    q.tiles_n = (p.N + bn - 1) / bn;
    q.group_m = 8;
    const int64_t per = (int64_t)q.tiles_m * q.tiles_n, most = 0xFFFFFFFFll / threads / per;
    HKQ_CHECK_ARG(most > 0, "too many tiles for one launch");
    for (int64_t e = 0; e < p.E; e += most) {
        q.E = (int)std::min<int64_t>(p.E - e, most);
        q.offs = p.offs + e;
        q.C = p.C + e * p.stride_e;
        kern<<<(unsigned)(per * q.E), threads, lds, stream>>>(q);
        if (int err = hkq_launch_status()) return err;
    }
    return 0;
}

// Tile size by the mean rows of a group: the least estimated time. A K-tile takes
// us + c * share with c workgroups on a CU; groups need about half a row tile more than
// their rows fill. Fitted to 5 sizes x 62 shapes (1 to 1024 rows in each of 8 or 64
// groups, N and K 1408 to 28672, Y and dX): 1.03 of the best size's time on average, 1.20
// at the most; smaller N and K and fewer groups lie outside the fit. What a size is for,
// Y in us:
//   64 groups 2816x2048, 4 rows:    64x64 127, 64x128 133, 128x256 142, 256x256 158
//   8 groups 4096x14336, 64 rows:   128x128 190, 64x128 240, 128x256 249, 256x256 235
//   8 groups 28672x4096, 1024 rows: 256x256 1546, 128x256 1806, 128x128 2226, 64x64 3560
struct RaggedSize {
    int bm, bn, slots;  // slots: workgroups per CU
    float us, share, e;  // e: start and epilogue
};
template <bool BT>
static int run_ragged(GroupedParams& p, hipStream_t stream) {
    static const RaggedSize S[] = {{256, 256, 1, 0.43f, 0.63f, 13.2f}, {128, 256, 1, 0.40f, 0.50f, 5.2f},
                                   {128, 128, 1, 0.28f, 0.32f, 1.4f}, {64, 128, 2, 0.15f, 0.34f, 1.6f},
                                   {64, 64, 3, 0.38f, 0.14f, 0.3f}};
    const double ncu = cu_count() > 0 ? cu_count() : 256;
    const double KT = (p.K + 63) / 64, live = (double)std::min(p.M, p.E), r = p.M / live;
    int best = 0;
    double best_us = 0;
    for (int i = 0; i < 5; ++i) {
        const RaggedSize& s = S[i];
        const double tiles = live * std::max(1.0, r / s.bm + 0.5) * ((p.N + s.bn - 1) / s.bn);
        auto round = [&](int c) { return c == 0 ? 0.0 : KT * (s.us + s.share * c) + s.e; };
        const double per = tiles / ncu;  // tiles of a CU
        const int full = (int)std::min(per / s.slots, 2.0);
        const double us = full == 2 ? (per / s.slots + 0.5) * round(s.slots)
                                    : full * round(s.slots) + round((int)std::ceil(per - full * s.slots - 1e-9));
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
    const int64_t ncu = cu_count() > 0 ? cu_count() : 256;
    const int64_t tiles = (int64_t)((p.K + 255) / 256) * ((p.N + 255) / 256) * p.E;
    if (tiles >= ncu && p.E <= STREAM_GROUPS && tiles < (1 << 23)) {
        p.tiles_m = (p.K + DENSE_BM - 1) / DENSE_BM;
        p.tiles_n = (p.N + DENSE_BN - 1) / DENSE_BN;
        p.group_m = 8;
        static std::atomic<uint64_t> attr{0};
        if (int e = set_device_lds(grouped_dw_stream_kernel, STREAM_LDS, attr)) return e;
        grouped_dw_stream_kernel<<<(unsigned)ncu, 256, STREAM_LDS, stream>>>(p);
        return hkq_launch_status();
    }
    if (tiles >= ncu) {
        static std::atomic<uint64_t> attr{0};
        return launch_dw(grouped_dw_whole_kernel, attr, WHOLE_LDS, DENSE_BM, DENSE_BN, 256, p, stream);
    }
    using Cfg = KgCfg<MODE_BF16, 4, 2, 1, 1, 2, 4>;
    static std::atomic<uint64_t> attr{0};
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
