// w4_tile.hip -- many rows times 4-bit weights: tiles of BM rows and 256 (128) columns,
// four waves side by side, each with all rows and 32 TN columns of its own.
//
// K goes in units of 128 values. Rows of X (bf16), codes and scales of a unit are
// staged in LDS by LDS-direct loads, NS stages. A wave turns its columns' codes into
// bf16 operands in registers, so that a code is converted once per BM rows, while the
// matrix instructions (32 x 32 x 16) work on the n-tile before. INT4: a group's sums
// P start from zero and acc += P * scale once the group ends; a lane holds one
// column's sums (rows of X are the first operand), so that is one multiplier per
// group. MXFP4 scales go into the operands.
//
// Bound by the issue port that conversion and matrix instructions share, one wave per
// SIMD: 2048x4096x14336, groups of 128, 214 to 220 us (bf16 weights 206 to 209), with zero
// points 232; 6006 rows of 64 groups 2816x2048, groups of 64, 129 to 147 us, 1.5 tiles of 96
// rows for a group's 94. Fewer tiles than CUs leave the rest idle, K is not split:
// 128x4096x14336 59 us on 128 CUs (bf16 weights 38).
#include <cmath>
#include <type_traits>

#include "gemm_kgroup.h"
#include "w4_chain.h"
#include "w4_core.h"

namespace hkq {

// G: values per group, 0 for MXFP4 (32); Z: zero points
template <int G_, bool Z_, int TM_, int TN_, int NS_>
struct W4Tile {
    static constexpr bool Z = Z_;
    static constexpr int G = G_, TM = TM_, TN = TN_, NS = NS_, NW = 4;
    static constexpr bool MX = G == 0;
    static constexpr int BM = 32 * TM, BN = NW * TN * 32, SB = MX ? 1 : 2;
    static constexpr int NG = MX ? 4 : 128 / G;  // groups in a unit
    // A row's scales of a unit start at any multiple of SB bytes (its zero points at
    // any byte): the aligned dwords that hold them
    static constexpr int SD = (NG * SB + 4 - SB + 3) / 4, ZD = Z ? (NG + 3 + 3) / 4 : 0;
    static constexpr int XB = 2 * BM * 128, WB = BN * 64, STAGE = XB + WB + NW * (SD + ZD) * 256;
    static constexpr int LX = 2 * BM / 8 / NW, LW = BN / 16 / NW, NLD = LX + LW + SD + ZD;
    static constexpr int EP_PITCH = TN * 64 + 16, EP = NW * BM * EP_PITCH;
    static constexpr int LDS = NS * STAGE > EP ? NS * STAGE : EP;
    static constexpr int OCC = TM == 1 && 2 * LDS <= 160 * 1024 ? 2 : 1;  // workgroups per CU (larger ones would spill)
    static_assert(LDS <= 160 * 1024 && NS >= 3 && (NS - 2) * NLD <= 63, "LDS and vmcnt budget");
    static constexpr int PARTS = MX ? 1 : NG, CH = 8 / PARTS;  // chains of matrix instructions per n-tile and m-tile
};

template <int I, int N, class F>
__device__ __forceinline__ void for_each_from(F&& f) {
    if constexpr (I < N) {
        f(std::integral_constant<int, I>{});
        for_each_from<I + 1, N>(f);
    }
}
template <int N, class F>
__device__ __forceinline__ void for_each_int(F&& f) {
    for_each_from<0, N>(f);
}

template <class T>
__global__ __launch_bounds__(256, T::OCC) void w4_tile_kernel(const W4Params p) {
    constexpr int TM = T::TM, TN = T::TN, NS = T::NS, BM = T::BM, NW = T::NW, SB = T::SB, NG = T::NG, CH = T::CH;
    constexpr bool MX = T::MX;
    using KT = KTile<128>;
    using KW = KTile<64>;
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem_raw[];
    HKQ_LDS uint8_t* smem = (HKQ_LDS uint8_t*)smem_raw;
    const int lane = threadIdx.x & 63, ln = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    RaggedTile t;
    if (p.offs) {
        if (!ragged_tile<BM>(p, t)) return;
    } else {
        t.e = 0;
        tile_coords(blockIdx.x, p.tiles_m, p.tiles_n, p.group_m, t.m0, t.tn);
        t.m0 *= BM;
        t.rows = p.M - t.m0;
    }
    const int n0 = t.tn * T::BN, cols = min(p.N - n0, T::BN), groups = p.K >> p.glog2;

    // sources: X rows, codes, scales and zero points of the tile's columns
    const uint8_t* x0 = p.gather ? p.X : p.X + t.m0 * p.ldx;
    const v4i dx = buffer_desc(x0, (uint32_t)((p.gather ? p.T - 1 : min(t.rows, BM) - 1) * p.ldx + p.K * 2));
    uint32_t x_off[T::LX / 2];
    const int xc = KT::load_chunk(lane, wave * 8 + lane / 8);  // the lane's chunk of every row that it loads
#pragma unroll
    for (int i = 0; i < T::LX / 2; ++i) {
        const int r = (i * NW + wave) * 8 + lane / 8;
        int row = r < t.rows ? r : -1;
        if (p.gather && row >= 0) {
            const int id = p.gather[t.m0 + r];
            row = id < 0 || id / p.topk >= p.T ? -1 : id / p.topk;
        }
        x_off[i] = row >= 0 ? (uint32_t)(row * p.ldx) + (uint32_t)(xc * 16) : OOB;
    }
    const v4i dq = buffer_desc(p.Q + t.e * p.stride_q + n0 * p.ldq, (uint32_t)((cols - 1) * p.ldq + p.K / 2));
    uint32_t w_off[T::LW];
#pragma unroll
    for (int i = 0; i < T::LW; ++i) {
        const int r = (i * NW + wave) * 16 + lane / 4;
        w_off[i] = (uint32_t)(r * p.ldq) + (uint32_t)(KW::load_chunk(lane, r) * 16);
    }
    auto dwords = [&](const uint8_t* base, int bytes, uint32_t& rem) {  // whole aligned dwords around [base, base + bytes)
        rem = (uint32_t)(reinterpret_cast<uintptr_t>(base) & 3);
        return buffer_desc(base - rem, bytes > 0 ? (uint32_t)(rem + bytes + 3) & ~3u : 0u);
    };
    uint32_t s_rem, z_rem = 0;
    const int64_t s_at = t.e * p.stride_s + n0 * p.lds, s_n = (cols - 1) * p.lds + groups;
    const v4i ds = dwords(p.S + s_at * SB, (int)(s_n * SB), s_rem);
    v4i dz{};
    if constexpr (T::Z) dz = dwords(p.Z + s_at, (int)s_n, z_rem);
    const uint32_t s_col = (uint32_t)((wave * TN * 32 + lane % (TN * 32)) * p.lds);  // the lane's column, in scales

    const int units = (p.K + 127) / 128;
    // the lane's chunk of the last unit's halves: past K it reads nothing
    const int last_k = (units - 1) * 128 + xc * 8;
    const uint32_t x_tail[2] = {last_k < p.K ? 0u : OOB, last_k + 64 < p.K ? 0u : OOB};
    // load l of a unit's into a stage; past the last unit they read nothing
    auto issue = [&](int u, int stage, int l) {
        HKQ_LDS uint8_t* st = smem + stage * T::STAGE;
        const uint32_t dead = u < units ? 0u : OOB;
        if (l < T::LX) {
            const int half = l / (T::LX / 2), r = l % (T::LX / 2);
            lds_load16_s(dx, st + half * BM * 128 + (r * NW + wave) * 1024, x_off[r] | (u + 1 < units ? 0u : x_tail[half] | dead),
                         dead ? 0u : (uint32_t)(u * 256 + half * 128));
        } else if (l < T::LX + T::LW) {
            const int i = l - T::LX;
            lds_load16_s(dq, st + T::XB + (i * NW + wave) * 1024, w_off[i] | dead, dead ? 0u : (uint32_t)(u * 64));
        } else {
            const int d = l - T::LX - T::LW;
            HKQ_LDS uint8_t* sc = st + T::XB + T::WB + (wave * (T::SD + T::ZD) + d) * 256;
            if (d < T::SD) lds_load4_s(ds, sc, ((s_rem + (s_col + (uint32_t)(u * NG)) * SB) & ~3u) | dead, 4 * d);
            else lds_load4_s(dz, sc, ((z_rem + s_col + (uint32_t)(u * NG)) & ~3u) | dead, 4 * (d - T::SD));
        }
    };

    // an n-tile's codes of a unit
    constexpr int NS_ = MX ? 2 : NG;  // scales of a lane (MXFP4: its block of each half)
    struct Raw {
        uint32_t w[8];  // word s: values 16 s + 8 h .. of the unit (MXFP4: 64 (s / 4) + 32 h + 8 (s % 4))
        uint32_t sb[NS_], zb[T::Z ? NG : 1];  // dwords that hold them
        float s[NS_], z[T::Z ? NG : 1];
    };
    // scales and zero points are bytes at any offset in the staged dwords of the lane's
    // column: the first group's, of n-tile i and unit u
    auto scale_at = [&](int u, int i, uint32_t rem, int bytes) {
        return (rem + ((uint32_t)((wave * TN * 32 + i * 32 + ln) * p.lds) + (uint32_t)(u * NG)) * bytes) & 3;
    };
    auto read_raw = [&](int u, int stage, int i, Raw& r) {
        const HKQ_LDS uint8_t* st = smem + stage * T::STAGE;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const v4i v = lds_read16(st + T::XB + KW::swz((wave * TN + i) * 32 + ln, 2 * half + h));
#pragma unroll
            for (int q = 0; q < 4; ++q) r.w[4 * half + q] = (uint32_t)v[q];
        }
        const HKQ_LDS uint8_t* sc = st + T::XB + T::WB + wave * (T::SD + T::ZD) * 256 + (i * 32 + ln) * 4;
        const uint32_t s0 = scale_at(u, i, s_rem, SB) + (MX ? h : 0), z0 = T::Z ? scale_at(u, i, z_rem, 1) : 0;
#pragma unroll
        for (int g = 0; g < NS_; ++g) r.sb[g] = *reinterpret_cast<const HKQ_LDS uint32_t*>(sc + ((s0 + 2 * g) >> 2) * 256);
        if constexpr (T::Z) {
#pragma unroll
            for (int g = 0; g < NG; ++g)
                r.zb[g] = *reinterpret_cast<const HKQ_LDS uint32_t*>(sc + T::SD * 256 + ((z0 + g) >> 2) * 256);
        }
    };
    // the scales as numbers; the words of INT4 change places between the lane halves, so
    // that an instruction's 16 values lie in one group
    auto finish_raw = [&](int u, int i, Raw& r) {
        const uint32_t s0 = scale_at(u, i, s_rem, SB) + (MX ? h : 0), z0 = T::Z ? scale_at(u, i, z_rem, 1) : 0;
#pragma unroll
        for (int g = 0; g < NS_; ++g) {
            const uint32_t v = r.sb[g] >> (8 * ((s0 + 2 * g) & 3));
            if constexpr (MX) {
                const uint32_t e = u * NG + 2 * g + h < groups ? v & 255 : 0u;
                // 2^(e - 127): the conversion takes the exponent, 0 of a subnormal, 255 of a NaN
                r.s[g] = __uint_as_float(e << 23 | (e == 255 ? 0x400000u : 0u));
            } else {
                r.s[g] = u * NG + g < groups ? __uint_as_float(v << 16) : 0.0f;
                if constexpr (T::Z) r.z[g] = (float)(r.zb[g] >> (8 * ((z0 + g) & 3)) & 255);
            }
        }
        if constexpr (!MX) {
#pragma unroll
            for (int q = 0; q < 8; q += 4) {
                swap32(r.w[q], r.w[q + 1]);  // words 0 and 1 of the first 32 values | of the next
                swap32(r.w[q + 2], r.w[q + 3]);
                const uint32_t v = r.w[q + 1];
                r.w[q + 1] = r.w[q + 2], r.w[q + 2] = v;
            }
        }
    };
    // Values 4 half .. 4 half + 3 of word s as a matrix operand's (INT4 without zero
    // points: a sixteenth of each).
    auto operand_half = [&](const Raw& r, int s, int half, v4i& b) {
        v2i o;
        if constexpr (MX) o = half ? fp4_operand2<1>(r.w[s], r.s[s / 4]) : fp4_operand2<0>(r.w[s], r.s[s / 4]);
        else if constexpr (T::Z) o = half ? int4_operand2<1>(r.w[s], r.z[s / CH]) : int4_operand2<0>(r.w[s], r.z[s / CH]);
        else o = half ? int4_sixteenths<1>(r.w[s]) : int4_sixteenths<0>(r.w[s]);
        b[2 * half] = o[0], b[2 * half + 1] = o[1];
    };
    // fragment f of the rows: values 16 (f % 8) of the unit (chains of CH: the same order),
    // m-tile f / 8
    uint32_t a_at[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) a_at[s] = (uint32_t)(uintptr_t)smem + (uint32_t)KT::swz(ln, MX ? 4 * h + s : 2 * s + h);
    auto read_a = [&](const uint32_t (&at)[4], int f) {
        return lds_read16(reinterpret_cast<const HKQ_LDS uint8_t*>(
            (uintptr_t)(at[f & 3] + (uint32_t)(f % 8 / 4 * BM * 128 + f / 8 * 32 * 128))));
    };

    v16f acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j) acc[i][j] = v16f{};

#pragma unroll
    for (int u = 0; u < NS - 1; ++u)
#pragma unroll
        for (int l = 0; l < T::NLD; ++l) issue(u, u, l);
    tile_barrier<(NS - 2) * T::NLD>();
    constexpr int SLOTS = 8 * TM;
    v4i B[2][8], A[SLOTS];
    Raw raw;
    float sc[2][MX ? 2 : NG];  // the scales of the operands in B
    read_raw(0, 0, 0, raw);
    finish_raw(0, 0, raw);
#pragma unroll
    for (int s = 0; s < 8; ++s) {
        operand_half(raw, s, 0, B[0][s]), operand_half(raw, s, 1, B[0][s]);
        // (inside the loop a step's conversions are a step ahead of its matrix instructions)
        if constexpr (!MX && !T::Z) int4_sixteenths_settle(B[0][s]);
    }
#pragma unroll
    for (int g = 0; g < NS_; ++g) sc[0][g] = raw.s[g];
    int stage = 0;
    for_each_int<SLOTS>([&](auto f) { A[decltype(f)::value] = read_a(a_at, decltype(f)::value); });
    v16f P{}, Pq{};  // a chain's sums; the chain's before, and their scale
    float sq = 0.0f;
    // n-tile i of unit u: matrix instructions on B[cur], one per slot, and between them
    // the sums of the chain before into acc, the next n-tile's operands into B[cur ^ 1]
    // and, at the last n-tile, the next unit's rows in place of those just used
    auto step = [&](int u, auto ii, auto par) {
        constexpr int i = decltype(ii)::value, cur = decltype(par)::value;
        constexpr bool LAST = i == TN - 1;
        const int next_stage = stage + 1 == NS ? 0 : stage + 1;
        if constexpr (LAST) {
            // unit u + 1 resident; every wave past unit u - 1, whose stage takes unit u + NS - 1.
            // (Reads of unit u may be on their way: nothing writes there.)
            __builtin_amdgcn_s_waitcnt(waitcnt_imm((NS - 3) * T::NLD, 15));
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
        }
        const int refill = stage == 0 ? NS - 1 : stage - 1;
        uint32_t at[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) at[s] = a_at[s] + (uint32_t)(next_stage * T::STAGE);
        read_raw(LAST ? u + 1 : u, LAST ? next_stage : stage, (i + 1) % TN, raw);
        __builtin_amdgcn_sched_barrier(0);
        constexpr int LPS = (T::NLD + SLOTS / 2 - 1) / (SLOTS / 2);  // loads per slot, in the step's first half
        constexpr int FIRST = 4;  // slots before the codes have arrived
        auto slot = [&](auto fi) {
            constexpr int f = decltype(fi)::value, j = f / 8, s = f % 8, part = s / CH;
            if constexpr (MX) {
                acc[i][j] = mfma_bf16(A[f], B[cur][s], acc[i][j]);
            } else {
                P = mfma_bf16(A[f], B[cur][s], s % CH == 0 ? v16f{} : P);
                // sums of the chain before
                constexpr int pc = f < CH ? SLOTS - 1 : f / CH * CH - 1, pi = f < CH ? (i + TN - 1) % TN : i, pj = pc / 8;
#pragma unroll
                for (int e = chain_added(s % CH, CH); e < chain_added(s % CH + 1, CH); ++e)
                    acc[pi][pj][e] = __builtin_fmaf(Pq[e], sq, acc[pi][pj][e]);
            }
            if constexpr (LAST) {
                A[f] = read_a(at, f);
#pragma unroll
                for (int l = f * LPS; l < (f + 1) * LPS && l < T::NLD; ++l) issue(u + NS - 1, refill, l);
            }
            // one wave per SIMD: rows live in the accumulation registers, the others are full
            if constexpr (T::OCC == 1) asm volatile("" : "+a"(A[(f + 1) % SLOTS]));
            if constexpr (f == FIRST) finish_raw(LAST ? u + 1 : u, (i + 1) % TN, raw);
            constexpr int N = SLOTS - FIRST, p0 = f < FIRST ? 0 : (f - FIRST) * 16 / N, p1 = f < FIRST ? 0 : (f - FIRST + 1) * 16 / N;
#pragma unroll
            for (int q = p0; q < p1; ++q) operand_half(raw, q / 2, q % 2, B[cur ^ 1][q / 2]);
            if constexpr (!MX && s % CH == CH - 1) Pq = P, sq = sc[cur][part];
            __builtin_amdgcn_sched_barrier(0);
        };
        for_each_int<SLOTS>(slot);
#pragma unroll
        for (int g = 0; g < NS_; ++g) sc[cur ^ 1][g] = raw.s[g];
        if constexpr (LAST) stage = next_stage;
    };
    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;
    if constexpr (TN == 2) {
        for (int u = 0; u < units; ++u) {
            step(u, I0{}, I0{});
            step(u, I1{}, I1{});
        }
    } else {
        int u = 0;
        for (; u + 1 < units; u += 2) {
            step(u, I0{}, I0{});
            step(u + 1, I0{}, I1{});
        }
        if (u < units) step(u, I0{}, I0{});
    }
    if constexpr (!MX) {
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[TN - 1][TM - 1][e] = __builtin_fmaf(Pq[e], sq, acc[TN - 1][TM - 1][e]);
    }
    mfma_drain();
    tile_barrier<0>();

    // the wave's BM x (32 TN) values through LDS, then row pieces of 8
    HKQ_LDS uint8_t* ep = smem + wave * BM * T::EP_PITCH;
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j)
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
                constexpr float unit = MX || T::Z ? 1.0f : 16.0f;  // (sixteenths of the codes)
                const uint32_t v = pk_bf16(acc[i][j][e] * unit, acc[i][j][e + 1] * unit);
                const int m = j * 32 + 8 * (e / 4) + 4 * h + e % 4;
                *reinterpret_cast<HKQ_LDS uint16_t*>(ep + m * T::EP_PITCH + (i * 32 + ln) * 2) = (uint16_t)v;
                *reinterpret_cast<HKQ_LDS uint16_t*>(ep + (m + 1) * T::EP_PITCH + (i * 32 + ln) * 2) = (uint16_t)(v >> 16);
            }
    constexpr int SEGS = TN * 4, RPP = 64 / SEGS;
    const bool c16 = p.ldc % 8 == 0 && reinterpret_cast<uintptr_t>(p.C) % 16 == 0;
    const int seg = lane % SEGS, nw = n0 + wave * TN * 32 + seg * 8, left = p.N - nw;
#pragma unroll 4
    for (int r0 = 0; r0 < BM; r0 += RPP) {
        const int r = r0 + lane / SEGS;
        const v4i v = lds_read16(ep + r * T::EP_PITCH + seg * 16);
        if (r >= t.rows || left <= 0) continue;
        uint16_t* dst = p.C + (int64_t)(t.m0 + r) * p.ldc + nw;
        if (c16 && left >= 8) {
            __builtin_nontemporal_store(v, reinterpret_cast<v4i*>(dst));
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < left) dst[e] = (uint16_t)((uint32_t)v[e / 2] >> (16 * (e & 1)));
        }
    }
}

template <class T>
static int launch_tile(W4Params& p, hipStream_t stream) {
    auto kern = w4_tile_kernel<T>;
    static std::atomic<uint64_t> attr{0};
    if (int e = set_device_lds(kern, T::LDS, attr)) return e;
    p.tiles_m = (int)ragged_most(p.M, p.E, T::BM);
    p.group_m = 8;
    return launch_columns(p, T::BN, 256, w4_from_column<T::MX>,
                          [&](const W4Params& q, unsigned blocks) { kern<<<blocks, 256, T::LDS, stream>>>(q); });
}

// Tile sizes, and us per unit and per tile on MI355X: a wave's instructions, one wave per
// SIMD (4.8 cycles each beside 9.5 per matrix instruction), so that converting the codes
// counts as much as multiplying. Two workgroups of the smallest share a CU. Measured at
// 32, 64 x 128, 64, 96, 128 x 256 and 128 x 128 (us): 24x28672x4096 22.7, 26.7, 42, 47, 56,
// 35; 300x4096x14336 109, 82, 140, 153, 184, 107; 2048x4096x14336 486, 362, 317, 334, 238,
// 271; 6016 rows of 64 groups 2816x2048 169, 169, 149, 123, 141, 157. Over 64 shapes of 8
// and 64 groups, 20 to 1024 rows each, the choice takes 1.016 of the best size's time on
// average, 1.3 at the most.
static const struct {
    int bm, bn;
    float us, e;
} W4_TILES[] = {{32, 128, 0.58f, 1.6f}, {64, 128, 0.68f, 3.1f}, {64, 256, 1.39f, 2.3f}, {96, 256, 1.44f, 1.7f}, {128, 256, 1.67f, 2.3f},
                {128, 128, 1.16f, 1.5f}};

float w4_tile_plan(const W4Params& p, int& tile) {
    const int ncu = cu_count() > 0 ? cu_count() : 256, units = (p.K + 127) / 128;
    const double live = (double)std::min(p.M, p.E), r = p.M / live;
    float best = 0.f;
    for (int t = 0; t < 6; ++t) {
        const auto& c = W4_TILES[t];
        // groups need about half a tile more than their rows fill, and how many tiles that
        // makes is known to some 8 %: the mean of the whole rounds in that range
        const bool guess = p.offs && r / c.bm + 0.48 > 1.0;
        const double rows = guess ? live * (r / c.bm + 0.48) : p.offs ? live : (double)((p.M + c.bm - 1) / c.bm);
        const double tiles = rows * ((p.N + c.bn - 1) / c.bn);
        const bool pairs = t == 0 && tiles > ncu;  // two on a CU slow each other down
        double rounds = 0.0;
        for (int i = -2; i <= 2; ++i) rounds += 0.2 * std::ceil(tiles * (guess ? 1.0 + 0.04 * i : 1.0) / (pairs ? 2 * ncu : ncu) - 1e-9);
        const float us = (float)rounds * ((float)units * (pairs ? 0.91f : c.us) + c.e);
        if (best == 0.f || us < best) best = us, tile = t;
    }
    return best;
}

template <int G, bool Z>
static int launch_rows(W4Params& p, int tile, hipStream_t stream) {
    switch (tile) {
        case 0: return launch_tile<W4Tile<G, Z, 1, 1, 4>>(p, stream);
        case 1: return launch_tile<W4Tile<G, Z, 2, 1, 4>>(p, stream);
        case 2: return launch_tile<W4Tile<G, Z, 2, 2, 3>>(p, stream);
        case 3: return launch_tile<W4Tile<G, Z, 3, 2, 3>>(p, stream);
        case 4: return launch_tile<W4Tile<G, Z, 4, 2, 3>>(p, stream);
    }
    return launch_tile<W4Tile<G, Z, 4, 1, 3>>(p, stream);
}
template <int G>
static int launch_group(W4Params& p, int tile, hipStream_t stream) {
    return p.Z ? launch_rows<G, true>(p, tile, stream) : launch_rows<G, false>(p, tile, stream);
}

int launch_w4_tile(W4Params& p, bool mx, int tile, hipStream_t stream) {
    if (mx) return launch_rows<0, false>(p, tile, stream);
    return p.glog2 == 5 ? launch_group<32>(p, tile, stream)
                        : p.glog2 == 6 ? launch_group<64>(p, tile, stream) : launch_group<128>(p, tile, stream);
}

}  // namespace hkq
