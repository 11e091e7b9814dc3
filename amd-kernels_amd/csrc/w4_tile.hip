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
#include <type_traits>

#include "w4_core.h"

namespace hkq {

// G: values per group, 0 for MXFP4 (32)
template <int G_, int TM_, int TN_, int NS_>
struct W4Tile {
    static constexpr int G = G_, TM = TM_, TN = TN_, NS = NS_, NW = 4;
    static constexpr bool MX = G == 0;
    static constexpr int BM = 32 * TM, BN = NW * TN * 32, SB = MX ? 1 : 2;
    static constexpr int NG = MX ? 4 : 128 / G;  // groups in a unit
    // A row's scales of a unit start at any multiple of SB bytes (its zero points at
    // any byte): the aligned dwords that hold them
    static constexpr int SD = (NG * SB + 4 - SB + 3) / 4, ZD = MX ? 0 : (NG + 3 + 3) / 4;
    static constexpr int XB = 2 * BM * 128, WB = BN * 64, STAGE = XB + WB + NW * (SD + ZD) * 256;
    static constexpr int LX = 2 * BM / 8 / NW, LW = BN / 16 / NW, NLD = LX + LW + SD + ZD;
    static constexpr int EP_PITCH = TN * 64 + 16, EP = NW * BM * EP_PITCH;
    static constexpr int LDS = NS * STAGE > EP ? NS * STAGE : EP;
    static_assert(LDS <= 160 * 1024 && NS >= 3 && (NS - 2) * NLD <= 63, "LDS and vmcnt budget");
    static constexpr int PARTS = MX ? 1 : NG, CH = 8 / PARTS;  // chains of matrix instructions per n-tile and m-tile
};

template <class T>
__global__ __launch_bounds__(256, 1) void w4_tile_kernel(const W4Params p) {
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
    if constexpr (!MX) dz = dwords(p.Z ? p.Z + s_at : nullptr, p.Z ? (int)s_n : 0, z_rem);
    const uint32_t s_col = (uint32_t)((wave * TN * 32 + lane % (TN * 32)) * p.lds);  // the lane's column, in scales

    const int units = (p.K + 127) / 128;
    // a unit's loads into a stage; past the last they read nothing
    auto issue = [&](int u, int stage) {
        HKQ_LDS uint8_t* st = smem + stage * T::STAGE;
        const bool live = u < units;
#pragma unroll
        for (int i = 0; i < T::LX; ++i) {
            const int half = i / (T::LX / 2), r = i % (T::LX / 2);
            const bool in = live && u * 128 + half * 64 + xc * 8 < p.K && x_off[r] != OOB;
            lds_load16_d(dx, st + half * BM * 128 + (r * NW + wave) * 1024, in ? x_off[r] + (uint32_t)(u * 256 + half * 128) : OOB);
        }
#pragma unroll
        for (int i = 0; i < T::LW; ++i)
            lds_load16_d(dq, st + T::XB + (i * NW + wave) * 1024, live ? w_off[i] + (uint32_t)(u * 64) : OOB);
        HKQ_LDS uint8_t* sc = st + T::XB + T::WB + wave * (T::SD + T::ZD) * 256;
#pragma unroll
        for (int d = 0; d < T::SD; ++d)
            lds_load4_d(ds, sc + d * 256, live ? ((s_rem + (s_col + (uint32_t)(u * NG)) * SB) & ~3u) + 4 * d : OOB);
#pragma unroll
        for (int d = 0; d < T::ZD; ++d)
            lds_load4_d(dz, sc + (T::SD + d) * 256, live && p.Z ? ((z_rem + s_col + (uint32_t)(u * NG)) & ~3u) + 4 * d : OOB);
    };

    // an n-tile's codes of a unit, and its operands
    struct Raw {
        uint32_t w[8];                // word s: values 16 s + 8 h .. of the unit (MXFP4: 64 (s / 4) + 32 h + 8 (s % 4))
        float s[NG], z[MX ? 1 : NG];  // MXFP4: s[half]: the lane's block
    };
    auto read_raw = [&](int u, int stage, int i, Raw& r) {
        const HKQ_LDS uint8_t* st = smem + stage * T::STAGE;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const v4i v = lds_read16(st + T::XB + KW::swz((wave * TN + i) * 32 + ln, 2 * half + h));
            uint32_t a = (uint32_t)v[0], b = (uint32_t)v[1], c = (uint32_t)v[2], d = (uint32_t)v[3];
            if constexpr (!MX) {
                swap32(a, b);  // a: words 0 and 1 of the 64 values' first 32, b: 4 and 5
                swap32(c, d);
                r.w[4 * half] = a, r.w[4 * half + 1] = c, r.w[4 * half + 2] = b, r.w[4 * half + 3] = d;
            } else {
                r.w[4 * half] = a, r.w[4 * half + 1] = b, r.w[4 * half + 2] = c, r.w[4 * half + 3] = d;
            }
        }
        // scales: bytes at any offset in the staged dwords of the lane's column
        const int cl = i * 32 + ln;
        const uint32_t col = (uint32_t)((wave * TN * 32 + cl) * p.lds) + (uint32_t)(u * NG);
        const HKQ_LDS uint8_t* sc = st + T::XB + T::WB + wave * (T::SD + T::ZD) * 256 + cl * 4;
        auto bits = [&](const HKQ_LDS uint8_t* at, uint32_t b) {
            return *reinterpret_cast<const HKQ_LDS uint32_t*>(at + (b >> 2) * 256) >> (8 * (b & 3));
        };
#pragma unroll
        for (int g = 0; g < (MX ? 2 : NG); ++g) {
            if constexpr (MX) {
                const uint32_t e = u * NG + 2 * g + h < groups ? bits(sc, ((s_rem + col) & 3) + 2 * g + h) & 255 : 0u;
                r.s[g] = e == 255 ? __builtin_nanf("") : exp2i((int)e - 127);
            } else {
                const bool live = u * NG + g < groups;
                const float v = __uint_as_float(bits(sc, ((s_rem + col * 2) & 3) + 2 * g) << 16);
                r.s[g] = live ? v : 0.0f;
                r.z[g] = p.Z ? (float)(bits(sc + T::SD * 256, ((z_rem + col) & 3) + g) & 255) : 8.0f;
            }
        }
    };
    auto operand = [&](const Raw& r, int s) {
        if constexpr (MX) return fp4_operand(r.w[s], r.s[s / 4]);
        else return int4_operand(r.w[s], r.z[s / CH]);
    };
    // fragment s of m-tile j
    uint32_t a_at[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        a_at[s] = (uint32_t)(uintptr_t)smem + (uint32_t)KT::swz(ln, MX ? 4 * h + s : 2 * s + h);
        asm volatile("" : "+v"(a_at[s]));
    }
    auto read_a = [&](int stage, int j, int s) {
        return lds_read16(reinterpret_cast<const HKQ_LDS uint8_t*>(
            (uintptr_t)(a_at[s & 3] + (uint32_t)(stage * T::STAGE + (s / 4) * BM * 128 + j * 32 * 128))));
    };

    v16f acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j) acc[i][j] = v16f{};

    auto bmfma = [](const v4i& a, const v4i& b, const v16f& c) { return mfma_bf16(a, b, c); };

#pragma unroll
    for (int u = 0; u < NS - 1; ++u) issue(u, u);
    tile_barrier<(NS - 2) * T::NLD>();
    v4i B[2][8];
    Raw raw[2];
    read_raw(0, 0, 0, raw[0]);
#pragma unroll
    for (int s = 0; s < 8; ++s) B[0][s] = operand(raw[0], s);
    int stage = 0;
    constexpr int CHUNKS = TM * T::PARTS;
    v16f Pq{};  // the chain before this one's sums, and their scale
    float sq = 0.0f;
    // n-tile i of unit u: matrix instructions on B[cur] while the next n-tile's
    // operands are formed in B[cur ^ 1]
    auto step = [&](int u, auto ii, auto par) {
        constexpr int i = decltype(ii)::value, cur = decltype(par)::value;
        const int next_stage = stage + 1 == NS ? 0 : stage + 1;
        if constexpr (i == TN - 1) {
            // unit u + 1 resident; every wave past unit u - 1, whose stage takes unit u + NS - 1
            tile_barrier<(NS - 3) * T::NLD>();
            issue(u + NS - 1, stage == 0 ? NS - 1 : stage - 1);
        }
        read_raw(i == TN - 1 ? u + 1 : u, i == TN - 1 ? next_stage : stage, (i + 1) % TN, raw[cur ^ 1]);
        v4i A[2][CH];
#pragma unroll
        for (int s = 0; s < CH; ++s) A[0][s] = read_a(stage, 0, s);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const int j = c / T::PARTS, part = c % T::PARTS;
            if (c + 1 < CHUNKS) {
#pragma unroll
                for (int s = 0; s < CH; ++s) A[(c + 1) & 1][s] = read_a(stage, (c + 1) / T::PARTS, (c + 1) % T::PARTS * CH + s);
            }
            v16f P = MX ? acc[i][j] : v16f{};
#pragma unroll
            for (int s = 0; s < CH; ++s) P = bmfma(A[c & 1][s], B[cur][part * CH + s], P);
#pragma unroll
            for (int s = c * 8 / CHUNKS; s < (c + 1) * 8 / CHUNKS; ++s) B[cur ^ 1][s] = operand(raw[cur ^ 1], s);
            if constexpr (MX) {
                acc[i][j] = P;
            } else {
                // the chain before: its matrix instructions are done by now
                const int pc = c == 0 ? CHUNKS - 1 : c - 1, pi = c == 0 ? (i + TN - 1) % TN : i;
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    acc[pi][pc / T::PARTS][e] = __builtin_fmaf(Pq[e], sq, acc[pi][pc / T::PARTS][e]);
                Pq = P;
                sq = raw[cur].s[part];
            }
#pragma unroll
            for (int s = 0; s < CH; ++s) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // one matrix instruction,
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // one LDS read,
                __builtin_amdgcn_sched_group_barrier(0x002, 8, 0);  // eight vector instructions
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;
    auto advance = [&] { stage = stage + 1 == NS ? 0 : stage + 1; };
    if constexpr (TN == 2) {
        for (int u = 0; u < units; ++u) {
            step(u, I0{}, I0{});
            step(u, I1{}, I1{});
            advance();
        }
    } else {
        int u = 0;
        for (; u + 1 < units; u += 2) {
            step(u, I0{}, I0{});
            advance();
            step(u + 1, I0{}, I1{});
            advance();
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
                const uint32_t v = pk_bf16(acc[i][j][e], acc[i][j][e + 1]);
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
    static bool attr = false;
    if (!attr) {
        hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, T::LDS);
        if (e != hipSuccess) {
            set_error("hipFuncSetAttribute(MaxDynamicSharedMemorySize=%d) failed: %s", T::LDS, hipGetErrorString(e));
            return (int)e;
        }
        attr = true;
    }
    p.tiles_m = (int)ragged_most(p.M, p.E, T::BM);
    p.tiles_n = (p.N + T::BN - 1) / T::BN;
    p.group_m = 8;
    const int64_t blocks = (int64_t)p.tiles_m * p.tiles_n;
    HKQ_CHECK_ARG(blocks < (1 << 23), "too many tiles for one launch");
    kern<<<(unsigned)blocks, 256, T::LDS, stream>>>(p);
    return hkq_launch_status();
}

template <int G>
static int launch_group(W4Params& p, hipStream_t stream) {
    const int64_t r = p.M / std::min(p.M, p.E);
    if (r <= 64) return launch_tile<W4Tile<G, 2, 1, 4>>(p, stream);
    return launch_tile<W4Tile<G, 4, 2, 3>>(p, stream);
}

int launch_w4_tile(W4Params& p, bool mx, hipStream_t stream) {
    if (mx) return launch_group<0>(p, stream);
    return p.glog2 == 5 ? launch_group<32>(p, stream) : p.glog2 == 6 ? launch_group<64>(p, stream) : launch_group<128>(p, stream);
}

}  // namespace hkq
