// w4.hip -- 4-bit weights: their quantizer, and products of bf16 rows with them.
//
//   hkq_w4_quant / hkq_w4_dequant   bf16 weights <-> codes with group scales
//   hkq_gemm_w4a16                  C = X . W^T
//   hkq_grouped_gemm_w4a16          the same over ragged groups of rows, a weight each
//
// A weight is (code - zero) * scale (HKQ_W4_INT4: bf16 scales, and zero points or 8,
// per 32, 64 or 128 values of K) or an E2M1 value times a power of two
// (HKQ_W4_MXFP4). Neither is rounded on its way: code - zero and the MXFP4 values from
// 2^-128 to below 2^128 are exact in bf16, as the matrix instruction's operand (which
// keeps values below the smallest normal number), and an INT4 scale multiplies the fp32
// sums of its group. MXFP4 values of 2^128 and more are infinities in the operand.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "w4_core.h"

namespace hkq {

// ---------------------------------------------------------------------------
// Quantizer: 2 bytes read and half a byte written per value, bound by the instructions
// beside them. A lane holds 16 values, G / 16 lanes a group, so that the group's
// part (maxima, divisions, the row's index) comes once per 16; a code is
// med3(rint(v / scale) + zero, 0, 15), and four of them are put together as one exact
// fp32 number. 14336x4096, groups of 128 with zero points, to codes and back: 56 us, 5.3
// TB/s (8 values per lane 69).
// ---------------------------------------------------------------------------
// at / per, in 32 bits where all of them fit
__device__ __forceinline__ int64_t row_of(int64_t at, int64_t per, int64_t total) {
    return total >> 32 == 0 ? (int64_t)((uint32_t)at / (uint32_t)per) : at / per;
}
template <int W, typename F>
__device__ __forceinline__ float group_fold(float v, F f) {
    if constexpr (W >= 2) v = f(v, butterfly_partner<1>(v));
    if constexpr (W >= 4) v = f(v, butterfly_partner<2>(v));
    if constexpr (W >= 8) v = f(v, butterfly_partner<4>(v));
    return v;
}

template <int G, bool Z>
__global__ __launch_bounds__(256) void w4_quant_kernel(const uint16_t* __restrict__ w, uint8_t* __restrict__ q,
                                                       uint16_t* __restrict__ s, uint8_t* __restrict__ z, int64_t N, int K,
                                                       int64_t ldw, int64_t ldq, int64_t lds) {
    typedef uint32_t codes_t __attribute__((ext_vector_type(2), aligned(4)));
    constexpr int L = G / 16;
    const int64_t per = K / 16, total = N * per;
    for (int64_t b = (int64_t)blockIdx.x * 256; b < total; b += (int64_t)gridDim.x * 256) {
        const int64_t at = b + threadIdx.x;  // whole groups: K is a multiple of G, 256 lanes of L
        if (at >= total) return;
        const int64_t row = row_of(at, per, total);
        const int k = (int)(at - row * per) * 16;
        const v4i* from = reinterpret_cast<const v4i*>(w + row * ldw + k);
        const v4i raw[2] = {from[0], from[1]};
        float v[16];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[2 * i] = bf16_to_f32((uint32_t)raw[i / 4][i % 4] & 0xFFFF);
            v[2 * i + 1] = __uint_as_float((uint32_t)raw[i / 4][i % 4] & 0xFFFF0000u);
        }
        // largest magnitude; a NaN orders above every number and is the scale then
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
        const float amax = group_max_abs<L>(__uint_as_float(top));
        float scale, zero = 8.0f;
        if constexpr (Z) {
            float lo = 0.0f, hi = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) lo = min_num(lo, v[i]), hi = max_num(hi, v[i]);
            lo = group_fold<L>(lo, min_num);
            hi = group_fold<L>(hi, max_num);
            scale = hi / 15.0f - lo / 15.0f;
            if (amax != amax) scale = amax;
            scale = bf16_to_f32(f32_to_bf16(scale));
            zero = -lo;
        } else {
            scale = bf16_to_f32(f32_to_bf16(amax / 7.0f));
        }
        // no reciprocal of zero, of a subnormal (it may overflow) or of a NaN: codes of zero
        const float inv = scale >= 0x1p-126f ? 1.0f / scale : 0.0f;
        auto clamp = [](float c) { return __builtin_amdgcn_fmed3f(c, 0.0f, 15.0f); };  // 0 of a NaN
        if constexpr (Z) zero = clamp(__builtin_rintf(zero * inv));
        codes_t code;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t part[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float c[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) c[i] = clamp(__builtin_rintf(v[8 * h + 4 * j + i] * inv) + zero);
                part[j] = (uint32_t)__builtin_fmaf(__builtin_fmaf(__builtin_fmaf(c[3], 16.0f, c[2]), 16.0f, c[1]), 16.0f, c[0]);
            }
            code[h] = part[1] << 16 | part[0];
        }
        *reinterpret_cast<codes_t*>(q + row * ldq + k / 2) = code;
        if (threadIdx.x % L == 0) {
            s[row * lds + k / G] = (uint16_t)f32_to_bf16(scale);
            if constexpr (Z) z[row * lds + k / G] = (uint8_t)(int)zero;
        }
    }
}

__global__ __launch_bounds__(256) void w4_dequant_kernel(const uint8_t* __restrict__ q, const uint16_t* __restrict__ s,
                                                         const uint8_t* __restrict__ z, uint16_t* __restrict__ out, int64_t N,
                                                         int K, int64_t ldq, int64_t lds, int64_t ldo, int glog2) {
    const int64_t per = K / 8, total = N * per;
    for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < total; at += (int64_t)gridDim.x * 256) {
        const int64_t row = row_of(at, per, total);
        const int k = (int)(at - row * per) * 8;
        const uint32_t code = *reinterpret_cast<const uint32_t*>(q + row * ldq + k / 2);
        const int64_t g = row * lds + (k >> glog2);
        const float scale = bf16_to_f32(s[g]), zero = z ? (float)z[g] : 8.0f;
        v4i o;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            o[i] = (int)pk_bf16(((float)(code >> (8 * i) & 15) - zero) * scale, ((float)(code >> (8 * i + 4) & 15) - zero) * scale);
        *reinterpret_cast<v4i*>(out + row * ldo + k) = o;
    }
}

__device__ __forceinline__ v4f mfma_bf16_16(const v4i& a, const v4i& b, const v4f& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf16, a), __builtin_bit_cast(v8bf16, b), c, 0, 0, 0);
}

// ---------------------------------------------------------------------------
// Few rows: the weights' way from memory. A workgroup owns 16 MT rows (4 XL with MT 1)
// of one group and 16 NT columns; its waves split K in units of 128 values, of which
// they hold D (codes) and XD (rows) in registers on their way. The sums of the waves
// meet in LDS.
//
// Loads are made for the memory path and turned in LDS (the wave's own, in order, no
// barrier): neighbouring lanes load neighbouring 16 bytes, a column's 64 bytes of codes
// four lanes, where the matrix instruction (16 x 16 x 32) wants lane c + 16 q to hold
// column c. Loaded as the instruction wants them, 16 columns side by side, each lane's
// 16 bytes were an access of their own, about 70 cycles a load (1x28672x4096 18.7 us,
// 16 rows 25.9).
//
// D[m][n]: rows of X are the instruction's first operand, so that a lane holds one
// column's sums. An instruction takes 32 consecutive values, which lie in one group:
// INT4 sums are multiplied by the group's scale, MXFP4 scales go into the operands. A
// wave's scales: one load for four units (lane c + 16 q: column c of unit q), handed to
// the lanes as each unit is worked on.
// ---------------------------------------------------------------------------
// G: values per group, 0 for MXFP4 (32); Z: zero points
template <int G, bool Z, int MT, int XL, int NT, int NW, int D, int XD, int OCC>
__global__ __launch_bounds__(64 * NW, OCC) void w4_stream_kernel(const W4Params p) {
    constexpr bool MX = G == 0;
    constexpr int NG = MX ? 4 : 128 / G, SB = MX ? 1 : 2;  // scales of a unit, bytes of each
    constexpr int SL = MX ? 1 : NG;                        // registers that hold them (MXFP4: one, four bytes)
    constexpr int XR = 4 * XL, ROWS = MT == 1 ? XR : 16 * MT;
    static_assert(MT == 1 || XL == 4, "whole row tiles");
    constexpr int BUF = (NT + MT * XL) * 1024, RED = MT * NT * 1024;
    __shared__ __attribute__((aligned(16))) uint8_t smem[NW][BUF > RED ? BUF : RED];
    const int lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    RaggedTile t;
    if (p.offs) {
        if (!ragged_tile<ROWS>(p, t)) return;
    } else {
        t.e = 0;
        tile_coords(blockIdx.x, p.tiles_m, p.tiles_n, p.group_m, t.m0, t.tn);
        t.m0 *= ROWS;
        t.rows = p.M - t.m0;
    }
    const int n0 = t.tn * 16 * NT, cols = min(p.N - n0, 16 * NT);
    const auto qr = make_rsrc(p.Q + t.e * p.stride_q + n0 * p.ldq, (uint32_t)((cols - 1) * p.ldq + p.K / 2));
    const int groups = p.K >> p.glog2;
    const uint8_t* s_base = p.S + (t.e * p.stride_s + n0 * p.lds) * SB;
    const auto sr = make_rsrc(s_base, (uint32_t)(((cols - 1) * p.lds + groups) * SB));
    const auto zr = make_rsrc(p.Z + (t.e * p.stride_s + n0 * p.lds), Z ? (uint32_t)((cols - 1) * p.lds + groups) : 0u);
    // rows: load l of XL brings pieces (16 bytes) 16 / XL l .. of the unit's 16 of XR rows;
    // 32-bit offsets from the tile's first row, or (gathered) from X
    constexpr int PL = 16 / XL;
    const int xrow = lane / PL, xpiece = lane % PL;
    uint32_t x_off[MT];
    const uint8_t* x0 = p.X;
    uint32_t x_bytes;
    if (p.gather) {
        x_bytes = (uint32_t)((p.T - 1) * p.ldx + p.K * 2);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const int r = 16 * i + xrow;
            const int id = r < t.rows ? p.gather[t.m0 + r] : -1;
            const int row = id < 0 ? -1 : id / p.topk;
            x_off[i] = row >= 0 && row < p.T ? (uint32_t)(row * p.ldx) : OOB;
        }
    } else {
        x0 += t.m0 * p.ldx;
        x_bytes = (uint32_t)((min(t.rows, ROWS) - 1) * p.ldx + p.K * 2);
#pragma unroll
        for (int i = 0; i < MT; ++i) x_off[i] = 16 * i + xrow < t.rows ? (uint32_t)((16 * i + xrow) * p.ldx) : OOB;
    }
    const auto xr = make_rsrc(x0, x_bytes);

    // LDS: codes piece k of column r in 16-byte slot 4 r + (k ^ r / 4), rows' piece 4 j + kg
    // of row r in slot 4 (XR j + r) + (kg ^ r / 4): the 16 lanes of a read fall on all banks
    HKQ_LDS uint8_t* lw = (HKQ_LDS uint8_t*)smem[wave];
    HKQ_LDS uint8_t* lx = lw + NT * 1024;
    HKQ_LDS uint8_t* w_put = lw + (lane / 4 * 4 + ((lane & 3) ^ (lane >> 4))) * 16;
    HKQ_LDS uint8_t *w_get[4], *x_put[XL], *x_get;
#pragma unroll
    for (int j = 0; j < 4; ++j) w_get[j] = lw + (c * 4 + (j ^ (c >> 2))) * 16 + q * 4;
#pragma unroll
    for (int l = 0; l < XL; ++l) {
        const int piece = l * PL + xpiece;
        x_put[l] = lx + ((piece / 4 * XR + xrow) * 4 + (piece % 4 ^ (xrow >> 2))) * 16;
    }
    x_get = lx + (c % XR * 4 + (q ^ (c % XR >> 2))) * 16;

    const int units = (p.K + 127) / 128, u0 = wave * units / NW, u1 = (wave + 1) * units / NW;
    struct Codes {
        v4i w[NT];
    };
    struct Rows {
        v4i x[MT][XL];
    };
    const uint32_t w_lane = (uint32_t)(lane / 4 * p.ldq + (lane & 3) * 16);
    auto load_codes = [&](int u, Codes& f, int i) {  // of n-tile i
        const bool live = u < u1 && u * 128 + 32 * (lane & 3) < p.K;
        f.w[i] = __builtin_amdgcn_raw_buffer_load_b128(qr, live ? w_lane + (uint32_t)(16 * i * p.ldq + u * 64) : OOB, 0, 0);
    };
    auto load_rows = [&](int u, Rows& f) {
#pragma unroll
        for (int l = 0; l < XL; ++l) {
            const int kx = u * 128 + 8 * (l * PL + xpiece);
            const bool live = u < u1 && kx < p.K;
#pragma unroll
            for (int i = 0; i < MT; ++i)
                f.x[i][l] = __builtin_amdgcn_raw_buffer_load_b128(xr, live && x_off[i] != OOB ? x_off[i] + (uint32_t)(kx * 2) : OOB, 0, 0);
        }
    };
    // scales and zero points of units u .. u + 3: lane c + 16 q those of unit u + q
    struct Four {
        uint32_t s[NT][SL], z[Z ? NT : 1][Z ? NG : 1];
    };
    const bool dwords = MX && ((reinterpret_cast<uintptr_t>(s_base) | (uintptr_t)p.lds | (uintptr_t)groups) & 3) == 0;
    auto load_scales = [&](int u, Four& f) {
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const int at = (u + q) * NG, col = (16 * i + c) * (int)p.lds;
            if (MX && dwords) {
                f.s[i][0] = __builtin_amdgcn_raw_buffer_load_b32(sr, u + q < u1 ? (uint32_t)(col + at) : OOB, 0, 0);
                continue;
            }
            if constexpr (MX) f.s[i][0] = 0;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const uint32_t off = u + q < u1 && at + g < groups ? (uint32_t)(col + at + g) : OOB;
                if constexpr (MX) {
                    f.s[i][0] |= (uint32_t)__builtin_amdgcn_raw_buffer_load_b8(sr, off, 0, 0) << (8 * g);
                } else {
                    f.s[i][g] = __builtin_amdgcn_raw_buffer_load_b16(sr, off == OOB ? OOB : off * 2, 0, 0);
                    if constexpr (Z) f.z[i][g] = __builtin_amdgcn_raw_buffer_load_b8(zr, off, 0, 0);
                }
            }
        }
    };
    v4f acc[MT][NT] = {};
    // unit u, place d in its four; the registers take unit u + D's codes and u + XD's rows
    // once they are in LDS
    auto work = [&](int u, Codes& f, Rows& xs, const Four& sc, int d) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int l = 0; l < XL; ++l) *reinterpret_cast<HKQ_LDS v4i*>(x_put[l] + m * XL * 1024) = xs.x[m][l];
#pragma unroll
        for (int i = 0; i < NT; ++i) *reinterpret_cast<HKQ_LDS v4i*>(w_put + i * 1024) = f.w[i];
        load_rows(u + XD, xs);
#pragma unroll
        for (int i = 0; i < NT; ++i) load_codes(u + D, f, i);
        v4i x[MT][4];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int j = 0; j < 4; ++j) x[m][j] = lds_read16(x_get + m * XL * 1024 + j * XR * 64);
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = *reinterpret_cast<const HKQ_LDS uint32_t*>(w_get[j] + i * 1024);
            v4f P[MT];
            float s[NG], z[NG];
            uint32_t v[SL];
#pragma unroll
            for (int g = 0; g < SL; ++g) {
                v[g] = MX ? sc.s[i][g] : sc.s[i][g] << 16;
                if constexpr (Z) v[g] |= sc.z[i][g];
                v[g] = (uint32_t)__builtin_amdgcn_ds_bpermute((c + 16 * d) * 4, (int)v[g]);
            }
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                if constexpr (MX) {
                    const uint32_t e = v[0] >> (8 * g) & 255;
                    s[g] = __uint_as_float(e << 23 | (e == 255 ? 0x400000u : 0u));
                } else {
                    if constexpr (Z) z[g] = (float)(v[g] & 255);
                    s[g] = __uint_as_float(Z ? v[g] & 0xFFFF0000u : v[g]);
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v4i b;
                if constexpr (MX) {
                    b = fp4_operand(w[j], s[j]);
                } else if constexpr (Z) {
                    b = int4_operand(w[j], z[j * NG / 4]);
                } else {
                    b = int4_sixteenths_operand(w[j]);
                }
                const bool first = !MX && j % (4 / NG) == 0, last = !MX && (j + 1) % (4 / NG) == 0;
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    if constexpr (MX) {
                        acc[m][i] = mfma_bf16_16(x[m][j], b, acc[m][i]);
                    } else {
                        P[m] = mfma_bf16_16(x[m][j], b, first ? v4f{0.f, 0.f, 0.f, 0.f} : P[m]);
                        if (last) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc[m][i][e] = __builtin_fmaf(P[m][e], s[j * NG / 4], acc[m][i][e]);
                        }
                    }
                }
            }
        }
    };
    static_assert(4 % D == 0 && 4 % XD == 0, "whole rings per four units");
    Codes codes[D];
    Rows rows[XD];
    Four sc;
    load_scales(u0, sc);
#pragma unroll
    for (int d = 0; d < (D > XD ? D : XD); ++d) {
        if (d < XD) load_rows(u0 + d, rows[d]);
        if (d < D) {
#pragma unroll
            for (int i = 0; i < NT; ++i) load_codes(u0 + d, codes[d], i);
        }
    }
    for (int u = u0; u < u1; u += 4) {
        Four next;
        load_scales(u + 4, next);
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            if (u + d >= u1) break;
            work(u + d, codes[d % D], rows[d % XD], sc, d);
        }
        sc = next;
    }
    // the waves' sums: each in its own area, added in wave order; tile o by wave o % NW
    v4f* red = reinterpret_cast<v4f*>(smem[wave]);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < NT; ++i) red[(m * NT + i) * 64 + lane] = acc[m][i];
    __syncthreads();
    constexpr float unit = MX || Z ? 1.0f : 16.0f;  // (sixteenths of the codes)
    for (int o = wave; o < MT * NT; o += NW) {
        v4f v = reinterpret_cast<const v4f*>(smem[0])[o * 64 + lane];
#pragma unroll
        for (int w = 1; w < NW; ++w) v = v + reinterpret_cast<const v4f*>(smem[w])[o * 64 + lane];
        const int m = o / NT, n = 16 * (o % NT) + c;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int r = 16 * m + 4 * q + e;
            if (4 * q + e < XR && r < t.rows && n < cols)
                p.C[(int64_t)(t.m0 + r) * p.ldc + n0 + n] = (uint16_t)f32_to_bf16(v[e] * unit);
        }
    }
}

template <int G, bool Z, int MT, int XL, int NT, int NW, int D, int XD, int OCC>
static int launch_w4_stream(W4Params& p, hipStream_t stream) {
    p.tiles_m = (int)ragged_most(p.M, p.E, MT == 1 ? 4 * XL : 16 * MT);
    p.group_m = 8;
    return launch_columns(p, 16 * NT, 64 * NW, w4_from_column<G == 0>, [&](const W4Params& q, unsigned blocks) {
        w4_stream_kernel<G, Z, MT, XL, NT, NW, D, XD, OCC><<<blocks, 64 * NW, 0, stream>>>(q);
    });
}

// Rows per group r (the mean) and columns. A row tile of r rows; more columns per
// workgroup once there are workgroups enough, so that a unit's rows are fetched for more
// columns: us at M x N x K, zero points, 1 | 2 | 4 column tiles: 16x4096x4096 6.1 | 7.8 |
// 11.4, 16x28672x4096 28.2 | 25.0 | 21.5, 6x28672x4096 23.9 | 20.2; MXFP4 16x28672x4096
// 27.8 | 22.8 | 17.9. Up to four rows, one column tile: eight waves 1x4096x14336 10.5,
// 1x28672x4096 20.7, four waves 13.1 and 17.4. Groups of unlike length: beyond a mean of
// two, tiles of 16 rows, where most groups have one, which reads their weights once (mean
// 8, tiles of 8 | 16 rows: 64 groups 2816x2048 103 | 71, 8 groups 28672x4096 150 | 115,
// 4096x4096 22.9 | 21.0; mean 3, 4 | 16: 63 | 68, 126 | 102, 21.0 | 20.4).
static bool ragged(const W4Params& p) { return p.offs && p.E > 1; }
template <int G, bool Z>
static int run_w4_stream(W4Params& p, int64_t r, hipStream_t stream) {
    const int64_t ncu = cu_count() > 0 ? cu_count() : 256;
    const bool many = std::min(p.M, p.E) * ((p.N + 15) / 16) > 3 * ncu;
    if (ragged(p) && r > 2) r = 16;
    if (r <= 4)
        return many ? launch_w4_stream<G, Z, 1, 1, 1, 4, 4, 4, 4>(p, stream) : launch_w4_stream<G, Z, 1, 1, 1, 8, 4, 4, 4>(p, stream);
    if (r <= 8)
        return many ? launch_w4_stream<G, Z, 1, 2, 2, 8, 2, 2, 4>(p, stream) : launch_w4_stream<G, Z, 1, 2, 1, 8, 2, 2, 4>(p, stream);
    if (r <= 16)
        return many ? launch_w4_stream<G, Z, 1, 4, 4, 8, 1, 1, 4>(p, stream) : launch_w4_stream<G, Z, 1, 4, 1, 8, 2, 2, 4>(p, stream);
    return launch_w4_stream<G, Z, 2, 4, 1, 8, 2, 1, 4>(p, stream);
}
template <int G>
static int run_w4_group(W4Params& p, int64_t r, hipStream_t stream) {
    return p.Z ? run_w4_stream<G, true>(p, r, stream) : run_w4_stream<G, false>(p, r, stream);
}

// Streamed or tiled, by estimated time. Up to 16 rows the stream reads a single weight once;
// beyond, once per 32 rows, in 5.8 us per 8192 units of K (128 values of 16 columns)
// (32x4096x4096 8.7 us, on 32-row tiles 22; 64x4096x4096 13.3 and 22; 24x28672x4096 57, 22.7).
// Groups on row tiles of 16: a workgroup's 64 columns take 1.2 us and 0.18 (MXFP4) to 0.4 us
// (scales per 32 values) per unit (stream and 32-row tiles, us: 3 rows of each of 64 groups
// 2816x2048, scales per 64, 68 and 60, 10 rows 73 and 61; 8 groups 4096x14336 58 and 66, 79 and
// 67; MXFP4 28672x4096 102 and 135, 127 and 138); beyond 16 rows they are tiled (20 rows of each
// of 8 groups 4096x4096 32.4 us, tiles 27.8).
static int run_w4(W4Params& p, bool mx, hipStream_t stream) {
    const int64_t live = std::min(p.M, p.E), r = p.M / live, ncu = cu_count() > 0 ? cu_count() : 256, units = (p.K + 127) / 128;
    const bool groups = ragged(p);
    if (r > (groups ? 2 : 16)) {
        int tile;
        const float us_tile = w4_tile_plan(p, tile);
        double us_stream;
        if (!groups) {
            const int64_t wgs = (r + 31) / 32 * ((p.N + 15) / 16);
            us_stream = 3.0 + (double)(std::max(wgs, ncu) * units) * (5.8 / 8192);
        } else {
            const double wgs = (double)live * std::max(1.0, (double)p.M / live / 16 + 0.5) * ((p.N + 63) / 64);
            const double unit = mx ? 0.18 : p.glog2 == 7 ? 0.21 : p.glog2 == 6 ? 0.29 : 0.40;
            us_stream = std::ceil(wgs / ncu) * (units * unit + 1.2);
        }
        // (from 2^27 rows on a grid of the stream's row tiles, of 512 threads, may be too large)
        if (us_tile < us_stream || (groups && r > 16) || p.M >= 1 << 27) return launch_w4_tile(p, mx, tile, stream);
    }
    if (mx) return run_w4_stream<0, false>(p, r, stream);
    return p.glog2 == 5 ? run_w4_group<32>(p, r, stream) : p.glog2 == 6 ? run_w4_group<64>(p, r, stream) : run_w4_group<128>(p, r, stream);
}

static int check_w4_weights(int64_t N, int64_t K, int64_t ldq, int64_t lds, int64_t group) {
    HKQ_CHECK_ARG(N >= 0 && K >= 0, "N and K must be >= 0");
    HKQ_CHECK_ARG(N < (1 << 22) && K < (1 << 22), "N and K must be < 2^22");
    HKQ_CHECK_ARG(group == 32 || group == 64 || group == 128, "group must be 32, 64 or 128");
    HKQ_CHECK_ARG(K % group == 0, "K must be a multiple of group");
    HKQ_CHECK_ARG(ldq >= K / 2 && ldq < (1 << 22), "ldq must be >= K / 2 and < 2^22");
    HKQ_CHECK_ARG(lds >= K / group && lds < (1 << 22), "lds must be >= K / group and < 2^22");
    return 0;
}

}  // namespace hkq

using namespace hkq;

extern "C" int hkq_w4_quant(const void* w, void* q, void* s, void* z, int64_t N, int64_t K, int64_t ldw, int64_t ldq, int64_t lds,
                            int64_t group, hipStream_t stream) {
    if (int e = check_w4_weights(N, K, ldq, lds, group)) return e;
    HKQ_CHECK_ARG(ldw >= K && ldw % 8 == 0 && ldw < (1 << 22), "ldw must be >= K, a multiple of 8 and < 2^22");
    HKQ_CHECK_ARG(ldq % 4 == 0, "ldq must be a multiple of 4");
    if (N == 0 || K == 0) return 0;
    HKQ_CHECK_ARG(w && q && s, "w, q and s are required");
    HKQ_CHECK_ALIGN(w, 16);
    HKQ_CHECK_ALIGN(q, 4);
    HKQ_CHECK_ALIGN(s, 2);
    const int64_t G = K / group;
    const MemRows mw{w, N, 2 * K, 2 * ldw}, mq{q, N, K / 2, ldq}, ms{s, N, 2 * G, 2 * lds}, mz{z, N, G, lds};
    HKQ_CHECK_ARG(!overlap(mq, mw) && !overlap(ms, mw) && !overlap(mz, mw) && !overlap(mq, ms) && !overlap(mq, mz) && !overlap(ms, mz),
                  "q, s and z must not overlap w or each other");
    const unsigned blocks = (unsigned)std::min<int64_t>((N * (K / 16) + 255) / 256, 1 << 16);
    auto kern = group == 32 ? (z ? w4_quant_kernel<32, true> : w4_quant_kernel<32, false>)
                : group == 64 ? (z ? w4_quant_kernel<64, true> : w4_quant_kernel<64, false>)
                              : (z ? w4_quant_kernel<128, true> : w4_quant_kernel<128, false>);
    kern<<<blocks, 256, 0, stream>>>(static_cast<const uint16_t*>(w), static_cast<uint8_t*>(q), static_cast<uint16_t*>(s),
                                     static_cast<uint8_t*>(z), N, (int)K, ldw, ldq, lds);
    return hkq_launch_status();
}

extern "C" int hkq_w4_dequant(const void* q, const void* s, const void* z, void* out, int64_t N, int64_t K, int64_t ldq,
                              int64_t lds, int64_t ldo, int64_t group, hipStream_t stream) {
    if (int e = check_w4_weights(N, K, ldq, lds, group)) return e;
    HKQ_CHECK_ARG(ldo >= K && ldo % 8 == 0 && ldo < (1 << 22), "ldo must be >= K, a multiple of 8 and < 2^22");
    HKQ_CHECK_ARG(ldq % 4 == 0, "ldq must be a multiple of 4");
    if (N == 0 || K == 0) return 0;
    HKQ_CHECK_ARG(q && s && out, "q, s and out are required");
    HKQ_CHECK_ALIGN(q, 4);
    HKQ_CHECK_ALIGN(s, 2);
    HKQ_CHECK_ALIGN(out, 16);
    const int64_t G = K / group;
    const MemRows mo{out, N, 2 * K, 2 * ldo};
    HKQ_CHECK_ARG(!overlap(mo, {q, N, K / 2, ldq}) && !overlap(mo, {s, N, 2 * G, 2 * lds}) && !overlap(mo, {z, N, G, lds}),
                  "out must not overlap q, s or z");
    const unsigned blocks = (unsigned)std::min<int64_t>((N * (K / 8) + 255) / 256, 1 << 16);
    w4_dequant_kernel<<<blocks, 256, 0, stream>>>(static_cast<const uint8_t*>(q), static_cast<const uint16_t*>(s),
                                                  static_cast<const uint8_t*>(z), static_cast<uint16_t*>(out), N, (int)K, ldq, lds,
                                                  ldo, group == 32 ? 5 : group == 64 ? 6 : 7);
    return hkq_launch_status();
}

static int w4_product(const void* X, const void* Q, const void* S, const void* Z, void* C, const int32_t* offs, const int32_t* gather,
                      int64_t M, int64_t T, int64_t E, int64_t N, int64_t K, int64_t topk, int64_t ldx, int64_t ldq, int64_t stride_q,
                      int64_t lds, int64_t stride_s, int64_t ldc, int64_t group, int kind, bool grouped, hipStream_t stream) {
    HKQ_CHECK_ARG(kind == HKQ_W4_INT4 || kind == HKQ_W4_MXFP4, "kind must be HKQ_W4_INT4 or HKQ_W4_MXFP4");
    HKQ_CHECK_ARG(M >= 0 && E >= 0 && T >= 0, "M, E and the rows of X must be >= 0");
    HKQ_CHECK_ARG(M < (1 << 28) && T < (1 << 28) && E < (1 << 16), "M and the rows of X must be < 2^28, E < 2^16");
    if (int e = check_w4_weights(N, K, ldq, lds, group)) return e;
    const bool mx = kind == HKQ_W4_MXFP4;
    HKQ_CHECK_ARG(!mx || (group == 32 && !Z), "MXFP4 weights have groups of 32 and no zero points");
    HKQ_CHECK_ARG(ldx >= K && ldx % 8 == 0 && ldx < (1 << 22), "ldx must be >= K, a multiple of 8 and < 2^22");
    HKQ_CHECK_ARG(ldq % 16 == 0, "ldq must be a multiple of 16");
    HKQ_CHECK_ARG(ldc >= N && ldc < (1 << 22), "ldc must be >= N and < 2^22");
    HKQ_CHECK_ARG(stride_q >= 0 && stride_q % 16 == 0 && stride_q < (1ll << 40), "stride_q must be >= 0, a multiple of 16 and < 2^40");
    HKQ_CHECK_ARG(stride_s >= 0 && stride_s < (1ll << 40), "stride_s must be >= 0 and < 2^40");
    HKQ_CHECK_ARG(!gather || (topk >= 1 && topk <= 65535), "topk must be in [1, 65535]");
    HKQ_CHECK_ARG(!gather || 2 * (int64_t)(T * ldx) < (1ll << 31), "with a gather, X must span less than 2^31 bytes");
    HKQ_CHECK_ARG(gather || !grouped || T >= M, "without a gather, X must have M rows");
    if (M == 0 || E == 0 || N == 0) return 0;
    HKQ_CHECK_ARG(C && (!grouped || offs) && (K == 0 || (Q && S && (X || T == 0))), "X, Q, S, the output and (grouped) offs are required");
    HKQ_CHECK_ALIGN(X, 16);
    HKQ_CHECK_ALIGN(Q, 16);
    HKQ_CHECK_ARG(mx || reinterpret_cast<uintptr_t>(S) % 2 == 0, "S (bf16) must be 2-byte aligned");
    HKQ_CHECK_ALIGN(C, 2);
    HKQ_CHECK_ALIGN(offs, 4);
    HKQ_CHECK_ALIGN(gather, 4);
    const int64_t G = K / group, sb = mx ? 1 : 2;
    const MemRows mc{C, M, 2 * N, 2 * ldc};
    HKQ_CHECK_ARG(!overlap(mc, {X, T, 2 * K, 2 * ldx}) && !overlap(mc, grouped_mem(Q, E, N, K / 2, ldq, stride_q)) &&
                      !overlap(mc, grouped_mem(S, E, N, G * sb, lds * sb, stride_s * sb)) &&
                      !overlap(mc, grouped_mem(Z, E, N, G, lds, stride_s)) && !overlap(mc, {offs, 1, 4 * (E + 1), 0}) &&
                      !overlap(mc, {gather, 1, 4 * M, 0}),
                  "the output must not overlap an operand");
    W4Params p{};
    p.X = static_cast<const uint8_t*>(X);
    p.Q = static_cast<const uint8_t*>(Q);
    p.S = static_cast<const uint8_t*>(S);
    p.Z = static_cast<const uint8_t*>(Z);
    p.C = static_cast<uint16_t*>(C);
    p.offs = offs;
    p.gather = gather;
    p.M = (int)M; p.T = (int)T; p.E = (int)E; p.N = (int)N; p.K = (int)K;
    // without rows X's span, (T - 1) ldx + 2 K bytes, has to be 0
    p.ldx = T > 0 ? 2 * ldx : 2 * K; p.ldq = ldq; p.lds = lds; p.ldc = ldc;
    p.stride_q = stride_q; p.stride_s = stride_s;
    p.glog2 = group == 32 ? 5 : group == 64 ? 6 : 7;
    p.topk = gather ? (int)topk : 1;
    return run_w4(p, mx, stream);
}

extern "C" size_t hkq_gemm_w4a16_workspace(int64_t, int64_t, int64_t) { return 0; }

extern "C" int hkq_gemm_w4a16(const void* X, const void* Q, const void* S, const void* Z, void* C, int64_t M, int64_t N, int64_t K,
                              int64_t ldx, int64_t ldq, int64_t lds, int64_t ldc, int64_t group, int kind, void*, size_t,
                              hipStream_t stream) {
    return w4_product(X, Q, S, Z, C, nullptr, nullptr, M, M, 1, N, K, 1, ldx, ldq, 0, lds, 0, ldc, group, kind, false, stream);
}

extern "C" size_t hkq_grouped_gemm_w4a16_workspace(int64_t, int64_t, int64_t, int64_t) { return 0; }

extern "C" int hkq_grouped_gemm_w4a16(const void* X, const void* Q, const void* S, const void* Z, void* Y, const int32_t* offs,
                                      const int32_t* gather, int64_t M, int64_t T, int64_t E, int64_t N, int64_t K, int64_t topk,
                                      int64_t ldx, int64_t ldq, int64_t stride_q, int64_t lds, int64_t stride_s, int64_t ldy,
                                      int64_t group, int kind, void*, size_t, hipStream_t stream) {
    return w4_product(X, Q, S, Z, Y, offs, gather, M, T, E, N, K, topk, ldx, ldq, stride_q, lds, stride_s, ldy, group, kind, true, stream);
}
