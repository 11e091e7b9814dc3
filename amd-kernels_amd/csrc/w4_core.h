// w4_core.h -- what the products with 4-bit weights share: parameters, and matrix
// operands made from codes.
#pragma once
#include "ragged.h"

namespace hkq {

struct W4Params {
    const uint8_t* X;  // bf16
    const uint8_t* Q;
    const uint8_t* S;  // bf16 or e8m0
    const uint8_t* Z;  // zero points (nullptr: 8)
    uint16_t* C;
    const int32_t* offs;    // nullptr: one group of M rows
    const int32_t* gather;  // row r is X row gather[r] / topk (nullptr: r itself)
    int M, T, E, N, K;      // T: rows of X
    int64_t ldx, ldq, lds, ldc;    // bytes, bytes, scales, values
    int64_t stride_q, stride_s;    // group to group: bytes, scales
    int glog2, topk;
    int tiles_m, tiles_n, group_m;
};

// ---------------------------------------------------------------------------
// Operands from codes.
// ---------------------------------------------------------------------------
typedef uint32_t v2u __attribute__((ext_vector_type(2)));

// Codes (value j in nibble j) 4 H .. 4 H + 3 -> bf16 values code - zero, exactly: a
// byte that holds 0 .. 15 is, as E4M3, that number times 2^-9, so one conversion with
// scale 2^9 gives two codes as fp32; the difference has at most 4 significant bits,
// and the upper half of its fp32 pattern is its bf16. 19 instructions per 8 codes.
template <int H>
__device__ __forceinline__ v2i int4_operand2(uint32_t w, float zero) {
    const f32x2_t e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w & 0x0F0F0F0Fu, 512.0f, H != 0);
    const f32x2_t d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w >> 4 & 0x0F0F0F0Fu, 512.0f, H != 0);
    return v2i{(int)__builtin_amdgcn_perm(__float_as_uint(d[0] - zero), __float_as_uint(e[0] - zero), 0x07060302u),
               (int)__builtin_amdgcn_perm(__float_as_uint(d[1] - zero), __float_as_uint(e[1] - zero), 0x07060302u)};
}
__device__ __forceinline__ v4i int4_operand(uint32_t w, float zero) {
    const v2i a = int4_operand2<0>(w, zero), b = int4_operand2<1>(w, zero);
    return v4i{a[0], a[1], b[0], b[1]};
}
// The same for zero = 8, as sixteenths (code - 8) / 16: with its upper bit inverted a
// code is a signed nibble, which v_cvt_off_f32_i4 converts from the low half of any
// byte. 14 instructions per 8 codes. A matrix instruction may read the result two wait
// states later; the compiler keeps that distance for instructions that it knows, not for
// these (int4_sixteenths_settle).
template <int H>
__device__ __forceinline__ v2i int4_sixteenths(uint32_t w) {
    const uint32_t ev = w ^ 0x88888888u, od = ev >> 4;
    // (one block: the compiler has no byte select for this conversion, and pads asm
    // results with wait states that whole-register writes do not need)
#define HKQ_NIBBLES(B0, B1)                                                           \
    "v_cvt_off_f32_i4_sdwa %0, %4 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:" B0 "\n\t" \
    "v_cvt_off_f32_i4_sdwa %2, %5 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:" B0 "\n\t" \
    "v_cvt_off_f32_i4_sdwa %1, %4 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:" B1 "\n\t" \
    "v_cvt_off_f32_i4_sdwa %3, %5 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:" B1 "\n\t" \
    "v_perm_b32 %0, %2, %0, %6\n\t"                                                   \
    "v_perm_b32 %1, %3, %1, %6"
    uint32_t o0, o1, t0, t1;
    if constexpr (H == 0)
        asm(HKQ_NIBBLES("BYTE_0", "BYTE_1") : "=&v"(o0), "=&v"(o1), "=&v"(t0), "=&v"(t1) : "v"(ev), "v"(od), "s"(0x07060302u));
    else
        asm(HKQ_NIBBLES("BYTE_2", "BYTE_3") : "=&v"(o0), "=&v"(o1), "=&v"(t0), "=&v"(t1) : "v"(ev), "v"(od), "s"(0x07060302u));
#undef HKQ_NIBBLES
    return v2i{(int)o0, (int)o1};
}
// Those two wait states: an operand that a matrix instruction reads next.
__device__ __forceinline__ void int4_sixteenths_settle(v4i& b) { asm("s_nop 1" : "+v"(b)); }
__device__ __forceinline__ v4i int4_sixteenths_operand(uint32_t w) {
    const v2i lo = int4_sixteenths<0>(w), hi = int4_sixteenths<1>(w);
    v4i b = v4i{lo[0], lo[1], hi[0], hi[1]};
    int4_sixteenths_settle(b);
    return b;
}
// E2M1 codes 4 H .. 4 H + 3 times 2^(e8m0 - 127), the scale as the fp32 of that exponent.
template <int H>
__device__ __forceinline__ v2i fp4_operand2(uint32_t w, float scale) {
    return v2i{__builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2 * H)),
               __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2 * H + 1))};
}
__device__ __forceinline__ v4i fp4_operand(uint32_t w, float scale) {
    const v2i a = fp4_operand2<0>(w, scale), b = fp4_operand2<1>(w, scale);
    return v4i{a[0], a[1], b[0], b[1]};
}

__device__ __forceinline__ void swap32(uint32_t& a, uint32_t& b) {
    const v2u r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = r[0], b = r[1];
}

// The weights, and the output, from column n on (launch_columns).
template <bool MX>
inline void w4_from_column(W4Params& q, int64_t n) {
    q.Q += n * q.ldq;
    q.S += n * q.lds * (MX ? 1 : 2);
    if (q.Z) q.Z += n * q.lds;
    q.C += n;
}

// The tiles of w4_tile.hip: the size with the least estimated time (us), and its launch.
float w4_tile_plan(const W4Params& p, int& tile);
int launch_w4_tile(W4Params& p, bool mx, int tile, hipStream_t stream);

}  // namespace hkq
