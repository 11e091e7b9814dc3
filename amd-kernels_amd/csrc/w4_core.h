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

// 8 codes (value j in nibble j) -> 8 bf16 values code - zero, exactly: a byte that
// holds 0 .. 15 is, as E4M3, that number times 2^-9, so one conversion with scale 2^9
// gives two codes as fp32; the difference has at most 4 significant bits, and the
// upper half of its fp32 pattern is its bf16.
__device__ __forceinline__ v4i int4_operand(uint32_t w, float zero) {
    const uint32_t ev = w & 0x0F0F0F0Fu, od = w >> 4 & 0x0F0F0F0Fu;
    v4i o;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const f32x2_t e = h ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(ev, 512.0f, true)
                            : __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(ev, 512.0f, false);
        const f32x2_t d = h ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(od, 512.0f, true)
                            : __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(od, 512.0f, false);
        o[2 * h] = (int)__builtin_amdgcn_perm(__float_as_uint(d[0] - zero), __float_as_uint(e[0] - zero), 0x07060302u);
        o[2 * h + 1] = (int)__builtin_amdgcn_perm(__float_as_uint(d[1] - zero), __float_as_uint(e[1] - zero), 0x07060302u);
    }
    return o;
}
// 8 E2M1 codes times 2^(e8m0 - 127), the scale as the fp32 of that exponent.
__device__ __forceinline__ v4i fp4_operand(uint32_t w, float scale) {
    v4i o;
    o[0] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0));
    o[1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1));
    o[2] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2));
    o[3] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3));
    return o;
}

__device__ __forceinline__ void swap32(uint32_t& a, uint32_t& b) {
    const v2u r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = r[0], b = r[1];
}
__device__ __forceinline__ void swap16(uint32_t& a, uint32_t& b) {
    const v2u r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    a = r[0], b = r[1];
}

// The tile kernel of w4_tile.hip.
int launch_w4_tile(W4Params& p, bool mx, hipStream_t stream);

}  // namespace hkq
