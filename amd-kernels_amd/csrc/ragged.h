// ragged.h -- rows in groups (the experts of a mixture) whose bounds are on the GPU:
// which tile of which group a workgroup takes. Params P have offs int32 [E + 1],
// M, E, tiles_m (the most there can be), tiles_n and group_m.
#pragma once
#include <algorithm>

#include "gemm_core.h"
#include "hkq_host.h"

namespace hkq {

// Rows [start, end) of group e: bounds outside [0, M], or decreasing ones, never
// leave the operands.
template <class P>
__device__ __forceinline__ int2 group_rows(const P& p, int e) {
    const int start = min(max(p.offs[e], 0), p.M);
    return make_int2(start, min(max(p.offs[e + 1], start), p.M));
}

// The bid-th workgroup's place in the order in which an XCD's workgroups, which are
// dealt out round robin, are neighbours.
__device__ __forceinline__ int xcd_order(int bid, int n) {
    const int q = n >> 3, rem = n & 7, xcd = bid & 7, idx = bid >> 3;
    return xcd < rem ? xcd * (q + 1) + idx : rem * (q + 1) + (xcd - rem) * q + idx;
}
// Tile `in` of a group with tiles_m x tiles_n of them, group_m row tiles at a time, rows
// first: neighbours share a group's weight columns and rows in their XCD's L2.
__device__ __forceinline__ void group_tile(int in, int tiles_m, int tiles_n, int group_m, int& tm, int& tn) {
    const int band = in / (group_m * tiles_n), first = band * group_m, size = min(tiles_m - first, group_m);
    const int at = in - band * group_m * tiles_n;
    tm = first + at % size;
    tn = at / size;
}

// Sums of tile counts, held at the largest int: bounds that count rows many times (65535
// groups of all rows) would pass it.
__device__ __forceinline__ int add_sat(int a, int b) { return __builtin_elementwise_add_sat(a, b); }

struct RaggedTile {
    int e, m0, rows;  // group, the tile's first row among all rows, the group's rows from there on
    int tn;
};

// Tile of this workgroup among the BM-row tiles of all groups, in group order, times
// the column tiles; false past the last. Each wave scans the groups' tile counts, 64
// groups at a time (twice where there are more: the order over the XCDs needs the
// total). One load's latency, hidden behind nothing: about 1 us of a call.
template <int BM, class P>
__device__ __forceinline__ bool ragged_tile(const P& p, RaggedTile& t) {
    const int lane = threadIdx.x & 63;
    auto count = [&](int e) {
        if (e >= p.E) return 0;
        const int2 r = group_rows(p, e);
        return (r.y - r.x + BM - 1) / BM;
    };
    auto scan = [&](int v) {  // inclusive sums over the wave
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int o = __shfl_up(v, d, 64);
            if (lane >= d) v = add_sat(v, o);
        }
        return v;
    };
    int n = count(lane), s = scan(n), total = __builtin_amdgcn_readlane(s, 63);
    for (int e0 = 64; e0 < p.E; e0 += 64) total = add_sat(total, __builtin_amdgcn_readlane(scan(count(e0 + lane)), 63));
    total = min(total, p.tiles_m);  // bounds that count a row twice: the tiles that the grid holds
    if ((int)blockIdx.x >= total * p.tiles_n) return false;
    const int id = xcd_order(blockIdx.x, total * p.tiles_n), at = id / p.tiles_n;
    int before = 0;  // tiles of the groups before e0
    for (int e0 = 0; e0 < p.E; e0 += 64) {
        if (e0 > 0) n = count(e0 + lane), s = scan(n);
        const uint64_t past = __ballot(add_sat(before, s) > at);
        if (past) {
            const int l = __builtin_ctzll(past);
            t.e = e0 + l;
            const int tiles = __builtin_amdgcn_readlane(n, l), first = before + __builtin_amdgcn_readlane(s, l) - tiles;
            int tm;
            group_tile(id - first * p.tiles_n, tiles, p.tiles_n, p.group_m, tm, t.tn);
            const int2 r = group_rows(p, t.e);
            t.m0 = __builtin_amdgcn_readfirstlane(r.x + tm * BM);
            t.rows = __builtin_amdgcn_readfirstlane(r.y) - t.m0;
            return true;
        }
        before = add_sat(before, __builtin_amdgcn_readlane(s, 63));
    }
    return false;
}

// Tiles that M rows in E groups can need at most: each group with rows wastes less
// than one.
inline int64_t ragged_most(int64_t M, int64_t E, int64_t bm) {
    const int64_t live = std::min(M, E);
    return (M - live) / bm + live;
}

// Launches of a product with p.N columns in tiles of bn: one, or as many as keep each below
// 2^32 threads (a grid's limit), of whole column tiles each. at(q, n) moves a copy's operands to
// column n. One column of row tiles always fits: below 2^28 rows make at most 2^22 + 2^16 of
// 64 rows with 512 threads, 2^23 + 2^16 of 32 with 256; shorter ones take below 2^27 rows.
template <class P, class At, class Launch>
inline int launch_columns(const P& p, int bn, int threads, At at, Launch launch) {
    const int64_t most = std::max<int64_t>(1, 0xFFFFFFFFll / threads / p.tiles_m);
    for (int64_t n = 0; n < p.N; n += most * bn) {
        P q = p;
        q.N = (int)std::min<int64_t>(p.N - n, most * bn);
        q.tiles_n = (q.N + bn - 1) / bn;
        at(q, n);
        launch(q, (unsigned)((int64_t)q.tiles_m * q.tiles_n));
        if (int e = hkq_launch_status()) return e;
    }
    return 0;
}

// E groups of R rows of `width` bytes, `pitch` apart, groups `stride` apart: one
// operand's memory for overlap().
inline MemRows grouped_mem(const void* p, int64_t E, int64_t R, int64_t width, int64_t pitch, int64_t stride) {
    if (E <= 0 || R <= 0) return MemRows{nullptr, 0, 0, 0};
    if (stride == R * pitch || E == 1) return MemRows{p, E * R, width, pitch};
    return MemRows{p, 1, (E - 1) * stride + (R - 1) * pitch + width, 0};
}

}  // namespace hkq
