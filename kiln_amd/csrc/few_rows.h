// Up to 16 rows times some column tiles of a packed weight, the groups of K dealt out to a block's wavefronts.
#pragma once
#include <type_traits>

#include "device_common.h"

namespace kiln {

// total[i] = this wavefront's share of 16 rows times column tile i, S of them: f32 sums, scales applied.  The G groups are dealt out GW side
// by side to `turns` wavefronts, of which this one is `turn`; its part of the rows stays in registers while the columns go by: per tile nothing is
// read but its chunks (GW KB, the next tile's asked for before the present one is multiplied) and their scales.  The rows' sums over
// the groups, which the zero-point and the bias of the expanded codes are taken off with, come out of products with ones, once, and go
// in as what the products start from.
//   row  this lane's row (lane & 15), 8 * (lane / 16) values in
//   b    chunk 0 of tile 0, this lane's word of it;  s  scale 0 of tile 0, this lane's column
//   meanwhile()  is called once, behind the first loads
//   also(x, first)  is called for every GW groups that this wavefront has, with its part of the rows; groups first + u, of which those from
//                   G on are none (x then holds the last one's)
template <int GW, int S, class F, class R>
__device__ __forceinline__ void few_rows_product(const uint16_t *__restrict__ row, const u32x4 *__restrict__ b, const uint16_t *__restrict__ s, int G,
                                                 bool per_column, int turn, int turns, const DequantConsts &dc, f32x4 (&total)[S], F &&meanwhile, R &&also) {
    const bf16x8 ones = bf16x8_splat_one();
    const int Gs = per_column ? 1 : G;
#pragma unroll
    for (int i = 0; i < S; ++i) total[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (turn * GW >= G) meanwhile();
    for (int first = turn * GW; first < G; first += turns * GW) {
        auto group = [&](int u) { return min(first + u, G - 1); };  // past the last: the last again, with a scale of zero
        u32x4 w[2][GW];
        uint16_t scale[2][GW];
        auto fetch = [&](int tile) {
#pragma unroll
            for (int u = 0; u < GW; ++u) {
                w[tile & 1][u] = b[(size_t)(tile * G + group(u)) * 64];
                scale[tile & 1][u] = s[(size_t)(tile * Gs + (per_column ? 0 : group(u))) * kTileN];
            }
        };
        fetch(0);
        bf16x8 x[GW][4];
        f32x4 start[GW];
#pragma unroll
        for (int u = 0; u < GW; ++u)
#pragma unroll
            for (int t = 0; t < 4; ++t) x[u][t] = *reinterpret_cast<const bf16x8 *>(row + group(u) * kGroupK + 32 * t);
        __builtin_amdgcn_sched_barrier(0);
        if (first == turn * GW) meanwhile();
#pragma unroll
        for (int u = 0; u < GW; ++u) {
            f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int t = 0; t < 4; ++t) sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[u][t], ones, sum, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) start[u][i] = -kCodeBias * sum[i];
        }
#pragma unroll
        for (int tile = 0; tile < S; ++tile) {
            if (tile + 1 < S) fetch(tile + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int u = 0; u < GW; ++u) {
                const u32x4 &v = w[tile & 1][u];
                f32x4 acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[u][0], codes_to_bf16x8(v.x, dc), start[u], 0, 0, 0);
                acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[u][1], codes_to_bf16x8(v.y, dc), acc, 0, 0, 0);
                acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[u][2], codes_to_bf16x8(v.z, dc), acc, 0, 0, 0);
                acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[u][3], codes_to_bf16x8(v.w, dc), acc, 0, 0, 0);
                const float sc = first + u < G ? f16_bits_to_f32(scale[tile & 1][u]) : 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i) total[tile][i] += sc * acc[i];
            }
        }
        also(x, first);
    }
}
template <int GW, int S>
__device__ __forceinline__ void few_rows_product(const uint16_t *__restrict__ row, const u32x4 *__restrict__ b, const uint16_t *__restrict__ s, int G,
                                                 bool per_column, int turn, int turns, const DequantConsts &dc, f32x4 (&total)[S]) {
    few_rows_product<GW, S>(row, b, s, G, per_column, turn, turns, dc, total, [] {}, [](const bf16x8(&)[GW][4], int) {});
}

// f(W, GW) as integral constants for G groups: five of them to a wavefront at most.
template <class F>
void with_few_rows_split(int G, F &&f) {
    using std::integral_constant;
    if (G <= 8) f(integral_constant<int, 4>{}, integral_constant<int, 2>{});
    else if (G <= 12) f(integral_constant<int, 4>{}, integral_constant<int, 3>{});
    else if (G <= 16) f(integral_constant<int, 4>{}, integral_constant<int, 4>{});
    else if (G <= 20) f(integral_constant<int, 4>{}, integral_constant<int, 5>{});
    else if (G <= 32) f(integral_constant<int, 8>{}, integral_constant<int, 4>{});
    else f(integral_constant<int, 8>{}, integral_constant<int, 5>{});
}

}  // namespace kiln
