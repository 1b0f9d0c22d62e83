// The projection of 16 rows onto their adapters as the work of one block, for launches that do other work beside it.
#pragma once
#include "bank.h"
#include "bank_expand.h"
#include "device_common.h"

namespace kiln {

// The adapters of 16 rows from p0 on, those whose turn (in the order they are met) is `turn0` modulo `turns`: f(adapter, mask of its rows)
template <class F>
__device__ __forceinline__ void adapters_of_turn(const BankRows &rows, int p0, int c, unsigned turn0, unsigned turns, F &&f) {
    int a = p0 + c < rows.rows ? rows.of[p0 + c] : -1;
    if ((unsigned)a >= (unsigned)rows.count) a = -1;
    unsigned left = (unsigned)__ballot(a >= 0) & 0xFFFFu;
    for (unsigned turn = 0; left; ++turn) {
        const int cur = __builtin_amdgcn_readlane(a, __builtin_ctz(left));
        const unsigned mine = (unsigned)__ballot(a == cur) & 0xFFFFu;
        left &= ~mine;
        if (turn % turns == turn0) f(cur, mine);
    }
}

// t[slice][row][rank] of the rows in `mine`, from what W wavefronts have of it
template <int W>
__device__ __forceinline__ void join_projected(const float (&part)[W][16][kBankMaxRank + 4], float *__restrict__ t, const BankRows &rows, int p0, int slice,
                                               int rank, unsigned mine) {
    __syncthreads();
    float *out = t + ((size_t)slice * rows.rows + p0) * rank;
    for (int e = threadIdx.x; e < 16 * rank; e += 64 * W) {
        const int r = e / rank, j = e - r * rank;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) v += part[w][r][j];
        if (mine >> r & 1) out[e] = v;
    }
    __syncthreads();
}

// T = x A^T over one slice of the contraction, rows as they stand: 16 of the rank at a time, W wavefronts 32 of the contraction each.
template <int W>
__device__ __forceinline__ void project_rows(const BankProjection &p, const BankRows &rows, int rank, int slice, int tile, unsigned turn0, unsigned turns,
                                             float (&part)[W][16][kBankMaxRank + 4]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, q = lane >> 4, p0 = 16 * tile;
    const int each = (p.K / 128 + p.slices - 1) / p.slices * 128, begin = slice * each + 32 * wave, end = min(p.K, (slice + 1) * each);
    const uint16_t *src = (const uint16_t *)p.src + (size_t)min(p0 + c, rows.rows - 1) * p.K + 8 * q;
    adapters_of_turn(rows, p0, c, turn0, turns, [&](int adapter, unsigned mine) {
        for (int j0 = 0; j0 < rank; j0 += 16) {  // rows past the rank: the last one again, their sums are dropped
            const uint16_t *mat = (const uint16_t *)p.mat + ((size_t)adapter * rank + min(j0 + c, rank - 1)) * p.K + 8 * q;
            f32x4 acc = {0.f, 0.f, 0.f, 0.f};
            for (int at = begin; at < end; at += 4 * 32 * W) {
                bf16x8 x[4], m[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    x[u] = load_bf16x8(src + min(at + 32 * W * u, p.K - 32));
                    m[u] = load_bf16x8(mat + min(at + 32 * W * u, p.K - 32));
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (at + 32 * W * u < end) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[u], m[u], acc, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) part[wave][4 * q + i][j0 + c] = acc[i];
        }
        join_projected<W>(part, p.t, rows, p0, slice, rank, mine);
    });
}

}  // namespace kiln
