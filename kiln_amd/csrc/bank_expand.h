// The rows of a call on a bank and the second half of their low-rank term, for the kernels that add it.
#pragma once
#include "bank.h"
#include "device_common.h"

namespace kiln {

__device__ __forceinline__ bf16x8 load_bf16x8(const uint16_t *p) {
    return __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4 *>(p));
}

// The row and the adapter (-1: none) of position p.
__device__ __forceinline__ void row_at(const BankRows &r, int p, int &row, int &a) {
    row = p < r.rows ? (r.order ? r.order[p] : p) : -1;
    a = row >= 0 ? r.of[row] : -1;
    if ((unsigned)a >= (unsigned)r.count) a = -1;
}

__device__ __forceinline__ __bf16 lower_part(float f, __bf16 hi) {  // what hi leaves of f; an infinity leaves nothing
    return (__bf16)((float)hi == f ? 0.f : f - (float)hi);
}

// y[row] += s_a T[row] B_a^T, formed as B_a (its rows the columns of y) times T^T, so that a lane holds consecutive columns of one row:
// two products of 16 columns, whose rows of B_a are dealt out such that their results are eight columns side by side.  T goes in as two
// bf16 parts whose sum is within 2^-17 of it, one product each with the same rows of B.  S: the contraction's steps of 32.
// A product's result is taken by the rows of its adapter alone (a lane has one row): what another adapter holds that is no number
// stays with its own rows.
__device__ __forceinline__ int column_of(int tile, int c) { return 32 * (tile >> 1) + 8 * (c >> 2) + 4 * (tile & 1) + (c & 3); }

template <int S>
struct ExpandRow {  // this lane's part of its row's T
    bf16x8 hi[S], lo[S];
    __device__ __forceinline__ void set(const float *t, float scale, bool live, int q, int rank) {
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const int at = 32 * s + 8 * q;
            hi[s] = lo[s] = bf16x8_zero();
            if (live && at < rank)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float f = t[at + i] * scale;
                    hi[s][i] = (__bf16)f;
                    lo[s][i] = lower_part(f, hi[s][i]);
                }
        }
    }
};
// 16 TILES columns from n0 on, of adapter `mat`'s rows of B (past the rank: the last eight again, times zeros)
template <int S, int TILES>
__device__ __forceinline__ void expand_rows(const uint16_t *__restrict__ mat, int c, int q, int rank, bf16x8 (&b)[TILES][S]) {
#pragma unroll
    for (int tile = 0; tile < TILES; ++tile)
#pragma unroll
        for (int s = 0; s < S; ++s) b[tile][s] = load_bf16x8(mat + (size_t)column_of(tile, c) * rank + min(32 * s + 8 * q, rank - 8));
}
template <int S, int TILES>
__device__ __forceinline__ void expand_product(const bf16x8 (&b)[TILES][S], const ExpandRow<S> &t, bool own, f32x4 (&acc)[TILES]) {
#pragma unroll
    for (int tile = 0; tile < TILES; ++tile) {
        f32x4 v = acc[tile];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            v = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[tile][s], t.hi[s], v, 0, 0, 0);
            v = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[tile][s], t.lo[s], v, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[tile][i] = own ? v[i] : acc[tile][i];
    }
}

// T's slices summed, [positions][rank] of this block's from p0 on: four of the rank at a time, eight slices' loads in flight together
template <int P>
__device__ __forceinline__ void sum_projected(const float *__restrict__ t, const BankRows &rows, int p0, int rank, int slices, int tid, int threads,
                                              float (&ts)[P][kBankMaxRank + 4]) {
    const size_t stride = (size_t)rows.rows * rank;
    for (int e = 4 * tid; e < P * rank; e += 4 * threads) {
        const int r = e / rank;
        const float *from = t + (size_t)min(p0 + r, rows.rows - 1) * rank + (e - r * rank);
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < slices; s += 8) {
            f32x4 d[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] = *reinterpret_cast<const f32x4 *>(from + min(s + i, slices - 1) * stride);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (s + i < slices) v += d[i];
        }
        *reinterpret_cast<f32x4 *>(&ts[r][e - r * rank]) = v;
    }
    __syncthreads();
}

}  // namespace kiln
