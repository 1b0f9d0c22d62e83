// The order of a call's rows by their adapters, as the work of one block per adapter.
#pragma once
#include "bank.h"

namespace kiln {

// order[] and first[]: a block per adapter (and one for the rows without) counts the rows of lower adapters and places its own, 64 rows
// per ballot, its W wavefronts a part of the rows each: no block waits for another and rows keep their order inside an adapter.  Up
// to 512 W rows a wavefront's part is in registers and read once.  2048 rows, 8 adapters: a wavefront for each took 14 us, a block 5.
constexpr int kOrderUnroll = 8;
template <int W>
struct OrderLds {
    int less_of[W], mine_of[W];
};
template <int W>
__device__ __forceinline__ void order_rows(const int *__restrict__ of, int *__restrict__ order, int *__restrict__ first, int rows, int count, int a,
                                           OrderLds<W> &lds) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int each = (rows + W * 64 - 1) / (W * 64) * 64;
    const int begin = wave * each, end = min(rows, begin + each);
    int key[kOrderUnroll];
    auto read = [&](int r0) {
#pragma unroll
        for (int u = 0; u < kOrderUnroll; ++u) {
            const int r = r0 + 64 * u + lane;
            key[u] = r < end ? of[r] : -1;
        }
#pragma unroll
        for (int u = 0; u < kOrderUnroll; ++u) {
            if ((unsigned)key[u] >= (unsigned)count) key[u] = count;
            if (r0 + 64 * u + lane >= end) key[u] = INT32_MAX;
        }
    };
    int less = 0, mine = 0;
    for (int r0 = begin; r0 < end; r0 += 64 * kOrderUnroll) {
        read(r0);
#pragma unroll
        for (int u = 0; u < kOrderUnroll; ++u) {
            less += __popcll(__ballot(key[u] < a));
            mine += __popcll(__ballot(key[u] == a));
        }
    }
    if (lane == 0) {
        lds.less_of[wave] = less;
        lds.mine_of[wave] = mine;
    }
    __syncthreads();
    int at = 0;
    for (int w = 0; w < W; ++w) at += lds.less_of[w];
    if (threadIdx.x == 0) {
        first[a] = at;
        if (a == count) first[count + 1] = rows;
    }
    for (int w = 0; w < wave; ++w) at += lds.mine_of[w];
    for (int r0 = begin; r0 < end; r0 += 64 * kOrderUnroll) {
        if (each > 64 * kOrderUnroll) read(r0);
#pragma unroll
        for (int u = 0; u < kOrderUnroll; ++u) {
            const unsigned long long all = __ballot(key[u] == a);
            if (key[u] == a) order[at + __popcll(all & ((1ull << lane) - 1))] = r0 + 64 * u + lane;
            at += __popcll(all);
        }
    }
}

}  // namespace kiln
