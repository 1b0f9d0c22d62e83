// A router's choices in the order of their experts, the tokens' rows in that order and back: what stands around products with experts
// for many tokens (w4a16_experts.hip), and the gradients.
//   sort              order = the pairs (token, choice) by expert, in their order inside one; place its inverse; first[e] where e begins
//   gather            rows[place[t, j]] = x[t]                          its gradient: a combine with weights of one
//   combine           y[t] = sum_j w[t, j] rows[place[t, j]]
//   combine backward  d_rows[place[t, j]] = w[t, j] dy[t],  d_w[t, j] = <rows[place[t, j]], dy[t]>
// Pairs without an expert come last, from position first[experts] on: rows of zeros where rows are written, never read.
// No counterpart in the reference, whose model family is dense.  All but the sort are bound by the rows, read and written once.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "device_common.h"
#include "kiln_w4a16.h"
#include "launch.h"
#include "pieces.h"

namespace kiln {
namespace {

constexpr int kMaxExperts = 1024, kMaxTop = 16;
constexpr int64_t kMaxPairs = 1 << 30;

// ---- the sort ------------------------------------------------------------------------------------------------------
// By counting: pairs go to blocks and their wavefronts in contiguous parts; a pair's position is where its expert begins, plus the expert's
// pairs in earlier blocks, earlier wavefronts and earlier turns of its own, plus those in lower lanes.  Nothing depends on who comes
// first.  Several blocks need their counts from a launch in front; one block's pairs are counted where they are placed.
constexpr int kSortWaves = 8, kSortThreads = kSortWaves * 64;
constexpr int kSortMaxBlocks = 256;
constexpr int kSortBlockPairs = 2048;
struct SortArgs {
    const int *of;
    int *order, *first, *place;
    int *counts;  // [blocks, experts + 1]
    int pairs, experts, each;  // pairs to a block, a multiple of kSortThreads
};
__device__ __forceinline__ int sort_key(const SortArgs &p, int pair) {
    const int e = p.of[pair];
    return (unsigned)e < (unsigned)p.experts ? e : p.experts;
}

__global__ __launch_bounds__(kSortThreads) void moe_count_kernel(SortArgs p) {
    __shared__ int count[kMaxExperts + 1];
    for (int e = threadIdx.x; e <= p.experts; e += kSortThreads) count[e] = 0;
    __syncthreads();
    const int begin = blockIdx.x * p.each, end = min(p.pairs, begin + p.each);
    for (int i = begin + threadIdx.x; i < end; i += kSortThreads) atomicAdd(&count[sort_key(p, i)], 1);
    __syncthreads();
    for (int e = threadIdx.x; e <= p.experts; e += kSortThreads) p.counts[(size_t)blockIdx.x * (p.experts + 1) + e] = count[e];
}

__global__ __launch_bounds__(kSortThreads) void moe_sort_kernel(SortArgs p) {
    __shared__ int count[kSortWaves][kMaxExperts + 1];  // of a wavefront; then where its next pair of the expert goes
    __shared__ int total[kMaxExperts + 1], before[kMaxExperts + 1];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, keys = p.experts + 1;
    const int part = p.each / kSortWaves, begin = blockIdx.x * p.each + wave * part, end = min(p.pairs, begin + part);
    for (int i = tid; i < kSortWaves * keys; i += kSortThreads) count[i / keys][i % keys] = 0;
    __syncthreads();
    for (int i = begin + lane; i < end; i += 64) atomicAdd(&count[wave][sort_key(p, i)], 1);
    __syncthreads();
    for (int e = tid; e < keys; e += kSortThreads) {
        int all = 0, earlier = 0;
        if (gridDim.x == 1) {
            for (int w = 0; w < kSortWaves; ++w) all += count[w][e];
        } else {
#pragma unroll 8
            for (int b = 0; b < (int)gridDim.x; ++b) {
                const int n = p.counts[(size_t)b * keys + e];
                all += n;
                earlier += b < (int)blockIdx.x ? n : 0;
            }
        }
        total[e] = all;
        before[e] = earlier;
    }
    __syncthreads();
    if (wave == 0) {  // where each expert begins: a lane adds up consecutive ones
        const int per = (keys + 63) / 64, e0 = lane * per, e1 = min(keys, e0 + per);
        int sum = 0;
        for (int e = e0; e < e1; ++e) sum += total[e];
        int upto = sum;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int below = __shfl_up(upto, d);
            if (lane >= d) upto += below;
        }
        int at = upto - sum;
        for (int e = e0; e < e1; ++e) {
            if (blockIdx.x == 0) p.first[e] = at;
            before[e] += at;
            at += total[e];
        }
    }
    __syncthreads();
    for (int e = tid; e < keys; e += kSortThreads) {
        int at = before[e];
        for (int w = 0; w < kSortWaves; ++w) {
            const int n = count[w][e];
            count[w][e] = at;
            at += n;
        }
    }
    __syncthreads();
    const int bits = 32 - __builtin_clz(keys - 1);
    for (int i0 = begin; i0 < end; i0 += 64) {
        const int i = i0 + lane;
        const bool here = i < end;
        const int key = here ? sort_key(p, i) : -1;
        unsigned long long same = __ballot(here);
        for (int b = 0; b < bits; ++b) {
            const unsigned long long set = __ballot(key >> b & 1);
            same &= key >> b & 1 ? set : ~set;
        }
        const int lower = __popcll(same & ((1ull << lane) - 1));
        int at = 0;
        if (here) at = count[wave][key];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (here && lower == 0) count[wave][key] = at + __popcll(same);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (here) {
            p.order[at + lower] = i;
            p.place[i] = at + lower;
        }
    }
}

// ---- rows ----------------------------------------------------------------------------------------------------------
// Units of 16 bytes, a thread for each of a token's: it is read or written once, its rows at `top` places.  The gather stores to one place after the other; the
// combine asks for a place, waits for it, asks for its row and for the next place, so that a thread's rows come one after the other, and then for the weights.
// Many tokens have enough wavefronts to cover that (8192 tokens of 8, 2048 wide 52 us, 6 TB/s; 1000 of 8, 2560 wide added up 8.4 us); one token's gather takes
// 2.9 us, 64 tokens' combine 4.3.
// (A place that no pair has is passed over: nothing is read or written out of bounds whatever `place` holds.)
struct RowsArgs {
    const uint16_t *in;      // gather: x; combine: rows; combine backward: dy
    const uint16_t *rows;    // combine backward
    const float *weights;    // [tokens, top], or null: one each
    const int *first, *place;
    uint16_t *out;
    float *d_weights;
    int tokens, top, experts, units;
};

// a thread's token and unit (a launch has less than 2^32 of them, rows_ok sees to that)
struct Place {
    int token, unit;
    size_t at;
    bool live;
};
__device__ __forceinline__ Place place_of(const RowsArgs &p) {
    const unsigned i = blockIdx.x * 256 + threadIdx.x, units = (unsigned)p.units, token = i / units;
    return {(int)token, (int)(i - token * units), i, i < (unsigned)p.tokens * units};
}

__global__ __launch_bounds__(256) void moe_gather_kernel(RowsArgs p) {
    const auto [token, unit, i, live] = place_of(p);
    if (!live) return;
    const int placed = p.first[p.experts], pairs = p.tokens * p.top;
    const u32x4 v = reinterpret_cast<const u32x4 *>(p.in)[i], zero = {0u, 0u, 0u, 0u};
    for (int j = 0; j < p.top; ++j) {
        const int at = p.place[(size_t)token * p.top + j];
        if ((unsigned)at < (unsigned)pairs) reinterpret_cast<u32x4 *>(p.out)[(size_t)at * p.units + unit] = at < placed ? v : zero;
    }
}

__device__ __forceinline__ float bf16_low(uint32_t v) { return __builtin_bit_cast(float, v << 16); }
__device__ __forceinline__ float bf16_high(uint32_t v) { return __builtin_bit_cast(float, v & 0xFFFF0000u); }
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t bf16_pair(float low, float high) { return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)low, (__bf16)high}); }

__global__ __launch_bounds__(256) void moe_combine_kernel(RowsArgs p) {
    const auto [token, unit, i, live] = place_of(p);
    if (!live) return;
    const int placed = min(p.first[p.experts], p.tokens * p.top);
    float sum[8] = {};
    for (int j0 = 0; j0 < p.top; j0 += 8) {
        u32x4 v[8];
        bool here[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int at = j0 + u < p.top ? p.place[(size_t)token * p.top + j0 + u] : placed;
            here[u] = at >= 0 && at < placed;
            if (here[u]) v[u] = reinterpret_cast<const u32x4 *>(p.in)[(size_t)at * p.units + unit];
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            if (!here[u]) continue;
            const float w = p.weights ? p.weights[(size_t)token * p.top + j0 + u] : 1.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                sum[2 * e] = fmaf(w, bf16_low(v[u][e]), sum[2 * e]);
                sum[2 * e + 1] = fmaf(w, bf16_high(v[u][e]), sum[2 * e + 1]);
            }
        }
    }
    u32x4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = bf16_pair(sum[2 * e], sum[2 * e + 1]);
    reinterpret_cast<u32x4 *>(p.out)[i] = o;
}

constexpr int kAhead = 4;  // units of a lane in flight
// A wavefront to a pair: its lanes go over the units of dy and of the pair's row together; the product is summed in f32 in the lanes and across them, in that
// order.  dy is read once from memory and by the token's other pairs from the caches.  4096 tokens, 8 of 64, 2560 wide (357 MB) 73 us, 4.9 TB/s; a block to a
// token, its wavefronts sharing out the units, 82 (five parts of 64 units do not go evenly to four), 64 tokens 3.9 and 7.9.
// LAST: the rows are read past the caches, for the last time, which leaves room for what is written and the next product reads -- where they are too many to
// have stayed there: 78 MB of rows 38 us without and 32, 58 MB 28 and 26, 39 MB level, but 27 MB 11.8 and 13.5; from 100 MB on level.
template <bool LAST>
__global__ __launch_bounds__(256) void moe_combine_backward_kernel(RowsArgs p) {
    const int lane = threadIdx.x & 63, pairs = p.tokens * p.top, placed = min(p.first[p.experts], pairs);
    const int pair = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    if (pair >= pairs) return;
    const int at = p.place[pair], token = (int)((unsigned)pair / (unsigned)p.top);
    const float w = p.weights[pair];
    const bool here = at >= 0 && at < placed;
    const u32x4 *dy = reinterpret_cast<const u32x4 *>(p.in) + (size_t)token * p.units;
    float dot = 0.f;
    if (here) {
        const u32x4 *row = reinterpret_cast<const u32x4 *>(p.rows) + (size_t)at * p.units;
        u32x4 *to = reinterpret_cast<u32x4 *>(p.out) + (size_t)at * p.units;
        for (int unit0 = lane; unit0 < p.units; unit0 += 64 * kAhead) {
            u32x4 d[kAhead], v[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const int unit = unit0 + 64 * i;
                if (unit < p.units) {
                    v[i] = LAST ? __builtin_nontemporal_load(row + unit) : row[unit];
                    d[i] = dy[unit];
                }
            }
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const int unit = unit0 + 64 * i;
                if (unit >= p.units) break;
                u32x4 o;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    o[e] = bf16_pair(w * bf16_low(d[i][e]), w * bf16_high(d[i][e]));
                    dot = fmaf(bf16_low(d[i][e]), bf16_low(v[i][e]), dot);
                    dot = fmaf(bf16_high(d[i][e]), bf16_high(v[i][e]), dot);
                }
                to[unit] = o;
            }
        }
    } else if ((unsigned)at < (unsigned)pairs) {
        for (int unit = lane; unit < p.units; unit += 64) reinterpret_cast<u32x4 *>(p.out)[(size_t)at * p.units + unit] = u32x4{0u, 0u, 0u, 0u};
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) dot += __shfl_xor(dot, d);
    if (lane == 0) p.d_weights[pair] = dot;
}

// ---- the entry points' checks --------------------------------------------------------------------------------------
// rows of `width` bf16 values for m tokens: KILN_W4A16_OK, or why not
kiln_marlin_status_t rows_ok(int m, int top_k, int experts, int width) {
    if (m < 0 || width < 1 || width % 8 != 0) return KILN_W4A16_ERR_PROB_SHAPE;
    if (top_k < 1 || top_k > kMaxTop || experts < 1 || experts > kMaxExperts || (int64_t)m * top_k > kMaxPairs) return KILN_W4A16_ERR_KERN_SHAPE;
    return launchable(((int64_t)m * (width / 8) + 255) / 256, 256) ? KILN_W4A16_OK : KILN_W4A16_ERR_KERN_SHAPE;
}
int sort_block_pairs(int pairs) {
    const int each = pairs <= kSortBlockPairs ? std::max(pairs, 1) : std::max(kSortBlockPairs, (pairs + kSortMaxBlocks - 1) / kSortMaxBlocks);
    return (each + kSortThreads - 1) / kSortThreads * kSortThreads;
}
int sort_blocks(int pairs) {
    const int each = sort_block_pairs(pairs);
    return pairs ? (pairs + each - 1) / each : 1;
}
kiln_marlin_status_t launched() { return hipGetLastError() == hipSuccess ? KILN_W4A16_OK : KILN_W4A16_ERR_LAUNCH; }
unsigned thread_blocks(int m, int units) { return (unsigned)(((size_t)m * units + 255) / 256); }

}  // namespace
}  // namespace kiln

using namespace kiln;

extern "C" {

size_t kiln_w4a16_moe_sort_scratch_bytes(int prob_m, int top_k, int experts) {
    if (rows_ok(prob_m, top_k, experts, 8) != KILN_W4A16_OK) return 0;
    const int blocks = sort_blocks(prob_m * top_k);
    return blocks == 1 ? 0 : (size_t)blocks * (experts + 1) * sizeof(int);
}

kiln_marlin_status_t kiln_w4a16_moe_sort(const int *expert_of, int prob_m, int top_k, int experts, int *order, int *first, int *place, int dev,
                                         void *stream, void *scratch) {
    (void)dev;
    if (const kiln_marlin_status_t st = rows_ok(prob_m, top_k, experts, 8)) return st;
    const int pairs = prob_m * top_k;
    const int each = sort_block_pairs(pairs), blocks = sort_blocks(pairs);
    if (!all_on(4, {first}) || (blocks > 1 && !all_on(4, {scratch})) || (pairs && !all_on(4, {expert_of, order, place}))) return KILN_W4A16_ERR_ARGUMENT;
    const size_t bytes = (size_t)pairs * 4;
    if (any_meet({{order, bytes}, {place, bytes}, {first, ((size_t)experts + 1) * 4}, {scratch, kiln_w4a16_moe_sort_scratch_bytes(prob_m, top_k, experts)}},
                 {{expert_of, bytes}}))
        return KILN_W4A16_ERR_ARGUMENT;
    hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
    const SortArgs a{expert_of, order, first, place, static_cast<int *>(scratch), pairs, experts, each};
    if (blocks > 1) moe_count_kernel<<<blocks, kSortThreads, 0, hs>>>(a);
    moe_sort_kernel<<<blocks, kSortThreads, 0, hs>>>(a);
    return launched();
}

kiln_marlin_status_t kiln_w4a16_moe_gather(const void *x, const int *first, const int *place, void *rows, int prob_m, int top_k, int experts,
                                           int width, int dev, void *stream) {
    (void)dev;
    if (const kiln_marlin_status_t st = rows_ok(prob_m, top_k, experts, width)) return st;
    if (prob_m == 0) return KILN_W4A16_OK;
    if (!all_on(16, {x, rows}) || !all_on(4, {first, place})) return KILN_W4A16_ERR_ARGUMENT;
    const size_t pairs = (size_t)prob_m * top_k, first_bytes = ((size_t)experts + 1) * 4;
    if (any_meet({{rows, pairs * width * 2}}, {{x, (size_t)prob_m * width * 2}, {first, first_bytes}, {place, pairs * 4}})) return KILN_W4A16_ERR_ARGUMENT;
    const RowsArgs a{(const uint16_t *)x, nullptr, nullptr, first, place, (uint16_t *)rows, nullptr, prob_m, top_k, experts, width / 8};
    moe_gather_kernel<<<thread_blocks(prob_m, width / 8), 256, 0, reinterpret_cast<hipStream_t>(stream)>>>(a);
    return launched();
}

kiln_marlin_status_t kiln_w4a16_moe_combine(const void *rows, const float *weights, const int *first, const int *place, void *y, int prob_m, int top_k,
                                            int experts, int width, int dev, void *stream) {
    (void)dev;
    if (const kiln_marlin_status_t st = rows_ok(prob_m, top_k, experts, width)) return st;
    if (prob_m == 0) return KILN_W4A16_OK;
    if (!all_on(16, {rows, y}) || !all_on(4, {first, place}) || reinterpret_cast<uintptr_t>(weights) % 4 != 0) return KILN_W4A16_ERR_ARGUMENT;
    const size_t pairs = (size_t)prob_m * top_k, first_bytes = ((size_t)experts + 1) * 4;
    if (any_meet({{y, (size_t)prob_m * width * 2}}, {{rows, pairs * width * 2}, {weights, pairs * 4}, {first, first_bytes}, {place, pairs * 4}}))
        return KILN_W4A16_ERR_ARGUMENT;
    const RowsArgs a{(const uint16_t *)rows, nullptr, weights, first, place, (uint16_t *)y, nullptr, prob_m, top_k, experts, width / 8};
    moe_combine_kernel<<<thread_blocks(prob_m, width / 8), 256, 0, reinterpret_cast<hipStream_t>(stream)>>>(a);
    return launched();
}

kiln_marlin_status_t kiln_w4a16_moe_combine_backward(const void *dy, const void *rows, const float *weights, const int *first, const int *place,
                                                     void *d_rows, float *d_weights, int prob_m, int top_k, int experts, int width, int dev, void *stream) {
    (void)dev;
    if (const kiln_marlin_status_t st = rows_ok(prob_m, top_k, experts, width)) return st;
    const int64_t blocks = ((int64_t)prob_m * top_k + 3) / 4;
    if (!launchable(blocks, 256)) return KILN_W4A16_ERR_KERN_SHAPE;
    if (prob_m == 0) return KILN_W4A16_OK;
    if (!all_on(16, {dy, rows, d_rows}) || !all_on(4, {weights, first, place, d_weights})) return KILN_W4A16_ERR_ARGUMENT;
    const size_t pairs = (size_t)prob_m * top_k, first_bytes = ((size_t)experts + 1) * 4;
    if (any_meet({{d_rows, pairs * width * 2}, {d_weights, pairs * 4}},
                 {{dy, (size_t)prob_m * width * 2}, {rows, pairs * width * 2}, {weights, pairs * 4}, {first, first_bytes}, {place, pairs * 4}}))
        return KILN_W4A16_ERR_ARGUMENT;
    const RowsArgs a{(const uint16_t *)dy, (const uint16_t *)rows, weights, first, place, (uint16_t *)d_rows, d_weights, prob_m, top_k, experts, width / 8};
    hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
    const bool last = pairs * width * 2 >= (size_t)48 << 20;
    if (last) moe_combine_backward_kernel<true><<<(unsigned)blocks, 256, 0, hs>>>(a);
    else moe_combine_backward_kernel<false><<<(unsigned)blocks, 256, 0, hs>>>(a);
    return launched();
}

}  // extern "C"
