// The experts of a mixture-of-experts MLP for a few tokens, and the router's choice of them.
//
// Two launches over the packs of the experts that have rows, which is what the call has to read (a token of 8 experts of 64 reads an
// eighth of the layer): gate, up and silu(gate) * up of every (token, expert) pair, then the down projection with the sum over a token's
// experts.  A block works out by itself which experts are present and which pairs are theirs: the ids of a run, 64 tokens at most, are a
// few KB, and a launch in front that sorts them costs more than reading them in every block.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "device_common.h"
#include "kiln_w4a16.h"

namespace kiln {
namespace {

constexpr int kMoeRun = 64;        // tokens of one pair of launches
constexpr int kMoeMaxTop = 16;
constexpr int kMoeMaxExperts = 1024;
constexpr int kMoeMaxPairs = kMoeRun * kMoeMaxTop;

struct MoeArgs {
    const uint16_t *x;          // bf16 [tokens, hidden]
    const int *expert_of;       // [tokens, top]
    const float *weights;       // [tokens, top]
    const u32x4 *b_in, *b_out;  // packs, one expert after the other
    const uint16_t *s_in, *s_out;
    uint16_t *h;                // bf16 [pairs, n_out]
    uint16_t *y;                // bf16 [tokens, n_down]
    int tokens, top, experts, hidden, n_out, n_down, per_column;
};

// The pairs of a run in LDS: ids (-1: none; also for a pair whose expert its token names earlier: that pair's weight goes to the earlier
// one) and which experts are present.
struct MoePairs {
    int id[kMoeMaxPairs];
    float weight[kMoeMaxPairs];
    unsigned present[kMoeMaxExperts / 32];
};

__device__ __forceinline__ void read_pairs(const MoeArgs &p, MoePairs &lds, int tid, int threads) {
    for (int i = tid; i < kMoeMaxExperts / 32; i += threads) lds.present[i] = 0u;
    __syncthreads();
    const int pairs = p.tokens * p.top;
    for (int i = tid; i < pairs; i += threads) {
        int e = p.expert_of[i];
        float w = p.weights[i];
        const int first = i - i % p.top;
        if ((unsigned)e >= (unsigned)p.experts) e = -1;
        for (int j = first; j < first + p.top; ++j)
            if (j != i && e >= 0 && p.expert_of[j] == e) {
                if (j < i) e = -1;
                else w += p.weights[j];
            }
        lds.id[i] = e;
        lds.weight[i] = w;
        if (e >= 0) atomicOr(&lds.present[e >> 5], 1u << (e & 31));
    }
    __syncthreads();
}

// How many experts are present, and the one in place `slot` among them (-1: there are fewer).  Every lane gets both.
__device__ __forceinline__ int expert_in_slot(const MoePairs &lds, int slot, int lane, int *count) {
    const unsigned word = lane < kMoeMaxExperts / 32 ? lds.present[lane] : 0u;
    int upto = __popc(word);
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int below = __shfl_up(upto, d);
        if (lane >= d) upto += below;
    }
    *count = __builtin_amdgcn_readlane(upto, 31);
    if (slot >= *count) return -1;
    const int at = __builtin_ctzll(__ballot(lane < 32 && upto > slot));
    unsigned w = __builtin_amdgcn_readlane(word, at);
    for (int skip = slot - (__builtin_amdgcn_readlane(upto, at) - __popc(w)); skip > 0; --skip) w &= w - 1;
    return at * 32 + __builtin_ctz(w);
}

// The pairs of expert e in their order, into a list of this wavefront's own (64: a token is there at most once).  Returns their count.
__device__ __forceinline__ int pairs_of(const MoePairs &lds, int pairs, int e, int lane, int *list) {
    int count = 0;
    for (int p0 = 0; p0 < pairs; p0 += 64) {
        const bool mine = p0 + lane < pairs && lds.id[p0 + lane] == e;
        const unsigned long long all = __ballot(mine);
        if (mine) list[count + __popcll(all & ((1ull << lane) - 1))] = p0 + lane;
        count += __popcll(all);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    return count;
}

// 16 rows times the chunks of column tiles nt ... nt + CT - 1, groups g0, g0 + stride, ... < G: the f32 sums, scales applied.
// row: this lane's row of the left operand, 8 * (lane / 16) values in.  The sum of a row over a group, which the zero-point and the
// bias of the expanded codes are taken off with, comes out of a product with ones.
template <int CT>
__device__ __forceinline__ void expert_product(const uint16_t *__restrict__ row, const u32x4 *__restrict__ b, const uint16_t *__restrict__ s, int G,
                                               int nt, int g0, int stride, bool per_column, int lane, const DequantConsts &dc, f32x4 (&total)[CT]) {
    const int c = lane & 15;
    const bf16x8 ones = bf16x8_splat_one();
    for (int g = g0; g < G; g += stride) {
        u32x4 w[CT];
        float scale[CT];
        bf16x8 x[4];
#pragma unroll
        for (int i = 0; i < CT; ++i) {
            w[i] = b[((size_t)(nt + i) * G + g) * 64 + lane];
            scale[i] = f16_bits_to_f32(s[scale_index(per_column ? 0 : g, (nt + i) * kTileN + c, per_column ? 1 : G)]);
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) x[t] = *reinterpret_cast<const bf16x8 *>(row + g * kGroupK + 32 * t);
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < 4; ++t) sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[t], ones, sum, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < CT; ++i) {
            f32x4 acc = {0.f, 0.f, 0.f, 0.f};
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[0], codes_to_bf16x8(w[i].x, dc), acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[1], codes_to_bf16x8(w[i].y, dc), acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[2], codes_to_bf16x8(w[i].z, dc), acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[3], codes_to_bf16x8(w[i].w, dc), acc, 0, 0, 0);
#pragma unroll
            for (int e = 0; e < 4; ++e) total[i][e] += scale[i] * (acc[e] - kCodeBias * sum[e]);
        }
    }
}

// h[pair] = silu(gate) * up: a block takes kInTiles column tiles (8 gate and 8 up columns each) of the expert in slot blockIdx.y, its
// wavefronts every fourth group; they meet in LDS.
constexpr int kInTiles = 2;
__global__ __launch_bounds__(256) void moe_in_kernel(MoeArgs p) {
    __shared__ MoePairs pairs;
    __shared__ int lists[4][kMoeRun];
    __shared__ float part[4][16][kInTiles * 16 + 1];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 15, q = lane >> 4;
    const DequantConsts dc = dequant_consts();
    read_pairs(p, pairs, tid, 256);
    int present;
    const int e = expert_in_slot(pairs, blockIdx.y, lane, &present);
    if (e < 0) return;
    int *list = lists[wave];
    const int count = pairs_of(pairs, p.tokens * p.top, e, lane, list);
    const int G = p.hidden / kGroupK, nt = blockIdx.x * kInTiles, N = 2 * p.n_out;
    const u32x4 *b = p.b_in + (size_t)e * (N / kTileN) * G * 64;
    const uint16_t *s = p.s_in + (size_t)e * N * (p.per_column ? 1 : G);
    for (int r0 = 0; r0 < count; r0 += 16) {
        const uint16_t *row = p.x + (size_t)(list[min(r0 + c, count - 1)] / p.top) * p.hidden + 8 * q;
        f32x4 total[kInTiles] = {};
        expert_product<kInTiles>(row, b, s, G, nt, wave, 4, p.per_column, lane, dc, total);
#pragma unroll
        for (int i = 0; i < kInTiles; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) part[wave][4 * q + r][16 * i + c] = total[i][r];
        __syncthreads();
        const int r = tid >> 4, col = (tid & 15) + (tid & 8);  // 8 gate columns of the first tile, 8 of the second
        if (r0 + r < count) {
            const float gate = (part[0][r][col] + part[1][r][col]) + (part[2][r][col] + part[3][r][col]);
            const float up = (part[0][r][col + 8] + part[1][r][col + 8]) + (part[2][r][col + 8] + part[3][r][col + 8]);
            p.h[(size_t)list[r0 + r] * p.n_out + nt * 8 + (tid & 15)] = f32_to_bf16_bits(gate * __builtin_amdgcn_rcpf(1.f + __expf(-gate)) * up);
        }
        __syncthreads();
    }
}

// y[token] = sum over its experts: a block takes one column tile for all tokens; its wavefronts share out the present experts (and, where
// those are fewer than wavefronts, parts of their groups), each with an f32 sum per token and column in LDS, added up at the end in the
// wavefronts' order.
constexpr int kOutWaves = 8;
__global__ __launch_bounds__(kOutWaves * 64) void moe_out_kernel(MoeArgs p) {
    __shared__ MoePairs pairs;
    __shared__ int lists[kOutWaves][kMoeRun];
    __shared__ float sums[kOutWaves][kMoeRun][16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 15, q = lane >> 4;
    const DequantConsts dc = dequant_consts();
    for (int i = lane; i < p.tokens * 16; i += 64) sums[wave][i >> 4][i & 15] = 0.f;
    read_pairs(p, pairs, tid, kOutWaves * 64);
    int present;
    expert_in_slot(pairs, 0, lane, &present);
    const int G = p.n_out / kGroupK, nt = blockIdx.x, N = p.n_down;
    if (present) {
        const int parts = min(G, (kOutWaves + present - 1) / present);
        int *list = lists[wave];
        for (int unit = wave; unit < present * parts; unit += kOutWaves) {
            int again;
            const int slot = unit / parts, e = expert_in_slot(pairs, slot, lane, &again);
            const int count = pairs_of(pairs, p.tokens * p.top, e, lane, list);
            const u32x4 *b = p.b_out + (size_t)e * (N / kTileN) * G * 64;
            const uint16_t *s = p.s_out + (size_t)e * N * (p.per_column ? 1 : G);
            for (int r0 = 0; r0 < count; r0 += 16) {
                const uint16_t *row = p.h + (size_t)list[min(r0 + c, count - 1)] * p.n_out + 8 * q;
                f32x4 total[1] = {};
                expert_product<1>(row, b, s, G, nt, unit - slot * parts, parts, p.per_column, lane, dc, total);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int at = r0 + 4 * q + r;
                    if (at < count) sums[wave][list[at] / p.top][c] += pairs.weight[list[at]] * total[0][r];
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
    }
    __syncthreads();
    for (int i = tid; i < p.tokens * 16; i += kOutWaves * 64) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kOutWaves; ++w) v += sums[w][i >> 4][i & 15];
        p.y[(size_t)(i >> 4) * N + nt * 16 + (i & 15)] = f32_to_bf16_bits(v);
    }
}

// ---- the router's choice -------------------------------------------------------------------------------------------
// A wavefront per row, V logits to a lane (expert lane + 64 v).  `top` times the largest that is left, ties to the lowest index, as
// one comparison of (value, index) across the lanes.
template <class T>
__device__ __forceinline__ float logit(const T *p) {
    if constexpr (sizeof(T) == 4) return *p;
    else return (float)*p;
}
template <class T, int V>
__global__ __launch_bounds__(256) void moe_route_kernel(const T *__restrict__ logits, int rows, int experts, int top, int renormalise,
                                                        int *__restrict__ expert_of, float *__restrict__ weights) {
    const int lane = threadIdx.x & 63, row = blockIdx.x * 4 + (int)(threadIdx.x >> 6);
    if (row >= rows) return;
    float v[V];
    float most = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int e = lane + 64 * i;
        v[i] = e < experts ? logit(logits + (size_t)row * experts + e) : -INFINITY;
        if (v[i] != v[i]) {
            nan = true;
            v[i] = -INFINITY;
        }
        most = fmaxf(most, v[i]);
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) most = fmaxf(most, __shfl_xor(most, d));
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) sum += __expf(v[i] - most);
#pragma unroll
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    const bool poisoned = __any(nan) || most == INFINITY, empty = most == -INFINITY;
    float my_weight = 0.f, chosen = 0.f;
    int my_id = -1;
    for (int k = 0; k < top; ++k) {
        float best = v[0];
        int at = lane;
#pragma unroll
        for (int i = 1; i < V; ++i)
            if (v[i] > best) {
                best = v[i];
                at = lane + 64 * i;
            }
#pragma unroll
        for (int d = 32; d; d >>= 1) {
            const float other = __shfl_xor(best, d);
            const int other_at = __shfl_xor(at, d);
            if (other > best || (other == best && other_at < at)) {
                best = other;
                at = other_at;
            }
        }
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (at == lane + 64 * i) v[i] = -INFINITY;
        const float w = best == -INFINITY ? 0.f : __expf(best - most);
        chosen += w;
        if (lane == k) {
            my_id = best == -INFINITY ? -1 : at;
            my_weight = w;
        }
    }
    if (lane < top) {
        const float over = renormalise ? chosen : sum;
        expert_of[(size_t)row * top + lane] = my_id;
        weights[(size_t)row * top + lane] = poisoned ? NAN : empty ? 0.f : my_weight / over;
    }
}

template <class T>
void launch_route(const void *logits, int rows, int experts, int top, int renormalise, int *of, float *weights, hipStream_t stream) {
    const T *l = (const T *)logits;
    const unsigned grid = (unsigned)((rows + 3) / 4);
    const int per_lane = (experts + 63) / 64;
    if (per_lane <= 1) moe_route_kernel<T, 1><<<grid, 256, 0, stream>>>(l, rows, experts, top, renormalise, of, weights);
    else if (per_lane <= 2) moe_route_kernel<T, 2><<<grid, 256, 0, stream>>>(l, rows, experts, top, renormalise, of, weights);
    else if (per_lane <= 4) moe_route_kernel<T, 4><<<grid, 256, 0, stream>>>(l, rows, experts, top, renormalise, of, weights);
    else if (per_lane <= 8) moe_route_kernel<T, 8><<<grid, 256, 0, stream>>>(l, rows, experts, top, renormalise, of, weights);
    else moe_route_kernel<T, 16><<<grid, 256, 0, stream>>>(l, rows, experts, top, renormalise, of, weights);
}

}  // namespace
}  // namespace kiln

using namespace kiln;

extern "C" {

size_t kiln_w4a16_moe_scratch_bytes(int prob_m, int top_k, int n_out, int n_down) {
    (void)n_down;
    if (prob_m < 1 || top_k < 1 || n_out < 1) return 256;
    return (size_t)(prob_m < kMoeRun ? prob_m : kMoeRun) * top_k * n_out * 2;
}

kiln_marlin_status_t kiln_w4a16_moe(const void *x, const int *expert_of, const float *weights, const void *b_gate_up, const void *s_gate_up,
                                    const void *b_down, const void *s_down, void *y, int prob_m, int top_k, int experts, int hidden, int n_out,
                                    int n_down, int groupsize, int dev, void *stream, void *scratch) {
    (void)dev;
    if (prob_m < 0 || hidden <= 0 || n_out <= 0 || n_down <= 0 || hidden % 128 != 0 || n_out % 128 != 0 || n_down % 256 != 0 ||
        n_out > INT32_MAX / 2 || (groupsize != -1 && groupsize != 128))
        return KILN_W4A16_ERR_PROB_SHAPE;
    if (top_k < 1 || top_k > kMoeMaxTop || experts < 1 || experts > kMoeMaxExperts) return KILN_W4A16_ERR_KERN_SHAPE;
    if (prob_m == 0) return KILN_W4A16_OK;
    if (!x || !expert_of || !weights || !b_gate_up || !s_gate_up || !b_down || !s_down || !y || !scratch) return KILN_W4A16_ERR_ARGUMENT;
    for (const void *p : {x, b_gate_up, s_gate_up, b_down, s_down, static_cast<const void *>(y), static_cast<const void *>(scratch)})
        if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return KILN_W4A16_ERR_ARGUMENT;
    hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
    for (int m0 = 0; m0 < prob_m; m0 += kMoeRun) {
        const int m = prob_m - m0 < kMoeRun ? prob_m - m0 : kMoeRun;
        MoeArgs a{(const uint16_t *)x + (size_t)m0 * hidden, expert_of + (size_t)m0 * top_k, weights + (size_t)m0 * top_k,
                  (const u32x4 *)b_gate_up, (const u32x4 *)b_down, (const uint16_t *)s_gate_up, (const uint16_t *)s_down,
                  (uint16_t *)scratch, (uint16_t *)y + (size_t)m0 * n_down, m, top_k, experts, hidden, n_out, n_down, groupsize == -1};
        const int slots = m * top_k < experts ? m * top_k : experts;
        moe_in_kernel<<<dim3(2 * n_out / (16 * kInTiles), slots), 256, 0, hs>>>(a);
        moe_out_kernel<<<n_down / 16, kOutWaves * 64, 0, hs>>>(a);
    }
    return hipGetLastError() == hipSuccess ? KILN_W4A16_OK : KILN_W4A16_ERR_LAUNCH;
}

kiln_marlin_status_t kiln_w4a16_moe_route(const void *logits, int dtype, int prob_m, int experts, int top_k, int renormalise, int *expert_of,
                                    float *weights, int dev, void *stream) {
    (void)dev;
    if (prob_m < 0) return KILN_W4A16_ERR_PROB_SHAPE;
    if (experts < 1 || experts > kMoeMaxExperts || top_k < 1 || top_k > kMoeMaxTop || top_k > experts || dtype < 0 || dtype > 2)
        return KILN_W4A16_ERR_KERN_SHAPE;
    if (prob_m == 0) return KILN_W4A16_OK;
    if (!logits || !expert_of || !weights) return KILN_W4A16_ERR_ARGUMENT;
    hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
    if (dtype == 0) launch_route<float>(logits, prob_m, experts, top_k, renormalise, expert_of, weights, hs);
    else if (dtype == 1) launch_route<__bf16>(logits, prob_m, experts, top_k, renormalise, expert_of, weights, hs);
    else launch_route<_Float16>(logits, prob_m, experts, top_k, renormalise, expert_of, weights, hs);
    return hipGetLastError() == hipSuccess ? KILN_W4A16_OK : KILN_W4A16_ERR_LAUNCH;
}

}  // extern "C"
