// The experts of a mixture-of-experts MLP for a few tokens, and the router's choice of them.
//
// Bound by the packs of the experts that have rows, read once (a token of 8 experts of 64 reads an eighth of the layer).  Two launches or
// three: gate, up and silu(gate) * up of every (token, expert) pair, then the down projection of every pair and the sum over a token's.  A
// block works out by itself which experts are present and which pairs are theirs: the ids of a run, 64 tokens at most, are a few KB,
// and a launch in front that sorts them costs more than reading them in every block.
//
// silu(gate) * up is rounded to bf16 in between, as in the MLP of one pack (kiln_w4a16_mlp) and in the reference's: the second product's operand is bf16.
// It is what takes the result's error against 64 bits from 0.0017 of its norm, its own rounding, to 0.0023.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "bank.h"
#include "device_common.h"
#include "few_rows.h"
#include "kiln_w4a16.h"
#include "launch.h"

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
    float *down;                // f32 [pairs, n_down]
    uint16_t *y;                // bf16 [tokens, n_down]
    int tokens, top, experts, hidden, n_out, n_down, per_column;
};

// Which experts are present among a run's pairs, and which pairs are theirs.  A wavefront looks at the pairs of as many whole tokens as
// fit its lanes at a time, ids in registers (FEW: all of them fit) or LDS.
struct MoePairs {
    int id[kMoeMaxPairs];  // -1: none
    unsigned present[kMoeMaxExperts / 32];
};

__device__ __forceinline__ int id_of(const MoeArgs &p, int pair, int pairs) {
    const int e = pair < pairs ? p.expert_of[pair] : -1;
    return (unsigned)e < (unsigned)p.experts ? e : -1;
}
// the expert in place `slot` in the order in which they are met (-1: there are fewer)
__device__ __forceinline__ int expert_in_lanes(int id, int slot) {
    for (unsigned long long left = __ballot(id >= 0); left; --slot) {
        const int e = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
        if (slot == 0) return e;
        left &= ~__ballot(id == e);
    }
    return -1;
}
__device__ __forceinline__ void read_pairs(const MoeArgs &p, MoePairs &lds, int tid, int threads) {
    for (int i = tid; i < kMoeMaxExperts / 32; i += threads) lds.present[i] = 0u;
    __syncthreads();
    const int pairs = p.tokens * p.top;
    for (int i = tid; i < pairs; i += threads) {
        const int e = id_of(p, i, pairs);
        lds.id[i] = e;
        if (e >= 0) atomicOr(&lds.present[e >> 5], 1u << (e & 31));
    }
    __syncthreads();
}
// ... and out of LDS, in the order of their ids
__device__ __forceinline__ int expert_in_lds(const MoePairs &lds, int slot, int lane) {
    const unsigned word = lane < kMoeMaxExperts / 32 ? lds.present[lane] : 0u;
    int upto = __popc(word);
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int below = __shfl_up(upto, d);
        if (lane >= d) upto += below;
    }
    if (slot >= __builtin_amdgcn_readlane(upto, 31)) return -1;
    const int at = __builtin_ctzll(__ballot(lane < 32 && upto > slot));
    unsigned w = __builtin_amdgcn_readlane(word, at);
    for (int skip = slot - (__builtin_amdgcn_readlane(upto, at) - __popc(w)); skip > 0; --skip) w &= w - 1;
    return at * 32 + __builtin_ctz(w);
}
// The pairs of expert e in their order, into a list of this wavefront's own; of a token that names e more than once the first, so 64 at
// most.  Returns their count.
__device__ __forceinline__ int pairs_of(const MoeArgs &p, const MoePairs *lds, int id_in_lane, int e, int lane, int *list) {
    const int pairs = p.tokens * p.top, step = 64 / p.top * p.top;
    const int before = lane - lane % p.top;                                        // the first of this lane's token
    const unsigned long long earlier = ((1ull << lane) - 1) & ~((1ull << before) - 1);  // ... and those between it and this lane
    int count = 0;
    for (int p0 = 0; p0 < pairs; p0 += step) {
        const int pair = p0 + lane, id = lds ? (lane < step && pair < pairs ? lds->id[pair] : -1) : id_in_lane;
        const bool mine = id == e && (__ballot(id == e) & earlier) == 0;
        const unsigned long long firsts = __ballot(mine);
        if (mine) list[count + __popcll(firsts & ((1ull << lane) - 1))] = pair;
        count += __popcll(firsts);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    return count;
}

// Up to 16 rows of one expert times S column tiles of its pack (few_rows.h); the wavefronts meet in LDS at the end.
// With the rows read again for every tile or two (64 tokens, 8 of 64 experts, 2560 -> 1024 -> 2560) the two launches took 54 and 51 us, not
// 39 and 25: the wavefronts waited for rows, 4 KB of them to a KB of codes.
template <bool IN, bool FEW, int W, int GW, int S>
__global__ __launch_bounds__(W * 64) void moe_expert_kernel(MoeArgs p) {
    __shared__ MoePairs pairs;
    __shared__ int lists[W][kMoeRun];
    constexpr int kPitch = S * 16 + 4;
    __shared__ float part[W][16][kPitch];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, q = lane >> 4;
    const DequantConsts dc = dequant_consts();
    int e, id = -1;
    if constexpr (FEW) {
        id = id_of(p, lane, p.tokens * p.top);
        e = expert_in_lanes(id, blockIdx.y);
    } else {
        read_pairs(p, pairs, tid, W * 64);
        e = expert_in_lds(pairs, blockIdx.y, lane);
    }
    if (e < 0) return;
    int *list = lists[wave];
    const int count = pairs_of(p, FEW ? nullptr : &pairs, id, e, lane, list);
    const int K = IN ? p.hidden : p.n_out, N = IN ? 2 * p.n_out : p.n_down, G = K / kGroupK, Gs = p.per_column ? 1 : G;
    const int nt0 = blockIdx.x * S;
    const u32x4 *b = (IN ? p.b_in : p.b_out) + ((size_t)e * (N / kTileN) + nt0) * G * 64 + lane;
    const uint16_t *s = (IN ? p.s_in : p.s_out) + ((size_t)e * (N / kTileN) + nt0) * Gs * kTileN + c;
    for (int r0 = 0; r0 < count; r0 += 16) {
        const int pair = list[min(r0 + c, count - 1)];
        const uint16_t *row = (IN ? p.x + (size_t)(pair / p.top) * K : p.h + (size_t)pair * K) + 8 * q;
        f32x4 total[S];
        few_rows_product<GW, S>(row, b, s, G, p.per_column, wave, W, dc, total);
#pragma unroll
        for (int i = 0; i < S; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) part[wave][4 * q + r][16 * i + c] = total[i][r];
        __syncthreads();
        auto sum_of = [&](int r, int col) {
            float v = 0.f;
#pragma unroll
            for (int i = 0; i < W; ++i) v += part[i][r][col];
            return v;
        };
        const int rows = min(16, count - r0);
        if constexpr (IN) {  // 8 gate columns of a tile, then the 8 matching up columns
            for (int i = tid; i < rows * S * 8; i += W * 64) {
                const int r = i / (S * 8), j = i % (S * 8), col = 16 * (j >> 3) + (j & 7);
                const float gate = sum_of(r, col), up = sum_of(r, col + 8);
                p.h[(size_t)list[r0 + r] * p.n_out + nt0 * 8 + j] = f32_to_bf16_bits(gate * __builtin_amdgcn_rcpf(1.f + __expf(-gate)) * up);
            }
        } else {
            for (int i = tid; i < rows * S * 16; i += W * 64) {
                const int r = i / (S * 16), col = i % (S * 16);
                p.down[(size_t)list[r0 + r] * N + nt0 * 16 + col] = sum_of(r, col);
            }
        }
        __syncthreads();
    }
}

// The down projection and the sum in one launch, for as many pairs as a block has wavefronts: a block takes one column tile for all tokens, its
// wavefronts share out the experts present (and, where those are fewer, parts of their groups), each with an f32 sum per token and column in
// LDS, added up in the wavefronts' order.  8 pairs (2560 -> 1024 -> 2560) 13.5 us a call against 15.4 with the two launches; experts beyond the
// wavefronts would come one after the other: 16 pairs 21.6 against 20.5.
constexpr int kJoinWaves = 8, kMoeJoinedPairs = kJoinWaves;
template <int GW>
__global__ __launch_bounds__(kJoinWaves * 64) void moe_join_kernel(MoeArgs p) {
    __shared__ int lists[kJoinWaves][kMoeRun];
    __shared__ float sums[kJoinWaves][kMoeJoinedPairs][16];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, q = lane >> 4;
    const DequantConsts dc = dequant_consts();
    const int pairs = p.tokens * p.top, id = id_of(p, lane, pairs);
    const float weight = lane < pairs ? p.weights[lane] : 0.f;
    for (int i = lane; i < p.tokens * 16; i += 64) sums[wave][i >> 4][i & 15] = 0.f;
    int present = 0;
    for (unsigned long long left = __ballot(id >= 0); left; ++present) left &= ~__ballot(id == __builtin_amdgcn_readlane(id, __builtin_ctzll(left)));
    const int G = p.n_out / kGroupK, Gs = p.per_column ? 1 : G, nt = blockIdx.x, tiles = p.n_down / kTileN;
    const int parts = present ? min((G + GW - 1) / GW, (kJoinWaves + present - 1) / present) : 1;
    int *list = lists[wave];
    for (int unit = wave; unit < present * parts; unit += kJoinWaves) {
        const int e = expert_in_lanes(id, unit / parts), count = pairs_of(p, nullptr, id, e, lane, list);
        const unsigned long long named = __ballot(id == e);
        for (int r0 = 0; r0 < count; r0 += 16) {
            f32x4 total[1];
            few_rows_product<GW, 1>(p.h + (size_t)list[min(r0 + c, count - 1)] * p.n_out + 8 * q, p.b_out + ((size_t)e * tiles + nt) * G * 64 + lane,
                                    p.s_out + ((size_t)e * tiles + nt) * Gs * kTileN + c, G, p.per_column, unit % parts, parts, dc, total);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int pair = list[min(r0 + 4 * q + i, count - 1)], token = pair / p.top;
                float w = __shfl(weight, pair);
                if (__popcll(named) != count)  // some token names the expert again: its weights together
                    for (int j = 1; j < p.top; ++j) {
                        const int other = min(pair + j, 63);
                        const float more = __shfl(weight, other);
                        if (pair + j < (token + 1) * p.top && (named >> other & 1)) w += more;
                    }
                if (r0 + 4 * q + i < count) sums[wave][token][c] += w * total[0][i];
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    __syncthreads();
    for (int i = tid; i < p.tokens * 16; i += kJoinWaves * 64) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kJoinWaves; ++w) v += sums[w][i >> 4][i & 15];
        p.y[(size_t)(i >> 4) * p.n_down + nt * 16 + (i & 15)] = f32_to_bf16_bits(v);
    }
}

// y[token] = sum of its pairs' rows times their weights, in the pairs' order, rounded once; four columns to a thread.  Bound by its
// start and two loads' latency: the rows of eight pairs are asked for together.
__global__ __launch_bounds__(256) void moe_sum_kernel(MoeArgs p) {
    const int lane = threadIdx.x & 63, col = (blockIdx.x * 256 + threadIdx.x) * 4, token = blockIdx.y;
    const int e = lane < p.top ? p.expert_of[(size_t)token * p.top + lane] : -1;
    const float weight = lane < p.top ? p.weights[(size_t)token * p.top + lane] : 0.f;
    const unsigned long long here = __ballot((unsigned)e < (unsigned)p.experts);
    const float *down = p.down + (size_t)token * p.top * p.n_down + min(col, p.n_down - 4);
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    for (int j0 = 0; j0 < p.top; j0 += 8) {
        f32x4 d[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {  // where an expert is named twice its row is with the first
            const int at = __builtin_ctzll(__ballot(e == __builtin_amdgcn_readlane(e, j0 + u)));
            if (here >> (j0 + u) & 1) d[u] = *reinterpret_cast<const f32x4 *>(down + (size_t)at * p.n_down);
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const float w = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, weight), j0 + u));
            if (here >> (j0 + u) & 1)
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] += w * d[u][i];
        }
    }
    if (col >= p.n_down) return;
    u32x2 o;
    o.x = f32_to_bf16_bits(v[0]) | (uint32_t)f32_to_bf16_bits(v[1]) << 16;
    o.y = f32_to_bf16_bits(v[2]) | (uint32_t)f32_to_bf16_bits(v[3]) << 16;
    *reinterpret_cast<u32x2 *>(p.y + (size_t)token * p.n_down + col) = o;
}

// Column tiles to a block: many where the blocks are enough all the same (their rows and lists are read once each), where the experts present
// are few as leave a block to every compute unit (two tokens of 8 experts, 2560 -> 1024 -> 2560: four 20.5 us, two 22.5; a token: 13.5, 13.8, one 15.9).
template <bool IN, bool FEW, int W, int GW>
void launch_expert(const MoeArgs &a, int slots, int cus, hipStream_t stream) {
    constexpr int kMany = W == 4 ? 8 : 4;
    const int tiles = (IN ? 2 * a.n_out : a.n_down) / kTileN;
    if (slots * (tiles / kMany) >= 2 * cus) moe_expert_kernel<IN, FEW, W, GW, kMany><<<dim3(tiles / kMany, slots), W * 64, 0, stream>>>(a);
    else if (slots * (tiles / 4) >= cus) moe_expert_kernel<IN, FEW, W, GW, 4><<<dim3(tiles / 4, slots), W * 64, 0, stream>>>(a);
    else moe_expert_kernel<IN, FEW, W, GW, 2><<<dim3(tiles / 2, slots), W * 64, 0, stream>>>(a);
}
template <bool IN, bool FEW>
void launch_experts(const MoeArgs &a, int slots, int cus, hipStream_t stream) {
    with_few_rows_split((IN ? a.hidden : a.n_out) / kGroupK,
                        [&](auto waves, auto groups) { launch_expert<IN, FEW, decltype(waves)::value, decltype(groups)::value>(a, slots, cus, stream); });
}

// ---- the router's choice -------------------------------------------------------------------------------------------
// A wavefront per row, V logits to a lane (expert lane + 64 v).  `top` times the largest that is left: its value by a reduction across the
// lanes in the vector unit, then the lowest index that holds it by comparison -- no LDS, through which the lanes' exchanges of (value, index)
// pairs took 8192 rows of 128 from 5 us to 14.
template <class F>
__device__ __forceinline__ float across_lanes(float v, float neutral, F &&join) {
    const int n = __builtin_bit_cast(int, neutral);
    auto step = [&](auto ctrl) {
        const int other = __builtin_amdgcn_update_dpp(n, __builtin_bit_cast(int, v), decltype(ctrl)::value, 0xF, 0xF, false);
        v = join(v, __builtin_bit_cast(float, other));
    };
    step(std::integral_constant<int, 0x111>{});  // row_shr 1, 2, 4, 8: each row of 16 lanes into its last
    step(std::integral_constant<int, 0x112>{});
    step(std::integral_constant<int, 0x114>{});
    step(std::integral_constant<int, 0x118>{});
    step(std::integral_constant<int, 0x142>{});  // row_bcast 15, 31: the rows' last lanes into the next rows
    step(std::integral_constant<int, 0x143>{});
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

template <class T, int V>
__global__ __launch_bounds__(256) void moe_route_kernel(const T *__restrict__ logits, int rows, int experts, int top, int renormalise,
                                                        int *__restrict__ expert_of, float *__restrict__ weights) {
    const int lane = threadIdx.x & 63, row = blockIdx.x * 4 + (int)(threadIdx.x >> 6);
    if (row >= rows) return;
    auto larger = [](float a, float b) { return fmaxf(a, b); };
    auto add = [](float a, float b) { return a + b; };
    float v[V];
    float most = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int e = lane + 64 * i;
        v[i] = e < experts ? (float)logits[(size_t)row * experts + e] : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
        nan |= v[i] != v[i];
        v[i] = v[i] != v[i] ? -INFINITY : v[i];
        most = fmaxf(most, v[i]);
    }
    most = across_lanes(most, -INFINITY, larger);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) sum += __expf(v[i] - most);
    sum = across_lanes(sum, 0.f, add);
    const bool poisoned = __any(nan) || most == INFINITY, empty = most == -INFINITY;
    float my_weight = 0.f, chosen = 0.f, best = most;
    int my_id = -1;
    for (int k = 0; k < top && best != -INFINITY; ++k) {
        int at = -1;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const unsigned long long holds = __ballot(v[i] == best);
            if (at < 0 && holds) at = 64 * i + __builtin_ctzll(holds);
        }
        const float w = __expf(best - most);
        chosen += w;
        if (lane == k) {
            my_id = at;
            my_weight = w;
        }
        best = -INFINITY;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (lane + 64 * i == at) v[i] = -INFINITY;
            best = fmaxf(best, v[i]);
        }
        best = across_lanes(best, -INFINITY, larger);
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
    const unsigned grid = ((unsigned)rows + 3) / 4;
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

static size_t moe_h_bytes(int m, int top_k, int n_out) {
    return ((size_t)(m < kMoeRun ? m : kMoeRun) * top_k * n_out * 2 + 255) & ~(size_t)255;
}

size_t kiln_w4a16_moe_scratch_bytes(int prob_m, int top_k, int n_out, int n_down) {
    if (prob_m < 1 || top_k < 1 || n_out < 1 || n_down < 1) return 256;
    return moe_h_bytes(prob_m, top_k, n_out) + (size_t)(prob_m < kMoeRun ? prob_m : kMoeRun) * top_k * n_down * 4;
}

kiln_marlin_status_t kiln_w4a16_moe(const void *x, const int *expert_of, const float *weights, const void *b_gate_up, const void *s_gate_up,
                                    const void *b_down, const void *s_down, void *y, int prob_m, int top_k, int experts, int hidden, int n_out,
                                    int n_down, int groupsize, int dev, void *stream, void *scratch) {
    if (prob_m < 0 || hidden <= 0 || n_out <= 0 || n_down <= 0 || hidden % 128 != 0 || n_out % 128 != 0 || n_down % 256 != 0 ||
        n_out > INT32_MAX / 2 || (groupsize != -1 && groupsize != 128))
        return KILN_W4A16_ERR_PROB_SHAPE;
    if (top_k < 1 || top_k > kMoeMaxTop || experts < 1 || experts > kMoeMaxExperts) return KILN_W4A16_ERR_KERN_SHAPE;
    if (prob_m == 0) return KILN_W4A16_OK;
    if (!x || !expert_of || !weights || !b_gate_up || !s_gate_up || !b_down || !s_down || !y || !scratch) return KILN_W4A16_ERR_ARGUMENT;
    for (const void *p : {x, b_gate_up, s_gate_up, b_down, s_down, static_cast<const void *>(y), static_cast<const void *>(scratch)})
        if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return KILN_W4A16_ERR_ARGUMENT;
    if (meet(y, (size_t)prob_m * n_down * 2, x, (size_t)prob_m * hidden * 2)) return KILN_W4A16_ERR_ARGUMENT;
    hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
    const int cus = compute_units(dev);
    for (int m0 = 0; m0 < prob_m; m0 += kMoeRun) {
        const int m = prob_m - m0 < kMoeRun ? prob_m - m0 : kMoeRun;
        const MoeArgs a{(const uint16_t *)x + (size_t)m0 * hidden, expert_of + (size_t)m0 * top_k, weights + (size_t)m0 * top_k,
                        (const u32x4 *)b_gate_up, (const u32x4 *)b_down, (const uint16_t *)s_gate_up, (const uint16_t *)s_down,
                        (uint16_t *)scratch, reinterpret_cast<float *>(static_cast<char *>(scratch) + moe_h_bytes(prob_m, top_k, n_out)),
                        (uint16_t *)y + (size_t)m0 * n_down, m, top_k, experts, hidden, n_out, n_down, groupsize == -1};
        const int slots = m * top_k < experts ? m * top_k : experts;
        const bool few = m <= 64 / top_k;  // whole tokens in a wavefront's lanes
        if (few) launch_experts<true, true>(a, slots, cus, hs);
        else launch_experts<true, false>(a, slots, cus, hs);
        if (few && m * top_k <= kMoeJoinedPairs) {
            // Groups of the down projection side by side in a wavefront: as many as divide them.  8 pairs of 2048 -> n_out -> 2048, us a call: of 5
            // groups 10.7 (four side by side 12.5), 6 11.7 (12.9), 8 12.7 (four 13.1, five 13.7), 10 16.0 (four 16.5, eight 18.1), 12 17.0
            // (four 17.9, eight 18.4); 7, by four, 13.2 (eight 12.5).  1 to 3 groups ask for their last again, times zero: 9.3, 10.0 and 10.3
            // where as many side by side as there are would take 8.4, 9.5 and 10.1.
            const int G = n_out / kGroupK;
            if (G % 8 == 0) moe_join_kernel<8><<<n_down / 16, kJoinWaves * 64, 0, hs>>>(a);
            else if (G % 6 == 0) moe_join_kernel<6><<<n_down / 16, kJoinWaves * 64, 0, hs>>>(a);
            else if (G % 5 == 0) moe_join_kernel<5><<<n_down / 16, kJoinWaves * 64, 0, hs>>>(a);
            else moe_join_kernel<4><<<n_down / 16, kJoinWaves * 64, 0, hs>>>(a);
            continue;
        }
        if (few) launch_experts<false, true>(a, slots, cus, hs);
        else launch_experts<false, false>(a, slots, cus, hs);
        moe_sum_kernel<<<dim3((n_down / 4 + 255) / 256, m), 256, 0, hs>>>(a);
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
