// A packed projection of up to 16 rows with low-rank adapters of their own, base product and low-rank term in one launch behind the
// projection of the rows onto their adapters (w4a16_bank.hip): the term lands on the f32 sums, and the result is rounded once.
#include "bank.h"
#include "bank_expand.h"
#include "few_rows.h"

namespace kiln {
namespace {

constexpr int kOwnRows = 2;
struct FewArgs {
    const uint16_t *x;
    const u32x4 *b;
    const uint16_t *s;
    uint16_t *y;
    const uint16_t *mat;   // [count, N, rank]
    const uint16_t *mat_a;  // [count, rank, K]
    const float *t;        // [slices, rows, rank], or null: the blocks project the rows by themselves
    const float *scales;
    BankRows rows;
    int K, N, rank, slices, per_column;
};

// One row or two onto their adapters, over the groups that a wavefront has of them: t[row][rank] += x A^T.  The loops are left as they are,
// 16 of the rank of one row a turn with its loads in flight together: unrolled, reading their code took longer.
template <int W, int GW, int SR>
__device__ __forceinline__ void project_own(const FewArgs &p, const bf16x8 (&x)[GW][4], int first, int G, int a, int lane, float (&t)[kOwnRows][32 * SR]) {
    const int c = lane & 15, q = lane >> 4;
#pragma unroll 1
    for (int r = 0; r < p.rows.rows; ++r) {
        const int adapter = __builtin_amdgcn_readlane(a, r);
        if ((unsigned)adapter >= (unsigned)p.rows.count) continue;
#pragma unroll 1
        for (int j0 = 0; j0 < p.rank; j0 += 16) {
            const uint16_t *m = p.mat_a + ((size_t)adapter * p.rank + min(j0 + c, p.rank - 1)) * p.K + 8 * q;
            bf16x8 b[GW][4];
#pragma unroll
            for (int u = 0; u < GW; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) b[u][i] = load_bf16x8(m + min(first + u, G - 1) * kGroupK + 32 * i);
            __builtin_amdgcn_sched_barrier(0);
            f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int u = 0; u < GW; ++u) {
                f32x4 sum = acc;
#pragma unroll
                for (int i = 0; i < 4; ++i) sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[u][i], b[u][i], sum, 0, 0, 0);
                if (first + u < G) acc = sum;
            }
            if (q == 0 && j0 + c < p.rank) t[r][j0 + c] += r == 0 ? acc[0] : acc[1];  // rows 0 and 1 of the product are with the first lanes
        }
    }
}

// S column tiles to a block of W wavefronts, which meet in LDS after the base product.  The adapters met among the rows are dealt out
// to the wavefronts; each finishes and stores the rows of its own (those without an adapter are the first one's).  What that needs of
// memory is touched while the first weights are on their way -- a lane a line or a few of its row's adapter -- and comes out of a cache.
// OWN: one row or two, and every block projects them onto their adapters by itself, out of the part of the rows that its wavefronts hold:
// the adapters' A read by every block is less than the launch in front that it saves.
template <int W, int GW, int S, int SR, bool OWN>
__global__ __launch_bounds__(W * 64) void bank_few_kernel(FewArgs p) {
    constexpr int kMost = 16 / W, kPitch = S * 16 + 4;
    __shared__ __align__(16) float part[W][16][kPitch];
    __shared__ __align__(16) float ts[16][kBankMaxRank + 4];
    __shared__ float parts_of_t[OWN ? W : 1][kOwnRows][32 * SR];
    if constexpr (OWN) {  // (this wavefront's own, until the block meets)
        for (int e = threadIdx.x & 63; e < kOwnRows * 32 * SR; e += 64) (&parts_of_t[threadIdx.x >> 6][0][0])[e] = 0.f;
    }
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, q = lane >> 4;
    const DequantConsts dc = dequant_consts();
    const int nt0 = blockIdx.x * S, G = p.K / kGroupK, Gs = p.per_column ? 1 : G, n0 = nt0 * kTileN;
    const uint16_t *mat = p.mat + (size_t)n0 * p.rank;
    int a = p.rows.of[min(c, p.rows.rows - 1)];
    constexpr int kLines = (S * 16 * SR * 32 / 64 + 4 * W - 1) / (4 * W);  // of 64 values, to a lane
    uint32_t touched[kLines];
    float scale;
    f32x4 total[S];
    few_rows_product<GW, S>(p.x + (size_t)min(c, p.rows.rows - 1) * p.K + 8 * q, p.b + (size_t)nt0 * G * 64 + lane,
                               p.s + (size_t)nt0 * Gs * kTileN + c, G, p.per_column, wave, W, dc, total, [&] {
                                   const size_t at = (unsigned)a < (unsigned)p.rows.count ? a : 0;
                                   scale = p.scales[at];
#pragma unroll
                                   for (int i = 0; i < kLines; ++i)
                                       touched[i] = mat[at * p.N * p.rank + min((4 * (W * i + wave) + q) * 64, S * 16 * p.rank - 1)];
                               },
                               [&](const bf16x8(&x)[GW][4], int first) {
                                   if constexpr (OWN) project_own<W, GW, SR>(p, x, first, G, a, lane, parts_of_t[wave]);
                               });
#pragma unroll
    for (int i = 0; i < kLines; ++i) asm volatile("" : : "v"(touched[i]));
    if (c >= p.rows.rows || (unsigned)a >= (unsigned)p.rows.count) a = -1;
    unsigned left = (unsigned)__ballot(a >= 0) & 0xFFFFu;
    int mine[kMost], count = 0;
    bool live = c < p.rows.rows && a < 0 && wave == 0;
    for (int turn = 0; left; ++turn) {
        const int cur = __builtin_amdgcn_readlane(a, __builtin_ctz(left));
        left &= ~((unsigned)__ballot(a == cur) & 0xFFFFu);
        if (turn % W != wave) continue;
#pragma unroll
        for (int i = 0; i < kMost; ++i)
            if (i == count) mine[i] = cur;
        ++count;
        live |= a == cur;
    }
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) part[wave][4 * q + r][16 * i + c] = total[i][r];
    auto rows_of_b = [&](int adapter, bf16x8 (&b)[S][SR]) {
#pragma unroll
        for (int tile = 0; tile < S; ++tile)
#pragma unroll
            for (int s = 0; s < SR; ++s)
                b[tile][s] = load_bf16x8(mat + (size_t)adapter * p.N * p.rank + (size_t)(16 * tile + c) * p.rank + min(32 * s + 8 * q, p.rank - 8));
    };
    bf16x8 b[2][S][SR];
    if (count > 0) rows_of_b(mine[0], b[0]);
    if constexpr (OWN) {
        __syncthreads();
        for (int e = tid; e < kOwnRows * 32 * SR; e += W * 64) {
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) v += parts_of_t[w][e / (32 * SR)][e % (32 * SR)];
            ts[e / (32 * SR)][e % (32 * SR)] = v;
        }
        __syncthreads();
    } else {
        sum_projected<16>(p.t, p.rows, 0, p.rank, p.slices, tid, W * 64, ts);
    }
    ExpandRow<SR> tv;
    tv.set(ts[c], scale, live && a >= 0, q, p.rank);
    f32x4 acc[S];
#pragma unroll
    for (int i = 0; i < S; ++i) {
        acc[i] = *reinterpret_cast<const f32x4 *>(&part[0][c][16 * i + 4 * q]);
#pragma unroll
        for (int w = 1; w < W; ++w) acc[i] += *reinterpret_cast<const f32x4 *>(&part[w][c][16 * i + 4 * q]);
    }
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
        if (i >= count) break;
        if (i + 1 < kMost && i + 1 < count) rows_of_b(mine[i + 1], b[(i + 1) & 1]);
        expand_product<SR, S>(b[i & 1], tv, a == mine[i], acc);
    }
    if (!live) return;
#pragma unroll
    for (int i = 0; i < S; ++i) {
        u32x2 v;
        v.x = f32_to_bf16_bits(acc[i][0]) | (uint32_t)f32_to_bf16_bits(acc[i][1]) << 16;
        v.y = f32_to_bf16_bits(acc[i][2]) | (uint32_t)f32_to_bf16_bits(acc[i][3]) << 16;
        *reinterpret_cast<u32x2 *>(p.y + (size_t)c * p.N + n0 + 16 * i + 4 * q) = v;
    }
}

template <int W, int GW, int S>
void launch_few(const FewArgs &a, hipStream_t stream) {
    const int blocks = a.N / (16 * S);
    if (!a.t) {
        if (a.rank <= 32) bank_few_kernel<W, GW, S, 1, true><<<blocks, W * 64, 0, stream>>>(a);
        else bank_few_kernel<W, GW, S, 2, true><<<blocks, W * 64, 0, stream>>>(a);
    } else {
        if (a.rank <= 32) bank_few_kernel<W, GW, S, 1, false><<<blocks, W * 64, 0, stream>>>(a);
        else bank_few_kernel<W, GW, S, 2, false><<<blocks, W * 64, 0, stream>>>(a);
    }
}

}  // namespace

void bank_few(const void *x, const void *b, const void *s, void *y, const kiln_w4a16_adapter_bank &bank, const BankRows &rows, const float *t, int slices,
              int K, int N, bool per_column, hipStream_t stream) {
    const FewArgs a{(const uint16_t *)x, (const u32x4 *)b, (const uint16_t *)s, (uint16_t *)y, (const uint16_t *)bank.lora_b, (const uint16_t *)bank.lora_a, t, bank.scales,
                    rows, K, N, bank.rank, slices, per_column};
    // two tiles to a block where that leaves a block to every compute unit
    with_few_rows_split(K / kGroupK, [&](auto waves, auto groups) {
        constexpr int W = decltype(waves)::value, GW = decltype(groups)::value;
        const int tiles = N / kTileN;
        if (tiles >= 512) launch_few<W, GW, 2>(a, stream);
        else launch_few<W, GW, 1>(a, stream);
    });
}

}  // namespace kiln
