// A packed projection of up to 16 rows with low-rank adapters of their own (w4a16_bank.hip): base product, projection and low-rank term of a
// row or two in one launch, or base product and projection in one and the term behind it.
#include "bank.h"
#include "bank_expand.h"
#include "bank_project.h"
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
    const float *scales;
    BankRows rows;
    int K, N, rank, per_column;
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

// One launch for a row or two.  S column tiles to a block of W wavefronts, which meet in LDS after the base product; every block projects the
// rows onto their adapters by itself, out of the part of the rows that its wavefronts hold: the adapters' A read by every block is less
// than a launch that it saves.  The first wavefront finishes and stores the rows of the first one's adapter (or of none), the second the other's, on
// the f32 sums.  What that needs of memory is touched while the first weights are on their way -- a lane a line or a few of its row's
// adapter -- and comes out of a cache.
template <int W, int GW, int S, int SR>
__global__ __launch_bounds__(W * 64) void bank_few_kernel(FewArgs p) {
    constexpr int kPitch = S * 16 + 4;
    __shared__ __align__(16) float part[W][16][kPitch];
    __shared__ __align__(16) float ts[kOwnRows][32 * SR];
    __shared__ float parts_of_t[W][kOwnRows][32 * SR];
    for (int e = threadIdx.x & 63; e < kOwnRows * 32 * SR; e += 64) (&parts_of_t[threadIdx.x >> 6][0][0])[e] = 0.f;  // (this wavefront's own, until the block meets)
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
                               [&](const bf16x8(&x)[GW][4], int first) { project_own<W, GW, SR>(p, x, first, G, a, lane, parts_of_t[wave]); });
#pragma unroll
    for (int i = 0; i < kLines; ++i) asm volatile("" : : "v"(touched[i]));
    if (c >= p.rows.rows || (unsigned)a >= (unsigned)p.rows.count) a = -1;
    const int mine = __builtin_amdgcn_readlane(a, wave & 1);
    const bool other = wave == 1 && mine == __builtin_amdgcn_readlane(a, 0);  // the first wavefront's
    const bool live = wave < kOwnRows && c < p.rows.rows && !other && (a == mine || (wave == 0 && a < 0));
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) part[wave][4 * q + r][16 * i + c] = total[i][r];
    bf16x8 b[S][SR];
    if (wave < kOwnRows && mine >= 0)
#pragma unroll
        for (int tile = 0; tile < S; ++tile)
#pragma unroll
            for (int s = 0; s < SR; ++s)
                b[tile][s] = load_bf16x8(mat + (size_t)mine * p.N * p.rank + (size_t)(16 * tile + c) * p.rank + min(32 * s + 8 * q, p.rank - 8));
    __syncthreads();
    for (int e = tid; e < kOwnRows * 32 * SR; e += W * 64) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) v += parts_of_t[w][e / (32 * SR)][e % (32 * SR)];
        ts[e / (32 * SR)][e % (32 * SR)] = v;
    }
    __syncthreads();
    if (wave >= kOwnRows) return;
    ExpandRow<SR> tv;
    tv.set(ts[min(c, kOwnRows - 1)], scale, live && a >= 0, q, p.rank);
    f32x4 acc[S];
#pragma unroll
    for (int i = 0; i < S; ++i) {
        acc[i] = *reinterpret_cast<const f32x4 *>(&part[0][c][16 * i + 4 * q]);
#pragma unroll
        for (int w = 1; w < W; ++w) acc[i] += *reinterpret_cast<const f32x4 *>(&part[w][c][16 * i + 4 * q]);
    }
    if (mine >= 0) expand_product<SR, S>(b, tv, a == mine, acc);
    if (!live) return;
#pragma unroll
    for (int i = 0; i < S; ++i) {
        u32x2 v;
        v.x = f32_to_bf16_bits(acc[i][0]) | (uint32_t)f32_to_bf16_bits(acc[i][1]) << 16;
        v.y = f32_to_bf16_bits(acc[i][2]) | (uint32_t)f32_to_bf16_bits(acc[i][3]) << 16;
        *reinterpret_cast<u32x2 *>(p.y + (size_t)c * p.N + n0 + 16 * i + 4 * q) = v;
    }
}

// The base product of up to 16 rows, and beside it in the same launch the rows' projections, which the launch behind it (w4a16_bank.hip)
// multiplies: the first `projecting` blocks, a slice of the contraction and a turn of the adapters each.  Tiles to a block: as many as leave
// a block to every compute unit, the rows are read once for all of them (2560 -> 18432, 16 rows: 5 15.6 us a call, 4 17.0, 2 18.0, 1 21.6).
template <int W, int GW, int S>
__global__ __launch_bounds__(W * 64) void bank_base_kernel(FewArgs p, BankProjection of_x, int projecting, int turns) {
    constexpr int kPitch = S * 16 + 4;
    union Lds {
        float projected[W][16][kBankMaxRank + 4];
        float part[W][16][kPitch];
    };
    __shared__ __align__(16) Lds lds;
    if ((int)blockIdx.x < projecting) {
        project_rows<W>(of_x, p.rows, p.rank, blockIdx.x / turns, 0, blockIdx.x % turns, turns, lds.projected);
        return;
    }
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, q = lane >> 4;
    const DequantConsts dc = dequant_consts();
    // (the last block's tiles may be the one's before it too: the same values twice)
    const int nt0 = min((int)(blockIdx.x - projecting) * S, p.N / kTileN - S), G = p.K / kGroupK, Gs = p.per_column ? 1 : G;
    f32x4 total[S];
    few_rows_product<GW, S>(p.x + (size_t)min(c, p.rows.rows - 1) * p.K + 8 * q, p.b + (size_t)nt0 * G * 64 + lane, p.s + (size_t)nt0 * Gs * kTileN + c, G,
                            p.per_column, wave, W, dc, total);
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) lds.part[wave][4 * q + r][16 * i + c] = total[i][r];
    __syncthreads();
    for (int e = tid; e < p.rows.rows * S * 8; e += W * 64) {
        const int r = e / (S * 8), col = e % (S * 8) * 2;
        float lo = 0.f, hi = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            lo += lds.part[w][r][col];
            hi += lds.part[w][r][col + 1];
        }
        *reinterpret_cast<uint32_t *>(p.y + (size_t)r * p.N + nt0 * kTileN + col) = f32_to_bf16_bits(lo) | (uint32_t)f32_to_bf16_bits(hi) << 16;
    }
}

template <int W, int GW, int S>
void launch_few(const FewArgs &a, hipStream_t stream) {
    const int blocks = a.N / (16 * S);
    if (a.rank <= 32) bank_few_kernel<W, GW, S, 1><<<blocks, W * 64, 0, stream>>>(a);
    else bank_few_kernel<W, GW, S, 2><<<blocks, W * 64, 0, stream>>>(a);
}
// Blocks of the projection are an adapter each; where those would be one round too many, up to four adapters each.
template <int W, int GW, int S>
void launch_base(const FewArgs &a, const BankProjection &of_x, int met, int cus, hipStream_t stream) {
    const int blocks = (a.N / 16 + S - 1) / S, room = cus * (W == 4 ? 2 : 1) - blocks;
    int turns = met;
    if (room > 0 && of_x.slices * turns > room) turns = room / of_x.slices > (met + 3) / 4 ? room / of_x.slices : (met + 3) / 4;
    bank_base_kernel<W, GW, S><<<of_x.slices * turns + blocks, W * 64, 0, stream>>>(a, of_x, of_x.slices * turns, turns);
}
template <int W, int GW>
void launch_base(const FewArgs &a, const BankProjection &of_x, int cus, hipStream_t stream) {
    const int met = a.rows.count < a.rows.rows ? a.rows.count : a.rows.rows, tiles = a.N / kTileN;
    // a unit holds one block of eight wavefronts, or two of four
    const int left = W == 4 ? cus : cus - of_x.slices * ((met + 1) / 2), units = left > 0 ? left : 1;
    int each = (tiles + units - 1) / units;
    if (W == 8 && each >= 7 && (tiles + 6) / 7 + of_x.slices * ((met + 3) / 4) > cus) each = 4;  // several rounds: small ones
    if (each <= 1) launch_base<W, GW, 1>(a, of_x, met, cus, stream);
    else if (each == 2) launch_base<W, GW, 2>(a, of_x, met, cus, stream);
    else if (each == 3) launch_base<W, GW, 3>(a, of_x, met, cus, stream);
    else if (each == 4) launch_base<W, GW, 4>(a, of_x, met, cus, stream);
    else if (each == 5) launch_base<W, GW, 5>(a, of_x, met, cus, stream);
    else if (each == 6) launch_base<W, GW, 6>(a, of_x, met, cus, stream);
    else launch_base<W, GW, 7>(a, of_x, met, cus, stream);
}

}  // namespace

// One row of rank 16, us, against two launches: 2560 -> 2560 6.0 to 7.1, 2560 -> 8192 7.6 to 8.5, 1024 -> 4096 4.6 to 7.0 (two rows 5.1); but 4096 -> 2560
// 7.6 to 7.1, two rows of 2560 -> 8192 10.1 to 8.6.
bool bank_projects_itself(int m, int n, int k, int rank) { return m <= kOwnRows && n <= 8192 && (int64_t)m * rank * k <= 48 * 1024; }

int bank_base_slices(int K) {  // one turn of a block's wavefronts each
    const int groups = K / kGroupK, each = groups <= 20 ? 4 : 8, slices = (groups + each - 1) / each;
    return bank_level_slices(groups, slices < kBankMaxSlices ? slices : kBankMaxSlices);
}

void bank_base(const void *x, const void *b, const void *s, void *y, const BankProjection &of_x, const BankRows &rows, int rank, int K, int N, bool per_column, int cus,
               hipStream_t stream) {
    const FewArgs a{(const uint16_t *)x, (const u32x4 *)b, (const uint16_t *)s, (uint16_t *)y, nullptr, nullptr, nullptr, rows, K, N, rank, per_column};
    with_few_rows_split(K / kGroupK, [&](auto waves, auto groups) {
        constexpr int W = decltype(waves)::value, GW = decltype(groups)::value;
        launch_base<W, GW>(a, of_x, cus, stream);
    });
}

void bank_few(const void *x, const void *b, const void *s, void *y, const kiln_w4a16_adapter_bank &bank, const BankRows &rows, int K, int N, bool per_column,
              hipStream_t stream) {
    const FewArgs a{(const uint16_t *)x, (const u32x4 *)b, (const uint16_t *)s, (uint16_t *)y, (const uint16_t *)bank.lora_b, (const uint16_t *)bank.lora_a,
                    bank.scales, rows, K, N, bank.rank, per_column};
    with_few_rows_split(K / kGroupK, [&](auto waves, auto groups) {
        constexpr int W = decltype(waves)::value, GW = decltype(groups)::value;
        if (N / kTileN >= 512) launch_few<W, GW, 2>(a, stream);
        else launch_few<W, GW, 1>(a, stream);
    });
}

}  // namespace kiln
