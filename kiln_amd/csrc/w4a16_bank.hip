// A packed projection whose rows have low-rank adapters of their own out of a bank:
// y[i] = x[i] W + s_a (x[i] A_a^T) B_a^T, a = adapter_of[i].
//
// Three steps: T = x A^T (w4a16_bank project, f32), the plain GEMM, and y += s T B^T in place.  Rows are handled in tiles of 16
// positions; a tile multiplies with each adapter that is present among its rows, once, and rows of other adapters are left out of
// the product, so any order of the rows is right and one in which an adapter's rows are together reads its matrices least often:
// from 65 rows on a launch in front puts them so.  The reference serves one adapter set per process
// (crates/kiln-model/src/lora_loader.rs:213-232); this is its formula with the adapter a row's own.
#include "bank.h"
#include "device_common.h"

namespace kiln {
namespace {

// order[] and first[]: a wavefront per adapter (and one for the rows without) counts the rows of lower adapters and places its own,
// 64 rows per ballot; no block waits for another and rows keep their order inside an adapter.
constexpr int kOrderUnroll = 8;
__global__ __launch_bounds__(256) void bank_order_kernel(const int *__restrict__ of, int *__restrict__ order, int *__restrict__ first, int rows,
                                                         int count) {
    const int lane = threadIdx.x & 63;
    const int a = blockIdx.x * 4 + (int)(threadIdx.x >> 6);
    if (a > count) return;
    int less = 0;
    for (int r0 = 0; r0 < rows; r0 += 64 * kOrderUnroll) {
        int v[kOrderUnroll];
#pragma unroll
        for (int u = 0; u < kOrderUnroll; ++u) {
            const int r = r0 + 64 * u + lane;
            v[u] = r < rows ? of[r] : -1;
        }
#pragma unroll
        for (int u = 0; u < kOrderUnroll; ++u) {
            const bool in = r0 + 64 * u + lane < rows;
            const int key = (unsigned)v[u] < (unsigned)count ? v[u] : count;
            less += __popcll(__ballot(in && key < a));
        }
    }
    if (lane == 0) {
        first[a] = less;
        if (a == count) first[count + 1] = rows;
    }
    for (int r0 = 0; r0 < rows; r0 += 64 * kOrderUnroll) {
        int v[kOrderUnroll];
#pragma unroll
        for (int u = 0; u < kOrderUnroll; ++u) {
            const int r = r0 + 64 * u + lane;
            v[u] = r < rows ? of[r] : -1;
        }
#pragma unroll
        for (int u = 0; u < kOrderUnroll; ++u) {
            const int r = r0 + 64 * u + lane;
            const int key = (unsigned)v[u] < (unsigned)count ? v[u] : count;
            const bool mine = r < rows && key == a;
            const unsigned long long all = __ballot(mine);
            if (mine) order[less + __popcll(all & ((1ull << lane) - 1))] = r;
            less += __popcll(all);
        }
    }
}

__device__ __forceinline__ bf16x8 load_bf16x8(const uint16_t *p) {
    return __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4 *>(p));
}

// The row and the adapter (-1: none) of position p0 + (lane & 15).
__device__ __forceinline__ void row_of_lane(const BankRows &r, int p, int &row, int &a) {
    row = p < r.rows ? (r.order ? r.order[p] : p) : -1;
    a = row >= 0 ? r.of[row] : -1;
    if ((unsigned)a >= (unsigned)r.count) a = -1;
}

// U steps of a projection's contraction, all their loads in front of their products.
constexpr int kProjectAhead = 4;
template <int JT, int U>
__device__ __forceinline__ void project_steps(const uint16_t *__restrict__ x, const uint16_t *__restrict__ m, int K, int rank, int c,
                                              f32x4 (&acc)[JT]) {
    bf16x8 xv[U], b[U][JT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        xv[u] = load_bf16x8(x + 128 * u);
#pragma unroll
        for (int j = 0; j < JT; ++j) b[u][j] = 16 * j + c < rank ? load_bf16x8(m + (size_t)16 * j * K + 128 * u) : bf16x8_zero();
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < JT; ++j) acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xv[u], b[u][j], acc[j], 0, 0, 0);
}

// A block: 16 positions, one slice of K, and of the adapters present among them those whose turn (in the order they are met) is
// blockIdx.z modulo gridDim.z.  Its four wavefronts take every fourth 32 of K and meet in LDS.
template <int JT>
__global__ __launch_bounds__(256) void bank_project_kernel(const uint16_t *__restrict__ src, const uint16_t *__restrict__ mat, BankRows rows,
                                                           float *__restrict__ t, int K, int steps, int rank) {
    __shared__ float part[4][16][JT * 16 + 4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 15, q = lane >> 4;
    const int p0 = blockIdx.x * kBankRowTile;
    int row, a;
    row_of_lane(rows, p0 + c, row, a);
    const int k0 = blockIdx.y * steps * 128 + 32 * wave + 8 * q;
    const int n_steps = min(steps, K / 128 - (int)blockIdx.y * steps);
    const uint16_t *x = src + (size_t)max(row, 0) * K + k0;
    unsigned left = (unsigned)__ballot(a >= 0) & 0xFFFFu;
    for (unsigned turn = 0; left; ++turn) {
        const int cur = __builtin_amdgcn_readlane(a, __builtin_ctz(left));
        const unsigned mine = (unsigned)__ballot(a == cur) & 0xFFFFu;
        left &= ~mine;
        if (turn % gridDim.z != blockIdx.z) continue;
        const uint16_t *m = mat + ((size_t)cur * rank + c) * K + k0;
        f32x4 acc[JT];
#pragma unroll
        for (int j = 0; j < JT; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
        int s = 0;
        for (; s + kProjectAhead <= n_steps; s += kProjectAhead) project_steps<JT, kProjectAhead>(x + 128 * s, m + 128 * s, K, rank, c, acc);
        for (; s < n_steps; ++s) project_steps<JT, 1>(x + 128 * s, m + 128 * s, K, rank, c, acc);
#pragma unroll
        for (int j = 0; j < JT; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) part[wave][4 * q + i][16 * j + c] = acc[j][i];
        __syncthreads();
        float *out = t + ((size_t)blockIdx.y * rows.rows + p0) * rank;
        for (int e = tid; e < 16 * rank; e += 256) {
            const int r = e / rank, j = e - r * rank;
            if (mine >> r & 1) out[e] = (part[0][r][j] + part[1][r][j]) + (part[2][r][j] + part[3][r][j]);
        }
        __syncthreads();
    }
}

// y[row] += s_a T[row] B_a^T on 16 positions x 256 columns, 64 to a wavefront, as B_a (its rows the columns of y) times T^T: a lane
// then holds four consecutive columns of one row.  T goes in as two bf16 parts whose sum is within 2^-17 of it, side by side on the
// contraction, which has room: 32 for a rank of 16.
template <int S>
__global__ __launch_bounds__(256) void bank_expand_kernel(uint16_t *__restrict__ y, const uint16_t *__restrict__ mat, const float *__restrict__ t,
                                                          const float *__restrict__ scales, BankRows rows, int N, int rank, int slices) {
    __shared__ float ts[16][kBankMaxRank + 4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 15, q = lane >> 4;
    const int p0 = blockIdx.y * kBankRowTile;
    int row, a;
    row_of_lane(rows, p0 + c, row, a);
    unsigned left = (unsigned)__ballot(a >= 0) & 0xFFFFu;
    if (!left) return;
    for (int e = tid; e < 16 * rank; e += 256) {
        const int r = e / rank, j = e - r * rank;
        float v = 0.f;
        if (p0 + r < rows.rows)
            for (int s = 0; s < slices; ++s) v += t[((size_t)s * rows.rows + p0 + r) * rank + j];
        ts[r][j] = v;
    }
    __syncthreads();
    const int n0 = blockIdx.x * 256 + wave * 64, octets = rank >> 3;
    const bool live = a >= 0;
    const float scale = live ? scales[a] : 0.f;
    uint16_t *dst = y + (size_t)max(row, 0) * N + n0 + 4 * q;
    f32x4 acc[4];
#pragma unroll
    for (int tile = 0; tile < 4; ++tile) {
        const u32x2 v = live ? *reinterpret_cast<const u32x2 *>(dst + 16 * tile) : u32x2{0u, 0u};
        acc[tile] = f32x4{__builtin_bit_cast(float, v.x << 16), __builtin_bit_cast(float, v.x & 0xFFFF0000u),
                          __builtin_bit_cast(float, v.y << 16), __builtin_bit_cast(float, v.y & 0xFFFF0000u)};
    }
    while (left) {
        const int cur = __builtin_amdgcn_readlane(a, __builtin_ctz(left));
        left &= ~((unsigned)__ballot(a == cur) & 0xFFFFu);
        const uint16_t *m = mat + ((size_t)cur * N + n0 + c) * rank;
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const int o = 4 * s + q;
            const bool lower = o >= octets, used = o < 2 * octets;
            const int at = 8 * (used ? (lower ? o - octets : o) : 0);
            bf16x8 tv = bf16x8_zero();
            if (used && a == cur)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float v = ts[c][at + i] * scale;
                    const __bf16 hi = (__bf16)v;
                    tv[i] = lower ? (__bf16)(v - (float)hi) : hi;
                }
#pragma unroll
            for (int tile = 0; tile < 4; ++tile) {
                const bf16x8 b = used ? load_bf16x8(m + (size_t)16 * tile * rank + at) : bf16x8_zero();
                acc[tile] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b, tv, acc[tile], 0, 0, 0);
            }
        }
    }
    if (!live) return;
#pragma unroll
    for (int tile = 0; tile < 4; ++tile) {
        u32x2 v;
        v.x = f32_to_bf16_bits(acc[tile][0]) | (uint32_t)f32_to_bf16_bits(acc[tile][1]) << 16;
        v.y = f32_to_bf16_bits(acc[tile][2]) | (uint32_t)f32_to_bf16_bits(acc[tile][3]) << 16;
        *reinterpret_cast<u32x2 *>(dst + 16 * tile) = v;
    }
}

int tiles_of(int rows) { return (rows + kBankRowTile - 1) / kBankRowTile; }

}  // namespace

bool bank_ok(const kiln_w4a16_adapter_bank &bank) {
    return bank.count >= 1 && bank.count <= 4096 && bank.rank >= 8 && bank.rank <= kBankMaxRank && bank.rank % 8 == 0;
}

size_t bank_order_bytes(int rows, int count) { return bank_up256((size_t)rows * 4) + bank_up256(((size_t)count + 2) * 4); }

BankRows bank_order(const int *of, int rows, int count, bool always, void *at, hipStream_t stream) {
    BankRows r{of, nullptr, nullptr, rows, count};
    if (rows < kBankOrderedFrom && !always) return r;
    int *order = reinterpret_cast<int *>(at);
    int *first = reinterpret_cast<int *>(reinterpret_cast<char *>(at) + bank_up256((size_t)rows * 4));
    bank_order_kernel<<<(count + 4) / 4, 256, 0, stream>>>(of, order, first, rows, count);
    r.order = order;
    r.first = first;
    return r;
}

// slices * rows <= this, and it does not fall with `rows`
size_t bank_projected_rows(int rows, int K) {
    const size_t tiles = tiles_of(rows), most = K / 128 < kBankMaxSlices ? K / 128 : kBankMaxSlices;
    return kBankRowTile * (tiles * most < tiles + 511 ? tiles * most : tiles + 511);
}

int bank_slices(int rows, int K) {
    const int groups = K / 128, want = (511 + tiles_of(rows)) / tiles_of(rows);
    int slices = want < kBankMaxSlices ? want : kBankMaxSlices;
    if (slices > groups) slices = groups;
    const int steps = (groups + slices - 1) / slices;
    return (groups + steps - 1) / steps;
}

void bank_project(const void *src, const void *mat, const BankRows &r, float *t, int K, int rank, int slices, hipStream_t stream) {
    const int groups = K / 128, steps = (groups + slices - 1) / slices;
    const int turns = r.count < (r.order ? 4 : 16) ? r.count : (r.order ? 4 : 16);
    const dim3 grid(tiles_of(r.rows), slices, turns);
    const uint16_t *s = (const uint16_t *)src, *m = (const uint16_t *)mat;
    switch ((rank + 15) / 16) {
        case 1: bank_project_kernel<1><<<grid, 256, 0, stream>>>(s, m, r, t, K, steps, rank); break;
        case 2: bank_project_kernel<2><<<grid, 256, 0, stream>>>(s, m, r, t, K, steps, rank); break;
        case 3: bank_project_kernel<3><<<grid, 256, 0, stream>>>(s, m, r, t, K, steps, rank); break;
        default: bank_project_kernel<4><<<grid, 256, 0, stream>>>(s, m, r, t, K, steps, rank); break;
    }
}

}  // namespace kiln

using namespace kiln;

extern "C" {

size_t kiln_w4a16_gemm_bank_scratch_bytes(int prob_m, int prob_n, int prob_k, int count, int rank) {
    if (prob_m < 1 || prob_n < 1 || prob_k < 128 || count < 1 || rank < 1) return 256;
    return bank_order_bytes(prob_m, count) + bank_up256(bank_projected_rows(prob_m, prob_k) * rank * 4);
}

kiln_marlin_status_t kiln_w4a16_gemm_bank(const void *A, const void *B, void *C, const void *s, int prob_m, int prob_n, int prob_k,
                                          void *workspace, int groupsize, int dev, void *stream, const kiln_w4a16_adapter_bank *bank,
                                          const int *adapter_of, void *scratch) {
    if (prob_m < 0 || prob_n < 0 || prob_k < 0) return KILN_W4A16_ERR_PROB_SHAPE;
    if (prob_m == 0 || prob_n == 0 || prob_k == 0)
        return kiln_marlin_w4a16_gemm(A, B, C, const_cast<void *>(s), prob_m, prob_n, prob_k, workspace, groupsize, dev, stream, -1, -1, -1, 16);
    if (!bank || !adapter_of || !scratch) return KILN_W4A16_ERR_ARGUMENT;
    if (!bank_ok(*bank)) return KILN_W4A16_ERR_KERN_SHAPE;
    if (!bank->lora_a || !bank->lora_b || !bank->scales) return KILN_W4A16_ERR_ARGUMENT;
    for (const void *p : {bank->lora_a, bank->lora_b, static_cast<const void *>(scratch)})
        if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return KILN_W4A16_ERR_ARGUMENT;
    // the plain GEMM's checks and its launches first: nothing is launched for a call that it refuses
    const kiln_marlin_status_t st =
        kiln_marlin_w4a16_gemm(A, B, C, const_cast<void *>(s), prob_m, prob_n, prob_k, workspace, groupsize, dev, stream, -1, -1, -1, 16);
    if (st != KILN_W4A16_OK) return st;
    hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
    char *at = reinterpret_cast<char *>(scratch);
    const BankRows rows = bank_order(adapter_of, prob_m, bank->count, false, at, hs);
    float *t = reinterpret_cast<float *>(at + bank_order_bytes(prob_m, bank->count));
    const int slices = bank_slices(prob_m, prob_k), rank = bank->rank;
    bank_project(A, bank->lora_a, rows, t, prob_k, rank, slices, hs);
    const dim3 grid(prob_n / 256, tiles_of(prob_m));
    uint16_t *y = (uint16_t *)C;
    const uint16_t *m = (const uint16_t *)bank->lora_b;
    switch ((2 * (rank / 8) + 3) / 4) {
        case 1: bank_expand_kernel<1><<<grid, 256, 0, hs>>>(y, m, t, bank->scales, rows, prob_n, rank, slices); break;
        case 2: bank_expand_kernel<2><<<grid, 256, 0, hs>>>(y, m, t, bank->scales, rows, prob_n, rank, slices); break;
        case 3: bank_expand_kernel<3><<<grid, 256, 0, hs>>>(y, m, t, bank->scales, rows, prob_n, rank, slices); break;
        default: bank_expand_kernel<4><<<grid, 256, 0, hs>>>(y, m, t, bank->scales, rows, prob_n, rank, slices); break;
    }
    return hipGetLastError() == hipSuccess ? KILN_W4A16_OK : KILN_W4A16_ERR_LAUNCH;
}

}  // extern "C"
