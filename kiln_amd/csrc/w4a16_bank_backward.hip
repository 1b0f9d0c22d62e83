// The gradients of a packed projection, with or without a bank of adapters (w4a16_bank.hip), the packed weight itself frozen:
//   dx[i]  = dy[i] W^T + s_a (dy[i] B_a) A_a            a = adapter_of[i]
//   dA_a   = s_a sum_{i of a} (dy[i] B_a)^T x[i]
//   dB_a   = s_a sum_{i of a} dy[i]^T (x[i] A_a^T)
// The reference trains adapters over a frozen base (crates/kiln-model/src/lora_loader.rs:213-232 is the forward it differentiates).
//
// Up to 64 rows two launches: dx straight from the codes with T = x A^T and U = dy B beside it, then dA, dB and dx's slices and U A.  45 rows of
// 4096 -> 2560: 19.2 us a call, 26.9 in four launches.
// Beyond: W as bf16 with its columns contiguous (what a product over the columns reads), the adapters' matrices transposed, T = x A^T and
// U = dy B in f32, then dx as one matrix product into which U A goes as further steps of the contraction, and dA, dB as sums over the
// rows of an adapter.  Rows are taken in the order of their adapters throughout.
#include <type_traits>

#include "async_loads.h"
#include "bank.h"
#include "bank_expand.h"
#include "bank_order.h"
#include "bank_project.h"
#include "device_common.h"
#include "launch.h"

namespace kiln {
namespace {

// Column e of eight rows of eight bf16 values each, as an operand of a product over the rows.
__device__ __forceinline__ bf16x8 column_of_rows(const u32x4 (&v)[8], int e) {
    u32x4 pairs;
#pragma unroll
    for (int i = 0; i < 4; ++i) pairs[i] = __builtin_amdgcn_perm(v[2 * i + 1][e >> 1], v[2 * i][e >> 1], e & 1 ? 0x07060302u : 0x05040100u);
    return __builtin_bit_cast(bf16x8, pairs);
}

// ---- what the products read ----------------------------------------------------------------------------------------
// One launch for what depends on the call's operands alone: the rows' order, the adapters' matrices turned, and W unpacked row by row.
struct PrepareArgs {
    const u32x4 *B;        // the packed weight
    const uint16_t *S;
    uint16_t *wt;          // bf16 [K, N]
    const uint16_t *a, *b;  // the bank's matrices, [count, rank, K] and [count, N, rank]
    uint16_t *at, *bt;      // ... turned: [count, K, rank] and [count, rank, N]
    uint8_t *odd;           // [count, K / 64]
    BankRows rows;
    int K, N, Gs, rank;
    int order_blocks, turn_blocks;
    const uint16_t *dy, *x;  // few rows: [m, N] and [m, K],
    float *partial;          // [slices, m, K],
    float *t, *u;            // ... and T and U, [slices, m, rank]
    int m, slices, t_slices, u_slices, turns;
};
constexpr int kPrepareThreads = 512, kTurnPitch = 128 + 8, kFewPitch = 128 + 4, kFewDyPitch = 256 + 8;
constexpr int kFewTiles = 16, kFewColumns = kFewTiles * kTileN;
union PrepareLds {
    uint16_t weight[128 * kTurnPitch];
    uint16_t bank[64][kBankMaxRank + 2];
    OrderLds<kPrepareThreads / 64> order;
};
union FewLds {
    struct {
        uint16_t dy[64 * kFewDyPitch];
        u32x4 codes[kFewTiles * 64];
        uint16_t scales[kFewColumns];
    } in;
    float sums[64 * kFewPitch];
    float projected[kPrepareThreads / 64][16][kBankMaxRank + 4];
};

// wt[k][n] = bf16((code - 8) * scale): a block takes one scale group (128 rows) x 128 columns, a chunk to each of its eight wavefronts.  The
// rounding of a weight to 8 bits is what every 16-bit product of the unpacked weight has (the reference's own bar is against
// bf16(dequant): crates/kiln-marlin-gemm/tests/parity.rs:150-157); the codes themselves would be exact, but the scales run along the
// contraction here and cannot be pulled out of it.
// A word has eight rows of one column and a row of wt wants many columns: the codes are turned, eight lanes' words of eight nibbles each,
// in three exchanges between lanes one, two and four apart, and a lane then has eight columns of one row, one 16-byte piece of LDS (as
// 32 pieces of 2 bytes these writes bounded the kernel: 2560 x 18432 22 us).
template <int S>
__device__ __forceinline__ uint32_t exchange_nibbles(uint32_t w, int lane) {
    constexpr uint32_t kLow = S == 1 ? 0x0F0F0F0Fu : S == 2 ? 0x00FF00FFu : 0x0000FFFFu;
    const bool lower = (lane & S) == 0;
    int other = (int)w;
    if constexpr (S == 1) other = __builtin_amdgcn_update_dpp(0, other, 0xB1, 0xF, 0xF, true);
    if constexpr (S == 2) other = __builtin_amdgcn_update_dpp(0, other, 0x4E, 0xF, 0xF, true);
    if constexpr (S == 4) {  // 7 - i, then 3 - i within four: four apart
        other = __builtin_amdgcn_update_dpp(0, other, 0x141, 0xF, 0xF, true);
        other = __builtin_amdgcn_update_dpp(0, other, 0x1B, 0xF, 0xF, true);
    }
    const uint32_t keep = lower ? kLow : ~kLow, turned = __builtin_amdgcn_alignbit(other, other, lower ? 32 - 4 * S : 4 * S);
    return (w & keep) | (turned & ~keep);
}
__device__ __forceinline__ void unpack_weight(const PrepareArgs &p, int block, PrepareLds &lds) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, i = lane & 7, h = lane >> 3 & 1, kq = lane >> 4;
    const int G = p.K / kGroupK, tiles = p.N / 128, g = block / tiles, n0 = block % tiles * 128, nt = n0 / kTileN + wave;
    const u32x4 w = p.B[((size_t)nt * G + g) * 64 + lane];
    const u32x4 scales = *reinterpret_cast<const u32x4 *>(p.S + scale_index(p.Gs == 1 ? 0 : g, nt * kTileN + 8 * h, p.Gs));
    const int j = i < 4 ? 2 * i : 2 * i - 7;  // the row in nibble i
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const uint32_t v = exchange_nibbles<4>(exchange_nibbles<2>(exchange_nibbles<1>(w[t], lane), lane), lane);
        bf16x8 o;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            const uint32_t pair = scales[c >> 1];
            o[c] = (__bf16)((float)((int)(v >> (4 * c) & 0xF) - 8) * f16_bits_to_f32((uint16_t)(c & 1 ? pair >> 16 : pair)));
        }
        *reinterpret_cast<bf16x8 *>(lds.weight + (32 * t + 8 * kq + j) * kTurnPitch + 16 * wave + 8 * h) = o;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int row = 32 * r + (tid >> 4), at = 8 * (tid & 15);
        *reinterpret_cast<u32x4 *>(p.wt + (size_t)(g * kGroupK + row) * p.N + n0 + at) = *reinterpret_cast<const u32x4 *>(lds.weight + row * kTurnPitch + at);
    }
}

// Up to 64 rows: partial[slice][row][k] = sum over the slice's columns of dy[row][n] W[k][n], the codes unpacked where they are multiplied.
// With the codes turned, and the lanes' words of a chunk dealt out for it (lane i + 8 kq + 32 h has column i + 8 h's), a word is the operand of
// a product of 32 rows of k x 16 columns as it stands: nothing of W goes through memory again or LDS, and of dy a row's 16 values serve 128 of k.
// A block takes one scale group and slice, a wavefront 32 rows of k and every other eight of sixteen column tiles; codes, scales and dy of
// sixteen tiles go through LDS, the next ones' on their way meanwhile, and the halves meet there.  Bound by its start, one round of loads, and
// its instructions and their fetch (straight-line code is read from memory once in every launch): 45 rows of 4096 <- 2560 20 us with eight
// tiles unrolled, 15 with four and codes from memory, 12 to 14 with a loop of one tile and everything through LDS.
constexpr int kFewProjected = 8;  // slices of T's and U's contraction at most
// (rows of a wavefront's ballot and of the tile of dy in LDS; beyond, W is unpacked for a product.  us a call at 64 rows straight from the codes / by that
// product, four adapters of rank 16: 2560 <- 2560 16.8 / 42.1, 4096 <- 2560 21.5 / 44.5, 9216 <- 2560 28.5 / 56.0, 2560 <- 18432 36.8 / 80.0;
// at 65 43.0, 46.7, 58.0 and 82)
constexpr int kFewRows = 64;
template <int RT>
__device__ __forceinline__ void few_dx(const PrepareArgs &p, int block, FewLds &lds) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, i = lane & 7, kq = lane >> 3 & 3, h = lane >> 5, r = lane & 31;
    const int t = wave & 3, half = wave >> 2, G = p.K / kGroupK, tiles = p.N / kTileN, g = block / p.slices, slice = block % p.slices;
    const int turns = (tiles + kFewTiles - 1) / kFewTiles, each = (turns + p.slices - 1) / p.slices * kFewTiles;
    const uint32_t *words = reinterpret_cast<const uint32_t *>(lds.in.codes) + (i + 8 * h + 16 * kq) * 4 + t;
    f32x16 acc[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[rt][e] = 0.f;
    u32x4 codes[kFewTiles / 8], scales = {0u, 0u, 0u, 0u}, dy[2 * RT];
    auto fetch = [&](int base) {  // (N is a multiple of kFewColumns)
#pragma unroll
        for (int u = 0; u < kFewTiles / 8; ++u) codes[u] = p.B[((size_t)(base + 8 * u + wave) * G + g) * 64 + lane];
        if (tid < 2 * kFewTiles)
            scales = *reinterpret_cast<const u32x4 *>(p.S + scale_index(p.Gs == 1 ? 0 : g, (base + (tid >> 1)) * kTileN + 8 * (tid & 1), p.Gs));
#pragma unroll
        for (int u = 0; u < 2 * RT; ++u)
            dy[u] = *reinterpret_cast<const u32x4 *>(p.dy + (size_t)min(16 * u + (tid >> 5), p.m - 1) * p.N + base * kTileN + 8 * (tid & 31));
    };
    const int last = min(tiles, (slice + 1) * each);
    fetch(slice * each);
    for (int base = slice * each; base < last; base += kFewTiles) {
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kFewTiles / 8; ++u) lds.in.codes[(8 * u + wave) * 64 + lane] = codes[u];
        if (tid < 2 * kFewTiles) *reinterpret_cast<u32x4 *>(lds.in.scales + 8 * tid) = scales;
#pragma unroll
        for (int u = 0; u < 2 * RT; ++u) *reinterpret_cast<u32x4 *>(lds.in.dy + (16 * u + (tid >> 5)) * kFewDyPitch + 8 * (tid & 31)) = dy[u];
        __syncthreads();
        fetch(min(base + kFewTiles, tiles - kFewTiles));
#pragma unroll 1
        for (int tile = kFewTiles / 2 * half; tile < kFewTiles / 2 * (half + 1); ++tile) {
            const uint32_t v = exchange_nibbles<4>(exchange_nibbles<2>(exchange_nibbles<1>(words[tile * 256], lane), lane), lane);
            const u32x4 s = *reinterpret_cast<const u32x4 *>(lds.in.scales + tile * kTileN + 8 * h);
            bf16x8 o;
#pragma unroll
            for (int c = 0; c < 8; ++c)
                o[c] = (__bf16)((float)((int)(v >> (4 * c) & 0xF) - 8) * f16_bits_to_f32((uint16_t)(c & 1 ? s[c >> 1] >> 16 : s[c >> 1])));
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
                acc[rt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(o, load_bf16x8(lds.in.dy + (32 * rt + r) * kFewDyPitch + tile * kTileN + 8 * h), acc[rt], 0, 0, 0);
        }
    }
    for (int w = 0; w < 2; ++w) {
        __syncthreads();
        if (half == w)
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int e = 0; e < 16; ++e) {  // row 8 (e / 4) + 4 h + e % 4 of the product: rows of k come in the nibbles' order
                    float *at = lds.sums + (32 * rt + r) * kFewPitch + 32 * t + 8 * (e >> 2) + 2 * (e & 3) + h;
                    *at = (w ? *at : 0.f) + acc[rt][e];
                }
    }
    __syncthreads();
    for (int e = tid; e < p.m * 32; e += kPrepareThreads)
        *reinterpret_cast<f32x4 *>(p.partial + ((size_t)slice * p.m + (e >> 5)) * p.K + g * kGroupK + 4 * (e & 31)) =
            *reinterpret_cast<const f32x4 *>(lds.sums + (e >> 5) * kFewPitch + 4 * (e & 31));
}

// Up to 64 rows: U = dy B of 16 rows and one slice of the columns (T: project_rows).  A lane reads eight of B's rank, [n, rank], for each of
// its eight n and pairs the n's values (v_perm), one product for each of the eight, as bank_grad_kernel does for its rows.
__device__ __forceinline__ void few_project_dy(const PrepareArgs &p, int slice, int tile, unsigned turn0, FewLds &lds) {
    constexpr int W = kPrepareThreads / 64;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, q = lane >> 4, p0 = 16 * tile, rank = p.rank;
    const int each = (p.N / 128 + p.u_slices - 1) / p.u_slices * 128, begin = slice * each + 32 * wave, end = min(p.N, (slice + 1) * each);
    const uint16_t *src = p.dy + (size_t)min(p0 + c, p.m - 1) * p.N + 8 * q;
    adapters_of_turn(p.rows, p0, c, turn0, p.turns, [&](int adapter, unsigned mine) {
        const uint16_t *mat = p.b + ((size_t)adapter * p.N + 8 * q) * rank + 8 * min(c, rank / 8 - 1);
        f32x4 acc[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int at = begin; at < end; at += 2 * 32 * W) {
            bf16x8 x[2];
            u32x4 v[2][8];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int n = min(at + 32 * W * u, p.N - 32);
                x[u] = load_bf16x8(src + n);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[u][i] = *reinterpret_cast<const u32x4 *>(mat + (size_t)(n + i) * rank);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int u = 0; u < 2; ++u)
                if (at + 32 * W * u < end)
#pragma unroll
                    for (int e = 0; e < 8; ++e) acc[e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[u], column_of_rows(v[u], e), acc[e], 0, 0, 0);
        }
        if (c < rank / 8)
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
                for (int i = 0; i < 4; ++i) lds.projected[wave][4 * q + i][8 * c + e] = acc[e][i];
        join_projected<W>(lds.projected, p.u, p.rows, p0, slice, rank, mine);
    });
}

// at[a][k][rank] of a[a][rank][k], or bt[a][rank][n] of b[a][n][rank]; 64 of k or n to a block.  `at` is multiplied with rows of several
// adapters at once, zeros for those of others, so it holds finite values alone; where A holds others, odd[a][k / 64] is set and
// bank_grad_kernel adds their products for the rows of that adapter.
__device__ __forceinline__ void turn_bank(const PrepareArgs &p, int block, PrepareLds &lds) {
    const int tid = threadIdx.x, rank = p.rank, of_a = p.K / 64, parts = of_a + p.N / 64, a = block / parts, part = block % parts;
    const bool is_a = part < of_a;
    const int len = is_a ? p.K : p.N, l0 = (is_a ? part : part - of_a) * 64;
    const size_t base = (size_t)a * rank * len;
    if (is_a) {
        bool any = false;
        for (int e = tid; e < rank * 64; e += kPrepareThreads) {
            uint16_t v = p.a[base + (size_t)(e >> 6) * len + l0 + (e & 63)];
            if ((v & 0x7F80u) == 0x7F80u) {
                any = true;
                v = 0;
            }
            lds.bank[e & 63][e >> 6] = v;
        }
        any = __syncthreads_or(any);
        if (tid == 0) p.odd[(size_t)a * of_a + part] = any;
        for (int e = tid; e < 64 * rank; e += kPrepareThreads) p.at[base + (size_t)l0 * rank + e] = lds.bank[e / rank][e % rank];
    } else {
        for (int e = tid; e < 64 * rank; e += kPrepareThreads) lds.bank[e / rank][e % rank] = p.b[base + (size_t)l0 * rank + e];
        __syncthreads();
        for (int e = tid; e < rank * 64; e += kPrepareThreads) p.bt[base + (size_t)(e >> 6) * len + l0 + (e & 63)] = lds.bank[e & 63][e >> 6];
    }
}

// RT: row tiles of a call of few rows, whose projections are here too, or 0 for a weight unpacked
template <int RT>
__global__ __launch_bounds__(kPrepareThreads, 4) void bank_prepare_kernel(PrepareArgs p) {
    __shared__ __align__(16) std::conditional_t<(RT > 0), FewLds, PrepareLds> lds;
    int block = blockIdx.x;
    if constexpr (RT > 0) {
        if (block < p.slices * (p.K / kGroupK)) {
            few_dx<RT>(p, block, lds);
            return;
        }
        block -= p.slices * (p.K / kGroupK);
        const int all = p.t_slices + p.u_slices, place = block % all, rest = block / all;
        const int tile = rest / p.turns, turn0 = rest % p.turns;
        if (place < p.u_slices) few_project_dy(p, place, tile, turn0, lds);
        else project_rows<kPrepareThreads / 64>(BankProjection{p.x, p.a, p.t, p.K, p.t_slices}, p.rows, p.rank, place - p.u_slices, tile, turn0, p.turns, lds.projected);
    } else {
        if (block < p.order_blocks) {
            order_rows(p.rows.of, p.rows.order, p.rows.first, p.rows.rows, p.rows.count, block, lds.order);
            return;
        }
        block -= p.order_blocks;
        if (block < p.turn_blocks) turn_bank(p, block, lds);
        else unpack_weight(p, block - p.turn_blocks, lds);
    }
}

// sums over slices: x[0][i] += x[1][i] + ... (both projections in one launch)
__global__ __launch_bounds__(256) void sum_slices_kernel(float *__restrict__ t, int t_slices, float *__restrict__ u, int u_slices, size_t count) {
    float *x = blockIdx.y ? u : t;
    const int slices = blockIdx.y ? u_slices : t_slices;
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= count || slices == 1) return;
    float v = x[i];
    for (int s = 1; s < slices; ++s) v += x[(size_t)s * count + i];
    x[i] = v;
}

// ---- dx --------------------------------------------------------------------------------------------------------
// dx[row][k] = sum_n dy[row][n] W[k][n] (+ s U A), both operands with the contraction contiguous.  A block of WM x WN wavefronts takes
// 32 TM WM rows x 32 TN WN of k, 32 of the contraction at a time: both tiles go straight to LDS, kStages - 1 of them in flight while one is
// multiplied.  A row of a tile is four 16-byte units, unit u at place u ^ (row / 2 & 3), so that the eight lanes that LDS serves together
// find their units in different banks.
constexpr int kStages = 4;
struct DxArgs {
    const uint16_t *dy, *wt, *at;   // [rows, N], [K, N], [count, K, rank]
    const float *u, *scales;        // [rows by position, rank], or null without a bank
    uint16_t *dx;
    float *partial;                 // [slices, rows, K], or null with one slice
    BankRows rows;
    int K, N, rank, steps;          // steps of 32 of the contraction to a slice
    int m_tiles, k_tiles;
};

__device__ __forceinline__ unsigned unit_at(int row, int unit) { return (unsigned)(row * 4 + (unit ^ (row >> 1 & 3))) * 16; }

template <int WM, int WN, int TM, int TN>
__global__ __launch_bounds__(WM * WN * 64) void bank_dx_kernel(DxArgs p) {
    constexpr int W = WM * WN, BM = 32 * TM * WM, BN = 32 * TN * WN, kStage = (BM + BN) * 64;
    constexpr int LM = BM / 16 / W, LN = BN / 16 / W;  // 16-row loads of either tile to a wavefront
    static_assert(BM % (16 * W) == 0 && BN % (16 * W) == 0, "");
    extern __shared__ __align__(16) char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave % WM, wn = wave / WM;
    // Blocks go to the eight dies in turn: a die's blocks are those side by side in (slice, k, m), m first, which share most of what
    // they read.
    const int total = gridDim.x, die = blockIdx.x % 8, each = total / 8, more = total % 8;
    const int id = die * each + min(die, more) + blockIdx.x / 8;
    const int m_tile = id % p.m_tiles, k_tile = id / p.m_tiles % p.k_tiles, slice = id / (p.m_tiles * p.k_tiles);
    const int k0 = k_tile * BN, p0 = m_tile * BM;
    const int first = slice * p.steps, last = min(p.N / 32, first + p.steps);
    const uint16_t *xs[LM], *ws[LN];
    const int unit = (lane & 3) ^ (lane >> 3 & 3);
#pragma unroll
    for (int i = 0; i < LM; ++i) {
        const int at = min(p0 + 16 * (LM * wave + i) + (lane >> 2), p.rows.rows - 1);
        xs[i] = p.dy + (size_t)(p.rows.order ? p.rows.order[at] : at) * p.N + 8 * unit;
    }
#pragma unroll
    for (int i = 0; i < LN; ++i) ws[i] = p.wt + (size_t)min(k0 + 16 * (LN * wave + i) + (lane >> 2), p.K - 1) * p.N + 8 * unit;
    const unsigned lds0 = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(lds_ptr_t)lds);
    auto fetch = [&](int step) {  // past the slice's end: its last step again, so that the count of loads in flight stays what it is
        const int buffer = (step - first) % kStages;
        const size_t from = (size_t)min(step, last - 1) * 32;
        const unsigned at = lds0 + buffer * kStage + wave * (LM * 1024), bt = lds0 + buffer * kStage + BM * 64 + wave * (LN * 1024);
#pragma unroll
        for (int i = 0; i < LM; ++i) load_to_lds_b128(xs[i] + from, at + i * 1024);
#pragma unroll
        for (int i = 0; i < LN; ++i) load_to_lds_b128(ws[i] + from, bt + i * 1024);
    };
    f32x16 acc[TN][TM];
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[j][i][e] = 0.f;
    const int r = lane & 31, h = lane >> 5;
    struct Operands {
        bf16x8 x[TM], w[TN];
    };
    auto read = [&](const char *stage, int kk, Operands &o) {
#pragma unroll
        for (int i = 0; i < TM; ++i) o.x[i] = *reinterpret_cast<const bf16x8 *>(stage + unit_at(32 * (TM * wm + i) + r, 2 * kk + h));
#pragma unroll
        for (int j = 0; j < TN; ++j) o.w[j] = *reinterpret_cast<const bf16x8 *>(stage + BM * 64 + unit_at(32 * (TN * wn + j) + r, 2 * kk + h));
    };
    auto multiply = [&](const Operands &o) {
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int i = 0; i < TM; ++i) acc[j][i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(o.w[j], o.x[i], acc[j][i], 0, 0, 0);
    };
    // Operands are read half a step ahead, and the wavefronts meet in mid-step, where the second half's are in registers and the
    // first half's products run: behind that, the present step's place is free for the step kStages on.
    Operands now, then;
#pragma unroll
    for (int s = 0; s < kStages; ++s) fetch(first + s);
    wait_vector_loads<(kStages - 1) * (LM + LN)>();
    __builtin_amdgcn_s_barrier();
    read(lds, 0, now);
    for (int step = first; step < last; ++step) {
        const int buffer = (step - first) % kStages;
        read(lds + buffer * kStage, 1, then);
        __builtin_amdgcn_sched_barrier(0);
        multiply(now);
        __builtin_amdgcn_sched_barrier(0);
        wait_vector_loads<(kStages - 2) * (LM + LN)>();
        wait_lds_reads();
        __builtin_amdgcn_s_barrier();
        fetch(step + kStages);
        read(lds + (buffer + 1) % kStages * kStage, 0, now);
        __builtin_amdgcn_sched_barrier(0);
        multiply(then);
        __builtin_amdgcn_sched_barrier(0);
    }
    wait_lds_reads();
    wait_vector_loads<0>();
    if (p.u && slice == 0) {
        // U A: the runs of rows of one adapter among the block's positions, 32 of the rank at a time, U's bf16 value and then what that
        // leaves, zeros for the rows of others (and `at` holds finite values alone: turn_bank_kernel).
        const int end = min(p0 + BM, p.rows.first[p.rows.count]);
        for (int q0 = p0; q0 < end;) {
            const int a = p.rows.of[p.rows.order[q0]], q1 = min(p.rows.first[a + 1], end);
            const float scale = p.scales[a];
            for (int c0 = 0; c0 < p.rank; c0 += 32)
                for (int side = 0; side < 2; ++side) {
                    __syncthreads();
                    for (int e = tid; e < BM * 4; e += W * 64) {
                        const int row = e >> 2, unit = e & 3, col = c0 + 8 * unit;
                        bf16x8 v = bf16x8_zero();
                        if (p0 + row >= q0 && p0 + row < q1 && col < p.rank) {
                            const float *u = p.u + (size_t)(p0 + row) * p.rank + col;
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                const float f = u[i] * scale;
                                const __bf16 hi = (__bf16)f;
                                v[i] = side ? lower_part(f, hi) : hi;
                            }
                        }
                        *reinterpret_cast<bf16x8 *>(lds + unit_at(row, unit)) = v;
                    }
                    if (side == 0)
                        for (int e = tid; e < BN * 4; e += W * 64) {
                            const int row = e >> 2, unit = e & 3, col = c0 + 8 * unit;
                            u32x4 v = {0u, 0u, 0u, 0u};
                            if (k0 + row < p.K && col < p.rank) v = *reinterpret_cast<const u32x4 *>(p.at + ((size_t)a * p.K + k0 + row) * p.rank + col);
                            *reinterpret_cast<u32x4 *>(lds + BM * 64 + unit_at(row, unit)) = v;
                        }
                    __syncthreads();
                    read(lds, 0, now);
                    read(lds, 1, then);
                    multiply(now);
                    multiply(then);
                }
            q0 = q1;
        }
    }
    // a lane holds column lane & 31 (a row of dx) and four consecutive k at 8 g + 4 (lane >> 5)
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const int at = p0 + 32 * (TM * wm + i) + r;
        if (at >= p.rows.rows) continue;
        const int row = p.rows.order ? p.rows.order[at] : at;
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int k = k0 + 32 * (TN * wn + j) + 8 * g + 4 * h;
                if (k >= p.K) continue;
                f32x4 v = {acc[j][i][4 * g], acc[j][i][4 * g + 1], acc[j][i][4 * g + 2], acc[j][i][4 * g + 3]};
                if (p.partial) {
                    *reinterpret_cast<f32x4 *>(p.partial + ((size_t)slice * p.rows.rows + row) * p.K + k) = v;
                } else {
                    u32x2 o;
                    o.x = f32_to_bf16_bits(v[0]) | (uint32_t)f32_to_bf16_bits(v[1]) << 16;
                    o.y = f32_to_bf16_bits(v[2]) | (uint32_t)f32_to_bf16_bits(v[3]) << 16;
                    *reinterpret_cast<u32x2 *>(p.dx + (size_t)row * p.K + k) = o;
                }
            }
    }
}

// dx = the slices' sum, rounded once
__global__ __launch_bounds__(256) void sum_dx_kernel(const f32x4 *__restrict__ partial, u32x2 *__restrict__ dx, int slices, size_t count) {
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= count) return;
    f32x4 v = partial[i];
    for (int s = 1; s < slices; ++s) v += partial[(size_t)s * count + i];
    dx[i] = u32x2{f32_to_bf16_bits(v[0]) | (uint32_t)f32_to_bf16_bits(v[1]) << 16, f32_to_bf16_bits(v[2]) | (uint32_t)f32_to_bf16_bits(v[3]) << 16};
}

// ---- dA and dB -------------------------------------------------------------------------------------------------
// out = s_a sum over the rows of adapter a of f[position][rank]^T src[row][columns], f = U with src = x (dA) or T with src = dy (dB).
// Bound by src, read once: a block takes 128 columns, its W wavefronts every W-th 32 rows.  The contraction runs over the rows, of which
// an operand of the matrix instruction wants eight to a lane: a lane reads eight columns of each of its eight rows and pairs the rows'
// values column by column (v_perm), so that nothing goes through LDS; its eight columns are eight products.  T and U go in as two bf16
// parts, within 2^-17 of their f32 values.  (With the f32 matrix instruction, which needs no pairing, the products took as long as the reads:
// 2048 rows, 20992 columns, rank 32: 62 us.)
struct GradArgs {
    const uint16_t *x, *dy;
    const float *t, *u, *scales;
    uint16_t *da, *db;
    BankRows rows;
    int K, N, rank;
    const uint16_t *a;   // the adapters' A as they lie, [count, rank, K]
    const uint8_t *odd;  // [count, K / 64]: where A holds values that are no finite numbers,
    uint16_t *dx;        // whose products are still to be added here
    const float *partial;  // few rows: [slices, rows, K], dx's to be summed and joined by U A here,
    int grad_blocks, slices, t_slices, u_slices;  // as are T's and U's slices
};

// T or U of few rows, their slices summed: ts[i] = row list[i]'s
__device__ __forceinline__ void sum_few(const GradArgs &p, bool of_t, const int *list, int count, int threads, float (&ts)[kFewRows][kBankMaxRank + 4]) {
    const size_t stride = (size_t)p.rows.rows * p.rank;
    const int slices = of_t ? p.t_slices : p.u_slices;
    for (int e = 4 * (int)threadIdx.x; e < count * p.rank; e += 4 * threads) {
        const int i = e / p.rank, col = e - i * p.rank;
        const float *from = (of_t ? p.t : p.u) + (size_t)list[i] * p.rank + col;
        f32x4 d[kFewProjected], v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < kFewProjected; ++s) d[s] = *reinterpret_cast<const f32x4 *>(from + min(s, slices - 1) * stride);
#pragma unroll
        for (int s = 0; s < kFewProjected; ++s)
            if (s < slices) v += d[s];
        *reinterpret_cast<f32x4 *>(&ts[i][col]) = v;
    }
    __syncthreads();
}

// dx of few rows: the slices' sum and the low-rank term, 4 W 64 of k of one row to a block
__device__ __forceinline__ void finish_dx(const GradArgs &p, int block, int threads, int *list, float (&ts)[kFewRows][kBankMaxRank + 4]) {
    const int parts = (p.K / 4 + threads - 1) / threads, row = block / parts, k = (block % parts * threads + (int)threadIdx.x) * 4;
    int a = p.rows.of[row];
    if ((unsigned)a >= (unsigned)p.rows.count) a = -1;
    if (a >= 0) {
        if (threadIdx.x == 0) list[0] = row;
        __syncthreads();
        sum_few(p, false, list, 1, threads, ts);
    }
    if (k >= p.K) return;
    const size_t stride = (size_t)p.rows.rows * p.K;
    const float *from = p.partial + (size_t)row * p.K + k;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    int s = 0;
    for (; s + 4 <= p.slices; s += 4) {
        f32x4 d[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) d[i] = *reinterpret_cast<const f32x4 *>(from + (s + i) * stride);
        v += (d[0] + d[1]) + (d[2] + d[3]);
    }
    for (; s < p.slices; ++s) v += *reinterpret_cast<const f32x4 *>(from + s * stride);
    if (a >= 0) {
        const uint16_t *m = p.a + (size_t)a * p.rank * p.K + k;
        const float *u = ts[0];
        f32x4 low = {0.f, 0.f, 0.f, 0.f};
        for (int r0 = 0; r0 < p.rank; r0 += 8) {
            u32x2 d[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] = *reinterpret_cast<const u32x2 *>(m + (size_t)(r0 + i) * p.K);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float f = u[r0 + i];
                low[0] += f * __builtin_bit_cast(float, d[i].x << 16);
                low[1] += f * __builtin_bit_cast(float, d[i].x & 0xFFFF0000u);
                low[2] += f * __builtin_bit_cast(float, d[i].y << 16);
                low[3] += f * __builtin_bit_cast(float, d[i].y & 0xFFFF0000u);
            }
        }
        const float scale = p.scales[a];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += scale * low[i];
    }
    u32x2 o;
    o.x = f32_to_bf16_bits(v[0]) | (uint32_t)f32_to_bf16_bits(v[1]) << 16;
    o.y = f32_to_bf16_bits(v[2]) | (uint32_t)f32_to_bf16_bits(v[3]) << 16;
    *reinterpret_cast<u32x2 *>(p.dx + (size_t)row * p.K + k) = o;
}

constexpr int kGradPitch = 128 + 4;
// FEW: rows as they stand, 64 at most, T and U still in slices
template <int JT, int W, bool FEW>
__global__ __launch_bounds__(W * 64) void bank_grad_kernel(GradArgs p) {
    __shared__ float sum[JT * 16 * kGradPitch];
    __shared__ int list[FEW ? kFewRows : 1];
    __shared__ __align__(16) float ts[FEW ? kFewRows : 1][kBankMaxRank + 4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 15, q = lane >> 4;
    if constexpr (FEW) {
        if ((int)blockIdx.x >= p.grad_blocks) {
            finish_dx(p, blockIdx.x - p.grad_blocks, W * 64, list, ts);
            return;
        }
    }
    const int parts = p.N / 128 + p.K / 128, a = blockIdx.x / parts, block = blockIdx.x % parts;
    const bool is_b = block < p.N / 128;
    const int c0 = (is_b ? block : block - p.N / 128) * 128, len = is_b ? p.N : p.K;
    const uint16_t *src = (is_b ? p.dy : p.x) + c0 + 8 * c;
    const float *f = is_b ? p.t : p.u;
    int begin = 0, end;
    if constexpr (FEW) {
        const bool mine = lane < p.rows.rows && p.rows.of[lane] == a;
        const unsigned long long all = __ballot(mine);
        end = __popcll(all);
        if (wave == 0 && mine) list[__popcll(all & ((1ull << lane) - 1))] = lane;
        __syncthreads();
        sum_few(p, is_b, list, end, W * 64, ts);
    } else {
        begin = p.rows.first[a], end = p.rows.first[a + 1];
    }
    int col[JT];  // past the rank: the last again, dropped at the end
#pragma unroll
    for (int j = 0; j < JT; ++j) col[j] = min(16 * j + c, p.rank - 1);
    f32x4 acc[8][JT];
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int j = 0; j < JT; ++j) acc[e][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    int row[8];
    auto rows_at = [&](int at) {  // positions past the last: the last again, times zeros
#pragma unroll
        for (int i = 0; i < 8; ++i) row[i] = FEW ? list[min(at + 8 * q + i, end - 1)] : p.rows.order[min(at + 8 * q + i, end - 1)];
    };
    int at = begin + 32 * wave;
    if (at < end) rows_at(at);
    for (; at < end; at += 32 * W) {
        u32x4 v[8];
        float w[JT][8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = *reinterpret_cast<const u32x4 *>(src + (size_t)row[i] * len);
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < JT; ++j)
                w[j][i] = FEW ? ts[FEW ? min(at + 8 * q + i, end - 1) : 0][col[j]] : f[(size_t)min(at + 8 * q + i, end - 1) * p.rank + col[j]];
        rows_at(at + 32 * W);
        __builtin_amdgcn_sched_barrier(0);
        bf16x8 hi[JT], lo[JT];
#pragma unroll
        for (int j = 0; j < JT; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float x = at + 8 * q + i < end ? w[j][i] : 0.f;
                hi[j][i] = (__bf16)x;
                lo[j][i] = lower_part(x, hi[j][i]);
            }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const bf16x8 b = column_of_rows(v, e);
#pragma unroll
            for (int j = 0; j < JT; ++j) {
                acc[e][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hi[j], b, acc[e][j], 0, 0, 0);
                acc[e][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(lo[j], b, acc[e][j], 0, 0, 0);
            }
        }
    }
    for (int w = 0; w < W; ++w) {  // the wavefronts' sums one after the other: the same order always
        if (wave == w)
#pragma unroll
            for (int j = 0; j < JT; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float *dst = sum + (16 * j + 4 * q + i) * kGradPitch + 8 * c;
#pragma unroll
                    for (int e = 0; e < 8; ++e) dst[e] = (w ? dst[e] : 0.f) + acc[e][j][i];
                }
        __syncthreads();
    }
    const float scale = begin < end ? p.scales[a] : 0.f;  // without rows: zeros, whatever the scale
    uint16_t *out = is_b ? p.db + ((size_t)a * p.N + c0) * p.rank : p.da + (size_t)a * p.rank * p.K + c0;
    for (int e = tid; e < p.rank * 16; e += W * 64) {  // eight results each
        const int r = is_b ? e % (p.rank / 8) : e >> 4, col = is_b ? e / (p.rank / 8) : e & 15;
        u32x4 o;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float lo = is_b ? sum[(8 * r + 2 * i) * kGradPitch + col] : sum[r * kGradPitch + 8 * col + 2 * i];
            const float hi = is_b ? sum[(8 * r + 2 * i + 1) * kGradPitch + col] : sum[r * kGradPitch + 8 * col + 2 * i + 1];
            o[i] = f32_to_bf16_bits(lo * scale) | (uint32_t)f32_to_bf16_bits(hi * scale) << 16;
        }
        *reinterpret_cast<u32x4 *>(is_b ? out + (size_t)col * p.rank + 8 * r : out + (size_t)r * p.K + 8 * col) = o;
    }
    if (FEW || is_b) return;
    const uint8_t *odd = p.odd + (size_t)a * (p.K / 64) + c0 / 64;
    if (!(odd[0] | odd[1])) return;
    for (int at = begin + (tid >> 7); at < end; at += W / 2) {
        const int k = c0 + (tid & 127);
        uint16_t *dx = p.dx + (size_t)p.rows.order[at] * p.K + k;
        float v = __builtin_bit_cast(float, (uint32_t)*dx << 16);
        for (int r = 0; r < p.rank; ++r) {
            const uint16_t bits = p.a[((size_t)a * p.rank + r) * p.K + k];
            if ((bits & 0x7F80u) == 0x7F80u) v += p.u[(size_t)at * p.rank + r] * scale * __builtin_bit_cast(float, (uint32_t)bits << 16);
        }
        *dx = f32_to_bf16_bits(v);
    }
}

template <int JT, int W>
void launch_grad(const GradArgs &g, bool few, hipStream_t stream) {
    if (few) {
        const int dx_blocks = g.rows.rows * ((g.K / 4 + W * 64 - 1) / (W * 64));
        bank_grad_kernel<JT, W, true><<<g.grad_blocks + dx_blocks, W * 64, 0, stream>>>(g);
    } else {
        bank_grad_kernel<JT, W, false><<<g.grad_blocks, W * 64, 0, stream>>>(g);
    }
}
template <int JT>
void launch_grad(GradArgs g, bool few, hipStream_t stream) {
    g.grad_blocks = (g.N / 128 + g.K / 128) * g.rows.count;
    if (g.grad_blocks >= 512) launch_grad<JT, 4>(g, few, stream);
    else launch_grad<JT, 8>(g, few, stream);
}

// ---- the plan ----------------------------------------------------------------------------------------------------
// The block of the product for dx and the slices of its contraction.  A block of 256 x 256 is the fastest by its area (2048 rows of n 18432, k
// 2560, three slices: 189 us, 1.02 PFLOP/s; 128 x 256 216, 128 x 128 237), a smaller one where those would leave compute units without
// work (777 rows, 2560 -> 9216: 128 x 256 49 us, 128 x 128 55, 256 x 256 79).  Times by a model: so many rounds of blocks, each its steps
// at what one takes, measured, and with slices what writing, reading and adding them takes.  (Of 256 compute units, the part's: the scratch that
// holds the slices is asked for without a device, and a plan of another count could need more.)
struct DxPlan {
    int kind;    // 0: 128 x 128, two blocks to a compute unit; 1: 128 x 256; 2: 256 x 256
    int slices;
};
constexpr int kMaxDxSlices = 8, kComputeUnits = 256;
constexpr int kDxTileM[3] = {128, 128, 256}, kDxTileK[3] = {128, 256, 256};
DxPlan dx_plan(int m, int n, int k) {
    DxPlan best{0, 1};
    float least = 0.f;
    for (int kind = 0; kind < 3; ++kind)
        for (int slices = 1; slices <= kMaxDxSlices; ++slices) {
            const int steps = n / 32, each = (steps + slices - 1) / slices;
            if (slices > 1 && (each < 8 || (steps + each - 1) / each != slices)) continue;
            const int64_t tiles = (int64_t)((m + kDxTileM[kind] - 1) / kDxTileM[kind]) * ((k + kDxTileK[kind] - 1) / kDxTileK[kind]) * slices;
            const float rounds = kind ? (float)((tiles + kComputeUnits - 1) / kComputeUnits)
                                      : tiles <= kComputeUnits ? 0.54f : (float)((tiles + 2 * kComputeUnits - 1) / (2 * kComputeUnits));
            const float step_us = kind == 2 ? 0.85f : kind == 1 ? 0.52f : 0.54f;
            const float t = rounds * (each + 6) * step_us + (slices > 1 ? 3.f + 2e-6f * slices * (float)m * (float)k : 0.f);
            if ((kind == 0 && slices == 1) || t < least) {
                least = t;
                best = DxPlan{kind, slices};
            }
        }
    return best;
}

void launch_prepare(const PrepareArgs &p, hipStream_t stream) {
    const int groups = p.K / kGroupK;
    if (p.m > kFewRows) {
        bank_prepare_kernel<0><<<p.order_blocks + p.turn_blocks + (p.N / 128) * groups, kPrepareThreads, 0, stream>>>(p);
        return;
    }
    const int blocks = p.slices * groups + (p.t_slices + p.u_slices) * ((p.m + 15) / 16) * p.turns;
    if (p.m > 32) bank_prepare_kernel<2><<<blocks, kPrepareThreads, 0, stream>>>(p);
    else bank_prepare_kernel<1><<<blocks, kPrepareThreads, 0, stream>>>(p);
}

template <int WM, int WN, int TM, int TN>
hipError_t launch_dx(DxArgs p, int slices, hipStream_t stream) {
    constexpr int BM = 32 * TM * WM, BN = 32 * TN * WN, kLds = kStages * (BM + BN) * 64;
    const hipError_t attr = allow_dynamic_lds<&bank_dx_kernel<WM, WN, TM, TN>>(kLds);
    if (attr != hipSuccess) return attr;
    p.m_tiles = (p.rows.rows + BM - 1) / BM;
    p.k_tiles = (p.K + BN - 1) / BN;
    p.steps = (p.N / 32 + slices - 1) / slices;
    bank_dx_kernel<WM, WN, TM, TN><<<p.m_tiles * p.k_tiles * slices, WM * WN * 64, kLds, stream>>>(p);
    return hipSuccess;
}

// Up to 64 rows: slices of the columns, of 256 at least; 16 at most, by what they add up to
int few_slices(int n) {
    const int turns = n / kFewColumns, slices = turns < 16 ? turns : 16, each = (turns + slices - 1) / slices;
    return (turns + each - 1) / each;
}

// ... and of their projections' contraction, of 1024 at least
int few_project_slices(int len) {
    const int groups = len / 128, slices = (groups + 7) / 8 < kFewProjected ? (groups + 7) / 8 : kFewProjected, each = (groups + slices - 1) / slices;
    return (groups + each - 1) / each;
}

struct BackwardScratch {
    size_t wt, at, bt, odd, order, t, u, partial, total;
    int t_slices, u_slices, few;
    DxPlan dx;
};
BackwardScratch backward_scratch(int m, int n, int k, int count, int rank) {
    BackwardScratch s{};
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += bank_up256(bytes);
        return here;
    };
    s.few = m <= kFewRows ? few_slices(n) : 0;
    s.wt = take(s.few ? 0 : (size_t)k * n * 2);
    if (count > 0) {
        if (s.few) {
            s.t_slices = few_project_slices(k);
            s.u_slices = few_project_slices(n);
        } else {
            s.at = take((size_t)count * rank * k * 2);
            s.bt = take((size_t)count * rank * n * 2);
            s.odd = take((size_t)count * (k / 64));
            s.order = take(bank_order_bytes(m, count));
            s.t_slices = bank_slices(m, k);
            s.u_slices = bank_slices(m, n);
        }
        s.t = take((size_t)s.t_slices * m * rank * 4);
        s.u = take((size_t)s.u_slices * m * rank * 4);
    }
    s.dx = s.few ? DxPlan{0, s.few} : dx_plan(m, n, k);
    s.partial = take(s.few || s.dx.slices > 1 ? (size_t)s.dx.slices * m * k * 4 : 0);
    s.total = at;
    return s;
}

}  // namespace
}  // namespace kiln

using namespace kiln;

extern "C" {

size_t kiln_w4a16_gemm_bank_backward_scratch_bytes(int prob_m, int prob_n, int prob_k, int count, int rank) {
    if (prob_n < 256 || prob_k < 128 || count < 0 || rank < 0) return 256;
    return backward_scratch(prob_m < 1 ? 1 : prob_m, prob_n, prob_k, count, rank).total;
}

int kiln_w4a16_debug_bank_backward_plan(int prob_m, int prob_n, int prob_k, int *out) {
    if (prob_m < 1 || prob_n < 256 || prob_n % 256 != 0 || prob_k < 128 || prob_k % 128 != 0) return 1;
    const BackwardScratch w = backward_scratch(prob_m, prob_n, prob_k, 0, 0);
    out[0] = w.few ? 0 : kDxTileM[w.dx.kind];
    out[1] = w.few ? 0 : kDxTileK[w.dx.kind];
    out[2] = w.dx.slices;
    return 0;
}

kiln_marlin_status_t kiln_w4a16_gemm_bank_backward(const void *dC, const void *A, const void *B, const void *s, int prob_m, int prob_n, int prob_k,
                                                   int groupsize, int dev, void *stream, const kiln_w4a16_adapter_bank *bank, const int *adapter_of,
                                                   void *dA, void *d_lora_a, void *d_lora_b, void *scratch) {
    (void)dev;
    if (prob_m < 0 || prob_n < 0 || prob_k < 0 || prob_k % 128 != 0 || prob_n % 256 != 0 || (groupsize != -1 && groupsize != 128))
        return KILN_W4A16_ERR_PROB_SHAPE;
    if (prob_n == 0 || prob_k == 0 || (prob_m == 0 && !bank)) return KILN_W4A16_OK;
    if (bank && !bank_ok(*bank)) return KILN_W4A16_ERR_KERN_SHAPE;
    if (prob_m > 0 && (!dC || !B || !s || !dA || !scratch)) return KILN_W4A16_ERR_ARGUMENT;
    if (bank && (!d_lora_a || !d_lora_b || !scratch || !bank->scales || (prob_m > 0 && (!A || !adapter_of || !bank->lora_a || !bank->lora_b))))
        return KILN_W4A16_ERR_ARGUMENT;
    for (const void *p : {dC, A, B, s, static_cast<const void *>(dA), static_cast<const void *>(scratch),
                          bank ? bank->lora_a : nullptr, bank ? bank->lora_b : nullptr, static_cast<const void *>(d_lora_a), static_cast<const void *>(d_lora_b)})
        if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return KILN_W4A16_ERR_ARGUMENT;
    const int m = prob_m, n = prob_n, k = prob_k, count = bank ? bank->count : 0, rank = bank ? bank->rank : 0;
    const struct {
        const void *p;
        size_t bytes;
    } results[3] = {{dA, (size_t)m * k * 2}, {d_lora_a, (size_t)count * rank * k * 2}, {d_lora_b, (size_t)count * rank * n * 2}},
      operands[4] = {{dC, (size_t)m * n * 2}, {A, bank ? (size_t)m * k * 2 : 0}, {bank ? bank->lora_a : nullptr, results[1].bytes},
                     {bank ? bank->lora_b : nullptr, results[2].bytes}};
    for (const auto &r : results) {
        if (r.bytes)
            for (const auto &o : operands)
                if (o.bytes && meet(r.p, r.bytes, o.p, o.bytes)) return KILN_W4A16_ERR_ARGUMENT;
    }
    hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
    const BackwardScratch w = backward_scratch(m > 0 ? m : 1, n, k, count, rank);
    char *at = reinterpret_cast<char *>(scratch);
    uint16_t *wt = reinterpret_cast<uint16_t *>(at + w.wt);
    DxArgs dx{};
    dx.dy = (const uint16_t *)dC;
    dx.wt = wt;
    dx.dx = (uint16_t *)dA;
    float *partial = w.few || w.dx.slices > 1 ? reinterpret_cast<float *>(at + w.partial) : nullptr;
    dx.partial = partial;
    dx.rows = BankRows{nullptr, nullptr, nullptr, m, 0};
    dx.K = k;
    dx.N = n;
    GradArgs grad{};
    PrepareArgs prepare{};
    prepare.B = (const u32x4 *)B;
    prepare.S = (const uint16_t *)s;
    prepare.wt = wt;
    prepare.K = k;
    prepare.N = n;
    prepare.Gs = groupsize == -1 ? 1 : k / 128;
    prepare.dy = (const uint16_t *)dC;
    prepare.partial = partial;
    prepare.m = m;
    prepare.slices = w.few;
    if (bank) {
        float *t = reinterpret_cast<float *>(at + w.t), *u = reinterpret_cast<float *>(at + w.u);
        const uint16_t *lora_a = (const uint16_t *)bank->lora_a;
        uint16_t *a_t = reinterpret_cast<uint16_t *>(at + w.at), *b_t = reinterpret_cast<uint16_t *>(at + w.bt);
        uint8_t *odd = reinterpret_cast<uint8_t *>(at + w.odd);
        dx.rows = w.few ? BankRows{adapter_of, nullptr, nullptr, m, count} : bank_rows(adapter_of, m, count, at + w.order);
        prepare.a = lora_a;
        prepare.b = (const uint16_t *)bank->lora_b;
        prepare.rows = dx.rows;
        prepare.rank = rank;
        if (w.few) {
            prepare.x = (const uint16_t *)A;
            prepare.t = t;
            prepare.u = u;
            prepare.t_slices = w.t_slices;
            prepare.u_slices = w.u_slices;
            prepare.turns = count < 16 ? count : 16;  // the adapters that 16 rows may have
            if (m > 0) launch_prepare(prepare, hs);
        } else {
            prepare.at = a_t;
            prepare.bt = b_t;
            prepare.odd = odd;
            prepare.order_blocks = count + 1;
            prepare.turn_blocks = count * (k / 64 + n / 64);
            launch_prepare(prepare, hs);
            const BankProjection of_x{A, lora_a, t, k, w.t_slices};
            bank_project(BankProjection{dC, b_t, u, n, w.u_slices}, &of_x, dx.rows, rank, hs);
            if (w.t_slices > 1 || w.u_slices > 1)
                sum_slices_kernel<<<dim3((unsigned)(((size_t)m * rank + 255) / 256), 2), 256, 0, hs>>>(t, w.t_slices, u, w.u_slices, (size_t)m * rank);
        }
        grad = GradArgs{(const uint16_t *)A, (const uint16_t *)dC, t, u, bank->scales, (uint16_t *)d_lora_a, (uint16_t *)d_lora_b,
                        dx.rows, k, n, rank, lora_a, odd, (uint16_t *)dA, partial, 0, w.few, w.t_slices, w.u_slices};
        dx.at = a_t;
        dx.u = u;
        dx.scales = bank->scales;
        dx.rank = rank;
    } else {
        launch_prepare(prepare, hs);
    }
    if (m > 0 && !w.few) {
        const hipError_t launched = w.dx.kind == 0   ? launch_dx<2, 2, 2, 2>(dx, w.dx.slices, hs)
                                    : w.dx.kind == 1 ? launch_dx<2, 4, 2, 2>(dx, w.dx.slices, hs)
                                                     : launch_dx<2, 2, 4, 4>(dx, w.dx.slices, hs);
        if (launched != hipSuccess) return KILN_W4A16_ERR_LAUNCH;
    }
    if (m > 0 && (!bank || !w.few) && partial) {
        const size_t units = (size_t)m * k / 4;
        sum_dx_kernel<<<(unsigned)((units + 255) / 256), 256, 0, hs>>>((const f32x4 *)partial, (u32x2 *)dA, w.dx.slices, units);
    }
    if (bank) {  // behind dx, to which it adds where an adapter holds what is no finite number
        switch ((rank + 15) / 16) {
            case 1: launch_grad<1>(grad, w.few, hs); break;
            case 2: launch_grad<2>(grad, w.few, hs); break;
            case 3: launch_grad<3>(grad, w.few, hs); break;
            default: launch_grad<4>(grad, w.few, hs); break;
        }
    }
    return hipGetLastError() == hipSuccess ? KILN_W4A16_OK : KILN_W4A16_ERR_LAUNCH;
}

}  // extern "C"
