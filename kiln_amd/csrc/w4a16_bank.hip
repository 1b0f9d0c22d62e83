// A packed projection whose rows have low-rank adapters of their own out of a bank:
// y[i] = x[i] W + s_a (x[i] A_a^T) B_a^T, a = adapter_of[i].
//
// Three steps: T = x A^T (f32), the plain GEMM, and y += s T B^T in place; up to 16 rows the first two share a launch where that is faster,
// and a row or two on few adapters take one launch for everything (w4a16_bank_few.hip).  Thousands of rows on wide outputs: rows are put in
// the order of their adapters and the product adds the term where it stores a tile (w4a16_prefill.hip).  Rows are handled in tiles of 16
// positions or 64; a tile multiplies with each adapter that is present among its rows, once, and rows of other adapters are left out
// of the product, so any order of the rows is right and one in which an adapter's rows are together reads its matrices least often:
// from 257 rows on a launch in front puts them so.  The reference serves one adapter set per process
// (crates/kiln-model/src/lora_loader.rs:213-232); this is its formula with the adapter a row's own.
//
// Where the term is a step of its own, y is rounded to bf16 between the product and the term, as the reference rounds its base before it adds a
// delta: the product is the plain GEMM, whose result is bf16 (a row without an adapter has its bits), and y in f32 would be twice the bytes
// written and read again.  The error against 64 bits is 0.0023 of the result's norm then, 0.0017 (the result's rounding) where the
// term lands on f32 sums.
#include "bank.h"
#include "bank_expand.h"
#include "bank_order.h"
#include "device_common.h"
#include "launch.h"
#include "lora_project.h"

namespace kiln {
namespace {

constexpr int kOrderWaves = 16;
__global__ __launch_bounds__(kOrderWaves * 64) void bank_order_kernel(const int *__restrict__ of, int *__restrict__ order, int *__restrict__ first,
                                                                      int rows, int count) {
    __shared__ OrderLds<kOrderWaves> lds;
    order_rows(of, order, first, rows, count, blockIdx.x, lds);
}

// Rows put in order for the product, and their sums over a group times the codes' bias, in the order of additions that the plain GEMM has:
// 16 lanes to a group, a position to a wavefront, 20 of its groups in flight together.
constexpr int kGatherRows = 8;
__device__ __forceinline__ void gather_rows(const BankGather &p, const BankRows &rows, int block, int waves) {
    constexpr int U = 5;
    const int G = p.K / kGroupK, lane = threadIdx.x & 63, sub = lane & 15, end = min(rows.rows, (block + 1) * kGatherRows);
    for (int at = block * kGatherRows + (int)(threadIdx.x >> 6); at < end; at += waves) {
        const int row = rows.order[at], a = rows.of[row];
        if (lane == 0) p.adapters[at] = (unsigned)a < (unsigned)rows.count ? a : -1;
        for (int g0 = lane >> 4; g0 < G; g0 += 4 * U) {
            u32x4 v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) v[u] = *reinterpret_cast<const u32x4 *>(p.x + (size_t)row * p.K + (size_t)min(g0 + 4 * u, G - 1) * kGroupK + sub * 8);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int g = g0 + 4 * u;
                float sum = sum_bf16x8(v[u]);
#pragma unroll
                for (int off = 8; off >= 1; off >>= 1) sum += __shfl_xor(sum, off, 16);
                if (g >= G) break;
                *reinterpret_cast<u32x4 *>(p.ordered + (size_t)at * p.K + (size_t)g * kGroupK + sub * 8) = v[u];
                if (sub == 0) store_row_sum(reinterpret_cast<u32x4 *>(p.sums), (size_t)g * rows.rows + at, sum, true);
            }
        }
    }
}

// s_a T, its slices summed, as the product takes it: eight of the rank to a thread, two bf16 parts in place of the first slice's f32.
__global__ __launch_bounds__(64) void bank_split_kernel(float *__restrict__ t, const float *__restrict__ scales, const int *__restrict__ adapters, int rows, int rank,
                                                        int slices) {
    const size_t unit = (size_t)blockIdx.x * 64 + threadIdx.x, stride = (size_t)rows * rank;
    const int per_row = rank / 8;
    if (unit >= (size_t)rows * per_row) return;
    const int a = adapters[unit / per_row];
    float *at = t + unit * 8;
    f32x4 v[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
    for (int s = 0; s < slices; s += 2) {
        f32x4 d[2][2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 2; ++i) d[u][i] = *reinterpret_cast<const f32x4 *>(at + min(s + u, slices - 1) * stride + 4 * i);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < 2; ++u)
            if (s + u < slices)
#pragma unroll
                for (int i = 0; i < 2; ++i) v[i] += d[u][i];
    }
    if (a < 0) return;
    const float scale = scales[a];
    bf16x8 hi, lo;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float f = v[i >> 2][i & 3] * scale;
        hi[i] = (__bf16)f;
        lo[i] = lower_part(f, hi[i]);
    }
    reinterpret_cast<bf16x8 *>(at)[0] = hi;
    reinterpret_cast<bf16x8 *>(at)[1] = lo;
}

// U pieces of a projection's contraction, 64 long each and 256 apart, all their loads in front of their products.  A lane's part of a
// piece is 16 values side by side, the first eight for one product and the rest for the next (which values meet in a product does not
// matter), so that four lanes read a row's 128 bytes together.
template <int JT, int RT, int W, int U>
__device__ __forceinline__ void project_pieces(const uint16_t *const (&x)[RT], const uint16_t *const (&m)[JT], int at, f32x4 (&acc)[RT][JT]) {
    bf16x8 xv[U][RT][2], b[U][JT][2];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < RT; ++i) xv[u][i][h] = load_bf16x8(x[i] + at + 64 * W * u + 8 * h);
#pragma unroll
            for (int j = 0; j < JT; ++j) b[u][j][h] = load_bf16x8(m[j] + at + 64 * W * u + 8 * h);
        }
    __builtin_amdgcn_sched_barrier(0);  // left alone, the compiler has eight loads in flight at a time
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int j = 0; j < JT; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xv[u][i][h], b[u][j][h], acc[i][j], 0, 0, 0);
}

// T: a block takes 16 RT positions, one slice of K, and of the adapters present among them those whose turn (in the order they are met)
// is blockIdx.y modulo gridDim.y.  Its W wavefronts take every W-th 64 of K and meet in LDS.  Blocks go through the slices first, so
// that with eight of them a die's blocks share one, whose part of the adapters' matrices its L2 then holds.  Two projections of the same
// rows share a launch: the second one's slices are behind the first one's.
template <int JT, int RT, int W>
__global__ __launch_bounds__(W * 64) void bank_project_kernel(BankProjection one, BankProjection two, BankRows rows, int rank, BankGather gather) {
    constexpr int P = 16 * RT, kAhead = JT + RT <= 4 ? 4 : 2;
    const int all = one.slices + two.slices, place = blockIdx.x % all, tile = blockIdx.x / all;
    if (tile * P >= rows.rows) {  // behind the projection's blocks
        if (blockIdx.y == 0) gather_rows(gather, rows, blockIdx.x - (rows.rows + P - 1) / P * all, W);
        return;
    }
    const bool second = place >= one.slices;
    const uint16_t *__restrict__ src = (const uint16_t *)(second ? two.src : one.src), *__restrict__ mat = (const uint16_t *)(second ? two.mat : one.mat);
    float *__restrict__ t = second ? two.t : one.t;
    const int K = second ? two.K : one.K, slices = second ? two.slices : one.slices, slice = second ? place - one.slices : place;
    const int steps = (K / 128 + slices - 1) / slices;
    __shared__ float part[W][P][JT * 16 + 4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 15, q = lane >> 4;
    const int p0 = tile * P;
    int row, a;
    row_at(rows, p0 + (lane & (P - 1)), row, a);
    constexpr unsigned long long kAll = P == 64 ? ~0ull : (1ull << P) - 1;
    unsigned long long left = __ballot(a >= 0) & kAll;
    const int k0 = slice * steps * 128, k1 = min(K, k0 + steps * 128), own = k0 + 64 * wave;
    const int pieces = own < k1 ? (k1 - own + 64 * W - 1) / (64 * W) : 0;
    const uint16_t *x[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) x[i] = src + (size_t)max(__shfl(row, 16 * i + c), 0) * K + own + 16 * q;
    for (unsigned turn = 0; left; ++turn) {
        const int cur = __builtin_amdgcn_readlane(a, __builtin_ctzll(left));
        const unsigned long long mine = __ballot(a == cur) & kAll;
        left &= ~mine;
        if (turn % gridDim.y != blockIdx.y) continue;
        const uint16_t *m[JT];  // rows past the rank: the last one again, their sums are dropped
#pragma unroll
        for (int j = 0; j < JT; ++j) m[j] = mat + ((size_t)cur * rank + min(16 * j + c, rank - 1)) * K + own + 16 * q;
        f32x4 acc[RT][JT] = {};
        int s = 0;
        for (; s + kAhead <= pieces; s += kAhead) project_pieces<JT, RT, W, kAhead>(x, m, 64 * W * s, acc);
        if (kAhead > 2 && s + 2 <= pieces) {
            project_pieces<JT, RT, W, 2>(x, m, 64 * W * s, acc);
            s += 2;
        }
        if (s < pieces) project_pieces<JT, RT, W, 1>(x, m, 64 * W * s, acc);
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int j = 0; j < JT; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) part[wave][16 * r + 4 * q + i][16 * j + c] = acc[r][j][i];
        __syncthreads();
        float *out = t + ((size_t)slice * rows.rows + p0) * rank;
        for (int e = tid; e < P * rank; e += 64 * W) {
            const int r = e / rank, j = e - r * rank;
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) v += part[w][r][j];
            if (mine >> r & 1) out[e] = v;
        }
        __syncthreads();
    }
}

// eight columns of y to the accumulators of two tiles, and back
__device__ __forceinline__ void take_columns(u32x4 v, f32x4 &even, f32x4 &odd) {
    even = f32x4{__builtin_bit_cast(float, v.x << 16), __builtin_bit_cast(float, v.x & 0xFFFF0000u), __builtin_bit_cast(float, v.y << 16),
                 __builtin_bit_cast(float, v.y & 0xFFFF0000u)};
    odd = f32x4{__builtin_bit_cast(float, v.z << 16), __builtin_bit_cast(float, v.z & 0xFFFF0000u), __builtin_bit_cast(float, v.w << 16),
                __builtin_bit_cast(float, v.w & 0xFFFF0000u)};
}
__device__ __forceinline__ u32x4 give_columns(const f32x4 &even, const f32x4 &odd) {
    auto pair = [](float lo, float hi) { return f32_to_bf16_bits(lo) | (uint32_t)f32_to_bf16_bits(hi) << 16; };
    return u32x4{pair(even[0], even[1]), pair(even[2], even[3]), pair(odd[0], odd[1]), pair(odd[2], odd[3])};
}
// Rows as they stand: 16 of them x 64 columns to a block, the adapters met dealt out to its four wavefronts, each of which takes the
// rows of its own: nothing to add up, and with an adapter per row (a decode step) the loads of four adapters' rows of B go out together.
// Bound by those loads' latency: 16 rows of 16 adapters, 18432 columns, rank 16, 6.4 us (27 with the adapters one after the other).
template <int S>
__global__ __launch_bounds__(256) void bank_expand_kernel(uint16_t *__restrict__ y, const uint16_t *__restrict__ mat, const float *__restrict__ t,
                                                          const float *__restrict__ scales, BankRows rows, int N, int rank, int slices) {
    constexpr int kTogether = S == 1 ? 4 : 2;
    __shared__ __align__(16) float ts[16][kBankMaxRank + 4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 15, q = lane >> 4;
    const int p0 = blockIdx.y * kBankRowTile, n0 = blockIdx.x * 64;
    int row, a;
    row_at(rows, p0 + c, row, a);
    unsigned left = (unsigned)__ballot(a >= 0) & 0xFFFFu;
    if (!left) return;
    int mine[4] = {0, 0, 0, 0}, count = 0;  // the adapters of this wavefront
    bool live = false;
    for (int turn = 0; left; ++turn) {
        const int cur = __builtin_amdgcn_readlane(a, __builtin_ctz(left));
        left &= ~((unsigned)__ballot(a == cur) & 0xFFFFu);
        if ((turn & 3) != wave) continue;
        if (count == 0) mine[0] = cur;
        else if (count == 1) mine[1] = cur;
        else if (count == 2) mine[2] = cur;
        else mine[3] = cur;
        ++count;
        live |= a == cur;
    }
    const float scale = live ? scales[a] : 0.f;
    uint16_t *dst = y + (size_t)max(row, 0) * N + n0 + 8 * q;
    u32x4 was[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) was[i] = *reinterpret_cast<const u32x4 *>(dst + 32 * i);
    f32x4 acc[4];
    ExpandRow<S> tv;
#pragma unroll
    for (int first = 0; first < 4; first += kTogether) {
        bf16x8 b[kTogether][4][S];
#pragma unroll
        for (int g = 0; g < kTogether; ++g) {
            if (first + g >= count) break;
            expand_rows<S, 4>(mat + ((size_t)mine[first + g] * N + n0) * rank, c, q, rank, b[g]);
        }
        if (first == 0) {
            sum_projected<16>(t, rows, p0, rank, slices, tid, 256, ts);
            tv.set(ts[c], scale, live, q, rank);
#pragma unroll
            for (int i = 0; i < 2; ++i) take_columns(was[i], acc[2 * i], acc[2 * i + 1]);
        }
#pragma unroll
        for (int g = 0; g < kTogether; ++g) {
            if (first + g >= count) break;
            expand_product<S, 4>(b[g], tv, a == mine[first + g], acc);
        }
    }
    if (live)
#pragma unroll
        for (int i = 0; i < 2; ++i) *reinterpret_cast<u32x4 *>(dst + 32 * i) = give_columns(acc[2 * i], acc[2 * i + 1]);
}

// Rows in the order of their adapters: 64 positions x `columns` columns to a block, 64 at a time to each wavefront, so that a wavefront's
// rows of B serve four tiles of rows; T is read and split once, y of the next columns on its way meanwhile.  Bound by y, read and written:
// 2048 rows of 18432 columns, rank 32, 45 us behind the GEMM that wrote them, 3.4 TB/s (with 16 positions to a wavefront, 128 columns at a time, the same).
template <int S>
__global__ __launch_bounds__(256) void bank_expand_ordered_kernel(uint16_t *__restrict__ y, const uint16_t *__restrict__ mat,
                                                                  const float *__restrict__ t, const float *__restrict__ scales, BankRows rows,
                                                                  int N, int rank, int slices, int columns) {
    __shared__ __align__(16) float ts[64][kBankMaxRank + 4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 15, q = lane >> 4;
    const int parts = (N + columns - 1) / columns, part = blockIdx.x % parts, p0 = blockIdx.x / parts * 64;
    int row, a;
    row_at(rows, p0 + lane, row, a);
    const unsigned long long present = __ballot(a >= 0);
    if (!present) return;
    const float scale = a >= 0 ? scales[a] : 0.f;
    const int end = min(N, (part + 1) * columns);
    int n0 = part * columns + 64 * wave;
    int a_of[4];
    uint16_t *dst[4];
    u32x4 was[4][2];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        a_of[r] = __shfl(a, 16 * r + c);
        dst[r] = y + (size_t)max(__shfl(row, 16 * r + c), 0) * N + 8 * q;
#pragma unroll
        for (int i = 0; i < 2; ++i) was[r][i] = *reinterpret_cast<const u32x4 *>(dst[r] + min(n0, end - 64) + 32 * i);
    }
    sum_projected<64>(t, rows, p0, rank, slices, tid, 256, ts);
    ExpandRow<S> tv[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) tv[r].set(ts[16 * r + c], __shfl(scale, 16 * r + c), a_of[r] >= 0, q, rank);
    for (; n0 < end; n0 += 256) {
        f32x4 acc[4][4];
        bool taken = false;
        for (unsigned long long left = present; left;) {
            const int cur = __builtin_amdgcn_readlane(a, __builtin_ctzll(left));
            const unsigned long long mine = __ballot(a == cur);
            left &= ~mine;
            bf16x8 b[4][S];
            expand_rows<S, 4>(mat + ((size_t)cur * N + n0) * rank, c, q, rank, b);
            __builtin_amdgcn_sched_barrier(0);
            if (!taken)
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        take_columns(was[r][i], acc[r][2 * i], acc[r][2 * i + 1]);
                        was[r][i] = *reinterpret_cast<const u32x4 *>(dst[r] + min(n0 + 256, end - 64) + 32 * i);
                    }
            taken = true;
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (mine >> (16 * r) & 0xFFFFu) expand_product<S, 4>(b, tv[r], a_of[r] == cur, acc[r]);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (a_of[r] >= 0)
#pragma unroll
                for (int i = 0; i < 2; ++i) *reinterpret_cast<u32x4 *>(dst[r] + n0 + 32 * i) = give_columns(acc[r][2 * i], acc[r][2 * i + 1]);
    }
}

int tiles_of(int rows, int tile) { return (rows + tile - 1) / tile; }

// Rows in order and a long contraction: 32 positions to a block, which the adapters' matrices are read for once, and eight slices (2048
// rows of K 18432 and rank 32: 33 us, 37 with 64 positions).  A short one has too few such blocks: 16 positions, eight wavefronts and
// slices of 1536 at most (K 2560, by itself: 6.9 us with 32 positions and five slices, 6.2).
constexpr int kLongContraction = 8192;
bool long_ordered(int rows, int K) { return rows >= kBankOrderedFrom && K >= kLongContraction; }

template <int JT, int RT, int W>
void launch_project(const BankProjection &one, const BankProjection &two, const BankRows &r, int rank, hipStream_t stream, const BankGather &gather) {
    const int tiles = tiles_of(r.rows, 16 * RT);
    // the adapters that a tile may hold side by side: as many as it has rows, but where they are together few tiles have more than one
    int turns = r.order ? 1 + r.count / tiles : 16;
    if (turns > 16) turns = 16;
    if (turns > r.count) turns = r.count;
    bank_project_kernel<JT, RT, W><<<dim3((one.slices + two.slices) * tiles + gather.blocks, turns), W * 64, 0, stream>>>(one, two, r, rank, gather);
}
template <int RT, int W>
void launch_project(const BankProjection &one, const BankProjection &two, const BankRows &r, int rank, hipStream_t stream, const BankGather &gather) {
    const int jt = (rank + 15) / 16;
    if (jt == 1) launch_project<1, RT, W>(one, two, r, rank, stream, gather);
    else if (jt == 2) launch_project<2, RT, W>(one, two, r, rank, stream, gather);
    else if (jt == 3) launch_project<3, RT, W>(one, two, r, rank, stream, gather);
    else launch_project<4, RT, W>(one, two, r, rank, stream, gather);
}

// Up to 16 rows: may the base product be the one with the projection beside it (bank_base)?  It saves a launch; the plain GEMM is the faster
// product of many rows of a long K.  1 / 8 / 16 rows of as many adapters, rank 16, us, against the plain GEMM with the projection behind it:
// 2560 -> 10240 8.2 / 10.2 / 13.1 against 11.4 / 13.6 / 16.0, 2560 -> 18432 9.6 / 12.9 / 15.6 against 12.5 / 15.4 / 18.7, 4096 -> 14336
// 10.3 / 12.0 / 14.6 against 14.0 / 16.0 / 18.9, 5120 -> 27648 17.5 / 24.8 / 29.8 against 22.9 / 26.6 / 30.9; but 9216 -> 2560 10.3 / 17.1 / 22.2 against
// 13.1 / 15.5 / 17.7.
bool takes_base(int m, int n, int k) { return m <= kBankFewRows && (k <= 5120 || m <= 4); }

}  // namespace

bool bank_ok(const kiln_w4a16_adapter_bank &bank) {
    return bank.count >= 1 && bank.count <= 4096 && bank.rank >= 8 && bank.rank <= kBankMaxRank && bank.rank % 8 == 0;
}

static size_t bank_ordered_x_bytes(int rows, int K) { return bank_up256((size_t)rows * K * 2); }

size_t bank_order_bytes(int rows, int count) { return bank_up256((size_t)rows * 4) + bank_up256(((size_t)count + 2) * 4); }

BankRows bank_rows(const int *of, int rows, int count, void *at) {
    return BankRows{of, reinterpret_cast<int *>(at), reinterpret_cast<int *>(reinterpret_cast<char *>(at) + bank_up256((size_t)rows * 4)), rows, count};
}

// Slices are 512 of K at least: two pieces to a wavefront, whose loads are in flight together; shorter ones leave whoever sums them more
// to read (16 rows of K 2560: 20 slices instead of 5 cost the next launch 20 KB a block).
int bank_slices(int rows, int K) {
    const int groups = K / 128;
    int slices;
    if (rows < kBankOrderedFrom) slices = (groups + 3) / 4 < kBankMaxSlices ? (groups + 3) / 4 : kBankMaxSlices;
    else slices = long_ordered(rows, K) ? 8 : (groups + 11) / 12;
    return bank_level_slices(groups, slices);
}

// slices * rows <= this for the slices of every plan (bank_plan), and it does not fall with `rows`
size_t bank_projected_rows(int rows, int K) {
    const int as_they_stand = bank_slices(1, K) > bank_base_slices(K) ? bank_slices(1, K) : bank_base_slices(K);
    const size_t below = (size_t)(rows < kBankOrderedFrom ? rows : kBankOrderedFrom) * as_they_stand;
    const size_t here = (size_t)rows * bank_slices(rows, K);
    return here > below ? here : below;
}

// (2048 rows of rank 32, 8 adapters, 2560 -> 18432: 186 us a call with the term in the product against 215 behind it, 4096 -> 14336 222 against 244; on
// narrow outputs the rows' copy costs what it saves: 4096 rows 14336 -> 4096 459 against 449)
BankPlan bank_plan(int m, int n, int k, int rank, int cus) {
    if (bank_projects_itself(m, n, k, rank)) return {BankMethod::kOneLaunch, 0};
    if (takes_base(m, n, k)) return {BankMethod::kBase, bank_base_slices(k)};
    const bool inside = m >= kBankOrderedFrom && n >= k && bank_in_product(m, n, k, cus);
    return {inside ? BankMethod::kInProduct : BankMethod::kBehind, bank_slices(m, k)};
}

void bank_project(const BankProjection &one, const BankProjection *two, const BankRows &r, int rank, hipStream_t stream, BankGather gather) {
    const BankProjection none{}, &other = two ? *two : none;
    if (!r.order || r.rows < kBankOrderedFrom) launch_project<1, 4>(one, other, r, rank, stream, gather);
    else if (two || long_ordered(r.rows, one.K)) launch_project<2, 4>(one, other, r, rank, stream, gather);
    else launch_project<1, 8>(one, other, r, rank, stream, gather);
}

namespace {

template <int S>
void launch_expand(uint16_t *y, const uint16_t *m, const float *t, const float *scales, const BankRows &r, int N, int rank, int slices, int cus,
                   hipStream_t stream) {
    if (!r.order) {
        bank_expand_kernel<S><<<dim3(N / 64, tiles_of(r.rows, 16)), 256, 0, stream>>>(y, m, t, scales, r, N, rank, slices);
        return;
    }
    const int tiles = tiles_of(r.rows, 64);
    int columns = 1024;  // (2048 rows of 18432 columns: 256 60 us, 512 49, 1024 45, 2048 50)
    while (columns > 256 && tiles * ((N + columns - 1) / columns) < 2 * cus) columns /= 2;
    bank_expand_ordered_kernel<S><<<(N + columns - 1) / columns * tiles, 256, 0, stream>>>(y, m, t, scales, r, N, rank, slices, columns);
}

}  // namespace

}  // namespace kiln

using namespace kiln;

extern "C" {

size_t kiln_w4a16_gemm_bank_scratch_bytes(int prob_m, int prob_n, int prob_k, int count, int rank) {
    if (prob_m < 1 || prob_n < 1 || prob_k < 128 || count < 1 || rank < 1) return 256;
    const size_t ordered = prob_m < kBankOrderedFrom ? 0 : bank_ordered_x_bytes(prob_m, prob_k) + (size_t)prob_m * (prob_k / 128 + 1) * 4;
    return bank_order_bytes(prob_m, count) + bank_up256(bank_projected_rows(prob_m, prob_k) * rank * 4) + ordered;
}

int kiln_w4a16_debug_bank_plan(int prob_m, int prob_n, int prob_k, int rank, int cus, int *out) {
    if (prob_m < 1 || prob_n < 256 || prob_n % 256 != 0 || prob_k < 128 || prob_k % 128 != 0 || rank < 8 || rank > kBankMaxRank || rank % 8 != 0 || cus < 1) return 1;
    const BankPlan plan = bank_plan(prob_m, prob_n, prob_k, rank, cus);
    out[0] = static_cast<int>(plan.method);
    out[1] = plan.slices;
    return 0;
}

kiln_marlin_status_t kiln_w4a16_gemm_bank(const void *A, const void *B, void *C, const void *s, int prob_m, int prob_n, int prob_k,
                                          void *workspace, int groupsize, int dev, void *stream, const kiln_w4a16_adapter_bank *bank,
                                          const int *adapter_of, void *scratch) {
    if (prob_m < 0 || prob_n < 0 || prob_k < 0) return KILN_W4A16_ERR_PROB_SHAPE;
    if (prob_m == 0 || prob_n == 0 || prob_k == 0)
        return kiln_marlin_w4a16_gemm(A, B, C, const_cast<void *>(s), prob_m, prob_n, prob_k, workspace, groupsize, dev, stream, -1, -1, -1, 16);
    if (!bank || !adapter_of || !scratch) return KILN_W4A16_ERR_ARGUMENT;
    if (!bank_ok(*bank)) return KILN_W4A16_ERR_KERN_SHAPE;
    if (prob_n % 256 != 0 || prob_k % 128 != 0 || (groupsize != -1 && groupsize != 128)) return KILN_W4A16_ERR_PROB_SHAPE;
    if (!A || !B || !C || !s || !workspace || !bank->lora_a || !bank->lora_b || !bank->scales) return KILN_W4A16_ERR_ARGUMENT;
    for (const void *p : {A, B, static_cast<const void *>(C), s, static_cast<const void *>(workspace), bank->lora_a, bank->lora_b,
                          static_cast<const void *>(scratch)})
        if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return KILN_W4A16_ERR_ARGUMENT;
    const size_t adapters = (size_t)bank->count * bank->rank * 2;
    if (meet(C, (size_t)prob_m * prob_n * 2, A, (size_t)prob_m * prob_k * 2) || meet(C, (size_t)prob_m * prob_n * 2, bank->lora_a, adapters * prob_k) ||
        meet(C, (size_t)prob_m * prob_n * 2, bank->lora_b, adapters * prob_n))
        return KILN_W4A16_ERR_ARGUMENT;
    hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
    char *at = reinterpret_cast<char *>(scratch);
    BankRows rows = bank_rows(adapter_of, prob_m, bank->count, at);
    float *t = reinterpret_cast<float *>(at + bank_order_bytes(prob_m, bank->count));
    const int rank = bank->rank;
    const int cus = compute_units(dev);
    const BankPlan plan = bank_plan(prob_m, prob_n, prob_k, rank, cus);
    if (plan.method == BankMethod::kOneLaunch) {
        rows.order = rows.first = nullptr;
        bank_few(A, B, s, C, *bank, rows, prob_k, prob_n, groupsize == -1, hs);
        return hipGetLastError() == hipSuccess ? KILN_W4A16_OK : KILN_W4A16_ERR_LAUNCH;
    }
    const int slices = plan.slices;
    const BankProjection of_x{A, bank->lora_a, t, prob_k, slices};
    if (plan.method == BankMethod::kInProduct) {
        char *ordered = at + bank_order_bytes(prob_m, bank->count) + bank_up256(bank_projected_rows(prob_m, prob_k) * rank * 4);
        float *sums = reinterpret_cast<float *>(ordered + bank_ordered_x_bytes(prob_m, prob_k));
        bank_order_kernel<<<bank->count + 1, kOrderWaves * 64, 0, hs>>>(adapter_of, rows.order, rows.first, prob_m, bank->count);
        int *adapters = reinterpret_cast<int *>(sums + (size_t)prob_m * (prob_k / 128));
        bank_project(of_x, nullptr, rows, rank, hs,
                     BankGather{(const uint16_t *)A, (uint16_t *)ordered, sums, adapters, prob_k, (prob_m + kGatherRows - 1) / kGatherRows});
        bank_split_kernel<<<(unsigned)(((size_t)prob_m * (rank / 8) + 63) / 64), 64, 0, hs>>>(t, bank->scales, adapters, prob_m, rank, slices);
        const PrefillBank term{(const uint16_t *)bank->lora_b, (const uint16_t *)t, rows.order, adapters, rank};
        return gemm_with_bank(ordered, B, C, s, prob_m, prob_n, prob_k, workspace, groupsize, dev, stream, sums, term);
    }
    if (plan.method == BankMethod::kBase) {
        rows.order = rows.first = nullptr;
        bank_base(A, B, s, C, of_x, rows, rank, prob_k, prob_n, groupsize == -1, cus, hs);
    } else {
        // the plain GEMM's checks and its launches first: nothing is launched for a call that it refuses
        const kiln_marlin_status_t st =
            kiln_marlin_w4a16_gemm(A, B, C, const_cast<void *>(s), prob_m, prob_n, prob_k, workspace, groupsize, dev, stream, -1, -1, -1, 16);
        if (st != KILN_W4A16_OK) return st;
        if (prob_m < kBankOrderedFrom) rows.order = rows.first = nullptr;
        else bank_order_kernel<<<bank->count + 1, kOrderWaves * 64, 0, hs>>>(adapter_of, rows.order, rows.first, prob_m, bank->count);
        bank_project(of_x, nullptr, rows, rank, hs);
    }
    uint16_t *y = (uint16_t *)C;
    const uint16_t *m = (const uint16_t *)bank->lora_b;
    if (rank <= 32) launch_expand<1>(y, m, t, bank->scales, rows, prob_n, rank, slices, cus, hs);
    else launch_expand<2>(y, m, t, bank->scales, rows, prob_n, rank, slices, cus, hs);
    return hipGetLastError() == hipSuccess ? KILN_W4A16_OK : KILN_W4A16_ERR_LAUNCH;
}

}  // extern "C"
