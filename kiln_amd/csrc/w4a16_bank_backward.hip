// The gradients of a packed projection, with or without a bank of adapters (w4a16_bank.hip), the packed weight itself frozen:
//   dx[i]  = dy[i] W^T + s_a (dy[i] B_a) A_a            a = adapter_of[i]
//   dA_a   = s_a sum_{i of a} (dy[i] B_a)^T x[i]
//   dB_a   = s_a sum_{i of a} dy[i]^T (x[i] A_a^T)
// The reference trains adapters over a frozen base (crates/kiln-model/src/lora_loader.rs:213-232 is the forward it differentiates).
//
// Steps: W as bf16 with its columns contiguous (what a product over the columns reads), the adapters' matrices transposed, T = x A^T and
// U = dy B in f32, then dx as one matrix product into which U A goes as further steps of the contraction, and dA, dB as sums over the
// rows of an adapter.  Rows are taken in the order of their adapters throughout.
#include "async_loads.h"
#include "bank.h"
#include "device_common.h"

namespace kiln {
namespace {

// ---- W, row by row ---------------------------------------------------------------------------------------------
// out[k][n] = bf16((code - 8) * scale): a block takes one scale group (128 rows) x 128 columns, a chunk to each of its eight
// wavefronts, and turns it through LDS.  The rounding of a weight to 8 bits is what every 16-bit product of the unpacked weight has
// (the reference's own bar is against bf16(dequant): crates/kiln-marlin-gemm/tests/parity.rs:150-157); the codes themselves would be exact,
// but the scales run along the contraction here and cannot be pulled out of it.
constexpr int kTurnPitch = 128 + 8;
__global__ __launch_bounds__(512) void dequant_rows_kernel(const u32x4 *__restrict__ B, const uint16_t *__restrict__ S, uint16_t *__restrict__ out, int K,
                                                           int N, int Gs) {
    __shared__ __align__(16) uint16_t tile[128 * kTurnPitch];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 15, kq = lane >> 4;
    const int G = K / kGroupK, g = blockIdx.y, nt = blockIdx.x * 8 + wave;
    const u32x4 w = B[((size_t)nt * G + g) * 64 + lane];
    const float s = f16_bits_to_f32(S[scale_index(Gs == 1 ? 0 : g, nt * kTileN + c, Gs)]);
    const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int code = (words[t] >> (4 * nibble_pos(j))) & 0xF;
            tile[(32 * t + 8 * kq + j) * kTurnPitch + 16 * wave + c] = f32_to_bf16_bits((float)(code - 8) * s);
        }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = 32 * i + (tid >> 4), at = 8 * (tid & 15);
        *reinterpret_cast<u32x4 *>(out + (size_t)(g * kGroupK + row) * N + blockIdx.x * 128 + at) =
            *reinterpret_cast<const u32x4 *>(tile + row * kTurnPitch + at);
    }
}

// ---- the adapters' matrices turned -------------------------------------------------------------------------------
// z = 0: at[a][k][rank] of a[a][rank][k]; z = 1: bt[a][rank][n] of b[a][n][rank]; 64 of k or n to a block
__global__ __launch_bounds__(256) void turn_bank_kernel(const uint16_t *__restrict__ a, const uint16_t *__restrict__ b, uint16_t *__restrict__ at,
                                                        uint16_t *__restrict__ bt, int K, int N, int rank) {
    __shared__ uint16_t tile[64][kBankMaxRank + 2];
    const int tid = threadIdx.x, which = blockIdx.z, len = which ? N : K, l0 = blockIdx.x * 64;
    if (l0 >= len) return;
    const size_t base = (size_t)blockIdx.y * rank * len;
    if (which == 0) {
        for (int e = tid; e < rank * 64; e += 256) tile[e & 63][e >> 6] = a[base + (size_t)(e >> 6) * len + l0 + (e & 63)];
        __syncthreads();
        for (int e = tid; e < 64 * rank; e += 256) at[base + (size_t)l0 * rank + e] = tile[e / rank][e % rank];
    } else {
        for (int e = tid; e < 64 * rank; e += 256) tile[e / rank][e % rank] = b[base + (size_t)l0 * rank + e];
        __syncthreads();
        for (int e = tid; e < rank * 64; e += 256) bt[base + (size_t)(e >> 6) * len + l0 + (e & 63)] = tile[e & 63][e >> 6];
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
// dx[row][k] = sum_n dy[row][n] W[k][n] (+ s U A), both operands with the contraction contiguous.  A block of four wavefronts takes
// 64 TM rows x 64 TN of k, 64 of the contraction at a time: both tiles go straight to LDS, one in flight while the other is
// multiplied.  A row of a tile is eight 16-byte units, unit u at place u ^ (row & 7), so that the eight lanes that LDS serves
// together find their units in different banks.
struct DxArgs {
    const uint16_t *dy, *wt, *at;   // [rows, N], [K, N], [count, K, rank]
    const float *u, *scales;        // [rows by position, rank], or null without a bank
    uint16_t *dx;
    float *partial;                 // [slices, rows, K], or null with one slice
    BankRows rows;
    int K, N, rank, steps;          // steps of 64 of the contraction to a slice
};

__device__ __forceinline__ unsigned unit_at(int row, int unit) { return (unsigned)(row * 8 + (unit ^ (row & 7))) * 16; }

template <int TM, int TN>
__device__ __forceinline__ void dx_product(const char *lds, int wm, int wn, int lane, f32x16 (&acc)[TN][TM]) {
    constexpr int BM = 64 * TM;
    const int r = lane & 31, h = lane >> 5;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
        bf16x8 x[TM], w[TN];
#pragma unroll
        for (int i = 0; i < TM; ++i) x[i] = *reinterpret_cast<const bf16x8 *>(lds + unit_at(32 * (TM * wm + i) + r, 2 * kk + h));
#pragma unroll
        for (int j = 0; j < TN; ++j) w[j] = *reinterpret_cast<const bf16x8 *>(lds + BM * 128 + unit_at(32 * (TN * wn + j) + r, 2 * kk + h));
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int i = 0; i < TM; ++i) acc[j][i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w[j], x[i], acc[j][i], 0, 0, 0);
    }
}

template <int TM, int TN>
__global__ __launch_bounds__(256) void bank_dx_kernel(DxArgs p) {
    constexpr int BM = 64 * TM, BN = 64 * TN, kStage = (BM + BN) * 128;
    extern __shared__ __align__(16) char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave & 1, wn = wave >> 1;
    const int k0 = blockIdx.x * BN, p0 = blockIdx.y * BM;
    const int first = blockIdx.z * p.steps, last = min(p.N / 64, first + p.steps);
    // this lane's part of a stage: rows 8 (i + TM.. * wave) + lane / 8 of either tile
    const uint16_t *xs[2 * TM], *ws[2 * TN];
    const int unit = (lane & 7) ^ (lane >> 3);
#pragma unroll
    for (int i = 0; i < 2 * TM; ++i) {
        const int at = min(p0 + 8 * (2 * TM * wave + i) + (lane >> 3), p.rows.rows - 1);
        xs[i] = p.dy + (size_t)(p.rows.order ? p.rows.order[at] : at) * p.N + 8 * unit;
    }
#pragma unroll
    for (int i = 0; i < 2 * TN; ++i) ws[i] = p.wt + (size_t)min(k0 + 8 * (2 * TN * wave + i) + (lane >> 3), p.K - 1) * p.N + 8 * unit;
    const unsigned lds0 = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(lds_ptr_t)lds);
    auto fetch = [&](int step, int buffer) {
        const unsigned at = lds0 + buffer * kStage + wave * (TM * 2048);
#pragma unroll
        for (int i = 0; i < 2 * TM; ++i) load_to_lds_b128(xs[i] + (size_t)step * 64, at + i * 1024);
        const unsigned bt = lds0 + buffer * kStage + BM * 128 + wave * (TN * 2048);
#pragma unroll
        for (int i = 0; i < 2 * TN; ++i) load_to_lds_b128(ws[i] + (size_t)step * 64, bt + i * 1024);
    };
    f32x16 acc[TN][TM];
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[j][i][e] = 0.f;
    fetch(first, 0);
    for (int step = first; step < last; ++step) {
        const int buffer = (step - first) & 1;
        wait_vector_loads<0>();
        __syncthreads();
        if (step + 1 < last) fetch(step + 1, buffer ^ 1);
        dx_product<TM, TN>(lds + buffer * kStage, wm, wn, lane, acc);
    }
    if (p.u && blockIdx.z == 0) {
        // U A: the runs of rows of one adapter among the block's positions, each as one step (rank <= 32: both parts of U side by
        // side on the 64 of the contraction) or two (U's bf16 value, then what that leaves)
        const int end = min(p0 + BM, p.rows.first[p.rows.count]);
        const int sides = p.rank <= 32 ? 1 : 2, half = p.rank <= 32 ? 32 : 64;
        for (int q0 = p0; q0 < end;) {
            const int a = p.rows.of[p.rows.order[q0]], q1 = min(p.rows.first[a + 1], end);
            const float scale = p.scales[a];
            for (int side = 0; side < sides; ++side) {
                __syncthreads();
                for (int e = tid; e < BM * 8; e += 256) {
                    const int row = e >> 3, unit = e & 7, col = (8 * unit) % half;
                    const bool lower = sides == 1 ? unit >= 4 : side == 1;
                    bf16x8 v = bf16x8_zero();
                    if (p0 + row >= q0 && p0 + row < q1 && col < p.rank) {
                        const float *u = p.u + (size_t)(p0 + row) * p.rank + col;
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float f = u[i] * scale;
                            const __bf16 hi = (__bf16)f;
                            v[i] = lower ? (__bf16)(f - (float)hi) : hi;
                        }
                    }
                    *reinterpret_cast<bf16x8 *>(lds + unit_at(row, unit)) = v;
                }
                for (int e = tid; e < BN * 8; e += 256) {
                    const int row = e >> 3, unit = e & 7, col = (8 * unit) % half;
                    u32x4 v = {0u, 0u, 0u, 0u};
                    if (k0 + row < p.K && col < p.rank) v = *reinterpret_cast<const u32x4 *>(p.at + ((size_t)a * p.K + k0 + row) * p.rank + col);
                    *reinterpret_cast<u32x4 *>(lds + BM * 128 + unit_at(row, unit)) = v;
                }
                __syncthreads();
                dx_product<TM, TN>(lds, wm, wn, lane, acc);
            }
            q0 = q1;
        }
    }
    // a lane holds column lane & 31 (a row of dx) and four consecutive k at 8 g + 4 (lane >> 5)
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const int at = p0 + 32 * (TM * wm + i) + (lane & 31);
        if (at >= p.rows.rows) continue;
        const int row = p.rows.order ? p.rows.order[at] : at;
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int k = k0 + 32 * (TN * wn + j) + 8 * g + 4 * (lane >> 5);
                if (k >= p.K) continue;
                const f32x16 &v = acc[j][i];
                if (p.partial) {
                    *reinterpret_cast<f32x4 *>(p.partial + ((size_t)blockIdx.z * p.rows.rows + row) * p.K + k) =
                        f32x4{v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]};
                } else {
                    u32x2 o;
                    o.x = f32_to_bf16_bits(v[4 * g]) | (uint32_t)f32_to_bf16_bits(v[4 * g + 1]) << 16;
                    o.y = f32_to_bf16_bits(v[4 * g + 2]) | (uint32_t)f32_to_bf16_bits(v[4 * g + 3]) << 16;
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
};

constexpr int kGradPitch = 128 + 4;
template <int JT, int W>
__global__ __launch_bounds__(W * 64) void bank_grad_kernel(GradArgs p) {
    __shared__ float sum[JT * 16 * kGradPitch];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 15, q = lane >> 4;
    const int a = blockIdx.y;
    const bool is_b = (int)blockIdx.x < p.N / 128;
    const int c0 = (is_b ? blockIdx.x : blockIdx.x - p.N / 128) * 128, len = is_b ? p.N : p.K;
    const uint16_t *src = (is_b ? p.dy : p.x) + c0 + 8 * c;
    const float *f = is_b ? p.t : p.u;
    const int begin = p.rows.first[a], end = p.rows.first[a + 1];
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
        for (int i = 0; i < 8; ++i) row[i] = p.rows.order[min(at + 8 * q + i, end - 1)];
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
            for (int j = 0; j < JT; ++j) w[j][i] = f[(size_t)min(at + 8 * q + i, end - 1) * p.rank + col[j]];
        rows_at(at + 32 * W);
        __builtin_amdgcn_sched_barrier(0);
        bf16x8 hi[JT], lo[JT];
#pragma unroll
        for (int j = 0; j < JT; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float x = at + 8 * q + i < end ? w[j][i] : 0.f;
                hi[j][i] = (__bf16)x;
                lo[j][i] = (__bf16)(x - (float)hi[j][i]);
            }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            u32x4 pairs;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                pairs[i] = __builtin_amdgcn_perm(v[2 * i + 1][e >> 1], v[2 * i][e >> 1], e & 1 ? 0x07060302u : 0x05040100u);
            const bf16x8 b = __builtin_bit_cast(bf16x8, pairs);
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
    const float scale = p.scales[a];
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
}

template <int JT>
void launch_grad(const GradArgs &g, hipStream_t stream) {
    const dim3 grid(g.N / 128 + g.K / 128, g.rows.count);
    if (grid.x * grid.y >= 512) bank_grad_kernel<JT, 4><<<grid, 256, 0, stream>>>(g);
    else bank_grad_kernel<JT, 8><<<grid, 512, 0, stream>>>(g);
}

// ---- the plan ----------------------------------------------------------------------------------------------------
constexpr int kMaxDxSlices = 8;
int dx_slices(int m, int n, int k) {
    const int tiles = ((m + 127) / 128) * (k / 128), steps = n / 64;
    int slices = 1;
    while (slices < kMaxDxSlices && tiles * slices < 384 && steps / (slices + 1) >= 4) ++slices;
    const int each = (steps + slices - 1) / slices;
    return (steps + each - 1) / each;
}

struct BackwardScratch {
    size_t wt, at, bt, order, t, u, partial, total;
    int t_slices, u_slices, dx_slices;
};
BackwardScratch backward_scratch(int m, int n, int k, int count, int rank) {
    BackwardScratch s{};
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += bank_up256(bytes);
        return here;
    };
    s.wt = take((size_t)k * n * 2);
    if (count > 0) {
        s.at = take((size_t)count * rank * k * 2);
        s.bt = take((size_t)count * rank * n * 2);
        s.order = take(bank_order_bytes(m, count));
        s.t_slices = bank_slices(m, k);
        s.u_slices = bank_slices(m, n);
        s.t = take((size_t)s.t_slices * m * rank * 4);
        s.u = take((size_t)s.u_slices * m * rank * 4);
    }
    s.dx_slices = dx_slices(m, n, k);
    s.partial = take(s.dx_slices > 1 ? (size_t)s.dx_slices * m * k * 4 : 0);
    s.total = at;
    return s;
}

constexpr int kTileM = 2, kTileK = 2;

}  // namespace
}  // namespace kiln

using namespace kiln;

extern "C" {

size_t kiln_w4a16_gemm_bank_backward_scratch_bytes(int prob_m, int prob_n, int prob_k, int count, int rank) {
    if (prob_m < 1 || prob_n < 256 || prob_k < 128 || count < 0 || rank < 0) return 256;
    return backward_scratch(prob_m, prob_n, prob_k, count, rank).total;
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
    hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
    const int m = prob_m, n = prob_n, k = prob_k, count = bank ? bank->count : 0, rank = bank ? bank->rank : 0;
    const BackwardScratch w = backward_scratch(m > 0 ? m : 1, n, k, count, rank);
    char *at = reinterpret_cast<char *>(scratch);
    uint16_t *wt = reinterpret_cast<uint16_t *>(at + w.wt);
    DxArgs dx{};
    dx.dy = (const uint16_t *)dC;
    dx.wt = wt;
    dx.dx = (uint16_t *)dA;
    dx.partial = w.dx_slices > 1 ? reinterpret_cast<float *>(at + w.partial) : nullptr;
    dx.rows = BankRows{nullptr, nullptr, nullptr, m, 0};
    dx.K = k;
    dx.N = n;
    dx.steps = (n / 64 + w.dx_slices - 1) / w.dx_slices;
    if (bank) {
        uint16_t *a_t = reinterpret_cast<uint16_t *>(at + w.at), *b_t = reinterpret_cast<uint16_t *>(at + w.bt);
        float *t = reinterpret_cast<float *>(at + w.t), *u = reinterpret_cast<float *>(at + w.u);
        dx.rows = bank_order(adapter_of, m, count, true, at + w.order, hs);
        if (m > 0) {
            turn_bank_kernel<<<dim3((k > n ? k : n) / 64, count, 2), 256, 0, hs>>>((const uint16_t *)bank->lora_a, (const uint16_t *)bank->lora_b, a_t, b_t, k, n, rank);
            bank_project(A, bank->lora_a, dx.rows, t, k, rank, w.t_slices, hs);
            bank_project(dC, b_t, dx.rows, u, n, rank, w.u_slices, hs);
            if (w.t_slices > 1 || w.u_slices > 1)
                sum_slices_kernel<<<dim3((unsigned)(((size_t)m * rank + 255) / 256), 2), 256, 0, hs>>>(t, w.t_slices, u, w.u_slices, (size_t)m * rank);
        }
        GradArgs g{(const uint16_t *)A, (const uint16_t *)dC, t, u, bank->scales, (uint16_t *)d_lora_a, (uint16_t *)d_lora_b, dx.rows, k, n, rank};
        switch ((rank + 15) / 16) {
            case 1: launch_grad<1>(g, hs); break;
            case 2: launch_grad<2>(g, hs); break;
            case 3: launch_grad<3>(g, hs); break;
            default: launch_grad<4>(g, hs); break;
        }
        dx.at = a_t;
        dx.u = u;
        dx.scales = bank->scales;
        dx.rank = rank;
    }
    if (m > 0) {
        dequant_rows_kernel<<<dim3(n / 128, k / 128), 512, 0, hs>>>((const u32x4 *)B, (const uint16_t *)s, wt, k, n, groupsize == -1 ? 1 : k / 128);
        constexpr int BM = 64 * kTileM, BN = 64 * kTileK;
        constexpr int lds = 2 * (BM + BN) * 128;
        bank_dx_kernel<kTileM, kTileK><<<dim3(k / BN, (m + BM - 1) / BM, w.dx_slices), 256, lds, hs>>>(dx);
        if (dx.partial) {
            const size_t units = (size_t)m * k / 4;
            sum_dx_kernel<<<(unsigned)((units + 255) / 256), 256, 0, hs>>>((const f32x4 *)dx.partial, (u32x2 *)dA, w.dx_slices, units);
        }
    }
    return hipGetLastError() == hipSuccess ? KILN_W4A16_OK : KILN_W4A16_ERR_LAUNCH;
}

}  // extern "C"
