// Rows in the order of their experts (kiln_w4a16_moe_sort) times their experts' packed weights, and the gradient of the rows:
//   y[p]  = x[p] W_e          (or of the token that position p is a pair of; or silu(gate) * up of it)
//   dx[p] = dy[p] W_e^T       for first[e] <= p < first[e + 1];  rows behind first[experts] are zero
// No counterpart in the reference, whose model family is dense: each expert is its packed GEMM (crates/kiln-marlin-gemm/csrc/marlin_kernel.cu:189-700).
//
// With many rows to an expert bound by the matrix cores, with few by the packs of the experts that have rows, read once.  One launch for all
// experts: the host knows how many rows there are, not whose, so it starts as many blocks as any choice could need and a block finds its
// expert, rows and columns in `first`; those without work leave.
//
// Either way a block is four wavefronts side by side, 32 MI rows x 256 columns of the result (64 to a wavefront: tiles of
// v_mfma_f32_32x32x16_bf16), 32 of the contraction to a stage.  Everything comes straight to LDS, four stages of the rows in flight.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <initializer_list>

#include "async_loads.h"
#include "bank.h"
#include "device_common.h"
#include "kiln_w4a16.h"
#include "launch.h"

namespace kiln {
namespace {

// 4 bytes per lane from an address of its own straight into LDS at lds_addr + 4 * lane (async_loads.h has the others)
__device__ __forceinline__ void lane_to_lds_b32(const void *gptr, unsigned lds_addr) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" : : "v"(gptr), "s"(lds_addr) : "memory", "m0");
}

constexpr int kMaxExperts = 1024;
constexpr int kWaves = 4, kThreads = kWaves * 64, kColumns = kWaves * 64, kStages = 4;

struct ExpertsArgs {
    const uint16_t *x;      // bf16 [rows, contraction], or with `order` [tokens, contraction]
    const int *first;       // [experts + 1]
    const int *order;       // [rows]: the pair of a position, or null
    const u32x4 *b;         // packs, one expert after the other
    const uint16_t *s;
    uint16_t *y;
    const float *sums;      // forward: -136 times the sums of x over a scale group, [K / 128][rows of x]
    int rows, x_rows, top, experts, K, N, Gs;
    int column_blocks;
};

// The work of a block: 32 MI rows of one expert at most, and a block of columns.  Blocks go to the eight dies in turn, a die's work is
// contiguous in (expert, columns, rows), rows first: what it reads at one time is a few blocks of a pack and one expert's rows.
struct Work {
    int expert, row0, rows, column;  // expert == experts: rows of no expert;  -1: nothing
};
template <int BM>
__device__ __forceinline__ Work find_work(const int *__restrict__ first, int experts, int rows, int column_blocks, int lane) {
    const int keys = experts + 1, per = (keys + 63) / 64, e0 = min(keys, lane * per), e1 = min(keys, e0 + per);
    auto begin_of = [&](int e) { return e < keys ? max(0, min(first[e], rows)) : rows; };  // (in bounds whatever `first` holds)
    auto tiles_of = [&](int e) { return (max(0, begin_of(e + 1) - begin_of(e)) + BM - 1) / BM; };
    int mine = 0;
    for (int e = e0; e < e1; ++e) mine += tiles_of(e);
    int upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int below = __shfl_up(upto, d);
        if (lane >= d) upto += below;
    }
    const unsigned total = (unsigned)__builtin_amdgcn_readlane(upto, 63) * (unsigned)column_blocks;
    const unsigned die = blockIdx.x & 7, seq = blockIdx.x >> 3, each = total >> 3, more = total & 7;
    if (seq >= each + (die < more ? 1u : 0u)) return {-1, 0, 0, 0};
    const unsigned id = die * each + min(die, more) + seq;
    const int tile = (int)(id / (unsigned)column_blocks);
    const int at = __builtin_ctzll(__ballot(upto > tile));
    int base = __builtin_amdgcn_readlane(upto - mine, at), e = at * per, count = 0;
    for (;; ++e) {
        count = __builtin_amdgcn_readfirstlane(tiles_of(e));
        if (tile < base + count) break;
        base += count;
    }
    const int inside = (int)(id - (unsigned)base * (unsigned)column_blocks), row0 = begin_of(e) + inside % count * BM;
    return {e, row0, min(BM, begin_of(e + 1) - row0), inside / count};
}

// rows of no expert: zeros in the block's columns
__device__ __forceinline__ void write_zeros(uint16_t *y, int width, int row0, int rows, int column0, int columns) {
    const int units = columns / 8;
    for (int i = threadIdx.x; i < rows * units; i += kThreads)
        *reinterpret_cast<u32x4 *>(y + (size_t)(row0 + i / units) * width + column0 + 8 * (i % units)) = u32x4{0u, 0u, 0u, 0u};
}

// A stage of the rows in LDS: 32 MI rows of 32 values, 64 bytes; four units of 16 bytes, unit u of row r at place u ^ (r / 4 & 3), so that the
// lanes that LDS serves together find their units in different banks.  One load fills 16 rows.
constexpr int kRowBytes = 64;
__device__ __forceinline__ unsigned unit_at(int row, int unit) { return (unsigned)(row * kRowBytes + ((unit ^ (row >> 2 & 3)) << 4)); }

template <int MI>
struct RowLoads {
    static constexpr int kEach = MI == 4 ? 2 : 1;  // loads of a wavefront (MI 1: two wavefronts fetch what the other two fetch)
    const char *from[kEach];
    unsigned to[kEach];
    template <class F>
    __device__ __forceinline__ RowLoads(const uint16_t *x, int width, int rows, int wave, int lane, F &&source_of) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int piece = MI == 1 ? wave & 1 : wave + kWaves * i, row = piece * 16 + (lane >> 2);
            from[i] = reinterpret_cast<const char *>(x + (size_t)source_of(min(row, rows - 1)) * width) + (((lane & 3) ^ (row >> 2 & 3)) << 4);
            to[i] = (unsigned)piece * 1024u;
        }
    }
    __device__ __forceinline__ void fetch(int stage, unsigned lds) const {
#pragma unroll
        for (int i = 0; i < kEach; ++i) load_to_lds_b128(from[i] + (size_t)stage * kRowBytes, lds + to[i]);
    }
};

template <int MI>
struct Tile {
    f32x16 acc[MI][2];
    __device__ __forceinline__ Tile() {
#pragma unroll
        for (int mi = 0; mi < MI; ++mi)
#pragma unroll
            for (int ni = 0; ni < 2; ++ni)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[mi][ni][r] = 0.f;
    }
};

// ---- forward -------------------------------------------------------------------------------------------------------
// The codes are multiplied as 128 + code; a group's scale is applied by a running rescale of the sums, (sums so far) / scale(g) times
// scale(g) / scale(g + 1) at each change of group, in f32, and the surplus of 136 comes off in the same multiply-add: -136 times the row's
// sum over the group, from a launch in front.  So a weight is exact: no rounding but the bf16 rows' own and the result's.
// A group's words, scales and row sums come to LDS two groups ahead.
template <int MI>
struct ForwardLds {
    static constexpr int kStage = 32 * MI * kRowBytes;
    static constexpr int kWords = kStages * kStage, kGroupWords = kWaves * 4096;
    static constexpr int kScales = kWords + 2 * kGroupWords, kSums = kScales + 2 * kWaves * 256, kBytes = kSums + 2 * kWaves * 256;
};

// -136 times the sums of a row's groups, [group][row]; 16 lanes to a group
__global__ __launch_bounds__(256) void expert_row_sums_kernel(const uint16_t *__restrict__ x, float *__restrict__ sums, int rows, int K) {
    const int G = K / kGroupK, sub = threadIdx.x & 15;
    const size_t item = (size_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    if (item >= (size_t)rows * G) return;
    const int row = (int)(item / G), g = (int)(item - (size_t)row * G);
    const u32x4 v = *reinterpret_cast<const u32x4 *>(x + (size_t)row * K + g * kGroupK + 8 * sub);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) sum += __builtin_bit_cast(float, v[i] << 16) + __builtin_bit_cast(float, v[i] & 0xFFFF0000u);
#pragma unroll
    for (int d = 8; d >= 1; d >>= 1) sum += __shfl_xor(sum, d, 16);
    if (sub == 0) sums[(size_t)g * rows + row] = -kCodeBias * sum;
}

__device__ __forceinline__ uint32_t pair_of(float low, float high) { return f32_to_bf16_bits(low) | (uint32_t)f32_to_bf16_bits(high) << 16; }
// Two values of a lane's column in neighbouring rows -> two of neighbouring columns in one row: even lanes get the first row's, odd lanes the second's.
__device__ __forceinline__ uint32_t across_columns(float first, float second, int lane) {
    const uint32_t own = pair_of(first, second);
    const uint32_t other = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)own, 0xB1, 0xF, 0xF, true);
    return __builtin_amdgcn_perm(own, other, lane & 1 ? 0x07060302u : 0x01000504u);
}

template <int MI, bool SWIGLU>
__global__ __launch_bounds__(kThreads, 2) void experts_kernel(ExpertsArgs p) {
    using L = ForwardLds<MI>;
    constexpr int BM = 32 * MI, LA = RowLoads<MI>::kEach, LW = 6;
    extern __shared__ __align__(16) char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l32 = lane & 31, h = lane >> 5;
    const Work work = find_work<BM>(p.first, p.experts, p.rows, p.column_blocks, lane);
    if (work.expert < 0) return;
    const int width = SWIGLU ? p.N / 2 : p.N, column0 = work.column * (SWIGLU ? kColumns / 2 : kColumns);
    if (work.expert == p.experts) {
        write_zeros(p.y, width, work.row0, work.rows, column0, SWIGLU ? kColumns / 2 : kColumns);
        return;
    }
    const int G = p.K / kGroupK, tiles = p.N / kTileN, nt0 = work.column * (kColumns / kTileN) + wave * 4;
    auto source_of = [&](int row) { return p.order ? (int)min((unsigned)p.order[work.row0 + row] / (unsigned)p.top, (unsigned)p.x_rows - 1) : work.row0 + row; };
    const RowLoads<MI> loads(p.x, p.K, work.rows, wave, lane, source_of);
    // the wavefront's four column tiles of a group, its scales and 64 of the block's row sums
    const char *const words = uniform(reinterpret_cast<const char *>(p.b) + ((size_t)work.expert * tiles + nt0) * G * 1024);
    const char *const scales = uniform(reinterpret_cast<const char *>(p.s + ((size_t)work.expert * tiles + nt0) * p.Gs * kTileN));
    const uint32_t scale_off = (uint32_t)(lane >> 3 & 3) * (uint32_t)p.Gs * (kTileN * 2) + (lane & 7) * 4;
    const char *const sums = reinterpret_cast<const char *>(p.sums + source_of(min((wave * 64 + lane) % BM, work.rows - 1)));
    const unsigned lds0 = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(lds_ptr_t)lds);
    const int stages = p.K / 32;
    auto fetch_rows = [&](int stage) {  // past the end: the last one again, so that the count of loads in flight stays what it is
        loads.fetch(min(stage, stages - 1), lds0 + (stage % kStages) * L::kStage);
    };
    auto fetch_group = [&](int g) {
        const int from = min(g, G - 1), slot = g & 1;
#pragma unroll
        for (int t = 0; t < 4; ++t)
            load_to_lds_b128(words + ((size_t)t * G + from) * 1024, (uint32_t)lane * 16u, lds0 + L::kWords + slot * L::kGroupWords + wave * 4096 + t * 1024);
        load_to_lds_b32(scales + (p.Gs == 1 ? 0 : (size_t)from * (kTileN * 2)), scale_off, lds0 + L::kScales + (slot * kWaves + wave) * 256);
        lane_to_lds_b32(sums + (size_t)from * p.x_rows * 4, lds0 + L::kSums + (slot * kWaves + wave) * 256);
    };
    // column sub-tile ni of the wavefront; SWIGLU: 0 the gate columns of its four tiles, 1 their up columns
    int word_at[2], scale_at[2];
#pragma unroll
    for (int ni = 0; ni < 2; ++ni) {
        const int t = SWIGLU ? l32 >> 3 : 2 * ni + (l32 >> 4), c = SWIGLU ? (l32 & 7) + 8 * ni : l32 & 15;
        word_at[ni] = L::kWords + wave * 4096 + t * 1024 + (c + 16 * h) * 16;
        scale_at[ni] = L::kScales + wave * 256 + (t * kTileN + c) * 2;
    }
    const DequantConsts dq = dequant_consts();
    Tile<MI> tile;
    u32x4 w[2][2];  // [ni][k16 step of a stage]: word t of a vector belongs to stage t
    float scale[2] = {1.f, 1.f};
    // the group's words and scales out of LDS, and its change of scale
    auto enter_group = [&](int g) {
        const int slot = g & 1;
        float f[2];
#pragma unroll
        for (int ni = 0; ni < 2; ++ni) {
#pragma unroll
            for (int v = 0; v < 2; ++v) w[ni][v] = *reinterpret_cast<const u32x4 *>(lds + word_at[ni] + slot * L::kGroupWords + v * 512);
            const float raw = f16_bits_to_f32(*reinterpret_cast<const uint16_t *>(lds + scale_at[ni] + slot * (kWaves * 256)));
            const float s = raw == 0.f ? 0x1p-40f : raw;  // a zero scale would end the running rescale: a value too small to matter
            f[ni] = scale[ni] * __builtin_amdgcn_rcpf(s);
            scale[ni] = s;
        }
        const char *c = lds + L::kSums + slot * (kWaves * 256) + h * 16;
#pragma unroll
        for (int mi = 0; mi < MI; ++mi)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x4 v = *reinterpret_cast<const f32x4 *>(c + mi * 128 + i * 32);
#pragma unroll
                for (int ni = 0; ni < 2; ++ni)
#pragma unroll
                    for (int r = 0; r < 4; ++r) tile.acc[mi][ni][4 * i + r] = fmaf(tile.acc[mi][ni][4 * i + r], f[ni], v[r]);
            }
    };
    struct Operands {
        bf16x8 a[MI];
    };
    auto read = [&](int slot, int step, Operands &o) {
#pragma unroll
        for (int mi = 0; mi < MI; ++mi) o.a[mi] = *reinterpret_cast<const bf16x8 *>(lds + slot * L::kStage + unit_at(32 * mi + l32, 2 * step + h));
    };
    auto multiply = [&](const Operands &o, auto tc, auto vc) {
#pragma unroll
        for (int ni = 0; ni < 2; ++ni) {
            const bf16x8 b = codes_to_bf16x8(w[ni][decltype(vc)::value][decltype(tc)::value], dq);
#pragma unroll
            for (int mi = 0; mi < MI; ++mi) tile.acc[mi][ni] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(o.a[mi], b, tile.acc[mi][ni], 0, 0, 0);
        }
    };
    using std::integral_constant;
    Operands now, then;
    fetch_group(0);
    fetch_group(1);
#pragma unroll
    for (int st = 0; st < kStages; ++st) fetch_rows(st);
    wait_vector_loads<3 * LA>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" : : : "memory");
    read(0, 0, now);
    for (int g = 0; g < G; ++g) {
        enter_group(g);
        unrolled<0, 4>([&](auto tc) {
            constexpr int t = decltype(tc)::value;
            read(t, 1, then);
            __builtin_amdgcn_sched_barrier(0);
            multiply(now, tc, integral_constant<int, 0>{});
            __builtin_amdgcn_sched_barrier(0);
            // The next stage has landed: behind it there are those of two more, and the group that was asked for one or two stages ago.  A next group's words
            // were asked for seven stages ago.
            wait_vector_loads<2 * LA + (t == 1 || t == 2 ? LW : 0)>();
            wait_lds_reads();
            __builtin_amdgcn_s_barrier();
            asm volatile("" : : : "memory");
            // every wavefront has this stage's rows in registers, and this group's words
            if constexpr (t == 0) fetch_group(g + 2);
            fetch_rows(4 * g + t + kStages);
            read((t + 1) & 3, 0, now);
            __builtin_amdgcn_sched_barrier(0);
            multiply(then, tc, integral_constant<int, 1>{});
            __builtin_amdgcn_sched_barrier(0);
        });
    }
    wait_vector_loads<0>();
    wait_lds_reads();
    __syncthreads();
    // 32 rows at a time through the wavefront's own part of LDS, so that a row's columns are written side by side
    constexpr int kPitch = (SWIGLU ? 64 : 128) + 16;
    char *mine = lds + wave * (32 * kPitch);
#pragma unroll
    for (int mi = 0; mi < MI; ++mi) {
#pragma unroll
        for (int r = 0; r < 16; r += 2) {
            char *at = mine + (8 * (r >> 2) + 4 * h + (r & 3) + (lane & 1)) * kPitch + (l32 & 30) * 2;
            if constexpr (SWIGLU) {
                float v[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float gate = tile.acc[mi][0][r + i] * scale[0], up = tile.acc[mi][1][r + i] * scale[1];
                    v[i] = gate * __builtin_amdgcn_rcpf(1.f + __expf(-gate)) * up;
                }
                *reinterpret_cast<uint32_t *>(at) = across_columns(v[0], v[1], lane);
            } else {
#pragma unroll
                for (int ni = 0; ni < 2; ++ni)
                    *reinterpret_cast<uint32_t *>(at + 64 * ni) = across_columns(tile.acc[mi][ni][r] * scale[ni], tile.acc[mi][ni][r + 1] * scale[ni], lane);
            }
        }
        wait_lds_reads();
        constexpr int kUnits = SWIGLU ? 4 : 8, kRowsAtOnce = 64 / kUnits;
#pragma unroll
        for (int i = 0; i < 32 / kRowsAtOnce; ++i) {
            const int r = i * kRowsAtOnce + lane / kUnits, unit = lane % kUnits;
            const u32x4 v = *reinterpret_cast<const u32x4 *>(mine + r * kPitch + unit * 16);
            if (32 * mi + r < work.rows)
                *reinterpret_cast<u32x4 *>(p.y + (size_t)(work.row0 + 32 * mi + r) * width + column0 + wave * (kUnits * 8) + unit * 8) = v;
        }
        wait_lds_reads();
    }
}

// ---- backward ------------------------------------------------------------------------------------------------------
// The contraction runs over a pack's columns, of which an operand of the matrix instruction wants eight to a lane, and a word holds eight rows
// of one column: LDS turns them on the way out (ds_read_b64_tr_b4: of 16 lanes' 16 codes each, lane i gets the i-th of every lane).  The
// scales run along the contraction too and cannot be pulled out of it, so a weight is rounded to bf16: (code - 8) * scale, exact in f32
// before, as for every 16-bit product of an unpacked weight.
// A stage is 32 columns of the pack, two column tiles: 32 lanes take one tile's, the others the other's.  A wavefront has 64 rows of
// the pack, half a scale group.
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i32x2 *lds_i32x2_ptr_t;
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

template <int MI>
struct BackwardLds {
    static constexpr int kRows = 32 * MI * kRowBytes, kCodes = kRows, kScales = kCodes + 4 * 1024, kStage = kScales + kWaves * 256;
    static constexpr int kBytes = kStages * kStage;
};

// eight codes of one row of the pack in eight columns, and those columns' scales: an operand
__device__ __forceinline__ bf16x8 weights_of(uint32_t codes, const u32x4 &scales) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // codes i and i + 4: 1024 + code in f16, less 1032
        const f16x2 d = __builtin_bit_cast(f16x2, (codes >> (4 * i) & 0x000F000Fu) | 0x64006400u) - f16x2{(_Float16)1032.f, (_Float16)1032.f};
        const f16x2 low = __builtin_bit_cast(f16x2, (uint32_t)scales[i >> 1]), high = __builtin_bit_cast(f16x2, (uint32_t)scales[2 + (i >> 1)]);
        v[i] = fmaf((float)d.x, (float)low[i & 1], 0.f);
        v[i + 4] = fmaf((float)d.y, (float)high[i & 1], 0.f);
    }
    bf16x8 o;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = (__bf16)v[i];
    return o;
}

template <int MI>
__global__ __launch_bounds__(kThreads, 2) void experts_backward_kernel(ExpertsArgs p) {
    using L = BackwardLds<MI>;
    constexpr int BM = 32 * MI, LA = RowLoads<MI>::kEach, LS = LA + 2;
    extern __shared__ __align__(16) char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l32 = lane & 31, h = lane >> 5;
    const Work work = find_work<BM>(p.first, p.experts, p.rows, p.column_blocks, lane);
    if (work.expert < 0) return;
    const int G = p.K / kGroupK, tiles = p.N / kTileN, k0 = work.column * kColumns;
    if (work.expert == p.experts) {
        write_zeros(p.y, p.K, work.row0, work.rows, k0, min(kColumns, p.K - k0));
        return;
    }
    const RowLoads<MI> loads(p.x, p.N, work.rows, wave, lane, [&](int row) { return work.row0 + row; });
    // of a stage's four chunks -- two tiles, two groups -- a wavefront fetches one; of the scales what it multiplies with
    const int group = min(2 * work.column + (wave >> 1), G - 1), group_fetched = min(2 * work.column + (wave & 1), G - 1), tile_fetched = wave >> 1;
    const char *const codes = uniform(reinterpret_cast<const char *>(p.b) + (((size_t)work.expert * tiles + tile_fetched) * G + group_fetched) * 1024);
    const char *const scales = uniform(reinterpret_cast<const char *>(p.s + ((size_t)work.expert * tiles * p.Gs + (p.Gs == 1 ? 0 : group)) * kTileN));
    const uint32_t scale_off = (uint32_t)(lane >> 3 & 1) * (uint32_t)p.Gs * (kTileN * 2) + (lane & 7) * 4;
    const unsigned lds0 = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(lds_ptr_t)lds);
    const int stages = p.N / 32;
    auto fetch = [&](int stage) {
        const int from = min(stage, stages - 1);
        const unsigned to = lds0 + (stage % kStages) * L::kStage;
        loads.fetch(from, to);
        load_to_lds_b128(codes + (size_t)from * 2 * G * 1024, (uint32_t)lane * 16u, to + L::kCodes + wave * 1024);
        load_to_lds_b32(scales + (size_t)from * 2 * p.Gs * (kTileN * 2), scale_off, to + L::kScales + wave * 256);
    };
    // chunk of tile h and the wavefront's group; in it the lane's column (lane % 16), its eight rows kq in each of two stages of 32 (half of the group)
    unsigned code_at[2];
#pragma unroll
    for (int ni = 0; ni < 2; ++ni) code_at[ni] = L::kCodes + (2 * h + (wave >> 1)) * 1024 + ((lane & 15) + 16 * (2 * ni + (l32 >> 4))) * 16 + 8 * (wave & 1);
    const unsigned scale_at = L::kScales + wave * 256 + h * 32;
    Tile<MI> tile;
    struct Operands {
        bf16x8 x[MI], w[2];
    };
    i32x2 turned[2];
    auto read_codes = [&](unsigned stage) {
#pragma unroll
        for (int ni = 0; ni < 2; ++ni)
            turned[ni] = __builtin_amdgcn_ds_read_tr4_b64_v2i32((lds_i32x2_ptr_t)(uintptr_t)(lds0 + stage + code_at[ni]));
    };
    auto read = [&](unsigned stage, auto uc, Operands &o) {
        constexpr int u = decltype(uc)::value;
#pragma unroll
        for (int mi = 0; mi < MI; ++mi) o.x[mi] = *reinterpret_cast<const bf16x8 *>(lds + stage + unit_at(32 * mi + l32, 2 * h + u));
        const u32x4 s = *reinterpret_cast<const u32x4 *>(lds + stage + scale_at + 16 * u);
#pragma unroll
        for (int ni = 0; ni < 2; ++ni) o.w[ni] = weights_of((uint32_t)turned[ni][u], s);
    };
    auto multiply = [&](const Operands &o) {
#pragma unroll
        for (int ni = 0; ni < 2; ++ni)
#pragma unroll
            for (int mi = 0; mi < MI; ++mi) tile.acc[mi][ni] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(o.w[ni], o.x[mi], tile.acc[mi][ni], 0, 0, 0);
    };
    using std::integral_constant;
    Operands now, then;
#pragma unroll
    for (int st = 0; st < kStages; ++st) fetch(st);
    wait_vector_loads<3 * LS>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" : : : "memory");
    read_codes(0);
    read(0, integral_constant<int, 0>{}, now);
    for (int st = 0; st < stages; ++st) {
        const unsigned stage = (st % kStages) * L::kStage, next = ((st + 1) % kStages) * L::kStage;
        read(stage, integral_constant<int, 1>{}, then);
        __builtin_amdgcn_sched_barrier(0);
        multiply(now);
        __builtin_amdgcn_sched_barrier(0);
        wait_vector_loads<2 * LS>();
        wait_lds_reads();
        __builtin_amdgcn_s_barrier();
        asm volatile("" : : : "memory");
        fetch(st + kStages);
        read_codes(next);
        read(next, integral_constant<int, 0>{}, now);
        __builtin_amdgcn_sched_barrier(0);
        multiply(then);
        __builtin_amdgcn_sched_barrier(0);
    }
    wait_vector_loads<0>();
    wait_lds_reads();
    if (2 * work.column + (wave >> 1) >= G) return;  // (a last block of half the columns)
    // A lane has row l32 of a row tile and of eight consecutive rows of the pack the even ones (lanes 32 ... 63: the odd ones): two such
    // eights change hands with the other half, and a lane writes one whole.
#pragma unroll
    for (int mi = 0; mi < MI; ++mi) {
        const int row = 32 * mi + l32;
#pragma unroll
        for (int ni = 0; ni < 2; ++ni)
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                u32x4 o;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float first = tile.acc[mi][ni][8 * b + i], second = tile.acc[mi][ni][8 * b + 4 + i];
                    const auto swapped = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, first), __builtin_bit_cast(unsigned, second), false, false);
                    o[i] = pair_of(__builtin_bit_cast(float, (unsigned)swapped[0]), __builtin_bit_cast(float, (unsigned)swapped[1]));
                }
                const int k = k0 + 64 * wave + 32 * h + 8 * (2 * ni + b);
                if (row < work.rows) *reinterpret_cast<u32x4 *>(p.y + (size_t)(work.row0 + row) * p.K + k) = o;
            }
    }
}

// ---- launches ------------------------------------------------------------------------------------------------------
// The most row tiles that rows sorted by expert can take: a part tile to every expert that has rows, and to the rows without one
int64_t most_tiles(int rows, int experts, int block_rows) {
    return (int64_t)rows / block_rows + std::min<int64_t>((int64_t)experts + 1, rows);
}
// Row tiles of a block by the rows that an expert has on average.
int row_tiles(int rows, int experts) {
    const int each = rows / experts;
    return each <= 32 ? 1 : each <= 64 ? 2 : 4;
}
template <auto Kernel>
bool launch(const ExpertsArgs &a, int block_rows, int lds_bytes, hipStream_t stream) {
    if (allow_dynamic_lds<Kernel>(lds_bytes) != hipSuccess) return false;
    Kernel<<<(unsigned)(most_tiles(a.rows, a.experts, block_rows) * a.column_blocks), kThreads, lds_bytes, stream>>>(a);
    return true;
}

kiln_marlin_status_t experts_ok(int rows, int n, int k, int experts, int groupsize) {
    if (rows < 0 || n <= 0 || k <= 0 || n % 256 != 0 || k % 128 != 0 || (groupsize != -1 && groupsize != 128)) return KILN_W4A16_ERR_PROB_SHAPE;
    if (experts < 1 || experts > kMaxExperts) return KILN_W4A16_ERR_KERN_SHAPE;
    return most_tiles(rows, experts, 32) * (std::max((int64_t)n, (int64_t)k) / 256 + 1) > INT32_MAX ? KILN_W4A16_ERR_KERN_SHAPE : KILN_W4A16_OK;
}
bool aligned(std::initializer_list<const void *> pointers) {
    for (const void *p : pointers)
        if (!p || reinterpret_cast<uintptr_t>(p) % 16 != 0) return false;
    return true;
}

}  // namespace
}  // namespace kiln

using namespace kiln;

extern "C" {

size_t kiln_w4a16_gemm_experts_scratch_bytes(int x_rows, int prob_k) {
    return x_rows < 1 || prob_k < kGroupK ? 256 : ((size_t)x_rows * (prob_k / kGroupK) * sizeof(float) + 255) & ~(size_t)255;
}

kiln_marlin_status_t kiln_w4a16_gemm_experts(const void *x, const int *first, const int *order, const void *b, const void *s, void *y, int rows, int x_rows,
                                             int top_k, int prob_n, int prob_k, int experts, int groupsize, int swiglu, int dev, void *stream, void *scratch) {
    (void)dev;
    if (const kiln_marlin_status_t st = experts_ok(rows, prob_n, prob_k, experts, groupsize)) return st;
    if (x_rows < 0 || top_k < 1 || (order ? (int64_t)x_rows * top_k != rows : x_rows != rows)) return KILN_W4A16_ERR_KERN_SHAPE;
    if ((int64_t)x_rows * (prob_k / kGroupK) > (int64_t)INT32_MAX * 16) return KILN_W4A16_ERR_KERN_SHAPE;
    if (rows == 0) return KILN_W4A16_OK;
    if (!aligned({x, b, s, y, scratch}) || !first) return KILN_W4A16_ERR_ARGUMENT;
    const int width = swiglu ? prob_n / 2 : prob_n;
    if (meet(y, (size_t)rows * width * 2, x, (size_t)x_rows * prob_k * 2)) return KILN_W4A16_ERR_ARGUMENT;
    hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
    const size_t items = (size_t)x_rows * (prob_k / kGroupK);
    expert_row_sums_kernel<<<(unsigned)((items + 15) / 16), 256, 0, hs>>>((const uint16_t *)x, (float *)scratch, x_rows, prob_k);
    const ExpertsArgs a{(const uint16_t *)x, first, order, (const u32x4 *)b, (const uint16_t *)s, (uint16_t *)y, (const float *)scratch,
                        rows, x_rows, top_k, experts, prob_k, prob_n, groupsize == -1 ? 1 : prob_k / kGroupK, prob_n / kColumns};
    bool ok = false;
    auto with = [&](auto mc) {
        constexpr int MI = decltype(mc)::value;
        ok = swiglu ? launch<experts_kernel<MI, true>>(a, 32 * MI, ForwardLds<MI>::kBytes, hs)
                    : launch<experts_kernel<MI, false>>(a, 32 * MI, ForwardLds<MI>::kBytes, hs);
    };
    switch (row_tiles(rows, experts)) {
        case 1: with(std::integral_constant<int, 1>{}); break;
        case 2: with(std::integral_constant<int, 2>{}); break;
        default: with(std::integral_constant<int, 4>{});
    }
    return ok && hipGetLastError() == hipSuccess ? KILN_W4A16_OK : KILN_W4A16_ERR_LAUNCH;
}

kiln_marlin_status_t kiln_w4a16_gemm_experts_backward(const void *dy, const int *first, const void *b, const void *s, void *dx, int rows, int prob_n, int prob_k,
                                                      int experts, int groupsize, int dev, void *stream) {
    (void)dev;
    if (const kiln_marlin_status_t st = experts_ok(rows, prob_n, prob_k, experts, groupsize)) return st;
    if (rows == 0) return KILN_W4A16_OK;
    if (!aligned({dy, b, s, dx}) || !first) return KILN_W4A16_ERR_ARGUMENT;
    if (meet(dx, (size_t)rows * prob_k * 2, dy, (size_t)rows * prob_n * 2)) return KILN_W4A16_ERR_ARGUMENT;
    hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
    const ExpertsArgs a{(const uint16_t *)dy, first, nullptr, (const u32x4 *)b, (const uint16_t *)s, (uint16_t *)dx, nullptr,
                        rows, rows, 1, experts, prob_k, prob_n, groupsize == -1 ? 1 : prob_k / kGroupK, (prob_k + kColumns - 1) / kColumns};
    bool ok = false;
    auto with = [&](auto mc) {
        constexpr int MI = decltype(mc)::value;
        ok = launch<experts_backward_kernel<MI>>(a, 32 * MI, BackwardLds<MI>::kBytes, hs);
    };
    switch (row_tiles(rows, experts)) {
        case 1: with(std::integral_constant<int, 1>{}); break;
        case 2: with(std::integral_constant<int, 2>{}); break;
        default: with(std::integral_constant<int, 4>{});
    }
    return ok && hipGetLastError() == hipSuccess ? KILN_W4A16_OK : KILN_W4A16_ERR_LAUNCH;
}

}  // extern "C"
