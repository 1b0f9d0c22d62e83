// Rows in the order of their experts (kiln_w4a16_moe_sort) times their experts' packed weights, and the gradient of the rows:
//   y[p]  = x[p] W_e          (or of the token that position p is a pair of; or silu(gate) * up of it)
//   dx[p] = dy[p] W_e^T       for first[e] <= p < first[e + 1];  rows behind first[experts] are zero
// No counterpart in the reference, whose model family is dense: each expert is its packed GEMM (crates/kiln-marlin-gemm/csrc/marlin_kernel.cu:189-700).
//
// With many rows to an expert bound by the matrix cores, with few by the packs of the experts that have rows, read once.  One launch for all
// experts: the host knows how many rows there are, not whose, so it starts as many blocks as any choice could need and a block finds its
// expert, rows and columns in `first`; those without work leave.
//
// A block is four wavefronts; tiles of v_mfma_f32_32x32x16_bf16, everything straight to LDS in stages of the contraction with several on their way.  By the rows
// that an expert has (choose_blocks) it takes
//   128 rows x 256 columns: four row tiles x 64 columns to a wavefront, products scheduled by hand,
//   64 or 32 rows x 256 columns: larger stages, the loads bound them,
//   the same with two sets of wavefronts, for half of the contraction each, where a compute unit gets one block at most,
//   32 rows x 64 columns (the gradient: 128), the wavefronts sharing out the contraction, where the others would leave compute units idle.
// In blocks of 128 and 64 rows what is left of an expert goes as in the smaller ones.
//
// us a call and what bounds it: 16384 rows of 64 experts, 2560 -> 2048 (172 GFLOP): 177-195, the gradient 209-217: rounds of blocks that do not come out even (the same rows in
// equal parts 167 and 187), and power: on values of this kind the matrix instructions alone reach 1.6 to 1.8 PFLOP/s, not the 2.2 that they do on zeros, and the vector
// instructions that expand the codes, reads of LDS and loads come on top (each left out for a measurement took 2 to 8 % off); 768 rows of 64 experts, 2560 -> 2048:
// 42, 4.1 TB/s of packs; 2331 rows of 24 experts, 1280 -> 2048: 24-27, a round and a half of blocks, each one's start (6 us with its stores), then 1.2 us to 128 of the
// contraction, 2.1 where two blocks share a compute unit: matrix products 0.5 of it, vector instructions, LDS and loads 0.1 to 0.2 each.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "async_loads.h"
#include "device_common.h"
#include "kiln_w4a16.h"
#include "launch.h"
#include "pieces.h"

namespace kiln {
namespace {

constexpr int kMaxExperts = 1024, kMaxRows = 1 << 29;  // (a row's sum has a 32-bit offset)
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

// The work of a block: up to BM rows of one expert, and a block of columns.  What is left of an expert behind its last whole row tile comes first where that is no more than half
// a tile: those blocks wait for their loads, and beside others they are no tail (ordered last: 16384 rows of 64
// experts, 2560 -> 2048 200 us, first 180; the gradient 217 and 203).
// Blocks go to the eight dies in turn, a die's share of either list is contiguous in (expert, columns, rows), rows first: what it reads at one time is a few
// blocks of a pack and one expert's rows.
struct Work {
    int expert, row0, rows, column;  // expert == experts: rows of no expert;  -1: nothing
};
// (Nothing else is on its way while a block finds its work: up to 63 experts are a lane's each, loaded together and read from the lanes again.)
__device__ __forceinline__ int sum_of_lanes_upto(int v) {
    auto add = [&](auto control, auto rows) { v += __builtin_amdgcn_update_dpp(0, v, decltype(control)::value, decltype(rows)::value, 0xF, false); };
    using std::integral_constant;
    add(integral_constant<int, 0x111>{}, integral_constant<int, 0xF>{});  // from 1, 2, 4, 8 lanes below in a row of 16
    add(integral_constant<int, 0x112>{}, integral_constant<int, 0xF>{});
    add(integral_constant<int, 0x114>{}, integral_constant<int, 0xF>{});
    add(integral_constant<int, 0x118>{}, integral_constant<int, 0xF>{});
    add(integral_constant<int, 0x142>{}, integral_constant<int, 0xA>{});  // the last lane of the row below to rows 1 and 3
    add(integral_constant<int, 0x143>{}, integral_constant<int, 0xC>{});  // lane 31 to rows 2 and 3
    return v;
}
template <int BM>
__device__ __forceinline__ Work find_work(const int *__restrict__ first, int experts, int rows, int column_blocks, int lane) {
    const int keys = experts + 1, per = (keys + 63) / 64, e0 = min(keys, lane * per), e1 = min(keys, e0 + per);
    auto begin_of = [&](int e) {  // (in bounds whatever `first` holds)
        const int begin = first[min(e, experts)];
        return e < keys ? max(0, min(begin, rows)) : rows;
    };
    auto tiles_of = [](int n) { return (n + BM / 2 - 1) / BM; };  // of more than half of BM rows
    auto has_rest = [](int n) { return n % BM != 0 && n % BM <= BM / 2; };
    int begin = begin_of(e0), end = begin_of(e0 + 1), n = max(0, end - begin);  // of the lane's first expert
    int tiles = tiles_of(n), rests = has_rest(n);  // of all of them
    for (int e = e0 + 1; e < e1; ++e) {
        const int next = begin_of(e + 1), m = max(0, next - end);
        tiles += tiles_of(m);
        rests += has_rest(m);
        end = next;
    }
    const int tiles_upto = sum_of_lanes_upto(tiles), rests_upto = sum_of_lanes_upto(rests);
    unsigned seq = blockIdx.x >> 3, id;
    auto mine = [&](unsigned total, unsigned die) {  // of a list: is this block's place in the die's share of it?
        const unsigned each = total >> 3, more = total & 7, count = each + (die < more ? 1u : 0u);
        id = die * each + min(die, more) + seq;
        if (seq < count) return true;
        seq -= count;
        return false;
    };
    // (what does not go evenly into eight is the first dies' of one list and the last dies' of the other: as many blocks as compute units are one to each)
    const unsigned die = blockIdx.x & 7;
    const bool is_rest = mine((unsigned)__builtin_amdgcn_readlane(rests_upto, 63) * (unsigned)column_blocks, die);
    if (!is_rest && !mine((unsigned)__builtin_amdgcn_readlane(tiles_upto, 63) * (unsigned)column_blocks, 7 - die)) return {-1, 0, 0, 0};
    const int tile = (int)(id / (unsigned)column_blocks), upto = is_rest ? rests_upto : tiles_upto;
    const int at = __builtin_ctzll(__ballot(upto > tile));
    int base = __builtin_amdgcn_readlane(upto - (is_rest ? rests : tiles), at), e = at * per;
    begin = __builtin_amdgcn_readlane(begin, at);
    n = __builtin_amdgcn_readlane(n, at);
    int count;
    for (;;) {
        count = is_rest ? has_rest(n) : tiles_of(n);
        if (tile < base + count) break;
        base += count;
        ++e;
        begin = __builtin_amdgcn_readfirstlane(begin_of(e));
        n = max(0, __builtin_amdgcn_readfirstlane(begin_of(e + 1)) - begin);
    }
    const int inside = (int)(id - (unsigned)base * (unsigned)column_blocks);
    if (is_rest) return {e, begin + n / BM * BM, n % BM, inside};
    const int t = inside % count;
    return {e, begin + t * BM, min(BM, n - t * BM), inside / count};
}

// rows of no expert: zeros in the block's columns
__device__ __forceinline__ void write_zeros(uint16_t *y, int width, int row0, int rows, int column0, int columns) {
    const int units = columns / 8;
    for (int i = threadIdx.x; i < rows * units; i += blockDim.x)
        *reinterpret_cast<u32x4 *>(y + (size_t)(row0 + i / units) * width + column0 + 8 * (i % units)) = u32x4{0u, 0u, 0u, 0u};
}

// A stage of the rows in LDS: 32 MI rows of 32 values, 64 bytes; four units of 16 bytes, unit u of row r at place u ^ (r / 4 & 3), so that the
// lanes that LDS serves together find their units in different banks.  One load fills 16 rows.
constexpr int kRowBytes = 64;
__device__ __forceinline__ unsigned unit_at(int row, int unit) { return (unsigned)(row * kRowBytes + ((unit ^ (row >> 2 & 3)) << 4)); }

template <int MI>
struct RowLoads {
    static constexpr int kEach = MI > 2 ? 2 : 1;  // loads of a wavefront (MI 1 and 3: two wavefronts fetch what another fetches)
    const char *from[kEach];
    unsigned to[kEach];
    template <class F>
    __device__ __forceinline__ RowLoads(const uint16_t *x, int width, int rows, int wave, int lane, F &&source_of) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int piece = (wave + kWaves * i) % (2 * MI), row = piece * 16 + (lane >> 2);
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
// The codes are multiplied as 128 + code, so a weight is exact: no rounding but the bf16 rows' own and the result's.  A group's scale is
// applied by a running rescale of the sums, (sums so far) / scale(g) times scale(g) / scale(g + 1) at each change of group, in f32.  The
// surplus of 136 times a row's sum over the group comes off
//   in blocks of 128 rows at the group's start, in the rescale's own multiply-add, from sums that a launch in front has formed: no work of its own;
//   in smaller ones at its end, by one product more with -136 throughout, of sums that a lane forms of the rows it multiplies (two values to an
//   instruction): calls of nothing else need no launch in front.  (Eight products, one beside every step's: 2331 rows of 24 experts, 1280 -> 2048 29 us, so 26.)
// A group's words and scales come to LDS two groups ahead.
struct ManyLds {
    static constexpr int kStage = 128 * kRowBytes;
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

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pair_of(float low, float high) { return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)low, (__bf16)high}); }
// Two values of a lane's column in neighbouring rows -> two of neighbouring columns in one row: even lanes get the first row's, odd lanes the second's.
__device__ __forceinline__ uint32_t across_columns(float first, float second, int lane) {
    const uint32_t own = pair_of(first, second);
    const uint32_t other = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)own, 0xB1, 0xF, 0xF, true);
    return __builtin_amdgcn_perm(own, other, lane & 1 ? 0x07060302u : 0x01000504u);
}

__device__ __forceinline__ int source_of(const ExpertsArgs &p, int pair) { return (int)min((unsigned)pair / (unsigned)p.top, (unsigned)p.x_rows - 1); }
__device__ __forceinline__ int source_of(const ExpertsArgs &p, const Work &work, int row) {
    return p.order ? source_of(p, p.order[work.row0 + row]) : work.row0 + row;
}

// A wavefront's four column tiles of its expert's pack, from tile nt0 on: a group's words and scales to LDS (five loads), and out of it, words_in and
// scales_in bytes into what is there for them.  Column sub-tile ni is what a lane multiplies; SWIGLU: 0 the gate columns of the four tiles, 1
// their up columns, so that a lane has both in the same register.
template <bool SWIGLU>
struct Columns {
    const char *words, *scales;
    uint32_t scale_off;
    unsigned lane16;
    int words_in, scales_in, word_at, scale_at, G, scale_step;
    static constexpr int kNextWords = SWIGLU ? 8 * 16 : 2 * 1024, kNextScale = SWIGLU ? 8 * 2 : 2 * kTileN * 2;  // from sub-tile 0's to sub-tile 1's
    __device__ __forceinline__ Columns(const ExpertsArgs &p, int expert, int nt0, int lane, int words_in, int scales_in)
        : lane16(lane * 16), words_in(words_in), scales_in(scales_in), G(p.K / kGroupK) {
        const int tiles = p.N / kTileN, l32 = lane & 31;
        words = uniform(reinterpret_cast<const char *>(p.b) + ((size_t)expert * tiles + nt0) * G * 1024);
        scales = uniform(reinterpret_cast<const char *>(p.s + ((size_t)expert * tiles + nt0) * p.Gs * kTileN));
        scale_off = (uint32_t)(lane >> 3 & 3) * (uint32_t)p.Gs * (kTileN * 2) + (lane & 7) * 4;
        scale_step = p.Gs == 1 ? 0 : kTileN * 2;
        const int t = SWIGLU ? l32 >> 3 : l32 >> 4, c = SWIGLU ? l32 & 7 : l32 & 15;
        word_at = words_in + t * 1024 + (c + 16 * (lane >> 5)) * 16;
        scale_at = scales_in + (t * kTileN + c) * 2;
    }
    __device__ __forceinline__ void fetch(int g, unsigned words_to, unsigned scales_to) const {
        const unsigned to = __builtin_amdgcn_readfirstlane(words_to + words_in), at = __builtin_amdgcn_readfirstlane(scales_to + scales_in);
#pragma unroll
        for (int t = 0; t < 4; ++t) load_to_lds_b128(words + ((size_t)t * G + g) * 1024, lane16, to + t * 1024);
        load_to_lds_b32(scales + (size_t)g * scale_step, scale_off, at);
    }
    // [ni][k16 step of 32]: word t of a vector belongs to the t-th 32 of the group
    __device__ __forceinline__ void read_words(const char *from, u32x4 (&w)[2][2]) const {
#pragma unroll
        for (int ni = 0; ni < 2; ++ni)
#pragma unroll
            for (int v = 0; v < 2; ++v) w[ni][v] = *reinterpret_cast<const u32x4 *>(from + word_at + ni * kNextWords + v * 512);
    }
    __device__ __forceinline__ float read_scale(const char *from, int ni) const {
        const float raw = f16_bits_to_f32(*reinterpret_cast<const uint16_t *>(from + scale_at + ni * kNextScale));
        return raw == 0.f ? 0x1p-40f : raw;  // a zero scale would end the running rescale: a value too small to matter
    }
};

constexpr int kStoreBytes = kWaves * 32 * (128 + 16);
// the scaled sums out, 32 rows at a time through the wavefront's own part of LDS (which nothing else uses any more), so that a row's columns are written
// side by side
template <int MI, bool SWIGLU>
__device__ __forceinline__ void store_tile(const ExpertsArgs &p, const Work &work, char *lds, int lane, int wave, Tile<MI> &tile, const float (&scale)[2]) {
    constexpr int kPitch = (SWIGLU ? 64 : 128) + 16;
    char *mine = lds + wave * (32 * kPitch);
    const int width = SWIGLU ? p.N / 2 : p.N, column0 = work.column * (SWIGLU ? kColumns / 2 : kColumns), l32 = lane & 31, h = lane >> 5;
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

// Up to 64 rows: bound by the loads, so a stage is a whole group -- 128 of the contraction, 256 bytes of a row in 16 units, unit u of row r at place
// u ^ (r & 15) --, with two or one more on their way while one is multiplied, and one barrier.  One stage to a turn of the loop: code that is not
// repeated is read from memory in every launch, which short blocks wait for.
template <int MI>
struct FewLds {
    static constexpr int kRing = MI == 1 ? 3 : 2, kRows = 32 * MI * 256, kScales = kRows + kWaves * 4096, kStage = kScales + kWaves * 256;
    static constexpr int kBytes = kRing * kStage;
};
// a group's eight k16 steps: the words' word t holds two of them.  Behind them the rows' surplus: a lane has summed its half of row lane % 32, and one more
// product, with -136 throughout, adds up the halves and takes them off -- the sum in three parts of 8 bits, which is all of it.
template <int MI>
__device__ __forceinline__ void few_product(const char *rows, const u32x4 (&w)[2][2], const DequantConsts &dq, int lane, Tile<MI> &tile) {
    const bf16x8 bias = bf16x8_splat(0xC308C308u);  // -136
    static_assert(kCodeBias == 136.f, "");
    const int l32 = lane & 31, h = lane >> 5;
    float sum[MI];
    unrolled<0, 8>([&](auto sc) {
        constexpr int step = decltype(sc)::value, t = step >> 1, v = step & 1;
        u32x4 a[MI];
#pragma unroll
        for (int mi = 0; mi < MI; ++mi) a[mi] = *reinterpret_cast<const u32x4 *>(rows + (32 * mi + l32) * 256 + (((2 * step + h) ^ (l32 & 15)) << 4));
#pragma unroll
        for (int ni = 0; ni < 2; ++ni) {
            const bf16x8 b = codes_to_bf16x8(w[ni][v][t], dq);
#pragma unroll
            for (int mi = 0; mi < MI; ++mi)
                tile.acc[mi][ni] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a[mi]), b, tile.acc[mi][ni], 0, 0, 0);
        }
#pragma unroll
        for (int mi = 0; mi < MI; ++mi)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                sum[mi] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, (uint32_t)a[mi][i]), bf16x2{(__bf16)1.f, (__bf16)1.f}, step + i == 0 ? 0.f : sum[mi], false);
    });
#pragma unroll
    for (int mi = 0; mi < MI; ++mi) {
        const uint32_t first = __builtin_bit_cast(uint32_t, sum[mi]);
        const float behind = sum[mi] - __builtin_bit_cast(float, first & 0xFFFF0000u);
        const uint32_t second = __builtin_bit_cast(uint32_t, behind);
        const uint32_t third = __builtin_bit_cast(uint32_t, behind - __builtin_bit_cast(float, second & 0xFFFF0000u));
        const bf16x8 parts = __builtin_bit_cast(bf16x8, u32x4{__builtin_amdgcn_perm(second, first, 0x07060302u), third >> 16, 0u, 0u});
#pragma unroll
        for (int ni = 0; ni < 2; ++ni) tile.acc[mi][ni] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(parts, bias, tile.acc[mi][ni], 0, 0, 0);
    }
}
// the sums in units of the next group's scale
template <int MI>
__device__ __forceinline__ void few_rescale(Tile<MI> &tile, const float (&by)[2]) {
#pragma unroll
    for (int mi = 0; mi < MI; ++mi)
#pragma unroll
        for (int ni = 0; ni < 2; ++ni)
#pragma unroll
            for (int r = 0; r < 16; ++r) tile.acc[mi][ni][r] *= by[ni];
}

// Where a compute unit gets one block at most, the block has a second set of four wavefronts for every other group (SETS), with LDS of its own; their sums
// meet there at the end, the first set's before the second's.
template <int MI>
__device__ __forceinline__ void add_second_set(char *lds, int lane, int wave, int set, Tile<MI> &tile) {
    static_assert(kStoreBytes + MI * 32768 <= 2 * FewLds<MI>::kBytes, "");
    wait_vector_loads<0>();  // stages asked for past the end still write to LDS
    wait_lds_reads();
    __syncthreads();
    float *box = reinterpret_cast<float *>(lds + kStoreBytes) + wave * (MI * 2048) + lane;
    if (set == 1)
#pragma unroll
        for (int i = 0; i < MI * 32; ++i) box[i * 64] = tile.acc[i >> 5][i >> 4 & 1][i & 15];
    __syncthreads();
    if (set == 0)
#pragma unroll
        for (int i = 0; i < MI * 32; ++i) tile.acc[i >> 5][i >> 4 & 1][i & 15] += box[i * 64];
}

template <int MI, bool SWIGLU, int SETS>
__device__ __forceinline__ void experts_few(const ExpertsArgs &p, const Work &work, char *all_lds, int lane, int wave_of_all) {
    using L = FewLds<MI>;
    const int wave = wave_of_all % kWaves, set = wave_of_all / kWaves;
    char *const lds = all_lds + set * L::kBytes;
    constexpr int LR = 2 * MI, LS = LR + 5;  // loads of a wavefront and stage: four rows each; with the words and scales
    const Columns<SWIGLU> cols(p, work.expert, work.column * (kColumns / kTileN) + wave * 4, lane, wave * 4096, wave * 256);
    const int G = p.K / kGroupK;
    const unsigned lds0 = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(lds_ptr_t)lds);
    auto group_of = [&](int turn) { return min(SETS * turn + set, G - 1); };  // past the end: the last one again, so that the count of loads in flight stays what it is
    auto stage_of = [&](int turn) { return lds0 + (unsigned)(turn % L::kRing) * L::kStage; };
    // The first stages' words wait for nothing, their rows for the order, which goes by the ring's last place.
    const unsigned spare = (unsigned)(L::kRing - 1) * L::kStage + wave * 256;
    if (p.order) load_to_lds_b32(uniform(reinterpret_cast<const char *>(p.order + work.row0)), (uint32_t)min(lane, work.rows - 1) * 4u, lds0 + spare);
#pragma unroll
    for (int turn = 0; turn < L::kRing - 1; ++turn) cols.fetch(group_of(turn), stage_of(turn) + L::kRows, stage_of(turn) + L::kScales);
    wait_vector_loads<(L::kRing - 1) * 5>();
    const char *rows[LR];
#pragma unroll
    for (int i = 0; i < LR; ++i) {
        const int row = 4 * (wave * LR + i) + (lane >> 4);
        const int source = p.order ? source_of(p, *reinterpret_cast<const int *>(lds + spare + 4 * row)) : work.row0 + min(row, work.rows - 1);
        rows[i] = reinterpret_cast<const char *>(p.x + (size_t)source * p.K) + (((lane & 15) ^ (row & 15)) << 4);
    }
    auto fetch_rows = [&](int turn) {
#pragma unroll
        for (int i = 0; i < LR; ++i) load_to_lds_b128(rows[i] + (size_t)group_of(turn) * 256, stage_of(turn) + (wave * LR + i) * 1024);
    };
    auto fetch = [&](int turn) {
        fetch_rows(turn);
        cols.fetch(group_of(turn), stage_of(turn) + L::kRows, stage_of(turn) + L::kScales);
    };
    const DequantConsts dq = dequant_consts();
    Tile<MI> tile;
    float scale[2] = {0.f, 0.f};
#pragma unroll
    for (int turn = 0; turn < L::kRing - 1; ++turn) fetch_rows(turn);
    wait_vector_loads<(L::kRing - 2) * LR>();  // the words and the first stage's rows; from here on a stage's rows are asked for before its words
#pragma unroll 1
    for (int turn = 0; SETS * turn < G; ++turn) {
        wait_vector_loads<(L::kRing - 2) * LS>();  // this stage has landed
        wait_lds_reads();
        __builtin_amdgcn_s_barrier();  // ... everywhere, and the one before has been read
        asm volatile("" : : : "memory");
        fetch(turn + L::kRing - 1);
        if (SETS > 1 && SETS * turn + set >= G) break;  // (the last turn of all)
        const char *stage = lds + (turn % L::kRing) * L::kStage;
        u32x4 w[2][2];
        float by[2];
        cols.read_words(stage + L::kRows, w);
#pragma unroll
        for (int ni = 0; ni < 2; ++ni) {
            const float next = cols.read_scale(stage + L::kScales, ni);
            by[ni] = scale[ni] * __builtin_amdgcn_rcpf(next);
            scale[ni] = next;
        }
        if (p.Gs != 1) few_rescale(tile, by);  // (of the first group: zeros)
        few_product<MI>(stage, w, dq, lane, tile);
    }
    few_rescale(tile, scale);
    if constexpr (SETS > 1) {
        add_second_set<MI>(all_lds, lane, wave, set, tile);
        if (set == 1) return;
    } else {
        wait_vector_loads<0>();
        wait_lds_reads();
        __syncthreads();
    }
    const float done[2] = {1.f, 1.f};
    store_tile<MI, SWIGLU>(p, work, all_lds, lane, wave, tile, done);
}

// Calls whose blocks would not fill the chip: a block takes 32 rows x 64 columns, its wavefronts every fourth group each.  They share nothing until
// the end, where their sums meet in LDS: no barriers, each waits for its own loads alone.
struct SplitLds {
    static constexpr int kRing = 3, kScales = 32 * 256 + 4096, kStage = kScales + 256, kWave = kRing * kStage, kBytes = kWaves * kWave;
};
template <bool SWIGLU>
__global__ __launch_bounds__(kThreads, 1) void experts_split_kernel(ExpertsArgs p) {
    using L = SplitLds;
    constexpr int LS = 8 + 5;  // loads of a stage: its rows', the words' and the scales'
    extern __shared__ __align__(16) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l32 = lane & 31, h = lane >> 5;
    const Work work = find_work<32>(p.first, p.experts, p.rows, p.column_blocks, lane);
    if (work.expert < 0) return;
    const int width = SWIGLU ? p.N / 2 : p.N, column0 = work.column * (SWIGLU ? 32 : 64), G = p.K / kGroupK;
    if (work.expert == p.experts) {
        write_zeros(p.y, width, work.row0, work.rows, column0, SWIGLU ? 32 : 64);
        return;
    }
    const Columns<SWIGLU> cols(p, work.expert, work.column * 4, lane, 0, 0);
    const unsigned lds0 = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(lds_ptr_t)lds + wave * L::kWave);
    auto group_of = [&](int turn) { return min(wave + kWaves * turn, G - 1); };  // past the end: the last group again, so that the count of loads in flight stays what it is
    auto stage_of = [&](int turn) { return lds0 + (unsigned)(turn % L::kRing) * L::kStage; };
    const unsigned spare = (unsigned)(L::kRing - 1) * L::kStage;  // (as in experts_few)
    if (p.order) load_to_lds_b32(uniform(reinterpret_cast<const char *>(p.order + work.row0)), (uint32_t)min(lane, work.rows - 1) * 4u, lds0 + spare);
#pragma unroll
    for (int turn = 0; turn < L::kRing - 1; ++turn) cols.fetch(group_of(turn), stage_of(turn) + 32 * 256, stage_of(turn) + L::kScales);
    wait_vector_loads<(L::kRing - 1) * 5>();
    const char *rows[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int row = 4 * i + (lane >> 4);
        const int source = p.order ? source_of(p, *reinterpret_cast<const int *>(lds + wave * L::kWave + spare + 4 * row)) : work.row0 + min(row, work.rows - 1);
        rows[i] = reinterpret_cast<const char *>(p.x + (size_t)source * p.K) + (((lane & 15) ^ (row & 15)) << 4);
    }
    auto fetch_rows = [&](int turn) {
#pragma unroll
        for (int i = 0; i < 8; ++i) load_to_lds_b128(rows[i] + (size_t)group_of(turn) * 256, stage_of(turn) + i * 1024);
    };
    const DequantConsts dq = dequant_consts();
    Tile<1> tile;
    float scale[2] = {0.f, 0.f};
#pragma unroll
    for (int turn = 0; turn < L::kRing - 1; ++turn) fetch_rows(turn);
#pragma unroll 1
    for (int turn = 0; wave + kWaves * turn < G; ++turn) {
        wait_lds_reads();  // the stage before has been read
        const int next = turn + L::kRing - 1;
        fetch_rows(next);
        cols.fetch(group_of(next), stage_of(next) + 32 * 256, stage_of(next) + L::kScales);
        if (turn == 0) wait_vector_loads<(L::kRing - 2) * 8 + LS>();  // (the first stages' words were asked for before all rows)
        else wait_vector_loads<(L::kRing - 1) * LS>();
        const char *stage = lds + wave * L::kWave + (turn % L::kRing) * L::kStage;
        u32x4 w[2][2];
        float by[2];
        cols.read_words(stage + 32 * 256, w);
#pragma unroll
        for (int ni = 0; ni < 2; ++ni) {
            const float next = cols.read_scale(stage + L::kScales, ni);
            by[ni] = scale[ni] * __builtin_amdgcn_rcpf(next);
            scale[ni] = next;
        }
        if (p.Gs != 1) few_rescale<1>(tile, by);
        few_product<1>(stage, w, dq, lane, tile);
    }
    few_rescale<1>(tile, scale);
    wait_vector_loads<0>();
    wait_lds_reads();
    __syncthreads();
    // [wavefront][sub-tile, register][lane]; then wavefront i takes registers 4 i ... 4 i + 3, rows 8 i + 4 h and the three behind
    float *parts = reinterpret_cast<float *>(lds);
#pragma unroll
    for (int ni = 0; ni < 2; ++ni)
#pragma unroll
        for (int r = 0; r < 16; ++r) parts[((wave * 2 + ni) * 16 + r) * 64 + lane] = tile.acc[0][ni][r];
    __syncthreads();
    float sum[2][4];
#pragma unroll
    for (int ni = 0; ni < 2; ++ni)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float *at = parts + (ni * 16 + 4 * wave + r) * 64 + lane;
            sum[ni][r] = ((at[0] + at[2048]) + at[4096]) + at[6144];
        }
#pragma unroll
    for (int r = 0; r < 4; r += 2) {
        const int row = 8 * wave + 4 * h + r + (lane & 1);
        uint16_t *to = p.y + (size_t)(work.row0 + row) * width + column0 + (l32 & 30);
        uint32_t v[2];
        if constexpr (SWIGLU) {
            float y[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) y[i] = sum[0][r + i] * __builtin_amdgcn_rcpf(1.f + __expf(-sum[0][r + i])) * sum[1][r + i];
            v[0] = across_columns(y[0], y[1], lane);
        } else {
#pragma unroll
            for (int ni = 0; ni < 2; ++ni) v[ni] = across_columns(sum[ni][r], sum[ni][r + 1], lane);
        }
        if (row < work.rows)
#pragma unroll
            for (int ni = 0; ni < (SWIGLU ? 1 : 2); ++ni) *reinterpret_cast<uint32_t *>(to + 32 * ni) = v[ni];
    }
}

// 128 rows: the matrix cores bound the loop, and everything else is placed under their products by hand.  A stage is four phases of four
// products, a row tile's each: two column sub-tiles, two k16 steps.
//   * Rows are read a stage ahead, a row tile's right behind its phase.  They are used four phases later, so no product waits for LDS.
//   * Behind phase 0 comes the stage's one barrier: the next stage has landed, and every wavefront holds all of this one, whose place takes
//     the fourth ahead.
//   * The next stage's operands of the pack are expanded half an operand behind a product.
//   * The change of scale goes in fours of registers behind products: of row tiles 0 and 1 in a group's last stage, when their products are done, of
//     2 and 3 in the next group's first, before theirs begin.
template <bool SWIGLU>
__device__ __forceinline__ void experts_many(const ExpertsArgs &p, const Work &work, char *lds, int lane, int wave) {
    constexpr int MI = 4, LA = RowLoads<MI>::kEach, LW = 6;  // loads of a stage's rows, of a group
    using L = ManyLds;
    const Columns<SWIGLU> cols(p, work.expert, work.column * (kColumns / kTileN) + wave * 4, lane, wave * 4096, wave * 256);
    const RowLoads<MI> rows(p.x, p.K, work.rows, wave, lane, [&](int row) { return source_of(p, work, row); });
    const uint32_t sum_off = (uint32_t)source_of(p, work, min(wave * 64 + lane, work.rows - 1)) * 4u;
    const int l32 = lane & 31, h = lane >> 5, G = p.K / kGroupK, stages = p.K / 32;
    const unsigned lds0 = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(lds_ptr_t)lds);
    auto fetch_rows = [&](int stage) {  // past the end: the last one again, so that the count of loads in flight stays what it is
        rows.fetch(min(stage, stages - 1), lds0 + (stage % kStages) * L::kStage);
    };
    auto fetch_group = [&](int g) {
        const int from = min(g, G - 1);
        cols.fetch(from, lds0 + L::kWords + (g & 1) * L::kGroupWords, lds0 + L::kScales + (g & 1) * (kWaves * 256));
        load_to_lds_b32(p.sums + (size_t)from * p.x_rows, sum_off, __builtin_amdgcn_readfirstlane(lds0 + L::kSums + ((g & 1) * kWaves + wave) * 256));
    };
    auto read_rows = [&](int slot, int mi, int step) {
        return *reinterpret_cast<const bf16x8 *>(lds + slot * L::kStage + unit_at(32 * mi + l32, 2 * step + h));
    };
    auto read_words = [&](int g, u32x4(&w)[2][2]) { cols.read_words(lds + L::kWords + (g & 1) * L::kGroupWords, w); };
    auto read_scale = [&](int g, int ni) { return cols.read_scale(lds + L::kScales + (g & 1) * (kWaves * 256), ni); };
    const DequantConsts dq = dequant_consts();
    Tile<MI> tile;
    u32x4 w[2][2];
    float scale[2], by[2] = {1.f, 1.f};
    bf16x8 a[MI][2], b[2][2];
    using std::integral_constant;
    fetch_group(0);
    fetch_group(1);
#pragma unroll
    for (int st = 0; st < kStages; ++st) fetch_rows(st);
    wait_vector_loads<3 * LA>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" : : : "memory");
    read_words(0, w);
#pragma unroll
    for (int ni = 0; ni < 2; ++ni) scale[ni] = read_scale(0, ni);
#pragma unroll
    for (int mi = 0; mi < MI; ++mi)
#pragma unroll
        for (int step = 0; step < 2; ++step) a[mi][step] = read_rows(0, mi, step);
#pragma unroll
    for (int ni = 0; ni < 2; ++ni)
#pragma unroll
        for (int step = 0; step < 2; ++step) b[ni][step] = codes_to_bf16x8(w[ni][step][0], dq);
    auto sums_at = [&](int g, int mi, int quarter) {
        return *reinterpret_cast<const f32x4 *>(lds + L::kSums + (g & 1) * (kWaves * 256) + h * 16 + mi * 128 + quarter * 32);
    };
#pragma unroll
    for (int mi = 0; mi < 2; ++mi)  // the others begin at zero and take theirs in the first stage
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x4 c = sums_at(0, mi, i);
#pragma unroll
            for (int r = 0; r < 4; ++r) tile.acc[mi][0][4 * i + r] = tile.acc[mi][1][4 * i + r] = c[r];
        }
    // items of the change: (row tile, quarter, column sub-tile), 16 of two row tiles, over kRoom products from kFrom on; sums are read kLead products ahead
    constexpr int kItems = 16, kRoom = 10, kFrom = 2, kLead = 2;
    auto group = [&](int g, auto lastc) {
        constexpr bool LAST = decltype(lastc)::value;
        unrolled<0, 4>([&](auto tc) {
            constexpr int t = decltype(tc)::value;
            constexpr bool ahead = !(LAST && t == 3);  // there is a next stage
            u32x4 next[2][2];
            f32x4 c[8];
            if constexpr (t == 3 && !LAST) {  // (this group's last words were expanded a stage ago)
                read_words(g + 1, w);
#pragma unroll
                for (int ni = 0; ni < 2; ++ni) {
                    const float n = read_scale(g + 1, ni);
                    by[ni] = scale[ni] * __builtin_amdgcn_rcpf(n);
                    scale[ni] = n;
                }
            }
            unrolled<0, MI>([&](auto mc) {
                constexpr int mi = decltype(mc)::value;
                unrolled<0, 4>([&](auto jc) {
                    constexpr int j = decltype(jc)::value, ni = j & 1, step = j >> 1, slot = 4 * mi + j;
                    tile.acc[mi][ni] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[mi][step], b[ni][step], tile.acc[mi][ni], 0, 0, 0);
                    // behind this product: halves of the next stage's operands ...
                    constexpr int from = t == 3 ? 4 : 0, room = 16 - from;  // (the next group's words are on their way first)
                    if constexpr (ahead && slot >= from) {
                        unrolled<(slot - from) * 8 / room, (slot - from + 1) * 8 / room>([&](auto hc) {
                            constexpr int half = decltype(hc)::value, en = half >> 1 & 1, es = half >> 2;
                            const uint32_t word = w[en][es][(t + 1) & 3];
                            if constexpr ((half & 1) == 0) {
                                next[en][es].x = (word & dq.mask) | dq.magic;
                                next[en][es].y = (word >> 4 & dq.mask) | dq.magic;
                            } else {
                                next[en][es].z = (word >> 8 & dq.mask) | dq.magic;
                                next[en][es].w = (word >> 12 & dq.mask) | dq.magic;
                            }
                        });
                    }
                    // ... and a part of the change of scale
                    if constexpr ((t == 3 && !LAST) || t == 0) {
                        constexpr int at = slot - (t == 3 ? 4 : 0) - kFrom, first = t == 3 ? 0 : 2;
                        constexpr auto begin_of = [](int i) { return i < 0 ? 0 : i > kRoom ? kItems : i * kItems / kRoom; };
                        unrolled<begin_of(at + kLead), begin_of(at + kLead + 1)>([&](auto ec) {
                            constexpr int e = decltype(ec)::value, quarter = e >> 1;
                            if constexpr ((e & 1) == 0) c[quarter] = sums_at(t == 3 ? g + 1 : g, first + (quarter >> 2), quarter & 3);
                        });
                        unrolled<begin_of(at), begin_of(at + 1)>([&](auto ec) {
                            constexpr int e = decltype(ec)::value, quarter = e >> 1, en = e & 1;
                            f32x16 &acc = tile.acc[first + (quarter >> 2)][en];
#pragma unroll
                            for (int r = 0; r < 4; ++r) acc[4 * (quarter & 3) + r] = fmaf(acc[4 * (quarter & 3) + r], by[en], c[quarter][r]);
                            // c outlives its last use: otherwise that one is written over c's registers, and the tile copied together again
                            if constexpr (en == 1) asm volatile("" : : "v"(c[quarter]));
                        });
                    }
                    __builtin_amdgcn_sched_barrier(0);
                });
                if constexpr (mi == 0) {
                    // The next stage has landed: behind it there are those of two more, and the group that was asked for one or two stages ago.  (At t == 0
                    // that is three stages ago and waited for with it.)
                    wait_vector_loads<2 * LA + (t == 2 || t == 3 ? LW : 0)>();
                    wait_lds_reads();
                    __builtin_amdgcn_s_barrier();
                    asm volatile("" : : : "memory");
                    fetch_rows(4 * g + t + kStages);
                }
                // the next group but one takes this one's places: its words and scales are in registers, its sums were read in the stage before
                if constexpr (mi == 0 && t == 1) fetch_group(g + 2);
                if constexpr (ahead) {
#pragma unroll
                    for (int step = 0; step < 2; ++step) a[mi][step] = read_rows((t + 1) & 3, mi, step);
                    __builtin_amdgcn_sched_barrier(0);
                }
            });
            if constexpr (ahead) {
#pragma unroll
                for (int ni = 0; ni < 2; ++ni)
#pragma unroll
                    for (int step = 0; step < 2; ++step) b[ni][step] = __builtin_bit_cast(bf16x8, next[ni][step]);
            }
        });
    };
    for (int g = 0; g + 1 < G; ++g) group(g, std::false_type{});
    group(G - 1, std::true_type{});
    wait_vector_loads<0>();  // stages asked for past the end still write to LDS
    wait_lds_reads();
    __syncthreads();
    store_tile<MI, SWIGLU>(p, work, lds, lane, wave, tile, scale);
}

// MAX: row tiles of the largest block.  A smaller one -- an expert's last rows -- multiplies no more row tiles than it needs.
template <int MAX, int SETS>
constexpr int kForwardLds = std::max({SETS * FewLds<1>::kBytes, MAX >= 2 ? SETS * FewLds<2>::kBytes : 0, MAX == 4 ? ManyLds::kBytes : 0});
template <int MAX, bool SWIGLU, int SETS>
__global__ __launch_bounds__(SETS * kThreads, 2) void experts_kernel(ExpertsArgs p) {
    extern __shared__ __align__(16) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Work work = find_work<32 * MAX>(p.first, p.experts, p.rows, p.column_blocks, lane);
    if (work.expert < 0) return;
    if (work.expert == p.experts) {
        constexpr int kOut = SWIGLU ? kColumns / 2 : kColumns;
        write_zeros(p.y, SWIGLU ? p.N / 2 : p.N, work.row0, work.rows, work.column * kOut, kOut);
        return;
    }
    if constexpr (MAX == 4) {
        if (work.rows > 64) {
            experts_many<SWIGLU>(p, work, lds, lane, wave);
            return;
        }
    }
    if constexpr (MAX >= 2) {
        if (work.rows > 32) {
            experts_few<2, SWIGLU, SETS>(p, work, lds, lane, wave);
            return;
        }
    }
    experts_few<1, SWIGLU, SETS>(p, work, lds, lane, wave);
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

__device__ __forceinline__ u32x2 turned_codes(unsigned lds_at, int offset) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr4_b64_v2i32((lds_i32x2_ptr_t)(uintptr_t)lds_at + offset / 8));
}
// masks and magic numbers of the codes' expansion, one instruction with both in registers that the compiler cannot see through (as dequant_consts)
struct TurnedConsts {
    uint32_t mask[2], magic[2];
};
__device__ __forceinline__ TurnedConsts turned_consts() {
    TurnedConsts c;
    asm volatile("s_mov_b32 %0, 0x000F000F" : "=s"(c.mask[0]));
    asm volatile("s_mov_b32 %0, 0x00F000F0" : "=s"(c.mask[1]));
    asm volatile("v_mov_b32 %0, 0x64006400" : "=v"(c.magic[0]));
    asm volatile("v_mov_b32 %0, 0x54005400" : "=v"(c.magic[1]));
    return c;
}
// Eight codes of one row of the pack in eight columns, and those columns' scales: half H of an operand's registers, codes 2 H, 2 H + 1 and four on.
// 1024 + code in f16, or 64 + code where the code lies four bits higher, less 1032 or 72, times the scale in f32: exact.
template <int H>
__device__ __forceinline__ void half_of_weights(uint32_t codes, const u32x4 &scales, const TurnedConsts &tc, u32x4 &operand) {
    const f16x2 low = __builtin_bit_cast(f16x2, (uint32_t)scales[H]), high = __builtin_bit_cast(f16x2, (uint32_t)scales[2 + H]);
    float v[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const _Float16 less = (_Float16)(i ? 72.f : 1032.f);
        const f16x2 d = __builtin_bit_cast(f16x2, (codes >> 8 * H & tc.mask[i]) | tc.magic[i]) - f16x2{less, less};
        v[0][i] = fmaf((float)d.x, (float)low[i], 0.f);
        v[1][i] = fmaf((float)d.y, (float)high[i], 0.f);
    }
    operand[H] = pair_of(v[0][0], v[0][1]);
    operand[2 + H] = pair_of(v[1][0], v[1][1]);
}
__device__ __forceinline__ bf16x8 weights_of(uint32_t codes, const u32x4 &scales, const TurnedConsts &tc) {
    u32x4 o;
    half_of_weights<0>(codes, scales, tc, o);
    half_of_weights<1>(codes, scales, tc, o);
    return __builtin_bit_cast(bf16x8, o);
}
// where a lane's row of the pack is in a chunk of its column tile: its column (lane % 16), and of the group's four times eight rows in two runs of 32 those of
// sub-tile ni -- + 512 bytes for ni 1, + 8 for the two runs behind
__device__ __forceinline__ int code_in_chunk(int lane) { return ((lane & 15) + (lane & 16)) * 16; }

// A lane has row l32 of a row tile and of eight consecutive rows of the pack the even ones (lanes 32 ... 63: the odd ones): two such eights change
// hands with the other half, and a lane writes one whole.  Sub-tile ni of 64 columns of the result from column k0 on.
__device__ __forceinline__ void store_eights(uint16_t *row, int k0, int ni, int h, bool live, const f32x16 &acc) {
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        u32x4 o;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float first = acc[8 * b + i], second = acc[8 * b + 4 + i];  // scalar copies: bit-casting an element in place reads element 0
            const auto swapped = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, first), __builtin_bit_cast(unsigned, second), false, false);
            o[i] = pair_of(__builtin_bit_cast(float, (unsigned)swapped[0]), __builtin_bit_cast(float, (unsigned)swapped[1]));
        }
        if (live) *reinterpret_cast<u32x4 *>(row + k0 + 32 * h + 8 * (2 * ni + b)) = o;
    }
}
template <int MI>
__device__ __forceinline__ void store_gradient(const ExpertsArgs &p, const Work &work, int lane, int k0, const Tile<MI> &tile) {
#pragma unroll
    for (int mi = 0; mi < MI; ++mi) {
        const int row = 32 * mi + (lane & 31);
#pragma unroll
        for (int ni = 0; ni < 2; ++ni) store_eights(p.y + (size_t)(work.row0 + row) * p.K, k0, ni, lane >> 5, row < work.rows, tile.acc[mi][ni]);
    }
}

// Up to 64 rows: a stage is 128 columns of the pack, eight column tiles, as in the forward product; one or two more are on their way.
template <int MI, int SETS>
__device__ __forceinline__ void experts_backward_few(const ExpertsArgs &p, const Work &work, char *all_lds, int lane, int wave_of_all) {
    using L = FewLds<MI>;
    const int wave = wave_of_all % kWaves, set = wave_of_all / kWaves;
    char *const lds = all_lds + set * L::kBytes;
    constexpr int LR = 2 * MI, LS = LR + 5;
    const int l32 = lane & 31, h = lane >> 5, G = p.K / kGroupK, tiles = p.N / kTileN, stages = p.N / 128;
    const unsigned lds0 = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(lds_ptr_t)lds);
    const char *rows[LR];
#pragma unroll
    for (int i = 0; i < LR; ++i) {
        const int row = 4 * (wave * LR + i) + (lane >> 4);
        rows[i] = reinterpret_cast<const char *>(p.x + (size_t)(work.row0 + min(row, work.rows - 1)) * p.N) + (((lane & 15) ^ (row & 15)) << 4);
    }
    // the block's two groups: a wavefront fetches four tiles' chunks of one, and the scales of its own half of one
    const int group = min(2 * work.column + (wave >> 1), G - 1), fetched = min(2 * work.column + (wave & 1), G - 1), tile0 = 4 * (wave >> 1);
    const char *const codes = uniform(reinterpret_cast<const char *>(p.b) + (((size_t)work.expert * tiles + tile0) * G + fetched) * 1024);
    const char *const scales = uniform(reinterpret_cast<const char *>(p.s + ((size_t)work.expert * tiles * p.Gs + (p.Gs == 1 ? 0 : group)) * kTileN));
    const uint32_t scale_off = (uint32_t)(lane >> 3) * (uint32_t)p.Gs * (kTileN * 2) + (lane & 7) * 4;
    auto fetch = [&](int turn) {  // past the end: the last one again, so that the count of loads in flight stays what it is
        const int from = min(SETS * turn + set, stages - 1);
        const unsigned to = lds0 + (unsigned)(turn % L::kRing) * L::kStage;
#pragma unroll
        for (int i = 0; i < LR; ++i) load_to_lds_b128(rows[i] + (size_t)from * 256, to + (wave * LR + i) * 1024);
        // chunks [group][tile]
        const unsigned words_to = __builtin_amdgcn_readfirstlane(to + L::kRows + ((wave & 1) * 8 + tile0) * 1024), scales_to = __builtin_amdgcn_readfirstlane(to + L::kScales + wave * 256);
#pragma unroll
        for (int t = 0; t < 4; ++t) load_to_lds_b128(codes + ((size_t)from * 8 + t) * G * 1024, (uint32_t)lane * 16u, words_to + t * 1024);
        load_to_lds_b32(scales + (size_t)from * 8 * p.Gs * (kTileN * 2), scale_off, scales_to);
    };
    const unsigned code_at = L::kRows + (wave >> 1) * 8192 + h * 1024 + code_in_chunk(lane) + 8 * (wave & 1);
    const unsigned scale_at = L::kScales + wave * 256 + h * 32;
    const TurnedConsts tc = turned_consts();
    Tile<MI> tile;
#pragma unroll
    for (int turn = 0; turn < L::kRing - 1; ++turn) fetch(turn);
#pragma unroll 1
    for (int turn = 0; SETS * turn < stages; ++turn) {
        wait_vector_loads<(L::kRing - 2) * LS>();  // this stage has landed
        wait_lds_reads();
        __builtin_amdgcn_s_barrier();  // ... everywhere, and the one before has been read
        asm volatile("" : : : "memory");
        fetch(turn + L::kRing - 1);
        if (SETS > 1 && SETS * turn + set >= stages) break;  // (the last turn of all)
        const unsigned at = (unsigned)(turn % L::kRing) * L::kStage;
        const char *stage = lds + at;
        // k16 steps: a pair of column tiles has two, lanes 32 ... 63 take the second tile.  A step's codes, scales and rows are read two steps ahead and its
        // weights made behind the products of the one before.
        u32x2 c[2][2];
        u32x4 sc[2];
        bf16x8 x[3][MI], w[2][2];
        auto read = [&](auto nc) {
            constexpr int n = decltype(nc)::value, q = n >> 1, u = n & 1;
            if constexpr (u == 0)
#pragma unroll
                for (int ni = 0; ni < 2; ++ni) c[q & 1][ni] = turned_codes(lds0 + at + code_at, q * 2048 + ni * 512);
            sc[u] = *reinterpret_cast<const u32x4 *>(stage + scale_at + q * 64 + 16 * u);
#pragma unroll
            for (int mi = 0; mi < MI; ++mi) x[n % 3][mi] = *reinterpret_cast<const bf16x8 *>(stage + (32 * mi + l32) * 256 + (((4 * q + 2 * h + u) ^ (l32 & 15)) << 4));
        };
        auto make = [&](auto nc) {
            constexpr int n = decltype(nc)::value;
#pragma unroll
            for (int ni = 0; ni < 2; ++ni) w[n & 1][ni] = weights_of(c[n >> 1 & 1][ni][n & 1], sc[n & 1], tc);
        };
        using std::integral_constant;
        read(integral_constant<int, 0>{});
        read(integral_constant<int, 1>{});
        make(integral_constant<int, 0>{});
        __builtin_amdgcn_sched_barrier(0);
        unrolled<0, 8>([&](auto nc) {
            constexpr int n = decltype(nc)::value;
            if constexpr (n + 1 < 8) make(integral_constant<int, n + 1>{});
            if constexpr (n + 2 < 8) read(integral_constant<int, n + 2>{});
#pragma unroll
            for (int ni = 0; ni < 2; ++ni)
#pragma unroll
                for (int mi = 0; mi < MI; ++mi) tile.acc[mi][ni] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w[n & 1][ni], x[n % 3][mi], tile.acc[mi][ni], 0, 0, 0);
            // a product, then vector work, in turn
#pragma unroll
            for (int i = 0; i < 2 * MI; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x2, 48 / (2 * MI), 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        });
    }
    if constexpr (SETS > 1) {
        add_second_set<MI>(all_lds, lane, wave, set, tile);
        if (set == 1) return;
    } else {
        wait_vector_loads<0>();  // stages asked for past the end still write to LDS
    }
    if (2 * work.column + (wave >> 1) < G) store_gradient<MI>(p, work, lane, work.column * kColumns + 64 * wave, tile);  // (a last block of half the columns)
}

// Calls whose blocks would not fill the chip: 32 rows x 128 columns of the result, one scale group, to a block, every fourth 128 of the contraction to a
// wavefront; the sums meet in LDS.
struct SplitBackwardLds {
    static constexpr int kRing = 2, kCodes = 32 * 256, kScales = kCodes + 8192, kStage = kScales + 256, kWave = kRing * kStage, kBytes = kWaves * kWave;
};
__global__ __launch_bounds__(kThreads, 1) void experts_split_backward_kernel(ExpertsArgs p) {
    using L = SplitBackwardLds;
    constexpr int LS = 8 + 8 + 1;
    extern __shared__ __align__(16) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l32 = lane & 31, h = lane >> 5;
    const Work work = find_work<32>(p.first, p.experts, p.rows, p.column_blocks, lane);
    if (work.expert < 0) return;
    const int G = p.K / kGroupK, tiles = p.N / kTileN, stages = p.N / 128, g = work.column;
    if (work.expert == p.experts) {
        write_zeros(p.y, p.K, work.row0, work.rows, g * kGroupK, kGroupK);
        return;
    }
    const unsigned lds0 = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(lds_ptr_t)lds + wave * L::kWave);
    const char *rows[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int row = 4 * i + (lane >> 4);
        rows[i] = reinterpret_cast<const char *>(p.x + (size_t)(work.row0 + min(row, work.rows - 1)) * p.N) + (((lane & 15) ^ (row & 15)) << 4);
    }
    const char *const codes = uniform(reinterpret_cast<const char *>(p.b) + ((size_t)work.expert * tiles * G + g) * 1024);
    const char *const scales = uniform(reinterpret_cast<const char *>(p.s + ((size_t)work.expert * tiles * p.Gs + (p.Gs == 1 ? 0 : g)) * kTileN));
    const uint32_t scale_off = (uint32_t)(lane >> 3) * (uint32_t)p.Gs * (kTileN * 2) + (lane & 7) * 4;
    auto fetch = [&](int turn) {
        const int from = min(wave + kWaves * turn, stages - 1);
        const unsigned to = lds0 + (unsigned)(turn % L::kRing) * L::kStage;
#pragma unroll
        for (int i = 0; i < 8; ++i) load_to_lds_b128(rows[i] + (size_t)from * 256, to + i * 1024);
#pragma unroll
        for (int t = 0; t < 8; ++t) load_to_lds_b128(codes + ((size_t)from * 8 + t) * G * 1024, (uint32_t)lane * 16u, to + L::kCodes + t * 1024);
        load_to_lds_b32(scales + (size_t)from * 8 * p.Gs * (kTileN * 2), scale_off, to + L::kScales);
    };
    const TurnedConsts tc = turned_consts();
    const unsigned code_at = L::kCodes + h * 1024 + code_in_chunk(lane);
    Tile<2> tile;  // [half of the group][sub-tile]
    fetch(0);
#pragma unroll 1
    for (int turn = 0; wave + kWaves * turn < stages; ++turn) {
        wait_lds_reads();  // the stage before has been read
        fetch(turn + 1);
        wait_vector_loads<LS>();
        const unsigned at = (unsigned)(turn % L::kRing) * L::kStage;
        const char *stage = lds + wave * L::kWave + at;
        unrolled<0, 4>([&](auto qc) {
            constexpr int q = decltype(qc)::value;
            u32x2 c[2][2];
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int ni = 0; ni < 2; ++ni)
                    c[half][ni] = turned_codes(lds0 + at + code_at, q * 2048 + ni * 512 + 8 * half);
            unrolled<0, 2>([&](auto uc) {
                constexpr int u = decltype(uc)::value;
                const u32x4 s = *reinterpret_cast<const u32x4 *>(stage + L::kScales + (2 * q + h) * 32 + 16 * u);
                const bf16x8 x = *reinterpret_cast<const bf16x8 *>(stage + l32 * 256 + (((4 * q + 2 * h + u) ^ (l32 & 15)) << 4));
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int ni = 0; ni < 2; ++ni)
                        tile.acc[half][ni] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(weights_of(c[half][ni][u], s, tc), x, tile.acc[half][ni], 0, 0, 0);
            });
        });
    }
    wait_vector_loads<0>();
    wait_lds_reads();
    __syncthreads();
    // [wavefront][half, sub-tile, register][lane]; then wavefront i takes half i / 2, sub-tile i % 2
    float *parts = reinterpret_cast<float *>(lds);
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int ni = 0; ni < 2; ++ni)
#pragma unroll
            for (int r = 0; r < 16; ++r) parts[(((wave * 2 + half) * 2 + ni) * 16 + r) * 64 + lane] = tile.acc[half][ni][r];
    __syncthreads();
    f32x16 sum;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const float *from = parts + (wave * 16 + r) * 64 + lane;
        sum[r] = ((from[0] + from[4096]) + from[8192]) + from[12288];
    }
    store_eights(p.y + (size_t)(work.row0 + l32) * p.K, g * kGroupK + 64 * (wave >> 1), wave & 1, h, l32 < work.rows, sum);
}

// 128 rows: four phases of four products to a stage of 32 columns, as experts_many, with the next stage's operands of the pack made behind the products.  Their
// codes and scales are read from LDS a stage before that, so a stage has landed two stages ahead of its products.
struct ManyBackwardLds {
    static constexpr int kRing = 6, kCodes = 128 * kRowBytes, kScales = kCodes + 4 * 1024, kStage = kScales + kWaves * 256, kBytes = kRing * kStage;
};
__device__ __forceinline__ void experts_backward_many(const ExpertsArgs &p, const Work &work, char *lds, int lane, int wave) {
    using L = ManyBackwardLds;
    constexpr int MI = 4, LS = RowLoads<MI>::kEach + 2;
    const int l32 = lane & 31, h = lane >> 5, G = p.K / kGroupK, tiles = p.N / kTileN, stages = p.N / 32;
    const RowLoads<MI> rows(p.x, p.N, work.rows, wave, lane, [&](int row) { return work.row0 + row; });
    // of a stage's four chunks -- two tiles, two groups -- a wavefront fetches one; of the scales what it multiplies with
    const int group = min(2 * work.column + (wave >> 1), G - 1), fetched = min(2 * work.column + (wave & 1), G - 1);
    const char *const codes = uniform(reinterpret_cast<const char *>(p.b) + (((size_t)work.expert * tiles + (wave >> 1)) * G + fetched) * 1024);
    const char *const scales = uniform(reinterpret_cast<const char *>(p.s + ((size_t)work.expert * tiles * p.Gs + (p.Gs == 1 ? 0 : group)) * kTileN));
    const uint32_t scale_off = (uint32_t)(lane >> 3 & 1) * (uint32_t)p.Gs * (kTileN * 2) + (lane & 7) * 4;
    const unsigned lds0 = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(lds_ptr_t)lds);
    auto fetch = [&](int stage, unsigned at) {  // past the end: the last one again, so that the count of loads in flight stays what it is
        const int from = min(stage, stages - 1);
        rows.fetch(from, lds0 + at);
        load_to_lds_b128(codes + (size_t)from * 2 * G * 1024, (uint32_t)lane * 16u, __builtin_amdgcn_readfirstlane(lds0 + at + L::kCodes + wave * 1024));
        load_to_lds_b32(scales + (size_t)from * 2 * p.Gs * (kTileN * 2), scale_off, __builtin_amdgcn_readfirstlane(lds0 + at + L::kScales + wave * 256));
    };
    const unsigned code_at = L::kCodes + (2 * h + (wave >> 1)) * 1024 + code_in_chunk(lane) + 8 * (wave & 1), scale_at = L::kScales + wave * 256 + h * 32;
    const TurnedConsts tc = turned_consts();
    Tile<MI> tile;
    bf16x8 x[MI][2], w[2][2];  // w: [ni][u]
    u32x2 c[2];
    u32x4 s;
    auto read_rows = [&](unsigned at, int mi) {
#pragma unroll
        for (int u = 0; u < 2; ++u) x[mi][u] = *reinterpret_cast<const bf16x8 *>(lds + at + unit_at(32 * mi + l32, 2 * h + u));
    };
    auto read_scales = [&](unsigned at, int u) { s = *reinterpret_cast<const u32x4 *>(lds + at + scale_at + 16 * u); };
    auto read_codes = [&](unsigned at) {
#pragma unroll
        for (int ni = 0; ni < 2; ++ni) c[ni] = turned_codes(lds0 + at + code_at, 512 * ni);
        read_scales(at, 0);
    };
#pragma unroll
    for (int st = 0; st < L::kRing; ++st) fetch(st, st * L::kStage);
    wait_vector_loads<(L::kRing - 2) * LS>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" : : : "memory");
    read_codes(0);
#pragma unroll
    for (int mi = 0; mi < MI; ++mi) read_rows(0, mi);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        if (u) read_scales(0, 1);
#pragma unroll
        for (int ni = 0; ni < 2; ++ni) w[ni][u] = weights_of(c[ni][u], s, tc);
    }
    read_codes(L::kStage);
    unsigned at = 0;  // this stage's place
    auto behind = [&](unsigned place, int stages_on) {
        const unsigned next = place + stages_on * L::kStage;
        return next < (unsigned)L::kBytes ? next : next - L::kBytes;
    };
#pragma unroll 1
    for (int st = 0; st < stages; ++st) {
        const unsigned next = behind(at, 1), after = behind(at, 2);
        u32x4 made[2][2];
        unrolled<0, MI>([&](auto mc) {
            constexpr int mi = decltype(mc)::value;
            unrolled<0, 4>([&](auto jc) {
                constexpr int j = decltype(jc)::value, ni = j & 1, u = j >> 1, slot = 4 * mi + j;
                tile.acc[mi][ni] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w[ni][u], x[mi][u], tile.acc[mi][ni], 0, 0, 0);
                // behind two products of three half an operand of the next stage: four of its first k16 step, then with the scales of the other that one's
                if constexpr ((slot >= 1 && slot < 7 && slot % 3 != 0) || (slot >= 10 && slot < 16 && slot % 3 != 0)) {
                    constexpr int eu = slot >= 10, half = eu ? (slot - 10) / 3 * 2 + (slot - 10) % 3 : (slot - 1) / 3 * 2 + (slot - 1) % 3;
                    half_of_weights<(half & 1)>(c[half >> 1][eu], s, tc, made[half >> 1][eu]);
                }
                if constexpr (slot == 6) read_scales(next, 1);
                __builtin_amdgcn_sched_barrier(0);
            });
            if constexpr (mi == 0) {
                wait_vector_loads<3 * LS>();  // the next stage but one has landed: behind it there are those of three more
                wait_lds_reads();
                __builtin_amdgcn_s_barrier();
                asm volatile("" : : : "memory");
                fetch(st + L::kRing, at);  // every wavefront has this stage's rows in registers, and the next one's codes
            }
            read_rows(next, mi);
            if constexpr (mi == MI - 1) read_codes(after);
            __builtin_amdgcn_sched_barrier(0);
        });
#pragma unroll
        for (int ni = 0; ni < 2; ++ni)
#pragma unroll
            for (int u = 0; u < 2; ++u) w[ni][u] = __builtin_bit_cast(bf16x8, made[ni][u]);
        at = next;
    }
    wait_vector_loads<0>();  // stages asked for past the end still write to LDS
    if (2 * work.column + (wave >> 1) < G) store_gradient<MI>(p, work, lane, work.column * kColumns + 64 * wave, tile);  // (a last block of half the columns)
}

template <int MAX, int SETS>
constexpr int kBackwardLds = std::max({SETS * FewLds<1>::kBytes, MAX >= 2 ? SETS * FewLds<2>::kBytes : 0, MAX == 4 ? ManyBackwardLds::kBytes : 0});
template <int MAX, int SETS>
__global__ __launch_bounds__(SETS * kThreads, 2) void experts_backward_kernel(ExpertsArgs p) {
    extern __shared__ __align__(16) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Work work = find_work<32 * MAX>(p.first, p.experts, p.rows, p.column_blocks, lane);
    if (work.expert < 0) return;
    if (work.expert == p.experts) {
        write_zeros(p.y, p.K, work.row0, work.rows, work.column * kColumns, min(kColumns, p.K - work.column * kColumns));
        return;
    }
    if constexpr (MAX == 4) {
        if (work.rows > 64) {
            experts_backward_many(p, work, lds, lane, wave);
            return;
        }
    }
    if constexpr (MAX >= 2) {
        if (work.rows > 32) {
            experts_backward_few<2, SETS>(p, work, lds, lane, wave);
            return;
        }
    }
    experts_backward_few<1, SETS>(p, work, lds, lane, wave);
}

// ---- launches ------------------------------------------------------------------------------------------------------
// The most row tiles that rows sorted by expert can take: a part tile to every expert that has rows, and to the rows without one
int64_t most_tiles(int rows, int experts, int block_rows) {
    return (int64_t)rows / block_rows + std::min<int64_t>((int64_t)experts + 1, rows);
}
// Which blocks a call takes, from what 128 of the contraction cost a block, us: `alone` on its compute unit, or `busy` where compute units have several (two side
// by side take nearly twice as long: what they have to issue bounds them, not what they wait for; an eighth longer again where every one has two blocks of up to 64
// rows, which load more to a product); `rest` of a block to an expert for its last rows, `least` of one to an expert of few; `launch` of the rows' sums, or of the
// sets' exchange.  An expert with rows has a block to each column block, whatever it costs.  Experts of up to 32 rows, and of up to 64, run the same code in every
// block that takes them, so what those cost agrees: `few`, and `busy` times `least`.  In the forward product the 128-row kernel has a launch in front beside, for
// nothing where no expert has more than 64 rows (64 experts, 2560 -> 2048, 40 rows 24 us and 22; 8 experts, 4096 -> 28672, 200 rows 165 and 135).
// us a call of blocks of 32 rows / 64 / 128, of 32 and 64 rows with two sets of wavefronts, and split:
//   forward    400 rows of 16 experts, 2560 -> 2048   24 /  29 /  36,   21 /  27,   28      800 of 32, 1280 -> 2048   20 /  21 /  23,  26 /  23,  36
//              400 rows of  4 experts, 2560 -> 1024   22 /  28 /  39,   20 /  26,   10     4000 of 64, 2560 -> 1024   53 /  44 /  59,  60 /  50,  91
//             3000 rows of 64 experts, 2560 -> 2048   74 /  75 /  76,   86 /  76,  137     3000 of  8,  384 ->  256    7 /   8 /  12,   7 /   8,   9
//             8000 rows of 64 experts, 2560 -> 2048  154 / 123 / 116,  189 / 139,  300    10000 of 16,  768 -> 1536   46 /  34 /  38,  66 /  45, 146
//            16384 rows of 64 experts, 2560 -> 2048  285 / 219 / 195,  348 / 251,  565     3000 of  2, 2560 -> 2048   52 /  48 /  44,  60 /  53, 108
//   gradient   400 rows of 16 experts, 2560 <- 2048   22 /  24 /  30,   21 /  23,   24      400 of 16,  768 <-  768   10 /  11 /  13,  10 /  11,   8
//             2331 rows of 24 experts, 1280 <- 2048   33 /  25 /  39,   38 /  25,   45     6000 of 32, 2048 <-  768   47 /  36 /  35,  66 /  45,  91
//             3000 rows of 64 experts, 2560 <- 2048   85 /  77 /  81,  107 /  90,  120     5900 of 28,  256 <- 1536   18 /  19 /  30,  17 /  18,  20
//            16384 rows of 64 experts, 2560 <- 2048  329 / 230 / 209,  412 / 270,  466
// (rows spread over the experts by weights of exp(normal / 2); in equal parts the 16384 rows take 266 / 198 / 167 and 313 / 211 / 187.)
// (The costs were fitted to 38 such sizes with their rows spread evenly and unevenly over the experts, packs in turn so that they come from memory, where what is
// chosen is within 1 % of the best on average, 15 % off at the worst; on 120 others, from 2 rows in all to 4000 of one expert, 2 %, and 49 % at the worst: the gradient of 16
// rows of 16 experts, 2560 <- 9216, 68, in split blocks, which would take two rounds, 46.)
// Two sets and split blocks are one to a compute unit (LDS) and taken where one round of them does.
enum class Blocks { kSplit, kOneTile, kTwoTiles, kFourTiles, kOneTileTwoSets, kTwoTilesTwoSets };
struct BlockCost {
    Blocks blocks;
    int rows;
    float alone, few, busy, rest, least, launch;  // few: alone, and up to kFewEach rows to an expert;  busy 0: one to a compute unit at most
};
constexpr float kFewEach = 24.f;  // (128-row blocks: a third, as an expert in 32 may have four times the rows of another, and one of more than 64 takes twice as long there)
Blocks choose_blocks(const BlockCost (&costs)[5], int rows, int experts, int contraction, int column_blocks, int split_columns, int cus) {
    const float present = (float)std::min(rows, experts), each = rows / present, groups = contraction / 128.f;
    if (present * std::max(1.f, each / 32 + 0.5f) * split_columns <= 1.05f * cus) return Blocks::kSplit;
    const BlockCost *best = nullptr;
    float least = 0.f;
    for (const BlockCost &c : costs) {
        const bool tall = c.rows == 128;
        if (tall && rows <= 64) continue;  // (what they are for needs an expert of more)
        const float blocks = each / c.rows + c.rest, share = present * std::max(c.least, blocks) * column_blocks / cus;
        float count = present * std::max(1.f, blocks) * column_blocks / cus;  // of blocks, to a compute unit
        // where one round is taken for all there is, a block too many takes a second: an expert in 32 may have four times the rows of another
        if ((tall || c.busy == 0.f) && each * 4 > c.rows) count += present / 32 * column_blocks / cus;
        if (c.busy == 0.f && count > 1.f) continue;
        const float side_by_side = tall ? 2.f : std::min(1.75f + share / 4, 2.25f);
        const float time = groups * (count > 1.f ? c.busy * std::max(share, side_by_side) : each <= (tall ? kFewEach / 3 : kFewEach) ? c.few : c.alone) + c.launch;
        if (!best || time < least) {
            best = &c;
            least = time;
        }
    }
    return best->blocks;
}
// (of equals the larger: an expert with more rows than others then takes no second block)
constexpr BlockCost kForwardCosts[5] = {{Blocks::kFourTiles, 128, 1.9f, 0.84f, 1.59f, 0.26f, 0.63f, 3.5f},  // (its rows' sums are a launch)
                                        {Blocks::kTwoTiles, 64, 1.37f, 0.84f, 1.f, 0.3f, 1.f, 0.f},
                                        {Blocks::kOneTile, 32, 0.84f, 0.84f, 1.f, 0.53f, 1.f, 0.f},
                                        {Blocks::kTwoTilesTwoSets, 64, 1.25f, 0.71f, 0.f, 0.3f, 1.f, 1.f},
                                        {Blocks::kOneTileTwoSets, 32, 0.71f, 0.71f, 0.f, 0.53f, 1.f, 1.f}};
constexpr BlockCost kGradientCosts[5] = {{Blocks::kFourTiles, 128, 3.05f, 1.16f, 2.2f, 0.41f, 0.62f, 0.f},
                                         {Blocks::kTwoTiles, 64, 1.54f, 1.16f, 1.36f, 0.3f, 1.f, 0.f},
                                         {Blocks::kOneTile, 32, 1.16f, 1.16f, 1.36f, 0.5f, 1.f, 0.f},
                                         {Blocks::kTwoTilesTwoSets, 64, 1.3f, 0.98f, 0.f, 0.3f, 1.f, 1.f},
                                         {Blocks::kOneTileTwoSets, 32, 0.99f, 0.99f, 0.f, 0.5f, 1.f, 1.f}};
Blocks forward_blocks(int rows, int n, int k, int experts, int cus) { return choose_blocks(kForwardCosts, rows, experts, k, n / kColumns, n / 64, cus); }
Blocks gradient_blocks(int rows, int n, int k, int experts, int cus) {
    return choose_blocks(kGradientCosts, rows, experts, n, (k + kColumns - 1) / kColumns, k / kGroupK, cus);
}
int rows_of(Blocks blocks) { return blocks == Blocks::kFourTiles ? 128 : blocks == Blocks::kTwoTiles || blocks == Blocks::kTwoTilesTwoSets ? 64 : 32; }
int threads_of(Blocks blocks) { return blocks == Blocks::kOneTileTwoSets || blocks == Blocks::kTwoTilesTwoSets ? 2 * kThreads : kThreads; }
int forward_columns(Blocks blocks, int n) { return blocks == Blocks::kSplit ? n / 64 : n / kColumns; }
int gradient_columns(Blocks blocks, int k) { return blocks == Blocks::kSplit ? k / kGroupK : (k + kColumns - 1) / kColumns; }
// (Eight blocks more: a die's shares of both lists may be rounded up.)
int64_t blocks_of(Blocks blocks, int rows, int experts, int column_blocks) { return most_tiles(rows, experts, rows_of(blocks)) * column_blocks + 8; }
bool one_launch(Blocks blocks, int rows, int experts, int column_blocks) {
    return launchable(blocks_of(blocks, rows, experts, column_blocks), threads_of(blocks));
}
template <auto Kernel>
bool launch(const ExpertsArgs &a, Blocks blocks, int lds_bytes, hipStream_t stream) {
    if (allow_dynamic_lds<Kernel>(lds_bytes) != hipSuccess) return false;
    Kernel<<<(unsigned)blocks_of(blocks, a.rows, a.experts, a.column_blocks), threads_of(blocks), lds_bytes, stream>>>(a);
    return true;
}

kiln_marlin_status_t experts_ok(int rows, int n, int k, int experts, int groupsize) {
    if (rows < 0 || n <= 0 || k <= 0 || n % 256 != 0 || k % 128 != 0 || (groupsize != -1 && groupsize != 128)) return KILN_W4A16_ERR_PROB_SHAPE;
    if (experts < 1 || experts > kMaxExperts) return KILN_W4A16_ERR_KERN_SHAPE;
    return most_tiles(rows, experts, 32) * (std::max((int64_t)n, (int64_t)k) / 64 + 1) > INT32_MAX - 8 ? KILN_W4A16_ERR_KERN_SHAPE : KILN_W4A16_OK;
}
// what a call reads of the packs and the order
Piece pack_of(const void *b, int n, int k, int experts) { return {b, (size_t)experts * k * n / 2}; }
Piece scales_of(const void *s, int n, int k, int experts, int groupsize) { return {s, (size_t)experts * (groupsize == -1 ? 1 : k / kGroupK) * n * 2}; }

}  // namespace
}  // namespace kiln

using namespace kiln;

extern "C" {

size_t kiln_w4a16_gemm_experts_scratch_bytes(int x_rows, int prob_k) {
    return x_rows < 1 || prob_k < kGroupK ? 256 : ((size_t)x_rows * (prob_k / kGroupK) * sizeof(float) + 255) & ~(size_t)255;
}

kiln_marlin_status_t kiln_w4a16_gemm_experts(const void *x, const int *first, const int *order, const void *b, const void *s, void *y, int rows, int x_rows,
                                             int top_k, int prob_n, int prob_k, int experts, int groupsize, int swiglu, int dev, void *stream, void *scratch) {
    if (const kiln_marlin_status_t st = experts_ok(rows, prob_n, prob_k, experts, groupsize)) return st;
    if (x_rows < 0 || top_k < 1 || (order ? (int64_t)x_rows * top_k != rows : x_rows != rows)) return KILN_W4A16_ERR_KERN_SHAPE;
    const int64_t items = (int64_t)x_rows * (prob_k / kGroupK);
    if (x_rows > kMaxRows || !launchable((items + 15) / 16, 256)) return KILN_W4A16_ERR_KERN_SHAPE;
    if (rows == 0) return KILN_W4A16_OK;
    const Blocks blocks = forward_blocks(rows, prob_n, prob_k, experts, compute_units(dev));
    const int column_blocks = forward_columns(blocks, prob_n);
    if (!one_launch(blocks, rows, experts, column_blocks)) return KILN_W4A16_ERR_KERN_SHAPE;
    if (!all_on(16, {x, b, s, y, scratch}) || !all_on(4, {first}) || reinterpret_cast<uintptr_t>(order) % 4 != 0) return KILN_W4A16_ERR_ARGUMENT;
    const size_t width = swiglu ? prob_n / 2 : prob_n;
    if (any_meet({{y, rows * width * 2}, {scratch, kiln_w4a16_gemm_experts_scratch_bytes(x_rows, prob_k)}},
                 {{x, (size_t)x_rows * prob_k * 2}, {first, ((size_t)experts + 1) * 4}, {order, (size_t)rows * 4}, pack_of(b, prob_n, prob_k, experts),
                  scales_of(s, prob_n, prob_k, experts, groupsize)}))
        return KILN_W4A16_ERR_ARGUMENT;
    hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
    if (blocks == Blocks::kFourTiles) {
        expert_row_sums_kernel<<<(unsigned)((items + 15) / 16), 256, 0, hs>>>((const uint16_t *)x, (float *)scratch, x_rows, prob_k);
    }
    ExpertsArgs a{(const uint16_t *)x, first, order, (const u32x4 *)b, (const uint16_t *)s, (uint16_t *)y, (const float *)scratch,
                  rows, x_rows, top_k, experts, prob_k, prob_n, groupsize == -1 ? 1 : prob_k / kGroupK, column_blocks};
    bool ok = false;
    auto with = [&](auto mc, auto sc) {
        constexpr int MI = decltype(mc)::value, SETS = decltype(sc)::value;
        ok = swiglu ? launch<experts_kernel<MI, true, SETS>>(a, blocks, kForwardLds<MI, SETS>, hs)
                    : launch<experts_kernel<MI, false, SETS>>(a, blocks, kForwardLds<MI, SETS>, hs);
    };
    using std::integral_constant;
    switch (blocks) {
        case Blocks::kSplit:
            ok = swiglu ? launch<experts_split_kernel<true>>(a, blocks, SplitLds::kBytes, hs) : launch<experts_split_kernel<false>>(a, blocks, SplitLds::kBytes, hs);
            break;
        case Blocks::kOneTile: with(integral_constant<int, 1>{}, integral_constant<int, 1>{}); break;
        case Blocks::kTwoTiles: with(integral_constant<int, 2>{}, integral_constant<int, 1>{}); break;
        case Blocks::kFourTiles: with(integral_constant<int, 4>{}, integral_constant<int, 1>{}); break;
        case Blocks::kOneTileTwoSets: with(integral_constant<int, 1>{}, integral_constant<int, 2>{}); break;
        case Blocks::kTwoTilesTwoSets: with(integral_constant<int, 2>{}, integral_constant<int, 2>{}); break;
    }
    return ok && hipGetLastError() == hipSuccess ? KILN_W4A16_OK : KILN_W4A16_ERR_LAUNCH;
}

kiln_marlin_status_t kiln_w4a16_gemm_experts_backward(const void *dy, const int *first, const void *b, const void *s, void *dx, int rows, int prob_n, int prob_k,
                                                      int experts, int groupsize, int dev, void *stream) {
    if (const kiln_marlin_status_t st = experts_ok(rows, prob_n, prob_k, experts, groupsize)) return st;
    if (rows == 0) return KILN_W4A16_OK;
    const Blocks blocks = gradient_blocks(rows, prob_n, prob_k, experts, compute_units(dev));
    const int column_blocks = gradient_columns(blocks, prob_k);
    if (!one_launch(blocks, rows, experts, column_blocks)) return KILN_W4A16_ERR_KERN_SHAPE;
    if (!all_on(16, {dy, b, s, dx}) || !all_on(4, {first})) return KILN_W4A16_ERR_ARGUMENT;
    if (any_meet({{dx, (size_t)rows * prob_k * 2}}, {{dy, (size_t)rows * prob_n * 2}, {first, ((size_t)experts + 1) * 4}, pack_of(b, prob_n, prob_k, experts),
                                                     scales_of(s, prob_n, prob_k, experts, groupsize)}))
        return KILN_W4A16_ERR_ARGUMENT;
    hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
    ExpertsArgs a{(const uint16_t *)dy, first, nullptr, (const u32x4 *)b, (const uint16_t *)s, (uint16_t *)dx, nullptr,
                  rows, rows, 1, experts, prob_k, prob_n, groupsize == -1 ? 1 : prob_k / kGroupK, column_blocks};
    bool ok = false;
    auto with = [&](auto mc, auto sc) {
        constexpr int MI = decltype(mc)::value, SETS = decltype(sc)::value;
        ok = launch<experts_backward_kernel<MI, SETS>>(a, blocks, kBackwardLds<MI, SETS>, hs);
    };
    using std::integral_constant;
    switch (blocks) {
        case Blocks::kSplit:
            ok = launch<experts_split_backward_kernel>(a, blocks, SplitBackwardLds::kBytes, hs);
            break;
        case Blocks::kOneTile: with(integral_constant<int, 1>{}, integral_constant<int, 1>{}); break;
        case Blocks::kTwoTiles: with(integral_constant<int, 2>{}, integral_constant<int, 1>{}); break;
        case Blocks::kFourTiles: with(integral_constant<int, 4>{}, integral_constant<int, 1>{}); break;
        case Blocks::kOneTileTwoSets: with(integral_constant<int, 1>{}, integral_constant<int, 2>{}); break;
        case Blocks::kTwoTilesTwoSets: with(integral_constant<int, 2>{}, integral_constant<int, 2>{}); break;
    }
    return ok && hipGetLastError() == hipSuccess ? KILN_W4A16_OK : KILN_W4A16_ERR_LAUNCH;
}

int kiln_w4a16_debug_experts_plan(int rows, int prob_n, int prob_k, int experts, int backward, int cus) {
    if (experts_ok(rows, prob_n, prob_k, experts, 128) != KILN_W4A16_OK || rows < 1 || cus < 1) return -1;
    const Blocks blocks = backward ? gradient_blocks(rows, prob_n, prob_k, experts, cus) : forward_blocks(rows, prob_n, prob_k, experts, cus);
    return one_launch(blocks, rows, experts, backward ? gradient_columns(blocks, prob_k) : forward_columns(blocks, prob_n)) ? (int)blocks : -1;
}

}  // extern "C"
