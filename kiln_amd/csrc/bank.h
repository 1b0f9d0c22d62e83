// What the calls on a bank of adapters share: the order of their rows, and the product of the rows with their own adapters' matrices.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "kiln_w4a16.h"

namespace kiln {

constexpr int kBankMaxRank = 64;
constexpr int kBankRowTile = 16;
// Calls of fewer rows take them as they stand.  Rank 16, us a call as they stand / in order: 32 adapters, rows mixed, 128 / 256 / 300 / 400 rows
// 2560 -> 18432 50.2 / 54.7, 72.1 / 61.2, 77.1 / 62.0, 98.3 / 71.9; 9216 -> 2560 33.9 / 45.6, 52.3 / 50.9, 57.5 / 53.4, 73.0 / 57.7; 5120 -> 5120
// 32.9 / 44.7, 47.8 / 46.2, 52.8 / 49.1, 73.6 / 61.9; 2560 -> 2560 19.6 / 34.4, 25.4 / 33.6, 26.1 / 33.4, 36.0 / 37.9.  Four adapters, each one's
// rows together, lose by order up to 400 rows of narrow outputs (5120 -> 5120 at 300 39.7 / 45.6) and gain beyond 300 on wide ones.
constexpr int kBankOrderedFrom = 257;
constexpr int kBankMaxSlices = 32;     // of the contraction of a projection

// do [a, a + a_bytes) and [b, b + b_bytes) share memory?
inline bool meet(const void *a, size_t a_bytes, const void *b, size_t b_bytes) {
    const uintptr_t i = reinterpret_cast<uintptr_t>(a), j = reinterpret_cast<uintptr_t>(b);
    return i < j + b_bytes && j < i + a_bytes;
}

// `groups` in at most `most` slices of the same number of groups, the last one's perhaps fewer: as many as none is left empty
inline int bank_level_slices(int groups, int most) {
    const int each = (groups + most - 1) / most;
    return (groups + each - 1) / each;
}

inline size_t bank_up256(size_t bytes) { return (bytes + 255) & ~(size_t)255; }

// The rows of a call by position: position p is row order[p] (p itself without `order`), rows of one adapter together.
// first[a] .. first[a + 1] are adapter a's positions, those of rows without an adapter come last.
struct BankRows {
    const int *of;      // [rows] adapter of a row; outside [0, count): none
    int *order;         // [rows], or null
    int *first;         // [count + 2], or null
    int rows, count;
};

bool bank_ok(const kiln_w4a16_adapter_bank &bank);
size_t bank_order_bytes(int rows, int count);
BankRows bank_rows(const int *of, int rows, int count, void *at);  // with order and first in bank_order_bytes of scratch from `at` on

// how a call on a bank goes, and the slices of K that its projection is cut into
enum class BankMethod { kOneLaunch, kBase, kBehind, kInProduct };
struct BankPlan {
    BankMethod method;
    int slices;
};
BankPlan bank_plan(int m, int n, int k, int rank, int cus);
// slices of K that a projection of `rows` rows is cut into in a launch of its own
int bank_slices(int rows, int K);
size_t bank_projected_rows(int rows, int K);  // slices * rows of any plan for up to `rows` rows
// t[slice][position][rank] = the slice's share of src[row, K] * mat[adapter of row][rank, K]^T, f32; positions without an adapter are not written
struct BankProjection {
    const void *src, *mat;
    float *t;
    int K, slices;
};
// Rows put in order beside a projection, for gemm_with_bank: x[row, K] to ordered[position, K], sums[K / 128][position] and adapters[position] (-1: none)
struct BankGather {
    const uint16_t *x;
    uint16_t *ordered;
    float *sums;
    int *adapters;
    int K, blocks;
};
void bank_project(const BankProjection &one, const BankProjection *two, const BankRows &r, int rank, hipStream_t stream, BankGather gather = {});

// up to 16 rows as they stand: y = x W, and their projection (bank_base_slices of it) in the same launch
constexpr int kBankFewRows = 16;
int bank_base_slices(int K);
void bank_base(const void *x, const void *b, const void *s, void *y, const BankProjection &of_x, const BankRows &rows, int rank, int K, int N, bool per_column, int cus,
               hipStream_t stream);
// ... or a row or two with their low-rank term in one launch
bool bank_projects_itself(int m, int n, int k, int rank);
void bank_few(const void *x, const void *b, const void *s, void *y, const kiln_w4a16_adapter_bank &bank, const BankRows &rows, int K, int N, bool per_column,
              hipStream_t stream);

// many rows: the plain GEMM with a bank's term in it (launch.h), for the sizes where it can
struct PrefillBank;
bool bank_in_product(int m, int n, int k, int cus);
// A: rows in the order of their adapters; row_sums: -136 times their sums, f32 [K/128][m]
kiln_marlin_status_t gemm_with_bank(const void *A, const void *B, void *C, const void *s, int m, int n, int k, void *workspace, int groupsize, int dev,
                                    void *stream, float *row_sums, const PrefillBank &bank);

}  // namespace kiln
