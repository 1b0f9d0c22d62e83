// silu(gate) * up in training: what the backward pass needs of gate and up is kept in 8 bits.
//   forward   h = silu(gate) * up from bf16 gate and up, 8 columns of one and the 8 matching ones of the other (the packed column order of
//             kiln_w4a16_gemm_swiglu), and beside it gate and up as 8-bit whole numbers sharing a power of two in blocks of 32 gate values
//             or 32 up values: 2.06 bytes for an (h, gate, up) where bf16 takes four
//   backward  with s = 1 / (1 + exp(-gate)):  d_up = dh gate s,  d_gate = dh up s (1 + gate (1 - s)),  and h again if asked for
// The reference keeps or recomputes bf16 gate and up (crates/kiln-model/src/forward.rs:2771-2819 is the forward it differentiates).
//
// A power of two instead of largest / 127: dividing by it and multiplying with it are exact, so the only rounding is to the whole number, at
// most 2^-7 of the block's largest magnitude (2^-8 where that is just below a power of two), and what is read back is a bf16 value.
// Bound by memory, every byte read and written once.  A lane takes 8 gate and 8 up values, two 16-byte pieces; four lanes have a block of
// each and meet in two exchanges inside the vector unit.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "device_common.h"
#include "kiln_w4a16.h"
#include "launch.h"
#include "pieces.h"

namespace kiln {
namespace {

constexpr int kNoNumber = 255;  // the exponent of a block that holds an infinity or NaN: it is read back as NaN

template <int CTRL>
__device__ __forceinline__ uint32_t from_quad(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true);
}
// the largest of four lanes
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
    v = max(v, from_quad<0xB1>(v));
    return max(v, from_quad<0x4E>(v));
}
__device__ __forceinline__ float half_of(const u32x4 &v, int i) {
    return __builtin_bit_cast(float, i & 1 ? v[i >> 1] & 0xFFFF0000u : v[i >> 1] << 16);
}
// biased exponent of the block's largest magnitude, at least 1
__device__ __forceinline__ int block_exponent(const u32x4 &v) {
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) most = max(most, max(v[i] & 0x7FFFu, v[i] >> 16 & 0x7FFFu));
    return max(1, (int)(quad_max(most) >> 7));
}
// value = whole * 2^(exponent - 127 - 6)
__device__ __forceinline__ u32x2 to_whole(const u32x4 &v, int exponent) {
    uint32_t o[2] = {0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float w = fminf(fmaxf(__builtin_rintf(__builtin_amdgcn_ldexpf(half_of(v, i), 133 - exponent)), -127.f), 127.f);
        o[i >> 2] |= ((uint32_t)(int)w & 0xFFu) << (8 * (i & 3));
    }
    if (exponent == kNoNumber) o[0] = o[1] = 0u;
    return u32x2{o[0], o[1]};
}
__device__ __forceinline__ float from_whole(uint32_t word, int i, int exponent) {
    const float v = __builtin_amdgcn_ldexpf((float)((int)(word << (24 - 8 * i)) >> 24), exponent - 133);
    return exponent == kNoNumber ? __builtin_nanf("") : v;
}
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pair_of(float low, float high) { return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)low, (__bf16)high}); }

struct KeepArgs {
    const u32x4 *gate_up;   // [rows, n / 8, 2] pieces of eight
    const u32x4 *dh;        // [rows, n / 8]
    u32x4 *whole;           // [rows, n / 8]: eight of gate, eight of up
    uint16_t *exponents;    // [rows, n / 32]: gate's, up's
    u32x4 *h, *d_gate_up;
    size_t pieces;          // rows * n / 8
};

__global__ __launch_bounds__(256) void swiglu_keep_kernel(KeepArgs p) {
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= p.pieces) return;  // (a row is a multiple of 16 pieces: whole blocks of four lanes)
    const u32x4 gate = p.gate_up[2 * i], up = p.gate_up[2 * i + 1];
    const int eg = block_exponent(gate), eu = block_exponent(up);
    const u32x2 wg = to_whole(gate, eg), wu = to_whole(up, eu);
    p.whole[i] = u32x4{wg.x, wg.y, wu.x, wu.y};
    if ((i & 3) == 0) p.exponents[i >> 2] = (uint16_t)(eg | eu << 8);
    u32x4 h;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float v[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const float g = half_of(gate, 2 * e + b);
            v[b] = g * __builtin_amdgcn_rcpf(1.f + __expf(-g)) * half_of(up, 2 * e + b);
        }
        h[e] = pair_of(v[0], v[1]);
    }
    p.h[i] = h;
}

template <bool AGAIN>
__global__ __launch_bounds__(256) void swiglu_keep_backward_kernel(KeepArgs p) {
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= p.pieces) return;
    const u32x4 w = p.whole[i], dh = p.dh[i];
    const uint32_t both = p.exponents[i >> 2];
    const int eg = both & 0xFF, eu = both >> 8;
    u32x4 d_gate, d_up, h;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float dg[2], du[2], hh[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int at = 2 * e + b;
            const float g = from_whole(w[at >> 2], at & 3, eg), u = from_whole(w[2 + (at >> 2)], at & 3, eu), d = half_of(dh, at);
            const float s = __builtin_amdgcn_rcpf(1.f + __expf(-g)), silu = g * s;
            du[b] = d * silu;
            dg[b] = d * u * s * fmaf(g, 1.f - s, 1.f);
            hh[b] = silu * u;
        }
        d_gate[e] = pair_of(dg[0], dg[1]);
        d_up[e] = pair_of(du[0], du[1]);
        if constexpr (AGAIN) h[e] = pair_of(hh[0], hh[1]);
    }
    p.d_gate_up[2 * i] = d_gate;
    p.d_gate_up[2 * i + 1] = d_up;
    if constexpr (AGAIN) p.h[i] = h;
}

kiln_marlin_status_t shape_ok(int m, int n_out) {
    if (m < 0 || n_out < 1 || n_out % 128 != 0 || n_out > INT32_MAX / 2) return KILN_W4A16_ERR_PROB_SHAPE;
    return launchable(((int64_t)m * (n_out / 8) + 255) / 256, 256) ? KILN_W4A16_OK : KILN_W4A16_ERR_KERN_SHAPE;
}

}  // namespace
}  // namespace kiln

using namespace kiln;

extern "C" {

kiln_marlin_status_t kiln_w4a16_swiglu_keep(const void *gate_up, void *h, void *whole, void *exponents, int prob_m, int n_out, int dev, void *stream) {
    (void)dev;
    if (const kiln_marlin_status_t st = shape_ok(prob_m, n_out)) return st;
    if (prob_m == 0) return KILN_W4A16_OK;
    if (!all_on(16, {gate_up, h, whole}) || !all_on(2, {exponents})) return KILN_W4A16_ERR_ARGUMENT;
    const size_t n = (size_t)prob_m * n_out;
    if (any_meet({{h, 2 * n}, {whole, 2 * n}, {exponents, n / 16}}, {{gate_up, 4 * n}})) return KILN_W4A16_ERR_ARGUMENT;
    const KeepArgs a{(const u32x4 *)gate_up, nullptr, (u32x4 *)whole, (uint16_t *)exponents, (u32x4 *)h, nullptr, n / 8};
    swiglu_keep_kernel<<<(unsigned)((a.pieces + 255) / 256), 256, 0, reinterpret_cast<hipStream_t>(stream)>>>(a);
    return hipGetLastError() == hipSuccess ? KILN_W4A16_OK : KILN_W4A16_ERR_LAUNCH;
}

kiln_marlin_status_t kiln_w4a16_swiglu_keep_backward(const void *dh, const void *whole, const void *exponents, void *d_gate_up, void *h, int prob_m,
                                                     int n_out, int dev, void *stream) {
    (void)dev;
    if (const kiln_marlin_status_t st = shape_ok(prob_m, n_out)) return st;
    if (prob_m == 0) return KILN_W4A16_OK;
    if (!all_on(16, {dh, whole, d_gate_up}) || !all_on(2, {exponents}) || reinterpret_cast<uintptr_t>(h) % 16 != 0) return KILN_W4A16_ERR_ARGUMENT;
    const size_t n = (size_t)prob_m * n_out;
    if (any_meet({{d_gate_up, 4 * n}, {h, 2 * n}}, {{dh, 2 * n}, {whole, 2 * n}, {exponents, n / 16}})) return KILN_W4A16_ERR_ARGUMENT;
    const KeepArgs a{nullptr, (const u32x4 *)dh, (u32x4 *)const_cast<void *>(whole), (uint16_t *)const_cast<void *>(exponents), (u32x4 *)h, (u32x4 *)d_gate_up, n / 8};
    const unsigned grid = (unsigned)((a.pieces + 255) / 256);
    hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
    if (h) swiglu_keep_backward_kernel<true><<<grid, 256, 0, hs>>>(a);
    else swiglu_keep_backward_kernel<false><<<grid, 256, 0, hs>>>(a);
    return hipGetLastError() == hipSuccess ? KILN_W4A16_OK : KILN_W4A16_ERR_LAUNCH;
}

}  // extern "C"
