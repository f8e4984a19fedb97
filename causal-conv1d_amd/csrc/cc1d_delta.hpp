// What the kernels of the gated delta rule share: reading of gates, where a chunk of tokens lies, and
// products of fp32 matrices on the 16-bit matrix cores.
#pragma once

#include "cc1d_device.hpp"
#include "cc1d_internal.hpp"
#include "cc1d_mixer.h"

namespace cc1d {

constexpr int kChunk = 64;               // tokens of a chunk
constexpr float kNormEps = 1e-6f;        // under the root of qk_l2norm

// exp(x) as 2^(x log2 e), the product in two floats: 6 instructions where expf takes 25.  Off by 2 units in the last place at most where the
// result is a normal number of 32 bits; 0 below that, from -87.4 on (the instruction gives no others), -inf included; an infinity or a NaN
// where it is too large, from 88.8 on, after which the recurrence has no finite value either (D^T k meets an infinity in every column).
__device__ __forceinline__ float exp_of(float x) {
    const float hi = x * 1.44269502f, lo = fmaf(x, 1.44269502f, -hi) + x * 1.92596299e-8f;
    const float e = __builtin_amdgcn_exp2f(hi);
    return x < -104.f ? 0.f : fmaf(e, lo * 0.693147182f, e);
}

// Sums over the 16 lanes of a row of a result tile, and over all 64, by DPP and half swaps: no LDS, the same order every time.
__device__ __forceinline__ float over_columns(float v) {
    v += dpp_moved<0xB1>(v);                             // quad_perm: lane ^ 1
    v += dpp_moved<0x4E>(v);                             // lane ^ 2
    v += dpp_moved<0x124>(v);                            // row_ror:4
    return v + dpp_moved<0x128>(v);                      // row_ror:8
}
__device__ __forceinline__ float over_rows(float v) {    // over lanes m, m + 16, m + 32, m + 48
    const auto a = __builtin_amdgcn_permlane16_swap(bitcast<uint32_t>(v), bitcast<uint32_t>(v), false, false);
    v = bitcast<float>((uint32_t)a[0]) + bitcast<float>((uint32_t)a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(bitcast<uint32_t>(v), bitcast<uint32_t>(v), false, false);
    return bitcast<float>((uint32_t)b[0]) + bitcast<float>((uint32_t)b[1]);
}
__device__ __forceinline__ float over_wave(float v) { return over_rows(over_columns(v)); }

// A double moved by DPP, 0 where a lane has no source or its row of 16 is not in ROWS.
template <int CTRL, int ROWS>
__device__ __forceinline__ double moved_or_zero(double v) {
    const uint64_t x = bitcast<uint64_t>(v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, CTRL, ROWS, 0xf, true);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(x >> 32), CTRL, ROWS, 0xf, true);
    return bitcast<double>((uint64_t)hi << 32 | lo);
}
// Running sums over the 64 lanes.
__device__ __forceinline__ double running_sum(double v) {
    v += moved_or_zero<0x111, 0xf>(v);                   // row_shr: 1, 2, 4, 8
    v += moved_or_zero<0x112, 0xf>(v);
    v += moved_or_zero<0x114, 0xf>(v);
    v += moved_or_zero<0x118, 0xf>(v);
    v += moved_or_zero<0x142, 0xa>(v);                   // row_bcast:15: the last lane of rows 0 and 2 to rows 1 and 3
    return v + moved_or_zero<0x143, 0xc>(v);             // row_bcast:31: the last lane of row 1 to rows 2 and 3
}
// What lane i and all behind it hold, summed.
__device__ __forceinline__ float sum_from_here(float v) {
    v += dpp_moved<0x101>(v);                            // row_shl: 1, 2, 4, 8
    v += dpp_moved<0x102>(v);
    v += dpp_moved<0x104>(v);
    v += dpp_moved<0x108>(v);
    const int bits = bitcast<int>(v), row = (threadIdx.x & 63) >> 4;
    const float c = bitcast<float>(__builtin_amdgcn_readlane(bits, 48));                   // rows' totals
    const float b = bitcast<float>(__builtin_amdgcn_readlane(bits, 32)) + c, a = bitcast<float>(__builtin_amdgcn_readlane(bits, 16)) + b;
    return v + (row == 0 ? a : row == 1 ? b : row == 2 ? c : 0.f);
}
__device__ __forceinline__ double of_lane(double v, int lane) {
    const uint64_t x = bitcast<uint64_t>(v);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)x, lane), hi = __builtin_amdgcn_readlane((int)(uint32_t)(x >> 32), lane);
    return bitcast<double>((uint64_t)hi << 32 | lo);
}

// An element as bits.  Loaded elements that cross a loop's end are kept so: __bf16 would be turned into a float in front of it,
// and waited for.
template <int DT> struct BitsOf { typedef uint16_t type; };
template <> struct BitsOf<CC1D_F32> { typedef uint32_t type; };

// A number of any of the three types, in two halves: the load, and what waits for it.
__device__ __forceinline__ uint32_t load_bits(const void *p, int64_t i, int dtype) {
    return dtype == CC1D_F32 ? static_cast<const uint32_t *>(p)[i] : (uint32_t)static_cast<const uint16_t *>(p)[i];
}
__device__ __forceinline__ float bits_as_float(uint32_t bits, int dtype) {
    if (dtype == CC1D_F16) return (float)bitcast<_Float16>((uint16_t)bits);
    return bitcast<float>(dtype == CC1D_F32 ? bits : bits << 16);
}
__device__ __forceinline__ void store_from_float(void *p, int64_t i, int dtype, float v) {
    if (dtype == CC1D_F32) static_cast<float *>(p)[i] = v;
    else if (dtype == CC1D_F16) static_cast<_Float16 *>(p)[i] = (_Float16)v;
    else static_cast<__bf16 *>(p)[i] = (__bf16)v;
}

// exp(-200) is 0 in fp32, and sums of such gates stay finite, so that differences of them do too: -inf ("forget
// everything") needs no other treatment.  A NaN stays one.
__device__ __forceinline__ float bounded_gate(float g) { return g < -200.f ? -200.f : g; }

__device__ __forceinline__ int64_t cu_entry(const void *cu, int is64, int i, int64_t most) {
    int64_t v = is64 ? static_cast<const int64_t *>(cu)[i] : (int64_t)static_cast<const int32_t *>(cu)[i];
    return v < 0 ? 0 : v > most ? most : v;
}
// Tokens [lo, hi) of sequence n, counted inside batch entry b.
struct TokenRange { int64_t lo, hi; int b; };
__device__ __forceinline__ TokenRange sequence_tokens(const cc1d_delta_params &p, int n) {
    if (p.cu_seqlens == nullptr) return {0, p.seqlen, n};
    const int64_t lo = cu_entry(p.cu_seqlens, p.cu_seqlens_is_int64, n, p.seqlen);
    const int64_t hi = cu_entry(p.cu_seqlens, p.cu_seqlens_is_int64, n + 1, p.seqlen);
    return {lo, hi < lo ? lo : hi, 0};
}

// Orders a wavefront's own LDS writes before its reads of what other lanes wrote.
__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

}  // namespace cc1d
