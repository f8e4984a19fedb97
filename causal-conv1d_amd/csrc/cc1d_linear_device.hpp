// Linear attention: reading of gates and of column pairs (cc1d_linear.hpp).
#pragma once

#include "cc1d_linear.hpp"

namespace cc1d {

// G of a segment's tokens as two floats, G at the end, and beta (1 without it; 0 behind the last token).
struct GateLds { float hi[kSegment], lo[kSegment], beta[kSegment]; double sums[kBlocks]; };

// All four wavefronts; ends with a barrier.  In front of it the LDS must be free.
__device__ __forceinline__ void segment_gates(const cc1d_delta_params &p, const SegmentAt &at, int h, int wave, int lane, GateLds &lds) {
    static_assert(kBlocks <= 4, "a wavefront a block");
    double sum = 0.0;
    float beta = 1.f;
    const int i = wave * kChunk + lane;
    if (wave < kBlocks) {
        const int64_t tok = at.lo + (i < at.count ? i : 0);
        const uint32_t bits = load_bits(p.g, at.b * p.g_stride_b + tok * p.g_stride_l + h * p.g_stride_h, p.g_dtype);
        if (p.beta != nullptr) beta = bits_as_float(load_bits(p.beta, at.b * p.beta_stride_b + tok * p.beta_stride_l + h * p.beta_stride_h, p.beta_dtype), p.beta_dtype);
        sum = running_sum(i < at.count ? (double)bounded_gate(bits_as_float(bits, p.g_dtype)) : 0.0);
        if (lane == 63) lds.sums[wave] = sum;
    }
    lds_barrier();
    if (wave < kBlocks) {
        double before = 0.0;
        for (int b = 0; b < wave; ++b) before += lds.sums[b];
        sum += before;
        const float hi = (float)sum;
        lds.hi[i] = hi;
        lds.lo[i] = (float)(sum - (double)hi);
        lds.beta[i] = i < at.count ? beta : 0.f;
    }
    lds_barrier();
}
__device__ __forceinline__ float decay_between(const GateLds &lds, int from, int to) {        // exp(G_to - G_from)
    return exp_of((lds.hi[to] - lds.hi[from]) + (lds.lo[to] - lds.lo[from]));
}
// exp of a sum of gates: what 32 bits leave of it (2^-19 of a sum of 32 to 64, and of its exponential) counts as well.
__device__ __forceinline__ float exp_of_sum(double x) {
    const float hi = (float)x, e = exp_of(hi);
    return fmaf(e, (float)(x - (double)hi), e);
}
__device__ __forceinline__ float decay_since_start(const GateLds &lds, int to) {
    const float e = exp_of(lds.hi[to]);
    return fmaf(e, lds.lo[to], e);       // |lo| < 2^-8 |hi| 2^-16: the next term is nothing
}

// Sums over the 16 lanes of a row of a result tile, and over all 64.
__device__ __forceinline__ double over_columns(double v) {
    v += moved_or_zero<0xB1, 0xf>(v);    // (quad_perm, row_ror: every lane has a source)
    v += moved_or_zero<0x4E, 0xf>(v);
    v += moved_or_zero<0x124, 0xf>(v);
    return v + moved_or_zero<0x128, 0xf>(v);
}
__device__ __forceinline__ double over_wave(double v) {
    v = over_columns(v);
    return (of_lane(v, 0) + of_lane(v, 16)) + (of_lane(v, 32) + of_lane(v, 48));
}

// Columns c, c + 1 (`c` even) of eight rows: the right operand of two result tiles, whose columns are the even and the odd ones of
// 32, so that a lane loads both with one access and stores both of its results with one.  Eight consecutive rows of one column are what
// the matrix instruction wants of a lane, and no 16-bit element has to cross lanes for it.
template <int DT>
struct Pair8 {
    static constexpr int W = DT == CC1D_F32 ? 2 : 1;
    uint32_t r[8][W];
    // at[i]: byte offset of row i from base; columns that are not there repeat the first.
    __device__ __forceinline__ void ask(const void *base, const uint32_t (&at)[8], int c, int cols) {
        const uint8_t *b = static_cast<const uint8_t *>(base);
        const uint32_t o = (c < cols ? c : 0) * (uint32_t)(DT == CC1D_F32 ? 4 : 2);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (DT == CC1D_F32) {
                const u32x2 v = *reinterpret_cast<const u32x2 *>(b + (at[i] + o));
                r[i][0] = v.x;
                r[i][W - 1] = v.y;
            } else {
                r[i][0] = *reinterpret_cast<const uint32_t *>(b + (at[i] + o));
            }
        }
    }
    // Column c + odd as numbers, and as an operand.
    __device__ __forceinline__ void get(int odd, float (&f)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (DT == CC1D_F32) f[i] = bitcast<float>(r[i][odd ? W - 1 : 0]);
            else if constexpr (DT == CC1D_F16) f[i] = (float)bitcast<_Float16>((uint16_t)(odd ? r[i][0] >> 16 : r[i][0]));
            else f[i] = bitcast<float>(odd ? r[i][0] & 0xffff0000u : r[i][0] << 16);
        }
    }
    template <int TERMS>
    __device__ __forceinline__ void operand(int odd, bf16x8 (&t)[TERMS]) const {
        if constexpr (DT == CC1D_BF16 && TERMS == 1) {
            u32x4 w;
            const uint32_t sel = odd ? 0x07060302u : 0x05040100u;
            w.x = __builtin_amdgcn_perm(r[1][0], r[0][0], sel);
            w.y = __builtin_amdgcn_perm(r[3][0], r[2][0], sel);
            w.z = __builtin_amdgcn_perm(r[5][0], r[4][0], sel);
            w.w = __builtin_amdgcn_perm(r[7][0], r[6][0], sel);
            t[0] = bitcast<bf16x8>(w);
        } else {
            float f[8];
            get(odd, f);
            split8<TERMS>(f, t);
        }
    }
};

// Two adjacent results to columns c, c + 1 of a row.
template <int DT>
__device__ __forceinline__ void store_pair(typename Elem<DT>::type *row, int c, int cols, float a, float b) {
    if (c >= cols) return;
    if constexpr (DT == CC1D_F32) {
        *reinterpret_cast<float2 *>(row + c) = make_float2(a, b);
    } else if constexpr (DT == CC1D_F16) {
        asm("" : "+v"(a), "+v"(b));      // (no fused multiply that rounds to fp16 in one step)
        f16x2 h;
        h.x = (_Float16)a;
        h.y = (_Float16)b;
        *reinterpret_cast<uint32_t *>(row + c) = bitcast<uint32_t>(h);
    } else {
        *reinterpret_cast<uint32_t *>(row + c) = rounded_pair(a, b);
    }
}

}  // namespace cc1d
