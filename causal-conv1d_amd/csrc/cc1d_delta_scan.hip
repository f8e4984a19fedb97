// The gated delta rule by chunks, second kernel: the states from chunk to chunk, and the outputs (cc1d_delta_chunk.hpp).
//
// A workgroup of four wavefronts takes 16 columns of one (sequence, value head)'s state, all of dim_k, and walks the chunks:
//
//   a  wavefront w: 16 tokens' rows of K S and Q S                      R = beta (V - gam K S) to LDS
//   b  the same rows of U = T R                                         U, and U to the chunk's end, to LDS
//   c  the same rows of O = scale gam Q S + P U; its share of S = gam_last S + K^T U'    S to LDS
//
// S stays in registers, spread over the wavefronts by rows; what travels through LDS are right operands, already split
// into their bfloat16 terms, and nothing needs to be turned around (row_of).  Left operands come from memory in the order in
// which lanes hold them, each asked for as soon as the one before it has been used, a whole chunk ahead.  The three barriers wait
// for LDS only.
#include "cc1d_delta_chunk.hpp"
#include "cc1d_delta_host.hpp"

namespace cc1d {
namespace {

template <int KS, int NU>
struct ScanLds {
    uint8_t s[KS * 3 * kFrag];           // S
    uint8_t r[2 * 3 * kFrag];            // R
    uint8_t u[2 * NU * kFrag];           // U for O
    uint8_t d[2 * 3 * kFrag];            // U to the chunk's end for S
};

// STATES: the state in front of every chunk, and U, go to memory too (for the backward), O does not.
template <int DT, int KS, bool STATES>
__global__ void __launch_bounds__(kBlock, 1)
delta_scan_kernel(const cc1d_delta_params p, const ChunkWork w, const uint32_t heads_total, const uint32_t col_tiles) {
    using T = typename Elem<DT>::type;
    constexpr int NT = Terms<DT>::n;
    constexpr int NU = DT == CC1D_F32 ? 3 : 2;           // terms of P, U and S in O: 16 bits where O has 8 or 11
    constexpr int OUT = NU - 1;
    constexpr int TW = (2 * KS + 3) / 4;                 // 16-row tiles of S a wavefront owns
    __shared__ ScanLds<KS, NU> lds;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, g = lane >> 4;
    // The slices of one head, which read the same operands, on one XCD.
    const uint32_t xcd = blockIdx.x & 7u, idx = blockIdx.x >> 3;
    const uint32_t nh = idx / col_tiles * 8u + xcd;
    if (nh >= heads_total) return;
    const int col = (int)(idx % col_tiles) * 16 + m;
    const int h = (int)(nh % (uint32_t)p.v_heads), n = (int)(nh / (uint32_t)p.v_heads);
    const int hk = h / (p.v_heads / p.heads);
    const bool has_col = col < p.dim_v;
    const TokenRange range = sequence_tokens(p, n);
    const int chunks = (int)((range.hi - range.lo + kChunk - 1) / kChunk);
    const int slot0 = first_slot(p, w, n, range);

    T *out = static_cast<T *>(p.out) + range.b * p.out_stride_b + h * p.out_stride_h + col;
    if (!STATES && p.cu_seqlens != nullptr && has_col) { // tokens in front of the first sequence and behind the last
        if (n == 0)
            for (int64_t t = wave * 4 + g; t < range.lo; t += 16) out[t * p.out_stride_l] = Elem<DT>::from_float(0.f);
        if (n == p.sequences - 1)
            for (int64_t t = range.hi + wave * 4 + g; t < p.seqlen; t += 16) out[t * p.out_stride_l] = Elem<DT>::from_float(0.f);
    }

    f32x4 s[TW];
#pragma unroll
    for (int i = 0; i < TW; ++i) {
        const int t = wave * TW + i;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int k = row_of(t, 4 * g + e);
            s[i][e] = p.initial_states != nullptr && t < 2 * KS && k < p.dim_k && has_col ? p.initial_states[n * p.init_stride_n + h * p.init_stride_h + k * p.init_stride_k + col] : 0.f;
        }
    }

    // Operands of the chunk at hand; each set is asked for again, for the next chunk, once it has been used.
    bf16x8 kf[KS][NT], qf[KS][NT], tf[2][3], pf[2][NU], ktf[TW][2][NT];
    float4 seen, beta, read, carry;
    float last;
    float v[4];
    const int64_t kb = w.kbytes(), tb = w.tbytes(), pb = w.pbytes();
    const int steps = (wave >> 1) + 1;                   // of a row of T and P
    auto ask_kq = [&](int c) {
        const int64_t at = ((int64_t)(slot0 + c) * p.heads + hk) * kb + (int64_t)wave * KS * NT * kFrag;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            load_frag<NT>(w.kf + at + i * NT * kFrag, lane, kf[i]);
            if (!STATES) load_frag<NT>(w.qf + at + i * NT * kFrag, lane, qf[i]);
        }
    };
    auto ask_v = [&](int c) {
        const float *sc = w.scalars + ((int64_t)(slot0 + c) * p.v_heads + h) * kScalars * kChunk;
        const int row = row_of(wave, 4 * g);
        seen = *reinterpret_cast<const float4 *>(sc + kSeenBeta * kChunk + row);
        beta = *reinterpret_cast<const float4 *>(sc + kBeta * kChunk + row);
        read = *reinterpret_cast<const float4 *>(sc + kReadGate * kChunk + row);
        carry = *reinterpret_cast<const float4 *>(sc + kCarry * kChunk + row);
        last = sc[kGate * kChunk + 63];
        const int64_t lo = range.lo + (int64_t)c * kChunk;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int64_t tok = lo + row + e;
            v[e] = has_col && tok < range.hi ? Elem<DT>::to_float(static_cast<const T *>(p.v)[range.b * p.v_stride_b + tok * p.v_stride_l + h * p.v_stride_h + col]) : 0.f;
        }
    };
    auto ask_t = [&](int c) {
        const uint8_t *f = w.tf + ((int64_t)(slot0 + c) * p.v_heads + h) * tb;
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (i < steps) load_frag<3>(f + lower_frag(wave, i) * 3 * kFrag, lane, tf[i]);
    };
    auto ask_p = [&](int c) {
        const uint8_t *f = w.pf + ((int64_t)(slot0 + c) * p.v_heads + h) * pb;
        if (!STATES)
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (i < steps) load_frag<NU>(f + lower_frag(wave, i) * NU * kFrag, lane, pf[i]);
        const uint8_t *kt = w.ktf + ((int64_t)(slot0 + c) * p.heads + hk) * kb;
#pragma unroll
        for (int i = 0; i < TW; ++i)
            if (wave * TW + i < 2 * KS)
#pragma unroll
                for (int j = 0; j < 2; ++j) load_frag<NT>(kt + ((wave * TW + i) * 2 + j) * NT * kFrag, lane, ktf[i][j]);
    };
    auto put = [&](uint8_t *base, int terms, int tile, int n_, const u32x2 &x) {  // a tile's half of a right operand
        *reinterpret_cast<u32x2 *>(base + ((tile >> 1) * terms + n_) * kFrag + lane * 16 + (tile & 1) * 8) = x;
    };
    if (chunks > 0) { ask_kq(0); ask_v(0); ask_t(0); ask_p(0); }

    for (int c = 0; c < chunks; ++c) {
        const bool more = c + 1 < chunks;
        const int64_t sv = (int64_t)(slot0 + c) * p.v_heads + h;
#pragma unroll
        for (int i = 0; i < TW; ++i) {
            const int t = wave * TW + i;
            if (t >= 2 * KS) break;
            const float x[4] = {s[i][0], s[i][1], s[i][2], s[i][3]};
            u32x2 f[3];
            split4<3>(x, f);
#pragma unroll
            for (int j = 0; j < 3; ++j) put(lds.s, 3, t, j, f[j]);
            if (STATES && has_col)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int k = row_of(t, 4 * g + e);
                    if (k < p.dim_k) w.s0[(sv * p.dim_k + k) * p.dim_v + col] = s[i][e];
                }
        }
        lds_barrier();
        f32x4 ks = {0.f, 0.f, 0.f, 0.f}, o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            bf16x8 b[3];
            load_frag<3>(lds.s + i * 3 * kFrag, lane, b);
            ks = product<2>(kf[i], b, ks);
            if (!STATES) o = product<OUT>(qf[i], b, o);
        }
        {
            const float x[4] = {beta.x * v[0] - seen.x * ks[0], beta.y * v[1] - seen.y * ks[1], beta.z * v[2] - seen.z * ks[2], beta.w * v[3] - seen.w * ks[3]};
            u32x2 f[3];
            split4<3>(x, f);
#pragma unroll
            for (int j = 0; j < 3; ++j) put(lds.r, 3, wave, j, f[j]);
        }
        o[0] *= read.x; o[1] *= read.y; o[2] *= read.z; o[3] *= read.w;
        const float4 to_end = carry;
        const float gam = last;
        if (more) { ask_kq(c + 1); ask_v(c + 1); }
        lds_barrier();
        f32x4 u = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (i < steps) {
                bf16x8 b[3];
                load_frag<3>(lds.r + i * 3 * kFrag, lane, b);
                u = product<2>(tf[i], b, u);
            }
        {
            const float x[4] = {u[0], u[1], u[2], u[3]}, y[4] = {u[0] * to_end.x, u[1] * to_end.y, u[2] * to_end.z, u[3] * to_end.w};
            u32x2 f[3];
            if (!STATES) {
                u32x2 fu[NU];
                split4<NU>(x, fu);
#pragma unroll
                for (int j = 0; j < NU; ++j) put(lds.u, NU, wave, j, fu[j]);
            } else if (has_col) {
#pragma unroll
                for (int e = 0; e < 4; ++e) w.u[(sv * kChunk + row_of(wave, 4 * g + e)) * p.dim_v + col] = x[e];
            }
            split4<3>(y, f);
#pragma unroll
            for (int j = 0; j < 3; ++j) put(lds.d, 3, wave, j, f[j]);
        }
        if (more) ask_t(c + 1);
        lds_barrier();
        if (!STATES) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (i < steps) {
                    bf16x8 b[NU];
                    load_frag<NU>(lds.u + i * NU * kFrag, lane, b);
                    o = product<OUT>(pf[i], b, o);
                }
            const int64_t lo = range.lo + (int64_t)c * kChunk;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int64_t tok = lo + row_of(wave, 4 * g + e);
                if (has_col && tok < range.hi) out[tok * p.out_stride_l] = Elem<DT>::from_float(o[e]);
            }
        }
#pragma unroll
        for (int i = 0; i < TW; ++i) {
            if (wave * TW + i >= 2 * KS) break;
            s[i] *= gam;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                bf16x8 b[3];
                load_frag<3>(lds.d + j * 3 * kFrag, lane, b);
                s[i] = product<2>(ktf[i][j], b, s[i]);
            }
        }
        if (more) ask_p(c + 1);
    }
    if (STATES || p.final_states == nullptr || !has_col) return;
#pragma unroll
    for (int i = 0; i < TW; ++i) {
        const int t = wave * TW + i;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int k = row_of(t, 4 * g + e);
            if (t < 2 * KS && k < p.dim_k) p.final_states[n * p.final_stride_n + h * p.final_stride_h + k * p.final_stride_k + col] = s[i][e];
        }
    }
}

template <int DT, int KS, bool STATES>
int launch(const cc1d_delta_params &p, const ChunkWork &w, hipStream_t stream) {
    const uint32_t tiles = (uint32_t)(p.dim_v + 15) / 16, nh = (uint32_t)((int64_t)p.sequences * p.v_heads);
    CC1D_LAUNCH((delta_scan_kernel<DT, KS, STATES>), dim3((nh + 7) / 8 * 8 * tiles), dim3(kBlock), 0, stream, p, w, nh, tiles);
    return launch_status();
}

}  // namespace

int launch_delta_scan(const cc1d_delta_params &p, const ChunkWork &w, bool states, hipStream_t stream) {
    return by_type_and_steps(p.x_dtype, w.ks, [&](auto dt, auto ks) {
        return states ? launch<decltype(dt)::value, decltype(ks)::value, true>(p, w, stream) : launch<decltype(dt)::value, decltype(ks)::value, false>(p, w, stream);
    });
}

}  // namespace cc1d
