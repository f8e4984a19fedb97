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

template <int KS, int NU, int CT>
struct ScanLds {
    uint8_t s[CT][KS * 3 * kFrag];       // S
    uint8_t r[CT][2 * 3 * kFrag];        // R
    uint8_t u[CT][2 * NU * kFrag];       // U for O
    uint8_t d[CT][2 * 3 * kFrag];        // U to the chunk's end for S
};

// STATES: the state in front of every chunk, and U, go to memory too (for the backward), O does not.
template <int DT, int KS, int CT, bool STATES>
__global__ void __launch_bounds__(kBlock, CT == 1 ? 2 : 1)
delta_scan_kernel(const cc1d_delta_params p, const ChunkWork w, const uint32_t heads_total, const uint32_t col_tiles) {
    using T = typename Elem<DT>::type;
    constexpr int NT = Terms<DT>::n, NU = Terms<DT>::p, OUT = NU - 1;
    constexpr int TW = (2 * KS + 3) / 4;                 // 16-row tiles of S a wavefront owns
    extern __shared__ uint4 raw[];
    ScanLds<KS, NU, CT> &lds = *reinterpret_cast<ScanLds<KS, NU, CT> *>(raw);
    const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // The slices of one head, which read the same operands, on one XCD.
    const uint32_t xcd = blockIdx.x & 7u, idx = blockIdx.x >> 3;
    const uint32_t nh = idx / col_tiles * 8u + xcd;
    if (nh >= heads_total) return;
    const int col0 = (int)(idx % col_tiles) * 16 * CT + m;
    const int h = (int)(nh % (uint32_t)p.v_heads), n = (int)(nh / (uint32_t)p.v_heads);
    const int hk = h / (p.v_heads / p.heads);
    const TokenRange range = sequence_tokens(p, n);
    const int chunks = (int)((range.hi - range.lo + kChunk - 1) / kChunk);
    const int slot0 = first_slot(p, w, n, range), total = (int)(range.hi - range.lo);
    const uint32_t v_pitch = (uint32_t)(p.v_stride_l * (int64_t)sizeof(T)), out_pitch = (uint32_t)(p.out_stride_l * (int64_t)sizeof(T));
    bool has_col[CT];
    int col[CT];                                         // a column that is there
#pragma unroll
    for (int i = 0; i < CT; ++i) {
        has_col[i] = col0 + 16 * i < p.dim_v;
        col[i] = has_col[i] ? col0 + 16 * i : 0;
    }

    T *out = static_cast<T *>(p.out) + range.b * p.out_stride_b + h * p.out_stride_h;
    if (!STATES && p.cu_seqlens != nullptr) {            // tokens in front of the first sequence and behind the last
        auto clear = [&](int64_t lo, int64_t hi) {
            for (int64_t t = lo + wave * 4 + g; t < hi; t += 16)
#pragma unroll
                for (int i = 0; i < CT; ++i)
                    if (has_col[i]) out[t * p.out_stride_l + col[i]] = Elem<DT>::from_float(0.f);
        };
        if (n == 0) clear(0, range.lo);
        if (n == p.sequences - 1) clear(range.hi, p.seqlen);
    }

    f32x4 s[CT][TW];
#pragma unroll
    for (int i = 0; i < TW; ++i) {
        const int t = wave * TW + i;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int k = row_of(t, 4 * g + e);
#pragma unroll
            for (int j = 0; j < CT; ++j)
                s[j][i][e] = p.initial_states != nullptr && t < 2 * KS && k < p.dim_k && has_col[j] ? p.initial_states[n * p.init_stride_n + h * p.init_stride_h + k * p.init_stride_k + col[j]] : 0.f;
        }
    }

    // Operands of the chunk at hand; each set is asked for again, for the next chunk, once it has been used.  No load stands behind a
    // condition (Row8): what a wavefront has no use for, and what lies behind the last token, is read from a place that exists.
    bf16x8 kf[KS][NT], qf[KS][NT], tf[2][3], pf[2][NU], ktf[TW][2][NT];
    float4 seen, beta, read, carry;
    float last;
    T v[CT][4];
    const int64_t kb = w.kbytes(), tb = w.tbytes(), pb = w.pbytes();
    const int steps = (wave >> 1) + 1;                   // of a row of T and P
    const int row = row_of(wave, 4 * g);
    const T *vp = static_cast<const T *>(p.v) + range.b * p.v_stride_b + range.lo * p.v_stride_l + h * p.v_stride_h;
    auto ask_kq = [&](int c, int i) {                    // step i
        const int64_t at = ((int64_t)(slot0 + c) * p.heads + hk) * kb + (int64_t)(wave * KS + i) * NT * kFrag;
        load_frag<NT>(w.kf + at, lane, kf[i]);
        if (!STATES) load_frag<NT>(w.qf + at, lane, qf[i]);
    };
    auto ask_v = [&](int c) {
        const float *sc = w.scalars + ((int64_t)(slot0 + c) * p.v_heads + h) * kScalars * kChunk;
        seen = *reinterpret_cast<const float4 *>(sc + kSeenBeta * kChunk + row);
        beta = *reinterpret_cast<const float4 *>(sc + kBeta * kChunk + row);
        read = *reinterpret_cast<const float4 *>(sc + kReadGate * kChunk + row);
        // Rows behind the last token take the last one's v: their beta is 0.
        const T *vc = vp + (int64_t)c * kChunk * p.v_stride_l;
        const int end = total - c * kChunk - 1;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t at = (uint32_t)(row + e < end ? row + e : end) * v_pitch;
#pragma unroll
            for (int j = 0; j < CT; ++j) v[j][e] = *reinterpret_cast<const T *>(reinterpret_cast<const uint8_t *>(vc) + (at + (uint32_t)col[j] * (uint32_t)sizeof(T)));
        }
    };
    auto ask_t = [&](int c, int i) {
        const uint8_t *f = w.tf + ((int64_t)(slot0 + c) * p.v_heads + h) * tb;
        load_frag<3>(f + lower_frag(wave, i < steps ? i : 0) * 3 * kFrag, lane, tf[i]);
    };
    auto ask_carry = [&](int c) {
        carry = *reinterpret_cast<const float4 *>(w.scalars + ((int64_t)(slot0 + c) * p.v_heads + h) * kScalars * kChunk + kCarry * kChunk + row);
    };
    auto ask_p = [&](int c, int i) {
        const uint8_t *f = w.pf + ((int64_t)(slot0 + c) * p.v_heads + h) * pb;
        load_frag<NU>(f + lower_frag(wave, i < steps ? i : 0) * NU * kFrag, lane, pf[i]);
    };
    auto ask_kt = [&](int c, int i) {                    // tile i of this wavefront's
        const int t = wave * TW + i < 2 * KS ? wave * TW + i : 0;
        const uint8_t *kt = w.ktf + ((int64_t)(slot0 + c) * p.heads + hk) * kb;
#pragma unroll
        for (int j = 0; j < 2; ++j) load_frag<NT>(kt + (t * 2 + j) * NT * kFrag, lane, ktf[i][j]);
    };
    auto ask_last = [&](int c) { last = w.scalars[((int64_t)(slot0 + c) * p.v_heads + h) * kScalars * kChunk + kGate * kChunk + 63]; };
    auto put = [&](uint8_t *base, int terms, int tile, int n_, const u32x2 &x) {  // a tile's half of a right operand
        *reinterpret_cast<u32x2 *>(base + ((tile >> 1) * terms + n_) * kFrag + lane * 16 + (tile & 1) * 8) = x;
    };
    if (chunks > 0) {
#pragma unroll
        for (int i = 0; i < KS; ++i) ask_kq(0, i);
        ask_v(0);
        ask_carry(0);
        ask_last(0);
#pragma unroll
        for (int i = 0; i < 2; ++i) ask_t(0, i);
#pragma unroll
        for (int i = 0; i < TW; ++i) ask_kt(0, i);
        if (!STATES)
#pragma unroll
            for (int i = 0; i < 2; ++i) ask_p(0, i);
    }

    for (int c = 0; c < chunks; ++c) {
        const int next = c + 1 < chunks ? c + 1 : c;
        const int64_t sv = (int64_t)(slot0 + c) * p.v_heads + h;
#pragma unroll
        for (int i = 0; i < TW; ++i) {
            const int t = wave * TW + i;
            if (t >= 2 * KS) break;
#pragma unroll
            for (int j = 0; j < CT; ++j) {
                const float x[4] = {s[j][i][0], s[j][i][1], s[j][i][2], s[j][i][3]};
                u32x2 f[3];
                split4<3>(x, f);
#pragma unroll
                for (int q = 0; q < 3; ++q) put(lds.s[j], 3, t, q, f[q]);
                if (STATES && has_col[j])
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int k = row_of(t, 4 * g + e);
                        if (k < p.dim_k) w.s0[(sv * p.dim_k + k) * p.dim_v + col[j]] = x[e];
                    }
            }
        }
        lds_barrier();
        f32x4 o[CT], ks[CT], rest[CT], orest[CT];
#pragma unroll
        for (int j = 0; j < CT; ++j) ks[j] = rest[j] = o[j] = orest[j] = (f32x4){0.f, 0.f, 0.f, 0.f};
        {
            bf16x8 b[CT][2][3];
#pragma unroll
            for (int j = 0; j < CT; ++j) load_frag<3>(lds.s[j], lane, b[j][0]);
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                if (i + 1 < KS)
#pragma unroll
                    for (int j = 0; j < CT; ++j) load_frag<3>(lds.s[j] + (i + 1) * 3 * kFrag, lane, b[j][(i + 1) & 1]);
                stay();
#pragma unroll
                for (int j = 0; j < CT; ++j) {
                    product2<2>(kf[i], b[j][i & 1], ks[j], rest[j]);
                    if (!STATES) product2<OUT>(qf[i], b[j][i & 1], o[j], orest[j]);
                }
                stay();
                ask_kq(next, i);
            }
        }
#pragma unroll
        for (int j = 0; j < CT; ++j) {
            ks[j] += rest[j];
            o[j] += orest[j];
            const float bt[4] = {beta.x, beta.y, beta.z, beta.w}, sn[4] = {seen.x, seen.y, seen.z, seen.w}, rd[4] = {read.x, read.y, read.z, read.w};
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[e] = bt[e] * Elem<DT>::to_float(v[j][e]) - sn[e] * ks[j][e];
                o[j][e] *= rd[e];
            }
            u32x2 f[3];
            split4<3>(x, f);
#pragma unroll
            for (int q = 0; q < 3; ++q) put(lds.r[j], 3, wave, q, f[q]);
        }
        lds_barrier();
        {
            bf16x8 b[CT][2][3];
            f32x4 u[CT], u2[CT];
#pragma unroll
            for (int j = 0; j < CT; ++j) {
                u[j] = u2[j] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < 2; ++i) load_frag<3>(lds.r[j] + i * 3 * kFrag, lane, b[j][i]);
            }
            stay();
#pragma unroll
            for (int j = 0; j < CT; ++j) product2<2>(tf[0], b[j][0], u[j], u2[j]);
            stay();
            ask_v(next);
            if (steps == 2)
#pragma unroll
                for (int j = 0; j < CT; ++j) product2<2>(tf[1], b[j][1], u[j], u2[j]);
            stay();
            ask_t(next, 0);
            ask_t(next, 1);
#pragma unroll
            for (int j = 0; j < CT; ++j) {
                u[j] += u2[j];
                const float x[4] = {u[j][0], u[j][1], u[j][2], u[j][3]}, y[4] = {x[0] * carry.x, x[1] * carry.y, x[2] * carry.z, x[3] * carry.w};
                u32x2 f[3];
                split4<3>(y, f);
#pragma unroll
                for (int q = 0; q < 3; ++q) put(lds.d[j], 3, wave, q, f[q]);
                if (!STATES) {
                    u32x2 fu[NU];
                    split4<NU>(x, fu);
#pragma unroll
                    for (int q = 0; q < NU; ++q) put(lds.u[j], NU, wave, q, fu[q]);
                } else if (has_col[j]) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) w.u[(sv * kChunk + row + e) * p.dim_v + col[j]] = x[e];
                }
            }
        }
        lds_barrier();
        {
            bf16x8 b[CT][2][3], bu[CT][2][NU];
#pragma unroll
            for (int j = 0; j < CT; ++j) {
#pragma unroll
                for (int q = 0; q < 2; ++q) load_frag<3>(lds.d[j] + q * 3 * kFrag, lane, b[j][q]);
                if (!STATES)
#pragma unroll
                    for (int q = 0; q < 2; ++q) load_frag<NU>(lds.u[j] + q * NU * kFrag, lane, bu[j][q]);
            }
            stay();
            ask_carry(next);
#pragma unroll
            for (int i = 0; i < TW; ++i) {
                if (wave * TW + i >= 2 * KS) break;
#pragma unroll
                for (int j = 0; j < CT; ++j) {
                    f32x4 small = {0.f, 0.f, 0.f, 0.f};
                    s[j][i] *= last;
#pragma unroll
                    for (int q = 0; q < 2; ++q) product2<2>(ktf[i][q], b[j][q], s[j][i], small);
                    s[j][i] += small;
                }
                stay();
                ask_kt(next, i);
            }
            if (!STATES) {
#pragma unroll
                for (int j = 0; j < CT; ++j) {
                    f32x4 small = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        if (i < steps) product2<OUT>(pf[i], bu[j][i], o[j], small);
                    o[j] += small;
                }
                stay();
                ask_p(next, 0);
                ask_p(next, 1);
            }
            ask_last(next);
        }
        if (!STATES) {
            uint8_t *oc = reinterpret_cast<uint8_t *>(out + (range.lo + (int64_t)c * kChunk) * p.out_stride_l);
            auto store = [&](int j, int e) {
                *reinterpret_cast<T *>(oc + ((uint32_t)(row + e) * out_pitch + (uint32_t)col[j] * (uint32_t)sizeof(T))) = Elem<DT>::from_float(o[j][e]);
            };
#pragma unroll
            for (int j = 0; j < CT; ++j)
                if (has_col[j]) {
                    if (total - c * kChunk >= kChunk) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) store(j, e);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (row + e < total - c * kChunk) store(j, e);
                    }
                }
        }
    }
    if (STATES || p.final_states == nullptr) return;
#pragma unroll
    for (int i = 0; i < TW; ++i) {
        const int t = wave * TW + i;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int k = row_of(t, 4 * g + e);
            if (t < 2 * KS && k < p.dim_k)
#pragma unroll
                for (int j = 0; j < CT; ++j)
                    if (has_col[j]) p.final_states[n * p.final_stride_n + h * p.final_stride_h + k * p.final_stride_k + col[j]] = s[j][i][e];
        }
    }
}

template <int DT, int KS, int CT, bool STATES>
int launch(const cc1d_delta_params &p, const ChunkWork &w, hipStream_t stream) {
    const uint32_t tiles = (uint32_t)(p.dim_v + 16 * CT - 1) / (16 * CT), nh = (uint32_t)((int64_t)p.sequences * p.v_heads);
    CC1D_LAUNCH((delta_scan_kernel<DT, KS, CT, STATES>), dim3((nh + 7) / 8 * 8 * tiles), dim3(kBlock), sizeof(ScanLds<KS, Terms<DT>::p, CT>), stream, p, w, nh, tiles);
    return launch_status();
}
template <int DT, int KS, int CT>
int launch_either(const cc1d_delta_params &p, const ChunkWork &w, bool states, hipStream_t stream) {
    return states ? launch<DT, KS, CT, true>(p, w, stream) : launch<DT, KS, CT, false>(p, w, stream);
}

}  // namespace

int launch_delta_scan(const cc1d_delta_params &p, const ChunkWork &w, bool states, hipStream_t stream) {
    return by_type_and_steps(p.x_dtype, w.ks, [&](auto dt, auto ks) {
        constexpr int DT = decltype(dt)::value, KS = decltype(ks)::value;
        return wide_columns(p) ? launch_either<DT, KS, 2>(p, w, states, stream) : launch_either<DT, KS, 1>(p, w, states, stream);
    });
}

}  // namespace cc1d
