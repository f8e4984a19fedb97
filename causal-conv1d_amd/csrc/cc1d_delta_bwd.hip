// The gated delta rule by chunks, backward (cc1d_delta_chunk.hpp).  The states in front of the chunks and U are computed
// again (prep and scan kernels); then, with dS1 the gradient of the state behind a chunk:
//
//   scan, last chunk first:   dU = P^T dO + diag(dec) K dS1,  dX = T^T dU,  dV = diag(beta) dX
//                             dS0 = gam_last dS1 + (scale diag(gam) Q)^T dO - (diag(gam beta) K)^T dX
//   then every chunk alone:   X1 = scale lower(dO U^T) * E,  X2 = -strict lower(dX U^T) * E
//                             dQ = scale diag(gam) dO S0^T + X1 K,   Z = -diag(gam) dX S0^T + X2 K,   W = diag(dec) U dS1^T
//                             Y = X1^T Q + (diag(beta) X2)^T K + W,  dK = diag(beta) Z + Y
//                             dbeta_i = dX_i.V_i + k_i.Z_i
//                             dG_i = q_i.dQ_i + beta_i k_i.Z_i - k_i.Y_i,  dG_last += sum_j k_j.W_j + gam_last <S0, dS1>
//                             dg = sums of dG from the chunk's end
//
// The gates' gradients need no products of their own: every place where G stands is a row of one of the terms above.
// Heads that share q and k are walked one after the other by one workgroup, which adds their dQ and dK up in
// registers: no atomics, the same bits every time.
#include "cc1d_delta_chunk.hpp"
#include "cc1d_delta_host.hpp"

namespace cc1d {
namespace {

template <int DT, int KS>
struct BwdScanLds {
    uint8_t s[KS * 3 * kFrag];                           // dS1
    uint8_t o[2 * Terms<DT>::n * kFrag];                 // dO
    uint8_t q[2 * 3 * kFrag];                            // scale gam rq dO
    uint8_t u[2 * 3 * kFrag];                            // dU
    uint8_t x[2 * 3 * kFrag];                            // -beta gam rk dX
};

template <int DT, int KS>
__global__ void __launch_bounds__(kBlock, 1)
delta_bwd_scan_kernel(const cc1d_delta_bwd_params bp, const ChunkWork w, const uint32_t heads_total, const uint32_t col_tiles) {
    using T = typename Elem<DT>::type;
    constexpr int NT = Terms<DT>::n;
    constexpr int TW = (2 * KS + 3) / 4;
    __shared__ BwdScanLds<DT, KS> lds;
    const cc1d_delta_params &p = bp.fwd;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, g = lane >> 4;
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

    T *dv = static_cast<T *>(bp.dv) + range.b * bp.dv_stride_b + h * bp.dv_stride_h + col;
    if (p.cu_seqlens != nullptr && has_col) {            // tokens in front of the first sequence and behind the last
        if (n == 0)
            for (int64_t t = wave * 4 + g; t < range.lo; t += 16) dv[t * bp.dv_stride_l] = Elem<DT>::from_float(0.f);
        if (n == p.sequences - 1)
            for (int64_t t = range.hi + wave * 4 + g; t < p.seqlen; t += 16) dv[t * bp.dv_stride_l] = Elem<DT>::from_float(0.f);
    }

    f32x4 s[TW];
#pragma unroll
    for (int i = 0; i < TW; ++i) {
        const int t = wave * TW + i;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int k = row_of(t, 4 * g + e);
            s[i][e] = bp.dfinal_states != nullptr && t < 2 * KS && k < p.dim_k && has_col ? bp.dfinal_states[n * bp.dfinal_stride_n + h * bp.dfinal_stride_h + k * bp.dfinal_stride_k + col] : 0.f;
        }
    }

    bf16x8 kf[KS][NT], tf[2][3], pf[2][3], ktf[TW][2][NT], qtf[TW][2][NT];
    float4 seen, beta, read, carry;
    float last;
    float d[4];
    const int64_t kb = w.kbytes(), tb = w.tbytes();
    const int from = wave >> 1;                          // first step of a row of T^T and P^T
    auto ask_k = [&](int c) {
        const int64_t at = ((int64_t)(slot0 + c) * p.heads + hk) * kb + (int64_t)wave * KS * NT * kFrag;
#pragma unroll
        for (int i = 0; i < KS; ++i) load_frag<NT>(w.kf + at + i * NT * kFrag, lane, kf[i]);
        const uint8_t *f = w.ptf + ((int64_t)(slot0 + c) * p.v_heads + h) * tb;
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (i >= from) load_frag<3>(f + upper_frag(wave, i) * 3 * kFrag, lane, pf[i]);
    };
    auto ask_d = [&](int c) {
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
            d[e] = has_col && tok < range.hi ? Elem<DT>::to_float(static_cast<const T *>(bp.dout)[range.b * bp.dout_stride_b + tok * bp.dout_stride_l + h * bp.dout_stride_h + col]) : 0.f;
        }
    };
    auto ask_t = [&](int c) {
        const uint8_t *f = w.ttf + ((int64_t)(slot0 + c) * p.v_heads + h) * tb;
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (i >= from) load_frag<3>(f + upper_frag(wave, i) * 3 * kFrag, lane, tf[i]);
    };
    auto ask_kt = [&](int c) {
        const int64_t at = ((int64_t)(slot0 + c) * p.heads + hk) * kb;
#pragma unroll
        for (int i = 0; i < TW; ++i)
            if (wave * TW + i < 2 * KS)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    load_frag<NT>(w.ktf + at + ((wave * TW + i) * 2 + j) * NT * kFrag, lane, ktf[i][j]);
                    load_frag<NT>(w.qtf + at + ((wave * TW + i) * 2 + j) * NT * kFrag, lane, qtf[i][j]);
                }
    };
    auto put = [&](uint8_t *base, int terms, int tile, int n_, const u32x2 &x) {
        *reinterpret_cast<u32x2 *>(base + ((tile >> 1) * terms + n_) * kFrag + lane * 16 + (tile & 1) * 8) = x;
    };
    if (chunks > 0) { ask_k(chunks - 1); ask_d(chunks - 1); ask_t(chunks - 1); ask_kt(chunks - 1); }

    for (int c = chunks - 1; c >= 0; --c) {
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
            if (has_col)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int k = row_of(t, 4 * g + e);
                    if (k < p.dim_k) w.ds1[(sv * p.dim_k + k) * p.dim_v + col] = s[i][e];
                }
        }
        {
            const float y[4] = {d[0] * read.x, d[1] * read.y, d[2] * read.z, d[3] * read.w};
            u32x2 fo[NT], f[3];
            split4<NT>(d, fo);
#pragma unroll
            for (int j = 0; j < NT; ++j) put(lds.o, NT, wave, j, fo[j]);
            split4<3>(y, f);
#pragma unroll
            for (int j = 0; j < 3; ++j) put(lds.q, 3, wave, j, f[j]);
        }
        const float4 sb = seen, bt = beta;
        lds_barrier();
        f32x4 u = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            bf16x8 b[3];
            load_frag<3>(lds.s + i * 3 * kFrag, lane, b);
            u = product<2>(kf[i], b, u);
        }
        u[0] *= carry.x; u[1] *= carry.y; u[2] *= carry.z; u[3] *= carry.w;
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (i >= from) {
                bf16x8 b[NT];
                load_frag<NT>(lds.o + i * NT * kFrag, lane, b);
                u = product<2>(pf[i], b, u);
            }
        {
            const float x[4] = {u[0], u[1], u[2], u[3]};
            u32x2 f[3];
            split4<3>(x, f);
#pragma unroll
            for (int j = 0; j < 3; ++j) put(lds.u, 3, wave, j, f[j]);
        }
        const float gam = last;
        if (c > 0) { ask_k(c - 1); ask_d(c - 1); }
        lds_barrier();
        f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (i >= from) {
                bf16x8 b[3];
                load_frag<3>(lds.u + i * 3 * kFrag, lane, b);
                x = product<2>(tf[i], b, x);
            }
        {
            const float y[4] = {-sb.x * x[0], -sb.y * x[1], -sb.z * x[2], -sb.w * x[3]}, bx[4] = {bt.x * x[0], bt.y * x[1], bt.z * x[2], bt.w * x[3]};
            u32x2 f[3];
            split4<3>(y, f);
#pragma unroll
            for (int j = 0; j < 3; ++j) put(lds.x, 3, wave, j, f[j]);
            if (has_col)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int row = row_of(wave, 4 * g + e);
                    const int64_t tok = range.lo + (int64_t)c * kChunk + row;
                    w.dx[(sv * kChunk + row) * p.dim_v + col] = x[e];
                    if (tok < range.hi) dv[tok * bp.dv_stride_l] = Elem<DT>::from_float(bx[e]);
                }
        }
        if (c > 0) ask_t(c - 1);
        lds_barrier();
#pragma unroll
        for (int i = 0; i < TW; ++i) {
            if (wave * TW + i >= 2 * KS) break;
            s[i] *= gam;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                bf16x8 b[3];
                load_frag<3>(lds.q + j * 3 * kFrag, lane, b);
                s[i] = product<2>(qtf[i][j], b, s[i]);
                load_frag<3>(lds.x + j * 3 * kFrag, lane, b);
                s[i] = product<2>(ktf[i][j], b, s[i]);
            }
        }
        if (c > 0) ask_kt(c - 1);
        lds_barrier();                                   // lds.q is written again before the next barrier
    }
    if (bp.dinitial_states == nullptr || !has_col) return;
#pragma unroll
    for (int i = 0; i < TW; ++i) {
        const int t = wave * TW + i;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int k = row_of(t, 4 * g + e);
            if (t < 2 * KS && k < p.dim_k) bp.dinitial_states[n * bp.dinit_stride_n + h * bp.dinit_stride_h + k * bp.dinit_stride_k + col] = s[i][e];
        }
    }
}

// 8 elements of a row from column c on, zeros behind `cols`.
template <int DT>
__device__ __forceinline__ void row8(const typename Elem<DT>::type *row, int c, int cols, bool vec, float (&f)[8]) {
    if (vec && c + 8 <= cols) {
        if constexpr (DT == CC1D_F32) {
            float lo[4], hi[4];
            Elem<DT>::unpack(*reinterpret_cast<const u32x4 *>(row + c), lo);
            Elem<DT>::unpack(*reinterpret_cast<const u32x4 *>(row + c + 4), hi);
#pragma unroll
            for (int i = 0; i < 4; ++i) { f[i] = lo[i]; f[i + 4] = hi[i]; }
        } else {
            Elem<DT>::unpack(*reinterpret_cast<const u32x4 *>(row + c), f);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = c + i < cols ? Elem<DT>::to_float(row[c + i]) : 0.f;
}

template <int KS>
struct GradStage { uint8_t u[4 * 3 * kFrag], s0[2 * KS * 3 * kFrag], ds1[2 * KS * 3 * kFrag]; };
struct GradLower { float x1[kChunk][68], x2[kChunk][68]; };
template <int KS>
struct GradLds {
    union { GradStage<KS> stage; GradLower lower; };
    float gate[kScalars][kChunk];
    float dg[kChunk], db[kChunk], end[4], inner[4];
};

__device__ __forceinline__ float over_columns(float v) {  // over the 16 lanes of a row of a result tile
    v += __shfl_xor(v, 1); v += __shfl_xor(v, 2); v += __shfl_xor(v, 4); v += __shfl_xor(v, 8);
    return v;
}

template <int DT, int KS>
__global__ void __launch_bounds__(kBlock, 1)
delta_grad_kernel(const cc1d_delta_bwd_params bp, const ChunkWork w, const int vec_x, const int vec_s) {
    using T = typename Elem<DT>::type;
    constexpr int NT = Terms<DT>::n;
    constexpr int TILES = 2 * KS;
    extern __shared__ uint4 raw[];
    GradLds<KS> &lds = *reinterpret_cast<GradLds<KS> *>(raw);
    const cc1d_delta_params &p = bp.fwd;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, g = lane >> 4;
    const int slot = (int)(blockIdx.x / (uint32_t)p.heads), hk = (int)(blockIdx.x % (uint32_t)p.heads);
    const int group = p.v_heads / p.heads;
    const ChunkAt at = chunk_at(p, w, slot);
    T *dq = static_cast<T *>(bp.dq) + hk * bp.dq_stride_h, *dk = static_cast<T *>(bp.dk) + hk * bp.dk_stride_h;
    if (p.cu_seqlens != nullptr && slot == 0) {          // tokens in front of the first sequence and behind the last
        auto clear = [&](int64_t lo, int64_t hi) {
            for (int64_t t = lo + wave; t < hi; t += 4) {
                for (int k = lane; k < p.dim_k; k += 64) {
                    dq[t * bp.dq_stride_l + k] = Elem<DT>::from_float(0.f);
                    dk[t * bp.dk_stride_l + k] = Elem<DT>::from_float(0.f);
                }
                for (int i = lane; i < group; i += 64) {
                    store_from_float(bp.dg, t * p.v_heads + hk * group + i, p.g_dtype, 0.f);
                    store_from_float(bp.dbeta, t * p.v_heads + hk * group + i, p.beta_dtype, 0.f);
                }
            }
        };
        clear(0, sequence_tokens(p, 0).lo);
        clear(sequence_tokens(p, p.sequences - 1).hi, p.seqlen);
    }
    if (at.count <= 0) return;
    const int64_t sh = (int64_t)slot * p.heads + hk;
    const int own = row_of(wave, m);                     // the token whose row this lane holds as a left operand
    const int row = row_of(wave, 4 * g);                 // the first of the four whose results it holds
    const bool there = own < at.count;

    f32x4 tq[TILES], tk[TILES];                          // dQ, dK of all heads of the group
#pragma unroll
    for (int t = 0; t < TILES; ++t) { tq[t] = (f32x4){0.f, 0.f, 0.f, 0.f}; tk[t] = (f32x4){0.f, 0.f, 0.f, 0.f}; }
    // An element of Q or K where the result tiles have it.
    auto element = [&](const void *base, int64_t sb, int64_t sl, int64_t sh_, int t, int e) {
        const int k = row_of(t, m);
        return k < p.dim_k && row + e < at.count ? Elem<DT>::to_float(static_cast<const T *>(base)[at.b * sb + (at.lo + row + e) * sl + hk * sh_ + k]) : 0.f;
    };

    for (int j = 0; j < group; ++j) {
        const int h = hk * group + j;
        const int64_t sv = (int64_t)slot * p.v_heads + h;
        for (int i = threadIdx.x; i < kScalars * kChunk; i += kBlock) (&lds.gate[0][0])[i] = w.scalars[sv * kScalars * kChunk + i];
        f32x4 aq[TILES], az[TILES], ay[TILES], x1[4], x2[4];
#pragma unroll
        for (int t = 0; t < TILES; ++t) { aq[t] = (f32x4){0.f, 0.f, 0.f, 0.f}; az[t] = aq[t]; ay[t] = aq[t]; }
#pragma unroll
        for (int t = 0; t < 4; ++t) { x1[t] = (f32x4){0.f, 0.f, 0.f, 0.f}; x2[t] = x1[t]; }
        float inner = 0.f, dxv = 0.f;
        const T *dop = static_cast<const T *>(bp.dout) + at.b * bp.dout_stride_b + (at.lo + (there ? own : 0)) * bp.dout_stride_l + h * bp.dout_stride_h;
        const T *vp = static_cast<const T *>(p.v) + at.b * p.v_stride_b + (at.lo + (there ? own : 0)) * p.v_stride_l + h * p.v_stride_h;
        const float *up = w.u + (sv * kChunk + own) * p.dim_v, *xp = w.dx + (sv * kChunk + own) * p.dim_v;
        for (int v0 = 0; v0 < p.dim_v; v0 += 32) {
            const int c = v0 + 8 * g;
            float f[8], f2[8];
            bf16x8 fo[NT], fx[3], fu[3];
            row8<DT>(dop, c, there ? p.dim_v : 0, vec_x, f);
            split8<NT>(f, fo);
            row8<CC1D_F32>(xp, c, p.dim_v, vec_s, f);
            row8<DT>(vp, c, there ? p.dim_v : 0, vec_x, f2);
#pragma unroll
            for (int e = 0; e < 8; ++e) dxv += f[e] * f2[e];
            split8<3>(f, fx);
            row8<CC1D_F32>(up, c, p.dim_v, vec_s, f);
            split8<3>(f, fu);
            __syncthreads();                             // the step before has been read
#pragma unroll
            for (int n = 0; n < 3; ++n) *reinterpret_cast<u32x4 *>(lds.stage.u + (wave * 3 + n) * kFrag + lane * 16) = bitcast<u32x4>(fu[n]);
#pragma unroll
            for (int i = 0; i < (TILES + 3) / 4; ++i) {
                const int t = wave + 4 * i;
                if (t >= TILES) break;
                const int k = row_of(t, m);
                bf16x8 fs[3];
                row8<CC1D_F32>(w.s0 + (sv * p.dim_k + (k < p.dim_k ? k : 0)) * p.dim_v, c, k < p.dim_k ? p.dim_v : 0, vec_s, f);
                row8<CC1D_F32>(w.ds1 + (sv * p.dim_k + (k < p.dim_k ? k : 0)) * p.dim_v, c, k < p.dim_k ? p.dim_v : 0, vec_s, f2);
#pragma unroll
                for (int e = 0; e < 8; ++e) inner += f[e] * f2[e];
                split8<3>(f, fs);
#pragma unroll
                for (int n = 0; n < 3; ++n) *reinterpret_cast<u32x4 *>(lds.stage.s0 + (t * 3 + n) * kFrag + lane * 16) = bitcast<u32x4>(fs[n]);
                split8<3>(f2, fs);
#pragma unroll
                for (int n = 0; n < 3; ++n) *reinterpret_cast<u32x4 *>(lds.stage.ds1 + (t * 3 + n) * kFrag + lane * 16) = bitcast<u32x4>(fs[n]);
            }
            __syncthreads();
#pragma unroll
            for (int t = 0; t < 4; ++t)
                if ((t >> 1) <= (wave >> 1)) {
                    bf16x8 b[3];
                    load_frag<3>(lds.stage.u + t * 3 * kFrag, lane, b);
                    x1[t] = product<2>(fo, b, x1[t]);
                    x2[t] = product<2>(fx, b, x2[t]);
                }
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
                bf16x8 b[3];
                load_frag<3>(lds.stage.s0 + t * 3 * kFrag, lane, b);
                aq[t] = product<2>(fo, b, aq[t]);
                az[t] = product<2>(fx, b, az[t]);
                load_frag<3>(lds.stage.ds1 + t * 3 * kFrag, lane, b);
                ay[t] = product<2>(fu, b, ay[t]);
            }
        }
        __syncthreads();                                 // the stage becomes X1, X2
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int jj = row_of(t, m);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = row + e;
                float decay = 0.f;
                if (i >= jj) decay = expf((lds.gate[kSumHi][i] - lds.gate[kSumHi][jj]) + (lds.gate[kSumLo][i] - lds.gate[kSumLo][jj]));
                lds.lower.x1[i][jj] = i >= jj ? p.scale * x1[t][e] * decay : 0.f;
                lds.lower.x2[i][jj] = i > jj ? -x2[t][e] * decay : 0.f;
            }
        }
        float to_last = 0.f;                             // sum over this lane's tokens of k.W
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float gam = lds.gate[kGate][row + e], dec = lds.gate[kToEnd][row + e], rk = lds.gate[kKeyNorm][row + e];
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
                aq[t][e] *= p.scale * gam;
                az[t][e] *= -gam;
                ay[t][e] *= dec;
                to_last += ay[t][e] * rk * element(p.k, p.k_stride_b, p.k_stride_l, p.k_stride_h, t, e);
            }
        }
        __syncthreads();
        const uint8_t *kt = w.ktf + sh * w.kbytes(), *qt = w.qtf + sh * w.kbytes();
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int c = 32 * s + 8 * g;
            float f[8];
            bf16x8 a[3], a2[3];
            if (s <= (wave >> 1)) {                      // rows of X1, X2
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = lds.lower.x1[own][c + e] * lds.gate[kKeyNorm][c + e];
                split8<3>(f, a);
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = lds.lower.x2[own][c + e] * lds.gate[kKeyNorm][c + e];
                split8<3>(f, a2);
#pragma unroll
                for (int t = 0; t < TILES; ++t) {
                    bf16x8 b[NT];
                    load_frag<NT>(kt + (t * 2 + s) * NT * kFrag, lane, b);
                    aq[t] = product<2>(a, b, aq[t]);
                    az[t] = product<2>(a2, b, az[t]);
                }
            }
            if (s >= (wave >> 1)) {                      // their columns
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = lds.lower.x1[c + e][own] * lds.gate[kQueryNorm][c + e];
                split8<3>(f, a);
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = lds.lower.x2[c + e][own] * (lds.gate[kBeta][c + e] * lds.gate[kKeyNorm][c + e]);
                split8<3>(f, a2);
#pragma unroll
                for (int t = 0; t < TILES; ++t) {
                    bf16x8 b[NT];
                    load_frag<NT>(qt + (t * 2 + s) * NT * kFrag, lane, b);
                    ay[t] = product<2>(a, b, ay[t]);
                    load_frag<NT>(kt + (t * 2 + s) * NT * kFrag, lane, b);
                    ay[t] = product<2>(a2, b, ay[t]);
                }
            }
        }
        dxv += __shfl_xor(dxv, 16); dxv += __shfl_xor(dxv, 32);
        if (g == 0) lds.db[own] = dxv;
        inner = wave_sum(inner);
        to_last = wave_sum(to_last);
        if (lane == 0) { lds.inner[wave] = inner; lds.end[wave] = to_last; }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float rk = lds.gate[kKeyNorm][row + e], rq = lds.gate[kQueryNorm][row + e], beta = lds.gate[kBeta][row + e];
            float qd = 0.f, kz = 0.f, ky = 0.f;
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
                const float ke = rk * element(p.k, p.k_stride_b, p.k_stride_l, p.k_stride_h, t, e);
                qd += aq[t][e] * rq * element(p.q, p.q_stride_b, p.q_stride_l, p.q_stride_h, t, e);
                kz += az[t][e] * ke;
                ky += ay[t][e] * ke;
                tq[t][e] += aq[t][e];
                tk[t][e] += beta * az[t][e] + ay[t][e];
            }
            qd = over_columns(qd); kz = over_columns(kz); ky = over_columns(ky);
            if (m == 0) {
                lds.dg[row + e] = qd + beta * kz - ky;
                lds.db[row + e] += kz;
            }
        }
        __syncthreads();
        if (wave == 0) {
            float d = lds.dg[lane];
            if (lane == 63) {
                const float both = (lds.inner[0] + lds.inner[1]) + (lds.inner[2] + lds.inner[3]);
                d += ((lds.end[0] + lds.end[1]) + (lds.end[2] + lds.end[3])) + lds.gate[kGate][63] * both;
            }
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const float other = __shfl_down(d, o);
                if (lane + o < 64) d += other;
            }
            // Nothing stands in front of a sequence's first token for its gate to act on; the terms cancel up to rounding.
            if (lane == 0 && p.initial_states == nullptr && at.lo == sequence_tokens(p, at.n).lo) d = 0.f;
            if (lane < at.count) {
                const int64_t to = ((int64_t)at.b * p.seqlen + at.lo + lane) * p.v_heads + h;
                store_from_float(bp.dg, to, p.g_dtype, d);
                store_from_float(bp.dbeta, to, p.beta_dtype, lds.db[lane]);
            }
        }
        __syncthreads();
    }

    // The lengths' share, and out.
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float rk = lds.gate[kKeyNorm][row + e], rq = lds.gate[kQueryNorm][row + e];
        float dotq = 0.f, dotk = 0.f;
        if (p.qk_l2norm) {
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
                dotq += tq[t][e] * element(p.q, p.q_stride_b, p.q_stride_l, p.q_stride_h, t, e);
                dotk += tk[t][e] * element(p.k, p.k_stride_b, p.k_stride_l, p.k_stride_h, t, e);
            }
            dotq = over_columns(dotq) * rq * rq;
            dotk = over_columns(dotk) * rk * rk;
        }
        if (row + e >= at.count) continue;
        const int64_t tok = at.lo + row + e;
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            const int k = row_of(t, m);
            if (k >= p.dim_k) continue;
            float a = tq[t][e], b = tk[t][e];
            if (p.qk_l2norm) {
                a = rq * (a - dotq * element(p.q, p.q_stride_b, p.q_stride_l, p.q_stride_h, t, e));
                b = rk * (b - dotk * element(p.k, p.k_stride_b, p.k_stride_l, p.k_stride_h, t, e));
            }
            dq[at.b * bp.dq_stride_b + tok * bp.dq_stride_l + k] = Elem<DT>::from_float(a);
            dk[at.b * bp.dk_stride_b + tok * bp.dk_stride_l + k] = Elem<DT>::from_float(b);
        }
    }
}

template <int DT, int KS>
int launch(const cc1d_delta_bwd_params &bp, const ChunkWork &w, hipStream_t stream) {
    const cc1d_delta_params &p = bp.fwd;
    const uint32_t tiles = (uint32_t)(p.dim_v + 15) / 16, nh = (uint32_t)((int64_t)p.sequences * p.v_heads);
    CC1D_LAUNCH((delta_bwd_scan_kernel<DT, KS>), dim3((nh + 7) / 8 * 8 * tiles), dim3(kBlock), 0, stream, bp, w, nh, tiles);
    int st = launch_status();
    if (st != CC1D_OK || w.slots == 0) return st;
    auto rows = [&](const void *x, int64_t b, int64_t l, int64_t h) {
        const int v = vec_elems(p.x_dtype);
        return aligned16(x) && b % v == 0 && l % v == 0 && h % v == 0;
    };
    const int vec_x = rows(bp.dout, bp.dout_stride_b, bp.dout_stride_l, bp.dout_stride_h) && rows(p.v, p.v_stride_b, p.v_stride_l, p.v_stride_h);
    CC1D_LAUNCH((delta_grad_kernel<DT, KS>), dim3((uint32_t)((int64_t)w.slots * p.heads)), dim3(kBlock), sizeof(GradLds<KS>), stream, bp, w, vec_x, (int)(p.dim_v % 4 == 0));
    return launch_status();
}

}  // namespace

int launch_delta_bwd(const cc1d_delta_bwd_params &bp, const ChunkWork &w, hipStream_t stream) {
    return by_type_and_steps(bp.fwd.x_dtype, w.ks, [&](auto dt, auto ks) { return launch<decltype(dt)::value, decltype(ks)::value>(bp, w, stream); });
}

}  // namespace cc1d
