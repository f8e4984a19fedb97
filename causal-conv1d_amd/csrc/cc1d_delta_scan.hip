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
//
// What bounds it is the chain from chunk to chunk, 3800 cycles for 128 x 16 columns in bfloat16: S split and through LDS 550, K S and Q S
// 680, R through LDS 400, T R 700, U through LDS 450, the last products 550, outputs 400.  512 tokens of 32 heads take 19 us.  A chunk's
// operands are 82 KB in 16 bytes a lane, 1300 cycles of a CU's 64 bytes a cycle, and two workgroups on a CU share that: 4096 packed tokens of 32
// heads take 114 us (121 with 104 KB; 156 with one workgroup a CU).  float16, two terms each of K and Q, has 130 KB and 7400 cycles: 16384 tokens of
// 16 heads, 128 workgroups, take 651 us.  The states and U that a training forward writes are bandwidth: 4 x 2048 tokens
// of 16 heads take 118 us without them and 167 with 200 MB of them.  Measured and not taken: 32 columns a workgroup, eight wavefronts
// with O in four of them, a wavefront for all of dim_k without LDS, operands two chunks ahead, results stored four columns at a time.
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

// SAVE: the state in front of every chunk, and U, go to memory for the backward.  K and Q come from the prep kernel's copy:
// read from their own rows, 64 bytes each, they made this kernel 10 to 20 % slower, as much as the copy costs.
template <int DT, int KS, bool SAVE>
__global__ void __launch_bounds__(kBlock, scan_waves(DT, KS))
delta_scan_kernel(const cc1d_delta_params p, const ChunkWork w, const uint32_t heads_total, const uint32_t col_tiles) {
    using T = typename Elem<DT>::type;
    using Bits = typename BitsOf<DT>::type;
    constexpr int NT = Terms<DT>::n, NU = Terms<DT>::p, OUT = NU - 1;
    constexpr int TW = (2 * KS + 3) / 4;                 // 16-row tiles of S a wavefront owns
    __shared__ ScanLds<KS, NU> lds;
    const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // The slices of one head, which read the same operands, on one XCD.
    const uint32_t xcd = blockIdx.x & 7u, idx = blockIdx.x >> 3;
    const uint32_t nh = idx / col_tiles * 8u + xcd;
    if (nh >= heads_total) return;
    int n = (int)divided(nh, w.by_v_heads);
    const int h = (int)nh - n * p.v_heads, hk = (int)divided((uint32_t)h, w.by_group);
    const bool mixed = w.shortest > 0;                   // n is f of a sequence, if there is one
    const int f = n;
    if (mixed) n = sequence_of(p, (int64_t)f * kChunk);
    const TokenRange range = sequence_tokens(p, n);
    if (mixed && !named(range, w, f)) return;
    const int chunks = (int)((range.hi - range.lo + kChunk - 1) / kChunk);
    const int slot0 = first_slot(p, w, n, range), total = (int)(range.hi - range.lo);
    const int col0 = (int)(idx % col_tiles) * 16 + m;
    const bool has_col = col0 < p.dim_v;
    const int col = has_col ? col0 : 0;                  // a column that is there
    // 64 rows are less than 2^31 bytes apart (checked on the host).
    const uint32_t v_pitch = (uint32_t)(p.v_stride_l * (int64_t)sizeof(T)), out_pitch = (uint32_t)(p.out_stride_l * (int64_t)sizeof(T));
    const uint32_t at_col = (uint32_t)col * (uint32_t)sizeof(T);

    T *out = static_cast<T *>(p.out) + range.b * p.out_stride_b + h * p.out_stride_h;
    if (p.cu_seqlens != nullptr && !mixed && has_col) {  // tokens in front of the first sequence and behind the last
        if (n == 0)
            for (int64_t t = wave * 4 + g; t < range.lo; t += 16) out[t * p.out_stride_l + col] = Elem<DT>::from_float(0.f);
        if (n == p.sequences - 1)
            for (int64_t t = range.hi + wave * 4 + g; t < p.seqlen; t += 16) out[t * p.out_stride_l + col] = Elem<DT>::from_float(0.f);
    }

    // Operands of the chunk at hand; each set is asked for again, for the next chunk, once it has been used.  No load stands behind a
    // condition (Row8): what a wavefront has no use for, and what lies behind the last token, is read from a place that exists.
    bf16x8 kf[KS][NT], qf[KS][NT], tf[2][3], pf[2][NU], ktf[TW][2][NT];
    float4 walk;                                         // of token row + (m & 3)
    float last;
    Bits v[4];
    const int64_t kb = w.kbytes(), tb = w.tbytes(), pb = w.pbytes();
    const int steps = (wave >> 1) + 1;                   // of a row of T and P
    const int row = row_of(wave, 4 * g);
    const T *vp = static_cast<const T *>(p.v) + range.b * p.v_stride_b + range.lo * p.v_stride_l + h * p.v_stride_h;
    auto scalars_of = [&](int c) { return w.scalars + ((int64_t)(slot0 + c) * p.v_heads + h) * kScalars * kChunk; };
    auto ask_kq = [&](int c, int i) {                    // step i
        const int64_t at = ((int64_t)(slot0 + c) * p.heads + hk) * kb + (int64_t)(wave * KS + i) * NT * kFrag;
        load_frag<NT>(w.kf + at, lane, kf[i]);
        load_frag<NT>(w.qf + at, lane, qf[i]);
    };
    auto ask_v = [&](int c) {
        // Rows behind the last token take the last one's v: their beta is 0.
        const uint8_t *vc = reinterpret_cast<const uint8_t *>(vp + (int64_t)c * kChunk * p.v_stride_l);
        const int end = total - c * kChunk - 1;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = *reinterpret_cast<const Bits *>(vc + ((uint32_t)(row + e < end ? row + e : end) * v_pitch + at_col));
    };
    auto ask_t = [&](int c, int i) {
        load_frag<3>(w.tf + ((int64_t)(slot0 + c) * p.v_heads + h) * tb + lower_frag(wave, i) * 3 * kFrag, lane, tf[i]);
    };
    auto ask_walk = [&](int c) { walk = *reinterpret_cast<const float4 *>(scalars_of(c) + 4 * (row + (m & 3))); };
    auto ask_p = [&](int c, int i) {
        load_frag<NU>(w.pf + ((int64_t)(slot0 + c) * p.v_heads + h) * pb + lower_frag(wave, i) * NU * kFrag, lane, pf[i]);
    };
    auto ask_kt = [&](int c, int i) {                    // tile i of this wavefront's
        const int t = wave * TW + i < 2 * KS ? wave * TW + i : 0;
        const uint8_t *kt = w.ktf + ((int64_t)(slot0 + c) * p.heads + hk) * kb;
#pragma unroll
        for (int j = 0; j < 2; ++j) load_frag<NT>(kt + (t * 2 + j) * NT * kFrag, lane, ktf[i][j]);
    };
    auto ask_last = [&](int c) { last = scalars_of(c)[kGate * kChunk + 63]; };
    auto put = [&](uint8_t *base, int terms, int tile, int n_, const u32x2 &x) {  // a tile's half of a right operand
        *reinterpret_cast<u32x2 *>(base + ((tile >> 1) * terms + n_) * kFrag + lane * 16 + (tile & 1) * 8) = x;
    };
    if (chunks > 0) {
#pragma unroll
        for (int i = 0; i < KS; ++i) ask_kq(0, i);
        ask_v(0);
        ask_walk(0);
        ask_last(0);
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (i < steps) ask_t(0, i);
#pragma unroll
        for (int i = 0; i < TW; ++i) ask_kt(0, i);
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (i < steps) ask_p(0, i);
    }

    f32x4 s[TW];
#pragma unroll
    for (int i = 0; i < TW; ++i) s[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (p.initial_states != nullptr) {
        const float *from = p.initial_states + n * p.init_stride_n + h * p.init_stride_h + col;
#pragma unroll
        for (int i = 0; i < TW; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int t = wave * TW + i, k = row_of(t, 4 * g + e);
                s[i][e] = from[(t < 2 * KS && k < p.dim_k ? k : 0) * p.init_stride_k];
            }
#pragma unroll
        for (int i = 0; i < TW; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int t = wave * TW + i, k = row_of(t, 4 * g + e);
                if (t >= 2 * KS || k >= p.dim_k || !has_col) s[i][e] = 0.f;
            }
    }

    for (int c = 0; c < chunks; ++c) {
        const int next = c + 1 < chunks ? c + 1 : c;
        const int64_t sv = (int64_t)(slot0 + c) * p.v_heads + h;
#pragma unroll
        for (int i = 0; i < TW; ++i) {
            const int t = wave * TW + i;
            if (t >= 2 * KS) break;
            const float x[4] = {s[i][0], s[i][1], s[i][2], s[i][3]};
            u32x2 f[3];
            split4<3>(x, f);
#pragma unroll
            for (int q = 0; q < 3; ++q) put(lds.s, 3, t, q, f[q]);
            if (SAVE && has_col) {
                float *to = w.s0 + sv * p.dim_k * p.dim_v;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int k = row_of(t, 4 * g + e);
                    if (k < p.dim_k) to[(uint32_t)(k * p.dim_v + col)] = x[e];
                }
            }
        }
        lds_barrier();
        const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
        f32x4 o = zero, o2 = zero, ks = zero, ks2 = zero;
        {
            bf16x8 b[2][3];
            load_frag<3>(lds.s, lane, b[0]);
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                if (i + 1 < KS) load_frag<3>(lds.s + (i + 1) * 3 * kFrag, lane, b[(i + 1) & 1]);
                stay();
                product2<2>(kf[i], b[i & 1], ks, ks2);
                product2<OUT>(qf[i], b[i & 1], o, o2);
                stay();
                ask_kq(next, i);
            }
        }
        {
            ks += ks2;
            o += o2;
            float x[4], sn[4], bt[4], rd[4];
            of_quad(walk.x, sn);
            of_quad(walk.y, bt);
            of_quad(walk.z, rd);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[e] = bt[e] * Elem<DT>::to_float(bitcast<T>(v[e])) - sn[e] * ks[e];
                o[e] *= rd[e];
            }
            u32x2 f[3];
            split4<3>(x, f);
#pragma unroll
            for (int q = 0; q < 3; ++q) put(lds.r, 3, wave, q, f[q]);
        }
        lds_barrier();
        {
            bf16x8 b[2][3];
            f32x4 u = zero, u2 = zero;
#pragma unroll
            for (int i = 0; i < 2; ++i) load_frag<3>(lds.r + i * 3 * kFrag, lane, b[i]);
            stay();
            product2<2>(tf[0], b[0], u, u2);
            stay();
            ask_v(next);
            if (steps == 2) product2<2>(tf[1], b[1], u, u2);
            stay();
            ask_t(next, 0);
            if (steps == 2) ask_t(next, 1);
            u += u2;
            float carry[4];
            of_quad(walk.w, carry);
            const float x[4] = {u[0], u[1], u[2], u[3]}, y[4] = {x[0] * carry[0], x[1] * carry[1], x[2] * carry[2], x[3] * carry[3]};
            u32x2 f[3], fu[NU];
            split4<3>(y, f);
#pragma unroll
            for (int q = 0; q < 3; ++q) put(lds.d, 3, wave, q, f[q]);
            split4<NU>(x, fu);
#pragma unroll
            for (int q = 0; q < NU; ++q) put(lds.u, NU, wave, q, fu[q]);
            if (SAVE && has_col) {
                float *to = w.u + sv * kChunk * p.dim_v;
#pragma unroll
                for (int e = 0; e < 4; ++e) to[(uint32_t)((row + e) * p.dim_v + col)] = x[e];
            }
        }
        lds_barrier();
        {
            bf16x8 b[2][3], bu[2][NU];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                load_frag<3>(lds.d + q * 3 * kFrag, lane, b[q]);
                load_frag<NU>(lds.u + q * NU * kFrag, lane, bu[q]);
            }
            stay();
            ask_walk(next);
#pragma unroll
            for (int i = 0; i < TW; ++i) {
                if (wave * TW + i >= 2 * KS) break;
                f32x4 small = zero;
                s[i] *= last;
#pragma unroll
                for (int q = 0; q < 2; ++q) product2<2>(ktf[i][q], b[q], s[i], small);
                s[i] += small;
                stay();
                ask_kt(next, i);
            }
            f32x4 small = zero;
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (i < steps) product2<OUT>(pf[i], bu[i], o, small);
            o += small;
            stay();
            ask_p(next, 0);
            if (steps == 2) ask_p(next, 1);
            ask_last(next);
        }
        if (has_col) {
            uint8_t *oc = reinterpret_cast<uint8_t *>(out + (range.lo + (int64_t)c * kChunk) * p.out_stride_l);
            auto store = [&](int e) { *reinterpret_cast<T *>(oc + ((uint32_t)(row + e) * out_pitch + at_col)) = Elem<DT>::from_float(o[e]); };
            const int left = total - c * kChunk;
            if (left >= kChunk) {
#pragma unroll
                for (int e = 0; e < 4; ++e) store(e);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (row + e < left) store(e);
            }
        }
    }
    if (p.final_states == nullptr || !has_col) return;
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

template <int DT, int KS, bool SAVE>
int launch(const cc1d_delta_params &p, const ChunkWork &w, hipStream_t stream) {
    const uint32_t tiles = (uint32_t)(p.dim_v + 15) / 16, nh = (uint32_t)(w.walks(p) * p.v_heads);
    CC1D_LAUNCH((delta_scan_kernel<DT, KS, SAVE>), dim3((nh + 7) / 8 * 8 * tiles), dim3(kBlock), 0, stream, p, w, nh, tiles);
    return launch_status();
}
}  // namespace

int launch_delta_scan(const cc1d_delta_params &p, const ChunkWork &w, bool save, hipStream_t stream) {
    return by_type_and_steps(p.x_dtype, w.ks, [&](auto dt, auto ks) {
        constexpr int DT = decltype(dt)::value, KS = decltype(ks)::value;
        return save ? launch<DT, KS, true>(p, w, stream) : launch<DT, KS, false>(p, w, stream);
    });
}

}  // namespace cc1d
