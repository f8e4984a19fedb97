// The gated delta rule by chunks, backward (cc1d_delta_chunk.hpp).  The states in front of the chunks and U come from the forward,
// T and P are made again (prep kernel); then, with dS1 the gradient of the state behind a chunk:
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
// Heads that share q and k leave their dQ and dK in fp32, and a last launch adds them up in their order: no atomics, the same bits
// every time (one workgroup for all heads of a key, adding in registers, was slower at every size: 4 x 2048 tokens of 8 and 16 heads
// 656 us for forward and backward and 637 now, 512 tokens of 2 and 16 heads 224 and 106).
//
// 4 x 2048 tokens of 16 heads of 128 x 128 in bfloat16, 2048 chunks: prep 54 us, scan 190, gradients 215.  The scan's chain is
// the forward's with one product more, and it writes 200 MB for the gradients.  Those read 550 MB and write 67, 2.9 TB/s: a third of a
// workgroup's time (24 us, one a CU) is the part behind the walk over dim_v, where nothing is on its way from memory.  Persistent workgroups that
// ask for their next chunk in that part were no faster (224 us): 38 to 70 registers more.
#include "cc1d_delta_chunk.hpp"
#include "cc1d_delta_host.hpp"

namespace cc1d {
namespace {

template <int DT, int KS>
struct BwdScanLds {
    uint8_t s[KS * 3 * kFrag];                           // dS1
    uint8_t o[2 * Terms<DT>::n * kFrag];                 // dO
    uint8_t q[2][2 * 3 * kFrag];                         // scale gam rq dO, this chunk's and the last one's (no barrier between their use)
    uint8_t u[2 * 3 * kFrag];                            // dU
    uint8_t x[2 * 3 * kFrag];                            // -beta gam rk dX
};

template <int DT, int KS>
__global__ void __launch_bounds__(kBlock, scan_waves(DT, KS))
delta_bwd_scan_kernel(const cc1d_delta_bwd_params bp, const ChunkWork w, const uint32_t heads_total, const uint32_t col_tiles) {
    using T = typename Elem<DT>::type;
    using Bits = typename BitsOf<DT>::type;
    constexpr int NT = Terms<DT>::n;
    constexpr int TW = (2 * KS + 3) / 4;                 // 16-row tiles of dS a wavefront owns
    __shared__ BwdScanLds<DT, KS> lds;
    const cc1d_delta_params &p = bp.fwd;
    const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t xcd = blockIdx.x & 7u, idx = blockIdx.x >> 3;
    const uint32_t nh = idx / col_tiles * 8u + xcd;
    if (nh >= heads_total) return;
    const int n = (int)divided(nh, w.by_v_heads), h = (int)nh - n * p.v_heads, hk = (int)divided((uint32_t)h, w.by_group);
    const TokenRange range = sequence_tokens(p, n);
    const int chunks = (int)((range.hi - range.lo + kChunk - 1) / kChunk);
    const int slot0 = first_slot(p, w, n, range), total = (int)(range.hi - range.lo);
    const int col0 = (int)(idx % col_tiles) * 16 + m;
    const bool has_col = col0 < p.dim_v;
    const int col = has_col ? col0 : 0;                  // a column that is there
    const uint32_t do_pitch = (uint32_t)(bp.dout_stride_l * (int64_t)sizeof(T)), dv_pitch = (uint32_t)(bp.dv_stride_l * (int64_t)sizeof(T));
    const uint32_t at_col = (uint32_t)col * (uint32_t)sizeof(T);

    T *dv = static_cast<T *>(bp.dv) + range.b * bp.dv_stride_b + h * bp.dv_stride_h;
    if (p.cu_seqlens != nullptr && has_col) {            // tokens in front of the first sequence and behind the last
        if (n == 0)
            for (int64_t t = wave * 4 + g; t < range.lo; t += 16) dv[t * bp.dv_stride_l + col] = Elem<DT>::from_float(0.f);
        if (n == p.sequences - 1)
            for (int64_t t = range.hi + wave * 4 + g; t < p.seqlen; t += 16) dv[t * bp.dv_stride_l + col] = Elem<DT>::from_float(0.f);
    }

    // As in the scan of the forward: operands asked for again between the products that have used them, without conditions.
    bf16x8 kf[KS][NT], tf[2][3], pf[2][3], ktf[TW][2][NT], qtf[TW][2][NT];
    float4 walk;                                         // of token row + (m & 3)
    float last;
    Bits d[4];
    const int64_t kb = w.kbytes(), tb = w.tbytes();
    const int from = wave >> 1;                          // first step of a row of T^T and P^T
    const int row = row_of(wave, 4 * g);
    const T *dop = static_cast<const T *>(bp.dout) + range.b * bp.dout_stride_b + range.lo * bp.dout_stride_l + h * bp.dout_stride_h;
    auto scalars_of = [&](int c) { return w.scalars + ((int64_t)(slot0 + c) * p.v_heads + h) * kScalars * kChunk; };
    auto ask_k = [&](int c, int i) { load_frag<NT>(w.kf + ((int64_t)(slot0 + c) * p.heads + hk) * kb + (int64_t)(wave * KS + i) * NT * kFrag, lane, kf[i]); };
    auto ask_p = [&](int c, int i) { load_frag<3>(w.ptf + ((int64_t)(slot0 + c) * p.v_heads + h) * tb + upper_frag(wave, i) * 3 * kFrag, lane, pf[i]); };
    auto ask_t = [&](int c, int i) { load_frag<3>(w.ttf + ((int64_t)(slot0 + c) * p.v_heads + h) * tb + upper_frag(wave, i) * 3 * kFrag, lane, tf[i]); };
    auto ask_d = [&](int c) {
        const uint8_t *dc = reinterpret_cast<const uint8_t *>(dop + (int64_t)c * kChunk * bp.dout_stride_l);
        const int end = total - c * kChunk - 1;
#pragma unroll
        for (int e = 0; e < 4; ++e) d[e] = *reinterpret_cast<const Bits *>(dc + ((uint32_t)(row + e < end ? row + e : end) * do_pitch + at_col));
    };
    auto ask_walk = [&](int c) { walk = *reinterpret_cast<const float4 *>(scalars_of(c) + 4 * (row + (m & 3))); };
    auto ask_last = [&](int c) { last = scalars_of(c)[kGate * kChunk + 63]; };
    auto ask_kt = [&](int c, int i) {
        const int64_t at = ((int64_t)(slot0 + c) * p.heads + hk) * kb + (int64_t)(wave * TW + i < 2 * KS ? wave * TW + i : 0) * 2 * NT * kFrag;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            load_frag<NT>(w.ktf + at + j * NT * kFrag, lane, ktf[i][j]);
            load_frag<NT>(w.qtf + at + j * NT * kFrag, lane, qtf[i][j]);
        }
    };
    auto put = [&](uint8_t *base, int terms, int tile, int n_, const u32x2 &x) {
        *reinterpret_cast<u32x2 *>(base + ((tile >> 1) * terms + n_) * kFrag + lane * 16 + (tile & 1) * 8) = x;
    };
    if (chunks > 0) {
        const int c = chunks - 1;
        ask_d(c);
#pragma unroll
        for (int i = 0; i < KS; ++i) ask_k(c, i);
        ask_walk(c);
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (i >= from) ask_p(c, i);
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (i >= from) ask_t(c, i);
        ask_last(c);
#pragma unroll
        for (int i = 0; i < TW; ++i) ask_kt(c, i);
    }

    f32x4 s[TW];
#pragma unroll
    for (int i = 0; i < TW; ++i) s[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (bp.dfinal_states != nullptr) {
        const float *from = bp.dfinal_states + n * bp.dfinal_stride_n + h * bp.dfinal_stride_h + col;
#pragma unroll
        for (int i = 0; i < TW; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int t = wave * TW + i, k = row_of(t, 4 * g + e);
                s[i][e] = from[(t < 2 * KS && k < p.dim_k ? k : 0) * bp.dfinal_stride_k];
            }
#pragma unroll
        for (int i = 0; i < TW; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int t = wave * TW + i, k = row_of(t, 4 * g + e);
                if (t >= 2 * KS || k >= p.dim_k || !has_col) s[i][e] = 0.f;
            }
    }

    for (int c = chunks - 1; c >= 0; --c) {
        const int next = c > 0 ? c - 1 : 0, left = total - c * kChunk;
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
            if (has_col) {
                float *to = w.ds1 + sv * p.dim_k * p.dim_v;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int k = row_of(t, 4 * g + e);
                    if (k < p.dim_k) to[(uint32_t)(k * p.dim_v + col)] = s[i][e];
                }
            }
        }
        {
            // Rows behind the last token have no dout.
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = left >= kChunk || row + e < left ? Elem<DT>::to_float(bitcast<T>(d[e])) : 0.f;
            float read[4];
            of_quad(walk.z, read);
            const float y[4] = {x[0] * read[0], x[1] * read[1], x[2] * read[2], x[3] * read[3]};
            u32x2 fo[NT], f[3];
            split4<NT>(x, fo);
#pragma unroll
            for (int j = 0; j < NT; ++j) put(lds.o, NT, wave, j, fo[j]);
            split4<3>(y, f);
#pragma unroll
            for (int j = 0; j < 3; ++j) put(lds.q[c & 1], 3, wave, j, f[j]);
        }
        lds_barrier();
        f32x4 u = {0.f, 0.f, 0.f, 0.f}, u2 = u, o = u, o2 = u;
        {
            bf16x8 b[2][3], bo[2][NT];
            load_frag<3>(lds.s, lane, b[0]);
#pragma unroll
            for (int i = 0; i < 2; ++i) load_frag<NT>(lds.o + i * NT * kFrag, lane, bo[i]);
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                if (i + 1 < KS) load_frag<3>(lds.s + (i + 1) * 3 * kFrag, lane, b[(i + 1) & 1]);
                stay();
                product2<2>(kf[i], b[i & 1], u, u2);
                if (i == 0) {
                    if (from == 0) product2<2>(pf[0], bo[0], o, o2);
                    product2<2>(pf[1], bo[1], o, o2);
                }
                stay();
                ask_k(next, i);
                if (i == 0) {
                    if (from == 0) ask_p(next, 0);
                    ask_p(next, 1);
                }
            }
        }
        const float4 now = walk;                             // the next chunk's are needed at its start
        ask_walk(next);
        ask_d(next);
        {
            u += u2;
            o += o2;
            float carry[4];
            of_quad(now.w, carry);
            const float x[4] = {u[0] * carry[0] + o[0], u[1] * carry[1] + o[1], u[2] * carry[2] + o[2], u[3] * carry[3] + o[3]};
            u32x2 f[3];
            split4<3>(x, f);
#pragma unroll
            for (int j = 0; j < 3; ++j) put(lds.u, 3, wave, j, f[j]);
        }
        lds_barrier();
        f32x4 x = {0.f, 0.f, 0.f, 0.f}, x2 = x;
        {
            bf16x8 b[2][3];
#pragma unroll
            for (int i = 0; i < 2; ++i) load_frag<3>(lds.u + i * 3 * kFrag, lane, b[i]);
            stay();
            if (from == 0) product2<2>(tf[0], b[0], x, x2);
            stay();
            product2<2>(tf[1], b[1], x, x2);
            stay();
            if (from == 0) ask_t(next, 0);
            ask_t(next, 1);
            x += x2;
        }
        {
            float seen[4], beta[4];
            of_quad(now.x, seen);
            of_quad(now.y, beta);
            const float y[4] = {-seen[0] * x[0], -seen[1] * x[1], -seen[2] * x[2], -seen[3] * x[3]}, bx[4] = {beta[0] * x[0], beta[1] * x[1], beta[2] * x[2], beta[3] * x[3]};
            u32x2 f[3];
            split4<3>(y, f);
#pragma unroll
            for (int j = 0; j < 3; ++j) put(lds.x, 3, wave, j, f[j]);
            if (has_col) {
                float *to = w.dx + sv * kChunk * p.dim_v;
                uint8_t *dc = reinterpret_cast<uint8_t *>(dv + (range.lo + (int64_t)c * kChunk) * bp.dv_stride_l);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    to[(uint32_t)((row + e) * p.dim_v + col)] = x[e];
                    if (left >= kChunk || row + e < left) *reinterpret_cast<T *>(dc + ((uint32_t)(row + e) * dv_pitch + at_col)) = Elem<DT>::from_float(bx[e]);
                }
            }
        }
        lds_barrier();
        {
            bf16x8 bq[2][3], bx[2][3];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                load_frag<3>(lds.q[c & 1] + j * 3 * kFrag, lane, bq[j]);
                load_frag<3>(lds.x + j * 3 * kFrag, lane, bx[j]);
            }
            stay();
#pragma unroll
            for (int i = 0; i < TW; ++i) {
                if (wave * TW + i >= 2 * KS) break;
                f32x4 small = {0.f, 0.f, 0.f, 0.f};
                s[i] *= last;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    product2<2>(qtf[i][j], bq[j], s[i], small);
                    product2<2>(ktf[i][j], bx[j], s[i], small);
                }
                s[i] += small;
                stay();
                ask_kt(next, i);
            }
            ask_last(next);
        }
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

constexpr int kGradBlock = 512;

// 32 columns of U, dX, S0 and dS1 as operands.  A lane's 16 bytes lie turned by 2 g places among the 16 of its group: lanes that have
// a row between them, 4 columns each, then write to different banks.
template <int KS>
struct GradStage {
    uint8_t u[4 * 3 * kFrag], x[4 * 3 * kFrag], s0[2 * KS * 3 * kFrag], ds1[2 * KS * 3 * kFrag];
    static constexpr int kCopies = KS <= 4 ? 2 : 1;      // as many as there is room for
};
// X1 and X2 as left operands: their rows (contraction over columns), scaled by rk of the column, in fp32; their columns
// (contraction over rows), scaled by rq, and by beta rk, of the row, split as operands.
struct GradLower { float rows[2][kChunk][68]; uint8_t columns[2][kTriFrags * 3 * kFrag]; };
template <int KS>
struct GradLds {
    union { GradStage<KS> stage[GradStage<KS>::kCopies]; GradLower lower; };
    float gate[kScalars][kChunk];
    float sums[2][3][kChunk];                            // q.dQ, k.Z, k.Y of each token, of either half of dim_k
    float db[kChunk], end[8], inner[8];
};

// dQ and dK leave through LDS, in whole rows; BOTH: at once.
template <int KS> constexpr int kOutPitch = 32 * KS + 8;
template <int DT, int KS> constexpr size_t kOutBytes = 2 * kChunk * kOutPitch<KS> * sizeof(typename Elem<DT>::type);
template <int DT, int KS> constexpr bool kJoinBoth = kOutBytes<DT, KS> <= 64 * 1024;
template <int DT, int KS, bool BOTH>
__device__ __forceinline__ void rows_leave(const f32x4 (&tq)[KS], const f32x4 (&tk)[KS], void *lds, const cc1d_delta_bwd_params &bp, const ChunkAt &at, int hk, int vec_out) {
    using T = typename Elem<DT>::type;
    constexpr int PITCH = kOutPitch<KS>;
    const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), tile = wave & 3, side = wave >> 2, row = row_of(tile, 4 * g);
    auto write = [&](const f32x4 (&v)[KS], T *rows) {
#pragma unroll
        for (int t = 0; t < KS; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) rows[(row + e) * PITCH + row_of(side * KS + t, m)] = Elem<DT>::from_float(v[t][e]);
    };
    auto leave = [&](const T *rows, T *to, int64_t sb, int64_t sl) {
        T *base = to + at.b * sb + at.lo * sl;
        for (int i = threadIdx.x; i < at.count * 4 * KS; i += kGradBlock) {    // 8 elements a lane
            const int token = i / (4 * KS), c = i % (4 * KS) * 8;
            if (c >= bp.fwd.dim_k) continue;
            const T *from = rows + token * PITCH + c;
            T *d = base + token * sl + c;
            if (vec_out && c + 8 <= bp.fwd.dim_k) {
#pragma unroll
                for (int v4 = 0; v4 < (int)sizeof(T) / 2; ++v4) reinterpret_cast<u32x4 *>(d)[v4] = reinterpret_cast<const u32x4 *>(from)[v4];
            } else {
                for (int e = 0; e < 8 && c + e < bp.fwd.dim_k; ++e) d[e] = from[e];
            }
        }
    };
    T *first = static_cast<T *>(lds), *second = first + (BOTH ? kChunk * PITCH : 0);
    write(tq, first);
    if (BOTH) write(tk, second);
    lds_barrier();
    leave(first, static_cast<T *>(bp.dq) + hk * bp.dq_stride_h, bp.dq_stride_b, bp.dq_stride_l);
    if (!BOTH) {
        lds_barrier();
        write(tk, second);
        lds_barrier();
    }
    leave(second, static_cast<T *>(bp.dk) + hk * bp.dk_stride_h, bp.dk_stride_b, bp.dk_stride_l);
}

// Every chunk's gradients alone.  Eight wavefronts: 16 tokens' rows of dQ, Z and Y each, of one half of dim_k; of X1 the first
// four, of X2 the others.  S0, dS1, dX and U pass through LDS once for all of them, 32 columns of dim_v at a time, split into their
// terms: eight lanes fetch a row's 128 bytes, and while the products of one step are under way other wavefronts split the
// next step's numbers into the other copy.  VEC: rows of v and dout are whole 16-byte vectors, rows of the fp32 matrices in the workspace too.
// A workgroup takes one value head; where several share a key head their shares of dq and dk go to the workspace in fp32.
template <int DT, int KS, bool VEC>
__global__ void __launch_bounds__(kGradBlock, 1)
delta_grad_kernel(const cc1d_delta_bwd_params bp, const ChunkWork w, const int vec_out) {
    using T = typename Elem<DT>::type;
    constexpr int NT = Terms<DT>::n;
    constexpr int TILES = KS, OWN = (2 * KS + 3) / 4;    // 16-column tiles of a half; that two wavefronts bring to LDS
    extern __shared__ uint4 raw[];
    GradLds<KS> &lds = *reinterpret_cast<GradLds<KS> *>(raw);
    const cc1d_delta_params &p = bp.fwd;
    const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), tile = wave & 3, side = wave >> 2;
    const int slot = (int)divided(blockIdx.x, w.by_v_heads), h = (int)blockIdx.x - slot * p.v_heads, hk = (int)divided((uint32_t)h, w.by_group);
    const ChunkAt at = chunk_at(p, w, slot);
    if (p.cu_seqlens != nullptr && slot == 0) {          // tokens in front of the first sequence and behind the last
        T *dq = static_cast<T *>(bp.dq) + hk * bp.dq_stride_h, *dk = static_cast<T *>(bp.dk) + hk * bp.dk_stride_h;     // (all heads of a group zeros)
        auto clear = [&](int64_t lo, int64_t hi) {
            for (int64_t t = lo + wave; t < hi; t += 8) {
                for (int k = lane; k < p.dim_k; k += 64) {
                    dq[t * bp.dq_stride_l + k] = Elem<DT>::from_float(0.f);
                    dk[t * bp.dk_stride_l + k] = Elem<DT>::from_float(0.f);
                }
                if (lane == 0) {
                    store_from_float(bp.dg, t * p.v_heads + h, p.g_dtype, 0.f);
                    store_from_float(bp.dbeta, t * p.v_heads + h, p.beta_dtype, 0.f);
                }
            }
        };
        clear(0, sequence_tokens(p, 0).lo);
        clear(sequence_tokens(p, p.sequences - 1).hi, p.seqlen);
    }
    if (at.count <= 0) return;
    const int64_t sh = (int64_t)slot * p.heads + hk, sv = (int64_t)slot * p.v_heads + h;
    const int own = row_of(tile, m);                     // the token whose row this lane holds as a left operand
    const int row = row_of(tile, 4 * g);                 // the first of the four whose results it holds
    const int half = tile >> 1;                          // where those four stand in K^T, Q^T: step, and first or second four
    const bool upper = tile & 1;
    const int cols = own < at.count ? p.dim_v : 0;
    const bool cut_k = p.dim_k < 32 * KS;
    const uint8_t *kt = w.ktf + sh * w.kbytes() + side * TILES * 2 * NT * kFrag, *qt = w.qtf + sh * w.kbytes() + side * TILES * 2 * NT * kFrag;

    // K^T and Q^T of the half of the chunk that holds this wavefront's own tokens; q.dQ and k.dK of those tokens.
    bf16x8 bk[TILES][NT], bq[TILES][NT];
    f32x4 tq[TILES], tk[TILES];                          // dQ, dK
    float rk[4], rq[4], dotq[4], dotk[4];

    {
        f32x4 aq[TILES], az[TILES], ay[TILES], x[4];
#pragma unroll
        for (int t = 0; t < TILES; ++t) { aq[t] = (f32x4){0.f, 0.f, 0.f, 0.f}; az[t] = aq[t]; ay[t] = aq[t]; }
#pragma unroll
        for (int t = 0; t < 4; ++t) x[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
        float inner = 0.f, dxv = 0.f;
        const T *dop = static_cast<const T *>(bp.dout) + at.b * bp.dout_stride_b + (at.lo + (cols ? own : 0)) * bp.dout_stride_l + h * bp.dout_stride_h;
        // What 32 columns of v need, asked for a step ahead: this lane's row of dO as a left operand, and of everything else 4 columns
        // of a row: eight rows of a tile are one wavefront's, the other eight its neighbour's.
        const int in_tile = (wave & 1) * 8 + (lane >> 3), c4 = 4 * (lane & 7), brought = row_of(wave >> 1, in_tile);
        const int place = (((lane & 7) >> 1) * 16 + ((in_tile + 2 * ((lane & 7) >> 1)) & 15)) * 16 + (lane & 1) * 8;
        const int turned = g * 16 + ((m + 2 * g) & 15);  // the lane whose place in the stage is this one's operand
        const T *vp = static_cast<const T *>(p.v) + at.b * p.v_stride_b + (at.lo + (brought < at.count ? brought : 0)) * p.v_stride_l + h * p.v_stride_h;
        Row8<DT, VEC> ro;
        Row4<DT, VEC> rv;
        Row4<CC1D_F32, VEC> rx, ru, rs[OWN], rd[OWN];
        const float *s0 = w.s0 + sv * p.dim_k * p.dim_v, *ds1 = w.ds1 + sv * p.dim_k * p.dim_v;
        const float *xp = w.dx + sv * kChunk * p.dim_v + (uint32_t)(brought * p.dim_v), *up = w.u + sv * kChunk * p.dim_v + (uint32_t)(brought * p.dim_v);
        auto ask = [&](int v0) {
            ro.ask(dop, v0 + 8 * g, cols);
            const int c = v0 + c4;
            rv.ask(vp, c, p.dim_v);
            rx.ask(xp, c, p.dim_v);
            ru.ask(up, c, p.dim_v);
#pragma unroll
            for (int i = 0; i < OWN; ++i) {
                const int t = (wave >> 1) + 4 * i, k = row_of(t, in_tile);
                const uint32_t to = (uint32_t)((t < 2 * KS && k < p.dim_k ? k : 0) * p.dim_v);
                rs[i].ask(s0 + to, c, p.dim_v);
                rd[i].ask(ds1 + to, c, p.dim_v);
            }
        };
        bf16x8 fo[NT];
        auto bring = [&](int v0, GradStage<KS> &stage) {
            const int c = v0 + c4;
            const bool cut = v0 + 32 > p.dim_v;
            float f[4], f2[4];
            u32x2 f3[3];
            auto put = [&](uint8_t *base, int t) {
#pragma unroll
                for (int n = 0; n < 3; ++n) *reinterpret_cast<u32x2 *>(base + (t * 3 + n) * kFrag + place) = f3[n];
            };
            ro.template operand<NT>(v0 + 8 * g, cols, true, fo);
            rx.get(c, p.dim_v, cut, f);
            rv.get(c, p.dim_v, cut, f2);
#pragma unroll
            for (int e = 0; e < 4; ++e) dxv += f[e] * f2[e];
            split4<3>(f, f3);
            put(stage.x, wave >> 1);
            ru.get(c, p.dim_v, cut, f);
            split4<3>(f, f3);
            put(stage.u, wave >> 1);
#pragma unroll
            for (int i = 0; i < OWN; ++i) {
                const int t = (wave >> 1) + 4 * i;
                if (t >= 2 * KS) break;
                const int in = row_of(t, in_tile) < p.dim_k ? p.dim_v : 0;
                rs[i].get(c, in, cut || cut_k, f);
                rd[i].get(c, in, cut || cut_k, f2);
#pragma unroll
                for (int e = 0; e < 4; ++e) inner += f[e] * f2[e];
                split4<3>(f, f3);
                put(stage.s0, t);
                split4<3>(f2, f3);
                put(stage.ds1, t);
            }
        };
        ask(0);
        for (int i = threadIdx.x; i < kScalars * kChunk; i += kGradBlock) (&lds.gate[0][0])[i] = w.scalars[sv * kScalars * kChunk + i];
        bring(0, lds.stage[0]);
        if (32 < p.dim_v) ask(32);
        lds_barrier();
        constexpr int COPIES = GradStage<KS>::kCopies;
        for (int v0 = 0; v0 < p.dim_v; v0 += 32) {
            const GradStage<KS> &stage = lds.stage[COPIES == 2 ? (v0 >> 5) & 1 : 0];
            bf16x8 fx[3], fu[3];
            load_frag<3>(stage.x + tile * 3 * kFrag, turned, fx);
            load_frag<3>(stage.u + tile * 3 * kFrag, turned, fu);
#pragma unroll
            for (int t = 0; t < 4; ++t)
                if ((t >> 1) <= half) {
                    bf16x8 b[3];
                    load_frag<3>(stage.u + t * 3 * kFrag, turned, b);
                    x[t] = side == 0 ? product<2>(fo, b, x[t]) : product<2>(fx, b, x[t]);
                    stay();
                }
            const uint8_t *sl = stage.s0 + side * TILES * 3 * kFrag, *dl = stage.ds1 + side * TILES * 3 * kFrag;
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
                bf16x8 b[3], d[3];
                load_frag<3>(sl + t * 3 * kFrag, turned, b);
                load_frag<3>(dl + t * 3 * kFrag, turned, d);
                aq[t] = product<2>(fo, b, aq[t]);
                az[t] = product<2>(fx, b, az[t]);
                ay[t] = product<2>(fu, d, ay[t]);
                stay();
            }
            if (v0 + 32 < p.dim_v) {
                if (COPIES == 1) lds_barrier();          // the step has been read
                bring(v0 + 32, lds.stage[COPIES == 2 ? ((v0 >> 5) + 1) & 1 : 0]);
                stay();
                if (v0 + 64 < p.dim_v) ask(v0 + 64);
                lds_barrier();
            }
        }
        auto ask_kq = [&](int s) {
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
                load_frag<NT>(kt + (t * 2 + s) * NT * kFrag, lane, bk[t]);
                load_frag<NT>(qt + (t * 2 + s) * NT * kFrag, lane, bq[t]);
            }
        };
        ask_kq(half);
        lds_barrier();                                   // the stage becomes X1, X2
        float beta[4], hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            rk[e] = lds.gate[kKeyNorm][row + e]; rq[e] = lds.gate[kQueryNorm][row + e]; beta[e] = lds.gate[kBeta][row + e];
            hi[e] = lds.gate[kSumHi][row + e]; lo[e] = lds.gate[kSumLo][row + e];
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            if ((t >> 1) > half) continue;
            const int jj = row_of(t, m);
            const float rj = lds.gate[kKeyNorm][jj], hj = lds.gate[kSumHi][jj], lj = lds.gate[kSumLo][jj];
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float d = x[t][e] * exp_of((hi[e] - hj) + (lo[e] - lj));
                const float z = side == 0 ? (row + e >= jj ? p.scale * d : 0.f) : (row + e > jj ? -d : 0.f);
                lds.lower.rows[side][row + e][jj] = z * rj;
                y[e] = z * (side == 0 ? rq[e] : beta[e] * rk[e]);
            }
            // Column jj as a row of the transposed matrix: tile t, four of its elements from token `row` on.
            u32x2 f[3];
            split4<3>(y, f);
            uint8_t *to = lds.lower.columns[side] + upper_frag(t, half) * 3 * kFrag + (g * 16 + m) * 16 + (tile & 1) * 8;
#pragma unroll
            for (int n = 0; n < 3; ++n) *reinterpret_cast<u32x2 *>(to + n * kFrag) = f[n];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float gam = lds.gate[kGate][row + e], dec = lds.gate[kToEnd][row + e];
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
                aq[t][e] *= p.scale * gam;
                az[t][e] *= -gam;
                ay[t][e] *= dec;
            }
        }
        dxv += dpp_moved<0xB1>(dxv);                     // over the eight lanes of a row
        dxv += dpp_moved<0x4E>(dxv);
        dxv += dpp_moved<0x141>(dxv);                    // row_half_mirror
        if ((lane & 7) == 0) lds.db[brought] = dxv;
        lds_barrier();
        // Rows of X1 and X2 against K, their columns against Q and K.  The operand of the step that holds this lane's own four
        // tokens also has their elements of K and Q, in the lane that has the results: what the gates' gradients multiply.
        float to_last = 0.f;                             // this lane's share of sum k.W, while Y is W alone
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            float ke[4];
            four_of(bk[t], upper, ke);
#pragma unroll
            for (int e = 0; e < 4; ++e) to_last += ay[t][e] * (rk[e] * ke[e]);
        }
        auto row_products = [&](int s) {
            float f[8];
            bf16x8 a1[3], a2[3];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float *from = &lds.lower.rows[i][own][32 * s + 8 * g];
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = from[e];
                if (i == 0) split8<3>(f, a1); else split8<3>(f, a2);
            }
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
                aq[t] = product<2>(a1, bk[t], aq[t]);
                az[t] = product<2>(a2, bk[t], az[t]);
            }
        };
        auto column_products = [&](int s) {
            bf16x8 a1[3], a2[3];
            load_frag<3>(lds.lower.columns[0] + upper_frag(tile, s) * 3 * kFrag, lane, a1);
            load_frag<3>(lds.lower.columns[1] + upper_frag(tile, s) * 3 * kFrag, lane, a2);
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
                ay[t] = product<2>(a1, bq[t], ay[t]);
                ay[t] = product<2>(a2, bk[t], ay[t]);
            }
        };
        row_products(half);
        stay();
        column_products(half);
        stay();
        ask_kq(1 - half);
        if (half == 0) column_products(1); else row_products(0);
        stay();
        ask_kq(half);
        float qd[4] = {0.f, 0.f, 0.f, 0.f}, kz[4] = {0.f, 0.f, 0.f, 0.f}, ky[4] = {0.f, 0.f, 0.f, 0.f};
        {
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
                float ke[4], qe[4];
                four_of(bk[t], upper, ke);
                four_of(bq[t], upper, qe);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    qd[e] += aq[t][e] * qe[e];
                    kz[e] += az[t][e] * ke[e];
                    ky[e] += ay[t][e] * ke[e];
                    tq[t][e] = aq[t][e];
                    tk[t][e] = beta[e] * az[t][e] + ay[t][e];
                }
            }
        }
        inner = over_wave(inner);
        to_last = over_wave(to_last);
        if (lane == 0) { lds.inner[wave] = inner; lds.end[wave] = to_last; }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float d = rq[e] * over_columns(qd[e]), z = rk[e] * over_columns(kz[e]), y = rk[e] * over_columns(ky[e]);
            if (m == 0) { lds.sums[side][0][row + e] = d; lds.sums[side][1][row + e] = z; lds.sums[side][2][row + e] = y; }
        }
        lds_barrier();
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            dotq[e] = lds.sums[0][0][row + e] + lds.sums[1][0][row + e];
            dotk[e] = beta[e] * (lds.sums[0][1][row + e] + lds.sums[1][1][row + e]) + (lds.sums[0][2][row + e] + lds.sums[1][2][row + e]);
        }
        if (wave == 0) {
            const float z = lds.sums[0][1][lane] + lds.sums[1][1][lane];
            float d = (lds.sums[0][0][lane] + lds.sums[1][0][lane]) + lds.gate[kBeta][lane] * z - (lds.sums[0][2][lane] + lds.sums[1][2][lane]);
            if (lane == 63) {
                float both = 0.f, ends = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) { both += lds.inner[i]; ends += lds.end[i]; }
                d += ends + lds.gate[kGate][63] * both;
            }
            d = sum_from_here(d);
            // Nothing stands in front of a sequence's first token for its gate to act on; the terms cancel up to rounding.
            if (lane == 0 && p.initial_states == nullptr && at.lo == sequence_tokens(p, at.n).lo) d = 0.f;
            if (lane < at.count) {
                const int64_t to = ((int64_t)at.b * p.seqlen + at.lo + lane) * p.v_heads + h;
                store_from_float(bp.dg, to, p.g_dtype, d);
                store_from_float(bp.dbeta, to, p.beta_dtype, lds.db[lane] + z);
            }
        }
    }

    // The lengths' share: what lies along a key or query; the sums have one factor rk or rq already.
    if (p.qk_l2norm) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            rk[e] = lds.gate[kKeyNorm][row + e]; rq[e] = lds.gate[kQueryNorm][row + e];
            dotq[e] *= rq[e];
            dotk[e] *= rk[e];
        }
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            float ke[4], qe[4];
            four_of(bk[t], upper, ke);
            four_of(bq[t], upper, qe);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                tq[t][e] = rq[e] * (tq[t][e] - dotq[e] * qe[e]);
                tk[t][e] = rk[e] * (tk[t][e] - dotk[e] * ke[e]);
            }
        }
    }
    if (p.v_heads > p.heads) {
        float *share = w.dqk + (sv * 2 * 8 + wave) * TILES * 256 + lane * 4;
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            *reinterpret_cast<f32x4 *>(share + t * 256) = tq[t];
            *reinterpret_cast<f32x4 *>(share + (8 * TILES + t) * 256) = tk[t];
        }
        return;
    }
    // The stage is free: all have read X1 and X2 in front of the last barrier.
    constexpr bool BOTH = kOutBytes<DT, KS> <= sizeof(GradStage<KS>) * GradStage<KS>::kCopies;
    rows_leave<DT, KS, BOTH>(tq, tk, raw, bp, at, hk, vec_out);
}

// dq and dk of a key head that several value heads share: their shares added up in the order of the heads.
template <int DT, int KS>
__global__ void __launch_bounds__(kGradBlock)
delta_join_kernel(const cc1d_delta_bwd_params bp, const ChunkWork w, const int vec_out) {
    extern __shared__ uint4 raw[];
    const cc1d_delta_params &p = bp.fwd;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, group = p.v_heads / p.heads;
    const int slot = (int)divided(blockIdx.x, w.by_heads), hk = (int)blockIdx.x - slot * p.heads;
    const ChunkAt at = chunk_at(p, w, slot);
    if (at.count <= 0) return;
    const float *share = w.dqk + (((int64_t)slot * p.v_heads + hk * group) * 2 * 8 + wave) * KS * 256 + lane * 4;
    f32x4 tq[KS], tk[KS];
#pragma unroll
    for (int t = 0; t < KS; ++t) { tq[t] = (f32x4){0.f, 0.f, 0.f, 0.f}; tk[t] = tq[t]; }
    for (int j = 0; j < group; ++j, share += 2 * 8 * KS * 256) {
        f32x4 a[KS], b[KS];
#pragma unroll
        for (int t = 0; t < KS; ++t) {
            a[t] = *reinterpret_cast<const f32x4 *>(share + t * 256);
            b[t] = *reinterpret_cast<const f32x4 *>(share + (8 * KS + t) * 256);
        }
#pragma unroll
        for (int t = 0; t < KS; ++t) { tq[t] += a[t]; tk[t] += b[t]; }
    }
    rows_leave<DT, KS, kJoinBoth<DT, KS>>(tq, tk, raw, bp, at, hk, vec_out);
}

// Without value heads nothing comes back to q and k: zeros, a wavefront a row of each.
template <typename Bits>
__global__ void __launch_bounds__(kBlock)
delta_no_values_kernel(const cc1d_delta_bwd_params bp, const int64_t rows) {
    const cc1d_delta_params &p = bp.fwd;
    for (int64_t r = blockIdx.x * 4 + (threadIdx.x >> 6); r < rows; r += (int64_t)gridDim.x * 4) {
        const int64_t h = r % p.heads, t = r / p.heads % p.seqlen, b = r / p.heads / p.seqlen;
        for (int k = threadIdx.x & 63; k < p.dim_k; k += 64) {
            static_cast<Bits *>(bp.dq)[b * bp.dq_stride_b + t * bp.dq_stride_l + h * bp.dq_stride_h + k] = 0;
            static_cast<Bits *>(bp.dk)[b * bp.dk_stride_b + t * bp.dk_stride_l + h * bp.dk_stride_h + k] = 0;
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
    const bool vec = p.dim_v % 8 == 0 && whole_rows(p.x_dtype, bp.dout, bp.dout_stride_b, bp.dout_stride_l, bp.dout_stride_h) &&
                     whole_rows(p.x_dtype, p.v, p.v_stride_b, p.v_stride_l, p.v_stride_h);
    const int vec_out = whole_rows(p.x_dtype, bp.dq, bp.dq_stride_b, bp.dq_stride_l, bp.dq_stride_h) &&
                        whole_rows(p.x_dtype, bp.dk, bp.dk_stride_b, bp.dk_stride_l, bp.dk_stride_h);
    auto go = [&](auto v) {
        CC1D_LAUNCH((delta_grad_kernel<DT, KS, decltype(v)::value>), dim3((uint32_t)((int64_t)w.slots * p.v_heads)), dim3(kGradBlock), sizeof(GradLds<KS>), stream, bp, w, vec_out);
    };
    vec ? go(std::true_type()) : go(std::false_type());
    st = launch_status();
    if (st != CC1D_OK || p.v_heads == p.heads) return st;
    CC1D_LAUNCH((delta_join_kernel<DT, KS>), dim3((uint32_t)((int64_t)w.slots * p.heads)), dim3(kGradBlock), kOutBytes<DT, KS> / (kJoinBoth<DT, KS> ? 1 : 2), stream, bp, w, vec_out);
    return launch_status();
}

}  // namespace

int launch_delta_no_values(const cc1d_delta_bwd_params &bp, hipStream_t stream) {
    const int64_t rows = (int64_t)bp.fwd.batch * bp.fwd.seqlen * bp.fwd.heads;
    if (rows == 0) return CC1D_OK;
    const dim3 grid((uint32_t)(rows < 4 * 8192 ? (rows + 3) / 4 : 8192));
    if (bp.fwd.x_dtype == CC1D_F32) CC1D_LAUNCH(delta_no_values_kernel<uint32_t>, grid, dim3(kBlock), 0, stream, bp, rows);
    else CC1D_LAUNCH(delta_no_values_kernel<uint16_t>, grid, dim3(kBlock), 0, stream, bp, rows);
    return launch_status();
}

int launch_delta_bwd(const cc1d_delta_bwd_params &bp, const ChunkWork &w, hipStream_t stream) {
    return by_type_and_steps(bp.fwd.x_dtype, w.ks, [&](auto dt, auto ks) { return launch<decltype(dt)::value, decltype(ks)::value>(bp, w, stream); });
}

}  // namespace cc1d
