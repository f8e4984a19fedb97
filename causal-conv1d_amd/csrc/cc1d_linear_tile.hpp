// Linear attention, the kernel of out, dq, dk and dv of 16-bit tensors with at most 128 columns (cc1d_linear_attend.hpp says what x, y, z and
// the factors are; that kernel takes everything else).
//
// A workgroup of eight wavefronts takes a segment of one head, or of several value heads of a key head one after the other, a wavefront 32 of its
// rows with all columns of z; its x stays in its registers.  y and z of the whole segment lie in LDS as operands, what belongs to the key head for all
// of its value heads; the state passes through the place of whichever of the two is the value head's own, in front of it.  What the next head
// needs is on its way while one is worked on.  A wavefront makes y_j.x_i of 32 y's and its own 32 x's: transposed, a lane has the products of one x
// with 4 + 4 consecutive y's, which is the left operand of the product with z.  So weighted products stay in their lanes, and there is no
// barrier between the blocks.  Rows near the end (REV: the start) meet the most blocks; wavefronts w and w + 4, which share a SIMD, get one of each.
//
// Columns of z are dealt so that a lane's W of them are adjacent (W tiles of 16 columns, of tile t column W m + t): it reads 8 or 16 bytes of a row of z,
// and stores as many of a result's.  Its 8 rows of one column are an operand.
//
// E between different 32 tokens is a product of three factors: from x to the border of its 32 tokens, from border to border, and from
// there to y; each token's two are made once, by one lane, of sums of 64 bits (exp_of_sum).  Among the same 32 tokens it is exp(G_i - B) exp(B - G_j), B in front of them all, unless
// the gates reach e^60 there: then an exponential an entry.
//
// 32 segments of 80 heads of 128 x 64 (a training step of 4 x 2048 tokens, one key head), bfloat16: out 119 us, dv 108, dq and dk 398 (traced means; the
// best 116, 105 and 383); out's matrix instructions come to 0.6 PFLOP/s.  A workgroup fills a CU's LDS, so that nobody hides what it waits for: of out's time the products take 40 (the
// matrix cores' own time 19), the product with the state 24 (32 KB of operands a head, 9 of matrix cores), the gates, barriers and start
// 37, z's way to LDS 11, stores 10.  Tried: half the rows a workgroup and two of them a CU (out 127: state and y are read twice); 16 rows a wavefront, balanced
// (equal, with spills in dq); dq and dk with two terms of state and products (22 us less each; the gates' gradients, small differences of their dots, would
// lose eight bits).
#pragma once

#include "cc1d_linear_attend.hpp"

namespace cc1d {

constexpr int kTileBlock = 512, kStep = 32, kSteps = kSegment / kStep;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// KS: 32-column steps of x and y, W: 16-column tiles of z.
template <int KS, int W>
struct TileLds {
    uint8_t y[kSteps * 2 * KS * kFrag], z[kSteps * W * kFrag];         // [32 tokens][tile][step], [32 tokens][tile]
    float hi[kSegment], lo[kSegment];    // G
    float of_x[kSegment], of_y[kSegment];                              // factors of E
    float weigh[kSegment], back[kSegment];                             // y's weight; where x and y share 32 tokens: exp(G at their start - G)
    float f[kSegment], s[kSegment];
    float of_self[kSegment], self_sum[kSegment];         // the weighted product of a token with itself, and over the heads
    double ends[kSteps + 1];             // G at the borders of 32 tokens
    double sums[kBlocks];
    int32_t steep[kSteps];               // whether `back` is too large to be used
};

// y.x of bfloat16 and of float16 are exact products on either's own instruction.
template <int DT>
__device__ __forceinline__ f32x4 same_type_product(const u32x4 &a, const u32x4 &b, f32x4 acc) {
    if constexpr (DT == CC1D_BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(bitcast<bf16x8>(a), bitcast<bf16x8>(b), acc, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(bitcast<f16x8>(a), bitcast<f16x8>(b), acc, 0, 0, 0);
}
template <int DT, int NT>
__device__ __forceinline__ void as_terms(const u32x4 &x, bf16x8 (&t)[NT]) {
    if constexpr (DT == CC1D_BF16) {
        t[0] = bitcast<bf16x8>(x);
    } else {
        float f[8];
        Elem<DT>::unpack(x, f);
        split8<NT>(f, t);
    }
}
// Two rows of tiles against one right operand, the chains of the two side by side.
template <int MOST, int NA, int NB>
__device__ __forceinline__ void product_rows(const bf16x8 (&a)[2][NA], const bf16x8 (&b)[NB], f32x4 &first, f32x4 &second) {
#pragma unroll
    for (int sum = MOST; sum >= 0; --sum)
#pragma unroll
        for (int i = 0; i < NA; ++i) {
            const int j = sum - i;
            if (j < 0 || j >= NB) continue;
            first = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[0][i], b[j], first, 0, 0, 0);
            second = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[1][i], b[j], second, 0, 0, 0);
        }
}

// W adjacent 16-bit columns of eight rows; element t of all eight as an operand.
template <int W>
struct Wide8 {
    uint32_t r[8][W / 2];
    __device__ __forceinline__ void ask(int i, const uint8_t *at) {
        if constexpr (W == 8) {
            const u32x4 v = *reinterpret_cast<const u32x4 *>(at);
            r[i][0] = v.x; r[i][1] = v.y; r[i][W / 2 - 2] = v.z; r[i][W / 2 - 1] = v.w;
        } else {
            const u32x2 v = *reinterpret_cast<const u32x2 *>(at);
            r[i][0] = v.x; r[i][1] = v.y;
        }
    }
    __device__ __forceinline__ u32x4 column(int t) const {
        const uint32_t sel = (t & 1) ? 0x07060302u : 0x05040100u;
        const int q = t >> 1;
        u32x4 w;
        w.x = __builtin_amdgcn_perm(r[1][q], r[0][q], sel);
        w.y = __builtin_amdgcn_perm(r[3][q], r[2][q], sel);
        w.z = __builtin_amdgcn_perm(r[5][q], r[4][q], sel);
        w.w = __builtin_amdgcn_perm(r[7][q], r[6][q], sel);
        return w;
    }
};
// W results to adjacent columns, all inside.
template <int DT, int W>
__device__ __forceinline__ void store_wide(typename Elem<DT>::type *to, const float (&o)[W]) {
    uint32_t w[W / 2];
#pragma unroll
    for (int i = 0; i < W / 2; ++i) {
        float a = o[2 * i], b = o[2 * i + 1];
        if constexpr (DT == CC1D_F16) {
            asm("" : "+v"(a), "+v"(b));  // (no fused multiply that rounds to fp16 in one step)
            f16x2 h;
            h.x = (_Float16)a;
            h.y = (_Float16)b;
            w[i] = bitcast<uint32_t>(h);
        } else {
            w[i] = rounded_pair(a, b);
        }
    }
    if constexpr (W == 8) { u32x4 v; v.x = w[0]; v.y = w[1]; v.z = w[W / 2 - 2]; v.w = w[W / 2 - 1]; *reinterpret_cast<u32x4 *>(to) = v; }
    else { u32x2 v; v.x = w[0]; v.y = w[1]; *reinterpret_cast<u32x2 *>(to) = v; }
}

// MANY: several value heads to a workgroup (DOTS: whose rows are added up, or leave as a share).
template <int DT, int KS, int W, bool REV, bool DOTS, bool MANY>
__device__ __forceinline__ void tile_rows(const cc1d_delta_params &p, const SegmentWork &w, const AttendArgs &a, const uint32_t workgroup, const uint32_t workgroups) {
    using T = typename Elem<DT>::type;
    constexpr bool JOIN = DOTS && MANY;
    constexpr int NT = Terms<DT>::n, PT = DOTS ? 3 : 2, MOST = PT - 1;
    constexpr int STATE = W * PT, ROOM = DOTS ? kSteps * 2 * KS : kSteps * W;          // KB: a step of the state, and its place
    constexpr int SB = ROOM / STATE >= KS ? KS : ROOM / STATE >= 2 ? 2 : 1, STAGES = KS / SB, IN_STATE = (SB * STATE + 7) / 8;
    extern __shared__ uint4 raw[];
    TileLds<KS, W> &lds = *reinterpret_cast<TileLds<KS, W> *>(raw);
    uint8_t *room = DOTS ? lds.y : lds.z;
    int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // Heads of one segment, which may share y and z, on one XCD.
    const uint32_t per = workgroups >> 3, at_item = (workgroup & 7u) * per + (workgroup >> 3);
    const uint32_t item = divided(at_item, a.by_col_tiles), ct = at_item - item * a.col_tiles;
    if (item >= a.items) return;
    const uint32_t sh = divided(item, a.by_shares), share = item - sh * a.shares;
    const int slot = (int)divided(sh, a.by_heads), hk = (int)sh - slot * p.heads;
    const int h_first = hk * a.group + (int)share * a.heads_each, h_left = a.group - (int)share * a.heads_each;
    const int h_count = !MANY ? 1 : h_left < a.heads_each ? h_left : a.heads_each;
    const int col0 = (int)ct * 16 * W;
    const SegmentAt at = segment_at(p, w, slot);

    if (p.cu_seqlens != nullptr && (!DOTS || share == 0)) {            // tokens in front of the first sequence and behind the last
        const int64_t front = sequence_tokens(p, 0).lo, back = sequence_tokens(p, p.sequences - 1).hi;
        auto clear = [&](int64_t t) {
            for (int c = col0 + lane; c < a.d2 && c < col0 + 16 * W; c += 64) {
                if (!DOTS) {
                    for (int i = 0; i < h_count; ++i) (static_cast<T *>(a.out) + (h_first + i) * a.out_h)[t * a.out_l + c] = Elem<DT>::from_float(0.f);
                } else if (a.share == nullptr) {
                    (static_cast<T *>(a.out) + hk * a.out_h)[t * a.out_l + c] = Elem<DT>::from_float(0.f);
                } else {
                    for (int i = 0; i < a.shares; ++i) a.share[(((int64_t)i * p.seqlen + t) * p.heads + hk) * a.d2 + c] = 0.f;
                }
            }
        };
        for (int64_t t = (int64_t)slot * 8 + wave; t < front; t += (int64_t)w.slots * 8) clear(t);
        for (int64_t t = back + (int64_t)slot * 8 + wave; t < p.seqlen; t += (int64_t)w.slots * 8) clear(t);
    }
    if (at.count <= 0) return;
    const int steps = (at.count + kStep - 1) / kStep;
    const bool has_state = (REV ? !at.last : at.c > 0) || a.first;
    const int64_t state = a.first ? (int64_t)slot : border_behind(p, w, at) - !REV;
    const int own = wave < 4 ? wave : 11 - wave;         // which 32 rows
    const bool rows = own < steps, whole = (own + 1) * kStep <= at.count;
    auto token = [&](int t) { return t < at.count ? t : at.count - 1; };           // (rows behind the last weigh nothing, or are not stored)

    f32x4 total[JOIN ? 2 : 1][JOIN ? W : 1], acc[2][W];
    if constexpr (JOIN)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int t = 0; t < W; ++t) total[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};

    int m = lane & 15, g = lane >> 4, h = h_first;
    const int mine = (int)threadIdx.x & (kSegment - 1);  // the token whose factors this lane makes (each twice)
    const uint32_t x_pitch = (uint32_t)(a.x.sl * (int64_t)sizeof(T)), y_pitch = (uint32_t)(a.y.sl * (int64_t)sizeof(T)), z_pitch = (uint32_t)(a.z.sl * (int64_t)sizeof(T));
    auto head_of = [&](const LinearRows &t) { return static_cast<const uint8_t *>(t.p) + (at.b * t.sb + at.lo * t.sl + (t.by_key ? hk : h) * t.sh) * (int64_t)sizeof(T); };
    // What is on its way.
    uint32_t gate_bits = 0, beta_bits = 0;
    u32x4 x[2][KS], yr[2][KS], in_state[IN_STATE];       // x, y: rows 16 i + m of 32, 8 columns: an operand either way
    Wide8<W> zr;
    auto ask_gates = [&]() {
        const int64_t tok = at.lo + token(mine);
        gate_bits = load_bits(p.g, at.b * p.g_stride_b + tok * p.g_stride_l + h * p.g_stride_h, p.g_dtype);
        if (p.beta != nullptr) beta_bits = load_bits(p.beta, at.b * p.beta_stride_b + tok * p.beta_stride_l + h * p.beta_stride_h, p.beta_dtype);
    };
    auto ask_x = [&]() {
        const uint8_t *xb = head_of(a.x);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t row = (uint32_t)token(own * kStep + 16 * i + m) * x_pitch;
#pragma unroll
            for (int s = 0; s < KS; ++s) x[i][s] = *reinterpret_cast<const u32x4 *>(xb + (row + (32 * s + 8 * g < a.d1 ? 32 * s + 8 * g : 0) * (uint32_t)sizeof(T)));
        }
    };
    auto ask_y = [&]() {
        const uint8_t *yb = head_of(a.y);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t row = (uint32_t)token(own * kStep + row_of(i, m)) * y_pitch;
#pragma unroll
            for (int s = 0; s < KS; ++s) yr[i][s] = *reinterpret_cast<const u32x4 *>(yb + (row + (32 * s + 8 * g < a.d1 ? 32 * s + 8 * g : 0) * (uint32_t)sizeof(T)));
        }
    };
    auto ask_z = [&]() {                                 // columns that are not there: the first
        const uint8_t *zb = head_of(a.z);
        const uint32_t col = (uint32_t)(col0 + W * m < a.d2 ? col0 + W * m : 0) * (uint32_t)sizeof(T);
#pragma unroll
        for (int e = 0; e < 8; ++e) zr.ask(e, zb + ((uint32_t)token(own * kStep + 8 * g + e) * z_pitch + col));
    };
    auto ask_state = [&](int stage) {                    // steps that are not there: the last
        const uint8_t *st = a.state + (state * p.v_heads + h) * a.steps * a.tiles * PT * kFrag + (int64_t)ct * STATE * kFrag + lane * 16;
#pragma unroll
        for (int i = 0; i < IN_STATE; ++i) {
            const int f = wave + 8 * i < SB * STATE ? wave + 8 * i : SB * STATE - 1, s = stage * SB + f / STATE, step = s < a.steps ? s : a.steps - 1;
            in_state[i] = *reinterpret_cast<const u32x4 *>(st + (step * a.tiles * PT + f % STATE) * kFrag);
        }
    };
    // DOTS, rows 16 i + 4 g + (0 .. 3) of this wavefront's 32: of u columns W m .. W m + W - 1, of z column W m + t.
    auto both_of = [](uint32_t two, float &first, float &second) {
        if constexpr (DT == CC1D_F16) { first = (float)bitcast<f16x2>(two).x; second = (float)bitcast<f16x2>(two).y; }
        else { first = bitcast<float>(two << 16); second = bitcast<float>(two & 0xffff0000u); }
    };
    auto ask_u = [&](int i, Wide8<W> &u) {
        const uint8_t *ub = static_cast<const uint8_t *>(a.u.p) + (at.b * a.u.sb + at.lo * a.u.sl + hk * a.u.sh) * (int64_t)sizeof(T);      // (of the key head)
        const uint32_t u_pitch = (uint32_t)(a.u.sl * (int64_t)sizeof(T)), col = (uint32_t)(W * m < a.d2 ? W * m : 0) * (uint32_t)sizeof(T);
#pragma unroll
        for (int e = 0; e < 4; ++e) u.ask(e, ub + ((uint32_t)token(own * kStep + 16 * i + 4 * g + e) * u_pitch + col));
    };
    auto z_rows = [&](int i, int t, float (&f)[4]) {
        const u32x2 r = *reinterpret_cast<const u32x2 *>(lds.z + (own * W + t) * kFrag + ((2 * i + (g >> 1)) * 16 + m) * 16 + (g & 1) * 8);
        both_of(r.x, f[0], f[1]);
        both_of(r.y, f[2], f[3]);
    };
    // In the order in which it is needed.  DOTS: y is the value head's, x too; else z is.
    ask_gates();
    if (has_state) ask_state(0);
    ask_x();
    ask_y();
    ask_z();

    for (int hi = 0; hi < h_count; ++hi) {
        asm volatile("" : "+v"(lane));                   // (addresses are made anew: kept over the loop they would take a hundred registers)
        m = lane & 15;
        g = lane >> 4;
        const int h_now = h;
        stay();
        if (hi > 0) lds_barrier();                       // the head before has been read
        // G, one token a lane.
        const bool first_half = threadIdx.x < kSegment;
        const float beta = p.beta != nullptr ? bits_as_float(beta_bits, p.beta_dtype) : 1.f;
        double sum = running_sum(mine < at.count ? (double)bounded_gate(bits_as_float(gate_bits, p.g_dtype)) : 0.0);
        if (first_half && lane == 63) lds.sums[wave] = sum;
        if (has_state) {
#pragma unroll
            for (int i = 0; i < IN_STATE; ++i)
                if (8 * i + 7 < SB * STATE || wave + 8 * i < SB * STATE) *reinterpret_cast<u32x4 *>(room + (wave + 8 * i) * kFrag + lane * 16) = in_state[i];
        }
        lds_barrier();
        if (has_state && STAGES > 1) ask_state(1);
#pragma unroll
        for (int b = 0; b < kBlocks - 1; ++b) sum += b < (wave & 3) ? lds.sums[b] : 0.0;
        if (first_half) {
            const float h0 = (float)sum;
            lds.hi[mine] = h0;
            lds.lo[mine] = (float)(sum - (double)h0);
            if ((mine & 31) == 31) lds.ends[(mine >> 5) + 1] = sum;
            if (mine == 0) lds.ends[0] = 0.0;
        }
        if (a.d1 < 32 * KS)                              // (y repeats its first columns there)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int s = 0; s < KS; ++s)
                    if (32 * s + 8 * g >= a.d1) x[i][s] = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int t = 0; t < W; ++t) acc[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (has_state) {
#pragma unroll
            for (int stage = 0; stage < STAGES; ++stage) {
                if (stage > 0) {
                    lds_barrier();                       // the steps before have been read
#pragma unroll
                    for (int i = 0; i < IN_STATE; ++i)
                        if (8 * i + 7 < SB * STATE || wave + 8 * i < SB * STATE) *reinterpret_cast<u32x4 *>(room + (wave + 8 * i) * kFrag + lane * 16) = in_state[i];
                    lds_barrier();
                    if (stage + 1 < STAGES) ask_state(stage + 1);
                }
                stay();
                if (rows)
#pragma unroll
                    for (int sb = 0; sb < SB; ++sb) {
                        bf16x8 f[2][NT];
#pragma unroll
                        for (int i = 0; i < 2; ++i) as_terms<DT, NT>(x[i][stage * SB + sb], f[i]);
#pragma unroll
                        for (int t = 0; t < W; ++t) {
                            bf16x8 b[PT];
                            load_frag<PT>(room + (sb * W + t) * PT * kFrag, lane, b);
                            product_rows<MOST>(f, b, acc[0][t], acc[1][t]);
                        }
                    }
                stay();
            }
        }
        lds_barrier();                                   // G; the state has been read
        if (first_half) {
            const double start = lds.ends[mine >> 5], end = lds.ends[(mine >> 5) + 1], last = lds.ends[kSteps];
            const float up = exp_of_sum(sum - start), down = exp_of_sum(end - sum), back = exp_of_sum(start - sum);
            const float weigh = mine >= at.count ? 0.f : REV ? p.scale : beta;
            lds.of_x[mine] = REV ? down : up;
            lds.of_y[mine] = weigh * (REV ? up : down);
            lds.weigh[mine] = weigh;
            lds.back[mine] = REV ? back : weigh * back;
            const uint64_t steep = __ballot(fabs(sum - start) > 60.0);
            if ((lane & 31) == 0) lds.steep[mine >> 5] = (uint32_t)(steep >> (lane & 32)) != 0u;
            lds.f[mine] = exp_of_sum(REV ? last - sum : sum);
            lds.s[mine] = REV ? beta : p.scale;
        }
        if (rows) {
            if (hi == 0 || DOTS)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int s = 0; s < KS; ++s) *reinterpret_cast<u32x4 *>(lds.y + ((own * 2 + i) * KS + s) * kFrag + lane * 16) = yr[i][s];
            if (hi == 0 || !DOTS)
#pragma unroll
                for (int t = 0; t < W; ++t) *reinterpret_cast<u32x4 *>(lds.z + (own * W + t) * kFrag + lane * 16) = zr.column(t);
        }
        lds_barrier();                                   // y, z, factors
        const bool more = MANY && hi + 1 < h_count;
        // x has arrived by now; without being told so the compiler waits for it in the loop below, and for all that is asked for here.
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int s = 0; s < KS; ++s) asm volatile("" : "+v"(x[i][s]));
        if (more) {                                      // the next head's
            h += 1;
            ask_gates();
            if (has_state) ask_state(0);
            if (DOTS) ask_y(); else ask_z();
        }
        stay();
        if (rows) {
            if (has_state)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const f32x4 by = *reinterpret_cast<const f32x4 *>(&lds.f[own * kStep + 16 * i + 4 * g]);
#pragma unroll
                    for (int t = 0; t < W; ++t) acc[i][t] *= by;
                }
            const float of_x[2] = {lds.of_x[own * kStep + m], lds.of_x[own * kStep + 16 + m]};
            const double border = lds.ends[REV ? own + 1 : own];
            const int turns = REV ? steps - own : own + 1;
            u32x4 y[2][KS];
            auto read_y = [&](int j) {
#pragma unroll
                for (int s = 0; s < KS; ++s)
#pragma unroll
                    for (int b = 0; b < 2; ++b) y[b][s] = *reinterpret_cast<const u32x4 *>(lds.y + ((j * 2 + b) * KS + s) * kFrag + lane * 16);
            };
            read_y(REV ? steps - 1 : 0);
            for (int k = 0; k < turns; ++k) {            // the 32 rows themselves come last
                const int j = REV ? steps - 1 - k : k;
                const bool self = k == turns - 1;
                f32x4 pt[2][2];                          // x's tile, y's tile
#pragma unroll
                for (int i = 0; i < 2; ++i) pt[i][0] = pt[i][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = 0; s < KS; ++s)
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int i = 0; i < 2; ++i) pt[i][b] = same_type_product<DT>(y[b][s], x[i][s], pt[i][b]);
                stay();
                // z's first half, and the next y: read while the products are weighted.
                u32x4 z[W / 2];
#pragma unroll
                for (int t = 0; t < W / 2; ++t) z[t] = *reinterpret_cast<const u32x4 *>(lds.z + (j * W + t) * kFrag + lane * 16);
                if (!self) read_y(REV ? j - 1 : j + 1);
                stay();
                bf16x8 f[2][PT];
                if (self) {
                    const int yj = own * kStep + 8 * g;
                    if constexpr (DOTS) {                // of x's row m: lane (m, 2 i + m / 8) has it
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const f32x4 lo = pt[i][0], up = pt[i][1];
                            const float b0 = m & 1 ? lo[1] : lo[0], b1 = m & 1 ? lo[3] : lo[2], b2 = m & 1 ? up[1] : up[0], b3 = m & 1 ? up[3] : up[2];
                            const float c0 = m & 2 ? b1 : b0, c1 = m & 2 ? b3 : b2, both = m & 4 ? c1 : c0;
                            if (g == 2 * i + (m >> 3)) lds.of_self[own * kStep + 16 * i + m] = both * lds.weigh[own * kStep + 16 * i + m];
                        }
                    }
                    if (lds.steep[own] != 0) {
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const int xi = own * kStep + 16 * i + m;
                            const float hx = lds.hi[xi], lx = lds.lo[xi];
#pragma unroll
                            for (int b = 0; b < 2; ++b) {
                                const f32x4 hy = *reinterpret_cast<const f32x4 *>(&lds.hi[yj + 4 * b]), ly = *reinterpret_cast<const f32x4 *>(&lds.lo[yj + 4 * b]);
                                const f32x4 cy = *reinterpret_cast<const f32x4 *>(&lds.weigh[yj + 4 * b]);
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const float d = (hx - hy[e]) + (lx - ly[e]);
                                    pt[i][b][e] *= cy[e] * exp_of(REV ? -d : d);
                                }
                            }
                        }
                    } else {
                        const float *to = REV ? lds.back : lds.of_x, *from = REV ? lds.of_y : lds.back;
                        const f32x4 y0 = *reinterpret_cast<const f32x4 *>(&from[yj]), y1 = *reinterpret_cast<const f32x4 *>(&from[yj + 4]);
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const float cx = to[own * kStep + 16 * i + m];
                            pt[i][0] *= cx * y0;
                            pt[i][1] *= cx * y1;
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float v[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) {    // (DOTS: without the token itself)
                            const int y_row = 8 * g + e, x_row = 16 * i + m;
                            v[e] = (DOTS ? (REV ? y_row > x_row : y_row < x_row) : REV ? y_row >= x_row : y_row <= x_row) ? pt[i][e >> 2][e & 3] : 0.f;
                        }
                        split8<PT>(v, f[i]);
                    }
                } else {
                    const float between = exp_of_sum(REV ? lds.ends[j] - border : border - lds.ends[j + 1]);
                    const f32x4 y0 = *reinterpret_cast<const f32x4 *>(&lds.of_y[j * kStep + 8 * g]), y1 = *reinterpret_cast<const f32x4 *>(&lds.of_y[j * kStep + 8 * g + 4]);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float cx = of_x[i] * between;
                        float v[8];
#pragma unroll
                        for (int e = 0; e < 4; ++e) { v[e] = pt[i][0][e] * (cx * y0[e]); v[4 + e] = pt[i][1][e] * (cx * y1[e]); }
                        split8<PT>(v, f[i]);
                    }
                }
                stay();
#pragma unroll
                for (int half = 0; half < 2; ++half) {
#pragma unroll
                    for (int t = 0; t < W / 2; ++t) {
                        bf16x8 zt[NT];
                        as_terms<DT, NT>(z[t], zt);
                        product_rows<MOST>(f, zt, acc[0][half * W / 2 + t], acc[1][half * W / 2 + t]);
                    }
                    if (half == 0) {
                        stay();
#pragma unroll
                        for (int t = 0; t < W / 2; ++t) z[t] = *reinterpret_cast<const u32x4 *>(lds.z + (j * W + W / 2 + t) * kFrag + lane * 16);
                        stay();
                    }
                }
            }
        }
        stay();
        if constexpr (DOTS) {
            if (more) ask_x();
            if (rows) {
                wave_lds_fence();                        // of_self
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int row = own * kStep + 16 * i + 4 * g;
                    Wide8<W> u;
                    ask_u(i, u);
                    stay();
                    double dot[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float sum_u = 0.f;
#pragma unroll
                        for (int t = 0; t < W / 2; ++t) {
                            float u0, u1;
                            both_of(u.r[e][t], u0, u1);
                            sum_u = fmaf(acc[i][2 * t][e], u0, fmaf(acc[i][2 * t + 1][e], u1, sum_u));
                        }
                        dot[e] = over_columns(W * m < a.d2 ? (double)sum_u : 0.0);
                    }
                    const double mine_dot = m == 1 ? dot[1] : m == 2 ? dot[2] : m == 3 ? dot[3] : dot[0];
                    if (m < 4) {
                        const float of_self = lds.of_self[row + m], weighed = of_self * lds.s[row + m];
                        lds.self_sum[row + m] = JOIN && hi > 0 ? lds.self_sum[row + m] + weighed : weighed;
                        if (row + m < at.count) {
                            const int64_t to = ((int64_t)at.b * p.v_heads + h_now) * p.seqlen + at.lo + row + m;
                            a.dots[to] = REV ? mine_dot : (double)p.scale * mine_dot;
                            if (a.selves != nullptr) a.selves[to] = of_self;
                        }
                    }
                    const f32x4 by = *reinterpret_cast<const f32x4 *>(&lds.s[row]);
#pragma unroll
                    for (int t = 0; t < W; ++t) {
                        if constexpr (JOIN) total[i][t] += acc[i][t] * by;
                        else acc[i][t] *= by;
                    }
                }
            }
        }
        if (rows && (!DOTS || !more)) {                  // rows leave
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int first = 16 * i + 4 * g;
                f32x4 s = {1.f, 1.f, 1.f, 1.f};
                if constexpr (!DOTS) s = *reinterpret_cast<const f32x4 *>(&lds.s[own * kStep + first]);
                if constexpr (DOTS) {                    // the tokens themselves
                    wave_lds_fence();
                    const f32x4 by = *reinterpret_cast<const f32x4 *>(&lds.self_sum[own * kStep + first]);
                    if (a.uz != nullptr && share == 0) {
                        Wide8<W> u;
                        ask_u(i, u);
                        float sum_uz[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int t = 0; t < W; t += 2) {
                            float z0[4], z1[4];
                            z_rows(i, t, z0);
                            z_rows(i, t + 1, z1);
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                float u0, u1;
                                both_of(u.r[e][t / 2], u0, u1);
                                sum_uz[e] = fmaf(u0, z0[e], fmaf(u1, z1[e], sum_uz[e]));
                            }
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float all = over_columns(W * m < a.d2 ? sum_uz[e] : 0.f);
                            if (m == e && own * kStep + first + e < at.count) a.uz[((int64_t)at.b * p.heads + hk) * p.seqlen + at.lo + own * kStep + first + e] = all;
                        }
                    }
#pragma unroll
                    for (int t = 0; t < W; ++t) {
                        float zt[4];
                        z_rows(i, t, zt);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if constexpr (JOIN) total[i][t][e] = fmaf(by[e], zt[e], total[i][t][e]);
                            else acc[i][t][e] = fmaf(by[e], zt[e], acc[i][t][e]);
                        }
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float o[W];
#pragma unroll
                    for (int t = 0; t < W; ++t) {
                        if constexpr (JOIN) o[t] = total[i][t][e];
                        else o[t] = s[e] * acc[i][t][e];
                    }
                    const int row = own * kStep + first + e;
                    if ((!whole && row >= at.count) || col0 + W * m >= a.d2) continue;
                    if (!JOIN || a.share == nullptr) {
                        const int64_t head = DOTS ? hk : h_now;
                        T *base = static_cast<T *>(a.out) + at.b * a.out_b + at.lo * a.out_l + head * a.out_h + col0;
                        store_wide<DT, W>(base + ((uint32_t)row * (uint32_t)a.out_l + W * m), o);
                    } else {
                        float *to = a.share + ((((int64_t)share * p.batch + at.b) * p.seqlen + at.lo + row) * p.heads + hk) * a.d2 + W * m;
#pragma unroll
                        for (int t = 0; t < W; t += 4) *reinterpret_cast<float4 *>(to + t) = make_float4(o[t], o[t + 1], o[t + 2], o[t + 3]);
                    }
                }
            }
        }
    }
}

template <int DT, int KS, int W, bool REV, bool MANY>
__global__ void __launch_bounds__(kTileBlock, 2)
linear_tile_kernel(const cc1d_delta_params p, const SegmentWork w, const AttendArgs a) {
    tile_rows<DT, KS, W, REV, false, MANY>(p, w, a, blockIdx.x, gridDim.x);
}
// dq and dk in one launch (linear_attend_pair_kernel).
template <int DT, int KS, int W, bool MANY>
__global__ void __launch_bounds__(kTileBlock, 2)
linear_tile_pair_kernel(const cc1d_delta_params p, const SegmentWork w, const AttendArgs q, const AttendArgs k, const uint32_t half) {
    if (blockIdx.x < half) tile_rows<DT, KS, W, false, true, MANY>(p, w, q, blockIdx.x, half);
    else tile_rows<DT, KS, W, true, true, MANY>(p, w, k, blockIdx.x - half, half);
}

// f(KS, W) for these columns of x and z.
template <typename F>
int by_tiles(const AttendArgs &a, F &&f) {
    using I2 = std::integral_constant<int, 2>;
    using I4 = std::integral_constant<int, 4>;
    using I8 = std::integral_constant<int, 8>;
    if (a.d2 <= 64) return a.d1 <= 64 ? f(I2(), I4()) : f(I4(), I4());
    return a.d1 <= 64 ? f(I2(), I8()) : f(I4(), I8());
}

// Steps of x and y at once, beyond 128 columns: eight, or four slab by slab where eight steps' LDS leaves fewer workgroups a CU and the barriers weigh less: float32's
// out and dv, and dq and dk of at most 64 columns of z.  16 heads, 4 x 2048 tokens, eight and four: bfloat16, 256 x 256 forward 329 us and 383, backward 953 and
// 1152, 256 x 64 forward 119 and 147, 64 x 256 backward 479 and 399; float32, 256 x 256 forward 971 and 802, 192 x 192 backward (dq and dk by eight) 1570 and 1821.
// (Backward since then, own shares out of the products: 3 to 5 % more.)
template <int DT, bool REV>
int launch_attend(const cc1d_delta_params &p, const SegmentWork &w, const AttendArgs &a, hipStream_t stream) {
    if constexpr (DT != CC1D_F32) {
        if (a.tile != 0)
            return by_tiles(a, [&](auto ks, auto width) {
                constexpr int KS = decltype(ks)::value, W = decltype(width)::value;
                const dim3 grid((a.items * a.col_tiles + 7) / 8 * 8);
                if constexpr (W == 4) {
                    if (a.heads_each > 1) {
                        CC1D_LAUNCH((linear_tile_kernel<DT, KS, W, REV, true>), grid, dim3(kTileBlock), sizeof(TileLds<KS, W>), stream, p, w, a);
                        return launch_status();
                    }
                }
                CC1D_LAUNCH((linear_tile_kernel<DT, KS, W, REV, false>), grid, dim3(kTileBlock), sizeof(TileLds<KS, W>), stream, p, w, a);
                return launch_status();
            });
    }
    const dim3 grid((a.items + 7) / 8 * 8 * kBlocks * a.col_tiles);
    auto go = [&](auto ks, auto rt) {
        constexpr int KS = decltype(ks)::value, RT = decltype(rt)::value;
        CC1D_LAUNCH((linear_attend_kernel<DT, KS, RT, REV>), grid, dim3(kBlock), sizeof(AttendLds<DT, KS, out_terms(DT)>), stream, p, w, a);
        return launch_status();
    };
    using I2 = std::integral_constant<int, 2>;
    using I4 = std::integral_constant<int, 4>;
    using I8 = std::integral_constant<int, 8>;
    if constexpr (DT == CC1D_F32) {
        if (a.steps <= 2) return a.d2 <= 64 ? go(I2(), I2()) : go(I2(), I4());
        return a.d2 <= 64 ? go(I4(), I2()) : go(I4(), I4());
    } else {                             // (more than 128 columns of x)
        return a.d2 <= 64 ? go(I8(), I2()) : go(I8(), I4());
    }
}

template <int DT>
int launch_attend_pair(const cc1d_delta_params &p, const SegmentWork &w, const AttendArgs &q, const AttendArgs &k, const AttendArgs *v, hipStream_t stream) {
    if constexpr (DT != CC1D_F32) {
        if (q.tile != 0)
            return by_tiles(q, [&](auto ks, auto width) {
                constexpr int KS = decltype(ks)::value, W = decltype(width)::value;
                const uint32_t half = (q.items + 7) / 8 * 8;
                if (q.share != nullptr || q.heads_each > 1)
                    CC1D_LAUNCH((linear_tile_pair_kernel<DT, KS, W, true>), dim3(2 * half), dim3(kTileBlock), sizeof(TileLds<KS, W>), stream, p, w, q, k, half);
                else
                    CC1D_LAUNCH((linear_tile_pair_kernel<DT, KS, W, false>), dim3(2 * half), dim3(kTileBlock), sizeof(TileLds<KS, W>), stream, p, w, q, k, half);
                return launch_status();
            });
    }
    const uint32_t half = (q.items + 7) / 8 * 8 * kBlocks;
    auto go = [&](auto ks, auto rt, auto cp) {
        constexpr int KS = decltype(ks)::value, RT = decltype(rt)::value, CP = decltype(cp)::value;
        constexpr size_t lds = sizeof(AttendLds<DT, KS, 3>), lds_v = DT == CC1D_F32 ? sizeof(AttendLds<DT, RT == 2 ? 2 : 4, 3>) : 0;
        const uint32_t more = v != nullptr ? (v->items + 7) / 8 * 8 * kBlocks * v->col_tiles : 0;
        CC1D_LAUNCH((linear_attend_pair_kernel<DT, KS, RT, CP>), dim3(2 * half + more), dim3(kBlock), lds > lds_v || v == nullptr ? lds : lds_v, stream, p, w, q, k, v != nullptr ? *v : q,
                    half);
        return launch_status();
    };
    using I1 = std::integral_constant<int, 1>;
    using I2 = std::integral_constant<int, 2>;
    using I4 = std::integral_constant<int, 4>;
    using I8 = std::integral_constant<int, 8>;
    auto by_columns = [&](auto ks) {
        if (q.d2 > 128) return go(ks, I4(), I2());
        return q.d2 <= 64 ? go(ks, I2(), I1()) : go(ks, I4(), I1());
    };
    if constexpr (DT == CC1D_F32) {
        if (q.steps <= 2) return by_columns(I2());
        if (q.steps <= 4 || q.d2 <= 64) return by_columns(I4());
    } else {                             // (more than 128 columns of x or z)
        if (q.steps <= 2) return go(I2(), I4(), I2());
        if (q.steps <= 4) return go(I4(), I4(), I2());
        if (q.d2 <= 64) return go(I4(), I2(), I1());
    }
    return q.d2 > 128 ? go(I8(), I4(), I2()) : go(I8(), I4(), I1());
}

}  // namespace cc1d
