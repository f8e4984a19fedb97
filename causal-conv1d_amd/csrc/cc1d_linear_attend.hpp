// Linear attention, the kernel of out, dq, dk and dv (cc1d_linear.hpp):
//
//   r_i = f_i x_i.State + sum over j <= i (REV: j >= i) of E_ij c_j (x_i.y_j) z_j,   result row i = s_i r_i
//
//   out   x = q     y = k     z = v     State = S0     f = exp(G)         c = beta   s = scale
//   dq    x = dout  y = v     z = k     State = S0^T   f = exp(G)         c = beta   s = scale      DOTS
//   dk    x = v     y = dout  z = q     State = dS1^T  f = exp(Gend - G)  c = scale  s = beta  REV  DOTS
//   dv    x = k     y = q     z = dout  State = dS1    f = exp(Gend - G)  c = scale  s = beta  REV
//
// A workgroup of four wavefronts makes 64 rows (one block of a segment) of up to 128 columns (CP = 2: 256).  A wavefront's result is 32 columns
// of z, all rows (RT = 4), or half the rows where z has at most 64 columns (RT = 2): State and z are right operands that it reads for itself,
// from memory in operand order and as column pairs (Pair8), so neither goes through LDS.  For the products x.y the wavefronts take 16 rows y_j each
// against all 64 x_i, so that the result, transposed, is the left operand of the product with z in the lane that has it, four tokens at a time: weighted,
// split into its terms and passed through LDS once, double-buffered, one barrier a block.
//
// E between two blocks is a product of two factors, exp(G_i - R) and exp(R - G_j), R between them, so that only a block with itself takes an exponential
// an entry; there the tiles beyond the diagonal are left out.  A factor below e^-87 is nothing, whatever
// the others are: with gates that add up to no more than 32 over any run of tokens, two of those lift it by e^64 at most, and what is lost weighs less than e^-23.
// (An exponential an entry wherever a gate is positive: linear_tile_pair_kernel<bfloat16, 2, 8, several heads> 4 % slower for all gates.)
//
// DOTS: several value heads of a key head one after the other, the sum of their rows kept in registers, and of each the rows' products with u
// (q or k), which the gates' gradients are made of.  There a row's own z stays out of the products; it joins the sum of the heads at the end, with a weight in fp32.  What several workgroups of a key head leave is joined by linear_join_kernel.
//
// float32 takes six matrix instructions a product, 16 heads of 128 x 128, 4 x 2048 tokens: forward 219 us (with sums, scan and the last states), backward 588; bfloat16 of 256 x 256:
// 352 and 994.  A block's chain of loads, splits, LDS and products is what it takes time for, with one or two workgroups a CU by registers
// and LDS: 24 workgroups of a small call take 19 us, the matrix cores' part of which is 5.
#pragma once

#include "cc1d_delta_host.hpp"
#include "cc1d_linear_device.hpp"

namespace cc1d {

// Two places for the products, or one and a barrier more where two would leave a CU a single workgroup.
constexpr int product_places(int dt, int ks) { return ks >= (dt == CC1D_F32 ? 4 : 8) ? 1 : 2; }
template <int DT, int KS, int PT>
struct AttendLds {
    uint8_t x[4 * KS * Terms<DT>::n * kFrag];
    uint8_t p[product_places(DT, KS)][8 * PT * kFrag];
    GateLds gates;
    float f[kChunk], s[kChunk];
    double dots[4][kChunk];
    float of_self[kChunk];               // the weighted product of a token with itself
};

// Left operands of four tiles against one right one, their chains side by side.
template <int MOST, int N, int NA, int NB>
__device__ __forceinline__ void products_left(const bf16x8 (&a)[N][NA], const bf16x8 (&b)[NB], f32x4 *const (&acc)[N]) {
#pragma unroll
    for (int sum = MOST; sum >= 0; --sum)
#pragma unroll
        for (int i = 0; i < NA; ++i) {
            const int j = sum - i;
            if (j < 0 || j >= NB) continue;
#pragma unroll
            for (int t = 0; t < N; ++t) *acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[t][i], b[j], *acc[t], 0, 0, 0);
        }
}

// Wavefronts a SIMD that the registers leave: two where nothing, or next to nothing, has to be kept in memory for that and LDS leaves two workgroups (dq and dk,
// 16 heads, 4 x 2048 tokens, backward with two and with one: float32, 128 x 128 603 us and 746, 64 x 256 741 and 1012; bfloat16, 128 x 256 447 and 605; float32,
// 128 x 256, whose LDS leaves one, 1262 and 1150; since then, with own shares out of the products, 3 % more).
constexpr int attend_waves(bool dots, int dt, int ks, int cp) { return dots && (cp > 1 || (dt == CC1D_F32 && ks == 8)) ? 1 : 2; }

// KS: 32-column steps of x and y at once (their LDS); wider ones, more than 256 columns, pass slab by slab.
template <int DT, int KS, int RT, int CP, bool REV, bool DOTS>
__device__ __forceinline__ void attend_rows(const cc1d_delta_params &p, const SegmentWork &w, const AttendArgs &a, const uint32_t workgroup) {
    using T = typename Elem<DT>::type;
    constexpr int NT = Terms<DT>::n, PT = DOTS ? 3 : out_terms(DT), MOST = PT - 1;
    constexpr bool XREG = KS * NT <= 4;                  // x stays in registers
    extern __shared__ uint4 raw[];
    AttendLds<DT, KS, PT> &lds = *reinterpret_cast<AttendLds<DT, KS, PT> *>(raw);
    int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // The blocks of one segment and head, which read the same state and y and z, on one XCD; those with the most to do first.
    const uint32_t idx = workgroup >> 3, rest = idx / kBlocks, of_block = idx % kBlocks;
    const uint32_t pos = divided(rest, a.by_col_tiles), ct = rest - pos * a.col_tiles, item = pos * 8u + (workgroup & 7u);
    if (item >= a.items) return;
    const int r = REV ? (int)of_block : kBlocks - 1 - (int)of_block;
    const uint32_t sh = divided(item, a.by_shares), share = item - sh * a.shares;
    const int slot = (int)divided(sh, a.by_heads), hk = (int)sh - slot * p.heads;
    const int h_first = hk * a.group + (int)share * a.heads_each, h_left = a.group - (int)share * a.heads_each;
    const int h_count = !DOTS ? 1 : h_left < a.heads_each ? h_left : a.heads_each;

    const int half = RT == 2 ? wave >> 1 : 0;            // which rows
    const int pair0 = RT == 2 ? wave & 1 : (int)ct * 4 + wave;         // CP = 2: and pair0 + 4
    const int i0 = 16 * RT * half;                       // first row of this wavefront's result
    const int out_head = DOTS ? hk : h_first;
    const SegmentAt at = segment_at(p, w, slot);

    if (p.cu_seqlens != nullptr && (!DOTS || share == 0)) {            // tokens in front of the first sequence and behind the last
        const int64_t front = sequence_tokens(p, 0).lo, back = sequence_tokens(p, p.sequences - 1).hi;
        const int64_t from = ((int64_t)slot * kBlocks + r) * 4 + wave, step = (int64_t)w.slots * kBlocks * 4;
        T *o = static_cast<T *>(a.out) + out_head * a.out_h;
        auto clear = [&](int64_t t) {
            if (a.share == nullptr) {
                for (int c = (int)ct * 128 + lane; c < a.d2 && c < ((int)ct + CP) * 128; c += 64) o[t * a.out_l + c] = Elem<DT>::from_float(0.f);
            } else {
                for (int i = 0; i < a.shares; ++i)
                    for (int c = lane; c < a.d2; c += 64) a.share[(((int64_t)i * p.seqlen + t) * p.heads + hk) * a.d2 + c] = 0.f;
            }
        };
        for (int64_t t = from; t < front; t += step) clear(t);
        for (int64_t t = back + from; t < p.seqlen; t += step) clear(t);
    }
    const int row0 = r * kChunk, own = at.count - row0;  // rows of this block, if any
    if (own <= 0) return;
    const int blocks = (at.count + kChunk - 1) / kChunk;
    const bool rows = i0 < own;                          // of this wavefront's result
    const int slabs = (a.steps + KS - 1) / KS;
    const bool cut = a.d1 < 32 * KS * slabs;
    const bool has_state = (REV ? !at.last : at.c > 0) || a.first;
    const int64_t state = a.first ? (int64_t)slot : border_behind(p, w, at) - !REV;

    auto token = [&](int t) { return t < at.count ? t : at.count - 1; };           // (rows behind the last weigh nothing, or are not stored)
    auto ask_rows = [&](const uint8_t *base, uint32_t pitch, int i, T (&r)[4][CP][2]) {          // rows as a result has them; columns that are not there: the first
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const T *row = reinterpret_cast<const T *>(base + (uint32_t)token(row0 + i0 + 16 * i + 4 * g + e) * pitch);
#pragma unroll
            for (int c = 0; c < CP; ++c) {
                const int col = 32 * (pair0 + 4 * c) + 2 * m;
                r[e][c][0] = row[col < a.d2 ? col : 0];
                r[e][c][1] = row[col + 1 < a.d2 ? col + 1 : 0];
            }
        }
    };
    f32x4 total[DOTS ? RT : 1][DOTS ? CP : 1][2];
    if constexpr (DOTS)
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int c = 0; c < CP; ++c) total[i][c][0] = total[i][c][1] = f32x4{0.f, 0.f, 0.f, 0.f};
    f32x4 acc[RT][CP][2];

    float self_sum = 0.f;                                // wavefront 0: of row `lane`, over the heads
    auto all_columns = [&]() {                           // of row `lane`, from the wavefronts that have it
        return RT == 2 ? lds.dots[2 * (lane >> 5)][lane] + lds.dots[2 * (lane >> 5) + 1][lane] : (lds.dots[0][lane] + lds.dots[1][lane]) + (lds.dots[2][lane] + lds.dots[3][lane]);
    };
    for (int hi = 0; hi < h_count; ++hi) {
        if constexpr (DOTS) {                            // (addresses are made anew: kept over the loop they would take a hundred registers)
            asm volatile("" : "+v"(lane));
            m = lane & 15;
            g = lane >> 4;
        }
        const int h = h_first + hi;
        auto rows_of = [&](const LinearRows &t) { return static_cast<const T *>(t.p) + at.b * t.sb + at.lo * t.sl + (t.by_key ? hk : h) * t.sh; };
        const T *xb = rows_of(a.x), *yb = rows_of(a.y);
        const uint8_t *zb = reinterpret_cast<const uint8_t *>(rows_of(a.z));
        const uint32_t z_pitch = (uint32_t)(a.z.sl * (int64_t)sizeof(T));

        Row8<DT, true> yr[KS];
        auto ask_y = [&](int c, int slab) {
            const T *row = yb + (int64_t)token(c * kChunk + row_of(wave, m)) * a.y.sl;
#pragma unroll
            for (int s = 0; s < KS; ++s) yr[s].ask(row, 32 * (slab * KS + s) + 8 * g, a.d1);
        };
        auto stage_x = [&](int slab) {                   // 16 rows a wavefront
            const T *row = xb + (int64_t)token(row0 + 16 * wave + m) * a.x.sl;
            Row8<DT, true> xr[KS];
#pragma unroll
            for (int s = 0; s < KS; ++s) xr[s].ask(row, 32 * (slab * KS + s) + 8 * g, a.d1);
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                bf16x8 f[NT];
                xr[s].template operand<NT>(32 * (slab * KS + s) + 8 * g, a.d1, cut, f);
#pragma unroll
                for (int n = 0; n < NT; ++n) *reinterpret_cast<u32x4 *>(lds.x + ((wave * KS + s) * NT + n) * kFrag + lane * 16) = bitcast<u32x4>(f[n]);
            }
        };
        const int turns = REV ? blocks - r : r + 1;
        auto block_of = [&](int k) { return REV ? blocks - 1 - k : k; };           // the block itself comes last

        if (hi > 0) lds_barrier();                       // the head before has read its gates and products
        if (slabs == 1) ask_y(block_of(0), 0);
        stage_x(0);
        segment_gates(p, at, h, wave, lane, lds.gates);  // (its barriers are x's too)
        if (wave == 0) {
            const int t = row0 + lane;
            lds.f[lane] = REV ? decay_between(lds.gates, t, kSegment - 1) : decay_since_start(lds.gates, t);
            lds.s[lane] = REV ? lds.gates.beta[t] : p.scale;
        }
        // x as a left operand (its products with the state) and as a right one (y's with it): the same 8 columns of row 16 t + m.
        bf16x8 xr[XREG ? 4 : 1][XREG ? KS : 1][NT];
        auto load_x = [&]() {
            if constexpr (XREG)
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int s = 0; s < KS; ++s) load_frag<NT>(lds.x + (t * KS + s) * NT * kFrag, lane, xr[t][s]);
        };
        load_x();
        auto x_of = [&](int t, int s, bf16x8 (&f)[NT]) {
            if constexpr (XREG) {
#pragma unroll
                for (int n = 0; n < NT; ++n) f[n] = xr[t][s][n];
            } else {
                load_frag<NT>(lds.x + (t * KS + s) * NT * kFrag, lane, f);
            }
        };

#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int c = 0; c < CP; ++c) acc[i][c][0] = acc[i][c][1] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (has_state) {
            const uint8_t *st = a.state + (state * p.v_heads + h) * a.steps * a.tiles * PT * kFrag;
            for (int slab = 0; slab < slabs; ++slab) {
                if (slab > 0) {
                    lds_barrier();
                    stage_x(slab);
                    lds_barrier();
                    load_x();
                }
#pragma unroll
                for (int c = 0; c < CP; ++c) {
                    const int pair = pair0 + 4 * c;
                    if (32 * pair >= a.d2 || !rows) continue;
                    int at_tile[2];
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        const int place = operand_place(32 * pair + 2 * m + n, a.width);
                        at_tile[n] = (place >> 4) * PT * kFrag + (g * 16 + (place & 15)) * 16;
                    }
                    bf16x8 b[2][2][PT];
                    auto ask_state = [&](int s) {        // (steps that are not there: the last, and x is 0)
                        const int step = slab * KS + s < a.steps ? slab * KS + s : a.steps - 1;
#pragma unroll
                        for (int n = 0; n < 2; ++n) load_frag<PT>(st + step * a.tiles * PT * kFrag + at_tile[n], 0, b[s & 1][n]);
                    };
                    ask_state(0);
#pragma unroll
                    for (int s = 0; s < KS; ++s) {
                        if (KS == 8 && slab * KS + s >= a.steps) break;
                        if (s + 1 < KS) ask_state(s + 1);
                        bf16x8 f[RT][NT];
                        f32x4 *to[2][RT];
#pragma unroll
                        for (int i = 0; i < RT; ++i) {
                            if constexpr (RT == 4) x_of(i, s, f[i]);
                            else load_frag<NT>(lds.x + ((half * RT + i) * KS + s) * NT * kFrag, lane, f[i]);
                            to[0][i] = &acc[i][c][0];
                            to[1][i] = &acc[i][c][1];
                        }
                        stay();
#pragma unroll
                        for (int n = 0; n < 2; ++n) products_left<MOST>(f, b[s & 1][n], to[n]);
                    }
                }
            }
        }
        lds_barrier();                                   // f, s
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            const float4 f = *reinterpret_cast<const float4 *>(&lds.f[i0 + 16 * i + 4 * g]);
            const f32x4 by = {f.x, f.y, f.z, f.w};
#pragma unroll
            for (int c = 0; c < CP; ++c)
#pragma unroll
                for (int n = 0; n < 2; ++n) acc[i][c][n] = has_state ? acc[i][c][n] * by : acc[i][c][n];
        }
        // Between blocks: R is G at the end of the block in front (REV: of this one).
        const int border = REV ? row0 + kChunk - 1 : row0 > 0 ? row0 - 1 : 0;
        float of_x[4];                                   // of row 16 t + m
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int i = row0 + 16 * t + m;
            of_x[t] = turns > 1 ? (REV ? decay_between(lds.gates, i, border) : decay_between(lds.gates, border, i)) : 0.f;
        }

        Pair8<DT> zr[CP][2];
        auto ask_z = [&](int block, int s) {
            uint32_t off[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) off[e] = (uint32_t)token(block * kChunk + 32 * s + 8 * g + e) * z_pitch;
#pragma unroll
            for (int c = 0; c < CP; ++c) zr[c][s].ask(zb, off, 32 * (pair0 + 4 * c) + 2 * m, a.d2);
        };
        ask_z(block_of(0), 0);
        ask_z(block_of(0), 1);
        for (int k = 0; k < turns; ++k) {
            const int c0 = block_of(k);
            const bool self = k == turns - 1;
            f32x4 pt[4];                                 // rows: y's four tokens, columns: x's rows 16 t + m
#pragma unroll
            for (int t = 0; t < 4; ++t) pt[t] = f32x4{0.f, 0.f, 0.f, 0.f};
            const int y_half = wave >> 1;
            for (int slab = 0; slab < slabs; ++slab) {
                if (slabs > 1) {
                    lds_barrier();
                    stage_x(slab);
                    ask_y(c0, slab);
                    lds_barrier();
                    load_x();
                }
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    if (KS == 8 && slab * KS + s >= a.steps) break;
                    bf16x8 f[NT], b[4][NT];
#pragma unroll
                    for (int t = 0; t < 4; ++t) x_of(t, s, b[t]);
                    yr[s].template operand<NT>(32 * (slab * KS + s) + 8 * g, a.d1, cut, f);
                    stay();
#pragma unroll
                    for (int sum = 2; sum >= 0; --sum)
#pragma unroll
                        for (int i = 0; i < NT; ++i) {
                            const int j = sum - i;
                            if (j < 0 || j >= NT) continue;
#pragma unroll
                            for (int t = 0; t < 4; ++t) pt[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f[i], b[t][j], pt[t], 0, 0, 0);
                        }
                }
            }
            if (slabs == 1 && !self) ask_y(block_of(k + 1), 0);
            // Weights, terms, and through LDS.
            uint8_t *place = lds.p[product_places(DT, KS) == 1 ? 0 : k & 1];
            if (product_places(DT, KS) == 1 && k > 0) lds_barrier();
            {
                const int j0 = c0 * kChunk + row_of(wave, 4 * g);
                float cj[4], hj[4], lj[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    cj[e] = REV ? (j0 + e < at.count ? p.scale : 0.f) : lds.gates.beta[j0 + e];
                    hj[e] = lds.gates.hi[j0 + e];
                    lj[e] = lds.gates.lo[j0 + e];
                    if (!self) cj[e] *= REV ? decay_between(lds.gates, border, j0 + e) : decay_between(lds.gates, j0 + e, border);
                }
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    float x[4];
                    if (self) {
                        const int i = row0 + 16 * t + m;
                        const float hx = lds.gates.hi[i], lx = lds.gates.lo[i];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float d = REV ? (hj[e] - hx) + (lj[e] - lx) : (hx - hj[e]) + (lx - lj[e]);
                            // DOTS: without the token itself
                            x[e] = (DOTS ? (REV ? j0 + e > i : j0 + e < i) : REV ? j0 + e >= i : j0 + e <= i) ? pt[t][e] * (cj[e] * exp_of(d)) : 0.f;
                            if (DOTS && j0 + e == i) lds.of_self[16 * t + m] = pt[t][e] * cj[e];
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[e] = pt[t][e] * (cj[e] * of_x[t]);
                    }
                    u32x2 f[PT];
                    split4<PT>(x, f);
#pragma unroll
                    for (int n = 0; n < PT; ++n)
                        *reinterpret_cast<u32x2 *>(place + ((t * 2 + y_half) * PT + n) * kFrag + lane * 16 + (wave & 1) * 8) = f[n];
                }
            }
            lds_barrier();
            if (!self || rows)
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    bf16x8 f[RT][PT];
#pragma unroll
                    for (int i = 0; i < RT; ++i) load_frag<PT>(place + ((half * RT + i) * 2 + s) * PT * kFrag, lane, f[i]);
#pragma unroll
                    for (int c = 0; c < CP; ++c) {
                        bf16x8 fz[2][NT];
                        f32x4 *to[2][RT];
#pragma unroll
                        for (int n = 0; n < 2; ++n) {
                            zr[c][s].template operand<NT>(n, fz[n]);
#pragma unroll
                            for (int i = 0; i < RT; ++i) to[n][i] = &acc[i][c][n];
                        }
                        if (c == CP - 1 && !self) ask_z(block_of(k + 1), s);
                        stay();
#pragma unroll
                        for (int n = 0; n < 2; ++n) products_left<MOST>(f, fz[n], to[n]);
                    }
                }
        }

        if constexpr (DOTS) {
            const uint8_t *ub = reinterpret_cast<const uint8_t *>(rows_of(a.u));
            const uint32_t u_pitch = (uint32_t)(a.u.sl * (int64_t)sizeof(T));
            double dot[RT][4];
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                T u[4][CP][2];
                ask_rows(ub, u_pitch, i, u);
                stay();
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    double sum = 0.0;
#pragma unroll
                    for (int c = 0; c < CP; ++c) {
                        const int col = 32 * (pair0 + 4 * c) + 2 * m;
                        sum += col < a.d2 ? (double)acc[i][c][0][e] * (double)Elem<DT>::to_float(u[e][c][0]) : 0.0;
                        sum += col + 1 < a.d2 ? (double)acc[i][c][1][e] * (double)Elem<DT>::to_float(u[e][c][1]) : 0.0;
                    }
                    dot[i][e] = over_columns(sum);
                }
            }
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                const int row = i0 + 16 * i + 4 * g;
                if (m < 4) lds.dots[wave][row + m] = m == 1 ? dot[i][1] : m == 2 ? dot[i][2] : m == 3 ? dot[i][3] : dot[i][0];
                const float4 s = *reinterpret_cast<const float4 *>(&lds.s[row]);
                const f32x4 by = {s.x, s.y, s.z, s.w};
#pragma unroll
                for (int c = 0; c < CP; ++c)
#pragma unroll
                    for (int n = 0; n < 2; ++n) total[i][c][n] += acc[i][c][n] * by;
            }
            lds_barrier();
            if (wave == 0 && lane < own) {
                const float of_self = lds.of_self[lane];
                self_sum = fmaf(of_self, lds.s[lane], self_sum);
                const int64_t to = ((int64_t)at.b * p.v_heads + h) * p.seqlen + at.lo + row0 + lane;
                if (a.selves != nullptr) a.selves[to] = of_self;
                const double d = all_columns();
                a.dots[to] = REV ? d : (double)p.scale * d;
            }
        }
    }

    if constexpr (DOTS) {                                // the tokens themselves
        if (wave == 0) lds.of_self[lane] = self_sum;     // (read by that lane alone so far)
        lds_barrier();
        auto of_key = [&](const LinearRows &t, int i, T (&r)[4][CP][2]) {
            ask_rows(reinterpret_cast<const uint8_t *>(static_cast<const T *>(t.p) + at.b * t.sb + at.lo * t.sl + hk * t.sh), (uint32_t)(t.sl * (int64_t)sizeof(T)), i, r);
        };
        const bool uz = a.uz != nullptr && share == 0;
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            T z[4][CP][2];
            of_key(a.z, i, z);
            const f32x4 by = *reinterpret_cast<const f32x4 *>(&lds.of_self[i0 + 16 * i + 4 * g]);
            stay();
            if (uz) {
                T u[4][CP][2];
                of_key(a.u, i, u);
                stay();
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    double sum = 0.0;
#pragma unroll
                    for (int c = 0; c < CP; ++c) {
                        const int col = 32 * (pair0 + 4 * c) + 2 * m;
#pragma unroll
                        for (int n = 0; n < 2; ++n) sum += col + n < a.d2 ? (double)Elem<DT>::to_float(z[e][c][n]) * (double)Elem<DT>::to_float(u[e][c][n]) : 0.0;
                    }
                    sum = over_columns(sum);
                    if (m == 0) lds.dots[wave][i0 + 16 * i + 4 * g + e] = sum;
                }
            }
#pragma unroll
            for (int c = 0; c < CP; ++c)
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) total[i][c][n][e] = fmaf(by[e], Elem<DT>::to_float(z[e][c][n]), total[i][c][n][e]);
        }
        if (uz) {
            lds_barrier();
            if (wave == 0 && lane < own) a.uz[((int64_t)at.b * p.heads + hk) * p.seqlen + at.lo + row0 + lane] = (float)all_columns();
        }
    }

    // Rows leave as column pairs.
    auto leave = [&](auto *to, uint32_t pitch, auto type) {  // the block's first row, bytes between rows
        using E = std::remove_pointer_t<decltype(to)>;
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            const int row = i0 + 16 * i + 4 * g;
            f32x4 s = {1.f, 1.f, 1.f, 1.f};
            if constexpr (!DOTS) s = *reinterpret_cast<const f32x4 *>(&lds.s[row]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (row + e >= own) continue;
                E *at_row = reinterpret_cast<E *>(reinterpret_cast<uint8_t *>(to) + (uint32_t)(row + e) * pitch);
#pragma unroll
                for (int c = 0; c < CP; ++c) {
                    float o0, o1;
                    if constexpr (DOTS) { o0 = total[i][c][0][e]; o1 = total[i][c][1][e]; }
                    else { o0 = s[e] * acc[i][c][0][e]; o1 = s[e] * acc[i][c][1][e]; }
                    store_pair<decltype(type)::value>(at_row, 32 * (pair0 + 4 * c) + 2 * m, a.d2, o0, o1);
                }
            }
        }
    };
    const int64_t tok = at.lo + row0;
    if (!DOTS || a.share == nullptr)
        leave(static_cast<T *>(a.out) + at.b * a.out_b + tok * a.out_l + out_head * a.out_h, (uint32_t)(a.out_l * (int64_t)sizeof(T)), std::integral_constant<int, DT>());
    else
        leave(a.share + ((((int64_t)share * p.batch + at.b) * p.seqlen + tok) * p.heads + hk) * a.d2, (uint32_t)p.heads * (uint32_t)a.d2 * 4u, std::integral_constant<int, CC1D_F32>());
}

template <int DT, int KS, int RT, bool REV>
__global__ void __launch_bounds__(kBlock, attend_waves(false, DT, KS, 1))
linear_attend_kernel(const cc1d_delta_params p, const SegmentWork w, const AttendArgs a) {
    attend_rows<DT, KS, RT, 1, REV, false>(p, w, a, blockIdx.x);
}
// dq and dk in one launch, `half` workgroups each: neither waits for the other, and one alone may leave CUs idle (24 workgroups each: 25 us, one
// after the other 47; 128 each of linear_tile_pair_kernel: 32 and 49; 256 each, which fill the card: 380 and 385 at best).  float32: dv's workgroups behind them, if all together
// are no more than CUs (24 each: 26 us, for 25 and 20); more of them leave no CU idle by themselves.
template <int DT, int KS, int RT, int CP>
__global__ void __launch_bounds__(kBlock, attend_waves(true, DT, KS, CP))
linear_attend_pair_kernel(const cc1d_delta_params p, const SegmentWork w, const AttendArgs q, const AttendArgs k, const AttendArgs v, const uint32_t half) {
    if (blockIdx.x < half) attend_rows<DT, KS, RT, CP, false, true>(p, w, q, blockIdx.x);
    else if (DT != CC1D_F32 || blockIdx.x < 2 * half) attend_rows<DT, KS, RT, CP, true, true>(p, w, k, blockIdx.x - half);
    else if constexpr (DT == CC1D_F32) attend_rows<DT, RT == 2 ? 2 : 4, KS == 2 ? 2 : 4, 1, true, false>(p, w, v, blockIdx.x - 2 * half);
}

}  // namespace cc1d
