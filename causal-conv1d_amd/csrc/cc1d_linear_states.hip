// Linear attention: the sums a segment adds to the state (or to its gradient), the recurrence over segments, and the gates' gradients
// (cc1d_linear.hpp).
#include "cc1d_delta_host.hpp"
#include "cc1d_linear_device.hpp"

namespace cc1d {
namespace {

// sum over a segment's tokens of weight_t a_t b_t^T, one workgroup a (slot, value head, 128 columns of b): a wavefront takes 32 columns of b, all
// columns of a; where b has at most 64, two wavefronts share those and take half of a each.  The weight goes to b, which is split into three
// terms then; a stays as it is, one term in bfloat16.  No operand goes through LDS: pairs of columns (Pair8) are loaded in the order
// of the matrix instruction, and the result tiles of a pair of a's are eight consecutive rows of a lane, the operand order of the next product.
// KT: 32-column steps of a that a wavefront takes.
// 32 segments of 80 heads of 128 x 64, bfloat16: 71 us, 86 MB read and 73 written, 2.2 TB/s; 64 segments of 16 heads of 128 x 128, float16: 63.  Splits, addresses
// and loads of 4 bytes share the time; two steps asked for ahead: 74 and 65; loads of 8 bytes with 4 x 4 tiles a wavefront: 89 and 71.
template <int DT, int KT>
__global__ void __launch_bounds__(kBlock, KT <= 4 && DT != CC1D_F32 ? 2 : 1)
linear_states_kernel(const cc1d_delta_params p, const SegmentWork w, const StatesArgs a, const int halves, const uint32_t col_tiles) {
    using T = typename Elem<DT>::type;
    constexpr int NT = Terms<DT>::n;
    __shared__ GateLds gates;
    __shared__ float weight[kSegment];
    const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t sv = blockIdx.x / col_tiles, ct = blockIdx.x - sv * col_tiles;
    const int slot = (int)divided(sv, w.by_v_heads), h = (int)sv - slot * p.v_heads, hk = (int)divided((uint32_t)h, w.by_group);
    const SegmentAt at = segment_at(p, w, slot);
    if (at.count <= 0 || !(a.all || (a.from_start ? at.c > 0 : !at.last))) return;

    segment_gates(p, at, h, wave, lane, gates);
    {
        const int i = threadIdx.x;
        if (i < kSegment) weight[i] = i >= at.count ? 0.f : a.from_start ? a.factor * decay_since_start(gates, i) : gates.beta[i] * decay_between(gates, i, kSegment - 1);
        if (i == 0 && ct == 0) w.decay[sv] = decay_since_start(gates, kSegment - 1);
    }
    lds_barrier();

    const int q = halves ? wave & 1 : (int)ct * 4 + wave, p0 = halves ? (wave >> 1) * KT : 0;
    if (q >= w.vp || p0 >= w.kp) return;
    const int cb = 32 * q + 2 * m;
    const uint8_t *ab = reinterpret_cast<const uint8_t *>(static_cast<const T *>(a.a.p) + at.b * a.a.sb + at.lo * a.a.sl + (a.a.by_key ? hk : h) * a.a.sh);
    const uint8_t *bb = reinterpret_cast<const uint8_t *>(static_cast<const T *>(a.b.p) + at.b * a.b.sb + at.lo * a.b.sl + (a.b.by_key ? hk : h) * a.b.sh);
    const uint32_t a_pitch = (uint32_t)(a.a.sl * (int64_t)sizeof(T)), b_pitch = (uint32_t)(a.b.sl * (int64_t)sizeof(T));

    f32x4 acc[KT][2][2];
#pragma unroll
    for (int i = 0; i < KT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][e >> 1][e & 1] = f32x4{0.f, 0.f, 0.f, 0.f};
    Pair8<DT> ra[KT], rb;
    auto ask = [&](int t0) {             // 32 tokens from t0 on; those behind the last take its rows, and their weight is 0
        uint32_t at_a[8], at_b[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int t = t0 + 8 * g + e;
            const uint32_t tok = (uint32_t)(t < at.count ? t : at.count - 1);
            at_a[e] = tok * a_pitch;
            at_b[e] = tok * b_pitch;
        }
        rb.ask(bb, at_b, cb, p.dim_v);
#pragma unroll
        for (int i = 0; i < KT; ++i) ra[i].ask(ab, at_a, 32 * (p0 + i) + 2 * m, p.dim_k);
    };
    // The matrix cores round their sums downwards by a little, 1e-8 of them over a segment, and S0 . dS0 does not average away what all elements are off by:
    // odd columns are summed up with the other sign.
    ask(0);
    for (int t0 = 0; t0 < at.count; t0 += 32) {
        bf16x8 fb[2][3], fa[KT][2][NT];
        {
            const float4 w0 = *reinterpret_cast<const float4 *>(&weight[t0 + 8 * g]), w1 = *reinterpret_cast<const float4 *>(&weight[t0 + 8 * g + 4]);
            const float wt[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                float f[8];
                rb.get(n, f);
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] *= n == 0 ? wt[e] : -wt[e];
                split8<3>(f, fb[n]);
            }
        }
#pragma unroll
        for (int i = 0; i < KT; ++i)
#pragma unroll
            for (int n = 0; n < 2; ++n) ra[i].template operand<NT>(n, fa[i][n]);
        if (t0 + 32 < at.count) ask(t0 + 32);
        stay();
#pragma unroll
        for (int i = 0; i < KT; ++i)
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) acc[i][n][c] = product<2>(fa[i][n], fb[c], acc[i][n][c]);
        stay();
    }
    const int64_t state = a.all ? (int64_t)slot : border_behind(p, w, at) - a.from_start;         // (of whom it meets)
    // Rows of a's pair i: dim_k index 32 (p0 + i) + 8 g + 2 e + n.  Padding is 0: it meets other operands' padding.
#pragma unroll
    for (int i = 0; i < KT; ++i) {
        if (p0 + i >= w.kp) break;
        float *to = w.local + (((state * p.v_heads + h) * w.kp + p0 + i) * w.vp + q) * 1024 + lane * 8;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            float f[8];
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int n = 0; n < 2; ++n)
                    f[2 * e + n] = 32 * (p0 + i) + 8 * g + 2 * e + n < p.dim_k && cb + c < p.dim_v ? (c == 0 ? acc[i][n][c][e] : -acc[i][n][c][e]) : 0.f;
            *reinterpret_cast<float4 *>(to + c * 512) = make_float4(f[0], f[1], f[2], f[3]);
            *reinterpret_cast<float4 *>(to + c * 512 + 4) = make_float4(f[4], f[5], f[6], f[7]);
        }
    }
}

// Rows to whole vectors and back, a wavefront a token of one tensor; single elements on the odd side.  62 heads of 41, 3676 tokens, float32 (37 MB read, 43
// written): 51 us.
template <typename E, bool OUT>
__global__ void __launch_bounds__(kBlock)
linear_copy_kernel(const CopyArgs a, const int64_t tokens) {
    const CopyRows &c = a.of[blockIdx.y];
    struct alignas(16) Vector { E e[kVector]; };
    const int lane = threadIdx.x & 63, vectors = padded(c.dim) / kVector;
    for (int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); t < tokens; t += (int64_t)gridDim.x * 4) {
        const int64_t b = divided((uint32_t)t, a.by_seqlen), l = t - b * a.seqlen;
        const uint8_t *from = c.from + b * c.from_b + l * c.from_l;
        uint8_t *to = c.to + b * c.to_b + l * c.to_l;
        for (int i = lane; i < c.heads * vectors; i += 64) {
            const int h = (int)divided((uint32_t)i, c.by_vectors), col = (i - h * vectors) * kVector;
            const E *x = reinterpret_cast<const E *>(from + h * c.from_h) + col;
            E *y = reinterpret_cast<E *>(to + h * c.to_h) + col;
            if constexpr (OUT) {
                const Vector v = *reinterpret_cast<const Vector *>(x);
#pragma unroll
                for (int k = 0; k < kVector; ++k)
                    if (col + k < c.dim) y[k] = v.e[k];
            } else {
                Vector v;
#pragma unroll
                for (int k = 0; k < kVector; ++k) v.e[k] = col + k < c.dim ? x[k] : (E)0;
                *reinterpret_cast<Vector *>(y) = v;
            }
        }
    }
}

// The recurrence over a sequence's segments, one wavefront a tile of 32 x 32 of one (sequence, value head): elementwise, bound by memory.  In front
// of every segment (REVERSE: behind it) the state leaves as operands: contracted over dim_k as it lies, contracted over dim_v turned around through LDS.
// 4 sequences of 8 segments, 80 heads of 128 x 64: 57 us forward (73 MB of sums read, 183 of operands of both kinds written, 4.5 TB/s), 88 backward (110 MB of the
// forward's operands more).  Those asked for ahead too: 92, their registers leave fewer wavefronts.
template <int KTERMS>
__global__ void __launch_bounds__(64)
linear_scan_kernel(const cc1d_delta_params p, const SegmentWork w, const ScanArgs a, const FastDiv by_tiles, const FastDiv by_vp) {
    __shared__ float turn[32][36];
    const int lane = threadIdx.x, m = lane & 15, g = lane >> 4;
    const uint32_t tiles = (uint32_t)w.tiles(), nh = divided(blockIdx.x, by_tiles), tile = blockIdx.x - nh * tiles;
    const int walk = (int)divided(nh, w.by_v_heads), h = (int)nh - walk * p.v_heads;
    const int n = w.shortest > 0 ? sequence_of(p, (int64_t)walk << kSegmentLog) : walk;             // (then of the sequence that holds that token, if it is the one that names it)
    const int pi = (int)divided(tile, by_vp), q = (int)tile - pi * w.vp;
    const TokenRange range = sequence_tokens(p, n);
    if (w.shortest > 0 && (range.hi - range.lo < w.shortest || naming(range) != walk)) return;
    const int chunks = (int)((range.hi - range.lo + kSegment - 1) >> kSegmentLog), slot0 = first_segment(p, w, n, range);
    const int k0 = 32 * pi + 8 * g, v0 = 32 * q + 2 * m;

    float s[2][8];
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            s[c][e] = 0.f;
            if (a.first != nullptr && k0 + e < p.dim_k && v0 + c < p.dim_v) s[c][e] = a.first[n * a.first_n + h * a.first_h + (k0 + e) * a.first_k + v0 + c];
        }
    // Segment c's own sum lies where the state does that it makes: behind it (REVERSE: in front), and states where the segment is that reads them.
    const int64_t border0 = border_behind(p, w, n, range.lo, 0);
    auto sum_of = [&](int c) { return a.to_end ? (int64_t)slot0 + c : border0 + c - a.reverse; };
    auto state_of = [&](int c) { return a.first != nullptr ? (int64_t)slot0 + c : border0 + c - 1 + a.reverse; };
    auto place = [&](int64_t state) { return (state * p.v_heads + h) * tiles + tile; };
    struct Step { float4 x[4]; float decay; };
    // Segment i of the walk; its sum is there only if somebody behind it in the walk needs it.
    auto chunk_of = [&](int i) { return a.reverse ? chunks - 1 - i : i; };
    const int summed = a.to_end ? chunks : chunks - 1;
    auto ask = [&](int i) {
        Step x;
        if (i >= summed) i = summed > 0 ? summed - 1 : 0;
        const float *from = w.local + place(sum_of(chunk_of(i))) * 1024 + lane * 8;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            x.x[2 * c] = *reinterpret_cast<const float4 *>(from + c * 512);
            x.x[2 * c + 1] = *reinterpret_cast<const float4 *>(from + c * 512 + 4);
        }
        x.decay = w.decay[(int64_t)(slot0 + chunk_of(i)) * p.v_heads + h];
        return x;
    };
    auto turned = [&](float (&t)[2][8]) {                // lane (m, g): rows 2 m + c of dim_k, columns 8 g + e of dim_v
        wave_lds_fence();
#pragma unroll
        for (int e = 0; e < 8; ++e) *reinterpret_cast<float2 *>(&turn[8 * g + e][2 * m]) = make_float2(s[0][e], s[1][e]);
        wave_lds_fence();
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const float4 lo = *reinterpret_cast<const float4 *>(&turn[2 * m + c][8 * g]), hi = *reinterpret_cast<const float4 *>(&turn[2 * m + c][8 * g + 4]);
            t[c][0] = lo.x; t[c][1] = lo.y; t[c][2] = lo.z; t[c][3] = lo.w;
            t[c][4] = hi.x; t[c][5] = hi.y; t[c][6] = hi.z; t[c][7] = hi.w;
        }
    };
    // Where this lane's two columns lie among a step's operands (of one term).
    int k_place[2], v_place[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const int kc = operand_place(v0 + c, w.k_width), vc = operand_place(32 * pi + 2 * m + c, w.v_width);
        k_place[c] = (kc >> 4) * KTERMS * kFrag + (g * 16 + (kc & 15)) * 16;
        v_place[c] = (vc >> 4) * 3 * kFrag + (g * 16 + (vc & 15)) * 16;
    }
    auto by_k_step = [&](int64_t state) { return (((state * p.v_heads + h) * w.kp + pi) * w.k_tiles) * KTERMS * kFrag; };
    auto by_v_step = [&](int64_t state) { return (((state * p.v_heads + h) * w.vp + q) * w.v_tiles) * 3 * kFrag; };
    // S0 . dS0 of a segment whose dS0 is at hand: S0 as the forward left it.
    auto inner = [&](int c, const float (&t)[2][8]) {
        const int64_t state = a.use_inner == 2 ? (int64_t)slot0 + c : border0 + c - 1;
        const uint8_t *from = w.first + by_v_step(state);
        double sum = 0.0;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            bf16x8 f[3];
            load_frag<3>(from + v_place[c], 0, f);
            float x[4];
            four_of(f, false, x);
#pragma unroll
            for (int e = 0; e < 4; ++e) sum = fma((double)x[e], (double)t[c][e], sum);
            four_of(f, true, x);
#pragma unroll
            for (int e = 0; e < 4; ++e) sum = fma((double)x[e], (double)t[c][4 + e], sum);
        }
        sum = over_wave(sum);
        if (lane == 0) w.inner[place(state)] = sum;
    };

    constexpr int AHEAD = 4;             // segments asked for ahead: the loop waits for memory alone
    Step next[AHEAD];
    if (summed > 0)
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) next[i] = ask(i);
    for (int i0 = 0; i0 < chunks; i0 += AHEAD) {
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            const int i = i0 + j;
            if (i >= chunks) break;
            const int c = chunk_of(i);
            if (i > 0 || a.first != nullptr) {
                if (a.write_k) {
                    uint8_t *to = w.by_k + by_k_step(state_of(c));
#pragma unroll
                    for (int o = 0; o < 2; ++o) {
                        bf16x8 f[KTERMS];
                        split8<KTERMS>(s[o], f);
#pragma unroll
                        for (int t = 0; t < KTERMS; ++t) *reinterpret_cast<u32x4 *>(to + k_place[o] + t * kFrag) = bitcast<u32x4>(f[t]);
                    }
                }
                if (a.write_v || a.use_inner) {
                    float t[2][8];
                    turned(t);
                    if (a.write_v) {
                        uint8_t *to = w.by_v + by_v_step(state_of(c));
#pragma unroll
                        for (int o = 0; o < 2; ++o) {
                            bf16x8 f[3];
                            split8<3>(t[o], f);
#pragma unroll
                            for (int k = 0; k < 3; ++k) *reinterpret_cast<u32x4 *>(to + v_place[o] + k * kFrag) = bitcast<u32x4>(f[k]);
                        }
                    }
                    if (a.use_inner && i > 0) inner(c + 1, t);               // (reverse: what is behind this segment is in front of the one behind it)
                }
            }
            if (i < summed) {
                const Step &x = next[j];
                const float add[2][8] = {{x.x[0].x, x.x[0].y, x.x[0].z, x.x[0].w, x.x[1].x, x.x[1].y, x.x[1].z, x.x[1].w},
                                         {x.x[2].x, x.x[2].y, x.x[2].z, x.x[2].w, x.x[3].x, x.x[3].y, x.x[3].z, x.x[3].w}};
#pragma unroll
                for (int o = 0; o < 2; ++o)
#pragma unroll
                    for (int e = 0; e < 8; ++e) s[o][e] = fmaf(x.decay, s[o][e], add[o][e]);
            }
            if (summed > 0) next[j] = ask(i + AHEAD);
        }
    }
    if (a.use_inner == 2 && chunks > 0) {                // there is an initial state, and its gradient is at hand
        float t[2][8];
        turned(t);
        inner(0, t);
    }
    if (a.last == nullptr) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if (k0 + e >= p.dim_k) continue;
        float *to = a.last + n * a.last_n + h * a.last_h + (k0 + e) * a.last_k + v0;
        if (v0 < p.dim_v) to[0] = s[0][e];
        if (v0 + 1 < p.dim_v) to[1] = s[1][e];
    }
}

// dg and dbeta of a segment, one wavefront each (slot, value head): bound by latency and by stores v_heads apart, 19 us for 2560 of them; sixteen heads a workgroup
// whose results pass through LDS 20 as well, and of 8 heads 8.5 for 6.
__global__ void __launch_bounds__(kBlock)
linear_gates_kernel(const cc1d_delta_bwd_params bp, const SegmentWork w, const uint32_t items, const int first) {
    const cc1d_delta_params &p = bp.fwd;
    const int lane = threadIdx.x & 63;
    const uint32_t sv = blockIdx.x * 4u + (threadIdx.x >> 6);
    if (sv >= items) return;
    const int slot = (int)divided(sv, w.by_v_heads), h = (int)sv - slot * p.v_heads;
    auto put = [&](int64_t at, float dg, float dbeta) {
        store_from_float(bp.dg, at, p.g_dtype, dg);
        if (p.beta != nullptr) store_from_float(bp.dbeta, at, p.beta_dtype, dbeta);
    };
    if (p.cu_seqlens != nullptr) {                       // tokens in front of the first sequence and behind the last
        const int64_t front = sequence_tokens(p, 0).lo, back = sequence_tokens(p, p.sequences - 1).hi;
        for (int64_t t = (int64_t)slot * 64 + lane; t < front; t += (int64_t)w.slots * 64) put(t * p.v_heads + h, 0.f, 0.f);
        for (int64_t t = back + (int64_t)slot * 64 + lane; t < p.seqlen; t += (int64_t)w.slots * 64) put(t * p.v_heads + h, 0.f, 0.f);
    }
    const SegmentAt at = segment_at(p, w, slot);
    if (at.count <= 0) return;
    const int64_t state = first ? (int64_t)slot : border_behind(p, w, at) - 1;
    auto inner = [&](int64_t of) {                       // S0 . dS0
        double sum = 0.0;
        for (int64_t i = lane; i < w.tiles(); i += 64) sum += w.inner[(of * p.v_heads + h) * w.tiles() + i];
        return over_wave(sum);
    };
    const int64_t token0 = ((int64_t)at.b * p.v_heads + h) * p.seqlen + at.lo;
    double change[kBlocks], size[kBlocks], total = 0.0, sizes = 0.0;
    float kz[kBlocks];
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
        const int t = b * kChunk + lane, there = t < at.count ? t : at.count - 1;
        float beta = 1.f;
        if (p.beta != nullptr) beta = bits_as_float(load_bits(p.beta, at.b * p.beta_stride_b + (at.lo + there) * p.beta_stride_l + h * p.beta_stride_h, p.beta_dtype), p.beta_dtype);
        const double qd = w.dot_q[token0 + there], z = w.dot_k[token0 + there];
        kz[b] = 0.f;
        if (p.beta != nullptr)
            kz[b] = (float)(z + (double)w.self_k[token0 + there] * (double)w.qk[((int64_t)at.b * p.heads + divided((uint32_t)h, w.by_group)) * p.seqlen + at.lo + there]);
        change[b] = t < at.count ? qd - (double)beta * z : 0.0;
        size[b] = t < at.count ? fabs(qd) + fabs((double)beta * z) : 0.0;
    }
    double dg = at.c > 0 || first ? inner(state) : 0.0, rest = 0.0;
    const bool known = !at.last || !bp.dfinal_states;    // what comes behind the last token
    const double end = at.last || !known ? 0.0 : inner(state + 1);
    double before[kBlocks], share[kBlocks];              // changes in front of each token, and the sizes of what they are differences of
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
        const double sum = running_sum(change[b]), all = running_sum(size[b]);
        before[b] = total + (sum - change[b]);
        share[b] = sizes + (all - size[b]);
        total += of_lane(sum, 63);
        sizes += of_lane(all, 63);
    }
    if (known) rest = end - (dg - total);
    rest = fabs(rest) < 1e300 && sizes > 0.0 ? rest / sizes : 0.0;       // (of numbers)
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
        const int t = b * kChunk + lane;
        if (t < at.count) put(((int64_t)at.b * p.seqlen + at.lo + t) * p.v_heads + h, (float)((dg - before[b]) + rest * share[b]), kz[b]);
    }
}

// dq and dk of a key head whose value heads were several workgroups': their shares in a fixed order.  Bound by memory: four shares of 8192 rows of 128 each, 34 MB, 13 us.
template <int DT>
__global__ void __launch_bounds__(kBlock)
linear_join_kernel(const cc1d_delta_bwd_params bp, const SegmentWork w, const int64_t rows) {
    using T = typename Elem<DT>::type;
    const cc1d_delta_params &p = bp.fwd;
    const int pitch = padded(p.dim_k);
    const int64_t plane = rows * pitch;
    for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < rows; r += (int64_t)gridDim.x * 4) {
        const int64_t t = r / p.heads, b = t / p.seqlen;
        const int hk = (int)(r - t * p.heads);
        for (int k = threadIdx.x & 63; k < p.dim_k; k += 64) {
            float dq = 0.f, dk = 0.f;
            for (int i = 0; i < w.shares; ++i) {
                dq += w.share_q[i * plane + r * pitch + k];
                dk += w.share_k[i * plane + r * pitch + k];
            }
            static_cast<T *>(bp.dq)[b * bp.dq_stride_b + (t - b * p.seqlen) * bp.dq_stride_l + hk * bp.dq_stride_h + k] = Elem<DT>::from_float(dq);
            static_cast<T *>(bp.dk)[b * bp.dk_stride_b + (t - b * p.seqlen) * bp.dk_stride_l + hk * bp.dk_stride_h + k] = Elem<DT>::from_float(dk);
        }
    }
}

template <int DT>
int launch_states(const cc1d_delta_params &p, const SegmentWork &w, const StatesArgs &a, hipStream_t stream) {
    const int halves = w.vp <= 2, each = halves ? (w.kp + 1) / 2 : w.kp;
    const uint32_t col_tiles = halves ? 1 : (uint32_t)(w.vp + 3) / 4;
    const dim3 grid((uint32_t)w.slots * (uint32_t)p.v_heads * col_tiles);
    auto go = [&](auto kt) {
        constexpr int KT = decltype(kt)::value;
        CC1D_LAUNCH((linear_states_kernel<DT, KT>), grid, dim3(kBlock), 0, stream, p, w, a, halves, col_tiles);
        return launch_status();
    };
    return each <= 1 ? go(std::integral_constant<int, 1>()) : each <= 2 ? go(std::integral_constant<int, 2>()) :
           each <= 4 ? go(std::integral_constant<int, 4>()) : go(std::integral_constant<int, 8>());
}

}  // namespace

int launch_linear_copy(const CopyArgs &a, int copies, bool out, hipStream_t stream) {
    const int64_t tokens = (int64_t)a.batch * a.seqlen, blocks = (tokens + 3) / 4;
    if (tokens == 0 || copies == 0) return CC1D_OK;
    const dim3 grid((uint32_t)(blocks < 16384 ? blocks : 16384), (uint32_t)copies);
    auto go = [&](auto e) {
        using E = decltype(e);
        if (out) CC1D_LAUNCH((linear_copy_kernel<E, true>), grid, dim3(kBlock), 0, stream, a, tokens);
        else CC1D_LAUNCH((linear_copy_kernel<E, false>), grid, dim3(kBlock), 0, stream, a, tokens);
        return launch_status();
    };
    return a.elem == 4 ? go(uint32_t()) : go(uint16_t());
}
int launch_linear_states(const cc1d_delta_params &p, const SegmentWork &w, const StatesArgs &a, hipStream_t stream) {
    if (w.slots == 0) return CC1D_OK;
    switch (p.x_dtype) {
        case CC1D_F32: return launch_states<CC1D_F32>(p, w, a, stream);
        case CC1D_F16: return launch_states<CC1D_F16>(p, w, a, stream);
        default: return launch_states<CC1D_BF16>(p, w, a, stream);
    }
}

int launch_linear_scan(const cc1d_delta_params &p, const SegmentWork &w, const ScanArgs &a, hipStream_t stream) {
    const dim3 grid((uint32_t)(w.walks(p) * p.v_heads * w.tiles()));
    const FastDiv by_tiles = fast_div((uint32_t)w.tiles()), by_vp = fast_div((uint32_t)w.vp);
    if (out_terms(p.x_dtype) == 3) CC1D_LAUNCH(linear_scan_kernel<3>, grid, dim3(64), 0, stream, p, w, a, by_tiles, by_vp);
    else CC1D_LAUNCH(linear_scan_kernel<2>, grid, dim3(64), 0, stream, p, w, a, by_tiles, by_vp);
    return launch_status();
}

int launch_linear_gates(const cc1d_delta_bwd_params &bp, const SegmentWork &w, hipStream_t stream) {
    const uint32_t items = (uint32_t)w.slots * (uint32_t)bp.fwd.v_heads;
    if (items == 0) return CC1D_OK;
    CC1D_LAUNCH(linear_gates_kernel, dim3((items + 3) / 4), dim3(kBlock), 0, stream, bp, w, items, (int)(bp.fwd.initial_states != nullptr));
    return launch_status();
}

int launch_linear_join(const cc1d_delta_bwd_params &bp, const SegmentWork &w, hipStream_t stream) {
    const cc1d_delta_params &p = bp.fwd;
    const int64_t rows = (int64_t)p.batch * p.seqlen * p.heads;
    if (rows == 0) return CC1D_OK;
    const dim3 grid((uint32_t)(rows < 4 * 8192 ? (rows + 3) / 4 : 8192));
    switch (p.x_dtype) {
        case CC1D_F32: CC1D_LAUNCH(linear_join_kernel<CC1D_F32>, grid, dim3(kBlock), 0, stream, bp, w, rows); break;
        case CC1D_F16: CC1D_LAUNCH(linear_join_kernel<CC1D_F16>, grid, dim3(kBlock), 0, stream, bp, w, rows); break;
        default: CC1D_LAUNCH(linear_join_kernel<CC1D_BF16>, grid, dim3(kBlock), 0, stream, bp, w, rows);
    }
    return launch_status();
}

}  // namespace cc1d
