// The gated delta rule by chunks, first kernel: everything of a chunk that needs no state (cc1d_delta_chunk.hpp).
// One workgroup a chunk and value head: K K^T and Q K^T on the matrix cores, T = (I + A)^-1, and the operands of the
// later kernels in the order in which these load them.
//
// T: the four 16 x 16 blocks on the diagonal by substitution, one wavefront each with a column a lane; below it by fp32 matrix
// instructions, first inside each half of 32, then between the halves: (I + A)^-1 of [[X, 0], [A, Y]] has -Y^-1 A X^-1 there.
// Substitution and not the series of powers of A: those of keys that resemble each other grow to 1e8 before they vanish.
//
// One workgroup a CU takes 11.6 us (256 chunks and heads of 128 in bfloat16), 15500 cycles of latency: 6000 until K and Q are in LDS and
// their lengths known, 2700 for the products, 2000 and 2400 for T's two parts, 2000 to write T and P.  Four to a CU share that: 2048 chunks 53 us, 160 MB
// written.  K and Q are written out again in operand order: it costs a third of the writes, and saves the scan 10 to 20 %.
#include "cc1d_delta_chunk.hpp"
#include "cc1d_delta_host.hpp"

namespace cc1d {
namespace {

constexpr int kPitch = 68;               // floats of a row of a 64 x 64 matrix in LDS

template <int DT, int KS>
struct PrepLds {
    union {
        uint8_t frags[4 * KS * Terms<DT>::n * kFrag];    // K, then Q; then T
        float t[kChunk][kPitch];
    };
    float a[kChunk][kPitch];
    float gate[kScalars][kChunk];
};

// Wavefronts a SIMD: as many as the workgroups that LDS has room for.
constexpr int prep_waves(int dt, int ks) {
    const int terms = dt == CC1D_BF16 ? 1 : dt == CC1D_F16 ? 2 : 3;
    return ks * terms <= 4 ? 4 : ks * terms <= 8 ? 3 : 1;
}

// The 16 x 16 product of two blocks in LDS, added to acc.
__device__ __forceinline__ f32x4 block_product(const float *x, int px, const float *y, int py, f32x4 acc, int m, int g) {
#pragma unroll
    for (int s = 0; s < 4; ++s)
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x[m * px + 4 * s + g], y[(4 * s + g) * py + m], acc, 0, 0, 0);
    return acc;
}

// x[i] -= a[i][k] x[k] for all i > k, k growing: a lane holds a column of both, a[i][k] is lane k's and the same for all.
template <int K>
__device__ __forceinline__ void below_diagonal(const float (&a)[16], float (&x)[16]) {
#pragma unroll
    for (int i = K + 1; i < 16; ++i) x[i] -= bitcast<float>(__builtin_amdgcn_readlane(bitcast<int>(a[i]), K)) * x[K];
    if constexpr (K < 14) below_diagonal<K + 1>(a, x);
}

template <int DT, int KS, bool VEC>
__global__ void __launch_bounds__(kBlock, prep_waves(DT, KS))
delta_prep_kernel(const cc1d_delta_params p, const ChunkWork w) {
    using T = typename Elem<DT>::type;
    constexpr int NT = Terms<DT>::n, PT = Terms<DT>::p;
    extern __shared__ uint4 raw[];
    PrepLds<DT, KS> &lds = *reinterpret_cast<PrepLds<DT, KS> *>(raw);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, g = lane >> 4;
    const int slot = (int)divided(blockIdx.x, w.by_v_heads), h = (int)blockIdx.x - slot * p.v_heads;
    const int hk = (int)divided((uint32_t)h, w.by_group);
    const bool first = h == 0 || (int)divided((uint32_t)h - 1u, w.by_group) != hk;                  // this workgroup writes what the heads of the group share
    const ChunkAt at = chunk_at(p, w, slot);
    if (at.count <= 0) return;
    const int64_t sh = (int64_t)slot * p.heads + hk, sv = (int64_t)slot * p.v_heads + h;

    // Gates: asked for first, summed while K and Q travel.
    uint32_t gate_bits = 0, beta_bits = 0;
    {
        const int64_t tok = at.lo + (lane < at.count ? lane : 0);
        gate_bits = load_bits(p.g, at.b * p.g_stride_b + tok * p.g_stride_l + h * p.g_stride_h, p.g_dtype);
        beta_bits = load_bits(p.beta, at.b * p.beta_stride_b + tok * p.beta_stride_l + h * p.beta_stride_h, p.beta_dtype);
    }
    stay();

    // Rows of K and Q as left operands; their lengths.
    const int token = row_of(wave, m);
    const bool there = token < at.count;
    const T *kp = static_cast<const T *>(p.k) + at.b * p.k_stride_b + (at.lo + (there ? token : 0)) * p.k_stride_l + hk * p.k_stride_h;
    const T *qp = static_cast<const T *>(p.q) + at.b * p.q_stride_b + (at.lo + (there ? token : 0)) * p.q_stride_l + hk * p.q_stride_h;
    bf16x8 kf[KS][NT], qf[KS][NT];
    float kk = 0.f, qq = 0.f;
    const int cols = there ? p.dim_k : 0;
    {
        Row8<DT, VEC> kr[KS], qr[KS];
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            kr[s].ask(kp, 32 * s + 8 * g, cols);
            qr[s].ask(qp, 32 * s + 8 * g, cols);
        }
        stay();
        // Sums of gates in 64 bits, kept as two floats: differences of large sums lose nothing.
        if (wave == 0) {
            const double sum = running_sum(lane < at.count ? (double)bounded_gate(bits_as_float(gate_bits, p.g_dtype)) : 0.0);
            const double last = of_lane(sum, 63);
            const float hi = (float)sum;
            lds.gate[kBeta][lane] = lane < at.count ? bits_as_float(beta_bits, p.beta_dtype) : 0.f;
            lds.gate[kGate][lane] = exp_of((float)sum);
            lds.gate[kToEnd][lane] = exp_of((float)(last - sum));
            lds.gate[kSumHi][lane] = hi;
            lds.gate[kSumLo][lane] = (float)(sum - (double)hi);
        }
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            float x[8];
            kr[s].get(32 * s + 8 * g, cols, true, x);
#pragma unroll
            for (int i = 0; i < 8; ++i) kk += x[i] * x[i];
            kr[s].template operand<NT>(32 * s + 8 * g, cols, true, kf[s]);
            qr[s].get(32 * s + 8 * g, cols, true, x);
#pragma unroll
            for (int i = 0; i < 8; ++i) qq += x[i] * x[i];
            qr[s].template operand<NT>(32 * s + 8 * g, cols, true, qf[s]);
#pragma unroll
            for (int n = 0; n < NT; ++n)
                *reinterpret_cast<u32x4 *>(lds.frags + ((wave * KS + s) * NT + n) * kFrag + lane * 16) = bitcast<u32x4>(kf[s][n]);
        }
    }
    kk = over_rows(kk);
    qq = over_rows(qq);
    if (g == 0) {
        lds.gate[kKeyNorm][token] = p.qk_l2norm ? rsqrtf(kk + kNormEps) : 1.f;
        lds.gate[kQueryNorm][token] = p.qk_l2norm ? rsqrtf(qq + kNormEps) : 1.f;
    }
    lds_barrier();

    // K K^T and Q K^T: this wavefront's 16 rows; columns behind the rows' last are nothing.
    f32x4 read[4];                                       // P waits in registers until A is used up
    float hi_i[4], lo_i[4], of_a[4], of_p[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int i = row_of(wave, 4 * g + e);
        hi_i[e] = lds.gate[kSumHi][i];
        lo_i[e] = lds.gate[kSumLo][i];
        of_a[e] = lds.gate[kBeta][i] * lds.gate[kKeyNorm][i];
        of_p[e] = p.scale * lds.gate[kQueryNorm][i];
    }
    auto half = [&](int c2) {                            // columns 32 c2 on
        f32x4 a[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}}, r[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
        float hi_j[2], lo_j[2], norm_j[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int j = row_of(2 * c2 + c, m);
            hi_j[c] = lds.gate[kSumHi][j];
            lo_j[c] = lds.gate[kSumLo][j];
            norm_j[c] = lds.gate[kKeyNorm][j];
        }
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                bf16x8 b[NT];
                load_frag<NT>(lds.frags + ((2 * c2 + c) * KS + s) * NT * kFrag, lane, b);
                a[c] = product<2>(kf[s], b, a[c]);
                r[c] = product<2>(qf[s], b, r[c]);
            }
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = row_of(wave, 4 * g + e), j = row_of(2 * c2 + c, m);
                const float decay = exp_of((hi_i[e] - hi_j[c]) + (lo_i[e] - lo_j[c])) * norm_j[c];       // (above the diagonal whatever it is)
                lds.a[i][j] = i > j ? a[c][e] * decay * of_a[e] : 0.f;
                read[2 * c2 + c][e] = i >= j ? r[c][e] * decay * of_p[e] : 0.f;
            }
    };
    half(0);
    if (wave >= 2) half(1);
    else read[2] = read[3] = f32x4{0.f, 0.f, 0.f, 0.f};
    // What needs no more work leaves only here: stores in front of the products would hold those up.
    if (wave == 0) {
        const float gam = lds.gate[kGate][lane], rk = lds.gate[kKeyNorm][lane];
        const float beta = lds.gate[kBeta][lane];
        float4 walk;
        walk.x = beta * gam * rk;                        // kSeenBeta, kWalkBeta, kReadGate, kCarry
        walk.y = beta;
        walk.z = p.scale * gam * lds.gate[kQueryNorm][lane];
        walk.w = lds.gate[kToEnd][lane] * rk;
        *reinterpret_cast<float4 *>(&lds.gate[0][0] + 4 * lane) = walk;
        wave_lds_fence();
#pragma unroll
        for (int i = 0; i < kScalars; ++i) w.scalars[(sv * kScalars + i) * kChunk + lane] = lds.gate[i][lane];
    }
    if (first) {
        uint8_t *kd = w.kf + sh * w.kbytes() + (int64_t)wave * KS * NT * kFrag, *qd = w.qf + sh * w.kbytes() + (int64_t)wave * KS * NT * kFrag;
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                *reinterpret_cast<u32x4 *>(kd + (s * NT + n) * kFrag + lane * 16) = bitcast<u32x4>(kf[s][n]);
                if (!w.backward) *reinterpret_cast<u32x4 *>(qd + (s * NT + n) * kFrag + lane * 16) = bitcast<u32x4>(qf[s][n]);
            }
    }
    // K^T, then Q^T, gathered from the operands in LDS: token 32 s + 8 g + e is row m' of tile ct, dim_k index k is
    // element k & 7 of lane group (k >> 3) & 3 of step k >> 5.
    auto transposed = [&](uint8_t *dst) {
#pragma unroll
        for (int i = 0; i < (2 * KS + 3) / 4; ++i) {
            const int t = wave + 4 * i;
            if (t >= 2 * KS) break;
            const int k = row_of(t, m);
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    uint16_t x[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int ct = 2 * s + (e >> 2), mm = 4 * g + (e & 3);
                        x[e] = *reinterpret_cast<const uint16_t *>(lds.frags + ((ct * KS + (k >> 5)) * NT + n) * kFrag + (((k >> 3) & 3) * 16 + mm) * 16 + (k & 7) * 2);
                    }
                    u32x4 f;
                    f.x = x[0] | (uint32_t)x[1] << 16; f.y = x[2] | (uint32_t)x[3] << 16;
                    f.z = x[4] | (uint32_t)x[5] << 16; f.w = x[6] | (uint32_t)x[7] << 16;
                    *reinterpret_cast<u32x4 *>(dst + ((t * 2 + s) * NT + n) * kFrag + lane * 16) = f;
                }
        }
    };
    if (first) {
        transposed(w.ktf + sh * w.kbytes());
        if (w.backward) {
            lds_barrier();
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int n = 0; n < NT; ++n)
                    *reinterpret_cast<u32x4 *>(lds.frags + ((wave * KS + s) * NT + n) * kFrag + lane * 16) = bitcast<u32x4>(qf[s][n]);
            lds_barrier();
            transposed(w.qtf + sh * w.kbytes());
        }
    }
    lds_barrier();                                       // T goes where the operands were

    // T.  Diagonal blocks: a lane has a column of A and one of T, and reads the other columns of A from the lanes that have them.
    {
        const int o = 16 * wave;
        float a[16], x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            a[i] = lds.a[o + i][o + m];
            x[i] = i == m ? 1.f : 0.f;
        }
        below_diagonal<0>(a, x);
        if (g == 0)
#pragma unroll
            for (int i = 0; i < 16; ++i) lds.t[o + i][o + m] = x[i];
        if ((wave & 1) == 0)                             // above the diagonal, where a step of 32 columns reads it
#pragma unroll
            for (int e = 0; e < 4; ++e) lds.t[o + 4 * g + e][o + 16 + m] = 0.f;
    }
    lds_barrier();
    auto put_block = [&](int i, int j, const f32x4 &acc, float sign) {
#pragma unroll
        for (int e = 0; e < 4; ++e) lds.t[16 * i + 4 * g + e][16 * j + m] = sign * acc[e];
    };
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    if (wave < 2) {                                      // inside the halves
        const int j = 2 * wave, i = j + 1;
        put_block(i, j, block_product(&lds.a[16 * i][16 * j], kPitch, &lds.t[16 * j][16 * j], kPitch, zero, m, g), 1.f);
        wave_lds_fence();
        const f32x4 acc = block_product(&lds.t[16 * i][16 * i], kPitch, &lds.t[16 * i][16 * j], kPitch, zero, m, g);
        wave_lds_fence();
        put_block(i, j, acc, -1.f);
    }
    lds_barrier();
    {                                                    // between them, a block a wavefront
        const int i = 2 + (wave >> 1), j = wave & 1;
        f32x4 acc = zero;
        for (int k = j; k < 2; ++k) acc = block_product(&lds.a[16 * i][16 * k], kPitch, &lds.t[16 * k][16 * j], kPitch, acc, m, g);
        put_block(i, j, acc, 1.f);
        lds_barrier();
        acc = zero;
        for (int k = 2; k <= i; ++k) acc = block_product(&lds.t[16 * i][16 * k], kPitch, &lds.t[16 * k][16 * j], kPitch, acc, m, g);
        lds_barrier();
        put_block(i, j, acc, -1.f);
    }
    lds_barrier();

    // T or, for the backward, its transpose as left operands.
    if (!w.backward)
        for (int s = 0; s <= (wave >> 1); ++s) {
        float x[8];
        bf16x8 f[3];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = lds.t[row_of(wave, m)][32 * s + 8 * g + e];
        split8<3>(x, f);
#pragma unroll
        for (int n = 0; n < 3; ++n)
            *reinterpret_cast<u32x4 *>(w.tf + sv * w.tbytes() + (lower_frag(wave, s) * 3 + n) * kFrag + lane * 16) = bitcast<u32x4>(f[n]);
    }
    if (w.backward)
        for (int s = wave >> 1; s < 2; ++s) {
            float x[8];
            bf16x8 f[3];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = lds.t[32 * s + 8 * g + e][row_of(wave, m)];
            split8<3>(x, f);
#pragma unroll
            for (int n = 0; n < 3; ++n)
                *reinterpret_cast<u32x4 *>(w.ttf + sv * w.tbytes() + (upper_frag(wave, s) * 3 + n) * kFrag + lane * 16) = bitcast<u32x4>(f[n]);
        }
    // P goes where A was.
#pragma unroll
    for (int ct = 0; ct < 4; ++ct)
#pragma unroll
        for (int e = 0; e < 4; ++e) lds.a[row_of(wave, 4 * g + e)][row_of(ct, m)] = read[ct][e];
    lds_barrier();
    if (!w.backward)
        for (int s = 0; s <= (wave >> 1); ++s) {
        float x[8];
        bf16x8 f[PT];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = lds.a[row_of(wave, m)][32 * s + 8 * g + e];
        split8<PT>(x, f);
#pragma unroll
        for (int n = 0; n < PT; ++n)
            *reinterpret_cast<u32x4 *>(w.pf + sv * w.pbytes() + (lower_frag(wave, s) * PT + n) * kFrag + lane * 16) = bitcast<u32x4>(f[n]);
    }
    if (w.backward)
        for (int s = wave >> 1; s < 2; ++s) {
            float x[8];
            bf16x8 f[3];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = lds.a[32 * s + 8 * g + e][row_of(wave, m)];
            split8<3>(x, f);
#pragma unroll
            for (int n = 0; n < 3; ++n)
                *reinterpret_cast<u32x4 *>(w.ptf + sv * w.tbytes() + (upper_frag(wave, s) * 3 + n) * kFrag + lane * 16) = bitcast<u32x4>(f[n]);
        }
}

template <int DT, int KS, bool VEC>
int launch(const cc1d_delta_params &p, const ChunkWork &w, hipStream_t stream) {
    CC1D_LAUNCH((delta_prep_kernel<DT, KS, VEC>), dim3((uint32_t)((int64_t)w.slots * p.v_heads)), dim3(kBlock), sizeof(PrepLds<DT, KS>), stream, p, w);
    return launch_status();
}

}  // namespace

int launch_delta_prep(const cc1d_delta_params &p, const ChunkWork &w, hipStream_t stream) {
    const bool vec = p.dim_k % 8 == 0 && whole_rows(p.x_dtype, p.q, p.q_stride_b, p.q_stride_l, p.q_stride_h) &&
                     whole_rows(p.x_dtype, p.k, p.k_stride_b, p.k_stride_l, p.k_stride_h);
    return by_type_and_steps(p.x_dtype, w.ks, [&](auto dt, auto ks) {
        return vec ? launch<decltype(dt)::value, decltype(ks)::value, true>(p, w, stream) : launch<decltype(dt)::value, decltype(ks)::value, false>(p, w, stream);
    });
}

}  // namespace cc1d
