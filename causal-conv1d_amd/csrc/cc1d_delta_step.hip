// The gated delta rule token by token: the step of a decode loop, and whole sequences that are too short
// to be worth cutting into chunks.
//
//   D = exp(g) S,  u = beta (v - D^T k),  S = D + k u^T,  out = scale S^T q
//
// The columns of S (dim_v) do not meet: a wavefront takes 32 of them, all of dim_k, in registers.  A lane holds
// 4 adjacent columns of KR rows (8 lanes make a row's 128 bytes, 8 groups of lanes take KR rows each), so every
// row of the state moves as whole 128-byte lines.  q and k go through LDS once, normalised, in fp32.  Both
// products of a token are formed before its update, out = D^T q + (k.q) u, so that one reduction over the
// lane groups serves both.  In a decode step nothing is computed worth mentioning: the state, read and written
// once, is the floor.  It is read and written past the caches (nothing reads it before the next step): 96 states of
// 32 heads of 128 x 128 take 73 us, 5.5 TB/s, and 100 through the caches; one request 7.5 us and 10, since no line is
// left to be written back when the kernel ends.  Four wavefronts to a workgroup: 73 us, one 83.
#include "cc1d_delta.hpp"
#include "cc1d_delta_host.hpp"

namespace cc1d {
namespace {

constexpr int kStepCols = 32;

struct StepArgs {
    cc1d_delta_params p;                 // initial_states / final_states: the state, or the caller's two
    const int32_t *indices;
    int32_t slots;
    int32_t longest;                     // sequences of this many tokens go by chunks; 0: none
    uint32_t items, col_tiles;
    uint32_t vec_state, vec_x;           // 16-byte rows of the state / 4 elements of v and out at once
};

// KR: rows of the state a lane holds, dim_k <= 8 KR.
template <int DT, int KR>
__global__ void __launch_bounds__(kBlock)
delta_step_kernel(const StepArgs a) {
    using T = typename Elem<DT>::type;
    using Bits = typename BitsOf<DT>::type;
    struct alignas(4 * sizeof(Bits)) Four { Bits x[4]; };
    __shared__ float lds[4][2][8 * KR + 8];
    const cc1d_delta_params &p = a.p;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t item = blockIdx.x * 4u + (uint32_t)wave;
    if (item >= a.items) return;                         // no barrier below: wavefronts work alone
    const int tile = (int)(item % a.col_tiles);
    const uint32_t nh = item / a.col_tiles;
    const int h = (int)(nh % (uint32_t)p.v_heads), n = (int)(nh / (uint32_t)p.v_heads);
    const int hk = h / (p.v_heads / p.heads);
    const int cg = lane & 7, rg = lane >> 3;
    const int c0 = tile * kStepCols + 4 * cg;
    const int cols = p.dim_v - c0;                       // of this lane's four
    const TokenRange range = sequence_tokens(p, n);

    if (p.cu_seqlens != nullptr && rg == 0) {            // tokens in front of the first sequence and behind the last
        auto clear = [&](int64_t lo, int64_t hi) {
            for (int64_t t = lo; t < hi; ++t)
                for (int i = 0; i < 4 && i < cols; ++i)
                    static_cast<T *>(p.out)[t * p.out_stride_l + h * p.out_stride_h + c0 + i] = Elem<DT>::from_float(0.f);
        };
        if (n == 0) clear(0, range.lo);
        if (n == p.sequences - 1) clear(range.hi, p.seqlen);
    }

    if (a.longest > 0 && range.hi - range.lo >= a.longest) return;

    int64_t slot = n;
    if (a.indices != nullptr) slot = a.indices[n];
    if (slot < 0 || slot >= a.slots) {                   // padding: zeros, no state touched
        if (rg == 0)
            for (int64_t t = range.lo; t < range.hi; ++t)
                for (int i = 0; i < 4 && i < cols; ++i)
                    static_cast<T *>(p.out)[range.b * p.out_stride_b + t * p.out_stride_l + h * p.out_stride_h + c0 + i] = Elem<DT>::from_float(0.f);
        return;
    }

    // Every load is made without a condition, of a place inside the tensor where the lane's own lies outside: a load behind
    // a branch is waited for before the next.  The token's own loads go out in front of the state's, and are summed while
    // those travel; the next token's in front of a token's products.
    constexpr int NE = (8 * KR + 63) / 64;               // elements of k and q a lane fetches
    const int cc = cols > 0 ? c0 : 0;                    // lanes behind the last column repeat the first, and store nothing
    struct Token { Bits k[NE], q[NE], v[4]; uint32_t g, beta; };
    const Bits *qp = static_cast<const Bits *>(p.q) + range.b * p.q_stride_b + range.lo * p.q_stride_l + hk * p.q_stride_h;
    const Bits *kp = static_cast<const Bits *>(p.k) + range.b * p.k_stride_b + range.lo * p.k_stride_l + hk * p.k_stride_h;
    const Bits *vp = static_cast<const Bits *>(p.v) + range.b * p.v_stride_b + range.lo * p.v_stride_l + h * p.v_stride_h + cc;
    int64_t at_g = range.b * p.g_stride_b + range.lo * p.g_stride_l + h * p.g_stride_h;
    int64_t at_beta = range.b * p.beta_stride_b + range.lo * p.beta_stride_l + h * p.beta_stride_h;
    auto ask = [&]() {                                   // the token after the one asked for last
        Token x;
#pragma unroll
        for (int e = 0; e < NE; ++e) {
            const int i = lane + 64 * e < p.dim_k ? lane + 64 * e : 0;
            x.k[e] = kp[i];
            x.q[e] = qp[i];
        }
        x.g = load_bits(p.g, at_g, p.g_dtype);
        x.beta = load_bits(p.beta, at_beta, p.beta_dtype);
        if (a.vec_x) {
            *reinterpret_cast<Four *>(x.v) = *reinterpret_cast<const Four *>(vp);
        } else {                                         // (lanes behind the last column: the first)
#pragma unroll
            for (int j = 0; j < 4; ++j) x.v[j] = vp[j < cols ? j : 0];
        }
        qp += p.q_stride_l; kp += p.k_stride_l; vp += p.v_stride_l; at_g += p.g_stride_l; at_beta += p.beta_stride_l;
        return x;
    };
    Token next = {};
    if (range.lo < range.hi) next = ask();
    stay();

    float s[KR][4];
    const float *src = p.initial_states == nullptr ? nullptr : p.initial_states + slot * p.init_stride_n + h * p.init_stride_h;
    if (src != nullptr) {
#pragma unroll
        for (int i = 0; i < KR; ++i) {
            const int row = rg * KR + i;
            const float *x = src + (row < p.dim_k ? row : 0) * p.init_stride_k + cc;
            if (a.vec_state) {
                const u32x4 r = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(x));
                Elem<CC1D_F32>::unpack(r, s[i]);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) s[i][j] = x[j < cols ? j : 0];
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < KR; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
    }
    stay();

    float *kq = &lds[wave][0][0], *qq = &lds[wave][1][0];
    for (int64_t t = range.lo; t < range.hi; ++t) {
        float ke[NE], qe[NE], kk = 0.f, qs = 0.f, dot = 0.f;
#pragma unroll
        for (int e = 0; e < NE; ++e) {
            const bool there = lane + 64 * e < p.dim_k;
            ke[e] = there ? Elem<DT>::to_float(bitcast<T>(next.k[e])) : 0.f;
            qe[e] = there ? Elem<DT>::to_float(bitcast<T>(next.q[e])) : 0.f;
            kk += ke[e] * ke[e]; qs += qe[e] * qe[e]; dot += ke[e] * qe[e];
        }
        const float decay = exp_of(bits_as_float(next.g, p.g_dtype)), beta = bits_as_float(next.beta, p.beta_dtype);
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = Elem<DT>::to_float(bitcast<T>(next.v[j]));
        if (t + 1 < range.hi) next = ask();
        float rk = 1.f, rq = p.scale;
        auto lengths = [&]() {
            dot = over_wave(dot);
            if (!p.qk_l2norm) return;
            rk = rsqrtf(over_wave(kk) + kNormEps);
            rq = p.scale * rsqrtf(over_wave(qs) + kNormEps);
        };
        if (KR == 32) lengths();                         // (behind the sums below it would take a register too many for two wavefronts a SIMD)
        wave_lds_fence();                                // the token before has been read
#pragma unroll
        for (int e = 0; e < NE; ++e) {
            const int i = lane + 64 * e;
            if (i < 8 * KR) { kq[i] = ke[e]; qq[i] = qe[e]; }
        }
        wave_lds_fence();
        // Sums with the state as it is, the decay and the lengths' factors on the sums: nothing waits for those.  Rows behind the
        // last, which hold what the first does, meet zeros.
        float sk[4] = {0.f, 0.f, 0.f, 0.f}, sq[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < KR; ++i) {
            const float ki = kq[rg * KR + i], qi = qq[rg * KR + i];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                sk[j] += s[i][j] * ki;
                sq[j] += s[i][j] * qi;
            }
        }
        if (KR < 32) lengths();
        float u[4], o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            sk[j] = over_rows(sk[j] + dpp_moved<0x128>(sk[j]));      // the lanes of a column are 8 apart
            sq[j] = over_rows(sq[j] + dpp_moved<0x128>(sq[j]));
            u[j] = beta * (v[j] - decay * rk * sk[j]) * rk;          // of k as it came
            o[j] = rq * (decay * sq[j] + dot * u[j]);
        }
#pragma unroll
        for (int i = 0; i < KR; ++i) {
            const float ki = kq[rg * KR + i];
#pragma unroll
            for (int j = 0; j < 4; ++j) s[i][j] = s[i][j] * decay + ki * u[j];
        }
        if (rg == 0) {
            T *op = static_cast<T *>(p.out) + range.b * p.out_stride_b + t * p.out_stride_l + h * p.out_stride_h + c0;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j < cols) op[j] = Elem<DT>::from_float(o[j]);
        }
    }

    if (p.final_states == nullptr) return;
    float *dst = p.final_states + slot * p.final_stride_n + h * p.final_stride_h;
#pragma unroll
    for (int i = 0; i < KR; ++i) {
        const int row = rg * KR + i;
        if (row >= p.dim_k || cols <= 0) continue;
        float *d = dst + row * p.final_stride_k + c0;
        if (a.vec_state) {
            const u32x4 r = Elem<CC1D_F32>::pack(s[i]);
            __builtin_nontemporal_store(r, reinterpret_cast<u32x4 *>(d));
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j < cols) d[j] = s[i][j];
        }
    }
}

template <int DT, int KR>
int launch_rows(const StepArgs &a, hipStream_t stream) {
    CC1D_LAUNCH((delta_step_kernel<DT, KR>), dim3((a.items + 3) / 4), dim3(kBlock), 0, stream, a);
    return launch_status();
}
template <int DT>
int launch_dtype(const StepArgs &a, hipStream_t stream) {
    return a.p.dim_k <= 64 ? launch_rows<DT, 8>(a, stream) : a.p.dim_k <= 128 ? launch_rows<DT, 16>(a, stream) : launch_rows<DT, 32>(a, stream);
}

}  // namespace


int launch_delta_tokens(const cc1d_delta_params &p, const int32_t *indices, int slots, int longest, hipStream_t stream) {
    StepArgs a = {};
    a.p = p;
    a.indices = indices;
    a.slots = slots;
    a.longest = longest;
    a.col_tiles = (uint32_t)((p.dim_v + kStepCols - 1) / kStepCols);
    const int64_t items = (int64_t)p.sequences * p.v_heads * a.col_tiles;
    if (items == 0) return CC1D_OK;
    if (items * 64 >= thread_limit()) return CC1D_ERR_TOO_LARGE;
    a.items = (uint32_t)items;
    auto whole = [&](const void *s, int64_t sn, int64_t sh, int64_t sk) {
        return s == nullptr || (aligned16(s) && sn % 4 == 0 && sh % 4 == 0 && sk % 4 == 0);
    };
    a.vec_state = p.dim_v % 4 == 0 && whole(p.initial_states, p.init_stride_n, p.init_stride_h, p.init_stride_k) &&
                  whole(p.final_states, p.final_stride_n, p.final_stride_h, p.final_stride_k);
    a.vec_x = p.dim_v % 4 == 0 && p.v_stride_b % 4 == 0 && p.v_stride_l % 4 == 0 && p.v_stride_h % 4 == 0 &&
              (reinterpret_cast<uintptr_t>(p.v) & (4u * (uint32_t)elem_bytes(p.x_dtype) - 1u)) == 0;
    switch (p.x_dtype) {
        case CC1D_F32: return launch_dtype<CC1D_F32>(a, stream);
        case CC1D_F16: return launch_dtype<CC1D_F16>(a, stream);
        default: return launch_dtype<CC1D_BF16>(a, stream);
    }
}

}  // namespace cc1d
