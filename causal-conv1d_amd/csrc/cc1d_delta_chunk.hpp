// The gated delta rule by chunks of 64 tokens: what its kernels share.
//
// With G the running sum of g inside a chunk, gam_i = exp(G_i), E_ij = exp(G_i - G_j), keys and queries of a chunk the
// rows of K and Q, S0 the state in front of it:
//
//   A = strict lower (beta_i E_ij k_i.k_j),  T = (I + A)^-1,  P = scale lower (E_ij q_i.k_j)
//   U = T diag(beta) (V - diag(gam) K S0)
//   O = scale diag(gam) Q S0 + P U,   S1 = gam_last S0 + K^T diag(gam_last / gam_j) U
//
// T and P need no state: the prep kernel makes them for all chunks at once.  What is left between one chunk and the
// next is three products, and columns of S (dim_v) do not meet, so the scan takes 16 of them to a workgroup.
//
// Products.  The matrix cores take 16-bit operands; a number x of 24 bits is the exact sum of three bfloat16
// (each the rest, rounded), so a product of two such is nine exact products, of which the six largest carry it to
// 2^-25, for numbers from 2^-90 on (the terms of smaller ones fall below the normal numbers; 2^-100 is off by 1e-8 still).  bfloat16 q, k, v, dout are one
// term each and cost nothing, float16 is two.
// Six products on the 16-bit cores take 0.38 of the time of the fp32 ones; one and three together a third of that.
//
// Operand order.  An MFMA of 16 x 16 x 32 wants of its left operand 8 consecutive columns of one row a lane, of its right one 8
// consecutive rows of one column, and leaves 4 rows of one column.  Which row of a matrix a tile's row is, is free as long
// as both sides agree: rows are dealt so that the 4 + 4 rows of two result tiles are 8 consecutive ones (row_of),
// and a result becomes the next product's right operand without leaving its lane.
#pragma once

#include "cc1d_delta.hpp"

namespace cc1d {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// The row of a matrix that row m of 16-row tile t is.
__device__ __host__ __forceinline__ constexpr int row_of(int t, int m) { return 32 * (t >> 1) + 8 * (m >> 2) + 4 * (t & 1) + (m & 3); }

// Terms of q, k, v, dout; of P, U and S where they make outputs of 16 bits.
template <int DT> struct Terms { static constexpr int n = DT == CC1D_BF16 ? 1 : DT == CC1D_F16 ? 2 : 3, p = DT == CC1D_F32 ? 3 : 2; };

// Scalars of a chunk's tokens per (chunk, value head): what the walks need of a token, four numbers side by side, then one
// vector of 64 each of what the gradients need.
enum { kSeenBeta, kWalkBeta, kReadGate, kCarry };        // of token i at 4 i + these
//     beta gam rk   beta       scale gam rq  dec rk
enum { kBeta = 4, kKeyNorm, kQueryNorm, kGate, kToEnd, kSumHi, kSumLo, kScalars };
//     beta       rk        rq          gam    dec     G = hi + lo

// Wavefronts a SIMD in the scans: two, or one with all registers where a chunk's operands do not fit in half of them.
constexpr int scan_waves(int dt, int ks) { return ks * (dt == CC1D_BF16 ? 1 : dt == CC1D_F16 ? 2 : 3) <= 8 && ks <= 4 ? 2 : 1; }

constexpr int kFrag = 1024;              // bytes of one operand of 16 x 32 bfloat16
constexpr int kTriFrags = 6;             // of a triangular 64 x 64 matrix: 2 tiles x 1 step + 2 tiles x 2 steps
__device__ __host__ __forceinline__ constexpr int lower_frag(int t, int s) { return t < 2 ? t : 2 + 2 * (t - 2) + s; }
__device__ __host__ __forceinline__ constexpr int upper_frag(int t, int s) { return t < 2 ? 2 * t + s : 4 + (t - 2); }

// Where everything lies in the workspace.  "slot": one chunk of one sequence; without cu_seqlens n ceil(seqlen / 64) + c, with
// it floor(first token / 64) + n + c, which no two chunks share.  Where only sequences of `shortest` tokens go by chunks, 64 at least, each holds
// a token whose number is a multiple of 64, and is named by the first of them, 64 f: slots 2 f + c, at most twice as many as it holds such
// tokens; workgroups are counted by tokens then, however many sequences there are.
struct ChunkWork {
    uint8_t *kf, *qf, *ktf, *qtf;        // per (slot, head): K, Q rows x dim_k; K^T, Q^T dim_k x rows
    uint8_t *tf, *pf, *ttf, *ptf;        // per (slot, value head): T, P lower; T^T, P^T upper
    float *scalars;                      // per (slot, value head): [kScalars][64]
    float *s0, *ds1;                     // per (slot, value head): (dim_k, dim_v)
    float *u, *dx;                       // per (slot, value head): (64, dim_v)
    float *dqk;                          // per (slot, value head) of shared keys: its share of dq and dk, 64 x 32 ks each, in the lanes' order
    int32_t slots, chunks;               // chunks: of one sequence without cu_seqlens; of all tokens
    int32_t ks, terms, pterms;           // 32-column steps of dim_k; terms of K and Q; of P
    int32_t backward;
    int32_t shortest;                    // packed sequences of fewer tokens are the token kernel's; 0: none
    FastDiv by_heads, by_v_heads, by_group, by_chunks;    // group: value heads of a key head
    // What the scan has workgroups for: the sequences, or the tokens that may name one.
    int64_t walks(const cc1d_delta_params &p) const { return shortest > 0 ? chunks : p.sequences; }
    __device__ __host__ int64_t kbytes() const { return (int64_t)4 * ks * terms * kFrag; }
    __device__ __host__ int64_t tbytes() const { return (int64_t)kTriFrags * 3 * kFrag; }
    __device__ __host__ int64_t pbytes() const { return (int64_t)kTriFrags * pterms * kFrag; }
};

// The last sequence whose place is not behind `target`; sequence 0's is not.  64 candidates at once, one a lane (the whole wavefront is here):
// one load's wait up to 64 sequences, two up to 4096.
template <typename F>
__device__ __forceinline__ int last_sequence(const cc1d_delta_params &p, int64_t target, F &&place) {
    int a = 0, b = p.sequences;
    while (b - a > 1) {
        const int step = (b - a + 63) >> 6, mine = a + (int)(threadIdx.x & 63) * step, i = mine < b ? mine : b - 1;
        const int64_t at = place(cu_entry(p.cu_seqlens, p.cu_seqlens_is_int64, i, p.seqlen), i);
        const int n = __popcll(__ballot(mine < b && (mine == a || at <= target)));
        a += (n - 1) * step;
        b = a + step < b ? a + step : b;
    }
    return a;
}
// The sequence that holds token `at`, if one does.
__device__ __forceinline__ int sequence_of(const cc1d_delta_params &p, int64_t at) {
    return last_sequence(p, at, [](int64_t first, int) { return first; });
}
// Whether a sequence goes by chunks and is named by token 64 f.
__device__ __forceinline__ bool named(const TokenRange &r, const ChunkWork &w, int64_t f) {
    return r.hi - r.lo >= w.shortest && (r.lo + kChunk - 1) / kChunk == f;
}

// Which chunk a slot is: tokens [lo, lo + count) of batch entry b, sequence n, or count = 0 if it is none.
struct ChunkAt { int64_t lo; int count, b, n; };
__device__ __forceinline__ ChunkAt chunk_at(const cc1d_delta_params &p, const ChunkWork &w, int slot) {
    if (p.cu_seqlens == nullptr) {
        const int n = (int)divided((uint32_t)slot, w.by_chunks), c = slot - n * w.chunks;
        const int64_t lo = (int64_t)c * kChunk, left = p.seqlen - lo;
        return {lo, (int)(left < kChunk ? left : kChunk), n, n};
    }
    if (w.shortest > 0) {
        const int n = sequence_of(p, (int64_t)(slot >> 1) * kChunk);
        const TokenRange r = sequence_tokens(p, n);
        const int64_t f = (r.lo + kChunk - 1) / kChunk, lo = r.lo + (slot - 2 * f) * kChunk, left = r.hi - lo;
        if (!named(r, w, f) || lo < r.lo || left <= 0) return {0, 0, 0, n};
        return {lo, (int)(left < kChunk ? left : kChunk), 0, n};
    }
    // The last sequence whose first slot is not behind this one; sequence 0 begins at slot floor(cu[0] / 64).
    const int a = last_sequence(p, slot, [](int64_t first, int i) { return first / kChunk + i; });
    const TokenRange r = sequence_tokens(p, a);
    const int64_t lo = r.lo + ((int64_t)slot - (r.lo / kChunk + a)) * kChunk, left = r.hi - lo;
    if (lo < r.lo || left <= 0) return {0, 0, 0, a};
    return {lo, (int)(left < kChunk ? left : kChunk), 0, a};
}
__device__ __forceinline__ int first_slot(const cc1d_delta_params &p, const ChunkWork &w, int n, const TokenRange &r) {
    if (p.cu_seqlens == nullptr) return n * w.chunks;
    return w.shortest > 0 ? 2 * (int)((r.lo + kChunk - 1) / kChunk) : (int)(r.lo / kChunk) + n;
}

// N bfloat16 terms of 4 (8) numbers, term i in two (four) words, each the rest rounded to nearest: two leave 2^-18 of a
// number, three nothing.  What a term leaves, x - hi, is one instruction, a dot product of the pair that hi stands in with
// (-1, 0) or (0, -1) added to x; it is exact.  The pairs are kept in scalar registers: as immediates the compiler puts them into
// the wrong half.
__device__ __forceinline__ uint32_t rounded_pair(float lo, float hi) {
    bf16x2 h;
    h.x = (__bf16)lo;
    h.y = (__bf16)hi;
    return bitcast<uint32_t>(h);
}
template <int N>
__device__ __forceinline__ void split4(const float (&x)[4], u32x2 (&t)[N]) {
    uint32_t low = 0x0000bf80u, high = 0xbf800000u;
    asm("" : "+s"(low), "+s"(high));
    float r[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
    for (int n = 0; n < N; ++n) {
        t[n].x = rounded_pair(r[0], r[1]);
        t[n].y = rounded_pair(r[2], r[3]);
        if (n + 1 < N) {
            r[0] = __builtin_amdgcn_fdot2_f32_bf16(bitcast<bf16x2>((uint32_t)t[n].x), bitcast<bf16x2>(low), r[0], false);
            r[1] = __builtin_amdgcn_fdot2_f32_bf16(bitcast<bf16x2>((uint32_t)t[n].x), bitcast<bf16x2>(high), r[1], false);
            r[2] = __builtin_amdgcn_fdot2_f32_bf16(bitcast<bf16x2>((uint32_t)t[n].y), bitcast<bf16x2>(low), r[2], false);
            r[3] = __builtin_amdgcn_fdot2_f32_bf16(bitcast<bf16x2>((uint32_t)t[n].y), bitcast<bf16x2>(high), r[3], false);
        }
    }
}
template <int N>
__device__ __forceinline__ void split8(const float (&x)[8], bf16x8 (&t)[N]) {
    const float lo[4] = {x[0], x[1], x[2], x[3]}, hi[4] = {x[4], x[5], x[6], x[7]};
    u32x2 a[N], b[N];
    split4<N>(lo, a);
    split4<N>(hi, b);
#pragma unroll
    for (int n = 0; n < N; ++n) {
        u32x4 w; w.x = a[n].x; w.y = a[n].y; w.z = b[n].x; w.w = b[n].y;
        t[n] = bitcast<bf16x8>(w);
    }
}

// acc += sum of a[i] b[j] with i + j <= MOST, the small ones first.
template <int MOST, int NA, int NB>
__device__ __forceinline__ f32x4 product(const bf16x8 (&a)[NA], const bf16x8 (&b)[NB], f32x4 acc) {
#pragma unroll
    for (int sum = MOST; sum >= 0; --sum)
#pragma unroll
        for (int i = 0; i < NA; ++i) {
            const int j = sum - i;
            if (j >= 0 && j < NB) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[j], acc, 0, 0, 0);
        }
    return acc;
}

// 8 elements of a row from column c on, `cols` columns long (none: a row that is not there), asked for without a branch and looked
// at later: a load behind a condition waits for itself, and with it for everything asked for before it.  VEC: cols is a multiple of 8
// and the row 16-byte aligned.
template <int DT, bool VEC>
struct Row8 {
    static constexpr int N = DT == CC1D_F32 ? 2 : 1;
    u32x4 r[N];
    __device__ __forceinline__ void ask(const typename Elem<DT>::type *row, int c, int cols) {
        if constexpr (VEC) {
            const u32x4 *at = reinterpret_cast<const u32x4 *>(row + (c < cols ? c : 0));
#pragma unroll
            for (int i = 0; i < N; ++i) r[i] = at[i];
        } else {
            uint32_t x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int j = c + i < cols ? c + i : 0;
                if constexpr (DT == CC1D_F32) x[i] = reinterpret_cast<const uint32_t *>(row)[j];
                else x[i] = reinterpret_cast<const uint16_t *>(row)[j];
            }
            if constexpr (DT == CC1D_F32) {
                r[0].x = x[0]; r[0].y = x[1]; r[0].z = x[2]; r[0].w = x[3];
                r[N - 1].x = x[4]; r[N - 1].y = x[5]; r[N - 1].z = x[6]; r[N - 1].w = x[7];
            } else {
                r[0].x = x[0] | x[1] << 16; r[0].y = x[2] | x[3] << 16; r[0].z = x[4] | x[5] << 16; r[0].w = x[6] | x[7] << 16;
            }
        }
    }
    // `cut`: some lane's elements are not all inside.
    __device__ __forceinline__ void get(int c, int cols, bool cut, float (&f)[8]) const {
        if constexpr (DT == CC1D_F32) {
            float lo[4], hi[4];
            Elem<DT>::unpack(r[0], lo);
            Elem<DT>::unpack(r[N - 1], hi);
#pragma unroll
            for (int i = 0; i < 4; ++i) { f[i] = lo[i]; f[i + 4] = hi[i]; }
        } else {
            Elem<DT>::unpack(r[0], f);
        }
        if (cut)
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = (VEC ? c : c + i) < cols ? f[i] : 0.f;
    }
    // As an operand of TERMS terms; bfloat16 is one as it stands.
    template <int TERMS>
    __device__ __forceinline__ void operand(int c, int cols, bool cut, bf16x8 (&t)[TERMS]) const {
        if constexpr (DT == CC1D_BF16 && VEC) {
            u32x4 w = r[0];
            if (cut && c >= cols) { w.x = 0; w.y = 0; w.z = 0; w.w = 0; }
            t[0] = bitcast<bf16x8>(w);
        } else {
            float f[8];
            get(c, cols, cut, f);
            split8<TERMS>(f, t);
        }
    }
};

// One of a token's four numbers, for the four tokens of a lane group's rows: lane b of a quad has loaded token b's.
__device__ __forceinline__ void of_quad(float x, float (&f)[4]) {
    f[0] = dpp_moved<0x00>(x);
    f[1] = dpp_moved<0x55>(x);
    f[2] = dpp_moved<0xAA>(x);
    f[3] = dpp_moved<0xFF>(x);
}

// 4 elements of a row in the same manner.
template <int DT, bool VEC>
struct Row4 {
    using T = typename Elem<DT>::type;
    using Bits = typename BitsOf<DT>::type;
    struct alignas(4 * sizeof(Bits)) Four { Bits x[4]; } r;
    __device__ __forceinline__ void ask(const T *row, int c, int cols) {
        const Bits *from = reinterpret_cast<const Bits *>(row);
        if constexpr (VEC) {
            r = *reinterpret_cast<const Four *>(from + (c < cols ? c : 0));
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) r.x[i] = from[c + i < cols ? c + i : 0];
        }
    }
    __device__ __forceinline__ void get(int c, int cols, bool cut, float (&f)[4]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = Elem<DT>::to_float(bitcast<T>(r.x[i]));
        if (cut)
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = (VEC ? c : c + i) < cols ? f[i] : 0.f;
    }
};

template <int N>
__device__ __forceinline__ void load_frag(const uint8_t *base, int lane, bf16x8 (&f)[N]) {
#pragma unroll
    for (int n = 0; n < N; ++n) f[n] = bitcast<bf16x8>(*reinterpret_cast<const u32x4 *>(base + n * kFrag + lane * 16));
}

// Two accumulators, the largest products in one and the rest in the other: two chains of instructions that do not wait for each other.
template <int MOST, int NA, int NB>
__device__ __forceinline__ void product2(const bf16x8 (&a)[NA], const bf16x8 (&b)[NB], f32x4 &large, f32x4 &rest) {
#pragma unroll
    for (int sum = MOST; sum >= 0; --sum)
#pragma unroll
        for (int i = 0; i < NA; ++i) {
            const int j = sum - i;
            if (j < 0 || j >= NB) continue;
            if (sum == 0) large = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[j], large, 0, 0, 0);
            else rest = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[j], rest, 0, 0, 0);
        }
}

// The numbers that elements 0..3 (or, `upper`, 4..7) of an operand's lane stand for.
template <int N>
__device__ __forceinline__ void four_of(const bf16x8 (&t)[N], bool upper, float (&f)[4]) {
#pragma unroll
    for (int n = N - 1; n >= 0; --n) {
        const u32x4 w = bitcast<u32x4>(t[n]);
        const uint32_t a = upper ? w.z : w.x, b = upper ? w.w : w.y;
        const float x[4] = {bitcast<float>(a << 16), bitcast<float>(a & 0xffff0000u), bitcast<float>(b << 16), bitcast<float>(b & 0xffff0000u)};
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = n == N - 1 ? x[i] : f[i] + x[i];
    }
}

}  // namespace cc1d
