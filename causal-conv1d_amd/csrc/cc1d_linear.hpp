// Linear attention with a decay for each head: what its kernels and its host side share.
//
//   S = exp(g[t]) S + beta[t] k[t] v[t]^T,   out[t] = scale S^T q[t]
//
// Sequences are cut into segments of kSegment tokens, segments into blocks of 64.  With G the running sum of g inside a segment,
// E_ij = exp(G_i - G_j), S0 the state in front of a segment and dS1 the gradient of the one behind it:
//
//   out_i = scale (exp(G_i) q_i S0 + sum over j <= i of E_ij (q_i.k_j) beta_j v_j)
//   dq_i  = scale (exp(G_i) dout_i S0^T + sum over j <= i of E_ij (dout_i.v_j) beta_j k_j)
//   dk_j  = beta_j (exp(Gend - G_j) v_j dS1^T + sum over i >= j of E_ij (v_j.dout_i) scale q_i)
//   dv_j  = beta_j (exp(Gend - G_j) k_j dS1 + sum over i >= j of E_ij (k_j.q_i) scale dout_i)
//
// These four are one kernel (linear_attend_kernel) on tensors x, y, z and a state: rows x_i of one block times the state, and products
// x_i.y_j, weighted, times z_j over the blocks in front (REV: behind).  No state is carried inside a segment, so every block of every segment
// is a workgroup of its own; what crosses segments is
//
//   S1 = exp(Gend) S0 + sum of exp(Gend - G_j) beta_j k_j v_j^T,   dS0 = exp(Gend) dS1 + sum of exp(G_i) scale q_i dout_i^T
//
// whose sums are one more kernel (linear_states_kernel), and whose recurrence over segments is elementwise (linear_scan_kernel).  The gates'
// gradients come out of sums that are there: dg at a segment's first token is S0 . dS0 over all elements (nothing else reads that gate's product), and
// dg[t + 1] = dg[t] - (q[t].dq[t] - k[t].dk[t]).  What a token reads of itself, scale beta_t (dout_t.v_t) (q_t.k_t), is in both products and is left out of both:
// where gates are strong it is nearly all of them, and nothing of dg (gates of -5, 320 tokens, heads of 128 x 64, bfloat16: dg off by 1.2e-6 of itself, with it 1.7e-4).
// What remains still cancels: S0 . dS0 is some 2^-11 of the norms' product, and what a segment's differences are off by adds
// up over its tokens.  So the sums are made in 64 bits (linear_tile_kernel: 32 for the four or eight products inside a lane), of dq and dk before they are rounded, and what the last token leaves over against the next segment's
// S0 . dS0 (or 0, behind the last one) is taken back in proportion to the sizes of the products in front: where the errors arise, and not among
// the small gradients in front of large ones (16 heads with a constant decay each, 2 x 1000 tokens, the sum of dg over the tokens, six seeds: off by
// 3e-8 to 5e-7 of itself, the plain form by 1e-7 to 6e-7; with sums of 32 bits, without that and without linear_states_kernel's alternating signs 7e-7 to 3e-6).
//
// Numbers of 24 bits on the 16-bit matrix cores: cc1d_delta_chunk.hpp.
#pragma once

#include "cc1d_delta_chunk.hpp"

namespace cc1d {

constexpr int kSegmentLog = 8, kSegment = 1 << kSegmentLog, kBlocks = kSegment / kChunk;

// A (batch, seqlen, heads, dim) tensor; by_key: its heads are the key heads.
struct LinearRows { const void *p; int64_t sb, sl, sh; int32_t by_key; };

// Terms of the states and weighted products where they make outputs of x_dtype alone; where they make the gates' gradients too, which are fp32 and
// small differences of large sums, three.  Two carry 2^-17 beside the 2^-8 or 2^-11 that out and dv are rounded to: against 64 bits both are off by 1.7e-3 (bfloat16) or
// 2.1e-4 (float16) of themselves with two as with three, and by 2e-5 to 1e-4 from what 32 bits all the way would have rounded to, with three by 1e-5 to 3.5e-5.  Three
// cost a prompt of 4 x 2048 tokens, 80 heads of 128 x 64, 224 us for 184, its training step 929 for 873.
constexpr int out_terms(int dt) { return dt == CC1D_F32 ? 3 : 2; }

// W of a state's operands, by sizes and type alone (what a forward saves has to be what its backward reads, whatever the layouts): those of
// linear_tile_kernel where it may take the product of `d1` by `d2` columns.
inline int operand_width(int dtype, int d1, int d2, bool gradient_of_keys) {
    const bool tile = dtype != CC1D_F32 && d1 <= 128 && (!gradient_of_keys || d2 <= 128);
    return !tile ? 2 : d2 <= 64 ? 4 : 8;
}
inline int operand_tiles(int width, int d2) { return (d2 + 16 * width - 1) / (16 * width) * width; }

// States lie by borders between a sequence's segments (border_behind), of which packed sequences of a few tokens have none; where a state in front of the
// first segment or behind the last is there too, by slots.
struct SegmentWork {
    int32_t slots, chunks;               // segments of the call; of one sequence without cu_seqlens
    int64_t borders;
    int32_t kp, vp;                      // 32-column steps of dim_k, dim_v
    FastDiv by_v_heads, by_chunks, by_group;
    float *local;                        // per (state, value head): a segment's own sum, [kp][vp] tiles of 32 x 32 in operand order
    float *decay;                        // per (slot, value head): exp(Gend)
    uint8_t *by_k, *by_v;                // per (state, value head): states split into operands, contracted over dim_k and over dim_v
    uint8_t *first;                      // S0 of the forward, contracted over dim_v: what a training forward saves
    double *dot_q, *dot_k;               // (batch, v_heads, seqlen): q.dq and k.(dk / beta) of each token, without its own share
    float *self_k, *qk;                  // that share of k.(dk / beta) is self_k qk: scale dout.v; (batch, heads, seqlen): q.k
    double *inner;                       // per (state, value head): S0 . dS0, a partial sum each tile
    float *share_q, *share_k;            // shares of dq, dk of heads_each value heads: (shares, batch, seqlen, heads, dim_k)
    int32_t k_width, v_width, k_tiles, v_tiles;                // of operands contracted over dim_k (out, dv), over dim_v (dq, dk)
    int32_t heads_each, shares;          // value heads of a workgroup of the gradients of q and k; such workgroups a key head
    int32_t shortest;                    // packed sequences of fewer tokens, kSegment at least, are the token kernel's; 0: none
    __host__ int64_t walks(const cc1d_delta_params &p) const { return shortest > 0 ? chunks : p.sequences; }
    __device__ __host__ int64_t tiles() const { return (int64_t)kp * vp; }
};

// Rows that are not whole 16-byte vectors (odd sizes, odd strides or addresses) are copied to rows that are, zeros behind their columns, and results
// from there: the kernels know no others.  16 heads of 100 x 100, 4 x 2048 tokens, bfloat16: 145 us forward and 358 backward, with kernels that read them element by
// element 254 and 1034; 56 heads of 154 x 80, 7 x 239 tokens: 530 us for 1510.
constexpr int kVector = 8;
__host__ __device__ inline int padded(int dim) { return (dim + kVector - 1) / kVector * kVector; }
struct CopyRows {
    const uint8_t *from; uint8_t *to;
    int64_t from_b, from_l, from_h, to_b, to_l, to_h;          // bytes
    int32_t heads, dim;                  // columns that are there
    FastDiv by_vectors;                  // vectors of a padded row
};
constexpr int kMostCopies = 4;
struct CopyArgs { CopyRows of[kMostCopies]; int32_t elem, batch, seqlen; FastDiv by_seqlen; };

__device__ __forceinline__ int64_t naming(const TokenRange &r) { return (r.lo + kSegment - 1) >> kSegmentLog; }
// Tokens [lo, lo + count) of batch entry b: segment c of sequence n, or count = 0 if a slot is none.
struct SegmentAt { int64_t lo; int count, b, n, c; bool last; };
__device__ __forceinline__ SegmentAt segment_at(const cc1d_delta_params &p, const SegmentWork &w, int slot) {
    if (p.cu_seqlens == nullptr) {
        const int n = (int)divided((uint32_t)slot, w.by_chunks), c = slot - n * w.chunks;
        const int64_t lo = (int64_t)c << kSegmentLog, left = p.seqlen - lo;
        return {lo, (int)(left < kSegment ? left : kSegment), n, n, c, left <= kSegment};
    }
    // As chunks of the gated delta rule.  Where only long sequences go by segments, each holds a token 256 f; with f of the first of these, its
    // segment c is slot 2 f + c, which no two share.
    if (w.shortest > 0) {
        const int n = sequence_of(p, (int64_t)(slot >> 1) << kSegmentLog);
        const TokenRange r = sequence_tokens(p, n);
        const int64_t f = naming(r), c = slot - 2 * f, lo = r.lo + (c << kSegmentLog), left = r.hi - lo;
        if (r.hi - r.lo < w.shortest || c < 0 || left <= 0) return {0, 0, 0, n, 0, false};
        return {lo, (int)(left < kSegment ? left : kSegment), 0, n, (int)c, left <= kSegment};
    }
    // Else sequence n begins at slot floor(first token / kSegment) + n, and no two share one.
    const int n = last_sequence(p, slot, [](int64_t first, int i) { return (first >> kSegmentLog) + i; });
    const TokenRange r = sequence_tokens(p, n);
    const int64_t c = slot - ((r.lo >> kSegmentLog) + n), lo = r.lo + (c << kSegmentLog), left = r.hi - lo;
    if (c < 0 || left <= 0) return {0, 0, 0, n, 0, false};
    return {lo, (int)(left < kSegment ? left : kSegment), 0, n, (int)c, left <= kSegment};
}
// The border behind a segment, which the one in front of it is 1 less than: borders between 256 tokens of a packed sequence and the next lie behind different
// tokens 256 f, as many segments as they are apart.
__device__ __forceinline__ int64_t border_behind(const cc1d_delta_params &p, const SegmentWork &w, int n, int64_t lo, int c) {
    return p.cu_seqlens == nullptr ? (int64_t)n * (w.chunks - 1) + c : lo >> kSegmentLog;
}
__device__ __forceinline__ int64_t border_behind(const cc1d_delta_params &p, const SegmentWork &w, const SegmentAt &at) { return border_behind(p, w, at.n, at.lo, at.c); }
__device__ __forceinline__ int first_segment(const cc1d_delta_params &p, const SegmentWork &w, int n, const TokenRange &r) {
    return p.cu_seqlens == nullptr ? n * w.chunks : w.shortest > 0 ? 2 * (int)naming(r) : (int)(r.lo >> kSegmentLog) + n;
}

// Which sums a segment's neighbours need: forward those in front of the last (and the last, if the states are asked for), backward those behind
// the first.
struct StatesArgs { LinearRows a, b; int32_t from_start, all; float factor; };
struct ScanArgs {
    const float *first; int64_t first_n, first_h, first_k;     // the state it begins with, or NULL
    float *last; int64_t last_n, last_h, last_k;               // where it ends, or NULL
    int32_t to_end;                      // the last segment's own sum is there too: `last`, or S0 . dS0 of the first, need it
    int32_t reverse, write_k, write_v, use_inner;
};
// A product with a state has a right operand of 16 columns a tile, PT terms of 1 KB each: [step of the contraction][tile][term].
// Which columns of an operand of a state stand for which of the matrix: of every 16 W, tile t (0 .. W - 1) and lane m are column W m + t; W = 2 for the
// general kernel, 4 or 8 for linear_tile_kernel.
__device__ __forceinline__ int operand_place(int col, int width) {     // of 1 KB tiles of 16 columns: tile << 4 | m
    const int in = col & (16 * width - 1);
    return (col / (16 * width) * width + in % width) << 4 | in / width;
}
struct AttendArgs {
    LinearRows x, y, z, u;               // u: what the rows of the result are multiplied with for the gates' gradients
    const uint8_t *state;
    int32_t d1, d2, steps;               // columns of x, y and of z; 32-column steps of x, y
    int32_t width, tiles;                // W of the state's operands, and their number in a step
    int32_t tile;                        // linear_tile_kernel takes it
    int32_t first;                       // the first segment (REV: the last) has a state too
    int32_t group, heads_each, shares;   // value heads of a key head, of a workgroup; workgroups of a key head
    uint32_t items, col_tiles;           // (slot, key head, share); 128-column tiles of d2
    FastDiv by_col_tiles, by_heads, by_shares;
    void *out; int64_t out_b, out_l, out_h;   // of x_dtype, by value head or (DOTS) by key head; NULL: to `share`
    float *share;
    double *dots;
    float *selves, *uz;                  // dk, with beta
};

// `out`: from whole vectors to rows as they are, else the other way round.
int launch_linear_copy(const CopyArgs &a, int copies, bool out, hipStream_t stream);
int launch_linear_states(const cc1d_delta_params &p, const SegmentWork &w, const StatesArgs &a, hipStream_t stream);
int launch_linear_scan(const cc1d_delta_params &p, const SegmentWork &w, const ScanArgs &a, hipStream_t stream);
// Instantiated one to a file: out (REV: dv), and dq and dk together, in float32 with dv if given.
template <int DT, bool REV>
int launch_attend(const cc1d_delta_params &p, const SegmentWork &w, const AttendArgs &a, hipStream_t stream);
template <int DT>
int launch_attend_pair(const cc1d_delta_params &p, const SegmentWork &w, const AttendArgs &q, const AttendArgs &k, const AttendArgs *v, hipStream_t stream);
int launch_linear_gates(const cc1d_delta_bwd_params &bp, const SegmentWork &w, hipStream_t stream);
int launch_linear_join(const cc1d_delta_bwd_params &bp, const SegmentWork &w, hipStream_t stream);

}  // namespace cc1d
