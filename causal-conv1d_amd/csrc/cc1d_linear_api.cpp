// C-ABI front of linear attention (cc1d_mixer.h): argument validation, layout of the workspace and the order of the launches.  Nothing
// here allocates or synchronises; validation never touches the GPU.
#include "cc1d_delta_host.hpp"
#include "cc1d_linear.hpp"

namespace cc1d {

#define CC1D_ATTEND(DT)                                                                                                                   \
    extern template int launch_attend<DT, false>(const cc1d_delta_params &, const SegmentWork &, const AttendArgs &, hipStream_t);     \
    extern template int launch_attend<DT, true>(const cc1d_delta_params &, const SegmentWork &, const AttendArgs &, hipStream_t);      \
    extern template int launch_attend_pair<DT>(const cc1d_delta_params &, const SegmentWork &, const AttendArgs &, const AttendArgs &, const AttendArgs *, hipStream_t);
CC1D_ATTEND(CC1D_F32)
CC1D_ATTEND(CC1D_F16)
CC1D_ATTEND(CC1D_BF16)
#undef CC1D_ATTEND

}  // namespace cc1d

using namespace cc1d;

namespace {

bool aligned256(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 255u) == 0; }

// The blocks are the gated delta rule's, whose checks want a beta.
template <typename P>
P with_beta(const P &p) {
    P q = p;
    if (q.beta == nullptr) {
        q.beta = q.g;
        q.beta_dtype = q.g_dtype;
    }
    return q;
}

// Rows of a segment are reached with 32 bits.
bool near(const cc1d_delta_params &p, int64_t stride) {
    return p.seqlen <= 1 || (stride >= 0 && stride * elem_bytes(p.x_dtype) < ((int64_t)1 << 31) / kSegment);
}
bool reachable(const cc1d_delta_params &p) { return near(p, p.q_stride_l) && near(p, p.k_stride_l) && near(p, p.v_stride_l); }
bool reachable_out(const cc1d_delta_params &p) { return reachable(p) && near(p, p.out_stride_l); }
bool reachable_gradients(const cc1d_delta_bwd_params &bp) {
    return reachable(bp.fwd) && near(bp.fwd, bp.dout_stride_l) && near(bp.fwd, bp.dq_stride_l) && near(bp.fwd, bp.dk_stride_l) && near(bp.fwd, bp.dv_stride_l);
}

// Sequences of this many tokens on average go by segments; `saved`: all do.  A token takes 0.7 to 1 us until the states of 512 heads of 128 x 128 (or as
// many elements of other heads) fill the card, then time by their number; a segment costs by heads and by their elements.  By tokens and
// by segments, us: 16-bit types, 128 x 128, 4 heads: 16 tokens 21 and 20; 256: 24 tokens 31 and 36, 32 tokens 39 and 36; 1024: 48 tokens 127 and 135,
// 64 tokens 162 and 138; 32 x 32, 1024 heads: 32 tokens 28 and 29; 2880: 64 tokens 80 and 82.  float32, whose products take six matrix instructions for
// one to three, 128 x 128, 4 heads: 24 tokens 27 and 24; 256: 48 tokens 51 and 60, 64 tokens 66 and 61; 512: 96 tokens 116 and 132, 128 tokens 150 and 140;
// 1024: 128 tokens 267 and 298, 256 tokens 540 and 420.  Many small ones go by tokens at any length: 2880 of 32 x 32: 256 tokens 286 and 447, 4096 tokens 4480
// and 7560; 2048 of 64 x 64: 256 tokens 395 and 379, 1024 tokens 1380 and 1580, 4096 tokens 6030 and 6410; 8192 of 64 x 64: 4096 tokens 21400 and 25600.
int64_t segments_from(const cc1d_delta_params &p, int64_t sequences) {
    const double heads = (double)sequences * p.v_heads, size = (double)p.dim_k * p.dim_v / 16384.0, most = heads < 1e6 ? heads : 1e6;
    if (p.x_dtype == CC1D_F32) {
        if (heads >= 2048.0 && size <= 0.25) return INT32_MAX;
        const int64_t from = 22 + (int64_t)(most * (0.05 + 0.14 * size));
        return from < 170 ? from : 170;
    }
    const int64_t from = 16 + (int64_t)(most * (0.016 + 0.03 * size)), cap = heads * size >= 512.0 ? 50 : 96;
    return from < cap ? from : cap;
}
// Whether any segment has a state in front of it.
bool has_states(const cc1d_delta_params &p, const SegmentWork &w) { return w.chunks > 1 || p.cu_seqlens != nullptr || p.initial_states != nullptr; }

struct Places {
    uint8_t *base;
    size_t used = 0;
    uint8_t *take(size_t bytes) {
        uint8_t *at = base + used;
        used += (bytes + 255) / 256 * 256;
        return at;
    }
    float *floats(size_t n) { return reinterpret_cast<float *>(take(n * sizeof(float))); }
    double *doubles(size_t n) { return reinterpret_cast<double *>(take(n * sizeof(double))); }
};

SegmentWork sizes_of(const cc1d_delta_params &p, bool alone) {
    SegmentWork w = {};
    w.shortest = alone ? kSegment : 0;
    w.chunks = (int32_t)(((int64_t)p.seqlen + kSegment - 1) / kSegment);
    const int64_t slots = p.cu_seqlens == nullptr ? (int64_t)p.batch * w.chunks : alone ? 2 * (int64_t)w.chunks : (int64_t)p.seqlen / kSegment + p.sequences + 1;
    w.slots = (int32_t)(slots < INT32_MAX ? slots : INT32_MAX);
    w.borders = (int64_t)p.batch * (w.chunks > 0 ? w.chunks - 1 : 0);      // (packed: one behind every token 256 f but the last)
    w.kp = (p.dim_k + 31) / 32;
    w.vp = (p.dim_v + 31) / 32;
    w.k_width = operand_width(p.x_dtype, p.dim_k, p.dim_v, false);
    w.v_width = operand_width(p.x_dtype, p.dim_v, p.dim_k, true);
    w.k_tiles = operand_tiles(w.k_width, p.dim_v);
    w.v_tiles = operand_tiles(w.v_width, p.dim_k);
    w.by_v_heads = fast_div((uint32_t)p.v_heads);
    w.by_chunks = fast_div((uint32_t)w.chunks);
    w.by_group = fast_div((uint32_t)(p.heads > 0 ? p.v_heads / p.heads : 1));
    return w;
}
// Numbers of 32 x 32 tiles of states, at every border or at every segment, for every value head; bytes of their operands.
size_t states_of(const cc1d_delta_params &p, const SegmentWork &w, bool all) { return (size_t)(all ? (int64_t)w.slots : w.borders) * p.v_heads; }
size_t state_tiles(const cc1d_delta_params &p, const SegmentWork &w, bool all) { return states_of(p, w, all) * w.tiles(); }
size_t by_k_bytes(const cc1d_delta_params &p, const SegmentWork &w, bool all) { return states_of(p, w, all) * w.kp * w.k_tiles * out_terms(p.x_dtype) * kFrag; }
size_t by_v_bytes(const cc1d_delta_params &p, const SegmentWork &w, bool all) { return states_of(p, w, all) * w.vp * w.v_tiles * 3 * kFrag; }
// `saved` is never nothing: it says that a backward follows.
constexpr size_t kLeastSaved = 256;

// One workgroup a (slot, block, value head, 128 columns) and less, of two such products at once in the backward; the scan's one wavefront a tile of each
// sequence's states.
bool grids_fit(const cc1d_delta_params &p, const SegmentWork &w, int products) {
    return ((int64_t)w.slots * p.v_heads + 8) * kBlocks * (products > (w.vp + 3) / 4 ? products : (w.vp + 3) / 4) < thread_limit() / kBlock &&
           w.walks(p) * p.v_heads * w.tiles() < thread_limit() / kWave;
}

LinearRows rows(const void *x, int64_t sb, int64_t sl, int64_t sh, bool by_key) { return {x, sb, sl, sh, by_key}; }
#define ROWS(P, NAME, KEY) rows(P.NAME, P.NAME##_stride_b, P.NAME##_stride_l, P.NAME##_stride_h, KEY)
bool whole(int dtype, const LinearRows &r, int dim) { return dim % kVector == 0 && whole_rows(dtype, r.p, r.sb, r.sl, r.sh); }

// A call's tensors as the kernels read and write them; those whose rows are not whole vectors at their places in the workspace, and what it takes to bring them
// there and back.
struct Tensors {
    const cc1d_delta_params &p;
    Places &work;
    CopyArgs in = {}, out = {};
    int ins = 0, outs = 0;
    Tensors(const cc1d_delta_params &params, Places &places) : p(params), work(places) {
        in.elem = out.elem = elem_bytes(p.x_dtype);
        in.batch = out.batch = p.batch;
        in.seqlen = out.seqlen = p.seqlen;
        in.by_seqlen = out.by_seqlen = fast_div((uint32_t)(p.seqlen > 0 ? p.seqlen : 1));
    }
    LinearRows place(const LinearRows &r, int dim, bool written) {
        if (whole(p.x_dtype, r, dim)) return r;
        const int heads = r.by_key ? p.heads : p.v_heads, pitch = padded(dim), e = elem_bytes(p.x_dtype);
        LinearRows at = {nullptr, (int64_t)p.seqlen * heads * pitch, (int64_t)heads * pitch, pitch, r.by_key};
        at.p = work.take((size_t)p.batch * at.sb * e);
        const LinearRows &from = written ? at : r, &to = written ? r : at;
        CopyRows &c = written ? out.of[outs++] : in.of[ins++];
        c.from = static_cast<const uint8_t *>(from.p);
        c.to = static_cast<uint8_t *>(const_cast<void *>(to.p));
        c.from_b = from.sb * e; c.from_l = from.sl * e; c.from_h = from.sh * e;
        c.to_b = to.sb * e; c.to_l = to.sl * e; c.to_h = to.sh * e;
        c.heads = heads;
        c.dim = dim;
        c.by_vectors = fast_div((uint32_t)(pitch / kVector));
        return at;
    }
    LinearRows read(const LinearRows &r, int dim) { return place(r, dim, false); }
    LinearRows written(const LinearRows &r, int dim) { return place(r, dim, true); }
};
// The rows of a segment of a copy are reached with 32 bits as well.
bool copies_reachable(const cc1d_delta_params &p) {
    return (int64_t)p.v_heads * padded(p.dim_k > p.dim_v ? p.dim_k : p.dim_v) * elem_bytes(p.x_dtype) < ((int64_t)1 << 31) / kSegment;
}

struct Forward { LinearRows q, k, v, out; CopyArgs in, back; int ins, backs; };
struct Backward { LinearRows q, k, v, dout, dq, dk, dv; CopyArgs in, back; int ins, backs; };

size_t lay_out_fwd(const cc1d_delta_params &p, bool alone, uint8_t *base, SegmentWork &w, Forward &f) {
    w = sizes_of(p, alone);
    Places work{base};
    if (has_states(p, w) || p.final_states != nullptr) {
        w.local = work.floats(state_tiles(p, w, p.final_states != nullptr) * 1024);
        w.decay = work.floats((size_t)w.slots * p.v_heads);
        w.by_k = work.take(by_k_bytes(p, w, p.initial_states != nullptr));
    }
    w.by_v = static_cast<uint8_t *>(p.saved);
    Tensors t(p, work);
    f.q = t.read(ROWS(p, q, true), p.dim_k);
    f.k = t.read(ROWS(p, k, true), p.dim_k);
    f.v = t.read(ROWS(p, v, false), p.dim_v);
    f.out = t.written(ROWS(p, out, false), p.dim_v);
    f.in = t.in; f.ins = t.ins; f.back = t.out; f.backs = t.outs;
    return work.used;
}

// Without `saved` the token kernel takes what the segments' do not.
bool segments_fit(const cc1d_delta_params &p, bool alone) {
    SegmentWork w;
    Forward f;
    lay_out_fwd(p, alone, nullptr, w, f);
    return grids_fit(p, w, 1) && reachable_out(p) && (f.ins + f.backs == 0 || copies_reachable(p));
}
// The average says nothing of the longest.  Packed sequences that go by tokens on average go by segments one by one, from 256 tokens on: the
// kernels see their lengths, the host does not.  Not where all their tokens together are few, nor where one sequence's heads fill
// the card with tokens.
enum class Way { tokens, segments, both };
Way way_of(const cc1d_delta_params &p) {
    if (p.batch == 0 || p.v_heads == 0 || p.sequences == 0 || p.seqlen == 0) return Way::tokens;
    if (p.saved != nullptr) return Way::segments;
    if (!reachable_out(p)) return Way::tokens;
    const Way way = p.seqlen >= segments_from(p, p.sequences) * (p.cu_seqlens == nullptr ? 1 : p.sequences) ? Way::segments :
                    p.cu_seqlens != nullptr && p.seqlen >= 2 * kSegment && segments_from(p, 1) <= kSegment ? Way::both : Way::tokens;
    return way == Way::tokens || segments_fit(p, way == Way::both) ? way : Way::tokens;
}

// Value heads that a workgroup takes one after the other, of `items` (slots and value heads): what belongs to their key head is read once for
// all of them, and of the gradients of q and k, whose workgroups of a shared key head each write a share in fp32, that is less too; but
// `workgroups` of them at least, one a CU (32 segments of 80 heads: out 112 us, with two 127).  Not where z has more than 64 columns: out of 64
// segments of 16 heads of 128 x 128, float16, 118 us each for itself and 138 in pairs, whose registers spill.
int heads_of_workgroup(int group, int64_t items, int workgroups) {
    const int64_t most = items / workgroups;
    const int each = most < 1 ? 1 : most > group ? group : (int)most, shares = (group + each - 1) / each;
    return (group + shares - 1) / shares;
}
void share_heads(const cc1d_delta_params &p, SegmentWork &w) {
    const int group = p.v_heads / p.heads;
    w.heads_each = heads_of_workgroup(group, (int64_t)w.slots * p.v_heads * (w.v_width > 2 ? 1 : kBlocks), 128);
    w.shares = (group + w.heads_each - 1) / w.heads_each;
}
bool gradient_of_states(const cc1d_delta_bwd_params &bp, const SegmentWork &w) {
    return has_states(bp.fwd, w) || bp.dfinal_states != nullptr || bp.dinitial_states != nullptr;
}
// Sums of all segments, the first's too: its S0 . dS0 or the gradient of the initial states.
bool needs_all_sums(const cc1d_delta_bwd_params &bp) { return bp.fwd.initial_states != nullptr || bp.dinitial_states != nullptr; }
size_t lay_out_bwd(const cc1d_delta_bwd_params &bp, uint8_t *base, SegmentWork &w, Backward &f) {
    const cc1d_delta_params &p = bp.fwd;
    w = sizes_of(p, false);
    w.first = static_cast<uint8_t *>(p.saved);
    Places work{base};
    share_heads(p, w);
    const size_t tokens = (size_t)p.batch * p.seqlen;
    if (gradient_of_states(bp, w)) {
        const bool initial = p.initial_states != nullptr, final = bp.dfinal_states != nullptr;
        w.local = work.floats(state_tiles(p, w, needs_all_sums(bp)) * 1024);
        w.decay = work.floats((size_t)w.slots * p.v_heads);
        w.by_k = work.take(by_k_bytes(p, w, final));
        w.by_v = work.take(by_v_bytes(p, w, final));
        w.inner = work.doubles(state_tiles(p, w, initial));
    }
    w.dot_q = work.doubles(tokens * p.v_heads);
    w.dot_k = work.doubles(tokens * p.v_heads);
    if (p.beta != nullptr) {
        w.self_k = work.floats(tokens * p.v_heads);
        w.qk = work.floats(tokens * p.heads);
    }
    if (w.shares > 1) {
        const size_t plane = (size_t)p.batch * p.seqlen * p.heads * padded(p.dim_k);
        w.share_q = work.floats(w.shares * plane);
        w.share_k = work.floats(w.shares * plane);
    }
    Tensors t(p, work);
    f.q = t.read(ROWS(p, q, true), p.dim_k);
    f.k = t.read(ROWS(p, k, true), p.dim_k);
    f.v = t.read(ROWS(p, v, false), p.dim_v);
    f.dout = t.read(ROWS(bp, dout, false), p.dim_v);
    f.dq = ROWS(bp, dq, true);
    f.dk = ROWS(bp, dk, true);
    if (w.shares == 1) {                 // (linear_join_kernel writes rows of any kind)
        f.dq = t.written(f.dq, p.dim_k);
        f.dk = t.written(f.dk, p.dim_k);
    }
    f.dv = t.written(ROWS(bp, dv, false), p.dim_v);
    f.in = t.in; f.ins = t.ins; f.back = t.out; f.backs = t.outs;
    return work.used;
}

AttendArgs prepared(const cc1d_delta_params &p, const SegmentWork &w, AttendArgs a, bool dots) {
    a.group = p.v_heads / p.heads;
    a.d1 = padded(a.d1);
    a.d2 = padded(a.d2);
    a.steps = (a.d1 + 31) / 32;
    a.width = dots ? w.v_width : w.k_width;
    a.tiles = dots ? w.v_tiles : w.k_tiles;
    a.tile = a.width > 2;
    a.heads_each = dots ? w.heads_each : a.width == 4 ? heads_of_workgroup(a.group, (int64_t)w.slots * p.v_heads, 256) : 1;
    a.shares = (a.group + a.heads_each - 1) / a.heads_each;
    a.items = (uint32_t)w.slots * (uint32_t)p.heads * (uint32_t)a.shares;
    a.col_tiles = dots ? 1u : (uint32_t)(a.d2 + (a.width == 4 ? 63 : 127)) / (a.width == 4 ? 64 : 128);
    a.by_col_tiles = fast_div(a.col_tiles);
    a.by_heads = fast_div((uint32_t)p.heads);
    a.by_shares = fast_div((uint32_t)a.shares);
    return a;
}
template <typename F>
int by_type(const cc1d_delta_params &p, F &&f) {
    switch (p.x_dtype) {
        case CC1D_F32: return f(std::integral_constant<int, CC1D_F32>());
        case CC1D_F16: return f(std::integral_constant<int, CC1D_F16>());
        default: return f(std::integral_constant<int, CC1D_BF16>());
    }
}
int attend(const cc1d_delta_params &p, const SegmentWork &w, const AttendArgs &given, hipStream_t stream) {
    if (w.slots == 0) return CC1D_OK;
    const AttendArgs a = prepared(p, w, given, false);
    return by_type(p, [&](auto dt) { return launch_attend<decltype(dt)::value, false>(p, w, a, stream); });
}
int attend_gradients(const cc1d_delta_params &p, const SegmentWork &w, const AttendArgs &dq, const AttendArgs &dk, const AttendArgs &dv, hipStream_t stream) {
    if (w.slots == 0) return CC1D_OK;
    const AttendArgs q = prepared(p, w, dq, true), k = prepared(p, w, dk, true), v = prepared(p, w, dv, false);
    const bool together = p.x_dtype == CC1D_F32 && (2 * (uint64_t)q.items + (uint64_t)v.items * v.col_tiles) * kBlocks <= 256;
    return by_type(p, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        const int st = launch_attend_pair<DT>(p, w, q, k, together ? &v : nullptr, stream);
        return st != CC1D_OK || together ? st : launch_attend<DT, true>(p, w, v, stream);
    });
}

void set_out(AttendArgs &a, const LinearRows &r) {
    a.out = const_cast<void *>(r.p);
    a.out_b = r.sb; a.out_l = r.sl; a.out_h = r.sh;
}

int forward(const cc1d_delta_params &p, const SegmentWork &w, const Forward &f, hipStream_t stream) {
    int st = launch_linear_copy(f.in, f.ins, false, stream);
    if (st != CC1D_OK) return st;
    const bool states = has_states(p, w);
    if (w.chunks > 1 || p.cu_seqlens != nullptr || p.final_states != nullptr) {
        StatesArgs a = {};
        a.a = f.k; a.b = f.v; a.all = p.final_states != nullptr;
        st = launch_linear_states(p, w, a, stream);
        if (st != CC1D_OK) return st;
    }
    if (states || p.final_states != nullptr) {
        ScanArgs a = {};
        a.first = p.initial_states; a.first_n = p.init_stride_n; a.first_h = p.init_stride_h; a.first_k = p.init_stride_k;
        a.last = p.final_states; a.last_n = p.final_stride_n; a.last_h = p.final_stride_h; a.last_k = p.final_stride_k;
        a.to_end = p.final_states != nullptr;
        a.write_k = states;
        a.write_v = states && p.saved != nullptr;
        st = launch_linear_scan(p, w, a, stream);
        if (st != CC1D_OK) return st;
    }
    AttendArgs a = {};
    a.x = f.q; a.y = f.k; a.z = f.v;
    a.d1 = p.dim_k; a.d2 = p.dim_v;
    a.state = w.by_k;
    a.first = p.initial_states != nullptr;
    set_out(a, f.out);
    st = attend(p, w, a, stream);
    return st != CC1D_OK ? st : launch_linear_copy(f.back, f.backs, true, stream);
}

int backward(const cc1d_delta_bwd_params &bp, const SegmentWork &w, const Backward &f, hipStream_t stream) {
    const cc1d_delta_params &p = bp.fwd;
    int st = launch_linear_copy(f.in, f.ins, false, stream);
    if (st != CC1D_OK) return st;
    const bool initial = p.initial_states != nullptr, to_end = needs_all_sums(bp);
    if (w.slots > 0 && (w.chunks > 1 || p.cu_seqlens != nullptr || to_end)) {
        StatesArgs a = {};
        a.a = f.q; a.b = f.dout; a.from_start = 1; a.all = to_end; a.factor = p.scale;
        st = launch_linear_states(p, w, a, stream);
        if (st != CC1D_OK) return st;
    }
    if (gradient_of_states(bp, w)) {
        ScanArgs a = {};
        a.first = bp.dfinal_states; a.first_n = bp.dfinal_stride_n; a.first_h = bp.dfinal_stride_h; a.first_k = bp.dfinal_stride_k;
        a.last = bp.dinitial_states; a.last_n = bp.dinit_stride_n; a.last_h = bp.dinit_stride_h; a.last_k = bp.dinit_stride_k;
        a.to_end = to_end;
        a.reverse = a.write_k = a.write_v = 1;
        a.use_inner = 1 + initial;
        st = launch_linear_scan(p, w, a, stream);
        if (st != CC1D_OK) return st;
    }
    AttendArgs dq = {}, dk = {};
    dq.x = f.dout; dq.y = f.v; dq.z = f.k; dq.u = f.q;
    dq.d1 = p.dim_v; dq.d2 = p.dim_k;
    dq.state = w.first;
    dq.first = initial;
    set_out(dq, f.dq);
    dq.share = w.share_q; dq.dots = w.dot_q;
    dk.x = f.v; dk.y = f.dout; dk.z = f.q; dk.u = f.k;
    dk.d1 = p.dim_v; dk.d2 = p.dim_k;
    dk.state = w.by_v;
    dk.first = bp.dfinal_states != nullptr;
    set_out(dk, f.dk);
    dk.share = w.share_k; dk.dots = w.dot_k; dk.selves = w.self_k; dk.uz = w.qk;
    AttendArgs d = {};                   // dv
    d.x = f.k; d.y = f.q; d.z = f.dout;
    d.d1 = p.dim_k; d.d2 = p.dim_v;
    d.state = w.by_k;
    d.first = bp.dfinal_states != nullptr;
    set_out(d, f.dv);
    st = attend_gradients(p, w, dq, dk, d, stream);
    if (st == CC1D_OK) st = launch_linear_gates(bp, w, stream);
    if (st == CC1D_OK && w.shares > 1 && w.slots > 0) st = launch_linear_join(bp, w, stream);
    if (st == CC1D_OK) st = launch_linear_copy(f.back, f.backs, true, stream);
    return st;
}

}  // namespace

extern "C" {

int cc1d_validate_linear(const cc1d_delta_params *p) {
    if (p == nullptr) return CC1D_ERR_NULL_POINTER;
    const cc1d_delta_params q = with_beta(*p);
    const int st = cc1d_validate_delta(&q);
    return st == CC1D_OK && p->qk_l2norm != 0 ? CC1D_ERR_OPTION : st;
}

int cc1d_linear_workspace_bytes(const cc1d_delta_params *p, size_t *bytes) {
    if (bytes == nullptr) return CC1D_ERR_NULL_POINTER;
    *bytes = 0;
    const int st = cc1d_validate_linear(p);
    const Way way = st == CC1D_OK ? way_of(*p) : Way::tokens;
    if (way == Way::tokens) return st;
    SegmentWork w;
    Forward f;
    *bytes = lay_out_fwd(*p, way == Way::both, nullptr, w, f);
    return p->saved == nullptr || segments_fit(*p, false) ? CC1D_OK : CC1D_ERR_TOO_LARGE;
}

int cc1d_linear_saved_bytes(const cc1d_delta_params *p, size_t *bytes) {
    if (bytes == nullptr) return CC1D_ERR_NULL_POINTER;
    *bytes = 0;
    if (p == nullptr) return CC1D_ERR_NULL_POINTER;
    cc1d_delta_params q = with_beta(*p);
    if (q.out == nullptr) q.out = const_cast<void *>(q.v);                 // (not needed for this)
    const int st = cc1d_validate_delta(&q);
    if (st != CC1D_OK) return st;
    const SegmentWork w = sizes_of(*p, false);
    *bytes = kLeastSaved + by_v_bytes(*p, w, p->initial_states != nullptr);
    return CC1D_OK;
}

int cc1d_linear_fwd(const cc1d_delta_params *p, void *workspace, size_t workspace_bytes, cc1d_stream_t stream) {
    size_t need = 0;
    const int st = cc1d_linear_workspace_bytes(p, &need);
    if (st != CC1D_OK) return st;
    if (need > 0 && (workspace == nullptr || !aligned256(workspace) || workspace_bytes < need)) return CC1D_ERR_WORKSPACE;
    if (p->batch == 0 || p->v_heads == 0 || p->sequences == 0) return CC1D_OK;
    const hipStream_t hs = static_cast<hipStream_t>(stream);
    const Way way = way_of(*p);
    if (way == Way::tokens) return launch_delta_tokens(*p, nullptr, p->sequences, 0, hs, false);
    SegmentWork w;
    Forward f;
    lay_out_fwd(*p, way == Way::both, static_cast<uint8_t *>(workspace), w, f);
    const int done = forward(*p, w, f, hs);
    return done != CC1D_OK || way == Way::segments ? done : launch_delta_tokens(*p, nullptr, p->sequences, w.shortest, hs, false);
}

int cc1d_validate_linear_bwd(const cc1d_delta_bwd_params *p) {
    if (p == nullptr) return CC1D_ERR_NULL_POINTER;
    cc1d_delta_bwd_params q = *p;
    q.fwd = with_beta(q.fwd);
    if (p->fwd.beta == nullptr) q.dbeta = q.dg;
    const int st = cc1d_validate_delta_bwd(&q);
    return st == CC1D_OK && p->fwd.qk_l2norm != 0 ? CC1D_ERR_OPTION : st;
}

int cc1d_linear_bwd_workspace_bytes(const cc1d_delta_bwd_params *p, size_t *bytes) {
    if (bytes == nullptr) return CC1D_ERR_NULL_POINTER;
    *bytes = 0;
    const int st = cc1d_validate_linear_bwd(p);
    if (st != CC1D_OK || p->fwd.batch == 0 || p->fwd.v_heads == 0 || p->fwd.sequences == 0) return st;
    SegmentWork w;
    Backward f;
    *bytes = lay_out_bwd(*p, nullptr, w, f);
    return grids_fit(p->fwd, w, 2) && reachable_gradients(*p) && (f.ins + f.backs == 0 || copies_reachable(p->fwd)) ? CC1D_OK : CC1D_ERR_TOO_LARGE;
}

int cc1d_linear_bwd(const cc1d_delta_bwd_params *p, void *workspace, size_t workspace_bytes, cc1d_stream_t stream) {
    size_t need = 0;
    const int st = cc1d_linear_bwd_workspace_bytes(p, &need);
    if (st != CC1D_OK) return st;
    if (need > 0 && (workspace == nullptr || !aligned256(workspace) || workspace_bytes < need)) return CC1D_ERR_WORKSPACE;
    const hipStream_t hs = static_cast<hipStream_t>(stream);
    if (p->fwd.v_heads == 0) return launch_delta_no_values(*p, hs);
    if (p->fwd.batch == 0 || p->fwd.sequences == 0) return CC1D_OK;
    SegmentWork w;
    Backward f;
    lay_out_bwd(*p, static_cast<uint8_t *>(workspace), w, f);
    return backward(*p, w, f, hs);
}

int cc1d_validate_linear_step(const cc1d_delta_step_params *p) {
    if (p == nullptr) return CC1D_ERR_NULL_POINTER;
    const cc1d_delta_step_params q = with_beta(*p);
    const int st = cc1d_validate_delta_step(&q);
    return st == CC1D_OK && p->qk_l2norm != 0 ? CC1D_ERR_OPTION : st;
}

int cc1d_linear_step(const cc1d_delta_step_params *p, cc1d_stream_t stream) {
    const int st = cc1d_validate_linear_step(p);
    if (st != CC1D_OK) return st;
    return launch_step_tokens(*p, static_cast<hipStream_t>(stream), false);
}

}  // extern "C"
