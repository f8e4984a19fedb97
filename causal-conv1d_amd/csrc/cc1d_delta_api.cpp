// C-ABI front of the gated delta rule (cc1d_mixer.h): argument validation and dispatch to the kernel
// launchers.  Nothing here allocates or synchronises; validation never touches the GPU.
#include "cc1d_delta_chunk.hpp"
#include "cc1d_delta_host.hpp"

using namespace cc1d;

namespace {

bool aligned256(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 255u) == 0; }
bool dtype_ok(int d) { return d == CC1D_F32 || d == CC1D_F16 || d == CC1D_BF16; }
bool on_elements(const void *p, int dtype) { return (reinterpret_cast<uintptr_t>(p) & ((uintptr_t)elem_bytes(dtype) - 1)) == 0; }

template <typename P>
int check_sizes(const P &p) {
    if (!dtype_ok(p.x_dtype) || !dtype_ok(p.g_dtype) || !dtype_ok(p.beta_dtype)) return CC1D_ERR_DTYPE;
    if (p.batch < 0 || p.seqlen < 0 || p.heads < 1 || p.v_heads < 0) return CC1D_ERR_SHAPE;
    if (p.v_heads % p.heads != 0) return CC1D_ERR_HEADS;
    if (p.dim_k < 1 || p.dim_k > 256 || p.dim_v < 1 || p.dim_v > 512) return CC1D_ERR_HEAD_DIM;
    return CC1D_OK;
}
template <typename P>
int check_inputs(const P &p) {
    if (p.q == nullptr || p.k == nullptr || p.v == nullptr || p.g == nullptr || p.beta == nullptr) return CC1D_ERR_NULL_POINTER;
    if (!on_elements(p.q, p.x_dtype) || !on_elements(p.k, p.x_dtype) || !on_elements(p.v, p.x_dtype) || !on_elements(p.g, p.g_dtype) ||
        !on_elements(p.beta, p.beta_dtype)) return CC1D_ERR_ROW_LAYOUT;
    return CC1D_OK;
}
int check_delta(const cc1d_delta_params &p) {
    int st = check_sizes(p);
    if (st != CC1D_OK) return st;
    if (p.sequences < 0 || (p.cu_seqlens == nullptr ? p.sequences != p.batch : p.batch != 1)) return CC1D_ERR_SHAPE;
    if (p.sequences == 0 && p.batch > 0 && p.seqlen > 0) return CC1D_ERR_SHAPE;        // nobody would write their zeros
    if (p.batch > 0 && p.seqlen > 0 && p.v_heads > 0) st = check_inputs(p);
    if (st != CC1D_OK) return st;
    if (p.saved != nullptr && !aligned256(p.saved)) return CC1D_ERR_WORKSPACE;
    if (!on_elements(p.initial_states, CC1D_F32) || !on_elements(p.final_states, CC1D_F32) || !on_elements(p.out, p.x_dtype)) return CC1D_ERR_ROW_LAYOUT;
    return CC1D_OK;
}

// Sequences of this many tokens on average go by chunks.  A token costs the token kernel 1.3 us as long as its states fill no more than the card,
// a chunk costs as much for one token as for 64.  Measured with heads of 128 x 128 and applied to all, token by token / by chunks, us:
//   bfloat16  32 heads:  8 tokens 15.9 / 14.9   256: 20 tokens 33.7 / 32.3   2048: 32 tokens 203 / 235, 48: 293 / 251
//   float32   32 heads: 12 tokens 20.5 / 19.4   256: 40 tokens 59.2 / 61.1   2048: 96 tokens 538 / 810, 128: 712 / 825
int chunked_from(const cc1d_delta_params &p) {
    const int64_t heads = (int64_t)p.sequences * p.v_heads;
    if (heads <= 128) return 10;
    if (heads <= 1024) return p.x_dtype == CC1D_F32 ? 40 : 20;
    return p.x_dtype == CC1D_F32 ? 160 : 40;
}
// The scans reach the 64 rows of a chunk with 32 bits; a single token's stride is nowhere taken.
bool near(const cc1d_delta_params &p, int64_t stride) {
    return p.seqlen <= 1 || (stride >= 0 && stride * elem_bytes(p.x_dtype) < ((int64_t)1 << 31) / kChunk);
}
bool reachable(const cc1d_delta_params &p) { return near(p, p.v_stride_l) && near(p, p.out_stride_l); }
// Grids of one workgroup a (slot, value head) and of one a (sequence or what names one, value head, 16 columns).
bool grids_fit(const cc1d_delta_params &p, int64_t slots, int64_t walks) {
    const int64_t limit = thread_limit() / 512;
    return slots * p.v_heads < limit && (walks * p.v_heads + 8) * ((p.dim_v + 15) / 16) < limit;
}
// The average says nothing of the longest.  Packed sequences that go by tokens on average go by chunks one by one, from chunked_from() tokens
// and from 64 on: the kernels see their lengths, the host does not.  One of 4096 tokens among 128 of one token, 32 heads: 6150 us by tokens
// alone, 245 so; four of 1000 among 128 of eight: 1556 and 302.  Where all are short the chunks' workgroups find nothing to do: 128 of 16 tokens 226 us
// and 247, 2048 of 4 tokens 1520 and 1611.  Not where the tokens are so few that one sequence of them all could not cost
// much more than that (255: 330 us).
int chunked_alone(const cc1d_delta_params &p) {
    const int from = chunked_from(p);
    return from > kChunk ? from : kChunk;
}
// How a call goes: by tokens, by chunks, or each packed sequence by its own length.
enum class Way { tokens, chunks, both };
Way way_of(const cc1d_delta_params &p) {
    if (p.batch == 0 || p.v_heads == 0 || p.sequences == 0 || p.seqlen == 0) return Way::tokens;
    if (p.saved != nullptr) return Way::chunks;
    if (!reachable(p)) return Way::tokens;
    if (p.seqlen >= (int64_t)chunked_from(p) * (p.cu_seqlens == nullptr ? 1 : p.sequences)) return Way::chunks;
    const int64_t chunks = ((int64_t)p.seqlen + kChunk - 1) / kChunk;
    return p.cu_seqlens != nullptr && p.seqlen >= 4 * kChunk && grids_fit(p, 2 * chunks, chunks) ? Way::both : Way::tokens;
}

struct Places {
    uint8_t *base;
    size_t used = 0;
    uint8_t *take(size_t bytes) {
        uint8_t *at = base + used;
        used += (bytes + 255) / 256 * 256;
        return at;
    }
};
// Places in the workspace and in `saved`; returns the workspace's size.
size_t lay_out(const cc1d_delta_params &p, bool backward, int shortest, uint8_t *base, ChunkWork &w, size_t *saved_bytes = nullptr) {
    w = ChunkWork();
    w.chunks = (int32_t)(((int64_t)p.seqlen + kChunk - 1) / kChunk);
    w.shortest = shortest;
    const int64_t slots = p.cu_seqlens == nullptr ? (int64_t)p.batch * w.chunks : w.shortest > 0 ? 2 * (int64_t)w.chunks : (int64_t)p.seqlen / kChunk + p.sequences + 1;
    w.slots = (int32_t)(slots < INT32_MAX ? slots : INT32_MAX);
    w.ks = key_steps(p.dim_k);
    w.terms = p.x_dtype == CC1D_BF16 ? 1 : p.x_dtype == CC1D_F16 ? 2 : 3;
    w.pterms = p.x_dtype == CC1D_F32 ? 3 : 2;
    w.backward = backward;
    w.by_heads = fast_div((uint32_t)p.heads);
    w.by_v_heads = fast_div((uint32_t)p.v_heads);
    w.by_group = fast_div((uint32_t)(p.heads > 0 ? p.v_heads / p.heads : 1));
    w.by_chunks = fast_div((uint32_t)w.chunks);
    const size_t keys = (size_t)w.slots * p.heads, values = (size_t)w.slots * p.v_heads;
    const size_t state = values * p.dim_k * p.dim_v * sizeof(float), rows = values * kChunk * p.dim_v * sizeof(float);
    Places saved{static_cast<uint8_t *>(p.saved)};
    w.s0 = reinterpret_cast<float *>(saved.take(state));
    w.u = reinterpret_cast<float *>(saved.take(rows));
    if (saved_bytes != nullptr) *saved_bytes = saved.used;
    Places work{base};
    w.kf = work.take(keys * w.kbytes());
    w.ktf = work.take(keys * w.kbytes());
    w.scalars = reinterpret_cast<float *>(work.take(values * kScalars * kChunk * sizeof(float)));
    if (backward) {
        w.qtf = work.take(keys * w.kbytes()); w.ttf = work.take(values * w.tbytes()); w.ptf = work.take(values * w.tbytes());
        w.ds1 = reinterpret_cast<float *>(work.take(state));
        w.dx = reinterpret_cast<float *>(work.take(rows));
        if (p.v_heads > p.heads) w.dqk = reinterpret_cast<float *>(work.take(values * 2 * kChunk * 32 * w.ks * sizeof(float)));
    } else {
        w.qf = work.take(keys * w.kbytes());
        w.tf = work.take(values * w.tbytes()); w.pf = work.take(values * w.pbytes());
    }
    return work.used;
}
}  // namespace

extern "C" {

int cc1d_validate_delta(const cc1d_delta_params *p) {
    if (p == nullptr) return CC1D_ERR_NULL_POINTER;
    const int st = check_delta(*p);
    if (st != CC1D_OK) return st;
    if (p->batch > 0 && p->seqlen > 0 && p->v_heads > 0 && p->out == nullptr) return CC1D_ERR_NULL_POINTER;
    return CC1D_OK;
}

int cc1d_delta_workspace_bytes(const cc1d_delta_params *p, size_t *bytes) {
    if (bytes == nullptr) return CC1D_ERR_NULL_POINTER;
    *bytes = 0;
    const int st = cc1d_validate_delta(p);
    const Way way = st == CC1D_OK ? way_of(*p) : Way::tokens;
    if (way == Way::tokens) return st;
    ChunkWork w;
    *bytes = lay_out(*p, false, way == Way::both ? chunked_alone(*p) : 0, nullptr, w);
    return grids_fit(*p, w.slots, w.walks(*p)) && reachable(*p) ? CC1D_OK : CC1D_ERR_TOO_LARGE;
}

int cc1d_delta_saved_bytes(const cc1d_delta_params *p, size_t *bytes) {
    if (bytes == nullptr) return CC1D_ERR_NULL_POINTER;
    *bytes = 0;
    if (p == nullptr) return CC1D_ERR_NULL_POINTER;
    const int st = check_delta(*p);
    if (st != CC1D_OK) return st;
    ChunkWork w;
    lay_out(*p, false, 0, nullptr, w, bytes);               // (of packed sequences without tokens too: what a traced call reckons with)
    return CC1D_OK;
}

int cc1d_delta_fwd(const cc1d_delta_params *p, void *workspace, size_t workspace_bytes, cc1d_stream_t stream) {
    size_t need = 0;
    const int st = cc1d_delta_workspace_bytes(p, &need);
    if (st != CC1D_OK) return st;
    if (need > 0 && (workspace == nullptr || !aligned256(workspace) || workspace_bytes < need)) return CC1D_ERR_WORKSPACE;
    if (p->batch == 0 || p->v_heads == 0 || p->sequences == 0) return CC1D_OK;
    const hipStream_t hs = static_cast<hipStream_t>(stream);
    const Way way = way_of(*p);
    if (way == Way::tokens) return launch_delta_tokens(*p, nullptr, p->sequences, 0, hs);
    ChunkWork w;
    lay_out(*p, false, way == Way::both ? chunked_alone(*p) : 0, static_cast<uint8_t *>(workspace), w);
    int done = launch_delta_prep(*p, w, hs);
    if (done == CC1D_OK) done = launch_delta_scan(*p, w, p->saved != nullptr, hs);
    return done != CC1D_OK || way == Way::chunks ? done : launch_delta_tokens(*p, nullptr, p->sequences, w.shortest, hs);
}

int cc1d_validate_delta_bwd(const cc1d_delta_bwd_params *p) {
    if (p == nullptr) return CC1D_ERR_NULL_POINTER;
    const int st = check_delta(p->fwd);
    if (st != CC1D_OK) return st;
    const cc1d_delta_params &f = p->fwd;
    if (f.batch > 0 && f.seqlen > 0 && f.v_heads > 0 &&
        (f.saved == nullptr || p->dout == nullptr || p->dv == nullptr || p->dg == nullptr || p->dbeta == nullptr)) return CC1D_ERR_NULL_POINTER;
    if (f.batch > 0 && f.seqlen > 0 && (p->dq == nullptr || p->dk == nullptr)) return CC1D_ERR_NULL_POINTER;           // (written without value heads too)
    if (!on_elements(p->dout, f.x_dtype) || !on_elements(p->dq, f.x_dtype) || !on_elements(p->dk, f.x_dtype) || !on_elements(p->dv, f.x_dtype) ||
        !on_elements(p->dg, f.g_dtype) || !on_elements(p->dbeta, f.beta_dtype) || !on_elements(p->dfinal_states, CC1D_F32) ||
        !on_elements(p->dinitial_states, CC1D_F32)) return CC1D_ERR_ROW_LAYOUT;
    return CC1D_OK;
}

int cc1d_delta_bwd_workspace_bytes(const cc1d_delta_bwd_params *p, size_t *bytes) {
    if (bytes == nullptr) return CC1D_ERR_NULL_POINTER;
    *bytes = 0;
    const int st = cc1d_validate_delta_bwd(p);
    if (st != CC1D_OK || p->fwd.batch == 0 || p->fwd.v_heads == 0 || p->fwd.sequences == 0) return st;
    ChunkWork w;
    *bytes = lay_out(p->fwd, true, 0, nullptr, w);
    const bool far = !near(p->fwd, p->dout_stride_l) || !near(p->fwd, p->dv_stride_l);
    return grids_fit(p->fwd, w.slots, w.walks(p->fwd)) && !far ? CC1D_OK : CC1D_ERR_TOO_LARGE;
}

int cc1d_delta_bwd(const cc1d_delta_bwd_params *p, void *workspace, size_t workspace_bytes, cc1d_stream_t stream) {
    size_t need = 0;
    int st = cc1d_delta_bwd_workspace_bytes(p, &need);
    if (st != CC1D_OK) return st;
    if (need > 0 && (workspace == nullptr || !aligned256(workspace) || workspace_bytes < need)) return CC1D_ERR_WORKSPACE;
    const hipStream_t hs = static_cast<hipStream_t>(stream);
    if (p->fwd.v_heads == 0) return launch_delta_no_values(*p, hs);
    if (p->fwd.batch == 0 || p->fwd.sequences == 0) return CC1D_OK;
    ChunkWork w;
    lay_out(p->fwd, true, 0, static_cast<uint8_t *>(workspace), w);
    if (w.slots > 0) st = launch_delta_prep(p->fwd, w, hs);
    if (st != CC1D_OK) return st;
    return launch_delta_bwd(*p, w, hs);
}

int cc1d_validate_delta_step(const cc1d_delta_step_params *p) {
    if (p == nullptr) return CC1D_ERR_NULL_POINTER;
    int st = check_sizes(*p);
    if (st != CC1D_OK) return st;
    if (p->state_slots < 0 || (p->state_indices == nullptr && p->state_slots != p->batch)) return CC1D_ERR_SHAPE;
    if (p->batch == 0 || p->seqlen == 0 || p->v_heads == 0) return CC1D_OK;
    st = check_inputs(*p);
    if (st != CC1D_OK) return st;
    if (p->out == nullptr || (p->state == nullptr && p->state_slots > 0)) return CC1D_ERR_NULL_POINTER;
    if (!on_elements(p->state, CC1D_F32) || !on_elements(p->out, p->x_dtype)) return CC1D_ERR_ROW_LAYOUT;
    return CC1D_OK;
}

int cc1d_delta_step(const cc1d_delta_step_params *s, cc1d_stream_t stream) {
    const int st = cc1d_validate_delta_step(s);
    if (st != CC1D_OK || s->batch == 0 || s->seqlen == 0 || s->v_heads == 0) return st;
    cc1d_delta_params p = {};
    p.batch = p.sequences = s->batch; p.seqlen = s->seqlen; p.heads = s->heads; p.v_heads = s->v_heads;
    p.dim_k = s->dim_k; p.dim_v = s->dim_v;
    p.x_dtype = s->x_dtype; p.g_dtype = s->g_dtype; p.beta_dtype = s->beta_dtype;
    p.qk_l2norm = s->qk_l2norm; p.scale = s->scale;
    p.q = s->q; p.q_stride_b = s->q_stride_b; p.q_stride_l = s->q_stride_l; p.q_stride_h = s->q_stride_h;
    p.k = s->k; p.k_stride_b = s->k_stride_b; p.k_stride_l = s->k_stride_l; p.k_stride_h = s->k_stride_h;
    p.v = s->v; p.v_stride_b = s->v_stride_b; p.v_stride_l = s->v_stride_l; p.v_stride_h = s->v_stride_h;
    p.g = s->g; p.g_stride_b = s->g_stride_b; p.g_stride_l = s->g_stride_l; p.g_stride_h = s->g_stride_h;
    p.beta = s->beta; p.beta_stride_b = s->beta_stride_b; p.beta_stride_l = s->beta_stride_l; p.beta_stride_h = s->beta_stride_h;
    p.initial_states = s->state; p.init_stride_n = s->state_stride_n; p.init_stride_h = s->state_stride_h; p.init_stride_k = s->state_stride_k;
    p.final_states = s->state; p.final_stride_n = s->state_stride_n; p.final_stride_h = s->state_stride_h; p.final_stride_k = s->state_stride_k;
    p.out = s->out; p.out_stride_b = s->out_stride_b; p.out_stride_l = s->out_stride_l; p.out_stride_h = s->out_stride_h;
    return launch_delta_tokens(p, s->state_indices, s->state_slots, 0, static_cast<hipStream_t>(stream));
}

}  // extern "C"
