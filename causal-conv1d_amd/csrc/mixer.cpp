// PyTorch binding of cc1d_mixer.h: the gated delta rule, linear attention and the norms as ops of the DaoAILab
// library, part of the extension module `causal_conv1d_cuda`.  Host-only C++: tensors are checked, results and
// workspaces come from the caching allocator, launches go to the current stream of the tensors' device.
#include <torch/extension.h>
#include <torch/library.h>
#include <torch/types.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>

#include <cmath>
#include <optional>
#include <tuple>

#include "cc1d_mixer.h"
#include "cc1d_torch_calls.hpp"

namespace {

using OptTensor = std::optional<at::Tensor>;

// Unit stride along the last dimension (of more than one element).
bool unit_last(const at::Tensor &t) { return t.size(-1) <= 1 || t.stride(-1) == 1; }
at::Tensor rows_of(const at::Tensor &t) { return unit_last(t) ? t : t.contiguous(); }

void check_gpu(const at::Tensor &t, const at::Tensor &like, const char *what) {
    TORCH_CHECK(t.is_cuda(), what, " must be on the GPU");
    TORCH_CHECK(t.device() == like.device(), what, " must be on the device of the other tensors");
}

// Memory on the device of `like`, past the dispatcher: 0.35 us of host time less for each (64 rows of 512 into 8 bits and their scales
// 6.3 -> 5.6).  Only the ops' GPU implementations allocate with it: fake tensors and modes have had a call before it arrives there.
at::Tensor empty_of(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor &like) {
    return at::Tensor(at::detail::empty_cuda(sizes, type, like.device(), std::nullopt));
}

at::Tensor workspace_of(size_t bytes, const at::Tensor &like) {
    return bytes ? empty_of({(int64_t)bytes}, at::kByte, like) : at::Tensor();
}

// ---- gated delta rule, linear attention ------------------------------------------------
// One binding for both: the same parameter blocks, the second without lengths of q and k and with an optional beta.
struct Recurrence {
    int (*workspace_bytes)(const cc1d_delta_params *, size_t *);
    int (*saved_bytes)(const cc1d_delta_params *, size_t *);
    int (*fwd)(const cc1d_delta_params *, void *, size_t, cc1d_stream_t);
    int (*bwd_workspace_bytes)(const cc1d_delta_bwd_params *, size_t *);
    int (*bwd)(const cc1d_delta_bwd_params *, void *, size_t, cc1d_stream_t);
    int (*step)(const cc1d_delta_step_params *, cc1d_stream_t);
    const char *name, *name_bwd, *name_update;
};
constexpr Recurrence kDelta = {cc1d_delta_workspace_bytes, cc1d_delta_saved_bytes, cc1d_delta_fwd, cc1d_delta_bwd_workspace_bytes, cc1d_delta_bwd, cc1d_delta_step,
                               "gated_delta_rule", "gated_delta_rule backward", "gated_delta_rule_update"};
constexpr Recurrence kLinear = {cc1d_linear_workspace_bytes, cc1d_linear_saved_bytes, cc1d_linear_fwd, cc1d_linear_bwd_workspace_bytes, cc1d_linear_bwd, cc1d_linear_step,
                                "linear_attention", "linear_attention backward", "linear_attention_update"};

struct DeltaInputs {
    at::Tensor q, k, v, g;
    OptTensor beta;
    int64_t batch, seqlen, heads, v_heads, dim_k, dim_v;
};

DeltaInputs delta_inputs(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &g, const OptTensor &opt_beta) {
    check_gpu(q, q, "q"); check_gpu(k, q, "k"); check_gpu(v, q, "v"); check_gpu(g, q, "g");
    if (opt_beta.has_value()) check_gpu(*opt_beta, q, "beta");
    TORCH_CHECK(q.dim() == 4, "q must be (batch, seqlen, heads, dim_k)");
    TORCH_CHECK(v.dim() == 4, "v must be (batch, seqlen, v_heads, dim_v)");
    DeltaInputs d;
    d.batch = q.size(0); d.seqlen = q.size(1); d.heads = q.size(2); d.dim_k = q.size(3);
    d.v_heads = v.size(2); d.dim_v = v.size(3);
    const int64_t batch = d.batch, seqlen = d.seqlen, heads = d.heads, v_heads = d.v_heads, dim_k = d.dim_k, dim_v = d.dim_v;
    CHECK_SHAPE(k, batch, seqlen, heads, dim_k);
    CHECK_SHAPE(v, batch, seqlen, v_heads, dim_v);
    CHECK_SHAPE(g, batch, seqlen, v_heads);
    if (opt_beta.has_value()) {
        const at::Tensor &beta = *opt_beta;
        CHECK_SHAPE(beta, batch, seqlen, v_heads);
    }
    TORCH_CHECK(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(), "q, k and v must have the same dtype");
    d.q = rows_of(q); d.k = rows_of(k); d.v = rows_of(v); d.g = g; d.beta = opt_beta;
    return d;
}

#define SET_STRIDES(P, NAME, T) P.NAME##_stride_b = T.stride(0); P.NAME##_stride_l = T.stride(1); P.NAME##_stride_h = T.stride(2)
#define SET_STATE(P, NAME, T) P.NAME##_stride_n = T.stride(0); P.NAME##_stride_h = T.stride(1); P.NAME##_stride_k = T.stride(2)

template <typename P>
void set_inputs(P &p, const DeltaInputs &d, double scale, bool qk_l2norm) {
    p.batch = size32(d.batch, "batch"); p.seqlen = size32(d.seqlen, "seqlen");
    p.heads = size32(d.heads, "heads"); p.v_heads = size32(d.v_heads, "v_heads");
    p.dim_k = size32(d.dim_k, "dim_k"); p.dim_v = size32(d.dim_v, "dim_v");
    p.x_dtype = to_cc1d_dtype(d.q.scalar_type(), "q");
    p.g_dtype = to_cc1d_dtype(d.g.scalar_type(), "g");
    p.beta_dtype = d.beta.has_value() ? to_cc1d_dtype(d.beta->scalar_type(), "beta") : p.g_dtype;
    p.qk_l2norm = qk_l2norm ? 1 : 0;
    p.scale = (float)scale;
    p.q = d.q.data_ptr(); SET_STRIDES(p, q, d.q);
    p.k = d.k.data_ptr(); SET_STRIDES(p, k, d.k);
    p.v = d.v.data_ptr(); SET_STRIDES(p, v, d.v);
    p.g = d.g.data_ptr(); SET_STRIDES(p, g, d.g);
    if (d.beta.has_value()) { p.beta = d.beta->data_ptr(); SET_STRIDES(p, beta, (*d.beta)); }
}

void check_states(const at::Tensor &s, const DeltaInputs &d, int64_t n, const char *what) {
    check_gpu(s, d.q, what);
    TORCH_CHECK(s.scalar_type() == at::kFloat, what, " must be float32");
    TORCH_CHECK(s.sizes() == at::IntArrayRef({n, d.v_heads, d.dim_k, d.dim_v}), what, " must have shape (sequences, v_heads, dim_k, dim_v)");
}

int64_t sequences_of(const DeltaInputs &d, const OptTensor &cu) {
    if (!cu.has_value()) return d.batch;
    check_gpu(*cu, d.q, "cu_seqlens");
    TORCH_CHECK(d.batch == 1, "cu_seqlens needs a batch of 1: sequences packed back to back");
    TORCH_CHECK(cu->dim() == 1 && cu->size(0) >= 1, "cu_seqlens must be (sequences + 1,)");
    TORCH_CHECK(cu->size(0) > 1 || d.seqlen == 0, "cu_seqlens names no sequence, but there are tokens");
    TORCH_CHECK(cu->is_contiguous(), "cu_seqlens must be contiguous");
    TORCH_CHECK(cu->scalar_type() == at::kInt || cu->scalar_type() == at::kLong, "cu_seqlens must be int32 or int64");
    return cu->size(0) - 1;
}

cc1d_delta_params delta_params(const DeltaInputs &d, const OptTensor &init, const OptTensor &cu, double scale, bool qk_l2norm) {
    cc1d_delta_params p = {};
    set_inputs(p, d, scale, qk_l2norm);
    p.sequences = size32(sequences_of(d, cu), "sequences");
    if (cu.has_value()) { p.cu_seqlens = cu->data_ptr(); p.cu_seqlens_is_int64 = cu->scalar_type() == at::kLong ? 1 : 0; }
    if (init.has_value()) {
        check_states(*init, d, p.sequences, "initial_states");
        TORCH_CHECK(unit_last(*init), "initial_states must have unit stride along dim_v");
        p.initial_states = init->data_ptr<float>(); SET_STATE(p, init, (*init));
    }
    return p;
}

// (out, saved): saved is what the backward needs of the forward, empty if not wanted.
std::tuple<at::Tensor, at::Tensor> delta_fwd_run(const Recurrence &of, const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &g, const OptTensor &beta,
                     const OptTensor &initial_states, const OptTensor &cu_seqlens, const OptTensor &final_states_out, double scale, bool qk_l2norm, bool save) {
    const DeltaInputs d = delta_inputs(q, k, v, g, beta);
    OptTensor init = initial_states;
    if (init.has_value()) init = rows_of(*init);
    cc1d_delta_params p = delta_params(d, init, cu_seqlens, scale, qk_l2norm);
    c10::DeviceGuard guard(q.device());
    at::Tensor out = empty_of({d.batch, d.seqlen, d.v_heads, d.dim_v}, d.v.scalar_type(), d.v);
    p.out = out.data_ptr(); SET_STRIDES(p, out, out);
    if (final_states_out.has_value()) {
        const at::Tensor &f = *final_states_out;
        check_states(f, d, p.sequences, "final_states_out");
        TORCH_CHECK(unit_last(f), "final_states_out must have unit stride along dim_v");
        p.final_states = f.data_ptr<float>(); SET_STATE(p, final, f);
    }
    size_t bytes = 0;
    at::Tensor saved;
    if (save) {
        check_status(of.saved_bytes(&p, &bytes), of.name);
        saved = empty_of({(int64_t)bytes}, at::kByte, q);
        p.saved = bytes ? saved.data_ptr() : nullptr;
    }
    check_status(of.workspace_bytes(&p, &bytes), of.name);
    const at::Tensor ws = workspace_of(bytes, q);
    check_status(of.fwd(&p, bytes ? ws.data_ptr() : nullptr, bytes, current_stream()), of.name);
    return {out, saved};
}
at::Tensor delta_fwd(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &g, const at::Tensor &beta,
                     const OptTensor &initial_states, const OptTensor &cu_seqlens, const OptTensor &final_states_out, double scale, bool qk_l2norm) {
    return std::get<0>(delta_fwd_run(kDelta, q, k, v, g, beta, initial_states, cu_seqlens, final_states_out, scale, qk_l2norm, false));
}
std::tuple<at::Tensor, at::Tensor> delta_fwd_save(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &g, const at::Tensor &beta,
                     const OptTensor &initial_states, const OptTensor &cu_seqlens, const OptTensor &final_states_out, double scale, bool qk_l2norm) {
    return delta_fwd_run(kDelta, q, k, v, g, beta, initial_states, cu_seqlens, final_states_out, scale, qk_l2norm, true);
}
at::Tensor linear_fwd(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &g, const OptTensor &beta,
                      const OptTensor &initial_states, const OptTensor &cu_seqlens, const OptTensor &final_states_out, double scale) {
    return std::get<0>(delta_fwd_run(kLinear, q, k, v, g, beta, initial_states, cu_seqlens, final_states_out, scale, false, false));
}
std::tuple<at::Tensor, at::Tensor> linear_fwd_save(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &g, const OptTensor &beta,
                      const OptTensor &initial_states, const OptTensor &cu_seqlens, const OptTensor &final_states_out, double scale) {
    return delta_fwd_run(kLinear, q, k, v, g, beta, initial_states, cu_seqlens, final_states_out, scale, false, true);
}

// dq, dk, dv, dg, dbeta in their inputs' types (dbeta empty without beta), and dinitial_states (empty if not wanted).
using Gradients6 = std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor>;
Gradients6 delta_bwd_run(const Recurrence &of, const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &g, const OptTensor &beta,
                     const OptTensor &initial_states, const OptTensor &cu_seqlens, const at::Tensor &saved, const at::Tensor &dout_,
                     const OptTensor &dfinal_states, double scale, bool qk_l2norm, bool want_dinitial) {
    const DeltaInputs d = delta_inputs(q, k, v, g, beta);
    OptTensor init = initial_states, dfinal = dfinal_states;
    if (init.has_value()) init = rows_of(*init);
    c10::DeviceGuard guard(q.device());
    cc1d_delta_bwd_params p = {};
    p.fwd = delta_params(d, init, cu_seqlens, scale, qk_l2norm);
    size_t bytes = 0;
    check_status(of.saved_bytes(&p.fwd, &bytes), of.name_bwd);
    check_gpu(saved, q, "saved");
    TORCH_CHECK(saved.is_contiguous() && saved.nbytes() >= bytes, "saved is not what the forward returned for these sizes");
    p.fwd.saved = bytes ? saved.data_ptr() : nullptr;
    check_gpu(dout_, q, "dout");
    TORCH_CHECK(dout_.sizes() == v.sizes() && dout_.scalar_type() == v.scalar_type(), "dout must have the shape and dtype of v");
    const at::Tensor dout = rows_of(dout_);
    p.dout = dout.data_ptr(); SET_STRIDES(p, dout, dout);
    if (dfinal.has_value()) {
        dfinal = rows_of(*dfinal);
        check_states(*dfinal, d, p.fwd.sequences, "dfinal_states");
        p.dfinal_states = dfinal->data_ptr<float>(); SET_STATE(p, dfinal, (*dfinal));
    }
    at::Tensor dq = empty_of(q.sizes(), q.scalar_type(), q), dk = empty_of(k.sizes(), k.scalar_type(), k), dv = empty_of(v.sizes(), v.scalar_type(), v);
    at::Tensor dg = empty_of(g.sizes(), g.scalar_type(), g), dbeta = beta.has_value() ? empty_of(beta->sizes(), beta->scalar_type(), q) : empty_of({0}, at::kFloat, q);
    p.dq = dq.data_ptr(); SET_STRIDES(p, dq, dq);
    p.dk = dk.data_ptr(); SET_STRIDES(p, dk, dk);
    p.dv = dv.data_ptr(); SET_STRIDES(p, dv, dv);
    p.dg = dg.data_ptr(); p.dbeta = beta.has_value() ? dbeta.data_ptr() : nullptr;
    at::Tensor dinit = want_dinitial ? empty_of({p.fwd.sequences, d.v_heads, d.dim_k, d.dim_v}, at::kFloat, q) : empty_of({0}, at::kFloat, q);
    if (want_dinitial) { p.dinitial_states = dinit.data_ptr<float>(); SET_STATE(p, dinit, dinit); }
    check_status(of.bwd_workspace_bytes(&p, &bytes), of.name_bwd);
    const at::Tensor ws = workspace_of(bytes, q);
    check_status(of.bwd(&p, bytes ? ws.data_ptr() : nullptr, bytes, current_stream()), of.name_bwd);
    return {dq, dk, dv, dg, dbeta, dinit};
}
Gradients6 delta_bwd(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &g, const at::Tensor &beta,
                     const OptTensor &initial_states, const OptTensor &cu_seqlens, const at::Tensor &saved, const at::Tensor &dout,
                     const OptTensor &dfinal_states, double scale, bool qk_l2norm, bool want_dinitial) {
    return delta_bwd_run(kDelta, q, k, v, g, beta, initial_states, cu_seqlens, saved, dout, dfinal_states, scale, qk_l2norm, want_dinitial);
}
Gradients6 linear_bwd(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &g, const OptTensor &beta,
                      const OptTensor &initial_states, const OptTensor &cu_seqlens, const at::Tensor &saved, const at::Tensor &dout,
                      const OptTensor &dfinal_states, double scale, bool want_dinitial) {
    return delta_bwd_run(kLinear, q, k, v, g, beta, initial_states, cu_seqlens, saved, dout, dfinal_states, scale, false, want_dinitial);
}

at::Tensor delta_update_run(const Recurrence &of, const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &g, const OptTensor &beta,
                        at::Tensor &state, const OptTensor &state_indices, double scale, bool qk_l2norm) {
    const bool flat = q.dim() == 3;                      // (batch, heads, dim): one token, no seqlen axis
    auto with_tokens = [&](const at::Tensor &t) { return flat ? t.unsqueeze(1) : t; };
    const DeltaInputs d = delta_inputs(with_tokens(q), with_tokens(k), with_tokens(v), with_tokens(g), beta.has_value() ? OptTensor(with_tokens(*beta)) : std::nullopt);
    cc1d_delta_step_params p = {};
    set_inputs(p, d, scale, qk_l2norm);
    check_gpu(state, q, "state");
    TORCH_CHECK(state.dim() == 4, "state must be (slots, v_heads, dim_k, dim_v)");
    check_states(state, d, state_indices.has_value() ? state.size(0) : d.batch, "state");
    TORCH_CHECK(unit_last(state), "state must have unit stride along dim_v");
    p.state_slots = size32(state.size(0), "state slots");
    p.state = state.data_ptr<float>(); SET_STATE(p, state, state);
    if (state_indices.has_value()) {
        const at::Tensor &i = *state_indices;
        check_gpu(i, q, "state_indices");
        TORCH_CHECK(i.scalar_type() == at::kInt, "state_indices must be int32");
        TORCH_CHECK(i.dim() == 1 && i.size(0) == d.batch && i.is_contiguous(), "state_indices must be (batch,), contiguous");
        p.state_indices = i.data_ptr<int32_t>();
    }
    c10::DeviceGuard guard(q.device());
    at::Tensor out = empty_of({d.batch, d.seqlen, d.v_heads, d.dim_v}, d.v.scalar_type(), d.v);
    p.out = out.data_ptr(); SET_STRIDES(p, out, out);
    check_status(of.step(&p, current_stream()), of.name_update);
    return flat ? out.squeeze(1) : out;
}
at::Tensor delta_update(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &g, const at::Tensor &beta,
                        at::Tensor &state, const OptTensor &state_indices, double scale, bool qk_l2norm) {
    return delta_update_run(kDelta, q, k, v, g, beta, state, state_indices, scale, qk_l2norm);
}
at::Tensor linear_update(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &g, at::Tensor &state,
                         const OptTensor &beta, const OptTensor &state_indices, double scale) {
    return delta_update_run(kLinear, q, k, v, g, beta, state, state_indices, scale, false);
}

at::Tensor delta_fwd_meta(const at::Tensor &, const at::Tensor &, const at::Tensor &v, const at::Tensor &, const at::Tensor &,
                          const OptTensor &, const OptTensor &, const OptTensor &, double, bool) {
    return at::empty_symint(v.sym_sizes(), v.options());
}
// How many bytes are saved shows only in the sizes that the kernel library lays out: the same sum.
std::tuple<at::Tensor, at::Tensor> delta_fwd_save_meta(const at::Tensor &q, const at::Tensor &, const at::Tensor &v, const at::Tensor &, const at::Tensor &,
                          const OptTensor &, const OptTensor &cu, const OptTensor &, double, bool) {
    const c10::SymInt chunks = (q.sym_size(1) + 63) / 64;
    const c10::SymInt slots = cu.has_value() ? q.sym_size(1) / 64 + cu->sym_size(0) : q.sym_size(0) * chunks;
    const c10::SymInt one = slots * v.sym_size(2) * v.sym_size(3) * 4, up = 255;
    const c10::SymInt bytes = (one * q.sym_size(3) + up) / 256 * 256 + (one * 64 + up) / 256 * 256;
    return {at::empty_symint(v.sym_sizes(), v.options()), at::empty_symint({bytes}, q.options().dtype(at::kByte))};
}
Gradients6 delta_bwd_meta(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &g, const at::Tensor &beta,
                          const OptTensor &, const OptTensor &cu, const at::Tensor &, const at::Tensor &, const OptTensor &, double, bool, bool want_dinitial) {
    auto like = [](const at::Tensor &t) { return at::empty_symint(t.sym_sizes(), t.options()); };
    const c10::SymInt n = cu.has_value() ? cu->sym_size(0) - 1 : q.sym_size(0);
    const auto f32 = q.options().dtype(at::kFloat);
    return {like(q), like(k), like(v), like(g), like(beta),
            want_dinitial ? at::empty_symint({n, v.sym_size(2), q.sym_size(3), v.sym_size(3)}, f32) : at::empty({0}, f32)};
}
at::Tensor delta_update_meta(const at::Tensor &, const at::Tensor &, const at::Tensor &v, const at::Tensor &, const at::Tensor &,
                             at::Tensor &, const OptTensor &, double, bool) {
    return at::empty_symint(v.sym_sizes(), v.options());
}
at::Tensor linear_fwd_meta(const at::Tensor &, const at::Tensor &, const at::Tensor &v, const at::Tensor &, const OptTensor &,
                           const OptTensor &, const OptTensor &, const OptTensor &, double) {
    return at::empty_symint(v.sym_sizes(), v.options());
}
// Three terms of 16 bits of every state between two segments of 256 tokens (with initial states: in front of every segment), in operands of 32 rows of dim_v and 16 columns of dim_k, whose number is
// whole to 2, 4 or 8 of them: the library's sum.
std::tuple<at::Tensor, at::Tensor> linear_fwd_save_meta(const at::Tensor &q, const at::Tensor &, const at::Tensor &v, const at::Tensor &, const OptTensor &,
                           const OptTensor &init, const OptTensor &cu, const OptTensor &, double) {
    const c10::SymInt chunks = (q.sym_size(1) + 255) / 256;
    const c10::SymInt states = !init.has_value() ? q.sym_size(0) * (chunks.max(1) - 1) : cu.has_value() ? q.sym_size(1) / 256 + cu->sym_size(0) : q.sym_size(0) * chunks;
    const int64_t dk = q.sym_size(3).guard_int(__FILE__, __LINE__), dv = v.sym_size(3).guard_int(__FILE__, __LINE__);
    const int64_t width = q.scalar_type() == at::kFloat || dk > 128 || dv > 128 ? 2 : dk <= 64 ? 4 : 8;
    const c10::SymInt bytes = 256 + states * v.sym_size(2) * ((dv + 31) / 32) * ((dk + 16 * width - 1) / (16 * width) * width) * 3 * 1024;
    return {at::empty_symint(v.sym_sizes(), v.options()), at::empty_symint({bytes}, q.options().dtype(at::kByte))};
}
Gradients6 linear_bwd_meta(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &g, const OptTensor &beta,
                           const OptTensor &init, const OptTensor &cu, const at::Tensor &saved, const at::Tensor &dout, const OptTensor &dfinal, double scale, bool want_dinitial) {
    return delta_bwd_meta(q, k, v, g, beta.has_value() ? *beta : at::empty({0}, q.options().dtype(at::kFloat)), init, cu, saved, dout, dfinal, scale, false, want_dinitial);
}
at::Tensor linear_update_meta(const at::Tensor &, const at::Tensor &, const at::Tensor &v, const at::Tensor &, at::Tensor &,
                              const OptTensor &, const OptTensor &, double) {
    return at::empty_symint(v.sym_sizes(), v.options());
}

// ---- root-mean-square norm -----------------------------------------------------------

// (rows, dim) view of t (..., dim) with one stride between rows, a copy where there is none.
at::Tensor as_rows(const at::Tensor &t) {
    TORCH_CHECK(t.dim() >= 1, "x must have at least one dimension");
    const int64_t dim = t.size(-1);
    int64_t rows = 1;
    for (int64_t i = 0; i + 1 < t.dim(); ++i) rows *= t.size(i);
    return rows_of(t.dim() == 2 ? t : t.reshape({rows, dim}));
}

struct NormInputs { at::Tensor x, residual, weight; };
NormInputs norm_inputs(const at::Tensor &x, const at::Tensor &weight, const OptTensor &residual) {
    check_gpu(x, x, "x"); check_gpu(weight, x, "weight");
    NormInputs n;
    n.x = as_rows(x);
    const int64_t dim = n.x.size(1);
    CHECK_SHAPE(weight, dim);
    n.weight = weight.contiguous();
    TORCH_CHECK(weight.scalar_type() == x.scalar_type() || weight.scalar_type() == at::kFloat, "weight must have the dtype of x or float32");
    if (residual.has_value()) {
        check_gpu(*residual, x, "residual");
        TORCH_CHECK(residual->sizes() == x.sizes(), "residual must have the shape of x");
        TORCH_CHECK(residual->scalar_type() == x.scalar_type() || residual->scalar_type() == at::kFloat, "residual must have the dtype of x or float32");
        n.residual = as_rows(*residual);
    }
    return n;
}

// y or (y8, scales), and h where there is a residual (else an empty tensor).
std::tuple<at::Tensor, at::Tensor, at::Tensor> norm_run(const at::Tensor &x, const at::Tensor &weight, const OptTensor &residual, double eps, bool quantised) {
    const NormInputs n = norm_inputs(x, weight, residual);
    c10::DeviceGuard guard(x.device());
    cc1d_norm_params p = {};
    p.rows = n.x.size(0); p.dim = size32(n.x.size(1), "dim"); p.eps = (float)eps;
    p.x_dtype = p.r_dtype = to_cc1d_dtype(x.scalar_type(), "x");
    p.w_dtype = to_cc1d_dtype(weight.scalar_type(), "weight");
    p.x = n.x.data_ptr(); p.x_stride = n.x.stride(0);
    p.weight = n.weight.data_ptr();
    at::Tensor h, scales;
    if (residual.has_value()) {
        p.r_dtype = to_cc1d_dtype(residual->scalar_type(), "residual");
        p.residual = n.residual.data_ptr(); p.residual_stride = n.residual.stride(0);
        h = empty_of(x.sizes(), residual->scalar_type(), x);
        p.h = h.data_ptr(); p.h_stride = p.dim;
    } else {
        h = empty_of({0}, x.scalar_type(), x);
    }
    at::Tensor y = empty_of(x.sizes(), quantised ? at::kFloat8_e4m3fn : x.scalar_type(), x);
    if (quantised) {
        scales = empty_of(x.sizes().slice(0, x.dim() - 1), at::kFloat, x);
        if (p.dim == 0) scales.zero_();
        p.y8 = y.data_ptr(); p.y8_stride = p.dim; p.scales = scales.data_ptr<float>();
    } else {
        p.y = y.data_ptr(); p.y_stride = p.dim;
    }
    check_status(cc1d_norm_fwd(&p, current_stream()), "rms_norm");
    return {y, scales, h};
}

std::tuple<at::Tensor, at::Tensor> norm_fwd(const at::Tensor &x, const at::Tensor &weight, const OptTensor &residual, double eps) {
    auto r = norm_run(x, weight, residual, eps, false);
    return {std::get<0>(r), std::get<2>(r)};
}
std::tuple<at::Tensor, at::Tensor, at::Tensor> norm_quant(const at::Tensor &x, const at::Tensor &weight, const OptTensor &residual, double eps) {
    return norm_run(x, weight, residual, eps, true);
}

// h: what was normalised.  dx in the dtype of dy, dresidual in that of h; where the two are the same type they are
// one tensor, and dresidual comes back empty.
std::tuple<at::Tensor, at::Tensor, at::Tensor> norm_bwd(const at::Tensor &h, const at::Tensor &weight, const at::Tensor &dy, const OptTensor &dh, double eps) {
    check_gpu(h, h, "h"); check_gpu(weight, h, "weight"); check_gpu(dy, h, "dy");
    TORCH_CHECK(dy.sizes() == h.sizes(), "dy must have the shape of h");
    const at::Tensor hr = as_rows(h), dyr = as_rows(dy), w = weight.contiguous();
    const int64_t dim = hr.size(1);
    CHECK_SHAPE(weight, dim);
    c10::DeviceGuard guard(h.device());
    cc1d_norm_bwd_params p = {};
    p.rows = hr.size(0); p.dim = size32(dim, "dim"); p.eps = (float)eps;
    p.x_dtype = to_cc1d_dtype(dy.scalar_type(), "dy");
    p.r_dtype = to_cc1d_dtype(h.scalar_type(), "h");
    p.w_dtype = to_cc1d_dtype(weight.scalar_type(), "weight");
    p.h = hr.data_ptr(); p.h_stride = hr.stride(0);
    p.weight = w.data_ptr();
    p.dy = dyr.data_ptr(); p.dy_stride = dyr.stride(0);
    at::Tensor dhr;
    if (dh.has_value()) {
        check_gpu(*dh, h, "dh");
        TORCH_CHECK(dh->sizes() == h.sizes() && dh->scalar_type() == h.scalar_type(), "dh must have the shape and dtype of h");
        dhr = as_rows(*dh);
        p.dh = dhr.data_ptr(); p.dh_stride = dhr.stride(0);
    }
    at::Tensor dx = empty_of(h.sizes(), dy.scalar_type(), h);
    p.dx = dx.data_ptr(); p.dx_stride = dim;
    const bool both = dy.scalar_type() != h.scalar_type();
    at::Tensor dres = both ? empty_of(h.sizes(), h.scalar_type(), h) : empty_of({0}, h.scalar_type(), h);
    if (both) { p.dresidual = dres.data_ptr(); p.dresidual_stride = dim; }
    at::Tensor dw = empty_of({dim}, weight.scalar_type(), h);
    p.dweight = dw.data_ptr();
    size_t bytes = 0;
    check_status(cc1d_norm_bwd_workspace_bytes(&p, &bytes), "rms_norm backward");
    const at::Tensor ws = workspace_of(bytes, h);
    check_status(cc1d_norm_bwd(&p, bytes ? ws.data_ptr() : nullptr, bytes, current_stream()), "rms_norm backward");
    return {dx, dres, dw};
}

// ---- layer norm ----------------------------------------------------------------------

const OptTensor &checked_bias(const OptTensor &bias, const at::Tensor &weight, int64_t dim) {
    if (bias.has_value()) {
        check_gpu(*bias, weight, "bias");
        TORCH_CHECK(bias->sizes() == at::IntArrayRef({dim}), "bias must have shape (dim)");
        TORCH_CHECK(bias->scalar_type() == weight.scalar_type(), "bias must have the dtype of weight");
    }
    return bias;
}

// y, h where there is a residual (else empty), and with `save` each row's mean and 1 / standard deviation (else empty).
std::tuple<at::Tensor, at::Tensor, at::Tensor> layer_norm_fwd(const at::Tensor &x, const at::Tensor &weight, const OptTensor &bias_, const OptTensor &residual, double eps, bool save) {
    const NormInputs n = norm_inputs(x, weight, residual);
    c10::DeviceGuard guard(x.device());
    const OptTensor bias = checked_bias(bias_, weight, n.x.size(1));
    cc1d_layer_norm_params p = {};
    p.rows = n.x.size(0); p.dim = size32(n.x.size(1), "dim"); p.eps = (float)eps;
    p.x_dtype = p.r_dtype = to_cc1d_dtype(x.scalar_type(), "x");
    p.w_dtype = to_cc1d_dtype(weight.scalar_type(), "weight");
    p.x = n.x.data_ptr(); p.x_stride = n.x.stride(0);
    p.weight = n.weight.data_ptr();
    at::Tensor b, h, stats = empty_of({save ? p.rows : 0, 2}, at::kFloat, x);
    if (bias.has_value()) { b = bias->contiguous(); p.bias = b.data_ptr(); }
    if (residual.has_value()) {
        p.r_dtype = to_cc1d_dtype(residual->scalar_type(), "residual");
        p.residual = n.residual.data_ptr(); p.residual_stride = n.residual.stride(0);
        h = empty_of(x.sizes(), residual->scalar_type(), x);
        p.h = h.data_ptr(); p.h_stride = p.dim;
    } else {
        h = empty_of({0}, x.scalar_type(), x);
    }
    if (save && p.rows > 0) p.stats = stats.data_ptr<float>();
    at::Tensor y = empty_of(x.sizes(), x.scalar_type(), x);
    p.y = y.data_ptr(); p.y_stride = p.dim;
    check_status(cc1d_layer_norm_fwd(&p, current_stream()), "layer_norm");
    return {y, h, stats};
}

// h: what was normalised.  dx in the dtype of dy, dresidual in that of h; where the two are the same type they are one tensor, and
// dresidual comes back empty.  dbias in the dtype of weight, empty if not wanted.
using Gradients4 = std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor>;
Gradients4 layer_norm_bwd(const at::Tensor &h, const at::Tensor &stats, const at::Tensor &weight, const at::Tensor &dy, const OptTensor &dh, bool want_dbias) {
    check_gpu(h, h, "h"); check_gpu(stats, h, "stats"); check_gpu(weight, h, "weight"); check_gpu(dy, h, "dy");
    TORCH_CHECK(dy.sizes() == h.sizes(), "dy must have the shape of h");
    const at::Tensor hr = as_rows(h), dyr = as_rows(dy), w = weight.contiguous();
    const int64_t dim = hr.size(1);
    CHECK_SHAPE(weight, dim);
    TORCH_CHECK(stats.is_contiguous() && stats.scalar_type() == at::kFloat && stats.numel() == 2 * hr.size(0), "stats is not what the forward returned for these sizes");
    c10::DeviceGuard guard(h.device());
    cc1d_layer_norm_bwd_params p = {};
    p.rows = hr.size(0); p.dim = size32(dim, "dim");
    p.x_dtype = to_cc1d_dtype(dy.scalar_type(), "dy");
    p.r_dtype = to_cc1d_dtype(h.scalar_type(), "h");
    p.w_dtype = to_cc1d_dtype(weight.scalar_type(), "weight");
    p.h = hr.data_ptr(); p.h_stride = hr.stride(0);
    p.stats = stats.data_ptr<float>();
    p.weight = w.data_ptr();
    p.dy = dyr.data_ptr(); p.dy_stride = dyr.stride(0);
    at::Tensor dhr;
    if (dh.has_value()) {
        check_gpu(*dh, h, "dh");
        TORCH_CHECK(dh->sizes() == h.sizes() && dh->scalar_type() == h.scalar_type(), "dh must have the shape and dtype of h");
        dhr = as_rows(*dh);
        p.dh = dhr.data_ptr(); p.dh_stride = dhr.stride(0);
    }
    at::Tensor dx = empty_of(h.sizes(), dy.scalar_type(), h);
    p.dx = dx.data_ptr(); p.dx_stride = dim;
    const bool both = dy.scalar_type() != h.scalar_type();
    at::Tensor dres = both ? empty_of(h.sizes(), h.scalar_type(), h) : empty_of({0}, h.scalar_type(), h);
    if (both) { p.dresidual = dres.data_ptr(); p.dresidual_stride = dim; }
    at::Tensor dw = empty_of({dim}, weight.scalar_type(), h), db = empty_of({want_dbias ? dim : 0}, weight.scalar_type(), h);
    p.dweight = dw.data_ptr();
    if (want_dbias) p.dbias = db.data_ptr();
    size_t bytes = 0;
    check_status(cc1d_layer_norm_bwd_workspace_bytes(&p, &bytes), "layer_norm backward");
    const at::Tensor ws = workspace_of(bytes, h);
    check_status(cc1d_layer_norm_bwd(&p, bytes ? ws.data_ptr() : nullptr, bytes, current_stream()), "layer_norm backward");
    return {dx, dres, dw, db};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> layer_norm_fwd_meta(const at::Tensor &x, const at::Tensor &, const OptTensor &, const OptTensor &residual, double, bool save) {
    c10::SymInt rows = 1;
    for (int64_t i = 0; i + 1 < x.dim(); ++i) rows *= x.sym_size(i);
    return {at::empty_symint(x.sym_sizes(), x.options()), residual.has_value() ? at::empty_symint(x.sym_sizes(), residual->options()) : at::empty({0}, x.options()),
            at::empty_symint({save ? rows : c10::SymInt(0), 2}, x.options().dtype(at::kFloat))};
}
Gradients4 layer_norm_bwd_meta(const at::Tensor &h, const at::Tensor &, const at::Tensor &weight, const at::Tensor &dy, const OptTensor &, bool want_dbias) {
    return {at::empty_symint(h.sym_sizes(), dy.options()), dy.scalar_type() != h.scalar_type() ? at::empty_symint(h.sym_sizes(), h.options()) : at::empty({0}, h.options()),
            at::empty_symint(weight.sym_sizes(), weight.options()), want_dbias ? at::empty_symint(weight.sym_sizes(), weight.options()) : at::empty({0}, weight.options())};
}

// ---- rows of 8 bits --------------------------------------------------------------------

at::Tensor dequantize(const at::Tensor &y8, const at::Tensor &scales, at::ScalarType dtype) {
    check_gpu(y8, y8, "y8"); check_gpu(scales, y8, "scales");
    TORCH_CHECK(y8.scalar_type() == at::kFloat8_e4m3fn, "y8 must be float8_e4m3fn");
    TORCH_CHECK(scales.scalar_type() == at::kFloat, "scales must be float32");
    TORCH_CHECK(y8.dim() >= 1 && scales.sizes() == y8.sizes().slice(0, y8.dim() - 1), "scales must have the shape of y8 without its last dimension");
    const at::Tensor r = as_rows(y8), s = scales.contiguous();
    c10::DeviceGuard guard(y8.device());
    at::Tensor y = empty_of(y8.sizes(), dtype, y8);
    cc1d_dequantize_params p = {};
    p.rows = r.size(0); p.dim = size32(r.size(1), "dim"); p.y_dtype = to_cc1d_dtype(dtype, "dtype");
    p.y8 = r.data_ptr(); p.y8_stride = r.stride(0);
    p.scales = s.data_ptr<float>();
    p.y = y.data_ptr(); p.y_stride = p.dim;
    check_status(cc1d_dequantize_rows(&p, current_stream()), "dequantize_rows");
    return y;
}

std::tuple<at::Tensor, at::Tensor> norm_fwd_meta(const at::Tensor &x, const at::Tensor &, const OptTensor &residual, double) {
    return {at::empty_symint(x.sym_sizes(), x.options()), residual.has_value() ? at::empty_symint(x.sym_sizes(), residual->options()) : at::empty({0}, x.options())};
}
std::tuple<at::Tensor, at::Tensor, at::Tensor> norm_quant_meta(const at::Tensor &x, const at::Tensor &, const OptTensor &residual, double) {
    return {at::empty_symint(x.sym_sizes(), x.options().dtype(at::kFloat8_e4m3fn)), at::empty_symint(x.sym_sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat)),
            residual.has_value() ? at::empty_symint(x.sym_sizes(), residual->options()) : at::empty({0}, x.options())};
}
std::tuple<at::Tensor, at::Tensor, at::Tensor> norm_bwd_meta(const at::Tensor &h, const at::Tensor &weight, const at::Tensor &dy, const OptTensor &, double) {
    return {at::empty_symint(h.sym_sizes(), dy.options()), dy.scalar_type() != h.scalar_type() ? at::empty_symint(h.sym_sizes(), h.options()) : at::empty({0}, h.options()),
            at::empty_symint(weight.sym_sizes(), weight.options())};
}
at::Tensor dequantize_meta(const at::Tensor &y8, const at::Tensor &, at::ScalarType dtype) {
    return at::empty_symint(y8.sym_sizes(), y8.options().dtype(dtype));
}

// ---- graphs recorded from C++, and direct calls from Python ---------------------------
// As in causal_conv1d.cpp: the same ops and the same graph without the interpreter in between.  Calls whose host time is longer than
// their kernels': normalising 64 rows and scaling them back 13.2 -> 11.4 us (10.0 by now), forward and
// backward of 777 rows of 1001 64 -> 54.

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
at::Tensor or_undefined(const OptTensor &t) { return t.value_or(at::Tensor()); }
OptTensor if_defined(const at::Tensor &t) { return t.defined() ? OptTensor(t) : std::nullopt; }

// (y, h) or (y): saves what was normalised, and the weight.
struct RMSNormNode : public torch::autograd::Function<RMSNormNode> {
    static variable_list forward(AutogradContext *ctx, const at::Tensor &x, const at::Tensor &weight, const OptTensor &residual, double eps) {
        static const auto op = typed_op<decltype(norm_fwd)>("DaoAILab::_rms_norm_fwd_cpp");
        std::tuple<at::Tensor, at::Tensor> r;
        {
            pybind11::gil_scoped_release no_gil;
            r = op.call(x, weight, residual, eps);
        }
        ctx->save_for_backward({residual.has_value() ? std::get<1>(r) : x, weight});
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["dtype"] = x.scalar_type();
        ctx->saved_data["residual"] = residual.has_value() && residual->requires_grad();
        ctx->set_materialize_grads(false);
        return residual.has_value() ? variable_list{std::get<0>(r), std::get<1>(r)} : variable_list{std::get<0>(r)};
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        static const auto op = typed_op<decltype(norm_bwd)>("DaoAILab::_rms_norm_bwd_cpp");
        const OptTensor dh = grads.size() > 1 ? if_defined(grads[1]) : std::nullopt;
        at::Tensor dy = grads[0];
        if (!dy.defined() && !dh.has_value()) return {at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
        const variable_list saved = ctx->get_saved_variables();
        const at::Tensor &h = saved[0], &weight = saved[1];
        if (!dy.defined()) dy = at::zeros(h.sizes(), h.options().dtype(ctx->saved_data["dtype"].toScalarType()));
        auto r = op.call(h, weight, dy, dh, ctx->saved_data["eps"].toDouble());
        const at::Tensor &dx = std::get<0>(r);
        at::Tensor dresidual;
        if (ctx->saved_data["residual"].toBool()) dresidual = dx.scalar_type() == h.scalar_type() ? dx : std::get<1>(r);
        return {dx, std::get<2>(r), dresidual, at::Tensor()};
    }
};

// (out, final_states) or (out): saves the inputs and what the forward keeps for its backward.
struct GatedDeltaRuleNode : public torch::autograd::Function<GatedDeltaRuleNode> {
    static variable_list forward(AutogradContext *ctx, const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &g, const at::Tensor &beta,
                                 const OptTensor &init, const OptTensor &cu, const OptTensor &final, double scale, bool qk_l2norm) {
        static const auto op = typed_op<decltype(delta_fwd_save)>("DaoAILab::_gated_delta_rule_fwd_save_cpp");
        std::tuple<at::Tensor, at::Tensor> r;
        {
            pybind11::gil_scoped_release no_gil;
            r = op.call(q, k, v, g, beta, init, cu, final, scale, qk_l2norm);
        }
        ctx->save_for_backward({q, k, v, g, beta, or_undefined(init), or_undefined(cu), std::get<1>(r)});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["l2norm"] = qk_l2norm;
        ctx->saved_data["dinit"] = init.has_value() && init->requires_grad();
        ctx->set_materialize_grads(false);
        return final.has_value() ? variable_list{std::get<0>(r), *final} : variable_list{std::get<0>(r)};
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        static const auto op = typed_op<decltype(delta_bwd)>("DaoAILab::_gated_delta_rule_bwd_cpp");
        const OptTensor dfinal = grads.size() > 1 ? if_defined(grads[1]) : std::nullopt;
        at::Tensor dout = grads[0];
        if (!dout.defined() && !dfinal.has_value()) return variable_list(10);
        const variable_list s = ctx->get_saved_variables();
        if (!dout.defined()) dout = at::zeros(s[2].sizes(), s[2].options());
        const bool dinit = ctx->saved_data["dinit"].toBool();
        auto r = op.call(s[0], s[1], s[2], s[3], s[4], if_defined(s[5]), if_defined(s[6]), s[7], dout, dfinal, ctx->saved_data["scale"].toDouble(),
                         ctx->saved_data["l2norm"].toBool(), dinit);
        variable_list all = {std::get<0>(r), std::get<1>(r), std::get<2>(r), std::get<3>(r), std::get<4>(r)};
        all.resize(10);
        if (dinit) all[5] = std::get<5>(r);
        return all;
    }
};

// As GatedDeltaRuleNode; beta may be missing.
struct LinearAttentionNode : public torch::autograd::Function<LinearAttentionNode> {
    static variable_list forward(AutogradContext *ctx, const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &g, const OptTensor &beta,
                                 const OptTensor &init, const OptTensor &cu, const OptTensor &final, double scale) {
        static const auto op = typed_op<decltype(linear_fwd_save)>("DaoAILab::_linear_attention_fwd_save_cpp");
        std::tuple<at::Tensor, at::Tensor> r;
        {
            pybind11::gil_scoped_release no_gil;
            r = op.call(q, k, v, g, beta, init, cu, final, scale);
        }
        ctx->save_for_backward({q, k, v, g, or_undefined(beta), or_undefined(init), or_undefined(cu), std::get<1>(r)});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["dinit"] = init.has_value() && init->requires_grad();
        ctx->set_materialize_grads(false);
        return final.has_value() ? variable_list{std::get<0>(r), *final} : variable_list{std::get<0>(r)};
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        static const auto op = typed_op<decltype(linear_bwd)>("DaoAILab::_linear_attention_bwd_cpp");
        const OptTensor dfinal = grads.size() > 1 ? if_defined(grads[1]) : std::nullopt;
        at::Tensor dout = grads[0];
        if (!dout.defined() && !dfinal.has_value()) return variable_list(9);
        const variable_list s = ctx->get_saved_variables();
        if (!dout.defined()) dout = at::zeros(s[2].sizes(), s[2].options());
        const bool dinit = ctx->saved_data["dinit"].toBool();
        auto r = op.call(s[0], s[1], s[2], s[3], if_defined(s[4]), if_defined(s[5]), if_defined(s[6]), s[7], dout, dfinal, ctx->saved_data["scale"].toDouble(), dinit);
        variable_list all = {std::get<0>(r), std::get<1>(r), std::get<2>(r), std::get<3>(r)};
        all.resize(9);
        if (s[4].defined()) all[4] = std::get<4>(r);
        if (dinit) all[5] = std::get<5>(r);
        return all;
    }
};

// (y, h) or (y): saves what was normalised, its rows' statistics and the weight.
struct LayerNormNode : public torch::autograd::Function<LayerNormNode> {
    static variable_list forward(AutogradContext *ctx, const at::Tensor &x, const at::Tensor &weight, const OptTensor &bias, const OptTensor &residual, double eps) {
        static const auto op = typed_op<decltype(layer_norm_fwd)>("DaoAILab::_layer_norm_fwd_cpp");
        std::tuple<at::Tensor, at::Tensor, at::Tensor> r;
        {
            pybind11::gil_scoped_release no_gil;
            r = op.call(x, weight, bias, residual, eps, true);
        }
        ctx->save_for_backward({residual.has_value() ? std::get<1>(r) : x, std::get<2>(r), weight});
        ctx->saved_data["dtype"] = x.scalar_type();
        ctx->saved_data["residual"] = residual.has_value() && residual->requires_grad();
        ctx->saved_data["bias"] = bias.has_value() && bias->requires_grad();
        ctx->set_materialize_grads(false);
        return residual.has_value() ? variable_list{std::get<0>(r), std::get<1>(r)} : variable_list{std::get<0>(r)};
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        static const auto op = typed_op<decltype(layer_norm_bwd)>("DaoAILab::_layer_norm_bwd_cpp");
        const OptTensor dh = grads.size() > 1 ? if_defined(grads[1]) : std::nullopt;
        at::Tensor dy = grads[0];
        variable_list all(5);
        if (!dy.defined() && !dh.has_value()) return all;
        const variable_list saved = ctx->get_saved_variables();
        const at::Tensor &h = saved[0];
        if (!dy.defined()) dy = at::zeros(h.sizes(), h.options().dtype(ctx->saved_data["dtype"].toScalarType()));
        const bool bias = ctx->saved_data["bias"].toBool();
        auto r = op.call(h, saved[1], saved[2], dy, dh, bias);
        all[0] = std::get<0>(r);
        all[1] = std::get<2>(r);
        if (bias) all[2] = std::get<3>(r);
        if (ctx->saved_data["residual"].toBool()) all[3] = all[0].scalar_type() == h.scalar_type() ? all[0] : std::get<1>(r);
        return all;
    }
};

bool wants_grad(std::initializer_list<const at::Tensor *> all) {
    if (!at::GradMode::is_enabled()) return false;
    for (const at::Tensor *t : all)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}
bool python_graph_needed(std::initializer_list<const at::Tensor *> all) {
    if (functorch_active()) return true;
    for (const at::Tensor *t : all)
        if (t->defined() && ::python_graph_needed(OptTensor(*t))) return true;
    return false;
}
PyObject *tuple_of(variable_list &&all) {
    PyObject *t = PyTuple_New((Py_ssize_t)all.size());
    if (t == nullptr) throw python_error();
    for (size_t i = 0; i < all.size(); ++i) PyTuple_SET_ITEM(t, (Py_ssize_t)i, THPVariable_Wrap(std::move(all[i])));
    return t;
}
bool plain_all(PyObject *const *a, int n) {
    for (int i = 0; i < n; ++i)
        if (!plain(a[i])) return false;
    return true;
}

// (x, weight, residual, eps) -> y or (y, h)
PyObject *norm_call(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 4 || !plain_all(a, 2) || !plain_or_none(a[2]) || !PyFloat_Check(a[3]) || generic_path_needed()) NOT_IMPLEMENTED();
    static const auto op = typed_op<decltype(norm_fwd)>("DaoAILab::_rms_norm_fwd_cpp");
    const at::Tensor x = THPVariable_Unpack(a[0]), weight = THPVariable_Unpack(a[1]);
    const OptTensor residual = optional_tensor(a[2]);
    const double eps = PyFloat_AS_DOUBLE(a[3]);
    const at::Tensor r = or_undefined(residual);
    variable_list all;
    if (wants_grad({&x, &weight, &r})) {
        if (python_graph_needed({&x, &weight, &r})) NOT_IMPLEMENTED();
        all = RMSNormNode::apply(x, weight, residual, eps);
    } else {
        pybind11::gil_scoped_release no_gil;
        auto t = op.call(x, weight, residual, eps);
        all = residual.has_value() ? variable_list{std::get<0>(t), std::get<1>(t)} : variable_list{std::get<0>(t)};
    }
    return residual.has_value() ? tuple_of(std::move(all)) : THPVariable_Wrap(std::move(all[0]));
    END_HANDLE_TH_ERRORS
}

// (x, weight, bias, residual, eps) -> y or (y, h)
PyObject *layer_norm_call(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 5 || !plain_all(a, 2) || !plain_or_none(a[2]) || !plain_or_none(a[3]) || !PyFloat_Check(a[4]) || generic_path_needed()) NOT_IMPLEMENTED();
    static const auto op = typed_op<decltype(layer_norm_fwd)>("DaoAILab::_layer_norm_fwd_cpp");
    const at::Tensor x = THPVariable_Unpack(a[0]), weight = THPVariable_Unpack(a[1]);
    const OptTensor bias = optional_tensor(a[2]), residual = optional_tensor(a[3]);
    const double eps = PyFloat_AS_DOUBLE(a[4]);
    const at::Tensor b = or_undefined(bias), r = or_undefined(residual);
    variable_list all;
    if (wants_grad({&x, &weight, &b, &r})) {
        if (python_graph_needed({&x, &weight, &b, &r})) NOT_IMPLEMENTED();
        all = LayerNormNode::apply(x, weight, bias, residual, eps);
    } else {
        pybind11::gil_scoped_release no_gil;
        auto t = op.call(x, weight, bias, residual, eps, false);
        all = residual.has_value() ? variable_list{std::get<0>(t), std::get<1>(t)} : variable_list{std::get<0>(t)};
    }
    return residual.has_value() ? tuple_of(std::move(all)) : THPVariable_Wrap(std::move(all[0]));
    END_HANDLE_TH_ERRORS
}

// (x, weight, residual, eps) -> (y8, scales) or (y8, scales, h)
PyObject *norm_quant_call(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 4 || !plain_all(a, 2) || !plain_or_none(a[2]) || !PyFloat_Check(a[3]) || generic_path_needed()) NOT_IMPLEMENTED();
    static const auto op = typed_op<decltype(norm_quant)>("DaoAILab::_rms_norm_quant_cpp");
    const at::Tensor x = THPVariable_Unpack(a[0]), weight = THPVariable_Unpack(a[1]), r = or_undefined(optional_tensor(a[2]));
    std::tuple<at::Tensor, at::Tensor, at::Tensor> t;
    {
        pybind11::gil_scoped_release no_gil;
        t = op.call(x, weight, if_defined(r), PyFloat_AS_DOUBLE(a[3]));
    }
    variable_list all = {std::get<0>(t), std::get<1>(t)};
    if (r.defined()) all.push_back(std::get<2>(t));
    return tuple_of(std::move(all));
    END_HANDLE_TH_ERRORS
}

// (y8, scales, dtype) -> y
PyObject *dequantize_call(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 3 || !plain_all(a, 2) || !THPDtype_Check(a[2]) || generic_path_needed()) NOT_IMPLEMENTED();
    static const auto op = typed_op<decltype(dequantize)>("DaoAILab::_dequantize_rows_cpp");
    const at::Tensor y8 = THPVariable_Unpack(a[0]), scales = THPVariable_Unpack(a[1]);
    const at::ScalarType dtype = reinterpret_cast<THPDtype *>(a[2])->scalar_type;
    at::Tensor y;
    {
        pybind11::gil_scoped_release no_gil;
        y = op.call(y8, scales, dtype);
    }
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// (q, k, v, g, beta, state, state_indices, scale or None, qk_l2norm) -> out
PyObject *delta_update_call(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 9 || !plain_all(a, 6) || !plain_or_none(a[6]) || !(a[7] == Py_None || PyFloat_Check(a[7])) || !PyBool_Check(a[8]) || generic_path_needed()) NOT_IMPLEMENTED();
    static const auto op = typed_op<decltype(delta_update)>("DaoAILab::_gated_delta_rule_update_cpp");
    const at::Tensor q = THPVariable_Unpack(a[0]), k = THPVariable_Unpack(a[1]), v = THPVariable_Unpack(a[2]), g = THPVariable_Unpack(a[3]), beta = THPVariable_Unpack(a[4]);
    at::Tensor state = THPVariable_Unpack(a[5]);
    const OptTensor indices = optional_tensor(a[6]);
    if (q.dim() < 1) NOT_IMPLEMENTED();
    const double scale = a[7] == Py_None ? 1.0 / std::sqrt((double)q.size(-1)) : PyFloat_AS_DOUBLE(a[7]);
    at::Tensor out;
    {
        pybind11::gil_scoped_release no_gil;
        out = op.call(q, k, v, g, beta, state, indices, scale, a[8] == Py_True);
    }
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// (q, k, v, g, beta, scale or None, initial_states, return_final_states, final_states_out, cu_seqlens, qk_l2norm)
// -> out or (out, final_states)
PyObject *delta_call(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 11 || !plain_all(a, 5) || !(a[5] == Py_None || PyFloat_Check(a[5])) || !plain_or_none(a[6]) || !PyBool_Check(a[7]) || !plain_or_none(a[8]) ||
        !plain_or_none(a[9]) || !PyBool_Check(a[10]) || generic_path_needed())
        NOT_IMPLEMENTED();
    static const auto op = typed_op<decltype(delta_fwd)>("DaoAILab::_gated_delta_rule_fwd_cpp");
    const at::Tensor q = THPVariable_Unpack(a[0]), k = THPVariable_Unpack(a[1]), v = THPVariable_Unpack(a[2]), g = THPVariable_Unpack(a[3]), beta = THPVariable_Unpack(a[4]);
    const OptTensor init = optional_tensor(a[6]), cu = optional_tensor(a[9]);
    const bool return_final = a[7] == Py_True, l2norm = a[10] == Py_True;
    OptTensor fin = return_final ? optional_tensor(a[8]) : std::nullopt;
    if (q.dim() != 4 || v.dim() != 4 || (cu.has_value() && (cu->dim() != 1 || cu->size(0) < 1 || !cu->is_contiguous()))) NOT_IMPLEMENTED();
    const double scale = a[5] == Py_None ? 1.0 / std::sqrt((double)q.size(-1)) : PyFloat_AS_DOUBLE(a[5]);
    const at::Tensor i = or_undefined(init);
    const bool graph = wants_grad({&q, &k, &v, &g, &beta, &i});
    if (graph && (fin.has_value() || python_graph_needed({&q, &k, &v, &g, &beta, &i}))) NOT_IMPLEMENTED();
    if (return_final && !fin.has_value())
        fin = at::empty({cu.has_value() ? cu->size(0) - 1 : q.size(0), v.size(2), q.size(3), v.size(3)}, v.options().dtype(at::kFloat));
    variable_list all;
    if (graph) {
        all = GatedDeltaRuleNode::apply(q, k, v, g, beta, init, cu, fin, scale, l2norm);
    } else {
        pybind11::gil_scoped_release no_gil;
        all.push_back(op.call(q, k, v, g, beta, init, cu, fin, scale, l2norm));
    }
    if (!return_final) return THPVariable_Wrap(std::move(all[0]));
    if (a[8] != Py_None) {                               // the caller's own object
        PyObject *pair = PyTuple_New(2);
        if (pair == nullptr) throw python_error();
        PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(std::move(all[0])));
        Py_INCREF(a[8]);
        PyTuple_SET_ITEM(pair, 1, a[8]);
        return pair;
    }
    if (!graph) all.push_back(*fin);
    return tuple_of(std::move(all));
    END_HANDLE_TH_ERRORS
}

// (q, k, v, g, state, beta, state_indices, scale or None) -> out
PyObject *linear_update_call(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 8 || !plain_all(a, 5) || !plain_or_none(a[5]) || !plain_or_none(a[6]) || !(a[7] == Py_None || PyFloat_Check(a[7])) || generic_path_needed()) NOT_IMPLEMENTED();
    static const auto op = typed_op<decltype(linear_update)>("DaoAILab::_linear_attention_update_cpp");
    const at::Tensor q = THPVariable_Unpack(a[0]), k = THPVariable_Unpack(a[1]), v = THPVariable_Unpack(a[2]);
    at::Tensor g = THPVariable_Unpack(a[3]), state = THPVariable_Unpack(a[4]);
    const OptTensor beta = optional_tensor(a[5]), indices = optional_tensor(a[6]);
    if (q.dim() < 1 || (g.dim() == 1 && v.dim() < 3)) NOT_IMPLEMENTED();
    const double scale = a[7] == Py_None ? 1.0 / std::sqrt((double)q.size(-1)) : PyFloat_AS_DOUBLE(a[7]);
    at::Tensor out;
    {
        pybind11::gil_scoped_release no_gil;
        if (g.dim() == 1) g = g.expand(v.sizes().slice(0, v.dim() - 1));
        out = op.call(q, k, v, g, state, beta, indices, scale);
    }
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// (q, k, v, g, beta, scale or None, initial_states, return_final_states, final_states_out, cu_seqlens) -> out or (out, final_states)
PyObject *linear_call(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 10 || !plain_all(a, 4) || !plain_or_none(a[4]) || !(a[5] == Py_None || PyFloat_Check(a[5])) || !plain_or_none(a[6]) || !PyBool_Check(a[7]) ||
        !plain_or_none(a[8]) || !plain_or_none(a[9]) || generic_path_needed())
        NOT_IMPLEMENTED();
    static const auto op = typed_op<decltype(linear_fwd)>("DaoAILab::_linear_attention_fwd_cpp");
    const at::Tensor q = THPVariable_Unpack(a[0]), k = THPVariable_Unpack(a[1]), v = THPVariable_Unpack(a[2]);
    at::Tensor g = THPVariable_Unpack(a[3]);
    const OptTensor beta = optional_tensor(a[4]), init = optional_tensor(a[6]), cu = optional_tensor(a[9]);
    const bool return_final = a[7] == Py_True;
    OptTensor fin = return_final ? optional_tensor(a[8]) : std::nullopt;
    if (q.dim() != 4 || v.dim() != 4 || (cu.has_value() && (cu->dim() != 1 || cu->size(0) < 1 || !cu->is_contiguous()))) NOT_IMPLEMENTED();
    const double scale = a[5] == Py_None ? 1.0 / std::sqrt((double)q.size(-1)) : PyFloat_AS_DOUBLE(a[5]);
    const at::Tensor b = or_undefined(beta), i = or_undefined(init);
    const bool graph = wants_grad({&q, &k, &v, &g, &b, &i});
    if (graph && (fin.has_value() || python_graph_needed({&q, &k, &v, &g, &b, &i}))) NOT_IMPLEMENTED();
    if (g.dim() == 1) g = g.expand(v.sizes().slice(0, 3));
    if (return_final && !fin.has_value())
        fin = at::empty({cu.has_value() ? cu->size(0) - 1 : q.size(0), v.size(2), q.size(3), v.size(3)}, v.options().dtype(at::kFloat));
    variable_list all;
    if (graph) {
        all = LinearAttentionNode::apply(q, k, v, g, beta, init, cu, fin, scale);
    } else {
        pybind11::gil_scoped_release no_gil;
        all.push_back(op.call(q, k, v, g, beta, init, cu, fin, scale));
    }
    if (!return_final) return THPVariable_Wrap(std::move(all[0]));
    if (a[8] != Py_None) {                               // the caller's own object
        PyObject *pair = PyTuple_New(2);
        if (pair == nullptr) throw python_error();
        PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(std::move(all[0])));
        Py_INCREF(a[8]);
        PyTuple_SET_ITEM(pair, 1, a[8]);
        return pair;
    }
    if (!graph) all.push_back(*fin);
    return tuple_of(std::move(all));
    END_HANDLE_TH_ERRORS
}

// ---- what autograd is told of an op ----------------------------------------------------
// The graphs above (and those of the Python functions) are recorded around the ops, with gradients off inside.  An op that is called on
// tensors that require a gradient all the same (the backward under create_graph, or the op itself) has no derivative: its results
// say so when somebody asks for one, where the dispatcher's fallback would give zeros and a warning.  A tangent would be lost here
// without a trace, so it is refused.

template <typename T> void add_edge(torch::autograd::edge_list &, const T &) {}
void add_edge(torch::autograd::edge_list &all, const at::Tensor &t) {
    if (t.defined() && t.requires_grad()) all.push_back(torch::autograd::impl::gradient_edge(t));
}
void add_edge(torch::autograd::edge_list &all, const OptTensor &t) { if (t.has_value()) add_edge(all, *t); }

template <typename T> void refuse_tangent(const char *, const T &) {}
void refuse_tangent(const char *name, const at::Tensor &t) {
    TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(), name, ": forward-mode derivatives (jvp) are not implemented");
}
void refuse_tangent(const char *name, const OptTensor &t) { if (t.has_value()) refuse_tangent(name, *t); }

void end_graph(const at::Tensor &t, const std::shared_ptr<torch::autograd::Node> &node) {
    if (t.defined() && torch::autograd::isDifferentiableType(t.scalar_type())) torch::autograd::set_history(t, node);
}
template <typename... R>
void end_graph(const std::tuple<R...> &all, const std::shared_ptr<torch::autograd::Node> &node) {
    std::apply([&](const R &...t) { (end_graph(t, node), ...); }, all);
}

// What an op writes in place: part of no graph that is being recorded, whose gradients it would make wrong.
void check_written(const char *name, const at::Tensor &t) {
    TORCH_CHECK(!t.defined() || !t.requires_grad() || !at::GradMode::is_enabled(), name, ": a tensor that is written in place requires a gradient");
}
void check_written(const char *name, const OptTensor &t) { if (t.has_value()) check_written(name, *t); }

// As torch's own operators do, so that a graph which has saved the tensor notices.  Tensors made in inference mode count nothing.
void count_write(const at::Tensor &t) { if (t.defined() && !t.is_inference()) torch::autograd::impl::bump_version(t); }
void count_write(const OptTensor &t) { if (t.has_value()) count_write(*t); }

// ENDS: the op has a function that records a graph around it.  The others have no backward: their results belong to no graph.
// WRITTEN: which argument is written in place, or -1.
template <const char *NAME, bool ENDS, int WRITTEN, typename F> struct Graphless;
template <const char *NAME, bool ENDS, int WRITTEN, typename R, typename... A>
struct Graphless<NAME, ENDS, WRITTEN, R(A...)> {
    static R call(A... args) {
        static const auto op = typed_op<R(A...)>(NAME);
        if constexpr (WRITTEN >= 0) check_written(NAME, std::get<WRITTEN>(std::tie(args...)));
        torch::autograd::edge_list edges;
        if constexpr (ENDS) {
            (refuse_tangent(NAME, args), ...);
            if (at::GradMode::is_enabled()) (add_edge(edges, args), ...);
        }
        R r = [&] {
            at::AutoDispatchBelowADInplaceOrView below;
            return op.call(args...);
        }();
        if constexpr (WRITTEN >= 0) count_write(std::get<WRITTEN>(std::tie(args...)));
        if (!edges.empty()) end_graph(r, std::shared_ptr<torch::autograd::Node>(new torch::autograd::NotImplemented(NAME, std::move(edges)), torch::autograd::deleteNode));
        return r;
    }
};
#define OP_NAME(ID, OP) constexpr char ID[] = "DaoAILab::" OP
OP_NAME(kDeltaFwd, "_gated_delta_rule_fwd_cpp");
OP_NAME(kDeltaFwdSave, "_gated_delta_rule_fwd_save_cpp");
OP_NAME(kDeltaBwd, "_gated_delta_rule_bwd_cpp");
OP_NAME(kDeltaUpdate, "_gated_delta_rule_update_cpp");
OP_NAME(kNormFwd, "_rms_norm_fwd_cpp");
OP_NAME(kNormBwd, "_rms_norm_bwd_cpp");
OP_NAME(kNormQuant, "_rms_norm_quant_cpp");
OP_NAME(kDequantize, "_dequantize_rows_cpp");
OP_NAME(kLinearFwd, "_linear_attention_fwd_cpp");
OP_NAME(kLinearFwdSave, "_linear_attention_fwd_save_cpp");
OP_NAME(kLinearBwd, "_linear_attention_bwd_cpp");
OP_NAME(kLinearUpdate, "_linear_attention_update_cpp");
OP_NAME(kLayerNormFwd, "_layer_norm_fwd_cpp");
OP_NAME(kLayerNormBwd, "_layer_norm_bwd_cpp");

#define DIRECT_CALL(NAME, F) {NAME, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&F)), METH_FASTCALL, nullptr}
PyMethodDef calls[] = {DIRECT_CALL("_rms_norm_call", norm_call),
                       DIRECT_CALL("_rms_norm_quant_call", norm_quant_call),
                       DIRECT_CALL("_dequantize_rows_call", dequantize_call),
                       DIRECT_CALL("_gated_delta_rule_call", delta_call),
                       DIRECT_CALL("_gated_delta_rule_update_call", delta_update_call),
                       DIRECT_CALL("_linear_attention_call", linear_call),
                       DIRECT_CALL("_linear_attention_update_call", linear_update_call),
                       DIRECT_CALL("_layer_norm_call", layer_norm_call),
                       {nullptr, nullptr, 0, nullptr}};

}  // namespace

PyMethodDef *mixer_direct_calls() { return calls; }

TORCH_LIBRARY_FRAGMENT(DaoAILab, m) {
    m.def("_gated_delta_rule_fwd_cpp(Tensor q, Tensor k, Tensor v, Tensor g, Tensor beta, Tensor? initial_states, "
          "Tensor? cu_seqlens, Tensor(a!)? final_states_out, float scale, bool qk_l2norm) -> Tensor", {at::Tag::pt2_compliant_tag});
    m.def("_gated_delta_rule_fwd_save_cpp(Tensor q, Tensor k, Tensor v, Tensor g, Tensor beta, Tensor? initial_states, "
          "Tensor? cu_seqlens, Tensor(a!)? final_states_out, float scale, bool qk_l2norm) -> (Tensor, Tensor)", {at::Tag::pt2_compliant_tag});
    m.def("_gated_delta_rule_bwd_cpp(Tensor q, Tensor k, Tensor v, Tensor g, Tensor beta, Tensor? initial_states, Tensor? cu_seqlens, "
          "Tensor saved, Tensor dout, Tensor? dfinal_states, float scale, bool qk_l2norm, bool want_dinitial) "
          "-> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)", {at::Tag::pt2_compliant_tag});
    m.def("_gated_delta_rule_update_cpp(Tensor q, Tensor k, Tensor v, Tensor g, Tensor beta, Tensor(a!) state, "
          "Tensor? state_indices, float scale, bool qk_l2norm) -> Tensor", {at::Tag::pt2_compliant_tag});
    m.def("_rms_norm_fwd_cpp(Tensor x, Tensor weight, Tensor? residual, float eps) -> (Tensor, Tensor)", {at::Tag::pt2_compliant_tag});
    m.def("_rms_norm_bwd_cpp(Tensor h, Tensor weight, Tensor dy, Tensor? dh, float eps) -> (Tensor, Tensor, Tensor)", {at::Tag::pt2_compliant_tag});
    m.def("_rms_norm_quant_cpp(Tensor x, Tensor weight, Tensor? residual, float eps) -> (Tensor, Tensor, Tensor)", {at::Tag::pt2_compliant_tag});
    m.def("_dequantize_rows_cpp(Tensor y8, Tensor scales, ScalarType dtype) -> Tensor", {at::Tag::pt2_compliant_tag});
    m.def("_linear_attention_fwd_cpp(Tensor q, Tensor k, Tensor v, Tensor g, Tensor? beta, Tensor? initial_states, "
          "Tensor? cu_seqlens, Tensor(a!)? final_states_out, float scale) -> Tensor", {at::Tag::pt2_compliant_tag});
    m.def("_linear_attention_fwd_save_cpp(Tensor q, Tensor k, Tensor v, Tensor g, Tensor? beta, Tensor? initial_states, "
          "Tensor? cu_seqlens, Tensor(a!)? final_states_out, float scale) -> (Tensor, Tensor)", {at::Tag::pt2_compliant_tag});
    m.def("_linear_attention_bwd_cpp(Tensor q, Tensor k, Tensor v, Tensor g, Tensor? beta, Tensor? initial_states, Tensor? cu_seqlens, "
          "Tensor saved, Tensor dout, Tensor? dfinal_states, float scale, bool want_dinitial) "
          "-> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)", {at::Tag::pt2_compliant_tag});
    m.def("_linear_attention_update_cpp(Tensor q, Tensor k, Tensor v, Tensor g, Tensor(a!) state, Tensor? beta, "
          "Tensor? state_indices, float scale) -> Tensor", {at::Tag::pt2_compliant_tag});
    m.def("_layer_norm_fwd_cpp(Tensor x, Tensor weight, Tensor? bias, Tensor? residual, float eps, bool save) -> (Tensor, Tensor, Tensor)", {at::Tag::pt2_compliant_tag});
    m.def("_layer_norm_bwd_cpp(Tensor h, Tensor stats, Tensor weight, Tensor dy, Tensor? dh, bool want_dbias) -> (Tensor, Tensor, Tensor, Tensor)", {at::Tag::pt2_compliant_tag});
}

TORCH_LIBRARY_IMPL(DaoAILab, CompositeExplicitAutograd, m) {
    m.impl("_gated_delta_rule_fwd_cpp", &delta_fwd);
    m.impl("_gated_delta_rule_fwd_save_cpp", &delta_fwd_save);
    m.impl("_gated_delta_rule_bwd_cpp", &delta_bwd);
    m.impl("_gated_delta_rule_update_cpp", &delta_update);
    m.impl("_rms_norm_fwd_cpp", &norm_fwd);
    m.impl("_rms_norm_bwd_cpp", &norm_bwd);
    m.impl("_rms_norm_quant_cpp", &norm_quant);
    m.impl("_dequantize_rows_cpp", &dequantize);
    m.impl("_linear_attention_fwd_cpp", &linear_fwd);
    m.impl("_linear_attention_fwd_save_cpp", &linear_fwd_save);
    m.impl("_linear_attention_bwd_cpp", &linear_bwd);
    m.impl("_linear_attention_update_cpp", &linear_update);
    m.impl("_layer_norm_fwd_cpp", &layer_norm_fwd);
    m.impl("_layer_norm_bwd_cpp", &layer_norm_bwd);
}

TORCH_LIBRARY_IMPL(DaoAILab, Meta, m) {
    m.impl("_gated_delta_rule_fwd_cpp", &delta_fwd_meta);
    m.impl("_gated_delta_rule_fwd_save_cpp", &delta_fwd_save_meta);
    m.impl("_gated_delta_rule_bwd_cpp", &delta_bwd_meta);
    m.impl("_gated_delta_rule_update_cpp", &delta_update_meta);
    m.impl("_rms_norm_fwd_cpp", &norm_fwd_meta);
    m.impl("_rms_norm_bwd_cpp", &norm_bwd_meta);
    m.impl("_rms_norm_quant_cpp", &norm_quant_meta);
    m.impl("_dequantize_rows_cpp", &dequantize_meta);
    m.impl("_linear_attention_fwd_cpp", &linear_fwd_meta);
    m.impl("_linear_attention_fwd_save_cpp", &linear_fwd_save_meta);
    m.impl("_linear_attention_bwd_cpp", &linear_bwd_meta);
    m.impl("_linear_attention_update_cpp", &linear_update_meta);
    m.impl("_layer_norm_fwd_cpp", &layer_norm_fwd_meta);
    m.impl("_layer_norm_bwd_cpp", &layer_norm_bwd_meta);
}

TORCH_LIBRARY_IMPL(DaoAILab, Autograd, m) {
    m.impl("_gated_delta_rule_fwd_cpp", &Graphless<kDeltaFwd, true, 7, decltype(delta_fwd)>::call);
    m.impl("_gated_delta_rule_fwd_save_cpp", &Graphless<kDeltaFwdSave, true, 7, decltype(delta_fwd_save)>::call);
    m.impl("_gated_delta_rule_bwd_cpp", &Graphless<kDeltaBwd, true, -1, decltype(delta_bwd)>::call);
    m.impl("_gated_delta_rule_update_cpp", &Graphless<kDeltaUpdate, false, 5, decltype(delta_update)>::call);
    m.impl("_rms_norm_fwd_cpp", &Graphless<kNormFwd, true, -1, decltype(norm_fwd)>::call);
    m.impl("_rms_norm_bwd_cpp", &Graphless<kNormBwd, true, -1, decltype(norm_bwd)>::call);
    m.impl("_rms_norm_quant_cpp", &Graphless<kNormQuant, false, -1, decltype(norm_quant)>::call);
    m.impl("_dequantize_rows_cpp", &Graphless<kDequantize, false, -1, decltype(dequantize)>::call);
    m.impl("_linear_attention_fwd_cpp", &Graphless<kLinearFwd, true, 7, decltype(linear_fwd)>::call);
    m.impl("_linear_attention_fwd_save_cpp", &Graphless<kLinearFwdSave, true, 7, decltype(linear_fwd_save)>::call);
    m.impl("_linear_attention_bwd_cpp", &Graphless<kLinearBwd, true, -1, decltype(linear_bwd)>::call);
    m.impl("_linear_attention_update_cpp", &Graphless<kLinearUpdate, false, 4, decltype(linear_update)>::call);
    m.impl("_layer_norm_fwd_cpp", &Graphless<kLayerNormFwd, true, -1, decltype(layer_norm_fwd)>::call);
    m.impl("_layer_norm_bwd_cpp", &Graphless<kLayerNormBwd, true, -1, decltype(layer_norm_bwd)>::call);
}
