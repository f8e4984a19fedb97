// Host-side contracts between the front of the gated delta rule (cc1d_delta_api.cpp) and its launchers.
#pragma once

#include <type_traits>

#include "cc1d_internal.hpp"
#include "cc1d_mixer.h"

namespace cc1d {

struct ChunkWork;

// Token by token.  initial_states / final_states of `p` are the states read and written, `slots` of them, picked by
// `indices` (NULL: sequence n has state n).  `longest`: sequences of that many tokens are left alone (0: none).  Without `rule`: linear
// attention, whose beta may be NULL.
int launch_delta_tokens(const cc1d_delta_params &p, const int32_t *indices, int slots, int longest, hipStream_t stream, bool rule = true);
// A decode step of either, whose arguments have been checked.
int launch_step_tokens(const cc1d_delta_step_params &step, hipStream_t stream, bool rule);
// By chunks: what needs no state; then the states and outputs (`save`: the states in front of the chunks and U are kept).
int launch_delta_prep(const cc1d_delta_params &p, const ChunkWork &w, hipStream_t stream);
int launch_delta_scan(const cc1d_delta_params &p, const ChunkWork &w, bool save, hipStream_t stream);
// Backward, behind its own prep: the gradients.
int launch_delta_bwd(const cc1d_delta_bwd_params &p, const ChunkWork &w, hipStream_t stream);

// Its gradients of q and k where there are no value heads.
int launch_delta_no_values(const cc1d_delta_bwd_params &bp, hipStream_t stream);

// Every row of a (batch, seqlen, heads, dim) tensor starts on 16 bytes.
inline bool whole_rows(int dtype, const void *x, int64_t sb, int64_t sl, int64_t sh) {
    const int v = vec_elems(dtype);
    return aligned16(x) && sb % v == 0 && sl % v == 0 && sh % v == 0;
}

// 32-column steps of dim_k that have kernels.  4 x 1024 tokens of 16 heads, forward and backward, dim_k 96 in three steps and in four: bfloat16
// 270 us and 307, float32 436 and 536; 192 in six and in eight: 404 and 566, 946 and 1332.  Five and seven would serve few sizes.
inline int key_steps(int dim_k) { return dim_k <= 128 ? (dim_k + 31) / 32 : dim_k <= 192 ? 6 : 8; }

template <typename F>
int by_type_and_steps(int dtype, int steps, F &&f) {
    auto with = [&](auto dt) {
        switch (steps) {
            case 1: return f(dt, std::integral_constant<int, 1>());
            case 2: return f(dt, std::integral_constant<int, 2>());
            case 3: return f(dt, std::integral_constant<int, 3>());
            case 4: return f(dt, std::integral_constant<int, 4>());
            case 6: return f(dt, std::integral_constant<int, 6>());
            default: return f(dt, std::integral_constant<int, 8>());
        }
    };
    switch (dtype) {
        case CC1D_F32: return with(std::integral_constant<int, CC1D_F32>());
        case CC1D_F16: return with(std::integral_constant<int, CC1D_F16>());
        default: return with(std::integral_constant<int, CC1D_BF16>());
    }
}

}  // namespace cc1d
