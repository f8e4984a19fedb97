// Host-side contracts between the front of the gated delta rule (cc1d_delta_api.cpp) and its launchers.
#pragma once

#include "cc1d_internal.hpp"
#include "cc1d_mixer.h"

namespace cc1d {

// Token by token.  initial_states / final_states of `p` are the states read and written, `slots` of them, picked by
// `indices` (NULL: sequence n has state n).
int launch_delta_tokens(const cc1d_delta_params &p, const int32_t *indices, int slots, hipStream_t stream);

}  // namespace cc1d
