// Linear attention, dq and dk of bf16 tensors (cc1d_linear_attend.hpp, cc1d_linear_tile.hpp).
#include "cc1d_linear_tile.hpp"

namespace cc1d {
template int launch_attend_pair<CC1D_BF16>(const cc1d_delta_params &, const SegmentWork &, const AttendArgs &, const AttendArgs &, const AttendArgs *, hipStream_t);
}
