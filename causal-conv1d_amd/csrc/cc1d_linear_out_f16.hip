// Linear attention, out of f16 tensors (cc1d_linear_attend.hpp, cc1d_linear_tile.hpp).
#include "cc1d_linear_tile.hpp"

namespace cc1d {
template int launch_attend<CC1D_F16, false>(const cc1d_delta_params &, const SegmentWork &, const AttendArgs &, hipStream_t);
}
