// swiftkv_paged_rows.hpp -- which rows of a call the paged cache's kernels read, as rules
// that a program without a device can check.
#pragma once

#ifdef __HIPCC__
#define SWIFTKV_RULE __host__ __device__ inline
#else
#define SWIFTKV_RULE inline
#endif

namespace swiftkv {

// Whether the step of tokens from tok0 on, one of those that tokens [p, end) of a call may
// touch, holds one of them.  (A tree may be without tokens: end == p, inside a step too.)
SWIFTKV_RULE bool step_has_new(int tok0, int p, int end) { return p < end && tok0 < end; }

// The row of the call that a lane of token `tok` loads: its own, or where the token is none
// of [p, end) the nearest.
SWIFTKV_RULE int nearest_row(int tok, int p, int end) { return (tok < p ? p : tok < end ? tok : end - 1) - p; }

}  // namespace swiftkv
