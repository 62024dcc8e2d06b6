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

// The position by which a token's query and key are turned: p cached tokens and its depth
// in the call.  Rows without a token and sequences that sit out (p < 0) are not turned by
// positions that the call's checks have bounded, and take 0.
SWIFTKV_RULE int turn_position(int p, int depth, bool live) { return p >= 0 && live ? p + depth : 0; }

// Whether the positions of a call's tokens, the deepest at `depth` (-1: none), are within a
// table of so many.
SWIFTKV_RULE bool turns_within(int p, int depth, int positions) { return p < 0 || static_cast<long long>(p) + depth < positions; }

}  // namespace swiftkv
