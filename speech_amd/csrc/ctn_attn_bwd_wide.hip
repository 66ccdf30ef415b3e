// Attention's backward pass for fp32 heads of 65 to 128 features, gfx950.  Three planes of keys and values and two accumulators
// take more registers than a wave at half occupancy has; left to itself the compiler then keeps every result of a matrix
// instruction in the accumulation registers and copies it out for each use.  This file is built with matrix results in
// plain registers, the overflow of long-lived fragments going to the accumulation registers instead (16 x 8 heads on 2 of 1024
// causal steps: 437 -> 385 us for dQ, 650 -> 443 us for dK and dV).
#include "ctn_attn_bwd.h"

namespace attn {

void launch_wide(const bool keys, const bwd_params& f, const int nw, const unsigned grid, hipStream_t s) {
    if (keys) launch_pair<float, 128>(f, nw, grid, s);
    else launch_dq<float, 128>(f, nw, grid, s);
}

}  // namespace attn
