// The rotation of a pair of values by a position: shared by the queries' kernel and the
// one that appends projected rows to the pages.
#pragma once

#include "moe_common.h"

namespace fleet_moe {
namespace rope {

// cos and sin of 2 pi * turns * position, times a magnitude. The product and its reduction
// to half a turn either way are in 64 bits: 2^31 positions of one radian are 2^28 turns, of
// which 2^-25 is left then; in 32 bits nothing of them would be.
__device__ __forceinline__ float2 angle(double turns, int position, float magnitude) {
    const double a = turns * (double)position;
    float s, c;
    sincospif((float)(2.0 * (a - rint(a))), &s, &c);
    return make_float2(c * magnitude, s * magnitude);
}

}  // namespace rope
}  // namespace fleet_moe
