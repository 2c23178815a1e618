// The rotation of a pair of values by a position: shared by the queries' kernel and the
// one that appends projected rows to the pages.
#pragma once

#include "moe_common.h"

namespace fleet_moe {
namespace rope {

// cos and sin of 2 pi * turns * position, times a magnitude. The product and its reduction
// to an eighth of a turn either way, with the quarter turns beside it, are in 64 bits: 2^31
// positions of one radian are 2^28 turns, of which 2^-25 is left then; in 32 bits nothing of them
// would be. What is left is rounded to 32 bits as at most 1/4 of a half turn, to 2^-25 radians
// (of a half turn either way 2^-23.3).
__device__ __forceinline__ float2 angle(double turns, int position, float magnitude) {
    double a = turns * (double)position;
    a -= rint(a);
    const double quarters = rint(4.0 * a);
    float s, c;
    sincospif((float)fma(-0.5, quarters, 2.0 * a), &s, &c);
    const int k = (int)quarters;                          // -2 .. 2
    const float cos = k & 1 ? s : c, sin = k & 1 ? c : s;
    return make_float2(((k + 1) & 2 ? -cos : cos) * magnitude, (k & 2 ? -sin : sin) * magnitude);
}

}  // namespace rope
}  // namespace fleet_moe
