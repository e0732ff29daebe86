// Device helpers of the operators around a prompt.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace pto {

// Of sequences that begin at cu[0] <= cu[1] <= .. the one that row r is in: how many of cu[1] .. cu[B] are at most r (B: none).
// Every lane looks at one of 64 evenly spaced entries.
__device__ __forceinline__ int sequence_of(const int32_t *cu, const int B, const long long r)
{
    const int l = threadIdx.x & 63;
    int lo = 0, n = B;                                     // the answer is in lo .. lo + n
    while (n > 0) {
        const int step = (n + 63) / 64, at = lo + (l + 1) * step - 1;
        const bool behind = at < lo + n && cu[at + 1] <= r;
        const int c = __popcll(__ballot(behind));
        const int end = lo + n;
        lo += c * step;
        n = step - 1 < end - lo ? step - 1 : end - lo;
    }
    return lo;
}

}  // namespace pto
