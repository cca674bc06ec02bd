// Cutting a launch that has too many threads for one; plain C++ so that it is checked on a host as well.
#pragma once
#include <stdint.h>

namespace seq {

// A launch's threads along x are counted in 32 bits, and what is above is dropped without an error (16 777 221 workgroups of 256 ran as 5): `blocks`
// workgroups of `threads` in launches of fewer than 2^32 threads, f(the first workgroup of the launch, how many).
template <typename F> void in_launches(int64_t blocks, int threads, F f) {
    const int64_t most = (((int64_t)1 << 32) - 1) / threads;
    for (int64_t first = 0; first < blocks; first += most) f((int32_t)first, (uint32_t)(blocks - first < most ? blocks - first : most));
}

}  // namespace seq
