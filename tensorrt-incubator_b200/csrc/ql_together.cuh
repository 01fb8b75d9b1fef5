// Steps that several warps take together, none of them further than the others.  Plain C++ as well, so that it runs on a host.
#pragma once

#include <type_traits>

#ifdef __CUDACC__
#define QL_ROLE __device__ __forceinline__
#else
#define QL_ROLE inline
#endif

namespace ql {

// What each warp of the group runs: step i (of n) is meet(slot, i, go), a barrier of the whole group that tells every warp the
// same, whether all of them go on, then take(slot, i), which may give up (false).  slot is i % 2, a constant.
// A warp that gave up comes to the next barrier nevertheless and says so there, and there all leave.  Were each to leave by
// itself, a warp whose wait had just been fulfilled would come to a barrier that the ones that gave up never reach.
template <typename Meet, typename Take> QL_ROLE void steps_together(int n, Meet &&meet, Take &&take) {
  bool go = true;
  for (int i = 0; i < n; i += 2) {
    if (!meet(std::integral_constant<int, 0>{}, i, go)) return;
    go = take(std::integral_constant<int, 0>{}, i);
    if (i + 1 >= n || !meet(std::integral_constant<int, 1>{}, i + 1, go)) return;
    go = take(std::integral_constant<int, 1>{}, i + 1);
  }
}

} // namespace ql
