// The waits that make up for one that ran out, for a warp with one stage: a K
// and a V tile, each with its barrier (0 and 1), whose phase for the warp's
// tile j has parity j & 1.  K of tile j + 1 is requested between the waits for K
// and for V of tile j, so still in flight are, after K's wait has run out, K and V of
// tile j; after V's, V of tile j and, if there are `more` tiles, K of tile j + 1.
// wait(barrier, parity) is a bounded wait.  Plain C++, so that it can be checked on a host.
#pragma once

#ifdef __CUDACC__
#define RKV_HOST_DEVICE __host__ __device__
#else
#define RKV_HOST_DEVICE
#endif

namespace rkv {

template <typename Wait>
RKV_HOST_DEVICE inline void drain_keys_and_values(int j, Wait wait) {
  wait(0, j & 1);
  wait(1, j & 1);
}

template <typename Wait>
RKV_HOST_DEVICE inline void drain_values(int j, bool more, Wait wait) {
  wait(1, j & 1);
  if (more) wait(0, (j + 1) & 1);
}

}  // namespace rkv
