// The running maximum of tree attention's softmax.  Plain C++ where nvcc does
// not compile it, so the rule can be run on the host.
//
// Weights are e^{scale (s - m)} for a maximum m of raw scores (before the
// scale) that moves only when a score lies more than the headroom above it.
// Whether it has to move is asked of single scores, and of a row's largest one
// when it moves: both subtract first, with one rounding, and rounding keeps
// order, so they cannot disagree.  The difference of near numbers is exact,
// however large they are, so the largest score's e^{..} stays between 1 and
// 2^8 even where one step of m is more than that.
#pragma once

#ifdef __CUDACC__
#define HALO_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define HALO_HOST_DEVICE inline
#endif

namespace halo {
namespace tree {

constexpr float kNoMax = -3.402823466e38f;   // nothing seen yet: any score raises it
constexpr float kRescaleLog2 = 8.f;          // headroom, in log2 units of a weight

// The headroom in units of a raw score.
HALO_HOST_DEVICE float raw_headroom(float scale_log2) { return kRescaleLog2 / scale_log2; }

HALO_HOST_DEVICE float excess(float s, float m) { return s - m; }

HALO_HOST_DEVICE bool rises(float s, float m, float headroom) { return excess(s, m) > headroom; }

}  // namespace tree
}  // namespace halo
