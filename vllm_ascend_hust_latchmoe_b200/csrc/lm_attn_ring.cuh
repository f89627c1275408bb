// Turns of the 16-row attention kernel's two query buffers. Plain C++ as well, for host models of the
// protocol.
#pragma once

#ifdef __CUDACC__
#define LM_RING_FN __host__ __device__ __forceinline__
#else
#define LM_RING_FN inline
#endif

namespace lm {

// A side (the loader warp, or a consumer warp) holds one of these and takes a turn for each segment that
// has key blocks, and for no other: both sides walk the same segments, so they count the same turns, and
// turn n uses buffer n & 1 for the n / 2-th time. A wait by parity tells a barrier's phase from its
// neighbours only. With a turn each, the loader waits for the consumers' release of turn n - 2 before it
// fills turn n and neither side is ever more than a phase from the other; turns that one side passed
// without waiting would let it run further ahead, and its next wait would take an older phase of the
// same parity for the one that it needs.
struct AttnQueryTurn {
  int taken = 0;
  static LM_RING_FN bool has_keys(int blk0, int blk1) { return blk1 > blk0; }
  LM_RING_FN int buffer() const { return taken & 1; }
  LM_RING_FN unsigned full_parity() const { return (static_cast<unsigned>(taken) >> 1) & 1u; }
  LM_RING_FN unsigned empty_parity() const { return full_parity() ^ 1u; }
  LM_RING_FN void next() { ++taken; }
};

}  // namespace lm
