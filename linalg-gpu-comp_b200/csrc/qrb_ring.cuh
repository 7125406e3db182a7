// A ring of shared-memory stages between a thread that loads items 0, 1, 2, ... and the threads that use
// them, with two mbarriers a stage: `full`, which the loads of an item complete, and `empty`, which its last
// reader does.
//
// A wait by parity cannot tell a phase from the one two before or behind it.  With a barrier pair of its own a
// stage's next phase needs its next item, which is not loaded before the loader has seen the last one freed, so
// no waiter can fall two phases behind, however long it is held up.  (One `empty` barrier for two stages has
// no such order: the other stage's item can be finished before the loader looks.)
//
// Plain C++, so that the protocol can be run on the host as well.
#pragma once

#ifdef __CUDACC__
#define QRB_RING_FN __host__ __device__ __forceinline__
#else
#define QRB_RING_FN inline
#endif

namespace qrb {

template <int S>
struct Ring {
  static_assert(S >= 1, "stages");
  // The stage of item i, and the parity of the phase that item i completes on either of its barriers.  Item i
  // may be loaded once item i - S has completed its phase of `empty`.
  QRB_RING_FN static constexpr int stage(int i) { return i % S; }
  QRB_RING_FN static constexpr unsigned phase(int i) { return (unsigned)(i / S) & 1u; }
};

}  // namespace qrb
