// The ring of K/V blocks of the chunk attention (mac_b200_chunk.cu): its shape, what a loading warp
// waits for before it fills a position, and what is taken out of a block of values there.  Plain C++, so
// that the host can walk through it (tests/chunk_ring_model.cpp).
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define MAC_RING_FN __device__ __forceinline__
#else
#define MAC_RING_FN inline
#endif

namespace mac_b200 {

// Positions of the ring, and groups of loading warps that fill them in turn: group g takes positions
// g, g + kGroups, ... of all that the CTA fills.  kSpare positions more where no unit has two tiles.
template <bool kE4m3>
struct RingShape {
  static constexpr int kGroups = kE4m3 ? 3 : 1;
  static constexpr int kStages = kE4m3 ? 3 : 5;
  static constexpr int kSpare = kE4m3 ? 1 : 0;
};

// Position p lies in stage p % stages and may be filled once p - stages was given back.  A barrier
// tells its phases apart by one bit, so that wait is only sound for a warp that knows p - 2 * stages to
// have been given back: else it could take the phase before for the one it waits for.  Where stages is not
// a multiple of the groups another group filled p - stages, and the positions that this warp did wait for
// say nothing: a stream gives a position of the other stream back at once, and its own only when
// the products on it, issued earlier, have run.  So the warp first waits until p - stages has been filled,
// which its group did after it had seen p - 2 * stages given back.  That wait is sound too: this warp has
// seen p - groups - stages given back (or filled its own first position), which both streams do only after
// they have seen every position up to it filled, p - 2 * stages among them (groups <= stages), and nobody
// fills p but this warp's group.  It costs no time: what has been given back has been filled.
// `wait(filled)`: the stage's barrier of filled positions, or of those given back, for the cursor's phase.
template <class Wait>
MAC_RING_FN bool wait_to_fill(Wait&& wait) {
  return wait(true) && wait(false);
}

// A pair of bf16 values with infinities and NaN replaced by zero.  The streams of a unit of two tiles share
// its blocks, and each takes these values out for itself before its own product, while the other's may
// run: so a word is changed by one store, which leaves it as it stays.  Whoever stores late stores
// what is there already.
MAC_RING_FN uint32_t finite_halves(uint32_t w) {
  if ((w & 0x00007f80u) == 0x00007f80u) w &= 0xffff0000u;
  if ((w & 0x7f800000u) == 0x7f800000u) w &= 0x0000ffffu;
  return w;
}

}  // namespace mac_b200
