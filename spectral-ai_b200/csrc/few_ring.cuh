// few_ring.cuh — the order in which a ring's slots are filled and used (no device code, so
// that a host program can check it).
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define SB_RING_FN __host__ __device__ __forceinline__
#else
#define SB_RING_FN inline
#endif

namespace sb {

// `depth` slots, filled and taken in turn; a slot's barrier completes one phase each time
// it is filled.
struct FewSlots {
  int depth, out;   // out: the next to be taken
  uint32_t parity;  // of the phase that fills `out`
  SB_RING_FN explicit FewSlots(int depth_) : depth(depth_), out(0), parity(0) {}
  SB_RING_FN void taken() {
    if (++out == depth) {
      out = 0;
      parity ^= 1u;
    }
  }
  // the slot of the i-th filling (0 .. depth - 1) that has not been taken, and its phase
  SB_RING_FN int ahead(int i, uint32_t* phase) const {
    const int slot = out + i;
    *phase = slot < depth ? parity : parity ^ 1u;
    return slot < depth ? slot : slot - depth;
  }
};

}  // namespace sb
