// Bookkeeping of a ring of at most 32 slots that asynchronous copies fill.
// Plain C++ too, so that its rules can be tested without a GPU.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define ADVOPT_HD __host__ __device__ __forceinline__
#else
#define ADVOPT_HD inline
#endif

namespace advopt {
namespace fp8 {

// For each slot (a bit each) whether it has been filled, and the parity of its
// latest fill.  A slot's barriers complete one phase a fill, so that is also
// the parity of the phase that ends when the fill has landed, and of the one
// that ends when it has been used up.
struct Fills {
  uint32_t begun = 0, parity = 0;
  ADVOPT_HD bool any(uint32_t slot) const { return begun >> slot & 1u; }
  ADVOPT_HD uint32_t latest(uint32_t slot) const { return parity >> slot & 1u; }
  ADVOPT_HD void next(uint32_t slot) {
    if (any(slot)) parity ^= 1u << slot;
    begun |= 1u << slot;
  }
};

// Waits for each slot's latest fill: wait(slot, parity).  An earlier fill has
// landed, since its slot was filled again; the other parity is that of the
// phase before, and waiting for it would return at once.
template <class Wait>
ADVOPT_HD void await_fills(const Fills& f, int slots, Wait wait) {
  for (int s = 0; s < slots; ++s)
    if (f.any((uint32_t)s)) wait(s, f.latest((uint32_t)s));
}

}  // namespace fp8
}  // namespace advopt
