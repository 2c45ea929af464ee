// A reader's place in a ring of stages.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define MOK_RING_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define MOK_RING_HOST_DEVICE inline
#endif

namespace mok {

// Stages are read in turn; the barrier of a stage tells rounds apart by one bit.  Once a wait has run out the reader goes on with its
// turns but never waits again: a round later the bit of a round that was served long ago would answer for one that never came.
template <int STAGES>
struct RingTurn {
    uint32_t stage = 0, phase = 0;
    bool ok = true;
    // wait(stage, phase): whether the stage of this turn is there.  False for this turn and all that follow it.
    template <class Wait>
    MOK_RING_HOST_DEVICE bool next(Wait&& wait) {
        ok = ok && wait(stage, phase);
        if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
        }
        return ok;
    }
};

}  // namespace mok
