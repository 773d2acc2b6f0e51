// Bookkeeping of a warp's ring of boxes in shared memory: which slot is filled next, which one is waited for and with which parity, and how many copies are on their way.
// Host and device, so that it can be run without a GPU.
#pragma once

#ifdef __CUDACC__
#define DX_RING_FN __host__ __device__ __forceinline__
#else
#define DX_RING_FN inline
#endif

namespace dx {

struct RingState {
    int stages, fill = 0, slot = 0, parity = 0, flying = 0;
    bool alive = true;
    DX_RING_FN explicit RingState(int stages_) : stages(stages_) {}
    // A copy into slot `fill` was started; none is once a wait has run out.
    DX_RING_FN void started() {
        fill = fill + 1 == stages ? 0 : fill + 1;
        ++flying;
    }
    // The box in slot `slot` has been waited for.
    DX_RING_FN void taken() {
        if (++slot == stages) {
            slot = 0;
            parity ^= 1;
        }
        --flying;
    }
    // The wait for the box in slot `slot` ran out: `wait(slot, parity)` for it and for each of the others that are still on their way, so that none writes to memory that
    // is not this warp's any more. To be called before the box counts as taken; later boxes of the loop are not there and are not waited for.
    template <typename Wait>
    DX_RING_FN void give_up(Wait wait) {
        const int next_slot = slot, next_parity = parity;
        while (flying > 0) {
            wait(slot, parity);
            taken();
        }
        slot = next_slot;
        parity = next_parity;
        alive = false;
    }
};

}  // namespace dx
