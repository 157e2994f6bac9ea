// ring.cuh -- a place in a ring of shared-memory stages and the parity of its barriers there. No CUDA
// header: the host's compiler reads it too, so that the walk can be checked without a GPU.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define SS_RING __host__ __device__ __forceinline__
#else
#define SS_RING inline
#endif

namespace ss {

// No division: next() is on the critical path of every step.
struct Ring {
    int n, at = 0;
    uint32_t parity = 0;
    SS_RING explicit Ring(int stages) : n(stages) {}
    SS_RING void next() {
        if (++at == n) {
            at = 0;
            parity ^= 1u;
        }
    }
    // the j-th stage before this one, j <= n
    SS_RING Ring before(int j) const {
        Ring r = *this;
        r.at -= j;
        if (r.at < 0) {
            r.at += n;
            r.parity ^= 1u;
        }
        return r;
    }
    // Waits for a barrier of each of the last `filled` stages, oldest first, in its last round: wait(stage,
    // parity), false once one ran out. `filled` is the smaller of the steps taken and n.
    template <typename W>
    SS_RING bool wait_for_each(int filled, W wait) const {
        bool ok = true;
        for (int j = filled; j > 0 && ok; --j) {
            const Ring r = before(j);
            ok = wait(r.at, r.parity);
        }
        return ok;
    }
};

}  // namespace ss
