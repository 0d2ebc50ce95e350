// Items that several thread blocks had a part of: who adds the parts up.
//
// Each block leaves its parts in the workspace, eight warps a part, and behind each warp's share raises a flag. A warp that has
// finished its share looks whether the same warp of every other block of the item has: the last one finds them all, takes the
// shares from the workspace, its own from its registers, and adds them up in the blocks' order, whichever block it is. Nothing
// waits. Two warps that finish together may both find all flags: they write the same values.
// A kernel before this one takes all flags down (clear_flags), so that neither what the workspace held before nor what a
// launch that gave up has left, a replay of the same captured call among them, is taken for a flag. (Flags that no earlier
// launch can have left, a new number every call, would save that kernel but not serve replays.)
#pragma once

#include "iq2xxs_common.cuh"

namespace iq2 {

constexpr uint32_t PART_WARPS = 8;
inline size_t part_flags_bytes(uint32_t blocks) { return ((size_t)blocks * 2 * PART_WARPS * sizeof(uint32_t) + 255) / 256 * 256; }

// The parts of an item: blocks c0 to c1, block c0's in its place `slot` (1 where it has begun in an earlier item), the others'
// in their place 0; this warp's share of this block's (c = self).
struct PartSet {
    uint32_t* flags;
    uint32_t c0, c1, slot, self, warp;

    __device__ __forceinline__ uint32_t part(uint32_t c) const { return c * 2 + (c == c0 ? slot : 0); }
    __device__ __forceinline__ uint32_t* flag(uint32_t c) const { return flags + part(c) * PART_WARPS + warp; }
    // Whether the other blocks' shares are there (the whole warp; what they wrote may then be read past the L1).
    __device__ __forceinline__ bool others_done() const {
        bool done = true;
        for (uint32_t c = c0 + threadIdx.x % 32; c <= c1; c += 32)
            if (c != self && ld_acquire_gpu_u32(flag(c)) == 0u) done = false;
        done = __all_sync(0xFFFFFFFFu, done);
        if (done) __threadfence();
        return done;
    }
    // After the share is written (the whole warp): shows it, and whether all the others' are there by now.
    __device__ __forceinline__ bool show() const {
        __threadfence();
        __syncwarp();
        if (threadIdx.x % 32 == 0) st_release_gpu_u32(flag(self), 1u);
        __threadfence();  // (of two warps that finish together, one at least sees the other's flag)
        __syncwarp();
        return others_done();
    }
};

}  // namespace iq2
