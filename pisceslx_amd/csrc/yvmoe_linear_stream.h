// The order in which a wavefront of int4_few_kernel reads codes and scales: plain index arithmetic, which
// the host checks against the weights' size (tests/test_int4_linear_stream.py).
#pragma once

#include <hip/hip_runtime.h>

namespace yvmoe {

// Groups wave, wave + 8, ... of each of the work-group's items (RB blocks of outputs each), then, for what is
// loaded ahead, the last item's again. A wavefront past the groups, whose loads are not used, reads the last
// one of each item.
template <int RB>
struct CodeStream {
    int blocks, groups, first, set, step, items;  // first: of an item's groups; step: sets to the next item
    int item, kg;

    __host__ __device__ __forceinline__ CodeStream(int blocks_, int groups_, int wave_, int wg, int grid)
        : blocks(blocks_), groups(groups_), first(wave_ < groups_ ? wave_ : groups_ - 1), set(wg), step(grid),
          items(((blocks + RB - 1) / RB - 1 - wg) / grid + 1), item(0), kg(first) {}

    // Place of block b's group, in groups from the start of all.
    __host__ __device__ __forceinline__ long long at(int b) const {
        const int block = (set + item * step) * RB + b;
        return (long long)(block < blocks ? block : blocks - 1) * groups + kg;
    }
    __host__ __device__ __forceinline__ void next() {
        if (kg + 8 < groups) kg += 8;
        else if (item + 1 < items) item += 1, kg = first;
    }
};

}  // namespace yvmoe
