// What a launch has to ask the driver about a kernel, asked once per device and kept: the driver's own
// answers cost a small call more than its launch does.  Thread safe; for host code.
#pragma once

#include <cuda_runtime.h>

namespace mmf {

// Lets `kernel` use `smem` bytes of dynamic shared memory on the current device (preferring shared memory
// over cache in the split, with `carveout`); throws std::runtime_error.
void allow_shared(const void* kernel, int smem, bool carveout = false);

// Blocks of `block` threads and `smem` bytes that an SM of the current device holds at once (at least 1,
// or it throws); allow_shared included.
int resident_blocks(const void* kernel, int block, int smem);

// Clusters of `blocks` such blocks (along y) that the current device holds at once: where a cluster's blocks
// have to be near one another that is less than the blocks alone would make.
int resident_clusters(const void* kernel, int block, int smem, int blocks);

}  // namespace mmf
