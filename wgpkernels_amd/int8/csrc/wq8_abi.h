// Internal declarations shared by the library's translation units (the public C-ABI is include/wq8.h).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#define WQ8_API extern "C" __attribute__((visibility("default")))

namespace wq8 {
// Row offset read on the GPU for CUDA-graph-style loops: rows first + counter[0] * step.
struct RowOffsetArgs { const long long* counter; long long first, step; };
// A grid's threads are counted in 32 bits: workgroups of 256 that one dimension holds.
constexpr int64_t MAX_BLOCKS_256 = (int64_t(1) << 24) - 1;
}  // namespace wq8
