// Rotary positions: angles by frequencies that a caller gives, and the rotation of rows of heads (rotation.hip); the
// frequencies of scaled rotations (rotary.cpp, host only).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace satori {

// Pair k of a head turned by position * frequencies[k], and both lanes made longer by `magnitude`. Pairs are lanes
// (k, k + pairs), or (2 k, 2 k + 1) where interleaved. The table has the sines, then the cosines, of positions
// 0 .. positions - 1, times the magnitude, as doubles [positions][2 * pairs].
struct RotationShape {
    const double* frequencies;
    const double* table;
    int positions, pairs;
    double magnitude;
    bool interleaved;
};

struct RotateArgs {
    const void* input;
    void* output;
    int64_t input_stride, output_stride;  // elements between rows
    const int* positions;
    int rows, heads, head_dim;
};

hipError_t launch_rotation_table(const RotationShape& shape, double* table, hipStream_t stream);
// `type`: Element (cache_ops.hpp).
hipError_t launch_rotate(const RotationShape& shape, int type, const RotateArgs& args, hipStream_t stream);

}  // namespace satori
