// The elements of a rotation by given frequencies, shared by the kernels that rotate so that all give the same values bit
// for bit: the angle in 64 bits, both rotated lanes in 64 bits, each rounded once.
#pragma once

#include <cmath>

#include "rope_device.hpp"

namespace satori {

__device__ __forceinline__ void rotation_angle(int k, int position, const double* frequencies, double magnitude, double& sn,
                                               double& cs) {
    const double angle = position * frequencies[k];
    sn = sin(angle) * magnitude;
    cs = cos(angle) * magnitude;
}

// Pair j of the N that two packs of N lanes hold: lane j of both, or, interleaved, the j-th two lanes of both in a row.
template <bool INTERLEAVED, int N>
__device__ __forceinline__ void rotate_pair(float (&x)[N], float (&y)[N], int j, double sn, double cs) {
    if constexpr (!INTERLEAVED) {
        rope_apply(x[j], y[j], sn, cs, x[j], y[j]);
    } else if constexpr (N == 1) {
        rope_apply(x[0], y[0], sn, cs, x[0], y[0]);
    } else {
        float(&in)[N] = 2 * j < N ? x : y;
        const int i = 2 * j < N ? 2 * j : 2 * j - N;
        rope_apply(in[i], in[i + 1], sn, cs, in[i], in[i + 1]);
    }
}

}  // namespace satori
