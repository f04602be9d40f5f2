// The elements of a position's attention inputs (DenseForward.cs:128-151): the bias add and RopeHalf, shared by the
// kernels that form them so that all give the same values bit for bit.
#pragma once

#include <cmath>

#include "device_common.hpp"

namespace satori {

__device__ __forceinline__ float biased(const float* x, const float* bias, int i) {
    return bias ? __fadd_rn(x[i], bias[i]) : x[i];
}

// RopeHalf of lane pair (kk, kk + rotary / 2) of one head (TransformerOps.cs:94-114): the angle
// position / base^(2 kk / rotary) in FP64, then both rotated lanes in FP64, each rounded once.
__device__ __forceinline__ void rope_angle(int kk, int position, double base, int rotary, double& sn, double& cs) {
    const double angle = position / pow(base, 2.0 * kk / rotary);
    sn = sin(angle);
    cs = cos(angle);
}

__device__ __forceinline__ void rope_apply(double x, double y, double sn, double cs, float& a, float& b) {
    a = static_cast<float>(x * cs - y * sn);
    b = static_cast<float>(x * sn + y * cs);
}

__device__ __forceinline__ void rope_pair(double x, double y, int kk, int position, double base, int rotary, float& a,
                                          float& b) {
    double sn, cs;
    rope_angle(kk, position, base, rotary, sn, cs);
    rope_apply(x, y, sn, cs, a, b);
}

}  // namespace satori
