// Rotary positions of rows of heads.
#include "rotation.hpp"

#include <algorithm>

#include "cache_ops.hpp"
#include "device_common.hpp"
#include "rotation_device.hpp"

namespace satori {
namespace {

constexpr int kThreads = 256;

__global__ __launch_bounds__(kThreads) void rotation_table_kernel(RotationShape s, double* table) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    if (i >= static_cast<int64_t>(s.positions) * s.pairs) return;
    const int p = static_cast<int>(i / s.pairs), k = static_cast<int>(i % s.pairs);
    double* row = table + static_cast<int64_t>(p) * 2 * s.pairs;
    rotation_angle(k, p, s.frequencies, s.magnitude, row[k], row[s.pairs + k]);
}

// N elements at any place of theirs, one access.
template <typename T, int N>
struct PackOf {
    typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};
template <typename T, int N>
__device__ __forceinline__ void load_pack(const T* p, float (&v)[N]) {
    typedef typename PackOf<T, N>::type pack;
    const pack x = *(const SATORI_GLOBAL pack*)(p);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = static_cast<float>(x[i]);
}
template <typename T, int N>
__device__ __forceinline__ void store_pack(T* p, const float (&v)[N]) {
    typedef typename PackOf<T, N>::type pack;
    pack x;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = static_cast<T>(v[i]);
    *(SATORI_GLOBAL pack*)(p) = x;
}

// A thread turns N pairs of one row in kHeads heads, whose angles it reads once: both lanes' 16 bytes a head and access.
// Behind the last whole N pairs of a head single ones, and packs for the lanes behind the rotated ones, which are copied
// unless the output is the input.
template <typename T, bool INTERLEAVED, int HEADS>
__global__ __launch_bounds__(kThreads) void rotate_kernel(RotationShape s, RotateArgs a, int units, int packs, int groups) {
    constexpr int N = 16 / sizeof(T);
    const uint32_t i = blockIdx.x * kThreads + threadIdx.x;
    const uint32_t unit = i % units, rest = i / units, group = rest % groups, row = rest / groups;
    if (row >= static_cast<uint32_t>(a.rows)) return;
    const int first = group * HEADS, heads = min(HEADS, a.heads - first), D = a.head_dim;
    const T* in = static_cast<const T*>(a.input) + row * a.input_stride + static_cast<int64_t>(first) * D;
    T* out = static_cast<T*>(a.output) + row * a.output_stride + static_cast<int64_t>(first) * D;
    if (static_cast<int>(unit) >= packs) {
        const int lane = 2 * s.pairs + (unit - packs) * N;
        for (int h = 0; h < heads; ++h) {
            if (lane + N <= D) {
                float v[N];
                load_pack<T, N>(in + h * D + lane, v);
                store_pack<T, N>(out + h * D + lane, v);
            } else {
                for (int j = lane; j < D; ++j) out[h * D + j] = in[h * D + j];
            }
        }
        return;
    }
    const int k = unit * N, position = a.positions[row], left = min(N, s.pairs - k);
    const bool listed = position >= 0 && position < s.positions;
    const double* angles = s.table + static_cast<int64_t>(listed ? position : 0) * 2 * s.pairs + k;
    const auto angle = [&](int j, double& sn, double& cs) {
        if (listed) {
            sn = angles[j];
            cs = angles[s.pairs + j];
        } else {
            rotation_angle(k + j, position, s.frequencies, s.magnitude, sn, cs);
        }
    };
    const int at = INTERLEAVED ? 2 * k : k, beside = INTERLEAVED ? N : s.pairs;
    if (left < N) {
        for (int j = 0; j < left; ++j) {
            double sn, cs;
            angle(j, sn, cs);
            const int x = INTERLEAVED ? at + 2 * j : at + j, y = INTERLEAVED ? x + 1 : x + s.pairs;
            for (int h = 0; h < heads; ++h) {
                float u, v;
                rope_apply(static_cast<float>(in[h * D + x]), static_cast<float>(in[h * D + y]), sn, cs, u, v);
                out[h * D + x] = static_cast<T>(u);
                out[h * D + y] = static_cast<T>(v);
            }
        }
        return;
    }
    float x[HEADS][N], y[HEADS][N];
#pragma unroll
    for (int h = 0; h < HEADS; ++h)
        if (h < heads) {
            load_pack<T, N>(in + h * D + at, x[h]);
            load_pack<T, N>(in + h * D + at + beside, y[h]);
        }
#pragma unroll
    for (int j = 0; j < N; ++j) {
        double sn, cs;
        angle(j, sn, cs);
#pragma unroll
        for (int h = 0; h < HEADS; ++h)
            if (h < heads) rotate_pair<INTERLEAVED>(x[h], y[h], j, sn, cs);
    }
#pragma unroll
    for (int h = 0; h < HEADS; ++h)
        if (h < heads) {
            store_pack<T, N>(out + h * D + at, x[h]);
            store_pack<T, N>(out + h * D + at + beside, y[h]);
        }
}

template <typename T, bool INTERLEAVED>
hipError_t rotate_of(const RotationShape& s, const RotateArgs& a, hipStream_t stream) {
    constexpr int N = 16 / sizeof(T);
    const int packs = (s.pairs + N - 1) / N, behind = a.output == a.input ? 0 : (a.head_dim - 2 * s.pairs + N - 1) / N;
    const int units = packs + behind;
    constexpr int kHeads = 4;
    const int groups = (a.heads + kHeads - 1) / kHeads;
    const int64_t row_units = static_cast<int64_t>(units) * groups;
    // (a launch's threads are counted in 32 bits)
    const int most = static_cast<int>(std::max<int64_t>(1, (int64_t(1) << 30) / row_units));
    for (int row = 0; row < a.rows; row += most) {
        RotateArgs part = a;
        part.rows = std::min(most, a.rows - row);
        part.input = static_cast<const T*>(a.input) + row * a.input_stride;
        part.output = static_cast<T*>(a.output) + row * a.output_stride;
        part.positions = a.positions + row;
        const unsigned blocks = static_cast<unsigned>((part.rows * row_units + kThreads - 1) / kThreads);
        rotate_kernel<T, INTERLEAVED, kHeads><<<blocks, kThreads, 0, stream>>>(s, part, units, packs, groups);
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace

hipError_t launch_rotation_table(const RotationShape& shape, double* table, hipStream_t stream) {
    const int64_t n = static_cast<int64_t>(shape.positions) * shape.pairs;
    if (n <= 0) return hipSuccess;
    rotation_table_kernel<<<static_cast<unsigned>((n + kThreads - 1) / kThreads), kThreads, 0, stream>>>(shape, table);
    return hipGetLastError();
}

hipError_t launch_rotate(const RotationShape& shape, int type, const RotateArgs& args, hipStream_t stream) {
    if (type == kF32)
        return shape.interleaved ? rotate_of<float, true>(shape, args, stream) : rotate_of<float, false>(shape, args, stream);
    return shape.interleaved ? rotate_of<_Float16, true>(shape, args, stream) : rotate_of<_Float16, false>(shape, args, stream);
}

}  // namespace satori
