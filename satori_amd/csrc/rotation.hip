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
    const int64_t all = static_cast<int64_t>(s.positions) * s.pairs, stride = static_cast<int64_t>(gridDim.x) * kThreads;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < all; i += stride) {
        const int p = static_cast<int>(i / s.pairs), k = static_cast<int>(i % s.pairs);
        double* row = table + static_cast<int64_t>(p) * 2 * s.pairs;
        rotation_angle(k, p, s.frequencies, s.magnitude, row[k], row[s.pairs + k]);
    }
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

// A workgroup turns some pairs (kThreads at most, all rows together) of some rows: its threads read, or compute, the sine and
// cosine of one pair of one row each and leave them in LDS, while what they turn first is on its way: four accesses of 16 bytes
// a thread and turn, each half a head apart its pairs' other one (two heads), or with whole pairs (four heads). Behind the
// last whole pack of a head single pairs; the lanes behind the rotated ones are copied, unless the output is the input.
// Bound by the launch (8 rows of 12 heads 3.2 us) or by memory: 4096 rows of 32 heads of 128 F16 lanes 13.2 us, 67 MB at 5.1 TB/s
// (13.0 where a sum was rounded by way of FP32's nearest number; with that two accesses a thread 14.4, eight 13.8; angles read by
// every thread, 64 bytes a pack, 18).

// A sum as an FP32 number that rounds to F16 as the sum itself does: its first 24 bits, the last of them set where any behind
// them is. That lies on the sum's side of every border between F16's numbers, which have 13 bits fewer. (FP32's nearest number may be
// such a border itself, and would round away from the sum.)
__device__ __forceinline__ float once(double v) {
    const uint64_t bits = __double_as_longlong(v);
    const uint32_t low = static_cast<uint32_t>(bits), behind = low & 0x1fffffffu;
    const uint32_t kept = (low | (behind + 0x1fffffffu)) & 0xe0000000u;
    return static_cast<float>(__longlong_as_double(bits >> 32 << 32 | kept));
}
// FP32 lanes have the bits of the cache write's (rope_apply); F16 ones fuse a product into each sum.
template <typename T>
__device__ __forceinline__ void turn_pair(double x, double y, double sn, double cs, float& a, float& b) {
    if constexpr (sizeof(T) == 4) {
        rope_apply(x, y, sn, cs, a, b);
    } else {
        a = once(fma(-y, sn, x * cs));
        b = once(fma(y, cs, x * sn));
    }
}

// Where a pair's angle lies: a pack's 128 bytes start at other banks than the next one's.
__device__ __forceinline__ int angle_at(int i) { return i + (i >> 3); }

template <typename T, bool INTERLEAVED>
__global__ __launch_bounds__(kThreads) void rotate_kernel(RotationShape s, RotateArgs a, int group_rows, int group_pairs) {
    constexpr int N = 16 / sizeof(T), kHeads = INTERLEAVED ? 4 : 2, kPairs = INTERLEAVED ? N / 2 : N;  // pairs of a pack
    typedef double f64x2 __attribute__((ext_vector_type(2)));
    __shared__ f64x2 angles[kThreads + kThreads / 8];
    const int thread = threadIdx.x, row0 = blockIdx.x * group_rows, k0 = blockIdx.y * group_pairs, D = a.head_dim;
    const int rows = min(group_rows, a.rows - row0), pairs = min(group_pairs, s.pairs - k0);
    const int packs = (pairs + kPairs - 1) / kPairs, groups = (a.heads + kHeads - 1) / kHeads;
    const bool copies = a.output != a.input && blockIdx.y + 1 == gridDim.y;
    const int units = packs + (copies ? (D - 2 * s.pairs + N - 1) / N : 0), row_units = units * groups;

    struct Unit {
        int row, pack, heads;  // past the pairs' packs: one to copy
        const T* in;
        T* out;
    };
    const auto locate = [&](int u) {
        Unit r;
        r.row = u / row_units;
        const int rest = u % row_units, first = rest / units * kHeads;
        r.pack = rest % units;
        r.heads = min(kHeads, a.heads - first);
        r.in = static_cast<const T*>(a.input) + (row0 + r.row) * a.input_stride + static_cast<int64_t>(first) * D;
        r.out = static_cast<T*>(a.output) + (row0 + r.row) * a.output_stride + static_cast<int64_t>(first) * D;
        return r;
    };
    float x[kHeads][N], y[INTERLEAVED ? 1 : kHeads][N];
    const auto load = [&](const Unit& r) {
        const int k = r.pack * kPairs;
        if (k + kPairs > pairs) return;
        const int at = INTERLEAVED ? 2 * (k0 + k) : k0 + k;
#pragma unroll
        for (int h = 0; h < kHeads; ++h)
            if (h < r.heads) {
                load_pack<T, N>(r.in + h * D + at, x[h]);
                if constexpr (!INTERLEAVED) load_pack<T, N>(r.in + h * D + at + s.pairs, y[h]);
            }
    };
    const auto turn = [&](const Unit& r) {
        const int k = r.pack * kPairs;
        if (r.pack >= packs) {
            const int lane = 2 * s.pairs + (r.pack - packs) * N;
            for (int h = 0; h < r.heads; ++h) {
                if (lane + N <= D) {
                    float v[N];
                    load_pack<T, N>(r.in + h * D + lane, v);
                    store_pack<T, N>(r.out + h * D + lane, v);
                } else {
                    for (int j = lane; j < D; ++j) r.out[h * D + j] = r.in[h * D + j];
                }
            }
        } else if (k + kPairs > pairs) {
            for (int i = k; i < pairs; ++i) {
                const f64x2 angle = angles[angle_at(r.row * pairs + i)];
                const int at = INTERLEAVED ? 2 * (k0 + i) : k0 + i, beside = INTERLEAVED ? 1 : s.pairs;
                for (int h = 0; h < r.heads; ++h) {
                    float u, v;
                    turn_pair<T>(static_cast<float>(r.in[h * D + at]), static_cast<float>(r.in[h * D + at + beside]), angle[0],
                                 angle[1], u, v);
                    r.out[h * D + at] = static_cast<T>(u);
                    r.out[h * D + at + beside] = static_cast<T>(v);
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < kPairs; ++j) {
                const f64x2 angle = angles[angle_at(r.row * pairs + k + j)];
#pragma unroll
                for (int h = 0; h < kHeads; ++h) {
                    float &u = INTERLEAVED ? x[h][2 * j] : x[h][j], &v = INTERLEAVED ? x[h][2 * j + 1] : y[INTERLEAVED ? 0 : h][j];
                    turn_pair<T>(u, v, angle[0], angle[1], u, v);
                }
            }
            const int at = INTERLEAVED ? 2 * (k0 + k) : k0 + k;
#pragma unroll
            for (int h = 0; h < kHeads; ++h)
                if (h < r.heads) {
                    store_pack<T, N>(r.out + h * D + at, x[h]);
                    if constexpr (!INTERLEAVED) store_pack<T, N>(r.out + h * D + at + s.pairs, y[h]);
                }
        }
    };

    const int all = rows * row_units;
    Unit now{};
    if (thread < all) {
        now = locate(thread);
        load(now);
    }
    if (thread < rows * pairs) {
        const int position = a.positions[row0 + thread / pairs], k = k0 + thread % pairs;
        f64x2 angle;
        if (position >= 0 && position < s.positions) {
            const double* row = s.table + static_cast<int64_t>(position) * 2 * s.pairs;
            angle[0] = row[k];
            angle[1] = row[s.pairs + k];
        } else {
            double sn, cs;
            rotation_angle(k, position, s.frequencies, s.magnitude, sn, cs);
            angle[0] = sn;
            angle[1] = cs;
        }
        angles[angle_at(thread)] = angle;
    }
    __syncthreads();
    for (int u = thread; u < all; u += kThreads) {
        if (u != thread) {
            now = locate(u);
            load(now);
        }
        turn(now);
    }
}

template <typename T, bool INTERLEAVED>
hipError_t rotate_of(const RotationShape& s, const RotateArgs& a, hipStream_t stream) {
    const int pairs = std::min(s.pairs, kThreads), parts = (s.pairs + pairs - 1) / pairs;
    const int rows = std::min(16, kThreads / pairs);
    constexpr int kMost = 1 << 22;  // (a launch's threads are counted in 32 bits)
    for (int64_t row = 0; row < a.rows; row += kMost) {
        RotateArgs part = a;
        part.rows = static_cast<int>(std::min<int64_t>(kMost, a.rows - row));
        part.input = static_cast<const T*>(a.input) + row * a.input_stride;
        part.output = static_cast<T*>(a.output) + row * a.output_stride;
        part.positions = a.positions + row;
        rotate_kernel<T, INTERLEAVED><<<dim3((part.rows + rows - 1) / rows, parts), kThreads, 0, stream>>>(s, part, rows, pairs);
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace

hipError_t launch_rotation_table(const RotationShape& shape, double* table, hipStream_t stream) {
    const int64_t n = static_cast<int64_t>(shape.positions) * shape.pairs;
    if (n <= 0) return hipSuccess;
    const int64_t groups = std::min<int64_t>((n + kThreads - 1) / kThreads, 1 << 20);  // (a launch's threads are counted in 32 bits)
    rotation_table_kernel<<<static_cast<unsigned>(groups), kThreads, 0, stream>>>(shape, table);
    return hipGetLastError();
}

hipError_t launch_rotate(const RotationShape& shape, int type, const RotateArgs& args, hipStream_t stream) {
    if (type == kF32)
        return shape.interleaved ? rotate_of<float, true>(shape, args, stream) : rotate_of<float, false>(shape, args, stream);
    return shape.interleaved ? rotate_of<_Float16, true>(shape, args, stream) : rotate_of<_Float16, false>(shape, args, stream);
}

}  // namespace satori
