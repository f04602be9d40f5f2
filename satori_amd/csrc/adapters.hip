// Low-rank adapters of many requests beside one projection: y[r] = base[r] + scale * up (down x[r]) with the adapter of
// row r. Two launches: the reduced vectors t = down x, split over the columns so that a few rows still reach every CU,
// then y = base + up t. Rows of one adapter are grouped in tiles of 16, the width of a matrix tile, so that its weights
// are read once per tile. The products are FP32 matrix instructions over the weights as they are (F16 converts exactly).
#include "adapters.hpp"

#include <algorithm>

#include "cache_ops.hpp"
#include "device_common.hpp"

namespace satori {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr int kMostSplits = 16;
constexpr int kStep = 32;  // columns a wave takes at once

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

// Elements at .. at + N - 1 of a row of `length`, zero behind it; as FP32. `aligned`: the addresses of the row's groups of
// N elements are multiples of their bytes (of 16 at most).
template <typename T, int N>
__device__ __forceinline__ void load_row(const T* row, int at, int length, bool aligned, float (&out)[N]) {
    if (aligned && at + N <= length) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < N; i += 4) {
                const f32x4 v = *(const SATORI_GLOBAL f32x4*)(row + at + i);
#pragma unroll
                for (int j = 0; j < 4; ++j) out[i + j] = v[j];
            }
        } else if constexpr (N == 8) {
            const f16x8 v = *(const SATORI_GLOBAL f16x8*)(row + at);
#pragma unroll
            for (int j = 0; j < 8; ++j) out[j] = static_cast<float>(v[j]);
        } else {
            const f16x4 v = *(const SATORI_GLOBAL f16x4*)(row + at);
#pragma unroll
            for (int j = 0; j < 4; ++j) out[j] = static_cast<float>(v[j]);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
        out[i] = at + i < length ? static_cast<float>(*(const SATORI_GLOBAL T*)(row + at + i)) : 0.0f;
}

// Workgroup (tile, 16 ranks, split): its waves take steps of 32 columns in turn; lane (c, g) holds columns 8 g .. 8 g + 7
// of rank c's weights and of row c's input.
template <typename T>
__global__ __launch_bounds__(kThreads) void adapter_down_kernel(AdapterShape s, AdapterTiles tiles,
                                                                const float* __restrict__ input,
                                                                float* __restrict__ reduced, int split_columns,
                                                                bool aligned) {
    const int tile = blockIdx.x, rank0 = blockIdx.y * 16, split = blockIdx.z;
    if (tiles.adapter[tile] == kNoAdapter) return;
    const Adapter a = s.adapters[tiles.adapter[tile]];
    if (rank0 >= a.rank) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
    const int begin = tiles.begin[tile], count = tiles.begin[tile + 1] - begin;
    const bool has_rank = rank0 + c < a.rank, has_row = c < count;
    const T* down = static_cast<const T*>(a.down) + static_cast<int64_t>(has_rank ? rank0 + c : 0) * s.columns;
    const int row = has_row ? tiles.order[begin + c] : 0;
    const float* x = input + static_cast<int64_t>(row) * s.columns;
    const int first = split * split_columns;
    const int end = first + split_columns < s.columns ? first + split_columns : s.columns;
    f32x4 sum{0, 0, 0, 0};
    for (int at = first + wave * kStep + 8 * g; at - 8 * g < end; at += kWaves * kStep) {
        float w[8], v[8];
        load_row(down, at, has_rank ? end : 0, aligned, w);
        load_row(x, at, has_row ? end : 0, aligned, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) sum = __builtin_amdgcn_mfma_f32_16x16x4f32(w[j], v[j], sum, 0, 0, 0);
    }
    __shared__ f32x4 parts[kWaves][64];
    parts[wave][lane] = sum;
    __syncthreads();
    if (wave == 0 && has_row) {
#pragma unroll
        for (int w = 1; w < kWaves; ++w) sum = sum + parts[w][lane];
        float* out = reduced + (static_cast<int64_t>(split) * tiles.positions + row) * s.rank_most + rank0 + 4 * g;
        *reinterpret_cast<f32x4*>(out) = sum;
    }
}

// Workgroup (tile, 256 output rows): the tile's reduced vectors summed over the splits into LDS, then 64 output rows a
// wave; lane (c, g) holds ranks 4 g .. 4 g + 3 of a step of 16.
template <typename T>
__global__ __launch_bounds__(kThreads) void adapter_up_kernel(AdapterShape s, AdapterTiles tiles,
                                                              const float* __restrict__ reduced, const float* base,
                                                              float* output, int splits) {
    extern __shared__ float t[];  // [16][rank_most + 4]
    const int tile = blockIdx.x;
    const int begin = tiles.begin[tile], count = tiles.begin[tile + 1] - begin;
    const bool none = tiles.adapter[tile] == kNoAdapter;
    const Adapter a = none ? Adapter{nullptr, nullptr, 0, 0.0f} : s.adapters[tiles.adapter[tile]];
    const int ranks = (a.rank + 15) / 16 * 16, stride = s.rank_most + 4;
    for (int i = threadIdx.x; i < count * ranks; i += kThreads) {
        const int r = i / ranks, k = i % ranks;
        float sum = 0;
        if (k < a.rank)
            for (int p = 0; p < splits; ++p)
                sum += reduced[(static_cast<int64_t>(p) * tiles.positions + tiles.order[begin + r]) * s.rank_most + k];
        t[r * stride + k] = sum * a.scale;
    }
    __syncthreads();
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.y * 256 + wave * 64;
    f32x4 sum[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) sum[n] = f32x4{0, 0, 0, 0};
    const T* up = static_cast<const T*>(a.up);
    const bool aligned = a.rank % 4 == 0 && reinterpret_cast<uintptr_t>(up) % 16 == 0;
    for (int k = 4 * g; k - 4 * g < ranks; k += 16) {
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = c < count ? t[c * stride + k + j] : 0.0f;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const int at = n0 + 16 * n + c;
            float w[4];
            load_row(up + static_cast<int64_t>(at < s.rows ? at : 0) * a.rank, k, at < s.rows ? a.rank : 0, aligned, w);
#pragma unroll
            for (int j = 0; j < 4; ++j) sum[n] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[j], v[j], sum[n], 0, 0, 0);
        }
    }
    if (c >= count) return;
    const int64_t row = static_cast<int64_t>(tiles.order[begin + c]) * s.rows;
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int at = n0 + 16 * n + 4 * g + j;
            if (at < s.rows) output[row + at] = base[row + at] + sum[n][j];
        }
}

template <typename T>
void launch(const AdapterShape& s, const AdapterTiles& tiles, const float* input, const float* base, float* output,
            float* workspace, hipStream_t stream) {
    const int ranks = s.rank_most / 16;
    // Splits of whole steps of the four waves, for about two workgroups a CU.
    const int steps = (s.columns + kWaves * kStep - 1) / (kWaves * kStep);
    const int want = std::min({std::max(1, 512 / (tiles.tiles * ranks)), steps, kMostSplits});
    const int per = (steps + want - 1) / want, splits = (steps + per - 1) / per;
    const bool aligned = s.aligned && reinterpret_cast<uintptr_t>(input) % 16 == 0;
    adapter_down_kernel<T><<<dim3(tiles.tiles, ranks, splits), kThreads, 0, stream>>>(
        s, tiles, input, workspace, per * kWaves * kStep, aligned);
    adapter_up_kernel<T><<<dim3(tiles.tiles, (s.rows + 255) / 256), kThreads, 16 * (s.rank_most + 4) * sizeof(float),
                           stream>>>(s, tiles, workspace, base, output, splits);
}

}  // namespace

size_t adapter_workspace_bytes(const AdapterShape& s) {
    return static_cast<size_t>(kMostSplits) * kAdapterRows * s.rank_most * sizeof(float);
}

hipError_t launch_adapters(const AdapterShape& s, const AdapterTiles& tiles, const float* input, const float* base,
                           float* output, float* workspace, hipStream_t stream) {
    if (tiles.tiles == 0) return hipSuccess;
    (s.type == kF32 ? launch<float> : launch<_Float16>)(s, tiles, input, base, output, workspace, stream);
    return hipGetLastError();
}

}  // namespace satori
