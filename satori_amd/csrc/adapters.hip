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
constexpr int kSplitGroups = 256;  // workgroups that the first launch's splits make up
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

constexpr int kRankTiles = 4;  // tiles of 16 ranks that share a workgroup's input rows

// Workgroup (tile, 64 ranks, split): its waves take steps of 32 columns in turn; lane (c, g) holds columns 8 g .. 8 g + 7
// of rank c's weights (of each tile of 16 ranks) and of row c's input.
template <typename T>
__global__ __launch_bounds__(kThreads) void adapter_down_kernel(AdapterShape s, AdapterTiles tiles,
                                                                const float* __restrict__ input,
                                                                float* __restrict__ reduced, int split_columns,
                                                                bool aligned) {
    const int tile = blockIdx.x, rank0 = blockIdx.y * 16 * kRankTiles, split = blockIdx.z;
    if (tiles.adapter[tile] == kNoAdapter) return;
    const Adapter a = s.adapters[tiles.adapter[tile]];
    if (rank0 >= a.rank) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
    const int begin = tiles.begin[tile], count = tiles.begin[tile + 1] - begin;
    const int rank_tiles = min(kRankTiles, (a.rank - rank0 + 15) / 16);
    const int row = c < count ? tiles.order[begin + c] : 0;
    const float* x = input + static_cast<int64_t>(row) * s.columns;
    const T* down = static_cast<const T*>(a.down) + static_cast<int64_t>(rank0) * s.columns;
    const int first = split * split_columns;
    const int end = first + split_columns < s.columns ? first + split_columns : s.columns;
    f32x4 sum[kRankTiles];
#pragma unroll
    for (int k = 0; k < kRankTiles; ++k) sum[k] = f32x4{0, 0, 0, 0};
#pragma unroll 2
    for (int at = first + wave * kStep + 8 * g; at - 8 * g < end; at += kWaves * kStep) {
        float v[8];
        load_row(x, at, c < count ? end : 0, aligned, v);
#pragma unroll
        for (int k = 0; k < kRankTiles; ++k) {
            if (k >= rank_tiles) break;
            const bool has_rank = rank0 + 16 * k + c < a.rank;
            float w[8];
            load_row(down + static_cast<int64_t>(has_rank ? 16 * k + c : 0) * s.columns, at, has_rank ? end : 0, aligned, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) sum[k] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[j], v[j], sum[k], 0, 0, 0);
        }
    }
    __shared__ f32x4 parts[kWaves][kRankTiles][64];
#pragma unroll
    for (int k = 0; k < kRankTiles; ++k)
        if (k < rank_tiles) parts[wave][k][lane] = sum[k];
    __syncthreads();
    if (wave < rank_tiles && c < count) {  // wave k joins tile k of the ranks
        f32x4 total = parts[0][wave][lane];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) total = total + parts[w][wave][lane];
        float* out = reduced + (static_cast<int64_t>(split) * tiles.positions + row) * s.rank_most + rank0 + 16 * wave + 4 * g;
        *reinterpret_cast<f32x4*>(out) = total;
    }
}

// Workgroup (tile, 256 output rows): the tile's reduced vectors summed over the splits into LDS (eight loads in flight),
// then 64 output rows a wave; lane (c, g) holds ranks 4 g .. 4 g + 3 of a step of 16. `whole`: rows of the output and the
// base start at multiples of 16 bytes.
template <typename T>
__global__ __launch_bounds__(kThreads) void adapter_up_kernel(AdapterShape s, AdapterTiles tiles,
                                                              const float* __restrict__ reduced, const float* base,
                                                              float* output, int splits, bool whole) {
    extern __shared__ float t[];  // [16][rank_most + 4]
    const int tile = blockIdx.x;
    const int begin = tiles.begin[tile], count = tiles.begin[tile + 1] - begin;
    const bool none = tiles.adapter[tile] == kNoAdapter;
    const Adapter a = none ? Adapter{nullptr, nullptr, 0, 0.0f} : s.adapters[tiles.adapter[tile]];
    const int ranks = (a.rank + 15) / 16 * 16, stride = s.rank_most + 4;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.y * 256 + wave * 64;
    const bool has_row = c < count;
    const int64_t row = static_cast<int64_t>(has_row ? tiles.order[begin + c] : 0) * s.rows;
    f32x4 kept[4];  // the base, on its way while the rest is computed
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        const int at = n0 + 16 * n + 4 * g;
        kept[n] = f32x4{0, 0, 0, 0};
        if (!has_row) continue;
        if (whole && at + 4 <= s.rows) {
            kept[n] = *(const SATORI_GLOBAL f32x4*)(base + row + at);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (at + j < s.rows) kept[n][j] = load_f32(base + row + at + j);
        }
    }
    const int64_t next = static_cast<int64_t>(tiles.positions) * s.rank_most;
    for (int i = threadIdx.x; i < count * (ranks / 4); i += kThreads) {
        const int r = i / (ranks / 4), k = i % (ranks / 4) * 4;
        const float* from = reduced + static_cast<int64_t>(tiles.order[begin + r]) * s.rank_most + k;
        f32x4 sum{0, 0, 0, 0};
        for (int p0 = 0; p0 < splits; p0 += 8) {
            f32x4 v[8];
#pragma unroll
            for (int p = 0; p < 8; ++p)
                v[p] = p0 + p < splits ? *(const SATORI_GLOBAL f32x4*)(from + (p0 + p) * next) : f32x4{0, 0, 0, 0};
#pragma unroll
            for (int p = 0; p < 8; ++p) sum = sum + v[p];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) t[r * stride + k + j] = k + j < a.rank ? sum[j] * a.scale : 0.0f;
    }
    __syncthreads();
    f32x4 sum[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) sum[n] = f32x4{0, 0, 0, 0};
    const T* up = static_cast<const T*>(a.up);
    const bool aligned = a.rank % 4 == 0 && reinterpret_cast<uintptr_t>(up) % 16 == 0;
    for (int k = 4 * g; k - 4 * g < ranks; k += 16) {
        float v[4], w[4][4];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const int at = n0 + 16 * n + c;
            load_row(up + static_cast<int64_t>(at < s.rows ? at : 0) * a.rank, k, at < s.rows ? a.rank : 0, aligned, w[n]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = has_row ? t[c * stride + k + j] : 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int n = 0; n < 4; ++n) sum[n] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[n][j], v[j], sum[n], 0, 0, 0);
    }
    if (!has_row) return;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        const int at = n0 + 16 * n + 4 * g;
        const f32x4 out = kept[n] + sum[n];
        if (whole && at + 4 <= s.rows) {
            *(SATORI_GLOBAL f32x4*)(output + row + at) = out;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (at + j < s.rows) store_f32(output + row + at + j, out[j]);
        }
    }
}

template <typename T>
void launch(const AdapterShape& s, const AdapterTiles& tiles, const float* input, const float* base, float* output,
            float* workspace, hipStream_t stream) {
    const int ranks = (s.rank_most / 16 + kRankTiles - 1) / kRankTiles;
    // Splits of whole steps of the four waves, for about one workgroup a CU.
    const int steps = (s.columns + kWaves * kStep - 1) / (kWaves * kStep);
    const int want = std::min({std::max(1, kSplitGroups / (tiles.tiles * ranks)), steps, kMostSplits});
    const int per = (steps + want - 1) / want, splits = (steps + per - 1) / per;
    const bool aligned = s.aligned && reinterpret_cast<uintptr_t>(input) % 16 == 0;
    const bool whole = s.rows % 4 == 0 && reinterpret_cast<uintptr_t>(base) % 16 == 0 &&
                       reinterpret_cast<uintptr_t>(output) % 16 == 0;
    adapter_down_kernel<T><<<dim3(tiles.tiles, ranks, splits), kThreads, 0, stream>>>(
        s, tiles, input, workspace, per * kWaves * kStep, aligned);
    adapter_up_kernel<T><<<dim3(tiles.tiles, (s.rows + 255) / 256), kThreads, 16 * (s.rank_most + 4) * sizeof(float),
                           stream>>>(s, tiles, workspace, base, output, splits, whole);
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
