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
constexpr int64_t kBothBytes = 24 << 20;  // weights that one launch may read, tiles times the workgroups that read them
constexpr int kSplitGroups = 256;  // workgroups that the first launch's splits make up
constexpr int kStep = 32;  // columns a wave takes at once

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

// N elements of a row from `at` on, as FP32, in one read (two for eight of FP32) at any element's address.
template <int N, typename T>
__device__ __forceinline__ void load_inside(const T* row, int at, float (&out)[N]) {
    constexpr int kGroup = N * sizeof(T) > 16 ? 16 / sizeof(T) : N;
    typedef T pack __attribute__((ext_vector_type(kGroup), aligned(sizeof(T))));
#pragma unroll
    for (int i = 0; i < N; i += kGroup) {
        const pack v = *(const SATORI_GLOBAL pack*)(row + at + i);
#pragma unroll
        for (int j = 0; j < kGroup; ++j) out[i + j] = static_cast<float>(v[j]);
    }
}
// The same where the row may end: zero from `end` on.
template <int N, typename T>
__device__ __forceinline__ void load_at_end(const T* row, int at, int end, float (&out)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const T v = *(const SATORI_GLOBAL T*)(row + min(at + i, end - 1));
        out[i] = at + i < end ? static_cast<float>(v) : 0.0f;
    }
}

// What a launch knows of a tile: its adapter and rows.
struct Tile {
    Adapter adapter;
    int begin, count;
    bool none;
};
__device__ __forceinline__ Tile tile_of(const AdapterShape& s, const AdapterTiles& tiles, int tile) {
    Tile t;
    t.begin = tiles.begin[tile];
    t.count = tiles.begin[tile + 1] - t.begin;
    t.none = tiles.adapter[tile] == kNoAdapter;
    t.adapter = t.none ? Adapter{nullptr, nullptr, 0, 0.0f} : s.adapters[tiles.adapter[tile]];
    return t;
}

// A wave's part of 16 ranks of a tile's reduced vectors: steps of 32 columns from `first` on, `stride` apart, four of them
// read at once; lane (c, g) holds columns 8 g .. 8 g + 7 of rank c's weights and of row c's input, and gets ranks
// 4 g .. 4 g + 3 of row c. (Ranks past the last repeat the first, rows past the last the tile's first: nobody takes those.)
template <typename T>
__device__ __forceinline__ f32x4 reduce(const AdapterShape& s, const Tile& tile, const float* x, int rank0, int first, int stride,
                                        int end) {
    constexpr int kAtOnce = 4;
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const T* down = static_cast<const T*>(tile.adapter.down) +
                    static_cast<int64_t>(rank0 + c < tile.adapter.rank ? rank0 + c : 0) * s.columns;
    f32x4 sum{0, 0, 0, 0};
    for (int at = first; at < end; at += kAtOnce * stride) {
        float w[kAtOnce][8] = {}, v[kAtOnce][8] = {};
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const int step = at + i * stride;
            if (step + kStep <= end) {
                load_inside(down, step + 8 * g, w[i]);
                load_inside(x, step + 8 * g, v[i]);
            } else if (step < end) {
                load_at_end(down, step + 8 * g, end, w[i]);
                load_at_end(x, step + 8 * g, end, v[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) sum = __builtin_amdgcn_mfma_f32_16x16x4f32(w[i][j], v[i][j], sum, 0, 0, 0);
    }
    return sum;
}

// Workgroup (tile, 16 ranks, split of the columns).
template <typename T>
__global__ __launch_bounds__(kThreads) void adapter_down_kernel(AdapterShape s, AdapterTiles tiles,
                                                                const float* __restrict__ input,
                                                                float* __restrict__ reduced, int split_columns) {
    const Tile tile = tile_of(s, tiles, blockIdx.x);
    const int rank0 = blockIdx.y * 16, split = blockIdx.z;
    if (rank0 >= tile.adapter.rank) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
    const int row = c < tile.count ? tiles.order[tile.begin + c] : 0;
    const int first = split * split_columns;
    f32x4 sum = reduce<T>(s, tile, input + static_cast<int64_t>(row) * s.columns, rank0, first + wave * kStep,
                                   kWaves * kStep, first + split_columns < s.columns ? first + split_columns : s.columns);
    __shared__ f32x4 parts[kWaves][64];
    parts[wave][lane] = sum;
    __syncthreads();
    if (wave == 0 && c < tile.count) {
#pragma unroll
        for (int w = 1; w < kWaves; ++w) sum = sum + parts[w][lane];
        *reinterpret_cast<f32x4*>(reduced + (static_cast<int64_t>(split) * tiles.positions + row) * s.rank_most + rank0 + 4 * g) = sum;
    }
}

// 64 output rows from n0 on of a tile's rows, with its reduced vectors `t` [16][stride] in LDS; lane (c, g) holds ranks
// 4 g .. 4 g + 3 of a step of 16 and gets output rows 4 g .. 4 g + 3 of each of four tiles, of row c. `whole`: rows of the
// output and the base start at multiples of 16 bytes.
struct Kept {
    f32x4 v[4];
};
__device__ __forceinline__ Kept load_base(const AdapterShape& s, const float* base, int64_t row, bool has_row, int n0, bool whole) {
    const int g = (threadIdx.x & 63) >> 4;
    Kept kept;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        const int at = n0 + 16 * n + 4 * g;
        kept.v[n] = f32x4{0, 0, 0, 0};
        if (!has_row) continue;
        if (whole && at + 4 <= s.rows) {
            kept.v[n] = *(const SATORI_GLOBAL f32x4*)(base + row + at);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (at + j < s.rows) kept.v[n][j] = load_f32(base + row + at + j);
        }
    }
    return kept;
}
// The weights of four steps of 16 ranks: read before what they are multiplied with is there.
template <typename T>
struct UpWeights {
    float w[4][4][4];
    __device__ __forceinline__ void load(const AdapterShape& s, const Tile& tile, int n0, int k) {
        const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4, rank = tile.adapter.rank;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int step = k + 16 * i;
            if (step >= rank) break;
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const T* up = static_cast<const T*>(tile.adapter.up) + static_cast<int64_t>(min(n0 + 16 * n + c, s.rows - 1)) * rank;
                if (step + 16 <= rank)
                    load_inside(up, step + 4 * g, w[i][n]);
                else
                    load_at_end(up, step + 4 * g, rank, w[i][n]);
            }
        }
    }
};
template <typename T>
__device__ __forceinline__ void expand(const AdapterShape& s, const Tile& tile, UpWeights<T>& up, const float* t, int stride,
                                       const Kept& kept, float* output, int64_t row, bool has_row, int n0, bool whole) {
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4, rank = tile.adapter.rank;
    f32x4 sum[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) sum[n] = f32x4{0, 0, 0, 0};
    for (int k = 0; k < rank; k += 64) {
        if (k > 0) up.load(s, tile, n0, k);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (k + 16 * i >= rank) break;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float v = t[c * stride + k + 16 * i + 4 * g + j];  // (rows past the last: nobody takes those)
#pragma unroll
                for (int n = 0; n < 4; ++n) sum[n] = __builtin_amdgcn_mfma_f32_16x16x4f32(up.w[i][n][j], v, sum[n], 0, 0, 0);
            }
        }
    }
    if (!has_row) return;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        const int at = n0 + 16 * n + 4 * g;
        const f32x4 out = kept.v[n] + sum[n];
        if (whole && at + 4 <= s.rows) {
            *(SATORI_GLOBAL f32x4*)(output + row + at) = out;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (at + j < s.rows) store_f32(output + row + at + j, out[j]);
        }
    }
}

// Workgroup (tile, 256 output rows): the tile's reduced vectors summed over the splits into LDS, then 64 output rows a wave.
template <typename T>
__global__ __launch_bounds__(kThreads) void adapter_up_kernel(AdapterShape s, AdapterTiles tiles,
                                                              const float* __restrict__ reduced, const float* base,
                                                              float* output, int splits, bool whole) {
    extern __shared__ float t[];  // [16][rank_most + 4]
    const Tile tile = tile_of(s, tiles, blockIdx.x);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15;
    const int n0 = blockIdx.y * 256 + wave * 64, stride = s.rank_most + 4;
    const bool has_row = c < tile.count;
    const int64_t row = static_cast<int64_t>(has_row ? tiles.order[tile.begin + c] : 0) * s.rows;
    UpWeights<T> up;
    up.load(s, tile, n0, 0);
    const Kept kept = load_base(s, base, row, has_row, n0, whole);
    const int quads = (tile.adapter.rank + 15) / 16 * 4;
    const int64_t next = static_cast<int64_t>(tiles.positions) * s.rank_most;
    for (int i = threadIdx.x; i < tile.count * quads; i += kThreads) {
        const int r = i / quads, k = i % quads * 4;
        const float* from = reduced + static_cast<int64_t>(tiles.order[tile.begin + r]) * s.rank_most + k;
        f32x4 sum{0, 0, 0, 0};
        for (int p0 = 0; p0 < splits; p0 += 4) {
            f32x4 v[4];
#pragma unroll
            for (int p = 0; p < 4; ++p)
                v[p] = p0 + p < splits ? *(const SATORI_GLOBAL f32x4*)(from + (p0 + p) * next) : f32x4{0, 0, 0, 0};
#pragma unroll
            for (int p = 0; p < 4; ++p) sum = sum + v[p];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) t[r * stride + k + j] = k + j < tile.adapter.rank ? sum[j] * tile.adapter.scale : 0.0f;
    }
    __syncthreads();
    expand<T>(s, tile, up, t, stride, kept, output, row, has_row, n0, whole);
}

// Both products in one launch, for small adapters and few tiles: workgroup (tile, 512 output rows or less) makes the tile's
// whole reduced vectors for itself.
constexpr int kBothWaves = 8;
constexpr int kBothRanks = 4;  // tiles of 16 ranks

template <typename T>
__global__ __launch_bounds__(kBothWaves * 64) void adapter_both_kernel(AdapterShape s, AdapterTiles tiles,
                                                                       const float* __restrict__ input, const float* base,
                                                                       float* output, int rows_each, bool whole) {
    __shared__ f32x4 parts[kBothWaves][64];
    __shared__ float t[16][16 * kBothRanks + 4];
    const Tile tile = tile_of(s, tiles, blockIdx.x);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
    const bool has_row = c < tile.count;
    const int order = has_row ? tiles.order[tile.begin + c] : 0;
    const int64_t row = static_cast<int64_t>(order) * s.rows;
    const int n0 = blockIdx.y * rows_each + wave * 64;
    const bool works = wave * 64 < rows_each && n0 < s.rows;
    Kept kept{};
    UpWeights<T> up;
    if (works) {
        up.load(s, tile, n0, 0);
        kept = load_base(s, base, row, has_row, n0, whole);
    }
    for (int rank0 = 0; rank0 < tile.adapter.rank; rank0 += 16) {
        const f32x4 sum = reduce<T>(s, tile, input + static_cast<int64_t>(order) * s.columns, rank0, wave * kStep,
                                             kBothWaves * kStep, s.columns);
        if (rank0) __syncthreads();
        parts[wave][lane] = sum;
        __syncthreads();
        if (wave == 0) {
            f32x4 total = sum;
#pragma unroll
            for (int w = 1; w < kBothWaves; ++w) total = total + parts[w][lane];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int k = rank0 + 4 * g + j;
                t[c][k] = k < tile.adapter.rank ? total[j] * tile.adapter.scale : 0.0f;
            }
        }
    }
    __syncthreads();
    if (works) expand<T>(s, tile, up, &t[0][0], 16 * kBothRanks + 4, kept, output, row, has_row, n0, whole);
}

template <typename T>
void launch(const AdapterShape& s, const AdapterTiles& tiles, const float* input, const float* base, float* output,
            float* workspace, hipStream_t stream) {
    const bool whole = s.rows % 4 == 0 && reinterpret_cast<uintptr_t>(base) % 16 == 0 &&
                       reinterpret_cast<uintptr_t>(output) % 16 == 0;
    const int ranks = s.rank_most / 16;
    const int64_t both_groups = static_cast<int64_t>(tiles.tiles) * ((s.rows + 511) / 512);
    if (ranks <= kBothRanks && both_groups * ranks * 16 * s.columns * static_cast<int64_t>(sizeof(T)) <= kBothBytes) {
        // 64 rows a wave and turn; fewer waves work on them where that lets more CUs share them.
        int each = 512;
        while (each > 64 && tiles.tiles * ((s.rows + each - 1) / each) < 128) each /= 2;
        adapter_both_kernel<T><<<dim3(tiles.tiles, (s.rows + each - 1) / each), kBothWaves * 64, 0, stream>>>(
            s, tiles, input, base, output, each, whole);
        return;
    }
    // Splits of whole steps of the four waves, for about one workgroup a CU.
    const int steps = (s.columns + kWaves * kStep - 1) / (kWaves * kStep);
    const int want = std::min({std::max(1, kSplitGroups / (tiles.tiles * ranks)), steps, kMostSplits});
    const int per = (steps + want - 1) / want, splits = (steps + per - 1) / per;
    adapter_down_kernel<T><<<dim3(tiles.tiles, ranks, splits), kThreads, 0, stream>>>(s, tiles, input, workspace,
                                                                                               per * kWaves * kStep);
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
