// Low-rank adapters of many requests beside one projection: y[r] = base[r] + scale * up (down x[r]) with the adapter of
// row r. Two launches: the reduced vectors t = down x, split over the columns so that a few rows still reach every CU,
// then y = base + up t; one launch for small adapters. Rows of one adapter are grouped in tiles of 16, the width of a matrix
// tile, so that its weights are read once per tile. The products are FP32 matrix instructions over the weights as they are
// (F16 converts exactly): what few rows have to multiply is little beside what they have to read.
#include "adapters.hpp"

#include <algorithm>

#include "cache_ops.hpp"
#include "device_common.hpp"

namespace satori {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr int kMostSplits = 16;  // (the second launch reads them all)
// Workgroups that the first launch's splits make up (11008 x 4096, rank 64, 256 rows of 2 adapters and 64 rows of 16: 128
// 33.4 and 33.0 us for both launches, 256 24.1 and 23.3, 512 24.4 and 22.7).
constexpr int kSplitGroups = 256;
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

// Workgroup (tile, 16 ranks, split of the columns). 256 rows of two adapters of rank 64 over 4096 columns: 8.9 us, of which the
// 0.13 GFLOP are 0.9 and the inputs' 4 x 4 MB (once per 16 ranks) through L2 the most; three splits leave 0.2 MB of sums.
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

// 16 * N output rows from n0 on of a tile's rows, with its reduced vectors `t` [16][stride] in LDS; lane (c, g) holds ranks
// 4 g .. 4 g + 3 of a step of 16 and gets output rows 4 g .. 4 g + 3 of each of N tiles, of row c. `whole`: rows of the
// output and the base start at multiples of 16 bytes.
template <int N>
struct Outputs {
    f32x4 base[N];
    int64_t row;  // of the tile's row c, in elements
    bool is;      // there is such a row
    __device__ __forceinline__ void load(const AdapterShape& s, const AdapterTiles& tiles, const Tile& tile, const float* from,
                                         int first, int n0, bool whole) {
        const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
        is = first + c < tile.count;
        row = static_cast<int64_t>(is ? tiles.order[tile.begin + first + c] : 0) * s.rows;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int at = n0 + 16 * n + 4 * g;
            base[n] = f32x4{0, 0, 0, 0};
            if (!is) continue;
            if (whole && at + 4 <= s.rows) {
                base[n] = *(const SATORI_GLOBAL f32x4*)(from + row + at);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (at + j < s.rows) base[n][j] = load_f32(from + row + at + j);
            }
        }
    }
    // `none`: the base as it is (a zero of its own sign among it).
    __device__ __forceinline__ void store(const AdapterShape& s, float* to, const f32x4 (&sum)[N], int n0, bool whole,
                                          bool none) const {
        const int g = (threadIdx.x & 63) >> 4;
        if (!is) return;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int at = n0 + 16 * n + 4 * g;
            const f32x4 out = none ? base[n] : base[n] + sum[n];
            if (whole && at + 4 <= s.rows) {
                *(SATORI_GLOBAL f32x4*)(to + row + at) = out;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (at + j < s.rows) store_f32(to + row + at + j, out[j]);
            }
        }
    }
};
// The weights of four steps of 16 ranks: read before what they are multiplied with is there.
template <typename T, int N>
struct UpWeights {
    float w[4][N][4];
    __device__ __forceinline__ void load(const AdapterShape& s, const Tile& tile, int n0, int k) {
        const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4, rank = tile.adapter.rank;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int step = k + 16 * i;
            if (step >= rank) break;
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const T* up = static_cast<const T*>(tile.adapter.up) + static_cast<int64_t>(min(n0 + 16 * n + c, s.rows - 1)) * rank;
                if (step + 16 <= rank)
                    load_inside(up, step + 4 * g, w[i][n]);
                else
                    load_at_end(up, step + 4 * g, rank, w[i][n]);
            }
        }
    }
    // Adds the product with those steps of t's rows.
    __device__ __forceinline__ void expand(const Tile& tile, const float* t, int stride, int k, f32x4 (&sum)[N]) const {
        const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (k + 16 * i >= tile.adapter.rank) break;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float v = t[c * stride + k + 16 * i + 4 * g + j];  // (rows past the last: nobody takes those)
#pragma unroll
                for (int n = 0; n < N; ++n) sum[n] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[i][n][j], v, sum[n], 0, 0, 0);
            }
        }
    }
};

// Workgroup (up to two tiles of one adapter, 128 output rows): the tiles' reduced vectors summed over the splits into LDS,
// then 32 output rows a wave, whose weights serve all the tiles (read once per tile they took 10 of 18 us at 256 rows, rank
// 64, 11008 output rows; four tiles a workgroup 16.8 us, two 15.6). That launch moves 27 MB at 1.7 TB/s: each workgroup is one
// chain of reads (its tile 0.9 us, up weights, reduced vectors and base together 3, the outputs 2.5) that starts with all
// the others.
template <typename T>
__global__ __launch_bounds__(kThreads) void adapter_up_kernel(AdapterShape s, AdapterTiles tiles,
                                                              const float* __restrict__ reduced, const float* base,
                                                              float* output, int splits, bool whole) {
    extern __shared__ float t[];  // [16 * kGroupTiles][rank_most + 4]
    Tile tile = tile_of(s, tiles, tiles.group[blockIdx.x]);
    tile.count = tiles.begin[tiles.group[blockIdx.x + 1]] - tile.begin;
    const int wave = threadIdx.x >> 6, n0 = blockIdx.y * 128 + wave * 32, stride = s.rank_most + 4;
    UpWeights<T, 2> up;
    up.load(s, tile, n0, 0);
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
    Outputs<2> out[kGroupTiles];
#pragma unroll
    for (int r = 0; r < kGroupTiles; ++r)
        if (16 * r < tile.count) out[r].load(s, tiles, tile, base, 16 * r, n0, whole);
    __syncthreads();
    f32x4 sum[kGroupTiles][2];
#pragma unroll
    for (int r = 0; r < kGroupTiles; ++r) sum[r][0] = sum[r][1] = f32x4{0, 0, 0, 0};
    for (int k = 0; k < tile.adapter.rank; k += 64) {
        if (k > 0) up.load(s, tile, n0, k);
#pragma unroll
        for (int r = 0; r < kGroupTiles; ++r)
            if (16 * r < tile.count) up.expand(tile, t + 16 * r * stride, stride, k, sum[r]);
    }
#pragma unroll
    for (int r = 0; r < kGroupTiles; ++r)
        if (16 * r < tile.count) out[r].store(s, output, sum[r], n0, whole, tile.none);
}

// Both products in one launch, for adapters of one tile of ranks and short rows: workgroup (tile, 512 output rows or less)
// makes the tile's whole reduced vectors for itself, 1024 columns a turn of its waves, which takes as long as the second
// launch would from some columns on. One launch against two, 32 rows of 32 adapters of rank 16, 1536 output rows: F16 1024
// columns 6.4 us and 9.1, 2048 8.2 and 8.9, 2560 10.0 and 9.0, 8192 21 and 11.7; FP32 1024 7.2 and 9.0, 1477 8.9 and 9.1, 2048
// 10.1 and 9.3; rank 32, F16, 1024 columns 9.5 and 9.0. And for few workgroups, each of which reads a tile's weights and rows:
// 1536 columns, adapters of one row, 64 over 1536 output rows (10.6 MB) 9.0 and 10.5, 128 (21 MB) 17.5 and 15.4, 32 over 4096
// (14 MB) 8.8 and 10.1, over 8192 (28 MB) 17.2 and 15.1; 256 rows of one adapter over 4096 (19 MB) 13.2 and 11.8.
constexpr int kBothWaves = 8;
constexpr int kBothRank = 16;
constexpr int64_t kBothBytes = 16 << 20;
constexpr int both_columns(int type) { return type == kF32 ? 1536 : 2048; }

template <typename T>
__global__ __launch_bounds__(kBothWaves * 64) void adapter_both_kernel(AdapterShape s, AdapterTiles tiles,
                                                                       const float* __restrict__ input, const float* base,
                                                                       float* output, int rows_each, bool whole) {
    __shared__ f32x4 parts[kBothWaves][64];
    __shared__ float t[16][kBothRank + 4];
    const Tile tile = tile_of(s, tiles, blockIdx.x);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.y * rows_each + wave * 64;
    const bool works = wave * 64 < rows_each && n0 < s.rows;
    UpWeights<T, 4> up;
    Outputs<4> out;
    if (works) {
        up.load(s, tile, n0, 0);
        out.load(s, tiles, tile, base, 0, n0, whole);
    }
    const float* x = input + static_cast<int64_t>(tiles.order[tile.begin + (c < tile.count ? c : 0)]) * s.columns;
    if (!tile.none) parts[wave][lane] = reduce<T>(s, tile, x, 0, wave * kStep, kBothWaves * kStep, s.columns);
    __syncthreads();
    if (wave == 0 && !tile.none) {
        f32x4 total = parts[0][lane];
#pragma unroll
        for (int w = 1; w < kBothWaves; ++w) total = total + parts[w][lane];
#pragma unroll
        for (int j = 0; j < 4; ++j) t[c][4 * g + j] = 4 * g + j < tile.adapter.rank ? total[j] * tile.adapter.scale : 0.0f;
    }
    __syncthreads();
    if (!works) return;
    f32x4 sum[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) sum[n] = f32x4{0, 0, 0, 0};
    up.expand(tile, &t[0][0], kBothRank + 4, 0, sum);
    out.store(s, output, sum, n0, whole, tile.none);
}

template <typename T>
hipError_t launch(const AdapterShape& s, const AdapterTiles& tiles, const float* input, const float* base, float* output,
            float* workspace, hipStream_t stream) {
    const bool whole = s.rows % 4 == 0 && reinterpret_cast<uintptr_t>(base) % 16 == 0 &&
                       reinterpret_cast<uintptr_t>(output) % 16 == 0;
    const int ranks = s.rank_most / 16;
    const int64_t both_bytes = (static_cast<int64_t>(tiles.tiles) * kBothRank * sizeof(T) + tiles.positions * sizeof(float)) *
                               s.columns * ((s.rows + 511) / 512);
    if (s.rank_most <= kBothRank && s.columns <= both_columns(s.type) && both_bytes <= kBothBytes) {
        // 64 rows a wave and turn; fewer waves work on them where that lets more CUs share them.
        int each = 512;
        while (each > 64 && tiles.tiles * ((s.rows + each - 1) / each) < 128) each /= 2;
        adapter_both_kernel<T><<<dim3(tiles.tiles, (s.rows + each - 1) / each), kBothWaves * 64, 0, stream>>>(
            s, tiles, input, base, output, each, whole);
        return hipGetLastError();
    }
    // Splits of whole steps of the four waves, for about one workgroup a CU.
    const int steps = (s.columns + kWaves * kStep - 1) / (kWaves * kStep);
    const int want = std::min({std::max(1, kSplitGroups / (tiles.tiles * ranks)), steps, kMostSplits});
    const int per = (steps + want - 1) / want, splits = (steps + per - 1) / per;
    adapter_down_kernel<T><<<dim3(tiles.tiles, ranks, splits), kThreads, 0, stream>>>(s, tiles, input, workspace,
                                                                                               per * kWaves * kStep);
    const int lds = 16 * kGroupTiles * (s.rank_most + 4) * static_cast<int>(sizeof(float));
    if (lds > 64 * 1024)
        if (const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(adapter_up_kernel<T>),
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, lds);
            e != hipSuccess)
            return e;
    adapter_up_kernel<T><<<dim3(tiles.groups, (s.rows + 127) / 128), kThreads, lds, stream>>>(s, tiles, workspace, base, output,
                                                                                             splits, whole);
    return hipGetLastError();
}

}  // namespace

size_t adapter_workspace_bytes(const AdapterShape& s) {
    return static_cast<size_t>(kMostSplits) * kAdapterRows * s.rank_most * sizeof(float);
}

hipError_t launch_adapters(const AdapterShape& s, const AdapterTiles& tiles, const float* input, const float* base,
                           float* output, float* workspace, hipStream_t stream) {
    if (tiles.tiles == 0) return hipSuccess;
    return (s.type == kF32 ? launch<float> : launch<_Float16>)(s, tiles, input, base, output, workspace, stream);
}

}  // namespace satori
