// Launchers of the low-rank adapters' kernels (adapters.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace satori {

// One adapter on the device: down [rank][columns] and up [rows][rank], row-major.
struct Adapter {
    const void* down;
    const void* up;
    int rank;
    float scale;
};

constexpr int kAdapterRows = 256;  // positions of one launch
constexpr int kMaxAdapters = 65535;
constexpr int kMaxRank = 512;     // a run of two tiles' reduced vectors lie in 66 KB of LDS then

// The rows of a launch by adapter: tile i is rows order[begin[i]] .. order[begin[i + 1] - 1] (16 at most) of adapter[i],
// kNoAdapter for rows without one. In the launch's arguments, so a captured launch keeps what it was called with.
constexpr uint16_t kNoAdapter = 65535;
constexpr int kGroupTiles = 2;
struct AdapterTiles {
    int tiles, positions, groups;
    uint8_t order[kAdapterRows];
    uint16_t begin[kAdapterRows + 1], adapter[kAdapterRows];
    uint16_t group[kAdapterRows + 1];  // runs of at most kGroupTiles tiles of one adapter: tiles group[i] .. group[i + 1] - 1
};

struct AdapterShape {
    const Adapter* adapters;  // device
    int rows, columns;
    int rank_most;            // largest rank, rounded up to a multiple of 16
    int type;                 // Element (cache_ops.hpp): kF32 or kF16
};

// Bytes of `workspace` (the rows' reduced vectors, [splits][positions][rank_most]).
size_t adapter_workspace_bytes(const AdapterShape& shape);
hipError_t launch_adapters(const AdapterShape& shape, const AdapterTiles& tiles, const float* input, const float* base,
                           float* output, float* workspace, hipStream_t stream);

}  // namespace satori
