// Launchers of the paged key/value cache's kernels (cache_ops.hip).
//
// A pool is [pages][layers][keys, values]: a page's keys of a layer [kv_heads][page_tokens][width], its values
// [kv_heads][width][page_tokens], `width` being the head dimension rounded up to a supported one (cache_width). Values lie
// transposed because that is the order in which the matrix instructions take them: a wave reads both operands of a tile
// with 16-byte loads from the cache straight into registers, and no page's bytes pass through LDS. A page of all layers
// is one run of bytes, so that copying it is one copy.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "pages.hpp"

namespace satori {

enum Element : int { kF32 = 0, kF16 = 1 };

inline int element_bytes(int type) { return type == kF32 ? 4 : 2; }

// The width that heads of `head_dim` lanes are kept at, or 0 past 256.
inline int cache_width(int head_dim) {
    for (int w : {32, 64, 96, 128, 192, 256})
        if (head_dim <= w) return w;
    return 0;
}

struct CacheShape {
    uint8_t* pool;
    int64_t page_bytes, layer_bytes;  // of one page; of one layer's keys and values in it
    int page_tokens, page_shift;      // 1 << page_shift tokens
    int heads, kv_heads, head_dim, width;
    int type;                         // Element
};

// Pairs of a wide attention workgroup (PlanShape::wide_pairs).
int cache_wide_pairs(int type, int width);

// Copies what a plan's arrays hold from pinned host memory to the same places of the image on the device.
hipError_t launch_plan_copy(const int* from, int* to, const PlanLayout& layout, const PlanLayout& used, hipStream_t stream);

constexpr int kMovesPerLaunch = 224;  // pairs of page numbers in a launch's arguments
struct PageMoves {
    int count, pad;
    int source[kMovesPerLaunch], destination[kMovesPerLaunch];
};
// pool page destination[i] = pool page source[i]; no page is in both lists.
hipError_t launch_copy_pages(uint8_t* pool, int64_t page_bytes, const PageMoves& moves, hipStream_t stream);

struct AppendArgs {
    const float *query, *query_bias, *key, *key_bias, *value, *value_bias;
    float* query_out;
    double base;
    int rotary;
    const double* rope;   // table of rope_positions rows, or null
    int rope_positions;
    int layer;
};
// `image`: a plan's on the device, `now` its header. `all`: the launch is captured and replays may read any plan, so its
// grid must do for any.
hipError_t launch_cache_append(const CacheShape& shape, const int* image, const PlanLayout& layout, const PlanHeader& now,
                               bool all, const AppendArgs& args, hipStream_t stream);

// `partials`: at least cache_partial_bytes for the plan's slots. Launches with no work now are left out unless `all`.
size_t cache_partial_bytes(const CacheShape& shape, int64_t slots);
hipError_t launch_cache_attention(const CacheShape& shape, const int* image, const PlanLayout& layout, const PlanHeader& now,
                                  bool all, int layer, const float* query, float* output, float* partials, size_t bytes,
                                  hipStream_t stream);

}  // namespace satori
