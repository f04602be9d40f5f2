// Kernels of the paged key/value cache: page copies, the write of new positions and the attention of a batch whose
// sequences share pages.
#include <algorithm>
#include <cmath>

#include "cache_ops.hpp"
#include "device_common.hpp"
#include "rope_device.hpp"

namespace satori {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kThreads = 256;

// ---- page copies ----

// Each workgroup copies kCopyBytes of one page, 16 bytes a thread and access, four accesses in flight.
constexpr int kCopyBytes = kThreads * 16 * 4;

__global__ __launch_bounds__(kThreads) void copy_pages_kernel(uint8_t* pool, int64_t page_bytes, PageMoves moves) {
    const int64_t at = static_cast<int64_t>(blockIdx.x) * kCopyBytes + threadIdx.x * 16;
    const uint8_t* src = pool + moves.source[blockIdx.y] * page_bytes;
    uint8_t* dst = pool + moves.destination[blockIdx.y] * page_bytes;
    u32x4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (at + i * kThreads * 16 < page_bytes) v[i] = *(const SATORI_GLOBAL u32x4*)(src + at + i * kThreads * 16);
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (at + i * kThreads * 16 < page_bytes) *(SATORI_GLOBAL u32x4*)(dst + at + i * kThreads * 16) = v[i];
}

// ---- the write of new positions ----

template <typename T, int N>
__device__ __forceinline__ void store_as(T* p, const float (&v)[N]) {
    typedef T pack __attribute__((ext_vector_type(N)));
    pack out;
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = static_cast<T>(v[i]);
    *(SATORI_GLOBAL pack*)(p) = out;
}
template <typename T>
__device__ __forceinline__ void store_as(T* p, const float (&v)[1]) {
    *(SATORI_GLOBAL T*)(p) = static_cast<T>(v[0]);
}

// N values of a row with their bias (biased()), in one load each.
template <int N>
__device__ __forceinline__ void load_biased(const float* x, const float* bias, int64_t at, int lane, float (&out)[N]) {
    typedef float pack __attribute__((ext_vector_type(N)));
    if constexpr (N == 1) {
        out[0] = biased(x + at, bias, lane);
    } else {
        const pack v = *(const SATORI_GLOBAL pack*)(x + at + lane);
        pack b{};
        if (bias) b = *(const SATORI_GLOBAL pack*)(bias + lane);
#pragma unroll
        for (int i = 0; i < N; ++i) out[i] = bias ? __fadd_rn(v[i], b[i]) : v[i];
    }
}

constexpr int kGroupTokens = 8;  // positions whose values a thread stores at once

// The rows of a run, spread over gridDim.y workgroups: N rotated lane pairs of a query or key head per thread and turn,
// then the lanes behind the rotated ones and the keys' padding, then the values. A page's values lie [lane][position], so a
// thread gathers one lane of up to eight positions (its neighbours the next lanes: the reads are whole lines) and stores
// them together where they fill an aligned group.
template <typename T, int N>
__global__ __launch_bounds__(kThreads) void cache_append_kernel(CacheShape s, const int* __restrict__ plan,
                                                                AppendArgs a) {
    const PlanHeader& h = *reinterpret_cast<const PlanHeader*>(plan);
    const PlanRun* runs = reinterpret_cast<const PlanRun*>(plan + h.runs_at);
    const PlanRow* rows = reinterpret_cast<const PlanRow*>(plan + h.rows_at);
    const int pairs = a.rotary / 2, D = s.head_dim, both = s.heads + s.kv_heads;
    const int64_t head_size = static_cast<int64_t>(s.page_tokens) * s.width;
    for (int u = blockIdx.x; u < h.runs; u += gridDim.x) {
        const PlanRun run = runs[u];
        const int position0 = rows[run.row].position;
        T* keys = reinterpret_cast<T*>(s.pool + run.page * s.page_bytes + a.layer * s.layer_bytes);
        T* values = keys + s.kv_heads * head_size;
        const int start = blockIdx.y * kThreads + threadIdx.x, stride = gridDim.y * kThreads;
        const int packs = pairs / N;
        for (int i = start; i < run.tokens * both * packs; i += stride) {
            const int kk = i % packs * N, rest = i / packs, head = rest % both, t = rest / both;
            const int position = position0 + t;
            const bool is_query = head < s.heads;
            const int lane = (is_query ? head : head - s.heads) * D + kk;
            const int64_t at = static_cast<int64_t>(run.row + t) * (is_query ? s.heads : s.kv_heads) * D;
            float x[N], y[N];
            load_biased(is_query ? a.query : a.key, is_query ? a.query_bias : a.key_bias, at, lane, x);
            load_biased(is_query ? a.query : a.key, is_query ? a.query_bias : a.key_bias, at, lane + pairs, y);
            const bool listed = a.rope && position < a.rope_positions;
            const double* angles = a.rope + static_cast<int64_t>(position) * a.rotary + kk;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                double sn, cs;
                if (listed) {
                    sn = angles[j];
                    cs = angles[pairs + j];
                } else {
                    rope_angle(kk + j, position, a.base, a.rotary, sn, cs);
                }
                rope_apply(x[j], y[j], sn, cs, x[j], y[j]);
            }
            if (is_query) {
                store_as(a.query_out + at + lane, x);
                store_as(a.query_out + at + lane + pairs, y);
            } else {
                T* out = keys + (head - s.heads) * head_size + static_cast<int64_t>(run.offset + t) * s.width + kk;
                store_as(out, x);
                store_as(out + pairs, y);
            }
        }
        const int behind = s.width - a.rotary;
        if (behind > 0)
            for (int i = start; i < run.tokens * both * behind; i += stride) {
                const int lane = a.rotary + i % behind, head = i / behind % both, t = i / behind / both;
                const int64_t row = run.row + t;
                if (head < s.heads) {
                    if (lane < D)
                        store_f32(a.query_out + row * s.heads * D + head * D + lane,
                                  biased(a.query + row * s.heads * D, a.query_bias, head * D + lane));
                } else {
                    const int kh = head - s.heads;
                    const float v[1] = {lane < D ? biased(a.key + row * s.kv_heads * D, a.key_bias, kh * D + lane) : 0.0f};
                    store_as(keys + kh * head_size + static_cast<int64_t>(run.offset + t) * s.width + lane, v);
                }
            }
        const int first = run.offset / kGroupTokens, groups = (run.offset + run.tokens - 1) / kGroupTokens - first + 1;
        for (int i = start; i < groups * s.kv_heads * D; i += stride) {
            const int lane = i % (s.kv_heads * D), group = first + i / (s.kv_heads * D);
            const int t0 = group * kGroupTokens - run.offset;  // of the run
            T* out = values + lane / D * head_size + static_cast<int64_t>(lane % D) * s.page_tokens + group * kGroupTokens;
            float v[kGroupTokens];
#pragma unroll
            for (int j = 0; j < kGroupTokens; ++j)
                v[j] = t0 + j >= 0 && t0 + j < run.tokens
                           ? biased(a.value + static_cast<int64_t>(run.row + t0 + j) * s.kv_heads * D, a.value_bias, lane)
                           : 0.0f;
            if (t0 >= 0 && t0 + kGroupTokens <= run.tokens) {
                store_as(out, v);
            } else {
#pragma unroll
                for (int j = 0; j < kGroupTokens; ++j)
                    if (t0 + j >= 0 && t0 + j < run.tokens) *(SATORI_GLOBAL T*)(out + j) = static_cast<T>(v[j]);
            }
        }
    }
}

// ---- attention ----
//
// A workgroup attends the tokens of one item for up to 16 * NB (row, query head) pairs of one key/value head; its four
// waves take tiles of 32 tokens in turn. With S^T = K Q^T and O^T = V^T P^T, both computed by 16 x 16 matrix tiles, a
// column of either product is a pair, so the running maximum and sum of a pair live in the lanes of its column
// (lane % 16), and what the first product leaves in a lane (four tokens of a pair per tile) is what the second takes
// from it: the tokens of the key tiles are numbered so that no value changes lanes (F16: row m of tile a is token
// 8 * (m / 4) + 4 * a + m % 4, which leaves lane group g the tokens 8 g .. 8 g + 7).
//
// F16 keys and values are exact in the matrix instructions; what they meet is not, so queries and probabilities go in as
// two halves of 11 bits, x = hi + lo, both products summed in the same FP32 accumulator: 2^-22 of a value is lost. Their
// scale is a power of two that puts the largest query lane of a pair (and a probability of one) at 2^14, far from
// where halves lose bits. F32 caches use the FP32 matrix instructions.

constexpr int kWaves = 4;
constexpr int kTileTokens = 32;
constexpr float kLog2e = 1.44269504088896340736f;

// Maximum and sum over the four lanes that hold one column (lane, lane ^ 16, lane ^ 32, lane ^ 48).
__device__ __forceinline__ float column_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float column_sum(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

__device__ __forceinline__ f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma32(float a, float b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// Operands of one wave's tile, by element type. Tokens are counted from the tile's first; token(i) is the i-th (of 8)
// that this lane's scores belong to.
template <typename T, int W>
struct Tile;

template <int W>
struct Tile<_Float16, W> {
    static constexpr float kTop = 14.0f;  // log2 of a probability of one, as the second product takes it
    struct Query {
        f16x8 hi[W / 32], lo[W / 32];
        float factor;  // of a score: 1 / sqrt(head_dim), the base of exp2 and the query's own scale
    };
    f16x8 k[2][W / 32], v[W / 16];

    static __device__ __forceinline__ int token(int g, int i) { return 8 * g + i; }

    __device__ __forceinline__ void load_keys(const uint8_t* page, int c, int g) {
        const _Float16* p = reinterpret_cast<const _Float16*>(page) + (8 * (c >> 2) + (c & 3)) * W + 8 * g;
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int s = 0; s < W / 32; ++s) k[a][s] = *(const SATORI_GLOBAL f16x8*)(p + 4 * a * W + 32 * s);
    }
    __device__ __forceinline__ void load_values(const uint8_t* page, int page_tokens, int c, int g) {
        const _Float16* p = reinterpret_cast<const _Float16*>(page) + c * page_tokens + 8 * g;
#pragma unroll
        for (int d = 0; d < W / 16; ++d) v[d] = *(const SATORI_GLOBAL f16x8*)(p + 16 * d * page_tokens);
    }
    // Values of tokens from `end` on become zero (they are nobody's, and may hold anything).
    __device__ __forceinline__ void clip_values(int end, int g) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (8 * g + i >= end)
#pragma unroll
                for (int d = 0; d < W / 16; ++d) v[d][i] = 0;
    }
    __device__ __forceinline__ bool values_finite() const {
        bool finite = true;
#pragma unroll
        for (int d = 0; d < W / 16; ++d)
#pragma unroll
            for (int i = 0; i < 8; ++i) finite &= __builtin_isfinite(static_cast<float>(v[d][i]));
        return finite;
    }
    static __device__ __forceinline__ void load_query(Query& q, const float* row, int head_dim, float scale, int g) {
        float x[W / 32][8];
        float top = 0;
#pragma unroll
        for (int s = 0; s < W / 32; ++s)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int d = 32 * s + 8 * g + j;
                x[s][j] = row && d < head_dim ? load_f32(row + d) : 0.0f;
                top = fmaxf(top, fabsf(x[s][j]));
            }
        top = column_max(top);
        const int exponent = static_cast<int>(__float_as_uint(top) >> 23) - 127;
        const int shift = top > 0 && exponent < 128 ? (14 - exponent < 100 ? 14 - exponent : 100) : 0;
        q.factor = ldexpf(scale, -shift);
#pragma unroll
        for (int s = 0; s < W / 32; ++s)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float y = ldexpf(x[s][j], shift);
                q.hi[s][j] = static_cast<_Float16>(y);
                q.lo[s][j] = static_cast<_Float16>(y - static_cast<float>(q.hi[s][j]));
            }
    }
    __device__ __forceinline__ void scores(const Query& q, f32x4 (&out)[2]) const {
#pragma unroll
        for (int a = 0; a < 2; ++a) out[a] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < W / 32; ++s) {
#pragma unroll
            for (int a = 0; a < 2; ++a) out[a] = mfma16(k[a][s], q.hi[s], out[a]);
#pragma unroll
            for (int a = 0; a < 2; ++a) out[a] = mfma16(k[a][s], q.lo[s], out[a]);
        }
    }
    static __device__ __forceinline__ void halves(const float (&p)[8], f16x8& hi, f16x8& lo) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            hi[i] = static_cast<_Float16>(p[i]);
            lo[i] = static_cast<_Float16>(p[i] - static_cast<float>(hi[i]));
        }
    }
    __device__ __forceinline__ void weigh(const float (&p)[8], f32x4 (&o)[W / 16]) const {
        f16x8 hi, lo;
        halves(p, hi, lo);
#pragma unroll
        for (int d = 0; d < W / 16; ++d) o[d] = mfma16(v[d], hi, o[d]);
#pragma unroll
        for (int d = 0; d < W / 16; ++d) o[d] = mfma16(v[d], lo, o[d]);
    }
    // The same for token t of the tile alone, added where `seen`.
    __device__ __forceinline__ void weigh_one(const float (&p)[8], int t, int g, bool seen, f32x4 (&o)[W / 16]) const {
        f16x8 hi, lo;
        halves(p, hi, lo);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (8 * g + i != t) hi[i] = lo[i] = 0;
#pragma unroll
        for (int d = 0; d < W / 16; ++d) {
            f16x8 one;
#pragma unroll
            for (int i = 0; i < 8; ++i) one[i] = 8 * g + i == t ? v[d][i] : static_cast<_Float16>(0);
            const f32x4 add = mfma16(one, lo, mfma16(one, hi, f32x4{0, 0, 0, 0}));
            if (seen) o[d] = o[d] + add;
        }
    }
};

template <int W>
struct Tile<float, W> {
    static constexpr float kTop = 0.0f;
    struct Query {
        f32x4 x[W / 16];
        float factor;
    };
    f32x4 k[2][W / 16], v[W / 16][2];

    static __device__ __forceinline__ int token(int g, int i) { return 16 * (i >> 2) + 4 * g + (i & 3); }

    __device__ __forceinline__ void load_keys(const uint8_t* page, int c, int g) {
        const float* p = reinterpret_cast<const float*>(page) + c * W + 4 * g;
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int s = 0; s < W / 16; ++s) k[a][s] = *(const SATORI_GLOBAL f32x4*)(p + 16 * a * W + 16 * s);
    }
    __device__ __forceinline__ void load_values(const uint8_t* page, int page_tokens, int c, int g) {
        const float* p = reinterpret_cast<const float*>(page) + c * page_tokens + 4 * g;
#pragma unroll
        for (int d = 0; d < W / 16; ++d)
#pragma unroll
            for (int a = 0; a < 2; ++a) v[d][a] = *(const SATORI_GLOBAL f32x4*)(p + 16 * d * page_tokens + 16 * a);
    }
    __device__ __forceinline__ void clip_values(int end, int g) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (token(g, i) >= end)
#pragma unroll
                for (int d = 0; d < W / 16; ++d) v[d][i >> 2][i & 3] = 0;
    }
    __device__ __forceinline__ bool values_finite() const {
        bool finite = true;
#pragma unroll
        for (int d = 0; d < W / 16; ++d)
#pragma unroll
            for (int i = 0; i < 8; ++i) finite &= __builtin_isfinite(v[d][i >> 2][i & 3]);
        return finite;
    }
    static __device__ __forceinline__ void load_query(Query& q, const float* row, int head_dim, float scale, int g) {
#pragma unroll
        for (int s = 0; s < W / 16; ++s)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int d = 16 * s + 4 * g + j;
                q.x[s][j] = row && d < head_dim ? load_f32(row + d) : 0.0f;
            }
        q.factor = scale;
    }
    __device__ __forceinline__ void scores(const Query& q, f32x4 (&out)[2]) const {
#pragma unroll
        for (int a = 0; a < 2; ++a) out[a] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < W / 16; ++s)
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int a = 0; a < 2; ++a) out[a] = mfma32(k[a][s][j], q.x[s][j], out[a]);
    }
    __device__ __forceinline__ void weigh(const float (&p)[8], f32x4 (&o)[W / 16]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int d = 0; d < W / 16; ++d) o[d] = mfma32(v[d][i >> 2][i & 3], p[i], o[d]);
    }
    __device__ __forceinline__ void weigh_one(const float (&p)[8], int t, int g, bool seen, f32x4 (&o)[W / 16]) const {
#pragma unroll
        for (int d = 0; d < W / 16; ++d) {
            f32x4 add{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const bool mine = token(g, i) == t;
                add = mfma32(mine ? v[d][i >> 2][i & 3] : 0.0f, mine ? p[i] : 0.0f, add);
            }
            if (seen) o[d] = o[d] + add;
        }
    }
};

// Partial results: [slots][heads][width] values, then [slots][heads] (maximum, sum) pairs, in units of exp2.
__device__ __forceinline__ float* partial_values(float* partials, int width, int64_t index) {
    return partials + index * width;
}
__device__ __forceinline__ float* partial_sums(float* partials, int width, int64_t all, int64_t index) {
    return partials + all * width + index * 2;
}

template <typename T, int W, int NB>
__global__ __launch_bounds__(kWaves * 64, NB == 1 && W <= 128 ? 2 : 1) void cache_attention_kernel(CacheShape s, const int* __restrict__ plan,
                                                                      int layer, const float* __restrict__ query,
                                                                      float* __restrict__ output, float* partials,
                                                                      float scale, int wide) {
    constexpr int kPart = W < 128 ? W : 128;  // lanes joined at once
    static_assert(W % 16 == 0 && (W <= 128 || W % 64 == 0), "widths");
    __shared__ float joined[kWaves][16][kPart + 4];
    __shared__ float stats[kWaves][16][2];
    const PlanHeader& h = *reinterpret_cast<const PlanHeader*>(plan);
    const PlanRow* rows = reinterpret_cast<const PlanRow*>(plan + h.rows_at);
    const PlanItem* items = reinterpret_cast<const PlanItem*>(plan + (wide ? h.wide_at : h.narrow_at));
    const int count = wide ? h.wide : h.narrow;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int group = s.heads / s.kv_heads;
    const int64_t head_bytes = static_cast<int64_t>(s.page_tokens) * W * sizeof(T);
    const int64_t partial_rows = static_cast<int64_t>(h.slots) * s.heads;
    for (int u = blockIdx.x; u < count; u += gridDim.x) {
        const PlanItem item = items[u];
        const int* pages = plan + h.pages_at + item.pages;
        const int* list = plan + h.list_at + item.rows;
        const uint8_t* base = s.pool + layer * s.layer_bytes + item.kv * head_bytes;
        const int blocks = (item.pairs + 15) / 16;

        typename Tile<T, W>::Query q[NB];
        f32x4 o[NB][W / 16];
        float m[NB], l[NB];
        int limit[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int p = item.pair + 16 * b + c;
            const float* row = nullptr;
            limit[b] = -1;
            if (16 * b + c < item.pairs) {
                const int r = list[p / group];
                row = query + (static_cast<int64_t>(r) * s.heads + item.kv * group + p % group) * s.head_dim;
                limit[b] = rows[r].position - item.first;
            }
            if (b < blocks) Tile<T, W>::load_query(q[b], row, s.head_dim, scale, g);
            m[b] = -INFINITY;
            l[b] = 0;
#pragma unroll
            for (int d = 0; d < W / 16; ++d) o[b][d] = f32x4{0, 0, 0, 0};
        }

        Tile<T, W> tile;
        const auto page_of = [&](int t) {  // the page and place of token item.first + t
            const int at = (item.first & (s.page_tokens - 1)) + t;
            return base + pages[at >> s.page_shift] * s.page_bytes;
        };
        const auto within = [&](int t) { return (item.first + t) & (s.page_tokens - 1); };
        int t = wave * kTileTokens;
        if (t < item.tokens) tile.load_keys(page_of(t) + static_cast<int64_t>(within(t)) * W * sizeof(T), c, g);
        for (; t < item.tokens; t += kWaves * kTileTokens) {
            tile.load_values(page_of(t) + s.kv_heads * head_bytes + within(t) * sizeof(T), s.page_tokens, c, g);
            f32x4 sc[NB][2];
#pragma unroll
            for (int b = 0; b < NB; ++b)
                if (b < blocks) tile.scores(q[b], sc[b]);
            const int next = t + kWaves * kTileTokens;
            if (next < item.tokens)
                tile.load_keys(page_of(next) + static_cast<int64_t>(within(next)) * W * sizeof(T), c, g);
            const int end = item.tokens - t;  // tokens of this tile that exist
            const bool hides = item.first + t + kTileTokens - 1 > item.limit;
            if (end < kTileTokens) tile.clip_values(end, g);
            // A value that one row sees and another must not can only spoil the other's sums if it is not finite.
            const bool one_by_one = hides && !__all(tile.values_finite());
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if (b >= blocks) continue;
                float x[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = sc[b][i >> 2][i & 3] * q[b].factor;
                if (hides || end < kTileTokens) {
                    const int seen = min(limit[b] - t + 1, end);
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[i] = Tile<T, W>::token(g, i) < seen ? x[i] : -INFINITY;
                }
                float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])),
                                  fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
                top = column_max(top);
                if (__any(top > m[b])) {
                    const float now = fmaxf(m[b], top);
                    const float shrink = __builtin_amdgcn_exp2f(m[b] - (now == -INFINITY ? 0.0f : now));
                    m[b] = now;
                    l[b] *= shrink;
#pragma unroll
                    for (int d = 0; d < W / 16; ++d) o[b][d] = o[b][d] * shrink;
                }
                const float from = Tile<T, W>::kTop - (m[b] == -INFINITY ? 0.0f : m[b]);
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = __builtin_amdgcn_exp2f(x[i] + from);
                l[b] += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
                if (!one_by_one) {
                    tile.weigh(x, o[b]);
                } else {
                    for (int k = 0; k < min(end, kTileTokens); ++k) tile.weigh_one(x, k, g, t + k <= limit[b], o[b]);
                }
            }
        }

        // The four waves' results joined, 16 pairs and up to 128 lanes at a time.
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            if (b >= blocks) continue;
            const float sum = column_sum(l[b]);
            if (g == 0) {
                stats[wave][c][0] = m[b];
                stats[wave][c][1] = sum;
            }
#pragma unroll
            for (int part = 0; part < (W + kPart - 1) / kPart; ++part) {
                constexpr int kTiles = kPart / 16;
#pragma unroll
                for (int d = 0; d < kTiles; ++d) {
                    const int of = part * kTiles + d;
                    if (of < W / 16) *reinterpret_cast<f32x4*>(&joined[wave][c][16 * d + 4 * g]) = o[b][of < W / 16 ? of : 0];
                }
                __syncthreads();
                const int pair = threadIdx.x >> 4;  // 16 threads a pair
                if (16 * b + pair < item.pairs) {
                    float top = -INFINITY, total = 0;
#pragma unroll
                    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, stats[w][pair][0]);
                    float weight[kWaves];
#pragma unroll
                    for (int w = 0; w < kWaves; ++w) {
                        // (a NaN maximum never arises; a NaN score leaves a NaN sum)
                        weight[w] = __builtin_amdgcn_exp2f(stats[w][pair][0] - (top == -INFINITY ? 0.0f : top));
                        total += weight[w] * stats[w][pair][1];
                    }
                    const int p = item.pair + 16 * b + pair;
                    const int r = list[p / group], head = item.kv * group + p % group;
                    const PlanRow row = rows[r];
                    const int64_t index = static_cast<int64_t>(row.slot + item.slot) * s.heads + head;
                    const int left = W - part * kPart < kPart ? W - part * kPart : kPart;
                    for (int d = threadIdx.x & 15; d < left; d += 16) {
                        float v = 0;
#pragma unroll
                        for (int w = 0; w < kWaves; ++w) v += weight[w] * joined[w][pair][d];
                        const int lane_of = part * kPart + d;
                        if (row.slots > 1)
                            partial_values(partials, W, index)[lane_of] = v;
                        else if (lane_of < s.head_dim)
                            output[(static_cast<int64_t>(r) * s.heads + head) * s.head_dim + lane_of] = v / total;
                    }
                    if (row.slots > 1 && part == 0 && (threadIdx.x & 15) == 0) {
                        float* sums = partial_sums(partials, W, partial_rows, index);
                        sums[0] = top;
                        sums[1] = total;
                    }
                }
                __syncthreads();
            }
        }
    }
}

// The partial results of one (row, head), joined by a wave: weight 2^(m_i - m) each.
__global__ __launch_bounds__(kThreads) void cache_join_kernel(CacheShape s, const int* __restrict__ plan,
                                                              float* partials, float* __restrict__ output) {
    const PlanHeader& h = *reinterpret_cast<const PlanHeader*>(plan);
    const PlanRow* rows = reinterpret_cast<const PlanRow*>(plan + h.rows_at);
    const int lane = threadIdx.x & 63;
    const int64_t units = static_cast<int64_t>(h.rows) * s.heads;
    const int64_t partial_rows = static_cast<int64_t>(h.slots) * s.heads;
    for (int64_t u = static_cast<int64_t>(blockIdx.x) * kWaves + (threadIdx.x >> 6); u < units; u += gridDim.x * kWaves) {
        const int r = static_cast<int>(u / s.heads), head = static_cast<int>(u % s.heads);
        const PlanRow row = rows[r];
        if (row.slots <= 1) continue;
        const int64_t first = static_cast<int64_t>(row.slot) * s.heads + head;
        float top = -INFINITY;
        for (int i = 0; i < row.slots; ++i)
            top = fmaxf(top, partial_sums(partials, s.width, partial_rows, first + static_cast<int64_t>(i) * s.heads)[0]);
        const float from = top == -INFINITY ? 0.0f : top;
        float total = 0, v[4] = {0, 0, 0, 0};
        for (int i = 0; i < row.slots; ++i) {
            const int64_t index = first + static_cast<int64_t>(i) * s.heads;
            const float* sums = partial_sums(partials, s.width, partial_rows, index);
            const float weight = __builtin_amdgcn_exp2f(sums[0] - from);
            total += weight * sums[1];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (lane + 64 * j < s.width) v[j] += weight * partial_values(partials, s.width, index)[lane + 64 * j];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (lane + 64 * j < s.head_dim) output[u * s.head_dim + lane + 64 * j] = v[j] / total;
    }
}

// Blocks of 16 pairs of a wide workgroup: what its registers hold beside a tile.
constexpr int wide_blocks(bool, int width) { return width <= 64 ? 4 : width <= 128 ? 2 : 1; }

constexpr int kMostGroups = 2048;  // workgroups of a launch whose work is only known when it is replayed

struct AttentionCall {
    const int* plan;
    PlanHeader now;
    bool all;
    int layer;
    const float* query;
    float *output, *partials;
    hipStream_t stream;
};

template <typename T, int W>
void attention_of_width(const CacheShape& s, const AttentionCall& a) {
    const float scale = static_cast<float>(static_cast<double>(kLog2e) / std::sqrt(static_cast<double>(s.head_dim)));
    if (a.now.wide || a.all)
        cache_attention_kernel<T, W, wide_blocks(sizeof(T) == 4, W)>
            <<<a.all ? kMostGroups : a.now.wide, kWaves * 64, 0, a.stream>>>(s, a.plan, a.layer, a.query, a.output,
                                                                             a.partials, scale, 1);
    if (a.now.narrow || a.all)
        cache_attention_kernel<T, W, 1><<<a.all ? kMostGroups : a.now.narrow, kWaves * 64, 0, a.stream>>>(
            s, a.plan, a.layer, a.query, a.output, a.partials, scale, 0);
}

template <typename T>
hipError_t attention_of_type(const CacheShape& s, const AttentionCall& a) {
    switch (s.width) {
        case 32: attention_of_width<T, 32>(s, a); break;
        case 64: attention_of_width<T, 64>(s, a); break;
        case 96: attention_of_width<T, 96>(s, a); break;
        case 128: attention_of_width<T, 128>(s, a); break;
        case 192: attention_of_width<T, 192>(s, a); break;
        case 256: attention_of_width<T, 256>(s, a); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace

int cache_wide_pairs(int type, int width) { return 16 * wide_blocks(type == kF32, width); }

hipError_t launch_copy_pages(uint8_t* pool, int64_t page_bytes, const PageMoves& moves, hipStream_t stream) {
    if (moves.count == 0) return hipSuccess;
    const dim3 grid(static_cast<unsigned>((page_bytes + kCopyBytes - 1) / kCopyBytes), moves.count);
    copy_pages_kernel<<<grid, kThreads, 0, stream>>>(pool, page_bytes, moves);
    return hipGetLastError();
}

hipError_t launch_cache_append(const CacheShape& s, const int* plan, const PlanHeader& now, bool all,
                               const AppendArgs& args, hipStream_t stream) {
    if (now.runs == 0 && !all) return hipSuccess;
    // Four lane pairs a thread and access where every row allows it.
    const auto whole = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    const bool packed = args.rotary % 8 == 0 && s.head_dim % 4 == 0 && whole(args.query) && whole(args.query_bias) &&
                        whole(args.query_out) && whole(args.key) && whole(args.key_bias);
    // One turn a thread for the longest run's rotations, and what a run of a few positions needs for its values.
    const int longest = all ? 8 : now.longest_run;
    const int64_t turns = static_cast<int64_t>(longest) * (s.heads + s.kv_heads) * (args.rotary / (packed ? 8 : 2));
    const int64_t values = (static_cast<int64_t>(longest) / kGroupTokens + 1) * s.kv_heads * s.head_dim;
    const int y = static_cast<int>(std::min<int64_t>((std::max(turns, values) + kThreads - 1) / kThreads, 1024));
    const dim3 grid(all ? 256 : now.runs, y);
    const auto launch = [&](auto kernel) { kernel<<<grid, kThreads, 0, stream>>>(s, plan, args); };
    if (s.type == kF32)
        packed ? launch(cache_append_kernel<float, 4>) : launch(cache_append_kernel<float, 1>);
    else
        packed ? launch(cache_append_kernel<_Float16, 4>) : launch(cache_append_kernel<_Float16, 1>);
    return hipGetLastError();
}

size_t cache_partial_bytes(const CacheShape& shape, int64_t slots) {
    return static_cast<size_t>(slots) * shape.heads * (shape.width + 2) * sizeof(float);
}

hipError_t launch_cache_attention(const CacheShape& shape, const int* plan, const PlanHeader& now, bool all, int layer,
                                  const float* query, float* output, float* partials, hipStream_t stream) {
    if (now.rows == 0 && !all) return hipSuccess;
    const AttentionCall call{plan, now, all, layer, query, output, partials, stream};
    const hipError_t e = shape.type == kF32 ? attention_of_type<float>(shape, call)
                                            : attention_of_type<_Float16>(shape, call);
    if (e != hipSuccess || (now.joined == 0 && !all)) return e;
    const int64_t groups = (static_cast<int64_t>(now.rows) * shape.heads + kWaves - 1) / kWaves;
    cache_join_kernel<<<all ? kMostGroups : static_cast<int>(std::min<int64_t>(groups, 65536)), kThreads, 0, stream>>>(
        shape, plan, partials, output);
    return hipGetLastError();
}

}  // namespace satori
