// Kernels of the paged key/value cache: page copies, the write of new positions and the attention of a batch whose
// sequences share pages.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "cache_ops.hpp"
#include "device_common.hpp"
#include "rope_device.hpp"
#include "rotation_device.hpp"

namespace satori {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;

// The same value, of which the compiler knows nothing.
__device__ __forceinline__ int unknown_scalar(int v) {
    __asm__ volatile("" : "+s"(v));
    return v;
}

// ---- page copies ----

// Each workgroup copies kCopyBytes of one page, 16 bytes a thread and access, four accesses in flight; a page of all layers is
// one run of bytes, so one launch serves any number of moves. Bound by memory: 224 moves of 917,504 bytes take 73 us (5.6
// TB/s read and written, the large copy's 4.9 being one of 2 GiB), 48 whose source is one page 10.9 us (the 44 MB written at
// 4.0 TB/s, launch included).
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

// ---- a plan's copy ----

constexpr int kPlanParts = 8;
struct PlanParts {
    int at[kPlanParts], end[kPlanParts];  // 16-byte units; end: of the parts up to this one, counted through
};

__global__ __launch_bounds__(kThreads) void plan_copy_kernel(const u32x4* from, u32x4* to, PlanParts parts) {
    int n = blockIdx.x * kThreads + threadIdx.x, part = 0;
    if (n >= parts.end[kPlanParts - 1]) return;
    while (n >= parts.end[part]) ++part;
    n += parts.at[part] - (part ? parts.end[part - 1] : 0);
    to[n] = from[n];
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
// them together where they fill an aligned group (one value a store took 93 us where this takes 9.8). Few rows are bound by
// the launch and two dependent reads (16 rows of 12 + 2 heads of 128 lanes 4.6 us), many by that and, half of the time, by memory: 8 x
// 61 rows of 32 + 8 heads move 22.6 MB in 9.8 us (2.3 TB/s, where a large copy reaches 4.9); in a captured step, whose grid does
// for any batch, 15.1. The rotation's angles come from the table in 64 bits, as the single-sequence operator's; where the host knows
// that the table has them all, the launch leaves out the code that computes them, and a wave takes 60 registers instead of 127:
// with that and the lanes behind the rotated ones in fours, 16 x 61 rows of a tree, 64 of 128 lanes rotated, 12.0 us instead of
// 21.4 (44 MB, a floor of 8.5).
enum class Turn { kPlain, kTree, kInterleaved };  // pairs half a head apart, rows no tree's; also a tree's; neighbouring lanes
template <typename T, int N, Turn TURN, bool LISTED>  // LISTED: the table has every position
__global__ __launch_bounds__(kThreads) void cache_append_kernel(CacheShape s, const int* __restrict__ image, int runs_at, int trees_at,
                                                                AppendArgs a) {
    constexpr bool kInterleaved = TURN == Turn::kInterleaved;
    const int count = reinterpret_cast<const PlanHeader*>(image)->runs;
    const int tree_stride = TURN == Turn::kPlain ? 0 : reinterpret_cast<const PlanHeader*>(image)->tree_stride;
    const PlanRun* runs = reinterpret_cast<const PlanRun*>(image + runs_at);
    const int pairs = a.rotary / 2, D = s.head_dim, both = s.heads + s.kv_heads;
    const int64_t head_size = static_cast<int64_t>(s.page_tokens) * s.width;
    for (int u = blockIdx.x; u < count; u += gridDim.x) {
        const PlanRun run = runs[u];
        const int position0 = run.position;
        T* keys = reinterpret_cast<T*>(s.pool + run.page * s.page_bytes + a.layer * s.layer_bytes);
        T* values = keys + s.kv_heads * head_size;
        const int start = blockIdx.y * kThreads + threadIdx.x, stride = gridDim.y * kThreads;
        const int packs = pairs / N;
        for (int i = start; i < run.tokens * both * packs; i += stride) {
            const int kk = i % packs * N, rest = i / packs, head = rest % both, t = rest / both;
            const int position = tree_stride ? image[trees_at + (run.row + t) * tree_stride] : position0 + t;
            const bool is_query = head < s.heads;
            const int first = (is_query ? head : head - s.heads) * D;
            const int lane = first + (kInterleaved ? 2 * kk : kk), beside = kInterleaved ? N : pairs;
            const int64_t at = static_cast<int64_t>(run.row + t) * (is_query ? s.heads : s.kv_heads) * D;
            float x[N], y[N];
            load_biased(is_query ? a.query : a.key, is_query ? a.query_bias : a.key_bias, at, lane, x);
            load_biased(is_query ? a.query : a.key, is_query ? a.query_bias : a.key_bias, at, lane + beside, y);
            const bool listed = LISTED || (a.rope && position < a.rope_positions);
            const double* angles = a.rope + static_cast<int64_t>(position) * a.rotary + kk;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                double sn, cs;
                if (LISTED || listed) {
                    sn = angles[j];
                    cs = angles[pairs + j];
                } else if (a.frequencies) {
                    rotation_angle(kk + j, position, a.frequencies, a.magnitude, sn, cs);
                } else {
                    rope_angle(kk + j, position, a.base, a.rotary, sn, cs);
                }
                rotate_pair<kInterleaved>(x, y, j, sn, cs);
            }
            if (is_query) {
                store_as(a.query_out + at + lane, x);
                store_as(a.query_out + at + lane + beside, y);
            } else {
                T* out = keys + (head - s.heads) * head_size + static_cast<int64_t>(run.offset + t) * s.width + lane - first;
                store_as(out, x);
                store_as(out + beside, y);
            }
        }
        // N lanes at once, as the rotated ones: a whole number of those, of heads and of what lies behind.
        const int behind = (s.width - a.rotary) / N;
        if (behind > 0)
            for (int i = start; i < run.tokens * both * behind; i += stride) {
                const int lane = a.rotary + i % behind * N, head = i / behind % both, t = i / behind / both;
                const int64_t row = run.row + t;
                float v[N] = {};
                if (head < s.heads) {
                    if (lane >= D) continue;
                    load_biased(a.query, a.query_bias, row * s.heads * D, head * D + lane, v);
                    store_as(a.query_out + row * s.heads * D + head * D + lane, v);
                } else {
                    const int kh = head - s.heads;
                    if (lane < D) load_biased(a.key, a.key_bias, row * s.kv_heads * D, kh * D + lane, v);
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

// ---- positions that a sequence keeps ----

// Moves the keys and values of a sequence's kept rows to the places behind its context, in all layers. A place that is
// written may be read by an earlier move and by no later one (rows go in ascending order, none behind where it was), so eight
// moves are read before they are written, and the next eight come behind them in the same wave. Of keys a thread takes 16 bytes
// through all moves. Of values, whose positions lie side by side, eight threads take a move each of one lane of the head, so
// that the destinations, which follow one another, are one access; a wave takes 32 lanes of a head. Few moves are bound by
// the launch (one sequence, 4 layers 3.1 us), many by the lines that hold the values, of which a move wants 2 bytes each: 245
// moves of 64 sequences, 28 layers of 2 heads of 128 lanes, F16, 14 MB, in 20 us. (A thread through all moves of a lane asks for
// 1.8 million writes instead of 0.5 and takes 25; a wave for all lanes of a head 31, the same with whole 64 bytes written through
// LDS 23.)
template <typename T>
__global__ __launch_bounds__(kThreads) void cache_keep_kernel(CacheShape s, int layers, KeepMoves moves) {
    typedef std::conditional_t<sizeof(T) == 2, uint16_t, uint32_t> Bits;
    constexpr int kSize = sizeof(T), kMoves = 8, kSteps = 4, kBlock = 64 / kMoves * kSteps;  // lanes of a head a wave takes
    const int begin = moves.begin[blockIdx.y], end = moves.begin[blockIdx.y + 1], lane = threadIdx.x & 63;
    const int wave = blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int pieces = s.width * kSize / 16, heads = layers * s.kv_heads, mask = s.page_tokens - 1;
    const int key_waves = (heads * pieces + 63) / 64, blocks = (s.head_dim + kBlock - 1) / kBlock;
    const int64_t head_bytes = static_cast<int64_t>(s.page_tokens) * s.width * kSize;
    if (wave < key_waves) {
        const int u = wave * 64 + lane;
        if (u >= heads * pieces) return;
        const int head = u / pieces;
        uint8_t* base = s.pool + head / s.kv_heads * s.layer_bytes + head % s.kv_heads * head_bytes + u % pieces * 16;
        const auto at = [&](int place) { return base + (place >> s.page_shift) * s.page_bytes + (place & mask) * (s.width * kSize); };
        for (int i0 = begin; i0 < end; i0 += kMoves) {
            u32x4 v[kMoves];
#pragma unroll
            for (int j = 0; j < kMoves; ++j) v[j] = *(const SATORI_GLOBAL u32x4*)(at(moves.source[min(i0 + j, end - 1)]));
#pragma unroll
            for (int j = 0; j < kMoves; ++j)
                if (i0 + j < end) *(SATORI_GLOBAL u32x4*)(at(moves.destination[i0 + j])) = v[j];
        }
        return;
    }
    const int head = (wave - key_waves) / blocks, first = (wave - key_waves) % blocks * kBlock;
    if (head >= heads) return;
    const int move = lane % kMoves, row = first + lane / kMoves, row_bytes = s.page_tokens * kSize;
    uint8_t* base = s.pool + head / s.kv_heads * s.layer_bytes + (s.kv_heads + head % s.kv_heads) * head_bytes +
                    static_cast<int64_t>(row) * row_bytes;
    for (int i0 = begin; i0 < end; i0 += kMoves) {
        // Each move's places are scalars, all read before any is chosen; those behind the last are the last, and not written.
        int of[kMoves], to[kMoves];
#pragma unroll
        for (int j = 0; j < kMoves; ++j) {
            of[j] = moves.source[min(i0 + j, end - 1)];
            to[j] = moves.destination[min(i0 + j, end - 1)];
        }
        int source = 0, destination = 0;
#pragma unroll
        for (int j = 0; j < kMoves; ++j) {
            const int x = unknown_scalar(of[j]), y = unknown_scalar(to[j]);
            source = move == j ? x : source;
            destination = move == j ? y : destination;
        }
        const auto at = [&](int place) { return base + (place >> s.page_shift) * s.page_bytes + (place & mask) * kSize; };
        const uint8_t* from = at(source);
        uint8_t* target = at(destination);
        const int left = (s.head_dim - row + kMoves - 1) / kMoves;  // steps that have a lane
        uint32_t v[kSteps];
#pragma unroll
        for (int j = 0; j < kSteps; ++j)
            v[j] = *(const SATORI_GLOBAL Bits*)(from + (j < left ? j : 0) * kMoves * row_bytes);
#pragma unroll
        for (int j = 0; j < kSteps; ++j)
            if (j < left && i0 + move < end) *(SATORI_GLOBAL Bits*)(target + j * kMoves * row_bytes) = static_cast<Bits>(v[j]);
    }
}

// ---- attention ----
//
// With S^T = K Q^T and O^T = V^T P^T, both computed by 16 x 16 matrix tiles, a column of either product is a (row, query
// head) pair, so the running maximum and sum of a pair live in the lanes of its column (lane % 16), and what the first
// product leaves in a lane (four tokens of a pair per tile) is what the second takes from it: the tokens of the key tiles
// are numbered so that no value changes lanes (F16: row m of tile a is token 8 * (m / 4) + 4 * a + m % 4, which leaves lane
// group g the tokens 8 g .. 8 g + 7; F32: row m of tile a is token 16 * a + m).
//
// F16 keys and values are exact in the matrix instructions; what they meet is not, so queries and probabilities go in as
// two halves of 11 bits, x = hi + lo, both products summed in the same FP32 accumulator. A power of two puts the largest
// query lane of a pair at 2^14 and its largest probability at 2^11 or more (2^15 at most), so that what is lost of either is
// 2^-22 of the value, or 2^-39 of the largest lane and 2^-36 of the largest probability where that is more (half a step of
// the smallest half). FP32 would keep 2^-24 of each; the difference shows where a row's output comes from weights far below its
// largest, whose value is near zero: with one token of value 0 and 1.5% of the weight on 16000 others about 5e-6 of the output, with
// 0.1% on them 1e-4, where rounding keys and values to F16 costs up to 2^-11 of each. Low halves times 2^12 with sums of their own, added
// to the others by the vector unit, would keep 2^-48 and cost 64 rows of one position over 16384 shared ones 73 us instead of 67,
// of 256 lanes 208 instead of 154. F32 caches use the FP32 matrix instructions and lose neither.

constexpr int kTileShift = 5, kTile = 1 << kTileShift;  // tokens that a wave attends at once
constexpr float kSlack = 4.0f;
constexpr float kLog2e = 1.44269504088896340736f;

// The larger one, NaN where either is: one instruction for three numbers, where fmaxf first quiets each of them.
__device__ __forceinline__ float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// Maximum and sum over the four lanes that hold one column (lane, lane ^ 16, lane ^ 32, lane ^ 48).
__device__ __forceinline__ float column_max(float v) {
    auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = larger(__uint_as_float(p[0]), __uint_as_float(p[1]));
    p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return larger(__uint_as_float(p[0]), __uint_as_float(p[1]));
}
__device__ __forceinline__ float column_sum(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

// N lanes of a query from d on, zero from head_dim on and where `is` does not hold. `row` is a row's address in any case.
template <int N>
__device__ __forceinline__ void load_lanes(const float* row, int d, int head_dim, bool quads, bool is, float (&x)[N]) {
#pragma unroll
    for (int j = 0; j < N; j += 4) {
        if (quads) {  // (heads of whole 16-byte pieces)
            const f32x4 v = *(const SATORI_GLOBAL f32x4*)(row + min(d + j, head_dim - 4));
#pragma unroll
            for (int k = 0; k < 4; ++k) x[j + k] = is && d + j < head_dim ? v[k] : 0.0f;
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float v = load_f32(row + min(d + j + k, head_dim - 1));
                x[j + k] = is && d + j + k < head_dim ? v : 0.0f;
            }
        }
    }
}

__device__ __forceinline__ float unknown_minus_one() {
    float v = -1.0f;
    __asm__("" : "+s"(v));
    return v;
}

// The arithmetic of an element type: W lanes a head. Lane (c, g) = (lane % 16, lane / 16).
template <typename T, int W>
struct Math;

template <int W>
struct Math<_Float16, W> {
    static constexpr float kTop = 11.0f;        // log2 of a probability of one, as the second product takes it
    static constexpr int kKeyParts = W / 32;    // fragments of a key tile's 16 rows, of a value tile's 16 lanes
    static constexpr int kValueParts = 1;
    typedef f16x8 Fragment;                     // 16 bytes: lanes 32 s + 8 g .. of a key, tokens 8 g .. of a value lane
    struct Query {
        f16x8 hi[W / 32], lo[W / 32];
        float factor;  // of a score: 1 / sqrt(head_dim), the base of exp2 and the query's own scale
    };
    struct Weights {
        f16x8 hi, lo;
    };

    static __device__ __forceinline__ int token(int g, int i) { return 8 * g + i; }     // of score i (of 8)
    static __device__ __forceinline__ int key_token(int a, int m) { return 8 * (m >> 2) + 4 * a + (m & 3); }
    static __device__ __forceinline__ int key_row(int t) { return 16 * ((t >> 2) & 1) + 4 * (t >> 3) + (t & 3); }
    static __device__ __forceinline__ void load_query(Query& q, const float* row, bool is, int head_dim, bool quads,
                                                      float scale, int g) {
        float x[W / 32][8];
        float top = 0;
#pragma unroll
        for (int s = 0; s < W / 32; ++s) load_lanes(row, 32 * s + 8 * g, head_dim, quads, is, x[s]);
#pragma unroll
        for (int s = 0; s < W / 32; ++s)
#pragma unroll
            for (int j = 0; j < 8; ++j) top = larger(top, fabsf(x[s][j]));
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
    static constexpr int kTerms = 2;  // products of a fragment: with the high halves, with the low ones
    static __device__ __forceinline__ f32x4 score(Fragment k, const Query& q, int s, int term, f32x4 sum) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(k, term ? q.lo[s] : q.hi[s], sum, 0, 0, 0);
    }
    static __device__ __forceinline__ void weights(const float (&p)[8], Weights& w) {
        // High halves in pairs, as the conversion takes them; a low one is a single mixed multiply-add, (-1) hi + p rounded to
        // a half (with a factor that the compiler knows it becomes three instructions).
        const float minus = unknown_minus_one();
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const f16x2 hi = __builtin_convertvector((f32x2{p[i], p[i + 1]}), f16x2);
            w.hi[i] = hi[0], w.hi[i + 1] = hi[1];
            w.lo[i] = static_cast<_Float16>(__builtin_fmaf(static_cast<float>(hi[0]), minus, p[i]));
            w.lo[i + 1] = static_cast<_Float16>(__builtin_fmaf(static_cast<float>(hi[1]), minus, p[i + 1]));
        }
    }
    static __device__ __forceinline__ f32x4 weigh(Fragment v, const Weights& w, int, int term, f32x4 sum) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(v, term ? w.lo : w.hi, sum, 0, 0, 0);
    }
};

template <int W>
struct Math<float, W> {
    static constexpr float kTop = 0.0f;
    static constexpr int kKeyParts = W / 16;
    static constexpr int kValueParts = 2;
    typedef f32x4 Fragment;  // lanes 16 s + 4 g .. of a key, tokens 16 a + 4 g .. of a value lane
    struct Query {
        f32x4 x[W / 16];
        float factor;
    };
    struct Weights {
        float p[8];
    };

    static __device__ __forceinline__ int token(int g, int i) { return 16 * (i >> 2) + 4 * g + (i & 3); }
    static __device__ __forceinline__ int key_token(int a, int m) { return 16 * a + m; }
    static __device__ __forceinline__ int key_row(int t) { return t; }
    static __device__ __forceinline__ void load_query(Query& q, const float* row, bool is, int head_dim, bool quads,
                                                      float scale, int g) {
        float x[W / 16][4];
#pragma unroll
        for (int s = 0; s < W / 16; ++s) load_lanes(row, 16 * s + 4 * g, head_dim, quads, is, x[s]);
#pragma unroll
        for (int s = 0; s < W / 16; ++s) q.x[s] = f32x4{x[s][0], x[s][1], x[s][2], x[s][3]};
        q.factor = scale;
    }
    static constexpr int kTerms = 4;  // products of a fragment: one per element
    static __device__ __forceinline__ f32x4 score(Fragment k, const Query& q, int s, int term, f32x4 sum) {
        return __builtin_amdgcn_mfma_f32_16x16x4f32(k[term], q.x[s][term], sum, 0, 0, 0);
    }
    static __device__ __forceinline__ void weights(const float (&p)[8], Weights& w) {
#pragma unroll
        for (int i = 0; i < 8; ++i) w.p[i] = p[i];
    }
    static __device__ __forceinline__ f32x4 weigh(Fragment v, const Weights& w, int part, int term, f32x4 sum) {
        return __builtin_amdgcn_mfma_f32_16x16x4f32(v[term], w.p[4 * part + term], sum, 0, 0, 0);
    }
};

// The state of 16 pairs: maximum (in units of exp2), the lane's part of the sum, and O^T: lane (c, g) holds lanes
// 16 d + 4 g .. 16 d + 4 g + 3 of pair c.
template <int W>
struct Softmax {
    float m, l;
    f32x4 o[W / 16];

    __device__ __forceinline__ void clear() {
        m = -INFINITY;
        l = 0;
#pragma unroll
        for (int d = 0; d < W / 16; ++d) o[d] = f32x4{0, 0, 0, 0};
    }
    // Takes a tile's scores (as they leave the first product) and gives their weights.
    __device__ __forceinline__ void take(const f32x4 (&score)[2], float factor, float top_weight, float (&p)[8]) {
        float top = larger(larger(score[0][0], score[0][1]), score[0][2]);
        top = larger(larger(top, score[0][3]), score[1][0]);
        top = larger(larger(larger(top, score[1][1]), score[1][2]), score[1][3]) * factor;
        // The maximum may fall behind by a factor of 2^kSlack before everything is scaled again (in the first tiles of random
        // scores some pair of a wave has a new maximum almost every time; 2^8 gives no more than 2^4, and leaves small
        // probabilities fewer bits).
        if (__any(top > m + kSlack)) {
            top = column_max(top);
            const float now = fmaxf(m, top);
            const float shrink = __builtin_amdgcn_exp2f(m - (now == -INFINITY ? 0.0f : now));
            m = now;
            l *= shrink;
#pragma unroll
            for (int d = 0; d < W / 16; ++d) o[d] = o[d] * shrink;
        }
        const float from = top_weight - (m == -INFINITY ? 0.0f : m);
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = __builtin_amdgcn_exp2f(__fmaf_rn(score[i >> 2][i & 3], factor, from));
        l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
    }
};

// The scores of the tokens that a pair does not see become -infinity: those from `seen` on, of the tile.
template <typename M>
__device__ __forceinline__ void hide(f32x4 (&score)[2], int seen, int g) {
    const int left = seen - M::token(g, 0);  // (a lane's tokens are its first one's plus numbers that all lanes share)
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (M::token(0, i) >= left) score[i >> 2][i & 3] = -INFINITY;
}

// The same where a bit of `sees` says of each of the tile's tokens whether the pair sees it.
template <typename M>
__device__ __forceinline__ void hide(f32x4 (&score)[2], uint32_t sees, int g) {
    const uint32_t mine = sees >> M::token(g, 0);
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (!(mine >> M::token(0, i) & 1)) score[i >> 2][i & 3] = -INFINITY;
}

// Of a token's number and what a pair sees of the tile, in either form: whether it sees the token.
__device__ __forceinline__ bool is_seen(int token, int seen) { return token < seen; }
__device__ __forceinline__ bool is_seen(int token, uint32_t sees) { return sees >> token & 1; }

// Values that are not finite. Where some pairs see a token and others must not, the second product would spoil the others'
// sums (0 * infinity), so such a tile's values get zeros in those places, and the sum of each (pair, lane) that sees one
// becomes NaN: here, with values in registers, a product tells which.
template <typename F>
__device__ __forceinline__ bool all_finite(F v) {
    bool all = true;
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(F) / sizeof(v[0])); ++i) all &= __builtin_isfinite(static_cast<float>(v[i]));
    return all;
}
template <typename F>
__device__ __forceinline__ F take_spoiled(F& v) {
    F spoiled;
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(F) / sizeof(v[0])); ++i) {
        const bool fine = __builtin_isfinite(static_cast<float>(v[i]));
        spoiled[i] = fine ? 0 : 1;
        v[i] = fine ? v[i] : 0;
    }
    return spoiled;
}
template <typename M, typename Seen>
__device__ __forceinline__ void spoil(typename M::Fragment spoiled, Seen seen, int part, int g, f32x4& o) {
    float one[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) one[i] = is_seen(M::token(g, i), seen) ? 1.0f : 0.0f;
    typename M::Weights w;
    M::weights(one, w);
    f32x4 hit{0, 0, 0, 0};
#pragma unroll
    for (int term = 0; term < M::kTerms; ++term) hit = M::weigh(spoiled, w, part, term, hit);
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = hit[j] > 0 ? NAN : o[j];
}

// Partial results: [slots][heads][width] values, then [slots][heads] (maximum, sum) pairs, in units of exp2; `all`: slots
// times heads that there is room for.
struct Partials {
    float* at;
    int64_t all;
    __device__ __forceinline__ float* values(int width, int64_t index) const { return at + index * width; }
    __device__ __forceinline__ float* sums(int width, int64_t index) const { return at + all * width + index * 2; }
};

struct AttentionArgs {
    CacheShape s;
    const int* image;
    PlanLayout at;
    int wide, narrow, rows;  // of the plan; -1: as its header says when the launch runs (a captured one)
    int layer;
    const float* query;
    float* output;
    Partials partials;
    float scale;
    bool quads;  // heads of a query start at multiples of 16 bytes and are whole 16-byte pieces
    int tree_stride;  // of the plan, as `wide` is
};

// A (row, query head) pair of an item, by its number; those past the item's last are the first, and not `is`.
struct Pair {
    PlanRow row;
    int head;
    bool is;
};

__device__ __forceinline__ int pair_place(const PlanItem& item, int p) { return item.pair + (p < item.pairs ? p : 0); }

template <bool TREES>
__device__ __forceinline__ Pair pair_of(const AttentionArgs& a, const PlanItem& item, int p) {
    const int group = a.s.heads / a.s.kv_heads, of = pair_place(item, p);
    Pair r;
    if (item.row_slots > 0) {
        const int behind = of / group - item.pair / group;
        r.row = PlanRow{item.limit + behind, item.row_slot + behind * item.row_slots, item.row_slots, item.row + behind};
    } else if (TREES && item.row_slots < 0) {
        const int behind = of / group - item.pair / group;
        r.row = PlanRow{-2 - item.limit, item.row_slot - behind * item.row_slots, -item.row_slots, item.row + behind};
    } else {
        r.row = reinterpret_cast<const PlanRow*>(a.image + a.at.list_at)[item.rows + of / group];
    }
    r.head = item.kv * group + of % group;
    r.is = p < item.pairs;
    return r;
}

__device__ __forceinline__ const float* query_of(const AttentionArgs& a, const Pair& p) {
    return a.query + (static_cast<int64_t>(p.row.row) * a.s.heads + p.head) * a.s.head_dim;
}

// What a pair sees of an item's tiles that its rows do not all see whole: the tokens before its row's position and that one.
template <bool TREES>
struct Sight {
    typedef int Seen;  // the first so many
    int limit;
    __device__ __forceinline__ Sight() = default;
    __device__ __forceinline__ Sight(const AttentionArgs&, const PlanItem& item, const Pair& p, int)
        : limit(p.is ? p.row.position - item.first : -1) {}
    __device__ __forceinline__ Seen of(const AttentionArgs&, const PlanItem&, int t, int end, int) const {
        return min(limit - t + 1, end);
    }
    static __device__ __forceinline__ uint32_t bits(Seen seen) {
        return seen <= 0 ? 0u : ~0u >> (kTile - min(seen, kTile));
    }
};

// The same where rows may be a tree's: a bit per token of the tile, which the plan has ready (a row sees what lies before
// its context's last multiple of 32, and nothing behind its own number's tile). One number a pair and tile, read a tile ahead
// (few pairs) or before the first product (many); tiles that all rows see whole, all but the last few, read none, and kernels
// of plans that never held a tree know of none.
template <>
struct Sight<true> {
    typedef uint32_t Seen;
    int limit;  // relative to the item; of a tree's row its context's last position
    int words;  // of the row, -1 for others
    __device__ __forceinline__ Sight() = default;
    __device__ __forceinline__ Sight(const AttentionArgs& a, const PlanItem& item, const Pair& p, int stride) {
        const bool tree = p.is && p.row.position < 0;
        limit = !p.is ? -1 : (tree ? -2 - p.row.position : p.row.position) - item.first;
        words = tree ? a.at.trees_at + p.row.row * stride + 1 : -1;
    }
    __device__ __forceinline__ Seen of(const AttentionArgs& a, const PlanItem& item, int t, int end, int stride) const {
        const int seen = min(words < 0 ? limit - t + 1 : kTile, end);
        uint32_t sees = seen <= 0 ? 0u : ~0u >> (kTile - min(seen, kTile));
        if (words < 0) return sees;
        const int k = ((item.first + t) >> kTileShift) - ((item.first + limit + 1) >> kTileShift);
        if (k >= 0) sees &= k < stride - 1 ? static_cast<uint32_t>(a.image[words + k]) : 0u;
        return sees;
    }
    static __device__ __forceinline__ uint32_t bits(Seen sees) { return sees; }
};

// One joined result of a pair, four lanes from `d` on: the output where it is the row's only one.
template <int W>
__device__ __forceinline__ void give(const AttentionArgs& a, const PlanItem& item, const Pair& p, int d, f32x4 o,
                                     float total) {
    if (p.row.slots > 1) {
        const int64_t index = static_cast<int64_t>(p.row.slot + item.slot) * a.s.heads + p.head;
        *(SATORI_GLOBAL f32x4*)(a.partials.values(W, index) + d) = o;
        return;
    }
    float* out = a.output + (static_cast<int64_t>(p.row.row) * a.s.heads + p.head) * a.s.head_dim + d;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (d + j < a.s.head_dim) store_f32(out + j, o[j] / total);
}
template <int W>
__device__ __forceinline__ void give_sums(const AttentionArgs& a, const PlanItem& item, const Pair& p, float m, float l) {
    if (p.row.slots <= 1) return;
    float* sums = a.partials.sums(W, static_cast<int64_t>(p.row.slot + item.slot) * a.s.heads + p.head);
    store_f32(sums, m);
    store_f32(sums + 1, l);
}

// Reads of what no kernel writes, at addresses that a wave has in common: through the scalar cache.
template <typename T>
__device__ __forceinline__ T scalar_load(const T* p) {
    const auto* words = (const __attribute__((address_space(4))) int*)(p);
    int w[sizeof(T) / 4];
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 4); ++i) w[i] = words[i];
    T out;
    __builtin_memcpy(&out, w, sizeof(T));
    return out;
}

// The same value, of which the compiler knows nothing: what is computed from it inside a loop stays there (hundreds of
// lane masks and addresses, moved out of the loop over items, would fill the registers).
__device__ __forceinline__ int unknown(int v) {
    __asm__ volatile("" : "+v"(v));
    return v;
}

// The pages of an item's tokens for one layer and key/value head.
struct Pages {
    const uint8_t* base;
    const int* list;
    int64_t page_bytes, head_bytes;
    int first, tokens, shift, kv_heads;
    __device__ __forceinline__ Pages(const AttentionArgs& a, const PlanItem& item, int64_t head) {
        head_bytes = head;
        base = a.s.pool + a.layer * a.s.layer_bytes + item.kv * head_bytes;
        list = a.image + a.at.pages_at + item.pages;
        page_bytes = a.s.page_bytes;
        tokens = a.s.page_tokens;
        first = item.first & (tokens - 1);
        shift = a.s.page_shift;
        kv_heads = a.s.kv_heads;
    }
    // Page number of the item's token t, and the bytes of the keys and values from a token within it.
    __device__ __forceinline__ int page(int t) const { return scalar_load(list + ((first + t) >> shift)); }
    __device__ __forceinline__ int within(int t) const { return (first + t) & (tokens - 1); }
    __device__ __forceinline__ const uint8_t* keys(int page) const { return base + page * page_bytes; }
    __device__ __forceinline__ const uint8_t* values(int page) const { return keys(page) + kv_heads * head_bytes; }
};

// A workgroup of four waves attends one item, in one of two ways.
//
// Few pairs (16 at most): each wave takes tiles of its own in turn, keys and values straight from the cache into registers
// (nobody else in the workgroup wants them), and the waves' results are joined through LDS. Bound by the chain of reads of one
// item (the item 0.8 us, keys and queries 1.3 to 3.4, of FP32 the 64 + 64 matrix instructions of a tile 1.9, the join 1.3): 4
// sequences of 20 to 120 positions 10.4 us in all, 9 x 5 rows over 1500 shared positions 12.7 with their join.
//
// Many pairs: each wave has 16 * kBlocks of them, and the tiles that all four want pass through LDS, in two buffers: while
// one is attended, the bytes of the next three are on their way, the nearest two in registers. Rows of a tile are 16-byte
// pieces, put where the 16 lanes that read a column of them reach different banks: piece p of row r lies at p ^ (r's bits that
// its place in a 256-byte line leaves open). A tile of 128 F16 lanes takes a wave 1.4 us: its 64 matrix instructions are 0.48
// of them, the softmax's and the tile's carrying's other instructions most of the rest, and a wave is alone on its SIMD (two
// workgroups a CU do a tile each in 1.8, but their twice as many partial results take the join that time). 64 sequences of 32
// heads over 16384 shared positions and 64 to 600 of their own: 65.6 us in all, 17.4 GFLOP of the definition and twice that in
// matrix instructions at 0.53 PFLOP/s, 133 MB read.
constexpr int kWaves = 4;

template <int PIECES>
__device__ __forceinline__ int piece_at(int row, int piece) {
    constexpr int kWhole = (PIECES & -PIECES) < 16 ? (PIECES & -PIECES) : 16;  // pieces that an XOR may permute
    constexpr int kShift = kWhole == 16 ? 0 : kWhole == 8 ? 1 : 2;
    return row * PIECES + (piece ^ ((row >> kShift) & (kWhole - 1)));
}

template <typename T, int W>
struct Shape {
    // Blocks of 16 pairs of a wave, as its registers allow: with two waves a SIMD up to 128 lanes, with one past them.
    static constexpr int kBlocks = (sizeof(T) == 2 && W <= 192) || W <= 64 ? 2 : 1;
    static constexpr int kWavesPerSimd = W <= 128 ? 2 : 1;
    static constexpr int kPairs = 16 * kBlocks * kWaves;
    static constexpr int kKeyPieces = W * sizeof(T) / 16, kValuePieces = kTile * sizeof(T) / 16;
    static constexpr int kKeys = kTile * kKeyPieces, kValues = W * kValuePieces;  // pieces of a tile
    static constexpr int kPieces = kKeys + kValues;
    static constexpr int kPer = (kPieces + kThreads - 1) / kThreads;             // pieces a thread moves
    // Whether all threads' i-th pieces belong to the keys, or all to the values.
    static constexpr bool kEven = kKeys % kThreads == 0 && kValues % kThreads == 0;
    static constexpr int kPart = W < 128 ? W : 128;                              // lanes of narrow results joined at once
    static constexpr int kTiles = 2 * kPieces * 16, kJoin = kWaves * 16 * (kPart + 4 + 2) * 4;
    // LDS: tiles or results, the pairs' rows, and a bit per token of every value lane (two buffers).
    static constexpr int kRowsAt = kTiles > kJoin ? kTiles : kJoin, kSpoiledAt = kRowsAt + kPairs * 16;
    static constexpr int kLds = kSpoiledAt + 2 * W * 4;
};

template <typename T, int W, bool TREES>
__device__ __forceinline__ void attend_few(const AttentionArgs& a, const PlanItem& item, uint8_t* lds, int wave, int stride) {
    using M = Math<T, W>;
    using S = Shape<T, W>;
    using Fragment = typename M::Fragment;
    constexpr int kPart = S::kPart;
    constexpr int kKeyUnit = sizeof(T) == 2 ? 32 : 16;  // lanes a key fragment's step covers
    constexpr int kGroupLanes = 16 / sizeof(T);         // elements of a fragment
    const int thread = unknown(threadIdx.x), lane = thread & 63, c = lane & 15, g = lane >> 4;
    const int head_dim = unknown_scalar(a.s.head_dim);
    const Pages pages(a, item, static_cast<int64_t>(a.s.page_tokens) * W * sizeof(T));
    Fragment k[2][M::kKeyParts], v[W / 16][M::kValueParts];
    const auto load_keys = [&](int page, int t) {
        const T* p = reinterpret_cast<const T*>(pages.keys(page)) + pages.within(t) * W + kGroupLanes * g;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int s = 0; s < M::kKeyParts; ++s)
                k[h][s] = *(const SATORI_GLOBAL Fragment*)(p + M::key_token(h, c) * W + kKeyUnit * s);
    };
    const auto load_values = [&](int page, int t) {
        const T* p = reinterpret_cast<const T*>(pages.values(page)) + pages.within(t) + c * pages.tokens + kGroupLanes * g;
#pragma unroll
        for (int d = 0; d < W / 16; ++d)
#pragma unroll
            for (int h = 0; h < M::kValueParts; ++h)
                v[d][h] = *(const SATORI_GLOBAL Fragment*)(p + 16 * d * pages.tokens + 16 * h);
    };
    int t = wave * kTile, page = 0;
    const Pair pair = pair_of<TREES>(a, item, c);
    if (t < item.tokens) {
        page = wave == 0 ? item.tile[0] : wave == 1 ? item.tile[1] : wave == 2 ? item.tile[2] : item.tile[3];
        load_keys(page, t);
        load_values(page, t);
        if (t + kWaves * kTile < item.tokens) page = pages.page(t + kWaves * kTile);
    }
    PlanRow* row_of = reinterpret_cast<PlanRow*>(lds + S::kRowsAt);
    if (thread < 16) row_of[thread] = pair.row;
    typename M::Query q;
    M::load_query(q, query_of(a, pair), pair.is, head_dim, a.quads, a.scale, g);
    const Sight<TREES> sight(a, item, pair, stride);
    const auto hidden = [&](int t) { return item.first + t + kTile - 1 > item.limit; };
    const auto in_part = [&](int t) { return hidden(t) || item.tokens - t < kTile; };
    typename Sight<TREES>::Seen ahead{};  // of the next tile that is not seen whole, read a tile before
    if (t < item.tokens && in_part(t)) ahead = sight.of(a, item, t, item.tokens - t, stride);
    Softmax<W> x;
    x.clear();
    while (t < item.tokens) {
        f32x4 score[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
#pragma unroll
        for (int s = 0; s < M::kKeyParts; ++s)
#pragma unroll
            for (int term = 0; term < M::kTerms; ++term)
#pragma unroll
                for (int h = 0; h < 2; ++h) score[h] = M::score(k[h][s], q, s, term, score[h]);
        const int next = t + kWaves * kTile;
        if (next < item.tokens) load_keys(page, next);
        const int end = item.tokens - t;  // tokens of this tile that exist
        const bool hides = hidden(t);
        const auto seen = ahead;
        if (next < item.tokens && in_part(next)) ahead = sight.of(a, item, next, item.tokens - next, stride);
        if (end < kTile) {
            // Values of tokens behind the end become zero (they are nobody's, and may hold anything).
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (M::token(g, i) >= end)
#pragma unroll
                    for (int d = 0; d < W / 16; ++d) v[d][i / kGroupLanes][i % kGroupLanes] = 0;
        }
        if (hides) {
            bool finite = true;
#pragma unroll
            for (int d = 0; d < W / 16; ++d)
#pragma unroll
                for (int h = 0; h < M::kValueParts; ++h) finite &= all_finite(v[d][h]);
            if (!__all(finite))
#pragma unroll
                for (int d = 0; d < W / 16; ++d)
#pragma unroll
                    for (int h = 0; h < M::kValueParts; ++h) {
                        const Fragment spoiled = take_spoiled(v[d][h]);
                        spoil<M>(spoiled, seen, h, g, x.o[d]);
                    }
        }
        if (hides || end < kTile) hide<M>(score, seen, g);
        float p[8];
        x.take(score, q.factor, M::kTop, p);
        typename M::Weights w;
        M::weights(p, w);
#pragma unroll
        for (int h = 0; h < M::kValueParts; ++h)
#pragma unroll
            for (int term = 0; term < M::kTerms; ++term)
#pragma unroll
                for (int d = 0; d < W / 16; ++d) x.o[d] = M::weigh(v[d][h], w, h, term, x.o[d]);
        if (next < item.tokens) {
            load_values(page, next);
            if (next + kWaves * kTile < item.tokens) page = pages.page(next + kWaves * kTile);
        }
        t = next;
    }

    // The waves' results joined, up to 128 lanes at a time: [wave][pair][kPart + 4], then (maximum, sum) of each.
    float* joined = reinterpret_cast<float*>(lds);
    float* stats = joined + kWaves * 16 * (kPart + 4);
    const float sum = column_sum(x.l);
    if (g == 0) {
        stats[(wave * 16 + c) * 2] = x.m;
        stats[(wave * 16 + c) * 2 + 1] = sum;
    }
    const int mine = thread >> 4;  // 16 threads a pair, four lanes each and turn
#pragma unroll
    for (int part = 0; part < (W + kPart - 1) / kPart; ++part) {
        if (part > 0) __syncthreads();
#pragma unroll
        for (int d = 0; d < kPart / 16; ++d) {
            const int of = part * (kPart / 16) + d;
            if (of < W / 16) *reinterpret_cast<f32x4*>(joined + (wave * 16 + c) * (kPart + 4) + 16 * d + 4 * g) = x.o[of < W / 16 ? of : 0];
        }
        __syncthreads();
        if (mine >= item.pairs) continue;
        const int group = a.s.heads / a.s.kv_heads;
        const Pair to{row_of[mine], item.kv * group + (item.pair + mine) % group, true};
        float top = -INFINITY, total = 0, weight[kWaves];
#pragma unroll
        for (int w = 0; w < kWaves; ++w) top = fmaxf(top, stats[(w * 16 + mine) * 2]);
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            weight[w] = __builtin_amdgcn_exp2f(stats[(w * 16 + mine) * 2] - (top == -INFINITY ? 0.0f : top));
            total += weight[w] * stats[(w * 16 + mine) * 2 + 1];
        }
        const int left = W - part * kPart < kPart ? W - part * kPart : kPart;
        for (int d = 4 * (thread & 15); d < left; d += 64) {
            f32x4 o{0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < kWaves; ++w)
                o = o + *reinterpret_cast<const f32x4*>(joined + (w * 16 + mine) * (kPart + 4) + d) * weight[w];
            give<W>(a, item, to, part * kPart + d, o, total);
        }
        if (part == 0 && (thread & 15) == 0) give_sums<W>(a, item, to, top, total);
    }
}

template <typename T, int W, bool TREES>
__device__ __forceinline__ void attend_many(const AttentionArgs& a, const PlanItem& item, uint8_t* lds, int wave, int stride) {
    using M = Math<T, W>;
    using S = Shape<T, W>;
    using Fragment = typename M::Fragment;
    constexpr int NB = S::kBlocks;
    const int thread = unknown(threadIdx.x), lane = thread & 63, c = lane & 15, g = lane >> 4;
    const int head_dim = unknown_scalar(a.s.head_dim);
    const Pages pages(a, item, static_cast<int64_t>(a.s.page_tokens) * W * sizeof(T));
    const int tiles = (item.tokens + kTile - 1) / kTile;
    const bool idle = 16 * NB * wave >= item.pairs;  // a wave without pairs only carries
    uint32_t* spoiled = reinterpret_cast<uint32_t*>(lds + S::kSpoiledAt);  // [2][W]

    // Where its pieces go and come from stays in a thread's registers from tile to tile if they are few.
    const auto of_thread = [&] { return S::kPer > 8 ? unknown(thread) : thread; };
    const auto fetch = [&](int page, int tile, u32x4 (&moved)[S::kPer]) {
        const int thread = of_thread();
        const int within = pages.within(tile * kTile);
        const uint8_t* keys = pages.keys(page) + within * (W * static_cast<int>(sizeof(T)));
        const uint8_t* values = pages.values(page) + within * static_cast<int>(sizeof(T));
#pragma unroll
        for (int i = 0; i < S::kPer; ++i) {
            const int piece = thread + i * kThreads;
            if (S::kPieces % kThreads != 0 && piece >= S::kPieces) continue;
            const uint32_t row = (piece - S::kKeys) / S::kValuePieces, of = (piece - S::kKeys) % S::kValuePieces;
            const uint32_t value = row * pages.tokens * static_cast<uint32_t>(sizeof(T)) + of * 16;
            if (S::kEven)  // (a scalar base and 32 bits that stay the same from tile to tile)
                moved[i] = i * kThreads < S::kKeys ? *(const SATORI_GLOBAL u32x4*)(keys + static_cast<uint32_t>(piece) * 16)
                                                   : *(const SATORI_GLOBAL u32x4*)(values + value);
            else
                moved[i] = *(const SATORI_GLOBAL u32x4*)(piece < S::kKeys ? keys + piece * 16 : values + value);
        }
    };
    const auto put = [&](int tile, const u32x4 (&moved)[S::kPer]) {
        const int thread = of_thread();
        u32x4* buffer = reinterpret_cast<u32x4*>(lds) + (tile & 1) * S::kPieces;
#pragma unroll
        for (int i = 0; i < S::kPer; ++i) {
            const int piece = thread + i * kThreads;
            if (S::kPieces % kThreads != 0 && piece >= S::kPieces) continue;
            if (S::kEven ? i * kThreads < S::kKeys : piece < S::kKeys) {
                buffer[piece_at<S::kKeyPieces>(M::key_row(piece / S::kKeyPieces), piece % S::kKeyPieces)] = moved[i];
            } else {
                const int row = (piece - S::kKeys) / S::kValuePieces, of = (piece - S::kKeys) % S::kValuePieces;
                buffer[S::kKeys + piece_at<S::kValuePieces>(row, of)] = moved[i];
            }
        }
    };
    // A tile that some pair does not see whole, once it is in LDS: values of tokens behind the item's end become zero (they
    // are nobody's, and may hold anything), and so do values that are not finite, whose places are kept as a bit per token
    // of every lane.
    const auto settle = [&](int tile) {
        const int left = item.tokens - tile * kTile;
        if (item.first + tile * kTile + kTile - 1 <= item.limit && left >= kTile) return;
        __syncthreads();
        constexpr int kOf = 16 / sizeof(T);
        Fragment* values = reinterpret_cast<Fragment*>(lds) + (tile & 1) * S::kPieces + S::kKeys;
#pragma unroll 1
        for (int row = thread; row < W; row += kThreads) {
            uint32_t where = 0;
#pragma unroll 1
            for (int piece = 0; piece < S::kValuePieces; ++piece) {
                Fragment v = values[piece_at<S::kValuePieces>(row, piece)];
#pragma unroll
                for (int j = 0; j < kOf; ++j) {
                    const int token = piece * kOf + j;
                    const bool fine = __builtin_isfinite(static_cast<float>(v[j]));
                    if (!fine && token < left) where |= 1u << token;
                    v[j] = fine && token < left ? v[j] : 0;
                }
                values[piece_at<S::kValuePieces>(row, piece)] = v;
            }
            spoiled[(tile & 1) * W + row] = where;
        }
    };

    u32x4 moved[2][S::kPer];  // tile i in set i % 2
    int page = 0;             // of the tile that is fetched next, read a tile before
    const auto page_of = [&](int tile) { return pages.page(min(tile, tiles - 1) * kTile); };
    if (tiles > 0) {
        fetch(item.tile[0], 0, moved[0]);
        if (tiles > 1) fetch(item.tile[1], 1, moved[1]);
    }
    typename M::Query q[NB];
    Softmax<W> x[NB];
    Sight<TREES> sight[NB];
    PlanRow* row_of = reinterpret_cast<PlanRow*>(lds + S::kRowsAt) + 16 * NB * wave;  // this wave's
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        x[b].clear();
        const Pair p = pair_of<TREES>(a, item, 16 * (NB * wave + b) + c);
        sight[b] = Sight<TREES>(a, item, p, stride);
        if (g == 0) row_of[16 * b + c] = p.row;
        M::load_query(q[b], query_of(a, p), p.is, head_dim, a.quads, a.scale, g);
    }
    if (tiles > 0) {
        put(0, moved[0]);
        if (tiles > 2) fetch(item.tile[2], 2, moved[0]);
        page = page_of(3);
        settle(0);
    }
    __syncthreads();
    const auto attend = [&](int tile, u32x4 (&next)[S::kPer]) {
        // The next tile's bytes, which came while the last two were attended, go into the other buffer (everyone has left it),
        // and the one three ahead sets out.
        const auto carry = [&] {
            if (tile + 1 < tiles) put(tile + 1, next);
            if (tile + 3 < tiles) {
                fetch(page, tile + 3, next);
                page = page_of(tile + 4);
            }
        };
        if (idle) {
            carry();
        } else {
            const int t = tile * kTile, end = item.tokens - t;
            const bool hides = item.first + t + kTile - 1 > item.limit;
            typename Sight<TREES>::Seen seen[NB] = {};
            if (hides || end < kTile)
#pragma unroll
                for (int b = 0; b < NB; ++b) seen[b] = sight[b].of(a, item, t, end, stride);
            const Fragment* keys = reinterpret_cast<const Fragment*>(lds) + (tile & 1) * S::kPieces;
            const Fragment* values = keys + S::kKeys;
            f32x4 score[NB][2];
#pragma unroll
            for (int b = 0; b < NB; ++b) score[b][0] = score[b][1] = f32x4{0, 0, 0, 0};
            // Fragments are read ahead of the products that take them: a read takes as long as eight products, and a wave is
            // alone on its SIMD. (The barriers keep the order: the compiler would read each right before its use.)
            Fragment k[2][2];
            const auto read_keys = [&](int s) {
#pragma unroll
                for (int h = 0; h < 2; ++h) k[s & 1][h] = keys[piece_at<S::kKeyPieces>(16 * h + c, 4 * s + g)];
            };
            read_keys(0);
#pragma unroll
            for (int s = 0; s < M::kKeyParts; ++s) {
                if (s + 1 < M::kKeyParts) read_keys(s + 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int term = 0; term < M::kTerms; ++term)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int b = 0; b < NB; ++b) score[b][h] = M::score(k[s & 1][h], q[b], s, term, score[b][h]);
                __builtin_amdgcn_sched_barrier(0);
            }
            constexpr int kAhead = W < 256 ? 4 : 2, kFragments = M::kValueParts * (W / 16);
            Fragment v[kAhead];
            const auto read_values = [&](int i) {
                v[i % kAhead] = values[piece_at<S::kValuePieces>(16 * (i % (W / 16)) + c, 4 * (i / (W / 16)) + g)];
            };
            carry();
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < kAhead; ++i) read_values(i);
            typename M::Weights w[NB];
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if (hides || end < kTile) hide<M>(score[b], seen[b], g);
                float p[8];
                x[b].take(score[b], q[b].factor, M::kTop, p);
                M::weights(p, w[b]);
                if (hides) {
                    const uint32_t sees = Sight<TREES>::bits(seen[b]);
                    const u32x4* bits = reinterpret_cast<const u32x4*>(spoiled + (tile & 1) * W);
#pragma unroll
                    for (int d = 0; d < W / 16; ++d) {
                        const u32x4 where = bits[4 * d + g];
#pragma unroll
                        for (int j = 0; j < 4; ++j) x[b].o[d][j] = where[j] & sees ? NAN : x[b].o[d][j];
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < kFragments; ++i) {
                __builtin_amdgcn_sched_barrier(0);
                const int d = i % (W / 16), h = i / (W / 16);
#pragma unroll
                for (int term = 0; term < M::kTerms; ++term)
#pragma unroll
                    for (int b = 0; b < NB; ++b) x[b].o[d] = M::weigh(v[i % kAhead], w[b], h, term, x[b].o[d]);
                if (i + kAhead < kFragments) read_values(i + kAhead);
            }
        }
        if (tile + 1 < tiles) settle(tile + 1);
        __syncthreads();
    };
    for (int tile = 0; tile < tiles; tile += 2) {
        attend(tile, moved[1]);
        if (tile + 1 < tiles) attend(tile + 1, moved[0]);
    }

    if (idle) return;
    const int group = a.s.heads / a.s.kv_heads;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const float total = column_sum(x[b].l);
        const int p = 16 * (NB * wave + b) + c;
        if (p >= item.pairs) continue;
        const Pair to{row_of[16 * b + c], item.kv * group + (item.pair + p) % group, true};
#pragma unroll
        for (int d = 0; d < W / 16; ++d) give<W>(a, item, to, 16 * d + 4 * g, x[b].o[d], total);
        if (g == 0) give_sums<W>(a, item, to, x[b].m, total);
    }
}

// Items of many pairs first, which take longest (one a CU, bound by arithmetic); those of few, bound by memory, run beside
// them (64 sequences as above, before later steps: two launches 64 + 27 us, one with the items in turn 92, with the many first
// 76). Workgroup u is u % 8 of its eight, which keeps items that read the same tokens on one XCD.
template <typename T, int W, bool TREES>
__global__ __launch_bounds__(kThreads, (Shape<T, W>::kWavesPerSimd)) void cache_attention_kernel(AttentionArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const PlanHeader* h = reinterpret_cast<const PlanHeader*>(a.image);
    const int wide = a.wide >= 0 ? a.wide : scalar_load(&h->wide), narrow = a.narrow >= 0 ? a.narrow : scalar_load(&h->narrow);
    const int stride = !TREES ? 0 : a.wide >= 0 ? a.tree_stride : scalar_load(&h->tree_stride);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (int u = blockIdx.x; u < wide + narrow; u += gridDim.x) {
        const bool many = u < wide;
        const int at = many ? a.at.wide_at : a.at.narrow_at;
        const PlanItem item = scalar_load(reinterpret_cast<const PlanItem*>(a.image + at) + (many ? u : u - wide));
        if (many)
            attend_many<T, W, TREES>(a, item, lds, wave, stride);
        else
            attend_few<T, W, TREES>(a, item, lds, wave, stride);
        if (u + static_cast<int>(gridDim.x) < wide + narrow) __syncthreads();  // the next item's tiles go where results lie
    }
}

// The partial results of one (row, head), joined by a workgroup with weights 2^(m_i - m): every wave finds the maximum, then
// groups of lanes read a part's values each, four lanes of the head a lane, and LDS joins the groups in order. Bound by the
// latency of its chain of reads (the parts come from other XCDs), so all parts of common plans are read at once: 24 x 12 pairs
// of up to 17 parts 3.9 us, 64 x 32 of 17 (18 MB) 7.2 us.
__global__ __launch_bounds__(kThreads) void cache_join_kernel(AttentionArgs a) {
    const CacheShape& s = a.s;
    const int count = a.rows >= 0 ? a.rows : scalar_load(&reinterpret_cast<const PlanHeader*>(a.image)->rows);
    const PlanRow* rows = reinterpret_cast<const PlanRow*>(a.image + a.at.rows_at);
    __shared__ f32x4 joined[kThreads];
    __shared__ float sums_of[kThreads];
    const int thread = threadIdx.x, lane = thread & 63;
    const int quads = s.width / 4, groups = kThreads / quads;  // 8 .. 64 threads take a part's values
    const int mine = thread / quads, d = thread % quads * 4;
    const int units = count * s.heads;
    for (int u = blockIdx.x; u < units; u += gridDim.x) {
        const int head = u % s.heads;
        const PlanRow row = scalar_load(rows + u / s.heads);
        if (row.slots <= 1) continue;
        const int64_t first = static_cast<int64_t>(row.slot) * s.heads + head;
        const float* sums = a.partials.sums(s.width, first);
        const float* values = a.partials.values(s.width, first) + d;
        float top = -INFINITY;
        for (int i = lane; i < row.slots; i += 64)
            top = fmaxf(top, load_f32(sums + static_cast<int64_t>(i) * s.heads * 2));
        float total = 0;
        f32x4 o{0, 0, 0, 0};
        float from = 0;
        for (int i0 = mine; i0 < row.slots || i0 == mine; i0 += 4 * groups) {
            f32x4 v[4];
            f32x2 part[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int64_t i = min(i0 + k * groups, row.slots - 1);
                part[k] = *(const SATORI_GLOBAL f32x2*)(sums + i * s.heads * 2);
                v[k] = *(const SATORI_GLOBAL f32x4*)(values + i * s.heads * s.width);
            }
            if (i0 == mine) {
#pragma unroll
                for (int k = 32; k > 0; k >>= 1) top = fmaxf(top, __shfl_xor(top, k, 64));
                from = top == -INFINITY ? 0.0f : top;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (mine >= groups || i0 + k * groups >= row.slots) break;
                const float weight = __builtin_amdgcn_exp2f(part[k][0] - from);
                total += weight * part[k][1];
                o = o + v[k] * weight;
            }
        }
        joined[thread] = o;
        sums_of[thread] = total;
        __syncthreads();
        if (thread < quads) {
            for (int k = 1; k < groups; ++k) {
                o = o + joined[k * quads + thread];
                total += sums_of[k * quads + thread];
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (d + j < s.head_dim) store_f32(a.output + static_cast<int64_t>(u) * s.head_dim + d + j, o[j] / total);
        }
        __syncthreads();
    }
}

// The same where rows have few parts: four lanes of a (row, head) a thread, all parts at once, added in the same order (the
// groups above would have one part each, and those without one add zeros). 512 x 32 pairs of 2 to 7 parts 10 us, where the
// workgroup a pair took 27; 1024 x 32 of 1 to 3 8 us instead of 34.
constexpr int kFewParts = 8;
__global__ __launch_bounds__(kThreads) void cache_join_few_kernel(AttentionArgs a) {
    const CacheShape& s = a.s;
    const uint32_t quads = s.width / 4, thread = blockIdx.x * kThreads + threadIdx.x, u = thread / quads;
    const int d = thread % quads * 4, head = u % s.heads;
    if (u / s.heads >= static_cast<uint32_t>(a.rows)) return;
    const PlanRow row = reinterpret_cast<const PlanRow*>(a.image + a.at.rows_at)[u / s.heads];
    if (row.slots <= 1) return;
    const int64_t first = static_cast<int64_t>(row.slot) * s.heads + head;
    const float* sums = a.partials.sums(s.width, first);
    const float* values = a.partials.values(s.width, first) + d;
    f32x2 part[kFewParts];
    f32x4 v[kFewParts];
#pragma unroll
    for (int i = 0; i < kFewParts; ++i) {
        const int64_t of = min(i, row.slots - 1);
        part[i] = *(const SATORI_GLOBAL f32x2*)(sums + of * s.heads * 2);
        v[i] = *(const SATORI_GLOBAL f32x4*)(values + of * s.heads * s.width);
    }
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kFewParts; ++i) top = fmaxf(top, part[i][0]);
    const float from = top == -INFINITY ? 0.0f : top;
    f32x4 o{0, 0, 0, 0};
    float total = 0;
#pragma unroll
    for (int i = 0; i < kFewParts; ++i)
        if (i < row.slots) {
            const float weight = __builtin_amdgcn_exp2f(part[i][0] - from);
            total += weight * part[i][1];
            o = o + v[i] * weight;
        }
    o = o + f32x4{0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (d + j < s.head_dim) store_f32(a.output + static_cast<int64_t>(u) * s.head_dim + d + j, o[j] / total);
}

constexpr int kMostGroups = 1024;  // workgroups of a launch whose work is only known when it is replayed

template <typename T, int W>
hipError_t attention_of_width(const AttentionArgs& a, int groups, bool trees, hipStream_t stream) {
    using S = Shape<T, W>;
    const auto kernel = trees ? cache_attention_kernel<T, W, true> : cache_attention_kernel<T, W, false>;
    // (more than 64 KB of LDS; set for the current device, where it is a table lookup after the first time)
    if (S::kLds > 64 * 1024)
        if (const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, S::kLds);
            e != hipSuccess)
            return e;
    kernel<<<groups, kThreads, S::kLds, stream>>>(a);
    return hipGetLastError();
}

// Calls f with the type and width of a shape as template arguments.
template <typename F>
auto of_shape(int type, int width, F&& f) {
    const auto of_type = [&](auto t) {
        switch (width) {
            case 32: return f(t, std::integral_constant<int, 32>{});
            case 64: return f(t, std::integral_constant<int, 64>{});
            case 96: return f(t, std::integral_constant<int, 96>{});
            case 128: return f(t, std::integral_constant<int, 128>{});
            case 192: return f(t, std::integral_constant<int, 192>{});
            default: return f(t, std::integral_constant<int, 256>{});
        }
    };
    return type == kF32 ? of_type(float{}) : of_type(_Float16{});
}

}  // namespace

int cache_wide_pairs(int type, int width) {
    return of_shape(type, width, [](auto t, auto w) { return Shape<decltype(t), decltype(w)::value>::kPairs; });
}

hipError_t launch_plan_copy(const int* from, int* to, const PlanLayout& layout, const PlanLayout& used, hipStream_t stream) {
    const int at[kPlanParts] = {0, layout.rows_at, layout.narrow_at, layout.wide_at, layout.runs_at, layout.pages_at,
                                layout.list_at, layout.trees_at};
    const size_t words[kPlanParts] = {sizeof(PlanHeader) / 4, used.rows * sizeof(PlanRow) / 4, used.narrow * sizeof(PlanItem) / 4,
                                      used.wide * sizeof(PlanItem) / 4, used.runs * sizeof(PlanRun) / 4,
                                      static_cast<size_t>(used.pages), used.list * sizeof(PlanRow) / 4,
                                      static_cast<size_t>(used.trees)};
    PlanParts parts;
    int end = 0;
    for (int i = 0; i < kPlanParts; ++i) {
        parts.at[i] = at[i] / 4;
        parts.end[i] = end += static_cast<int>((words[i] + 3) / 4);
    }
    plan_copy_kernel<<<(end + kThreads - 1) / kThreads, kThreads, 0, stream>>>(reinterpret_cast<const u32x4*>(from),
                                                                              reinterpret_cast<u32x4*>(to), parts);
    return hipGetLastError();
}

hipError_t launch_copy_pages(uint8_t* pool, int64_t page_bytes, const PageMoves& moves, hipStream_t stream) {
    if (moves.count == 0) return hipSuccess;
    const dim3 grid(static_cast<unsigned>((page_bytes + kCopyBytes - 1) / kCopyBytes), moves.count);
    copy_pages_kernel<<<grid, kThreads, 0, stream>>>(pool, page_bytes, moves);
    return hipGetLastError();
}

hipError_t launch_cache_append(const CacheShape& s, const int* image, const PlanLayout& layout, const PlanHeader& now,
                               bool all, bool trees, const AppendArgs& args, hipStream_t stream) {
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
    const dim3 grid(all ? 256 : std::min(now.runs, 1 << 16), y);
    const auto launch = [&](auto kernel) {
        kernel<<<grid, kThreads, 0, stream>>>(s, image, layout.runs_at, layout.trees_at, args);
    };
    const auto of_turn = [&](auto turn, auto listed) {
        constexpr Turn kTurn = decltype(turn)::value;
        constexpr bool kListed = decltype(listed)::value;
        if (s.type == kF32)
            packed ? launch(cache_append_kernel<float, 4, kTurn, kListed>) : launch(cache_append_kernel<float, 1, kTurn, kListed>);
        else
            packed ? launch(cache_append_kernel<_Float16, 4, kTurn, kListed>)
                   : launch(cache_append_kernel<_Float16, 1, kTurn, kListed>);
    };
    // Without the code that computes angles a wave takes half the registers. (A captured launch may meet any position.)
    const bool listed = !all && args.rope && now.most_position < args.rope_positions;
    const auto with = [&](auto turn) {
        listed ? of_turn(turn, std::true_type{}) : of_turn(turn, std::false_type{});
    };
    if (args.interleaved)
        with(std::integral_constant<Turn, Turn::kInterleaved>{});
    else if (trees || args.frequencies)
        with(std::integral_constant<Turn, Turn::kTree>{});
    else
        with(std::integral_constant<Turn, Turn::kPlain>{});
    return hipGetLastError();
}

hipError_t launch_cache_keep(const CacheShape& s, int layers, const KeepMoves& moves, hipStream_t stream) {
    if (moves.sequences == 0) return hipSuccess;
    const int64_t heads = static_cast<int64_t>(layers) * s.kv_heads;
    const int64_t waves = (heads * (s.width * element_bytes(s.type) / 16) + 63) / 64 + heads * ((s.head_dim + 31) / 32);
    if (waves > INT32_MAX / 128) return hipErrorInvalidValue;
    const dim3 grid(static_cast<unsigned>((waves + kThreads / 64 - 1) / (kThreads / 64)), moves.sequences);
    if (s.type == kF32)
        cache_keep_kernel<float><<<grid, kThreads, 0, stream>>>(s, layers, moves);
    else
        cache_keep_kernel<_Float16><<<grid, kThreads, 0, stream>>>(s, layers, moves);
    return hipGetLastError();
}

size_t cache_partial_bytes(const CacheShape& shape, int64_t slots) {
    return static_cast<size_t>(slots) * shape.heads * (shape.width + 2) * sizeof(float);
}

hipError_t launch_cache_attention(const CacheShape& shape, const int* image, const PlanLayout& layout, const PlanHeader& now,
                                  bool all, bool trees, int layer, const float* query, float* output, float* partials,
                                  size_t bytes, hipStream_t stream) {
    if (now.rows == 0 && !all) return hipSuccess;
    const int64_t room = static_cast<int64_t>(bytes / cache_partial_bytes(shape, 1)) * shape.heads;
    const float scale = static_cast<float>(static_cast<double>(kLog2e) / std::sqrt(static_cast<double>(shape.head_dim)));
    const AttentionArgs a{shape,
                          image,
                          layout,
                          all ? -1 : now.wide,
                          all ? -1 : now.narrow,
                          all ? -1 : now.rows,
                          layer,
                          query,
                          output,
                          Partials{partials, room},
                          scale,
                          shape.head_dim % 4 == 0 && reinterpret_cast<uintptr_t>(query) % 16 == 0,
                          now.tree_stride};
    const int groups = all ? kMostGroups : std::min(now.wide + now.narrow, 1 << 20);
    const hipError_t e = of_shape(shape.type, shape.width, [&](auto t, auto w) {
        return attention_of_width<decltype(t), decltype(w)::value>(a, groups, trees, stream);
    });
    if (e != hipSuccess || (now.joined == 0 && !all)) return e;
    const int64_t joins = static_cast<int64_t>(now.rows) * shape.heads;
    const int quads = shape.width / 4;
    if (!all && now.most_slots <= std::min(kFewParts, kThreads / quads) && joins * quads < INT32_MAX) {
        cache_join_few_kernel<<<static_cast<unsigned>((joins * quads + kThreads - 1) / kThreads), kThreads, 0, stream>>>(a);
        return hipGetLastError();
    }
    cache_join_kernel<<<all ? kMostGroups : static_cast<int>(std::min<int64_t>(joins, 65536)), kThreads, 0, stream>>>(a);
    return hipGetLastError();
}

}  // namespace satori
