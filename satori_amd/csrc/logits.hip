// What stands between a model's logits and the chosen token: penalties for tokens that a row has had, biases, grammar masks
// and the best token.
#include "logits.hpp"

#include <algorithm>
#include <cmath>

#include "device_common.hpp"

namespace satori {
namespace {

constexpr int kThreads = 256;
constexpr int kPlaces = 1024;  // workgroups at once: four a CU, by their LDS and registers
constexpr int kListed = 2048;  // (where a row has had more of a slice's tokens, each thread looks at its own)
constexpr int kPacks = kLogitSlice / kThreads / 4;  // of four logits a thread

typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));

// A number that orders keys as their values do, values of zero alike.
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t bits = __float_as_uint(v + 0.0f);
    return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

__device__ __forceinline__ unsigned long long greater(unsigned long long a, unsigned long long b) { return a > b ? a : b; }

// What a thread has of one row's slice.
struct Slice {
    f32x4 x[kPacks];
    uint32_t allowed[kPacks];  // bit j of 4: of lane j of the pack
};

// One slice of the tokens of up to kLogitGroup rows, one row after another. How often a row has had each token (its history
// and, where it is a draft, its branch) is counted in LDS, with a list of the tokens that it has had. Rows of one history follow
// one another (a tree's, a request's), so the counts stay and only the branches change. What is listed, and what has a bias, is
// changed in LDS, one token a thread (each thread at its own tokens would divide for whole waves, 16 times a row); a row's
// logits and mask set out while the row before is at work. A row's slices meet in one atomic maximum each; the last to
// arrive, which sees them all (each waits for its maximum before it counts itself in), gives the best token. Sums and
// quotients in FP32, each rounded, in the order of the definition. Few rows are bound by the chain of reads and of the three
// atomics (one row of 151936 tokens and 2000 it has had 7.8 us, launch included), many by memory and the lists: 512 rows of 8 trees
// of 64 over 151936, histories of 100 to 16384, 156 us, 624 MB at 4.0 TB/s (without penalties 136, nothing but the copy 128).
__global__ __launch_bounds__(kThreads, 4) void logits_kernel(LogitArgs a) {
    __shared__ __attribute__((aligned(16))) int counts[kLogitSlice];
    __shared__ __attribute__((aligned(16))) float values[kLogitSlice];
    __shared__ uint16_t listed[kListed];
    __shared__ int list_length;
    __shared__ unsigned long long branches[kLogitGroup];
    __shared__ unsigned long long top[kLogitGroup][kThreads / 64];
    __shared__ LogitRow params[kLogitGroup];
    const int thread = threadIdx.x, slice = blockIdx.x, local = blockIdx.y * a.group, first = a.first + local;
    const int rows = min(a.group, a.first + a.count - first);
    const int begin = slice * kLogitSlice, end = min(a.vocabulary - begin, kLogitSlice);

    const auto load = [&](int i, Slice& to) {
        const float* in = a.logits + (first + i) * a.logits_stride + begin;
#pragma unroll
        for (int k = 0; k < kPacks; ++k) {
            const int at = k * kThreads * 4 + thread * 4;
            to.x[k] = f32x4{0, 0, 0, 0};
            if (at + 4 <= end) {
                to.x[k] = *(const SATORI_GLOBAL f32x4_a4*)(in + at);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (at + j < end) to.x[k][j] = load_f32(in + at + j);
            }
        }
    };
    const auto load_mask = [&](int i, Slice& to) {
        const int mask = __builtin_amdgcn_readfirstlane(params[i].mask);
        const bool is = mask >= 0 && mask < a.mask_count;
        const uint32_t* words = a.masks + (is ? mask : 0) * a.mask_stride + begin / 32;
#pragma unroll
        for (int k = 0; k < kPacks; ++k) {
            const int at = k * kThreads * 4 + thread * 4;
            to.allowed[k] = is && at < end ? words[at / 32] >> at % 32 : ~0u;
        }
    };
    Slice now, next;
    load(0, now);
    if (thread < rows * static_cast<int>(sizeof(LogitRow) / 4))
        reinterpret_cast<int*>(params)[thread] = reinterpret_cast<const int*>(a.rows + first)[thread];
    // The branches' rows: those of a window of 64 lie in the lanes of a wave, at first the last 64 up to the group's end.
    const int lane = thread & 63, latest = max(0, first + rows - 64);
    int base = latest, parent = -1, token = -1;
    const auto look = [&](int from) {
        base = from;
        const int mine = min(base + lane, first + rows - 1);
        parent = a.rows[mine].parent;
        token = a.rows[mine].token;
    };
    look(latest);
    __syncthreads();
    load_mask(0, now);
    // A bit for every row of that window that a row's branch has, or none where it goes back further.
    for (int i = __builtin_amdgcn_readfirstlane(thread / 64); i < rows; i += kThreads / 64) {
        unsigned long long has = 0;
        for (int at = first + i; at >= 0;) {
            if (at < base) {
                has = 0;
                break;
            }
            has |= 1ull << (at - base);
            const int up = __builtin_amdgcn_readlane(parent, at - base);
            at = up < at ? up : -1;
        }
        if (lane == 0) branches[i] = has;
    }

    const auto count = [&](int of, int by) {
        const uint32_t at = static_cast<uint32_t>(of) - static_cast<uint32_t>(begin);
        if (at >= static_cast<uint32_t>(end) || atomicAdd(counts + at, by) != 0 || by < 0) return;
        const int place = atomicAdd(&list_length, 1);
        if (place < kListed) listed[place] = static_cast<uint16_t>(at);
    };
    // Counts a row's branch (the first wave): the rows that it has, at once, or window after window.
    const auto count_branch = [&](int row, int by) {
        const unsigned long long has = branches[row - first];
        if (has) {
            if (has >> lane & 1) count(token, by);
            return;
        }
        for (int at = row; at >= 0;) {
            if (at < base || at > base + 63) look(at > base ? latest : max(0, at - 63));
            const int of = __builtin_amdgcn_readfirstlane(at - base);
            if (lane == of) count(token, by);
            const int up = __builtin_amdgcn_readlane(parent, of);
            at = up < at ? up : -1;
        }
        look(latest);
    };
    // A bias set's entries of the slice: a thread's first one stays with it.
    int put = -1, bias_end = 0, bias_from = 0, bias_at = 0;
    float bias_by = 0;
    const auto take_biases = [&](int set) {
        const int* starts = a.biases.sets + static_cast<int64_t>(set) * a.biases.words;
        put = set;
        bias_from = starts[slice] + thread;
        bias_end = starts[slice + 1];
        if (bias_from < bias_end) {
            bias_at = starts[gridDim.x + 1 + bias_from] - begin;
            bias_by = reinterpret_cast<const float*>(starts)[gridDim.x + 1 + a.biases.entries + bias_from];
        }
    };
    int counted = -2, of_history = 0, walked = -1;  // the history that LDS holds, its part of the list, and the branch
    const auto pass = [&](int i, const Slice& now, Slice& next) {
        const int row = first + i;
        if (i + 1 < rows) {
            load(i + 1, next);
            load_mask(i + 1, next);
        }
        const LogitRow r = params[i];
        const bool penalises = r.repetition != 1.0f || r.presence != 0.0f || r.frequency != 0.0f;
        const int set = r.biases >= 0 && r.biases < a.biases.count ? r.biases : -1;
        const int history = r.history >= 0 && r.history < a.histories ? r.history : -1;
        if (penalises && history != counted) {
            for (int k = thread; k < kLogitSlice / 4; k += kThreads) reinterpret_cast<u32x4*>(counts)[k] = u32x4{0, 0, 0, 0};
            if (thread == 0) list_length = 0;
            __syncthreads();
            counted = history;
            walked = -1;
            if (history >= 0) {
                const int* tokens = a.history + history * a.history_stride;
                // (unsigned: the last turn's places pass 2^31 where the longest history's tokens end just below it)
                const uint32_t length = static_cast<uint32_t>(min(static_cast<int64_t>(max(a.lengths[history], 0)), a.history_stride));
                // Sixteen tokens a thread and turn, all on their way at once.
                for (uint32_t k0 = 0; k0 < length; k0 += kThreads * 16) {
                    i32x4_a4 had[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t at = k0 + (k * kThreads + thread) * 4;
                        if (at + 4 <= length) {
                            had[k] = *(const SATORI_GLOBAL i32x4_a4*)(tokens + at);
                        } else {
#pragma unroll
                            for (int j = 0; j < 4; ++j) had[k][j] = at + j < length ? tokens[at + j] : -1;
                        }
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k)
#pragma unroll
                        for (int j = 0; j < 4; ++j) count(had[k][j], 1);
                }
            }
            __syncthreads();
            of_history = list_length;  // (the first wave's own is what counts)
        }
        if (penalises && thread < 64) {
            if (walked >= 0) {
                count_branch(walked, -1);
                if (thread == 0) list_length = of_history;
            }
            count_branch(row, 1);
        }
        if (penalises) walked = row;
        if (set >= 0 && set != put) take_biases(set);
        Slice mine = now;
        if (penalises || set >= 0) {
#pragma unroll
            for (int k = 0; k < kPacks; ++k) *reinterpret_cast<f32x4*>(values + k * kThreads * 4 + thread * 4) = now.x[k];
            __syncthreads();
            if (penalises) {
                const auto penalise = [&](int at) {
                    const float x = values[at];
                    const float v = x > 0 ? x / r.repetition : x * r.repetition;
                    values[at] = v - (r.presence + r.frequency * static_cast<float>(counts[at]));
                };
                const int length = list_length;
                if (length <= kListed)
                    for (int k = thread; k < length; k += kThreads) penalise(listed[k]);
                else
                    for (int at = thread; at < end; at += kThreads)
                        if (counts[at] > 0) penalise(at);
            }
            if (set >= 0) {
                if (penalises) __syncthreads();
                const auto add = [&](int at, float by) {
                    if (by != 0) values[at] = values[at] + by;
                };
                if (bias_from < bias_end) add(bias_at, bias_by);
                const int* tokens = a.biases.sets + static_cast<int64_t>(set) * a.biases.words + gridDim.x + 1;
                for (int k = bias_from + kThreads; k < bias_end; k += kThreads)
                    add(tokens[k] - begin, reinterpret_cast<const float*>(tokens)[a.biases.entries + k]);
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < kPacks; ++k) mine.x[k] = *reinterpret_cast<const f32x4*>(values + k * kThreads * 4 + thread * 4);
        }

        float best = -INFINITY;
        int best_at = -1;  // a thread's tokens go up, so an equal one is a higher one
#pragma unroll
        for (int k = 0; k < kPacks; ++k) {
            const int at = k * kThreads * 4 + thread * 4;
            if (at >= end) break;
            f32x4 x = mine.x[k];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[j] = now.allowed[k] >> j & 1 ? x[j] : -INFINITY;
                if (x[j] > best && at + j < end) {
                    best = x[j];
                    best_at = at + j;
                }
            }
            if (!a.output) continue;
            float* out = a.output + row * a.output_stride + begin + at;
            if (at + 4 <= end) {
                *(SATORI_GLOBAL f32x4_a4*)(out) = x;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (at + j < end) store_f32(out + j, x[j]);
            }
        }
        if (a.best) {
            const uint32_t value = best_at < 0 ? 0 : ordered(best), most = wave_extreme_u32<true>(value);
            const uint32_t place = wave_extreme_u32<false>(value == most ? static_cast<uint32_t>(begin + best_at) : ~0u);
            if (lane == 0) top[i][thread / 64] = most ? static_cast<unsigned long long>(most) << 32 | ~place : 0;
        }
    };
    for (int i = 0; i < rows; i += 2) {
        pass(i, now, next);
        if (i + 1 < rows) pass(i + 1, next, now);
    }
    __syncthreads();
    if (!a.best || thread >= rows) return;
    unsigned long long key = top[thread][0];
#pragma unroll
    for (int k = 1; k < kThreads / 64; ++k) key = greater(key, top[thread][k]);
    if (gridDim.x == 1) {
        a.best[first + thread] = key ? static_cast<int>(~static_cast<uint32_t>(key)) : -1;
        return;
    }
    LogitBest* found = a.found + local + thread;
    __hip_atomic_fetch_max(&found->key, key, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const unsigned long long seen = __hip_atomic_fetch_add(&found->arrived, 1ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if ((seen + 1) % gridDim.x != 0) return;
    key = __hip_atomic_exchange(&found->key, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    a.best[first + thread] = key ? static_cast<int>(~static_cast<uint32_t>(key)) : -1;
}

}  // namespace

hipError_t launch_logits(LogitArgs args, hipStream_t stream) {
    if (args.count <= 0) return hipSuccess;
    // Rows of a workgroup: four rounds of the workgroups that the card holds (four a CU), as the last one is not full. (512 x
    // 151936: two rounds 171 us, four 156, eight 165, each row by itself 320.)
    const int64_t units = static_cast<int64_t>(logit_slices(args.vocabulary)) * args.count;
    args.group = static_cast<int>(std::min<int64_t>(kLogitGroup, std::max<int64_t>(1, units / (4 * kPlaces))));
    const dim3 grid(logit_slices(args.vocabulary), (args.count + args.group - 1) / args.group);
    logits_kernel<<<grid, kThreads, 0, stream>>>(args);
    return hipGetLastError();
}

}  // namespace satori
