// What stands between a model's logits and the chosen token: penalties for tokens that a row has had, biases, grammar masks
// and the best token.
#include "logits.hpp"

#include <cmath>

#include "device_common.hpp"

namespace satori {
namespace {

constexpr int kThreads = 256;
constexpr int kPacks = kLogitSlice / kThreads / 4;  // of four logits a thread

typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));

// A number that orders keys as their values do, values of zero alike.
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t bits = __float_as_uint(v + 0.0f);
    return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

__device__ __forceinline__ unsigned long long greater(unsigned long long a, unsigned long long b) { return a > b ? a : b; }

// One slice of a row's tokens: how often the row has had each (its history and, where it is a draft, its branch) is counted
// in LDS, the biases put beside, then all of it meets the logits, which set out first. A row's slices meet in one atomic
// maximum each; the last to arrive, which sees them all (each waits for its maximum before it counts itself in), gives the
// best token. Sums and quotients in FP32, each rounded, in the order of the definition.
__global__ __launch_bounds__(kThreads) void logits_kernel(LogitArgs a) {
    __shared__ int counts[kLogitSlice];
    __shared__ float biases[kLogitSlice];
    __shared__ unsigned long long top[kThreads / 64];
    const int thread = threadIdx.x, slice = blockIdx.x, local = blockIdx.y, row = a.first + local;
    const int begin = slice * kLogitSlice, end = min(a.vocabulary - begin, kLogitSlice);
    const LogitRow r = a.rows[row];
    const float* in = a.logits + row * a.logits_stride + begin;

    f32x4 x[kPacks];
#pragma unroll
    for (int i = 0; i < kPacks; ++i) {
        const int at = i * kThreads * 4 + thread * 4;
        x[i] = f32x4{0, 0, 0, 0};
        if (at + 4 <= end) {
            x[i] = *(const SATORI_GLOBAL f32x4_a4*)(in + at);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (at + j < end) x[i][j] = load_f32(in + at + j);
        }
    }

    const bool penalises = r.repetition != 1.0f || r.presence != 0.0f || r.frequency != 0.0f;
    const bool biased = r.biases >= 0 && r.biases < a.biases.count;
    if (penalises)
        for (int i = thread; i < kLogitSlice; i += kThreads) counts[i] = 0;
    if (biased)
        for (int i = thread; i < kLogitSlice; i += kThreads) biases[i] = 0;
    __syncthreads();
    const auto count = [&](int token) {
        const uint32_t at = static_cast<uint32_t>(token) - static_cast<uint32_t>(begin);
        if (at < static_cast<uint32_t>(end)) atomicAdd(counts + at, 1);
    };
    if (penalises) {
        if (r.history >= 0 && r.history < a.histories) {
            const int* history = a.history + r.history * a.history_stride;
            const int length = static_cast<int>(min(static_cast<int64_t>(max(a.lengths[r.history], 0)), a.history_stride));
            for (int i = thread; i < length; i += kThreads) count(history[i]);
        }
        if (thread < 64) {
            // Up the branch: the rows of a window of 64 lie in the lanes.
            int at = row, base = row + 1, parent = -1, token = -1;
            while (at >= 0) {
                if (at < base) {
                    base = max(0, at - 63);
                    const int mine = min(base + thread, row);
                    parent = a.rows[mine].parent;
                    token = a.rows[mine].token;
                }
                const int of = __builtin_amdgcn_readfirstlane(at - base);
                if (thread == 0) count(__builtin_amdgcn_readlane(token, of));
                const int up = __builtin_amdgcn_readlane(parent, of);
                at = up < at ? up : -1;
            }
        }
    }
    if (biased) {
        const int* set = a.biases.sets + static_cast<int64_t>(r.biases) * a.biases.words;
        const int* tokens = set + gridDim.x + 1;
        const float* values = reinterpret_cast<const float*>(tokens + a.biases.entries);
        for (int i = set[slice] + thread; i < set[slice + 1]; i += kThreads) biases[tokens[i] - begin] = values[i];
    }
    __syncthreads();

    const bool masked = r.mask >= 0 && r.mask < a.mask_count;
    const uint32_t* mask = masked ? a.masks + r.mask * a.mask_stride + begin / 32 : nullptr;
    unsigned long long key = 0;
#pragma unroll
    for (int i = 0; i < kPacks; ++i) {
        const int at = i * kThreads * 4 + thread * 4;
        if (at >= end) break;
        const uint32_t allowed = masked ? mask[at / 32] >> at % 32 : ~0u;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float v = x[i][j];
            if (penalises) {
                const int n = counts[at + j];
                if (n > 0) {
                    v = v > 0 ? v / r.repetition : v * r.repetition;
                    v = v - (r.presence + r.frequency * static_cast<float>(n));
                }
            }
            if (biased) {
                const float b = biases[at + j];
                v = b != 0 ? v + b : v;
            }
            v = allowed >> j & 1 ? v : -INFINITY;
            x[i][j] = v;
            if (at + j < end && v > -INFINITY)
                key = greater(key, static_cast<unsigned long long>(ordered(v)) << 32 | ~static_cast<uint32_t>(begin + at + j));
        }
        if (!a.output) continue;
        float* out = a.output + row * a.output_stride + begin + at;
        if (at + 4 <= end) {
            *(SATORI_GLOBAL f32x4_a4*)(out) = x[i];
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (at + j < end) store_f32(out + j, x[i][j]);
        }
    }
    if (!a.best) return;
#pragma unroll
    for (int k = 32; k > 0; k >>= 1) key = greater(key, __shfl_xor(key, k, 64));
    if (thread % 64 == 0) top[thread / 64] = key;
    __syncthreads();
    if (thread != 0) return;
#pragma unroll
    for (int i = 1; i < kThreads / 64; ++i) key = greater(key, top[i]);
    LogitBest* found = a.found + local;
    __hip_atomic_fetch_max(&found->key, key, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const unsigned long long seen = __hip_atomic_fetch_add(&found->arrived, 1ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if ((seen + 1) % gridDim.x != 0) return;
    key = __hip_atomic_exchange(&found->key, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    a.best[row] = key ? static_cast<int>(~static_cast<uint32_t>(key)) : -1;
}

}  // namespace

hipError_t launch_logits(const LogitArgs& args, hipStream_t stream) {
    if (args.count <= 0) return hipSuccess;
    logits_kernel<<<dim3(logit_slices(args.vocabulary), args.count), kThreads, 0, stream>>>(args);
    return hipGetLastError();
}

}  // namespace satori
