// Launchers of the logits' kernels (logits.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace satori {

constexpr int kLogitSlice = 4096;  // tokens of a workgroup
constexpr int kLogitGroup = 16;    // rows of a workgroup, at most
constexpr int kLogitRows = 1024;   // rows of a launch, for each of which the workspace has a LogitBest
inline int logit_slices(int vocabulary) { return (vocabulary + kLogitSlice - 1) / kLogitSlice; }

// One row's parameters, as callers write them (satori_hip_logit_row).
struct LogitRow {
    float repetition, presence, frequency;
    int history, parent, token, biases, mask;
};

// The greatest value of a row so far, above its place's complement (0: none yet), and how many slices of it were done, counted
// through all launches, so that what a launch leaves behind is right for the next even after launches that overlapped.
struct LogitBest {
    unsigned long long key, arrived;
};

// The bias sets of a handle: each `starts` [slices + 1] (entries of slice s: starts[s] .. starts[s + 1] - 1), tokens and values
// [entries], tokens ascending, in `words` 4-byte words.
struct LogitBiases {
    const int* sets;
    int count, entries, words;
};
inline int64_t logit_bias_words(int vocabulary, int entries) {
    return (logit_slices(vocabulary) + 1 + 2 * static_cast<int64_t>(entries) + 3) / 4 * 4;
}

struct LogitArgs {
    const LogitRow* rows;  // of the whole batch
    int first, count;      // the launch's rows
    int vocabulary;
    const float* logits;
    float* output;         // or null
    int* best;             // or null
    int64_t logits_stride, output_stride;
    const int *history, *lengths;
    int64_t history_stride;
    int histories, mask_count;
    const uint32_t* masks;
    int64_t mask_stride;   // words
    LogitBiases biases;
    LogitBest* found;      // of the launch's rows
    int group;             // rows of a workgroup (launch_logits says)
};
hipError_t launch_logits(LogitArgs args, hipStream_t stream);

}  // namespace satori
