// sample.hpp -- vkml_sample's parameter checks, how a row is split and what the
// workspace holds. Code without HIP's runtime, so that it can be tested on any
// machine.
#pragma once

#include <cstdint>

#include "../../include/vkml_hip.h"

namespace vkml::sample {

constexpr uint32_t kThreads = 1024;
constexpr uint32_t kVectors = 8;                         // of four values, a thread's of a slice
constexpr uint32_t kSlice = 4 * kVectors * kThreads;     // values a workgroup holds in registers
constexpr uint32_t kBins = 2048;
constexpr uint32_t kMaxVocab = 1u << 22;
constexpr uint32_t kMaxSlices = 1u << 21;

inline uint32_t slices(uint32_t vocab) { return (vocab + kSlice - 1) / kSlice; }

inline const char* check(const vkml_sample_params& p) {
    if (p.vocab == 0 || p.vocab > kMaxVocab) return "rows must hold 1 to 2^22 logits";
    if (p.row_stride < p.vocab) return "rows overlap";
    if (p.row_stride > (1ull << 40)) return "row_stride is too large";
    // (a launch has less than 2^32 threads)
    if (static_cast<uint64_t>(p.rows) * slices(p.vocab) > kMaxSlices) return "too many rows";
    return nullptr;
}

// What a row of several slices keeps: a slice's largest, its sums and counts by
// bin, and its mass past min_p.
struct SliceSums {
    uint64_t mass[kBins];
    uint32_t count[kBins];
    uint64_t likely;
};
inline uint64_t peaks_bytes(const vkml_sample_params& p) { return (static_cast<uint64_t>(p.rows) * slices(p.vocab) * 8 + 15) / 16 * 16; }
inline uint64_t workspace_bytes(const vkml_sample_params& p) {
    const uint64_t n = slices(p.vocab);
    return n == 1 ? 0 : peaks_bytes(p) + static_cast<uint64_t>(p.rows) * n * sizeof(SliceSums);
}

}  // namespace vkml::sample
