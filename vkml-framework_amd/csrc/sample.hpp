// sample.hpp -- vkml_sample's parameter checks, how a row is split and what the
// workspace holds. Code without HIP's runtime, so that it can be tested on any
// machine.
#pragma once

#include <cstdint>

#include "../../include/vkml_hip.h"

namespace vkml::sample {

// A workgroup holds a slice of a row, or the whole, in registers: so many threads,
// vectors of four values each.
constexpr uint32_t kWideThreads = 1024, kNarrowThreads = 256;
constexpr uint32_t kVectors = 8;
constexpr uint32_t kSlice = 4 * kVectors * kWideThreads;
constexpr uint32_t kNarrowRow = 4 * kVectors * kNarrowThreads;  // rows up to that many take the narrow one
constexpr uint32_t kBins = 2048;  // of weights
constexpr uint32_t kList = 2048;  // candidates in the LDS
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

// Weights and counts by bin, and the mass within min_p: a slice's, or a row's up to
// each bin.
struct Sums {
    uint64_t mass[kBins];
    uint32_t count[kBins];
    uint64_t likely;
    uint64_t unused;
};
// What a row of several slices keeps of one: its sums, and the ids of candidates, more
// than kList where these are not all.
struct Slice {
    Sums sums;
    uint32_t id[kList];
    uint32_t listed, unused[3];
};
inline uint64_t peaks_bytes(const vkml_sample_params& p) { return (static_cast<uint64_t>(p.rows) * slices(p.vocab) * 8 + 15) / 16 * 16; }
inline uint64_t workspace_bytes(const vkml_sample_params& p) {
    const uint64_t n = slices(p.vocab);
    return n == 1 ? 0 : peaks_bytes(p) + static_cast<uint64_t>(p.rows) * (sizeof(Sums) + n * sizeof(Slice));
}

}  // namespace vkml::sample
