// paged.hpp -- what PagedCache's sources share.
#pragma once

#include <cstdint>
#include <string>
#include <vector>

#include "runtime.hpp"
#include "vkml/pages.hpp"

namespace vkml::detail::paged {

// What a batch of the kernels holds at most (csrc/pages.hpp).
inline constexpr std::int64_t kMaxSeqs = 1 << 16, kMaxTokens = 1 << 22, kMaxKeys = 1 << 26, kMaxNodes = 1 << 12;

inline std::uint32_t u32(std::int64_t v) {
    if (v < 0 || v > 0xFFFFFFFFll) throw Error("PagedCache: size " + std::to_string(v) + " does not fit 32 bits");
    return static_cast<std::uint32_t>(v);
}

inline Tensor array(Runtime& runtime, Shape shape) { return TensorAccess::empty(runtime, std::move(shape), DType::I32); }

inline void upload(const Tensor& t, const std::vector<std::int32_t>& values, const char* name = "PagedCache::batch") {
    if (!values.empty()) check(vkml_memcpy_h2d(t.data(), values.data(), values.size() * sizeof(std::int32_t)), name);
}

inline const std::int32_t* ints(const Tensor& t) { return static_cast<const std::int32_t*>(t.data()); }

}  // namespace vkml::detail::paged
