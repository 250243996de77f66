// vkml::Tensor's release when host memory runs out, without a device: the calls of the C
// ABI that it makes are here, over host memory. A buffer that the pool has no room to
// note goes back to the device. Prints "ok" or what is wrong.
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <new>
#include <optional>

#include "vkml/tensor.hpp"
#include "vkml/context.hpp"
#include "vkml_hip.h"

namespace {
bool no_memory = false;
int held = 0;  // buffers
}  // namespace

void* operator new(std::size_t n) {
    if (no_memory) throw std::bad_alloc();
    if (void* p = std::malloc(n ? n : 1)) return p;
    throw std::bad_alloc();
}
void operator delete(void* p) noexcept { std::free(p); }
void operator delete(void* p, std::size_t) noexcept { std::free(p); }

extern "C" {
const char* vkml_last_error(void) { return "made to fail"; }
int vkml_is_initialized(void) { return 1; }
int vkml_init(const char*) { return VKML_OK; }
int vkml_shutdown(void) { return VKML_OK; }
int vkml_synchronize(void) { return VKML_OK; }
int vkml_get_device_info(vkml_device_info* info) { return *info = {}, VKML_OK; }
int vkml_set_profiling(int) { return VKML_OK; }
int vkml_get_profiling(void) { return 0; }
int vkml_profile(vkml_kernel_time*, uint32_t, uint32_t* count) { return *count = 0, VKML_OK; }
int vkml_reset_profile(void) { return VKML_OK; }
int vkml_malloc(uint64_t bytes, void** out) { return *out = std::malloc(bytes), ++held, VKML_OK; }
int vkml_free(void* p) { return std::free(p), --held, VKML_OK; }
int vkml_fill_u32(void*, uint32_t, uint64_t) { return VKML_OK; }
int vkml_memcpy_h2d(void* d, const void* h, uint64_t n) { return std::memcpy(d, h, n), VKML_OK; }
int vkml_memcpy_d2h(void* h, const void* d, uint64_t n) { return std::memcpy(h, d, n), VKML_OK; }
}

int main() {
    bool ok = true;
    const auto expect = [&](int n, const char* what) {
        if (held != n) std::printf("%s: %d buffers\n", what, held), ok = false;
    };
    {
        vkml::Context ctx;
        std::optional<vkml::Tensor> a = vkml::Tensor::empty(ctx, {100}, vkml::DType::F32), b = vkml::Tensor::empty(ctx, {100}, vkml::DType::F32);
        expect(2, "two tensors");
        no_memory = true;
        a.reset();
        no_memory = false;
        expect(1, "one released without memory");
        b.reset();
        expect(1, "one in the pool");
        const vkml::Tensor c = vkml::Tensor::empty(ctx, {100}, vkml::DType::F32), d = vkml::Tensor::empty(ctx, {100}, vkml::DType::F32);
        expect(2, "one from the pool, and a new one");
    }
    expect(0, "the end");
    std::printf("%s\n", ok ? "ok" : "WRONG");
    return !ok;
}
