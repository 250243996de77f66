// The checks and the batch arithmetic of csrc/pages.hpp as C functions, for
// test_pages.py.
#include "pages.hpp"

using namespace vkml::pages;

extern "C" const char* check_attend_c(const vkml_attend_pages_params* p) { return check(*p); }
extern "C" const char* check_rope_c(const vkml_rope_kv_pages_params* p) { return check(*p); }
extern "C" const char* check_copy_c(const vkml_copy_pages_params* p) { return check(*p); }
extern "C" const char* check_copies_c(uint32_t pages, uint32_t count, const int32_t* src, const int32_t* dst, uint64_t* marks) {
    return check_copies(pages, count, src, dst, marks);
}

// out [seqs, 5]: first row, rows, length, group, shared keys
extern "C" void batch_c(const Batch* b, int32_t* out) {
    for (int32_t s = 0; s < b->seqs; ++s) {
        const int32_t g = b->group_of(s);
        out[5 * s] = b->start(s);
        out[5 * s + 1] = b->count(s);
        out[5 * s + 2] = b->length(s);
        out[5 * s + 3] = g;
        out[5 * s + 4] = g < 0 ? 0 : b->group_shared(g);
    }
}
