// vkml::PagedCache's drafts without a device: the calls of the C ABI that it makes are
// here, over host memory, and the n-th of them, or of the host's allocations, fails on
// demand.
// Usage: drafts_host_check PART. Prints a line a check ("ok" or what is wrong).
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <new>
#include <string>
#include <vector>

#include "vkml/pages.hpp"
#include "vkml_hip.h"

namespace {

long calls_left = -1, memory_left = -1;  // until one fails; negative: none does
bool fails(long& left) { return left >= 0 && left-- == 0; }

}  // namespace

void* operator new(std::size_t n) {
    if (fails(memory_left)) throw std::bad_alloc();
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
int vkml_malloc(uint64_t bytes, void** out) {
    if (fails(calls_left)) return VKML_ERROR_OUT_OF_MEMORY;
    *out = std::malloc(bytes);
    return VKML_OK;
}
int vkml_free(void* p) { return std::free(p), VKML_OK; }
int vkml_fill_u32(void* d, uint32_t v, uint64_t words) {
    for (uint64_t i = 0; i < words; ++i) static_cast<uint32_t*>(d)[i] = v;
    return VKML_OK;
}
int vkml_memcpy_h2d(void* d, const void* h, uint64_t n) { return std::memcpy(d, h, n), VKML_OK; }
int vkml_memcpy_d2h(void* h, const void* d, uint64_t n) {
    if (fails(calls_left)) return VKML_ERROR_DEVICE;
    return std::memcpy(h, d, n), VKML_OK;
}
int vkml_copy_pages(const vkml_copy_pages_params* p, const int32_t* src, const int32_t* dst, void* k, void* v) {
    for (uint32_t layer = 0; layer < p->layers; ++layer)
        for (uint32_t i = 0; i < p->count; ++i)
            for (void* pool : {k, v}) {
                char* base = static_cast<char*>(pool) + layer * p->pages * p->page_bytes;
                std::memcpy(base + dst[i] * p->page_bytes, base + src[i] * p->page_bytes, p->page_bytes);
            }
    return VKML_OK;
}
int vkml_rope_kv_pages(const vkml_rope_kv_pages_params*, const float*, const float*, const int32_t*, const int32_t*, const int32_t*, const int32_t*, float*, void*,
                       void*) {
    return VKML_OK;
}
uint64_t vkml_attend_pages_workspace_bytes(const vkml_attend_pages_params*) { return 64; }
int vkml_attend_pages(const vkml_attend_pages_params*, const float*, const void*, const void*, const int32_t*, const int32_t*, const int32_t*, const int32_t*,
                      const int32_t*, void*, float*) {
    return VKML_OK;
}
int vkml_attend_pages_tree(const vkml_attend_pages_params*, uint32_t, const float*, const void*, const void*, const int32_t*, const int32_t*, const int32_t*,
                           const int32_t*, const int32_t*, const uint32_t*, void*, float*) {
    return VKML_OK;
}
int vkml_attend_pages_window(const vkml_attend_pages_params*, uint32_t, uint32_t, const float*, const void*, const void*, const int32_t*, const int32_t*,
                             const int32_t*, void*, float*) {
    return VKML_OK;
}
// (one layer of keys of one head; row by row in the path's order)
int vkml_keep_drafts(const vkml_keep_drafts_params* p, const int32_t* parents, const int32_t* drafted, const int32_t* picked, const int32_t* table,
                     const int32_t* lengths, const int32_t* starts, int32_t* path, int32_t* counts, int32_t* next, void* k, void* v) {
    if (fails(calls_left)) return VKML_ERROR_DEVICE;
    const uint64_t bytes = p->head_dim * 4;
    for (uint32_t s = 0; s < p->seqs; ++s) {
        const int32_t first = starts[s], n = starts[s + 1] - first, base = lengths[s] - n;
        int32_t at = -1, count = 0;
        const auto row = [&](void* pool, int32_t pos) {
            return static_cast<char*>(pool) + (static_cast<uint64_t>(table[s * p->table_stride + static_cast<uint32_t>(pos) / p->page_size]) * p->page_size + static_cast<uint32_t>(pos) % p->page_size) * bytes;
        };
        for (int32_t i = 0; i < n; ++i) path[first + i] = -1;
        for (int32_t i = 0; i < n; ++i) {
            if (i > 0 && (parents[first + i] != at || drafted[first + i] != picked[first + at])) continue;
            for (void* pool : {k, v}) std::memmove(row(pool, base + count), row(pool, base + i), bytes);
            path[first + count++] = at = i;
        }
        counts[s] = count;
        next[s] = n > 0 ? picked[first + at] : -1;
    }
    return VKML_OK;
}
}

namespace {

using Ids = std::vector<std::int64_t>;
using Ints = std::vector<std::int32_t>;
using vkml::DType;
using vkml::Tensor;
constexpr std::int64_t kPages = 40, kPage = 16;

int wrong = 0;
void expect(bool ok, const std::string& what) {
    if (!ok && wrong++ < 10) std::printf("%s\n", what.c_str());
}
void throws(const char* why, const char* what, const std::function<void()>& f) {
    try {
        f();
    } catch (const vkml::Error& e) {
        expect(std::string(e.what()).find(why) != std::string::npos, std::string(what) + ": \"" + e.what() + "\" for \"" + why + "\"");
        return;
    }
    expect(false, std::string(what) + ": not refused: " + why);
}

// A cache of one layer, with keys of one head of two dims.
struct Cache {
    vkml::Context ctx;
    vkml::PagedCache c{ctx, 1, 1, 2, kPages, kPage, DType::F32};

    Tensor ints(const Ints& x) { return Tensor::from_data<std::int32_t>(ctx, x, {static_cast<std::int64_t>(x.size())}); }
    Tensor qkv(const vkml::PagedBatch& b) { return Tensor::zeros(ctx, {b.tokens, 6}, DType::F32); }
    Tensor q(const vkml::PagedBatch& b) { return Tensor::zeros(ctx, {b.tokens, 1, 2}, DType::F32); }
};

void trees() {
    Cache x;
    vkml::PagedCache& c = x.c;
    const std::int64_t a = c.create(), b = c.create();
    c.batch(Ids{a, b}, Ids{10, 3});
    const Ints parents = {-1, 0, 0, -1, 0, 1};
    const vkml::PagedBatch first = c.batch(Ids{a, b}, Ids{3, 3});
    const vkml::PagedTrees of_first = c.trees(first, parents);
    const Tensor none, drafted = x.ints({5, 6, 7, 8, 9, 4}), picked = x.ints({6, 0, 0, 9, 4, 1});
    const auto refused = [&](const char* what, const vkml::PagedBatch& batch) {
        const std::int64_t la = c.table().length(a), lb = c.table().length(b);
        throws("another batch", what, [&] { c.append(0, batch, x.qkv(batch), none, vkml::RopeStyle::Interleaved, &of_first); });
        throws("another batch", what, [&] { c.attention_tree(0, batch, of_first, x.q(batch)); });
        throws("another batch", what, [&] { c.keep(batch, of_first, drafted, picked); });
        expect(c.table().length(a) == la && c.table().length(b) == lb, std::string(what) + ": a refused call changed a sequence");
    };
    const auto back = [&] { c.truncate(a, 10), c.truncate(b, 3); };
    back();
    refused("the sequences in another order", c.batch(Ids{b, a}, Ids{3, 3}));
    back();
    refused("as many new tokens in all, not of each", c.batch(Ids{a, b}, Ids{2, 4}));
    back();
    refused("one sequence of as many", c.batch(Ids{a}, Ids{6}));
    back();
    refused("a third, without tokens", c.batch(Ids{a, b, c.create()}, Ids{3, 3, 0}));
    back();
    c.batch(Ids{a}, Ids{1});
    refused("the next step's", c.batch(Ids{a, b}, Ids{3, 3}));
    // What the trees say is as true of a batch of as many earlier keys and new tokens.
    back();
    const vkml::PagedBatch again = c.batch(Ids{a, b}, Ids{3, 3});
    c.append(0, again, x.qkv(again), none, vkml::RopeStyle::Interleaved, &of_first);
    c.attention_tree(0, again, of_first, x.q(again));
    const vkml::KeptDrafts kept = c.keep(again, of_first, drafted, picked);
    expect(kept.paths == std::vector<Ints>{{0, 1}, {0, 1, 2}} && kept.next == Ints{0, 1}, "another path");
    expect(c.table().length(a) == 12 && c.table().length(b) == 6, "another length");
}

// A sequence that was cut and has as many keys again, in the same pages, holds others
// than the batch's.
void stale() {
    Cache x;
    vkml::PagedCache& c = x.c;
    const std::int64_t a = c.create(), b = c.create();
    c.batch(Ids{a, b}, Ids{10, 3});
    const Tensor drafted = x.ints({5, 6, 7}), others = x.ints({4, 4, 4}), all = x.ints({6, 7, 0});
    const Ints parents = {-1, 0, 1};
    const auto refused = [&](const char* what, const vkml::PagedBatch& batch, const vkml::PagedTrees& trees) {
        const std::int64_t length = c.table().length(a);
        throws("not as the batch left it", what, [&] { c.keep(batch, trees, drafted, all); });
        expect(c.table().length(a) == length, std::string(what) + ": a refused call changed a sequence");
    };
    const vkml::PagedBatch first = c.batch(Ids{a}, Ids{3});
    const vkml::PagedTrees trees = c.trees(first, parents);
    c.keep(first, trees, drafted, others);  // one stays
    const vkml::PagedBatch second = c.batch(Ids{a}, Ids{2});
    expect(c.table().length(a) == 13, "the test's own lengths");
    refused("kept, and grown to as many", first, trees);
    c.truncate(a, 10);
    refused("cut", first, trees);
    const vkml::PagedBatch third = c.batch(Ids{a}, Ids{3});
    refused("cut, and grown to as many", first, trees);
    throws("not as the batch left it", "cut, and grown past", [&] { c.keep(second, c.trees(second, Ints{-1, 0}), x.ints({7, 4}), x.ints({0, 0})); });
    // What leaves a sequence's keys as they are does not matter.
    c.release(c.fork(a));
    c.batch(Ids{b, a}, Ids{20, 0});
    c.truncate(a, 13);
    c.truncate(b, 1);
    try {
        c.batch(Ids{a}, Ids{kPages * kPage});
    } catch (const vkml::Error&) {
    }
    expect(c.keep(third, trees, drafted, all).paths == std::vector<Ints>{{0, 1, 2}}, "another path");
}

// Three sequences, the third without new tokens, and a step of drafts for them that is
// kept after `fail`, which has the n-th call or allocation from there on fail. Whether
// that was reached. However it ends, no sequence has a key that it had not: all are as
// the batch left them, and keep then does what it should, or (where the device failed)
// they end at their earlier keys.
bool keeps_or_not(const char* what, long n, bool on_device, const std::function<void(long)>& fail, bool& ended) {
    Cache x;
    vkml::PagedCache& c = x.c;
    const Ids ids = {c.create(), c.create(), c.create()};
    float next = 1;
    const auto at = [&](std::int64_t id, std::int64_t p) -> float& {
        return static_cast<float*>(c.k_pages().data())[(c.table().row(id)[static_cast<std::size_t>(p / kPage)] * kPage + p % kPage) * 2];
    };
    const auto keys = [&](std::int64_t id) {
        std::vector<float> k;
        for (std::int64_t p = 0; p < c.table().length(id); ++p) k.push_back(at(id, p));
        return k;
    };
    const Ids held = {14, 3, 5}, added = {40, 3, 0};
    for (std::size_t i = 0; i < 3; ++i) {
        c.batch(Ids{ids[i]}, Ids{held[i]});
        for (std::int64_t p = 0; p < held[i]; ++p) at(ids[i], p) = next++;
    }
    c.release(c.fork(ids[0]));
    const vkml::PagedBatch b = c.batch(ids, added);
    Ints parents, drafted(43), picked(43);
    for (std::size_t i = 0; i < 2; ++i)
        for (std::int64_t t = 0; t < added[i]; ++t) {
            parents.push_back(static_cast<std::int32_t>(t == 0 ? -1 : t < 3 ? 0 : t - 2));  // chains of the odd and of the even ones
            at(ids[i], held[i] + t) = next++;
        }
    for (std::size_t t = 0; t < 43; ++t) drafted[t] = static_cast<std::int32_t>(t);
    for (std::size_t t = 0; t < 40; ++t) picked[t] = static_cast<std::int32_t>(t + 2 < 32 ? t + 2 : 99);  // the even ones, 0 to 30
    picked[40] = 41;
    const vkml::PagedTrees trees = c.trees(b, parents);
    const Tensor d = x.ints(drafted), p = x.ints(picked);
    const std::vector<std::vector<float>> before = {keys(ids[0]), keys(ids[1]), keys(ids[2])};
    std::vector<std::vector<float>> after = {before[0], before[1], before[2]};
    for (std::size_t k = 1; k < 16; ++k) after[0][14 + k] = before[0][14 + 2 * k];
    after[0].resize(30);
    after[1].resize(5);
    const std::string text = std::string(what) + ", failure " + std::to_string(n);
    bool threw = false;
    vkml::KeptDrafts kept;
    fail(n);
    try {
        kept = c.keep(b, trees, d, p);
    } catch (const std::exception&) {
        threw = true;
    }
    const bool reached = calls_left < 0 && memory_left < 0;
    fail(-1);
    expect(!threw || reached, text + ": threw without a failure");  // (the pool lives with some)
    if (threw) {
        bool as_left = true, as_held = true;
        for (std::size_t i = 0; i < 3; ++i) {
            std::vector<float> earlier = before[i];
            earlier.resize(static_cast<std::size_t>(held[i]));
            as_left &= keys(ids[i]) == before[i];
            as_held &= keys(ids[i]) == earlier;
        }
        expect(as_left || (on_device && as_held), text + ": the sequences are not as they were");
        ended |= !as_left;
        if (!as_left) return reached;
        kept = c.keep(b, trees, d, p);
    }
    for (std::size_t i = 0; i < 3; ++i) expect(keys(ids[i]) == after[i], text + ": other keys are kept");
    Ints even;
    for (std::int32_t k = 0; k < 16; ++k) even.push_back(2 * k);
    expect(kept.paths == std::vector<Ints>{even, {0, 1}, {}} && kept.next == Ints{99, 0, -1}, text + ": another path");
    return reached;
}

void failures() {
    bool ended = false;
    long n = 0;
    while (keeps_or_not("host memory", n, false, [](long left) { memory_left = left; }, ended)) ++n;
    expect(n >= 10, "fewer allocations than expected");
    n = 0;
    while (keeps_or_not("a call", n, true, [](long left) { calls_left = left; }, ended)) ++n;
    expect(n >= 4 && ended, "fewer calls than expected");
}

}  // namespace

int main(int argc, char** argv) {
    const std::string part = argc == 2 ? argv[1] : "";
    if (part == "trees") trees();
    else if (part == "stale") stale();
    else if (part == "failures") failures();
    else return 2;
    std::printf("%s %s\n", wrong ? "WRONG" : "ok", part.c_str());
    return wrong != 0;
}
