// vkml::PagedCache without a device: the calls of the C ABI that it makes are
// here, over host memory, and the n-th of them fails on demand. After every
// failure the sequences have the lengths, pages and keys that they had, and the
// same step then succeeds.
// Prints a line a check ("ok" or what is wrong).
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <map>
#include <string>
#include <type_traits>
#include <vector>

#include "vkml/pages.hpp"
#include "vkml_hip.h"

namespace {

long calls_left = -1;  // until one fails; negative: none does

bool fails(long& left) { return left >= 0 && left-- == 0; }

}  // namespace

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
int vkml_memcpy_h2d(void* d, const void* h, uint64_t n) {
    if (fails(calls_left)) return VKML_ERROR_OUT_OF_MEMORY;
    return std::memcpy(d, h, n), VKML_OK;
}
int vkml_memcpy_d2h(void* h, const void* d, uint64_t n) { return std::memcpy(h, d, n), VKML_OK; }
int vkml_copy_pages(const vkml_copy_pages_params* p, const int32_t* src, const int32_t* dst, void* k, void* v) {
    if (fails(calls_left)) return VKML_ERROR_OUT_OF_MEMORY;
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
    return fails(calls_left) ? VKML_ERROR_OUT_OF_MEMORY : VKML_OK;
}
uint64_t vkml_attend_pages_workspace_bytes(const vkml_attend_pages_params*) { return 64; }
int vkml_attend_pages(const vkml_attend_pages_params*, const float*, const void*, const void*, const int32_t*, const int32_t*, const int32_t*, const int32_t*,
                      const int32_t*, void*, float*) {
    return fails(calls_left) ? VKML_ERROR_OUT_OF_MEMORY : VKML_OK;
}
}

namespace {

static_assert(!std::is_copy_constructible_v<vkml::PagedCache> && !std::is_copy_assignable_v<vkml::PagedCache>);  // one table for its pools
static_assert(std::is_move_constructible_v<vkml::PagedCache> && std::is_move_assignable_v<vkml::PagedCache>);

using Ids = std::vector<std::int64_t>;
constexpr std::int64_t kPages = 40, kPage = 16;

// What a table holds, and in a cache each key's first element (a key is one KV
// head of two f32 dims here).
struct Seen {
    std::map<std::int64_t, std::pair<std::int64_t, std::vector<std::int32_t>>> rows;
    std::map<std::int64_t, std::vector<float>> keys;
    std::int64_t free = 0;
    bool operator==(const Seen&) const = default;
};
Seen look(const vkml::PageTable& t, const Ids& ids, const vkml::PagedCache* cache) {
    Seen s;
    s.free = t.free_pages();
    for (const std::int64_t id : ids) {
        s.rows[id] = {t.length(id), t.row(id)};
        for (std::int64_t p = 0; cache && p < t.length(id); ++p)
            s.keys[id].push_back(static_cast<const float*>(cache->k_pages().data())[(t.row(id)[static_cast<std::size_t>(p / kPage)] * kPage + p % kPage) * 2]);
    }
    return s;
}

int wrong = 0;
void expect(bool ok, const std::string& what) {
    if (!ok && wrong++ < 10) std::printf("%s\n", what.c_str());
}

// The action, with every n-th call (or allocation) of it failing; then without.
// Whenever it throws, the table is as it was. Returns how many failures there
// were.
int every_failure(const char* what, long& left, const vkml::PageTable& table, const Ids& ids, const vkml::PagedCache* cache, const std::function<void()>& act) {
    for (int n = 0;; ++n) {
        const Seen before = look(table, ids, cache);
        const std::string text = std::string(what) + ", failure " + std::to_string(n);
        bool threw = false;
        left = n;
        try {
            act();
        } catch (const std::exception&) {
            threw = true;
        }
        const bool reached = left < 0;
        left = -1;
        expect(threw == reached, text + (threw ? ": threw without a failure" : ": failed without an error"));
        if (!reached || !threw) return n;
        expect(look(table, ids, cache) == before, text + ": the table or its keys changed");
    }
}

void say(const char* what, int failures, int least) {
    std::printf("%s %s: %d failures\n", wrong == 0 && failures >= least ? "ok" : "WRONG", what, failures);
    if (failures < least) ++wrong;
}

// The new keys' numbers, so that sequences can be told apart.
void write(vkml::PagedCache& c, std::int64_t id, std::int64_t n, float first) {
    const auto& t = c.table();
    for (std::int64_t p = t.length(id) - n; p < t.length(id); ++p)
        static_cast<float*>(c.k_pages().data())[(t.row(id)[static_cast<std::size_t>(p / kPage)] * kPage + p % kPage) * 2] = first + static_cast<float>(p);
}

void batches() {
    vkml::Context ctx;
    vkml::PagedCache c(ctx, 1, 1, 2, kPages, kPage, vkml::DType::F32);
    const std::int64_t a = c.create();
    std::vector<vkml::PagedBatch> kept = {c.batch(Ids{a}, Ids{37})};  // so that the pool has nothing to hand out
    write(c, a, 37, 100);
    const std::int64_t b = c.fork(a), d = c.fork(a), e = c.create();
    const Ids ids = {a, b, d, e};
    const Ids counts = {1, 30, 2, 17}, groups = {3};
    // A part-filled page that all three hold: two copies, and new pages.
    const int n = every_failure("a batch", calls_left, c.table(), ids, &c, [&] { kept.push_back(c.batch(ids, counts, groups)); });
    for (std::size_t i = 0; i < 4; ++i) c.truncate(ids[i], i < 3 ? 37 : 0);
    say("a batch that fails", n, 6);  // five uploads and the copies
    c.batch(ids, counts, groups);
    for (const std::int64_t id : {a, b, d}) {
        const Seen s = look(c.table(), ids, &c);
        for (std::int64_t p = 0; p < 37; ++p) expect(s.keys.at(id)[static_cast<std::size_t>(p)] == 100 + static_cast<float>(p), "a key of the prompt is lost");
    }
    expect(c.table().row(a).back() != c.table().row(b)[2] && c.table().row(b)[2] != c.table().row(d)[2], "writers share a page");
    write(c, b, 30, 500);
    c.release(a);
    c.release(e);
    const Ids left = {b, d};
    const auto keys = [&] { return look(c.table(), left, &c).keys; };
    const auto before = keys();
    // Move the sequences up: forks that come and go leave holes.
    const std::int64_t hole = c.create();
    c.batch(Ids{hole}, Ids{100});
    c.batch(left, Ids{20, 40});
    c.truncate(b, 67), c.truncate(d, 39);
    c.batch(left, Ids{100, 60});
    c.release(hole);
    const int m = every_failure("a compaction", calls_left, c.table(), left, &c, [&] { c.compact(); });
    say("a compaction that fails", m, 1);
    for (const std::int64_t id : left) {
        std::vector<float> now = keys().at(id);
        now.resize(before.at(id).size());
        expect(now == before.at(id), "a key is lost in the compaction");
    }
    std::printf("%s keys\n", wrong ? "WRONG" : "ok");
}

void limits() {
    vkml::Context ctx;
    vkml::PagedCache c(ctx, 1, 1, 2, kPages, kPage, vkml::DType::F32);
    Ids ids, one;
    for (int i = 0; i < (1 << 16) + 1; ++i) {
        ids.push_back(c.create());
        one.push_back(0);
    }
    const auto refused = [&](const char* why, const Ids& i, const Ids& n) {
        const Seen before = look(c.table(), Ids(ids.begin(), ids.begin() + 4), &c);
        try {
            c.batch(i, n);
            expect(false, std::string("not refused: ") + why);
        } catch (const vkml::Error& e) {
            expect(std::string(e.what()).find(why) != std::string::npos, e.what());
        }
        expect(look(c.table(), Ids(ids.begin(), ids.begin() + 4), &c) == before, std::string(why) + ": the table changed");
    };
    refused("65536 sequences", ids, one);
    refused("2^22 new tokens", {ids[0], ids[1]}, {1 << 21, (1 << 21) + 1});
    refused("2^26 keys", {ids[0], ids[1]}, {1, (1 << 26) + 1});
    refused("-1 tokens", {ids[0], ids[1]}, {1, -1});
    refused("twice", {ids[0], ids[0]}, {1, 1});
    refused("no sequence", {ids[0], 1 << 20}, {1, 1});
    refused("pages needed", {ids[0], ids[1]}, {1, kPages * kPage});
    refused("counts", {ids[0], ids[1]}, {1});
    std::printf("%s limits\n", wrong ? "WRONG" : "ok");
}

void construction() {
    vkml::Context ctx;
    const auto refused = [&](const char* why, std::int64_t layers, std::int64_t kv_heads, std::int64_t head_dim, std::int64_t pages, std::int64_t page) {
        try {
            vkml::PagedCache c(ctx, layers, kv_heads, head_dim, pages, page, vkml::DType::F32);
            expect(false, std::string("not refused: ") + why);
        } catch (const vkml::Error& e) {
            expect(std::string(e.what()).find(why) != std::string::npos, e.what());
        }
    };
    refused("65535 layers", 65536, 1, 2, 4, 16);
    refused("2^24 pages", 1, 1, 2, (1 << 24) + 1, 16);
    refused("KV heads", 1, 4097, 2, 4, 16);
    refused("KV heads", 1, 1, 1026, 4, 16);
    refused("KV heads", 1, 1, 3, 4, 16);
    refused("2^30 bytes", 1, 4096, 1024, 4, 128);
    refused("2^62 bytes", 1 << 14, 512, 512, 1 << 24, 1024);  // 2^68 in all: 0 in 64 bits
    refused("0 pages", 1, 1, 2, 0, 16);
    vkml::PagedCache(ctx, 65535, 1, 2, 1, 16, vkml::DType::F16);
    std::printf("%s construction\n", wrong ? "WRONG" : "ok");
}

void tables() {
    vkml::Context ctx;
    vkml::PagedCache c(ctx, 1, 1, 2, kPages, kPage, vkml::DType::F32);
    const std::int64_t a = c.create(), b = c.create();
    const vkml::PagedBatch first = c.batch(Ids{a, b}, Ids{40, 7}), idle = c.batch(Ids{a, b}, Ids{0, 1});
    const auto takes = [&](const vkml::PagedBatch& batch, const vkml::Tensor& table) {
        try {
            c.append(0, batch, vkml::Tensor::empty(ctx, {batch.tokens, 6}, vkml::DType::F32), table, vkml::RopeStyle::Interleaved);
        } catch (const vkml::Error& e) {
            expect(std::string(e.what()).find("positions") != std::string::npos, e.what());
            return false;
        }
        return true;
    };
    const auto rows = [&](std::int64_t n) { return vkml::Tensor::empty(ctx, {n, 1, 2}, vkml::DType::F32); };
    expect(takes(first, rows(40)) && takes(first, vkml::Tensor()), "a table that holds every position is refused");
    expect(!takes(first, rows(39)) && !takes(first, rows(0)), "a table that is too short is taken");
    expect(takes(idle, rows(8)) && !takes(idle, rows(7)), "positions of a sequence without new tokens count");
    std::printf("%s tables\n", wrong ? "WRONG" : "ok");
}

}  // namespace

int main() {
    tables();
    construction();
    batches();
    limits();
    return wrong ? 1 : 0;
}
