// vkml::PageTable when host memory runs out: random calls, each with its first,
// second, ... allocation failing until it succeeds. A call that throws leaves
// the table as it was (a copy taken before it says the same), and a call on a
// copy of the table too, whose heap has no room to spare.
#include <cstdio>
#include <cstdlib>
#include <new>
#include <random>

#include "vkml/error.hpp"
#include "vkml/pages.hpp"

namespace {
long left = -1;  // allocations until one fails; negative: none does
}

void* operator new(std::size_t n) {
    if (left >= 0 && left-- == 0) throw std::bad_alloc();
    if (void* p = std::malloc(n ? n : 1)) return p;
    throw std::bad_alloc();
}
void operator delete(void* p) noexcept { std::free(p); }
void operator delete(void* p, std::size_t) noexcept { std::free(p); }

int main() {
    std::mt19937 gen(7);
    const auto below = [&](std::size_t n) { return static_cast<std::int64_t>(gen() % n); };
    vkml::PageTable table(40, 4);
    std::vector<std::int64_t> ids;
    int failures = 0, wrong = 0;
    const auto same = [&](const vkml::PageTable& a, const vkml::PageTable& b) {
        if (a.free_pages() != b.free_pages()) return false;
        for (const std::int64_t id : ids)
            if (a.length(id) != b.length(id) || a.row(id) != b.row(id)) return false;
        // what is free, by taking all of it
        vkml::PageTable x = a, y = b;
        const std::int64_t i = x.create(), j = y.create();
        if (i != j) return false;
        x.append(i, 4 * x.free_pages());
        y.append(j, 4 * y.free_pages());
        return x.row(i) == y.row(j);
    };
    for (int step = 0; step < 3000; ++step) {
        const std::int64_t what = below(7), id = ids.empty() ? -1 : ids[static_cast<std::size_t>(below(ids.size()))];
        std::vector<std::int64_t> some, counts;
        for (const std::int64_t i : ids)
            if (below(2)) some.push_back(i), counts.push_back(below(7));
        const std::int64_t length = id < 0 ? 0 : below(static_cast<std::size_t>(table.length(id)) + 1);
        const auto act = [&](vkml::PageTable& t) -> std::int64_t {
            if (what == 0 && ids.size() < 5) return t.create();
            if (what == 1 && id >= 0 && ids.size() < 9) return t.fork(id);
            if (what == 2 && ids.size() > 2) return t.release(id), -1;
            if (what == 3 && id >= 0) return t.truncate(id, length), -1;
            if (what == 4 && below(4) == 0) return t.compact(), -1;
            if (what > 4) return t.append(some, counts), -1;
            return -1;
        };
        const bool copied = below(3) == 0;
        for (long n = 0;; ++n) {
            const vkml::PageTable before = table;
            if (copied) table = vkml::PageTable(before);
            std::int64_t made = -1;
            bool threw = false;
            const auto state = gen;
            left = n;
            try {
                made = act(table);
            } catch (const std::bad_alloc&) {
                threw = true;
            } catch (const vkml::Error&) {
                left = -1;
                if (!same(table, before)) ++wrong;
                break;  // refused: too few pages
            }
            left = -1;
            if (!threw) {
                if (made >= 0) ids.push_back(made);
                if (what == 2 && ids.size() > 2) std::erase(ids, id);
                break;
            }
            gen = state;
            ++failures;
            if (!same(table, before) && wrong++ < 5) std::printf("step %d, call %lld, allocation %ld: the table changed\n", step, static_cast<long long>(what), n);
        }
    }
    std::printf("%s: %d failures\n", wrong ? "WRONG" : "ok", failures);
    return wrong || failures < 1000;
}
