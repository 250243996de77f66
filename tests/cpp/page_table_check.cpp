// Runs vkml::PageTable on commands from stdin, a line each, and answers with
// a line of numbers (a call's result), "error: ..." or, for "state", the free
// pages and every given sequence's length and pages. Host only.
#include <cstdio>
#include <iostream>
#include <sstream>
#include <string>

#include "vkml/error.hpp"
#include "vkml/pages.hpp"

int main(int argc, char** argv) {
    if (argc != 3) return 2;
    std::string line;
    try {
        vkml::PageTable table(std::atoll(argv[1]), std::atoll(argv[2]));
        while (std::getline(std::cin, line)) {
            std::istringstream in(line);
            std::string verb;
            in >> verb;
            std::vector<std::int64_t> a;
            for (std::int64_t v; in >> v;) a.push_back(v);
            try {
                std::vector<vkml::PageCopy> copies;
                std::vector<std::int64_t> ids, counts;
                for (std::size_t i = 0; i + 1 < a.size(); i += 2) {
                    ids.push_back(a[i]);
                    counts.push_back(a[i + 1]);
                }
                if (verb == "create") std::printf("%lld", static_cast<long long>(table.create()));
                if (verb == "fork") std::printf("%lld", static_cast<long long>(table.fork(a.at(0))));
                if (verb == "release") table.release(a.at(0));
                if (verb == "truncate") table.truncate(a.at(0), a.at(1));
                if (verb == "append") copies = table.append(ids, counts);
                if (verb == "compact") copies = table.compact();
                if (verb == "shared") std::printf("%lld", static_cast<long long>(table.shared(ids, counts)));
                if (verb == "state") {
                    std::printf("%lld", static_cast<long long>(table.free_pages()));
                    for (const std::int64_t id : a) {
                        std::printf(" | %lld", static_cast<long long>(table.length(id)));
                        for (const std::int32_t page : table.row(id)) std::printf(" %d", page);
                    }
                }
                for (const vkml::PageCopy& c : copies) std::printf("%d %d ", c.from, c.to);
                std::printf("\n");
            } catch (const vkml::Error& e) {
                std::printf("error: %s\n", e.what());
            }
            std::fflush(stdout);
        }
    } catch (const vkml::Error& e) {
        std::printf("error: %s\n", e.what());
    }
    return 0;
}
