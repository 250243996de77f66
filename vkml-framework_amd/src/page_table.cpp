// page_table.cpp -- the pages of a paged KV cache's sequences: taken, shared,
// copied before a write into a shared one, given back, compacted. Host code
// without a device.
#include <algorithm>
#include <functional>
#include <string>

#include "vkml/error.hpp"
#include "vkml/pages.hpp"

namespace vkml {

PageTable::PageTable(std::int64_t pages, std::int64_t page_size) : page_size_(page_size) {
    if (pages < 1 || pages > 0x7FFFFFFF) throw Error("PageTable: " + std::to_string(pages) + " pages");
    if (page_size < 1) throw Error("PageTable: pages of " + std::to_string(page_size) + " keys");
    users_.resize(static_cast<std::size_t>(pages));
    free_.resize(users_.size());
    for (std::size_t i = 0; i < free_.size(); ++i) free_[i] = static_cast<std::int32_t>(i);  // in order: a heap
}

const PageTable::Row& PageTable::at(std::int64_t id) const {
    const auto it = rows_.find(id);
    if (it == rows_.end()) throw Error("PageTable: no sequence " + std::to_string(id));
    return it->second;
}

std::int32_t PageTable::take() {
    std::pop_heap(free_.begin(), free_.end(), std::greater<>());
    const std::int32_t page = free_.back();
    free_.pop_back();
    users_[static_cast<std::size_t>(page)] = 1;
    return page;
}

void PageTable::give(std::int32_t page) {
    if (--users_[static_cast<std::size_t>(page)] != 0) return;
    free_.push_back(page);
    std::push_heap(free_.begin(), free_.end(), std::greater<>());
}

std::int64_t PageTable::create() {
    rows_.emplace(next_id_, Row{});
    return next_id_++;
}

std::int64_t PageTable::fork(std::int64_t id) {
    const auto& [to, row] = *rows_.emplace(next_id_, at(id)).first;
    for (const std::int32_t page : row.pages) ++users_[static_cast<std::size_t>(page)];
    return next_id_++, to;
}

void PageTable::release(std::int64_t id) {
    free_.reserve(users_.size());  // (a copied table's has room for its free pages alone)
    for (const std::int32_t page : at(id).pages) give(page);
    rows_.erase(id);
}

void PageTable::truncate(std::int64_t id, std::int64_t length) {
    const Row& row = at(id);
    if (length < 0 || length > row.length) {
        throw Error("PageTable::truncate: length " + std::to_string(length) + " of a sequence of " + std::to_string(row.length));
    }
    free_.reserve(users_.size());
    Row& mine = rows_.find(id)->second;
    while (static_cast<std::int64_t>(mine.pages.size()) > pages_for(length)) {
        give(mine.pages.back());
        mine.pages.pop_back();
    }
    mine.length = length;
}

std::vector<PageCopy> PageTable::append(std::span<const std::int64_t> ids, std::span<const std::int64_t> tokens) {
    if (ids.size() != tokens.size()) throw Error("PageTable::append: " + std::to_string(ids.size()) + " sequences, " + std::to_string(tokens.size()) + " counts");
    // What it takes: new pages, and copies of the part-filled ones that are
    // written into while another sequence still holds them.
    std::int64_t need = 0;
    std::map<std::int32_t, std::int32_t> writers;
    std::map<std::int64_t, int> seen;
    for (std::size_t i = 0; i < ids.size(); ++i) {
        const Row& row = at(ids[i]);
        if (tokens[i] < 0 || tokens[i] > 0x7FFFFFFF - row.length) throw Error("PageTable::append: " + std::to_string(tokens[i]) + " tokens");
        if (seen[ids[i]]++) throw Error("PageTable::append: sequence " + std::to_string(ids[i]) + " twice");
        need += pages_for(row.length + tokens[i]) - static_cast<std::int64_t>(row.pages.size());
        if (tokens[i] > 0 && row.length % page_size_ != 0) ++writers[row.pages.back()];
    }
    std::size_t most = 0;  // copies
    for (const auto& [page, n] : writers) most += static_cast<std::size_t>(n);
    for (const auto& [page, n] : writers) need += users_[static_cast<std::size_t>(page)] > n ? n : n - 1;
    if (need > free_pages()) {
        throw Error("PageTable::append: " + std::to_string(need) + " pages needed, " + std::to_string(free_pages()) + " of " + std::to_string(pages()) + " free");
    }
    // The memory that it takes, before anything changes.
    std::vector<PageCopy> copies;
    copies.reserve(most);
    for (std::size_t i = 0; i < ids.size(); ++i) {
        Row& row = rows_.find(ids[i])->second;
        const auto pages = static_cast<std::size_t>(pages_for(row.length + tokens[i]));
        if (row.pages.capacity() < pages) row.pages.reserve(std::max(pages, 2 * row.pages.size()));
    }
    for (std::size_t i = 0; i < ids.size(); ++i) {
        Row& row = rows_.find(ids[i])->second;
        if (tokens[i] > 0 && row.length % page_size_ != 0 && users_[static_cast<std::size_t>(row.pages.back())] > 1) {
            const std::int32_t page = take();
            copies.push_back({row.pages.back(), page});
            give(row.pages.back());
            row.pages.back() = page;
        }
        row.length += tokens[i];
        while (static_cast<std::int64_t>(row.pages.size()) < pages_for(row.length)) row.pages.push_back(take());
    }
    return copies;
}

void PageTable::undo(std::span<const std::int64_t> ids, std::span<const std::int64_t> tokens, std::span<const PageCopy> copies) {
    if (ids.size() != tokens.size()) throw Error("PageTable::undo: " + std::to_string(ids.size()) + " sequences, " + std::to_string(tokens.size()) + " counts");
    for (std::size_t i = 0; i < ids.size(); ++i) {
        if (tokens[i] < 0 || tokens[i] > at(ids[i]).length) throw Error("PageTable::undo: " + std::to_string(tokens[i]) + " tokens");
    }
    auto copy = copies.begin();  // in the order of the sequences
    for (std::size_t i = 0; i < ids.size(); ++i) {
        Row& row = rows_.find(ids[i])->second;
        row.length -= tokens[i];
        while (static_cast<std::int64_t>(row.pages.size()) > pages_for(row.length)) {
            give(row.pages.back());
            row.pages.pop_back();
        }
        if (tokens[i] > 0 && copy != copies.end() && !row.pages.empty() && row.pages.back() == copy->to) {
            give(copy->to);
            row.pages.back() = copy->from;
            ++users_[static_cast<std::size_t>(copy->from)];
            ++copy;
        }
    }
}

std::vector<PageCopy> PageTable::compact() {
    const std::int64_t used = pages() - free_pages();
    std::vector<std::int32_t> to(users_.size(), -1), holes;
    for (std::int64_t p = 0; p < used; ++p)
        if (users_[static_cast<std::size_t>(p)] == 0) holes.push_back(static_cast<std::int32_t>(p));
    std::vector<PageCopy> copies;
    for (std::int64_t p = used; p < pages(); ++p) {
        if (users_[static_cast<std::size_t>(p)] == 0) continue;
        const std::int32_t hole = holes[copies.size()];
        copies.push_back({static_cast<std::int32_t>(p), hole});
        to[static_cast<std::size_t>(p)] = hole;
    }
    std::vector<std::int32_t> left;
    left.reserve(users_.size());
    for (std::int64_t p = used; p < pages(); ++p) left.push_back(static_cast<std::int32_t>(p));
    for (const PageCopy& c : copies) std::swap(users_[static_cast<std::size_t>(c.from)], users_[static_cast<std::size_t>(c.to)]);
    for (auto& [id, row] : rows_)
        for (std::int32_t& page : row.pages)
            if (to[static_cast<std::size_t>(page)] >= 0) page = to[static_cast<std::size_t>(page)];
    free_ = std::move(left);
    return copies;
}

std::int64_t PageTable::shared(std::span<const std::int64_t> ids, std::span<const std::int64_t> before) const {
    if (ids.size() != before.size()) throw Error("PageTable::shared: " + std::to_string(ids.size()) + " sequences, " + std::to_string(before.size()) + " counts");
    if (ids.empty()) return 0;
    const std::vector<std::int32_t>& first = row(ids[0]);
    std::size_t same = first.size();
    std::int64_t keys = INT64_MAX;
    for (std::size_t i = 0; i < ids.size(); ++i) {
        const Row& r = at(ids[i]);
        if (before[i] < 0) throw Error("PageTable::shared: " + std::to_string(before[i]) + " keys");
        const auto end = std::mismatch(first.begin(), first.begin() + static_cast<std::ptrdiff_t>(std::min(same, r.pages.size())), r.pages.begin());
        same = static_cast<std::size_t>(end.first - first.begin());
        keys = std::min(keys, r.length - before[i]);
    }
    return std::max<std::int64_t>(0, std::min(keys, static_cast<std::int64_t>(same) * page_size_));
}

}  // namespace vkml
