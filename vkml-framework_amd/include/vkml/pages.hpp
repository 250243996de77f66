#pragma once

#include <cstdint>
#include <map>
#include <span>
#include <vector>

#include "vkml/context.hpp"
#include "vkml/ops.hpp"
#include "vkml/tensor.hpp"

// Several sequences over one paged KV cache. The reference keeps one sequence
// in contiguous caches (include/vkml/llama.hpp:199-209 there) and has no
// counterpart.
namespace vkml {

// Page `from`'s contents go to page `to`, in every layer.
struct PageCopy {
    std::int32_t from, to;
    bool operator==(const PageCopy&) const = default;
};

// Which pages of a pool hold which sequence's keys (host only): key p of a
// sequence is row p % page_size of its page p / page_size. Sequences that were
// forked share pages; one that writes into a shared page gets a copy first.
// What throws (vkml::Error, or std::bad_alloc) changes nothing.
class PageTable {
public:
    PageTable(std::int64_t pages, std::int64_t page_size);

    std::int64_t create();                  // a new, empty sequence
    std::int64_t fork(std::int64_t id);     // a new sequence with the same keys, in the same pages
    void release(std::int64_t id);          // its pages go back, those that others share excepted
    void truncate(std::int64_t id, std::int64_t length);

    // Room for tokens[i] more keys of sequence ids[i] (each id once). The
    // copies are to be made before those keys are written.
    std::vector<PageCopy> append(std::span<const std::int64_t> ids, std::span<const std::int64_t> tokens);
    std::vector<PageCopy> append(std::int64_t id, std::int64_t tokens) { return append(std::span(&id, 1), std::span(&tokens, 1)); }
    // Takes back the append that returned `copies`, where they or the keys could
    // not be written; no other call may have changed the table since.
    void undo(std::span<const std::int64_t> ids, std::span<const std::int64_t> tokens, std::span<const PageCopy> copies);

    // The pages in use become the lowest ones: the rows change, and the copies
    // are to be made before anything is read or written through them.
    std::vector<PageCopy> compact();

    // Keys that all of these sequences hold in the same pages, none of them
    // among a sequence's last before[i].
    std::int64_t shared(std::span<const std::int64_t> ids, std::span<const std::int64_t> before) const;

    std::int64_t length(std::int64_t id) const { return at(id).length; }
    const std::vector<std::int32_t>& row(std::int64_t id) const { return at(id).pages; }
    std::int64_t pages() const noexcept { return static_cast<std::int64_t>(users_.size()); }
    std::int64_t page_size() const noexcept { return page_size_; }
    std::int64_t free_pages() const noexcept { return static_cast<std::int64_t>(free_.size()); }

private:
    struct Row {
        std::vector<std::int32_t> pages;
        std::int64_t length = 0;
    };
    const Row& at(std::int64_t id) const;
    std::int64_t pages_for(std::int64_t length) const { return (length + page_size_ - 1) / page_size_; }
    std::int32_t take();
    void give(std::int32_t page);

    std::int64_t page_size_;
    std::int64_t next_id_ = 0;
    std::vector<std::int32_t> users_;  // sequences that hold each page
    std::vector<std::int32_t> free_;   // a heap, the lowest first
    std::map<std::int64_t, Row> rows_;
};

// A step's sequences as the kernels read them, good until the table changes.
struct PagedBatch {
    Tensor table, lengths, starts;     // i32 [seqs, stride], [seqs], [seqs + 1]
    Tensor group_starts, group_keys;   // i32 [groups + 1], [groups]; null without groups
    std::int64_t seqs = 0, tokens = 0, groups = 0;
    std::int64_t positions = 0;        // past the last position of a new token
};

// The keys and values of several sequences, in up to 2^24 pages of `page_size`
// (a power of two, 16 to 1024) and 2^30 bytes, f32 or f16, for every layer of a
// model (up to 65535), of up to 4096 KV heads of up to 1024 dims. What
// throws changes nothing: a batch that is refused, or for which there is no
// memory, leaves every sequence with the keys that it had.
class PagedCache {
public:
    PagedCache(Context& context, std::int64_t layers, std::int64_t kv_heads, std::int64_t head_dim, std::int64_t pages, std::int64_t page_size,
               DType dtype);
    // (a copy would have the same pools under a table of its own)
    PagedCache(const PagedCache&) = delete;
    PagedCache& operator=(const PagedCache&) = delete;
    PagedCache(PagedCache&&) = default;
    PagedCache& operator=(PagedCache&&) = default;

    std::int64_t create() { return table_.create(); }
    std::int64_t fork(std::int64_t id) { return table_.fork(id); }
    void release(std::int64_t id) { table_.release(id); }
    void truncate(std::int64_t id, std::int64_t length) { table_.truncate(id, length); }
    void compact();
    const PageTable& table() const noexcept { return table_; }

    // A step in which sequence ids[i] gets tokens[i] new keys: makes room for
    // them and uploads what the step's calls read. group_sizes: so many
    // neighbours in ids read the keys that they share once, from the first on
    // (sequences past the last group each read their own). At most 65536
    // sequences, 2^22 new tokens and 2^26 keys a sequence. The new keys count
    // from here on: where a step is given up before its appends, truncate.
    PagedBatch batch(std::span<const std::int64_t> ids, std::span<const std::int64_t> tokens, std::span<const std::int64_t> group_sizes = {});

    // The new tokens' q | k | v, f32 [tokens, (heads + 2 kv_heads) * head_dim],
    // sequence after sequence: q and k rotated at their positions by a table
    // from rope_table (for a part of the head: of that many dims; null: not
    // rotated) that holds them all, k and v into a layer's pages. Returns q
    // [tokens, heads, head_dim].
    Tensor append(std::int64_t layer, const PagedBatch& batch, const Tensor& qkv, const Tensor& rope_table, RopeStyle style);

    // softmax(q k^T / sqrt(head_dim)) v of each new token over its sequence's
    // keys up to its own; q and the result [tokens, heads, head_dim].
    // head_dim 64 or 128.
    Tensor attention(std::int64_t layer, const PagedBatch& batch, const Tensor& q, float softcap = 0.0f) const;

    const Tensor& k_pages() const noexcept { return k_; }  // [layers, pages, kv_heads, page_size, head_dim]
    const Tensor& v_pages() const noexcept { return v_; }

private:
    void copy(const std::vector<PageCopy>& copies);
    void* pool(const Tensor& pools, std::int64_t layer) const;

    std::int64_t layers_, kv_heads_, head_dim_;
    PageTable table_;
    Tensor k_, v_;
};

}  // namespace vkml
