// pages.cpp -- vkml::PagedCache over the C ABI (vkml_rope_kv_pages,
// vkml_attend_pages, vkml_copy_pages).
#include <algorithm>
#include <cmath>
#include <string>

#include "runtime.hpp"
#include "vkml/pages.hpp"

namespace vkml {

using detail::check;
using detail::TensorAccess;

namespace {

std::uint32_t u32(std::int64_t v) {
    if (v < 0 || v > 0xFFFFFFFFll) throw Error("PagedCache: size " + std::to_string(v) + " does not fit 32 bits");
    return static_cast<std::uint32_t>(v);
}

std::int64_t positive(std::int64_t v, const char* what) {
    if (v < 1) throw Error("PagedCache: " + std::to_string(v) + " " + what);
    return v;
}

// What a batch of the kernels holds at most (csrc/pages.hpp).
constexpr std::int64_t kMaxSeqs = 1 << 16, kMaxTokens = 1 << 22, kMaxKeys = 1 << 26;

// The table of a cache whose every call the kernels take (csrc/pages.hpp), and
// whose pools' bytes can be counted.
PageTable table_of(std::int64_t layers, std::int64_t kv_heads, std::int64_t head_dim, std::int64_t pages, std::int64_t page_size, DType dtype) {
    if (dtype != DType::F32 && dtype != DType::F16) throw Error("PagedCache: no kernel for " + std::string(to_string(dtype)) + " yet");
    if (page_size < 16 || page_size > 1024 || (page_size & (page_size - 1)) != 0) {
        throw Error("PagedCache: page_size must be a power of two from 16 to 1024, got " + std::to_string(page_size));
    }
    if (pages > std::int64_t{1} << 24) throw Error("PagedCache: more than 2^24 pages");
    if (layers > 65535) throw Error("PagedCache: more than 65535 layers");
    if (kv_heads > 4096 || head_dim > 1024 || head_dim % 2 != 0) {
        throw Error("PagedCache: at most 4096 KV heads of an even number of dims up to 1024, got " + std::to_string(kv_heads) + " of " + std::to_string(head_dim));
    }
    const std::int64_t page_bytes = kv_heads * page_size * head_dim * static_cast<std::int64_t>(element_size(dtype));
    if (page_bytes > std::int64_t{1} << 30) throw Error("PagedCache: a page of more than 2^30 bytes");
    if (page_bytes > (std::int64_t{1} << 62) / layers / std::max<std::int64_t>(pages, 1)) throw Error("PagedCache: pools of more than 2^62 bytes");
    return PageTable(pages, page_size);
}

Tensor array(detail::Runtime& runtime, Shape shape) { return TensorAccess::empty(runtime, std::move(shape), DType::I32); }

void upload(const Tensor& t, const std::vector<std::int32_t>& values) {
    if (!values.empty()) check(vkml_memcpy_h2d(t.data(), values.data(), values.size() * sizeof(std::int32_t)), "PagedCache::batch");
}

const std::int32_t* ints(const Tensor& t) { return static_cast<const std::int32_t*>(t.data()); }

}  // namespace

PagedCache::PagedCache(Context& context, std::int64_t layers, std::int64_t kv_heads, std::int64_t head_dim, std::int64_t pages, std::int64_t page_size,
                       DType dtype)
    : layers_(positive(layers, "layers")), kv_heads_(positive(kv_heads, "KV heads")), head_dim_(positive(head_dim, "dims a head")),
      table_(table_of(layers, kv_heads, head_dim, pages, page_size, dtype)) {
    const Shape shape = {layers, pages, kv_heads, page_size, head_dim};
    k_ = Tensor::empty(context, shape, dtype);
    v_ = Tensor::empty(context, shape, dtype);
}

void* PagedCache::pool(const Tensor& pools, std::int64_t layer) const {
    if (layer < 0 || layer >= layers_) throw Error("PagedCache: no layer " + std::to_string(layer) + " of " + std::to_string(layers_));
    return static_cast<std::byte*>(pools.data()) + static_cast<std::uint64_t>(layer) * (pools.nbytes() / static_cast<std::uint64_t>(layers_));
}

void PagedCache::copy(const std::vector<PageCopy>& copies) {
    if (copies.empty()) return;
    std::vector<std::int32_t> from, to;
    for (const PageCopy& c : copies) {
        from.push_back(c.from);
        to.push_back(c.to);
    }
    vkml_copy_pages_params p{};
    p.pages = u32(table_.pages());
    p.layers = u32(layers_);
    p.count = u32(static_cast<std::int64_t>(copies.size()));
    p.page_bytes = k_.nbytes() / static_cast<std::uint64_t>(layers_ * table_.pages());
    check(vkml_copy_pages(&p, from.data(), to.data(), k_.data(), v_.data()), "PagedCache");
}

void PagedCache::compact() {
    PageTable compacted = table_;
    copy(compacted.compact());
    table_ = std::move(compacted);
}

PagedBatch PagedCache::batch(std::span<const std::int64_t> ids, std::span<const std::int64_t> tokens, std::span<const std::int64_t> group_sizes) {
    if (ids.size() != tokens.size()) throw Error("PagedCache::batch: " + std::to_string(ids.size()) + " sequences, " + std::to_string(tokens.size()) + " counts");
    std::int64_t grouped = 0;
    for (const std::int64_t n : group_sizes) {
        if (n < 1 || n > static_cast<std::int64_t>(ids.size()) - grouped) throw Error("PagedCache::batch: a group of " + std::to_string(n) + " sequences");
        grouped += n;
    }
    // Whatever can be refused or fail comes before the table changes, but for
    // the uploads and copies of what it changes to.
    PagedBatch b;
    b.seqs = static_cast<std::int64_t>(ids.size());
    b.groups = static_cast<std::int64_t>(group_sizes.size());
    if (b.seqs > kMaxSeqs) throw Error("PagedCache::batch: more than 65536 sequences");
    std::int64_t most = 1;
    for (std::size_t i = 0; i < ids.size(); ++i) {
        const std::int64_t length = table_.length(ids[i]);
        if (tokens[i] < 0) throw Error("PagedCache::batch: " + std::to_string(tokens[i]) + " tokens");
        if (tokens[i] > kMaxKeys - length) throw Error("PagedCache::batch: a sequence of more than 2^26 keys");
        b.tokens += tokens[i];
        if (b.tokens > kMaxTokens) throw Error("PagedCache::batch: more than 2^22 new tokens");
        most = std::max(most, length + tokens[i]);
        if (tokens[i] > 0) b.positions = std::max(b.positions, length + tokens[i]);
    }
    const std::int64_t stride = (most + table_.page_size() - 1) / table_.page_size();
    detail::Runtime& runtime = TensorAccess::runtime(k_);
    b.table = array(runtime, {b.seqs, stride});
    b.lengths = array(runtime, {b.seqs});
    b.starts = array(runtime, {b.seqs + 1});
    if (b.groups > 0) {
        b.group_starts = array(runtime, {b.groups + 1});
        b.group_keys = array(runtime, {b.groups});
    }
    const std::vector<PageCopy> copies = table_.append(ids, tokens);
    try {
        std::vector<std::int32_t> table(ids.size() * static_cast<std::size_t>(stride), -1), lengths, starts = {0}, group_starts = {0}, group_keys;
        for (std::size_t i = 0; i < ids.size(); ++i) {
            const auto& row = table_.row(ids[i]);
            std::copy(row.begin(), row.end(), table.begin() + static_cast<std::ptrdiff_t>(i * static_cast<std::size_t>(stride)));
            lengths.push_back(static_cast<std::int32_t>(table_.length(ids[i])));
            starts.push_back(static_cast<std::int32_t>(starts.back() + tokens[i]));
        }
        std::size_t at = 0;
        for (const std::int64_t n : group_sizes) {
            const auto count = static_cast<std::size_t>(n);
            group_keys.push_back(static_cast<std::int32_t>(table_.shared(ids.subspan(at, count), tokens.subspan(at, count))));
            at += count;
            group_starts.push_back(static_cast<std::int32_t>(at));
        }
        upload(b.table, table);
        upload(b.lengths, lengths);
        upload(b.starts, starts);
        if (b.groups > 0) {
            upload(b.group_starts, group_starts);
            upload(b.group_keys, group_keys);
        }
        copy(copies);  // (into pages that were free, should it fail)
    } catch (...) {
        table_.undo(ids, tokens, copies);
        throw;
    }
    return b;
}

Tensor PagedCache::append(std::int64_t layer, const PagedBatch& batch, const Tensor& qkv, const Tensor& rope_table, RopeStyle style) {
    const Shape& s = qkv.shape();
    const std::int64_t heads = s.size() == 2 && s[1] % head_dim_ == 0 ? s[1] / head_dim_ - 2 * kv_heads_ : 0;
    if (qkv.dtype() != DType::F32 || heads < 1 || s[0] != batch.tokens) {
        throw Error("PagedCache::append: qkv must be f32 [" + std::to_string(batch.tokens) + ", (heads + " + std::to_string(2 * kv_heads_) + ") * " +
                    std::to_string(head_dim_) + "], got " + std::string(to_string(qkv.dtype())) + " " + to_string(s));
    }
    const Shape& t = rope_table.shape();
    const bool rotated = t != Tensor().shape();
    if (rotated && (rope_table.dtype() != DType::F32 || t.size() != 3 || t[1] * 2 > head_dim_ || t[2] != 2)) {
        throw Error("PagedCache::append: heads of " + std::to_string(head_dim_) + " do not match the table " + to_string(t) + " from rope_table");
    }
    if (rotated && batch.positions > t[0]) {
        throw Error("PagedCache::append: positions up to " + std::to_string(batch.positions - 1) + " are outside the table's " + std::to_string(t[0]) + " positions");
    }
    Tensor q = TensorAccess::empty(TensorAccess::runtime(qkv), {batch.tokens, heads, head_dim_}, DType::F32);
    if (batch.tokens == 0) return q;
    vkml_rope_kv_pages_params p{};
    p.heads = u32(heads);
    p.kv_heads = u32(kv_heads_);
    p.head_dim = u32(head_dim_);
    p.kv_type = detail::type_code(k_.dtype());
    p.page_size = u32(table_.page_size());
    p.pages = u32(table_.pages());
    p.seqs = u32(batch.seqs);
    p.tokens = u32(batch.tokens);
    p.table_stride = u32(batch.table.shape().back());
    p.row_stride = u32(s[1]);
    p.rotary_dim = rotated ? u32(2 * t[1]) : 0;
    p.style = style == RopeStyle::Interleaved ? 0 : 1;
    p.positions = rotated ? u32(t[0]) : 0;
    check(vkml_rope_kv_pages(&p, static_cast<const float*>(qkv.data()), rotated ? static_cast<const float*>(rope_table.data()) : nullptr, ints(batch.table),
                             ints(batch.lengths), ints(batch.starts), nullptr, static_cast<float*>(q.data()), pool(k_, layer), pool(v_, layer)),
          "PagedCache::append");
    return q;
}

Tensor PagedCache::attention(std::int64_t layer, const PagedBatch& batch, const Tensor& q, float softcap) const {
    const Shape& s = q.shape();
    if (q.dtype() != DType::F32 || s.size() != 3 || s[0] != batch.tokens || s[1] < 1 || s[1] % kv_heads_ != 0 || s[2] != head_dim_) {
        throw Error("PagedCache::attention: q must be f32 [" + std::to_string(batch.tokens) + ", heads, " + std::to_string(head_dim_) + "] with heads a multiple of " +
                    std::to_string(kv_heads_) + ", got " + std::string(to_string(q.dtype())) + " " + to_string(s));
    }
    detail::Runtime& runtime = TensorAccess::runtime(q);
    Tensor out = TensorAccess::empty(runtime, s, DType::F32);
    if (batch.tokens == 0) return out;
    vkml_attend_pages_params p{};
    p.heads = u32(s[1]);
    p.kv_heads = u32(kv_heads_);
    p.head_dim = u32(head_dim_);
    p.kv_type = detail::type_code(k_.dtype());
    p.page_size = u32(table_.page_size());
    p.pages = u32(table_.pages());
    p.seqs = u32(batch.seqs);
    p.tokens = u32(batch.tokens);
    p.table_stride = u32(batch.table.shape().back());
    p.groups = u32(batch.groups);
    p.scale = 1.0f / std::sqrt(static_cast<float>(head_dim_));
    p.softcap = softcap;
    const std::uint64_t bytes = vkml_attend_pages_workspace_bytes(&p);
    // Released when this returns: later work on the stream runs after the call's.
    const Tensor workspace = TensorAccess::empty(runtime, {static_cast<std::int64_t>(std::max<std::uint64_t>(bytes, 16) / 4)}, DType::F32);
    check(vkml_attend_pages(&p, static_cast<const float*>(q.data()), pool(k_, layer), pool(v_, layer), ints(batch.table), ints(batch.lengths), ints(batch.starts),
                            batch.groups > 0 ? ints(batch.group_starts) : nullptr, batch.groups > 0 ? ints(batch.group_keys) : nullptr, workspace.data(),
                            static_cast<float*>(out.data())),
          "PagedCache::attention");
    return out;
}

}  // namespace vkml
