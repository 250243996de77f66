// pages.hpp -- the paged KV cache of several sequences: what a call's
// parameters must be, and which rows, keys and shared prefix the sequences of
// a batch have. Code without HIP's runtime, so that the checks can be tested
// on any machine.
#pragma once

#include <cstdint>

#include "../../include/vkml_hip.h"

#if defined(__HIPCC__)
#define VKML_HD __host__ __device__ __forceinline__
#else
#define VKML_HD inline
#endif

namespace vkml::pages {

constexpr uint32_t kMaxGroup = 128;       // query heads a KV head
constexpr uint32_t kMaxSeqs = 1u << 16;   // sequences a batch
constexpr uint32_t kMaxTokens = 1u << 22;  // new tokens a batch
constexpr float kFinite = 3.402823466e+38f;

VKML_HD int32_t clamp_to(int32_t v, int32_t lo, int32_t hi) { return v < lo ? lo : v > hi ? hi : v; }

// An element of a call's arrays, which no launch that reads them writes: for
// an index that a workgroup's threads share, through the scalar unit.
VKML_HD int32_t element(const int32_t* p, int32_t i) {
#if defined(__HIP_DEVICE_COMPILE__)
    return *reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(reinterpret_cast<uintptr_t>(p + i));
#else
    return p[i];
#endif
}

// The batch as the device reads it. Its values are device memory, so the host
// cannot check them: every read here clamps what it finds, so that no value
// leads outside q, the table or the pools.
struct Batch {
    const int32_t* lengths;
    const int32_t* starts;        // null: token s is sequence s's
    const int32_t* group_starts;  // groups + 1
    const int32_t* group_keys;
    int32_t seqs, tokens, groups, table_keys;

    VKML_HD int32_t start(int32_t s) const { return starts ? clamp_to(element(starts, s), 0, tokens) : s < tokens ? s : tokens; }
    // New tokens of sequence s from start(s) on.
    VKML_HD int32_t count(int32_t s) const {
        const int32_t n = start(s + 1) - start(s);
        return n > 0 ? n : 0;
    }
    VKML_HD int32_t length(int32_t s) const { return clamp_to(element(lengths, s), 0, table_keys); }
    VKML_HD int32_t group_start(int32_t g) const { return clamp_to(element(group_starts, g), 0, seqs); }
    VKML_HD int32_t group_key(int32_t g) const { return clamp_to(element(group_keys, g), 0, table_keys); }
    // The group that sequence s is in, if it is in any.
    VKML_HD int32_t group_near(int32_t s) const {
        int32_t lo = 0, hi = groups;
        while (hi - lo > 1) {
            const int32_t mid = (lo + hi) / 2;
            if (group_start(mid) <= s) lo = mid;
            else hi = mid;
        }
        return lo;
    }
};

// ---------------------------------------------------------------- the work of vkml_attend_pages

// A KV head's work is a list of segments: for each group its shared keys by
// all of its tokens, then for each sequence its other keys by its tokens. A
// segment's tokens go in tiles: all of them where they are at most kFewRows
// rows (token, query head), else kTileRows / (query heads a KV head) at a time.
// A tile has a cost, and the whole of all KV heads' tiles, laid end to end, is
// cut into equal parts of it, one a workgroup: what a workgroup takes of a tile
// is a piece. A cut within a tile's own cost is made at its start instead, and one
// near its end there: the rest would cost more by itself than it evens out. (The
// parts follow the tiles one by one: a group of more than 128 rows reads its shared
// keys once for each tile, far apart in time.)
constexpr int32_t kFewRows = 16;
constexpr int32_t kTileRows = 128;
constexpr int32_t kLeadStep = 128;  // a multiple of every block of keys

// A tile's cost: a key's times its keys, and one of its own for its queries,
// its first loads, its joining and storing. Measured (us, 64 keys, two
// workgroups a compute unit): f16, head_dim 128, a tile of few rows, which
// memory bounds, 1.1 beside one of many, and that one 3.4 beside it, 4.0 beside
// its like; by themselves the tiles take 8 and 10, some of it while the other
// workgroup works. f32, head_dim 64: 1.6 and 3.8; 1.7 and 1.2. f16 at 64 and f32
// at 128 are not measured: a key's cost goes by its bytes, a tile's own stays.
struct Costs {
    int32_t few_key, tile_key, few_own, tile_own;
};
// The cost below which work is not cut further. Measured (us a call, with 1024, 512
// and 256): 8 sequences, 2000 shared keys, f32, head_dim 64, 19.6, 17.8, 17.8; one
// sequence of 2000 keys 13.3, 12.1, 13.8; three of 5 to 40 11.2, 11.0, 12.5.
constexpr int32_t kMinPart = 512;
VKML_HD Costs costs(uint32_t head_dim, bool f16) {
    const int32_t few = static_cast<int32_t>(head_dim / (f16 ? 16 : 8));
    return {few, f16 ? 3 * few : few + few * 3 / 4, f16 ? 2600 : 600, f16 ? 3600 : 600};
}

VKML_HD int32_t tile_tokens(int32_t group) { return kTileRows / group > 1 ? kTileRows / group : 1; }

// The keys of a segment lie on one axis: first the `lead` keys that its tokens
// read through the table row of their group's first sequence, filled up to a
// multiple of kLeadStep, then those from position lo on, of its own row.
struct Segment {
    int32_t row = 0;       // the sequence whose table holds the keys from lo on
    int32_t lead_row = 0;  // and the `lead` keys
    int32_t lead = 0;
    int32_t token0 = 0;    // the first token
    int32_t n = 0;         // tokens
    int32_t from = 0;      // the first position that counts
    int32_t base = 0;      // positions from lo() on before the first token's; shared keys: all
    int32_t tiles = 0, step = 1;
    bool few = false, shared = false;
    int32_t key_cost = 0, own_cost = 0;

    // The first position read, a multiple of 16.
    VKML_HD int32_t lo() const { return from & ~15; }
    VKML_HD int32_t lead_span() const { return (lead + kLeadStep - 1) / kLeadStep * kLeadStep; }
    // The axis' length for tile i's tokens.
    VKML_HD int32_t keys(int32_t i) const {
        int32_t own = base;
        if (!shared) {
            own += base < 0 || (i + 1) * step > n ? n : (i + 1) * step;
            own = own > 0 ? own : 0;
        }
        return lead_span() + own;
    }
    VKML_HD int32_t tile_cost(int32_t i) const { return own_cost + key_cost * keys(i); }  // (2^26 keys' fits)
    // The cost of the tiles before tile i.
    VKML_HD int64_t before(int32_t i) const {
        if (i == 0) return 0;
        const bool equal = shared || base < 0;
        const int64_t k = i, each = own_cost + static_cast<int64_t>(key_cost) * (equal ? keys(0) : lead_span() + base);
        return equal ? k * each : k * each + key_cost * (step * (k * (k + 1) / 2));
    }
    VKML_HD int64_t cost() const { return tiles ? before(tiles - 1) + tile_cost(tiles - 1) : 0; }
    // The tile that holds unit u of the segment, 0 <= u < cost().
    VKML_HD int32_t tile_at(int64_t u) const {
        int32_t first = 0, hi = tiles;
        while (hi - first > 1) {
            const int32_t mid = first + (hi - first) / 2;
            if (before(mid) <= u) first = mid;
            else hi = mid;
        }
        return first;
    }
    // The position past the last that token i of the segment sees.
    VKML_HD int32_t limit(int32_t i) const { return shared ? base : lo() + base + i + 1; }
    VKML_HD int32_t tile_n(int32_t i) const { return n - i * step < step ? n - i * step : step; }
};

// Segment i of a batch: groups 0 .. groups - 1, then the sequences. (Loads that
// don't depend on one another come before what branches on them.)
//
// A group's shared keys are a segment of their own unless its sequences have
// half a tile of tokens or more on average: then their own tiles read few
// blocks more than the group's would, and no rows are in two parts. A group of
// one sequence shares nothing.
VKML_HD Segment segment(const Batch& b, int32_t group, Costs costs, int32_t i) {
    const bool of_group = i < b.groups;
    const int32_t q = of_group ? 0 : i - b.groups;
    const int32_t own0 = b.start(q), own1 = b.start(q + 1), length = b.length(q);
    int32_t first = 0, last = 0, keys = 0;
    if (b.groups > 0) {
        const int32_t g = of_group ? i : b.group_near(q);
        first = b.group_start(g);
        last = b.group_start(g + 1);
        keys = b.group_key(g);
        if (last - first < 2 || !(of_group || (first <= q && q < last))) keys = 0;
    }
    int32_t group0 = 0, group1 = 0;
    if (keys > 0) {
        group0 = b.start(first);
        group1 = b.start(last);
    }
    const int64_t tokens = static_cast<int64_t>(group1) - group0;
    const bool shares = keys > 0 && tokens > 0 && 2 * tokens <= static_cast<int64_t>(last - first) * tile_tokens(group);
    Segment s;
    if (of_group) {
        s.row = first;
        s.shared = true;
        s.base = keys;
        s.token0 = group0;
        s.n = shares ? group1 - group0 : 0;
    } else {
        s.row = q;
        s.from = keys;
        if (!shares) s.lead = keys, s.lead_row = keys > 0 ? first : 0;
        s.token0 = own0;
        s.n = own1 > own0 ? own1 - own0 : 0;
        s.base = length - s.n - s.lo();
    }
    s.few = s.n <= kFewRows && s.n * group <= kFewRows;
    s.step = s.few ? (s.n > 0 ? s.n : 1) : tile_tokens(group);
    s.tiles = s.few ? (s.n > 0 ? 1 : 0) : (s.n + s.step - 1) / s.step;
    s.key_cost = s.few ? costs.few_key : costs.tile_key;
    s.own_cost = s.few ? costs.few_own : costs.tile_own;
    return s;
}

// The parts of a cost, as a power of two: one a workgroup, at least one an
// XCD, and fewer where a part would be less than kMinPart.
VKML_HD int32_t parts_log2(int64_t cost, int32_t workgroups_log2) {
    int32_t n = 3;
    while (n < workgroups_log2 && cost >> n >= 2 * kMinPart) ++n;
    return n;
}
// The first unit of part w, and the part that unit u is in (the quotient,
// found in f32 and set right).
VKML_HD int64_t part_start(int64_t cost, int32_t n_log2, int32_t w) {
    return (cost >> n_log2) * w + (static_cast<int64_t>(static_cast<uint32_t>(cost) & ((1u << n_log2) - 1)) * w >> n_log2);
}
VKML_HD int32_t part_of(int64_t cost, int32_t n_log2, int64_t u) {
    int32_t w = static_cast<int32_t>(static_cast<float>(u) / static_cast<float>(cost) * static_cast<float>(1 << n_log2));
    while (part_start(cost, n_log2, w) > u) --w;
    while (part_start(cost, n_log2, w + 1) <= u) ++w;
    return w;
}
// Where the tile of s with `cost` is cut at unit x of it: at its start (0), its
// end (cost) or between (x). Its end comes first: a tile without keys has its own
// cost alone, and the part that ends with it takes it.
VKML_HD int32_t snap(int64_t x, const Segment& s, int32_t cost) {
    if (x >= cost) return cost;
    if (x <= s.own_cost) return 0;
    return x >= cost - s.own_cost / 8 ? cost : static_cast<int32_t>(x);
}
// Where on its keys' axis a tile is cut at unit x: at whole blocks (or the
// end), so that every part cuts at the same places. f32's quotient is a block
// off at most, for all parts alike.
VKML_HD int32_t cut(int32_t x, const Segment& s, int32_t keys, int32_t block) {
    if (x <= s.own_cost) return 0;
    const float at = static_cast<float>(x - s.own_cost) / static_cast<float>(s.key_cost * block);
    const int32_t blocks = (keys + block - 1) / block;
    if (at >= static_cast<float>(blocks)) return keys;
    const int32_t up = (static_cast<int32_t>(at) + 1) * block;
    return up < keys ? up : keys;
}
// Pieces of a tile of s whose unit 0 is the whole's `start`, the first of them
// in part `first`.
VKML_HD int32_t pieces_of(int64_t cost, int32_t n_log2, const Segment& s, int64_t start, int32_t tile_cost, int32_t first) {
    const int32_t last = tile_cost - s.own_cost / 8 - 1;  // the last unit a cut can be made at
    return last <= s.own_cost ? 1 : part_of(cost, n_log2, start + last) - first + 1;
}

// What a call keeps of unfinished rows: slots of kFewRows or kTileRows rows,
// for each piece of a tile that is not the whole of its rows' work. Piece (w,
// i), workgroup w's of the i-th tile of its kind, takes slot w + i: the next
// piece has a larger w, a larger i or both.
struct Slots {
    int64_t few, tile;  // of each kind
    VKML_HD int64_t rows() const { return few * kFewRows + tile * kTileRows; }
};
// A KV head's tiles of more than kFewRows rows, at most. A batch whose sequences
// or groups overlap (which the rules exclude) may have any number, as many as would
// keep the GPU busy for hours: nothing is done for one that has more.
VKML_HD int64_t most_tiles(int64_t group, int64_t seqs, int64_t groups, int64_t tokens) {
    const int64_t many = tokens * group / (kFewRows + 1);  // segments of each kind with more than kFewRows rows, at most
    const int64_t step = tile_tokens(static_cast<int32_t>(group));
    return 2 * (tokens / step) + (seqs < many ? seqs : many) + (groups < many ? groups : many);
}
VKML_HD Slots slots(int64_t kv_heads, int64_t group, int64_t seqs, int64_t groups, int64_t tokens, int64_t workgroups) {
    return {workgroups + kv_heads * (seqs + groups), workgroups + kv_heads * most_tiles(group, seqs, groups, tokens)};
}

// The grid of `workgroups`, numbered y * x + x's own: a launch has less than 2^32
// threads in x.
struct Grid {
    uint32_t x, y;
};
VKML_HD Grid grid_of(uint32_t workgroups) {
    constexpr uint32_t kMost = 1u << 23;  // of 256 threads
    return workgroups <= kMost ? Grid{workgroups, 1} : Grid{kMost, (workgroups + kMost - 1) / kMost};
}

// ---------------------------------------------------------------- checks

inline const char* check_cache(uint32_t kv_heads, uint32_t head_dim, uint32_t kv_type, uint32_t page_size, uint32_t pages, uint64_t page_stride) {
    if (kv_type != VKML_F16 && kv_type != VKML_F32) return "caches must be f16 or f32";
    if (page_size < 16 || page_size > 1024 || (page_size & (page_size - 1))) return "page_size must be a power of two from 16 to 1024";
    if (pages == 0 || pages > 0x7FFFFFFFu) return "the pools must hold 1 to 2^31 - 1 pages";
    if (page_stride && page_stride < static_cast<uint64_t>(kv_heads) * page_size * head_dim) return "pages overlap";
    if (page_stride % 8) return "page_stride must be a multiple of 8";
    if (page_stride > (1ull << 33) || static_cast<uint64_t>(kv_heads) * page_size * head_dim > (1ull << 33)) return "pages are too large";
    return nullptr;
}

inline const char* check_batch(uint32_t seqs, uint32_t tokens, uint32_t table_stride, uint32_t page_size) {
    if (seqs > kMaxSeqs) return "more than 65536 sequences";
    if (tokens > kMaxTokens) return "more than 2^22 new tokens";
    if (table_stride == 0 || static_cast<uint64_t>(table_stride) * page_size > (1u << 26)) return "a table row must hold 1 to 2^26 keys";
    return nullptr;
}

inline const char* check(const vkml_attend_pages_params& p) {
    if (p.kv_heads == 0 || p.heads == 0 || p.heads % p.kv_heads) return "heads must be a multiple of kv_heads";
    if (p.heads / p.kv_heads > kMaxGroup) return "more than 128 query heads a KV head";
    if (static_cast<uint64_t>(p.heads) * p.tokens > 0x7FFFFFFFu) return "too many rows";
    if (p.head_dim != 64 && p.head_dim != 128) return "head_dim must be 64 or 128";
    if (const char* why = check_cache(p.kv_heads, p.head_dim, p.kv_type, p.page_size, p.pages, p.page_stride)) return why;
    if (const char* why = check_batch(p.seqs, p.tokens, p.table_stride, p.page_size)) return why;
    if (p.groups > p.seqs) return "more groups than sequences";
    if (!(p.softcap >= 0.0f && p.softcap <= kFinite)) return "softcap must be finite and not negative";
    if (!(p.scale >= -kFinite && p.scale <= kFinite)) return "scale must be finite";
    return nullptr;
}

inline const char* check(const vkml_rope_kv_pages_params& p) {
    if (p.kv_heads == 0 || p.heads == 0 || p.head_dim == 0 || p.head_dim % 2 || p.head_dim > 1024 || p.heads > 4096 || p.kv_heads > 4096) return "bad head layout";
    if (const char* why = check_cache(p.kv_heads, p.head_dim, p.kv_type, p.page_size, p.pages, p.page_stride)) return why;
    if (const char* why = check_batch(p.seqs, p.tokens, p.table_stride, p.page_size)) return why;
    if (p.rotary_dim % 2 || p.rotary_dim > p.head_dim) return "rotary_dim must be even and at most head_dim";
    if (p.style > 1) return "style must be 0 (interleaved pairs) or 1 (rotate-half)";
    if (p.row_stride < static_cast<uint64_t>(p.heads + 2 * p.kv_heads) * p.head_dim) return "rows overlap";
    return nullptr;
}

inline const char* check(const vkml_copy_pages_params& p) {
    if (p.pages == 0 || p.pages > (1u << 24)) return "the pools must hold 1 to 2^24 pages";
    if (p.page_bytes == 0 || p.page_bytes % 16 || p.page_stride % 16 || p.layer_stride % 16) return "page_bytes and the strides must be multiples of 16";
    if (p.page_bytes > (1u << 30)) return "a page must have at most 2^30 bytes";
    if (p.page_stride && p.page_stride < p.page_bytes) return "pages overlap";
    const uint64_t stride = p.page_stride ? p.page_stride : p.page_bytes;
    if (stride > (1ull << 40)) return "page_stride is too large";
    if (p.layer_stride && p.layer_stride < (p.pages - 1) * stride + p.page_bytes) return "layers overlap";
    if (p.layers == 0 || p.layers > 65535) return "1 to 65535 layers";
    return nullptr;
}

// The copy list of vkml_copy_pages: every page in the pools, no destination
// twice, and none that is also a source, so that the copies may run in any
// order. marks: (pages + 63) / 64 words, zeroed.
inline const char* check_copies(uint32_t pages, uint32_t count, const int32_t* src, const int32_t* dst, uint64_t* marks) {
    for (uint32_t i = 0; i < count; ++i) {
        const uint32_t d = static_cast<uint32_t>(dst[i]);
        if (d >= pages) return "a destination is outside the pools";
        if (marks[d / 64] >> (d % 64) & 1) return "a page is a destination twice";
        marks[d / 64] |= 1ull << (d % 64);
    }
    for (uint32_t i = 0; i < count; ++i) {
        const uint32_t s = static_cast<uint32_t>(src[i]);
        if (s >= pages) return "a source is outside the pools";
        if (marks[s / 64] >> (s % 64) & 1) return "a page is both a source and a destination";
    }
    return nullptr;
}

}  // namespace vkml::pages
