// k_pages.hip -- rotary positions into a paged KV cache, copies of its pages,
// and the drafted tokens that stay in it (vkml_rope_kv_pages, vkml_copy_pages,
// vkml_keep_drafts). All move bytes and compute next to nothing: what bounds them
// is memory, and a launch's latency where there are few.
#include <hip/hip_runtime.h>

#include <new>
#include <string>
#include <vector>

#include "device.hpp"
#include "internal.hpp"
#include "pages.hpp"

using namespace vkml::dev;
using vkml::pages::Batch;

namespace {

constexpr uint32_t kThreads = 256;

// ---------------------------------------------------------------- rope and append

struct RopeArgs {
    const float* qkv;
    const float* angles;     // [positions, rotary_dim / 2, 2]
    const int32_t* table;    // [seqs, table_stride]
    const int32_t* at;       // each token's position for the turn, or null
    float* q;
    void* k;
    void* v;
    Batch batch;
    uint64_t page_stride;
    uint32_t heads, kv_heads, head_dim, page_size, pages, table_stride, row_stride, rotary_dim, style, positions;
};

template <int W>
struct Part {
    float x[W];
};

template <int W>
__device__ __forceinline__ Part<W> read(const float* p) {
    Part<W> r;
    if constexpr (W == 4) {
        const float4 f = ldg(reinterpret_cast<const float4*>(p));
        r.x[0] = f.x, r.x[1] = f.y, r.x[2] = f.z, r.x[3] = f.w;
    } else {
        r.x[0] = ldg(p);
    }
    return r;
}

// W values to a row of q or of a pool (each rounded once, to nearest even).
template <int W, typename T>
__device__ __forceinline__ void write(T* p, const Part<W>& r) {
    if constexpr (W == 1) {
        stg(p, static_cast<T>(r.x[0]));
    } else if constexpr (sizeof(T) == 4) {
        stg(reinterpret_cast<float4*>(p), make_float4(r.x[0], r.x[1], r.x[2], r.x[3]));
    } else {
        typedef T t4 __attribute__((ext_vector_type(4)));
        const t4 h = {static_cast<T>(r.x[0]), static_cast<T>(r.x[1]), static_cast<T>(r.x[2]), static_cast<T>(r.x[3])};
        stg(reinterpret_cast<uint2*>(p), __builtin_bit_cast(uint2, h));
    }
}

// Workgroup (x, y): kThreads units of token x. A unit is 2 W values of one head
// that one thread takes: W pairs of a turned part, or 2 W consecutive dims of an
// unturned one (v, and q's and k's dims from rotary_dim on). A thread's values
// are loaded first; where its token stands is found meanwhile. Bound by memory:
// 7900 tokens of 32 + 2 * 8 heads of 128 (355 MB read and written) in 68 us, 5.2
// TB/s, where a large copy reaches 5.0; 32 such tokens 3.6 us, a launch. Two or
// three units a thread, their loads in flight together, took as long.
template <int W, typename T>
__global__ void __launch_bounds__(kThreads) k_rope_kv_pages(RopeArgs a) {
    const int32_t t = static_cast<int32_t>(blockIdx.x);
    const uint32_t hd = a.head_dim, r = a.rotary_dim, per_head = hd / (2 * W), turned = r / (2 * W), units = (a.heads + 2 * a.kv_heads) * per_head;
    const float* row = a.qkv + static_cast<uint64_t>(t) * a.row_stride;
    const uint32_t unit = blockIdx.y * kThreads + threadIdx.x, u = min(unit, units - 1);  // past the last: that again, not stored
    const uint32_t head = u / per_head;
    const bool is_v = head >= a.heads + a.kv_heads;
    const bool turns = !is_v && u % per_head < turned;
    const uint32_t e = u % per_head, ia = turns && a.style == 1 ? W * e : 2 * W * e, ib = turns && a.style == 1 ? r / 2 + W * e : ia + W;
    Part<W> x = read<W>(row + head * hd + ia), y = read<W>(row + head * hd + ib);
    int32_t s = t;
    if (a.batch.starts) {  // the sequences that end at or before the token
        s = 0;
        for (int32_t i = 0; i < a.batch.seqs; i += kThreads) {
            const int32_t j = i + static_cast<int32_t>(threadIdx.x);
            s += __syncthreads_count(j < a.batch.seqs && a.batch.start(j + 1) <= t);
        }
    }
    if (s >= a.batch.seqs || t < a.batch.start(s) || unit >= units) return;
    const int32_t pos = a.batch.length(s) - a.batch.count(s) + t - a.batch.start(s);
    const int32_t page =
        head >= a.heads && pos >= 0 && pos < a.batch.table_keys ? ldg(a.table + static_cast<uint64_t>(s) * a.table_stride + pos / a.page_size) : -1;
    if (turns) {
        const int32_t turn = a.at ? a.at[t] : pos;
        float c[W], d[W];  // cos and sin of the unit's pairs
#pragma unroll
        for (int j = 0; j < W; ++j) c[j] = d[j] = __builtin_nanf("");
        if (static_cast<uint32_t>(turn) < a.positions) {
            const float* angles = a.angles + static_cast<uint64_t>(turn) * r;
            if constexpr (W == 4) {
                const Part<4> lo = read<4>(angles + 8 * e), hi = read<4>(angles + 8 * e + 4);
                c[0] = lo.x[0], d[0] = lo.x[1], c[1] = lo.x[2], d[1] = lo.x[3];
                c[2] = hi.x[0], d[2] = hi.x[1], c[3] = hi.x[2], d[3] = hi.x[3];
            } else {
                c[0] = ldg(angles + 2 * e);
                d[0] = ldg(angles + 2 * e + 1);
            }
        }
        const Part<W> f = x, g = y;
        if (W == 1 || a.style == 1) {  // the pairs are (f[j], g[j])
#pragma unroll
            for (int j = 0; j < W; ++j) {
                x.x[j] = f.x[j] * c[j] - g.x[j] * d[j];
                y.x[j] = f.x[j] * d[j] + g.x[j] * c[j];
            }
        } else {  // neighbours in the 2 W values
#pragma unroll
            for (int j = 0; j < W / 2; ++j) {
                x.x[2 * j] = f.x[2 * j] * c[j] - f.x[2 * j + 1] * d[j];
                x.x[2 * j + 1] = f.x[2 * j] * d[j] + f.x[2 * j + 1] * c[j];
                y.x[2 * j] = g.x[2 * j] * c[W / 2 + j] - g.x[2 * j + 1] * d[W / 2 + j];
                y.x[2 * j + 1] = g.x[2 * j] * d[W / 2 + j] + g.x[2 * j + 1] * c[W / 2 + j];
            }
        }
    }
    if (head < a.heads) {
        float* to = a.q + (static_cast<uint64_t>(t) * a.heads + head) * hd;
        write<W>(to + ia, x);
        write<W>(to + ib, y);
        return;
    }
    if (static_cast<uint32_t>(page) >= a.pages) return;
    const uint32_t kvh = head - a.heads - (is_v ? a.kv_heads : 0);
    T* to = static_cast<T*>(is_v ? a.v : a.k) + static_cast<uint64_t>(page) * a.page_stride +
            (static_cast<uint64_t>(kvh) * a.page_size + pos % a.page_size) * hd;
    write<W>(to + ia, x);
    write<W>(to + ib, y);
}

// ---------------------------------------------------------------- page copies

// The pairs of one launch, in its arguments: a captured graph keeps them, and
// no buffer has to outlive the call.
constexpr uint32_t kPairs = 448;
struct CopyArgs {
    uint8_t* pool[2];
    uint64_t page_stride, layer_stride;
    uint32_t vectors;  // 16-byte vectors a page
    uint32_t pieces;   // workgroups a page
    uint32_t src[kPairs], dst[kPairs];
};
constexpr uint32_t kVectors = 4;  // vectors a thread has in flight

// Workgroup x: piece x % pieces of pair x / pieces; y the layer, z the pool.
// Bound by memory: 31 pages of 128 KiB in 32 layers of two pools (260 MB read and
// as much written) in 98 us, 5.3 TB/s; a large copy reaches 5.0.
__global__ void __launch_bounds__(kThreads) k_copy_pages(CopyArgs a) {
    const uint32_t pair = blockIdx.x / a.pieces, piece = blockIdx.x % a.pieces;
    uint8_t* base = a.pool[blockIdx.z] + blockIdx.y * a.layer_stride;
    const uint4* src = reinterpret_cast<const uint4*>(base + a.src[pair] * a.page_stride);
    uint4* dst = reinterpret_cast<uint4*>(base + a.dst[pair] * a.page_stride);
    const uint32_t first = piece * kVectors * kThreads + threadIdx.x;
    uint4 v[kVectors];
#pragma unroll
    for (uint32_t i = 0; i < kVectors; ++i)
        if (first + i * kThreads < a.vectors) v[i] = ldg(src + first + i * kThreads);
#pragma unroll
    for (uint32_t i = 0; i < kVectors; ++i)
        if (first + i * kThreads < a.vectors) stg(dst + first + i * kThreads, v[i]);
}

// ---------------------------------------------------------------- drafts that stay

struct KeepArgs {
    const int32_t* parents;  // [tokens]
    const int32_t* drafted;
    const int32_t* picked;
    const int32_t* table;
    int32_t* path;    // [tokens]
    int32_t* counts;  // [seqs]
    int32_t* next;
    uint8_t* pool[2];
    Batch batch;
    uint64_t page_bytes, layer_bytes;  // from one to the next
    uint32_t row_bytes;                // a key's of one head
    uint32_t kv_heads, page_shift, pages, table_stride;
};
constexpr uint32_t kKeepVectors = 4;  // a thread has in flight

// Workgroup (sequence, layer). It walks the tree: the first node after the one it is
// at, of that parent, whose drafted token is the parent's pick, 64 nodes looked at at
// once. (Every workgroup for itself: a walk is some 0.3 us, a launch of its own were
// 2.) A tree of up to 64 nodes is in the lanes of each wave; a larger one in the LDS,
// walked by the first. Then the rows of the path move to the places after one another
// that it takes, both pools'. They are read and written by turns, 16 KB at most, since a
// row may go to where another one comes from: never to where one of a later turn does, as
// a path's k-th node is the k-th of the tree or a later one.
// Bound by its waits (arrays, the walk, pages, rows: four in a chain) rather than by bytes:
// one sequence's 16 layers 5.4 us, 24 sequences' 32 layers 9.2 (16 MB read and written, 3.2
// us at a copy's rate; 11.2 with a workgroup a pool, which walks every tree twice).
template <typename V>
__global__ void __launch_bounds__(kThreads) k_keep_drafts(KeepArgs a) {
    constexpr int32_t kNodes = static_cast<int32_t>(vkml::pages::kMaxNodes);
    static_assert(kNodes <= 0x7FFF);
    __shared__ int16_t s_parent[kNodes], s_path[kNodes];
    __shared__ int32_t s_count;
    const int32_t s = static_cast<int32_t>(blockIdx.x), token0 = a.batch.start(s), all = a.batch.count(s), n = min(all, kNodes);
    const int32_t base = a.batch.length(s) - all, l = static_cast<int32_t>(threadIdx.x % kWave);
    const bool small = n <= kWave;
    const int32_t* table = a.table + static_cast<uint64_t>(s) * a.table_stride;
    // The pages that the new tokens are in, from the first one's on, for a small tree
    // (5 at most) a lane each, loaded beside the tree.
    const auto page_at = [&](int32_t i) { return i >= 0 && i < static_cast<int32_t>(a.table_stride) ? static_cast<uint32_t>(ldg(table + i)) : ~0u; };
    const int32_t first_page = base >> a.page_shift;
    uint32_t held = ~0u;
    if (small && l < 8) held = page_at(first_page + l);
    int32_t count = n > 0 ? 1 : 0, path = 0;  // small: node l of the path
    if (small) {
        int32_t parent = -1, drafted = 0, picked = 0;
        if (l < n) parent = ldg(a.parents + token0 + l), drafted = ldg(a.drafted + token0 + l), picked = ldg(a.picked + token0 + l);
        // The parent of a node that its parent's pick is the token of; of the others none.
        const bool earlier = parent >= 0 && parent < l;
        const int32_t pick = __shfl(picked, earlier ? parent : 0);
        if (!earlier || pick != drafted) parent = -1;
        for (int32_t at = 0;;) {
            const uint64_t found = __ballot(parent == at);
            if (found == 0) break;
            at = static_cast<int32_t>(__builtin_ctzll(found));
            if (l == count) path = at;
            ++count;
        }
    } else {
        for (int32_t i = static_cast<int32_t>(threadIdx.x); i < n; i += kThreads) {
            const int32_t parent = ldg(a.parents + token0 + i);
            s_parent[i] = static_cast<int16_t>(parent >= 0 && parent < i && ldg(a.picked + token0 + parent) == ldg(a.drafted + token0 + i) ? parent : -1);
        }
        __syncthreads();
        if (threadIdx.x < kWave) {
            if (l == 0) s_path[0] = 0;
            int32_t at = 0;
            for (int32_t i = 0; i < n;) {
                const uint64_t found = __ballot(i + l > at && i + l < n && s_parent[min(i + l, n - 1)] == at);
                if (found == 0) {
                    i += kWave;
                    continue;
                }
                at = i + static_cast<int32_t>(__builtin_ctzll(found));
                i = at / kWave * kWave;
                if (l == 0) s_path[count] = static_cast<int16_t>(at);
                ++count;
            }
            if (l == 0) s_count = count;
        }
        __syncthreads();
        count = s_count;
    }
    // (by all of a wave's lanes at once)
    const auto node_of = [&](int32_t j) { return small ? __shfl(path, min(j, kWave - 1)) : static_cast<int32_t>(s_path[min(j, kNodes - 1)]); };
    if (blockIdx.y == 0) {
        for (int32_t i0 = 0; i0 < all; i0 += kThreads) {
            const int32_t i = i0 + static_cast<int32_t>(threadIdx.x), node = node_of(i);
            if (i < all) stg(a.path + token0 + i, i < count ? node : -1);
        }
        const int32_t last = node_of(max(count, 1) - 1);
        if (threadIdx.x == 0) {
            stg(a.counts + s, count);
            stg(a.next + s, count > 0 ? ldg(a.picked + token0 + last) : -1);
        }
    }
    const uint32_t pieces = a.row_bytes / sizeof(V), per_pool = a.kv_heads * pieces, per_node = 2 * per_pool;
    const uint32_t head_bytes = a.row_bytes << a.page_shift;
    const uint64_t units = static_cast<uint64_t>(count) * per_node, layer = blockIdx.y * a.layer_bytes;
    const auto page_of = [&](int32_t pos) {  // (as node_of; no page outside the table)
        const int32_t i = pos >> a.page_shift;
        return small ? static_cast<uint32_t>(__shfl(static_cast<int>(held), i - first_page)) : page_at(i);
    };
    for (uint64_t first = per_node; first < units; first += kKeepVectors * kThreads) {  // (node 0 stays)
        V v[kKeepVectors];
        uint8_t* to[kKeepVectors];
#pragma unroll
        for (uint32_t i = 0; i < kKeepVectors; ++i) {
            const uint64_t u = min(first + i * kThreads + threadIdx.x, units - 1);
            const int32_t j = static_cast<int32_t>(u / per_node), node = node_of(j);
            const uint32_t unit = static_cast<uint32_t>(u % per_node), in_pool = unit % per_pool;
            const uint32_t from_page = page_of(base + node), to_page = page_of(base + j);
            to[i] = nullptr;
            if (node == j || first + i * kThreads + threadIdx.x >= units || from_page >= a.pages || to_page >= a.pages) continue;
            uint8_t* pool = a.pool[unit / per_pool] + layer + static_cast<uint64_t>(in_pool / pieces) * head_bytes + in_pool % pieces * sizeof(V);
            const uint32_t mask = (1u << a.page_shift) - 1;
            to[i] = pool + to_page * a.page_bytes + (static_cast<uint32_t>(base + j) & mask) * a.row_bytes;
            v[i] = ldg(reinterpret_cast<const V*>(pool + from_page * a.page_bytes + (static_cast<uint32_t>(base + node) & mask) * a.row_bytes));
        }
        // Every load of the turn has landed before the first store.
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < kKeepVectors; ++i)
            if (to[i]) stg(reinterpret_cast<V*>(to[i]), v[i]);
    }
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace

extern "C" {

int vkml_rope_kv_pages(const vkml_rope_kv_pages_params* p, const float* qkv, const float* rope_table, const int32_t* table,
                       const int32_t* lengths, const int32_t* starts, const int32_t* positions, float* q, void* k_pages, void* v_pages) {
    VKML_REQUIRE_INIT();
    VKML_CHECK_ARG(p, "rope_kv_pages: null params");
    if (const char* why = vkml::pages::check(*p)) return vkml::abi::fail(VKML_ERROR_INVALID_ARGUMENT, std::string("rope_kv_pages: ") + why);
    if (p->seqs == 0 || p->tokens == 0) return VKML_OK;
    VKML_CHECK_ARG(starts || p->tokens == p->seqs, "rope_kv_pages: without starts every sequence has one token");
    VKML_CHECK_ARG(qkv && table && lengths && q && k_pages && v_pages && (rope_table || p->rotary_dim == 0), "rope_kv_pages: null buffer");
    const Batch batch{lengths, starts, nullptr, nullptr, static_cast<int32_t>(p->seqs), static_cast<int32_t>(p->tokens), 0,
                      static_cast<int32_t>(p->table_stride * p->page_size)};
    const uint64_t stride = p->page_stride ? p->page_stride : static_cast<uint64_t>(p->kv_heads) * p->page_size * p->head_dim;
    const RopeArgs a{qkv, rope_table, table, positions, q, k_pages, v_pages, batch, stride, p->heads, p->kv_heads, p->head_dim, p->page_size, p->pages,
                     p->table_stride, p->row_stride, p->rotary_dim, p->style, p->positions};
    // Four values a load where every part starts on 16 bytes.
    const bool wide = p->head_dim % 8 == 0 && p->rotary_dim % 8 == 0 && p->row_stride % 4 == 0 && aligned16(qkv) && aligned16(rope_table) &&
                      aligned16(q) && aligned16(k_pages) && aligned16(v_pages);
    const uint32_t units = (p->heads + 2 * p->kv_heads) * (p->head_dim / (wide ? 8 : 2));
    const dim3 grid(p->tokens, (units + kThreads - 1) / kThreads);
    vkml::abi::ProfileScope prof("rope_kv_pages");
    const auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, vkml::abi::stream(), a); };
    if (p->kv_type == VKML_F16) wide ? go(k_rope_kv_pages<4, _Float16>) : go(k_rope_kv_pages<1, _Float16>);
    else wide ? go(k_rope_kv_pages<4, float>) : go(k_rope_kv_pages<1, float>);
    return vkml::abi::check_launch("rope_kv_pages");
}

int vkml_keep_drafts(const vkml_keep_drafts_params* p, const int32_t* parents, const int32_t* drafted, const int32_t* picked, const int32_t* table,
                     const int32_t* lengths, const int32_t* starts, int32_t* path, int32_t* counts, int32_t* next, void* k_pages, void* v_pages) {
    VKML_REQUIRE_INIT();
    VKML_CHECK_ARG(p, "keep_drafts: null params");
    if (const char* why = vkml::pages::check(*p)) return vkml::abi::fail(VKML_ERROR_INVALID_ARGUMENT, std::string("keep_drafts: ") + why);
    if (p->seqs == 0) return VKML_OK;
    VKML_CHECK_ARG(starts || p->tokens == p->seqs, "keep_drafts: without starts every sequence has one token");
    VKML_CHECK_ARG(table && lengths && counts && next && k_pages && v_pages && (p->tokens == 0 || (parents && drafted && picked && path)), "keep_drafts: null buffer");
    const uint32_t size = p->kv_type == VKML_F16 ? 2 : 4;
    const uint64_t page = p->page_stride ? p->page_stride : static_cast<uint64_t>(p->kv_heads) * p->page_size * p->head_dim;
    KeepArgs a{};
    a.parents = parents;
    a.drafted = drafted;
    a.picked = picked;
    a.table = table;
    a.path = path;
    a.counts = counts;
    a.next = next;
    a.pool[0] = static_cast<uint8_t*>(k_pages);
    a.pool[1] = static_cast<uint8_t*>(v_pages);
    a.batch = Batch{lengths, starts, nullptr, nullptr, static_cast<int32_t>(p->seqs), static_cast<int32_t>(p->tokens), 0,
                    static_cast<int32_t>(p->table_stride * p->page_size)};
    a.page_bytes = page * size;
    a.layer_bytes = (p->layer_stride ? p->layer_stride : p->pages * page) * size;
    a.row_bytes = p->head_dim * size;
    a.kv_heads = p->kv_heads;
    a.page_shift = static_cast<uint32_t>(__builtin_ctz(p->page_size));
    a.pages = p->pages;
    a.table_stride = p->table_stride;
    // (strides are multiples of 8 elements, so that rows start on 16 bytes as the pools and a row's bytes do)
    const bool wide = a.row_bytes % 16 == 0 && a.page_bytes % 16 == 0 && a.layer_bytes % 16 == 0 && aligned16(k_pages) && aligned16(v_pages);
    vkml::abi::ProfileScope prof("keep_drafts");
    const auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(p->seqs, p->layers), dim3(kThreads), 0, vkml::abi::stream(), a); };
    wide ? go(k_keep_drafts<uint4>) : go(k_keep_drafts<uint32_t>);
    return vkml::abi::check_launch("keep_drafts");
}

int vkml_copy_pages(const vkml_copy_pages_params* p, const int32_t* src, const int32_t* dst, void* k_pages, void* v_pages) {
    VKML_REQUIRE_INIT();
    VKML_CHECK_ARG(p, "copy_pages: null params");
    if (const char* why = vkml::pages::check(*p)) return vkml::abi::fail(VKML_ERROR_INVALID_ARGUMENT, std::string("copy_pages: ") + why);
    if (p->count == 0) return VKML_OK;
    VKML_CHECK_ARG(src && dst && k_pages && v_pages, "copy_pages: null buffer");
    VKML_CHECK_ARG(aligned16(k_pages) && aligned16(v_pages), "copy_pages: the pools must be 16-byte aligned");
    try {
        std::vector<uint64_t> marks((p->pages + 63) / 64);
        if (const char* why = vkml::pages::check_copies(p->pages, p->count, src, dst, marks.data()))
            return vkml::abi::fail(VKML_ERROR_INVALID_ARGUMENT, std::string("copy_pages: ") + why);
    } catch (const std::bad_alloc&) {
        return vkml::abi::fail(VKML_ERROR_OUT_OF_MEMORY, "copy_pages: out of host memory");
    }
    CopyArgs a;
    a.pool[0] = static_cast<uint8_t*>(k_pages);
    a.pool[1] = static_cast<uint8_t*>(v_pages);
    a.page_stride = p->page_stride ? p->page_stride : p->page_bytes;
    a.layer_stride = p->layer_stride ? p->layer_stride : p->pages * a.page_stride;
    a.vectors = static_cast<uint32_t>(p->page_bytes / 16);
    a.pieces = (a.vectors + kVectors * kThreads - 1) / (kVectors * kThreads);
    // (a launch has less than 2^32 threads)
    const uint32_t most = (1u << 31) / kThreads / a.pieces < kPairs ? (1u << 31) / kThreads / a.pieces : kPairs;
    vkml::abi::ProfileScope prof("copy_pages");
    for (uint32_t i = 0, n; i < p->count; i += n) {
        n = p->count - i < most ? p->count - i : most;
        for (uint32_t j = 0; j < kPairs; ++j) {
            a.src[j] = j < n ? static_cast<uint32_t>(src[i + j]) : 0;
            a.dst[j] = j < n ? static_cast<uint32_t>(dst[i + j]) : 0;
        }
        hipLaunchKernelGGL(k_copy_pages, dim3(n * a.pieces, p->layers, 2), dim3(kThreads), 0, vkml::abi::stream(), a);
        if (const int r = vkml::abi::check_launch("copy_pages")) return r;
    }
    return VKML_OK;
}

}  // extern "C"
