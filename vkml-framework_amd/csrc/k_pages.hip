// k_pages.hip -- rotary positions into a paged KV cache, and copies of its
// pages (vkml_rope_kv_pages, vkml_copy_pages). Both move bytes and compute
// next to nothing: what bounds them is memory, and a launch's latency where
// there are few.
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
