// k_attend_pages.hip -- attention of a batch's new tokens over a paged KV
// cache (vkml_attend_pages): softmax(q k^T scale) v over each token's keys,
// the ones that a group shares through its first sequence's table, for 128 of its
// rows at a time, the rest through the sequence's own.
//
// Softmax in one pass: a row (token, query head) keeps the running maximum m
// of its scores in log2 units, the sum l of 2^(x - m) and the sum o of
// 2^(x - m) v; parts (m, l, o) of a row's keys join as
//   M = max m,  l = sum 2^(m - M) l,  o = sum 2^(m - M) o,  out = o / l.
//
// The work, (KV head, rows, keys), is cut into equal parts by what it costs
// (pages.hpp), one a workgroup, whatever the lengths of the batch; two
// workgroups a compute unit are on the GPU at once. The parts follow the KV
// heads, and workgroup b takes part (b % 8) of eight first: the workgroups are
// dealt to the 8 XCDs round-robin, so an XCD's L2 sees a few KV heads only.
//
// A piece of a tile of few rows (at most 16, a sequence's in its decode step)
// is bound by the memory it streams: the four waves take blocks of keys in
// turn, each by itself, K straight into the registers of the matrix operand, V
// by global_load_lds into the wave's part of the LDS, the next block's loads
// issued before the current one is used; the waves join at the end. Of a tile
// of many rows (a group's shared keys, a prompt) a wave takes 16 or 32 rows,
// and the workgroup's waves share each block of K and V in the LDS, the next
// one loaded meanwhile.
//
// Scores S^T = K . Q^T and O^T = V^T . P^T by v_mfma_f32_16x16x32_f16 (f32
// caches: v_mfma_f32_16x16x4_f32): a row is a lane column in both, and the
// scores' accumulators are the second product's operand as they are, the keys
// permuted alike in V^T's, which ds_read_b64_tr_b16 reads transposed from the
// rows of V. f16: every product is exact, q (scaled by a power of two a row to
// [1, 2)) and the weights (times 2^14) split in two f16 terms, sums in f32.
//
// Rows of a block that hold no key that counts (past the sequence's keys, below
// the first that counts, in no page) are read from where they would be, within
// the pools; their scores are masked, and what is not finite in their V is
// cleared in the LDS before the product. So are infinities and NaN of keys that
// some rows see and others don't, which are added to those rows at the end.
//
// Measured (a whole call, 32 query and 8 KV heads of 128, f16): one token over
// 32768 keys 35 us, 5 of them to join its pieces, 134 MB at 4.4 TB/s before that (a
// large copy reaches 5.0); 64 sequences with 32768 shared keys and 1000 of their own
// 122 us, 8 to join (71 GFLOP, the split counted twice, and 547 MB read where 407
// are needed: the group's 256 rows are two tiles, one after the other, and each
// reads the shared keys from memory); 2600 tokens of six prompts 147 us, 16 to join
// (115 GFLOP).
// What the three ways through a tile need at once is more than the scalar registers
// hold: 161 to 195 are spilled to lanes of vector registers; of those none is.
// Short ones are a chain of waits: 1.0 us for the batch's arrays, 0.8 to find the
// part, 1.3 its first tile, 1.2 for pages and keys, 2 to 3 the block, 0.8 the end.
//
// The same kernel with another mask, as its own instances (MASK), so that the one above
// keeps its registers. Trees (vkml_attend_pages_tree): the new tokens' keys are masked by
// bits, up to three words a lane for 64 keys, read for blocks that hold new keys only;
// the keys before these cost nothing more. Windows (vkml_attend_pages_window): a tile of
// tokens whose window no longer begins at key 0 takes an axis of its own, the sinks and
// then the keys from its first token's window on, as long as the longest such tile's
// whatever the lengths (pages.hpp), so that the work is still cut without looking at
// lengths; what is behind the window is neither read nor counted as cost.
// Measured (a whole call, f16, 32 query and 8 KV heads of 128): 60 nodes over 8100 keys
// 40 us, 31 of them the pieces (7.9 GFLOP: with the split counted twice 12.6 us at a
// large product's rate) and 8.7 to join 512 pieces of 128 rows, 34 MB written and read;
// 24 trees of 13 over 4100 shared keys 71 us, 8 to join (18.6 GFLOP: 29.7 us); 16 chats
// of up to 30000 keys, windows of 4096, 56 us, 5 to join (245 MB: 4.3 TB/s); three prompts
// of 1400 tokens, windows of 1024, 126 us, 15 to join (41 GFLOP: 65 us). Of many rows the
// pieces are bound by the chain within a block (scores, weights, products; the next
// block's loads run meanwhile): 17 us for four blocks of 64 keys with two workgroups a
// compute unit, where the matrix units alone need 8. Of what is known from the start on,
// 4 to 6 vector registers are in scratch memory with bits at f16 and head_dim 128, 3 with
// a window and a soft cap.
#include <hip/hip_runtime.h>

#include <string>

#include "attend.hpp"
#include "attend_fast.hpp"
#include "device.hpp"
#include "internal.hpp"
#include "pages.hpp"

using namespace vkml::dev;
using namespace vkml::pages;
using vkml::attend_fast::f32x4;
using vkml::attend_fast::half8;
using vkml::attend_fast::kLog2e;

namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kWaves = kThreads / kWave;
constexpr float kLowest = -__FLT_MAX__;

// The pieces of a row's work that the merge joins: their first row in the
// workspace and how many there are (a slot of their kind apart).
struct Parts {
    uint32_t row, count;  // count: 2 n + (1 for kTileRows rows a slot)
};

struct PagesArgs {
    const float* q;  // [tokens, heads, hd]
    const uint8_t* k;
    const uint8_t* v;
    const int32_t* table;
    float* out;
    Parts* parts;  // [kv_heads, tokens, 2]: of the shared keys, of the own ones
    float2* stats;  // [rows]: m, l
    float* o;       // [rows, hd]
    Batch batch;
    uint32_t page_units;  // 16 bytes each, from a page to the next
    int64_t few_slots, tile_slots;
    uint32_t heads, kv_heads, group, page_shift, pages, table_stride;
    int32_t workgroups_log2;
    uint32_t most_tiles;
    float score_scale;  // what turns q k^T into a score in log2 units; with a soft cap, into tanh's argument
    float softcap, group_inverse;
    Costs costs;
    Window window;         // kWindow
    const uint32_t* seen;  // kTree: [tokens, seen_words]
    uint32_t seen_words;
};

// What a row sees of its sequence's keys up to its own position: all, those before
// the new tokens and its bits' among these, or a window and the sinks.
enum Mask { kCausal, kTree, kWindow };

template <int MASK>
__device__ __forceinline__ Window window_of(const PagesArgs& a) {
    if constexpr (MASK == kWindow) return a.window;
    else return {};
}

// A value that a wave's lanes share, in a scalar register.
__device__ __forceinline__ int32_t uniform(int32_t x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t uniform(int64_t x) {
    return static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(uniform(static_cast<int32_t>(x >> 32)))) << 32 |
                                static_cast<uint32_t>(uniform(static_cast<int32_t>(x))));
}

// The blocks: 16 KiB each of K and V for a workgroup, 8 KiB for a wave alone.
template <typename T, int HD>
struct Block {
    static constexpr bool kF16 = sizeof(T) == 2;
    static constexpr uint32_t kRow = HD * sizeof(T);      // bytes
    static constexpr uint32_t kPieces = kRow / 16;        // 16-byte pieces a row
    static constexpr uint32_t kSteps = kRow / 64;         // operand reads a key
    static constexpr uint32_t kKeys = 16384 / kRow, kTiles = kKeys / 16;
    static constexpr uint32_t kWaveKeys = kKeys / 2, kWaveTiles = kTiles / 2;
    static constexpr uint32_t kDims = HD / 16;            // tiles of 16 dims
    // Where a row's pieces lie in the LDS, so that the lanes of an operand
    // read hit different banks: K's piece p at p ^ swizzle_k(row). V's f16
    // pieces stay in pairs, the 16 dims that a transposed read takes.
    static constexpr uint32_t kRowsABank = kRow < 256 ? 256 / kRow : 1;
    static constexpr uint32_t kMix = kPieces < 16 ? kPieces : 16;
    __device__ static uint32_t swizzle_k(uint32_t row) { return row / kRowsABank % kMix; }
    __device__ static uint32_t swizzle_v(uint32_t row) { return kF16 ? 2 * (row / kRowsABank % (kMix / 2)) : swizzle_k(row); }
};

struct Buffer {
    alignas(16) uint8_t k[16384];
    alignas(16) uint8_t v[16384];
    __device__ __forceinline__ uint8_t* all() { return reinterpret_cast<uint8_t*>(this); }
};

// Where the keys of a tile are (pages.hpp's axis: the lead, then its own).
struct Tile {
    const int32_t* lead_table;  // the table row that the lead is read through
    const int32_t* table;       // and the other keys
    int32_t span, lead;         // the axis' part that the lead takes, its keys
    int32_t lo, from, end;      // of the others: the first read, the first and past the last that count
    uint32_t kvh;
};

// A block's keys: positions key0 on through a table row, those that count.
struct Keys {
    const int32_t* table;
    int32_t key0, from, end;
    bool lead;
};
__device__ __forceinline__ Keys keys_at(const Tile& t, int32_t x) {
    const bool lead = x < t.span;
    return {lead ? t.lead_table : t.table, lead ? x : t.lo + x - t.span, lead ? 0 : t.from, lead ? t.lead : t.end, lead};
}
// A block's keys and the pages that hold them: lane i has the page of the table
// row's entry first + i, -1 past the keys. Neighbouring blocks share a window.
struct Pages {
    Keys keys;
    int32_t ids, first;
};
__device__ __forceinline__ void load_window(const PagesArgs& a, Pages& p) {
    p.first = p.keys.key0 >> a.page_shift;
    const int32_t i = p.first + static_cast<int32_t>(thread_index() % kWave);
    p.ids = -1;
    if (i < (p.keys.end + (1 << a.page_shift) - 1) >> a.page_shift) p.ids = ldg(p.keys.table + i);
}
__device__ __forceinline__ Pages pages_at(const PagesArgs& a, const Tile& t, int32_t x) {
    Pages p{keys_at(t, x), 0, 0};
    load_window(a, p);
    return p;
}
// The block at x, `span` keys, whose predecessor is p's.
__device__ __forceinline__ Pages pages_after(const PagesArgs& a, const Tile& t, const Pages& p, int32_t x, int32_t span) {
    Pages n{keys_at(t, x), p.ids, p.first};
    if (n.keys.lead != p.keys.lead || ((n.keys.key0 + span - 1) >> a.page_shift) - n.first >= static_cast<int32_t>(kWave)) load_window(a, n);
    return n;
}
__device__ __forceinline__ int32_t page_of(const PagesArgs& a, const Pages& p, int32_t key) {
    return __builtin_amdgcn_readlane(p.ids, (key >> a.page_shift) - p.first);
}
// A bit for each of the block's 16-key tiles that is in no page.
template <int TT>
__device__ __forceinline__ uint32_t dead_tiles(const PagesArgs& a, const Pages& p) {
    uint32_t dead = 0;
#pragma unroll
    for (int i = 0; i < TT; ++i) dead |= static_cast<uint32_t>(page_of(a, p, p.keys.key0 + 16 * i)) < a.pages ? 0u : 1u << i;
    return dead;
}
// Where the 16 keys from `key` on of page id are (page 0's for none), from a
// pool's first on.
template <uint32_t ROW>
__device__ __forceinline__ uint64_t offset_of(const PagesArgs& a, uint32_t kvh, int32_t id, int32_t key) {
    const uint32_t held = static_cast<uint32_t>(id) < a.pages ? static_cast<uint32_t>(id) : 0u;
    const uint32_t row = (kvh << a.page_shift) + (static_cast<uint32_t>(key) & ((1u << a.page_shift) - 1));
    return (static_cast<uint64_t>(held) * a.page_units + row * (ROW / 16)) * 16;
}
// pool + offset, in scalar registers as one: the lanes' offsets are added by
// the loads, not to the pool ahead of a loop, where their sums would take two
// registers each.
__device__ __forceinline__ const uint8_t* at_offset(const uint8_t* pool, uint64_t offset) {
    uint64_t p = static_cast<uint64_t>(uniform(static_cast<int64_t>(reinterpret_cast<uint64_t>(pool) + offset)));
    asm volatile("" : "+s"(p));
    return reinterpret_cast<const uint8_t*>(p);
}

// The `bytes` of a pool from `from` on, as loads take them: nothing past them is
// read (of 0 bytes nothing at all: zeros).
__device__ __forceinline__ __amdgpu_buffer_rsrc_t part_of_pool(const uint8_t* from, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(from), 0, static_cast<int>(bytes), 0x00020000);
}
// 16 bytes a lane to `to` (the wave's first lane's) in the LDS. (A buffer load: the
// compiler takes global_load_lds for one that the waits for the LDS count too, and
// every read of the LDS after it for late.)
__device__ __forceinline__ void part_to_lds(__amdgpu_buffer_rsrc_t part, uint32_t lane_offset, uint8_t* to) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(part, (__attribute__((address_space(3))) void*)to, 16, static_cast<int>(lane_offset), 0, 0, 0);
}

// ---------------------------------------------------------------- q

// Eight f32 values as two f16 terms each, two at a time, the remainder by an
// fma that widens the f16 term itself.
__device__ __forceinline__ void split(f32x4 a, f32x4 b, half8& hi, half8& lo) {
    typedef float float2v __attribute__((ext_vector_type(2)));
    typedef _Float16 half2v __attribute__((ext_vector_type(2)));
    uint32_t h[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2v x = i < 2 ? float2v{a[2 * i], a[2 * i + 1]} : float2v{b[2 * i - 4], b[2 * i - 3]};
        h[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(x, half2v));
        float2v r;
        asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r[0]) : "v"(h[i]), "v"(x[0]));
        asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r[1]) : "v"(h[i]), "v"(x[1]));
        l[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(r, half2v));
    }
    hi = __builtin_bit_cast(half8, make_uint4(h[0], h[1], h[2], h[3]));
    lo = __builtin_bit_cast(half8, make_uint4(l[0], l[1], l[2], l[3]));
}

// RT tiles of 16 rows of q as the matrix instructions take them: lane (j, g)
// has row j's pieces 4 s + g. c[rt]: what turns a product with them into a
// score in log2 units (with a soft cap: into tanh's argument), positive and
// finite, so that it makes no NaN of 0 or -inf; the scale's sign is in q.
template <typename T, int HD, int RT>
struct Queries;

// A row as loaded, in the order of the keys' 16-byte pieces.
template <typename T, int HD>
struct RawRow {
    static constexpr int N = HD / 16;
    float4 x[N];
    __device__ __forceinline__ void load(const float* row, uint32_t g) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t at = sizeof(T) == 2 ? 32 * (i / 2) + 8 * g + 4 * (i % 2) : 16 * i + 4 * g;
            x[i] = ldg(reinterpret_cast<const float4*>(row + at));
        }
    }
};

template <int HD, int RT>
struct Queries<_Float16, HD, RT> {
    half8 hi[RT][HD / 32], lo[RT][HD / 32];
    float c[RT];
    __device__ __forceinline__ void take(int rt, const RawRow<_Float16, HD>& raw, float scale) {
        float most = 0.0f;
#pragma unroll
        for (int i = 0; i < raw.N; ++i)
            most = fmaxf(most, fmaxf(fmaxf(fabsf(raw.x[i].x), fabsf(raw.x[i].y)), fmaxf(fabsf(raw.x[i].z), fabsf(raw.x[i].w))));
        const uint2 r16 = swap_rows<16>(__float_as_uint(most));
        most = fmaxf(__uint_as_float(r16.x), __uint_as_float(r16.y));
        const uint2 r32 = swap_rows<32>(__float_as_uint(most));
        most = fmaxf(__uint_as_float(r32.x), __uint_as_float(r32.y));
        // The row's largest value to [1/2, 1), by a power of two that f32 holds:
        // neither term leaves f16's range.
        const int e2 = max(__builtin_amdgcn_frexp_expf(most), -100);
        const float f = __builtin_amdgcn_ldexpf(scale < 0.0f ? -1.0f : 1.0f, -e2);
#pragma unroll
        for (int s = 0; s < HD / 32; ++s) {
            const float4 x = raw.x[2 * s], y = raw.x[2 * s + 1];
            split(f32x4{x.x * f, x.y * f, x.z * f, x.w * f}, f32x4{y.x * f, y.y * f, y.z * f, y.w * f}, hi[rt][s], lo[rt][s]);
        }
        c[rt] = fminf(fmaxf(__builtin_amdgcn_ldexpf(fabsf(scale), e2), __FLT_MIN__), __FLT_MAX__);
    }
    // The products of step s with N of the keys' tiles, in turn, so that an
    // instruction does not wait for the one before it.
    template <int N, int TT>
    __device__ __forceinline__ void score(int s, const uint4 (&k)[N], int t0, f32x4 (&acc)[RT][TT]) const {
#pragma unroll
        for (int term = 0; term < 2; ++term)
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int i = 0; i < N; ++i)
                    acc[rt][t0 + i] =
                        __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, k[i]), term ? lo[rt][s] : hi[rt][s], acc[rt][t0 + i], 0, 0, 0);
    }
};

template <int HD, int RT>
struct Queries<float, HD, RT> {
    float4 x[RT][HD / 16];
    float c[RT];
    __device__ __forceinline__ void take(int rt, const RawRow<float, HD>& raw, float scale) {
        const float sign = scale < 0.0f ? -1.0f : 1.0f;
#pragma unroll
        for (int i = 0; i < raw.N; ++i) x[rt][i] = make_float4(raw.x[i].x * sign, raw.x[i].y * sign, raw.x[i].z * sign, raw.x[i].w * sign);
        c[rt] = fminf(fmaxf(fabsf(scale), __FLT_MIN__), __FLT_MAX__);
    }
    template <int N, int TT>
    __device__ __forceinline__ void score(int s, const uint4 (&k)[N], int t0, f32x4 (&acc)[RT][TT]) const {
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const f32x4 y = __builtin_bit_cast(f32x4, k[i]);
                    const float4 z = x[rt][s];
                    acc[rt][t0 + i] = __builtin_amdgcn_mfma_f32_16x16x4f32(y[e], e == 0 ? z.x : e == 1 ? z.y : e == 2 ? z.z : z.w, acc[rt][t0 + i], 0, 0, 0);
                }
    }
};

// ---------------------------------------------------------------- a block

// What a wave has of RT tiles of 16 rows: lane (j, g) has row j's dims 16 dt +
// 4 g + e, its maximum (of the scores as attend_block has them), and the sum over
// the keys of its own lane.
template <int HD, int RT>
struct Running {
    f32x4 o[RT][HD / 16];
    float m[RT], l[RT];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            m[rt] = kLowest;  // finite: a score of -inf has the weight 2^-inf = 0 whatever came before
            l[rt] = 0.0f;
#pragma unroll
            for (int dt = 0; dt < HD / 16; ++dt) o[rt][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }
};

// The rows' own limits: row j of tile rt sees positions below limit[rt], of
// the lead all.
template <int RT>
struct Limits {
    int32_t limit[RT];
};

// kTree: the position of a piece's sequence's first new token, and what makes a
// row's limit its token.
struct Sees {
    int32_t base, to_token;
};

// The 64 bits from new token b on (b < 0: before the first; keys there are seen) of a
// token's words.
__device__ __forceinline__ uint64_t seen_bits(const PagesArgs& a, int32_t token, int32_t b) {
    const int32_t w = b >> 5, words = static_cast<int32_t>(a.seen_words);
    const uint32_t* row = a.seen + static_cast<uint64_t>(static_cast<uint32_t>(token)) * a.seen_words;
    const auto word = [&](int32_t i) { return i < 0 ? ~0u : i < words ? ldg(row + i) : 0u; };
    const uint64_t two = static_cast<uint64_t>(word(w + 1)) << 32 | word(w);
    return b & 31 ? two >> (b & 31) | static_cast<uint64_t>(word(w + 2)) << (64 - (b & 31)) : two;
}

// Zeros for the infinities and NaN among a masked block's V values, N 16-byte
// pieces a thread; whether any of the thread's were those of keys that count.
template <typename T, uint32_t ROW, int N>
__device__ __forceinline__ bool clear_unbounded(uint8_t* v, uint32_t thread, uint32_t threads, const Keys& keys, uint32_t dead) {
    // One more in the exponent carries into the sign's bit from those alone.
    constexpr uint32_t kOne = sizeof(T) == 2 ? 0x04000400u : 0x00800000u, kSign = sizeof(T) == 2 ? 0x80008000u : 0x80000000u;
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint4 x = *reinterpret_cast<const uint4*>(v + 16 * (thread + i * threads));
        any |= ((x.x & ~kSign) + kOne) | ((x.y & ~kSign) + kOne) | ((x.z & ~kSign) + kOne) | ((x.w & ~kSign) + kOne);
    }
    bool found = false;
    if (!__any(any & kSign)) return found;
#pragma unroll 1
    for (uint32_t i = 16 * thread; i < 16 * N * threads; i += 16 * threads) {
        const uint4 x = *reinterpret_cast<const uint4*>(v + i);
        uint32_t y[4] = {x.x, x.y, x.z, x.w};
        bool here = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t mask = sizeof(T) == 2 ? 0x7C00u : 0x7F800000u;
            uint32_t keep = (y[e] & mask) == mask ? (sizeof(T) == 2 ? 0xFFFF0000u : 0u) : ~0u;
            if (sizeof(T) == 2 && (y[e] >> 16 & mask) == mask) keep &= 0xFFFFu;
            here |= keep != ~0u;
            y[e] &= keep;
        }
        if (here) *reinterpret_cast<uint4*>(v + i) = make_uint4(y[0], y[1], y[2], y[3]);
        const int32_t row = static_cast<int32_t>(i / ROW), key = keys.key0 + row;
        found |= here && key >= keys.from && key < keys.end && !(dead >> (row / 16) & 1);
    }
    return found;
}

// What may move across the order that a loop of reads and products fixes: the
// other VALU, SALU and transcendental instructions.
constexpr int kOnlyAlu = 0x406;

// tanh y: below sqrt(0.4) y + y^3 p(y^2), p of degree 4 fitted to (tanh y / y -
// 1) / y^2 for the least relative error of the whole (5e-9, and f32's rounding);
// above, 1 - 2 / (e^2|y| + 1), whose subtraction loses less than a bit there. No
// division, but the compiler makes the choice a branch, one a score: 256 rows over
// 32768 keys 107 us with a soft cap and 98 without at head_dim 128, 87 and 59 at 64.
__device__ __forceinline__ float tanh_of(float y) {
    const float z = y * y;
    float p = __builtin_fmaf(z, -0.00566077698f, 0.0206019953f);
    p = __builtin_fmaf(z, p, -0.053729225f);
    p = __builtin_fmaf(z, p, 0.133313283f);
    p = __builtin_fmaf(z, p, -0.333332777f);
    const float e = __builtin_amdgcn_exp2f(2.0f * kLog2e * fabsf(y)), far = 1.0f - 2.0f * __builtin_amdgcn_rcpf(e + 1.0f);
    return z < 0.4f ? __builtin_fmaf(y * z, p, y) : __builtin_copysignf(far, y);
}

// What turns a row's maximum as attend_block keeps it into log2 units: f16 caches
// keep the product with the row of q as it is, a soft cap natural units. Within
// f32's range, so that the maxima of two parts can be subtracted.
template <typename T, bool CAP>
__device__ __forceinline__ float in_log2(float m, float c) {
    return __builtin_amdgcn_fmed3f(CAP ? m * kLog2e : sizeof(T) == 2 ? m * c : m, kLowest, __FLT_MAX__);
}

// One block of TT tiles of 16 keys, K in the lane's registers (REGS) or as
// swizzled rows in the LDS, V's rows in the LDS. masked: some rows don't see
// all of its keys. dead: a bit for each tile that is in no page.
//
// A weight is 2^(c (x - m)), the difference taken of the values whose maximum m is:
// its exponent is 0 at the maximum, however large x is. (2^(c x - c m) by an fma is one
// instruction less, but its two products round apart: at scores of 2^25 the
// maximum's weight was up to four times too large, past f16's range.)
template <typename T, int HD, int RT, int TT, bool REGS, bool CAP, int MASK>
__device__ __forceinline__ void attend_block(const PagesArgs& a, const Sees& sees, const Queries<T, HD, RT>& q, const Limits<RT>& lim, const Keys& keys, bool masked, uint32_t dead, float softcap,
                                             const uint4 (*k_regs)[Block<T, HD>::kSteps], const uint8_t* k, const uint8_t* v,
                                             Running<HD, RT>& run) {
#pragma clang fp contract(off)
    using B = Block<T, HD>;
    // (from a fresh thread index, so that the addresses are not kept in
    // registers from one block to the next)
    const uint32_t l = thread_index() % kWave, j = l % 16, g = l / 16;
    const uint32_t k_at = j * B::kRow + 16 * (g ^ B::swizzle_k(j));
    f32x4 s[RT][TT];
    // Where two waves share a SIMD's matrix unit (tiles of many rows), the one
    // in its products goes first: 3 % of a prompt's time.
    if constexpr (!REGS) __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) s[rt][tt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (REGS) {
#pragma unroll
        for (int st = 0; st < static_cast<int>(B::kSteps); ++st) {
            uint4 kk[TT];
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) kk[tt] = k_regs[tt][st];
            q.score(st, kk, 0, s);
        }
    } else {
        // N tiles of a step at a time, the next ones' read before the products.
        constexpr int N = RT == 1 && TT >= 4 ? 4 : 2, kGroups = static_cast<int>(B::kSteps) * TT / N;
        uint4 kk[2][N];
        const auto fetch = [&](int i, uint4 (&to)[N]) {
#pragma unroll
            for (int n = 0; n < N; ++n) to[n] = *reinterpret_cast<const uint4*>(k + (k_at ^ (64 * (i / (TT / N)))) + 16 * (i % (TT / N) * N + n) * B::kRow);
        };
        fetch(0, kk[0]);
#pragma unroll
        for (int i = 0; i < kGroups; ++i) {
            if (i + 1 < kGroups) fetch(i + 1, kk[(i + 1) % 2]);
            __builtin_amdgcn_sched_barrier(kOnlyAlu);
            q.score(i / (TT / N), kk[i % 2], i % (TT / N) * N, s);
            __builtin_amdgcn_sched_barrier(kOnlyAlu);
        }
        __builtin_amdgcn_s_setprio(0);
    }
    constexpr float kShift = B::kF16 ? 14.0f : 0.0f;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        float c = q.c[rt];
        if constexpr (CAP) {
#pragma unroll
            for (int tt = 0; tt < TT; ++tt)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[rt][tt][e] = softcap * tanh_of(s[rt][tt][e] * c);
            c = kLog2e;
        } else if constexpr (!B::kF16) {  // q k^T itself may be near the end of f32's range
#pragma unroll
            for (int tt = 0; tt < TT; ++tt)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[rt][tt][e] *= c;
        }
        if (masked) {
            const int32_t limit = keys.lead ? keys.end : lim.limit[rt];
            uint64_t bits[(TT + 3) / 4];  // of the lane's first key in each four tiles on
            if constexpr (MASK == kTree) {
#pragma unroll
                for (int i = 0; i < (TT + 3) / 4; ++i)
                    bits[i] = keys.lead ? ~0ull : seen_bits(a, lim.limit[rt] + sees.to_token, keys.key0 + 64 * i + 4 * static_cast<int32_t>(g) - sees.base);
            }
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) {
                const int32_t key0 = keys.key0 + 16 * tt + 4 * static_cast<int32_t>(g);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int32_t key = key0 + e;
                    bool hidden = key < keys.from || key >= limit || (dead >> tt & 1);
                    if constexpr (MASK == kTree) hidden |= !(bits[tt / 4] >> (tt % 4 * 16 + e) & 1);
                    if constexpr (MASK == kWindow) hidden |= !keys.lead && key < limit - a.window.keys && key >= a.window.sinks;
                    if (hidden) s[rt][tt][e] = -__builtin_inff();
                }
            }
        }
        float bm = -__builtin_inff();
#pragma unroll
        for (int tt = 0; tt < TT; ++tt)
#pragma unroll
            for (int e = 0; e < 4; ++e) bm = fmaxf(bm, s[rt][tt][e]);
        const uint2 a16 = swap_rows<16>(__float_as_uint(bm));
        bm = fmaxf(__uint_as_float(a16.x), __uint_as_float(a16.y));
        const uint2 a32 = swap_rows<32>(__float_as_uint(bm));
        bm = fmaxf(__uint_as_float(a32.x), __uint_as_float(a32.y));
        constexpr bool kLog2 = !B::kF16 && !CAP;  // in log2 units already
        const float mn = fmaxf(run.m[rt], bm), down = run.m[rt] - mn, factor = __builtin_amdgcn_exp2f(kLog2 ? down : down * c);
        float bs = 0.0f;
#pragma unroll
        for (int tt = 0; tt < TT; ++tt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = s[rt][tt][e] - mn, p = __builtin_amdgcn_exp2f(kLog2 ? x : __builtin_fmaf(x, c, kShift));
                s[rt][tt][e] = p;
                bs += p;
            }
        run.l[rt] = __builtin_fmaf(run.l[rt], factor, bs);
        run.m[rt] = mn;
        // Once the maxima have settled, most blocks leave the output's scale.
        if (__any(factor != 1.0f)) {
#pragma unroll
            for (int dt = 0; dt < HD / 16; ++dt)
#pragma unroll
                for (int e = 0; e < 4; ++e) run.o[rt][dt][e] *= factor;
        }
    }
    if constexpr (B::kF16) {
        typedef __fp16 half4v __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) half4v* lds4;
        // The lane's part of a transposed read of 4 keys by 16 dims a lane
        // group: it points at row 4 g + j / 4, dims 4 (j % 4) on, and gets dim
        // j of the four rows.
        const uint32_t row = 4 * g + j / 4, at = row * B::kRow + 16 * ((j % 4 / 2) ^ B::swizzle_v(row)) + 8 * (j % 2);
        // D tiles of dims at a time; the next ones' read before the products where
        // K comes from the LDS too.
        constexpr int D = REGS ? (HD == 128 ? 8 : 4) : RT == 1 ? 4 : 2, kAt = HD / 16 / D, kGroups = TT / 2 * kAt;
        const auto fetch = [&](int i, half8 (&to)[D]) {
#pragma unroll
            for (int d = 0; d < D; ++d) {
                const uint8_t* from = v + (at ^ (32 * (i % kAt * D + d))) + 32 * (i / kAt) * B::kRow;
                const auto x = __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds4)(from));
                const auto y = __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds4)(from + 16 * B::kRow));
                const uint2 xx = __builtin_bit_cast(uint2, x), yy = __builtin_bit_cast(uint2, y);
                to[d] = __builtin_bit_cast(half8, make_uint4(xx.x, xx.y, yy.x, yy.y));
            }
        };
        half8 ph[RT], pl[RT], vv[REGS ? 1 : 2][D];
        if constexpr (!REGS) {
            __builtin_amdgcn_s_setprio(1);
            fetch(0, vv[0]);
        }
#pragma unroll
        for (int i = 0; i < kGroups; ++i) {
            if (i % kAt == 0) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) split(s[rt][2 * (i / kAt)], s[rt][2 * (i / kAt) + 1], ph[rt], pl[rt]);
            }
            half8(&now)[D] = vv[REGS ? 0 : i % 2];
            if constexpr (REGS) fetch(i, now);
            else if (i + 1 < kGroups) fetch(i + 1, vv[(i + 1) % 2]);
            if constexpr (!REGS) __builtin_amdgcn_sched_barrier(kOnlyAlu);
#pragma unroll
            for (int term = 0; term < 2; ++term)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int d = 0; d < D; ++d) {
                        f32x4& o = run.o[rt][i % kAt * D + d];
                        o = __builtin_amdgcn_mfma_f32_16x16x32_f16(now[d], term ? pl[rt] : ph[rt], o, 0, 0, 0);
                    }
            if constexpr (!REGS) __builtin_amdgcn_sched_barrier(kOnlyAlu);
        }
        if constexpr (!REGS) __builtin_amdgcn_s_setprio(0);
    } else {
        // Instruction e of a tile takes keys 4 g + e: V's element of dim j.
#pragma unroll
        for (int tt = 0; tt < TT; ++tt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t row = 16 * tt + 4 * g + e;
#pragma unroll
                for (int dt = 0; dt < HD / 16; ++dt) {
                    const float vv = *reinterpret_cast<const float*>(v + (row * B::kRow + 16 * ((4 * dt + j / 4) ^ B::swizzle_v(row)) + 4 * (j % 4)));
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) run.o[rt][dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(vv, s[rt][tt][e], run.o[rt][dt], 0, 0, 0);
                }
            }
    }
}

// ---------------------------------------------------------------- pieces

// A piece of a tile: [x0, x1) of its keys' axis, rows from token0 on.
struct Piece {
    Tile tile;
    int32_t x0, x1;
    int32_t token0, tokens;
    int32_t limit0;    // the position below which the first token sees
    Sees sees;
    bool causal;       // and each further token one more
    bool whole;        // all of its rows' work: the output itself
    int64_t slot_row;  // else the rows of the workspace, -1 for none
};

// The LDS of the workgroup's waves is theirs together from here on: what they
// wrote there is there, and what they read is read (unlike __syncthreads(),
// stores to memory need not have arrived).
__device__ __forceinline__ void lds_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Every load of the wave has landed, those to the LDS among them. (The builtin:
// what asm waits for, the compiler would wait for again.)
__device__ __forceinline__ void loads_landed() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    asm volatile("" ::: "memory");
}
// And what the wave has read from the LDS is read, so that loads into it may be
// issued: where no barrier says so.
__device__ __forceinline__ void loads_and_reads_landed() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
    asm volatile("" ::: "memory");
}

__device__ __forceinline__ float lanes_sum(float v) {  // over a row's four lanes
    const uint2 l16 = swap_rows<16>(__float_as_uint(v));
    v = __uint_as_float(l16.x) + __uint_as_float(l16.y);
    const uint2 l32 = swap_rows<32>(__float_as_uint(v));
    return __uint_as_float(l32.x) + __uint_as_float(l32.y);
}

// The token of row r < 128 of a tile: r / group, (r + 1/2) / group being at
// least 1/256 from a whole number.
__device__ __forceinline__ uint32_t token_of(const PagesArgs& a, uint32_t r) { return static_cast<uint32_t>((static_cast<float>(r) + 0.5f) * a.group_inverse); }

template <typename T, int HD, int RT>
__device__ __forceinline__ void load_rows(const PagesArgs& a, const Piece& p, uint32_t first_row, RawRow<T, HD> (&raw)[RT], Limits<RT>& lim) {
    const uint32_t l = thread_index() % kWave, j = l % 16, g = l / 16, rows = p.tokens * a.group;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const uint32_t r = min(first_row + 16 * rt + j, rows - 1), t = token_of(a, r);
        raw[rt].load(a.q + (static_cast<uint64_t>(p.token0 + t) * a.heads + p.tile.kvh * a.group + r - t * a.group) * HD, g);
        lim.limit[rt] = p.causal ? p.limit0 + static_cast<int32_t>(t) : p.limit0;
    }
}

// Where row r of a piece goes, and what its values are multiplied by there: the
// output, divided by the sum of weights l, or the workspace, with (m, l) beside
// it. null: nowhere.
template <int HD>
__device__ __forceinline__ float* row_to(const PagesArgs& a, const Piece& p, uint32_t r, bool first_lane, float m, float l, float& times) {
    if (p.whole) {
        const uint32_t t = token_of(a, r);
        times = l == 0.0f ? 0.0f : 1.0f / l;
        return a.out + (static_cast<uint64_t>(p.token0 + t) * a.heads + p.tile.kvh * a.group + r - t * a.group) * HD;
    }
    times = 1.0f;
    if (p.slot_row < 0) return nullptr;
    if (first_lane) stg(a.stats + p.slot_row + r, make_float2(m, l));
    return a.o + (p.slot_row + r) * HD;
}

// Whether some of a tile's rows don't see all of a block of `span` keys.
template <int MASK>
__device__ __forceinline__ bool is_masked(const PagesArgs& a, const Piece& p, const Keys& keys, int32_t span, uint32_t dead) {
    const bool cut = keys.key0 < keys.from || keys.key0 + span > (keys.lead ? keys.end : MASK == kTree ? p.sees.base : p.limit0) || dead;
    if constexpr (MASK == kWindow) return cut || (!keys.lead && keys.key0 < p.limit0 + p.tokens - 1 - a.window.keys && keys.key0 + span > a.window.sinks);
    else return cut;
}

// The infinities and NaN of V in a piece's masked blocks, which the products
// have left out, for the rows that see them, where the workgroup has stored
// those: a row's value there is their sum, whatever the finite ones are.
template <typename T, int HD, int MASK>
__device__ __forceinline__ void add_unbounded(const PagesArgs& a, const Piece& p) {
    using B = Block<T, HD>;
    if (!p.whole && p.slot_row < 0) return;
    const uint32_t thread = thread_index(), dim = thread % HD, rows = p.tokens * a.group;
    __syncthreads();  // the rows are stored
    for (int32_t x = p.x0; x < p.x1; x += B::kKeys) {
        const Pages at = pages_at(a, p.tile, x);
        if (!is_masked<MASK>(a, p, at.keys, B::kKeys, dead_tiles<B::kTiles>(a, at))) continue;
#pragma unroll 1
        for (int32_t key = max(at.keys.key0, at.keys.from); key < min(at.keys.key0 + static_cast<int32_t>(B::kKeys), at.keys.end); ++key) {
            const int32_t id = ld_scalar_i32(at.keys.table + (key >> a.page_shift));
            if (static_cast<uint32_t>(id) >= a.pages) continue;
            const float v = static_cast<float>(reinterpret_cast<const T*>(a.v + offset_of<B::kRow>(a, p.tile.kvh, id, key))[dim]);
            if (fabsf(v) <= __FLT_MAX__) continue;
#pragma unroll 1
            for (uint32_t r = thread / HD; r < rows; r += kThreads / HD) {
                const uint32_t t = token_of(a, r);
                const int32_t limit = p.limit0 + static_cast<int32_t>(t);
                if (!at.keys.lead && p.causal && key >= limit) continue;
                if constexpr (MASK == kTree) {
                    if (!at.keys.lead && !(seen_bits(a, p.token0 + static_cast<int32_t>(t), key - p.sees.base) & 1)) continue;
                }
                if constexpr (MASK == kWindow) {
                    if (!at.keys.lead && key < limit - a.window.keys && key >= a.window.sinks) continue;
                }
                float* to = p.whole ? a.out + (static_cast<uint64_t>(p.token0 + t) * a.heads + p.tile.kvh * a.group + r - t * a.group) * HD + dim
                                    : a.o + (p.slot_row + r) * HD + dim;
                stg(to, ldg(to) + v);
            }
        }
    }
}

// At most 16 rows: each wave by itself over blocks of kWaveKeys keys in turn.
template <typename T, int HD, bool CAP, int MASK>
__device__ __forceinline__ void few_rows(const PagesArgs& a, const Piece& p, Buffer& buf0, Buffer& buf1) {
    using B = Block<T, HD>;
    constexpr int TT = B::kWaveTiles;
    const uint32_t thread = thread_index(), w = __builtin_amdgcn_readfirstlane(thread / kWave), l = thread % kWave, j = l % 16, g = l / 16;
    Queries<T, HD, 1> q;
    q.c[0] = 1.0f;  // where there are no keys
    Limits<1> lim{{p.limit0}};
    Running<HD, 1> run;
    run.clear();
    constexpr int32_t kStep = kWaves * B::kWaveKeys, kSpan = B::kWaveKeys;
    int32_t x = p.x0 + static_cast<int32_t>(w) * kSpan;
    const auto issue = [&](const Pages& at, uint4 (&k)[TT][B::kSteps], uint8_t* to) {
        __amdgpu_buffer_rsrc_t k_part[TT], v_part[TT];
#pragma unroll
        for (int i = 0; i < TT; ++i) {
            const int32_t key = at.keys.key0 + 16 * i;
            const uint64_t part = offset_of<B::kRow>(a, p.tile.kvh, page_of(a, at, key), key);
            k_part[i] = part_of_pool(at_offset(a.k, part), 16 * B::kRow);
            v_part[i] = part_of_pool(at_offset(a.v, part), 16 * B::kRow);
        }
#pragma unroll
        for (int tt = 0; tt < TT; ++tt)
#pragma unroll
            for (int s = 0; s < static_cast<int>(B::kSteps); ++s)
                k[tt][s] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(k_part[tt], static_cast<int>(j * B::kRow + 64 * s + 16 * g), 0, 0));
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) {
            const uint32_t u = 64 * i + l, row = u / B::kPieces;
            part_to_lds(v_part[64 * i / B::kPieces / 16], row % 16 * B::kRow + 16 * (u % B::kPieces ^ B::swizzle_v(row)), to + 1024 * i);
        }
    };
    // Values of V that are not finite in blocks that some rows see less of than
    // others are left out of the product and added at the end.
    bool unbounded = false;
    // The buffers are variables of their own, used by turns, and a load into each
    // (for the second, of nothing) is on every way to the loop: that is what it takes
    // for the compiler not to let reads of one wait for the loads into the other.
    const auto blocks = [&](uint8_t* v0, uint8_t* v1) {
        uint4 k0[TT][B::kSteps], k1[TT][B::kSteps];
        RawRow<T, HD> raw[1];
        Pages cur = pages_at(a, p.tile, x);
        load_rows(a, p, 0, raw, lim);
        part_to_lds(part_of_pool(a.v, 0), 0, v1);
        issue(cur, k0, v0);
        Pages nxt = pages_after(a, p.tile, cur, x + kStep, kSpan);
        q.take(0, raw[0], a.score_scale);
        const auto block = [&](uint4 (&k)[TT][B::kSteps], uint8_t* here, uint4 (&k_next)[TT][B::kSteps], uint8_t* there) {
            loads_and_reads_landed();  // this block's, the next one's pages; the last block's reads
            const uint32_t dead = dead_tiles<TT>(a, cur);
            if (x + kStep < p.x1) issue(nxt, k_next, there);
            const Pages after = pages_after(a, p.tile, nxt, x + 2 * kStep, kSpan);
            const bool masked = is_masked<MASK>(a, p, cur.keys, kSpan, dead);
            if (masked) unbounded |= clear_unbounded<T, B::kRow, 8>(here, l, kWave, cur.keys, dead);
            attend_block<T, HD, 1, TT, true, CAP, MASK>(a, p.sees, q, lim, cur.keys, masked, dead, a.softcap, k, nullptr, here, run);
            cur = nxt;
            nxt = after;
            x += kStep;
        };
        for (;;) {
            block(k0, v0, k1, v1);
            if (x >= p.x1) break;
            block(k1, v1, k0, v0);
            if (x >= p.x1) break;
        }
    };
    if (x < p.x1) blocks(buf0.all() + 8192 * w, buf1.all() + 8192 * w);
    // The waves' parts join in the LDS, rows HD + 4 floats apart.
    const float sum = lanes_sum(run.l[0]);
    constexpr uint32_t kStride = HD + 4;
    // [16][kStride] of a wave, two waves a buffer; then [waves][16] of (m, l)
    const auto part = [&](uint32_t wave) { return reinterpret_cast<float*>(wave < 2 ? buf0.all() : buf1.all()) + wave % 2 * 16 * kStride; };
    float2* ml = reinterpret_cast<float2*>(part(0) + 2 * 16 * kStride);
    uint32_t* found = reinterpret_cast<uint32_t*>(ml + kWaves * 16);  // [waves]
    const bool mine = __any(unbounded);
    lds_barrier();
#pragma unroll
    for (int dt = 0; dt < HD / 16; ++dt)
        *reinterpret_cast<f32x4*>(part(w) + j * kStride + 16 * dt + 4 * g) = run.o[0][dt];
    if (g == 0) ml[16 * w + j] = make_float2(in_log2<T, CAP>(run.m[0], q.c[0]), sum);
    if (l == 0) found[w] = mine;
    lds_barrier();
    const uint32_t r = thread / 16;
    if (r < p.tokens * a.group) {
        float m = kLowest, f[kWaves], lsum = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < kWaves; ++i) m = fmaxf(m, ml[16 * i + r].x);
#pragma unroll
        for (uint32_t i = 0; i < kWaves; ++i) {
            f[i] = __builtin_amdgcn_exp2f(ml[16 * i + r].x - m);
            lsum += f[i] * ml[16 * i + r].y;
        }
        float times;
        float* to = row_to<HD>(a, p, r, thread % 16 == 0, m, lsum, times);
#pragma unroll
        for (uint32_t d = 0; d < HD / 64; ++d) {
            const uint32_t dim = 64 * d + 4 * (thread % 16);
            f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (uint32_t i = 0; i < kWaves; ++i) {
                const f32x4 y = *reinterpret_cast<const f32x4*>(part(i) + r * kStride + dim);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] += f[i] * y[e];
            }
            if (to) stg(reinterpret_cast<float4*>(to + dim), make_float4(o[0] * times, o[1] * times, o[2] * times, o[3] * times));
        }
    }
    if (uniform(static_cast<int32_t>(found[0] | found[1] | found[2] | found[3]))) add_unbounded<T, HD, MASK>(a, p);
}

// Many rows: RT tiles of 16 a wave, the blocks shared.
template <typename T, int HD, int RT, bool CAP, int MASK>
__device__ __forceinline__ void many_rows(const PagesArgs& a, const Piece& p, Buffer& buf0, Buffer& buf1) {
    using B = Block<T, HD>;
    constexpr int TT = B::kTiles;
    constexpr int32_t kSpan = B::kKeys;
    const uint32_t thread = thread_index(), w = __builtin_amdgcn_readfirstlane(thread / kWave), l = thread % kWave, j = l % 16, g = l / 16;
    const uint32_t rows = p.tokens * a.group, first = 16 * RT * w;
    Queries<T, HD, RT> q;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) q.c[rt] = 1.0f;  // where there are no keys
    Limits<RT> lim;
    Running<HD, RT> run;
    run.clear();
    const auto issue = [&](const Pages& at, uint8_t* to) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t u = i * kThreads + thread, row = u / B::kPieces;
            // the first of the 16 keys that the wave's i-th load is in
            const int32_t key = at.keys.key0 + static_cast<int32_t>((i * kThreads + w * kWave) / B::kPieces / 16 * 16);
            const uint64_t part = offset_of<B::kRow>(a, p.tile.kvh, page_of(a, at, key), key);
            uint8_t* k_to = to + 16 * (i * kThreads + w * kWave);
            part_to_lds(part_of_pool(at_offset(a.k, part), 16 * B::kRow), row % 16 * B::kRow + 16 * (u % B::kPieces ^ B::swizzle_k(row)), k_to);
            part_to_lds(part_of_pool(at_offset(a.v, part), 16 * B::kRow), row % 16 * B::kRow + 16 * (u % B::kPieces ^ B::swizzle_v(row)), k_to + sizeof buf0.k);
        }
    };
    int32_t x = p.x0;
    // (Waves without rows, and blocks past all that a wave's rows see, are not left
    // out: the sums would be copied where the ways join, 64 registers twice a
    // block, and the workgroup's other waves are waited for in any case.)
    bool unbounded = false;
    const auto blocks = [&](uint8_t* b0, uint8_t* b1) {  // as in few_rows
        RawRow<T, HD> raw[RT];
        Pages cur = pages_at(a, p.tile, x);
        load_rows(a, p, first, raw, lim);
        part_to_lds(part_of_pool(a.v, 0), 0, b1 + 1024 * w);
        issue(cur, b0);
        Pages nxt = pages_after(a, p.tile, cur, x + kSpan, kSpan);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) q.take(rt, raw[rt], a.score_scale);
        const auto block = [&](uint8_t* here, uint8_t* there) {
            loads_landed();
            lds_barrier();  // every wave's loads have landed, and the other buffer is read no more
            const uint32_t dead = dead_tiles<TT>(a, cur);
            if (x + kSpan < p.x1) issue(nxt, there);
            const Pages after = pages_after(a, p.tile, nxt, x + 2 * kSpan, kSpan);
            const bool masked = is_masked<MASK>(a, p, cur.keys, kSpan, dead);
            if (masked) {
                unbounded |= clear_unbounded<T, B::kRow, 4>(here + sizeof buf0.k, thread, kThreads, cur.keys, dead);
                lds_barrier();
            }
            attend_block<T, HD, RT, TT, false, CAP, MASK>(a, p.sees, q, lim, cur.keys, masked, dead, a.softcap, nullptr, here, here + sizeof buf0.k, run);
            cur = nxt;
            nxt = after;
            x += kSpan;
        };
        for (;;) {
            block(b0, b1);
            if (x >= p.x1) break;
            block(b1, b0);
            if (x >= p.x1) break;
        }
    };
    if (x < p.x1) blocks(buf0.all(), buf1.all());
    const bool found = __syncthreads_or(unbounded);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const float sum = lanes_sum(run.l[rt]);
        const uint32_t r = first + 16 * rt + j;
        if (r < rows) {
            float times;
            float* to = row_to<HD>(a, p, r, g == 0, in_log2<T, CAP>(run.m[rt], q.c[rt]), sum, times);
            if (to) {
#pragma unroll
                for (int dt = 0; dt < HD / 16; ++dt) {
                    const f32x4 o = run.o[rt][dt];
                    stg(reinterpret_cast<float4*>(to + 16 * dt + 4 * g), make_float4(o[0] * times, o[1] * times, o[2] * times, o[3] * times));
                }
            }
        }
    }
    if (found) add_unbounded<T, HD, MASK>(a, p);
}

// ---------------------------------------------------------------- the launch

// Segments as the workgroup keeps them, the first kThreads of a batch.
struct Kept {
    int32_t v[10];
};
__device__ __forceinline__ Kept kept(const Segment& s) {
    return {{s.row, s.lead_row, s.lead, s.token0, s.n, s.from, s.base, s.tiles, s.step, (s.few ? 1 : 0) + (s.shared ? 2 : 0)}};
}
__device__ __forceinline__ Segment taken(const Kept& k, Costs costs, Window window) {
    Segment s;
    s.row = uniform(k.v[0]);
    s.lead_row = uniform(k.v[1]);
    s.lead = uniform(k.v[2]);
    s.token0 = uniform(k.v[3]);
    s.n = uniform(k.v[4]);
    s.from = uniform(k.v[5]);
    s.base = uniform(k.v[6]);
    s.tiles = uniform(k.v[7]);
    s.step = uniform(k.v[8]);
    const int32_t flags = uniform(k.v[9]);
    s.few = flags & 1;
    s.shared = flags & 2;
    s.key_cost = s.few ? costs.few_key : costs.tile_key;
    s.own_cost = s.few ? costs.few_own : costs.tile_own;
    s.set(window);
    return s;
}

struct Scratch {
    int64_t cost[kThreads];    // inclusive sums of a wave
    int64_t counts[kThreads];  // of tiles: few rows' in the low half, others' in the high
    Kept segments[kThreads];
};

// Where a workgroup's part begins, and the whole of the work.
struct Place {
    int64_t cost;          // all KV heads'
    int64_t unit;          // the part's first, from the segment's on
    int32_t kvh, segment;  // the first that the part has work of
    int32_t few, tiles;    // tiles of each kind before the segment
    int32_t part, parts_log2;
};

// Every thread sums its run of segments (one, up to kThreads of them), and the
// waves' sums place the part's first unit among them.
template <int MASK>
__device__ __forceinline__ bool find_place(const PagesArgs& a, Place& out, Scratch& lds) {
    const int32_t n = a.batch.groups + a.batch.seqs, each = n <= static_cast<int32_t>(kThreads) ? 1 : (n + kThreads - 1) / kThreads;
    const int32_t t = static_cast<int32_t>(threadIdx.x), i0 = t * each, i1 = min(i0 + each, n);
    int64_t cost = 0, counts = 0;
    for (int32_t i = i0; i < i1; ++i) {
        const Segment s = segment(a.batch, a.group, a.costs, i, window_of<MASK>(a));
        if (each == 1) lds.segments[t] = kept(s);
        cost += s.cost();
        counts += s.few ? static_cast<int64_t>(s.tiles) : static_cast<int64_t>(s.tiles) << 32;
        if (counts >> 32 > a.most_tiles) break;  // and more in all: nothing is done below
    }
    lds.cost[t] = inclusive_sum(cost);
    lds.counts[t] = inclusive_sum(counts);
    lds_barrier();
    const uint32_t l = threadIdx.x % kWave;
    int64_t sums[kWaves], per_head = 0, counts_head = 0;
#pragma unroll
    for (uint32_t i = 0; i < kWaves; ++i) {
        sums[i] = uniform(lds.cost[kWave * i + kWave - 1]);
        per_head += sums[i];
        counts_head += uniform(lds.counts[kWave * i + kWave - 1]);
    }
    out.cost = per_head * a.kv_heads;
    out.parts_log2 = parts_log2(out.cost, a.workgroups_log2);
    // dealt to the XCDs round-robin: the parts of one are neighbours
    const int32_t b = static_cast<int32_t>(blockIdx.x);
    if (out.cost == 0 || b >> out.parts_log2 || static_cast<uint64_t>(counts_head) >> 32 > a.most_tiles) return false;
    out.part = (b % 8 << (out.parts_log2 - 3)) + b / 8;
    out.kvh = static_cast<int32_t>(static_cast<int64_t>(a.kv_heads) * out.part >> out.parts_log2);
    const int64_t unit = part_start(out.cost, out.parts_log2, out.part) - out.kvh * per_head;
    int64_t off = 0, before = 0;  // of the wave whose segments hold the unit
    uint32_t w = 0;
#pragma unroll
    for (uint32_t i = 0; i + 1 < kWaves; ++i)
        if (w == i && unit >= off + sums[i]) {
            off += sums[i];
            before += uniform(lds.counts[kWave * i + kWave - 1]);
            ++w;
        }
    const int64_t mine = lds.cost[kWave * w + l], my_counts = lds.counts[kWave * w + l];
    const uint32_t lane = static_cast<uint32_t>(__builtin_ctzll(__ballot(off + mine > unit)));
    if (lane > 0) {
        const auto from_lane = [&](int64_t v) {
            return static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v >> 32), lane - 1))) << 32 |
                                        static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), lane - 1)));
        };
        off += from_lane(mine);
        before += from_lane(my_counts);
    }
    int32_t i = static_cast<int32_t>(kWave * w + lane) * each;
    for (; each > 1; ++i) {
        const Segment s = segment(a.batch, a.group, a.costs, i, window_of<MASK>(a));
        if (unit < off + s.cost()) break;
        off += s.cost();
        before += s.few ? static_cast<int64_t>(s.tiles) : static_cast<int64_t>(s.tiles) << 32;
    }
    out.segment = i;
    out.unit = unit - off;
    out.few = static_cast<int32_t>(before) + out.kvh * static_cast<int32_t>(counts_head);
    out.tiles = static_cast<int32_t>(before >> 32) + out.kvh * static_cast<int32_t>(counts_head >> 32);
    return true;
}

template <typename T, int HD, bool CAP, int MASK>
__global__ void __launch_bounds__(kThreads, 2) k_attend_pages(PagesArgs a) {
    using B = Block<T, HD>;
    __shared__ Buffer buf0, buf1;  // apart: the compiler then knows that they are
    __shared__ Scratch scratch;
    Place at;
    if (!find_place<MASK>(a, at, scratch)) return;
    const int64_t part_end = part_start(at.cost, at.parts_log2, at.part + 1);
    const int32_t segments = a.batch.groups + a.batch.seqs;
    int32_t kvh = at.kvh, i = at.segment, few = at.few, tiles = at.tiles, tile = 0;
    // The part's ends, from the segment's (then the tile's) first unit on.
    int64_t begin = at.unit, end = begin + part_end - part_start(at.cost, at.parts_log2, at.part);
    bool again = false;
    for (;;) {
        const Segment s = segments <= static_cast<int32_t>(kThreads) ? taken(scratch.segments[i], a.costs, window_of<MASK>(a)) : segment(a.batch, a.group, a.costs, i, window_of<MASK>(a));
        tile = 0;
        if (begin > 0 && s.tiles > 1) {
            tile = s.tile_at(begin);
            const int64_t before = s.before(tile);
            begin -= before;
            end -= before;
        }
        for (; tile < s.tiles; ++tile) {
            const int32_t keys = s.keys(tile), cost = s.tile_cost(tile);
            const int32_t from = snap(begin, s, cost), to = snap(end, s, cost);
            begin = 0;
            if (to == 0) return;  // the next part's
            const int64_t start = part_end - end;  // the tile's, in the whole
            end -= cost;
            if (from == cost) continue;  // the part before has taken the rest
            const bool ends = to == cost;
            Piece p;
            p.x0 = cut(from, s, keys, B::kKeys);
            p.x1 = ends ? keys : cut(to, s, keys, B::kKeys);
            const Segment::Where in = s.where(tile);
            p.tile = {a.table + static_cast<uint64_t>(s.lead_row) * a.table_stride, a.table + static_cast<uint64_t>(s.row) * a.table_stride,
                      in.span, in.lead, in.lo, in.from, in.end, static_cast<uint32_t>(kvh)};
            p.token0 = s.token0 + tile * s.step;
            p.tokens = s.tile_n(tile);
            p.limit0 = s.limit(tile * s.step);
            p.sees = {s.shared ? p.limit0 : s.lo() + s.base, p.token0 - p.limit0};
            p.causal = !s.shared;
            // the rows' own keys are all there is, but for a shared segment's
            const bool all = !s.shared && s.from == s.lead;
            p.whole = all && ends && from == 0;
            const int32_t slot = at.part + (s.few ? few : tiles + tile);
            p.slot_row = s.few ? (slot < a.few_slots ? static_cast<int64_t>(slot) * kFewRows : -1)
                               : (slot < a.tile_slots ? a.few_slots * kFewRows + static_cast<int64_t>(slot) * kTileRows : -1);
            // The tile's first piece tells the merge where they all are, and
            // where there is no shared segment, that there is none.
            if (from == 0) {
                const uint32_t count = p.whole || p.slot_row < 0 ? 0 : ends ? 1 : pieces_of(at.cost, at.parts_log2, s, start, cost, at.part);
                for (uint32_t k = threadIdx.x; k < static_cast<uint32_t>(p.tokens); k += kThreads) {
                    Parts* to = a.parts + (static_cast<uint64_t>(kvh) * a.batch.tokens + p.token0 + k) * 2;
                    const uint2 mine = make_uint2(static_cast<uint32_t>(p.slot_row + k * a.group), 2 * count + (s.few ? 0u : 1u));
                    if (all) stg(reinterpret_cast<uint4*>(to), make_uint4(0, 0, mine.x, mine.y));
                    else stg(reinterpret_cast<uint2*>(to + (s.shared ? 0 : 1)), mine);
                }
            }
            if (again) lds_barrier();  // the last piece's LDS
            again = true;
            if (s.few) few_rows<T, HD, CAP, MASK>(a, p, buf0, buf1);
            else if (p.tokens * a.group <= kTileRows / 2) many_rows<T, HD, 1, CAP, MASK>(a, p, buf0, buf1);
            else many_rows<T, HD, 2, CAP, MASK>(a, p, buf0, buf1);
            if (end <= 0) return;
        }
        (s.few ? few : tiles) += s.tiles;
        if (++i == segments) {
            i = 0;
            if (++kvh == static_cast<int32_t>(a.kv_heads)) return;
        }
    }
}

// What the merge joins for a (token, KV head): its pieces' rows in the
// workspace, those of the shared keys first.
struct Joins {
    int64_t row0, row1;
    uint32_t n0, n, step0, step1;
    __device__ __forceinline__ int64_t row(uint32_t p) const {
        return p < n0 ? row0 + static_cast<int64_t>(p) * step0 : row1 + static_cast<int64_t>(p - n0) * step1;
    }
};
// (none where there is nothing to join, or for rows of no sequence)
__device__ __forceinline__ Joins joins_of(const PagesArgs& a, uint32_t at, int64_t ws_rows) {  // at: [kv_heads, tokens]
    const uint4 both = ldg(reinterpret_cast<const uint4*>(a.parts + static_cast<uint64_t>(at) * 2));
    const int32_t t = static_cast<int32_t>(at % a.batch.tokens), first = a.batch.start(0), end = a.batch.start(a.batch.seqs);
    const uint32_t n0 = both.y / 2, n = n0 + both.w / 2;
    Joins j{both.x, both.z, n0, n, static_cast<uint32_t>(both.y & 1 ? kTileRows : kFewRows), static_cast<uint32_t>(both.w & 1 ? kTileRows : kFewRows)};
    const int64_t last = ws_rows - a.group;
    if (n == 0 || t < first || t >= end || j.row(n - 1) > last || (n0 && j.row(n0 - 1) > last)) j.n = 0;
    return j;
}

// Dims N l .. N l + N - 1 of a row.
template <int N>
__device__ __forceinline__ void load_dims(float (&x)[N], const float* row, uint32_t l) {
    if constexpr (N == 2) {
        const float2 y = ldg(reinterpret_cast<const float2*>(row) + l);
        x[0] = y.x, x[1] = y.y;
    } else {
        x[0] = ldg(row + l);
    }
}
template <int N>
__device__ __forceinline__ void store_dims(float* row, const float (&x)[N], uint32_t l) {
    if constexpr (N == 2) stg(reinterpret_cast<float2*>(row) + l, make_float2(x[0], x[1]));
    else stg(row + l, x[0]);
}

// Joins the pieces of the rows that are in several, few of them: a workgroup a
// row, the pieces' (m, l) a lane each, then each wave its share of their o,
// HD / 64 dims a lane, kFlight pieces in flight.
template <int HD>
__global__ void __launch_bounds__(kThreads) k_attend_pages_merge(PagesArgs a, int64_t ws_rows) {
    constexpr int N = HD / 64, kFlight = 8;
    __shared__ float s_o[kWaves][HD];
    const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), l = threadIdx.x % kWave;
    const uint32_t at = blockIdx.x / a.group, head = blockIdx.x % a.group;
    const Joins j = joins_of(a, at, ws_rows);
    if (j.n == 0) return;
    float m = kLowest, lsum = 0.0f, o[N] = {};
    for (uint32_t p0 = 0; p0 < j.n; p0 += kWave) {
        const uint32_t many = min(j.n - p0, static_cast<uint32_t>(kWave));
        const float2 ml = l < many ? ldg(a.stats + j.row(p0 + l) + head) : make_float2(kLowest, 0.0f);
        // the first pieces' o before their weights are known
        float x[kFlight][N];
        const auto fetch = [&](uint32_t k0) {
#pragma unroll
            for (uint32_t k = 0; k < kFlight; ++k)  // past the last: its o again, not used
                load_dims<N>(x[k], a.o + (j.row(p0 + min(k0 + kWaves * k, many - 1)) + head) * HD, l);
        };
        fetch(w);
        const float mn = fmaxf(m, wave_max(ml.x)), factor = __builtin_amdgcn_exp2f(m - mn), weight = __builtin_amdgcn_exp2f(ml.x - mn);
        lsum = lsum * factor + wave_sum(l < many ? weight * ml.y : 0.0f);
        m = mn;
#pragma unroll
        for (int i = 0; i < N; ++i) o[i] *= factor;
        for (uint32_t k0 = w; k0 < many; k0 += kWaves * kFlight) {
            if (k0 >= kWaves) fetch(k0);
#pragma unroll
            for (uint32_t k = 0; k < kFlight; ++k) {
                if (k0 + kWaves * k >= many) break;
                const float f = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(weight), k0 + kWaves * k));
#pragma unroll
                for (int i = 0; i < N; ++i) o[i] += f * x[k][i];
            }
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) s_o[w][N * l + i] = o[i];
    __syncthreads();
    if (threadIdx.x < HD) {
        float y = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < kWaves; ++i) y += s_o[i][threadIdx.x];
        const uint32_t t = at % a.batch.tokens, kvh = at / a.batch.tokens;
        stg(a.out + (static_cast<uint64_t>(t) * a.heads + kvh * a.group + head) * HD + threadIdx.x, y * (lsum == 0.0f ? 0.0f : 1.0f / lsum));
    }
}

// The same for many rows, most of them in one piece or two: a wave up to four
// query heads of a (token, KV head), (m, l) of 16 pieces of each in the lanes,
// two pieces of each head in flight.
template <int HD>
__global__ void __launch_bounds__(kThreads) k_attend_pages_merge_many(PagesArgs a, int64_t ws_rows) {
    constexpr int N = HD / 64, kHeads = 4, kLanes = kWave / kHeads, kFlight = 2;
    const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), l = threadIdx.x % kWave;
    const uint32_t splits = (a.group + kHeads - 1) / kHeads;
    const uint32_t item = (blockIdx.y * gridDim.x + blockIdx.x) * kWaves + w;  // less than 2^31 + 2^25
    const uint32_t at = item / splits, head = item % splits * kHeads;
    if (at >= a.kv_heads * static_cast<uint32_t>(a.batch.tokens)) return;
    const Joins j = joins_of(a, at, ws_rows);
    if (j.n == 0) return;
    const uint32_t last = min(head + kHeads, a.group) - 1;  // heads past it: its work again, not stored
    const uint32_t mine = min(head + l / kLanes, last);
    float m = kLowest, lsum = 0.0f, o[kHeads][N] = {};  // m and l of the lane's head
    for (uint32_t p0 = 0; p0 < j.n; p0 += kLanes) {
        const uint32_t many = min(j.n - p0, static_cast<uint32_t>(kLanes));
        const float2 ml = l % kLanes < many ? ldg(a.stats + j.row(p0 + l % kLanes) + mine) : make_float2(kLowest, 0.0f);
        float x[kFlight][kHeads][N];
        const auto fetch = [&](uint32_t k0) {
#pragma unroll
            for (uint32_t k = 0; k < kFlight; ++k) {
                const int64_t row = j.row(p0 + min(k0 + k, many - 1));
#pragma unroll
                for (uint32_t h = 0; h < kHeads; ++h) load_dims<N>(x[k][h], a.o + (row + min(head + h, last)) * HD, l);
            }
        };
        fetch(0);
        const float mn = fmaxf(m, group_max<kLanes>(ml.x)), factor = __builtin_amdgcn_exp2f(m - mn), weight = __builtin_amdgcn_exp2f(ml.x - mn);
        lsum = lsum * factor + group_sum<kLanes>(weight * ml.y);
        m = mn;
#pragma unroll
        for (uint32_t h = 0; h < kHeads; ++h) {
            const float f = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(factor), kLanes * h));
#pragma unroll
            for (int i = 0; i < N; ++i) o[h][i] *= f;
        }
        for (uint32_t k0 = 0; k0 < many; k0 += kFlight) {
            if (k0) fetch(k0);
#pragma unroll
            for (uint32_t k = 0; k < kFlight; ++k) {
                if (k0 + k >= many) break;
#pragma unroll
                for (uint32_t h = 0; h < kHeads; ++h) {
                    const float f = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(weight), kLanes * h + k0 + k));
#pragma unroll
                    for (int i = 0; i < N; ++i) o[h][i] += f * x[k][h][i];
                }
            }
        }
    }
    const uint32_t t = at % a.batch.tokens, kvh = at / a.batch.tokens;
#pragma unroll
    for (uint32_t h = 0; h < kHeads; ++h) {
        if (head + h > last) break;
        const float sum = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(lsum), kLanes * h)), inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
        for (int i = 0; i < N; ++i) o[h][i] *= inv;
        store_dims<N>(a.out + (static_cast<uint64_t>(t) * a.heads + kvh * a.group + head + h) * HD, o[h], l);
    }
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Two workgroups a compute unit, or the power of two below.
int32_t workgroups_log2() {
    int32_t n = 3;
    while ((2u << n) <= 2 * vkml::abi::compute_units()) ++n;
    return n;
}

Slots slots_of(const vkml_attend_pages_params& p) {
    return slots(p.kv_heads, p.heads / p.kv_heads, p.seqs, p.groups, p.tokens, int64_t{1} << workgroups_log2());
}

uint64_t up16(uint64_t bytes) { return (bytes + 15) / 16 * 16; }

struct Call {
    const char* name;
    const float* q;
    const void* k;
    const void* v;
    const int32_t* table;
    const int32_t* lengths;
    const int32_t* starts;
    const int32_t* group_starts;
    const int32_t* group_keys;
    void* workspace;
    float* out;
};

// One of the calls, whose own arguments `set` takes and checks.
template <int MASK, typename Set>
int attend(const vkml_attend_pages_params* p, const Call& c, const Set& set) {
    VKML_REQUIRE_INIT();
    const auto refuse = [&](const char* why) { return vkml::abi::fail(VKML_ERROR_INVALID_ARGUMENT, std::string(c.name) + ": " + why); };
    if (!p) return refuse("null params");
    if (const char* why = check(*p)) return refuse(why);
    PagesArgs a{};
    if (const char* why = set(a)) return refuse(why);
    if (p->seqs == 0 || p->tokens == 0) return VKML_OK;
    if (!c.starts && p->tokens != p->seqs) return refuse("without starts every sequence has one token");
    if (!(c.q && c.k && c.v && c.table && c.lengths && c.workspace && c.out && (p->groups == 0 || (c.group_starts && c.group_keys)))) return refuse("null buffer");
    if (!(aligned16(c.q) && aligned16(c.k) && aligned16(c.v) && aligned16(c.workspace) && aligned16(c.out)))
        return refuse("q, the pools, the workspace and out must be 16-byte aligned");
    const Batch batch{c.lengths, c.starts, c.group_starts, c.group_keys, static_cast<int32_t>(p->seqs), static_cast<int32_t>(p->tokens),
                      static_cast<int32_t>(p->groups), static_cast<int32_t>(p->table_stride * p->page_size)};
    const uint64_t stride = p->page_stride ? p->page_stride : static_cast<uint64_t>(p->kv_heads) * p->page_size * p->head_dim;
    const Slots s = slots_of(*p);
    auto* at = static_cast<uint8_t*>(c.workspace);
    a.q = c.q;
    a.k = static_cast<const uint8_t*>(c.k);
    a.v = static_cast<const uint8_t*>(c.v);
    a.table = c.table;
    a.out = c.out;
    a.parts = reinterpret_cast<Parts*>(at);
    at += up16(static_cast<uint64_t>(p->kv_heads) * p->tokens * 2 * sizeof(Parts));
    a.stats = reinterpret_cast<float2*>(at);
    a.o = reinterpret_cast<float*>(at + up16(s.rows() * sizeof(float2)));
    a.batch = batch;
    a.page_units = static_cast<uint32_t>(stride * (p->kv_type == VKML_F16 ? 2 : 4) / 16);
    a.few_slots = s.few;
    a.tile_slots = s.tile;
    a.heads = p->heads;
    a.kv_heads = p->kv_heads;
    a.group = p->heads / p->kv_heads;
    a.page_shift = static_cast<uint32_t>(__builtin_ctz(p->page_size));
    a.pages = p->pages;
    a.table_stride = p->table_stride;
    a.workgroups_log2 = workgroups_log2();
    a.most_tiles = static_cast<uint32_t>(most_tiles(a.group, p->seqs, p->groups, p->tokens));  // at most 2^23 + 2^17
    a.score_scale = p->softcap > 0.0f ? p->scale / p->softcap : p->scale * kLog2e;
    a.softcap = p->softcap;
    a.costs = costs(p->head_dim, p->kv_type == VKML_F16);
    a.group_inverse = 1.0f / static_cast<float>(a.group);
    vkml::abi::ProfileScope prof(c.name);
    const auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(1u << a.workgroups_log2), dim3(kThreads), 0, vkml::abi::stream(), a); };
    const bool wide = p->head_dim == 128;
    if (p->kv_type == VKML_F16) {
        if (p->softcap > 0.0f) wide ? go(k_attend_pages<_Float16, 128, true, MASK>) : go(k_attend_pages<_Float16, 64, true, MASK>);
        else wide ? go(k_attend_pages<_Float16, 128, false, MASK>) : go(k_attend_pages<_Float16, 64, false, MASK>);
    } else {
        if (p->softcap > 0.0f) wide ? go(k_attend_pages<float, 128, true, MASK>) : go(k_attend_pages<float, 64, true, MASK>);
        else wide ? go(k_attend_pages<float, 128, false, MASK>) : go(k_attend_pages<float, 64, false, MASK>);
    }
    if (const int r = vkml::abi::check_launch(c.name)) return r;
    // Few rows, in many pieces: a workgroup a row. Many, in a piece or two: a wave
    // for four. Measured (us a call): one token of 32 heads over 32768 keys, 64
    // pieces a row, 35.4, the waves' 57.2; 64 tokens of 32 heads in two pieces 64.4
    // and 63.1; 2600 tokens 222.6 and 149.4.
    const uint32_t rows = p->tokens * p->heads, fours = p->tokens * p->kv_heads * ((a.group + 3) / 4);
    const auto merge = [&](auto kernel, uint32_t workgroups) {
        const Grid grid = grid_of(workgroups);
        hipLaunchKernelGGL(kernel, dim3(grid.x, grid.y), dim3(kThreads), 0, vkml::abi::stream(), a, s.rows());
    };
    if (rows <= 4096) wide ? merge(k_attend_pages_merge<128>, rows) : merge(k_attend_pages_merge<64>, rows);
    else wide ? merge(k_attend_pages_merge_many<128>, (fours + kWaves - 1) / kWaves) : merge(k_attend_pages_merge_many<64>, (fours + kWaves - 1) / kWaves);
    return vkml::abi::check_launch(c.name);
}

}  // namespace

extern "C" {

uint64_t vkml_attend_pages_workspace_bytes(const vkml_attend_pages_params* p) {
    if (!p || !vkml::abi::initialized() || check(*p)) return 0;
    const uint64_t rows = slots_of(*p).rows();
    return up16(static_cast<uint64_t>(p->kv_heads) * p->tokens * 2 * sizeof(Parts)) + up16(rows * sizeof(float2)) + rows * p->head_dim * sizeof(float);
}

int vkml_attend_pages(const vkml_attend_pages_params* p, const float* q, const void* k_pages, const void* v_pages, const int32_t* table,
                      const int32_t* lengths, const int32_t* starts, const int32_t* group_starts, const int32_t* group_keys, void* workspace,
                      float* out) {
    const Call c{"attend_pages", q, k_pages, v_pages, table, lengths, starts, group_starts, group_keys, workspace, out};
    return attend<kCausal>(p, c, [](PagesArgs&) -> const char* { return nullptr; });
}

int vkml_attend_pages_tree(const vkml_attend_pages_params* p, uint32_t seen_words, const float* q, const void* k_pages, const void* v_pages,
                           const int32_t* table, const int32_t* lengths, const int32_t* starts, const int32_t* group_starts,
                           const int32_t* group_keys, const uint32_t* seen, void* workspace, float* out) {
    const Call c{"attend_pages_tree", q, k_pages, v_pages, table, lengths, starts, group_starts, group_keys, workspace, out};
    return attend<kTree>(p, c, [=](PagesArgs& a) -> const char* {
        a.seen = seen;
        a.seen_words = seen_words;
        const char* why = check_tree(seen_words);
        return why ? why : seen || p->seqs == 0 || p->tokens == 0 ? nullptr : "null buffer";
    });
}

int vkml_attend_pages_window(const vkml_attend_pages_params* p, uint32_t window, uint32_t sinks, const float* q, const void* k_pages,
                             const void* v_pages, const int32_t* table, const int32_t* lengths, const int32_t* starts, void* workspace, float* out) {
    const Call c{"attend_pages_window", q, k_pages, v_pages, table, lengths, starts, nullptr, nullptr, workspace, out};
    return attend<kWindow>(p, c, [=](PagesArgs& a) -> const char* {
        // (whole blocks of many rows, Block::kKeys)
        a.window = vkml::pages::window_of(*p, window, sinks, 16384 / (p->head_dim * (p->kv_type == VKML_F16 ? 2 : 4)));
        return check_window(*p, window);
    });
}

}  // extern "C"
