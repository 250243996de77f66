// k_attend_pages.hip -- attention of a batch's new tokens over a paged KV
// cache (vkml_attend_pages): softmax(q k^T scale) v over each token's keys,
// the ones that a group shares through its first sequence's table and once for
// all of its tokens, the rest through the sequence's own.
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
// Rows of a block past the sequence's keys, below the first that counts or in
// no page are read as zeros, so that what lies there, NaN included, has no part.
#include <hip/hip_runtime.h>

#include <string>

#include "attend.hpp"
#include "attend_fast.hpp"
#include "device.hpp"
#include "internal.hpp"
#include "pages.hpp"

using namespace vkml::dev;
using namespace vkml::pages;
using vkml::attend::load_to_lds16;
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
    uint64_t page_bytes;  // from a page to the next
    int64_t few_slots, tile_slots;
    uint32_t heads, kv_heads, group, page_shift, pages, table_stride, workgroups;
    float scale, softcap;
};

// 16 bytes of zeros that the rows without a key are read from.
__device__ const uint4 g_zeros = {0, 0, 0, 0};

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
};

// The pages that a wave's N loads of a block from key0 on read, 16 keys or
// less each, and a bit for each of the block's tiles that is in no page.
template <int N>
struct Pages {
    int32_t id[N];
    int32_t key0;
    uint32_t dead;
};

// What a tile's pieces have in common.
struct Tile {
    const int32_t* table;  // its sequence's row
    uint32_t kvh;
    int32_t from, end;     // the keys that count
};

__device__ __forceinline__ int32_t page_id(const PagesArgs& a, const Tile& t, int32_t key) {
    return key < t.end ? ld_scalar_i32(t.table + (key >> a.page_shift)) : -1;
}

// 16 keys of a block: where their first row is, and whether all of them count.
struct Rows {
    const uint8_t* k;
    const uint8_t* v;
    bool whole;
    int32_t first, last;  // the rows that count
};
template <uint32_t ROW>
__device__ __forceinline__ Rows rows_at(const PagesArgs& a, const Tile& t, int32_t id, int32_t key) {
    const bool held = static_cast<uint32_t>(id) < a.pages;
    const uint64_t at = static_cast<uint64_t>(held ? id : 0) * a.page_bytes +
                        ((static_cast<uint64_t>(t.kvh) << a.page_shift) + (key & ((1 << a.page_shift) - 1))) * ROW;
    Rows r{a.k + at, a.v + at, false, held ? max(t.from - key, 0) : 16, min(t.end - key, 16)};
    r.whole = r.first == 0 && r.last == 16;
    return r;
}

// The bytes at `offset`, in row r of 16 rows, or zeros where the row holds no key.
__device__ __forceinline__ const uint8_t* piece_at(const uint8_t* base, const Rows& rows, uint32_t r, uint32_t offset) {
    return static_cast<int32_t>(r) >= rows.first && static_cast<int32_t>(r) < rows.last ? base + offset : reinterpret_cast<const uint8_t*>(&g_zeros);
}

// ---------------------------------------------------------------- q

// RT tiles of 16 rows of q as the matrix instructions take them: lane (j, g)
// has row j's pieces 4 s + g. c[rt]: what turns a product with them into a
// score in log2 units (with a soft cap: into a score).
template <typename T, int HD, int RT>
struct Queries;

template <int HD, int RT>
struct Queries<_Float16, HD, RT> {
    half8 hi[RT][HD / 32], lo[RT][HD / 32];
    float c[RT];
    __device__ __forceinline__ void load(int rt, const float* row, uint32_t g, float scale) {
        float x[HD / 32][8], most = 0.0f;
#pragma unroll
        for (int s = 0; s < HD / 32; ++s) {
            const float4 a = ldg(reinterpret_cast<const float4*>(row + 32 * s + 8 * g)), b = ldg(reinterpret_cast<const float4*>(row + 32 * s + 8 * g + 4));
            const float y[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[s][e] = y[e];
                most = fmaxf(most, fabsf(y[e]));
            }
        }
        const uint2 r16 = swap_rows<16>(__float_as_uint(most));
        most = fmaxf(__uint_as_float(r16.x), __uint_as_float(r16.y));
        const uint2 r32 = swap_rows<32>(__float_as_uint(most));
        most = fmaxf(__uint_as_float(r32.x), __uint_as_float(r32.y));
        // The row's largest value to [1/2, 1): neither term leaves f16's range.
        const int e2 = __builtin_amdgcn_frexp_expf(most);
#pragma unroll
        for (int s = 0; s < HD / 32; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float y = __builtin_amdgcn_ldexpf(x[s][e], -e2);
                hi[rt][s][e] = static_cast<_Float16>(y);
                lo[rt][s][e] = static_cast<_Float16>(y - static_cast<float>(hi[rt][s][e]));
            }
        c[rt] = __builtin_amdgcn_ldexpf(scale, e2);
    }
    // The products of step s with the keys' tiles, in turn, so that an
    // instruction does not wait for the one before it.
    template <int TT>
    __device__ __forceinline__ void score(int s, const uint4 (&k)[TT], f32x4 (&acc)[RT][TT]) const {
#pragma unroll
        for (int term = 0; term < 2; ++term)
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int tt = 0; tt < TT; ++tt)
                    acc[rt][tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, k[tt]), term ? lo[rt][s] : hi[rt][s], acc[rt][tt], 0, 0, 0);
    }
};

template <int HD, int RT>
struct Queries<float, HD, RT> {
    float4 x[RT][HD / 16];
    float c[RT];
    __device__ __forceinline__ void load(int rt, const float* row, uint32_t g, float scale) {
#pragma unroll
        for (int s = 0; s < HD / 16; ++s) x[rt][s] = ldg(reinterpret_cast<const float4*>(row + 16 * s + 4 * g));
        c[rt] = scale;
    }
    template <int TT>
    __device__ __forceinline__ void score(int s, const uint4 (&k)[TT], f32x4 (&acc)[RT][TT]) const {
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int tt = 0; tt < TT; ++tt) {
                    const f32x4 y = __builtin_bit_cast(f32x4, k[tt]);
                    const float4 z = x[rt][s];
                    acc[rt][tt] = __builtin_amdgcn_mfma_f32_16x16x4f32(y[e], e == 0 ? z.x : e == 1 ? z.y : e == 2 ? z.z : z.w, acc[rt][tt], 0, 0, 0);
                }
    }
};

// ---------------------------------------------------------------- a block

// What a wave has of RT tiles of 16 rows: lane (j, g) has row j's dims 16 dt +
// 4 g + e, its maximum, and the sum over the keys of its own lane.
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

// The rows' own limits: row j of tile rt sees keys below limit[rt]. low: the
// least of the piece's tile; mixed: they differ.
template <int RT>
struct Limits {
    int32_t limit[RT];
    int32_t low;
    bool mixed;
};

// Zeros for the infinities and NaN among a block's V values; whether there
// were any among the thread's.
template <typename T>
__device__ __forceinline__ bool clear_unbounded(uint8_t* v, uint32_t bytes, uint32_t thread, uint32_t threads) {
    bool found = false;
#pragma unroll 1
    for (uint32_t i = 16 * thread; i < bytes; i += 16 * threads) {
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
        found |= here;
    }
    return found;
}

// The infinities and NaN of V at keys [k0, k1) for the rows that see them: a
// row's output there is their sum, whatever its finite values are.
template <typename T, int HD, int RT>
__device__ __forceinline__ void add_unbounded(const PagesArgs& a, const Tile& t, const Limits<RT>& lim, int32_t k0, int32_t k1, Running<HD, RT>& run) {
    const uint32_t g = threadIdx.x % kWave / 16;
#pragma unroll 1
    for (int32_t key = k0; key < k1; ++key) {
        const int32_t id = ld_scalar_i32(t.table + (key >> a.page_shift));
        if (static_cast<uint32_t>(id) >= a.pages || key < t.from) continue;
        const Rows at = rows_at<Block<T, HD>::kRow>(a, t, id, key);
        const T* row = reinterpret_cast<const T*>(at.v) + 4 * g;
#pragma unroll
        for (int dt = 0; dt < HD / 16; ++dt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = static_cast<float>(row[16 * dt + e]);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
                    if (key < lim.limit[rt] && !(fabsf(x) <= __FLT_MAX__)) run.o[rt][dt][e] += x;
            }
    }
}

// One block: TT tiles of 16 keys from key0, K in the lane's registers (REGS)
// or as swizzled rows in the LDS, V's rows in the LDS. dead: a bit for each
// tile that is in no page.
template <typename T, int HD, int RT, int TT, bool REGS>
__device__ __forceinline__ void attend_block(const Queries<T, HD, RT>& q, const Limits<RT>& lim, const Tile& tile, int32_t key0, uint32_t dead,
                                             float softcap, const uint4 (*k_regs)[Block<T, HD>::kSteps], const uint8_t* k, const uint8_t* v,
                                             Running<HD, RT>& run) {
    using B = Block<T, HD>;
    const uint32_t l = threadIdx.x % kWave, j = l % 16, g = l / 16;
    const uint32_t k_at = j * B::kRow + 16 * (g ^ B::swizzle_k(j));
    f32x4 s[RT][TT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) s[rt][tt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int st = 0; st < static_cast<int>(B::kSteps); ++st) {
        uint4 kk[TT];
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) {
            if constexpr (REGS) kk[tt] = k_regs[tt][st];
            else kk[tt] = *reinterpret_cast<const uint4*>(k + (k_at ^ (64 * st)) + 16 * tt * B::kRow);
        }
        q.score(st, kk, s);
    }
    const bool masked = key0 < tile.from || key0 + 16 * TT > lim.low || dead;
    constexpr float kShift = B::kF16 ? 14.0f : 0.0f;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const float c = q.c[rt];
#pragma unroll
        for (int tt = 0; tt < TT; ++tt)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[rt][tt][e] *= c;
        if (softcap > 0.0f) {
#pragma unroll
            for (int tt = 0; tt < TT; ++tt)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[rt][tt][e] = softcap * tanhf(s[rt][tt][e] / softcap) * kLog2e;
        }
        if (masked) {
#pragma unroll
            for (int tt = 0; tt < TT; ++tt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int32_t key = key0 + 16 * tt + 4 * static_cast<int32_t>(g) + e;
                    if (key < tile.from || key >= lim.limit[rt] || (dead >> tt & 1)) s[rt][tt][e] = -__builtin_inff();
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
        const float mn = fmaxf(run.m[rt], bm), factor = __builtin_amdgcn_exp2f(run.m[rt] - mn), mm = mn - kShift;
        float bs = 0.0f;
#pragma unroll
        for (int tt = 0; tt < TT; ++tt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float p = __builtin_amdgcn_exp2f(s[rt][tt][e] - mm);
                s[rt][tt][e] = p;
                bs += p;
            }
        run.l[rt] = run.l[rt] * factor + bs;
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
        constexpr int D = RT == 1 && HD == 128 ? 8 : 4;  // tiles of dims read at a time
#pragma unroll
        for (int u = 0; u < TT / 2; ++u) {
            half8 ph[RT], pl[RT];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float p = s[rt][2 * u + e / 4][e % 4];
                    ph[rt][e] = static_cast<_Float16>(p);
                    pl[rt][e] = static_cast<_Float16>(p - static_cast<float>(ph[rt][e]));
                }
#pragma unroll
            for (int d0 = 0; d0 < HD / 16; d0 += D) {
                half8 vv[D];
#pragma unroll
                for (int i = 0; i < D; ++i) {
                    const uint8_t* to = v + (at ^ (32 * (d0 + i))) + 32 * u * B::kRow;
                    const auto x = __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds4)(to));
                    const auto y = __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds4)(to + 16 * B::kRow));
                    const uint2 xx = __builtin_bit_cast(uint2, x), yy = __builtin_bit_cast(uint2, y);
                    vv[i] = __builtin_bit_cast(half8, make_uint4(xx.x, xx.y, yy.x, yy.y));
                }
#pragma unroll
                for (int term = 0; term < 2; ++term)
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                        for (int i = 0; i < D; ++i)
                            run.o[rt][d0 + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vv[i], term ? pl[rt] : ph[rt], run.o[rt][d0 + i], 0, 0, 0);
            }
        }
    } else {
        // Instruction e of a tile takes keys 4 g + e: V's element of dim j.
#pragma unroll
        for (int tt = 0; tt < TT; ++tt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t row = 16 * tt + 4 * g + e;
#pragma unroll
                for (int dt = 0; dt < HD / 16; ++dt) {
                    const float vv = *reinterpret_cast<const float*>(v + row * B::kRow + 16 * ((4 * dt + j / 4) ^ B::swizzle_v(row)) + 4 * (j % 4));
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) run.o[rt][dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(vv, s[rt][tt][e], run.o[rt][dt], 0, 0, 0);
                }
            }
    }
}

// ---------------------------------------------------------------- pieces

// A piece of a tile: keys [k0, k1) of rows `rows` from token0 on.
struct Piece {
    Tile tile;
    int32_t k0, k1;
    int32_t token0, tokens;
    int32_t limit0;   // the keys below which the first token sees
    bool causal;      // and each further token one more
    bool whole;       // all of its rows' work: the output itself
    int64_t slot_row;  // else the rows of the workspace, -1 for none
};

template <typename T, int HD, int RT>
__device__ __forceinline__ void load_rows(const PagesArgs& a, const Piece& p, uint32_t first_row, Queries<T, HD, RT>& q, Limits<RT>& lim) {
    const uint32_t l = threadIdx.x % kWave, j = l % 16, g = l / 16, rows = p.tokens * a.group;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const uint32_t r = min(first_row + 16 * rt + j, rows - 1), t = r / a.group;
        const float* row = a.q + (static_cast<uint64_t>(p.token0 + t) * a.heads + p.tile.kvh * a.group + r % a.group) * HD;
        q.load(rt, row, g, a.softcap > 0.0f ? a.scale : a.scale * kLog2e);
        lim.limit[rt] = p.causal ? p.limit0 + static_cast<int32_t>(t) : p.limit0;
    }
    lim.low = p.limit0;
    lim.mixed = p.causal && p.tokens > 1;
}

// dims of a row, 4 a lane, to the output or the workspace
template <int HD>
__device__ __forceinline__ void store_row(const PagesArgs& a, const Piece& p, uint32_t r, uint32_t dim, f32x4 o, float m, float l) {
    if (p.whole) {
        const uint32_t t = r / a.group;
        float* to = a.out + (static_cast<uint64_t>(p.token0 + t) * a.heads + p.tile.kvh * a.group + r % a.group) * HD + dim;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        stg(reinterpret_cast<float4*>(to), make_float4(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv));
    } else if (p.slot_row >= 0) {
        stg(reinterpret_cast<float4*>(a.o + (p.slot_row + r) * HD + dim), make_float4(o[0], o[1], o[2], o[3]));
        if (dim == 0) stg(a.stats + p.slot_row + r, make_float2(m, l));
    }
}

// At most 16 rows: each wave by itself over blocks of kWaveKeys keys in turn.
template <typename T, int HD>
__device__ __forceinline__ void few_rows(const PagesArgs& a, const Piece& p, Buffer* buf) {
    using B = Block<T, HD>;
    constexpr int TT = B::kWaveTiles, N = TT;
    const uint32_t w = threadIdx.x / kWave, l = threadIdx.x % kWave, j = l % 16, g = l / 16;
    Queries<T, HD, 1> q;
    Limits<1> lim;
    Running<HD, 1> run;
    run.clear();
    uint8_t* v = reinterpret_cast<uint8_t*>(buf) + 8192 * w;  // and as far into the second buffer
    const int32_t step = kWaves * B::kWaveKeys;
    int32_t key = p.k0 + static_cast<int32_t>(w * B::kWaveKeys);
    key = __builtin_amdgcn_readfirstlane(key);
    const int32_t first = key;
    const auto issue = [&](const Pages<N>& ids, uint4 (&k)[TT][B::kSteps], uint8_t* to) {
        Rows rows[N];
        bool whole = true;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            rows[i] = rows_at<B::kRow>(a, p.tile, ids.id[i], ids.key0 + 16 * i);
            whole &= rows[i].whole;
        }
        const auto loads = [&](auto piece) {
#pragma unroll
            for (int tt = 0; tt < TT; ++tt)
#pragma unroll
                for (int s = 0; s < static_cast<int>(B::kSteps); ++s)
                    k[tt][s] = ldg(reinterpret_cast<const uint4*>(piece(rows[tt].k, rows[tt], j, j * B::kRow + 64 * s + 16 * g)));
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {
                const uint32_t u = 64 * i + l, row = u / B::kPieces, r = row % 16;
                const Rows& at = rows[64 * i / B::kPieces / 16];
                load_to_lds16(piece(at.v, at, r, r * B::kRow + 16 * (u % B::kPieces ^ B::swizzle_v(row))), to + 1024 * i);
            }
        };
        if (whole) loads([](const uint8_t* base, const Rows&, uint32_t, uint32_t offset) { return base + offset; });
        else loads(piece_at);
    };
    uint4 k[TT][B::kSteps];
    const auto pages_at = [&](int32_t key0) {
        Pages<N> r{{}, key0, 0};
#pragma unroll
        for (int i = 0; i < N; ++i) {
            r.id[i] = page_id(a, p.tile, key0 + 16 * i);
            r.dead |= static_cast<uint32_t>(r.id[i]) < a.pages ? 0u : 1u << i;
        }
        return r;
    };
    Pages<N> cur = pages_at(key), nxt = pages_at(key + step);
    // Values that are not finite in blocks that some rows see less of than
    // others are left out of the product and added at the end.
    bool unbounded = false;
    // The buffers don't overlap. Said so (__restrict__), and with both's loads
    // issued in here, the reads of one do not wait for the loads into the other.
    const auto block = [&](uint8_t* __restrict__ here, uint8_t* __restrict__ there) {
        if (key == first) {
            issue(cur, k, here);
            load_rows(a, p, 0, q, lim);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this block has landed
        uint4 k_next[TT][B::kSteps] = {};
        if (key + step < p.k1) issue(nxt, k_next, there);
        const Pages<N> after = pages_at(key + 2 * step);
        if (lim.mixed && key + static_cast<int32_t>(B::kWaveKeys) > lim.low) unbounded |= clear_unbounded<T>(here, 8192, l, kWave);
        attend_block<T, HD, 1, TT, true>(q, lim, p.tile, key, cur.dead, a.softcap, k, nullptr, here, run);
        cur = nxt;
        nxt = after;
        key += step;
#pragma unroll
        for (int tt = 0; tt < TT; ++tt)
#pragma unroll
            for (int s = 0; s < static_cast<int>(B::kSteps); ++s) k[tt][s] = k_next[tt][s];
    };
    for (uint32_t n = 0; key < p.k1; n ^= sizeof(Buffer)) block(v + n, v + (n ^ sizeof(Buffer)));
    if (__any(unbounded)) {
        for (int32_t k = p.k0 + static_cast<int32_t>(w * B::kWaveKeys); k < p.k1; k += step) {
            const int32_t end = min(k + static_cast<int32_t>(B::kWaveKeys), p.k1);
            if (k + static_cast<int32_t>(B::kWaveKeys) > lim.low)
                add_unbounded<T, HD, 1>(a, p.tile, lim, __builtin_amdgcn_readfirstlane(k), __builtin_amdgcn_readfirstlane(end), run);
        }
    }
    // The waves' parts join in the LDS, rows HD + 4 floats apart.
    const uint2 l16 = swap_rows<16>(__float_as_uint(run.l[0]));
    float sum = __uint_as_float(l16.x) + __uint_as_float(l16.y);
    const uint2 l32 = swap_rows<32>(__float_as_uint(sum));
    sum = __uint_as_float(l32.x) + __uint_as_float(l32.y);
    constexpr uint32_t kStride = HD + 4;
    float* part = reinterpret_cast<float*>(buf);  // [waves][16][kStride], then [waves][16] of (m, l)
    float2* ml = reinterpret_cast<float2*>(part + kWaves * 16 * kStride);
    __syncthreads();
#pragma unroll
    for (int dt = 0; dt < HD / 16; ++dt)
        *reinterpret_cast<f32x4*>(part + (16 * w + j) * kStride + 16 * dt + 4 * g) = run.o[0][dt];
    if (g == 0) ml[16 * w + j] = make_float2(run.m[0], sum);
    __syncthreads();
    const uint32_t r = threadIdx.x / 16;
    if (r < p.tokens * a.group) {
        float m = kLowest, f[kWaves], lsum = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < kWaves; ++i) m = fmaxf(m, ml[16 * i + r].x);
#pragma unroll
        for (uint32_t i = 0; i < kWaves; ++i) {
            f[i] = __builtin_amdgcn_exp2f(ml[16 * i + r].x - m);
            lsum += f[i] * ml[16 * i + r].y;
        }
#pragma unroll
        for (uint32_t d = 0; d < HD / 64; ++d) {
            const uint32_t dim = 64 * d + 4 * (threadIdx.x % 16);
            f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (uint32_t i = 0; i < kWaves; ++i) {
                const f32x4 x = *reinterpret_cast<const f32x4*>(part + (16 * i + r) * kStride + dim);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] += f[i] * x[e];
            }
            store_row<HD>(a, p, r, dim, o, m, lsum);
        }
    }
    __syncthreads();  // the next piece loads into this memory
}

// Many rows: RT tiles of 16 a wave, the blocks shared.
template <typename T, int HD, int RT>
__device__ __forceinline__ void many_rows(const PagesArgs& a, const Piece& p, Buffer* buf) {
    using B = Block<T, HD>;
    constexpr int TT = B::kTiles, N = 4;
    const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), l = threadIdx.x % kWave, j = l % 16, g = l / 16;
    const uint32_t rows = p.tokens * a.group, first = 16 * RT * w;
    Queries<T, HD, RT> q;
    Limits<RT> lim;
    Running<HD, RT> run;
    run.clear();
    // The first of the 16 keys that the wave's i-th load is in.
    const auto part_of_load = [&](int i) { return static_cast<int32_t>((i * kThreads + w * kWave) / B::kPieces / 16 * 16); };
    const auto issue = [&](const Pages<N>& ids, uint8_t* k_all, uint8_t* v_all) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t u = i * kThreads + threadIdx.x, row = u / B::kPieces, r = row % 16;
            const Rows at = rows_at<B::kRow>(a, p.tile, ids.id[i], ids.key0 + part_of_load(i));
            const uint32_t k_offset = r * B::kRow + 16 * (u % B::kPieces ^ B::swizzle_k(row));
            const uint32_t v_offset = r * B::kRow + 16 * (u % B::kPieces ^ B::swizzle_v(row));
            uint8_t* k_to = k_all + 16 * (i * kThreads + w * kWave);
            uint8_t* v_to = v_all + 16 * (i * kThreads + w * kWave);
            if (at.whole) {
                load_to_lds16(at.k + k_offset, k_to);
                load_to_lds16(at.v + v_offset, v_to);
            } else {
                load_to_lds16(piece_at(at.k, at, r, k_offset), k_to);
                load_to_lds16(piece_at(at.v, at, r, v_offset), v_to);
            }
        }
    };
    int32_t key = p.k0;
    const auto pages_at = [&](int32_t key0) {
        Pages<N> r{{}, key0, 0};
#pragma unroll
        for (int i = 0; i < N; ++i) r.id[i] = page_id(a, p.tile, key0 + part_of_load(i));
#pragma unroll
        for (int i = 0; i < TT; ++i) r.dead |= static_cast<uint32_t>(page_id(a, p.tile, key0 + 16 * i)) < a.pages ? 0u : 1u << i;
        return r;
    };
    Pages<N> cur = pages_at(key), nxt = pages_at(key + B::kKeys);
    // The wave's rows that are none of the tile's take no part; nor do blocks
    // past all that the wave's rows see.
    const int32_t last_row = static_cast<int32_t>(min(first + 16 * RT, rows)) - 1;
    const int32_t wave_end = first >= rows ? 0 : p.causal ? p.limit0 + last_row / static_cast<int32_t>(a.group) : p.limit0;
    bool unbounded = false;  // as in few_rows
    const auto block = [&](uint8_t* __restrict__ k, uint8_t* __restrict__ v, uint8_t* __restrict__ k_next, uint8_t* __restrict__ v_next) {
        if (key == p.k0) {
            issue(cur, k, v);
            load_rows(a, p, first, q, lim);
            lim.low = p.causal ? p.limit0 + static_cast<int32_t>(first / a.group) : p.limit0;
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();  // every wave's loads have landed, and the other buffer is read no more
        if (key + static_cast<int32_t>(B::kKeys) < p.k1) issue(nxt, k_next, v_next);
        const Pages<N> after = pages_at(key + 2 * B::kKeys);
        if (lim.mixed && key + static_cast<int32_t>(B::kKeys) > p.limit0) {
            unbounded |= clear_unbounded<T>(v, sizeof buf[0].v, threadIdx.x, kThreads);
            __syncthreads();
        }
        if (key < wave_end) attend_block<T, HD, RT, TT, false>(q, lim, p.tile, key, cur.dead, a.softcap, nullptr, k, v, run);
        cur = nxt;
        nxt = after;
        key += B::kKeys;
    };
    for (uint32_t n = 0; key < p.k1; n ^= 1) block(buf[n].k, buf[n].v, buf[n ^ 1].k, buf[n ^ 1].v);
    if (p.causal && p.tokens > 1 && __syncthreads_or(unbounded)) {
        // the blocks from the one that holds the first limit on
        const int32_t first_block = max(p.limit0 - p.k0, 0) / static_cast<int32_t>(B::kKeys) * static_cast<int32_t>(B::kKeys);
        add_unbounded<T, HD, RT>(a, p.tile, lim, p.k0 + first_block, p.k1, run);
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const uint2 l16 = swap_rows<16>(__float_as_uint(run.l[rt]));
        float sum = __uint_as_float(l16.x) + __uint_as_float(l16.y);
        const uint2 l32 = swap_rows<32>(__float_as_uint(sum));
        sum = __uint_as_float(l32.x) + __uint_as_float(l32.y);
        const uint32_t r = first + 16 * rt + j;
        if (r < rows) {
#pragma unroll
            for (int dt = 0; dt < HD / 16; ++dt) store_row<HD>(a, p, r, 16 * dt + 4 * g, run.o[rt][dt], run.m[rt], sum);
        }
    }
    __syncthreads();  // the next piece loads into this memory
}

// ---------------------------------------------------------------- the launch

// Where a workgroup's part begins, and the whole of the work.
struct Place {
    int64_t cost;          // all KV heads'
    int64_t off;           // the cost before the segment
    int32_t kvh, segment;  // the first that the part has work of
    int32_t few, tiles;    // tiles of each kind before the segment
    int32_t part, parts;
};

// Every thread sums its run of segments; the workgroup's exclusive sums then
// place them, and the thread whose run holds the part's first unit finds it.
__device__ __forceinline__ bool find_place(const PagesArgs& a, Place& out, uint8_t* lds) {
    const int32_t n = a.batch.groups + a.batch.seqs, each = (n + kThreads - 1) / kThreads;
    const int32_t i0 = min(static_cast<int32_t>(threadIdx.x) * each, n), i1 = min(i0 + each, n);
    int64_t cost = 0;
    int32_t few = 0, tiles = 0;
    for (int32_t i = i0; i < i1; ++i) {
        const Segment s = segment(a.batch, a.group, i);
        cost += s.cost();
        (s.few ? few : tiles) += s.tiles;
    }
    int64_t* costs = reinterpret_cast<int64_t*>(lds);
    int32_t* fews = reinterpret_cast<int32_t*>(costs + kThreads);
    int32_t* tile_sums = fews + kThreads;
    Place* place = reinterpret_cast<Place*>(tile_sums + kThreads);
    // inclusive sums in the wave, then across the waves
    const uint32_t l = threadIdx.x % kWave, w = threadIdx.x / kWave;
    int64_t c = cost;
    int32_t f = few, t = tiles;
#pragma unroll
    for (uint32_t d = 1; d < kWave; d *= 2) {
        const int64_t cc = __shfl_up(static_cast<long long>(c), d, kWave);
        const int32_t ff = __shfl_up(f, d, kWave), tt = __shfl_up(t, d, kWave);
        if (l >= d) c += cc, f += ff, t += tt;
    }
    if (l == kWave - 1) costs[w] = c, fews[w] = f, tile_sums[w] = t;
    __syncthreads();
    int64_t per_head = 0;
    int32_t few_head = 0, tiles_head = 0;
#pragma unroll
    for (uint32_t i = 0; i < kWaves; ++i) {
        if (i < w) c += costs[i], f += fews[i], t += tile_sums[i];
        per_head += costs[i], few_head += fews[i], tiles_head += tile_sums[i];
    }
    const int64_t all = per_head * a.kv_heads;
    const int32_t n_parts = parts(all, a.workgroups);
    // dealt to the XCDs round-robin: part p is with its neighbours on one
    const int32_t b = static_cast<int32_t>(blockIdx.x);
    if (all == 0 || b >= n_parts) return false;
    const int32_t part = b % 8 * (n_parts / 8) + b / 8;
    const int64_t u0 = part_start(all, n_parts, part);
    const int32_t kvh = static_cast<int32_t>(u0 / per_head);
    const int64_t rem = u0 - kvh * per_head;
    int64_t off = c - cost;
    f -= few, t -= tiles;
    if (rem >= off && rem < c) {
        for (int32_t i = i0; i < i1; ++i) {
            const Segment s = segment(a.batch, a.group, i);
            if (rem < off + s.cost()) {
                place->cost = all;
                place->off = kvh * per_head + off;
                place->kvh = kvh;
                place->segment = i;
                place->few = kvh * few_head + f;
                place->tiles = kvh * tiles_head + t;
                place->part = part;
                place->parts = n_parts;
                break;
            }
            off += s.cost();
            (s.few ? f : t) += s.tiles;
        }
    }
    __syncthreads();
    // the workgroup's, in scalar registers
    const auto whole = [](int32_t x) { return __builtin_amdgcn_readfirstlane(x); };
    const auto whole64 = [&](int64_t x) {
        return static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(whole(static_cast<int32_t>(x >> 32)))) << 32 |
                                    static_cast<uint32_t>(whole(static_cast<int32_t>(x))));
    };
    out.cost = whole64(place->cost);
    out.off = whole64(place->off);
    out.kvh = whole(place->kvh);
    out.segment = whole(place->segment);
    out.few = whole(place->few);
    out.tiles = whole(place->tiles);
    out.part = whole(place->part);
    out.parts = whole(place->parts);
    __syncthreads();
    return true;
}

template <typename T, int HD>
__global__ void __launch_bounds__(kThreads, 2) k_attend_pages(PagesArgs a) {
    using B = Block<T, HD>;
    __shared__ Buffer buf[2];
    Place at;
    if (!find_place(a, at, buf[0].k)) return;
    const int64_t u0 = part_start(at.cost, at.parts, at.part), u1 = part_start(at.cost, at.parts, at.part + 1);
    const int32_t segments = a.batch.groups + a.batch.seqs;
    int32_t kvh = at.kvh, i = at.segment, few = at.few, tiles = at.tiles;
    int64_t off = at.off;
    while (off < u1 && kvh < static_cast<int32_t>(a.kv_heads)) {
        const Segment s = segment(a.batch, a.group, i);
        for (int32_t t = s.tiles && u0 > off ? s.tile_at(u0 - off) : 0; t < s.tiles; ++t) {
            const int64_t start = off + s.before(t);
            if (start >= u1) break;
            const int32_t keys = s.keys(t);
            const int64_t end = start + kOverhead + keys;
            Piece p;
            p.tile = {a.table + static_cast<uint64_t>(s.row) * a.table_stride, static_cast<uint32_t>(kvh), s.from, s.lo + keys};
            p.k0 = s.lo + (u0 > start ? cut(u0 - start, keys, B::kKeys) : 0);
            p.k1 = s.lo + (u1 >= end ? keys : cut(u1 - start, keys, B::kKeys));
            p.token0 = s.token0 + t * s.step;
            p.tokens = s.tile_n(t);
            p.limit0 = s.limit(t * s.step);
            p.causal = !s.shared;
            const bool alone = u0 <= start && u1 >= end;
            p.whole = alone && !s.shared && s.from == 0;
            const int32_t slot = at.part + (s.few ? few : tiles + t);
            p.slot_row = s.few ? (slot < a.few_slots ? static_cast<int64_t>(slot) * kFewRows : -1)
                               : (slot < a.tile_slots ? a.few_slots * kFewRows + static_cast<int64_t>(slot) * kTileRows : -1);
            // The tile's first piece tells the merge where they all are; of
            // tokens without shared keys also that those have none.
            if (start >= u0) {
                const uint32_t count = p.whole || p.slot_row < 0 ? 0 : part_of(at.cost, at.parts, end - 1) - at.part + 1;
                for (uint32_t k = threadIdx.x; k < static_cast<uint32_t>(p.tokens); k += kThreads) {
                    Parts* to = a.parts + (static_cast<uint64_t>(kvh) * a.batch.tokens + p.token0 + k) * 2;
                    const Parts mine = {static_cast<uint32_t>(p.slot_row + k * a.group), 2 * count + (s.few ? 0u : 1u)};
                    stg(reinterpret_cast<uint2*>(to + (s.shared ? 0 : 1)), make_uint2(mine.row, mine.count));
                    if (!s.shared && s.from == 0) stg(reinterpret_cast<uint2*>(to), make_uint2(0, 0));
                }
            }
            if (s.few) few_rows<T, HD>(a, p, buf);
            else if (p.tokens * a.group <= kTileRows / 2) many_rows<T, HD, 1>(a, p, buf);
            else many_rows<T, HD, 2>(a, p, buf);
        }
        off += s.cost();
        (s.few ? few : tiles) += s.tiles;
        if (++i == segments) i = 0, ++kvh;
    }
}

// Joins the pieces of the rows that are in several: a wave a row, the pieces'
// (m, l) a lane each, then their o, HD / 64 dims a lane.
template <int HD>
__global__ void __launch_bounds__(kThreads) k_attend_pages_merge(PagesArgs a, int64_t ws_rows) {
    constexpr int N = HD / 64;
    const uint64_t row = static_cast<uint64_t>(blockIdx.x) * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint32_t l = threadIdx.x % kWave;
    if (row >= static_cast<uint64_t>(a.batch.tokens) * a.heads) return;
    const int32_t t = static_cast<int32_t>(row / a.heads);
    if (t < a.batch.start(0) || t >= a.batch.start(a.batch.seqs)) return;
    const uint32_t h = static_cast<uint32_t>(row % a.heads), kvh = h / a.group;
    const uint4 both = ldg(reinterpret_cast<const uint4*>(a.parts + (static_cast<uint64_t>(kvh) * a.batch.tokens + t) * 2));
    const uint32_t n0 = both.y / 2, n1 = both.w / 2, n = n0 + n1;
    if (n == 0) return;
    const auto row_of = [&](uint32_t p) -> int64_t {
        const bool own = p >= n0;
        const uint32_t kind = own ? both.w : both.y;
        return static_cast<int64_t>(own ? both.z : both.x) + h % a.group + static_cast<int64_t>(own ? p - n0 : p) * (kind & 1 ? kTileRows : kFewRows);
    };
    if (row_of(n - 1) >= ws_rows || (n0 && row_of(n0 - 1) >= ws_rows)) return;
    float m = kLowest, lsum = 0.0f, o[N];
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = 0.0f;
    for (uint32_t p0 = 0; p0 < n; p0 += kWave) {
        const uint32_t p = p0 + l;
        const float2 ml = p < n ? ldg(a.stats + row_of(p)) : make_float2(kLowest, 0.0f);
        const float mn = fmaxf(m, wave_max(ml.x)), factor = __builtin_amdgcn_exp2f(m - mn), weight = __builtin_amdgcn_exp2f(ml.x - mn);
        lsum = lsum * factor + wave_sum(p < n ? weight * ml.y : 0.0f);
        m = mn;
#pragma unroll
        for (int i = 0; i < N; ++i) o[i] *= factor;
        const uint32_t many = min(n - p0, static_cast<uint32_t>(kWave));
#pragma unroll 8
        for (uint32_t k = 0; k < many; ++k) {
            const float f = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(weight), k));
            const float* from = a.o + row_of(p0 + k) * HD + N * l;
#pragma unroll
            for (int i = 0; i < N; ++i) o[i] += f * ldg(from + i);
        }
    }
    const float inv = lsum == 0.0f ? 0.0f : 1.0f / lsum;
#pragma unroll
    for (int i = 0; i < N; ++i) stg(a.out + row * HD + N * l + i, o[i] * inv);
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

uint32_t workgroups() { return std::max(8u, 2 * vkml::abi::compute_units() / 8 * 8); }

Slots slots_of(const vkml_attend_pages_params& p) {
    return slots(p.kv_heads, p.heads / p.kv_heads, p.seqs, p.groups, p.tokens, workgroups());
}

uint64_t up16(uint64_t bytes) { return (bytes + 15) / 16 * 16; }

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
    VKML_REQUIRE_INIT();
    VKML_CHECK_ARG(p, "attend_pages: null params");
    if (const char* why = check(*p)) return vkml::abi::fail(VKML_ERROR_INVALID_ARGUMENT, std::string("attend_pages: ") + why);
    if (p->seqs == 0 || p->tokens == 0) return VKML_OK;
    VKML_CHECK_ARG(starts || p->tokens == p->seqs, "attend_pages: without starts every sequence has one token");
    VKML_CHECK_ARG(q && k_pages && v_pages && table && lengths && workspace && out && (p->groups == 0 || (group_starts && group_keys)),
                   "attend_pages: null buffer");
    VKML_CHECK_ARG(aligned16(q) && aligned16(k_pages) && aligned16(v_pages) && aligned16(workspace) && aligned16(out),
                   "attend_pages: q, the pools, the workspace and out must be 16-byte aligned");
    const Batch batch{lengths, starts, group_starts, group_keys, static_cast<int32_t>(p->seqs), static_cast<int32_t>(p->tokens),
                      static_cast<int32_t>(p->groups), static_cast<int32_t>(p->table_stride * p->page_size)};
    const uint64_t stride = p->page_stride ? p->page_stride : static_cast<uint64_t>(p->kv_heads) * p->page_size * p->head_dim;
    const Slots s = slots_of(*p);
    auto* at = static_cast<uint8_t*>(workspace);
    PagesArgs a{};
    a.q = q;
    a.k = static_cast<const uint8_t*>(k_pages);
    a.v = static_cast<const uint8_t*>(v_pages);
    a.table = table;
    a.out = out;
    a.parts = reinterpret_cast<Parts*>(at);
    at += up16(static_cast<uint64_t>(p->kv_heads) * p->tokens * 2 * sizeof(Parts));
    a.stats = reinterpret_cast<float2*>(at);
    a.o = reinterpret_cast<float*>(at + up16(s.rows() * sizeof(float2)));
    a.batch = batch;
    a.page_bytes = stride * (p->kv_type == VKML_F16 ? 2 : 4);
    a.few_slots = s.few;
    a.tile_slots = s.tile;
    a.heads = p->heads;
    a.kv_heads = p->kv_heads;
    a.group = p->heads / p->kv_heads;
    a.page_shift = static_cast<uint32_t>(__builtin_ctz(p->page_size));
    a.pages = p->pages;
    a.table_stride = p->table_stride;
    a.workgroups = workgroups();
    a.scale = p->scale;
    a.softcap = p->softcap;
    vkml::abi::ProfileScope prof("attend_pages");
    const auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(a.workgroups), dim3(kThreads), 0, vkml::abi::stream(), a); };
    if (p->kv_type == VKML_F16) p->head_dim == 128 ? go(k_attend_pages<_Float16, 128>) : go(k_attend_pages<_Float16, 64>);
    else p->head_dim == 128 ? go(k_attend_pages<float, 128>) : go(k_attend_pages<float, 64>);
    if (const int r = vkml::abi::check_launch("attend_pages")) return r;
    const dim3 merge(static_cast<uint32_t>((static_cast<uint64_t>(p->tokens) * p->heads + kWaves - 1) / kWaves));
    if (p->head_dim == 128) hipLaunchKernelGGL(k_attend_pages_merge<128>, merge, dim3(kThreads), 0, vkml::abi::stream(), a, s.rows());
    else hipLaunchKernelGGL(k_attend_pages_merge<64>, merge, dim3(kThreads), 0, vkml::abi::stream(), a, s.rows());
    return vkml::abi::check_launch("attend_pages: merge");
}

}  // extern "C"
