// k_sample.hip -- a token for each row of logits (vkml_sample): vkml::Sampler's
// definition (src/sampling.cpp) for the device, from given random numbers.
//
// Candidates are ranked by logit, then id. With peak the row's largest logit a
// candidate weighs e^((l - peak) / T); top_k, top_p and min_p each keep a first part
// of the ranking, so that only the kept mass M has to be known, and the pick is the
// first candidate whose weight and those before it pass random * M. Nothing is
// sorted: a candidate is found by its count or mass before it, in a histogram of the
// weights' logarithms, then among its bin's candidates.
//
// Where top_k (at most three quarters of a workgroup's threads, fewer in long rows) or
// min_p alone leave few, these are listed first, and the rest is never weighed: the k-th
// largest of the threads' own largest logits is a bound that at least k reach, and few
// more do. A list of up to a quarter of the threads is ranked outright, every candidate
// against every other; a longer one goes through a histogram of its own.
//
// Weights are whole numbers, units of 2^-shift of the largest (45 bits for 2^17
// logits, so that all of a row's fit 62 bits): sums of them are exact in any order,
// so that the same row gives the same token whatever the atomics' order. e^x is
// found in 64 bits, 2^(-n / 1024) from a table times a polynomial of degree 3: within
// 2^-50 of the largest weight (weight_of), not of itself, before it is rounded to units;
// the picks are those of sums in f64 unless a border is nearer than that.
//
// A row of up to 32768 logits is read once and stays in a workgroup's registers; a longer
// one is cut into slices of as many, for a launch each of largest, weights, lists and
// picks, since one workgroup for a row of 128256 would leave most of the GPU idle (40 rows)
// and could not hold it.
//
// Measured (us): 1 row of 32768 with top_k 40 9.8 (5 of it the launch and the load),
// greedy 4.9, min_p 0.05 7.9, top_p 0.95 20.5, no cut 18.8; 40 24; 416 of requests that
// differ 32 (54 MB: 1.7 TB/s), all with top_k 40 26, with top_p 0.95 56, without a cut 53;
// 1024 74; 300 of 4096 15; 40 of 128256 46 to 53: 5 peaks, 14 weights, 14 lists, 14 picks.
// Flat rows take longer, since a bin, 1/32 of a factor of two in weight, has more than the
// list holds and the row is read again for it: normal logits at temperature 30, top_p
// 0.95, 72 for 1 of 32768, 162 for 416, 241 for 40 of 128256. Not bound by bytes (10.6 us for
// the 416, 4.0 for the 40 at a large copy's rate): a row whose candidates are all weighed
// (top_p alone, or nothing) takes 18 by itself, 2 to load, 7 for 32 weights a thread, two
// f64 products and polynomials and two LDS atomics each, 2 for the bins' sums, 2 to list, 4
// for the rest, a chain of steps a few hundred clocks each between barriers; and a
// workgroup of 1024 threads that holds a slice has a compute unit to itself (128 vector
// registers a thread: with 64, so that two fit, they spill, and all rows got slower).
#include <hip/hip_runtime.h>

#include <string>

#include "device.hpp"
#include "internal.hpp"
#include "sample.hpp"

using namespace vkml::dev;
using namespace vkml::sample;

namespace {

constexpr uint32_t kSubs = 1024;  // parts of a range of candidates
constexpr uint64_t kNone = ~0ull;
constexpr int32_t kTurnsLog2 = 10, kTurns = 1 << kTurnsLog2;  // to a factor of two between weights
constexpr int32_t kBinTurns = 32;
static_assert(kTurns / kBinTurns * 53 <= kBins);
constexpr double kMagic = 6755399441055744.0;  // 1.5 2^52: a sum with it is whole, in the low bits

struct Args {
    const float* logits;
    const vkml_sampling* options;
    const double* random;
    int32_t* tokens;
    uint64_t* peaks;  // [rows, slices]: the places of the slices' largest
    Sums* totals;     // [rows]
    Slice* parts;     // [rows, slices]
    uint64_t row_stride;
    uint32_t rows, vocab, slices;
    int32_t shift;
    bool ordered;  // rows of one slice: the long ones first
};

// A candidate's place in the ranking: its logit's bits as a number that falls as the
// logit rises (zeros alike), then its id.
__device__ __forceinline__ uint32_t falling(float l) {
    const uint32_t u = __float_as_uint(l + 0.0f);
    return u & 0x80000000u ? u : ~u & 0x7FFFFFFFu;
}
__device__ __forceinline__ uint64_t place_of(float l, uint32_t id) { return static_cast<uint64_t>(falling(l)) << 32 | id; }
__device__ __forceinline__ float logit_at(uint64_t place) {
    const uint32_t u = static_cast<uint32_t>(place >> 32);
    return __uint_as_float(u & 0x80000000u ? u : ~u & 0x7FFFFFFFu);
}

// ---------------------------------------------------------------- weights

// More turns below the largest than any that is within min_p.
__device__ __forceinline__ double likely_turns(const vkml_sampling& o) { return fmax(2.0 - kTurns * static_cast<double>(log2f(o.min_p)), 2.0); }

// Whether top_p asks for the mass of all, or nothing leaves any out.
__device__ __forceinline__ bool weighs_all(const vkml_sampling& o) { return o.top_p < 1.0f || !(o.min_p > 0.0f); }

struct Row {
    double peak;
    double turns;    // kTurns log2(e) / T
    double nats;     // 1 / T
    double limit;    // a candidate is less turns below the largest (and kMagic)
    uint64_t least;  // weights below it are not within min_p; 0 without
    int32_t shift;
    bool all;        // weighs_all
};

__device__ __forceinline__ Row row_of(float peak, const vkml_sampling& o, int32_t shift) {
    Row r;
    r.peak = static_cast<double>(peak);
    r.nats = fmax(1.0 / static_cast<double>(o.temperature), 1e-300);  // (not 0, of which -infinity makes NaN)
    r.turns = kTurns * 1.4426950408889634 * r.nats;
    r.limit = kTurns * (shift + 1);  // less than half a unit from there on
    r.least = 0;
    if (o.min_p > 0.0f) r.least = o.min_p <= 1.0f ? static_cast<uint64_t>(__builtin_ceil(static_cast<double>(o.min_p) * __builtin_ldexp(1.0, shift))) : ~0ull;
    r.shift = shift;
    r.all = weighs_all(o);
    // Where top_p does not ask for the mass of all, those that min_p leaves out need no
    // weight.
    if (!r.all) r.limit = fmin(r.limit, likely_turns(o));
    r.limit += kMagic;
    return r;
}

// How far a logit's weight is below the largest, in turns: with kMagic, to the next whole
// number n of them. (+infinity beside itself is none below; beside it, as -infinity
// always, the rest is no candidate. NaN comes as -infinity.)
struct Turns {
    double below, sum;  // below: the logits' difference
    __device__ __forceinline__ uint32_t n() const { return static_cast<uint32_t>(__builtin_bit_cast(uint64_t, sum)); }
    __device__ __forceinline__ uint32_t bin() const { return n() / kBinTurns; }
    __device__ __forceinline__ bool candidate(const Row& r) const { return sum < r.limit; }
};
__device__ __forceinline__ Turns turns_of(const Row& r, float l) {
    const double d = fmax(r.peak - static_cast<double>(l), 0.0);
    return {d, __builtin_fma(d, r.turns, kMagic)};
}
// e^(-below / T) 2^shift as a whole number: 2^(shift - n / kTurns) from the table and n's
// upper bits, the rest, at most half a turn, by e^f's first terms. Before it is rounded
// it is off, as a part of itself, by f^4 / 24 < 2^-50.7, the table's 2^-52, the last fma's
// 2^-53 and x = below / T times 3.5 2^-53 (below, 1 / T, their product and n's factor, each
// rounded): 2^-50 (0.99 + 0.44 x). Times e^-x that is at most 2^-50 of the largest weight,
// at x = 0 (largest found in 2 10^7 draws on the CPU: 2^-50.3), but 2^-46.6 of itself at
// x = 36.
__device__ __forceinline__ uint64_t weight_of(const Row& r, const Turns& t, const double* table) {
    const uint32_t n = t.n();
    const double f = __builtin_fma(t.sum - kMagic, 0.6931471805599453 / kTurns, -t.below * r.nats);
    double p = __builtin_fma(f, 1.0 / 6.0, 0.5);
    p = __builtin_fma(p, f, 1.0);
    p = __builtin_fma(p, f, 1.0);
    const uint64_t power = __builtin_bit_cast(uint64_t, table[n & (kTurns - 1)]);
    const uint32_t high = static_cast<uint32_t>(power >> 32) - ((n & ~(kTurns - 1u)) << (20 - kTurnsLog2));
    const double w = __builtin_bit_cast(double, static_cast<uint64_t>(high) << 32 | static_cast<uint32_t>(power));
    return __builtin_bit_cast(uint64_t, __builtin_fma(w, p, 4503599627370496.0)) & 0xFFFFFFFFFFFFFull;
}

// The least logit whose turns are below `sum` (there is one: the largest's are least),
// found among all floats in their order, a 64th of what is left at a time.
__device__ __forceinline__ float edge_of(const Row& r, double sum) {
    uint32_t lo = 0x007FFFFFu, hi = 0xFF800000u;  // -infinity and +infinity, in numbers that rise
    const auto value = [](uint32_t u) { return __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u); };
    while (lo < hi) {
        const uint32_t step = (hi - lo) / kWave + 1, at = lo + min(threadIdx.x % kWave * step, hi - lo);
        const uint64_t below = __ballot(turns_of(r, value(at)).sum < sum);
        if (below == 0) {
            lo += (kWave - 1) * step + 1;
            continue;
        }
        const uint32_t first = static_cast<uint32_t>(__builtin_ctzll(below));
        hi = lo + min(first * step, hi - lo);
        if (first > 0) lo += min((first - 1) * step, hi - lo) + 1;
        lo = min(lo, hi);
    }
    return value(hi);
}

// The logits of the candidates of bins first .. last (or of none).
struct Bounds {
    float from = __builtin_nanf(""), to = __builtin_nanf("");  // to: NaN for +infinity and beyond
    Bounds() = default;
    __device__ __forceinline__ Bounds(const Row& r, uint32_t first, uint32_t last)
        : from(edge_of(r, fmin(r.limit, kMagic + static_cast<double>(last + 1) * kBinTurns))),
          to(first ? edge_of(r, kMagic + static_cast<double>(first) * kBinTurns) : __builtin_nanf("")) {}
    __device__ __forceinline__ bool hold(float l) const { return l >= from && !(l >= to); }
};

// The mass that top_p, `share` of it, asks for at the least, and the unit of it that
// the draw falls on.
__device__ __forceinline__ uint64_t reach_of(float share, uint64_t mass) {
    const double of = __builtin_ceil(static_cast<double>(fmaxf(share, 0.0f)) * static_cast<double>(mass));
    const uint64_t least = static_cast<uint64_t>(of);
    return least < 1 ? 1 : least < mass ? least : mass;
}
__device__ __forceinline__ uint64_t unit_of(double random, uint64_t mass) {
    const double at = random * static_cast<double>(mass);
    const uint64_t unit = at > 0.0 ? (at < 9.2e18 ? static_cast<uint64_t>(at) : mass) : 0;
    return unit < mass ? unit : mass - 1;
}
// What min_p leaves of a mass: the first candidate at least.
__device__ __forceinline__ uint64_t within(const Row& r, uint64_t mass, uint64_t likely) {
    if (r.least == 0) return mass;
    const uint64_t first = 1ull << r.shift, some = likely < first ? first : likely;
    return some < mass ? some : mass;
}

__device__ __forceinline__ bool greedy(const vkml_sampling& o) { return !(o.temperature > 0.0f) || o.top_k == 1; }
__device__ __forceinline__ vkml_sampling options_of(const Args& a, uint32_t row) {
    const uint4 x = ldg(reinterpret_cast<const uint4*>(a.options + row));
    return {__uint_as_float(x.x), static_cast<int32_t>(x.y), __uint_as_float(x.z), __uint_as_float(x.w)};
}

// A row: its vectors of four values from the first multiple of 16 bytes on, and up
// to three values before them and behind.
struct Source {
    const float* row;
    uint32_t vocab, head, vectors;
    __device__ __forceinline__ float4 load(uint32_t v) const {
        const float4 x = ldg(reinterpret_cast<const float4*>(row + head) + v);
        return make_float4(number(x.x), number(x.y), number(x.z), number(x.w));
    }
    __device__ __forceinline__ float value(uint32_t id) const { return number(ldg(row + id)); }
    __device__ __forceinline__ static float number(float l) { return fmaxf(l, -__builtin_inff()); }  // NaN: -infinity
    __device__ __forceinline__ uint32_t id(uint32_t v) const { return head + 4 * v; }
    // The values outside the vectors, six at most: their ids.
    __device__ __forceinline__ uint32_t edges() const { return vocab - 4 * vectors; }
    __device__ __forceinline__ uint32_t edge(uint32_t i) const { return i < head ? i : i + 4 * vectors; }
};
__device__ __forceinline__ Source source_of(const Args& a, uint32_t row) {
    const float* p = a.logits + row * a.row_stride;
    const uint32_t head = min(static_cast<uint32_t>(-(reinterpret_cast<uintptr_t>(p) / 4) % 4), a.vocab);
    return {p, a.vocab, head, (a.vocab - head) / 4};
}

__device__ __forceinline__ uint64_t exchanged(uint64_t v, int o) {
    return static_cast<uint64_t>(static_cast<uint32_t>(__shfl_xor(static_cast<int>(v >> 32), o))) << 32 | static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), o));
}
__device__ __forceinline__ uint64_t wave_min(uint64_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint64_t w = exchanged(v, o);
        v = w < v ? w : v;
    }
    return v;
}
__device__ __forceinline__ uint64_t lane_of(uint64_t v, uint32_t lane) {
    return static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v >> 32), lane))) << 32 |
           static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), lane));
}
__device__ __forceinline__ void add(uint64_t* to, uint64_t v) { __hip_atomic_fetch_add(to, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP); }
__device__ __forceinline__ void add(uint32_t* to, uint32_t v) { __hip_atomic_fetch_add(to, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP); }
__device__ __forceinline__ uint32_t taken(uint32_t* from, uint32_t n) { return __hip_atomic_fetch_add(from, n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP); }

// ---------------------------------------------------------------- a workgroup's work on a row

// Of kThreads threads, which hold kVectors vectors each of a slice.
template <uint32_t kThreads>
struct Picker {
    static constexpr uint32_t kWaves = kThreads / kWave;
    static constexpr uint32_t kFew = kThreads / 4;  // candidates that are ranked one by one, by four threads each

    struct Scratch {
        uint64_t mass[kBins];  // of a bin, then of it and those before
        uint32_t count[kBins];
        uint64_t place[kList], weight[kList];
        union {
            uint32_t id[kList];  // of what is listed, until its places are
            struct {
                uint64_t sub_mass[kSubs];
                uint32_t sub_count[kSubs];
            };
            struct {
                uint64_t few_place[kFew], few_weight[kFew];
                uint64_t ranked_mass[kFew];  // of the ranked candidates up to each
                uint32_t ranked_id[kFew];
            };
        };
        uint64_t wave_mass[kWaves];
        uint32_t wave_count[kWaves];
        double table[kTurns];
        uint64_t lo, hi, likely;  // a range of places; the mass within min_p
        uint64_t found_mass, found_before;
        uint32_t found, found_count, listed, lowest;
    };

    static __device__ __forceinline__ void fill_table(int32_t shift, Scratch& lds) {
        for (uint32_t i = threadIdx.x; i < kTurns; i += kThreads) lds.table[i] = exp2(shift - static_cast<double>(i) / kTurns);
    }

    // A slice in the workgroup's registers, the first one's with the values outside the
    // vectors. (What is none of the row's is -infinity.)
    struct Held {
        float4 x[kVectors];
        float edge;
        uint32_t id0, edge_id;
        __device__ __forceinline__ void load(const Source& s, uint32_t slice) {
            const uint32_t v0 = slice * kVectors * kThreads + threadIdx.x;
            const float none = -__builtin_inff();
            id0 = s.id(v0);
#pragma unroll
            for (uint32_t i = 0; i < kVectors; ++i) {
                x[i] = make_float4(none, none, none, none);
                if (v0 + i * kThreads < s.vectors) x[i] = s.load(v0 + i * kThreads);
            }
            edge = none;
            edge_id = s.edge(threadIdx.x);
            if (slice == 0 && threadIdx.x < s.edges()) edge = s.value(edge_id);
        }
        // f(value, id). (Through an empty asm, so that what one pass finds of the values
        // and ids is not kept in registers for the next.)
        template <typename F>
        __device__ __forceinline__ void each(const F& f) {
#pragma unroll
            for (uint32_t i = 0; i < kVectors; ++i) {
                asm volatile("" : "+v"(x[i].x), "+v"(x[i].y), "+v"(x[i].z), "+v"(x[i].w), "+v"(id0));
                const uint32_t id = id0 + 4 * i * kThreads;
                f(x[i].x, id);
                f(x[i].y, id + 1);
                f(x[i].z, id + 2);
                f(x[i].w, id + 3);
            }
            f(edge, edge_id);
        }
        __device__ __forceinline__ float largest() const {
            float m = edge;
#pragma unroll
            for (uint32_t i = 0; i < kVectors; ++i) m = fmaxf(fmaxf(m, fmaxf(x[i].x, x[i].y)), fmaxf(x[i].z, x[i].w));
            return m;
        }
        // The ids of the candidates in some bins to the list, lds.listed of them:
        // which they are as bits first, then one addition a wave for their places there.
        __device__ __forceinline__ void list(const Bounds& some, const Bounds& others, Scratch& lds) {
            static_assert(4 * kVectors == 32);
            uint32_t bits = 0, k = 0, at_edge = 0;
            each([&](float l, uint32_t) {
                const uint32_t hit = some.hold(l) || others.hold(l);
                if (k < 32) bits |= hit << k++;
                else at_edge = hit;
            });
            const uint32_t n = static_cast<uint32_t>(__builtin_popcount(bits)) + at_edge;
            const uint32_t upto = static_cast<uint32_t>(inclusive_sum(static_cast<int32_t>(n))), all = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(upto), kWave - 1));
            if (all == 0) return;
            uint32_t base = 0;
            if (threadIdx.x % kWave == 0) base = taken(&lds.listed, all);
            uint32_t to = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(base))) + upto - n;
            if (at_edge) {
                if (to < kList) lds.id[to] = edge_id;
                ++to;
            }
            for (; bits && to < kList; bits &= bits - 1, ++to) {
                const uint32_t i = static_cast<uint32_t>(__builtin_ctz(bits));
                lds.id[to] = id0 + 4 * (i / 4) * kThreads + i % 4;
            }
        }
    };

    // A row read again each time.
    struct Streamed {
        Source s;
        template <typename F>
        __device__ __forceinline__ void each(const F& f) {
            constexpr uint32_t kFlight = 2;
            for (uint32_t v = threadIdx.x; v < s.vectors; v += kFlight * kThreads) {
                float4 x[kFlight];
#pragma unroll
                for (uint32_t i = 0; i < kFlight; ++i) x[i] = s.load(min(v + i * kThreads, s.vectors - 1));
#pragma unroll
                for (uint32_t i = 0; i < kFlight; ++i) {
                    if (v + i * kThreads >= s.vectors) break;
                    const uint32_t id = s.id(v + i * kThreads);
                    f(x[i].x, id);
                    f(x[i].y, id + 1);
                    f(x[i].z, id + 2);
                    f(x[i].w, id + 3);
                }
            }
            if (threadIdx.x < s.edges()) f(s.value(s.edge(threadIdx.x)), s.edge(threadIdx.x));
        }
        __device__ __forceinline__ void list(const Bounds& some, const Bounds& others, Scratch& lds) {
            for (uint32_t i = 0; i * kVectors * kThreads < s.vectors || i == 0; ++i) {
                Held h;
                h.load(s, i);
                h.list(some, others, lds);
            }
        }
    };

    // The largest of the threads' values.
    static __device__ __forceinline__ float peak_of(float largest, Scratch& lds) {
        const float m = wave_max(largest);
        if (threadIdx.x % kWave == 0) lds.wave_count[threadIdx.x / kWave] = __float_as_uint(m);
        __syncthreads();
        float all = -__builtin_inff();
#pragma unroll
        for (uint32_t i = 0; i < kWaves; ++i) all = fmaxf(all, __uint_as_float(lds.wave_count[i]));
        return all;
    }
    // The first id of those with the value peak, ~0 where there is none.
    template <typename V>
    static __device__ __forceinline__ uint32_t first_with(V& values, float peak, Scratch& lds) {
        if (threadIdx.x == 0) lds.lowest = ~0u;
        __syncthreads();
        uint32_t id = ~0u;
        values.each([&](float l, uint32_t i) {
            if (l == peak) id = i < id ? i : id;
        });
        if (id != ~0u) __hip_atomic_fetch_min(&lds.lowest, id, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        __syncthreads();
        return lds.lowest;
    }

    // The workgroup's row of up to kThreads: those whose candidates are all weighed first,
    // greedy ones last. (Rows come to more than the compute units, one each at a time, and
    // what begins last should not take longest.)
    static __device__ __forceinline__ uint32_t ordered_row(const Args& a, Scratch& lds) {
        const uint32_t t = threadIdx.x, w = t / kWave, l = t % kWave;
        uint32_t kind = 3;
        if (t < a.rows) {
            const vkml_sampling o = options_of(a, t);
            kind = greedy(o) ? 2 : lists_first(o, 1) ? 1 : 0;
        }
        uint32_t* counts = lds.sub_count;  // [3, kWaves]
        uint64_t mine = 0;
#pragma unroll
        for (uint32_t k = 0; k < 3; ++k) {
            const uint64_t of = __ballot(kind == k);
            if (kind == k) mine = of;
            if (l == 0) counts[k * kWaves + w] = static_cast<uint32_t>(__builtin_popcountll(of));
        }
        __syncthreads();
        static_assert(3 * kWaves <= kWave);
        const uint32_t n = l < 3 * kWaves ? counts[l] : 0u, upto = static_cast<uint32_t>(inclusive_sum(static_cast<int32_t>(n)));
        const uint32_t in = static_cast<uint32_t>(__builtin_ctzll(__ballot(upto > blockIdx.x)));  // the kind's and wave's
        const uint32_t before = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(upto - n), in));
        if (kind == in / kWaves && w == in % kWaves && static_cast<uint32_t>(__builtin_popcountll(mine & ((1ull << l) - 1))) == blockIdx.x - before) lds.found = t;
        __syncthreads();
        return lds.found;
    }

    // Clears the bins; with a barrier after it.
    static __device__ __forceinline__ void clear_bins(Scratch& lds) {
        for (uint32_t i = threadIdx.x; i < kBins; i += kThreads) lds.mass[i] = 0, lds.count[i] = 0;
        if (threadIdx.x == 0) lds.likely = 0, lds.listed = 0;
        __syncthreads();
    }
    // The candidates' weights to the bins, and the mass within min_p. A barrier has to
    // follow.
    template <typename V>
    static __device__ __forceinline__ void fill_bins(V& values, const Row& r, const vkml_sampling& o, Scratch& lds) {
        values.each([&](float l, uint32_t) {
            const Turns t = turns_of(r, l);
            if (!t.candidate(r)) return;
            add(&lds.count[t.bin()], 1u);
            add(&lds.mass[t.bin()], weight_of(r, t, lds.table));
        });
        if (r.least == 0) return;
        uint64_t likely = 0;
        const double to = kMagic + likely_turns(o);
        values.each([&](float l, uint32_t) {
            const Turns t = turns_of(r, l);
            if (t.sum >= to || !t.candidate(r)) return;
            const uint64_t w = weight_of(r, t, lds.table);
            if (w >= r.least) likely += w;
        });
        if (likely) add(&lds.likely, likely);
    }

    // What of N parts becomes that of the part and all before it. A barrier has to come
    // before; one comes after.
    template <uint32_t N, bool MASS>
    static __device__ __forceinline__ void sum_up(uint64_t* mass, uint32_t* count, Scratch& lds) {
        constexpr uint32_t kEach = N / kThreads;
        const uint32_t t = threadIdx.x, w = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(t / kWave)));
        uint64_t m[kEach], ms = 0, mi = 0;
        uint32_t c[kEach], cs = 0;
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
            if constexpr (MASS) ms = m[i] = ms + mass[kEach * t + i];
            cs = c[i] = cs + count[kEach * t + i];
        }
        if constexpr (MASS) mi = static_cast<uint64_t>(inclusive_sum(static_cast<int64_t>(ms)));
        const uint32_t ci = static_cast<uint32_t>(inclusive_sum(static_cast<int32_t>(cs)));
        if (t % kWave == kWave - 1) lds.wave_mass[w] = mi, lds.wave_count[w] = ci;
        __syncthreads();
        // the sums of the waves before: a lane each, summed up by every wave
        const uint32_t l = t % kWave % kWaves;
        uint64_t m0 = 0;
        uint32_t c0 = 0;
        if constexpr (MASS) {
            const uint64_t all = static_cast<uint64_t>(inclusive_sum(static_cast<int64_t>(lds.wave_mass[l])));
            if (w > 0) m0 = lane_of(all, w - 1);
        }
        const int32_t all = inclusive_sum(static_cast<int32_t>(lds.wave_count[l]));
        if (w > 0) c0 = static_cast<uint32_t>(__builtin_amdgcn_readlane(all, w - 1));
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
            if constexpr (MASS) mass[kEach * t + i] = m0 + mi - ms + m[i];
            count[kEach * t + i] = c0 + ci - cs + c[i];
        }
        __syncthreads();
    }

    // What is searched for: the candidate that `before` others come before, or that
    // holds unit `before` of the mass.
    struct Wanted {
        bool by_count;
        uint64_t before;
    };

    // The part of N (summed up) that holds it: its number, what is in it, and what comes
    // before it.
    struct Part {
        uint32_t i, count;
        uint64_t mass_before;
        uint32_t count_before;
    };
    template <uint32_t N>
    static __device__ __forceinline__ Part part_with(const uint64_t* mass, const uint32_t* count, Wanted x, Scratch& lds) {
#pragma unroll
        for (uint32_t i = threadIdx.x; i < N; i += kThreads) {
            const uint64_t m0 = i ? mass[i - 1] : 0;
            const uint32_t c0 = i ? count[i - 1] : 0;
            const bool here = x.by_count ? c0 <= x.before && x.before < count[i] : m0 <= x.before && x.before < mass[i];
            if (here) lds.found = i, lds.found_count = count[i] - c0, lds.found_mass = m0, lds.found_before = c0;
        }
        __syncthreads();
        const Part p{lds.found, lds.found_count, lds.found_mass, static_cast<uint32_t>(lds.found_before)};
        __syncthreads();
        return p;
    }

    // What was found: its mass and all before it, and its id.
    struct Found {
        uint64_t mass;
        uint32_t id;
    };

    // The candidate with x before it, of those that visit(f) gives, f(place, weight), with
    // places in lo .. hi, n of them in all; mass: what comes before these.
    template <typename Visit>
    static __device__ __forceinline__ Found among(const Visit& visit, Wanted x, uint64_t lo, uint64_t hi, uint32_t n, uint64_t mass, Scratch& lds) {
        // Ranges of a thousandth of the last, until few are in one. (Places are all
        // different: the seventh at the latest is a place.)
        for (int level = 0; n > kFew && level < 7; ++level) {
            const int bits = 64 - __builtin_clzll(hi - lo | 1);
            const int step = bits > 10 ? bits - 10 : 0;
            for (uint32_t i = threadIdx.x; i < kSubs; i += kThreads) lds.sub_mass[i] = 0, lds.sub_count[i] = 0;
            __syncthreads();
            visit([&](uint64_t at, uint64_t w) {
                if (at < lo || at > hi) return;
                const uint32_t i = static_cast<uint32_t>((at - lo) >> step);
                add(&lds.sub_mass[i], w);
                add(&lds.sub_count[i], 1u);
            });
            __syncthreads();
            sum_up<kSubs, true>(lds.sub_mass, lds.sub_count, lds);
            const Part p = part_with<kSubs>(lds.sub_mass, lds.sub_count, x, lds);
            mass += p.mass_before;
            x.before -= x.by_count ? p.count_before : p.mass_before;
            n = p.count;
            lo += static_cast<uint64_t>(p.i) << step;
            const uint64_t end = lo + ((1ull << step) - 1);
            hi = end < hi ? end : hi;
        }
        if (threadIdx.x == 0) lds.listed = 0;
        __syncthreads();
        visit([&](uint64_t at, uint64_t w) {
            if (at < lo || at > hi) return;
            const uint32_t i = taken(&lds.listed, 1);
            if (i < kFew) lds.few_place[i] = at, lds.few_weight[i] = w;
        });
        __syncthreads();
        const uint32_t j = threadIdx.x / 4;
        if (j < min(n, kFew)) {
            const Ranked k = ranked(lds.few_place, lds.few_weight, j, min(n, kFew));
            const bool here = x.by_count ? k.before == x.before : k.mass <= x.before && x.before < k.mass + lds.few_weight[j];
            if (here && threadIdx.x % 4 == 0) lds.found_mass = mass + k.mass + lds.few_weight[j], lds.found = static_cast<uint32_t>(lds.few_place[j]);
        }
        __syncthreads();
        const Found f{lds.found_mass, lds.found};
        __syncthreads();
        return f;
    }

    // How many of n come before the j-th, and their mass, by four threads.
    struct Ranked {
        uint32_t before;
        uint64_t mass;
    };
    static __device__ __forceinline__ Ranked ranked(const uint64_t* places, const uint64_t* weights, uint32_t j, uint32_t n) {
        const uint64_t at = places[j];
        uint64_t m = 0;
        uint32_t c = 0;
        for (uint32_t i = threadIdx.x % 4; i < n; i += 4)
            if (places[i] < at) m += weights[i], ++c;
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) m += exchanged(m, o), c += static_cast<uint32_t>(__shfl_xor(static_cast<int>(c), o));
        return {c, m};
    }

    // Which bins' candidates the list in the LDS holds all of.
    struct Range {
        uint32_t first = 1, last = 0;
        __device__ __forceinline__ bool holds(uint32_t b) const { return first <= b && b <= last; }
    };
    struct Listed {
        Range some, others;
        uint32_t n = 0;
        __device__ __forceinline__ bool holds(uint32_t b) const { return some.holds(b) || others.holds(b); }
    };

    // The places and weights of the n listed ids. With a barrier after it.
    static __device__ __forceinline__ void weigh_listed(const Source& source, const Row& r, uint32_t n, Scratch& lds) {
        for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
            const uint32_t id = lds.id[i];
            const float l = source.value(id);
            lds.place[i] = place_of(l, id);
            lds.weight[i] = weight_of(r, turns_of(r, l), lds.table);
        }
        __syncthreads();
    }

    // The bins that the draw may fall in once top_p has cut within part p.
    static __device__ __forceinline__ Range drawn_after(const Part& p, const Row& r, double random, Scratch& lds) {
        const uint64_t least = within(r, p.mass_before + 1, lds.likely), most = within(r, lds.mass[p.i], lds.likely);
        const uint32_t first = part_with<kBins>(lds.mass, lds.count, {false, unit_of(random, least)}, lds).i;
        return {first, part_with<kBins>(lds.mass, lds.count, {false, unit_of(random, most)}, lds).i};
    }

    // What to list of a row whose bins are summed up, for part p: its candidates, and all
    // before them if they fit too; else those that the draw may ask for, if that comes
    // next. None where its own are more than fit.
    static __device__ __forceinline__ Listed to_list(const Part& p, bool cut, const Row& r, double random, Scratch& lds) {
        Listed listed;
        if (p.count > kList) return listed;
        listed.n = p.count_before + p.count;
        listed.some = {0, p.i};
        if (listed.n <= kList) return listed;
        listed.n = p.count;
        listed.some.first = p.i;
        if (cut) {
            Range next = drawn_after(p, r, random, lds);
            if (next.last == p.i) --next.last;  // (wraps where that is 0: then all before it fit)
            const uint32_t n = next.holds(next.first) ? lds.count[next.last] - (next.first ? lds.count[next.first - 1] : 0) : 0;
            if (n > 0 && n + listed.n <= kList) listed.others = next, listed.n += n;
        }
        return listed;
    }
    static __device__ __forceinline__ Bounds bounds_of(const Row& r, const Range& bins) { return bins.holds(bins.first) ? Bounds{r, bins.first, bins.last} : Bounds{}; }

    // The candidate with x before it, in the bins' sums and the row's values; cut: the
    // draw comes next.
    static __device__ __forceinline__ Found find(Streamed values, const Row& r, Wanted x, bool cut, double random, Listed& listed, Scratch& lds) {
        const Part p = part_with<kBins>(lds.mass, lds.count, x, lds);
        x.before -= x.by_count ? p.count_before : p.mass_before;
        const uint32_t b = p.i;
        if (p.count <= kList && !listed.holds(b)) {
            listed = to_list(p, cut, r, random, lds);
            if (threadIdx.x == 0) lds.listed = 0;
            __syncthreads();
            values.list(bounds_of(r, listed.some), bounds_of(r, listed.others), lds);
            __syncthreads();
            weigh_listed(values.s, r, listed.n, lds);
        }
        const bool from_list = listed.holds(b);
        const auto visit = [&](const auto& f) {  // (more than the list holds: they are read again)
            if (from_list) {
                for (uint32_t i = threadIdx.x; i < listed.n; i += kThreads)
                    if (turns_of(r, logit_at(lds.place[i])).bin() == b) f(lds.place[i], lds.weight[i]);
            } else {
                values.each([&](float l, uint32_t id) {
                    const Turns t = turns_of(r, l);
                    if (t.candidate(r) && t.bin() == b) f(place_of(l, id), weight_of(r, t, lds.table));
                });
            }
        };
        uint64_t lo = 0, hi = kNone;
        if (p.count > kFew) {  // how far apart the bin's are
            if (threadIdx.x == 0) lds.lo = kNone, lds.hi = 0;
            __syncthreads();
            lo = kNone, hi = 0;
            visit([&](uint64_t at, uint64_t) {
                lo = at < lo ? at : lo;
                hi = at > hi ? at : hi;
            });
            lo = wave_min(lo);
            hi = ~wave_min(~hi);
            if (threadIdx.x % kWave == 0) {
                __hip_atomic_fetch_min(&lds.lo, lo, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                __hip_atomic_fetch_max(&lds.hi, hi, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            }
            __syncthreads();
            lo = lds.lo;
            hi = lds.hi;
        }
        return among(visit, x, lo, hi, p.count, p.mass_before, lds);
    }

    // The steps of a pick, each looking for a candidate by what the one before leaves:
    // top_k, top_p, the draw. Step `step`, or the next that there is; mass: what is kept.
    static __device__ __forceinline__ Wanted wanted(int& step, uint64_t& mass, uint32_t count, const Row& r, const vkml_sampling& o, double random, const Scratch& lds) {
        if (step == 0) {
            if (o.top_k > 0 && static_cast<uint32_t>(o.top_k) < count) return {true, static_cast<uint64_t>(o.top_k - 1)};
            ++step;
        }
        if (step == 1) {
            if (o.top_p < 1.0f) return {false, reach_of(o.top_p, mass) - 1};  // the last unit that top_p asks for
            ++step;
        }
        mass = within(r, mass, lds.likely);
        return {false, unit_of(random, mass)};
    }
    // The pick of a row whose bins are summed up.
    static __device__ __forceinline__ uint32_t pick(const Streamed& values, const Row& r, const vkml_sampling& o, double random, Listed listed, Scratch& lds) {
        uint64_t mass = lds.mass[kBins - 1];
        const uint32_t count = lds.count[kBins - 1];
#pragma unroll 1
        for (int step = 0;; ++step) {
            const Wanted x = wanted(step, mass, count, r, o, random, lds);
            const Found f = find(values, r, x, step == 1, random, listed, lds);
            if (step == 2) return f.id;
            mass = f.mass;
        }
    }
    // What to list for the first of its steps.
    static __device__ __forceinline__ Listed first_listed(const Row& r, const vkml_sampling& o, double random, Scratch& lds) {
        uint64_t mass = lds.mass[kBins - 1];
        int step = 0;
        const Wanted x = wanted(step, mass, lds.count[kBins - 1], r, o, random, lds);
        return to_list(part_with<kBins>(lds.mass, lds.count, x, lds), step == 1, r, random, lds);
    }

    // The same of n candidates that are listed, up to kFew: all ranked, then looked for
    // by halves.
    static __device__ __forceinline__ uint32_t pick_few(const Row& r, const vkml_sampling& o, double random, uint32_t n, Scratch& lds) {
        const uint32_t j = threadIdx.x / 4;
        if (j < n) {
            const Ranked k = ranked(lds.place, lds.weight, j, n);
            if (threadIdx.x % 4 == 0) lds.ranked_mass[k.before] = k.mass + lds.weight[j], lds.ranked_id[k.before] = static_cast<uint32_t>(lds.place[j]);
        }
        __syncthreads();
        const auto holds = [&](uint64_t unit) {  // the first whose mass and all before it pass it
            uint32_t lo = 0, hi = n - 1;
            while (lo < hi) {
                const uint32_t mid = (lo + hi) / 2;
                if (lds.ranked_mass[mid] > unit) hi = mid;
                else lo = mid + 1;
            }
            return lo;
        };
        const uint32_t k = o.top_k > 0 && static_cast<uint32_t>(o.top_k) < n ? static_cast<uint32_t>(o.top_k) : n;
        uint64_t mass = lds.ranked_mass[k - 1];
        if (o.top_p < 1.0f) mass = lds.ranked_mass[holds(reach_of(o.top_p, mass) - 1)];
        mass = within(r, mass, lds.likely);
        return lds.ranked_id[holds(unit_of(random, mass))];
    }

    // Whether the candidates that top_k or min_p keep are listed first. (top_k: of values
    // in no order the slices list about n (1 - (1 - top_k / kThreads)^(1 / 32)) of their n each:
    // 1387 of one slice at three quarters of the threads, 1178 of four at a quarter. With more
    // the list does not hold them all, and they are weighed after all: top_k 1000 of 40 rows
    // of 128256 so 78 us, weighed at once 47.)
    static __device__ __forceinline__ bool lists_first(const vkml_sampling& o, uint32_t slices) {
        return (o.top_k > 0 && static_cast<uint32_t>(o.top_k) <= kThreads / 4 * 3 && static_cast<uint64_t>(o.top_k) * slices <= kThreads) || !weighs_all(o);
    }
    // Lists them, and what else is in their bins: the ids, lds.listed of them (more than
    // the list holds: some). Largest: of the thread's values. The counts are as they were,
    // 0, and lds.listed has to be. With a barrier after it.
    static __device__ __forceinline__ void list_kept(Held& values, float largest, const Row& r, const vkml_sampling& o, Scratch& lds) {
        uint32_t last = kBins - 1;
        if (o.top_k > 0 && static_cast<uint32_t>(o.top_k) <= kThreads) {
            const Turns t = turns_of(r, largest);
            if (t.candidate(r)) add(&lds.count[t.bin()], 1u);
            __syncthreads();
            sum_up<kBins, false>(lds.mass, lds.count, lds);
            const uint32_t most = lds.count[kBins - 1], k = static_cast<uint32_t>(o.top_k);
            if (k <= most) last = part_with<kBins>(lds.mass, lds.count, {true, k - 1}, lds).i;
            else __syncthreads();
            for (uint32_t i = threadIdx.x; i < kBins; i += kThreads) lds.count[i] = 0;
        }
        values.list(Bounds{r, 0, last}, Bounds{}, lds);
        __syncthreads();
    }
    // The n listed candidates, weighed: their mass within min_p, and where they are more
    // than few, their bins. With a barrier after it.
    static __device__ __forceinline__ void bin_listed(const Row& r, uint32_t n, Scratch& lds) {
        uint64_t likely = 0;
        for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
            const uint64_t w = lds.weight[i];
            if (r.least != 0 && w >= r.least) likely += w;
            if (n > kFew) {
                const uint32_t b = turns_of(r, logit_at(lds.place[i])).bin();
                add(&lds.count[b], 1u);
                add(&lds.mass[b], w);
            }
        }
        if (likely) add(&lds.likely, likely);
        __syncthreads();
    }
};

// ---------------------------------------------------------------- the launches

// Rows of one slice: a workgroup a row, its values in registers. (Of up to 8192 logits:
// 256 threads, two workgroups a compute unit. Measured, us with 256 and 1024 threads, all
// rows with top_p 0.95: 1 of 1000 12.0 and 13.3, of 4096 13.6 and 14.0, of 8192 15.7 and
// 15.0; 256 of 8192 16.9 and 16.6; 300 of 4096 16.5 and 29.6; 1024 of 4096 31 and 58, of
// 8192 37 and 64. With top_k 40 256 are ahead at all of these.)
template <uint32_t kThreads>
__global__ void __launch_bounds__(kThreads) k_sample(Args a) {
    using P = Picker<kThreads>;
    __shared__ typename P::Scratch lds;
    const uint32_t row = a.ordered ? static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(P::ordered_row(a, lds)))) : blockIdx.x;
    const vkml_sampling o = options_of(a, row);
    const typename P::Streamed again{source_of(a, row)};
    typename P::Held values;
    values.load(again.s, 0);
    P::fill_table(a.shift, lds);
    P::clear_bins(lds);
    const float largest = values.largest(), peak = P::peak_of(largest, lds);
    uint32_t id = ~0u;  // -1
    if (!(peak > -__builtin_inff())) {
    } else if (greedy(o)) {
        id = P::first_with(values, peak, lds);
    } else {
        const Row r = row_of(peak, o, a.shift);
        uint32_t n = kList + 1;
        if (P::lists_first(o, 1)) {
            P::list_kept(values, largest, r, o, lds);
            n = lds.listed;
        }
        typename P::Listed listed;
        if (n <= kList) {
            P::weigh_listed(again.s, r, n, lds);
            P::bin_listed(r, n, lds);
            listed.some = {0, kBins - 1};
            listed.n = n;
        } else {
            P::fill_bins(values, r, o, lds);
            __syncthreads();
        }
        if (n <= P::kFew) {
            id = P::pick_few(r, o, a.random[row], n, lds);
        } else {
            P::template sum_up<kBins, true>(lds.mass, lds.count, lds);
            id = P::pick(again, r, o, a.random[row], listed, lds);
        }
    }
    if (threadIdx.x == 0) stg(a.tokens + row, static_cast<int32_t>(id));
}

// Longer rows, workgroups on slices of them: each slice's largest; then what top_k or
// min_p keep of it, or its bins; for the latter rows then those candidates of each slice
// that their picks begin with, found in all slices' bins (by each slice's workgroup for
// itself: 98 KB of a row of 128256), and the bins of those that listed too much; then the
// picks. (40 rows of 128256: 48 us, 56 with the picks' workgroups looking through their
// rows by themselves.)
using Wide = Picker<kWideThreads>;

__global__ void __launch_bounds__(kWideThreads) k_sample_peaks(Args a) {
    __shared__ Wide::Scratch lds;
    Wide::Held values;
    values.load(source_of(a, blockIdx.x / a.slices), blockIdx.x % a.slices);
    const float peak = Wide::peak_of(values.largest(), lds);
    const uint32_t id = greedy(options_of(a, blockIdx.x / a.slices)) ? Wide::first_with(values, peak, lds) : 0;
    if (threadIdx.x == 0) stg(a.peaks + blockIdx.x, peak > -__builtin_inff() ? place_of(peak, id) : kNone);
}

// The place of a row's largest: the slices', a lane each.
__device__ __forceinline__ uint64_t first_of(const Args& a, uint32_t row) {
    uint64_t first = kNone;
    for (uint32_t i = threadIdx.x % kWave; i < a.slices; i += kWave) {
        const uint64_t p = ldg(a.peaks + static_cast<uint64_t>(row) * a.slices + i);
        first = p < first ? p : first;
    }
    return wave_min(first);
}

// The sums of a row's slices to the bins, two a thread, four slices' loads in flight.
// Likely has to be 0.
__device__ __forceinline__ void add_slices(const Slice* from, uint32_t slices, Wide::Scratch& lds) {
    static_assert(2 * kWideThreads == kBins);
    const uint32_t i = 2 * threadIdx.x;
    uint64_t m0 = 0, m1 = 0;
    uint32_t c0 = 0, c1 = 0;
    for (uint32_t s = 0; s < slices; s += 4) {
        uint4 m[4];
        uint2 c[4];
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
            const Sums& of = from[min(s + k, slices - 1)].sums;
            m[k] = ldg(reinterpret_cast<const uint4*>(of.mass + i));
            c[k] = ldg(reinterpret_cast<const uint2*>(of.count + i));
        }
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
            if (s + k >= slices) break;
            m0 += static_cast<uint64_t>(m[k].y) << 32 | m[k].x, m1 += static_cast<uint64_t>(m[k].w) << 32 | m[k].z;
            c0 += c[k].x, c1 += c[k].y;
        }
    }
    lds.mass[i] = m0, lds.mass[i + 1] = m1, lds.count[i] = c0, lds.count[i + 1] = c1;
    for (uint32_t s = threadIdx.x; s < slices; s += kWideThreads) add(&lds.likely, ldg(&from[s].sums.likely));
}

// How many a row's slices have listed (more than kList where these are not all).
__device__ __forceinline__ uint32_t listed_in(const Slice* from, uint32_t slices) {
    uint32_t n = 0;
    for (uint32_t s0 = 0; s0 < slices; s0 += kWave) {
        const uint32_t s = s0 + threadIdx.x % kWave, of = s < slices ? min(ldg(&from[s].listed), kList + 1) : 0u;
        n = min(n + static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(inclusive_sum(static_cast<int32_t>(of))), kWave - 1)), kList + 1);
    }
    return n;
}
// The lists, one after another, each wave some of the slices'; how many as above.
__device__ __forceinline__ uint32_t join_lists(const Slice* from, uint32_t slices, Wide::Scratch& lds) {
    uint32_t n = 0;
    for (uint32_t s0 = 0; s0 < slices; s0 += kWave) {
        const uint32_t l = threadIdx.x % kWave, of = s0 + l < slices ? min(ldg(&from[s0 + l].listed), kList + 1) : 0u;
        const uint32_t upto = static_cast<uint32_t>(inclusive_sum(static_cast<int32_t>(of)));
        for (uint32_t s = threadIdx.x / kWave; s < min(static_cast<uint32_t>(kWave), slices - s0); s += kWideThreads / kWave) {
            const uint32_t mine = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(of), s)), to = n + static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(upto), s)) - mine;
            for (uint32_t i = l; i < mine && to + i < kList; i += kWave) lds.id[to + i] = ldg(from[s0 + s].id + i);
        }
        n = min(n + static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(upto), kWave - 1)), kList + 1);
    }
    return n;
}

__device__ __forceinline__ void store_sums(Sums& to, const Wide::Scratch& lds) {
    for (uint32_t i = threadIdx.x; i < kBins; i += kWideThreads) stg(to.mass + i, lds.mass[i]), stg(to.count + i, lds.count[i]);
    if (threadIdx.x == 0) stg(&to.likely, lds.likely);
}
// A slice's weights, by bins that are 0.
__device__ __forceinline__ void sum_slice(const Args& a, Wide::Held& values, const Row& r, const vkml_sampling& o, Sums& to, Wide::Scratch& lds) {
    Wide::fill_table(a.shift, lds);
    __syncthreads();
    Wide::fill_bins(values, r, o, lds);
    __syncthreads();
    store_sums(to, lds);
}

__global__ void __launch_bounds__(kWideThreads) k_sample_slices(Args a) {
    __shared__ Wide::Scratch lds;
    const uint32_t row = blockIdx.x / a.slices;
    const vkml_sampling o = options_of(a, row);
    const uint64_t first = first_of(a, row);
    if (first == kNone || greedy(o)) return;
    const Source source = source_of(a, row);
    Wide::Held values;
    values.load(source, blockIdx.x % a.slices);
    const Row r = row_of(logit_at(first), o, a.shift);
    Wide::clear_bins(lds);
    Slice* to = a.parts + blockIdx.x;
    if (Wide::lists_first(o, a.slices)) {
        Wide::list_kept(values, values.largest(), r, o, lds);
        const uint32_t n = lds.listed;
        if (threadIdx.x == 0) stg(&to->listed, n);
        if (n > kList) return;
        for (uint32_t i = threadIdx.x; i < n; i += kWideThreads) stg(to->id + i, lds.id[i]);
        return;
    }
    sum_slice(a, values, r, o, to->sums, lds);
}

__global__ void __launch_bounds__(kWideThreads) k_sample_list(Args a) {
    __shared__ Wide::Scratch lds;
    const uint32_t row = blockIdx.x / a.slices, slice = blockIdx.x % a.slices;
    const vkml_sampling o = options_of(a, row);
    const uint64_t first = first_of(a, row);
    if (greedy(o) || first == kNone) return;
    const Slice* parts = a.parts + static_cast<uint64_t>(row) * a.slices;
    const bool lists = Wide::lists_first(o, a.slices);
    if (lists && listed_in(parts, a.slices) <= kList) return;
    Wide::Held values;
    values.load(source_of(a, row), slice);
    const Row r = row_of(logit_at(first), o, a.shift);
    if (lists) {
        Wide::clear_bins(lds);
        return sum_slice(a, values, r, o, a.parts[blockIdx.x].sums, lds);
    }
    if (threadIdx.x == 0) lds.likely = 0, lds.listed = 0;
    __syncthreads();
    add_slices(parts, a.slices, lds);
    __syncthreads();
    Wide::sum_up<kBins, true>(lds.mass, lds.count, lds);
    if (slice == 0) store_sums(a.totals[row], lds);
    const Wide::Listed listed = Wide::first_listed(r, o, a.random[row], lds);
    if (listed.n > 0) values.list(Wide::bounds_of(r, listed.some), Wide::bounds_of(r, listed.others), lds);
    __syncthreads();
    Slice* to = a.parts + blockIdx.x;
    const uint32_t n = min(lds.listed, kList);
    for (uint32_t i = threadIdx.x; i < n; i += kWideThreads) stg(to->id + i, lds.id[i]);
    if (threadIdx.x == 0) stg(&to->listed, n);
}

__global__ void __launch_bounds__(kWideThreads) k_sample_pick(Args a) {
    __shared__ Wide::Scratch lds;
    const uint32_t row = blockIdx.x;
    const vkml_sampling o = options_of(a, row);
    const uint64_t first = first_of(a, row);
    uint32_t id = ~0u;  // -1
    if (first == kNone) {
    } else if (greedy(o)) {
        id = static_cast<uint32_t>(first);
    } else {
        const Row r = row_of(logit_at(first), o, a.shift);
        Wide::Streamed values{source_of(a, row)};
        const bool lists = Wide::lists_first(o, a.slices);
        Wide::fill_table(a.shift, lds);
        if (lists) {
            Wide::clear_bins(lds);
        } else {
            const Sums* sums = a.totals + row;
            for (uint32_t i = threadIdx.x; i < kBins; i += kWideThreads) lds.mass[i] = ldg(sums->mass + i), lds.count[i] = ldg(sums->count + i);
            if (threadIdx.x == 0) lds.likely = ldg(&sums->likely);
        }
        const Slice* parts = a.parts + static_cast<uint64_t>(row) * a.slices;
        const uint32_t n = join_lists(parts, a.slices, lds);
        __syncthreads();
        Wide::Listed listed;
        if (n <= kList) Wide::weigh_listed(values.s, r, n, lds);
        if (!lists) {
            if (n > 0) listed = Wide::first_listed(r, o, a.random[row], lds);
        } else if (n <= kList) {
            Wide::bin_listed(r, n, lds);
            listed.some = {0, kBins - 1};
            listed.n = n;
        } else {
            add_slices(parts, a.slices, lds);
            __syncthreads();
        }
        if (lists && n <= Wide::kFew) {
            id = Wide::pick_few(r, o, a.random[row], n, lds);
        } else {
            if (lists) Wide::sum_up<kBins, true>(lds.mass, lds.count, lds);
            id = Wide::pick(values, r, o, a.random[row], listed, lds);
        }
    }
    if (threadIdx.x == 0) stg(a.tokens + row, static_cast<int32_t>(id));
}

bool aligned(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

}  // namespace

extern "C" {

uint64_t vkml_sample_workspace_bytes(const vkml_sample_params* p) { return !p || check(*p) ? 0 : workspace_bytes(*p); }

int vkml_sample(const vkml_sample_params* p, const float* logits, const vkml_sampling* options, const double* random, void* workspace, int32_t* tokens) {
    VKML_REQUIRE_INIT();
    VKML_CHECK_ARG(p, "sample: null params");
    if (const char* why = check(*p)) return vkml::abi::fail(VKML_ERROR_INVALID_ARGUMENT, std::string("sample: ") + why);
    if (p->rows == 0) return VKML_OK;
    VKML_CHECK_ARG(logits && options && random && tokens && (workspace || workspace_bytes(*p) == 0), "sample: null buffer");
    VKML_CHECK_ARG(aligned(logits, 4) && aligned(options, 16) && aligned(random, 8) && aligned(tokens, 4) && aligned(workspace, 16),
                   "sample: options and the workspace must be 16-byte aligned, the other buffers as their types are");
    Args a{};
    a.logits = logits;
    a.options = options;
    a.random = random;
    a.tokens = tokens;
    a.row_stride = p->row_stride;
    a.rows = p->rows;
    a.vocab = p->vocab;
    a.slices = slices(p->vocab);
    if (a.slices > 1) {
        a.peaks = static_cast<uint64_t*>(workspace);
        a.totals = reinterpret_cast<Sums*>(static_cast<uint8_t*>(workspace) + peaks_bytes(*p));
        a.parts = reinterpret_cast<Slice*>(a.totals + p->rows);
    }
    // a row's weights fit 62 bits, one of them 51
    int32_t bits = 0;
    while ((1u << bits) < p->vocab) ++bits;
    a.shift = 62 - bits < 51 ? 62 - bits : 51;
    vkml::abi::ProfileScope prof("sample");
    const auto go = [&](auto kernel, uint32_t workgroups, uint32_t threads) {
        hipLaunchKernelGGL(kernel, dim3(workgroups), dim3(threads), 0, vkml::abi::stream(), a);
        return vkml::abi::check_launch("sample");
    };
    if (p->vocab <= kNarrowRow) return go(k_sample<kNarrowThreads>, p->rows, kNarrowThreads);
    // Measured (us, the requests mixed): 416 rows of 32768 47 as they come, 32 in order;
    // 1024 97 and 76.
    a.ordered = p->rows > vkml::abi::compute_units() && p->rows <= kWideThreads;
    if (a.slices == 1) return go(k_sample<kWideThreads>, p->rows, kWideThreads);
    if (const int r = go(k_sample_peaks, p->rows * a.slices, kWideThreads)) return r;
    if (const int r = go(k_sample_slices, p->rows * a.slices, kWideThreads)) return r;
    if (const int r = go(k_sample_list, p->rows * a.slices, kWideThreads)) return r;
    return go(k_sample_pick, p->rows, kWideThreads);
}

}  // extern "C"
