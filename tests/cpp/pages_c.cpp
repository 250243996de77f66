// The checks and the batch arithmetic of csrc/pages.hpp as C functions, for
// test_pages.py.
#include "pages.hpp"

using namespace vkml::pages;

extern "C" const char* check_attend_c(const vkml_attend_pages_params* p) { return check(*p); }
extern "C" const char* check_rope_c(const vkml_rope_kv_pages_params* p) { return check(*p); }
extern "C" const char* check_copy_c(const vkml_copy_pages_params* p) { return check(*p); }
extern "C" const char* check_copies_c(uint32_t pages, uint32_t count, const int32_t* src, const int32_t* dst, uint64_t* marks) {
    return check_copies(pages, count, src, dst, marks);
}

// out [seqs, 5]: first row, rows, length, group, shared keys
extern "C" void batch_c(const Batch* b, int32_t* out) {
    for (int32_t s = 0; s < b->seqs; ++s) {
        const int32_t g = b->groups > 0 && b->group_start(b->group_near(s)) <= s && s < b->group_start(b->group_near(s) + 1) ? b->group_near(s) : -1;
        out[5 * s] = b->start(s);
        out[5 * s + 1] = b->count(s);
        out[5 * s + 2] = b->length(s);
        out[5 * s + 3] = g;
        out[5 * s + 4] = g < 0 ? 0 : b->group_start(g + 1) - b->group_start(g) > 1 ? b->group_key(g) : 0;
    }
}

// The whole work of a call as its workgroups cut it, a piece a row: workgroup,
// KV head, segment, tile, first key, last key + 1, slot, few, whole, pieces of
// the tile (as its first piece says). Returns the number of pieces.
extern "C" int64_t pieces_c(const Batch* b, int32_t kv_heads, int32_t group, int32_t head_dim, int32_t f16, int32_t workgroups_log2, int32_t block, int64_t* out, int64_t most) {
    const int32_t segments = b->groups + b->seqs;
    const Costs cost_of = costs(head_dim, f16 != 0);
    int64_t per_head = 0, n = 0;
    for (int32_t i = 0; i < segments; ++i) per_head += segment(*b, group, cost_of, i).cost();
    const int64_t cost = per_head * kv_heads;
    if (cost == 0) return 0;
    const int32_t w_log2 = parts_log2(cost, workgroups_log2);
    for (int32_t w = 0; w < 1 << w_log2; ++w) {
        const int64_t u0 = part_start(cost, w_log2, w), u1 = part_start(cost, w_log2, w + 1);
        int64_t off = 0, few = 0, tiles = 0;
        for (int32_t h = 0; h < kv_heads; ++h)
            for (int32_t i = 0; i < segments; ++i) {
                const Segment s = segment(*b, group, cost_of, i);
                for (int32_t t = 0; t < s.tiles; ++t) {
                    const int64_t at = off + s.before(t);
                    const int32_t c = s.tile_cost(t), keys = s.keys(t);
                    // the part's range within the tile, as its workgroup finds it
                    if (u0 >= at + c || u1 <= at) continue;
                    const int32_t from = u0 > at ? snap(u0 - at, s, c) : 0, to = snap(u1 - at, s, c);
                    if (from >= to) continue;
                    if (n >= most) return -1;
                    int64_t* o = out + 10 * n++;
                    o[0] = w, o[1] = h, o[2] = i, o[3] = t;
                    o[4] = cut(from, s, keys, block);
                    o[5] = to == c ? keys : cut(to, s, keys, block);
                    o[6] = w + (s.few ? few : tiles + t);
                    o[7] = s.few;
                    o[8] = from == 0 && to == c;
                    o[9] = from == 0 ? (to == c ? 1 : pieces_of(cost, w_log2, s, at, c, w)) : -1;
                }
                off += s.cost();
                (s.few ? few : tiles) += s.tiles;
            }
    }
    return n;
}

// The KV head that part w of the work of kv_heads equal ones begins in, found by division, and by shift.
extern "C" int32_t first_head_c(int64_t per_head, int32_t kv_heads, int32_t w_log2, int32_t w) {
    return static_cast<int32_t>(part_start(per_head * kv_heads, w_log2, w) / per_head) - (kv_heads * w >> w_log2);
}

// {few, tile} slots
extern "C" void slots_c(int64_t kv_heads, int64_t group, int64_t seqs, int64_t groups, int64_t tokens, int64_t workgroups, int64_t* out) {
    const Slots s = slots(kv_heads, group, seqs, groups, tokens, workgroups);
    out[0] = s.few, out[1] = s.tile;
}
// A segment's token0, n, lo, from, keys of its last tile, tiles, step, row, shared, lead, lead_row, lead_span
extern "C" void segment_c(const Batch* b, int32_t group, int32_t i, int32_t* out) {
    const Segment s = segment(*b, group, costs(128, true), i);
    const int32_t v[] = {s.token0, s.n, s.lo(), s.from, s.tiles ? s.keys(s.tiles - 1) : 0, s.tiles, s.step, s.row, s.shared, s.lead, s.lead_row, s.lead_span()};
    for (int k = 0; k < 12; ++k) out[k] = v[k];
}
extern "C" int32_t limit_c(const Batch* b, int32_t group, int32_t i, int32_t token) { return segment(*b, group, costs(128, true), i).limit(token); }

extern "C" void grid_c(uint32_t workgroups, uint32_t* out) {
    const Grid g = grid_of(workgroups);
    out[0] = g.x, out[1] = g.y;
}

// Segment i's cost, and for each tile: its cost, what comes before it, and the
// tile that its first and its last unit are found in.
extern "C" int64_t costs_c(const Batch* b, int32_t group, int32_t head_dim, int32_t f16, int32_t i, int64_t* out, int64_t most) {
    const Segment s = segment(*b, group, costs(head_dim, f16 != 0), i);
    for (int32_t t = 0; t < s.tiles && t < most; ++t) {
        int64_t* o = out + 4 * t;
        o[0] = s.tile_cost(t), o[1] = s.before(t);
        o[2] = s.tile_at(o[1]), o[3] = s.tile_at(o[1] + o[0] - 1);
    }
    return s.cost();
}

extern "C" int64_t most_tiles_c(int64_t group, int64_t seqs, int64_t groups, int64_t tokens) { return most_tiles(group, seqs, groups, tokens); }
