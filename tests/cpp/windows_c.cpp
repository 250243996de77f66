// The checks of trees, windows, kept drafts and samples, and the division of a
// windowed call's work (csrc/pages.hpp, csrc/sample.hpp) as C functions, for
// test_windows.py.
#include "pages.hpp"
#include "sample.hpp"

using namespace vkml::pages;

extern "C" const char* check_tree_c(uint32_t words) { return check_tree(words); }
extern "C" const char* check_window_c(const vkml_attend_pages_params* p, uint32_t window) { return check_window(*p, window); }
extern "C" const char* check_keep_c(const vkml_keep_drafts_params* p) { return check(*p); }
extern "C" const char* check_sample_c(const vkml_sample_params* p) { return vkml::sample::check(*p); }
extern "C" uint64_t sample_workspace_c(const vkml_sample_params* p) { return vkml::sample::workspace_bytes(*p); }
extern "C" void window_c(const vkml_attend_pages_params* p, uint32_t window, uint32_t sinks, uint32_t block, int32_t* out) {
    const Window w = window_of(*p, window, sinks, block);
    out[0] = w.keys, out[1] = w.sinks, out[2] = w.span;
}

// A segment's token0, n, tiles, step, straight, few, lead_row, row; then for each of
// its tiles: cost, what comes before it, the tile that its first and last unit are
// found in, keys, the five of Where, the first token's limit.
extern "C" int64_t tiles_c(const Batch* b, int32_t group, int32_t head_dim, int32_t f16, int32_t i, const int32_t* window, int32_t* head, int64_t* out, int64_t most) {
    const Segment s = segment(*b, group, costs(head_dim, f16 != 0), i, Window{window[0], window[1], window[2]});
    const int32_t v[] = {s.token0, s.n, s.tiles, s.step, s.straight, s.few, s.lead_row, s.row};
    for (int k = 0; k < 8; ++k) head[k] = v[k];
    for (int32_t t = 0; t < s.tiles && t < most; ++t) {
        int64_t* o = out + 11 * t;
        const Segment::Where in = s.where(t);
        o[0] = s.tile_cost(t), o[1] = s.before(t);
        o[2] = s.tile_at(o[1]), o[3] = s.tile_at(o[1] + o[0] - 1);
        o[4] = s.keys(t);
        o[5] = in.span, o[6] = in.lead, o[7] = in.lo, o[8] = in.from, o[9] = in.end;
        o[10] = s.limit(t * s.step);
    }
    return s.cost();
}

// The pieces of a windowed call: KV head, segment, tile, first key, last key + 1.
extern "C" int64_t window_pieces_c(const Batch* b, int32_t kv_heads, int32_t group, int32_t head_dim, int32_t f16, const int32_t* window, int32_t workgroups_log2, int32_t block, int64_t* out, int64_t most) {
    const Costs cost_of = costs(head_dim, f16 != 0);
    const Window win{window[0], window[1], window[2]};
    int64_t per_head = 0, n = 0;
    for (int32_t i = 0; i < b->seqs; ++i) per_head += segment(*b, group, cost_of, i, win).cost();
    const int64_t cost = per_head * kv_heads;
    if (cost == 0) return 0;
    const int32_t w_log2 = parts_log2(cost, workgroups_log2);
    for (int32_t w = 0; w < 1 << w_log2; ++w) {
        const int64_t u0 = part_start(cost, w_log2, w), u1 = part_start(cost, w_log2, w + 1);
        int64_t off = 0;
        for (int32_t h = 0; h < kv_heads; ++h)
            for (int32_t i = 0; i < b->seqs; ++i) {
                const Segment s = segment(*b, group, cost_of, i, win);
                for (int32_t t = 0; t < s.tiles; ++t) {
                    const int64_t at = off + s.before(t);
                    const int32_t c = s.tile_cost(t), keys = s.keys(t);
                    if (u0 >= at + c || u1 <= at) continue;
                    const int32_t from = u0 > at ? snap(u0 - at, s, c) : 0, to = snap(u1 - at, s, c);
                    if (from >= to) continue;
                    if (n >= most) return -1;
                    int64_t* o = out + 6 * n++;
                    o[0] = h, o[1] = i, o[2] = t;
                    o[3] = cut(from, s, keys, block);
                    o[4] = to == c ? keys : cut(to, s, keys, block);
                    o[5] = from == 0 ? (to == c ? 1 : pieces_of(cost, w_log2, s, at, c, w)) : -1;
                }
                off += s.cost();
            }
    }
    return n;
}
