"""Trees of drafted tokens and windows over the paged cache
(vkml_attend_pages_tree, vkml_attend_pages_window), and the drafts that stay
(vkml_keep_drafts), against plain implementations in float64. Attention's bound
is that of test_gpu_pages.py, of the keys that a token sees."""
import ctypes as C
import math

import numpy as np
import pytest

import test_gpu_pages as P
from vkml_amd import hip as H

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    H.init()
    yield
    H.synchronize()


dev, ptr, close = P.dev, P.ptr, P.close


def attention_f64(q, cache, batch, scale, sees, softcap=0.0):
    """(out, bound) of every token; sees(s, i): the positions that new token i of
    sequence s sees, those that no page holds left out here."""
    heads, hd = q.shape[1:]
    G = heads // cache.kv_heads
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for s, (length, n) in enumerate(zip(batch.lengths, batch.new)):
        kk, held = P.rows_of(cache, cache.k, batch.table[s], length)
        vv, _ = P.rows_of(cache, cache.v, batch.table[s], length)
        for i in range(n):
            t = batch.starts[s] + i
            on = np.asarray(sees(s, i), int)
            on = on[held[on]] if on.size else on
            if on.size == 0:
                continue
            for g in range(cache.kv_heads):
                K, V = kk[on, g].astype(np.float64), vv[on, g].astype(np.float64)
                Q = q[t, g * G:(g + 1) * G].astype(np.float64)
                with np.errstate(all="ignore"):
                    x = Q @ K.T * scale
                    off = scale * (2.0 ** -22 * np.abs(Q).max(1)[:, None] * np.abs(K).sum(1) + (hd + 8) * 2.0 ** -24 * (np.abs(Q) @ np.abs(K).T))
                    extra = 0.0
                    if softcap:
                        x, extra = softcap * np.tanh(x / softcap), 2.0 ** -20 * softcap
                    p = np.exp(x - x.max(1, keepdims=True))
                    p /= p.sum(1, keepdims=True)
                    out[t, g * G:(g + 1) * G] = p @ V
                    rel = 2 * (off.max(1) + extra) + 2.0 ** -22 * np.abs(x).max(1) + (on.size / 16 + 64) * 2.0 ** -24 + 2.0 ** -20
                    bound[t, g * G:(g + 1) * G] = (p @ np.abs(V)) * rel[:, None]
    return out, bound


class Call:
    """One call of the trees' or the window's attention and its buffers."""

    def __init__(self, q, cache, batch, scale, softcap=0.0, starts=True, workspace=None, seen=None, window=None):
        self.p = P.params(cache, batch, q.shape[1], scale, softcap)
        self.cache, self.batch, self.shape, self.window = cache, batch, q.shape, window
        self.q, self.out = dev(q), dev(np.full(q.shape, 7.5, np.float32))
        self.starts = batch.d_starts if starts else None
        if seen is not None:
            self.words, self.seen = seen.shape[1], dev(seen)
        need = H.lib().vkml_attend_pages_workspace_bytes(C.byref(self.p))
        self.workspace = workspace or dev(np.full(max(need, 16) // 4 + 4, -1, np.int32))

    def run(self):
        b, where = self.batch, (self.q.p, self.cache.dk.p, self.cache.dv.p, self.batch.d_table.p, self.batch.d_lengths.p, ptr(self.starts))
        if self.window is None:
            H.call("vkml_attend_pages_tree", C.byref(self.p), self.words, *where, b.d_group_starts.p if b.groups else None, b.d_group_keys.p if b.groups else None,
                   self.seen.p, self.workspace.p, self.out.p)
        else:
            H.call("vkml_attend_pages_window", C.byref(self.p), *self.window, *where, self.workspace.p, self.out.p)
        return self

    def result(self):
        return self.out.download(np.float32, self.shape)


# ---------------------------------------------------------------- trees

def random_parents(rng, n, width=4):
    return [-1] + [int(rng.integers(max(0, i - 1 - width), i)) for i in range(1, n)]


def bits_of(rows, words):
    """rows: for each token the new tokens that it sees."""
    seen = np.zeros((len(rows), words), np.uint32)
    for t, on in enumerate(rows):
        for j in on:
            seen[t, j // 32] |= np.uint32(1 << j % 32)
    return seen


def ancestors(parents):
    rows = []
    for i, p in enumerate(parents):
        rows.append((rows[p] if p >= 0 else []) + [i])
    return rows


def tree(seed, heads, kv_heads, hd, page, kv, lengths, new, groups=(), softcap=0.0, rows=None, words=None, starts=True, q_scale=1.0, stride=0, spoil=None):
    rng = np.random.default_rng(seed)
    batch = P.Batch(rng, lengths, new, page, groups)
    cache = P.Cache(rng, batch.pages, kv_heads, page, hd, kv, stride)
    batch.share(cache)
    q = (rng.standard_normal((batch.tokens, heads, hd)) * q_scale).astype(np.float32)
    if rows is None:
        rows = [r for n in new for r in ancestors(random_parents(rng, n) if n else [])]
    words = words or max(1, -(-max(new) // 32))
    seen = bits_of(rows, max(words, max([j // 32 + 1 for r in rows for j in r] or [1])))[:, :words]

    def sees(s, i):
        base = lengths[s] - new[s]
        return list(range(base)) + sorted(base + j for j in rows[batch.starts[s] + i] if j <= i and j < 32 * words)

    scale = 1.0 / math.sqrt(hd)
    want, bound = attention_f64(q, cache, batch, scale, sees, softcap)
    if spoil:
        spoil(cache, batch, rows)
    cache.upload()
    batch.upload()
    print("tree", seed, heads, kv_heads, hd, page, kv, list(lengths)[:8], list(new)[:8], groups, softcap, words, flush=True)
    got = Call(q, cache, batch, scale, softcap, starts, seen=np.ascontiguousarray(seen)).run().result()
    close(got, want, bound, loose=max(1.0, q_scale))
    return got


@pytest.mark.parametrize("kv", [H.F16, H.F32])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(4, 2), (32, 8), (8, 8), (6, 2), (5, 1), (16, 1), (128, 1)])
def test_trees(heads, kv_heads, hd, kv):
    tree(1, heads, kv_heads, hd, 16, kv, [1, 2, 17, 40, 65, 129, 300, 33], [1, 2, 3, 7, 13, 4, 31, 33])


@pytest.mark.parametrize("kv", [H.F16, H.F32])
@pytest.mark.parametrize("page", [16, 32, 128, 1024])
def test_trees_over_pages_of_any_size(page, kv):
    # ... whose new tokens begin anywhere in a page, and span several
    tree(2, 8, 2, 128, page, kv, [page + 3, 2 * page, 2 * page + 70, 900], [5, 16, 70, 60])
    tree(3, 8, 2, 64, page, kv, [page - 1, 40, 700], [12, 40, 64])


@pytest.mark.parametrize("kv", [H.F16, H.F32])
@pytest.mark.parametrize("hd", [64, 128])
def test_trees_of_many_nodes(hd, kv):
    tree(4, 8, 2, hd, 32, kv, [600, 301, 1000], [300, 301, 140])


@pytest.mark.parametrize("kv", [H.F16, H.F32])
@pytest.mark.parametrize("shared", [1, 16, 100, 1000])
def test_trees_behind_a_shared_prefix(shared, kv):
    new = [5, 1, 13, 30, 2, 8]
    tree(5, 8, 2, 128, 16, kv, [shared + n + k for n, k in zip(new, (0, 3, 20, 1, 64, 9))], new, [(0, 6, shared)])
    # many rows each: their own tiles read the shared keys
    new = [70, 64, 90]
    tree(6, 8, 2, 64, 16, kv, [shared + n + k for n, k in zip(new, (0, 3, 20))], new, [(0, 3, shared)])


@pytest.mark.parametrize("kv", [H.F16, H.F32])
def test_trees_with_a_soft_cap(kv):
    tree(7, 8, 2, 128, 16, kv, [5, 200, 333], [5, 60, 2], softcap=30.0, q_scale=6.0)


@pytest.mark.parametrize("kv", [H.F16, H.F32])
@pytest.mark.parametrize("heads,kv_heads", [(8, 2), (4, 4)])
def test_a_token_sees_what_its_bits_say(heads, kv_heads, kv):
    """Any bits: none (zeros where there are no earlier keys), not the token's
    own, and those of later tokens, which count as none."""
    rng = np.random.default_rng(8)
    new = [3, 20, 70, 2]
    rows = []
    for n in new:
        for i in range(n):
            rows.append([j for j in range(n) if rng.random() < 0.3])
    rows[0] = []      # of a sequence without earlier keys
    rows[1] = [2, 1]  # sees itself alone: 2 comes later
    rows[2] = []
    got = tree(9, heads, kv_heads, 128, 16, kv, [3, 50, 300, 2], new, rows=rows)
    assert not got[0].any() and not got[2].any()


def test_new_tokens_past_the_bits_are_seen_by_none():
    rng = np.random.default_rng(10)
    rows = ancestors(random_parents(rng, 100, 6))
    tree(11, 8, 2, 128, 16, H.F16, [150], [100], rows=rows, words=2)
    tree(11, 8, 2, 64, 16, H.F32, [100], [100], rows=rows, words=1)


def test_words_past_the_tokens_are_none():
    rng = np.random.default_rng(12)
    rows = ancestors(random_parents(rng, 7))
    tree(13, 8, 2, 128, 16, H.F16, [50], [7], rows=rows, words=128)


@pytest.mark.parametrize("kv", [H.F16, H.F32])
@pytest.mark.parametrize("hd", [64, 128])
def test_a_chain_is_causal_attention(hd, kv):
    rng = np.random.default_rng(14)
    lengths, new = [5, 64, 300, 513, 90], [5, 1, 33, 300, 2]
    batch = P.Batch(rng, lengths, new, 16)
    cache = P.Cache(rng, batch.pages, 2, 16, hd, kv).upload()
    batch.upload()
    q = rng.standard_normal((batch.tokens, 8, hd)).astype(np.float32)
    rows = [list(range(i + 1)) for n in new for i in range(n)]
    got = Call(q, cache, batch, 0.1, seen=bits_of(rows, 10)).run().result()
    want = P.Call(q, cache, batch, 0.1).run().result()
    assert np.array_equal(got.view(np.uint32), want.view(np.uint32))


@pytest.mark.parametrize("kv", [H.F16, H.F32])
@pytest.mark.parametrize("heads,kv_heads,hd", [(8, 2, 128), (4, 4, 64), (40, 2, 128)])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_what_is_not_finite_on_another_branch_leaves_a_token_alone(bad, heads, kv_heads, hd, kv):
    """Two branches; the keys and values of one are spoilt, and the other's
    outputs are as before."""
    n, rows = 21, [[0]]
    for i in range(1, n):
        rows.append((rows[i - 2] if i > 2 else rows[0]) + [i])
    odd = np.array([i for i in range(1, n, 2)])

    rng = np.random.default_rng(15)
    batch = P.Batch(rng, [n + 40], [n], 16)
    cache = P.Cache(rng, batch.pages, kv_heads, 16, hd, kv)
    q = rng.standard_normal((n, heads, hd)).astype(np.float32)
    want, bound = attention_f64(q, cache, batch, 0.1, lambda s, i: list(range(40)) + [40 + j for j in rows[i]])
    pos = 40 + odd
    cache.k[batch.table[0, pos // 16], :, pos % 16] = bad
    cache.v[batch.table[0, pos // 16], :, pos % 16] = bad
    cache.upload()
    batch.upload()
    print("branches", bad, heads, kv_heads, hd, kv, flush=True)
    got = Call(q, cache, batch, 0.1, seen=bits_of(rows, 1)).run().result()
    even = np.array([i for i in range(0, n, 2)])
    close(got[even], want[even], bound[even])
    assert not np.isfinite(got[odd]).any()


@pytest.mark.parametrize("kv", [H.F16, H.F32])
def test_infinite_values_reach_those_who_see_them(kv):
    n = 30
    rng = np.random.default_rng(16)
    rows = ancestors(random_parents(rng, n, 5))
    batch = P.Batch(rng, [n + 20], [n], 16)
    cache = P.Cache(rng, batch.pages, 2, 16, 64, kv)
    q = rng.standard_normal((n, 8, 64)).astype(np.float32)
    want, bound = attention_f64(q, cache, batch, 0.1, lambda s, i: list(range(20)) + [20 + j for j in rows[i]])
    cache.v[batch.table[0, 27 // 16], :, 27 % 16, 5] = np.inf  # node 7
    cache.upload()
    batch.upload()
    got = Call(q, cache, batch, 0.1, seen=bits_of(rows, 1)).run().result()
    hit = np.array([7 in r for r in rows])
    assert hit.any() and not hit.all()
    assert np.all(got[hit][:, :, 5] == np.inf)
    got[hit, :, 5] = want[hit, :, 5]
    close(got, want, bound)


def test_rows_behind_the_last_sequence_stay_as_they_were():
    rng = np.random.default_rng(17)
    for seen, window in ((True, None), (False, (20, 2))):
        batch = P.Batch(rng, [60, 33], [5, 3], 16)
        batch.tokens = 12  # four rows of no sequence
        cache = P.Cache(rng, batch.pages, 2, 16, 128, H.F16).upload()
        batch.upload()
        q = rng.standard_normal((12, 8, 128)).astype(np.float32)
        got = Call(q, cache, batch, 0.1, seen=np.full((12, 1), 0xFF, np.uint32) if seen else None, window=window).run().result()
        assert np.all(got[8:] == 7.5) and np.all(np.isfinite(got)) and not np.any(got[:8] == 7.5)


# ---------------------------------------------------------------- windows

def visible(window, sinks):
    def sees(length, n, i):
        pos = length - n + i
        return [p for p in range(pos + 1) if p > pos - window or p < sinks]
    return sees


def windowed(seed, heads, kv_heads, hd, page, kv, lengths, new, window, sinks, softcap=0.0, starts=True, q_scale=1.0, stride=0, give_back=True, bad=None):
    rng = np.random.default_rng(seed)
    batch = P.Batch(rng, lengths, new, page)
    cache = P.Cache(rng, batch.pages, kv_heads, page, hd, kv, stride)
    q = (rng.standard_normal((batch.tokens, heads, hd)) * q_scale).astype(np.float32)
    sees = visible(window, sinks)
    scale = 1.0 / math.sqrt(hd)
    want, bound = attention_f64(q, cache, batch, scale, lambda s, i: sees(lengths[s], new[s], i), softcap)
    for s, (length, n) in enumerate(zip(lengths, new)):
        on = np.zeros(batch.stride * page, bool)
        for i in range(n):
            on[sees(length, n, i)] = True
        if bad is not None:  # what no token sees
            pos = np.flatnonzero(~on[:length])
            cache.k[batch.table[s, pos // page], :, pos % page] = bad
            cache.v[batch.table[s, pos // page], :, pos % page] = bad
        if give_back:
            batch.table[s, ~on.reshape(-1, page).any(1)] = -1
    cache.upload()
    batch.upload()
    print("window", seed, heads, kv_heads, hd, page, kv, list(lengths)[:8], list(new)[:8], window, sinks, softcap, flush=True)
    got = Call(q, cache, batch, scale, softcap, starts, window=(window, sinks)).run().result()
    close(got, want, bound, loose=max(1.0, q_scale))


@pytest.mark.parametrize("kv", [H.F16, H.F32])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 4), (15, 0), (16, 16), (17, 4), (64, 130), (200, 4), (300, 0), (5000, 3), (2 ** 32 - 1, 2 ** 32 - 1)])
def test_decode_in_a_window(window, sinks, hd, kv):
    windowed(20, 8, 2, hd, 16, kv, [1, 2, 15, 16, 17, 33, 65, 129, 200, 301, 1000, 1333], [1] * 12, window, sinks, starts=False)


@pytest.mark.parametrize("kv", [H.F16, H.F32])
@pytest.mark.parametrize("heads,kv_heads", [(4, 2), (32, 8), (6, 2), (5, 1), (4, 4), (128, 1)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (20, 4), (150, 1)])
def test_prompts_in_a_window(window, sinks, heads, kv_heads, kv):
    windowed(21, heads, kv_heads, 128, 16, kv, [3, 70, 1, 330, 600, 45], [3, 33, 1, 130, 2, 45], window, sinks)
    windowed(22, heads, kv_heads, 64, 32, kv, [500, 700, 90, 64], [200, 3, 90, 0], window, sinks)


@pytest.mark.parametrize("kv", [H.F16, H.F32])
@pytest.mark.parametrize("page", [16, 64, 1024])
def test_windows_over_pages_of_any_size(page, kv):
    windowed(23, 8, 2, 128, page, kv, [1, page, page + 1, 3 * page + 5, 1300], [1, 1, 1, 20, 40], 100, 4)
    windowed(24, 8, 2, 64, page, kv, [3 * page + 5, 1300], [1, 100], page + 3, page + 1)


@pytest.mark.parametrize("kv", [H.F16, H.F32])
def test_windows_with_a_soft_cap(kv):
    windowed(25, 8, 2, 128, 16, kv, [5, 200, 1333], [1, 70, 2], 50, 4, softcap=30.0, q_scale=6.0)


@pytest.mark.parametrize("kv", [H.F16, H.F32])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("give_back", [True, False])
def test_what_no_token_sees_is_left_out(give_back, bad, kv):
    windowed(26, 8, 2, 128, 16, kv, [40, 500, 1000, 700], [1, 60, 1, 3], 100, 5, give_back=give_back, bad=bad)
    windowed(27, 4, 2, 64, 32, kv, [40, 500, 1000, 700], [1, 60, 1, 3], 33, 0, give_back=give_back, bad=bad)


@pytest.mark.parametrize("kv", [H.F16, H.F32])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_what_some_tokens_see_reaches_those_alone(bad, kv):
    rng = np.random.default_rng(28)
    length, n, window, sinks = 500, 80, 40, 3
    batch = P.Batch(rng, [length], [n], 16)
    cache = P.Cache(rng, batch.pages, 2, 16, 128, kv)
    q = rng.standard_normal((n, 8, 128)).astype(np.float32)
    sees = visible(window, sinks)
    want, bound = attention_f64(q, cache, batch, 0.1, lambda s, i: sees(length, n, i))
    hit = np.zeros(n, bool)
    for pos in (400, 470):
        cache.v[batch.table[0, pos // 16], :, pos % 16, 7] = bad
        hit |= np.array([pos in sees(length, n, i) for i in range(n)])
    cache.upload()
    batch.upload()
    got = Call(q, cache, batch, 0.1, window=(window, sinks)).run().result()
    assert hit.any() and not hit.all() and not np.isfinite(got[hit][:, :, 7]).any()
    got[hit, :, 7] = want[hit, :, 7]
    close(got, want, bound)


def test_a_long_window():
    windowed(29, 8, 2, 64, 64, H.F16, [70001, 9000], [1, 1], 60000, 4)
    windowed(30, 4, 1, 128, 64, H.F32, [20011], [3], 4096, 64)


@pytest.mark.parametrize("kv", [H.F16, H.F32])
@pytest.mark.parametrize("hd", [64, 128])
def test_a_window_of_all_keys_is_causal_attention(hd, kv):
    rng = np.random.default_rng(31)
    batch = P.Batch(rng, [5, 64, 300, 513, 90], [5, 1, 33, 300, 2], 16)
    cache = P.Cache(rng, batch.pages, 2, 16, hd, kv).upload()
    batch.upload()
    q = rng.standard_normal((batch.tokens, 8, hd)).astype(np.float32)
    want = P.Call(q, cache, batch, 0.1).run().result()
    for window in ((513, 0), (2 ** 32 - 1, 4)):
        got = Call(q, cache, batch, 0.1, window=window).run().result()
        assert np.array_equal(got.view(np.uint32), want.view(np.uint32))


# ---------------------------------------------------------------- both: graphs, workspaces, refusals

def test_captured_calls_follow_their_arrays_and_share_a_workspace():
    """Two graphs on one workspace, replayed by turns, with eager calls between;
    lengths, tables and bits change between replays."""
    rng = np.random.default_rng(32)
    new = [9, 20, 1]
    batch = P.Batch(rng, [300, 200, 77], new, 16, spare=40)
    cache = P.Cache(rng, batch.pages, 2, 16, 128, H.F16).upload()
    batch.upload()
    q = rng.standard_normal((batch.tokens, 8, 128)).astype(np.float32)
    rows = [r for n in new for r in ancestors(random_parents(rng, n))]
    trees = Call(q, cache, batch, 0.1, seen=bits_of(rows, 1))
    windows = Call(q, cache, batch, 0.1, window=(50, 4), workspace=trees.workspace)
    graphs = []
    for call in (trees, windows):
        H.call("vkml_graph_begin")
        call.run()
        g = C.c_uint64()
        H.call("vkml_graph_end", C.byref(g))
        graphs.append(g)
    sees = visible(50, 4)
    for k in range(4):
        if k:
            batch.lengths = [int(x) for x in rng.integers(30, 300, 3)]
            batch.d_lengths.upload(np.asarray(batch.lengths, np.int32))
            batch.table = rng.permutation(batch.pages)[:batch.table.size].reshape(batch.table.shape).astype(np.int32)
            batch.d_table.upload(batch.table)
            rows = [r for n in new for r in ancestors(random_parents(rng, n))]
            trees.seen.upload(bits_of(rows, 1))
        for g in graphs:
            H.call("vkml_graph_launch", g)
        first, second = trees.result(), windows.result()
        bases = [n - m for n, m in zip(batch.lengths, new)]
        close(first, *attention_f64(q, cache, batch, 0.1, lambda s, i: list(range(bases[s])) + [bases[s] + j for j in rows[batch.starts[s] + i]]))
        close(second, *attention_f64(q, cache, batch, 0.1, lambda s, i: sees(batch.lengths[s], new[s], i)))
        assert np.array_equal(trees.run().result(), first) and np.array_equal(windows.run().result(), second)
    for g in graphs:
        H.call("vkml_graph_destroy", g)


def refused(name, *args):
    assert getattr(H.lib(), name)(*args) == 1
    return H.lib().vkml_last_error().decode()


def test_trees_and_windows_refuse():
    rng = np.random.default_rng(33)
    batch = P.Batch(rng, [20, 30], [1, 1], 16)
    cache = P.Cache(rng, batch.pages, 2, 16, 64, H.F16).upload()
    batch.upload()
    b, q, out, seen, ws = batch, dev(np.zeros((2, 4, 64), np.float32)), dev(np.zeros((2, 4, 64), np.float32)), dev(np.ones((2, 1), np.uint32)), dev(np.zeros(100000, np.int32))
    p = P.params(cache, batch, 4, 0.1)

    def args(own, seen=None, q=q, ws=ws, table=b.d_table, k=cache.dk, window=False):
        where = (ptr(q), ptr(k), cache.dv.p, ptr(table), b.d_lengths.p, None)
        return (C.byref(p), *own, *where, ptr(ws), out.p) if window else (C.byref(p), *own, *where, None, None, ptr(seen), ptr(ws), out.p)

    for why, a in (("seen_words", args((0,), seen)), ("seen_words", args((129,), seen)), ("null buffer", args((1,))), ("null buffer", args((1,), seen, q=None)),
                   ("null buffer", args((1,), seen, ws=None))):
        assert why in refused("vkml_attend_pages_tree", *a), why
    for why, a in (("window", args((0, 4), window=True)), ("null buffer", args((5, 4), table=None, window=True)), ("null buffer", args((5, 4), k=None, window=True))):
        assert why in refused("vkml_attend_pages_window", *a), why
    p.groups = 1
    assert "groups" in refused("vkml_attend_pages_window", *args((5, 4), window=True))
    p.groups, p.head_dim = 0, 96
    assert "head_dim" in refused("vkml_attend_pages_tree", *args((1,), seen)) and "head_dim" in refused("vkml_attend_pages_window", *args((5, 4), window=True))
    assert "null params" in refused("vkml_attend_pages_tree", None, 1, *[None] * 11)
    assert "null params" in refused("vkml_attend_pages_window", None, 1, 1, *[None] * 8)
    p.head_dim, p.seqs, p.tokens = 64, 0, 0
    for name, own in (("vkml_attend_pages_tree", args((1,))), ("vkml_attend_pages_window", args((5, 4), window=True))):
        assert getattr(H.lib(), name)(*own) == 0


# ---------------------------------------------------------------- the drafts that stay

def walk(parents, drafted, picked):
    path = []
    if len(parents):
        path = [0]
        while True:
            after = [i for i in range(path[-1] + 1, min(len(parents), 4096)) if parents[i] == path[-1] and drafted[i] == picked[path[-1]]]
            if not after:
                break
            path.append(after[0])
    return path


class Keep:
    def __init__(self, rng, lengths, new, kv_heads, hd, page, kv, layers=2, stride=0, layer_stride=0, spare=2, base16=True):
        self.batch = P.Batch(rng, lengths, new, page, spare=spare)
        self.dtype = np.float16 if kv == H.F16 else np.float32
        self.layers, self.pages, self.kv_heads, self.hd, self.page = layers, self.batch.pages, kv_heads, hd, page
        self.stride = stride or kv_heads * page * hd
        self.layer_stride = layer_stride or self.pages * self.stride
        self.k, self.v = (rng.standard_normal((layers, self.layer_stride)).astype(self.dtype) for _ in range(2))
        self.p = H.KeepDraftsParams(kv_heads=kv_heads, head_dim=hd, kv_type=kv, page_size=page, pages=self.pages, layers=layers, seqs=len(lengths), tokens=self.batch.tokens,
                                    table_stride=self.batch.stride, page_stride=stride, layer_stride=layer_stride)
        self.offset = 0 if base16 else 4 // np.dtype(self.dtype).itemsize  # pools that start 4 bytes past a multiple of 16

    def upload(self, parents, drafted, picked):
        self.batch.upload()
        self.dk, self.dv = (dev(np.concatenate([np.zeros(self.offset, self.dtype), x.ravel()])) for x in (self.k, self.v))
        self.lists = [dev(np.concatenate([np.asarray(x, np.int64).astype(np.int32), np.zeros(1, np.int32)])) for x in (parents, drafted, picked)]
        n = max(1, self.batch.tokens)
        self.path, self.counts, self.next = dev(np.full(n, 77, np.int32)), dev(np.full(len(self.batch.lengths) + 1, 77, np.int32)), dev(np.full(len(self.batch.lengths) + 1, 77, np.int32))
        return self

    def run(self, starts=True):
        b, size = self.batch, np.dtype(self.dtype).itemsize
        pools = [C.c_void_p(x.p.value + self.offset * size) for x in (self.dk, self.dv)]
        H.call("vkml_keep_drafts", C.byref(self.p), *[x.p for x in self.lists], b.d_table.p, b.d_lengths.p, b.d_starts.p if starts else None, self.path.p, self.counts.p, self.next.p,
               *pools)
        return self

    def place(self, s, pos):
        """The elements of a key's rows in a layer, [kv_heads, hd], or None."""
        if not 0 <= pos < self.batch.stride * self.page:
            return None
        page = self.batch.table[s, pos // self.page]
        if not 0 <= page < self.pages:
            return None
        return page * self.stride + (np.arange(self.kv_heads)[:, None] * self.page + pos % self.page) * self.hd + np.arange(self.hd)

    def check(self, parents, drafted, picked, what=""):
        b = self.batch
        n = len(b.lengths)
        path, counts, nxt = self.path.download(np.int32, (max(1, b.tokens),)), self.counts.download(np.int32, (n + 1,)), self.next.download(np.int32, (n + 1,))
        k, v = (x.download(self.dtype, (self.offset + self.layers * self.layer_stride,))[self.offset:].reshape(self.layers, -1) for x in (self.dk, self.dv))
        want_k, want_v = self.k.copy(), self.v.copy()
        free = np.zeros(self.layer_stride, bool)  # rows of drafts that are not kept
        for s in range(n):
            lo, hi = b.starts[s], b.starts[s + 1]
            own = walk(parents[lo:hi], drafted[lo:hi], picked[lo:hi])
            assert counts[s] == len(own), what
            assert path[lo:hi].tolist() == own + [-1] * (hi - lo - len(own)), what
            assert nxt[s] == (picked[lo + own[-1]] if own else -1), what
            base = b.lengths[s] - (hi - lo)
            for j, i in enumerate(own):
                a, c = self.place(s, base + i), self.place(s, base + j)
                if a is not None and c is not None:
                    want_k[:, c], want_v[:, c] = self.k[:, a], self.v[:, a]
            for j in range(len(own), hi - lo):
                c = self.place(s, base + j)
                if c is not None:
                    free[c] = True
        for got, want in ((k, want_k), (v, want_v)):
            got, want = got.view(np.uint16 if self.dtype == np.float16 else np.uint32), want.view(np.uint16 if self.dtype == np.float16 else np.uint32)
            assert np.array_equal(got[:, ~free], want[:, ~free]), what
        return counts[:n]


def drafts(rng, new, right=0.7, vocab=50):
    """Trees, their tokens, and picks that agree with a child's token often."""
    parents, drafted, picked = [], [], []
    for n in new:
        p = random_parents(rng, n) if n else []
        t = rng.integers(0, vocab, n).tolist()
        k = rng.integers(0, vocab, n).tolist()
        for i in range(1, n):
            if rng.random() < right:
                k[p[i]] = t[i]
        parents += p
        drafted += t
        picked += k
    return parents, drafted, picked


@pytest.mark.parametrize("kv", [H.F16, H.F32])
@pytest.mark.parametrize("hd,kv_heads", [(128, 8), (64, 2), (6, 3), (2, 1), (80, 5)])
@pytest.mark.parametrize("page", [16, 64])
def test_drafts_that_are_picked_stay(page, hd, kv_heads, kv):
    rng = np.random.default_rng(40)
    new = [1, 2, 5, 13, 64, 65, 0, 200]
    lengths = [n + k for n, k in zip(new, (0, 5, 11, 100, 15, 0, 9, 40))]
    x = drafts(rng, new, 0.9)
    print("keep", hd, kv_heads, page, kv, flush=True)
    call = Keep(rng, lengths, new, kv_heads, hd, page, kv, layers=3).upload(*x).run()
    assert call.check(*x).max() >= 5  # (of its inputs: some paths are long)


@pytest.mark.parametrize("kv", [H.F16, H.F32])
@pytest.mark.parametrize("n", [40, 300])
def test_a_path_whose_rows_move_by_one(n, kv):
    """Node 1 is wrong and all others right, in a chain: each row goes where
    the next one's was."""
    rng = np.random.default_rng(41)
    parents = [-1, 0, 0] + list(range(2, n - 1))
    drafted, picked = list(range(n)), [2] + [0] + list(range(3, n + 1))
    call = Keep(rng, [n + 21], [n], 8, 128, 16, kv).upload(parents, drafted, picked).run()
    assert call.check(parents, drafted, picked).tolist() == [n - 1]


def test_lists_of_any_values():
    """Parents that are no earlier node, equal tokens of siblings (the first
    is taken), nodes past the 4096th, and sequences without tokens."""
    rng = np.random.default_rng(42)
    new = [0, 30, 4100, 9, 1]
    parents, drafted, picked = drafts(rng, new, 1.0, 3)
    parents[0:30] = [5, 0, 0, 0, 3, 2 ** 31 - 1, -2 ** 31, 7, 6, -1] + [int(rng.integers(0, i)) for i in range(10, 30)]
    chain = 30
    parents[chain:chain + 4100] = [-1] + list(range(4099))
    drafted[chain:chain + 4100] = [9] * 4100
    picked[chain:chain + 4100] = [9] * 4100
    parents[4130:4139] = [2 ** 31 - 1] * 9
    call = Keep(rng, [7, 33, 4100, 20, 1], new, 1, 64, 16, H.F16, layers=1).upload(parents, drafted, picked).run()
    got = call.check(parents, drafted, picked)
    assert got.tolist()[2:] == [4096, 1, 1] and got[0] == 0


@pytest.mark.parametrize("base16", [True, False])
def test_gaps_and_pools_that_start_anywhere(base16):
    rng = np.random.default_rng(43)
    new = [9, 20]
    x = drafts(rng, new, 0.95)
    for kv in (H.F16, H.F32):
        for hd in (64, 10):
            pages = 3 + 2 + 4  # of [40, 29 + 20] keys, and spare ones
            stride = 2 * 16 * hd + 24
            call = Keep(rng, [40, 29], new, 2, hd, 16, kv, layers=3, stride=stride, layer_stride=pages * stride + 40, spare=4, base16=base16).upload(*x)
            call.run().check(*x)


def test_keys_in_no_page_stay():
    rng = np.random.default_rng(44)
    new = [40]
    n = 40
    parents, drafted, picked = [-1, 0, 0] + list(range(2, n - 1)), list(range(n)), [2, 0] + list(range(3, n + 1))
    call = Keep(rng, [60], new, 2, 64, 16, H.F16)
    call.batch.table[0, 2] = -1
    call.upload(parents, drafted, picked).run().check(parents, drafted, picked)
    call = Keep(rng, [30], new, 2, 64, 16, H.F16)  # fewer keys than new tokens
    call.upload(parents, drafted, picked).run()
    H.synchronize()


def test_one_token_a_sequence_without_starts():
    rng = np.random.default_rng(45)
    x = ([-1] * 5, [1] * 5, [4, 5, 6, 7, 8])
    call = Keep(rng, [1, 9, 20, 5, 3], [1] * 5, 2, 64, 16, H.F16).upload(*x).run(starts=False)
    assert call.check(*x).tolist() == [1] * 5


def test_a_captured_keep_follows_its_arrays():
    rng = np.random.default_rng(46)
    new = [9, 20, 33]
    x = drafts(rng, new, 0.9)
    call = Keep(rng, [40, 20, 100], new, 2, 64, 16, H.F16).upload(*x)
    H.call("vkml_graph_begin")
    call.run()
    g = C.c_uint64()
    H.call("vkml_graph_end", C.byref(g))
    for k in range(4):
        x = drafts(rng, new, 0.9)
        for buf, values in zip(call.lists, x):
            buf.upload(np.asarray(values, np.int32))
        call.dk.upload(call.k)
        call.dv.upload(call.v)
        H.call("vkml_graph_launch", g)
        call.check(*x, what=k)
    H.call("vkml_graph_destroy", g)


def test_keep_refuses():
    rng = np.random.default_rng(47)
    x = ([-1, 0], [1, 2], [2, 3])
    call = Keep(rng, [9], [2], 2, 64, 16, H.F16).upload(*x)
    b = call.batch

    def args(p=None, **change):
        named = dict(parents=call.lists[0], drafted=call.lists[1], picked=call.lists[2], table=b.d_table, lengths=b.d_lengths, starts=b.d_starts, path=call.path, counts=call.counts,
                     next=call.next, k=call.dk, v=call.dv)
        named.update(change)
        return (C.byref(p or call.p), *[ptr(y) for y in named.values()])

    for name in ("parents", "drafted", "picked", "table", "lengths", "path", "counts", "next", "k", "v"):
        assert "null buffer" in refused("vkml_keep_drafts", *args(**{name: None})), name
    assert "without starts" in refused("vkml_keep_drafts", *args(starts=None))
    assert "null params" in refused("vkml_keep_drafts", None, *[None] * 11)
    p = H.KeepDraftsParams.from_buffer_copy(call.p)
    p.layers = 0
    assert "layers" in refused("vkml_keep_drafts", *args(p))
    p.layers, p.seqs, p.tokens = 2, 0, 0
    assert H.lib().vkml_keep_drafts(*args(p, k=None)) == 0
