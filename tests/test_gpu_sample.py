"""vkml_sample against its definition in float64 (numpy), row by row, and against
vkml::Sampler on the host.

Tokens have to be equal. A pick differs from float64's only where a border, the
draw's, top_p's or min_p's, lies nearer to a sum of weights (for min_p to a weight)
than both computations' error: each weight is rounded to 2^-shift of the largest
(shift = min(51, 62 - ceil(log2(vocab)))) and found to 2^-50, so that n of them are
off by n 2^-(shift + 1) of the largest and 2^-50 of themselves at the most, and the
cumulated float64 sums of the reference by n 2^-53 of the total. pick_f64 says
whether the nearest border is further away than that; a row where it is not has no
one answer and is left out (a few in a million, which the test counts)."""
import ctypes as C
import math

import numpy as np
import pytest

from vkml_amd import hip as H
from vkml_amd import llama as L

pytestmark = pytest.mark.gpu
OPTIONS = np.dtype([("temperature", np.float32), ("top_k", np.int32), ("top_p", np.float32), ("min_p", np.float32)])
LOWEST = np.finfo(np.float32).min


@pytest.fixture(scope="module", autouse=True)
def device():
    H.init()
    yield
    H.synchronize()


def dev(a):
    return H.to_device(np.ascontiguousarray(a))


def pick_f64(row, temperature, top_k, top_p, min_p, u):
    """(token, whether no border is within the errors)."""
    with np.errstate(all="ignore"):
        ids = np.flatnonzero(row > -np.inf)  # (not NaN)
        if ids.size == 0:
            return -1, True
        if row.max(where=row > -np.inf, initial=-np.inf) == np.inf:
            ids = np.flatnonzero(row == np.inf)
        ranked = ids[np.lexsort((ids, -(row[ids] + 0.0).astype(np.float64)))]
        if not temperature > 0 or top_k == 1:
            return int(ranked[0]), True
        x = row[ranked].astype(np.float64)
        d = np.where(x == x[0], 0.0, x - x[0])
        w = np.exp(d / float(temperature)) if temperature < np.inf else np.ones(x.size)
        near = 1.0
        rounding, sums_off = row.size * 2.0 ** -(shift_of(row.size) + 1), 2.0 ** -50 + row.size * 2.0 ** -53
        if top_k > 0:
            w = w[:top_k]
        if top_p < 1:
            sums, target = np.cumsum(w), max(float(top_p), 0.0) * w.sum()
            m = min(int(np.searchsorted(sums, target, side="left")) + 1, w.size)
            near = min(near, np.abs(sums - target).min() / sums[-1] - rounding / sums[-1] - sums_off)
            w = w[:m]
        if min_p > 0:
            near = min(near, np.abs(w / float(min_p) - 1).min() - 2.0 ** -(shift_of(row.size) + 1) / float(min_p) - 2.0 ** -50)
            w = w[:max(1, int((w >= float(min_p) * w[0]).sum()))]
        sums = np.cumsum(w)
        at = min(max(u, 0.0), 1.0) * sums[-1]
        i = min(int(np.searchsorted(sums, at, side="right")), int((w > 0).sum()) - 1)
        near = min(near, np.abs(sums[w > 0][:-1] - at).min(initial=np.inf) / sums[-1] - rounding / sums[-1] - sums_off)
        return int(ranked[i]), near > 0


def shift_of(vocab):
    return min(51, 62 - math.ceil(math.log2(vocab)))


class Call:
    def __init__(self, logits, options, random, stride=0, offset=0):
        rows, vocab = logits.shape
        stride = stride or vocab
        flat = np.full(offset + rows * stride, np.inf, np.float32)  # gaps are never read as logits
        for i in range(rows):
            flat[offset + i * stride:offset + i * stride + vocab] = logits[i]
        self.rows, self.p = rows, H.SampleParams(rows=rows, vocab=vocab, row_stride=stride)
        self.logits, self.at = dev(flat), 4 * offset
        self.options, self.random = dev(options), dev(np.asarray(random, np.float64))
        self.workspace = dev(np.full(max(16, H.lib().vkml_sample_workspace_bytes(C.byref(self.p))) // 4, -1, np.int32))  # of any content
        self.tokens = dev(np.full(rows, 77, np.int32))

    def run(self):
        H.call("vkml_sample", C.byref(self.p), C.c_void_p(self.logits.p.value + self.at), self.options.p, self.random.p, self.workspace.p, self.tokens.p)
        return self

    def result(self):
        return self.tokens.download(np.int32, (self.rows,))


def check(logits, options, random, exact_borders=False, **where):
    options = np.array(options, OPTIONS)
    print("sample", logits.shape, where, flush=True)
    call = Call(logits, options, random, **where).run()
    got = call.result()
    left_out = 0
    for i, (row, o, u) in enumerate(zip(logits, options, random)):
        want, sure = pick_f64(row, *o, u)
        left_out += not (sure or exact_borders)
        assert got[i] == want or not (sure or exact_borders), (i, o, u, got[i], want)
    assert left_out <= 1
    assert np.array_equal(call.run().result(), got)
    return got


ASKED = [(0.7, 40, 0.9, 0.0), (1.0, 0, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (0.8, 0, 0.95, 0.0), (1.2, 0, 1.0, 0.05), (0.6, 50, 0.8, 0.02), (1.0, 1, 1.0, 0.0), (1.5, 5, 1.0, 0.0),
         (2.0, 0, 0.5, 0.3), (1.0, 10 ** 9, 0.999, 1e-4), (0.05, 0, 1.0, 0.0), (5.0, 0, 0.97, 0.0)]


def like_a_model(rng, rows, vocab, spread=1.7):
    x = (spread * rng.standard_normal((rows, vocab))).astype(np.float32)
    n = min(vocab, 64)
    for r in x:
        r[rng.integers(0, vocab, n)] += (12 * rng.random(n) ** 2).astype(np.float32)
    return x


def asked(rng, rows):
    return [ASKED[i % len(ASKED)] for i in range(rows)], rng.random(rows)


@pytest.mark.parametrize("vocab", [1, 2, 3, 4, 5, 63, 64, 65, 1000, 1023, 4096, 4099, 32764, 32765, 32766, 32768, 65531, 128256, 300001])
def test_rows_of_any_size(vocab):
    rng = np.random.default_rng(vocab)
    rows = 24 if vocab < 100000 else 12
    check(like_a_model(rng, rows, vocab), *asked(rng, rows))


@pytest.mark.parametrize("rows", [255, 256, 257, 300, 511, 1023, 1024, 1025])
def test_many_rows(rows):
    """Of every kind of request, in an order that changes (rows that take long come
    first); the same row gives the same token wherever it stands."""
    rng = np.random.default_rng(rows)
    x, (o, u) = like_a_model(rng, rows, 8200), asked(rng, rows)
    order = rng.permutation(rows)
    o = [o[i] for i in order]
    got = check(x, o, u)
    back = np.argsort(order)
    assert np.array_equal(Call(x[back], np.array(o, OPTIONS)[back], u[back]).run().result(), got[back])
    # one kind alone
    assert np.array_equal(Call(x, np.array([ASKED[1]] * rows, OPTIONS), u).run().result(), Call(x[::-1], np.array([ASKED[1]] * rows, OPTIONS), u[::-1]).run().result()[::-1])


@pytest.mark.parametrize("vocab", [7, 1000, 32763, 32765, 40000])
@pytest.mark.parametrize("offset,gap", [(0, 1), (1, 0), (2, 3), (3, 2), (3, 4)])
def test_rows_that_start_anywhere(offset, gap, vocab):
    rng = np.random.default_rng(2)
    check(like_a_model(rng, 13, vocab), *asked(rng, 13), stride=vocab + gap, offset=offset)


@pytest.mark.parametrize("vocab", [192, 6000, 32768, 40000, 128256, 200000])
def test_many_are_kept(vocab):
    """By top_k on both sides of what is listed first, and by a min_p that leaves more
    than a list holds."""
    rng = np.random.default_rng(vocab + 1)
    ks = [128, 191, 192, 193, 256, 257, 341, 512, 513, 768, 769, 1000, 1024, 1025, 5000]
    o = [(1.0, k, p, 0.0) for k in ks for p in (0.9, 1.0)] + [(1.0, k, 1.0, m) for k in (0, 300, 2000) for m in (1e-5, 1e-3, 0.02)]
    check(like_a_model(rng, len(o), vocab), o, rng.random(len(o)))


@pytest.mark.parametrize("vocab", [1000, 32768, 128256])
@pytest.mark.parametrize("step", [1 / 32, 1.0, 4.0])
def test_equal_logits(step, vocab):
    """Of a few values, so that hundreds or thousands are alike: the lowest ids first."""
    rng = np.random.default_rng(3)
    x = (np.round(like_a_model(rng, 24, vocab) / step) * step).astype(np.float32)
    check(x, *asked(rng, 24))


@pytest.mark.parametrize("vocab", [5, 128, 2049, 32768, 131072])
def test_all_logits_alike(vocab):
    """Every weight is 1: token floor(u m) of the m that are kept."""
    n = 9
    u = (np.arange(n) + 0.5) / n
    for value in (0.0, -3.25, LOWEST, np.inf, -0.0):
        x = np.full((n, vocab), value, np.float32)
        x[::2] *= np.float32(1.0) if value else np.float32(-1.0)  # zeros of both signs are alike
        got = check(x, [(1.0, 0, 1.0, 0.0)] * n, u, exact_borders=True)
        assert got.tolist() == [int(y * vocab) for y in u]
        k = max(2, vocab // 3)
        got = check(x, [(0.5, k, 1.0, 0.5)] * n, u, exact_borders=True)
        assert got.tolist() == [int(y * k) for y in u]
        got = check(x, [(0.5, 0, 0.5, 1.0)] * n, u, exact_borders=True)
        assert got.tolist() == [int(y * ((vocab + 1) // 2)) for y in u]


@pytest.mark.parametrize("vocab", [50, 32768, 40000])
def test_masked_and_bad_logits(vocab):
    rng = np.random.default_rng(4)
    x = like_a_model(rng, 30, vocab)
    for i, bad in enumerate((-np.inf, LOWEST, np.nan, np.inf, -np.inf)):
        r = x[i::5]
        r[rng.random(r.shape) < (0.002 if bad == np.inf else 0.5)] = bad
        x[i::5] = r
    x[7, :] = -np.inf
    x[8, :] = np.nan
    x[9, :] = np.nan
    x[9, vocab // 2] = -np.inf
    x[10, :] = -np.inf
    x[10, vocab - 1] = -50.0
    x[11, :] = np.nan
    x[11, 3] = LOWEST
    got = check(x, *asked(rng, 30))
    assert got[7:12].tolist() == [-1, -1, -1, vocab - 1, 3]


@pytest.mark.parametrize("vocab", [1000, 32768, 50000])
def test_options_at_their_ends(vocab):
    rng = np.random.default_rng(5)
    nan = float("nan")
    o = [(1.0, 0, 0.0, 0.0), (1.0, 0, -1.0, 0.0), (1.0, 0, 1e-30, 0.0), (1.0, 0, nan, nan), (1.0, -5, 2.0, -1.0), (nan, 0, 1.0, 0.0), (-1.0, 0, 1.0, 0.0), (1e-30, 0, 1.0, 0.0),
         (1e-45, 0, 1.0, 0.0), (1.0, 2 ** 31 - 1, 1.0, 0.0), (1.0, -2 ** 31, 1.0, 0.0), (1.0, 0, 1.0, 1.0), (1.0, 0, 1.0, 7.0), (100.0, 0, 1.0, 0.0), (1.0, 2, 1.0, 0.0),
         (1.0, vocab - 1, 1.0, 0.0), (1.0, vocab, 1.0, 0.0), (1.0, 0, 0.9999999, 0.0), (1e4, 3000, 1.0, 0.0)]
    x = like_a_model(rng, len(o), vocab)
    check(x, o, rng.random(len(o)))
    x[:, 5] = x.max(1) + 1e-3  # two near the top
    check(x, o, rng.random(len(o)))


def test_infinitely_hot():
    rng = np.random.default_rng(6)
    x = like_a_model(rng, 5, 1000)
    x[1, 500:] = -np.inf
    u = np.array([0.1, 0.5, 0.999, 0.0, 0.3])
    got = check(x, [(float("inf"), 0, 1.0, 0.0)] * 5, u, exact_borders=True)
    assert x[1, got[1]] > -np.inf


def test_draws_at_their_ends():
    rng = np.random.default_rng(7)
    for vocab in (1000, 40000):
        x = like_a_model(rng, 8, vocab)
        u = [0.0, -3.0, float("nan"), -np.inf, 1.0 - 2.0 ** -53, 1.0, 5.0, np.inf]
        o = [(1.0, 7, 1.0, 0.0)] * 8
        got = Call(x, np.array(o, OPTIONS), u).run().result()
        for i, row in enumerate(x):
            ranked = np.argsort(-row, kind="stable")
            assert got[i] == ranked[0 if i < 4 else 6]


def test_draws_follow_the_weights():
    """Every token of a small row at the middle of its share, and at its ends."""
    row = np.array([0.0, math.log(3.0), -1.0, 2.0, 2.0, -20.0, 0.5], np.float32)  # the least has a share of 10^-10
    w = np.exp(row.astype(np.float64))
    ranked = np.argsort(-row, kind="stable")
    ends = np.cumsum(w[ranked]) / w.sum()
    starts = np.concatenate([[0.0], ends[:-1]])
    eps = 1e-13
    u = np.concatenate([(starts + ends) / 2, starts + eps, ends - eps])
    got = Call(np.tile(row, (21, 1)), np.array([(1.0, 0, 1.0, 0.0)] * 21, OPTIONS), u).run().result()
    assert got.tolist() == ranked.tolist() * 3


def test_twenty_thousand_small_rows():
    rng = np.random.default_rng(8)
    rows = 20000
    x = rng.standard_normal((rows, 6)).astype(np.float32)
    o = np.array([ASKED[i % len(ASKED)] for i in range(rows)], OPTIONS)
    u = rng.random(rows)
    got = Call(x, o, u).run().result()
    some = rng.integers(0, rows, 2000)
    for i in some:
        want, sure = pick_f64(x[i], *o[i], u[i])
        assert got[i] == want or not sure


def test_the_largest_row():
    rng = np.random.default_rng(9)
    check(like_a_model(rng, 4, 2 ** 22), ASKED[:2] + ASKED[3:5], rng.random(4))


def test_rows_past_32_bit_offsets():
    """Rows 2^30 floats apart."""
    rng = np.random.default_rng(10)
    stride, vocab = 1 << 30, 1000
    x = like_a_model(rng, 4, vocab)
    o, u = asked(rng, 4)
    call = Call(x, np.array(o, OPTIONS), u)
    buf = H.empty(4 * (3 * stride + vocab))
    for i in range(4):
        H.call("vkml_memcpy_h2d", C.c_void_p(buf.p.value + 4 * i * stride), np.ascontiguousarray(x[i]).ctypes.data_as(C.c_void_p), 4 * vocab)
    call.logits, call.p.row_stride = buf, stride
    assert call.run().result().tolist() == [pick_f64(x[i], *np.array(o, OPTIONS)[i], u[i])[0] for i in range(4)]


@pytest.mark.parametrize("vocab", [1000, 40000])
def test_the_host_s_sampler_picks_the_same(vocab):
    """vkml::Sampler's draw is its generator's uniform number times the kept weight."""
    import oracle as O
    rng = np.random.default_rng(11)
    for k, (t, top_k, top_p, min_p) in enumerate(ASKED):
        x = like_a_model(rng, 20, vocab)
        host, raw = L.Sampler(temperature=t, top_k=min(top_k, 2 ** 31 - 1), top_p=top_p, min_p=min_p, seed=k), O.Sampler(seed=k)
        want = [host.sample(row) for row in x]
        u = [raw.draw_uniform(1.0) for _ in x]
        got = Call(x, np.array([(t, top_k, top_p, min_p)] * 20, OPTIONS), u).run().result()
        assert got.tolist() == want, (k, vocab)


def test_captured_calls_follow_their_arrays():
    rng = np.random.default_rng(12)
    graphs, calls = [], []
    for vocab in (1000, 40000):
        call = Call(like_a_model(rng, 12, vocab), np.array(asked(rng, 12)[0], OPTIONS), rng.random(12))
        H.call("vkml_graph_begin")
        call.run()
        g = C.c_uint64()
        H.call("vkml_graph_end", C.byref(g))
        graphs.append(g)
        calls.append(call)
    for _ in range(4):
        for call, g in zip(calls, graphs):
            x, u, o = like_a_model(rng, 12, call.p.vocab), rng.random(12), np.array(rng.permutation(np.array(asked(rng, 12)[0], OPTIONS)), OPTIONS)
            call.logits.upload(x)
            call.random.upload(u)
            call.options.upload(o)
            H.call("vkml_graph_launch", g)
            got = call.result()
            assert got.tolist() == [pick_f64(row, *oo, uu)[0] for row, oo, uu in zip(x, o, u)]
            assert np.array_equal(call.run().result(), got)
    for g in graphs:
        H.call("vkml_graph_destroy", g)


def test_sample_refuses():
    def refused(*args):
        assert H.lib().vkml_sample(*args) == 1
        return H.lib().vkml_last_error().decode()

    call = Call(np.zeros((2, 40000), np.float32), np.array([(1.0, 0, 1.0, 0.0)] * 2, OPTIONS), [0.5, 0.5])
    fine = [C.byref(call.p), call.logits.p, call.options.p, call.random.p, call.workspace.p, call.tokens.p]
    for i in range(1, 6):
        assert "null buffer" in refused(*fine[:i], None, *fine[i + 1:])
    assert "null params" in refused(None, *fine[1:])
    assert "aligned" in refused(*fine[:2], C.c_void_p(call.options.p.value + 4), *fine[3:])
    assert "aligned" in refused(*fine[:3], C.c_void_p(call.random.p.value + 4), *fine[4:])
    assert "aligned" in refused(*fine[:4], C.c_void_p(call.workspace.p.value + 8), *fine[5:])
    p = H.SampleParams(rows=2, vocab=1000, row_stride=999)
    assert "overlap" in refused(C.byref(p), *fine[1:])
    p = H.SampleParams(rows=0, vocab=1000, row_stride=1000)
    assert H.lib().vkml_sample(C.byref(p), None, None, None, None, None) == 0
    p = H.SampleParams(rows=1, vocab=1000, row_stride=1000)
    assert H.lib().vkml_sample(C.byref(p), call.logits.p, call.options.p, call.random.p, None, call.tokens.p) == 0  # no workspace needed
    H.synchronize()
