"""Several sequences over one paged KV cache (vkml_rope_kv_pages,
vkml_attend_pages, vkml_copy_pages) against plain implementations in float64.

Attention's bound, element by element. A score x_j = scale sum_d q_d k_jd is
off by at most delta_j = scale (2^-22 max|q| sum_d |k_jd| + (hd + 8) 2^-24
sum_d |q_d k_jd|): q in two f16 terms (relative to the row's largest value),
the products exact, the sum in f32. In log2 units its rounding adds
2^-23 |x_j|. The weights e^(x_j - M) carry twice the largest such error as a
relative one, 2^-20 more for the exponential and their own two terms; the
sums of n weighted values go through at most n / 16 + 64 f32 additions each
(blocks of 16 keys or more in the matrix unit, then the blocks, then the
parts of a split). With P_d = sum_j p_j |v_jd| of the float64 softmax:

    |out_d - exact_d| <= P_d (2 max_j delta_j + 2^-22 max|x| + (n / 16 + 64) 2^-24 + 2^-20)

A soft cap turns a score's error by at most one; its own f32 tanh adds 2^-20
cap. Rotations: two products and a sum, each rounded: 2^-23 (|a| + |b|), then
the cache type's half step.
"""
import ctypes as C
import math

import numpy as np
import pytest

from vkml_amd import hip as H

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    H.init()
    yield
    H.synchronize()


def dev(a):
    return H.to_device(a)


def ptr(b):
    return b.p if b is not None else None


class Cache:
    """Host pools [pages, kv_heads, page, hd] with their device copies, pages
    `stride` elements apart."""

    def __init__(self, rng, pages, kv_heads, page, hd, kv, stride=0, fill=None):
        self.pages, self.kv_heads, self.page, self.hd, self.kv = pages, kv_heads, page, hd, kv
        self.dtype = np.float16 if kv == H.F16 else np.float32
        self.stride = stride or kv_heads * page * hd
        shape = (pages, kv_heads, page, hd)
        gain = 0.5 + 1.5 * rng.random(hd)
        self.k = (rng.standard_normal(shape) * gain).astype(self.dtype) if fill is None else np.full(shape, fill, self.dtype)
        self.v = rng.standard_normal(shape).astype(self.dtype) if fill is None else np.full(shape, fill, self.dtype)

    def upload(self):
        out = []
        for x in (self.k, self.v):
            whole = np.full((self.pages, self.stride), np.nan, self.dtype)  # gaps between pages are never read as keys
            whole[:, :x[0].size] = x.reshape(self.pages, -1)
            out.append(dev(whole))
        self.dk, self.dv = out
        return self

    def download(self):
        n = self.kv_heads * self.page * self.hd
        return [b.download(self.dtype, (self.pages, self.stride))[:, :n].reshape(self.k.shape) for b in (self.dk, self.dv)]


class Batch:
    """Sequences of shared + own keys, `new` of them new, with a page table."""

    def __init__(self, rng, lengths, new, page, groups=(), spare=2, stride=0, pages=None):
        # groups: (first sequence, last + 1, shared keys)
        self.lengths, self.new, self.page, self.groups = list(lengths), list(new), page, list(groups)
        self.starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.tokens = int(self.starts[-1])
        need = [-(-n // page) for n in lengths]
        self.stride = stride or max(need + [1])
        self.table = np.full((len(lengths), self.stride), -1, np.int32)
        shared = {}
        for a, b, keys in groups:
            for s in range(a, b):
                shared[s] = (a, keys // page)
        count = 0
        for s, n in enumerate(need):
            first, full = shared.get(s, (s, 0))
            full = 0 if first == s else full
            self.table[s, :full] = self.table[first, :full]
            self.table[s, full:n] = np.arange(count, count + n - full)
            count += n - full
        self.pages = pages or count + spare
        order = rng.permutation(self.pages).astype(np.int32)
        self.table = np.where(self.table >= 0, order[np.maximum(self.table, 0)], -1).astype(np.int32)

    def share(self, cache):
        """The part-filled shared page is each sequence's own copy."""
        for a, b, keys in self.groups:
            part = keys % self.page
            for s in range(a + 1, b):
                if part:
                    for pool in (cache.k, cache.v):
                        pool[self.table[s, keys // self.page], :, :part] = pool[self.table[a, keys // self.page], :, :part]

    def upload(self):
        self.d_table, self.d_lengths, self.d_starts = dev(self.table), dev(np.asarray(self.lengths, np.int32)), dev(self.starts)
        gs = [a for a, _, _ in self.groups] + ([self.groups[-1][1]] if self.groups else [0])
        self.d_group_starts = dev(np.asarray(gs, np.int32))
        self.d_group_keys = dev(np.asarray([k for _, _, k in self.groups] or [0], np.int32))
        return self


def rows_of(cache, pool, table_row, n):
    """Keys 0 .. n - 1 of a sequence, [n, kv_heads, hd], and whether a page holds each."""
    pos = np.arange(n)
    page = table_row[pos // cache.page]
    held = (page >= 0) & (page < cache.pages)
    return pool[np.where(held, page, 0), :, pos % cache.page], held


def attention_f64(q, cache, batch, scale, softcap=0.0, k=None, v=None):
    """(out, bound) of every token, [tokens, heads, hd]."""
    k, v = cache.k if k is None else k, cache.v if v is None else v
    heads, hd = q.shape[1:]
    G = heads // cache.kv_heads
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for s, (length, n) in enumerate(zip(batch.lengths, batch.new)):
        kk, held = rows_of(cache, k, batch.table[s], length)
        vv, _ = rows_of(cache, v, batch.table[s], length)
        for i in range(n):
            t, seen = batch.starts[s] + i, max(0, length - n + i + 1)
            on = np.flatnonzero(held[:seen])
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


def params(cache, batch, heads, scale, softcap=0.0):
    return H.AttendPagesParams(heads=heads, kv_heads=cache.kv_heads, head_dim=cache.hd, kv_type=cache.kv, page_size=cache.page, pages=cache.pages,
                               seqs=len(batch.lengths), tokens=batch.tokens, table_stride=batch.stride, groups=len(batch.groups),
                               page_stride=cache.stride, scale=scale, softcap=softcap)


class Call:
    """One vkml_attend_pages call and its buffers."""

    def __init__(self, q, cache, batch, scale, softcap=0.0, starts=True, workspace=None):
        self.p = params(cache, batch, q.shape[1], scale, softcap)
        self.cache, self.batch, self.shape = cache, batch, q.shape
        self.q, self.out = dev(q), dev(np.full(q.shape, 7.5, np.float32))
        self.starts = batch.d_starts if starts else None
        need = H.lib().vkml_attend_pages_workspace_bytes(C.byref(self.p))
        # of any content: NaN bits here
        self.workspace = workspace or dev(np.full(max(need, 16) // 4 + 4, -1, np.int32))

    def run(self):
        b = self.batch
        H.call("vkml_attend_pages", C.byref(self.p), self.q.p, self.cache.dk.p, self.cache.dv.p, b.d_table.p, b.d_lengths.p, ptr(self.starts),
               b.d_group_starts.p if b.groups else None, b.d_group_keys.p if b.groups else None, self.workspace.p, self.out.p)
        return self

    def result(self):
        return self.out.download(np.float32, self.shape)


def close(got, want, bound, what="", loose=1.0):
    err = np.abs(got.astype(np.float64) - want)
    worst = np.unravel_index(np.argmax(err - bound), err.shape)
    assert np.all(err <= bound), f"{what}: |err| {err[worst]:.3g} above {bound[worst]:.3g} at {worst}"
    # and in the 2-norm, where roundings average out, far below the worst case
    # (scores `loose` times as large carry errors as many times as large)
    norm = np.linalg.norm(want)
    assert np.linalg.norm(err) <= 1e-5 * loose * norm, f"{what}: relative error {np.linalg.norm(err) / norm:.3g}"


def attend(seed, heads, kv_heads, hd, page, kv, lengths, new, groups=(), softcap=0.0, stride=0, table_stride=0, starts=True, q_scale=1.0):
    rng = np.random.default_rng(seed)
    batch = Batch(rng, lengths, new, page, groups, stride=table_stride)
    cache = Cache(rng, batch.pages, kv_heads, page, hd, kv, stride)
    batch.share(cache)
    q = (rng.standard_normal((batch.tokens, heads, hd)) * q_scale).astype(np.float32)
    scale = 1.0 / math.sqrt(hd)
    cache.upload()
    batch.upload()
    print("attend", seed, heads, kv_heads, hd, page, kv, list(lengths)[:8], list(new)[:8], groups, softcap, flush=True)
    got = Call(q, cache, batch, scale, softcap, starts).run().result()
    want, bound = attention_f64(q, cache, batch, scale, softcap)
    close(got, want, bound, loose=max(1.0, q_scale))


HEADS = [(4, 2), (32, 8), (8, 8), (6, 2), (5, 1), (16, 1), (48, 2), (128, 1)]


@pytest.mark.parametrize("kv", [H.F16, H.F32])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", HEADS)
def test_decode_over_ragged_lengths(heads, kv_heads, hd, kv):
    attend(1, heads, kv_heads, hd, 16, kv, [1, 2, 15, 16, 17, 31, 33, 64, 65, 127, 129, 300], [1] * 12, starts=False)


@pytest.mark.parametrize("kv", [H.F16, H.F32])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 1024])
def test_page_sizes(page, kv):
    attend(2, 8, 2, 128, page, kv, [1, page - 1, page, page + 1, 3 * page + 5, 700], [1] * 6, starts=False)
    attend(3, 8, 2, 64, page, kv, [40, page + 7, 2 * page + 100], [40, 5, 33])


@pytest.mark.parametrize("kv", [H.F16, H.F32])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("shared", [1, 15, 16, 100, 128, 1000])
def test_shared_prefix(shared, hd, kv):
    lengths = [shared + n for n in (1, 2, 17, 64, 130, 5, 33, 16, 1)]
    attend(4, 8, 2, hd, 16, kv, lengths, [1] * 9, [(0, 9, shared)], starts=False)
    # two groups, and sequences in none
    attend(5, 8, 2, hd, 32, kv, [50] + lengths + [77], [1] * 11, [(1, 4, shared), (4, 10, shared // 2)], starts=False)


def test_many_sequences_share_a_long_prefix():
    rng = np.random.default_rng(6)
    own = rng.integers(1, 90, 40)
    attend(6, 32, 8, 128, 64, H.F16, [3000 + int(n) for n in own], [1] * 40, [(0, 40, 3000)])
    attend(7, 16, 2, 128, 16, H.F32, [900 + int(n) for n in own], [1] * 40, [(0, 40, 900)])


@pytest.mark.parametrize("kv", [H.F16, H.F32])
@pytest.mark.parametrize("heads,kv_heads", [(4, 2), (32, 8), (6, 2), (5, 1), (4, 4), (128, 1)])
def test_ragged_new_tokens_are_causal(heads, kv_heads, kv):
    attend(8, heads, kv_heads, 128, 16, kv, [3, 70, 1, 130, 200, 45], [3, 33, 1, 130, 2, 45])
    attend(9, heads, kv_heads, 64, 32, kv, [120, 103, 150, 100, 164], [20, 1, 50, 0, 64], [(0, 5, 100)])


def test_long_prompts():
    attend(10, 8, 2, 128, 64, H.F16, [700, 513], [700, 300])
    attend(11, 8, 2, 64, 128, H.F32, [300, 400], [300, 129])


def test_a_group_of_one_and_an_empty_prefix_share_nothing():
    attend(12, 8, 2, 128, 16, H.F16, [90, 50, 60], [1, 1, 1], [(0, 1, 40), (1, 3, 0)])


@pytest.mark.parametrize("kv", [H.F16, H.F32])
def test_softcap(kv):
    attend(13, 8, 2, 128, 16, kv, [5, 200, 333], [1, 70, 2], softcap=30.0, q_scale=6.0)


@pytest.mark.parametrize("q_scale", [1e-20, 1e-4, 30.0])
def test_queries_of_any_size(q_scale):
    attend(14, 8, 2, 128, 16, H.F16, [5, 200, 333], [1, 20, 2], q_scale=q_scale)


def test_gaps_between_pages_and_in_the_table():
    attend(15, 8, 2, 128, 16, H.F16, [5, 200, 333], [1, 20, 2], stride=2 * 16 * 128 + 8, table_stride=40)


def test_one_long_sequence():
    attend(16, 8, 2, 64, 16, H.F16, [70001], [1])
    attend(17, 4, 1, 128, 64, H.F32, [20011], [3])


def test_pools_past_32_bit_offsets():
    """Pages 2^28 elements apart: byte offsets past 4 GiB, element offsets past 2^32."""
    rng = np.random.default_rng(18)
    batch = Batch(rng, [300, 250], [1, 2], 16, pages=40)
    cache = Cache(rng, 40, 2, 16, 64, H.F16)
    cache.stride = 1 << 28
    cache.dk, cache.dv = H.empty(40 * cache.stride * 2), H.empty(40 * cache.stride * 2)
    for buf, x in ((cache.dk, cache.k), (cache.dv, cache.v)):
        for i in range(40):
            page = np.ascontiguousarray(x[i])
            H.call("vkml_memcpy_h2d", C.c_void_p(buf.p.value + i * cache.stride * 2), page.ctypes.data_as(C.c_void_p), page.nbytes)
    batch.upload()
    q = rng.standard_normal((3, 8, 64)).astype(np.float32)
    got = Call(q, cache, batch, 0.125).run().result()
    close(got, *attention_f64(q, cache, batch, 0.125))


@pytest.mark.parametrize("kv", [H.F16, H.F32])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_rows_that_hold_no_key_are_not_read(kv, bad):
    """Rows past a sequence's length, rows of a forked page below the shared
    keys' end and pages of no sequence hold NaN or infinities."""
    rng = np.random.default_rng(19)
    shared = 37
    batch = Batch(rng, [shared + 10, shared + 70, shared + 1, 20, 1], [1, 9, 1, 20, 1], 16, [(0, 3, shared)], spare=5)
    cache = Cache(rng, batch.pages, 2, 16, 128, kv)
    batch.share(cache)
    live = np.zeros((batch.pages, 16), bool)
    for s, n in enumerate(batch.lengths):
        pos = np.arange(n)
        live[batch.table[s, pos // 16], pos % 16] = True
    q = rng.standard_normal((batch.tokens, 8, 128)).astype(np.float32)
    want = attention_f64(q, cache, batch, 0.1)
    for s in (1, 2):  # their copies of the shared part of the page: read through the first sequence only
        live[batch.table[s, 2], :shared % 16] = False
    for pool in (cache.k, cache.v):
        pool.transpose(0, 2, 1, 3)[~live] = bad
    cache.upload()
    batch.upload()
    close(Call(q, cache, batch, 0.1).run().result(), *want)


@pytest.mark.parametrize("kv", [H.F16, H.F32])
@pytest.mark.parametrize("heads,kv_heads,hd", [(8, 2, 128), (4, 2, 64), (40, 2, 128)])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_a_later_token_that_is_not_finite_leaves_earlier_ones_alone(bad, heads, kv_heads, hd, kv):
    rng = np.random.default_rng(20)
    batch = Batch(rng, [50, 100, 33], [3, 60, 33], 16)
    cache = Cache(rng, batch.pages, kv_heads, 16, hd, kv)
    q = rng.standard_normal((batch.tokens, heads, hd)).astype(np.float32)
    want, bound = attention_f64(q, cache, batch, 0.1)
    hit = {0: 48, 1: 70, 2: 1}  # the key of each sequence that is spoilt: tokens at or past it see it
    for s, pos in hit.items():
        cache.v[batch.table[s, pos // 16], :, pos % 16, 5] = bad
    cache.upload()
    batch.upload()
    got = Call(q, cache, batch, 0.1).run().result()
    for s, pos in hit.items():
        for i in range(batch.new[s]):
            t = batch.starts[s] + i
            if batch.lengths[s] - batch.new[s] + i < pos:
                close(got[t], want[t], bound[t], f"sequence {s} token {i}")
            else:
                rest = np.arange(hd) != 5
                assert not np.isfinite(got[t][:, 5]).any()
                close(got[t][:, rest], want[t][:, rest], bound[t][:, rest], f"sequence {s} token {i}")
    for s, pos in hit.items():  # a key that is not finite: masked scores are left out, not added to
        cache.v[batch.table[s, pos // 16], :, pos % 16, 5] = 0
        cache.k[batch.table[s, pos // 16], :, pos % 16, 5] = np.nan
    want, bound = attention_f64(q, cache, batch, 0.1)
    cache.upload()
    got = Call(q, cache, batch, 0.1).run().result()
    for s, pos in hit.items():
        for i in range(batch.new[s]):
            t = batch.starts[s] + i
            if batch.lengths[s] - batch.new[s] + i < pos:
                close(got[t], want[t], bound[t], f"sequence {s} token {i}, K")
            else:
                assert np.isnan(got[t]).all()


@pytest.mark.parametrize("kv", [H.F16, H.F32])
def test_entries_that_are_no_page_hold_no_keys(kv):
    rng = np.random.default_rng(21)
    batch = Batch(rng, [200, 200, 40, 16], [1, 30, 1, 1], 16)
    cache = Cache(rng, batch.pages, 2, 16, 128, kv)
    batch.table[0, 3] = -1
    batch.table[0, 12] = batch.pages
    batch.table[1, :5] = 2 ** 31 - 1
    batch.table[3, 0] = -2 ** 31
    cache.upload()
    batch.upload()
    q = rng.standard_normal((batch.tokens, 8, 128)).astype(np.float32)
    got = Call(q, cache, batch, 0.1).run().result()
    want, bound = attention_f64(q, cache, batch, 0.1)
    close(got, want, bound)
    assert not got[batch.starts[3]].any()  # no key left: zeros


def test_tokens_without_keys_and_rows_of_no_sequence():
    rng = np.random.default_rng(22)
    batch = Batch(rng, [0, 20, 0, 2, 33], [1, 0, 2, 4, 2], 16)
    batch.starts += 3  # rows before the first sequence and past the last
    batch.tokens += 8
    cache = Cache(rng, batch.pages, 2, 16, 64, H.F16)
    cache.upload()
    batch.upload()
    q = rng.standard_normal((batch.tokens, 4, 64)).astype(np.float32)
    got = Call(q, cache, batch, 0.125).run().result()
    want, bound = attention_f64(q, cache, batch, 0.125)
    first, last = batch.starts[0], batch.starts[-1]
    close(got[first:last], want[first:last], bound[first:last])
    # lengths 0, 0, 0 and 2 of four new tokens: five rows without a key
    assert np.array_equal(np.flatnonzero(~got.any((1, 2))), [3, 4, 5, 6, 7])
    assert np.all(got[:first] == 7.5) and np.all(got[last:] == 7.5)


def test_nothing_to_do():
    rng = np.random.default_rng(23)
    batch = Batch(rng, [5], [1], 16)
    cache = Cache(rng, batch.pages, 2, 16, 64, H.F16)
    cache.upload()
    batch.upload()
    q = rng.standard_normal((1, 4, 64)).astype(np.float32)
    for change in ({"seqs": 0, "tokens": 0}, {"tokens": 0}):
        c = Call(q, cache, batch, 0.125)
        for name, value in change.items():
            setattr(c.p, name, value)
        assert np.all(c.run().result() == 7.5)


def test_the_same_call_twice_gives_the_same_bits():
    rng = np.random.default_rng(24)
    batch = Batch(rng, [500 + 13 * i for i in range(20)], [1] * 19 + [40], 16, [(0, 20, 300)])
    cache = Cache(rng, batch.pages, 8, 16, 128, H.F16)
    batch.share(cache)
    cache.upload()
    batch.upload()
    q = rng.standard_normal((batch.tokens, 32, 128)).astype(np.float32)
    first = Call(q, cache, batch, 0.1).run().result()
    for _ in range(3):
        assert np.array_equal(Call(q, cache, batch, 0.1).run().result().view(np.uint32), first.view(np.uint32))


def test_calls_of_other_shapes_share_a_workspace():
    rng = np.random.default_rng(25)
    calls = []
    for lengths, new, groups in (([900 + i for i in range(12)], [1] * 12, [(0, 12, 800)]), ([40, 300], [40, 7], []), ([5], [1], [])):
        batch = Batch(rng, lengths, new, 16, groups)
        cache = Cache(rng, batch.pages, 2, 16, 128, H.F16)
        batch.share(cache)
        cache.upload()
        batch.upload()
        q = rng.standard_normal((batch.tokens, 8, 128)).astype(np.float32)
        calls.append((q, cache, batch))
    most = max(H.lib().vkml_attend_pages_workspace_bytes(C.byref(params(c, b, 8, 0.1))) for _, c, b in calls)
    workspace = H.empty(max(most, 16))
    for _ in range(2):
        runs = [Call(q, c, b, 0.1, workspace=workspace).run() for q, c, b in calls]
        for run, (q, c, b) in zip(runs, calls):
            close(run.result(), *attention_f64(q, c, b, 0.1))


def test_a_captured_call_follows_the_lengths():
    rng = np.random.default_rng(26)
    batch = Batch(rng, [100, 333, 57], [1, 1, 1], 16, [(0, 3, 40)], stride=40)
    batch.table[:] = rng.integers(0, batch.pages, batch.table.shape)
    batch.table[1:, :2] = batch.table[0, :2]
    cache = Cache(rng, batch.pages, 2, 16, 128, H.F16)
    # the shared part of page 2 of each
    for s in (1, 2):
        batch.table[s, 2] = batch.table[0, 2]
    cache.upload()
    batch.upload()
    q = rng.standard_normal((3, 8, 128)).astype(np.float32)
    call = Call(q, cache, batch, 0.1, starts=False)
    graph = C.c_uint64()
    H.call("vkml_graph_begin")
    call.run()
    H.call("vkml_graph_end", C.byref(graph))
    try:
        for step in range(4):
            batch.lengths = [n + 61 * step for n in (100, 333, 57)]
            batch.d_lengths.upload(np.asarray(batch.lengths, np.int32))
            H.call("vkml_graph_launch", graph)
            got = call.result()
            close(got, *attention_f64(q, cache, batch, 0.1))
            eager = Call(q, cache, batch, 0.1, starts=False).run().result()
            assert np.array_equal(got.view(np.uint32), eager.view(np.uint32))
    finally:
        H.call("vkml_graph_destroy", graph)


def refused(name, *args):
    status = getattr(H.lib(), name)(*args)
    assert status == 1, status  # VKML_ERROR_INVALID_ARGUMENT
    return H.lib().vkml_last_error().decode()


def test_attend_refusals():
    rng = np.random.default_rng(27)
    batch = Batch(rng, [40, 30], [1, 1], 16)
    cache = Cache(rng, batch.pages, 2, 16, 64, H.F16)
    cache.upload()
    batch.upload()
    q = rng.standard_normal((2, 4, 64)).astype(np.float32)

    def with_(**change):
        c = Call(q, cache, batch, 0.125)
        for name, value in change.items():
            setattr(c.p, name, value)
        return c

    def args(c, **swap):
        b = c.batch
        names = ["q", "k", "v", "table", "lengths", "starts", "gs", "gk", "workspace", "out"]
        values = dict(zip(names, [c.q.p, cache.dk.p, cache.dv.p, b.d_table.p, b.d_lengths.p, b.d_starts.p, None, None, c.workspace.p, c.out.p]))
        values.update(swap)
        return [C.byref(c.p)] + [values[n] for n in names]

    assert "head_dim must be 64 or 128" in refused("vkml_attend_pages", *args(with_(head_dim=96)))
    assert "multiple of kv_heads" in refused("vkml_attend_pages", *args(with_(heads=5)))
    assert "f16 or f32" in refused("vkml_attend_pages", *args(with_(kv_type=H.BF16)))
    assert "power of two" in refused("vkml_attend_pages", *args(with_(page_size=24)))
    assert "groups" in refused("vkml_attend_pages", *args(with_(groups=3)))
    assert "null buffer" in refused("vkml_attend_pages", *args(with_(groups=1)))
    assert "null buffer" in refused("vkml_attend_pages", *args(with_(), workspace=None))
    assert "16-byte" in refused("vkml_attend_pages", *args(with_(), q=C.c_void_p(4096 + 4)))
    assert "one token" in refused("vkml_attend_pages", *args(with_(seqs=1), starts=None))
    assert "null params" in refused("vkml_attend_pages", None, *args(with_())[1:])
    c = with_()
    assert np.all(c.result() == 7.5)  # nothing ran


# ---------------------------------------------------------------- rope and append

def rope_f64(qkv, heads, kv_heads, hd, angles, pos, r, style):
    x = qkv[:, :(heads + 2 * kv_heads) * hd].astype(np.float64).reshape(len(qkv), heads + 2 * kv_heads, hd)
    y, size = x.copy(), np.abs(x)
    turn = np.where((pos >= 0) & (pos < len(angles)), pos, 0)
    c, s = angles[turn, :, 0].astype(np.float64)[:, None], angles[turn, :, 1].astype(np.float64)[:, None]
    ia, ib = (np.arange(0, r, 2), np.arange(1, r, 2)) if style == 0 else (np.arange(r // 2), np.arange(r // 2, r))
    n = heads + kv_heads
    a, b = x[:, :n, ia], x[:, :n, ib]
    y[:, :n, ia], y[:, :n, ib] = a * c - b * s, a * s + b * c
    size[:, :n, ia] = size[:, :n, ib] = np.abs(a) + np.abs(b)
    y[:, :n, :r][(pos < 0) | (pos >= len(angles))] = np.nan
    return y, 2.0 ** -23 * size


def rope_case(seed, heads, kv_heads, hd, page, kv, lengths, new, r, style, pad=0, positions=None, table_rows=None, drop=(), lead=0, trail=0, starts=True,
              stride=0):
    rng = np.random.default_rng(seed)
    batch = Batch(rng, lengths, new, page)
    batch.starts += lead
    batch.tokens += lead + trail
    cache = Cache(rng, batch.pages, kv_heads, page, hd, kv, stride)
    for s, i, value in drop:
        batch.table[s, i] = value
    cache.upload()
    batch.upload()
    width = (heads + 2 * kv_heads) * hd + pad
    qkv = rng.standard_normal((batch.tokens, width)).astype(np.float32)
    rows = table_rows or max(list(lengths) + [1])
    angle = rng.uniform(0, 2 * np.pi, (rows, max(r // 2, 1)))
    angles = np.stack([np.cos(angle), np.sin(angle)], -1).astype(np.float32)
    p = H.RopeKvPagesParams(heads=heads, kv_heads=kv_heads, head_dim=hd, kv_type=kv, page_size=page, pages=cache.pages, seqs=len(lengths),
                            tokens=batch.tokens, table_stride=batch.stride, row_stride=width, page_stride=cache.stride, rotary_dim=r, style=style,
                            positions=rows)
    d_qkv, d_angles, d_q = dev(qkv), dev(angles), dev(np.full((batch.tokens, heads, hd), 7.5, np.float32))
    d_pos = None if positions is None else dev(np.asarray(positions, np.int32))
    print("rope", seed, heads, kv_heads, hd, page, kv, lengths, new, r, style, flush=True)
    H.call("vkml_rope_kv_pages", C.byref(p), d_qkv.p, d_angles.p if r else None, batch.d_table.p, batch.d_lengths.p, batch.d_starts.p if starts else None,
           ptr(d_pos), d_q.p, cache.dk.p, cache.dv.p)
    q, (k, v) = d_q.download(np.float32, (batch.tokens, heads, hd)), cache.download()
    want_k, want_v = cache.k.astype(np.float64), cache.v.astype(np.float64)
    tol_k, tol_v = np.zeros(want_k.shape), np.zeros(want_v.shape)
    want_q, tol_q = np.full(q.shape, 7.5), np.zeros(q.shape)
    half = 2.0 ** -11 if kv == H.F16 else 0.0
    for s, (length, n) in enumerate(zip(lengths, new)):
        a = batch.starts[s]
        pos = np.arange(length - n, length)
        turn = pos if positions is None else np.asarray(positions)[a:a + n]
        y, tol = rope_f64(qkv[a:a + n], heads, kv_heads, hd, angles, turn, r, style)
        want_q[a:a + n], tol_q[a:a + n] = y[:, :heads], tol[:, :heads]
        for i in range(n):
            at = batch.table[s, pos[i] // page] if 0 <= pos[i] < batch.stride * page else -1
            if 0 <= at < cache.pages:
                yk, yv = y[i, heads:heads + kv_heads], y[i, heads + kv_heads:]
                want_k[at, :, pos[i] % page], want_v[at, :, pos[i] % page] = yk, yv
                # f16: the half step, or that of its smallest values
                tol_k[at, :, pos[i] % page] = tol[i, heads:heads + kv_heads] + np.maximum(half * np.abs(yk), 2.0 ** -25 if half else 0)
                tol_v[at, :, pos[i] % page] = np.maximum(half * np.abs(yv), 2.0 ** -25 if half else 0)
    for got, want, tol, name in ((q, want_q, tol_q, "q"), (k, want_k, tol_k, "k"), (v, want_v, tol_v, "v")):
        nan = np.isnan(want)
        assert np.array_equal(np.isnan(got), nan), name
        err = np.abs(got.astype(np.float64) - want)
        assert np.all(err[~nan] <= tol[~nan] * 1.001), (name, np.nanmax(err - tol))


@pytest.mark.parametrize("kv", [H.F16, H.F32])
@pytest.mark.parametrize("style", [0, 1])
@pytest.mark.parametrize("hd,r", [(128, 128), (64, 64), (128, 64), (64, 16), (64, 0), (64, 2), (128, 100), (96, 24), (80, 80), (6, 4)])
def test_rope_into_pages(hd, r, style, kv):
    rope_case(30, 8, 2, hd, 16, kv, [1, 17, 40, 33, 300], [1, 3, 40, 17, 20], r, style)


@pytest.mark.parametrize("kv", [H.F16, H.F32])
@pytest.mark.parametrize("style", [0, 1])
def test_rope_of_decoding_sequences(style, kv):
    lengths = [1 + 37 * i for i in range(50)]
    rope_case(31, 32, 8, 128, 64, kv, lengths, [1] * 50, 128, style, starts=False)
    rope_case(32, 32, 8, 128, 64, kv, lengths, [1] * 50, 128, style)


def test_rope_of_more_sequences_than_a_workgroup_has_threads():
    rope_case(33, 4, 2, 64, 16, H.F16, [3 + i % 5 for i in range(600)], [1 + i % 3 for i in range(600)], 64, 0)


def test_rope_rows_with_gaps():
    for pad in (3, 4):
        rope_case(34, 8, 2, 64, 16, H.F16, [40, 33], [40, 17], 64, 1, pad=pad)
    rope_case(35, 8, 2, 64, 16, H.F32, [40, 33], [40, 17], 64, 0, stride=2 * 16 * 64 + 24)


def test_rope_at_positions_of_its_own():
    rope_case(36, 8, 2, 64, 16, H.F16, [40, 33], [4, 3], 64, 0, positions=[900, 3, 3, 12, 0, 999, 5], table_rows=1000)


def test_rope_past_the_table_gives_nan():
    rope_case(37, 8, 2, 64, 16, H.F16, [40, 33], [40, 3], 32, 0, table_rows=31)
    rope_case(38, 8, 2, 64, 16, H.F32, [40, 33], [2, 2], 32, 1, positions=[-1, 5, 50, -2 ** 31], table_rows=50)


def test_rope_leaves_other_rows_and_pages_alone():
    rope_case(39, 8, 2, 64, 16, H.F16, [40, 33, 20], [20, 17, 0], 64, 0, lead=3, trail=5, drop=[(0, 2, -1), (1, 1, 10 ** 6)])
    # more new tokens than keys: the first stand before position 0
    rope_case(40, 8, 2, 64, 16, H.F16, [3, 33], [5, 1], 64, 0)


def test_rope_refusals():
    H.init()
    good = dict(heads=4, kv_heads=2, head_dim=64, kv_type=H.F16, page_size=16, pages=3, seqs=1, tokens=1, table_stride=2, row_stride=512, page_stride=0,
                rotary_dim=64, style=0, positions=8)
    some = C.c_void_p(4096)

    def why(ptrs=None, **change):
        p = H.RopeKvPagesParams(**{**good, **change})
        return refused("vkml_rope_kv_pages", C.byref(p), *(ptrs or [some] * 9))

    assert "rotary_dim" in why(rotary_dim=66)
    assert "rotary_dim" in why(rotary_dim=3)
    assert "style" in why(style=2)
    assert "rows overlap" in why(row_stride=511)
    assert "head layout" in why(heads=0)
    assert "pages overlap" in why(page_stride=8)
    assert "one token" in why([some] * 4 + [None] + [some] * 4, seqs=2)
    assert "null buffer" in why([None] + [some] * 8)
    assert "null buffer" in why([some, None] + [some] * 7)


# ---------------------------------------------------------------- page copies

@pytest.mark.parametrize("count", [1, 7, 447, 448, 449, 1000])
@pytest.mark.parametrize("layers,vectors,gap", [(1, 1, 0), (3, 5, 0), (2, 1025, 3)])
def test_copy_pages(layers, vectors, gap, count):
    rng = np.random.default_rng(50)
    pages, n = 2 * count + 3, 2 * vectors  # u64s a page
    stride = n + 2 * gap
    layer = pages * stride + 2 * gap
    pools = [rng.integers(0, 2 ** 63, layers * layer, dtype=np.uint64) for _ in range(2)]
    order = rng.permutation(pages).astype(np.int32)
    src, dst = order[:count].copy(), order[count:2 * count].copy()
    src[count // 2:] = src[0]  # the same page may be copied to several
    p = H.CopyPagesParams(pages=pages, layers=layers, count=count, page_bytes=8 * n, page_stride=8 * stride if gap else 0, layer_stride=8 * layer if gap else 0)
    d = [dev(x) for x in pools]
    print("copy", layers, vectors, gap, count, flush=True)
    H.call("vkml_copy_pages", C.byref(p), src.ctypes.data_as(C.c_void_p), dst.ctypes.data_as(C.c_void_p), d[0].p, d[1].p)
    for x, b in zip(pools, d):
        want = x.copy()
        for m in range(layers):
            rows = want[m * layer:m * layer + pages * stride].reshape(pages, stride)
            rows[dst, :n] = rows[src, :n]
        assert np.array_equal(b.download(np.uint64, want.shape), want)


def test_copy_refusals():
    src, dst = np.array([0, 1], np.int32), np.array([2, 3], np.int32)
    pool = dev(np.zeros(1024, np.uint8))

    def why(s=src, d=dst, k=pool.p, v=pool.p, **change):
        p = H.CopyPagesParams(**{**dict(pages=4, layers=1, count=2, page_bytes=16, page_stride=0, layer_stride=0), **change})
        s, d = (None if x is None else np.asarray(x, np.int32) for x in (s, d))
        return refused("vkml_copy_pages", C.byref(p), None if s is None else s.ctypes.data_as(C.c_void_p), None if d is None else d.ctypes.data_as(C.c_void_p), k, v)

    assert "destination is outside" in why(d=[2, 4])
    assert "destination is outside" in why(d=[-1, 3])
    assert "source is outside" in why(s=[0, 4])
    assert "twice" in why(d=[2, 2])
    assert "both a source and a destination" in why(s=[0, 2])
    assert "multiples of 16" in why(page_bytes=24)
    assert "pages overlap" in why(page_bytes=32, page_stride=16)
    assert "layers overlap" in why(layers=2, layer_stride=48)
    assert "null buffer" in why(k=None)
    assert "16-byte" in why(k=C.c_void_p(pool.p.value + 8))
    assert H.lib().vkml_copy_pages(C.byref(H.CopyPagesParams(pages=4, layers=1, count=0, page_bytes=16)), None, None, None, None) == 0


# ---------------------------------------------------------------- together

@pytest.mark.parametrize("kv,style", [(H.F16, 0), (H.F32, 1)])
def test_prompts_forks_decoding_and_compaction(kv, style):
    """A prompt into pages, five forks of it that decode side by side, some
    that end, their pages compacted, and more steps, against each sequence's
    own contiguous float64 history."""
    rng = np.random.default_rng(60)
    heads, kv_heads, hd, page, pages, stride = 8, 2, 128, 16, 64, 12
    cache = Cache(rng, pages, kv_heads, page, hd, kv, fill=np.nan).upload()
    angle = np.arange(200)[:, None] * 10000.0 ** (-np.arange(hd // 2) / (hd // 2))
    angles = np.stack([np.cos(angle), np.sin(angle)], -1).astype(np.float32)
    d_angles = dev(angles)
    width = (heads + 2 * kv_heads) * hd
    free = list(range(pages))[::-1]

    def step(tables, lengths, new, shared, history):
        total = sum(new)
        qkv = rng.standard_normal((total, width)).astype(np.float32)
        starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        table = np.full((len(tables), stride), -1, np.int32)
        for s, t in enumerate(tables):
            table[s, :len(t)] = t
        d = [dev(x) for x in (qkv, table, np.asarray(lengths, np.int32), starts, np.array([0, len(tables)], np.int32), np.array([shared], np.int32))]
        d_q, d_out = dev(np.zeros((total, heads, hd), np.float32)), dev(np.zeros((total, heads, hd), np.float32))
        common = dict(heads=heads, kv_heads=kv_heads, head_dim=hd, kv_type=kv, page_size=page, pages=pages, seqs=len(tables), tokens=total, table_stride=stride)
        rp = H.RopeKvPagesParams(row_stride=width, rotary_dim=hd, style=style, positions=200, **common)
        ap = H.AttendPagesParams(groups=1, scale=hd ** -0.5, softcap=0.0, **common)
        ws = H.empty(max(16, H.lib().vkml_attend_pages_workspace_bytes(C.byref(ap))))
        H.call("vkml_rope_kv_pages", C.byref(rp), d[0].p, d_angles.p, d[1].p, d[2].p, d[3].p, None, d_q.p, cache.dk.p, cache.dv.p)
        H.call("vkml_attend_pages", C.byref(ap), d_q.p, cache.dk.p, cache.dv.p, d[1].p, d[2].p, d[3].p, d[4].p, d[5].p, ws.p, d_out.p)
        out, q = d_out.download(np.float32, (total, heads, hd)), d_q.download(np.float32, (total, heads, hd))
        for s, n in enumerate(new):
            pos = np.arange(lengths[s] - n, lengths[s])
            y, _ = rope_f64(qkv[starts[s]:starts[s + 1]], heads, kv_heads, hd, angles, pos, hd, style)
            for i in range(n):
                # what the cache holds: rounded to its type
                history[s].append((y[i, heads:heads + kv_heads].astype(np.float32).astype(cache.dtype), y[i, heads + kv_heads:].astype(cache.dtype)))
            flat = Batch(rng, [lengths[s]], [n], page)
            mine = Cache(rng, flat.pages, kv_heads, page, hd, kv)
            at = np.arange(lengths[s])
            mine.k[flat.table[0, at // page], :, at % page] = np.stack([h[0] for h in history[s]])
            mine.v[flat.table[0, at // page], :, at % page] = np.stack([h[1] for h in history[s]])
            want, bound = attention_f64(q[starts[s]:starts[s + 1]], mine, flat, hd ** -0.5)
            # a key's rounding to f16 may fall on the other side of a half step: one f16 step of a few of its dims
            slack = 2.0 ** -10 if kv == H.F16 else 2.0 ** -20
            err = np.abs(out[starts[s]:starts[s + 1]] - want)
            assert np.all(err <= bound + slack * np.abs(mine.v.astype(np.float64)).max()), (s, err.max())

    prompt = 43
    tables, history = [[free.pop() for _ in range(3)]], [[]]
    step(tables, [prompt], [prompt], 0, history)
    # four forks: the two whole pages shared, the part-filled third copied
    src, dst = [], []
    for _ in range(4):
        page_id = free.pop()
        src.append(tables[0][2])
        dst.append(page_id)
        tables.append(tables[0][:2] + [page_id])
        history.append(list(history[0]))
    cp = H.CopyPagesParams(pages=pages, layers=1, count=4, page_bytes=kv_heads * page * hd * np.dtype(cache.dtype).itemsize)
    i32 = [np.asarray(x, np.int32) for x in (src, dst)]
    H.call("vkml_copy_pages", C.byref(cp), i32[0].ctypes.data_as(C.c_void_p), i32[1].ctypes.data_as(C.c_void_p), cache.dk.p, cache.dv.p)
    lengths = [prompt] * 5
    for n in ([1] * 5, [1] * 5, [4, 1, 2, 1, 9]):
        lengths = [a + b for a, b in zip(lengths, n)]
        for t, m in zip(tables, lengths):
            while len(t) * page < m:
                t.append(free.pop())
        step(tables, lengths, n, prompt, history)
    # two end; the pages of the others move to the lowest free ones
    for s in (3, 1):
        free += [x for x in tables[s] if sum(x in t for t in tables) == 1]
        del tables[s], lengths[s], history[s]
    used = sorted({x for t in tables for x in t}, reverse=True)
    holes = sorted(set(range(pages)) - set(used))
    moves = {}
    for x in used:
        if holes and holes[0] < x:
            moves[x] = holes.pop(0)
    cp.count = len(moves)
    i32 = [np.asarray(list(x), np.int32) for x in (moves.keys(), moves.values())]
    H.call("vkml_copy_pages", C.byref(cp), i32[0].ctypes.data_as(C.c_void_p), i32[1].ctypes.data_as(C.c_void_p), cache.dk.p, cache.dv.p)
    tables = [[moves.get(x, x) for x in t] for t in tables]
    free = sorted(set(range(pages)) - {x for t in tables for x in t}, reverse=True)
    assert len(moves) > 0 and max(x for t in tables for x in t) < len({x for t in tables for x in t})
    for n in ([1] * 3, [3, 1, 20]):
        lengths = [a + b for a, b in zip(lengths, n)]
        for t, m in zip(tables, lengths):
            while len(t) * page < m:
                t.append(free.pop())
        step(tables, lengths, n, prompt, history)


# ---------------------------------------------------------------- further calls


@pytest.mark.parametrize("kv", [H.F16, H.F32])
@pytest.mark.parametrize("softcap", [0.0, 4.0])
def test_scales_of_either_sign_and_zero(kv, softcap):
    rng = np.random.default_rng(40)
    batch = Batch(rng, [5, 200, 77], [1, 30, 2], 16)
    cache = Cache(rng, batch.pages, 2, 16, 64, kv).upload()
    batch.upload()
    q = rng.standard_normal((batch.tokens, 8, 64)).astype(np.float32)
    close(Call(q, cache, batch, -0.125, softcap).run().result(), *attention_f64(-q, cache, batch, 0.125, softcap), what="negative")
    close(Call(q, cache, batch, 0.0, softcap).run().result(), *attention_f64(q * 0, cache, batch, 0.125, softcap), what="zero")


@pytest.mark.parametrize("kv", [H.F16, H.F32])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_a_row_of_q_that_is_not_finite_leaves_the_others_alone(kv, bad):
    rng = np.random.default_rng(41)
    batch = Batch(rng, [60, 200, 300, 301], [1, 70, 1, 1], 16, [(2, 4, 256)])
    cache = Cache(rng, batch.pages, 2, 16, 128, kv)
    batch.share(cache)
    cache.upload()
    batch.upload()
    q = rng.standard_normal((batch.tokens, 8, 128)).astype(np.float32)
    want, bound = attention_f64(q, cache, batch, 0.1)
    rows = [(0, 3), (5, 0), (70, 7), (71, 2)]
    for t, h in rows:
        q[t, h, 17] = bad
    got = Call(q, cache, batch, 0.1).run().result()
    for t, h in rows:
        assert not np.isfinite(got[t, h]).any()
        got[t, h] = want[t, h]
    close(got, want, bound)


@pytest.mark.parametrize("kv", [H.F16, H.F32])
def test_more_sequences_than_a_workgroup_has_threads(kv):
    rng = np.random.default_rng(42)
    lengths = rng.integers(1, 60, 700)
    new = np.minimum(lengths, rng.choice([0, 1, 1, 1, 2, 9], 700))
    lengths[100:400] += 40
    batch = Batch(rng, lengths.tolist(), new.tolist(), 16, [(100, 400, 37), (400, 502, 0)])
    cache = Cache(rng, batch.pages, 2, 16, 64, kv)
    batch.share(cache)
    cache.upload()
    batch.upload()
    q = rng.standard_normal((batch.tokens, 4, 64)).astype(np.float32)
    close(Call(q, cache, batch, 0.125).run().result(), *attention_f64(q, cache, batch, 0.125))


def test_two_graphs_share_a_workspace():
    rng = np.random.default_rng(43)
    calls = []
    for lengths, new, groups in (([900 + i for i in range(12)], [1] * 12, [(0, 12, 800)]), ([400, 3000], [60, 1], [])):
        batch = Batch(rng, lengths, new, 16, groups)
        cache = Cache(rng, batch.pages, 2, 16, 128, H.F16)
        batch.share(cache)
        cache.upload()
        batch.upload()
        calls.append((rng.standard_normal((batch.tokens, 8, 128)).astype(np.float32), cache, batch))
    workspace = H.empty(max(H.lib().vkml_attend_pages_workspace_bytes(C.byref(params(c, b, 8, 0.1))) for _, c, b in calls))
    runs, graphs = [], []
    try:
        for q, c, b in calls:
            runs.append(Call(q, c, b, 0.1, workspace=workspace))
            graph = C.c_uint64()
            H.call("vkml_graph_begin")
            runs[-1].run()
            H.call("vkml_graph_end", C.byref(graph))
            graphs.append(graph)
        for _ in range(3):
            for graph in graphs:
                H.call("vkml_graph_launch", graph)
            for run, (q, c, b) in zip(runs, calls):
                close(run.result(), *attention_f64(q, c, b, 0.1))
                run.out.upload(np.full(run.shape, 7.5, np.float32))
    finally:
        for graph in graphs:
            H.call("vkml_graph_destroy", graph)


def test_copies_past_a_launch_of_pairs():
    """More pairs than one launch takes, one source for several destinations."""
    rng = np.random.default_rng(44)
    pages, vectors = 1500, 3
    pool = rng.integers(0, 2 ** 32, (2, pages, vectors * 4), dtype=np.uint32)
    dst = rng.permutation(pages)[:1000]
    src = rng.choice(np.setdiff1d(np.arange(pages), dst), 1000)
    k, v = dev(pool[0]), dev(pool[1])
    p = H.CopyPagesParams(pages=pages, layers=1, count=1000, page_bytes=16 * vectors)
    s, d = np.ascontiguousarray(src, np.int32), np.ascontiguousarray(dst, np.int32)
    H.call("vkml_copy_pages", C.byref(p), s.ctypes.data_as(C.c_void_p), d.ctypes.data_as(C.c_void_p), k.p, v.p)
    pool[:, dst] = pool[:, src]
    assert np.array_equal(k.download(np.uint32, pool[0].shape), pool[0]) and np.array_equal(v.download(np.uint32, pool[1].shape), pool[1])


@pytest.mark.parametrize("kv", [H.F16, H.F32])
@pytest.mark.parametrize("scale,softcap", [(0.125, 1e-39), (3e38, 0.0), (-3e38, 2.0)])
def test_extreme_scales_of_rows_that_are_zero(kv, scale, softcap):
    """Every score is 0 (or a cap that is as good as 0): the values' mean."""
    rng = np.random.default_rng(45)
    batch = Batch(rng, [5, 200], [1, 30], 16)
    cache = Cache(rng, batch.pages, 2, 16, 64, kv).upload()
    batch.upload()
    q = np.zeros((batch.tokens, 8, 64), np.float32)
    close(Call(q, cache, batch, scale, softcap).run().result(), *attention_f64(q, cache, batch, 0.125))


@pytest.mark.parametrize("kv", [H.F16, H.F32])
@pytest.mark.parametrize("softcap", [0.25, 1.0, 7.0, 50.0])
def test_softcaps_small_and_large(kv, softcap):
    attend(46, 8, 2, 64, 16, kv, [90, 300, 400], [1, 100, 2], softcap=softcap, q_scale=3.0)


def test_a_captured_step_appends_and_copies():
    """Rope into pages, a page copy and attention in one graph: replayed with
    new lengths and inputs between eager work, each replay as the eager calls."""
    rng = np.random.default_rng(47)
    heads, kv_heads, hd, page, stride, pages = 8, 2, 64, 16, 4, 12
    table = rng.permutation(pages - 2)[:8].astype(np.int32).reshape(2, stride)
    cache = Cache(rng, pages, kv_heads, page, hd, H.F16)
    angles = rng.standard_normal((64, hd // 2, 2)).astype(np.float32)
    src, dst = np.asarray([table[0, 0], table[1, 1]], np.int32), np.asarray([pages - 2, pages - 1], np.int32)
    order = dict(heads=heads, kv_heads=kv_heads, head_dim=hd, kv_type=H.F16, page_size=page, pages=pages, seqs=2, tokens=2, table_stride=stride)
    r = H.RopeKvPagesParams(**order, row_stride=(heads + 2 * kv_heads) * hd, rotary_dim=hd, positions=64)
    a = H.AttendPagesParams(**order, scale=0.125)
    c = H.CopyPagesParams(pages=pages, layers=1, count=2, page_bytes=2 * kv_heads * page * hd)
    workspace = H.empty(H.lib().vkml_attend_pages_workspace_bytes(C.byref(a)))
    d_table, d_angles, src_p, dst_p = dev(table), dev(angles), src.copy(), dst.copy()

    class Side:
        def __init__(self):
            self.k, self.v = dev(cache.k), dev(cache.v)
            self.qkv, self.lengths = dev(np.zeros((2, (heads + 2 * kv_heads) * hd), np.float32)), dev(np.zeros(2, np.int32))
            self.q, self.out = dev(np.zeros((2, heads, hd), np.float32)), dev(np.zeros((2, heads, hd), np.float32))

        def step(self):
            H.call("vkml_rope_kv_pages", C.byref(r), self.qkv.p, d_angles.p, d_table.p, self.lengths.p, None, None, self.q.p, self.k.p, self.v.p)
            H.call("vkml_copy_pages", C.byref(c), src_p.ctypes.data_as(C.c_void_p), dst_p.ctypes.data_as(C.c_void_p), self.k.p, self.v.p)
            H.call("vkml_attend_pages", C.byref(a), self.q.p, self.k.p, self.v.p, d_table.p, self.lengths.p, None, None, None, workspace.p, self.out.p)

        def results(self):
            return [b.download(t, n) for b, t, n in ((self.k, np.uint16, cache.k.shape), (self.v, np.uint16, cache.k.shape),
                                                    (self.q, np.uint32, (2, heads, hd)), (self.out, np.uint32, (2, heads, hd)))]

    replayed, eager = Side(), Side()
    graph = C.c_uint64()
    H.call("vkml_graph_begin")
    replayed.step()
    H.call("vkml_graph_end", C.byref(graph))
    src_p[:], dst_p[:] = -1, -1  # read when the calls were made
    try:
        for i in range(4):
            qkv, lengths = rng.standard_normal((2, (heads + 2 * kv_heads) * hd)).astype(np.float32), np.asarray([1 + i, 30 + 9 * i], np.int32)
            for side in (replayed, eager):
                side.qkv.upload(qkv)
                side.lengths.upload(lengths)
            H.call("vkml_graph_launch", graph)
            got = replayed.results()
            src_p[:], dst_p[:] = src, dst
            eager.step()
            src_p[:], dst_p[:] = -1, -1
            for x, y in zip(got, eager.results()):
                assert np.array_equal(x, y)
    finally:
        H.call("vkml_graph_destroy", graph)


@pytest.mark.parametrize("kv", [H.F16, H.F32])
@pytest.mark.parametrize("lengths,new,groups", [([0], [1], []), ([100, 0], [1, 1], []), ([40, 0], [1, 40], []), ([0] * 64, [1] * 64, []),
                                                ([700, 33, 512] + [0] * 13, [1] * 16, []), ([520, 501, 505, 0, 0], [1] * 5, [(0, 3, 500)]), ([0, 90, 3], [33, 20, 9], [])])
def test_empty_sequences_get_zeros(lengths, new, groups, kv):
    """A padded batch's empty slots, last among them, over a workspace that
    holds another call's pieces and records."""
    rng = np.random.default_rng(48)
    other = Batch(rng, [900 + i for i in range(70)], [1] * 70, 16, [(0, 70, 800)])
    other_cache = Cache(rng, other.pages, 8, 16, 64, kv)
    other.share(other_cache)
    other_cache.upload()
    other.upload()
    batch = Batch(rng, lengths, new, 16, groups)
    cache = Cache(rng, batch.pages, 8, 16, 64, kv)
    batch.share(cache)
    cache.upload()
    batch.upload()
    q = rng.standard_normal((max(70, batch.tokens), 32, 64)).astype(np.float32)
    print("empty sequences", lengths, new, groups, kv, flush=True)
    workspace = H.empty(max(H.lib().vkml_attend_pages_workspace_bytes(C.byref(params(c, b, 32, 0.125))) for c, b in ((other_cache, other), (cache, batch))))
    Call(q[:70], other_cache, other, 0.125, workspace=workspace).run()
    got = Call(q[:batch.tokens], cache, batch, 0.125, starts=max(new) > 1, workspace=workspace).run().result()
    close(got, *attention_f64(q[:batch.tokens], cache, batch, 0.125))
    seen = [length - n + i + 1 for length, n in zip(lengths, new) for i in range(n)]
    for t, keys in enumerate(seen):
        assert got[t].any() == (keys > 0), t


def test_a_captured_call_follows_sequences_that_end():
    rng = np.random.default_rng(49)
    batch = Batch(rng, [300, 200, 100, 50], [1] * 4, 16, stride=20)
    cache = Cache(rng, batch.pages, 8, 16, 64, H.F16).upload()
    batch.upload()
    q = rng.standard_normal((4, 32, 64)).astype(np.float32)
    call = Call(q, cache, batch, 0.125, starts=False)
    graph = C.c_uint64()
    H.call("vkml_graph_begin")
    call.run()
    H.call("vkml_graph_end", C.byref(graph))
    try:
        for lengths in ([300, 200, 100, 50], [300, 200, 100, 0], [300, 0, 0, 0], [0, 0, 0, 0], [0, 0, 0, 50]):
            batch.lengths = lengths
            batch.d_lengths.upload(np.asarray(lengths, np.int32))
            call.out.upload(np.full(call.shape, 7.5, np.float32))
            H.call("vkml_graph_launch", graph)
            got = call.result()
            close(got, *attention_f64(q, cache, batch, 0.125))
            assert got.any((1, 2)).tolist() == [n > 0 for n in lengths]
    finally:
        H.call("vkml_graph_destroy", graph)


LARGE = [(2.0 ** 25, 0.0), (2.0 ** 27, 0.0), (2.0 ** 30, 0.0), (2.0 ** 33, 0.0), (2.0 ** 60, 0.0), (2.0 ** 100, 0.0), (2.0 ** 25, 2.0 ** 28), (2.0 ** 30, 1e30)]


def large_scores(seed, kv, heads, kv_heads, lengths, new, groups, make_k):
    rng = np.random.default_rng(seed)
    batch = Batch(rng, lengths, new, 16, groups)
    cache = Cache(rng, batch.pages, kv_heads, 16, 128, kv)
    cache.k[:] = make_k(rng, cache.k.shape)
    batch.share(cache)
    cache.upload()
    batch.upload()
    return rng, batch, cache


@pytest.mark.parametrize("kv", [H.F16, H.F32])
@pytest.mark.parametrize("size,softcap", LARGE)
@pytest.mark.parametrize("sign", [1, -1])
def test_large_scores_that_are_equal(sign, size, softcap, kv):
    """Every key of a head is the same, so that a row's scores, of about
    `size`, are equal to the last bit: each is the same products in the same
    order. All weights are 1 and the output is the values' mean, whatever the
    score's own rounding: the sums' share of the bound above, without delta
    and x."""
    lengths, new, groups = [40, 700, 900, 20, 333], [1, 1, 1, 1, 60], [(1, 3, 300)]
    rng, batch, cache = large_scores(51, kv, 8, 2, lengths, new, groups,
                                     lambda r, shape: np.broadcast_to(np.abs(r.standard_normal((1, shape[1], 1, shape[3]))) + 0.5, shape))
    q = np.abs(rng.standard_normal((batch.tokens, 8, 128))).astype(np.float32)
    scale = sign * size / 100  # q k is 80 to 160
    got = Call(q, cache, batch, scale, softcap).run().result()
    want, _ = attention_f64(q * 0, cache, batch, 0.1)
    plain, _ = attention_f64(q * 0, cache, batch, 0.1, v=np.abs(cache.v))
    keys = np.concatenate([np.arange(length - n, length) + 1 for length, n in zip(lengths, new)])
    close(got, want, plain * ((keys / 16 + 64) * 2.0 ** -24 + 2.0 ** -20)[:, None, None], f"{size} {softcap}")


@pytest.mark.parametrize("kv", [H.F16, H.F32])
@pytest.mark.parametrize("size", [2.0 ** 20, 2.0 ** 25, 2.0 ** 27, 2.0 ** 30, 2.0 ** 33, 2.0 ** 60, 2.0 ** 100])
def test_large_scores_pick_the_largest(size, kv):
    """Scores of random signs of about `size`: a row whose largest stands out
    by more than the scores' errors (delta and 2^-22 max|x| of the bound
    above, on either side) and 64 more has the weight 1 for that key and less
    than e^-64 for each other one, so that its output is that key's value,
    within the weight's and the sums' rounding. Rows without such a key stay
    finite and among the values."""
    lengths, new, groups = [40, 700, 900, 20, 333], [1, 1, 1, 1, 60], [(1, 3, 300)]
    rng, batch, cache = large_scores(52, kv, 8, 2, lengths, new, groups, lambda r, shape: r.standard_normal(shape))
    q = rng.standard_normal((batch.tokens, 8, 128)).astype(np.float32)
    scale = size / 11.3
    got = Call(q, cache, batch, scale).run().result().astype(np.float64)
    picked = 0
    for s, (length, n) in enumerate(zip(lengths, new)):
        kk, _ = rows_of(cache, cache.k, batch.table[s], length)
        vv, _ = rows_of(cache, cache.v, batch.table[s], length)
        for i in range(n):
            t, seen = batch.starts[s] + i, length - n + i + 1
            for h in range(8):
                K, V, Q = kk[:seen, h // 4].astype(np.float64), vv[:seen, h // 4].astype(np.float64), q[t, h].astype(np.float64)
                x = K @ Q * scale
                off = scale * (2.0 ** -22 * np.abs(Q).max() * np.abs(K).sum(1) + 136 * 2.0 ** -24 * (np.abs(K) @ np.abs(Q))).max() + 2.0 ** -22 * np.abs(x).max()
                most = np.abs(V).max(0)
                assert np.all(np.abs(got[t, h]) <= most * (1 + 2.0 ** -10)), (t, h, got[t, h])
                order = np.argsort(x)
                if seen == 1 or x[order[-1]] - x[order[-2]] > 2 * off + 64:
                    picked += 1
                    assert np.all(np.abs(got[t, h] - V[order[-1]]) <= np.abs(V[order[-1]]) * ((seen / 16 + 64) * 2.0 ** -24 + 2.0 ** -20) + seen * math.exp(-64) * most), (t, h)
    assert picked > 8 * batch.tokens * 0.9


def test_more_rows_than_a_launch_has_threads_for():
    """2129920 new tokens of 32 heads with KV heads of their own: the join's
    waves are 2^32 threads and more. All sequences read the same pages, and q
    is zero: each token's output is the mean of the values up to its own."""
    rng = np.random.default_rng(53)
    heads, hd, page, seqs, n = 32, 64, 16, 4096, 520
    tokens = seqs * n
    assert tokens * heads * 64 >= 2 ** 32
    cache = Cache(rng, 33, heads, page, hd, H.F16).upload()
    p = H.AttendPagesParams(heads=heads, kv_heads=heads, head_dim=hd, kv_type=H.F16, page_size=page, pages=33, seqs=seqs, tokens=tokens, table_stride=33, scale=0.125)
    table = np.broadcast_to(rng.permutation(33).astype(np.int32), (seqs, 33))
    bufs = [dev(table), dev(np.full(seqs, n, np.int32)), dev(np.arange(0, tokens + 1, n, dtype=np.int32))]
    row = heads * hd * 4
    q, out, workspace = H.empty(tokens * row), H.empty(tokens * row), H.empty(H.lib().vkml_attend_pages_workspace_bytes(C.byref(p)))
    print("large", tokens, workspace.nbytes, flush=True)
    H.call("vkml_fill_u32", q.p, 0, tokens * row // 4)
    H.call("vkml_fill_u32", out.p, 0x7FC00000, tokens * row // 4)
    H.call("vkml_attend_pages", C.byref(p), q.p, cache.dk.p, cache.dv.p, *(b.p for b in bufs), None, None, workspace.p, out.p)
    at = np.arange(n)
    v = cache.v[table[0, at // page], :, at % page].astype(np.float64)
    keys = at[:, None, None] + 1
    mean, size = np.cumsum(v, 0) / keys, np.cumsum(np.abs(v), 0) / keys
    bound = size * ((keys / 16 + 64) * 2.0 ** -24 + 2.0 ** -20)
    # the parts of a KV head's work end at every 256th sequence or so
    for s in sorted({min(max(256 * i + d, 0), seqs - 1) for i in range(17) for d in (-2, -1, 0, 1)}):
        got = np.empty((n, heads, hd), np.float32)
        H.call("vkml_memcpy_d2h", got.ctypes.data_as(C.c_void_p), C.c_void_p(out.p.value + s * n * row), got.nbytes)
        close(got, mean, bound, f"sequence {s}")


@pytest.mark.parametrize("heads,kv_heads", [(8, 2), (40, 2)])
def test_scores_of_minus_infinity_weigh_nothing(heads, kv_heads):
    """f32 caches, queries of positive values: a key of -infinity in a dim is
    left out, and a token that sees no other gets zeros."""
    rng = np.random.default_rng(54)
    batch = Batch(rng, [30, 200, 3], [30, 1, 3], 16)
    cache = Cache(rng, batch.pages, kv_heads, 16, 64, H.F32)
    q = (np.abs(rng.standard_normal((batch.tokens, heads, 64))) + 0.1).astype(np.float32)
    out = {0: [0, 1, 2, 17], 1: [5, 190], 2: [0, 1, 2]}
    for s, keys in out.items():
        for pos in keys:
            cache.k[batch.table[s, pos // 16], :, pos % 16, 7] = -np.inf
    cache.upload()
    batch.upload()
    got = Call(q, cache, batch, 0.1).run().result()
    for s, keys in out.items():
        n, length = batch.new[s], batch.lengths[s]
        for i in range(n):
            t = batch.starts[s] + i
            on = [p for p in range(length - n + i + 1) if p not in keys]
            if not on:
                assert not got[t].any(), (s, i)
                continue
            for h in range(heads):
                K, V = (np.stack([x[batch.table[s, p // 16], h // (heads // kv_heads), p % 16] for p in on]).astype(np.float64) for x in (cache.k, cache.v))
                Q = q[t, h].astype(np.float64)
                x = K @ Q * 0.1
                w = np.exp(x - x.max())
                w /= w.sum()
                delta = 0.1 * 72 * 2.0 ** -24 * (np.abs(K) @ np.abs(Q)).max()
                bound = (w @ np.abs(V)) * (2 * delta + 2.0 ** -22 * np.abs(x).max() + (len(on) / 16 + 64) * 2.0 ** -24 + 2.0 ** -20)
                assert np.all(np.abs(got[t, h] - w @ V) <= bound), (s, i, h)


@pytest.mark.parametrize("seed", range(24))
def test_random_batches(seed):
    """Batches of every make: ragged, padded, grouped or not, decoding and
    prompts, more new tokens than keys, over a workspace of NaN bits."""
    rng = np.random.default_rng(1000 + seed)
    heads, kv_heads = HEADS[int(rng.integers(len(HEADS)))]
    hd, page, kv = int(rng.choice([64, 128])), int(rng.choice([16, 32, 128])), [H.F16, H.F32][int(rng.integers(2))]
    n = int(rng.choice([1, 2, 7, 20, 70]))
    new = rng.integers(0, 40, n) if rng.random() < 0.5 and n < 20 else np.ones(n, int)
    own = np.where(rng.random(n) < 0.2, 0, rng.integers(0, 400, n))
    groups, lengths = [], own.copy()
    if n > 1 and rng.random() < 0.7:
        a, b = sorted(rng.choice(n + 1, 2, replace=False).tolist())
        shared = int(rng.integers(1, 600))
        lengths[a:b] = shared + new[a:b] + own[a:b]  # at most the keys before a sequence's new tokens
        groups = [(a, b, shared)]
    if new.sum() == 0:
        new[0] = 1
        lengths[0] = max(lengths[0], 1)
    attend(seed, heads, kv_heads, hd, page, kv, lengths.tolist(), new.tolist(), groups, softcap=float(rng.choice([0.0, 0.0, 20.0])),
           starts=not bool(np.all(new == 1) and rng.random() < 0.5))


@pytest.mark.parametrize("new", [1, 40])
def test_the_longest_sequence(new):
    """2^26 keys, the same 64 pages over and over: key p's score and value are
    those of key p % 1024, so that the softmax is over those with 2^16 times
    their weight (short of the last keys that a token does not see)."""
    rng = np.random.default_rng(55)
    heads, hd, page, keys = 4, 64, 16, 2 ** 26
    cache = Cache(rng, 64, 1, page, hd, H.F16).upload()
    order = rng.permutation(64).astype(np.int32)
    p = H.AttendPagesParams(heads=heads, kv_heads=1, head_dim=hd, kv_type=H.F16, page_size=page, pages=64, seqs=1, tokens=new, table_stride=keys // page, scale=0.125)
    q = rng.standard_normal((new, heads, hd)).astype(np.float32)
    bufs = [dev(np.tile(order, keys // 1024)), dev(np.array([keys], np.int32)), dev(np.array([0, new], np.int32))]
    d_q, out, workspace = dev(q), dev(np.full(q.shape, 7.5, np.float32)), H.empty(H.lib().vkml_attend_pages_workspace_bytes(C.byref(p)))
    print("longest", new, flush=True)
    H.call("vkml_attend_pages", C.byref(p), d_q.p, cache.dk.p, cache.dv.p, *(b.p for b in bufs), None, None, workspace.p, out.p)
    got = out.download(np.float32, q.shape)
    at = np.arange(1024)
    K, V = (x[order[at // page], 0, at % page].astype(np.float64) for x in (cache.k, cache.v))
    want = np.empty(q.shape)
    for t in range(new):
        x = q[t].astype(np.float64) @ K.T * 0.125
        w = np.exp(x - x.max(1, keepdims=True)) * (2 ** 16 - (at >= 1024 - (new - 1 - t)))
        want[t] = (w / w.sum(1, keepdims=True)) @ V
    # Scores off by up to 2e-6, as in the bound above (scale (2^-22 4 * 52 + 72 2^-24 52)), twice;
    # the sums go through blocks of 64 or 128 keys, a wave's or workgroup's run of them and the
    # parts: at most 2^26 / 512 / 64 + 1024 additions in a row, 2^-24 each, of Sum p |v| < 4
    bound = 4 * (4e-5 + (2 ** 26 / 512 / 64 + 1024) * 2.0 ** -24 + 2.0 ** -20)
    assert np.abs(got - want).max() <= bound, np.abs(got - want).max()
    assert np.linalg.norm(got - want) <= 1e-4 * np.linalg.norm(want)


def test_as_many_sequences_as_a_batch_takes():
    """65536 sequences of 0 to 2 keys in a decode step: rope into their pages
    (16 rows a page, a sequence each), then attention."""
    rng = np.random.default_rng(56)
    heads, kv_heads, hd, seqs = 2, 1, 64, 65536
    lengths = rng.integers(0, 3, seqs).astype(np.int32)
    lengths[-5:] = [2, 1, 0, 0, 0]
    table = rng.permutation(seqs).astype(np.int32)
    cache = Cache(rng, seqs, kv_heads, 16, hd, H.F32).upload()
    qkv = rng.standard_normal((seqs, (heads + 2 * kv_heads) * hd)).astype(np.float32)
    common = dict(heads=heads, kv_heads=kv_heads, head_dim=hd, kv_type=H.F32, page_size=16, pages=seqs, seqs=seqs, tokens=seqs, table_stride=1)
    rp, ap = H.RopeKvPagesParams(row_stride=qkv.shape[1], **common), H.AttendPagesParams(scale=0.125, **common)
    d = [dev(qkv), dev(table), dev(lengths), dev(np.arange(seqs + 1, dtype=np.int32))]
    d_q, out, workspace = H.empty(seqs * heads * hd * 4), dev(np.full((seqs, heads, hd), 7.5, np.float32)), H.empty(H.lib().vkml_attend_pages_workspace_bytes(C.byref(ap)))
    print("sequences", seqs, workspace.nbytes, flush=True)
    H.call("vkml_rope_kv_pages", C.byref(rp), d[0].p, None, d[1].p, d[2].p, d[3].p, None, d_q.p, cache.dk.p, cache.dv.p)
    H.call("vkml_attend_pages", C.byref(ap), d_q.p, cache.dk.p, cache.dv.p, d[1].p, d[2].p, d[3].p, None, None, workspace.p, out.p)
    x = qkv.reshape(seqs, heads + 2 * kv_heads, hd)
    assert np.array_equal(d_q.download(np.float32, (seqs, heads, hd)), x[:, :heads])
    some = lengths > 0
    for pool, got, lane in zip((cache.k, cache.v), cache.download(), (heads, heads + 1)):
        pool[table[some], 0, lengths[some] - 1] = x[some, lane]
        assert np.array_equal(got, pool)
    got = out.download(np.float32, (seqs, heads, hd))
    K, V = (p[table, 0, :2].astype(np.float64) for p in (cache.k, cache.v))
    s = np.matmul(x[:, :heads].astype(np.float64), np.ascontiguousarray(K.transpose(0, 2, 1))) * 0.125
    s[lengths < 2, :, 1] = -np.inf
    w = np.exp(s - s.max(2, keepdims=True))
    w /= w.sum(2, keepdims=True)
    w[~some] = 0
    size = np.matmul(w, np.abs(V))
    # delta = 0.125 * 72 2^-24 sum|q k|, at most that of both keys
    delta = 0.125 * 72 * 2.0 ** -24 * np.matmul(np.abs(x[:, :heads].astype(np.float64)), np.abs(K).sum(1)[:, :, None])
    top = np.where(np.isfinite(s), np.abs(s), 0).max(2, keepdims=True)
    close(got, np.matmul(w, V), size * (2 * delta + 2.0 ** -22 * top + 65 * 2.0 ** -24 + 2.0 ** -20))


@pytest.mark.parametrize("seqs,each", [(40, 300), (300, 300)])
def test_sequences_that_overlap_are_not_worked_on(seqs, each):
    """Starts that go up and down, which the rules exclude: the call returns
    and touches the named arrays alone; the next one is as ever."""
    rng = np.random.default_rng(57)
    batch = Batch(rng, [each] * seqs, [each] + [0] * (seqs - 1), 16)
    cache = Cache(rng, batch.pages, 2, 16, 64, H.F16).upload()
    batch.upload()
    q = rng.standard_normal((each, 8, 64)).astype(np.float32)
    call = Call(q, cache, batch, 0.125)
    want = call.run().result()
    close(want, *attention_f64(q, cache, batch, 0.125))
    batch.d_starts.upload(np.asarray([0, each] * (seqs // 2) + [0], np.int32))
    call.run().result()
    k, v = cache.download()
    assert np.array_equal(k, cache.k) and np.array_equal(v, cache.v) and np.array_equal(call.q.download(np.float32, q.shape), q)
    batch.d_starts.upload(batch.starts)
    assert np.array_equal(call.run().result().view(np.uint32), want.view(np.uint32))
