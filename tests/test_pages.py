"""The paged cache's argument checks and batch arithmetic
(vkml-framework_amd/csrc/pages.hpp), compiled with the host's compiler."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from vkml_amd import hip as H

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def pages(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("pages") / "libpages.so")
    subprocess.run(["g++", "-std=c++20", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I" + os.path.join(ROOT, "vkml-framework_amd", "csrc"),
                    os.path.join(ROOT, "tests", "cpp", "pages_c.cpp"), "-o", so], check=True)
    lib = C.CDLL(so)
    for name in ("check_attend_c", "check_rope_c", "check_copy_c", "check_copies_c"):
        getattr(lib, name).restype = C.c_char_p
    return lib


ATTEND = dict(heads=8, kv_heads=2, head_dim=128, kv_type=H.F16, page_size=16, pages=10, seqs=4, tokens=4, table_stride=8, groups=1, page_stride=0,
              scale=0.1, softcap=0.0)
BAD_ATTEND = [
    (dict(heads=0), "kv_heads"), (dict(kv_heads=0), "kv_heads"), (dict(heads=9), "kv_heads"), (dict(heads=258), "128 query heads"),
    (dict(head_dim=0), "head_dim"), (dict(head_dim=96), "head_dim"), (dict(head_dim=256), "head_dim"), (dict(kv_type=H.BF16), "f16 or f32"),
    (dict(kv_type=H.Q8_0), "f16 or f32"), (dict(page_size=0), "power of two"), (dict(page_size=8), "power of two"), (dict(page_size=48), "power of two"),
    (dict(page_size=2048), "power of two"), (dict(pages=0), "pages"), (dict(pages=2 ** 31), "pages"), (dict(page_stride=16 * 2 * 128 - 8), "overlap"),
    (dict(page_stride=16 * 2 * 128 + 4), "multiple of 8"), (dict(seqs=65537), "65536"), (dict(tokens=2 ** 22 + 1), "2^22"), (dict(table_stride=0), "table row"),
    (dict(table_stride=2 ** 22 + 1), "table row"), (dict(groups=5), "groups"), (dict(softcap=-1.0), "softcap"), (dict(softcap=float("nan")), "softcap"),
    (dict(heads=2 ** 10, kv_heads=8, tokens=2 ** 22), "too many rows"), (dict(page_stride=2 ** 33 + 8), "too large"),
    (dict(heads=2 ** 28, kv_heads=2 ** 28), "too large"),
]


@pytest.mark.parametrize("change,why", BAD_ATTEND)
def test_attend_refuses(pages, change, why):
    assert pages.check_attend_c(C.byref(H.AttendPagesParams(**ATTEND))) is None
    got = pages.check_attend_c(C.byref(H.AttendPagesParams(**{**ATTEND, **change})))
    assert got is not None and why in got.decode(), got


def test_attend_takes_the_whole_range(pages):
    for change in (dict(heads=2, kv_heads=2), dict(heads=256), dict(head_dim=64), dict(kv_type=H.F32), dict(page_size=1024), dict(page_stride=16 * 2 * 128 + 8),
                   dict(seqs=65536), dict(table_stride=2 ** 22), dict(groups=0), dict(groups=4), dict(seqs=0, tokens=0, groups=0), dict(softcap=50.0),
                   dict(pages=2 ** 31 - 1)):
        assert pages.check_attend_c(C.byref(H.AttendPagesParams(**{**ATTEND, **change}))) is None, change


ROPE = dict(heads=8, kv_heads=2, head_dim=128, kv_type=H.F16, page_size=16, pages=10, seqs=4, tokens=4, table_stride=8, row_stride=12 * 128, page_stride=0,
            rotary_dim=128, style=0, positions=100)
BAD_ROPE = [
    (dict(heads=0), "head layout"), (dict(kv_heads=0), "head layout"), (dict(head_dim=0), "head layout"), (dict(head_dim=65), "head layout"),
    (dict(head_dim=2048), "head layout"), (dict(heads=5000), "head layout"), (dict(kv_type=H.BF16), "f16 or f32"), (dict(page_size=17), "power of two"),
    (dict(rotary_dim=130), "rotary_dim"), (dict(rotary_dim=7), "rotary_dim"), (dict(style=2), "style"), (dict(row_stride=12 * 128 - 1), "rows overlap"),
    (dict(tokens=2 ** 23), "2^22"), (dict(pages=0), "pages"),
]


@pytest.mark.parametrize("change,why", BAD_ROPE)
def test_rope_refuses(pages, change, why):
    assert pages.check_rope_c(C.byref(H.RopeKvPagesParams(**ROPE))) is None
    got = pages.check_rope_c(C.byref(H.RopeKvPagesParams(**{**ROPE, **change})))
    assert got is not None and why in got.decode(), got


COPY = dict(pages=8, layers=2, count=1, page_bytes=64, page_stride=0, layer_stride=0)
BAD_COPY = [
    (dict(pages=0), "pages"), (dict(pages=2 ** 24 + 1), "pages"), (dict(page_bytes=0), "multiples of 16"), (dict(page_bytes=40), "multiples of 16"),
    (dict(page_stride=72), "multiples of 16"), (dict(layer_stride=520), "multiples of 16"), (dict(page_stride=48), "pages overlap"),
    (dict(layer_stride=496), "layers overlap"), (dict(layers=0), "layers"), (dict(layers=70000), "layers"), (dict(page_bytes=2 ** 30 + 16), "2^30"),
    (dict(page_stride=2 ** 41), "too large"),
]


@pytest.mark.parametrize("change,why", BAD_COPY)
def test_copy_refuses(pages, change, why):
    assert pages.check_copy_c(C.byref(H.CopyPagesParams(**COPY))) is None
    got = pages.check_copy_c(C.byref(H.CopyPagesParams(**{**COPY, **change})))
    assert got is not None and why in got.decode(), got


def _i32(x):
    return np.asarray(x, np.int32)


def test_copy_lists(pages):
    def why(n, src, dst):
        src, dst, marks = _i32(src), _i32(dst), np.zeros((n + 63) // 64, np.uint64)
        got = pages.check_copies_c(n, len(src), src.ctypes.data_as(C.c_void_p), dst.ctypes.data_as(C.c_void_p), marks.ctypes.data_as(C.c_void_p))
        return got and got.decode()

    assert why(130, [0, 0, 64, 1], [129, 128, 63, 65]) is None
    assert "destination is outside" in why(130, [0], [130])
    assert "destination is outside" in why(130, [0], [-1])
    assert "source is outside" in why(130, [130], [0])
    assert "source is outside" in why(130, [-2 ** 31], [0])
    assert "twice" in why(130, [0, 1], [64, 64])
    assert "both" in why(130, [0, 64], [64, 65])
    assert "both" in why(130, [5], [5])


class Batch(C.Structure):
    _fields_ = [("lengths", C.c_void_p), ("starts", C.c_void_p), ("group_starts", C.c_void_p), ("group_keys", C.c_void_p), ("seqs", C.c_int32),
                ("tokens", C.c_int32), ("groups", C.c_int32), ("table_keys", C.c_int32)]


def batch(lengths, starts, group_starts, group_keys, tokens, table_keys):
    keep = [None if x is None else _i32(x) for x in (lengths, starts, group_starts, group_keys)]
    ptrs = [None if x is None else x.ctypes.data for x in keep]
    return Batch(*ptrs, len(lengths), tokens, 0 if group_keys is None else len(group_keys), table_keys), keep


def rows(pages, *args):
    b, keep = batch(*args)
    out = np.zeros((b.seqs, 5), np.int32)
    pages.batch_c(C.byref(b), out.ctypes.data_as(C.c_void_p))
    return out.tolist()


def test_a_batch_is_read_as_given(pages):
    assert rows(pages, [5, 9, 3], None, None, None, 3, 64) == [[0, 1, 5, -1, 0], [1, 1, 9, -1, 0], [2, 1, 3, -1, 0]]
    # sequences 1 and 2 in a group, 3 alone in one (sharing nothing), 0 and 4 in none
    assert rows(pages, [5, 40, 50, 60, 7], [0, 2, 2, 6, 7, 8], [1, 3, 4], [32, 16], 8, 64) == [
        [0, 2, 5, -1, 0], [2, 0, 40, 0, 32], [2, 4, 50, 0, 32], [6, 1, 60, 1, 0], [7, 1, 7, -1, 0]]
    # many groups: the search finds each
    n = 37
    got = rows(pages, [100] * 3 * n, None, range(0, 3 * n + 1, 3), range(1, n + 1), 3 * n, 4096)
    assert [r[3:] for r in got] == [[s // 3, s // 3 + 1] for s in range(3 * n)]


def test_a_batch_that_breaks_the_rules_stays_in_bounds(pages):
    rng = np.random.default_rng(0)
    edge = [-2 ** 31, -1, 0, 1, 5, 64, 65, 1000, 2 ** 31 - 1]
    for _ in range(200):
        n = int(rng.integers(1, 9))
        pick = lambda k: rng.choice(edge, k)  # noqa: E731
        g = int(rng.integers(0, n + 1))
        for first, count, length, group, shared in rows(pages, pick(n), pick(n + 1), pick(g + 1), pick(g), 20, 64):
            assert 0 <= first <= 20 and 0 <= count and first + count <= 20
            assert 0 <= length <= 64 and -1 <= group < max(g, 1) and 0 <= shared <= 64


# ---------------------------------------------------------------- the work of a call, cut into parts

def pieces(pages, b, kv_heads, group, workgroups_log2=9, block=64):
    out = np.zeros((200000, 10), np.int64)
    # blocks of 16 KiB: 32 keys are f32's of 128, 64 f16's of 128, 128 f16's of 64
    hd, f16 = {32: (128, 0), 64: (128, 1), 128: (64, 1)}[block]
    n = pages.pieces_c(C.byref(b), kv_heads, group, hd, f16, workgroups_log2, block, out.ctypes.data_as(C.c_void_p), C.c_int64(len(out)))
    assert n >= 0
    return out[:n]


def segments(pages, b, group):
    out = np.zeros((b.groups + b.seqs, 12), np.int32)
    for i in range(len(out)):
        pages.segment_c(C.byref(b), group, i, out[i].ctypes.data_as(C.c_void_p))
    return out


def check_cut(pages, lengths, new, group_starts, group_keys, kv_heads, group, workgroups_log2, block, table_keys=1 << 20):
    starts = np.concatenate([[0], np.cumsum(new)])
    b, keep = batch(lengths, starts, group_starts, group_keys, int(starts[-1]), table_keys)
    got, seg = pieces(pages, b, kv_heads, group, workgroups_log2, block), segments(pages, b, group)
    s = np.zeros(2, np.int64)
    pages.slots_c(*[C.c_int64(int(x)) for x in (kv_heads, group, len(lengths), b.groups, starts[-1], 1 << workgroups_log2)], s.ctypes.data_as(C.c_void_p))
    # every key of every token is in exactly one of its segments, or in the lead of one
    seen = {}
    for i, (token0, n, lo, first, keys, tiles, step, row, shared, lead, lead_row, span) in enumerate(seg):
        assert lo % 16 == 0 and lo <= first < lo + 16 and n <= max(1, tiles) * step and span % 128 == 0 and lead <= span < lead + 128
        assert tiles == 0 or (tiles - 1) * step < n
        assert lead in (0, first)
        for k in range(n):
            t, end = token0 + k, pages.limit_c(C.byref(b), group, i, int(k))
            seen.setdefault(t, []).extend([(0, lead), (first, max(first, end))])
            assert end - lo <= keys - span or end <= first
    for q, (length, n) in enumerate(zip(lengths, new)):
        for k in range(n):
            end = 0
            for a, z in sorted(x for x in seen[starts[q] + k] if x[1] > x[0]):
                assert a == end
                end = z
            assert end == max(0, length - n + k + 1)
    # the pieces of a tile follow one another and cover it; the first one knows how many there are
    used, tiles = {0: set(), 1: set()}, {}
    for w, h, i, t, k0, k1, slot, is_few, whole, count in got.tolist():
        assert 0 <= slot < s[0 if is_few else 1] and slot not in used[is_few]
        used[is_few].add(slot)
        tiles.setdefault((h, i, t), []).append((w, k0, k1, slot, whole, count))
        assert k0 % block == 0 or k0 == k1
    assert len(tiles) == kv_heads * sum(x[5] for x in seg)
    for (h, i, t), p in tiles.items():
        keys, count = seg[i][4:6]
        assert [x[0] for x in p] == list(range(p[0][0], p[0][0] + len(p))) and [x[3] for x in p] == list(range(p[0][3], p[0][3] + len(p)))
        assert p[0][5] == len(p) and all(x[5] == -1 for x in p[1:])
        assert (len(p) == 1) == bool(p[0][4]) and p[0][1] == 0
        for x, y in zip(p, p[1:]):
            assert x[2] == y[1]
        if t == count - 1:
            assert p[-1][2] == keys
    return got


@pytest.mark.parametrize("block", [32, 64, 128])
@pytest.mark.parametrize("workgroups_log2", [3, 9])
@pytest.mark.parametrize("kv_heads,group", [(1, 1), (2, 4), (8, 4), (2, 3), (1, 16), (1, 128)])
def test_the_parts_cover_the_work(pages, kv_heads, group, workgroups_log2, block):
    rng = np.random.default_rng(1)
    for k in range(12):
        n = int(rng.integers(1, 12))
        new = rng.integers(0, [2, 5, 200][k % 3], n)
        own = new + rng.integers(0, [1, 40, 3000][k // 3 % 3], n)
        if k % 2:
            shared = int(rng.integers(1, 2000))
            check_cut(pages, own + shared, new, [0, n], [shared if n > 1 else 0], kv_heads, group, workgroups_log2, block)
        else:
            check_cut(pages, own, new, None, None, kv_heads, group, workgroups_log2, block)
    cuts = sorted(int(x) for x in rng.integers(0, 10, 4))
    keys = [int(x) for x in rng.integers(1, 700, 3)]
    total = np.full(10, 700) + rng.integers(1, 50, 10)
    check_cut(pages, total, np.ones(10, int), cuts, keys, kv_heads, group, workgroups_log2, block)


def test_shared_keys_are_a_segment_where_tokens_are_few(pages):
    def lead(new, group):
        n = len(new)
        b, keep = batch([500 + x for x in new], np.concatenate([[0], np.cumsum(new)]), [0, n], [500], sum(new), 4096)
        s = segments(pages, b, group)
        assert (s[0][5] > 0) == all(x[9] == 0 for x in s[1:])
        return [int(x[9]) for x in s[1:]]
    assert lead([1] * 8, 4) == [0] * 8
    assert lead([1, 31], 4) == [0, 0]  # 32 tokens of 128 rows a tile
    assert lead([1, 32], 4) == [500, 500]
    assert lead([1] * 5, 64) == [0] * 5
    assert lead([1] * 5, 65) == [500] * 5  # a tile a token either way


def test_a_large_prompt_is_cut_evenly(pages):
    got = check_cut(pages, [4096, 33], [4096, 1], None, None, 8, 4, 9, 64)
    load = np.zeros(512)
    for w, _, _, _, k0, k1, *_ in got.tolist():
        load[w] += k1 - k0 + 171
    assert load.max() < 1.1 * load.mean()


def test_the_first_head_of_a_part(pages):
    for per_head in (1, 7, 129, 1000003, 2 ** 40 + 5):
        for kv_heads in (1, 2, 3, 8, 96):
            for w_log2 in (3, 9):
                assert not any(pages.first_head_c(C.c_int64(per_head), kv_heads, w_log2, w) for w in range(1 << w_log2))


def test_parts_of_long_batches_fit_64_bits(pages):
    n = 2 ** 22
    b, keep = batch([n], [0, n], None, None, n, 2 ** 26)
    out = np.zeros(12, np.int32)
    pages.segment_c(C.byref(b), 128, 0, out.ctypes.data_as(C.c_void_p))
    assert out[4:7].tolist() == [n, n, 1]  # a tile a token


def test_the_work_of_a_batch_that_breaks_the_rules_is_finite(pages):
    rng = np.random.default_rng(2)
    edge = [-2 ** 31, -1, 0, 1, 5, 64, 65, 1000, 2 ** 31 - 1]
    for _ in range(100):
        n = int(rng.integers(1, 9))
        pick = lambda k: rng.choice(edge, k)  # noqa: E731
        g = int(rng.integers(0, n + 1))
        b, keep = batch(pick(n), pick(n + 1), pick(g + 1), pick(g), 20, 640)
        for token0, rows, lo, first, keys, tiles, step, row, shared, lead, lead_row, span in segments(pages, b, 4).tolist():
            assert 0 <= token0 and token0 + rows <= 20 and 0 <= lo <= first <= 640 and lo + keys - span <= 660 and 0 <= tiles <= 20
            assert 0 <= lead <= 640 and 0 <= lead_row < n and (tiles == 0 or 0 <= row < n)
        for w, h, i, t, k0, k1, slot, few, whole, count in pieces(pages, b, 2, 4).tolist():
            assert 0 <= k0 <= k1 <= 660 + 768 and slot >= 0


@pytest.mark.parametrize("change,why", [(dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(scale=float("-inf")), "scale"),
                                        (dict(softcap=float("inf")), "softcap")])
def test_attend_refuses_what_is_not_finite(pages, change, why):
    got = pages.check_attend_c(C.byref(H.AttendPagesParams(**{**ATTEND, **change})))
    assert got is not None and why in got.decode(), got
    for fine in (dict(scale=0.0), dict(scale=-0.1), dict(scale=3.0e38)):
        assert pages.check_attend_c(C.byref(H.AttendPagesParams(**{**ATTEND, **fine}))) is None


EMPTY = [([0], [1]), ([100, 0], [1, 1]), ([2, 2, 2, 0], [1, 1, 1, 1]), ([40, 0], [1, 40]), ([0] * 64, [1] * 64), ([0, 0, 0], [40, 1, 200]), ([0, 700, 0, 3, 0], [1, 300, 33, 7, 4]),
         ([3000] * 5 + [0] * 27, [1] * 32), ([33, 20, 5], [50, 20, 40])]


@pytest.mark.parametrize("block", [32, 64, 128])
@pytest.mark.parametrize("workgroups_log2", [3, 9])
@pytest.mark.parametrize("kv_heads,group", [(1, 1), (2, 4), (8, 4), (2, 3), (1, 16), (1, 128)])
def test_the_parts_cover_tokens_without_keys(pages, kv_heads, group, workgroups_log2, block):
    """Empty slots of a padded batch, last, alone and among others, and more
    new tokens than keys: a tile whose cost is its own cost alone belongs to
    the part that reaches its end."""
    for lengths, new in EMPTY:
        check_cut(pages, lengths, new, None, None, kv_heads, group, workgroups_log2, block)
    # behind and before a group, and in one that shares nothing
    check_cut(pages, [520, 501, 505, 0, 0], [1] * 5, [0, 3], [500], kv_heads, group, workgroups_log2, block)
    check_cut(pages, [0, 520, 501, 0], [1] * 4, [1, 3], [500], kv_heads, group, workgroups_log2, block)
    check_cut(pages, [0, 0, 0], [1] * 3, [0, 3], [0], kv_heads, group, workgroups_log2, block)


def test_the_parts_of_a_batch_that_breaks_the_rules_cover_its_tiles(pages):
    rng = np.random.default_rng(3)
    edge = [-2 ** 31, -1, 0, 1, 5, 64, 65, 1000, 2 ** 31 - 1]
    for _ in range(200):
        n = int(rng.integers(1, 9))
        pick = lambda k: rng.choice(edge, k)  # noqa: E731
        g = int(rng.integers(0, n + 1))
        b, keep = batch(pick(n), pick(n + 1), pick(g + 1), pick(g), 20, 640)
        got, seg = pieces(pages, b, 2, 4), segments(pages, b, 4)
        tiles = {}
        for w, h, i, t, k0, k1, slot, few, whole, count in got.tolist():
            tiles.setdefault((h, i, t), []).append(count)
        assert len(tiles) == 2 * sum(x[5] for x in seg.tolist())
        assert all(p[0] == len(p) for p in tiles.values())


def test_a_grid_holds_every_workgroup_below_2_32_threads(pages):
    for n in (1, 2, 4096, 2 ** 23 - 1, 2 ** 23, 2 ** 23 + 1, 2 ** 24, 3 * 2 ** 23 + 5, 2 ** 29 - 1, 2 ** 29):
        out = np.zeros(2, np.uint32)
        pages.grid_c(C.c_uint32(n), out.ctypes.data_as(C.c_void_p))
        x, y = out.tolist()
        assert n <= x * y < n + x and x * 256 < 2 ** 32 and 0 < y < 65536
        # the waves' numbers, four a workgroup, fit 32 bits
        assert x * y * 4 < 2 ** 32


def tile_costs(pages, b, group, hd, f16, i, most):
    out = np.zeros((most, 4), np.int64)
    pages.costs_c.restype = C.c_int64
    total = pages.costs_c(C.byref(b), group, hd, f16, i, out.ctypes.data_as(C.c_void_p), C.c_int64(most))
    return total, out


@pytest.mark.parametrize("hd,f16", [(64, 0), (64, 1), (128, 0), (128, 1)])
@pytest.mark.parametrize("length,new,group", [(2 ** 26, 2 ** 22, 128), (2 ** 26, 2 ** 22, 1), (2 ** 22, 2 ** 22, 128), (2 ** 26, 1, 1), (5, 2 ** 20, 4), (0, 100, 8)])
def test_costs_of_long_batches_fit_64_bits(pages, length, new, group, hd, f16):
    """Tile costs against whole numbers of any size: their sums, the order and
    what is found from a unit."""
    b, keep = batch([length], [0, new], None, None, new, 2 ** 26)
    step = max(1, 128 // group)
    few = new * group <= 16
    tiles = 1 if few else -(-new // step)
    total, got = tile_costs(pages, b, group, hd, f16, 0, tiles)
    key = {(64, 1): (4, 12), (128, 1): (8, 24), (64, 0): (8, 14), (128, 0): (16, 28)}[hd, f16][0 if few else 1]
    own = (2600 if few else 3600) if f16 else 600
    # the keys that a tile's last token sees; where the first tokens see none, all that any sees
    last = np.full(tiles, new) if few or length < new else np.minimum((np.arange(tiles) + 1) * step, new)
    want = own + key * np.maximum(0, length - new + last).astype(np.int64)
    assert want.max() < 2 ** 31 and int(want.max()) * tiles < 2 ** 63
    assert np.array_equal(got[:, 0], want)
    assert np.array_equal(got[:, 1], np.cumsum(want) - want)
    assert np.array_equal(got[:, 2], np.arange(tiles)) and np.array_equal(got[:, 3], np.arange(tiles))
    assert total == want.sum()


@pytest.mark.parametrize("kv_heads,group,lengths,new", [(8, 4, [4096, 33], [4096, 1]), (8, 4, [30, 4000, 900, 2500], [1] * 4), (32, 1, [32768], [1]), (8, 4, [2000] * 64, [1] * 64)])
def test_parts_cost_the_same_but_for_their_ends(pages, kv_heads, group, lengths, new):
    """What a workgroup takes, in the rule's own costs: a part's share, and at
    most a tile's own cost and a block of keys more at each end."""
    got = check_cut(pages, lengths, new, None, None, kv_heads, group, 9, 64)
    b, keep = batch(lengths, np.concatenate([[0], np.cumsum(new)]), None, None, sum(new), 1 << 20)
    seg = segments(pages, b, group)
    few = [bool(n * group <= 16) for n in new]
    key, own = {True: 8, False: 24}, {True: 2600, False: 3600}
    load, parts, total = np.zeros(512), set(), 0
    for i in range(len(lengths)):
        total += kv_heads * tile_costs(pages, b, group, 128, 1, i, int(seg[i][5]))[0]
    for w, h, i, t, k0, k1, *_ in got.tolist():
        load[w] += (own[few[i]] if k0 == 0 else 0) + key[few[i]] * (k1 - k0)
    n = 512
    while n > 8 and total // n < 512:
        n //= 2
    ends = max(own[f] + 64 * key[f] for f in few)
    assert load.max() <= total / n + 2 * ends
    assert abs(load.sum() - total) <= sum(own[f] / 8 + 1 for f in few) * kv_heads * len(got)


def test_most_tiles(pages):
    """No batch within the rules has more tiles of more than 16 rows a KV head;
    one whose sequences or groups overlap does. 256 threads' sums of one more
    than that each fit the 32 bits in which they are counted."""
    pages.most_tiles_c.restype = C.c_int64
    most = lambda *n: pages.most_tiles_c(*[C.c_int64(int(x)) for x in n])  # noqa: E731
    assert max(most(g, 65536, 65536, 2 ** 22) for g in (1, 2, 3, 4, 64, 65, 128)) * 257 < 2 ** 32
    rng = np.random.default_rng(4)
    for k in range(300):
        n, group = int(rng.integers(1, 30)), int(rng.choice([1, 3, 4, 16, 65, 128]))
        new = rng.integers(0, [2, 9, 300][k % 3], n)
        cuts = sorted(int(x) for x in rng.integers(0, n + 1, 4))
        starts = np.concatenate([[0], np.cumsum(new)])
        b, keep = batch(new + 700, starts, cuts, [int(x) for x in rng.integers(0, 700, 3)], int(starts[-1]), 4096)
        seg = segments(pages, b, group)
        assert sum(x[5] for x in seg.tolist() if x[1] * group > 16) <= most(group, n, 3, starts[-1])
    b, keep = batch([500] * 40, [0, 300] * 20 + [0], None, None, 300, 4096)
    assert sum(x[5] for x in segments(pages, b, 4).tolist()) == 200 > most(4, 40, 0, 300)
