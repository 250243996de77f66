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
    (dict(table_stride=2 ** 27), "table row"), (dict(groups=5), "groups"), (dict(softcap=-1.0), "softcap"), (dict(softcap=float("nan")), "softcap"),
    (dict(heads=2 ** 10, kv_heads=8, tokens=2 ** 22), "too many rows"),
]


@pytest.mark.parametrize("change,why", BAD_ATTEND)
def test_attend_refuses(pages, change, why):
    assert pages.check_attend_c(C.byref(H.AttendPagesParams(**ATTEND))) is None
    got = pages.check_attend_c(C.byref(H.AttendPagesParams(**{**ATTEND, **change})))
    assert got is not None and why in got.decode(), got


def test_attend_takes_the_whole_range(pages):
    for change in (dict(heads=2, kv_heads=2), dict(heads=256), dict(head_dim=64), dict(kv_type=H.F32), dict(page_size=1024), dict(page_stride=16 * 2 * 128 + 8),
                   dict(seqs=65536), dict(table_stride=2 ** 27 - 1), dict(groups=0), dict(groups=4), dict(seqs=0, tokens=0, groups=0), dict(softcap=50.0),
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
