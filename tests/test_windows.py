"""Checks of trees, windows, kept drafts and samples, and how a windowed call's
work is divided (vkml-framework_amd/csrc/pages.hpp, sample.hpp), compiled with
the host's compiler."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from vkml_amd import hip as H

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("windows") / "libwindows.so")
    subprocess.run(["g++", "-std=c++20", "-O1", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover=undefined", "-shared", "-fPIC",
                    "-I" + os.path.join(ROOT, "vkml-framework_amd", "csrc"), os.path.join(ROOT, "tests", "cpp", "windows_c.cpp"), "-o", so], check=True)
    lib = C.CDLL(so)
    for name in ("check_tree_c", "check_window_c", "check_keep_c", "check_sample_c"):
        getattr(lib, name).restype = C.c_char_p
    lib.sample_workspace_c.restype = C.c_uint64
    lib.tiles_c.restype = C.c_int64
    lib.window_pieces_c.restype = C.c_int64
    return lib


def said(why):
    return None if why is None else why.decode()


ATTEND = dict(heads=8, kv_heads=2, head_dim=128, kv_type=H.F16, page_size=16, pages=10, seqs=4, tokens=4, table_stride=8, groups=0, page_stride=0, scale=0.1, softcap=0.0)


def test_trees_and_windows_refuse(host):
    assert host.check_tree_c(1) is None and host.check_tree_c(128) is None
    assert "seen_words" in said(host.check_tree_c(0)) and "seen_words" in said(host.check_tree_c(129))
    p = H.AttendPagesParams(**ATTEND)
    assert host.check_window_c(C.byref(p), 1) is None and host.check_window_c(C.byref(p), 2 ** 32 - 1) is None
    assert "window" in said(host.check_window_c(C.byref(p), 0))
    assert "groups" in said(host.check_window_c(C.byref(H.AttendPagesParams(**{**ATTEND, "groups": 1})), 5))


KEEP = dict(kv_heads=2, head_dim=128, kv_type=H.F16, page_size=16, pages=10, layers=3, seqs=4, tokens=20, table_stride=8, page_stride=0, layer_stride=0)


@pytest.mark.parametrize("change,why", [
    (dict(kv_heads=0), "head layout"), (dict(head_dim=0), "head layout"), (dict(head_dim=3), "head layout"), (dict(head_dim=1026), "head layout"),
    (dict(kv_heads=4097), "head layout"), (dict(kv_type=H.BF16), "f16 or f32"), (dict(page_size=24), "power of two"), (dict(pages=0), "pages"),
    (dict(layers=0), "layers"), (dict(layers=65536), "layers"), (dict(seqs=65537), "65536"), (dict(tokens=2 ** 22 + 1), "2^22"), (dict(table_stride=0), "table row"),
    (dict(page_stride=8), "pages overlap"), (dict(page_stride=4100), "multiple of 8"), (dict(layer_stride=4096 * 9), "layers overlap"),
    (dict(layer_stride=4096 * 10 + 4), "multiple of 8"), (dict(layer_stride=2 ** 46 + 8), "too large"), (dict(layer_stride=2 ** 46, layers=65535), "too large"),
    (dict(pages=2 ** 31 - 1, page_stride=2 ** 33), "too large")])
def test_keep_refuses(host, change, why):
    assert host.check_keep_c(C.byref(H.KeepDraftsParams(**KEEP))) is None
    assert why in said(host.check_keep_c(C.byref(H.KeepDraftsParams(**{**KEEP, **change}))))


def test_keep_takes_the_whole_range(host):
    for change in (dict(seqs=0, tokens=0), dict(head_dim=2, page_stride=0), dict(kv_type=H.F32), dict(layers=65535), dict(layer_stride=4096 * 10), dict(page_stride=4104)):
        assert host.check_keep_c(C.byref(H.KeepDraftsParams(**{**KEEP, **change}))) is None, change


@pytest.mark.parametrize("change,why", [(dict(vocab=0), "logits"), (dict(vocab=2 ** 22 + 1, row_stride=2 ** 23), "logits"), (dict(row_stride=999), "overlap"),
                                        (dict(row_stride=2 ** 41), "too large"), (dict(rows=2 ** 21 + 1), "too many"),
                                        (dict(rows=2 ** 20 + 1, vocab=40000, row_stride=40000), "too many")])
def test_sample_refuses(host, change, why):
    fine = dict(rows=5, vocab=1000, row_stride=1000)
    assert host.check_sample_c(C.byref(H.SampleParams(**fine))) is None
    assert why in said(host.check_sample_c(C.byref(H.SampleParams(**{**fine, **change}))))


def test_the_workspace_of_a_sample(host):
    need = lambda rows, vocab: host.sample_workspace_c(C.byref(H.SampleParams(rows=rows, vocab=vocab, row_stride=vocab)))  # noqa: E731
    assert need(7, 1) == need(7, 32768) == 0
    assert need(1, 32769) > 0 and need(3, 128256) % 8 == 0 and need(1, 2 ** 22) > 0
    assert need(40, 128256) < 7 << 20


class Batch(C.Structure):
    _fields_ = [("lengths", C.c_void_p), ("starts", C.c_void_p), ("group_starts", C.c_void_p), ("group_keys", C.c_void_p), ("seqs", C.c_int32),
                ("tokens", C.c_int32), ("groups", C.c_int32), ("table_keys", C.c_int32)]


def batch(lengths, new, table_keys):
    keep = [np.asarray(lengths, np.int32), np.concatenate([[0], np.cumsum(new)]).astype(np.int32)]
    return Batch(keep[0].ctypes.data, keep[1].ctypes.data, None, None, len(lengths), int(keep[1][-1]), 0, table_keys), keep


def blocks(hd, f16):
    return 16384 // (hd * (2 if f16 else 4))


def window_of(host, window, sinks, block, table_keys):
    p = H.AttendPagesParams(**{**ATTEND, "table_stride": table_keys // 16})
    out = np.zeros(3, np.int32)
    host.window_c(C.byref(p), C.c_uint32(window), C.c_uint32(sinks), block, out.ctypes.data_as(C.c_void_p))
    return out


def tiles(host, b, group, hd, f16, i, win):
    head, out = np.zeros(8, np.int32), np.zeros((70000, 11), np.int64)
    cost = host.tiles_c(C.byref(b), group, hd, int(f16), i, win.ctypes.data_as(C.c_void_p), head.ctypes.data_as(C.c_void_p), out.ctypes.data_as(C.c_void_p), C.c_int64(len(out)))
    return cost, head.tolist(), out[:head[2]].tolist()


def check(host, lengths, new, window, sinks, group, hd, f16, kv_heads=2, workgroups_log2=9, table_keys=1 << 20):
    block = blocks(hd, f16)
    win = window_of(host, window, sinks, block, table_keys)
    assert win[2] % block == 0 and win[1] <= win[2] < win[1] + block
    b, keep = batch(lengths, new, table_keys)
    ends = {}
    for s, (length, n) in enumerate(zip(lengths, new)):
        cost, (token0, rows, count, step, straight, few, lead_row, row), each = tiles(host, b, group, hd, f16, s, win)
        assert rows == n and token0 == sum(new[:s]) and row == s and 0 <= straight <= count
        before = 0
        for t, (own, at, first, last, keys, span, lead, lo, start, end, limit) in enumerate(each):
            assert at == before and first == last == t and own > 0
            before += own
            ends[s, t] = keys
            assert lo % 16 == 0 and lo <= start and (lead == 0 or (lead_row == s and lead <= span and span % block == 0))
            # every key that a token of the tile sees is on the axis, once
            for k in range(t * step, min(n, (t + 1) * step)):
                pos = length - n + k
                assert limit + k - t * step == pos + 1
                low = pos - min(window, 1 << 27) + 1
                for a, z in ((0, min(sinks, pos + 1, max(0, low))), (max(0, low), pos + 1)):
                    if z <= a:
                        continue
                    if lead and z <= lead:
                        continue  # the sinks
                    assert start <= a and z <= end and span + z - lo <= keys and (lead == 0 or a >= lead), (s, t, k, a, z)
            assert end <= max(0, length)
        assert before == cost
    out = np.zeros((300000, 6), np.int64)
    n = host.window_pieces_c(C.byref(b), kv_heads, group, hd, int(f16), win.ctypes.data_as(C.c_void_p), workgroups_log2, block, out.ctypes.data_as(C.c_void_p), C.c_int64(len(out)))
    assert n >= 0
    found = {}
    for h, i, t, k0, k1, count in out[:n].tolist():
        found.setdefault((h, i, t), []).append((k0, k1, count))
    assert len(found) == kv_heads * len(ends)
    for (h, i, t), p in found.items():
        assert p[0][0] == 0 and p[-1][1] == ends[i, t] and p[0][2] == len(p)
        assert all(x[1] == y[0] and (y[0] % block == 0 or y[0] == y[1]) for x, y in zip(p, p[1:])), (p, block)


@pytest.mark.parametrize("hd,f16", [(64, True), (128, True), (64, False), (128, False)])
@pytest.mark.parametrize("group", [1, 3, 4, 16, 128])
def test_a_window_s_tiles_hold_every_key_that_is_seen(host, group, hd, f16):
    rng = np.random.default_rng(group * hd + f16)
    for k in range(25):
        n = int(rng.integers(1, 7))
        new = rng.integers(0, [2, 5, 200][k % 3], n).tolist()
        lengths = [x + int(rng.integers(0, [1, 40, 3000][k // 3 % 3])) for x in new]
        window = int(rng.choice([1, 2, 15, 16, 17, 64, 300, 1000, 5000, 2 ** 31, 2 ** 32 - 1]))
        sinks = int(rng.choice([0, 1, 4, 16, 100, 128, 129, 700, 2 ** 32 - 1]))
        check(host, lengths, new, window, sinks, group, hd, f16, workgroups_log2=int(rng.choice([3, 9])))


def test_a_window_s_edges(host):
    check(host, [2 ** 20], [1], 4096, 4, 4, 128, True)
    check(host, [2 ** 20 - 5, 1, 0], [700, 1, 0], 1, 0, 4, 128, True)
    check(host, [4101] * 4, [1] * 4, 4096, 4, 4, 128, True)  # about to slide
    for length in range(150, 290, 7):
        check(host, [length], [3], 100, 4, 4, 64, True)


def test_windows_of_a_batch_that_breaks_the_rules_stay_in_bounds(host):
    rng = np.random.default_rng(2)
    edge = [-2 ** 31, -1, 0, 1, 5, 64, 65, 1000, 2 ** 31 - 1]
    for _ in range(300):
        n = int(rng.integers(1, 9))
        lengths, starts = _i32(rng.choice(edge, n)), _i32(rng.choice(edge, n + 1))
        b = Batch(lengths.ctypes.data, starts.ctypes.data, None, None, n, 20, 0, 640)
        win = window_of(host, int(rng.choice([1, 7, 100, 640, 2 ** 32 - 1])), int(rng.choice([0, 4, 200, 2 ** 32 - 1])), 64, 640)
        for i in range(n):
            cost, (token0, rows, count, step, straight, few, lead_row, row), each = tiles(host, b, 4, 128, True, i, win)
            assert 0 <= token0 and token0 + rows <= 20 and 0 <= count <= 20 and 0 <= lead_row < n and 0 <= row < n
            for own, at, first, last, keys, span, lead, lo, start, end, limit in each:
                assert own > 0 and 0 <= lead <= 640 and 0 <= lo <= start <= 640 and end <= 660 and first == last


def test_the_largest_window_fits_32_bits(host):
    win = window_of(host, 2 ** 26 - 200, 4, 128, 2 ** 26)
    b, keep = batch([2 ** 26], [2 ** 12], 2 ** 26)
    cost, head, each = tiles(host, b, 128, 64, False, 0, win)
    assert each[-1][0] > 0 and each[-1][4] <= 2 ** 26 + 400 and cost == each[-1][1] + each[-1][0]
    assert head[4] < head[2]  # the last ones slide


def _i32(x):
    return np.asarray(x).astype(np.int64).astype(np.int32)
