"""vkml::PageTable (vkml-framework_amd/src/page_table.cpp) on the CPU, through
a check program built from that file alone: random calls, with the pages'
contents kept here as the cache would have them. Whatever is called, every
sequence reads its own tokens back through its pages."""
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def exe(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("bin") / "page_table_check")
    subprocess.run(["g++", "-std=c++20", "-O1", "-Wall", "-Werror", "-I" + os.path.join(ROOT, "vkml-framework_amd", "include"),
                    os.path.join(ROOT, "tests", "cpp", "page_table_check.cpp"), os.path.join(ROOT, "vkml-framework_amd", "src", "page_table.cpp"), "-o", out],
                   check=True)
    return out


class Table:
    """The program, the tokens that each sequence should hold, and the pools'
    contents as the returned copies and the writes make them."""

    def __init__(self, exe, pages, page):
        self.p = subprocess.Popen([exe, str(pages), str(page)], stdin=subprocess.PIPE, stdout=subprocess.PIPE, text=True, bufsize=1)
        self.pages, self.page = pages, page
        self.pool = np.full((pages, page), -1)
        self.want = {}
        self.token = 0

    def ask(self, *words):
        self.p.stdin.write(" ".join(str(w) for w in words) + "\n")
        self.p.stdin.flush()
        return self.p.stdout.readline().rstrip("\n")

    def numbers(self, *words):
        got = self.ask(*words)
        assert not got.startswith("error"), (words, got)
        return [int(x) for x in got.split()]

    def state(self):
        parts = self.ask("state", *self.want).split("|")
        rows = [[int(x) for x in p.split()] for p in parts[1:]]
        return int(parts[0]), {i: (r[0], r[1:]) for i, r in zip(self.want, rows)}

    def copies(self, got):
        pairs = list(zip(got[::2], got[1::2]))
        sources, targets = {a for a, _ in pairs}, [b for _, b in pairs]
        assert len(set(targets)) == len(targets) and not sources & set(targets)
        for a, b in pairs:
            self.pool[b] = self.pool[a]
        return pairs

    def append(self, ids, counts):
        words = [w for pair in zip(ids, counts) for w in pair]
        before = self.state()
        need = 0
        for i, n in zip(ids, counts):
            need += -(-(before[1][i][0] + n) // self.page) - len(before[1][i][1])
        # A part-filled page that k of its holders write into gets k copies,
        # or k - 1 if nobody else holds it.
        writers = {}
        for i, n in zip(ids, counts):
            if n and before[1][i][0] % self.page:
                writers[before[1][i][1][-1]] = writers.get(before[1][i][1][-1], 0) + 1
        for page, k in writers.items():
            holders = sum(page in row for _, row in before[1].values())
            need += k if holders > k else k - 1
        got = self.ask("append", *words)
        if need > before[0]:
            assert got.startswith("error") and "%d pages needed" % need in got, (got, need, before)
            assert self.state() == before
            return False
        assert not got.startswith("error"), got
        self.copies([int(x) for x in got.split()])
        free, rows = self.state()
        assert free == before[0] - need
        for i, n in zip(ids, counts):
            for _ in range(n):
                at = len(self.want[i])
                self.pool[rows[i][1][at // self.page], at % self.page] = self.token
                self.want[i].append(self.token)
                self.token += 1
        return True

    def check(self):
        free, rows = self.state()
        held = set()
        for i, tokens in self.want.items():
            length, row = rows[i]
            assert length == len(tokens) and len(row) == -(-length // self.page)
            assert all(0 <= p < self.pages for p in row) and len(set(row)) == len(row)
            held.update(row)
            got = self.pool[row].reshape(-1)[:length].tolist() if row else []
            assert got == tokens, (i, got, tokens)
        assert free == self.pages - len(held)
        return rows

    def close(self):
        self.p.stdin.close()
        assert self.p.wait(timeout=10) == 0


@pytest.mark.parametrize("seed,pages,page", [(0, 40, 4), (1, 12, 4), (2, 64, 16), (3, 9, 1), (4, 200, 16)])
def test_every_sequence_reads_its_own_tokens(exe, seed, pages, page):
    rng = np.random.default_rng(seed)
    t = Table(exe, pages, page)
    refused = 0
    for _ in range(400):
        ids = list(t.want)
        what = rng.choice(["create", "fork", "append", "append", "append", "truncate", "release", "compact", "shared"])
        if what == "create" and len(ids) < 8:
            t.want[t.numbers("create")[0]] = []
        elif what == "fork" and ids and len(ids) < 12:
            i = int(rng.choice(ids))
            t.want[t.numbers("fork", i)[0]] = list(t.want[i])
        elif what == "append" and ids:
            some = [int(i) for i in rng.permutation(ids)[:rng.integers(1, len(ids) + 1)]]
            refused += not t.append(some, [int(rng.choice([0, 1, 1, 2, page, 3 * page + 1])) for _ in some])
        elif what == "truncate" and ids:
            i = int(rng.choice(ids))
            n = int(rng.integers(0, len(t.want[i]) + 1))
            assert t.ask("truncate", i, n) == ""
            del t.want[i][n:]
        elif what == "release" and len(ids) > 3:
            i = int(rng.choice(ids))
            assert t.ask("release", i) == ""
            del t.want[i]
        elif what == "compact":
            t.copies(t.numbers("compact"))
            _, rows = t.state()
            held = {p for _, row in rows.values() for p in row}
            assert held == set(range(len(held)))
        elif what == "shared" and ids:
            some = [int(i) for i in rng.permutation(ids)[:3]]
            before = [int(rng.integers(0, 3)) for _ in some]
            n = t.numbers("shared", *[w for pair in zip(some, before) for w in pair])[0]
            _, rows = t.state()
            most = max(0, min(rows[i][0] - b for i, b in zip(some, before)))
            same = 0
            while same < most and len({rows[i][1][same // page] for i in some}) == 1:
                same += 1
            assert n == same
        t.check()
    t.close()
    assert refused > 0 or pages >= 200


def test_a_fork_shares_until_it_writes(exe):
    t = Table(exe, 10, 4)
    a = t.numbers("create")[0]
    t.want[a] = []
    t.append([a], [10])                       # three pages, the last of two keys
    b, c = t.numbers("fork", a)[0], t.numbers("fork", a)[0]
    t.want[b], t.want[c] = list(t.want[a]), list(t.want[a])
    assert t.state()[0] == 7
    assert t.numbers("shared", a, 0, b, 0, c, 0) == [10]
    t.append([a, b, c], [1, 1, 1])            # two copies: the last one that writes keeps the page
    rows = t.check()
    assert t.state()[0] == 5 and [rows[i][1][:2] for i in (a, b, c)] == [rows[a][1][:2]] * 3
    assert t.numbers("shared", a, 1, b, 1, c, 1) == [8]
    t.append([a], [1])                        # its own page now: no copy
    assert t.state()[0] == 5
    t.check()
    t.close()


def test_refusals(exe):
    for args, why in ((("0", "4"), "0 pages"), (("4", "0"), "pages of 0 keys")):
        out = subprocess.run([exe, *args], input="", capture_output=True, text=True, timeout=10).stdout
        assert out.startswith("error: PageTable") and why in out
    t = Table(exe, 4, 4)
    a = t.numbers("create")[0]
    t.want[a] = []
    t.append([a], [5])
    before = t.state()
    for words, why in ((("append", a, -1), "-1 tokens"), (("append", a, 2 ** 31), "tokens"), (("append", a, 1, a, 1), "twice"), (("append", 7, 1), "no sequence 7"),
                       (("append", a, 12), "3 pages needed, 2 of 4 free"), (("truncate", a, 6), "length 6 of a sequence of 5"), (("truncate", a, -1), "length -1"),
                       (("truncate", 7, 0), "no sequence"), (("fork", 7), "no sequence"), (("release", 7), "no sequence"), (("shared", 7, 0), "no sequence")):
        got = t.ask(*words)
        assert got.startswith("error: PageTable") and why in got, (words, got)
        assert t.state() == before
    t.close()


@pytest.fixture(scope="module")
def host_check(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("bin") / "paged_cache_host_check")
    pkg = os.path.join(ROOT, "vkml-framework_amd")
    subprocess.run(["g++", "-std=c++20", "-O1", "-g", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover", "-I" + os.path.join(pkg, "include"),
                    "-I" + os.path.join(ROOT, "include"), "-I" + os.path.join(pkg, "src"), os.path.join(ROOT, "tests", "cpp", "paged_cache_host_check.cpp"),
                    *(os.path.join(pkg, "src", f) for f in ("pages.cpp", "page_table.cpp", "runtime.cpp")), "-o", out], check=True)
    return out


def test_a_cache_that_fails_changes_nothing(host_check):
    """vkml::PagedCache over a C ABI in host memory whose n-th call fails:
    every batch and compaction that throws leaves the lengths, the pages and
    the keys as they were."""
    r = subprocess.run([host_check], capture_output=True, text=True, timeout=100)
    print(r.stdout)
    assert r.returncode == 0, r.stdout + r.stderr
    assert sum(line.startswith("ok ") for line in r.stdout.split("\n")) == 6


@pytest.fixture(scope="module")
def exe_undo(tmp_path_factory):
    """The check program with two verbs more: "undo", and "append-undo", an
    append that is taken back where it succeeded."""
    d = tmp_path_factory.mktemp("bin")
    with open(os.path.join(ROOT, "tests", "cpp", "page_table_check.cpp")) as f:
        source = f.read()
    verb = 'if (verb == "compact")'
    assert source.count(verb) == 1
    more = ['if (verb == "append-undo") table.undo(ids, counts, table.append(ids, counts));', 'if (verb == "undo") table.undo(ids, counts, copies);', verb]
    (d / "undo.cpp").write_text(source.replace(verb, "\n                ".join(more)))
    out = str(d / "undo")
    subprocess.run(["g++", "-std=c++20", "-O1", "-Wall", "-Werror", "-I" + os.path.join(ROOT, "vkml-framework_amd", "include"), str(d / "undo.cpp"),
                    os.path.join(ROOT, "vkml-framework_amd", "src", "page_table.cpp"), "-o", out], check=True)
    return out


@pytest.mark.parametrize("seed", [0, 1, 2])
def test_an_append_taken_back_leaves_no_trace(exe_undo, seed):
    rng = np.random.default_rng(seed)
    t = Table(exe_undo, 30, 4)
    for _ in range(300):
        ids = list(t.want)
        what = rng.choice(["create", "fork", "append", "undo", "undo", "truncate", "release", "compact"])
        if what == "create" and len(ids) < 6:
            t.want[t.numbers("create")[0]] = []
        elif what == "fork" and ids and len(ids) < 9:
            i = int(rng.choice(ids))
            t.want[t.numbers("fork", i)[0]] = list(t.want[i])
        elif what in ("append", "undo") and ids:
            some = [int(i) for i in rng.permutation(ids)[:rng.integers(1, len(ids) + 1)]]
            counts = [int(rng.choice([0, 1, 1, 2, 4, 7])) for _ in some]
            if what == "append":
                t.append(some, counts)
            else:
                before = t.state()
                t.ask("append-undo", *[w for pair in zip(some, counts) for w in pair])
                assert t.state() == before
        elif what == "truncate" and ids:
            i = int(rng.choice(ids))
            n = int(rng.integers(0, len(t.want[i]) + 1))
            assert t.ask("truncate", i, n) == ""
            del t.want[i][n:]
        elif what == "release" and len(ids) > 3:
            i = int(rng.choice(ids))
            assert t.ask("release", i) == ""
            del t.want[i]
        elif what == "compact":
            t.copies(t.numbers("compact"))
        t.check()
    assert t.ask("undo", 99, 1).startswith("error: PageTable") and t.ask("undo", next(iter(t.want)), 10 ** 6).startswith("error: PageTable")
    t.check()
    t.close()


def test_shared_refuses_negative_counts(exe):
    """Keys past the end of a sequence's pages' used part are nobody's."""
    t = Table(exe, 8, 4)
    a = t.numbers("create")[0]
    t.want[a] = []
    t.append([a], [5])
    b = t.numbers("fork", a)[0]
    assert t.numbers("shared", a, 0, b, 0) == [5] and t.numbers("shared", a, 9, b, 0) == [0]
    for words in ((a, -1, b, -1), (a, 0, b, -3), (a, -2 ** 63, b, 0)):
        assert "error: PageTable::shared" in t.ask("shared", *words)
    t.close()


def test_a_table_without_memory_changes_nothing(tmp_path):
    exe = str(tmp_path / "page_table_memory_check")
    subprocess.run(["g++", "-std=c++20", "-O1", "-Wall", "-I" + os.path.join(ROOT, "vkml-framework_amd", "include"),
                    os.path.join(ROOT, "tests", "cpp", "page_table_memory_check.cpp"), os.path.join(ROOT, "vkml-framework_amd", "src", "page_table.cpp"), "-o", exe],
                   check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.startswith("ok: ")
