"""Performance cases of speculative decoding and of long chats over the paged
cache, through the C ABI (include/vkml_hip.h).

Each case is a dict of plain values; its "kind" says which operator it runs:

  tree    vkml_attend_pages_tree: attention of each sequence's tree of
          drafted tokens, a token seeing the sequence's earlier keys and its
          own ancestors; the sequences may share their first `shared` keys
  window  vkml_attend_pages_window: attention of a batch whose tokens see the
          last `window` keys and the first `sinks` ones
  sample  vkml_sample: a token for each row of logits by its own temperature,
          top_k, top_p and min_p, from a given random number
  keep    vkml_keep_drafts: the drafted tokens that the model's picks confirm,
          whose keys and values move to the end of their sequence

With `own` false `run` computes them in elementary torch operations in 32
bits (the weights of `sample`, whose sums decide whole numbers, in 64); with
`own` true it makes the framework's calls.
"""
import ctypes as C
import math
import os
import random
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16}
# (query heads, KV heads, head_dim) of the repository's tiny, 1B- and
# 7B-shaped configurations, and a grouping of eight.
HEADS = {"tiny": (4, 2, 64), "1b": (32, 8, 64), "7b": (32, 8, 128), "wide": (16, 2, 128)}
GOLDEN = 0.6180339887498949
LOWEST = float(np.finfo(np.float32).min)
# (temperature, top_k, top_p, min_p) as requests bring them, greedy ones among them
REQUESTS = [(0.7, 40, 0.9, 0.0), (1.0, 0, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (0.8, 0, 0.95, 0.0), (1.2, 0, 1.0, 0.05), (0.6, 50, 0.8, 0.02)]


def listed():
    return [
        # Two chats of a tiny f32 model with a handful of drafts each: launches are everything.
        {"name": "tree-tiny-2seq-f32", "kind": "tree", "heads": "tiny", "kv": "f32", "page": 16, "seqs": 2, "shared": 0, "own_lo": 9, "own_hi": 40, "nodes": 7, "softcap": 0.0},
        # One chat, a large tree of guesses checked in one step.
        {"name": "tree-7b-1seq-60nodes", "kind": "tree", "heads": "7b", "kv": "f16", "page": 64, "seqs": 1, "shared": 0, "own_lo": 8100, "own_hi": 8100, "nodes": 60, "softcap": 0.0},
        # Unrelated chats of very different lengths, each with its tree.
        {"name": "tree-1b-16seq-ragged", "kind": "tree", "heads": "1b", "kv": "f16", "page": 16, "seqs": 16, "shared": 0, "own_lo": 40, "own_hi": 4000, "nodes": 26, "softcap": 0.0},
        # Replies drafted side by side from one few-shot prompt: the largest tree step.
        {"name": "tree-7b-24seq-shared4k", "kind": "tree", "heads": "7b", "kv": "f16", "page": 64, "seqs": 24, "shared": 4100, "own_lo": 40, "own_hi": 1200, "nodes": 13, "softcap": 0.0},
        # Three short chats with a window not much longer than they are.
        {"name": "window-tiny-3seq-f32", "kind": "window", "heads": "tiny", "kv": "f32", "page": 16, "seqs": 3, "own_lo": 3, "own_hi": 90, "new": 1, "window": 32, "sinks": 3, "softcap": 0.0},
        # Chats that have outgrown their window, pages behind it given back.
        {"name": "window-7b-16chats", "kind": "window", "heads": "7b", "kv": "f16", "page": 64, "seqs": 16, "own_lo": 500, "own_hi": 30000, "new": 1, "window": 4096, "sinks": 4, "softcap": 0.0},
        # Chunks of long prompts beside a chat that decodes.
        {"name": "window-7b-3prompts", "kind": "window", "heads": "7b", "kv": "f16", "page": 32, "seqs": 3, "own_lo": 1400, "own_hi": 5000, "new": 1400, "window": 1024, "sinks": 4, "softcap": 0.0},
        # The next token of one chat.
        {"name": "sample-7b-1row", "kind": "sample", "rows": 1, "vocab": 32768},
        # A decode step of 40 requests with a large vocabulary.
        {"name": "sample-1b-40rows", "kind": "sample", "rows": 40, "vocab": 128256},
        # Every node of 32 trees of drafts: the picks that confirm them.
        {"name": "sample-7b-416rows", "kind": "sample", "rows": 416, "vocab": 32768},
        # One chat with a large tree, a few of its tokens right.
        {"name": "keep-1b-1seq", "kind": "keep", "heads": "1b", "kv": "f16", "page": 16, "layers": 16, "seqs": 1, "before": 5000, "nodes": 60, "kept": 6},
        # A step of 24 chats in every layer of a 7B-shaped model.
        {"name": "keep-7b-24seq", "kind": "keep", "heads": "7b", "kv": "f16", "page": 64, "layers": 32, "seqs": 24, "before": 30000, "nodes": 13, "kept": 6},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "window", "window", "sample", "sample", "keep"])
    heads, kv, page = rng.choice(["tiny", "1b", "7b", "7b", "wide"]), rng.choice(["f16", "f16", "f32"]), rng.choice([16, 32, 64, 128])
    if kind == "tree":
        nodes = _log(rng, 2, 100)
        seqs = _log(rng, 1, max(2, min(24, 300 // nodes)))
        lo = _log(rng, nodes, nodes + 300)
        return {"kind": kind, "heads": heads, "kv": kv, "page": page, "seqs": seqs, "shared": rng.choice([0, _log(rng, 3, 4000)]), "own_lo": lo, "own_hi": lo + _log(rng, 1, 1000),
                "nodes": nodes, "softcap": rng.choice([0.0, 0.0, 0.0, 30.0])}
    if kind == "window":
        prompts = rng.random() < 0.3
        new = _log(rng, 2, 500) if prompts else 1
        lo = _log(rng, new, new + 500)
        return {"kind": kind, "heads": heads, "kv": kv, "page": page, "seqs": _log(rng, 1, 4 if prompts else 16), "own_lo": lo, "own_hi": lo + _log(rng, 1, 2000 if prompts else 20000),
                "new": new, "window": _log(rng, 5, 600 if prompts else 5000), "sinks": rng.choice([0, 4, _log(rng, 1, 150)]), "softcap": rng.choice([0.0, 0.0, 0.0, 30.0])}
    if kind == "sample":
        vocab = rng.choice([1000, 4096, 32768, 128256, _log(rng, 300, 128256)])
        return {"kind": kind, "rows": _log(rng, 1, min(400, 5000000 // vocab)), "vocab": vocab}
    nodes = _log(rng, 3, 64)
    return {"kind": kind, "heads": heads, "kv": kv, "page": page, "layers": rng.randint(1, 16), "seqs": _log(rng, 1, 24), "before": _log(rng, 1, 60000), "nodes": nodes,
            "kept": rng.randint(2, max(2, min(12, nodes // 3)))}


# ---------------------------------------------------------------- inputs

class _Rng:
    """Tensors from a seed, on the GPU, one stream per tensor."""

    def __init__(self, seed):
        self.seed, self.index = seed, 0

    def _gen(self):
        self.index += 1
        g = torch.Generator(device=DEV)
        g.manual_seed(self.seed * 100003 + self.index)
        return g

    def normal(self, *shape, dtype=torch.float32):
        return torch.randn(shape, generator=self._gen(), device=DEV, dtype=dtype)

    def uniform(self, *shape, dtype=torch.float32):
        return torch.rand(shape, generator=self._gen(), device=DEV, dtype=dtype)

    def order(self, n):
        return torch.randperm(n, generator=self._gen(), device=DEV).to(torch.int32)


def _spread(i, lo, hi):
    """The i-th of numbers spread over lo..hi."""
    return lo + int((hi - lo) * ((i + 1) * GOLDEN % 1.0) + 0.5)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _starts(new):
    return [0] + np.cumsum(new).tolist()


def _batch(case):
    """Each sequence's own keys and its new tokens (the last of them)."""
    n = range(case["seqs"])
    if case["kind"] == "tree":
        new = [_spread(i, (case["nodes"] + 1) // 2, case["nodes"]) if case["seqs"] > 1 else case["nodes"] for i in n]
    else:
        # Among prompts every third sequence is a chat in its decode step.
        new = [1 if case["new"] == 1 or i % 3 == 1 else _spread(i, (case["new"] + 1) // 2, case["new"]) for i in n]
    return [max(new[i], _spread(3 * i, case["own_lo"], case["own_hi"])) for i in n], new


def _tree(rng, nodes):
    """Parents of a tree: each node after its own, most of them near."""
    return [-1] + [rng.randrange(max(0, i - 1 - nodes // 4), i) for i in range(1, nodes)]


def _pools(rng, shape, dtype):
    # keys as after a projection: some dims larger than others
    gain = 0.5 + 1.5 * rng.uniform(shape[-1])
    return rng.normal(*shape, dtype=dtype) * gain.to(dtype), rng.normal(*shape, dtype=dtype)


def _tree_inputs(case, seed):
    rng, host = _Rng(seed), random.Random(seed)
    H, KVH, hd = HEADS[case["heads"]]
    page, shared = case["page"], case["shared"] if case["seqs"] > 1 else 0
    owned, new = _batch(case)
    full = shared // page  # whole shared pages; the part-filled one is each sequence's own copy
    stride = -(-(shared + max(owned)) // page)
    count = [-(-(shared + o) // page) - full for o in owned]
    pages = full + sum(count) + 3
    ids = rng.order(pages)
    table = torch.full((case["seqs"], stride), -1, dtype=torch.int32, device=DEV)
    table[:, :full] = ids[:full]
    at = full
    for s, c in enumerate(count):
        table[s, full:full + c] = ids[at:at + c]
        at += c
    k, v = _pools(rng, (pages, KVH, page, hd), TYPES[case["kv"]])
    if shared % page:
        to = table[1:, full].long()
        k[to, :, :shared % page] = k[table[0, full].long(), :, :shared % page]
        v[to, :, :shared % page] = v[table[0, full].long(), :, :shared % page]
    q = rng.normal(sum(new), H, hd)
    parents = [_tree(host, n) for n in new]
    words = -(-max(new) // 32)
    seen = np.zeros((sum(new), words), np.uint32)
    at = 0
    for tree in parents:
        for i, p in enumerate(tree):
            if p >= 0:
                seen[at + i] = seen[at + p]
            seen[at + i, i // 32] |= np.uint32(1 << i % 32)
        at += len(tree)
    lengths = [shared + o for o in owned]
    return {"kind": "tree", "case": case, "shape": (H, KVH, hd), "q": q, "k": k, "v": v, "table": table, "lengths": _i32(lengths), "starts": _i32(_starts(new)),
            "group_starts": _i32([0, case["seqs"]]), "group_keys": _i32([shared]), "shared": shared, "own": owned, "new": new, "parents": parents,
            "seen": torch.from_numpy(seen.view(np.int32)).to(DEV), "scale": 1.0 / math.sqrt(hd)}


def _window_inputs(case, seed):
    rng = _Rng(seed)
    H, KVH, hd = HEADS[case["heads"]]
    page, W, sinks = case["page"], case["window"], case["sinks"]
    lengths, new = _batch(case)
    stride = -(-max(lengths) // page)
    # the pages that hold keys some token still sees; the others are given back
    held = [[p for p in range(-(-n // page)) if p * page < sinks or (p + 1) * page > n - m - W + 1] for n, m in zip(lengths, new)]
    pages = sum(map(len, held)) + 2
    ids = rng.order(pages)
    table = torch.full((case["seqs"], stride), -1, dtype=torch.int32, device=DEV)
    at = 0
    for s, h in enumerate(held):
        table[s, torch.tensor(h, device=DEV)] = ids[at:at + len(h)]
        at += len(h)
    k, v = _pools(rng, (pages, KVH, page, hd), TYPES[case["kv"]])
    return {"kind": "window", "case": case, "shape": (H, KVH, hd), "q": rng.normal(sum(new), H, hd), "k": k, "v": v, "table": table, "lengths": _i32(lengths),
            "starts": _i32(_starts(new)), "own": lengths, "new": new, "scale": 1.0 / math.sqrt(hd)}


def _sample_inputs(case, seed):
    """Logits of a few likely tokens above many unlikely ones; every second row
    as a 16-bit model leaves them, with ties; some rows with tokens that must
    not come (masked by -inf, or by the type's lowest value)."""
    rng, rows, vocab = _Rng(seed), case["rows"], case["vocab"]
    x = 1.7 * rng.normal(rows, vocab)
    likely = (rng.uniform(rows, 64) * vocab).long().clamp(max=vocab - 1)
    x.scatter_add_(1, likely, 12.0 * rng.uniform(rows, 64) ** 2)
    x[1::2] = torch.round(x[1::2] * 32) / 32
    banned = (rng.uniform(rows, 16) * vocab).long().clamp(max=vocab - 1)
    x[0::3] = x[0::3].scatter(1, banned[0::3], -math.inf)
    x[1::3] = x[1::3].scatter(1, banned[1::3], LOWEST)
    asked = [REQUESTS[i % len(REQUESTS)] for i in range(rows)]
    options = np.zeros((rows, 4), np.float32)
    options[:, [0, 2, 3]] = np.array([(t, p, m) for t, _, p, m in asked], np.float32)
    options.view(np.int32)[:, 1] = [k for _, k, _, _ in asked]
    return {"kind": "sample", "case": case, "logits": x, "options": torch.from_numpy(options).to(DEV), "random": rng.uniform(rows, dtype=torch.float64),
            "tokens": torch.zeros(rows, dtype=torch.int32, device=DEV)}


def _kept(case):
    """Each sequence's nodes, how many of them are confirmed, and its keys."""
    n = range(case["seqs"])
    nodes = [case["nodes"] - i % 2 if case["nodes"] > 4 else case["nodes"] for i in n]
    return nodes, [min(_spread(i, 1, case["kept"]), (nodes[i] + 1) // 2) for i in n], [_spread(2 * i, case["before"] // 2, case["before"]) for i in n]


def _keep_inputs(case, seed):
    """Trees of drafts with distinct tokens, and picks that confirm a path of
    them. (The path's later nodes stand behind the rows that it moves to, so a
    pass leaves rows that another one finds and moves alike.)"""
    rng, host = _Rng(seed), random.Random(seed)
    _, KVH, hd = HEADS[case["heads"]]
    page = case["page"]
    nodes, kept, before = _kept(case)
    lengths = [n + b for n, b in zip(nodes, before)]
    stride = -(-max(lengths) // page)
    first = [b // page for b in before]
    count = [-(-n // page) - f for n, f in zip(lengths, first)]
    pages = sum(count) + 2
    ids = rng.order(pages)
    table = torch.full((case["seqs"], stride), -1, dtype=torch.int32, device=DEV)
    parents, drafted, picked, at = [], [], [], 0
    for s, (n, m) in enumerate(zip(nodes, kept)):
        table[s, first[s]:first[s] + count[s]] = ids[at:at + count[s]]
        at += count[s]
        path = [0] + sorted(host.sample(range(m, n), m - 1))
        tree = _tree(host, n)
        for a, b in zip(path, path[1:]):
            tree[b] = a
        tokens = host.sample(range(1000), n)
        picks = [host.randrange(1000, 2000) for _ in range(n)]
        for a, b in zip(path, path[1:]):
            picks[a] = tokens[b]
        parents += tree
        drafted += tokens
        picked += picks
    shape = (case["layers"], pages, KVH, page, hd)
    dtype = TYPES[case["kv"]]
    total = sum(nodes)
    return {"kind": "keep", "case": case, "k": rng.normal(*shape, dtype=dtype), "v": rng.normal(*shape, dtype=dtype), "table": table, "lengths": _i32(lengths),
            "starts": _i32(_starts(nodes)), "parents": _i32(parents), "drafted": _i32(drafted), "picked": _i32(picked), "most": max(nodes),
            "path": torch.zeros(total, dtype=torch.int32, device=DEV), "counts": torch.zeros(len(nodes), dtype=torch.int32, device=DEV),
            "next": torch.zeros(len(nodes), dtype=torch.int32, device=DEV)}


INPUTS = {"tree": _tree_inputs, "window": _window_inputs, "sample": _sample_inputs, "keep": _keep_inputs}


def prepare(case, seed):
    state = INPUTS[case["kind"]](case, seed)
    if own:
        _bind(state)
    return state


# ---------------------------------------------------------------- the framework's calls

def _ptr(t):
    return C.c_void_p(t.data_ptr())


def _workspace(nbytes):
    return torch.zeros(max(int(nbytes), 16) // 4, device=DEV)


def _bind(state):
    """The call's parameters, its output and its workspace, as a serving
    program keeps them from one step to the next."""
    path = os.path.join(os.getcwd(), "vkml-framework_amd", "python")
    if path not in sys.path:
        sys.path.insert(0, path)
    from vkml_amd import hip as H
    H.init()
    state["H"], case = H, state["case"]
    if state["kind"] == "sample":
        state["params"] = H.SampleParams(rows=case["rows"], vocab=case["vocab"], row_stride=case["vocab"])
        state["workspace"] = _workspace(H.lib().vkml_sample_workspace_bytes(C.byref(state["params"])))
        return
    _, kv_heads, hd = HEADS[case["heads"]]
    common = dict(kv_heads=kv_heads, head_dim=hd, kv_type={"f32": H.F32, "f16": H.F16}[case["kv"]], page_size=case["page"], pages=state["k"].shape[-4], seqs=case["seqs"],
                  table_stride=state["table"].shape[1])
    if state["kind"] == "keep":
        state["params"] = H.KeepDraftsParams(layers=case["layers"], tokens=state["parents"].shape[0], **common)
        return
    state["params"] = H.AttendPagesParams(heads=state["shape"][0], tokens=state["q"].shape[0], groups=1 if state["kind"] == "tree" else 0, scale=state["scale"],
                                          softcap=case["softcap"], **common)
    state["out"] = torch.zeros_like(state["q"])
    state["workspace"] = _workspace(H.lib().vkml_attend_pages_workspace_bytes(C.byref(state["params"])))


def _run_own(s):
    H, p = s["H"], C.byref(s["params"])
    if s["kind"] == "tree":
        H.call("vkml_attend_pages_tree", p, s["seen"].shape[1], _ptr(s["q"]), _ptr(s["k"]), _ptr(s["v"]), _ptr(s["table"]), _ptr(s["lengths"]), _ptr(s["starts"]),
               _ptr(s["group_starts"]), _ptr(s["group_keys"]), _ptr(s["seen"]), _ptr(s["workspace"]), _ptr(s["out"]))
        return s["out"]
    if s["kind"] == "window":
        starts = _ptr(s["starts"]) if max(s["new"]) > 1 else None  # NULL: a token a sequence
        H.call("vkml_attend_pages_window", p, s["case"]["window"], s["case"]["sinks"], _ptr(s["q"]), _ptr(s["k"]), _ptr(s["v"]), _ptr(s["table"]), _ptr(s["lengths"]), starts,
               _ptr(s["workspace"]), _ptr(s["out"]))
        return s["out"]
    if s["kind"] == "sample":
        H.call("vkml_sample", p, _ptr(s["logits"]), _ptr(s["options"]), _ptr(s["random"]), _ptr(s["workspace"]), _ptr(s["tokens"]))
        return s["tokens"]
    H.call("vkml_keep_drafts", p, _ptr(s["parents"]), _ptr(s["drafted"]), _ptr(s["picked"]), _ptr(s["table"]), _ptr(s["lengths"]), _ptr(s["starts"]), _ptr(s["path"]),
           _ptr(s["counts"]), _ptr(s["next"]), _ptr(s["k"]), _ptr(s["v"]))
    return {"path": s["path"], "counts": s["counts"], "next": s["next"], "k": s["k"], "v": s["v"]}


# ---------------------------------------------------------------- plain forms

def _softcapped(x, cap):
    return cap * torch.tanh(x / cap) if cap else x


def _padded(s, most):
    """Queries by sequence, padded to the longest one's: [KVH, S, most * G, hd]."""
    H, KVH, hd = s["shape"]
    starts = s["starts"].long()
    at = (starts[:-1, None] + torch.arange(most, device=DEV)).clamp(max=s["q"].shape[0] - 1)
    return s["q"][at].view(-1, most, KVH, H // KVH, hd).permute(2, 0, 1, 3, 4).reshape(KVH, at.shape[0], -1, hd)


def _unpadded(s, o, most):
    """[KVH, S, most * G, hd] back to the tokens' [tokens, H, hd]."""
    H, KVH, hd = s["shape"]
    starts = s["starts"].long()
    t = torch.arange(s["q"].shape[0], device=DEV)
    seq = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    return o.view(KVH, starts.shape[0] - 1, most, H // KVH, hd)[:, seq, t - starts[seq]].permute(1, 0, 2, 3).reshape(-1, H, hd)


def _held(s, pos):
    """K and V of each sequence's positions pos [S, n] (any that the table holds): [KVH, S, hd, n] and [KVH, S, n, hd]."""
    page = s["case"]["page"]
    table = s["table"].long()
    ids = table.gather(1, (pos // page).clamp(0, table.shape[1] - 1)).clamp(min=0)
    k, v = s["k"][ids, :, pos % page].float(), s["v"][ids, :, pos % page].float()
    return k.permute(2, 0, 3, 1).contiguous(), v.permute(2, 0, 1, 3).contiguous()


def _plain_tree(s):
    H, KVH, hd = s["shape"]
    G, page, shared, cap = H // KVH, s["case"]["page"], s["shared"], s["case"]["softcap"]
    S, most, most_own = len(s["own"]), max(s["new"]), max(s["own"])
    starts, lengths = s["starts"].long(), s["lengths"].long()
    new = starts[1:] - starts[:-1]
    q = _padded(s, most)
    # the keys that all share, once
    at = torch.arange(shared, device=DEV)
    table = s["table"].long()
    ks = s["k"][table[0, at // page], :, at % page].float().permute(1, 2, 0).contiguous()
    vs = s["v"][table[0, at // page], :, at % page].float().transpose(0, 1).contiguous()
    x1 = _softcapped(torch.matmul(q.reshape(KVH, S * most * G, hd), ks).view(KVH, S, most * G, shared) * s["scale"], cap)
    # each sequence's own: [KVH, S, own, hd]
    pos = (shared + torch.arange(most_own, device=DEV)).expand(S, -1)
    ko, vo = _held(s, pos)
    x2 = _softcapped(torch.matmul(q, ko) * s["scale"], cap)
    # a token sees what came before its sequence's new ones, and its bits' among those
    bits = (s["seen"][(starts[:-1, None] + torch.arange(most, device=DEV)).clamp(max=s["q"].shape[0] - 1)].long()[..., None] >> torch.arange(32, device=DEV)) & 1
    index = pos - (lengths - new)[:, None]  # [S, own]
    among = bits.flatten(2).gather(2, index.clamp(0, 32 * bits.shape[2] - 1)[:, None].expand(-1, most, -1)).bool()
    seen = (index < 0)[:, None] | (among & (index < new[:, None])[:, None])
    x2 = x2.masked_fill(~seen.repeat_interleave(G, 1), -math.inf)
    m = x2.amax(-1, keepdim=True)
    if shared:
        m = torch.maximum(m, x1.amax(-1, keepdim=True))
    m = m.clamp(min=LOWEST)  # rows of the padding see nothing
    p1, p2 = torch.exp(x1 - m), torch.exp(x2 - m)
    o = torch.matmul(p2, vo) + torch.matmul(p1.view(KVH, S * most * G, shared), vs).view(KVH, S, most * G, hd)
    return _unpadded(s, o / (p1.sum(-1, keepdim=True) + p2.sum(-1, keepdim=True)), most)


def _plain_window(s):
    H, KVH, hd = s["shape"]
    G, W, sinks, cap = H // KVH, s["case"]["window"], s["case"]["sinks"], s["case"]["softcap"]
    S, most = len(s["own"]), max(s["new"])
    starts, lengths = s["starts"].long(), s["lengths"].long()
    first = lengths - (starts[1:] - starts[:-1])  # the first new token's position
    q = _padded(s, most)
    # the sinks, then the keys from the first token's window on
    sink = torch.arange(sinks, device=DEV).expand(S, -1)
    late = first[:, None] - W + 1 + torch.arange(W + most - 1, device=DEV)
    pos = torch.cat([sink, late], 1)
    k, v = _held(s, pos.clamp(min=0))
    at = (first[:, None] + torch.arange(most, device=DEV))[..., None]  # [S, most, 1]
    seen = torch.cat([(sink[:, None] <= at), (late[:, None] >= sinks) & (late[:, None] <= at) & (late[:, None] > at - W)], -1)
    x = _softcapped(torch.matmul(q, k) * s["scale"], cap).masked_fill(~seen.repeat_interleave(G, 1), -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=LOWEST))
    return _unpadded(s, torch.matmul(p, v) / p.sum(-1, keepdim=True), most)


def _plain_sample(s):
    t, k, top_p, min_p = s["options"][:, 0], s["options"].view(torch.int32)[:, 1], s["options"][:, 2], s["options"][:, 3]
    x, ids = torch.sort(s["logits"], dim=1, descending=True, stable=True)
    heat = torch.where(t > 0, t, torch.ones_like(t)).double()[:, None]
    w = torch.exp((x.double() - x[:, :1].double()) / heat)
    rank = torch.arange(x.shape[1], device=DEV)
    w = w * ((k[:, None] == 0) | (rank < k[:, None]))
    mass = w.cumsum(1)
    w = w * ((rank == 0) | (mass - w < top_p.double()[:, None] * mass[:, -1:]))
    w = w * ((rank == 0) | (w >= min_p.double()[:, None] * w[:, :1]))
    mass = w.cumsum(1)
    kept = (w > 0).sum(1, keepdim=True)
    at = torch.minimum((mass <= s["random"][:, None] * mass[:, -1:]).sum(1, keepdim=True), kept - 1)
    at = torch.where(t[:, None] > 0, at, torch.zeros_like(at))
    s["tokens"].copy_(ids.gather(1, at)[:, 0])
    return s["tokens"]


def _plain_keep(s):
    page = s["case"]["page"]
    starts, lengths, most = s["starts"].long(), s["lengths"].long(), s["most"]
    S, total = lengths.shape[0], s["parents"].shape[0]
    new = starts[1:] - starts[:-1]
    t = torch.arange(total, device=DEV)
    seq = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    index = t - starts[seq]
    # a node is right where its parent's pick is its token; confirmed, where all before it on its way are
    parent = starts[seq] + s["parents"].long().clamp(min=0)
    right = (s["parents"] >= 0) & (s["picked"][parent] == s["drafted"]) | (index == 0)
    up = torch.zeros(S, most, most, device=DEV)
    up[seq, index, index] = 1
    up[seq, index, s["parents"].long().clamp(min=0)] = 1
    reach = up
    for _ in range(max(1, (most - 1).bit_length())):
        reach = (torch.matmul(reach, reach) > 0).float()
    wrong = torch.zeros(S, most, device=DEV)
    wrong[seq, index] = (~right).float()
    confirmed = (torch.matmul(reach, wrong[..., None])[..., 0] == 0)[seq, index]
    s["counts"].copy_(torch.zeros(S, dtype=torch.int32, device=DEV).index_add_(0, seq, confirmed.int()))
    place = torch.cumsum(confirmed.int(), 0) - confirmed.int()
    place = place - place[starts[seq]]
    s["path"].fill_(-1)
    keep = torch.nonzero(confirmed)[:, 0]
    s["path"][starts[seq[keep]] + place[keep]] = index[keep].int()
    last = s["path"].long()[starts[:-1] + s["counts"].long() - 1]
    s["next"].copy_(s["picked"][starts[:-1] + last])
    table = s["table"].long()
    base = (lengths - new)[seq[keep]]
    src, dst = base + index[keep], base + place[keep]
    a, b = table[seq[keep], src // page], table[seq[keep], dst // page]
    s["k"][:, b, :, dst % page] = s["k"][:, a, :, src % page]
    s["v"][:, b, :, dst % page] = s["v"][:, a, :, src % page]
    return {"path": s["path"], "counts": s["counts"], "next": s["next"], "k": s["k"], "v": s["v"]}


PLAIN = {"tree": _plain_tree, "window": _plain_window, "sample": _plain_sample, "keep": _plain_keep}


def run(state):
    if own:
        return _run_own(state)
    return PLAIN[state["kind"]](state)


# ---------------------------------------------------------------- work

def work(case):
    if case["kind"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + 28 * case["rows"], "flops": 4 * n}
    H, KVH, hd = HEADS[case["heads"]]
    size = 2 if case["kv"] == "f16" else 4
    if case["kind"] == "keep":
        nodes, kept, _ = _kept(case)
        return {"bytes": 2 * 2 * case["layers"] * sum(m - 1 for m in kept) * KVH * hd * size + 16 * sum(nodes), "flops": 0}
    total, new = _batch(case)
    tokens = sum(new)
    if case["kind"] == "tree":
        # a node sees its ancestors, half of the nodes before it at the most
        shared = case["shared"] if case["seqs"] > 1 else 0
        seen = sum(n * (shared + o - n) + n for o, n in zip(total, new))
        keys = shared + sum(total)
    else:
        W, sinks = case["window"], case["sinks"]
        seen = sum(sum(min(o - n + i + 1, W + min(sinks, max(0, o - n + i + 1 - W))) for i in range(n)) for o, n in zip(total, new))
        keys = sum(min(o, W + n - 1 + min(sinks, max(0, o - n + 1 - W))) for o, n in zip(total, new))
    return {"bytes": 2 * tokens * H * hd * 4 + 2 * keys * KVH * hd * size, "flops": 4 * H * hd * seen}


# ---------------------------------------------------------------- 64 bits

def _attend_64(s, hidden_of):
    """Softmax attention of each sequence over its keys through its own table,
    in 64 bits; hidden_of(sequence, keys): what its tokens [n, keys] don't see."""
    H, KVH, hd = s["shape"]
    page, cap, out, t = s["case"]["page"], s["case"]["softcap"], [], 0
    for b, n in enumerate(s["new"]):
        keys = int(s["lengths"][b])
        pages = s["table"][b, :-(-keys // page)].long()
        gone = (pages < 0)[:, None, None, None]
        k = s["k"][pages.clamp(min=0)].double().masked_fill(gone, 0).transpose(0, 1).reshape(KVH, -1, hd)[:, :keys]
        v = s["v"][pages.clamp(min=0)].double().masked_fill(gone, 0).transpose(0, 1).reshape(KVH, -1, hd)[:, :keys]
        q = s["q"][t:t + n].double().view(n, KVH, H // KVH, hd)
        hidden = hidden_of(b, keys)
        rows = []
        for h in range(KVH):
            x = (q[:, h].reshape(-1, hd) @ k[h].t().contiguous()).view(n, -1, keys) * s["scale"]
            if cap:
                x = cap * torch.tanh(x / cap)
            w = torch.softmax(x.masked_fill(hidden[:, None], -math.inf), -1)
            rows.append((w.view(-1, keys) @ v[h]).view(n, -1, hd))
        out.append(torch.cat(rows, 1))
        t += n
    return torch.cat(out)


def _exact_tree(s):
    def hidden(b, keys):
        n = s["new"][b]
        h = np.zeros((n, keys), bool)
        h[:, keys - n:] = True
        for i in range(n):
            at = i
            while at >= 0:
                h[i, keys - n + at] = False
                at = s["parents"][b][at]
        return torch.from_numpy(h).to(DEV)
    return _attend_64(s, hidden)


def _exact_window(s):
    def hidden(b, keys):
        key, at = torch.arange(keys, device=DEV)[None], torch.arange(keys - s["new"][b], keys, device=DEV)[:, None]
        return (key > at) | ((key <= at - s["case"]["window"]) & (key >= s["case"]["sinks"]))
    return _attend_64(s, hidden)


def _exact_sample(s):
    """A request at a time, candidate by candidate in the order of their
    logits (equal ones by index), in 64 bits on the host."""
    out = []
    logits, u = s["logits"].cpu().numpy(), s["random"].cpu().numpy()
    options = s["options"].cpu().numpy()
    top_ks = options.view(np.int32)[:, 1]
    for row, r, (t, _, top_p, min_p), top_k in zip(logits, u, options, top_ks):
        ranked = np.lexsort((np.arange(row.size), -row))
        if t == 0:
            out.append(int(ranked[0]))
            continue
        w = np.exp((row[ranked].astype(np.float64) - float(row[ranked[0]])) / float(t))
        if top_k:
            w = w[:top_k]
        if top_p < 1:
            w = w[:max(1, int(np.searchsorted(np.cumsum(w), float(top_p) * w.sum(), side="left")) + 1)]
        if min_p > 0:
            w = w[:max(1, int((w >= float(min_p) * w[0]).sum()))]
        sums = np.cumsum(w)
        out.append(int(ranked[min(int(np.searchsorted(sums, r * sums[-1], side="right")), w.size - 1)]))
    return torch.tensor(out, dtype=torch.int32)


def _exact_keep(s):
    """Node by node on the host; rows as they are, moved."""
    page = s["case"]["page"]
    starts, lengths, table = s["starts"].tolist(), s["lengths"].tolist(), s["table"].tolist()
    parents, drafted, picked = s["parents"].tolist(), s["drafted"].tolist(), s["picked"].tolist()
    k, v = s["k"].clone(), s["v"].clone()
    paths, counts, nexts = [-1] * len(parents), [], []
    for b, (lo, hi) in enumerate(zip(starts, starts[1:])):
        path = [0]
        while True:
            after = [i for i in range(hi - lo) if parents[lo + i] == path[-1] and drafted[lo + i] == picked[lo + path[-1]]]
            if not after:
                break
            path.append(after[0])
        paths[lo:lo + len(path)] = path
        counts.append(len(path))
        nexts.append(picked[lo + path[-1]])
        base = lengths[b] - (hi - lo)
        for j, i in enumerate(path):
            (p, r), (o, w) = divmod(base + i, page), divmod(base + j, page)
            k[:, table[b][o], :, w] = s["k"][:, table[b][p], :, r]
            v[:, table[b][o], :, w] = s["v"][:, table[b][p], :, r]
    return {"path": _i32(paths), "counts": _i32(counts), "next": _i32(nexts), "k": k, "v": v}


EXACT = {"tree": _exact_tree, "window": _exact_window, "sample": _exact_sample, "keep": _exact_keep}


def exact(case, seed):
    return EXACT[case["kind"]](INPUTS[case["kind"]](case, seed))
