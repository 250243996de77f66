"""Performance cases of the paged-cache operators: several sequences decoded
at once over one cache of pages, through the C ABI (include/vkml_hip.h).

Each case is a dict of plain values; its "kind" says which operator it runs:

  attend  vkml_attend_pages: attention of a batch whose sequences share the
          first `shared` keys and have own ones after them, `new` tokens of
          them in this call (1: a decode step)
  rope    vkml_rope_kv_pages: rotary positions of a batch's new queries and
          keys, with the keys and values appended to the sequences' pages
  copy    vkml_copy_pages: pages copied in every layer of the cache, as a
          fork or a compaction asks for

With `own` false `run` computes them in elementary torch operations in 32
bits; with `own` true it makes the framework's calls.
"""
import ctypes as C
import math
import os
import sys

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16}
# (query heads, KV heads, head_dim) of the repository's tiny, 1B- and
# 7B-shaped configurations, and a grouping of eight.
HEADS = {"tiny": (4, 2, 64), "1b": (32, 8, 64), "7b": (32, 8, 128), "wide": (16, 2, 128)}
GOLDEN = 0.6180339887498949


def listed():
    return [
        # Three short chats on a tiny f32 model: launches are everything.
        {"name": "attend-tiny-3seq", "kind": "attend", "heads": "tiny", "kv": "f32", "page": 16, "seqs": 3, "shared": 0, "own_lo": 5, "own_hi": 40, "new": 1, "softcap": 0.0},
        # Unrelated chats of very different lengths in one decode step.
        {"name": "attend-1b-16seq-ragged", "kind": "attend", "heads": "1b", "kv": "f16", "page": 16, "seqs": 16, "shared": 0, "own_lo": 30, "own_hi": 4000, "new": 1, "softcap": 0.0},
        # Replies sampled side by side from one few-shot prompt.
        {"name": "attend-7b-32seq-shared4k", "kind": "attend", "heads": "7b", "kv": "f16", "page": 64, "seqs": 32, "shared": 4100, "own_lo": 1, "own_hi": 400, "new": 1, "softcap": 0.0},
        # Many questions to one long document: the largest decode step.
        {"name": "attend-7b-64seq-shared32k", "kind": "attend", "heads": "7b", "kv": "f16", "page": 128, "seqs": 64, "shared": 32768, "own_lo": 100, "own_hi": 2000, "new": 1, "softcap": 0.0},
        # A system prompt, then chunks of new prompts beside decoding chats.
        {"name": "attend-7b-6seq-prompts", "kind": "attend", "heads": "7b", "kv": "f16", "page": 32, "seqs": 6, "shared": 1000, "own_lo": 700, "own_hi": 900, "new": 700, "softcap": 0.0},
        # The default f32 cache: best-of-8 after a 2000-token prompt.
        {"name": "attend-1b-8seq-f32", "kind": "attend", "heads": "1b", "kv": "f32", "page": 64, "seqs": 8, "shared": 2000, "own_lo": 10, "own_hi": 600, "new": 1, "softcap": 0.0},
        # One long chat alone, kept in pages.
        {"name": "attend-7b-1seq-32k", "kind": "attend", "heads": "7b", "kv": "f16", "page": 64, "seqs": 1, "shared": 0, "own_lo": 32768, "own_hi": 32768, "new": 1, "softcap": 0.0},
        # A decode step of 32 chats: one token each, far apart in position.
        {"name": "rope-7b-32tok", "kind": "rope", "heads": "7b", "kv": "f16", "page": 64, "seqs": 32, "new": 1, "before": 30000, "rotary": 128, "style": 0},
        # Ragged prompts, half of each head rotated in the split-half layout.
        {"name": "rope-1b-5prompts-half", "kind": "rope", "heads": "1b", "kv": "f32", "page": 16, "seqs": 5, "new": 901, "before": 777, "rotary": 32, "style": 1},
        # Long prompts of a 7B-shaped model.
        {"name": "rope-7b-8192tok", "kind": "rope", "heads": "7b", "kv": "f16", "page": 128, "seqs": 2, "new": 5461, "before": 100, "rotary": 128, "style": 0},
        # 31 forks of one chat: each copies the part-filled last page.
        {"name": "copy-7b-fork31", "kind": "copy", "heads": "7b", "kv": "f16", "page": 64, "layers": 32, "count": 31},
        # A pool of small pages compacted after chats have ended.
        {"name": "copy-1b-compact500", "kind": "copy", "heads": "1b", "kv": "f16", "page": 16, "layers": 16, "count": 500},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "rope", "copy"])
    heads, kv, page = rng.choice(["tiny", "1b", "7b", "7b", "wide"]), rng.choice(["f16", "f16", "f32"]), rng.choice([16, 32, 64, 128])
    if kind == "attend":
        prompts = rng.random() < 0.3
        new = _log(rng, 2, 400) if prompts else 1
        lo = _log(rng, new, new + 300)
        return {"kind": kind, "heads": heads, "kv": kv, "page": page, "seqs": _log(rng, 1, 4 if prompts else 48), "shared": rng.choice([0, _log(rng, 3, 1500 if prompts else 16000)]),
                "own_lo": lo, "own_hi": lo + _log(rng, 1, 600 if prompts else 1000), "new": new, "softcap": rng.choice([0.0, 0.0, 0.0, 30.0])}
    if kind == "rope":
        hd = HEADS[heads][2]
        return {"kind": kind, "heads": heads, "kv": kv, "page": page, "seqs": _log(rng, 1, 40), "new": rng.choice([1, _log(rng, 2, 300)]), "before": _log(rng, 1, 60000),
                "rotary": rng.choice([hd, hd, hd // 2, hd // 4, 2 * rng.randint(1, hd // 2)]), "style": rng.randint(0, 1)}
    _, kv_heads, hd = HEADS[heads]
    layers = rng.randint(1, 12)
    most = (400 << 20) // (layers * 4 * page * kv_heads * hd * (2 if kv == "f16" else 4))
    return {"kind": kind, "heads": heads, "kv": kv, "page": page, "layers": layers, "count": _log(rng, 1, min(300, most))}


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

    def order(self, n):
        return torch.randperm(n, generator=self._gen(), device=DEV).to(torch.int32)


def _spread(i, lo, hi):
    """The i-th of numbers spread over lo..hi."""
    return lo + int((hi - lo) * ((i + 1) * GOLDEN % 1.0) + 0.5)


def _batch(case):
    """Each sequence's own keys and its new tokens (the last of them)."""
    n = range(case["seqs"])
    if case["kind"] == "attend":
        # Among prompts every third sequence is a chat in its decode step.
        new = [1 if case["new"] == 1 or i % 3 == 1 else _spread(i, (case["new"] + 1) // 2, case["new"]) for i in n]
        return [max(new[i], _spread(3 * i, case["own_lo"], case["own_hi"])) for i in n], new
    new = [_spread(i, (case["new"] + 1) // 2, case["new"]) for i in n]
    return [_spread(2 * i, case["before"] // 2, case["before"]) + new[i] for i in n], new


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _starts(new):
    total, out = 0, [0]
    for n in new:
        total += n
        out.append(total)
    return out


def _attend_inputs(case, seed):
    rng = _Rng(seed)
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
    dtype = TYPES[case["kv"]]
    # keys as after a projection: some dims larger than others
    gain = 0.5 + 1.5 * torch.rand(hd, generator=rng._gen(), device=DEV)
    k = (rng.normal(pages, KVH, page, hd, dtype=dtype) * gain.to(dtype))
    v = rng.normal(pages, KVH, page, hd, dtype=dtype)
    part = shared % page
    if part:
        to = table[1:, full].long()
        for pool in (k, v):
            pool[to, :, :part] = pool[table[0, full].long(), :, :part]
    q = rng.normal(sum(new), H, hd)
    lengths, starts = [shared + o for o in owned], _starts(new)
    return {"kind": "attend", "case": case, "shape": (H, KVH, hd), "q": q, "k": k, "v": v, "table": table, "lengths": _i32(lengths), "starts": _i32(starts),
            "group_starts": _i32([0, case["seqs"]]), "group_keys": _i32([shared]), "shared": shared, "own": owned, "new": new, "scale": 1.0 / math.sqrt(hd)}


def _rope_inputs(case, seed):
    rng = _Rng(seed)
    H, KVH, hd = HEADS[case["heads"]]
    page, r = case["page"], case["rotary"]
    lengths, new = _batch(case)
    stride = -(-max(lengths) // page)
    first = [(n - m) // page for n, m in zip(lengths, new)]  # the page that the first new key goes to
    count = [-(-n // page) - f for n, f in zip(lengths, first)]
    pages = sum(count) + 2
    ids = rng.order(pages)
    table = torch.full((case["seqs"], stride), int(ids[-1]), dtype=torch.int32, device=DEV)
    at = 0
    for s, (f, c) in enumerate(zip(first, count)):
        table[s, f:f + c] = ids[at:at + c]
        at += c
    dtype = TYPES[case["kv"]]
    k, v = rng.normal(pages, KVH, page, hd, dtype=dtype), rng.normal(pages, KVH, page, hd, dtype=dtype)
    qkv = rng.normal(sum(new), (H + 2 * KVH) * hd)
    return {"kind": "rope", "case": case, "shape": (H, KVH, hd), "qkv": qkv, "k": k, "v": v, "q": torch.zeros(sum(new), H, hd, device=DEV), "table": table,
            "lengths": _i32(lengths), "starts": _i32(_starts(new)), "angles": _angles(max(lengths), r)}


def _angles(positions, r):
    """cos and sin of the positions, frequencies below one turn in 8192
    positions divided by 8 (a linear scaling of the low ones), in 64 bits."""
    inv = 500000.0 ** (-torch.arange(0, r, 2, device=DEV, dtype=torch.float64) / r)
    inv = torch.where(inv < 2 * math.pi / 8192, inv / 8, inv)
    a = torch.arange(positions, device=DEV, dtype=torch.float64)[:, None] * inv
    return torch.stack([a.cos(), a.sin()], -1).to(torch.float32).contiguous()


def _copy_inputs(case, seed):
    rng = _Rng(seed)
    _, KVH, hd = HEADS[case["heads"]]
    n, dtype = case["count"], TYPES[case["kv"]]
    pages = 2 * n + 5
    k, v = rng.normal(case["layers"], pages, KVH, case["page"], hd, dtype=dtype), rng.normal(case["layers"], pages, KVH, case["page"], hd, dtype=dtype)
    order = rng.order(pages)
    return {"kind": "copy", "case": case, "k": k, "v": v, "src": order[:n].contiguous(), "dst": order[n:2 * n].contiguous(), "pages": pages}


INPUTS = {"attend": _attend_inputs, "rope": _rope_inputs, "copy": _copy_inputs}


def prepare(case, seed):
    state = INPUTS[case["kind"]](case, seed)
    if own:
        _bind(state)
    return state


# ---------------------------------------------------------------- the framework's calls

def _ptr(t):
    return C.c_void_p(t.data_ptr())


def _bind(state):
    """The call's parameters, its output and its workspace, as a serving
    program keeps them from one step to the next."""
    path = os.path.join(os.getcwd(), "vkml-framework_amd", "python")
    if path not in sys.path:
        sys.path.insert(0, path)
    from vkml_amd import hip as H
    H.init()
    state["H"], case = H, state["case"]
    kind = {"f32": H.F32, "f16": H.F16}[case["kv"]]
    if state["kind"] == "copy":
        k = state["k"]
        page_bytes = k[0, 0].numel() * k.element_size()
        state["params"] = H.CopyPagesParams(pages=state["pages"], layers=case["layers"], count=case["count"], page_bytes=page_bytes)
        # the lists are the host's: a page table decides them
        state["src"], state["dst"] = state["src"].cpu(), state["dst"].cpu()
        return
    heads, kv_heads, hd = state["shape"]
    common = dict(heads=heads, kv_heads=kv_heads, head_dim=hd, kv_type=kind, page_size=case["page"], pages=state["k"].shape[0], seqs=case["seqs"],
                  table_stride=state["table"].shape[1])
    if state["kind"] == "attend":
        state["params"] = H.AttendPagesParams(tokens=state["q"].shape[0], groups=1, scale=state["scale"], softcap=case["softcap"], **common)
        state["out"] = torch.zeros_like(state["q"])
        need = int(H.lib().vkml_attend_pages_workspace_bytes(C.byref(state["params"])))
        state["workspace"] = torch.zeros(max(need, 4) // 4, device=DEV)
    else:
        state["params"] = H.RopeKvPagesParams(tokens=state["q"].shape[0], row_stride=state["qkv"].shape[1], rotary_dim=case["rotary"], style=case["style"],
                                              positions=state["angles"].shape[0], **common)


def _run_own(s):
    H, p = s["H"], C.byref(s["params"])
    if s["kind"] == "attend":
        starts = _ptr(s["starts"]) if max(s["new"]) > 1 else None  # NULL: a token a sequence
        H.call("vkml_attend_pages", p, _ptr(s["q"]), _ptr(s["k"]), _ptr(s["v"]), _ptr(s["table"]), _ptr(s["lengths"]), starts, _ptr(s["group_starts"]),
               _ptr(s["group_keys"]), _ptr(s["workspace"]), _ptr(s["out"]))
        return s["out"]
    if s["kind"] == "rope":
        H.call("vkml_rope_kv_pages", p, _ptr(s["qkv"]), _ptr(s["angles"]), _ptr(s["table"]), _ptr(s["lengths"]), _ptr(s["starts"]), None, _ptr(s["q"]), _ptr(s["k"]),
               _ptr(s["v"]))
        return {"q": s["q"], "k": s["k"], "v": s["v"]}
    H.call("vkml_copy_pages", p, _ptr(s["src"]), _ptr(s["dst"]), _ptr(s["k"]), _ptr(s["v"]))
    return {"k": s["k"], "v": s["v"]}


# ---------------------------------------------------------------- plain forms

def _tokens(s):
    """Each token's sequence, its index among that sequence's new ones, and its position."""
    starts, lengths = s["starts"].long(), s["lengths"].long()
    total = s["q"].shape[0]
    t = torch.arange(total, device=DEV)
    seq = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    index = t - starts[seq]
    return seq, index, lengths[seq] - (starts[seq + 1] - starts[seq]) + index


def _softcapped(x, cap):
    return cap * torch.tanh(x / cap) if cap else x


def _plain_attend(s):
    H, KVH, hd = s["shape"]
    G, page, shared, cap = H // KVH, s["case"]["page"], s["shared"], s["case"]["softcap"]
    S, most_new, most_own = len(s["own"]), max(s["new"]), max(s["own"])
    starts, lengths, table = s["starts"].long(), s["lengths"].long(), s["table"].long()
    new = starts[1:] - starts[:-1]
    # queries, padded to the longest sequence's: [KVH, S, new * G, hd]
    i = torch.arange(most_new, device=DEV)
    q = s["q"][(starts[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)].view(S, most_new, KVH, G, hd).permute(2, 0, 1, 3, 4).reshape(KVH, S, most_new * G, hd)
    # the keys that all share, once
    at = torch.arange(shared, device=DEV)
    ks = s["k"][table[0, at // page], :, at % page].float().permute(1, 2, 0).contiguous()
    vs = s["v"][table[0, at // page], :, at % page].float().transpose(0, 1).contiguous()
    x1 = _softcapped(torch.matmul(q.reshape(KVH, S * most_new * G, hd), ks).view(KVH, S, most_new * G, shared) * s["scale"], cap)
    # each sequence's own: [KVH, S, own, hd]
    pos = shared + torch.arange(most_own, device=DEV)
    ids = table[:, (pos // page).clamp(max=table.shape[1] - 1)].clamp(min=0)
    ko = s["k"][ids, :, pos % page].float().permute(2, 0, 3, 1).contiguous()
    vo = s["v"][ids, :, pos % page].float().permute(2, 0, 1, 3).contiguous()
    x2 = _softcapped(torch.matmul(q, ko) * s["scale"], cap)
    seen = pos <= (lengths - new)[:, None, None] + i[:, None]  # [S, new, own]
    x2 = x2.masked_fill(~seen.repeat_interleave(G, 1), -math.inf)
    m = x2.amax(-1, keepdim=True)
    if shared:
        m = torch.maximum(m, x1.amax(-1, keepdim=True))
    p1, p2 = torch.exp(x1 - m), torch.exp(x2 - m)
    o = torch.matmul(p2, vo) + torch.matmul(p1.view(KVH, S * most_new * G, shared), vs).view(KVH, S, most_new * G, hd)
    o = o / (p1.sum(-1, keepdim=True) + p2.sum(-1, keepdim=True))
    seq, index, _ = _tokens(s)
    return o.view(KVH, S, most_new, G, hd)[:, seq, index].permute(1, 0, 2, 3).reshape(-1, H, hd)


def _rotate(x, angles, style, r):
    """x [tokens, heads, hd], its first r dims turned by angles [tokens, r / 2, 2]."""
    c, d = angles[:, None, :, 0], angles[:, None, :, 1]
    head, rest = x[..., :r], x[..., r:]
    a, b = (head[..., 0::2], head[..., 1::2]) if style == 0 else (head[..., :r // 2], head[..., r // 2:])
    ra, rb = a * c - b * d, a * d + b * c
    turned = torch.stack([ra, rb], -1).flatten(-2) if style == 0 else torch.cat([ra, rb], -1)
    return torch.cat([turned, rest], -1)


def _plain_rope(s):
    H, KVH, hd = s["shape"]
    page, r, style = s["case"]["page"], s["case"]["rotary"], s["case"]["style"]
    seq, _, pos = _tokens(s)
    x = s["qkv"].view(-1, H + 2 * KVH, hd)
    turned = _rotate(x[:, :H + KVH], s["angles"][pos], style, r)
    s["q"].copy_(turned[:, :H])
    where = s["table"].long()[seq, pos // page]
    s["k"][where, :, pos % page] = turned[:, H:].to(s["k"].dtype)
    s["v"][where, :, pos % page] = x[:, H + KVH:].to(s["v"].dtype)
    return {"q": s["q"], "k": s["k"], "v": s["v"]}


def _plain_copy(s):
    src, dst = s["src"].long(), s["dst"].long()
    s["k"][:, dst] = s["k"][:, src]
    s["v"][:, dst] = s["v"][:, src]
    return {"k": s["k"], "v": s["v"]}


PLAIN = {"attend": _plain_attend, "rope": _plain_rope, "copy": _plain_copy}


def run(state):
    if own:
        return _run_own(state)
    return PLAIN[state["kind"]](state)


# ---------------------------------------------------------------- work

def work(case):
    H, KVH, hd = HEADS[case["heads"]]
    size = 2 if case["kv"] == "f16" else 4
    if case["kind"] == "copy":
        return {"bytes": 2 * 2 * case["layers"] * case["count"] * KVH * case["page"] * hd * size, "flops": 0}
    total, new = _batch(case)
    tokens = sum(new)
    if case["kind"] == "rope":
        positions = tokens * case["rotary"] * 4
        return {"bytes": tokens * ((2 * H + 2 * KVH) * hd * 4 + 2 * KVH * hd * size) + positions, "flops": tokens * (H + KVH) * case["rotary"] * 3}
    shared = case["shared"] if case["seqs"] > 1 else 0
    # token i of n sees the shared keys and all but the last n - 1 - i own ones
    seen = sum(n * (shared + o) - n * (n - 1) // 2 for o, n in zip(total, new))
    return {"bytes": 2 * tokens * H * hd * 4 + 2 * (shared + sum(total)) * KVH * hd * size, "flops": 4 * H * hd * seen}


# ---------------------------------------------------------------- 64 bits

def _exact_attend(s):
    """Softmax attention of each sequence over all its keys through its own
    table, in 64 bits."""
    H, KVH, hd = s["shape"]
    page, cap, out, t = s["case"]["page"], s["case"]["softcap"], [], 0
    for b, (o, n) in enumerate(zip(s["own"], s["new"])):
        keys = s["shared"] + o
        pages = s["table"][b, :-(-keys // page)].long()
        k = s["k"][pages].double().transpose(0, 1).reshape(KVH, -1, hd)[:, :keys]
        v = s["v"][pages].double().transpose(0, 1).reshape(KVH, -1, hd)[:, :keys]
        q = s["q"][t:t + n].double().view(n, KVH, H // KVH, hd)
        hidden = torch.arange(keys, device=DEV)[None, :] > keys - n + torch.arange(n, device=DEV)[:, None]
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


def _exact_rope(s):
    """The turn as a complex product, token by sequence, in 64 bits."""
    H, KVH, hd = s["shape"]
    page, r = s["case"]["page"], s["case"]["rotary"]
    angles = s["angles"].double()
    k, v, q = s["k"].double(), s["v"].double(), []
    lengths, starts, table = s["lengths"].tolist(), s["starts"].tolist(), s["table"].long()
    for b, n in enumerate(lengths):
        x = s["qkv"][starts[b]:starts[b + 1]].double().view(-1, H + 2 * KVH, hd)
        pos = torch.arange(n - x.shape[0], n, device=DEV)
        turn = torch.view_as_complex(angles[pos])[:, None]
        y = x.clone()
        if s["case"]["style"] == 0:
            z = torch.complex(x[..., 0:r:2], x[..., 1:r:2]) * turn
            y[..., 0:r:2], y[..., 1:r:2] = z.real, z.imag
        else:
            z = torch.complex(x[..., :r // 2], x[..., r // 2:r]) * turn
            y[..., :r // 2], y[..., r // 2:r] = z.real, z.imag
        q.append(y[:, :H])
        k[table[b, pos // page], :, pos % page] = y[:, H:H + KVH]
        v[table[b, pos // page], :, pos % page] = x[:, H + KVH:]
    return {"q": torch.cat(q), "k": k, "v": v}


def _exact_copy(s):
    k, v = s["k"].clone(), s["v"].clone()
    for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
        k[:, b] = s["k"][:, a]
        v[:, b] = s["v"][:, a]
    return {"k": k, "v": v}


EXACT = {"attend": _exact_attend, "rope": _exact_rope, "copy": _exact_copy}


def exact(case, seed):
    return EXACT[case["kind"]](INPUTS[case["kind"]](case, seed))
