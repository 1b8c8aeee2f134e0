"""The operators of a step of several drafted tokens, and of models that normalise queries and keys, as cases that can be timed one by one.

Six kinds of work:

  norm     grl_qk_norm_rope: every query and key head of a prompt normalised (root mean square, learned weight) and rotated, one call
  grad     grl_qk_norm_rope_backward: gradients of its inputs and weights
  append   grl_kv_append_norm: the same for new tokens, with their values, into the paged cache; a tree's tokens stand at their depth
  attend   grl_tree_attention: the nodes of a drafted tree over the cache; a node sees the prefix, its ancestors and itself
  keep     append of a drafted tree, then grl_kv_commit: the rows of the accepted path close up behind the prefix
  step     all of it: append, attend, commit, as a speculating server runs a step

Plain forms are elementary torch operations in float32 (angles in float64); the framework's calls go through its C ABI.
"""
import ctypes as C
import functools
import math
import os
import random
import sys

import numpy as np
import torch

own = False

EPS = 1e-6
THETA = 10000.0
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # The prompt batch of the benchmark, 4 x 2048 tokens with 32 query and 8 kv heads, out in the layout attention takes.
        {"name": "norm_prompt", "kind": "norm", "batch": 4, "seq": 2048, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128,
         "rope": "half", "scaled": False, "start": 0, "packed": False, "head_major": True, "dtype": "bf16"},
        # A short float32 call of a small model: half of the head rotated, inputs cut out of one packed projection; latency.
        {"name": "norm_small", "kind": "norm", "batch": 1, "seq": 37, "heads": 6, "kv_heads": 2, "dim": 64, "rotary": 32,
         "rope": "interleaved", "scaled": True, "start": 120011, "packed": True, "head_major": False, "dtype": "f32"},
        # The backward pass of a training batch.
        {"name": "grad_batch", "kind": "grad", "batch": 2, "seq": 2048, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128,
         "rope": "half", "scaled": False, "start": 0, "packed": False, "head_major": True, "dtype": "bf16"},
        # The backward pass of a small float32 model of an odd length, inputs and gradients packed.
        {"name": "grad_small", "kind": "grad", "batch": 3, "seq": 333, "heads": 12, "kv_heads": 12, "dim": 64, "rotary": 64,
         "rope": "interleaved", "scaled": False, "start": 0, "packed": True, "head_major": False, "dtype": "f32"},
        # The cache fill behind a prompt: 4 x 2048 tokens, keys and queries normalised and rotated on the way.
        {"name": "append_prompt", "kind": "append", "batch": 4, "new": 2048, "cached": 0, "kv_heads": 8, "group": 4, "dim": 128, "rotary": 128,
         "rope": "half", "scaled": False, "page": 64, "tree": False, "ragged": False, "dtype": "bf16"},
        # The append of a drafted tree of 12 nodes, 7 sequences of some 900 tokens: latency.
        {"name": "append_tree", "kind": "append", "batch": 7, "new": 12, "cached": 900, "kv_heads": 8, "group": 4, "dim": 128, "rotary": 64,
         "rope": "half", "scaled": True, "page": 16, "tree": True, "ragged": True, "dtype": "bf16"},
        # One user, a short run of drafted tokens (a chain) over about a thousand cached ones: latency.
        {"name": "attend_chain", "kind": "attend", "batch": 1, "nodes": 5, "kv_heads": 8, "group": 4, "dim": 128, "tokens": 1001, "page": 16,
         "tree": False, "ragged": False, "dtype": "bf16"},
        # The batch of the benchmark's decode step, 32 sequences of 4096 cached tokens, with a tree of 16 nodes each.
        {"name": "attend_batch", "kind": "attend", "batch": 32, "nodes": 16, "kv_heads": 8, "group": 4, "dim": 128, "tokens": 4096, "page": 64,
         "tree": True, "ragged": False, "dtype": "bf16"},
        # Long context: one sequence of 131072 tokens and a tree of 61 nodes.
        {"name": "attend_long", "kind": "attend", "batch": 1, "nodes": 61, "kv_heads": 8, "group": 4, "dim": 128, "tokens": 131072, "page": 64,
         "tree": True, "ragged": False, "dtype": "bf16"},
        # A float32 cache with an odd page size, ragged lengths and trees: the exact path of a small model.
        {"name": "attend_fp32", "kind": "attend", "batch": 5, "nodes": 11, "kv_heads": 2, "group": 3, "dim": 64, "tokens": 777, "page": 24,
         "tree": True, "ragged": True, "dtype": "f32"},
        # 32 sequences append a tree of 24 nodes and keep what was accepted.
        {"name": "keep_batch", "kind": "keep", "batch": 32, "new": 24, "cached": 1000, "kv_heads": 8, "group": 4, "dim": 128, "rotary": 128,
         "rope": "half", "scaled": False, "page": 64, "tree": True, "ragged": True, "dtype": "bf16"},
        # A whole step of a small server: 4 sequences of up to 1500 tokens, a tree of 31 nodes each.
        {"name": "step_server", "kind": "step", "batch": 4, "new": 31, "cached": 1500, "kv_heads": 8, "group": 4, "dim": 128, "rotary": 128,
         "rope": "half", "scaled": False, "page": 64, "tree": True, "ragged": True, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    kind = rng.choice(["norm", "norm", "grad", "grad", "append", "append", "attend", "attend", "attend", "attend", "keep", "step"])
    rope = rng.choice(["half", "interleaved"])
    if kind in ("norm", "grad"):
        most = listed()[0 if kind == "norm" else 2]
        while True:
            d = rng.choice([32, 64, 80, 128, 128, 256])
            hkv = rng.choice([1, 2, 4, 8])
            c = {"kind": kind, "batch": rng.randint(1, 4), "seq": _log(rng, 1, 4096), "heads": hkv * rng.choice([1, 2, 3, 4, 8]), "kv_heads": hkv,
                 "dim": d, "rotary": rng.choice([d, d, d // 2]), "rope": rope, "scaled": rng.random() < 0.4, "start": rng.choice([0, 0, 120011]),
                 "packed": rng.random() < 0.4, "head_major": rng.random() < 0.4, "dtype": rng.choice(["bf16", "bf16", "f32"])}
            if work(c)["bytes"] <= work(most)["bytes"]:
                return c
    if kind == "append":
        tree = rng.random() < 0.6
        while True:
            d = rng.choice([64, 128, 128])
            c = {"kind": kind, "batch": _log(rng, 1, 32), "new": _log(rng, 1, 128) if tree else _log(rng, 1, 2048), "cached": _log(rng, 1, 4096),
                 "kv_heads": rng.choice([2, 4, 8]), "group": rng.choice([1, 2, 3, 4, 8]), "dim": d, "rotary": rng.choice([d, d, d // 2]), "rope": rope,
                 "scaled": rng.random() < 0.4, "page": rng.choice([16, 24, 32, 64]), "tree": tree, "ragged": tree and rng.random() < 0.6,
                 "dtype": rng.choice(["bf16", "bf16", "f32"])}
            if work(c)["bytes"] <= work(listed()[4])["bytes"] and c["batch"] * (c["cached"] + c["new"]) * c["kv_heads"] * d <= 32 * 4096 * 8 * 128:
                return c
    if kind == "attend":
        while True:
            f32 = rng.random() < 0.25
            c = {"kind": kind, "batch": _log(rng, 1, 64), "nodes": _log(rng, 1, 128), "kv_heads": rng.choice([2, 4, 8]),
                 "group": rng.choice([1, 2, 3, 4, 8]), "dim": rng.choice([64, 128, 128]), "tokens": _log(rng, 32, 131072),
                 "page": rng.choice([16, 24, 32, 64]) if f32 else rng.choice([16, 32, 64, 64]), "tree": rng.random() < 0.7,
                 "ragged": rng.random() < 0.4, "dtype": "f32" if f32 else "bf16"}
            w = work(c)
            if w["bytes"] <= (0.05 if f32 else 1.0) * work(listed()[7])["bytes"] and w["flops"] <= (0.02 if f32 else 1.0) * work(listed()[8])["flops"]:
                return c
    while True:
        c = {"kind": kind, "batch": _log(rng, 1, 32), "new": _log(rng, 1, 64), "cached": _log(rng, 1, 4096), "kv_heads": rng.choice([2, 4, 8]),
             "group": rng.choice([1, 2, 3, 4, 8]), "dim": rng.choice([64, 128, 128]), "rope": rope, "scaled": rng.random() < 0.4,
             "page": rng.choice([16, 32, 64]), "tree": rng.random() < 0.8, "ragged": rng.random() < 0.6, "dtype": "bf16"}
        c["rotary"] = rng.choice([c["dim"], c["dim"], c["dim"] // 2])
        if c["batch"] * c["cached"] * c["kv_heads"] * c["dim"] <= 8 * 4096 * 8 * 128:
            return c


# ------------------------------------------------------------------------------ what a case fixes besides its sizes
def _rng(case, salt):
    return random.Random("%s %s" % (salt, sorted((k, v) for k, v in case.items() if k != "name")))


def _tokens(case):
    """Cached tokens of every sequence ahead of the step."""
    t = case["tokens"] if case["kind"] == "attend" else case["cached"]
    r = _rng(case, "tokens")
    return [r.randint(t // 2, t) if case["ragged"] else t for _ in range(case["batch"])]


def _width(case):
    return case["nodes"] if case["kind"] == "attend" else case["new"]


def _nodes(case):
    """New tokens of every sequence, at most the width of the step; a ragged batch has sequences that sat the step out."""
    n, r = _width(case), _rng(case, "nodes")
    return [(0 if i and r.random() < 0.1 else r.randint((n + 1) // 2, n)) if case["ragged"] else n for i in range(case["batch"])]


def _parents(case):
    """(batch, width) parents of drafted trees: node 0 hangs on the prefix, children follow their parents, depth about 8 at most."""
    r, rows = _rng(case, "parents"), []
    for _ in range(case["batch"]):
        row, depth = [-1], [0]
        for t in range(1, _width(case)):
            p = r.randrange(max(0, t - 8), t)
            while depth[p] >= 7:
                p = row[p]
            row.append(p)
            depth.append(depth[p] + 1)
        rows.append(row)
    return rows


def _paths(case, parents, nodes):
    """The accepted path of every sequence: some node and its ancestors, ascending."""
    r, paths = _rng(case, "paths"), []
    for row, n in zip(parents, nodes):
        path, t = [], (r.randrange(n) if n else -1)
        while t >= 0:
            path.append(t)
            t = row[t] if case["tree"] else t - 1
        paths.append(path[::-1])
    return paths


def _elem(case):
    return 4 if case["dtype"] == "f32" else 2


def work(case):
    k, e, d = case["kind"], _elem(case), case["dim"]
    if k in ("norm", "grad"):
        values = float(case["batch"] * case["seq"] * (case["heads"] + case["kv_heads"]) * d)
        return {"bytes": (2 if k == "norm" else 3) * values * e, "flops": (8 if k == "norm" else 20) * values}
    hkv, hq = case["kv_heads"], case["kv_heads"] * case["group"]
    lens, new = _tokens(case), _nodes(case)
    fresh = float(sum(new)) * (2 * hkv + hq) * d * e          # keys, values and queries of the new tokens
    attend = {"bytes": float(sum(n + m for n, m in zip(lens, new) if m)) * 2 * hkv * d * e + 2.0 * sum(new) * hq * d * e,
              "flops": 4.0 * d * hq * sum(m * (n + (m + 1) / 2) for n, m in zip(lens, new))}
    append = {"bytes": 2 * fresh, "flops": 8.0 * sum(new) * (hkv + hq) * d}
    if k == "append":
        return append
    if k == "attend":
        return attend
    kept = sum(len(p) for p in _paths(case, _parents(case), new))
    moved = 2.0 * kept * 2 * hkv * d * e
    if k == "keep":
        return {"bytes": append["bytes"] + moved, "flops": append["flops"]}
    return {"bytes": append["bytes"] + attend["bytes"] + moved, "flops": append["flops"] + attend["flops"]}


# ---------------------------------------------------------------------------------------------- preparation
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _freq(case):
    """Inverse frequencies of a model scaled for long contexts: the slow pairs by 8, the fast ones not, a ramp between; float32, as stored."""
    half = case["rotary"] // 2
    j = torch.arange(half, dtype=torch.float64)
    base = THETA ** (-2.0 * j / case["rotary"])
    ramp = ((j / max(1, half - 1) - 0.25) / 0.5).clamp(0, 1)
    return (base * (1 - ramp) + base / 8 * ramp).to(torch.float32).cuda()


def _weights(case, g):
    return [1 + 0.1 * torch.randn(case["dim"], generator=g, device="cuda") for _ in range(2)]


def _prepare_norm(case, seed):
    g, dt = _generator(seed), DTYPES[case["dtype"]]
    b, s, h, hk, d = case["batch"], case["seq"], case["heads"], case["kv_heads"], case["dim"]
    if case["packed"]:           # one projection's rows [q | k | v]
        rows = torch.randn((b, s, h + 2 * hk, d), generator=g, device="cuda").to(dt)
        q, k = rows[:, :, :h], rows[:, :, h:h + hk]
    else:
        q, k = (torch.randn((b, s, n, d), generator=g, device="cuda").to(dt) for n in (h, hk))
    wq, wk = _weights(case, g)

    def results():               # (B,S,H,D) in index order, in memory (B,H,S,D) where attention wants it so
        return [torch.empty((b, n, s, d), dtype=dt, device="cuda").transpose(1, 2) if case["head_major"]
                else torch.empty((b, s, n, d), dtype=dt, device="cuda") for n in (h, hk)]

    state = {"q": q, "k": k, "wq": wq, "wk": wk, "freq": _freq(case) if case["scaled"] else None, "y": results()}
    if case["kind"] == "grad":
        dy = results()
        for t in dy:
            t.normal_(generator=g)
        if case["packed"]:
            grads = torch.zeros((b, s, h + 2 * hk, d), dtype=dt, device="cuda")
            dq, dk = grads[:, :, :h], grads[:, :, h:h + hk]
        else:
            dq, dk = torch.empty_like(q), torch.empty_like(k)
        state.update(dy=dy, dx=[dq, dk], dw=[torch.empty_like(wq), torch.empty_like(wk)])
    return state


def _prepare_cache(case, seed):
    g, dt = _generator(seed), DTYPES[case["dtype"]]
    b, hkv, hq, d, t = case["batch"], case["kv_heads"], case["kv_heads"] * case["group"], case["dim"], _width(case)
    lens, new, parents = _tokens(case), _nodes(case), _parents(case)
    page, pages = case["page"], -(-(max(lens) + t) // case["page"])
    table = torch.randperm(pages * b, generator=g, device="cuda").to(torch.int32).reshape(b, pages).contiguous()
    make = torch.zeros if case["kind"] in ("append", "keep") else torch.empty
    pools = [make((pages * b, hkv, page, d), dtype=dt, device="cuda") for _ in range(2)]
    if case["kind"] not in ("append", "keep"):
        for p in pools:
            p.normal_(generator=g)
    before = torch.tensor(lens, dtype=torch.int32, device="cuda")
    count = torch.tensor(new, dtype=torch.int32, device="cuda")
    state = {"pools": pools, "table": table, "before": before, "after": before + count, "count": count, "most": max(lens) + t,
             "parents": torch.tensor(parents, dtype=torch.int32, device="cuda") if case["tree"] else None,
             "q": torch.randn((b, t, hq, d), generator=g, device="cuda").to(dt)}
    if case["kind"] != "append":
        state["out"] = torch.empty((b, t, hq, d), dtype=dt, device="cuda")
    if case["kind"] != "attend":
        state["k"], state["v"] = (torch.randn((b, t, hkv, d), generator=g, device="cuda").to(dt) for _ in range(2))
        state["wq"], state["wk"] = _weights(case, g)
        state["freq"] = _freq(case) if case["scaled"] else None
        state["q_out"] = torch.empty_like(state["q"])
    if case["kind"] in ("keep", "step"):
        paths = _paths(case, parents, new)
        most = max(1, max(len(p) for p in paths))
        state["path"] = torch.tensor([p + [0] * (most - len(p)) for p in paths], dtype=torch.int32, device="cuda")
        state["accepted"] = torch.tensor([len(p) for p in paths], dtype=torch.int32, device="cuda")
        state["kept"] = torch.zeros_like(before)
    return state


def prepare(case, seed):
    state = _prepare_norm(case, seed) if case["kind"] in ("norm", "grad") else _prepare_cache(case, seed)
    state["case"] = dict(case)
    return state


# ---------------------------------------------------------------------------------------------- plain forms
def _angles(case, pos, freq):
    """cos and sin of (B,S) positions x pairs, angles in float64."""
    f = freq.double() if freq is not None else THETA ** (-2.0 * torch.arange(case["rotary"] // 2, device="cuda", dtype=torch.float64) / case["rotary"])
    a = pos.double()[..., None] * f
    return a.cos().float()[:, :, None], a.sin().float()[:, :, None]


def _turn(case, x, c, s):
    """The rotation of the first `rotary` elements of (B,S,H,D), by (c, s); by (c, -s) it is undone."""
    r = case["rotary"]
    if case["rope"] == "half":
        a, b = x[..., :r // 2], x[..., r // 2:r]
        return torch.cat([a * c - b * s, a * s + b * c, x[..., r:]], -1)
    a, b = x[..., 0:r:2], x[..., 1:r:2]
    return torch.cat([torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2), x[..., r:]], -1)


def _norm_rope(case, x, w, c, s):
    x = x.float()
    return _turn(case, x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w, c, s)


def _positions(case):
    return (case["start"] + torch.arange(case["seq"], device="cuda")).expand(case["batch"], -1)


def _plain_norm(st):
    case = st["case"]
    c, s = _angles(case, _positions(case), st["freq"])
    st["y"][0].copy_(_norm_rope(case, st["q"], st["wq"], c, s))
    st["y"][1].copy_(_norm_rope(case, st["k"], st["wk"], c, s))
    return list(st["y"])


def _norm_rope_grad(case, x, w, dy, c, s):
    x, g = x.float(), _turn(case, dy.float(), c, -s)
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    dw = (g * (x * r)).double().sum((0, 1, 2)).float()
    g = g * w
    return g * r - x * (r * r * r * (g * x).mean(-1, keepdim=True)), dw


def _plain_grad(st):
    case = st["case"]
    c, s = _angles(case, _positions(case), st["freq"])
    dq, dwq = _norm_rope_grad(case, st["q"], st["wq"], st["dy"][0], c, s)
    dk, dwk = _norm_rope_grad(case, st["k"], st["wk"], st["dy"][1], c, s)
    st["dx"][0].copy_(dq)
    st["dx"][1].copy_(dk)
    st["dw"][0].copy_(dwq)
    st["dw"][1].copy_(dwk)
    return list(st["dx"]) + list(st["dw"])


def _seen(st):
    """(B,T,T): whether node t sees node u, itself and its ancestors among them; rows past a sequence's nodes see nothing."""
    t = st["q"].shape[1]
    i = torch.arange(t, device="cuda")
    live = i < st["count"][:, None]
    if st["parents"] is None:
        seen = (i[:, None] >= i).expand(live.shape[0], -1, -1)
    else:
        m = (torch.eye(t, device="cuda") + (st["parents"][:, :, None] == i)).float()      # 7 squarings reach 128 generations
        m = (m @ m).clamp(max=1)
        m = (m @ m).clamp(max=1)
        m = (m @ m).clamp(max=1)
        m = (m @ m).clamp(max=1)
        m = (m @ m).clamp(max=1)
        m = (m @ m).clamp(max=1)
        seen = (m @ m) > 0
    return seen & live[:, :, None] & live[:, None, :]


def _rows(st, at):
    """Page and slot of positions (B,N) of the sequences."""
    page = st["pools"][0].shape[2]
    return st["table"].long().gather(1, at // page), at % page


def _plain_append(st):
    case = st["case"]
    i = torch.arange(st["q"].shape[1], device="cuda")
    depth = _seen(st).sum(-1).clamp(min=1) - 1
    c, s = _angles(case, st["before"][:, None] + depth, st["freq"])
    live = (i < st["count"][:, None])[:, :, None, None]
    dt = st["q"].dtype
    st["q_out"].copy_(torch.where(live, _norm_rope(case, st["q"], st["wq"], c, s), 0.0))
    k = _norm_rope(case, st["k"], st["wk"], c, s).to(dt)
    page, slot = _rows(st, st["before"][:, None] + i)
    kp, vp = st["pools"]
    kp[page, :, slot] = torch.where(live, k, kp[page, :, slot])
    vp[page, :, slot] = torch.where(live, st["v"], vp[page, :, slot])


def _plain_attend(st, q):
    b, t, hq, d = q.shape
    kp, vp = st["pools"]
    hkv, page = kp.shape[1], kp.shape[2]
    table = st["table"].long()
    k, v = (p[table].transpose(2, 3).reshape(b, -1, hkv, d).transpose(1, 2).float() for p in (kp, vp))     # (B,Hkv,L,D)
    at = torch.arange(k.shape[2], device="cuda")
    u = at - st["before"][:, None]                                                   # which node a cached row is
    live = torch.arange(t, device="cuda") < st["count"][:, None]
    seen = torch.where((u < 0)[:, None], live[:, :, None], _seen(st).gather(2, u.clamp(0, t - 1)[:, None].expand(-1, t, -1)) & (u < t)[:, None])
    rows = q.float().reshape(b, t, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d)
    score = (rows @ k.transpose(-1, -2) / math.sqrt(d)).reshape(b, hkv, hq // hkv, t, -1)
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    p = (score - score.amax(-1, keepdim=True).clamp(min=-3e38)).exp()
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-38)
    # rows past a sequence's end weigh nothing, whatever they hold
    v = torch.where((at < st["after"][:, None])[:, None, :, None], v, 0.0)
    out = p.reshape(b, hkv, -1, p.shape[-1]) @ v
    st["out"].copy_(out.reshape(b, hkv, hq // hkv, t, d).permute(0, 3, 1, 2, 4).reshape(b, t, hq, d))


def _plain_commit(st):
    n = st["path"].shape[1]
    i = torch.arange(n, device="cuda")
    live = (i < st["accepted"][:, None])[:, :, None, None]
    source, target = _rows(st, st["before"][:, None] + st["path"]), _rows(st, st["before"][:, None] + i)
    kp, vp = st["pools"]
    k, v = kp[source[0], :, source[1]], vp[source[0], :, source[1]]
    kp[target[0], :, target[1]] = torch.where(live, k, kp[target[0], :, target[1]])
    vp[target[0], :, target[1]] = torch.where(live, v, vp[target[0], :, target[1]])
    st["kept"].copy_(st["before"] + st["accepted"])


# ---------------------------------------------------------------------------------------------- the framework's calls
@functools.lru_cache(maxsize=None)
def _abi():
    """The device a program opens once; its launches go to torch's stream."""
    sys.path.insert(0, os.path.join(os.getcwd(), "grilly-next_b200", "python"))
    from grilly_next import cabi
    dev = cabi.Device(0)
    cabi.check(dev.L.grl_device_use_stream(dev.h, C.c_void_p(torch.cuda.current_stream().cuda_stream or 1)))
    return cabi, dev


def _ptr(t):
    return None if t is None else t.data_ptr()


def _rope_spec(cabi, st):
    case, r = st["case"], cabi.RopeSpec()
    r.mode = cabi.ROPE_HALF if case["rope"] == "half" else cabi.ROPE_INTERLEAVED
    r.rotary_dim, r.theta, r.scaling, r.inv_freq = case["rotary"], THETA, 1.0, _ptr(st["freq"])
    return r


def _norm_params(cabi, st):
    case, p = st["case"], cabi.QKNormParams()
    p.q, p.k, p.q_out, p.k_out = _ptr(st["q"]), _ptr(st["k"]), _ptr(st["y"][0]), _ptr(st["y"][1])
    p.q_weight, p.k_weight, p.eps, p.rope = _ptr(st["wq"]), _ptr(st["wk"]), EPS, _rope_spec(cabi, st)
    p.in_dtype = p.out_dtype = cabi.F32 if case["dtype"] == "f32" else cabi.BF16
    p.batch, p.seq_len, p.num_q_heads, p.num_kv_heads, p.head_dim = case["batch"], case["seq"], case["heads"], case["kv_heads"], case["dim"]
    p.q_strides[:], p.k_strides[:] = st["q"].stride()[:3], st["k"].stride()[:3]
    p.q_out_strides[:], p.k_out_strides[:] = st["y"][0].stride()[:3], st["y"][1].stride()[:3]
    p.pos_base = case["start"]
    return p


def _layout(cabi, st, lens):
    case, kv = st["case"], cabi.KVLayout()
    kv.k_pages, kv.v_pages = st["pools"][0].data_ptr(), st["pools"][1].data_ptr()
    kv.cache_dtype = cabi.F32 if case["dtype"] == "f32" else cabi.BF16
    kv.block_table, kv.seq_lens = st["table"].data_ptr(), lens.data_ptr()
    kv.batch, kv.num_kv_heads, kv.head_dim = case["batch"], case["kv_heads"], case["dim"]
    kv.page_tokens, kv.max_pages, kv.num_pages = case["page"], st["table"].shape[1], st["table"].numel()
    return kv


def _calls(st):
    """The calls of a pass, their parameters filled in once."""
    cabi, dev = _abi()
    case, kind = st["case"], st["case"]["kind"]
    dtype = cabi.F32 if case["dtype"] == "f32" else cabi.BF16
    if kind == "norm":
        p = _norm_params(cabi, st)
        return [(dev.L.grl_qk_norm_rope, dev.h, C.byref(p), p)]
    if kind == "grad":
        p = cabi.QKNormGradParams()
        p.fwd = _norm_params(cabi, st)
        p.q_out_grad, p.k_out_grad = _ptr(st["dy"][0]), _ptr(st["dy"][1])
        p.q_grad, p.k_grad, p.q_weight_grad, p.k_weight_grad = _ptr(st["dx"][0]), _ptr(st["dx"][1]), _ptr(st["dw"][0]), _ptr(st["dw"][1])
        p.q_grad_strides[:], p.k_grad_strides[:] = st["dx"][0].stride()[:3], st["dx"][1].stride()[:3]
        size = C.c_size_t()
        cabi.check(dev.L.grl_qk_norm_rope_backward_workspace_bytes(dev.h, C.byref(p), C.byref(size)))
        st["space"] = torch.empty(max(16, size.value), dtype=torch.uint8, device="cuda")
        p.workspace, p.workspace_bytes = _ptr(st["space"]), st["space"].numel()
        return [(dev.L.grl_qk_norm_rope_backward, dev.h, C.byref(p), p)]
    calls = []
    if kind != "attend":
        p = cabi.AppendNormParams()
        p.kv = _layout(cabi, st, st["before"])
        p.k_new, p.v_new, p.q_in, p.q_out = _ptr(st["k"]), _ptr(st["v"]), _ptr(st["q"]), _ptr(st["q_out"])
        p.in_dtype = p.q_out_dtype = dtype
        p.n_new, p.num_q_heads = st["q"].shape[1], st["q"].shape[2]
        p.q_weight, p.k_weight, p.eps, p.rope = _ptr(st["wq"]), _ptr(st["wk"]), EPS, _rope_spec(cabi, st)
        p.parents, p.n_nodes = _ptr(st["parents"]), _ptr(st["count"])
        calls.append((dev.L.grl_kv_append_norm, dev.h, C.byref(p), p))
    if kind in ("attend", "step"):
        p = cabi.TreeParams()
        p.kv = _layout(cabi, st, st["after"])
        p.q, p.out, p.io_dtype = _ptr(st["q_out"] if kind == "step" else st["q"]), _ptr(st["out"]), dtype
        p.num_q_heads, p.n_tree = st["q"].shape[2], st["q"].shape[1]
        p.parents, p.n_nodes, p.max_seq_len = _ptr(st["parents"]), _ptr(st["count"]), st["most"]
        size = C.c_size_t()
        cabi.check(dev.L.grl_tree_workspace_bytes(dev.h, C.byref(p), C.byref(size)))
        st["space"] = torch.empty(max(16, size.value), dtype=torch.uint8, device="cuda")
        p.workspace, p.workspace_bytes = _ptr(st["space"]), st["space"].numel()
        calls.append((dev.L.grl_tree_attention, dev.h, C.byref(p), p))
    if kind in ("keep", "step"):
        p = cabi.CommitParams()
        p.kv = _layout(cabi, st, st["after"])
        p.path, p.n_path, p.max_path = _ptr(st["path"]), _ptr(st["accepted"]), st["path"].shape[1]
        p.n_nodes, p.n_tree, p.lens_out = _ptr(st["count"]), st["q"].shape[1], _ptr(st["kept"])
        calls.append((dev.L.grl_kv_commit, dev.h, C.byref(p), p))
    return calls


# ---------------------------------------------------------------------------------------------- one pass
def _outputs(st):
    kind = st["case"]["kind"]
    if kind == "norm":
        return list(st["y"])
    if kind == "grad":
        return list(st["dx"]) + list(st["dw"])
    if kind == "attend":
        return [st["out"]]
    if kind == "append":
        return list(st["pools"]) + [st["q_out"]]
    if kind == "keep":
        return list(st["pools"]) + [st["q_out"], st["kept"]]
    return [st["out"]] + list(st["pools"]) + [st["q_out"], st["kept"]]


def run(state):
    kind = state["case"]["kind"]
    if own:
        calls = state.get("calls")
        if calls is None:
            calls = state["calls"] = _calls(state)
        for call in calls:
            rc = call[0](call[1], call[2])
            if rc:
                _abi()[0].check(rc)
        return _outputs(state)
    if kind == "norm":
        return _plain_norm(state)
    if kind == "grad":
        return _plain_grad(state)
    if kind == "attend":
        _plain_attend(state, state["q"])
        return _outputs(state)
    _plain_append(state)
    if kind == "step":
        _plain_attend(state, state["q_out"])
    if kind in ("keep", "step"):
        _plain_commit(state)
    return _outputs(state)


# ---------------------------------------------------------------------------------------------- the definition in 64 bits
def _exact_rotation(case, pos, freq):
    """(N, D, D) rotation matrices of positions."""
    r, d = case["rotary"], case["dim"]
    m = np.broadcast_to(np.eye(d), (len(pos), d, d)).copy()
    for j in range(r // 2):
        f = float(freq[j]) if freq is not None else THETA ** (-2.0 * j / r)
        lo, hi = (j, j + r // 2) if case["rope"] == "half" else (2 * j, 2 * j + 1)
        c, s = np.cos(pos * f), np.sin(pos * f)
        m[:, lo, lo], m[:, lo, hi], m[:, hi, lo], m[:, hi, hi] = c, -s, s, c
    return torch.from_numpy(m).cuda()


def _exact_norm(x, w):
    x = x.double()
    return x / ((x ** 2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * w.double()


def exact(case, seed):
    st = prepare(case, seed)
    freq = st["freq"].cpu().numpy().astype(np.float64) if st.get("freq") is not None else None
    if case["kind"] in ("norm", "grad"):
        turn = _exact_rotation(case, case["start"] + np.arange(case["seq"], dtype=np.float64), freq)
        if case["kind"] == "norm":
            return [torch.einsum("sij,bshj->bshi", turn, _exact_norm(st[n], st["w" + n])) for n in "qk"]
        dx, dw = [], []
        for n, dy in zip("qk", st["dy"]):
            x, w = st[n].double(), st["w" + n].double()
            g = torch.einsum("sji,bshj->bshi", turn, dy.double())
            size = ((x ** 2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt()
            dw.append((g * x / size).sum((0, 1, 2)))
            dx.append(w * g / size - x * (w * g * x).sum(-1, keepdim=True) / (x.shape[-1] * size ** 3))
        return dx + dw
    b, t, hq, d = st["q"].shape
    kp, vp = (p.double() for p in st["pools"])
    hkv, page, dt = kp.shape[1], kp.shape[2], st["q"].dtype
    q, q_out = st["q"].double(), torch.zeros((b, t, hq, d), dtype=torch.float64, device="cuda")
    out, kept = torch.zeros_like(q_out), []
    table, parents = st["table"].cpu().numpy(), st["parents"].cpu().numpy() if case["tree"] else None
    for i, (n, m) in enumerate(zip(_tokens(case), _nodes(case))):
        above = []                                # above[u]: node u's ancestors and itself
        for u in range(m):
            p = int(parents[i, u]) if case["tree"] else u - 1
            above.append((above[p] if p >= 0 else []) + [u])
        at = lambda rows: (torch.tensor(table[i][np.asarray(rows) // page], device="cuda").long(), torch.tensor(np.asarray(rows) % page, device="cuda"))  # noqa: E731
        if case["kind"] != "attend" and m:
            turn = _exact_rotation(case, n + np.array([len(a) - 1 for a in above], dtype=np.float64), freq)
            pages, slots = at(n + np.arange(m))
            kp[pages, :, slots] = torch.einsum("sij,shj->shi", turn, _exact_norm(st["k"][i, :m], st["wk"]))
            vp[pages, :, slots] = st["v"][i, :m].double()
            q_out[i, :m] = torch.einsum("sij,shj->shi", turn, _exact_norm(st["q"][i, :m], st["wq"]))
        if case["kind"] in ("attend", "step") and m:
            rows = (q if case["kind"] == "attend" else q_out.to(dt).double())[i, :m]
            pages, slots = at(np.arange(n + m))
            k, v = (x[pages, :, slots].to(dt).double().transpose(0, 1) for x in (kp, vp))       # (Hkv, n + m, D)
            seen = torch.zeros((m, n + m), dtype=torch.bool, device="cuda")
            seen[:, :n] = True
            for u in range(m):
                seen[u, [n + a for a in above[u]]] = True
            score = torch.einsum("uhgd,hld->hgul", rows.reshape(m, hkv, hq // hkv, d), k) / math.sqrt(d)
            weight = torch.softmax(score.masked_fill(~seen, -math.inf), -1)
            out[i, :m] = torch.einsum("hgul,hld->uhgd", weight, v).reshape(m, hq, d)
        if case["kind"] in ("keep", "step"):
            path = st["path"][i, :int(st["accepted"][i])].cpu().numpy()
            kept.append(n + len(path))
            if len(path):
                old, new = at(n + path), at(n + np.arange(len(path)))
                for x in (kp, vp):
                    x[new[0], :, new[1]] = x[old[0], :, old[1]].clone()
    if case["kind"] == "attend":
        return [out]
    if case["kind"] == "append":
        return [kp, vp, q_out]
    kept = torch.tensor(kept, dtype=torch.int32, device="cuda")
    return [kp, vp, q_out, kept] if case["kind"] == "keep" else [out, kp, vp, q_out, kept]
