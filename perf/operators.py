"""Cases of the paged-cache operators for many requests: query/key norms with the position
rotation, the append of new keys and values to a paged cache, and attention of new tokens
(a chunk of a prompt, or single tokens) over that cache.

With ``own`` false the operators run in their plain form (elementary torch operations in 32
bits); with ``own`` true they run through the library's entry points.  ``exact`` restates
their definitions in 64 bits.
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_CODES = {"f32": 0, "f16": 1, "bf16": 2}
_EPS = 1e-6


def _lib():
    """The ctypes binding; its package folder is not on the path by itself."""
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tiny-llm_b200")
    if here not in sys.path:
        sys.path.append(here)
    from tqb200 import lib
    return lib


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one request of the fp16-cache decode configuration at its full context
        dict(name="attn 1 x 4096 f32/f16", op="attention", type="f32", cache="f16", heads=32,
             kv_heads=8, dim=128, page=16, heads_first=True, seqs=1, q_min=1, q_max=1,
             ctx_min=4095, ctx_max=4095, pad=0, mix=1),
        # the shortest contexts of the smallest model (7 query heads per KV head), fp32 cache:
        # the call's latency
        dict(name="attn 3 x 1..40 f32/f32 d64", op="attention", type="f32", cache="f32", heads=14,
             kv_heads=2, dim=64, page=16, heads_first=False, seqs=3, q_min=1, q_max=1,
             ctx_min=0, ctx_max=40, pad=0, mix=2),
        # a serving batch of single tokens over contexts of very different lengths
        dict(name="attn 64 x 100..8192 bf16", op="attention", type="bf16", cache="bf16", heads=32,
             kv_heads=8, dim=128, page=32, heads_first=False, seqs=64, q_min=1, q_max=1,
             ctx_min=100, ctx_max=8191, pad=0, mix=3),
        # the 512-token prompt of the MoE configuration (8 query heads per KV head)
        dict(name="attn prompt 512 f32/f16", op="attention", type="f32", cache="f16", heads=32,
             kv_heads=4, dim=128, page=16, heads_first=True, seqs=1, q_min=512, q_max=512,
             ctx_min=0, ctx_max=0, pad=0, mix=4),
        # one chunk of a long prompt over what is cached of it
        dict(name="attn chunk 2048+14336 bf16", op="attention", type="bf16", cache="bf16", heads=32,
             kv_heads=8, dim=128, page=64, heads_first=True, seqs=1, q_min=2048, q_max=2048,
             ctx_min=14336, ctx_max=14336, pad=0, mix=5),
        # prompt chunks of odd lengths in one batch with single tokens, rows behind the last
        # sequence left alone
        dict(name="attn mixed 8 x 1..509 f16 d64", op="attention", type="f16", cache="f16", heads=14,
             kv_heads=2, dim=64, page=24, heads_first=False, seqs=8, q_min=1, q_max=509,
             ctx_min=7, ctx_max=4093, pad=3, mix=6),
        # one new token: its norms, rotation and append between the projections and attention
        dict(name="append 1 f32/f16", op="append", type="f32", cache="f16", heads=32, kv_heads=8,
             dim=128, rotary=128, theta=1e6, norm=True, page=16, heads_first=True, seqs=1, q_min=1,
             q_max=1, ctx_min=4000, ctx_max=4000, pad=0, mix=7),
        # a serving batch of single tokens, padded to a fixed row count
        dict(name="append 61+3 bf16", op="append", type="bf16", cache="bf16", heads=32, kv_heads=8,
             dim=128, rotary=128, theta=1e6, norm=True, page=32, heads_first=False, seqs=61, q_min=1,
             q_max=1, ctx_min=0, ctx_max=8000, pad=3, mix=8),
        # prompts of odd lengths, no norms (the smallest model), fp32 cache
        dict(name="append 5 x 30..700 f32 d64", op="append", type="f32", cache="f32", heads=14,
             kv_heads=2, dim=64, rotary=64, theta=1e6, norm=False, page=16, heads_first=False,
             seqs=5, q_min=30, q_max=700, ctx_min=0, ctx_max=300, pad=0, mix=9),
        # a long prompt's chunk out of a fused q/k/v projection
        dict(name="append 8192 bf16", op="append", type="bf16", cache="bf16", heads=32, kv_heads=8,
             dim=128, rotary=128, theta=1e6, norm=True, page=64, heads_first=True, seqs=2,
             q_min=4096, q_max=4096, ctx_min=0, ctx_max=100000, pad=0, mix=10),
        # the 512-token prompt's norms and rotation (the cache kept elsewhere)
        dict(name="norm+rope 512 f32", op="rotate", type="f32", heads=32, kv_heads=4, dim=128,
             rotary=128, theta=1e6, norm=True, tokens=512, far=512, mix=11),
        # a long chunk with rotation over a quarter of each head only
        dict(name="norm+rope 8191 f16 part", op="rotate", type="f16", heads=32, kv_heads=8, dim=128,
             rotary=32, theta=1e4, norm=True, tokens=8191, far=131072, mix=12),
    ]


def _spread(rng, lo, hi):
    """A whole number of lo..hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(max(lo, 0.5)), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "append", "rotate"])
    heads, kv_heads, dim = rng.choice([(32, 8, 128), (32, 4, 128), (16, 8, 128), (14, 2, 64), (4, 2, 64),
                                       (16, 4, 64), (5, 5, 64)])
    kind, cache = rng.choice([("f32", "f16"), ("f32", "f32"), ("f16", "f16"), ("bf16", "bf16")])
    c = dict(op=op, type=kind, heads=heads, kv_heads=kv_heads, dim=dim, mix=rng.randrange(1 << 20))
    if op == "rotate":
        tokens = _spread(rng, 1, 8191)
        c.update(rotary=rng.choice([dim, dim, dim // 2, dim // 4]), theta=rng.choice([1e4, 1e6]),
                 norm=rng.random() < 0.6, tokens=tokens, far=_spread(rng, tokens, 131072))
        return c
    c.update(cache=cache, page=rng.choice([1, 5, 8, 16, 16, 24, 32, 64, 128]),
             heads_first=rng.random() < 0.5, pad=rng.choice([0, 0, 0, 1, 7]))
    if op == "append":
        seqs = _spread(rng, 1, 64)
        q_max = 1 if rng.random() < 0.4 else _spread(rng, 2, 8000 // seqs)
        c.update(rotary=rng.choice([dim, dim, dim // 4]), theta=rng.choice([1e4, 1e6]),
                 norm=rng.random() < 0.6, seqs=seqs, q_min=1, q_max=q_max, ctx_min=0,
                 ctx_max=_spread(rng, 1, 100000 // seqs))
        return c
    if rng.random() < 0.5:  # single tokens
        seqs = _spread(rng, 1, 64)
        c.update(seqs=seqs, q_min=1, q_max=1, ctx_min=0, ctx_max=_spread(rng, 1, 200000 // seqs))
    else:
        seqs = _spread(rng, 1, 8)
        c.update(seqs=seqs, q_min=1, q_max=_spread(rng, 2, 2048 // seqs), ctx_min=0,
                 ctx_max=_spread(rng, 1, 12000 // seqs))
    return c


def _lengths(case):
    """Every sequence's new tokens and cached positions after them; the first has the most of
    both (the rest spread evenly over the logarithm)."""
    r = random.Random(case["mix"])
    new = [case["q_max"]] + [_spread(r, case["q_min"], case["q_max"]) for _ in range(case["seqs"] - 1)]
    ctx = [case["ctx_max"]] + [_spread(r, case["ctx_min"], max(1, case["ctx_max"])) for _ in range(case["seqs"] - 1)]
    ctx = [min(c, case["ctx_max"]) for c in ctx]
    return new, [n + c for n, c in zip(new, ctx)]


def work(case):
    size = _TYPES[case["type"]].itemsize
    h, kvh, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "rotate":
        n = case["tokens"] * (h + kvh) * d
        return {"bytes": 2 * n * size, "flops": 8 * n}
    new, total = _lengths(case)
    held = _TYPES[case["cache"]].itemsize
    if case["op"] == "append":
        n = sum(new) * d
        return {"bytes": n * (2 * h * size + 2 * kvh * (size + held)), "flops": 8 * n * (h + kvh)}
    pairs = sum(n * (t - n) + n * (n + 1) // 2 for n, t in zip(new, total))
    return {"bytes": 2 * sum(new) * h * d * size + 2 * sum(total) * kvh * d * held,
            "flops": 4 * d * h * pairs}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    kind = _TYPES[case["type"]]
    h, kvh, d = case["heads"], case["kv_heads"], case["dim"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    s = dict(case=dict(case))
    if case["op"] != "attention" and case["norm"]:
        s["q_norm"] = 1.0 + 0.3 * normal(d)
        s["k_norm"] = 1.0 + 0.3 * normal(d)
    if case["op"] == "rotate":
        n = case["tokens"]
        # rows of a fused projection's output: q heads, k heads, v heads
        s["qkv"] = (3.0 * normal(n, (h + 2 * kvh) * d)).to(kind)
        s["positions"] = torch.randint(0, case["far"], (n,), generator=g, device=dev, dtype=torch.int32)
        s["q_out"] = torch.zeros(n, h, d, device=dev, dtype=kind)
        s["k_out"] = torch.zeros(n, kvh, d, device=dev, dtype=kind)
        return s
    new, total = _lengths(case)
    page, n = case["page"], sum(new) + case["pad"]
    used = [-(-t // page) for t in total]
    pool = sum(used) + 2
    order = torch.randperm(pool, generator=g, device=dev).to(torch.int32)
    table = torch.full((len(new), max(used)), -1, device=dev, dtype=torch.int32)
    at = 0
    for i, u in enumerate(used):
        table[i, :u] = order[at:at + u]
        at += u
    start = [0]
    for x in new:
        start.append(start[-1] + x)
    s["q_start"] = torch.tensor(start, device=dev, dtype=torch.int32)
    s["kv_len"] = torch.tensor(total, device=dev, dtype=torch.int32)
    s["table"], s["n"], s["q_most"], s["kv_most"] = table, n, max(new), max(total)
    shape = (pool + 1, kvh, page, d) if case["heads_first"] else (pool + 1, page, kvh, d)
    held = _TYPES[case["cache"]]
    lean = 1.0 + 2.0 * (torch.arange(d, device=dev) % 16 == 3)  # some channels stand out, as in trained keys
    # one page more than the pool: where the plain form puts the rows that it has to drop
    s["k_all"] = (normal(*shape) * lean).to(held)
    s["v_all"] = normal(*shape).to(held)
    s["k"], s["v"] = s["k_all"][:pool], s["v_all"][:pool]
    if case["op"] == "append":
        s["qkv"] = (3.0 * normal(n, (h + 2 * kvh) * d)).to(kind)
        s["q_out"] = torch.zeros(n, h, d, device=dev, dtype=kind)
    else:
        s["q"] = (1.5 * normal(n, h, d)).to(kind)
        s["out"] = torch.zeros(n, h, d, device=dev, dtype=kind)
    if own:
        lib = _lib()
        s["lib"] = lib
        where = ((kvh * page * d, page * d, d) if case["heads_first"] else (page * kvh * d, d, kvh * d))
        s["cache"] = lib.PagedCache(s["k"].data_ptr(), s["v"].data_ptr(), _CODES[case["cache"]], pool, page,
                                    kvh, d, *where)
        s["batch"] = lib.PagedBatch(s["q_start"].data_ptr(), s["kv_len"].data_ptr(), table.data_ptr(),
                                    len(new), table.shape[1], n, max(new))
        if case["op"] == "attention":
            need = lib.paged_attention_workspace_bytes(s["cache"], s["batch"], h)
            s["work"] = torch.zeros(max(1, need), device=dev, dtype=torch.uint8)
    return s


# ------------------------------------------------------------------ the plain forms
def _rotated(x, weight, pos, rotary, theta):
    """Each head's RMS norm (where there are weights), then the rotation of its first `rotary`
    dimensions by the row's position; x [rows, heads, dim], pos [rows]."""
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * weight
    half = rotary // 2
    freq = torch.pow(torch.tensor(theta, dtype=torch.float64, device=x.device),
                     -2.0 * torch.arange(half, device=x.device, dtype=torch.float64) / rotary)
    angle = pos.double()[:, None] * freq
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    a, b = x[..., :half], x[..., half:rotary]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., rotary:]], -1)


def _plain_rotate(s):
    c = s["case"]
    h, kvh, d = c["heads"], c["kv_heads"], c["dim"]
    rows = s["qkv"].view(c["tokens"], h + 2 * kvh, d)
    q = _rotated(rows[:, :h], s.get("q_norm"), s["positions"], c["rotary"], c["theta"])
    k = _rotated(rows[:, h:h + kvh], s.get("k_norm"), s["positions"], c["rotary"], c["theta"])
    return {"q": q.to(rows.dtype), "k": k.to(rows.dtype)}


def _plain_append(s):
    c = s["case"]
    h, kvh, d, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    rows = s["qkv"].view(s["n"], h + 2 * kvh, d)
    start, row = s["q_start"].long(), torch.arange(s["n"], device=rows.device)
    seq = (row[:, None] >= start[None, 1:-1]).sum(-1)
    live = row < start[-1]
    pos = s["kv_len"].long()[seq] - start[seq + 1] + row
    pos = torch.where(live, pos, torch.zeros_like(pos))
    q = _rotated(rows[:, :h], s.get("q_norm"), pos, c["rotary"], c["theta"]).to(rows.dtype)
    k = _rotated(rows[:, h:h + kvh], s.get("k_norm"), pos, c["rotary"], c["theta"])
    to = torch.where(live, s["table"].long()[seq, pos // page], s["k"].shape[0])
    slot = pos % page
    at = (to, slice(None), slot) if c["heads_first"] else (to, slot)
    s["k_all"][at] = k.to(s["k"].dtype)
    s["v_all"][at] = rows[:, h + kvh:].to(s["v"].dtype)
    s["q_out"].copy_(torch.where(live[:, None, None], q, s["q_out"]))
    return {"q": s["q_out"], "k": s["k"], "v": s["v"]}


def _plain_attention(s):
    c = s["case"]
    h, kvh, d, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    dev, group = s["q"].device, h // kvh
    pos = torch.arange(s["kv_most"], device=dev)
    pages = s["table"].long()[:, pos // page].clamp(min=0)
    at = (pages, slice(None), pos % page) if c["heads_first"] else (pages, pos % page)
    k = s["k"][at].float().permute(0, 2, 3, 1)  # [seqs, kv heads, dim, positions]
    v = s["v"][at].float().permute(0, 2, 1, 3)
    start, length = s["q_start"].long(), s["kv_len"].long()
    i = torch.arange(s["q_most"], device=dev)
    live = i < (start[1:] - start[:-1])[:, None]
    row = torch.where(live, start[:-1, None] + i, s["n"])
    q = torch.cat([s["q"], s["q"][:1]])[row].float()
    seqs, most = row.shape
    q = q.view(seqs, most, kvh, group, d).permute(0, 2, 3, 1, 4).reshape(seqs, kvh, group * most, d)
    score = torch.matmul(q, k).mul_(1.0 / math.sqrt(d)).view(seqs, kvh, group, most, -1)
    last = length[:, None] - (start[1:] - start[:-1])[:, None] + i  # the row's own position
    seen = pos <= last[..., None]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    score -= score.amax(-1, keepdim=True).clamp(min=-1e30)
    p = score.exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(seqs, kvh, group * most, -1), v).view(seqs, kvh, group, most, d)
    o = (o / total.clamp(min=1e-30)).permute(0, 3, 1, 2, 4).reshape(seqs, most, h, d)
    out = torch.cat([s["out"], s["out"][:1]])
    out[row] = o.to(out.dtype)
    return {"out": out[:-1]}


# ------------------------------------------------------------------ the library's operators
def _own_rotate(s):
    c, lib = s["case"], _lib()
    size, width = s["qkv"].element_size(), s["qkv"].shape[1]
    h, kvh, d = c["heads"], c["kv_heads"], c["dim"]
    at = s["qkv"].data_ptr()
    lib.dev_qk_norm_rope(at, at + h * d * size, s["q_out"].data_ptr(), s["k_out"].data_ptr(),
                         _CODES[c["type"]], c["tokens"], h, kvh, d, c["rotary"], width, width, h * d, kvh * d,
                         s["q_norm"].data_ptr() if c["norm"] else None,
                         s["k_norm"].data_ptr() if c["norm"] else None, _EPS, c["theta"],
                         s["positions"].data_ptr())
    return {"q": s["q_out"], "k": s["k_out"]}


def _own_append(s):
    c, lib = s["case"], s["lib"]
    size, width = s["qkv"].element_size(), s["qkv"].shape[1]
    h, kvh, d = c["heads"], c["kv_heads"], c["dim"]
    at = s["qkv"].data_ptr()
    lib.dev_paged_append(at, at + h * d * size, at + (h + kvh) * d * size, s["q_out"].data_ptr(),
                         _CODES[c["type"]], h, c["rotary"], width, width, width, h * d,
                         s["q_norm"].data_ptr() if c["norm"] else None,
                         s["k_norm"].data_ptr() if c["norm"] else None, _EPS, c["theta"], None,
                         s["cache"], s["batch"])
    return {"q": s["q_out"], "k": s["k"], "v": s["v"]}


def _own_attention(s):
    c, lib = s["case"], s["lib"]
    h, d = c["heads"], c["dim"]
    lib.dev_paged_attention(s["q"].data_ptr(), s["out"].data_ptr(), _CODES[c["type"]], h, h * d, h * d,
                            1.0 / math.sqrt(d), s["cache"], s["batch"], s["work"].data_ptr(),
                            s["work"].numel())
    return {"out": s["out"]}


def run(state):
    op = state["case"]["op"]
    if own:
        return _own_rotate(state) if op == "rotate" else _own_append(state) if op == "append" else _own_attention(state)
    return _plain_rotate(state) if op == "rotate" else _plain_append(state) if op == "append" else _plain_attention(state)


# ------------------------------------------------------------------ the definitions in 64 bits
def _turned(x, weight, pos, rotary, theta):
    """One head's rows [rows, dim] in 64 bits, as complex numbers turned by their angles."""
    x = x.double()
    if weight is not None:
        x = x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + _EPS).sqrt() * weight.double()
    half = rotary // 2
    step = torch.tensor([theta ** (-2.0 * i / rotary) for i in range(half)], dtype=torch.float64, device=x.device)
    turn = torch.polar(torch.ones_like(step).expand(len(pos), half), pos.double()[:, None] * step)
    z = torch.complex(x[:, :half].contiguous(), x[:, half:rotary].contiguous()) * turn
    return torch.cat([z.real, z.imag, x[:, rotary:]], 1)


def exact(case, seed):
    s = prepare(case, seed)
    h, kvh, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "rotate":
        rows = s["qkv"].view(case["tokens"], h + 2 * kvh, d)
        pos, (rotary, theta) = s["positions"], (case["rotary"], case["theta"])
        q = [_turned(rows[:, i], s.get("q_norm"), pos, rotary, theta) for i in range(h)]
        k = [_turned(rows[:, h + i], s.get("k_norm"), pos, rotary, theta) for i in range(kvh)]
        return {"q": torch.stack(q, 1), "k": torch.stack(k, 1)}
    new, total = _lengths(case)
    page, table = case["page"], s["table"].tolist()
    first, dev = 0, s["k"].device
    if case["op"] == "append":
        rows = s["qkv"].view(s["n"], h + 2 * kvh, d)
        k, v = s["k"].double(), s["v"].double()
        q = torch.zeros(s["n"], h, d, device=dev, dtype=torch.float64)
        for i, (n, t) in enumerate(zip(new, total)):
            mine, pos = rows[first:first + n], torch.arange(t - n, t, device=dev)
            to = torch.tensor([table[i][x // page] for x in range(t - n, t)], device=dev)
            for j in range(h):
                q[first:first + n, j] = _turned(mine[:, j], s.get("q_norm"), pos, case["rotary"], case["theta"])
            for j in range(kvh):
                key = _turned(mine[:, h + j], s.get("k_norm"), pos, case["rotary"], case["theta"])
                val = mine[:, h + kvh + j].double()
                if case["heads_first"]:
                    k[to, j, pos % page], v[to, j, pos % page] = key, val
                else:
                    k[to, pos % page, j], v[to, pos % page, j] = key, val
            first += n
        return {"q": q, "k": k, "v": v}
    out = torch.zeros(s["n"], h, d, device=dev, dtype=torch.float64)
    for i, (n, t) in enumerate(zip(new, total)):
        pos = torch.arange(t, device=dev)
        to = torch.tensor([table[i][x // page] for x in range(t)], device=dev)
        seen = pos[None, :] <= torch.arange(t - n, t, device=dev)[:, None]
        for j in range(h):
            head = j * kvh // h
            at = (to, head, pos % page) if case["heads_first"] else (to, pos % page, head)
            score = s["q"][first:first + n, j].double() @ s["k"][at].double().T / math.sqrt(d)
            score[~seen] = -math.inf
            out[first:first + n, j] = torch.softmax(score, -1) @ s["v"][at].double()
        first += n
    return {"out": out}
