"""Paged-cache operators at sizes that reach what small cases do not: an item joined from more than
128 parts, more sequences than a CTA of the tcgen05 kernel has threads, inputs in pinned host memory."""
from __future__ import annotations

import math

import pytest
import torch

from paged_ref import TYPES, Case
from test_gpu_paged import KINDS, SIXTEEN, WIDE, check, near

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,cache", KINDS)
@pytest.mark.parametrize("H,KVH,D", [(8, 1, 64), (14, 2, 64), (8, 1, 128)])
@pytest.mark.parametrize("n", [33001, 70000])
@pytest.mark.parametrize("rising", [True, False])
def test_one_token_over_a_long_context(tq, kind, cache, H, KVH, D, n, rising):
    """A long context is cut into more parts than are joined at a time, so the running maximum, sum and values
    are carried from one round of the join to the next.  rising: scores grow (or fall) by 24
    over the context, so that the maximum is raised in the later rounds (or never).

    Tolerance: a part has at most 8 tiles of 64 positions, 32 additions for each of a lane's sums, and at most
    300 parts are added in a row: under 400 fp32 additions, as a context of 400 positions has."""
    c = Case([1], [1], H, KVH, D, 64, True, kind, cache, seed=n)
    g = torch.Generator().manual_seed(n + D)
    c.total, c.pool = [n], -(-n // 64)
    c.table_cpu = torch.randperm(c.pool, generator=g).to(torch.int32)[None]
    q = c.q_cpu.view(H, D).double()
    # along the mean of a KV head's queries, whose scores then rise alike
    lean = q.view(KVH, H // KVH, D).mean(1)
    slope = 24.0 / c.scale / float((q * lean.repeat_interleave(H // KVH, 0)).sum(-1).abs().max())
    x = torch.arange(c.pool * 64, dtype=torch.float64) / n
    ramp = (x if rising else 1 - x)[None, :, None] * slope * lean[:, None]
    k = torch.randn(KVH, c.pool * 64, D, generator=g) + ramp.float()
    v = torch.randn(KVH, c.pool * 64, D, generator=g)
    order = torch.empty_like(c.table_cpu[0]).long()
    order[c.table_cpu[0].long()] = torch.arange(c.pool)
    place = lambda t: t.view(KVH, c.pool, 64, D).transpose(0, 1)[order].contiguous().to(TYPES[cache])  # noqa: E731
    c.k_cpu, c.v_cpu = place(k), place(v)
    c.upload()
    got = c.attend(tq).double().cpu().view(H, D)
    assert int(c.status) == 0
    kk = k.to(TYPES[cache]).double()[:, :n].repeat_interleave(H // KVH, 0)
    vv = v.to(TYPES[cache]).double()[:, :n].repeat_interleave(H // KVH, 0)
    s = torch.einsum("hd,hxd->hx", q, kk) * c.scale
    want = torch.einsum("hx,hxd->hd", torch.softmax(s, -1), vv)
    most = float((torch.einsum("hd,hxd->hx", q.abs(), kk.abs()) * c.scale).max())
    c.total = [400]
    near(got, want, c.tolerance(most, float(vv.abs().max())))


@pytest.mark.parametrize("kind,cache", SIXTEEN)
@pytest.mark.parametrize("seqs,new", [(140, 5), (500, 5), (1000, 7)])
def test_many_sequences_on_tcgen05(tq, kind, cache, seqs, new):
    """More sequences than the threads of a CTA (448), several to a thread; some without rows."""
    new = [0 if i % 7 == 3 else new for i in range(seqs)]
    total = [n + (i * 37) % 70 for i, n in enumerate(new)]
    c = Case(new, total, 8, 2, 64, 16, True, kind, cache, pad=1, seed=seqs, room=WIDE)
    check(c, tq)
    assert int(c.status) == 0


@pytest.mark.parametrize("new", [1, 40])
def test_lengths_and_tables_in_pinned_host_memory(tq, new):
    """Memory that the device reads, so it is taken; pageable memory is refused (test_gpu_paged)."""
    c = Case([new, new], [70, 90], 8, 2, 64, 16, True, "f16", "f16", seed=1, room=WIDE if new > 1 else 0)
    c.start, c.len, c.table = (t.cpu().pin_memory() for t in (c.start, c.len, c.table))
    check(c, tq)
    assert int(c.status) == 0


def test_a_workspace_serves_every_batch(tq):
    """Its bytes depend on the device and head_dim alone, so a call of few rows leaves it ready for many."""
    a = Case([90] * 3, [2500, 700, 91], 8, 2, 64, 16, True, "f16", "f16", seed=8, room=WIDE)
    b = Case([1, 2], [1000, 1500], 32, 8, 64, 16, True, "f32", "f32", seed=1)
    w = a.workspace(tq, *a.handles(tq))
    assert w.numel() == b.workspace(tq, *b.handles(tq)).numel()
    for _ in range(2):
        check(a, tq, work=w)
        check(b, tq, work=w)
