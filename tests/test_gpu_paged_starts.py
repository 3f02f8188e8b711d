"""Malformed q_start entries: the sequences whose numbers do not fit are skipped and reported,
the rows of every other sequence are served, by append and by every attention kernel."""
from __future__ import annotations

import pytest
import torch

from paged_ref import CODES, TYPES, Case
from test_gpu_paged import KINDS, WIDE, near

pytestmark = pytest.mark.gpu

SPOILT = ["negative", "backwards", "too large", "past its rows", "last too small"]


def spoil(c, what, at):
    """The starts with entry `at` spoilt, and which sequence each row belongs to (-1: none)."""
    st, n, most = c.start.tolist(), c.n, max(c.new)
    if what == "last too small":
        st[-1] = 0
    else:
        st[at] = {"negative": -1, "backwards": 0, "too large": n + 5, "past its rows": n}[what]
    c.start.copy_(torch.tensor(st, dtype=torch.int32))
    owner = [-1] * n
    bad = 0
    for s, (lo, hi) in enumerate(zip(st, st[1:])):
        if not (0 <= lo <= hi <= n and hi - lo <= most):
            bad += 1
            continue
        for t in range(lo, hi):
            assert owner[t] == -1
            owner[t] = s
    assert bad and any(o >= 0 for o in owner)
    return st, torch.tensor(owner)


def batch(seqs, each, kind, cache, D, H=2, KVH=1, room=0, gap=0, shift=0):
    new = [each] * seqs
    total = [each + (i * 7) % 23 for i in range(seqs)]
    return Case(new, total, H, KVH, D, 16, True, kind, cache, pad=3, seed=seqs + D, room=room, gap=gap, shift=shift)


WHERE = [(7, 1), (7, 4), (50, 16), (50, 33), (100, 32), (100, 64), (100, 97)]


@pytest.mark.parametrize("what", SPOILT)
@pytest.mark.parametrize("seqs,at", WHERE)
@pytest.mark.parametrize("kind,cache,D,shift", [("f32", "f32", 64, 0), ("f32", "f16", 128, 0), ("bf16", "bf16", 64, 1),
                                                ("f16", "f16", 40, 0)])
@pytest.mark.parametrize("each", [1, 3])
def test_append_serves_the_other_sequences(tq, what, seqs, at, kind, cache, D, shift, each):
    c = batch(seqs, each, kind, cache, D)
    st, owner = spoil(c, what, at)
    g = torch.Generator().manual_seed(at)
    H, n = 2, c.n
    rows = torch.randn(n * (H + 2) * D + 8, generator=g).to(TYPES[kind]).cuda()
    x = rows[shift:shift + n * (H + 2) * D].view(n, H + 2, D)
    q = torch.full((n, H, D), 7.0, dtype=TYPES[kind], device="cuda")
    want_k, want_v = c.kview.clone(), c.vview.clone()
    for t in range(n):
        s = int(owner[t])
        if s >= 0:
            pos = c.total[s] - (st[s + 1] - st[s]) + t - st[s]
            p = int(c.table_cpu[s, pos // 16])
            want_k[p, :, pos % 16] = x[t, H:H + 1].cpu().to(TYPES[cache])
            want_v[p, :, pos % 16] = x[t, H + 1:].cpu().to(TYPES[cache])
    ch, b = c.handles(tq, max_q=each)
    size, width = rows.element_size(), (H + 2) * D
    at_ = x.data_ptr()
    tq.dev_paged_append(at_, at_ + H * D * size, at_ + (H + 1) * D * size, q.data_ptr(), CODES[kind], H, 0, width, width,
                        width, H * D, None, None, 0.0, 1e4, None, ch, b, c.status.data_ptr())
    torch.cuda.synchronize()
    assert int(c.status) == tq.PAGED_BAD_SEQ
    served = owner >= 0
    assert torch.equal(q.cpu()[served], x.cpu()[served, :H])
    assert bool((q.cpu()[~served] == 7.0).all())
    for got, want in ((c.k, want_k), (c.v, want_v)):
        got = got.cpu()
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())


@pytest.mark.parametrize("what", SPOILT)
@pytest.mark.parametrize("seqs,at", WHERE)
@pytest.mark.parametrize("kind,cache", KINDS)
@pytest.mark.parametrize("D,H,KVH,each,room", [(96, 2, 1, 1, 0), (40, 4, 2, 3, 0), (64, 2, 1, 1, 0), (64, 8, 1, 3, WIDE)])
def test_attention_serves_the_other_sequences(tq, what, seqs, at, kind, cache, D, H, KVH, each, room):
    c = batch(seqs, each, kind, cache, D, H, KVH, room=room)
    want, most, vmax = c.want()
    h = c.handles(tq, max_q=each)
    _, owner = spoil(c, what, at)
    want[owner < 0] = 7.0
    got = c.attend(tq, handles=h)
    torch.cuda.synchronize()
    near(got, want, c.tolerance(most, vmax))
    assert int(c.status) == tq.PAGED_BAD_SEQ


@pytest.mark.parametrize("D", [64, 96, 40])
@pytest.mark.parametrize("seqs,at", [(3, 1), (3, 2), (40, 37), (100, 50)])
def test_a_bad_sequence_without_rows_is_reported(tq, D, seqs, at):
    """No row leads to it: append and attention record it all the same."""
    new = [0 if i == at else 1 for i in range(seqs)]
    total = [0 if i == at else 9 for i in range(seqs)]
    c = Case(new, total, 2, 1, D, 16, True, "f16", "f16", seed=seqs)
    want, most, vmax = c.want()
    c.len[at] = -4
    near(c.attend(tq), want, c.tolerance(most, vmax))
    assert int(c.status) == tq.PAGED_BAD_SEQ
    c.status.zero_()
    x = torch.ones(c.n, D, dtype=torch.float16, device="cuda")
    ch, b = c.handles(tq)
    tq.dev_paged_append(None, x.data_ptr(), x.data_ptr(), None, CODES["f16"], 0, 0, 0, D, D, 0, None, None, 0.0, 1e4, None,
                        ch, b, c.status.data_ptr())
    assert int(c.status) == tq.PAGED_BAD_SEQ
