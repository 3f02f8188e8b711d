"""Paged attention over keys and values that are not finite: every row against 64 bits, those
that see such a position too, whatever the number of new rows and the kernel that serves them."""
from __future__ import annotations

import math

import pytest
import torch

from paged_ref import Case
from test_gpu_paged import KINDS, WIDE, near

pytestmark = pytest.mark.gpu

# one new row (alone, or beside others), a few, and more than a block of the mma.sync kernel; the
# last goes to the tcgen05 kernel where the cache has 16 bits
ROWS = [([1], [40], 0), ([1], [900], 0), ([1, 1, 1], [5, 333, 70], 0), ([2, 1], [30, 50], 0), ([1, 20], [7, 200], 0),
        ([40, 1], [700, 66], WIDE)]


def spoil(c, seq, x, key=None, value=None):
    """KV head 0 of position x of sequence `seq`: an element of its key, of its value."""
    p = int(c.table_cpu[seq, x // c.page])
    if key is not None:
        c.kview[p, 0, x % c.page, 5] = key
    if value is not None:
        c.vview[p, 0, x % c.page, 7] = value


def same(got, want, tol):
    """Infinities and NaN where the definition has them, the rest within tol."""
    got = got.double().cpu()
    fine = torch.isfinite(want)
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got[~fine & ~want.isnan()], want[~fine & ~want.isnan()])
    near(got[fine], want[fine], tol)


def rows_of(c, seq):
    return slice(sum(c.new[:seq]), sum(c.new[:seq + 1]))


@pytest.mark.parametrize("kind,cache", KINDS)
@pytest.mark.parametrize("new,total,room", ROWS)
@pytest.mark.parametrize("H,KVH,D", [(8, 2, 64), (32, 8, 128), (2, 2, 96)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("whole", [False, True])
def test_a_key_that_weighs_nothing(tq, kind, cache, new, total, room, H, KVH, D, sign, whole):
    """An infinite element whose product with the query is -inf: weight 0, a finite result.  whole:
    a query element of one bit, of whose split the second part is 0."""
    c = Case(new, total, H, KVH, D, 16, True, kind, cache, seed=len(new) + D, room=room)
    _, most, vmax = c.want()
    seq = len(new) - 1
    mine = c.q_cpu[rows_of(c, seq)].view(-1, H, D)
    mine[:, :H // KVH, 5] = -sign * (torch.ones_like(mine[:, :H // KVH, 5]) if whole else mine[:, :H // KVH, 5].abs() + 0.25)
    spoil(c, seq, total[seq] // 2, key=sign * math.inf)
    c.upload()
    want, _, _ = c.want()
    assert torch.isfinite(want).all()
    same(c.attend(tq), want, c.tolerance(most + 1.0, vmax))
    assert int(c.status) == 0


@pytest.mark.parametrize("kind,cache", KINDS)
@pytest.mark.parametrize("new,total,room", ROWS + [([1], [1], 0)])
@pytest.mark.parametrize("H,KVH,D", [(8, 2, 64), (32, 8, 128), (2, 2, 96)])
@pytest.mark.parametrize("what", [math.inf, -math.inf, math.nan])
def test_a_value_that_is_not_finite(tq, kind, cache, new, total, room, H, KVH, D, what):
    """It makes one element of the rows that see it what the definition says, and no other."""
    c = Case(new, total, H, KVH, D, 16, True, kind, cache, seed=len(new) + D, room=room)
    _, most, vmax = c.want()
    seq = len(new) - 1
    spoil(c, seq, total[seq] // 2, value=what)
    c.upload()
    want, _, _ = c.want()
    # 0 * inf in the restatement: rows that do not see the position
    x, first = total[seq] // 2, total[seq] - new[seq]
    blind = max(0, x - first)
    clean = Case(new, total, H, KVH, D, 16, True, kind, cache, seed=len(new) + D, room=room).want()[0]
    r = rows_of(c, seq)
    want[r][:blind] = clean[r][:blind]
    assert int((~torch.isfinite(want)).sum()) == (new[seq] - blind) * (H // KVH)
    same(c.attend(tq), want, c.tolerance(most, vmax))
    assert int(c.status) == 0


@pytest.mark.parametrize("kind,cache", KINDS)
@pytest.mark.parametrize("new,total,room", ROWS)
@pytest.mark.parametrize("D", [64, 128])
def test_a_nan_key_spoils_its_own_heads(tq, kind, cache, new, total, room, D):
    c = Case(new, total, 8, 2, D, 16, True, kind, cache, seed=len(new) + D, room=room)
    clean, most, vmax = c.want()
    seq = len(new) - 1
    spoil(c, seq, total[seq] // 2, key=math.nan)
    c.upload()
    want, _, _ = c.want()
    r, blind = rows_of(c, seq), max(0, total[seq] // 2 - (total[seq] - new[seq]))
    want[r][:blind] = clean[r][:blind]
    same(c.attend(tq), want, c.tolerance(most, vmax))


@pytest.mark.parametrize("kind,cache", [("bf16", "bf16"), ("f32", "f16")])
def test_rows_computed_again_for_long_do_not_touch_other_sequences(tq, kind, cache):
    """One sequence's infinity among 262 thousand positions.  Its 32 rows belong to one warp, whose passes
    over what they see (0.2 us a position and row: 1.6 s) outlast the limit of the kernel's waits (2e9
    clocks, 1.0 s), so they must not run beside them.  The rows of the sequences that the same
    CTAs serve after it stay right, and nothing is reported.

    Every sequence's page table names one page over and over (the first of sequence 0 its copy with the
    infinity), so row i of n sees each of the page's positions N / P times, the last n - 1 - i of them
    once less: the softmax of the page's scores with these counts.

    Bound: N / 16 products in the tensor core, each cut by less than 2^-23 of the running sum, and
    N / 64 fp32 additions of the weights' sum, beside what short contexts have."""
    H, D, P, N, seqs = 16, 64, 64, 1 << 18, 200
    new = [2] + [3] * (seqs - 1)
    c = Case(new, [n + 61 for n in new], H, 1, D, P, True, kind, cache, seed=3, spare=0)
    _, most, vmax = c.want()
    c.pool = 2
    g = torch.Generator().manual_seed(4)
    c.k_cpu, c.v_cpu = (torch.randn(1, 1, P, D, generator=g).to(c.k_cpu.dtype).repeat(2, 1, 1, 1) for _ in range(2))
    k, v = c.k_cpu[0, 0].double(), c.v_cpu[0, 0].double()
    c.v_cpu[1, 0, 3, 7] = math.inf
    c.table_cpu = torch.zeros(seqs, N // P, dtype=torch.int32)
    c.table_cpu[0, 0] = 1
    c.total = [N] * seqs
    c.upload()
    got = c.attend(tq).double().cpu()
    torch.cuda.synchronize()
    assert int(c.status) == 0
    q = c.q_cpu[:, :H * D].double().view(c.n, H, D)
    count = torch.full((c.n, P), float(N // P), dtype=torch.float64)
    row = 0
    for n in new:
        for i in range(n):
            count[row, P - (n - 1 - i):] -= 1
            row += 1
    s = torch.einsum("rhd,xd->rhx", q, k) * c.scale
    w = (s - s.amax(-1, keepdim=True)).exp() * count[:, None]
    want = torch.einsum("rhx,xd->rhd", w / w.sum(-1, keepdim=True), v).reshape(c.n, H * D)
    want[:2].view(2, H, D)[..., 7] = math.inf
    c.total = [P] * seqs  # the bound's terms of one page
    same(got, want, c.tolerance(max(most, float(s.abs().max())), float(v.abs().max())) +
         float(v.abs().max()) * (N / 16 * 2.0 ** -23 + N / 64 * 2.0 ** -24))


def test_an_early_infinity_in_a_long_chunk(tq):
    """Every row of a chunk sees it: element 7 is infinite, the others as without it."""
    for kind, cache in (("bf16", "bf16"), ("f32", "f16")):
        c = Case([256], [4096], 8, 2, 128, 16, True, kind, cache, seed=6, room=WIDE)
        clean, most, vmax = c.want()
        spoil(c, 0, 100, value=math.inf)
        c.upload()
        want = clean.clone()
        want.view(256, 8, 128)[:, :4, 7] = math.inf
        same(c.attend(tq), want, c.tolerance(most, vmax))


@pytest.mark.parametrize("kind,cache", [("bf16", "bf16"), ("f16", "f16"), ("f32", "f16")])
@pytest.mark.parametrize("D", [64, 128])
def test_shared_items_computed_again_leave_the_workspace_ready(tq, kind, cache, D):
    """Items that several CTAs share, some of whose parts come out not finite: their tickets are taken
    late.  The call repeats bit for bit, in a graph too, and the next calls find the workspace ready."""
    new, total, at = [90, 60, 17], [2500, 700, 3000], {0: 100, 2: 2990}
    c = Case(new, total, 8, 2, D, 16, True, kind, cache, seed=8, room=WIDE)
    h = c.handles(tq)
    w = c.workspace(tq, *h)
    first = c.attend(tq, work=w, handles=h).clone()
    clean, most, vmax = c.want()
    near(first, clean, c.tolerance(most, vmax))
    finite = c.v.clone()
    for seq, x in at.items():
        spoil(c, seq, x, value=math.inf)
    want = clean.clone()
    for seq, x in at.items():
        r = rows_of(c, seq)
        blind = max(0, x - (total[seq] - new[seq]))
        want[r][blind:].view(-1, 8, D)[:, :4, 7] = math.inf
    c.v.copy_(c.v_cpu.to(c.v.device))
    again = c.attend(tq, work=w, handles=h).clone()
    same(again, want, c.tolerance(most, vmax))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        c.attend(tq, work=w, handles=h)
    for _ in range(3):
        c.obuf.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(c.out().view(torch.uint8), again.view(torch.uint8))
    c.v.copy_(finite)
    c.obuf.fill_(7.0)
    assert torch.equal(c.attend(tq, work=w, handles=h), first)
    assert int(c.status) == 0


@pytest.mark.parametrize("seqs", [40, 500])
@pytest.mark.parametrize("kind,cache", [("bf16", "bf16"), ("f32", "f16")])
def test_rows_computed_again_among_many_sequences(tq, kind, cache, seqs):
    """The second look finds its way through more sequences than a warp's lanes, than a CTA's threads."""
    new = [0 if i % 7 == 3 else 5 for i in range(seqs)]
    total = [n + 9 + (i * 37) % 120 for i, n in enumerate(new)]
    c = Case(new, total, 8, 2, 64, 16, True, kind, cache, pad=1, seed=seqs, room=WIDE)
    want, most, vmax = c.want()
    for seq in (0, 2, seqs // 2, seqs - 1):
        if new[seq]:
            spoil(c, seq, 3, value=math.inf)
            want[rows_of(c, seq)].view(-1, 8, 64)[:, :4, 7] = math.inf
    c.upload()
    same(c.attend(tq), want, c.tolerance(most, vmax))
    assert int(c.status) == 0
