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
