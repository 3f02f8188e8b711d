"""Paged-cache operators on the GPU against their definitions in 64 bits: types, head layouts,
page sizes, ragged and empty sequences, what lies in masked places, streams and graphs, and a
run of append and attention together."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from paged_ref import CODES, TYPES, Case, turn_tolerance, turned

pytestmark = pytest.mark.gpu

KINDS = [("f32", "f32"), ("f32", "f16"), ("f16", "f16"), ("bf16", "bf16")]
SIXTEEN = KINDS[1:]   # caches that the tcgen05 kernel reads
WIDE = 1 << 21        # positions of a table that is wide enough for it whatever the rows


def near(got, want, tol, same_nan=False):
    got, want = got.double().cpu(), want.double()
    if same_nan:
        assert torch.equal(got.isnan(), want.isnan())
        got, want = got[~want.isnan()], want[~want.isnan()]
    assert torch.isfinite(got).all()
    if not got.numel():
        return
    d = (got - want).abs()
    tol = torch.as_tensor(tol, dtype=torch.float64).expand_as(d)
    worst = (d - tol).argmax()
    assert bool((d <= tol).all()), f"{float(d.flatten()[worst]):.3g} off, {float(tol.flatten()[worst]):.3g} allowed"


def check(c, tq, drop=(), **kw):
    got = c.attend(tq, **kw)
    torch.cuda.synchronize()
    want, most, vmax = c.want(drop)
    near(got, want, c.tolerance(most, max(vmax, 1e-3)))
    return got


# ------------------------------------------------------------------ attention
SHAPES = [(32, 8, 128), (14, 2, 64), (16, 8, 128), (4, 4, 64), (8, 1, 128), (40, 2, 64)]


@pytest.mark.parametrize("kind,cache", KINDS)
@pytest.mark.parametrize("H,KVH,D", SHAPES)
@pytest.mark.parametrize("page,first", [(16, True), (5, False), (128, True), (1, False)])
def test_single_tokens(tq, kind, cache, H, KVH, D, page, first):
    total = [1, 300, 16, 17, 64, 129, 2]
    c = Case([1] * len(total), total, H, KVH, D, page, first, kind, cache, pad=2, seed=page + D)
    check(c, tq)
    assert int(c.status) == 0


@pytest.mark.parametrize("kind,cache", KINDS)
@pytest.mark.parametrize("H,KVH,D", SHAPES)
@pytest.mark.parametrize("page,first", [(16, False), (24, True), (1, True)])
def test_chunks(tq, kind, cache, H, KVH, D, page, first):
    new, total = [37, 1, 130, 5], [37, 90, 261, 5]
    c = Case(new, total, H, KVH, D, page, first, kind, cache, pad=1, seed=page + H)
    check(c, tq)
    assert int(c.status) == 0


@pytest.mark.parametrize("kind,cache", KINDS)
@pytest.mark.parametrize("new,total", [([2], [2]), ([3, 3], [3, 200]), ([4, 1, 2], [40, 1, 33]), ([16], [600])])
@pytest.mark.parametrize("H,KVH,D", [(32, 8, 128), (14, 2, 64), (5, 5, 64)])
def test_a_few_tokens_at_a_time(tq, kind, cache, new, total, H, KVH, D):
    check(Case(new, total, H, KVH, D, 16, True, kind, cache, seed=sum(total)), tq)


@pytest.mark.parametrize("kind,cache", KINDS)
@pytest.mark.parametrize("H,KVH,D", [(4, 4, 96), (6, 1, 256), (2, 2, 8), (3, 3, 40)])
def test_other_head_dims(tq, kind, cache, H, KVH, D):
    check(Case([3, 1], [20, 77], H, KVH, D, 16, False, kind, cache, seed=D), tq)


@pytest.mark.parametrize("kind,cache", KINDS)
@pytest.mark.parametrize("new,total", [
    ([0, 1, 0, 4], [0, 9, 12, 30]),   # sequences without rows, without positions
    ([5, 3], [2, 0]),                 # more rows than positions: rows that see nothing
    ([1, 0, 0], [0, 0, 0]),           # nothing at all
    ([200, 1], [100, 1]),
])
def test_empty_rows_and_sequences(tq, kind, cache, new, total):
    c = Case(new, total, 8, 2, 64, 16, True, kind, cache, pad=3, seed=5)
    got = check(c, tq)
    assert torch.equal(got[sum(new):].float(), torch.full_like(got[sum(new):].float(), 7.0))
    assert int(c.status) == 0


@pytest.mark.parametrize("kind,cache", KINDS)
@pytest.mark.parametrize("shift,gap", [(0, 64), (0, 8), (1, 0), (3, 1)])
@pytest.mark.parametrize("new,total", [([1, 1], [70, 3]), ([40, 2], [50, 60])])
def test_strides_and_alignment(tq, kind, cache, shift, gap, new, total):
    """q and out as a part of wider rows, and off 16 bytes; what lies between rows is kept."""
    c = Case(new, total, 8, 2, 64, 16, True, kind, cache, shift=shift, gap=gap, seed=9)
    check(c, tq)
    rows = c.obuf[shift:shift + c.n * c.qw].view(c.n, c.qw)
    assert bool((rows[:, c.H * c.D:] == 7.0).all()) and bool((c.obuf[shift + c.n * c.qw:] == 7.0).all())


@pytest.mark.parametrize("kind,cache", KINDS)
@pytest.mark.parametrize("new", [1, 3, 150])
def test_large_scores(tq, kind, cache, new):
    """Scores far apart (one position holds nearly all the weight, late or early)."""
    check(Case([new], [300], 8, 2, 64, 16, True, kind, cache, qk=4.0, seed=3), tq)


@pytest.mark.parametrize("kind,cache", KINDS)
@pytest.mark.parametrize("new,total,x", [(4, 40, 38), (150, 200, 120), (150, 200, 199), (2, 3, 2), (130, 700, 571)])
@pytest.mark.parametrize("H,KVH,D", [(8, 2, 64), (8, 2, 128)])
@pytest.mark.parametrize("what", [math.nan, math.inf])
def test_non_finite_values_reach_only_the_rows_that_see_them(tq, kind, cache, new, total, x, H, KVH, D, what):
    c = Case([new], [total], H, KVH, D, 16, True, kind, cache, seed=x)
    want, most, vmax = c.want()
    p = int(c.table_cpu[0, x // 16])
    c.kview[p, 0, x % 16, 5] = what
    c.vview[p, 0, x % 16, 7] = what
    c.upload()
    got = c.attend(tq).double().cpu()
    torch.cuda.synchronize()
    blind = max(0, x - (total - new))  # rows before position x
    near(got[:blind], want[:blind], c.tolerance(most, vmax))
    half = (H // KVH) * D              # the other KV head's queries
    near(got[:, half:], want[:, half:], c.tolerance(most, vmax))
    assert bool(got[blind:, 7].isnan().any() or not torch.isfinite(got[blind:, 7]).all())


@pytest.mark.parametrize("kind,cache", KINDS)
@pytest.mark.parametrize("new", [1, 100])
def test_a_non_finite_query_spoils_its_own_row_only(tq, kind, cache, new):
    c = Case([new, 1], [150, 20], 8, 2, 64, 16, True, kind, cache, seed=2)
    want, most, vmax = c.want()
    c.q_cpu[0, 3] = math.nan
    c.upload()
    got = c.attend(tq).double().cpu()
    torch.cuda.synchronize()
    assert bool(got[0, :64].isnan().all())
    near(got[0, 64:], want[0, 64:], c.tolerance(most, vmax))
    near(got[1:], want[1:], c.tolerance(most, vmax))


@pytest.mark.parametrize("kind,cache", KINDS)
@pytest.mark.parametrize("new,total", [([1, 1], [60, 33]), ([70, 2], [90, 33])])
@pytest.mark.parametrize("page_id", [-1, 1 << 30, -(1 << 31)])
def test_bad_pages_are_masked_and_reported(tq, kind, cache, new, total, page_id):
    c = Case(new, total, 8, 2, 64, 16, True, kind, cache, seed=4)
    c.table_cpu[0, 1] = page_id
    c.upload()
    check(c, tq, drop={(0, x) for x in range(16, 32)})
    assert int(c.status) == tq.PAGED_BAD_PAGE


@pytest.mark.parametrize("kind,cache", KINDS)
@pytest.mark.parametrize("what", ["len over the table", "len negative", "rows past n_tokens", "rows decreasing",
                                  "more rows than max_q_len", "negative start"])
@pytest.mark.parametrize("new", [1, 60])
def test_bad_sequences_are_skipped_and_reported(tq, kind, cache, what, new):
    c = Case([new, new, new], [70, 80, 90], 8, 2, 64, 16, True, kind, cache, seed=6)
    want, most, vmax = c.want()
    c_, b = c.handles(tq)
    rows = slice(0, new)  # the sequence that is spoilt
    if what == "len over the table":
        c.len[0] = c.table.shape[1] * 16 + 1
    elif what == "len negative":
        c.len[0] = -5
    elif what == "rows past n_tokens":
        rows = slice(2 * new, 3 * new)
        c.start[3] = 3 * new + 1
    elif what == "rows decreasing":
        rows = slice(0, 2 * new)
        c.start[1] = 3 * new + 1  # the first past its end, the second backwards
    elif what == "more rows than max_q_len":
        rows = slice(0, 2 * new)
        c.start[1] = 2 * new
    else:
        c.start[0] = -1
    got = c.attend(tq, handles=(c_, b)).double().cpu()
    torch.cuda.synchronize()
    assert int(c.status) == tq.PAGED_BAD_SEQ
    want[rows] = 7.0
    near(got, want, c.tolerance(most, vmax))


@pytest.mark.parametrize("room", [0, WIDE])
def test_rows_where_none_were_announced(tq, room):
    c = Case([1, 2], [9, 30], 8, 2, 64, 16, True, "f16", "f16", room=room)
    got = c.attend(tq, handles=c.handles(tq, max_q=0))
    assert int(c.status) == tq.PAGED_BAD_SEQ and bool((got == 7.0).all())


@pytest.mark.parametrize("kind,cache", KINDS)
@pytest.mark.parametrize("new", [1, 90])
def test_calls_repeat_bit_for_bit_and_leave_the_workspace_ready(tq, kind, cache, new):
    c = Case([new] * 3, [2500, 700, 91], 8, 2, 64, 16, True, kind, cache, seed=8)
    h = c.handles(tq)
    w = c.workspace(tq, *h)
    first = c.attend(tq, work=w, handles=h).clone()
    for _ in range(5):
        c.obuf.fill_(7.0)
        assert torch.equal(c.attend(tq, work=w, handles=h), first)
    other = Case([1, 2], [1000, 1500], 8, 2, 64, 16, True, kind, cache, seed=1)
    if other.workspace(tq, *other.handles(tq)).numel() <= w.numel():
        check(other, tq, work=w)
    c.obuf.fill_(7.0)
    assert torch.equal(c.attend(tq, work=w, handles=h), first)


@pytest.mark.parametrize("kind,cache", KINDS)
@pytest.mark.parametrize("new", [1, 80])
def test_a_captured_call_follows_lengths_and_tables(tq, kind, cache, new):
    """Captured once, replayed with other lengths, pages and queries."""
    c = Case([new, new], [300, 90], 8, 2, 64, 16, True, kind, cache, seed=11)
    h = c.handles(tq)
    w = c.workspace(tq, *h)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        c.attend(tq, work=w, handles=h)
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        c.attend(tq, work=w, handles=h)
    for lens in ([300, 90], [new + 1, 90], [250, new]):
        c.total = lens
        c.len.copy_(torch.tensor(lens, dtype=torch.int32))
        c.obuf.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        want, most, vmax = c.want()
        near(c.out(), want, c.tolerance(most, vmax))


def test_two_streams_with_a_workspace_each(tq):
    a = Case([1, 1], [900, 40], 8, 2, 128, 16, True, "bf16", "bf16", seed=1)
    b = Case([70], [300], 8, 2, 128, 16, True, "bf16", "bf16", seed=2)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    work = [x.workspace(tq, *x.handles(tq)) for x in (a, b)]
    torch.cuda.synchronize()
    for _ in range(20):
        for x, w, s in zip((a, b), work, streams):
            x.attend(tq, work=w, stream=s.cuda_stream)
    torch.cuda.synchronize()
    for x in (a, b):
        want, most, vmax = x.want()
        near(x.out(), want, x.tolerance(most, vmax))


@pytest.mark.parametrize("kind,cache,new", [("f16", "f16", 1), ("f16", "f16", 40), ("f32", "f32", 1)])
def test_offsets_past_32_bits(tq, kind, cache, new):
    """Pages far apart in one large allocation: element offsets above 2^32."""
    c = Case([new], [120], 4, 2, 64, 16, True, kind, cache, seed=3)
    far = (1 << 32) // (c.pool - 1) // 16 * 16 + 4096
    dt = TYPES[cache]
    big = torch.zeros(far * c.pool + 4096, dtype=dt, device="cuda")
    n = c.KVH * c.page * c.D
    at = n
    for p in range(c.pool):
        big[p * far:p * far + n] = c.k[p].reshape(-1)
        big[p * far + at:p * far + at + n] = c.v[p].reshape(-1)
    ch, b = c.handles(tq)
    ch.k, ch.v, ch.page_stride = big.data_ptr(), big.data_ptr() + at * big.element_size(), far
    assert far * (c.pool - 1) >= 1 << 32
    check(c, tq, handles=(ch, b))


def test_a_host_pointer_is_refused(tq):
    c = Case([1], [5], 4, 2, 64, 16, True, "f32", "f32")
    ch, b = c.handles(tq)
    host = torch.zeros(4, dtype=torch.int32)
    b.kv_len = host.data_ptr()
    with pytest.raises(tq.TQB200Error, match="kv_len is not device memory"):
        c.attend(tq, handles=(ch, b))


def test_matches_the_contiguous_decode_attention(tq):
    """One sequence whose pages lie in order holds the cache of tqb200_attention_decode: each
    is within its own tolerance of the other."""
    H, KVH, D, n, most = 32, 8, 128, 333, 352
    rng = np.random.default_rng(0)
    q = rng.normal(size=H * D).astype(np.float32)
    kc, vc = (rng.normal(size=(KVH, most, D)).astype(np.float32) for _ in range(2))
    want = tq.attention_decode(q, kc, vc, n, most, H, KVH, D, 1.0 / math.sqrt(D))
    c = Case([1], [n], H, KVH, D, most, True, "f32", "f32", spare=0)
    c.k_cpu, c.v_cpu = torch.tensor(kc)[None], torch.tensor(vc)[None]
    c.kview, c.vview = c.k_cpu, c.v_cpu
    c.q_cpu = torch.tensor(q)[None]
    c.upload()
    got = c.attend(tq).cpu().numpy().reshape(-1)
    _, m, vmax = c.want()
    assert np.abs(got - want).max() <= 2 * c.tolerance(m, vmax)


# ------------------------------------------------------------------ the tcgen05 kernel on small cases
@pytest.mark.parametrize("kind,cache", SIXTEEN)
@pytest.mark.parametrize("H,KVH,D", SHAPES + [(130, 1, 64), (300, 1, 128)])
@pytest.mark.parametrize("page,first", [(16, False), (24, True), (1, True), (64, True), (128, False), (8, True)])
def test_chunks_on_tcgen05(tq, kind, cache, H, KVH, D, page, first):
    new, total = [37, 1, 130, 17], [37, 90, 261, 64]
    c = Case(new, total, H, KVH, D, page, first, kind, cache, pad=1, seed=page + H, room=WIDE)
    check(c, tq)
    assert int(c.status) == 0


@pytest.mark.parametrize("kind,cache", SIXTEEN)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page,first", [(40, False), (48, True), (96, False), (192, True), (72, True)])
def test_pages_that_tiles_do_not_divide_on_tcgen05(tq, kind, cache, D, page, first):
    """Pages that begin and end inside a tile of 64 positions."""
    new, total = [33, 1, 70, 20], [400, 257, 641, 192]
    c = Case(new, total, 8, 2, D, page, first, kind, cache, pad=1, seed=page + D, room=WIDE)
    check(c, tq)
    assert int(c.status) == 0


@pytest.mark.parametrize("kind,cache", SIXTEEN)
@pytest.mark.parametrize("new,total", [
    ([0, 20, 0, 40], [0, 29, 12, 60]), ([50, 30], [20, 0]), ([17, 0, 0], [0, 0, 0]), ([200, 17], [100, 17]),
    ([64], [64]), ([64], [128]), ([65], [129]), ([63], [65]), ([300], [300])])
def test_lengths_on_tcgen05(tq, kind, cache, new, total):
    c = Case(new, total, 8, 2, 128, 16, True, kind, cache, pad=3, seed=5, room=WIDE)
    got = check(c, tq)
    assert torch.equal(got[sum(new):].float(), torch.full_like(got[sum(new):].float(), 7.0))


@pytest.mark.parametrize("kind,cache", SIXTEEN)
@pytest.mark.parametrize("gap,qk", [(8, 1.0), (64, 1.0), (0, 4.0)])
def test_strides_and_large_scores_on_tcgen05(tq, kind, cache, gap, qk):
    c = Case([100, 40], [300, 60], 8, 2, 64, 16, True, kind, cache, gap=gap, qk=qk, seed=9, room=WIDE)
    check(c, tq)
    rows = c.obuf[:c.n * c.qw].view(c.n, c.qw)
    assert bool((rows[:, c.H * c.D:] == 7.0).all()) and bool((c.obuf[c.n * c.qw:] == 7.0).all())


@pytest.mark.parametrize("kind,cache", SIXTEEN)
@pytest.mark.parametrize("new,total,x", [(150, 200, 120), (150, 200, 199), (130, 700, 571), (20, 900, 30)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("what", [math.nan, math.inf])
def test_non_finite_values_on_tcgen05(tq, kind, cache, new, total, x, D, what):
    c = Case([new], [total], 8, 2, D, 16, True, kind, cache, seed=x, room=WIDE)
    want, most, vmax = c.want()
    p = int(c.table_cpu[0, x // 16])
    c.kview[p, 0, x % 16, 5] = what
    c.vview[p, 0, x % 16, 7] = what
    c.upload()
    got = c.attend(tq).double().cpu()
    torch.cuda.synchronize()
    blind = max(0, x - (total - new))
    near(got[:blind], want[:blind], c.tolerance(most, vmax))
    half = 4 * D
    near(got[:, half:], want[:, half:], c.tolerance(most, vmax))
    assert not torch.isfinite(got[blind:, 7]).all()


@pytest.mark.parametrize("kind,cache", SIXTEEN)
@pytest.mark.parametrize("page_id", [-1, 1 << 30])
def test_bad_pages_and_sequences_on_tcgen05(tq, kind, cache, page_id):
    c = Case([70, 20, 30], [290, 33, 90], 8, 2, 64, 16, True, kind, cache, seed=4, room=WIDE)
    c.table_cpu[0, 1] = page_id
    c.upload()
    drop = {(0, x) for x in range(16, 32)}
    check(c, tq, drop=drop)
    assert int(c.status) == tq.PAGED_BAD_PAGE
    want, most, vmax = c.want(drop)
    c.obuf.fill_(7.0)
    c.status.zero_()
    c.len[1] = -1
    got = c.attend(tq).double().cpu()
    want[70:90] = 7.0
    near(got, want, c.tolerance(most, vmax))
    assert int(c.status) in (tq.PAGED_BAD_SEQ, tq.PAGED_BAD_PAGE)


@pytest.mark.parametrize("kind,cache", SIXTEEN)
@pytest.mark.parametrize("D", [64, 128])
def test_a_prompt_from_its_beginning(tq, kind, cache, D):
    """Whole items, one query tile each: a table with room for the prompt only."""
    c = Case([400, 211], [400, 230], 16, 4, D, 16, True, kind, cache, seed=D)
    check(c, tq)


@pytest.mark.parametrize("new,total", [
    ([0, 200, 0, 40], [0, 290, 12, 60]), ([170, 30], [120, 0]), ([200, 170], [100, 170]), ([641], [641]),
    ([129], [1290]), ([65, 90, 1], [4000, 3333, 700])])
@pytest.mark.parametrize("H,KVH", [(8, 2), (7, 1), (4, 4)])
def test_one_query_tile_per_item(tq, new, total, H, KVH):
    """fp32 over fp16 with head_dim 128 and a table of some thousand positions."""
    c = Case(new, total, H, KVH, 128, 16, True, "f32", "f16", pad=3, seed=len(new) + H, room=4096)
    first = check(c, tq).clone()
    assert torch.equal(first[sum(new):], torch.full_like(first[sum(new):], 7.0))
    assert torch.equal(c.attend(tq)[:sum(new)], first[:sum(new)])


@pytest.mark.parametrize("what", [math.nan, math.inf, -1])
def test_masked_places_with_one_query_tile_per_item(tq, what):
    new, total, x = 150, 900, 810
    c = Case([new], [total], 8, 2, 128, 16, True, "f32", "f16", seed=3, room=4096)
    if what == -1:  # a bad page
        c.table_cpu[0, x // 16] = -1
        c.upload()
        check(c, tq, drop={(0, y) for y in range(x // 16 * 16, x // 16 * 16 + 16)})
        assert int(c.status) == tq.PAGED_BAD_PAGE
        return
    want, most, vmax = c.want()
    p = int(c.table_cpu[0, x // 16])
    c.kview[p, 0, x % 16, 5] = what
    c.vview[p, 0, x % 16, 7] = what
    c.upload()
    got = c.attend(tq).double().cpu()
    blind = x - (total - new)
    near(got[:blind], want[:blind], c.tolerance(most, vmax))
    near(got[:, 4 * 128:], want[:, 4 * 128:], c.tolerance(most, vmax))
    assert not torch.isfinite(got[blind:, 7]).all()


@pytest.mark.parametrize("kind,cache", SIXTEEN)
def test_tcgen05_calls_repeat_and_follow_a_graph(tq, kind, cache):
    """Items split over CTAs and joined: bit for bit the same every time, whatever other call used
    the workspace in between; captured and replayed with other lengths."""
    c = Case([90, 60, 17], [2500, 700, 3000], 8, 2, 128, 16, True, kind, cache, seed=8, room=WIDE)
    h = c.handles(tq)
    w = c.workspace(tq, *h)
    first = check(c, tq, work=w, handles=h).clone()
    other = Case([1, 1], [1000, 1500], 8, 2, 64, 16, True, kind, cache, seed=1)
    for _ in range(4):
        c.obuf.fill_(7.0)
        assert torch.equal(c.attend(tq, work=w, handles=h), first)
        check(other, tq, work=w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        c.attend(tq, work=w, handles=h)
    for lens in ([2500, 700, 3000], [90, 500, 17], [1111, 60, 2999]):
        c.total = lens
        c.len.copy_(torch.tensor(lens, dtype=torch.int32))
        c.obuf.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        want, most, vmax = c.want()
        near(c.out(), want, c.tolerance(most, vmax))


@pytest.mark.parametrize("cache,room,new", [("f16", WIDE, 64), ("f16", 0, 1), ("f32", 0, 1), ("f32", 0, 20)])
def test_fp32_results_keep_their_precision_over_long_contexts(tq, cache, room, new):
    """Tensor-core sums are cut, not rounded, so an error that grows with the context shows in the
    2-norm.  Bound: sums of at most 8 tiles of 8 products, each cut by less than 2^-24 of the sum
    (64), the scores' 16 products likewise, splits to 2^-21 twice, and as much again for what
    fp32 additions round at random: 2 * (80 * 2^-24 + 2 * 2^-21) / 2 on average half of it."""
    c = Case([new], [12000], 2, 1, 128, 16, True, "f32", cache, qk=1.0, seed=1, room=room)
    got = c.attend(tq).double().cpu()
    want, _, _ = c.want()
    assert float((got - want).norm() / want.norm()) <= 80 * 2.0 ** -24 + 2 * 2.0 ** -21


@pytest.mark.parametrize("kind,cache", KINDS)
@pytest.mark.parametrize("seqs,new", [(33, 1), (150, 1), (300, 1), (40, 6), (140, 3)])
def test_many_sequences(tq, kind, cache, seqs, new):
    """More sequences than a warp's lanes, than a CTA's threads; some without rows."""
    new = [0 if i % 7 == 3 else new for i in range(seqs)]
    total = [n + (i * 37) % 90 for i, n in enumerate(new)]
    for room in (0, WIDE):
        c = Case(new, total, 8, 2, 64, 16, True, kind, cache, pad=1, seed=seqs, room=room)
        check(c, tq)
        assert int(c.status) == 0


# ------------------------------------------------------------------ norms and rotation
def rope_inputs(n, H, KVH, D, kind, seed, gap=0, far=200000):
    g = torch.Generator().manual_seed(seed)
    qkv = (torch.randn(n, (H + 2 * KVH) * D + gap, generator=g) * 3).to(TYPES[kind])
    w = [1 + 0.3 * torch.randn(D, generator=g) for _ in range(2)]
    pos = torch.randint(-5, far, (n,), generator=g, dtype=torch.int32)
    return qkv, w, pos


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,KVH,D,rotary", [(32, 8, 128, 128), (14, 2, 64, 64), (5, 5, 64, 16), (4, 1, 256, 64),
                                           (3, 1, 96, 48), (2, 2, 8, 2), (32, 4, 128, 32), (2, 1, 128, 0), (3, 0, 64, 64),
                                           (0, 3, 64, 64), (2, 2, 64, 6)])
@pytest.mark.parametrize("n", [1, 7, 300])
@pytest.mark.parametrize("norm", [True, False])
def test_norm_and_rotation(tq, kind, H, KVH, D, rotary, n, norm):
    qkv, w, pos = rope_inputs(n, H, KVH, D, kind, seed=n + D)
    dev, (wq, wk), p = qkv.cuda(), [x.cuda() for x in w], pos.cuda()
    q = torch.full((n, max(1, H), D), 7.0, dtype=TYPES[kind], device="cuda")
    k = torch.full((n, max(1, KVH), D), 7.0, dtype=TYPES[kind], device="cuda")
    width, size = qkv.shape[1], qkv.element_size()
    tq.dev_qk_norm_rope(dev.data_ptr(), dev.data_ptr() + H * D * size, q.data_ptr(), k.data_ptr(), CODES[kind], n, H, KVH,
                        D, rotary, width, width, H * D, KVH * D, wq.data_ptr() if norm else None,
                        wk.data_ptr() if norm else None, 1e-6, 1e6, p.data_ptr() if rotary else None)
    torch.cuda.synchronize()
    rows = qkv[:, :(H + 2 * KVH) * D].view(n, H + 2 * KVH, D)
    for got, x, ww in ((q, rows[:, :H], w[0]), (k, rows[:, H:H + KVH], w[1])):
        if x.shape[1]:
            want = turned(x, ww if norm else None, pos, rotary, 1e6, 1e-6)
            near(got, want, turn_tolerance(want, kind, norm))
        else:
            assert bool((got == 7.0).all())


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D,rotary,gap,shift", [(64, 64, 0, 0), (128, 32, 8, 0), (64, 64, 3, 0), (64, 64, 0, 1)])
def test_norm_and_rotation_in_place(tq, kind, D, rotary, gap, shift):
    """In place within a fused projection's rows (the value part is kept), aligned or not."""
    n, H, KVH = 33, 6, 2
    qkv, w, pos = rope_inputs(n, H, KVH, D, kind, seed=D, gap=gap)
    width, size = qkv.shape[1], qkv.element_size()
    buf = torch.zeros(n * width + 8, dtype=TYPES[kind], device="cuda")
    buf[shift:shift + n * width] = qkv.cuda().reshape(-1)
    (wq, wk), p = [x.cuda() for x in w], pos.cuda()
    at = buf.data_ptr() + shift * size
    tq.dev_qk_norm_rope(at, at + H * D * size, at, at + H * D * size, CODES[kind], n, H, KVH, D, rotary, width, width,
                        width, width, wq.data_ptr(), wk.data_ptr(), 1e-6, 1e4, p.data_ptr())
    torch.cuda.synchronize()
    got = buf[shift:shift + n * width].view(n, width).cpu()
    rows = qkv[:, :(H + 2 * KVH) * D].view(n, H + 2 * KVH, D)
    want = torch.cat([turned(rows[:, :H], w[0], pos, rotary, 1e4, 1e-6),
                      turned(rows[:, H:H + KVH], w[1], pos, rotary, 1e4, 1e-6)], 1)
    near(got[:, :(H + KVH) * D].reshape(want.shape), want, turn_tolerance(want, kind, True))
    assert torch.equal(got[:, (H + KVH) * D:], qkv[:, (H + KVH) * D:])


def test_a_position_turns_by_its_own_angle(tq):
    """Far positions keep their phase: the unit vector's angle at 2^31 - 1, against 64 bits."""
    pos = torch.tensor([0, 1, 12345, 1 << 20, (1 << 31) - 1, -(1 << 31)], dtype=torch.int32)
    x = torch.zeros(len(pos), 64)
    x[:, :32] = 1.0
    d, p = x.cuda(), pos.cuda()
    tq.dev_qk_norm_rope(d.data_ptr(), None, d.data_ptr(), None, 0, len(pos), 1, 0, 64, 64, 64, 0, 64, 0, None, None, 0.0,
                        1e4, p.data_ptr())
    torch.cuda.synchronize()
    f = torch.tensor([1e4 ** (-i / 32) for i in range(32)], dtype=torch.float64)
    a = pos.double()[:, None] * f
    # fp32: 4 roundings of a value up to 1 and the angle's own 4 * 2^-24; the frequency's and the
    # product's 64-bit roundings, 8 of 2^-53 of the angle each
    tol = 8 * 2.0 ** -24 + a.abs() * 8 * 2.0 ** -53
    near(d[:, :32], torch.cos(a), tol)
    near(d[:, 32:], torch.sin(a), tol)


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("kind,cache", KINDS)
@pytest.mark.parametrize("H,KVH,D,rotary,norm", [(32, 8, 128, 128, True), (14, 2, 64, 64, False), (0, 3, 64, 16, True),
                                                (3, 1, 96, 96, True), (2, 2, 40, 0, False), (4, 2, 256, 64, True)])
@pytest.mark.parametrize("new,total,page,first", [([1] * 5, [1, 17, 16, 300, 2], 16, True),
                                                  ([40, 0, 3, 1], [40, 9, 70, 1], 5, False),
                                                  ([6, 2], [3, 0], 1, True), ([70], [128], 64, False)])
@pytest.mark.parametrize("shift", [0, 1])
def test_append(tq, kind, cache, H, KVH, D, rotary, norm, new, total, page, first, shift):
    c = Case(new, total, max(H, KVH), KVH, D, page, first, kind, cache, pad=2, seed=D + page)
    n = c.n
    qkv, w, pos = rope_inputs(n, H, KVH, D, kind, seed=7)
    width, size = qkv.shape[1], qkv.element_size()
    buf = torch.zeros(n * width + 8, dtype=TYPES[kind], device="cuda")
    buf[shift:shift + n * width] = qkv.cuda().reshape(-1)
    qo = torch.full((n, max(1, H), D), 7.0, dtype=TYPES[kind], device="cuda")
    (wq, wk), own = [x.cuda() for x in w], pos.cuda()
    use_own = page == 16  # rotary positions other than the cache's
    ch, b = c.handles(tq)
    at = buf.data_ptr() + shift * size
    tq.dev_paged_append(at if H else None, at + H * D * size, at + (H + KVH) * D * size, qo.data_ptr() if H else None,
                        CODES[kind], H, rotary, width, width, width, H * D, wq.data_ptr() if norm else None,
                        wk.data_ptr() if norm else None, 1e-6, 1e4, own.data_ptr() if use_own else None, ch, b,
                        c.status.data_ptr())
    torch.cuda.synchronize()
    assert int(c.status) == 0
    rows = qkv.view(n, H + 2 * KVH, D)
    want_k, want_v = c.kview.double(), c.vview.double()
    place = torch.zeros(n, dtype=torch.int64)
    first_row, kept = 0, torch.ones(c.pool, page, dtype=torch.bool)
    for m, t in zip(new, total):
        place[first_row:first_row + m] = torch.arange(t - m, t)
        first_row += m
    turn_at = pos if use_own else place
    q64 = turned(rows[:, :H], w[0] if norm else None, turn_at, rotary, 1e4, 1e-6)
    k64 = turned(rows[:, H:H + KVH], w[1] if norm else None, turn_at, rotary, 1e4, 1e-6)
    tol_k = torch.zeros_like(want_k)
    tol_v = torch.zeros_like(want_v)
    u = torch.finfo(TYPES[cache]).eps / 2
    at_row = 0
    for i, (m, t) in enumerate(zip(new, total)):
        for r in range(m):
            x = t - m + r
            if x >= 0:
                p, s = int(c.table_cpu[i, x // page]), x % page
                want_k[p, :, s], want_v[p, :, s] = k64[at_row + r], rows[at_row + r, H + KVH:].double()
                tol_k[p, :, s] = turn_tolerance(k64[at_row + r], cache, norm)
                tol_v[p, :, s] = rows[at_row + r, H + KVH:].double().abs() * (u if kind != cache else 0.0)
        at_row += m
    for got, want, tol in ((c.k, want_k, tol_k), (c.v, want_v, tol_v)):
        got = got.cpu().double() if first else got.cpu().transpose(1, 2).double()
        assert torch.equal(got.isnan(), want.isnan())  # nothing else is written
        near(got.nan_to_num(), want.nan_to_num(), tol)
    if H:
        used = sum(new)
        near(qo[:used], q64[:used], turn_tolerance(q64[:used], kind, norm))
        assert bool((qo[used:] == 7.0).all())


@pytest.mark.parametrize("kind,cache", KINDS)
@pytest.mark.parametrize("D", [64, 96])
def test_append_passes_over_bad_pages_and_sequences(tq, kind, cache, D):
    c = Case([2, 2, 2], [20, 30, 40], 2, 1, D, 16, True, kind, cache, seed=1)
    c.table[0, 1] = c.pool
    c.len[2] = -1
    before = c.k.clone()
    x = torch.ones(c.n, D, dtype=TYPES[kind], device="cuda")
    ch, b = c.handles(tq)
    tq.dev_paged_append(None, x.data_ptr(), x.data_ptr(), None, CODES[kind], 0, 0, 0, D, D, 0, None, None, 0.0, 1e4, None,
                        ch, b, c.status.data_ptr())
    torch.cuda.synchronize()
    assert int(c.status) in (tq.PAGED_BAD_PAGE, tq.PAGED_BAD_SEQ)
    p = int(c.table_cpu[1, 28 // 16])
    before[p, :, 28 % 16:28 % 16 + 2] = 1.0
    assert torch.equal(c.k.isnan(), before.isnan()) and torch.equal(c.k.nan_to_num(), before.nan_to_num())


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("kind,cache", KINDS)
@pytest.mark.parametrize("H,KVH,D", [(8, 2, 64), (16, 4, 128)])
def test_prompts_in_chunks_then_tokens(tq, kind, cache, H, KVH, D):
    """Two sequences' prompts appended and attended in chunks, then token by token in one
    captured graph, against dense causal attention in 64 bits over the same rounded rows."""
    page, lens, steps = 16, [75, 130], 3
    g = torch.Generator().manual_seed(D)
    L = [n + steps for n in lens]
    qkv = [(torch.randn(x, (H + 2 * KVH) * D, generator=g) * 2).to(TYPES[kind]) for x in L]
    w = [1 + 0.3 * torch.randn(D, generator=g) for _ in range(2)]
    c = Case([0, 0], L, H, KVH, D, page, False, kind, cache, pad=max(L) * 2)
    c.k.fill_(math.nan), c.v.fill_(math.nan)
    wq, wk = (x.cuda() for x in w)
    dev = [x.cuda() for x in qkv]
    out = [torch.zeros(x, H * D, dtype=TYPES[kind]) for x in L]
    q_kept = [torch.zeros(x, H * D, dtype=TYPES[kind]) for x in L]
    most = 64
    rows = torch.zeros(2 * most, (H + 2 * KVH) * D, dtype=TYPES[kind], device="cuda")
    q, o = (torch.zeros(2 * most, H * D, dtype=TYPES[kind], device="cuda") for _ in range(2))
    size, width = rows.element_size(), rows.shape[1]

    def handles(n, m):
        ch, _ = c.handles(tq)
        return ch, tq.PagedBatch(c.start.data_ptr(), c.len.data_ptr(), c.table.data_ptr(), 2, c.table.shape[1], n, m)

    def layer(n, m, work):
        ch, b = handles(n, m)
        at = rows.data_ptr()
        tq.dev_paged_append(at, at + H * D * size, at + (H + KVH) * D * size, q.data_ptr(), CODES[kind], H, D, width, width,
                            width, H * D, wq.data_ptr(), wk.data_ptr(), 1e-6, 1e4, None, ch, b, c.status.data_ptr())
        tq.dev_paged_attention(q.data_ptr(), o.data_ptr(), CODES[kind], H, H * D, H * D, c.scale, ch, b, work.data_ptr(),
                               work.numel(), c.status.data_ptr())

    ch, b = handles(2 * most, most)
    work = torch.zeros(tq.paged_attention_workspace_bytes(ch, b, H), dtype=torch.uint8, device="cuda")
    done = [0, 0]
    while any(d < n for d, n in zip(done, lens)):
        take = [min(most if i else 29, n - d) for i, (d, n) in enumerate(zip(done, lens))]
        rows[:take[0]] = dev[0][done[0]:done[0] + take[0]]
        rows[take[0]:sum(take)] = dev[1][done[1]:done[1] + take[1]]
        c.start.copy_(torch.tensor([0, take[0], sum(take)], dtype=torch.int32))
        c.len.copy_(torch.tensor([d + t for d, t in zip(done, take)], dtype=torch.int32))
        layer(2 * most, most, work)
        for i, (lo, t) in enumerate(zip((0, take[0]), take)):
            out[i][done[i]:done[i] + t] = o[lo:lo + t].cpu()
            q_kept[i][done[i]:done[i] + t] = q[lo:lo + t].cpu()
        done = [d + t for d, t in zip(done, take)]
    c.start.copy_(torch.tensor([0, 1, 2], dtype=torch.int32))
    graph, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=s):
        layer(2, 1, work)
    for t in range(steps):
        rows[0], rows[1] = dev[0][lens[0] + t], dev[1][lens[1] + t]
        c.len.copy_(torch.tensor([n + t + 1 for n in lens], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        for i in range(2):
            out[i][lens[i] + t], q_kept[i][lens[i] + t] = o[i].cpu(), q[i].cpu()
    assert int(c.status) == 0
    for i, x in enumerate(L):
        r = qkv[i].view(x, H + 2 * KVH, D)
        pos = torch.arange(x)
        k64 = turned(r[:, H:H + KVH], w[1], pos, D, 1e4, 1e-6)
        pages = c.table_cpu[i, :].tolist()
        got_k = torch.stack([c.k.cpu()[pages[y // page], y % page] for y in range(x)])
        near(got_k, k64, turn_tolerance(k64, cache, True))
        # attention over the cache as it was rounded
        ref = Case([x], [x], H, KVH, D, page, False, kind, cache, device="cpu")
        ref.q_cpu = q_kept[i]
        for y in range(x):
            p = int(ref.table_cpu[0, y // page])
            ref.kview[p, :, y % page] = got_k[y]
            ref.vview[p, :, y % page] = r[y, H + KVH:].to(TYPES[cache])
        want, m, vmax = ref.want()
        near(out[i], want, ref.tolerance(m, vmax))
