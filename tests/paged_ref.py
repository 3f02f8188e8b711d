"""Inputs and 64-bit restatements for the paged-cache operator tests (test infrastructure)."""
from __future__ import annotations

import math

import torch

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f32": 0, "f16": 1, "bf16": 2}


class Case:
    """A batch of sequences (new[i] rows, total[i] cached positions with them) over a cache in
    pages of random order.  Slots that no sequence holds are NaN in k and v, table entries
    past a sequence's pages an impossible page."""

    def __init__(self, new, total, heads=8, kv_heads=2, dim=64, page=16, heads_first=True, kind="f32",
                 cache="f32", pad=0, seed=0, device="cuda", gap=0, qk=1.0, shift=0, spare=3, room=0):
        g = torch.Generator().manual_seed(seed)
        self.new, self.total, self.H, self.KVH, self.D = list(new), list(total), heads, kv_heads, dim
        self.page, self.kind, self.cache, self.dev = page, kind, cache, device
        self.n = sum(new) + pad
        used = [-(-t // page) for t in total]
        self.pool = sum(used) + spare
        order = torch.randperm(self.pool, generator=g).tolist()
        # `room`: positions that the page table has space for (a wide one sends a call with many
        # rows to the tcgen05 kernel, which the lengths themselves do not show on the host)
        width = max(max(used + [1]) + 1, room // page)
        self.table_cpu = torch.full((max(1, len(new)), width), 1 << 29, dtype=torch.int32)
        at = 0
        for i, u in enumerate(used):
            self.table_cpu[i, :u] = torch.tensor(order[at:at + u], dtype=torch.int32)
            at += u
        shape = (self.pool, kv_heads, page, dim) if heads_first else (self.pool, page, kv_heads, dim)
        dt = TYPES[cache]
        k = torch.full(shape, math.nan, dtype=dt)
        v = torch.full(shape, math.nan, dtype=dt)
        self.kview = k if heads_first else k.transpose(1, 2)   # [page][head][slot][dim]
        self.vview = v if heads_first else v.transpose(1, 2)
        for i, t in enumerate(total):
            for x in range(t):
                p, s = int(self.table_cpu[i, x // page]), x % page
                self.kview[p, :, s] = (torch.randn(kv_heads, dim, generator=g) * qk).to(dt)
                self.vview[p, :, s] = torch.randn(kv_heads, dim, generator=g).to(dt)
        self.k_cpu, self.v_cpu, self.heads_first = k, v, heads_first
        self.shift = shift  # elements by which q and out are moved off their allocation
        self.qw = heads * dim + gap
        self.q_cpu = (torch.randn(self.n, self.qw, generator=g) * qk).to(TYPES[kind])
        self.scale = 1.0 / math.sqrt(dim)
        self.upload()

    def upload(self):
        d = self.dev
        st = [0]
        for x in self.new:
            st.append(st[-1] + x)
        self.start = torch.tensor(st, dtype=torch.int32, device=d)
        self.len = torch.tensor(self.total or [0], dtype=torch.int32, device=d)
        self.table = self.table_cpu.to(d)
        self.k, self.v = self.k_cpu.to(d), self.v_cpu.to(d)
        dt = TYPES[self.kind]
        self.qbuf = torch.empty(self.n * self.qw + 16, dtype=dt, device=d)
        self.qbuf[self.shift:self.shift + self.n * self.qw] = self.q_cpu.to(d).reshape(-1)
        self.obuf = torch.full((self.n * self.qw + 16,), 7.0, dtype=dt, device=d)
        self.status = torch.zeros(1, dtype=torch.int32, device=d)

    def handles(self, lib, k=None, v=None, max_q=None):
        P, KVH, D = self.page, self.KVH, self.D
        where = (KVH * P * D, P * D, D) if self.heads_first else (P * KVH * D, D, KVH * D)
        c = lib.PagedCache((self.k if k is None else k).data_ptr(), (self.v if v is None else v).data_ptr(),
                           CODES[self.cache], self.pool, P, KVH, D, *where)
        b = lib.PagedBatch(self.start.data_ptr(), self.len.data_ptr(), self.table.data_ptr(), len(self.new),
                           self.table.shape[1], self.n, max(self.new + [0]) if max_q is None else max_q)
        return c, b

    def workspace(self, lib, c, b):
        return torch.zeros(max(16, lib.paged_attention_workspace_bytes(c, b, self.H)), dtype=torch.uint8,
                           device=self.dev)

    def attend(self, lib, work=None, stream=None, handles=None):
        """One call; returns out [n, H * D] (rows as the library left them)."""
        c, b = handles or self.handles(lib)
        w = self.workspace(lib, c, b) if work is None else work
        esz = self.qbuf.element_size()
        lib.dev_paged_attention(self.qbuf.data_ptr() + self.shift * esz, self.obuf.data_ptr() + self.shift * esz,
                                CODES[self.kind], self.H, self.qw, self.qw, self.scale, c, b, w.data_ptr(),
                                w.numel(), self.status.data_ptr(), stream)
        return self.out()

    def out(self):
        return self.obuf[self.shift:self.shift + self.n * self.qw].view(self.n, self.qw)[:, :self.H * self.D]

    def want(self, drop=()):
        """(out [n, H, D], bound of the score sum |q.k| scale, largest |v|) in 64 bits; rows that
        no sequence has keep the 7 they were filled with.  drop: positions masked, (seq, x)."""
        H, KVH, D = self.H, self.KVH, self.D
        out = torch.full((self.n, H, D), 7.0, dtype=torch.float64)
        q = self.q_cpu[:, :H * D].double().view(self.n, H, D)
        most, vmax, first = 0.0, 0.0, 0
        for i, (n, t) in enumerate(zip(self.new, self.total)):
            x = torch.arange(t)
            pages = self.table_cpu[i].long()[x // self.page]
            held = (pages >= 0) & (pages < self.pool)
            for lost in drop:
                if lost[0] == i:
                    held[lost[1]] = False
            at = torch.where(held, pages, torch.zeros_like(pages)), slice(None), x % self.page
            k, v = self.kview[at].double(), self.vview[at].double()
            k[~held], v[~held] = 0.0, 0.0
            k, v = k.repeat_interleave(H // KVH, 1), v.repeat_interleave(H // KVH, 1)
            rows = q[first:first + n]
            seen = held[None] & (x[None] <= torch.arange(t - n, t)[:, None])
            s = torch.einsum("rhd,xhd->hrx", rows, k) * self.scale
            s.masked_fill_(~seen, -math.inf)
            w = torch.softmax(s, -1).masked_fill(~seen, 0.0)  # a row that sees nothing: zeros
            out[first:first + n] = torch.einsum("hrx,xhd->rhd", w, v)
            if n and t:
                most = max(most, float((torch.einsum("rhd,xhd->hrx", rows.abs(), k.abs()) * self.scale).max()))
                vmax = max(vmax, float(v.abs().max()))
            first += n
        return out.view(self.n, H * D), most, vmax

    def tolerance(self, most, vmax):
        """Largest distance of a right result from the 64-bit one, from its roundings.
        Scores: products of D terms in at most 24 sequential fp32 additions, the operands split
        to 2^-21: absolute error ds <= most * (24 * 2^-24 + 2^-21).  Weights: relative error
        ds + 2^-21 (exponential and running maximum) + u (their rounding to the type).  Sums
        over n positions: n 2^-24.  Numerator and denominator each carry these; the result is
        rounded to u."""
        u = torch.finfo(TYPES[self.kind]).eps / 2
        n = max(self.total + [1])
        ds = most * (24 * 2.0 ** -24 + 2.0 ** -21)
        return vmax * (2 * (ds + 2.0 ** -21 + n * 2.0 ** -24) + 2 * u)


def turned(x, w, pos, rotary, theta, eps):
    """RMS norm and rotation of rows x [n, heads, dim] in 64 bits."""
    x = x.double()
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    h = rotary // 2
    f = torch.tensor([float(theta) ** (-2.0 * i / rotary) for i in range(h)], dtype=torch.float64)
    a = pos.double()[:, None] * f
    c, s = torch.cos(a)[:, None], torch.sin(a)[:, None]
    return torch.cat([x[..., :h] * c - x[..., h:rotary] * s, x[..., h:rotary] * c + x[..., :h] * s,
                      x[..., rotary:]], -1)


def turn_tolerance(want, kind, normed):
    """Roundings of a rotated value: the sum of squares (at most 13 fp32 additions, half of
    which reaches the root), the root (2 ulp), the factors and the two products (6), the angle
    (its fraction rounded once: 2^-24 of half a turn, pi 2^-24 <= 4 * 2^-24, and sine and
    cosine 2 ulp): 24 half steps of the pair's length in all; then the type's own rounding."""
    u = torch.finfo(TYPES[kind]).eps / 2
    length = want.abs().amax(-1, keepdim=True) * math.sqrt(2.0)
    return length * 24 * 2.0 ** -24 + want.abs() * u + (2.0 ** -25 if kind == "f16" else 0.0)
