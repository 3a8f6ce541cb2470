"""The 8-bit cache in 64 bits, from its definition, and inputs for it: whole sequences on the host, one function per operator."""
import math
import random

import torch

BLOCK = 16
# the non-negative values of the code: three bits of fraction, exponents -6 to 8, steps of 2^-9 below; 480 would be the NaN
GRID = torch.tensor([m * 2.0 ** -9 for m in range(8)] + [(8 + m) / 8.0 * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-1],
                    dtype=torch.float64)


def scale_for(top: float) -> float:
    """The smallest power of two from 2^-126 on with top <= 448 s."""
    s = 2.0 ** -126
    if top > 448.0 * s:
        s = 2.0 ** (math.frexp(top / 448.0)[1] - 2)
        while top > 448.0 * s:
            s *= 2.0
    return s


def nearest(x: torch.Tensor) -> torch.Tensor:
    """The nearest value of the grid, of two equally near ones that with the even code; infinities and NaN give NaN."""
    a = x.abs().nan_to_num(0.0, 0.0, 0.0)
    hi = torch.searchsorted(GRID, a).clamp(max=len(GRID) - 1)
    lo = (hi - 1).clamp(min=0)
    up, down = (GRID[hi] - a).abs(), (a - GRID[lo]).abs()
    take = (up < down) | ((up == down) & (hi % 2 == 0))
    got = torch.where(take, GRID[hi], GRID[lo]) * torch.where(x < 0, -1.0, 1.0)
    return torch.where(torch.isfinite(x), got, torch.nan)


def values_of(pool: torch.Tensor) -> torch.Tensor:
    return pool.cpu().float().double()


class Batch:
    """A step over a cache: ``each`` lists (tokens cached after the step, new tokens) of every request."""

    def __init__(self, each, page, *, seed=0, spare_pages=2, spare_slots=1, table_pages=None):
        rng = random.Random(seed)
        self.each, self.page = each, page
        n = len(each)
        width = table_pages or max(1, max(-(-k // page) for k, _ in each))
        used = [-(-k // page) for k, _ in each]
        self.n_pages = sum(used) + spare_pages
        ids = rng.sample(range(self.n_pages), self.n_pages)
        self.slots = rng.sample(range(n + spare_slots), n)
        self.table = torch.full((n + spare_slots, width), -1, dtype=torch.int32)
        at = 0
        for r, u in enumerate(used):
            self.table[self.slots[r], :u] = torch.tensor(ids[at:at + u], dtype=torch.int32)
            at += u
        self.q_start = [0]
        self.positions, self.req = [], []
        for r, (k, q) in enumerate(each):
            self.q_start.append(self.q_start[-1] + q)
            self.positions += range(k - q, k)
            self.req += [r] * q
        self.tiles = [(r, t) for r, (k, q) in enumerate(each) if q > 1 for t in range(0, q, 64)]
        self.single = [r for r, (k, q) in enumerate(each) if q == 1]
        self.tokens = len(self.req)

    def arrays(self, device):
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
        return dict(block_table=self.table.to(device), positions=i32(self.positions), req_of_token=i32(self.req), q_start=i32(self.q_start),
                    slots=i32(self.slots), kv_len=i32([k for k, _ in self.each]), tiles=i32(self.tiles).reshape(-1, 2), decode_reqs=i32(self.single))

    def row_of(self, r, pos):
        """(page, row in the page) of a position of request r."""
        return int(self.table[self.slots[r], pos // self.page]), pos % self.page


def write(batch: Batch, k, v, codes, scales):
    """The operator on host tensors in place: k, v [tokens, heads, dim] float64, codes (values) float64, scales float64."""
    for r, (n, q) in enumerate(batch.each):
        at, first = batch.q_start[r], n - q
        for b in range(first // BLOCK, -(-n // BLOCK)):
            lo, hi = max(first, b * BLOCK), min(n, (b + 1) * BLOCK)
            if lo >= hi:
                continue
            page, row = batch.row_of(r, b * BLOCK)
            sub, ahead = row // BLOCK, lo - b * BLOCK
            for plane, x in enumerate((k, v)):
                new = x[at + lo - first:at + hi - first]
                for h in range(new.shape[1]):
                    fine = new[:, h][torch.isfinite(new[:, h])]
                    s = scale_for(float(fine.abs().max()) if fine.numel() else 0.0)
                    if ahead:
                        was = float(scales[page, plane, h, sub])
                        s = max(s, was)
                        codes[page, plane, h, row:row + ahead] = nearest(codes[page, plane, h, row:row + ahead] * (was / s))
                    codes[page, plane, h, row + ahead:row + ahead + hi - lo] = nearest(new[:, h] / s)
                    scales[page, plane, h, sub] = s


def attention(batch: Batch, q, codes, scales, heads, scale, window=None):
    """(outputs, bound of their error but for the output's own rounding, for f16 and for split operands) in float64, [tokens, heads, dim].

    The bound: a score's error e moves its probability by e relative; the sum of probabilities times |v| is the output's size A.  The
    products of a score are summed 16 at a time with an error of 2^-19 of the largest partial sum a step, of which the bound |q|max sum |k| is
    many times the size: (steps) 2^-22 |q|max sum |k| scale.  A probability is rounded to 2^-11 (as two halves: 2^-22), the exponential is off by
    2^-22 + 2^-24 |score|, and sums of n products add 2^-22 a step of 16 keys."""
    n_kv, dim = codes.shape[2], codes.shape[4]
    group = heads // n_kv
    out = torch.zeros(batch.tokens, heads, dim, dtype=torch.float64)
    rough, fine = torch.zeros_like(out), torch.zeros_like(out)
    for r, (n, nq) in enumerate(batch.each):
        if n == 0 or nq == 0:
            continue
        at = [batch.row_of(r, j) for j in range(n)]
        pages, rows = torch.tensor([a for a, _ in at]), torch.tensor([b for _, b in at])
        there = pages >= 0
        kv = codes[pages.clamp(min=0), :, :, rows] * scales[pages.clamp(min=0), :, :, rows // BLOCK][..., None]  # [n, 2, heads, dim]
        x = q[batch.q_start[r]:batch.q_start[r + 1]].unflatten(1, (n_kv, group))
        t = torch.einsum("qhgd,khd->hgqk", x, kv[:, 0]) * scale
        p = torch.arange(n - nq, n)[:, None]
        j = torch.arange(n)[None]
        hide = (j > p) | ~there[None] | ((j <= p - window) if window else torch.zeros(1, 1, dtype=torch.bool))
        t = t.masked_fill(hide, -math.inf)
        w = torch.exp(t - t.nan_to_num(-math.inf).amax(dim=3, keepdim=True).clamp(min=-1e300))
        total = w.sum(dim=3, keepdim=True)
        w = torch.where(total == 0, 0.0, w / total)
        # a value that is NaN reaches the rows that see it, whatever its weight, and no others
        clean = kv[:, 1].nan_to_num(0.0)
        bad = torch.einsum("hgqk,khd->qhgd", (~hide).double().expand(n_kv, group, nq, n), torch.isnan(kv[:, 1]).double()) > 0
        o = torch.einsum("hgqk,khd->qhgd", w, clean)
        size = torch.einsum("hgqk,khd->qhgd", w.nan_to_num(0.0), clean.abs())
        most = x.abs().amax(dim=3).permute(1, 2, 0)[..., None] * kv[:, 0].nan_to_num(0.0).abs().sum(dim=2).T[:, None, None] * scale
        most = most.masked_fill(hide, 0.0).nan_to_num(0.0).amax(dim=3).permute(2, 0, 1)[..., None]
        common = 2 * most * (dim / 16) * 2.0 ** -22 + most * 2.0 ** -22 + 2.0 ** -21 + (n / 16 + 8) * 2.0 ** -22
        s = slice(batch.q_start[r], batch.q_start[r + 1])
        out[s] = torch.where(bad, torch.nan, o).flatten(1, 2)
        rough[s] = (size * (2.0 ** -11 + common)).flatten(1, 2)
        fine[s] = (size * (2.0 ** -21 + common)).flatten(1, 2)
    return out, rough, fine
