"""Plain float64 forms of latent attention and plain Python forms of the page bookkeeping, for the tests (CPU).

Tolerances, per output element, with u = finfo(type).eps / 2 (one rounding to the type), A = sum_j softmax_j |v_j|, D the
length of the dot products, Z the largest scale * sum |q||k| of the row and L its number of keys:
    final rounding                           u |o|
    weights rounded to the type              u A
    scores in fp32: |dz| <= D 2^-24 Z, which changes each weight and the sum by e^dz - 1    2 D 2^-24 Z A
    fp32 sums over the keys and exponentials                                                (L + 8) 2^-24 A
    fp16 weights and results below the smallest number                                      (L + 1) 2^-24 max|v|
lse: D 2^-24 Z + (L + 16) 2^-24 + 2^-23 |lse|."""
import math

import torch

LAT, PE, HEAD = 512, 64, 128
ROW = LAT + PE
SCALE = (HEAD + PE) ** -0.5


def attend(q, keys, vals, visible, scale):
    """(o, lse, tol of o, tol of lse but for the type's rounding) of float64 rows; visible bool [rows, keys].  Values of keys
    that no row sees are never used."""
    rows, L = q.shape[0], keys.shape[0]
    o = torch.zeros(rows, vals.shape[1], dtype=torch.float64)
    A = torch.zeros_like(o)
    lse = torch.full((rows,), -math.inf, dtype=torch.float64)
    Z = torch.zeros(rows, dtype=torch.float64)
    vmax = torch.zeros(rows, dtype=torch.float64)
    for pattern in torch.unique(visible, dim=0) if rows and L else []:
        r = (visible == pattern).all(dim=1).nonzero().flatten()
        j = pattern.nonzero().flatten()
        if len(j) == 0:
            continue
        z = q[r] @ keys[j].T * scale
        lse[r] = torch.logsumexp(z, dim=1)
        p = torch.exp(z - lse[r][:, None])
        o[r] = p @ vals[j]
        A[r] = p @ vals[j].abs()
        Z[r] = (q[r].abs() @ keys[j].abs().T * abs(scale)).max(dim=1).values
        vmax[r] = vals[j].abs().max()
    return o, A, lse, Z, vmax, L


def check(got, got_lse, ref, dtype, D, what):
    """Asserts the tolerances above; prints the largest share of them that is used."""
    o, A, lse, Z, vmax, L = ref
    u = torch.finfo(dtype).eps / 2
    f = 2.0 ** -24
    tol = u * (o.abs() + A) + ((2 * D * Z + L + 8) * f)[:, None] * A
    if dtype == torch.float16:
        tol = tol + ((L + 1) * f * vmax)[:, None]
    d = (got.double().cpu() - o).abs()
    bad = d > tol
    assert not torch.isnan(d).any(), f"{what}: NaN"
    used = float((d / tol.clamp(min=1e-300)).max()) if d.numel() else 0.0
    print(f"[err] {what}: largest share of the tolerance {used:.3f}", flush=True)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} elements off, worst share {used:.3f}"
    if got_lse is not None:
        g = got_lse.double().cpu()
        empty = torch.isinf(lse)
        assert torch.equal(g[empty], lse[empty]), f"{what}: lse of rows that see nothing"
        tl = D * f * Z + (L + 16) * f + 2 * f * lse.abs()
        dl = (g - lse).abs()[~empty]
        assert (dl <= tl[~empty]).all(), f"{what}: lse off by {float(dl.max()):.3e}"


def cache_rows(cache, table, n):
    """(rows [n, 576] float64, present bool [n]) of a sequence; tokens in holes are zeros and absent."""
    pages, size, _ = cache.shape
    rows = torch.zeros(n, ROW, dtype=torch.float64)
    there = torch.zeros(n, dtype=torch.bool)
    for j in range(n):
        page = int(table[j // size])
        if 0 <= page < pages:
            rows[j] = cache[page, j % size].double()
            there[j] = True
    return rows, there


def decode(ql, qp, cache, table, lens, S, scale=SCALE, prefix_table=None, prefix_len=0):
    """latent_decode on CPU tensors, one (o, A, lse, Z, vmax, L) of the S * H rows of every sequence."""
    out = []
    H, size = ql.shape[1], cache.shape[1]
    head, head_there = cache_rows(cache, prefix_table, max(0, min(prefix_len, size * len(prefix_table)))) \
        if prefix_table is not None else cache_rows(cache, [], 0)
    P = head.shape[0]
    for n in range(len(lens)):
        length = max(0, min(int(lens[n]), size * table.shape[1]))
        rows, there = cache_rows(cache, table[n], length)
        rows, there = torch.cat([head, rows]), torch.cat([head_there, there])
        q = torch.cat([ql, qp], dim=-1)[n * S:(n + 1) * S].double().reshape(S * H, ROW)
        j = torch.arange(P + length)
        s = torch.arange(S).repeat_interleave(H)
        visible = there[None, :] & (j[None, :] < P + length - (S - 1 - s)[:, None]) | (there & (j < P))[None, :]
        out.append(attend(q, rows, rows[:, :LAT], visible, scale))
    return out


def prefill(q, k, v, pe, cu_q, cu_k, causal, scale=SCALE):
    """latent_prefill on CPU tensors: one (o, A, lse, Z, vmax, L) for each (sequence, head)."""
    out = []
    for n in range(len(cu_q) - 1):
        a, b, c, d = cu_q[n], cu_q[n + 1], cu_k[n], cu_k[n + 1]
        i, j = torch.arange(b - a)[:, None], torch.arange(d - c)[None, :]
        visible = (j <= i + (d - c) - (b - a)) if causal else torch.ones(b - a, d - c, dtype=torch.bool)
        for h in range(q.shape[1]):
            keys = torch.cat([k[c:d, h], pe[c:d]], dim=-1).double()
            out.append((n, h, attend(q[a:b, h].double(), keys, v[c:d, h].double(), visible, scale)))
    return out


# ------------------------------------------------------------------------------------------------ page bookkeeping
class Book:
    """The bookkeeping of kda355/pages.py as plain lists, with the pools' rows as a list of page contents."""

    def __init__(self, table, lens, refs, free, num, size):
        self.table, self.lens = [list(r) for r in table], list(lens)
        self.refs, self.free, self.num, self.size = list(refs), list(free), num, size
        self.moves = []  # (src, dst) in the order made

    def _length(self, r):
        return max(0, min(self.lens[r], len(self.table[r]) * self.size))

    def fork(self, parents, children):
        pages, rows = len(self.refs), len(self.table)
        jobs = []
        for p, c in zip(parents, children):
            if not (0 <= p < rows and 0 <= c < rows and p != c):
                continue
            n = self._length(p)
            full, new = n // self.size, None
            if n % self.size and 0 <= self.table[p][full] < pages:  # (a hole stays one: there is nothing to copy)
                new = -2
                if self.num > 0:
                    self.num -= 1
                    new, self.free[self.num] = self.free[self.num], -1
                    if not 0 <= new < pages:
                        new = -2
            jobs.append((p, c, n, full, new))
        for p, c, n, full, new in jobs:
            width = len(self.table[c])
            if new == -2:
                self.table[c], self.lens[c] = [-1] * width, 0
                continue
            row = self.table[p][:full]
            for g in row:
                if 0 <= g < pages:
                    self.refs[g] += 1
            if new is not None:
                self.moves.append((self.table[p][full], new))
                self.refs[new] = 1
                row = row + [new]
            self.table[c], self.lens[c] = row + [-1] * (width - len(row)), n

    def release(self, which):
        pages, gone = len(self.refs), []
        for r in which:
            if not 0 <= r < len(self.table):
                continue
            used = -(-self._length(r) // self.size)
            for g in self.table[r][:used]:
                if 0 <= g < pages and self.refs[g] > 0:
                    self.refs[g] -= 1
                    if self.refs[g] == 0:
                        gone.append(g)
            self.table[r], self.lens[r] = [-1] * len(self.table[r]), 0
        for g in sorted(gone, reverse=True):
            self.free[self.num] = g
            self.num += 1

    def compact(self):
        pages = len(self.refs)
        live = sum(r > 0 for r in self.refs)
        holes = [p for p in range(live) if self.refs[p] <= 0]
        movers = [p for p in range(live, pages) if self.refs[p] > 0]
        to = dict(zip(movers, holes))
        for s, d in to.items():
            self.moves.append((s, d))
            self.refs[d], self.refs[s] = self.refs[s], 0
        self.table = [[to.get(g, g) for g in r] for r in self.table]
        self.free = [pages - 1 - j if j < pages - live else -1 for j in range(pages)]
        self.num = pages - live
