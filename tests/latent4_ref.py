"""Plain forms of the 4-bit latent rows, the accumulated attention weights and the eviction by them, for the tests (CPU)."""
import math

import torch

from latent_ref import LAT, PE, ROW, SCALE, cache_rows

ROW4, GROUP = 400, 32
SIZES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
LEAST = {torch.bfloat16: -125, torch.float16: -23}
MOST = {torch.bfloat16: 125, torch.float16: 13}


def rounded(latent, pe):
    """[T, 512] and [T, 64] of one 16-bit type -> rows [T, 400] uint8, a value at a time."""
    out = torch.zeros(latent.shape[0], ROW4, dtype=torch.uint8)
    out[:, 272:] = pe.contiguous().view(torch.uint8)
    for t in range(latent.shape[0]):
        values = latent[t].double().tolist()
        for g in range(LAT // GROUP):
            x = values[g * GROUP:(g + 1) * GROUP]
            if not all(math.isfinite(v) for v in x):
                out[t, 256 + g] = 255
                continue
            a = max(abs(v) for v in x)
            e = math.frexp(a)[1] - 3 if a else LEAST[latent.dtype]
            if a > 7 * 2.0 ** e:
                e += 1
            e = min(max(e, LEAST[latent.dtype]), MOST[latent.dtype])
            out[t, 256 + g] = e + 127
            for i, v in enumerate(x):
                y = abs(v) / 2.0 ** e
                # the nearest, of two equally near ones the even
                code = min(range(8), key=lambda k: (abs(SIZES[k] - y), k % 2))
                code |= 8 if math.copysign(1.0, v) < 0 else 0
                j = g * GROUP + i
                out[t, j // 2] |= code << 4 * (j % 2)
    return out


def ends(dtype):
    """[21, 512]: groups about the largest and the smallest numbers of the type, where the scale's exponent is held."""
    info = torch.finfo(dtype)
    top, step, rows = MOST[dtype], info.tiny * info.eps, []
    for a in (info.max, 6.0 * 2.0 ** top, 6.5 * 2.0 ** top, 7.0 * 2.0 ** top, 7.0 * 2.0 ** top * (1 + info.eps), 7.75 * 2.0 ** top):
        rows.append(a * torch.linspace(-1, 1, LAT, dtype=torch.float64))
    for k in (1, 2, 3, 5, 7, 8, 11, 60, 64, 100, 127, 128, 250, 255, 1000):  # the largest is the k-th number
        rows.append(step * torch.round(k * torch.linspace(-1, 1, LAT, dtype=torch.float64)))
    return torch.stack(rows).to(dtype)


def values(rows, dtype):
    """[..., 400] uint8 -> [..., 576] of the type"""
    size = torch.tensor(SIZES + [-s for s in SIZES], dtype=torch.float64)
    size[8] = -0.0
    lat = size[torch.stack([rows[..., :256] & 15, rows[..., :256] >> 4], dim=-1).flatten(-2).long()]
    power = torch.tensor([2.0 ** (b - 127) for b in range(255)] + [math.nan], dtype=torch.float64)
    lat = lat * power[rows[..., 256:272].long()].repeat_interleave(GROUP, dim=-1)
    # (codes times powers of two are numbers of float32, or below its smallest normal one and 0 or exact in either type)
    return torch.cat([lat.float().to(dtype), rows[..., 272:].contiguous().view(dtype)], dim=-1)


def weights(ql, qp, cache, table, lens, S, lse, before, scale=SCALE):
    """(weights afterwards [B, W], tolerance) of latent_weights on CPU tensors, cache in 16 bits.

    Tolerance, f = 2^-24: dz = D f Z of a score (D = 576 products, Z the sum of their sizes), f (|z| + |lse|) of the difference,
    f |z - lse| of its product with log2 e; the exponential 2^-22; each of n rows' additions f of the sum; the last one f of the
    result."""
    H, size = ql.shape[1], cache.shape[1]
    f = 2.0 ** -24
    out, tol = before.double().clone(), torch.zeros_like(before, dtype=torch.float64)
    for n in range(len(lens)):
        length = max(0, min(int(lens[n]), size * table.shape[1]))
        rows, there = cache_rows(cache, table[n], length)
        q = torch.cat([ql, qp], dim=-1)[n * S:(n + 1) * S].double().reshape(S * H, ROW)
        s = torch.arange(S).repeat_interleave(H)
        seen = there[None, :] & (torch.arange(length)[None, :] < length - (S - 1 - s)[:, None])
        z, Z = q @ rows.T * scale, q.abs() @ rows.abs().T * scale
        m = lse[n * S:(n + 1) * S].double().reshape(S * H, 1)
        w = torch.where(seen & (m != -math.inf), torch.exp(z - m), torch.zeros_like(z))
        t = 2 * w * (ROW * f * Z + 2 * f * (z.abs() + m.abs()) + 2.0 ** -22)
        t = torch.where(w > 0, t, torch.zeros_like(t))
        out[n, :length] += w.sum(dim=0)
        tol[n, :length] = t.sum(dim=0) + (S * H + 8) * f * w.sum(dim=0) + f * out[n, :length].abs()
    return out, tol


def evict(pools, mass, table, lens, refs, free, num, rows, keep, recent, size):
    """evict_tokens on plain lists: pools[l][page][offset] and mass[l][row][j] anything that can be moved."""
    start, push, done = list(refs), [], set()
    left = keep - recent
    for r in rows:
        if not 0 <= r < len(table) or r in done:
            continue
        done.add(r)
        n = min(lens[r], len(table[r]) * size)
        used = -(-n // size)
        if n <= keep or any(not 0 <= g < len(refs) for g in table[r][:used]):
            continue
        fixed = max([0] + [(j + 1) * size for j in range(used) if start[table[r][j]] > 1])
        if fixed > left:
            continue
        at = lambda j: (table[r][j // size], j % size)  # noqa: E731
        for pool, w in zip(pools, mass):
            w = w[r]
            key = lambda j: (not math.isnan(w[j]), -w[j] if not math.isnan(w[j]) else 0.0, j)  # noqa: E731
            stays = set(range(fixed)) | set(sorted(range(fixed, n - recent), key=key)[:left - fixed])
            holes = [j for j in range(left) if j not in stays]
            movers = [j for j in range(left, n - recent) if j in stays]
            assert len(holes) == len(movers)
            for a, b in list(zip(holes, movers)) + [(left + k, n - recent + k) for k in range(recent)]:
                (p, o), (q, u) = at(a), at(b)
                pool[p][o] = pool[q][u]
                w[a] = w[b]
            w[keep:n] = [0.0] * (n - keep)
        kept = -(-keep // size)
        push += table[r][kept:used]
        table[r][:] = table[r][:kept] + table[r][used:] + [-1] * (used - kept)
        lens[r] = keep
    gone = []
    for g in push:
        if refs[g] == 1:
            refs[g] = 0
            gone.append(g)
    for g in sorted(gone, reverse=True):
        free[num] = g
        num += 1
    return num


__all__ = ["ROW4", "GROUP", "LAT", "PE", "ends", "rounded", "values", "weights", "evict"]
