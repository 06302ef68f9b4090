"""Accumulated attention weights against float64 (tolerances in latent4_ref), eviction by them bit for bit against plain lists, and
both together with append, decode and the pages, as a sequence under a budget runs them."""
import random

import pytest
import torch

import kda355
import latent4_ref as Q
import latent_ref as R
from latent_ref import LAT, PE, ROW, SCALE
from test_gpu_latent import DECODE, Absorbed, _i32, _randn
from test_gpu_latent4 import _narrow

pytestmark = pytest.mark.gpu
DEV, BF, HF = "cuda", torch.bfloat16, torch.float16
NAN, INF = float("nan"), float("inf")


# ================================================================================================ weights
def _weights(x, bits, lse, before, wide=False, scale=None):
    ql, qp, table = x.ql.to(DEV), x.qp.to(DEV), x.table.to(DEV)
    cache = x.bytes if bits == 4 else x.cache.to(DEV)
    if wide:
        both = torch.cat([ql, qp], dim=-1)
        ql, qp = both[..., :LAT], both[..., LAT:]
        row = cache.shape[2]
        page = torch.zeros(cache.shape[0], x.size * row + 80, dtype=cache.dtype, device=DEV)
        view = page.as_strided(cache.shape, (page.shape[1], row, 1))
        view.copy_(cache)
        cache = view
        table = torch.cat([table, torch.full_like(table, 1 << 20)], dim=1)[:, :table.shape[1]]
    W = before.shape[1]
    buf = torch.full((before.shape[0], W + 5), 9.0, device=DEV)
    buf[:, :W] = before.to(DEV)
    got = kda355.latent_weights(ql, qp, cache, table, _i32(x.lens), lse.to(DEV), buf[:, :W], scale)
    assert got.data_ptr() == buf.data_ptr() and (buf[:, W:] == 9.0).all()
    return got.cpu()


def _check_weights(x, bits, what="", **kw):
    if bits == 4:
        _narrow(x)
    S, H, B = x.S, x.H, len(x.lens)
    lse = torch.cat([ref[2].view(S, H) for ref in R.decode(x.ql, x.qp, x.cache, x.table, x.lens, S, prefix_table=x.prefix_table,
                                                          prefix_len=x.prefix or 0)]).float()
    before = torch.rand(B, x.table.shape[1] * x.size, generator=torch.Generator().manual_seed(3))
    want, tol = Q.weights(x.ql, x.qp, x.cache, x.table, x.lens, S, lse, before)
    got = _weights(x, bits, lse, before, **kw)
    d = (got.double() - want).abs()
    used = float((d / tol.clamp(min=1e-300))[tol > 0].max()) if (tol > 0).any() else 0.0
    print(f"[err] {what}: largest share of the tolerance {used:.3f}", flush=True)
    assert (d <= tol).all(), f"{what}: {int((d > tol).sum())} off, worst share {used:.3f}"
    assert torch.equal(got, _weights(x, bits, lse, before, **kw))
    return got, want, lse


@pytest.mark.parametrize("lens,S,H,size", DECODE, ids=[f"{len(c[0])}seq-{max(c[0])}-S{c[1]}-H{c[2]}-p{c[3]}" for c in DECODE])
@pytest.mark.parametrize("bits,dtype", [(16, BF), (16, HF), (4, BF), (4, HF)])
def test_weights_lengths(lens, S, H, size, bits, dtype):
    _check_weights(Absorbed(lens, S, H, size, dtype), bits)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("lens,S,H,size,prefix", [([400, 90], 1, 12, 64, None), ([130, 77, 1], 4, 17, 16, None), ([513], 1, 128, 100, 70)])
def test_weights_views_and_prefix(lens, S, H, size, prefix, bits):
    _check_weights(Absorbed(lens, S, H, size, BF, prefix=prefix), bits, wide=True)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("H", [8, 64, 200])
def test_weights_long(bits, H):
    got, want, lse = _check_weights(Absorbed([9000, 3333, 1], 1, H, 64, BF, std=2.0), bits)


@pytest.mark.parametrize("bits", [16, 4])
def test_weights_of_every_row_sum_to_one(bits):
    """With the step's own log-sums: what the tokens of a sequence get are its rows' softmax weights, which add up to one a row."""
    x = Absorbed([3000, 77], 3, 20, 16, BF)
    if bits == 4:
        _narrow(x)
    cache = x.bytes if bits == 4 else x.cache.to(DEV)
    lse = torch.empty(6, 20, device=DEV)
    kda355.latent_decode(x.ql.to(DEV), x.qp.to(DEV), cache, x.table.to(DEV), _i32(x.lens), lse=lse)
    got = _weights(x, bits, lse, torch.zeros(2, x.table.shape[1] * 16))
    # scores of up to Z ~ 100: 2 ROW 2^-24 Z, and the sum's own additions
    assert (got.double().sum(dim=1) - 60).abs().max() < 60 * (2 * ROW * 100 + 3100) * 2.0 ** -24


@pytest.mark.parametrize("bits", [16, 4])
def test_weights_holes_and_odd_lengths(bits):
    x = Absorbed([300, 64, 700, 5], 2, 24, 16, BF)
    x.table[0, 3], x.table[0, 7], x.table[1, :] = -1, x.cache.shape[0], -9
    x.table[2, 10:30] = 1 << 30
    x.lens[3] = -4
    _check_weights(x, bits)
    x = Absorbed([64, 30], 1, 8, 16, BF)
    x.lens, x.table = [1 << 30, 30], x.table[:, :4].contiguous()
    _check_weights(x, bits)


@pytest.mark.parametrize("bits", [16, 4])
def test_weights_of_special_rows(bits):
    """A row whose log-sum is -inf gives nothing; a row or a token with a NaN makes NaN of what sees it and of nothing else; a later
    draft token reaches no earlier row."""
    x = Absorbed([200, 40], 2, 18, 16, HF)
    _narrow(x)
    lse = torch.cat([ref[2].view(2, 18) for ref in R.decode(x.ql, x.qp, x.cache, x.table, x.lens, 2)]).float()
    zero = torch.zeros(2, x.table.shape[1] * 16)
    base = _weights(x, bits, lse, zero)
    l2 = lse.clone()
    l2[0, 3], l2[2, 17] = -INF, NAN
    got = _weights(x, bits, l2, zero)
    assert (got[0, :199] < base[0, :199]).all() and torch.isfinite(got[0]).all()
    assert torch.isnan(got[1, :39]).all() and torch.equal(got[1, 39:], base[1, 39:])  # row 2 does not see the last token
    # the last token of sequence 0, seen by its 18 last rows only: a NaN there is nobody else's
    at = (int(x.table[0, 199 // 16]), 199 % 16)
    x.cache[at][5] = NAN
    x.bytes[at][256] = 255
    got = _weights(x, bits, lse, zero)
    assert torch.isnan(got[0, 199]) and torch.equal(got[0, :199], base[0, :199]) and torch.equal(got[1], base[1])


@pytest.mark.parametrize("seed", range(10))
def test_weights_any(seed):
    rng = random.Random(seed)
    H, S = rng.choice([1, 5, 16, 33, 64, 96, 128]), rng.choice([1, 1, 2, 5, 8])
    lens = [rng.choice([0, 1, S, rng.randint(1, 700)]) for _ in range(rng.choice([1, 3, 20, 66]))]
    x = Absorbed(lens, S, H, rng.choice([1, 3, 16, 64, 272]), rng.choice([BF, HF]), prefix=rng.choice([None, 40]), seed=seed)
    _check_weights(x, rng.choice([4, 16]))


def test_weights_in_wide_tables():
    """Tables with room for many more tokens than there are."""
    x = Absorbed([300, 5, 0, 129], 1, 12, 16, BF)
    _, _, lse = _check_weights(x, 4)
    W = x.table.shape[1] * 16
    a = _weights(x, 4, lse, torch.zeros(4, W))
    x.widen(1 << 16)
    b = _weights(x, 4, lse, torch.zeros(4, x.table.shape[1] * 16))
    assert torch.equal(a, b[:, :W]) and (b[:, W:] == 0).all()
    _check_weights(x, 4)


def test_weights_far_offsets():
    """Pages beyond 2^32 bytes of the cache; on another stream, with the weights of one row far from the next one's."""
    pages, size = 90000, 128  # 4.6 GB
    x = Absorbed([700, 90], 2, 20, size, BF)
    _, _, lse = _check_weights(x, 4)
    W = x.table.shape[1] * size
    want = _weights(x, 4, lse, torch.zeros(2, W))
    cache = torch.empty(pages, size, 400, dtype=torch.uint8, device=DEV)
    to = [pages - 1 - 3 * i for i in range(x.bytes.shape[0])]
    assert min(to) * size * 400 > 1 << 32
    cache[to] = x.bytes
    table = torch.where(x.table >= 0, torch.tensor(to)[x.table.clamp(min=0).long()].int(), x.table)
    far = torch.empty((1 << 30) + W + 64, device=DEV)  # row 1 begins 2^32 + 256 bytes behind row 0
    weights = far.as_strided((2, W), ((1 << 30) + 64, 1)).zero_()
    args = (x.ql.to(DEV), x.qp.to(DEV), cache, table.to(DEV), _i32(x.lens), lse.to(DEV), weights)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kda355.latent_weights(*args)
    side.synchronize()
    assert torch.equal(weights.cpu(), want)


def test_weights_refusals():
    x = _narrow(Absorbed([20, 5], 1, 4, 16, BF))
    ql, qp, table, lens = x.ql.to(DEV), x.qp.to(DEV), x.table.to(DEV), _i32(x.lens)
    lse, w = torch.zeros(2, 4, device=DEV), torch.zeros(2, table.shape[1] * 16, device=DEV)
    ok = dict(q_latent=ql, q_pe=qp, cache=x.bytes, block_table=table, seq_lens=lens, lse=lse, weights=w)
    kda355.latent_weights(**ok)
    for kw in (dict(weights=w[:, :-1]), dict(weights=w[:1]), dict(weights=w.t()), dict(weights=w[0]), dict(lse=lse[:, :3]), dict(lse=lse.t()),
               dict(weights=w[:1].expand(2, -1)), dict(seq_lens=lens[:1]), dict(q_latent=ql[..., :500]), dict(q_pe=qp[:1]),
               dict(cache=x.bytes[..., :300]), dict(block_table=table[0]), dict(scale=0.0), dict(scale=NAN), dict(scale=-1.0)):
        with pytest.raises(ValueError):
            kda355.latent_weights(**{**ok, **kw})
    for kw in (dict(weights=w.half()), dict(weights=w.cpu()), dict(lse=lse.double()), dict(lse=None), dict(weights=None), dict(q_latent=ql.float()),
               dict(cache=x.cache.half().to(DEV)), dict(block_table=table.long()), dict(seq_lens=lens.cpu())):
        with pytest.raises(TypeError):
            kda355.latent_weights(**{**ok, **kw})
    kda355.latent_weights(**ok)


# ================================================================================================ eviction
class Budget:
    """Sequences on scattered pages with their books; pools and weights whose values name their place."""

    def __init__(self, lens, size, layers=1, seed=0, token=(16,), dtype=torch.int32, spare=3, reserve=0, shared=(), ties=0.3, span=0):
        rng = random.Random(seed)
        self.size, need = size, [-(-n // size) for n in lens]
        width = max(max([1] + need) + reserve + 1, -(-span // size))
        pages = sum(need) + len(lens) * reserve + spare
        perm = list(range(pages))
        rng.shuffle(perm)
        self.lens, self.table, self.refs = list(lens), [], [0] * pages
        for n, k in enumerate(need):
            row = [perm.pop() for _ in range(k + reserve)]
            self.table.append(row + [-1] * (width - len(row)))
        for child, parent, k in shared:  # the first k pages of a parent
            self.table[child][:k] = self.table[parent][:k]
        for row in self.table:
            for g in row:
                if g >= 0:
                    self.refs[g] += 1
        gone = [p for p in range(pages) if not self.refs[p]]
        self.free, self.num = gone[::-1] + [-1] * (pages - len(gone)), len(gone)
        g = torch.Generator().manual_seed(seed)
        W = width * size
        self.pools = [torch.randint(-2 ** 31, 2 ** 31 - 1, (pages, size, *token), generator=g).to(dtype) for _ in range(layers)]
        self.mass = [torch.rand(len(lens), W + 3, generator=g) for _ in range(layers)]
        for w in self.mass:
            w[torch.rand(w.shape, generator=g) < ties] = 0.25
            w[torch.rand(w.shape, generator=g) < ties / 4] = 0.0
            w[torch.rand(w.shape, generator=g) < ties / 8] = -0.0

    def device(self, layout="dense"):
        d = dict(block_table=_i32(self.table), seq_lens=_i32(self.lens), ref_counts=_i32(self.refs), free_pages=_i32(self.free),
                 num_free=_i32([self.num]))
        pools, mass = [p.to(DEV) for p in self.pools], [w.to(DEV) for w in self.mass]
        if layout == "apart":  # pages and rows of weights and of the table with others between them
            for i, p in enumerate(pools):
                row = p[0].numel()
                pad = torch.full((p.shape[0], row + 16 // p.element_size() * 3), 7, dtype=p.dtype, device=DEV)
                view = pad.as_strided(p.shape, (pad.shape[1], *p.stride()[1:]))
                view.copy_(p)
                pools[i] = view
            mass = [torch.cat([w, torch.full((len(w), 6), 5.0, device=DEV)], dim=1)[:, :w.shape[1]] for w in mass]
            t = d["block_table"]
            d["block_table"] = torch.cat([t, torch.full_like(t, 77)], dim=1)[:, :t.shape[1]]
        return pools, mass, d

    def run(self, rows, keep, recent, layout="dense"):
        pools, mass, d = self.device(layout)
        kda355.evict_tokens(pools, mass, *d.values(), _i32(rows), keep, recent, self.size)
        return pools, mass, d

    def check(self, rows, keep, recent, layout="dense"):
        pools, mass, d = self.run(rows, keep, recent, layout)
        p0, w0 = [p.clone() for p in self.pools], [w.clone() for w in self.mass]
        lists = [[w[r].tolist() for r in range(len(w))] for w in w0]
        table, lens, refs, free = [list(r) for r in self.table], list(self.lens), list(self.refs), list(self.free)
        rows_of = [[[p[g, o] for o in range(self.size)] for g in range(p.shape[0])] for p in p0]
        rows_of = [[[t.clone() for t in page] for page in p] for p in rows_of]
        num = Q.evict(rows_of, lists, table, lens, refs, free, self.num, rows, keep, recent, self.size)
        assert d["block_table"].tolist() == table
        assert d["seq_lens"].tolist() == lens
        assert d["ref_counts"].tolist() == refs
        assert d["free_pages"].tolist() == free and d["num_free"].tolist() == [num]
        for got, want in zip(pools, rows_of):
            want = torch.stack([torch.stack(page) for page in want])
            assert torch.equal(got.cpu().view(torch.uint8) if got.dtype == torch.uint8 else got.cpu(), want)
        for got, want in zip(mass, lists):
            got, want = got.cpu(), torch.tensor(want)
            assert torch.equal(torch.isnan(got), torch.isnan(want))
            assert torch.equal(got.nan_to_num(3.0), want.nan_to_num(3.0))
        return lens


EVICT = [
    # lens, keep, recent, page size, layers
    ([2], 1, 0, 1, 1), ([2], 1, 1, 1, 1), ([5], 4, 2, 16, 1), ([17, 16, 15, 1, 0], 16, 4, 16, 2), ([64, 65, 130], 64, 0, 64, 1),
    ([64, 65, 130], 64, 64, 64, 1), ([300, 20, 299], 7, 3, 5, 3), ([1000, 1500], 600, 100, 16, 2), ([1100], 1030, 1025, 64, 1),
    ([2500, 90], 1200, 1150, 64, 1), ([4160], 4096, 256, 64, 1), ([3000, 2999], 1, 0, 100, 1), ([3000], 2999, 0, 100, 1),
    ([3000], 2999, 2999, 272, 1), ([40] * 70, 30, 5, 8, 2), ([2000], 1024, 0, 16, 1), ([2049, 2048], 1000, 24, 16, 1),
]


@pytest.mark.parametrize("lens,keep,recent,size,layers", EVICT, ids=[f"{len(c[0])}seq-{max(c[0])}-to{c[1]}-r{c[2]}-p{c[3]}" for c in EVICT])
@pytest.mark.parametrize("layout", ["dense", "apart"])
def test_evict(lens, keep, recent, size, layers, layout):
    x = Budget(lens, size, layers, token=(4,), seed=sum(lens))
    after = x.check(list(range(len(lens))), keep, recent, layout)
    assert after == [min(n, keep) for n in lens]


@pytest.mark.parametrize("token,dtype", [((400,), torch.uint8), ((ROW,), torch.int16), ((2, 3, 8), torch.int32), ((4,), torch.int32),
                                         ((33, 4), torch.int32)])
def test_evict_token_rows(token, dtype):
    """Rows of 400 bytes, of 1152, of 16 and of odd counts of 16."""
    x = Budget([300, 70, 180], 16, 2, token=token, dtype=dtype)
    x.check([0, 1, 2], 64, 9)


def test_evict_layers_of_different_rows():
    x = Budget([300, 70, 180], 16, 3, token=(4,))
    x.pools[1] = torch.randint(0, 255, (len(x.refs), 16, 400), dtype=torch.uint8)
    x.pools[2] = torch.randint(0, 255, (len(x.refs), 16, 7, 8), dtype=torch.int16)
    x.check([0, 1, 2], 100, 30)


@pytest.mark.parametrize("layers", [24, 25, 50])
def test_evict_many_layers(layers):
    """More layers than a launch takes: the books change once."""
    Budget([90, 30, 55], 8, layers, token=(4,)).check([0, 1, 2], 40, 11)


@pytest.mark.parametrize("ties", [0.0, 1.0, 4.0])
def test_evict_ties_and_odd_weights(ties):
    """Equal weights, zeros of both signs, NaN, infinities, negative and subnormal numbers."""
    x = Budget([700, 650], 16, 1, token=(4,), ties=ties)
    x.check([0, 1], 500, 20)
    w = x.mass[0]
    w[0, 5:600:7], w[0, 6:600:9], w[0, 7:600:11], w[0, 8:600:13] = NAN, -INF, INF, 1e-42
    w[1, :300] = NAN
    w[1, 300:] = -w[1, 300:]
    for keep in (30, 200, 301, 500, 649):
        x.check([0, 1], keep, 7)


def test_evict_shared_pages_stay():
    """Pages that others hold too stay whole, in front; where they and the recent tokens are too many nothing changes."""
    shared = [(1, 0, 5), (2, 0, 5), (3, 0, 2)]
    x = Budget([400, 333, 90, 300, 200], 16, 2, token=(4,), shared=shared, reserve=1)
    assert x.check([0, 1, 2, 3, 4], 200, 100) == [200, 200, 90, 200, 200]
    assert x.check([0, 1, 2, 3, 4], 120, 40) == [120, 120, 90, 120, 120]  # (fixed = left)
    assert x.check([0, 1, 2, 3, 4], 120, 41) == [400, 333, 90, 120, 120]
    assert x.check([0, 1, 2, 3, 4], 79, 0) == [400, 333, 90, 79, 79]


def test_evict_holes_rows_outside_and_twice():
    x = Budget([100, 100, 100, 100], 16, 1, token=(4,))
    for row, col, what in ((0, 2, -1), (1, 6, len(x.refs)), (2, 7, -1)):  # (column 7 is behind the tokens)
        x.refs[x.table[row][col]] -= x.table[row][col] >= 0
        x.table[row][col] = what
    assert x.check([3, -1, 2, 4, 0, 3, 1, 1 << 30, 2, 3, -(1 << 31)], 50, 10) == [100, 100, 50, 50]


def test_evict_reserved_pages_move_down():
    x = Budget([100, 20, 64], 16, 1, token=(4,), reserve=3)
    pools, mass, d = x.run([0, 1, 2], 40, 10)
    assert d["block_table"].tolist()[0][:6] == x.table[0][:3] + x.table[0][7:10]
    x.check([0, 1, 2], 40, 10)


def test_evict_lengths_past_the_table():
    x = Budget([64, 30], 16, 1, token=(4,))
    x.table = [r[:4] for r in x.table]
    x.lens = [1 << 30, -3]
    assert x.check([0, 1], 20, 4) == [20, -3]


def test_evict_nothing():
    x = Budget([64, 30], 16, 1, token=(4,))
    assert x.check([], 20, 4) == [64, 30]
    assert x.check([0, 1], 64, 4) == [64, 30]
    assert x.check([0, 1], 1 << 29, 4) == [64, 30]


@pytest.mark.parametrize("seed", range(14))
def test_evict_any(seed):
    rng = random.Random(seed)
    size = rng.choice([1, 3, 16, 64, 100])
    lens = [rng.randint(0, rng.choice([40, 700, 1500])) for _ in range(rng.choice([1, 2, 9, 33]))]
    shared = [(n, 0, min(2, lens[n] // size, lens[0] // size)) for n in range(1, len(lens)) if rng.random() < 0.3]
    x = Budget(lens, size, rng.choice([1, 2, 4]), seed=seed, token=(4,), reserve=rng.choice([0, 2]), shared=shared)
    keep = rng.randint(1, max(2, max(lens)))
    rows = list(range(len(lens)))
    rng.shuffle(rows)
    x.check(rows, keep, rng.randint(0, keep))


@pytest.mark.parametrize("n", [40000, 70001, 140000])
def test_evict_long(n):
    """Sequences whose weights no workgroup holds at once; every byte of the weights' keys decides somewhere."""
    x = Budget([n, n // 3], 272, 1, token=(4,), seed=n)
    x.mass[0][0, :n // 2] = 1.0 + torch.arange(n // 2) * 2.0 ** -23  # neighbouring numbers
    for keep, recent in ((n // 4, n // 16), (n - 100, 3000), (n // 2, 0)):
        pools, mass, d = x.run([0, 1], keep, recent)
        left, w = keep - recent, x.mass[0][0, :n]
        order = torch.sort(w[:n - recent], descending=True, stable=True).indices[:left]
        stays = torch.zeros(n - recent, dtype=torch.bool)
        stays[order] = True
        place = torch.arange(keep)
        place[torch.nonzero(~stays[:left]).flatten()] = left + torch.nonzero(stays[left:]).flatten()
        place[left:] = torch.arange(n - recent, n)
        assert torch.equal(mass[0][0, :keep].cpu(), w[place]) and (mass[0][0, keep:n] == 0).all()
        t = torch.tensor(x.table[0])
        flat = x.pools[0].view(-1, 4)
        at = lambda j: t[j // 272] * 272 + j % 272  # noqa: E731
        assert torch.equal(pools[0].cpu().view(-1, 4)[at(torch.arange(keep))], flat[at(place)])
        assert d["seq_lens"].tolist()[0] == keep


def _cut(w, n, fixed, keep, recent):
    """Where the tokens of a row of n come from after a cut, by torch's stable sort."""
    left = keep - recent
    order = fixed + torch.sort(w[fixed:n - recent], descending=True, stable=True).indices[:left - fixed]
    stays = torch.zeros(n - recent, dtype=torch.bool)
    stays[:fixed], stays[order] = True, True
    place = torch.arange(keep)
    place[torch.nonzero(~stays[:left]).flatten()] = left + torch.nonzero(stays[left:]).flatten()
    place[left:] = torch.arange(n - recent, n)
    return place


@pytest.mark.parametrize("n,kind", [(540000, "ties"), (600000, "few"), (1100000, "ties"), (700001, "heads"), (1000000, "none")])
def test_evict_beyond_64_parts(n, kind):
    """More parts of a sequence than a wave has lanes (540672 tokens): how many ties, places and movers stand before a part goes from one
    64 of them to the next.  Ties alone; a few heavier tokens between them; all movers behind the first 64 parts; neighbouring numbers.  Rows
    of other lengths beside it, one of them with shared pages, another left as it is; all books and both layers' rows and weights."""
    size = 272
    lens = [n, 9000, n // 3, 700]
    x = Budget(lens, size, 2, token=(4,), seed=n, shared=[(2, 0, 5)], reserve=1)
    g = torch.Generator().manual_seed(n + 1)
    for w in x.mass:
        W = w.shape[1]
        if kind == "ties":
            w[:] = (torch.rand(w.shape, generator=g) < 0.5).float()
        elif kind == "few":
            w[:] = 0.25
            w[0, torch.randint(0, n, (500,), generator=g)] = 1.0
            w[0, torch.randint(0, n, (500,), generator=g)] = 0.0
        elif kind == "heads":
            w[0] = torch.arange(W).float()
        else:
            w[0] = 1.0 + torch.randperm(W, generator=g) * 2.0 ** -23
    for keep, recent in ((n // 2, n // 50), (n - 5000, 9000), (7 * size, 0)):
        pools, mass, d = x.run([3, 0, 2, 1, 0], keep, recent)
        after, table, refs, gone = list(lens), [list(r) for r in x.table], list(x.refs), []
        for l in range(2):
            want, rows = x.mass[l].clone(), x.pools[l].view(-1, 4).clone()
            for r, length in enumerate(lens):
                if length <= keep:
                    continue
                fixed = 5 * size if r in (0, 2) else 0
                place = _cut(x.mass[l][r], length, fixed, keep, recent)
                t = torch.tensor(x.table[r])
                at = lambda j: t[j // size] * size + j % size  # noqa: E731
                rows[at(torch.arange(keep))] = x.pools[l].view(-1, 4)[at(place)]
                want[r, :keep] = x.mass[l][r][place]
                want[r, keep:length] = 0
            assert torch.equal(pools[l].cpu().view(-1, 4), rows)
            assert torch.equal(mass[l].cpu(), want)
        for r, length in enumerate(lens):
            if length > keep:
                kept, used = -(-keep // size), -(-length // size)
                gone += table[r][kept:used]
                table[r] = table[r][:kept] + table[r][used:] + [-1] * (used - kept)
                after[r] = keep
        for page in gone:
            refs[page] = 0
        free = x.free[:x.num] + sorted(gone, reverse=True)
        assert d["seq_lens"].tolist() == after and d["block_table"].tolist() == table and d["ref_counts"].tolist() == refs
        assert d["num_free"].tolist() == [len(free)] and d["free_pages"].tolist() == free + [-1] * (len(refs) - len(free))


@pytest.mark.parametrize("seed", range(8))
def test_evict_any_in_wide_tables(seed):
    """Tables with room for more tokens than a workgroup selects from: the sequences are short, or end behind the first 8192 tokens."""
    rng = random.Random(seed)
    size = rng.choice([16, 64, 100])
    lens = [rng.randint(0, rng.choice([700, 1500])) for _ in range(rng.choice([1, 2, 9]))] + [rng.choice([8190, 8200, 9500])]
    shared = [(n, 0, min(2, lens[n] // size, lens[0] // size)) for n in range(1, len(lens)) if rng.random() < 0.3]
    x = Budget(lens, size, rng.choice([1, 2]), seed=seed, token=(4,), reserve=rng.choice([0, 2]), shared=shared, span=40000,
               ties=rng.choice([0.1, 1.0]))
    if seed % 2:
        x.mass[0][:, 1:900:5], x.mass[0][0, 2:900:7] = NAN, -INF
    keep = rng.randint(1, max(lens)) if seed % 4 else max(lens) - 9
    rows = list(range(len(lens)))
    rng.shuffle(rows)
    x.check(rows + rows[:1], keep, rng.randint(0, keep))


def test_evict_many_rows_in_wide_tables():
    """More sequences and layers than one run of the selecting workgroups takes."""
    lens = [20 + n % 60 for n in range(47)]
    x = Budget(lens, 16, 24, seed=3, token=(4,), span=20000)
    assert x.check(list(range(47)), 40, 11) == [min(n, 40) for n in lens]


@pytest.mark.parametrize("layers,B,size,span,keep,recent", [(24, 130, 16, 16384, 7000, 30), (24, 47, 16, 20000, 400, 0),
                                                            (3, 48, 272, 300000, 125000, 64)])
def test_evict_in_runs(layers, B, size, span, keep, recent):
    """More lists of pairs than are held at a time (100, 42 and 44 rows): a call is the calls for a few of its rows, one after the other,
    but for the order in which pages come onto the stack.  Rows given twice stand in different runs."""
    x = Budget([keep - 20 + (7 * n) % 500 for n in range(B)], size, layers, seed=layers, token=(4,), shared=[(9, 2, 1), (B - 1, 2, 1)])
    width = span // size
    outs = []
    for parts in (1, 5):
        pools, _, d = x.device()
        g = torch.Generator(device=DEV).manual_seed(layers)
        mass = [torch.rand(B, width * size, generator=g, device=DEV) for _ in range(layers)]
        d["block_table"] = torch.cat([d["block_table"], _i32([[-1] * (width - d["block_table"].shape[1])] * B)], dim=1)
        order = list(range(B)) + [0, B // 2]
        step = -(-len(order) // parts)
        for i in range(0, len(order), step):
            kda355.evict_tokens(pools, mass, *d.values(), _i32(order[i:i + step]), keep, recent, size)
        top = int(d["num_free"])
        d["free_pages"][:top] = d["free_pages"][:top].sort().values
        outs.append([*pools, *mass, *d.values()])
        assert d["seq_lens"].tolist() == [min(n, keep) for n in x.lens]
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def test_evict_far_offsets():
    """Pages beyond 2^32 bytes of the pool, on another stream."""
    pages, size = 90000, 128  # 4.6 GB
    x = Budget([700, 300, 129], size, 1, token=(400,), dtype=torch.uint8)
    for keep, recent in ((260, 30), (128, 100), (600, 500)):
        pools, mass, d = x.run([0, 1, 2], keep, recent)
        to = [pages - 1 - 3 * i for i in range(len(x.refs))]
        assert min(to) * size * 400 > 1 << 32
        cache = torch.empty(pages, size, 400, dtype=torch.uint8, device=DEV)
        cache[to] = x.pools[0].to(DEV)
        table = _i32([[to[g] if g >= 0 else -1 for g in row] for row in x.table])
        refs = torch.zeros(pages, dtype=torch.int32, device=DEV)
        refs[to] = _i32(x.refs)
        free, num, lens = torch.full((pages,), -1, dtype=torch.int32, device=DEV), _i32([0]), _i32(x.lens)
        w, rows = x.mass[0].to(DEV), _i32([0, 1, 2])
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            kda355.evict_tokens([cache], [w], table, lens, refs, free, num, rows, keep, recent, size)
        side.synchronize()
        assert torch.equal(cache[to], pools[0]) and torch.equal(w, mass[0]) and torch.equal(lens, d["seq_lens"])
        assert torch.equal(refs[to], d["ref_counts"]) and int(num) == int(d["num_free"]) - x.num
        assert table.tolist() == [[to[g] if g >= 0 else -1 for g in row] for row in d["block_table"].tolist()]


@pytest.mark.parametrize("span", [0, 20000])
def test_evict_captured(span):
    """One graph, replayed over other lengths, tables and weights; every replay against the eager call."""
    xs = [Budget(lens, 16, 2, seed=s, token=(4,), spare=40 - sum(-(-n // 16) for n in lens), reserve=0, span=span)
          for s, lens in enumerate(([100, 40, 7], [3, 200, 60], [150, 2, 133]))]
    width = max(len(x.table[0]) for x in xs)
    pools, mass, d = Budget([150] * 3, 16, 2, token=(4,), spare=40 - 30, span=16 * width).device()
    rows = _i32([2, 0, 1])

    def step():
        kda355.evict_tokens(pools, mass, *d.values(), rows, 50, 12, 16)

    def load(x):
        for a, b in zip(pools, x.pools):
            a.copy_(b)
        for a, b in zip(mass, x.mass):
            a.zero_()
            a[:, :b.shape[1]] = b
        d["block_table"].fill_(-1)
        d["block_table"][:, :len(x.table[0])] = _i32(x.table)
        for name, v in (("seq_lens", x.lens), ("ref_counts", x.refs), ("free_pages", x.free), ("num_free", [x.num])):
            d[name].copy_(_i32(v))

    load(xs[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for x in xs + xs:
        load(x)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (*pools, *mass, *d.values())]
        load(x)
        step()
        for a, b in zip(got, (*pools, *mass, *d.values())):
            assert torch.equal(a, b)
        assert d["seq_lens"].tolist() == [min(n, 50) for n in x.lens]


def test_evict_refusals():
    x = Budget([64, 30], 16, 2, token=(4,))
    pools, mass, d = x.device()
    rows = _i32([0, 1])

    def call(p=pools, w=mass, keep=20, recent=4, size=16, r=rows, **kw):
        kda355.evict_tokens(p, w, *{**d, **kw}.values(), r, keep, recent, size)

    W = mass[0].shape[1]
    short = [mass[0][:, :len(x.table[0]) * 16 - 1]] * 2
    for kw in (dict(keep=0), dict(recent=-1), dict(recent=21), dict(size=8), dict(size=0), dict(p=pools[:1]), dict(p=[], w=[]), dict(w=short),
               dict(w=[m[:1] for m in mass]), dict(w=[m.t() for m in mass]), dict(w=[m[:1].expand(2, W) for m in mass]),
               dict(p=[q[:3] for q in pools]), dict(p=[q[:, ::2] for q in pools]), dict(p=[q[..., :3] for q in pools]),
               dict(p=[torch.zeros(len(x.refs), 16, 2, dtype=torch.int32, device=DEV)] * 2), dict(p=[q.view(len(x.refs), -1) for q in pools]),
               dict(p=pools[:1] * 2), dict(w=mass[:1] * 2), dict(seq_lens=d["seq_lens"][:1]), dict(free_pages=d["free_pages"][:2]), dict(num_free=d["free_pages"]), dict(r=rows[None])):
        with pytest.raises(ValueError):
            call(**kw)
    for kw in (dict(w=[m.half() for m in mass]), dict(w=[m.cpu() for m in mass]), dict(p=[q.cpu() for q in pools]), dict(r=rows.long()),
               dict(p=[None, None]), dict(w=[None, None]), dict(seq_lens=d["seq_lens"].long()), dict(block_table=d["block_table"].cpu())):
        with pytest.raises(TypeError):
            call(**kw)
    assert d["seq_lens"].tolist() == [64, 30]
    call()
    assert d["seq_lens"].tolist() == [20, 20]


@pytest.mark.parametrize("keep,recent", [((1 << 32) + 20, 4), ((1 << 63) - 1, 4), (20, (1 << 32) + 4), (1 << 31, 1 << 31)])
def test_evict_budgets_beyond_32_bits(keep, recent):
    x = Budget([64, 30], 16, 2, token=(4,))
    pools, mass, d = x.device()
    for _ in range(2):  # (nothing is kept of a call that was refused)
        with pytest.raises(ValueError, match="32 bits"):
            kda355.evict_tokens(pools, mass, *d.values(), _i32([0, 1]), keep, recent, 16)
    assert d["seq_lens"].tolist() == [64, 30]
    assert x.check([0, 1], (1 << 29), 4) == [64, 30]


# ================================================================================================ together
@pytest.mark.parametrize("bits,dtype", [(16, BF), (4, BF), (4, HF)])
def test_a_sequence_under_a_budget(bits, dtype):
    """Steps of append, decode, weights and eviction, beside a plain model that keeps each token's row and weight in lists: what the
    layers attend to after every step, and the pages held, are the model's."""
    size, H, keep, recent, layers, B = 16, 6, 40, 8, 2, 3
    g = torch.Generator().manual_seed(11)
    rnd = lambda *shape: torch.randn(*shape, generator=g).to(dtype)  # noqa: E731
    pages, width = 20, 5
    row = 400 if bits == 4 else ROW
    pools = [torch.zeros(pages, size, row, dtype=torch.uint8 if bits == 4 else dtype, device=DEV) for _ in range(layers)]
    mass = [torch.zeros(B, width * size, device=DEV) for _ in range(layers)]
    table, lens = torch.full((B, width), -1, dtype=torch.int32, device=DEV), _i32([0] * B)
    refs, free, num = _i32([0] * pages), _i32(list(range(pages))), _i32([pages])
    kept = [[[] for _ in range(B)] for _ in range(layers)]  # (row of 576 values in the type, weight, the kernel's weight)
    evicted = 0
    for step, new in enumerate([30, 9, 1, 8, 1, 1, 17, 5, 1, 12, 12]):
        # pages for the new tokens from the stack, on the host as a scheduler does
        t, n, top = table.tolist(), lens.tolist(), int(num)
        stack = free.tolist()
        slots = []
        for r in range(B):
            for j in range(n[r], n[r] + new):
                if j % size == 0 and t[r][j // size] < 0:
                    top -= 1
                    t[r][j // size], stack[top] = stack[top], -1
                    refs[t[r][j // size]] = 1
                slots.append(t[r][j // size] * size + j % size)
        table.copy_(_i32(t)), free.copy_(_i32(stack)), num.fill_(top)
        lens += new
        for layer in range(layers):
            latent, pe = rnd(B * new, LAT), rnd(B * new, PE)
            kda355.latent_append(latent.to(DEV), pe.to(DEV), pools[layer], torch.tensor(slots, device=DEV))
            rows = Q.values(Q.rounded(latent, pe), dtype) if bits == 4 else torch.cat([latent, pe], dim=1)
            S = min(new, 4)
            ql, qp = rnd(B * S, H, LAT), rnd(B * S, H, PE)
            lse = torch.empty(B * S, H, device=DEV)
            out = kda355.latent_decode(ql.to(DEV), qp.to(DEV), pools[layer], table, lens, lse=lse)
            kda355.latent_weights(ql.to(DEV), qp.to(DEV), pools[layer], table, lens, lse, mass[layer])
            for r in range(B):
                seen = kept[layer][r]
                seen += [[rows[r * new + i].double(), 0.0] for i in range(new)]
                have = torch.stack([x[0] for x in seen])
                q = torch.cat([ql, qp], dim=-1)[r * S:(r + 1) * S].double().reshape(S * H, ROW)
                vis = torch.arange(len(seen))[None] < len(seen) - (S - 1 - torch.arange(S).repeat_interleave(H))[:, None]
                ref = R.attend(q, have, have[:, :LAT], vis, SCALE)
                R.check(out[r * S:(r + 1) * S].cpu().reshape(S * H, LAT), lse[r * S:(r + 1) * S].cpu().reshape(-1), ref, dtype, ROW,
                        f"step {step} layer {layer} seq {r}")
                z = torch.where(vis, q @ have.T * SCALE, torch.tensor(-INF, dtype=torch.float64))
                w = torch.softmax(z, dim=1).sum(dim=0)
                for x, a in zip(seen, w.tolist()):
                    x[1] += a
                got = mass[layer][r].cpu().double()
                want = torch.tensor([x[1] for x in seen], dtype=torch.float64)
                # scores of up to Z = 40, weights of 24 rows a step: dz twice (here and in lse) and the additions
                assert (got[:len(seen)] - want).abs().max() < (step + 1) * 24 * (4 * ROW * 40 + 64) * 2.0 ** -24
                assert (got[len(seen):] == 0).all()
        before = [m.cpu().clone() for m in mass]
        kda355.evict_tokens(pools, mass, table, lens, refs, free, num, _i32(list(range(B))), keep, recent, size)
        for layer in range(layers):
            for r in range(B):
                seen, w = kept[layer][r], before[layer][r].tolist()
                n = len(seen)
                if n <= keep:
                    continue
                evicted += n - keep
                left = keep - recent
                stays = set(sorted(range(n - recent), key=lambda j: (-w[j], j))[:left])
                place = list(range(keep))
                for a, b in zip([j for j in range(left) if j not in stays], [j for j in range(left, n - recent) if j in stays]):
                    place[a] = b
                place[left:] = range(n - recent, n)
                kept[layer][r] = [seen[j] for j in place]
        want = [len(kept[0][r]) for r in range(B)]
        assert lens.tolist() == want and int(num) == pages - sum(-(-n // size) for n in want)
        assert int(refs.sum()) == sum(-(-n // size) for n in want)
    assert evicted > 100
