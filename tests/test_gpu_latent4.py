"""The latent cache in 4 bits: rows rounded into pages and read back, bit for bit against a plain form, and attention over them against
float64 (tolerances of latent_ref; the widened rows are numbers of the 16-bit type).  Where values are not finite: what is not
finite in the outputs against the same call over the widened cache, which has tests of its own."""
import random

import pytest
import torch

import kda355
import latent4_ref as Q
import latent_ref as R
from latent_ref import LAT, PE, ROW, SCALE
from test_gpu_latent import DECODE, Absorbed, _i32, _randn

pytestmark = pytest.mark.gpu
DEV, BF, HF = "cuda", torch.bfloat16, torch.float16
NAN, INF = float("nan"), float("inf")


def _same(a, b):
    """The same bits, and any NaN for a NaN."""
    a, b = a.cpu(), b.cpu()
    na, nb = torch.isnan(a), torch.isnan(b)
    assert torch.equal(na, nb)
    kind = {2: torch.int16, 4: torch.int32}[a.element_size()]
    assert torch.equal(a.contiguous().view(kind)[~na], b.contiguous().view(kind)[~nb])


# ================================================================================================ rows
def _rows_of_all_kinds(dtype):
    """Rows of 512 values where rounding can go wrong: ties and both their neighbours at several scales, largest values around 6, 7 and 8
    steps, zeros of both signs, the smallest and the largest numbers, infinities and NaN."""
    info = torch.finfo(dtype)
    out = [torch.zeros(LAT), -torch.zeros(LAT), torch.full((LAT,), info.tiny), torch.full((LAT,), info.max), torch.full((LAT,), -info.max)]
    small = torch.tensor([info.tiny * info.eps * k for k in range(LAT)], dtype=torch.float64)  # subnormal numbers
    out.append(small)
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0], dtype=torch.float64)
    for scale in (1.0, 2.0 ** -9, 2.0 ** 9):
        for top in (4.0, 5.0, 6.0, 6.96875, 7.0, 7.03125, 7.96875):
            near = torch.cat([ties, ties * (1 + info.eps), ties * (1 - info.eps / 2), torch.tensor([0.0, -0.0, 0.1, 2.2, 3.0, 0.5, 1.0])])
            row = torch.cat([near, torch.tensor([top], dtype=torch.float64)])[:32]
            row[-1] = top
            row = torch.where(row.abs() > top, torch.zeros_like(row), row).repeat(16)
            out.append(row * scale * torch.where(torch.arange(LAT) % 3 == 0, -1.0, 1.0))
    x = torch.stack([r.double() for r in out]).to(dtype)
    odd = _randn(6, LAT, dtype=dtype, seed=5)
    odd[0, 7], odd[1, 100], odd[2, 511], odd[3, 0] = INF, -INF, NAN, NAN
    odd[4, 32:64] = NAN
    return torch.cat([x, odd, _randn(40, LAT, dtype=dtype, seed=6)])


@pytest.mark.parametrize("dtype", [BF, HF])
def test_append_rounds(dtype):
    latent = _rows_of_all_kinds(dtype)
    T = latent.shape[0]
    pe = _randn(T, PE, dtype=dtype, seed=7)
    pe[3, 5], pe[4, 6] = NAN, INF
    cache = torch.full((T // 5 + 1, 5, 400), 170, dtype=torch.uint8, device=DEV)
    kda355.latent_append(latent.to(DEV), pe.to(DEV), cache, torch.arange(T, device=DEV))
    assert torch.equal(cache.view(-1, 400)[:T].cpu(), Q.rounded(latent, pe))
    assert (cache.view(-1, 400)[T:] == 170).all()


@pytest.mark.parametrize("dtype", [BF, HF])
def test_append_and_gather_at_the_ends_of_the_type(dtype):
    latent = Q.ends(dtype)
    T = len(latent)
    pe = _randn(T, PE, dtype=dtype, seed=8)
    cache = torch.zeros(T, 1, 400, dtype=torch.uint8, device=DEV)
    kda355.latent_append(latent.to(DEV), pe.to(DEV), cache, torch.arange(T, device=DEV))
    rows = Q.rounded(latent, pe)
    assert torch.equal(cache.cpu()[:, 0], rows)
    out = torch.empty(T, ROW, dtype=dtype, device=DEV)
    kda355.latent_gather(cache, torch.arange(T, dtype=torch.int32, device=DEV)[None], _i32([0, T]), out)
    assert torch.isfinite(out).all()
    _same(out, Q.values(rows, dtype))


@pytest.mark.parametrize("T,pages,size,dtype", [(1, 1, 1, BF), (7, 5, 3, HF), (8, 2, 16, BF), (9, 4, 7, BF), (100, 9, 16, HF)])
def test_append_anywhere(T, pages, size, dtype):
    """Views of wider rows, pages apart, slots in any order and outside."""
    g = torch.Generator().manual_seed(T)
    wide = _randn(T, 600, dtype=dtype, seed=T)
    latent, pe = wide[:, :LAT], wide[:, LAT:LAT + PE]
    slots = torch.randperm(pages * size, generator=g)[:T]
    slots = torch.cat([slots, torch.full((T - len(slots),), -1, dtype=torch.int64)])
    for i, bad in enumerate((-1, pages * size, 1 << 40, -(1 << 50))):
        if T > 3 * i + 4:
            slots[3 * i + 2] = bad
    buf = torch.full((pages, size * 400 + 48), 9, dtype=torch.uint8, device=DEV)
    cache = buf.as_strided((pages, size, 400), (buf.shape[1], 400, 1))
    dev = wide.to(DEV)
    assert kda355.latent_append(dev[:, :LAT], dev[:, LAT:LAT + PE], cache, slots.to(DEV)) is cache
    want = torch.full((pages, size * 400 + 48), 9, dtype=torch.uint8)
    rows = Q.rounded(latent, pe)
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < pages * size:
            want[s // size, s % size * 400:(s % size + 1) * 400] = rows[t]
    assert torch.equal(buf.cpu(), want)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_gather_any_bytes(dtype):
    """Every code under every scale, rounded to the type; NaN groups; holes, lengths past the table, rows past the last one."""
    cache = torch.randint(0, 256, (40, 16, 400), dtype=torch.uint8, generator=torch.Generator().manual_seed(1))
    cache.view(-1, 400)[:, 256:272] = (torch.arange(640)[:, None] * 16 + torch.arange(16)) % 256
    cache.view(-1, 400)[:, :256] = torch.arange(256, dtype=torch.uint8)
    table = torch.full((4, 12), -1, dtype=torch.int32)
    perm = torch.randperm(40, generator=torch.Generator().manual_seed(2)).int()
    table[0, :11], table[1, 0], table[2, :12], table[3, :6] = perm[:11], perm[11], perm[12:24], perm[24:30]
    table[0, 4], table[2, 3], table[3, 2] = 40, -3, 1 << 30
    lens = [170, 0, 12 * 16 + 30, 90]
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    out = torch.full((cu[-1] + 3, ROW + 8), 3.0, dtype=dtype, device=DEV)
    got = kda355.latent_gather(cache.to(DEV), table.to(DEV), _i32(cu), out[:, :ROW])
    want = torch.zeros(cu[-1], ROW, dtype=dtype)
    wide = Q.values(cache, dtype)
    for n, length in enumerate(lens):
        for j in range(min(length, 12 * 16)):
            p = int(table[n, j // 16])
            if 0 <= p < 40:
                want[cu[n] + j] = wide[p, j % 16]
    _same(got[:cu[-1]], want)
    assert (out[cu[-1]:] == 3.0).all() and (out[:, ROW:] == 3.0).all()


def test_append_and_gather_nothing():
    cache = torch.full((2, 4, 400), 7, dtype=torch.uint8, device=DEV)
    empty = torch.empty(0, LAT, dtype=BF, device=DEV)
    kda355.latent_append(empty, torch.empty(0, PE, dtype=BF, device=DEV), cache, torch.empty(0, dtype=torch.int64, device=DEV))
    kda355.latent_gather(cache, _i32([[0, 1]]), _i32([0, 0]), torch.empty(0, ROW, dtype=BF, device=DEV))
    torch.cuda.synchronize()
    assert (cache == 7).all()


# ================================================================================================ attention
def _narrow(x):
    """The case's cache in 4 bits: x.cache becomes what its rows stand for, x.bytes the rows."""
    flat = x.cache.reshape(-1, ROW)
    dev = flat.to(DEV)
    buf = torch.empty(flat.shape[0], 1, 400, dtype=torch.uint8, device=DEV)  # (the rounding has its own tests)
    kda355.latent_append(dev[:, :LAT], dev[:, LAT:], buf, torch.arange(flat.shape[0], device=DEV))
    x.bytes = buf.view(x.cache.shape[0], x.size, 400)
    x.cache = Q.values(x.bytes.cpu(), x.dtype)
    return x


def _run4(x, wide=False, workspace=None, scale=None, cache=None):
    ql, qp, cache, table = x.ql.to(DEV), x.qp.to(DEV), x.bytes if cache is None else cache, x.table.to(DEV)
    out = None
    if wide:  # queries as one 576-wide tensor, pages and table rows apart, an output between other values
        both = torch.cat([ql, qp], dim=-1)
        ql, qp = both[..., :LAT], both[..., LAT:]
        page = torch.full((cache.shape[0], x.size * 400 + 80), 255, dtype=torch.uint8, device=DEV)
        view = page.as_strided(cache.shape, (page.shape[1], 400, 1))
        view.copy_(cache)
        cache = view
        table = torch.cat([table, torch.full_like(table, 1 << 20)], dim=1)[:, :table.shape[1]]
        out = torch.full((ql.shape[0], x.H + 1, LAT + 8), 3.0, dtype=x.dtype, device=DEV)[:, 1:, :LAT]
    lse = torch.full((ql.shape[0], x.H), 7.0, device=DEV)
    kw = {}
    if x.prefix is not None:
        kw = dict(prefix_table=x.prefix_table.to(DEV), prefix_len=_i32([x.prefix]))
    o = kda355.latent_decode(ql, qp, cache, table, _i32(x.lens), scale, out=out, lse=lse, workspace=workspace, **kw)
    return o, lse


def _check4(x, what="", **kw):
    o, lse = _run4(x, **kw)
    S, H = x.S, x.H
    oc, lc = o.cpu(), lse.cpu()
    for n, ref in enumerate(R.decode(x.ql, x.qp, x.cache, x.table, x.lens, S, prefix_table=x.prefix_table, prefix_len=x.prefix or 0)):
        R.check(oc[n * S:(n + 1) * S].reshape(S * H, LAT), lc[n * S:(n + 1) * S].reshape(S * H), ref, x.dtype, ROW, f"{what} seq {n}")
    return o, lse


def _like_the_widened(x, o, lse):
    """What is not finite stands where the call over the widened cache has it; the rest is near that: both are off from the exact
    result by latent_ref's tolerance at most, whose weights add up to one and so A to the largest value."""
    o16, lse16 = x.run()
    u, f = torch.finfo(x.dtype).eps / 2, 2.0 ** -24
    size = x.cache.double().nan_to_num(0, 0, 0).abs()
    Z = SCALE * torch.cat([x.ql, x.qp], dim=-1).double().abs().sum(dim=-1).max() * size.max()
    L = x.table.shape[1] * x.size + (x.prefix or 0)
    for a, b, tol in ((o, o16, 2 * (2 * u + (2 * ROW * Z + 2 * L + 9) * f) * size.max()), (lse, lse16, 2 * (ROW * Z + L + 16 + 4 * Z) * f)):
        a, b = a.cpu().double(), b.cpu().double()
        for kind in (torch.isnan, torch.isposinf, torch.isneginf):
            assert torch.equal(kind(a), kind(b))
        fine = torch.isfinite(a)
        assert ((a - b).abs()[fine] <= tol).all()


IDS = [f"{len(c[0])}seq-{max(c[0])}-S{c[1]}-H{c[2]}-p{c[3]}" for c in DECODE]


@pytest.mark.parametrize("lens,S,H,size", DECODE, ids=IDS)
@pytest.mark.parametrize("dtype", [BF, HF])
def test_decode_lengths(lens, S, H, size, dtype):
    _check4(_narrow(Absorbed(lens, S, H, size, dtype)))


@pytest.mark.parametrize("lens,S,H,size", DECODE, ids=IDS)
def test_decode_lengths_in_wide_tables(lens, S, H, size):
    """Tables with room for many more tokens: groups of 64 rows."""
    _check4(_narrow(Absorbed(lens, S, H, size, BF)).widen())


@pytest.mark.parametrize("n", [1, 31, 32, 33, 64, 65, 96, 97, 128, 129, 160, 161, 192, 193, 224, 225, 256, 257, 300])
@pytest.mark.parametrize("H", [12, 64])
def test_decode_tiles_of_a_run(n, H):
    """Runs of one tile, of two, ...: every fill of the rings that the tiles pass through, in one workgroup's run and in several."""
    x = _narrow(Absorbed([n, n + 2000], 1, H, 16, BF))
    _check4(x)
    _check4(x.widen())


@pytest.mark.parametrize("lens,S,H,size", [([400, 90], 1, 12, 64), ([130, 77, 1], 4, 16, 16), ([513], 1, 128, 100)])
def test_decode_views(lens, S, H, size):
    x = _narrow(Absorbed(lens, S, H, size, BF))
    _check4(x, wide=True)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("H", [8, 64, 128])
def test_decode_long(dtype, H):
    _check4(_narrow(Absorbed([9000, 3333], 1, H, 64, dtype)))


@pytest.mark.parametrize("H", [4, 40, 128])
@pytest.mark.parametrize("widen", [False, True])
def test_decode_holes(H, widen):
    x = Absorbed([300, 64, 700], 1, H, 16, BF)
    x.table[0, 3], x.table[0, 7], x.table[1, :] = -1, x.cache.shape[0], -9
    x.table[2, 10:30] = 1 << 30
    x = _narrow(x)
    if widen:
        x.widen()
    o, lse = _check4(x)
    assert (o[1] == 0).all() and torch.isinf(lse[1]).all()


def test_decode_lengths_past_the_table():
    x = _narrow(Absorbed([64, 30], 1, 8, 16, BF))
    o, lse = _run4(x)
    x.lens, x.table = [1 << 30, 30], x.table[:, :4].contiguous()
    o2, _ = _check4(x)
    assert torch.equal(o, o2)
    x.lens = [-5, 30]
    o3, lse3 = _run4(x)
    assert (o3[0] == 0).all() and torch.isinf(lse3[0]).all() and torch.equal(o3[1], o[1])


@pytest.mark.parametrize("kind", ["scale", "infinite", "pe"])
@pytest.mark.parametrize("H,S", [(4, 3), (40, 2), (96, 4)])
@pytest.mark.parametrize("widen", [False, True])
def test_decode_later_draft_tokens_do_not_matter(kind, H, S, widen):
    """A draft token is seen by itself and the tokens after it only, whatever it holds: NaN groups, products past the type's end, NaN in
    the positional part."""
    x = _narrow(Absorbed([130, 64, 33], S, H, 16, HF))
    if widen:
        x.widen()
    o, lse = _run4(x)
    cache = x.bytes.clone()
    for n in range(3):
        row = cache[int(x.table[n, (x.lens[n] - 1) // 16]), (x.lens[n] - 1) % 16]
        if kind == "pe":
            row[272:274] = 255
        else:
            row[256 + 3] = 255 if kind == "scale" else 200
    o2, lse2 = _run4(x, cache=cache)
    for n in range(3):
        a, b = n * S, (n + 1) * S - 1
        assert torch.equal(o[a:b], o2[a:b]) and torch.equal(lse[a:b], lse2[a:b])
        assert torch.isnan(o2[b]).any(dim=-1).all()
    x.cache = Q.values(cache.cpu(), HF)
    _like_the_widened(x, o2, lse2)


@pytest.mark.parametrize("at", [3, 33, 60, 66, 97, 100, 103])
@pytest.mark.parametrize("H,S,prefix", [(4, 1, None), (12, 3, None), (96, 1, None), (12, 1, 75), (96, 2, 75)])
def test_decode_values_past_the_end_of_the_type(at, H, S, prefix):
    """Codes under a scale that takes them past fp16: infinite, as the widened cache has them, in tiles that all rows see and others."""
    x = _narrow(Absorbed([105, 64, 40], S, H, 16, HF, prefix=prefix))
    if prefix is not None and at >= prefix:
        return
    pages = x.prefix_table if prefix is not None else x.table[0]
    row = x.bytes[int(pages[at // 16]), at % 16]
    row[256 + 5] = 142  # 2^15: codes from 4 (2 x 2^15) on are infinite
    x.cache = Q.values(x.bytes.cpu(), HF)
    for _ in range(2):
        o, lse = _run4(x)
        assert not torch.isfinite(o).all()
        _like_the_widened(x, o, lse)
        x.widen()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("lens,S,H,size,prefix", [
    ([1, 33, 64, 100, 7, 250, 18, 90], 1, 12, 16, 2000), ([5, 300], 3, 40, 64, 129), ([1, 1, 1], 1, 128, 100, 31), ([0, 0], 1, 4, 16, 0),
    ([0, 9], 1, 16, 16, 64), ([40, 7], 8, 96, 7, 300)])
def test_decode_prefix(lens, S, H, size, prefix, dtype):
    _check4(_narrow(Absorbed(lens, S, H, size, dtype, prefix=prefix)))


@pytest.mark.parametrize("lens,S,H,size,prefix", [([1, 33, 64, 100], 1, 12, 16, 2000), ([5, 300], 3, 40, 64, 129), ([40, 7], 8, 96, 7, 300)])
def test_decode_prefix_in_wide_tables(lens, S, H, size, prefix):
    _check4(_narrow(Absorbed(lens, S, H, size, BF, prefix=prefix)).widen())


def _tails(x, byte):
    """The cache's rows, the places of pages behind the tokens of a sequence and of the prefix full of a byte."""
    cache = x.bytes.clone()
    ends = [(x.table[n], length) for n, length in enumerate(x.lens)]
    if x.prefix is not None:
        ends.append((x.prefix_table, x.prefix))
    for pages, length in ends:
        if length % x.size:
            cache[int(pages[length // x.size]), length % x.size:] = byte
    return cache


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("lens,S,H,size,prefix", [
    ([1, 33, 64, 100, 7, 250, 18, 90], 1, 12, 16, 2001), ([5, 300, 1031], 3, 40, 64, 129), ([513, 1], 1, 128, 100, None), ([61], 8, 4, 8, None),
    ([40, 7, 500], 8, 96, 7, 300), ([1025], 1, 64, 272, None)])
def test_decode_what_stands_behind_the_tokens(lens, S, H, size, prefix, dtype):
    """Places of a page that hold no token yet: NaN groups, products past the type's end, the largest finite ones.  The same bits."""
    x = _narrow(Absorbed(lens, S, H, size, dtype, prefix=prefix))
    for _ in range(2):
        o, lse = _run4(x, cache=_tails(x, 0))
        for byte in (255, 254, 200, 139, 1):
            o2, lse2 = _run4(x, cache=_tails(x, byte))
            assert torch.equal(o, o2) and torch.equal(lse, lse2), byte
        x.widen()


@pytest.mark.parametrize("n,S,H", [(4127, 1, 12), (4127, 1, 64), (31, 1, 4), (2079, 8, 96)])
def test_decode_time_does_not_follow_what_stands_behind_the_tokens(n, S, H):
    """Recycled pages hold anything.  Best times of calls in a row, a quarter for noise; the last tile has 31 tokens and a place behind
    them, so that a walk through its tokens for what is not finite would be 31 dependent reads."""
    x = _narrow(Absorbed([n], S, H, 64, BF))
    args = [t.to(DEV) for t in (x.ql, x.qp)], x.table.to(DEV), _i32(x.lens)
    caches = [_tails(x, 0), _tails(x, 255)]
    best = [float("inf")] * 2
    for _ in range(12):
        for i, cache in enumerate(caches):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            kda355.latent_decode(*args[0], cache, *args[1:])
            a.record()
            for _ in range(20):
                kda355.latent_decode(*args[0], cache, *args[1:])
            b.record()
            b.synchronize()
            best[i] = min(best[i], a.elapsed_time(b) / 20 * 1e3)
    print(f"[time] {best[0]:.1f} us over zeros, {best[1]:.1f} over NaN groups", flush=True)
    assert best[1] < 1.25 * best[0]


@pytest.mark.parametrize("seed", range(12))
def test_decode_any(seed):
    rng = random.Random(seed)
    H, S = rng.choice([1, 5, 16, 33, 64, 96, 128]), rng.choice([1, 1, 2, 5, 8])
    lens = [rng.choice([0, 1, S, rng.randint(1, 2500)]) for _ in range(rng.choice([1, 3, 20, 66]))]
    x = Absorbed(lens, S, H, rng.choice([1, 3, 16, 64, 272]), rng.choice([BF, HF]), prefix=rng.choice([None, 40, 1111]), seed=seed)
    x = _narrow(x)
    _check4(x.widen() if rng.random() < 0.5 else x)


def test_decode_far_offsets():
    """Pages beyond 2^32 bytes of the cache."""
    pages, size = 90000, 128  # 4.6 GB
    x = _narrow(Absorbed([700, 90], 1, 16, size, BF))
    cache = torch.empty(pages, size, 400, dtype=torch.uint8, device=DEV)
    to = [pages - 1 - 3 * i for i in range(x.bytes.shape[0])]
    cache[to] = x.bytes
    o, lse = _run4(x)
    x.table = torch.where(x.table >= 0, torch.tensor(to)[x.table.clamp(min=0).long()].int(), x.table)
    assert min(to) * size * 400 > 1 << 32
    o2, lse2 = _run4(x, cache=cache)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)
    out = torch.zeros(790, ROW, dtype=BF, device=DEV)
    kda355.latent_gather(cache, x.table.to(DEV), _i32([0, 700, 790]), out)
    rows = torch.cat([R.cache_rows(x.cache, x.table.new_tensor([to.index(int(p)) if int(p) >= 0 else -1 for p in x.table[n]]), k)[0]
                      for n, k in ((0, 700), (1, 90))])
    assert torch.equal(out.cpu().double(), rows)


def test_decode_workspace_and_stream():
    x = _narrow(Absorbed([900, 33, 2000], 1, 12, 64, BF))
    o, lse = _run4(x)
    need = kda355.latent_decode_workspace_bytes(3, 1, 12, 64, x.table.shape[1], num_cus=torch.cuda.get_device_properties(0).multi_processor_count)
    ws = torch.full((need + 512,), 171, dtype=torch.uint8, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o2, lse2 = _run4(x, workspace=ws[:need])
    side.synchronize()
    assert torch.equal(o, o2) and torch.equal(lse, lse2) and (ws[need:] == 171).all()
    with pytest.raises(ValueError):
        _run4(x, workspace=ws[:need - 1])


def test_captured_steps():
    """append, decode, weights and gather in one graph, replayed with other data, lengths and tables."""
    xs = [_narrow(Absorbed(lens, 2, 12, 16, BF, seed=s)) for s, lens in enumerate(([90, 40, 7], [3, 200, 60], [150, 2, 33]))]
    width = max(x.table.shape[1] for x in xs)
    pages = max(x.bytes.shape[0] for x in xs)
    ql, qp = torch.zeros(6, 12, LAT, dtype=BF, device=DEV), torch.zeros(6, 12, PE, dtype=BF, device=DEV)
    cache, table = torch.zeros(pages, 16, 400, dtype=torch.uint8, device=DEV), torch.zeros(3, width, dtype=torch.int32, device=DEV)
    lens, lse = _i32([0, 0, 0]), torch.zeros(6, 12, device=DEV)
    out, weights = torch.zeros(6, 12, LAT, dtype=BF, device=DEV), torch.zeros(3, width * 16, device=DEV)
    latent, pe, slots = torch.zeros(6, LAT, dtype=BF, device=DEV), torch.zeros(6, PE, dtype=BF, device=DEV), torch.zeros(6, dtype=torch.int64, device=DEV)
    cu, rows = _i32([0, 0, 0, 0]), torch.zeros(300, ROW, dtype=BF, device=DEV)

    def step():
        kda355.latent_append(latent, pe, cache, slots)
        kda355.latent_decode(ql, qp, cache, table, lens, out=out, lse=lse)
        kda355.latent_weights(ql, qp, cache, table, lens, lse, weights)
        kda355.latent_gather(cache, table, cu, rows)

    def load(x, seed):
        cache.zero_()
        cache[:x.bytes.shape[0]] = x.bytes
        table.fill_(-1)
        table[:, :x.table.shape[1]] = x.table.to(DEV)
        lens.copy_(_i32(x.lens))
        ql.copy_(x.ql), qp.copy_(x.qp)
        latent.copy_(_randn(6, LAT, dtype=BF, seed=seed)), pe.copy_(_randn(6, PE, dtype=BF, seed=seed + 1))
        t = [(n, x.lens[n] - 2 + s) for n in range(3) for s in range(2)]
        slots.copy_(torch.tensor([int(x.table[n, j // 16]) * 16 + j % 16 for n, j in t]))
        cu.copy_(_i32([0, x.lens[0], x.lens[0] + x.lens[1], sum(x.lens)]))
        weights.fill_(0.5)
        rows.zero_()

    load(xs[0], 0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i, x in enumerate(xs + xs[:2]):
        load(x, 50 + i)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (cache, out, lse, weights, rows)]
        load(x, 50 + i)
        step()
        for a, b in zip(got, (cache, out, lse, weights, rows)):
            assert torch.equal(a, b)
        graph.replay()  # the weights add up
        torch.cuda.synchronize()
        assert torch.allclose(weights, got[3] + (got[3] - 0.5), rtol=1e-5, atol=1e-6)


def test_pages_in_4_bits_forked_freed_and_compacted():
    """The page bookkeeping takes a cache in 4 bits like any pool: a fork reads as its parent, and nothing changes for those that stay."""
    size, H = 16, 10
    x = _narrow(Absorbed([90, 33, 70, 0], 1, H, size, HF))
    used = x.bytes.shape[0]
    pages = used + 9
    cache = torch.zeros(pages, size, 400, dtype=torch.uint8, device=DEV)
    cache[:used] = x.bytes
    need = [-(-n // size) for n in x.lens]
    table = [[int(p) for p in x.table[n][:need[n]]] for n in range(4)]
    held = sorted(p for row in table for p in row)
    left = [p for p in range(pages) if p not in held]
    width = max(need) + 1
    table = _i32([row + [-1] * (width - len(row)) for row in table])
    lens, num = _i32(x.lens), _i32([len(left)])
    refs, free = _i32([int(p in held) for p in range(pages)]), _i32(left + [-1] * (pages - len(left)))
    ql, qp = x.ql.to(DEV), x.qp.to(DEV)

    def step(what):
        """The rows of every sequence; the step over them within the tolerances.  (How a sequence is cut depends on those beside it.)"""
        n = lens.tolist()
        cu = [sum(n[:i]) for i in range(5)]
        rows = torch.zeros(cu[4], ROW, dtype=HF, device=DEV)
        kda355.latent_gather(cache, table, _i32(cu), rows)
        out = kda355.latent_decode(ql, qp, cache, table, lens).cpu()
        rows = [rows[cu[i]:cu[i + 1]].cpu() for i in range(4)]
        for i in range(4):
            q, k = torch.cat([ql[i], qp[i]], dim=-1).cpu().double(), rows[i].double()
            R.check(out[i], None, R.attend(q, k, k[:, :LAT], torch.ones(H, n[i], dtype=torch.bool), R.SCALE), HF, ROW, f"{what} seq {i}")
        return rows

    before = step("before")
    kda355.fork_pages([cache], table, lens, refs, free, num, _i32([0]), _i32([3]), size)
    assert lens.tolist() == [90, 33, 70, 90]
    after = step("forked")
    assert all(torch.equal(a, b) for a, b in zip(after, before[:3] + before[:1]))
    kda355.free_pages(table, lens, refs, free, num, _i32([0, 1]), size)
    kda355.compact_pages([cache], table, refs, free, num)
    assert lens.tolist() == [0, 0, 70, 90] and int(table.max()) == need[0] + need[2] - 1
    last = step("compacted")
    assert torch.equal(last[2], before[2]) and torch.equal(last[3], before[0])


def test_refusals():
    x = _narrow(Absorbed([20, 5], 1, 4, 16, BF))
    ql, qp, table, lens = x.ql.to(DEV), x.qp.to(DEV), x.table.to(DEV), _i32(x.lens)
    for bad in (x.bytes[..., :399], x.bytes[..., ::2], x.bytes.view(-1, 400), x.bytes[:0], x.bytes[:, :0],
                x.bytes.repeat(1, 2, 1)[:, ::2], torch.zeros(3, 16, ROW, dtype=torch.uint8, device=DEV)):
        with pytest.raises(ValueError):
            kda355.latent_decode(ql, qp, bad, table, lens)
        with pytest.raises(ValueError):
            kda355.latent_append(ql[:, 0], qp[:, 0], bad, torch.zeros(2, dtype=torch.int64, device=DEV))
        with pytest.raises(ValueError):
            kda355.latent_gather(bad, table, _i32([0, 20, 25]), torch.empty(25, ROW, dtype=BF, device=DEV))
    for bad in (x.bytes.view(torch.int8), x.bytes.cpu(), x.bytes.float(), None):
        with pytest.raises(TypeError):
            kda355.latent_decode(ql, qp, bad, table, lens)
        with pytest.raises(TypeError):
            kda355.latent_append(ql[:, 0], qp[:, 0], bad, torch.zeros(2, dtype=torch.int64, device=DEV))
    with pytest.raises(TypeError):
        kda355.latent_gather(x.bytes, table, _i32([0, 20, 25]), torch.empty(25, ROW, device=DEV))
    with pytest.raises(TypeError):
        kda355.latent_gather(x.bytes, table, _i32([0, 20, 25]), None)
    odd = torch.zeros(x.bytes.numel() + 16, dtype=torch.uint8, device=DEV)[8:8 + x.bytes.numel()].view_as(x.bytes)
    with pytest.raises(ValueError):  # not aligned
        kda355.latent_decode(ql, qp, odd, table, lens)
    apart = torch.zeros(x.bytes.shape[0], 16 * 400 + 8, dtype=torch.uint8, device=DEV)
    with pytest.raises(ValueError):  # pages not aligned
        kda355.latent_decode(ql, qp, apart.as_strided(x.bytes.shape, (apart.shape[1], 400, 1)), table, lens)
