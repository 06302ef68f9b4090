"""Latent attention on the GPU against the float64 forms of latent_ref.py (tolerances derived there)."""
import pytest
import torch

import kda355
import latent_ref as R
from latent_ref import HEAD, LAT, PE, ROW, SCALE

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _offsets(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


def _randn(*shape, dtype, seed, std=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


# ================================================================================================ expanded form
class Expanded:
    """Inputs on the CPU, and on the GPU in the layout named: "dense", "joint" (k | v of a head side by side, k_pe the tail
    of 576-wide rows, as projections leave them) or "wide" (every tensor a view with padding, heads outermost for q)."""

    def __init__(self, lq, lk, H, dtype, layout="joint", seed=0, std=1.5):
        self.H, self.dtype = H, dtype
        self.cu_q, self.cu_k = _offsets(lq), _offsets(lk)
        Tq, Tk = self.cu_q[-1], self.cu_k[-1]
        self.q = _randn(Tq, H, HEAD + PE, dtype=dtype, seed=seed, std=std)
        self.k, self.v = _randn(Tk, H, HEAD, dtype=dtype, seed=seed + 1), _randn(Tk, H, HEAD, dtype=dtype, seed=seed + 2)
        self.pe = _randn(Tk, PE, dtype=dtype, seed=seed + 3)
        self.layout = layout

    def run(self, causal=True, scale=SCALE, out=None, stream=None):
        H, dt = self.H, self.dtype
        q, k, v, pe = (t.to(DEV) for t in (self.q, self.k, self.v, self.pe))
        if self.layout == "joint":
            kv = torch.cat([k, v], dim=-1)
            k, v = kv[..., :HEAD], kv[..., HEAD:]
            pe = torch.cat([torch.full((pe.shape[0], LAT), float("nan"), device=DEV, dtype=dt), pe], dim=-1)[:, LAT:]
        elif self.layout == "wide":
            q = q.transpose(0, 1).contiguous().transpose(0, 1)
            k = torch.cat([k, torch.full_like(k[..., :8], float("nan"))], dim=-1)[..., :HEAD]
            v = v.transpose(0, 1).contiguous().transpose(0, 1)
        lse = torch.full((q.shape[0], H), 7.0, device=DEV)
        o = kda355.latent_prefill(q, k, v, pe, _i32(self.cu_q), _i32(self.cu_k), scale, causal, out=out, lse=lse)
        return o, lse

    def check(self, causal=True, scale=SCALE, what=""):
        o, lse = self.run(causal, scale)
        o, lse = o.cpu(), lse.cpu()
        parts = R.prefill(self.q, self.k, self.v, self.pe, self.cu_q, self.cu_k, causal, scale)
        for n, h, ref in parts:
            a, b = self.cu_q[n], self.cu_q[n + 1]
            R.check(o[a:b, h], lse[a:b, h], ref, self.dtype, HEAD + PE, f"{what} seq {n} head {h}")
        return o, lse


LENS = [
    ([1], [1]), ([1], [2]), ([2], [1]), ([5], [5]), ([31, 32, 33], [31, 32, 33]), ([63, 64, 65], [63, 64, 65]),
    ([127, 128, 129], [127, 130, 300]), ([1, 0, 40, 7, 0], [70, 3, 40, 0, 0]), ([0], [5]), ([257], [513]),
    ([70, 3], [20, 2]),  # fewer keys than queries: the first queries see nothing
    ([1, 1, 1, 1], [1000, 64, 65, 1]),
]


@pytest.mark.parametrize("lq,lk", LENS, ids=[f"{a}-{b}".replace(" ", "") for a, b in LENS])
@pytest.mark.parametrize("causal", [True, False])
def test_prefill_lengths(lq, lk, causal):
    Expanded(lq, lk, 2, BF).check(causal)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("layout", ["dense", "joint", "wide"])
@pytest.mark.parametrize("H", [1, 3, 8])
def test_prefill_layouts(dtype, layout, H):
    Expanded([100, 37], [164, 37], H, dtype, layout).check()


@pytest.mark.parametrize("dtype", [BF, HF])
def test_prefill_long(dtype):
    Expanded([200, 1], [2000, 5001], 1, dtype).check()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("kind", ["rising", "spike_first", "spike_last", "huge", "zero"])
def test_prefill_score_ranges(dtype, kind):
    """Running maxima that rise key by key, one key above all others at either end, scores in the thousands, all equal."""
    x = Expanded([96], [700], 1, dtype, std=0.0 if kind == "zero" else 1.0)
    j = torch.arange(700)[:, None, None].float()
    if kind == "rising":
        x.q[..., 0] = 8.0
        x.k[..., :1] = (j / 8).to(dtype)
    elif kind.startswith("spike"):
        x.q[..., 0] = 16.0
        x.k[..., 0] = 0.0
        x.k[0 if kind == "spike_first" else 600, :, 0] = 24.0
    elif kind == "huge":
        x.q *= 64.0
        x.k *= 16.0
    x.check()


def test_prefill_fp16_many_small_weights():
    """One key at weight 1 and thousands at 2^-13 to 2^-17 each, whose sum matters."""
    x = Expanded([3], [6000], 1, HF, std=0.0)
    x.q[..., 0] = 4.0
    x.k[..., 0] = -_randn(6000, 1, dtype=HF, seed=9).abs() * 3 - 24.0
    x.k[10, :, 0] = 9.0
    x.v.abs_()
    x.check()


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("lq,lk", [(130, 130), (64, 200), (9, 40)])
def test_prefill_unseen_keys_do_not_matter(value, lq, lk):
    """Keys and values that a query does not see, NaN and infinite among them, leave its output bit for bit as it is; a
    neighbouring sequence's do too."""
    x = Expanded([lq, 5, lq], [lk, 5, lk], 2, BF)
    o, lse = x.run()
    for j in (lk - 1, lk - 2, lk - lq // 2):  # seen by the later queries only
        y = Expanded([lq, 5, lq], [lk, 5, lk], 2, BF)
        y.v[j, 0, 3] = value
        y.k[j, 1, 5] = value
        y.v[x.cu_k[1]:x.cu_k[2]] = value
        y.k[x.cu_k[1]:x.cu_k[2]] = value
        y.pe[x.cu_k[1]:x.cu_k[2]] = value
        o2, lse2 = y.run()
        last = j - (lk - lq)  # queries before this one do not see key j
        for a, b in ((0, last), (x.cu_q[2], x.cu_q[3])):
            assert torch.equal(o2[a:b], o[a:b]) and torch.equal(lse2[a:b], lse[a:b])
        # the ones that do: the value itself in that output channel, the rest of head 0 as before
        got = o2[last:lq, 0].float().cpu()
        if value != value:
            assert torch.isnan(got[:, 3]).all()
        else:
            assert (got[:, 3] == value).all()
        keep = [c for c in range(HEAD) if c != 3]
        assert torch.equal(got[:, keep], o[last:lq, 0].float().cpu()[:, keep])


def test_prefill_far_offsets():
    """Rows further apart than 32 bits can address, in elements and in bytes."""
    x = Expanded([40], [300], 1, BF)
    wide = torch.empty(300, 1 << 23, dtype=BF, device=DEV)  # 5 GB
    rows = wide[:, :HEAD * 2 + PE]
    rows.copy_(torch.cat([x.k[:, 0], x.v[:, 0], x.pe], dim=-1))
    out = torch.empty(40, 1, HEAD, dtype=BF, device=DEV)
    lse = torch.empty(40, 1, device=DEV)
    kda355.latent_prefill(x.q.to(DEV), rows[:, None, :HEAD], rows[:, None, HEAD:2 * HEAD], rows[:, 2 * HEAD:], _i32([0, 40]),
                          _i32([0, 300]), out=out, lse=lse)
    o, l = x.run()
    assert torch.equal(o, out) and torch.equal(l, lse)


def test_prefill_out_slice_and_repeat():
    """`out` as a view: nothing beside it changes; the same call twice gives the same bits."""
    x = Expanded([150, 3], [150, 90], 3, BF)
    wide = torch.full((153, 5, HEAD + 16), 3.0, dtype=BF, device=DEV)
    o1, l1 = x.run(out=wide[:, 1:4, 8:8 + HEAD])
    o2, l2 = x.run()
    assert torch.equal(o1, o2) and torch.equal(l1, l2)
    wide[:, 1:4, 8:8 + HEAD] = 3.0
    assert (wide == 3.0).all()


def test_prefill_bad_offsets_stay_inside():
    """cu_seqlens past the tensors are clamped to them: nothing outside is read or written."""
    x = Expanded([20], [50], 2, BF)
    o, _ = x.run()
    q, k, v, pe = (t.to(DEV) for t in (x.q, x.k, x.v, x.pe))
    out = torch.zeros_like(o)
    kda355.latent_prefill(q, k, v, pe, _i32([0, 20]), _i32([0, 1 << 30]), out=out)
    assert torch.equal(out, o)
    kda355.latent_prefill(q, k, v, pe, _i32([-5, 1 << 30]), _i32([50, 0]), out=out)  # no keys left
    assert (out == 0).all() or torch.equal(out, o)


def test_prefill_cut_along_the_keys():
    """Few queries over many keys: pieces of a sequence that come together again, empty ones and rows that see nothing among
    them; a workspace full of NaN leaves no trace, on another stream too."""
    x = Expanded([40, 3, 0, 300, 9], [20, 6000, 100, 900, 0], 3, BF)
    o, lse = x.check()
    assert (o[:20] == 0).all() and torch.isinf(lse[:20]).all() and (o[343:] == 0).all()
    need = kda355.latent_prefill_workspace_bytes(5, 3, 352, 7020, num_cus=torch.cuda.get_device_properties(0).multi_processor_count)
    ws = torch.full((need,), 255, dtype=torch.uint8, device=DEV)
    q, k, v, pe = (t.to(DEV) for t in (x.q, x.k, x.v, x.pe))
    cu_q, cu_k = _i32(x.cu_q), _i32(x.cu_k)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        l2 = torch.empty_like(lse, device=DEV)
        o2 = kda355.latent_prefill(q, k, v, pe, cu_q, cu_k, lse=l2, workspace=ws)
    side.synchronize()
    assert torch.equal(o2.cpu(), o) and torch.equal(l2.cpu(), lse)


@pytest.mark.parametrize("seed", range(6))
def test_prefill_any(seed):
    g = torch.Generator().manual_seed(100 + seed)
    pick = lambda top, n: torch.randint(0, top, (n,), generator=g).tolist()  # noqa: E731
    n = 1 + pick(6, 1)[0]
    lq = pick(200, n)
    lk = [a + b if c else b for a, b, c in zip(lq, pick(700, n), pick(4, n))]
    Expanded(lq, lk, 1 + pick(5, 1)[0], (BF, HF)[seed % 2], ("dense", "joint", "wide")[seed % 3], seed=seed).check(seed != 4)


@pytest.mark.parametrize("N", [64, 65, 150])
def test_prefill_many_sequences(N):
    """More sequences than a wave has lanes, empty ones and one that is cut among them."""
    g = torch.Generator().manual_seed(N)
    lq = torch.randint(0, 30, (N,), generator=g).tolist()
    lk = [a + b for a, b in zip(lq, torch.randint(0, 60, (N,), generator=g).tolist())]
    lq[N - 1], lk[N - 1], lq[3], lk[3] = 5, 6000, 200, 3
    lk[N // 2] = 0
    Expanded(lq, lk, 2, BF).check()


def test_prefill_captured_with_other_lengths():
    """One graph replayed with other boundaries, every replay against the eager result and the plain form."""
    xs = [Expanded(lq, lk, 2, BF, "dense", seed=i) for i, (lq, lk) in enumerate(
        [([100, 7, 43], [300, 50, 150]), ([1, 148, 1], [400, 90, 10]), ([0, 150, 0], [0, 200, 300]), ([5, 5, 140], [1, 498, 1])])]
    q, k, v, pe = (torch.empty_like(t, device=DEV) for t in (xs[0].q, xs[0].k, xs[0].v, xs[0].pe))
    cu_q, cu_k = _i32([0] * 4), _i32([0] * 4)
    out, lse = torch.empty(150, 2, HEAD, dtype=BF, device=DEV), torch.empty(150, 2, device=DEV)

    def step():
        kda355.latent_prefill(q, k, v, pe, cu_q, cu_k, out=out, lse=lse)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for x in xs + xs[:1]:
        for t, y in ((q, x.q), (k, x.k), (v, x.v), (pe, x.pe)):
            t.copy_(y)
        cu_q.copy_(_i32(x.cu_q))
        cu_k.copy_(_i32(x.cu_k))
        graph.replay()
        torch.cuda.synchronize()
        got, got_lse = out.clone(), lse.clone()
        step()
        assert torch.equal(got, out) and torch.equal(got_lse, lse)
        for n, h, ref in R.prefill(x.q, x.k, x.v, x.pe, x.cu_q, x.cu_k, True, SCALE):
            a, b = x.cu_q[n], x.cu_q[n + 1]
            R.check(got[a:b, h].cpu(), got_lse[a:b, h].cpu(), ref, BF, HEAD + PE, f"replay seq {n} head {h}")


# ================================================================================================ absorbed form
class Absorbed:
    def __init__(self, lens, S, H, size, dtype, prefix=None, seed=0, std=1.0, spare=2):
        self.S, self.H, self.size, self.dtype = S, H, size, dtype
        self.lens, self.prefix = list(lens), prefix
        B = len(lens)
        need = [-(-n // size) for n in lens]
        width = max([1] + need) + 1
        extra = -(-prefix // size) if prefix is not None else 0
        pages = sum(need) + extra + spare
        g = torch.Generator().manual_seed(seed)
        perm = torch.randperm(pages, generator=g).int()
        self.table = torch.full((B, width), -1, dtype=torch.int32)
        at = 0
        for n, k in enumerate(need):
            self.table[n, :k] = perm[at:at + k]
            at += k
        self.prefix_table = None
        if prefix is not None:
            self.prefix_table = torch.full((extra + 1,), -1, dtype=torch.int32)
            self.prefix_table[:extra] = perm[at:at + extra]
            at += extra
        self.cache = _randn(pages, size, ROW, dtype=dtype, seed=seed + 1)
        # what no sequence holds is never seen: pages of nobody and the ends of last pages are NaN
        self.cache[perm[at:].long()] = float("nan")
        for n in range(B):
            if lens[n] % size:
                self.cache[int(self.table[n, lens[n] // size]), lens[n] % size:] = float("nan")
        if prefix is not None and prefix % size:
            self.cache[int(self.prefix_table[prefix // size]), prefix % size:] = float("nan")
        self.ql = _randn(B * S, H, LAT, dtype=dtype, seed=seed + 2, std=std)
        self.qp = _randn(B * S, H, PE, dtype=dtype, seed=seed + 3, std=std)

    def run(self, wide=False, workspace=None, scale=SCALE):
        ql, qp, cache, table = (t.to(DEV) for t in (self.ql, self.qp, self.cache, self.table))
        out = None
        if wide:  # queries as one 576-wide tensor, pages and table rows apart, an output between other values
            both = torch.cat([ql, qp], dim=-1)
            ql, qp = both[..., :LAT], both[..., LAT:]
            page = torch.full((cache.shape[0], self.size * ROW + 40), float("nan"), dtype=self.dtype, device=DEV)
            view = page.as_strided(cache.shape, (page.shape[1], ROW, 1))
            view.copy_(cache)
            cache = view
            table = torch.cat([table, torch.full_like(table, 1 << 20)], dim=1)[:, :table.shape[1]]
            out = torch.full((ql.shape[0], self.H + 1, LAT + 8), 3.0, dtype=self.dtype, device=DEV)[:, 1:, :LAT]
        lse = torch.full((ql.shape[0], self.H), 7.0, device=DEV)
        kw = {}
        if self.prefix is not None:
            kw = dict(prefix_table=self.prefix_table.to(DEV), prefix_len=_i32([self.prefix]))
        o = kda355.latent_decode(ql, qp, cache, table, _i32(self.lens), scale, out=out, lse=lse, workspace=workspace, **kw)
        return o, lse

    def check(self, what="", **kw):
        o, lse = self.run(**kw)
        o, lse = o.cpu(), lse.cpu()
        refs = R.decode(self.ql, self.qp, self.cache, self.table, self.lens, self.S, prefix_table=self.prefix_table,
                        prefix_len=self.prefix or 0)
        S, H = self.S, self.H
        for n, ref in enumerate(refs):
            R.check(o[n * S:(n + 1) * S].reshape(S * H, LAT), lse[n * S:(n + 1) * S].reshape(S * H), ref, self.dtype, ROW,
                    f"{what} seq {n}")
        return o, lse


    def widen(self, entries=1 << 20):
        """Tables with room for many more tokens: the work is grouped for long lists of pages."""
        pad = torch.full((len(self.lens), entries // self.size // len(self.lens)), -1, dtype=torch.int32)
        self.table = torch.cat([self.table, pad], dim=1)
        if self.prefix_table is not None:
            self.prefix_table = torch.cat([self.prefix_table, torch.full((entries // self.size,), -1, dtype=torch.int32)])
        return self


DECODE = [
    ([1], 1, 1, 1), ([1], 1, 12, 16), ([2, 31, 32, 33], 1, 4, 16), ([63, 64, 65, 127, 128, 129], 1, 16, 64),
    ([0, 5, 0, 300], 1, 12, 64), ([1000], 1, 32, 272), ([500, 3], 1, 33, 100), ([700, 40], 1, 64, 64), ([290], 1, 96, 16),
    ([300, 5], 1, 128, 64), ([300, 5], 1, 130, 64), ([40, 7, 8, 300], 8, 4, 16), ([9, 130], 3, 12, 7),
    ([200, 64], 8, 40, 64), ([3, 1, 0, 600], 4, 8, 16),  # fewer tokens than S: the first rows see nothing
    ([37] * 70, 1, 2, 16), ([5] * 300 + [900], 1, 1, 16),
]


@pytest.mark.parametrize("lens,S,H,size", DECODE, ids=[f"{len(c[0])}seq-{max(c[0])}-S{c[1]}-H{c[2]}-p{c[3]}" for c in DECODE])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_decode_lengths(lens, S, H, size, dtype):
    Absorbed(lens, S, H, size, dtype).check()


@pytest.mark.parametrize("lens,S,H,size", DECODE, ids=[f"{len(c[0])}seq-{max(c[0])}-S{c[1]}-H{c[2]}-p{c[3]}" for c in DECODE])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_decode_lengths_in_wide_tables(lens, S, H, size, dtype):
    Absorbed(lens, S, H, size, dtype).widen().check()


@pytest.mark.parametrize("lens,S,H,size", [([400, 90], 1, 12, 64), ([130, 77, 1], 4, 16, 16), ([513], 1, 128, 100)])
def test_decode_views(lens, S, H, size):
    x = Absorbed(lens, S, H, size, BF)
    o, lse = x.check(wide=True)
    o2, lse2 = x.run()
    assert torch.equal(o, o2.cpu()) and torch.equal(lse, lse2.cpu())


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("H", [8, 64, 128])
def test_decode_long(dtype, H):
    Absorbed([6000, 20], 1, H, 64, dtype).check()


@pytest.mark.parametrize("kind", ["rising", "spike_first", "spike_last", "huge", "zero"])
@pytest.mark.parametrize("H,dtype", [(2, BF), (40, BF), (100, HF)])
def test_decode_score_ranges(kind, H, dtype):
    x = Absorbed([1500], 1, H, 64, dtype, std=0.0 if kind == "zero" else 1.0)
    rows = x.table[0, :24].long()
    flat = x.cache[rows].reshape(-1, ROW)
    if kind == "rising":
        x.qp[..., 0] = 8.0
        flat[:, LAT] = (torch.arange(24 * 64) / 16).to(dtype)
    elif kind.startswith("spike"):
        x.qp[..., 0] = 16.0
        flat[:, LAT] = 0.0
        flat[0 if kind == "spike_first" else 1400, LAT] = 24.0
    elif kind == "huge":
        x.ql *= 30.0
    flat[1500:] = float("nan")
    x.cache[rows] = flat.view(24, 64, ROW)
    x.check()


@pytest.mark.parametrize("kind", ["rising", "spike_first", "spike_last"])
@pytest.mark.parametrize("H,dtype", [(2, BF), (40, HF), (100, BF)])
def test_decode_score_ranges_in_wide_tables(kind, H, dtype):
    x = Absorbed([1500], 1, H, 64, dtype)
    rows = x.table[0, :24].long()
    flat = x.cache[rows].reshape(-1, ROW)
    x.qp[..., 0] = 8.0 if kind == "rising" else 16.0
    flat[:, LAT] = (torch.arange(24 * 64) / 16).to(dtype) if kind == "rising" else 0.0
    if kind != "rising":
        flat[0 if kind == "spike_first" else 1400, LAT] = 24.0
    flat[1500:] = float("nan")
    x.cache[rows] = flat.view(24, 64, ROW)
    x.widen().check()


def test_decode_fp16_many_small_weights():
    x = Absorbed([6000], 1, 4, 64, HF, std=0.0)
    x.qp[..., 0] = 4.0
    rows = x.table[0, :94].long()
    flat = x.cache[rows].reshape(-1, ROW)
    flat[:, LAT] = -_randn(94 * 64, dtype=HF, seed=9).abs() * 3 - 24.0
    flat[10, LAT] = 9.0
    flat[:, :LAT] = flat[:, :LAT].abs()
    x.cache[rows] = flat.view(94, 64, ROW)
    x.check()


@pytest.mark.parametrize("H", [4, 40, 128])
def test_decode_holes(H):
    """Page numbers outside the cache: their tokens take no part; a sequence of holes alone gives zeros and -inf."""
    x = Absorbed([300, 64, 700], 1, H, 16, BF)
    x.table[0, 3] = -1
    x.table[0, 7] = x.cache.shape[0]
    x.table[1, :] = -9
    x.table[2, 10:30] = 1 << 30
    o, lse = x.check()
    assert (o[1] == 0).all() and torch.isinf(lse[1]).all()


def test_decode_lengths_past_the_table():
    x = Absorbed([64, 30], 1, 8, 16, BF)
    o, lse = x.run()
    x.lens = [1 << 30, 30]
    x.table = x.table[:, :4].contiguous()
    x.check()
    o2, _ = x.run()
    assert torch.equal(o, o2)
    x.lens = [-5, 30]
    o3, lse3 = x.run()
    assert (o3[0] == 0).all() and torch.isinf(lse3[0]).all() and torch.equal(o3[1], o[1])


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("H,S", [(4, 3), (40, 2), (96, 4)])
def test_decode_later_draft_tokens_do_not_matter(value, H, S):
    """A draft token is seen by itself and the tokens after it only, whatever it holds."""
    x = Absorbed([130, 64, 33], S, H, 16, BF)
    o, lse = x.run()
    for n in range(3):
        j = x.lens[n] - 1
        x.cache[int(x.table[n, j // 16]), j % 16, 7] = value
    o2, lse2 = x.run()
    for n in range(3):
        a, b = n * S, (n + 1) * S - 1
        assert torch.equal(o[a:b], o2[a:b]) and torch.equal(lse[a:b], lse2[a:b])


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("H,S", [(4, 3), (40, 2), (96, 4)])
def test_decode_later_draft_tokens_do_not_matter_in_wide_tables(value, H, S):
    x = Absorbed([130, 64, 33], S, H, 16, BF).widen()
    o, lse = x.check()
    for n in range(3):
        j = x.lens[n] - 1
        x.cache[int(x.table[n, j // 16]), j % 16, 7] = value
    o2, lse2 = x.run()
    for n in range(3):
        a, b = n * S, (n + 1) * S - 1
        assert torch.equal(o[a:b], o2[a:b].cpu()) and torch.equal(lse[a:b], lse2[a:b].cpu())


@pytest.mark.parametrize("lens,S,H,size,prefix", [
    ([1, 33, 64], 1, 12, 16, 100), ([5, 0, 300], 1, 12, 64, 1000), ([40, 7], 2, 96, 64, 129), ([10, 20, 30], 1, 128, 272, 500),
    ([12] * 40, 1, 4, 16, 257), ([50, 60], 1, 8, 16, 0), ([0, 2], 3, 8, 16, 0)])
def test_decode_prefix_in_wide_tables(lens, S, H, size, prefix):
    Absorbed(lens, S, H, size, BF, prefix=prefix).widen().check()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("lens,S,H,size,prefix", [
    ([1], 1, 1, 16, 1), ([1, 33, 64], 1, 12, 16, 100), ([5, 0, 300], 1, 12, 64, 1000), ([5, 9], 4, 16, 16, 33),
    ([40, 7], 2, 96, 64, 129), ([10, 20, 30], 1, 128, 272, 500), ([12] * 40, 1, 4, 16, 257), ([50, 60], 1, 8, 16, 0),
    ([0, 0], 1, 8, 16, 70), ([0, 2], 3, 8, 16, 0)])
def test_decode_prefix(lens, S, H, size, prefix, dtype):
    Absorbed(lens, S, H, size, dtype, prefix=prefix).check()


@pytest.mark.parametrize("B,S,H", [(64, 1, 3), (65, 2, 16), (150, 1, 40)])
def test_decode_many_sequences_behind_a_prefix(B, S, H):
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, 90, (B,), generator=g).tolist()
    lens[B - 1] = 1500
    Absorbed(lens, S, H, 16, BF, prefix=333).check()


def test_decode_prefix_long():
    Absorbed([700, 3], 1, 40, 64, BF, prefix=5000).check()


def test_decode_prefix_equals_copies():
    """The shared prefix gives what every sequence holding its own copy of it gives, within both calls' tolerances."""
    x = Absorbed([33, 90, 7], 2, 16, 16, BF, prefix=160)
    o, lse = x.check()
    y = Absorbed([193, 250, 167], 2, 16, 16, BF)
    y.ql, y.qp = x.ql, x.qp
    for n in range(3):
        rows = torch.cat([R.cache_rows(x.cache, x.prefix_table, 160)[0], R.cache_rows(x.cache, x.table[n], x.lens[n])[0]])
        for j in range(len(rows)):
            y.cache[int(y.table[n, j // 16]), j % 16] = rows[j].to(BF)
    o2, lse2 = y.check()
    assert (lse - lse2).abs().max() < 1e-4


@pytest.mark.parametrize("seed", range(10))
def test_decode_any(seed):
    g = torch.Generator().manual_seed(200 + seed)
    pick = lambda top, n: torch.randint(0, top, (n,), generator=g).tolist()  # noqa: E731
    B, S, H = 1 + pick(9, 1)[0], 1 + pick(8, 1)[0], 1 + pick(130, 1)[0]
    top = (40, 600, 2500)[seed % 3]
    Absorbed(pick(top, B), S, H, 1 + pick(150, 1)[0], (BF, HF)[seed % 2], prefix=pick(900, 1)[0] if seed % 4 == 1 else None,
             seed=seed).check()


def test_decode_far_offsets():
    """Pages further apart than 32 bits can address."""
    x = Absorbed([900], 1, 12, 64, BF)
    o, lse = x.run()
    wide = torch.empty(x.cache.shape[0], 1 << 28, dtype=BF, device=DEV)  # 9 GB
    view = wide.as_strided(x.cache.shape, (wide.stride(0), ROW, 1))
    view.copy_(x.cache)
    l2 = torch.empty_like(lse)
    o2 = kda355.latent_decode(x.ql.to(DEV), x.qp.to(DEV), view, x.table.to(DEV), _i32(x.lens), lse=l2)
    assert torch.equal(o, o2) and torch.equal(lse, l2)


@pytest.mark.parametrize("prefix", [None, 200])
def test_decode_captured_with_other_lengths(prefix):
    """One graph replayed with other lengths, tables, queries and prefix lengths, every replay against the eager result."""
    xs = [Absorbed(lens, 2, 12, 16, BF, prefix=prefix, seed=i, spare=40) for i, lens in
          enumerate([[50, 7, 90], [2, 300, 64], [128, 0, 1], [301, 290, 33]])]
    width = max(x.table.shape[1] for x in xs)
    pages = max(x.cache.shape[0] for x in xs)
    cache = torch.zeros(pages, 16, ROW, dtype=BF, device=DEV)
    table = torch.full((3, width), -1, dtype=torch.int32, device=DEV)
    ql, qp, lens = xs[0].ql.to(DEV), xs[0].qp.to(DEV), _i32(xs[0].lens)
    ptab = torch.full((14,), -1, dtype=torch.int32, device=DEV) if prefix else None
    plen = _i32([0]) if prefix else None
    out, lse = torch.empty_like(ql), torch.empty(6, 12, device=DEV)

    def step():
        kda355.latent_decode(ql, qp, cache, table, lens, out=out, lse=lse, prefix_table=ptab, prefix_len=plen)

    def fill(x):
        cache[:x.cache.shape[0]] = x.cache.to(DEV)
        table.fill_(-1)
        table[:, :x.table.shape[1]] = x.table.to(DEV)
        ql.copy_(x.ql)
        qp.copy_(x.qp)
        lens.copy_(_i32(x.lens))
        if prefix:
            ptab.fill_(-1)
            ptab[:x.prefix_table.numel()] = x.prefix_table.to(DEV)
            plen.fill_(x.prefix)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for x in xs + xs[:1]:
        fill(x)
        graph.replay()
        torch.cuda.synchronize()
        got, got_lse = out.clone(), lse.clone()
        step()
        assert torch.equal(got, out) and torch.equal(got_lse, lse)
        refs = R.decode(x.ql, x.qp, x.cache, x.table, x.lens, 2, prefix_table=x.prefix_table, prefix_len=x.prefix or 0)
        for n, ref in enumerate(refs):
            R.check(got[2 * n:2 * n + 2].reshape(24, LAT), got_lse[2 * n:2 * n + 2].reshape(24), ref, BF, ROW, f"replay seq {n}")


def test_side_stream_and_workspace():
    """Calls on another stream than the default one; a workspace of the caller's, full of NaN, leaves no trace."""
    x = Absorbed([700, 64, 9], 1, 40, 16, BF, prefix=90)
    o, lse = x.run()
    need = kda355.latent_decode_workspace_bytes(3, 1, 40, 16, x.table.shape[1], x.prefix_table.numel(),
                                                num_cus=torch.cuda.get_device_properties(0).multi_processor_count)
    ws = torch.full((need + 4,), 255, dtype=torch.uint8, device=DEV)[:need]
    y = Expanded([100], [300], 2, BF)
    o3, _ = y.run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        o2, lse2 = x.run(workspace=ws)
        o4, _ = y.run()
    side.synchronize()
    assert torch.equal(o, o2) and torch.equal(lse, lse2) and torch.equal(o3, o4)


# ================================================================================================ refusals
def test_refusals():
    x = Expanded([8], [8], 2, BF, "dense")
    q, k, v, pe = (t.to(DEV) for t in (x.q, x.k, x.v, x.pe))
    cu = _i32([0, 8])
    call = kda355.latent_prefill
    for bad in (dict(q=q[..., :128]), dict(k=k[:7]), dict(v=v[:, :1]), dict(k_pe=pe[:, :32]), dict(cu_seqlens_k=_i32([0, 4, 8])),
                dict(out=torch.empty(8, 2, 64, device=DEV, dtype=BF)), dict(lse=torch.empty(8, 3, device=DEV)),
                dict(q=q.transpose(1, 2).contiguous().transpose(1, 2)), dict(cu_seqlens_q=_i32([]))):
        with pytest.raises(ValueError):
            call(**{**dict(q=q, k=k, v=v, k_pe=pe, cu_seqlens_q=cu, cu_seqlens_k=cu), **bad})
    for bad in (dict(q=q.float()), dict(k=k.half()), dict(k_pe=x.pe), dict(cu_seqlens_q=cu.long()),
                dict(lse=torch.empty(8, 2, device=DEV, dtype=BF)), dict(v=None), dict(cu_seqlens_k=[0, 8])):
        with pytest.raises(TypeError):
            call(**{**dict(q=q, k=k, v=v, k_pe=pe, cu_seqlens_q=cu, cu_seqlens_k=cu), **bad})
    with pytest.raises(ValueError):  # a token stride that is no multiple of 8 elements
        call(torch.empty(8, 2 * 192 + 4, device=DEV, dtype=BF).as_strided((8, 2, 192), (388, 192, 1)), k, v, pe, cu, cu)
    a = Absorbed([20, 5], 1, 4, 16, BF)
    ql, qp, cache, table = (t.to(DEV) for t in (a.ql, a.qp, a.cache, a.table))
    args = dict(q_latent=ql, q_pe=qp, cache=cache, block_table=table, seq_lens=_i32([20, 5]))
    call = kda355.latent_decode
    for bad in (dict(q_latent=ql[:, :, :256]), dict(q_pe=qp[:1]), dict(cache=cache[:, :, :512]), dict(block_table=table[0]),
                dict(seq_lens=_i32([1])), dict(prefix_table=_i32([0])), dict(prefix_len=_i32([0])),
                dict(prefix_table=_i32([0]), prefix_len=_i32([0, 1])), dict(out=torch.empty(2, 4, 511, device=DEV, dtype=BF)),
                dict(prefix_table=_i32([]), prefix_len=_i32([0])), dict(cache=cache.transpose(1, 2).contiguous().transpose(1, 2))):
        with pytest.raises(ValueError):
            call(**{**args, **bad})
    with pytest.raises(ValueError):
        call(**{**args, "q_latent": ql[:1], "q_pe": qp[:1]})
    for bad in (dict(q_pe=qp.half()), dict(cache=cache.float()), dict(block_table=table.long()), dict(seq_lens=a.lens),
                dict(workspace=torch.empty(1 << 20, device=DEV))):
        with pytest.raises(TypeError):
            call(**{**args, **bad})


def test_ops_run_the_same_kernels():
    x = Expanded([30], [50], 2, BF, "dense")
    o, _ = x.run()
    q, k, v, pe = (t.to(DEV) for t in (x.q, x.k, x.v, x.pe))
    out = torch.empty_like(o)
    torch.ops.kda355.latent_prefill(q, k, v, pe, _i32([0, 30]), _i32([0, 50]), out)
    assert torch.equal(out, o)
    a = Absorbed([20, 5], 1, 4, 16, BF)
    o, _ = a.run()
    out = torch.empty_like(o)
    torch.ops.kda355.latent_decode(a.ql.to(DEV), a.qp.to(DEV), a.cache.to(DEV), a.table.to(DEV), _i32(a.lens), out)
    assert torch.equal(out, o)


def test_refused_after_a_like_call_was_taken():
    """What a call of the same shapes had found right does not let another one through."""
    x = Expanded([8], [8], 2, BF, "dense")
    q, k, v, pe = (t.to(DEV) for t in (x.q, x.k, x.v, x.pe))
    cu = _i32([0, 8])
    for _ in range(2):
        kda355.latent_prefill(q, k, v, pe, cu, cu)
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    few = torch.empty(kda355.latent_prefill_workspace_bytes(1, 2, 8, 8, num_cus=cus) - 1, dtype=torch.uint8, device=DEV)
    odd = torch.empty(8 * 2 * 192 + 1, device=DEV, dtype=BF)[1:].view(8, 2, 192)  # the same shape and strides, 2 bytes off
    for bad in (dict(q=odd), dict(k=k[:7]), dict(cu_seqlens_k=_i32([0, 4, 8])), dict(workspace=few)):
        with pytest.raises(ValueError):
            kda355.latent_prefill(**{**dict(q=q, k=k, v=v, k_pe=pe, cu_seqlens_q=cu, cu_seqlens_k=cu), **bad})
    for bad in (dict(q=q.half()), dict(cu_seqlens_q=cu.cpu()), dict(v=v.cpu())):
        with pytest.raises(TypeError):
            kda355.latent_prefill(**{**dict(q=q, k=k, v=v, k_pe=pe, cu_seqlens_q=cu, cu_seqlens_k=cu), **bad})
    a = Absorbed([20, 5], 1, 4, 16, BF)
    args = dict(q_latent=a.ql.to(DEV), q_pe=a.qp.to(DEV), cache=a.cache.to(DEV), block_table=a.table.to(DEV), seq_lens=_i32([20, 5]))
    few = torch.empty(kda355.latent_decode_workspace_bytes(2, 1, 4, 16, a.table.shape[1], num_cus=cus) - 1, dtype=torch.uint8,
                      device=DEV)
    for _ in range(2):
        kda355.latent_decode(**args)
    for bad in (dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(seq_lens=_i32([1])),
                dict(workspace=few)):
        with pytest.raises(ValueError):
            kda355.latent_decode(**{**args, **bad})
    for bad in (dict(cache=args["cache"].half()), dict(seq_lens=_i32([20, 5]).float()), dict(q_pe=a.qp)):
        with pytest.raises(TypeError):
            kda355.latent_decode(**{**args, **bad})


def test_a_scale_that_is_written_again_counts_anew():
    """A scale may be given as anything that float() takes: its value at the call is the one that counts, and nothing that
    is kept from one call for the next holds on to it."""
    x, a = Expanded([9], [20], 2, BF), Absorbed([20, 5], 1, 4, 16, BF, prefix=30)
    s, flag = torch.tensor(0.25), torch.tensor(True)
    for value in (0.25, 0.03125, 0.25):
        s.fill_(value)
        for run in (lambda z: x.run(scale=z), lambda z: a.run(scale=z)):
            (o, lse), (o2, lse2) = run(s), run(value)
            assert torch.equal(o, o2) and torch.equal(lse, lse2)
    for value in (True, False, True):
        flag.fill_(value)
        (o, lse), (o2, lse2) = x.run(flag), x.run(value)
        assert torch.equal(o, o2) and torch.equal(lse, lse2)
    for seen in (kda355.latent._prefill_seen, kda355.latent._decode_seen):
        assert not any(isinstance(part, torch.Tensor) for key in seen for part in key)
    for bad in ("much", [1.0]):
        with pytest.raises((TypeError, ValueError)):
            x.run(scale=bad)


@pytest.mark.parametrize("value", [float("inf"), -float("inf")])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("H,S,prefix", [(4, 1, None), (12, 3, None), (40, 2, None), (96, 1, None), (12, 1, 75), (96, 2, 75)])
def test_decode_infinite_values_that_are_seen(value, wide, H, S, prefix):
    """A token whose score is -inf because one of its values is infinite has a weight of 0, and 0 times that value is NaN: in
    that channel of every row that sees it, wherever the token stands (a tile that all rows see whole or not), and nowhere
    else."""
    lens, size = [105, 64, 40], 16
    for at in (3, 33, 60, 66, 97, 100, 103):  # within sequence 0, or within the prefix; tiles end at 64 and 96
        x = Absorbed(lens, S, H, size, BF, prefix=prefix)
        if prefix is not None and at >= prefix:
            continue
        x.ql[..., 7] = -1.0 if value > 0 else 1.0
        pages = x.prefix_table if prefix is not None else x.table[0]
        x.cache[int(pages[at // size]), at % size, 7] = value
        if wide:
            x.widen()
        o, lse = x.run()
        o, lse = o.cpu(), lse.cpu()
        head, head_there = R.cache_rows(x.cache, x.prefix_table, prefix) if prefix is not None else R.cache_rows(x.cache, [], 0)
        for n, length in enumerate(lens):
            rows, there = R.cache_rows(x.cache, x.table[n], length)
            rows, there = torch.cat([head, rows]), torch.cat([head_there, there])
            P, j = len(head), torch.arange(len(head) + length)
            s = torch.arange(S).repeat_interleave(H)
            visible = there[None, :] & (j[None, :] < P + length - (S - 1 - s)[:, None])
            sees = visible[:, at].clone() if prefix is not None or n == 0 else torch.zeros(S * H, dtype=torch.bool)
            if prefix is not None or n == 0:  # the token adds nothing but its NaN
                visible[:, at] = False
                rows[at] = 0.0
            q = torch.cat([x.ql, x.qp], dim=-1)[n * S:(n + 1) * S].double().reshape(S * H, ROW)
            ref, A, ref_lse, Z, vmax, L = R.attend(q, rows, rows[:, :LAT], visible, SCALE)
            got, got_lse = o[n * S:(n + 1) * S].reshape(S * H, LAT), lse[n * S:(n + 1) * S].reshape(S * H)
            assert torch.isnan(got[sees, 7]).all(), f"token {at} of sequence {n}: {got[sees, 7]}"
            keep = [c for c in range(LAT) if c != 7]
            R.check(got[:, keep], got_lse, (ref[:, keep], A[:, keep], ref_lse, Z, vmax, L), BF, ROW, f"token {at} seq {n}")
            if not sees.all():
                r = ~sees
                R.check(got[r], got_lse[r], (ref[r], A[r], ref_lse[r], Z[r], vmax[r], L), BF, ROW, f"token {at} seq {n}, unseen")


@pytest.mark.parametrize("cu_q,cu_k,keys", [([-5, 1 << 30], [50, 0], 0), ([-5, 1 << 30], [0, 1 << 30], 50), ([0, 25], [-3, 50], 50),
                                            ([0, 1 << 31 - 1], [1 << 30, 1 << 30], 0), ([0, 20], [0, -1], 0)])
def test_prefill_offsets_outside_leave_the_rest_alone(cu_q, cu_k, keys):
    """cu_seqlens past the tensors, or falling: clamped, every row of the 20 queries is written, with zeros and -inf where no
    key is left, and nothing around the outputs is."""
    x = Expanded([20], [50], 2, BF, "dense")
    o, lse = x.run()
    q, k, v, pe = (t.to(DEV) for t in (x.q, x.k, x.v, x.pe))
    wide = torch.full((20 + 300, 4, HEAD + 16), 3.0, dtype=BF, device=DEV)
    lines = torch.full((20 + 300, 2), 5.0, device=DEV)
    kda355.latent_prefill(q, k, v, pe, _i32(cu_q), _i32(cu_k), out=wide[150:170, 1:3, 8:8 + HEAD], lse=lines[150:170])
    got, got_lse = wide[150:170, 1:3, 8:8 + HEAD].clone(), lines[150:170].clone()
    if keys:
        assert torch.equal(got, o) and torch.equal(got_lse, lse)
    else:
        assert (got == 0).all() and (got_lse == -float("inf")).all()
    wide[150:170, 1:3, 8:8 + HEAD] = 3.0
    lines[150:170] = 5.0
    assert (wide == 3.0).all() and (lines == 5.0).all()
