"""Latent attention, its paged cache and its pages through torch.ops.kda355.*: every op against the Python entry point of its
name, bit for bit, eager and as torch.compile traces it (aot_eager, fullgraph: functionalized, the lists of pools too)."""
import pytest
import torch

import kda355
from latent_ref import HEAD, LAT, PE, ROW

pytestmark = pytest.mark.gpu
DEV, BF = "cuda", torch.bfloat16


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _state():
    """A cache of two layers with its books, queries for both forms, and a KDA layer's state rows."""
    g = torch.Generator().manual_seed(21)
    rnd = lambda *shape: torch.randn(*shape, generator=g).to(BF).to(DEV)  # noqa: E731
    size, pages = 16, 24
    st = dict(pools=[rnd(pages, size, ROW) for _ in range(2)], rows=torch.randn(6, 4, 32, generator=g).to(DEV),
              table=_i32([[0, 3, 6, -1], [9, 12, -1, -1], [15, -1, -1, -1], [-1] * 4, [-1] * 4, [-1] * 4]),
              lens=_i32([40, 17, 9, 0, 0, 0]), refs=_i32([1 if p in (0, 3, 6, 9, 12, 15) else 0 for p in range(pages)]),
              parents=_i32([0, 1, 0]), children=_i32([3, 4, 5]), gone=_i32([1, 4]),
              latent=rnd(5, LAT), k_pe=rnd(5, PE), slots=torch.tensor([3, 50, -1, 100, 9], device=DEV),
              q_latent=rnd(6, 4, LAT), q_pe=rnd(6, 4, PE), q=rnd(20, 2, HEAD + PE), k=rnd(30, 2, HEAD), v=rnd(30, 2, HEAD),
              pe=rnd(30, PE), cu_q=_i32([0, 7, 20]), cu_k=_i32([0, 10, 30]), cu=_i32([0, 40, 57, 66, 106, 123, 163]))
    left = [p for p in range(pages) if not int(st["refs"][p])]
    st.update(free=_i32(left + [-1] * (pages - len(left))), num=_i32([len(left)]), prefix=_i32([20, 21]), prefix_len=_i32([23]),
              gathered=torch.zeros(163, ROW, dtype=BF, device=DEV), out=torch.zeros(6, 4, LAT, dtype=BF, device=DEV),
              lse=torch.zeros(6, 4, device=DEV), behind=torch.zeros(6, 4, LAT, dtype=BF, device=DEV),
              pout=torch.zeros(20, 2, HEAD, dtype=BF, device=DEV), plse=torch.zeros(20, 2, device=DEV))
    return st


def _python(s):
    kda355.latent_append(s["latent"], s["k_pe"], s["pools"][0], s["slots"])
    kda355.fork_pages(s["pools"], s["table"], s["lens"], s["refs"], s["free"], s["num"], s["parents"], s["children"], 16)
    kda355.copy_rows([s["rows"]], s["parents"], s["children"])
    kda355.latent_gather(s["pools"][0], s["table"], s["cu"], s["gathered"])
    kda355.latent_decode(s["q_latent"], s["q_pe"], s["pools"][0], s["table"], s["lens"], out=s["behind"], prefix_table=s["prefix"],
                         prefix_len=s["prefix_len"])
    kda355.free_pages(s["table"], s["lens"], s["refs"], s["free"], s["num"], s["gone"], 16)
    kda355.compact_pages(s["pools"], s["table"], s["refs"], s["free"], s["num"])
    kda355.latent_decode(s["q_latent"], s["q_pe"], s["pools"][1], s["table"], s["lens"], 0.11, out=s["out"], lse=s["lse"])
    kda355.latent_prefill(s["q"], s["k"], s["v"], s["pe"], s["cu_q"], s["cu_k"], None, False, out=s["pout"], lse=s["plse"])


def _ops(s):
    o = torch.ops.kda355
    o.latent_append(s["latent"], s["k_pe"], s["pools"][0], s["slots"])
    o.fork_pages(s["pools"], s["table"], s["lens"], s["refs"], s["free"], s["num"], s["parents"], s["children"], 16)
    o.copy_rows([s["rows"]], s["parents"], s["children"])
    o.latent_gather(s["pools"][0], s["table"], s["cu"], s["gathered"])
    o.latent_decode(s["q_latent"], s["q_pe"], s["pools"][0], s["table"], s["lens"], s["behind"], prefix_table=s["prefix"],
                    prefix_len=s["prefix_len"])
    o.free_pages(s["table"], s["lens"], s["refs"], s["free"], s["num"], s["gone"], 16)
    o.compact_pages(s["pools"], s["table"], s["refs"], s["free"], s["num"])
    o.latent_decode(s["q_latent"], s["q_pe"], s["pools"][1], s["table"], s["lens"], s["out"], 0.11, s["lse"])
    o.latent_prefill(s["q"], s["k"], s["v"], s["pe"], s["cu_q"], s["cu_k"], s["pout"], None, False, s["plse"])


def _same(a, b):
    for name in a:
        for x, y in zip(*([s[name]] if isinstance(s[name], torch.Tensor) else s[name] for s in (a, b))):
            assert torch.equal(x, y), name


def test_ops_are_the_entry_points():
    first, a, b = _state(), _state(), _state()
    _python(a)
    _ops(b)
    _same(a, b)
    for name in ("rows", "table", "lens", "refs", "free", "gathered", "out", "lse", "behind", "pout", "plse"):
        assert not torch.equal(a[name], first[name]), f"{name} was not written"
    assert all(not torch.equal(x, y) for x, y in zip(a["pools"], first["pools"]))
    assert a["num"].tolist() == [18]  # 18, three taken by the forks, three given up (9, 12 and the second fork's own)


@pytest.mark.parametrize("which", ["whole", "append", "gather", "copy", "fork", "free", "compact", "decode", "prefill"])
def test_ops_compiled(which):
    """One graph without breaks; what the ops write into is what the eager calls write."""
    o = torch.ops.kda355
    steps = dict(
        whole=_ops,
        append=lambda s: o.latent_append(s["latent"], s["k_pe"], s["pools"][0], s["slots"]),
        gather=lambda s: o.latent_gather(s["pools"][0], s["table"], s["cu"], s["gathered"]),
        copy=lambda s: o.copy_rows([s["rows"], s["pools"][0][:6], s["pools"][1][6:]], s["parents"], s["children"]),
        fork=lambda s: o.fork_pages(s["pools"], s["table"], s["lens"], s["refs"], s["free"], s["num"], s["parents"],
                                    s["children"], 16),
        free=lambda s: o.free_pages(s["table"], s["lens"], s["refs"], s["free"], s["num"], s["gone"], 16),
        compact=lambda s: o.compact_pages(s["pools"], s["table"], s["refs"], s["free"], s["num"]),
        decode=lambda s: o.latent_decode(s["q_latent"], s["q_pe"], s["pools"][0], s["table"], s["lens"], s["out"], lse=s["lse"]),
        prefill=lambda s: o.latent_prefill(s["q"], s["k"], s["v"], s["pe"], s["cu_q"], s["cu_k"], s["pout"], lse=s["plse"]))
    step = steps[which]

    def run(s):
        step(s)
        return s["lens"] + 1

    torch._dynamo.reset()
    a, b = _state(), _state()
    x, y = run(a), torch.compile(run, backend="aot_eager", fullgraph=True)(b)
    torch.cuda.synchronize()
    assert torch.equal(x, y)
    _same(a, b)


def test_ops_refuse_like_the_entry_points():
    s = _state()
    o = torch.ops.kda355
    with pytest.raises(ValueError):
        o.fork_pages(s["pools"], s["table"], s["lens"], s["refs"], s["free"], s["num"], s["parents"], s["children"], 0)
    with pytest.raises(ValueError):
        o.compact_pages([s["pools"][0][:5]], s["table"], s["refs"], s["free"], s["num"])
    with pytest.raises(TypeError):
        o.latent_append(s["latent"].half(), s["k_pe"], s["pools"][0], s["slots"])
    with pytest.raises(ValueError):
        o.latent_gather(s["pools"][0], s["table"], s["cu"][:3], s["gathered"])
    with pytest.raises(TypeError):
        o.copy_rows([s["rows"]], s["parents"].long(), s["children"])
    with pytest.raises(NotImplementedError):
        o.free_pages(*(s[n].cpu() for n in ("table", "lens", "refs", "free", "num", "gone")), 16)
