"""The latent cache in 4 bits, accumulated attention weights and eviction through torch.ops.kda355.*: every op against the Python
entry point of its name, bit for bit, eager and as torch.compile traces it (aot_eager, fullgraph)."""
import pytest
import torch

import kda355

pytestmark = pytest.mark.gpu
DEV, BF = "cuda", torch.bfloat16
LAT, PE, ROW, ROW4 = 512, 64, 576, 400


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _state(bits):
    """Two layers' caches with their books, and a step's queries."""
    g = torch.Generator().manual_seed(33)
    rnd = lambda *shape: torch.randn(*shape, generator=g).to(BF).to(DEV)  # noqa: E731
    size, pages, T = 16, 12, 90
    row, dtype = (ROW, BF) if bits == 16 else (ROW4, torch.uint8)
    table = [[0, 3, 6, 9], [1, 4, -1, -1], [5, 2, 8, -1]]
    lens = [60, 17, 40]
    slots = [table[n][j // size] * size + j % size for n in range(3) for j in range(lens[n])]
    st = dict(pools=[torch.zeros(pages, size, row, dtype=dtype, device=DEV) for _ in range(2)], table=_i32(table), lens=_i32(lens),
              refs=_i32([1] * 7 + [0, 1, 1, 0, 0]), free=_i32([7, 10, 11] + [-1] * 9), num=_i32([3]), latent=rnd(sum(lens), LAT),
              k_pe=rnd(sum(lens), PE), slots=torch.tensor(slots, device=DEV), q_latent=rnd(6, 4, LAT), q_pe=rnd(6, 4, PE),
              cu=_i32([0, 60, 77, 117]), gathered=torch.zeros(T + 27, ROW, dtype=BF, device=DEV),
              out=torch.zeros(6, 4, LAT, dtype=BF, device=DEV), lse=torch.zeros(6, 4, device=DEV), rows=_i32([2, 0, 1]),
              weights=[torch.zeros(3, 64, device=DEV) for _ in range(2)])
    return st


def _books(s):
    return [s[n] for n in ("table", "lens", "refs", "free", "num", "rows")]


def _python(s):
    for pool, w, scale in zip(s["pools"], s["weights"], (0.05, 0.11)):
        kda355.latent_append(s["latent"], s["k_pe"], pool, s["slots"])
        kda355.latent_decode(s["q_latent"], s["q_pe"], pool, s["table"], s["lens"], scale, out=s["out"], lse=s["lse"])
        kda355.latent_weights(s["q_latent"], s["q_pe"], pool, s["table"], s["lens"], s["lse"], w, scale)
    kda355.evict_tokens(s["pools"], s["weights"], *_books(s), 24, 5, 16)
    kda355.latent_gather(s["pools"][1], s["table"], s["cu"], s["gathered"])


def _ops(s):
    o = torch.ops.kda355
    for pool, w, scale in zip(s["pools"], s["weights"], (0.05, 0.11)):
        o.latent_append(s["latent"], s["k_pe"], pool, s["slots"])
        o.latent_decode(s["q_latent"], s["q_pe"], pool, s["table"], s["lens"], s["out"], scale, s["lse"])
        o.latent_weights(s["q_latent"], s["q_pe"], pool, s["table"], s["lens"], s["lse"], w, scale)
    o.evict_tokens(s["pools"], s["weights"], *_books(s), 24, 5, 16)
    o.latent_gather(s["pools"][1], s["table"], s["cu"], s["gathered"])


def _same(a, b):
    for name in a:
        for x, y in zip(*([s[name]] if isinstance(s[name], torch.Tensor) else s[name] for s in (a, b))):
            assert torch.equal(x, y), name


@pytest.mark.parametrize("bits", [16, 4])
def test_ops_are_the_entry_points(bits):
    first, a, b = _state(bits), _state(bits), _state(bits)
    _python(a)
    _ops(b)
    _same(a, b)
    for name in ("table", "lens", "refs", "free", "num", "gathered", "out", "lse"):
        assert not torch.equal(a[name], first[name]), f"{name} was not written"
    for name in ("pools", "weights"):
        assert all(not torch.equal(x, y) for x, y in zip(a[name], first[name]))
    assert a["lens"].tolist() == [24, 17, 24] and a["num"].tolist() == [6]  # two pages of the first, one of the third


@pytest.mark.parametrize("which", ["whole", "append", "gather", "decode", "weights", "evict"])
def test_ops_compiled(which):
    """One graph without breaks; what the ops write into is what the eager calls write."""
    o = torch.ops.kda355
    steps = dict(
        whole=_ops,
        append=lambda s: o.latent_append(s["latent"], s["k_pe"], s["pools"][0], s["slots"]),
        gather=lambda s: o.latent_gather(s["pools"][0], s["table"], s["cu"], s["gathered"]),
        decode=lambda s: o.latent_decode(s["q_latent"], s["q_pe"], s["pools"][0], s["table"], s["lens"], s["out"], lse=s["lse"]),
        weights=lambda s: o.latent_weights(s["q_latent"], s["q_pe"], s["pools"][0], s["table"], s["lens"], s["lse"], s["weights"][0]),
        evict=lambda s: o.evict_tokens(s["pools"], s["weights"], *_books(s), 24, 5, 16))
    step = steps[which]

    def run(s):
        step(s)
        return s["lens"] + 1

    torch._dynamo.reset()
    a, b = _state(4), _state(4)
    x, y = run(a), torch.compile(run, backend="aot_eager", fullgraph=True)(b)
    torch.cuda.synchronize()
    assert torch.equal(x, y)
    _same(a, b)


def test_ops_refuse_like_the_entry_points():
    s = _state(4)
    o = torch.ops.kda355
    with pytest.raises(ValueError):
        o.evict_tokens(s["pools"], s["weights"], *_books(s), 0, 0, 16)
    with pytest.raises(ValueError):
        o.latent_weights(s["q_latent"], s["q_pe"], s["pools"][0], s["table"], s["lens"], s["lse"], s["weights"][0][:, :60])
    with pytest.raises(TypeError):
        o.latent_weights(s["q_latent"], s["q_pe"], s["pools"][0], s["table"], s["lens"], s["lse"].half(), s["weights"][0])
    with pytest.raises(NotImplementedError):
        o.evict_tokens([p.cpu() for p in s["pools"]], [w.cpu() for w in s["weights"]], *(t.cpu() for t in _books(s)), 24, 5, 16)
