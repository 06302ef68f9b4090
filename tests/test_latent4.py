"""Caches in 4 bits, accumulated weights and eviction without a GPU: the argument structs, the refusals of the C entries (all before any
device call) and of the Python functions, the op schemas, the plain forms that the GPU tests go by."""
import ctypes
import subprocess
import sys
import tempfile

import pytest
import torch

import latent4_ref as Q
from test_latent import FAKE, ROOT, _decode_args, _lib, _tokens_args


def test_struct_layout_matches_header():
    m = _lib()
    names = ["KdaLatentTokensArgs", "KdaLatentWeightsArgs", "KdaEvictLayer", "KdaEvictArgs"]
    src = '#include "kda355.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(){\n'
    for n in names:
        src += f'printf("%zu", sizeof({n}));\n'
        for f, _ in getattr(m, n)._fields_:
            src += f'printf(" %zu", offsetof({n}, {f}));\n'
        src += 'printf("\\n");\n'
    src += 'printf("%d %d %u\\n", KDA355_LATENT_ROW_4BIT, KDA355_LATENT_GROUP, KDA355_EVICT_MORE); return 0;}\n'
    with tempfile.TemporaryDirectory() as d:
        with open(f"{d}/m.c", "w") as f:
            f.write(src)
        subprocess.run(["gcc", "-I", str(ROOT / "include"), f"{d}/m.c", "-o", f"{d}/m"], check=True)
        lines = subprocess.run([f"{d}/m"], capture_output=True, text=True, check=True).stdout.splitlines()
    for n, line in zip(names, lines):
        cls = getattr(m, n)
        assert [int(x) for x in line.split()] == [ctypes.sizeof(cls)] + [getattr(cls, f).offset for f, _ in cls._fields_], n
    assert lines[-1] == f"{Q.ROW4} {Q.GROUP} {m.EVICT_MORE}"
    import kda355
    assert kda355.latent.ROW_4BIT == Q.ROW4


def _tokens4(**kw):
    return _tokens_args(**{**dict(page_stride=16 * 400), **kw})


def _decode4(**kw):
    return _decode_args(**{**dict(page_stride=64 * 400), **kw})


def _weights_args(**kw):
    a = dict(q_latent=FAKE, q_pe=FAKE, cache=FAKE, block_table=FAKE, seq_lens=FAKE, lse=FAKE, weights=FAKE, ql_row=1024, ql_head=512,
             qp_row=128, qp_head=64, weights_row=256, page_stride=64 * 576, pages=4, table_stride=4, B=1, S=1, H=2, page_size=64,
             table_width=4, cache_bits=16, scale=1.0)
    a.update(kw)
    return _lib().KdaLatentWeightsArgs(**a)


def _evict_args(layers=((FAKE, 400, 6400, FAKE, 64),), **kw):
    m = _lib()
    a = dict(num_layers=len(layers), n=2, src=FAKE, block_table=FAKE, seq_lens=FAKE, ref_counts=FAKE, free_pages=FAKE, num_free=FAKE,
             workspace=FAKE, workspace_bytes=1 << 40, table_stride=4, rows=4, table_width=4, pages=8, page_size=16, keep=20, recent=4)
    a.update(kw)
    a = m.KdaEvictArgs(**a)
    for i, y in enumerate(layers[:m.MAX_POOLS]):
        a.layer[i] = m.KdaEvictLayer(*y)
    return a


BAD = [(op, _tokens4, kw, msg) for op in ("latent4_append", "latent4_gather") for kw, msg in [
    (dict(T=-1), b"T=-1"), (dict(pages=0), b"pages=0"), (dict(page_size=0), b"page_size=0"), (dict(cache=0), b"null"),
    (dict(T=1 << 25), b"2^25"), (dict(page_stride=16 * 400 - 16), b"dense"), (dict(page_stride=16 * 400 + 8), b"aligned"),
    (dict(cache=FAKE + 8), b"aligned"), (dict(dtype=2), b"dtype"), (dict(dtype=-1), b"dtype")]]
BAD += [("latent4_append", _tokens4, kw, msg) for kw, msg in [
    (dict(slots=0), b"null"), (dict(latent=0), b"null"), (dict(latent_row=513), b"aligned"), (dict(k_pe=FAKE + 2), b"aligned")]]
BAD += [("latent4_gather", _tokens4, kw, msg) for kw, msg in [
    (dict(out=0), b"null"), (dict(out_row=577), b"aligned"), (dict(table_width=0), b"table_width"), (dict(table_stride=2), b""), (dict(N=-1), b"N=-1")]]
BAD += [("latent4_decode", _decode4, kw, msg) for kw, msg in [
    (dict(page_stride=64 * 400 - 16), b"dense"), (dict(page_stride=64 * 400 + 8), b"aligned"), (dict(cache=FAKE + 8), b"aligned"),
    (dict(flags=1), b"flags"), (dict(flags=2), b"flags"), (dict(dtype=3), b"dtype"), (dict(cache=0), b"null"), (dict(S=0), b"S=0"),
    (dict(prefix_table=FAKE), b"prefix_len"), (dict(scale=0.0), b"positive"), (dict(workspace=0), b"workspace"),
    (dict(workspace_bytes=0), b"workspace"), (dict(table_width=1 << 30), b"2^31")]]
BAD += [("latent_weights", _weights_args, kw, msg) for kw, msg in [
    (dict(B=-1), b"B=-1"), (dict(S=0), b"S=0"), (dict(H=0), b"H=0"), (dict(page_size=0), b"page_size"), (dict(table_width=1 << 30), b"2^31"),
    (dict(table_width=(1 << 25) - 1, weights_row=1 << 31), b"2^31"), (dict(B=1 << 20, S=1 << 10), b"too large"), (dict(B=1 << 22), b"too large"),
    (dict(B=1 << 20, table_width=1 << 20, weights_row=1 << 26), b"2^38"), (dict(dtype=3), b"dtype"), (dict(cache_bits=8), b"cache_bits"),
    (dict(flags=1), b"flags"), (dict(lse=0), b"null"), (dict(weights=0), b"null"), (dict(seq_lens=0), b"null"), (dict(table_width=0), b"null"),
    (dict(pages=0), b"pages"), (dict(table_stride=3), b"table_stride"), (dict(weights_row=255), b"shorter"), (dict(q_pe=FAKE + 8), b"aligned"),
    (dict(ql_head=4), b"aligned"), (dict(page_stride=64 * 576 - 8), b"dense"), (dict(cache_bits=4, page_stride=64 * 400 - 16), b"dense"),
    (dict(cache_bits=4, page_stride=64 * 400 + 8), b"aligned"), (dict(scale=0.0), b"positive"), (dict(scale=float("nan")), b"positive"),
    (dict(num_cus=-1), b"num_cus")]]
BAD += [("evict_tokens", _evict_args, kw, msg) for kw, msg in [
    (dict(num_layers=-1), b"num_layers"), (dict(num_layers=25), b"num_layers"), (dict(layers=()), b"no layers"), (dict(n=-1), b"n=-1"),
    (dict(n=1 << 20), b"n="), (dict(n=65536), b"65535"), (dict(rows=0), b"rows=0"), (dict(table_width=0), b"table_width=0"), (dict(pages=0), b"pages=0"),
    (dict(page_size=0), b"page_size=0"), (dict(table_width=1 << 27), b"2^30"), (dict(keep=0), b"keep=0"), (dict(recent=-1), b"recent=-1"),
    (dict(recent=21), b"recent=21"), (dict(flags=2), b"flags"), (dict(table_stride=3), b"table_stride"), (dict(src=0), b"null"),
    (dict(block_table=0), b"null"), (dict(seq_lens=0), b"null"), (dict(num_free=0), b"null"), (dict(workspace=0), b"workspace"),
    (dict(workspace=FAKE + 4), b"workspace"), (dict(workspace_bytes=8), b"workspace"),
    (dict(layers=((0, 400, 6400, FAKE, 64),)), b"null"), (dict(layers=((FAKE, 400, 6400, 0, 64),)), b"null"),
    (dict(layers=((FAKE, 392, 6400, FAKE, 64),)), b"multiple of 16"), (dict(layers=((FAKE, 400, 6392, FAKE, 64),)), b"dense"),
    (dict(layers=((FAKE, 400, 6384, FAKE, 64),)), b"dense"), (dict(layers=((FAKE + 8, 400, 6400, FAKE, 64),)), b"aligned"),
    (dict(layers=((FAKE, 400, 6400, FAKE, 63),)), b"shorter"), (dict(layers=((FAKE, 400, 6400, FAKE, 64), (FAKE, 0, 16, FAKE, 64))), b"layer 1")]]


@pytest.mark.parametrize("op,make,kw,msg", BAD, ids=[f"{b[0]}-{'-'.join(b[2])}-{i}" for i, b in enumerate(BAD)])
def test_c_entry_refuses(op, make, kw, msg):
    m = _lib()
    a = make(**kw)
    assert getattr(m.lib(), f"kda355_{op}_launch")(ctypes.byref(a), None) == m.EINVAL
    assert msg in m.lib().kda355_last_error()


@pytest.mark.parametrize("op", ["latent4_append", "latent4_gather", "latent4_decode", "latent_weights", "evict_tokens"])
def test_c_entry_refuses_null(op):
    m = _lib()
    assert getattr(m.lib(), f"kda355_{op}_launch")(None, None) == m.EINVAL


def test_empty_calls_launch_nothing():
    m = _lib()
    for op, a in (("latent4_append", _tokens4(T=0)), ("latent4_gather", _tokens4(T=0)), ("latent4_gather", _tokens4(N=0)),
                  ("latent4_decode", _decode4(B=0)), ("latent_weights", _weights_args(B=0)), ("evict_tokens", _evict_args(n=0)),
                  ("evict_tokens", _evict_args(keep=64))):  # (no row can be longer)
        assert getattr(m.lib(), f"kda355_{op}_launch")(ctypes.byref(a), None) == 0, op


def test_evict_workspace():
    m = _lib()
    for n, layers, keep, recent in ((1, 1, 20, 4), (100, 24, 63, 0), (7, 3, 30, 30)):
        need = m.lib().kda355_evict_tokens_workspace_bytes(ctypes.byref(_evict_args(n=n, keep=keep, recent=recent, num_layers=layers)))
        assert 4 * n < need <= 1024 + n * layers * (64 * 8 + 64)
    assert m.lib().kda355_evict_tokens_workspace_bytes(ctypes.byref(_evict_args(keep=0))) == m.EINVAL
    assert m.lib().kda355_evict_tokens_workspace_bytes(None) == m.EINVAL


@pytest.mark.parametrize("n,layers,width,keep,recent", [(256, 24, 2048, 32768, 512), (65535, 24, 256, 8192, 100), (1000, 7, 200, 6000, 0),
                                                        (4, 24, 1 << 15, 1 << 20, 4096)])
def test_evict_workspace_is_bounded(n, layers, width, keep, recent):
    """Of the pairs that could move 128 MiB are held at a time, and those of one sequence's layers where they are more; 25 KiB and 16 bytes
    a part for 1024 (sequence, layer)s of long tables; lengths, counts and pages of recent tokens for all."""
    m = _lib()
    L = m.lib()
    a = _evict_args(n=n, num_layers=layers, table_width=width, page_size=64, pages=1 << 16, keep=keep, recent=recent)
    need = L.kda355_evict_tokens_workspace_bytes(ctypes.byref(a))
    pairs = 8 * layers * min(keep - recent, width * 64 - keep)
    parts = 1024 * (25 * 1024 + 16 * (width // 128 + 1)) if width * 64 - recent > 16384 else 0
    assert 4 * n < need <= max(128 << 20, pairs) + parts + 4 * n * (4 + recent // 64 + layers)


def test_evict_workspace_and_launch_take_the_same_rows():
    """A size that the launch refuses has no workspace; where no row can be longer than the budget both take more rows."""
    m = _lib()
    L = m.lib()
    assert L.kda355_evict_tokens_workspace_bytes(ctypes.byref(_evict_args(n=65535))) > 0
    for n in (65536, (1 << 20) - 1):
        assert L.kda355_evict_tokens_workspace_bytes(ctypes.byref(_evict_args(n=n))) == m.EINVAL
        assert b"65535" in L.kda355_last_error()
        assert L.kda355_evict_tokens_launch(ctypes.byref(_evict_args(n=n)), None) == m.EINVAL
        a = _evict_args(n=n, keep=64)  # (the table's tokens)
        assert L.kda355_evict_tokens_workspace_bytes(ctypes.byref(a)) > 0 and L.kda355_evict_tokens_launch(ctypes.byref(a), None) == 0


def test_cpu_tensors_raise():
    import kda355
    pe, i32 = torch.zeros(4, 64).bfloat16(), torch.zeros(4, dtype=torch.int32)
    cache, table = torch.zeros(2, 16, 400, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.int32)
    with pytest.raises(TypeError):
        kda355.latent_append(torch.zeros(4, 512).bfloat16(), pe, cache, torch.zeros(4, dtype=torch.int64))
    with pytest.raises(TypeError):
        kda355.latent_gather(cache, table, i32[:3], torch.zeros(4, 576).bfloat16())
    with pytest.raises(TypeError):
        kda355.latent_decode(torch.zeros(2, 2, 512).bfloat16(), torch.zeros(2, 2, 64).bfloat16(), cache, table, i32[:2])
    with pytest.raises(TypeError):
        kda355.latent_weights(torch.zeros(2, 2, 512).bfloat16(), torch.zeros(2, 2, 64).bfloat16(), cache, table, i32[:2], torch.zeros(2, 2),
                              torch.zeros(2, 32))
    with pytest.raises(TypeError):
        kda355.evict_tokens([cache], [torch.zeros(2, 32)], table, i32[:2], i32[:2], i32[:2], i32[:1], i32[:1], 20, 4, 16)


@pytest.mark.parametrize("kw", [dict(keep=(1 << 32) + 20), dict(keep=sys.maxsize), dict(keep=-(1 << 40)), dict(keep=1 << 31, recent=1 << 31),
                                dict(recent=(1 << 32) + 4), dict(size=(1 << 32) + 16)], ids=str)
def test_evict_sizes_beyond_32_bits(kw):
    """Refused before the tensors are looked at: the argument struct would take their low 32 bits."""
    import kda355
    i32 = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="32 bits"):
        kda355.evict_tokens([torch.zeros(2, 16, 400, dtype=torch.uint8)], [torch.zeros(2, 32)], torch.zeros(2, 2, dtype=torch.int32), i32[:2],
                            i32[:2], i32[:2], i32[:1], i32[:1], kw.get("keep", 20), kw.get("recent", 4), kw.get("size", 16))


def test_ops_are_registered():
    import kda355  # noqa: F401
    for name in ("latent_weights", "evict_tokens"):
        schema = str(getattr(torch.ops.kda355, name).default._schema)
        assert schema.endswith("-> ()")
    assert "Tensor(a0!) weights" in str(torch.ops.kda355.latent_weights.default._schema) or \
        "Tensor(a!) weights" in str(torch.ops.kda355.latent_weights.default._schema)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_plain_rounding(dtype):
    """What the plain rounding of the GPU tests gives back is nearest in its group: within half a step below 6, a fifth of the largest
    value in all, and unchanged where it is rounded again."""
    x = torch.randn(50, 512, generator=torch.Generator().manual_seed(0)).to(dtype)
    x[7] *= 1e-3
    rows = Q.rounded(x, torch.zeros(50, 64).to(dtype))
    y = Q.values(rows, dtype)[:, :512]
    top = x.double().abs().view(50, 16, 32).amax(dim=-1)
    assert ((y.double() - x.double()).abs().view(50, 16, 32).amax(dim=-1) <= top / 5).all()
    again = Q.values(Q.rounded(y, torch.zeros(50, 64).to(dtype)), dtype)[:, :512]
    assert torch.equal(again, y)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_plain_rounding_at_the_ends_of_the_type(dtype):
    """The stated bounds where the scale's limits hold: a / 4 for the largest numbers, 2^-127 or a / 5 for the smallest; a / 5 just inside."""
    top, x = Q.MOST[dtype], Q.ends(dtype)
    y = Q.values(Q.rounded(x, torch.zeros(len(x), 64).to(dtype)), dtype)[:, :512]
    assert torch.isfinite(y).all()
    a = x.double().abs().view(-1, 16, 32).amax(dim=-1)
    off = (y.double() - x.double()).abs().view(-1, 16, 32).amax(dim=-1)
    held = a > 7 * 2.0 ** top
    low = 2.0 ** -127 if dtype is torch.bfloat16 else 0.0
    bound = torch.where(held, a / 4, torch.where(a < 2.0 ** -123, (a / 5).clamp(min=low), a / 5))
    assert (off <= bound).all()
    assert (off > a / 5)[held].any() and held[0, 0]  # (the bound of the others does not hold there)
    if dtype is torch.bfloat16:
        assert (off > a / 5)[a < 2.0 ** -123].any()
