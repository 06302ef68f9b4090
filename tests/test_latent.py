"""Latent attention and the pages of its cache without a GPU: the argument structs, the refusals of the C entries (all before
any device call) and of the Python functions, the op schemas."""
import ctypes
import subprocess
import tempfile
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parent.parent
OPS = ("latent_prefill", "latent_decode", "latent_append", "latent_gather", "copy_rows", "fork_pages", "free_pages",
       "compact_pages")


def _lib():
    from kda355 import _lib
    return _lib


def test_struct_layout_matches_header():
    m = _lib()
    names = ["KdaLatentPrefillArgs", "KdaLatentDecodeArgs", "KdaLatentTokensArgs", "KdaPool", "KdaPagesArgs"]
    src = '#include "kda355.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(){\n'
    for n in names:
        src += f'printf("%zu", sizeof({n}));\n'
        for f, _ in getattr(m, n)._fields_:
            src += f'printf(" %zu", offsetof({n}, {f}));\n'
        src += 'printf("\\n");\n'
    src += f'printf("%d\\n", KDA355_MAX_POOLS); return 0;}}\n'
    with tempfile.TemporaryDirectory() as d:
        (Path(d) / "m.c").write_text(src)
        subprocess.run(["gcc", "-I", str(ROOT / "include"), str(Path(d) / "m.c"), "-o", str(Path(d) / "m")], check=True)
        lines = subprocess.run([str(Path(d) / "m")], capture_output=True, text=True, check=True).stdout.splitlines()
    for n, line in zip(names, lines):
        cls = getattr(m, n)
        want = [ctypes.sizeof(cls)] + [getattr(cls, f).offset for f, _ in cls._fields_]
        assert [int(x) for x in line.split()] == want, n
    assert int(lines[-1]) == m.MAX_POOLS


FAKE = 1 << 20  # a 16-byte aligned address that is never read: every call below is refused before any device call


def _prefill_args(**kw):
    a = dict(q=FAKE, k=FAKE, v=FAKE, k_pe=FAKE, out=FAKE, cu_q=FAKE, cu_k=FAKE, q_row=384, q_head=192, k_row=256, k_head=128,
             v_row=256, v_head=128, pe_row=64, out_row=256, out_head=128, Tq=8, Tk=8, N=1, H=2, scale=1.0,
             workspace=FAKE, workspace_bytes=1 << 40)
    a.update(kw)
    return _lib().KdaLatentPrefillArgs(**a)


def _decode_args(**kw):
    a = dict(q_latent=FAKE, q_pe=FAKE, cache=FAKE, block_table=FAKE, seq_lens=FAKE, out=FAKE, workspace=FAKE,
             workspace_bytes=1 << 40, ql_row=1024, ql_head=512, qp_row=128, qp_head=64, out_row=1024, out_head=512,
             page_stride=64 * 576, pages=4, table_stride=4, B=1, S=1, H=2, page_size=64, table_width=4, scale=1.0)
    a.update(kw)
    return _lib().KdaLatentDecodeArgs(**a)


def _tokens_args(**kw):
    a = dict(latent=FAKE, k_pe=FAKE, cache=FAKE, slots=FAKE, block_table=FAKE, cu=FAKE, out=FAKE, latent_row=512, pe_row=64,
             out_row=576, page_stride=16 * 576, pages=4, table_stride=4, T=3, page_size=16, table_width=4, N=1)
    a.update(kw)
    return _lib().KdaLatentTokensArgs(**a)


def _pages_args(pools=((FAKE, 1024, 1024, 8),), **kw):
    m = _lib()
    a = dict(num_pools=len(pools), n=2, src=FAKE, dst=FAKE, block_table=FAKE, seq_lens=FAKE, ref_counts=FAKE, free_pages=FAKE,
             num_free=FAKE, workspace=FAKE, table_stride=4, rows=4, table_width=4, pages=8, page_size=16)
    a.update(kw)
    a = m.KdaPagesArgs(**a)
    for i, p in enumerate(pools[:m.MAX_POOLS]):
        a.pool[i] = m.KdaPool(*p)
    return a


BAD = [("latent_prefill", _prefill_args, kw, msg) for kw, msg in [
    (dict(N=-1), b"N=-1"), (dict(H=0), b"H=0"), (dict(Tq=-1), b"Tq"), (dict(dtype=2), b"dtype"), (dict(flags=2), b"flags"),
    (dict(q=0), b"null"), (dict(k=0), b"null"), (dict(cu_k=0), b"null"), (dict(q=FAKE + 8), b"aligned"),
    (dict(k_row=260), b"aligned"), (dict(v_head=4), b"aligned"), (dict(pe_row=65), b"aligned"), (dict(out_head=4), b"aligned"),
    (dict(Tk=1 << 30), b"2^30"), (dict(Tq=1 << 30), b"2^30"), (dict(scale=0.0), b"positive"), (dict(scale=-1.0), b"positive"),
    (dict(scale=float("nan")), b"positive"), (dict(k_row=(1 << 23) + 8), b"2^23"), (dict(H=1 << 23), b"grid"), (dict(workspace=0), b"workspace"),
    (dict(workspace=FAKE + 16), b"workspace"), (dict(workspace_bytes=100), b"workspace"), (dict(num_cus=-1), b"num_cus")]]
BAD += [("latent_decode", _decode_args, kw, msg) for kw, msg in [
    (dict(B=-1), b"B=-1"), (dict(S=0), b"S=0"), (dict(H=0), b"H=0"), (dict(page_size=0), b"page_size"),
    (dict(table_width=1 << 30), b"2^31"), (dict(prefix_width=1 << 30), b"2^31"), (dict(B=1 << 20, S=1 << 10, H=2), b"too large"),
    (dict(dtype=3), b"dtype"), (dict(flags=1), b"flags"), (dict(cache=0), b"null"), (dict(seq_lens=0), b"null"),
    (dict(table_width=0), b"null"), (dict(prefix_table=FAKE), b"prefix_len"),
    (dict(prefix_table=FAKE, prefix_len=FAKE, prefix_width=0), b"prefix_len"), (dict(pages=0), b"pages"),
    (dict(table_stride=3), b"table_stride"), (dict(q_latent=FAKE + 8), b"aligned"), (dict(qp_row=4), b"aligned"),
    (dict(out=FAKE + 2), b"aligned"), (dict(page_stride=64 * 576 - 8), b"dense"), (dict(cache=FAKE + 8), b"aligned"),
    (dict(scale=0.0), b"positive"), (dict(scale=float("nan")), b"positive"), (dict(num_cus=-1), b"num_cus"),
    (dict(table_width=1 << 28, page_size=1), b"2^28"), (dict(prefix_width=8), b"prefix_table"),
    (dict(B=1 << 22), b"too large"), (dict(workspace=0), b"workspace"), (dict(workspace_bytes=0), b"workspace")]]
BAD += [(op, _tokens_args, kw, msg) for op in ("latent_append", "latent_gather") for kw, msg in [
    (dict(T=-1), b"T=-1"), (dict(pages=0), b"pages=0"), (dict(page_size=0), b"page_size=0"), (dict(cache=0), b"null"),
    (dict(T=1 << 25), b"2^25"), (dict(page_stride=100), b"dense"), (dict(cache=FAKE + 4), b"aligned")]]
BAD += [("latent_append", _tokens_args, kw, msg) for kw, msg in [
    (dict(slots=0), b"null"), (dict(latent_row=513), b"aligned"), (dict(k_pe=FAKE + 2), b"aligned")]]
BAD += [("latent_gather", _tokens_args, kw, msg) for kw, msg in [
    (dict(out=0), b"null"), (dict(out_row=577), b"aligned"), (dict(table_width=0), b"table_width"), (dict(table_stride=2), b"")]]
BAD += [("copy_rows", _pages_args, kw, msg) for kw, msg in [
    (dict(num_pools=-1), b"num_pools"), (dict(num_pools=25), b"num_pools"), (dict(pools=((0, 16, 16, 1),)), b"empty"),
    (dict(pools=((FAKE, 24, 32, 1),)), b"aligned"), (dict(pools=((FAKE + 8, 16, 16, 1),)), b"aligned"),
    (dict(pools=((FAKE, 32, 16, 2),)), b"aligned"), (dict(pools=((FAKE, 1 << 31, 1 << 31, 2),)), b"too long"),
    (dict(n=-1), b"n=-1"), (dict(n=1 << 23), b"n="), (dict(src=0), b"null")]]
BAD += [(op, _pages_args, kw, msg) for op in ("fork_pages", "free_pages", "compact_pages") for kw, msg in [
    (dict(rows=0), b"rows=0"), (dict(table_width=0), b"table_width=0"), (dict(pages=0), b"pages=0"),
    (dict(page_size=0), b"page_size=0"), (dict(table_width=1 << 28), b"2^31"), (dict(table_stride=3), b"table_stride"),
    (dict(block_table=0), b"null"), (dict(num_free=0), b"null")]]
BAD += [("fork_pages", _pages_args, kw, msg) for kw, msg in [
    (dict(seq_lens=0), b"null"), (dict(workspace=0), b"null"), (dict(n=-2), b"n=-2"), (dict(dst=0), b"null")]]
BAD += [("free_pages", _pages_args, kw, msg) for kw, msg in [(dict(seq_lens=0), b"null"), (dict(src=0), b"null")]]
BAD += [("compact_pages", _pages_args, dict(workspace=0), b"null")]


@pytest.mark.parametrize("op,make,kw,msg", BAD, ids=[f"{b[0]}-{'-'.join(b[2])}-{i}" for i, b in enumerate(BAD)])
def test_c_entry_refuses(op, make, kw, msg):
    m = _lib()
    a = make(**kw)
    assert getattr(m.lib(), f"kda355_{op}_launch")(ctypes.byref(a), None) == m.EINVAL
    assert msg in m.lib().kda355_last_error()


@pytest.mark.parametrize("op", OPS)
def test_c_entry_refuses_null(op):
    m = _lib()
    assert getattr(m.lib(), f"kda355_{op}_launch")(None, None) == m.EINVAL


def test_empty_calls_launch_nothing():
    """Sizes of zero return 0 before any device call (there is no GPU here)."""
    m = _lib()
    for op, a in (("latent_prefill", _prefill_args(N=0)), ("latent_prefill", _prefill_args(Tq=0)),
                  ("latent_decode", _decode_args(B=0)), ("latent_append", _tokens_args(T=0)),
                  ("latent_gather", _tokens_args(T=0)), ("copy_rows", _pages_args(n=0)),
                  ("copy_rows", _pages_args(pools=())), ("fork_pages", _pages_args(n=0)), ("free_pages", _pages_args(n=0))):
        assert getattr(m.lib(), f"kda355_{op}_launch")(ctypes.byref(a), None) == 0, op


def test_workspace_is_checked():
    import kda355
    m = _lib()
    for B, S, H, width in ((1, 1, 12, 64), (64, 1, 64, 100), (16, 8, 96, 200)):
        need = kda355.latent_decode_workspace_bytes(B, S, H, 64, width)
        assert 0 <= need < 1 << 30
        if need:
            a = _decode_args(B=B, S=S, H=H, table_width=width, table_stride=width, workspace_bytes=need - 1)
            assert m.lib().kda355_latent_decode_launch(ctypes.byref(a), None) == m.EINVAL
            assert b"workspace" in m.lib().kda355_last_error()
            a = _decode_args(B=B, S=S, H=H, table_width=width, table_stride=width, workspace=FAKE + 16)
            assert m.lib().kda355_latent_decode_launch(ctypes.byref(a), None) == m.EINVAL
    with pytest.raises(ValueError):
        kda355.latent_decode_workspace_bytes(1, 0, 1, 1, 1)
    for N, H, Tq, Tk in ((1, 16, 77, 1277), (1, 32, 8192, 8192), (64, 96, 64, 1 << 20)):
        assert 0 < kda355.latent_prefill_workspace_bytes(N, H, Tq, Tk) < 1 << 30
    assert kda355.latent_prefill_workspace_bytes(0, 1, 0, 0) == 0
    with pytest.raises(ValueError):
        kda355.latent_prefill_workspace_bytes(1, 0, 1, 1)


def test_cpu_tensors_raise():
    import kda355
    q, kv, pe = torch.zeros(4, 2, 192).bfloat16(), torch.zeros(4, 2, 128).bfloat16(), torch.zeros(4, 64).bfloat16()
    cu, i32 = torch.tensor([0, 4], dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    cache, table = torch.zeros(2, 16, 576).bfloat16(), torch.zeros(2, 2, dtype=torch.int32)
    with pytest.raises(TypeError):
        kda355.latent_prefill(q, kv, kv, pe, cu, cu)
    with pytest.raises(TypeError):
        kda355.latent_prefill(q.float(), kv, kv, pe, cu, cu)
    with pytest.raises(TypeError):
        kda355.latent_decode(torch.zeros(2, 2, 512).bfloat16(), pe, cache, table, i32[:2])
    with pytest.raises(TypeError):
        kda355.latent_append(torch.zeros(4, 512).bfloat16(), pe, cache, torch.zeros(4, dtype=torch.int64))
    with pytest.raises(TypeError):
        kda355.latent_gather(cache, table, cu, torch.zeros(4, 576).bfloat16())
    with pytest.raises(TypeError):
        kda355.copy_rows([cache], i32, i32)
    with pytest.raises(TypeError):
        kda355.fork_pages([cache], table, i32[:2], i32[:2], i32[:2], i32[:1], i32[:1], i32[:1], 16)
    with pytest.raises(TypeError):
        kda355.free_pages(table, i32[:2], i32[:2], i32[:2], i32[:1], i32[:1], 16)
    with pytest.raises(TypeError):
        kda355.compact_pages([cache], table, i32[:2], i32[:2], i32[:1])


@pytest.mark.parametrize("op", OPS)
def test_op_registered(op):
    import kda355  # noqa: F401
    schema = getattr(torch.ops.kda355, op).default._schema
    assert len(schema.returns) == 0
    assert any(a.alias_info is not None and a.alias_info.is_write for a in schema.arguments)
