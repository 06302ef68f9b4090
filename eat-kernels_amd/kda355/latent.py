"""Latent attention and its paged cache (host side of kda355_latent_*): the attention layers that stand between the KDA
layers of a hybrid model.  No counterpart in the reference, which holds KDA layers only.

Every token leaves one latent vector of 512 values and a positional part of 64 that all heads share (rotated or not, as the
model has it).  A cache is [pages, page_size, 576] bf16 or fp16: token rows (latent | positional part) dense within a page,
any page stride; page numbers outside the cache are holes whose tokens take no part.

    latent_append(latent, k_pe, cache, slots)                              # token rows into their pages
    rows = latent_gather(cache, block_table, cu_seqlens, out)              # and back, dense
    o = latent_prefill(q, k, v, k_pe, cu_seqlens_q, cu_seqlens_k)          # expanded form, packed sequences
    o = latent_decode(q_latent, q_pe, cache, block_table, seq_lens)        # absorbed form, S tokens a sequence
    o = latent_decode(..., prefix_table=pages, prefix_len=n)               # the same behind one shared prefix

The expanded form takes keys and values as the up-projection leaves them (views with any token and head stride), the
absorbed form queries that carry the key up-projection, and returns outputs in the latent space.  The default scale is
192^-1/2 for both.  Lengths and tables stay on the device: nothing is read back, so every call can be captured in a HIP
graph and replayed with other lengths, tables and data.

Errors: TypeError for a wrong dtype or device, ValueError for a wrong shape or stride.
"""
from __future__ import annotations

import ctypes
import struct

import torch

from . import _lib
from .recurrent import _need

LATENT, PE, HEAD = 512, 64, 128
ROW = LATENT + PE
SCALE = (HEAD + PE) ** -0.5
_DTYPES = {torch.bfloat16: 0, torch.float16: 1}
_cus = {}


# A decode step makes dozens of these calls, each of a few microseconds on the GPU.  What the checks look at (types, devices,
# shapes, strides) comes back call after call, so every entry keeps what it found for it: the checked sizes and strides, packed as
# the C struct's bytes.  The addresses are the call's own.  (Host time of a call whose sizes were not there before: latent_prefill
# 18 us instead of 12, latent_append 9.7 instead of 5.1, latent_gather 8.8 instead of 5.0.)
_MOST = 4096  # kept at a time, per entry


def _keep(seen, key, plan):
    if len(seen) >= _MOST:
        seen.clear()
    seen[key] = plan
    return plan


_raw_stream = torch._C._cuda_getCurrentRawStream  # the handle alone: current_stream() builds an object (2 us)


def _stream(device):
    return _raw_stream(device.index)


def _num_cus(device):
    n = _cus.get(device)
    if n is None:
        n = _cus[device] = torch.cuda.get_device_properties(device).multi_processor_count
    return n


def _first(name, t):
    """(device, dtype) of the tensor that the others have to match."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"kda355: {name} must be a tensor")
    if t.dtype not in _DTYPES:
        raise TypeError(f"kda355: {name} must be bfloat16 or float16, got {t.dtype}")
    if t.device.type != "cuda":
        raise TypeError("kda355: tensors must be on a GPU")
    return t.device, t.dtype


def _rows(name, t, shape, dtype, device):
    """The tensor has this shape and a dense last dimension; returns its other strides."""
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.device != device:
        _need(name, t, dtype, device)
    if t.shape != shape:
        raise ValueError(f"kda355: {name} must be {list(shape)}, got {list(t.shape)}")
    st = t.stride()
    if st[-1] != 1:
        raise ValueError(f"kda355: the last dimension of {name} must be dense")
    # the stride of a dimension of one is never used: any value is valid there, odd ones too
    if len(st) == 3:
        return st[0] if shape[0] > 1 else 0, st[1] if shape[1] > 1 else 0
    return (st[0] if shape[0] > 1 else 0,)


def _index(name, t, shape, device, dtype=torch.int32):
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.device != device:
        _need(name, t, dtype, device)
    if t.shape != shape or not t.is_contiguous():
        raise ValueError(f"kda355: {name} must be a contiguous {dtype} {list(shape)} tensor, got {list(t.shape)}")


def _table(name, t, device):
    """Row stride of a [rows, width] int32 page table with dense rows."""
    if not isinstance(t, torch.Tensor) or t.dtype is not torch.int32 or t.device != device:
        _need(name, t, torch.int32, device)
    sh, st = t.shape, t.stride()
    if len(sh) != 2 or sh[1] < 1 or (sh[1] > 1 and st[1] != 1):
        raise ValueError(f"kda355: {name} must be [rows, width >= 1] with dense rows, got {list(sh)}")
    return st[0] if sh[0] > 1 else sh[1]


def _cache(cache, dtype, device):
    """(pages, page_size, page stride) of a cache."""
    if not isinstance(cache, torch.Tensor) or cache.dtype is not dtype or cache.device != device:
        _need("cache", cache, dtype, device)
    sh, st = cache.shape, cache.stride()
    if len(sh) != 3 or sh[2] != ROW or sh[0] < 1 or sh[1] < 1:
        raise ValueError(f"kda355: cache must be [pages, page_size, {ROW}], got {list(sh)}")
    pages, size, _ = sh
    if st[2] != 1 or (size > 1 and st[1] != ROW):
        raise ValueError("kda355: cache must be dense within a page")
    return pages, size, st[0] if pages > 1 else size * ROW


def _workspace(need, workspace, device):
    """The caller's workspace or one from torch's allocator, kept by the call until its launch (None for none)."""
    if workspace is None:
        return torch.empty(need, dtype=torch.uint8, device=device) if need else None
    _need("workspace", workspace, torch.uint8, device)
    if not workspace.is_contiguous() or workspace.numel() < need:
        raise ValueError(f"kda355: workspace must be contiguous with >= {need} bytes")
    return workspace


def _bytes_needed(name, a):
    need = getattr(_lib.lib(), f"kda355_{name}_workspace_bytes")(ctypes.byref(a))
    if need < 0:
        _lib.check(int(need), name)
    return int(need)


def _sig(t):
    """What the checks look at of an optional argument."""
    return None if t is None else (t.shape, t.stride(), t.dtype, t.device)


_prefill_seen, _decode_seen, _append_seen, _gather_seen = {}, {}, {}, {}
_PTR2, _PTR7, _PTR8, _PTR10 = (struct.Struct(f"{n}Q") for n in (2, 7, 8, 10))


def _plan_prefill(q, k, v, k_pe, cu_q, cu_k, scale, causal, out, lse):
    """(device, dtype, out shape, bytes of workspace, struct bytes behind the pointers, those behind the workspace)."""
    dev, dt = _first("q", q)
    if q.dim() != 3 or q.shape[2] != HEAD + PE:
        raise ValueError(f"kda355: q must be [Tq, H, {HEAD + PE}], got {list(q.shape)}")
    Tq, H = q.shape[0], q.shape[1]
    Tk = k.shape[0] if isinstance(k, torch.Tensor) and k.dim() else 0
    strides = (_rows("q", q, (Tq, H, HEAD + PE), dt, dev) + _rows("k", k, (Tk, H, HEAD), dt, dev) +
               _rows("v", v, (Tk, H, HEAD), dt, dev) + _rows("k_pe", k_pe, (Tk, PE), dt, dev))
    N = cu_q.numel() - 1 if isinstance(cu_q, torch.Tensor) else 0
    if isinstance(cu_q, torch.Tensor) and N < 0:
        raise ValueError("kda355: cu_seqlens_q must have at least one entry")
    _index("cu_seqlens_q", cu_q, (N + 1,), dev)
    _index("cu_seqlens_k", cu_k, (N + 1,), dev)
    strides += (H * HEAD, HEAD) if out is None else _rows("out", out, (Tq, H, HEAD), dt, dev)
    if lse is not None:
        _index("lse", lse, (Tq, H), dev, torch.float32)
    a = _lib.KdaLatentPrefillArgs(*[None] * 8, *strides, Tq, Tk, None, 0, N, H, _DTYPES[dt], 1 if causal else 0,
                                  scale, _num_cus(dev))
    b, at = bytes(a), _lib.KdaLatentPrefillArgs.workspace.offset
    return dev, dt, (Tq, H, HEAD), _bytes_needed("latent_prefill", a), b[_PTR8.size:at], b[at + 16:]


def latent_prefill(q, k, v, k_pe, cu_seqlens_q, cu_seqlens_k, scale=None, causal=True, *, out=None, lse=None,
                   workspace=None):
    """The expanded form over packed sequences: q [Tq, H, 192] (128 | 64), k and v [Tk, H, 128], k_pe [Tk, 64] shared by the
    heads.  cu_seqlens_q / cu_seqlens_k int32 [N + 1] on the device; the queries are the last tokens of their sequences, so
    with `causal` query i of Lq sees keys j <= i + Lk - Lq.  Returns out [Tq, H, 128]; `lse` (fp32 [Tq, H]) receives the
    logarithms of the softmax sums, for joining with the attention over other keys.  A query that sees no key gets zeros and
    -inf, and keys it does not see never reach it, whatever they hold; rows of no sequence are not written.

    workspace: uint8 tensor of latent_prefill_workspace_bytes(...) (up to 136 MB); by default one is taken from torch's
    allocator for the call.  Calls that may overlap need workspaces of their own."""
    scale, causal = SCALE if scale is None else float(scale), bool(causal)  # (what is kept is keyed by their values)
    try:
        key = (q.shape, q.stride(), q.dtype, q.device, k.shape, k.stride(), k.dtype, k.device, v.shape, v.stride(), v.dtype,
               v.device, k_pe.shape, k_pe.stride(), k_pe.dtype, k_pe.device, cu_seqlens_q.shape, cu_seqlens_q.stride(),
               cu_seqlens_q.dtype, cu_seqlens_q.device, cu_seqlens_k.shape, cu_seqlens_k.stride(), cu_seqlens_k.dtype,
               cu_seqlens_k.device, scale, causal, _sig(out), _sig(lse))
        plan = _prefill_seen.get(key)
    except (AttributeError, TypeError):  # something that is no tensor: the checks say what
        key = plan = None
    if plan is None:
        plan = _keep(_prefill_seen, key, _plan_prefill(q, k, v, k_pe, cu_seqlens_q, cu_seqlens_k, scale, causal, out, lse))
    dev, dt, shape, need, mid, tail = plan
    if out is None:
        out = torch.empty_strided(shape, (shape[1] * shape[2], shape[2], 1), dtype=dt, device=dev)  # (0.4 us less than empty)
    ws = _workspace(need, workspace, dev)
    args = (_PTR8.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), k_pe.data_ptr(), out.data_ptr(),
                       0 if lse is None else lse.data_ptr(), cu_seqlens_q.data_ptr(), cu_seqlens_k.data_ptr()) + mid +
            _PTR2.pack(0 if ws is None else ws.data_ptr(), need) + tail)
    rc = _lib.LAUNCH["latent_prefill"](args, _stream(dev))
    if rc:
        _lib.check(rc, "latent_prefill")
    return out


def latent_prefill_workspace_bytes(N, H, Tq, Tk, *, num_cus=256):
    """Bytes of device workspace that latent_prefill() needs for these sizes (host only)."""
    return _bytes_needed("latent_prefill", _lib.KdaLatentPrefillArgs(N=N, H=H, Tq=Tq, Tk=Tk, num_cus=num_cus))


def _plan_decode(q_latent, q_pe, cache, block_table, seq_lens, scale, out, lse, prefix_table, prefix_len):
    """(device, dtype, out shape, bytes of workspace, struct bytes behind the pointers)."""
    dev, dt = _first("q_latent", q_latent)
    if q_latent.dim() != 3 or q_latent.shape[2] != LATENT:
        raise ValueError(f"kda355: q_latent must be [B * S, H, {LATENT}], got {list(q_latent.shape)}")
    T, H = q_latent.shape[0], q_latent.shape[1]
    strides = _rows("q_latent", q_latent, (T, H, LATENT), dt, dev) + _rows("q_pe", q_pe, (T, H, PE), dt, dev)
    pages, size, page_stride = _cache(cache, dt, dev)
    table_stride = _table("block_table", block_table, dev)
    B = block_table.shape[0]
    _index("seq_lens", seq_lens, (B,), dev)
    if T % B if B else T:
        raise ValueError(f"kda355: {T} rows of q_latent are not B x S for B = {B}")
    S = max(1, T // B) if B else 1
    if B and T < B:
        raise ValueError("kda355: q_latent must hold at least one token a sequence")
    width = 0
    if (prefix_table is None) != (prefix_len is None):
        raise ValueError("kda355: pass prefix_table and prefix_len together")
    if prefix_table is not None:
        width = prefix_table.numel() if isinstance(prefix_table, torch.Tensor) else 0
        _index("prefix_table", prefix_table, (max(1, width),), dev)
        _index("prefix_len", prefix_len, (1,), dev)
    strides += (H * LATENT, LATENT) if out is None else _rows("out", out, (T, H, LATENT), dt, dev)
    if lse is not None:
        _index("lse", lse, (T, H), dev, torch.float32)
    a = _lib.KdaLatentDecodeArgs(*[None] * 10, *strides, page_stride, pages, table_stride, 0, B, S, H, size, block_table.shape[1],
                                 width, _DTYPES[dt], _num_cus(dev), scale, 0)
    a.workspace_bytes = need = _bytes_needed("latent_decode", a)
    return dev, dt, (T, H, LATENT), need, bytes(a)[_PTR10.size:]


def latent_decode(q_latent, q_pe, cache, block_table, seq_lens, scale=None, *, out=None, lse=None, prefix_table=None,
                  prefix_len=None, workspace=None):
    """The absorbed form over the paged cache: q_latent [B * S, H, 512] and q_pe [B * S, H, 64], S tokens a sequence (row
    n * S + s), block_table int32 [B, width], seq_lens int32 [B] the cached tokens of each sequence, its S new ones among
    them (token s sees j < seq_lens[n] - (S - 1 - s)).  Returns out [B * S, H, 512] in the latent space; `lse` (fp32
    [B * S, H]) as in latent_prefill.

    prefix_table (int32 [width]) and prefix_len (int32 [1]) name the pages of a prefix that all B sequences share and see in
    front of their own tokens; it is read once for the whole batch.  block_table and seq_lens then hold what follows it.

    workspace: uint8 tensor of latent_decode_workspace_bytes(...) (17 MB for one sequence, 42 MB for 64 of 64 heads, 303 MB
    for 128 of 8 tokens and 128 heads); by default one is taken from torch's allocator for the call.  Calls that may overlap
    need workspaces of their own."""
    scale = SCALE if scale is None else float(scale)  # (what is kept is keyed by its value)
    try:
        key = (q_latent.shape, q_latent.stride(), q_latent.dtype, q_latent.device, q_pe.shape, q_pe.stride(), q_pe.dtype,
               q_pe.device, cache.shape, cache.stride(), cache.dtype, cache.device, block_table.shape, block_table.stride(),
               block_table.dtype, block_table.device, seq_lens.shape, seq_lens.stride(), seq_lens.dtype, seq_lens.device, scale,
               _sig(out), _sig(lse), _sig(prefix_table), _sig(prefix_len))
        plan = _decode_seen.get(key)
    except (AttributeError, TypeError):  # something that is no tensor: the checks say what
        key = plan = None
    if plan is None:
        plan = _keep(_decode_seen, key, _plan_decode(q_latent, q_pe, cache, block_table, seq_lens, scale, out, lse, prefix_table,
                                                     prefix_len))
    dev, dt, shape, need, tail = plan
    if out is None:
        out = torch.empty_strided(shape, (shape[1] * shape[2], shape[2], 1), dtype=dt, device=dev)  # (0.4 us less than empty)
    ws = _workspace(need, workspace, dev)
    args = (_PTR10.pack(q_latent.data_ptr(), q_pe.data_ptr(), cache.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(),
                        0 if prefix_table is None else prefix_table.data_ptr(),
                        0 if prefix_len is None else prefix_len.data_ptr(),
                        out.data_ptr(), 0 if lse is None else lse.data_ptr(), 0 if ws is None else ws.data_ptr()) + tail)
    rc = _lib.LAUNCH["latent_decode"](args, _stream(dev))
    if rc:
        _lib.check(rc, "latent_decode")
    return out


def latent_decode_workspace_bytes(B, S, H, page_size, table_width, prefix_width=0, *, num_cus=256):
    """Bytes of device workspace that latent_decode() needs for these sizes (host only)."""
    return _bytes_needed("latent_decode", _lib.KdaLatentDecodeArgs(B=B, S=S, H=H, page_size=page_size, table_width=table_width,
                                                                   prefix_width=prefix_width, num_cus=num_cus))


def latent_append(latent, k_pe, cache, slots):
    """cache row slots[t] (= page * page_size + offset, int64 [T]) <- latent [T, 512] | k_pe [T, 64]; slots outside the cache
    (padding: -1) are skipped.  The cache is written in place and returned."""
    try:
        key = (latent.shape, latent.stride(), latent.dtype, latent.device, k_pe.shape, k_pe.stride(), k_pe.dtype, k_pe.device,
               cache.shape, cache.stride(), cache.dtype, cache.device, slots.shape, slots.stride(), slots.dtype, slots.device)
        plan = _append_seen.get(key)
    except (AttributeError, TypeError):  # something that is no tensor: the checks say what
        key = plan = None
    if plan is None:
        dev, dt = _first("latent", latent)
        T = latent.shape[0] if latent.dim() else 0
        strides = _rows("latent", latent, (T, LATENT), dt, dev) + _rows("k_pe", k_pe, (T, PE), dt, dev)
        pages, size, page_stride = _cache(cache, dt, dev)
        _index("slots", slots, (T,), dev, torch.int64)
        a = _lib.KdaLatentTokensArgs(*[None] * 7, *strides, 0, page_stride, pages, 0, T, size, 0, 0, 0)
        plan = _keep(_append_seen, key, (dev, bytes(a)[_PTR7.size:]))
    dev, tail = plan
    args = _PTR7.pack(latent.data_ptr(), k_pe.data_ptr(), cache.data_ptr(), slots.data_ptr(), 0, 0, 0) + tail
    rc = _lib.LAUNCH["latent_append"](args, _stream(dev))
    if rc:
        _lib.check(rc, "latent_append")
    return cache


def latent_gather(cache, block_table, cu_seqlens, out):
    """out [T, 576] row cu_seqlens[n] + j <- token j of sequence n (block_table int32 [N, width], cu_seqlens int32 [N + 1] on
    the device); tokens in holes or past the table give zero rows, rows of `out` past the last sequence stay as they are."""
    try:
        key = (cache.shape, cache.stride(), cache.dtype, cache.device, block_table.shape, block_table.stride(), block_table.dtype,
               block_table.device, cu_seqlens.shape, cu_seqlens.stride(), cu_seqlens.dtype, cu_seqlens.device, out.shape,
               out.stride(), out.dtype, out.device)
        plan = _gather_seen.get(key)
    except (AttributeError, TypeError):  # something that is no tensor: the checks say what
        key = plan = None
    if plan is None:
        dev, dt = _first("cache", cache)
        pages, size, page_stride = _cache(cache, dt, dev)
        table_stride = _table("block_table", block_table, dev)
        N = block_table.shape[0]
        _index("cu_seqlens", cu_seqlens, (N + 1,), dev)
        T = out.shape[0] if isinstance(out, torch.Tensor) and out.dim() else 0
        o_st = _rows("out", out, (T, ROW), dt, dev)
        a = _lib.KdaLatentTokensArgs(*[None] * 7, 0, 0, *o_st, page_stride, pages, table_stride, T, size, block_table.shape[1], N,
                                     0)
        plan = _keep(_gather_seen, key, (dev, bytes(a)[_PTR7.size:]))
    dev, tail = plan
    args = _PTR7.pack(0, 0, cache.data_ptr(), 0, block_table.data_ptr(), cu_seqlens.data_ptr(), out.data_ptr()) + tail
    rc = _lib.LAUNCH["latent_gather"](args, _stream(dev))
    if rc:
        _lib.check(rc, "latent_gather")
    return out
