"""Pages of a cache (host side of kda355_{copy_rows, fork_pages, free_pages, compact_pages}_launch): sequences forked, freed
and compacted on the device, with the copies in every layer's pool.  No counterpart in the reference (its caller manages
slots on the host).

The bookkeeping is five int32 tensors that the caller keeps on the device:
    block_table [rows, width]   the pages of each sequence, in order; entries outside [0, pages) are holes
    seq_lens    [rows]          its tokens
    ref_counts  [pages]         how many sequences hold a page
    free_pages  [pages]         a stack of the pages nobody holds, the next one at its top; entries past it are -1
    num_free    [1]             its height
`pools` are the tensors that hold the pages' data, one per layer (latent caches, but also any [pages, ...] tensor with dense
rows): everything of a row is copied.  State rows of KDA layers are not paged: copy_rows() copies them for forked sequences.

Nothing is read back to the host, results do not depend on timing, and every call can be captured in a HIP graph.
Errors: TypeError for a wrong dtype or device, ValueError for a wrong shape or stride.
"""
from __future__ import annotations

import ctypes
import struct

import torch

from . import _lib
from .latent import _index, _stream, _table
from .recurrent import _need


def _pools(pools, slots=None):
    """(device, [(address, row bytes, slot stride, slots)]) of a list of [slots, ...] tensors with dense rows."""
    if isinstance(pools, torch.Tensor):
        pools = (pools,)
    out, dev = [], None
    for i, t in enumerate(pools):
        if not isinstance(t, torch.Tensor):
            raise TypeError("kda355: pools must be tensors")
        if dev is None:
            dev = t.device
        if t.device != dev or dev.type != "cuda":
            raise TypeError("kda355: pools must be on one GPU")
        sh = t.shape
        if len(sh) < 1 or (slots is not None and sh[0] != slots):
            raise ValueError(f"kda355: pool {i} must be [{slots if slots is not None else 'slots'}, ...], "
                             f"got {list(sh)}")
        n = sh[0]
        if n == 0:
            continue
        size = t.element_size()
        if t.is_contiguous():
            row = t.numel() // n * size
            stride = row
        else:
            st, exp = t.stride(), 1
            for d in range(len(sh) - 1, 0, -1):
                if sh[d] != 1 and st[d] != exp:
                    raise ValueError(f"kda355: the rows of pool {i} must be dense")
                exp *= sh[d]
            row = exp * size
            stride = st[0] * size if n > 1 else row
        if row == 0:
            continue
        out.append((t.data_ptr(), row, stride, n))
    return dev, out


# KdaPagesArgs in one go: its 24 pools would be as many objects
_PACK = struct.Struct(f"={4 * _lib.MAX_POOLS}q2i8Qq4i")
assert _PACK.size == ctypes.sizeof(_lib.KdaPagesArgs)
_NO_POOLS = (0,) * (4 * _lib.MAX_POOLS)


def _launch(name, dev, pools, n, src, dst, ws, table=0, lens=0, refs=0, free=0, num=0, stride=0, rows=0, width=0, pages=0,
            size=1):
    flat = _NO_POOLS
    if pools:
        flat = [v for p in pools for v in p]
        flat += _NO_POOLS[len(flat):]
    try:
        a = _lib.KdaPagesArgs.from_buffer_copy(
            _PACK.pack(*flat, len(pools), n, src, dst, table, lens, refs, free, num, ws, stride, rows, width, pages, size))
    except struct.error as e:
        raise ValueError(f"kda355: {name}: a size is out of range ({e})") from None
    _lib.check(_LAUNCH[name](ctypes.byref(a), _stream(dev)), name)


class _Entries(dict):
    def __missing__(self, name):
        f = self[name] = getattr(_lib.lib(), f"kda355_{name}_launch")
        return f


_LAUNCH = _Entries()


def _copy(dev, pools, n, src, dst):
    for i in range(0, len(pools), _lib.MAX_POOLS):
        _launch("copy_rows", dev, pools[i:i + _lib.MAX_POOLS], n, src, dst, 0)


def _book(block_table, ref_counts, free_pages, num_free):
    dev = block_table.device if isinstance(block_table, torch.Tensor) else None
    if dev is None or dev.type != "cuda":
        raise TypeError("kda355: block_table must be a tensor on a GPU")
    stride = _table("block_table", block_table, dev)
    pages = ref_counts.numel() if isinstance(ref_counts, torch.Tensor) else 0
    _index("ref_counts", ref_counts, (max(1, pages),), dev)
    _index("free_pages", free_pages, (pages,), dev)
    _index("num_free", num_free, (1,), dev)
    return dev, pages, dict(table=block_table.data_ptr(), refs=ref_counts.data_ptr(), free=free_pages.data_ptr(),
                            num=num_free.data_ptr(), stride=stride, rows=block_table.shape[0], width=block_table.shape[1],
                            pages=pages)


def copy_rows(pools, src, dst):
    """pool[dst[i]] <- pool[src[i]] in every pool of the list (int32 [n] rows; pairs with a row outside a pool are skipped
    there).  No dst may be another pair's src or dst."""
    dev, ps = _pools(pools)
    if dev is None:
        return
    n = src.numel() if isinstance(src, torch.Tensor) else 0
    _index("src", src, (n,), dev)
    _index("dst", dst, (n,), dev)
    _copy(dev, ps, n, src.data_ptr(), dst.data_ptr())


def fork_pages(pools, block_table, seq_lens, ref_counts, free_pages, num_free, parents, children, page_size):
    """Sequence children[i] becomes a copy of parents[i] (int32 [n] rows of block_table): full pages are shared, a part-filled
    last page is copied in every pool to a page from the stack.  Where the stack is empty the child gets length 0 and no
    pages.  What a child row held before is overwritten, not released (free_pages() first).  Pairs outside the table are
    skipped; children must differ from one another and from every parent."""
    dev, pages, book = _book(block_table, ref_counts, free_pages, num_free)
    _index("seq_lens", seq_lens, (block_table.shape[0],), dev)
    pool_dev, ps = _pools(pools, pages)
    if pool_dev is not None and pool_dev != dev:
        raise TypeError(f"kda355: pools must be on {dev}, got {pool_dev}")
    n = parents.numel() if isinstance(parents, torch.Tensor) else 0
    _index("parents", parents, (n,), dev)
    _index("children", children, (n,), dev)
    if n == 0:
        return
    ws = torch.empty(2 * n, dtype=torch.int32, device=dev)
    at = ws.data_ptr()
    first, rest = ps[:_lib.MAX_POOLS], ps[_lib.MAX_POOLS:]
    _launch("fork_pages", dev, first, n, parents.data_ptr(), children.data_ptr(), at, lens=seq_lens.data_ptr(),
            size=int(page_size), **book)
    _copy(dev, rest, n, at, at + 4 * n)


def free_pages(block_table, seq_lens, ref_counts, free_pages, num_free, rows, page_size):
    """The sequences rows[i] (int32 [n], all different) give up the pages of their tokens: their table rows become holes and
    their lengths 0; pages that nobody holds any more go onto the stack, the highest first (the lowest is taken next)."""
    dev, _, book = _book(block_table, ref_counts, free_pages, num_free)
    _index("seq_lens", seq_lens, (block_table.shape[0],), dev)
    n = rows.numel() if isinstance(rows, torch.Tensor) else 0
    _index("rows", rows, (n,), dev)
    _launch("free_pages", dev, [], n, rows.data_ptr(), 0, 0, lens=seq_lens.data_ptr(), size=int(page_size), **book)


def compact_pages(pools, block_table, ref_counts, free_pages, num_free):
    """Moves the held pages to the start of every pool: with L pages held, the i-th held page at or above L goes into the
    i-th free one below L.  block_table, ref_counts and the stack (L is taken next) follow.  Afterwards pages L and up hold
    nothing: the pools can be cut there."""
    dev, pages, book = _book(block_table, ref_counts, free_pages, num_free)
    pool_dev, ps = _pools(pools, pages)
    if pool_dev is not None and pool_dev != dev:
        raise TypeError(f"kda355: pools must be on {dev}, got {pool_dev}")
    ws = torch.empty(2 * pages + 2, dtype=torch.int32, device=dev)
    at = ws.data_ptr()
    _launch("compact_pages", dev, ps[:_lib.MAX_POOLS], 0, 0, 0, at, **book)
    half = pages // 2
    if half:
        _copy(dev, ps[_lib.MAX_POOLS:], half, at + 4 * pages, at + 4 * (pages + half))
