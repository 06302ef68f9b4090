"""Pages of a cache (host side of kda355_{copy_rows, fork_pages, free_pages, compact_pages, evict_tokens}_launch): sequences
forked, freed, compacted and cut to a budget of tokens on the device, with the copies in every layer's pool.  No counterpart in the reference (its caller manages
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
from .latent import _index, _keep, _table
from .recurrent import _need


def _sequence(pools):
    return pools if isinstance(pools, (list, tuple)) else (pools,) if isinstance(pools, torch.Tensor) else tuple(pools)


def _pools(pools, slots=None):
    """(device, [(row bytes, slot stride, slots)]) of a list of [slots, ...] tensors with dense rows; None for an empty one."""
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
        if t.numel() == 0:
            out.append(None)
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
        out.append((row, stride, n))
    return dev, out


# KdaPagesArgs in three pieces (its 24 pools would be as many objects): the pools that there are, zeros, what follows the pools
_POOLS = [struct.Struct(f"={4 * n}q") for n in range(_lib.MAX_POOLS + 1)]
_REST = [bytes(32 * (_lib.MAX_POOLS - n)) for n in range(_lib.MAX_POOLS + 1)]
_PACK = struct.Struct("=2i8Qq4i")
assert 32 * _lib.MAX_POOLS + _PACK.size == ctypes.sizeof(_lib.KdaPagesArgs)


# What was found right is kept by what the checks look at (latent.py): (device, pages, table stride, rows, width, page size,
# [(row bytes, slot stride, slots) of each pool])
_seen = {}


def _key(name, page_size, pools, tensors):
    return (name, page_size, tuple([(t.shape, t.stride(), t.dtype, t.device) for t in pools]),
            tuple([(t.shape, t.stride(), t.dtype, t.device) for t in tensors]))


def _launch(name, dev, pools, n, src, dst, ws, book=(0, 0, 0, 0, 0), stride=0, rows=0, width=0, pages=0, size=1):
    """`pools`: address, row bytes, slot stride and slots of one after the other; `book`: the addresses of the bookkeeping."""
    count = len(pools) // 4
    try:
        args = (_POOLS[count].pack(*pools) + _REST[count] +
                _PACK.pack(count, n, src, dst, *book, ws, stride, rows, width, pages, size))
    except struct.error as e:
        raise ValueError(f"kda355: {name}: a size is out of range ({e})") from None
    rc = _lib.launch(_lib.LAUNCH[name], args, dev)
    if rc:
        _lib.check(rc, name)


def _addresses(pools, found):
    """The flat list of _launch() for pools that were found right (empty ones have no entry)."""
    out = []
    for t, p in zip(pools, found):
        if p is not None:
            out += (t.data_ptr(), *p)
    return out


def _copy(dev, flat, n, src, dst):
    for i in range(0, len(flat), 4 * _lib.MAX_POOLS):
        _launch("copy_rows", dev, flat[i:i + 4 * _lib.MAX_POOLS], n, src, dst, 0)


def _book(block_table, ref_counts, free_pages, num_free):
    """(device, pages, table stride, rows, width)"""
    dev = block_table.device if isinstance(block_table, torch.Tensor) else None
    if dev is None or dev.type != "cuda":
        raise TypeError("kda355: block_table must be a tensor on a GPU")
    stride = _table("block_table", block_table, dev)
    pages = ref_counts.numel() if isinstance(ref_counts, torch.Tensor) else 0
    _index("ref_counts", ref_counts, (max(1, pages),), dev)
    _index("free_pages", free_pages, (pages,), dev)
    _index("num_free", num_free, (1,), dev)
    return dev, pages, stride, block_table.shape[0], block_table.shape[1]


def _check(name, page_size, pools, block_table, ref_counts, free_pages, num_free, seq_lens=None, **rows):
    """The checks of a bookkeeping call, or what they found for the like of it before."""
    page_size = int(page_size)  # (what is kept is keyed by its value)
    try:
        key = _key(name, page_size, pools, (block_table, ref_counts, free_pages, num_free, *rows.values()) +
                   (() if seq_lens is None else (seq_lens,)))
        plan = _seen.get(key)
    except (AttributeError, TypeError):  # something that is no tensor: the checks say what
        key = plan = None
    if plan is None:
        found = _book(block_table, ref_counts, free_pages, num_free)
        dev, pages = found[:2]
        if name != "compact_pages":
            _index("seq_lens", seq_lens, (found[3],), dev)
        pool_dev, ps = _pools(pools, pages)
        if pool_dev is not None and pool_dev != dev:
            raise TypeError(f"kda355: pools must be on {dev}, got {pool_dev}")
        n = None
        for what, t in rows.items():
            n = t.numel() if n is None and isinstance(t, torch.Tensor) else n or 0
            _index(what, t, (n,), dev)
        plan = _keep(_seen, key, found + (page_size, ps))
    return plan


def copy_rows(pools, src, dst):
    """pool[dst[i]] <- pool[src[i]] in every pool of the list (int32 [n] rows; pairs with a row outside a pool are skipped
    there).  No dst may be another pair's src or dst."""
    pools = _sequence(pools)
    dev, ps = _pools(pools)
    if dev is None:
        return
    n = src.numel() if isinstance(src, torch.Tensor) else 0
    _index("src", src, (n,), dev)
    _index("dst", dst, (n,), dev)
    _copy(dev, _addresses(pools, ps), n, src.data_ptr(), dst.data_ptr())


def fork_pages(pools, block_table, seq_lens, ref_counts, free_pages, num_free, parents, children, page_size):
    """Sequence children[i] becomes a copy of parents[i] (int32 [n] rows of block_table): full pages are shared, a part-filled
    last page is copied in every pool to a page from the stack.  Holes stay holes: a part-filled last page that is one takes no
    page.  Where the stack is empty the child gets length 0 and no pages.  What a child row held before is overwritten, not
    released (free_pages() first).  Pairs outside the table are skipped; children must differ from one another and from every
    parent."""
    pools = _sequence(pools)
    dev, pages, stride, rows, width, size, ps = _check(
        "fork_pages", page_size, pools, block_table, ref_counts, free_pages, num_free, seq_lens, parents=parents, children=children)
    n = parents.numel()
    if n == 0:
        return
    ws = torch.empty(2 * n, dtype=torch.int32, device=dev)
    at, flat = ws.data_ptr(), _addresses(pools, ps)
    most = 4 * _lib.MAX_POOLS
    _launch("fork_pages", dev, flat[:most], n, parents.data_ptr(), children.data_ptr(), at,
            (block_table.data_ptr(), seq_lens.data_ptr(), ref_counts.data_ptr(), free_pages.data_ptr(), num_free.data_ptr()),
            stride, rows, width, pages, size)
    if len(flat) > most:
        _copy(dev, flat[most:], n, at, at + 4 * n)


def free_pages(block_table, seq_lens, ref_counts, free_pages, num_free, rows, page_size):
    """The sequences rows[i] (int32 [n], all different) give up the pages of their tokens: their table rows become holes and
    their lengths 0; pages that nobody holds any more go onto the stack, the highest first (the lowest is taken next).

    Only the ceil(length / page_size) first entries of a row are given up.  Entries after them become holes without being given
    up, and their pages would stay counted as held: where pages are reserved ahead of the tokens, or tokens were taken back,
    raise the lengths to cover them first (seq_lens[rows] = width * page_size covers a whole row; holes in it are skipped)."""
    dev, pages, stride, count, width, size, _ = _check("free_pages", page_size, (), block_table, ref_counts, free_pages, num_free,
                                                       seq_lens, rows=rows)
    _launch("free_pages", dev, [], rows.numel(), rows.data_ptr(), 0, 0,
            (block_table.data_ptr(), seq_lens.data_ptr(), ref_counts.data_ptr(), free_pages.data_ptr(), num_free.data_ptr()),
            stride, count, width, pages, size)


def compact_pages(pools, block_table, ref_counts, free_pages, num_free):
    """Moves the held pages to the start of every pool: with L pages held, the i-th held page at or above L goes into the
    i-th free one below L.  block_table, ref_counts and the stack (L is taken next) follow.  Afterwards pages L and up hold
    nothing: the pools can be cut there.  Lists of pages kept elsewhere are not rewritten: keep the pages of a shared prefix as a
    row of block_table and pass that row to latent_decode."""
    pools = _sequence(pools)
    dev, pages, stride, rows, width, _, ps = _check("compact_pages", 1, pools, block_table, ref_counts, free_pages, num_free)
    ws = torch.empty(2 * pages + 2, dtype=torch.int32, device=dev)
    at, flat = ws.data_ptr(), _addresses(pools, ps)
    most = 4 * _lib.MAX_POOLS
    _launch("compact_pages", dev, flat[:most], 0, 0, 0, at,
            (block_table.data_ptr(), 0, ref_counts.data_ptr(), free_pages.data_ptr(), num_free.data_ptr()),
            stride, rows, width, pages)
    half = pages // 2
    if half and len(flat) > most:
        _copy(dev, flat[most:], half, at + 4 * pages, at + 4 * (pages + half))


_LAYER = struct.Struct("=5q")
_EVICT = struct.Struct("=2i7Q2q6iIi")
assert _LAYER.size * _lib.MAX_POOLS + _EVICT.size == ctypes.sizeof(_lib.KdaEvictArgs)


def _check_evict(pools, weights, block_table, seq_lens, ref_counts, free_pages, num_free, rows, keep, recent, page_size):
    """(device, table stride, rows, width, pages, [(token bytes, page stride, weights stride)], bytes of workspace of each call)"""
    for name, x in (("keep", keep), ("recent", recent), ("page_size", page_size)):
        if not -1 << 31 <= x < 1 << 31:  # (the struct would take the low 32 bits)
            raise ValueError(f"kda355: evict_tokens: {name}={x} does not fit in 32 bits")
    dev, pages, stride, count, width = _book(block_table, ref_counts, free_pages, num_free)
    _index("seq_lens", seq_lens, (count,), dev)
    n = rows.numel() if isinstance(rows, torch.Tensor) else 0
    _index("rows", rows, (n,), dev)
    if len(pools) != len(weights) or not pools:
        raise ValueError(f"kda355: {len(pools)} pools and {len(weights)} weights: one of each for every layer")
    pool_dev, found = _pools(pools, pages)
    if pool_dev != dev:
        raise TypeError(f"kda355: pools must be on {dev}, got {pool_dev}")
    layers = []
    for i, (t, p, w) in enumerate(zip(pools, found, weights)):
        if p is None or t.dim() < 2 or t.shape[1] != page_size:
            raise ValueError(f"kda355: pool {i} must be [pages, {page_size}, ...], got {list(t.shape)}")
        if not isinstance(w, torch.Tensor) or w.dtype is not torch.float32 or w.device != dev:
            _need(f"weights {i}", w, torch.float32, dev)
        sh, st = w.shape, w.stride()
        if len(sh) != 2 or sh[0] != count or sh[1] < width * page_size or (sh[1] > 1 and st[1] != 1):
            raise ValueError(f"kda355: weights {i} must be [{count}, >= {width * page_size}] with dense rows, got {list(sh)}")
        row = st[0] if count > 1 else sh[1]
        if row < sh[1]:
            raise ValueError(f"kda355: rows of weights {i} overlap")
        layers.append((p[0] // page_size, p[1], row))
    need = []
    for i in range(0, len(layers), _lib.MAX_POOLS):
        a = _lib.KdaEvictArgs(num_layers=len(layers[i:i + _lib.MAX_POOLS]), n=n, rows=count, table_width=width, pages=pages,
                              page_size=page_size, keep=keep, recent=recent)
        need.append(_lib.lib().kda355_evict_tokens_workspace_bytes(ctypes.byref(a)))
        if need[-1] < 0:
            _lib.check(int(need[-1]), "evict_tokens")
    return dev, stride, count, width, pages, layers, need


def evict_tokens(pools, weights, block_table, seq_lens, ref_counts, free_pages, num_free, rows, keep, recent, page_size):
    """Cuts the sequences rows[i] (int32 [n] rows of block_table) that are longer than `keep` tokens to `keep`, in every layer:
    pools[l] is [pages, page_size, ...] with token rows of a multiple of 16 bytes, weights[l] fp32 [rows, >= width * page_size]
    what latent_weights added up for the layer.

    The `recent` last tokens stay, and so do all up to the end of the sequence's last page that others hold too.  Of the tokens
    between, those with the largest weights of the layer stay, as many as make `keep` in all (ties: the lower index; a NaN is
    larger than any number).  With left = keep - recent, the i-th place below left whose token goes is filled by the i-th staying
    token from left on; the recent ones follow in order.  Layers choose on their own, so that place j is another token in each.
    Weights move along, and those of the places that became free are 0.  Pages behind the first ceil(keep / page_size) are given
    up as in free_pages; pages reserved ahead of the tokens move down in the table behind the kept ones.

    A sequence stays as it is where one of its pages is a hole, or where shared pages and recent tokens are more than `keep`.

    Afterwards seq_lens is the number of cached tokens and no longer the position of the next one: whoever rotates by
    positions keeps them elsewhere.  Draft tokens that may still be taken back have to be among the `recent`.  A table that spans
    more than recent + 16384 tokens takes the form for long sequences, whatever their lengths: 64 sequences of some 400
    tokens in 4 layers 18 us in a table of their size, 66 in one of 32768 tokens, 159 in one of 131072.

    Rows outside the table are skipped; a row that is given twice is taken once.  No two layers may have the same memory.  At most 65535
    rows; the workspace (up to some 160 MB, more only where one sequence's layers need it) comes from torch's allocator for the call."""
    pools, weights = _sequence(pools), _sequence(weights)
    keep, recent, page_size = int(keep), int(recent), int(page_size)  # (what is kept is keyed by their values)
    try:
        key = (keep, recent) + _key("evict_tokens", page_size, pools, (block_table, seq_lens, ref_counts, free_pages, num_free, rows, *weights))
        plan = _seen.get(key)
    except (AttributeError, TypeError):  # something that is no tensor: the checks say what
        key = plan = None
    if plan is None:
        plan = _keep(_seen, key, _check_evict(pools, weights, block_table, seq_lens, ref_counts, free_pages, num_free, rows, keep,
                                              recent, page_size))
    dev, stride, count, width, total, layers, need = plan
    n = rows.numel()
    if n == 0:
        return
    if len({t.data_ptr() for t in pools}) < len(pools) or len({w.data_ptr() for w in weights}) < len(weights):
        raise ValueError("kda355: evict_tokens: a pool or its weights are given twice: layers are cut at the same time")
    ws = torch.empty(max(need), dtype=torch.uint8, device=dev)
    books = (rows.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(), ref_counts.data_ptr(), free_pages.data_ptr(),
             num_free.data_ptr(), ws.data_ptr())
    for c, first in enumerate(range(0, len(layers), _lib.MAX_POOLS)):
        some = layers[first:first + _lib.MAX_POOLS]
        args = b"".join([_LAYER.pack(t.data_ptr(), y[0], y[1], w.data_ptr(), y[2])
                         for t, w, y in zip(pools[first:], weights[first:], some)])
        more = _lib.EVICT_MORE if first + len(some) < len(layers) else 0
        args += bytes(_LAYER.size * (_lib.MAX_POOLS - len(some))) + _EVICT.pack(
            len(some), n, *books, need[c], stride, count, width, total, page_size, keep, recent, more, 0)
        rc = _lib.launch(_lib.LAUNCH["evict_tokens"], args, dev)
        if rc:
            _lib.check(rc, "evict_tokens")
