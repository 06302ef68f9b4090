"""Pages of a cache on the GPU: bookkeeping exact against the plain Python form, page contents bit for bit."""
import random

import pytest
import torch

import kda355
from latent_ref import ROW, Book

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _bits(t):
    return t.view(torch.int16) if t.element_size() == 2 else t.view(torch.int32)


def _random(shape, dtype, seed):
    """Random bits, NaN patterns among them."""
    g = torch.Generator().manual_seed(seed)
    n = torch.int16 if dtype.itemsize == 2 else torch.int32
    return torch.randint(-(1 << 15), 1 << 15, shape, generator=g).to(n).view(dtype).to(DEV)


# ------------------------------------------------------------------------------------------------ token rows
@pytest.mark.parametrize("T,pages,size,dtype", [(1, 1, 1, torch.bfloat16), (7, 5, 3, torch.float16),
                                                (64, 40, 16, torch.bfloat16), (1000, 9, 272, torch.bfloat16)])
def test_append(T, pages, size, dtype):
    rng = random.Random(T)
    pool = _random((pages, size * ROW + 64), dtype, 1)
    cache = pool[:, :size * ROW].view(pages, size, ROW) if pages == 1 else pool.as_strided((pages, size, ROW),
                                                                                         (size * ROW + 64, ROW, 1))
    before = _bits(pool).cpu().clone()
    latent, pe = _random((T, 520), dtype, 2)[:, :512], _random((T, 640), dtype, 3)[:, 576:]
    slots = rng.sample(range(pages * size), min(T, pages * size))
    slots += [-1] * (T - len(slots))
    slots[0] = pages * size  # outside: skipped
    if T > 3:
        slots[1], slots[2] = -5, 1 << 40
    kda355.latent_append(latent, pe, cache, torch.tensor(slots, dtype=torch.int64, device=DEV))
    want = before
    rows = _bits(torch.cat([latent, pe], dim=1)).cpu()
    for t, s in enumerate(slots):
        if 0 <= s < pages * size:
            want[s // size, (s % size) * ROW:(s % size + 1) * ROW] = rows[t]
    assert torch.equal(_bits(pool).cpu(), want)


@pytest.mark.parametrize("lens,size,dtype", [([1], 1, torch.bfloat16), ([5, 0, 17, 1], 16, torch.float16),
                                             ([300, 64, 63, 65], 64, torch.bfloat16), ([0, 0], 4, torch.bfloat16)])
def test_gather(lens, size, dtype):
    width = max(1, max(-(-n // size) for n in lens)) + 1
    pages = width * len(lens) + 3
    cache = _random((pages, size, ROW), dtype, 4)
    g = torch.Generator().manual_seed(5)
    table = torch.randperm(pages, generator=g)[:width * len(lens)].view(len(lens), width).int()
    table[0, 0] = pages  # a hole
    lens = list(lens)
    lens[-1] += size * width  # runs past the table
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    out = _random((cu[-1] + 3, ROW + 8), dtype, 6)
    want = _bits(out).cpu().clone()
    bits = _bits(cache).cpu()
    for n, length in enumerate(lens):
        for j in range(length):
            p = int(table[n, j // size]) if j // size < width else -1
            want[cu[n] + j, :ROW] = bits[p, j % size] if 0 <= p < pages else 0
    kda355.latent_gather(cache, table.to(DEV), _i32(cu), out[:, :ROW])
    assert torch.equal(_bits(out).cpu(), want)


# ------------------------------------------------------------------------------------------------ rows
@pytest.mark.parametrize("pools", [1, 3, 30])
def test_copy_rows(pools):
    ts = []
    for i in range(pools):
        slots = 6 + i % 3
        t = _random((slots, 3, 8 * (1 + 5 * i) + 2000 * (i == 2)), torch.bfloat16 if i % 2 else torch.float32, i)
        if i % 4 == 1:  # rows a stride apart
            wide = _random((slots, 3 * t.shape[2] + 16), t.dtype, 100 + i)
            t = wide.as_strided(t.shape, (wide.shape[1], t.shape[2], 1))
        ts.append(t)
    want = [_bits(t.contiguous()).cpu().clone() for t in ts]
    src, dst = [0, 1, -1, 7, 2, 5], [3, 4, 5, 2, 100, 5]
    for w in want:
        old = w.clone()
        for s, d in zip(src, dst):
            if 0 <= s < len(w) and 0 <= d < len(w):
                w[d] = old[s]
    kda355.copy_rows(ts, _i32(src), _i32(dst))
    for t, w in zip(ts, want):
        assert torch.equal(_bits(t.contiguous()).cpu(), w)


def _make(rng, rows, width, size, pages, live, dtype=torch.bfloat16, layers=2):
    """A bookkeeping state: `live` random pages over random rows, some of them shared."""
    perm = list(range(pages))
    rng.shuffle(perm)
    used, free = perm[:live], perm[live:]
    table, lens = [[-1] * width for _ in range(rows)], [0] * rows
    for r in range(rows):
        n = rng.randrange(width + 1)
        own = [used.pop() for _ in range(min(n, len(used)))]
        if own and r and rng.random() < 0.5:
            own[0] = next((g for g in table[r - 1] if g >= 0), own[0])
        table[r][:len(own)] = own
        lens[r] = max(0, len(own) * size - rng.randrange(size)) if own else 0
    refs = [0] * pages
    for row in table:
        for g in row:
            if g >= 0:
                refs[g] += 1
    free = [p for p in range(pages) if refs[p] == 0]
    rng.shuffle(free)
    stack = free + [-1] * (pages - len(free))
    pools = [_random((pages, size, ROW), dtype, 50 + i) for i in range(layers)]
    return Book(table, lens, refs, stack, len(free), size), pools


class _Device:
    def __init__(self, book, pad=3):
        rows, width = len(book.table), len(book.table[0])
        self.wide = torch.full((rows, width + pad), 77, dtype=torch.int32, device=DEV)
        self.table = self.wide[:, :width]
        self.table.copy_(_i32(book.table))
        self.lens, self.refs, self.free, self.num = _i32(book.lens), _i32(book.refs), _i32(book.free), _i32([book.num])

    def same(self, book):
        assert self.table.tolist() == book.table
        assert self.refs.tolist() == book.refs
        assert self.free.tolist() == book.free
        assert self.num.tolist() == [book.num]
        assert (self.wide[:, self.table.shape[1]:] == 77).all()


def _contents(pools, before, moves):
    for t, b in zip(pools, before):
        want = b.clone()
        for s, d in moves:
            want[d] = b[s]
        assert torch.equal(_bits(t).cpu(), want)


@pytest.mark.parametrize("n,size,layers,seed", [(1, 1, 1, 0), (3, 16, 2, 1), (20, 5, 2, 2), (40, 16, 26, 3),
                                                (1500, 3, 1, 4), (5, 64, 0, 5)])
def test_fork(n, size, layers, seed):
    rng = random.Random(seed)
    rows = 6 + n + 2
    book, pools = _make(rng, rows, 7, size, 200 + n // 2, 40, layers=layers)
    for r in range(6, rows):  # the children's rows: whatever they hold is overwritten
        for g in book.table[r]:
            if g >= 0:
                book.refs[g] -= 1
        book.table[r], book.lens[r] = [rng.choice([-1, 3, 999])] * 7, rng.randrange(50)
    book.lens[1] = 10 ** 6  # past the table
    if n > 4:
        book.table[2][0] = 10 ** 6  # a hole in a shared part
    d = _Device(book)
    before = [_bits(t).cpu().clone() for t in pools]
    parents = [rng.randrange(6) for _ in range(n)]
    children = list(range(6, 6 + n))
    if n > 2:
        parents[1], children[2] = -1, rows  # skipped
    kda355.fork_pages(pools, d.table, d.lens, d.refs, d.free, d.num, _i32(parents), _i32(children), size)
    book.fork(parents, children)
    d.same(book)
    assert d.lens.tolist() == book.lens
    _contents(pools, before, book.moves)


def test_fork_without_free_pages():
    """The stack runs dry in the middle of a call: the later children that need a page get nothing, the others live."""
    book = Book([[0, 1], [2, 3]] + [[-1, -1]] * 6, [20, 32, 0, 0, 0, 0, 0, 0], [1, 1, 1, 1, 0, 0], [5, 4, -1, -1, -1, -1], 2, 16)
    d = _Device(book)
    pools = [_random((6, 16, ROW), torch.float16, 9)]
    before = [_bits(t).cpu().clone() for t in pools]
    parents, children = [0, 1, 0, 0, 1, 0], [2, 3, 4, 5, 6, 7]
    kda355.fork_pages(pools, d.table, d.lens, d.refs, d.free, d.num, _i32(parents), _i32(children), 16)
    book.fork(parents, children)
    assert book.lens[5] == 0 and book.lens[6] == 32 and book.num == 0
    d.same(book)
    assert d.lens.tolist() == book.lens
    _contents(pools, before, book.moves)


@pytest.mark.parametrize("rows,width,pages,live,seed", [(1, 1, 1, 1, 0), (8, 5, 60, 30, 1), (70, 9, 5000, 500, 2),
                                                        (300, 40, 9000, 8000, 3)])
def test_free(rows, width, pages, live, seed):
    rng = random.Random(seed)
    book, _ = _make(rng, rows, width, 16, pages, live, layers=0)
    if rows > 4:
        book.lens[2] = 0          # holds pages that its length does not cover
        book.table[3][0] = -7     # a hole
        book.lens[4] = 10 ** 7
    d = _Device(book)
    which = rng.sample(range(rows), max(1, rows * 2 // 3)) + ([-1, rows] if rows > 4 else [])
    kda355.free_pages(d.table, d.lens, d.refs, d.free, d.num, _i32(which), 16)
    book.release(which)
    d.same(book)
    assert d.lens.tolist() == book.lens


def test_free_few_of_many_pages():
    rng = random.Random(7)
    book, _ = _make(rng, 8, 5, 16, 40000, 30, layers=0)
    d = _Device(book)
    kda355.free_pages(d.table, d.lens, d.refs, d.free, d.num, _i32([1, 6, 3]), 16)
    book.release([1, 6, 3])
    d.same(book)


@pytest.mark.parametrize("rows,size", [(20, 4), (300, 4)])
@pytest.mark.parametrize("extra", [0, 1, 200])
def test_free_shared_by_many(rows, size, extra):
    """Pages that all sequences share, given up by all of them or by all but `extra`; a page whose count is too low by two and
    by all but one is freed once."""
    width, pages = 20, 64
    extra = min(extra, rows - 1)
    table = [[5, 9, 40, 41] + [-1] * 16 for _ in range(rows)]
    refs = [0] * pages
    for p in (5, 9):
        refs[p] = rows
    refs[40], refs[41] = rows - 2, 1
    free = [p for p in range(pages) if refs[p] == 0]
    book = Book(table, [4 * size - 1] * rows, refs, free + [-1] * (pages - len(free)), len(free), size)
    d = _Device(book)
    which = list(range(extra, rows))
    kda355.free_pages(d.table, d.lens, d.refs, d.free, d.num, _i32(which), size)
    book.release(which)
    d.same(book)
    assert d.lens.tolist() == book.lens


@pytest.mark.parametrize("rows,width,pages,live,layers,seed", [(1, 1, 1, 1, 1, 0), (1, 1, 1, 0, 1, 0), (8, 5, 61, 30, 2, 1),
                                                               (20, 9, 300, 170, 27, 2), (300, 40, 9000, 6000, 0, 3),
                                                               (4, 3, 2, 1, 1, 4)])
def test_compact(rows, width, pages, live, layers, seed):
    rng = random.Random(seed)
    book, pools = _make(rng, rows, width, 4, pages, live, layers=layers)
    if rows > 4:
        book.table[2][-1] = pages + 5  # holes stay as they are
    d = _Device(book)
    before = [_bits(t).cpu().clone() for t in pools]
    kda355.compact_pages(pools, d.table, d.refs, d.free, d.num)
    book.compact()
    d.same(book)
    _contents(pools, before, book.moves)
    kda355.compact_pages(pools, d.table, d.refs, d.free, d.num)  # a compact pool stays as it is
    d.same(book)
    _contents(pools, before, book.moves)


def test_fork_free_compact_captured():
    """A step of drop, fork and compact recorded once and replayed, against the plain form, with eager work between."""
    rng = random.Random(11)
    book, pools = _make(rng, 12, 6, 8, 80, 40)
    for r in range(8, 12):
        for g in book.table[r]:
            if g >= 0:
                book.refs[g] -= 1
        book.table[r], book.lens[r] = [-1] * 6, 0
    book.free = [p for p in range(80) if book.refs[p] == 0]
    book.num = len(book.free)
    book.free += [-1] * (80 - book.num)
    d = _Device(book)
    parents, children = _i32([0, 1, 2, 3]), _i32([8, 9, 10, 11])

    def step():
        kda355.free_pages(d.table, d.lens, d.refs, d.free, d.num, children, 8)
        kda355.fork_pages(pools, d.table, d.lens, d.refs, d.free, d.num, parents, children, 8)
        kda355.compact_pages(pools, d.table, d.refs, d.free, d.num)

    def plain():
        book.release(children.tolist())
        book.fork(parents.tolist(), children.tolist())
        book.compact()

    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()  # the first pass outside the capture
    torch.cuda.current_stream().wait_stream(side)
    plain()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        parents.copy_(_i32([i, (i + 3) % 8, (i + 5) % 8, 0]))
        graph.replay()
        torch.cuda.synchronize()
        plain()
        d.same(book)
        (torch.randn(64, 64, device=DEV) @ torch.randn(64, 64, device=DEV)).sum().item()


def test_page_refusals():
    book, pools = _make(random.Random(1), 4, 3, 4, 20, 5)
    d = _Device(book, pad=0)
    one = _i32([0])
    with pytest.raises(ValueError):
        kda355.fork_pages([pools[0][:10]], d.table, d.lens, d.refs, d.free, d.num, one, one, 4)
    with pytest.raises(ValueError):
        kda355.fork_pages(pools, d.table, d.lens, d.refs, d.free, d.num, one, _i32([1, 2]), 4)
    with pytest.raises(ValueError):
        kda355.fork_pages(pools, d.table, d.lens, d.refs, d.free[:5], d.num, one, one, 4)
    with pytest.raises(ValueError):
        kda355.fork_pages(pools, d.table, d.lens, d.refs, d.free, d.num, one, one, 0)
    with pytest.raises(TypeError):
        kda355.free_pages(d.table, d.lens.long(), d.refs, d.free, d.num, one, 4)
    with pytest.raises(TypeError):
        kda355.free_pages(d.table, d.lens, d.refs, d.free, d.num, one.cpu(), 4)
    with pytest.raises(ValueError):
        kda355.compact_pages([pools[0].transpose(1, 2)], d.table, d.refs, d.free, d.num)
    with pytest.raises(ValueError):
        kda355.copy_rows([torch.zeros(4, 3, device=DEV)], one, one)  # rows of 12 bytes
    with pytest.raises(TypeError):
        kda355.copy_rows([pools[0], torch.zeros(4, 8)], one, one)
    with pytest.raises(ValueError):
        kda355.latent_append(torch.zeros(2, 511, device=DEV).bfloat16(), torch.zeros(2, 64, device=DEV).bfloat16(), pools[0],
                             torch.zeros(2, dtype=torch.int64, device=DEV))
    with pytest.raises(TypeError):
        kda355.latent_append(torch.zeros(2, 512, device=DEV).half(), torch.zeros(2, 64, device=DEV).half(), pools[0],
                             torch.zeros(2, dtype=torch.int64, device=DEV))
    with pytest.raises(TypeError):
        kda355.latent_gather(pools[0], d.table.long(), _i32([0] * 5), torch.zeros(1, ROW, device=DEV).bfloat16())
    with pytest.raises(ValueError):
        kda355.latent_gather(pools[0], d.table, _i32([0] * 4), torch.zeros(1, ROW, device=DEV).bfloat16())


def test_refused_after_a_like_call_was_taken():
    """What a call of the same shapes had found right does not let another one through."""
    book, pools = _make(random.Random(1), 4, 3, 4, 20, 5)
    d = _Device(book, pad=0)
    one, cache = _i32([0]), pools[0]
    lat, pe, slots = _random((2, 512), torch.bfloat16, 1), _random((2, 64), torch.bfloat16, 2), torch.tensor([0, 1], device=DEV)
    out = torch.empty(4, ROW, dtype=torch.bfloat16, device=DEV)
    for _ in range(2):
        kda355.free_pages(d.table, d.lens, d.refs, d.free, d.num, one, 4)
        kda355.latent_append(lat, pe, cache, slots)
        kda355.latent_gather(cache, d.table, _i32([0, 1, 2, 3, 4]), out)
    for size in (0, -1, 1 << 31):
        with pytest.raises(ValueError):
            kda355.free_pages(d.table, d.lens, d.refs, d.free, d.num, one, size)
    for bad in (dict(latent=lat.half()), dict(k_pe=pe.float()), dict(slots=slots.int()), dict(cache=cache.cpu())):
        with pytest.raises(TypeError):
            kda355.latent_append(**{**dict(latent=lat, k_pe=pe, cache=cache, slots=slots), **bad})
    with pytest.raises(ValueError):
        kda355.latent_append(lat, pe, cache, slots[:1])
    with pytest.raises(ValueError):  # the same shape, 2 bytes off
        kda355.latent_append(_random((1026,), torch.bfloat16, 1)[1:1025].view(2, 512), pe, cache, slots)
    with pytest.raises(TypeError):
        kda355.latent_gather(cache, d.table, torch.zeros(5, dtype=torch.int64, device=DEV), out)


@pytest.mark.parametrize("hole", [-1, -7, 6, 10 ** 6])
def test_fork_with_a_hole_as_last_page(hole):
    """A part-filled last page outside the pool: the child has a hole there too and no page is taken for it, so that the
    child sees what its parent sees, and not what some page's last owner left."""
    size, pages = 16, 6
    d = _Device(Book([[0, hole, -1], [2, 3, -1], [9, 9, 9], [9, 9, 9], [9, 9, 9]], [20, 24, 5, 5, 5], [1, 0, 1, 1, 0, 0],
                     [5, 4, 1, -1, -1, -1], 3, size))
    pools = [_random((pages, size, ROW), torch.bfloat16, 60 + i) for i in range(2)]
    pools[0][:] = torch.randn(pages, size, ROW, generator=torch.Generator().manual_seed(5)).to(torch.bfloat16)
    before = [_bits(t).cpu().clone() for t in pools]
    kda355.fork_pages(pools, d.table, d.lens, d.refs, d.free, d.num, _i32([0, 1, 0]), _i32([2, 3, 4]), size)
    assert d.table.tolist() == [[0, hole, -1], [2, 3, -1], [0, -1, -1], [2, 1, -1], [0, -1, -1]]
    assert d.lens.tolist() == [20, 24, 20, 24, 20]
    assert d.refs.tolist() == [3, 1, 2, 1, 0, 0]
    assert d.free.tolist() == [5, 4, -1, -1, -1, -1] and d.num.tolist() == [2]
    _contents(pools, before, [(3, 1)])
    g = torch.Generator().manual_seed(6)
    ql, qp = (torch.randn(1, 4, n, generator=g).to(torch.bfloat16).to(DEV) for n in (512, 64))
    seen = [kda355.latent_decode(ql, qp, pools[0], d.table[r:r + 1].contiguous(), d.lens[r:r + 1].contiguous()) for r in range(5)]
    assert torch.isfinite(seen[0]).all()
    for parent, child in ((0, 2), (1, 3), (0, 4)):
        assert torch.equal(seen[parent], seen[child])


def test_fork_holes_do_not_use_up_the_stack():
    """Two pages left, three forks that need one among four whose last page is a hole: the pages go to the first two."""
    size = 8
    book = Book([[0, 1], [2, -1]] + [[-1, -1]] * 7, [12, 12] + [0] * 7, [1, 1, 1, 0, 0], [4, 3, -1, -1, -1], 2, size)
    d = _Device(book)
    pools = [_random((5, size, ROW), torch.float16, 70)]
    before = [_bits(t).cpu().clone() for t in pools]
    kda355.fork_pages(pools, d.table, d.lens, d.refs, d.free, d.num, _i32([1, 0, 1, 1, 0, 0, 1]), _i32([2, 3, 4, 5, 6, 7, 8]), size)
    assert d.table.tolist()[2:] == [[2, -1], [0, 3], [2, -1], [2, -1], [0, 4], [-1, -1], [2, -1]]
    assert d.lens.tolist()[2:] == [12, 12, 12, 12, 12, 0, 12]
    assert d.refs.tolist() == [3, 1, 5, 1, 1] and d.free.tolist() == [-1] * 5 and d.num.tolist() == [0]
    _contents(pools, before, [(1, 3), (1, 4)])


def test_a_page_size_that_is_written_again_counts_anew():
    """A page size may be given as anything that int() takes: its value at the call is the one that counts, and nothing that
    is kept from one call for the next holds on to it."""
    size = torch.tensor(4)
    for value in (4, 8, 4):
        size.fill_(value)
        book, pools = _make(random.Random(12), 6, 5, value, 30, 12)
        book.table[4], book.lens[4], book.table[5], book.lens[5] = [-1] * 5, 0, [-1] * 5, 0
        pools = [_random((30, 8, ROW), torch.bfloat16, 80)]  # (the same shape for either size)
        before = [_bits(t).cpu().clone() for t in pools]
        d = _Device(book)
        kda355.fork_pages(pools, d.table, d.lens, d.refs, d.free, d.num, _i32([0, 1]), _i32([4, 5]), size)
        book.fork([0, 1], [4, 5])
        d.same(book)
        _contents(pools, before, book.moves)
        kda355.free_pages(d.table, d.lens, d.refs, d.free, d.num, _i32([1, 2]), size)
        book.release([1, 2])
        d.same(book)
        assert d.lens.tolist() == book.lens
    assert not any(isinstance(part, torch.Tensor) for key in kda355.pages._seen for part in key)


def test_captured_steps_move_the_contents():
    """A step of drop, fork and compact recorded once and replayed: after every replay the pages hold what the plain form's
    moves leave, bit for bit, and the lengths agree."""
    rng = random.Random(13)
    book, pools = _make(rng, 12, 6, 8, 80, 40)
    for r in range(8, 12):
        for g in book.table[r]:
            if g >= 0:
                book.refs[g] -= 1
        book.table[r], book.lens[r] = [-1] * 6, 0
    book.free = [p for p in range(80) if book.refs[p] == 0]
    book.num = len(book.free)
    book.free += [-1] * (80 - book.num)
    d = _Device(book)
    parents, children = _i32([0, 1, 2, 3]), _i32([8, 9, 10, 11])
    want = [_bits(t).cpu().clone() for t in pools]

    def step():
        kda355.free_pages(d.table, d.lens, d.refs, d.free, d.num, children, 8)
        kda355.fork_pages(pools, d.table, d.lens, d.refs, d.free, d.num, parents, children, 8)
        kda355.compact_pages(pools, d.table, d.refs, d.free, d.num)

    def compare(what):
        book.moves = []
        book.release(children.tolist())
        book.fork(parents.tolist(), children.tolist())
        book.compact()
        for w in want:
            for s, t in book.moves:
                w[t] = w[s]
        d.same(book)
        assert d.lens.tolist() == book.lens, what
        for t, w in zip(pools, want):
            assert torch.equal(_bits(t).cpu(), w), what
        return len(book.moves)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()  # the first pass outside the capture
    torch.cuda.current_stream().wait_stream(side)
    moved = compare("eager")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(5):
        parents.copy_(_i32([(i + 1) % 8, (i + 3) % 8, (i + 6) % 8, 2]))
        graph.replay()
        torch.cuda.synchronize()
        moved += compare(f"replay {i}")
        (torch.randn(64, 64, device=DEV) @ torch.randn(64, 64, device=DEV)).sum().item()
    assert moved > 12  # (forks of part-filled pages and moved pages in more than one replay)


@pytest.mark.parametrize("rows,width,pages", [(6, 5, 60), (70, 9, 5000), (300, 40, 9000)])
def test_free_gives_up_reserved_pages_that_the_length_covers(rows, width, pages):
    """Pages reserved past a sequence's tokens are given up with it when its length is raised to cover them first."""
    rng = random.Random(rows)
    size = 16
    perm = list(range(pages))
    rng.shuffle(perm)
    table, lens, refs = [], [], [0] * pages
    for r in range(rows):
        n = rng.randrange(1, width + 1)
        own = [perm.pop() for _ in range(n)]
        for g in own:
            refs[g] = 1
        table.append(own + [-1] * (width - n))
        lens.append(rng.randrange(n * size + 1))  # anything from no token to all pages full
    free = [p for p in range(pages) if not refs[p]]
    d = _Device(Book(table, lens, refs, free + [-1] * (pages - len(free)), len(free), size))
    which = _i32(list(range(rows)))
    d.lens[which.long()] = width * size
    kda355.free_pages(d.table, d.lens, d.refs, d.free, d.num, which, size)
    assert (d.table == -1).all() and (d.lens == 0).all() and (d.refs == 0).all()
    assert d.num.tolist() == [pages] and sorted(d.free.tolist()) == list(range(pages))
