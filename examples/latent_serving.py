"""One latent attention layer of a hybrid model through a serving day in miniature: prompts over a paged cache (expanded form),
parallel samples forked from them, a step of new tokens (absorbed form), samples dropped, the pool compacted, a batch behind a
shared document.  Prints how far the two forms of the layer are apart at every stage.

    python examples/latent_serving.py            (needs an MI355X and the built library)
"""
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "eat-kernels_amd"))

import kda355  # noqa: E402

DEV, DT = "cuda", torch.bfloat16
HEADS, LAT, PE, HEAD, PAGE = 16, 512, 64, 128, 64


def _int32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


class Layer:
    """The up-projections of the layer: keys and values of a head from the latent vector.  The absorbed form multiplies the
    queries by the keys' part, and its output by the values'."""

    def __init__(self, gen):
        self.k = torch.randn(HEADS, LAT, HEAD, generator=gen, device=DEV) * LAT ** -0.5
        self.v = torch.randn(HEADS, LAT, HEAD, generator=gen, device=DEV) * LAT ** -0.5

    def expand(self, rows):
        """[T, 576] cache rows -> keys and values [T, H, 128], the shared part [T, 64]"""
        latent = rows[:, :LAT].float()
        heads = [torch.cat([latent @ self.k[h], latent @ self.v[h]], dim=-1) for h in range(HEADS)]
        kv = torch.stack(heads, dim=1).to(DT)
        return kv[..., :HEAD], kv[..., HEAD:], rows[:, LAT:]

    def absorb(self, q):
        """[T, H, 192] queries -> [T, H, 512] in the latent space, [T, H, 64]"""
        lat = torch.stack([q[:, h, :HEAD].float() @ self.k[h].t() for h in range(HEADS)], dim=1)
        return lat.to(DT), q[..., HEAD:]

    def values(self, o):
        """[T, H, 512] outputs of the absorbed form -> [T, H, 128]"""
        return torch.stack([o[:, h].float() @ self.v[h] for h in range(HEADS)], dim=1)


def expanded(layer, cache, table, lens, q, new):
    """The expanded form of the last `new` tokens of every sequence over its whole cached history."""
    cu_k = _int32([0] + torch.tensor(lens).cumsum(0).tolist())
    rows = kda355.latent_gather(cache, table, cu_k, torch.empty(sum(lens), LAT + PE, dtype=DT, device=DEV))
    k, v, pe = layer.expand(rows)
    cu_q = _int32([0] + torch.tensor(new).cumsum(0).tolist())
    return kda355.latent_prefill(q, k, v, pe, cu_q, cu_k)


def apart(a, b):
    """Largest difference over the RMS of the first."""
    return float((a.float() - b.float()).abs().max() / a.float().pow(2).mean().sqrt())


def main():
    gen = torch.Generator(device=DEV).manual_seed(7)
    rnd = lambda *shape: torch.randn(*shape, generator=gen, device=DEV).to(DT)  # noqa: E731
    layer = Layer(gen)
    prompts, samples, pages = [700, 90, 1030], 2, 96
    rows, width = len(prompts) * (1 + samples), 24
    cache = torch.zeros(pages, PAGE, LAT + PE, dtype=DT, device=DEV)
    state = torch.zeros(rows, 8, 128, dtype=torch.float32, device=DEV)  # a KDA layer's state rows, one a sequence

    # ---- the books: pages 0, 3, 6, ... to the prompts, the rest on the stack
    table = torch.full((rows, width), -1, dtype=torch.int32)
    lens, refs, at = [0] * rows, [0] * pages, 0
    for n, length in enumerate(prompts):
        for i in range(-(-length // PAGE)):
            table[n, i] = at
            refs[at] = 1
            at += 3
        lens[n] = length
    left = [p for p in range(pages) if not refs[p]]
    table, lens, refs = table.to(DEV), _int32(lens), _int32(refs)
    free, num_free = _int32(left + [-1] * (pages - len(left))), _int32([len(left)])

    def slots(which, first, count):
        """Cache rows of tokens first[i] .. + count[i] - 1 of sequences which[i]"""
        t = table.cpu()
        return torch.tensor([int(t[n, j // PAGE]) * PAGE + j % PAGE for n, f, c in zip(which, first, count)
                             for j in range(f, f + c)], dtype=torch.int64, device=DEV)

    # ---- prompts: their tokens into the pages, then the expanded form, against the absorbed form a token at a time
    total = sum(prompts)
    kda355.latent_append(rnd(total, LAT), rnd(total, PE), cache, slots(range(3), [0] * 3, prompts))
    q = rnd(total, HEADS, HEAD + PE)
    out = expanded(layer, cache, table[:3], prompts, q, prompts)
    ends = torch.tensor(prompts).cumsum(0) - 1
    ql, qp = layer.absorb(q[ends.to(DEV)])
    found = {"prompt": apart(out[ends.to(DEV)], layer.values(kda355.latent_decode(ql, qp, cache, table[:3], lens[:3])))}

    # ---- samples: full pages shared, the last one copied; the KDA layers' states by copy_rows
    parents = _int32([n for n in range(3) for _ in range(samples)])
    children = _int32(list(range(3, rows)))
    kda355.fork_pages([cache], table, lens, refs, free, num_free, parents, children, PAGE)
    kda355.copy_rows([state], parents, children)

    # ---- a step of 4 new tokens for every sequence (they fit the last page): absorbed form against expanded form
    new = 4
    before = lens.tolist()
    kda355.latent_append(rnd(rows * new, LAT), rnd(rows * new, PE), cache, slots(range(rows), before, [new] * rows))
    lens += new
    q = rnd(rows * new, HEADS, HEAD + PE)
    ql, qp = layer.absorb(q)
    step = layer.values(kda355.latent_decode(ql, qp, cache, table, lens))
    found["step"] = apart(step, expanded(layer, cache, table, lens.tolist(), q, [new] * rows))

    # ---- the first sample of every prompt dropped (other lengths: the work is cut elsewhere, sums round otherwise), then the
    # pool made dense (the same lengths: the same bits)
    keep = [0, 1, 2, 4, 6, 8]
    left = lambda: layer.values(  # noqa: E731
        kda355.latent_decode(ql, qp, cache, table, lens)).view(rows, new, HEADS, HEAD)[keep]
    kda355.free_pages(table, lens, refs, free, num_free, _int32([3, 5, 7]), PAGE)
    dropped = left()
    found["dropped"] = apart(step.view(rows, new, HEADS, HEAD)[keep], dropped)
    kda355.compact_pages([cache], table, refs, free, num_free)
    found["compacted"] = apart(dropped, left())

    # ---- the second prompt's sequences behind the third as a shared document: against the two lists of pages as one
    doc, own = 1024, [1, 6]  # (rows of the table; whole pages of the document, so that lists can be put together)
    ql, qp = ql[:2 * new], qp[:2 * new]
    shared = kda355.latent_decode(ql, qp, cache, table[own].contiguous(), lens[own].contiguous(),
                                  prefix_table=table[2, :doc // PAGE].contiguous(), prefix_len=_int32([doc]))
    lists = torch.cat([table[2:3, :doc // PAGE].expand(2, -1), table[own][:, :8]], dim=1).contiguous()
    found["prefix"] = apart(shared, kda355.latent_decode(ql, qp, cache, lists, lens[own].clamp(max=8 * PAGE) + doc))
    torch.cuda.synchronize()
    for name, x in found.items():
        print(f"{name:10s} {x:.4f}")
    return found


if __name__ == "__main__":
    main()
