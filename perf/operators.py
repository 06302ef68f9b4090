"""Timed cases of latent attention and its paged cache: the attention layers between the KDA layers of a hybrid model.

A case is a dict of plain values.  `op` names the operator:
  prefill   the expanded form over packed sequences: per-head keys (128 | a 64-wide part shared by the heads) and
            values of 128; `q` are the new tokens of each sequence, `ctx` the tokens of history before them
  decode    the absorbed form over a paged cache of 512 + 64 wide token rows, S tokens a sequence; `lens` are the
            cached tokens of each sequence, the S new ones among them
  prefix    the same for a batch whose sequences share one prefix of `prefix` tokens, held once; `lens` follow it
  tokens    `new` token rows written to their pages and the whole sequences (`lens`) read back as dense rows, as the
            expanded form over a cached history needs them
  fork      `n` samples dropped and as many forked anew: full pages shared, the last one copied in every layer's pool
  compact   the live pages of a fragmented pool moved down to its start in every layer's pool, tables rewritten
`dtype` is the type of the tokens ("bf16" or "fp16"), `page` the tokens of a page.
"""
import math
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda"
NOPE, PE, VD, LAT = 128, 64, 128, 512
ROW = LAT + PE
SCALE = (NOPE + PE) ** -0.5


def listed():
    return [
        # a user's next short turn on top of their history: latency counts
        dict(name="prefill_77_over_1200_h16", op="prefill", q="77", ctx="1200", H=16, causal=True, dtype="bf16"),
        # a serving step of prompts of very different lengths, single tokens among them, most with a history
        dict(name="prefill_mixed_h32", op="prefill", q="2048,1000,517,64,17,1", ctx="0,2000,0,4096,333,8191", H=32,
             causal=True, dtype="fp16"),
        # one long prompt
        dict(name="prefill_8192_h32", op="prefill", q="8192", ctx="0", H=32, causal=True, dtype="bf16"),
        # one user's next token, a tensor-parallel share of the heads: the smallest decode call
        dict(name="decode_b1_4k_h12", op="decode", lens="4097", S=1, H=12, page=64, dtype="bf16"),
        # decode of a large batch at very different lengths, on the odd page size of a hybrid page layout
        dict(name="decode_b64_ragged_h64", op="decode", S=1, H=64, page=272, dtype="bf16",
             lens=",".join(str(200 + (n * 7919) % 15000) for n in range(64))),
        # speculative verify of 8 tokens with all 96 heads on the GPU
        dict(name="verify_b16_s8_h96", op="decode", S=8, H=96, page=64, dtype="fp16",
             lens=",".join(str(6000 + 257 * n) for n in range(16))),
        # a few samples of one short system prompt
        dict(name="prefix_b8_2k_h12", op="prefix", prefix=2000, S=1, H=12, page=16, dtype="bf16",
             lens="1,33,64,100,7,250,18,90"),
        # a batch of requests over one long document
        dict(name="prefix_b64_32k_h32", op="prefix", prefix=32768, S=1, H=32, page=64, dtype="bf16",
             lens=",".join(str(1 + (n * 613) % 1000) for n in range(64))),
        # the cache write of a decode step, with the histories read back for a short turn
        dict(name="tokens_b4_short", op="tokens", new="1,1,16,77", lens="130,1,400,1277", page=64, dtype="bf16"),
        # a chunk of long prompts written and their histories gathered
        dict(name="tokens_64k", op="tokens", new="4096,2000,1,517", lens="32768,20001,4000,9000", page=272, dtype="bf16"),
        # parallel samples: 64 of the step before dropped, and each of 8 prompts forked into 8 new ones
        dict(name="fork_64_of_8", op="fork", n=64, lens="700,1025,64,333,2000,4097,90,1500", page=64, layers=4,
             dtype="bf16"),
        # a pool fragmented by many finished requests made dense again
        dict(name="compact_4096", op="compact", pages=4096, rows=64, live=0.5, page=64, layers=4, dtype="bf16"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["prefill", "prefill", "decode", "decode", "prefix", "prefix", "tokens", "fork", "compact"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    page = rng.choice([1, 16, 16, 64, 64, 100, 272])
    if op == "prefill":
        H = rng.choice([1, 4, 8, 16, 32, 64, 96])
        n = _log_uniform(rng, 1, 16)
        causal = rng.random() < 0.8
        q, ctx = [], []
        for _ in range(n):
            a = _log_uniform(rng, 1, 8000)
            c = 0 if rng.random() < 0.4 else _log_uniform(rng, 1, 16000)
            pairs = _pairs(a, c, causal) + sum(_pairs(x, y, causal) for x, y in zip(q, ctx))
            if H * pairs > 1.0e9 or H * (a + c + sum(q) + sum(ctx)) > 600000:
                a, c = min(a, 64), min(c, 300)
            q.append(a)
            ctx.append(c)
        return dict(op=op, H=H, causal=causal, dtype=dtype, q=_text(q), ctx=_text(ctx))
    if op in ("decode", "prefix"):
        H = rng.choice([1, 4, 8, 12, 16, 32, 64, 96, 128])
        S = rng.choice([1, 1, 1, 2, 3, 4, 8])
        B = _log_uniform(rng, 1, 128)
        most = _log_uniform(rng, 64, 60000)
        most = max(S, min(most, int(1.0e8 / (B * S * H)), 450000 // B))
        lens = [max(S, int(most * rng.uniform(0.02, 1.0))) for _ in range(B)]
        case = dict(op=op, H=H, S=S, page=page, dtype=dtype, lens=_text(lens))
        if op == "prefix":
            case["prefix"] = min(_log_uniform(rng, 100, 60000), max(1, int(6.0e7 / (B * S * H))))
        return case
    if op == "tokens":
        n = _log_uniform(rng, 1, 32)
        lens = [_log_uniform(rng, 1, 30000) for _ in range(n)]
        scale = min(1.0, 60000 / sum(lens))
        lens = [max(1, int(x * scale)) for x in lens]
        return dict(op=op, page=page, dtype=dtype, lens=_text(lens),
                    new=_text([min(x, _log_uniform(rng, 1, 4096)) for x in lens]))
    if op == "fork":
        page = max(16, page)
        lens = [_log_uniform(rng, 1, 8000) for _ in range(_log_uniform(rng, 1, 16))]
        return dict(op=op, n=_log_uniform(rng, 1, 128), lens=_text(lens), page=page, layers=rng.choice([1, 2, 4, 8]),
                    dtype=dtype)
    return dict(op=op, pages=_log_uniform(rng, 64, 4096), rows=_log_uniform(rng, 4, 200), live=rng.uniform(0.1, 0.95),
                page=rng.choice([16, 64]), layers=rng.choice([1, 2, 4]), dtype=dtype)


def _text(values):
    return ",".join(str(v) for v in values)


def _ints(text):
    return [int(v) for v in text.split(",")]


def _pairs(a, c, causal):
    """Visible (query, key) pairs of `a` new tokens after `c` tokens of history."""
    return a * c + (a * (a + 1) // 2 if causal else a * a)


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float16


# ------------------------------------------------------------------------------------------------------------- inputs
class _Random:
    """Device normals and permutations from one seeded generator each."""

    def __init__(self, seed):
        self.dev = torch.Generator(device=DEV).manual_seed(seed)
        self.cpu = torch.Generator().manual_seed(seed)

    def normal(self, *shape, dtype, std=1.0):
        return (torch.randn(*shape, generator=self.dev, device=DEV) * std).to(dtype)

    def pages(self, count):
        return torch.randperm(count, generator=self.cpu).to(torch.int32)


def _offsets(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _table(rnd, lens, page, spare=0):
    """Sequences of `lens` tokens on scattered pages: (block table on the host, pages in the pool)."""
    need = [-(-n // page) for n in lens]
    total = sum(need) + spare
    perm = rnd.pages(total)
    table = torch.full((len(lens), max(1, max(need))), -1, dtype=torch.int32)
    at = 0
    for i, k in enumerate(need):
        table[i, :k] = perm[at:at + k]
        at += k
    return table, total, perm[at:]


def prepare(case, seed):
    rnd = _Random(seed)
    dt = _dtype(case)
    st = dict(case)
    op = case["op"]
    if op == "prefill":
        H, q, ctx = case["H"], _ints(case["q"]), _ints(case["ctx"])
        cu_q, cu_k = _offsets(q), _offsets([a + c for a, c in zip(q, ctx)])
        # what the projections leave: queries of 128 | 64 a head, keys and values side by side, the shared part as
        # the tail of the latent rows
        kv = rnd.normal(cu_k[-1], H, NOPE + VD, dtype=dt)
        rows = rnd.normal(cu_k[-1], ROW, dtype=dt)
        st.update(q=rnd.normal(cu_q[-1], H, NOPE + PE, dtype=dt, std=1.5), k=kv[..., :NOPE], v=kv[..., NOPE:],
                  k_pe=rows[:, LAT:], host_q=cu_q, host_k=cu_k, cu_q=_int32(cu_q), cu_k=_int32(cu_k))
    elif op in ("decode", "prefix"):
        lens, S, H, page = _ints(case["lens"]), case["S"], case["H"], case["page"]
        every = lens + [case["prefix"]] if op == "prefix" else lens
        table, total, _ = _table(rnd, every, page)
        T = len(lens) * S
        st.update(q_latent=rnd.normal(T, H, LAT, dtype=dt), q_pe=rnd.normal(T, H, PE, dtype=dt),
                  cache=rnd.normal(total, page, ROW, dtype=dt), host_lens=lens)
        if op == "prefix":
            st.update(prefix_table=table[-1].contiguous().to(DEV), prefix_len=_int32([case["prefix"]]))
            table = table[:-1, :max(1, max(-(-n // page) for n in lens))].contiguous()
        st.update(table=table.to(DEV), seq_lens=_int32(lens))
    elif op == "tokens":
        lens, new, page = _ints(case["lens"]), _ints(case["new"]), case["page"]
        table, total, _ = _table(rnd, lens, page)
        slots = []
        for row, n, k in zip(table.tolist(), lens, new):
            slots += [row[t // page] * page + t % page for t in range(n - k, n)]
        T = len(slots)
        st.update(cache=rnd.normal(total, page, ROW, dtype=dt), latent=rnd.normal(T, LAT, dtype=dt),
                  k_pe=rnd.normal(T, ROW, dtype=dt)[:, LAT:], slots=torch.tensor(slots, dtype=torch.int64, device=DEV),
                  table=table.to(DEV), cu=_int32(_offsets(lens)), host_lens=lens,
                  out=torch.empty(sum(lens), ROW, dtype=dt, device=DEV))
    elif op == "fork":
        lens, n, page = _ints(case["lens"]), case["n"], case["page"]
        table, total, spare = _table(rnd, lens, page, spare=n + 5)
        # the samples of the step before are there already, so that a pass (drop, then fork) can be repeated
        refs = torch.zeros(total, dtype=torch.int32)
        refs[table[table >= 0].long()] = 1
        spare = torch.sort(spare, descending=True).values.tolist()
        rows = torch.full((len(lens) + n, table.shape[1]), -1, dtype=torch.int32)
        rows[:len(lens)] = table
        parents = [i % len(lens) for i in range(n)]
        for i, p in enumerate(parents):
            full = lens[p] // page
            rows[len(lens) + i, :full] = table[p, :full]
            refs[table[p, :full].long()] += 1
            if lens[p] % page:
                rows[len(lens) + i, full] = spare.pop()
                refs[rows[len(lens) + i, full].long()] = 1
        free = torch.full((total,), -1, dtype=torch.int32)
        free[:len(spare)] = torch.tensor(spare, dtype=torch.int32)
        st.update(pools=[rnd.normal(total, page, ROW, dtype=dt) for _ in range(case["layers"])],
                  table=rows.to(DEV), seq_lens=_int32(lens + [lens[p] for p in parents]), refs=refs.to(DEV),
                  free=free.to(DEV), num_free=_int32([len(spare)]), parents=_int32(parents),
                  children=_int32([len(lens) + i for i in range(n)]))
    else:
        pages, rows, page = case["pages"], case["rows"], case["page"]
        live = max(1, int(pages * case["live"]))
        perm = rnd.pages(pages)
        per = -(-live // rows)
        width = per + 2
        table = torch.full((rows, width), -1, dtype=torch.int32)
        for i in range(rows):
            own_pages = perm[min(i * per, live):min((i + 1) * per, live)]
            shared = perm[:min(2, live)] if i else perm[:0]  # every sequence after the first shares its first pages
            table[i, :len(shared)] = shared
            table[i, len(shared):len(shared) + len(own_pages)] = own_pages
        refs = torch.bincount(table[table >= 0].long(), minlength=pages).to(torch.int32)
        gone = torch.nonzero(refs == 0).flatten().to(torch.int32)
        free = torch.full((pages,), -1, dtype=torch.int32)
        free[:len(gone)] = gone.flip(0)
        st.update(pools=[rnd.normal(pages, page, ROW, dtype=dt) for _ in range(case["layers"])],
                  table0=table.to(DEV), refs0=refs.to(DEV), free0=free.to(DEV), num_free0=_int32([len(gone)]))
    return st


# -------------------------------------------------------------------------------------------------------- plain forms
def _softmax_rows(s):
    """(exp(s - max), row sum, log-sum-exp); rows of -inf only give zeros and -inf."""
    m = s.max(dim=-1, keepdim=True).values
    e = torch.exp(s - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    l = e.sum(dim=-1, keepdim=True)
    return e, l, (torch.log(l) + m).squeeze(-1)


def _plain_prefill(st):
    q, k, v, pe = st["q"], st["k"], st["v"], st["k_pe"]
    H = q.shape[1]
    out = torch.empty(q.shape[0], H, VD, dtype=q.dtype, device=DEV)
    lse = torch.empty(q.shape[0], H, device=DEV)
    for i in range(len(st["host_q"]) - 1):
        a, b, c, d = st["host_q"][i], st["host_q"][i + 1], st["host_k"][i], st["host_k"][i + 1]
        keys = torch.arange(d - c, device=DEV)
        pos = torch.arange(b - a, device=DEV) + (d - c) - (b - a)
        step = max(1, (1 << 27) // (d - c))
        for h in range(H):
            kk = torch.cat([k[c:d, h], pe[c:d]], dim=-1).float().t().contiguous()
            vv = v[c:d, h].float()
            for r in range(a, b, step):
                e = min(b, r + step)
                s = (q[r:e, h].float() @ kk) * SCALE
                if st["causal"]:
                    s = s.masked_fill(keys[None, :] > pos[r - a:e - a, None], -math.inf)
                p, l, lse[r:e, h] = _softmax_rows(s)
                out[r:e, h] = ((p @ vv) / l).to(out.dtype)
    return out, lse


def _plain_decode(st):
    S, H = st["S"], st["H"]
    ql, qp, cache, table = st["q_latent"], st["q_pe"], st["cache"], st["table"].long()
    page = cache.shape[1]
    out = torch.empty(ql.shape[0], H, LAT, dtype=ql.dtype, device=DEV)
    lse = torch.empty(ql.shape[0], H, device=DEV)
    shared = None
    if "prefix_table" in st:
        n = st["prefix"]
        shared = cache[st["prefix_table"].long()[:-(-n // page)]].reshape(-1, ROW)[:n]
    for i, n in enumerate(st["host_lens"]):
        rows = cache[table[i, :-(-n // page)]].reshape(-1, ROW)[:n]
        if shared is not None:
            rows = torch.cat([shared, rows])
        rows = rows.float()
        total = rows.shape[0]
        q = torch.cat([ql[i * S:(i + 1) * S], qp[i * S:(i + 1) * S]], dim=-1).float().reshape(S * H, ROW)
        s = (q @ rows.t().contiguous()) * SCALE
        if S > 1:
            last = torch.arange(S, device=DEV).repeat_interleave(H) + total - S
            first = total - n
            keys = torch.arange(total, device=DEV)
            s = s.masked_fill((keys[None, :] > last[:, None]) & (keys[None, :] >= first), -math.inf)
        p, l, z = _softmax_rows(s)
        l = torch.where(l == 0, torch.ones_like(l), l)
        out[i * S:(i + 1) * S] = ((p @ rows[:, :LAT]) / l).to(out.dtype).view(S, H, LAT)
        lse[i * S:(i + 1) * S] = z.view(S, H)
    return out, lse


def _plain_tokens(st):
    cache, page = st["cache"], st["page"]
    cache.view(-1, ROW)[st["slots"]] = torch.cat([st["latent"], st["k_pe"]], dim=-1)
    table = st["table"].long()
    rows = [cache[table[i, :-(-n // page)]].reshape(-1, ROW)[:n] for i, n in enumerate(st["host_lens"])]
    return cache, torch.cat(rows)


def _count(pages, values):
    """How often each page stands in `values` (entries below 0 left out)."""
    return torch.bincount(torch.where(values >= 0, values, torch.full_like(values, pages)).flatten().long(),
                          minlength=pages + 1)[:pages].int()


def _plain_fork(st):
    table, lens, refs, free, page = st["table"], st["seq_lens"], st["refs"], st["free"], st["page"]
    par, child = st["parents"].long(), st["children"].long()
    n, width, pages = par.numel(), table.shape[1], refs.numel()
    top = st["num_free"].long()
    at = torch.arange(pages, device=DEV)
    # the old samples dropped: references taken back, pages left without any pushed, the highest first
    gone = _count(pages, table[child])
    refs -= gone
    mine = (gone > 0) & (refs == 0)
    order = torch.flip(torch.cumsum(torch.flip(mine.long(), [0]), 0), [0]) - 1 + top
    grown = torch.cat([free, free.new_zeros(1)])
    grown[torch.where(mine, order, torch.full_like(order, pages))] = at.int()
    free.copy_(grown[:-1])
    top = top + mine.long().sum()
    # the new ones: full pages shared, a page from the stack for the part-filled one
    cols = torch.arange(width, device=DEV)
    ln = lens[par].long()
    full, tail = ln // page, (ln % page) > 0
    rank = torch.cumsum(tail.long(), 0) - tail.long()
    taken = torch.where(tail, free.long()[(top - 1 - rank).clamp(min=0)], torch.full_like(rank, -1))
    old = table[par]
    share = cols[None, :] < full[:, None]
    table[child] = torch.where(share, old, torch.where((cols[None, :] == full[:, None]) & tail[:, None],
                                                       taken[:, None].int(), torch.full_like(old, -1)))
    refs += _count(pages, table[child])
    # one page copied for each fork; a fork without a part-filled page copies its first page onto itself
    src = torch.where(tail, old.gather(1, full.clamp(max=width - 1)[:, None]).flatten(), old[:, 0]).long()
    dst = torch.where(tail, taken, src)
    for pool in st["pools"]:
        pool[dst] = pool[src]
    lens[child] = ln.int()
    left = top - tail.long().sum()
    free.masked_fill_(at >= left, -1)
    st["num_free"].copy_(left.int())
    return (table, lens, refs, free, st["num_free"]) + tuple(st["pools"])


def _plain_compact(st):
    table, refs = st["table0"], st["refs0"]
    pages = refs.numel()
    live = refs > 0
    count = live.long().sum()
    idx = torch.arange(pages, device=DEV)
    mover = live & (idx >= count)
    hole = ~live & (idx < count)
    # the i-th hole takes the i-th page above the live count (there are as many of either)
    holes = torch.argsort((~hole).long(), stable=True)
    movers = torch.argsort((~mover).long(), stable=True)
    some = idx < hole.long().sum()
    rank = torch.cumsum(mover.long(), 0) - 1
    remap = torch.where(mover, holes[rank.clamp(min=0)], idx)
    source = torch.cat([idx, idx[:1]])
    source[torch.where(some, holes, torch.full_like(idx, pages))] = movers
    for pool in st["pools"]:
        pool.copy_(pool[source[:-1]])
    new = torch.where(table >= 0, remap[table.clamp(min=0).long()].int(), table)
    left = torch.where(idx < count, torch.where(hole, torch.zeros_like(refs), refs), torch.zeros_like(refs))
    left = left.scatter_add(0, torch.where(mover, remap, idx), torch.where(mover, refs, torch.zeros_like(refs)))
    free = torch.where(idx < pages - count, pages - 1 - idx, torch.full_like(idx, -1)).int()
    return (new, left, free, (pages - count).int().view(1)) + tuple(st["pools"])


# --------------------------------------------------------------------------------------------------------- own kernels
def _kda355():
    if "kda355" not in sys.modules:  # a program finds its package once, not at every call
        sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "eat-kernels_amd"))
    import kda355
    return kda355


def _own_run(st):
    kda355 = _kda355()
    op = st["op"]
    if op == "prefill":
        lse = torch.empty(st["q"].shape[:2], dtype=torch.float32, device=DEV)
        out = kda355.latent_prefill(st["q"], st["k"], st["v"], st["k_pe"], st["cu_q"], st["cu_k"], scale=SCALE,
                                    causal=st["causal"], lse=lse)
        return out, lse
    if op in ("decode", "prefix"):
        lse = torch.empty(st["q_latent"].shape[:2], dtype=torch.float32, device=DEV)
        out = kda355.latent_decode(st["q_latent"], st["q_pe"], st["cache"], st["table"], st["seq_lens"], scale=SCALE,
                                   lse=lse, prefix_table=st.get("prefix_table"), prefix_len=st.get("prefix_len"))
        return out, lse
    if op == "tokens":
        kda355.latent_append(st["latent"], st["k_pe"], st["cache"], st["slots"])
        return st["cache"], kda355.latent_gather(st["cache"], st["table"], st["cu"], st["out"])
    if op == "fork":
        kda355.free_pages(st["table"], st["seq_lens"], st["refs"], st["free"], st["num_free"], st["children"],
                          st["page"])
        kda355.fork_pages(st["pools"], st["table"], st["seq_lens"], st["refs"], st["free"], st["num_free"],
                          st["parents"], st["children"], st["page"])
        return (st["table"], st["seq_lens"], st["refs"], st["free"], st["num_free"]) + tuple(st["pools"])
    # the bookkeeping is copied first, so that a pass can be repeated (the pages moved are the same each time)
    table, refs, free, num = (st[k].clone() for k in ("table0", "refs0", "free0", "num_free0"))
    kda355.compact_pages(st["pools"], table, refs, free, num)
    return (table, refs, free, num) + tuple(st["pools"])


def run(state):
    if own:
        return _own_run(state)
    return {"prefill": _plain_prefill, "decode": _plain_decode, "prefix": _plain_decode, "tokens": _plain_tokens,
            "fork": _plain_fork, "compact": _plain_compact}[state["op"]](state)


# --------------------------------------------------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op == "prefill":
        H, q, ctx = case["H"], _ints(case["q"]), _ints(case["ctx"])
        Tq, Tk = sum(q), sum(q) + sum(ctx)
        pairs = sum(_pairs(a, c, case["causal"]) for a, c in zip(q, ctx))
        return {"bytes": 2 * (Tq * H * (NOPE + PE + VD) + Tk * (H * (NOPE + VD) + PE)) + 4 * Tq * H,
                "flops": 2 * H * pairs * (NOPE + PE + VD)}
    if op in ("decode", "prefix"):
        lens, S, H = _ints(case["lens"]), case["S"], case["H"]
        P = case.get("prefix", 0)
        seen = sum(max(0, n - S + 1 + s) + P for n in lens for s in range(S))
        rows = len(lens) * S * H
        return {"bytes": 2 * ((sum(lens) + P) * ROW + rows * (ROW + LAT)) + 4 * rows,
                "flops": 2 * H * seen * (ROW + LAT)}
    if op == "tokens":
        return {"bytes": 4 * ROW * (sum(_ints(case["new"])) + sum(_ints(case["lens"]))), "flops": 0}
    if op == "fork":
        lens, n, page = _ints(case["lens"]), case["n"], case["page"]
        copied = sum(1 for i in range(n) if lens[i % len(lens)] % page)
        width = max(-(-x // page) for x in lens)
        total = sum(-(-x // page) for x in lens) + n + 5
        return {"bytes": copied * case["layers"] * page * ROW * 4 + 4 * (6 * n * width + 8 * total), "flops": 0}
    pages = case["pages"]
    live = max(1, int(pages * case["live"]))
    moved = int(live * (pages - live) / pages)  # pages above the live count, for live pages spread evenly
    return {"bytes": moved * case["layers"] * case["page"] * ROW * 4 + 16 * pages, "flops": 0}


# ------------------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    """The definitions in float64: o = sum_j w_j v_j / sum_j w_j over the visible keys, w_j = e^(z_j), lse = log sum w_j.
    The token and page cases move values and whole numbers: nothing there is computed."""
    if case["op"] not in ("prefill", "decode", "prefix"):
        return None
    if work(case)["flops"] > 8.0e12:
        return None
    st = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "prefill":
        H = case["H"]
        o = torch.zeros(st["q"].shape[0], H, VD, dtype=f64, device=DEV)
        z = torch.zeros(st["q"].shape[0], H, dtype=f64, device=DEV)
        for n in range(len(st["host_q"]) - 1):
            q0, q1, k0, k1 = st["host_q"][n], st["host_q"][n + 1], st["host_k"][n], st["host_k"][n + 1]
            shift = (k1 - k0) - (q1 - q0)
            shared = st["k_pe"][k0:k1].to(f64)
            for h in range(H):
                key, val = st["k"][k0:k1, h].to(f64), st["v"][k0:k1, h].to(f64)
                for i in range(q0, q1, 1024):
                    j = min(q1, i + 1024)
                    seen = min(k1 - k0, shift + j - q0) if case["causal"] else k1 - k0
                    qq = st["q"][i:j, h].to(f64)
                    x = qq[:, :NOPE] @ key[:seen].T + qq[:, NOPE:] @ shared[:seen].T
                    x = x / math.sqrt(NOPE + PE)
                    if case["causal"]:
                        hidden = torch.ones(j - i, seen, dtype=torch.bool, device=DEV).triu(shift + i - q0 + 1)
                        x[hidden] = -math.inf
                    z[i:j, h] = torch.logsumexp(x, dim=1)
                    o[i:j, h] = torch.exp(x - z[i:j, h, None]) @ val[:seen]
        return o, z
    S, H, page = case["S"], case["H"], case["page"]
    T = st["q_latent"].shape[0]
    o = torch.zeros(T, H, LAT, dtype=f64, device=DEV)
    z = torch.full((T, H), -math.inf, dtype=f64, device=DEV)
    P = case.get("prefix", 0)
    flat = st["cache"].reshape(-1, ROW)

    def token_rows(pages_of, n):
        t = torch.arange(n, device=DEV)
        return flat[pages_of.long()[t // page] * page + t % page].to(f64)

    head = token_rows(st["prefix_table"], P) if P else flat[:0].to(f64)
    for n, length in enumerate(st["host_lens"]):
        rows = torch.cat([head, token_rows(st["table"][n], length)])
        for s in range(S):
            seen = P + max(0, length - (S - 1 - s))
            if seen == 0:
                continue
            t = n * S + s
            x = st["q_latent"][t].to(f64) @ rows[:seen, :LAT].T + st["q_pe"][t].to(f64) @ rows[:seen, LAT:].T
            x = x / math.sqrt(NOPE + PE)
            z[t] = torch.logsumexp(x, dim=1)
            o[t] = torch.exp(x - z[t][:, None]) @ rows[:seen, :LAT]
    return o, z
