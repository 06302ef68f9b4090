"""Timed cases of long latent caches made cheaper: rows held in 4 bits, and sequences kept to a budget of tokens.

A case is a dict of plain values.  `op` names the operator:
  tokens    `new` token rows rounded to 4 bits into their pages, and the whole sequences (`lens`) read back as dense
            16-bit rows, as the expanded form over a cached history needs them
  decode    attention in the absorbed form over a paged cache in 4 bits, S tokens a sequence; `lens` are the cached
            tokens of each sequence, the S new ones among them; `prefix` tokens in front of them that all share, if any
  weights   what every cached token was given by the softmax of a decode step, over its heads and S tokens, added to the
            tokens' accumulated weights; `bits` is the cache's
  evict     sequences longer than `keep` tokens cut to `keep` in every layer: the `recent` last ones stay, and of the
            others those with the largest accumulated weights of the layer; `shared` of them were forked from the first and
            share its first pages, which stay.  A pass begins from the same books and weights
`dtype` is the type of queries and 16-bit rows ("bf16" or "fp16"), `page` the tokens of a page.

A row in 4 bits is 400 bytes: 256 of codes (value 2 i in the low half of byte i), 16 scales of 32 consecutive values each, the
positional part of 64 values in 16 bits.  A code is a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6; a scale byte b stands for
2^(b - 127), 255 for NaN.
"""
import math
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda"
PE, LAT, GROUP = 64, 512, 32
ROW, ROW4 = LAT + PE, LAT // 2 + LAT // GROUP + 2 * PE
SCALE = 192 ** -0.5


def listed():
    return [
        # a decode step's cache write, with the histories read back for a short turn: latency counts
        dict(name="tokens_b4_short", op="tokens", new="1,1,16,77", lens="130,1,400,1277", page=64, dtype="bf16"),
        # a chunk of long prompts written and their histories gathered, on the odd page size of a hybrid page layout
        dict(name="tokens_64k", op="tokens", new="4096,2000,1,517", lens="32768,20001,4000,9000", page=272, dtype="fp16"),
        # one user's next token, a tensor-parallel share of the heads: the smallest decode call
        dict(name="decode_b1_4k_h12", op="decode", lens="4097", S=1, H=12, page=64, prefix=0, dtype="bf16"),
        # decode of a large batch at very different lengths
        dict(name="decode_b64_ragged_h32", op="decode", S=1, H=32, page=272, prefix=0, dtype="bf16",
             lens=",".join(str(200 + (n * 7919) % 15000) for n in range(64))),
        # speculative verify of 8 tokens with all 96 heads on the GPU
        dict(name="verify_b16_s8_h96", op="decode", S=8, H=96, page=64, prefix=0, dtype="fp16",
             lens=",".join(str(6000 + 257 * n) for n in range(16))),
        # a batch of requests over one long document
        dict(name="prefix_b64_32k_h64", op="decode", prefix=32768, S=1, H=64, page=64, dtype="bf16",
             lens=",".join(str(1 + (n * 613) % 1000) for n in range(64))),
        # the weights of one user's step
        dict(name="weights_b1_4k_h12", op="weights", bits=16, lens="4097", S=1, H=12, page=64, dtype="bf16"),
        # the weights of a large ragged batch over a 4-bit cache
        dict(name="weights4_b64_ragged_h64", op="weights", bits=4, S=1, H=64, page=272, dtype="bf16",
             lens=",".join(str(200 + (n * 7919) % 15000) for n in range(64))),
        # the weights of a verify step with all heads
        dict(name="weights_b16_s8_h96", op="weights", bits=16, S=8, H=96, page=64, dtype="fp16",
             lens=",".join(str(6000 + 257 * n) for n in range(16))),
        # one user's sequence a page above its budget
        dict(name="evict_b1_4k", op="evict", bits=16, lens="4160", keep=4096, recent=256, shared=0, page=64, layers=1,
             dtype="bf16"),
        # a batch around its budget, some of it parallel samples of one prompt
        dict(name="evict4_b64_l4", op="evict", bits=4, keep=4096, recent=512, shared=8, page=64, layers=4, dtype="bf16",
             lens=",".join(str(2500 + (n * 7919) % 6000) for n in range(64))),
        # long documents just read, cut to a quarter
        dict(name="evict_128k_l7", op="evict", bits=16, lens="131072,100001", keep=32768, recent=4096, shared=0, page=272,
             layers=7, dtype="bf16"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tokens", "decode", "decode", "decode", "weights", "weights", "evict", "evict"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    page = rng.choice([1, 16, 16, 64, 64, 100, 272])
    if op == "tokens":
        lens = [_log_uniform(rng, 1, 30000) for _ in range(_log_uniform(rng, 1, 32))]
        scale = min(1.0, 60000 / sum(lens))
        lens = [max(1, int(x * scale)) for x in lens]
        return dict(op=op, page=page, dtype=dtype, lens=_text(lens),
                    new=_text([min(x, _log_uniform(rng, 1, 4096)) for x in lens]))
    if op in ("decode", "weights"):
        H = rng.choice([1, 4, 8, 12, 16, 32, 64, 96, 128])
        S = rng.choice([1, 1, 1, 2, 3, 4, 8])
        B = _log_uniform(rng, 1, 128)
        most = _log_uniform(rng, 64, 60000)
        most = max(S, min(most, int(1.0e8 / (B * S * H)), 450000 // B))
        lens = [max(S, int(most * rng.uniform(0.02, 1.0))) for _ in range(B)]
        case = dict(op=op, H=H, S=S, page=page, dtype=dtype, lens=_text(lens))
        if op == "decode":
            case["prefix"] = min(_log_uniform(rng, 100, 60000), int(6.0e7 / (B * S * H))) if rng.random() < 0.3 else 0
        else:
            case["bits"] = rng.choice([4, 16])
        return case
    B = _log_uniform(rng, 1, 64)
    layers = rng.choice([1, 1, 2, 4, 7])
    most = min(_log_uniform(rng, 64, 100000), 400000 // (B * layers))
    lens = [max(2, int(most * rng.uniform(0.2, 1.0))) for _ in range(B)]
    keep = max(1, int(max(lens) * rng.uniform(0.1, 0.99)))
    recent = int(keep * rng.uniform(0.0, 0.6))
    return dict(op=op, bits=rng.choice([4, 16]), lens=_text(lens), keep=keep, recent=recent,
                shared=rng.choice([0, 0, B // 4]), page=rng.choice([1, 16, 64, 100, 272]), layers=layers, dtype=dtype)


def _text(values):
    return ",".join(str(v) for v in values)


def _ints(text):
    return [int(v) for v in text.split(",")]


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float16


# ------------------------------------------------------------------------------------------------------------- inputs
class _Random:
    """Device normals and permutations from one seeded generator each; latent vectors have channels of different size."""

    def __init__(self, seed):
        self.dev = torch.Generator(device=DEV).manual_seed(seed)
        self.cpu = torch.Generator().manual_seed(seed)
        self.gain = torch.exp(0.5 * torch.randn(LAT, generator=self.cpu)).to(DEV)

    def normal(self, *shape, dtype):
        return torch.randn(*shape, generator=self.dev, device=DEV).to(dtype)

    def latent(self, n, dtype):
        return (torch.randn(n, LAT, generator=self.dev, device=DEV) * self.gain).to(dtype)

    def cache(self, pages, page, bits, dtype):
        n = pages * page
        if bits == 16:
            out = torch.empty(n, ROW, dtype=dtype, device=DEV)
        else:
            out = torch.empty(n, ROW4, dtype=torch.uint8, device=DEV)
        power = _powers()
        for i in range(0, n, 1 << 17):
            rows = out[i:i + (1 << 17)]
            lat, pe = self.latent(len(rows), dtype), self.normal(len(rows), PE, dtype=dtype)
            rows.copy_(torch.cat([lat, pe], dim=-1) if bits == 16 else _rounded(lat, pe, power))
        return out.view(pages, page, out.shape[1])

    def pages(self, count):
        return torch.randperm(count, generator=self.cpu).to(torch.int32)


def _powers():
    """What the scale bytes stand for."""
    return torch.tensor([2.0 ** (b - 127) for b in range(255)] + [math.nan], dtype=torch.float64).float().to(DEV)


def _codes():
    """What the codes stand for."""
    size = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    return torch.tensor(size + [-x for x in size], device=DEV)


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
    perm = rnd.pages(sum(need) + spare)
    table = torch.full((len(lens), max(1, max(need))), -1, dtype=torch.int32)
    at = 0
    for i, k in enumerate(need):
        table[i, :k] = perm[at:at + k]
        at += k
    return table, len(perm)


def prepare(case, seed):
    rnd = _Random(seed)
    dt = _dtype(case)
    st = dict(case, power=_powers(), code=_codes())
    op, page, lens = case["op"], case["page"], _ints(case["lens"])
    if op == "tokens":
        new = _ints(case["new"])
        table, total = _table(rnd, lens, page)
        slots = []
        for row, n, k in zip(table.tolist(), lens, new):
            slots += [row[t // page] * page + t % page for t in range(n - k, n)]
        # the new rows as the projection leaves them: the positional part is the tail of wider rows
        st.update(cache=rnd.cache(total, page, 4, dt), latent=rnd.latent(len(slots), dt),
                  k_pe=rnd.normal(len(slots), ROW, dtype=dt)[:, LAT:],
                  slots=torch.tensor(slots, dtype=torch.int64, device=DEV), table=table.to(DEV), seq_lens=_int32(lens),
                  cu=_int32(_offsets(lens)), total=sum(lens), out=torch.empty(sum(lens), ROW, dtype=dt, device=DEV))
    elif op in ("decode", "weights"):
        S, H, P = case["S"], case["H"], case.get("prefix", 0)
        table, total = _table(rnd, lens + [P] if P else lens, page)
        T = len(lens) * S
        st.update(q_latent=rnd.normal(T, H, LAT, dtype=dt), q_pe=rnd.normal(T, H, PE, dtype=dt), most=max(lens),
                  cache=rnd.cache(total, page, case.get("bits", 4), dt), seq_lens=_int32(lens))
        if P:
            st.update(prefix_table=table[-1].contiguous().to(DEV), prefix_len=_int32([P]))
            table = table[:-1, :max(1, max(-(-n // page) for n in lens))].contiguous()
        st.update(table=table.to(DEV))
        if op == "weights":  # the sums that the step's attention left, and the weights of the steps before
            st["lse"] = _softmax(_scores(st, _rows(st, st["table"], st["most"])))[2].view(T, H)
            st["weights"] = torch.rand(len(lens), table.shape[1] * page, generator=rnd.dev, device=DEV)
    else:
        keep = case["keep"]
        table, total = _table(rnd, lens, page, spare=3)
        refs = torch.zeros(total, dtype=torch.int32)
        first = min(lens[0], max(0, keep - case["recent"]) // 2) // page  # whole pages of the first sequence
        for n in range(1, 1 + case["shared"]):
            k = min(first, lens[n] // page)
            table[n, :k] = table[0, :k]
        refs.index_add_(0, table[table >= 0].long(), torch.ones(int((table >= 0).sum()), dtype=torch.int32))
        gone = torch.nonzero(refs == 0).flatten().to(torch.int32)
        free = torch.full((total,), -1, dtype=torch.int32)
        free[:len(gone)] = gone.flip(0)
        B, W = table.shape[0], table.shape[1] * page
        # books and weights of all layers in a buffer each: a pass begins from copies of both
        books = torch.cat([table.flatten(), torch.tensor(lens, dtype=torch.int32), refs, free,
                           torch.tensor([len(gone)], dtype=torch.int32)]).to(DEV)
        weights = torch.exp(2 * torch.randn(case["layers"], B, W, generator=rnd.dev, device=DEV))
        weights *= torch.rand(case["layers"], B, W, generator=rnd.dev, device=DEV) > 0.1  # (some were never looked at)
        weights *= torch.arange(W, device=DEV) < _int32(lens)[:, None]
        st.update(pools=[rnd.cache(total, page, case["bits"], dt) for _ in range(case["layers"])], books0=books,
                  books=books.clone(), weights0=weights, weights=weights.clone(), rows=_int32(list(range(B))))
        at, parts = 0, {}
        for name, shape in (("table", table.shape), ("seq_lens", (B,)), ("refs", (total,)), ("free", (total,)),
                            ("num_free", (1,))):
            n = math.prod(shape)
            parts[name] = st["books"][at:at + n].view(shape)
            at += n
        st.update(parts, masses=list(st["weights"]))
    return st


# -------------------------------------------------------------------------------------------------------- plain forms
def _rounded(latent, pe, power):
    """Rows of 400 bytes: groups scaled by a power of two, values to the nearest code, ties to the even one."""
    x = latent.float().view(-1, LAT // GROUP, GROUP)
    a = x.abs().amax(dim=-1)
    low = -125 if latent.dtype == torch.bfloat16 else -23  # every value is one of the type
    good = torch.isfinite(a)
    e = torch.frexp(torch.where(good, a, torch.ones_like(a))).exponent - 3
    e = torch.where(a > 7 * power[(e + 127).clamp(min=0)], e + 1, e).clamp(min=low)
    y = x.abs() * power[127 - e][..., None]
    code = ((y > 0.25).byte() + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5) + (y >= 3.5) + (y > 5)).byte()
    code = (code | torch.signbit(x).byte() << 3) * good[..., None]
    code = code.view(-1, LAT // 2, 2)
    scale = torch.where(good, e + 127, torch.full_like(e, 255)).byte()
    return torch.cat([code[..., 0] | code[..., 1] << 4, scale, pe.contiguous().view(torch.uint8)], dim=-1)


def _values(st, rows):
    """fp32 values [..., 576] of cache rows, in 16 or 4 bits"""
    if rows.dtype != torch.uint8:
        return rows.float()
    byte = rows[..., :LAT // 2]
    code = st["code"][torch.stack([byte & 15, byte >> 4], dim=-1).int()].unflatten(-2, (LAT // GROUP, GROUP // 2))
    lat = code * st["power"][rows[..., LAT // 2:LAT // 2 + LAT // GROUP].int()][..., None, None]
    pe = rows[..., LAT // 2 + LAT // GROUP:].contiguous().view(_dtype(st)).float()
    return torch.cat([lat.flatten(-3), pe], dim=-1)


def _rows(st, table, n):
    """The first n rows of the table's sequences [B, n, 576] (behind their ends: any)"""
    t = torch.arange(n, device=DEV)
    page = st["page"]
    return _values(st, st["cache"][table[:, t // page].clamp(min=0).long(), (t % page)[None]])


def _scores(st, rows):
    """[B, S * H, n], -inf where a row does not see a token"""
    S, H, B, n = st["S"], st["H"], rows.shape[0], rows.shape[1]
    q = torch.cat([st["q_latent"], st["q_pe"]], dim=-1).float().view(B, S * H, ROW)
    z = torch.bmm(q, rows.transpose(1, 2).contiguous()) * SCALE
    sees = st["seq_lens"][:, None] - (S - 1 - torch.arange(S, device=DEV).repeat_interleave(H))[None]
    return z.masked_fill(torch.arange(n, device=DEV) >= sees[..., None], -math.inf)


def _softmax(s):
    """(exp(s - max), row sums, log-sum-exp); rows of -inf only give zeros and -inf."""
    m = s.amax(dim=-1, keepdim=True)
    e = torch.exp(s - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    l = e.sum(dim=-1, keepdim=True)
    return e, l, (torch.log(l) + m).squeeze(-1)


def _plain_tokens(st):
    cache, cu = st["cache"], st["cu"].long()
    cache.view(-1, ROW4)[st["slots"]] = _rounded(st["latent"], st["k_pe"], st["power"])
    t = torch.arange(st["total"], device=DEV)
    n = torch.searchsorted(cu, t, right=True) - 1
    j = t - cu[n]
    rows = cache[st["table"][n, j // st["page"]].long(), j % st["page"]]
    return _values(st, rows).to(st["latent"].dtype)


def _plain_decode(st):
    S, H, T = st["S"], st["H"], st["q_latent"].shape[0]
    rows = _rows(st, st["table"], st["most"])
    s = _scores(st, rows)
    P = st["prefix"]
    if P:
        head = _rows(st, st["prefix_table"][None], P)[0]
        q = torch.cat([st["q_latent"], st["q_pe"]], dim=-1).float().view(T * H, ROW)
        s = torch.cat([(q @ head.t().contiguous() * SCALE).view(*s.shape[:2], P), s], dim=-1)
    p, l, lse = _softmax(s)
    o = torch.bmm(p[..., P:].contiguous(), rows[..., :LAT].contiguous())
    if P:
        o += (p[..., :P].reshape(T * H, P) @ head[:, :LAT].contiguous()).view_as(o)
    return (o / torch.where(l == 0, torch.ones_like(l), l)).to(st["q_latent"].dtype).view(T, H, LAT), lse.view(T, H)


def _plain_weights(st):
    z = _scores(st, _rows(st, st["table"], st["most"]))
    lse = st["lse"].view(z.shape[0], -1, 1)
    w = torch.exp(torch.where(torch.isinf(lse), torch.full_like(z, -math.inf), z - lse))
    st["weights"][:, :st["most"]] += w.sum(dim=1)
    return st["weights"]


def _plain_evict(st):
    table, lens, refs, free, page = st["table"], st["seq_lens"], st["refs"], st["free"], st["page"]
    keep, recent, pages, width = st["keep"], st["recent"], st["refs"].numel(), st["table"].shape[1]
    W = width * page
    j, cols = torch.arange(W, device=DEV), torch.arange(width, device=DEV)
    n = lens.long()
    used = (n + page - 1) // page
    held = cols < used[:, None]
    at = table.clamp(min=0).long()
    # the tokens up to the end of the last page that others hold too stay
    fixed = ((cols + 1) * page * (held & (refs[at] > 1))).amax(dim=1)
    cut = (n > keep) & (fixed <= keep - recent)
    older = (n - recent)[:, None]
    free_to_go = (j >= fixed[:, None]) & (j < older)
    new = torch.where(cut, torch.full_like(n, keep), n)
    left = keep - recent
    for pool, mass in zip(st["pools"], st["masses"]):
        w = torch.where(j < fixed[:, None], math.inf, torch.where(free_to_go, mass, -math.inf))
        order = torch.sort(w, dim=1, descending=True, stable=True).indices[:, :left]
        stays = torch.zeros_like(w, dtype=torch.bool).scatter_(1, order, True)
        drop = ~stays & (j < left)
        move = stays & (j >= left)
        # the i-th place that is left gets the i-th token that has to move
        drops = torch.argsort((~drop).byte(), dim=1, stable=True)[:, :left]
        moves = torch.argsort((~move).byte(), dim=1, stable=True)[:, :left]
        some = cut[:, None] & (j[:left] < drop.sum(dim=1, keepdim=True))
        place = j.repeat(len(n), 1)
        place = torch.cat([place, place[:, :1]], dim=1).scatter_(1, torch.where(some, drops, W), moves)[:, :keep]
        place = torch.where((j[:keep] >= left) & cut[:, None], j[:keep] + (n - keep)[:, None], place)
        place, here = (torch.minimum(x, (n - 1)[:, None]) for x in (place, j[:keep].expand_as(place)))
        src, dst = (at.gather(1, x // page) * page + x % page for x in (place, here))
        flat = pool.view(pages * page, -1)
        flat[dst] = flat[src]
        moved = torch.cat([mass.gather(1, place), mass[:, keep:]], dim=1)
        moved = torch.where((j >= keep) & (j < n[:, None]), torch.zeros_like(moved), moved)
        mass.copy_(torch.where(cut[:, None], moved, mass))
    # pages behind the new ends given up, the highest first onto the stack
    first = (new + page - 1) // page
    gone = held & (cols >= first[:, None])
    given = torch.zeros(pages + 1, dtype=torch.int32, device=DEV)
    given.index_put_((torch.where(gone, at, torch.full_like(at, pages)).flatten(),), torch.ones(1, dtype=torch.int32, device=DEV),
                     accumulate=True)
    given = given[:pages]
    refs -= given
    mine = (given > 0) & (refs == 0)
    rank = torch.flip(torch.cumsum(torch.flip(mine.long(), [0]), 0), [0]) - 1 + st["num_free"].long()
    grown = torch.cat([free, free.new_zeros(1)])
    grown[torch.where(mine, rank, torch.full_like(rank, pages))] = torch.arange(pages, device=DEV).int()
    free.copy_(grown[:-1])
    st["num_free"] += mine.sum().int()
    table.masked_fill_(gone, -1)
    lens.copy_(new)
    return (table, lens, refs, free, st["num_free"], *st["masses"], *st["pools"])


# --------------------------------------------------------------------------------------------------------- own kernels
def _kda355():
    if "kda355" not in sys.modules:  # a program finds its package once, not at every call
        sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "eat-kernels_amd"))
    import kda355
    return kda355


def _own_run(st):
    kda355 = _kda355()
    op = st["op"]
    if op == "tokens":
        kda355.latent_append(st["latent"], st["k_pe"], st["cache"], st["slots"])
        return kda355.latent_gather(st["cache"], st["table"], st["cu"], st["out"])
    if op == "decode":
        lse = torch.empty(st["q_latent"].shape[:2], dtype=torch.float32, device=DEV)
        out = kda355.latent_decode(st["q_latent"], st["q_pe"], st["cache"], st["table"], st["seq_lens"], scale=SCALE, lse=lse,
                                   prefix_table=st.get("prefix_table"), prefix_len=st.get("prefix_len"))
        return out, lse
    if op == "weights":
        return kda355.latent_weights(st["q_latent"], st["q_pe"], st["cache"], st["table"], st["seq_lens"], st["lse"],
                                     st["weights"], scale=SCALE)
    kda355.evict_tokens(st["pools"], st["masses"], st["table"], st["seq_lens"], st["refs"], st["free"], st["num_free"],
                        st["rows"], st["keep"], st["recent"], st["page"])
    return (st["table"], st["seq_lens"], st["refs"], st["free"], st["num_free"], *st["masses"], *st["pools"])


def run(state):
    if state["op"] == "evict":
        state["books"].copy_(state["books0"])
        state["weights"].copy_(state["weights0"])
    if own:
        return _own_run(state)
    return {"tokens": _plain_tokens, "decode": _plain_decode, "weights": _plain_weights,
            "evict": _plain_evict}[state["op"]](state)


# --------------------------------------------------------------------------------------------------------------- work
def work(case):
    op, lens = case["op"], _ints(case["lens"])
    if op == "tokens":
        return {"bytes": (2 * ROW + ROW4) * (sum(_ints(case["new"])) + sum(lens)), "flops": 0}
    row = ROW4 if case.get("bits", 4) == 4 else 2 * ROW
    if op in ("decode", "weights"):
        S, H, P = case["S"], case["H"], case.get("prefix", 0)
        seen = sum(max(0, n - S + 1 + s) + P for n in lens for s in range(S))
        rows = len(lens) * S * H
        if op == "decode":
            return {"bytes": (sum(lens) + P) * row + 2 * rows * (ROW + LAT) + 4 * rows, "flops": 2 * H * seen * (ROW + LAT)}
        return {"bytes": sum(lens) * (row + 8) + rows * (2 * ROW + 4), "flops": 2 * H * seen * ROW}
    # of the older tokens a share of 1 - d stays, and as many leave the first places as are taken from behind them
    keep, recent, total = case["keep"], case["recent"], 0
    for n in lens:
        if n > keep:
            d = (n - keep) / (n - recent)
            total += 4 * (n - recent) + int((keep - recent) * d + recent) * (2 * row + 8)
    width = max(-(-n // case["page"]) for n in lens)
    return {"bytes": case["layers"] * total + 8 * len(lens) * width, "flops": 0}


# ------------------------------------------------------------------------------------------------------------ 64 bits
def _token_rows(case, st, pages_of, n):
    """Token rows 0 .. n - 1 as float64 values."""
    t = torch.arange(n, device=DEV)
    rows = st["cache"].reshape(-1, st["cache"].shape[2])[pages_of.long()[t // case["page"]] * case["page"] + t % case["page"]]
    if rows.dtype != torch.uint8:
        return rows.double()
    x = torch.empty(n, ROW, dtype=torch.float64, device=DEV)
    for half in (0, 1):
        c = (rows[:, :256].long() >> (4 * half)) & 15
        two = c & 7  # 2-bit exponent, 1-bit fraction
        size = torch.where(two < 2, two * 0.5, (1 + (two & 1) * 0.5) * (1 << (two >> 1)).double() * 0.5)
        x[:, half:512:2] = torch.where(c > 7, -size, size)
    b = rows[:, 256:272].double()
    x[:, :512] *= torch.exp2(b - 127).repeat_interleave(32, dim=1)
    x[:, 512:] = rows[:, 272:].clone().view(_dtype(case)).double()
    return x


def _nearest(x, dtype):
    """float64 rows as 4 bits hold them, by distance to every value that there is."""
    sizes = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=DEV)
    g = x.reshape(-1, 16, 32)
    top = g.abs().amax(dim=2)
    e = torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top)))) - 2
    e = torch.where(top > 0, e, torch.full_like(e, -1000.0))
    e = torch.where(top > 7 * torch.exp2(e), e + 1, e).clamp(min=-125 if dtype == torch.bfloat16 else -23)
    unit = torch.exp2(e)[:, :, None]
    y = g.abs() / unit
    best, at = torch.zeros_like(y), torch.full_like(y, math.inf)
    for k in (0, 2, 4, 6, 1, 3, 5, 7):  # the even ones first: an odd one has to be nearer
        d = (y - sizes[k]).abs()
        best, at = torch.where(d < at, sizes[k], best), torch.minimum(d, at)
    return (torch.where(g < 0, -best, best) * unit).reshape(x.shape)


def exact(case, seed):
    """The definitions in float64: values to the nearest of their group; o = sum_j w_j c_j / sum_j w_j over the visible
    tokens, w_j = e^(z_j), lse = log sum w_j; weights increased by the sums of e^(z_j - lse).  Evicting moves values."""
    if case["op"] == "evict" or work(case)["flops"] > 8.0e12:
        return None
    st = prepare(case, seed)
    lens, page = _ints(case["lens"]), case["page"]
    if case["op"] == "tokens":
        out, at = [], 0
        flat = torch.cat([_nearest(st["latent"].double(), st["latent"].dtype), st["k_pe"].double()], dim=1)
        for n, (length, k) in enumerate(zip(lens, _ints(case["new"]))):
            rows = _token_rows(case, st, st["table"][n], length)
            rows[length - k:] = flat[at:at + k]
            at += k
            out.append(rows)
        return torch.cat(out)
    S, H, P = case["S"], case["H"], case.get("prefix", 0)
    T = st["q_latent"].shape[0]
    o = torch.zeros(T, H, LAT, dtype=torch.float64, device=DEV)
    z = torch.full((T, H), -math.inf, dtype=torch.float64, device=DEV)
    head = _token_rows(case, st, st["prefix_table"], P) if P else o.new_zeros(0, ROW)
    sums = st["weights"].double() if case["op"] == "weights" else None
    for n, length in enumerate(lens):
        rows = torch.cat([head, _token_rows(case, st, st["table"][n], length)])
        for s in range(S):
            seen = P + max(0, length - (S - 1 - s))
            if seen == 0:
                continue
            t = n * S + s
            x = st["q_latent"][t].double() @ rows[:seen, :LAT].T + st["q_pe"][t].double() @ rows[:seen, LAT:].T
            x = x / math.sqrt(192)
            if sums is not None:
                sums[n, :seen] += torch.exp(x - st["lse"][t].double()[:, None]).sum(dim=0)
                continue
            z[t] = torch.logsumexp(x, dim=1)
            o[t] = torch.exp(x - z[t][:, None]) @ rows[:seen, :LAT]
    return (o, z) if sums is None else sums
