"""Timed cases of the operators for several continuations of a prompt over a paged cache: attention that reads a
common prefix once, the selection of beams, forking, compacting and copying of pages.

``listed()`` are fixed cases, ``draw(rng)`` gives more of the same ranges, ``prepare(case, seed)`` the inputs
that a program holds before the call, ``run(state)`` one pass, ``work(case)`` what the pass cannot do without and
``exact(case, seed)`` the same outputs in 64 bits. With ``own`` false, ``run`` computes the operators from
elementary torch operations; with ``own`` true it calls this package.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
NEG_INF = float("-inf")


def listed():
    shared = dict(op="shared", dtype="bf16", H=16, Hk=4, d=128, page=16, window=0, softcap=0.0, slopes=False)
    beam = dict(op="beam", dtype="bf16", done=0)
    fork = dict(op="fork", page=16)
    copy = dict(op="copy", dtype="bf16", Hk=4, d=128, page=16, gaps=True)
    compact = dict(op="compact", page=16)
    return [
        # the beams of one short prompt: latency
        dict(shared, name="shared short", groups=1, B=4, prefix=300, tail=40, H=8, Hk=8, d=64, dtype="fp16"),
        # a batch of beam searches over documents of different lengths, capped scores
        dict(shared, name="shared beams", groups=9, B=67, prefix=4099, tail=300, softcap=30.0),
        # many requests behind one long system prompt: the matrix product's end
        dict(shared, name="shared prompt", groups=1, B=256, prefix=8192, tail=200, page=64),
        # one search of four beams: latency
        dict(beam, name="beam one search", G=1, W=4, k=4, V=32000),
        # wide beams over a catalogue of items, an odd number of them, logits in fp32
        dict(beam, name="beam wide", G=4, W=50, k=50, V=10007, dtype="fp32", done=5),
        # a batch of searches over a large vocabulary; twice the beams, so that as many can go on as end
        dict(beam, name="beam batch", G=64, W=8, k=16, V=128000, done=7),
        # one search's step: latency
        dict(fork, name="fork one search", groups=1, W=4, longest=300, drop=0),
        # a batch of searches with long prompts, some of them ended and freed
        dict(fork, name="fork batch", groups=64, W=8, longest=8192, drop=9),
        # the last pages of a step's forked beams, one row in two without a copy
        dict(copy, name="copy forked", n=67, d=64),
        # a cache's pages moved together
        dict(copy, name="copy many", n=2000, Hk=8, page=64, dtype="fp16", gaps=False),
        # a small cache
        dict(compact, name="compact small", N=8, longest=500, spare=30),
        # a large cache, a third of it free in holes
        dict(compact, name="compact large", N=500, longest=4099, spare=20000),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    op = rng.choice(["shared", "shared", "shared", "beam", "beam", "fork", "copy", "compact"])
    page = rng.choice([8, 16, 32, 64, 128])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "shared":
        Hk, ratio = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 8])
        B = _log(rng, 1, 256)
        longest = min(16384, 2400000 // (B * Hk))
        return dict(op=op, dtype=dtype, H=min(Hk * ratio, max(16 // Hk, 1) * Hk), Hk=Hk, d=rng.choice([64, 128]), B=B, groups=min(B, _log(rng, 1, 40)),
                    prefix=_log(rng, 1, longest), tail=_log(rng, 1, 300), page=page, window=rng.choice([0, 0, _log(rng, 1, 8192)]),
                    softcap=rng.choice([0.0, 0.0, 20.0, 50.0]), slopes=rng.random() < 0.3)
    if op == "beam":
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        G, W = _log(rng, 1, 64), _log(rng, 1, 64)
        V = _log(rng, 50, min(151936, 60000000 // (G * W)))
        return dict(op=op, dtype=dtype, G=G, W=W, V=V, k=min(64, V, rng.choice([1, W, W, 2 * W])), done=rng.choice([0, 3, 10]))
    if op == "fork":
        W = _log(rng, 1, 32)
        return dict(op=op, groups=_log(rng, 1, 512 // W), W=W, longest=_log(rng, 1, 8192), page=page, drop=rng.choice([0, 2, 9]))
    if op == "copy":
        Hk, d = rng.choice([1, 2, 4, 8]), rng.choice([64, 128])
        return dict(op=op, dtype=dtype, Hk=Hk, d=d, page=page, n=_log(rng, 1, min(4000, 120000000 // (Hk * d * page))), gaps=rng.random() < 0.5)
    return dict(op=op, N=_log(rng, 1, 500), longest=_log(rng, 1, 4099), spare=_log(rng, 1, 20000), page=page)


# sizes that follow from a case alone: what a scheduler's host side would hold

def _shared_lens(c):
    """(offsets of the groups, prefix lengths, lengths): prompts of different lengths, each with some requests; the
    last of several groups has an ended request, and the last request of many belongs to none."""
    B, G = c["B"], c["groups"]
    r = random.Random(B * 131 + G * 7 + c["prefix"])
    most = B - 1 if B > 8 and G < B else B
    cuts = sorted(r.sample(range(1, most), G - 1)) if G > 1 else []
    cu = [0] + cuts + [most]
    prefix = [c["prefix"]] + [r.randint((c["prefix"] + 1) // 2, c["prefix"]) for _ in range(G - 1)]
    lens = []
    for g in range(G):
        lens += [prefix[g] + r.randint(1, c["tail"]) for _ in range(cu[g + 1] - cu[g])]
    lens += [r.randint(1, c["tail"]) for _ in range(B - most)]
    if G > 3:
        lens[most - 1] = 0
    return cu, prefix, lens


def _row_lens(c):
    """Lengths of the rows before a fork: a search's beams are equally long."""
    r = random.Random(c["groups"] * 17 + c["W"] + c["longest"] * 3)
    lens = [c["longest"]] + [r.randint(1, c["longest"]) for _ in range(c["groups"] - 1)]
    return [n for n in lens for _ in range(c["W"])]


def _fork_sizes(c):
    """(columns, pages): searches whose beams share their prompts' pages, three quarters of a search's."""
    M = -(-c["longest"] // c["page"]) + 1
    pages = 0
    for n in _row_lens(c)[::c["W"]]:
        held = -(-n // c["page"])
        pages += held * 3 // 4 + c["W"] * (held - held * 3 // 4)
    return M, pages + 2 * c["groups"] * c["W"] + 5


def _compact_lens(c):
    r = random.Random(c["N"] * 31 + c["longest"] + c["spare"])
    return [c["longest"]] + [r.randint(0, c["longest"]) for _ in range(c["N"] - 1)]


# inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _slopes(H):
    """Geometric distance slopes, one for each head."""
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], dtype=torch.float32, device="cuda")


def _numbered(wanted, M, ids):
    """A table [rows, M]: the first wanted[r] entries of row r are the next of ids, the others -1."""
    at = torch.cumsum(wanted, 0) - wanted
    col = torch.arange(M, device="cuda")[None]
    nth = (at[:, None] + col).clamp_max(ids.numel() - 1)
    return torch.where(col < wanted[:, None], ids[nth], torch.full_like(ids[nth], -1))


def _beam_inputs(c, g):
    """Logits as a language model's: a bulk of unlikely words, forty likely ones or a tenth of a small vocabulary."""
    G, W, V = c["G"], c["W"], c["V"]
    x = torch.randn(G, W, V, generator=g, device="cuda") * 2.0
    strong = max(1, min(40, V // 10))
    bins = V // strong
    where = torch.randint(0, bins, (G, W, strong), generator=g, device="cuda") + bins * torch.arange(strong, device="cuda")
    lift = 6.0 + 3.0 * torch.randn(G, W, strong, generator=g, device="cuda")
    x.scatter_(2, where, lift + torch.rand(G, W, 1, generator=g, device="cuda") * 4.0)
    scores = -20.0 * torch.rand(G, W, generator=g, device="cuda")
    done = (torch.rand(G, W, generator=g, device="cuda") * 100 < c["done"]) if c["done"] else None
    return dict(logits=x.to(DTYPES[c["dtype"]]), scores=scores, k=c["k"], finished=done, eos=min(2, V - 1))


def _shared_inputs(c, g):
    dt, H, Hk, d, page, B = DTYPES[c["dtype"]], c["H"], c["Hk"], c["d"], c["page"], c["B"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dt)

    cu, prefix, lens = _shared_lens(c)
    M = -(-max(lens + prefix) // page)
    group = [next((i for i in range(c["groups"]) if cu[i] <= b < cu[i + 1]), -1) for b in range(B)]
    whole = [prefix[i] // page if i >= 0 else 0 for i in group]   # pages that a group's requests share
    held = [-(-n // page) for n in lens]
    P = sum(p // page for p in prefix) + sum(max(h - w, 0) for h, w in zip(held, whole)) + 3
    ids = torch.randperm(P, generator=g, device="cuda").int()
    common = _numbered(_int32([p // page for p in prefix]).long(), M, ids)
    mine = _numbered(_int32([max(h - w, 0) for h, w in zip(held, whole)]).long(), M, ids[sum(p // page for p in prefix):])
    col = torch.arange(M, device="cuda")[None]
    w = _int32(whole).long()[:, None]
    table = torch.where(col < w, common[_int32(group).long().clamp_min(0)], mine.gather(1, (col - w).clamp_min(0)))
    k_cache, v_cache = normal(P, Hk, page, d), normal(P, Hk, page, d)
    for i in range(c["groups"]):   # a prompt's last, partly filled page: each request has its copy
        rest, a, b = prefix[i] % page, cu[i], cu[i + 1]
        if rest and b > a:
            rows = table[a:b, prefix[i] // page].long()
            rows = rows[rows >= 0]
            for cache in (k_cache, v_cache):
                cache[rows, :, :rest] = cache[rows[:1], :, :rest]
    return dict(q=normal(B, H, d), k_cache=k_cache, v_cache=v_cache, block_table=table, kv_lens=_int32(lens), cu_groups=_int32(cu),
                prefix_lens=_int32(prefix), scale=d ** -0.5, softcap=c["softcap"], window=c["window"], slopes=_slopes(H) if c["slopes"] else None)


def _fork_inputs(c, g):
    page, W, G = c["page"], c["W"], c["groups"]
    lens = _row_lens(c)
    M, P = _fork_sizes(c)
    ids = torch.randperm(P, generator=g, device="cuda").int()
    held = [-(-n // page) for n in lens]
    first = [h * 3 // 4 for h in held]   # whole pages of the prompt: the beams share them
    common = _numbered(_int32(first[::W]).long(), M, ids)
    mine = _numbered(_int32([h - f for h, f in zip(held, first)]).long(), M, ids[sum(first[::W]):])
    col = torch.arange(M, device="cuda")[None]
    f = _int32(first).long()[:, None]
    group = torch.arange(G * W, device="cuda") // W
    table = torch.where(col < f, common[group], mine.gather(1, (col - f).clamp_min(0)))
    parents = group * W + torch.randint(0, W, (G * W,), generator=g, device="cuda")   # as a selection gives them
    if c["drop"]:
        ended = torch.rand(G, generator=g, device="cuda") * 100 < c["drop"]
        parents = torch.where(ended[group], torch.full_like(parents, -1), parents)
    return dict(block_table=table, seq_lens=_int32(lens), parents=parents.int(), page_size=page, num_pages=P)


def _copy_inputs(c, g):
    n = c["n"]
    P = 2 * n + 3

    def normal():
        return torch.randn(P, c["Hk"], c["page"], c["d"], generator=g, device="cuda", dtype=torch.float32).to(DTYPES[c["dtype"]])

    ids = torch.randperm(P, generator=g, device="cuda").int()
    src, dst = ids[:n].clone(), ids[n:2 * n].clone()
    if c["gaps"] and n > 1:
        gone = torch.arange(n, device="cuda") % 2 == 1
        src[gone] = -1
        dst[gone] = -1
    return dict(k_cache=normal(), v_cache=normal(), src=src, dst=dst)


def _compact_inputs(c, g):
    lens, page = _compact_lens(c), c["page"]
    held = _int32([-(-n // page) for n in lens]).long()
    M, used = -(-c["longest"] // page), sum(-(-n // page) for n in lens)
    ids = torch.randperm(used + c["spare"], generator=g, device="cuda").int()
    return dict(block_table=_numbered(held, M, ids), seq_lens=_int32(lens), page_size=page, num_pages=used + c["spare"])


MAKE = {"shared": _shared_inputs, "beam": _beam_inputs, "fork": _fork_inputs, "copy": _copy_inputs, "compact": _compact_inputs}


def prepare(case, seed):
    return case["op"], MAKE[case["op"]](case, _gen(seed))


# plain forms

def _attend(s, v):
    """softmax over the last axis of scores that hold -inf where hidden, times v; rows that see nothing give 0."""
    top = s.amax(dim=-1, keepdim=True)
    e = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = e.sum(dim=-1, keepdim=True)
    return torch.matmul(e, v) / torch.where(total == 0, torch.ones_like(total), total)


def _shared(q, k_cache, v_cache, block_table, kv_lens, cu_groups, prefix_lens, scale, softcap, window, slopes):
    B, H, d = q.shape
    P, Hk, page, _ = k_cache.shape
    b, j = torch.arange(B, device=q.device), torch.arange(block_table.shape[1] * page, device=q.device)
    g = torch.searchsorted(cu_groups.long(), b, right=True) - 1
    inside = (g >= 0) & (g < prefix_lens.numel())
    g = g.clamp(0, max(prefix_lens.numel() - 1, 0))
    prefix = torch.where(inside, prefix_lens.long()[g], torch.zeros_like(b))
    row = torch.where(j[None] < prefix[:, None], cu_groups.long()[g][:, None], b[:, None])
    entry = block_table[row, (j // page)[None].expand(B, -1)].long()
    at, rest = entry.clamp_min(0), (j % page)[None].expand(B, -1)
    k, v = (x[at, :, rest].transpose(1, 2).float() for x in (k_cache, v_cache))
    back = kv_lens.long()[:, None] - 1 - j[None]   # distance from the last token, which asks
    seen = (back >= 0) & (entry >= 0) & (entry < P)
    if window:
        seen = seen & (back < window)
    s = torch.matmul(q.float().view(B, Hk, -1, d), k.transpose(2, 3)) * scale
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    if slopes is not None:
        s = s - slopes.view(1, Hk, -1, 1) * back[:, None, None].float()
    return _attend(s.masked_fill(~seen[:, None, None], NEG_INF), v).view(B, H, d).to(q.dtype)


def _beam(logits, scores, k, finished, eos):
    G, W, V = logits.shape
    x = logits.double()   # the order of neighbours is lost in 32 bits
    top = x.amax(dim=-1, keepdim=True)
    s = x - (top + torch.log(torch.exp(x - top).sum(dim=-1, keepdim=True))) + scores.double()[..., None]
    if finished is not None:
        only = torch.full_like(s, NEG_INF)
        only[..., eos] = scores.double()
        s = torch.where(finished[..., None], only, s)
    s = s.view(G, W * V)
    index = torch.arange(W * V, device=s.device)
    best, where = [], []
    for _ in range(k):   # one after the other, the lowest index first among equals
        top = s.amax(dim=-1, keepdim=True)
        at = torch.where(s == top, index, torch.full_like(index, W * V)).amin(dim=-1, keepdim=True)
        best.append(top)
        where.append(at)
        s = s.scatter(1, at, NEG_INF)
    best, where = torch.cat(best, 1), torch.cat(where, 1)
    real = best > NEG_INF
    parents = torch.arange(G, device=s.device)[:, None] * W + where // V
    return best.float(), torch.where(real, where % V, -1).int(), torch.where(real, parents, -1).int()


def _held(block_table, lens, page, num_pages):
    """(columns' whole pages, the pages as indices with num_pages for none)."""
    col = torch.arange(block_table.shape[1], device=lens.device)[None]
    ok = (block_table >= 0) & (block_table < num_pages) & (col < (lens + page - 1)[:, None] // page)
    return ok & (col < lens[:, None] // page), torch.where(ok, block_table.long(), num_pages), ok


def _marked(pages, num_pages):
    marks = torch.zeros(num_pages + 1, dtype=torch.bool, device=pages.device)
    marks[pages.reshape(-1)] = True
    return marks[:num_pages]


def _listed_pages(free):
    """The marked pages in ascending order, -1 behind them, and how many there are."""
    n = free.numel()
    order = torch.argsort((~free).int(), stable=True)
    count = free.sum()
    return torch.where(torch.arange(n, device=free.device) < count, order, -1), count


def _fork(block_table, seq_lens, parents, page_size, num_pages):
    (N, M), R = block_table.shape, parents.numel()
    real = (parents >= 0) & (parents < N)
    up = parents.long().clamp(0, N - 1)
    lens = torch.where(real, seq_lens.long()[up].clamp(0, M * page_size), 0)
    whole, pages, ok = _held(block_table[up], lens, page_size, num_pages)
    col = torch.arange(M, device=lens.device)[None]
    last = (lens // page_size).clamp_max(M - 1)[:, None]
    part = torch.where((lens % page_size != 0)[:, None], pages.gather(1, last), num_pages)[:, 0]
    i = torch.arange(R, device=lens.device)
    firsts = torch.full((num_pages + 1,), R, dtype=torch.int64, device=lens.device).scatter_reduce(0, part, i, "amin")
    full = _marked(torch.where(whole, pages, num_pages), num_pages + 1)
    mine = (firsts[part] == i) & ~full[part]
    wants = (part < num_pages) & ~mine
    free, count = _listed_pages(~_marked(pages, num_pages))
    nth = torch.cumsum(wants.long(), 0) - 1
    has = wants & (nth < count)
    dst = torch.where(has, free[nth.clamp(0, num_pages - 1)], -1)
    table = torch.where(ok, pages, -1)
    table = torch.where((col == last) & wants[:, None], dst[:, None], table)
    taken = has.sum()
    free = free.gather(0, (torch.arange(num_pages, device=lens.device) + taken).clamp_max(num_pages - 1))
    free = torch.where(torch.arange(num_pages, device=lens.device) < count - taken, free, -1)
    counts = torch.stack([count - taken, taken, wants.sum() - taken])
    return table.int(), lens.int(), torch.where(has, part, -1).int(), dst.int(), free.int(), counts.int()


def _compact(block_table, seq_lens, page_size, num_pages):
    N, M = block_table.shape
    lens = seq_lens.long().clamp(0, M * page_size)
    _, pages, ok = _held(block_table, lens, page_size, num_pages)
    used = _marked(pages, num_pages)
    page = torch.arange(num_pages, device=lens.device)
    count = used.sum()
    move, nmove = _listed_pages(used & (page >= count))
    hole, _ = _listed_pages(~used & (page < count))
    half = num_pages // 2
    remap = torch.where(used & (page < count), page, -1)
    remap = torch.cat([remap, remap.new_full((1,), -1)])
    remap[torch.where(move >= 0, move, num_pages)] = torch.where(move >= 0, hole, -1)
    free = torch.where(page + count < num_pages, page + count, -1)
    table = torch.where(ok, remap[pages], -1)
    return (table.int(), move[:half].int(), torch.where(move >= 0, hole, -1)[:half].int(), remap[:num_pages].int(), free.int(),
            torch.stack([count, nmove]).int())


def _copy(k_cache, v_cache, src, dst):
    P = k_cache.shape[0]
    ok = (src >= 0) & (src < P) & (dst >= 0) & (dst < P)
    a, b = src[ok].long(), dst[ok].long()
    k_cache[b] = k_cache[a]
    v_cache[b] = v_cache[a]
    return k_cache, v_cache


PLAIN = {"shared": _shared, "beam": _beam, "fork": _fork, "copy": _copy, "compact": _compact}


def run(state):
    op, x = state
    if not own:
        return PLAIN[op](**x)
    from custom_ops_amd import ops

    if op == "shared":
        return ops.mha_shared_decode(x["q"], x["k_cache"], x["v_cache"], x["block_table"], x["kv_lens"], x["cu_groups"], x["prefix_lens"],
                                     scale=x["scale"], softcap=x["softcap"], window=x["window"], slopes=x["slopes"])
    if op == "beam":
        return ops.beam_select(x["logits"], x["scores"], x["k"], finished=x["finished"], eos=x["eos"])
    if op == "fork":
        return ops.paged_fork(x["block_table"], x["seq_lens"], x["parents"], x["page_size"], x["num_pages"])
    if op == "compact":
        return ops.paged_compact(x["block_table"], x["seq_lens"], x["page_size"], x["num_pages"])
    ops.paged_copy(x["k_cache"], x["v_cache"], x["src"], x["dst"])
    return x["k_cache"], x["v_cache"]


# what a pass cannot do without

def work(case):
    c = case
    if c["op"] == "shared":
        cu, prefix, lens = _shared_lens(c)
        H, Hk, d, B = c["H"], c["Hk"], c["d"], c["B"]
        lo = [max(0, n - c["window"]) if c["window"] else 0 for n in lens]
        keys = 0
        for g, p in enumerate(prefix):
            rows = [b for b in range(cu[g], cu[g + 1]) if lens[b] > 0]
            keys += max([0] + [p - lo[b] for b in rows])
            keys += sum(max(0, lens[b] - max(lo[b], p)) for b in rows)
        keys += sum(lens[b] - lo[b] for b in range(cu[-1], B))
        pairs = sum(n - a for n, a in zip(lens, lo))
        return {"bytes": 2.0 * d * (2 * Hk * keys + 2 * H * B) + 4.0 * (keys // c["page"]), "flops": 4.0 * H * d * pairs}
    if c["op"] == "beam":
        rows = c["G"] * c["W"]
        return {"bytes": float(BYTES[c["dtype"]]) * rows * c["V"] + 5.0 * rows + 12.0 * c["G"] * c["k"], "flops": 3.0 * rows * c["V"]}
    if c["op"] == "fork":
        M, P = _fork_sizes(c)
        entries = sum(-(-n // c["page"]) for n in _row_lens(c))
        R = c["groups"] * c["W"]
        return {"bytes": 4.0 * (entries + R * M + P + 5 * R + 3), "flops": 0.0}
    if c["op"] == "compact":
        lens = _compact_lens(c)
        used = sum(-(-n // c["page"]) for n in lens)
        P = used + c["spare"]
        return {"bytes": 4.0 * (used + c["N"] * (-(-c["longest"] // c["page"])) + 2 * (P // 2) + 2 * P + c["N"] + 2), "flops": 0.0}
    n = (c["n"] + 1) // 2 if c["gaps"] else c["n"]
    return {"bytes": 2.0 * 2 * n * 2.0 * c["Hk"] * c["page"] * c["d"] + 8.0 * c["n"], "flops": 0.0}


# the same outputs in 64 bits, from the definitions

def exact(case, seed):
    c = case
    if c["op"] in ("fork", "compact"):
        return None   # whole numbers: the plain form is exact
    x = prepare(c, seed)[1]
    if c["op"] == "copy":
        origin = torch.arange(x["k_cache"].shape[0], device="cuda")   # where a page's values come from
        real = x["dst"] >= 0
        origin[x["dst"][real].long()] = x["src"][real].long()
        return x["k_cache"].double()[origin], x["v_cache"].double()[origin]
    if c["op"] == "beam":
        logits, scores, k = x["logits"], x["scores"].double(), c["k"]
        out = []
        for g in range(c["G"]):
            rows = []
            for w in range(c["W"]):
                if x["finished"] is not None and bool(x["finished"][g, w]):
                    rows.append(scores[g, w:w + 1])
                else:
                    rows.append(torch.log_softmax(logits[g, w].double(), dim=0).topk(min(k, c["V"])).values + scores[g, w])
            every = torch.cat(rows)
            best = every.topk(min(k, every.numel())).values
            out.append(torch.cat([best, best.new_full((k - best.numel(),), NEG_INF)]))
        return torch.stack(out), None, None   # tokens and parents are whole numbers
    cu, prefix, lens = _shared_lens(c)
    H, Hk, d = c["H"], c["Hk"], c["d"]
    out = torch.zeros(c["B"], H, d, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        if n == 0:
            continue
        pages = x["block_table"][b, :-(-n // c["page"])].long()
        first = max(0, n - c["window"]) if c["window"] else 0
        dist = (n - 1 - torch.arange(first, n, device="cuda")).double().view(1, 1, -1)
        k, v = (x[m][pages].transpose(0, 1).reshape(Hk, -1, d)[:, first:n].double() for m in ("k_cache", "v_cache"))
        s = (x["q"][b].double().view(Hk, -1, d) @ k.transpose(1, 2).contiguous()) * d ** -0.5
        if c["softcap"]:
            s = torch.tanh(s / c["softcap"]) * c["softcap"]
        if c["slopes"]:
            s = s - dist * x["slopes"].double().view(Hk, -1, 1)
        p = torch.exp(s - s.max(dim=-1, keepdim=True).values)
        out[b] = ((p @ v) / p.sum(dim=-1, keepdim=True)).reshape(H, d)
    return out
