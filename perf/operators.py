"""Timed cases of the serving operators: attention over packed sequences, one-token attention over a paged
key-value cache, rotary positions with the write into that cache, and the cache's layout on the device.

``listed()`` are fixed cases, ``draw(rng)`` gives more of the same ranges, ``prepare(case, seed)`` the inputs
that a program holds before the call, ``run(state)`` one pass, ``work(case)`` what the pass cannot do without and
``exact(case, seed)`` the same outputs in 64 bits. With ``own`` false, ``run`` computes the operators from
elementary torch operations in fp32; with ``own`` true it calls this package.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
NEG_INF = float("-inf")


def listed():
    packed = dict(op="packed", dtype="bf16", H=16, Hk=4, d=128, docs=1, pad=0, causal=True, window=0, softcap=0.0,
                  slopes=False, prefix=0)
    decode = dict(op="decode", dtype="bf16", H=16, Hk=4, d=128, page=16, window=0, softcap=0.0, slopes=False)
    rope = dict(op="rope", dtype="bf16", H=16, Hk=4, d=128, rot=128, interleaved=False, page=16, far=8192)
    layout = dict(op="layout", page=16)
    return [
        # one long prompt, grouped heads: the matrix-product-bound end
        dict(packed, name="packed one prompt", T=8192),
        # a ragged batch of documents in fp16 with a distance bias, a padded tail behind the last
        dict(packed, name="packed documents bias", T=8000, docs=24, pad=77, dtype="fp16", H=8, Hk=8, d=64, slopes=True),
        # capped scores, a sliding window and a prefix that every row sees
        dict(packed, name="packed capped window", T=4099, docs=3, H=16, Hk=8, softcap=50.0, window=1000, prefix=130),
        # a short prompt: latency
        dict(packed, name="packed short", T=131, docs=2, H=8, Hk=8, d=64),
        # one request with a short context: latency
        dict(decode, name="decode one short", B=1, longest=200, H=8, Hk=8, d=64, dtype="fp16"),
        # a ragged batch in service
        dict(decode, name="decode ragged batch", B=32, longest=8192),
        # one request with a very long context, capped scores
        dict(decode, name="decode one long", B=1, longest=131072, page=64, H=32, softcap=30.0),
        # a large batch without shared heads, a distance bias and a window
        dict(decode, name="decode window bias", B=100, longest=4099, H=16, Hk=16, d=64, window=2048, slopes=True, page=32),
        # a decoding step's tokens
        dict(rope, name="rope step", T=33),
        # a prompt's tokens: neighbours paired, half of the head, far positions
        dict(rope, name="rope prompt", T=8191, dtype="fp16", rot=64, interleaved=True, page=64, far=1000000, Hk=8),
        # a decoding step: one token for each request
        dict(layout, name="layout step", N=256, longest=8192, new=1),
        # new prompts beside running requests, a page budget that runs out
        dict(layout, name="layout prompts", N=67, longest=4099, new=1500, page=32),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    op = rng.choice(["packed", "packed", "decode", "decode", "rope", "layout"])
    dtype = rng.choice(["bf16", "fp16"])
    d = rng.choice([64, 128])
    Hk = rng.choice([1, 2, 4, 8])
    ratio = rng.choice([1, 2, 3, 4, 8])
    slopes, softcap = rng.random() < 0.3, rng.choice([0.0, 0.0, 20.0, 50.0])
    if op == "packed":
        H = min(Hk * ratio, 16 // Hk * Hk)
        causal = rng.random() < 0.8
        T = _log(rng, 1, 8192 if causal else 5700)
        return dict(op=op, dtype=dtype, H=H, Hk=Hk, d=d, T=T, docs=min(T, _log(rng, 1, 40)), pad=rng.choice([0, 0, 1, 50]),
                    causal=causal, window=rng.choice([0, 0, _log(rng, 1, 4096)]), softcap=softcap, slopes=slopes,
                    prefix=rng.choice([0, 0, _log(rng, 1, 500)]))
    if op == "decode":
        B = _log(rng, 1, 128)
        longest = _log(rng, 1, min(131072, 400000 // B))
        return dict(op=op, dtype=dtype, H=Hk * ratio, Hk=Hk, d=d, B=B, longest=longest, page=rng.choice([8, 16, 32, 64, 128]),
                    window=rng.choice([0, 0, _log(rng, 1, 8192)]), softcap=softcap, slopes=slopes)
    if op == "rope":
        return dict(op=op, dtype=dtype, H=min(Hk * ratio, 32), Hk=Hk, d=d, T=_log(rng, 1, 8192),
                    rot=rng.choice([d, d, d // 2, d // 4]), interleaved=rng.random() < 0.5, page=rng.choice([8, 16, 32, 64, 128]),
                    far=_log(rng, 100, 1000000))
    return dict(op=op, N=_log(rng, 1, 1000), longest=_log(rng, 1, 8192), new=_log(rng, 1, 2000), page=rng.choice([8, 16, 32, 64, 128]))


# sizes that follow from a case alone: what a scheduler's host side would hold

def _doc_lens(c):
    """Ragged lengths of a packed batch: the documents' sum is T, each has a token."""
    n, T = c["docs"], c["T"]
    r = random.Random(T * 31 + n)
    cuts = sorted(r.sample(range(1, T), n - 1)) if n > 1 else []
    return [b - a for a, b in zip([0] + cuts, cuts + [T])]


def _prefix_lens(c):
    return [c["prefix"] if i % 2 == 0 else c["prefix"] // 3 for i in range(c["docs"])]


def _kv_lens(c):
    """Cached lengths of a decoding batch: the first the longest, an empty one among many."""
    r = random.Random(c["B"] * 131 + c["longest"])
    lens = [c["longest"]] + [r.randint(1, c["longest"]) for _ in range(c["B"] - 1)]
    if c["B"] > 8:
        lens[5] = 0
    return lens


def _layout_lens(c):
    """(cached, new) lengths: decoding requests and, for longer steps, new prompts (cached 0) and idle ones (new 0)."""
    r = random.Random(c["N"] * 17 + c["longest"] * 3 + c["new"])
    cached, new = [], []
    for i in range(c["N"]):
        prompt = c["new"] > 1 and i % 3 == 0
        cached.append(0 if prompt else r.randint(0, c["longest"]))
        new.append(r.randint(1, c["new"]) if prompt else 0 if c["new"] > 1 and i % 7 == 1 else 1)
    return cached, new


def _layout_sizes(c):
    cached, new = _layout_lens(c)
    p = c["page"]
    grow = sum(-(-(a + b) // p) + (-a // p) for a, b in zip(cached, new))
    M = -(-(c["longest"] + c["new"]) // p)
    return M, max(1, grow - grow // 16), sum(new) + 5   # a 16th of the pages is missing


# inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _slopes(H):
    """Geometric distance slopes, one for each head."""
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], dtype=torch.float32, device="cuda")


def _cu(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return _int32(out)


def _inv_freq(rot):
    return torch.tensor([10000.0 ** (-2.0 * i / rot) for i in range(rot // 2)], dtype=torch.float64, device="cuda")


def _inputs(c, seed):
    g, op = _gen(seed), c["op"]
    if op == "layout":
        cached, new = _layout_lens(c)
        M, F, max_tokens = _layout_sizes(c)
        pool = c["N"] * M + F
        order = torch.randperm(pool, generator=g, device="cuda").int()
        col = torch.arange(M, device="cuda")[None]
        held = -(-_int32(cached) // c["page"])
        table = torch.where(col < held[:, None], order[F:].view(c["N"], M), torch.full_like(order[F:].view(c["N"], M), -1))
        return dict(seq_lens=_int32(cached), new_lens=_int32(new), block_table=table, free_pages=order[:F].contiguous(),
                    page_size=c["page"], max_tokens=max_tokens)
    dt, H, Hk, d = DTYPES[c["dtype"]], c["H"], c["Hk"], c["d"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dt)

    scores = dict(scale=d ** -0.5, softcap=c.get("softcap", 0.0), window=c.get("window", 0),
                  slopes=_slopes(H) if c.get("slopes") else None)
    if op == "packed":
        T = c["T"] + c["pad"]
        qkv = normal(T, H + 2 * Hk, d)   # views of one projection, as a block has them
        cu = _cu(_doc_lens(c))
        return dict(q=qkv[:, :H], k=qkv[:, H:H + Hk], v=qkv[:, H + Hk:], cu_q=cu, cu_k=cu, causal=c["causal"],
                    prefix_lens=_int32(_prefix_lens(c)) if c["prefix"] else None, **scores)
    page = c["page"]
    if op == "decode":
        lens = _kv_lens(c)
        M = -(-c["longest"] // page)
        held = [-(-n // page) for n in lens]
        P = sum(held) + 3
        ids = torch.randperm(P, generator=g, device="cuda").int()
        table = torch.full((c["B"], M), -1, dtype=torch.int32, device="cuda")
        at = _cu(held)[:-1].long()[:, None] + torch.arange(M, device="cuda")[None]
        mine = torch.arange(M, device="cuda")[None] < _int32(held)[:, None]
        table = torch.where(mine, ids[at.clamp_max(P - 1)], table)
        return dict(q=normal(c["B"], H, d), k_cache=normal(P, Hk, page, d), v_cache=normal(P, Hk, page, d), block_table=table,
                    kv_lens=_int32(lens), **scores)
    T = c["T"]
    P = -(-T // page) + 2
    qkv = normal(T, H + 2 * Hk, d)
    slots = torch.randperm(P * page, generator=g, device="cuda")[:T]
    if T > 8:
        slots[T // 2] = -1   # a token without a page
    first = torch.randint(0, max(1, c["far"] - T + 1), (1,), generator=g, device="cuda")
    return dict(q=qkv[:, :H], k=qkv[:, H:H + Hk], v=qkv[:, H + Hk:], positions=(first + torch.arange(T, device="cuda")).int(),
                inv_freq=_inv_freq(c["rot"]), slot_map=slots, k_cache=normal(P, Hk, page, d), v_cache=normal(P, Hk, page, d),
                interleaved=c["interleaved"], amplitude=1.0)


def prepare(case, seed):
    return case["op"], _inputs(case, seed)


# plain forms

def _attend(s, v):
    """softmax over the last axis of scores that hold -inf where hidden, times v; rows that see nothing give 0."""
    top = s.amax(dim=-1, keepdim=True)
    e = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = e.sum(dim=-1, keepdim=True)
    return torch.matmul(e, v) / torch.where(total == 0, torch.ones_like(total), total)


def _packed(q, k, v, cu_q, cu_k, causal, prefix_lens, scale, softcap, window, slopes):
    (Tq, H, d), (Tk, Hk, _) = q.shape, k.shape
    n = cu_q.numel() - 1
    iq, ik = (torch.arange(t, device=q.device) for t in (Tq, Tk))
    sq, sk = (torch.searchsorted(cu[1:].long(), i, right=True) for cu, i in ((cu_q, iq), (cu_k, ik)))
    lq, lk = cu_q[1:] - cu_q[:-1], cu_k[1:] - cu_k[:-1]
    ends = sq.clamp_max(n - 1)
    pq = (iq - cu_q[:-1].long()[ends] + (lk - lq).long()[ends])[:, None]   # a row's place among the keys
    pk = (ik - cu_k[:-1].long()[sk.clamp_max(n - 1)])[None]
    seen = pk <= pq if causal else pk == pk
    if window:
        seen = seen & ((pq - pk).abs() < window)
    if prefix_lens is not None:
        seen = seen | (pk < prefix_lens.long()[ends][:, None])
    seen = seen & (sq[:, None] == sk[None]) & (sq < n)[:, None]
    s = torch.matmul(q.float().transpose(0, 1).reshape(Hk, -1, d), k.float().permute(1, 2, 0)) * scale
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    s = s.view(H, Tq, Tk)
    if slopes is not None:
        s = s - slopes.view(H, 1, 1) * (pq - pk).abs().float()
    s = s.masked_fill(~seen, NEG_INF)
    return _attend(s.view(Hk, -1, Tk), v.float().transpose(0, 1)).view(H, Tq, d).transpose(0, 1).contiguous().to(q.dtype)


def _decode(q, k_cache, v_cache, block_table, kv_lens, scale, softcap, window, slopes):
    B, H, d = q.shape
    P, Hk, page, _ = k_cache.shape
    at = block_table.long().clamp_min(0)
    k, v = (x[at].transpose(1, 2).reshape(B, Hk, -1, d).float() for x in (k_cache, v_cache))
    j = torch.arange(k.shape[2], device=q.device)[None]
    back = kv_lens.long()[:, None] - 1 - j   # distance from the last token, which asks
    seen = (back >= 0) & (block_table >= 0).repeat_interleave(page, dim=1)
    if window:
        seen = seen & (back < window)
    s = torch.matmul(q.float().view(B, Hk, -1, d), k.transpose(2, 3)) * scale
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    if slopes is not None:
        s = s - slopes.view(1, Hk, -1, 1) * back[:, None, None].float()
    return _attend(s.masked_fill(~seen[:, None, None], NEG_INF), v).view(B, H, d).to(q.dtype)


def _rotate(x, cos, sin, interleaved):
    x, r = x.float(), cos.shape[-1]
    a, b = (x[..., 0:2 * r:2], x[..., 1:2 * r:2]) if interleaved else (x[..., :r], x[..., r:2 * r])
    turned = (a * cos - b * sin, b * cos + a * sin)
    turned = torch.stack(turned, dim=-1).flatten(-2) if interleaved else torch.cat(turned, dim=-1)
    return torch.cat([turned, x[..., 2 * r:]], dim=-1)


def _rope(q, k, v, positions, inv_freq, slot_map, k_cache, v_cache, interleaved, amplitude):
    angle = positions.double()[:, None, None] * inv_freq
    cos, sin = (amplitude * torch.cos(angle)).float(), (amplitude * torch.sin(angle)).float()
    qr, kr = (_rotate(x, cos, sin, interleaved).to(x.dtype) for x in (q, k))
    kept = slot_map >= 0
    page = k_cache.shape[2]
    where = slot_map[kept]
    k_cache[where // page, :, where % page] = kr[kept]
    v_cache[where // page, :, where % page] = v[kept]
    return qr, kr, k_cache, v_cache


def _layout(seq_lens, new_lens, block_table, free_pages, page_size, max_tokens):
    (N, M), F = block_table.shape, free_pages.numel()
    seq, new = seq_lens.long(), new_lens.long()
    total = seq + new
    held, wanted = (seq + page_size - 1) // page_size, (total + page_size - 1) // page_size
    need = wanted.clamp_max(M)
    grow = (need - held).clamp_min(0)
    at = torch.cumsum(grow, 0) - grow
    col = torch.arange(M, device=seq.device)[None]
    nth = at[:, None] + col - held[:, None]
    fresh = (col >= held[:, None]) & (col < need[:, None]) & (nth < F)
    table = torch.where(fresh, free_pages[nth.clamp(0, max(F - 1, 0))], torch.full_like(block_table, -1))
    table = torch.where((col < held[:, None]) & (col < need[:, None]), block_table, table)
    cu = torch.cat([torch.zeros_like(seq[:1]), torch.cumsum(new, 0)])
    t = torch.arange(max_tokens, device=seq.device)
    r = torch.searchsorted(cu[1:].contiguous(), t, right=True).clamp_max(N - 1)
    real = t < cu[N]
    pos = torch.where(real, seq[r] + t - cu[r], torch.zeros_like(t))
    page = pos // page_size
    entry = table[r, page.clamp_max(M - 1)].long()
    slot = torch.where(real & (page < M) & (entry >= 0), entry * page_size + pos % page_size, torch.full_like(t, -1))
    taken = grow.sum().clamp_max(F)
    counts = torch.stack([cu[N], taken, (wanted - held).clamp_min(0).sum() - taken])
    return total.int(), cu.int(), pos.int(), slot, table, counts.int()


PLAIN = {"packed": _packed, "decode": _decode, "rope": _rope, "layout": _layout}


def run(state):
    op, x = state
    if not own:
        return PLAIN[op](**x)
    from custom_ops_amd import ops

    if op == "packed":
        return ops.mha_packed_fwd(x["q"], x["k"], x["v"], x["cu_q"], x["cu_k"], causal=x["causal"], scale=x["scale"],
                                  softcap=x["softcap"], window=x["window"], slopes=x["slopes"], prefix_lens=x["prefix_lens"])
    if op == "decode":
        return ops.mha_paged_decode(x["q"], x["k_cache"], x["v_cache"], x["block_table"], x["kv_lens"], scale=x["scale"],
                                    softcap=x["softcap"], window=x["window"], slopes=x["slopes"])
    if op == "rope":
        q, k = ops.rope_paged_store(x["q"], x["k"], x["v"], x["positions"], x["inv_freq"], x["slot_map"], x["k_cache"],
                                    x["v_cache"], interleaved=x["interleaved"], amplitude=x["amplitude"])
        return q, k, x["k_cache"], x["v_cache"]
    return ops.paged_layout(x["seq_lens"], x["new_lens"], x["block_table"], x["free_pages"], x["page_size"], x["max_tokens"])


# what a pass cannot do without

def _row_range(c, i, n, prefix):
    """(visible keys of row i in a document of n, outside and inside the prefix)."""
    hi = i + 1 if c["causal"] else min(n, i + c["window"]) if c["window"] else n
    lo = max(0, i - c["window"] + 1) if c["window"] else 0
    p = min(prefix, n)
    return max(0, hi - max(lo, p)) + p


def work(case):
    c = case
    if c["op"] == "layout":
        M, F, max_tokens = _layout_sizes(c)
        cached, new = _layout_lens(c)
        grown = min(F, sum(-(-(a + b) // c["page"]) + (-a // c["page"]) for a, b in zip(cached, new)))
        held = sum(-(-a // c["page"]) for a in cached)
        return {"bytes": 4.0 * (4 * c["N"] + 4 + held + grown + c["N"] * M + 3 * max_tokens), "flops": 0.0}
    H, Hk, d = c["H"], c["Hk"], c["d"]
    if c["op"] == "packed":
        rows = 0
        for n, p in zip(_doc_lens(c), _prefix_lens(c)):
            rows += sum(_row_range(c, i, n, p) for i in range(n))
        return {"bytes": 2.0 * d * ((2 * H + 2 * Hk) * c["T"] + H * c["pad"]), "flops": 4.0 * H * d * rows}
    if c["op"] == "decode":
        keys = sum(min(n, c["window"]) if c["window"] else n for n in _kv_lens(c))
        return {"bytes": 2.0 * d * (2 * Hk * keys + 2 * H * c["B"]) + 4.0 * (keys // c["page"]), "flops": 4.0 * H * d * keys}
    stored = c["T"] - (1 if c["T"] > 8 else 0)
    return {"bytes": c["T"] * (2.0 * d * (2 * H + 2 * Hk + Hk) + 12) + 2.0 * d * 2 * Hk * stored + 4.0 * c["rot"],
            "flops": 3.0 * (H + Hk) * c["rot"] * c["T"]}


# the same outputs in 64 bits, from the definitions

def _exact_rows(q, k, v, scale, softcap, bias, seen):
    """One head's rows: softmax of the seen scores times v."""
    s = (q @ k.t().contiguous()) * scale
    if softcap:
        s = torch.tanh(s / softcap) * softcap
    if bias is not None:
        s = s + bias
    s = torch.where(seen, s, torch.full_like(s, NEG_INF))
    top = s.max(dim=1, keepdim=True).values
    p = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    p = torch.where(seen, p, torch.zeros_like(p))
    total = p.sum(dim=1, keepdim=True)
    return (p @ v) / torch.where(total > 0, total, torch.ones_like(total))


def exact(case, seed):
    c, x = case, _inputs(case, seed)
    if c["op"] == "layout":
        return None   # whole numbers: the plain form is exact
    H, Hk, d = c["H"], c["Hk"], c["d"]
    if c["op"] == "packed":
        q, k, v = (x[n].double() for n in ("q", "k", "v"))
        out = torch.zeros_like(q, memory_format=torch.contiguous_format)
        at = 0
        for n, p in zip(_doc_lens(c), _prefix_lens(c)):
            i, j = torch.arange(n, device="cuda").view(-1, 1), torch.arange(n, device="cuda").view(1, -1)
            dist = (i - j).abs()
            seen = (j <= i) if c["causal"] else (dist >= 0)
            seen = seen & ((dist < c["window"]) if c["window"] else (dist >= 0)) | ((j < p) & (dist >= 0))
            for h in range(H):
                kv = h * Hk // H
                bias = -dist * x["slopes"][h].double() if c["slopes"] else None
                out[at:at + n, h] = _exact_rows(q[at:at + n, h], k[at:at + n, kv], v[at:at + n, kv], d ** -0.5, c["softcap"], bias, seen)
            at += n
        return out
    if c["op"] == "decode":
        out = torch.zeros(c["B"], H, d, dtype=torch.float64, device="cuda")
        for b, n in enumerate(_kv_lens(c)):
            if n == 0:
                continue
            pages = x["block_table"][b, :-(-n // c["page"])].long()
            first = max(0, n - c["window"]) if c["window"] else 0
            dist = (n - 1 - torch.arange(first, n, device="cuda")).view(1, -1)
            for kv in range(Hk):
                k, v = (x[m][pages, kv].double().view(-1, d)[first:n] for m in ("k_cache", "v_cache"))
                hs = slice(kv * (H // Hk), (kv + 1) * (H // Hk))
                bias = -dist * x["slopes"][hs].double().view(-1, 1) if c["slopes"] else None
                out[b, hs] = _exact_rows(x["q"][b, hs].double(), k, v, d ** -0.5, c["softcap"], bias, dist >= 0)
        return out
    r = c["rot"] // 2
    turn = x["positions"].double().view(-1, 1, 1) * x["inv_freq"].view(1, 1, -1)
    z = torch.polar(torch.ones_like(turn), turn)   # a rotation is a product with exp(i·angle)
    turned = []
    for name in ("q", "k"):
        t = x[name].double().clone()
        first, second = (slice(0, 2 * r, 2), slice(1, 2 * r, 2)) if c["interleaved"] else (slice(0, r), slice(r, 2 * r))
        w = torch.complex(t[..., first], t[..., second]) * z
        t[..., first], t[..., second] = w.real, w.imag
        turned.append(t)
    caches = []
    for name, rows in (("k_cache", turned[1]), ("v_cache", x["v"].double())):
        flat = x[name].double().transpose(1, 2).reshape(-1, Hk, d)   # by slot
        ok = x["slot_map"] >= 0
        flat[x["slot_map"][ok]] = rows[ok]
        caches.append(flat.view(-1, c["page"], Hk, d).transpose(1, 2).contiguous())
    return turned[0], turned[1], caches[0], caches[1]
