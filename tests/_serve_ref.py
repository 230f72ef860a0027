"""Plain 64-bit implementations of the serving operators, and the tolerances that the
operators' roundings allow, for the tests.

A result rounded to a type t is off by at most u_t = eps_t / 2 of its value. The
attention kernels round P to t (weights that are off by u_t each, normalised by
their own sum, move O by at most u_t·Σ p|v − O|), round O to t once, and form scores
in fp32: a sum of d products is off by at most (d + 2)·2^-24·Σ|q·k| (in any order), the
exponential and the factors around it by a few 2^-23 of the exponent's size."""
import math

import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def seen_mask(n_q, n_k, causal, window, prefix, device="cpu"):
    """[n_q, n_k]: which keys each row of a sequence sees (the last row is at the last key)."""
    i = torch.arange(n_q, device=device).view(-1, 1) + (n_k - n_q)
    j = torch.arange(n_k, device=device).view(1, -1)
    seen = (j <= i) if causal else torch.ones(n_q, n_k, dtype=torch.bool, device=device)
    if window:
        seen = seen & ((i - j).abs() < window)
    return seen | (j < prefix)


def attend(q, k, v, seen, *, scale, softcap=0.0, slope=0.0, dtype):
    """One head: (O, tolerance), both 64-bit [n_q, d]. q, k, v hold values of dtype; what is
    not seen is left out of every sum, whatever it holds."""
    n_q, n_k = seen.shape
    d = q.shape[1]
    out = torch.zeros(n_q, d, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    if n_k == 0 or n_q == 0:
        return out, tol
    q, k, v = q.double(), k.double(), v.double()
    used = seen.any(dim=0)
    k = torch.where(used[:, None], k, torch.zeros_like(k))
    raw = q @ k.T * scale
    size = q.abs() @ k.abs().T * scale
    s = softcap * torch.tanh(raw / softcap) if softcap else raw
    i = torch.arange(n_q, device=q.device).view(-1, 1) + (n_k - n_q)
    dist = (i - torch.arange(n_k, device=q.device).view(1, -1)).abs()
    s = s - slope * dist
    s = torch.where(seen, s, torch.full_like(s, -math.inf))
    top = s.max(dim=1, keepdim=True).values
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    p = torch.exp(s - top)
    total = p.sum(dim=1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    if bool((seen | ~used[None]).all()):   # no key is seen by some rows only
        v = torch.where(used[:, None], v, torch.zeros_like(v))
        out = p @ v
        mag = p @ v.abs()
    else:   # a key that only some rows see reaches those only
        bad = ~torch.isfinite(v).all(dim=1)
        clean = torch.where(bad[:, None], torch.zeros_like(v), v)
        out, mag = p @ clean, p @ clean.abs()
        for j in torch.nonzero(bad).flatten().tolist():
            row = torch.where(seen[:, j:j + 1], p[:, j:j + 1] * v[j:j + 1], torch.zeros_like(out))
            out, mag = out + row, mag + row.abs()
    u = HALF_STEP[dtype]
    err_s = ((d + 2) * 2.0 ** -24 * size).masked_fill(~seen, 0)
    # the exponent's terms (score, distance, running max) are each rounded at their own size
    span = s.masked_fill(~seen, 0).abs().amax(dim=1, keepdim=True) + (slope * dist).masked_fill(~seen, 0).amax(dim=1, keepdim=True)
    span = torch.where(torch.isfinite(span), span, torch.zeros_like(span))
    err_e = err_s.amax(dim=1, keepdim=True) + 8 * 2.0 ** -23 * (1 + span + 4 * softcap)
    tiny = 2.0 ** -24 * n_k if dtype == torch.float16 else 0.0   # fp16 steps near 0: P below 2^-14
    vmax = torch.where(torch.isfinite(v), v.abs(), torch.zeros_like(v)).amax(dim=0, keepdim=True)
    tol = (u + 2 * err_e) * (mag + out.abs()) + (u + n_k * 2.0 ** -24) * out.abs() + n_k * 2.0 ** -24 * mag + tiny * vmax + 2.0 ** -24
    return out, tol


def packed(q, k, v, cu_q, cu_k, *, causal=True, scale=None, softcap=0.0, window=0, slopes=None, prefix_lens=None):
    Tq, H, d = q.shape
    ratio = H // k.shape[1]
    scale = d ** -0.5 if scale is None else scale
    out = torch.zeros(Tq, H, d, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    for n in range(len(cu_q) - 1):
        a, b, e, f = cu_q[n], cu_q[n + 1], cu_k[n], cu_k[n + 1]
        seen = seen_mask(b - a, f - e, causal, window, prefix_lens[n] if prefix_lens is not None else 0, q.device)
        for h in range(H):
            out[a:b, h], tol[a:b, h] = attend(q[a:b, h], k[e:f, h // ratio], v[e:f, h // ratio], seen, scale=scale, softcap=softcap,
                                              slope=float(slopes[h]) if slopes is not None else 0.0, dtype=q.dtype)
    return out, tol


def decode(q, k_cache, v_cache, table, lens, *, scale=None, softcap=0.0, window=0, slopes=None):
    B, H, d = q.shape
    P, Hk, page, _ = k_cache.shape
    ratio = H // Hk
    scale = d ** -0.5 if scale is None else scale
    out = torch.zeros(B, H, d, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    for b in range(B):
        n = max(0, min(int(lens[b]), table.shape[1] * page))
        if n == 0 or P == 0:
            continue
        entries = table[b, :-(-n // page)].long()
        ok = ((entries >= 0) & (entries < P)).repeat_interleave(page)[:n]
        at = entries.clamp(0, P - 1)
        seen = seen_mask(1, n, True, window, 0, q.device) & ok[None]
        for h in range(H):
            k = k_cache[at, h // ratio].reshape(-1, d)[:n]
            v = v_cache[at, h // ratio].reshape(-1, d)[:n]
            o, t = attend(q[b, h:h + 1], k, v, seen, scale=scale, softcap=softcap,
                          slope=float(slopes[h]) if slopes is not None else 0.0, dtype=q.dtype)
            out[b, h], tol[b, h] = o[0], t[0]
    return out, tol


def rotate(x, positions, inv_freq, interleaved, amplitude):
    """(turned, tolerance) of x [T, heads, d]: products and sum in fp32 with cosine and sine
    off by 2^-22 at most, one rounding to the type."""
    r = inv_freq.numel()
    y = x.double().clone()
    angle = positions.double().view(-1, 1, 1) * inv_freq.view(1, 1, -1)
    c, s = amplitude * torch.cos(angle), amplitude * torch.sin(angle)
    a, b = (slice(0, 2 * r, 2), slice(1, 2 * r, 2)) if interleaved else (slice(0, r), slice(r, 2 * r))
    p, w = x.double()[..., a], x.double()[..., b]
    y[..., a], y[..., b] = p * c - w * s, w * c + p * s
    tol = torch.zeros_like(y)
    grow = 2.0 ** -20 * abs(amplitude) * (p.abs() + w.abs())
    floor = 2.0 ** -25 if x.dtype == torch.float16 else 0.0   # half a step of fp16 near 0
    tol[..., a] = tol[..., b] = grow + floor
    tol[..., :2 * r] += HALF_STEP[x.dtype] * (y.abs() + tol)[..., :2 * r]
    return y, tol


def layout(seq, new, table, free, page, max_tokens):
    """Lists in, lists out, one request and one token after the other."""
    n, M = len(seq), len(table[0]) if table else 0
    seq, new = [max(0, x) for x in seq], [max(0, x) for x in new]
    out, used, missing, cu, positions, slots = [], 0, 0, [0], [], []
    wanted = 0
    for r in range(n):
        held, want = -(-seq[r] // page), -(-(seq[r] + new[r]) // page)
        row = []
        for c in range(M):
            if c >= want:
                row.append(-1)
            elif c < held:
                row.append(table[r][c])
            else:
                row.append(free[used] if used < len(free) else -1)
                used += 1
        wanted += want - held
        out.append(row)
        cu.append(cu[-1] + new[r])
        for t in range(new[r]):
            pos = seq[r] + t
            c = pos // page
            entry = row[c] if c < M else -1
            positions.append(pos)
            slots.append(entry * page + pos % page if entry >= 0 else -1)
    taken = min(used, len(free))
    positions = (positions + [0] * max_tokens)[:max_tokens]
    slots = (slots + [-1] * max_tokens)[:max_tokens]
    return [a + b for a, b in zip(seq, new)], cu, positions, slots, out, [cu[-1], taken, wanted - taken]


def check(got, want, tol, name=""):
    got = got.double()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    bad = ~((got - want).abs() <= tol) & ~((got != got) & (want != want))
    if bad.any():
        at = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} outside the tolerance, first at {at}: "
                             f"{got[at].item()} for {want[at].item()} ± {tol[at].item()}")
