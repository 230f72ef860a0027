"""Plain 64-bit implementations of the operators for several continuations of a prompt, one
request, row and page after the other, for the tests. Attention's tolerance is
tests/_serve_ref.py's: the same roundings of P, O and the scores, whatever is shared."""
import math

import torch

from tests._serve_ref import HALF_STEP, attend, check, seen_mask  # noqa: F401


def shared(q, k_cache, v_cache, table, lens, cu, prefix, *, scale=None, softcap=0.0, window=0, slopes=None):
    """(O, tolerance), 64-bit [B, H, d]."""
    B, H, d = q.shape
    P, Hk, page, _ = k_cache.shape
    ratio = H // Hk
    scale = d ** -0.5 if scale is None else scale
    cap = table.shape[1] * page
    out = torch.zeros(B, H, d, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    for b in range(B):
        n = max(0, min(int(lens[b]), cap))
        if n == 0 or P == 0:
            continue
        g = next((i for i in range(len(prefix)) if int(cu[i]) <= b < int(cu[i + 1])), None)
        common = 0 if g is None else max(0, min(int(prefix[g]), cap))
        j = torch.arange(n, device=q.device)
        row = torch.where(j < common, 0 if g is None else int(cu[g]), b)
        entry = table[row, j // page].long()
        ok = (entry >= 0) & (entry < P)
        at = entry.clamp(0, P - 1)
        seen = seen_mask(1, n, True, window, 0, q.device) & ok[None]
        for h in range(H):
            k, v = (x[at, h // ratio, j % page] for x in (k_cache, v_cache))
            o, t = attend(q[b, h:h + 1], k, v, seen, scale=scale, softcap=softcap, slope=float(slopes[h]) if slopes is not None else 0.0,
                          dtype=q.dtype)
            out[b, h], tol[b, h] = o[0], t[0]
    return out, tol


def select(logits, scores, k, finished=None, eos=-1):
    """Lists: the k best of every search as (score, token, parent), in 64 bits, one sort."""
    G, W, V = logits.shape
    x = logits.double()
    out = []
    for g in range(G):
        every = []
        for w in range(W):
            run = float(scores[g, w])
            if not math.isfinite(run):
                continue
            if finished is not None and bool(finished[g, w]):
                every.append((-run, w, eos))
                continue
            r = x[g, w]
            if bool(torch.isnan(r).any()) or bool((r == math.inf).any()) or bool((r == -math.inf).all()):
                continue
            top = r.max()
            s = run + (r - (top + torch.log(torch.exp(r - top).sum())))
            least = s.topk(min(k, V)).values[-1]   # (what is below k others is not looked at)
            best = torch.nonzero((s >= least) & (s > -math.inf)).flatten()
            every += [(-a, w, v) for a, v in zip(s[best].tolist(), best.tolist())]
        every.sort()
        best = every[:k]
        out.append([(-s, v, g * W + w) for s, w, v in best] + [(-math.inf, -1, -1)] * (k - len(best)))
    return out


def _used(n, page, M):
    n = max(0, min(n, M * page))
    return n, -(-n // page)


def fork(table, seq, parents, page, num_pages, held=()):
    """Lists in, lists out: table, lens, src, dst, free pages, counts."""
    N, M = len(table), len(table[0]) if table else 0
    rows, lens = [], []
    for p in parents:
        n, used = _used(seq[p], page, M) if 0 <= p < N else (0, 0)
        lens.append(n)
        rows.append([table[p][c] if c < used and 0 <= table[p][c] < num_pages else -1 for c in range(M)])
    kept = {h for h in held if 0 <= h < num_pages}
    whole = set(kept)
    for r, n in zip(rows, lens):
        whole |= {e for e in r[:n // page] if e >= 0}
    used = kept | {e for r in rows for e in r if e >= 0}
    free = [p for p in range(num_pages) if p not in used]
    src, dst, taken, missing, owners = [], [], 0, 0, set()
    for r, n in zip(rows, lens):
        a = b = -1
        c = n // page
        e = r[c] if n % page else -1
        if e >= 0:
            if e in whole or e in owners:
                if taken < len(free):
                    a, b = e, free[taken]
                    taken += 1
                else:
                    missing += 1
                r[c] = b
            owners.add(e)
        src.append(a)
        dst.append(b)
    left = free[taken:]
    return rows, lens, src, dst, left + [-1] * (num_pages - len(left)), [len(left), taken, missing]


def compact(table, seq, page, num_pages, held=()):
    N, M = len(table), len(table[0]) if table else 0
    rows = []
    for r in range(N):
        _, used = _used(seq[r], page, M)
        rows.append([table[r][c] if c < used and 0 <= table[r][c] < num_pages else -1 for c in range(M)])
    used = {h for h in held if 0 <= h < num_pages} | {e for r in rows for e in r if e >= 0}
    u = len(used)
    src = [p for p in range(u, num_pages) if p in used]
    dst = [p for p in range(u) if p not in used]
    remap = [p if p in used and p < u else -1 for p in range(num_pages)]
    for a, b in zip(src, dst):
        remap[a] = b
    half = num_pages // 2
    pad = [-1] * (half - len(src))
    return ([[remap[e] if e >= 0 else -1 for e in r] for r in rows], src + pad, dst + pad, remap,
            list(range(u, num_pages)) + [-1] * u, [u, len(src)])
