"""GPU tests of the operators for several continuations of a prompt, against the plain
64-bit forms of tests/_beam_ref.py: shapes, types, masks, what is unseen, odd sizes,
strides, ranges, graphs, streams, and a run of all of them together."""
import math
import random

import pytest
import torch

from tests import _beam_ref as ref
from tests._beam_ref import check

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
INF = math.inf


@pytest.fixture(scope="module")
def ops(gpu):
    from custom_ops_amd import ops
    ops.ensure_loaded("beam", "serve")
    return ops


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def batch(seed, groups, tail, H, Hk, d, page, dtype, alone=0, own=True):
    """Groups (prefix, requests) and requests of none. Rows of a group share its whole pages; own:
    each has a copy of the partly filled one, else only the first row names the prefix."""
    r, g = random.Random(seed), gen(seed)
    cu, prefix, lens, rows, nxt = [0], [], [], [], [0]

    def pages(n):
        nxt[0] += n
        return list(range(nxt[0] - n, nxt[0]))
    copies = []
    for p, n in groups:
        common = pages(p // page)
        first = None
        for i in range(n):
            length = p + r.randint(1, tail)
            row = list(common) + pages(-(-length // page) - p // page)
            if p % page and i:
                copies.append((first, row[p // page], p % page))
            elif p % page:
                first = row[p // page]
            if not own and i:
                row = [-7] * (p // page) + row[p // page:]
            rows.append(row)
            lens.append(length)
        cu.append(len(rows))
        prefix.append(p)
    for _ in range(alone):
        n = r.randint(1, tail)
        rows.append(pages(-(-n // page)))
        lens.append(n)
    M = max(map(len, rows)) + 1
    table = ints([x + [-1] * (M - len(x)) for x in rows])
    P = nxt[0] + 2
    order = torch.randperm(P, generator=g, device="cuda").int()
    table = torch.where(table >= 0, order[table.clamp_min(0).long()], table)
    kc, vc = (torch.randn(P, Hk, page, d, generator=g, device="cuda").to(dtype) for _ in range(2))
    for a, b, n in copies:
        a, b = int(order[a]), int(order[b])
        kc[b, :, :n], vc[b, :, :n] = kc[a, :, :n], vc[a, :, :n]
    q = torch.randn(len(rows), H, d, generator=g, device="cuda").to(dtype)
    return dict(q=q, kc=kc, vc=vc, table=table, lens=lens, cu=cu, prefix=prefix)


def shared(ops, x, **kw):
    out = ops.mha_shared_decode(x["q"], x["kc"], x["vc"], x["table"], ints(x["lens"]), ints(x["cu"]), ints(x["prefix"]), **kw)
    want, tol = ref.shared(x["q"], x["kc"], x["vc"], x["table"], x["lens"], x["cu"], x["prefix"], **kw)
    check(out, want, tol)
    return out


# ── attention over shared prefixes ────────────────────────────────────────────

@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("H,Hk", [(4, 4), (8, 2), (6, 1), (20, 1), (12, 4)])
def test_shared_heads(ops, dtype, d, H, Hk):
    x = batch(1, [(70, 3), (133, 5), (5, 2)], 50, H, Hk, d, 16, DT[dtype], alone=2)
    shared(ops, x)


@pytest.mark.parametrize("page", [8, 16, 64, 256, 1024])
@pytest.mark.parametrize("groups", [[(1, 1)], [(1, 2)], [(31, 4)], [(32, 4)], [(33, 2)], [(64, 9)], [(300, 4)], [(1000, 2), (63, 7)], [(0, 3), (200, 3)],
                                    [(257, 40)], [(96, 1), (96, 1), (97, 2)]])
def test_shared_lengths(ops, page, groups):
    x = batch(sum(p for p, _ in groups) + page, groups, 40, 8, 4, 64, page, torch.bfloat16)
    shared(ops, x)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("softcap,window,slopes", [(30.0, 0, False), (0.0, 50, False), (0.0, 0, True), (20.0, 200, True), (0.0, 1, False), (0.0, 100000, True)])
def test_shared_scores(ops, d, softcap, window, slopes):
    x = batch(5, [(400, 9), (77, 4)], 60, 8, 2, d, 16, torch.float16, alone=1)
    s = torch.tensor([2.0 ** (-8 * (h + 1) / 8) for h in range(8)], device="cuda") if slopes else None
    shared(ops, x, softcap=softcap, window=window, slopes=s)
    shared(ops, x, softcap=softcap, window=window, slopes=s, scale=0.3)


@pytest.mark.parametrize("d", [64, 128])
def test_shared_many_columns(ops, d):
    """More columns of a KV head than a workgroup takes, the last block odd; long enough to be split."""
    x = batch(9, [(2100, 37), (900, 19)], 90, 16, 2, d, 32, torch.bfloat16)
    shared(ops, x)


def test_shared_prefix_is_the_first_rows(ops):
    """The others' rows need not name the prefix's pages: whatever they have there is not read."""
    x = batch(3, [(160, 4), (99, 3)], 30, 4, 2, 128, 16, torch.bfloat16, own=False)
    a = shared(ops, x)
    y = batch(3, [(160, 4), (99, 3)], 30, 4, 2, 128, 16, torch.bfloat16, own=True)
    assert torch.equal(a, ops.mha_shared_decode(y["q"], y["kc"], y["vc"], y["table"], ints(y["lens"]), ints(y["cu"]), ints(y["prefix"])))


def test_shared_agrees_with_paged(ops):
    """Within both operators' tolerances, and exactly where nothing is shared and nothing split."""
    x = batch(4, [(333, 6)], 40, 8, 2, 128, 16, torch.bfloat16)
    a = shared(ops, x)
    b = ops.mha_paged_decode(x["q"], x["kc"], x["vc"], x["table"], ints(x["lens"]))
    _, tol = ref.shared(x["q"], x["kc"], x["vc"], x["table"], x["lens"], x["cu"], x["prefix"])
    check(a, b.double(), 2 * tol)


@pytest.mark.parametrize("lens", [[0, 0, 0], [0, 140, 150], [140, 0, 150], [100, 150, 151], [5, 150, 160], [1, 1, 160], [-3, 150, 2 ** 31 - 1]])
def test_shared_short_and_ended_requests(ops, lens):
    """Requests without keys, shorter than the prefix, longer than their tables."""
    x = batch(6, [(130, 3)], 20, 4, 2, 64, 16, torch.bfloat16)
    x["table"][:, -1] = x["table"][0, 0]   # (a longest request reaches over the whole row)
    x["lens"] = lens
    out = shared(ops, x)
    for b, n in enumerate(lens):
        if n <= 0:
            assert (out[b] == 0).all()


@pytest.mark.parametrize("cu,prefix", [([0, 0, 0], [50, 60]), ([2, 4], [70]), ([0, 3, 3, 5], [70, 9, 64]), ([1, 6], [64]), ([0], []), ([0, 6], [10 ** 9]),
                                       ([0, 6], [-5]), ([0, 100], [64]), ([3, 3, 6], [40, 70])])
def test_shared_offsets(ops, cu, prefix):
    """Empty groups, requests before, between and behind groups, prefixes past the table, offsets past the batch."""
    x = batch(7, [(70, 6)], 90, 4, 2, 64, 16, torch.float16)
    x["cu"], x["prefix"] = cu, prefix
    shared(ops, x)


@pytest.mark.parametrize("cu", [[5, 2, 6], [6, 0, 3], [-4, 3, 9], [0, 5, 2, 6], [2 ** 31 - 1, -2 ** 31, 0]])
def test_shared_offsets_that_do_not_ascend(ops, cu):
    """Nothing outside the tensors is reached, and all that comes back is finite."""
    x = batch(7, [(70, 6)], 90, 4, 2, 64, 16, torch.float16)
    out = ops.mha_shared_decode(x["q"], x["kc"], x["vc"], x["table"], ints(x["lens"]), ints(cu), ints([70] * (len(cu) - 1)))
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("where", ["prefix", "own"])
@pytest.mark.parametrize("value", [-1, 10 ** 6, -2 ** 31])
def test_shared_bad_pages(ops, where, value):
    x = batch(8, [(128, 5)], 70, 4, 2, 64, 16, torch.bfloat16)
    if where == "prefix":
        x["table"][0, 3] = value
    else:
        x["table"][2, 8] = value
    shared(ops, x)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bad", [math.nan, INF, -INF, 3e4])
def test_shared_unseen_keys_have_no_influence(ops, d, bad):
    """Rows of pages behind the last key, before the window, of pages that no row has."""
    for window in (0, 60):
        x = batch(10, [(90, 5), (40, 3)], 30, 8, 2, d, 16, torch.bfloat16)
        args = (x["table"], ints(x["lens"]), ints(x["cu"]), ints(x["prefix"]))
        want = ops.mha_shared_decode(x["q"], x["kc"], x["vc"], *args, window=window)
        seen = torch.zeros(x["kc"].shape[0], 16, dtype=torch.bool, device="cuda")
        for b, n in enumerate(x["lens"]):
            j = torch.arange(max(0, n - window) if window else 0, n, device="cuda")
            seen[x["table"][b, j // 16].long(), j % 16] = True
            g = next(i for i in range(2) if x["cu"][i] <= b < x["cu"][i + 1])
            j = j[j < x["prefix"][g]]
            seen[x["table"][x["cu"][g], j // 16].long(), j % 16] = True
        for c in (x["kc"], x["vc"]):
            c.masked_fill_(~seen[:, None, :, None], bad)
        assert torch.equal(want, ops.mha_shared_decode(x["q"], x["kc"], x["vc"], *args, window=window))


@pytest.mark.parametrize("bad", [math.nan, INF])
def test_shared_values_that_are_not_finite(ops, bad):
    """A seen V reaches the rows that see it and no other request's."""
    x = batch(11, [(96, 4)], 30, 4, 2, 64, 16, torch.bfloat16)
    args = (x["table"], ints(x["lens"]), ints(x["cu"]), ints(x["prefix"]))
    want = ops.mha_shared_decode(x["q"], x["kc"], x["vc"], *args)
    own = x["table"][1, 6].long()
    x["vc"][own, 1, 0, 5] = bad
    out = ops.mha_shared_decode(x["q"], x["kc"], x["vc"], *args)
    same = torch.ones_like(out, dtype=torch.bool)
    same[1, 2:, 5] = False
    assert torch.equal(out[same], want[same]) and not torch.isfinite(out[1, 2:, 5]).any()


def test_shared_strides(ops):
    """q out of one projection, K and V in one cache, rows before heads, a table with a wider row."""
    x = batch(12, [(150, 6)], 40, 8, 4, 64, 16, torch.float16)
    want = shared(ops, x)
    P, Hk, page, d = x["kc"].shape
    both = torch.empty(P, page, 2, Hk, d, dtype=torch.float16, device="cuda")
    both[:, :, 0] = x["kc"].transpose(1, 2)
    both[:, :, 1] = x["vc"].transpose(1, 2)
    proj = torch.randn(x["q"].shape[0], 16, d, device="cuda").half()
    proj[:, 2:10] = x["q"]
    wide = torch.full((x["table"].shape[0], x["table"].shape[1] + 5), -9, dtype=torch.int32, device="cuda")
    wide[:, :-5] = x["table"]
    out = ops.mha_shared_decode(proj[:, 2:10], both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2), wide[:, :-5], ints(x["lens"]),
                                ints(x["cu"]), ints(x["prefix"]))
    assert torch.equal(out, want)


def test_shared_empty(ops):
    x = batch(13, [(40, 2)], 9, 4, 2, 64, 16, torch.bfloat16)
    none = ops.mha_shared_decode(x["q"][:0], x["kc"], x["vc"], x["table"][:0], ints([]), ints([0]), ints([]))
    assert none.shape == (0, 4, 64)
    out = ops.mha_shared_decode(x["q"], x["kc"][:0], x["vc"][:0], x["table"], ints(x["lens"]), ints(x["cu"]), ints(x["prefix"]))
    assert (out == 0).all()
    out = ops.mha_shared_decode(x["q"], x["kc"], x["vc"], x["table"][:, :0], ints(x["lens"]), ints(x["cu"]), ints(x["prefix"]))
    assert (out == 0).all()


def test_shared_most_requests(ops):
    """The most requests a call takes, in groups of all sizes."""
    r = random.Random(2)
    groups, left = [], 1024
    while left:
        n = min(left, r.choice([1, 2, 3, 17, 90]))
        groups.append((r.choice([0, 33, 64, 90]), n))
        left -= n
    x = batch(14, groups, 12, 2, 1, 64, 16, torch.bfloat16)
    out = ops.mha_shared_decode(x["q"], x["kc"], x["vc"], x["table"], ints(x["lens"]), ints(x["cu"]), ints(x["prefix"]))
    b = ops.mha_paged_decode(x["q"], x["kc"], x["vc"], x["table"], ints(x["lens"]))
    pick = list(range(0, 1024, 37))
    for i in pick:
        g = next(g for g in range(len(groups)) if x["cu"][g] <= i < x["cu"][g + 1])
        y = dict(x, q=x["q"][i:i + 1], table=x["table"][i:i + 1], lens=[x["lens"][i]], cu=[0], prefix=[])
        want, tol = ref.shared(y["q"], y["kc"], y["vc"], y["table"], y["lens"], y["cu"], y["prefix"])
        check(out[i:i + 1], want, tol, f"request {i} of group {g}")
        check(b[i:i + 1], want, tol)


# Columns of a KV head of a group of 5: a workgroup of 32, 64 or 128 of them.
@pytest.mark.parametrize("H", [8, 16, 32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page", [8, 16, 32, 128])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_shared_shapes(ops, H, d, page, dtype):
    x = batch(H + d + page, [(330, 5), (140, 5)], 60, H, 2, d, page, DT[dtype], alone=1)
    shared(ops, x)
    slopes = torch.tensor([2.0 ** (-8 * (h + 1) / H) for h in range(H)], device="cuda")
    shared(ops, x, softcap=20.0, window=250, slopes=slopes)


@pytest.mark.parametrize("H", [8, 16, 32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page", [8, 64])
def test_shared_bad_pages_of_shapes(ops, H, d, page):
    """In the first group's prefix, in the other's only for one request."""
    x = batch(H + d, [(330, 5), (200, 5)], 60, H, 2, d, page, torch.bfloat16)
    x["table"][0, 2], x["table"][7, 200 // page] = -1, 10 ** 6
    shared(ops, x)
    shared(ops, x, softcap=15.0, window=290)


def means(x, lens, cu, prefix):
    """O where all scores are equal: the mean of V, [B, Hk, d]."""
    page, out = x["vc"].shape[2], []
    for b, n in enumerate(lens):
        g = next((i for i in range(len(prefix)) if cu[i] <= b < cu[i + 1]), None)
        j = torch.arange(n, device="cuda")
        row = torch.where(j < (0 if g is None else prefix[g]), 0 if g is None else cu[g], b)
        at = x["table"][row, j // page].long() * page + j % page
        times = torch.bincount(at, minlength=x["vc"].shape[0] * page).double()
        v = x["vc"].double().transpose(1, 2).reshape(len(times), -1)
        out.append(times @ v / n)
    return torch.stack(out).reshape(len(lens), x["vc"].shape[1], -1)


@pytest.mark.parametrize("ratio,B,Hk,prefix", [(1, 2, 32, 80000), (16, 3, 32, 280000), (16, 8, 32, 260000)])
def test_shared_long_parts(ops, ratio, B, Hk, prefix):
    """Parts of more pages than the kernel holds the numbers of at once; V are small integers and all
    scores equal, so that 32-bit sums are exact and what is read shows."""
    g, page, P, d = gen(B), 8, 300, 128
    lens = [prefix + 100 * b + 1 for b in range(B)]
    table = torch.randint(0, P // 2, (B, max(lens) // page + 1), generator=g, device="cuda").int()
    table[:, 3 * table.shape[1] // 4:] += P // 2
    vc = torch.randint(-3, 4, (P, Hk, page, d), generator=g, device="cuda").bfloat16()
    vc[P // 2:] += 5
    kc = torch.randn(P, Hk, page, d, generator=g, device="cuda").bfloat16()
    q = torch.zeros(B, Hk * ratio, d, dtype=torch.bfloat16, device="cuda")
    out = ops.mha_shared_decode(q, kc, vc, table, ints(lens), ints([0, B]), ints([prefix]))
    want = means(dict(vc=vc, table=table), lens, [0, B], [prefix])
    got = out.double().view(B, Hk, ratio, d)
    # the sums are exact (below 2^24), their quotient and its rounding are not; 1/l is of one ulp
    check(got, want[:, :, None].expand_as(got), (2.0 ** -9 * 2 + 2.0 ** -21) * want[:, :, None].abs().expand_as(got))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens", [[700] * 9, [3, 0, 0, 2100, 0, 33, 1, 0, 900], [0] * 8 + [5000], [5000] + [0] * 8])
def test_shared_own_keys_only(ops, d, lens):
    """No groups: requests of very different lengths, whose keys are one sequence for the kernel's waves."""
    x = batch(21, [(5000, 1)] * 9, 1, 6, 3, d, 64, torch.float16)
    x["lens"], x["cu"], x["prefix"] = lens, [0], []
    shared(ops, x)


@pytest.mark.parametrize("d", [64, 128])
def test_shared_plan_of_many(ops, d):
    """More requests and groups than one wave plans."""
    groups = [(70 + i % 50, 1 + i % 4) for i in range(60)]
    x = batch(15, groups, 40, 2, 1, d, 16, torch.bfloat16, alone=9)
    x["lens"][3] = x["lens"][17] = 0
    shared(ops, x)


@pytest.mark.parametrize("d,H", [(64, 4), (128, 32)])
def test_shared_past_32_bits(ops, d, H):
    """Pages that lie more than 4 GiB apart, and prefixes whose keys reach past them."""
    x = batch(16, [(200, 5)], 60, H, 2, d, 16, torch.bfloat16)
    want = shared(ops, x)
    P, Hk, page, _ = x["kc"].shape
    stride = (1 << 33) // P // 8 * 8
    far = []
    for c in (x["kc"], x["vc"]):
        buf = torch.empty(stride * P, dtype=c.dtype, device="cuda")
        y = buf.as_strided((P, Hk, page, d), (stride, page * d, d, 1))
        y.copy_(c)
        far.append(y)
    assert far[0].stride(0) * (P - 1) > 1 << 32
    out = ops.mha_shared_decode(x["q"], *far, x["table"], ints(x["lens"]), ints(x["cu"]), ints(x["prefix"]))
    assert torch.equal(out, want)


# ── selection ─────────────────────────────────────────────────────────────────

def logits_of(seed, G, W, V, dtype, spread=3.0):
    g = gen(seed)
    return (torch.randn(G, W, V, generator=g, device="cuda") * spread).to(dtype), -10 * torch.rand(G, W, generator=g, device="cuda")


def select(ops, x, scores, k, finished=None, eos=-1):
    s, t, p = ops.beam_select(x, scores, k, finished=finished, eos=eos)
    want = ref.select(x, scores, k, finished, eos)
    assert t.tolist() == [[c[1] for c in row] for row in want]
    assert p.tolist() == [[c[2] for c in row] for row in want]
    # one rounding of a value that 64 bits give to 10^-12 of the sum's logarithm
    w = torch.tensor([[c[0] for c in row] for row in want], dtype=torch.float64, device="cuda")
    none = torch.isinf(w)
    assert torch.equal(torch.isinf(s), none)
    check(s.masked_fill(none, 0), w.masked_fill(none, 0), 2.0 ** -24 * w.masked_fill(none, 0).abs() + 1e-10)
    return s, t, p


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("G,W,V,k", [(1, 1, 1, 1), (1, 1, 7, 3), (1, 4, 5, 64), (2, 3, 1000, 3), (3, 8, 2049, 16), (1, 50, 777, 50), (1, 2, 40001, 64), (5, 1, 8200, 1),
                                     (130, 9, 100, 9), (1, 256, 300, 5), (300, 4, 9000, 8)])
def test_select(ops, dtype, G, W, V, k):
    x, scores = logits_of(V + W, G, W, V, dtype)
    select(ops, x, scores, k)


@pytest.mark.parametrize("k", [1, 5, 64])
@pytest.mark.parametrize("kind", ["equal", "two values", "steps", "one row's", "zeros"])
def test_select_ties(ops, kind, k):
    """The lowest place among equals, however many there are."""
    V, W = 20000, 3
    x = torch.zeros(2, W, V, device="cuda")
    if kind == "two values":
        x[:, :, 5000:] = 1.0
    elif kind == "steps":
        x = (torch.arange(V, device="cuda") // 3000 % 4).float().expand(2, W, V).contiguous()
    elif kind == "one row's":
        x[:, 1] = torch.randn(V, generator=gen(1), device="cuda")
    elif kind == "zeros":
        x[..., ::2] = -0.0
        x[..., 7:12] = 0.0
    for dtype in (torch.float32, torch.bfloat16):
        select(ops, x.to(dtype), torch.zeros(2, W, device="cuda"), k)


def test_select_neighbours_in_the_last_digits(ops):
    """Beams whose candidates differ by less than 32 bits tell apart."""
    g = gen(2)
    x = torch.randn(64, 4, 3001, generator=g, device="cuda")
    x[:, 1] = x[:, 0].flip(-1)                       # the same sum in another order
    x[:, 2] = x[:, 0] * 1.0000001
    scores = torch.zeros(64, 4, device="cuda")
    scores[:, 3] = 1e-7
    x[:, 3] = x[:, 0]
    x[:, 1] += 2.0 ** -20
    s, t, p = ops.beam_select(x, scores, 8)
    want = ref.select(x, scores, 8)
    for g in range(64):
        for i in range(8):
            got = (int(t[g, i]), int(p[g, i]))
            if got != want[g][i][1:]:   # only candidates that 64 bits cannot tell apart may change places
                w = int(p[g, i]) % 4
                r = x[g, w].double()
                true = float(scores[g, w]) + float(r[got[0]] - (r.max() + torch.log(torch.exp(r - r.max()).sum())))
                assert abs(true - want[g][i][0]) < 1e-11, (g, i)


def test_select_finished(ops):
    x, scores = logits_of(3, 6, 5, 900, torch.bfloat16)
    done = torch.rand(6, 5, generator=gen(4), device="cuda") < 0.4
    done[0], done[1] = True, False
    s, t, p = select(ops, x, scores, 5, done, 17)
    assert (t[0] == 17).all() and sorted(p[0].tolist()) == list(range(5))


def test_select_what_is_not_finite(ops):
    x, scores = logits_of(5, 8, 3, 500, torch.float32)
    x[0, 1, 17] = math.nan
    x[1, 0, 3] = INF
    x[2, 2, ::2] = -INF
    x[3, :, :498] = -INF          # few candidates
    x[4] = -INF                   # none
    x[5, 0], x[5, 1, 499] = -INF, 3e38
    x[6] = math.nan
    x[7, 0] = 3e38
    scores[2, 0], scores[3, 0], scores[3, 1] = math.nan, -INF, INF
    select(ops, x, scores, 10)
    for v in (0, 255, 256, 499):   # a NaN anywhere, in every type
        for dtype in (torch.bfloat16, torch.float16):
            y = x[2:3].to(dtype).clone()
            y[0, 1, v] = math.nan
            select(ops, y, scores[2:3], 4)


def test_select_first_step(ops):
    """All beams but the first do not exist yet."""
    x, scores = logits_of(6, 3, 4, 100, torch.float16)
    scores[:, 1:] = -INF
    s, t, p = select(ops, x, scores, 4)
    assert (p % 4 == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_select_strides(ops, dtype):
    """Rows at odd distances and addresses; all beams with the same logits, as one row expanded."""
    x, scores = logits_of(7, 3, 4, 1003, dtype)
    wide = torch.empty(3, 5, 1017, dtype=dtype, device="cuda")
    view = wide[:, 1:, 5:1008]
    view.copy_(x)
    for a, b in zip(select(ops, x, scores, 7), select(ops, view, scores, 7)):
        assert torch.equal(a, b)
    one = x[:, :1].expand(3, 4, 1003)
    select(ops, one, scores, 7)
    select(ops, x[:1].expand(3, 4, 1003), scores, 7)


def test_select_large_values(ops):
    """Logits far apart: sums that underflow beside the largest one; steps of the type's last place."""
    g = gen(8)
    x = (torch.randn(4, 2, 5000, generator=g, device="cuda") * 1e4)
    select(ops, x, torch.zeros(4, 2, device="cuda"), 6)
    select(ops, (x * 1e30).bfloat16(), torch.zeros(4, 2, device="cuda"), 6)
    select(ops, torch.randn(4, 2, 5000, generator=g, device="cuda") * 1e-6, torch.zeros(4, 2, device="cuda"), 6)


# ── pages ─────────────────────────────────────────────────────────────────────

def flat(got):
    return [x.tolist() for x in got]


def fork(ops, table, seq, parents, page, P, held=None):
    M = len(table[0]) if table else 0
    got = ops.paged_fork(ints(table).view(len(table), M), ints(seq), ints(parents), page, P, held=None if held is None else ints(held))
    want = ref.fork(table, seq, parents, page, P, held or ())
    for name, a, b in zip(("table", "lens", "src", "dst", "free", "counts"), flat(got), want):
        assert a == b, name
    return got


def pool(seed, N, M, page, P, share=0.5):
    """Rows of random lengths whose first pages are partly those of the row before."""
    r = random.Random(seed)
    order = list(range(P))
    r.shuffle(order)
    table, seq, at = [], [], 0
    for i in range(N):
        n = r.choice([0, 1, page, M * page, r.randint(0, M * page)])
        used = -(-n // page)
        row = []
        for c in range(used):
            if i and c < len(table[-1]) and table[-1][c] >= 0 and r.random() < share and (c == 0 or row[-1] == table[-1][c - 1]):
                row.append(table[-1][c])
            else:
                row.append(order[at % P])
                at += 1
        table.append(row + [-1] * (M - used))
        seq.append(n)
    return table, seq


@pytest.mark.parametrize("page", [1, 3, 16, 1000])
@pytest.mark.parametrize("N,M,P,R", [(1, 1, 1, 1), (4, 6, 40, 8), (4, 6, 12, 8), (60, 33, 3000, 60), (300, 20, 9000, 700), (5, 2, 33, 1000), (3, 500, 70000, 40)])
def test_fork(ops, page, N, M, P, R):
    table, seq = pool(N + page, N, M, page, P)
    r = random.Random(R)
    parents = [r.randint(-1, N - 1) for _ in range(R)]
    fork(ops, table, seq, parents, page, P)
    fork(ops, table, seq, parents, page, P, held=[r.randint(-3, P + 3) for _ in range(min(P, 50))])


def test_fork_of_beams(ops):
    """Three beams of one row of 20 tokens in pages of 16: one keeps the second page, two get copies."""
    t, lens, src, dst, free, counts = fork(ops, [[4, 7, -1], [5, 6, -1]], [20, 33], [0, 0, -1, 0], 16, 10)
    assert t.tolist() == [[4, 7, -1], [4, 0, -1], [-1, -1, -1], [4, 1, -1]]
    assert src.tolist() == [-1, 7, -1, 7] and dst.tolist() == [-1, 0, -1, 1] and counts.tolist() == [6, 2, 0]


def test_fork_rows_out_of_range(ops):
    fork(ops, [[0, 1], [2, 3]], [20, 40], [2, -1, 1, 2 ** 31 - 1, -2 ** 31, 0, 1], 16, 6)
    fork(ops, [[0, 9], [-5, 3]], [20, 10 ** 9], [0, 0, 1, 1], 16, 6)      # entries that are no pages; a length past the row
    fork(ops, [[0, 1], [2, 3]], [-4, 20], [0, 0, 1, 1], 16, 4)
    fork(ops, [[0, 0], [0, 0]], [20, 20], [0, 1], 16, 4)                   # a page twice in a row


def test_fork_without_room(ops):
    t, lens, src, dst, free, counts = fork(ops, [[0, 1]], [17], [0, 0, 0, 0], 16, 4)
    assert counts.tolist() == [0, 2, 1] and t[:, 1].tolist() == [1, 2, 3, -1]


def test_fork_empty(ops):
    fork(ops, [[0, 1]], [17], [], 16, 4)
    got = ops.paged_fork(ints([]).view(0, 3), ints([]), ints([0, 0]), 16, 5)
    assert got[0].tolist() == [[-1] * 3] * 2 and got[4].tolist() == [0, 1, 2, 3, 4]
    got = ops.paged_fork(ints([[]]).view(1, 0), ints([5]), ints([0, 0]), 16, 0)
    assert got[0].shape == (2, 0) and got[1].tolist() == [0, 0] and got[5].tolist() == [0, 0, 0]


def test_fork_most(ops):
    """The most rows and pages a call takes, and every row with a page of its own to want."""
    P, page = 1 << 19, 16
    table, seq = [[i * 7, P - 1 - i] for i in range(2000)], [17 + i % 15 for i in range(2000)]
    r = random.Random(1)
    fork(ops, table, seq, [r.randint(0, 1999) for _ in range(4096)], page, P, held=list(range(100, 9000, 3)))


def compact(ops, table, seq, page, P, held=None):
    M = len(table[0]) if table else 0
    got = ops.paged_compact(ints(table).view(len(table), M), ints(seq), page, P, held=None if held is None else ints(held))
    want = ref.compact(table, seq, page, P, held or ())
    for name, a, b in zip(("table", "src", "dst", "remap", "free", "counts"), flat(got), want):
        assert a == b, name
    return got


@pytest.mark.parametrize("page", [1, 16, 1000])
@pytest.mark.parametrize("N,M,P", [(1, 1, 1), (1, 1, 2), (4, 6, 40), (4, 6, 10), (9, 7, 32), (60, 33, 3000), (300, 20, 70001), (3, 500, 1300), (50, 40, 1 << 19), (40, 700, 30000), (17, 300, 2048)])
def test_compact(ops, page, N, M, P):
    table, seq = pool(N + M, N, M, page, P)
    compact(ops, table, seq, page, P)
    r = random.Random(P)
    compact(ops, table, seq, page, P, held=[r.randint(-3, P + 3) for _ in range(min(P, 40))])


def test_compact_edges(ops):
    compact(ops, [[0, 1], [2, 3]], [32, 32], 16, 4)                        # all in use
    compact(ops, [[0, 1], [2, 3]], [0, 0], 16, 64)                         # none
    compact(ops, [[63, 62], [61, 60]], [32, 17], 16, 64)
    compact(ops, [[99, -1], [-7, 5]], [32, 10 ** 9], 16, 8)
    got = ops.paged_compact(ints([]).view(0, 3), ints([]), 16, 5)
    assert got[4].tolist() == [0, 1, 2, 3, 4] and got[5].tolist() == [0, 0]
    got = ops.paged_compact(ints([[0]]), ints([3]), 16, 0)
    assert got[0].tolist() == [[-1]] and got[5].tolist() == [0, 0]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("Hk,page,d,P,n", [(1, 1, 64, 9, 3), (1, 8, 64, 20, 7), (2, 16, 128, 30, 15), (3, 5, 64, 400, 190), (8, 64, 128, 20, 10), (1, 1024, 64, 5, 2)])
def test_copy(ops, dtype, Hk, page, d, P, n):
    g = gen(P)
    kc, vc = (torch.randn(P, Hk, page, d, generator=g, device="cuda").to(DT[dtype]) for _ in range(2))
    ids = torch.randperm(P, generator=g, device="cuda").int()
    dst, rest = ids[:n].clone(), ids[n:]
    src = rest[torch.randint(0, P - n, (n,), generator=g, device="cuda")].clone()   # one page to several places
    if n > 5:
        src[1], dst[2], src[3], dst[4] = -1, -1, P, 2 ** 31 - 1
    want = [c.clone() for c in (kc, vc)]
    for a, b in zip(src.tolist(), dst.tolist()):
        if 0 <= a < P and 0 <= b < P:
            for w in want:
                w[b] = w[a]
    # rows first, K and V in one tensor
    both = torch.empty(P, page, 2, Hk, d, dtype=kc.dtype, device="cuda")
    views = [both[:, :, i].transpose(1, 2) for i in range(2)]
    for view, c in zip(views, (kc, vc)):
        view.copy_(c)
    assert ops.paged_copy(kc, vc, src, dst) is None
    ops.paged_copy(*views, src, dst)
    for c, view, w in zip((kc, vc), views, want):
        assert torch.equal(c, w) and torch.equal(view, w)


def test_copy_nothing(ops):
    kc = torch.randn(4, 2, 16, 64, device="cuda").half()
    vc, want = kc.clone(), kc.clone()
    ops.paged_copy(kc, vc, ints([]), ints([]))
    ops.paged_copy(kc, vc, ints([-1, 9]), ints([2, 1]))
    ops.paged_copy(kc[:0], vc[:0], ints([1]), ints([0]))
    assert torch.equal(kc, want) and torch.equal(vc, want)


def test_copy_past_32_bits(ops):
    """Pages that lie more than 2^32 bytes into a cache."""
    P, Hk, page, d = 2200, 8, 1024, 128
    kc, vc = (torch.zeros(P, Hk, page, d, dtype=torch.float16, device="cuda") for _ in range(2))
    kc[2150], vc[2199] = 1.5, 2.5
    ops.paged_copy(kc, vc, ints([2150, 2199]), ints([2198, 3]))
    assert (kc[2198] == 1.5).all() and (vc[3] == 2.5).all() and (kc[3] == 0).all() and (vc[2198] == 0).all()


# ── graphs, streams, refusals ─────────────────────────────────────────────────

def test_streams_and_graphs(ops):
    """All five on a side stream, and captured and replayed with other contents, eager work between."""
    x = batch(20, [(200, 6), (90, 5)], 40, 8, 2, 64, 16, torch.bfloat16)
    lens, cu, prefix = ints(x["lens"]), ints(x["cu"]), ints(x["prefix"])
    lx, scores = logits_of(9, 2, 6, 5000, torch.bfloat16)
    parents = ints([0, 0, 2, 2, 2, 5, 6, 7, 7, -1, 10])
    P = x["kc"].shape[0]

    def step():
        f = ops.paged_fork(x["table"], lens, parents, 16, P + 40)
        c = ops.paged_compact(x["table"], lens, 16, P + 40)
        out = [ops.mha_shared_decode(x["q"], x["kc"], x["vc"], x["table"], lens, cu, prefix), *ops.beam_select(lx, scores, 6), *f, *c]
        return out

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(4):
        g = gen(seed)
        x["q"].copy_(torch.randn(x["q"].shape, generator=g, device="cuda"))
        lx.copy_(torch.randn(lx.shape, generator=g, device="cuda") * 3)
        parents.copy_(torch.randint(-1, 11, parents.shape, generator=g, device="cuda"))
        lens.copy_(ints(x["lens"]) - seed)
        graph.replay()
        got = [h.clone() for h in held]
        for a, b in zip(step(), got):
            assert torch.equal(a, b)
        torch.cuda.synchronize()


def test_two_graphs_at_once(ops):
    """Two graphs captured apart, replayed on two streams together: neither uses the other's workspace."""
    x = batch(21, [(1500, 9)], 60, 8, 2, 128, 16, torch.bfloat16)
    y = batch(22, [(1400, 8)], 60, 8, 2, 128, 16, torch.bfloat16)
    lx, scores = logits_of(10, 2, 6, 30000, torch.bfloat16)
    runs = []
    for z, scale in ((x, 1.0), (y, 2.0)):
        args = (z["q"], z["kc"], z["vc"], z["table"], ints(z["lens"]), ints(z["cu"]), ints(z["prefix"]))
        mine = lx * scale

        def call(args=args, mine=mine):
            return [ops.mha_shared_decode(*args), *ops.beam_select(mine, scores, 9), *ops.paged_fork(args[3], args[4], args[4], 16, 4000)]
        want = call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = call()
        runs.append((graph, held, want, torch.cuda.Stream(), call))   # (call holds the graph's inputs)
    for _ in range(5):
        torch.cuda.synchronize()
        for graph, _, _, stream, _ in runs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _, held, want, _, _ in runs:
            for a, b in zip(held, want):
                assert torch.equal(a, b)


def test_refusals(ops):
    x = batch(23, [(40, 3)], 9, 4, 2, 64, 16, torch.bfloat16)
    good = dict(q=x["q"], k_cache=x["kc"], v_cache=x["vc"], block_table=x["table"], kv_lens=ints(x["lens"]), cu_groups=ints(x["cu"]),
                prefix_lens=ints(x["prefix"]))
    for bad, text in [(dict(q=x["q"].float()), "float16 or bfloat16"), (dict(q=x["q"].half()), "dtype must match"), (dict(q=x["q"][:, :3]), "divisible"),
                      (dict(q=x["q"][..., :32]), "head_dim"), (dict(kv_lens=good["kv_lens"].long()), "kv_lens"), (dict(kv_lens=good["kv_lens"][:2]), "kv_lens"),
                      (dict(cu_groups=ints([0])), "cu_groups"), (dict(prefix_lens=ints([[1]])), "prefix_lens must be 1D"),
                      (dict(prefix_lens=ints(x["prefix"]).cpu()), "prefix_lens must be a CUDA tensor"), (dict(block_table=x["table"][:2]), "block_table"),
                      (dict(block_table=x["table"].t().contiguous().t()), "innermost"), (dict(scale=-1.0), "scale"), (dict(softcap=2000.0), "softcap"),
                      (dict(window=-1), "window"), (dict(slopes=torch.ones(3, device="cuda")), "slopes"), (dict(v_cache=x["vc"][:-1]), "same shape"),
                      (dict(backend="tilelang"), "tilelang")]:
        with pytest.raises(RuntimeError, match=text):
            ops.mha_shared_decode(**{**good, **bad})
    many = torch.zeros(1025, 4, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="1024 requests"):
        ops.mha_shared_decode(many, x["kc"], x["vc"], x["table"][:1].expand(1025, -1), ints([0] * 1025), ints([0]), ints([]))
    lx, s = logits_of(1, 2, 3, 50, torch.float32)
    done = torch.zeros(2, 3, dtype=torch.bool, device="cuda")
    good = dict(logits=lx, scores=s, k=3)
    for bad, text in [(dict(logits=lx.double()), "float16, bfloat16 or float32"), (dict(logits=lx[0]), "3D"), (dict(logits=lx.transpose(1, 2)), "innermost"),
                      (dict(logits=lx.cpu()), "CUDA"), (dict(scores=s.half()), "float32"), (dict(scores=s[:1]), "scores"), (dict(scores=s.t().contiguous().t()), "scores"),
                      (dict(k=0), "k must"), (dict(k=65), "k must"), (dict(finished=done), "eos"), (dict(finished=done, eos=50), "eos"),
                      (dict(finished=done.float(), eos=1), "bool"), (dict(finished=done[:1], eos=1), "finished"), (dict(logits=lx[:, :0]), "beams"),
                      (dict(logits=lx[..., :0]), "vocabulary"), (dict(logits=lx[:, :1].expand(2, 257, 50)), "beams")]:
        with pytest.raises(RuntimeError, match=text):
            ops.beam_select(**{**good, **bad})
    t, n = x["table"], ints(x["lens"])
    for f, args, text in [(ops.paged_fork, (t, n, n.long(), 16, 9), "parents"), (ops.paged_fork, (t, n[:2], n, 16, 9), "seq_lens"), (ops.paged_fork, (t, n, n, 0, 9), "page_size"),
                          (ops.paged_fork, (t, n, n, 16, -1), "num_pages"), (ops.paged_fork, (t, n, n, 16, 2 ** 19 + 1), "num_pages"), (ops.paged_fork, (t.long(), n, n, 16, 9), "block_table"),
                          (ops.paged_fork, (t, n, n, 16, 9, t), "held"), (ops.paged_fork, (t, n, ints([0] * 4097), 16, 9), "4096 rows"), (ops.paged_fork, (t, n, n.cpu(), 16, 9), "CUDA"),
                          (ops.paged_compact, (t[:1].expand(4097, -1), ints([0] * 4097), 16, 9), "4096 rows"), (ops.paged_compact, (t, n, 16, 2 ** 19 + 1), "num_pages"),
                          (ops.paged_copy, (x["kc"], x["vc"].half(), n, n), "dtype"), (ops.paged_copy, (x["kc"], x["vc"][:2], n, n), "same shape"),
                          (ops.paged_copy, (x["kc"], x["kc"], n, n), "overlap|memory"), (ops.paged_copy, (x["kc"], x["vc"], n, n[:2]), "dst"),
                          (ops.paged_copy, (x["kc"].float(), x["vc"].float(), n, n), "float16 or bfloat16"), (ops.paged_copy, (x["kc"], x["vc"], n.long(), n), "src")]:
        with pytest.raises(RuntimeError, match=text):
            f(*args)


# ── together ──────────────────────────────────────────────────────────────────

def test_a_search(ops):
    """Steps of a beam search through all operators (a model of one attention layer whose keys, values
    and logits depend on the token): after each, the cache holds for every beam the keys of its own
    history, and attention gives what the history's rows give, computed alone."""
    G, W, V, H, Hk, d, page, prompt = 3, 4, 60, 4, 2, 64, 8, 21
    g = gen(30)
    emb = torch.randn(V, H + 2 * Hk, d, generator=g, device="cuda").bfloat16()
    head = torch.randn(H * d, V, generator=g, device="cuda") * 0.2
    P = 64
    kc, vc = (torch.full((P, Hk, page, d), math.nan, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    freq, _ = ops.rotary_frequencies(d, device="cuda")
    free = torch.randperm(P, generator=g, device="cuda").int()
    words = torch.randint(0, V, (G, prompt), generator=g, device="cuda")
    M = 8
    # the prompts, one row each
    lens = ints([0] * G)
    table = torch.full((G, M), -1, dtype=torch.int32, device="cuda")
    lens, cu, pos, slots, table, counts = ops.paged_layout(lens, ints([prompt] * G), table, free, page, G * prompt)
    x = emb[words.flatten()]
    ops.rope_paged_store(x[:, :H], x[:, H:H + Hk], x[:, H + Hk:], pos, freq, slots, kc, vc)
    # the beams: rows of a prompt, of which only the first exists
    rows = torch.arange(G, device="cuda").repeat_interleave(W).int()
    history = words.repeat_interleave(W, 0)
    table, lens, src, dst, free, _ = ops.paged_fork(table, lens, rows, page, P)
    ops.paged_copy(kc, vc, src, dst)
    scores = torch.full((G, W), -INF, device="cuda")
    scores[:, 0] = 0
    logits = torch.randn(G, W, V, generator=g, device="cuda").bfloat16()
    groups, prefix = ints([W * i for i in range(G + 1)]), ints([prompt] * G)
    done = torch.zeros(G, W, dtype=torch.bool, device="cuda")
    for step in range(7):
        want = ref.select(logits, scores, W, done, 1)
        scores, tokens, parents = ops.beam_select(logits, scores, W, finished=done, eos=1)
        assert tokens.tolist() == [[c[1] for c in r] for r in want] and parents.tolist() == [[c[2] for c in r] for r in want]
        done = tokens == 1
        up = parents.flatten()
        history = torch.cat([history[up.long().clamp_min(0)], tokens.flatten()[:, None].long().clamp_min(0)], 1)
        table, lens, src, dst, free, counts = ops.paged_fork(table, lens, up, page, P)
        ops.paged_copy(kc, vc, src, dst)
        if step == 3:
            table, src, dst, remap, free, counts = ops.paged_compact(table, lens, page, P)
            ops.paged_copy(kc, vc, src, dst)
        lens, cu, pos, slots, table, counts = ops.paged_layout(lens, torch.ones_like(lens), table, free, page, G * W)
        assert int(counts[2]) == 0
        x = emb[history[:, -1]]
        q, _ = ops.rope_paged_store(x[:, :H], x[:, H:H + Hk], x[:, H + Hk:], pos, freq, slots, kc, vc)
        out = ops.mha_shared_decode(q, kc, vc, table, lens, groups, prefix)
        n = history.shape[1]
        y = emb[history.flatten()]
        at = torch.arange(n, device="cuda").int().repeat(G * W)
        none = torch.full((G * W * n,), -1, dtype=torch.int64, device="cuda")
        qr, kr = ops.rope_paged_store(y[:, :H], y[:, H:H + Hk], y[:, H + Hk:], at, freq, none, kc, vc)
        off = torch.arange(G * W + 1, device="cuda").int() * n
        alone = ops.mha_packed_fwd(qr, kr, y[:, H + Hk:], off, off).view(G * W, n, H, d)[:, -1]
        assert lens.tolist() == [n] * (G * W)
        for b in range(G * W):   # both are within the tolerance of the same row
            k, v = (z.view(G * W, n, Hk, d)[b] for z in (kr, y[:, H + Hk:]))
            for h in range(H):
                want, tol = ref.attend(q[b, h:h + 1], k[:, h * Hk // H], v[:, h * Hk // H], torch.ones(1, n, dtype=torch.bool, device="cuda"),
                                       scale=d ** -0.5, dtype=torch.bfloat16)
                check(out[b, h:h + 1], want, tol, f"step {step} beam {b}")
                check(alone[b, h:h + 1], want, tol)
        logits = (out.float().flatten(1) @ head).view(G, W, V).bfloat16()
