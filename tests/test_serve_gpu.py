"""The serving operators on the GPU against plain 64-bit implementations
(tests/_serve_ref.py), at the sizes, masks, lengths, strides and pages where they can
go wrong. Tolerances are derived there, from the operators' roundings."""
import math

import pytest
import torch

from tests import _serve_ref as ref

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]
NAN = float("nan")


@pytest.fixture(scope="module")
def ops(gpu):
    from custom_ops_amd import ops as o
    o.ensure_loaded("serve")
    return o


def randn(*shape, seed=0, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def cu_of(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


def slopes_of(H):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], device="cuda")


# ── packed attention ──────────────────────────────────────────────────────────

def packed_case(ops, lens_q, lens_k=None, H=4, Hk=2, d=128, dtype=torch.bfloat16, pad=0, seed=1, slopes=False, prefix=None, **kw):
    lens_k = lens_q if lens_k is None else lens_k
    cq, ck = cu_of(lens_q), cu_of(lens_k)
    q = randn(cq[-1] + pad, H, d, seed=seed, dtype=dtype)
    k, v = randn(ck[-1] + pad, Hk, d, seed=seed + 1, dtype=dtype), randn(ck[-1] + pad, Hk, d, seed=seed + 2, dtype=dtype)
    s = slopes_of(H) if slopes else None
    got = ops.mha_packed_fwd(q, k, v, i32(cq), i32(ck), slopes=s, prefix_lens=i32(prefix) if prefix else None, **kw)
    want, tol = ref.packed(q, k, v, cq, ck, slopes=s, prefix_lens=prefix, **kw)
    ref.check(got, want, tol, f"{lens_q} {lens_k} {kw}")
    if pad:
        assert (got[cq[-1]:] == 0).all()
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens", [[1], [2, 1, 63], [64], [65, 127, 128], [200, 0, 31, 300], [513]])
def test_packed_causal_lengths(ops, dtype, d, lens):
    packed_case(ops, lens, d=d, dtype=dtype, pad=3)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens", [[1], [65, 30], [300, 129]])
def test_packed_not_causal(ops, d, lens):
    packed_case(ops, lens, d=d, causal=False)


@pytest.mark.parametrize("H,Hk", [(1, 1), (3, 1), (6, 2), (8, 8), (16, 1)])
def test_packed_head_groups(ops, H, Hk):
    packed_case(ops, [70, 129], H=H, Hk=Hk, d=64)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 200, 2 ** 31 - 1])
def test_packed_window(ops, causal, window):
    packed_case(ops, [300, 65], causal=causal, window=window)


@pytest.mark.parametrize("prefix", [[0, 0], [1, 40], [64, 65], [300, 1000], [-5, 2 ** 31 - 1]])
@pytest.mark.parametrize("window", [0, 20])
def test_packed_prefix(ops, prefix, window):
    held = [min(max(p, 0), 10 ** 6) for p in prefix]
    q, k, v = randn(420, 4, 64, seed=1), randn(420, 2, 64, seed=2), randn(420, 2, 64, seed=3)
    cu = [0, 290, 420]
    got = ops.mha_packed_fwd(q, k, v, i32(cu), i32(cu), window=window, prefix_lens=i32(prefix))
    want, tol = ref.packed(q, k, v, cu, cu, window=window, prefix_lens=held)
    ref.check(got, want, tol)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("softcap,slopes", [(0.0, True), (5.0, False), (50.0, True), (1000.0, False)])
def test_packed_scores(ops, dtype, d, softcap, slopes):
    packed_case(ops, [257, 40], d=d, dtype=dtype, softcap=softcap, slopes=slopes, window=130, prefix=[9, 0])
    packed_case(ops, [100], d=d, dtype=dtype, softcap=softcap, slopes=slopes, causal=False, scale=0.3)


@pytest.mark.parametrize("lens_q,lens_k", [([5], [300]), ([300], [5]), ([1, 1, 1], [100, 0, 64]), ([0, 70], [50, 65]), ([130, 3], [0, 700])])
@pytest.mark.parametrize("causal", [True, False])
def test_packed_rows_and_keys_differ(ops, lens_q, lens_k, causal):
    """Fewer rows than keys (a chunk behind a context), more (rows that see nothing), none."""
    packed_case(ops, lens_q, lens_k, causal=causal, pad=1)


def test_packed_eight_wave_grid(ops):
    """Enough rows for workgroups of 256, ragged."""
    packed_case(ops, [1000, 1, 2000, 1537, 77], H=16, Hk=4, pad=9)
    packed_case(ops, [2100, 2000], H=16, Hk=16, d=64, window=700, softcap=30.0, slopes=True, prefix=[100, 3], dtype=torch.float16)


@pytest.mark.parametrize("T", [4300, 5000, 7900, 8300])
def test_packed_between_one_and_two_workgroups_a_cu(ops, T):
    packed_case(ops, [T], H=8, Hk=8, d=64, window=300)
    packed_case(ops, [T // 2, 33, T // 3], H=4, Hk=1, d=64)


def test_packed_many_sequences(ops):
    """More sequences than a wave has lanes, empty ones among them."""
    packed_case(ops, [(i * 7) % 40 for i in range(200)], H=2, Hk=1, d=64)


def test_packed_no_tokens_no_sequences_no_keys(ops):
    q, k = randn(0, 4, 64), randn(0, 2, 64)
    assert ops.mha_packed_fwd(q, k, k, i32([0]), i32([0])).shape == (0, 4, 64)
    q = randn(7, 4, 64)
    assert (ops.mha_packed_fwd(q, k, k, i32([0]), i32([0])) == 0).all()
    assert (ops.mha_packed_fwd(q, k, k, i32([0, 7]), i32([0, 0])) == 0).all()
    assert (ops.mha_packed_fwd(q, k, k, i32([0, 7]), i32([0, 0]), prefix_lens=i32([5])) == 0).all()


def test_packed_strided_views(ops):
    """q, k and v as slices of one projection, padded rows, other orders of the dimensions."""
    T, H, Hk, d = 150, 4, 2, 64
    qkv = randn(T, H + 2 * Hk + 1, d, seed=4)
    q, k, v = qkv[:, :H], qkv[:, H:H + Hk], qkv[:, H + Hk:-1]
    cu = [0, 60, 150]
    want, tol = ref.packed(q, k, v, cu, cu)
    ref.check(ops.mha_packed_fwd(q, k, v, i32(cu), i32(cu)), want, tol)
    hq, hk, hv = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v))   # head-major
    ref.check(ops.mha_packed_fwd(hq, hk, hv, i32(cu), i32(cu)), want, tol)
    wide = torch.zeros(T, H, d + 8, dtype=q.dtype, device="cuda")
    wide[..., :d] = q
    ref.check(ops.mha_packed_fwd(wide[..., :d], k, v, i32(cu), i32(cu)), want, tol)


def test_packed_offsets_outside_the_tensors_are_held(ops):
    """Offsets past the ends count as the ends; nothing outside is touched."""
    q, k, v = randn(50, 2, 64, seed=1), randn(50, 2, 64, seed=2), randn(50, 2, 64, seed=3)
    got = ops.mha_packed_fwd(q, k, v, i32([0, 50]), i32([0, 50]))
    assert torch.equal(ops.mha_packed_fwd(q, k, v, i32([-7, 90]), i32([-1, 10 ** 9])), got)


# ── decode ────────────────────────────────────────────────────────────────────

def decode_case(ops, lens, H=4, Hk=2, d=128, page=16, dtype=torch.bfloat16, seed=1, cols=None, slopes=False, spoil=True, **kw):
    B = len(lens)
    held = [-(-n // page) for n in lens]
    M = max(max(held), 1) if cols is None else cols
    P = sum(held) + 2
    g = torch.Generator().manual_seed(seed)
    ids = torch.randperm(P, generator=g).tolist()
    table, at = [], 0
    for n in held:
        table.append((ids[at:at + n] + [-1] * M)[:M])
        at += n
    k, v = randn(P, Hk, page, d, seed=seed + 1, dtype=dtype), randn(P, Hk, page, d, seed=seed + 2, dtype=dtype)
    if spoil:   # what lies behind a sequence's end, and in pages of nobody, is garbage
        for b, n in enumerate(lens):
            if n % page and held[b] <= M:
                k[table[b][held[b] - 1], :, n % page:] = NAN
                v[table[b][held[b] - 1], :, n % page:] = math.inf
        for p in ids[at:]:
            k[p], v[p] = NAN, NAN
    q = randn(B, H, d, seed=seed + 3, dtype=dtype)
    s = slopes_of(H) if slopes else None
    t = i32(table)
    got = ops.mha_paged_decode(q, k, v, t, i32(lens), slopes=s, **kw)
    want, tol = ref.decode(q, k, v, t, lens, slopes=s, **kw)
    ref.check(got, want, tol, f"{lens} {page} {kw}")
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens", [[1], [0, 5, 16, 17], [31, 32, 33, 127, 128, 129], [1000, 3, 0, 511]])
def test_decode_lengths(ops, dtype, d, lens):
    decode_case(ops, lens, d=d, dtype=dtype)


@pytest.mark.parametrize("page", [8, 16, 32, 64, 1024])
def test_decode_page_sizes(ops, page):
    decode_case(ops, [1, 777, page, page + 1, 2 * page - 1], page=page)


@pytest.mark.parametrize("H,Hk", [(1, 1), (3, 1), (8, 8), (16, 1), (17, 1), (40, 2), (64, 2)])
def test_decode_head_groups(ops, H, Hk):
    decode_case(ops, [100, 333], H=H, Hk=Hk, d=64)


@pytest.mark.parametrize("window", [1, 31, 32, 33, 500, 2 ** 31 - 1])
def test_decode_window(ops, window):
    decode_case(ops, [700, 20, 33], window=window)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("softcap,slopes", [(0.0, True), (5.0, False), (50.0, True), (1000.0, False)])
def test_decode_scores(ops, dtype, d, softcap, slopes):
    decode_case(ops, [300, 1, 45], d=d, dtype=dtype, softcap=softcap, slopes=slopes, window=250)


def test_decode_long_and_many(ops):
    decode_case(ops, [20000], H=8, Hk=2, page=64, softcap=30.0)
    decode_case(ops, [(i * 37) % 900 for i in range(130)], H=4, Hk=4, d=64, page=32, slopes=True)


def test_decode_wide_table_and_long_lens(ops):
    """A table far wider than the sequences; lengths past the table count as its span; negative as 0."""
    decode_case(ops, [40, 7], cols=4096)
    q, k, v = randn(2, 4, 64, seed=1), randn(3, 2, 16, 64, seed=2), randn(3, 2, 16, 64, seed=3)
    t = i32([[2, 0], [1, 1]])
    got = ops.mha_paged_decode(q, k, v, t, i32([10 ** 9, -3]))
    want, tol = ref.decode(q, k, v, t, [32, 0])
    ref.check(got, want, tol)


def test_decode_pages_outside_the_cache_are_hidden(ops):
    q, k, v = randn(3, 4, 128, seed=1), randn(4, 2, 16, 128, seed=2), randn(4, 2, 16, 128, seed=3)
    t = i32([[0, -1, 3], [4, 2 ** 31 - 1, 1], [-2 ** 31, -1, 99]])
    got = ops.mha_paged_decode(q, k, v, t, i32([48, 48, 48]))
    want, tol = ref.decode(q, k, v, t, [48, 48, 48])
    ref.check(got, want, tol)
    assert (got[2] == 0).all()


def test_decode_empty(ops):
    k = randn(3, 2, 16, 64)
    assert ops.mha_paged_decode(randn(0, 4, 64), k, k, i32([]).view(0, 2), i32([])).shape == (0, 4, 64)
    assert (ops.mha_paged_decode(randn(2, 4, 64), k, k, i32([[], []]).view(2, 0), i32([5, 5])) == 0).all()
    none = randn(0, 2, 16, 64)
    assert (ops.mha_paged_decode(randn(2, 4, 64), none, none, i32([[0], [0]]), i32([5, 5])) == 0).all()


def test_decode_strided(ops):
    """Keys and values in one cache tensor, other orders, a table that is a slice, a q that is."""
    P, Hk, page, d, H, B = 7, 2, 16, 64, 6, 2
    both = randn(P, 2, Hk, page, d, seed=5)
    k, v = both[:, 0], both[:, 1]
    t = i32([[3, 1, 6, 0, 9], [2, 5, 4, 1, 9]])[:, :3]
    q = randn(B, H + 3, d, seed=6)[:, 1:1 + H]
    lens = [40, 33]
    want, tol = ref.decode(q, k, v, t, lens)
    ref.check(ops.mha_paged_decode(q, k, v, t, i32(lens)), want, tol)
    k2, v2 = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v))   # rows before heads
    ref.check(ops.mha_paged_decode(q, k2, v2, t, i32(lens)), want, tol)


# ── rotary positions and the cache ────────────────────────────────────────────

def rope_case(ops, T, H=4, Hk=2, d=128, rot=None, interleaved=False, dtype=torch.bfloat16, page=16, first=0, amplitude=1.0, seed=1, views=True,
              slots=None, base=10000.0):
    rot = d if rot is None else rot
    P = T // page + 3
    qkv = randn(T, H + 2 * Hk, d, seed=seed, dtype=dtype)
    q, k, v = qkv[:, :H], qkv[:, H:H + Hk], qkv[:, H + Hk:]
    if not views:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    g = torch.Generator().manual_seed(seed)
    if slots is None:
        slots = torch.randperm(P * page, generator=g)[:T].tolist()
        if T > 3:
            slots[1] = -1
    pos = i32([first + (t * 3) % max(T, 1) for t in range(T)])
    freq = ops.rotary_frequencies(rot, base, device="cuda")[0]
    kc, vc = randn(P, Hk, page, d, seed=seed + 1, dtype=dtype), randn(P, Hk, page, d, seed=seed + 2, dtype=dtype)
    kc0, vc0 = kc.clone(), vc.clone()
    qo, ko = ops.rope_paged_store(q, k, v, pos, freq, torch.tensor(slots, dtype=torch.int64, device="cuda"), kc, vc, interleaved=interleaved,
                                  amplitude=amplitude)
    for got, x in ((qo, q), (ko, k)):
        want, tol = ref.rotate(x, pos, freq, interleaved, amplitude)
        ref.check(got, want, tol)
        assert torch.equal(got[..., rot:], x[..., rot:])
    for t, s in enumerate(slots):
        if 0 <= s < P * page:
            kc0[s // page, :, s % page] = ko[t]
            vc0[s // page, :, s % page] = v[t]
    assert torch.equal(kc, kc0) and torch.equal(vc, vc0)
    return qo, ko


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rot", [0, 16, 48, 64])
def test_rope(ops, dtype, d, interleaved, rot):
    rope_case(ops, 37, d=d, rot=rot, interleaved=interleaved, dtype=dtype)


@pytest.mark.parametrize("T", [1, 2, 5, 64, 3001])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_tokens(ops, T, interleaved):
    rope_case(ops, T, interleaved=interleaved, page=8)


@pytest.mark.parametrize("H,Hk", [(1, 1), (7, 1), (64, 8), (12, 12)])
def test_rope_heads(ops, H, Hk):
    rope_case(ops, 9, H=H, Hk=Hk, views=False)


def test_rope_far_positions_and_amplitude(ops):
    rope_case(ops, 50, first=10 ** 6, dtype=torch.float16)
    rope_case(ops, 50, first=2 ** 31 - 200, dtype=torch.float16, amplitude=1.2)
    rope_case(ops, 50, first=-1000, base=5e5, amplitude=-0.5, interleaved=True)


def test_rope_slots_outside_the_cache_store_nothing(ops):
    rope_case(ops, 6, page=8, slots=[-1, 3 * 8, 2 ** 40, -2 ** 62, 5, 23])


def test_rope_cache_views(ops):
    T, H, Hk, d, page, P = 20, 4, 2, 64, 8, 5
    q, k, v = randn(T, H, d, seed=1), randn(T, Hk, d, seed=2), randn(T, Hk, d, seed=3)
    both = randn(P, 2, page, Hk, d, seed=4)
    kc, vc = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    kc0, vc0 = kc.contiguous(), vc.contiguous()
    args = (q, k, v, i32(list(range(T))), ops.rotary_frequencies(64, device="cuda")[0], torch.arange(3, 3 + T, device="cuda"))
    a, b = ops.rope_paged_store(*args, kc, vc)
    c, e = ops.rope_paged_store(*args, kc0, vc0)
    assert torch.equal(a, c) and torch.equal(b, e) and torch.equal(kc, kc0) and torch.equal(vc, vc0)


# ── layout ────────────────────────────────────────────────────────────────────

def layout_case(ops, seq, new, page=16, M=None, F=None, max_tokens=None, seed=0):
    n = len(seq)
    want_pages = [-(-(max(0, a) + max(0, b)) // page) for a, b in zip(seq, new)]
    M = max(want_pages + [1]) if M is None else M
    total = sum(max(0, b) for b in new)
    F = sum(want_pages) if F is None else F
    max_tokens = total + 3 if max_tokens is None else max_tokens
    g = torch.Generator().manual_seed(seed)
    ids = torch.randperm(n * M + F, generator=g).int()
    free, table = ids[:F], ids[F:].view(n, M)
    got = ops.paged_layout(i32(seq), i32(new), table.cuda(), free.cuda(), page, max_tokens)
    want = ref.layout(seq, new, table.tolist(), free.tolist(), page, max_tokens)
    for name, a, b in zip(("kv_lens", "cu_new", "positions", "slot_map", "table", "counts"), got, want):
        assert a.tolist() == b, name
    return got


@pytest.mark.parametrize("page", [1, 7, 16, 64])
def test_layout_steps(ops, page):
    layout_case(ops, [0, 1, 15, 16, 17, 100], [1, 1, 1, 1, 1, 1], page)
    layout_case(ops, [0, 5, 0, 33], [40, 0, 1, 100], page)


def test_layout_pages_run_out(ops):
    for F in (0, 1, 3, 5):
        layout_case(ops, [0, 10, 30], [50, 40, 20], F=F)


def test_layout_table_too_narrow(ops):
    layout_case(ops, [0, 40, 100], [60, 5, 3], M=2)
    layout_case(ops, [0, 40], [60, 5], M=0)


def test_layout_token_buffer(ops):
    layout_case(ops, [3, 0], [10, 20], max_tokens=0)
    layout_case(ops, [3, 0], [10, 20], max_tokens=13)
    layout_case(ops, [3, 0], [10, 20], max_tokens=500)


def test_layout_negative_and_empty(ops):
    layout_case(ops, [-5, 3], [2, -7])
    layout_case(ops, [0, 0], [0, 0])
    out = ops.paged_layout(i32([]), i32([]), i32([]).view(0, 4), i32([1, 2]), 16, 3)
    assert out[1].tolist() == [0] and out[3].tolist() == [-1] * 3 and out[5].tolist() == [0, 0, 0]


@pytest.mark.parametrize("n", [255, 256, 257, 1000, 8192])
def test_layout_many_requests(ops, n):
    layout_case(ops, [(i * 13) % 70 for i in range(n)], [(i * 5) % 4 for i in range(n)], F=n // 2)


def test_layout_table_slice(ops):
    table = torch.arange(30, dtype=torch.int32, device="cuda").view(3, 10)
    a = ops.paged_layout(i32([20, 0, 33]), i32([1, 2, 3]), table[:, 2:6], i32([90, 91, 92]), 16, 10)
    b = ops.paged_layout(i32([20, 0, 33]), i32([1, 2, 3]), table[:, 2:6].contiguous(), i32([90, 91, 92]), 16, 10)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


# ── what a row does not see ───────────────────────────────────────────────────

@pytest.mark.parametrize("wild", [NAN, math.inf, -math.inf])
@pytest.mark.parametrize("d,H,lens,kw", [
    (64, 2, [70, 200], {}),                                                    # 128 rows a workgroup
    (128, 2, [300, 65], dict(window=50)),
    (128, 4, [600], dict(window=33, prefix=[20])),                            # 64 rows
    (64, 4, [600], dict(softcap=9.0)),
    (128, 16, [1500, 3000, 1100], dict(window=700, slopes=True)),             # 256 rows
    (64, 2, [129], dict(causal=False, window=10)),
])
def test_packed_unseen_keys_reach_nothing(ops, wild, d, H, lens, kw):
    """Values that are not finite, in keys and values, reach only the rows that see them."""
    kw = dict(kw)
    slopes = slopes_of(H) if kw.pop("slopes", False) else None
    prefix = kw.pop("prefix", None)
    cu, Hk = cu_of(lens), max(1, H // 2)
    T = cu[-1] + 9
    q, k, v = randn(T, H, d, seed=1), randn(T, Hk, d, seed=2), randn(T, Hk, d, seed=3)
    v[cu[-1]:], k[cu[-1]:] = wild, wild             # behind the last sequence
    for c, n in zip(cu, lens):
        v[c + n // 2, 0, 5] = wild                  # one element in the middle of each sequence
        v[c + n - 1, -1] = wild                     # the last key's
        k[c + n - 2, 0, 7] = NAN
    got = ops.mha_packed_fwd(q, k, v, i32(cu), i32(cu), slopes=slopes, prefix_lens=i32(prefix) if prefix else None, **kw)
    want, tol = ref.packed(q, k, v, cu, cu, slopes=slopes, prefix_lens=prefix, **kw)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine)
    ref.check(torch.where(fine, got.double(), 0), torch.where(fine, want, 0), torch.where(fine, tol, 1), f"{lens} {kw}")


@pytest.mark.parametrize("wild", [NAN, math.inf])
@pytest.mark.parametrize("d,H,lens_q,lens_k", [(64, 2, [40], [10]), (128, 4, [300], [70]), (128, 16, [1500, 3000, 1100], [700, 2900, 1])])
def test_packed_rows_that_see_nothing_stay_0(ops, wild, d, H, lens_q, lens_k):
    """Rows in front of the first key share tiles with rows that see keys; no value reaches them."""
    cq, ck = cu_of(lens_q), cu_of(lens_k)
    q, k, v = randn(cq[-1], H, d, seed=1), randn(ck[-1], H // 2, d, seed=2), randn(ck[-1], H // 2, d, seed=3)
    for c, n in zip(ck, lens_k):
        v[c + n // 2:c + n] = wild
    got = ops.mha_packed_fwd(q, k, v, i32(cq), i32(ck))
    for c, n, m in zip(cq, lens_q, lens_k):
        assert (got[c:c + n - m] == 0).all()
        assert torch.isfinite(got[c:c + n - m + m // 2]).all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("wild", [NAN, -math.inf])
def test_packed_seen_infinity_beside_unseen_values(ops, d, wild):
    """An infinity that a row sees is its result, whatever unseen keys of the tile hold there."""
    n = 200
    q, k, v = randn(n, 2, d, seed=1), randn(n, 2, d, seed=2), randn(n, 2, d, seed=3)
    v[130, :, 5], v[150, :, 5] = math.inf, wild
    v[140, :, 6], v[150, :, 6] = NAN, wild
    got = ops.mha_packed_fwd(q, k, v, i32([0, n]), i32([0, n]))
    assert torch.isfinite(got[:130]).all()
    assert (got[130:150, :, 5] == math.inf).all() and got[150:, :, 5].isnan().all()
    assert torch.isfinite(got[:140, :, 6]).all() and got[140:, :, 6].isnan().all()
    rest = [c for c in range(d) if c not in (5, 6)]
    assert torch.isfinite(got[:, :, rest]).all()


def test_decode_unseen_keys_reach_nothing(ops):
    """Keys before the window, in the tile where it starts, hold NaN."""
    q, k, v = randn(2, 4, 128, seed=1), randn(40, 2, 16, 128, seed=2), randn(40, 2, 16, 128, seed=3)
    t = torch.arange(40, dtype=torch.int32, device="cuda").view(2, 20)
    lens = [300, 111]
    for b, n in enumerate(lens):
        for j in range(max(0, n - 45)):
            k[b * 20 + j // 16, :, j % 16] = NAN
            v[b * 20 + j // 16, :, j % 16] = math.inf
    got = ops.mha_paged_decode(q, k, v, t, i32(lens), window=45)
    want, tol = ref.decode(q, k, v, t, lens, window=45)
    assert torch.isfinite(got).all()
    ref.check(got, want, tol)


def test_seen_nan_stays(ops):
    q, k, v = randn(80, 2, 64, seed=1), randn(80, 2, 64, seed=2), randn(80, 2, 64, seed=3)
    v[3] = NAN
    out = ops.mha_packed_fwd(q, k, v, i32([0, 80]), i32([0, 80]))
    assert torch.isfinite(out[:3]).all() and out[3:].isnan().all()
    q[50, 0] = NAN
    v[3] = 0
    out = ops.mha_packed_fwd(q, k, v, i32([0, 80]), i32([0, 80]))
    assert out[50, 0].isnan().all() and torch.isfinite(out[:50]).all() and torch.isfinite(out[51:]).all()
    kc, vc = randn(3, 1, 16, 64, seed=4), randn(3, 1, 16, 64, seed=5)
    kc[1, 0, 2] = NAN
    out = ops.mha_paged_decode(randn(2, 2, 64, seed=6), kc, vc, i32([[0, 1, 2], [0, 2, 1]]), i32([48, 20]))
    assert out[0].isnan().all() and torch.isfinite(out[1]).all()


# ── streams, graphs, far offsets, a whole step ────────────────────────────────

def test_other_stream(ops):
    """The calls run on the current stream: inputs made there are seen without a wait."""
    side = torch.cuda.Stream()
    k, v = randn(64, 2, 16, 128, seed=1), randn(64, 2, 16, 128, seed=2)
    t = torch.arange(64, dtype=torch.int32, device="cuda").view(1, 64)
    q0 = randn(1, 4, 128, seed=3)
    want = ops.mha_paged_decode(q0 * 2, k, v, t, i32([1000]))
    lens = i32([1000])
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(10 ** 7)
        got = ops.mha_paged_decode(q0 * 2, k, v, t, lens)
    side.synchronize()
    assert torch.equal(got, want)


def test_results_do_not_depend_on_the_run(ops):
    """Twenty calls, and calls on two streams at once, give the same bits."""
    q, k, v = randn(3, 16, 128, seed=1), randn(600, 4, 16, 128, seed=2), randn(600, 4, 16, 128, seed=3)
    t = torch.arange(600, dtype=torch.int32, device="cuda").view(3, 200)
    lens = i32([3200, 17, 1500])
    want = ops.mha_paged_decode(q, k, v, t, lens)
    for _ in range(20):
        assert torch.equal(ops.mha_paged_decode(q, k, v, t, lens), want)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(ops.mha_paged_decode(q, k, v, t, lens))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


class Model:
    """One attention block's state and a step of it: the operators as a program runs them."""

    def __init__(self, ops, H=8, Hk=2, d=128, page=16, pages=80, N=3, M=20, dtype=torch.bfloat16, softcap=0.0, rot=64):
        self.ops, self.H, self.Hk, self.d, self.page = ops, H, Hk, d, page
        self.kc, self.vc = (torch.full((pages, Hk, page, d), NAN, dtype=dtype, device="cuda") for _ in range(2))
        self.table = torch.full((N, M), -1, dtype=torch.int32, device="cuda")
        self.lens = torch.zeros(N, dtype=torch.int32, device="cuda")
        g = torch.Generator().manual_seed(5)
        self.free = torch.randperm(pages, generator=g).int().cuda()
        self.freq, self.amp = ops.rotary_frequencies(rot, scaling="yarn", factor=4.0, original_len=64, device="cuda")
        self.softcap = softcap

    def store(self, qkv, new, max_tokens):
        o, H, Hk = self.ops, self.H, self.Hk
        lens, cu, pos, slots, table, counts = o.paged_layout(self.lens, new, self.table, self.free, self.page, max_tokens)
        q, k = o.rope_paged_store(qkv[:, :H], qkv[:, H:H + Hk], qkv[:, H + Hk:], pos, self.freq, slots, self.kc, self.vc, amplitude=self.amp)
        return q, k, qkv[:, H + Hk:], lens, cu, table, counts

    def prompt(self, qkv, new):
        q, k, v, lens, cu, table, counts = self.store(qkv, new, qkv.shape[0])
        out = self.ops.mha_packed_fwd(q, k, v, cu, cu, softcap=self.softcap)
        self.lens, self.table, self.free = lens, table, self.free[int(counts[1]):].contiguous()
        return out

    def token(self, qkv, new):
        q, _, _, lens, _, table, counts = self.store(qkv, new, qkv.shape[0])
        return self.ops.mha_paged_decode(q, self.kc, self.vc, table, lens, softcap=self.softcap), lens, table, counts


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("softcap", [0.0, 20.0])
def test_prompt_and_tokens_together(ops, dtype, softcap):
    """Prompts, then tokens one by one, against attention in 64 bits over everything seen so far:
    positions, slots, pages and lengths all have to agree for it to match."""
    m = Model(ops, dtype=dtype, softcap=softcap)
    H, Hk, d = m.H, m.Hk, m.d
    lens = [37, 1, 90]
    seen_q, seen_k, seen_v = ([[] for _ in lens] for _ in range(3))

    def rotated(qkv, at):
        pos = torch.tensor(at, device="cuda")
        y, tol = ref.rotate(qkv[:, :H + Hk], pos, m.freq, False, m.amp)
        return y.to(dtype), tol    # rounded as the operator rounds (ties apart, see below)

    def compare(got, qkv, rows):
        """rows: (request, position) of each row of got."""
        turned, _ = rotated(qkv, [p for _, p in rows])
        for i, (r, p) in enumerate(rows):
            seen_k[r].append(turned[i, H:])
            seen_v[r].append(qkv[i, H + Hk:])
        for i, (r, p) in enumerate(rows):
            k, v = torch.stack(seen_k[r])[:p + 1], torch.stack(seen_v[r])[:p + 1]
            for h in range(H):
                want, tol = ref.attend(turned[i, h:h + 1], k[:, h // (H // Hk)], v[:, h // (H // Hk)], ref.seen_mask(1, p + 1, True, 0, 0, "cuda"),
                                       scale=d ** -0.5, softcap=softcap, dtype=dtype)
                # a turned value may round the other way (its fp32 sum is off by 2^-20): a step of
                # q or k in one of d products, d times at most, moves a score by u·Σ|q·k|·2^-7
                u = ref.HALF_STEP[dtype]
                slack = 2 * (u * 2.0 ** -7) * float((turned[i, h].double().abs() @ k[:, h // (H // Hk)].double().abs().T).max()) * d ** -0.5
                ref.check(got[i, h:h + 1], want, tol + slack * (want.abs() + v.abs().double().amax()), f"request {r} position {p} head {h}")

    qkv = randn(sum(lens), H + 2 * Hk, d, seed=9, dtype=dtype)
    out = m.prompt(qkv, i32(lens))
    compare(out, qkv, [(r, p) for r, n in enumerate(lens) for p in range(n)])
    for step in range(4):
        qkv = randn(3, H + 2 * Hk, d, seed=20 + step, dtype=dtype)
        out, lens_t, table, counts = m.token(qkv, i32([1, 1, 1]))
        m.lens, m.table, m.free = lens_t, table, m.free[int(counts[1]):].contiguous()
        compare(out, qkv, [(r, n + step) for r, n in enumerate(lens)])
    assert m.lens.tolist() == [n + 4 for n in lens]


def test_step_in_a_graph(ops):
    """A captured step, replayed with other lengths, tables and tokens in its inputs, between eager
    work of the same kind and of a second graph that shares the memory pool: each replay is the
    eager result."""
    def inputs(seed):
        qkv = randn(3, 12, 128, seed=seed)
        lens = i32([100 + seed, 3 * seed, 33])
        return qkv, lens

    def fresh():
        m = Model(ops)
        m.kc.normal_()
        m.vc.normal_()
        m.table.copy_(torch.arange(60, dtype=torch.int32, device="cuda").view(3, 20))
        return m

    def eager(seed):
        torch.manual_seed(3)
        m = fresh()
        qkv, lens = inputs(seed)
        m.lens = lens
        return (*m.token(qkv, i32([1, 1, 1])), m.kc.clone(), m.vc.clone())

    torch.manual_seed(3)
    m = fresh()
    base_k, base_v = m.kc.clone(), m.vc.clone()
    qkv, lens = inputs(1)
    m.lens = lens
    one = i32([1, 1, 1])
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        m.token(qkv, one)
    torch.cuda.current_stream().wait_stream(warm)
    graphs, outs = [], []
    pool = torch.cuda.graph_pool_handle()
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            outs.append(m.token(qkv, one))
        graphs.append(g)
    for round_, seed in enumerate([1, 4, 2, 7, 4, 1]):
        want = eager(seed)
        q2, l2 = inputs(seed)
        qkv.copy_(q2)
        lens.copy_(l2)
        m.kc.copy_(base_k)
        m.vc.copy_(base_v)
        i = round_ % 2
        graphs[i].replay()
        torch.cuda.synchronize()
        for a, b in zip((*outs[i], m.kc, m.vc), want):
            assert torch.equal(a, b), (round_, seed)


def test_cache_offsets_past_32_bits(ops):
    """A cache of more than 2^32 elements: pages at its far end are written and read."""
    P, Hk, page, d = 2 ** 32 // (2 * 16 * 128) + 40, 2, 16, 128
    kc, vc = (torch.empty(P, Hk, page, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    T, H = 100, 4
    far = [P - 1 - i * 2 for i in range(7)]
    slots = torch.tensor([far[t // page] * page + t % page for t in range(T)], device="cuda")
    q, k, v = randn(T, H, d, seed=1), randn(T, Hk, d, seed=2), randn(T, Hk, d, seed=3)
    freq = ops.rotary_frequencies(d, device="cuda")[0]
    qo, ko = ops.rope_paged_store(q, k, v, i32(list(range(T))), freq, slots, kc, vc)
    small = torch.stack([kc[p] for p in far]), torch.stack([vc[p] for p in far])
    assert torch.equal(small[0].transpose(1, 2).reshape(-1, Hk, d)[:T], ko)
    got = ops.mha_paged_decode(qo[-1:], kc, vc, i32([far]), i32([T]))
    assert torch.equal(got, ops.mha_paged_decode(qo[-1:], *small, i32([list(range(7))]), i32([T])))
    del kc, vc
    torch.cuda.empty_cache()


def test_packed_offsets_past_32_bits(ops):
    """Rows so far apart that their offsets pass 2^32 elements."""
    d, H, Hk, T, step = 64, 2, 1, 1100, 2 ** 22 + 64
    raw = torch.empty(T * step, dtype=torch.bfloat16, device="cuda")
    x = raw.as_strided((T, H + 2 * Hk, d), (step, d, 1))
    x.copy_(randn(T, H + 2 * Hk, d, seed=3))
    cu = i32([0, 30, T])
    far = ops.mha_packed_fwd(x[:, :H], x[:, H:H + Hk], x[:, H + Hk:], cu, cu)
    y = x.contiguous()
    assert torch.equal(far, ops.mha_packed_fwd(y[:, :H], y[:, H:H + Hk], y[:, H + Hk:], cu, cu))
    del raw, x
    torch.cuda.empty_cache()


# ── refusals ──────────────────────────────────────────────────────────────────

def refused(text, f, *args, **kw):
    with pytest.raises(RuntimeError, match=text):
        f(*args, **kw)


def test_refusals_packed(ops):
    q, k, cu = randn(8, 4, 64), randn(8, 2, 64), i32([0, 8])
    f = ops.mha_packed_fwd
    refused("float16 or bfloat16", f, q.float(), k.float(), k.float(), cu, cu)
    refused("k dtype must match q", f, q, k.half(), k, cu, cu)
    refused("k must be a CUDA tensor", f, q, k.cpu(), k, cu, cu)
    refused("q must be 3D", f, q[0], k, k, cu, cu)
    refused("head_dim mismatch", f, q, randn(8, 2, 128), k, cu, cu)
    refused("token count mismatch", f, q, k, k[:7], cu, cu)
    refused("n_kv_heads mismatch", f, q, k, randn(8, 1, 64), cu, cu)
    refused("divisible", f, randn(8, 3, 64), k, k, cu, cu)
    refused("Only head_dim", f, randn(8, 4, 96), randn(8, 2, 96), randn(8, 2, 96), cu, cu)
    refused("innermost stride", f, randn(8, 64, 4).transpose(1, 2), k, k, cu, cu)
    refused("multiples of 8", f, randn(8, 4, 65)[..., :64], k, k, cu, cu)
    refused("16-byte aligned", f, randn(8 * 4 * 64 + 8)[4:-4].view(8, 4, 64), k, k, cu, cu)
    refused("cu_q must be", f, q, k, k, cu.long(), cu)
    refused("cu_k must have", f, q, k, k, cu, i32([0, 4, 8]))
    refused("cu_q must be 1D", f, q, k, k, i32([]), i32([]))
    refused("prefix_lens must have", f, q, k, k, cu, cu, prefix_lens=i32([1, 2]))
    refused("slopes must be float32", f, q, k, k, cu, cu, slopes=slopes_of(4).double())
    refused("slopes must be contiguous with 4", f, q, k, k, cu, cu, slopes=slopes_of(3))
    for bad in (0.0, -1.0, math.inf, NAN):
        refused("scale", f, q, k, k, cu, cu, scale=bad)
    for bad in (-1.0, 1000.5, math.inf, NAN):
        refused("softcap", f, q, k, k, cu, cu, softcap=bad)
    refused("window", f, q, k, k, cu, cu, window=-1)
    refused("forward only", f, q.clone().requires_grad_(), k, k, cu, cu)
    with torch.no_grad():
        f(q.clone().requires_grad_(), k, k, cu, cu)


def test_refusals_decode(ops):
    q, k, t, n = randn(2, 4, 64), randn(5, 2, 16, 64), i32([[0, 1], [2, 3]]), i32([20, 30])
    f = ops.mha_paged_decode
    refused("float16 or bfloat16", f, q.float(), k, k, t, n)
    refused("v_cache dtype", f, q, k, k.half(), t, n)
    refused("k_cache must be 4D", f, q, k[0], k, t, n)
    refused("same shape", f, q, k, k[:4], t, n)
    refused("head_dim mismatch", f, q, randn(5, 2, 16, 128), randn(5, 2, 16, 128), t, n)
    refused("divisible", f, randn(2, 3, 64), k, k, t, n)
    for page in (4, 24, 2048):
        refused("page_size", f, q, randn(5, 2, page, 64), randn(5, 2, page, 64), t, n)
    refused("block_table must be int32", f, q, k, k, t.long(), n)
    refused("block_table must be int32", f, q, k, k, t[:1], n)
    refused("block_table must have an innermost", f, q, k, k, i32([[0, 2], [1, 3]]).t(), n)
    refused("kv_lens must be", f, q, k, k, t, n.long())
    refused("kv_lens must have", f, q, k, k, t, i32([1]))
    refused("window", f, q, k, k, t, n, window=2 ** 31)
    refused("slopes", f, q, k, k, t, n, slopes=slopes_of(4).half())
    refused("forward only", f, q, k.clone().requires_grad_(), k, t, n)


def test_refusals_rope(ops):
    T = 5
    q, k, pos, slots = randn(T, 4, 64), randn(T, 2, 64), i32(range(T)), torch.arange(T, device="cuda")
    freq, kc, vc = ops.rotary_frequencies(64, device="cuda")[0], randn(3, 2, 16, 64), randn(3, 2, 16, 64)
    f = ops.rope_paged_store
    refused("positions must be", f, q, k, k, pos.long(), freq, slots, kc, vc)
    refused("slot_map must be", f, q, k, k, pos, freq, slots.int(), kc, vc)
    refused("slot_map must have", f, q, k, k, pos, freq, slots[:4], kc, vc)
    refused("inv_freq must be", f, q, k, k, pos, freq.float(), slots, kc, vc)
    refused("inv_freq must be 1D", f, q, k, k, pos, freq[:12], slots, kc, vc)
    refused("inv_freq must be 1D", f, q, k, k, pos, torch.cat([freq, freq]), slots, kc, vc)
    refused("token count", f, q, k[:4], k, pos, freq, slots, kc, vc)
    refused("k_cache must be", f, q, k, k, pos, freq, slots, randn(3, 1, 16, 64), vc)
    refused("same shape", f, q, k, k, pos, freq, slots, kc, vc[:2])
    refused("single memory location", f, q, k, k, pos, freq, slots, kc[:1].expand(3, 2, 16, 64), vc)
    refused("overlap|same memory|single memory", f, q, k, k, pos, freq, slots, kc, kc)
    refused("amplitude", f, q, k, k, pos, freq, slots, kc, vc, amplitude=NAN)
    inner = kc.view(-1)[: T * 2 * 64].view(T, 2, 64)
    refused("overlap|same memory|single memory", f, q, inner, k, pos, freq, slots, kc, vc)
    refused("overlap|same memory|single memory", f, q, k, inner, pos, freq, slots, kc, vc)
    refused("forward only", f, q, k.clone().requires_grad_(), k, pos, freq, slots, kc, vc)


def test_refusals_of_launches_past_32_bits(ops):
    """2^24 workgroups of 256 threads are more than a launch counts."""
    T = 2 ** 24
    row, pos = randn(1, 1, 64), torch.zeros(T, dtype=torch.int32, device="cuda")
    freq, c = ops.rotary_frequencies(64, device="cuda")[0], torch.zeros(2, 1, 1, 16, 64, dtype=torch.bfloat16, device="cuda")
    x = row.expand(T, 1, 64)
    refused("too large", ops.rope_paged_store, x, x, x, pos, freq, pos.long(), c[0], c[1])
    t = torch.zeros(1, 1, dtype=torch.int32, device="cuda").expand(T, 1)
    refused("too large", ops.mha_paged_decode, x, c[0], c[1], t, pos)


def test_refusals_layout(ops):
    a, t, fr = i32([1, 2]), i32([[0, 1], [2, 3]]), i32([4, 5])
    f = ops.paged_layout
    refused("seq_lens must be a CUDA", f, a.cpu(), a, t, fr, 16, 8)
    refused("new_lens must have", f, a, a[:1], t, fr, 16, 8)
    refused("new_lens must be", f, a, a.long(), t, fr, 16, 8)
    refused("block_table", f, a, a, t.long(), fr, 16, 8)
    refused("block_table", f, a, a, t[:1], fr, 16, 8)
    refused("free_pages", f, a, a, t, fr.long(), 16, 8)
    refused("free_pages", f, a, a, t, t, 16, 8)
    refused("page_size", f, a, a, t, fr, 0, 8)
    refused("max_tokens", f, a, a, t, fr, 16, -1)
    many = torch.zeros(8193, dtype=torch.int32, device="cuda")
    refused("at most 8192", f, many, many, many.view(-1, 1), fr, 16, 8)


def test_decode_more_requests_than_are_scanned(ops):
    """Beyond 1024 requests a workgroup serves a request each, whatever its length."""
    decode_case(ops, [(i * 7) % 50 for i in range(1100)] + [900], H=2, Hk=1, d=64)
