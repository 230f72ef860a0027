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
