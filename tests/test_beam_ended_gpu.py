"""GPU tests of shared prefixes where a group's first requests have ended: rows that a fork
left empty are passed over, a row that still names its pages is read."""
import pytest
import torch

from tests import _beam_ref as ref
from tests._beam_ref import check
from tests.test_beam_gpu import batch, ints

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(gpu):
    from custom_ops_amd import ops
    ops.ensure_loaded("beam", "serve")
    return ops


def led(x):
    """The same batch with each group's prefix in the row of its first request, for the plain form."""
    table, P = x["table"].clone(), x["kc"].shape[0]
    for a, b in zip(x["cu"], x["cu"][1:]):
        first = next((r for r in range(a, b) if x["lens"][r] > 0 or 0 <= int(x["table"][r, 0]) < P), a)
        if b > a and first != a:   # (row a has no keys, so only the prefix is read of it)
            table[a] = x["table"][first]
    return table


def run(ops, x, **kw):
    out = ops.mha_shared_decode(x["q"], x["kc"], x["vc"], x["table"], ints(x["lens"]), ints(x["cu"]), ints(x["prefix"]), **kw)
    want, tol = ref.shared(x["q"], x["kc"], x["vc"], led(x), x["lens"], x["cu"], x["prefix"], **kw)
    check(out, want, tol)
    for b, n in enumerate(x["lens"]):
        assert n > 0 or (out[b] == 0).all()
    return out


def end(x, rows, entry=-1):
    for r in rows:
        x["lens"][r] = 0
        x["table"][r] = entry


# Columns of a KV head of a group of 5: a workgroup of 32, 64 or 128 of them.
@pytest.mark.parametrize("H", [8, 16, 32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("ended", [[0], [0, 1], [0, 1, 2, 3], [0, 5], [1, 6, 9], [0, 1, 2, 3, 4], list(range(10))])
@pytest.mark.parametrize("entry", [-1, 10 ** 6])
def test_rows_left_empty(ops, H, d, ended, entry):
    x = batch(H + d, [(330, 5), (141, 5)], 60, H, 2, d, 16, torch.bfloat16, alone=1)
    end(x, ended, entry)
    run(ops, x)
    run(ops, x, softcap=20.0, window=250)


def test_a_row_kept_for_its_prefix(ops):
    """An ended first request whose row names the prefix, which the others' rows do not."""
    x = batch(3, [(160, 4), (99, 3)], 30, 4, 2, 128, 16, torch.bfloat16, own=False)
    x["lens"][0] = x["lens"][4] = 0
    out = run(ops, x)
    y = batch(3, [(160, 4), (99, 3)], 30, 4, 2, 128, 16, torch.bfloat16, own=True)
    y["lens"][0] = y["lens"][4] = 0
    assert torch.equal(out, run(ops, y))


@pytest.mark.parametrize("d", [64, 128])
def test_many_groups(ops, d):
    """More requests and groups than one wave plans, the first of every other group ended."""
    x = batch(15, [(70 + i % 50, 1 + i % 4) for i in range(60)], 40, 2, 1, d, 16, torch.bfloat16, alone=9)
    end(x, x["cu"][:-1:2])
    run(ops, x)


def test_a_fork_that_ends_the_first(ops):
    """Samples of one prompt of which the first, then the second, ends: the others attend as each would by itself."""
    page, P, H, Hk, d, T, W = 16, 60, 8, 2, 64, 53, 5
    g = torch.Generator(device="cuda").manual_seed(5)
    kc, vc = (torch.randn(P, Hk, page, d, generator=g, device="cuda").bfloat16() for _ in range(2))
    table = ints([[9, 4, 30, 17, -1, -1]])
    lens = ints([T])
    table, lens, src, dst, free, _ = ops.paged_fork(table, lens, ints([0] * W), page, P)
    ops.paged_copy(kc, vc, src, dst)
    for parents in ([0, 1, 2, 3, 4], [-1, 1, 2, 3, 4], [-1, -1, 2, 4, 3], [-1, -1, -1, 3, 4], [3, -1, -1, 3, 4]):
        table, lens, src, dst, free, counts = ops.paged_fork(table, lens, ints(parents), page, P)
        ops.paged_copy(kc, vc, src, dst)
        q = torch.randn(W, H, d, generator=g, device="cuda").bfloat16()
        out = ops.mha_shared_decode(q, kc, vc, table, lens, ints([0, W]), ints([T]))
        want, tol = ref.shared(q, kc, vc, table, lens.tolist(), [0], [])
        check(out, want, tol)
        assert [bool((o != 0).any()) for o in out] == [p >= 0 for p in parents]


def test_replays_as_requests_end(ops):
    """One captured call, replayed as requests end one after the other, with eager calls between."""
    x = batch(8, [(200, 4), (90, 3)], 40, 8, 2, 64, 16, torch.bfloat16)
    lens, cu, prefix = ints(x["lens"]), ints(x["cu"]), ints(x["prefix"])
    args = (x["q"], x["kc"], x["vc"], x["table"], lens, cu, prefix)
    ops.mha_shared_decode(*args)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = ops.mha_shared_decode(*args)
    for row in (None, 0, 4, 1, 6, 2):
        if row is not None:
            end(x, [row])
            lens.copy_(ints(x["lens"]))
        graph.replay()
        got = held.clone()
        assert torch.equal(got, run(ops, x))
        torch.cuda.synchronize()
