"""GPU tests of selections over the largest vocabularies that a call takes: the last part's
tokens count and can be chosen, where a row is cut finely and where a part is cut at 2^30."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(gpu):
    from custom_ops_amd import ops
    ops.ensure_loaded("beam")
    return ops


def planted(V, places, dtype):
    """Logits of 0 but for one after the other at `places`, and the scores that follow."""
    x = torch.zeros(1, 1, V, dtype=dtype, device="cuda")
    values = [3.0 + 0.5 * i for i in range(len(places))]
    for p, v in zip(places, values):
        x[0, 0, p] = v
    total = math.log(sum(math.exp(v) for v in values) + (V - len(places)))
    return x, [v - total for v in values]


def close(got, want):
    """One rounding of a value that 64 bits give to 10^-12 of the sum's logarithm."""
    assert abs(got - want) <= 2.0 ** -24 * abs(want) + 1e-10, (got, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("k", [4, 64])
def test_largest_vocabulary(ops, dtype, k):
    V = 2 ** 31 - 1
    places = [0, 2 ** 30, V - 2 ** 21, V - 9, V - 1]
    x, want = planted(V, places, dtype)
    s, t, p = ops.beam_select(x, torch.zeros(1, 1, device="cuda"), k)
    best = list(zip(places, want))[::-1][:k]
    assert t[0, :len(best)].tolist() == [v for v, _ in best]
    assert (p == 0).all()
    for i, (_, w) in enumerate(best):
        close(float(s[0, i]), w)
    # the others: the lowest tokens that hold 0
    rest = [v for v in range(70) if v not in places][:k - len(best)] if k > len(best) else []
    assert t[0, len(best):].tolist() == rest


def test_parts_cut_at_their_most(ops):
    """So many rows that each would be one part, of more tokens than a part holds."""
    V, G, k = 2 ** 30 + 7, 129, 33
    places = [5, 2 ** 30 - 1, 2 ** 30, V - 1]
    x, want = planted(V, places, torch.float16)
    s, t, p = ops.beam_select(x.expand(G, 1, V), torch.zeros(G, 1, device="cuda"), k)
    best = list(zip(places, want))[::-1]
    rest = [v for v in range(60) if v not in places][:k - len(best)]
    assert t.tolist() == [[v for v, _ in best] + rest] * G
    assert p.tolist() == [[g] * k for g in range(G)]
    for i, (_, w) in enumerate(best):
        close(float(s[0, i]), w)
    assert (s == s[:1]).all()
