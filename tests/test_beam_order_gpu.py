"""GPU tests of the order among candidates whose scores are the same in 64 bits: the lower beam,
then the larger logit, then the lower token, however many are asked for and however rows are split."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(gpu):
    from custom_ops_amd import ops
    ops.ensure_loaded("beam")
    return ops


def best_of(x, scores, k):
    """(tokens, parents, scores) of one search by the definition, on the host, in 64 bits."""
    W, V = x.shape
    x = x.double().cpu()
    every = []
    for w in range(W):
        top = x[w].max()
        s = float(scores[w]) + (x[w] - (top + torch.log(torch.exp(x[w] - top).sum())))
        first = x[w].sort(descending=True, stable=True).indices[:k]   # a row's are in the order of its logits
        every += [(-float(s[v]), w, -float(x[w, v]), int(v)) for v in first]
    every.sort()
    best = every[:k]
    return [v for _, _, _, v in best], [w for _, w, _, _ in best], [-s for s, _, _, _ in best]


def agrees(ops, x, scores, k):
    """One search by itself (many parts a row) and among 1200 (a part a row): the same, and as defined."""
    W, V = x.shape
    tokens, parents, values = best_of(x, scores, k)
    n = len(tokens)
    one = ops.beam_select(x[None], scores[None], k)
    assert one[1][0, :n].tolist() == tokens and one[2][0, :n].tolist() == parents
    for got, want in zip(one[0][0, :n].tolist(), values):
        assert abs(got - want) <= 2.0 ** -24 * abs(want) + 1e-10
    G = max(1, 1200 // W)
    many = ops.beam_select(x[None].expand(G, W, V), scores[None].expand(G, W).contiguous(), k)
    assert torch.equal(many[0], one[0].expand(G, k)) and torch.equal(many[1], one[1].expand(G, k))
    step = W * torch.arange(G, device="cuda", dtype=torch.int32)[:, None]
    assert torch.equal(torch.where(many[2] >= 0, many[2] - step, -1), one[2].expand(G, k))


@pytest.mark.parametrize("k", [1, 2, 5, 64])
@pytest.mark.parametrize("V", [20, 700, 2500, 40001])
@pytest.mark.parametrize("score", [-3e38, -1e9])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_scores_that_swallow_the_logits(ops, k, V, score, dtype):
    """Running scores so large that a row's candidates have few values in 64 bits, or one."""
    g = torch.Generator(device="cuda").manual_seed(V + k)
    x = torch.randn(1, V, generator=g, device="cuda")
    if score == -1e9:   # (a step of 1.2e-7: neighbours share it)
        x = x * 1e-7 if dtype == torch.float32 else x * 1e-3
    agrees(ops, x.to(dtype).expand(3, V), torch.full((3,), score, device="cuda"), k)


@pytest.mark.parametrize("k", [1, 2, 5, 64])
@pytest.mark.parametrize("V", [20, 700, 2500, 40001])
def test_logits_closer_than_the_scores(ops, k, V):
    """Logits whose differences are lost beside the row's logarithm."""
    g = torch.Generator(device="cuda").manual_seed(V - k)
    x = torch.randint(-50, 51, (2, V), generator=g, device="cuda").float() * 1e-20
    agrees(ops, x, torch.zeros(2, device="cuda"), k)


def test_tokens_beside_a_far_larger_one(ops):
    """All but one token of a row at the same distance in 64 bits."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(2, 3000, generator=g, device="cuda")
    x[:, 1234] = 3e38
    agrees(ops, x, torch.tensor([-1.0, -2.0], device="cuda"), 9)
    assert math.isfinite(float(ops.beam_select(x[None], torch.zeros(1, 2, device="cuda"), 9)[0][0, 8]))
