"""Packed attention at d = 128 in each shape of workgroup (row waves by key groups), against the
64-bit plain form: both types, no cap and caps that take either form of the tanh, or both, with
and without a distance bias, windows, prefixes, and chunks behind a context.

The shape follows from the sizes (csrc/serve.hip): blocks of 256 rows and half a sequence each,
times heads, over 256 CUs is 4x1, over a quarter of them 4x2; below, keys of more than 512 a
sequence 2x4, else 2x2. A block holds 128 rows (4x1, 4x2) or 64 of all heads it packs."""
import pytest
import torch

from tests import _serve_ref as ref

pytestmark = pytest.mark.gpu

#        rows of each sequence, heads, KV heads
CASES = {"4x1": ([1000, 1, 900, 1537, 960], 16, 4),
         "4x1, no shared heads": ([1900, 2300], 16, 16),
         "4x2": ([700, 33, 1467], 8, 8),
         "2x4": ([650, 651], 4, 2),
         "2x2": ([200, 0, 97], 4, 1)}


@pytest.fixture(scope="module")
def ops(gpu):
    from custom_ops_amd import ops as o
    o.ensure_loaded("serve")
    return o


def shape_of(lens, keys, H):
    full = (-(-sum(lens) // 256) + len(lens) // 2) * H
    return "4x1" if full > 256 else "4x2" if full > 64 else "2x4" if sum(keys) // len(keys) > 512 else "2x2"


def inputs(lens, keys, H, Hk, dtype):
    g = torch.Generator(device="cuda").manual_seed(7)
    cq, ck = [0], [0]
    for a, b in zip(lens, keys):
        cq.append(cq[-1] + a)
        ck.append(ck[-1] + b)
    q, k, v = (torch.randn(t + 3, h, 128, generator=g, device="cuda").to(dtype) for t, h in ((cq[-1], H), (ck[-1], Hk), (ck[-1], Hk)))
    return q, k, v, cq, ck


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("slopes", [False, True])
@pytest.mark.parametrize("softcap,scale", [(0.0, None), (50.0, None), (5.0, None), (50.0, 3.0)])
@pytest.mark.parametrize("case", CASES)
def test_shapes(ops, case, softcap, scale, slopes, dtype):
    lens, H, Hk = CASES[case]
    assert shape_of(lens, lens, H) == case[:3]
    q, k, v, cu, _ = inputs(lens, lens, H, Hk, dtype)
    s = torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], device="cuda") if slopes else None
    for kw in (dict(), dict(window=300, prefix_lens=[70 * (n % 2) for n in range(len(lens))])):
        got = ops.mha_packed_fwd(q, k, v, i32(cu), i32(cu), softcap=softcap, scale=scale, slopes=s,
                                 **{x: i32(y) if x == "prefix_lens" else y for x, y in kw.items()})
        want, tol = ref.packed(q, k, v, cu, cu, softcap=softcap, scale=scale, slopes=s, **kw)
        ref.check(got, want, tol, f"{case} {kw}")
        assert (got[cu[-1]:] == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("softcap,causal", [(0.0, True), (20.0, True), (20.0, False)])
@pytest.mark.parametrize("case", CASES)
def test_chunks_behind_a_context(ops, case, softcap, causal, dtype):
    lens, H, Hk = CASES[case]
    keys = [n + 5 + 100 * (i % 3) for i, n in enumerate(lens)]
    q, k, v, cq, ck = inputs(lens, keys, H, Hk, dtype)
    got = ops.mha_packed_fwd(q, k, v, i32(cq), i32(ck), softcap=softcap, causal=causal)
    want, tol = ref.packed(q, k, v, cq, ck, softcap=softcap, causal=causal)
    ref.check(got, want, tol, case)
