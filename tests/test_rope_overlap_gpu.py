"""rope_paged_store writes both caches: ones that share memory are refused, in views that are not
dense too, and K and V side by side in one tensor are not."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(gpu):
    from custom_ops_amd import ops as o
    o.ensure_loaded("serve")
    return o


def store(ops, kc, vc):
    T, Hk, d = 4, kc.shape[1], kc.shape[3]
    x = torch.zeros(T, Hk, d, dtype=torch.bfloat16, device="cuda")
    at = torch.arange(T, dtype=torch.int32, device="cuda")
    return ops.rope_paged_store(x, x, x, at, ops.rotary_frequencies(d, device="cuda")[0], at.long(), kc, vc)


BASES = {   # what holds both, and how a cache [pages, heads, rows, d] is cut from it at one of its places
    "pages": ((6, 2, 2, 16, 64), lambda x, i: x[:, i]),
    "rows first": ((6, 2, 16, 2, 64), lambda x, i: x[:, i].transpose(1, 2)),
    "heads": ((6, 4, 16, 64), lambda x, i: x[:, 2 * i:2 * i + 2]),
    "columns": ((6, 2, 16, 128), lambda x, i: x[..., 64 * i:64 * i + 64]),
    "alternate rows": ((6, 2, 32, 64), lambda x, i: x[:, :, i::2]),
}


@pytest.mark.parametrize("name", BASES)
def test_caches_in_one_tensor(ops, name):
    shape, cut = BASES[name]
    base = torch.zeros(shape, dtype=torch.bfloat16, device="cuda")
    store(ops, cut(base, 0), cut(base, 1))
    store(ops, cut(base, 1), cut(base, 0))
    for i in (0, 1):
        with pytest.raises(RuntimeError, match="overlap|same memory|single memory"):
            store(ops, cut(base, i), cut(base, i))
    a, b = cut(base, 0)[:4], cut(base, 0)[2:]
    assert a.shape == b.shape
    for x, y in ((a, b), (b, a)):
        with pytest.raises(RuntimeError, match="overlap|same memory|single memory"):
            store(ops, x, y)
    store(ops, cut(base, 0)[:3], cut(base, 0)[3:])


def test_heads_that_overlap_in_part(ops):
    base = torch.zeros(6, 4, 16, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="overlap|same memory|single memory"):
        store(ops, base[:, 0:2], base[:, 1:3])
    with pytest.raises(RuntimeError, match="overlap|same memory|single memory"):
        store(ops, base[1:, 2:4], base[:-1, 1:3])   # one page apart, one head in common
