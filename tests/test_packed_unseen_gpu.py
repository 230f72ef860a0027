"""Packed attention, to the bit: a row's result does not change with keys that it does not
see, nor with what an earlier launch left in the LDS.

Each shape of workgroup has its sizes here, by the rule in csrc/serve.hip (blocks of 256
rows times heads, against the 256 CUs): 2 row waves by 2 key groups, 2 by 4, 4 by 2, 4 by 1."""
import pytest
import torch

pytestmark = pytest.mark.gpu

SHAPES = {"2x2": (100, 2), "2x4": (600, 2), "4x2": (4096, 8), "4x1": (5000, 16)}   # tokens, heads


@pytest.fixture(scope="module")
def ops(gpu):
    from custom_ops_amd import ops as o
    o.ensure_loaded("serve")
    return o


def qkv(T, H, d, dtype, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(T, h, d, generator=g, device="cuda").to(dtype) for h in (H, max(1, H // 2), max(1, H // 2))]


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("softcap", [0.0, 50.0, 1000.0])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("shape", SHAPES)
def test_unseen_keys_change_no_bit(ops, shape, d, softcap, dtype):
    """Keys in front of the window of the last rows, and behind the first ones, grow a hundredfold:
    |z| of their scores passes 1/2, where capped scores take another form of the tanh."""
    T, H = SHAPES[shape]
    q, k, v = qkv(T, H, d, dtype)
    cu, window = i32([0, T]), 20
    at = T // 2 // 64 * 64 + 6      # inside a tile of 64 keys and one of 32
    big = k.clone()
    big[at:at + 3] *= 100
    for kw in (dict(), dict(window=window)):
        a, b = (ops.mha_packed_fwd(q, x, v, cu, cu, softcap=softcap, **kw) for x in (k, big))
        assert torch.equal(a[:at], b[:at])
        assert not torch.equal(a[at:at + 3], b[at:at + 3])   # those rows do see them
        if kw:
            assert torch.equal(a[at + 2 + window:], b[at + 2 + window:])


@pytest.mark.parametrize("softcap", [0.0, 50.0, 1000.0])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("shape", SHAPES)
def test_equal_calls_give_equal_bits(ops, shape, d, softcap):
    """A last tile of 4 to 36 keys beside rows of K that nothing loaded: what a launch of large
    keys left there, or one of small keys."""
    T, H = SHAPES[shape]
    q, k, v = qkv(T, H, d, torch.bfloat16)
    cu = i32([0, T])
    want = ops.mha_packed_fwd(q, k, v, cu, cu, softcap=softcap)
    for factor in (1000, 0, 1000, 0):
        ops.mha_packed_fwd(q, k * factor, v, cu, cu)
        assert torch.equal(ops.mha_packed_fwd(q, k, v, cu, cu, softcap=softcap), want), factor
