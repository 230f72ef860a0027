"""Packed attention over keys whose rows overlap in memory: one key, one row expanded over
all tokens, rows that start 8 elements apart. Nothing of them is found behind the last key."""
import math

import pytest
import torch

from tests import _serve_ref as ref

pytestmark = pytest.mark.gpu


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


@pytest.mark.parametrize("wild", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("d", [64, 128])
def test_one_key(ops, d, wild):
    """The rows that see it get its value, which is no copy of it behind the end times 0."""
    q, k, v = randn(5, 4, d, seed=1), randn(1, 2, d, seed=2), randn(1, 2, d, seed=3)
    v[0, :, 5] = wild
    want = v.repeat_interleave(2, dim=1)
    for causal in (False, True):
        for _ in range(5):
            out = ops.mha_packed_fwd(q, k, v, i32([0, 5]), i32([0, 1]), causal=causal)
            seen = out[4:] if causal else out
            assert torch.equal(seen.nan_to_num(nan=7.0), want.expand_as(seen).nan_to_num(nan=7.0))
            assert not causal or (out[:4] == 0).all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("T,H", [(1, 2), (70, 2), (610, 2), (4100, 8), (5003, 16)])   # each shape of workgroup
def test_values_expanded_over_the_tokens(ops, T, H, d):
    """Softmax weights sum to 1, so each row is that value: P is rounded and normalised by the
    sum of the rounded, so only the sums in fp32 and the output's rounding are left."""
    q, k, v = randn(T, H, d, seed=1), randn(T, H // 2, d, seed=2), randn(1, H // 2, d, seed=3)
    v[0, :, 5] = math.inf
    cu = i32([0, T])
    for _ in range(5):
        out = ops.mha_packed_fwd(q, k, v.expand(T, H // 2, d), cu, cu).double()
        want = v.repeat_interleave(2, dim=1).double().expand(T, H, d)
        assert (out[..., 5] == math.inf).all()
        rest = [c for c in range(d) if c != 5]
        tol = (ref.HALF_STEP[torch.bfloat16] + 2 * T * 2.0 ** -24 + 2.0 ** -20) * want.abs()
        ref.check(out[..., rest], want[..., rest], tol[..., rest])


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("T,step", [(70, 0), (70, 8), (129, 24), (610, 8)])
def test_keys_and_values_overlap(ops, T, step, d):
    q = randn(T, 4, d, seed=1)
    raw = randn(2, 2, T * step + d, seed=2)
    k, v = (x.as_strided((T, 2, d), (step, x.stride(0), 1), x.storage_offset()) for x in raw)
    cu = [0, T // 3, T]
    want, tol = ref.packed(q, k, v, cu, cu)
    ref.check(ops.mha_packed_fwd(q, k, v, i32(cu), i32(cu)), want, tol)


@pytest.mark.parametrize("d", [64, 128])
def test_one_row_of_any_stride(ops, d):
    """Through the C entry: the output of a single row is that row, whatever its token stride."""
    import ctypes

    from custom_ops_amd import build
    from tests.test_serve import Packed, call, make
    q, k, v = randn(1, 4, d, seed=1), randn(40, 2, d, seed=2), randn(40, 2, d, seed=3)
    cq, ck = i32([0, 1]), i32([0, 40])
    want = ops.mha_packed_fwd(q, k, v, cq, ck)
    lib = ctypes.CDLL(build.SERVE_LIB_PATH)
    for o_ts in (0, 8, 4 * d):
        out = torch.full_like(q, 3.0)
        torch.cuda.synchronize()
        rc = call(lib, "mi355_packed_fwd", make(Packed, dict(
            q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), o=out.data_ptr(), cu_q=cq.data_ptr(), cu_k=ck.data_ptr(), q_ts=4 * d, q_hs=d,
            k_ts=2 * d, k_hs=d, v_ts=2 * d, v_hs=d, o_ts=o_ts, o_hs=d, total_q=1, total_k=40, n_seqs=1, h=4, h_k=2, d=d, dtype=1, causal=1,
            window=0, scale=1.0 / d ** 0.5, softcap=0.0)))
        torch.cuda.synchronize()
        assert rc == (0, "") and torch.equal(out, want), (o_ts, rc)
