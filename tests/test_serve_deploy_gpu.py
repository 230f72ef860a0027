"""A sealed deployment of the serving operators, loaded in strict mode in a fresh
process on the GPU, gives the in-tree build's results."""
import os
import subprocess
import sys
import textwrap

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "custom_ops_amd", "deploy", "libmi355_serve.so")

CALLS = """
import torch
def results(ops):
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(50, 6, 64, generator=g, device="cuda").half()
    cu = torch.tensor([0, 20, 50], dtype=torch.int32, device="cuda")
    kc, vc = torch.randn(2, 4, 1, 16, 64, generator=g, device="cuda").half()
    t = torch.tensor([[0, 3], [2, 1]], dtype=torch.int32, device="cuda")
    n = torch.tensor([17, 30], dtype=torch.int32, device="cuda")
    return [ops.mha_packed_fwd(x[:, :4], x[:, 4:5], x[:, 5:], cu, cu), ops.mha_paged_decode(x[:2, :4], kc, vc, t, n),
            *ops.paged_layout(n, n, t, t[0], 16, 60)]
"""


@pytest.mark.gpu
def test_deployment(gpu, tmp_path):
    if not os.path.exists(LIB):
        pytest.skip("no deployment exported (run __graft_entry__.build())")
    code = textwrap.dedent(f"""
        import sys
        sys.path.insert(0, {ROOT!r})
        from custom_ops_amd import ops, serve
        ops.load_precompiled("serve", {LIB!r})
        assert not ops.allow_jit and serve.loaded_path() == {os.path.realpath(LIB)!r}
    """) + CALLS + f"torch.save(results(ops), {str(tmp_path / 'out.pt')!r})\n"
    res = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=110)
    assert res.returncode == 0, res.stderr[-3000:]
    ns = {}
    exec(CALLS, ns)
    from custom_ops_amd import ops
    ops.ensure_loaded("serve")
    for a, b in zip(torch.load(tmp_path / "out.pt", weights_only=True), ns["results"](ops)):
        assert torch.equal(a, b)
