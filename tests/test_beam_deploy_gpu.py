"""A sealed deployment of the operators for several continuations of a prompt, loaded in
strict mode in a fresh process on the GPU, gives the in-tree build's results."""
import os
import subprocess
import sys
import textwrap

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "custom_ops_amd", "deploy", "libmi355_beam.so")

CALLS = """
import torch
def results(ops):
    g = torch.Generator(device="cuda").manual_seed(3)
    q = torch.randn(3, 4, 64, generator=g, device="cuda").half()
    kc, vc = torch.randn(2, 9, 1, 16, 64, generator=g, device="cuda").half()
    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")
    t, n = ints([[0, 3, 4], [0, 3, 5], [0, 3, 8]]), ints([40, 41, 47])
    fork = ops.paged_fork(t, n, ints([0, 0, 2]), 16, 9)
    ops.paged_copy(kc, vc, fork[2], fork[3])
    return [ops.mha_shared_decode(q, kc, vc, t, n, ints([0, 3]), ints([32])), *fork, *ops.paged_compact(t, n, 16, 9), kc, vc,
            *ops.beam_select(torch.randn(2, 3, 999, generator=g, device="cuda"), torch.zeros(2, 3, device="cuda"), 5)]
"""


@pytest.mark.gpu
def test_deployment(gpu, tmp_path):
    if not os.path.exists(LIB):
        pytest.skip("no deployment exported (run __graft_entry__.build())")
    code = textwrap.dedent(f"""
        import sys
        sys.path.insert(0, {ROOT!r})
        from custom_ops_amd import ops, beam
        ops.load_precompiled("beam", {LIB!r})
        assert not ops.allow_jit and beam.loaded_path() == {os.path.realpath(LIB)!r}
    """) + CALLS + f"torch.save(results(ops), {str(tmp_path / 'out.pt')!r})\n"
    res = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=110)
    assert res.returncode == 0, res.stderr[-3000:]
    ns = {}
    exec(CALLS, ns)
    from custom_ops_amd import ops
    ops.ensure_loaded("beam")
    for a, b in zip(torch.load(tmp_path / "out.pt", weights_only=True), ns["results"](ops)):
        assert torch.equal(a, b)
