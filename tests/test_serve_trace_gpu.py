"""The serving operators in a compiled program on the GPU: the eager calls' results, and the
caches written."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_compiled_step(gpu):
    from custom_ops_amd import ops
    ops.ensure_loaded("serve")
    o = torch.ops.recsys_ops
    g = torch.Generator(device="cuda").manual_seed(1)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda").bfloat16()

    freq = ops.rotary_frequencies(64, device="cuda")[0]
    table = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    free = torch.zeros(0, dtype=torch.int32, device="cuda")

    def step(x, w, lens, new, kc, vc):
        qkv = (x @ w).view(-1, 8, 64)
        lens, cu, pos, slots, t, _ = o.paged_layout(lens, new, table, free, 16, x.shape[0])
        q, k = o.rope_paged_store(qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], pos, freq, slots, kc, vc)
        return o.mha_packed_fwd(q, k, qkv[:, 6:], cu, cu), o.mha_paged_decode(q[:2], kc, vc, t, lens)

    x, w = randn(9, 32), randn(32, 512)
    lens, new = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([3, 30], [4, 5]))
    kc, vc = randn(2, 8, 2, 16, 64)
    compiled = torch.compile(step, backend="aot_eager", fullgraph=True)
    with torch.no_grad():
        for _ in range(2):
            a, b = (kc.clone(), vc.clone()), (kc.clone(), vc.clone())
            before = b[0]._version
            want, got = step(x, w, lens, new, *a), compiled(x, w, lens, new, *b)
            for p, q in zip((*want, *a), (*got, *b)):
                assert torch.equal(p, q)
            assert not torch.equal(b[0], kc) and b[0]._version > before
    w.requires_grad_()
    with pytest.raises(RuntimeError, match="forward only"):
        torch.compile(step, backend="aot_eager", fullgraph=True)(x, w, lens, new, kc, vc)
