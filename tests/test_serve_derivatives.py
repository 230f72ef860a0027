"""CPU tests that no derivative is lost: the serving operators have none, so a call that needs
one is refused in eager mode, while tracing (fake and meta tensors) and under torch.func."""
import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch._subclasses.fake_tensor import FakeTensorMode


@pytest.fixture(scope="module")
def o():
    from custom_ops_amd import ops
    ops.ensure_loaded("serve")
    return torch.ops.recsys_ops


def packed(o, dev, **given):
    a = dict(q=torch.ones(9, 4, 64, device=dev), k=torch.ones(9, 2, 64, device=dev), v=torch.ones(9, 2, 64, device=dev),
             slopes=torch.ones(4, device=dev))
    a.update(given)
    cu = torch.zeros(3, dtype=torch.int32, device=dev)
    return o.mha_packed_fwd(a["q"], a["k"], a["v"], cu, cu, slopes=a["slopes"])


def decode(o, dev, **given):
    a = dict(q=torch.ones(9, 4, 64, device=dev), k=torch.ones(5, 2, 16, 64, device=dev), v=torch.ones(5, 2, 16, 64, device=dev),
             slopes=torch.ones(4, device=dev))
    a.update(given)
    return o.mha_paged_decode(a["q"], a["k"], a["v"], torch.zeros(9, 2, dtype=torch.int32, device=dev),
                              torch.zeros(9, dtype=torch.int32, device=dev), slopes=a["slopes"])


def rope(o, dev, **given):
    a = dict(q=torch.ones(9, 4, 64, device=dev), k=torch.ones(9, 2, 64, device=dev), v=torch.ones(9, 2, 64, device=dev),
             freq=torch.ones(32, dtype=torch.float64, device=dev), kc=torch.ones(5, 2, 16, 64, device=dev), vc=torch.ones(5, 2, 16, 64, device=dev))
    a.update(given)
    return o.rope_paged_store(a["q"], a["k"], a["v"], torch.zeros(9, dtype=torch.int32, device=dev), a["freq"],
                              torch.zeros(9, dtype=torch.int64, device=dev), a["kc"], a["vc"])[0]


CALLS = [(packed, n) for n in ("q", "k", "v", "slopes")] + [(decode, n) for n in ("q", "k", "v", "slopes")] + \
        [(rope, n) for n in ("q", "k", "v", "freq", "kc", "vc")]
SHAPES = {(packed, "q"): (9, 4, 64), (packed, "k"): (9, 2, 64), (packed, "v"): (9, 2, 64), (packed, "slopes"): (4,),
          (decode, "q"): (9, 4, 64), (decode, "k"): (5, 2, 16, 64), (decode, "v"): (5, 2, 16, 64), (decode, "slopes"): (4,),
          (rope, "q"): (9, 4, 64), (rope, "k"): (9, 2, 64), (rope, "v"): (9, 2, 64), (rope, "freq"): (32,),
          (rope, "kc"): (5, 2, 16, 64), (rope, "vc"): (5, 2, 16, 64)}


def leaf(call, name, dev, **kw):
    return torch.ones(SHAPES[call, name], dtype=torch.float64 if name == "freq" else torch.float32, device=dev, **kw)


@pytest.mark.parametrize("kind", ["fake", "meta", "cpu"])
@pytest.mark.parametrize("call,name", CALLS)
def test_gradients_are_refused(o, call, name, kind):
    dev = {"fake": "cuda", "meta": "meta", "cpu": "cpu"}[kind]
    import contextlib
    with FakeTensorMode() if kind == "fake" else contextlib.nullcontext():
        x = leaf(call, name, dev, requires_grad=True)
        with pytest.raises(RuntimeError, match="forward only"):
            call(o, dev, **{name: x})
        with pytest.raises(RuntimeError, match="forward only"):
            call(o, dev, **{name: x * 2})
        if kind == "cpu":   # no kernel there, for a call that is let through either
            with torch.no_grad(), pytest.raises(RuntimeError, match="only supported on CUDA"):
                call(o, dev, **{name: x})
            return
        with torch.no_grad():
            assert not call(o, dev, **{name: x}).requires_grad
        with torch.inference_mode():
            call(o, dev, **{name: x})
        assert not call(o, dev, **{name: x.detach()}).requires_grad
        assert not call(o, dev).requires_grad


@pytest.mark.parametrize("call,name", CALLS)
def test_tangents_are_refused(o, call, name):
    x = leaf(call, name, "meta")
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward only"):
                call(o, "meta", **{name: dual})
        call(o, "meta", **{name: x})
    with pytest.raises(RuntimeError, match="forward only"):
        torch.func.jvp(lambda t: call(o, "meta", **{name: t}), (x,), (torch.ones_like(x),))
    with pytest.raises(RuntimeError, match="forward only"):
        torch.func.grad(lambda t: call(o, "meta", **{name: t}).sum())(x)


def test_compiled_calls_keep_no_secret(o):
    """A traced call with a weight that requires a gradient raises instead of leaving it out."""
    w = torch.ones(64, 64, device="meta", requires_grad=True)
    x = torch.ones(9, 4, 64, device="meta")
    f = torch.compile(lambda t: packed(o, "meta", q=t @ w).sum(), backend="aot_eager", fullgraph=True)
    with pytest.raises(RuntimeError, match="forward only"):
        f(x)
    torch._dynamo.reset()
    with torch.no_grad():
        assert f(x).shape == ()


def test_layout_takes_no_gradients(o):
    n = torch.zeros(4, dtype=torch.int32, device="meta")
    t = torch.zeros(4, 6, dtype=torch.int32, device="meta")
    assert o.paged_layout(n, n, t, n, 16, 11)[0].shape == (4,)


# ── caches written in place ───────────────────────────────────────────────────

@pytest.mark.parametrize("mode", ["grad", "no_grad", "inference"])
def test_cache_versions_move(o, mode):
    kc, vc = (torch.ones(5, 2, 16, 64, device="meta") for _ in range(2))
    view = kc[1:3]
    with {"grad": torch.enable_grad, "no_grad": torch.no_grad, "inference": torch.inference_mode}[mode]():
        for n in (1, 2):
            rope(o, "meta", kc=kc, vc=vc)
            assert kc._version == n and vc._version == n and view._version == n


def test_a_saved_cache_is_noticed(o):
    w = torch.ones(64, device="meta", requires_grad=True)
    for which in ("kc", "vc"):
        cache = torch.ones(5, 2, 16, 64, device="meta")
        y = (w * cache).sum()
        rope(o, "meta", **{which: cache})
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()


def test_inference_caches(o):
    """Made in inference mode, they are written there and outside."""
    with torch.inference_mode():
        kc, vc = (torch.ones(5, 2, 16, 64, device="meta") for _ in range(2))
        rope(o, "meta", kc=kc, vc=vc)
    with torch.no_grad():
        rope(o, "meta", kc=kc, vc=vc)


def test_traced_writes_stay(o):
    """A compiled step that writes the caches and returns nothing of them still writes them."""
    from torch._dynamo.testing import CompileCounterWithBackend
    seen = CompileCounterWithBackend("aot_eager")
    kc, vc = (torch.ones(5, 2, 16, 64, device="meta") for _ in range(2))
    f = torch.compile(lambda q, a, b: rope(o, "meta", q=q, kc=a, vc=b) * 2, backend=seen, fullgraph=True)
    with torch.no_grad():
        f(torch.ones(9, 4, 64, device="meta"), kc, vc)
    assert kc._version > 0 and vc._version > 0
    assert any("rope_paged_store" in str(n.target) for g in seen.graphs for n in g.graph.nodes)
