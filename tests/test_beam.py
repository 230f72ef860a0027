"""CPU tests of the host side of the operators for several continuations of a prompt: the
C ABI's refusals, exports and workspace sizes, schemas and fake kernels, derivatives, the
op group in the facade, deployment."""
import ctypes
import json
import math
import os
import re
import shutil

import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch._subclasses.fake_tensor import FakeTensorMode

from custom_ops_amd import beam, build
from tests.test_serve import EINVAL, F, I32, I64, P, _fields, call, make, run_py

WS = ((P, "workspace"), (ctypes.c_size_t, "bytes"))


class Shared(ctypes.Structure):
    _fields_ = _fields((P, "q k v o table lens cu prefix slopes"), (I64, "q_bs q_hs o_bs o_hs kp kh kr vp vh vr ts"),
                       (I32, "b groups h h_k d dtype num_pages page_size cols window"), (F, "scale softcap"), *WS)


class Select(ctypes.Structure):
    _fields_ = _fields((P, "x scores done os ot op"), (I64, "gs bs"), (I32, "groups beams vocab k eos dtype"), *WS)


class Fork(ctypes.Structure):
    _fields_ = _fields((P, "table_in seq parents held table lens src dst free counts"), (I64, "ts"), (I32, "n r cols num_pages page_size n_held"), *WS)


class Compact(ctypes.Structure):
    _fields_ = _fields((P, "table_in seq held table src dst remap free counts"), (I64, "ts"), (I32, "n cols num_pages page_size n_held"), *WS)


class Copy(ctypes.Structure):
    _fields_ = _fields((P, "k v src dst"), (I64, "kp kh kr vp vh vr"), (I32, "n num_pages h_k page_size d"))


SHARED = dict(q=4096, k=4096, v=4096, o=4096, table=4096, lens=4096, cu=4096, prefix=4096, q_bs=256, q_hs=64, o_bs=256, o_hs=64, kp=2048, kh=1024, kr=64,
              vp=2048, vh=1024, vr=64, ts=4, b=2, groups=1, h=4, h_k=2, d=64, dtype=1, num_pages=5, page_size=16, cols=4, window=0, scale=0.125, softcap=0.0)
SELECT = dict(x=4096, scores=4096, os=4096, ot=4096, op=4096, gs=400, bs=100, groups=2, beams=4, vocab=100, k=4, dtype=1)
FORK = dict(table_in=4096, seq=4096, parents=4096, table=4096, lens=4096, src=4096, dst=4096, free=4096, counts=4096, ts=4, n=3, r=3, cols=4, num_pages=9,
            page_size=16)
COMPACT = dict(table_in=4096, seq=4096, table=4096, src=4096, dst=4096, remap=4096, free=4096, counts=4096, ts=4, n=3, cols=4, num_pages=9, page_size=16)
COPY = dict(k=4096, v=8192, src=4096, dst=4096, kp=2048, kh=1024, kr=64, vp=2048, vh=1024, vr=64, n=3, num_pages=5, h_k=2, page_size=16, d=64)
CALLS = [("mi355_shared_decode", Shared, SHARED), ("mi355_beam_select", Select, SELECT), ("mi355_paged_fork", Fork, FORK),
         ("mi355_paged_compact", Compact, COMPACT), ("mi355_paged_copy", Copy, COPY)]


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(build.BEAM_LIB_PATH):
        build.build_beam()
    return ctypes.CDLL(build.BEAM_LIB_PATH)


@pytest.mark.parametrize("name,cls,base,bad,text", [
    *[("mi355_shared_decode", Shared, SHARED, bad, text) for bad, text in [
        (dict(dtype=2), "float16 or bfloat16"), (dict(d=96), "head_dim"), (dict(h=3), "divisible"), (dict(h_k=0), "divisible"), (dict(b=-1), "requests"),
        (dict(b=1025), "1024 requests"), (dict(groups=-1), "groups"), (dict(groups=1025), "groups"), (dict(h=2 ** 17), "heads"), (dict(cols=-1), "negative"),
        (dict(num_pages=-1), "negative"), (dict(page_size=4), "page_size"), (dict(page_size=48), "page_size"), (dict(page_size=2048), "page_size"),
        (dict(cols=2 ** 27), "2\\^30 keys"),
        (dict(cols=2 ** 26, h=64, h_k=64), "too many requests, heads and keys"), (dict(cols=2 ** 26, b=1024), "too many requests, heads and keys"), (dict(window=-1), "window"), (dict(scale=0.0), "scale"), (dict(scale=math.nan), "scale"),
        (dict(softcap=1001.0), "softcap"), (dict(lens=0), "NULL"), (dict(cu=0), "NULL"), (dict(prefix=0), "NULL"), (dict(table=0), "NULL"), (dict(v=0), "NULL"),
        (dict(q=4104), "16-byte"), (dict(kr=68), "multiples of 8"), (dict(kr=2 ** 24), "row strides"), (dict(vr=-64), "row strides"), (dict(o_hs=68), "multiples of 8")]],
    *[("mi355_beam_select", Select, SELECT, bad, text) for bad, text in [
        (dict(dtype=3), "float32"), (dict(groups=-1), "beams"), (dict(beams=0), "beams"), (dict(beams=257), "beams"), (dict(vocab=0), "vocab"),
        (dict(vocab=2 ** 30), "vocab"), (dict(groups=2 ** 30), "vocab"), (dict(k=0), "k must"), (dict(k=65), "k must"), (dict(done=4096, eos=-1), "eos"),
        (dict(done=4096, eos=100), "eos"), (dict(bs=-1), "strides"), (dict(x=0), "NULL"), (dict(scores=0), "NULL"), (dict(op=0), "NULL"), (dict(x=4097), "aligned"),
        (dict(x=4098, dtype=2), "aligned")]],
    *[("mi355_paged_fork", Fork, FORK, bad, text) for bad, text in [
        (dict(n=-1), "rows"), (dict(r=-1), "rows"), (dict(r=4097), "4096 rows"), (dict(cols=-1), "columns"), (dict(cols=2 ** 30 + 1), "2\\^30 columns"),
        (dict(num_pages=-1), "num_pages"), (dict(num_pages=2 ** 19 + 1), "num_pages"), (dict(page_size=0), "page_size"), (dict(n_held=-1), "negative"),
        (dict(n_held=2), "NULL"), (dict(parents=0), "NULL"), (dict(table=0), "NULL"), (dict(free=0), "NULL"), (dict(counts=0), "NULL"), (dict(dst=0), "NULL")]],
    *[("mi355_paged_compact", Compact, COMPACT, bad, text) for bad, text in [
        (dict(n=-1), "rows"), (dict(n=4097), "4096 rows"), (dict(num_pages=2 ** 20), "num_pages"), (dict(page_size=-16), "page_size"), (dict(remap=0), "NULL"),
        (dict(src=0), "NULL"), (dict(seq=0), "NULL"), (dict(counts=0), "NULL")]],
    *[("mi355_paged_copy", Copy, COPY, bad, text) for bad, text in [
        (dict(d=96), "head_dim"), (dict(n=-1), "negative"), (dict(num_pages=-1), "negative"), (dict(h_k=-2), "negative"), (dict(page_size=-1), "negative"),
        (dict(h_k=2 ** 12, page_size=2 ** 12), "2\\^27 elements"), (dict(n=2 ** 31 - 1), "too many"), (dict(src=0), "NULL"), (dict(v=0), "NULL"),
        (dict(k=4104), "16-byte"), (dict(vh=1028), "multiples of 8")]],
])
def test_entry_points_refuse(lib, name, cls, base, bad, text):
    rc, err = call(lib, name, make(cls, base, **bad))
    assert rc == EINVAL and re.search(text, err), (rc, err)


def test_entry_points_refuse_null_and_take_empty_calls(lib):
    for name, _, _ in CALLS:
        assert call(lib, name, None)[0] == EINVAL
    for name, cls, base, empty in (("mi355_shared_decode", Shared, SHARED, dict(b=0)), ("mi355_beam_select", Select, SELECT, dict(groups=0)),
                                   ("mi355_paged_copy", Copy, COPY, dict(n=0))):
        assert call(lib, name, make(cls, base, **empty)) == (0, "")


def test_workspaces(lib):
    """Room for every part and its record; 0 for a call that is refused or does nothing."""
    def size(name, cls, base, **kw):
        f = getattr(lib, name + "_workspace_bytes")
        f.argtypes, f.restype = [P], ctypes.c_size_t
        assert f(None) == 0
        return f(ctypes.addressof(make(cls, base, **kw)))

    for b, g, h, hk, d in ((1, 1, 4, 4, 128), (67, 9, 40, 2, 64), (1024, 1024, 8, 8, 128), (1024, 1, 64, 1, 64), (5, 0, 8, 8, 64)):
        units = b * hk * -(-(h // hk) // 16)   # of own keys, 16 heads each
        assert size(*CALLS[0], b=b, groups=g, h=h, h_k=hk, d=d) >= (units + 1) * 16 * (d + 2) * 4 + (b + g) * 16
    assert size(*CALLS[0], b=0) == 0 and size(*CALLS[0], d=96) == 0
    for g, w, v, k in ((1, 4, 32000, 4), (64, 8, 128000, 16), (3, 1, 5, 64)):
        assert size(*CALLS[1], groups=g, beams=w, vocab=v, k=k) >= g * w * (16 + 8 * k)
    assert size(*CALLS[1], groups=0) == 0 and size(*CALLS[1], k=99) == 0
    for name, cls, base in CALLS[2:4]:
        assert size(name, cls, base, num_pages=2 ** 19) >= 2 * 2 ** 16 and size(name, cls, base, num_pages=-1) == 0


def test_exports_are_the_headers(lib):
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(build.INCLUDE, "mi355_beam.h")).read(), flags=re.S)
    names = set(re.findall(r"\b(mi355_\w+)\s*\(", text))
    assert names == {n for n, _, _ in CALLS} | {n + "_workspace_bytes" for n, _, _ in CALLS[:4]} | {"mi355_beam_abi_version"}
    for n in names:
        assert hasattr(lib, n), n
    assert lib.mi355_beam_abi_version() == beam.ABI_VERSION


def test_group_beside_the_others():
    """Loading or naming the group changes nothing for a program that does not."""
    out = run_py("""
        import torch
        from custom_ops import ops
        ops.ensure_loaded()
        ops.ensure_loaded("serve")
        assert ops.groups == {"fa": "loaded", "serve": "loaded"}
        calls = dict(mha_shared_decode=7, beam_select=2, paged_fork=3, paged_compact=2, paged_copy=4)
        more = dict(beam_select=(3,), paged_fork=(16, 5), paged_compact=(16, 5))
        for name, n in calls.items():
            try:
                getattr(ops, name)(*[torch.zeros(1)] * n, *more.get(name, ()))
                raise SystemExit(name)
            except RuntimeError as e:
                assert "only supported on CUDA" in str(e), (name, e)
            for key in ("CUDA", "CPU", "Meta"):
                assert torch._C._dispatch_has_kernel_for_dispatch_key("recsys_ops::" + name, key), (name, key)
        assert ops.groups == {"fa": "loaded", "serve": "loaded", "beam": "loaded"}
        try:
            ops.beam_select(torch.zeros(1), torch.zeros(1), 1, backend="tilelang")
        except RuntimeError as e:
            assert "tilelang" in str(e)
        print("ok")
    """)
    assert "ok" in out


def test_strict_facade_refuses_the_group():
    out = run_py("""
        import torch
        from custom_ops_amd import ops, CustomOpsError
        ops.disable_jit()
        try:
            ops.beam_select(torch.zeros(1), torch.zeros(1), 1)
        except CustomOpsError as e:
            assert "JIT is disabled" in str(e) and "beam" in str(e)
            print("ok")
    """)
    assert "ok" in out


@pytest.fixture(scope="module")
def o():
    from custom_ops_amd import ops
    ops.ensure_loaded("beam")
    return torch.ops.recsys_ops


def shared(o, dev, **given):
    a = dict(q=torch.ones(9, 4, 64, device=dev), k=torch.ones(5, 2, 16, 64, device=dev), v=torch.ones(5, 2, 16, 64, device=dev),
             slopes=torch.ones(4, device=dev))
    a.update(given)
    n = torch.zeros(9, dtype=torch.int32, device=dev)
    return o.mha_shared_decode(a["q"], a["k"], a["v"], torch.zeros(9, 2, dtype=torch.int32, device=dev), n, n[:3], n[:2], slopes=a["slopes"])


def select(o, dev, **given):
    a = dict(logits=torch.ones(2, 3, 50, device=dev), scores=torch.ones(2, 3, device=dev))
    a.update(given)
    return o.beam_select(a["logits"], a["scores"], 4)[0]


def copy(o, dev, **given):
    a = dict(k=torch.ones(5, 2, 16, 64, device=dev), v=torch.ones(5, 2, 16, 64, device=dev))
    a.update(given)
    n = torch.zeros(3, dtype=torch.int32, device=dev)
    o.paged_copy(a["k"], a["v"], n, n)
    return torch.zeros((), device=dev)


def test_fake_kernels(o):
    with FakeTensorMode():
        def x(*s, dtype=torch.int32):
            return torch.empty(*s, dtype=dtype, device="cuda")
        assert shared(o, "cuda").shape == (9, 4, 64)
        got = o.beam_select(x(2, 3, 50, dtype=torch.bfloat16), x(2, 3, dtype=torch.float32), 7, x(2, 3, dtype=torch.bool), 1)
        assert [(tuple(t.shape), t.dtype) for t in got] == [((2, 7), torch.float32), ((2, 7), torch.int32), ((2, 7), torch.int32)]
        got = o.paged_fork(x(4, 6), x(4), x(9), 16, 31)
        assert [tuple(t.shape) for t in got] == [(9, 6), (9,), (9,), (9,), (31,), (3,)] and all(t.dtype == torch.int32 for t in got)
        got = o.paged_compact(x(4, 6), x(4), 16, 31, x(2))
        assert [tuple(t.shape) for t in got] == [(4, 6), (15,), (15,), (31,), (31,), (2,)]
        copy(o, "cuda")


NEEDS = [(shared, n) for n in ("q", "k", "v", "slopes")] + [(select, n) for n in ("logits", "scores")] + [(copy, n) for n in ("k", "v")]
SHAPES = {(shared, "q"): (9, 4, 64), (shared, "k"): (5, 2, 16, 64), (shared, "v"): (5, 2, 16, 64), (shared, "slopes"): (4,),
          (select, "logits"): (2, 3, 50), (select, "scores"): (2, 3), (copy, "k"): (5, 2, 16, 64), (copy, "v"): (5, 2, 16, 64)}


@pytest.mark.parametrize("call,name", NEEDS)
def test_derivatives_are_refused(o, call, name):
    x = torch.ones(SHAPES[call, name], device="meta", requires_grad=True)
    with pytest.raises(RuntimeError, match="forward only"):
        call(o, "meta", **{name: x})
    with pytest.raises(RuntimeError, match="forward only"):
        call(o, "meta", **{name: x * 2})
    with torch.no_grad():
        assert not call(o, "meta", **{name: x}).requires_grad
    with torch.inference_mode():
        call(o, "meta", **{name: x})
    call(o, "meta", **{name: x.detach()})
    x = x.detach()
    with fwd.dual_level():
        with pytest.raises(RuntimeError, match="forward only"):
            call(o, "meta", **{name: fwd.make_dual(x, torch.ones_like(x))})
    with pytest.raises(RuntimeError, match="forward only"):
        torch.func.grad(lambda t: call(o, "meta", **{name: t}).sum())(x)


@pytest.mark.parametrize("mode", ["grad", "no_grad", "inference"])
def test_cache_versions_move(o, mode):
    k, v = (torch.ones(5, 2, 16, 64, device="meta") for _ in range(2))
    view = k[1:3]
    with {"grad": torch.enable_grad, "no_grad": torch.no_grad, "inference": torch.inference_mode}[mode]():
        for n in (1, 2):
            copy(o, "meta", k=k, v=v)
            assert k._version == n and v._version == n and view._version == n


def test_traced_copies_stay(o):
    """A compiled step that copies pages and returns nothing of them still copies them."""
    from torch._dynamo.testing import CompileCounterWithBackend
    seen = CompileCounterWithBackend("aot_eager")
    k, v = (torch.ones(5, 2, 16, 64, device="meta") for _ in range(2))
    f = torch.compile(lambda a, b: copy(o, "meta", k=a, v=b) * 2, backend=seen, fullgraph=True)
    with torch.no_grad():
        f(k, v)
    assert k._version > 0 and v._version > 0
    assert any("paged_copy" in str(n.target) for g in seen.graphs for n in g.graph.nodes)


# ── deployment ────────────────────────────────────────────────────────────────

def test_sealed_deployment(lib, tmp_path, monkeypatch):
    from custom_ops_amd.loader import BeamOps
    monkeypatch.setattr(build, "compile_checked", lambda out, flags, verbose=False, src=None: shutil.copy2(build.BEAM_LIB_PATH, out))
    path = BeamOps().build(tmp_path)
    md = json.loads(open(str(path) + ".json").read())
    assert set(md["contract"]["schemas"]) == {f"recsys_ops::{n}" for n in beam.SCHEMAS}
    assert md["companion"]["file"] == "libmi355_beam_ops.so" and md["targets"] == ["gfx950"]
    out = run_py(f"""
        import torch
        from custom_ops_amd import ops, beam
        ops.load_precompiled("beam", {str(path)!r})
        assert ops.groups == {{"fa": "not_loaded", "beam": "loaded"}} and not ops.allow_jit
        assert torch._C._dispatch_has_kernel_for_dispatch_key("recsys_ops::beam_select", "CUDA")
        print("loaded", beam.loaded_path())
    """)
    assert f"loaded {path}" in out
    (path.parent / "libmi355_beam_ops.so").unlink()
    out = run_py(f"""
        from custom_ops_amd import ops, beam, CustomOpsError
        try:
            ops.load_precompiled("beam", {str(path)!r})
        except CustomOpsError as e:
            print("ERR", e, beam.loaded_path())
    """)
    assert "was not deployed" in out and out.rstrip().endswith("None"), out
