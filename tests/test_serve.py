"""CPU tests of the serving operators' host side: the C ABI's refusals, exports and
workspace sizes, schemas and fake kernels, the op group in the facade, deployment, and
the rotary frequencies."""
import ctypes
import json
import math
import os
import re
import shutil
import subprocess
import sys
import textwrap

import pytest
import torch

from custom_ops_amd import build, serve

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P, I32, I64, F = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float
EINVAL, EWORKSPACE = 1, 2


def _fields(*groups):
    return [(name, t) for t, names in groups for name in names.split()]


class Packed(ctypes.Structure):
    _fields_ = _fields((P, "q k v o cu_q cu_k prefix_lens slopes"), (I64, "q_ts q_hs k_ts k_hs v_ts v_hs o_ts o_hs"),
                       (I32, "total_q total_k n_seqs h h_k d dtype causal window"), (F, "scale softcap"))


class Decode(ctypes.Structure):
    _fields_ = _fields((P, "q k v o table lens slopes"), (I64, "q_bs q_hs o_bs o_hs kp kh kr vp vh vr ts"),
                       (I32, "b h h_k d dtype num_pages page_size cols window"), (F, "scale softcap"), (P, "workspace"), (ctypes.c_size_t, "bytes"))


class Rope(ctypes.Structure):
    _fields_ = _fields((P, "q k v qo ko kc vc positions inv_freq slots"),
                       (I64, "q_ts q_hs k_ts k_hs v_ts v_hs qo_ts qo_hs ko_ts ko_hs kcp kch kcr vcp vch vcr"),
                       (I32, "t h h_k d dtype rot interleaved num_pages page_size"), (F, "amplitude"))


class Layout(ctypes.Structure):
    _fields_ = _fields((P, "seq new table_in free kv_lens cu positions slots table counts"), (I64, "ts"), (I32, "n cols n_free page_size max_tokens"))


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(build.SERVE_LIB_PATH):
        build.build_serve()
    return ctypes.CDLL(build.SERVE_LIB_PATH)


def call(lib, name, params):
    f = getattr(lib, name)
    f.argtypes = [P, P, ctypes.c_char_p, ctypes.c_size_t]
    err = ctypes.create_string_buffer(256)
    return f(None if params is None else ctypes.addressof(params), None, err, 256), err.value.decode()


def make(cls, base, **kw):
    p = cls()
    for k, v in {**base, **kw}.items():
        setattr(p, k, v)
    return p


PACKED = dict(q=4096, k=4096, v=4096, o=4096, cu_q=4096, cu_k=4096, q_ts=256, q_hs=64, k_ts=128, k_hs=64, v_ts=128, v_hs=64, o_ts=256, o_hs=64,
              total_q=8, total_k=8, n_seqs=1, h=4, h_k=2, d=64, dtype=1, causal=1, window=0, scale=0.125, softcap=0.0)
DECODE = dict(q=4096, k=4096, v=4096, o=4096, table=4096, lens=4096, q_bs=256, q_hs=64, o_bs=256, o_hs=64, kp=2048, kh=1024, kr=64, vp=2048, vh=1024, vr=64,
              ts=4, b=2, h=4, h_k=2, d=64, dtype=1, num_pages=5, page_size=16, cols=4, window=0, scale=0.125, softcap=0.0)
ROPE = dict(q=4096, k=4096, v=4096, qo=4096, ko=4096, kc=4096, vc=4096, positions=4096, inv_freq=4096, slots=4096, q_ts=256, q_hs=64, k_ts=128, k_hs=64,
            v_ts=128, v_hs=64, qo_ts=256, qo_hs=64, ko_ts=128, ko_hs=64, kcp=2048, kch=1024, kcr=64, vcp=2048, vch=1024, vcr=64, t=8, h=4, h_k=2, d=64,
            dtype=1, rot=64, interleaved=0, num_pages=5, page_size=16, amplitude=1.0)
LAYOUT = dict(seq=4096, new=4096, table_in=4096, free=4096, kv_lens=4096, cu=4096, positions=4096, slots=4096, table=4096, counts=4096, ts=4, n=3, cols=4,
              n_free=5, page_size=16, max_tokens=9)


@pytest.mark.parametrize("name,cls,base,bad,text", [
    *[("mi355_packed_fwd", Packed, PACKED, bad, text) for bad, text in [
        (dict(dtype=2), "float16 or bfloat16"), (dict(d=96), "head_dim"), (dict(h=3), "divisible"), (dict(h_k=0), "divisible"),
        (dict(total_q=-1), "total_q"), (dict(total_k=2 ** 30 + 1), "total_q"), (dict(n_seqs=-1), "n_seqs"), (dict(window=-1), "window"),
        (dict(scale=0.0), "scale"), (dict(scale=math.inf), "scale"), (dict(scale=math.nan), "scale"), (dict(softcap=-1.0), "softcap"),
        (dict(softcap=1001.0), "softcap"), (dict(softcap=math.nan), "softcap"), (dict(scale=1e-38), "scale"), (dict(softcap=1e-39), "softcap"),
        (dict(q=0), "NULL"), (dict(k=0), "NULL"), (dict(cu_k=0), "NULL"), (dict(q=4098), "16-byte"), (dict(k_ts=130), "multiples of 8"),
        (dict(v_ts=2 ** 24), "token strides"), (dict(o_ts=-256), "token strides")]],
    *[("mi355_paged_decode", Decode, DECODE, bad, text) for bad, text in [
        (dict(dtype=-1), "float16 or bfloat16"), (dict(d=32), "head_dim"), (dict(h=5), "divisible"), (dict(b=-1), "negative"), (dict(cols=-1), "negative"),
        (dict(page_size=4), "page_size"), (dict(page_size=48), "page_size"), (dict(page_size=2048), "page_size"), (dict(window=-2), "window"),
        (dict(cols=2 ** 27), "2\\^30 keys"), (dict(scale=-1.0), "scale"), (dict(softcap=math.inf), "softcap"), (dict(lens=0), "NULL"), (dict(table=0), "NULL"), (dict(k=0), "NULL"),
        (dict(k=4104), "16-byte"), (dict(vr=68), "multiples of 8")]],
    *[("mi355_rope_paged_store", Rope, ROPE, bad, text) for bad, text in [
        (dict(dtype=7), "float16 or bfloat16"), (dict(d=256), "head_dim"), (dict(h=3), "divisible"), (dict(rot=8), "rot"), (dict(rot=80), "rot"),
        (dict(rot=-16), "rot"), (dict(page_size=0), "page_size"), (dict(amplitude=math.nan), "amplitude"), (dict(t=-1), "t and num_pages"),
        (dict(inv_freq=0), "NULL"), (dict(kc=0), "NULL"), (dict(qo=4100), "16-byte"), (dict(vcr=60), "multiples of 8")]],
    *[("mi355_paged_layout", Layout, LAYOUT, bad, text) for bad, text in [
        (dict(n=-1), "requests"), (dict(n=8193), "requests"), (dict(cols=-1), "negative"), (dict(n_free=-1), "negative"), (dict(max_tokens=-1), "negative"),
        (dict(page_size=0), "page_size"), (dict(cu=0), "NULL"), (dict(table=0), "NULL"), (dict(free=0), "NULL"), (dict(slots=0), "NULL")]],
])
def test_entry_points_refuse(lib, name, cls, base, bad, text):
    rc, err = call(lib, name, make(cls, base, **bad))
    assert rc == EINVAL and re.search(text, err), (rc, err)


def test_entry_points_refuse_null_and_take_empty_calls(lib):
    for name in ("mi355_packed_fwd", "mi355_paged_decode", "mi355_rope_paged_store", "mi355_paged_layout"):
        assert call(lib, name, None)[0] == EINVAL
    for name, cls, base, empty in (("mi355_packed_fwd", Packed, PACKED, dict(total_q=0)), ("mi355_paged_decode", Decode, DECODE, dict(b=0)),
                                   ("mi355_rope_paged_store", Rope, ROPE, dict(t=0))):
        assert call(lib, name, make(cls, base, **empty)) == (0, "")


def test_workspace_covers_every_part(lib):
    """Slots for every part and every request's record; none where no request can be split."""
    f = lib.mi355_paged_decode_workspace_bytes
    f.argtypes, f.restype = [P], ctypes.c_size_t

    def size(**kw):
        return f(ctypes.addressof(make(Decode, DECODE, **kw)))

    assert size(cols=4) == 0                                    # 64 keys
    assert size(page_size=3) == 0 and size(b=0) == 0 and f(None) == 0
    for b, h, hk, d in ((1, 4, 1, 128), (3, 40, 2, 64), (1000, 8, 8, 128)):
        groups = hk * -(-(h // hk) // 16)
        got = size(b=b, h=h, h_k=hk, d=d, cols=4096)
        assert got >= (b * groups + 240) * 16 * (d + 2) * 4 + b * groups * 8
    assert size(b=1025, cols=4096) == 0                          # lengths too many to scan


def test_exports_are_the_headers(lib):
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(build.INCLUDE, "mi355_serve.h")).read(), flags=re.S)
    names = set(re.findall(r"\b(mi355_\w+)\s*\(", text))
    assert names == {"mi355_packed_fwd", "mi355_paged_decode", "mi355_paged_decode_workspace_bytes", "mi355_rope_paged_store", "mi355_paged_layout",
                     "mi355_serve_abi_version"}
    for n in names:
        assert hasattr(lib, n), n
    assert lib.mi355_serve_abi_version() == serve.ABI_VERSION


def run_py(code):
    env = dict(os.environ, PYTHONPATH=ROOT)
    env.pop("CUSTOM_OPS_BACKEND", None)
    res = subprocess.run([sys.executable, "-c", textwrap.dedent(code)], cwd=ROOT, env=env, capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, (res.stdout[-2000:], res.stderr[-3000:])
    return res.stdout


def test_group_beside_the_references():
    """Loading or naming the serving group changes nothing for a program that does not."""
    out = run_py("""
        import torch
        from custom_ops import ops
        assert ops.groups == {"fa": "not_loaded"}
        ops.ensure_loaded()
        assert ops.groups == {"fa": "loaded"}
        try:
            ops.mha_paged_decode(*[torch.zeros(1)] * 5)
        except RuntimeError as e:
            assert "only supported on CUDA" in str(e), e
        assert ops.groups == {"fa": "loaded", "serve": "loaded"}
        for name in ("mha_packed_fwd", "mha_paged_decode", "rope_paged_store", "paged_layout"):
            for key in ("CUDA", "CPU", "Meta"):
                assert torch._C._dispatch_has_kernel_for_dispatch_key("recsys_ops::" + name, key), (name, key)
        try:
            ops.paged_layout(*[torch.zeros(1)] * 4, 16, 1, backend="tilelang")
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
            ops.mha_packed_fwd(*[torch.zeros(1)] * 5)
        except CustomOpsError as e:
            assert "JIT is disabled" in str(e) and "serve" in str(e)
            print("ok")
    """)
    assert "ok" in out


def test_fake_kernels():
    from torch._subclasses.fake_tensor import FakeTensorMode

    from custom_ops_amd import ops
    ops.ensure_loaded("serve")
    o = torch.ops.recsys_ops
    with FakeTensorMode():
        def x(*s, dtype=torch.bfloat16):
            return torch.empty(*s, dtype=dtype, device="cuda")
        qkv, n = x(9, 12, 64), x(4, dtype=torch.int32)
        q, k = qkv[:, :8], qkv[:, 8:10]
        out = o.mha_packed_fwd(q, k, k, n, n)
        assert out.shape == q.shape and out.is_contiguous() and out.dtype == q.dtype
        assert o.mha_paged_decode(q, x(5, 2, 16, 64), x(5, 2, 16, 64), x(9, 7, dtype=torch.int32), x(9, dtype=torch.int32)).shape == q.shape
        a, b = o.rope_paged_store(q, k, k, x(9, dtype=torch.int32), x(32, dtype=torch.float64), x(9, dtype=torch.int64), x(5, 2, 16, 64), x(5, 2, 16, 64))
        assert a.shape == q.shape and b.shape == k.shape and a.is_contiguous() and b.is_contiguous()
        got = o.paged_layout(n, n, x(4, 6, dtype=torch.int32), x(3, dtype=torch.int32), 16, 11)
        assert [tuple(t.shape) for t in got] == [(4,), (5,), (11,), (11,), (4, 6), (3,)] and got[3].dtype == torch.int64


# ── deployment ────────────────────────────────────────────────────────────────

@pytest.fixture(scope="module")
def exported(tmp_path_factory, lib):
    """ServeOps.build with the in-tree library in place of a new compilation."""
    from custom_ops_amd.loader import ServeOps
    mp = pytest.MonkeyPatch()
    mp.setattr(build, "compile_checked", lambda out, flags, verbose=False, src=None: shutil.copy2(build.SERVE_LIB_PATH, out))
    try:
        return ServeOps().build(tmp_path_factory.mktemp("sealed"))
    finally:
        mp.undo()


def load(path):
    return run_py(f"""
        import torch
        from custom_ops_amd import ops, serve, CustomOpsError
        try:
            ops.load_precompiled("serve", {str(path)!r})
            assert ops.groups == {{"fa": "not_loaded", "serve": "loaded"}} and not ops.allow_jit
            assert torch._C._dispatch_has_kernel_for_dispatch_key("recsys_ops::mha_packed_fwd", "CUDA")
            print("loaded", serve.loaded_path())
        except CustomOpsError as e:
            print("ERR", e, serve.loaded_path())
    """)


def test_sealed_deployment(exported):
    md = json.loads(open(str(exported) + ".json").read())
    assert set(md["contract"]["schemas"]) == {f"recsys_ops::{n}" for n in serve.SCHEMAS}
    assert md["companion"]["file"] == "libmi355_serve_ops.so" and md["targets"] == ["gfx950"]
    assert f"loaded {exported}" in load(exported)


def test_deployment_without_its_implementation_is_refused(exported, tmp_path):
    for name in (exported.name, exported.name + ".json"):
        shutil.copy2(exported.parent / name, tmp_path / name)
    out = load(tmp_path / exported.name)
    assert "was not deployed" in out and out.rstrip().endswith("None"), out
    data = bytearray((exported.parent / "libmi355_serve_ops.so").read_bytes())
    data[4096] ^= 0xFF
    (tmp_path / "libmi355_serve_ops.so").write_bytes(bytes(data))
    out = load(tmp_path / exported.name)
    assert "companion digest mismatch" in out and out.rstrip().endswith("None"), out


# ── rotary frequencies ────────────────────────────────────────────────────────

def test_rotary_frequencies():
    f, amp = serve.rotary_frequencies(64, 10000.0)
    assert f.dtype == torch.float64 and amp == 1.0
    want = [10000.0 ** (-2 * i / 64) for i in range(32)]
    assert torch.allclose(f, torch.tensor(want, dtype=torch.float64), rtol=1e-14, atol=0)
    lin, _ = serve.rotary_frequencies(64, scaling="linear", factor=4.0)
    assert torch.allclose(lin, f / 4, rtol=1e-14, atol=0)
    ntk, _ = serve.rotary_frequencies(64, scaling="ntk", factor=4.0)
    assert ntk[0] == 1.0 and abs(float(ntk[-1] * 4 / f[-1]) - 1) < 1e-12   # the slowest pair exactly divided
    y, amp = serve.rotary_frequencies(64, scaling="yarn", factor=8.0, original_len=4096)
    assert abs(amp - (0.1 * math.log(8) + 1)) < 1e-15
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(y[turns >= 32], f[turns >= 32]) and torch.allclose(y[turns <= 1], f[turns <= 1] / 8, rtol=1e-14, atol=0)
    assert (y[1:] < y[:-1]).all()
    assert serve.rotary_frequencies(0)[0].numel() == 0


@pytest.mark.parametrize("args,kw", [((24,), {}), ((-16,), {}), ((64, 1.0), {}), ((64, math.inf), {}), ((64,), dict(factor=0.5)),
                                     ((64,), dict(scaling="cubic")), ((64,), dict(scaling="yarn", factor=2.0)),
                                     ((64,), dict(scaling="yarn", factor=2.0, original_len=100, beta_slow=40.0))])
def test_rotary_frequencies_refuse(args, kw):
    with pytest.raises(RuntimeError):
        serve.rotary_frequencies(*args, **kw)
