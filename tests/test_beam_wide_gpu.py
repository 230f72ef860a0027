"""GPU tests of selections whose parts take several wide steps, as those of real vocabularies do:
ties across steps, lists that overflow, references that move, values that the count of bf16 logits
leaves out, and what is not finite in the first, a middle and the last step."""
import ctypes
import math

import pytest
import torch

from custom_ops_amd import beam
from tests.test_beam import SELECT, Select
from tests.test_serve import make

pytestmark = pytest.mark.gpu
INF = math.inf
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
STEP = {"fp32": 4096, "bf16": 8192, "fp16": 8192}   # tokens of a wide step


@pytest.fixture(scope="module")
def ops(gpu):
    from custom_ops_amd import ops
    ops.ensure_loaded("beam")
    return ops


def best_of(x, scores, k, done=None, eos=-1):
    """The k best of one search, (-score, row, -logit, token), by the definition in 64 bits."""
    W, V = x.shape
    x = x.double()
    every = []
    for w in range(W):
        run, r = float(scores[w]), x[w]
        if not math.isfinite(run):
            continue
        if done is not None and bool(done[w]):
            every.append((-run, w, 0.0, eos))
            continue
        top = r.max()
        if bool(torch.isnan(r).any()) or float(top) in (INF, -INF):
            continue
        s = run + (r - (top + torch.log(torch.exp(r - top).sum())))
        first = r.sort(descending=True, stable=True).indices[:k]
        every += [(-a, w, -b, v) for a, b, v in zip(s[first].tolist(), r[first].tolist(), first.tolist()) if b > -INF]
    every.sort()
    return every[:k]


def parts(G, W, V, k, dtype):
    """Of a row, from the workspace: 16 bytes a part, in whole 256, then 8 for each of its k."""
    lib = beam._lib
    lib.mi355_beam_select_workspace_bytes.argtypes, lib.mi355_beam_select_workspace_bytes.restype = [ctypes.c_void_p], ctypes.c_size_t
    kind = {"fp16": 0, "bf16": 1, "fp32": 2}[dtype]
    have = lib.mi355_beam_select_workspace_bytes(ctypes.addressof(make(Select, SELECT, groups=G, beams=W, vocab=V, k=k, dtype=kind)))
    return next(n for n in range(1, 1100) if have == (G * W * n * 16 + 255) // 256 * 256 + G * W * n * k * 8)


def look(ops, x, dtype, k, scores=None, done=None, eos=-1, rows=600):
    W, V = x.shape
    x = x.to(TYPES[dtype])
    if scores is None:
        scores = torch.tensor([-0.37 * w for w in range(W)], device="cuda")
    G = -(-rows // W)
    n = parts(G, W, V, k, dtype)
    assert V > 3 * n * STEP[dtype]   # four steps a part and more
    s, t, p = ops.beam_select(x.expand(G, W, V), scores.expand(G, W).contiguous(), k,
                              finished=None if done is None else done.expand(G, W).contiguous(), eos=eos)
    want = best_of(x, scores, k, done, eos)
    pad = [-1] * (k - len(want))
    assert t[0].tolist() == [v for *_, v in want] + pad
    assert p[0].tolist() == [w for _, w, _, _ in want] + pad
    for got, (w, *_) in zip(s[0].tolist(), want):   # one rounding of a value that 64 bits give to 10^-12 of the sum's logarithm
        assert abs(got + w) <= 2.0 ** -24 * abs(w) + 1e-10
    assert (s[0, len(want):] == -INF).all()
    assert torch.equal(s, s[:1].expand(G, k)) and torch.equal(t, t[:1].expand(G, k))
    first = W * torch.arange(G, device="cuda", dtype=torch.int32)[:, None]
    assert torch.equal(torch.where(p >= 0, p - first, -1), p[:1].expand(G, k))


def normal(V, seed, spread=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(3, V, generator=g, device="cuda") * spread


def values(kind, V, step):
    """Three rows of logits; the second is always the common kind."""
    x, i = normal(V, V % 1000), torch.arange(V, device="cuda")
    if kind == "ascending":
        x[0], x[2] = i / 1000.0, i / 700.0 - 50
    elif kind == "descending":
        x[0], x[2] = -i / 1000.0, 30 - i / 700.0
    elif kind == "equal":
        x[0], x[2] = 1.5, -0.25
    elif kind == "zeros":
        x[0], x[2] = 0.0, -0.0
        x[0, ::3] = -0.0
    elif kind == "ties at the steps' ends":
        for s in range(step, V, step):
            x[0, s - 2:s + 2] = 40.0
            x[2, s - 1] = x[2, s] = 41.0 + s // step % 2
    elif kind == "beyond the count":   # at and outside the values that are counted: 2^-10 .. 64 and their negatives
        x[0] = torch.tensor([64.0, 63.75, -64.0, -63.75, 2.0 ** -10, 2.0 ** -11, -2.0 ** -10, -2.0 ** -12, 0.0, 70.0, -500.0], device="cuda")[i % 11]
        x[2] = x[2] * 30
    elif kind == "far beyond":
        x[0], x[2] = x[0] * 4000, x[2] * 1e5
    elif kind == "past 10^6":
        x[0, step:] = x[0, step:] * 1e5 + 3e6
        x[2] = x[2] * 1e5 - 5e6
    elif kind == "past 10^6 first":
        x[0, :step // 2] += 2e6
        x[2, V - 5:] = 4e7
    elif kind == "from below":   # -5·10^6, then the common kind
        x[0, :2 * step] -= 5e6
        x[2, : V - step] -= 5e6
    elif kind == "rising reference":   # by 150 a step, and by 30
        x[0] += 150.0 * (i // step)
        x[2] += 30.0 * (i // step)
    elif kind == "falling reference":
        x[0] -= 150.0 * (i // step)
        x[2] -= 500.0 * (i // step)
    elif kind == "largest in the last step":
        x[0, V - 3] = x[0, V - 1] = 63.0
        x[2, V - 1] = 900.0
    elif kind == "banned":   # a tenth, and nine tenths
        x[0, i % 10 == 3] = -INF
        x[2, i % 10 != 3] = -INF
    elif kind == "few left":
        x[0, :V - 7] = -INF
        x[2, 3:] = -INF
    elif kind == "none left":
        x[0] = -INF
        x[2, step:] = -INF
    else:
        assert kind == "normal"
    return x


KINDS = ["normal", "ascending", "descending", "equal", "zeros", "ties at the steps' ends", "beyond the count", "far beyond", "past 10^6", "past 10^6 first",
         "from below", "rising reference", "falling reference", "largest in the last step", "banned", "few left", "none left"]


def fits(kind, dtype):
    return dtype != "fp16" or not any(x in kind for x in ("10^6", "below", "far"))   # (65504 at most)


@pytest.mark.parametrize("k", [1, 16, 64])
@pytest.mark.parametrize("V", [40960, 40001, 70003])
@pytest.mark.parametrize("dtype,kind", [(t, kind) for t in TYPES for kind in KINDS if fits(kind, t)])
def test_values(ops, dtype, kind, V, k):
    look(ops, values(kind, V, STEP[dtype]), dtype, k)


@pytest.mark.parametrize("dtype,kind", [(t, kind) for t in TYPES for kind in KINDS if fits(kind, t)])
def test_values_of_two_parts(ops, dtype, kind):
    """Rows of two parts, whose references and lists are joined."""
    look(ops, values(kind, 100003, STEP[dtype]), dtype, 8, rows=400)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("bad", [math.nan, INF])
@pytest.mark.parametrize("where", ["first", "middle", "last", "end"])
def test_rows_that_hold_no_number(ops, dtype, bad, where):
    V, step = 40001, STEP[dtype]
    at = {"first": 77, "middle": 2 * step + 4321 % step, "last": V // step * step + 1, "end": V - 1}[where]
    x = normal(V, 4)
    x[0, at] = bad
    look(ops, x, dtype, 9)
    x[2, at] = -bad
    look(ops, x, dtype, 9)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_finished_rows(ops, dtype):
    x = normal(50003, 5)
    x[1, 40000] = math.nan   # of a finished beam: not read
    for done in ([False, True, False], [True, True, False], [True, True, True]):
        look(ops, x, dtype, 7, done=torch.tensor(done, device="cuda"), eos=33333)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_rows_at_odd_places(ops, dtype):
    wide = normal(50021, 6)
    look(ops, wide[:, 5:50008], dtype, 16)
    x = wide.to(TYPES[dtype])[:, 7:50010]   # rows 50021 elements apart, from the 7th on
    one = ops.beam_select(x.expand(200, 3, 50003), torch.zeros(200, 3, device="cuda"), 16)
    two = ops.beam_select(x.contiguous().expand(200, 3, 50003), torch.zeros(200, 3, device="cuda"), 16)
    for a, b in zip(one, two):
        assert torch.equal(a, b)
