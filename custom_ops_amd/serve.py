"""The serving operators on MI355X, around ``recsys_ops::mha_fwd_with_mask``: what a
program that generates token by token needs next to it.

  * ``paged_layout``      page tables, slots and positions of a step, on the device
  * ``rope_paged_store``  rotary positions of q and k; k and v into a paged cache
  * ``mha_packed_fwd``    attention over packed sequences: prompts, documents
  * ``mha_paged_decode``  attention of one new token per request over the cache

A step: ``paged_layout`` gives slots and positions, ``rope_paged_store`` fills the
cache, then prompts with nothing cached attend with ``mha_packed_fwd`` (q and k as
``rope_paged_store`` returns them, ``cu_new`` as offsets: the step's own tokens alone)
and single tokens with ``mha_paged_decode`` (``kv_lens`` and the table of
``paged_layout``). Several new tokens behind cached ones need their keys gathered, with
offsets of their own as cu_k. Nothing reads device data on the host, so a step can be
captured into a graph; from one step to the next the program drops the pages taken
(``counts[1]``) from the front of its free ones.

The kernels are HIP (csrc/serve.hip, ``libmi355_serve.so``, C ABI in
include/mi355_serve.h); the checks and launches are csrc/serve_binding.cpp
(``libmi355_serve_ops.so``). There is no fallback: forward only, on the GPU only; a
call that needs a derivative is refused, while tracing too.
Every failure of a check is a ``RuntimeError``, as of the operators of fa.py.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

NAMESPACE = "recsys_ops"
ABI_VERSION = 1

SCHEMAS = {
    "mha_packed_fwd":
        "mha_packed_fwd(Tensor q, Tensor k, Tensor v, Tensor cu_q, Tensor cu_k, bool causal=True, float? scale=None, "
        "float softcap=0., int window=0, Tensor? slopes=None, Tensor? prefix_lens=None) -> Tensor",
    "mha_paged_decode":
        "mha_paged_decode(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_table, Tensor kv_lens, float? scale=None, "
        "float softcap=0., int window=0, Tensor? slopes=None) -> Tensor",
    "rope_paged_store":
        "rope_paged_store(Tensor q, Tensor k, Tensor v, Tensor positions, Tensor inv_freq, Tensor slot_map, "
        "Tensor(a!) k_cache, Tensor(b!) v_cache, bool interleaved=False, float amplitude=1.) -> (Tensor, Tensor)",
    "paged_layout":
        "paged_layout(Tensor seq_lens, Tensor new_lens, Tensor block_table, Tensor free_pages, int page_size, "
        "int max_tokens) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)",
}

_lib: Optional[ctypes.CDLL] = None
_ops_lib: Optional[ctypes.CDLL] = None
_torch_lib = None
_path: Optional[str] = None


def loaded_path() -> Optional[str]:
    """The library this process opened, if any."""
    return _path


def _fakes() -> dict:
    def attention(q, *args, **kwargs):
        return q.new_empty(q.shape)

    def rope(q, k, *args, **kwargs):
        return q.new_empty(q.shape), k.new_empty(k.shape)

    def layout(seq_lens, new_lens, block_table, free_pages, page_size, max_tokens):
        n = seq_lens.shape[0]
        return (seq_lens.new_empty(n), seq_lens.new_empty(n + 1), seq_lens.new_empty(max_tokens),
                seq_lens.new_empty(max_tokens, dtype=torch.int64), block_table.new_empty(block_table.shape),
                seq_lens.new_empty(3))

    return {"mha_packed_fwd": attention, "mha_paged_decode": attention, "rope_paged_store": rope, "paged_layout": layout}


def _cpu(name: str):
    def refuse(*args, **kwargs):
        raise RuntimeError(f"{name} is only supported on CUDA")
    return refuse


def register(library: str, native: str) -> None:
    """Open the library and the compiled implementation over it, and register the
    operators with the dispatcher (idempotent)."""
    global _lib, _ops_lib, _torch_lib, _path
    if _torch_lib is not None:
        return
    lib = ctypes.CDLL(library)
    version = getattr(lib, "mi355_serve_abi_version", None)
    if version is None or version() != ABI_VERSION:
        raise RuntimeError(f"{library}: not a library of ABI version {ABI_VERSION}; rebuild it")
    ops = ctypes.CDLL(native)
    torch_lib = torch.library.Library(NAMESPACE, "FRAGMENT")
    for schema in SCHEMAS.values():
        torch_lib.define(schema)
    ops.mi355_serve_connect.argtypes = [ctypes.c_void_p]
    ops.mi355_serve_connect.restype = ctypes.c_int
    if ops.mi355_serve_connect(lib._handle) != 0:
        raise RuntimeError(f"{native} does not fit {library}; rebuild both")
    for name, fake in _fakes().items():
        torch_lib.impl(name, _cpu(name), "CPU")
        torch.library.register_fake(f"{NAMESPACE}::{name}", fake, lib=torch_lib)
    _lib, _ops_lib, _torch_lib, _path = lib, ops, torch_lib, library


def rotary_frequencies(rot: int, base: float = 10000.0, *, scaling: Optional[str] = None, factor: float = 1.0,
                       original_len: int = 0, beta_fast: float = 32.0, beta_slow: float = 1.0, device=None):
    """``(inv_freq, amplitude)`` for ``rope_paged_store``: the float64 radians per
    position of the rot / 2 pairs, and the factor of q and k.

    ``scaling`` stretches the positions for contexts ``factor`` times as long:
    ``"linear"`` divides every frequency by it; ``"ntk"`` raises the base by
    factor^(rot / (rot - 2)), which leaves the fastest pair and divides the slowest;
    ``"yarn"`` (Peng et al. 2023) leaves pairs that turn more than ``beta_fast`` times
    over ``original_len`` positions, divides those under ``beta_slow``, blends
    between, and has the amplitude 0.1·ln(factor) + 1."""
    if rot < 0 or rot % 16:
        raise RuntimeError("rot must be a multiple of 16")
    if not (base > 1 and math.isfinite(base) and factor >= 1 and math.isfinite(factor)):
        raise RuntimeError("base must be above 1 and factor at least 1, both finite")
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise RuntimeError("scaling must be None, 'linear', 'ntk' or 'yarn'")
    if scaling == "ntk" and rot:
        base = base * factor ** (rot / (rot - 2))
    i = torch.arange(rot // 2, dtype=torch.float64)
    freq = base ** (-2.0 * i / max(rot, 1))
    amplitude = 1.0
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "yarn":
        if original_len <= 0 or not beta_fast > beta_slow > 0:
            raise RuntimeError("yarn needs original_len > 0 and beta_fast > beta_slow > 0")
        turns = original_len * freq / (2 * math.pi)
        keep = ((turns - beta_slow) / (beta_fast - beta_slow)).clamp(0, 1)
        freq = freq * keep + freq / factor * (1 - keep)
        amplitude = 0.1 * math.log(factor) + 1.0
    return freq.to(device) if device is not None else freq, amplitude
