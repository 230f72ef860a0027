"""Operators for several continuations of a prompt on MI355X, beside the serving operators
(serve.py): beam search, parallel samples, batches behind one system prompt.

  * ``mha_shared_decode``  attention of one new token per request over the paged cache,
                           the prefix that requests share read once for all of them
  * ``beam_select``        the best continuations of each search's beams
  * ``paged_fork``         the page table of the chosen continuations; pages of the others freed
  * ``paged_copy``         the pages that a fork or a compaction moves, in a layer's caches
  * ``paged_compact``      pages in use moved to the front of the cache

A step of beam search: the model's logits go to ``beam_select``; ``paged_fork`` takes its
parents and gives the new table, lengths and free pages; ``paged_copy`` copies the last,
partly filled pages of beams with a common parent, in each layer's caches; then
``paged_layout`` (serve.py) gives slots of the new tokens, ``rope_paged_store`` fills them
and ``mha_shared_decode`` attends. Nothing reads device data on the host, so a step can be
captured into a graph.

The kernels are HIP (csrc/beam.hip, ``libmi355_beam.so``, C ABI in
include/mi355_beam.h); the checks and launches are csrc/beam_binding.cpp
(``libmi355_beam_ops.so``). There is no fallback: forward only, on the GPU only; a
call that needs a derivative is refused, while tracing too.
Every failure of a check is a ``RuntimeError``, as of the operators of fa.py.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from .serve import NAMESPACE, _cpu

ABI_VERSION = 1

SCHEMAS = {
    "mha_shared_decode":
        "mha_shared_decode(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_table, Tensor kv_lens, Tensor cu_groups, "
        "Tensor prefix_lens, float? scale=None, float softcap=0., int window=0, Tensor? slopes=None) -> Tensor",
    "beam_select":
        "beam_select(Tensor logits, Tensor scores, int k, Tensor? finished=None, int eos=-1) -> (Tensor, Tensor, Tensor)",
    "paged_fork":
        "paged_fork(Tensor block_table, Tensor seq_lens, Tensor parents, int page_size, int num_pages, Tensor? held=None) -> "
        "(Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)",
    "paged_compact":
        "paged_compact(Tensor block_table, Tensor seq_lens, int page_size, int num_pages, Tensor? held=None) -> "
        "(Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)",
    "paged_copy":
        "paged_copy(Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor src, Tensor dst) -> ()",
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

    def select(logits, scores, k, *args, **kwargs):
        shape = (logits.shape[0], k)
        return (logits.new_empty(shape, dtype=torch.float32), logits.new_empty(shape, dtype=torch.int32),
                logits.new_empty(shape, dtype=torch.int32))

    def fork(block_table, seq_lens, parents, page_size, num_pages, held=None):
        r, new = parents.shape[0], block_table.new_empty
        return new((r, block_table.shape[1])), new(r), new(r), new(r), new(num_pages), new(3)

    def compact(block_table, seq_lens, page_size, num_pages, held=None):
        new = block_table.new_empty
        return new(block_table.shape), new(num_pages // 2), new(num_pages // 2), new(num_pages), new(num_pages), new(2)

    def copy(k_cache, v_cache, src, dst):
        return None

    return {"mha_shared_decode": attention, "beam_select": select, "paged_fork": fork, "paged_compact": compact, "paged_copy": copy}


def register(library: str, native: str) -> None:
    """Open the library and the compiled implementation over it, and register the
    operators with the dispatcher (idempotent)."""
    global _lib, _ops_lib, _torch_lib, _path
    if _torch_lib is not None:
        return
    lib = ctypes.CDLL(library)
    version = getattr(lib, "mi355_beam_abi_version", None)
    if version is None or version() != ABI_VERSION:
        raise RuntimeError(f"{library}: not a library of ABI version {ABI_VERSION}; rebuild it")
    ops = ctypes.CDLL(native)
    torch_lib = torch.library.Library(NAMESPACE, "FRAGMENT")
    for schema in SCHEMAS.values():
        torch_lib.define(schema)
    ops.mi355_beam_connect.argtypes = [ctypes.c_void_p]
    ops.mi355_beam_connect.restype = ctypes.c_int
    if ops.mi355_beam_connect(lib._handle) != 0:
        raise RuntimeError(f"{native} does not fit {library}; rebuild both")
    for name, fake in _fakes().items():
        torch_lib.impl(name, _cpu(name), "CPU")
        torch.library.register_fake(f"{NAMESPACE}::{name}", fake, lib=torch_lib)
    _lib, _ops_lib, _torch_lib, _path = lib, ops, torch_lib, library
