"""The package's front door: ``ops``, one object per process that hands out the
operator groups and the operators themselves.

Public surface (names, signatures and behaviour of the reference facade
``RecsysOps``, recsys.py:451-656, for the one group built here):

    ops.mha_fwd_with_mask(q, k, v, mask, backend=None)   recsys.py:641-656
    ops.is_available(group=None), ops.load_error(group=None), ops.groups
    ops.ensure_loaded(*groups), ops.load()
    ops.load_precompiled(group, library_path, metadata_path=None)
    ops.allow_jit / ops.configure(allow_jit=...) / ops.disable_jit()
    ops.<op name>  -> the dispatcher op, after its group is loaded

How it is organised here: the facade owns one ``_Slot`` per group. A slot
records the group's loader (created on first need) and where its library came
from: ``"tree"`` (development: the in-tree build, compiled by hipcc if it is
missing) or ``"artifact"`` (deployment: a sealed, validated export). The
policy is a single flag, ``allow_jit``; turning it off (explicitly, or by
loading an artifact) freezes the facade: from then on a slot is only ever
read, never loaded, and asking for an unloaded group raises
``CustomOpsError``.
"""
from __future__ import annotations

import os
import threading
from typing import Optional

import torch

from . import serve
from .loader import CustomOpsError, FAOps, ServeOps

# group name -> loader class; operator name -> group name
GROUP_LOADERS = {"fa": FAOps, "serve": ServeOps}
OP_GROUPS = {"mha_fwd_with_mask": "fa", **{name: "serve" for name in serve.SCHEMAS}}

# Groups that calls naming no group stand for: the reference's. The others load by
# name or at their operators' first call, and appear in ``ops.groups`` from then on,
# so a program that uses the attention alone deploys and reports it alone.
_DEFAULT_GROUPS = ("fa",)

_BACKENDS = ("auto", "cuda", "hip")


def resolve_backend(backend: Optional[str]) -> str:
    """The backend a call runs on: the argument, else ``CUSTOM_OPS_BACKEND``,
    else ``"auto"`` (the reference's order, recsys.py:140-158).

    Every accepted name means the same thing here, the HIP library (the device
    type is still called "cuda" on PyTorch-ROCm). ``"tilelang"`` is refused:
    there is no second backend and no silent fallback to one."""
    name = backend if backend is not None else os.environ.get("CUSTOM_OPS_BACKEND", "auto")
    name = str(name).strip().lower()
    if name == "tilelang":
        raise RuntimeError(
            "backend 'tilelang': the Tile-lang backend does not exist in this build; "
            "the HIP kernels for MI355X are the only backend (use backend='auto')")
    if name not in _BACKENDS:
        raise ValueError(f"backend {name!r} is not one of {list(_BACKENDS)} "
                         f"(argument or CUSTOM_OPS_BACKEND)")
    return name


def _as_flag(value) -> bool:
    if type(value) is not bool:
        raise TypeError(f"allow_jit must be a bool, not {type(value).__name__}")
    return value


class _Slot:
    """One op group as the facade sees it."""

    __slots__ = ("loader", "origin")

    def __init__(self) -> None:
        self.loader: Optional[FAOps] = None
        self.origin: Optional[str] = None     # None | "tree" | "artifact"

    @property
    def ready(self) -> bool:
        return self.loader is not None and self.loader.is_available()

    @property
    def state(self) -> str:
        if self.loader is None:
            return "not_loaded"
        return "loaded" if self.loader.is_available() else "failed"


class RecsysOps:
    """Facade over the operator groups: the reference's ``fa``, and ``serve``."""

    def __init__(self, *, allow_jit: bool = True) -> None:
        self._mu = threading.RLock()
        self._slots = {name: _Slot() for name in GROUP_LOADERS}
        self._jit = _as_flag(allow_jit)
        self._serve_ops = None   # torch.ops.recsys_ops once the group "serve" is ready

    # ── policy ──────────────────────────────────────────────────────────────
    @property
    def allow_jit(self) -> bool:
        """True: groups load lazily from the in-tree build. False: only groups
        loaded with ``load_precompiled`` are usable."""
        return self._jit

    @allow_jit.setter
    def allow_jit(self, value: bool) -> None:
        self.configure(allow_jit=value)

    def configure(self, *, allow_jit: bool) -> "RecsysOps":
        """Set the policy for this facade and every loader it holds; loads nothing."""
        flag = _as_flag(allow_jit)
        with self._mu:
            self._jit = flag
            for slot in self._slots.values():
                if slot.loader is not None:
                    slot.loader.configure(allow_jit=flag)
        return self

    def disable_jit(self) -> "RecsysOps":
        return self.configure(allow_jit=False)

    # ── groups ──────────────────────────────────────────────────────────────
    def _slot(self, group: str) -> _Slot:
        try:
            return self._slots[group]
        except (KeyError, TypeError):
            raise ValueError(f"unknown group {group!r}: this build provides "
                             f"{sorted(self._slots)}") from None

    def _acquire(self, group: str) -> FAOps:
        """The group's loader with its library loaded, loading it if the policy allows."""
        with self._mu:
            slot = self._slot(group)
            if slot.ready:
                return slot.loader
            if not self._jit:
                why = slot.loader.load_error() if slot.loader is not None else None
                raise CustomOpsError(
                    f"JIT is disabled and group {group!r} is not loaded: deploy it with "
                    f"ops.load_precompiled({group!r}, library_path, metadata_path=None)"
                    + (f"; its last load failed with: {why}" if why else ""))
            if slot.loader is None:
                slot.loader = GROUP_LOADERS[group](allow_jit=True)
            slot.loader.load()                  # raises CustomOpsError on failure
            slot.origin = "tree"
            return slot.loader

    def load_precompiled(self, group: str, library_path, metadata_path=None) -> "RecsysOps":
        """Validate and load a deployed library (sidecar defaults to
        ``<library_path>.json``). The facade stays in strict mode afterwards,
        whether or not the load succeeds."""
        with self._mu:
            slot = self._slot(group)
            self.configure(allow_jit=False)
            self._serve_ops = None
            if slot.loader is None:
                slot.loader = GROUP_LOADERS[group](allow_jit=False)
            slot.loader.load_precompiled(library_path, metadata_path)
            slot.origin = "artifact"
        return self

    def ensure_loaded(self, *groups: str) -> "RecsysOps":
        """Load the named groups (the reference's when none is named). Unknown names
        are rejected before anything loads."""
        with self._mu:
            for g in groups:
                self._slot(g)
            for g in groups or _DEFAULT_GROUPS:
                self._acquire(g)
        return self

    def load(self) -> "RecsysOps":
        return self.ensure_loaded()

    @property
    def groups(self) -> dict:
        """``{group: "loaded" | "failed" | "not_loaded"}``, of the reference's groups and
        those beside them that were asked for."""
        with self._mu:
            return {name: slot.state for name, slot in self._slots.items()
                    if name in _DEFAULT_GROUPS or slot.loader is not None}

    def is_available(self, group: Optional[str] = None) -> bool:
        """Whether the named group (else the facade as a whole) can run.

        With ``allow_jit`` the question loads what it asks about; in strict mode
        it only reads the current state. Without a group it also needs a
        visible GPU, and in strict mode at least one deployed group."""
        with self._mu:
            if group is not None:
                slot = self._slot(group)
                if not self._jit:
                    return slot.ready
                try:
                    self._acquire(group)
                except CustomOpsError:
                    return False
                return True
            if not torch.cuda.is_available():
                return False
            if not self._jit:
                created = [s for s in self._slots.values() if s.loader is not None]
                return bool(created) and all(s.ready for s in created)
            try:
                self.ensure_loaded()
            except CustomOpsError:
                return False
            return True

    def load_error(self, group: Optional[str] = None) -> Optional[str]:
        """The last load error of the named group, else of the first failed
        one; never loads anything."""
        with self._mu:
            slots = [self._slot(group)] if group is not None else list(self._slots.values())
            for slot in slots:
                if slot.loader is not None and (group is not None or not slot.ready):
                    err = slot.loader.load_error()
                    if err or group is not None:
                        return err
        return None

    # ── operators ───────────────────────────────────────────────────────────
    def mha_fwd_with_mask(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                          mask: torch.Tensor, backend: Optional[str] = None) -> torch.Tensor:
        """FlashAttention-2 forward with an additive fp16/bf16 mask (recsys.py:641-656).

        q [B,H,Sq,d], k/v [B,Hk,Sk,d] (H % Hk == 0), mask [B,1,>=Sq,>=Sk] with
        0 = visible, -inf = blocked, finite = bias. d in {64, 128}."""
        if backend is not None or "CUSTOM_OPS_BACKEND" in os.environ:
            resolve_backend(backend)
        # (a slot that is ready is only read: no lock on the per-call path)
        slot = self._slots["fa"]
        if not slot.ready:
            self._acquire("fa")
        return torch.ops.recsys_ops.mha_fwd_with_mask(q, k, v, mask)

    def _serve(self, backend: Optional[str]):
        """The dispatcher's operators, with the group ``serve`` loaded. (The environment's
        backend is looked up when the group loads: a look costs 0.6 us, a tenth of a
        small call.)"""
        if backend is not None:
            resolve_backend(backend)
        found = self._serve_ops
        if found is None:
            with self._mu:
                resolve_backend(None)
                self._acquire("serve")
                found = self._serve_ops = torch.ops.recsys_ops
        return found

    def mha_packed_fwd(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor, cu_k: torch.Tensor,
                       causal: bool = True, scale: Optional[float] = None, softcap: float = 0.0, window: int = 0,
                       slopes: Optional[torch.Tensor] = None, prefix_lens: Optional[torch.Tensor] = None,
                       backend: Optional[str] = None) -> torch.Tensor:
        """Attention over packed sequences; rows of different sequences do not see each other.

        q [Tq,H,d], k/v [Tk,Hk,d] (fp16/bf16, H % Hk == 0, d in {64, 128}; views whose
        strides are multiples of 8 elements do); cu_q/cu_k [N+1] int32: sequence n's
        rows and keys, ascending. Position: the last row stands at the last key. Row i sees key j
        if j <= i (causal) and |i - j| < window (window > 0), and sees the first
        prefix_lens[n] keys in any case. Scores: scale·q·k (default 1/sqrt(d)), then
        softcap·tanh(s/softcap), then - slopes[h]·|i - j| (slopes [H] float32). A row
        that sees no key, and one of no sequence, gives 0. Returns [Tq,H,d]."""
        return self._serve(backend).mha_packed_fwd(q, k, v, cu_q, cu_k, causal, scale, softcap, window, slopes, prefix_lens)

    def mha_paged_decode(self, q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                         kv_lens: torch.Tensor, scale: Optional[float] = None, softcap: float = 0.0, window: int = 0,
                         slopes: Optional[torch.Tensor] = None, backend: Optional[str] = None) -> torch.Tensor:
        """Attention of one new token per request over a paged cache that holds it.

        q [B,H,d]; caches [pages,Hk,page_size,d], page_size a power of two in 8 .. 1024;
        block_table [B,M] int32; kv_lens [B] int32, the new token among them. Scores as
        in ``mha_packed_fwd``, for the row at the last key. A page number outside the
        cache hides its keys; a request that sees no key gives 0. Returns [B,H,d]."""
        return self._serve(backend).mha_paged_decode(q, k_cache, v_cache, block_table, kv_lens, scale, softcap, window, slopes)

    def rope_paged_store(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
                         inv_freq: torch.Tensor, slot_map: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                         interleaved: bool = False, amplitude: float = 1.0, backend: Optional[str] = None):
        """Rotary positions of q and k, and the turned k and v into a paged cache.

        q [T,H,d], k/v [T,Hk,d] (views do, as above); positions [T] int32; inv_freq
        [rot/2] float64 radians per position (see ``rotary_frequencies``), rot a multiple
        of 16 up to d; slot_map [T] int64, slot = page·page_size + row, one outside the
        cache (-1) stores nothing, two tokens of a call may not share one. Pairs are
        elements (i, i + rot/2), or (2i, 2i + 1) if interleaved. Writes the caches
        [pages,Hk,page_size,d] in place; returns the turned (q, k), contiguous."""
        return self._serve(backend).rope_paged_store(q, k, v, positions, inv_freq, slot_map, k_cache, v_cache, interleaved,
                                                     amplitude)

    def paged_layout(self, seq_lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor,
                     free_pages: torch.Tensor, page_size: int, max_tokens: int, backend: Optional[str] = None):
        """Page tables, slots and positions of a step, from the requests' lengths.

        seq_lens/new_lens [N] int32 (N <= 8192): tokens cached and to add; block_table
        [N,M] int32: the pages held; free_pages [F] int32: requests take the pages they
        lack from its front, in order. Returns ``(kv_lens [N], cu_new [N+1], positions
        [max_tokens], slot_map [max_tokens] int64, table [N,M], counts [3])``: lengths
        after the step, offsets, position and slot of each new token (0 and -1 behind the
        last), the new table (-1 where there is no page) and {new tokens, pages taken,
        pages wanted and not had}. Tokens without a page have the slot -1."""
        return self._serve(backend).paged_layout(seq_lens, new_lens, block_table, free_pages, page_size, max_tokens)

    @staticmethod
    def rotary_frequencies(*args, **kwargs):
        """``(inv_freq, amplitude)`` for ``rope_paged_store``: see serve.rotary_frequencies."""
        return serve.rotary_frequencies(*args, **kwargs)

    def __getattr__(self, name: str):
        if name.startswith("_"):
            raise AttributeError(name)
        group = OP_GROUPS.get(name)
        if group is None:
            raise AttributeError(f"No op '{name}' in this build: it provides "
                                 f"{sorted(OP_GROUPS)} in groups {sorted(GROUP_LOADERS)}")
        self._acquire(group)
        return getattr(torch.ops.recsys_ops, name)

    def __repr__(self) -> str:
        origins = {n: s.origin for n, s in self._slots.items() if s.origin}
        return (f"RecsysOps(allow_jit={self._jit}, namespace='recsys_ops', backend='hip', "
                f"groups={self.groups}, origins={origins})")
