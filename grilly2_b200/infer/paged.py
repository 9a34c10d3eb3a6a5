"""A paged int8 KV cache for several requests at once: block tables and slot maps built on the device, the append that
fills the blocks, and the attention that reads them. No counterpart in the reference, whose cache is contiguous, float32
and of batch 1 (crates/grilly-infer/src/kv_cache.rs:1-33).

    cache = PagedKvCache.for_model(cfg, seqs=32, blocks=4096)
    step = PagedStep(cache, max_tokens=32)
    cache.plan(counts, step)                        # once per step
    q = cache.append(layer, qkv, heads, cos, sin, step)   # per layer
    y = cache.attend(layer, q, heads, step, max_count=1)
    cache.advance(step)                             # once per step
    cache.release(finished)                         # blocks of finished requests go back on the free list

Everything a step depends on (lengths, counts, tables, the free list) lives on the device, so a captured step replays.
"""
from __future__ import annotations

import ctypes

import numpy as np

from .. import _C, _lib
from .._lib import check

__all__ = ["PagedKvCache", "PagedStep"]

_BUFFERS = {"k": "int32", "v": "int32", "kscale": "float32", "vscale": "float32", "table": "int32", "lens": "int32", "free": "int32",
            "free_count": "int32"}


def _held(buffers, name, dtype, size, make):
    """The caller's tensor, or a new one: `size` elements of `dtype` at the start of their buffer."""
    t = buffers.pop(name, None)
    if t is None:
        return make()
    if not isinstance(t, _C.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if t.dtype != dtype or t.offset or t.numel() < size:
        raise RuntimeError(f"{name} must hold at least {size} {dtype} values at offset 0, got {list(t.shape)} {t.dtype} at {t.offset}")
    return t


def _filled(shape, dtype="int32", word=0):
    """A tensor of one 32-bit word, written on the device: a pool may be larger than the host's memory."""
    t = _C.Tensor.empty(shape, dtype, persistent=True)
    check(_lib.load().gq_fill(_C.context(), t.storage.handle, 0, 4 * t.numel(), word))
    return t


def _operand(t, dtype, what, size=None):
    if not isinstance(t, _C.Tensor):
        raise TypeError(f"{what} must be a tensor, got {type(t).__name__}")
    if t.dtype != dtype:
        raise NotImplementedError(f"grilly: {what} with dtype {t.dtype} is not implemented yet (expected {dtype})")
    if t.offset:
        raise RuntimeError(f"{what} must lie at offset 0 of its buffer, got {t.offset}")
    if size is not None and t.numel() != size:
        raise RuntimeError(f"{what} must hold {size} values, got {list(t.shape)}")
    return t.storage.handle


class PagedKvCache:
    """The pool, the block tables and the free list (the layouts are include/gq.h's). ``buffers`` may supply any of
    ``k``, ``v`` (int8 codes as int32 words), ``kscale``, ``vscale``, ``table``, ``lens``, ``free``, ``free_count``; what is missing
    is allocated, the tables empty and every block free."""

    def __init__(self, *, layers: int, kv_heads: int, head_dim: int, blocks: int, seqs: int, max_blocks: int, block_size: int = 64,
                 buffers: dict | None = None) -> None:
        self.layers, self.kv_heads, self.head_dim = int(layers), int(kv_heads), int(head_dim)
        self.blocks, self.seqs, self.max_blocks, self.block_size = int(blocks), int(seqs), int(max_blocks), int(block_size)
        if min(self.layers, self.kv_heads, self.head_dim, self.blocks, self.seqs, self.max_blocks, self.block_size) < 1:
            raise RuntimeError("a paged cache needs at least one layer, head, block and request")
        if self.block_size not in (16, 32, 64, 128):
            raise RuntimeError(f"block_size must be 16, 32, 64 or 128, got {self.block_size}")
        if self.head_dim not in (32, 64, 128):
            raise RuntimeError(f"head_dim must be 32, 64 or 128, got {self.head_dim}")
        given = dict(buffers or {})
        scales = self.layers * self.blocks * self.kv_heads
        words = scales * self.block_size * self.head_dim // 4
        sizes = {"k": words, "v": words, "kscale": scales, "vscale": scales, "table": self.seqs * self.max_blocks, "lens": self.seqs,
                 "free": self.blocks, "free_count": 1}
        make = {"table": lambda: _filled((self.seqs, self.max_blocks), word=0xFFFFFFFF),
                "free": lambda: _C.Tensor.from_numpy(np.arange(self.blocks, dtype=np.int32)[::-1].copy(), persistent=True),
                "free_count": lambda: _C.Tensor.from_numpy(np.array([self.blocks], dtype=np.int32), persistent=True)}
        for name, dtype in _BUFFERS.items():
            setattr(self, name, _held(given, name, dtype, sizes[name], make.get(name, lambda n=sizes[name], d=dtype: _filled((n,), d))))
        if given:
            raise RuntimeError(f"a paged cache has no buffers {sorted(given)}")
        self._desc = _lib.PagedCache(layers=self.layers, blocks=self.blocks, block_size=self.block_size, kv_heads=self.kv_heads, dim=self.head_dim,
                                     seqs=self.seqs, max_blocks=self.max_blocks, **{n: getattr(self, n).storage.handle for n in _BUFFERS
                                                                                   if not n.startswith("free")})
        self._ref = ctypes.byref(self._desc)

    @classmethod
    def for_model(cls, cfg, *, seqs: int, blocks: int, block_size: int = 64) -> "PagedKvCache":
        """A cache for a ``LlamaConfig``; a request may grow to ``cfg.max_cache_len`` tokens."""
        return cls(layers=cfg.num_hidden_layers, kv_heads=cfg.num_key_value_heads, head_dim=cfg.head_dim, blocks=blocks, seqs=seqs,
                   max_blocks=-(-cfg.max_cache_len // block_size), block_size=block_size)

    def nbytes(self) -> int:
        return 4 * (2 * self.k.numel() + 2 * self.kscale.numel())

    def lengths(self) -> np.ndarray:
        return self.lens.numpy()

    def free_blocks(self) -> int:
        return int(self.free_count.numpy()[0])

    def plan(self, counts: "_C.Tensor", step: "PagedStep") -> "PagedStep":
        """Where the next counts[b] tokens of every request go (gq_paged_plan)."""
        check(_lib.load().gq_paged_plan(_C.context(), self._ref, _operand(counts, "int32", "counts", self.seqs), self.free.storage.handle,
                                        self.free_count.storage.handle, step._ref))
        return step

    def advance(self, step: "PagedStep") -> None:
        check(_lib.load().gq_paged_advance(_C.context(), self._ref, step._ref))

    def release(self, which: "_C.Tensor") -> None:
        """which: int32 [seqs], non-zero for the requests whose blocks go back on the free list."""
        check(_lib.load().gq_paged_release(_C.context(), self._ref, _operand(which, "int32", "which", self.seqs), self.free.storage.handle,
                                           self.free_count.storage.handle))

    def append(self, layer: int, qkv: "_C.Tensor", heads: int, cos: "_C.Tensor", sin: "_C.Tensor", step: "PagedStep",
               q_out: "_C.Tensor | None" = None) -> "_C.Tensor":
        """Rotary, then k and v of the fused rows into the blocks; returns the rotated q [max_tokens, heads * head_dim]."""
        rows, width = step.max_tokens, heads * self.head_dim
        q = q_out if q_out is not None else _C.Tensor.empty((rows, width), "float32")
        if cos.numel() % self.head_dim or cos.numel() != sin.numel():
            raise RuntimeError(f"cos and sin must be (positions, {self.head_dim}), got {list(cos.shape)} and {list(sin.shape)}")
        check(_lib.load().gq_paged_append(
            _C.context(), self._ref, layer, _operand(qkv, "float32", "qkv", rows * (width + 2 * self.kv_heads * self.head_dim)), heads,
            _operand(cos, "float32", "cos"), _operand(sin, "float32", "sin"), cos.numel() // self.head_dim, step._ref,
            _operand(q, "float32", "q_out", rows * width)))
        return q

    def attend(self, layer: int, q: "_C.Tensor", heads: int, step: "PagedStep", *, scale: float | None = None, max_count: int | None = None,
               out: "_C.Tensor | None" = None) -> "_C.Tensor":
        """Causal grouped-query attention of the step's rows over the cache. ``max_count``: the largest count the caller
        expects of a request (1 for a decode step; the default is the step's room), which chooses how the work is cut."""
        rows, width = step.max_tokens, heads * self.head_dim
        y = out if out is not None else _C.Tensor.empty((rows, width), "float32")
        check(_lib.load().gq_paged_attn(
            _C.context(), self._ref, layer, _operand(q, "float32", "q", rows * width), heads,
            float(self.head_dim) ** -0.5 if scale is None else float(scale), step._ref, rows if max_count is None else max_count,
            _operand(y, "float32", "out", rows * width)))
        return y


class PagedStep:
    """The maps of one step with room for ``max_tokens`` rows (include/gq.h, gq_paged_step), reused from step to step."""

    def __init__(self, cache: PagedKvCache, max_tokens: int, buffers: dict | None = None) -> None:
        self.max_tokens = int(max_tokens)
        if self.max_tokens < 1:
            raise RuntimeError("a step needs room for at least one row")
        given = dict(buffers or {})
        runs = min(self.max_tokens, self.max_tokens // cache.block_size + 2 * cache.seqs)
        sizes = {"starts": cache.seqs + 1, "slots": self.max_tokens, "positions": self.max_tokens, "runs": runs + 1, "last": cache.seqs, "info": 2}
        for name, n in sizes.items():
            setattr(self, name, _held(given, name, "int32", n, lambda n=n: _filled((n,))))
        if given:
            raise RuntimeError(f"a step has no buffers {sorted(given)}")
        self._desc = _lib.PagedStep(max_tokens=self.max_tokens, **{n: getattr(self, n).storage.handle for n in sizes})
        self._ref = ctypes.byref(self._desc)

    def shortfall(self) -> int:
        """Blocks that the last plan's rows lack: the free list was empty, then or when the entry's first tokens came (a host
        copy; waits for the device)."""
        return int(self.info.numpy()[1])

    def dropped(self) -> int:
        """Rows of the last plan whose token has no place in the pool and so is neither cached nor seen: the blocks that
        ``shortfall`` counts were missing, or the request has outgrown its table, which it does not count (a host copy; waits for the device)."""
        return int((self.slots.numpy()[:int(self.info.numpy()[0])] < 0).sum())
