"""bf16 KV cache with O(1) rollback, laid out for the verify-attention kernel.

Semantics follow the caches the reference drives (mlx-lm ``KVCache``; its own ``BatchCache``,
batch_engine.py:193-224): buffers ``[B, Hk, capacity, D]`` grown in steps of :data:`STEP` rows
(batch_engine.py:38, :226-227); :meth:`update_and_fetch` writes T rows at ``offset`` and returns
``[..., :offset, :]`` views (no copy — the kernel reads the strides); :meth:`trim` is pure
metadata: ``offset -= n`` clamped at 0, the next write overwrites the stale tail
(batch_engine.py:220-224; tests/test_batch_engine.py:57-73). Dense rollback trims every layer's
cache by the rejected count (target.py:679-696).

MI355X layout note: with 288 GB of HBM the cache is allocated once at its final capacity when
the caller knows it (``capacity=``), so verify rounds never reallocate; growth copies only when
an unknown length overflows.
"""

from __future__ import annotations

import torch

from . import ops

STEP = 256


def _round_step(n: int) -> int:
    return ((n + STEP - 1) // STEP) * STEP


class KVCache:
    def __init__(self, batch: int, kv_heads: int, head_dim: int, *, device, capacity: int = 0,
                 dtype=torch.bfloat16):
        self.batch, self.kv_heads, self.head_dim = batch, kv_heads, head_dim
        self.device, self.dtype = torch.device(device), dtype
        cap = _round_step(max(capacity, 1))
        self.keys = torch.zeros((batch, kv_heads, cap, head_dim), dtype=dtype, device=self.device)
        self.values = torch.zeros_like(self.keys)
        self.offset = 0

    @property
    def capacity(self) -> int:
        return self.keys.shape[2]

    def _grow(self, need: int) -> None:
        cap = _round_step(need)
        nk = torch.zeros((self.batch, self.kv_heads, cap, self.head_dim), dtype=self.dtype, device=self.device)
        nv = torch.zeros_like(nk)
        nk[:, :, :self.offset] = self.keys[:, :, :self.offset]
        nv[:, :, :self.offset] = self.values[:, :, :self.offset]
        self.keys, self.values = nk, nv

    def update_and_fetch(self, keys: torch.Tensor, values: torch.Tensor):
        """Write ``keys``/``values`` [B, Hk, T, D] at ``offset``; return the ``[..., :offset, :]`` views."""
        t = keys.shape[2]
        if self.offset + t > self.capacity:
            self._grow(self.offset + t)
        self.keys[:, :, self.offset:self.offset + t] = keys
        self.values[:, :, self.offset:self.offset + t] = values
        self.offset += t
        return self.fetch()

    def reserve(self, t: int) -> None:
        """Make room for ``t`` more rows at ``offset`` (a kernel then writes them in place)."""
        if self.offset + t > self.capacity:
            self._grow(self.offset + t)

    def advance(self, t: int) -> None:
        """Commit ``t`` rows a kernel wrote at ``offset`` (after :meth:`reserve`)."""
        if self.offset + t > self.capacity:
            raise ValueError(f"advance({t}) past capacity {self.capacity} at offset {self.offset}")
        self.offset += t

    def fetch(self):
        return self.keys[:, :, :self.offset, :], self.values[:, :, :self.offset, :]

    def trim(self, n: int) -> int:
        """Roll back ``n`` rows (metadata only). Returns how many were removed."""
        n = min(self.offset, max(0, int(n)))
        self.offset -= n
        return n

    def is_trimmable(self) -> bool:
        return True

    @property
    def state(self):
        return self.fetch()


class QuantizedKVCache:
    """KV cache holding affine-quantized rows: mlx-lm's ``QuantizedKVCache`` layout, which the
    reference's targets use when ``kv_bits`` is set (target.py:166-184). Keys and values are
    each ``(words int32 [B, Hk, cap, D*bits/32], scales [B, Hk, cap, D/64], biases ...)`` with
    scales and biases in the model dtype; rows are quantized as they are written
    (:func:`dspark_rocm.quant.quantize_rows`). Offset, ``trim`` and growth behave as in
    :class:`KVCache`; :meth:`update_and_fetch` returns the two triples as ``[..., :offset, :]``
    views, which ``ops.verify_attention_quantized`` reads in place."""

    def __init__(self, batch: int, kv_heads: int, head_dim: int, *, bits: int = 8, group_size: int = 64, device,
                 capacity: int = 0, dtype=torch.bfloat16):
        self.batch, self.kv_heads, self.head_dim = batch, kv_heads, head_dim
        self.bits, self.group_size = bits, group_size
        self.device, self.dtype = torch.device(device), dtype
        self.keys = self._alloc(_round_step(max(capacity, 1)))
        self.values = self._alloc(self.keys[0].shape[2])
        self.offset = 0

    def _alloc(self, cap: int):
        B, H, D = self.batch, self.kv_heads, self.head_dim
        w = torch.zeros((B, H, cap, D * self.bits // 32), dtype=torch.int32, device=self.device)
        s = torch.zeros((B, H, cap, D // self.group_size), dtype=self.dtype, device=self.device)
        return (w, s, torch.zeros_like(s))

    @property
    def capacity(self) -> int:
        return self.keys[0].shape[2]

    def _grow(self, need: int) -> None:
        cap = _round_step(need)
        nk, nv = self._alloc(cap), self._alloc(cap)
        for new, old in zip(nk + nv, self.keys + self.values):
            new[:, :, :self.offset] = old[:, :, :self.offset]
        self.keys, self.values = nk, nv

    def update_and_fetch(self, keys: torch.Tensor, values: torch.Tensor):
        """Quantize ``keys``/``values`` [B, Hk, T, D] into rows ``offset..offset+T``; return the
        ``[..., :offset, :]`` views of both triples."""
        from .quant import quantize_rows

        t = keys.shape[2]
        if self.offset + t > self.capacity:
            self._grow(self.offset + t)
        if self._kernel(keys, values):
            rows = lambda trip: tuple(a[:, :, self.offset:self.offset + t] for a in trip)
            ops.quantize_kv(keys, values, rows(self.keys), rows(self.values), bits=self.bits, group_size=self.group_size)
        else:
            for dst, src in ((self.keys, keys), (self.values, values)):
                for buf, part in zip(dst, quantize_rows(src, self.bits, self.group_size, self.dtype)):
                    buf[:, :, self.offset:self.offset + t] = part
        self.offset += t
        return self.fetch()

    def _kernel(self, keys: torch.Tensor, values: torch.Tensor) -> bool:
        """Whether ``ops.quantize_kv`` writes these rows (the same values in one launch): rows and cache on
        one GPU, whole rows of the cache's own shape, nothing recording gradients."""
        if not ops.eager_inference(keys, values, *self.keys, *self.values):
            return False
        return (keys.shape == values.shape and keys.dim() == 4 and keys.dtype == values.dtype
                and keys.dtype in ops.DEQUANT_DTYPES and self.dtype in ops.KV_CACHE_DTYPES and keys.shape[2] > 0
                and tuple(keys.shape[:2]) == (self.batch, self.kv_heads) and keys.shape[3] == self.head_dim
                and self.bits in ops.KV_BITS and self.group_size == ops.GROUP
                and self.head_dim % ops.GROUP == 0 and self.head_dim <= 4096
                and 2 * self.batch * self.kv_heads <= 65535
                and self._buffers_fit(self.keys) and self._buffers_fit(self.values))

    def _buffers_fit(self, trip) -> bool:
        """Whether a triple is as :meth:`_alloc` makes it, but for its capacity: buffers put in its place may not be."""
        w, s, b = trip
        B, H, cap, n = w.shape
        st = s.stride()
        return (w.dtype in (torch.int32, torch.uint32) and (B, H, 32 * n) == (self.batch, self.kv_heads, self.head_dim * self.bits)
                and s.dtype is self.dtype and b.dtype is self.dtype
                and s.shape == b.shape == (B, H, cap, self.head_dim // self.group_size)
                and w.stride(3) == 1 and st[3] == 1 and st == b.stride())

    def reserve(self, t: int) -> None:
        """Make room for ``t`` more rows at ``offset`` (a kernel then writes them in place)."""
        if self.offset + t > self.capacity:
            self._grow(self.offset + t)

    def advance(self, t: int) -> None:
        """Commit ``t`` rows a kernel wrote at ``offset`` (after :meth:`reserve`)."""
        if self.offset + t > self.capacity:
            raise ValueError(f"advance({t}) past capacity {self.capacity} at offset {self.offset}")
        self.offset += t

    def fetch(self):
        view = lambda trip: tuple(a[:, :, :self.offset] for a in trip)
        return view(self.keys), view(self.values)

    def trim(self, n: int) -> int:
        n = min(self.offset, max(0, int(n)))
        self.offset -= n
        return n

    def is_trimmable(self) -> bool:
        return True

    @property
    def state(self):
        return self.fetch()
