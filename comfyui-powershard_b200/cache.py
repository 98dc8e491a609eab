"""Keys and values of earlier tokens in 8 bits, in pages, and attention over them.

Streaming generation appends the tokens of a few frames at a time and attends
all that came before; 40 layers of 32760 tokens x 40 heads hold 26.8 GB in 16
bits and half of it here.  ``KVCache`` is one layer's storage: ``write``
quantises new rows as it stores them (e4m3 or int8 codes, one fp32 scale per
token and head), ``read`` gives rows back in 16 bits for the attention, into
one workspace that all layers share.  Page tables and lengths are device
tensors and nothing synchronises, so a step can be captured into a CUDA graph.

``StreamingAttention`` runs a step: append, read back, attend (dense or
block-sparse).
"""
from __future__ import annotations

import torch
from torch.autograd.graph import increment_version

from . import _lib, ops
from .contract import AttentionOptions
from .provider import B200Provider
from .sparse import SparseProvider, _no_grad


class KVCache:
    """Codes k, v [pages, page_rows, heads, head_dim] and scales k_scale, v_scale
    [pages, page_rows, heads] of one layer.

    Position p of sequence b is row ``p % page_rows`` of page
    ``table[b, p // page_rows]`` (int32 [B, n], on the cache's device).  Which
    pages a sequence owns is the caller's book-keeping; sequences may share
    pages that they only read.  One ``write`` must not name a position twice.
    Both calls run forward only (rows that require grad are refused while
    autograd records) and count as operations in place on what they change."""

    def __init__(self, pages: int, page_rows: int, heads: int, head_dim: int = 128,
                 dtype: torch.dtype = torch.float8_e4m3fn, device=None):
        if min(pages, page_rows, heads) < 1:
            raise ValueError("KVCache: pages, page_rows and heads must be positive")
        if dtype not in ops._CODES or head_dim not in (64, 128, 256):
            raise _lib.UnsupportedAttention("KVCache: float8_e4m3fn or int8 codes and heads of 64, 128 or 256, "
                                            f"got {dtype} and {head_dim}")
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        shape = (pages, page_rows, heads, head_dim)
        self._set(*(torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype) for _ in range(2)),
                  *(torch.zeros(shape[:3], dtype=torch.float32, device=device) for _ in range(2)))

    @classmethod
    def over(cls, k, v, k_scale, v_scale) -> "KVCache":
        """A cache in tensors the caller owns (a slice of one pool for all layers)."""
        self = cls.__new__(cls)
        self._set(k, v, k_scale, v_scale)
        return self

    def _set(self, k, v, k_scale, v_scale):
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale

    def write(self, k, v, table, start=None, lengths=None):
        """Rows i < lengths[b] (None: all) of k, v [B, n, heads, head_dim] to
        positions start[b] + i (None: i) of sequence b.  Rows without a page are dropped."""
        _no_grad(k, v)
        ops.cache_write((self.k, self.v), (self.k_scale, self.v_scale), (k, v), table, start, lengths)
        increment_version((self.k, self.v, self.k_scale, self.v_scale))

    def read(self, table, lengths, k_out, v_out, first=None):
        """Positions first[b] + i (None: i) below lengths[b] into row i of k_out,
        v_out [B, n, heads, head_dim] (bf16 or fp16); the other rows stay as they are."""
        _no_grad(k_out, v_out)
        ops.cache_read((self.k, self.v), (self.k_scale, self.v_scale), (k_out, v_out), table, lengths, first)
        increment_version((k_out, v_out))


class StreamingAttention:
    """Attention of new tokens over a cache that they are appended to.

    ``provider``: a ``SparseProvider``, or a dense ``B200Provider`` where every
    sequence holds the same number of rows."""

    def __init__(self, cache: KVCache, provider):
        self.cache, self.provider = cache, provider

    def __call__(self, q, k, v, table, start, options: AttentionOptions | None = None, *, context: int | None = None,
                 lengths=None, **selection):
        """q, k, v [B, n, H, D] new rows -> [B, n, Hq, D].

        start: rows that the sequences hold already, an int for all of them or
        an int32 device tensor [B]; lengths: new rows in use, int32 [B] (taken
        as within [0, n]) or None for all; context: rows of the longest sequence
        with the new ones, needed with a tensor (rows behind it are held but not
        attended); selection: ``allowed`` of a sparse provider.

        The table must name a page for every position below the rows held with
        the new ones and below ``context``: that it has as many entries is
        checked, but the pages are on the device, and a position whose page is
        out of range is attended as a key and a value of zeros."""
        _no_grad(q, k, v)
        b, n = k.shape[:2]
        ragged = lengths is not None or not isinstance(start, int)
        if ragged and not isinstance(self.provider, SparseProvider):
            raise ValueError("sequences of different lengths need a SparseProvider")
        if isinstance(start, int):
            if start < 0 or context not in (None, start + n):
                raise ValueError(f"start {start} with {n} new rows makes a context of {start + n}, got {context}")
            context = start + n
        elif context is None:
            raise ValueError("context: the rows of the longest sequence, with start on the device")
        rows = table.shape[-1] * self.cache.k.shape[1]
        if context > rows:
            raise ValueError(f"the page table names {rows} rows of a sequence, a context of {context} needs more pages")
        keys, values = (torch.empty((b, context, *k.shape[2:]), dtype=k.dtype, device=k.device) for _ in range(2))
        if isinstance(self.provider, B200Provider):  # before the write: a refused step changes nothing
            self.provider.check(q, keys, values, options or AttentionOptions())
            if isinstance(self.provider, SparseProvider):
                self.provider.check_selection(q, keys, selection.get("allowed"), selection.get("key_means"))
            elif selection:
                raise ValueError(f"a dense provider takes no {', '.join(selection)}")
        if isinstance(start, int):
            start = torch.full((b,), start, dtype=torch.int32, device=k.device)
        if lengths is not None:
            lengths = lengths.clamp(0, n)  # of what the write takes
        self.cache.write(k, v, table, start, lengths)
        held = start + (n if lengths is None else lengths)
        self.cache.read(table, held, keys, values)
        if not ragged:
            return self.provider(q, keys, values, options, **selection)
        return self.provider(q, keys, values, options, query_lengths=lengths, key_lengths=held, **selection)
