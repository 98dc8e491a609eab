"""Attention over the key blocks that a cheap score selects for each query block.

``SparseProvider(keep)(q, k, v, options)`` has the calling convention of the
dense ``B200Provider``, so a dispatcher (or the wrapper that H3 puts around
it: VedaDispatch, powershard/veda/runtime.py:95-110) calls one like the other.
It runs three steps, each also an entry point of its own for callers that keep
a plan (the selected blocks) or the key means between calls:

* ``block_means(x, block)`` - the mean row of each block, held in fp32;
* ``select_blocks(query_means, key_means, keep)`` - the ``keep`` key blocks
  with the largest <mean query, mean key> for each query block, among those
  that ``allowed`` and the lengths leave (ties: the lower index);
* ``sparse_attention(q, k, v, blocks, counts)`` - softmax attention of each
  query block over its listed key blocks.

Query blocks are multiples of 256 rows (the two query tiles of a CTA share
their keys), key blocks multiples of 64.  Lengths are int32 device tensors
[B]: rows behind them are not used whatever they hold, and are zeros in the
output, as is a query that has no key.  Scores are 32-bit numbers: scaled, times
log2 e, they may reach 2^27 in magnitude (2^30 in bf16), as in the dense kernel.
Nothing here synchronises, so every call can be captured into a CUDA graph.
"""
from __future__ import annotations

import contextlib
import math

import torch
from torch.autograd import forward_ad

from . import _lib, ops
from .contract import AttentionOptions, UnsupportedAttention
from .provider import B200Provider, _tma_ok

NAME = "b200_sparse"
_DEFAULT = AttentionOptions()
QUERY_BLOCK, KEY_BLOCK = 256, 128


def _readable(t: torch.Tensor) -> torch.Tensor:
    """t, or a contiguous copy where its strides do not suit the kernels'
    loads (an expanded axis has stride 0, which a tensor map cannot hold)."""
    if t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t
    return t if _tma_ok(t) and all(s > 0 or n == 1 for s, n in zip(t.stride(), t.shape)) else t.clone(
        memory_format=torch.contiguous_format)


_HERE = contextlib.nullcontext()


def _on(device: torch.device):
    """Context in which `device` is current (nothing to do where it is)."""
    return _HERE if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _broadcast(allowed, shape):
    try:
        return allowed.broadcast_to(shape)
    except RuntimeError as error:
        raise ValueError(f"allowed {tuple(allowed.shape)} does not broadcast to {shape} "
                         "(batch, heads, query blocks, key blocks)") from error


def _no_grad(*tensors):
    """The kernels run forward only: a call that autograd would record, or whose tangents it would carry on, is refused."""
    for t in tensors:
        if t.requires_grad and torch.is_grad_enabled():
            raise UnsupportedAttention("b200_sparse: forward only, an input requires grad")
    if forward_ad._current_level >= 0:  # inside a dual_level only
        for t in tensors:
            if forward_ad.unpack_dual(t).tangent is not None:
                raise UnsupportedAttention("b200_sparse: an input has a forward-mode tangent, which would be lost")


def block_means(x, block: int, lengths=None):
    """Mean over the rows in use of each block of ``block`` rows of x [B, L, H, 128]:
    fp32 [B, ceil(L/block), H, 128] (a block without any row in use: zeros)."""
    ops._check16(x, "block_means")
    _no_grad(x)
    shape = x.shape
    if len(shape) != 4 or block < 1:
        raise ValueError(f"block_means: expected [B, L, H, D] and a positive block, got {tuple(shape)}, {block}")
    x = _readable(x)
    b, n, h, d = shape
    out = x.new_empty((b, -(-n // block), h, d), dtype=torch.float32)
    with _on(x.device):
        ops.block_means([x], [block], [lengths], [out])
    return out


def select_blocks(query_means, key_means, keep: int, *, allowed=None, query_block: int = QUERY_BLOCK,
                  key_block: int = KEY_BLOCK, query_lengths=None, key_lengths=None):
    """(blocks int32 [B, Hq, nq, n], counts int32 [B, Hq, nq]) with n = min(keep, nk): the chosen
    key blocks of each query block in ascending order, -1 behind the first ``counts`` of them.

    query_means [B, nq, Hq, 128], key_means [B, nk, Hk, 128] as ``block_means``
    gives them; allowed: bool, broadcastable to [B, Hq, nq, nk]."""
    if query_means.dim() != 4 or key_means.dim() != 4:
        raise ValueError("select_blocks: means are [B, blocks, H, D]")
    b, nq, h, _ = query_means.shape
    nk = key_means.shape[1]
    for t in (query_means, key_means):
        _lib.require_cuda(t, "select_blocks")
    _no_grad(query_means, key_means)
    if keep < 1:
        raise ValueError(f"select_blocks: keep must be at least 1, got {keep}")
    if allowed is not None:
        allowed = _broadcast(allowed, (b, h, nq, nk))
    keep = min(int(keep), nk)
    device = query_means.device
    blocks = query_means.new_empty((b, h, nq, keep), dtype=torch.int32)
    counts = query_means.new_empty((b, h, nq), dtype=torch.int32)
    with _on(device):
        ops.block_select(query_means, key_means, keep, blocks, counts, query_block, key_block, allowed, query_lengths,
                         key_lengths)
    return blocks, counts


_status: dict[int, ops.PinnedStatus] = {}


def _status_for(device: torch.device) -> ops.PinnedStatus:
    if device.index not in _status:
        _status[device.index] = ops.PinnedStatus(device)
    return _status[device.index]


def sparse_attention(q, k, v, blocks, counts=None, *, query_block: int = QUERY_BLOCK, key_block: int = KEY_BLOCK,
                     softmax_scale: float | None = None, query_lengths=None, key_lengths=None):
    """Attention of q [B, Lq, Hq, 128] over the key blocks of k/v [B, Lk, Hk, 128] that ``blocks``
    [B, Hq, ceil(Lq/query_block), n] names (``counts``: entries in use, None: all).  An entry
    outside the key blocks names no key; an entry that occurs twice counts twice."""
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        ops._check16(t, f"sparse_attention {name}")
        if t.dim() != 4:
            raise ValueError(f"sparse_attention {name}: expected [B, L, H, D], got {tuple(t.shape)}")
    _no_grad(q, k, v)
    status = _status_for(q.device)
    status.poll()
    q, k, v = _readable(q), _readable(k), _readable(v)
    scale = q.shape[-1] ** -0.5 if softmax_scale is None else float(softmax_scale)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    with _on(q.device):
        workspace = ops.sparse_attention_workspace(q.shape[0], q.shape[2], q.shape[1], blocks.shape[-1], key_block,
                                                   q.device)
        ops.sparse_attention(q, k, v, out, blocks, counts, query_block, key_block, scale, status, workspace,
                             query_lengths, key_lengths)
    return out


class SparseProvider(B200Provider):
    """Block-sparse attention behind the provider API.

    keep: key blocks that each query block attends - a number of blocks, or a
    fraction of them in (0, 1] as a float."""

    name = NAME

    def __init__(self, keep, *, query_block: int = QUERY_BLOCK, key_block: int = KEY_BLOCK):
        super().__init__()
        if isinstance(keep, float) and not 0 < keep <= 1 or not isinstance(keep, float) and keep < 1:
            raise ValueError(f"keep: a positive number of blocks or a fraction in (0, 1], got {keep}")
        if query_block < 256 or query_block % 256 or key_block < 64 or key_block % 64:
            raise ValueError("query_block is a multiple of 256 and key_block of 64, "
                             f"got {query_block} and {key_block}")
        self.keep, self.query_block, self.key_block = keep, query_block, key_block
        self.identity["provider"] = NAME

    def check(self, q, k, v, o: AttentionOptions):
        # What needs no word is seen at a glance (the checks one by one take 3 us
        # of a 25 us call); anything else gets them, and their errors.
        dtype, at, qs, ks = q.dtype, q.get_device(), q.shape, k.shape
        if not (o is _DEFAULT and (dtype is torch.bfloat16 or dtype is torch.float16) and len(qs) == len(ks) == 4
                and qs[3] == ks[3] == 128 and v.shape == ks and qs[0] == ks[0] > 0 and ks[1] and qs[2] and ks[2]
                and qs[2] % ks[2] == 0 and k.dtype is dtype and v.dtype is dtype
                and at == k.get_device() == v.get_device() >= 0):
            super().check(q, k, v, o)
        if o.softmax_scale is not None and not o.softmax_scale > 0:
            raise UnsupportedAttention("b200_sparse: the selection ranks by a positive softmax_scale")
        _no_grad(q, k, v)

    def check_selection(self, q, k, allowed=None, key_means=None):
        """(key blocks, allowed broadcast to [B, Hq, query blocks, key blocks]) of a call; errors before any launch."""
        (b, lq, h, d), (_, lk, hk, _) = q.shape, k.shape
        nq, nk = -(-lq // self.query_block), -(-lk // self.key_block)
        if allowed is not None:
            allowed = _broadcast(allowed, (b, h, nq, nk))
            if allowed.dtype != torch.bool or allowed.device != q.device:
                raise ValueError(f"allowed must be bool on {q.device}, got {allowed.dtype} on {allowed.device}")
        if key_means is not None and (tuple(key_means.shape) != (b, nk, hk, d) or key_means.dtype != torch.float32
                                      or not key_means.is_contiguous() or key_means.device != q.device):
            raise ValueError(f"key_means: expected contiguous fp32 {(b, nk, hk, d)} on {q.device}")
        return nk, allowed

    def blocks_kept(self, key_blocks: int) -> int:
        """Key blocks each query block attends, of ``key_blocks``."""
        # 0.07 * 100 is a little above 7
        n = max(1, math.ceil(self.keep * key_blocks - 1e-9)) if isinstance(self.keep, float) else self.keep
        return min(n, key_blocks)

    def __call__(self, q, k, v, o: AttentionOptions | None = None, *, allowed=None, key_means=None,
                 query_lengths=None, key_lengths=None):
        """q [B, Lq, Hq, 128], k/v [B, Lk, Hk, 128] -> [B, Lq, Hq, 128].

        key_means: ``block_means(k, key_block, key_lengths)`` kept from an
        earlier call (of a cache that grew, its new blocks' means appended);
        allowed: bool, broadcastable to [B, Hq, query blocks, key blocks]."""
        o = o or _DEFAULT
        self.check(q, k, v, o)
        device = q.device
        status = _status_for(device)
        status.poll()
        q, k, v = _readable(q), _readable(k), _readable(v)
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        if q.shape[1] == 0:
            return out
        nk, allowed = self.check_selection(q, k, allowed, key_means)
        scale = q.shape[-1] ** -0.5 if o.softmax_scale is None else float(o.softmax_scale)
        with _on(device):
            ops.sparse_forward(q, k, v, out, self.blocks_kept(nk), self.query_block, self.key_block, scale, status,
                               key_means, allowed, query_lengths, key_lengths)
        return out
