"""The streaming KV cache of a decoder layer in 8 bits, and attention over it, on the B200 kernels
(csrc/kv_cache.cu, csrc/kv_attend.cu).  No counterpart in the reference, whose decode keeps
transformers' 16-bit DynamicCache (src/duplex/streaming/clock.py:155-156).

  kv_append(k_new, v_new, k, v, k_scale, v_scale, block_table, kv_len, *, cu_q, weights, err)
  kv_attend(q, k, v, k_scale, v_scale, block_table, kv_len, *, cu_q, window, sinks, softmax_scale,
            weights, out, lse, return_lse, err) -> out or (out, lse)
  kv_evict(k, v, k_scale, v_scale, block_table, kv_len, weights, dst_table, *, keep, sinks, recent,
           err) -> kv_len of the kept tokens
  PackedKVCache(n_blocks, kv_heads, ...): the buffers of one layer with these as methods

Storage (include/duplex_b200.h): codes k, v [n_blocks, kv_heads, block, dim], torch.float8_e4m3fn or
torch.int8; one fp32 scale per (block, head), k_scale, v_scale [n_blocks, kv_heads]; value = code *
scale, and the scales that `kv_append` and `kv_evict` write are powers of two.  dim 64 or 128, block
16, 32, 64 or 128 tokens.  A sequence's tokens lie in order in the blocks of its row of block_table
[batch, width] (int32); kv_len [batch] (int32) counts them, the rows of the call included: call
`kv_append` and then `kv_attend` with the same kv_len.  cu_q [batch + 1] (int32) gives the
sequences' row offsets in q (or k_new and v_new); without it every sequence has as many rows.
Row t of a sequence's T is its token kv_len - T + t.

All index tensors are read on the device: a call makes no host synchronisation, and a captured one
follows new lengths, tables and values.  Calls run on the current stream of the cache's device;
`kv_attend` and `kv_evict` take their workspace from torch's allocator, so calls on several streams
do not share one.  Inference only, no autograd formula.  Errors in arguments raise RuntimeError;
what the device arrays get wrong is reported in `err` (int32 [1]) if it is given: block ids out of
range (_lib.DEVERR_BLOCK), values that are not finite (_lib.DEVERR_NONFINITE), a kv_len beyond what its
row of the table holds (_lib.DEVERR_LENGTH; tokens past the table are left out: not stored, not seen,
not kept), and row offsets that fall (_lib.DEVERR_OFFSETS; the call then does nothing else, `out` and
the caches stay as they were).
"""

from __future__ import annotations

import torch

from duplex import _lib

FORMATS = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}

_ops = None


def _op(name):
    global _ops
    if _ops is None:
        _ops = _lib.load_torch_ops()
    return getattr(_ops, name)


def _inference(*ts):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts):
        raise _lib.DuplexError("the KV cache's operators have no gradients: pass detached tensors")


def kv_append(k_new, v_new, k, v, k_scale, v_scale, block_table, kv_len, *, cu_q=None, weights=None,
              err=None) -> None:
    """Store rows k_new, v_new [n, kv_heads, dim] (fp16 or bf16, any row and head strides: views of a
    q|k|v buffer need no copy) as the last tokens of their sequences.

    A block's scale is 2^e, the least e >= -126 with max|x| <= top * 2^e over its tokens (top 448 for
    e4m3, 127 for int8); a code is x * 2^-e rounded once, ties to even.  In a block that already holds
    older tokens of the sequence e never falls; when it rises, their codes are rounded again at the new
    scale.  With `weights` the new tokens' accumulated weights become 0.  Values that are not finite
    are stored as 0 (DEVERR_NONFINITE).  Rows that would lie before token 0 are not stored.  Two
    sequences may share blocks that are full, not one that either appends to."""
    _inference(k_new, v_new)
    _op("kv_append")(k_new, v_new, k, v, k_scale, v_scale, block_table, kv_len, cu_q, weights, err)


def kv_attend(q, k, v, k_scale, v_scale, block_table, kv_len, *, cu_q=None, window=0, sinks=0,
              softmax_scale=None, weights=None, out=None, lse=None, return_lse=False, err=None):
    """Causal attention of rows q [n, heads, dim] (fp16 or bf16; heads a multiple of kv_heads) over the
    cache: out [n, heads, dim] in q's type and, if asked for, lse [n, heads] fp32, the natural
    logarithm of each row's sum of exp(q.k * softmax_scale) (default 1 / sqrt(dim)).

    window = 0: a row sees its own token and all before.  window > 0: the last `window` of those, and
    the sequence's first `sinks` tokens.  Windows count cached tokens, so after `kv_evict` they count
    kept ones.  Blocks that no row sees are not read, and their table entries may be anything; slots
    that no row sees may hold any code.  (An e4m3 NaN in a token that one row of a call sees may reach
    rows that do not: 0 * NaN.  kv_append stores none.)  A row that sees nothing (kv_len smaller than
    its sequence's rows) gets 0 and -inf.  Rows behind the last sequence's are left as they were
    (without `out` and `lse`: they may hold anything).

    Scales need not be powers of two, nor near one another; prompts are slower where a sequence and head
    has others than powers of two within 2^14 of its largest.  Beside its relative error a row's out may
    be off by 2^-28 of the largest value it sees (a probability times a block's scale is held in fp16).

    weights [n_blocks, kv_heads, block] fp32: each seen token's entry grows by its attention weights,
    summed over the call's rows and the query heads of its KV head.  `out` must not overlap q."""
    _inference(q)
    if out is None and lse is None:
        out, lse = _op("kv_attend")(q, k, v, k_scale, v_scale, block_table, kv_len, cu_q, softmax_scale,
                                    window, sinks, weights, err)
        return (out, lse) if return_lse else out
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if lse is None and return_lse:
        lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
    _op("kv_attend_into")(q, k, v, k_scale, v_scale, block_table, kv_len, cu_q, softmax_scale, window,
                          sinks, weights, out, lse, err)
    return (out, lse) if return_lse else out


def kv_evict(k, v, k_scale, v_scale, block_table, kv_len, weights, dst_table, *, keep, sinks=0,
             recent=0, err=None) -> torch.Tensor:
    """Keep at most `keep` tokens of each (sequence, KV head): the first `sinks`, the last `recent`, and
    of the rest those with the largest `weights` (ties: the earlier one; NaN counts as the largest).
    They move, in their order, to the blocks of dst_table [batch, >= keep / block] with their weights,
    rounded at scales of the destination blocks; returns their number, [batch] int32, the kv_len to go
    on with (and dst_table as the block_table).  Sequences of at most `keep` tokens are copied whole.

    The source blocks are not written, so shared ones stay valid for the other sequences and the caller
    can free the rest.  A destination block must not be a source block of the call, nor appear twice."""
    return _op("kv_evict")(k, v, k_scale, v_scale, block_table, kv_len, weights, dst_table, keep, sinks,
                           recent, err)


class PackedKVCache:
    """One layer's cache: codes, scales and (track_weights) accumulated attention weights of n_blocks
    blocks, and the operators on them.  Block tables and lengths are the caller's, one set for all
    layers."""

    def __init__(self, n_blocks, kv_heads, head_dim=128, block=64, fmt="e4m3", track_weights=False,
                 device="cuda"):
        if fmt not in FORMATS:
            raise _lib.DuplexError(f"unknown KV format {fmt!r}: one of {sorted(FORMATS)}")
        if head_dim not in (64, 128) or block not in (16, 32, 64, 128):
            raise _lib.DuplexError(f"unsupported KV cache geometry: head_dim {head_dim}, block {block}")
        shape = (n_blocks, kv_heads, block, head_dim)
        self.block, self.fmt = block, fmt
        self.k = torch.zeros(shape, dtype=torch.uint8, device=device).view(FORMATS[fmt])
        self.v = torch.zeros(shape, dtype=torch.uint8, device=device).view(FORMATS[fmt])
        self.k_scale = torch.ones(shape[:2], dtype=torch.float32, device=device)
        self.v_scale = torch.ones(shape[:2], dtype=torch.float32, device=device)
        self.weights = torch.zeros(shape[:3], dtype=torch.float32, device=device) if track_weights else None
        self.err = torch.zeros(1, dtype=torch.int32, device=device)

    def _buffers(self):
        return self.k, self.v, self.k_scale, self.v_scale

    def append(self, k_new, v_new, block_table, kv_len, cu_q=None) -> None:
        kv_append(k_new, v_new, *self._buffers(), block_table, kv_len, cu_q=cu_q, weights=self.weights,
                  err=self.err)

    def attend(self, q, block_table, kv_len, cu_q=None, window=0, sinks=0, softmax_scale=None, out=None,
               lse=None, return_lse=False, accumulate=True):
        """kv_attend; with track_weights the weights grow unless accumulate is False."""
        return kv_attend(q, *self._buffers(), block_table, kv_len, cu_q=cu_q, window=window, sinks=sinks,
                         softmax_scale=softmax_scale, weights=self.weights if accumulate else None,
                         out=out, lse=lse, return_lse=return_lse, err=self.err)

    def evict(self, block_table, kv_len, dst_table, keep, sinks=0, recent=0) -> torch.Tensor:
        if self.weights is None:
            raise _lib.DuplexError("eviction needs the accumulated weights: build the cache with track_weights")
        return kv_evict(*self._buffers(), block_table, kv_len, self.weights, dst_table, keep=keep,
                        sinks=sinks, recent=recent, err=self.err)

    def device_errors(self) -> int:
        """The device error word (DUPLEX_DEVERR_* bits) of this cache's launches, read and cleared."""
        n = int(self.err.item())
        self.err.zero_()
        return n
