"""Attention over sequences of tokens: the global counterpart of the local operators (``qk``, ``av``, ``sapa_fused``), for the encoders and
decoders around an upsampler.  The reference has no such operator.

``packed_attention`` takes whole sequences packed one behind the other and is differentiable; ``paged_attention`` takes new tokens, one or
many a sequence, over a cache of keys and values in pages, into which ``paged_write`` puts the new keys and values.  Checks, allocation and
the autograd node are native (``csrc/host_attention.inc``), the kernels are in ``csrc/attention.cu``.
"""
from __future__ import annotations

from torch.autograd import Function, forward_ad

from . import _lib


def packed_attention(query, key, value, offsets, key_offsets=None, causal=True, scale=None):
    """``out[t, h] = sum_j softmax_j(scale * <query[t, h], key[j, g]>) value[j, g]`` over the keys j that token t sees; g is the key head that
    query head h shares, ``h // (heads // groups)``.  Differentiable with respect to query, key and value.

    ``query`` [T, heads, dim]; ``key``, ``value`` [S, groups, dim]: float32, float16 or bfloat16, dim a multiple of 8 up to 128, any strides (a
    tensor whose rows are not dense and 16-byte aligned is copied).  ``offsets`` [B + 1], int32 on the device: sequence b is the tokens
    ``offsets[b]`` to ``offsets[b + 1]``, and its keys ``key_offsets[b]`` to ``key_offsets[b + 1]`` (``offsets`` where not given).  With ``causal``
    token i of a sequence sees the keys j <= i + keys - tokens, without it all of its sequence.  ``scale``: 1 / sqrt(dim) where not given.

    A token that sees no key gets 0, and so do rows of no sequence.  What a token does not see has no part in its output or in any
    gradient, not even if it is infinite or NaN.  The lengths stay on the device: the call can be captured into a graph and replayed with
    others.  Deterministic.

    ``offsets`` do not decrease.  Where they do, nothing outside the tensors is read or written, but rows of sequences that overlap, or that the last offset
    leaves out, hold any numbers.  In 16 bits the softmax's weights, and dS in the gradients, are rounded to the type for the products that take them (up
    to 64 tokens dS keeps what that leaves out; in float16 it is held by a power of two, so that gradients of any size neither vanish nor overflow on the
    way), and a quarter of the forward's exponentials are off by up to 1.0e-4 (bfloat16) or 2.8e-6 (float16) of themselves; sums, statistics and delta are
    float32."""
    if _lib.transformed():
        return PackedAttentionFunction.apply(query, key, value, offsets, key_offsets, causal, scale)
    return (_lib.host or _lib.load_host()).packed_attention(query, key, value, offsets, key_offsets, causal, scale)


class PackedAttentionFunction(Function):
    """``packed_attention`` for traces and transforms."""

    @staticmethod
    def forward(ctx, query, key, value, offsets, key_offsets, causal, scale):
        out, lse, low, scale = _lib.load_host().packed_attention_forward(query, key, value, offsets, key_offsets, causal, scale)
        ctx.config = (causal, scale)
        ctx.save_for_backward(query, key, value, out, lse, low, offsets, offsets if key_offsets is None else key_offsets)
        return out

    @staticmethod
    def backward(ctx, grad_output):
        return (*_lib.load_host().packed_attention_backward(grad_output, *ctx.saved_tensors, *ctx.config), None, None, None, None)


def paged_attention(query, key_pages, value_pages, page_table, key_lengths, offsets, causal=True, scale=None):
    """Attention of new tokens over a paged cache; forward only.

    ``query`` [T, heads, dim], packed as in :func:`packed_attention`; ``key_pages``, ``value_pages`` [pages, page, groups, dim] of any strides that are
    multiples of 16 bytes; ``page_table`` [B, most pages] and ``key_lengths`` [B], int32 on the device.  Position p of sequence b lies in slot
    ``p % page`` of page ``page_table[b, p // page]``; its keys are the positions below ``key_lengths[b]``, which counts the new tokens: with ``causal``
    token i of Lq sees the positions up to ``key_lengths[b] - Lq + i``.

    In 16 bits pages of 8, 16, 32, ... slots (powers of two) go through the tensor cores.  Pages of other sizes are served by the kernel of float32, which takes
    15 times as long for single tokens and 40 times for chunks (48 sequences of up to 8190 keys: 150 and 2200 us; six chunks of 512 tokens: 165 and 6500).

    Entries of the table behind a sequence's last page are not read.  A token that sees a position whose page number lies outside the
    cache, or that the table has no entry for, gets NaN; the page is not read."""
    if _lib.transformed():
        return PagedAttentionFunction.apply(query, key_pages, value_pages, page_table, key_lengths, offsets, causal, scale)
    return (_lib.host or _lib.load_host()).paged_attention(query, key_pages, value_pages, page_table, key_lengths, offsets, causal, scale)


class PagedAttentionFunction(Function):
    """``paged_attention`` for traces; under transforms it raises."""

    @staticmethod
    def forward(ctx, query, key_pages, value_pages, page_table, key_lengths, offsets, causal, scale):
        _forward_only("paged_attention", ctx)
        return _lib.load_host().paged_attention(query, key_pages, value_pages, page_table, key_lengths, offsets, causal, scale)

    @staticmethod
    def backward(ctx, grad_output):
        raise NotImplementedError("paged_attention is forward only")


def paged_write(key, value, key_pages, value_pages, page_table, key_lengths, offsets):
    """Put new keys and values, [T, groups, dim] packed by ``offsets``, into the cache in place: token i of the Lq new ones of sequence b goes to
    position ``key_lengths[b] - Lq + i``, so ``key_lengths`` already counts them.  Positions below 0 or without a page inside the cache
    are skipped; nothing else of the cache is touched.  No two tokens of a call may go to the same slot."""
    if _lib.transformed():
        if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in (key, value, key_pages, value_pages)):
            raise NotImplementedError("paged_write is not differentiable")      # here: the Function would first write
        PagedWriteFunction.apply(key, value, key_pages, value_pages, page_table, key_lengths, offsets)
        return
    (_lib.host or _lib.load_host()).paged_write(key, value, key_pages, value_pages, page_table, key_lengths, offsets)


class PagedWriteFunction(Function):
    """``paged_write`` for traces, as a step without a result that is used; under transforms it raises."""

    @staticmethod
    def forward(ctx, key, value, key_pages, value_pages, page_table, key_lengths, offsets):
        _forward_only("paged_write", ctx)
        _lib.load_host().paged_write(key, value, key_pages, value_pages, page_table, key_lengths, offsets)
        return key.new_empty(0)                          # a trace keeps no step without one

    @staticmethod
    def backward(ctx, grad_output):
        raise NotImplementedError("paged_write is not differentiable")


def _forward_only(name, ctx):
    if any(ctx.needs_input_grad):
        raise NotImplementedError(f"{name} has no gradients")
