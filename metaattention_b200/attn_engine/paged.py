"""Paged key / value caches of softmax attention with grouped heads: writing, reading back, and attention of new tokens
(csrc/paged_ops.cu, csrc/paged_attention.cu).  They stand beside the paged MLA decode of attn_engine/mla.py, whose
``block_table`` and ``cache_seqlens`` they share (the reference pages only that cache:
core/template/cute_template_kvshared/flash_api.cpp:61-210).

A step of a server, layer by layer::

    cache.append(k, v, block_table, cache_seqlens, cu_seqlens, rotary=rope)      # the new tokens' keys and values
    o = cache.attention(rope(q, positions=positions), block_table, cache_seqlens, cu_seqlens)

``cache_seqlens`` counts the tokens of each sequence WITH the new ones, which are its last; append, then attend.
"""

from __future__ import annotations

import torch

from core.native import lib as native


class PagedKVCache:
    """Pools of pages ``k``, ``v`` [num_pages, page_size, heads_kv, head_dim] in float16, bfloat16 or float8_e4m3fn, the last
    with ``k_scale``, ``v_scale`` [num_pages, page_size, heads_kv] (float8_e8m0fnu, or uint8 exponents): a code stands for
    code * 2^(exponent - 127), a row of exponent 255 for NaN.  The codes 0x7f and 0xff belong to such rows alone, as ``append`` writes
    them: in other rows ``read`` gives NaN for them, and ``attention``, which does not look for them, may take them for 480 times the
    scale.
    Any strides of whole 16 bytes with a contiguous last dimension; page_size a power of two of at least 8, head_dim 64 or 128.
    The pools are the caller's tensors and are written in place; they stay where they are (a call after one was resized or given
    other memory is refused).

    Common arguments: ``block_table`` int32 [batch, max_blocks] names the page of each page_size tokens of a sequence (entries
    behind its end may hold anything); ``cache_seqlens`` int32 [batch], tokens of each sequence with the new ones among them, at
    most max_blocks * page_size.  New tokens come as [batch, seq, heads, head_dim], the same number for every sequence, or
    with ``cu_seqlens`` int32 [batch + 1], which do not decrease, as packed rows [rows, heads, head_dim], those of sequence b being
    rows cu_seqlens[b] to cu_seqlens[b + 1] - 1.  Rows behind cu_seqlens[batch] take no part (padding of a captured step).  All
    of them on the cache's device; calls run on the current stream of that device."""

    def __init__(self, k, v, k_scale=None, v_scale=None):
        self._pools = (k, v, k_scale, v_scale)
        self._native = native.host().make_cache(*self._pools)

    def __getstate__(self):
        return {**self.__dict__, "_native": None}

    def __setstate__(self, state):
        self.__dict__.update(state)
        self._native = native.host().make_cache(*self._pools)

    k = property(lambda self: self._pools[0])
    v = property(lambda self: self._pools[1])
    k_scale = property(lambda self: self._pools[2])
    v_scale = property(lambda self: self._pools[3])

    @classmethod
    def allocate(cls, num_pages: int, page_size: int, heads_kv: int, head_dim: int, dtype=torch.bfloat16, device="cuda"):
        """A cache of zeros.  Page by page and head by head in memory, so that a head's rows of a page are one piece."""
        def pool():
            return torch.zeros(num_pages, heads_kv, page_size, head_dim, dtype=dtype, device=device).transpose(1, 2)

        def scale():
            if dtype != torch.float8_e4m3fn:
                return None
            return torch.zeros(num_pages, heads_kv, page_size, dtype=torch.uint8, device=device).view(torch.float8_e8m0fnu).transpose(1, 2)
        return cls(pool(), pool(), scale(), scale())

    @property
    def page_size(self) -> int:
        return self.k.shape[1]

    def append(self, k, v, block_table, cache_seqlens, cu_seqlens=None, rotary=None):
        """Writes the new tokens' k, v [.., heads_kv, head_dim] (float16 or bfloat16, the cache's own dtype unless that is 8
        bits) to the last positions of their sequences.  8 bits: a scale for each token and head, the least power of two that
        brings its largest magnitude to 448 at most; a row with a value that is not finite becomes NaN.  ``rotary`` (a
        RotaryEmbedding with a rotary_dim that is a multiple of 16) turns k by its positions on the way, rounded once.  Tokens at
        negative positions, and those whose table entry names no page, are not written; no two may have the same place, nor may the
        pools k and v be one."""
        turns = None
        if rotary is not None and self.k.is_cuda:
            turns = rotary.native_on(self.k.device)
        native.host().cache_append(self._native, k, v, block_table, cache_seqlens, cu_seqlens, turns)

    def read(self, block_table, cache_seqlens, max_len: int, dtype=None):
        """(k, v) [batch, max_len, heads_kv, head_dim]: the first ``max_len`` tokens of each sequence one after the other,
        zeros behind its end; float16 or bfloat16 ``dtype`` for an 8-bit cache (default bfloat16), else the cache's own."""
        if dtype is None:
            dtype = self.k.dtype if self.k_scale is None else torch.bfloat16
        if dtype not in native.DTYPE_CODES:
            raise ValueError(f"a cache is read in float16 or bfloat16 (got {dtype})")
        return tuple(native.host().cache_read(self._native, block_table, cache_seqlens, int(max_len), dtype == torch.bfloat16))

    def attention(self, q, block_table, cache_seqlens, cu_seqlens=None, scale=None, causal: bool = True, window=None, out=None,
                  return_lse: bool = False):
        """Softmax attention of the new tokens' q [.., heads, head_dim] over their sequences' keys, ``heads`` a multiple of
        heads_kv (query head h reads KV head h // (heads / heads_kv)): o like q, and with ``return_lse`` (o, lse), lse the
        log-sum-exp of each row in float32 [batch, heads, seq], packed [heads, rows].  With ``causal`` the row at position p sees the
        keys up to its own, with ``window`` only the last ``window`` of those, at a negative position none; without, every row sees
        all keys of its sequence, wherever it is.  A row that sees none gives 0 and -inf.  ``scale`` defaults to head_dim ** -0.5.
        Written to ``out`` if given; packed rows behind the last sequence are left as they are there (and are not initialised
        otherwise).  An 8-bit cache is read as the values of q's dtype that its codes stand for.  Keys and values inside a sequence
        must be finite; what lies behind its end is not looked at.  No backward pass, and no forward-mode one."""
        if window is not None and window <= 0:
            raise ValueError(f"window must be positive (got {window})")
        o, lse = native.host().cache_attention(self._native, q, block_table, cache_seqlens, cu_seqlens,
                                               self.k.shape[-1] ** -0.5 if scale is None else float(scale), bool(causal),
                                               0 if window is None else int(window), out, return_lse)
        return (o, lse) if return_lse else o
