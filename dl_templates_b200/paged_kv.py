"""Serving form of the operators in ``rope_axes.py`` and ``sink_swa.py``: a paged cache of keys and values.

  ``kv_append_rope(q, k, v, positions, tables, k_cache, v_cache, page_table, seq_lens, new_lens=None) -> q_rot``
  ``sink_swa_decode(q, k_cache, v_cache, page_table, seq_lens, window, n_sink, sm_scale) -> o``

``k_cache [pages, Hkv, page_size, d_qk]``, ``v_cache [pages, Hkv, page_size, d_v]`` (any strides: a ``[pages, page_size, Hkv, d]``
tensor as a permuted view too) and ``page_table`` int32 ``[B, max_pages]``: position ``p`` of sequence ``b`` lies in slot ``p % page_size`` of page
``page_table[b, p // page_size]``.  ``seq_lens`` int32 ``[B]``: the tokens of each sequence, those of the step included, so that one tensor serves
both calls of a step.  All three live on the device and are read there: a step can be captured into a CUDA graph and replayed
while they change.  A page number outside the cache is no page -- nothing is written to it and nothing of it is seen -- so that
pages that neither the window nor the sinks reach can be given back and their entries set to -1.

Two new tokens of one call never share a slot: the pages they fall into belong to one sequence each (a page that several sequences
read, a shared prefix, may stand in all their tables).  Neither call records gradients, tangents or a jit trace: inputs that ask for one are refused.
"""
from __future__ import annotations

from . import _lib
from ._lib import native as _native

_NO_TABLES = ()


def kv_append_rope(q, k, v, positions, tables, k_cache, v_cache, page_table, seq_lens, new_lens=None):
    """Writes new tokens into the cache: ``k [B,Hkv,T,d_qk]`` rotated by ``positions`` (int32 ``[axes, T]`` or ``[B, axes, T]``) and ``tables`` as in
    ``RotaryPEAxes``, ``v [B,Hkv,T,d_v]`` as it is, and returns ``q [B,Hq,T,d_qk]`` rotated the same way in a new tensor; one launch.

    Row ``t`` of sequence ``b`` becomes position ``seq_lens[b] - n + t`` with ``n = new_lens[b]`` (``None``: ``T``); rows from ``n`` on are padding and
    written nowhere.  ``q`` may be ``None`` (returns ``None``); ``positions`` may be ``None``: nothing is rotated."""
    return _native.kv_append(q, k, v, positions, _NO_TABLES if tables is None else tables, k_cache, v_cache, page_table, seq_lens,
                             new_lens)


def sink_swa_decode(q, k_cache, v_cache, page_table, seq_lens, window, n_sink, sm_scale=1.0, impl="auto", out=None):
    """Attention of one new token per sequence: ``q [B,Hq,1,d_qk]`` stands at position ``seq_lens[b] - 1`` (its key and value are in the cache
    already) and sees positions ``p >= seq_lens[b] - window`` and ``p < n_sink``.  Returns ``o [B,Hq,1,d_v]`` (``out``: a tensor to write it
    into, apart from ``q`` and the cache); zeros for a sequence of no tokens."""
    return _native.sink_decode(q, k_cache, v_cache, page_table, seq_lens, window, n_sink, sm_scale, _lib.impl_code(impl), out)
