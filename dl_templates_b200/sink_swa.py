"""Attention over a token sequence with a sliding window and sink tokens: token ``i`` sees token ``j`` if ``j <= i`` and
(``j > i - window`` or ``j < n_sink``) -- the ``window`` latest tokens up to itself, and the ``n_sink`` first ones.

  ``SinkSwa.apply(q, k, v, seq_lens, window, n_sink, sm_scale) -> o``                       differentiable
  ``sink_swa_fwd(q, k, v, window, n_sink, sm_scale=1.0, seq_lens=None) -> o``               forward only
  ``sink_swa_forward`` / ``sink_swa_backward``                                              with the softmax statistic, into given outputs

Layout: ``q [B,Hq,N,d_qk]``, ``k [B,Hkv,N,d_qk]``, ``v [B,Hkv,N,d_v]``, ``o [B,Hq,N,d_v]``; ``Hq`` is a multiple of ``Hkv`` and query head
``h`` attends with key head ``h // (Hq // Hkv)``.  ``seq_lens``: ``None`` or int32 ``[B]`` on the device, the tokens of each sequence of a
padded batch; rows behind a sequence's end take no part, whatever they hold, and their outputs and
gradients are zeros.

fp16 / bf16 with head dims up to 128 run on the tensor cores, fp32 with such head dims in tiles on the CUDA cores; both want rows of whole
16-byte units, so that other head dims are padded with zero columns and tensors in other layouts (expanded gradients,
misaligned views) are copied.  Head dims up to 256 run on the CUDA cores, a warp a row.  Sums and softmax statistics are fp32; the weights P and dS are rounded to
the type of the inputs before the second product.  Results do not depend on the order in which blocks finish.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from ._lib import native as _native

MAX_SINKS = 1024                    # SINK_MAX_SINKS of include/swa_sequence.h


def sink_swa_forward(q, k, v, window, n_sink, sm_scale, seq_lens=None, impl="auto", out=None):
    """No autograd graph (tangents and jit traces are refused).  Returns ``(o, lse)``, ``lse`` fp32 ``[B,Hq,N]`` in the base-2 domain (``-inf`` for rows behind a sequence's end).  ``out``: an
    optional ``[B,Hq,N,d_v]`` tensor or strided view that O is written into; it shares no memory with the inputs."""
    return _native.sink_forward(q, k, v, seq_lens, window, n_sink, sm_scale, _lib.impl_code(impl), out)


def sink_swa_backward(q, k, v, o, lse, do, window, n_sink, sm_scale, seq_lens=None, impl="auto", out=None):
    """Returns ``(dq, dk, dv)`` in the input dtype; ``out``: optional ``(dq, dk, dv)`` tensors or strided views to write
    into, which share no memory with one another or with the inputs."""
    return _native.sink_backward(q, k, v, o, lse, do, seq_lens, window, n_sink, sm_scale, _lib.impl_code(impl), *(out or (None,) * 3))


def sink_swa_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int, n_sink: int, sm_scale: float = 1.0,
                 seq_lens=None) -> torch.Tensor:
    """Forward only, no autograd graph."""
    return sink_swa_forward(q, k, v, window, n_sink, sm_scale, seq_lens)[0]


def sink_selected_impl(q, k, v, window, n_sink, sm_scale=1.0, impl="auto"):
    """'tc' or 'simt': the kernel family that runs these shapes as they are."""
    g = _lib.SinkGeom(_lib.dtype_code(q.dtype), q.shape[0], q.shape[1], k.shape[1], q.shape[2], q.shape[3], v.shape[3], window, n_sink,
                      float(sm_scale), _lib.impl_code(impl), None)
    code = _lib.lib.sink_swa_select(C.byref(g))
    if code < 0:
        _lib.check(code, "sink_swa_select")
    return {_lib.IMPL_SIMT: "simt", _lib.IMPL_TC: "tc"}[code]


class SinkSwa(torch.autograd.Function):
    """``SinkSwa.apply(q, k, v, seq_lens, window, n_sink, sm_scale)``.  ``apply`` runs natively; ``forward`` and ``backward`` are the
    general path (functorch, tracing), as in ``TiledSwa``.  Gradients of shared key heads are summed in a fixed order."""

    apply = staticmethod(_native.sink_swa)

    @staticmethod
    def forward(ctx, q, k, v, seq_lens, *win):
        o, lse = _native.sink_forward_body(q, k, v, seq_lens, *win, _lib.IMPL_AUTO, None)
        ctx.save_for_backward(q, k, v, lse, o, *(() if seq_lens is None else (seq_lens,)))
        ctx.win = win
        return o

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do):
        q, k, v, lse, o, *lens = ctx.saved_tensors
        return (*_native.sink_backward_body(q, k, v, o, lse, do, lens[0] if lens else None, *ctx.win, _lib.IMPL_AUTO, None, None, None), *(None,) * 4)
