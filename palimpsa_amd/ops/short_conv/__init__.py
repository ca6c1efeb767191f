"""The short causal convolution in front of the operators, as fused HIP kernels.

Both layers of the reference convolve the projections over time before they call an operator, one filter of a few taps per
channel, and keep the last inputs for generation: ``Palimpsa`` through ``fla.modules.ShortConvolution``
(palimpsa/layers/palimpsa.py:240-257), ``MetaMamba2`` through a ``conv1d`` over x, B and C together
(palimpsa/layers/meta_mamba2.py:264-279).  Neither module is part of the reference tree; their published behaviour is
restated here:

    p[t, c] = bias[c] + sum_i weight[c, W-1-i] * x[t-i, c]          y = p * sigmoid(p)   (activation "silu")  or  p

A state ``[N, D, W]`` in the type of the rows holds the last ``W`` inputs of each sequence, oldest first, which is what the
layers keep in their cache.

    y, state = short_conv(x, weight, bias, output_final_state=True)      # prompts, packed batches, training
    y = short_conv_step(x, state, weight, bias)                          # tokens of a generation; state in place
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from ... import _lib as L
from ..palimpsa import _common as cm

__all__ = ["short_conv", "short_conv_step", "ShortConv"]

MAX_WIDTH = 8


def _silu(activation: Optional[str]) -> int:
    if activation not in (None, "silu", "swish"):
        raise ValueError(f"activation must be None, 'silu' or 'swish', got {activation!r}")
    return 0 if activation is None else 1


def _filters(weight: torch.Tensor, bias: Optional[torch.Tensor], D: int):
    """(weight [D, W], bias, W) in one type that the kernels read."""
    if weight.dim() == 3 and weight.shape[1] == 1:     # nn.Conv1d's layout
        weight = weight.squeeze(1)
    if weight.dim() != 2 or weight.shape[0] != D:
        raise ValueError(f"weight must be [{D}, W] or [{D}, 1, W], got {tuple(weight.shape)}")
    W = weight.shape[1]
    if not 2 <= W <= MAX_WIDTH:
        raise ValueError(f"the convolution takes 2 to {MAX_WIDTH} taps, got {W}")
    if bias is not None and tuple(bias.shape) != (D,):
        raise ValueError(f"bias must be [{D}], got {tuple(bias.shape)}")
    if bias is not None and bias.dtype != weight.dtype:
        weight, bias = weight.float(), bias.float()
    return cm.param(weight), cm.param(bias), W


def _dims(B, T, N, D, W, chunks, cd, weight, silu, flags, x):
    xb, xt = cm.token_strides(x)
    return L.PalConvDims(batch=B, seq_len=T, n_seqs=N, channels=D, width=W, total_chunks=chunks, dtype=cm._pal_dtype(cd),
                         weight_dtype=cm._pal_dtype(weight.dtype), silu=silu, flags=flags, x_batch_stride=xb, x_token_stride=xt)


class ShortConv(torch.autograd.Function):
    """forward(ctx, x, weight, bias, silu, initial_state, output_final_state, cu_seqlens) -> (y, final_state | None).
    Gradients for x, weight, bias and initial_state; one that reaches the final state is taken."""

    @staticmethod
    def forward(ctx, x, weight, bias, silu, initial_state, output_final_state, cu_seqlens):
        dev = cm._require_gpu(x, weight, bias, initial_state)
        B, T, D = x.shape
        w, b, W = _filters(weight, bias, D)
        cd = torch.bfloat16 if x.dtype == torch.bfloat16 else torch.float32
        xc = cm.token_rows(x if x.dtype == cd else x.to(cd))
        cu = table = None
        N, chunks, flags = B, 0, 0
        if cu_seqlens is not None:
            cu, table, chunks, N = cm.packed_batch(cu_seqlens, B, T, dev)
            flags |= L.PAL_FLAG_VARLEN
        init = None
        if initial_state is not None:
            if tuple(initial_state.shape) != (N, D, W):
                raise ValueError(f"initial_state must be {(N, D, W)}, got {tuple(initial_state.shape)}")
            init = cm._plain(initial_state, cd)
            flags |= L.PAL_FLAG_HAS_INIT
        y = torch.empty(B, T, D, dtype=cd, device=dev)
        final = torch.empty(N, D, W, dtype=cd, device=dev) if output_final_state else None
        dims = _dims(B, T, N, D, W, chunks, cd, w, silu, flags | (L.PAL_FLAG_STORE_FINAL if output_final_state else 0), xc)
        pt = cm._ptr
        tens = L.PalConvTensors(x=pt(xc), weight=pt(w), bias=pt(b), y=pt(y), init=pt(init), final_=pt(final), cu_seqlens=pt(cu),
                                chunk_table=pt(table))
        with torch.cuda.device(dev):
            rc = L.load().pal_short_conv_fwd(dims, tens, cm.current_stream_ptr(dev))
        L.check(rc, "pal_short_conv_fwd")
        ctx.set_materialize_grads(False)
        if any(ctx.needs_input_grad):
            ctx.save_for_backward(xc, w, b, init, cu, table)
            ctx.meta = dict(N=N, W=W, chunks=chunks, cd=cd, silu=silu, flags=flags, wshape=tuple(weight.shape),
                            dtypes=[None if t is None else t.dtype for t in (x, weight, bias, initial_state)])
        if y.dtype != x.dtype:
            y = y.to(x.dtype)
        if final is not None and final.dtype != x.dtype:
            final = final.to(x.dtype)
        return y, final

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, d_final):
        x, w, b, init, cu, table = ctx.saved_tensors
        m = ctx.meta
        dev, cd = x.device, m["cd"]
        B, T, D = x.shape
        dy = torch.zeros(B, T, D, dtype=cd, device=dev) if dy is None else cm._plain(dy, cd)
        d_final = None if d_final is None else cm._plain(d_final, cd)
        dx = torch.empty(B, T, D, dtype=cd, device=dev)
        dw = torch.empty(D, m["W"], dtype=torch.float32, device=dev)
        db = None if b is None else torch.empty(D, dtype=torch.float32, device=dev)
        d_init = torch.empty_like(init) if init is not None and ctx.needs_input_grad[4] else None
        dims = _dims(B, T, m["N"], D, m["W"], m["chunks"], cd, w, m["silu"], m["flags"], x)
        pt = cm._ptr
        tens = L.PalConvTensors(x=pt(x), weight=pt(w), bias=pt(b), y=pt(dx), init=pt(init), cu_seqlens=pt(cu), chunk_table=pt(table))
        grads = L.PalConvGrads(dy=pt(dy), d_final=pt(d_final), dx=pt(dx), dweight=pt(dw), dbias=pt(db), d_init=pt(d_init))
        lib = L.load()
        ws_bytes = int(lib.pal_short_conv_bwd_workspace_bytes(dims))
        ws = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=dev)
        with torch.cuda.device(dev):
            rc = lib.pal_short_conv_bwd(dims, tens, grads, C.c_void_p(ws.data_ptr()), ws_bytes, cm.current_stream_ptr(dev))
        L.check(rc, "pal_short_conv_bwd")
        dt = m["dtypes"]
        return (dx.to(dt[0]), dw.reshape(m["wshape"]).to(dt[1]), None if db is None else db.to(dt[2]), None,
                None if d_init is None else d_init.to(dt[3]), None, None)


def short_conv(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: Optional[str] = "silu",
               initial_state: Optional[torch.Tensor] = None, output_final_state: bool = False,
               cu_seqlens: Optional[torch.Tensor] = None):
    """Causal convolution over time with one filter of ``W`` taps (2 to 8) per channel; returns ``(y, final_state | None)``.

    x ``[B, T, D]`` with at least one token (bf16, or computed in fp32); a slice of a wider projection is read where it is.
    weight ``[D, W]`` or ``[D, 1, W]``, the last tap meets the token itself; bias ``[D]``; ``activation`` "silu" (or "swish") or
    None.  ``initial_state`` ``[N, D, W]`` holds the ``W`` inputs before the first token, oldest first (the oldest meets no tap;
    it is there because layers keep it); final states have the same form and the type of x.  ``cu_seqlens`` ``[N + 1]`` makes x one
    packed row of N sequences, some of which may be empty: each starts from its own state, and an empty one hands its state on.
    Gradients for x, weight, bias and initial_state, through y and the final state."""
    if not torch.compiler.is_compiling() and x.is_cuda and x.dim() == 3 and activation in (None, "silu", "swish"):
        cu = table = None
        if cu_seqlens is not None:
            cu, table, _, _ = cm.packed_batch(cu_seqlens, x.shape[0], x.shape[1], x.device)
        r = L.host().short_conv(x, weight, bias, activation is not None, initial_state, output_final_state, cu, table)
        if r is not None:
            return r
    return _short_conv(x, weight, bias, activation, initial_state, output_final_state, cu_seqlens)


@cm.no_compile
def _short_conv(x, weight, bias, activation, initial_state, output_final_state, cu_seqlens):
    cm._require_gpu(x, weight, bias, initial_state)
    if x.dim() != 3:
        raise ValueError(f"x must be [B, T, D], got {tuple(x.shape)}")
    return ShortConv.apply(x, weight, bias, _silu(activation), initial_state, output_final_state, cu_seqlens)


def short_conv_step(x: torch.Tensor, state: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                    activation: Optional[str] = "silu") -> torch.Tensor:
    """The next token (x ``[B, D]``) or the next few (x ``[B, T, D]``) of ``B`` generations; returns y in the shape of x.

    ``state`` ``[B, D, W]``, packed and in the type of x (bf16 or fp32), is read and written in place.  Nothing but y is allocated,
    so a step can be recorded into a HIP graph.  No gradients: call it under ``torch.no_grad()``, or ``short_conv`` for training."""
    if not torch.compiler.is_compiling() and x.is_cuda and activation in (None, "silu", "swish"):
        r = L.host().short_conv_step(x, state, weight, bias, activation is not None)
        if r is not None:
            return r
    return _short_conv_step(x, state, weight, bias, activation)


@cm.no_compile
def _short_conv_step(x, state, weight, bias, activation):
    silu = _silu(activation)
    dev = cm._require_gpu(x, state, weight, bias)
    if x.dim() not in (2, 3):
        raise ValueError(f"x must be [B, D] or [B, T, D], got {tuple(x.shape)}")
    if cm.wants_grad(x, state, weight, bias):
        raise ValueError("short_conv_step writes its state in place and has no gradient: use short_conv, or torch.no_grad()")
    x3 = cm.token_rows(x.unsqueeze(1) if x.dim() == 2 else x)
    B, T, D = x3.shape
    w, b, W = _filters(weight, bias, D)
    if x.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"x must be bf16 or fp32, got {x.dtype}")
    if tuple(state.shape) != (B, D, W) or state.dtype != x.dtype or not state.is_contiguous():
        raise ValueError(f"state must be contiguous {x.dtype} {(B, D, W)}, got {state.dtype} {tuple(state.shape)}")
    y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    dims = _dims(B, T, B, D, W, 0, x.dtype, w, silu, 0, x3)
    pt = cm._ptr
    tens = L.PalConvTensors(x=pt(x3), weight=pt(w), bias=pt(b), y=pt(y), final_=pt(state))
    with torch.cuda.device(dev):
        rc = L.load().pal_short_conv_step(dims, tens, cm.current_stream_ptr(dev))
    L.check(rc, "pal_short_conv_step")
    cm.bump_version(state)
    return y
