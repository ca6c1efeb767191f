"""Gated feed-forward block, the second half of the reference's block (fla.modules.GatedMLP, restated from its published behaviour):
both projections, the activation and their product in one kernel, the projection back, and the gradients of all of them."""
from __future__ import annotations

import ctypes as C

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from ... import _lib as L
from ..layer_glue import _norm_rows
from ..palimpsa import _common as cm

__all__ = ["gated_mlp", "ACTIVATIONS", "MAX_DIM"]

ACTIVATIONS = tuple(L.PAL_ACT)
MAX_DIM = 1 << 20
MAX_ROWS = 1 << 30


def _up8(n: int) -> int:
    return cm._round_up(n, 8)


def _matrix(w: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """A weight as the kernels read it: of ``dtype``, packed, both dims multiples of eight (zeros behind), 16-byte aligned."""
    w = cm._plain(w, dtype)
    n, k = w.shape
    if n % 8 or k % 8:
        return F.pad(w, (0, _up8(k) - k, 0, _up8(n) - n))
    return w.clone() if w.data_ptr() % 16 else w


def _rows(x: torch.Tensor, dtype: torch.dtype):
    """x [.., D] as rows the kernels read, and the distance between them; D a multiple of eight, rows 16-byte aligned."""
    x, stride = _norm_rows(x, dtype)
    D = x.shape[-1]
    if D % 8:
        return F.pad(x, (0, _up8(D) - D)), _up8(D)
    if x.data_ptr() % 16 or stride % 8 or stride > MAX_DIM:
        x = x.contiguous() if not x.is_contiguous() else x.clone()
        return x, D
    return x, stride


def _check(x, w_gate, w_up, w_down, activation):
    if activation not in L.PAL_ACT:
        raise ValueError(f"activation must be one of {', '.join(ACTIVATIONS)}, got {activation!r}")
    if x.dim() < 1 or any(w.dim() != 2 for w in (w_gate, w_up, w_down)):
        raise ValueError("expected x [.., D], w_gate and w_up [F, D], w_down [D_out, F]")
    Fh, D = w_gate.shape
    if x.shape[-1] != D or w_up.shape != w_gate.shape or w_down.shape[1] != Fh:
        raise ValueError(f"expected x [.., D], w_gate and w_up [F, D], w_down [D_out, F]; got {tuple(x.shape)}, {tuple(w_gate.shape)}, "
                         f"{tuple(w_up.shape)}, {tuple(w_down.shape)}")
    if min(D, Fh, w_down.shape[0]) < 1 or max(D, Fh, w_down.shape[0]) > MAX_DIM:
        raise ValueError(f"dims must be between 1 and {MAX_DIM}, got D={D}, F={Fh}, D_out={w_down.shape[0]}")
    if x.numel() // D > MAX_ROWS:
        raise ValueError(f"up to {MAX_ROWS} rows are served, got {x.numel() // D}")


class GatedMlp(torch.autograd.Function):
    """forward(ctx, x, w_gate, w_up, w_down, activation) -> y."""

    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, activation):
        dev = cm._require_gpu(x, w_gate, w_up, w_down)
        _check(x, w_gate, w_up, w_down, activation)
        D, Fh, Do = x.shape[-1], w_gate.shape[0], w_down.shape[0]
        rows = x.numel() // D
        ctx.shapes = (x.shape, w_gate.shape, w_up.shape, w_down.shape)
        ctx.dtypes = [t.dtype for t in (x, w_gate, w_up, w_down)]
        if rows == 0:
            ctx.dims = None
            return x.new_empty(x.shape[:-1] + (Do,))
        cd = torch.bfloat16 if all(t.dtype == torch.bfloat16 for t in (x, w_gate, w_up, w_down)) else torch.float32
        xc, xs = _rows(x, cd)
        wg, wu, wd = (_matrix(w, cd) for w in (w_gate, w_up, w_down))
        dims = L.PalMlpDims(rows=rows, x_stride=xs, dim=_up8(D), hidden=_up8(Fh), out_dim=_up8(Do), dtype=cm._pal_dtype(cd),
                            activation=L.PAL_ACT[activation], hidden_pad=_up8(Fh) - Fh)
        y = torch.empty((rows, _up8(Do)), dtype=cd, device=dev)
        lib = L.load()
        kept = torch.empty(int(lib.pal_gated_mlp_kept_bytes(dims)), dtype=torch.uint8, device=dev) if any(ctx.needs_input_grad) else None
        pt = cm._ptr
        tens = L.PalMlpTensors(x=pt(xc), w_gate=pt(wg), w_up=pt(wu), w_down=pt(wd), y=pt(y), kept=pt(kept))
        ws_bytes = int(lib.pal_gated_mlp_fwd_workspace_bytes(dims, kept is not None))
        ws = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=dev)
        with torch.cuda.device(dev):
            rc = lib.pal_gated_mlp_fwd(dims, tens, C.c_void_p(ws.data_ptr()), ws_bytes, cm.current_stream_ptr(dev))
        L.check(rc, "pal_gated_mlp_fwd")
        if kept is not None:
            ctx.save_for_backward(xc, wg, wu, wd, kept)
            ctx.dims = dims
            ctx.form = cm.saved_form(xc, wg, wu, wd, kept)
        return cm.unpad_last(y, Do).reshape(x.shape[:-1] + (Do,)).to(x.dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        shapes, dtypes, need = ctx.shapes, ctx.dtypes, ctx.needs_input_grad
        if ctx.dims is None:
            return tuple(torch.zeros(s, dtype=t, device=dy.device) if n else None for s, t, n in zip(shapes, dtypes, need)) + (None,)
        saved = ctx.saved_tensors
        cm.check_saved(saved, ctx.form, "gated_mlp")
        dev, cd = saved[0].device, saved[0].dtype
        dims = L.PalMlpDims.from_buffer_copy(ctx.dims)
        xc, dims.x_stride = _rows(saved[0], cd)
        wg, wu, wd = (_matrix(w, cd) for w in saved[1:4])
        kept = saved[4].contiguous()
        d, _ = _rows(dy.reshape(dims.rows, shapes[3][0]).to(cd).contiguous(), cd)
        out = [torch.empty(s, dtype=cd, device=dev) if n else None
               for s, n in zip(((dims.rows, dims.dim), wg.shape, wu.shape, wd.shape), need)]
        pt = cm._ptr
        tens = L.PalMlpTensors(x=pt(xc), w_gate=pt(wg), w_up=pt(wu), w_down=pt(wd), kept=pt(kept))
        grads = L.PalMlpGrads(dy=pt(d), dx=pt(out[0]), dw_gate=pt(out[1]), dw_up=pt(out[2]), dw_down=pt(out[3]))
        lib = L.load()
        ws_bytes = int(lib.pal_gated_mlp_bwd_workspace_bytes(dims, grads))
        ws = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=dev)
        with torch.cuda.device(dev):
            rc = lib.pal_gated_mlp_bwd(dims, tens, grads, C.c_void_p(ws.data_ptr()), ws_bytes, cm.current_stream_ptr(dev))
        L.check(rc, "pal_gated_mlp_bwd")
        res = []
        for t, s, dt in zip(out, shapes, dtypes):
            if t is not None:
                t = cm.unpad_last(t, s[-1])
                t = (t if len(s) != 2 else t[:s[0]]).reshape(s).to(dt)
            res.append(t)
        return (*res, None)


def gated_mlp(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, activation: str = "silu") -> torch.Tensor:
    """``y = (act(x @ w_gate.T) * (x @ w_up.T)) @ w_down.T`` of rows x ``[.., D]`` and weights as ``torch.nn.Linear`` holds them: w_gate,
    w_up ``[F, D]``, w_down ``[D_out, F]``; returns y ``[.., D_out]`` in the type of x.  ``activation``: "silu" (the reference's), "gelu",
    "gelu_tanh" (its form by a tanh) or "relu".

    Gradients for x and the weights.  The product of the two projections is rounded once to the type of the rows between the kernels, and so
    are the gradients of the projections; sums are in fp32.  For the backward pass the two projections and their product are kept, six bytes per
    row and hidden entry of bf16 rows, twelve of fp32 rows.  Rows and weights all in bf16, or everything is computed from fp32, under autocast too
    (fp32 master weights beside bf16 rows: pass ``w.bfloat16()``, a sixth of the time).  Dims that are no multiple of eight, up to 2^20, are padded by
    a copy; up to 2^30 rows.  Calls of few rows are bound by the reading of the weights."""
    if not torch.compiler.is_compiling() and x.is_cuda and activation in L.PAL_ACT:
        r = L.host().gated_mlp(x, w_gate, w_up, w_down, L.PAL_ACT[activation])
        if r is not None:
            return r
    return _gated_mlp(x, w_gate, w_up, w_down, activation)


@cm.no_compile
def _gated_mlp(x, w_gate, w_up, w_down, activation):
    cm._require_gpu(x, w_gate, w_up, w_down)
    return GatedMlp.apply(x, w_gate, w_up, w_down, activation)
