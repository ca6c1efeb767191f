"""The element-wise work of the reference layer either side of the operator, as fused HIP kernels.

``Palimpsa.forward`` of the reference (palimpsa/layers/palimpsa.py) turns the projections into the
operator's inputs with about a dozen framework kernels (:266-279) and post-processes the operator's
output with a residual and a gated RMS norm (:337-343).  Here each side is one kernel forward and one
backward behind the C ABI (``pal_prologue_fwd/bwd``, ``pal_epilogue_fwd/bwd``):

    q, k, v, b, gt = palimpsa_inputs(q_raw, k_raw, x, dt_raw, dt_bias, bs_raw, b_raw, b_scale)
    o = chunk_palimpsa(q, k, v, b, gt, A, Ip, ...)
    y = palimpsa_output_norm(o, x, D, gate, weight, eps)

A maintainer of the reference would replace lines :266-279 and :337-343 of the layer by these two calls;
the projections, the short convolutions and ``o_proj`` stay as they are.  There is no CPU fallback.

The reference's other caller of the operator, ``MetaMamba2.forward`` (palimpsa/layers/meta_mamba2.py), wraps it
in different element-wise work (:283-299 before, :355-363 after); the same kernels serve it in a second form:

    v, b, dt = metamamba2_inputs(x, dt_raw, dt_bias, b_raw, b_scale, dt_limit)     # dt clamped, v = x dt, b = .. dt
    o = chunk_palimpsa(C, B, v, b, dt, A, Ip, scale=1.0, ...)                       # B, C rows as they are
    y = metamamba2_output_norm(o, x, D, gate, weight, eps)                          # gate first, norm over the token

Between two blocks stands a norm with the residual's addition (the pre-norm of the reference's blocks, ``fla.modules.RMSNorm`` called with
a residual; models/palimpsa/modeling_palimpsa.py:84-114), for training and, with rows in 8 bits, for serving:

    y, residual = residual_rms_norm(x, residual, weight, eps)
    q, scales, residual = residual_rms_norm_fp8(x, residual, weight, eps, group_size=128)   # y = q * scales, e4m3

Blocks with a layer norm in that place, and with a dropout of what is added to the stream, take

    y, residual = residual_layer_norm(x, residual, weight, bias, eps, dropout_p=0.1, seed=seed, site=layer)
    y = layer_norm(x, weight, bias, eps)
    x = dropout(x, 0.1, seed, site)
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from ... import _lib as L
from ..palimpsa import _common as cm

__all__ = ["palimpsa_inputs", "palimpsa_output_norm", "PalimpsaInputs", "PalimpsaOutputNorm",
           "metamamba2_inputs", "metamamba2_output_norm", "MetaMamba2Inputs", "MetaMamba2OutputNorm",
           "residual_rms_norm", "residual_rms_norm_fp8", "ResidualRmsNorm",
           "layer_norm", "residual_layer_norm", "LayerNorm", "dropout", "Dropout"]


def _rows_dtype(*tensors) -> torch.dtype:
    return torch.bfloat16 if all(t is None or t.dtype == torch.bfloat16 for t in tensors) else torch.float32


def _check_dims(dk: int, dv: int) -> None:
    for name, d in (("dk", dk), ("dv", dv)):
        if d % 8 or not 8 <= d <= 256:
            raise ValueError(f"{name} must be a multiple of 8 in [8, 256], got {d}")


def _glue_dims(tokens, H, Hqk, dk, dv, dtype, eps, dt_min=0.0, dt_max=0.0, norm_over_heads=False):
    return L.PalGlueDims(tokens=tokens, n_heads=H, n_qk_heads=Hqk, dk=dk, dv=dv, dtype=cm._pal_dtype(dtype), eps=float(eps),
                         dt_min=float(dt_min), dt_max=float(dt_max), norm_over_heads=1 if norm_over_heads else 0)


class PalimpsaInputs(torch.autograd.Function):
    """forward(ctx, q_raw, k_raw, x, dt_raw, dt_bias, bs_raw, b_raw, b_scale, eps) -> (q, k, v, b | None, gt)."""

    @staticmethod
    def forward(ctx, q_raw, k_raw, x, dt_raw, dt_bias, bs_raw, b_raw, b_scale, eps):
        dev = cm._require_gpu(q_raw, k_raw, x, dt_raw, dt_bias, bs_raw, b_raw, b_scale)
        if q_raw.shape != k_raw.shape or q_raw.shape[:-2] != x.shape[:-2]:
            raise ValueError("expected q_raw, k_raw [..., Hqk, dk] and x [..., H, dv] with the same leading dims")
        lead = tuple(x.shape[:-2])
        H, dv = x.shape[-2:]
        Hqk, dk = q_raw.shape[-2:]
        if H % Hqk:
            raise ValueError(f"the {H} value heads must be a multiple of the {Hqk} query/key heads")
        if tuple(dt_raw.shape) != lead + (H,) or tuple(bs_raw.shape) != lead + (H,):
            raise ValueError(f"dt_raw and bs_raw must be {lead + (H,)}")
        if (b_raw is None) != (b_scale is None):
            raise ValueError("b_raw and b_scale go together")
        if b_raw is not None and b_raw.shape != x.shape:
            raise ValueError("b_raw must have the shape of x")
        _check_dims(dk, dv)
        cd = _rows_dtype(q_raw, k_raw, x, dt_raw, bs_raw, b_raw)
        prep = lambda t: None if t is None else t.to(cd).contiguous()
        q_raw_c, k_raw_c, x_c, dt_c, bs_c, b_c = (prep(t) for t in (q_raw, k_raw, x, dt_raw, bs_raw, b_raw))
        bias = dt_bias.reshape(H).float().contiguous()
        bsc = None if b_scale is None else b_scale.reshape(H).float().contiguous()
        tokens = x_c.numel() // (H * dv)
        q = torch.empty(lead + (H, dk), dtype=cd, device=dev)
        k = torch.empty_like(q)
        v = torch.empty(lead + (H, dv), dtype=cd, device=dev)
        b = torch.empty_like(v) if b_raw is not None else None
        gt = torch.empty(lead + (H,), dtype=torch.float32, device=dev)
        dims = _glue_dims(tokens, H, Hqk, dk, dv, cd, eps)
        pt = cm._ptr
        tens = L.PalPrologueTensors(q_raw=pt(q_raw_c), k_raw=pt(k_raw_c), x=pt(x_c), dt_raw=pt(dt_c), bs_raw=pt(bs_c),
                                    b_raw=pt(b_c), dt_bias=pt(bias), b_scale=pt(bsc), q=pt(q), k=pt(k), v=pt(v), b=pt(b),
                                    gt=pt(gt))
        with torch.cuda.device(dev):
            rc = L.load().pal_prologue_fwd(dims, tens, cm.current_stream_ptr(dev))
        L.check(rc, "pal_prologue_fwd")
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(q_raw_c, k_raw_c, x_c, dt_c, bs_c, b_c, bias, bsc)
        ctx.meta = dict(tokens=tokens, H=H, Hqk=Hqk, dk=dk, dv=dv, cd=cd, eps=float(eps), lead=lead,
                        dtypes=[None if t is None else t.dtype for t in (q_raw, k_raw, x, dt_raw, dt_bias, bs_raw, b_raw, b_scale)],
                        bias_shape=tuple(dt_bias.shape), bscale_shape=None if b_scale is None else tuple(b_scale.shape))
        return q, k, v, b, gt

    @staticmethod
    def backward(ctx, dq, dk, dv, db, dgt):
        q_raw, k_raw, x, dt_raw, bs_raw, b_raw, bias, bsc = ctx.saved_tensors
        m = ctx.meta
        dev = x.device
        cd, lead, H, Hqk = m["cd"], m["lead"], m["H"], m["Hqk"]

        def grad_in(g, shape, dtype):
            if g is None:
                return torch.zeros(shape, dtype=dtype, device=dev)
            return g.to(dtype).contiguous()

        dq = grad_in(dq, lead + (H, m["dk"]), cd)
        dk = grad_in(dk, lead + (H, m["dk"]), cd)
        dv = grad_in(dv, lead + (H, m["dv"]), cd)
        db = grad_in(db, lead + (H, m["dv"]), cd) if b_raw is not None else None
        dgt = grad_in(dgt, lead + (H,), torch.float32)
        dq_raw, dk_raw, dx = torch.empty_like(q_raw), torch.empty_like(k_raw), torch.empty_like(x)
        db_raw = torch.empty_like(b_raw) if b_raw is not None else None
        ddt_raw, dbs_raw = torch.empty_like(dt_raw), torch.empty_like(bs_raw)
        ddt_bias = torch.empty(H, dtype=torch.float32, device=dev)
        db_scale = torch.empty(H, dtype=torch.float32, device=dev) if b_raw is not None else None
        dims = _glue_dims(m["tokens"], H, Hqk, m["dk"], m["dv"], cd, m["eps"])
        pt = cm._ptr
        tens = L.PalPrologueTensors(q_raw=pt(q_raw), k_raw=pt(k_raw), x=pt(x), dt_raw=pt(dt_raw), bs_raw=pt(bs_raw),
                                    b_raw=pt(b_raw), dt_bias=pt(bias), b_scale=pt(bsc), q=pt(dq), k=pt(dk), v=pt(dv),
                                    b=pt(db), gt=pt(dgt))   # outputs are not touched by the backward; any valid pointers
        grads = L.PalPrologueGrads(dq=pt(dq), dk=pt(dk), dv=pt(dv), db=pt(db), dgt=pt(dgt), dq_raw=pt(dq_raw),
                                   dk_raw=pt(dk_raw), dx=pt(dx), db_raw=pt(db_raw), ddt_raw=pt(ddt_raw), dbs_raw=pt(dbs_raw),
                                   ddt_bias=pt(ddt_bias), db_scale=pt(db_scale))
        lib = L.load()
        ws_bytes = int(lib.pal_prologue_bwd_workspace_bytes(dims))
        ws = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=dev)
        with torch.cuda.device(dev):
            rc = lib.pal_prologue_bwd(dims, tens, grads, C.c_void_p(ws.data_ptr()), ws_bytes, cm.current_stream_ptr(dev))
        L.check(rc, "pal_prologue_bwd")
        dt = m["dtypes"]
        return (dq_raw.to(dt[0]), dk_raw.to(dt[1]), dx.to(dt[2]), ddt_raw.to(dt[3]),
                ddt_bias.reshape(m["bias_shape"]).to(dt[4]), dbs_raw.to(dt[5]),
                None if db_raw is None else db_raw.to(dt[6]),
                None if db_scale is None else db_scale.reshape(m["bscale_shape"]).to(dt[7]), None)


class PalimpsaOutputNorm(torch.autograd.Function):
    """forward(ctx, o, x, D, gate, weight, eps) -> y = rmsnorm(o + x * D) * weight * gate * sigmoid(gate)."""

    @staticmethod
    def forward(ctx, o, x, D, gate, weight, eps):
        dev = cm._require_gpu(o, x, D, gate, weight)
        lead = tuple(o.shape[:-2])
        H, dv = o.shape[-2:]
        if (x is None) != (D is None):
            raise ValueError("x and D go together")
        for name, t in (("x", x), ("gate", gate)):
            if t is not None and t.shape != o.shape:
                raise ValueError(f"{name} must have the shape of o")
        if weight.numel() != dv:
            raise ValueError(f"weight must have {dv} entries")
        _check_dims(8, dv)
        cd = _rows_dtype(o, x, gate)
        prep = lambda t: None if t is None else t.to(cd).contiguous()
        o_c, x_c, g_c = prep(o), prep(x), prep(gate)
        Dc = None if D is None else D.reshape(H).float().contiguous()
        w = weight.reshape(dv).float().contiguous()
        tokens = o_c.numel() // (H * dv)
        y = torch.empty_like(o_c)
        rstd = torch.empty(lead + (H,), dtype=torch.float32, device=dev)
        dims = _glue_dims(tokens, H, H, 8, dv, cd, eps)
        pt = cm._ptr
        tens = L.PalEpilogueTensors(o=pt(o_c), x=pt(x_c), D=pt(Dc), gate=pt(g_c), weight=pt(w), y=pt(y), rstd=pt(rstd))
        with torch.cuda.device(dev):
            rc = L.load().pal_epilogue_fwd(dims, tens, cm.current_stream_ptr(dev))
        L.check(rc, "pal_epilogue_fwd")
        ctx.save_for_backward(o_c, x_c, Dc, g_c, w, rstd)
        ctx.meta = dict(tokens=tokens, H=H, dv=dv, cd=cd, eps=float(eps),
                        dtypes=[None if t is None else t.dtype for t in (o, x, D, gate, weight)],
                        D_shape=None if D is None else tuple(D.shape), w_shape=tuple(weight.shape))
        return y

    @staticmethod
    def backward(ctx, dy):
        o, x, D, gate, w, rstd = ctx.saved_tensors
        m = ctx.meta
        dev = o.device
        cd, H, dv = m["cd"], m["H"], m["dv"]
        dy = dy.to(cd).contiguous()
        d_o = torch.empty_like(o)
        dx = torch.empty_like(x) if x is not None else None
        dgate = torch.empty_like(gate) if gate is not None else None
        dD = torch.empty(H, dtype=torch.float32, device=dev) if x is not None else None
        dw = torch.empty(dv, dtype=torch.float32, device=dev)
        dims = _glue_dims(m["tokens"], H, H, 8, dv, cd, m["eps"])
        pt = cm._ptr
        tens = L.PalEpilogueTensors(o=pt(o), x=pt(x), D=pt(D), gate=pt(gate), weight=pt(w), y=pt(d_o), rstd=pt(rstd))
        grads = L.PalEpilogueGrads(dy=pt(dy), d_o=pt(d_o), dx=pt(dx), dgate=pt(dgate), dD=pt(dD), dweight=pt(dw))
        lib = L.load()
        ws_bytes = int(lib.pal_epilogue_bwd_workspace_bytes(dims))
        ws = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=dev)
        with torch.cuda.device(dev):
            rc = lib.pal_epilogue_bwd(dims, tens, grads, C.c_void_p(ws.data_ptr()), ws_bytes, cm.current_stream_ptr(dev))
        L.check(rc, "pal_epilogue_bwd")
        dt = m["dtypes"]
        return (d_o.to(dt[0]), None if dx is None else dx.to(dt[1]),
                None if dD is None else dD.reshape(m["D_shape"]).to(dt[2]),
                None if dgate is None else dgate.to(dt[3]), dw.reshape(m["w_shape"]).to(dt[4]), None)


class MetaMamba2Inputs(torch.autograd.Function):
    """forward(ctx, x, dt_raw, dt_bias, b_raw, b_scale, dt_min, dt_max) -> (v, b | None, dt)."""

    @staticmethod
    def forward(ctx, x, dt_raw, dt_bias, b_raw, b_scale, dt_min, dt_max):
        dev = cm._require_gpu(x, dt_raw, dt_bias, b_raw, b_scale)
        lead = tuple(x.shape[:-2])
        H, dv = x.shape[-2:]
        if tuple(dt_raw.shape) != lead + (H,):
            raise ValueError(f"dt_raw must be {lead + (H,)}")
        if (b_raw is None) != (b_scale is None):
            raise ValueError("b_raw and b_scale go together")
        if b_raw is not None and b_raw.shape != x.shape:
            raise ValueError("b_raw must have the shape of x")
        if not dt_min <= dt_max:
            raise ValueError(f"dt_limit must be an ordered pair, got ({dt_min}, {dt_max})")
        _check_dims(8, dv)
        cd = _rows_dtype(x, dt_raw, b_raw)
        prep = lambda t: None if t is None else t.to(cd).contiguous()
        x_c, dt_c, b_c = prep(x), prep(dt_raw), prep(b_raw)
        bias = dt_bias.reshape(H).float().contiguous()
        bsc = None if b_scale is None else b_scale.reshape(H).float().contiguous()
        tokens = x_c.numel() // (H * dv)
        v = torch.empty(lead + (H, dv), dtype=cd, device=dev)
        b = torch.empty_like(v) if b_raw is not None else None
        gt = torch.empty(lead + (H,), dtype=torch.float32, device=dev)
        dims = _glue_dims(tokens, H, H, 8, dv, cd, 0.0, dt_min, dt_max)
        pt = cm._ptr
        tens = L.PalPrologueTensors(x=pt(x_c), dt_raw=pt(dt_c), b_raw=pt(b_c), dt_bias=pt(bias), b_scale=pt(bsc),
                                    v=pt(v), b=pt(b), gt=pt(gt))
        with torch.cuda.device(dev):
            rc = L.load().pal_prologue_fwd(dims, tens, cm.current_stream_ptr(dev))
        L.check(rc, "pal_prologue_fwd")
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x_c, dt_c, b_c, bias, bsc)
        ctx.meta = dict(tokens=tokens, H=H, dv=dv, cd=cd, lead=lead, dt_min=float(dt_min), dt_max=float(dt_max),
                        dtypes=[None if t is None else t.dtype for t in (x, dt_raw, dt_bias, b_raw, b_scale)],
                        bias_shape=tuple(dt_bias.shape), bscale_shape=None if b_scale is None else tuple(b_scale.shape))
        return v, b, gt

    @staticmethod
    def backward(ctx, dv, db, dgt):
        x, dt_raw, b_raw, bias, bsc = ctx.saved_tensors
        m = ctx.meta
        dev = x.device
        cd, lead, H = m["cd"], m["lead"], m["H"]

        def grad_in(g, shape, dtype):
            if g is None:
                return torch.zeros(shape, dtype=dtype, device=dev)
            return g.to(dtype).contiguous()

        dv = grad_in(dv, lead + (H, m["dv"]), cd)
        db = grad_in(db, lead + (H, m["dv"]), cd) if b_raw is not None else None
        dgt = grad_in(dgt, lead + (H,), torch.float32)
        dx = torch.empty_like(x)
        db_raw = torch.empty_like(b_raw) if b_raw is not None else None
        ddt_raw = torch.empty_like(dt_raw)
        ddt_bias = torch.empty(H, dtype=torch.float32, device=dev)
        db_scale = torch.empty(H, dtype=torch.float32, device=dev) if b_raw is not None else None
        dims = _glue_dims(m["tokens"], H, H, 8, m["dv"], cd, 0.0, m["dt_min"], m["dt_max"])
        pt = cm._ptr
        tens = L.PalPrologueTensors(x=pt(x), dt_raw=pt(dt_raw), b_raw=pt(b_raw), dt_bias=pt(bias), b_scale=pt(bsc),
                                    v=pt(dv), b=pt(db), gt=pt(dgt))   # outputs are not touched by the backward
        grads = L.PalPrologueGrads(dv=pt(dv), db=pt(db), dgt=pt(dgt), dx=pt(dx), db_raw=pt(db_raw), ddt_raw=pt(ddt_raw),
                                   ddt_bias=pt(ddt_bias), db_scale=pt(db_scale))
        lib = L.load()
        ws_bytes = int(lib.pal_prologue_bwd_workspace_bytes(dims))
        ws = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=dev)
        with torch.cuda.device(dev):
            rc = lib.pal_prologue_bwd(dims, tens, grads, C.c_void_p(ws.data_ptr()), ws_bytes, cm.current_stream_ptr(dev))
        L.check(rc, "pal_prologue_bwd")
        dt = m["dtypes"]
        return (dx.to(dt[0]), ddt_raw.to(dt[1]), ddt_bias.reshape(m["bias_shape"]).to(dt[2]),
                None if db_raw is None else db_raw.to(dt[3]),
                None if db_scale is None else db_scale.reshape(m["bscale_shape"]).to(dt[4]), None, None)


class MetaMamba2OutputNorm(torch.autograd.Function):
    """forward(ctx, o, x, D, gate, weight, eps) -> y = rmsnorm over all heads of ((o + x * D) * gate * sigmoid(gate)) * weight."""

    @staticmethod
    def forward(ctx, o, x, D, gate, weight, eps):
        dev = cm._require_gpu(o, x, D, gate, weight)
        lead = tuple(o.shape[:-2])
        H, dv = o.shape[-2:]
        if (x is None) != (D is None):
            raise ValueError("x and D go together")
        for name, t in (("x", x), ("gate", gate)):
            if t is not None and tuple(t.shape) not in (tuple(o.shape), lead + (H * dv,)):
                raise ValueError(f"{name} must have the entries of o ({tuple(o.shape)} or {lead + (H * dv,)})")
        if weight.numel() != H * dv:
            raise ValueError(f"weight must have {H * dv} entries")
        if H * dv > 4096:
            raise ValueError(f"the norm over all heads serves up to 4096 entries per token, got {H * dv}")
        _check_dims(8, dv)
        cd = _rows_dtype(o, x, gate)
        prep = lambda t: None if t is None else t.to(cd).contiguous()
        o_c, x_c, g_c = prep(o), prep(x), prep(gate)
        Dc = None if D is None else D.reshape(H).float().contiguous()
        w = weight.reshape(H * dv).float().contiguous()
        tokens = o_c.numel() // (H * dv)
        y = torch.empty_like(o_c)
        rstd = torch.empty(lead, dtype=torch.float32, device=dev)
        dims = _glue_dims(tokens, H, H, 8, dv, cd, eps, norm_over_heads=True)
        pt = cm._ptr
        tens = L.PalEpilogueTensors(o=pt(o_c), x=pt(x_c), D=pt(Dc), gate=pt(g_c), weight=pt(w), y=pt(y), rstd=pt(rstd))
        with torch.cuda.device(dev):
            rc = L.load().pal_epilogue_fwd(dims, tens, cm.current_stream_ptr(dev))
        L.check(rc, "pal_epilogue_fwd")
        ctx.save_for_backward(o_c, x_c, Dc, g_c, w, rstd)
        ctx.meta = dict(tokens=tokens, H=H, dv=dv, cd=cd, eps=float(eps),
                        dtypes=[None if t is None else t.dtype for t in (o, x, D, gate, weight)],
                        shapes=[None if t is None else tuple(t.shape) for t in (o, x, D, gate, weight)])
        return y

    @staticmethod
    def backward(ctx, dy):
        o, x, D, gate, w, rstd = ctx.saved_tensors
        m = ctx.meta
        dev = o.device
        cd, H, dv = m["cd"], m["H"], m["dv"]
        dy = dy.to(cd).contiguous()
        d_o = torch.empty_like(o)
        dx = torch.empty_like(x) if x is not None else None
        dgate = torch.empty_like(gate) if gate is not None else None
        dD = torch.empty(H, dtype=torch.float32, device=dev) if x is not None else None
        dw = torch.empty(H * dv, dtype=torch.float32, device=dev)
        dims = _glue_dims(m["tokens"], H, H, 8, dv, cd, m["eps"], norm_over_heads=True)
        pt = cm._ptr
        tens = L.PalEpilogueTensors(o=pt(o), x=pt(x), D=pt(D), gate=pt(gate), weight=pt(w), y=pt(d_o), rstd=pt(rstd))
        grads = L.PalEpilogueGrads(dy=pt(dy), d_o=pt(d_o), dx=pt(dx), dgate=pt(dgate), dD=pt(dD), dweight=pt(dw))
        lib = L.load()
        ws_bytes = int(lib.pal_epilogue_bwd_workspace_bytes(dims))
        ws = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=dev)
        with torch.cuda.device(dev):
            rc = lib.pal_epilogue_bwd(dims, tens, grads, C.c_void_p(ws.data_ptr()), ws_bytes, cm.current_stream_ptr(dev))
        L.check(rc, "pal_epilogue_bwd")
        dt, sh = m["dtypes"], m["shapes"]
        return (d_o.to(dt[0]), None if dx is None else dx.reshape(sh[1]).to(dt[1]),
                None if dD is None else dD.reshape(sh[2]).to(dt[2]),
                None if dgate is None else dgate.reshape(sh[3]).to(dt[3]), dw.reshape(sh[4]).to(dt[4]), None)


MAX_NORM_ROW = 16384


def _norm_rows(x: torch.Tensor, dtype: torch.dtype):
    """x ``[.., D]`` in ``dtype`` with one distance between its rows, and that distance (a slice of a wider tensor stays where it is)."""
    x = x if x.dtype == dtype else x.to(dtype)
    D = x.shape[-1]
    if x.stride(-1) == 1 or D == 1:
        stride = None
        for d in range(x.dim() - 2, -1, -1):
            if x.shape[d] == 1:
                continue
            if stride is None:
                stride, span = x.stride(d), x.stride(d) * x.shape[d]
                if stride < D:
                    break
            elif x.stride(d) == span:
                span *= x.shape[d]
            else:
                break
        else:
            return x, D if stride is None else stride
    x = x.contiguous()
    return x, D


def _norm_call(x, residual, weight, eps, residual_in_fp32, group=None):
    """Checks a norm call and fills its structs: (dims, tensors, outputs) with everything that has to stay alive in ``outputs``."""
    dev = cm._require_gpu(x, residual, weight)
    if x.dim() < 1 or x.numel() == 0:
        raise ValueError(f"x must be [.., D] with at least one row, got {tuple(x.shape)}")
    D = x.shape[-1]
    if D > MAX_NORM_ROW:
        raise ValueError(f"the norm serves rows of up to {MAX_NORM_ROW} entries, got {D}")
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f"residual must have the shape of x, {tuple(x.shape)}, got {tuple(residual.shape)}")
    if tuple(weight.shape) != (D,):
        raise ValueError(f"weight must be [{D}], got {tuple(weight.shape)}")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    cd = _rows_dtype(x)
    rd = torch.float32 if residual_in_fp32 or _rows_dtype(x, residual) == torch.float32 else torch.bfloat16
    xc, xs = _norm_rows(x, cd)
    rc, rs = (None, D) if residual is None else _norm_rows(residual, rd)
    w = cm.param(weight)
    res_out = torch.empty(x.shape, dtype=rd, device=dev)
    dims = L.PalNormDims(rows=x.numel() // D, x_stride=xs, res_stride=rs, dim=D, dtype=cm._pal_dtype(cd), res_dtype=cm._pal_dtype(rd),
                         weight_dtype=cm._pal_dtype(w.dtype), group=group or 0, eps=float(eps))
    tens = L.PalNormTensors(x=cm._ptr(xc), residual=cm._ptr(rc), weight=cm._ptr(w), residual_out=cm._ptr(res_out))
    return dims, tens, (dev, cd, rd, xc, rc, w, res_out)


class ResidualRmsNorm(torch.autograd.Function):
    """forward(ctx, x, residual, weight, eps, residual_in_fp32) -> (y, residual_out): s = x + residual, y = rmsnorm(s) * weight."""

    @staticmethod
    def forward(ctx, x, residual, weight, eps, residual_in_fp32):
        dims, tens, (dev, cd, rd, xc, rc_, w, res_out) = _norm_call(x, residual, weight, eps, residual_in_fp32)
        y = torch.empty(x.shape, dtype=cd, device=dev)
        tens.y = y.data_ptr()
        with torch.cuda.device(dev):
            rc = L.load().pal_residual_norm_fwd(dims, tens, cm.current_stream_ptr(dev))
        L.check(rc, "pal_residual_norm_fwd")
        ctx.set_materialize_grads(False)
        if any(ctx.needs_input_grad):
            ctx.save_for_backward(res_out, w)
            ctx.dims = dims
            ctx.meta = dict(cd=cd, rd=rd, dtypes=[None if t is None else t.dtype for t in (x, residual, weight)])
        return (y if y.dtype == x.dtype else y.to(x.dtype)), res_out

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dres):
        res_out, w = ctx.saved_tensors
        m = ctx.meta
        dev, cd, rd = res_out.device, m["cd"], m["rd"]
        if dy is None and dres is None:
            return None, None, None, None, None
        dy = None if dy is None else cm._plain(dy, cd)
        dres = None if dres is None else cm._plain(dres, rd)
        dx = torch.empty(res_out.shape, dtype=cd, device=dev)
        d_res = dx if cd == rd else torch.empty(res_out.shape, dtype=rd, device=dev)
        dw = torch.empty(w.shape, dtype=torch.float32, device=dev)
        pt = cm._ptr
        tens = L.PalNormTensors(weight=pt(w), residual_out=pt(res_out))
        grads = L.PalNormGrads(dy=pt(dy), dresidual_out=pt(dres), dx=pt(dx), dresidual=None if cd == rd else pt(d_res), dweight=pt(dw))
        lib = L.load()
        ws_bytes = int(lib.pal_residual_norm_bwd_workspace_bytes(ctx.dims))
        ws = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=dev)
        with torch.cuda.device(dev):
            rc = lib.pal_residual_norm_bwd(ctx.dims, tens, grads, C.c_void_p(ws.data_ptr()), ws_bytes, cm.current_stream_ptr(dev))
        L.check(rc, "pal_residual_norm_bwd")
        dt = m["dtypes"]
        return dx.to(dt[0]), None if dt[1] is None else d_res.to(dt[1]), dw.to(dt[2]), None, None


def residual_rms_norm(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor, eps: float = 1e-5,
                      residual_in_fp32: bool = False):
    """``s = x + residual``, ``y = s * rsqrt(mean(s ** 2) + eps) * weight``; returns ``(y, s)``: the block's input and the residual
    stream to hand on.  x, residual ``[.., D]`` (D up to 16384, residual None for the first block), weight ``[D]``.

    y has the type of x; s is bf16 where x and residual are bf16 and ``residual_in_fp32`` is not set, else fp32 (bf16 rows beside an
    fp32 stream are the usual choice for deep models).  The norm is that of s as it is handed on.  Gradients for x, residual and weight."""
    if not torch.compiler.is_compiling() and x.is_cuda:
        r = L.host().residual_norm(x, residual, weight, eps, residual_in_fp32)
        if r is not None:
            return r
    return _residual_rms_norm(x, residual, weight, eps, residual_in_fp32)


@cm.no_compile
def _residual_rms_norm(x, residual, weight, eps, residual_in_fp32):
    cm._require_gpu(x, residual, weight)
    return ResidualRmsNorm.apply(x, residual, weight, eps, residual_in_fp32)


def residual_rms_norm_fp8(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor, eps: float = 1e-5,
                          group_size: Optional[int] = None, residual_in_fp32: bool = False):
    """``residual_rms_norm`` with y in 8 bits for a projection that takes such rows; returns ``(q, scales, s)`` with ``y = q * scales``:
    q ``[.., D]`` ``torch.float8_e4m3fn``, scales fp32 ``[.., D / group_size]``, one for each group of ``group_size`` entries (32, 64, 128
    or 256, a divisor of D), or ``[.., 1]``, one for the row (``group_size`` None).  A scale is the largest absolute y of its group (at least
    1e-12) over 448.  A row whose sum of squares is not a finite number has NaN scales.  No gradients: call it under ``torch.no_grad()``."""
    if not torch.compiler.is_compiling() and x.is_cuda and group_size in (None, 32, 64, 128, 256):
        r = L.host().residual_norm_fp8(x, residual, weight, eps, residual_in_fp32, group_size or 0)
        if r is not None:
            return r
    return _residual_rms_norm_fp8(x, residual, weight, eps, group_size, residual_in_fp32)


@cm.no_compile
def _residual_rms_norm_fp8(x, residual, weight, eps, group_size, residual_in_fp32):
    cm._require_gpu(x, residual, weight)
    if cm.wants_grad(x, residual, weight):
        raise ValueError("residual_rms_norm_fp8 has no gradient: use residual_rms_norm, or torch.no_grad()")
    D = x.shape[-1] if x.dim() else 0
    if group_size is not None and (group_size not in (32, 64, 128, 256) or D % group_size):
        raise ValueError(f"group_size must be 32, 64, 128 or 256 and divide the {D} entries of a row, or None; got {group_size}")
    dims, tens, (dev, _, _, xc, rc_, w, res_out) = _norm_call(x, residual, weight, eps, residual_in_fp32, group_size)
    q = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=dev)
    scales = torch.empty(x.shape[:-1] + (D // group_size if group_size else 1,), dtype=torch.float32, device=dev)
    tens.y, tens.scales = q.data_ptr(), scales.data_ptr()
    with torch.cuda.device(dev):
        rc = L.load().pal_residual_norm_fwd(dims, tens, cm.current_stream_ptr(dev))
    L.check(rc, "pal_residual_norm_fwd")
    return q, scales, res_out


def _seed(seed, site, dev):
    """(64 bits of the seed as a signed number, tensor | None, site) of a dropout."""
    if not isinstance(site, int) or not 0 <= site < 1 << 32:
        raise ValueError(f"site must be a whole number below 2^32, got {site!r}")
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1 or seed.device != dev:
            raise ValueError(f"a seed tensor must be one int64 number on {dev}, got {seed.dtype} {tuple(seed.shape)} on {seed.device}")
        return 0, seed, site
    if not isinstance(seed, int) or not -(1 << 63) <= seed < 1 << 64:
        raise ValueError(f"seed must be a whole number of 64 bits or an int64 tensor, got {seed!r}")
    return ((seed + (1 << 63)) % (1 << 64)) - (1 << 63), None, site


def _probability(p) -> float:
    p = float(p)
    if not 0.0 <= p < 1.0:
        raise ValueError(f"the probability of being dropped must be at least 0 and below 1, got {p}")
    return p


def _drop_struct(p, seed, seed_t, site):
    return L.PalDropout(p=p, seed=seed, seed_at=cm._ptr(seed_t), site=site)


class Dropout(torch.autograd.Function):
    """forward(ctx, x, p, seed, seed_t, site) -> y."""

    @staticmethod
    def _run(x, p, seed, seed_t, site):
        cd = _rows_dtype(x)
        y = torch.empty(x.shape, dtype=cd, device=x.device)
        if x.numel():
            xc, stride = _norm_rows(x if x.dim() else x.reshape(1), cd)
            D = xc.shape[-1]
            with torch.cuda.device(x.device):
                rc = L.load().pal_dropout(_drop_struct(p, seed, seed_t, site), cm._ptr(xc), cm._ptr(y), x.numel() // D, D, stride,
                                          cm._pal_dtype(cd), cm.current_stream_ptr(x.device))
            L.check(rc, "pal_dropout")
        return y if y.dtype == x.dtype else y.to(x.dtype)

    @staticmethod
    def forward(ctx, x, p, seed, seed_t, site):
        ctx.meta = (p, seed, site)
        ctx.save_for_backward(seed_t)
        ctx.form = cm.saved_form(seed_t)
        return Dropout._run(x, p, seed, seed_t, site)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        p, seed, site = ctx.meta
        saved = ctx.saved_tensors
        cm.check_saved(saved, ctx.form, "dropout")
        return Dropout._run(dy, p, seed, saved[0], site), None, None, None, None


def dropout(x: torch.Tensor, p: float, seed, site: int = 0) -> torch.Tensor:
    """Entries of x ``[.., D]`` are zero with probability p (0 <= p < 1), the others are multiplied by ``1 / (1 - p)``.

    Which ones is a function of the seed (a whole number of 64 bits, or an int64 tensor of one element on the device, which a captured graph
    reads at every replay) and of the entry's row and column alone: word ``column % 4`` of Philox4x32 with seven rounds of the counter
    ``(column // 4, row, row >> 32, site)`` under the key ``seed``, kept where it is not below ``p * 2 ** 32``.  So nothing is stored for
    the backward pass, the strides of x and the order of the work change nothing, and ``site`` numbers the places of a model that share a
    step's seed.  A dropped entry is zero whatever it held.  A seed tensor must not be changed between the forward and the backward pass."""
    if not torch.compiler.is_compiling() and x.is_cuda and isinstance(p, float) and 0.0 <= p < 1.0:
        bits, seed_t, site = _seed(seed, site, x.device)
        r = L.host().dropout(x, p, bits, seed_t, site)
        if r is not None:
            return r
    return _dropout(x, p, seed, site)


@cm.no_compile
def _dropout(x, p, seed, site):
    cm._require_gpu(x)
    return Dropout.apply(x, _probability(p), *_seed(seed, site, x.device))


class LayerNorm(torch.autograd.Function):
    """forward(ctx, x, residual, weight, bias, eps, residual_in_fp32, handed_on, p, seed, seed_t, site) -> y, or (y, s) where the
    stream is handed on."""

    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps, residual_in_fp32, handed_on, p, seed, seed_t, site):
        dev = cm._require_gpu(x, residual, weight, bias)
        if x.dim() < 1 or x.numel() == 0:
            raise ValueError(f"x must be [.., D] with at least one row, got {tuple(x.shape)}")
        D = x.shape[-1]
        if D > MAX_NORM_ROW:
            raise ValueError(f"the norm serves rows of up to {MAX_NORM_ROW} entries, got {D}")
        if residual is not None and residual.shape != x.shape:
            raise ValueError(f"residual must have the shape of x, {tuple(x.shape)}, got {tuple(residual.shape)}")
        if tuple(weight.shape) != (D,) or (bias is not None and tuple(bias.shape) != (D,)):
            raise ValueError(f"weight and bias must be [{D}], got {tuple(weight.shape)} and {None if bias is None else tuple(bias.shape)}")
        if not eps >= 0:
            raise ValueError(f"eps must not be negative, got {eps}")
        cd = _rows_dtype(x)
        rd = cd
        if handed_on and (residual_in_fp32 or _rows_dtype(x, residual) == torch.float32):
            rd = torch.float32
        xc, xs = _norm_rows(x, cd)
        rc_, rs = (None, D) if residual is None else _norm_rows(residual, rd)
        w, b = cm.param(weight), cm.param(bias)
        if b is not None and b.dtype != w.dtype:
            w, b = w.float(), b.float()
        y = torch.empty(x.shape, dtype=cd, device=dev)
        s = torch.empty(x.shape, dtype=rd, device=dev) if handed_on else None
        rows = x.numel() // D
        stats = torch.empty((rows, 2), dtype=torch.float32, device=dev) if any(ctx.needs_input_grad) else None
        pt = cm._ptr
        dims = L.PalLayerNormDims(rows=rows, x_stride=xs, res_stride=rs, dim=D, dtype=cm._pal_dtype(cd), res_dtype=cm._pal_dtype(rd),
                                  weight_dtype=cm._pal_dtype(w.dtype), eps=float(eps), drop=_drop_struct(p, seed, seed_t, site))
        tens = L.PalLayerNormTensors(x=pt(xc), residual=pt(rc_), weight=pt(w), bias=pt(b), residual_out=pt(s), y=pt(y), stats=pt(stats))
        with torch.cuda.device(dev):
            rc = L.load().pal_layer_norm_fwd(dims, tens, cm.current_stream_ptr(dev))
        L.check(rc, "pal_layer_norm_fwd")
        ctx.set_materialize_grads(False)
        if stats is not None:
            ctx.save_for_backward(s if handed_on else xc, w, stats, seed_t)
            ctx.form = cm.saved_form(s if handed_on else xc, w, stats, seed_t)
            ctx.meta = dict(cd=cd, rd=rd, handed_on=handed_on, dims=dims, drop=(p, seed, site),
                            dtypes=[None if t is None else t.dtype for t in (x, residual, weight, bias)])
        y = y if y.dtype == x.dtype else y.to(x.dtype)
        return (y, s) if handed_on else y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dres=None):
        rows, w, stats, seed_t = saved = ctx.saved_tensors
        cm.check_saved(saved, ctx.form, "layer_norm")
        m = ctx.meta
        w, stats = w.contiguous(), stats.contiguous()
        rows, stride = _norm_rows(rows.contiguous() if m["handed_on"] else rows, rows.dtype)
        dev, cd, rd, dt = rows.device, m["cd"], m["rd"], m["dtypes"]
        if dy is None and dres is None:
            return (None,) * 11
        dy = None if dy is None else cm._plain(dy, cd)
        dres = None if dres is None else cm._plain(dres, rd)
        dx = torch.empty(rows.shape, dtype=cd, device=dev)
        p, seed, site = m["drop"]
        apart = dt[1] is not None and (p > 0.0 or cd != rd)
        ds = torch.empty(rows.shape, dtype=rd, device=dev) if apart else None
        dw = torch.empty(w.shape, dtype=torch.float32, device=dev)
        db = None if dt[3] is None else torch.empty_like(dw)
        pt = cm._ptr
        dims = L.PalLayerNormDims.from_buffer_copy(m["dims"])
        dims.drop = _drop_struct(p, seed, seed_t, site)
        dims.x_stride = stride
        tens = L.PalLayerNormTensors(weight=pt(w), bias=pt(w) if db is not None else None, stats=pt(stats),
                                     **{"residual_out" if m["handed_on"] else "x": pt(rows)})
        grads = L.PalLayerNormGrads(dy=pt(dy), dresidual_out=pt(dres), dx=pt(dx), dresidual=pt(ds), dweight=pt(dw), dbias=pt(db))
        lib = L.load()
        ws_bytes = int(lib.pal_layer_norm_bwd_workspace_bytes(dims))
        ws = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=dev)
        with torch.cuda.device(dev):
            rc = lib.pal_layer_norm_bwd(dims, tens, grads, C.c_void_p(ws.data_ptr()), ws_bytes, cm.current_stream_ptr(dev))
        L.check(rc, "pal_layer_norm_bwd")
        d_res = None if dt[1] is None else (ds if apart else dx).to(dt[1])
        return (dx.to(dt[0]), d_res, dw.to(dt[2]), None if db is None else db.to(dt[3])) + (None,) * 7


def layer_norm(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean(x)) * rsqrt(var(x) + eps) * weight + bias`` over the last dim of x ``[.., D]`` (D up to 16384; var the mean square around
    the mean); weight, bias ``[D]`` in fp32 or bf16.  y has the type of x.  Gradients for x, weight and bias."""
    if not torch.compiler.is_compiling() and x.is_cuda:
        r = L.host().layer_norm(x, None, weight, bias, eps, False, False, 0.0, 0, None, 0)
        if r is not None:
            return r[0]
    return _layer_norm(x, None, weight, bias, eps, False, False, 0.0, 0, None, 0)


@cm.no_compile
def _layer_norm(x, residual, weight, bias, *rest):
    cm._require_gpu(x, residual, weight, bias)
    return LayerNorm.apply(x, residual, weight, bias, *rest)


def residual_layer_norm(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                        eps: float = 1e-5, residual_in_fp32: bool = False, dropout_p: float = 0.0, seed=None, site: int = 0):
    """``s = dropout(x) + residual``, ``y = layer_norm(s)``; returns ``(y, s)``: the block's input and the residual stream to hand on, as
    ``residual_rms_norm`` does (types, rows and the missing residual of a first block are as there), with the bias of a layer norm and the
    dropout of ``dropout(x, dropout_p, seed, site)`` in the same pass.  The norm is that of s as it is handed on.  Gradients for x, residual,
    weight and bias."""
    p = _probability(dropout_p)
    bits, seed_t = 0, None
    if p > 0.0:
        if seed is None:
            raise ValueError("a dropout needs a seed")
        bits, seed_t, site = _seed(seed, site, x.device)
    if not torch.compiler.is_compiling() and x.is_cuda:
        r = L.host().layer_norm(x, residual, weight, bias, eps, residual_in_fp32, True, p, bits, seed_t, site)
        if r is not None:
            return r
    return _layer_norm(x, residual, weight, bias, eps, residual_in_fp32, True, p, bits, seed_t, site)


@cm.no_compile
def palimpsa_inputs(q_raw: torch.Tensor, k_raw: torch.Tensor, x: torch.Tensor, dt_raw: torch.Tensor,
                    dt_bias: torch.Tensor, bs_raw: torch.Tensor, b_raw: Optional[torch.Tensor] = None,
                    b_scale: Optional[torch.Tensor] = None, eps: float = 1e-12):
    """Operator inputs from the layer's projections (layers/palimpsa.py:266-279 of the reference).

    q_raw, k_raw ``[..., Hqk, dk]`` and x ``[..., H, dv]`` are the (convolved, activated) q/k/v projections
    split into heads; dt_raw, bs_raw ``[..., H]`` the outputs of ``dt_proj`` / ``bs_proj``; b_raw ``[..., H, dv]``
    the output of ``b_proj`` (None with metaplasticity off).  Returns ``(q, k, v, b | None, gt)``: q, k
    L2-normalised with their heads repeated ``H / Hqk`` times, ``v = x * bs``, ``b = sigmoid(b_raw) *
    softplus(b_scale) * bs`` with ``bs = sigmoid(bs_raw)`` rounded to the row dtype, and
    ``gt = softplus(dt_raw + dt_bias)`` in fp32."""
    return PalimpsaInputs.apply(q_raw, k_raw, x, dt_raw, dt_bias, bs_raw, b_raw, b_scale, eps)


@cm.no_compile
def palimpsa_output_norm(o: torch.Tensor, x: Optional[torch.Tensor], D: Optional[torch.Tensor],
                         gate: Optional[torch.Tensor], weight: torch.Tensor, eps: float = 1e-5) -> torch.Tensor:
    """Residual and output norm of the layer (layers/palimpsa.py:337-343): ``rmsnorm(o + x * D) * weight``,
    times ``gate * sigmoid(gate)`` when a gate is given; o, x, gate ``[..., H, dv]``, D ``[H]``, weight ``[dv]``."""
    return PalimpsaOutputNorm.apply(o, x, D, gate, weight, eps)


@cm.no_compile
def metamamba2_inputs(x: torch.Tensor, dt_raw: torch.Tensor, dt_bias: torch.Tensor, b_raw: Optional[torch.Tensor] = None,
                      b_scale: Optional[torch.Tensor] = None, dt_limit=(0.0, float("inf"))):
    """Operator inputs of ``MetaMamba2.forward`` from its projections (layers/meta_mamba2.py:283-299 of the reference).

    x ``[..., H, dv]`` is the convolved value stream split into heads, dt_raw ``[..., H]`` the time-step columns of
    ``in_proj``, b_raw ``[..., H, dv]`` the output of ``b_proj`` (None with metaplasticity off).  Returns
    ``(v, b | None, dt)``: ``dt = clamp(softplus(dt_raw + dt_bias), *dt_limit)`` in fp32 (the operator's ``gt``),
    ``v = x * dt`` and ``b = sigmoid(b_raw) * softplus(b_scale) * dt`` in the row dtype.  The layer's ``B`` and ``C``
    rows go to the operator as they are (``k = B``, ``q = C``; fewer heads than ``H`` are shared inside the kernels)."""
    return MetaMamba2Inputs.apply(x, dt_raw, dt_bias, b_raw, b_scale, float(dt_limit[0]), float(dt_limit[1]))


@cm.no_compile
def metamamba2_output_norm(o: torch.Tensor, x: Optional[torch.Tensor], D: Optional[torch.Tensor],
                           gate: Optional[torch.Tensor], weight: torch.Tensor, eps: float = 1e-5) -> torch.Tensor:
    """Residual, gate and output norm of ``MetaMamba2.forward`` (layers/meta_mamba2.py:355-363):
    ``rmsnorm((o + x * D) * gate * sigmoid(gate)) * weight`` with the mean square taken over all ``H * dv`` entries of a
    token (``RMSNormGated(intermediate_size, norm_before_gate=False)``); o ``[..., H, dv]``, x and gate with the same
    entries (``[..., H, dv]`` or ``[..., H * dv]``), D ``[H]``, weight ``[H * dv]``.  Returns ``[..., H, dv]``."""
    return MetaMamba2OutputNorm.apply(o, x, D, gate, weight, eps)
