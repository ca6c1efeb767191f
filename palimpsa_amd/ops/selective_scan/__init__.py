"""Selective scan: the recurrence of this family whose decay differs for every channel and state entry.

``simple_gla`` has one decay per head and token; here (Gu and Dao, "Mamba: Linear-Time Sequence Modeling with Selective State
Spaces", 2023) every channel ``d`` walks ``N`` state entries of its own:

    dt = softplus(delta + delta_bias)
    h[d, n] = exp(dt[d] * A[d, n]) * h[d, n] + dt[d] * u[d] * B[n]
    y[d] = (sum_n C[n] * h[d, n] + D[d] * u[d]) * z[d] * sigmoid(z[d])

It takes the output of ``short_conv`` and the projections as they are (slices of a wider projection are read in place), fuses
the softplus, the skip and the gate, and keeps its states ``[N_seqs, D, N]`` in fp32.

    y, state = selective_scan(u, delta, A, B, C, D, z, delta_bias, output_final_state=True)     # prompts, packed, training
    y = selective_scan_step(u, state, delta, A, B, C, D, z, delta_bias)                         # tokens of a generation, in place
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from ... import _lib as L
from ..palimpsa import _common as cm

__all__ = ["selective_scan", "selective_scan_step", "SelectiveScan"]

MAX_STATE = 64


def _check(u, delta, A, B, C_, D, z, delta_bias):
    """Shapes of a call on ``[B, T, ..]`` tensors; (channels, state entries, groups)."""
    ch = u.shape[-1]
    if A.dim() != 2 or A.shape[0] != ch:
        raise ValueError(f"A must be [{ch}, N], got {tuple(A.shape)}")
    N = A.shape[1]
    if not 1 <= N <= MAX_STATE:
        raise ValueError(f"the scan takes 1 to {MAX_STATE} state entries per channel, got {N}")
    for name, t in (("delta", delta), ("z", z)):
        if t is not None and t.shape != u.shape:
            raise ValueError(f"{name} must have the shape of u, {tuple(u.shape)}, got {tuple(t.shape)}")
    G = B.shape[-2] if B.dim() == 4 else 1
    lead = tuple(u.shape[:2])
    if B.dim() != 4 or tuple(B.shape) != lead + (G, N) or C_.shape != B.shape:
        raise ValueError(f"B and C must be {lead + (N,)} or {lead + ('G', N)}, got {tuple(B.shape)} and {tuple(C_.shape)}")
    if G < 1 or ch % G:
        raise ValueError(f"the {G} groups of B and C must divide the {ch} channels")
    for name, t in (("D", D), ("delta_bias", delta_bias)):
        if t is not None and tuple(t.shape) != (ch,):
            raise ValueError(f"{name} must be [{ch}], got {tuple(t.shape)}")
    return ch, N, G


def _dims(u, delta, z, B, C_, N, G, seqs, cd, softplus, flags):
    (ub, ut), (db, dt), (Bb, Bt), (Cb, Ct) = (cm.token_strides(u), cm.token_strides(delta), cm.token_strides(B, 2),
                                              cm.token_strides(C_, 2))
    zb, zt = cm.token_strides(z) if z is not None else (0, 0)
    return L.PalScanDims(batch=u.shape[0], seq_len=u.shape[1], n_seqs=seqs, channels=u.shape[2], state=N, groups=G,
                         dtype=cm._pal_dtype(cd), softplus=1 if softplus else 0, flags=flags, u_batch=ub, u_token=ut, delta_batch=db,
                         delta_token=dt, z_batch=zb, z_token=zt, B_batch=Bb, B_token=Bt, C_batch=Cb, C_token=Ct)


def _rows(t, inner):
    t = cm.token_rows(t, inner)
    return t if cm.token_strides(t, inner)[1] < 1 << 24 else t.contiguous()   # (the kernels' limit)


def _aligned(t):
    """t in fp32, packed, from a multiple of 16 bytes on (parameters and states are read in pieces of that size)."""
    if t is None:
        return None
    t = cm._plain(t, torch.float32)
    return t if t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


class SelectiveScan(torch.autograd.Function):
    """forward(ctx, u, delta, A, B, C, D, z, delta_bias, softplus, initial_state, output_final_state, cu_seqlens) -> (y, final | None)
    on ``pal_scan_fwd`` / ``pal_scan_bwd``; B, C ``[B, T, G, N]``.  Gradients for every tensor; one that reaches the final state is taken."""

    @staticmethod
    def forward(ctx, u, delta, A, B, C_, D, z, delta_bias, softplus, initial_state, output_final_state, cu_seqlens):
        dev = cm._require_gpu(u, delta, A, B, C_, D, z, delta_bias, initial_state)
        ch, N, G = _check(u, delta, A, B, C_, D, z, delta_bias)
        bt, T = u.shape[:2]
        cd = torch.bfloat16 if all(t is None or t.dtype == torch.bfloat16 for t in (u, delta, B, C_, z)) else torch.float32
        rows = lambda t, inner=1: None if t is None else _rows(t if t.dtype == cd else t.to(cd), inner)  # noqa: E731
        uc, dc, zc, Bc, Cc = rows(u), rows(delta), rows(z), rows(B, 2), rows(C_, 2)
        f32 = _aligned
        Ac, Dc, bc = f32(A), f32(D), f32(delta_bias)
        cu, seqs, flags = None, bt, 0
        if cu_seqlens is not None:
            cu, _, _, seqs = cm.packed_batch(cu_seqlens, bt, T, dev)
            flags |= L.PAL_FLAG_VARLEN
        init = None
        if initial_state is not None:
            if tuple(initial_state.shape) != (seqs, ch, N):
                raise ValueError(f"initial_state must be {(seqs, ch, N)}, got {tuple(initial_state.shape)}")
            init = f32(initial_state)
            flags |= L.PAL_FLAG_HAS_INIT
        y = torch.empty(bt, T, ch, dtype=cd, device=dev)
        final = torch.empty(seqs, ch, N, dtype=torch.float32, device=dev) if output_final_state else None
        dims = _dims(uc, dc, zc, Bc, Cc, N, G, seqs, cd, softplus, flags | (L.PAL_FLAG_STORE_FINAL if output_final_state else 0))
        lib = L.load()
        kept = None
        if any(ctx.needs_input_grad):
            kept = torch.empty(max(int(lib.pal_scan_checkpoint_bytes(dims)), 16), dtype=torch.uint8, device=dev)
        ws_bytes = int(lib.pal_scan_fwd_workspace_bytes(dims))
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
        pt = cm._ptr
        tens = L.PalScanTensors(u=pt(uc), delta=pt(dc), A=pt(Ac), B=pt(Bc), C=pt(Cc), D=pt(Dc), z=pt(zc), delta_bias=pt(bc), y=pt(y),
                                init=pt(init), final_=pt(final), cu_seqlens=pt(cu), checkpoints=pt(kept))
        with torch.cuda.device(dev):
            rc = lib.pal_scan_fwd(dims, tens, pt(ws), ws_bytes, cm.current_stream_ptr(dev))
        L.check(rc, "pal_scan_fwd")
        ctx.set_materialize_grads(False)
        if kept is not None:
            ctx.save_for_backward(uc, dc, Ac, Bc, Cc, Dc, zc, bc, init, cu, kept)
            ctx.meta = dict(N=N, G=G, seqs=seqs, cd=cd, softplus=softplus, flags=flags,
                            dtypes=[None if t is None else t.dtype for t in (u, delta, A, B, C_, D, z, delta_bias, initial_state)])
        return (y if y.dtype == u.dtype else y.to(u.dtype)), final

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, d_final):
        u, delta, A, B, C_, D, z, bias, init, cu, kept = ctx.saved_tensors
        m = ctx.meta
        dev, cd = u.device, m["cd"]
        dy = torch.zeros(u.shape, dtype=cd, device=dev) if dy is None else cm._plain(dy, cd)
        d_final = _aligned(d_final)
        like = lambda t: None if t is None else torch.empty(t.shape, dtype=t.dtype, device=dev)  # noqa: E731
        du, dd, dA, dB, dC, dD, dz, dbias = (like(t) for t in (u, delta, A, B, C_, D, z, bias))
        d_init = like(init) if init is not None and ctx.needs_input_grad[9] else None
        dims = _dims(u, delta, z, B, C_, m["N"], m["G"], m["seqs"], cd, m["softplus"], m["flags"])
        pt = cm._ptr
        tens = L.PalScanTensors(u=pt(u), delta=pt(delta), A=pt(A), B=pt(B), C=pt(C_), D=pt(D), z=pt(z), delta_bias=pt(bias),
                                init=pt(init), cu_seqlens=pt(cu), checkpoints=pt(kept))
        grads = L.PalScanGrads(dy=pt(dy), d_final=pt(d_final), du=pt(du), ddelta=pt(dd), dA=pt(dA), dB=pt(dB), dC=pt(dC), dD=pt(dD),
                               dz=pt(dz), ddelta_bias=pt(dbias), d_init=pt(d_init))
        lib = L.load()
        ws_bytes = int(lib.pal_scan_bwd_workspace_bytes(dims))
        ws = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=dev)
        with torch.cuda.device(dev):
            rc = lib.pal_scan_bwd(dims, tens, grads, C.c_void_p(ws.data_ptr()), ws_bytes, cm.current_stream_ptr(dev))
        L.check(rc, "pal_scan_bwd")
        back = lambda t, k: None if t is None else t if t.dtype == m["dtypes"][k] else t.to(m["dtypes"][k])  # noqa: E731
        return (back(du, 0), back(dd, 1), back(dA, 2), back(dB, 3), back(dC, 4), back(dD, 5), back(dz, 6), back(dbias, 7), None,
                back(d_init, 8), None, None)


def _grouped(t: torch.Tensor) -> torch.Tensor:
    return t.unsqueeze(-2) if t.dim() == 3 else t


def selective_scan(u: torch.Tensor, delta: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                   D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None, delta_bias: Optional[torch.Tensor] = None,
                   delta_softplus: bool = True, initial_state: Optional[torch.Tensor] = None, output_final_state: bool = False,
                   cu_seqlens: Optional[torch.Tensor] = None):
    """Selective scan over prompts and training batches; returns ``(y, final_state | None)``.

    u, delta, z ``[B, T, D]`` with at least one token, B, C ``[B, T, N]`` or, for ``G`` groups of channels, ``[B, T, G, N]`` (all
    bf16, or computed in fp32), slices of wider projections among them; A ``[D, N]`` (negative for a decay; up to 64 entries), D,
    delta_bias ``[D]`` and states ``[N_seqs, D, N]`` in fp32.  Without ``delta_softplus`` the time step is ``delta + delta_bias`` as
    it is.  ``cu_seqlens`` ``[N_seqs + 1]`` makes the batch one packed row of sequences, some of which may be empty: each starts
    from its own state, and an empty one hands its state on.  Gradients for every tensor, through y and the final state."""
    if not torch.compiler.is_compiling() and u.is_cuda and u.dim() == 3:
        cu = None
        if cu_seqlens is not None:
            cu, _, _, _ = cm.packed_batch(cu_seqlens, u.shape[0], u.shape[1], u.device)
        r = L.host().selective_scan(u, delta, A, B, C, D, z, delta_bias, bool(delta_softplus), initial_state, output_final_state, cu)
        if r is not None:
            return r
    return _selective_scan(u, delta, A, B, C, D, z, delta_bias, delta_softplus, initial_state, output_final_state, cu_seqlens)


@cm.no_compile
def _selective_scan(u, delta, A, B, C, D, z, delta_bias, delta_softplus, initial_state, output_final_state, cu_seqlens):
    cm._require_gpu(u, delta, A, B, C, D, z, delta_bias, initial_state)
    if u.dim() != 3:
        raise ValueError(f"u must be [B, T, D], got {tuple(u.shape)}")
    return SelectiveScan.apply(u, delta, A, _grouped(B), _grouped(C), D, z, delta_bias, bool(delta_softplus), initial_state,
                               output_final_state, cu_seqlens)


def selective_scan_step(u: torch.Tensor, state: torch.Tensor, delta: torch.Tensor, A: torch.Tensor, B: torch.Tensor,
                        C: torch.Tensor, D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None,
                        delta_bias: Optional[torch.Tensor] = None, delta_softplus: bool = True) -> torch.Tensor:
    """The next token (u, delta, z ``[B, D]``, B, C ``[B, N]`` or ``[B, G, N]``) or the next few (``[B, T, ..]``) of ``B``
    generations; returns y in the shape of u.

    ``state`` ``[B, D, N]`` fp32, packed, is read and written in place.  Of a few tokens nothing but y is allocated; a step
    can be recorded into a HIP graph.  No gradients: call it under ``torch.no_grad()``, or ``selective_scan`` for training."""
    if not torch.compiler.is_compiling() and u.is_cuda:
        r = L.host().selective_scan_step(u, state, delta, A, B, C, D, z, delta_bias, bool(delta_softplus))
        if r is not None:
            return r
    return _selective_scan_step(u, state, delta, A, B, C, D, z, delta_bias, delta_softplus)


@cm.no_compile
def _selective_scan_step(u, state, delta, A, B, C, D, z, delta_bias, delta_softplus):
    dev = cm._require_gpu(u, state, delta, A, B, C, D, z, delta_bias)
    if u.dim() not in (2, 3):
        raise ValueError(f"u must be [B, D] or [B, T, D], got {tuple(u.shape)}")
    if cm.wants_grad(u, state, delta, A, B, C, D, z, delta_bias):
        raise ValueError("selective_scan_step writes its state in place and has no gradient: use selective_scan, or torch.no_grad()")
    shape = u.shape
    if u.dim() == 2:
        u, delta, B, C = (t.unsqueeze(1) for t in (u, delta, B, C))
        z = None if z is None else z.unsqueeze(1)
    B, C = _grouped(B), _grouped(C)
    ch, N, G = _check(u, delta, A, B, C, D, z, delta_bias)
    bt = u.shape[0]
    if tuple(state.shape) != (bt, ch, N) or state.dtype != torch.float32 or not state.is_contiguous():
        raise ValueError(f"state must be contiguous fp32 {(bt, ch, N)}, got {state.dtype} {tuple(state.shape)}")
    if state.data_ptr() % 16:
        raise ValueError("state must start at a multiple of 16 bytes")
    cd = torch.bfloat16 if all(t is None or t.dtype == torch.bfloat16 for t in (u, delta, B, C, z)) else torch.float32
    dtype = u.dtype
    rows = lambda t, inner=1: None if t is None else _rows(t if t.dtype == cd else t.to(cd), inner)  # noqa: E731
    u, delta, z, B, C = rows(u), rows(delta), rows(z), rows(B, 2), rows(C, 2)
    f32 = _aligned
    A, D, delta_bias = f32(A), f32(D), f32(delta_bias)
    y = torch.empty(u.shape, dtype=cd, device=dev)
    dims = _dims(u, delta, z, B, C, N, G, bt, cd, delta_softplus, L.PAL_FLAG_HAS_INIT | L.PAL_FLAG_STORE_FINAL)
    lib = L.load()
    ws_bytes = int(lib.pal_scan_fwd_workspace_bytes(dims))
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
    pt = cm._ptr
    tens = L.PalScanTensors(u=pt(u), delta=pt(delta), A=pt(A), B=pt(B), C=pt(C), D=pt(D), z=pt(z), delta_bias=pt(delta_bias), y=pt(y),
                            init=pt(state), final_=pt(state))
    with torch.cuda.device(dev):
        rc = lib.pal_scan_fwd(dims, tens, pt(ws), ws_bytes, cm.current_stream_ptr(dev))
    L.check(rc, "pal_scan_fwd")
    cm.bump_version(state)
    return y.reshape(shape) if y.dtype == dtype else y.to(dtype).reshape(shape)
