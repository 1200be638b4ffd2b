"""Torch-facing operators over the C ABI (libgdn_b200.so).

Two surfaces:

* functional ops (``prefill``, ``decode_step``, ``rmsnorm``, ``gated_rmsnorm``,
  ``proj_conv_silu``) taking torch CUDA tensors, shape-generic, launching on
  ``torch.cuda.current_stream()``;
* drop-in module objects with the reference's operator surface -- the
  ``exts`` dict consumed by ``gdn_layer.GDNLayerCustom`` (gdn_layer.py:206-217):
  ``exts()['prefill'].prefill(...)`` (kernels/prefill_chunked.cu:512-526),
  ``['decode'].forward(...)`` (kernels/decode.cu:172-218),
  ``['proj'].forward(...)`` (kernels/fused_proj_conv_silu.cu:298-360),
  ``['rmsnorm'].forward(...)`` (kernels/rmsnorm.cu:280-298).

torch is only the allocator / stream provider here; all arithmetic runs in
the sm_100a kernels of the library.
"""
from __future__ import annotations

import ctypes
import functools
import math

import torch

from . import _lib
from ._lib import (GDN_DTYPE_BF16, GDN_DTYPE_F32, GDN_LAYOUT_BHTD, GDN_LAYOUT_BTHD)

CHUNK = 64


def _stream() -> int:
    # the current stream of the current device as a handle, without building a Stream object
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def _ptr(t):
    return None if t is None else t.data_ptr()


def _gate_dtype(t: torch.Tensor, name: str) -> int:
    if t.dtype == torch.bfloat16:
        return GDN_DTYPE_BF16
    if t.dtype == torch.float32:
        return GDN_DTYPE_F32
    raise RuntimeError(f"{name}: gate tensors must be bfloat16 or float32, got {t.dtype}")


def _need(cond: bool, msg: str) -> None:
    if not cond:
        raise RuntimeError(msg)


def _cuda_contig(t: torch.Tensor, name: str, dtype=None) -> None:
    _need(t.is_cuda, f"{name} must be a CUDA tensor")
    _need(t.is_contiguous(), f"{name} must be contiguous")
    if dtype is not None:
        _need(t.dtype == dtype, f"{name} must be {dtype}, got {t.dtype}")


# ---------------------------------------------------------------------------
# functional ops
# ---------------------------------------------------------------------------


_SCHEDULES = {None: 0, "auto": 0, "single": 1, "pieced": 2, "stream": 3}


def prefill(q, k, v, A_log, a, b_logits, *, dt_bias=0.0, mask=None, state_in=None,
            scale=0.0, layout="bhtd", out=None, state_out=None, return_state=True, gates="bht", schedule=None):
    """Chunked gated-delta-rule prefill (reference/prefill_ref.py semantics).

    layout "bhtd": q,k [B,Hqk,T,dk], v [B,Hv,T,dv]; "bthd": q,k [B,T,Hqk,dk], v [B,T,Hv,dv].
    a, b_logits [B,Hv,T] (bf16 or f32), or with gates="bth" [B,T,Hv] views whose
    token rows share one stride (read in place, e.g. the halves of a [B,T,2Hv]
    projection); A_log [Hv] f32; dt_bias float or f32 [Hv]; mask [B,T] f32 or None;
    state_in [B,Hv,dk,dv] f32 or None; schedule None/"auto", "single", "pieced" or
    "stream" for this call (gdn_prefill_fwd_ex).
    Returns (out bf16 in v's layout, state_out f32 [B,Hv,dk,dv] or None).
    """
    _need(gates in ("bht", "bth"), f"gates must be 'bht' or 'bth', got {gates!r}")
    _need(schedule in _SCHEDULES, f"schedule must be one of {sorted(k_ for k_ in _SCHEDULES if k_)}, got {schedule!r}")
    lay, B, T, Hqk, Hv, dk, dv, gdt, dt_scalar, dt_vec = _prefill_checks(q, k, v, A_log, a, b_logits, dt_bias, mask,
                                                                         state_in, layout, gates)
    if out is None:
        out = torch.empty_like(v)
    if state_out is None and return_state:
        state_out = torch.empty(B, Hv, dk, dv, dtype=torch.float32, device=q.device)
    ws_bytes = _lib.lib().gdn_prefill_workspace_bytes(B, T, Hv, dk, dv)
    ws = torch.empty(max(int(ws_bytes), 1), dtype=torch.uint8, device=q.device)
    opts = _lib.PrefillOpts(_SCHEDULES[schedule], _lib.GDN_GATES_BTH if gates == "bth" else _lib.GDN_GATES_BHT,
                            a.stride(1) if gates == "bth" else 0)
    _lib.call("gdn_prefill_fwd_ex", _ptr(q), _ptr(k), _ptr(v), _ptr(A_log), _ptr(a), _ptr(b_logits), gdt,
              dt_scalar, _ptr(dt_vec), _ptr(mask), _ptr(state_in), _ptr(out), _ptr(state_out),
              B, T, Hqk, Hv, dk, dv, lay, float(scale), ctypes.byref(opts), _ptr(ws), int(ws_bytes), _stream())
    return out, state_out


def prefill_window(q, k, v, A_log, a, b_logits, t0, Tw, *, out, dt_bias=0.0, mask=None, state_in=None,
                   state_out=None, scale=0.0, layout="bhtd", workspace=None):
    """``prefill`` over the tokens [t0, t0 + Tw) of the given (whole) tensors
    (gdn_prefill_window_ws): reads the window's q, k, v, gates and mask in place
    and writes its o into the same tokens of ``out``; ``state_in`` is the state
    before token t0, ``state_out`` the state after the window.  ``workspace``: a
    uint8 CUDA tensor of at least gdn_prefill_workspace_bytes(B, Tw, Hv, dk, dv)
    bytes (allocated per call if None)."""
    lay, B, T, Hqk, Hv, dk, dv, gdt, dt_scalar, dt_vec = _prefill_checks(q, k, v, A_log, a, b_logits, dt_bias, mask,
                                                                         state_in, layout)
    _cuda_contig(out, "out", torch.bfloat16)
    _need(tuple(out.shape) == tuple(v.shape), "out must have v's shape")
    if state_out is not None:
        _cuda_contig(state_out, "state_out", torch.float32)
    ws_bytes = int(_lib.lib().gdn_prefill_workspace_bytes(B, max(int(Tw), 1), Hv, dk, dv))
    if workspace is None:
        workspace = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=q.device)
    _need(workspace.is_cuda and workspace.dtype == torch.uint8 and workspace.numel() >= ws_bytes,
          f"workspace: uint8 CUDA tensor of at least {ws_bytes} bytes required")
    _lib.call("gdn_prefill_window_ws", _ptr(q), _ptr(k), _ptr(v), _ptr(A_log), _ptr(a), _ptr(b_logits), gdt,
              dt_scalar, _ptr(dt_vec), _ptr(mask), _ptr(state_in), _ptr(out), _ptr(state_out),
              B, T, int(t0), int(Tw), Hqk, Hv, dk, dv, lay, float(scale), _ptr(workspace), workspace.numel(),
              _stream())
    return out, state_out


def _prefill_checks(q, k, v, A_log, a, b_logits, dt_bias, mask, state_in, layout, gates="bht"):
    """Shape, dtype and device checks shared by the prefill wrappers; returns
    (layout code, B, T, Hqk, Hv, dk, dv, gate dtype code, dt_bias scalar, dt_bias vector).
    ``gates`` "bht": a, b_logits contiguous [B, Hv, T]; "bth": [B, T, Hv] views whose
    tokens are rows of one stride (e.g. the halves of a [B, T, 2 Hv] projection)."""
    lay = GDN_LAYOUT_BHTD if layout == "bhtd" else GDN_LAYOUT_BTHD
    for name, t in (("q", q), ("k", k), ("v", v)):
        _cuda_contig(t, name, torch.bfloat16)
    if lay == GDN_LAYOUT_BHTD:
        B, Hqk, T, dk = q.shape
        Hv, dv = v.shape[1], v.shape[3]
    else:
        B, T, Hqk, dk = q.shape
        Hv, dv = v.shape[2], v.shape[3]
    _need(tuple(k.shape) == tuple(q.shape), "k must have q's shape")
    gdt = _gate_dtype(a, "a")
    _need(b_logits.dtype == a.dtype, "a and b_logits must share a dtype")
    if gates == "bth":
        _need(a.is_cuda and b_logits.is_cuda, "a and b_logits must be CUDA tensors")
        _need(tuple(a.shape) == (B, T, Hv) and tuple(b_logits.shape) == (B, T, Hv),
              "a, b_logits must be [B, T, Hv] with gates='bth'")
        ld = a.stride(1)
        _need(a.stride(2) == 1 and tuple(b_logits.stride()) == tuple(a.stride()) and a.stride(0) == T * ld
              and ld >= Hv, "a, b_logits (gates='bth'): token rows of one stride, heads contiguous")
    else:
        _cuda_contig(a, "a")
        _cuda_contig(b_logits, "b_logits")
        _need(tuple(a.shape) == (B, Hv, T) and tuple(b_logits.shape) == (B, Hv, T), "a, b_logits must be [B, Hv, T]")
    _cuda_contig(A_log, "A_log", torch.float32)
    dt_vec = None
    dt_scalar = 0.0
    if isinstance(dt_bias, torch.Tensor) and dt_bias.numel() > 1:
        _cuda_contig(dt_bias, "dt_bias", torch.float32)
        dt_vec = dt_bias
    else:
        dt_scalar = float(dt_bias)
    if mask is not None:
        _cuda_contig(mask, "mask", torch.float32)
    if state_in is not None:
        _cuda_contig(state_in, "state_in", torch.float32)
    return lay, B, T, Hqk, Hv, dk, dv, gdt, dt_scalar, dt_vec


def _contig(t: torch.Tensor, name: str, dtype=None) -> None:
    _need(t.is_contiguous(), f"{name} must be contiguous")
    if dtype is not None:
        _need(t.dtype == dtype, f"{name} must be {dtype}, got {t.dtype}")


def prefill_host(q, k, v, A_log, a, b_logits, *, dt_bias=0.0, mask=None, state_in=None, scale=0.0,
                 layout="bhtd", out=None, state_out=None, return_state=True, seg_tokens=0, device=None,
                 synchronize=True):
    """``prefill`` on host tensors (gdn_prefill_host): the inputs are copied to the
    GPU and the results back in token segments that overlap the prefill of the
    neighbouring segments.  Tensors may live on the host (pinned, for the copies
    to overlap) or on the device; outputs default to pinned host tensors.
    ``seg_tokens`` 0 picks the segment length.  With ``synchronize`` the current
    stream is synchronised before returning; without it the host outputs are
    valid once the stream completes, and the caller keeps the host inputs alive
    until then.  Same result as ``prefill`` on the whole sequence."""
    lay = GDN_LAYOUT_BHTD if layout == "bhtd" else GDN_LAYOUT_BTHD
    for name, t in (("q", q), ("k", k), ("v", v)):
        _contig(t, name, torch.bfloat16)
    if lay == GDN_LAYOUT_BHTD:
        B, Hqk, T, dk = q.shape
        Hv, dv = v.shape[1], v.shape[3]
    else:
        B, T, Hqk, dk = q.shape
        Hv, dv = v.shape[2], v.shape[3]
    _need(tuple(k.shape) == tuple(q.shape), "k must have q's shape")
    gdt = _gate_dtype(a, "a")
    _need(b_logits.dtype == a.dtype, "a and b_logits must share a dtype")
    _contig(a, "a")
    _contig(b_logits, "b_logits")
    _need(tuple(a.shape) == (B, Hv, T) and tuple(b_logits.shape) == (B, Hv, T), "a, b_logits must be [B, Hv, T]")
    _contig(A_log, "A_log", torch.float32)
    dt_vec, dt_scalar = None, 0.0
    if isinstance(dt_bias, torch.Tensor) and dt_bias.numel() > 1:
        _contig(dt_bias, "dt_bias", torch.float32)
        dt_vec = dt_bias
    else:
        dt_scalar = float(dt_bias)
    if mask is not None:
        _contig(mask, "mask", torch.float32)
    if state_in is not None:
        _contig(state_in, "state_in", torch.float32)
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    if out is None:
        out = torch.empty(v.shape, dtype=torch.bfloat16, pin_memory=True)
    if state_out is None and return_state:
        state_out = torch.empty(B, Hv, dk, dv, dtype=torch.float32, pin_memory=True)
    ws_bytes = int(_lib.lib().gdn_prefill_host_workspace_bytes(B, T, Hqk, Hv, dk, dv, gdt, int(seg_tokens)))
    _need(ws_bytes > 0, f"prefill_host: unsupported shapes or seg_tokens={seg_tokens}")
    ws = torch.empty(ws_bytes + 256, dtype=torch.uint8, device=dev)
    ws_ptr = (ws.data_ptr() + 255) // 256 * 256
    with torch.cuda.device(dev):
        _lib.call("gdn_prefill_host", _ptr(q), _ptr(k), _ptr(v), _ptr(A_log), _ptr(a), _ptr(b_logits), gdt,
                  dt_scalar, _ptr(dt_vec), _ptr(mask), _ptr(state_in), _ptr(out), _ptr(state_out),
                  B, T, Hqk, Hv, dk, dv, lay, float(scale), int(seg_tokens), ws_ptr, ws_bytes, _stream())
        if synchronize:
            torch.cuda.current_stream().synchronize()
    return out, state_out


def prefill_varlen(q, k, v, A_log, a, b_logits, cu_seqlens, *, max_len=None, dt_bias=0.0, state_in=None,
                   scale=0.0, out=None, state_out=None, return_state=True):
    """Prefill of N sequences packed along the token axis (gdn_prefill_varlen_fwd_ws).

    q,k [Ttot,Hqk,dk], v [Ttot,Hv,dv] bf16; a, b_logits [Hv,Ttot]; cu_seqlens int32 [N+1]
    on the device (sequence i = tokens cu_seqlens[i]:cu_seqlens[i+1]); max_len = the
    longest sequence (read from cu_seqlens with a device->host copy when not given);
    state_in [N,Hv,dk,dv] f32 or None.  Returns (out [Ttot,Hv,dv] bf16, state_out
    [N,Hv,dk,dv] f32 or None); per sequence the result of ``prefill`` on it alone."""
    for name, t in (("q", q), ("k", k), ("v", v)):
        _cuda_contig(t, name, torch.bfloat16)
    _need(q.dim() == 3 and v.dim() == 3, "q, k, v must be [Ttot, H, D]")
    Ttot, Hqk, dk = q.shape
    Hv, dv = v.shape[1], v.shape[2]
    _need(tuple(k.shape) == tuple(q.shape) and v.shape[0] == Ttot, "k must have q's shape, v Ttot rows")
    gdt = _gate_dtype(a, "a")
    _need(b_logits.dtype == a.dtype, "a and b_logits must share a dtype")
    _cuda_contig(a, "a")
    _cuda_contig(b_logits, "b_logits")
    _need(tuple(a.shape) == (Hv, Ttot) and tuple(b_logits.shape) == (Hv, Ttot), "a, b_logits must be [Hv, Ttot]")
    _cuda_contig(cu_seqlens, "cu_seqlens", torch.int32)
    N = cu_seqlens.numel() - 1
    _need(N >= 1, "cu_seqlens needs at least two entries")
    if max_len is None:
        max_len = int((cu_seqlens[1:] - cu_seqlens[:-1]).max())
    max_len = max(int(max_len), 1)
    _cuda_contig(A_log, "A_log", torch.float32)
    dt_vec, dt_scalar = None, 0.0
    if isinstance(dt_bias, torch.Tensor) and dt_bias.numel() > 1:
        _cuda_contig(dt_bias, "dt_bias", torch.float32)
        dt_vec = dt_bias
    else:
        dt_scalar = float(dt_bias)
    if state_in is not None:
        _cuda_contig(state_in, "state_in", torch.float32)
    if out is None:
        out = torch.empty_like(v)
    if state_out is None and return_state:
        state_out = torch.empty(N, Hv, dk, dv, dtype=torch.float32, device=q.device)
    ws_bytes = _lib.lib().gdn_prefill_varlen_workspace_bytes(N, max_len, Hv, dk, dv)
    ws = torch.empty(max(int(ws_bytes), 1), dtype=torch.uint8, device=q.device)
    _lib.call("gdn_prefill_varlen_fwd_ws", _ptr(q), _ptr(k), _ptr(v), _ptr(A_log), _ptr(a), _ptr(b_logits), gdt,
              dt_scalar, _ptr(dt_vec), _ptr(cu_seqlens), N, Ttot, max_len, _ptr(state_in), _ptr(out),
              _ptr(state_out), Hqk, Hv, dk, dv, float(scale), _ptr(ws), int(ws_bytes), _stream())
    return out, state_out


def prefill_backward(q, k, v, A_log, a, b_logits, dO, *, dt_bias=0.0, mask=None, state_in=None, dS_final=None,
                     scale=0.0, need_dstate=True, window=None, algorithm=None):
    """Gradients of ``prefill`` (gdn_prefill_bwd): q, k [B,H,T,dk], v [B,H,T,dv] bf16
    (layout "bhtd", Hqk == Hv), gates as ``prefill``, dO [B,H,T,dv] (bf16 or f32),
    dS_final [B,H,dk,dv] or None.  ``algorithm``: "token" (token-recurrent, in
    windows), "chunked" (64-token chunks) or None (the library's choice).
    ``window``: tokens per window of the token-recurrent backward (None: automatic,
    max(256, sqrt T)).  Returns a dict of fp32 tensors
    dq, dk, dv, da, db, dA_log [H], ddt_bias ([H] for a per-head dt_bias, a scalar
    tensor otherwise) and dstate_in (or None)."""
    for name, t in (("q", q), ("k", k), ("v", v)):
        _cuda_contig(t, name, torch.bfloat16)
    B, H, T, dk = q.shape
    dv = v.shape[-1]
    gdt = _gate_dtype(a, "a")
    _need(b_logits.dtype == a.dtype, "a and b_logits must share a dtype")
    _cuda_contig(a, "a")
    _cuda_contig(b_logits, "b_logits")
    _need(dO.dtype in (torch.bfloat16, torch.float32), "dO must be bf16 or f32")
    _cuda_contig(dO, "dO")
    dod = GDN_DTYPE_BF16 if dO.dtype == torch.bfloat16 else GDN_DTYPE_F32
    dt_vec = dt_bias if isinstance(dt_bias, torch.Tensor) and dt_bias.numel() > 1 else None
    dt_scalar = 0.0 if dt_vec is not None else float(dt_bias)
    f32 = dict(dtype=torch.float32, device=q.device)
    g = dict(dq=torch.empty(B, H, T, dk, **f32), dk=torch.empty(B, H, T, dk, **f32), dv=torch.empty(B, H, T, dv, **f32),
             da=torch.empty(B, H, T, **f32), db=torch.empty(B, H, T, **f32), dA_log=torch.empty(H, **f32),
             ddt_bias=torch.empty(H, **f32),
             dstate_in=torch.empty(B, H, dk, dv, **f32) if need_dstate else None)
    _need(window is None or int(window) > 0, f"window must be a positive token count, got {window!r}")
    algos = {None: 0, "token": 1, "chunked": 2}
    _need(algorithm in algos, f"algorithm must be None, 'token' or 'chunked', got {algorithm!r}")
    lib = _lib.lib()
    _lib.call("gdn_prefill_bwd_set_window", 0 if window is None else int(window))
    _lib.call("gdn_prefill_bwd_set_algorithm", algos[algorithm])
    try:
        ws_bytes = lib.gdn_prefill_bwd_workspace_bytes(B, T, H, dk, dv)
        ws = torch.empty(max(int(ws_bytes), 1), dtype=torch.uint8, device=q.device)
        _lib.call("gdn_prefill_bwd", _ptr(q), _ptr(k), _ptr(v), _ptr(A_log), _ptr(a), _ptr(b_logits), gdt,
                  dt_scalar, _ptr(dt_vec), _ptr(mask), _ptr(state_in), _ptr(dO), dod, _ptr(dS_final), _ptr(g["dq"]),
                  _ptr(g["dk"]), _ptr(g["dv"]), _ptr(g["da"]), _ptr(g["db"]), _ptr(g["dA_log"]),
                  _ptr(g["ddt_bias"]), _ptr(g["dstate_in"]), B, T, H, dk, dv, float(scale), _ptr(ws),
                  int(ws_bytes), _stream())
    finally:
        _lib.call("gdn_prefill_bwd_set_window", 0)
        _lib.call("gdn_prefill_bwd_set_algorithm", 0)
    if dt_vec is None:
        g["ddt_bias"] = g["ddt_bias"].sum()
    return g


class _FirstDerivative(torch.autograd.Function):
    """run(), a gradient of functions of ``tensors``, as a node that cannot be differentiated."""

    @staticmethod
    def forward(ctx, run, *tensors):
        return run()

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("this operator's gradient is computed by a kernel: it is differentiable once only")


def _once(backward):
    """For Function.backward: under create_graph the gradients stay tied to what they were
    computed from, so that a second derivative is an error rather than a number without their
    share (torch's once_differentiable ties them to nothing, and torch.autograd.grad passes
    over its error)."""
    @functools.wraps(backward)
    def tied(ctx, *grads):
        if not torch.is_grad_enabled():
            return backward(ctx, *grads)
        return _FirstDerivative.apply(lambda: backward(ctx, *grads), *grads, *ctx.saved_tensors)
    return tied


class PrefillFunction(torch.autograd.Function):
    """``prefill`` as an autograd op (layout "bhtd", Hqk == Hv): forward is the
    chunked tcgen05 prefill, backward gdn_prefill_backward.  Differentiable
    inputs (once): q, k, v, A_log, a, b_logits, dt_bias (tensor) and
    state_in; outputs (o, state_out)."""

    @staticmethod
    def forward(ctx, q, k, v, A_log, a, b_logits, dt_bias, state_in, scale):
        o, S = prefill(q, k, v, A_log, a, b_logits, dt_bias=dt_bias, state_in=state_in, scale=scale)
        ctx.save_for_backward(q, k, v, A_log, a, b_logits, dt_bias, state_in)
        ctx.scale = scale
        return o, S

    @staticmethod
    @_once
    def backward(ctx, do, dS):
        q, k, v, A_log, a, b_logits, dt_bias, state_in = ctx.saved_tensors
        if do is None:
            do = torch.zeros_like(v, dtype=torch.float32)
        g = prefill_backward(q, k, v, A_log, a, b_logits, do.contiguous(), dt_bias=dt_bias, state_in=state_in,
                             dS_final=None if dS is None else dS.contiguous(), scale=ctx.scale)
        ddt = g["ddt_bias"].reshape(dt_bias.shape).to(dt_bias.dtype)
        return (g["dq"].to(q.dtype), g["dk"].to(k.dtype), g["dv"].to(v.dtype), g["dA_log"], g["da"].to(a.dtype),
                g["db"].to(b_logits.dtype), ddt, g["dstate_in"], None)


def prefill_autograd(q, k, v, A_log, a, b_logits, dt_bias, state_in, scale=0.0):
    """Differentiable ``prefill`` (see PrefillFunction); dt_bias a tensor ([H] or [1])."""
    return PrefillFunction.apply(q, k, v, A_log, a, b_logits, dt_bias, state_in, scale)


def decode_step(q, k, v, a, b, A_log, dt_bias, state, *, scale=0.0, out=None, state_out=None, l2norm_qk=False):
    """One decode step; updates ``state`` in place unless ``state_out`` is given.
    q,k [B,Hqk,dk] bf16; v [B,Hv,dv] bf16; a,b [B,Hv]; state [B,Hv,dk,dv] f32.
    With ``l2norm_qk`` q and k are L2-normalised per head inside the kernel.
    Returns out f32 [B,Hv,dv]."""
    B, Hqk, dk = q.shape
    Hv, dv = v.shape[1], v.shape[2]
    for name, t in (("q", q), ("k", k), ("v", v)):
        _cuda_contig(t, name, torch.bfloat16)
    _cuda_contig(state, "state", torch.float32)
    gdt = _gate_dtype(a, "a")
    if out is None:
        out = torch.empty(B, Hv, dv, dtype=torch.float32, device=q.device)
    if state_out is None:
        state_out = state
    _lib.call("gdn_decode_step_ex", _ptr(q), _ptr(k), _ptr(v), _ptr(a), _ptr(b), gdt, _ptr(A_log),
              _ptr(dt_bias), _ptr(state), _ptr(state_out), _ptr(out), B, Hqk, Hv, dk, dv, float(scale),
              _lib.GDN_DECODE_L2NORM_QK if l2norm_qk else 0, _stream())
    return out


def decode_step_gated(q, k, v, a, b, A_log, dt_bias, state, z, norm_gamma, eps, *, scale=0.0, y=None,
                      out=None, state_out=None, l2norm_qk=False):
    """``decode_step`` with the layer's gated output norm applied to each head's o row in
    the same kernel (gdn_decode_step_gated): y = rmsnorm_dv(o) * norm_gamma * silu(z), bf16.
    z [B,Hv,dv] bf16; norm_gamma [dv] bf16.  ``out`` (the fp32 o) is written only when
    given.  Returns y [B,Hv,dv] bf16."""
    B, Hqk, dk = q.shape
    Hv, dv = v.shape[1], v.shape[2]
    for name, t in (("q", q), ("k", k), ("v", v), ("z", z), ("norm_gamma", norm_gamma)):
        _cuda_contig(t, name, torch.bfloat16)
    _cuda_contig(state, "state", torch.float32)
    _need(z.numel() == B * Hv * dv and norm_gamma.numel() == dv, "z must be [B, Hv, dv] and norm_gamma [dv]")
    gdt = _gate_dtype(a, "a")
    if y is None:
        y = torch.empty(B, Hv, dv, dtype=torch.bfloat16, device=q.device)
    if state_out is None:
        state_out = state
    _lib.call("gdn_decode_step_gated", _ptr(q), _ptr(k), _ptr(v), _ptr(a), _ptr(b), gdt, _ptr(A_log),
              _ptr(dt_bias), _ptr(state), _ptr(state_out), _ptr(out), _ptr(z), _ptr(norm_gamma), float(eps),
              _ptr(y), B, Hqk, Hv, dk, dv, float(scale), _lib.GDN_DECODE_L2NORM_QK if l2norm_qk else 0, _stream())
    return y


def outproj_rs(x, W, recv_ptrs, rank, world):
    """This rank's share of a head-sharded output projection, sent to its owners
    (gdn_outproj_rs_fwd): the partial product x [M, K] @ W[N, K]^T, cut into row
    blocks of M/world tokens, block s written into slot ``rank`` of the receive
    buffer at ``recv_ptrs[s]`` (device pointers of every rank's [world, M/world, N]
    bf16 buffer, peers' mapped into this process).  Only launches; ordering the
    reduction after every rank's call is the caller's job."""
    _cuda_contig(x, "x", torch.bfloat16)
    _cuda_contig(W, "W", torch.bfloat16)
    _need(x.dim() == 2 and W.dim() == 2 and x.shape[1] == W.shape[1], "x [M, K] and W [N, K] required")
    _need(len(recv_ptrs) == world, "one receive buffer per rank")
    arr = (ctypes.c_void_p * world)(*[int(p) for p in recv_ptrs])
    _lib.call("gdn_outproj_rs_fwd", _ptr(x), _ptr(W), arr, x.shape[0], W.shape[0], x.shape[1], int(rank), int(world),
              _stream())


def gather_window(gathered, peer_ptrs, rank, t0, Tw, layout="bhtd", stream=None):
    """Pull tokens [t0, t0 + Tw) of every peer's slot of a head-sharded o into the
    same slots of ``gathered`` [world, B, H_local, T, dv] ("bhtd") or [world, B, T,
    H_local, dv] ("bthd") (gdn_gather_window): one copy-engine transfer per peer
    from ``peer_ptrs[p]`` (rank p's gathered buffer, mapped into this process),
    enqueued on ``stream`` (default: the current stream).  Only enqueues; the
    caller orders it after the peers wrote the window."""
    _cuda_contig(gathered, "gathered", torch.bfloat16)
    _need(gathered.dim() == 5, "gathered must be [world, B, H, T, dv] or [world, B, T, H, dv]")
    _need(layout in ("bhtd", "bthd"), f"layout must be 'bhtd' or 'bthd', got {layout!r}")
    world = gathered.shape[0]
    _need(len(peer_ptrs) == world, "one peer pointer per rank")
    if layout == "bhtd":
        _, B, H, T, dv = gathered.shape
        lay = GDN_LAYOUT_BHTD
    else:
        _, B, T, H, dv = gathered.shape
        lay = GDN_LAYOUT_BTHD
    arr = (ctypes.c_void_p * world)(*[int(p) for p in peer_ptrs])
    s = stream.cuda_stream if stream is not None else _stream()
    _lib.call("gdn_gather_window", _ptr(gathered), arr, world, int(rank), B, T, H, dv, lay, int(t0), int(Tw), s)


def outproj_reduce(recv, out=None):
    """out [rows, N] = bf16(sum over slots of recv [world, rows, N]) (gdn_outproj_reduce)."""
    _cuda_contig(recv, "recv", torch.bfloat16)
    world, rows, N = recv.shape
    if out is None:
        out = torch.empty(rows, N, dtype=torch.bfloat16, device=recv.device)
    _lib.call("gdn_outproj_reduce", _ptr(recv), _ptr(out), rows, N, world, _stream())
    return out


def rmsnorm(x, gamma, eps=1e-6, out=None):
    """y = x * rsqrt(mean(x^2) + eps) * gamma over the last dim; bf16 in/out."""
    _cuda_contig(x, "x", torch.bfloat16)
    _cuda_contig(gamma, "gamma", torch.bfloat16)
    D = x.shape[-1]
    R = x.numel() // D
    if out is None:
        out = torch.empty_like(x)
    _lib.call("gdn_rmsnorm_fwd", _ptr(x), _ptr(gamma), _ptr(out), R, D, float(eps), _stream())
    return out


def gated_rmsnorm(x, z, gamma, eps=1e-6, out=None):
    """y = rmsnorm(x) * gamma * silu(z) over the last dim (x bf16 or f32, z bf16)."""
    _cuda_contig(x, "x")
    _cuda_contig(z, "z", torch.bfloat16)
    _cuda_contig(gamma, "gamma", torch.bfloat16)
    xdt = _gate_dtype(x, "x")
    D = x.shape[-1]
    R = x.numel() // D
    if out is None:
        out = torch.empty(x.shape, dtype=torch.bfloat16, device=x.device)
    _lib.call("gdn_gated_rmsnorm_fwd", _ptr(x), xdt, _ptr(z), _ptr(gamma), _ptr(out), R, D, float(eps),
              _stream())
    return out


def proj_conv_silu(x, W, conv_w, *, conv_state_in=None, conv_state_out=None, l2norm_group=0, out=None):
    """SiLU(causal_conv4(x @ W^T)) with optional conv history and per-group L2 norm.
    x [B,T,D] bf16; W [Dout,D] bf16; conv_w [Dout,4] bf16 -> [B,T,Dout] bf16."""
    _cuda_contig(x, "x", torch.bfloat16)
    _cuda_contig(W, "W", torch.bfloat16)
    _cuda_contig(conv_w, "conv_w", torch.bfloat16)
    B, T, D = x.shape
    Dout = W.shape[0]
    if out is None:
        out = torch.empty(B, T, Dout, dtype=torch.bfloat16, device=x.device)
    _lib.call("gdn_proj_conv_silu_fwd", _ptr(x), _ptr(W), _ptr(conv_w), _ptr(out), B, T, D, Dout,
              _ptr(conv_state_in), _ptr(conv_state_out), int(l2norm_group), _stream())
    return out


def proj_multi(x, segments):
    """Several projections of the same x [B,T,D] bf16 in one launch (gdn_proj_multi_fwd).
    ``segments``: up to 6 dicts with ``W`` [Dout, D] bf16 and optionally ``conv_w``
    [Dout, 4] (without it: a plain projection x @ W^T rounded to bf16),
    ``conv_state_in`` / ``conv_state_out`` [B, Dout, 3], ``l2norm_group`` and ``out``
    [B, T, Dout].  Returns the list of outputs, each as ``proj_conv_silu`` (or the
    plain projection) would give it."""
    _cuda_contig(x, "x", torch.bfloat16)
    _need(x.dim() == 3, "x must be [B, T, D]")
    B, T, D = x.shape
    segs = (_lib.ProjOutSeg * len(segments))()
    outs = []
    for i, sg in enumerate(segments):
        W = sg["W"]
        _cuda_contig(W, f"segments[{i}].W", torch.bfloat16)
        _need(W.dim() == 2 and W.shape[1] == D, f"segments[{i}].W must be [Dout, {D}]")
        Dout = W.shape[0]
        out = sg.get("out")
        if out is None:
            out = torch.empty(B, T, Dout, dtype=torch.bfloat16, device=x.device)
        _cuda_contig(out, f"segments[{i}].out", torch.bfloat16)
        cw = sg.get("conv_w")
        if cw is not None:
            _cuda_contig(cw, f"segments[{i}].conv_w", torch.bfloat16)
        segs[i].W, segs[i].y, segs[i].conv_w = _ptr(W), _ptr(out), _ptr(cw)
        segs[i].conv_state_in, segs[i].conv_state_out = _ptr(sg.get("conv_state_in")), _ptr(sg.get("conv_state_out"))
        segs[i].Dout, segs[i].l2norm_group = Dout, int(sg.get("l2norm_group", 0))
        outs.append(out)
    _lib.call("gdn_proj_multi_fwd", _ptr(x), B, T, D, segs, len(segments), _stream())
    return outs


def decode_proj(x, segments, *, norm_gamma=None, eps=1e-6):
    """Input projections of one decode step in one launch (gdn_decode_proj_fwd).

    x [B, D] bf16 (B <= 8); ``segments``: list of dicts with ``W`` [C, D] bf16 and
    optionally ``conv_w`` [C, 4], ``conv_state_in`` / ``conv_state_out`` [B, C, 3]
    (may be the same tensor: updated in place), ``l2_group`` and ``out`` [B, C].
    With ``norm_gamma`` x is RMS-normalised first.  Returns the list of outputs,
    each [B, C] bf16: SiLU(conv4) (L2-normalised per group when asked) for the
    segments with ``conv_w``, plain bf16(x W^T) rows for the others."""
    _cuda_contig(x, "x", torch.bfloat16)
    _need(x.dim() == 2, "x must be [B, D]")
    B, D = x.shape
    if norm_gamma is not None:
        _cuda_contig(norm_gamma, "norm_gamma", torch.bfloat16)
    segs = (_lib.ProjSegment * len(segments))()
    outs = []
    for i, sg in enumerate(segments):
        W = sg["W"]
        _cuda_contig(W, f"segments[{i}].W", torch.bfloat16)
        _need(W.shape[1] == D, f"segments[{i}].W must be [C, {D}]")
        C = W.shape[0]
        out = sg.get("out")
        if out is None:
            out = torch.empty(B, C, dtype=torch.bfloat16, device=x.device)
        _need(out.dtype == torch.bfloat16 and out.is_cuda and out.shape[-1] == C and out.stride(-1) == 1,
              f"segments[{i}].out must be bf16 [B, {C}] with unit inner stride")
        for name in ("conv_w", "conv_state_in", "conv_state_out"):
            if sg.get(name) is not None:
                _cuda_contig(sg[name], f"segments[{i}].{name}", torch.bfloat16)
        segs[i] = _lib.ProjSegment(_ptr(W), _ptr(out), _ptr(sg.get("conv_w")), _ptr(sg.get("conv_state_in")),
                                   _ptr(sg.get("conv_state_out")), C, out.stride(0) if B > 1 else C,
                                   int(sg.get("l2_group", 0)))
        outs.append(out)
    _lib.call("gdn_decode_proj_fwd", _ptr(x), _ptr(norm_gamma), float(eps), B, D, segs, len(segments), _stream())
    return outs


# ---------------------------------------------------------------------------
# the softmax-attention block of a hybrid stack: the norms around a block, rotary
# positions, the paged cache and its attention
# ---------------------------------------------------------------------------


_INT_MAX = 0x7FFFFFFF


def _int(n):
    """n as a C int that compares with every size as n does (ctypes would take its low 32 bits)."""
    return max(-1, min(n, _INT_MAX))


def _dense(t, name, dtype):
    """A contiguous CUDA tensor of that type (one test on the way that is right)."""
    if not (t.dtype is dtype and t.is_cuda and t.is_contiguous()):
        _cuda_contig(t, name, dtype)


def _shaped(t, name, shape, dtype):
    _dense(t, name, dtype)
    if t.shape != shape:
        raise RuntimeError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")


def _like(t):
    """An uninitialised contiguous tensor of t's shape, type and device."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _norm_args(y, h, hname, gamma_post, gate, gamma_pre):
    """Checks shared by block_norm and its backward; returns (rows, columns, residual type
    code, gate rows, whether every row has its own gate row)."""
    _dense(y, "y", torch.bfloat16)
    hdt = _gate_dtype(h, hname)
    if h.shape != y.shape or y.dim() < 1 or y.shape[-1] == 0:
        raise RuntimeError(f"{hname} must have y's shape, with at least one column")
    _dense(h, hname, h.dtype)
    D = y.shape[-1]
    R = y.numel() // D
    if R > _INT_MAX:
        raise RuntimeError(f"at most {_INT_MAX} rows, got {R}")
    for name, w in (("gamma_post", gamma_post), ("gamma_pre", gamma_pre)):
        if w is not None:
            _dense(w, name, torch.bfloat16)
            if w.dim() != 1 or w.shape[0] != D:
                raise RuntimeError(f"{name} must be [{D}]")
    if gate is None:
        return R, D, hdt, 0, False
    _dense(gate, "gate", torch.bfloat16)
    if gate.dim() not in (1, 2) or gate.shape[-1] != D:
        raise RuntimeError(f"gate must be [{D}] or [G, {D}]")
    if gate.dim() == 1:
        return R, D, hdt, 1, False
    G = gate.shape[0]
    if G < 1 and R > 0 or G > 0 and R % G != 0:
        raise RuntimeError(f"gate rows ({G}) must divide the {R} rows")
    return R, D, hdt, G, G == R


def block_norm(y, h, *, gamma_post=None, gate=None, gamma_pre=None, residual_scale=1.0, eps=1e-6, h_out=None,
               x_out=None):
    """The norms around a block, with its gate and the residual scale, in one pass
    (gdn_block_norm_fwd): h' = residual_scale * h + gate * u with u = RMSNorm(y) *
    gamma_post (u = y without it), and x = RMSNorm(h') * gamma_pre, the next block's input.

    y [..., D] bf16; h [..., D] bf16 or f32 (the residual stream); gate None, [D], or
    [G, D] bf16 with G dividing the rows (a gate row per sequence, or per token);
    gammas [D] bf16.  Returns (h', x): h' in h's type, x bf16 or None without
    gamma_pre.  ``h_out=h`` updates the residual stream in place."""
    R, D, hdt, G, _ = _norm_args(y, h, "h", gamma_post, gate, gamma_pre)
    if h_out is None:
        h_out = torch.empty_like(h)
    else:
        _shaped(h_out, "h_out", h.shape, h.dtype)
    if gamma_pre is None:
        x_out = None
    elif x_out is None:
        x_out = torch.empty_like(y)
    else:
        _shaped(x_out, "x_out", y.shape, torch.bfloat16)
    if R == 0:
        return h_out, x_out
    _lib.call("gdn_block_norm_fwd", y.data_ptr(), h.data_ptr(), hdt, _ptr(gamma_post), _ptr(gate), G, _ptr(gamma_pre),
              float(residual_scale), h_out.data_ptr(), _ptr(x_out), R, D, float(eps), _stream())
    return h_out, x_out


def block_norm_backward(y, h_out, dh_out=None, dx=None, *, gamma_post=None, gate=None, gamma_pre=None,
                        residual_scale=1.0, eps=1e-6):
    """Gradients of ``block_norm`` from y and its stored result h_out (gdn_block_norm_bwd):
    dh_out [..., D] in h_out's type or None (zero), dx bf16 (with gamma_pre).  Returns a
    dict of dy bf16, dh in h_out's type, dgamma_post and dgamma_pre [D] f32 and dgate
    (f32 [D] or [G, D], sums over the rows that share a gate row; bf16 [R, D] for a gate
    row per row), None where there is no such input."""
    R, D, hdt, G, per_row = _norm_args(y, h_out, "h_out", gamma_post, gate, gamma_pre)
    if dh_out is not None:
        _shaped(dh_out, "dh_out", y.shape, h_out.dtype)
    if gamma_pre is None:
        dx = None
    elif dx is None:
        raise RuntimeError("dx is required with gamma_pre")
    else:
        _shaped(dx, "dx", y.shape, torch.bfloat16)
    # the sums over rows share an allocation
    summed = gate is not None and not per_row
    rows = torch.empty(2 + (G if summed else 0), D, dtype=torch.float32, device=y.device)
    g = dict(dy=torch.empty_like(y), dh=torch.empty_like(h_out),
             dgate=None if gate is None else torch.empty_like(gate) if per_row else rows[2:].view(gate.shape),
             dgamma_post=None if gamma_post is None else rows[0], dgamma_pre=None if gamma_pre is None else rows[1])
    if R == 0:
        return {n: None if t is None else t.zero_() for n, t in g.items()}
    ws_bytes = _lib.lib().gdn_block_norm_bwd_workspace_bytes(R, D, G)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=y.device)
    at = rows.data_ptr()
    _lib.call("gdn_block_norm_bwd", y.data_ptr(), h_out.data_ptr(), hdt, _ptr(dh_out), _ptr(dx), _ptr(gamma_post),
              _ptr(gate), G, _ptr(gamma_pre), float(residual_scale), g["dy"].data_ptr(), g["dh"].data_ptr(),
              _ptr(g["dgate"]), GDN_DTYPE_BF16 if per_row else GDN_DTYPE_F32, None if gamma_post is None else at,
              None if gamma_pre is None else at + 4 * D, R, D, float(eps), ws.data_ptr(), ws_bytes, _stream())
    return g


class BlockNormFunction(torch.autograd.Function):
    """``block_norm`` as an autograd op: differentiable in y, h, gamma_post, gate and
    gamma_pre, once; outputs (h', x)."""

    @staticmethod
    def forward(ctx, y, h, gamma_post, gate, gamma_pre, residual_scale, eps):
        h_out, x = block_norm(y, h, gamma_post=gamma_post, gate=gate, gamma_pre=gamma_pre,
                              residual_scale=residual_scale, eps=eps)
        ctx.save_for_backward(y, h_out, gamma_post, gate, gamma_pre)
        ctx.scale, ctx.eps = residual_scale, eps
        return h_out, x

    @staticmethod
    @_once
    def backward(ctx, dh, dx):
        y, h_out, gamma_post, gate, gamma_pre = ctx.saved_tensors
        if dx is None and gamma_pre is not None:
            dx = torch.zeros_like(y)
        g = block_norm_backward(y, h_out, None if dh is None else dh.contiguous(),
                                None if dx is None else dx.contiguous(), gamma_post=gamma_post, gate=gate,
                                gamma_pre=gamma_pre, residual_scale=ctx.scale, eps=ctx.eps)
        like = lambda d, p: None if p is None else d.to(p.dtype)  # noqa: E731
        return (g["dy"], g["dh"], like(g["dgamma_post"], gamma_post), like(g["dgate"], gate),
                like(g["dgamma_pre"], gamma_pre), None, None)


def block_norm_autograd(y, h, *, gamma_post=None, gate=None, gamma_pre=None, residual_scale=1.0, eps=1e-6):
    """Differentiable ``block_norm`` (see BlockNormFunction)."""
    return BlockNormFunction.apply(y, h, gamma_post, gate, gamma_pre, residual_scale, eps)


_ROPE_STYLES = {"half": _lib.GDN_ROPE_HALF, "interleaved": _lib.GDN_ROPE_INTERLEAVED}


def _token_rows(t, name):
    """(tokens, heads, D, elements between tokens) of [..., H, D] bf16 whose heads and
    values are contiguous and whose tokens are rows of one stride (a slice of a fused
    projection is one)."""
    if not (t.is_cuda and t.dtype is torch.bfloat16):
        raise RuntimeError(f"{name} must be a bfloat16 CUDA tensor")
    shape = t.shape
    if len(shape) < 3:
        raise RuntimeError(f"{name} must be [..., heads, head dim]")
    H, D = shape[-2], shape[-1]
    if t.is_contiguous():
        return (shape[0] if len(shape) == 3 else t.numel() // (H * D) if H * D else 0), H, D, H * D
    _need(t.stride(-1) == 1 and (H == 1 or t.stride(-2) == D), f"{name}: heads and values must be contiguous")
    T, ld = 1, None
    for n, s in zip(reversed(shape[:-2]), reversed(t.stride()[:-2])):
        if n == 1:
            continue
        if ld is None:
            ld = s
        elif s != ld * T:
            raise RuntimeError(f"{name}: tokens must be rows of one stride")
        T *= n
    return T, H, D, (H * D if ld is None else ld)


@functools.lru_cache(maxsize=64)
def _int_array(values):
    """A C array of these ints (they are few and known at the call)."""
    return (ctypes.c_int * len(values))(*values)


def _rope_spec(positions, inv_freq, sections, style, T):
    code = _ROPE_STYLES.get(style)
    if code is None:
        raise RuntimeError(f"style must be 'half' or 'interleaved', got {style!r}")
    if not (positions.is_cuda and positions.dtype is torch.int32):
        raise RuntimeError("positions must be an int32 CUDA tensor")
    if not (inv_freq.is_cuda and inv_freq.dtype is torch.float32 and inv_freq.dim() == 1 and inv_freq.is_contiguous()):
        raise RuntimeError("inv_freq must be a contiguous float32 CUDA vector")
    pairs = inv_freq.shape[0]
    sections = (pairs,) if sections is None else tuple(sections)
    axes = len(sections)
    shape = positions.shape
    if not positions.is_contiguous() or positions.numel() != axes * T or (axes > 1 and (len(shape) < 2 or shape[0] != axes)):
        raise RuntimeError(f"positions must be contiguous, [{axes}, tokens] ([tokens] for one axis), got {tuple(shape)}")
    counts = _int_array(sections)
    spec = _lib.RopeSpec(positions.data_ptr(), T, inv_freq.data_ptr(), ctypes.addressof(counts), axes, 2 * pairs, code)
    spec.counts = counts            # the structure holds an address only
    return spec


def rope(q, k, positions, inv_freq, sections=None, *, style="half", inverse=False, q_out=None, k_out=None):
    """Rotary positions with several axes (gdn_rope_fwd): pair i of the first
    2 * len(inv_freq) values of each head is turned by positions[axis][t] * inv_freq[i],
    where ``sections`` counts the pairs of each axis in turn (None: one axis).

    q [..., Hq, D], k [..., Hk, D] bf16 or None (tokens may be strided rows); positions
    int32 [axes, tokens] ([tokens] for one axis); inv_freq f32 [rot / 2]; style "half" pairs values (i, i + rot/2),
    "interleaved" (2i, 2i + 1).  ``inverse`` turns back, which is the gradient.
    Returns (q_out, k_out), contiguous; ``q_out=q`` works in place."""
    T, Hq, D, q_ld = _token_rows(q, "q")
    Hk = k_ld = 0
    if k is not None:
        Tk, Hk, Dk, k_ld = _token_rows(k, "k")
        _need(Tk == T and Dk == D, "k must have q's tokens and head dim")
    spec = _rope_spec(positions, inv_freq, sections, style, T)
    if q_out is None:
        q_out = _like(q)
    else:
        _shaped(q_out, "q_out", q.shape, torch.bfloat16)
    if k is None:
        k_out = None
    elif k_out is None:
        k_out = _like(k)
    else:
        _shaped(k_out, "k_out", k.shape, torch.bfloat16)
    if T == 0:
        return q_out, k_out
    _lib.call("gdn_rope_fwd", q.data_ptr(), q_ld, _ptr(k), k_ld, q_out.data_ptr(), _ptr(k_out), ctypes.byref(spec),
              1 if inverse else 0, T, Hq, Hk, D, _stream())
    return q_out, k_out


class RopeFunction(torch.autograd.Function):
    """``rope`` as an autograd op, differentiable in q and k, once."""

    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, sections, style):
        ctx.save_for_backward(positions, inv_freq)
        ctx.sections, ctx.style = sections, style
        return rope(q, k, positions, inv_freq, sections, style=style)

    @staticmethod
    @_once
    def backward(ctx, dq, dk):
        positions, inv_freq = ctx.saved_tensors
        dq, dk = rope(dq.contiguous(), None if dk is None else dk.contiguous(), positions, inv_freq, ctx.sections,
                      style=ctx.style, inverse=True)
        return dq, dk, None, None, None, None


def rope_autograd(q, k, positions, inv_freq, sections=None, *, style="half"):
    """Differentiable ``rope`` (see RopeFunction)."""
    return RopeFunction.apply(q, k, positions, inv_freq, sections, style)


def _paged_cache(k_cache, v_cache, block_table, layout):
    if not (k_cache.is_cuda and v_cache.is_cuda and k_cache.dtype is torch.bfloat16 and v_cache.dtype is torch.bfloat16):
        raise RuntimeError("k_cache and v_cache must be bfloat16 CUDA tensors")
    shape, st = k_cache.shape, k_cache.stride()
    if len(shape) != 4 or v_cache.shape != shape or v_cache.stride() != st or st[3] != 1:
        raise RuntimeError("k_cache and v_cache must be 4-d and share shape and strides, the values of a row contiguous")
    ts = block_table.shape
    if not (block_table.is_cuda and block_table.dtype is torch.int32 and len(ts) == 2
            and (block_table.is_contiguous() or block_table.stride(1) == 1)):
        raise RuntimeError("block_table must be int32 [B, pages] CUDA rows")
    if layout == "bthd":
        pages, page_size, n_kv, D = shape
        token, head = st[1], st[2]
    elif layout == "bhtd":
        pages, n_kv, page_size, D = shape
        token, head = st[2], st[1]
    else:
        raise RuntimeError(f"layout must be 'bthd' or 'bhtd', got {layout!r}")
    return _lib.PagedCache(k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(),
                           block_table.stride(0) if ts[0] > 1 else ts[1], st[0], token, head, pages, page_size, ts[1],
                           n_kv, D)


def _sequences(cu_seqlens, kv_lens, block_table):
    _dense(cu_seqlens, "cu_seqlens", torch.int32)
    _dense(kv_lens, "kv_lens", torch.int32)
    B = kv_lens.numel()
    if B < 1 or cu_seqlens.numel() != B + 1 or block_table.shape[0] != B:
        raise RuntimeError("cu_seqlens must have B + 1 entries, kv_lens and block_table B rows")
    return B


def rope_append(q, k, v, positions, inv_freq, sections, k_cache, v_cache, block_table, cu_seqlens, kv_lens, *,
                style="half", layout="bthd", q_out=None):
    """The step before ``paged_attention`` (gdn_rope_append): q is turned as by ``rope``
    and returned, the turned keys and the values are written into the paged cache.

    q [T, Hq, D], k, v [T, Hkv, D] bf16: the new tokens of B sequences, packed
    (cu_seqlens int32 [B + 1]); they are the last ones of kv_lens int32 [B] positions.
    k_cache, v_cache [pages, page_size, Hkv, D] (layout "bthd") or [pages, Hkv, page_size,
    D] ("bhtd"), strided slices of a larger pool too; block_table int32 [B, max_pages].
    Sequence lengths live on the device, so the call can be captured in a CUDA graph."""
    T, Hq, D, q_ld = _token_rows(q, "q")
    Tk, Hk, Dk, k_ld = _token_rows(k, "k")
    Tv, Hv, Dv, v_ld = _token_rows(v, "v")
    cache = _paged_cache(k_cache, v_cache, block_table, layout)
    B = _sequences(cu_seqlens, kv_lens, block_table)
    if not (Tk == T == Tv and Hk == Hv == cache.n_kv and D == Dk == Dv == cache.head_dim):
        raise RuntimeError("q, k, v must have the same tokens and the cache's heads and head dim")
    spec = _rope_spec(positions, inv_freq, sections, style, T)
    if q_out is None:
        q_out = _like(q)
    else:
        _shaped(q_out, "q_out", q.shape, torch.bfloat16)
    if T == 0:
        return q_out
    _lib.call("gdn_rope_append", q.data_ptr(), q_ld, k.data_ptr(), k_ld, v.data_ptr(), v_ld, q_out.data_ptr(),
              ctypes.byref(spec), ctypes.byref(cache), cu_seqlens.data_ptr(), kv_lens.data_ptr(), B, T, Hq, _stream())
    return q_out


def paged_attention(q, k_cache, v_cache, block_table, cu_seqlens, kv_lens, *, max_q=None, max_kv=None, scale=0.0,
                    causal=True, window=0, layout="bthd", out=None, return_lse=False, workspace=None):
    """Softmax attention of new tokens over a paged cache that holds them already
    (gdn_paged_attn_fwd): single tokens, drafted ones and chunks of a prompt alike.

    q [T, Hq, D] bf16, the new tokens of B sequences, packed; caches, block_table,
    cu_seqlens and kv_lens as ``rope_append``.  Token i of a sequence sees its positions
    0 .. kv_len - q_len + i (``causal``; otherwise all), with ``window`` only the last
    ``window`` of them.  max_q, max_kv: the longest new chunk and an upper bound of the
    lengths, on the host (max_q is read from cu_seqlens with a device->host copy when not
    given, max_kv defaults to the block table's width).  scale 0 -> 1/sqrt(D).
    ``workspace``: uint8 CUDA tensor of at least paged_attention_workspace(...) bytes
    (allocated per call if None).  Returns out [T, Hq, D] bf16, with ``return_lse`` also
    the log of the softmax's sum, f32 [T, Hq].  A token that sees nothing gets zeros
    and -inf, one that sees a score of NaN or +inf gets NaN in both; rows of q past
    cu_seqlens[B] are not written.  The softmax's weights are rounded to bf16 before
    they meet the values (fp32 sums)."""
    T, Hq, D, q_ld = _token_rows(q, "q")
    cache = _paged_cache(k_cache, v_cache, block_table, layout)
    B = _sequences(cu_seqlens, kv_lens, block_table)
    if D != cache.head_dim:
        raise RuntimeError("q must have the cache's head dim")
    if max_q is None:
        max_q = int((cu_seqlens[1:] - cu_seqlens[:-1]).max())
    if max_kv is None:
        max_kv = cache.max_pages * cache.page_size
    if out is None:
        out = _like(q)
    else:
        _shaped(out, "out", q.shape, torch.bfloat16)
    lse = torch.empty(q.shape[:-1], dtype=torch.float32, device=q.device) if return_lse else None
    if T == 0:
        return (out, lse) if return_lse else out
    if not (0 <= max_q <= _INT_MAX and 0 <= max_kv <= _INT_MAX and 0 <= window <= _INT_MAX):
        max_q, max_kv, window = _int(max_q), _int(max_kv), _int(window)
    ws_bytes = _lib.lib().gdn_paged_attn_workspace_bytes(B, T, Hq, cache.n_kv, D, max_q, max_kv, window)
    if workspace is None:
        workspace = q.new_empty(ws_bytes // 2)
    elif not (workspace.is_cuda and workspace.dtype is torch.uint8 and workspace.numel() >= ws_bytes):
        raise RuntimeError(f"workspace: uint8 CUDA tensor of at least {ws_bytes} bytes required")
    _lib.call("gdn_paged_attn_fwd", q.data_ptr(), q_ld, ctypes.byref(cache), cu_seqlens.data_ptr(), kv_lens.data_ptr(),
              out.data_ptr(), _ptr(lse), B, T, Hq, max_q, max_kv, 1 if causal else 0, window, float(scale),
              workspace.data_ptr(), ws_bytes, _stream())
    return (out, lse) if return_lse else out


def paged_attention_workspace(B, T, Hq, n_kv, head_dim, max_q, max_kv, window=0):
    """Bytes of workspace ``paged_attention`` needs for calls up to these sizes."""
    return int(_lib.lib().gdn_paged_attn_workspace_bytes(_int(B), _int(T), _int(Hq), _int(n_kv), _int(head_dim), _int(max_q),
                                                         _int(max_kv), _int(window)))


# ---------------------------------------------------------------------------
# reference-surface modules (drop-in for GDNLayerCustom's ``exts`` dict)
# ---------------------------------------------------------------------------


class PrefillModule:
    """``prefill(q,k,v,A_log,a,dt_bias,b_logits,mask,state_in,scale) -> (out, state_out)``
    with the argument meaning of kernels/prefill_chunked.cu:422-433 (q,k,v [B,H,T,*]
    bf16; a,b_logits [B,H,T] bf16; dt_bias float; mask [B,T] f32; state_in empty =
    zeros).  Shape-generic: H, dk in {64,128}, dv in {64,128,256}, any T."""

    # the reference layer's shapes (gdn_layer.py:24-28); C_DIM is the chunk length
    H_DIM = 16
    K_DIM = 128
    V_DIM = 256
    C_DIM = CHUNK

    def prefill(self, q, k, v, A_log, a, dt_bias, b_logits, mask, state_in, scale):
        for name, t in (("q", q), ("k", k), ("v", v), ("a", a), ("b_logits", b_logits)):
            _need(t.is_cuda and t.is_contiguous() and t.dtype == torch.bfloat16,
                  f"{name}: contiguous bfloat16 CUDA required")
        s_in = state_in if (state_in is not None and state_in.numel() > 0) else None
        return prefill(q, k, v, A_log, a, b_logits, dt_bias=float(dt_bias), mask=mask, state_in=s_in,
                       scale=float(scale), layout="bhtd")


class DecodeModule:
    """``forward(q,k,v,a_sc,b_sc,A_log,dt_bias,S_in,scale,o_out,S_out) -> None``
    (kernels/decode.cu:172-214): q,k [B,H,K], v [B,H,V] bf16, a,b [B,H] bf16,
    A_log, dt_bias [H] f32, S_in/S_out [B,H,K,V] f32 (may alias), o_out [B,H,V] f32."""

    def forward(self, q, k, v, a_sc, b_sc, A_log, dt_bias, S_in, scale, o_out, S_out):
        for name, t in (("q", q), ("k", k), ("v", v), ("a_sc", a_sc), ("b_sc", b_sc), ("A_log", A_log),
                        ("dt_bias", dt_bias), ("S_in", S_in), ("o_out", o_out), ("S_out", S_out)):
            _need(t.is_cuda, f"{name} must be a CUDA tensor")
            _need(t.is_contiguous(), f"{name} must be contiguous")
        decode_step(q, k, v, a_sc, b_sc, A_log, dt_bias, S_in, scale=float(scale), out=o_out, state_out=S_out)


class ProjModule:
    """``forward(input [B,T,D], weight [D_out,D], conv_w [D_out,4]) -> [B,T,D_out]``
    bf16 (kernels/fused_proj_conv_silu.cu:298-355)."""

    def forward(self, input, weight, conv_w):
        _need(input.is_cuda and weight.is_cuda and conv_w.is_cuda, "all tensors must be on CUDA")
        _need(input.is_contiguous() and weight.is_contiguous() and conv_w.is_contiguous(),
              "all tensors must be contiguous")
        _need(input.dtype == torch.bfloat16 and weight.dtype == torch.bfloat16 and conv_w.dtype == torch.bfloat16,
              "all tensors must be bfloat16")
        _need(weight.shape[1] == input.shape[2], "weight dim-1 must equal D")
        _need(conv_w.shape[0] == weight.shape[0], "conv_w dim-0 must equal D_out")
        _need(conv_w.shape[1] == 4, "conv_w dim-1 must equal CONV_K")
        return proj_conv_silu(input, weight, conv_w)


class RMSNormModule:
    """``forward(x [R,D] bf16, gamma [D] bf16, eps, block_threads, rows_per_block)``
    (kernels/rmsnorm.cu:280-293).  The launch-shape arguments are validated like the
    reference's (:133-144) and otherwise unused; any D % 8 == 0 up to 8192 works."""

    def forward(self, x, gamma, eps, block_threads, rows_per_block):
        _need(x.is_cuda, "x must be CUDA")
        _need(gamma.is_cuda, "gamma must be CUDA")
        _need(x.dtype == torch.bfloat16, "x must be BF16")
        _need(gamma.dtype == torch.bfloat16, "gamma must be BF16")
        _need(x.dim() == 2, "x must be [R, D]")
        _need(gamma.dim() == 1 and gamma.shape[0] == x.shape[1], "gamma must be [D]")
        _need(x.is_contiguous() and gamma.is_contiguous(), "inputs must be contiguous")
        _need(rows_per_block >= 1, "rows_per_block must be >= 1")
        _need(32 <= block_threads <= 1024, "block_threads must be in [32, 1024]")
        _need(block_threads % rows_per_block == 0, "block_threads must be divisible by rows_per_block")
        tpr = block_threads // rows_per_block
        _need(tpr >= 32 and tpr % 32 == 0, "threads_per_row must be a multiple of 32")
        return rmsnorm(x, gamma, float(eps))


def exts() -> dict:
    """The ``exts`` dict of gdn_layer.GDNLayerCustom (gdn_layer.py:209-217)."""
    _lib.lib()  # fail loudly now if the library is missing
    return dict(rmsnorm=RMSNormModule(), proj=ProjModule(), prefill=PrefillModule(), decode=DecodeModule())
