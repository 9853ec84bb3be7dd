"""Tensor-level entry points over the C ABI (one function per kernel).

These take and return ``torch`` tensors on an AMD GPU and do nothing but
validate, allocate outputs and pass raw pointers to ``libdaisy_hip.so``.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import _lib

ATTN_SCALE = 0.12  # the reference's constant softmax scale (models/daisy/attention.py:88)


def _check_bf16(name: str, t: torch.Tensor, ndim: int) -> None:
    if t.dtype != torch.bfloat16:
        raise TypeError(f"{name} must be bfloat16, got {t.dtype}")
    if t.dim() != ndim:
        raise ValueError(f"{name} must have {ndim} dims, got shape {tuple(t.shape)}")
    if t.stride(-1) != 1:
        raise ValueError(f"{name} must be contiguous in its last dim")


def prefill_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
                      window: Optional[int], scale: float = ATTN_SCALE,
                      cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None,
                      doc_start: Optional[torch.Tensor] = None,
                      out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Sliding-window causal attention over ``[B, T, H, D]`` bf16 tensors.

    ``cos``/``sin`` (fp32 ``[>=T, D/2]``) rotate q and k inside the call;
    ``doc_start`` (int32 ``[T]``) confines each query to its document; ``window``
    counts the visible keys including the query itself (``None``/``<=0`` = full
    causal).  Returns ``(o, k_rot)``: ``o`` is ``[B, T, H, D]`` bf16 and ``k_rot``
    the rotated keys (``None`` without ``cos``/``sin``).

    Contract of ``doc_start``: ``0 <= doc_start[t] <= t`` and non-decreasing in ``t`` (the kernel
    picks the key tiles of a block of queries from the block's first row).  It is not checked
    here, since that would synchronise; ``check_doc_start`` does, for callers that want it.
    """
    fast = _lib.native().prefill_attention(q, k, v, 0 if window is None else int(window), float(scale), cos, sin, doc_start, out, k_out)
    if fast is not None:
        return fast
    dev = _lib.require_gpu(q, k, v, cos, sin, doc_start, out, k_out)
    for name, t in (("q", q), ("k", k), ("v", v)):
        _check_bf16(name, t, 4)
    B, T, H, D = q.shape
    if k.shape != q.shape or v.shape != q.shape:
        raise ValueError(f"q, k, v shapes differ: {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin must be given together")
    if cos is not None:
        for name, t in (("cos", cos), ("sin", sin)):
            if t.dtype != torch.float32 or t.dim() != 2 or t.shape[1] != D // 2 or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous fp32 [rows, {D // 2}] table, got {tuple(t.shape)} {t.dtype}")
            torch._assert(T <= t.shape[0], f"Rotary buffers too small {t.shape[0]} < {T}")
    if doc_start is not None:
        if doc_start.dtype != torch.int32 or doc_start.shape != (T,) or not doc_start.is_contiguous():
            raise ValueError("doc_start must be a contiguous int32 [T] tensor")
    if out is None:
        out = torch.empty((B, T, H, D), dtype=torch.bfloat16, device=dev)
    else:
        _check_bf16("out", out, 4)
    if cos is not None and k_out is None:
        k_out = torch.empty((B, T, H, D), dtype=torch.bfloat16, device=dev)
    if k_out is not None:
        _check_bf16("k_out", k_out, 4)
        if cos is None:
            raise ValueError("k_out is only produced when cos/sin are given")
    w = 0 if window is None else int(window)
    flags = 0
    lib = _lib.load()
    with _lib.on_device(dev):
        rc = lib.daisy_prefill_fwd(
            q.data_ptr(), _lib.strides(q, (0, 1, 2)),
            k.data_ptr(), _lib.strides(k, (0, 1, 2)),
            v.data_ptr(), _lib.strides(v, (0, 1, 2)),
            _lib.ptr(cos), _lib.ptr(sin), _lib.ptr(doc_start),
            out.data_ptr(), _lib.strides(out, (0, 1, 2)),
            _lib.ptr(k_out), None if k_out is None else _lib.strides(k_out, (0, 1, 2)),
            B, T, H, D, w, float(scale), flags, _lib.current_stream(dev))
    _lib.check(rc, "daisy_prefill_fwd")
    return out, k_out


def _check_f32(name: str, t: torch.Tensor, ndim: int) -> None:
    if t.dtype != torch.float32:
        raise TypeError(f"{name} must be float32, got {t.dtype}")
    if t.dim() != ndim:
        raise ValueError(f"{name} must have {ndim} dims, got shape {tuple(t.shape)}")
    if t.stride(-1) != 1:
        raise ValueError(f"{name} must be contiguous in its last dim")


def prefill_attention_f32(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
                          window: Optional[int], scale: float = ATTN_SCALE,
                          cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None,
                          doc_start: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``prefill_attention`` on fp32 ``[B, T, H, D]`` tensors with fp32 arithmetic (``daisy_prefill_fwd_f32``):
    the mode of a module with fp32 parameters.  Any even ``D <= 256``.  Returns fp32 ``(o, k_rot)``."""
    dev = _lib.require_gpu(q, k, v, cos, sin, doc_start)
    for name, t in (("q", q), ("k", k), ("v", v)):
        _check_f32(name, t, 4)
    B, T, H, D = q.shape
    if k.shape != q.shape or v.shape != q.shape:
        raise ValueError(f"q, k, v shapes differ: {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin must be given together")
    if cos is not None:
        for name, t in (("cos", cos), ("sin", sin)):
            if t.dtype != torch.float32 or t.dim() != 2 or t.shape[1] != D // 2 or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous fp32 [rows, {D // 2}] table, got {tuple(t.shape)} {t.dtype}")
            torch._assert(T <= t.shape[0], f"Rotary buffers too small {t.shape[0]} < {T}")
    if doc_start is not None:
        if doc_start.dtype != torch.int32 or doc_start.shape != (T,) or not doc_start.is_contiguous():
            raise ValueError("doc_start must be a contiguous int32 [T] tensor")
    out = torch.empty((B, T, H, D), dtype=torch.float32, device=dev)
    k_out = torch.empty((B, T, H, D), dtype=torch.float32, device=dev) if cos is not None else None
    d3 = (0, 1, 2)
    lib = _lib.load()
    with _lib.on_device(dev):
        rc = lib.daisy_prefill_fwd_f32(
            q.data_ptr(), _lib.strides(q, d3), k.data_ptr(), _lib.strides(k, d3), v.data_ptr(), _lib.strides(v, d3),
            _lib.ptr(cos), _lib.ptr(sin), _lib.ptr(doc_start),
            out.data_ptr(), _lib.strides(out, d3),
            _lib.ptr(k_out), None if k_out is None else _lib.strides(k_out, d3),
            B, T, H, D, 0 if window is None else int(window), float(scale), _lib.current_stream(dev))
    _lib.check(rc, "daisy_prefill_fwd_f32")
    return out, k_out


def decode_attention_f32(q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor,
                         k_rows: Optional[torch.Tensor], v_rows: Optional[torch.Tensor], *,
                         n_rows: int, new_idx: int, scale: float = ATTN_SCALE,
                         cos_row: Optional[torch.Tensor] = None, sin_row: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``decode_attention`` on fp32 tensors with fp32 arithmetic (``daisy_decode_fwd_f32``); the
    cache rows ``[B, H, rows, D]`` are only read."""
    dev = _lib.require_gpu(q, k_new, v_new, k_rows, v_rows, cos_row, sin_row)
    for name, t in (("q", q), ("k_new", k_new), ("v_new", v_new)):
        _check_f32(name, t, 3)
    B, H, D = q.shape
    if k_new.shape != q.shape or v_new.shape != q.shape:
        raise ValueError("q, k_new, v_new must all be [B, H, D]")
    if k_rows is not None:
        _check_f32("k_rows", k_rows, 4)
        _check_f32("v_rows", v_rows, 4)
    out = torch.empty((B, H, D), dtype=torch.float32, device=dev)
    lib = _lib.load()
    with _lib.on_device(dev):
        rc = lib.daisy_decode_fwd_f32(
            q.data_ptr(), _lib.strides(q, (0, 1)), k_new.data_ptr(), _lib.strides(k_new, (0, 1)),
            v_new.data_ptr(), _lib.strides(v_new, (0, 1)),
            _lib.ptr(k_rows), None if k_rows is None else _lib.strides(k_rows, (0, 1, 2)),
            _lib.ptr(v_rows), None if v_rows is None else _lib.strides(v_rows, (0, 1, 2)),
            _lib.ptr(cos_row), _lib.ptr(sin_row), out.data_ptr(), _lib.strides(out, (0, 1)),
            B, H, D, int(n_rows), int(new_idx), 0, float(scale), _lib.current_stream(dev))
    _lib.check(rc, "daisy_decode_fwd_f32")
    return out


def check_doc_start(doc_start: torch.Tensor) -> None:
    """Raises ``ValueError`` unless ``0 <= doc_start[t] <= t`` and ``doc_start`` does not decrease
    (the contract of ``prefill_attention``).  Synchronises with the device."""
    pos = torch.arange(doc_start.numel(), device=doc_start.device, dtype=doc_start.dtype)
    ok = (doc_start >= 0) & (doc_start <= pos)
    if doc_start.numel() > 1:
        ok[1:] &= doc_start[1:] >= doc_start[:-1]
    if not bool(ok.all()):
        raise ValueError("doc_start must satisfy 0 <= doc_start[t] <= t and must not decrease")


def decode_workspace_bytes(B: int, H: int, D: int, n_rows: int, nsplit: int = 0) -> int:
    return int(_lib.load().daisy_decode_workspace_bytes(B, H, D, n_rows, nsplit))


def decode_attention(q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor,
                     k_rows: Optional[torch.Tensor], v_rows: Optional[torch.Tensor], *,
                     n_rows: int, new_idx: int, write_back: bool,
                     scale: float = ATTN_SCALE,
                     cos_row: Optional[torch.Tensor] = None, sin_row: Optional[torch.Tensor] = None,
                     out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None,
                     nsplit: int = 0) -> torch.Tensor:
    """One decode step for every (batch, head).

    ``q``, ``k_new``, ``v_new``: bf16 ``[B, H, D]`` (any batch/head strides).
    ``k_rows``/``v_rows``: bf16 tensors addressed as ``[B, H, rows, D]`` through
    their strides (dims 0, 1, 2); logical rows ``0..n_rows-1`` are attended,
    except that row ``new_idx`` is taken from ``k_new``/``v_new`` (after RoPE
    with ``cos_row``/``sin_row``) and stored back when ``write_back``.
    Returns ``o`` bf16 ``[B, H, D]``.
    """
    dev = _lib.require_gpu(q, k_new, v_new, k_rows, v_rows, cos_row, sin_row, out, workspace)
    for name, t in (("q", q), ("k_new", k_new), ("v_new", v_new)):
        _check_bf16(name, t, 3)
    B, H, D = q.shape
    if k_new.shape != q.shape or v_new.shape != q.shape:
        raise ValueError("q, k_new, v_new must all be [B, H, D]")
    if k_rows is not None:
        _check_bf16("k_rows", k_rows, 4)
        _check_bf16("v_rows", v_rows, 4)
    if out is None:
        out = torch.empty((B, H, D), dtype=torch.bfloat16, device=dev)
    else:
        _check_bf16("out", out, 3)
    lib = _lib.load()
    need = int(lib.daisy_decode_workspace_bytes(B, H, D, n_rows, nsplit))
    if need > 0 and (workspace is None or workspace.numel() * workspace.element_size() < need):
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    ws_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    with _lib.on_device(dev):
        rc = lib.daisy_decode_fwd(
            q.data_ptr(), _lib.strides(q, (0, 1)),
            k_new.data_ptr(), _lib.strides(k_new, (0, 1)),
            v_new.data_ptr(), _lib.strides(v_new, (0, 1)),
            _lib.ptr(k_rows), None if k_rows is None else _lib.strides(k_rows, (0, 1, 2)),
            _lib.ptr(v_rows), None if v_rows is None else _lib.strides(v_rows, (0, 1, 2)),
            _lib.ptr(cos_row), _lib.ptr(sin_row),
            out.data_ptr(), _lib.strides(out, (0, 1)),
            B, H, D, int(n_rows), int(new_idx), 1 if write_back else 0,
            float(scale), int(nsplit),
            _lib.ptr(workspace), ws_bytes, _lib.current_stream(dev))
    _lib.check(rc, "daisy_decode_fwd")
    return out


def decode_attention_at(q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor,
                        k_ring: torch.Tensor, v_ring: torch.Tensor, pos: torch.Tensor, *,
                        scale: float = ATTN_SCALE, out: Optional[torch.Tensor] = None,
                        workspace: Optional[torch.Tensor] = None, nsplit: int = 0) -> torch.Tensor:
    """``decode_attention`` over a ring cache with the position in device memory.

    ``k_ring``/``v_ring``: bf16 ``[B, H, W, D]`` (slot order); ``pos``: one-element int32 device tensor
    holding ``t``, the number of positions already in the ring.  The kernel reads ``t`` when it
    runs, attends the ``min(t + 1, W)`` live rows and writes the new row (``k_new``, ``v_new``, already
    rotated) to slot ``t % W``; the launch can therefore be recorded in a HIP graph and replayed
    while the caller increments ``pos``.  Returns ``o`` bf16 ``[B, H, D]``.
    """
    dev = _lib.require_gpu(q, k_new, v_new, k_ring, v_ring, pos, out, workspace)
    for name, t in (("q", q), ("k_new", k_new), ("v_new", v_new)):
        _check_bf16(name, t, 3)
    _check_bf16("k_ring", k_ring, 4)
    _check_bf16("v_ring", v_ring, 4)
    B, H, D = q.shape
    if k_new.shape != q.shape or v_new.shape != q.shape:
        raise ValueError("q, k_new, v_new must all be [B, H, D]")
    W = k_ring.shape[2]
    if k_ring.shape != (B, H, W, D) or v_ring.shape != k_ring.shape:
        raise ValueError(f"k_ring, v_ring must be [B, H, W, D] = [{B}, {H}, W, {D}], got {tuple(k_ring.shape)}, {tuple(v_ring.shape)}")
    if pos.dtype != torch.int32 or pos.numel() != 1:
        raise ValueError("pos must be a one-element int32 tensor")
    if out is None:
        out = torch.empty((B, H, D), dtype=torch.bfloat16, device=dev)
    else:
        _check_bf16("out", out, 3)
    lib = _lib.load()
    need = int(lib.daisy_decode_workspace_bytes(B, H, D, W, nsplit))
    if need > 0 and (workspace is None or workspace.numel() * workspace.element_size() < need):
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    ws_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    with _lib.on_device(dev):
        rc = lib.daisy_decode_fwd_at(
            q.data_ptr(), _lib.strides(q, (0, 1)),
            k_new.data_ptr(), _lib.strides(k_new, (0, 1)),
            v_new.data_ptr(), _lib.strides(v_new, (0, 1)),
            k_ring.data_ptr(), _lib.strides(k_ring, (0, 1, 2)),
            v_ring.data_ptr(), _lib.strides(v_ring, (0, 1, 2)),
            out.data_ptr(), _lib.strides(out, (0, 1)),
            B, H, D, int(W), pos.data_ptr(), float(scale), int(nsplit),
            _lib.ptr(workspace), ws_bytes, _lib.current_stream(dev))
    _lib.check(rc, "daisy_decode_fwd_at")
    return out


def attn_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_ring: torch.Tensor, v_ring: torch.Tensor,
              pos: Union[int, torch.Tensor], *, cos: torch.Tensor, sin: torch.Tensor, eps: float,
              ve: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
              scale: float = ATTN_SCALE, out: Optional[torch.Tensor] = None,
              workspace: Optional[torch.Tensor] = None, nsplit: int = 0,
              status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The attention part of one decode step in one launch (``daisy_attn_step_fwd``).

    ``q``, ``k``, ``v``: the new token's rows of the QKV projection output, bf16 ``[B, H, D]`` views;
    the kernel normalises them, rotates q and k with row ``pos`` of ``cos``/``sin`` (fp32
    ``[rows, D/2]``), mixes ``v`` with ``ve [B, H, D]`` through ``gate`` (one fp32), writes the new rows
    into slot ``pos % W`` of ``k_ring``/``v_ring [B, H, W, D]`` (bf16 or fp16) and attends the live rows.  ``pos`` is an
    int or a one-element int32 device tensor (read when the kernel runs).  Returns ``o [B, H, D]``.

    ``status``: one-element int32 device tensor.  A device position past the rotary tables cannot
    be refused on the host; the kernel then writes NaN outputs and raises bit
    ``_lib.STATUS_POSITION_PAST_TABLES`` in ``status`` (see ``raise_for_status``).
    """
    pos_dev = pos if isinstance(pos, torch.Tensor) else None
    dev = _lib.require_gpu(q, k, v, k_ring, v_ring, cos, sin, ve, gate, pos_dev, out, workspace, status)
    _check_status(status)
    for name, t in (("q", q), ("k", k), ("v", v)):
        _check_bf16(name, t, 3)
    if k_ring.dtype == torch.float16 and v_ring.dtype == torch.float16 and k_ring.dim() == 4 and k_ring.stride(-1) == 1 \
            and v_ring.stride(-1) == 1:
        ring_f16 = True       # the reference generator's default cache dtype
    else:
        ring_f16 = False
        _check_bf16("k_ring", k_ring, 4)
        _check_bf16("v_ring", v_ring, 4)
    B, H, D = q.shape
    if k.shape != q.shape or v.shape != q.shape:
        raise ValueError("q, k, v must all be [B, H, D]")
    W = k_ring.shape[2]
    if k_ring.shape != (B, H, W, D) or v_ring.shape != k_ring.shape:
        raise ValueError(f"k_ring, v_ring must be [{B}, {H}, W, {D}], got {tuple(k_ring.shape)}, {tuple(v_ring.shape)}")
    for name, t in (("cos", cos), ("sin", sin)):
        if t.dtype != torch.float32 or t.dim() != 2 or t.shape[1] != D // 2 or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous fp32 [rows, {D // 2}] table, got {tuple(t.shape)} {t.dtype}")
    if pos_dev is not None:
        if pos_dev.dtype != torch.int32 or pos_dev.numel() != 1:
            raise ValueError("a device position must be a one-element int32 tensor")
        live = W
    else:
        torch._assert(0 <= pos < cos.shape[0], f"Rotary buffers too small {cos.shape[0]} < {pos + 1}")
        live = min(int(pos) + 1, W)
    if (ve is None) != (gate is None):
        raise ValueError("ve and gate must be given together")
    if ve is not None:
        _check_bf16("ve", ve, 3)
        if ve.shape != q.shape or gate.dtype != torch.float32 or gate.numel() != 1:
            raise ValueError("ve must be [B, H, D] and gate a one-element fp32 tensor")
    if out is None:
        out = torch.empty((B, H, D), dtype=torch.bfloat16, device=dev)
    else:
        _check_bf16("out", out, 3)
    lib = _lib.load()
    need = int(lib.daisy_decode_workspace_bytes(B, H, D, live, nsplit))
    if need > 0 and (workspace is None or workspace.numel() * workspace.element_size() < need):
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    ws_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    d2 = (0, 1)
    with _lib.on_device(dev):
        rc = lib.daisy_attn_step_fwd(
            q.data_ptr(), _lib.strides(q, d2), k.data_ptr(), _lib.strides(k, d2), v.data_ptr(), _lib.strides(v, d2),
            _lib.ptr(ve), None if ve is None else _lib.strides(ve, d2), _lib.ptr(gate),
            cos.data_ptr(), sin.data_ptr(), int(cos.shape[0]),
            0 if pos_dev is not None else int(pos), _lib.ptr(pos_dev), _lib.ptr(status), float(eps),
            k_ring.data_ptr(), _lib.strides(k_ring, (0, 1, 2)), v_ring.data_ptr(), _lib.strides(v_ring, (0, 1, 2)),
            1 if ring_f16 else 0,
            out.data_ptr(), _lib.strides(out, d2), B, H, D, int(W), float(scale), int(nsplit),
            _lib.ptr(workspace), ws_bytes, _lib.current_stream(dev))
    _lib.check(rc, "daisy_attn_step_fwd")
    return out


def attn_layer_step(x: torch.Tensor, w_qkv: torch.Tensor, w_out: torch.Tensor, k_ring: torch.Tensor,
                    v_ring: torch.Tensor, pos: Union[int, torch.Tensor], *, cos: torch.Tensor, sin: torch.Tensor,
                    eps: float, ve: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
                    scale: float = ATTN_SCALE, nsplit: int = 0, status: Optional[torch.Tensor] = None,
                    workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One decode step of an attention layer in one call (``daisy_attn_layer_step_fwd``): QKV projection of
    ``x [B, dim]`` (or ``[B, 1, dim]``) with ``w_qkv [3*H*D, dim]``, the one-launch attention step of ``attn_step`` on
    the rings ``[B, H, W, D]``, output projection with ``w_out [dim, H*D]``.  bf16 throughout (the rings may be fp16),
    ``B`` at most ``_lib.LINEAR_MAX_ROWS``.  Returns ``y`` shaped like ``x``.  Same results as ``linear_rows``,
    ``attn_step``, ``linear_rows`` one after the other; what it saves is the host's time between the launches."""
    pos_dev = pos if isinstance(pos, torch.Tensor) else None
    dev = _lib.require_gpu(x, w_qkv, w_out, k_ring, v_ring, cos, sin, ve, gate, pos_dev, status, workspace)
    _check_status(status)
    if x.dtype != torch.bfloat16 or w_qkv.dtype != torch.bfloat16 or w_out.dtype != torch.bfloat16:
        raise TypeError("attn_layer_step: x, w_qkv and w_out must be bf16")
    if k_ring.dtype != v_ring.dtype or k_ring.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"attn_layer_step: the rings must both be bf16 or both fp16, got {k_ring.dtype}, {v_ring.dtype}")
    if k_ring.dim() != 4 or v_ring.shape != k_ring.shape or k_ring.stride(3) != 1 or v_ring.stride(3) != 1:
        raise ValueError("attn_layer_step: k_ring, v_ring must be [B, H, W, D] with a contiguous last dim")
    B, H, W, D = k_ring.shape
    dim = x.shape[-1]
    if x.numel() != B * dim or w_qkv.shape != (3 * H * D, dim) or w_out.shape != (dim, H * D):
        raise ValueError(f"attn_layer_step: x {tuple(x.shape)}, w_qkv {tuple(w_qkv.shape)}, w_out {tuple(w_out.shape)} do not "
                         f"fit rings of {B} x {H} x {D}")
    if not (x.is_contiguous() and w_qkv.stride(1) == 1 and w_out.stride(1) == 1):
        raise ValueError("attn_layer_step: x must be contiguous and the weights' last dims contiguous")
    for name, t in (("cos", cos), ("sin", sin)):
        if t.dtype != torch.float32 or t.dim() != 2 or t.shape[1] != D // 2 or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous fp32 [rows, {D // 2}] table, got {tuple(t.shape)} {t.dtype}")
    if pos_dev is not None:
        if pos_dev.dtype != torch.int32 or pos_dev.numel() != 1:
            raise ValueError("a device position must be a one-element int32 tensor")
    else:
        torch._assert(0 <= pos < cos.shape[0], f"Rotary buffers too small {cos.shape[0]} < {pos + 1}")
    if (ve is None) != (gate is None):
        raise ValueError("ve and gate must be given together")
    ve_strides = None
    if ve is not None:
        if ve.dtype != torch.bfloat16 or ve.shape != (B, H, D) or ve.stride(2) != 1:
            raise ValueError(f"ve must be bf16 [{B}, {H}, {D}] with a contiguous last dim, got {tuple(ve.shape)} {ve.dtype}")
        if gate.dtype != torch.float32 or gate.numel() != 1:
            raise ValueError("gate must be a one-element fp32 tensor")
        ve_strides = _lib.strides(ve, (0, 1))
    lib = _lib.load()
    need = int(lib.daisy_attn_layer_step_workspace_bytes(B, H, D, W, nsplit))
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    y = torch.empty_like(x)
    with _lib.on_device(dev):
        rc = lib.daisy_attn_layer_step_fwd(
            x.data_ptr(), dim, w_qkv.data_ptr(), w_qkv.stride(0), w_out.data_ptr(), w_out.stride(0),
            _lib.ptr(ve), ve_strides, _lib.ptr(gate), cos.data_ptr(), sin.data_ptr(), int(cos.shape[0]),
            0 if pos_dev is not None else int(pos), _lib.ptr(pos_dev), _lib.ptr(status), float(eps),
            k_ring.data_ptr(), _lib.strides(k_ring, (0, 1, 2)), v_ring.data_ptr(), _lib.strides(v_ring, (0, 1, 2)),
            1 if k_ring.dtype == torch.float16 else 0, y.data_ptr(), dim, B, H, D, dim, W, float(scale), int(nsplit),
            workspace.data_ptr(), workspace.numel() * workspace.element_size(), _lib.current_stream(dev))
    _lib.check(rc, "daisy_attn_layer_step_fwd")
    return y


def _check_status(status: Optional[torch.Tensor]) -> None:
    if status is not None and (status.dtype != torch.int32 or status.numel() != 1):
        raise ValueError("status must be a one-element int32 tensor")


def raise_for_status(status: torch.Tensor) -> None:
    """Reads a status word (synchronises) and raises what the kernels reported in it."""
    bits = int(status.item())
    if bits & _lib.STATUS_POSITION_PAST_TABLES:
        raise RuntimeError("a decode step ran at a position past the rotary tables (Rotary buffers too small); "
                           "its outputs are NaN")
    if bits & _lib.STATUS_LENGTH_PAST_PAGES:
        raise RuntimeError("a length or position of a paged call lies past what the page table has room for; its outputs are NaN")
    if bits & _lib.STATUS_PAGE_OUT_OF_RANGE:
        raise RuntimeError("a paged call needed a page table entry that names no page of the pool; its outputs are NaN")
    if bits & _lib.STATUS_INDEX_OUT_OF_ORDER:
        raise RuntimeError("an index of rows to be moved in a paged cache does not rise; its sequence is as it was")


def kda_workspace_bytes(B: int, T: int, H: int, Dk: int, Dv: int, chunk: int = 64) -> int:
    return int(_lib.load().daisy_kda_workspace_bytes(B, T, H, Dk, Dv, chunk))


def _check_cu_seqlens(cu_seqlens: torch.Tensor, B: int) -> int:
    """Validates what the host can see of packed-sequence bounds; returns the sequence count."""
    if B != 1:
        raise ValueError("cu_seqlens needs batch size 1 (sequences packed along T)")
    if cu_seqlens.dtype != torch.int32 or cu_seqlens.dim() != 1 or cu_seqlens.numel() < 2 or not cu_seqlens.is_contiguous():
        raise ValueError("cu_seqlens must be a contiguous int32 [n_seq + 1] tensor")
    return cu_seqlens.numel() - 1


def _kda_inputs(q, k, v, g, beta, initial_state, n_states, scale, fresh_state_copy=True):
    for name, t in (("q", q), ("k", k), ("v", v)):
        _check_bf16(name, t, 4)
    B, T, H, Dk = q.shape
    Dv = v.shape[-1]
    if k.shape != q.shape or g.shape != q.shape or v.shape[:3] != q.shape[:3] or beta.shape != (B, T, H):
        raise ValueError("kda: expected q,k,g [B,T,H,Dk], v [B,T,H,Dv], beta [B,T,H]")
    if g.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"g must be fp32 or bf16, got {g.dtype}")
    q, k, v, g = q.contiguous(), k.contiguous(), v.contiguous(), g.contiguous()
    beta = beta.to(torch.float32).contiguous()
    if scale is None:
        scale = Dk ** -0.5
    if initial_state is not None:
        if initial_state.shape != (n_states, H, Dk, Dv):
            raise ValueError(f"initial_state must be [{n_states},H,Dk,Dv], got {tuple(initial_state.shape)}")
        if fresh_state_copy:
            initial_state = initial_state.to(torch.float32).contiguous()
    return q, k, v, g, beta, initial_state, scale


def kda_chunk_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor, *,
                  scale: Optional[float] = None, initial_state: Optional[torch.Tensor] = None,
                  output_final_state: bool = False, use_qk_l2norm_in_kernel: bool = True,
                  l2_eps: float = 1e-6, chunk: int = 64, cu_seqlens: Optional[torch.Tensor] = None,
                  workspace: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Chunked KDA forward; see ``daisy_kda_chunk_fwd`` / ``daisy_kda_chunk_varlen_fwd`` in ``include/daisy_hip.h``.

    ``cu_seqlens`` (int32 ``[N + 1]`` on the GPU, from 0 to T, non-decreasing): the batch is 1 and
    holds N sequences packed along T, each with its own state ``[N, H, Dk, Dv]``.  The kernels read
    the bounds on the device; the host never does, so the call does not synchronise.
    """
    if workspace is None and chunk == 64:
        fast = _lib.native().kda_chunk(q, k, v, g, beta, scale, initial_state, bool(output_final_state), bool(use_qk_l2norm_in_kernel),
                                       float(l2_eps), cu_seqlens)
        if fast is not None:
            return fast
    dev = _lib.require_gpu(q, k, v, g, beta, initial_state, workspace, cu_seqlens)
    B, T, H, Dk = q.shape
    Dv = v.shape[-1]
    n_seq = _check_cu_seqlens(cu_seqlens, B) if cu_seqlens is not None else 0
    n_states = n_seq if n_seq else B
    q, k, v, g, beta, initial_state, scale = _kda_inputs(q, k, v, g, beta, initial_state, n_states, scale)
    o = torch.empty((B, T, H, Dv), dtype=torch.bfloat16, device=dev)
    final = torch.empty((n_states, H, Dk, Dv), dtype=torch.float32, device=dev) if output_final_state else None
    lib = _lib.load()
    if n_seq:
        need = int(lib.daisy_kda_varlen_workspace_bytes(T, n_seq, H, Dk, Dv, chunk))
    else:
        need = int(lib.daisy_kda_workspace_bytes(B, T, H, Dk, Dv, chunk))
    if need > 0 and (workspace is None or workspace.numel() * workspace.element_size() < need):
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    ws_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    head = (q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), 1 if g.dtype == torch.bfloat16 else 0, beta.data_ptr())
    tail = (int(chunk), float(scale), 1 if use_qk_l2norm_in_kernel else 0, float(l2_eps),
            _lib.ptr(workspace), ws_bytes, _lib.current_stream(dev))
    with _lib.on_device(dev):
        if n_seq:
            rc = lib.daisy_kda_chunk_varlen_fwd(*head, cu_seqlens.data_ptr(), n_seq, _lib.ptr(initial_state), o.data_ptr(),
                                                _lib.ptr(final), T, H, Dk, Dv, *tail)
        else:
            rc = lib.daisy_kda_chunk_fwd(*head, _lib.ptr(initial_state), o.data_ptr(), _lib.ptr(final), B, T, H, Dk, Dv, *tail)
    _lib.check(rc, "daisy_kda_chunk_fwd")
    return o, final


def kda_recurrent_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor, *,
                      scale: Optional[float] = None, initial_state: Optional[torch.Tensor] = None,
                      output_final_state: bool = True, use_qk_l2norm_in_kernel: bool = True,
                      l2_eps: float = 1e-6, inplace_state: bool = False,
                      cu_seqlens: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Token-by-token KDA with the state in registers; see ``daisy_kda_recurrent_fwd``.

    With ``inplace_state`` the final state overwrites ``initial_state`` (which must then be a
    contiguous fp32 ``[B, H, Dk, Dv]`` tensor) and is returned as such -- the decode loop's mode.
    ``cu_seqlens``: packed sequences as in ``kda_chunk_fwd``.
    """
    dev = _lib.require_gpu(q, k, v, g, beta, initial_state, cu_seqlens)
    B, T, H, Dk = q.shape
    Dv = v.shape[-1]
    n_seq = _check_cu_seqlens(cu_seqlens, B) if cu_seqlens is not None else 0
    n_states = n_seq if n_seq else B
    if inplace_state:
        if initial_state is None:
            raise ValueError("inplace_state needs an initial_state")
        if initial_state.dtype != torch.float32 or not initial_state.is_contiguous():
            raise ValueError("inplace_state needs a contiguous fp32 initial_state")
    q, k, v, g, beta, initial_state, scale = _kda_inputs(q, k, v, g, beta, initial_state, n_states, scale,
                                                         fresh_state_copy=not inplace_state)
    o = (torch.zeros if n_seq else torch.empty)((B, T, H, Dv), dtype=torch.bfloat16, device=dev)
    if inplace_state:
        final = initial_state
    else:
        final = torch.empty((n_states, H, Dk, Dv), dtype=torch.float32, device=dev) if output_final_state else None
    lib = _lib.load()
    head = (q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), 1 if g.dtype == torch.bfloat16 else 0, beta.data_ptr())
    tail = (float(scale), 1 if use_qk_l2norm_in_kernel else 0, float(l2_eps), _lib.current_stream(dev))
    with _lib.on_device(dev):
        if n_seq:
            rc = lib.daisy_kda_recurrent_varlen_fwd(*head, cu_seqlens.data_ptr(), n_seq, _lib.ptr(initial_state), o.data_ptr(),
                                                    _lib.ptr(final), T, H, Dk, Dv, *tail)
        else:
            rc = lib.daisy_kda_recurrent_fwd(*head, _lib.ptr(initial_state), o.data_ptr(), _lib.ptr(final), B, T, H, Dk, Dv, *tail)
    _lib.check(rc, "daisy_kda_recurrent_fwd")
    return o, final


def kda_gate_fwd(g: torch.Tensor, A_log: torch.Tensor, head_k_dim: int,
                 g_bias: Optional[torch.Tensor] = None, beta: float = 1.0, threshold: float = 20.0) -> torch.Tensor:
    """``-exp(A_log[h]) * softplus(g + bias)``; ``g [..., H*Dk]`` -> ``[..., H, Dk]`` in ``g.dtype``."""
    dev = _lib.require_gpu(g, A_log, g_bias)
    if g.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"g must be fp32 or bf16, got {g.dtype}")
    last = g.shape[-1]
    if last % head_k_dim != 0:
        raise RuntimeError("last dim must be divisible by head_k_dim")
    H = last // head_k_dim
    if A_log.numel() != H:
        raise RuntimeError(f"A_log must be shape [H] or [1,1,H,1]; got {tuple(A_log.shape)} with H={H}")
    a = A_log.detach().reshape(H).to(device=dev, dtype=torch.float32).contiguous()
    bias = None
    if g_bias is not None:
        b = g_bias.detach().to(device=dev, dtype=torch.float32)
        if b.numel() == H * head_k_dim:
            bias = b.reshape(H, head_k_dim).contiguous()
        elif b.numel() == H:
            bias = b.reshape(H, 1).expand(H, head_k_dim).contiguous()
        else:
            raise RuntimeError(f"g_bias must be one of [(H*D,), (H,D), (1,1,H,D), (H,)]; got {tuple(b.shape)}")
    gc = g.contiguous()
    out = torch.empty((*g.shape[:-1], H, head_k_dim), dtype=g.dtype, device=dev)
    rows = gc.numel() // last
    lib = _lib.load()
    with _lib.on_device(dev):
        rc = lib.daisy_kda_gate_fwd(gc.data_ptr(), a.data_ptr(), _lib.ptr(bias), out.data_ptr(),
                                    rows, H, head_k_dim, 1 if g.dtype == torch.bfloat16 else 0,
                                    float(beta), float(threshold), _lib.current_stream(dev))
    _lib.check(rc, "daisy_kda_gate_fwd")
    return out


def linear_rows_ok(x: torch.Tensor, weight: torch.Tensor) -> bool:
    """Whether ``linear_rows`` takes this pair: bf16 on a GPU, at most ``_lib.LINEAR_MAX_ROWS`` rows of ``x``,
    rows of both starting on 16-byte boundaries."""
    if not (x.is_cuda and weight.is_cuda and x.dtype == torch.bfloat16 and weight.dtype == torch.bfloat16):
        return False
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1] or weight.shape[1] % 8 != 0:
        return False
    rows = x.numel() // x.shape[-1] if x.shape[-1] else 0
    if not 1 <= rows <= _lib.LINEAR_MAX_ROWS:
        return False
    return weight.stride(1) == 1 and weight.stride(0) % 8 == 0 and weight.data_ptr() % 16 == 0


def linear_rows(x: torch.Tensor, weight: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``F.linear(x, weight)`` for the few activation rows of a decode step (``daisy_linear_rows_fwd``):
    ``x [..., K]`` bf16 with at most ``_lib.LINEAR_MAX_ROWS`` rows in all, ``weight [N, K]`` bf16 (rows may be
    strided); returns ``[..., N]`` bf16.  Reads the weights once; fp32 accumulation, one rounding."""
    dev = _lib.require_gpu(x, weight, out)
    if x.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16:
        raise TypeError(f"linear_rows: x and weight must be bf16, got {x.dtype}, {weight.dtype}")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"linear_rows: x [..., K] and weight [N, K] do not fit: {tuple(x.shape)}, {tuple(weight.shape)}")
    if weight.stride(1) != 1:
        raise ValueError("linear_rows: the weight's last dim must be contiguous")
    N, K = weight.shape
    x2 = x.reshape(-1, K)
    if x2.stride(1) != 1 or (x2.size(0) > 1 and x2.stride(0) % 8 != 0) or x2.data_ptr() % 16 != 0:
        x2 = x2.contiguous()
    M = x2.size(0)
    if out is None:
        out = torch.empty(*x.shape[:-1], N, dtype=torch.bfloat16, device=dev)
    elif out.dtype != torch.bfloat16 or out.shape != (*x.shape[:-1], N) or not out.is_contiguous():
        raise ValueError(f"linear_rows: out must be a contiguous bf16 {(*x.shape[:-1], N)} tensor")
    lib = _lib.load()
    with _lib.on_device(dev):
        rc = lib.daisy_linear_rows_fwd(x2.data_ptr(), x2.stride(0) if M > 1 else K, weight.data_ptr(), weight.stride(0),
                                       out.data_ptr(), N, M, N, K, _lib.current_stream(dev))
    _lib.check(rc, "daisy_linear_rows_fwd")
    return out


def qkv_prep(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, eps: float,
             cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None,
             pos0: Union[int, torch.Tensor] = 0,
             ve: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
             q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None,
             v_out: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None
             ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """RMS norm of q, k, v + RoPE of q, k at rows ``pos0 + t`` + ``gate*v + (1-gate)*ve`` in one pass.

    ``q``, ``k``, ``v`` (and ``ve``) are bf16 ``[B, T, H, D]`` tensors or views with a
    contiguous last dim; ``gate`` is a one-element fp32 tensor holding the (bf16-rounded)
    sigmoid of the gate logit.  Outputs default to new contiguous ``[B, T, H, D]`` tensors;
    any strided bf16 ``[B, T, H, D]`` view may be passed instead.

    ``pos0`` may be a one-element int32 device tensor: the kernel then reads the position when
    it runs (a launch recorded in a HIP graph follows the tensor's value from replay to replay);
    ``pos0 + T`` beyond the tables cannot be refused here: the kernel then writes NaN for the rotated
    outputs and raises ``_lib.STATUS_POSITION_PAST_TABLES`` in ``status`` (one-element int32 tensor).
    """
    pos_dev = pos0 if isinstance(pos0, torch.Tensor) else None
    if pos_dev is not None:
        if pos_dev.dtype != torch.int32 or pos_dev.numel() != 1:
            raise ValueError("a device position must be a one-element int32 tensor")
        if cos is None:
            raise ValueError("a device position needs the rotary tables")
        pos0 = 0
    dev = _lib.require_gpu(q, k, v, ve, gate, cos, sin, q_out, k_out, v_out, pos_dev, status)
    _check_status(status)
    for name, t in (("q", q), ("k", k), ("v", v)):
        _check_bf16(name, t, 4)
    B, T, H, D = q.shape
    if k.shape != q.shape or v.shape != q.shape:
        raise ValueError(f"q, k, v shapes differ: {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin must be given together")
    if cos is not None:
        for name, t in (("cos", cos), ("sin", sin)):
            if t.dtype != torch.float32 or t.dim() != 2 or t.shape[1] != D // 2 or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous fp32 [rows, {D // 2}] table, got {tuple(t.shape)} {t.dtype}")
            torch._assert(pos0 + T <= t.shape[0], f"Rotary buffers too small {t.shape[0]} < {pos0 + T}")
    if (ve is None) != (gate is None):
        raise ValueError("ve and gate must be given together")
    if ve is not None:
        _check_bf16("ve", ve, 4)
        if ve.shape != q.shape:
            raise ValueError(f"ve must have shape {tuple(q.shape)}, got {tuple(ve.shape)}")
        if gate.dtype != torch.float32 or gate.numel() != 1:
            raise ValueError("gate must be a one-element fp32 tensor")
    outs = []
    for name, t in (("q_out", q_out), ("k_out", k_out), ("v_out", v_out)):
        if t is None:
            t = torch.empty((B, T, H, D), dtype=torch.bfloat16, device=dev)
        else:
            _check_bf16(name, t, 4)
            if t.shape != q.shape:
                raise ValueError(f"{name} must have shape {tuple(q.shape)}, got {tuple(t.shape)}")
        outs.append(t)
    qo, ko, vo = outs
    d3 = (0, 1, 2)
    lib = _lib.load()
    ins = (q.data_ptr(), _lib.strides(q, d3), k.data_ptr(), _lib.strides(k, d3), v.data_ptr(), _lib.strides(v, d3),
           _lib.ptr(ve), None if ve is None else _lib.strides(ve, d3), _lib.ptr(gate), _lib.ptr(cos), _lib.ptr(sin))
    outs = (qo.data_ptr(), _lib.strides(qo, d3), ko.data_ptr(), _lib.strides(ko, d3), vo.data_ptr(), _lib.strides(vo, d3),
            B, T, H, D, float(eps))
    with _lib.on_device(dev):
        if pos_dev is None:
            rc = lib.daisy_qkv_prep_fwd(*ins, int(pos0), *outs, _lib.current_stream(dev))
        else:
            rc = lib.daisy_qkv_prep_fwd_at(*ins, pos_dev.data_ptr(), int(cos.shape[0]), _lib.ptr(status), *outs,
                                           _lib.current_stream(dev))
    _lib.check(rc, "daisy_qkv_prep_fwd")
    return qo, ko, vo


def short_conv(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
               cache: Optional[torch.Tensor] = None, output_final_state: bool = False,
               activation: Optional[str] = "silu", inplace_cache: bool = False,
               cu_seqlens: Optional[torch.Tensor] = None
               ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Depthwise causal convolution over time + SiLU for ``x [B, T, C]`` bf16 (``daisy_short_conv_fwd``).

    ``weight [C, 1, K]`` or ``[C, K]``; ``cache [B, C, K]`` holds the last K inputs of the sequence
    so far.  Returns ``(y [B, T, C], new cache or None)``.  ``inplace_cache``: the new window is
    written into ``cache`` itself (bf16, contiguous, ``T <= 32``: decode steps) and ``cache`` is returned.
    ``cu_seqlens`` (int32 ``[N + 1]`` on the GPU): ``B == 1`` and N sequences are packed along T; no tap
    reaches across the start of its sequence and the windows are ``[N, C, K]`` (``daisy_short_conv_varlen_fwd``).
    """
    dev = _lib.require_gpu(x, weight, bias, cache, cu_seqlens)
    _check_bf16("x", x, 3)
    B, T, C = x.shape
    n_seq = _check_cu_seqlens(cu_seqlens, B) if cu_seqlens is not None else 0
    n_win = n_seq if n_seq else B
    w = weight.reshape(C, -1)
    K = w.shape[1]
    if w.dtype != torch.bfloat16 or (bias is not None and bias.dtype != torch.bfloat16):
        raise TypeError("short_conv: weight and bias must be bf16")
    if activation not in (None, "silu"):
        raise ValueError(f"short_conv: activation {activation!r} not supported")
    if x.stride(2) != 1:
        x = x.contiguous()
    w = w.contiguous()
    if cache is not None:
        if cache.shape != (n_win, C, K):
            raise ValueError(f"short_conv: cache must be [{n_win}, {C}, {K}], got {tuple(cache.shape)}")
        if inplace_cache and (cache.dtype != torch.bfloat16 or not cache.is_contiguous()):
            raise ValueError("short_conv: a window updated in place must be a contiguous bf16 tensor")
        cache = cache.to(torch.bfloat16).contiguous()
    elif inplace_cache:
        raise ValueError("short_conv: inplace_cache needs a cache")
    y = torch.empty(B, T, C, dtype=torch.bfloat16, device=dev)
    if inplace_cache:
        new_cache = cache
    else:
        new_cache = torch.empty(n_win, C, K, dtype=torch.bfloat16, device=dev) if output_final_state else None
    lib = _lib.load()
    if n_seq:
        if inplace_cache:
            raise ValueError("short_conv: inplace_cache does not combine with cu_seqlens")
        if bias is not None:
            bias = bias.contiguous()
        with _lib.on_device(dev):
            rc = lib.daisy_short_conv_varlen_fwd(x.data_ptr(), x.stride(1), w.data_ptr(), _lib.ptr(bias),
                                                 cu_seqlens.data_ptr(), n_seq, _lib.ptr(cache),
                                                 y.data_ptr(), y.stride(1), _lib.ptr(new_cache),
                                                 T, C, K, 1 if activation == "silu" else 0, _lib.current_stream(dev))
        _lib.check(rc, "daisy_short_conv_varlen_fwd")
        return y, new_cache
    with _lib.on_device(dev):
        rc = lib.daisy_short_conv_fwd(x.data_ptr(), _lib.strides(x, (0, 1)), w.data_ptr(), _lib.ptr(bias), _lib.ptr(cache),
                                      y.data_ptr(), _lib.strides(y, (0, 1)), _lib.ptr(new_cache),
                                      B, T, C, K, 1 if activation == "silu" else 0, _lib.current_stream(dev))
    _lib.check(rc, "daisy_short_conv_fwd")
    return y, new_cache


def gated_rmsnorm(x: torch.Tensor, gate: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5) -> torch.Tensor:
    """``x * rsqrt(mean(x^2) + eps) * weight * sigmoid(gate)`` over the last dim (64 or 128), bf16."""
    dev = _lib.require_gpu(x, gate, weight)
    if x.dtype != torch.bfloat16 or gate.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16:
        raise TypeError("gated_rmsnorm: x, gate and weight must be bf16")
    if gate.shape != x.shape or weight.numel() != x.shape[-1]:
        raise ValueError(f"gated_rmsnorm: shapes {tuple(x.shape)}, {tuple(gate.shape)}, {tuple(weight.shape)} do not match")
    xc, gc, wc = x.contiguous(), gate.contiguous(), weight.contiguous()
    out = torch.empty_like(xc)
    D = x.shape[-1]
    lib = _lib.load()
    with _lib.on_device(dev):
        rc = lib.daisy_gated_rmsnorm_fwd(xc.data_ptr(), gc.data_ptr(), wc.data_ptr(), out.data_ptr(),
                                         xc.numel() // D, D, float(eps), _lib.current_stream(dev))
    _lib.check(rc, "daisy_gated_rmsnorm_fwd")
    return out


# ----------------------------------------------------------------------------------------------
# sequences of unequal length: a paged cache, and the logits of a batch of requests
# ----------------------------------------------------------------------------------------------
_HALF_TYPES = (torch.bfloat16, torch.float16)


def _no_autograd(what: str, *tensors: Optional[torch.Tensor]) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{what} has no backward: call it under torch.no_grad() or with tensors that need no gradient")


def _check_rows(name: str, t: torch.Tensor, ndim: int, dtypes) -> None:
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d)[6:] for d in dtypes)}, got {t.dtype}")
    if t.dim() != ndim:
        raise ValueError(f"{name} must have {ndim} dims, got shape {tuple(t.shape)}")
    if t.stride(-1) != 1:
        raise ValueError(f"{name} must be contiguous in its last dim")


def _check_index(name: str, t: torch.Tensor, n: int) -> None:
    if t.dtype != torch.int32 or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 [{n}] tensor, got {tuple(t.shape)} {t.dtype}")


def _check_pages(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor) -> Tuple[int, int, int, int]:
    """Validates what the host can see of a paged cache; returns (pages, H, page size, D)."""
    _check_rows("k_pages", k_pages, 4, _HALF_TYPES)
    _check_rows("v_pages", v_pages, 4, (k_pages.dtype,))
    if v_pages.shape != k_pages.shape or 0 in k_pages.shape:
        raise ValueError(f"k_pages, v_pages must be [pages, H, page_size, D], got {tuple(k_pages.shape)}, {tuple(v_pages.shape)}")
    if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.shape[1] == 0 or page_table.stride(1) != 1:
        raise ValueError(f"page_table must be an int32 [sequences, pages] tensor, contiguous in its last dim, got {tuple(page_table.shape)} {page_table.dtype}")
    return tuple(k_pages.shape)


def paged_append(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                 positions: torch.Tensor, *, rows: Optional[torch.Tensor] = None, q: Optional[torch.Tensor] = None,
                 cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None, eps: Optional[float] = None,
                 ve: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None,
                 k_out: Optional[torch.Tensor] = None, v_out: Optional[torch.Tensor] = None,
                 status: Optional[torch.Tensor] = None, slots: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Appends keys and values to a paged cache, preparing them (and the queries) on the way, in one launch.

    ``k``, ``v`` ``[N, H, D]`` and ``q [N, Hq, D]``: rows of the QKV projection for N tokens, bf16 or fp16, any token and head
    strides; ``positions`` int32 ``[N]``: each token's position in its sequence, ``rows`` int32 ``[N]``: its sequence, a row of
    ``page_table`` (``None``: token i belongs to sequence i, a decode step).  ``k_pages``, ``v_pages`` ``[pages, H, page_size, D]``, bf16 or fp16;
    position t of sequence s is row ``t % page_size`` of page ``page_table[s, t // page_size]`` (int32).  Page size: a multiple of 16;
    D: 64, 128 or 256.  ``slots`` int32 ``[N]``: the position whose place a token's rows take, where that is not the one it is rotated by (the nodes of a
    drafted tree, see ``draft_tree``).

    ``eps``: RMS norm of q, k and v first (``None``: none).  ``cos``/``sin`` (fp32 ``[rows, D/2]``) rotate q and k at the token's position.
    ``ve [N, H, D]`` and ``gate`` (one fp32): v becomes ``gate * v + (1 - gate) * ve``.  Fp32 throughout, one rounding.

    Returns the prepared queries in the cache's dtype, or ``q_out`` (the cache's dtype or k's); ``None`` without ``q``.  ``k_out``, ``v_out``: ``[N, H, D]`` in k's
    dtype, receive k and v too (for the attention over a prompt); they and ``q_out`` may be k, v and q themselves, and share no memory with what else the
    call reads or writes (rows beside each other in one buffer, with the same strides, are fine).  A token at a negative position or slot is skipped: the cache and rows of buffers
    that the caller gave stay as they are, a query row of a tensor made here is zero.  Two tokens of one call must not share a place.

    The device reads positions, rows and table when the kernel runs.  One that leads to no page or past the rotary tables writes nothing to
    the cache, gives NaN elsewhere, and raises a bit in ``status`` (one-element int32, see ``raise_for_status``).
    """
    if eps is not None and not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    fast = _lib.native().paged_append(k, v, k_pages, v_pages, page_table, positions, rows, q, cos, sin, -1.0 if eps is None else eps, ve, gate, q_out, k_out, v_out, status, slots)
    if fast is not None:
        return fast if fast is not True else None
    dev = _lib.require_gpu(k, v, k_pages, v_pages, page_table, positions, rows, q, cos, sin, ve, gate, q_out, k_out, v_out, status, slots)
    _no_autograd("paged_append", k, v, q, ve, gate, k_pages, v_pages, q_out, k_out, v_out)
    _check_status(status)
    P, H, size, D = _check_pages(k_pages, v_pages, page_table)
    _check_rows("k", k, 3, _HALF_TYPES)
    _check_rows("v", v, 3, (k.dtype,))
    N = k.shape[0]
    if k.shape != (N, H, D) or v.shape != k.shape:
        raise ValueError(f"k, v must be [N, {H}, {D}] to fit the pages, got {tuple(k.shape)}, {tuple(v.shape)}")
    _check_index("positions", positions, N)
    if rows is not None:
        _check_index("rows", rows, N)
    elif N > page_table.shape[0]:
        raise ValueError(f"without rows, token i belongs to sequence i: {N} tokens, {page_table.shape[0]} sequences")
    if slots is not None:
        _check_index("slots", slots, N)
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin must be given together")
    if cos is not None:
        for name, t in (("cos", cos), ("sin", sin)):
            if t.dtype != torch.float32 or t.dim() != 2 or t.shape[1] != D // 2 or not t.is_contiguous() or t.shape != cos.shape:
                raise ValueError(f"{name} must be a contiguous fp32 [rows, {D // 2}] table, got {tuple(t.shape)} {t.dtype}")
    if (ve is None) != (gate is None):
        raise ValueError("ve and gate must be given together")
    if ve is not None:
        _check_rows("ve", ve, 3, (k.dtype,))
        if ve.shape != k.shape or gate.dtype != torch.float32 or gate.numel() != 1:
            raise ValueError(f"ve must be [N, {H}, {D}] and gate a one-element fp32 tensor")
    Hq, zero_skipped = 0, False
    if q is not None:
        _check_rows("q", q, 3, (k.dtype,))
        Hq = q.shape[1]
        if q.shape != (N, Hq, D) or Hq == 0:
            raise ValueError(f"q must be [{N}, Hq, {D}], got {tuple(q.shape)}")
        if q_out is None:
            q_out, zero_skipped = torch.empty((N, Hq, D), dtype=k_pages.dtype, device=dev), True
        _check_rows("q_out", q_out, 3, tuple({k_pages.dtype, k.dtype}))
        if q_out.shape != q.shape:
            raise ValueError(f"q_out must be {tuple(q.shape)}, got {tuple(q_out.shape)}")
    elif q_out is not None:
        raise ValueError("q_out is only produced when q is given")
    for name, t in (("k_out", k_out), ("v_out", v_out)):
        if t is not None:
            _check_rows(name, t, 3, (k.dtype,))
            if t.shape != k.shape:
                raise ValueError(f"{name} must be {tuple(k.shape)}, got {tuple(t.shape)}")
    if N == 0:
        return q_out
    d2, d3 = (0, 1), (0, 1, 2)
    st = lambda t: None if t is None else _lib.strides(t, d2)      # noqa: E731
    lib = _lib.load()
    with _lib.on_device(dev):
        rc = lib.daisy_paged_append_slots_fwd(
            _lib.ptr(q), st(q), k.data_ptr(), st(k), v.data_ptr(), st(v), 1 if k.dtype == torch.float16 else 0, _lib.ptr(ve), st(ve), _lib.ptr(gate),
            _lib.ptr(cos), _lib.ptr(sin), 0 if cos is None else int(cos.shape[0]),
            k_pages.data_ptr(), _lib.strides(k_pages, d3), v_pages.data_ptr(), _lib.strides(v_pages, d3), 1 if k_pages.dtype == torch.float16 else 0,
            page_table.data_ptr(), page_table.stride(0), page_table.shape[0], page_table.shape[1], P, size, positions.data_ptr(), _lib.ptr(rows), _lib.ptr(slots),
            _lib.ptr(q_out), st(q_out), 1 if q_out is not None and q_out.dtype == torch.float16 else 0, _lib.ptr(k_out), st(k_out), _lib.ptr(v_out), st(v_out), 1 if zero_skipped else 0,
            N, Hq, H, D, -1.0 if eps is None else float(eps), _lib.ptr(status), _lib.current_stream(dev))
    _lib.check(rc, "daisy_paged_append_slots_fwd")
    return q_out


def paged_attention_workspace_bytes(B: int, Hq: int, H: int, D: int, max_pages: int, page_size: int) -> int:
    return int(_lib.load().daisy_paged_attn_workspace_bytes(B, Hq, H, D, max_pages, page_size))


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, lens: torch.Tensor, *,
                    window: Optional[int] = None, scale: float = ATTN_SCALE, out: Optional[torch.Tensor] = None,
                    workspace: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The attention of one new token per sequence over a paged cache that holds its key and value already (``paged_append``).

    ``q [B, Hq, D]`` in the cache's dtype (bf16 or fp16), any batch and head strides; ``k_pages``, ``v_pages``, ``page_table`` as for ``paged_append``, row b of
    the table for sequence b; Hq a multiple of the cache's H, ``Hq // H`` query heads to a key head.  ``lens`` int32 ``[B]``: the number of
    positions of each sequence, the new token's among them; the last ``window`` of them are seen (``None``: all).  A sequence of length zero gives
    zeros.  Returns ``o [B, Hq, D]`` in q's dtype, or ``out``, which may be bf16 with an fp16 cache, and q itself, but share no
    memory with q otherwise, or with the pages.

    Rows of a page that are not visible may hold anything.  A visible value that is not finite makes its channel not finite for the heads that share it (an infinity may
    give NaN: a probability's rounding is a term of its own in the sum).

    Lengths and table are read when the kernels run, and the work is split over the lengths that are found there: nothing but shapes is fixed by a
    recording.  ``workspace``: at least ``paged_attention_workspace_bytes`` on the GPU, whatever it holds, for one call at a time (two that run at
    once, recorded ones too, need one each); ``None``: a tensor made for the call.  A length beyond the table's room, or a page that is none, gives NaN for the heads of that sequence and raises a bit in ``status``.
    """
    if window is not None and window <= 0:
        raise ValueError(f"window must be positive or None, got {window}")
    fast = _lib.native().paged_attention(q, k_pages, v_pages, page_table, lens, 0 if window is None else window, scale, out, workspace, status)
    if fast is not None:
        return fast
    dev = _lib.require_gpu(q, k_pages, v_pages, page_table, lens, out, workspace, status)
    _no_autograd("paged_attention", q, k_pages, v_pages, out)
    _check_status(status)
    P, H, size, D = _check_pages(k_pages, v_pages, page_table)
    _check_rows("q", q, 3, (k_pages.dtype,))
    B, Hq = q.shape[:2]
    if q.shape[2] != D or Hq == 0 or Hq % H != 0:
        raise ValueError(f"q must be [B, a multiple of {H}, {D}] to fit the pages, got {tuple(q.shape)}")
    if page_table.shape[0] < B:
        raise ValueError(f"page_table has {page_table.shape[0]} rows for {B} sequences")
    _check_index("lens", lens, B)
    if out is None:
        out = torch.empty((B, Hq, D), dtype=q.dtype, device=dev)
    else:
        _check_rows("out", out, 3, (torch.bfloat16,) if q.dtype == torch.bfloat16 else _HALF_TYPES)
        if out.shape != q.shape:
            raise ValueError(f"out must be {tuple(q.shape)}, got {tuple(out.shape)}")
    if B == 0:
        return out
    lib = _lib.load()
    max_pages = page_table.shape[1]
    need = int(lib.daisy_paged_attn_workspace_bytes(B, Hq, H, D, max_pages, size))
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    elif not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous")
    with _lib.on_device(dev):
        rc = lib.daisy_paged_attn_fwd(
            q.data_ptr(), _lib.strides(q, (0, 1)), k_pages.data_ptr(), _lib.strides(k_pages, (0, 1, 2)),
            v_pages.data_ptr(), _lib.strides(v_pages, (0, 1, 2)), 1 if q.dtype == torch.float16 else 0,
            page_table.data_ptr(), page_table.stride(0), max_pages, P, size, lens.data_ptr(), out.data_ptr(), _lib.strides(out, (0, 1)),
            1 if out.dtype == torch.float16 else 0, B, Hq, H, D, min(int(window), 2 ** 31 - 1) if window is not None else 0, float(scale), _lib.ptr(status),
            workspace.data_ptr(), workspace.numel() * workspace.element_size(), _lib.current_stream(dev))
    _lib.check(rc, "daisy_paged_attn_fwd")
    return out


_LOGITS_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MAX_HISTORY = 131071      # tokens of a row's history that process_logits can count


def process_logits(logits: torch.Tensor, history: Optional[torch.Tensor] = None, history_lens: Optional[torch.Tensor] = None, *,
                   repetition: Union[float, torch.Tensor] = 1.0, half_life: Optional[float] = None, cap: Optional[float] = None,
                   presence: Union[float, torch.Tensor] = 0.0, frequency: Union[float, torch.Tensor] = 0.0, lookback: Optional[int] = None,
                   bias: Optional[torch.Tensor] = None, allowed: Optional[torch.Tensor] = None,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Penalties for repeated tokens, biases and grammar masks on ``logits [B, V]`` (or ``[V]``; fp32, bf16 or fp16) in one launch.

    ``history [B, T]`` (int64 or int32 token ids, ``history_lens`` int32 ``[B]`` of them; ``None``: all T): of the last ``lookback`` (``None``: all, at most
    ``MAX_HISTORY``), a token that was seen n times, at ages (1 = the newest) that add up to ``w = sum 2 ** (-age / half_life)`` (``None``: w = n),
    has its logit divided by ``repetition ** min(w, cap)`` where positive and multiplied by it otherwise; ``frequency * n`` and, for n > 0, ``presence``
    are subtracted.  ``cap=1`` without a half life is the usual penalty; ``half_life=140, cap=3, lookback=128`` is the generator's
    (``penalise_repeats``).  Ids outside the vocabulary count for nothing.  ``repetition`` (positive and finite), ``presence``, ``frequency``: a number, or fp32 ``[B]`` on the GPU.

    ``bias`` (fp32 ``[V]`` or ``[B, V]``) is added.  ``allowed`` (int32 ``[ceil(V / 32)]`` or ``[B, ceil(V / 32)]``, see ``pack_allowed``): tokens whose bit
    (``v % 32`` of word ``v // 32``) is clear become -inf, whatever they were; a row without a set bit is -inf throughout.

    Returns a new tensor in the dtype of ``logits``, or ``out`` (``logits`` itself, or memory of its own).  The result does not depend on any order of
    summation.
    """
    if lookback is not None and lookback < 0:
        raise ValueError(f"lookback must not be negative, got {lookback}")
    fast = _lib.native().process_logits(logits, history, history_lens, repetition, 0.0 if half_life is None else half_life or -1.0, float("inf") if cap is None else cap,
                                        presence, frequency, -1 if lookback is None else lookback, bias, allowed, out)
    if fast is not None:
        return fast
    settings = [t for t in (repetition, presence, frequency) if isinstance(t, torch.Tensor)]
    dev = _lib.require_gpu(logits, history, history_lens, bias, allowed, out, *settings)
    _no_autograd("process_logits", logits, bias, out, *settings)
    if logits.dtype not in _LOGITS_TYPES:
        raise TypeError(f"logits must be float32, bfloat16 or float16, got {logits.dtype}")
    if logits.dim() not in (1, 2) or logits.stride(-1) != 1 and logits.shape[-1] > 1:
        raise ValueError(f"logits must be [B, V] or [V], contiguous in the last dim, got {tuple(logits.shape)}")
    x = logits.unsqueeze(0) if logits.dim() == 1 else logits
    B, V = x.shape
    if out is None:
        out = torch.empty(logits.shape, dtype=logits.dtype, device=dev)
    elif out.dtype != logits.dtype or out.shape != logits.shape or (V > 1 and out.stride(-1) != 1):
        raise ValueError(f"out must be {tuple(logits.shape)} {logits.dtype}, contiguous in the last dim")
    T = 0
    if history is not None:
        if history.dim() == 1 and logits.dim() == 1:
            history = history.unsqueeze(0)
        if history.dtype not in (torch.int64, torch.int32) or history.dim() != 2 or history.shape[0] != B or (history.shape[1] > 1 and history.stride(1) != 1):
            raise ValueError(f"history must be int64 or int32 [{B}, T], contiguous in the last dim, got {tuple(history.shape)} {history.dtype}")
        T = history.shape[1]
        if history_lens is not None:
            _check_index("history_lens", history_lens, B)
    elif history_lens is not None:
        raise ValueError("history_lens needs a history")
    lookback = T if lookback is None else min(int(lookback), T)
    if lookback > MAX_HISTORY:
        raise ValueError(f"a history of {lookback} tokens is too long: give a lookback of at most {MAX_HISTORY}")
    if half_life is not None and not half_life > 0.0:
        raise ValueError(f"half_life must be positive, got {half_life}")
    if cap is not None and not cap >= 0.0:
        raise ValueError(f"cap must not be negative, got {cap}")
    numbers = []
    for name, t in (("repetition", repetition), ("presence", presence), ("frequency", frequency)):
        if isinstance(t, torch.Tensor):
            if t.dtype != torch.float32 or t.shape != (B,) or not t.is_contiguous():
                raise ValueError(f"{name} must be a number or a contiguous fp32 [{B}] tensor, got {tuple(t.shape)} {t.dtype}")
            numbers += [t.data_ptr(), 0.0]
        else:
            numbers += [None, float(t)]
    if not isinstance(repetition, torch.Tensor) and not 0.0 < repetition < float("inf"):
        raise ValueError(f"repetition must be positive and finite, got {repetition}")
    strides = []
    for name, t, width, dtype in (("bias", bias, V, torch.float32), ("allowed", allowed, (V + 31) // 32, torch.int32)):
        if t is None:
            strides.append(0)
            continue
        if t.dtype != dtype or t.shape not in ((width,), (B, width)) or (width > 1 and t.stride(-1) != 1):
            raise ValueError(f"{name} must be {str(dtype)[6:]} [{width}] or [{B}, {width}], contiguous in the last dim, got {tuple(t.shape)} {t.dtype}")
        strides.append(t.stride(0) if t.dim() == 2 else 0)
    if B == 0 or V == 0:
        return out
    y = out.unsqueeze(0) if out.dim() == 1 else out
    lib = _lib.load()
    with _lib.on_device(dev):
        rc = lib.daisy_logits_process_fwd(
            x.data_ptr(), x.stride(0), y.data_ptr(), y.stride(0), _LOGITS_TYPES[logits.dtype], _lib.ptr(history),
            0 if history is None else history.stride(0), 0 if history is None or history.dtype == torch.int32 else 1, _lib.ptr(history_lens),
            T, lookback, *numbers, 0.0 if half_life is None else max(float(half_life), torch.finfo(torch.float32).tiny), float("inf") if cap is None else float(cap),
            _lib.ptr(bias), strides[0], _lib.ptr(allowed), strides[1], B, V, _lib.current_stream(dev))
    _lib.check(rc, "daisy_logits_process_fwd")
    return out


def pack_allowed(mask: torch.Tensor) -> torch.Tensor:
    """The bits that ``process_logits`` takes as ``allowed``: bool ``[..., V]`` -> int32 ``[..., ceil(V / 32)]`` on the same device."""
    if mask.dtype != torch.bool or mask.dim() == 0:
        raise TypeError(f"mask must be a bool [..., V] tensor, got {tuple(mask.shape)} {mask.dtype}")
    V = mask.shape[-1]
    words = torch.zeros(*mask.shape[:-1], (V + 31) // 32 * 32, dtype=torch.bool, device=mask.device)
    words[..., :V] = mask
    bits = words.view(*mask.shape[:-1], -1, 32).to(torch.int64) << torch.arange(32, device=mask.device)
    total = bits.sum(dim=-1)
    return (total - ((total >> 31) << 32)).to(torch.int32)


# ----------------------------------------------------------------------------------------------
# several drafted tokens per sequence in one step over a paged cache
# ----------------------------------------------------------------------------------------------
MAX_TREE_NODES = _lib.MAX_TREE_NODES


class DraftTree(NamedTuple):
    """What a step over trees of drafted tokens needs to know of them (``draft_tree``)."""
    mask: torch.Tensor           # int32 [B, T, ceil(T / 32)]: bit j % 32 of word j // 32 of node i: node i sees node j
    positions: torch.Tensor      # int32 [B * T]: the position that each node is rotated by, -1 for nodes that there are not
    slots: torch.Tensor          # int32 [B * T]: the position whose place in the cache it takes
    rows: torch.Tensor           # int32 [B * T]: its sequence


def _check_nodes(nodes: Optional[torch.Tensor], B: int, T: int) -> None:
    if not 0 < T <= MAX_TREE_NODES:
        raise ValueError(f"a tree must have 1 to {MAX_TREE_NODES} nodes, got {T}")
    if nodes is not None:
        _check_index("nodes", nodes, B)


def _check_parents(parents: torch.Tensor, B: int, T: Optional[int] = None) -> int:
    """Nodes of a tree."""
    T = parents.shape[-1] if T is None and parents.dim() else T
    if parents.dtype != torch.int32 or parents.shape not in ((T,), (B, T)) or (T > 1 and parents.stride(-1) != 1):
        raise ValueError(f"parents must be int32 [T] or [{B}, T], contiguous in the last dim, got {tuple(parents.shape)} {parents.dtype}")
    return T


def _row_stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.dim() == 2 and t.shape[0] > 1 else 0


def draft_tree(parents: torch.Tensor, lens: torch.Tensor, *, nodes: Optional[torch.Tensor] = None) -> DraftTree:
    """What the nodes of trees of drafted tokens see, the positions that they are rotated by and the places that they take in a paged cache, in one launch.

    ``parents`` int32 ``[B, T]`` (``[T]``: one tree for all; at most ``MAX_TREE_NODES``): the node that each comes from, ahead of it in the tree; anything else (-1, by
    convention) for a root.  Node 0 is the root that the step's tokens follow (``verify_drafts``).  ``lens`` int32 ``[B]``: the positions of each sequence's context
    (negative: a free slot, which has no nodes; ``PagedKVCache.positions``), ``nodes`` int32 ``[B]``: how many of its nodes there are (``None``: all).

    Node i of sequence b takes the place of position ``lens[b] + i`` and is rotated as position ``lens[b]`` plus the number of its ancestors: what ``paged_append``
    takes as ``slots`` and ``positions``, with ``rows``.  It sees the context, its ancestors and itself: ``mask``, for ``paged_tree_attention``.
    """
    fast = _lib.native().draft_tree(parents, lens, nodes)
    if fast is not None:
        return DraftTree(*fast)
    if lens.dtype != torch.int32 or lens.dim() != 1 or not lens.is_contiguous():
        raise ValueError(f"lens must be a contiguous int32 [B] tensor, got {tuple(lens.shape)} {lens.dtype}")
    dev = _lib.require_gpu(parents, lens, nodes)
    B = lens.shape[0]
    T = _check_parents(parents, B)
    _check_nodes(nodes, B, T)
    W = (T + 31) // 32
    room = torch.empty(B * T * (W + 3), dtype=torch.int32, device=dev)
    mask, positions, slots, rows = room.split([B * T * W, B * T, B * T, B * T])
    tree = DraftTree(mask.view(B, T, W), positions, slots, rows)
    if B == 0:
        return tree
    lib = _lib.load()
    with _lib.on_device(dev):
        rc = lib.daisy_draft_tree_fwd(parents.data_ptr(), _row_stride(parents), lens.data_ptr(), _lib.ptr(nodes), mask.data_ptr(), positions.data_ptr(),
                                      slots.data_ptr(), rows.data_ptr(), B, T, _lib.current_stream(dev))
    _lib.check(rc, "daisy_draft_tree_fwd")
    return tree


def paged_tree_attention_workspace_bytes(B: int, T: int, Hq: int, H: int, D: int, max_pages: int, page_size: int) -> int:
    return int(_lib.load().daisy_paged_tree_attn_workspace_bytes(B, T, Hq, H, D, max_pages, page_size))


def paged_tree_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, lens: torch.Tensor, mask: torch.Tensor, *,
                         nodes: Optional[torch.Tensor] = None, window: Optional[int] = None, scale: float = ATTN_SCALE, out: Optional[torch.Tensor] = None,
                         workspace: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The attention of a tree of drafted tokens per sequence over a paged cache that holds their keys and values already (``paged_append`` with ``slots``).

    ``q [B, T, Hq, D]`` in the cache's dtype (bf16 or fp16), any strides of the first three dims; pages and table as for ``paged_attention``.  ``lens`` int32 ``[B]``: the
    positions of each context, ahead of its tree (negative: a free slot); node i lies at position ``lens[b] + i``.  Every node sees the context, itself and the nodes whose bits ``mask``
    (int32 ``[B, T, ceil(T / 32)]``, see ``draft_tree``; any set of nodes) has; with ``window``, the last ``window`` of these, in the order of the cache.  ``nodes`` int32 ``[B]``: as for
    ``draft_tree``; the rows of the others become zero.  Returns ``o [B, T, Hq, D]``, or ``out``, as ``paged_attention`` does.

    Rows of a page that no node sees may hold anything.  A value that is not finite makes its channel not finite for the nodes that see it and the heads that share it (an infinity may
    come out as NaN); the others do not feel it.

    Lengths, nodes, mask and table are read when the kernels run.  ``workspace``: at least ``paged_tree_attention_workspace_bytes``, as for ``paged_attention``.  A tree that goes beyond the
    table's room, or a page that is none, gives NaN for the heads of that sequence and raises a bit in ``status``.
    """
    if window is not None and window <= 0:
        raise ValueError(f"window must be positive or None, got {window}")
    fast = _lib.native().paged_tree_attention(q, k_pages, v_pages, page_table, lens, mask, nodes, 0 if window is None else window, scale, out, workspace, status)
    if fast is not None:
        return fast
    dev = _lib.require_gpu(q, k_pages, v_pages, page_table, lens, mask, nodes, out, workspace, status)
    _no_autograd("paged_tree_attention", q, k_pages, v_pages, out)
    _check_status(status)
    P, H, size, D = _check_pages(k_pages, v_pages, page_table)
    _check_rows("q", q, 4, (k_pages.dtype,))
    B, T, Hq = q.shape[:3]
    if q.shape[3] != D or Hq == 0 or Hq % H != 0:
        raise ValueError(f"q must be [B, T, a multiple of {H}, {D}] to fit the pages, got {tuple(q.shape)}")
    if page_table.shape[0] < B:
        raise ValueError(f"page_table has {page_table.shape[0]} rows for {B} sequences")
    _check_index("lens", lens, B)
    _check_nodes(nodes, B, T)
    W = (T + 31) // 32
    if mask.dtype != torch.int32 or mask.shape != (B, T, W) or (W > 1 and mask.stride(2) != 1):
        raise ValueError(f"mask must be an int32 [{B}, {T}, {W}] tensor, contiguous in its last dim, got {tuple(mask.shape)} {mask.dtype}")
    if out is None:
        out = torch.empty((B, T, Hq, D), dtype=q.dtype, device=dev)
    else:
        _check_rows("out", out, 4, (torch.bfloat16,) if q.dtype == torch.bfloat16 else _HALF_TYPES)
        if out.shape != q.shape:
            raise ValueError(f"out must be {tuple(q.shape)}, got {tuple(out.shape)}")
    if B == 0:
        return out
    lib = _lib.load()
    max_pages, d3 = page_table.shape[1], (0, 1, 2)
    need = int(lib.daisy_paged_tree_attn_workspace_bytes(B, T, Hq, H, D, max_pages, size))
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    elif not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous")
    with _lib.on_device(dev):
        rc = lib.daisy_paged_tree_attn_fwd(
            q.data_ptr(), _lib.strides(q, d3), k_pages.data_ptr(), _lib.strides(k_pages, d3), v_pages.data_ptr(), _lib.strides(v_pages, d3),
            1 if q.dtype == torch.float16 else 0, page_table.data_ptr(), page_table.stride(0), max_pages, P, size, lens.data_ptr(), _lib.ptr(nodes),
            mask.data_ptr(), _lib.strides(mask, (0, 1)), out.data_ptr(), _lib.strides(out, d3), 1 if out.dtype == torch.float16 else 0, B, T, Hq, H, D,
            min(int(window), 2 ** 31 - 1) if window is not None else 0, float(scale), _lib.ptr(status),
            workspace.data_ptr(), workspace.numel() * workspace.element_size(), _lib.current_stream(dev))
    _lib.check(rc, "daisy_paged_tree_attn_fwd")
    return out


def verify_drafts_workspace_bytes(B: int, T: int, V: int) -> int:
    return int(_lib.load().daisy_verify_workspace_bytes(B, T, V))


def verify_drafts(logits: torch.Tensor, tokens: torch.Tensor, parents: torch.Tensor, *, nodes: Optional[torch.Tensor] = None,
                  temperature: Union[float, torch.Tensor] = 0.0, accept: Optional[torch.Tensor] = None, noise: Optional[torch.Tensor] = None,
                  draft: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Which nodes of trees of drafted tokens the target's probabilities accept, and the token that follows them, in two launches (four with ``draft``) that the host does not wait for.

    ``logits [B, T, V]`` (fp32, bf16 or fp16; any strides of the first two dims): row u says what may follow node u, ``p = softmax(logits[b, u] / temperature)``, -inf what may not (what
    ``process_logits`` or a filter has left).  ``tokens`` int64 or int32 ``[B, T]``: the nodes' tokens, of which node 0's is taken; ``parents``, ``nodes``: as for ``draft_tree``.
    ``temperature``: a number or fp32 ``[B]``; zero (in rows, less too): the likeliest token alone is accepted, and follows (of equal ones the lowest).

    From node 0 on, the children of the node are tried in their order.  Child c, with token y, is accepted where ``accept[b, c] * (1 - what rejected children took of p) < p(y)``; its p is
    taken where it is rejected (a token that an earlier child had has none left).  Where none is accepted, the token that follows is drawn from what is left: the
    largest ``log p(v) + noise[b, v]``.  With ``draft`` (fp32 ``[B, T, V]``: row u the probabilities q that the children of u were drawn from, independently) each rejection
    makes p ``max(p - q, 0)``, normalised (p as it was at first where that leaves nothing), and a child is accepted where ``accept[b, c] * q(y) < p(y)``.  Either way tokens come out as if drawn
    from p one by one.  ``accept`` fp32 ``[B, T]`` in [0, 1), ``noise`` fp32 ``[B, V]``, Gumbel (``generate.gumbel_noise``): the random numbers; not needed at temperature zero.

    Returns ``path`` int32 ``[B, T]`` (the accepted nodes from node 0 on, -1 behind them: an ``index`` for ``paged_move``), ``counts`` int32 ``[B]`` (how many) and the tokens that follow, int64 ``[B]``;
    -1 where nothing may: a row that is -inf throughout beside its children, a row with NaN or +inf, a row's temperature that is NaN or +inf, no nodes.

    Temperature zero compares the scores as they are.  Otherwise sums of exponentials are fp32 within up to 1024 tokens and 64 bits beyond them, within 2^-17 of themselves: so near are the probabilities that a child is accepted
    with.  What rejections of drawn children leave is held in 64 bits, however little it is, and the token that follows is looked for in 64 bits where fp32 does not tell it.  The same call gives the same results.

    ``workspace``: at least ``verify_drafts_workspace_bytes``, whatever it holds, for one call at a time; ``None``: a tensor made for the call.
    """
    fast = _lib.native().verify_drafts(logits, tokens, parents, nodes, temperature, accept, noise, draft, workspace)
    if fast is not None:
        return fast
    rows = temperature if isinstance(temperature, torch.Tensor) else None
    dev = _lib.require_gpu(logits, tokens, parents, nodes, rows, accept, noise, draft, workspace)
    _no_autograd("verify_drafts", logits, rows, accept, noise, draft)
    if logits.dtype not in _LOGITS_TYPES:
        raise TypeError(f"logits must be float32, bfloat16 or float16, got {logits.dtype}")
    if logits.dim() != 3 or logits.shape[2] == 0 or (logits.shape[2] > 1 and logits.stride(2) != 1):
        raise ValueError(f"logits must be [B, T, V], contiguous in the last dim, got {tuple(logits.shape)}")
    B, T, V = logits.shape
    _check_nodes(nodes, B, T)
    _check_parents(parents, B, T)
    if tokens.dtype not in (torch.int64, torch.int32) or tokens.shape != (B, T) or (T > 1 and tokens.stride(1) != 1):
        raise ValueError(f"tokens must be int64 or int32 [{B}, {T}], contiguous in the last dim, got {tuple(tokens.shape)} {tokens.dtype}")
    if rows is not None:
        if rows.dtype != torch.float32 or rows.shape != (B,) or not rows.is_contiguous():
            raise ValueError(f"temperature must be a number or a contiguous fp32 [{B}] tensor, got {tuple(rows.shape)} {rows.dtype}")
    elif not 0.0 <= temperature < float("inf"):
        raise ValueError(f"temperature must not be negative, and finite, got {temperature}")
    if (rows is not None or temperature > 0.0) and (accept is None or noise is None):
        raise ValueError("a temperature needs accept and noise")
    for name, t, shape in (("accept", accept, (B, T)), ("noise", noise, (B, V)), ("draft", draft, (B, T, V))):
        if t is not None and (t.dtype != torch.float32 or t.shape != shape or (shape[-1] > 1 and t.stride(-1) != 1)):
            raise ValueError(f"{name} must be fp32 {list(shape)}, contiguous in the last dim, got {tuple(t.shape)} {t.dtype}")
    path = torch.empty(B, T, dtype=torch.int32, device=dev)
    counts = torch.empty(B, dtype=torch.int32, device=dev)
    following = torch.empty(B, dtype=torch.int64, device=dev)
    if B == 0:
        return path, counts, following
    lib = _lib.load()
    need = int(lib.daisy_verify_workspace_bytes(B, T, V))
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    elif not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous")
    with _lib.on_device(dev):
        rc = lib.daisy_verify_fwd(
            logits.data_ptr(), _lib.strides(logits, (0, 1)), _LOGITS_TYPES[logits.dtype], tokens.data_ptr(), tokens.stride(0), 1 if tokens.dtype == torch.int64 else 0,
            parents.data_ptr(), _row_stride(parents), _lib.ptr(nodes), _lib.ptr(rows), 0.0 if rows is not None else float(temperature),
            _lib.ptr(accept), 0 if accept is None else accept.stride(0), _lib.ptr(noise), 0 if noise is None else noise.stride(0),
            _lib.ptr(draft), None if draft is None else _lib.strides(draft, (0, 1)), path.data_ptr(), counts.data_ptr(), following.data_ptr(), B, T, V,
            workspace.data_ptr(), workspace.numel() * workspace.element_size(), _lib.current_stream(dev))
    _lib.check(rc, "daisy_verify_fwd")
    return path, counts, following


def paged_move(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, starts: torch.Tensor, counts: torch.Tensor, *, rows: Optional[int] = None,
               index: Optional[torch.Tensor] = None, sources: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> None:
    """Rows of a paged cache to other places of it, in all layers, in one launch.

    ``k_pages``, ``v_pages`` ``[L, pages, H, page_size, D]`` (``PagedKVCache.k``, ``.v``; or one layer without the first dim), ``page_table`` as for ``paged_append``.  For
    sequence b, a row of the table, and ``i < counts[b]`` (int32 ``[B]``): position ``starts[b] + i`` (int32 ``[B]``; negative: nothing to do) becomes what position ``starts[b] + index[b, i]`` of
    sequence ``sources[b]`` held.  ``index`` int32 ``[B, M]`` (at most M rows of a sequence; ``None``: i itself, at most ``rows`` of them), ``sources`` int32 ``[B]`` (``None``: b itself).

    With ``index=path, counts=counts`` of ``verify_drafts`` and the context's lengths as ``starts``, the accepted nodes of a tree become the context's next positions.  With ``sources``
    a sequence gets another one's rows into pages of its own (a fork's last page).

    An index must rise from 0 or more on, so that a sequence can be closed up in place; what other sequences of the call read or write is the caller's to keep apart.  The device
    reads all of it when the kernel runs: an index that does not rise leaves its sequence as it was, a row that leads to no page is left out, and either raises a bit in
    ``status``.
    """
    if _lib.native().paged_move(k_pages, v_pages, page_table, starts, counts, -1 if rows is None else rows, index, sources, status) is not None:
        return
    dev = _lib.require_gpu(k_pages, v_pages, page_table, starts, counts, index, sources, status)
    _no_autograd("paged_move", k_pages, v_pages)
    _check_status(status)
    if k_pages.dim() == 4 and v_pages.dim() == 4:
        k_pages, v_pages = k_pages[None], v_pages[None]
    if k_pages.dim() != 5 or v_pages.shape != k_pages.shape or 0 in k_pages.shape:
        raise ValueError(f"k_pages, v_pages must be [L, pages, H, page_size, D] or [pages, H, page_size, D], got {tuple(k_pages.shape)}, {tuple(v_pages.shape)}")
    P, H, size, D = _check_pages(k_pages[0], v_pages[0], page_table)
    B = starts.shape[0] if starts.dim() else 0
    _check_index("starts", starts, B)
    _check_index("counts", counts, B)
    if B > page_table.shape[0]:
        raise ValueError(f"page_table has {page_table.shape[0]} rows for {B} sequences")
    if sources is not None:
        _check_index("sources", sources, B)
    if index is not None:
        if index.dtype != torch.int32 or index.dim() != 2 or index.shape[0] != B or (index.shape[1] > 1 and index.stride(1) != 1):
            raise ValueError(f"index must be an int32 [{B}, M] tensor, contiguous in its last dim, got {tuple(index.shape)} {index.dtype}")
        rows = index.shape[1]
    elif sources is None:
        raise ValueError("paged_move needs an index or sources: without them every row stays where it is")
    elif rows is None or rows < 0:
        raise ValueError(f"without an index, rows must say how many a sequence has at most, got {rows}")
    if B == 0 or rows == 0:
        return
    d4 = (0, 1, 2, 3)
    lib = _lib.load()
    with _lib.on_device(dev):
        rc = lib.daisy_paged_move_fwd(
            k_pages.data_ptr(), _lib.strides(k_pages, d4), v_pages.data_ptr(), _lib.strides(v_pages, d4), page_table.data_ptr(), page_table.stride(0),
            page_table.shape[0], page_table.shape[1], P, size, starts.data_ptr(), counts.data_ptr(), _lib.ptr(index), 0 if index is None else index.stride(0),
            _lib.ptr(sources), B, rows, k_pages.shape[0], H, D, _lib.ptr(status), _lib.current_stream(dev))
    _lib.check(rc, "daisy_paged_move_fwd")
