"""Sequence operators on device tensors: the query/key norm with its rotation,
and linear attention with a decay for each head.

Both are thin callers of the C ABI (to_qk_norm_rotary*, to_linear_attention*):
an object holds what stays fixed (type, heads, widths), a call takes torch
tensors and the stream to launch on (0: the default stream) and allocates
nothing.  Rows are tensors [tokens, heads, width] whose last dimension is
contiguous; they may be views into wider packed rows.  Shapes, types, devices
and sizes are checked here, the rest by the library; a failed check raises
before anything is launched (ValueError here, abi.ToError from the library).
The caller orders the streams: a tensor written on another stream has to be
ready on `stream`, and may be freed or overwritten only after it.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional, Sequence

import torch

from . import abi

DTYPES = {torch.bfloat16: abi.TO_BF16, torch.float32: abi.TO_F32}


def _dtype(dtype) -> torch.dtype:
    kind = {"bf16": torch.bfloat16, "f32": torch.float32}.get(dtype, dtype)
    if kind not in DTYPES:
        raise ValueError(f"dtype {dtype!r}: 'bf16' or 'f32'")
    return kind


def _rows(t, name: str, dtype: torch.dtype, tokens: int, heads: int, width: int, device) -> abi.Rows:
    if t.shape != (tokens, heads, width):
        raise ValueError(f"{name}: shape {tuple(t.shape)} is not {(tokens, heads, width)}")
    if t.dtype != dtype:
        raise ValueError(f"{name}: {t.dtype} is not {dtype}")
    if t.device != device:
        raise ValueError(f"{name}: on {t.device}, not on {device}")
    if width > 1 and t.stride(2) != 1:
        raise ValueError(f"{name}: the last dimension is not contiguous")
    return abi.Rows(t.data_ptr() if t.numel() else None, t.stride(0), t.stride(1))


def _flat(t, name: str, dtype: torch.dtype, shape, device, optional: bool = False) -> Optional[int]:
    if t is None:
        if optional:
            return None
        raise ValueError(f"{name} is missing")
    if t.shape != tuple(shape):
        raise ValueError(f"{name}: shape {tuple(t.shape)} is not {tuple(shape)}")
    if t.dtype != dtype:
        raise ValueError(f"{name}: {t.dtype} is not {dtype}")
    if t.device != device:
        raise ValueError(f"{name}: on {t.device}, not on {device}")
    if not t.is_contiguous():
        raise ValueError(f"{name} is not contiguous")
    return t.data_ptr()


def _cuda(t, name: str):
    if t.device.type != "cuda":
        raise ValueError(f"{name}: on {t.device}; the operators run on CUDA tensors")
    if t.device.index != torch.cuda.current_device():
        raise ValueError(f"{name}: on {t.device}; the current device is {torch.cuda.current_device()}")
    return t.device


def _scratch(t, need: int, device):
    """(pointer, bytes) of a workspace; none is needed where `need` is 0."""
    if t is None:
        if need:
            raise ValueError(f"a workspace of {need} bytes is needed")
        return None, 0
    if t.device != device or not t.is_contiguous():
        raise ValueError(f"workspace: on {t.device}, contiguous {t.is_contiguous()}; wanted on {device}")
    return t.data_ptr(), t.numel() * t.element_size()


class QkNormRotary:
    """Norm of every query and key head and its rotation by position, in one pass.

    `sections` names the rotated pairs of each position axis (their sum is
    rotary_dim / 2; one axis by default).  `interleaved` pairs neighbours
    (2j, 2j+1) instead of halves (j, j + rotary_dim/2).
    """

    def __init__(self, dtype, q_heads: int, k_heads: int, head_dim: int, rotary_dim: Optional[int] = None,
                 sections: Optional[Sequence[int]] = None, interleaved: bool = False, theta: float = 10000.0,
                 eps: float = 1e-6):
        self.dtype = _dtype(dtype)
        self.q_heads, self.k_heads, self.head_dim = q_heads, k_heads, head_dim
        self.rotary_dim = head_dim if rotary_dim is None else rotary_dim
        sections = [self.rotary_dim // 2] if sections is None else list(sections)
        if not 1 <= len(sections) <= 4:
            raise ValueError(f"{len(sections)} axes: 1 to 4 are supported")
        self.axes = len(sections)
        d = abi.QkDesc(DTYPES[self.dtype], q_heads, k_heads, head_dim, self.rotary_dim, self.axes)
        d.section[:self.axes] = sections
        d.interleaved, d.theta, d.eps = int(bool(interleaved)), theta, eps
        self._h = C.c_void_p()
        abi.check(abi.lib.to_qk_plan_create(C.byref(d), C.byref(self._h)), "to_qk_plan_create")

    def __del__(self):
        h = getattr(self, "_h", None)
        if h is not None and h.value and abi is not None and abi.lib is not None:
            abi.lib.to_qk_plan_destroy(h)
            self._h = None

    def _pair(self, q, k, names, tokens, device):
        return (C.byref(_rows(q, names[0], self.dtype, tokens, self.q_heads, self.head_dim, device)),
                C.byref(_rows(k, names[1], self.dtype, tokens, self.k_heads, self.head_dim, device)))

    def _fixed(self, positions, wq, wk, tokens, device):
        pos = None
        if self.rotary_dim:
            pos = _flat(positions, "positions", torch.int32, (self.axes, tokens), device)
        w = [_flat(x, n, torch.float32, (self.head_dim,), device, True) for x, n in ((wq, "wq"), (wk, "wk"))]
        return pos, w[0], w[1]

    def forward(self, q, k, positions, wq, wk, q_out, k_out, stream: int = 0):
        """q_out, k_out <- the normed, weighted and rotated q, k (in place where they are q, k).

        positions: int32 [axes, tokens]; wq, wk: f32 [head_dim] or None.
        """
        tokens, device = q.shape[0], _cuda(q, "q")
        i = self._pair(q, k, ("q", "k"), tokens, device)
        o = self._pair(q_out, k_out, ("q_out", "k_out"), tokens, device)
        abi.check(abi.lib.to_qk_norm_rotary(self._h, tokens, *i, *self._fixed(positions, wq, wk, tokens, device),
                                            *o, stream), "to_qk_norm_rotary")

    def workspace_bytes(self, tokens: int) -> int:
        """Bytes of `workspace` that backward() needs."""
        return abi.lib.to_qk_norm_rotary_workspace_bytes(self._h, tokens)

    def backward(self, q, k, positions, wq, wk, gq, gk, dq, dk, dwq, dwk, workspace, stream: int = 0):
        """dq, dk, dwq, dwk <- gradients from gq, gk (those of q_out, k_out); q, k are forward()'s inputs."""
        tokens, device = q.shape[0], _cuda(q, "q")
        i = self._pair(q, k, ("q", "k"), tokens, device)
        g = self._pair(gq, gk, ("gq", "gk"), tokens, device)
        o = self._pair(dq, dk, ("dq", "dk"), tokens, device)
        dw = [_flat(x, n, torch.float32, (self.head_dim,), device, True) for x, n in ((dwq, "dwq"), (dwk, "dwk"))]
        ws, size = _scratch(workspace, 1, device)
        abi.check(abi.lib.to_qk_norm_rotary_backward(self._h, tokens, *i,
                                                     *self._fixed(positions, wq, wk, tokens, device), *g, *o, *dw,
                                                     ws, size, stream), "to_qk_norm_rotary_backward")


class LinearAttention:
    """o_t = scale * S_t^T q_t with S_t = exp(log_decay) S_{t-1} + k_t v_t^T for each query head.

    Prompts (`forward`) are packed sequences in chunked form, single tokens
    (`step`) update the states in place, `backward` gives the gradients of
    `forward`.  log_decay: f32 [q_heads], <= 0.  States: f32
    [slots, q_heads, key_dim, value_dim].  scale: key_dim ** -0.5 by default.
    """

    def __init__(self, dtype, q_heads: int, kv_heads: int, key_dim: int, value_dim: int,
                 scale: Optional[float] = None):
        self.dtype = _dtype(dtype)
        self.q_heads, self.kv_heads, self.key_dim, self.value_dim = q_heads, kv_heads, key_dim, value_dim
        self.scale = 1.0 / math.sqrt(key_dim) if scale is None else scale
        self._desc(0, 0)
        abi.check(abi.lib.to_linear_attention(self._desc(0, 0), C.byref(abi.LinearAttentionArgs()), 0),
                  "LinearAttention")

    def _desc(self, tokens: int, nseq: int, slots: int = 0):
        return C.byref(abi.LinearAttentionDesc(DTYPES[self.dtype], self.q_heads, self.kv_heads, self.key_dim,
                                               self.value_dim, nseq, tokens, slots, self.scale))

    def workspace_bytes(self, tokens: int, sequences: int) -> int:
        """Bytes of `workspace` that forward() needs (0: none)."""
        return abi.lib.to_linear_attention_workspace_bytes(self._desc(tokens, sequences))

    def backward_workspace_bytes(self, tokens: int, sequences: int) -> int:
        return abi.lib.to_linear_attention_backward_workspace_bytes(self._desc(tokens, sequences))

    def _kv(self, t, name, tokens, width, device):
        return _rows(t, name, self.dtype, tokens, self.kv_heads, width, device)

    def _q(self, t, name, tokens, width, device):
        return _rows(t, name, self.dtype, tokens, self.q_heads, width, device)

    def _state(self, t, name, device, slots=None):
        n = t.shape[0] if slots is None and t is not None else slots
        return _flat(t, name, torch.float32, (n, self.q_heads, self.key_dim, self.value_dim), device, True)

    def _sequences(self, cu_seqlens, device):
        n = cu_seqlens.numel() - 1
        if n < 0:
            raise ValueError("cu_seqlens is empty")
        return n, _flat(cu_seqlens, "cu_seqlens", torch.int32, (n + 1,), device)

    def _decay(self, log_decay, device):
        return _flat(log_decay, "log_decay", torch.float32, (self.q_heads,), device)

    def forward(self, q, k, v, log_decay, cu_seqlens, o, state_in=None, state_out=None, slots=None, workspace=None,
                stream: int = 0):
        """o <- the outputs of packed sequences; state_out (may be state_in) <- the states they leave.

        cu_seqlens: int32 [sequences + 1], on the device.  slots: int32
        [sequences], each sequence's place in state_in and state_out (None:
        its number); one outside them means no state.
        """
        tokens, device = q.shape[0], _cuda(q, "q")
        n, cu = self._sequences(cu_seqlens, device)
        have = next((t.shape[0] for t in (state_in, state_out) if t is not None), n)
        if slots is None and have != n:
            raise ValueError(f"{have} states for {n} sequences, and no slots")
        need = self.workspace_bytes(tokens, n)
        ws, size = _scratch(workspace, need, device)
        a = abi.LinearAttentionArgs(
            self._q(q, "q", tokens, self.key_dim, device), self._kv(k, "k", tokens, self.key_dim, device),
            self._kv(v, "v", tokens, self.value_dim, device), self._q(o, "o", tokens, self.value_dim, device),
            self._decay(log_decay, device), cu, _flat(slots, "slots", torch.int32, (n,), device, True),
            self._state(state_in, "state_in", device, have if state_in is not None else None),
            self._state(state_out, "state_out", device, have if state_out is not None else None), ws, size)
        abi.check(abi.lib.to_linear_attention(self._desc(tokens, n, have), C.byref(a), stream),
                  "to_linear_attention")

    def step(self, q, k, v, log_decay, state, o, slots=None, stream: int = 0):
        """One token of each request: its state is updated in place, o <- its output."""
        tokens, device = q.shape[0], _cuda(q, "q")
        if slots is None and state.shape[0] < tokens:
            raise ValueError(f"{state.shape[0]} states for {tokens} requests, and no slots")
        a = abi.LinearAttentionArgs(
            self._q(q, "q", tokens, self.key_dim, device), self._kv(k, "k", tokens, self.key_dim, device),
            self._kv(v, "v", tokens, self.value_dim, device), self._q(o, "o", tokens, self.value_dim, device),
            self._decay(log_decay, device), None, _flat(slots, "slots", torch.int32, (tokens,), device, True),
            None, self._state(state, "state", device))
        abi.check(abi.lib.to_linear_attention_step(self._desc(tokens, 0, state.shape[0]), C.byref(a), stream),
                  "to_linear_attention_step")

    def backward(self, q, k, v, log_decay, cu_seqlens, do, dq, dk, dv, state_in=None, dstate_out=None,
                 dstate_in=None, workspace=None, stream: int = 0):
        """dq, dk, dv (and dstate_in) <- gradients of forward() from do and dstate_out.

        State tensors hold one state a sequence, in order.  log_decay gets no gradient.
        """
        tokens, device = q.shape[0], _cuda(q, "q")
        n, cu = self._sequences(cu_seqlens, device)
        need = self.backward_workspace_bytes(tokens, n)
        ws, size = _scratch(workspace, need, device)
        states = [self._state(t, name, device, n) if t is not None else None
                  for t, name in ((state_in, "state_in"), (dstate_out, "dstate_out"), (dstate_in, "dstate_in"))]
        a = abi.LinearAttentionGradArgs(
            self._q(q, "q", tokens, self.key_dim, device), self._kv(k, "k", tokens, self.key_dim, device),
            self._kv(v, "v", tokens, self.value_dim, device), self._q(do, "do", tokens, self.value_dim, device),
            self._q(dq, "dq", tokens, self.key_dim, device), self._kv(dk, "dk", tokens, self.key_dim, device),
            self._kv(dv, "dv", tokens, self.value_dim, device), self._decay(log_decay, device), cu, *states, ws, size)
        abi.check(abi.lib.to_linear_attention_backward(self._desc(tokens, n, n), C.byref(a), stream),
                  "to_linear_attention_backward")
