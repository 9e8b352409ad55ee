"""Sequence operators on device tensors: the query/key norm with its rotation,
and linear attention with a decay for each head.

Both are thin callers of the C ABI (to_qk_norm_rotary*, to_linear_attention*):
an object holds what stays fixed (type, heads, widths), a call takes torch
tensors and the stream to launch on (torch's current one where none is given;
0: the default stream) and allocates nothing.  Rows are tensors [tokens, heads, width] whose last dimension is
contiguous; they may be views into wider packed rows.  Shapes, types, devices
and sizes are checked here, the rest by the library; a failed check raises
before anything is launched (ValueError here, abi.ToError from the library).
Outputs share no memory with what the call reads, but for q_out, k_out and
state_out, which may be the inputs themselves.
No call records a graph for autograd; a torch.autograd.Function around forward
and backward does.  Autograd is told what a call has written.
The caller orders the streams: a tensor written on another stream has to be
ready on the call's, and may be freed or overwritten only after it.
"""
from __future__ import annotations

import ctypes as C
import math
import struct
from typing import Optional, Sequence

import torch
from torch.autograd.graph import increment_version  # tells autograd that a saved tensor has changed

from . import abi

# to_rows, to_linear_attention_desc / _args / _grad_args as the C compiler lays
# them out: a call packs its arguments into bytes of its own (a ctypes structure
# filled field by field took longer than the smallest kernels).
_ROWS = struct.Struct("@Pqq")
_DESC = struct.Struct("@6i2qd")
_ARGS = struct.Struct("@" + 4 * "Pqq" + "6PN")
_GRAD_ARGS = struct.Struct("@" + 7 * "Pqq" + "6PN")

DTYPES = {torch.bfloat16: abi.TO_BF16, torch.float32: abi.TO_F32}


def _dtype(dtype) -> torch.dtype:
    kind = {"bf16": torch.bfloat16, "f32": torch.float32}.get(dtype, dtype)
    if kind not in DTYPES:
        raise ValueError(f"dtype {dtype!r}: 'bf16' or 'f32'")
    return kind


def _sizes(**sizes):
    """Sizes that the descriptors hold (32-bit fields, which would cut longer ones short)."""
    for name, n in sizes.items():
        if not -2**31 <= n < 2**31:
            raise ValueError(f"{name} {n} does not fit 32 bits")


def _rows(t, name: str, dtype: torch.dtype, shape, device):
    """(data, token stride, head stride) of rows, as in to_rows."""
    if t.shape != shape or t.dtype != dtype or t.device != device:
        _refuse(t, name, dtype, shape, device)
    stride = t.stride()
    if stride[2] != 1 and shape[2] > 1:
        raise ValueError(f"{name}: the last dimension is not contiguous")
    return t.data_ptr(), stride[0], stride[1]


def _flat(t, name: str, dtype: torch.dtype, shape, device) -> int:
    """Data of a contiguous tensor; 0 where there is none."""
    if t is None:
        return 0
    if t.shape != shape or t.dtype != dtype or t.device != device:
        _refuse(t, name, dtype, shape, device)
    if not t.is_contiguous():
        raise ValueError(f"{name} is not contiguous")
    return t.data_ptr()


def _refuse(t, name, dtype, shape, device):
    if t.shape != shape:
        raise ValueError(f"{name}: shape {tuple(t.shape)} is not {tuple(shape)}")
    if t.dtype != dtype:
        raise ValueError(f"{name}: {t.dtype} is not {dtype}")
    raise ValueError(f"{name}: on {t.device}, not on {device}")


def _needed(t, name: str):
    if t is None:
        raise ValueError(f"{name} is missing")
    return t


def _cuda(t, name: str):
    if t.device.type != "cuda":
        raise ValueError(f"{name}: on {t.device}; the operators run on CUDA tensors")
    if t.device.index != torch.cuda.current_device():
        raise ValueError(f"{name}: on {t.device}; the current device is {torch.cuda.current_device()}")
    return t.device


def _on(stream: Optional[int], device) -> int:
    return torch.cuda.current_stream(device).cuda_stream if stream is None else stream


def _scratch(t, need: int, device):
    """(pointer, bytes) of a workspace; none is needed where `need` is 0."""
    if t is None:
        if need:
            raise ValueError(f"a workspace of {need} bytes is needed")
        return 0, 0
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
        _sizes(q_heads=q_heads, k_heads=k_heads, head_dim=head_dim, rotary_dim=self.rotary_dim,
               section=max(sections, key=abs))
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
        d = self.head_dim
        return (_ROWS.pack(*_rows(q, names[0], self.dtype, (tokens, self.q_heads, d), device)),
                _ROWS.pack(*_rows(k, names[1], self.dtype, (tokens, self.k_heads, d), device)))

    def _fixed(self, positions, wq, wk, tokens, device):
        pos = 0
        if self.rotary_dim:
            pos = _flat(_needed(positions, "positions"), "positions", torch.int32, (self.axes, tokens), device)
        shape = (self.head_dim,)
        return (pos, _flat(wq, "wq", torch.float32, shape, device), _flat(wk, "wk", torch.float32, shape, device))

    def forward(self, q, k, positions, wq, wk, q_out, k_out, stream: Optional[int] = None):
        """q_out, k_out <- the normed, weighted and rotated q, k (in place where they are q, k).

        positions: int32 [axes, tokens]; wq, wk: f32 [head_dim] or None.
        """
        tokens, device = q.shape[0], _cuda(q, "q")
        i = self._pair(q, k, ("q", "k"), tokens, device)
        o = self._pair(q_out, k_out, ("q_out", "k_out"), tokens, device)
        st = abi.lib.to_qk_norm_rotary(self._h, tokens, *i, *self._fixed(positions, wq, wk, tokens, device), *o,
                                       _on(stream, device))
        if st:
            abi.check(st, "to_qk_norm_rotary")
        increment_version((q_out, k_out))

    def workspace_bytes(self, tokens: int) -> int:
        """Bytes of `workspace` that backward() needs."""
        return abi.lib.to_qk_norm_rotary_workspace_bytes(self._h, tokens)

    def backward(self, q, k, positions, wq, wk, gq, gk, dq, dk, dwq, dwk, workspace, stream: Optional[int] = None):
        """dq, dk, dwq, dwk <- gradients from gq, gk (those of q_out, k_out); q, k are forward()'s inputs."""
        tokens, device, shape = q.shape[0], _cuda(q, "q"), (self.head_dim,)
        i = self._pair(q, k, ("q", "k"), tokens, device)
        g = self._pair(gq, gk, ("gq", "gk"), tokens, device)
        o = self._pair(dq, dk, ("dq", "dk"), tokens, device)
        dw = _flat(dwq, "dwq", torch.float32, shape, device), _flat(dwk, "dwk", torch.float32, shape, device)
        abi.check(abi.lib.to_qk_norm_rotary_backward(self._h, tokens, *i,
                                                     *self._fixed(positions, wq, wk, tokens, device), *g, *o, *dw,
                                                     *_scratch(workspace, 1, device), _on(stream, device)),
                  "to_qk_norm_rotary_backward")
        increment_version([t for t in (dq, dk, dwq, dwk) if t is not None])


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
        _sizes(q_heads=q_heads, kv_heads=kv_heads, key_dim=key_dim, value_dim=value_dim)
        self.scale = 1.0 / math.sqrt(max(key_dim, 1)) if scale is None else scale  # (widths below 1 are refused)
        abi.check(abi.lib.to_linear_attention(self._desc(0, 0), bytes(_ARGS.size), 0), "LinearAttention")

    def _desc(self, tokens: int, nseq: int, slots: int = 0) -> bytes:
        return _DESC.pack(DTYPES[self.dtype], self.q_heads, self.kv_heads, self.key_dim, self.value_dim, nseq, tokens,
                          slots, self.scale)

    def workspace_bytes(self, tokens: int, sequences: int) -> int:
        """Bytes of `workspace` that forward() needs (0: none)."""
        return abi.lib.to_linear_attention_workspace_bytes(self._desc(tokens, sequences))

    def backward_workspace_bytes(self, tokens: int, sequences: int) -> int:
        return abi.lib.to_linear_attention_backward_workspace_bytes(self._desc(tokens, sequences))

    def _inputs(self, tokens, device, tensors):
        """Rows of (tensor, name, is a query head's, width) each, in one list."""
        out = []
        for t, name, query, width in tensors:
            out += _rows(t, name, self.dtype, (tokens, self.q_heads if query else self.kv_heads, width), device)
        return out

    def _state(self, t, name, device, slots):
        return _flat(t, name, torch.float32, (slots, self.q_heads, self.key_dim, self.value_dim), device)

    def _sequences(self, cu_seqlens, device):
        n = cu_seqlens.numel() - 1
        if n < 0:
            raise ValueError("cu_seqlens is empty")
        return n, _flat(cu_seqlens, "cu_seqlens", torch.int32, (n + 1,), device)

    def _decay(self, log_decay, device):
        return _flat(_needed(log_decay, "log_decay"), "log_decay", torch.float32, (self.q_heads,), device)

    def forward(self, q, k, v, log_decay, cu_seqlens, o, state_in=None, state_out=None, slots=None, workspace=None,
                stream: Optional[int] = None):
        """o <- the outputs of packed sequences; state_out (may be state_in) <- the states they leave.

        cu_seqlens: int32 [sequences + 1], on the device.  slots: int32
        [sequences], each sequence's place in state_in and state_out (None:
        its number); one outside them means no state.
        """
        tokens, device = q.shape[0], _cuda(q, "q")
        n, cu = self._sequences(cu_seqlens, device)
        have = n if state_in is None and state_out is None else (state_out if state_in is None else state_in).shape[0]
        if slots is None and have != n:
            raise ValueError(f"{have} states for {n} sequences, and no slots")
        desc, dk, dv = self._desc(tokens, n, have), self.key_dim, self.value_dim
        args = _ARGS.pack(
            *self._inputs(tokens, device, ((q, "q", True, dk), (k, "k", False, dk), (v, "v", False, dv),
                                           (o, "o", True, dv))),
            self._decay(log_decay, device), cu, _flat(slots, "slots", torch.int32, (n,), device),
            self._state(state_in, "state_in", device, have), self._state(state_out, "state_out", device, have),
            *_scratch(workspace, abi.lib.to_linear_attention_workspace_bytes(desc), device))
        st = abi.lib.to_linear_attention(desc, args, _on(stream, device))
        if st:
            abi.check(st, "to_linear_attention")
        increment_version((o,) if state_out is None else (o, state_out))

    def step(self, q, k, v, log_decay, state, o, slots=None, stream: Optional[int] = None):
        """One token of each request: its state is updated in place, o <- its output."""
        tokens, device, have = q.shape[0], _cuda(q, "q"), state.shape[0]
        if slots is None and have < tokens:
            raise ValueError(f"{have} states for {tokens} requests, and no slots")
        dk, dv = self.key_dim, self.value_dim
        args = _ARGS.pack(
            *self._inputs(tokens, device, ((q, "q", True, dk), (k, "k", False, dk), (v, "v", False, dv),
                                           (o, "o", True, dv))),
            self._decay(log_decay, device), 0, _flat(slots, "slots", torch.int32, (tokens,), device), 0,
            self._state(state, "state", device, have), 0, 0)
        st = abi.lib.to_linear_attention_step(self._desc(tokens, 0, have), args, _on(stream, device))
        if st:
            abi.check(st, "to_linear_attention_step")
        increment_version((o, state))

    def backward(self, q, k, v, log_decay, cu_seqlens, do, dq, dk, dv, state_in=None, dstate_out=None,
                 dstate_in=None, workspace=None, stream: Optional[int] = None):
        """dq, dk, dv (and dstate_in) <- gradients of forward() from do and dstate_out.

        State tensors hold one state a sequence, in order.  log_decay gets no gradient.
        """
        tokens, device = q.shape[0], _cuda(q, "q")
        n, cu = self._sequences(cu_seqlens, device)
        desc, wk, wv = self._desc(tokens, n, n), self.key_dim, self.value_dim
        args = _GRAD_ARGS.pack(
            *self._inputs(tokens, device, ((q, "q", True, wk), (k, "k", False, wk), (v, "v", False, wv),
                                           (do, "do", True, wv), (dq, "dq", True, wk), (dk, "dk", False, wk),
                                           (dv, "dv", False, wv))),
            self._decay(log_decay, device), cu, self._state(state_in, "state_in", device, n),
            self._state(dstate_out, "dstate_out", device, n), self._state(dstate_in, "dstate_in", device, n),
            *_scratch(workspace, abi.lib.to_linear_attention_backward_workspace_bytes(desc), device))
        st = abi.lib.to_linear_attention_backward(desc, args, _on(stream, device))
        if st:
            abi.check(st, "to_linear_attention_backward")
        increment_version((dq, dk, dv) if dstate_in is None else (dq, dk, dv, dstate_in))
