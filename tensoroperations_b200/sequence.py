"""Sequence operators on device tensors: the query/key norm with its rotation,
linear attention with a decay for each head, the gated linear recurrence of
channels, the norms around a block with its gate and residual scale, and rows
kept in 8 bits for a backward pass.

All are thin callers of the C ABI (to_qk_norm_rotary*, to_linear_attention*,
to_gated_recurrence*, to_block_norm*, to_rows8*): an object holds what stays fixed (type, heads, widths), a call takes torch
tensors and the stream to launch on (torch's current one where none is given;
0: the default stream) and allocates nothing.  Rows are tensors [tokens, heads, width] or, without heads,
[tokens, width], whose last dimension is contiguous; they may be views into wider packed rows.  Shapes, types, devices
and sizes are checked here, the rest by the library; a failed check raises
before anything is launched (ValueError here, abi.ToError from the library).
Outputs share no memory with what the call reads, but for q_out, k_out,
state_out, r_out and dr, which may be the inputs themselves.
No call records a graph for autograd; a torch.autograd.Function around forward
and backward does.  Autograd is told what a call has written.
The caller orders the streams: a tensor written on another stream has to be
ready on the call's, and may be freed or overwritten only after it.
"""
from __future__ import annotations

import ctypes as C
import math
import struct
from typing import NamedTuple, Optional, Sequence

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
# to_rows8; to_gated_recurrence_desc / _args / _grad_args; to_block_norm_desc / _args / _grad_args
_ROWS8 = struct.Struct("@PPqq")
_REC_DESC = struct.Struct("@4i2q")
_REC_ARGS = struct.Struct("@" + 3 * "Pqq" + 2 * "PPqq" + "7PN")
_REC_GRAD_ARGS = struct.Struct("@" + 5 * "Pqq" + 2 * "PPqq" + "7PN")
_NORM_DESC = struct.Struct("@6i2d")
_NORM_ARGS = struct.Struct("@" + 5 * "Pqq" + 3 * "PPqq" + "2P")
_NORM_GRAD_ARGS = struct.Struct("@" + 8 * "Pqq" + 3 * "PPqq" + "5PN")
_NO_ROWS, _NO_ROWS8 = (0, 0, 0), (0, 0, 0, 0)

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


def _row(t, name: str, dtype: torch.dtype, shape, device):
    """(data, token stride, 0) of rows without heads, as in to_rows."""
    if t.shape != shape or t.dtype != dtype or t.device != device:
        _refuse(t, name, dtype, shape, device)
    stride = t.stride()
    if stride[1] != 1 and shape[1] > 1:
        raise ValueError(f"{name}: the last dimension is not contiguous")
    return t.data_ptr(), stride[0], 0


def _row8(t, name: str, tokens: int, width: int, device):
    """(codes, scales, their token strides) of rows in 8 bits, as in to_rows8."""
    if not isinstance(t, Rows8):
        raise ValueError(f"{name}: {type(t).__name__} is not Rows8")
    codes = _row(t.codes, f"{name}.codes", torch.int8, (tokens, width), device)
    scales = _row(t.scales, f"{name}.scales", torch.uint8, (tokens, -(-width // GROUP8)), device)
    return codes[0], scales[0], codes[1], scales[1]


def _row_or_8(t, name: str, dtype: torch.dtype, shape, device):
    """A to_rows and a to_rows8, one of them empty."""
    if isinstance(t, Rows8):
        return _NO_ROWS, _row8(t, name, *shape, device)
    return _row(t, name, dtype, shape, device), _NO_ROWS8


def _written(*outputs):
    """Tells autograd which tensors a call has written (None, tensors and Rows8)."""
    seen = []
    for t in outputs:
        if isinstance(t, Rows8):
            seen += t
        elif t is not None:
            seen.append(t)
    increment_version(seen)


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
    # (torch.cuda.current_stream makes an object, which takes longer than the smallest kernels)
    return torch._C._cuda_getCurrentRawStream(device.index) if stream is None else stream


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


GROUP8 = 32  # neighbouring values of Rows8 that share a scale


class Rows8(NamedTuple):
    """Rows in 8 bits: value = codes * 2^(scales - 127), a scale for every 32 neighbouring values.

    codes: int8 [tokens, width]; scales: uint8 [tokens, ceil(width / 32)]
    (255: the group held an infinity or a NaN and reads as NaN).  A value is off
    by at most half a scale, 1/127 of the largest one of its 32.
    """
    codes: torch.Tensor
    scales: torch.Tensor

    @classmethod
    def empty(cls, tokens: int, width: int, device="cuda") -> "Rows8":
        """Uninitialised rows."""
        return cls(torch.empty(tokens, width, dtype=torch.int8, device=device),
                   torch.empty(tokens, -(-width // GROUP8), dtype=torch.uint8, device=device))


class Checkpoint8:
    """Activations into 8 bits (Rows8) and back.

    GatedRecurrence and BlockNorm write the same form while they hold the rows
    (keep_*), and their backward passes read it in the place of the rows.
    """

    def __init__(self, dtype, width: int):
        self.dtype, self.width = _dtype(dtype), width
        _sizes(width=width)
        abi.check(abi.lib.to_rows8_pack(DTYPES[self.dtype], width, 0, bytes(_ROWS.size), bytes(_ROWS8.size), 0),
                  "Checkpoint8")

    def _call(self, fn, name, x, x8, first, stream, device):
        tokens = x.shape[0]
        rows = _ROWS.pack(*_row(x, "x", self.dtype, (tokens, self.width), device))
        kept = _ROWS8.pack(*_row8(x8, "x8", tokens, self.width, device))
        st = fn(DTYPES[self.dtype], self.width, tokens, *((rows, kept) if first else (kept, rows)), _on(stream, device))
        if st:
            abi.check(st, name)

    def pack(self, x, x8: Rows8, stream: Optional[int] = None):
        """x8 <- x in 8 bits."""
        self._call(abi.lib.to_rows8_pack, "to_rows8_pack", x, x8, True, stream, _cuda(x, "x"))
        _written(x8)

    def unpack(self, x8: Rows8, x, stream: Optional[int] = None):
        """x <- the values that x8 stands for."""
        self._call(abi.lib.to_rows8_unpack, "to_rows8_unpack", x, x8, False, stream, _cuda(x, "x"))
        _written(x)


class GatedRecurrence:
    """h_t = a_t h_{t-1} + (1 - a_t) x_t for every channel, with a_t = sigmoid(f_t + bias).

    With complement=False x_t is added as it is.  Prompts (`forward`) are packed
    sequences, single tokens (`step`) update the states in place, `backward`
    gives the gradients of `forward`.  bias: f32 [channels] or None.  States:
    f32 [slots, channels].
    """

    def __init__(self, dtype, channels: int, complement: bool = True):
        self.dtype, self.channels, self.complement = _dtype(dtype), channels, bool(complement)
        _sizes(channels=channels)
        abi.check(abi.lib.to_gated_recurrence(self._desc(0, 0), bytes(_REC_ARGS.size), 0), "GatedRecurrence")

    def _desc(self, tokens: int, nseq: int, slots: int = 0) -> bytes:
        return _REC_DESC.pack(DTYPES[self.dtype], self.channels, nseq, self.complement, tokens, slots)

    def saved_rows(self, tokens: int, sequences: int) -> int:
        """Rows of `saved` (f32 [rows, channels]): a state for every 128 tokens begun, at most."""
        return abi.lib.to_gated_recurrence_saved_rows(self._desc(tokens, sequences))

    def workspace_bytes(self, tokens: int, sequences: int) -> int:
        """Bytes of `workspace` that forward() needs (0: none)."""
        return abi.lib.to_gated_recurrence_workspace_bytes(self._desc(tokens, sequences))

    def backward_workspace_bytes(self, tokens: int, sequences: int) -> int:
        return abi.lib.to_gated_recurrence_backward_workspace_bytes(self._desc(tokens, sequences))

    def _flat(self, t, name, rows, device):
        return _flat(t, name, torch.float32, (rows, self.channels), device)

    def _bias(self, bias, device, name="bias"):
        return _flat(bias, name, torch.float32, (self.channels,), device)

    def _sequences(self, cu_seqlens, device):
        n = cu_seqlens.numel() - 1
        if n < 0:
            raise ValueError("cu_seqlens is empty")
        return n, _flat(cu_seqlens, "cu_seqlens", torch.int32, (n + 1,), device)

    def forward(self, x, f, bias, cu_seqlens, h, state_in=None, state_out=None, slots=None, saved=None,
                keep_x: Optional[Rows8] = None, keep_f: Optional[Rows8] = None, workspace=None,
                stream: Optional[int] = None):
        """h <- the outputs of packed sequences; state_out (may be state_in) <- the states they leave.

        cu_seqlens: int32 [sequences + 1], on the device.  slots: int32
        [sequences], each sequence's place in state_in and state_out (None:
        its number); one outside them means no state.  For backward(): saved
        <- the states that enter every 128 tokens, keep_x, keep_f <- x, f in 8 bits.
        """
        tokens, device = x.shape[0], _cuda(x, "x")
        n, cu = self._sequences(cu_seqlens, device)
        have = n if state_in is None and state_out is None else (state_out if state_in is None else state_in).shape[0]
        if slots is None and have != n:
            raise ValueError(f"{have} states for {n} sequences, and no slots")
        desc, shape = self._desc(tokens, n, have), (tokens, self.channels)
        args = _REC_ARGS.pack(
            *_row(x, "x", self.dtype, shape, device), *_row(f, "f", self.dtype, shape, device),
            *_row(h, "h", self.dtype, shape, device),
            *(_NO_ROWS8 if keep_x is None else _row8(keep_x, "keep_x", *shape, device)),
            *(_NO_ROWS8 if keep_f is None else _row8(keep_f, "keep_f", *shape, device)),
            self._bias(bias, device), cu, _flat(slots, "slots", torch.int32, (n,), device),
            self._flat(state_in, "state_in", have, device), self._flat(state_out, "state_out", have, device),
            0 if saved is None else self._flat(saved, "saved", abi.lib.to_gated_recurrence_saved_rows(desc), device),
            *_scratch(workspace, abi.lib.to_gated_recurrence_workspace_bytes(desc), device))
        st = abi.lib.to_gated_recurrence(desc, args, _on(stream, device))
        if st:
            abi.check(st, "to_gated_recurrence")
        _written(h, state_out, saved, keep_x, keep_f)

    def step(self, x, f, bias, state, h, slots=None, stream: Optional[int] = None):
        """One token of each request: its state is updated in place, h <- its output."""
        tokens, device, have = x.shape[0], _cuda(x, "x"), state.shape[0]
        if slots is None and have < tokens:
            raise ValueError(f"{have} states for {tokens} requests, and no slots")
        shape = (tokens, self.channels)
        args = _REC_ARGS.pack(
            *_row(x, "x", self.dtype, shape, device), *_row(f, "f", self.dtype, shape, device),
            *_row(h, "h", self.dtype, shape, device), *_NO_ROWS8, *_NO_ROWS8, self._bias(bias, device), 0,
            _flat(slots, "slots", torch.int32, (tokens,), device), 0, self._flat(state, "state", have, device), 0, 0, 0)
        st = abi.lib.to_gated_recurrence_step(self._desc(tokens, 0, have), args, _on(stream, device))
        if st:
            abi.check(st, "to_gated_recurrence_step")
        increment_version((h, state))

    def backward(self, x, f, bias, cu_seqlens, saved, dh, dx, df, dbias=None, dstate_out=None, dstate_in=None,
                 workspace=None, stream: Optional[int] = None):
        """dx, df (and dbias, dstate_in) <- gradients of forward() from dh and dstate_out.

        x, f: forward()'s rows, or what it kept of them (Rows8); saved: what it
        saved.  State gradients hold one row a sequence, in order.
        """
        tokens, device = dh.shape[0], _cuda(dh, "dh")
        n, cu = self._sequences(cu_seqlens, device)
        desc, shape = self._desc(tokens, n, n), (tokens, self.channels)
        (rx, x8), (rf, f8) = (_row_or_8(t, name, self.dtype, shape, device) for t, name in ((x, "x"), (f, "f")))
        args = _REC_GRAD_ARGS.pack(
            *rx, *rf, *_row(dh, "dh", self.dtype, shape, device), *_row(dx, "dx", self.dtype, shape, device),
            *_row(df, "df", self.dtype, shape, device), *x8, *f8, self._bias(bias, device), cu,
            self._flat(_needed(saved, "saved"), "saved", abi.lib.to_gated_recurrence_saved_rows(desc), device),
            self._flat(dstate_out, "dstate_out", n, device), self._flat(dstate_in, "dstate_in", n, device),
            self._bias(dbias, device, "dbias"),
            *_scratch(workspace, abi.lib.to_gated_recurrence_backward_workspace_bytes(desc), device))
        st = abi.lib.to_gated_recurrence_backward(desc, args, _on(stream, device))
        if st:
            abi.check(st, "to_gated_recurrence_backward")
        _written(dx, df, dbias, dstate_in)


class BlockNorm:
    """What lies between two blocks: norm of a block's output, gate, residual sum and the next block's norm.

    u = w_post * y / rms(y), r_out = r + scale * u * act(g), n = w_pre * r_out / rms(r_out).

    residual: type of r and r_out (dtype by default, or f32).  gate: None, "linear"
    (act(g) = g), "sigmoid" or "silu".  post_norm=False leaves u = w_post * y.
    w_post, w_pre: f32 [width] or None.
    """

    GATES = {None: 0, "linear": 1, "sigmoid": 2, "silu": 3}

    def __init__(self, dtype, width: int, residual=None, gate: Optional[str] = None, post_norm: bool = True,
                 scale: float = 1.0, eps: float = 1e-6):
        self.dtype, self.width = _dtype(dtype), width
        self.residual = self.dtype if residual is None else _dtype(residual)
        if gate not in self.GATES:
            raise ValueError(f"gate {gate!r}: None, 'linear', 'sigmoid' or 'silu'")
        self.gate = gate
        _sizes(width=width)
        self._desc = _NORM_DESC.pack(DTYPES[self.dtype], DTYPES[self.residual], width, self.GATES[gate],
                                     int(bool(post_norm)), 0, scale, eps)
        abi.check(abi.lib.to_block_norm(self._desc, 0, bytes(_NORM_ARGS.size), 0), "BlockNorm")

    def _gate(self, g, y, name):
        if (g is not None) != (self.gate is not None and y is not None):
            raise ValueError(f"{name} is {'missing' if g is None else 'given'} with gate {self.gate!r}"
                             f"{'' if y is not None else ' and no y'}")

    def forward(self, r, y, g, w_post, w_pre, r_out, n, keep_r: Optional[Rows8] = None,
                keep_y: Optional[Rows8] = None, keep_g: Optional[Rows8] = None, stream: Optional[int] = None):
        """r_out (may be r) <- the residual stream with y joined, n <- the next block's input.

        Without y (None, then r_out and g are None too) n is made of r alone; n
        may be None.  keep_r, keep_y, keep_g <- r_out (r without y), y, g in 8 bits.
        """
        tokens, device = r.shape[0], _cuda(r, "r")
        self._gate(g, y, "g")
        if (y is None) != (r_out is None):
            raise ValueError("y and r_out: one is None, the other is not")
        if y is None and (n is None or keep_y is not None):
            raise ValueError("without y there has to be n, and no keep_y")
        if g is None and keep_g is not None:
            raise ValueError("keep_g without g")
        shape = (tokens, self.width)
        row = lambda t, name, kind: _NO_ROWS if t is None else _row(t, name, kind, shape, device)  # noqa: E731
        kept = lambda t, name: _NO_ROWS8 if t is None else _row8(t, name, *shape, device)  # noqa: E731
        args = _NORM_ARGS.pack(
            *_row(r, "r", self.residual, shape, device), *row(y, "y", self.dtype), *row(g, "g", self.dtype),
            *row(r_out, "r_out", self.residual), *row(n, "n", self.dtype),
            *kept(keep_r, "keep_r"), *kept(keep_y, "keep_y"), *kept(keep_g, "keep_g"),
            _flat(w_post, "w_post", torch.float32, (self.width,), device),
            _flat(w_pre, "w_pre", torch.float32, (self.width,), device))
        st = abi.lib.to_block_norm(self._desc, tokens, args, _on(stream, device))
        if st:
            abi.check(st, "to_block_norm")
        _written(r_out, n, keep_r, keep_y, keep_g)

    def workspace_bytes(self, tokens: int) -> int:
        """Bytes of `workspace` that backward() needs."""
        return abi.lib.to_block_norm_workspace_bytes(self._desc, tokens)

    def backward(self, r_out, y, g, w_post, w_pre, dr_out, dn, dr, dy, dg, dw_post, dw_pre, workspace,
                 stream: Optional[int] = None):
        """dr (may be dr_out), dy, dg, dw_post, dw_pre <- gradients from dr_out and dn (None: zero).

        r_out, y, g: forward()'s rows (r_out without y: r), or what it kept of
        them (Rows8).  dw_post, dw_pre: f32 [width] or None.
        """
        tokens, device = dr.shape[0], _cuda(dr, "dr")
        self._gate(g, y, "g")
        if (y is None) != (dy is None) or (g is None) != (dg is None) or (y is None and dw_post is not None):
            raise ValueError("y and dy, g and dg: one is None, the other is not; or dw_post without y")
        shape = (tokens, self.width)
        row = lambda t, name, kind: _NO_ROWS if t is None else _row(t, name, kind, shape, device)  # noqa: E731
        read = [(_NO_ROWS, _NO_ROWS8) if t is None else _row_or_8(t, name, kind, shape, device)
                for t, name, kind in ((_needed(r_out, "r_out"), "r_out", self.residual), (y, "y", self.dtype),
                                      (g, "g", self.dtype))]
        weights = [_flat(t, name, torch.float32, (self.width,), device)
                   for t, name in ((w_post, "w_post"), (w_pre, "w_pre"), (dw_post, "dw_post"), (dw_pre, "dw_pre"))]
        args = _NORM_GRAD_ARGS.pack(
            *read[0][0], *read[1][0], *read[2][0], *row(dr_out, "dr_out", self.residual), *row(dn, "dn", self.dtype),
            *_row(dr, "dr", self.residual, shape, device), *row(dy, "dy", self.dtype), *row(dg, "dg", self.dtype),
            *read[0][1], *read[1][1], *read[2][1], *weights,
            *_scratch(workspace, int(dw_post is not None or dw_pre is not None), device))
        st = abi.lib.to_block_norm_backward(self._desc, tokens, args, _on(stream, device))
        if st:
            abi.check(st, "to_block_norm_backward")
        _written(dr, dy, dg, dw_post, dw_pre)
