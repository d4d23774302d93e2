"""Selective state space layers over slots: the short causal convolution and
the selective scan, for prompts (batched or packed) and for single tokens.

A layer's mixer is: projection -> short convolution -> projections of dt, B
and C -> selective scan -> output projection. Both operators keep a state per
request, and both states are families of a bank
(:class:`wkvm_b200.state.SSMStateBank`), read and written in place by slot id:

  conv [L, S+1, W-1, D] activation dtype: the last W-1 inputs, oldest first
  ssm  [L, S+1, D, N] fp32

Activations are [B, T, D], or [1, total, D] with cu_seqlens; views whose last
axis is contiguous (one half of a projection's output, a slice of it) are read
where they are. Outputs are new contiguous tensors; tokens of a packed axis
that no sequence covers are not written. Slot ids of one call differ, but for
padding rows, which may share slot 0. The operators are forward only: inputs
that ask for gradients are refused.
"""

from __future__ import annotations

import struct

import torch

from . import _lib
from . import ops as _ops

_STATES = (8, 16, 32, 64, 128)
_WIDTHS = (2, 3, 4)
_INT32 = (1 << 31) - 1
_ACTIVATIONS = {None: 0, "silu": 1, "swish": 1}
_strides = struct.Struct("10q").pack  # the C call's array of ten int64


def _check(ts) -> int:
    """The index of the one device that holds every tensor of ``ts``; refuses
    CPU tensors and inputs that ask for gradients."""
    idx = ts[0].get_device()
    for t in ts:
        if t.get_device() != idx or idx < 0:
            _ops._require_cuda(*ts)
            if len({t.device for t in ts}) > 1:
                raise ValueError(f"tensors lie on different devices: {sorted({str(t.device) for t in ts})}")
            break
    if torch.is_grad_enabled():
        for t in ts:
            if t.requires_grad:
                raise RuntimeError("this operator has no backward pass: call it under torch.no_grad() or "
                                   "with detached tensors")
    return idx


def _rows(t: torch.Tensor, tail: int = 1):
    """(tensor, its strides): ``t`` itself when its last ``tail`` axes are
    dense, else a contiguous copy."""
    s = t.stride()
    if s[-1] != 1 or (tail == 2 and s[-2] != t.shape[-1]):
        t = t.contiguous()
        s = t.stride()
    return t, s


def _new_like(x: torch.Tensor) -> torch.Tensor:
    # (torch.empty with a shape, a dtype and a device takes three times as long)
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def _f32(t: torch.Tensor | None) -> torch.Tensor | None:
    if t is None or (t.dtype is torch.float32 and t.is_contiguous()):
        return t
    return t.float().contiguous()


def _sequences(x: torch.Tensor, cu_seqlens):
    """(number of sequences, tokens for the C call, cu_seqlens on the device)."""
    B, T, D = x.shape
    if B > _INT32 or T > _INT32 or D > _INT32:
        raise ValueError(f"a size of {(B, T, D)} is more than an int32 counts")
    if cu_seqlens is None:
        return B, T, None
    _ops._check_varlen(x, None, cu_seqlens)
    if cu_seqlens.dim() != 1 or len(cu_seqlens) < 1 or cu_seqlens.is_floating_point():
        raise ValueError("cu_seqlens must be a vector of sequence offsets")
    if not cu_seqlens.is_cuda:
        c = cu_seqlens.to(torch.int64)
        if int(c[0]) < 0 or int(c[-1]) > T or bool((c[1:] < c[:-1]).any()):
            raise ValueError(f"cu_seqlens must ascend within [0, {T}]")
    return len(cu_seqlens) - 1, T, _ops._cu(cu_seqlens, x.device)


def _output(out: torch.Tensor, x: torch.Tensor, dtype, inputs) -> torch.Tensor:
    """``out`` once it is a contiguous tensor like x that no input shares."""
    if out.shape != x.shape or out.dtype != dtype or out.device != x.device or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous {tuple(x.shape)} {dtype} tensor on {x.device}")
    lo, hi = out.data_ptr(), out.data_ptr() + out.numel() * out.element_size()
    for t in inputs:
        if t is None or t.numel() == 0 or lo == hi:
            continue
        a = t.data_ptr()
        b = a + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()
        if a < hi and lo < b:
            raise ValueError("out overlaps an input")
    return out


def _bank_rows(bank: torch.Tensor, layer: int, rows: int, cols: int, dtype: torch.dtype, what: str):
    """(address, number of slots) of one layer of a family tensor [L, S+1, rows, cols]."""
    if bank.dtype is not dtype or bank.dim() != 4 or not bank.is_contiguous():
        raise ValueError(f"the {what} bank must be a contiguous {dtype} tensor [L, S+1, {rows}, {cols}]")
    L, slots, r, c = bank.shape
    if r != rows or c != cols:
        raise ValueError(f"bank rows of shape ({r}, {c}), not ({rows}, {cols})")
    if not 0 <= layer < L:
        raise IndexError(f"layer {layer} out of range [0, {L})")
    return bank.data_ptr() + layer * slots * rows * cols * bank.element_size(), slots


def _slot_ids(slot_ids, num_slots: int, nseq: int, x: torch.Tensor) -> torch.Tensor:
    ids = _ops.slot_ids_tensor(slot_ids, num_slots, x.device)
    if ids.get_device() != x.get_device():
        raise ValueError(f"slot ids lie on {ids.device}, not {x.device}")
    if ids.numel() != nseq:
        raise ValueError(f"{ids.numel()} slot ids for {nseq} sequences")
    return ids


# ---------------------------------------------------------------------------
# short causal convolution
# ---------------------------------------------------------------------------

def _conv_args(x, weight, bias, activation, *state):
    """(device index, D, W, weight, bias, activation code), checked."""
    idx = _check([t for t in (x, weight, bias, *state) if t is not None])
    if x.dim() != 3:
        raise ValueError(f"x must be [B, T, D], not {tuple(x.shape)}")
    dtype, D = x.dtype, x.shape[2]
    if dtype not in _ops._DTYPES:
        raise ValueError(f"unsupported dtype {dtype}")
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation must be None or 'silu', not {activation!r}")
    if weight.dim() == 3 and weight.shape[1] == 1:  # a depthwise Conv1d's [D, 1, W]
        weight = weight[:, 0]
    if weight.dim() != 2 or weight.shape[0] != D:
        raise ValueError(f"weight must be [{D}, W], not {tuple(weight.shape)}")
    W = weight.shape[1]
    if W not in _WIDTHS:
        raise ValueError(f"a width of {W} is not supported (2, 3 or 4)")
    if weight.dtype is not dtype or not weight.is_contiguous():
        weight = weight.to(dtype).contiguous()
    if bias is not None:
        if bias.dim() != 1 or bias.shape[0] != D:
            raise ValueError(f"bias must be [{D}], not {tuple(bias.shape)}")
        if bias.dtype is not dtype or not bias.is_contiguous():
            bias = bias.to(dtype).contiguous()
    return idx, D, W, weight, bias, _ACTIVATIONS[activation]


def short_conv(x, weight, bias=None, activation: str | None = None, initial_state=None,
               output_final_state: bool = False, cu_seqlens=None):
    """Short causal convolution: o[t, d] = act(bias[d] + sum_j weight[d, j] x[t-W+1+j, d]).

    x [B, T, D] or packed [1, total, D] with ``cu_seqlens``; weight [D, W] (or
    [D, 1, W]) with W in 2..4; activation None or "silu". A weight, bias or
    state of another dtype is rounded to x's; sums are fp32. ``initial_state``
    [N, W-1, D] in x's dtype holds the inputs before each sequence's first
    token, oldest first (None: zeros). Returns (o, final_state), the last W-1
    inputs of each sequence when ``output_final_state``, else None."""
    idx, D, W, weight, bias, act = _conv_args(x, weight, bias, activation, initial_state)
    N, T, cu = _sequences(x, cu_seqlens)
    if initial_state is not None:
        if tuple(initial_state.shape) != (N, W - 1, D):
            raise ValueError(f"initial_state must be {(N, W - 1, D)}, not {tuple(initial_state.shape)}")
        initial_state = initial_state.to(x.dtype).contiguous()
    x, (bs, ts, _) = _rows(x)
    o = _new_like(x)
    st = torch.empty(N, W - 1, D, dtype=x.dtype, device=x.device) if output_final_state else None
    p = _ops._ptr
    _ops._launch("wkvm_short_conv", idx, p(x), bs, ts, p(weight), p(bias), p(o), p(initial_state), p(st), p(cu),
                 N, T, D, W, act, _ops._DTYPES[x.dtype])
    return o, st


def _conv_slots(x, weight, bank_conv, layer, slot_ids, bias, activation, cu_seqlens, out):
    idx, D, W, weight, bias, act = _conv_args(x, weight, bias, activation, bank_conv)
    N, T, cu = _sequences(x, cu_seqlens)
    rows, slots = _bank_rows(bank_conv, layer, W - 1, D, x.dtype, "conv")
    ids = _slot_ids(slot_ids, slots, N, x)
    x, (bs, ts, _) = _rows(x)
    if out is None:
        out = _new_like(x)
    else:
        _output(out, x, x.dtype, (x, weight, bias, bank_conv))
    p = _ops._ptr
    _ops._launch("wkvm_short_conv_slots", idx, p(x), bs, ts, p(weight), p(bias), p(out), rows, slots, p(ids), p(cu),
                 N, T, D, W, act, _ops._DTYPES[x.dtype])
    return out


def short_conv_decode_slots(x, weight, bank_conv: torch.Tensor, layer: int, slot_ids, bias=None,
                            activation: str | None = None,
                            out: torch.Tensor | None = None) -> torch.Tensor:
    """Short causal convolution of T new tokens per row, x [B, T, D], with the
    last W-1 inputs of row i in bank_conv[layer, slot_ids[i]] ([L, S+1, W-1, D]
    in x's dtype, updated in place). Returns o [B, T, D]."""
    return _conv_slots(x, weight, bank_conv, layer, slot_ids, bias, activation, None, out)


def short_conv_prefill_slots(x, weight, bank_conv: torch.Tensor, layer: int, slot_ids, bias=None,
                             activation: str | None = None, cu_seqlens=None,
                             out: torch.Tensor | None = None) -> torch.Tensor:
    """The same over prompts: x [B, T, D], or [1, total, D] with cu_seqlens."""
    return _conv_slots(x, weight, bank_conv, layer, slot_ids, bias, activation, cu_seqlens, out)


# ---------------------------------------------------------------------------
# selective scan
# ---------------------------------------------------------------------------

class _Scan:
    """Checked arguments of a selective scan, and its C call."""

    __slots__ = ("idx", "dtype", "code", "nseq", "T", "d", "n", "g", "cu", "x", "inputs", "strides")

    def __init__(self, x, dt, A, B, C, D, z, dt_bias, state, cu_seqlens):
        self.idx = _check([t for t in (x, dt, A, B, C, D, z, dt_bias, state) if t is not None])
        shape = x.shape
        if len(shape) != 3:
            raise ValueError(f"x must be [B, T, D], not {tuple(shape)}")
        d = shape[2]
        if dt.shape != shape:
            raise ValueError(f"dt must have x's shape {tuple(shape)}, not {tuple(dt.shape)}")
        if z is not None and z.shape != shape:
            raise ValueError(f"z must have x's shape {tuple(shape)}, not {tuple(z.shape)}")
        if A.dim() != 2 or A.shape[0] != d:
            raise ValueError(f"A must be [{d}, N], not {tuple(A.shape)}")
        n = A.shape[1]
        if n not in _STATES:
            raise ValueError(f"{n} states per channel are not supported (8, 16, 32, 64 or 128)")
        grouped = B.dim() == 4
        want = (shape[0], shape[1], B.shape[2], n) if grouped else (shape[0], shape[1], n)
        for name, t in (("B", B), ("C", C)):
            if t.shape != want:
                raise ValueError(f"{name} must be [B, T, N] or [B, T, G, N] with N = {n} and as many groups as B, "
                                 f"not {tuple(t.shape)}")
        g = want[2] if grouped else 1
        if g < 1 or d % g:
            raise ValueError(f"{d} channels do not split into {g} groups")
        for name, t in (("D", D), ("dt_bias", dt_bias)):
            if t is not None and (t.dim() != 1 or t.shape[0] != d):
                raise ValueError(f"{name} must be [{d}], not {tuple(t.shape)}")
        self.dtype = dtype = x.dtype  # the output's
        if dtype not in _ops._DTYPES:
            raise ValueError(f"unsupported dtype {dtype}")
        if (dt.dtype is not dtype or B.dtype is not dtype or C.dtype is not dtype
                or (z is not None and z.dtype is not dtype)):
            # mixed dtypes are widened to fp32 (lossless), as the other ops do
            x, dt, B, C, z = (None if t is None else t.float() for t in (x, dt, B, C, z))
        self.nseq, self.T, self.cu = _sequences(x, cu_seqlens)
        self.d, self.n, self.g, self.code = d, n, g, _ops._DTYPES[x.dtype]
        tail = 2 if grouped else 1
        x, xs = _rows(x)
        dt, ds = _rows(dt)
        B, bs = _rows(B, tail)
        C, cs = _rows(C, tail)
        z, zs = (None, (0, 0)) if z is None else _rows(z)
        self.x = x
        # kept until the launch: some are copies made here
        self.inputs = (x, dt, _f32(A), B, C, _f32(D), z, _f32(dt_bias))
        self.strides = _strides(xs[0], xs[1], ds[0], ds[1], zs[0], zs[1], bs[0], bs[1], cs[0], cs[1])

    def output(self):
        return _new_like(self.x)

    def call(self, entry, o, softplus, *state):
        p = _ops._ptr
        x, dt, A, B, C, D, z, bias = self.inputs
        _ops._launch(entry, self.idx, x.data_ptr(), dt.data_ptr(), A.data_ptr(), B.data_ptr(), C.data_ptr(), p(D),
                     p(z), p(bias), o.data_ptr(), self.strides, *state, p(self.cu), self.nseq, self.T, self.d,
                     self.n, self.g, 1 if softplus else 0, self.code)


def selective_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, dt_softplus: bool = True,
                   initial_state=None, output_final_state: bool = False, cu_seqlens=None):
    """Selective state space scan. Per token, channel d and state n, with
    delta = softplus(dt + dt_bias) (dt + dt_bias without ``dt_softplus``):

      h[d, n] = exp(delta A[d, n]) h[d, n] + delta x[d] B[g, n]
      o[d] = (sum_n C[g, n] h[d, n] + D[d] x[d]) * silu(z[d])

    x, dt, z [B, T, D] or packed [1, total, D] with ``cu_seqlens``; A [D, N];
    B, C [B, T, N] or [B, T, G, N], channel d in group g = d // (D // G);
    D, dt_bias [D]; z, D and dt_bias optional. N in 8, 16, 32, 64, 128.
    States are fp32 [sequences, D, N]; A and states start on 16 bytes.
    Returns (o, final_state): o in x's dtype, final_state fp32 when
    ``output_final_state``, else None."""
    a = _Scan(x, dt, A, B, C, D, z, dt_bias, initial_state, cu_seqlens)
    want = (a.nseq, a.d, a.n)
    if initial_state is not None and tuple(initial_state.shape) != want:
        raise ValueError(f"initial_state must be {want}, not {tuple(initial_state.shape)}")
    h0 = _ops._state(initial_state)
    o = a.output()
    ht = torch.empty(want, dtype=torch.float32, device=x.device) if output_final_state else None
    a.call("wkvm_selective_scan", o, dt_softplus, _ops._ptr(h0), _ops._ptr(ht))
    return o.to(a.dtype), ht


def _scan_slots(x, dt, A, B, C, bank_ssm, layer, slot_ids, D, z, dt_bias, dt_softplus, cu_seqlens, out):
    a = _Scan(x, dt, A, B, C, D, z, dt_bias, bank_ssm, cu_seqlens)
    rows, slots = _bank_rows(bank_ssm, layer, a.d, a.n, torch.float32, "ssm")
    ids = _slot_ids(slot_ids, slots, a.nseq, x)
    if out is not None:
        _output(out, x, a.dtype, (x, *a.inputs, bank_ssm))
    # a call of mixed dtypes computes in fp32 and rounds into `out` afterwards
    direct = a.x.dtype is a.dtype
    o = out if direct and out is not None else a.output()
    a.call("wkvm_selective_scan_slots", o, dt_softplus, rows, slots, ids.data_ptr())
    if direct:
        return o
    return o.to(a.dtype) if out is None else out.copy_(o)


def selective_scan_decode_slots(x, dt, A, B, C, bank_ssm: torch.Tensor, layer: int, slot_ids, D=None,
                                z=None, dt_bias=None, dt_softplus: bool = True,
                                out: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`selective_scan` of T new tokens per row with the state of row i
    in bank_ssm[layer, slot_ids[i]] ([L, S+1, D, N] fp32, updated in place).
    Returns o [B, T, D]."""
    return _scan_slots(x, dt, A, B, C, bank_ssm, layer, slot_ids, D, z, dt_bias, dt_softplus, None, out)


def selective_scan_prefill_slots(x, dt, A, B, C, bank_ssm: torch.Tensor, layer: int, slot_ids, D=None,
                                 z=None, dt_bias=None, dt_softplus: bool = True, cu_seqlens=None,
                                 out: torch.Tensor | None = None) -> torch.Tensor:
    """The same over prompts: x [B, T, D], or [1, total, D] with cu_seqlens."""
    return _scan_slots(x, dt, A, B, C, bank_ssm, layer, slot_ids, D, z, dt_bias, dt_softplus, cu_seqlens,
                       out)
