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
where they are. Outputs are new contiguous tensors. The operators are
forward only: inputs that ask for gradients are refused.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from . import ops as _ops

_STATES = (8, 16, 32, 64, 128)
_WIDTHS = (2, 3, 4)
_ACTIVATIONS = {None: 0, "silu": 1, "swish": 1}


def _no_grad(*ts):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts):
        raise RuntimeError("this operator has no backward pass: call it under torch.no_grad() or "
                           "with detached tensors")


def _same_device(*ts):
    _ops._require_cuda(*ts)
    ts = [t for t in ts if t is not None]
    if any(t.device != ts[0].device for t in ts):
        raise ValueError(f"tensors lie on different devices: {sorted({str(t.device) for t in ts})}")


def _rows(t: torch.Tensor | None, tail: int = 1):
    """(tensor, batch stride, token stride): ``t`` itself when its last
    ``tail`` axes are dense, else a contiguous copy. Strides of axes of one
    element do not matter and are given as 0."""
    if t is None:
        return None, 0, 0
    want = 1
    for i in range(1, tail + 1):
        if t.shape[-i] > 1 and t.stride(-i) != want:
            t = t.contiguous()
            break
        want *= t.shape[-i]
    return t, t.stride(0) if t.shape[0] > 1 else 0, t.stride(1) if t.shape[1] > 1 else 0


def _sequences(x: torch.Tensor, cu_seqlens):
    """(number of sequences, tokens for the C call, cu_seqlens on the device)."""
    _ops._check_varlen(x, None, cu_seqlens)
    if x.shape[1] >= 1 << 31:
        raise ValueError(f"{x.shape[1]} tokens are more than an int32 counts")
    if cu_seqlens is None:
        return x.shape[0], x.shape[1], None
    if cu_seqlens.dim() != 1 or len(cu_seqlens) < 1:
        raise ValueError("cu_seqlens must be a vector of sequence offsets")
    if not cu_seqlens.is_cuda:
        c = cu_seqlens.to(torch.int64)
        if int(c[0]) < 0 or int(c[-1]) > x.shape[1] or bool((c[1:] < c[:-1]).any()):
            raise ValueError(f"cu_seqlens must ascend within [0, {x.shape[1]}]")
    return len(cu_seqlens) - 1, x.shape[1], _ops._cu(cu_seqlens, x.device)


def _output(out: torch.Tensor | None, x: torch.Tensor, *inputs) -> torch.Tensor:
    """A new contiguous tensor like x, or ``out`` once it is one that no input shares."""
    if out is None:
        return torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if out.shape != x.shape or out.dtype != x.dtype or out.device != x.device or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous {tuple(x.shape)} {x.dtype} tensor on {x.device}")
    lo, hi = out.data_ptr(), out.data_ptr() + out.numel() * out.element_size()
    for t in inputs:
        if t is None or t.numel() == 0 or lo == hi:
            continue
        a = t.data_ptr()
        b = a + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()
        if a < hi and lo < b:
            raise ValueError("out overlaps an input")
    return out


def _bank(bank: torch.Tensor, layer: int, tail: tuple[int, ...], dtype: torch.dtype, what: str):
    if bank.dtype != dtype or not bank.is_contiguous() or bank.dim() != 2 + len(tail):
        raise ValueError(f"the {what} bank must be a contiguous {dtype} tensor [L, S+1, "
                         f"{', '.join(map(str, tail))}]")
    if not 0 <= layer < bank.shape[0]:
        raise IndexError(f"layer {layer} out of range [0, {bank.shape[0]})")
    if tuple(bank.shape[2:]) != tail:
        raise ValueError(f"bank rows of shape {tuple(bank.shape[2:])}, not {tail}")
    return bank[layer]


def _slot_ids(slot_ids, num_slots: int, nseq: int, device) -> torch.Tensor:
    ids = _ops.slot_ids_tensor(slot_ids, num_slots, device)
    if ids.device != device:
        raise ValueError(f"slot ids lie on {ids.device}, not {device}")
    if ids.numel() != nseq:
        raise ValueError(f"{ids.numel()} slot ids for {nseq} sequences")
    return ids


# ---------------------------------------------------------------------------
# short causal convolution
# ---------------------------------------------------------------------------

def _conv_args(x, weight, bias, activation):
    _same_device(x, weight, bias)
    _no_grad(x, weight, bias)
    if x.dim() != 3:
        raise ValueError(f"x must be [B, T, D], not {tuple(x.shape)}")
    if x.dtype not in _ops._DTYPES:
        raise ValueError(f"unsupported dtype {x.dtype}")
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation must be None or 'silu', not {activation!r}")
    D = x.shape[2]
    if weight.dim() == 3 and weight.shape[1] == 1:  # a depthwise Conv1d's [D, 1, W]
        weight = weight[:, 0]
    if weight.dim() != 2 or weight.shape[0] != D:
        raise ValueError(f"weight must be [{D}, W], not {tuple(weight.shape)}")
    if weight.shape[1] not in _WIDTHS:
        raise ValueError(f"a width of {weight.shape[1]} is not supported (2, 3 or 4)")
    if bias is not None and tuple(bias.shape) != (D,):
        raise ValueError(f"bias must be [{D}], not {tuple(bias.shape)}")
    weight = weight.to(x.dtype).contiguous()
    bias = None if bias is None else bias.to(x.dtype).contiguous()
    return weight, bias, _ACTIVATIONS[activation]


def short_conv(x, weight, bias=None, activation: str | None = None, initial_state=None,
               output_final_state: bool = False, cu_seqlens=None):
    """Short causal convolution: o[t, d] = act(bias[d] + sum_j weight[d, j] x[t-W+1+j, d]).

    x [B, T, D] or packed [1, total, D] with ``cu_seqlens``; weight [D, W] (or
    [D, 1, W]) with W in 2..4; activation None or "silu". ``initial_state``
    [N, W-1, D] in x's dtype holds the inputs before each sequence's first
    token, oldest first (None: zeros). Returns (o, final_state), the last W-1
    inputs of each sequence when ``output_final_state``, else None."""
    weight, bias, act = _conv_args(x, weight, bias, activation)
    _same_device(x, initial_state)
    N, T, cu = _sequences(x, cu_seqlens)
    D, W = weight.shape
    if initial_state is not None:
        _no_grad(initial_state)
        if tuple(initial_state.shape) != (N, W - 1, D):
            raise ValueError(f"initial_state must be {(N, W - 1, D)}, not {tuple(initial_state.shape)}")
        initial_state = initial_state.to(x.dtype).contiguous()
    x, bs, ts = _rows(x)
    o = _output(None, x)
    st = torch.empty(N, W - 1, D, dtype=x.dtype, device=x.device) if output_final_state else None
    p = _ops._ptr
    with torch.cuda.device(x.device):
        _lib.call("wkvm_short_conv", p(x), bs, ts, p(weight), p(bias), p(o), p(initial_state), p(st),
                  p(cu), N, T, D, W, act, _ops._DTYPES[x.dtype], p(_ops.status_word(x.device)),
                  _ops._stream(x.device))
    return o, st


def _conv_slots(x, weight, bank_conv, layer, slot_ids, bias, activation, cu_seqlens, out):
    weight, bias, act = _conv_args(x, weight, bias, activation)
    _same_device(x, bank_conv)
    N, T, cu = _sequences(x, cu_seqlens)
    D, W = weight.shape
    layer_t = _bank(bank_conv, layer, (W - 1, D), x.dtype, "conv")
    ids = _slot_ids(slot_ids, layer_t.shape[0], N, x.device)
    x, bs, ts = _rows(x)
    o = _output(out, x, x, layer_t)
    p = _ops._ptr
    with torch.cuda.device(x.device):
        _lib.call("wkvm_short_conv_slots", p(x), bs, ts, p(weight), p(bias), p(o), p(layer_t),
                  layer_t.shape[0], p(ids), p(cu), N, T, D, W, act, _ops._DTYPES[x.dtype],
                  p(_ops.status_word(x.device)), _ops._stream(x.device))
    return o


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
    """Checked arguments of a selective scan in the C call's order."""

    def __init__(self, x, dt, A, B, C, D, z, dt_bias, cu_seqlens):
        _same_device(x, dt, A, B, C, D, z, dt_bias)
        _no_grad(x, dt, A, B, C, D, z, dt_bias)
        if x.dim() != 3:
            raise ValueError(f"x must be [B, T, D], not {tuple(x.shape)}")
        d = x.shape[2]
        for name, t in (("dt", dt), ("z", z)):
            if t is not None and t.shape != x.shape:
                raise ValueError(f"{name} must have x's shape {tuple(x.shape)}, not {tuple(t.shape)}")
        if A.dim() != 2 or A.shape[0] != d:
            raise ValueError(f"A must be [{d}, N], not {tuple(A.shape)}")
        n = A.shape[1]
        if n not in _STATES:
            raise ValueError(f"{n} states per channel are not supported (8, 16, 32, 64 or 128)")
        B, C = (t.unsqueeze(2) if t.dim() == 3 else t for t in (B, C))
        for name, t in (("B", B), ("C", C)):
            if t.dim() != 4 or t.shape[:2] != x.shape[:2] or t.shape[3] != n or t.shape != B.shape:
                raise ValueError(f"{name} must be [B, T, N] or [B, T, G, N] with N = {n}, "
                                 f"not {tuple(t.shape)}")
        g = B.shape[2]
        if g < 1 or d % g:
            raise ValueError(f"{d} channels do not split into {g} groups")
        for name, t in (("D", D), ("dt_bias", dt_bias)):
            if t is not None and tuple(t.shape) != (d,):
                raise ValueError(f"{name} must be [{d}], not {tuple(t.shape)}")
        self.dtype = x.dtype  # the output's
        acts = [t for t in (x, dt, B, C, z) if t is not None]
        if x.dtype not in _ops._DTYPES or any(t.dtype != x.dtype for t in acts):
            # mixed dtypes are widened to fp32 (lossless), as the other ops do
            x, dt, B, C, z = (None if t is None else t.float() for t in (x, dt, B, C, z))
        self.nseq, self.T, self.cu = _sequences(x, cu_seqlens)
        self.x, self.shape = x, (self.nseq, self.T, d, n, g)
        rows = [_rows(x), _rows(dt), _rows(z), _rows(B, 2), _rows(C, 2)]
        x, dt, z, B, C = (r[0] for r in rows)
        f32 = lambda t: None if t is None else t.float().contiguous()  # noqa: E731
        # kept alive until the launch: some are copies made here
        self.inputs = (x, dt, f32(A), B, C, f32(D), z, f32(dt_bias))
        self.strides = (ctypes.c_int64 * 10)(*(s for r in rows for s in r[1:]))

    def call(self, entry, o, *state, softplus):
        p, dev = _ops._ptr, self.x.device
        with torch.cuda.device(dev):
            _lib.call(entry, *(p(t) for t in self.inputs), p(o), self.strides, *state, p(self.cu),
                      *self.shape, int(bool(softplus)), _ops._DTYPES[self.x.dtype],
                      p(_ops.status_word(dev)), _ops._stream(dev))


def selective_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, dt_softplus: bool = True,
                   initial_state=None, output_final_state: bool = False, cu_seqlens=None):
    """Selective state space scan. Per token, channel d and state n, with
    delta = softplus(dt + dt_bias) (dt + dt_bias without ``dt_softplus``):

      h[d, n] = exp(delta A[d, n]) h[d, n] + delta x[d] B[g, n]
      o[d] = (sum_n C[g, n] h[d, n] + D[d] x[d]) * silu(z[d])

    x, dt, z [B, T, D] or packed [1, total, D] with ``cu_seqlens``; A [D, N];
    B, C [B, T, N] or [B, T, G, N], channel d in group g = d // (D // G);
    D, dt_bias [D]; z, D and dt_bias optional. N in 8, 16, 32, 64, 128.
    States are fp32 [sequences, D, N]. Returns (o, final_state): o in x's
    dtype, final_state fp32 when ``output_final_state``, else None."""
    a = _Scan(x, dt, A, B, C, D, z, dt_bias, cu_seqlens)
    want = (a.nseq, a.shape[2], a.shape[3])
    if initial_state is not None:
        _same_device(x, initial_state)
        _no_grad(initial_state)
        if tuple(initial_state.shape) != want:
            raise ValueError(f"initial_state must be {want}, not {tuple(initial_state.shape)}")
    h0 = _ops._state(initial_state)
    o = _output(None, a.x)
    ht = torch.empty(want, dtype=torch.float32, device=x.device) if output_final_state else None
    a.call("wkvm_selective_scan", o, _ops._ptr(h0), _ops._ptr(ht), softplus=dt_softplus)
    return o.to(a.dtype), ht


def _scan_slots(x, dt, A, B, C, bank_ssm, layer, slot_ids, D, z, dt_bias, dt_softplus, cu_seqlens, out):
    a = _Scan(x, dt, A, B, C, D, z, dt_bias, cu_seqlens)
    _same_device(x, bank_ssm)
    layer_t = _bank(bank_ssm, layer, a.shape[2:4], torch.float32, "ssm")
    ids = _slot_ids(slot_ids, layer_t.shape[0], a.nseq, x.device)
    # a promoted call computes in fp32 and rounds into `out` afterwards
    direct = a.x.dtype == a.dtype
    if out is not None:
        _output(out, x, *a.inputs, layer_t)
    o = out if direct and out is not None else _output(None, a.x)
    a.call("wkvm_selective_scan_slots", o, _ops._ptr(layer_t), layer_t.shape[0], _ops._ptr(ids),
           softplus=dt_softplus)
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
