"""Choice of the next tokens from logits and given uniform numbers."""

from __future__ import annotations

import torch

from . import _lib
from . import ops as _ops


# WKVM_SAMPLE_MAX_VOCAB: there the masses' rounding reaches two steps of an fp32 u
MAX_VOCAB = 1 << 20


def _setting(name: str, value, rows: int, dtype: torch.dtype, logits: torch.Tensor):
    """(per-row device tensor or None, scalar) of one sampling setting."""
    if not isinstance(value, torch.Tensor):
        if value is None or not value >= 0:
            raise ValueError(f"{name} must be >= 0, not {value!r}")
        if dtype is torch.int32:
            if value == float("inf") or value != int(value):
                raise ValueError(f"{name} must be a whole number, not {value!r}")
            value = int(value)
        return None, value
    if value.dim() == 0:
        value = value.expand(rows)
    if value.dim() != 1 or value.shape[0] != rows:
        raise ValueError(f"{name} must be a number or [{rows}], not {tuple(value.shape)}")
    if value.dtype is dtype and value.get_device() == logits.get_device() and value.is_contiguous():
        return value, 0
    if dtype is torch.int32 and value.dtype is not torch.int32:
        # a fraction is rounded up, so that it never becomes the 0 that keeps all
        value = (value.ceil() if value.is_floating_point() else value).clamp(0, 1 << 30)
    return value.to(device=logits.device, dtype=dtype).contiguous(), 0


def sample_tokens(logits: torch.Tensor, u: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0,
                  min_p=0.0) -> tuple[torch.Tensor, torch.Tensor]:
    """One token per row of ``logits`` [B, V], drawn with the uniform numbers
    ``u`` [B] in [0, 1) under temperature, top-k, top-p and min-p (each a
    number, or a [B] tensor with a value per row). Returns (tokens int64 [B],
    logprobs fp32 [B]), the log-probabilities under the filtered distribution.

    With w_i = exp((l_i - max l) / temperature): ``top_k`` keeps the k largest
    logits (0: all; a whole number, fractions in a tensor are rounded up);
    ``top_p`` keeps, of those in descending order, the shortest prefix that
    holds at least that share of their mass (1: all); ``min_p`` keeps, of
    those, w_i >= min_p (0: all). The token is the first kept id whose running
    mass, over ascending ids, exceeds u times the mass kept. Masses count in
    units of 2^-46 at 65,536 logits; a weight of less than half a unit is never
    drawn. Ties go to the lowest ids; temperature 0 is greedy. -inf (and NaN)
    logits are never chosen; a row of nothing else gives token -1 and
    log-probability -inf. The same inputs give the same tokens on every run,
    eagerly and in a captured graph. Forward only: inputs that ask for
    gradients are refused."""
    idx = logits.get_device()
    if idx < 0 or u.get_device() != idx:
        _ops._require_cuda(logits, u)
        if u.device != logits.device:
            raise ValueError(f"u must be on {logits.device}, not {u.device}")
    if torch.is_grad_enabled():
        for t in (logits, u, temperature, top_p, min_p):
            if isinstance(t, torch.Tensor) and t.requires_grad:
                raise RuntimeError("this operator has no backward pass: call it under torch.no_grad() or "
                                   "with detached tensors")
    if logits.dim() != 2:
        raise ValueError(f"logits must be [B, V], not {tuple(logits.shape)}")
    if logits.dtype not in _ops._DTYPES:
        raise ValueError(f"unsupported dtype {logits.dtype}")
    B, V = logits.shape
    if V < 1 or V > MAX_VOCAB:
        raise ValueError(f"a vocabulary of {V} is not supported")
    if B >= 1 << 31:
        raise ValueError(f"{B} rows are more than an int32 counts")
    if u.dim() != 1 or u.shape[0] != B:
        raise ValueError(f"u must be [{B}], not {tuple(u.shape)}")
    temp, temp0 = _setting("temperature", temperature, B, torch.float32, logits)
    k, k0 = _setting("top_k", top_k, B, torch.int32, logits)
    tp, tp0 = _setting("top_p", top_p, B, torch.float32, logits)
    mp, mp0 = _setting("min_p", min_p, B, torch.float32, logits)
    if mp0 > 1:
        raise ValueError(f"min_p must be <= 1, not {mp0!r}")
    stride, last = logits.stride()
    if last != 1 and V > 1:
        logits = logits.contiguous()
        stride = V
    if u.dtype is not torch.float32 or not u.is_contiguous():
        u = u.to(torch.float32).contiguous()
    tokens, logprobs = torch.empty_like(u, dtype=torch.int64), torch.empty_like(u)
    p = _ops._ptr
    _ops._launch("wkvm_sample_tokens", idx, logits.data_ptr(), stride, u.data_ptr(), p(temp), p(k), p(tp), p(mp),
                 float(temp0), min(k0, V), float(tp0), float(mp0), tokens.data_ptr(), logprobs.data_ptr(), B, V,
                 _ops._DTYPES[logits.dtype])
    return tokens, logprobs
