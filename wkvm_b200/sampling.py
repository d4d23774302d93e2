"""Choice of the next tokens from logits and given uniform numbers."""

from __future__ import annotations

import torch

from . import _lib
from . import ops as _ops


def _setting(name: str, value, rows: int, dtype: torch.dtype, device):
    """(per-row device tensor or None, scalar) of one sampling setting."""
    if not isinstance(value, torch.Tensor):
        return None, value
    if value.dim() == 0:
        value = value.expand(rows)
    if tuple(value.shape) != (rows,):
        raise ValueError(f"{name} must be a number or [{rows}], not {tuple(value.shape)}")
    return value.to(device=device, dtype=dtype).contiguous(), 0


def sample_tokens(logits: torch.Tensor, u: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0,
                  min_p=0.0) -> tuple[torch.Tensor, torch.Tensor]:
    """One token per row of ``logits`` [B, V], drawn with the uniform numbers
    ``u`` [B] in [0, 1) under temperature, top-k, top-p and min-p (each a
    number, or a [B] tensor with a value per row). Returns (tokens int64 [B],
    logprobs fp32 [B]), the log-probabilities under the filtered distribution.

    With w_i = exp((l_i - max l) / temperature): ``top_k`` keeps the k largest
    logits (0: all); ``top_p`` keeps, of those in descending order, the
    shortest prefix that holds at least that share of their mass (1: all);
    ``min_p`` keeps, of those, w_i >= min_p (0: all). The token is the first
    kept id whose running mass, over ascending ids, exceeds u times the mass
    kept. Ties go to the lowest ids; temperature 0 is greedy. -inf (and NaN)
    logits are never chosen; a row of nothing else gives token -1 and
    log-probability -inf. The same inputs give the same tokens on every run,
    eagerly and in a captured graph."""
    _ops._require_cuda(logits, u)
    if logits.dim() != 2:
        raise ValueError(f"logits must be [B, V], not {tuple(logits.shape)}")
    if logits.dtype not in _ops._DTYPES:
        raise ValueError(f"unsupported dtype {logits.dtype}")
    B, V = logits.shape
    if V < 1 or V >= 1 << 31:
        raise ValueError(f"a vocabulary of {V} is not supported")
    if tuple(u.shape) != (B,) or u.device != logits.device:
        raise ValueError(f"u must be [{B}] on {logits.device}")
    dev = logits.device
    temp, temp0 = _setting("temperature", temperature, B, torch.float32, dev)
    k, k0 = _setting("top_k", top_k, B, torch.int32, dev)
    tp, tp0 = _setting("top_p", top_p, B, torch.float32, dev)
    mp, mp0 = _setting("min_p", min_p, B, torch.float32, dev)
    for name, v in (("temperature", temp0), ("top_k", k0), ("top_p", tp0), ("min_p", mp0)):
        if v is None or not v >= 0:
            raise ValueError(f"{name} must be >= 0, not {v!r}")
    if mp0 > 1:
        raise ValueError(f"min_p must be <= 1, not {mp0!r}")
    if V > 1 and logits.stride(1) != 1:
        logits = logits.contiguous()
    u = u.to(torch.float32).contiguous()
    tokens = torch.empty(B, dtype=torch.int64, device=dev)
    logprobs = torch.empty(B, dtype=torch.float32, device=dev)
    p = _ops._ptr
    with torch.cuda.device(dev):
        _lib.call("wkvm_sample_tokens", p(logits), logits.stride(0) if B > 1 else V, p(u), p(temp), p(k),
                  p(tp), p(mp), float(temp0), min(int(k0), V), float(tp0), float(mp0), p(tokens), p(logprobs),
                  B, V, _ops._DTYPES[logits.dtype], _ops._stream(dev))
    return tokens, logprobs
