"""64-bit references of the short convolution, the selective scan and token
sampling, with bounds on what 32-bit arithmetic may lose, for the GPU tests.

The bounds are propagated through the same recurrence: every rounding enters
as a relative error of the term it touches, in units of 2^-24 (half a step of
fp32) or of the documented error of the function used."""

import math

import numpy as np
import torch

HALF = {d: torch.finfo(d).eps / 2 for d in (torch.float32, torch.bfloat16, torch.float16)}


def spans(cu, B, T):
    return [(int(a), int(b)) for a, b in zip(cu[:-1], cu[1:])] if cu is not None else [(0, T)] * B


def conv(x, w, bias, act, s0, cu=None):
    """(o, bound on |error| of o, new state). x [B, T, D] or [1, total, D]; s0 [N, W-1, D]."""
    x, w = x.double().cpu(), w.double().cpu()
    o, tol = torch.zeros_like(x), torch.zeros_like(x)
    W, new = w.shape[1], []
    b = torch.zeros(x.shape[2], dtype=torch.float64) if bias is None else bias.double().cpu()
    for n, (lo, hi) in enumerate(spans(cu, *x.shape[:2])):
        row = 0 if cu is not None else n
        line = torch.cat([s0[n].double().cpu(), x[row, lo:hi]])
        new.append(line[len(line) - (W - 1):])
        for t in range(hi - lo):
            terms = line[t:t + W].T * w
            y, mag = terms.sum(1) + b, terms.abs().sum(1) + b.abs()
            if act:
                # slope at most 1.1; e^-y to 2^-21 + |y| 2^-23, the quotient to 2^-22
                y, mag = y * torch.sigmoid(y), 1.1 * mag + (y.abs() * (1 + y.abs() / 4))
            o[row, lo + t], tol[row, lo + t] = y, mag * 2.0 ** -20
    return o, tol, torch.stack(new)


def scan(x, dt, A, B, C, D, z, bias, softplus, h0, cu=None):
    """(o, bound, final state, bound). B, C [.., G, N]; h0 [N, D, N]."""
    x, dt, A, B, C = (t.double().cpu() for t in (x, dt, A, B, C))
    rep = x.shape[2] // B.shape[2]
    o, tol = torch.zeros_like(x), torch.zeros_like(x)
    fin, ftol = [], []
    for n, (lo, hi) in enumerate(spans(cu, *x.shape[:2])):
        row = 0 if cu is not None else n
        h = h0[n].double().cpu()
        H, E = h.abs(), torch.zeros_like(h)  # magnitudes, and the error bound
        for t in range(lo, hi):
            s = dt[row, t] + (0 if bias is None else bias.double().cpu())
            delta = torch.nn.functional.softplus(s, threshold=60.0) if softplus else s
            # the sum rounds once (|s| 2^-24 of e^s), expf and log1pf lose 2^-21
            e_d = 2.0 ** -20 * (1 + s.abs() / 8)
            a = torch.exp(delta[:, None] * A)
            e_a = 2.0 ** -22 + (delta[:, None] * A).abs() * (e_d[:, None] + 2.0 ** -23)
            b, c = (v[row, t].repeat_interleave(rep, 0) for v in (B, C))
            inp = (delta * x[row, t])[:, None] * b
            h, prev = a * h + inp, a * H
            H = prev + inp.abs()
            E = a * E + prev * e_a + inp.abs() * (e_d[:, None] + 2.0 ** -23) + H * 2.0 ** -23
            skip = 0 if D is None else D.double().cpu() * x[row, t]
            y = (h * c).sum(1) + skip
            ey = (E * c.abs()).sum(1) + ((H * c.abs()).sum(1) + abs(skip)) * 2.0 ** -20
            if z is not None:
                zz = z[row, t].double().cpu()
                g = zz * torch.sigmoid(zz)
                y, ey = y * g, ey * g.abs() + (y * g).abs() * 2.0 ** -20 * (1 + zz.abs() / 8)
            o[row, t], tol[row, t] = y, ey
        fin.append(h)
        ftol.append(E)
    return o, tol, torch.stack(fin), torch.stack(ftol)


def check(got, want, tol, what):
    """|got - want| <= tol + half a step of got's own rounding."""
    g = got.detach().double().cpu()
    bound = tol * (1 + 2.0 ** -7) + HALF[got.dtype] * want.abs() + 1e-37
    if got.dtype == torch.float16:
        bound = bound + 2.0 ** -25  # half a step of fp16's smallest values
    bad = ~((g - want).abs() <= bound)
    if bad.any():
        i = int(((g - want).abs() / bound).nan_to_num(1e30).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside their bound; worst "
                             f"{float(g.reshape(-1)[i])} for {float(want.reshape(-1)[i])} +- "
                             f"{float(bound.reshape(-1)[i])}")


def sample(logits, u, temperature, top_k, top_p, min_p):
    """(tokens, logprobs) from the definition, one row after the other; settings are per-row lists."""
    tok, lp = [], []
    for row, uu, t, k, p, m in zip(logits.detach().double().cpu().numpy(), u, temperature, top_k, top_p, min_p):
        ok = np.flatnonzero(row > -np.inf)  # neither -inf nor NaN
        if len(ok) == 0:
            tok.append(-1)
            lp.append(-math.inf)
            continue
        order = ok[np.argsort(-row[ok], kind="stable")]
        best = row[order[0]]
        if not t > 0:
            k, t = 1, 1.0
        if k > 0:
            order = order[:k]
        with np.errstate(invalid="ignore", over="ignore"):
            w = np.where(row[order] == best, 1.0, 0.0 if np.isinf(best) else np.exp((row[order] - best) / t))
        if p < 1:
            before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
            n = max(1, int((before < p * w.sum()).sum()))
            order, w = order[:n], w[:n]
        keep = ((w >= m) | (row[order] == best)) & (w > 0)
        order, w = order[keep], w[keep]
        by = np.argsort(order)
        order, w = order[by], w[by]
        c = np.cumsum(w)
        j = min(int((c <= uu * c[-1]).sum()), len(w) - 1)
        tok.append(int(order[j]))
        lp.append(math.log(w[j] / c[-1]))
    return np.array(tok), np.array(lp)
