"""Token sampling at the edges of what its documentation allows: rows whose
CTAs start apart, two host threads, settings and numbers at their limits."""

import math

import numpy as np
import pytest
import torch

import ssm_ref
import wkvm_b200 as wk

pytestmark = pytest.mark.gpu

BF, FH, F32 = torch.bfloat16, torch.float16, torch.float32
INF, NAN = math.inf, math.nan


def _logits(B, V, seed, cuda, dtype=F32):
    g = torch.Generator(device=cuda).manual_seed(seed)
    x = 2.5 * torch.randn(B, V, generator=g, device=cuda)
    x.scatter_add_(1, torch.randint(0, V, (B, 8), generator=g, device=cuda),
                   4 + 6 * torch.rand(B, 8, generator=g, device=cuda))
    return x.to(dtype), torch.rand(B, generator=g, device=cuda)


def _want(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(tokens, log-probabilities) of the definition in 64 bits."""
    f = lambda v: [float(np.float32(v))] * len(x)  # noqa: E731
    return ssm_ref.sample(x, u.float().tolist(), f(temperature), [int(top_k)] * len(x), f(top_p), f(min_p))


def _near(lp, want, V):
    """fp32's rounding, and V weights each rounded to a unit of 2^-s, against a mass of at least 1."""
    s = min(52, 62 - math.ceil(math.log2(V)))
    return (np.abs(lp.double().cpu().numpy() - want) <=
            2.0 ** -24 * np.abs(want) + 1e-12 + V * 2.0 ** -(s + 1)).all()


@pytest.mark.parametrize("V", [2048, 4097, 16400, 50257])
@pytest.mark.parametrize("B", [1, 5, 130])
def test_rows_whose_ctas_start_apart(cuda, B, V):
    """A row's CTAs with nothing to load (the last ones of these vocabularies)
    reach each other's shared memory at once, while another stream's kernels
    hold their neighbours back."""
    x, u = _logits(B, V, V + B, cuda)
    s = dict(top_k=30, top_p=0.95, temperature=0.9)
    want, wlp = _want(x, u, **s)
    load = torch.randn(4096, 4096, device=cuda)
    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))
    for i in range(30):
        with torch.cuda.stream(side):
            for n in (64, 640, 4096):
                load[:n].sin_()
        tok, lp = wk.sample_tokens(x, u, **s)
        assert tok.tolist() == want.tolist() and _near(lp, wlp, V), i
    torch.cuda.synchronize()
