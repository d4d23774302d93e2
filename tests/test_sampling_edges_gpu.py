"""Token sampling at the edges of what its documentation allows: rows whose
CTAs start apart, two host threads, settings and numbers at their limits."""

import ctypes
import math
import threading

import numpy as np
import pytest
import torch

import ssm_ref
import wkvm_b200 as wk
from wkvm_b200 import _lib

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


def test_threads_with_vocabularies_of_their_own(cuda):
    """Host threads sample from vocabularies whose kernels need different
    amounts of shared memory: no call makes another thread's fail. The C entry
    is called without the interpreter's lock, as ctypes does."""
    entry, f, p = _lib.load().wkvm_sample_tokens, ctypes.c_float, ctypes.c_void_p
    sizes, wrong = (131072, 131072, 700, 700), []
    start = threading.Barrier(len(sizes))

    def serve(V):
        with torch.cuda.device(cuda), torch.cuda.stream(torch.cuda.Stream(cuda)):
            stream = torch.cuda.current_stream(cuda)
            x, u = _logits(1, V, V, cuda, BF)
            tok, lp = torch.empty(1, dtype=torch.int64, device=cuda), torch.empty(1, device=cuda)
            args = (p(x.data_ptr()), V, p(u.data_ptr()), None, None, None, None, f(1), 0, f(0.9), f(0),
                    p(tok.data_ptr()), p(lp.data_ptr()), 1, V, 1, None, p(stream.cuda_stream))
            start.wait()
            rc = [entry(*args) for _ in range(2000)]
            stream.synchronize()
            want, _ = _want(x, u, top_p=0.9)
            if any(rc) or tok.tolist() != want.tolist():
                wrong.append((V, sum(c != 0 for c in rc), tok.tolist(), want.tolist()))

    threads = [threading.Thread(target=serve, args=(V,)) for V in sizes]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("V", [900, 3000, 40000])
def test_temperature_without_limit_and_min_p(cuda, V):
    """At an infinite temperature every weight is 1, and so at least min_p."""
    x, u = _logits(6, V, V, cuda)
    x[:, V // 2:] = -INF
    inf = torch.full((6,), INF, device=cuda)
    for s in (dict(min_p=1.0), dict(min_p=0.5), dict(min_p=1.0, top_p=0.5), dict(min_p=1.0, top_k=V)):
        n = V // 2
        if "top_p" in s:  # the largest half of them
            tok, lp = wk.sample_tokens(x, u, temperature=inf, **s)
            kept = math.ceil(n / 2)
            rank = (x > x.gather(1, tok[:, None])).sum(1)
            assert bool((rank < kept).all())
        else:
            kept = n
            tok, lp = wk.sample_tokens(x, u, temperature=inf, **s)
            assert torch.equal(tok, (u.double() * n).long())
        assert bool(((lp + math.log(kept)).abs() < 1e-6).all())
    for t in (1e30, 1e18):  # weights round to 1
        for s in (dict(min_p=1.0), dict(min_p=0.5), dict()):
            tok, lp = wk.sample_tokens(x, u, temperature=t, **s)
            want, wlp = _want(x, u, temperature=t, **s)
            assert tok.tolist() == want.tolist() and _near(lp, wlp, V)


def test_weights_below_half_a_unit_are_never_drawn(cuda):
    """Weights are rounded to units of 2^-s: the smallest number draws the first id with one."""
    V = 5000  # s = 62 - 13 = 49
    x = torch.full((3, V), -200.0, device=cuda)  # e^-200: no unit
    x[:, 4000] = 0.0
    x[1, 3000] = -48 * math.log(2)               # two units
    x[2, 3000] = -51 * math.log(2)               # a quarter of one
    zero = torch.zeros(3, device=cuda)
    for s in (dict(), dict(top_k=100), dict(top_p=1 - 2.0 ** -24)):
        tok, lp = wk.sample_tokens(x, zero, **s)
        assert tok.tolist()[::2] == [4000, 4000] and bool((lp[::2] == 0).all())
        if "top_p" not in s:
            assert tok[1] == 3000 and abs(lp[1].item() + 48 * math.log(2)) < 1e-5


def test_largest_vocabulary(cuda):
    """2^20 logits: a border moves by V 2^-43 = 2^-23 of the largest weight at most."""
    V = wk.sampling.MAX_VOCAB
    assert V == 1 << 20
    x, u = _logits(3, V, 1, cuda, BF)
    for s in (dict(), dict(top_p=0.9), dict(top_k=100, top_p=0.9), dict(min_p=0.05)):
        tok, lp = wk.sample_tokens(x, u, **s)
        want, wlp = _want(x, u, **s)
        assert tok.tolist() == want.tolist() and _near(lp, wlp, V)


@pytest.mark.parametrize("s", [dict(), dict(top_k=9), dict(top_p=0.9), dict(min_p=0.01)], ids=str)
def test_numbers_outside_their_range(cuda, s):
    """Below 0 as 0, at or past 1 the last kept id with a mass, against the definition."""
    x, _ = _logits(6, 2000, 4, cuda)
    for u, like in ((-1.0, 0.0), (NAN, 0.0), (-INF, 0.0), (1.0, 1.0), (2.0, 1.0), (INF, 1.0)):
        tok, lp = wk.sample_tokens(x, torch.full((6,), u, device=cuda), **s)
        want, wlp = _want(x, torch.full((6,), like), **s)
        assert tok.tolist() == want.tolist() and _near(lp, wlp, 2000)
