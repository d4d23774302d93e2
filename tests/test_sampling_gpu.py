"""Token sampling on the GPU against the definition in 64 bits: tokens equal,
log-probabilities to fp32's rounding."""

import math

import numpy as np
import pytest
import torch

import ssm_ref
import wkvm_b200 as wk

pytestmark = pytest.mark.gpu

BF, FH, F32 = torch.bfloat16, torch.float16, torch.float32
INF, NAN = math.inf, math.nan


def _check(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    B = logits.shape[0]
    tok, lp = wk.sample_tokens(logits, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    # settings as fp32, as the operator takes them
    rows = [(v.float().tolist() if isinstance(v, torch.Tensor) else [float(np.float32(v))] * B)
            for v in (temperature, top_k, top_p, min_p)]
    want, wlp = ssm_ref.sample(logits, u.float().tolist(), rows[0], [int(k) for k in rows[1]], rows[2], rows[3])
    assert tok.dtype == torch.int64 and lp.dtype == torch.float32 and tok.shape == lp.shape == (B,)
    assert tok.tolist() == want.tolist()
    fin = np.isfinite(wlp)
    got = lp.double().cpu().numpy()
    assert (got[~fin] == wlp[~fin]).all()
    # rounding to fp32; weights to 2e-13; and the mass, a sum of V weights each rounded to a unit of 2^-s
    # with s = min(52, 62 - ceil(log2 V)): off by V 2^-(s+1) at most, against a mass of at least 1
    V = logits.shape[1]
    s = min(52, 62 - math.ceil(math.log2(V)))
    assert (np.abs(got[fin] - wlp[fin]) <= 2.0 ** -24 * np.abs(wlp[fin]) + 1e-12 + V * 2.0 ** -(s + 1)).all()
    return tok, lp


def _logits(B, V, seed, cuda, dtype=F32, scale=2.5, peaks=8):
    g = torch.Generator(device=cuda).manual_seed(seed)
    x = scale * torch.randn(B, V, generator=g, device=cuda)
    if peaks:
        x.scatter_add_(1, torch.randint(0, V, (B, peaks), generator=g, device=cuda),
                       4 + 6 * torch.rand(B, peaks, generator=g, device=cuda))
    return x.to(dtype), torch.rand(B, generator=g, device=cuda)


SETTINGS = [dict(), dict(temperature=0.0), dict(temperature=0.7), dict(top_k=1), dict(top_k=40), dict(top_p=0.9),
            dict(top_p=0.3, temperature=1.7), dict(min_p=0.05), dict(top_k=50, top_p=0.95, min_p=0.01, temperature=0.8),
            dict(top_k=10 ** 6, top_p=0.999), dict(top_k=700, top_p=0.99, temperature=2.5), dict(top_p=0.0),
            dict(min_p=1.0), dict(temperature=1e-6), dict(temperature=1e6, top_p=0.5), dict(top_k=3000)]


@pytest.mark.parametrize("setting", SETTINGS, ids=str)
@pytest.mark.parametrize("dtype,V", [(BF, 65536), (F32, 65536), (FH, 50000), (F32, 1001), (BF, 31)])
def test_against_definition(cuda, setting, dtype, V):
    x, u = _logits(6, V, V + len(setting), cuda, dtype)
    _check(x, u, **setting)


@pytest.mark.parametrize("V", [1, 2, 3, 32, 33, 127, 1024, 1025, 4097, 16383, 16385, 40000, 131071, 200001, 262144, 300008, 400001])
def test_vocabulary_sizes(cuda, V):
    x, u = _logits(3, V, V, cuda, BF)
    for s in (dict(), dict(top_p=0.9), dict(top_k=20, top_p=0.8), dict(temperature=0)):
        _check(x, u, **s)


@pytest.mark.parametrize("B", [1, 2, 7, 37, 300])
def test_batches_with_settings_per_row(cuda, B):
    x, u = _logits(B, 5003, B, cuda, F32)
    g = torch.Generator(device=cuda).manual_seed(B)
    r = lambda: torch.rand(B, generator=g, device=cuda)  # noqa: E731
    temp = torch.where(r() < 0.2, 0.0, 0.3 + r())
    k = torch.where(r() < 0.4, 0.0, 1 + 200 * r()).to(torch.int32)
    p = torch.where(r() < 0.4, 1.0, r())
    _check(x, u, temp, k, p, torch.where(r() < 0.5, 0.0, 0.2 * r()))


def test_ties(cuda):
    """Equal logits go to the lowest ids, at the k-th place, at the edge of the nucleus and in the draw."""
    V = 3000
    x = torch.zeros(9, V, device=cuda)
    u = torch.tensor([0.0, 0.1, 0.25, 0.5, 0.5 + 2 ** -20, 0.75, 0.9, 1 - 2 ** -24, 0.999], device=cuda)
    for s in (dict(), dict(top_k=7), dict(top_p=0.5), dict(top_p=0.25, top_k=64), dict(min_p=1.0), dict(temperature=0),
              dict(top_k=2999), dict(top_p=0.001)):
        _check(x, u, **s)
    x[:, 1500:] = 1.0
    x[:, 2000] = 2.0
    for s in (dict(), dict(top_k=7), dict(top_k=1600), dict(top_p=0.5), dict(top_p=0.9), dict(top_k=1501)):
        _check(x, u, **s)
    few = torch.randint(0, 4, (9, V), device=cuda).float()  # four values, 750 ids each
    for s in (dict(), dict(top_k=100), dict(top_k=800, top_p=0.7), dict(top_p=0.95), dict(top_p=0.2)):
        _check(few, u, **s)


def test_masked_and_special_values(cuda):
    V = 2500
    x, u = _logits(8, V, 5, cuda, F32)
    x[0] = -INF                                  # nothing to choose
    x[1, :] = -INF
    x[1, 1234] = -3.0                            # one choice
    x[2, ::2] = -INF
    x[3, :] = torch.finfo(F32).min               # masks of the type's lowest value
    x[3, [7, 900]] = torch.tensor([1.0, 2.0], device=cuda)
    x[4, 17] = NAN                               # never chosen
    x[5, [3, 2000]] = INF                        # share the mass
    x[6] = NAN
    x[7, 100:] = torch.finfo(F32).min
    for s in (dict(), dict(top_k=5), dict(top_p=0.9), dict(top_k=1000, top_p=0.99), dict(temperature=0),
              dict(min_p=0.1), dict(temperature=0.01)):
        tok, _ = _check(x, u, **s)
        assert tok[0] == -1 and tok[6] == -1 and tok[1] == 1234
    y = torch.full((3, V), torch.finfo(F32).min, device=cuda)  # every logit the lowest value
    for s in (dict(), dict(top_k=5), dict(top_p=0.5)):
        _check(y, u[:3], **s)
    h = torch.full((3, V), -INF, device=cuda, dtype=FH)
    h[1] = torch.finfo(FH).min
    h[2, 5], h[2, 9] = 3, torch.finfo(FH).max
    for s in (dict(), dict(top_k=2), dict(top_p=0.5)):
        _check(h, u[:3], **s)
    z = torch.zeros(2, V, device=cuda)
    z[:, 1::2] = -0.0                            # zeros of both signs are equal
    _check(z, u[:2], top_k=3)


def test_odd_settings(cuda):
    """Numbers outside [0, 1), settings that are NaN, negative or beyond the
    vocabulary: each row still gets a token, as the settings' nearest meaning
    has it."""
    V = 2000
    x, _ = _logits(6, V, 4, cuda, F32)
    first, last = torch.full((6,), 0.0, device=cuda), torch.full((6,), 1 - 2.0 ** -24, device=cuda)
    for s in (dict(), dict(top_k=9), dict(top_p=0.9), dict(min_p=0.01)):
        a = wk.sample_tokens(x, first, **s)
        for u in (-1.0, NAN, -INF):
            b = wk.sample_tokens(x, torch.full((6,), u, device=cuda), **s)
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        # at or past 1: the last kept id, which is never below the last number's
        for u in (1.0, 2.0, INF):
            b = wk.sample_tokens(x, torch.full((6,), u, device=cuda), **s)
            assert bool((b[0] >= wk.sample_tokens(x, last, **s)[0]).all()) and bool((b[0] < V).all())
            assert bool(b[1].isfinite().all())
    u = torch.rand(6, device=cuda)
    t = lambda v: torch.full((6,), v, device=cuda)  # noqa: E731
    plain = wk.sample_tokens(x, u)
    for s in (dict(top_p=t(NAN)), dict(min_p=t(NAN)), dict(min_p=t(-1.0)), dict(top_p=t(7.0)),
              dict(top_k=torch.full((6,), -5, device=cuda)), dict(top_k=torch.full((6,), 10 ** 12, device=cuda))):
        assert torch.equal(wk.sample_tokens(x, u, **s)[0], plain[0])
    best = x.argmax(1)
    for s in (dict(temperature=t(NAN)), dict(temperature=t(-1.0)), dict(top_p=t(-1.0)), dict(min_p=t(2.0)),
              dict(top_k=1, top_p=0.5)):
        assert torch.equal(wk.sample_tokens(x, u, **s)[0], best)
    # a temperature without limit: every finite logit alike
    x[:, 1000:] = -INF
    tok, lp = wk.sample_tokens(x, u, temperature=t(INF))
    assert torch.equal(tok, (u.double() * 1000).long()) and bool(((lp + math.log(1000)).abs() < 1e-6).all())


def test_wide_ranges(cuda):
    """Logits over many orders of magnitude, near-equal neighbours, outliers on both sides."""
    V = 20000
    g = torch.Generator(device=cuda).manual_seed(11)
    sign = torch.where(torch.rand(4, V, generator=g, device=cuda) < 0.5, -1.0, 1.0)
    x = sign * torch.exp(20 * torch.rand(4, V, generator=g, device=cuda) - 12)
    near = 1.0 + torch.arange(V, device=cuda) * 2.0 ** -23  # one step of fp32 apart
    x[1] = near[torch.randperm(V, generator=g, device=cuda)]
    x[2] = near.flip(0)
    x[2, 5], x[2, 6] = 30.0, -1e30
    u = torch.rand(4, generator=g, device=cuda)
    for s in (dict(), dict(top_k=300), dict(top_p=0.5), dict(top_k=9000, top_p=0.9), dict(top_p=0.97, temperature=50.0),
              dict(temperature=1e-7, top_p=0.9)):
        _check(x, u, **s)


def test_strided_rows_and_types(cuda):
    x, u = _logits(4, 3001, 2, cuda, BF)
    wide = torch.randn(4, 3, 4000, device=cuda).to(BF)
    wide[:, 1, 5:3006] = x
    view = wide[:, 1, 5:3006]
    a = wk.sample_tokens(x, u, top_p=0.9)
    for v in (view, x.t().contiguous().t()):
        b = wk.sample_tokens(v, u.double(), top_p=torch.full((4,), 0.9, device=cuda, dtype=torch.float64))
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # widening the logits changes nothing
    c = wk.sample_tokens(x.float(), u, top_p=0.9)
    assert torch.equal(a[0], c[0]) and torch.equal(a[1], c[1])
    e = wk.sample_tokens(x[:0], u[:0])
    assert e[0].shape == e[1].shape == (0,)


def test_row_offsets_past_32_bits(cuda):
    V, B = 131072, 16500  # 2.2e9 elements
    x = torch.zeros(B, V, dtype=BF, device=cuda)
    x[-1, 77777] = 50.0
    tok, lp = wk.sample_tokens(x, torch.full((B,), 0.5, device=cuda), top_k=1)
    assert tok[-1].item() == 77777 and tok[0].item() == 0 and not lp.any()


def test_frequencies(cuda):
    """Uniform numbers in even steps give every token its share of them."""
    n = 4096
    x = torch.randn(1, 50, device=cuda).expand(n, 50)
    u = (torch.arange(n, device=cuda) + 0.5) / n
    tok, _ = wk.sample_tokens(x, u)
    share = torch.bincount(tok, minlength=50).double().cpu() / n
    assert (share - torch.softmax(x[0].double().cpu(), 0)).abs().max() <= 1.0 / n


def test_graph_replay_and_streams(cuda):
    x, u = _logits(5, 9000, 1, cuda, F32)
    temp, p = torch.full((5,), 0.9, device=cuda), torch.full((5,), 0.8, device=cuda)
    sx, su = torch.zeros_like(x), torch.zeros_like(u)
    wk.sample_tokens(sx, su)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = wk.sample_tokens(sx, su, temperature=temp, top_p=p)
    for seed in range(4):
        x, u = _logits(5, 9000, seed, cuda, F32)
        sx.copy_(x)
        su.copy_(u)
        temp.fill_(0.5 + 0.2 * seed)
        graph.replay()
        side = torch.cuda.Stream(cuda)
        side.wait_stream(torch.cuda.current_stream(cuda))
        with torch.cuda.stream(side):
            ref = wk.sample_tokens(x, u, temperature=temp, top_p=p)
        side.synchronize()
        assert torch.equal(out[0], ref[0]) and torch.equal(out[1], ref[1])
