"""Short convolution and selective scan at the edges of what their
documentation allows: every launch shape of the step, values that are not
numbers, offsets out of order, states that grow, the longest token axis."""

import pytest
import torch

import ssm_ref
import wkvm_b200 as wk
from wkvm_b200 import _lib, ops

pytestmark = pytest.mark.gpu

BF, FH, F32 = torch.bfloat16, torch.float16, torch.float32
NAMES = ("x", "dt", "A", "B", "C")


def _inputs(cuda, lead, D, N, G, dtype, seed=0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=cuda)  # noqa: E731
    return dict(x=r(*lead, D).to(dtype), dt=r(*lead, D).to(dtype), A=-torch.exp(r(D, N)), B=r(*lead, G, N).to(dtype),
                C=r(*lead, G, N).to(dtype), D=r(D), z=r(*lead, D).to(dtype), dt_bias=r(D) - 4)


def _call(fn, a, *state, **more):
    return fn(*[a[k] for k in NAMES], *state, D=a["D"], z=a["z"], dt_bias=a["dt_bias"], **more)


@pytest.mark.parametrize("T", [2 ** 26 + 7, 2 ** 31 - 1])
def test_scan_longest_token_axis(cuda, T):
    """One channel of as many tokens as an int32 counts, the inputs repeated by
    a stride of 0: the state settles where x delta / (1 - e^-delta) has it."""
    one = torch.ones(1, 1, 1, device=cuda, dtype=BF)
    row = torch.ones(1, 1, 8, device=cuda, dtype=BF).expand(1, T, 8)
    o, ht = wk.selective_scan(one.expand(1, T, 1), (0.5 * one).expand(1, T, 1), -torch.ones(1, 8, device=cuda), row, row,
                              dt_softplus=False, output_final_state=True)
    h = 0.5 / (1 - torch.tensor(-0.5, dtype=torch.float64).exp().item())
    # 1 / (1 - e^-1/2) < 3 roundings of 2^-22 settle; the output's own half step
    assert (ht.double() - h).abs().max().item() <= 3 * 2.0 ** -22 * h
    rest = o[0, 60:, 0]  # e^-30 of the empty start
    assert rest.min() == rest.max() and abs(rest[0].item() - 8 * h) <= (2.0 ** -8 + 2.0 ** -19) * 8 * h
    assert abs(o[0, 0, 0].item() - 4) <= 2.0 ** -8 * 4


SHAPES = [(2, 5, 40, 16, 2), (160, 2, 1000, 16, 2),  # steps, one and four channels a thread
          (2, 50, 40, 16, 2), (1, 60, 24, 128, 2),   # prompts
          (64, 20, 2048, 16, 2),                     # many of them
          (1, 2100, 40, 16, 2), (1, 1100, 8, 64, 2)]  # few long ones, split in time


@pytest.mark.parametrize("B,T,D,N,G", SHAPES)
@pytest.mark.parametrize("what", ["x", "dt", "A", "B", "C", "D", "z", "dt_bias", "state"])
def test_scan_keeps_nan(cuda, B, T, D, N, G, what):
    """A NaN in any input reaches what the formula makes of it, and nothing else."""
    a = _inputs(cuda, (B, T), D, N, G, F32, seed=T)
    h0 = torch.randn(B, D, N, device=cuda)
    o, ht = _call(wk.selective_scan, a, initial_state=h0, output_final_state=True)
    bad, g0, b, t, d, n = dict(a), h0.clone(), B - 1, T // 2, D // 2 + 1, N - 2
    g = d // (D // G)
    at = {"x": (b, t, d), "dt": (b, t, d), "z": (b, t, d), "A": (d, n), "B": (b, t, g, n), "C": (b, t, g, n), "D": (d,),
          "dt_bias": (d,), "state": (b, d, n)}[what]
    if what == "state":
        g0[at] = float("nan")
    else:
        bad[what] = a[what].clone()
        bad[what][at] = float("nan")
    o2, ht2 = _call(wk.selective_scan, bad, initial_state=g0, output_final_state=True)
    mo, mh = torch.zeros_like(o, dtype=torch.bool), torch.zeros_like(ht, dtype=torch.bool)
    lo, hi = g * (D // G), (g + 1) * (D // G)
    if what in ("x", "dt"):
        mo[b, t:, d] = mh[b, d] = True
    elif what == "A":
        mo[:, :, d] = mh[:, d, n] = True
    elif what == "B":
        mo[b, t:, lo:hi] = mh[b, lo:hi, n] = True
    elif what == "C":
        mo[b, t, lo:hi] = True
    elif what == "z":
        mo[b, t, d] = True
    elif what == "D":
        mo[:, :, d] = True
    elif what == "dt_bias":
        mo[:, :, d] = mh[:, d] = True
    else:
        mo[b, :, d] = mh[b, d, n] = True
    assert torch.equal(o2.isnan(), mo) and torch.equal(ht2.isnan(), mh)
    assert torch.equal(o2[~mo], o[~mo]) and torch.equal(ht2[~mh], ht[~mh])


@pytest.mark.parametrize("cu", [[0, 50, 10, 40], [0, 50, 60, -2, 1], [60, 100, 0, 40], [40, 100, 35, 38], [0, 33, 500, 70, 90],
                                [5, 5, 64, 3, 3, 5]])
@pytest.mark.parametrize("D", [40, 1032])
def test_conv_offsets_out_of_order(cuda, cu, D):
    """Sequences between offsets that descend or leave the axis are skipped;
    every other one is computed, wherever it stands."""
    T, W = 100, 4
    x, w = torch.randn(1, T, D, device=cuda).to(BF), torch.randn(D, W, device=cuda).to(BF)
    n = len(cu) - 1
    bank = torch.randn(1, n + 1, W - 1, D, device=cuda).to(BF)
    start, o = bank.clone(), torch.full_like(x, float("nan"))
    wk.short_conv_prefill_slots(x, w, bank, 0, list(range(1, n + 1)), activation="silu",
                                cu_seqlens=torch.tensor(cu, device=cuda), out=o)
    with pytest.raises(_lib.WkvmError, match="INVALID_ARG"):
        ops.check_device_status(cuda)
    ok = [i for i in range(n) if 0 <= cu[i] <= cu[i + 1] <= T]
    cover = torch.zeros(T, dtype=torch.int64)
    for i in ok:
        cover[cu[i]:cu[i + 1]] += 1
    assert torch.equal(o[0].isnan().all(1).cpu(), cover == 0) and torch.equal(o[0].isnan().any(1).cpu(), cover == 0)
    ref = start.clone()
    for i in ok:
        s = slice(cu[i], cu[i + 1])
        want = wk.short_conv_prefill_slots(x[:, s], w, ref, 0, [i + 1], activation="silu")
        one = (cover[s] == 1).to(cuda)  # tokens of two sequences may hold either's
        assert torch.equal(o[0, s][one], want[0][one])
    assert torch.equal(bank, ref)


@pytest.mark.parametrize("D,N", [(40, 16), (8, 64)])
def test_scan_states_that_grow_between_parts(cuda, D, N):
    """Without softplus steps may have any sign. Over a part of a long row a
    state may grow by more than fp32's range: from nothing it stays nothing,
    from a small value it is what the tokens one by one give."""
    T = 2304
    a = _inputs(cuda, (1, T), D, N, 1, F32, seed=N)
    a["A"] = torch.ones(D, N, device=cuda)
    a["dt_bias"] = None
    sign = torch.where(torch.arange(T, device=cuda) // 144 % 2 == 0, 1.0, -1.0)
    a["dt"] = (0.68 * sign)[None, :, None].expand(1, T, D).contiguous()  # e^98 up, e^98 down
    a["x"] = torch.zeros_like(a["x"])
    h0 = torch.zeros(1, D, N, device=cuda)
    h0[:, ::2] = 1e-20 * (1 + torch.rand(1, (D + 1) // 2, N, device=cuda))
    o, ht = _call(wk.selective_scan, a, dt_softplus=False, initial_state=h0, output_final_state=True)
    ro, tol, rh, htol = ssm_ref.scan(*[a[k] for k in NAMES], a["D"], a["z"], None, False, h0)
    assert bool(o.isfinite().all()) and not o[..., 1::2].any() and not ht[:, 1::2].any()
    # a part's decay is the exponential of a sum of 144 steps, each rounded once:
    # 144 x 2^-24 of a sum of 98 at most, that is 2^-10.2, sixteen parts
    ssm_ref.check(o, ro, tol + 2.0 ** -6 * ro.abs(), "o")
    ssm_ref.check(ht, rh, htol + 2.0 ** -6 * rh.abs(), "state")


# rows enough for four channels a thread (B D N >= 16 x 148 x 1024), with a
# last block of channels that is not full and groups that end inside a block
@pytest.mark.parametrize("dtype,B,D,N,G", [(BF, 160, 1002, 16, 3), (F32, 310, 1001, 8, 1), (FH, 304, 1002, 8, 6),
                                           (BF, 80, 1001, 32, 7), (F32, 40, 990, 64, 10), (FH, 20, 1002, 128, 2),
                                           (F32, 160, 1002, 16, 1)])
@pytest.mark.parametrize("T", [1, 3, 8])
def test_scan_steps_of_many_rows(cuda, dtype, B, D, N, G, T):
    assert B * D * N >= 16 * 148 * 1024
    a = _inputs(cuda, (B, T), D, N, G, dtype, seed=N + T)
    bank = torch.randn(1, B + 3, D, N, device=cuda)
    before = bank.clone()
    ids = (1 + torch.randperm(B + 2, generator=torch.Generator().manual_seed(T))[:B]).tolist()
    o = _call(wk.selective_scan_decode_slots, a, bank, 0, ids)
    ro, tol, rh, htol = ssm_ref.scan(*[a[k] for k in NAMES], a["D"], a["z"], a["dt_bias"], True, before[0, ids])
    ssm_ref.check(o, ro, tol, "o")
    ssm_ref.check(bank[0, ids], rh, htol, "state")
    rest = [i for i in range(B + 3) if i not in ids]
    assert torch.equal(bank[0, rest], before[0, rest])
    ops.check_device_status(cuda)


@pytest.mark.parametrize("dtype,B,T,D,N,G", [(BF, 16, 19, 2050, 16, 2), (F32, 33, 9, 2001, 8, 3), (FH, 9, 33, 2004, 32, 4),
                                             (F32, 9, 17, 1000, 64, 1), (BF, 5, 40, 1030, 128, 2), (F32, 17, 16, 2048, 16, 1)])
def test_scan_prompts_of_many_rows(cuda, dtype, B, T, D, N, G):
    """The wide launch shape (B D N >= 2048 x 256) against 64 bits."""
    assert B * D * N >= 2048 * 256 and D % G == 0
    a = _inputs(cuda, (B, T), D, N, G, dtype, seed=B)
    h0 = torch.randn(B, D, N, device=cuda)
    o, ht = _call(wk.selective_scan, a, initial_state=h0, output_final_state=True)
    ro, tol, rh, htol = ssm_ref.scan(*[a[k] for k in NAMES], a["D"], a["z"], a["dt_bias"], True, h0)
    ssm_ref.check(o, ro, tol, "o")
    ssm_ref.check(ht, rh, htol, "state")


@pytest.mark.parametrize("D,N", [(40, 16), (8, 64), (12, 128)])
def test_scan_parts_join_without_loss(cuda, D, N):
    """Steps of 1/4 add up exactly and slow decays carry states over every part
    of a long row: the bounds of the tokens one by one hold as they are."""
    T = 2100
    a = _inputs(cuda, (1, T), D, N, 1, F32, seed=N)
    a["dt"], a["dt_bias"] = torch.full_like(a["dt"], 0.25), None
    a["A"] = -torch.exp(-7 * torch.rand(D, N, device=cuda))  # e-folds from 4 to 4,400 tokens
    a["x"] = a["x"] * (torch.rand(1, T, 1, device=cuda) < 0.02)
    h0 = 10 * torch.randn(1, D, N, device=cuda)
    o, ht = _call(wk.selective_scan, a, dt_softplus=False, initial_state=h0, output_final_state=True)
    ro, tol, rh, htol = ssm_ref.scan(*[a[k] for k in NAMES], a["D"], a["z"], None, False, h0)
    ssm_ref.check(o, ro, tol, "o")
    ssm_ref.check(ht, rh, htol, "state")


@pytest.mark.parametrize("B,D,N", [(6, 96, 16), (300, 1024, 16)])
def test_padded_batches(cuda, B, D, N):
    """Rows padded with slot 0, as a graphed step pads them, share that row and change no other."""
    a = _inputs(cuda, (B, 1), D, N, 1, BF)
    w = torch.randn(D, 4, device=cuda).to(BF)
    n = B // 2 + 1
    ids = torch.zeros(B, dtype=torch.int32, device=cuda)
    ids[:n] = 1 + torch.randperm(n, device=cuda)
    conv, ssm = torch.randn(1, n + 2, 3, D, device=cuda).to(BF), torch.randn(1, n + 2, D, N, device=cuda)
    conv2, ssm2 = conv.clone(), ssm.clone()
    y = wk.short_conv_decode_slots(a["x"], w, conv, 0, ids)
    o = _call(wk.selective_scan_decode_slots, a, ssm, 0, ids)
    real = {k: v[:n] if k in ("x", "dt", "B", "C", "z") else v for k, v in a.items()}
    y2 = wk.short_conv_decode_slots(real["x"], w, conv2, 0, ids[:n])
    o2 = _call(wk.selective_scan_decode_slots, real, ssm2, 0, ids[:n])
    assert torch.equal(y[:n], y2) and torch.equal(o[:n], o2)
    assert torch.equal(conv[:, 1:], conv2[:, 1:]) and torch.equal(ssm[:, 1:], ssm2[:, 1:])
    ops.check_device_status(cuda)


def test_captured_prompts(cuda):
    """Packed prompts captured once and replayed over other inputs, lengths and
    slots: tiles, and long rows split in time."""
    D, N, total = 64, 16, 3000
    w = torch.randn(D, 4, device=cuda).to(BF)
    s = _inputs(cuda, (1, total), D, N, 1, BF)
    cu, ids = torch.tensor([0, 1400, 3000], device=cuda), torch.tensor([1, 2], dtype=torch.int32, device=cuda)
    conv, ssm = torch.zeros(1, 4, 3, D, device=cuda, dtype=BF), torch.zeros(1, 4, D, N, device=cuda)

    def call(v, c, h):
        y = wk.short_conv_prefill_slots(v["x"], w, c, 0, ids, activation="silu", cu_seqlens=cu)
        return _call(wk.selective_scan_prefill_slots, dict(v, x=y), h, 0, ids, cu_seqlens=cu)

    call(s, conv, ssm)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = call(s, conv, ssm)
    for seed, (offsets, slots) in enumerate([([0, 1400, 3000], [1, 2]), ([0, 3, 3000], [3, 1]), ([0, 2990, 2990], [2, 3])]):
        fresh = _inputs(cuda, (1, total), D, N, 1, BF, seed=10 + seed)
        for k in s:
            s[k].copy_(fresh[k])
        cu.copy_(torch.tensor(offsets, device=cuda))
        ids.copy_(torch.tensor(slots, dtype=torch.int32, device=cuda))
        conv.normal_()
        ssm.normal_()
        conv2, ssm2 = conv.clone(), ssm.clone()
        graph.replay()
        end = offsets[-1]
        assert torch.equal(o[:, :end], call(fresh, conv2, ssm2)[:, :end])
        assert torch.equal(conv, conv2) and torch.equal(ssm, ssm2)
    ops.check_device_status(cuda)


def test_conv_keeps_nan(cuda):
    """A NaN reaches the W outputs whose window holds it and the state, in its channel alone."""
    for T, D, W in ((5, 40, 4), (70, 40, 3), (70, 7, 4)):
        x, w = torch.randn(2, T, D, device=cuda).to(BF), torch.randn(D, W, device=cuda).to(BF)
        s0 = torch.randn(2, W - 1, D, device=cuda).to(BF)
        o, st = wk.short_conv(x, w, activation="silu", initial_state=s0, output_final_state=True)
        x[1, T - 2, 3] = s0[0, 0, 5] = float("nan")
        o2, st2 = wk.short_conv(x, w, activation="silu", initial_state=s0, output_final_state=True)
        mo, ms = torch.zeros_like(o, dtype=torch.bool), torch.zeros_like(st, dtype=torch.bool)
        mo[1, T - 2:, 3] = mo[0, 0, 5] = ms[1, W - 3, 3] = True
        assert torch.equal(o2.isnan(), mo) and torch.equal(st2.isnan(), ms)
        assert torch.equal(o2[~mo], o[~mo]) and torch.equal(st2[~ms], st[~ms])


@pytest.mark.parametrize("n,T", [(256, 16), (200, 3), (64, 9)])
def test_many_short_prompts_cost_what_their_tokens_do(cuda, n, T):
    """Packed prompts of a few tokens each take about as long as the same
    tokens in a batch: what a CTA does per sequence ahead of them is small."""
    D, N = 2048, 16
    a = _inputs(cuda, (1, n * T), D, N, 1, BF)
    cu = torch.arange(0, n * T + 1, T, device=cuda)
    h0 = torch.randn(n, D, N, device=cuda)
    batch = {k: v.view(n, T, *v.shape[2:]) if k in ("x", "dt", "B", "C", "z") else v for k, v in a.items()}
    calls = [lambda: _call(wk.selective_scan, a, initial_state=h0, output_final_state=True, cu_seqlens=cu),
             lambda: _call(wk.selective_scan, batch, initial_state=h0, output_final_state=True)]
    (o, ht), (o2, ht2) = (f() for f in calls)
    times = []
    for f in calls:
        best = []
        for _ in range(5):
            b, e = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            b.record()
            for _ in range(10):
                f()
            e.record()
            e.synchronize()
            best.append(b.elapsed_time(e))
        times.append(min(best))
    ro, tol, rh, htol = ssm_ref.scan(*[a[k][..., :64] if k in ("x", "dt") else a[k][:64] if k == "A" else a[k] for k in NAMES],
                                     a["D"][:64], a["z"][..., :64], a["dt_bias"][:64], True, h0[:, :64], cu.tolist())
    ssm_ref.check(o[..., :64], ro, tol, "o")
    ssm_ref.check(ht[:, :64], rh, htol, "state")
    assert times[0] < 5 * times[1], times
