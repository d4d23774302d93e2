"""Short convolution and selective scan on the GPU against 64-bit references,
over dtypes, widths, head layouts, lengths, strides and packings."""

import pytest
import torch

import ssm_ref
import wkvm_b200 as wk
from wkvm_b200 import _lib, ops

pytestmark = pytest.mark.gpu

BF, FH, F32 = torch.bfloat16, torch.float16, torch.float32


def _cu(lengths, cuda):
    return torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], dtype=torch.int64, device=cuda)


def _ids(n, slots, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (1 + torch.randperm(slots, generator=g)[:n]).tolist()


# ---------------------------------------------------------------- convolution

@pytest.mark.parametrize("dtype", [BF, FH, F32])
@pytest.mark.parametrize("B,T,D,W", [(1, 1, 64, 4), (3, 1, 200, 2), (2, 2, 33, 4), (3, 3, 8, 3), (5, 16, 136, 4),
                                     (2, 17, 24, 4), (2, 47, 1, 3), (1, 129, 72, 2), (3, 33, 1032, 4)])
@pytest.mark.parametrize("act", [None, "silu"])
def test_conv_slots(cuda, dtype, B, T, D, W, act):
    torch.manual_seed(B * T + D)
    x = torch.randn(B, T, D, device=cuda).to(dtype)
    w = torch.randn(D, W, device=cuda).to(dtype)
    bias = torch.randn(D, device=cuda).to(dtype) if act else None
    bank = torch.randn(2, 8, W - 1, D, device=cuda).to(dtype)
    before, ids = bank.clone(), _ids(B, 7)
    fn = wk.short_conv_decode_slots if T <= 3 else wk.short_conv_prefill_slots
    o = fn(x, w, bank, 1, ids, bias=bias, activation=act)
    ro, tol, new = ssm_ref.conv(x, w, bias, act, before[1, ids])
    ssm_ref.check(o, ro, tol, "o")
    assert torch.equal(bank[1, ids].double().cpu(), new)
    rest = [i for i in range(8) if i not in ids]
    assert torch.equal(bank[1, rest], before[1, rest]) and torch.equal(bank[0], before[0])
    ops.check_device_status(cuda)


@pytest.mark.parametrize("dtype,D", [(BF, 256), (F32, 37), (FH, 1028)])
@pytest.mark.parametrize("W", [2, 4])
@pytest.mark.parametrize("lengths", [[5], [0, 1, 2, 3, 0, 40, 1, 16, 15, 17, 0], [31, 1, 0, 0, 96],
                                     [1] * 70, [0, 0, 0], [200, 3]])
def test_conv_packed(cuda, dtype, D, W, lengths):
    torch.manual_seed(len(lengths) + D)
    x = torch.randn(1, sum(lengths), D, device=cuda).to(dtype)
    w = torch.randn(D, W, device=cuda).to(dtype)
    cu, n = _cu(lengths, cuda), len(lengths)
    s0 = torch.randn(n, W - 1, D, device=cuda).to(dtype)
    ro, tol, new = ssm_ref.conv(x, w, None, "silu", s0, cu.tolist())
    o, st = wk.short_conv(x, w, activation="silu", initial_state=s0, output_final_state=True, cu_seqlens=cu)
    ssm_ref.check(o, ro, tol, "o")
    assert torch.equal(st.double().cpu(), new)
    bank = torch.zeros(1, n + 1, W - 1, D, device=cuda, dtype=dtype)
    ids = _ids(n, n)
    bank[0, ids] = s0
    o2 = wk.short_conv_prefill_slots(x, w, bank, 0, ids, activation="silu", cu_seqlens=cu)
    assert torch.equal(o2, o) and torch.equal(bank[0, ids], st)
    # without a state: as after zeros, and none returned unless asked for
    o3, none = wk.short_conv(x, w, activation="silu", cu_seqlens=cu)
    ro3, tol3, _ = ssm_ref.conv(x, w, None, "silu", torch.zeros_like(s0), cu.tolist())
    ssm_ref.check(o3, ro3, tol3, "o without a state")
    assert none is None
    ops.check_device_status(cuda)


@pytest.mark.parametrize("off,D", [(0, 64), (3, 64), (8, 40), (1, 7)])
def test_conv_strided_views(cuda, off, D):
    """Halves and odd slices of a wider projection, read where they are."""
    big = torch.randn(2, 21, 3 * D + 9, device=cuda).to(BF)
    x = big[..., off:off + D]
    w, bank = torch.randn(D, 4, device=cuda).to(BF), torch.randn(1, 4, 3, D, device=cuda).to(BF)
    ro, tol, new = ssm_ref.conv(x, w, None, None, bank[0, [2, 1]])
    o = wk.short_conv_prefill_slots(x, w.unsqueeze(1), bank, 0, [2, 1])
    ssm_ref.check(o, ro, tol, "o")
    assert torch.equal(bank[0, [2, 1]].double().cpu(), new)
    # tokens and channels swapped in memory: a copy is made
    xt = x.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(wk.short_conv(xt, w)[0], wk.short_conv(x.contiguous(), w)[0])


def test_conv_split_prompt_and_steps_agree(cuda):
    """A prompt at once, in pieces, and token by token: the same bits."""
    D, T = 96, 75
    x, w = torch.randn(2, T, D, device=cuda).to(BF), torch.randn(D, 4, device=cuda).to(BF)
    banks = [torch.zeros(1, 3, 3, D, device=cuda, dtype=BF) for _ in range(3)]
    whole = wk.short_conv_prefill_slots(x, w, banks[0], 0, [1, 2], activation="silu")
    cuts = [0, 1, 3, 40, 58, T]
    parts = [wk.short_conv_prefill_slots(x[:, a:b], w, banks[1], 0, [1, 2], activation="silu")
             for a, b in zip(cuts, cuts[1:])]
    steps = [wk.short_conv_decode_slots(x[:, t:t + 1], w, banks[2], 0, [1, 2], activation="silu") for t in range(T)]
    assert torch.equal(torch.cat(parts, 1), whole) and torch.equal(torch.cat(steps, 1), whole)
    assert torch.equal(banks[1], banks[0]) and torch.equal(banks[2], banks[0])


# ----------------------------------------------------------------------- scan

def _scan_inputs(cuda, lead, D, N, G, dtype, gated=True, skip=True, bias=True, seed=0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=cuda)  # noqa: E731
    return dict(x=r(*lead, D).to(dtype), dt=(r(*lead, D) - (0 if bias else 3)).to(dtype),
                A=-torch.exp(r(D, N)), B=r(*lead, G, N).to(dtype), C=r(*lead, G, N).to(dtype),
                D=r(D) if skip else None, z=r(*lead, D).to(dtype) if gated else None,
                dt_bias=r(D) - 4 if bias else None)


def _ref(a, h0, cu=None, softplus=True):
    return ssm_ref.scan(a["x"], a["dt"], a["A"], a["B"], a["C"], a["D"], a["z"], a["dt_bias"], softplus, h0,
                        None if cu is None else cu.tolist())


@pytest.mark.parametrize("dtype", [BF, FH, F32])
@pytest.mark.parametrize("B,T,D,N,G", [(1, 1, 64, 16, 1), (3, 1, 100, 16, 2), (5, 2, 33, 8, 1), (2, 5, 6, 64, 3),
                                       (1, 3, 40, 128, 4), (2, 1, 1, 32, 1), (2, 65, 48, 16, 1), (1, 257, 130, 16, 2),
                                       (3, 40, 17, 32, 1), (1, 100, 36, 8, 4), (2, 31, 9, 128, 1), (1, 70, 129, 64, 1)])
def test_scan_slots(cuda, dtype, B, T, D, N, G):
    a = _scan_inputs(cuda, (B, T), D, N, G, dtype, seed=D + T)
    bank = torch.randn(2, 9, D, N, device=cuda)
    before, ids = bank.clone(), _ids(B, 8)
    fn = wk.selective_scan_decode_slots if T <= 5 else wk.selective_scan_prefill_slots
    o = fn(a["x"], a["dt"], a["A"], a["B"], a["C"], bank, 1, ids, D=a["D"], z=a["z"], dt_bias=a["dt_bias"])
    ro, tol, rh, htol = _ref(a, before[1, ids])
    ssm_ref.check(o, ro, tol, "o")
    ssm_ref.check(bank[1, ids], rh, htol, "state")
    rest = [i for i in range(9) if i not in ids]
    assert torch.equal(bank[1, rest], before[1, rest]) and torch.equal(bank[0], before[0])
    ops.check_device_status(cuda)


@pytest.mark.parametrize("gated,skip,bias,softplus", [(False, False, False, True), (True, False, True, True),
                                                      (False, True, False, False), (True, True, True, False)])
@pytest.mark.parametrize("T", [1, 50])
def test_scan_optional_inputs(cuda, gated, skip, bias, softplus, T):
    a = _scan_inputs(cuda, (2, T), 70, 16, 1, BF, gated, skip, bias, seed=T)
    if not softplus:  # steps as they are: small and positive, some zero
        a["dt"] = (0.1 * a["dt"].float().abs() * (a["x"] > -1)).to(BF)
        a["dt_bias"] = None if a["dt_bias"] is None else torch.zeros(70, device=cuda)
    o, ht = wk.selective_scan(a["x"], a["dt"], a["A"], a["B"][:, :, 0], a["C"][:, :, 0], D=a["D"], z=a["z"],
                              dt_bias=a["dt_bias"], dt_softplus=softplus, output_final_state=True)
    ro, tol, rh, htol = _ref(a, torch.zeros(2, 70, 16), softplus=softplus)
    ssm_ref.check(o, ro, tol, "o")
    ssm_ref.check(ht, rh, htol, "state")


@pytest.mark.parametrize("dtype,D,N,G", [(BF, 192, 16, 1), (F32, 35, 16, 5), (FH, 66, 64, 1), (BF, 10, 8, 2)])
@pytest.mark.parametrize("lengths", [[7], [0, 1, 2, 33, 0, 64, 65, 31, 0], [130, 1, 0, 20], [1] * 40, [0, 0]])
def test_scan_packed(cuda, dtype, D, N, G, lengths):
    a = _scan_inputs(cuda, (1, sum(lengths)), D, N, G, dtype, seed=len(lengths))
    cu, n = _cu(lengths, cuda), len(lengths)
    h0 = torch.randn(n, D, N, device=cuda)
    args = [a[k] for k in ("x", "dt", "A", "B", "C")]
    more = {k: a[k] for k in ("D", "z", "dt_bias")}
    ro, tol, rh, htol = _ref(a, h0, cu)
    o, ht = wk.selective_scan(*args, **more, initial_state=h0, output_final_state=True, cu_seqlens=cu)
    ssm_ref.check(o, ro, tol, "o")
    ssm_ref.check(ht, rh, htol, "state")
    bank, ids = torch.zeros(1, n + 1, D, N, device=cuda), _ids(n, n)
    bank[0, ids] = h0
    o2 = wk.selective_scan_prefill_slots(*args, bank, 0, ids, **more, cu_seqlens=cu)
    assert torch.equal(o2, o) and torch.equal(bank[0, ids], ht)
    o3, none = wk.selective_scan(*args, **more, cu_seqlens=cu)
    ro3, tol3, _, _ = _ref(a, torch.zeros_like(h0), cu)
    ssm_ref.check(o3, ro3, tol3, "o without a state")
    assert none is None
    ops.check_device_status(cuda)


@pytest.mark.parametrize("T", [1, 90])
@pytest.mark.parametrize("rank", [0, 1, 6, 8])
def test_scan_strided_views(cuda, T, rank):
    """x and z as halves of one projection, B and C as slices of another at
    offsets that are no multiple of any vector."""
    D, N, G = 80, 16, 2
    a = _scan_inputs(cuda, (2, T), D, N, G, BF, seed=rank)
    xz = torch.cat([a["x"], a["z"]], -1)
    proj = torch.cat([a["dt"][..., :rank], a["B"].flatten(2), a["C"].flatten(2)], -1)
    x, z = xz[..., :D], xz[..., D:]
    Bv = proj[..., rank:rank + G * N].unflatten(-1, (G, N))
    Cv = proj[..., rank + G * N:].unflatten(-1, (G, N))
    o, ht = wk.selective_scan(x, a["dt"], a["A"], Bv, Cv, z=z, D=a["D"], dt_bias=a["dt_bias"], output_final_state=True)
    o2, ht2 = wk.selective_scan(a["x"], a["dt"], a["A"], a["B"], a["C"], z=a["z"], D=a["D"], dt_bias=a["dt_bias"],
                                output_final_state=True)
    assert torch.equal(o, o2) and torch.equal(ht, ht2)
    # axes in another order: a copy is made
    o3, _ = wk.selective_scan(x.transpose(1, 2).contiguous().transpose(1, 2), a["dt"], a["A"].t().contiguous().t(),
                              Bv.transpose(2, 3).contiguous().transpose(2, 3), Cv, z=z, D=a["D"],
                              dt_bias=a["dt_bias"])
    assert torch.equal(o3, o2)


@pytest.mark.parametrize("dtype,D,N,G", [(BF, 64, 16, 1), (F32, 37, 8, 1), (FH, 40, 64, 2), (BF, 12, 128, 1), (F32, 24, 32, 3)])
@pytest.mark.parametrize("lengths", [[900, 0, 3, 700, 1201], [2100], [1025, 1023]])
def test_scan_long_rows_split_in_time(cuda, dtype, D, N, G, lengths):
    """Few rows of many tokens: their parts run side by side; short sequences
    among them leave parts empty."""
    a = _scan_inputs(cuda, (1, sum(lengths)), D, N, G, dtype, seed=D)
    cu, n = _cu(lengths, cuda), len(lengths)
    h0 = torch.randn(n, D, N, device=cuda)
    bank, ids = torch.zeros(1, n + 1, D, N, device=cuda), _ids(n, n)
    bank[0, ids] = h0
    o = wk.selective_scan_prefill_slots(*[a[k] for k in ("x", "dt", "A", "B", "C")], bank, 0, ids, D=a["D"], z=a["z"],
                                        dt_bias=a["dt_bias"], cu_seqlens=cu)
    ro, tol, rh, htol = _ref(a, h0, cu)
    # a part's decay is the exponential of a sum of up to 2101 / 4 steps, each
    # rounded once: 2^-24 of it a step at most, 2^-15 in all, on what came before
    ssm_ref.check(o, ro, tol + 2.0 ** -15 * ro.abs().max() * (dtype == F32), "o")
    ssm_ref.check(bank[0, ids], rh, htol + 2.0 ** -15 * h0.abs().max().double().cpu(), "state")
    ops.check_device_status(cuda)


def test_scan_pieces_and_steps_agree(cuda):
    """A prompt at once, in pieces of every kind, and token by token."""
    D, N, T = 40, 16, 600
    a = _scan_inputs(cuda, (2, T), D, N, 2, F32, seed=9)
    names = ("x", "dt", "B", "C", "z")
    run = lambda fn, bank, lo, hi: fn(*[a[k][:, lo:hi] if k in names else a[k] for k in ("x", "dt", "A", "B", "C")],  # noqa: E731
                                      bank, 0, [2, 1], D=a["D"], z=a["z"][:, lo:hi], dt_bias=a["dt_bias"])
    ro, tol, rh, htol = _ref(a, torch.zeros(2, D, N))
    cuts = [0, 1, 9, 17, 19, 300, T]
    for bounds, fn in (([0, T], wk.selective_scan_prefill_slots), (cuts, wk.selective_scan_prefill_slots),
                       (list(range(T + 1)), wk.selective_scan_decode_slots)):
        bank = torch.zeros(1, 3, D, N, device=cuda)
        o = torch.cat([run(fn, bank, lo, hi) for lo, hi in zip(bounds, bounds[1:])], 1)
        ssm_ref.check(o, ro, tol, f"o in {len(bounds) - 1} pieces")
        ssm_ref.check(bank[0, [2, 1]], rh, htol, "state")


@pytest.mark.parametrize("dtype,B,T,D,N,G,skew", [(BF, 64, 41, 2048, 16, 1, 0), (FH, 64, 17, 2048, 16, 4, 3),
                                                  (F32, 90, 33, 1001, 32, 1, 0), (BF, 33, 20, 2050, 64, 2, 0),
                                                  (BF, 40, 35, 1030, 128, 1, 0), (FH, 130, 12, 2051, 8, 1, 1)])
def test_scan_many_rows(cuda, dtype, B, T, D, N, G, skew):
    """Enough rows for the wide launch shape, against the packed form of the
    same sequences (another shape; the tests above hold that to 64 bits): the
    same states to the bit, outputs within their sums' order."""
    a = _scan_inputs(cuda, (B, T), D + skew, N, 1, dtype, seed=B)
    for k in ("x", "dt", "z"):
        a[k] = a[k][..., skew:]
    for k in ("D", "dt_bias"):
        a[k] = a[k][skew:].contiguous()
    a["A"] = a["A"][skew:].contiguous()
    a["B"], a["C"] = (t.expand(B, T, G, N).contiguous() * torch.arange(1, G + 1, device=cuda).view(1, 1, G, 1).to(dtype)
                      for t in (a["B"], a["C"]))
    if D % G:
        a["B"], a["C"] = a["B"][:, :, :1], a["C"][:, :, :1]
    h0 = torch.randn(B, D, N, device=cuda)
    more = {k: a[k] for k in ("D", "dt_bias")}
    o, ht = wk.selective_scan(a["x"], a["dt"], a["A"], a["B"], a["C"], z=a["z"], initial_state=h0,
                              output_final_state=True, **more)
    flat = lambda t: t.reshape(1, B * T, *t.shape[2:])  # noqa: E731
    cu = torch.arange(0, B * T + 1, T, device=cuda)
    o2, ht2 = wk.selective_scan(flat(a["x"]), flat(a["dt"]), a["A"], flat(a["B"]), flat(a["C"]), z=flat(a["z"]),
                                initial_state=h0, output_final_state=True, cu_seqlens=cu, **more)
    assert torch.equal(ht, ht2)
    # fp32 sums of N terms in two orders: N 2^-24 of their magnitudes, which stay
    # below 2^7 of the largest output here; then half a step of each rounding
    u = torch.finfo(dtype).eps / 2
    w = o2.view(B, T, D).double()
    assert bool(((o.double() - w).abs() <= 2 * u * w.abs() + N * 2.0 ** -17 * w.abs().max() * 2.0 ** -7).all())


def test_scan_mixed_dtypes(cuda):
    """fp32 B and C beside bf16 activations: computed in fp32, returned in x's dtype."""
    a = _scan_inputs(cuda, (2, 9), 24, 16, 1, BF)
    a["B"], a["C"] = a["B"].float() * 1.001, a["C"].float() * 0.999
    bank = torch.randn(1, 3, 24, 16, device=cuda)
    ro, tol, rh, htol = _ref(a, bank[0, [1, 2]])
    out = torch.empty_like(a["x"])
    args = [a[k] for k in ("x", "dt", "A", "B", "C")]
    o = wk.selective_scan_prefill_slots(*args, bank, 0, [1, 2], D=a["D"], z=a["z"], dt_bias=a["dt_bias"], out=out)
    assert o.data_ptr() == out.data_ptr() and o.dtype == BF
    ssm_ref.check(o, ro, tol, "o")
    ssm_ref.check(bank[0, [1, 2]], rh, htol, "state")


def test_scan_extreme_steps(cuda):
    """Steps of e^-80 and of 90, decays that underflow, and one infinite input
    that stays in its own channel."""
    a = _scan_inputs(cuda, (1, 40), 32, 16, 1, F32, seed=3)
    a["dt"][0, 5], a["dt"][0, 6], a["dt"][0, 7] = -80.0, 94.0, 30.0
    ref = dict(a)
    ro, tol, rh, htol = _ref(ref, torch.ones(1, 32, 16))
    args = lambda v: [v[k] for k in ("x", "dt", "A", "B", "C")]  # noqa: E731
    more = {k: a[k] for k in ("D", "z", "dt_bias")}
    o, ht = wk.selective_scan(*args(a), **more, initial_state=torch.ones(1, 32, 16, device=cuda), output_final_state=True)
    ssm_ref.check(o, ro, tol, "o")
    ssm_ref.check(ht, rh, htol, "state")
    bad = dict(a, x=a["x"].clone())
    bad["x"][0, 20, 7] = float("inf")
    o2, ht2 = wk.selective_scan(*args(bad), **more, initial_state=torch.ones(1, 32, 16, device=cuda),
                                output_final_state=True)
    keep = [c for c in range(32) if c != 7]
    assert torch.equal(o2[..., keep], o[..., keep]) and torch.equal(o2[0, :20], o[0, :20])
    assert torch.equal(ht2[:, keep], ht[:, keep]) and not ht2[:, 7].isfinite().any()


# ----------------------------------------------- slots, offsets, streams, graphs

def test_bad_device_ids_skip_their_rows(cuda):
    D, N, lengths = 48, 16, [30, 25, 40]
    cu = _cu(lengths, cuda)
    a = _scan_inputs(cuda, (1, sum(lengths)), D, N, 1, BF)
    args, more = [a[k] for k in ("x", "dt", "A", "B", "C")], {k: a[k] for k in ("D", "z", "dt_bias")}
    w = torch.randn(D, 4, device=cuda).to(BF)
    good, bad = [1, 2, 3], torch.tensor([1, 77, 3], dtype=torch.int32, device=cuda)
    keep = torch.ones(sum(lengths), dtype=torch.bool)
    keep[30:55] = False
    runs = [(lambda b, i, out: wk.selective_scan_prefill_slots(*args, b, 0, i, **more, cu_seqlens=cu, out=out),
             torch.randn(1, 5, D, N, device=cuda)),
            (lambda b, i, out: wk.short_conv_prefill_slots(a["x"], w, b, 0, i, cu_seqlens=cu, out=out),
             torch.randn(1, 5, 3, D, device=cuda).to(BF))]
    for run, bank in runs:
        start, ref_bank = bank.clone(), bank.clone()
        o = torch.full_like(a["x"], 7.0)
        run(bank, bad, o)
        with pytest.raises(_lib.WkvmError, match="SLOT_RANGE"):
            ops.check_device_status(cuda)
        ref = run(ref_bank, good, None)
        assert torch.equal(o[0, keep], ref[0, keep]) and bool((o[0, ~keep] == 7).all())
        assert torch.equal(bank[0, [1, 3]], ref_bank[0, [1, 3]])
        assert torch.equal(bank[0, [0, 2, 4]], start[0, [0, 2, 4]])


def test_bad_offsets_are_reported(cuda):
    """Offsets given on the device that descend or leave the token axis: their
    sequences are skipped, the others computed, nothing outside is touched."""
    D, N = 40, 16
    a = _scan_inputs(cuda, (1, 60), D, N, 1, BF)
    args, more = [a[k] for k in ("x", "dt", "A", "B", "C")], {k: a[k] for k in ("D", "z", "dt_bias")}
    w = torch.randn(D, 4, device=cuda).to(BF)
    for cu in ([0, 20, 10, 30], [0, 25, 61], [-3, 10, 20]):
        cu = torch.tensor(cu, device=cuda)
        n = len(cu) - 1
        ok = [i for i in range(n) if 0 <= cu[i] <= cu[i + 1] <= 60]
        for fn, bank in ((lambda b: wk.selective_scan_prefill_slots(*args, b, 0, list(range(1, n + 1)), **more,
                                                                    cu_seqlens=cu), torch.randn(1, 5, D, N, device=cuda)),
                         (lambda b: wk.short_conv_prefill_slots(a["x"], w, b, 0, list(range(1, n + 1)),
                                                                cu_seqlens=cu), torch.randn(1, 5, 3, D, device=cuda).to(BF))):
            start = bank.clone()
            fn(bank)
            with pytest.raises(_lib.WkvmError, match="INVALID_ARG"):
                ops.check_device_status(cuda)
            changed = [i for i in range(5) if not torch.equal(bank[0, i], start[0, i])]
            assert changed == [i + 1 for i in ok if cu[i + 1] > cu[i]]


def test_tokens_behind_the_last_sequence_stay(cuda):
    D, N = 40, 16
    a = _scan_inputs(cuda, (1, 100), D, N, 1, BF)
    args = [a[k] for k in ("x", "dt", "A", "B", "C")]
    w, cu = torch.randn(D, 4, device=cuda).to(BF), torch.tensor([3, 40, 71], device=cuda)
    for fn, bank in ((lambda b, o: wk.selective_scan_prefill_slots(*args, b, 0, [1, 2], cu_seqlens=cu, out=o),
                      torch.randn(1, 3, D, N, device=cuda)),
                     (lambda b, o: wk.short_conv_prefill_slots(a["x"], w, b, 0, [1, 2], cu_seqlens=cu, out=o),
                      torch.randn(1, 3, 3, D, device=cuda).to(BF))):
        o = torch.full_like(a["x"], float("nan"))  # a value that no output takes here
        fn(bank, o)
        assert bool(o[0, :3].isnan().all()) and bool(o[0, 71:].isnan().all()) and not bool(o[0, 3:71].isnan().any())


def test_offsets_past_32_bits(cuda):
    """Slots and tokens whose element offsets do not fit 32 bits."""
    D, N, S = 4096, 128, 4200  # 2.2e9 state elements
    bank = torch.zeros(1, S, D, N, device=cuda)
    small = torch.zeros(1, 3, D, N, device=cuda)
    a = _scan_inputs(cuda, (2, 1), D, N, 1, BF)
    args = [a[k] for k in ("x", "dt", "A", "B", "C")]
    bank[0, S - 1] = small[0, 1] = 0.5
    o = wk.selective_scan_decode_slots(*args, bank, 0, [S - 1, S - 2])
    ref = wk.selective_scan_decode_slots(*args, small, 0, [1, 2])
    assert torch.equal(o, ref) and torch.equal(bank[0, [S - 1, S - 2]], small[0, [1, 2]])
    del bank, small
    # tokens 2^26 elements apart
    T, d = 40, 64
    buf = torch.empty(T * (1 << 26), dtype=BF, device=cuda)
    b = _scan_inputs(cuda, (1, T), d, 16, 1, BF)
    far = buf.as_strided((1, T, d), (0, 1 << 26, 1))
    far.copy_(b["x"])
    rest = [b[k] for k in ("dt", "A", "B", "C")]
    assert torch.equal(wk.selective_scan(far, *rest)[0], wk.selective_scan(b["x"], *rest)[0])
    w = torch.randn(d, 4, device=cuda).to(BF)
    assert torch.equal(wk.short_conv(far, w)[0], wk.short_conv(b["x"], w)[0])


def test_other_stream_and_graph_replay(cuda):
    """Decode steps captured into a graph and replayed equal the same steps
    run eagerly, on another stream than the default."""
    D, N, B = 64, 16, 4
    w = torch.randn(D, 4, device=cuda).to(BF)
    p = _scan_inputs(cuda, (B, 1), D, N, 1, BF)
    ids = torch.tensor([4, 1, 3, 2], dtype=torch.int32, device=cuda)
    conv = torch.randn(1, 5, 3, D, device=cuda).to(BF)
    ssm = torch.randn(1, 5, D, N, device=cuda)
    conv2, ssm2 = conv.clone(), ssm.clone()
    x = torch.zeros(B, 1, D, device=cuda, dtype=BF)

    def step(inp, c, s):
        y = wk.short_conv_decode_slots(inp, w, c, 0, ids, activation="silu")
        return wk.selective_scan_decode_slots(y, p["dt"], p["A"], p["B"], p["C"], s, 0, ids, D=p["D"], z=p["z"],
                                              dt_bias=p["dt_bias"])

    inputs = [torch.randn(B, 1, D, device=cuda).to(BF) for _ in range(6)]
    side = torch.cuda.Stream(cuda)
    with torch.cuda.stream(side):
        ref = [step(i, conv2, ssm2) for i in inputs]
    side.synchronize()
    ops.status_word(cuda)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = step(x, conv, ssm)
    got = []
    for i in inputs:
        x.copy_(i)
        graph.replay()
        got.append(o.clone())
    torch.cuda.synchronize()
    assert all(torch.equal(g, r) for g, r in zip(got, ref))
    assert torch.equal(conv, conv2) and torch.equal(ssm, ssm2)


def test_two_streams_at_once(cuda):
    """Prompts over disjoint slots of one bank on two streams at once."""
    D, N, T = 512, 16, 700
    bank = torch.randn(1, 5, D, N, device=cuda)
    ref = bank.clone()
    sets = [_scan_inputs(cuda, (2, T), D, N, 1, BF, seed=s) for s in (1, 2)]
    args = [[a[k] for k in ("x", "dt", "A", "B", "C")] for a in sets]
    want = [wk.selective_scan_prefill_slots(*v, ref, 0, i) for v, i in zip(args, ([1, 2], [3, 4]))]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(cuda) for _ in sets]
    got = []
    for s, v, i in zip(streams, args, ([1, 2], [3, 4])):
        with torch.cuda.stream(s):
            got.append(wk.selective_scan_prefill_slots(*v, bank, 0, torch.tensor(i, dtype=torch.int32).to(cuda)))
    torch.cuda.synchronize()
    assert all(torch.equal(g, w) for g, w in zip(got, want)) and torch.equal(bank, ref)


def test_empty_calls(cuda):
    D, N = 24, 16
    bank, conv = torch.randn(1, 3, D, N, device=cuda), torch.randn(1, 3, 3, D, device=cuda).to(BF)
    b0, c0 = bank.clone(), conv.clone()
    w = torch.randn(D, 4, device=cuda).to(BF)
    for B, T, ids in ((0, 4, []), (2, 0, [1, 2])):
        a = _scan_inputs(cuda, (B, T), D, N, 1, BF)
        args = [a[k] for k in ("x", "dt", "A", "B", "C")]
        assert wk.selective_scan_prefill_slots(*args, bank, 0, ids).shape == (B, T, D)
        assert wk.short_conv_prefill_slots(a["x"], w, conv, 0, ids).shape == (B, T, D)
        o, ht = wk.selective_scan(*args, output_final_state=True)
        assert o.shape == (B, T, D) and ht.shape == (B, D, N) and not ht.any()
        o, st = wk.short_conv(a["x"], w, output_final_state=True)
        assert st.shape == (B, 3, D) and not st.any()
    assert torch.equal(bank, b0) and torch.equal(conv, c0)
