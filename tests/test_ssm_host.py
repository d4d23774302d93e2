"""Refusals of the selective state space operators and of sampling, found on
the host (no GPU, nothing launched)."""

import ctypes

import pytest
import torch

import wkvm_b200 as wk
from wkvm_b200 import _lib, ssm


@pytest.fixture(scope="module")
def lib():
    from wkvm_b200 import build
    build.build()
    return _lib.load()


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(1, 2, 8), torch.zeros(8, 4)
    with pytest.raises(ValueError, match="CUDA"):
        wk.short_conv(x, w)
    with pytest.raises(ValueError, match="CUDA"):
        wk.selective_scan(x, x, torch.zeros(8, 16), torch.zeros(1, 2, 16), torch.zeros(1, 2, 16))
    with pytest.raises(ValueError, match="CUDA"):
        wk.sample_tokens(torch.zeros(2, 8), torch.zeros(2))


@pytest.fixture
def anywhere(monkeypatch):
    """The checks behind the one for CUDA tensors, with nothing launched."""
    from wkvm_b200 import ops
    monkeypatch.setattr(ops, "_require_cuda", lambda *t: None)

    def call(name, *args):
        raise AssertionError(f"{name} would have been launched")

    monkeypatch.setattr(_lib, "call", call)


def test_conv_refusals(anywhere):
    x, w = torch.zeros(2, 3, 8), torch.zeros(8, 4)
    bank = torch.zeros(2, 5, 3, 8)
    bad = [
        (dict(x=x[0]), ValueError, r"x must be \[B, T, D\]"),
        (dict(x=x.double()), ValueError, "unsupported dtype"),
        (dict(weight=torch.zeros(7, 4)), ValueError, "weight must be"),
        (dict(weight=torch.zeros(8, 5)), ValueError, "width of 5"),
        (dict(weight=torch.zeros(8, 1)), ValueError, "width of 1"),
        (dict(bias=torch.zeros(9)), ValueError, "bias must be"),
        (dict(activation="gelu"), ValueError, "activation"),
        (dict(bank_conv=bank.to(torch.bfloat16)), ValueError, "conv bank"),
        (dict(bank_conv=bank[:, :, :2]), ValueError, "conv bank"),
        (dict(bank_conv=torch.zeros(2, 5, 2, 8)), ValueError, "bank rows"),
        (dict(layer=2), IndexError, "layer 2"),
        (dict(layer=-1), IndexError, "layer -1"),
        (dict(slot_ids=[1]), ValueError, "1 slot ids for 2"),
        (dict(slot_ids=[1, 1]), _lib.WkvmError, "DUPLICATE"),
        (dict(slot_ids=[1, 5]), _lib.WkvmError, "SLOT_RANGE"),
        (dict(out=torch.zeros(2, 3, 9)), ValueError, "out must be"),
        (dict(cu_seqlens=torch.tensor([0, 3])), ValueError, "batch size is expected to be 1"),
        (dict(x=torch.zeros(2, 3, 8, requires_grad=True)), RuntimeError, "no backward"),
    ]
    for change, err, text in bad:
        kw = dict(x=torch.zeros(2, 3, 8), weight=w, bank_conv=bank, layer=0, slot_ids=[1, 2]) | change
        with pytest.raises(err, match=text):
            wk.short_conv_prefill_slots(**kw)
    with pytest.raises(ValueError, match="overlaps"):
        wk.short_conv_decode_slots(x, w, bank, 0, [1, 2], out=x)
    with pytest.raises(ValueError, match="initial_state must be"):
        wk.short_conv(torch.zeros(2, 3, 8), w, initial_state=torch.zeros(2, 4, 8))
    with pytest.raises(ValueError, match="must ascend"):
        wk.short_conv(torch.zeros(1, 6, 8), w, cu_seqlens=torch.tensor([0, 4, 3]))
    with pytest.raises(ValueError, match="must ascend"):
        wk.short_conv(torch.zeros(1, 6, 8), w, cu_seqlens=torch.tensor([0, 7]))


def test_scan_refusals(anywhere):
    def args(**change):
        x = torch.zeros(2, 3, 12)
        bc = torch.zeros(2, 3, 2, 16)
        return dict(x=x, dt=x, A=torch.zeros(12, 16), B=bc, C=bc, bank_ssm=torch.zeros(1, 4, 12, 16), layer=0,
                    slot_ids=[1, 2]) | change

    bad = [
        (dict(x=torch.zeros(3, 12)), "x must be"),
        (dict(x=torch.zeros(2, 3, 12, dtype=torch.float64)), "unsupported dtype"),
        (dict(dt=torch.zeros(2, 3, 1)), "dt must have x's shape"),
        (dict(z=torch.zeros(2, 4, 12)), "z must have x's shape"),
        (dict(A=torch.zeros(16, 12)), "A must be"),
        (dict(A=torch.zeros(12, 20)), "20 states"),
        (dict(A=torch.zeros(12, 256)), "256 states"),
        (dict(B=torch.zeros(2, 3, 2, 8)), "B must be"),
        (dict(C=torch.zeros(2, 3, 1, 16)), "C must be"),
        (dict(B=torch.zeros(2, 3, 5, 16), C=torch.zeros(2, 3, 5, 16)), "5 groups"),
        (dict(B=torch.zeros(2, 3, 0, 16), C=torch.zeros(2, 3, 0, 16)), "0 groups"),
        (dict(D=torch.zeros(13)), "D must be"),
        (dict(dt_bias=torch.zeros(1)), "dt_bias must be"),
        (dict(bank_ssm=torch.zeros(1, 4, 16, 12)), "bank rows"),
        (dict(bank_ssm=torch.zeros(1, 4, 12, 16, dtype=torch.float16)), "ssm bank"),
        (dict(bank_ssm=torch.zeros(1, 4, 12, 32)[..., ::2]), "ssm bank"),
        (dict(slot_ids=[1, 2, 3]), "3 slot ids for 2"),
        (dict(out=torch.zeros(2, 3, 12, dtype=torch.float16)), "out must be"),
    ]
    for change, text in bad:
        with pytest.raises(ValueError, match=text):
            wk.selective_scan_prefill_slots(**args(**change))
    with pytest.raises(RuntimeError, match="no backward"):
        wk.selective_scan_decode_slots(**args(A=torch.zeros(12, 16, requires_grad=True)))
    kw = args()
    with pytest.raises(ValueError, match="overlaps"):
        wk.selective_scan_prefill_slots(**kw, z=torch.zeros(2, 3, 12), out=kw["x"])
    a = args()
    with pytest.raises(ValueError, match="initial_state must be"):
        wk.selective_scan(a["x"], a["dt"], a["A"], a["B"], a["C"], initial_state=torch.zeros(2, 16, 12))


def test_sampling_refusals(anywhere):
    x, u = torch.zeros(3, 9), torch.zeros(3)
    for change, text in [(dict(logits=x[0]), "logits must be"), (dict(logits=x.double()), "unsupported dtype"),
                         (dict(logits=x[:, :0]), "vocabulary of 0"), (dict(u=u[:2]), "u must be"),
                         (dict(temperature=-1.0), "temperature must be >= 0"), (dict(top_k=-1), "top_k must be >= 0"),
                         (dict(top_p=float("nan")), "top_p must be >= 0"), (dict(min_p=1.5), "min_p must be <= 1"),
                         (dict(top_p=torch.zeros(2)), "top_p must be a number"), (dict(top_k=None), "top_k must be")]:
        with pytest.raises(ValueError, match=text):
            wk.sample_tokens(**(dict(logits=x, u=u) | change))


def test_strides_given_to_the_kernels():
    t = torch.zeros(4, 5, 6)
    assert ssm._rows(t)[0] is t and ssm._rows(t)[1] == (30, 6, 1)
    half = torch.zeros(4, 5, 12)[..., 6:]
    assert ssm._rows(half)[0] is half and ssm._rows(half)[1] == (60, 12, 1)
    turned = torch.zeros(4, 6, 5).transpose(1, 2)
    assert ssm._rows(turned)[0].is_contiguous() and ssm._rows(turned)[1] == (30, 6, 1)
    groups = torch.zeros(4, 5, 40)[..., 3:35].unflatten(-1, (2, 16))
    assert ssm._rows(groups, 2)[0] is groups and ssm._rows(groups, 2)[1] == (200, 40, 16, 1)
    gapped = torch.zeros(4, 5, 2, 20)[..., :16]
    assert ssm._rows(gapped, 2)[0].is_contiguous()


def test_c_entry_refusals(lib):
    """Status codes of the C entry points; every call is refused or empty, so
    nothing is launched."""
    P, n = ctypes.c_void_p, None
    d = P(4096)
    s = (ctypes.c_int64 * 10)()

    def conv(B=1, T=1, D=8, W=4, act=0, dt=1, x=d, w=d, o=d):
        return lib.wkvm_short_conv(x, 0, 0, w, n, o, n, n, n, B, T, D, W, act, dt, n, n)

    assert conv(B=-1) == -1 and conv(T=-1) == -1 and conv(D=0) == -1 and conv(act=2) == -1
    assert conv(W=5) == -2 and conv(W=1) == -2 and conv(dt=3) == -3
    assert conv(x=n) == -1 and conv(w=n) == -1 and conv(o=n) == -1 and conv(B=0) == 0
    slots = lambda bank=d, ns=4, ids=d, B=1: lib.wkvm_short_conv_slots(  # noqa: E731
        d, 0, 0, d, n, d, bank, ns, ids, n, B, 1, 8, 4, 0, 1, n, n)
    assert slots(bank=n) == -1 and slots(ns=0) == -1 and slots(ids=n) == -1 and slots(B=0) == 0

    def scan(B=1, T=1, D=8, N=16, G=1, dt=1, A=d, x=d, st=s, h0=n):
        return lib.wkvm_selective_scan(x, d, A, d, d, n, n, n, d, st, h0, n, n, B, T, D, N, G, 1, dt, n, n)

    assert scan(B=-1) == -1 and scan(T=-1) == -1 and scan(D=0) == -1 and scan(G=0) == -1 and scan(N=0) == -1
    assert scan(N=24) == -2 and scan(G=3) == -2 and scan(dt=9) == -3 and scan(A=n) == -1 and scan(x=n) == -1
    assert scan(st=n) == -1 and scan(A=P(4100)) == -7 and scan(h0=P(4100)) == -7 and scan(B=0) == 0
    sslots = lambda bank=d, ns=4, ids=d, B=1: lib.wkvm_selective_scan_slots(  # noqa: E731
        d, d, d, d, d, n, n, n, d, s, bank, ns, ids, n, B, 1, 8, 16, 1, 1, 1, n, n)
    assert sslots(bank=n) == -1 and sslots(ns=0) == -1 and sslots(ids=n) == -1 and sslots(B=0) == 0

    def sample(B=1, V=8, dt=1, x=d, u=d, o=d):
        f = ctypes.c_float
        return lib.wkvm_sample_tokens(x, 8, u, n, n, n, n, f(1), 0, f(1), f(0), o, o, B, V, dt, n, n)

    assert sample(B=-1) == -1 and sample(V=0) == -1 and sample(dt=5) == -3 and sample(x=n) == -1
    assert sample(u=n) == -1 and sample(o=n) == -1 and sample(B=0) == 0


def test_bank_layout():
    from wkvm_b200.state import SSMStateBank, SSMStateLayout
    lay = SSMStateLayout(2, 24, 8, 3, torch.float16)
    bank = SSMStateBank(lay, num_slots=3, device="cpu")
    assert bank.ssm.shape == (2, 4, 24, 8) and bank.conv.shape == (2, 4, 2, 24) and bank.conv.dtype == torch.float16
    with pytest.raises(ValueError, match="multiples of 16 bytes"):
        SSMStateLayout(2, 25, 16, 4)
    with pytest.raises(_lib.WkvmError, match="SLOT_RANGE"):
        bank.device_ids([4])
