"""Calls of the selective state space operators and of sampling that are
refused on the host, and the host's checks of tokens (no GPU, nothing launched)."""

import ctypes
import math

import pytest
import torch

import wkvm_b200 as wk


@pytest.fixture
def anywhere(monkeypatch):
    """The checks behind the one for CUDA tensors; a launch is recorded instead."""
    from wkvm_b200 import ops
    calls = []
    monkeypatch.setattr(ops, "_require_cuda", lambda *t: None)
    monkeypatch.setattr(ops, "_launch", lambda name, idx, *args: calls.append((name, args)))
    return calls


def _top_k0(call):
    return call[1][8]  # of wkvm_sample_tokens: the scalar beside the device array


def test_top_k_is_a_whole_number(anywhere):
    x, u = torch.zeros(3, 9), torch.zeros(3)
    for k in (0.5, 2.7, math.inf):
        with pytest.raises(ValueError, match="top_k must be a whole number"):
            wk.sample_tokens(x, u, top_k=k)
    assert not anywhere
    for k, want in ((4, 4), (4.0, 4), (0, 0), (10 ** 12, 9)):
        wk.sample_tokens(x, u, top_k=k)
        assert _top_k0(anywhere[-1]) == want


def test_top_k_tensors_become_whole_numbers():
    """Per-row values of any type reach the kernel as int32; a fraction never as the 0 that keeps everything."""
    from wkvm_b200.sampling import _setting
    x = torch.zeros(4, 9)
    for value, want in ((torch.tensor([0.0, 0.5, 2.7, 1e12]), [0, 1, 3, 1 << 30]),
                        (torch.tensor([-3, 0, 7, 1 << 40]), [0, 0, 7, 1 << 30]),
                        (torch.tensor(0.25, dtype=torch.float64), [1] * 4)):
        got, scalar = _setting("top_k", value, 4, torch.int32, x)
        assert got.dtype is torch.int32 and got.tolist() == want and scalar == 0


def test_sampling_refuses_inputs_that_ask_for_gradients(anywhere):
    x, u = torch.zeros(3, 9), torch.zeros(3)
    t = lambda: torch.ones(3, requires_grad=True)  # noqa: E731
    for change in (dict(logits=torch.zeros(3, 9, requires_grad=True)), dict(u=t()), dict(temperature=t()),
                   dict(top_p=t()), dict(min_p=t())):
        kw = dict(logits=x, u=u) | change
        with pytest.raises(RuntimeError, match="no backward"):
            wk.sample_tokens(**kw)
        assert not anywhere
        with torch.no_grad():
            wk.sample_tokens(**kw)
        assert anywhere.pop()


def test_vocabularies_beyond_the_masses_resolution(anywhere):
    """Past 2^20 logits the masses' rounding would exceed two steps of an fp32 u."""
    x = torch.zeros(1, 1).expand(1, (1 << 20) + 1)
    with pytest.raises(ValueError, match="a vocabulary of 1048577 is not supported"):
        wk.sample_tokens(x, torch.zeros(1))
    assert not anywhere
    from wkvm_b200 import _lib, build
    build.build()
    p, f, n = ctypes.c_void_p(4096), ctypes.c_float, None
    assert _lib.load().wkvm_sample_tokens(p, 8, p, n, n, n, n, f(1), 0, f(1), f(0), p, p, 1, (1 << 20) + 1, 1, n, n) == -2


class _Model:
    """Stands in for a causal language model; a forward pass would be recorded."""

    def __init__(self, vocab):
        self.table, self.seen = torch.nn.Embedding(vocab, 2), []

    def get_input_embeddings(self):
        return self.table

    def __call__(self, input_ids, **kw):
        self.seen.append(input_ids)
        raise AssertionError("the model was called")


class _Bank:
    device, num_slots = torch.device("cpu"), 4

    def gather_cache(self, slot_batch):
        return None


@pytest.mark.parametrize("tokens", [[3, -1], [50, 7], [-1, 2 ** 40]])
def test_tokens_outside_the_vocabulary_never_reach_the_model(tokens):
    """-1 is what sampling gives for a row with nothing to choose; the
    embedding's lookup would fault on the device."""
    from wkvm_b200.graph import GraphedDecode
    from wkvm_b200.runner import RWKV7Runner, checked_tokens
    model, batch = _Model(50), [{"wkv": 1, "shift": 1}, {"wkv": 2, "shift": 2}]
    runner = RWKV7Runner(model, _Bank())
    graphed = GraphedDecode.__new__(GraphedDecode)  # a captured step, without its graph
    graphed.runner, graphed.batch_size = runner, 2
    for call in (lambda: runner.decode_step(batch, tokens), lambda: runner.prefill(tokens, batch[0]),
                 lambda: runner.sample_step(batch, tokens, torch.zeros(2)), lambda: graphed.decode_step(batch, tokens),
                 lambda: graphed.sample_step(batch, tokens, torch.zeros(2))):
        with pytest.raises(ValueError, match="leave the vocabulary of 50"):
            call()
    assert not model.seen
    with pytest.raises(AssertionError, match="the model was called"):
        runner.decode_step(batch, [0, 49])
    assert model.seen[0].tolist() == [[0], [49]]
    assert checked_tokens([], model).numel() == 0


def test_sizes_beyond_32_bits_are_refused(anywhere):
    """The kernels count in int32: a larger size would wrap in the call, to a smaller one that runs."""
    big = (1 << 32) + 8
    e = lambda *s: torch.empty(*s, device="meta")  # noqa: E731
    for B, T, D in ((1, 1, big), (1, big, 8), (big, 1, 8)):
        x, bc = e(B, T, D), e(B, T, 8)
        with pytest.raises(ValueError, match="more than an int32 counts"):
            wk.short_conv(x, e(D, 4))
        with pytest.raises(ValueError, match="more than an int32 counts"):
            wk.selective_scan(x, x, e(D, 8), bc, bc)
    with pytest.raises(ValueError, match="more than an int32 counts"):
        wk.sample_tokens(e(big, 1), e(big))
    assert not anywhere


def test_restored_host_copies_live_until_the_kernels_have_read_them(monkeypatch):
    """The restore kernels read pinned memory directly, and its allocator does
    not know: a copy freed ahead of the synchronise could be handed out again."""
    import gc
    import weakref

    from wkvm_b200 import state
    staged, read = [], []

    class Stream:
        def synchronize(self):
            gc.collect()
            read.append([r() is not None for r in staged])

    monkeypatch.setattr(state, "_pinned", lambda t: t.clone())
    monkeypatch.setattr(state.ops, "slot_restore", lambda fam, dim, ids, packed: staged.append(weakref.ref(packed)))
    monkeypatch.setattr(state.torch.cuda, "current_stream", lambda dev: Stream())
    bank = state.SSMStateBank(state.SSMStateLayout(2, 24, 8, 3, torch.float16), num_slots=3, device="cpu")
    bank.restore([1, 2], {"ssm": torch.zeros(2, 2, 24, 8), "conv": torch.zeros(2, 2, 2, 24, dtype=torch.float16)})
    lay = state.RWKV7StateLayout(n_layer=2, hidden_size=8, num_heads=1, head_dim=4, head_v_dim=4)
    bank = state.RWKV7StateBank(lay, num_slots=3, device="cpu")
    bank.restore({"wkv": 1, "shift": 1}, {"wkv": torch.zeros(2, 1, 4, 4), "shift": torch.zeros(2, 2, 8)})
    assert read[0] == [True, True] and read[1][2:] == [True, True]
