"""The operators as they are used together: a small selective state space
language model over bank slots, prompts packed, decode steps with the choice
of tokens inside one captured graph; the bank's slot operations; sampling
behind the RWKV-7 runner."""

import pytest
import torch

import wkvm_b200 as wk
from wkvm_b200 import ops
from wkvm_b200.state import SSMStateBank, SSMStateLayout

pytestmark = pytest.mark.gpu

L, H, D, N, W, R, VOCAB = 2, 48, 96, 16, 4, 6, 700


def _weights(device, dtype):
    g = torch.Generator().manual_seed(3)
    r = lambda *s, k: (torch.randn(*s, generator=g) / k ** 0.5)  # noqa: E731
    layers = [dict(inp=r(2 * D, H, k=H), conv=r(D, W, k=W), conv_b=0.1 * r(D, k=1), proj=r(R + 2 * N, D, k=D),
                   dt=r(D, R, k=R), dt_b=-3 + r(D, k=1), A=-torch.exp(0.5 * r(D, N, k=1)), D=1 + 0.1 * r(D, k=1),
                   out=r(H, D, k=D)) for _ in range(L)]
    top = dict(emb=r(VOCAB, H, k=1), head=3 * r(VOCAB, H, k=H))
    f32 = ("A", "D", "dt_b")
    return ([{n: t.to(device, torch.float32 if n in f32 and dtype != torch.float64 else dtype) for n, t in w.items()}
             for w in layers], {n: t.to(device, dtype) for n, t in top.items()})


def _forward(bank, layers, top, tokens, ids, cu=None):
    """Logits of every token; tokens [B, T] (decode) or [1, total] with cu."""
    h = top["emb"][tokens]
    for i, w in enumerate(layers):
        x, z = (h @ w["inp"].t()).split(D, -1)
        x = bank.conv_prefill(i, ids, x, w["conv"], w["conv_b"], cu_seqlens=cu)
        dt, B, C = (x @ w["proj"].t()).split([R, N, N], -1)
        y = bank.scan_prefill(i, ids, x, dt @ w["dt"].t(), w["A"], B, C, cu_seqlens=cu, D=w["D"], z=z,
                              dt_bias=w["dt_b"])
        h = h + y @ w["out"].t()
    return h @ top["head"].t()


def _reference(layers, top, tokens):
    """Logits of every token of one sequence in 64 bits, from an empty state."""
    h = top["emb"][tokens]
    for w in layers:
        x, z = (h @ w["inp"].t()).split(D, -1)
        x = torch.cat([x.new_zeros(W - 1, D), x]).unfold(0, W, 1)
        x = torch.nn.functional.silu((x * w["conv"]).sum(-1) + w["conv_b"])
        dt, B, C = (x @ w["proj"].t()).split([R, N, N], -1)
        step = torch.nn.functional.softplus(dt @ w["dt"].t() + w["dt_b"], threshold=60.0)
        s, y = x.new_zeros(D, N), []
        for t in range(len(x)):
            s = torch.exp(step[t, :, None] * w["A"]) * s + (step[t] * x[t])[:, None] * B[t]
            y.append(s @ C[t])
        h = h + ((torch.stack(y) + w["D"] * x) * torch.nn.functional.silu(z)) @ w["out"].t()
    return h @ top["head"].t()


def test_prompts_then_graphed_decode_with_sampling(cuda, monkeypatch):
    monkeypatch.setattr(torch.backends.cuda.matmul, "allow_tf32", False)
    layers, top = _weights(cuda, torch.float32)
    bank = SSMStateBank(SSMStateLayout(L, D, N, W, torch.float32), num_slots=6, device=cuda)
    g = torch.Generator().manual_seed(1)
    lengths, slots, steps = [37, 1, 70], [5, 2, 3], 12
    prompts = [torch.randint(0, VOCAB, (n,), generator=g) for n in lengths]
    cu = torch.tensor([0, 37, 38, 108], device=cuda)
    ids = bank.device_ids(slots)
    u = torch.rand(steps + 1, 3, generator=g).to(cuda)
    settings = dict(temperature=torch.tensor([0.8, 1.0, 1.3], device=cuda),
                    top_k=torch.tensor([0, 50, 200], dtype=torch.int32, device=cuda), top_p=0.95)
    with torch.inference_mode():
        logits = _forward(bank, layers, top, torch.cat(prompts)[None].to(cuda), ids, cu)
        first, first_lp = wk.sample_tokens(logits[0, cu[1:] - 1], u[0], **settings)
        start = bank.snapshot(slots)

        def step(tok, uu):
            return wk.sample_tokens(_forward(bank, layers, top, tok[:, None], ids)[:, 0], uu, **settings)

        eager, lps = [first], [first_lp]
        for i in range(steps):
            t, lp = step(eager[-1], u[i + 1])
            eager.append(t)
            lps.append(lp)
        end = bank.snapshot(slots)
        # the same steps as one captured graph, replayed
        bank.restore(slots, start)
        tok, uu = first.clone(), u[1].clone()
        warm = bank.device_ids([1, 4, 6])  # other slots, for the first calls of each kernel
        _forward(bank, layers, top, tok[:, None], warm)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(tok, uu)
        replayed = [first]
        for i in range(steps):
            tok.copy_(replayed[-1])
            uu.copy_(u[i + 1])
            graph.replay()
            replayed.append(out[0].clone())
        again = bank.snapshot(slots)
    ops.check_device_status(cuda)
    assert torch.equal(torch.stack(replayed), torch.stack(eager))
    assert all(torch.equal(end[n], again[n]) for n in end)
    assert not bank.ssm[:, 0].any() and not bank.conv[:, 0].any()
    # the whole run in 64 bits on the tokens that were drawn: each one's
    # probability, and its place in the distribution
    rl, rt = _weights("cpu", torch.float64)
    drawn, lps = torch.stack(eager).cpu(), torch.stack(lps).double().cpu()
    import ssm_ref
    for i, p in enumerate(prompts):
        ref = _reference(rl, rt, torch.cat([p, drawn[:-1, i]]))[len(p) - 1:]
        temp, k = float(settings["temperature"][i]), int(settings["top_k"][i])
        want, wlp = ssm_ref.sample(ref, u[:, i].tolist(), [temp] * len(ref), [k] * len(ref),
                                   [float(torch.tensor(0.95))] * len(ref), [0.0] * len(ref))
        same = torch.from_numpy(want) == drawn[:, i]
        # fp32 logits are off by some 1e-5: a token changes where the uniform
        # number or the nucleus' edge falls that close to a border
        assert same.double().mean() >= 0.9
        assert ((torch.from_numpy(wlp) - lps[:, i])[same].abs() < 1e-3).all()


def test_bank_slot_operations(cuda):
    bank = SSMStateBank(SSMStateLayout(3, 64, 16, 4, torch.bfloat16), num_slots=5, device=cuda)
    bank.ssm.normal_()
    bank.conv.normal_()
    ssm, conv = bank.ssm.clone(), bank.conv.clone()
    bank.fork([1, 2], [4, 5])
    assert torch.equal(bank.ssm[:, [4, 5]], ssm[:, [1, 2]]) and torch.equal(bank.conv[:, [4, 5]], conv[:, [1, 2]])
    snap = bank.snapshot([3, 1])
    assert torch.equal(snap["ssm"][0], ssm[:, 3].cpu()) and torch.equal(snap["conv"][1], conv[:, 1].cpu())
    bank.zero([3])
    assert not bank.ssm[:, 3].any() and not bank.conv[:, 3].any()
    bank.restore([2, 3], snap)
    assert torch.equal(bank.ssm[:, [2, 3]], ssm[:, [3, 1]]) and torch.equal(bank.conv[:, [2, 3]], conv[:, [3, 1]])
    assert torch.equal(bank.ssm[:, [0, 1]], ssm[:, [0, 1]])
    assert bank.state_bytes() == ssm.numel() * 4 + conv.numel() * 2


def test_sampling_behind_the_runner(cuda):
    """RWKV7Runner.sample_step and GraphedDecode.sample_step choose what
    sample_tokens chooses on decode_step's logits."""
    fla_models = pytest.importorskip("fla.models.rwkv7")
    from wkvm_b200 import fla_compat
    from wkvm_b200.graph import GraphedDecode
    from wkvm_b200.runner import RWKV7Runner
    from wkvm_b200.state import RWKV7StateBank, RWKV7StateLayout
    torch.manual_seed(0)
    cfg = fla_models.RWKV7Config(hidden_size=128, num_hidden_layers=2, head_dim=64, vocab_size=512)
    with torch.device(cuda):
        model = fla_models.RWKV7ForCausalLM(cfg)
    model = model.to(torch.bfloat16).eval()
    lay = RWKV7StateLayout(n_layer=2, hidden_size=128, num_heads=2, head_dim=64, head_v_dim=64)
    banks = [RWKV7StateBank(lay, num_slots=4, device=cuda) for _ in range(3)]
    batch = [{"wkv": 2, "shift": 2}, {"wkv": 4, "shift": 4}]
    u = torch.tensor([0.3, 0.8], device=cuda)
    kw = dict(temperature=0.9, top_k=100, top_p=0.9)
    try:
        gd = GraphedDecode(RWKV7Runner(model, banks[0]), batch_size=2)  # installs the fused ops
        tok = [[7, 9]] * 3
        for _ in range(4):
            got = [gd.sample_step(batch, tok[0], u, **kw),
                   RWKV7Runner(model, banks[1]).sample_step(batch, tok[1], u, **kw),
                   wk.sample_tokens(RWKV7Runner(model, banks[2]).decode_step(batch, tok[2]), u, **kw)]
            assert torch.equal(got[1][0], got[2][0]) and torch.equal(got[1][1], got[2][1])
            assert torch.equal(got[0][0], got[2][0])
            tok = [t.tolist() for t, _ in got]
    finally:
        fla_compat.uninstall()
