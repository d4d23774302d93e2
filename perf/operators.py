"""The selective state space scan with its short causal convolution, and the
choice of the next tokens, as one pass each over slots of a state bank or over
a batch of logits rows: what is measured, in elementary torch operations and
as calls of wkvm_b200.

A case is one call:
  conv_step, conv   short causal convolution over bank slots: T new tokens of
                    every slot, or packed prompts of unequal lengths
  scan_step, scan   selective scan over bank slots, the same two forms
  sample            one token for each row of logits, from a given uniform
                    number, under temperature, top-k, top-p and min-p
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # a handful of sessions decode one token: launch latency
        dict(name="conv_step_8", op="conv_step", batch=8, tokens=1, slots=64, channels=4096, width=4,
             silu=True, bias=True, dtype="bf16"),
        # a full decode batch of a served model
        dict(name="conv_step_512", op="conv_step", batch=512, tokens=1, slots=1024, channels=8192,
             width=4, silu=True, bias=True, dtype="bf16"),
        # sixteen prompts of unequal lengths, packed
        dict(name="conv_packed", op="conv", seqs=16, total=32768, slots=64, channels=4096, width=4,
             silu=True, bias=True, dtype="bf16"),
        # an odd channel count and width, 32-bit activations, no activation function
        dict(name="conv_odd", op="conv", seqs=5, total=9001, slots=8, channels=1537, width=3,
             silu=False, bias=False, dtype="fp32"),
        # one session decodes one token: launch latency
        dict(name="scan_step_1", op="scan_step", batch=1, tokens=1, slots=64, channels=4096, states=16,
             groups=1, gated=True, dtype="bf16"),
        # a full decode batch: the state's traffic
        dict(name="scan_step_512", op="scan_step", batch=512, tokens=1, slots=1024, channels=4096,
             states=16, groups=1, gated=True, dtype="bf16"),
        # one long prompt: few rows, a long chain
        dict(name="scan_long", op="scan", seqs=1, total=8192, slots=8, channels=4096, states=16,
             groups=1, gated=True, dtype="bf16"),
        # sixteen prompts of unequal lengths, packed
        dict(name="scan_packed", op="scan", seqs=16, total=32768, slots=64, channels=2048, states=16,
             groups=1, gated=True, dtype="fp16"),
        # grouped B and C, a wide state, odd sizes, 32-bit activations
        dict(name="scan_odd", op="scan", seqs=3, total=1999, slots=4, channels=1002, states=64,
             groups=3, gated=False, dtype="fp32"),
        # one session's next token
        dict(name="sample_1", op="sample", rows=1, vocab=65536, mode="top_p", dtype="bf16"),
        # a decode batch as a runner hands it over (32-bit logits), every session with its own settings
        dict(name="sample_256", op="sample", rows=256, vocab=65536, mode="mixed", dtype="fp32"),
        # a large vocabulary of an odd size, short candidate lists
        dict(name="sample_wide", op="sample", rows=96, vocab=131071, mode="top_k", dtype="fp16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["conv_step", "conv", "scan_step", "scan", "scan", "sample", "sample"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "sample":
        rows, vocab = _log(rng, 1, 256), _log(rng, 1000, 131072)
        return dict(op=op, rows=rows, vocab=vocab, mode=rng.choice(["top_k", "top_p", "plain", "mixed"]),
                    dtype=dtype)
    channels = _log(rng, 64, 4096)
    if rng.random() < 0.6:
        channels = max(64, channels // 64 * 64)
    if op in ("conv_step", "scan_step"):
        batch = _log(rng, 1, 512)
        c = dict(op=op, batch=batch, tokens=rng.choice([1, 1, 1, 2, 5]), slots=batch + _log(rng, 1, 300),
                 channels=channels)
    else:
        total = _log(rng, 16, 32768)
        seqs = min(_log(rng, 1, 64), total)
        c = dict(op=op, seqs=seqs, total=total, slots=seqs + 3, channels=channels)
    if op in ("conv_step", "conv"):
        return dict(c, width=rng.choice([2, 3, 4, 4]), silu=rng.random() < 0.7, bias=rng.random() < 0.7,
                    dtype=dtype)
    states = rng.choice([8, 16, 16, 16, 32, 64, 128])
    if op == "scan_step":
        while c["batch"] * channels * states > 512 * 4096 * 16:
            c["batch"] = (c["batch"] + 1) // 2
    else:
        while c["total"] * channels * states > 32768 * 2048 * 16:
            c["total"] = (c["total"] + 1) // 2
        c["seqs"] = min(c["seqs"], c["total"])
    groups = rng.choice([g for g in (1, 1, 2, 4) if channels % g == 0])
    return dict(c, states=states, groups=groups, gated=rng.random() < 0.7, dtype=dtype)


def _lengths(case):
    """Lengths of the packed prompts: they sum to `total`; one is empty and one a single token where there is room."""
    n, total = case["seqs"], case["total"]
    rng = random.Random(1000003 * total + n)
    if n == 1:
        return [total]
    part = [rng.uniform(0.2, 1.8) for _ in range(n)]
    got = [int(total * p / sum(part)) for p in part]
    if n >= 5 and total >= 64:
        got[1], got[3] = 0, 1
    got[-1] += total - sum(got)
    if got[-1] < 0:
        got[0] += got[-1]
        got[-1] = 0
    return got


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def randn(*s):
        return torch.randn(*s, generator=g, device=dev)

    def rand(*s):
        return torch.rand(*s, generator=g, device=dev)

    dt = DTYPES[case["dtype"]]
    s = dict(case=case, op=case["op"])
    if case["op"] == "sample":
        b, v = case["rows"], case["vocab"]
        # a broad bulk of unlikely tokens, some likely ones, and a tenth of the rows under a mask
        x = 2.5 * randn(b, v)
        x.scatter_add_(1, torch.randint(0, v, (b, 24), generator=g, device=dev), 5.0 + 5.0 * rand(b, 24))
        masked = (rand(b, 1) < 0.1) & (rand(b, v) < 0.5)
        s["logits"] = x.masked_fill_(masked, -math.inf).to(dt)
        s["u"] = rand(b)
        on = torch.ones(b, device=dev)
        s["temperature"] = 0.6 + 0.6 * rand(b)
        s["top_k"] = torch.zeros(b, dtype=torch.int32, device=dev)
        s["top_p"], s["min_p"] = on, 0 * on
        k = (5 + 95 * rand(b)).to(torch.int32)
        p = 0.8 + 0.19 * rand(b)
        if case["mode"] == "top_k":
            s["top_k"], s["top_p"] = k, p
        elif case["mode"] == "top_p":
            s["top_p"] = p
        elif case["mode"] == "mixed":
            kind = torch.randint(0, 6, (b,), generator=g, device=dev)
            s["temperature"] = torch.where(kind == 0, 0.0, s["temperature"])  # greedy
            s["top_k"] = torch.where((kind == 1) | (kind == 2), k, 0).to(torch.int32)
            s["top_p"] = torch.where((kind == 2) | (kind == 3), p, on)
            s["min_p"] = torch.where(kind == 4, 0.02 + 0.08 * rand(b), 0 * on)
        return s

    d = case["channels"]
    if case["op"] in ("conv_step", "scan_step"):
        n, lead = case["batch"], (case["batch"], case["tokens"])
    else:
        n, lead = case["seqs"], (1, case["total"])
        ends = torch.tensor(_lengths(case)).cumsum(0)
        s["cu_seqlens"] = torch.cat([torch.zeros(1, dtype=torch.int64), ends]).to(dev)
        s["lengths"] = _lengths(case)
    rows = case["slots"] + 1  # the bank keeps row 0 for padding
    s["ids"] = (1 + torch.randperm(case["slots"], generator=g, device=dev)[:n]).to(torch.int32)
    s["layer"] = 1
    if case["op"] in ("conv_step", "conv"):
        # the convolution's input is one half of a projection's output
        s["x"] = randn(*lead, 2 * d).to(dt)[..., :d]
        s["weight"] = (randn(d, case["width"]) / math.sqrt(case["width"])).to(dt)
        s["bias"] = (0.1 * randn(d)).to(dt) if case["bias"] else None
        s["bank"] = randn(2, rows, case["width"] - 1, d).to(dt)
        return s
    m, groups = case["states"], case["groups"]
    s["x"] = torch.nn.functional.silu(randn(*lead, d)).to(dt)
    s["z"] = randn(*lead, 2 * d).to(dt)[..., d:] if case["gated"] else None
    rank = max(1, d // 16)
    proj = randn(*lead, rank + 2 * groups * m).to(dt)  # the projection that holds dt's factor, B and C
    s["B"] = proj[..., rank:rank + groups * m].unflatten(-1, (groups, m))
    s["C"] = proj[..., rank + groups * m:].unflatten(-1, (groups, m))
    s["dt"] = (0.5 * randn(*lead, d)).to(dt)
    step = torch.exp(math.log(1e-3) + rand(d) * math.log(100.0))  # typical steps from 0.001 to 0.1
    s["dt_bias"] = step + torch.log(-torch.expm1(-step))
    s["A"] = -torch.arange(1, m + 1, device=dev).float() * torch.exp(0.1 * randn(d, m))
    s["D"] = 1 + 0.1 * randn(d)
    s["bank"] = 0.3 * randn(2, rows, d, m)
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------

def _starts(s):
    """(index of the first token of every non-empty prompt, which prompt each token belongs to, its place in it)."""
    cu = s["cu_seqlens"]
    seq = torch.repeat_interleave(torch.arange(len(cu) - 1, device=cu.device), cu[1:] - cu[:-1],
                                  output_size=s["case"]["total"])
    return cu[:-1], seq, torch.arange(len(seq), device=cu.device) - cu[seq]


def _plain_conv(s):
    x, w = s["x"].float(), s["weight"].float()
    width, ids, layer = w.shape[1], s["ids"].long(), s["bank"][s["layer"]]
    old = layer[ids].float()  # [n, width - 1, D], the oldest first
    if s["op"] == "conv_step":
        full = torch.cat([old, x], 1)
        y = sum(full[:, j:j + x.shape[1]] * w[:, j] for j in range(width))
        new = full[:, -(width - 1):]
    else:
        x = x[0]
        _, seq, place = _starts(s)
        at = torch.arange(len(seq), device=x.device)
        y = 0
        for j in range(width):
            back = width - 1 - j
            prev = torch.where((place >= back)[:, None], x[(at - back).clamp(min=0)],
                               old[seq, (place + j).clamp(max=width - 2)])
            y = y + prev * w[:, j]
        y = y[None]
        cu = s["cu_seqlens"]
        length, end = (cu[1:] - cu[:-1])[:, None], cu[1:, None]
        back = torch.arange(width - 1, 0, -1, device=x.device)[None]  # how far before the end
        from_x = x[(end - back).clamp(min=0, max=len(seq) - 1)]
        from_old = old.gather(1, (width - 1 + length - back).clamp(max=width - 2)[..., None].expand_as(old))
        new = torch.where((length >= back)[..., None], from_x, from_old)
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if s["case"]["silu"]:
        y = y * torch.sigmoid(y)
    layer[ids] = new.to(layer.dtype)
    return y.to(s["x"].dtype), layer


def _softplus(x):
    return torch.clamp(x, min=0) + torch.log1p(torch.exp(-x.abs()))


def _plain_scan(s):
    x, ids, layer = s["x"].float(), s["ids"].long(), s["bank"][s["layer"]]
    d, groups = x.shape[-1], s["case"]["groups"]
    step = _softplus(s["dt"].float() + s["dt_bias"])
    b, c = (t.float().repeat_interleave(d // groups, -2) for t in (s["B"], s["C"]))  # [.., D, N]
    if s["op"] == "scan_step":
        h, y = layer[ids], []
        for t in range(x.shape[1]):
            h = torch.exp(step[:, t, :, None] * s["A"]) * h + (step[:, t] * x[:, t])[..., None] * b[:, t]
            y.append((h * c[:, t]).sum(-1))
        y, new = torch.stack(y, 1), h
    else:
        cu = s["cu_seqlens"]
        start, seq, place = _starts(s)
        decay = torch.exp(step[0, ..., None] * s["A"])  # [L, D, N]
        h = (step[0] * x[0])[..., None] * b[0]
        old = layer[ids]
        full = cu[1:] > cu[:-1]
        h[start[full]] += decay[start[full]] * old[full]
        decay[start[full]] = 0
        for k in range(max(s["lengths"]).bit_length()):  # h_t over 2^k tokens, then twice as many
            far = 1 << k
            if far >= len(h):
                break
            h[far:] += decay[far:] * h[:-far]
            decay[far:] *= decay[:-far].clone()
        y = (h * c[0]).sum(-1)[None]
        new = torch.where(full[:, None, None], h[(cu[1:] - 1).clamp(min=0)], old)
    y = y + s["D"] * x
    if s["z"] is not None:
        z = s["z"].float()
        y = y * (z * torch.sigmoid(z))
    layer[ids] = new
    return y.to(s["x"].dtype), layer


def _plain_sample(s):
    x = s["logits"]
    greedy = (s["temperature"] == 0)[:, None]
    t = torch.where(greedy, 1.0, s["temperature"][:, None]).double()
    k = torch.where(greedy[:, 0] | (s["top_k"] <= 0), torch.where(greedy[:, 0], 1, x.shape[1]), s["top_k"])
    w = torch.exp((x.double() - x.amax(1, keepdim=True).double()) / t)  # relative to the likeliest
    order = torch.sort(x, dim=1, descending=True, stable=True).indices  # ties: the lowest index first
    ws = w.gather(1, order)
    ws = ws * (torch.arange(x.shape[1], device=x.device) < k[:, None])
    before = torch.cumsum(ws, 1)
    total = before[:, -1:]
    before = torch.cat([torch.zeros_like(total), before[:, :-1]], 1)
    p = s["top_p"][:, None].double()
    keep = ((p >= 1) | (before < p * total)) & (ws > 0) & (ws >= s["min_p"][:, None].double())
    ws = ws * keep
    mass = torch.zeros_like(w).scatter_(1, order, ws)
    c = torch.cumsum(mass, 1)
    hit = (c > s["u"][:, None].double() * c[:, -1:]) & (mass > 0)
    token = hit.int().argmax(1)
    return token, torch.log(mass.gather(1, token[:, None]) / c[:, -1:])[:, 0].float()


def run(state):
    s = state
    if not own:
        return {"sample": _plain_sample, "scan": _plain_scan, "scan_step": _plain_scan, "conv": _plain_conv,
                "conv_step": _plain_conv}[s["op"]](s)
    import wkvm_b200 as wk
    if s["op"] == "sample":
        return wk.sample_tokens(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"],
                                top_p=s["top_p"], min_p=s["min_p"])
    bank, layer = s["bank"], s["layer"]
    if s["op"] in ("conv_step", "conv"):
        act = "silu" if s["case"]["silu"] else None
        if s["op"] == "conv_step":
            o = wk.short_conv_decode_slots(s["x"], s["weight"], bank, layer, s["ids"], bias=s["bias"],
                                           activation=act)
        else:
            o = wk.short_conv_prefill_slots(s["x"], s["weight"], bank, layer, s["ids"], bias=s["bias"],
                                            activation=act, cu_seqlens=s["cu_seqlens"])
        return o, bank[layer]
    args = (s["x"], s["dt"], s["A"], s["B"], s["C"], bank, layer, s["ids"])
    more = dict(D=s["D"], z=s["z"], dt_bias=s["dt_bias"], dt_softplus=True)
    if s["op"] == "scan_step":
        return wk.selective_scan_decode_slots(*args, **more), bank[layer]
    return wk.selective_scan_prefill_slots(*args, cu_seqlens=s["cu_seqlens"], **more), bank[layer]


# ---------------------------------------------------------------------------
# what a pass cannot do without, and the definitions in 64 bits
# ---------------------------------------------------------------------------

def work(case):
    es = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        # a maximum, a scaled difference, an exponential and a sum for every logit
        return {"bytes": n * es + case["rows"] * 32, "flops": 4 * n}
    d = case["channels"]
    if case["op"] in ("conv_step", "scan_step"):
        rows, tokens = case["batch"], case["batch"] * case["tokens"]
    else:
        rows, tokens = case["seqs"], case["total"]
    if case["op"] in ("conv_step", "conv"):
        w = case["width"]
        return {"bytes": es * d * (2 * tokens + 2 * rows * (w - 1) + w + case["bias"]),
                "flops": tokens * d * (2 * w + (5 if case["silu"] else 0))}
    n, g = case["states"], case["groups"]
    streams = 4 if case["gated"] else 3  # x, dt, z in, the output out
    return {"bytes": es * tokens * (streams * d + 2 * g * n) + 4 * (2 * rows * d * n + d * n + 2 * d),
            "flops": tokens * d * (7 * n + 12)}


def _exact_sample(s):
    import numpy as np
    x = s["logits"].double().cpu().numpy()
    temp, top_k, top_p, min_p, u = (s[n].double().cpu().numpy() for n in
                                    ("temperature", "top_k", "top_p", "min_p", "u"))
    tokens, logp = np.empty(len(x), np.int64), np.empty(len(x))
    for i, row in enumerate(x):
        k = 1 if temp[i] == 0 else int(top_k[i]) if top_k[i] > 0 else len(row)
        top = np.argsort(-row, kind="stable")[:k]
        w = np.exp((row[top] - row[top[0]]) / (temp[i] or 1.0))
        if top_p[i] < 1:
            size = 1 + np.searchsorted(np.cumsum(w), top_p[i] * w.sum(), side="left")
            top, w = top[:size], w[:size]
        top, w = top[(w >= min_p[i]) & (w > 0)], w[(w >= min_p[i]) & (w > 0)]
        by_id = np.argsort(top)
        top, w = top[by_id], w[by_id]
        c = np.cumsum(w)
        j = min(np.searchsorted(c, u[i] * c[-1], side="right"), len(w) - 1)
        tokens[i], logp[i] = top[j], np.log(w[j] / c[-1])
    return torch.from_numpy(tokens), torch.from_numpy(logp)


def _exact_conv(s):
    layer = s["bank"][s["layer"]].double()
    x, w = s["x"].double(), s["weight"].double()
    parts = x.unbind(0) if s["op"] == "conv_step" else x[0].split(s["lengths"])
    y = []
    for i, part in zip(s["ids"].tolist(), parts):
        line = torch.cat([layer[i], part])
        y.append(torch.einsum("tdw,dw->td", line.unfold(0, w.shape[1], 1), w) if len(part) else part)
        layer[i] = line[len(part):]
    y = torch.stack(y) if s["op"] == "conv_step" else torch.cat(y)[None]
    if s["bias"] is not None:
        y = y + s["bias"].double()
    return torch.nn.functional.silu(y) if s["case"]["silu"] else y, layer


def _exact_scan(s):
    layer, ids = s["bank"][s["layer"]].double(), s["ids"].long()
    names = [n for n in ("x", "dt", "B", "C", "z") if s[n] is not None]
    if s["op"] == "scan_step":
        live = torch.ones(s["x"].shape[:2], dtype=torch.bool, device=layer.device)
        v = {n: s[n].double() for n in names}
    else:  # the prompts side by side, padded behind their ends
        most = max(s["lengths"])
        live = torch.arange(most)[None] < torch.tensor(s["lengths"])[:, None]
        live = live.to(layer.device)
        v = {}
        for n in names:
            t = s[n][0]
            v[n] = torch.zeros(*live.shape, *t.shape[1:], dtype=torch.float64, device=t.device)
            v[n][live] = t.double()
    a, rep = s["A"].double(), s["x"].shape[-1] // s["case"]["groups"]
    h = layer[ids]
    delta = torch.nn.functional.softplus(v["dt"] + s["dt_bias"].double(), threshold=60.0)
    y = torch.zeros_like(v["x"])
    for t in range(live.shape[1]):
        b, c = (v[n][:, t].repeat_interleave(rep, 1) for n in ("B", "C"))
        new = torch.exp(delta[:, t, :, None] * a) * h + (delta[:, t] * v["x"][:, t])[..., None] * b
        h = torch.where(live[:, t, None, None], new, h)
        y[:, t] = torch.einsum("rdn,rdn->rd", h, c) + s["D"].double() * v["x"][:, t]
    if s["z"] is not None:
        y = y * torch.nn.functional.silu(v["z"])
    layer[ids] = h
    return y if s["op"] == "scan_step" else y[live][None], layer


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(s)
    return _exact_conv(s) if case["op"] in ("conv_step", "conv") else _exact_scan(s)
