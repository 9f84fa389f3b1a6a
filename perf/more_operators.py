"""The operators that training the whole model needs beside its blocks' own, as cases that can be timed and checked.

* ``embedding``      rows of the embedding by token, scaled, and the weight's gradient
* ``scan``           the gated linear recurrence h_t = a_t h_{t-1} + u_t and its gradients
* ``orthogonalize``  a matrix, or a stack of them, brought near its closest semi-orthogonal one by Newton-Schulz steps
* ``muon``           one Muon step over a model's matrices: momentum, orthogonalization, update

With ``own`` the package's calls are made; without it the same is computed in elementary torch operations in
32 bits. ``exact`` restates everything in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

LR, MOMENTUM, DECAY, EPS, STEPS = 0.02, 0.95, 0.1, 1e-7, 5
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
PAD = 0
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ======================================================================================
# the cases
# ======================================================================================

def listed():
    return [
        # the next token of 64 generated streams
        dict(name="embedding_decode", op="embedding", B=64, T=1, V=16_384, D=1024, dtype="bf16", out="bf16", scaled=False,
             train=False, pad=False),
        # a training step of the promoted model: fp32 weights, text whose frequent words come often
        dict(name="embedding_train", op="embedding", B=4, T=2048, V=16_384, D=1024, dtype="fp32", out="fp32",
             scaled=False, train=True, pad=False),
        # more text and a large vocabulary, weights in bf16
        dict(name="embedding_train_large", op="embedding", B=8, T=4096, V=131_072, D=1024, dtype="bf16", out="bf16",
             scaled=False, train=True, pad=False),
        # short texts padded to one length, odd width and vocabulary, rows scaled by the width's root, bf16 activations
        dict(name="embedding_train_ragged", op="embedding", B=3, T=333, V=32_001, D=714, dtype="fp32", out="bf16",
             scaled=True, train=True, pad=True),
        # one token of 64 streams, the state carried
        dict(name="scan_step", op="scan", B=64, T=1, C=1024, gate="fp32", drive="fp32", per_token=False, state=True,
             train=False),
        # the softpatch's recurrence in a training step: one gate a token, 64 channels
        dict(name="scan_softpatch", op="scan", B=4, T=2048, C=64, gate="fp32", drive="fp32", per_token=True, state=False,
             train=True),
        # a batch of sequences, a gate for each channel
        dict(name="scan_train", op="scan", B=8, T=2048, C=1024, gate="fp32", drive="fp32", per_token=False, state=True,
             train=True),
        # one long document, bf16 activations
        dict(name="scan_long", op="scan", B=1, T=65_536, C=1024, gate="fp32", drive="bf16", per_token=False, state=False,
             train=True),
        # one matrix of a small model
        dict(name="orthogonalize_small", op="orthogonalize", N=1, M=256, K=632, dtype="fp32"),
        # the projections of all Field blocks, stacked
        dict(name="orthogonalize_stack", op="orthogonalize", N=18, M=1536, K=1024, dtype="bf16"),
        # a small model with widths that are no multiple of a tile, weights in bf16
        dict(name="muon_ragged", op="muon", blocks=7, dim=714, hidden=1531, dtype="bf16", nesterov=False),
        # all matrices of 22 blocks
        dict(name="muon_model", op="muon", blocks=22, dim=1024, hidden=2528, dtype="fp32", nesterov=True),
    ]


def _log_uniform(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["embedding", "embedding", "scan", "scan", "scan", "orthogonalize", "muon"])
    if op == "embedding":
        b = rng.choice([1, 2, 3, 4, 8])
        return dict(op=op, B=b, T=_log_uniform(rng, 1, 32_768 // b), V=_log_uniform(rng, 500, 131_072),
                    D=_log_uniform(rng, 24, 1024), dtype=rng.choice(["fp32", "bf16"]), out=rng.choice(["fp32", "bf16"]),
                    scaled=rng.random() < 0.5, train=rng.random() < 0.7, pad=rng.random() < 0.3)
    if op == "scan":
        c = _log_uniform(rng, 1, 2048)
        t = _log_uniform(rng, 1, 65_536)
        b = _log_uniform(rng, 1, max(1, min(64, (1 << 26) // (c * t))))
        return dict(op=op, B=b, T=max(1, min(t, (1 << 26) // (b * c))), C=c, gate=rng.choice(["fp32", "fp32", "bf16"]),
                    drive=rng.choice(["fp32", "bf16"]), per_token=rng.random() < 0.4, state=rng.random() < 0.5,
                    train=rng.random() < 0.6)
    if op == "orthogonalize":
        m, k = _log_uniform(rng, 8, 2048), _log_uniform(rng, 8, 2048)
        return dict(op=op, N=_log_uniform(rng, 1, max(1, min(18, (1 << 24) // (m * k)))), M=m, K=k,
                    dtype=rng.choice(["fp32", "bf16"]))
    return dict(op=op, blocks=rng.randint(1, 12), dim=2 * _log_uniform(rng, 24, 512), hidden=_log_uniform(rng, 16, 2528),
                dtype=rng.choice(["fp32", "bf16"]), nesterov=rng.random() < 0.5)


def _matrices(case):
    """Shapes of the matrices of ``blocks`` Field blocks."""
    d, h = case["dim"], case["hidden"]
    return [(3 * (d // 2), d), (d, 2 * d), (d, d), (2 * h, d), (d, h)] * case["blocks"]


def _size(name):
    return 2 if name == "bf16" else 4


def _products(m, k):
    """Operations of the Newton-Schulz steps of one matrix through its Gram matrix: that and the last product with the
    matrix once, between them four products of symmetric matrices a step (three less in all), half of whose results are
    computed."""
    m, k = min(m, k), max(m, k)
    return m * m * k + 2 * m * m * k + (4 * STEPS - 3) * m ** 3


def work(case):
    if case["op"] == "embedding":
        n, d = case["B"] * case["T"], case["D"]
        rows = 8 * n + n * d * (_size(case["dtype"]) + _size(case["out"]))
        grad = n * d * _size(case["out"]) + case["V"] * d * _size(case["dtype"])
        return {"bytes": rows + case["train"] * grad, "flops": n * d * (1 + case["train"])}
    if case["op"] == "scan":
        n, gates = case["B"] * case["T"] * case["C"], case["B"] * case["T"] * (1 if case["per_token"] else case["C"])
        u, a = n * _size(case["drive"]), gates * _size(case["gate"])
        state = 4 * case["B"] * case["C"] * case["state"]
        return {"bytes": a + 2 * u + 2 * state + case["train"] * (2 * a + 3 * u + 2 * state),
                "flops": n * (2 + 5 * case["train"])}
    if case["op"] == "orthogonalize":
        n = case["N"] * case["M"] * case["K"]
        return {"bytes": 2 * n * _size(case["dtype"]), "flops": case["N"] * _products(case["M"], case["K"])}
    shapes = _matrices(case)
    n = sum(m * k for m, k in shapes)
    return {"bytes": n * (3 * _size(case["dtype"]) + 8), "flops": sum(_products(m, k) for m, k in shapes)}


# ======================================================================================
# what a program has in hand
# ======================================================================================

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    def rand(*shape):
        return torch.rand(*shape, device="cuda", generator=gen)

    state = dict(case=case)
    if case["op"] == "embedding":
        b, t, v, d = case["B"], case["T"], case["V"], case["D"]
        # words by their frequency: the r-th most frequent comes 1 / r as often as the first
        rank = torch.exp(rand(b, t) * math.log(v)).long().clamp_(1, v) - 1
        tokens = torch.randperm(v, device="cuda", generator=gen)[rank]
        if case["pad"]:  # every text but the first ends early
            ends = (rand(b, 1) * t).long()
            ends[0] = t
            tokens[torch.arange(t, device="cuda") >= ends] = PAD
        state.update(tokens=tokens, weight=(0.02 * randn(v, d)).to(DTYPES[case["dtype"]]),
                     scale=math.sqrt(d) if case["scaled"] else 1.0,
                     grad=(randn(b, t, d) * 1e-3).to(DTYPES[case["out"]]))
    elif case["op"] == "scan":
        b, t, c = case["B"], case["T"], case["C"]
        # gates of memories from a few steps to some thousands, closed at the borders of packed texts
        gate = torch.sigmoid(2.0 + 2.0 * randn(b, t, *([] if case["per_token"] else [c])))
        gate = 1.0 - (1.0 - gate) * (1.0 if case["per_token"] else torch.exp(-4.0 * rand(c)))
        gate[rand(b, t) < 1e-3] = 0.0
        state.update(gate=gate.to(DTYPES[case["gate"]]), drive=randn(b, t, c).mul_(0.3).to(DTYPES[case["drive"]]),
                     state=randn(b, c) if case["state"] else None,
                     grads=[randn(b, t, c).mul_(1e-2).to(DTYPES[case["drive"]]), 1e-2 * randn(b, c)])
    elif case["op"] == "orthogonalize":
        state["matrix"] = _gradient(gen, case["N"], case["M"], case["K"]).to(DTYPES[case["dtype"]])
    else:
        shapes, dtype = _matrices(case), DTYPES[case["dtype"]]
        state["params"], state["param"] = _parts([randn(m, k) / math.sqrt(k) for m, k in shapes], dtype)
        state["grads"], _ = _parts([1e-3 * _gradient(gen, 1, m, k)[0] for m, k in shapes], dtype)
        state["buffers"], state["buffer"] = _parts([1e-3 * _gradient(gen, 1, m, k)[0] for m, k in shapes], torch.float32)
    return state


def _parts(matrices, dtype):
    """The matrices as parts of one buffer, each at a multiple of 64 values, and the buffer."""
    starts, total = [], 0
    for x in matrices:
        starts.append(total)
        total += -(-x.numel() // 64) * 64
    flat = torch.zeros(total, dtype=dtype, device=matrices[0].device)
    parts = [flat[at:at + x.numel()].view(x.shape) for at, x in zip(starts, matrices)]
    for part, x in zip(parts, matrices):
        part.copy_(x)
    return parts, flat


def _gradient(gen, n, m, k):
    """Matrices with what gradients have: rows and columns of unlike sizes, a few strong directions."""
    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    x = randn(n, m, k) * torch.exp(0.5 * randn(n, m, 1)) * torch.exp(0.5 * randn(n, 1, k))
    return x + 0.5 * torch.matmul(randn(n, m, 4), randn(n, 4, k))


# ======================================================================================
# one pass
# ======================================================================================

def run(state):
    return {"embedding": _run_embedding, "scan": _run_scan, "orthogonalize": _run_orthogonalize,
            "muon": _run_muon}[state["case"]["op"]](state)


def _run_embedding(state):
    c, tokens, weight, scale = state["case"], state["tokens"], state["weight"], state["scale"]
    pad, out = (PAD if c["pad"] else None), DTYPES[c["out"]]
    if own:
        import fields_lm_amd as fl

        if not c["train"]:
            return {"rows": fl.embedding(tokens, weight, scale=scale, padding_idx=pad, dtype=out)}
        weight = weight.detach().requires_grad_()
        rows = fl.embedding(tokens, weight, scale=scale, padding_idx=pad, dtype=out)
        grad, = torch.autograd.grad(rows, weight, state["grad"])
        return {"rows": rows.detach(), "grad": grad}
    got = {"rows": (weight[tokens].float() * scale).to(out)}
    if c["train"]:
        g = state["grad"].float() * scale
        if pad is not None:
            g = torch.where((tokens == pad)[..., None], 0.0, g)
        grad = torch.zeros(weight.shape, device=weight.device)
        grad.index_add_(0, tokens.reshape(-1), g.reshape(-1, g.shape[-1]))
        got["grad"] = grad.to(weight.dtype)
    return got


def _run_scan(state):
    c, gate, drive, first = state["case"], state["gate"], state["drive"], state["state"]
    if own:
        import fields_lm_amd as fl

        if not c["train"]:
            if first is None:
                return {"out": fl.gated_scan(gate, drive)}
            out, last = fl.gated_scan(gate, drive, first, return_state=True)
            return {"out": out, "state": last}
        inputs = [t.detach().requires_grad_() for t in (gate, drive, first) if t is not None]
        out, last = fl.gated_scan(*inputs, return_state=True)
        grads = torch.autograd.grad([out, last], inputs, state["grads"])
        return {"out": out.detach(), "state": last.detach(),
                **dict(zip(("grad_gate", "grad_drive", "grad_state"), grads))}
    a, u = gate.float(), drive.float()
    if c["per_token"]:
        a = a[..., None]
    h = _plain_scan(a, u, first)
    got = {"out": h.to(drive.dtype)}
    if c["train"] or first is not None:
        got["state"] = h[:, -1].clone()
    if c["train"]:
        g, g_last = state["grads"][0].float(), state["grads"][1]
        # the same recurrence from the end: g_t = dh_t + a_{t+1} g_{t+1}
        after = torch.cat((torch.ones_like(a[:, :1]), a[:, 1:].flip(1)), 1)
        g = _plain_scan(after, g.flip(1), g_last).flip(1)
        before = torch.cat(((torch.zeros_like(h[:, 0]) if first is None else first)[:, None], h[:, :-1]), 1)
        da = g * before
        got["grad_gate"] = (da.sum(-1) if c["per_token"] else da).to(gate.dtype)
        got["grad_drive"] = g.to(drive.dtype)
        if first is not None:
            got["grad_state"] = a[:, 0] * g[:, 0]
    return got


def _run_orthogonalize(state):
    x = state["matrix"]
    if own:
        import fields_lm_amd as fl

        return {"matrix": fl.orthogonalize(x, steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)}
    return {"matrix": torch.stack([_plain_orthogonalize(m.float()) for m in x]).to(x.dtype)}


def _run_muon(state):
    c, params, grads, buffers = state["case"], state["params"], state["grads"], state["buffers"]
    if own:
        import fields_lm_amd as fl

        fl.muon_step(params, grads, buffers, lr=LR, momentum=MOMENTUM, nesterov=c["nesterov"], weight_decay=DECAY,
                     steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)
    else:
        for p, g, buf in zip(params, grads, buffers):
            g = g.float()
            buf.mul_(MOMENTUM).add_(g * (1 - MOMENTUM))
            update = g * (1 - MOMENTUM) + buf * MOMENTUM if c["nesterov"] else buf
            update = _plain_orthogonalize(update) * math.sqrt(max(1.0, p.shape[0] / p.shape[1]))
            p.copy_(p.float() * (1 - LR * DECAY) - LR * update)
    return {"param": state["param"], "buffer": state["buffer"]}


# ======================================================================================
# the plain forms
# ======================================================================================

def _plain_scan(a, u, first):
    """All states by doubling: after k rounds a step holds what the last 2^k steps make of it."""
    p, s = a, u
    if first is not None:
        s = torch.cat(((a[:, 0] * first + u[:, 0])[:, None], u[:, 1:]), 1)
    reach = 1
    while reach < u.shape[1]:
        s = torch.cat((s[:, :reach], p[:, reach:] * s[:, :-reach] + s[:, reach:]), 1)
        p = torch.cat((p[:, :reach], p[:, reach:] * p[:, :-reach]), 1)
        reach *= 2
    return s


def _plain_orthogonalize(g):
    a, b, c = COEFFICIENTS
    tall = g.shape[0] > g.shape[1]
    x = g.t().contiguous() if tall else g
    x = x / (torch.sqrt(x.double().square().sum()).float() + EPS)
    for _ in range(STEPS):
        gram = x @ x.t()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.t() if tall else x


# ======================================================================================
# 64 bits
# ======================================================================================

def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "embedding":
        return _exact_embedding(case, state)
    if case["op"] == "scan":
        return _exact_scan(case, state)
    if case["op"] == "orthogonalize":
        return {"matrix": torch.stack([_exact_polar(x.double()) for x in state["matrix"]])}
    params, buffers = [], []
    for p, g, buf in zip(state["params"], state["grads"], state["buffers"]):
        g, buf = g.double(), buf.double()
        buf = buf + (1 - MOMENTUM) * (g - buf)
        step = g + MOMENTUM * (buf - g) if case["nesterov"] else buf
        shape = max(1.0, p.shape[0] / p.shape[1]) ** 0.5
        params.append(p.double() - LR * DECAY * p.double() - LR * shape * _exact_polar(step))
        buffers.append(buf)
    return {"param": _parts(params, torch.float64)[1], "buffer": _parts(buffers, torch.float64)[1]}


def _exact_embedding(case, state):
    tokens, weight = state["tokens"], state["weight"].double()
    out = {"rows": torch.index_select(weight, 0, tokens.view(-1)).view(*tokens.shape, -1) * state["scale"]}
    if case["train"]:
        flat = tokens.view(-1)
        order = torch.argsort(flat)
        if case["pad"]:
            order = order[flat[order] != PAD]
        sums = torch.zeros_like(weight)
        sums.index_put_((flat[order],), state["grad"].view(flat.numel(), -1)[order].double(), accumulate=True)
        out["grad"] = sums * state["scale"]
    return out


def _exact_scan(case, state):
    a, u = state["gate"].double(), state["drive"].double()
    a = a[..., None] if case["per_token"] else a
    t = u.shape[1]
    start = torch.zeros_like(u[:, 0]) if state["state"] is None else state["state"].double()
    h, now = torch.empty_like(u), start
    for i in range(t):
        now = torch.addcmul(u[:, i], a[:, i], now)
        h[:, i] = now
    out = {"out": h}
    if case["train"] or case["state"]:
        out["state"] = now
    if case["train"]:
        g = state["grads"][0].double()
        carry = state["grads"][1].double()
        for i in range(t - 1, -1, -1):
            carry = carry + g[:, i]
            g[:, i] = carry
            carry = a[:, i] * carry
        da = torch.empty_like(u)
        da[:, 0] = g[:, 0] * start
        torch.mul(g[:, 1:], h[:, :-1], out=da[:, 1:])
        out["grad_gate"] = da.sum(-1) if case["per_token"] else da
        out["grad_drive"] = g
        if case["state"]:
            out["grad_state"] = carry
    return out


def _exact_polar(g):
    a, b, c = COEFFICIENTS
    x = (g if g.shape[0] <= g.shape[1] else g.mT).contiguous()
    x = x / (torch.linalg.matrix_norm(x) + EPS)
    for _ in range(STEPS):
        gram = torch.mm(x, x.mT.contiguous())
        x = torch.addmm(x, torch.addmm(gram, gram, gram, beta=b, alpha=c), x, beta=a)
    return x if g.shape[0] <= g.shape[1] else x.mT.contiguous()
