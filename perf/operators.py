"""The operators of a training step and of scoring around the blocks, as cases that can be timed and checked.

* ``logprobs``  log probabilities of given tokens with entropy and top alternatives, and their gradient
* ``norm``      the 2-norm of all gradients and the scale that clips it
* ``adamw``     one AdamW step over many tensors, states in 32 or 8 bits
* ``update``    the norm, then the clipped AdamW step, as a training loop calls them

With ``own`` the package's calls are made; without it the same is computed in elementary torch operations in
32 bits. ``exact`` restates everything in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

LR, BETA1, BETA2, EPS, DECAY, MAX_NORM, STEPS = 1e-3, 0.9, 0.95, 1e-8, 0.1, 1.0, 41
IGNORE = -100
BLOCK, TOP_CODE, SMALLEST = 256, 448.0, 2.0 ** -9  # 8-bit states: values per scale; e4m3's largest and smallest
TINY = 1e-30  # a block whose largest value is below this is held as zeros
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ======================================================================================
# the cases
# ======================================================================================

def listed():
    return [
        # a generation loop of 64 streams returns each sampled token's log probability with five alternatives
        dict(name="logprobs_decode", op="logprobs", B=64, T=1, V=16_384, dtype="bf16", k=5, entropy=True, train=False,
             temperature=1.0, shift=False),
        # one stream, a large vocabulary, twenty alternatives
        dict(name="logprobs_one_stream", op="logprobs", B=1, T=1, V=131_072, dtype="fp32", k=20, entropy=True,
             train=False, temperature=0.8, shift=False),
        # scoring a batch of texts: every token given the ones before it, the logits of all positions but the
        # last read in place
        dict(name="logprobs_score", op="logprobs", B=4, T=2048, V=16_384, dtype="bf16", k=0, entropy=False, train=False,
             temperature=1.0, shift=True),
        # the same with the top twenty of every position, as an evaluation or a distillation set stores them
        dict(name="logprobs_score_top", op="logprobs", B=4, T=2048, V=16_384, dtype="bf16", k=20, entropy=True,
             train=False, temperature=1.0, shift=False),
        # the loss of a training step and its gradient, a part of the rows padding
        dict(name="logprobs_train", op="logprobs", B=4, T=2048, V=16_384, dtype="bf16", k=0, entropy=True, train=True,
             temperature=1.0, shift=False),
        # fp32 logits of an odd vocabulary, short texts, gradients through the alternatives too
        dict(name="logprobs_train_ragged", op="logprobs", B=3, T=333, V=32_001, dtype="fp32", k=8, entropy=True,
             train=True, temperature=0.7, shift=False),
        # one Field block of width 1,024 trained by itself
        dict(name="norm_block", op="norm", blocks=1, dim=1024, hidden=2528, vocab=0, dtype="fp32"),
        # all gradients of a model of 22 blocks and its embedding, 0.29 G values
        dict(name="norm_model", op="norm", blocks=22, dim=1024, hidden=2528, vocab=16_384, dtype="fp32"),
        # the step of a small model, where the launch counts
        dict(name="adamw_small", op="adamw", blocks=2, dim=256, hidden=632, vocab=1024, dtype="fp32", bits=32),
        # the step of that whole model, states in 8 bits
        dict(name="adamw8_model", op="adamw", blocks=22, dim=1024, hidden=2528, vocab=16_384, dtype="fp32", bits=8),
        # widths that are no multiple of a vector or of a block of 256, weights in bf16
        dict(name="adamw8_ragged", op="adamw", blocks=7, dim=714, hidden=1531, vocab=5003, dtype="bf16", bits=8),
        # clip and step of the whole model, states in 32 bits
        dict(name="update_model", op="update", blocks=22, dim=1024, hidden=2528, vocab=16_384, dtype="fp32", bits=32),
    ]


def _log_uniform(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["logprobs", "logprobs", "norm", "adamw", "adamw", "update"])
    if op == "logprobs":
        v = _log_uniform(rng, 500, 131_072)
        rows = _log_uniform(rng, 1, max(2, min(8192, 4 * 2048 * 16_384 // v)))
        b = rng.choice([1, 2, 3, 4, 8])
        train = rng.random() < 0.5
        return dict(op=op, B=min(b, rows), T=max(1, rows // b), V=v, dtype=rng.choice(["bf16", "fp32"]) if v < 65_536
                    else "bf16", k=rng.choice([0, 1, 5, 20, rng.randint(1, 64)]), entropy=rng.random() < 0.6, train=train,
                    temperature=rng.choice([1.0, 0.7, 1.3]), shift=rows // b > 1 and rng.random() < 0.3)
    case = dict(op=op, blocks=rng.randint(1, 20), dim=2 * _log_uniform(rng, 24, 512), hidden=_log_uniform(rng, 16, 2528),
                vocab=rng.choice([0, _log_uniform(rng, 100, 16_384)]), dtype=rng.choice(["fp32", "bf16"]))
    if op != "norm":
        case["bits"] = 32 if op == "update" else rng.choice([8, 32])
    return case


def _sizes(case):
    """Value counts of the tensors of ``blocks`` Field blocks and an embedding."""
    d, h = case["dim"], case["hidden"]
    block = [d // 2, d // 2, 3 * (d // 2) * d, 3 * (d // 2), 2 * d, 2 * d * d, d, d * d, d, d, 2 * h * d, h * d]
    return block * case["blocks"] + ([case["vocab"] * d, d] if case["vocab"] else [])


def work(case):
    if case["op"] == "logprobs":
        rows = case["B"] * (case["T"] - (1 if case["shift"] else 0))
        n, size = rows * case["V"], 2 if case["dtype"] == "bf16" else 4
        small = rows * (8 + 4 + 4 * case["entropy"] + 12 * case["k"])
        return {"bytes": n * size * (2 if case["train"] else 1) + small,
                "flops": n * (4 + 2 * case["entropy"] + 6 * case["train"])}
    n, size = sum(_sizes(case)), 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "norm":
        return {"bytes": n * size, "flops": 2 * n}
    state = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
    return {"bytes": int(n * (3 * size + state)), "flops": n * (16 if case["op"] == "update" else 14)}


# ======================================================================================
# what a program has in hand
# ======================================================================================

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "logprobs":
        b, t, v, k = case["B"], case["T"], case["V"], case["k"]
        logits = torch.randn(b, t, v, device="cuda", generator=gen).mul_(2.5)
        tokens = torch.randint(0, v, (b, t), device="cuda", generator=gen)
        # the given token is a likely one in most rows, as in text
        lift = torch.rand(b, t, 1, device="cuda", generator=gen) * 14
        logits.scatter_add_(-1, tokens[..., None], lift)
        logits[..., torch.randint(0, v, (max(1, v // 97),), device="cuda", generator=gen)] = float("-inf")  # banned
        logits.scatter_(-1, tokens[..., None], lift)
        logits = logits.to(dtype)
        if case["train"]:
            tokens[torch.rand(b, t, device="cuda", generator=gen) < 0.06] = IGNORE  # padding
        if case["shift"]:
            logits, tokens = logits[:, :-1], tokens[:, 1:]
        shape = tuple(tokens.shape)
        grads = [torch.randn(shape, device="cuda", generator=gen) / tokens.numel(),
                 0.1 * torch.randn(shape, device="cuda", generator=gen) / tokens.numel(),
                 0.1 * torch.randn(*shape, k, device="cuda", generator=gen) / tokens.numel()]
        return dict(case=case, logits=logits, tokens=tokens, grads=grads)
    # one buffer for all tensors of a kind, each tensor's part a multiple of the 8-bit states' block
    sizes = _sizes(case)
    padded = [-(-n // BLOCK) * BLOCK for n in sizes]
    total, at = sum(padded), 0
    starts, pads = [], []
    for n, p in zip(sizes, padded):
        starts.append(at)
        pads.extend(range(at + n, at + p))
        at += p
    pads = torch.tensor(pads, dtype=torch.int64, device="cuda")

    def values(scale, spread):
        x = torch.randn(total, device="cuda", generator=gen)
        if spread:
            x *= torch.randn(total, device="cuda", generator=gen).mul_(spread).exp_()
        x *= scale
        x[pads] = 0
        return x

    def parts(flat):
        return [flat[a:a + n] for a, n in zip(starts, sizes)]

    grad = values(3e-4, 1.0).to(dtype)
    state = dict(case=case, grad=grad, grads=parts(grad))
    if case["op"] == "norm":
        return state
    param = values(0.02, 0.0).to(dtype)
    avg, sq = values(1e-4, 1.0), values(3e-4, 1.0).square_()
    steps = torch.full((len(sizes),), STEPS, dtype=torch.int64, device="cuda")
    state.update(param=param, params=parts(param), steps=steps)
    if case["bits"] == 32:
        state.update(avg=avg, sq=sq, avgs=parts(avg), sqs=parts(sq))
    else:
        avg, avg_scale = _to8(avg, False)
        sq, sq_scale = _to8(sq.sqrt_(), True)

        def scales(flat):
            return [flat[a // BLOCK:(a + n + BLOCK - 1) // BLOCK] for a, n in zip(starts, sizes)]

        state.update(avg=avg, sq=sq, avgs=parts(avg), sqs=parts(sq), avg_scale=avg_scale, sq_scale=sq_scale,
                     avg_scales=scales(avg_scale), sq_scales=scales(sq_scale))
    return state


# ======================================================================================
# one pass
# ======================================================================================

def run(state):
    op = state["case"]["op"]
    if op == "logprobs":
        return _run_logprobs(state)
    out = {}
    scale = None
    if op in ("norm", "update"):
        if own:
            import fields_lm_amd as fl

            out["norm"], scale = fl.grad_norm(state["grads"], max_norm=MAX_NORM)
        else:
            out["norm"], scale = _plain_norm(state["grad"])
        out["scale"] = scale
    if op in ("adamw", "update"):
        eight = state["case"]["bits"] == 8
        if own:
            import fields_lm_amd as fl

            fl.adamw_step(state["params"], state["grads"], state["avgs"], state["sqs"], state["steps"], lr=LR,
                          betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY, grad_scale=scale,
                          exp_avg_scales=state.get("avg_scales"), exp_avg_sq_scales=state.get("sq_scales"))
        else:
            _plain_adamw(state, scale)
        out.update({n: state[n] for n in ("param", "avg", "sq", "steps")})
        if eight:
            out.update(avg_scale=state["avg_scale"], sq_scale=state["sq_scale"])
    return out


def _run_logprobs(state):
    c, logits, tokens = state["case"], state["logits"], state["tokens"]
    g_lp, g_ent, g_top = state["grads"]
    if not own:
        return _plain_logprobs(c, logits, tokens, g_lp, g_ent, g_top)
    import fields_lm_amd as fl

    if c["train"]:
        logits = logits.detach().requires_grad_()
    r = fl.token_logprobs(logits, tokens, temperature=c["temperature"], top_k=c["k"], entropy=c["entropy"],
                          ignore_index=IGNORE)
    out = {"logprobs": r.logprobs.detach()}
    if c["entropy"]:
        out["entropy"] = r.entropy.detach()
    if c["k"]:
        out["top_logprobs"], out["top_tokens"] = r.top_logprobs.detach(), r.top_tokens
    if c["train"]:
        outs, grads = [r.logprobs], [g_lp]
        if c["entropy"]:
            outs, grads = outs + [r.entropy], grads + [g_ent]
        if c["k"]:
            outs, grads = outs + [r.top_logprobs], grads + [g_top]
        out["grad"], = torch.autograd.grad(outs, [logits], grads)
    return out


# ======================================================================================
# the plain forms
# ======================================================================================

def _top(x, k):
    """The k largest values' indices, of equal values the lowest index first: the largest of
    (value's order as an integer, reversed index)."""
    bits = (x + 0.0).view(torch.int32)  # (+ 0.0: -0 counts as 0)
    order = torch.where(bits < 0, bits ^ 0x7fffffff, bits).to(torch.int64)
    key = (order << 32) | (0xffffffff - torch.arange(x.shape[-1], device=x.device))
    return 0xffffffff - (torch.topk(key, k, dim=-1).values & 0xffffffff)


def _plain_logprobs(c, logits, tokens, g_lp, g_ent, g_top):
    x = logits.float()
    top = x.amax(-1, keepdim=True)
    d = (x - top) / c["temperature"]
    e = torch.exp(d)
    total = e.sum(-1, keepdim=True)
    logp = d - torch.log(total)
    kept = tokens != IGNORE
    at = torch.where(kept, tokens, 0)[..., None]
    out = {"logprobs": torch.where(kept, logp.gather(-1, at)[..., 0], 0.0)}
    ent = torch.where(e > 0, e * d, 0.0).sum(-1, keepdim=True) / total
    ent = torch.log(total) - ent
    if c["entropy"]:
        out["entropy"] = ent[..., 0]
    if c["k"]:
        out["top_tokens"] = _top(x, c["k"])
        out["top_logprobs"] = logp.gather(-1, out["top_tokens"])
    if c["train"]:
        g = torch.where(kept, g_lp, 0.0)[..., None]
        p = e / total
        a = g + (g_top.sum(-1, keepdim=True) if c["k"] else 0.0)
        grad = -p * a
        if c["entropy"]:
            grad = grad - g_ent[..., None] * torch.where(p > 0, p * (logp + ent), 0.0)
        grad.scatter_add_(-1, at, g)
        if c["k"]:
            grad.scatter_add_(-1, out["top_tokens"], g_top)
        out["grad"] = (grad / c["temperature"]).to(logits.dtype)
    return out


def _plain_norm(grad):
    norm = torch.sqrt(grad.double().square().sum()).float()
    return norm, torch.clamp(MAX_NORM / (norm + 1e-6), max=1.0)


def _to8(x, positive):
    """Blocks of 256 as e4m3 codes and fp32 scales; what is positive keeps at least the smallest code."""
    x = x.view(-1, BLOCK)
    top = x.abs().amax(1, keepdim=True)
    inv = torch.where(top >= TINY, TOP_CODE / top, 0.0)
    y = x * inv
    if positive:
        y = torch.where((y < SMALLEST) & (y > 0), SMALLEST, y)
    scale = torch.where(top >= TINY, top * (1.0 / TOP_CODE), 0.0)
    return y.to(torch.float8_e4m3fn).view(-1), scale.view(-1)


def _from8(code, scale):
    return (code.float().view(-1, BLOCK) * scale[:, None]).view(-1)


def _plain_adamw(state, scale):
    eight = state["case"]["bits"] == 8
    state["steps"] += 1
    t = state["steps"][0].double()  # every tensor has taken the same number of steps
    step_size = (LR / (1 - BETA1 ** t)).float()
    root_scale = (1 / torch.sqrt(1 - BETA2 ** t)).float()
    g = state["grad"].float()
    if scale is not None:
        g = g * scale
    if eight:
        m = _from8(state["avg"], state["avg_scale"])
        v = _from8(state["sq"], state["sq_scale"]).square()
    else:
        m, v = state["avg"], state["sq"]
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + (g * (1 - BETA2)) * g
    root = torch.sqrt(v)
    p = state["param"].float() * (1 - LR * DECAY) - step_size * (m / (root * root_scale + EPS))
    state["param"].copy_(p)
    if eight:
        for name, x in (("avg", m), ("sq", root)):
            code, s = _to8(x, name == "sq")
            state[name].copy_(code)
            state[name + "_scale"].copy_(s)
    else:
        state["avg"].copy_(m)
        state["sq"].copy_(v)


# ======================================================================================
# 64 bits
# ======================================================================================

def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "logprobs":
        return _exact_logprobs(case, state["logits"].double(), state["tokens"], state["grads"])
    out = {}
    g = state["grad"].double()
    if case["op"] in ("norm", "update"):
        norm = torch.linalg.vector_norm(g)
        out["norm"], out["scale"] = norm, torch.minimum(MAX_NORM / (norm + 1e-6), torch.ones_like(norm))
        g = g * out["scale"]
    if case["op"] == "norm":
        return out
    if case["bits"] == 8:
        m = state["avg"].double() * state["avg_scale"].double().repeat_interleave(BLOCK)
        v = (state["sq"].double() * state["sq_scale"].double().repeat_interleave(BLOCK)) ** 2
    else:
        m, v = state["avg"].double(), state["sq"].double()
    m = m + (1 - BETA1) * (g - m)
    v = v + (1 - BETA2) * (g * g - v)
    t = STEPS + 1
    ratio = (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)).sqrt() + EPS)
    p = state["param"].double()
    out["param"] = p - LR * DECAY * p - LR * ratio
    out["steps"] = state["steps"] + 1
    # a code next to a border between two has no exact value: rounding the sums decides it
    out["avg"], out["sq"] = (m, v) if case["bits"] == 32 else (None, None)
    if case["bits"] == 8:
        out["avg_scale"] = m.abs().view(-1, BLOCK).amax(1) / TOP_CODE
        out["sq_scale"] = v.view(-1, BLOCK).amax(1).sqrt() / TOP_CODE
    return out


def _exact_logprobs(case, x, tokens, grads):
    temp, k = case["temperature"], case["k"]
    logp = torch.log_softmax(x / temp, -1)
    p = logp.exp()
    plogp = torch.where(p > 0, p * logp, 0.0)
    kept = tokens != IGNORE
    one = torch.where(kept, tokens, 0)
    out = {"logprobs": torch.where(kept, torch.take_along_dim(logp, one[..., None], -1)[..., 0], 0.0)}
    h = -plogp.sum(-1)
    if case["entropy"]:
        out["entropy"] = h
    if k:
        index = torch.sort(x, dim=-1, descending=True, stable=True).indices[..., :k]
        out["top_tokens"], out["top_logprobs"] = index, torch.take_along_dim(logp, index, -1)
    if case["train"]:
        g_lp, g_ent, g_top = (g.double() for g in grads)
        g_lp = torch.where(kept, g_lp, 0.0)
        up = torch.zeros_like(x).scatter_add_(-1, one[..., None], g_lp[..., None])  # dL / d log p
        if k:
            up.scatter_add_(-1, index, g_top)
        grad = up - p * up.sum(-1, keepdim=True)
        if case["entropy"]:
            grad = grad - g_ent[..., None] * (plogp + p * h[..., None])
        out["grad"] = grad / temp
    return out
