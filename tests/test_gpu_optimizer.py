"""GPU: gradient norm and AdamW against float64 formulas, the 8-bit states against the same steps on the CPU.

Tolerances count roundings, u = 2^-24. m' = b1 m + c1 g is two products and a sum, of constants that are
themselves rounded: 4 u (|b1 m| + |c1 g|), g's own scale one more. v' likewise with one product more: 6 u v'. The root of
it then carries 4 u, the ratio m' / (root s + eps) beside m's error 8 u, the update one more for its step size (two more where
the device's 64-bit powers round another way), and p' two products and a difference: 3 u (|p| + |update|). A bf16
parameter is rounded once at the end (half a step, eps / 2). The 8-bit codes are compared bit for bit: every
operation up to them is correctly rounded on both sides and they come in one order.
"""
from __future__ import annotations

import copy
import math

import numpy as np
import pytest
import torch

import fields_lm_amd as fl
from fields_lm_amd.optim import STATE8_DTYPE

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HYPER = dict(lr=3e-3, betas=(0.9, 0.98), eps=1e-8, weight_decay=0.1)


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm device")
    return torch.device("cuda:0")


# ------------------------------------------------------------------ norm
SIZES = [[1], [0, 5], [255, 256, 257], [4095, 4096, 4097, 0, 1], [7] * 200, [100003, 3, 65536], [0], [(1 << 22) + 5]]


def tensors(dev, sizes, dtype, seed, scale=1.0, shift=0):
    """Tensors of these sizes, each ``shift`` elements behind its allocation's start."""
    g = torch.Generator(device=dev).manual_seed(seed)
    return [(torch.randn(n + shift, device=dev, generator=g) * scale).to(dtype)[shift:] for n in sizes]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{max(s)}")
def test_grad_norm(dev, sizes, shift, dtype):
    print(f"[case] grad_norm {sizes[:5]} shift={shift} {dtype}", flush=True)
    grads = tensors(dev, sizes, dtype, len(sizes), 0.1, shift)
    exp = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    norm, scale = fl.grad_norm(grads, 0.5)
    assert norm.dtype == torch.float32 and norm.shape == () == scale.shape
    assert abs(float(norm) - exp) <= 2 * U * exp
    assert abs(float(scale) - min(1.0, 0.5 / (exp + 1e-6))) <= 6 * U * float(scale)
    assert torch.equal(fl.grad_norm(grads), norm) and torch.equal(fl.grad_norm(grads, 0.5)[1], scale)


@pytest.mark.parametrize("n", [63, 64, 65, 191, 192, 193, 500])
def test_grad_norm_of_many_mixed_tensors(dev, n):
    """Lists at and past a launch's tensors, types in turn of 1, 2, 3 and empty ones between."""
    print(f"[case] grad_norm, {n} mixed tensors", flush=True)
    sizes = [0 if i % 11 == 5 else 1 + 37 * i % 9000 for i in range(n)]
    g = [t.bfloat16() if i % 6 in (1, 3, 4) else t for i, t in enumerate(tensors(dev, sizes, torch.float32, n))]
    exp = math.sqrt(sum(float(t.double().square().sum()) for t in g))
    assert abs(float(fl.grad_norm(g)) - exp) <= 2 * U * exp


def test_grad_norm_of_mixed_types_shapes_and_extremes(dev):
    print("[case] grad_norm, mixed types", flush=True)
    g = tensors(dev, [300, 64], torch.float32, 1) + tensors(dev, [129], torch.bfloat16, 2)
    g[0] = g[0].view(30, 10).t()
    exp = math.sqrt(sum(float(t.double().square().sum()) for t in g))
    assert abs(float(fl.grad_norm(g)) - exp) <= 2 * U * exp
    big = [torch.full((1000,), 1e30, device=dev), torch.full((3,), 1e-30, device=dev)]  # squares past fp32
    exp = math.sqrt(sum(float(t.double().square().sum()) for t in big))
    assert abs(float(fl.grad_norm(big)) - exp) <= 2 * U * exp
    tiny = [torch.full((1000,), 1e-35, device=dev)]
    exp = math.sqrt(float(tiny[0].double().square().sum()))
    assert abs(float(fl.grad_norm(tiny)) - exp) <= 2 * U * exp
    for bad in (float("inf"), float("nan")):
        t = torch.zeros(5000, device=dev)
        t[4321] = bad
        norm, scale = fl.grad_norm([torch.ones(3, device=dev), t], 1.0)
        assert not math.isfinite(float(norm)) and math.isnan(float(scale))
    norm, scale = fl.grad_norm([torch.zeros(3, device=dev)], 0.0)
    assert float(norm) == 0.0 == float(scale)
    assert float(fl.grad_norm([torch.ones(4, device=dev)], float("inf"))[1]) == 1.0


def test_grad_norm_refuses_on_the_device(dev):
    print("[case] grad_norm refusals", flush=True)
    with pytest.raises(TypeError):
        fl.grad_norm([torch.ones(3, device=dev, dtype=torch.float16)])
    with pytest.raises(ValueError):
        fl.grad_norm([torch.ones(3, device=dev), torch.ones(3)])
    with pytest.raises(ValueError):
        fl.grad_norm([torch.ones(3, device=dev)], -1.0)
    with pytest.raises(TypeError):
        fl.grad_norm([torch.ones(3, device=dev).to_sparse()])


# ------------------------------------------------------------------ AdamW, fp32 states
def exact(p, g, m, v, t, gs=1.0, lr=3e-3, betas=(0.9, 0.98), eps=1e-8, weight_decay=0.1):
    """One step in float64 with its tolerances: (p, m, v) and (tol_p, tol_m, tol_v)."""
    p, g, m, v = (x.double() for x in (p, g, m, v))
    g = g * gs
    b1, b2 = betas
    tol_m = 5 * U * ((b1 * m).abs() + ((1 - b1) * g).abs())
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    c = 1 / (1 - b1 ** t)
    denom = (v / (1 - b2 ** t)).sqrt() + eps
    update = lr * c * m / denom
    tol_p = 3 * U * (p.abs() + update.abs()) + lr * c * (tol_m + 12 * U * m.abs()) / denom
    return (p * (1 - lr * weight_decay) - update, m, v), (tol_p, tol_m + 1e-45, 8 * U * v + 1e-45)


def near(got, exp, tol, what):
    off = (got.double() - exp).abs()
    tol = tol + exp.abs() * (torch.finfo(got.dtype).eps / 2 if got.dtype == torch.bfloat16 else 0)
    assert bool((off <= tol).all()), (what, float((off / tol.clamp_min(1e-60)).max()))


def start32(dev, sizes, dtype, seed, shift=0):
    p, g = tensors(dev, sizes, dtype, seed, 0.5, shift), tensors(dev, sizes, dtype, seed + 1, 0.1, shift)
    m = tensors(dev, sizes, torch.float32, seed + 2, 0.05, shift)
    v = [x.square_() for x in tensors(dev, sizes, torch.float32, seed + 3, 0.1, shift)]
    return p, g, m, v


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{max(s)}")
def test_adamw_step(dev, sizes, shift, dtype):
    print(f"[case] adamw_step {sizes[:5]} shift={shift} {dtype}", flush=True)
    p, g, m, v = start32(dev, sizes, dtype, len(sizes), shift)
    before = [[t.clone() for t in l] for l in (p, g, m, v)]
    steps = torch.arange(len(sizes), device=dev)
    scale = torch.tensor(0.37, device=dev) if shift else None
    fl.adamw_step(p, g, m, v, steps, grad_scale=scale, **HYPER)
    assert torch.equal(steps, torch.arange(len(sizes), device=dev) + 1)
    for i in range(len(sizes)):
        if sizes[i] == 0:
            continue
        exp, tol = exact(*(l[i] for l in before), i + 1, float(scale) if shift else 1.0)
        for got, e, t, what in zip((p[i], m[i], v[i]), exp, tol, "pmv"):
            near(got, e, t, (i, what))
        assert torch.equal(g[i], before[1][i])


def test_adamw_neighbours_stay_as_they_were(dev):
    """Values beside a tensor in its buffer (before it, after it, between blocks) are not written."""
    print("[case] adamw_step leaves neighbours alone", flush=True)
    for eight in (False, True):
        for dtype in (torch.float32, torch.bfloat16):
            n, total = 777, 2048
            buf = [torch.full((total,), 3.0, device=dev, dtype=dtype) for _ in range(2)]
            st = [torch.full((total,), 0.5, device=dev).to(STATE8_DTYPE if eight else torch.float32) for _ in range(2)]
            sc = [torch.full((16,), 0.25, device=dev) for _ in range(2)]
            cut = slice(5, 5 + n)
            step = torch.zeros(1, dtype=torch.long, device=dev)
            fl.adamw_step([buf[0][cut]], [buf[1][cut]], [st[0][cut]], [st[1][cut]], step, **HYPER,
                          **(dict(exp_avg_scales=[sc[0][3:7]], exp_avg_sq_scales=[sc[1][3:7]]) if eight else {}))
            for t, old in [(buf[0], 3.0)] + [(s.float(), 0.5) for s in st]:
                outside = torch.cat((t[:5], t[5 + n:]))
                # inside, all change but a bf16 weight: m' / (1 - 0.9) = 7.5 over sqrt(v' / (1 - 0.98)) = 5.8 (v = 0.5) or
                # less than 5.0 (8 bits: v = 1 / 64) makes a step below lr (2.5 + 0.3) = 0.0084 at most and 0.0048 with
                # v = 0.5, around or below half a step of bf16 at 3, 2^-7
                assert bool((outside == old).all()) and (t.dtype == torch.bfloat16 or not bool((t[cut] == old).all()))
            if eight:
                assert all(bool((torch.cat((s[:3], s[7:])) == 0.25).all()) for s in sc)


@pytest.mark.parametrize("eight", [False, True])
def test_one_tensor_past_2_to_31_values(dev, eight):
    print(f"[case] adamw_step and grad_norm past 2^31 values, 8 bits: {eight}", flush=True)
    n = (1 << 31) + 300
    p, g = (torch.zeros(n, device=dev, dtype=torch.bfloat16) for _ in range(2))
    at = torch.tensor([0, 1, (1 << 31) - 1, 1 << 31, n - 1], device=dev)
    p[at], g[at] = torch.tensor([1.0, -2.0, 3.0, -4.0, 5.0], device=dev).bfloat16(), torch.tensor([2.0, 1.0, -1.0, 3.0, -2.0],
                                                                                                 device=dev).bfloat16()
    assert abs(float(fl.grad_norm([g])) - math.sqrt(19.0)) <= 2 * U * math.sqrt(19.0)
    def new():
        return torch.zeros(n, device=dev, dtype=torch.uint8 if eight else torch.float32).view(
            STATE8_DTYPE if eight else torch.float32)

    m, v = new(), new()
    scales = [[torch.zeros(-(-n // 256), device=dev)] for _ in range(2)] if eight else [None, None]
    old = p[at].clone()
    fl.adamw_step([p], [g], [m], [v], torch.zeros(1, dtype=torch.long, device=dev), exp_avg_scales=scales[0],
                  exp_avg_sq_scales=scales[1], **{**HYPER, "lr": 0.1})
    exp, tol = exact(old, g[at], torch.zeros(5, device=dev), torch.zeros(5, device=dev), 1, **{**HYPER, "lr": 0.1})
    near(p[at], exp[0], tol[0], "p")
    assert int((p != 0).sum()) == 5 and int((m.view(torch.uint8) if eight else m).ne(0).sum()) == 5


def test_adamw_lr_and_scale_are_read_on_the_device(dev):
    print("[case] adamw_step with lr on the device, and steps that are skipped", flush=True)
    p, g, m, v = start32(dev, [1000, 3], torch.float32, 3)
    q, g2, m2, v2 = ([t.clone() for t in l] for l in (p, g, m, v))
    steps, steps2 = (torch.full((2,), 4, device=dev) for _ in range(2))
    lr = torch.tensor(3e-3, device=dev)
    fl.adamw_step(p, g, m, v, steps, **HYPER)
    fl.adamw_step(q, g2, m2, v2, [steps2[0], steps2[1]], **{**HYPER, "lr": lr})
    # the device's lr is the fp32 neighbour of the host's: 2^-24 of the update and of the decay
    for a, b in zip(p, q):
        assert float((a - b).abs().max()) <= 4 * U * float(a.abs().max())
    assert all(torch.equal(a, b) for a, b in zip(m + v, m2 + v2)) and torch.equal(steps, steps2)
    kept = [t.clone() for t in p + m + v]
    for bad in (float("nan"), float("inf"), -float("inf")):
        fl.adamw_step(p, g, m, v, steps, grad_scale=torch.tensor(bad, device=dev), **HYPER)
    assert all(torch.equal(a, b) for a, b in zip(kept, p + m + v)) and steps.tolist() == [5, 5]
    fl.adamw_step(p, g, m, v, steps, grad_scale=torch.zeros((), device=dev), **HYPER)
    assert steps.tolist() == [6, 6] and all(torch.equal(a, 0.9 * b) for a, b in zip(m, kept[2:4]))


def test_adamw_first_step_and_edges_of_the_hyperparameters(dev):
    print("[case] adamw_step, first step, betas 0, eps 0", flush=True)
    for hyper in (dict(lr=1e-2, betas=(0.0, 0.0), eps=1e-8, weight_decay=0.0), dict(lr=0.0, betas=(0.9, 0.999), eps=1e-8,
                  weight_decay=0.3), dict(lr=1e-2, betas=(0.9, 0.999), eps=0.0, weight_decay=0.0)):
        p, g, m, v = start32(dev, [513], torch.float32, 9)
        m[0].zero_(), v[0].zero_()
        old = [t[0].clone() for t in (p, g, m, v)]
        fl.adamw_step(p, g, m, v, torch.zeros(1, dtype=torch.long, device=dev), **hyper)
        exp, tol = exact(*old, 1, **hyper)
        for got, e, t in zip((p[0], m[0], v[0]), exp, tol):
            near(got, e, t, hyper)


def test_adamw_reads_gradients_of_any_strides_and_counts_as_a_write(dev):
    print("[case] adamw_step, strides and versions", flush=True)
    w = torch.nn.Parameter(torch.randn(6, 5, device=dev))
    g = torch.randn(5, 6, device=dev).t()
    a, b = w.detach().clone(), w.detach().clone()
    zeros = [torch.zeros_like(w) for _ in range(4)]
    fl.adamw_step([a], [g], zeros[:1], zeros[1:2], torch.zeros(1, dtype=torch.long, device=dev), **HYPER)
    fl.adamw_step([b], [g.contiguous()], zeros[2:3], zeros[3:], torch.zeros(1, dtype=torch.long, device=dev), **HYPER)
    assert torch.equal(a, b) and not torch.equal(a, w)
    y = (w * w).sum()
    fl.adamw_step([w], [g], zeros[:1], zeros[1:2], torch.zeros(1, dtype=torch.long, device=dev), **HYPER)
    with pytest.raises(RuntimeError):  # w was changed after the product saved it
        y.backward()


def test_adamw_refuses_on_the_device(dev):
    print("[case] adamw_step refusals", flush=True)
    def one(dtype=torch.float32, n=4):
        return torch.zeros(n, device=dev, dtype=dtype)

    step = torch.zeros(1, dtype=torch.long, device=dev)
    p = one()
    for bad in (([one(torch.float16)], [one(torch.float16)], [one()], [one()], step),
                ([p], [one(torch.bfloat16)], [one()], [one()], step),
                ([p], [one()], [one(torch.bfloat16)], [one()], step),
                ([p], [one().to_sparse()], [one()], [one()], step)):
        with pytest.raises(TypeError):
            fl.adamw_step(*bad)
    for bad in (([p], [one(n=5)], [one()], [one()], step), ([p], [one()], [one(n=5)], [one()], step),
                ([p], [torch.zeros(4)], [one()], [one()], step), ([p], [one()], [one()], [one()], step.int()),
                ([p], [one()], [one()], [one()], [step.expand(2)]),
                ([p], [one()], [one()], [one()], [step[0], step[0]]), ([p], [one()], [one()], [one()], step.cpu()),
                ([one(n=8)[::2]], [one()], [one()], [one()], step), ([p], [one()], [one(n=8)[::2]], [one()], step),
                ([p, p], [one(), one()], [one(), one()], [one(), one()], torch.zeros(2, dtype=torch.long, device=dev)),
                ([p, one()], [one(), one()], [one(), one()], [one(), one()], [step, step])):
        with pytest.raises(ValueError):
            fl.adamw_step(*bad)
    with pytest.raises(TypeError):
        fl.adamw_step([p], [one()], [one()], [one()], [step.int()])
    with pytest.raises(TypeError):
        fl.adamw_step([p], [3], [one()], [one()], step)
    with pytest.raises(ValueError):
        fl.adamw_step([p], [one()], [one()], [one()], step, grad_scale=torch.zeros(2, device=dev))
    with pytest.raises(ValueError):
        fl.adamw_step([p], [one()], [one()], [one()], step, lr=torch.zeros((), dtype=torch.float64, device=dev))
    with pytest.raises(ValueError):
        fl.adamw_step([p], [one()], [one(STATE8_DTYPE)], [one(STATE8_DTYPE)], step, exp_avg_scales=[one(n=2)],
                      exp_avg_sq_scales=[one(n=1)])
    shared, m, sc = one(n=12), one(), one(n=1)
    codes = one(STATE8_DTYPE)
    for bad in (([shared[:8], shared[4:]], [one(n=8), one(n=8)], [one(n=8), one(n=8)], [one(n=8), one(n=8)],
                 torch.zeros(2, dtype=torch.long, device=dev)),   # two parameters overlap
                ([p], [one()], [m], [m], step),                   # both moments are one
                ([p], [one()], [p], [m], step),                   # a moment is the parameter
                ([shared[:4]], [shared[2:6]], [m], [one()], step),  # a gradient lies in a parameter
                ([p], [m], [m], [one()], step)):
        with pytest.raises(ValueError):
            fl.adamw_step(*bad)
    with pytest.raises(ValueError):
        fl.adamw_step([p], [one()], [codes], [one(STATE8_DTYPE)], step, exp_avg_scales=[sc], exp_avg_sq_scales=[sc])
    with pytest.raises(RuntimeError):
        torch.jit.trace(lambda g: fl.grad_norm([g]), (p,))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda g: fl.grad_norm([g]))(one(n=8).view(2, 4))
    grad = one()  # one gradient of two parameters is read twice
    fl.adamw_step([one(), one()], [grad, grad], [one(), one()], [one(), one()],
                  torch.zeros(2, dtype=torch.long, device=dev))
    assert float(p.abs().sum()) == 0.0 and int(step) == 0


# ------------------------------------------------------------------ AdamW, 8-bit states
def quantised(x, root):
    """Codes and scales of the flat fp32 x on the CPU, in the kernel's operations (numpy's reciprocal and root are
    correctly rounded; torch's on the CPU are not: of 10^6 roots 6,558 came out next to the nearest float)."""
    n = x.numel()
    b = torch.zeros(-(-n // 256) * 256)
    b[:n] = x
    b = b.view(-1, 256)
    top = b.abs().amax(1, keepdim=True)
    held = top >= 1e-30
    y = b * torch.where(held, torch.from_numpy(np.float32(1) / top.clamp_min(1e-38).numpy()) * 448.0, 0.0)
    if root:
        y = torch.where((y > 0) & (y < 2.0 ** -9), torch.tensor(2.0 ** -9), y)
    return y.to(STATE8_DTYPE).view(-1)[:n], torch.where(held, top * (1.0 / 448.0), 0.0).view(-1)


def step8(p, g, mc, ms, vc, vs, t, gs=1.0, lr=3e-3, betas=(0.9, 0.98), eps=1e-8, weight_decay=0.1):
    """The 8-bit step on the CPU: (new codes and scales of both, exact p and its tolerance)."""
    n = p.numel()

    def back(code, scale):
        return code.float() * scale.repeat_interleave(256)[:n]

    m, v = back(mc, ms), back(vc, vs)
    v = v * v
    exp, tol = exact(p, g, m, v, t, gs, lr, betas, eps, weight_decay)
    b1, b2 = betas
    g = g.float() * torch.tensor(gs)
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * (1 - b2)) * g
    return (*quantised(m, False), *quantised(torch.from_numpy(np.sqrt(v.numpy())), True)), exp[0], tol[0]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("sizes", SIZES[:-2], ids=lambda s: f"{len(s)}x{max(s)}")
def test_adamw_step_8_bits(dev, sizes, shift, dtype):
    print(f"[case] adamw_step 8 bits {sizes[:5]} shift={shift} {dtype}", flush=True)
    n = len(sizes)
    p = tensors(dev, sizes, dtype, n, 0.5, shift)
    blocks = [-(-s // 256) for s in sizes]
    mc, vc = ([t.to(STATE8_DTYPE) for t in tensors(dev, sizes, torch.float32, 0, 0.0, shift)] for _ in range(2))
    ms, vs = ([torch.zeros(b, device=dev) for b in blocks] for _ in range(2))
    steps = torch.zeros(n, dtype=torch.long, device=dev)
    for turn in range(3):
        g = tensors(dev, sizes, dtype, n + turn, 1e-3, shift)
        g = [x * torch.exp(3 * y) for x, y in zip(g, tensors(dev, sizes, dtype, 50 + turn, 1.0, shift))]  # over decades
        before = [[t.cpu() for t in l] for l in (p, g, mc, ms, vc, vs)]
        fl.adamw_step(p, g, mc, vc, steps, grad_scale=torch.tensor(0.7, device=dev) if shift else None, exp_avg_scales=ms,
                      exp_avg_sq_scales=vs, **HYPER)
        for i in range(n):
            if sizes[i] == 0:
                continue
            (emc, ems, evc, evs), ep, tol = step8(*(l[i] for l in before), turn + 1, 0.7 if shift else 1.0)
            near(p[i].cpu(), ep, tol, (turn, i, "p"))
            for got, exp, what in ((ms[i], ems, "ms"), (vs[i], evs, "vs"), (mc[i].view(torch.uint8), emc.view(torch.uint8), "mc"),
                                   (vc[i].view(torch.uint8), evc.view(torch.uint8), "vc")):
                assert torch.equal(got.cpu(), exp), (turn, i, what)
    assert bool((steps == 3).all())


def test_adamw_8_bits_of_uneven_blocks(dev):
    """Blocks of zeros, of one value, of values over all of fp32's range, of subnormals, of infinity."""
    print("[case] adamw_step 8 bits, uneven blocks", flush=True)
    g = torch.zeros(8, 256)
    g[1, 17] = 2.0
    g[2] = 10.0 ** torch.linspace(-18, 3, 256)
    g[3] = 1e-38
    g[4] = torch.where(torch.arange(256) % 2 == 0, 1.0, -1.0)
    g[5] = 10.0 ** torch.linspace(0, 18, 256)
    g[6, 3] = 1e-20
    g = g.view(-1)
    n = g.numel()
    p = torch.randn(n, generator=torch.Generator().manual_seed(0))
    state = [torch.zeros(n).to(STATE8_DTYPE), torch.zeros(8), torch.zeros(n).to(STATE8_DTYPE), torch.zeros(8)]
    on = [t.to(dev) for t in (p, *state)]
    steps = torch.zeros(1, dtype=torch.long, device=dev)
    for turn in range(4):
        grad = g if turn % 2 == 0 else torch.zeros(n)
        (mc, ms, vc, vs), ep, tol = step8(p, grad, *state, turn + 1)
        fl.adamw_step([on[0]], [grad.to(dev)], [on[1]], [on[3]], steps, exp_avg_scales=[on[2]], exp_avg_sq_scales=[on[4]], **HYPER)
        near(on[0].cpu(), ep, tol, turn)
        for got, exp in zip(on[1:], (mc, ms, vc, vs)):
            assert torch.equal(got.cpu().view(torch.uint8), exp.view(torch.uint8)), turn
        assert bool(on[0].isfinite().all())
        # a root that is not 0 never rounds to 0 beside a moment that does not: no step without a gradient runs away
        assert not bool(((mc.float() != 0) & (vc.float() == 0) & (vs.repeat_interleave(256) > 0)).any())
        p, state = on[0].cpu(), [mc, ms, vc, vs]
    bad = torch.zeros(n)
    bad[300] = float("nan")
    before = [t.clone() for t in on]
    fl.adamw_step([on[0]], [bad.to(dev)], [on[1]], [on[3]], steps, exp_avg_scales=[on[2]], exp_avg_sq_scales=[on[4]], **HYPER)
    nan = on[0].isnan().view(8, 256).any(1).tolist()
    assert nan == [False, True] + [False] * 6 and before[0].isfinite().all()


# ------------------------------------------------------------------ the optimizer, and a run of all together
def stock_pair(dev, **kw):
    torch.manual_seed(0)
    own = torch.nn.Sequential(torch.nn.Linear(40, 300), torch.nn.SiLU(), torch.nn.Linear(300, 17, bias=False)).to(dev)
    stock = torch.nn.Sequential(torch.nn.Linear(40, 300), torch.nn.SiLU(), torch.nn.Linear(300, 17, bias=False)).to(dev)
    stock.load_state_dict(own.state_dict())
    return own, stock


def test_optimizer_matches_torch_adamw(dev):
    """Groups, clipping, a parameter without a gradient for a while, a changed lr; ten steps."""
    print("[case] AdamW against torch.optim.AdamW", flush=True)
    own, stock = stock_pair(dev)
    groups = lambda m: [dict(params=[m[0].weight, m[2].weight], weight_decay=0.2), dict(params=[m[0].bias], lr=1e-2)]  # noqa: E731
    a = fl.AdamW(groups(own), lr=3e-3, betas=(0.9, 0.95), max_grad_norm=0.5)
    b = torch.optim.AdamW(groups(stock), lr=3e-3, betas=(0.9, 0.95))
    for turn in range(10):
        x = torch.randn(32, 40, device=dev, generator=torch.Generator(device=dev).manual_seed(turn))
        for m, opt in ((own, a), (stock, b)):
            m[0].bias.requires_grad_(turn != 3)
            opt.zero_grad(set_to_none=True)
            (m(x).square().mean() * 30).backward()
            opt.param_groups[0]["lr"] = 3e-3 / (1 + turn)
        norm = torch.nn.utils.clip_grad_norm_(stock.parameters(), 0.5)
        a.step()
        b.step()
        assert abs(float(a.grad_norm) - float(norm)) <= 1e-4 * float(norm)
    for p, q in zip(own.parameters(), stock.parameters()):
        # ten steps of at most 3e-3 / 1e-2 each; a gradient that differs by its own rounding noise moves its step by that share
        assert float((p - q).abs().max()) <= 1e-3 * 10 * 1e-2
    assert int(a.state[own[0].bias]["step"]) == 9 and int(a.state[own[0].weight]["step"]) == 10


def test_optimizer_continues_from_its_checkpoint(dev):
    print("[case] AdamW checkpoint", flush=True)
    for bits in (32, 8):
        own, other = stock_pair(dev)
        a = fl.AdamW(own.parameters(), state_bits=bits)
        grads = [[torch.randn_like(p) for p in own.parameters()] for _ in range(4)]

        def take(model, opt, gs):
            for p, g in zip(model.parameters(), gs):
                p.grad = g.clone()
            opt.step()

        take(own, a, grads[0])
        take(own, a, grads[1])
        other.load_state_dict(own.state_dict())
        b = fl.AdamW(other.parameters())
        b.load_state_dict(a.state_dict())
        for gs in grads[2:]:
            take(own, a, gs)
            take(other, b, gs)
        assert all(torch.equal(p, q) for p, q in zip(own.parameters(), other.parameters()))


def test_optimizer_in_a_graph(dev):
    """Norm, clip and step captured and replayed, with eager steps between, equal eager steps alone."""
    print("[case] AdamW in a graph", flush=True)
    for bits in (32, 8):
        own, other = stock_pair(dev)
        kw = dict(state_bits=bits, max_grad_norm=1.0, lr=torch.tensor(1e-2, device=dev))
        a, b = fl.AdamW(own.parameters(), **kw), fl.AdamW(other.parameters(), **kw)
        for p, q in zip(own.parameters(), other.parameters()):
            p.grad, q.grad = torch.randn_like(p), torch.zeros_like(q)
        fresh = fl.AdamW([torch.nn.Parameter(torch.zeros(3, device=dev))])
        fresh.param_groups[0]["params"][0].grad = torch.ones(3, device=dev)
        a.step()
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            a.step()
            with pytest.raises(RuntimeError):
                fresh.step()
        for turn in range(6):
            for p in own.parameters():
                p.grad.normal_(generator=torch.Generator(device=dev).manual_seed(turn)) if turn else None
            if turn == 4:
                own[0].weight.grad[0, 0] = float("inf")  # skipped
            kw["lr"].fill_(1e-2 / (turn + 1))
            for p, q in zip(own.parameters(), other.parameters()):
                q.grad.copy_(p.grad)
            b.step()
            if turn in (0, 3):
                a.step() if turn else None
            else:
                g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(own.parameters(), other.parameters())), turn
        assert int(a.state[own[0].weight]["step"]) == 5


@pytest.mark.parametrize("bits", [32, 8])
def test_a_training_step_of_field_blocks(dev, bits):
    """Embedding, two Field blocks, head, token log probabilities as the loss, clip and AdamW: gradients against the
    stock loss, and the step against torch's AdamW (fp32 states) or run for its result (8 bits)."""
    print(f"[case] a training step of Field blocks, {bits} bits", flush=True)
    torch.manual_seed(0)
    vocab, dim = 501, 64
    emb = torch.nn.Embedding(vocab, dim).to(dev)
    blocks = torch.nn.ModuleList(fl.FieldBlock(dim, "triton", 32, 32, 64, 96) for _ in range(2)).to(dev)
    head = torch.nn.Linear(dim, vocab, bias=False).to(dev)
    params = [p for m in (emb, blocks, head) for p in m.parameters()]
    ids = torch.randint(0, vocab, (3, 40), device=dev)
    target = ids[:, 1:].clone()
    target[1, 20:] = -100  # padding

    def logits():
        x = emb(ids)
        for b in blocks:
            x = b(x)
        return head(x)

    r = fl.token_logprobs(logits()[:, :-1], target, entropy=True)
    kept = int((target != -100).sum())
    loss = -r.logprobs.sum() / kept
    stock = torch.nn.functional.cross_entropy(logits()[:, :-1].reshape(-1, vocab), target.reshape(-1))
    assert abs(float(loss) - float(stock)) <= 1e-5 * float(stock)  # fp32 sums over 117 rows of 501
    grads = torch.autograd.grad(loss, params)
    for a, b in zip(grads, torch.autograd.grad(stock, params)):
        assert float((a - b).norm()) <= 1e-4 * float(b.norm()) + 1e-9
    opt = fl.AdamW(params, lr=1e-2, state_bits=bits, max_grad_norm=0.1)
    before = [p.detach().clone() for p in params]
    for p, g in zip(params, grads):
        p.grad = g.clone()
    opt.step()
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    assert abs(float(opt.grad_norm) - norm) <= 1e-6 * norm
    for p, old, g in zip(params, before, grads):
        exp, tol = exact(old, g, torch.zeros_like(g), torch.zeros_like(g), 1, min(1.0, 0.1 / (norm + 1e-6)), 1e-2,
                         (0.9, 0.999), 1e-8, 1e-2)
        # (the clip's own roundings move g by 4 u, which a first step's ratio hardly sees)
        near(p.detach(), exp[0], 2 * tol[0], "p")
        assert bool(p.isfinite().all())
    again = fl.token_logprobs(logits()[:, :-1], target).logprobs
    assert bool(again.isfinite().all()) and int(opt.state[params[0]]["step"]) == 1


def test_adamw_values_with_the_negative_flag(dev):
    """lr and grad_scale whose memory holds their negative are read as they are; step counters are refused."""
    print("[case] adamw_step, values with the negative flag", flush=True)
    p, g, m, v = start32(dev, [100], torch.float32, 5)
    lr, scale = torch.tensor(3e-3, device=dev), torch.tensor(0.5, device=dev)
    results = []
    for a, b in ((lr, scale), (torch._neg_view(-lr), torch._neg_view(-scale)),
                 (torch.complex(lr, -lr).conj().imag, torch.complex(scale, -scale).conj().imag)):
        q, m2, v2 = ([t.clone() for t in l] for l in (p, m, v))
        fl.adamw_step(q, g, m2, v2, torch.zeros(1, dtype=torch.long, device=dev), grad_scale=b, **{**HYPER, "lr": a})
        results.append(q + m2 + v2)
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))
    steps = torch._neg_view(torch.zeros(1, dtype=torch.long, device=dev))
    for bad in (steps, [steps]):
        with pytest.raises(ValueError):
            fl.adamw_step(p, g, m, v, bad, **HYPER)


def test_adamw_refuses_values_without_memory(dev):
    """A scale of zero that torch holds without memory is no missing scale."""
    print("[case] adamw_step, values without memory", flush=True)
    p, g, m, v = start32(dev, [10], torch.float32, 5)
    before = p[0].clone()
    zero = torch._efficientzerotensor((), device=dev)
    step = torch.zeros(1, dtype=torch.long, device=dev)
    for kw in (dict(grad_scale=zero), dict(lr=zero)):
        with pytest.raises(ValueError):
            fl.adamw_step(p, g, m, v, step, **{**HYPER, **kw})
    assert torch.equal(p[0], before) and int(step) == 0


def test_optimizer_copy_steps_as_its_original(dev):
    print("[case] AdamW, a deep copy", flush=True)
    own, _ = stock_pair(dev)
    a = fl.AdamW(own.parameters(), state_bits=8, max_grad_norm=0.1, lr=1e-2)

    def step(model, opt, seed):
        for i, p in enumerate(model.parameters()):
            p.grad = torch.randn(p.shape, device=dev, generator=torch.Generator(device=dev).manual_seed(seed + i))
        opt.step()

    step(own, a, 0)
    other, b = copy.deepcopy((own, a))
    for model, opt in ((own, a), (other, b)):
        step(model, opt, 10)
    assert torch.equal(a.grad_norm, b.grad_norm)
    assert all(torch.equal(p, q) for p, q in zip(own.parameters(), other.parameters()))


def test_optimizer_continues_from_a_checkpoint_read_on_the_host(dev, tmp_path):
    """As a program resumes: saved, read with its tensors on the host, loaded; the learning rate lies on the device."""
    print("[case] AdamW checkpoint by way of the host", flush=True)
    own, other = stock_pair(dev)
    kw = dict(state_bits=8, max_grad_norm=1.0)
    a = fl.AdamW(own.parameters(), lr=torch.tensor(1e-2, device=dev), **kw)
    grads = [[torch.randn_like(p) for p in own.parameters()] for _ in range(2)]

    def take(model, opt, gs):
        for p, g in zip(model.parameters(), gs):
            p.grad = g.clone()
        opt.step()

    take(own, a, grads[0])
    torch.save(a.state_dict(), tmp_path / "opt.pt")
    other.load_state_dict(own.state_dict())
    b = fl.AdamW(other.parameters(), lr=torch.tensor(1.0, device=dev), **kw)
    b.load_state_dict(torch.load(tmp_path / "opt.pt", map_location="cpu", weights_only=True))
    for model, opt in ((own, a), (other, b)):
        take(model, opt, grads[1])
    assert all(torch.equal(p, q) for p, q in zip(own.parameters(), other.parameters()))


def test_adamw_counts_as_a_write_of_states_and_counters(dev):
    """A product that saved a moment, a scale or a step counter does not take the stepped one for it in its backward."""
    print("[case] adamw_step, versions of states", flush=True)
    for eight in (False, True):
        for listed in (False, True):
            p, g, m, v = start32(dev, [300], torch.float32, 5)
            scales = [torch.ones(2, device=dev) for _ in range(2)] if eight else []
            if eight:
                m, v = ([t.to(STATE8_DTYPE) for t in l] for l in (m, v))
            step = torch.zeros(1, dtype=torch.long, device=dev)
            w = torch.ones((), device=dev, requires_grad=True)
            sums = [(w * t).sum() for t in (*([] if eight else [m[0], v[0]]), step, *scales)]
            before = [t._version for t in (p[0], m[0], v[0])]
            fl.adamw_step(p, g, m, v, [step] if listed else step, **HYPER,
                          **(dict(exp_avg_scales=scales[:1], exp_avg_sq_scales=scales[1:]) if eight else {}))
            assert all(t._version > n for t, n in zip((p[0], m[0], v[0]), before))
            for y in sums:
                with pytest.raises(RuntimeError):
                    y.backward()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_adamw_8_bit_moments_are_the_formulas(dev, dtype):
    """Code times scale against the moments in 64 bits, step by step from the held ones: a first moment is off by half a
    step of e4m3 (2^-4 of itself, or half of the smallest code, 2^-10 of a block's largest over 448), a root by as much
    or raised to the smallest code, both by their roundings before (16 u)."""
    print(f"[case] adamw_step 8 bits, moments in 64 bits {dtype}", flush=True)
    n, (b1, b2) = 5000, HYPER["betas"]
    gen = torch.Generator(device=dev).manual_seed(7)
    p = torch.randn(n, device=dev, generator=gen).to(dtype)
    mc, vc = (torch.zeros(n, device=dev).to(STATE8_DTYPE) for _ in range(2))
    ms, vs = (torch.zeros(-(-n // 256), device=dev) for _ in range(2))
    steps = torch.zeros(1, dtype=torch.long, device=dev)

    def held(code, scale):
        return code.double() * scale.double().repeat_interleave(256)[:n]

    def largest(x):
        full = torch.zeros(ms.numel() * 256, device=dev, dtype=torch.float64)
        full[:n] = x.abs()
        return full.view(-1, 256).amax(1).repeat_interleave(256)[:n]

    for turn in range(4):
        g = (torch.randn(n, device=dev, generator=gen) * torch.exp(2 * torch.randn(n, device=dev, generator=gen))).to(dtype)
        parts = b1 * held(mc, ms), (1 - b1) * g.double()
        m = parts[0] + parts[1]
        root = (b2 * held(vc, vs) ** 2 + (1 - b2) * g.double() ** 2).sqrt()
        fl.adamw_step([p], [g], [mc], [vc], steps, exp_avg_scales=[ms], exp_avg_sq_scales=[vs], **HYPER)
        low = 2.0 ** -10 / 448 * largest(m)
        off = (held(mc, ms) - m).abs()
        assert bool((off <= 2.0 ** -4 * m.abs() + low + 16 * U * (parts[0].abs() + parts[1].abs() + largest(m))).all()), turn
        small = 2.0 ** -9 / 448 * largest(root)  # a root that is not 0 keeps at least this
        off = (held(vc, vs) - root).abs()
        assert bool((off <= torch.maximum(2.0 ** -4 * root + small / 2, small - root) + 16 * U * largest(root)).all()), turn
        assert bool((held(vc, vs)[root > 0] > 0).all())


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("n", [479, 480, 481, 1000])
def test_adamw_step_of_many_tensors(dev, n, eight):
    """Past one launch's step counters and many of its tables: each tensor's step is that of a call of its own."""
    print(f"[case] adamw_step, {n} tensors, 8 bits: {eight}", flush=True)
    sizes = [0 if i % 13 == 7 else 1 + 37 * i % 5000 for i in range(n)]
    p, g, m, v = start32(dev, sizes, torch.float32, n)
    if eight:
        m, v = ([t.clamp(-1, 1).to(STATE8_DTYPE) for t in l] for l in (m, v))
    scales = [[torch.rand(-(-s // 256), device=dev) for s in sizes] for _ in range(2)] if eight else [None, None]

    def call(pick, steps, lists):
        lists = [None if l is None else [l[i] for i in pick] for l in lists]
        fl.adamw_step(*lists[:4], steps, exp_avg_scales=lists[4], exp_avg_sq_scales=lists[5],
                      grad_scale=torch.tensor(0.5, device=dev), **HYPER)

    steps = torch.arange(n, device=dev) % 50
    checked = sorted({*range(0, n, 97), 478, n - 1})
    lists = [p, g, m, v, *scales]
    alone = [None if l is None else [t.clone() for t in l] for l in lists]
    for i in checked:
        counter = steps[i:i + 1].clone()
        call([i], counter, alone)
        assert int(counter) == int(steps[i]) + 1
    call(range(n), steps, lists)
    assert torch.equal(steps, torch.arange(n, device=dev) % 50 + 1)
    for i in checked:
        for a, b in zip(lists, alone):
            assert a is None or torch.equal(a[i].view(torch.uint8), b[i].view(torch.uint8)), i
    for i in range(0, n, 5):  # the others are no longer what they were
        assert sizes[i] == 0 or not torch.equal(p[i], alone[0][i]) or i in checked


def test_one_tensor_of_the_most_values(dev):
    """2^34 bf16 values with 8-bit states (106 GB): as many blocks as a launch takes, behind a small tensor's own."""
    print("[case] adamw_step and grad_norm of 2^34 values", flush=True)
    n = 1 << 34
    if torch.cuda.mem_get_info()[0] < 130 << 30:
        torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 130 << 30:
        pytest.skip("needs 130 GiB of free device memory")
    at = torch.tensor([0, 1, (1 << 31) - 1, 1 << 32, (1 << 33) + 255, n - 257, n - 1], device=dev)
    vals = torch.tensor([2.0, 1.0, -1.0, 3.0, -2.0, 0.5, 4.0], device=dev).bfloat16()
    p, g = (torch.zeros(n, device=dev, dtype=torch.bfloat16) for _ in range(2))
    m, v = (torch.zeros(n, device=dev, dtype=torch.uint8).view(STATE8_DTYPE) for _ in range(2))
    ms, vs = (torch.zeros(n // 256, device=dev) for _ in range(2))
    p[at], g[at] = -vals, vals
    small = [torch.ones(3, device=dev, dtype=torch.bfloat16) for _ in range(2)]
    codes = [torch.zeros(3, device=dev, dtype=torch.uint8).view(STATE8_DTYPE) for _ in range(2)]
    tops = [torch.zeros(1, device=dev) for _ in range(2)]
    norm = math.sqrt(float(vals.double().square().sum()) + 3)
    assert abs(float(fl.grad_norm([small[1], g])) - norm) <= 2 * U * norm
    hyper = {**HYPER, "lr": 0.1}
    fl.adamw_step([small[0], p], [small[1], g], [codes[0], m], [codes[1], v], torch.zeros(2, dtype=torch.long, device=dev),
                  exp_avg_scales=[tops[0], ms], exp_avg_sq_scales=[tops[1], vs], **hyper)
    exp, tol = exact(-vals, vals, *(torch.zeros(7, device=dev) for _ in range(2)), 1, **hyper)
    near(p[at], exp[0], tol[0], "p")
    held = m[at].float() * ms[at // 256]
    assert bool(((held - 0.1 * vals.float()).abs() <= 2.0 ** -4 * 0.1 * vals.float().abs() + 1e-6).all())
    assert bool((small[0] != 1).all())
    assert sum(int(c.count_nonzero()) for c in p.split(1 << 31)) == 7
    assert sum(int(c.count_nonzero()) for c in m.view(torch.uint8).split(1 << 31)) == 7 == int(ms.count_nonzero()) + 1
    del p, g, m, v, ms, vs
    torch.cuda.empty_cache()
