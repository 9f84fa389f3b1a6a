"""GPU: the gated scan and its gradients against 64-bit formulas.

u = 2^-24. With H the scan of magnitudes (|a|, |u|, |h_-1|), a step rounds its product and its sum: 2 u H_t, carried on by
the gates after it. A tile composed of maps rounds the product of up to 256 gates once each: 256 u of what enters the
tile, which is at most H there, and the same again where a step's value is formed from the tile's start. So
    E = scan(|a|, 2 u H + [first step of a tile] 260 u H) + 260 u H.
The reverse recurrence has the same bound with G, the reverse scan of |dh|. da = g h_-1: E_g |h| + G E_h + u G H, and a sum
over C channels C roundings of the sum of those magnitudes. A result in bf16 is rounded once: half a step.
"""
from __future__ import annotations

import pytest
import torch

import fields_lm_amd as fl
from fields_lm_amd._train import gated_scan_ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16
TILE = 256


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm device")
    return torch.device("cuda:0")


def half_step(dtype):
    return 0.0 if dtype == F32 else torch.finfo(dtype).eps / 2


def scan64(a, u, first):
    h, now = torch.empty_like(u), first
    for t in range(u.shape[1]):
        now = a[:, t] * now + u[:, t]
        h[:, t] = now
    return h


def carried(a, e, H):
    """Errors e added at every step, and a tile's, carried on by the gates."""
    add = 2 * U * H + e
    add[:, ::TILE] += 260 * U * H[:, ::TILE]
    return scan64(a.abs(), add, torch.zeros_like(H[:, 0])) + 260 * U * H


def expected(gate, drive, first, g_out, g_last):
    """(value, bound) of out, state, and the gradients of gate, drive and state."""
    a = gate.double()
    token = a.ndim == 2
    a = (a[..., None] if token else a).expand(drive.shape)
    u = drive.double()
    start = torch.zeros_like(u[:, 0]) if first is None else first.double()
    h, H = scan64(a, u, start), scan64(a.abs(), u.abs(), start.abs())
    E = carried(a, 0.0, H)
    out = {"out": (h, E + half_step(drive.dtype) * h.abs()), "state": (h[:, -1], E[:, -1])}
    dh = torch.zeros_like(u) if g_out is None else g_out.double()
    last = torch.zeros_like(start) if g_last is None else g_last.double()
    after = torch.cat((torch.ones_like(a[:, :1]), a.flip(1)[:, :-1]), 1)
    g = scan64(after, dh.flip(1), last)
    G = scan64(after.abs(), dh.abs().flip(1), last.abs())
    # tiles lie from the start, so that their ends come at any place of the reversed steps: a tile's error at every step
    # that could be one would be far too much, so it is added where they are
    add = 2 * U * G
    ends = torch.zeros(u.shape[1], dtype=torch.bool, device=u.device)
    ends[TILE - 1::TILE] = True
    ends[-1] = True
    add += 260 * U * G * ends.flip(0)[None, :, None]
    Eg = (scan64(after.abs(), add, torch.zeros_like(start)) + 260 * U * G).flip(1)
    g, G = g.flip(1), G.flip(1)
    before = torch.cat((start[:, None], h[:, :-1]), 1)
    Hb = torch.cat((start.abs()[:, None], H[:, :-1]), 1)
    Eb = torch.cat((torch.zeros_like(start)[:, None], E[:, :-1]), 1)
    da, Ea = g * before, Eg * Hb + G * (Eb + 260 * U * Hb) + U * G * Hb
    if token:
        Ea = Ea.sum(-1) + drive.shape[2] * U * (G * Hb).sum(-1)
        da = da.sum(-1)
    out["gate"] = (da, Ea + half_step(gate.dtype) * da.abs())
    out["drive"] = (g, Eg + half_step(drive.dtype) * g.abs())
    s = a[:, 0] * g[:, 0]
    out["state_in"] = (s, a[:, 0].abs() * Eg[:, 0] + 260 * U * (a[:, 0].abs() * G[:, 0]))
    return out


def close(got, pair, what):
    value, bound = pair
    assert got.shape == value.shape, (what, got.shape, value.shape)
    far = (got.double() - value).abs() - bound - 1e-38
    assert bool((far <= 0).all()), (what, float(far.max()))


def inputs(dev, B, T, C, token, gt, dt, state, seed, low=0.0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    shape = (B, T) if token else (B, T, C)
    gate = torch.sigmoid(3 + 2 * torch.randn(shape, device=dev, generator=gen))
    gate = torch.where(torch.rand(shape, device=dev, generator=gen) < 0.02, low, gate)
    gate = torch.where(torch.rand(shape, device=dev, generator=gen) < 0.02, 1.0, gate)
    gate = torch.where(torch.rand(shape, device=dev, generator=gen) < 0.1, -gate, gate)
    drive = torch.randn(B, T, C, device=dev, generator=gen)
    first = torch.randn(B, C, device=dev, generator=gen) * 3 if state else None
    g_out = torch.randn(B, T, C, device=dev, generator=gen).to(dt)
    g_last = torch.randn(B, C, device=dev, generator=gen)
    return gate.to(gt), drive.to(dt), first, g_out, g_last


SHAPES = [(70_001, 2, 3), (1, 8, 70), (2, 9, 70), (1, 1, 1), (64, 1, 96), (2, 2, 3), (3, 15, 5), (1, 16, 64), (2, 17, 65), (1, 63, 7), (2, 64, 64), (1, 65, 130),
          (3, 255, 31), (1, 256, 4), (2, 257, 66), (1, 300, 1), (2, 511, 62), (1, 513, 257), (3, 1025, 64), (1, 4099, 33),
          (2, 2048, 192)]


@pytest.mark.parametrize("types", [(F32, F32), (F32, BF16), (BF16, F32), (BF16, BF16)], ids=str)
@pytest.mark.parametrize("token", [False, True])
@pytest.mark.parametrize("B,T,C", SHAPES, ids=str)
def test_scan_and_gradients(dev, B, T, C, token, types):
    state = (T + C) % 2 == 0
    print(f"[case] gated_scan {B}x{T}x{C} token={token} {types} state={state}", flush=True)
    gate, drive, first, g_out, g_last = inputs(dev, B, T, C, token, *types, state, B + T + C)
    exp = expected(gate, drive, first, g_out, g_last)
    out, last = fl.gated_scan(gate, drive, first, return_state=True)
    assert out.dtype == drive.dtype and last.dtype == F32
    close(out, exp["out"], "out")
    close(last, exp["state"], "state")
    assert torch.equal(fl.gated_scan(gate, drive, first), out)
    leaves = [t.detach().requires_grad_() for t in (gate, drive, first) if t is not None]
    out2, last2 = fl.gated_scan(*leaves, return_state=True)
    assert torch.equal(out2.detach(), out) and torch.equal(last2.detach(), last)
    got = torch.autograd.grad([out2, last2], leaves, [g_out, g_last], retain_graph=True)
    for name, g, leaf in zip(("gate", "drive", "state_in"), got, leaves):
        assert g.dtype == leaf.dtype
        close(g, exp[name], name)
    again = torch.autograd.grad([out2, last2], leaves, [g_out, g_last])
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("T,C", [(40, 70), (600, 70), (5000, 8)])
@pytest.mark.parametrize("token", [False, True])
def test_one_upstream_gradient_and_frozen_inputs(dev, token, T, C):
    print(f"[case] gated_scan, one upstream gradient, T={T} token={token}", flush=True)
    gate, drive, first, g_out, g_last = inputs(dev, 2, T, C, token, F32, F32, True, T)
    for up in ((g_out, None), (None, g_last)):
        exp = expected(gate, drive, first, *up)
        for frozen in (None, 0, 1, 2):
            leaves = [t.detach().requires_grad_(i != frozen) for i, t in enumerate((gate, drive, first))]
            outs = fl.gated_scan(*leaves, return_state=True)
            wanted = [t for t in leaves if t.requires_grad]
            i = 0 if up[0] is not None else 1
            got = torch.autograd.grad(outs[i], wanted, up[i])
            names = [n for j, n in enumerate(("gate", "drive", "state_in")) if j != frozen]
            for name, g in zip(names, got):
                close(g, exp[name], (name, frozen))


@pytest.mark.parametrize("T", [1000, 70_001])
def test_long(dev, T):
    print(f"[case] gated_scan T={T}", flush=True)
    gate, drive, first, g_out, g_last = inputs(dev, 1, T, 5, False, F32, F32, True, 11)
    gate = 1.0 - (1.0 - gate.abs()) * 1e-3  # memories of thousands of steps
    gate[0, 700] = 0.0
    exp = expected(gate, drive, first, g_out, g_last)
    leaves = [t.detach().requires_grad_() for t in (gate, drive, first)]
    out, last = fl.gated_scan(*leaves, return_state=True)
    close(out.detach(), exp["out"], "out")
    close(last.detach(), exp["state"], "state")
    got = torch.autograd.grad([out, last], leaves, [g_out, g_last])
    for name, g in zip(("gate", "drive", "state_in"), got):
        close(g, exp[name], name)


def test_many_chains(dev):
    """More chains of tiles than the card holds blocks."""
    print("[case] gated_scan, many chains", flush=True)
    gate, drive, first, g_out, g_last = inputs(dev, 9, 700, 2000, False, F32, BF16, True, 12)
    exp = expected(gate, drive, first, g_out, g_last)
    leaves = [t.detach().requires_grad_() for t in (gate, drive, first)]
    for _ in range(3):
        out, last = fl.gated_scan(*leaves, return_state=True)
        close(out.detach(), exp["out"], "out")
        got = torch.autograd.grad([out, last], leaves, [g_out, g_last])
        for name, g in zip(("gate", "drive", "state_in"), got):
            close(g, exp[name], name)


def test_closed_gates_open_gates_and_the_split(dev):
    """A gate of 0 starts anew, bit for bit; of 1 without drive passes the state on; two calls carry on as one."""
    print("[case] gated_scan, closed and open gates", flush=True)
    gate, drive, first, _, _ = inputs(dev, 2, 900, 40, False, F32, F32, True, 13)
    gate[:, 300] = 0.0
    out = fl.gated_scan(gate, drive, first)
    assert torch.equal(out[:, 300], drive[:, 300])
    other = fl.gated_scan(gate, drive, first + 5)
    assert torch.equal(out[:, 300:], other[:, 300:])
    ones, none = torch.ones(2, 900, device=dev), torch.zeros_like(drive)
    held, last = fl.gated_scan(ones, none, first, return_state=True)
    assert torch.equal(held, first[:, None].expand_as(held)) and torch.equal(last, first)
    a, mid = fl.gated_scan(gate[:, :256], drive[:, :256], first, return_state=True)
    b = fl.gated_scan(gate[:, 256:], drive[:, 256:], mid)
    exp = expected(gate, drive, first, None, None)["out"]
    close(torch.cat((a, b), 1), exp, "split")


def test_strides(dev):
    """Column slices of one projection, [B, T, 1] gates, expanded and transposed tensors, negated memory."""
    print("[case] gated_scan, strides", flush=True)
    gen = torch.Generator(device=dev).manual_seed(14)
    packed = torch.rand(3, 270, 2 * 37 + 3, device=dev, generator=gen)
    g, d = packed[..., 1:38], packed[..., 38:75]
    wide = torch.rand(270, 3, 37, device=dev, generator=gen)
    first = torch.randn(37, 3, device=dev, generator=gen).t()
    up = torch.randn(270, 3, 37, device=dev, generator=gen).transpose(0, 1)
    for gate, drive in ((g, d), (wide.transpose(0, 1), d), (g, wide.transpose(0, 1)), (g[..., :1], d), (g[..., 0], d),
                        (g[:, :1].expand_as(g), d), (g, d[:, :1].expand_as(d)), (torch._neg_view(g), torch._neg_view(d)),
                        (g[..., ::2][..., :18], d[..., ::2][..., :18]), (wide[..., 0].t(), d)):
        c = drive.shape[-1]
        f, w = first[:, :c], up[..., :c]
        flat = gate[..., 0] if gate.ndim == 3 and gate.shape[-1] == 1 else gate
        exp = expected(flat, drive, f, w, None)
        leaves = [t.detach().requires_grad_() for t in (gate, drive, f)]
        out = fl.gated_scan(*leaves)
        close(out.detach(), exp["out"], "out")
        got = torch.autograd.grad(out, leaves, w)
        close(got[0].reshape(flat.shape), exp["gate"], "gate")
        close(got[1], exp["drive"], "drive")
        close(got[2], exp["state_in"], "state_in")


def test_empty(dev):
    print("[case] gated_scan, empty", flush=True)
    state = torch.randn(2, 5, device=dev, requires_grad=True)
    out, last = fl.gated_scan(torch.rand(2, 0, device=dev), torch.rand(2, 0, 5, device=dev), state, return_state=True)
    assert out.shape == (2, 0, 5) and torch.equal(last, state)
    got, = torch.autograd.grad(last.sum(), state)
    assert bool((got == 1).all())
    out, last = fl.gated_scan(torch.rand(0, 4, 5, device=dev), torch.rand(0, 4, 5, device=dev), return_state=True)
    assert out.shape == (0, 4, 5) and last.shape == (0, 5)
    for shape in ((2, 0, 5), (2, 0)):
        gate, drive = torch.rand(shape, device=dev, requires_grad=True), torch.rand(2, 0, 5, device=dev, requires_grad=True)
        got = torch.autograd.grad(fl.gated_scan(gate, drive).sum(), (gate, drive))
        assert got[0].shape == shape and got[1].shape == (2, 0, 5)


def test_special_values(dev):
    """NaN and infinities reach what comes after them in their channel, up to a closed gate's product with them."""
    print("[case] gated_scan, special values", flush=True)
    gate, drive = torch.full((1, 700, 9), 0.5, device=dev), torch.ones(1, 700, 9, device=dev)
    drive[0, 290, 2], drive[0, 310, 4] = float("nan"), float("inf")
    out = fl.gated_scan(gate, drive)
    assert bool(out[0, 290:, 2].isnan().all()) and bool(out[0, :290].isfinite().all())
    assert bool((out[0, 310:, 4] == float("inf")).all())
    out[0, :, 2] = out[0, :, 4] = 0
    assert bool(out.isfinite().all())


@pytest.mark.parametrize("token", [False, True])
def test_same_bits(dev, token):
    """Wherever a tile finds the state that enters it, the results are the same bits."""
    print(f"[case] gated_scan, same bits, token={token}", flush=True)
    gate, drive, first, g_out, g_last = inputs(dev, 3, 9000, 300, token, F32, F32, True, 16)
    gate = 1.0 - (1.0 - gate.abs()) * 1e-3
    leaves = [t.detach().requires_grad_() for t in (gate, drive, first)]
    busy = torch.randn(2048, 2048, device=dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    kept = None
    for i in range(12):
        if i % 3:
            with torch.cuda.stream(side):  # other work takes some of the card
                for _ in range(i):
                    busy.mm(busy)
        out, last = fl.gated_scan(*leaves, return_state=True)
        got = [out.detach(), last.detach(), *torch.autograd.grad([out, last], leaves, [g_out, g_last])]
        kept = kept or got
        assert all(torch.equal(a, b) for a, b in zip(got, kept))
    torch.cuda.synchronize()


def test_states_of_zero_before_growing_gates(dev):
    """A state of 0 stays 0 whatever the product of the gates behind it; products over several tiles may overflow."""
    print("[case] gated_scan, growing gates", flush=True)
    gate, drive = torch.full((1, 2000, 3), 2.0, device=dev), torch.zeros(1, 2000, 3, device=dev)
    drive[0, 1990] = 1.0
    leaves = [t.requires_grad_() for t in (gate, drive)]
    out = fl.gated_scan(*leaves)
    exp = torch.zeros_like(drive)
    exp[0, 1990:] = 2.0 ** torch.arange(10.0, device=dev)[:, None]
    assert torch.equal(out, exp)
    up = torch.zeros_like(drive)
    up[0, 5] = 1.0
    got = torch.autograd.grad(out, leaves, up)
    back = torch.zeros_like(drive)
    back[0, :6] = 2.0 ** torch.arange(5.0, -1.0, -1.0, device=dev)[:, None]
    assert torch.equal(got[1], back) and bool((got[0] == 0).all())
    # 2^-60 times 2^90 over 1,920 steps: the product over eight tiles is 2^90, over the steps after the first tile 2^78;
    # a gate of 2^(3 / 64) is off by a rounding a step, so that 1,920 steps are off by 1,920 * 2^-24 and their own roundings
    gate = torch.full((1, 1920), 2.0 ** (3 / 64), device=dev)
    first = torch.full((1, 3), 2.0 ** -60, device=dev)
    out, last = fl.gated_scan(gate, torch.zeros(1, 1920, 3, device=dev), first, return_state=True)
    assert bool(((last / 2.0 ** 30 - 1).abs() <= 1920 * 2.0 ** -22).all())


def gates(dev, T, *runs):
    """[1, T] of 1, but (from, to, value) for each of `runs`."""
    gate = torch.ones(1, T, device=dev)
    for lo, hi, value in runs:
        gate[:, lo:hi] = value
    return gate


# with a state of `size` before and a gradient of the last state of as much; every state, gradient and product of both is an
# ordinary number in fp32, the products of gates over a segment or a tile are not
RUNS = [(1e15, (3, 19, 1e-3)), (1e15, (250, 266, 1e-3)), (1e15, (3, 19, 1e-3), (300, 305, 1e3)),
        (1e15, (3, 19, 1e-3), (40, 45, 1e3)), (1e15, (3, 19, -1e-3), (530, 533, -1e3)), (1e-30, (3, 48, 10.0)),
        (1e-30, (3, 33, 10.0), (40, 55, -10.0)), (1e-30, (240, 285, 10.0))]


@pytest.mark.parametrize("token", [False, True])
@pytest.mark.parametrize("size,runs", [(r[0], r[1:]) for r in RUNS], ids=str)
def test_products_outside_fp32(dev, size, runs, token):
    print(f"[case] gated_scan, products of {runs} token={token}", flush=True)
    T, C = 700, 5
    gate = gates(dev, T, *runs)
    if not token:
        gate = gate[..., None].expand(1, T, C).contiguous()
    first = torch.linspace(0.5, 1.5, C, device=dev)[None] * size
    drive, g_out, g_last = torch.zeros(1, T, C, device=dev), torch.zeros(1, T, C, device=dev), first.flip(1)
    exp = expected(gate, drive, first, g_out, g_last)
    leaves = [t.detach().requires_grad_() for t in (gate, drive, first)]
    out, last = fl.gated_scan(*leaves, return_state=True)
    close(out.detach(), exp["out"], "out")
    close(last.detach(), exp["state"], "state")
    got = torch.autograd.grad([out, last], leaves, [g_out, g_last])
    for name, g in zip(("gate", "drive", "state_in"), got):
        close(g, exp[name], name)


@pytest.mark.parametrize("value", [1e-3, -1e-3, 1e-30])
def test_infinite_states_before_small_gates(dev, value):
    """Infinite step by step, also where a tile's product of gates is too small for any number; a finite state is gone."""
    print(f"[case] gated_scan, infinite states before gates of {value}", flush=True)
    gate, drive = torch.full((1, 700), value, device=dev), torch.ones(1, 700, 2, device=dev)
    first = torch.tensor([[float("inf"), 1e30]], device=dev)
    out, last = fl.gated_scan(gate, drive, first, return_state=True)
    sign = torch.full((700,), value, device=dev).sign().cumprod(0)
    assert torch.equal(out[0, :, 0], sign * float("inf")) and torch.equal(last[0, 0], out[0, -1, 0])
    exp = expected(gate, drive[..., 1:].contiguous(), first[:, 1:], None, None)
    close(out[..., 1:], exp["out"], "out")


def test_infinities_stay_in_their_channel(dev):
    """Bits of the channels beside an infinite state, forward and back."""
    print("[case] gated_scan, infinities beside", flush=True)
    gate, drive, first, g_out, g_last = inputs(dev, 2, 1500, 70, False, F32, F32, True, 51, low=1e-3)
    wild, wild_last = first.clone(), g_last.clone()
    wild[:, ::7], wild_last[:, ::7] = float("inf"), float("-inf")
    rest = torch.arange(70, device=dev) % 7 != 0
    kept = None
    for f, k in ((first, g_last), (wild, wild_last)):
        leaves = [t.detach().requires_grad_() for t in (gate, drive, f)]
        outs = fl.gated_scan(*leaves, return_state=True)
        got = [t[..., rest] for t in (*(o.detach() for o in outs), *torch.autograd.grad(outs, leaves, [g_out, k]))]
        kept = kept or got
        assert all(torch.equal(a, b) for a, b in zip(got, kept))


def test_many_sequences(dev):
    """More threads than one dimension of a launch holds: 2^23 chains of one tile back, 2^26 of one step forward."""
    print("[case] gated_scan, 2^23 + 5 sequences", flush=True)
    B = 2 ** 23 + 5
    gen = torch.Generator(device=dev).manual_seed(17)
    leaves = [torch.rand(shape, device=dev, generator=gen).requires_grad_() for shape in ((B, 1), (B, 1, 1), (B, 1))]
    out = fl.gated_scan(*leaves)
    exp = torch.addcmul(leaves[1].detach().double()[:, 0], leaves[0].detach().double(), leaves[2].detach().double())
    assert bool(((out.detach()[:, 0] - exp).abs() <= exp * 2.0 ** -24).all())
    got = torch.autograd.grad(out, leaves, torch.ones_like(out))
    assert torch.equal(got[0], leaves[2]) and bool((got[1] == 1).all()) and torch.equal(got[2], leaves[0])
    del leaves, out, exp, got
    print("[case] gated_scan, 2^24 sequences of 257 channels", flush=True)
    B, C = 2 ** 24, 257
    drive = torch.randn(2 ** 20, C, device=dev, dtype=BF16, generator=gen).repeat(B // 2 ** 20, 1).view(B, 1, C)
    out = fl.gated_scan(torch.rand(B, 1, device=dev, generator=gen), drive)
    assert torch.equal(out, drive)


def test_gradients_by_differences(dev):
    """The loss's quotient of differences, in a direction of each input. It is off by the outputs' roundings over the step,
    and by what the same quotient in 64 bits is off the derivative."""
    print("[case] gated_scan, differences", flush=True)
    gate, drive, first, w, _ = inputs(dev, 2, 9, 6, False, F32, F32, True, 15)
    leaves = [t.detach().requires_grad_() for t in (gate, drive, first)]
    got = torch.autograd.grad(fl.gated_scan(*leaves), leaves, w)
    gen = torch.Generator(device=dev).manual_seed(16)
    step = 2.0 ** -7
    for i, t in enumerate((gate, drive, first)):
        d = torch.randn(t.shape, device=dev, generator=gen)

        def moved(by):
            return [x + by * d if j == i else x for j, x in enumerate((gate, drive, first))]

        plus, minus = moved(step), moved(-step)
        quotient = float(((fl.gated_scan(*plus).double() - fl.gated_scan(*minus).double()) * w.double()).sum()) / (2 * step)
        exact = float(((scan64(*[x.double() for x in plus]) - scan64(*[x.double() for x in minus])) * w.double()).sum()) / (2 * step)
        E = sum(float((expected(*x, w, None)["out"][1] * w.abs()).sum()) for x in (plus, minus)) / (2 * step)
        exp = expected(gate, drive, first, w, None)[("gate", "drive", "state_in")[i]]
        slope = float((exp[0] * d.double()).sum())
        bound = E + abs(exact - slope) + float((exp[1] * d.double().abs()).sum())
        assert abs(float((got[i].double() * d.double()).sum()) - quotient) <= bound, i


@pytest.mark.parametrize("token", [False, True])
def test_differentiable_backward(dev, token):
    """Second derivatives, against the same in 64 bits on the CPU."""
    print(f"[case] gated_scan, create_graph token={token}", flush=True)
    gate, drive, first, w, _ = inputs(dev, 2, 12, 5, token, F32, F32, True, 17)

    def second(op, *ts):
        leaves = [t.detach().requires_grad_() for t in ts]
        out = op(*leaves)
        grads = torch.autograd.grad((out * w.to(out)).sum(), leaves, create_graph=True)
        return torch.autograd.grad(sum((g.square()).sum() for g in grads), leaves)

    got = second(lambda a, u, s: fl.gated_scan(a, u, s), gate, drive, first)

    def ops(a, u, s):
        h, now = [], s
        for t in range(u.shape[1]):
            now = (a[:, t, None] if a.ndim == 2 else a[:, t]) * now + u[:, t]
            h.append(now)
        return torch.stack(h, 1)

    exp = second(ops, *[t.double().cpu() for t in (gate, drive, first)])
    # magnitudes: the same with everything positive; stock operations round a few hundred times
    size = second(ops, *[t.double().abs().cpu() for t in (gate, drive, first)])
    w = w.abs()
    size = second(ops, *[t.double().abs().cpu() for t in (gate, drive, first)])
    for a, b, s in zip(got, exp, size):
        assert bool(((a.double().cpu() - b).abs() <= 400 * U * (s.abs() + 1)).all())


@pytest.mark.parametrize("types", [(F32, F32), (BF16, F32), (F32, BF16)], ids=str)
@pytest.mark.parametrize("token", [False, True])
def test_differentiable_backward_over_tiles(dev, token, types):
    """First derivatives of a backward with create_graph, by the bounds of an ordinary one: many tiles; and gates above 1
    whose products leave fp32, with states of 0 and gradients that end early."""
    print(f"[case] gated_scan, create_graph over tiles, token={token} {types}", flush=True)
    for state in (False, True):
        gate, drive, first, g_out, g_last = inputs(dev, 2, 1300, 9, token, *types, state, 41)
        exp = expected(gate, drive, first, g_out, g_last)
        leaves = [t.detach().requires_grad_() for t in (gate, drive, first) if t is not None]
        outs = fl.gated_scan(*leaves, return_state=True)
        got = torch.autograd.grad(outs, leaves, [g_out, g_last], create_graph=True)
        for name, g, leaf in zip(("gate", "drive", "state_in"), got, leaves):
            assert g.dtype == leaf.dtype and g.shape == leaf.shape and g.requires_grad
            close(g.detach(), exp[name], name)
    T = 2500
    for value in (1.05, 2.0):
        gate = torch.full((1, T) if token else (1, T, 3), value, device=dev, dtype=types[0], requires_grad=True)
        drive = torch.zeros(1, T, 3, device=dev, dtype=types[1])
        drive[:, T - 10:] = 0.5
        drive.requires_grad_()
        up = torch.zeros(1, T, 3, device=dev, dtype=types[1])
        up[:, 5] = 1.0
        exp = expected(gate.detach(), drive.detach(), None, up, None)
        got = torch.autograd.grad(fl.gated_scan(gate, drive), (gate, drive), up, create_graph=True)
        for name, g in zip(("gate", "drive"), got):
            close(g.detach(), exp[name], name)


@pytest.mark.parametrize("token", [False, True])
def test_second_derivatives_over_tiles(dev, token):
    """Of a sum of weighted gradients, against the same in 64 bits on the CPU; bounds as test_differentiable_backward's."""
    print(f"[case] gated_scan, second derivatives over tiles, token={token}", flush=True)
    gate, drive, first, w, _ = inputs(dev, 1, 530, 3, token, F32, F32, True, 42)
    gen = torch.Generator(device=dev).manual_seed(43)
    weights = [torch.randn(t.shape, device=dev, generator=gen) for t in (gate, drive, first)]

    def second(op, ts, w, weights):
        leaves = [t.detach().requires_grad_() for t in ts]
        grads = torch.autograd.grad((op(*leaves) * w).sum(), leaves, create_graph=True)
        return torch.autograd.grad(sum((g * v).sum() for g, v in zip(grads, weights)), leaves[:2])

    def ops(a, u, s):
        h, now = [], s
        for t in range(u.shape[1]):
            now = (a[:, t, None] if a.ndim == 2 else a[:, t]) * now + u[:, t]
            h.append(now)
        return torch.stack(h, 1)

    got = second(fl.gated_scan, (gate, drive, first), w, weights)
    args = [[t.double().cpu() for t in x] if isinstance(x, list) else x.double().cpu()
            for x in ([gate, drive, first], w, weights)]
    exp = second(ops, *args)
    size = second(ops, *[[t.abs() for t in x] if isinstance(x, list) else x.abs() for x in args])
    # four scans behind each other, each with 2 x 260 u of a tile and as many tiles as three: 4 * 3 * 520 u of the magnitudes
    for a, b, s in zip(got, exp, size):
        assert bool(((a.double().cpu() - b).abs() <= 6240 * U * (s.abs() + 1)).all())


def test_stock_form(dev):
    print("[case] gated_scan, stock form", flush=True)
    for token in (False, True):
        gate, drive, first, _, _ = inputs(dev, 2, 300, 7, token, F32, F32, True, 18)
        out, last = gated_scan_ops(gate, drive, first)
        exp = expected(gate, drive, first, None, None)
        # doubling rounds products of runs of gates, at most once a round and gate: the bound's 260 u covers its 300
        close(out, (exp["out"][0], 2 * exp["out"][1]), "out")
        close(last, (exp["state"][0], 2 * exp["state"][1]), "state")


def test_captured_in_a_graph(dev):
    print("[case] gated_scan, graph", flush=True)
    data = inputs(dev, 2, 1500, 70, False, F32, F32, True, 19)
    gate, drive, first, g_out, g_last = data
    leaves = [t.requires_grad_() for t in (gate, drive, first)]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.autograd.grad(fl.gated_scan(*leaves, return_state=True), leaves, [g_out, g_last])
    torch.cuda.synchronize()
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = fl.gated_scan(*leaves, return_state=True)
        grads = torch.autograd.grad(outs, leaves, [g_out, g_last])
    with torch.cuda.graph(second, stream=side, pool=graph.pool()):
        outs2 = fl.gated_scan(gate.detach(), drive.detach(), first.detach(), return_state=True)
    for i in range(4):
        fresh = inputs(dev, 2, 1500, 70, False, F32, F32, True, 20 + i)
        with torch.no_grad():
            for to, x in zip(data, fresh):
                to.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        exp = expected(*fresh)
        close(outs[0].detach(), exp["out"], "out")
        for name, g in zip(("gate", "drive", "state_in"), grads):
            close(g, exp[name], name)
        second.replay()
        torch.cuda.synchronize()
        close(outs2[0], exp["out"], "out of the second graph")


def test_two_streams_at_once(dev):
    print("[case] gated_scan, two streams", flush=True)
    sets = [inputs(dev, 1, 20_000, 64, False, F32, F32, True, 30 + i) for i in range(2)]
    want = []
    for gate, drive, first, g_out, g_last in sets:
        leaves = [t.detach().requires_grad_() for t in (gate, drive, first)]
        outs = fl.gated_scan(*leaves, return_state=True)
        want.append((outs, torch.autograd.grad(outs, leaves, [g_out, g_last], retain_graph=True)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        got = []
        for s, (gate, drive, first, g_out, g_last) in zip(streams, sets):
            with torch.cuda.stream(s):
                leaves = [t.detach().requires_grad_() for t in (gate, drive, first)]
                outs = fl.gated_scan(*leaves, return_state=True)
                got.append((outs, torch.autograd.grad(outs, leaves, [g_out, g_last], retain_graph=True)))
        torch.cuda.synchronize()
        for (o, g), (o2, g2) in zip(got, want):
            assert all(torch.equal(a, b) for a, b in zip((*o, *g), (*o2, *g2)))


def test_a_captured_backward_refuses_leaves_of_the_default_stream(dev):
    print("[case] gated_scan, capture beside an eager graph", flush=True)
    gate = torch.rand(2, 30, 4, device=dev, requires_grad=True)
    drive = torch.rand(2, 30, 4, device=dev)
    eager = fl.gated_scan(gate, drive)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with pytest.raises(RuntimeError, match="default stream"):
        with torch.cuda.graph(graph, stream=side):
            torch.autograd.grad(fl.gated_scan(gate, drive).sum(), gate)
    torch.cuda.synchronize()
    eager.sum().backward()
    assert bool(gate.grad.isfinite().all())


def test_refuses(dev):
    print("[case] gated_scan, refusals", flush=True)
    g, d, s = torch.rand(2, 5, 3, device=dev), torch.rand(2, 5, 3, device=dev), torch.rand(2, 3, device=dev)
    for bad in ((g.half(), d, s), (g, d.double(), s), (g, d, s.bfloat16()), (None, d), (g, d, 3.0)):
        with pytest.raises(TypeError):
            fl.gated_scan(*bad)
    for bad in ((g[:, :4], d), (g[..., :2], d), (g[0], d), (g, d[0]), (g, d, s[:1]), (g.cpu(), d), (g, d, s.cpu())):
        with pytest.raises(ValueError):
            fl.gated_scan(*bad)
    with pytest.raises(RuntimeError):
        torch.jit.trace(lambda x: fl.gated_scan(x, d), g)
