"""GPU: orthogonalization and the Muon step against 64-bit formulas.

How far a result may be off, in the Frobenius norm, u = 2^-24: an operand is held in 22 bits (2^-23 of it at most, and as
much for the product of both low parts that is left out: 2^-21 a product) and summed in fp32 over K terms, whose roundings
add up as sqrt(K) u does (they have no common sign). A step's factor Q(A) = P_k .. P_1 of a stage moves X by at most
D |E| where E is A's error and D the largest |Q[l, m]| sqrt(m) of divided differences over A's eigenvalues l, m, taken from a
grid below; the stages after it multiply that by at most the largest slope of theirs. A stage's own products of squares
(four a step) carry the same relative error each, which that slope covers too. Eigenvalues reach 1 in the first stage and
the square of what the steps before leave (1.21^2) behind it. |A| is at most |X|^2, which is 1 at first and m behind.
"""
from __future__ import annotations

import copy
import math

import pytest
import torch

import fields_lm_amd as fl

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16
ABC = (3.4445, -4.7750, 2.0315)


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm device")
    return torch.device("cuda:0")


def half_step(dtype):
    return 0.0 if dtype == F32 else torch.finfo(dtype).eps / 2


def polar64(x, steps=5, abc=ABC, eps=1e-7):
    a, b, c = abc
    x = x.double()
    tall = x.shape[-2] > x.shape[-1]
    x = (x.mT if tall else x).contiguous()
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    for _ in range(steps):
        gram = x @ x.mT.contiguous()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.mT if tall else x


def stages(steps, most=3):
    n = -(-steps // most)
    out, left = [], steps
    for i in range(n):
        out.append(-(-left // (n - i)))
        left -= out[-1]
    return out


def growth(abc, steps):
    """Of every stage: D, the slope, the norm's bound before it."""
    a, b, c = abc
    out, top = [], 1.0
    for k in stages(steps):
        lam = torch.cat((torch.zeros(1, dtype=torch.float64), torch.logspace(-9, 0, 600, dtype=torch.float64) * top ** 2))

        def run(l):
            q = torch.ones_like(l)
            for _ in range(k):
                p = a + b * l + c * l * l
                q, l = q * p, l * p * p
            return q, l

        q, after = run(lam)
        diff = (q[:, None] - q[None, :]).abs() / (lam[:, None] - lam[None, :]).abs().clamp_min(1e-30)
        diff.fill_diagonal_(0.0)
        out.append((float((diff * lam.sqrt()[None, :]).max()), float(q.abs().max()), top))
        top = max(1.0, float(after.sqrt().max()))
    return out


def allowed(m, n, steps=5, abc=ABC):
    """Of the Frobenius norm of the result's error."""
    g, err = growth(abc, steps), 0.0
    for i, (d, slope, top) in enumerate(g):
        norm = 1.0 if i == 0 else top * math.sqrt(m)
        e = (2.0 ** -21 + math.sqrt(n) * U) * norm * top      # A = X X^T: |X| of the Frobenius norm, |X| of the spectral one
        e += 4 * stages(steps)[i] * (2.0 ** -21 + math.sqrt(m) * U) * norm * top
        err = err * slope + d * e + (2.0 ** -21 + math.sqrt(m) * U) * slope * norm
    return err


def check(got, x, steps=5, abc=ABC, eps=1e-7):
    exp = polar64(x, steps, abc, eps)
    m, n = min(x.shape[-2:]), max(x.shape[-2:])
    off = (got.double() - exp).square().sum((-2, -1)).sqrt()
    size = exp.square().sum((-2, -1)).sqrt()
    assert bool((off <= allowed(m, n, steps, abc) + half_step(got.dtype) * size).all()), (off, size)


def matrices(dev, shape, seed, kind="rows"):
    gen = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(shape, device=dev, generator=gen)
    if kind == "rows":
        x = x * torch.exp(0.7 * torch.randn(*shape[:-1], 1, device=dev, generator=gen))
    if kind == "low":
        r = min(4, *shape[-2:])
        x = 0.03 * x + torch.matmul(torch.randn(*shape[:-1], r, device=dev, generator=gen),
                                    torch.randn(*shape[:-2], r, shape[-1], device=dev, generator=gen))
    return x


SHAPES = [(1, 1), (1, 9), (9, 1), (2, 2), (7, 5), (31, 33), (32, 64), (33, 200), (64, 64), (65, 127), (128, 128), (129, 129),
          (130, 60), (200, 1001), (257, 255), (384, 128), (256, 632), (640, 640), (1000, 301)]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_orthogonalize(dev, shape, dtype):
    print(f"[case] orthogonalize {shape} {dtype}", flush=True)
    for i, kind in enumerate(("plain", "rows", "low")):
        x = matrices(dev, shape, i, kind).to(dtype)
        got = fl.orthogonalize(x)
        assert got.shape == x.shape and got.dtype == dtype
        check(got, x)
        assert torch.equal(fl.orthogonalize(x), got)


def test_as_near_as_steps_in_fp32(dev):
    """Nearer than eight times what the same steps on X in fp32 are off (numerical experiment: a stage of A's own steps
    loses up to a factor of four on them)."""
    print("[case] orthogonalize, beside fp32", flush=True)
    for shape in ((256, 640), (500, 512)):
        for kind in ("plain", "rows", "low"):
            x = matrices(dev, shape, 3, kind)
            exp = polar64(x)
            y = x / (x.norm() + 1e-7)
            for _ in range(5):
                gram = y @ y.t()
                y = ABC[0] * y + (ABC[1] * gram + ABC[2] * (gram @ gram)) @ y
            stock = float((y.double() - exp).norm())
            assert float((fl.orthogonalize(x).double() - exp).norm()) <= 8 * stock + 1e-6 * float(exp.norm())


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 6, 7, 10])
@pytest.mark.parametrize("abc", [ABC, (1.5, -0.5, 0.0), (1.875, -1.25, 0.375), (2.0, -1.5, 0.5)], ids=str)
def test_steps_and_coefficients(dev, steps, abc):
    print(f"[case] orthogonalize, {steps} steps of {abc}", flush=True)
    for shape in ((40, 90), (150, 140)):
        x = matrices(dev, shape, steps, "plain")
        check(fl.orthogonalize(x, steps=steps, coefficients=abc), x, steps, abc)


def divided(fn, l):
    """|fn[l_i, l_j]|, the divided differences of a polynomial; its slope where two are close."""
    f, d = fn(l), l[:, None] - l[None, :]
    close = d.abs() < 1e-6 * l.abs().max()
    mid, h = (l[:, None] + l[None, :]) / 2, 1e-5 * l.abs().max()
    slope = (fn(mid + h) - fn(mid - h)) / (2 * h)
    return torch.where(close, slope, (f[:, None] - f[None, :]) / torch.where(close, 1.0, d)).abs()


def held(k):
    """Of a product over k terms, relative to |L| |R| (one of them the Frobenius, one the spectral norm): what is stored of it
    is two parts of 11 bits, 2^-22 off at most; the product of both low parts, left out, is as much; sums in fp32 are off
    by sqrt(k) u and their scales by 4 u. Mirroring half a square makes that sqrt(2) as much at most."""
    return 1.5 * (2.0 ** -21 + (math.sqrt(k) + 4) * U)


def off_at_most(x, steps, abc, eps=1e-7):
    """Of the Frobenius norm of one matrix's error, to first order, from its own singular values s; l = s^2. Everything of a
    stage is a function of A, so that in A's eigenvectors an error E of what is held passes on entry by entry: that of A with
    the divided differences of the factor still to come, times q s, what it meets on its right; that of a step's P as
    itself in the product of the factors and as A P E + E P A in the next A; that of X by those of s -> Q(s^2) s, which
    are, of a matrix that is not symmetric, (f_i - f_j) / (s_i - s_j), (f_i + f_j) / (s_i + s_j) and f_i / s_i."""
    # (a stage has one step where the short side of an fp32 matrix is below 256, at most three elsewhere)
    a, b, c = abc
    m, n = min(x.shape), max(x.shape)
    s = torch.linalg.svdvals(x.double().cpu())
    s = s / (s.square().sum().sqrt() + eps)

    def p(l):
        return a + b * l + c * l * l

    def factor(k):  # of k steps, from A's eigenvalues before them
        def q(l):
            out = torch.ones_like(l)
            for _ in range(k):
                out, l = out * p(l), l * p(l) ** 2
            return out
        return q

    def size(v):
        return float(v.square().sum().sqrt())

    def top(v):
        return float(v.abs().max())

    err = 0.0
    for k in stages(steps, 1 if x.dtype == F32 and m < 256 else 3):
        l, q = s * s, torch.ones_like(s)
        f = factor(k)(l) * s
        plus = (f[:, None] + f[None, :]) / (s[:, None] + s[None, :]).clamp_min(1e-300)
        of_x = max(top(divided(lambda t: factor(k)(t * t) * t, s)), top(plus), top(factor(k)(l)))
        total = of_x * (err + 2.0 ** -22 * size(s))
        e_a = held(n) * size(s) * top(s)
        for e in range(k):
            total += float((divided(factor(k - e), l) * (q * s).abs()[None, :]).max()) * e_a
            pl = p(l)
            after = l * pl * pl
            rest = factor(k - e - 1)(after)
            e_p = (abs(c) * held(m) * size(l) * top(l) + 1.5 * 2.0 ** -21 * size(pl) +
                   4 * U * (abs(a) * math.sqrt(m) + abs(b) * size(l)))
            total += top(rest * q) * e_p * top(s)
            if e:
                total += held(m) * size(q) * top(pl) * top(rest) * top(s)  # the product of the factors, as it is held
            e_a = (2 * top(l) * top(pl) * e_p + held(m) * size(l) * top(pl) * top(pl) + held(m) * size(l * pl) * top(pl))
            q, l = q * pl, after
        err = total + held(m) * min(size(q) * top(s), top(q) * size(s))
        s = (q * s).abs()
    return err


def beyond(got, x, steps, abc):
    """How far a matrix is past that and its type's rounding, and both, relative to the result's norm."""
    exp = polar64(x, steps, abc)
    size, bound = float(exp.norm()), off_at_most(x, steps, abc)
    return float((got.double() - exp).norm()) / size - bound / size - half_step(got.dtype), bound / size


def spectrum(dev, shape, seed):
    """Singular values over six decades."""
    gen = torch.Generator(device="cpu").manual_seed(seed)
    m = min(shape)
    u, v = (torch.linalg.qr(torch.randn(k, m, generator=gen, dtype=torch.float64))[0] for k in shape)
    return ((u * torch.logspace(0, -6, m, dtype=torch.float64)) @ v.t()).float().to(dev)


ABCS = [ABC, (1.5, -0.5, 0.0), (1.875, -1.25, 0.375), (2.0, -1.5, 0.5)]
NEAR_SHAPES = [(1, 1), (1, 9), (9, 1), (7, 5), (33, 200), (130, 60), (257, 255), (640, 640), (1000, 301)]
# at most this much of the result, so that the bound says something: small singular values that the usual coefficients
# raise by 3.4 a step, over more than five steps, may end as far off as they are large
SAYS = 0.3


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 5, 6, 7, 10])
@pytest.mark.parametrize("abc", ABCS, ids=str)
def test_near_at_every_step(dev, steps, abc):
    print(f"[case] orthogonalize, by its own singular values: {steps} steps of {abc}", flush=True)
    tried = 0
    for shape in NEAR_SHAPES:
        for i, kind in enumerate(("plain", "rows", "low", "wide")):
            x = spectrum(dev, shape, steps) if kind == "wide" else matrices(dev, shape, 10 * steps + i, kind)
            for dtype in (F32, BF16):
                y = x.to(dtype)
                far, bound = beyond(fl.orthogonalize(y, steps=steps, coefficients=abc), y, steps, abc)
                assert far <= 0 or bound > SAYS, (shape, kind, dtype, far, bound)
                tried += bound <= SAYS
    assert tried >= (20 if steps > 7 and abc == ABC else 50)


def steps32(x, steps=5, abc=ABC):
    """The formula's steps on one X in fp32."""
    tall = x.shape[0] > x.shape[1]
    y = x.t().contiguous() if tall else x
    y = (y / (y.double().norm() + 1e-7)).float()
    for _ in range(steps):
        gram = y @ y.t()
        y = abc[0] * y + (abc[1] * gram + abc[2] * (gram @ gram)) @ y
    return y.t() if tall else y


@pytest.mark.parametrize("shape", [(8, 10), (18, 15), (24, 25), (33, 20), (65, 65), (100, 100), (11, 1286), (1654, 40), (160, 1900),
                                   (200, 200), (255, 300), (256, 256), (300, 1500), (700, 600)], ids=str)
def test_errors_are_those_of_steps_in_fp32(dev, shape):
    """In the mean square over matrices that look like gradients, at most twice as far as steps on X in fp32. What is held
    of a value is off by 0.35 of fp32's last place in the mean square (up to half of it, less where the low part is
    small) where fp32 is off by 0.29; a sum is rounded once to 16 terms where fp32's is to each; matrices of more
    than one step a stage are those whose sums, a few hundred terms at least, make up for what a stage adds."""
    print(f"[case] orthogonalize, errors beside fp32 {shape}", flush=True)
    gen = torch.Generator(device=dev).manual_seed(sum(shape))
    count = 32 if max(shape) < 300 else 6
    x = torch.randn(count, *shape, device=dev, generator=gen)
    x = x * torch.exp(0.5 * torch.randn(count, shape[0], 1, device=dev, generator=gen))
    x = x * torch.exp(0.5 * torch.randn(count, 1, shape[1], device=dev, generator=gen))
    x = x + 0.5 * torch.matmul(torch.randn(count, shape[0], 4, device=dev, generator=gen),
                               torch.randn(count, 4, shape[1], device=dev, generator=gen))
    got = fl.orthogonalize(x)
    own = stock = 0.0
    for i in range(count):
        exp = polar64(x[i])
        own += float(((got[i].double() - exp).norm() / exp.norm()) ** 2)
        stock += float(((steps32(x[i]).double() - exp).norm() / exp.norm()) ** 2)
    assert own <= 4 * stock, math.sqrt(own / stock)
    print(f"[measured] {math.sqrt(own / stock):.2f} of fp32's {math.sqrt(stock / count):.1e}", flush=True)


def test_results_are_a_matter_of_the_matrix_alone(dev):
    """In lists of long and short sides, in either tile, in fp32 and in bf16."""
    print("[case] muon_step, long and short sides", flush=True)
    shapes = [(255, 300), (256, 300), (300, 255), (40, 40), (257, 256), (1, 700), (0, 3), (1024, 1024)] + [(64, 200)] * 30
    for dtype in (F32, BF16):
        params, grads, bufs = model(dev, dtype, 21, shapes)
        before = [(p.clone(), b.clone()) for p, b in zip(params, bufs)]
        fl.muon_step(params, grads, bufs, lr=0.1)
        for (p, b), g, now, buf in zip(before, grads, params, bufs):
            fl.muon_step([p], [g], [b], lr=0.1)
            assert torch.equal(p, now) and torch.equal(b, buf)


@pytest.mark.parametrize("shape", [(3, 1024, 1100), (40, 300, 200), (18, 500, 130)], ids=str)
def test_near_in_large_tiles(dev, shape):
    """Enough matrices for tiles of 128; in bf16 each value is, besides, the nearest to one within the bound."""
    print(f"[case] orthogonalize, by their own singular values: {shape}", flush=True)
    x = matrices(dev, shape, 7)
    for steps in (5, 7):
        got = fl.orthogonalize(x, steps=steps)
        for i in range(shape[0]):
            far, bound = beyond(got[i], x[i], steps, ABC)
            assert far <= 0 and bound <= SAYS, (i, steps, far, bound)
    y = x.bfloat16()
    got = fl.orthogonalize(y)
    for i in range(shape[0]):
        exp = polar64(y[i])
        off = (got[i].double() - exp).abs()
        assert bool((off <= half_step(BF16) * exp.abs() + 1.01 * off_at_most(y[i], 5, ABC)).all())
    assert all(torch.equal(fl.orthogonalize(y), got) for _ in range(3))


def test_stacks_and_strides(dev):
    print("[case] orthogonalize, stacks and strides", flush=True)
    x = matrices(dev, (3, 2, 50, 70), 5)
    got = fl.orthogonalize(x)
    check(got, x)
    for i in range(3):
        for j in range(2):
            assert torch.equal(fl.orthogonalize(x[i, j]), got[i, j])
    for y in (x.mT, x[..., 1::2], x[:, :1, 3:], torch._neg_view(x), x.permute(2, 3, 0, 1)[..., 0].permute(2, 0, 1),
              x[0, 0].expand(3, 50, 70)):
        check(fl.orthogonalize(y), y)
    assert torch.allclose(fl.orthogonalize(x.mT), got.mT, rtol=0, atol=2 * allowed(50, 70))
    for shape in ((0, 5, 4), (3, 0, 4), (3, 4, 0)):
        assert fl.orthogonalize(torch.empty(shape, device=dev)).shape == shape
    wide = fl.orthogonalize(x.requires_grad_())
    assert not wide.requires_grad


@pytest.mark.parametrize("n", [63, 64, 65, 128, 4096, 4097, 10_000])
def test_many_matrices(dev, n):
    """A stack's matrices are found at any count of them, with one tile and with several to each."""
    for shape in ((5, 9), (65, 130)):
        print(f"[case] orthogonalize, {n} of {shape}", flush=True)
        x = matrices(dev, (n, *shape), n)
        got = fl.orthogonalize(x)
        check(got, x)
        for i in (0, 1, n // 2, n - 2, n - 1):
            assert torch.equal(fl.orthogonalize(x[i]), got[i])


def test_many_ragged_matrices(dev):
    print("[case] muon_step, 5,000 ragged matrices", flush=True)
    shapes = [(1 + i % 13, 1 + i * 7 % 90) for i in range(4990)] + [(140, 300)] * 10
    params, grads, bufs = model(dev, F32, 9, shapes)
    before = [p.clone() for p in params]
    fl.muon_step(params, grads, bufs, lr=0.5, weight_decay=0.0, momentum=0.0, nesterov=False)
    for i in (*range(0, 5000, 333), 4988, 4989, 4990, 4999):
        r, c = shapes[i]
        step = 0.5 * max(1.0, r / c) ** 0.5 * fl.orthogonalize(grads[i])
        # the parameter's rounding and that of r as it is multiplied
        assert torch.allclose(params[i], before[i] - step, rtol=2.0 ** -22, atol=2.0 ** -22)


def test_sizes_of_values(dev):
    """Zeros, large and small scales, a row or column alone, an identity; NaN and infinities spoil their matrix alone."""
    print("[case] orthogonalize, values", flush=True)
    x = matrices(dev, (60, 80), 6)
    for eps in (1e-7, 0.0):
        assert bool((fl.orthogonalize(torch.zeros(5, 60, 80, device=dev), eps=eps) == 0).all())
    base = fl.orthogonalize(x, eps=0.0)
    for scale in (2.0 ** 100, 2.0 ** -100):
        assert torch.equal(fl.orthogonalize(x * scale, eps=0.0), base)
    check(fl.orthogonalize(x * 1e-7), x * 1e-7)  # eps as large as the norm
    one = torch.zeros(60, 80, device=dev)
    one[7] = x[7]
    check(fl.orthogonalize(one), one)
    check(fl.orthogonalize(one.t()), one.t())
    check(fl.orthogonalize(torch.eye(130, device=dev)), torch.eye(130, device=dev))
    stack = x.repeat(4, 1, 1)
    stack[1, 3, 4], stack[2, 5, 6] = float("nan"), float("inf")
    got = fl.orthogonalize(stack)
    assert bool(got[1:3].isnan().all()) and torch.equal(got[0], got[3]) and bool(got[0].isfinite().all())


def model(dev, dtype, seed, shapes):
    gen = torch.Generator(device=dev).manual_seed(seed)

    def make(scale, t):
        return [(torch.randn(s, device=dev, generator=gen) * scale).to(t) for s in shapes]

    return make(0.05, dtype), make(1e-3, dtype), make(1e-3, F32)


SETS = [[(1, 1)], [(33, 70), (70, 33), (5, 5)], [(129, 64)] * 5 + [(64, 300)], [(30 + i % 7, 40 - i % 5) for i in range(150)],
        [(0, 4), (16, 16), (4, 0)], [(513, 257), (100, 700), (384, 128)]]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
@pytest.mark.parametrize("nesterov", [False, True])
@pytest.mark.parametrize("shapes", SETS, ids=lambda s: f"{len(s)}x{s[0]}")
def test_muon_step(dev, shapes, nesterov, dtype):
    print(f"[case] muon_step {shapes[:3]} nesterov={nesterov} {dtype}", flush=True)
    for adjust in ("original", "match_rms_adamw"):
        params, grads, bufs = model(dev, dtype, len(shapes), shapes)
        scale = torch.tensor(0.37, device=dev)
        before = [p.clone() for p in params], [b.clone() for b in bufs]
        versions = [p._version for p in params]
        fl.muon_step(params, grads, bufs, lr=0.02, momentum=0.9, nesterov=nesterov, weight_decay=0.1, adjust_lr=adjust,
                     grad_scale=scale)
        assert all(p._version > v for p, v in zip(params, versions))
        for p, g, b, p0, b0 in zip(params, grads, bufs, *before):
            g, b0 = g.double() * float(scale), b0.double()
            m = 0.9 * b0 + 0.1 * g
            bound = 5 * U * (0.9 * b0.abs() + 0.1 * g.abs())
            assert bool(((b.double() - m).abs() <= bound + 1e-38).all())
            if p.numel() == 0:
                continue
            # the rounding of what is orthogonalized is far below that of its operands, which `allowed` counts
            u = 0.1 * g + 0.9 * m if nesterov else m
            rows, cols = p.shape
            rate = 0.02 * (math.sqrt(max(1.0, rows / cols)) if adjust == "original" else 0.2 * math.sqrt(max(rows, cols)))
            exp = p0.double() * (1 - 0.02 * 0.1) - rate * polar64(u)
            off = rate * allowed(min(p.shape), max(p.shape)) + 4 * U * float(p0.double().norm() + rate * math.sqrt(min(p.shape)))
            off += half_step(dtype) * float(exp.norm())
            assert float((p.double() - exp).norm()) <= off


def test_muon_step_is_the_same_every_time_and_of_every_grouping(dev):
    """A matrix's result is its own: alone, among others, and where the list takes several groups of workspace."""
    print("[case] muon_step, grouping", flush=True)
    shapes = [(300, 200)] * 3 + [(2048, 4096)] * 8 + [(77, 130)]
    params, grads, bufs = model(dev, F32, 1, shapes)
    alone = [(p.clone(), b.clone()) for p, b in zip(params, bufs)]
    twice = [(p.clone(), b.clone()) for p, b in zip(params, bufs)]
    fl.muon_step(params, grads, bufs, lr=0.02)
    fl.muon_step([p for p, _ in twice], grads, [b for _, b in twice], lr=0.02)
    for i in (0, 2, 3, 10, 11):
        fl.muon_step([alone[i][0]], [grads[i]], [alone[i][1]], lr=0.02)
        assert torch.equal(alone[i][0], params[i]) and torch.equal(alone[i][1], bufs[i])
    assert all(torch.equal(a, p) and torch.equal(m, b) for (a, m), p, b in zip(twice, params, bufs))
    check((model(dev, F32, 1, shapes)[0][3] * (1 - 0.02 * 0.1) - params[3]) / 0.02,
          0.05 * grads[3].double() + 0.95 * (0.95 * model(dev, F32, 1, shapes)[2][3].double() + 0.05 * grads[3].double()))


def test_scales_that_are_not_finite_and_rates_on_the_device(dev):
    print("[case] muon_step, scales and rates", flush=True)
    for dtype in (F32, BF16):
        for bad in (float("nan"), float("inf"), float("-inf")):
            params, grads, bufs = model(dev, dtype, 2, [(40, 50), (50, 40)])
            before = [t.clone() for t in params + bufs]
            fl.muon_step(params, grads, bufs, grad_scale=torch.tensor(bad, device=dev))
            assert all(torch.equal(a, b) for a, b in zip(before, params + bufs))
        params, grads, bufs = model(dev, dtype, 2, [(40, 50)])
        other = [p.clone() for p in params], [b.clone() for b in bufs]
        lr = torch.tensor(0.03, device=dev)
        fl.muon_step(params, grads, bufs, lr=lr)
        fl.muon_step(other[0], grads, other[1], lr=float(lr))
        assert torch.equal(params[0], other[0][0])
        negated = [p.clone() for p in other[0]], [b.clone() for b in other[1]]
        fl.muon_step(params, grads, bufs, lr=torch._neg_view(-lr), grad_scale=torch._neg_view(-torch.ones((), device=dev)))
        fl.muon_step(negated[0], grads, negated[1], lr=lr)
        assert torch.equal(params[0], negated[0][0])


def test_muon_class(dev):
    """The optimizer against muon_step, with a clip, groups, missing gradients, checkpoints and copies."""
    print("[case] Muon", flush=True)
    gen = torch.Generator(device=dev).manual_seed(3)

    def leaves():
        g = torch.Generator(device=dev).manual_seed(4)
        return [torch.nn.Parameter(torch.randn(s, device=dev, generator=g).to(t))
                for s, t in (((30, 50), F32), ((64, 20), F32), ((30, 30), BF16), ((9, 9), F32))]

    ps = leaves()
    opt = fl.Muon([dict(params=ps[:3]), dict(params=ps[3:], lr=0.5, nesterov=False, adjust_lr="match_rms_adamw")], lr=0.02,
                  max_grad_norm=1.0)
    ref = [p.detach().clone() for p in ps]
    bufs = [torch.zeros(p.shape, device=dev) for p in ps]
    for step in range(3):
        for i, p in enumerate(ps):
            p.grad = None if (step, i) == (1, 1) else torch.randn(p.shape, device=dev, generator=gen).to(p.dtype)
        opt.step()
        norm, scale = fl.grad_norm([p.grad for p in ps if p.grad is not None], 1.0)
        assert torch.equal(norm, opt.grad_norm)
        for i, p in enumerate(ps):
            if p.grad is not None:
                kw = dict(lr=0.5, nesterov=False, adjust_lr="match_rms_adamw") if i == 3 else dict(lr=0.02)
                fl.muon_step([ref[i]], [p.grad], [bufs[i]], grad_scale=scale, **kw)
            assert torch.equal(ref[i], p.detach()) and torch.equal(opt.state[p]["momentum_buffer"], bufs[i])
    twin = leaves()
    with torch.no_grad():
        for a, b in zip(twin, ps):
            a.copy_(b)
    other = fl.Muon([dict(params=twin[:3]), dict(params=twin[3:])], lr=1.0, max_grad_norm=1.0)
    other.load_state_dict(copy.deepcopy(opt.state_dict()))
    assert other.state[twin[2]]["momentum_buffer"].dtype == F32 and other.param_groups[1]["lr"] == 0.5
    for a, b in zip(twin, ps):
        a.grad = b.grad.clone()
    opt.step()
    other.step()
    assert all(torch.equal(a, b) for a, b in zip(twin, ps))
    ps[0].grad = torch.full_like(ps[0], float("inf"))
    before = [p.detach().clone() for p in ps]
    opt.step()
    assert all(torch.equal(a, b) for a, b in zip(before, ps))


def test_captured_steps(dev):
    print("[case] Muon, graph", flush=True)
    shapes = [(70, 90), (128, 64), (33, 33)]
    params, grads, _ = model(dev, F32, 5, shapes)
    ps = [torch.nn.Parameter(p) for p in params]
    mirror = [torch.nn.Parameter(p.clone()) for p in params]
    opt, eager = (fl.Muon(q, lr=0.02, max_grad_norm=1.0) for q in (ps, mirror))
    for p, q, g in zip(ps, mirror, grads):
        p.grad, q.grad = g, g
    with pytest.raises(RuntimeError, match="capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    torch.cuda.synchronize()
    opt.step()
    eager.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    gen = torch.Generator(device=dev).manual_seed(6)
    for _ in range(4):
        for g in grads:
            g.copy_(torch.randn(g.shape, device=dev, generator=gen))
        graph.replay()
        eager.step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(ps, mirror))


def test_two_streams_at_once(dev):
    print("[case] orthogonalize, two streams", flush=True)
    xs = [matrices(dev, (6, 300, 500), i) for i in range(2)]
    want = [fl.orthogonalize(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(4):
        got = []
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                got.append(fl.orthogonalize(x))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refuses(dev):
    print("[case] muon, refusals", flush=True)
    x = torch.randn(4, 5, device=dev)
    for bad in (x.half(), None, x.to_sparse()):
        with pytest.raises(TypeError):
            fl.orthogonalize(bad)
    for kw in (dict(steps=0), dict(steps=65), dict(eps=-1.0), dict(eps=float("nan")), dict(coefficients=(30.0, 50.0, 9.0)),
               dict(coefficients=(float("nan"), 0.0, 0.0))):
        with pytest.raises(ValueError):
            fl.orthogonalize(x, **kw)
    with pytest.raises(ValueError):
        fl.orthogonalize(x[0])
    buf = torch.zeros(4, 5, device=dev)
    for params, grads, bufs in (([x], [x], [buf]), ([x], [buf], [buf]), ([x], [buf], [x]), ([x, x], [buf, buf], [buf, buf.clone()]),
                                ([x[0]], [buf[0]], [buf[0].clone()]), ([x], [], [buf]), ([x.t()], [buf.t()], [buf.clone()]),
                                ([x], [buf[:2]], [buf.clone()]), ([], [], []), ([x], [buf.cpu()], [buf.clone()])):
        with pytest.raises(ValueError):
            fl.muon_step(params, grads, bufs)
    with pytest.raises(TypeError):
        fl.muon_step([x], [buf], [buf.bfloat16()])
    with pytest.raises(TypeError):
        fl.muon_step([x.half()], [buf.half()], [buf])
    fl.muon_step([x], [torch.ones_like(x)], [buf])
