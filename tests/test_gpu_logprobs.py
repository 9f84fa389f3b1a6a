"""GPU: token log probabilities, entropy, top alternatives and their gradients against a plain float64 form.

Tolerances count roundings, u = 2^-24. With D the largest |d| = |x - max| / temperature among logits that weigh
anything (e^d > 2^-40 of the row's sum; the others' errors vanish in it), a power e^d carries (4 D + 4) u: the
difference, two products and the base-2 argument each move d by D u at most, the power itself rounds twice. A sum of V of them
carries that and its own additions, at most V / 256 + 64 u for any order that adds in at least 256 lanes. So with
E = (4 D + V / 256 + 72) u: ln s is off by E + 2 u |ln s|; a log probability by that and 4 u |d_t|; an entropy by
E (2 + 2 D), its sum of e^d d over s being two such sums with terms up to D; a weight p (relative) by
2 E + 8 u D. A gradient is a sum of terms (|g|, p |a|, p |h| (|ln p| + H)) each with that relative error, and is
rounded to its type (half a step, eps / 2) at the end.
"""
from __future__ import annotations

import pytest
import torch

import fields_lm_amd as fl

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm device")
    return torch.device("cuda:0")


def plain(x, t, temperature, k, ignore=-100):
    """float64: (log p [R, V], log probabilities, entropy, top logprobs, top tokens, D per row)."""
    x = x.double().cpu()
    t = t.cpu()
    empty = (x == float("-inf")).all(-1)
    top = torch.where(empty, 0.0, x.amax(-1))[..., None]
    d = (x - top) / temperature
    s = d.exp().sum(-1, keepdim=True)
    logp = torch.where(empty[..., None], float("-inf"), d - s.log())
    p = logp.exp()
    h = -torch.where(p > 0, p * logp, 0.0).sum(-1)
    h = torch.where(x.isnan().any(-1) | (x == float("inf")).any(-1), float("nan"), h)
    inside = (t >= 0) & (t < x.shape[-1])
    lp = logp.gather(-1, torch.where(inside, t, 0)[..., None])[..., 0]
    lp = torch.where(t == ignore, 0.0, torch.where(inside, lp, float("nan")))
    order = torch.where(x.isnan(), float("inf"), x)  # NaN above +inf: sorted by (nan, value), stable
    idx = torch.sort(order, dim=-1, descending=True, stable=True).indices
    idx = idx.gather(-1, torch.sort(x.gather(-1, idx).isnan().int(), dim=-1, descending=True, stable=True).indices)[..., :k]
    weighs = (logp > -40 * 0.6931471805599453)
    big = torch.where(weighs, d.abs(), 0.0).amax(-1)
    return logp, lp, h, logp.gather(-1, idx), idx, big


def bounds(x, temperature, ref):
    logp, lp, h, top, idx, big = ref
    v = x.shape[-1]
    e = (4 * big + v / 256 + 72) * U
    x64 = x.double().cpu()
    m = x64.amax(-1, keepdim=True)
    logs = e + 2 * U * (big + 12)  # |ln s| <= ln V < 12 here
    return e, logs, lambda values: logs[..., None] + 4 * U * ((m - values).abs() / temperature)


def check(got, ref, tol, what):
    got = got.double().cpu()
    # (3e38 - -3e38 has no fp32 value but infinity)
    ref = torch.where(ref.abs() > torch.finfo(torch.float32).max, ref.sign() * float("inf"), ref)
    assert torch.equal(got.isnan(), ref.isnan()), what
    special = ~ref.isfinite()
    assert torch.equal(got[special & ~ref.isnan()], ref[special & ~ref.isnan()]), what
    off = torch.where(special, 0.0, (got - ref).abs())
    worst = (off - torch.where(special, 1.0, tol)).nan_to_num(1e300).flatten().argmax()
    assert bool((off <= torch.where(special, 1.0, tol)).all()), \
        (what, int(worst), *(float(z.expand_as(off).flatten()[worst]) for z in (got, ref, tol)))


def check_forward(x, t, temperature, k, entropy, r, ignore=-100):
    ref = logp, lp, h, top, idx, big = plain(x, t, temperature, k, ignore)
    e, logs, lp_tol = bounds(x, temperature, ref)
    xt = x.double().cpu().gather(-1, t.cpu().clamp(0, x.shape[-1] - 1)[..., None])
    check(r.logprobs, lp, lp_tol(xt)[..., 0], "logprobs")
    assert r.logprobs.dtype == torch.float32 and r.logprobs.shape == t.shape
    if entropy:
        check(r.entropy, h, (2 + 2 * big) * e + 4 * U * big + logs, "entropy")
    else:
        assert r.entropy is None
    if k:
        assert torch.equal(r.top_tokens.cpu(), idx), "top_tokens"
        check(r.top_logprobs, top, lp_tol(x.double().cpu().gather(-1, idx)), "top_logprobs")
    else:
        assert r.top_tokens is None and r.top_logprobs is None
    return ref


def make(dev, rows, vocab, dtype, seed, spread=2.5):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(rows, vocab, device=dev, generator=g) * spread
    t = torch.randint(0, vocab, (rows,), device=dev, generator=g)
    x.scatter_add_(-1, t[:, None], 8 * torch.rand(rows, 1, device=dev, generator=g))
    return x.to(dtype), t


# one logit; less than a vector, a wave and a block; odd; around the sizes that change the tile
VOCABS = [1, 2, 7, 63, 65, 255, 257, 1000, 1024, 1025, 2047, 2049, 4096, 4097, 5003, 8191, 8193, 16384, 16385, 32767, 32769,
          40001, 65537, 131073, 600011]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", VOCABS)
def test_forward_over_vocabularies(dev, vocab, dtype):
    print(f"[case] token_logprobs V={vocab} {dtype}", flush=True)
    for rows, k, entropy, temperature in ((3, min(5, vocab), True, 1.0), (1, 0, False, 0.7), (2, min(64, vocab), False, 1.4)):
        x, t = make(dev, rows, vocab, dtype, vocab + rows)
        r = fl.token_logprobs(x, t, temperature=temperature, top_k=k, entropy=entropy)
        check_forward(x, t, temperature, k, entropy, r)


def test_forward_of_the_longest_row(dev):
    """2^23 logits: 1,024 segments; with the largest in the last and equal ones in others."""
    print("[case] token_logprobs V=2^23", flush=True)
    x, t = make(dev, 2, 1 << 23, torch.float32, 3)
    x[0, -1], x[1, 5], x[1, 1 << 22] = 30.0, 29.0, 29.0
    check_forward(x, t, 1.0, 64, True, fl.token_logprobs(x, t, top_k=64, entropy=True))
    with pytest.raises(ValueError):
        fl.token_logprobs(torch.empty(1, (1 << 23) + 1, device=dev), t[:1])


@pytest.mark.parametrize("rows,vocab", [(1, 16384), (64, 16384), (300, 16384), (700, 501), (5000, 33), (257, 12345),
                                        (40, 70000)])
def test_forward_over_rows(dev, rows, vocab):
    print(f"[case] token_logprobs rows={rows} V={vocab}", flush=True)
    x, t = make(dev, rows, vocab, torch.bfloat16, rows)
    check_forward(x, t, 1.0, 20, True, fl.token_logprobs(x, t, top_k=20, entropy=True))


def test_forward_reads_slices_in_place(dev):
    print("[case] token_logprobs, slices and strides", flush=True)
    for dtype in (torch.bfloat16, torch.float32):
        x, t = make(dev, 3 * 9, 1001, dtype, 5)
        x, t = x.view(3, 9, 1001), t.view(3, 9)
        for a, b in ((x[:, :-1], t[:, 1:]), (x.transpose(0, 1), t.t()), (x[:, ::2], t[:, ::2]), (x[..., 3:], t % 998),
                     (x[1:2, 4], t[1:2, 4]), (x[0, 0], t[0, 0]), (x[..., ::2], t % 501), (x[:, :1].expand(3, 9, 1001), t)):
            r = fl.token_logprobs(a, b, top_k=3, entropy=True)
            check_forward(a.reshape(-1, a.shape[-1]), b.reshape(-1), 1.0, 3, True,
                          fl.TokenLogprobs(r.logprobs.reshape(-1), r.entropy.reshape(-1), r.top_logprobs.reshape(-1, 3),
                                           r.top_tokens.reshape(-1, 3)))
            assert r.logprobs.shape == b.shape and r.top_tokens.shape == (*b.shape, 3)


def special_rows(dev, vocab, dtype):
    """Rows that go wrong first: masked, empty, equal, of the type's lowest value, infinite, NaN, large."""
    g = torch.Generator(device=dev).manual_seed(vocab)
    x = (torch.randn(18, vocab, device=dev, generator=g) * 3).to(dtype)
    low = torch.finfo(dtype).min
    x[0, 1:] = float("-inf")                     # one token left
    x[1] = float("-inf")                         # none left
    x[2] = 0.0                                   # all equal
    x[3] = low                                   # all masked by the type's lowest value
    x[4, ::2] = low
    x[5, vocab // 2] = float("nan")
    x[6, vocab - 1] = float("inf")
    x[7] = -0.0
    x[7, ::3] = 0.0                              # both zeros are equal
    x[8] = torch.arange(vocab, device=dev).to(dtype) / 64
    x[9] = -torch.arange(vocab, device=dev).to(dtype) / 64
    x[10] = x[10] * 1e4                          # large logits
    x[11, : vocab // 2] = float("-inf")
    x[12] = 3.0
    x[12, vocab // 3] = torch.finfo(dtype).max   # the difference overflows to -inf
    x[12, vocab // 4] = low
    x[13, 0], x[13, vocab - 1] = float("inf"), float("nan")
    x[14] = float("nan")
    x[15] = torch.randint(0, 3, (vocab,), device=dev, generator=g).to(dtype)  # a few values, many times each
    x[16] = torch.where(torch.arange(vocab, device=dev) % 131 == 7, x[16], float("-inf"))  # few and far between
    x[17, vocab // 3:vocab // 3 + 90] = float("-inf")
    x[17, :vocab // 3] = float("-inf")
    return x


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [3, 300, 8193, 70001])
def test_forward_of_special_rows(dev, vocab, dtype):
    print(f"[case] token_logprobs special rows V={vocab} {dtype}", flush=True)
    x = special_rows(dev, vocab, dtype)
    for k in sorted({min(vocab, n) for n in (1, 20, 21, 64)}):
        for at in (0, vocab - 1):
            t = torch.full((18,), at, device=dev)
            check_forward(x, t, 1.0, k, True, fl.token_logprobs(x, t, top_k=k, entropy=True))


@pytest.mark.parametrize("k", [1, 3, 20, 64])
@pytest.mark.parametrize("vocab", [16388, 131072, 64 * 8192, 64 * 8192 + 1])
def test_alternatives_of_long_rows(dev, vocab, k):
    """Rows of several segments (fp32 segments of 8,192), up to 64 and one more: the largest logits in one of them, one in
    each, equal in all, masked but in the last, fewer left than are wanted."""
    print(f"[case] alternatives of long rows V={vocab} k={k}", flush=True)
    g = torch.Generator(device=dev).manual_seed(vocab + k)
    x = torch.randn(8, vocab, device=dev, generator=g) * 3
    x[1, 8192:8292] += 50
    x[2, 17::8192] += 50
    x[3] = 1.0
    x[4, :-70] = float("-inf")
    x[5] = float("-inf")
    x[5, ::vocab // 2] = 2.0
    x[6, -1] = float("nan")
    x[7] = x[7].round()  # many equal ones
    t = torch.randint(0, vocab, (8,), device=dev, generator=g)
    check_forward(x, t, 1.0, k, True, fl.token_logprobs(x, t, top_k=k, entropy=True))


def test_tokens_outside_the_vocabulary_and_ignored_ones(dev):
    print("[case] token_logprobs, tokens outside", flush=True)
    x, _ = make(dev, 6, 400, torch.float32, 9)
    t = torch.tensor([5, -100, 400, -1, 1 << 40, -(1 << 40)], device=dev)
    check_forward(x, t, 1.0, 2, True, fl.token_logprobs(x, t, top_k=2, entropy=True))
    x[1] = float("nan")
    assert float(fl.token_logprobs(x, t).logprobs[1]) == 0.0
    assert fl.token_logprobs(x, t, ignore_index=5).logprobs.cpu()[:2].isnan().tolist() == [False, True]


def test_no_rows(dev):
    print("[case] token_logprobs without rows", flush=True)
    x = torch.randn(4, 0, 7, device=dev, requires_grad=True)
    r = fl.token_logprobs(x, torch.zeros(4, 0, dtype=torch.long, device=dev), top_k=3, entropy=True)
    assert r.logprobs.shape == r.entropy.shape == (4, 0) and r.top_logprobs.shape == r.top_tokens.shape == (4, 0, 3)
    assert r.top_tokens.dtype == torch.int64
    assert torch.autograd.grad(r.logprobs.sum(), x)[0].shape == x.shape


def test_many_rows_past_32_bit_offsets(dev):
    """Logits of more than 2^31 values: rows on both sides of the border."""
    print("[case] token_logprobs past 2^31 values", flush=True)
    vocab, rows = 16384, (1 << 17) + 3
    x = torch.zeros(rows, vocab, device=dev, dtype=torch.bfloat16)
    t = torch.arange(rows, device=dev) % vocab
    at = torch.tensor([0, 1, (1 << 16) + 1, (1 << 17) - 1, 1 << 17, rows - 1], device=dev)
    part, _ = make(dev, len(at), vocab, torch.bfloat16, 11)
    x[at] = part
    x.requires_grad_()
    r = fl.token_logprobs(x, t, top_k=3, entropy=True)
    check_forward(part, t[at], 1.0, 3, True, fl.TokenLogprobs(*[o.detach()[at] for o in r]))
    w = torch.zeros(rows, device=dev)
    w[at] = 1.0
    grad, = torch.autograd.grad(r.logprobs, x, w)
    check_grad(part, t[at], 1.0, 0, w[at], None, None, grad[at])
    assert float(grad.float().abs().sum(-1)[(w == 0)].max()) == 0.0


# ------------------------------------------------------------------ gradients
def check_grad(x, t, temperature, k, g, h, gt, got, ignore=-100):
    ref = logp, lp, ent, top, idx, big = plain(x, t, temperature, max(k, 1), ignore)
    x64, t = x.double().cpu(), t.cpu()
    p = logp.exp()
    g = torch.where(t == ignore, 0.0, g.double().cpu()) if g is not None else torch.zeros(t.shape, dtype=torch.float64)
    h = h.double().cpu() if h is not None else torch.zeros_like(g)
    gt = gt.double().cpu() if gt is not None else torch.zeros(*t.shape, 0, dtype=torch.float64)
    inside = (t >= 0) & (t < x.shape[-1])
    up = torch.zeros_like(x64).scatter_add_(-1, torch.where(inside, t, 0)[..., None], torch.where(inside, g, 0.0)[..., None])
    size = up.abs()
    if gt.shape[-1]:
        up.scatter_add_(-1, idx[..., :gt.shape[-1]], gt)
        size.scatter_add_(-1, idx[..., :gt.shape[-1]], gt.abs())
    a = g + gt.sum(-1)
    inner = torch.where(p > 0, logp + ent[..., None], 0.0)
    exp = (up - p * (a[..., None] + h[..., None] * inner)) / temperature
    weight = (g.abs() + gt.abs().sum(-1))[..., None] \
        + h.abs()[..., None] * (torch.where(p > 0, logp.abs(), 0.0) + ent.abs()[..., None])
    size = (size + p * weight) / temperature
    live = (g != 0) | (h != 0) | (gt != 0).any(-1)
    empty = (x64 == float("-inf")).all(-1)
    exp = torch.where((live & ~empty)[..., None], exp, 0.0)
    exp = torch.where((live & ~empty & (g != 0) & ~inside)[..., None], float("nan"), exp)
    e, logs, _ = bounds(x, temperature, ref)
    rel = (2 * e + 8 * U * big + 8 * U)[..., None] + 8 * U * torch.where(p > 0, logp.abs(), 0.0)  # (small p: its own exponent)
    # ln p + H cancels near p = e^-H: its parts' errors
    part = (p * h.abs()[..., None] * (2 * logs + (2 + 2 * big) * e)[..., None]) / temperature
    # a p below 2^-126 is 0 (the hardware's power has no subnormal results): up to 2^-126 of its factor, whose ln p is
    # above -104 where fp32 has a value at all
    flushed = 2.0 ** -126 * (1 + torch.where(p > 2.0 ** -150, weight, 0.0)) / temperature
    tol = size * (rel + 8 * U) + part + exp.abs() * torch.finfo(x.dtype).eps / 2 + flushed
    check(got, exp, tol, "grad")
    assert got.dtype == x.dtype and got.shape == x.shape


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [1, 2, 65, 501, 2048, 5003, 16384, 32769, 70001])
def test_gradients(dev, vocab, dtype):
    print(f"[case] token_logprobs gradients V={vocab} {dtype}", flush=True)
    rows = 5
    x, t = make(dev, rows, vocab, dtype, vocab)
    t[1] = -100
    k = min(7, vocab)
    gen = torch.Generator(device=dev).manual_seed(1)
    g, h, gt = (torch.randn(*s, device=dev, generator=gen) for s in ((rows,), (rows,), (rows, k)))
    g[2] = h[2] = 0.0
    gt[2] = 0.0  # a row that passes nothing
    for temperature in (1.0, 0.6):
        for use in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 1)):
            z = x.detach().clone().requires_grad_()
            r = fl.token_logprobs(z, t, temperature=temperature, top_k=k if use[2] else 0, entropy=bool(use[1]))
            outs = [o for o, u in zip((r.logprobs, r.entropy, r.top_logprobs), use) if u]
            ups = [o for o, u in zip((g, h, gt), use) if u]
            got, = torch.autograd.grad(outs, z, ups)
            check_grad(x, t, temperature, k if use[2] else 0, *(o if u else None for o, u in zip((g, h, gt), use)), got)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [3, 300, 8193])
def test_gradients_of_special_rows(dev, vocab, dtype):
    print(f"[case] token_logprobs gradients of special rows V={vocab} {dtype}", flush=True)
    x = special_rows(dev, vocab, dtype)
    t = torch.full((18,), vocab - 1, device=dev)
    t[3], t[4] = vocab, -100
    k = min(5, vocab)
    g = torch.linspace(-1, 1, 18, device=dev) + 0.01
    z = x.clone().requires_grad_()
    r = fl.token_logprobs(z, t, top_k=k, entropy=True)
    got, = torch.autograd.grad([r.logprobs, r.entropy], z, [g, g / 3])
    check_grad(x, t, 1.0, 0, g, g / 3, None, got)
    z = x.clone().requires_grad_()  # nothing flows: zeros, also from rows with NaN
    got, = torch.autograd.grad(fl.token_logprobs(z, t).logprobs, z, torch.zeros(18, device=dev))
    assert float(got.float().abs().max()) == 0.0


def test_gradients_of_slices_and_broadcast_logits(dev):
    print("[case] token_logprobs gradients of slices and broadcast logits", flush=True)
    for dtype in (torch.bfloat16, torch.float32):
        x, t = make(dev, 3 * 9, 1001, dtype, 5)
        x, t = x.view(3, 9, 1001), t.view(3, 9)
        g = torch.randn(3, 9, device=dev, generator=torch.Generator(device=dev).manual_seed(2))
        z = x.clone().requires_grad_()
        got, = torch.autograd.grad(fl.token_logprobs(z[:, :-1], t[:, 1:]).logprobs, z, g[:, 1:])
        assert float(got[:, -1].float().abs().max()) == 0.0
        check_grad(x[:, :-1].reshape(-1, 1001), t[:, 1:].reshape(-1), 1.0, 0, g[:, 1:].reshape(-1), None, None,
                   got[:, :-1].reshape(-1, 1001))
        one = x[:, :1].clone().requires_grad_()  # every position reads one row's logits
        wide = one.expand(3, 9, 1001)
        got, = torch.autograd.grad(fl.token_logprobs(wide, t).logprobs, wide, g)
        check_grad(x[:, :1].expand(3, 9, 1001).reshape(-1, 1001), t.reshape(-1), 1.0, 0, g.reshape(-1), None, None,
                   got.reshape(-1, 1001))
        total, = torch.autograd.grad(fl.token_logprobs(one.expand(3, 9, 1001), t).logprobs, one, g)
        assert total.shape == one.shape
        z = x.clone().requires_grad_()  # gradients that are broadcast themselves (a mean's)
        got, = torch.autograd.grad(fl.token_logprobs(z.transpose(0, 1), t.t()).logprobs.mean(), z)
        check_grad(x.reshape(-1, 1001), t.reshape(-1), 1.0, 0, torch.full((27,), 1 / 27, device=dev), None, None,
                   got.reshape(-1, 1001))


def test_gradient_against_differences(dev):
    print("[case] token_logprobs gradient against differences", flush=True)
    x, t = make(dev, 3, 50, torch.float32, 2, spread=1.0)
    w = torch.randn(3, 2, device=dev, generator=torch.Generator(device=dev).manual_seed(4))

    def loss(z):
        r = fl.token_logprobs(z, t, temperature=0.8, entropy=True)
        return (w[:, 0] * r.logprobs + w[:, 1] * r.entropy).double().sum()

    z = x.clone().requires_grad_()
    got, = torch.autograd.grad(loss(z), z)
    step = 2.0 ** -6
    for i, j in [(0, int(t[0])), (0, 3), (1, 17), (2, 49)]:
        d = torch.zeros_like(x)
        d[i, j] = step
        diff = float(loss(x + d) - loss(x - d)) / (2 * step)
        # third derivatives of these sums below 60 (weights to 2.5, 1 / 0.8^3, entropy's up to 4 of p ln p): 10 step^2,
        # and the two losses' roundings, 2^-20 each
        assert abs(diff - float(got[i, j])) <= 10 * step ** 2 + 2 ** -20 / step, (i, j)


def test_double_backward_matches_log_softmax(dev):
    print("[case] token_logprobs double backward", flush=True)
    x, t = make(dev, 4, 40, torch.float32, 6, spread=1.0)
    t[2] = -100

    def second(fn):
        z = x.clone().requires_grad_()
        g, = torch.autograd.grad(fn(z).square().sum(), z, create_graph=True)
        return torch.autograd.grad(g.square().sum(), z)[0].double()

    def stock(z):
        lp = torch.log_softmax(z / 0.9, -1)
        ent = -(lp.exp() * lp).sum(-1)
        return torch.where(t == -100, 0.0, lp.gather(-1, t.clamp_min(0)[:, None])[:, 0]) + ent

    def own(z):
        r = fl.token_logprobs(z, t, temperature=0.9, entropy=True)
        return r.logprobs + r.entropy

    a, b = second(own), second(stock)
    assert float((a - b).norm() / b.norm()) <= 1e-4  # two fp32 chains of some 40 roundings over sums of 40 terms


def test_partial_outputs_and_no_gradient(dev):
    print("[case] token_logprobs, parts of the outputs", flush=True)
    x, t = make(dev, 3, 100, torch.bfloat16, 8)
    with torch.no_grad():
        assert not fl.token_logprobs(x.requires_grad_(), t).logprobs.requires_grad
    r = fl.token_logprobs(x, t, top_k=4, entropy=True)
    assert r.logprobs.requires_grad and r.entropy.requires_grad and r.top_logprobs.requires_grad
    assert not r.top_tokens.requires_grad
    got, = torch.autograd.grad(r.top_logprobs[:, 1].sum(), x)
    gt = torch.zeros(3, 4, device=dev)
    gt[:, 1] = 1
    check_grad(x.detach(), t, 1.0, 4, None, None, gt, got)
    import torch.autograd.forward_ad as fwad

    with fwad.dual_level():
        for z in (x.detach(), x):
            with pytest.raises(NotImplementedError):  # a tangent is refused, not lost
                fl.token_logprobs(fwad.make_dual(z, torch.ones_like(x)), t)
    with pytest.raises(RuntimeError):  # a transform's wrapper has no memory to read
        torch.func.vmap(lambda a, b: fl.token_logprobs(a, b).logprobs)(x.detach(), t)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda a: fl.token_logprobs(a, t).logprobs.sum())(x.detach())
    with pytest.raises(RuntimeError):  # a trace would hold this call's results
        torch.jit.trace(lambda a, b: fl.token_logprobs(a, b).logprobs, (x.detach(), t))
    from torch._subclasses.fake_tensor import FakeTensorMode

    plain = x.detach()
    with FakeTensorMode(allow_non_fake_inputs=True):
        with pytest.raises(TypeError):
            fl.token_logprobs(x.detach(), t)  # a fake tensor
        with pytest.raises(ValueError):  # outputs without memory
            fl.token_logprobs(plain, t)
    with pytest.raises(ValueError):
        fl.token_logprobs(x, t.cpu())
    changed = x.detach().clone().requires_grad_()
    y = changed * 1.0
    r = fl.token_logprobs(y, t)
    y.add_(1.0)
    with pytest.raises(RuntimeError):  # what the backward reads was changed in place
        r.logprobs.sum().backward()


def test_two_streams_and_graph_replays(dev):
    """Calls on two streams at once, and two captured graphs replayed in turn with eager calls between."""
    print("[case] token_logprobs on streams and in graphs", flush=True)
    cases = [make(dev, r, v, torch.bfloat16, r + v) for r, v in ((64, 16384), (2, 131072))]
    eager = [fl.token_logprobs(x, t, top_k=20, entropy=True) for x, t in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    outs = [[], []]
    for _ in range(4):
        for i, (s, (x, t)) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(s):
                outs[i].append(fl.token_logprobs(x, t, top_k=20, entropy=True))
    torch.cuda.synchronize()
    for got, exp in zip(outs, eager):
        for r in got:
            assert all(torch.equal(a, b) for a, b in zip(r, exp))
    graphs, results, inputs = [], [], []
    for x, t in cases:
        x = x.clone()
        up = torch.ones(t.shape, device=dev)
        z = x.requires_grad_()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            torch.autograd.grad(fl.token_logprobs(z, t, top_k=20, entropy=True).logprobs, z, up)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = fl.token_logprobs(z, t, top_k=20, entropy=True)
            grad, = torch.autograd.grad(r.logprobs, z, up)
        graphs.append(g)
        results.append((*(o.detach() for o in r), grad))
        inputs.append((z, t, up))
    for turn in range(3):
        for z, _, _ in inputs:
            with torch.no_grad():
                z.copy_(z.flip(-1) if turn else z)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for (z, t, up), got in zip(inputs, results):
            r = fl.token_logprobs(z, t, top_k=20, entropy=True)
            grad, = torch.autograd.grad(r.logprobs, z, up)
            assert all(torch.equal(a, b) for a, b in zip(got, (*(o.detach() for o in r), grad))), turn


@pytest.mark.parametrize("leaf", [True, False])
def test_captured_backward_refuses_leaves_of_a_living_eager_graph(dev, leaf):
    """A graph of the default stream that holds the leaves: the captured backward raises; without it, it replays."""
    print(f"[case] captured backward, a living eager graph, leaf {leaf}", flush=True)
    x, t = make(dev, 8, 301, torch.float32, 5)
    z = x.clone().requires_grad_()
    up = torch.ones(8, device=dev)

    def loss():
        return fl.token_logprobs(z if leaf else z * 2.0, t, top_k=3).logprobs

    living = loss()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r = loss()
        with pytest.raises(RuntimeError, match="default stream"):
            r.backward(up)
        del r
    del living
    torch.cuda.synchronize()
    assert z.grad is None
    z.grad = torch.zeros_like(z)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        z.grad.zero_()
        loss().backward(up)
    for turn in range(3):
        with torch.no_grad():
            z.add_(0.25 * turn).copy_(z.flip(-1))
        g.replay()
        torch.cuda.synchronize()
        got = z.grad.clone()
        exp, = torch.autograd.grad(loss(), z, up)
        assert torch.equal(got, exp), turn


def test_score_of_the_model_is_its_logits_log_softmax(dev):
    print("[case] FieldsForCausalLM.score", flush=True)
    from fields_lm_amd import model as M

    torch.manual_seed(0)
    core = M.FieldTokenSystem(vocab=211, dim=64, ff_hidden=96, refresh_windows=(64,), mamba_positions=(3,), layers=6, q_heads=4,
                              kv_heads=2, latent_dim=16, landmark_chunk=32, softpatch_rank=8, late_ff_delta=0,
                              mamba=dict(d_state=16, headdim=16, chunk_size=32)).to(dev)
    lm = fl.FieldsForCausalLM(core, backend_name="test", source_audit={}, topology_audit={})
    ids = torch.randint(0, 211, (2, 33), device=dev)
    with torch.no_grad():
        logits = lm(ids).logits[:, :-1]
    r = lm.score(ids, top_k=3, entropy=True)
    flat = fl.TokenLogprobs(*(o.reshape(-1, *o.shape[2:]) for o in r))
    check_forward(logits.reshape(-1, 211), ids[:, 1:].reshape(-1), 1.0, 3, True, flat)
    assert lm.score(ids[:, :1]).logprobs.shape == (2, 0)
    with pytest.raises(TypeError):
        lm.score(ids.int())


@pytest.mark.parametrize("rows", [1, 5])
def test_gradients_with_the_negative_flag(dev, rows):
    """Upstream gradients whose memory holds their negative (the imaginary part of a conjugate), of one row and more."""
    print(f"[case] token_logprobs gradients with the negative flag, rows {rows}", flush=True)
    x, t = make(dev, rows, 300, torch.float32, rows)
    gen = torch.Generator(device=dev).manual_seed(rows)
    ups = [torch.randn(*s, device=dev, generator=gen) for s in ((rows,), (rows,), (rows, 4))]
    z = x.clone().requires_grad_()
    r = fl.token_logprobs(z, t, top_k=4, entropy=True)
    outs = [r.logprobs, r.entropy, r.top_logprobs]
    for use in ((0,), (1,), (2,), (0, 1, 2)):
        o, g = [outs[i] for i in use], [ups[i] for i in use]
        exp, = torch.autograd.grad(o, z, g, retain_graph=True)
        got, = torch.autograd.grad(o, z, [torch._neg_view(-u) for u in g], retain_graph=True)
        assert torch.equal(got, exp), use
    lp = fl.token_logprobs(z, t).logprobs
    exp, = torch.autograd.grad(2 * lp.sum(), z, retain_graph=True)
    got, = torch.autograd.grad((torch.complex(torch.zeros_like(lp), lp).conj() * (1 + 2j)).real.sum(), z)
    assert torch.equal(got, exp)


def test_tokens_with_the_negative_flag(dev):
    print("[case] token_logprobs, tokens with the negative flag", flush=True)
    x, t = make(dev, 6, 400, torch.float32, 9)
    t[1], t[2] = -100, 400
    z = x.clone().requires_grad_()
    a, b = (fl.token_logprobs(z, s).logprobs for s in (t, torch._neg_view(-t)))
    assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))
    a, b = (torch.autograd.grad(o.sum(), z)[0].nan_to_num(7.0) for o in (a, b))
    assert torch.equal(a, b)


def test_upstream_gradients_without_memory_are_refused(dev):
    """What follows in the graph may hand over a gradient that dispatches to Python, with no memory at its address."""
    print("[case] token_logprobs, upstream gradients without memory", flush=True)
    x, t = make(dev, 3, 20, torch.float32, 1)

    class Wrapped(torch.Tensor):
        @staticmethod
        def __new__(cls, like):
            return torch.Tensor._make_wrapper_subclass(cls, like.shape, dtype=like.dtype, device=like.device)

        @classmethod
        def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
            return func(*(torch.ones(a.shape, dtype=a.dtype, device=a.device) if isinstance(a, cls) else a for a in args),
                        **(kwargs or {}))

    class Hands(torch.autograd.Function):
        @staticmethod
        def forward(ctx, a):
            return a.clone()

        @staticmethod
        def backward(ctx, g):
            return Wrapped(g)

    for entropy in (False, True):
        z = x.clone().requires_grad_()
        r = fl.token_logprobs(z, t, entropy=entropy)
        with pytest.raises(TypeError):
            torch.autograd.grad(Hands.apply(r.entropy if entropy else r.logprobs).sum(), z)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_differentiable_gradients_of_special_rows(dev, dtype):
    """A backward that can be differentiated again has the plain backward's zeros and NaN: rows that pass nothing, ignored
    and outside tokens, rows of -inf, NaN and +inf."""
    print(f"[case] token_logprobs differentiable gradients of special rows {dtype}", flush=True)
    x = special_rows(dev, 300, dtype)
    for turn, (token, use) in enumerate([(299, (1, 0, 0)), (-100, (1, 0, 0)), (300, (1, 0, 0)), (300, (1, 1, 1)),
                                         (-100, (0, 1, 1)), (0, (1, 1, 1))]):
        t = torch.full((18,), token, device=dev)
        gen = torch.Generator(device=dev).manual_seed(turn)
        ups = [torch.randn(*s, device=dev, generator=gen) for s in ((18,), (18,), (18, 5))]
        for u in ups:
            u[turn % 2::2] = 0.0
        z = x.clone().requires_grad_()
        r = fl.token_logprobs(z, t, top_k=5, entropy=True)
        o, g = ([a for a, u in zip(l, use) if u] for l in ((r.logprobs, r.entropy, r.top_logprobs), ups))
        exp, = torch.autograd.grad(o, z, g, retain_graph=True)
        got, = torch.autograd.grad(o, z, g, create_graph=True)
        got, weights = got.detach(), [u if w else None for u, w in zip(ups, use)]
        if weights[0] is not None:
            weights[0] = torch.where(t == -100, 0.0, weights[0])
        quiet = torch.stack([(u.view(18, -1) == 0).all(-1) for u in weights if u is not None]).all(0)
        for grad in (exp, got):
            assert bool((grad[quiet] == 0).all()), (token, use)
            assert bool((grad[1] == 0).all())  # -inf alone
            if not bool(quiet.all()):
                check_grad(x[~quiet], t[~quiet], 1.0, 5 * use[2], *(None if u is None else u[~quiet] for u in weights),
                           grad[~quiet])


def flat_bounds(x, big, temperature=1.0):
    """(ln s, entropy) tolerances of rows whose additions are counted one by one: up to 8 packs and one logit to a
    thread (at most 65), 6 in a wave, 3 between waves, and where segments are joined 6 and 16 more: 96 with the
    roundings of each segment's ln and of its shift (three of at most 40 each in base 2, 120 u) beside."""
    e = (4 * big + 96 + 120 + 8) * U
    logs = e + 2 * U * (big + 16)  # |ln s| <= ln 2^23 < 16
    return logs, (2 + 2 * big) * e + 4 * U * big + logs


def test_sums_of_the_longest_row(dev):
    """2^23 logits in 1,024 segments, each of which weighs: all equal, a small spread, and all the weight in one
    segment, early, late or last. A lost segment of equal logits would move ln s by 2^-10."""
    print("[case] token_logprobs, sums of V=2^23", flush=True)
    vocab, seg = 1 << 23, 8192
    g = torch.Generator(device=dev).manual_seed(1)
    x = torch.zeros(6, vocab, device=dev)
    x[1] = 0.1 * torch.randn(vocab, device=dev, generator=g)
    for row, at in ((2, 3), (3, 130), (4, 700), (5, 1023)):
        x[row, at * seg:(at + 1) * seg] = 20.0 + 0.01 * torch.randn(seg, device=dev, generator=g)
    t = torch.tensor([5, vocab - 1, 3 * seg + 1, 130 * seg + 7, 0, vocab - 2], device=dev)
    r = fl.token_logprobs(x, t, entropy=True, top_k=3)
    _, lp, h, top, idx, _ = plain(x, t, 1.0, 3)
    big = torch.tensor([0.0, 1.2, 20.1, 20.1, 20.1, 20.1], dtype=torch.float64)  # (outside the heavy segment too)
    logs, ent = flat_bounds(x, big)
    assert float(logs.max()) < 3e-5  # far below what a segment weighs
    check(r.logprobs, lp, logs + 4 * U * big, "logprobs")
    check(r.entropy, h, ent, "entropy")
    assert torch.equal(r.top_tokens.cpu(), idx)
    check(r.top_logprobs, top, (logs + 4 * U * big)[:, None], "top_logprobs")


@pytest.mark.parametrize("dtype,vocab,k", [(torch.float32, 9, 3), (torch.bfloat16, 600, 20), (torch.float32, 1025, 5),
                                           (torch.float32, 1030, 40), (torch.bfloat16, 8200, 20), (torch.float32, 8193, 5),
                                           (torch.float32, 8199, 64)])
def test_rows_past_one_launch(dev, dtype, vocab, k):
    """More than 2^20 rows, so that blocks take a second one: overlapping windows of one long tensor, against the same
    rows in calls that hold them at once, bit for bit, and some of them in 64 bits."""
    print(f"[case] token_logprobs, 2^20 + 9 rows of {vocab} {dtype}", flush=True)
    rows, half = (1 << 20) + 9, 1 << 19
    g = torch.Generator(device=dev).manual_seed(vocab)
    line = (torch.randn(rows + vocab, device=dev, generator=g) * 3).to(dtype)
    line[half:half + 2 * vocab] = float("-inf")  # windows of -inf alone, and few logits left beside
    line[rows - 3 - vocab // 2] = float("nan")   # the last rows, that their blocks' first rows are far from
    x = line.as_strided((rows, vocab), (1, 1))
    t = torch.randint(0, vocab, (rows,), device=dev, generator=g)
    t[::7] = -100
    outs = fl.token_logprobs(x, t, top_k=k, entropy=True)
    parts = [fl.token_logprobs(x[lo:hi], t[lo:hi], top_k=k, entropy=True)
             for lo, hi in ((0, half), (half, 2 * half), (2 * half, rows))]
    for a, *b in zip(outs, *parts):
        assert torch.equal(a.view(torch.int32), torch.cat(b).view(torch.int32))
    at = torch.tensor([0, 1, 8, half - 1, 2 * half - 1, 2 * half, 2 * half + 1, rows - 1], device=dev)
    check_forward(x[at], t[at], 1.0, k, True, fl.TokenLogprobs(*(o[at] for o in outs)))


@pytest.mark.parametrize("dtype,vocab", [(torch.float32, 9), (torch.bfloat16, 600), (torch.float32, 1030)])
def test_gradients_of_rows_past_one_launch(dev, dtype, vocab):
    print(f"[case] token_logprobs gradients, 2^20 + 9 rows of {vocab} {dtype}", flush=True)
    rows, half = (1 << 20) + 9, 1 << 19
    g = torch.Generator(device=dev).manual_seed(vocab)
    x = (torch.randn(rows + vocab, device=dev, generator=g) * 3).to(dtype).as_strided((rows, vocab), (1, 1))
    t = torch.randint(0, vocab, (rows,), device=dev, generator=g)
    t[::7] = -100
    ups = [torch.randn(*s, device=dev, generator=g) for s in ((rows,), (rows,), (rows, 3))]

    def grad(lo, hi):
        z = x[lo:hi].detach().requires_grad_()
        r = fl.token_logprobs(z, t[lo:hi], top_k=3, entropy=True)
        return torch.autograd.grad([r.logprobs, r.entropy, r.top_logprobs], z, [u[lo:hi] for u in ups])[0]

    whole = grad(0, rows)
    for lo, hi in ((0, half), (half, 2 * half), (2 * half, rows)):
        assert torch.equal(whole[lo:hi], grad(lo, hi)), lo
    at = torch.tensor([0, 1, 8, 2 * half - 1, 2 * half, 2 * half + 1, rows - 1], device=dev)
    check_grad(x[at], t[at], 1.0, 3, *(u[at] for u in ups), whole[at])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [3, 300, 8193])
def test_gradients_of_alternatives_of_special_rows(dev, vocab, dtype):
    """Masked alternatives, ties, fewer logits left than alternatives, with tokens among the alternatives and ignored."""
    print(f"[case] token_logprobs gradients of special rows' alternatives V={vocab} {dtype}", flush=True)
    x = special_rows(dev, vocab, dtype)
    for k in sorted({min(vocab, n) for n in (1, 5, 64)}):
        gen = torch.Generator(device=dev).manual_seed(k)
        g, h, gt = (torch.randn(*s, device=dev, generator=gen) for s in ((18,), (18,), (18, k)))
        for token in (0, vocab - 1, -100):
            t = torch.full((18,), token, device=dev)
            for use in ((0, 0, 1), (1, 1, 1)):
                z = x.clone().requires_grad_()
                r = fl.token_logprobs(z, t, top_k=k, entropy=True)
                outs, ups = ([a for a, u in zip(l, use) if u]
                             for l in ((r.logprobs, r.entropy, r.top_logprobs), (g, h, gt)))
                got, = torch.autograd.grad(outs, z, ups)
                check_grad(x, t, 1.0, k, *(o if u else None for o, u in zip((g, h, gt), use)), got)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [300, 8193, 70001])
def test_alternatives_around_the_groups_that_bound_them(dev, vocab, dtype):
    """The largest number of alternatives that 64 groups bound, and one more: special rows, ordinary ones, and logits
    that lie in a few groups alone."""
    print(f"[case] 32 and 33 alternatives V={vocab} {dtype}", flush=True)
    g = torch.Generator(device=dev).manual_seed(vocab)
    x = torch.cat((special_rows(dev, vocab, dtype), (torch.randn(6, vocab, device=dev, generator=g) * 3).to(dtype)))
    x[20, :200] += 40
    x[21, torch.arange(vocab, device=dev) % 64 < 31] += 40
    x[22, torch.arange(vocab, device=dev) // 8 % 64 < 32] += 40
    t = torch.randint(0, vocab, (24,), device=dev, generator=g)
    for k in (32, 33):
        check_forward(x, t, 1.0, k, True, fl.token_logprobs(x, t, top_k=k, entropy=True))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("temperature", [2.0 ** -20, 2.0 ** -9, 2.0 ** 9, 2.0 ** 20])
def test_temperatures_at_the_ends_of_their_range(dev, temperature, dtype):
    print(f"[case] token_logprobs T={temperature} {dtype}", flush=True)
    for vocab in (501, 16385):
        x, t = make(dev, 6, vocab, dtype, vocab)
        z = x.clone().requires_grad_()
        r = fl.token_logprobs(z, t, temperature=temperature, top_k=5, entropy=True)
        check_forward(x, t, temperature, 5, True, fl.TokenLogprobs(*(o.detach() for o in r)))
        g = torch.Generator(device=dev).manual_seed(1)
        ups = [torch.randn(*s, device=dev, generator=g) for s in ((6,), (6,), (6, 5))]
        got, = torch.autograd.grad([r.logprobs, r.entropy, r.top_logprobs], z, ups)
        check_grad(x, t, temperature, 5, *ups, got)


@pytest.mark.parametrize("vocab", [501, 8193])
def test_logits_far_from_zero(dev, vocab):
    """A maximum on both sides of 2^20 over log2(e) / T, where the difference is taken another way: differences of a few
    units, in steps of 1 / 16, keep their digits."""
    print(f"[case] token_logprobs, logits far from zero V={vocab}", flush=True)
    base = 2.0 ** 20 / 1.4426950408889634
    offsets = torch.tensor([0.5 * base, base - 20, base - 1, base + 20, 1.4 * base, -base - 20, -base + 20, 0.0], device=dev)
    x, t = make(dev, 8, vocab, torch.float32, vocab)
    x = x + offsets[:, None]
    g = torch.Generator(device=dev).manual_seed(1)
    ups = [torch.randn(*s, device=dev, generator=g) for s in ((8,), (8,), (8, 5))]
    for temperature in (1.0, 0.75):
        z = x.clone().requires_grad_()
        r = fl.token_logprobs(z, t, temperature=temperature, top_k=5, entropy=True)
        check_forward(x, t, temperature, 5, True, fl.TokenLogprobs(*(o.detach() for o in r)))
        got, = torch.autograd.grad([r.logprobs, r.entropy, r.top_logprobs], z, ups)
        check_grad(x, t, temperature, 5, *ups, got)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradient_of_the_longest_row(dev, dtype):
    print(f"[case] token_logprobs gradient V=2^23 {dtype}", flush=True)
    vocab = 1 << 23
    x, t = make(dev, 2, vocab, dtype, 5)
    x[1, : vocab // 2] = float("-inf")
    t[0] = vocab - 1
    ups = [torch.randn(*s, device=dev, generator=torch.Generator(device=dev).manual_seed(1)) for s in ((2,), (2,), (2, 5))]
    z = x.clone().requires_grad_()
    r = fl.token_logprobs(z, t, top_k=5, entropy=True)
    check_forward(x, t, 1.0, 5, True, fl.TokenLogprobs(*(o.detach() for o in r)))
    got, = torch.autograd.grad([r.logprobs, r.entropy, r.top_logprobs], z, ups)
    check_grad(x, t, 1.0, 5, *ups, got)


def test_rows_past_32_bits(dev):
    """More than 2^32 rows in two groups, which all read one of three rows: where a row lies is a 64-bit quotient."""
    print("[case] token_logprobs, 3 x (2^31 - 5) rows", flush=True)
    inner = (1 << 31) - 5
    line = torch.tensor([0.5, -1.0, 2.0, 0.25], device=dev)
    x = line.as_strided((3, inner, 2), (1, 0, 1))
    t = torch.ones(1, 1, dtype=torch.long, device=dev).expand(3, inner)
    got = fl.token_logprobs(x, t).logprobs
    exp = torch.log_softmax(line.double().unfold(0, 2, 1), -1)[:, 1]
    for i in range(3):
        low, high = float(got[i].min()), float(got[i].max())
        assert low == high and abs(low - float(exp[i])) <= 16 * U * (1 + abs(float(exp[i]))), i
