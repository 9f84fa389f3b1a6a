"""GPU: embedding rows and the weight's gradient against 64-bit formulas.

u = 2^-24. A row is one product in fp32 (u), rounded to its type (half a step, eps / 2). A gradient's row is a sum of k
products-free terms in fp32, in any fixed grouping at most k roundings of partial sums, each at most the sum of the terms'
magnitudes, then one product: (k + 1) u sum |g| |s|, and the rounding to its type.
"""
from __future__ import annotations

import math

import pytest
import torch

import fields_lm_amd as fl

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm device")
    return torch.device("cuda:0")


def half_step(dtype):
    return 0.0 if dtype == F32 else torch.finfo(dtype).eps / 2


def expected_grad(tokens, g, V, scale, padding):
    """The gradient in 64 bits, the sums of magnitudes and the counts."""
    flat, g = tokens.reshape(-1), g.reshape(tokens.numel(), -1).double()
    kept = (flat >= 0) & (flat < V)
    if padding is not None:
        kept &= flat != padding % V
    out = torch.zeros(V, g.shape[1], dtype=torch.float64, device=g.device)
    size, count = torch.zeros_like(out), torch.zeros(V, dtype=torch.float64, device=g.device)
    out.index_add_(0, flat[kept], g[kept])
    size.index_add_(0, flat[kept], g[kept].abs())
    count.index_add_(0, flat[kept], torch.ones_like(flat[kept], dtype=torch.float64))
    return out * scale, size * abs(scale), count


def check_grad(got, tokens, g, scale, padding):
    exp, size, count = expected_grad(tokens, g, got.shape[0], scale, padding)
    bound = (count[:, None] + 1) * U * size + half_step(got.dtype) * exp.abs() + 1e-40
    assert bool(((got.double() - exp).abs() <= bound).all())
    assert bool((got[count == 0] == 0).all())


SHAPES = [((1,), 1, 1), ((1,), 7, 3), ((64,), 100, 64), ((3, 5), 11, 7), ((2, 33), 500, 24), ((4, 77), 37, 129),
          ((5, 200), 1000, 513), ((3, 333), 3201, 714), ((2, 1030), 64, 8), ((1, 4097), 5, 1030), ((8, 1024), 16_384, 72)]


@pytest.mark.parametrize("types", [(F32, F32), (F32, BF16), (BF16, BF16), (BF16, F32)], ids=str)
@pytest.mark.parametrize("shape,V,D", SHAPES, ids=str)
def test_embedding_and_its_gradient(dev, shape, V, D, types):
    print(f"[case] embedding {shape} V={V} D={D} {types}", flush=True)
    wt, ot = types
    gen = torch.Generator(device=dev).manual_seed(V + D)
    tokens = torch.randint(0, V, shape, device=dev, generator=gen)
    tokens = torch.where(torch.rand(shape, device=dev, generator=gen) < 0.2, V // 2, tokens)  # one that comes often
    weight = torch.randn(V, D, device=dev, generator=gen).to(wt).requires_grad_()
    g = torch.randn(*shape, D, device=dev, generator=gen).to(ot)
    for scale, padding in ((1.0, None), (math.sqrt(D), V // 2), (-0.37, -1)):
        rows = fl.embedding(tokens, weight, scale=scale, padding_idx=padding, dtype=ot)
        assert rows.dtype == ot and rows.shape == (*shape, D)
        exp = weight.detach().double()[tokens] * torch.tensor(scale, dtype=F32).double()
        assert bool(((rows.detach().double() - exp).abs() <= (U + half_step(ot)) * exp.abs() + 1e-40).all())
        if scale == 1.0 and wt == ot:
            assert torch.equal(rows.detach(), weight.detach()[tokens])
        got, = torch.autograd.grad(rows, weight, g)
        assert got.dtype == wt and got.shape == (V, D)
        check_grad(got, tokens, g, torch.tensor(scale, dtype=F32).item(), padding)
        again, = torch.autograd.grad(fl.embedding(tokens, weight, scale=scale, padding_idx=padding, dtype=ot), weight, g)
        assert torch.equal(got, again)


@pytest.mark.parametrize("n", [1, 63, 64, 65, 1000, 16_384, 16_385, 40_000])
@pytest.mark.parametrize("V", [1, 31, 33, 2049, 70_001])
def test_gradient_of_counts_and_vocabularies(dev, n, V):
    """One token alone, all tokens the same, each of its own, words by their frequency."""
    print(f"[case] embedding gradient n={n} V={V}", flush=True)
    gen = torch.Generator(device=dev).manual_seed(n + V)
    D = 40
    g = torch.randn(n, D, device=dev, generator=gen)
    same = torch.full((n,), V - 1, device=dev)
    own = torch.arange(n, device=dev) % V
    frequent = torch.exp(torch.rand(n, device=dev, generator=gen) * math.log(V + 1)).long().clamp_(1, V) - 1
    for tokens in (same, own, own.flip(0), frequent):
        weight = torch.zeros(V, D, device=dev, requires_grad=True)
        got, = torch.autograd.grad(fl.embedding(tokens, weight), weight, g)
        check_grad(got, tokens, g, 1.0, None)


@pytest.mark.parametrize("V,D,n", [(1 << 23, 3, 5000), ((1 << 23) - 5, 1, 70), (3, 5000, 700), (1, 1, 200_000), (4097, 33, 100_000)])
def test_ends_of_the_ranges(dev, V, D, n):
    """The largest vocabulary, wide rows, many tokens, a bucket of few rows and one of thousands."""
    print(f"[case] embedding gradient V={V} D={D} n={n}", flush=True)
    gen = torch.Generator(device=dev).manual_seed(n)
    g = torch.randn(n, D, device=dev, generator=gen)
    tokens = torch.randint(0, V, (n,), device=dev, generator=gen)
    tokens[::3] = V - 1
    tokens[1::7] = max(0, V - 1500)
    weight = torch.zeros(V, D, device=dev, requires_grad=True)
    got, = torch.autograd.grad(fl.embedding(tokens, weight), weight, g)
    check_grad(got, tokens, g, 1.0, None)


def test_refuses_a_vocabulary_past_the_largest(dev):
    print("[case] embedding, vocabulary past the largest", flush=True)
    w = torch.empty(1, 1, device=dev).expand((1 << 23) + 1, 1)
    with pytest.raises(ValueError):
        fl.embedding(torch.zeros(1, dtype=torch.long, device=dev), w)


def test_tokens_outside(dev):
    print("[case] embedding, tokens outside", flush=True)
    weight = torch.randn(9, 20, device=dev, requires_grad=True)
    tokens = torch.tensor([3, -1, 9, 0, 8, 1 << 40, -(1 << 40), 3], device=dev)
    rows = fl.embedding(tokens, weight, scale=2.0)
    bad = torch.tensor([False, True, True, False, False, True, True, False], device=dev)
    assert bool(rows[bad].isnan().all()) and torch.equal(rows[~bad].detach(), weight.detach()[tokens[~bad]] * 2)
    g = torch.randn(8, 20, device=dev)
    got, = torch.autograd.grad(rows, weight, g)
    check_grad(got, tokens, g, 2.0, None)
    none = torch.tensor([-1, 9], device=dev)
    got, = torch.autograd.grad(fl.embedding(none, weight), weight, g[:2])
    assert bool((got == 0).all())


def test_no_tokens(dev):
    print("[case] embedding, no tokens", flush=True)
    weight = torch.randn(9, 20, device=dev, requires_grad=True)
    rows = fl.embedding(torch.zeros(3, 0, dtype=torch.long, device=dev), weight)
    assert rows.shape == (3, 0, 20)
    got, = torch.autograd.grad(rows.sum(), weight)
    assert got.shape == (9, 20) and bool((got == 0).all())


def test_special_values(dev):
    """Infinities and NaN of a weight or a gradient stay in their rows and columns."""
    print("[case] embedding, special values", flush=True)
    weight = torch.randn(6, 24, device=dev)
    weight[2, 3], weight[4, 5] = float("nan"), float("-inf")
    tokens = torch.tensor([0, 2, 4, 4, 1], device=dev)
    assert torch.equal(fl.embedding(tokens, weight).nan_to_num(7.0), weight[tokens].nan_to_num(7.0))
    g = torch.randn(5, 24, device=dev)
    g[1, 0], g[2, 1] = float("nan"), float("inf")
    w = weight.clone().requires_grad_()
    got, = torch.autograd.grad(fl.embedding(tokens, w), w, g)
    assert bool(got[2, 0].isnan()) and float(got[4, 1]) == float("inf")
    got[2, 0], got[4, 1] = 0.0, 0.0
    assert bool(got.isfinite().all())


def test_strides(dev):
    """Rows of a wider weight, a transposed weight, tokens that are a slice, upstream gradients of other strides."""
    print("[case] embedding, strides", flush=True)
    gen = torch.Generator(device=dev).manual_seed(5)
    wide = torch.randn(50, 61, device=dev, generator=gen)
    ids = torch.randint(0, 30, (6, 14), device=dev, generator=gen)
    for weight in (wide[:30, 1:42], wide.t()[:30, :20], wide[0].expand(30, 61), torch._neg_view(wide)[:30]):
        for tokens in (ids, ids[:, 1::2], ids.t(), ids[2].expand(4, 14)):
            leaf = weight.detach().requires_grad_()
            rows = fl.embedding(tokens, leaf)
            assert torch.equal(rows.detach(), weight[tokens])
            wide_g = torch.randn(*tokens.shape[::-1], leaf.shape[1], device=dev, generator=gen)
            g = wide_g.transpose(0, 1) if tokens.ndim == 2 else wide_g
            for up in (g, torch._neg_view(g), g[..., :1].expand(g.shape)):
                got, = torch.autograd.grad(rows, leaf, up, retain_graph=True)
                check_grad(got, tokens, up, 1.0, None)


def test_gradient_by_differences_and_of_the_gradient(dev):
    print("[case] embedding, differences", flush=True)
    gen = torch.Generator(device=dev).manual_seed(6)
    weight = torch.randn(12, 10, device=dev, generator=gen, requires_grad=True)
    tokens = torch.tensor([[3, 11, 3], [0, 5, 40]], device=dev)
    w = torch.randn(2, 3, 10, device=dev, generator=gen)
    w[1, 2] = 0
    d = torch.randn(12, 10, device=dev, generator=gen)

    def loss(x):
        rows = fl.embedding(tokens, x, scale=1.5, padding_idx=5)
        return (torch.where(w == 0, 0.0, rows.double()) * w.double()).sum()

    got, = torch.autograd.grad(loss(weight), weight)
    d[5] = 0
    step = 2.0 ** -6
    moved = (loss(weight.detach() + step * d) - loss(weight.detach() - step * d)) / (2 * step)
    # rows carry 2 u each (the sum and the product), the quotient divides that by the step
    bound = 4 * U * float((fl.embedding(tokens.clamp(max=11), weight.detach().abs() + d.abs()) * 1.5 * w.abs()).sum()) / step
    assert abs(float((got.double() * d.double()).sum()) - float(moved)) <= bound

    g = torch.randn(2, 3, 10, device=dev, generator=gen, requires_grad=True)
    grad, = torch.autograd.grad(fl.embedding(tokens, weight, scale=1.5, padding_idx=5), weight, g, create_graph=True)
    v = torch.randn(12, 10, device=dev, generator=gen, requires_grad=True)
    back, = torch.autograd.grad((grad * v).sum(), g, create_graph=True)
    exp = torch.where(((tokens == 5) | (tokens > 11))[..., None], 0.0, v.detach()[tokens.clamp(max=11)] * 1.5)
    assert torch.equal(back.detach(), exp)
    third, = torch.autograd.grad((back * g.detach()).sum(), v)
    check_grad(third, tokens, g.detach(), 1.5, 5)


def test_captured_in_a_graph(dev):
    print("[case] embedding, graph", flush=True)
    gen = torch.Generator(device=dev).manual_seed(7)
    weight = torch.randn(300, 65, device=dev, generator=gen, requires_grad=True)
    tokens = torch.randint(0, 300, (4, 90), device=dev, generator=gen)
    g = torch.randn(4, 90, 65, device=dev, generator=gen)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.autograd.grad(fl.embedding(tokens, weight), weight, g)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        rows = fl.embedding(tokens, weight)
        grad, = torch.autograd.grad(rows, weight, g)
    for i in range(4):
        tokens.copy_(torch.randint(0, 300 if i < 3 else 2, (4, 90), device=dev, generator=gen))
        g.copy_(torch.randn(4, 90, 65, device=dev, generator=gen))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(rows, weight.detach()[tokens])
        check_grad(grad, tokens, g, 1.0, None)
        leaf = weight.detach().clone().requires_grad_()
        eager, = torch.autograd.grad(fl.embedding(tokens, leaf), leaf, g)
        assert torch.equal(eager, grad)


def test_a_captured_backward_refuses_leaves_of_the_default_stream(dev):
    print("[case] embedding, capture beside an eager graph", flush=True)
    weight = torch.randn(30, 16, device=dev, requires_grad=True)
    tokens = torch.arange(8, device=dev)
    eager = fl.embedding(tokens, weight)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with pytest.raises(RuntimeError, match="default stream"):
        with torch.cuda.graph(graph, stream=side):
            torch.autograd.grad(fl.embedding(tokens, weight).sum(), weight)
    torch.cuda.synchronize()
    eager.sum().backward()
    assert float(weight.grad.sum()) == 8 * 16


def test_another_stream_and_a_weight_written_before_the_backward(dev):
    print("[case] embedding, streams", flush=True)
    gen = torch.Generator(device=dev).manual_seed(8)
    weight = torch.randn(500, 130, device=dev, generator=gen, requires_grad=True)
    tokens = torch.randint(0, 500, (2000,), device=dev, generator=gen)
    g = torch.randn(2000, 130, device=dev, generator=gen)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        rows = fl.embedding(tokens, weight)
        with torch.no_grad():
            weight.mul_(2.0)
        got, = torch.autograd.grad(rows, weight, g)
    side.synchronize()
    check_grad(got, tokens, g, 1.0, None)


def test_refuses(dev):
    print("[case] embedding, refusals", flush=True)
    w, t = torch.randn(5, 4, device=dev), torch.zeros(3, dtype=torch.long, device=dev)
    for bad in ((t.int(), w), (t, w.half()), (t, w.to_sparse()), (t.float(), w), (t, None)):
        with pytest.raises(TypeError):
            fl.embedding(*bad)
    for bad in ((t.cpu(), w), (t, w[0]), (t, w[:0]), (t, w[:, :0])):
        with pytest.raises(ValueError):
            fl.embedding(*bad)
    for padding in (5, -6):
        with pytest.raises(ValueError):
            fl.embedding(t, w, padding_idx=padding)
    with pytest.raises(TypeError):
        fl.embedding(t, w, dtype=torch.float16)
    with pytest.raises(ValueError):
        fl.embedding(t, w, scale=float("nan"))
    with pytest.raises(RuntimeError):
        torch.jit.trace(lambda x: fl.embedding(t, x), w)


def test_more_rows_than_a_launch_holds(dev):
    """2^26 + 8 rows of 512, a wave to each."""
    print("[case] embedding, 2^26 + 8 tokens", flush=True)
    n, V = 2 ** 26 + 8, 1000
    weight = torch.randn(V, 512, device=dev, dtype=torch.bfloat16)
    tokens = torch.randint(V, (n,), device=dev)
    out = fl.embedding(tokens, weight)
    for at in (0, 2 ** 25 - 4, 2 ** 26 - 4):
        assert torch.equal(out[at:at + 12], weight[tokens[at:at + 12]])
    some = torch.arange(0, n, 4099, device=dev)
    assert torch.equal(out[some], weight[tokens[some]])


@pytest.mark.parametrize("n", [2 ** 28 + 2048, 2 ** 29 + 7])
def test_gradient_of_more_pieces_than_a_launch_holds(dev, n):
    """Narrow rows and so many tokens that pieces of 32 would need 2^32 threads and more; whole numbers, whose sums are exact."""
    print(f"[case] embedding gradient, {n} tokens", flush=True)
    V = 2048
    tokens = torch.arange(n, device=dev) % V
    g = torch.randint(-1, 2, (n, 1), device=dev, dtype=torch.int8).float()
    weight = torch.zeros(V, 1, device=dev, requires_grad=True)
    got, = torch.autograd.grad(fl.embedding(tokens, weight), weight, g)
    whole = n // V * V
    exp = g[:whole].view(-1, V).sum(0, dtype=torch.float64)
    exp[:n - whole] += g[whole:, 0].double()
    assert torch.equal(got[:, 0].double(), exp)
