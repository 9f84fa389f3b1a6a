"""Embedding, gated scan, orthogonalization and Muon on the host: refusals (Python's and the C ABI's, none of which reaches
a launch), workspaces, the optimizer's bookkeeping and the stock form that a differentiable backward runs.
"""
from __future__ import annotations

import copy
import ctypes
import pickle

import pytest
import torch

import fields_lm_amd as fl
from fields_lm_amd import _native as nat
from fields_lm_amd import _train as train


def test_cpu_tensors_are_refused():
    x = torch.randn(4, 6, requires_grad=True)
    with pytest.raises(RuntimeError):
        fl.embedding(torch.zeros(3, dtype=torch.long), x)
    with pytest.raises(RuntimeError):
        fl.gated_scan(torch.rand(2, 3), torch.rand(2, 3, 4))
    with pytest.raises(RuntimeError):
        fl.orthogonalize(x)
    with pytest.raises(RuntimeError):
        fl.muon_step([x.detach()], [torch.ones(4, 6)], [torch.zeros(4, 6)])


def test_fake_tensors_are_refused():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x, t = torch.empty(4, 6, device="cuda"), torch.zeros(3, dtype=torch.long, device="cuda")
        d = torch.empty(2, 3, 4, device="cuda")
    for call in (lambda: fl.embedding(t, x), lambda: fl.gated_scan(d, d), lambda: fl.orthogonalize(x),
                 lambda: fl.muon_step([x], [x], [x])):
        with pytest.raises(TypeError):
            call()


def test_types_and_shapes_are_refused():
    t, w = torch.zeros(3, dtype=torch.long), torch.randn(5, 4)
    for bad in ((t.int(), w), (t, w.half()), (t, 3), (None, w), (t, w.to_sparse())):
        with pytest.raises(TypeError):
            fl.embedding(*bad)
    for bad in ((t, w[0]), (t, w[:0]), (t, w[:, :0])):
        with pytest.raises(ValueError):
            fl.embedding(*bad)
    for kw in (dict(padding_idx=5), dict(padding_idx=-6), dict(scale=float("inf"))):
        with pytest.raises(ValueError):
            fl.embedding(t, w, **kw)
    for dtype in (torch.float16, 3):
        with pytest.raises(TypeError):
            fl.embedding(t, w, dtype=dtype)
    g, d, s = torch.rand(2, 5, 3), torch.rand(2, 5, 3), torch.rand(2, 3)
    for bad in ((g.half(), d, s), (g, d.double(), s), (g, d, s.bfloat16()), (None, d), (g, d, 3.0)):
        with pytest.raises(TypeError):
            fl.gated_scan(*bad)
    for bad in ((g[:, :4], d), (g[..., :2], d), (g[0], d), (g, d[0]), (g, d, s[:1])):
        with pytest.raises(ValueError):
            fl.gated_scan(*bad)


def test_forward_mode_is_refused():
    from torch.autograd import forward_ad

    with forward_ad.dual_level():
        x = forward_ad.make_dual(torch.randn(3, 4, 5), torch.randn(3, 4, 5))
        with pytest.raises(NotImplementedError):
            fl.gated_scan(x, torch.randn(3, 4, 5))
        with pytest.raises(NotImplementedError):
            fl.embedding(torch.zeros(2, dtype=torch.long), x[0])


def test_steps_and_coefficients_are_refused():
    x = torch.randn(4, 5)
    for kw in (dict(steps=0), dict(steps=65), dict(eps=-1.0), dict(eps=float("nan")), dict(coefficients=(30.0, 50.0, 9.0)),
               dict(coefficients=(float("nan"), 0.0, 0.0)), dict(coefficients=(2.0, 0.0, 0.0), steps=11)):
        with pytest.raises(ValueError):
            fl.orthogonalize(x, **kw)
    with pytest.raises(TypeError):
        fl.orthogonalize(x, steps=2.5)
    for kw in (dict(momentum=1.0), dict(momentum=-0.1), dict(lr=-1.0), dict(lr=float("nan")), dict(weight_decay=-1.0),
               dict(adjust_lr="none")):
        with pytest.raises(ValueError):
            fl.muon_step([x], [x.clone()], [torch.zeros(4, 5)], **kw)


@pytest.mark.parametrize("steps,abc", [(5, (3.4445, -4.7750, 2.0315)), (64, (1.5, -0.5, 0.0)), (10, (2.0, 0.0, 0.0)),
                                       (8, (1.875, -1.25, 0.375)), (3, (-4.0, 1.0, 0.5)), (2, (0.0, 0.0, 0.0))])
def test_bounds_hold(steps, abc):
    """What the check lets pass keeps singular values and factors within 1024, on a fine grid of them."""
    lib = nat.load()
    a, b, c = abc
    if lib.fl_orthogonalize_check(steps, a, b, c) == nat.FL_OK:
        x = torch.linspace(0, 1, 100_001, dtype=torch.float64)
        for _ in range(steps):
            p = a + b * x ** 2 + c * x ** 4
            x = (p * x).abs()
            assert float(p.abs().max()) <= 1024 and float(x.max()) <= 1024
    else:
        assert (steps, abc) == (3, (-4.0, 1.0, 0.5))
    assert lib.fl_orthogonalize_check(10, 2.0, 0.0, 0.0) == nat.FL_OK
    assert lib.fl_orthogonalize_check(11, 2.0, 0.0, 0.0) == nat.FL_ERR_INVALID_ARGUMENT


def _sizes(*values):
    return (ctypes.c_int64 * len(values))(*values)


def test_abi_refusals():
    lib = nat.load()
    tokens = (ctypes.c_int64 * 4)()
    data = (ctypes.c_float * 64)()
    at, k = ctypes.addressof(data), ctypes.addressof(tokens)
    bad, dtype, ws = nat.FL_ERR_INVALID_ARGUMENT, nat.FL_ERR_DTYPE, nat.FL_ERR_WORKSPACE

    def rows(n=4, w=at, wt=0, V=2, D=4, stride=4, out=at, ot=0, t=k):
        return lib.fl_embedding(t, n, w, wt, V, D, stride, 1.0, 0, -1, out, ot, None)

    assert rows(wt=2) == dtype == rows(ot=-1)
    assert {rows(n=-1), rows(V=0), rows(D=0), rows(stride=-1), rows(w=None), rows(out=None), rows(t=None), rows(w=at + 2),
            rows(t=k + 4)} == {bad}
    assert rows(n=0) == nat.FL_OK

    def grad(n=4, g=at, gt=0, V=2, D=4, out=at, ot=0, w=at, size=1 << 20, t=k):
        return lib.fl_embedding_backward(t, n, g, gt, V, D, -1, 1.0, out, ot, w, size, None)

    assert grad(gt=2) == dtype == grad(ot=7)
    assert {grad(n=-1), grad(V=0), grad(g=None), grad(out=None), grad(t=None), grad(out=at + 1), grad(w=at + 4)} == {bad}
    assert grad(w=None) == ws == grad(size=1)
    assert lib.fl_embedding_backward_workspace_bytes(-1, 2, 4) == 0

    def scan(a=at, at_=0, u=at, ut=0, B=1, T=2, C=3, out=at, w=at, size=1 << 20, sb=6, st=3):
        return lib.fl_gated_scan(a, at_, 0, sb, st, u, ut, sb, st, B, T, C, None, None, None, out, w, size, None)

    assert scan(at_=3) == dtype == scan(ut=2)
    assert {scan(a=None), scan(u=None), scan(out=None), scan(B=0), scan(T=0), scan(C=0), scan(B=1 << 40), scan(T=1 << 40),
            scan(C=1 << 40), scan(sb=-1), scan(st=-1), scan(a=at + 2), scan(w=at + 4)} == {bad}
    # (a workspace is asked for at any size)
    assert scan(w=None, T=5000) == ws == scan(size=0, T=5000)

    def back(starts=at, g=at, ga=at, gu=at, w=at, size=1 << 20):
        return lib.fl_gated_scan_backward(at, 0, 0, 6, 3, at, 0, 6, 3, 1, 5000, 3, starts, g, None, ga, gu, None, w, size, None)

    assert {back(starts=None), back(gu=None), back(g=at + 1), back(ga=at + 2), back(starts=at + 2)} == {bad}
    assert back(w=None) == ws == back(size=8)
    assert lib.fl_gated_scan_workspace_bytes(0, 1, 1, 0) == 0

    ptrs = (ctypes.c_void_p * 1)(at)
    odd = (ctypes.c_void_p * 1)(at + 2)
    none = (ctypes.c_void_p * 1)(None)
    m, n = _sizes(4), _sizes(5)

    def orth(x=ptrs, t=0, r=m, c=n, steps=5, a=3.4445, eps=1e-7, out=ptrs, w=at, size=1 << 40, count=1):
        return lib.fl_orthogonalize(count, x, t, r, c, steps, a, -4.775, 2.0315, eps, out, w, size, None)

    assert orth(t=5) == dtype
    assert {orth(x=none), orth(x=odd), orth(out=none), orth(x=None), orth(r=_sizes(-1)), orth(c=_sizes(1 << 21)),
            orth(r=_sizes(1 << 20), c=_sizes(1 << 20)), orth(steps=0), orth(steps=65), orth(a=float("inf")), orth(eps=-1.0),
            orth(count=0), orth(w=at + 8)} == {bad}
    assert orth(w=None) == ws == orth(size=64)
    scale = (ctypes.c_double * 1)(1.0)

    def muon(p=ptrs, g=ptrs, buf=ptrs, t=0, momentum=0.9, rate=scale, w=at, size=1 << 40):
        return lib.fl_muon_step(1, p, g, t, buf, m, n, 0.1, None, rate, momentum, 1, 0.1, 5, 3.4445, -4.775, 2.0315, 1e-7,
                                None, w, size, None)

    assert muon(t=2) == dtype
    assert {muon(p=none), muon(g=odd), muon(buf=none), muon(momentum=1.0), muon(momentum=float("nan")), muon(rate=None)} == {bad}
    assert muon(w=None) == ws == muon(size=0)


@pytest.mark.parametrize("V", [1, 2048, 2049, 1 << 23])
@pytest.mark.parametrize("D", [1, 2, 3, 4, 5, 64])
def test_gradient_launches_hold_few_enough_threads(D, V):
    """The gradient's sums are launched with 256 threads to each bucket and each piece behind a bucket's first, their join
    with 512 to each such piece; a dimension of a launch holds fewer than 2^32 threads. The number of pieces is read off the
    workspace: 4 bytes each, a bit to each of two pieces' rows in words of 4, and two places of fp32 rows."""
    lib = nat.load()
    rows = 1
    while -(-V // rows) > 2048:
        rows *= 2
    buckets = -(-V // rows)
    for n in (1 << 20, (1 << 28) - 1, 1 << 28, (1 << 28) + 1, 1 << 29, (1 << 30) - 1, 1 << 30):
        size = lib.fl_embedding_backward_workspace_bytes(n, V, D)
        fixed = 64 * 2048 * 4 + (buckets + 1) * 4 + 4 + buckets * 4 + n * 8
        per = 4 + 2 * 4 * -(-rows // 32) + 2 * rows * D * 4
        extras = (size - fixed) // per  # (rounded up by what the parts are aligned with: 6 times up to 15 bytes)
        assert 0 < extras <= n // 32 + 8
        assert extras * 512 < 1 << 32 and (extras + buckets) * 256 < 1 << 32, (n, extras)


def test_workspaces_stay_within_groups():
    """Up to 2 GiB where the matrices fit in that, whatever their number."""
    lib = nat.load()
    many = lib.fl_orthogonalize_workspace_bytes(400, _sizes(*[1024] * 400), _sizes(*[1024] * 400))
    assert 1 << 30 < many <= (2 << 30) + (1 << 20)
    one = lib.fl_orthogonalize_workspace_bytes(1, _sizes(16384), _sizes(16384))
    assert one > 2 << 30


def test_stock_scan_gradients():
    """Against a loop over the steps in float64, and differentiable."""
    g = torch.Generator().manual_seed(1)
    for token in (False, True):
        a = torch.rand((2, 11) if token else (2, 11, 3), generator=g, dtype=torch.float64, requires_grad=True)
        u = torch.randn(2, 11, 3, generator=g, dtype=torch.float64, requires_grad=True)
        s = torch.randn(2, 3, generator=g, dtype=torch.float64, requires_grad=True)
        w, k = torch.randn(2, 11, 3, generator=g), torch.randn(2, 3, generator=g)
        h, now = [], s
        for t in range(11):
            now = (a[:, t, None] if token else a[:, t]) * now + u[:, t]
            h.append(now)
        exp = torch.autograd.grad((torch.stack(h, 1) * w).sum() + (now * k).sum(), (a, u, s))
        low = [t.detach().float().requires_grad_() for t in (a, u, s)]
        got = train.stock_scan_gradients(*low, w, k)
        assert all(torch.allclose(x.double(), y, rtol=0, atol=1e-4) for x, y in zip(got, exp))
        assert all(x.requires_grad for x in got)
        got = train.stock_scan_gradients(low[0], low[1], None, w, None)
        assert got[2] is None and got[0].shape == a.shape


def _steps64(a, u, s, w, k):
    """The gradients of the scan, a loop over its steps in float64."""
    a, u, s = (t.detach().double().requires_grad_() for t in (a, u, s))
    h, now = [], s
    for t in range(u.shape[1]):
        now = (a[:, t, None] if a.ndim == 2 else a[:, t]) * now + u[:, t]
        h.append(now)
    return torch.autograd.grad((torch.stack(h, 1) * w).sum() + (now * k).sum(), (a, u, s))


@pytest.mark.parametrize("token", [False, True])
def test_stock_scan_gradients_over_tiles(token):
    """Gates above 1, whose product over all steps leaves fp32 while those within a tile are finite, states of 0 before a late
    drive, gradients that end early: everything the formulas form is an ordinary number."""
    T, late, early = 2500, 2490, 5
    a = torch.full((1, T) if token else (1, T, 2), 1.05, requires_grad=True)
    u = torch.zeros(1, T, 2)
    u[:, late:] = torch.linspace(0.5, 1.5, 20).view(1, 10, 2)
    u.requires_grad_()
    s = torch.zeros(1, 2, requires_grad=True)
    w = torch.zeros(1, T, 2)
    w[:, early] = 1.0
    # forward sums at most 10 terms of at most 10 gates each, backward 6 gates: 30 roundings are ample
    states, last = train.gated_scan_ops(a, u, s)
    now = torch.zeros(2, dtype=torch.float64)
    for t in range(late, T):
        now = 1.05 * now + u.detach().double()[0, t]
    assert bool(states.isfinite().all()) and torch.allclose(last.double()[0], now, rtol=30 * 2.0 ** -24, atol=0)
    exp = _steps64(a, u, s, w, torch.zeros(1, 2))
    got = train.stock_scan_gradients(a, u, s, w, None)
    for x, y in zip(got, exp):
        assert bool(x.isfinite().all())
        assert bool(((x.detach().double() - y).abs() <= 30 * 2.0 ** -24 * y.abs() + 1e-30).all())


def test_muon_bookkeeping():
    with pytest.raises(ValueError, match="matrices"):
        fl.Muon([torch.zeros(3)])
    with pytest.raises(TypeError):
        fl.Muon([torch.zeros(3, 3, dtype=torch.float16)])
    for kw in (dict(lr=-1.0), dict(momentum=1.0), dict(weight_decay=-1.0), dict(steps=0), dict(eps=-1.0), dict(adjust_lr="x"),
               dict(coefficients=(50.0, 50.0, 50.0)), dict(max_grad_norm=-1.0)):
        with pytest.raises(ValueError):
            fl.Muon([torch.zeros(3, 3)], **kw)
    p = torch.nn.Parameter(torch.zeros(3, 4))
    opt = fl.Muon([p], max_grad_norm=2.0)
    with pytest.raises(ValueError):
        opt.add_param_group(dict(params=[torch.nn.Parameter(torch.zeros(3))]))
    assert len(opt.param_groups) == 1
    assert opt.step() is None and opt.step(lambda: 5.0) == 5.0
    for twin in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        assert twin.max_grad_norm == 2.0 and twin.param_groups[0]["coefficients"] == opt.param_groups[0]["coefficients"]
    state = opt.state_dict()
    state["state"] = {0: dict(momentum_buffer=torch.ones(3, 4))}
    opt.load_state_dict(state)
    assert torch.equal(opt.state[p]["momentum_buffer"], torch.ones(3, 4))
    for wrong in (dict(momentum_buffer=torch.ones(3, 5)), dict(momentum_buffer=torch.ones(3, 4).bfloat16()),
                  dict(exp_avg=torch.ones(3, 4))):
        state["state"] = {0: wrong}
        with pytest.raises(ValueError):
            opt.load_state_dict(state)
    adam = fl.AdamW([torch.nn.Parameter(torch.zeros(3, 4))])
    with pytest.raises(ValueError, match="lacks"):
        opt.load_state_dict(adam.state_dict())
    with pytest.raises(ValueError, match="lacks"):
        adam.load_state_dict(opt.state_dict())


@pytest.mark.parametrize("make,names", [(lambda p: fl.Muon([p]), ("momentum_buffer",)),
                                        (lambda p: fl.AdamW([p]), ("exp_avg", "exp_avg_sq"))], ids=["Muon", "AdamW"])
def test_states_of_other_shapes_and_strides(make, names):
    """A state of as many values in another shape belongs to other positions: refused, and nothing is changed. One of other
    strides is loaded as the contiguous one that a step takes."""
    p = torch.nn.Parameter(torch.zeros(3, 4))
    opt = make(p)
    turned = torch.arange(12.0).view(4, 3)
    rest = {} if len(names) == 1 else {"step": torch.ones((), dtype=torch.int64)}
    saved = opt.state_dict()
    for wrong in (turned, turned.view(2, 6), turned.view(1, 3, 4), turned.view(3, 4)[None].transpose(0, 1)):
        for name in names:
            state = {**rest, **{n: torch.zeros(3, 4) for n in names}, name: wrong}
            with pytest.raises(ValueError, match="shape"):
                opt.load_state_dict({**saved, "state": {0: state}})
            assert not opt.state
    opt.load_state_dict({**saved, "state": {0: {**rest, **{n: turned.t() for n in names}}}})
    for name in names:
        got = opt.state[p][name]
        assert got.is_contiguous() and torch.equal(got, turned.t())


def test_flat_states():
    """AdamW goes value by value, and takes a state that lies flat; a flat momentum says nothing of rows and columns."""
    p = torch.nn.Parameter(torch.zeros(3, 4))
    adam, muon = fl.AdamW([p]), fl.Muon([p])
    flat = torch.arange(12.0)
    adam.load_state_dict({**adam.state_dict(), "state": {0: dict(step=torch.ones((), dtype=torch.int64), exp_avg=flat,
                                                                 exp_avg_sq=flat)}})
    assert torch.equal(adam.state[p]["exp_avg"].view(-1), flat)
    with pytest.raises(ValueError, match="shape"):
        muon.load_state_dict({**muon.state_dict(), "state": {0: dict(momentum_buffer=flat)}})


def _polar_of_high_parts(x, steps, abc):
    """Steps whose products' operands have the 11 bits of fp16."""
    def high(t):
        return (t * 1024).half().float() / 1024

    tall = x.shape[0] > x.shape[1]
    y = x.t() if tall else x
    y = (y / (y.double().norm() + 1e-7)).float()
    for _ in range(steps):
        y = high(y)
        gram = high(y @ y.t())
        y = high(abc[0] * torch.eye(len(y)) + abc[1] * gram + abc[2] * (gram @ gram)) @ y
    return y.t() if tall else y


@pytest.mark.parametrize("steps", [1, 2, 3, 5, 7, 10])
def test_the_bound_of_orthogonalization_finds_mistakes(steps):
    """What the GPU tests' bound lets pass is neither zeros nor a step fewer nor, where errors are not magnified past
    it, operands of 11 bits."""
    import test_gpu_muon as muon

    cpu = torch.device("cpu")
    found = {"zeros": 0, "fewer": 0, "high": 0}
    for abc in muon.ABCS:
        for shape in ((7, 5), (33, 200), (130, 60), (150, 140)):
            for kind in ("plain", "rows", "low", "wide"):
                x = muon.spectrum(cpu, shape, steps) if kind == "wide" else muon.matrices(cpu, shape, steps, kind)

                def far(got):
                    return muon.beyond(got, x, steps, abc)[0]

                right = muon.polar64(x, steps, abc)
                bound = muon.beyond(right, x, steps, abc)[1]
                assert far(right.float()) <= 0
                if bound > muon.SAYS:
                    continue
                assert far(torch.zeros_like(right)) > 0
                found["zeros"] += 1
                if abc == muon.ABC:  # (the others stand still where they have arrived)
                    assert far(muon.polar64(x, steps - 1, abc)) > 0
                    found["fewer"] += 1
                found["high"] += far(_polar_of_high_parts(x, steps, abc)) > 0
    assert found["zeros"] >= 48 and found["fewer"] >= 8 and found["high"] >= (48 if steps <= 3 else 20), found
