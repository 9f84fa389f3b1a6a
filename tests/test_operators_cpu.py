"""Token log probabilities, gradient norm and AdamW on the host: refusals (Python's and the C ABI's, none of which
reaches a launch), how rows and strides are seen, the optimizer's bookkeeping and the stock form that a
differentiable backward runs.
"""
from __future__ import annotations

import copy
import ctypes
import pickle

import pytest
import torch

import fields_lm_amd as fl
from fields_lm_amd import _native as nat
from fields_lm_amd import logprobs as L


def test_fake_tensors_are_refused():
    """Tensors that dispatch to Python have no memory behind their addresses."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x, t = torch.empty(4, 9, device="cuda"), torch.zeros(3, dtype=torch.long, device="cuda")
        step = torch.zeros(1, dtype=torch.long, device="cuda")
    for call in (lambda: fl.token_logprobs(x[1:], t), lambda: fl.grad_norm([x[1:]]),
                 lambda: fl.adamw_step([x], [x], [x], [x], step)):
        with pytest.raises(TypeError):
            call()


# ------------------------------------------------------------------ token_logprobs
def test_token_logprobs_refuses_what_it_does_not_take():
    x, t = torch.randn(3, 7), torch.zeros(3, dtype=torch.long)
    with pytest.raises(RuntimeError):
        fl.token_logprobs(x, t)
    for bad in ((x.half(), t), (x, t.int()), (x, 3), (None, t), (x.to_sparse(), t)):
        with pytest.raises(TypeError):
            fl.token_logprobs(*bad)
    with pytest.raises(ValueError):
        fl.token_logprobs(x, t[:2])
    with pytest.raises(ValueError):
        fl.token_logprobs(torch.tensor(1.0), t)
    with pytest.raises(ValueError):
        fl.token_logprobs(torch.randn(3, 0), t)
    with pytest.raises(ValueError):
        fl.token_logprobs(torch.empty(1).expand(3, (1 << 23) + 1), t)
    for temperature in (0.0, -1.0, float("nan"), float("inf"), 1e-40, 1e7):
        with pytest.raises(ValueError):
            fl.token_logprobs(x, t, temperature=temperature)
    for top_k in (-1, 8, 65):
        with pytest.raises(ValueError):
            fl.token_logprobs(x, t, top_k=top_k)
    with pytest.raises(ValueError):
        fl.token_logprobs(torch.randn(3, 100), t, top_k=65)
    with pytest.raises(TypeError):
        fl.token_logprobs(x, t, top_k=2.5)


def _rows(logits, tokens):
    x, t, outer, inner, so, si, to, ti = nat.host().where(logits, tokens)
    return x, t, (outer, inner, so, si), (to, ti)


def _flat_rows(t, groups, dims):
    """The elements (or rows) that (outer, inner, strides) reach, in order."""
    outer, inner, so, si = groups
    base = t.storage_offset()
    at = torch.tensor([base + o * so + i * si for o in range(outer) for i in range(inner)])
    store = torch.as_strided(t, (t.untyped_storage().nbytes() // t.element_size(),), (1,), 0)
    if dims == t.ndim:
        return store[at]
    return store[at[:, None] + torch.arange(t.shape[-1])]


@pytest.mark.parametrize("make", [
    lambda: (torch.randn(5), torch.zeros((), dtype=torch.long)),
    lambda: (torch.randn(6, 5), torch.arange(6)),
    lambda: (torch.randn(6, 9)[:, 2:7], torch.arange(12)[::2]),
    lambda: (torch.randn(3, 4, 5)[:, :-1], torch.arange(12).view(3, 4)[:, 1:]),
    lambda: (torch.randn(3, 4, 5), torch.arange(12).view(3, 4)),
    lambda: (torch.randn(3, 4, 5), torch.arange(12).view(4, 3).t()),
    lambda: (torch.randn(4, 3, 5).transpose(0, 1), torch.arange(12).view(3, 4)),
    lambda: (torch.randn(2, 3, 4, 5)[:, :, 1:], torch.arange(24).view(2, 3, 4)[:, :, 1:]),
    lambda: (torch.randn(2, 3, 4, 5)[:, 1:, 1:], torch.arange(24).view(2, 3, 4)[:, 1:, 1:]),
    lambda: (torch.randn(2, 3, 4, 5)[:, 1:], torch.arange(24).view(2, 3, 4)[:, :2]),
    lambda: (torch.randn(2, 6, 4, 5)[:, ::2], torch.arange(48).view(2, 3, 8)[..., ::2]),
    lambda: (torch.randn(1, 4, 5).expand(3, 4, 5), torch.arange(4).expand(3, 4)),
    lambda: (torch.randn(5, 6).t(), torch.arange(6)),
    lambda: (torch.randn(1, 1, 5), torch.arange(7)[3:4].view(1, 1)),
])
def test_rows_are_found_where_they_are(make):
    x, t = make()
    x2, t2, a, b = _rows(x, t)
    assert a[0] * a[1] == t.numel()
    assert torch.equal(_flat_rows(x2, a, x2.ndim - 1), x.reshape(-1, x.shape[-1]))
    assert torch.equal(_flat_rows(t2, (*a[:2], *b), t2.ndim), t.reshape(-1))


def test_rows_of_a_slice_are_not_copied():
    x, t = torch.randn(3, 4, 5), torch.arange(12).view(3, 4)
    x2, t2, _, _ = _rows(x[:, :-1], t[:, 1:])
    assert x2.data_ptr() == x.data_ptr() and t2.data_ptr() == t[:, 1:].data_ptr()


def test_stock_form_and_its_gradient():
    """The form a differentiable backward runs, against log_softmax in float64 and against differences."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(4, 9, generator=g, dtype=torch.float64)
    x[1, 3] = float("-inf")
    t = torch.tensor([2, 5, -100, 0])
    top = torch.topk(x, 3).indices
    lp, ent, tops = L._ops(x.float(), t, top, 0.7, -100)
    ref = torch.log_softmax(x / 0.7, -1)
    assert torch.allclose(lp.double(), torch.where(t == -100, 0.0, ref.gather(-1, t.clamp_min(0)[:, None])[:, 0]), atol=1e-5)
    assert torch.allclose(ent.double(), -(ref.exp() * ref.masked_fill(ref == float("-inf"), 0)).sum(-1), atol=1e-5)
    assert torch.allclose(tops.double(), ref.gather(-1, top), atol=1e-5)
    x32 = x.float().requires_grad_()
    weights = [torch.randn(4, generator=g), torch.randn(4, generator=g), torch.randn(4, 3, generator=g)]

    def loss(z):
        return sum((w * o).sum() for w, o in zip(weights, L._ops(z, t, top, 0.7, -100)))

    got, = torch.autograd.grad(loss(x32), x32)
    step = 1e-2
    for i, j in [(0, 2), (0, 7), (1, 5), (1, 0), (2, 4), (3, 0)]:
        d = torch.zeros_like(x32)
        d[i, j] = step
        diff = (loss(x32.detach() + d) - loss(x32.detach() - d)) / (2 * step)
        # the third derivative of these sums is below 30: 30 step^2 / 6, and 2^-22 of a loss below 30 over a step
        assert abs(float(diff - got[i, j])) <= 5 * step ** 2 + 30 * 2 ** -22 / step
    empty = torch.full((1, 9), float("-inf"), requires_grad=True)
    lp, ent, tops = L._ops(empty, torch.tensor([1]), top[:1], 1.0, -100)
    assert torch.autograd.grad(lp.sum() + ent.sum() + tops.sum(), empty)[0].abs().max() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_stock_gradient_of_rows_that_pass_nothing(dtype):
    """The kernel's zeros and NaN: rows that pass nothing whatever they hold, tokens outside with and without a gradient."""
    g = torch.Generator().manual_seed(2)
    nan, inf = float("nan"), float("inf")
    x = torch.randn(10, 9, generator=g).to(dtype)
    x[1], x[2, 4], x[3, 0], x[6], x[8], x[9] = nan, inf, nan, nan, -inf, -inf
    t = torch.tensor([1, -100, 2, 3, 9, -1, -100, 40, 9, -100])
    up = torch.tensor([1.0, 2.0, 0.0, -0.0, 0.0, 0.5, 1.0, 0.0, 1.0, 1.0])
    x.requires_grad_()
    got = L.stock_gradient(x, t, None, 0.8, -100, up, None, None).detach()
    assert got.dtype == dtype and bool(got[5].isnan().all()) and bool(got[0].isfinite().all()) and float(got[0].abs().max()) > 0
    assert all(float(got[i].abs().max()) == 0.0 for i in (1, 2, 3, 4, 6, 7, 8, 9))
    h = torch.zeros(10)
    h[6] = h[7] = 1.0  # an ignored and an outside token's row passes its entropy
    got = L.stock_gradient(x, t, None, 0.8, -100, up, h, None).detach()
    assert bool(got[6].isnan().all()) and bool(got[7].isfinite().all()) and float(got[7].abs().max()) > 0
    top = torch.topk(x.detach().float().nan_to_num(0.0), 2).indices
    gt = torch.zeros(10, 2)
    gt[0, 1] = gt[2, 0] = 1.0
    got = L.stock_gradient(x, t, top, 0.8, -100, None, None, gt).detach()
    assert bool(got[2].isnan().all()) and float(got[[1, 3, 4, 5, 6, 7, 8, 9]].abs().max()) == 0.0
    got = L.stock_gradient(x, t, top, 0.8, -100, 0 * up, 0 * h, 0 * gt).detach()
    assert float(got.abs().max()) == 0.0


def test_stock_gradient_can_be_differentiated_by_a_gradient_of_zero():
    """A product with the Jacobian by two backward passes: the first one's upstream gradient is zero everywhere."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(4, 9, generator=g).requires_grad_()
    t = torch.tensor([2, 5, -100, 0])
    up, v = torch.zeros(4, requires_grad=True), torch.randn(4, 9, generator=g)
    got, = torch.autograd.grad(L.stock_gradient(x, t, None, 0.7, -100, up, None, None), up, v)
    p = torch.softmax(x.detach().double() / 0.7, -1)
    exp = (v.double().gather(-1, t.clamp_min(0)[:, None])[:, 0] - (p * v).sum(-1)) / 0.7
    # sums of nine products below 4: 40 roundings of 2^-24
    assert float((got.double() - torch.where(t == -100, 0.0, exp)).abs().max()) <= 40 * 4 * 2 ** -24


def test_c_abi_token_logprobs_refusals():
    lib = nat.load()

    def call(logits=256, dtype=0, outer=1, inner=4, V=10, so=40, si=10, tokens=256, temperature=1.0, k=0, lp=256, ent=None,
             top=None, tok=None, stats=None, ws=None, ws_bytes=0):
        return lib.fl_token_logprobs(logits, dtype, outer, inner, V, so, si, tokens, 4, 1, -100, temperature, k, lp, ent, top,
                                     tok, stats, ws, ws_bytes, None)

    bad = nat.FL_ERR_INVALID_ARGUMENT
    assert call(dtype=7) == nat.FL_ERR_DTYPE
    for kw in (dict(logits=None), dict(logits=257), dict(outer=0), dict(inner=-1), dict(V=0), dict(V=1 << 31), dict(si=-1),
               dict(tokens=None), dict(tokens=260), dict(temperature=0.0), dict(temperature=float("nan")),
               dict(temperature=float("inf")), dict(k=-1), dict(k=65), dict(k=11, top=256, tok=256), dict(k=2), dict(lp=None),
               dict(lp=258), dict(ent=258), dict(stats=258), dict(k=2, top=256), dict(k=2, top=256, tok=260),
               dict(outer=1 << 40, inner=1 << 40)):
        assert call(**kw) == bad, kw

    def back(logits=256, dtype=0, V=10, k=0, stats=256, ent=None, tok=None, g=None, gh=None, gt=None, out=256, t=1.0):
        return lib.fl_token_logprobs_backward(logits, dtype, 1, 4, V, 40, 10, 256, 4, 1, -100, t, k, stats, ent, tok, g, gh, gt,
                                              out, None)

    assert back(dtype=9) == nat.FL_ERR_DTYPE
    for kw in (dict(logits=None), dict(V=-1), dict(stats=None), dict(out=None), dict(out=258), dict(gh=256), dict(gt=256),
               dict(k=2, gt=256), dict(g=258), dict(t=-1.0)):
        assert back(**kw) == bad, kw


# ------------------------------------------------------------------ grad_norm, adamw_step
def _array(*addresses):
    return (ctypes.c_void_p * len(addresses))(*addresses)


def test_grad_norm_refusals():
    with pytest.raises(ValueError):
        fl.grad_norm([])
    with pytest.raises(RuntimeError):
        fl.grad_norm([torch.randn(3)])
    lib = nat.load()
    n = (ctypes.c_int64 * 2)(5, 0)
    codes = (ctypes.c_int * 2)(0, 1)

    def call(count=2, grads=_array(256, None), codes=codes, n=n, most=1.0, scaled=1, out=256, ws=256, ws_bytes=1 << 20):
        return lib.fl_grad_norm(count, grads, codes, n, most, scaled, out, ws, ws_bytes, None)

    bad = nat.FL_ERR_INVALID_ARGUMENT
    assert call(codes=(ctypes.c_int * 2)(0, 5)) == nat.FL_ERR_DTYPE
    for kw in (dict(count=0), dict(grads=None), dict(codes=None), dict(n=None), dict(n=(ctypes.c_int64 * 2)(5, -1)),
               dict(n=(ctypes.c_int64 * 2)(5, 1 << 35)), dict(grads=_array(None, None)), dict(grads=_array(258, None)),
               dict(most=-1.0), dict(most=float("nan")), dict(out=None), dict(ws=260), dict(n=(ctypes.c_int64 * 2)(5, 3))):
        assert call(**kw) == bad, kw
    assert call(ws=None) == nat.FL_ERR_WORKSPACE == call(ws_bytes=4)
    assert lib.fl_grad_norm_workspace_bytes(2, n) >= 8 and lib.fl_grad_norm_workspace_bytes(0, n) == 0


def test_adamw_refusals_on_the_host():
    p, g, m, v = (torch.zeros(4) for _ in range(4))
    step = torch.zeros(1, dtype=torch.long)
    with pytest.raises(RuntimeError):
        fl.adamw_step([p], [g], [m], [v], step)
    with pytest.raises(ValueError):
        fl.adamw_step([], [], [], [], step)
    with pytest.raises(ValueError):
        fl.adamw_step([p], [g, g], [m], [v], step)
    with pytest.raises(ValueError):
        fl.adamw_step([p], [g], [m], [v], step, exp_avg_scales=[m])
    for kw in (dict(lr=-1.0), dict(lr=float("nan")), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1e-8),
               dict(eps=float("inf")), dict(weight_decay=-0.1)):
        with pytest.raises(ValueError):
            fl.adamw_step([p], [g], [m], [v], step, **kw)


def test_c_abi_adamw_refusals():
    lib = nat.load()
    n = (ctypes.c_int64 * 1)(5)
    one = _array(256)

    def call(count=1, p=one, g=one, dtype=0, m=one, v=one, ms=None, vs=None, n=n, steps=one, lr_ptr=None, b1=0.9, b2=0.99,
             eps=1e-8, gs=None, ws=256, ws_bytes=16):
        return lib.fl_adamw_step(count, p, g, dtype, m, v, ms, vs, n, steps, 1e-3, lr_ptr, b1, b2, eps, 0.1, gs, ws, ws_bytes,
                                 None)

    bad = nat.FL_ERR_INVALID_ARGUMENT
    assert call(dtype=3) == nat.FL_ERR_DTYPE
    for kw in (dict(count=0), dict(p=None), dict(p=_array(None)), dict(p=_array(258)), dict(g=_array(None)), dict(m=None),
               dict(v=_array(258)), dict(ms=one), dict(vs=one), dict(ms=one, vs=_array(None)), dict(n=None), dict(steps=None),
               dict(n=(ctypes.c_int64 * 1)(-1)), dict(n=(ctypes.c_int64 * 1)((1 << 34) + 1)), dict(steps=_array(None)),
               dict(steps=_array(260)), dict(lr_ptr=258), dict(b1=1.0), dict(b1=float("nan")), dict(b2=-0.5), dict(eps=-1.0),
               dict(gs=258), dict(ws=264)):
        assert call(**kw) == bad, kw
    assert call(ws=None) == nat.FL_ERR_WORKSPACE == call(ws_bytes=15)


def test_optimizer_refuses_groups_it_cannot_step():
    w = torch.nn.Parameter(torch.zeros(3))
    for kw in (dict(state_bits=16), dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(max_grad_norm=-1.0),
               dict(max_grad_norm=float("nan"))):
        with pytest.raises(ValueError):
            fl.AdamW([w], **kw)
    with pytest.raises(TypeError):
        fl.AdamW([torch.nn.Parameter(torch.zeros(3, dtype=torch.float16))])
    opt = fl.AdamW([w])
    with pytest.raises(ValueError):
        opt.add_param_group(dict(params=[torch.nn.Parameter(torch.zeros(2))], eps=-1.0))
    assert len(opt.param_groups) == 1 and opt.step() is None  # no gradients: nothing to do


def test_optimizer_state_keeps_its_types_through_a_checkpoint(tmp_path):
    """8-bit codes and 64-bit counters come back as they were saved, also beside bf16 parameters."""
    ws = [torch.nn.Parameter(torch.zeros(300, dtype=torch.bfloat16)), torch.nn.Parameter(torch.zeros(4, 5, dtype=torch.bfloat16))]
    opt = fl.AdamW(ws, state_bits=8)
    for w in ws:
        n = w.numel()
        opt.state[w] = dict(step=torch.tensor(7), exp_avg=torch.randn(w.shape).to(torch.float8_e4m3fn),
                            exp_avg_sq=torch.rand(w.shape).to(torch.float8_e4m3fn),
                            exp_avg_scale=torch.rand(-(-n // 256)), exp_avg_sq_scale=torch.rand(-(-n // 256)))
    torch.save(opt.state_dict(), tmp_path / "opt.pt")
    new = fl.AdamW(ws, state_bits=32)
    new.load_state_dict(torch.load(tmp_path / "opt.pt", weights_only=True))
    assert new.param_groups[0]["state_bits"] == 8
    for w in ws:
        for k, t in opt.state[w].items():
            u = new.state[w][k]
            assert u.dtype == t.dtype and u.shape == t.shape and u.data_ptr() != t.data_ptr()
            assert torch.equal(u.float(), t.float())


def _with_state(ws, bits, step=7):
    """An optimizer whose states are as after some steps, without a device."""
    opt = fl.AdamW(ws, state_bits=bits)
    code = torch.float8_e4m3fn if bits == 8 else torch.float32
    for w in ws:
        opt.state[w] = dict(step=torch.tensor(step), exp_avg=torch.randn(w.shape).to(code), exp_avg_sq=torch.rand(w.shape).to(code))
        if bits == 8:
            opt.state[w].update({k: torch.rand(-(-w.numel() // 256)) for k in ("exp_avg_scale", "exp_avg_sq_scale")})
    return opt


@pytest.mark.parametrize("bits", [8, 32])
def test_optimizer_loads_through_its_hooks(bits):
    """What pre-hooks return and what post-hooks write is what the optimizer holds; types are kept all the same."""
    ws = [torch.nn.Parameter(torch.zeros(300, dtype=torch.bfloat16)), torch.nn.Parameter(torch.zeros(4, dtype=torch.bfloat16))]
    saved = _with_state(ws, bits).state_dict()
    new, seen = fl.AdamW(ws), []

    def replace(opt, d):
        state = {i: {**s, "step": torch.tensor(40 + i)} for i, s in d["state"].items()}
        return {**d, "state": state, "param_groups": [{**g, "lr": 0.5} for g in d["param_groups"]]}

    def look(opt):
        seen.append([int(opt.state[w]["step"]) for w in ws])
        opt.state[ws[1]]["step"] = torch.tensor(99)

    new.register_load_state_dict_pre_hook(replace)
    new.register_load_state_dict_post_hook(look, prepend=True)
    for _ in range(2):  # the hooks stay those that were registered
        new.load_state_dict(saved)
    assert seen == [[40, 41]] * 2 and new.param_groups[0]["lr"] == 0.5
    assert int(new.state[ws[0]]["step"]) == 40 and int(new.state[ws[1]]["step"]) == 99
    for i, w in enumerate(ws):
        assert {k: t.dtype for k, t in new.state[w].items()} == {k: t.dtype for k, t in saved["state"][i].items()}
        assert all(torch.equal(new.state[w][k].float(), t.float()) for k, t in saved["state"][i].items() if k != "step")
    assert int(saved["state"][0]["step"]) == 7


def test_optimizer_refuses_checkpoints_it_cannot_go_on_from():
    """Another optimizer's, and states of other types, sizes and kinds: refused at once, with nothing changed."""
    ws = [torch.nn.Parameter(torch.zeros(300)), torch.nn.Parameter(torch.zeros(4))]
    stock = torch.optim.AdamW(ws)
    for w in ws:
        w.grad = torch.ones_like(w)
    stock.step()
    good = {bits: _with_state(ws, bits).state_dict() for bits in (8, 32)}
    own = _with_state(ws, 32, step=3)
    before = own.state_dict()

    def changed(bits, name, value):
        d = good[bits]
        return {**d, "state": {**d["state"], 1: {k: v for k, v in {**d["state"][1], name: value}.items() if v is not None}}}

    def regrouped(**kw):
        return {**good[32], "param_groups": [{**g, **kw} for g in good[32]["param_groups"]]}

    bad = [stock.state_dict(), regrouped(state_bits=8), regrouped(state_bits=16), regrouped(lr=-1.0), regrouped(eps=float("nan")),
           changed(32, "step", torch.tensor(7.0)), changed(32, "step", 7), changed(32, "exp_avg", None),
           changed(32, "exp_avg_sq", torch.zeros(5)), changed(32, "exp_avg", torch.zeros(4, dtype=torch.bfloat16)),
           changed(8, "exp_avg_scale", None), changed(8, "exp_avg_sq_scale", torch.zeros(2)),
           changed(8, "exp_avg", torch.zeros(4)), {**good[32], "param_groups": []}]
    for d in bad:
        with pytest.raises(ValueError):
            own.load_state_dict(d)
        after = own.state_dict()
        assert after["param_groups"] == before["param_groups"]
        assert all(after["state"][i][k] is t for i, s in before["state"].items() for k, t in s.items())
    for bits in (8, 32):
        own.load_state_dict(good[bits])
        assert own.param_groups[0]["state_bits"] == bits and int(own.state[ws[1]]["step"]) == 7
    own.load_state_dict({**good[32], "state": {0: good[32]["state"][0], 1: {}}})  # one that has not stepped yet
    assert int(own.state[ws[0]]["step"]) == 7 and not own.state[ws[1]]


def test_optimizer_copies_keep_the_clip():
    ws = [torch.nn.Parameter(torch.zeros(3))]
    for most in (None, 0.5):
        opt = fl.AdamW(ws, max_grad_norm=most)
        for new in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
            assert new.max_grad_norm == most and new.grad_norm is None and new.step() is None
            assert new.param_groups[0]["state_bits"] == 32


def test_optimizer_loads_a_learning_rate_onto_the_parameters_device():
    """A checkpoint read on the host, as most are: its tensors come to the parameters' device."""
    ws = [torch.nn.Parameter(torch.zeros(3))]
    saved = _with_state(ws, 32).state_dict()
    for g in saved["param_groups"]:
        g["lr"] = torch.tensor(0.25)
    new = fl.AdamW([torch.nn.Parameter(torch.zeros(3, device="meta"))])
    new.load_state_dict(saved)
    p, = new.param_groups[0]["params"]
    assert {t.device.type for t in (new.param_groups[0]["lr"], *new.state[p].values())} == {"meta"}
    here = fl.AdamW(ws)
    here.load_state_dict(saved)
    assert float(here.param_groups[0]["lr"]) == 0.25 and here.param_groups[0]["lr"] is not saved["param_groups"][0]["lr"]
