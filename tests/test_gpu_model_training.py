"""GPU: a small model trained through the package's own operators: embedding, softpatch's scan, log probabilities, Muon for
its matrices and AdamW for the rest.

Gradients are compared with the same model's whose embedding and recurrence are stock operations. Both round the same
operations elsewhere; a row of the embedding's gradient sums at most 60 terms, a step of the recurrence carries the
roundings of at most 60 steps, and what follows passes both on: 1,000 u of a gradient's norm, u = 2^-24, is ample for
either and far below what a missing or doubled term leaves.
"""
from __future__ import annotations

import copy

import pytest
import torch
import torch.nn.functional as F

import fields_lm_amd as fl
from fields_lm_amd import model as M
from fields_lm_amd._train import gated_scan_ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm device")
    return torch.device("cuda:0")


def small_model(dev, padding=None):
    torch.manual_seed(7)
    core = M.FieldTokenSystem(vocab=331, dim=128, ff_hidden=192, refresh_windows=(32,), mamba_positions=(1,), layers=6,
                              q_heads=2, kv_heads=1, latent_dim=32, landmark_chunk=16, softpatch_rank=24,
                              mamba=dict(d_state=16, d_conv=4, expand=2, headdim=32, ngroups=1, chunk_size=32),
                              late_ff_delta=0)
    M.tied_embedding_init(core, 11)
    torch.nn.init.normal_(core.softpatch.up.weight, std=0.05)
    torch.nn.init.normal_(core.softpatch.score.weight, std=0.05)
    core.emb.padding_idx = padding
    return core.to(dev)


def loss_of(core, tokens):
    logits = core.states_logits(tokens)[1]
    return -fl.token_logprobs(logits[:, :-1], tokens[:, 1:]).logprobs.mean()


def trained(core):
    """Parameters that the loss reaches (the cache's are kept for checkpoints alone)."""
    return {n: p for n, p in core.named_parameters() if not n.startswith("cache.")}


@pytest.mark.parametrize("autocast", [False, True])
@pytest.mark.parametrize("padding", [None, 5])
def test_gradients(dev, monkeypatch, padding, autocast):
    print(f"[case] model gradients padding={padding} autocast={autocast}", flush=True)
    core = small_model(dev, padding)
    gen = torch.Generator(device=dev).manual_seed(3)
    tokens = torch.randint(0, 331, (3, 61), device=dev, generator=gen)
    tokens[1, 40:] = 5
    named = trained(core)

    def gradients():
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
            loss = loss_of(core, tokens)
        return torch.autograd.grad(loss, list(named.values()))

    calls = []
    monkeypatch.setattr(M, "embedding", lambda *a, **k: (calls.append("embedding"), fl.embedding(*a, **k))[1])
    monkeypatch.setattr(M, "gated_scan", lambda *a, **k: (calls.append("scan"), fl.gated_scan(*a, **k))[1])
    got = gradients()
    assert sorted(calls) == ["embedding", "scan"]
    monkeypatch.setattr(M, "embedding", lambda t, w, *, padding_idx: F.embedding(t, w, padding_idx))
    monkeypatch.setattr(M, "gated_scan", lambda a, u, *, return_state: gated_scan_ops(a, u, None))
    for (name, p), a, b in zip(named.items(), got, gradients()):
        # (under autocast a changed last bit can move a bf16 value by a step of 2^-8, of which a norm holds many)
        bound = (2.0 ** -8 if autocast else 1000 * U) * float(b.norm())
        assert float((a - b).norm()) <= bound, name
    down = dict(zip(named, got))["softpatch.down.weight"]
    assert float(down.norm()) > 0


def test_the_recurrence_passes_its_gradient(dev):
    """The state is part of the softpatch's gradient: closing its columns of `up` changes that of `down`."""
    print("[case] softpatch gradient", flush=True)
    mixer = small_model(dev).softpatch
    gen = torch.Generator(device=dev).manual_seed(4)
    x = torch.randn(2, 40, 128, device=dev, generator=gen)
    tokens = torch.zeros(2, 40, dtype=torch.long, device=dev)
    w = torch.randn(2, 40, 128, device=dev, generator=gen)
    full, = torch.autograd.grad((mixer(x, tokens) * w).sum(), mixer.down.weight)
    with torch.no_grad():
        assert torch.allclose(mixer(x, tokens), mixer(x.requires_grad_(), tokens).detach(), atol=1e-4)
        mixer.up.weight[:, 24:] = 0
    less, = torch.autograd.grad((mixer(x.detach(), tokens) * w).sum(), mixer.down.weight)
    assert float((full - less).norm()) > 0.05 * float(less.norm())


def _contexts():
    import contextlib

    from torch.utils._python_dispatch import TorchDispatchMode
    from torch.utils.flop_counter import FlopCounterMode

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    return {"nothing": contextlib.nullcontext, "a dispatch mode": Watch, "a flop counter": lambda: FlopCounterMode(display=False)}


@pytest.mark.parametrize("watched", ["nothing", "a dispatch mode", "a flop counter", "selective checkpoints",
                                     "torch.func", "compilation"])
def test_the_recurrence_passes_its_gradient_to_whatever_watches(dev, watched):
    """Where the kernels do not run the gradient is that of stock operations: both round the recurrence's 300 steps, each at
    most by 2 u of what a sum of magnitudes is, and the rest alike: 1,000 u of the norm."""
    print(f"[case] softpatch gradient under {watched}", flush=True)
    mixer = small_model(dev).softpatch
    gen = torch.Generator(device=dev).manual_seed(6)
    x = torch.randn(2, 300, 128, device=dev, generator=gen)
    tokens = torch.zeros(2, 300, dtype=torch.long, device=dev)
    w = torch.randn(2, 300, 128, device=dev, generator=gen)
    named = dict(mixer.named_parameters())

    def gradients(run):
        out = run(x)
        return torch.autograd.grad((out * w).sum(), list(named.values()))

    want = gradients(lambda y: mixer(y, tokens))
    if watched == "selective checkpoints":
        import functools

        from torch.utils.checkpoint import CheckpointPolicy, checkpoint, create_selective_checkpoint_contexts

        contexts = functools.partial(create_selective_checkpoint_contexts,
                                     lambda ctx, op, *a, **k: CheckpointPolicy.PREFER_RECOMPUTE)
        got = gradients(lambda y: checkpoint(mixer, y, tokens, use_reentrant=False, context_fn=contexts))
    elif watched == "compilation":
        got = gradients(lambda y: torch.compile(mixer, backend="aot_eager")(y, tokens))
    elif watched == "torch.func":
        def loss(params):
            return (torch.func.functional_call(mixer, params, (x, tokens)) * w).sum()

        got = list(torch.func.grad(loss)({n: p.detach() for n, p in named.items()}).values())
        with pytest.raises(RuntimeError):  # a batched tensor says of no gradient: refused, not lost
            torch.vmap(lambda a, t: mixer(a[None], t[None])[0])(x, tokens)
    else:
        with _contexts()[watched]():
            got = gradients(lambda y: mixer(y, tokens))
    for (name, _), a, b in zip(named.items(), got, want):
        assert float((a - b).norm()) <= 1000 * U * float(b.norm()), name
    assert float(dict(zip(named, got))["down.weight"].norm()) > 0


def test_training_steps(dev):
    """Every parameter gets a gradient and a step, Muon's is muon_step's, and checkpoints carry on."""
    print("[case] training steps", flush=True)
    core = small_model(dev)
    gen = torch.Generator(device=dev).manual_seed(5)
    named = trained(core)
    matrices = [p for n, p in named.items() if p.ndim == 2 and not n.startswith("emb")]
    others = [p for p in named.values() if not any(p is m for m in matrices)]
    assert len(matrices) > 15 and any(p is core.emb.weight for p in others)
    muon = fl.Muon(matrices, lr=0.01, adjust_lr="match_rms_adamw", max_grad_norm=1.0)
    adam = fl.AdamW(others, lr=1e-3, max_grad_norm=1.0)
    buffers = [torch.zeros_like(p) for p in matrices]
    for step in range(3):
        tokens = torch.randint(0, 331, (2, 50), device=dev, generator=gen)
        for p in named.values():
            p.grad = None
        loss_of(core, tokens).backward()
        assert all(p.grad is not None and bool(p.grad.isfinite().all()) for p in named.values())
        mirror = [p.detach().clone() for p in matrices]
        _, scale = fl.grad_norm([p.grad for p in matrices], 1.0)
        fl.muon_step(mirror, [p.grad for p in matrices], buffers, lr=0.01, adjust_lr="match_rms_adamw", grad_scale=scale)
        before = [p.detach().clone() for p in others]
        muon.step()
        adam.step()
        assert all(torch.equal(a, b) for a, b in zip(matrices, mirror))
        assert all(not torch.equal(a, b) for a, b in zip(others, before))
    state = copy.deepcopy(muon.state_dict()), copy.deepcopy(adam.state_dict())
    muon.load_state_dict(state[0])
    adam.load_state_dict(state[1])
    muon.step()
    adam.step()
    assert all(bool(p.isfinite().all()) for p in named.values())


@pytest.mark.parametrize("rows", [2 ** 23, 2 ** 23 + 1])
def test_the_largest_vocabulary(dev, rows):
    """Past the kernel's rows the model's embedding is the stock one."""
    print(f"[case] model's embedding of {rows} rows", flush=True)
    core = small_model(dev)
    core.emb = torch.nn.Embedding(rows, 5, device=dev)
    tokens = torch.tensor([[0, rows - 1, 7, rows - 1]], device=dev)
    up = torch.randn(1, 4, 5, device=dev)
    x = core._embed(tokens)
    assert torch.equal(x, core.emb.weight[tokens])
    got, = torch.autograd.grad(x, core.emb.weight, up)
    assert torch.equal(got[[0, 7]], up[0, [0, 2]]) and torch.equal(got[rows - 1], up[0, 1] + up[0, 3])
    assert int(got.ne(0).any(1).sum()) == 3


@pytest.mark.parametrize("rows,tokens,dtype,kernels", [(1 << 15, 383, torch.float32, False), (1 << 15, 384, torch.float32, True),
                                                       ((1 << 15) - 1, 383, torch.float32, True),
                                                       (1 << 15, 383, torch.bfloat16, True)], ids=str)
def test_a_few_tokens_of_a_large_weight(dev, monkeypatch, rows, tokens, dtype, kernels):
    """Whose gradient the kernels make, and that either is the sum of the tokens' (whole numbers, exact in any order)."""
    print(f"[case] model's embedding of {rows} rows, {tokens} tokens, {dtype}", flush=True)
    core = small_model(dev)
    core.emb = torch.nn.Embedding(rows, 1024, device=dev, dtype=dtype)
    gen = torch.Generator(device=dev).manual_seed(8)
    ids = torch.randint(0, 9, (1, tokens), device=dev, generator=gen) * (rows // 9)
    up = torch.randint(-1, 2, (1, tokens, 1024), device=dev, generator=gen).to(dtype)
    calls = []
    monkeypatch.setattr(M, "embedding", lambda *a, **k: (calls.append(1), fl.embedding(*a, **k))[1])
    x = core._embed(ids)
    assert bool(calls) == kernels and torch.equal(x, core.emb.weight[ids])
    got, = torch.autograd.grad(x, core.emb.weight, up)
    exp = torch.zeros(rows, 1024, device=dev).index_add_(0, ids[0], up[0].float())
    assert torch.equal(got.float(), exp)
