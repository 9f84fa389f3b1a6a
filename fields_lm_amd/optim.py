"""What follows a training step's backward, on the HIP path only (``csrc/optimizer.hip``, host side
``csrc/host.cpp`` and ``csrc/host_train.cpp``):

* :func:`grad_norm`   the 2-norm over many gradients and the scale that clips it, in one pass over them;
* :func:`adamw_step`  one AdamW step over many tensors, moments in fp32 or in 8 bits;
* :class:`AdamW`      the optimizer around both;
* :func:`orthogonalize`, :func:`muon_step`, :class:`Muon`  the same for matrices (``csrc/muon.hip``): Newton-Schulz
  steps, the Muon step over many matrices, the optimizer.

Nothing here waits for the device: norms and scales stay there, step counters too, so a step can be captured
in a HIP graph and replayed.
"""
from __future__ import annotations

import math
from operator import itemgetter
from typing import Iterable, List, Optional, Sequence, Tuple, Union

import torch

from . import _native as nat

STATE_BLOCK = 256                   # values that share a scale in the 8-bit states
STATE8_DTYPE = torch.float8_e4m3fn  # their codes

_TYPES = (torch.float32, torch.bfloat16)
NEWTON_SCHULZ = (3.4445, -4.7750, 2.0315)  # a, b, c: steep at 0, singular values within 0.7 to 1.2 after five steps
ADJUST_LR = ("original", "match_rms_adamw")

_STATES = {32: itemgetter("step", "exp_avg", "exp_avg_sq"),
           8: itemgetter("step", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")}


def _listed(tensors):
    return tensors if isinstance(tensors, (list, tuple)) else list(tensors)


def grad_norm(grads: Iterable[torch.Tensor], max_norm: Optional[float] = None
              ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """2-norm over all values of ``grads`` (fp32 / bf16, any mix, on one ROCm device): fp32 0-d, summed in
    64 bits in a fixed order.

    With ``max_norm`` also the scale that clips it, min(1, max_norm / (norm + 1e-6)), which
    :func:`adamw_step` takes as ``grad_scale``; the gradients are not rewritten. The scale of a norm that is
    not finite is NaN, on which :func:`adamw_step` leaves everything as it was. Neither is differentiable.
    """
    if max_norm is not None and not float(max_norm) >= 0.0:
        raise ValueError(f"max_norm must be 0 or more, got {max_norm}")
    norm, scale = nat.host().grad_norm(_listed(grads), -1.0 if max_norm is None else float(max_norm))
    return norm if max_norm is None else (norm, scale)


def _check_hyper(lr, betas, eps, weight_decay) -> None:
    if not isinstance(lr, torch.Tensor) and not (float(lr) >= 0.0 and math.isfinite(lr)):
        raise ValueError(f"lr must be finite and 0 or more, got {lr}")
    if not all(0.0 <= float(b) < 1.0 for b in betas):
        raise ValueError(f"betas must lie in [0, 1), got {tuple(betas)}")
    if not (float(eps) >= 0.0 and math.isfinite(eps)):
        raise ValueError(f"eps must be finite and 0 or more, got {eps}")
    if not (float(weight_decay) >= 0.0 and math.isfinite(weight_decay)):
        raise ValueError(f"weight_decay must be finite and 0 or more, got {weight_decay}")


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], exp_avgs: Sequence[torch.Tensor],
               exp_avg_sqs: Sequence[torch.Tensor], steps: Union[torch.Tensor, Sequence[torch.Tensor]], *,
               lr: Union[float, torch.Tensor] = 1e-3, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 1e-2, grad_scale: Optional[torch.Tensor] = None,
               exp_avg_scales: Optional[Sequence[torch.Tensor]] = None,
               exp_avg_sq_scales: Optional[Sequence[torch.Tensor]] = None) -> None:
    """One AdamW step over all tensors, in place (``fl_adamw_step``). With g = grad * grad_scale and t the
    tensor's step counter, advanced first:

        m = beta1 m + (1 - beta1) g;  v = beta2 v + (1 - beta2) g^2
        p = p (1 - lr weight_decay) - lr / (1 - beta1^t) * m / (sqrt(v / (1 - beta2^t)) + eps)

    params: contiguous, all fp32 or all bf16, on one ROCm device; grads of their shapes and type. Maths in
    fp32, a bf16 parameter rounded once. steps: an int64 value per tensor, one tensor [N] or N of one value.
    lr: a number, or one fp32 value on the device, read when the step runs.

    Without scales exp_avgs / exp_avg_sqs are contiguous fp32 tensors of the parameters' sizes. With scales they
    hold 8 bits a value: float8_e4m3fn codes of m and of sqrt(v) in blocks of 256 consecutive values, whose
    largest magnitude / 448 is the block's fp32 scale ([ceil(numel / 256)]); zeros are a valid start. A root
    that is not 0 keeps at least the smallest code. A non-finite value in a gradient spoils its block's states.

    grad_scale: one fp32 value on the device (:func:`grad_norm`'s second), or None for 1. Where it is not finite the
    call leaves parameters, states and step counters as they were. To autograd the call is a write of all of them.
    """
    _check_hyper(lr, betas, eps, weight_decay)
    nat.host().adamw_step(
        _listed(params), _listed(grads), _listed(exp_avgs), _listed(exp_avg_sqs),
        steps if isinstance(steps, torch.Tensor) else _listed(steps), lr, betas[0], betas[1], eps, weight_decay,
        grad_scale, None if exp_avg_scales is None else _listed(exp_avg_scales),
        None if exp_avg_sq_scales is None else _listed(exp_avg_sq_scales))


def orthogonalize(x: torch.Tensor, *, steps: int = 5, coefficients: Tuple[float, float, float] = NEWTON_SCHULZ,
                  eps: float = 1e-7) -> torch.Tensor:
    """Matrices [..., M, N] (up to 2^20 of them, sides up to 2^20, 2^30 values each; fp32 or bf16, on a ROCm device)
    brought near their closest semi-orthogonal ones by Newton-Schulz steps (``fl_orthogonalize``): from
    X = x / (|x| + eps), |x| the Frobenius norm, ``steps`` (1 to 64) times X = a X + (b A + c A^2) X with A = X X^T
    (X^T X for a tall matrix), (a, b, c) the ``coefficients``.

    Everything is computed in fp32 and in products of 22 bits, whose errors are about those of the same steps in fp32 (0.4
    to 1.3 times), and rounded once, to x's type; a matrix of zeros stays zeros, one with NaN or infinities becomes NaN. Coefficients with which singular values, or a step's factor, could
    pass 1024 are refused. Not differentiable. A call takes up to 2 GiB of workspace, or what its largest matrix needs.
    """
    a, b, c = coefficients
    return nat.host().orthogonalize(x, steps, a, b, c, eps)


def _check_muon(lr, momentum, weight_decay, adjust_lr) -> None:
    if not isinstance(lr, torch.Tensor) and not (float(lr) >= 0.0 and math.isfinite(lr)):
        raise ValueError(f"lr must be finite and 0 or more, got {lr}")
    if not 0.0 <= float(momentum) < 1.0:
        raise ValueError(f"momentum must lie in [0, 1), got {momentum}")
    if not (float(weight_decay) >= 0.0 and math.isfinite(weight_decay)):
        raise ValueError(f"weight_decay must be finite and 0 or more, got {weight_decay}")
    if adjust_lr not in ADJUST_LR:
        raise ValueError(f"adjust_lr must be one of {ADJUST_LR}, got {adjust_lr!r}")


def muon_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], momentum_buffers: Sequence[torch.Tensor], *,
              lr: Union[float, torch.Tensor] = 1e-3, momentum: float = 0.95, nesterov: bool = True,
              weight_decay: float = 0.1, steps: int = 5, coefficients: Tuple[float, float, float] = NEWTON_SCHULZ,
              eps: float = 1e-7, adjust_lr: str = "original", grad_scale: Optional[torch.Tensor] = None) -> None:
    """One Muon step over all matrices, in place (``fl_muon_step``). With g = grad * grad_scale:

        m = momentum m + (1 - momentum) g;  u = (1 - momentum) g + momentum m with ``nesterov``, else m
        p = p (1 - lr weight_decay) - lr r orthogonalize(u)

    r is sqrt(max(1, rows / columns)) for ``adjust_lr`` "original" and 0.2 sqrt(max(rows, columns)) for
    "match_rms_adamw", with which the update is as large as AdamW's and takes its learning rate.

    params: contiguous matrices, all fp32 or all bf16, on one ROCm device; grads of their shapes and type; buffers
    contiguous fp32 of their sizes, zeros at first. Maths as :func:`orthogonalize`'s, a parameter rounded once. lr and
    grad_scale as in :func:`adamw_step`: where grad_scale is not finite parameters and buffers stay as they were. To
    autograd the call is a write of both.
    """
    _check_muon(lr, momentum, weight_decay, adjust_lr)
    a, b, c = coefficients
    nat.host().muon_step(_listed(params), _listed(grads), _listed(momentum_buffers), lr, momentum, nesterov, weight_decay,
                         steps, a, b, c, eps, adjust_lr == "match_rms_adamw", grad_scale)


class _Optimizer(torch.optim.Optimizer):
    """What the optimizers share: a step over parameters by group, type and device, with its clip, and checkpoints whose
    states keep their types. A subclass has ``_group`` (what a step reads of its group), ``_check_group``,
    ``_check_parameter``, ``_wanted`` (a state's types and counts), ``_like_parameter`` (which of them have a value to each of
    the parameter's), ``_new`` (fresh states) and ``_step``."""

    _group: Tuple[str, ...] = ()
    _like_parameter: Tuple[str, ...] = ()

    def __init__(self, params, defaults: dict, max_grad_norm: Optional[float]) -> None:
        if max_grad_norm is not None and not float(max_grad_norm) >= 0.0:
            raise ValueError(f"max_grad_norm must be 0 or more, got {max_grad_norm}")
        self.max_grad_norm = max_grad_norm
        self.grad_norm: Optional[torch.Tensor] = None
        super().__init__(params, defaults)

    def __getstate__(self) -> dict:
        """What copies and pickles hold: the base class's, and the clip."""
        return {**super().__getstate__(), "max_grad_norm": self.max_grad_norm, "grad_norm": self.grad_norm}

    def _check_parameter(self, p: torch.Tensor) -> None:
        if p.dtype not in _TYPES:
            raise TypeError(f"parameters must be float32 or bfloat16, got {p.dtype}")

    def add_param_group(self, param_group) -> None:
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            self._check_group(group)
            for p in group["params"]:
                self._check_parameter(p)
        except (TypeError, ValueError):
            self.param_groups.pop()
            raise

    def _state(self, p: torch.Tensor, group: dict) -> dict:
        st = self.state[p]
        if not st:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("a parameter's first step makes its states and must not be under graph capture")
            st.update(self._new(p, group))
        return st

    def _check_state(self, state: dict, p: torch.Tensor, group: dict) -> None:
        """A saved state of ``p`` is one that a step can go on from."""
        for name, (dtype, count) in self._wanted(p, group).items():
            t = state.get(name)
            if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.numel() != count:
                got = f"{t.numel()} of {t.dtype}" if isinstance(t, torch.Tensor) else repr(t)
                raise ValueError(f"{name} of a parameter of {p.numel()} values must be {count} of {dtype}, got {got}")
            if name in self._like_parameter and not self._lies_as(t, p):
                raise ValueError(f"{name} of a parameter of the shape {tuple(p.shape)} has the shape {tuple(t.shape)}")

    def _lies_as(self, t: torch.Tensor, p: torch.Tensor) -> bool:
        """Whether a saved state's values belong to the parameter's in their order."""
        return t.shape == p.shape

    def load_state_dict(self, state_dict) -> None:
        """As the base class, hooks included, but every state keeps the type it was saved in, and a learning rate held in
        a tensor comes to the parameters' device, as states do, which become contiguous. What no step can go on from
        (another optimizer's checkpoint, states of other types, sizes or shapes) is refused before anything is changed."""
        loaded: dict = {}

        def last(_, final) -> None:  # behind the other pre-hooks: what the base class is about to load
            for group, own in zip(final["param_groups"], self.param_groups):
                if missing := [k for k in self._group if k not in group]:
                    raise ValueError(f"no checkpoint of this optimizer: a group lacks {', '.join(missing)}")
                self._check_group(group)
                for i, p in zip(group["params"], own["params"]):
                    if final["state"].get(i):
                        self._check_state(final["state"][i], p, group)
            loaded.update(final)

        def first(_) -> None:  # ahead of the other post-hooks: the base class has cast states to their parameters' type
            for group in self.param_groups:
                if isinstance(group["lr"], torch.Tensor) and group["params"]:
                    group["lr"] = group["lr"].to(group["params"][0].device)
            ids = [i for g in loaded["param_groups"] for i in g["params"]]
            for i, p in zip(ids, (p for g in self.param_groups for p in g["params"])):
                if i in loaded["state"]:
                    self.state[p] = {k: v.detach().to(p.device, copy=True, memory_format=torch.contiguous_format)
                                     if isinstance(v, torch.Tensor) else v for k, v in loaded["state"][i].items()}

        hooks = (self.register_load_state_dict_pre_hook(last),
                 self.register_load_state_dict_post_hook(first, prepend=True))
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        work: List[Tuple[dict, List[torch.Tensor], List[torch.Tensor]]] = []  # a group's parameters and gradients
        for group in self.param_groups:
            kinds: dict = {}
            for p in group["params"]:
                grad = p.grad
                if grad is not None:
                    key = (p.dtype, p.device)
                    kind = kinds.get(key)
                    if kind is None:
                        kind = kinds[key] = (group, [], [])
                    kind[1].append(p)
                    kind[2].append(grad)
            work += kinds.values()
        if not work:
            return loss
        scale = None
        if self.max_grad_norm is not None:
            self.grad_norm, scale = grad_norm([g for _, _, grads in work for g in grads], self.max_grad_norm)
        for group, ps, grads in work:
            self._step(group, ps, grads, scale)
        return loss


class AdamW(_Optimizer):
    """AdamW over :func:`adamw_step`: one call per parameter group, type and device.

    ``state_bits`` 32 keeps both moments in fp32 (8 bytes a value), 8 in 8-bit blocks (2 bytes and 1 / 32).
    ``max_grad_norm`` clips the norm over all groups' gradients inside the step, without rewriting them; the norm
    stays in ``self.grad_norm`` (fp32, on the device; all gradients on one), and a step whose norm is not finite changes
    nothing.
    A parameter without a gradient is left alone and its step not counted. States are made at a parameter's
    first step, which must not be under graph capture.
    """

    _group = ("lr", "betas", "eps", "weight_decay", "state_bits")
    _like_parameter = ("exp_avg", "exp_avg_sq")

    def __init__(self, params, lr: Union[float, torch.Tensor] = 1e-3, betas: Tuple[float, float] = (0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 1e-2, *, state_bits: int = 32,
                 max_grad_norm: Optional[float] = None) -> None:
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits),
                         max_grad_norm)

    def _check_group(self, group: dict) -> None:
        _check_hyper(group["lr"], group["betas"], group["eps"], group["weight_decay"])
        if group["state_bits"] not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {group['state_bits']}")

    def _wanted(self, p: torch.Tensor, group: dict) -> dict:
        n, blocks, bits = p.numel(), -(-p.numel() // STATE_BLOCK), group["state_bits"]
        code = torch.float32 if bits == 32 else STATE8_DTYPE
        wanted = dict(step=(torch.int64, 1), exp_avg=(code, n), exp_avg_sq=(code, n))
        if bits == 8:
            wanted.update(exp_avg_scale=(torch.float32, blocks), exp_avg_sq_scale=(torch.float32, blocks))
        return wanted

    def _lies_as(self, t: torch.Tensor, p: torch.Tensor) -> bool:
        return super()._lies_as(t, p) or t.ndim == 1  # (a step goes value by value)

    def _new(self, p: torch.Tensor, group: dict) -> dict:
        new = dict(device=p.device)
        st = dict(step=torch.zeros((), dtype=torch.int64, **new))
        if group["state_bits"] == 32:
            st["exp_avg"], st["exp_avg_sq"] = (torch.zeros(p.shape, dtype=torch.float32, **new) for _ in range(2))
        else:
            blocks = -(-p.numel() // STATE_BLOCK)
            for name in ("exp_avg", "exp_avg_sq"):
                st[name] = torch.zeros(p.shape, dtype=torch.uint8, **new).view(STATE8_DTYPE)
                st[name + "_scale"] = torch.zeros(blocks, dtype=torch.float32, **new)
        return st

    def _step(self, group: dict, ps: List[torch.Tensor], grads: List[torch.Tensor], scale) -> None:
        state = self.state
        states = [state[p] or self._state(p, group) for p in ps]
        steps, avgs, sqs, *scales = zip(*map(_STATES[group["state_bits"]], states))
        adamw_step(ps, grads, avgs, sqs, steps, lr=group["lr"], betas=group["betas"], eps=group["eps"],
                   weight_decay=group["weight_decay"], grad_scale=scale,
                   **dict(zip(("exp_avg_scales", "exp_avg_sq_scales"), scales)))


class Muon(_Optimizer):
    """Muon over :func:`muon_step`, for a model's matrices (embeddings, norms and biases are AdamW's): one call per
    parameter group, type and device.

    The momentum is kept in fp32 (4 bytes a value). ``max_grad_norm`` clips as :class:`AdamW`'s does, over this
    optimizer's gradients. A parameter without a gradient is left alone. States are made at a parameter's first step,
    which must not be under graph capture.
    """

    _group = ("lr", "momentum", "nesterov", "weight_decay", "steps", "coefficients", "eps", "adjust_lr")
    _like_parameter = ("momentum_buffer",)

    def __init__(self, params, lr: Union[float, torch.Tensor] = 1e-3, momentum: float = 0.95, nesterov: bool = True,
                 weight_decay: float = 0.1, *, steps: int = 5,
                 coefficients: Tuple[float, float, float] = NEWTON_SCHULZ, eps: float = 1e-7,
                 adjust_lr: str = "original", max_grad_norm: Optional[float] = None) -> None:
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps,
                                      coefficients=coefficients, eps=eps, adjust_lr=adjust_lr), max_grad_norm)

    def _check_group(self, group: dict) -> None:
        _check_muon(group["lr"], group["momentum"], group["weight_decay"], group["adjust_lr"])
        nat.host().check_steps(group["steps"], *group["coefficients"], group["eps"])

    def _check_parameter(self, p: torch.Tensor) -> None:
        super()._check_parameter(p)
        if p.ndim != 2:
            raise ValueError(f"parameters must be matrices, got the shape {tuple(p.shape)}")

    def _wanted(self, p: torch.Tensor, group: dict) -> dict:
        return dict(momentum_buffer=(torch.float32, p.numel()))

    def _new(self, p: torch.Tensor, group: dict) -> dict:
        return dict(momentum_buffer=torch.zeros(p.shape, dtype=torch.float32, device=p.device))

    def _step(self, group: dict, ps: List[torch.Tensor], grads: List[torch.Tensor], scale) -> None:
        buffers = [(self.state[p] or self._state(p, group))["momentum_buffer"] for p in ps]
        muon_step(ps, grads, buffers, lr=group["lr"], momentum=group["momentum"], nesterov=group["nesterov"],
                  weight_decay=group["weight_decay"], steps=group["steps"], coefficients=group["coefficients"],
                  eps=group["eps"], adjust_lr=group["adjust_lr"], grad_scale=scale)
