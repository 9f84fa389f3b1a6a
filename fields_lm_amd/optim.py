"""What follows a training step's backward, on the HIP path only (``csrc/optimizer.hip``, host side
``csrc/host.cpp``):

* :func:`grad_norm`   the 2-norm over many gradients and the scale that clips it, in one pass over them;
* :func:`adamw_step`  one AdamW step over many tensors, moments in fp32 or in 8 bits;
* :class:`AdamW`      the optimizer around both.

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
_GROUP = ("lr", "betas", "eps", "weight_decay", "state_bits")  # what a step reads of its group
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


def _check_group(group: dict) -> None:
    _check_hyper(group["lr"], group["betas"], group["eps"], group["weight_decay"])
    if group["state_bits"] not in (8, 32):
        raise ValueError(f"state_bits must be 8 or 32, got {group['state_bits']}")


def _check_state(state: dict, p: torch.Tensor, bits: int) -> None:
    """A saved state of ``p`` is one that a step can go on from."""
    n, blocks, code = p.numel(), -(-p.numel() // STATE_BLOCK), torch.float32 if bits == 32 else STATE8_DTYPE
    wanted = dict(step=(torch.int64, 1), exp_avg=(code, n), exp_avg_sq=(code, n))
    if bits == 8:
        wanted.update(exp_avg_scale=(torch.float32, blocks), exp_avg_sq_scale=(torch.float32, blocks))
    for name, (dtype, count) in wanted.items():
        t = state.get(name)
        if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.numel() != count:
            got = f"{t.numel()} of {t.dtype}" if isinstance(t, torch.Tensor) else repr(t)
            raise ValueError(f"{name} of a parameter of {n} values must be {count} of {dtype} ({bits}-bit states), got {got}")


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


class AdamW(torch.optim.Optimizer):
    """AdamW over :func:`adamw_step`: one call per parameter group, type and device.

    ``state_bits`` 32 keeps both moments in fp32 (8 bytes a value), 8 in 8-bit blocks (2 bytes and 1 / 32).
    ``max_grad_norm`` clips the norm over all groups' gradients inside the step, without rewriting them; the norm
    stays in ``self.grad_norm`` (fp32, on the device; all gradients on one), and a step whose norm is not finite changes
    nothing.
    A parameter without a gradient is left alone and its step not counted. States are made at a parameter's
    first step, which must not be under graph capture.
    """

    def __init__(self, params, lr: Union[float, torch.Tensor] = 1e-3, betas: Tuple[float, float] = (0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 1e-2, *, state_bits: int = 32,
                 max_grad_norm: Optional[float] = None) -> None:
        if max_grad_norm is not None and not float(max_grad_norm) >= 0.0:
            raise ValueError(f"max_grad_norm must be 0 or more, got {max_grad_norm}")
        self.max_grad_norm = max_grad_norm
        self.grad_norm: Optional[torch.Tensor] = None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits))

    def __getstate__(self) -> dict:
        """What copies and pickles hold: the base class's, and the clip."""
        return {**super().__getstate__(), "max_grad_norm": self.max_grad_norm, "grad_norm": self.grad_norm}

    def add_param_group(self, param_group) -> None:
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            _check_group(group)
            for p in group["params"]:
                if p.dtype not in _TYPES:
                    raise TypeError(f"parameters must be float32 or bfloat16, got {p.dtype}")
        except (TypeError, ValueError):
            self.param_groups.pop()
            raise

    def _state(self, p: torch.Tensor, bits: int) -> dict:
        st = self.state[p]
        if not st:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("a parameter's first step makes its states and must not be under graph capture")
            new = dict(device=p.device)
            st["step"] = torch.zeros((), dtype=torch.int64, **new)
            if bits == 32:
                st["exp_avg"], st["exp_avg_sq"] = (torch.zeros(p.shape, dtype=torch.float32, **new) for _ in range(2))
            else:
                blocks = -(-p.numel() // STATE_BLOCK)
                for name in ("exp_avg", "exp_avg_sq"):
                    st[name] = torch.zeros(p.shape, dtype=torch.uint8, **new).view(STATE8_DTYPE)
                    st[name + "_scale"] = torch.zeros(blocks, dtype=torch.float32, **new)
        return st

    def load_state_dict(self, state_dict) -> None:
        """As the base class, hooks included, but every state keeps the type it was saved in, and a learning rate held in
        a tensor comes to the parameters' device, as states do. What no step can go on from
        (another optimizer's checkpoint, states of other types or sizes) is refused before anything is changed."""
        loaded: dict = {}

        def last(_, final) -> None:  # behind the other pre-hooks: what the base class is about to load
            for group, own in zip(final["param_groups"], self.param_groups):
                if missing := [k for k in _GROUP if k not in group]:
                    raise ValueError(f"no checkpoint of this optimizer: a group lacks {', '.join(missing)}")
                _check_group(group)
                for i, p in zip(group["params"], own["params"]):
                    if final["state"].get(i):
                        _check_state(final["state"][i], p, group["state_bits"])
            loaded.update(final)

        def first(_) -> None:  # ahead of the other post-hooks: the base class has cast states to their parameters' type
            for group in self.param_groups:
                if isinstance(group["lr"], torch.Tensor) and group["params"]:
                    group["lr"] = group["lr"].to(group["params"][0].device)
            ids = [i for g in loaded["param_groups"] for i in g["params"]]
            for i, p in zip(ids, (p for g in self.param_groups for p in g["params"])):
                if i in loaded["state"]:
                    self.state[p] = {k: v.detach().to(p.device, copy=True) if isinstance(v, torch.Tensor) else v
                                     for k, v in loaded["state"][i].items()}

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
            bits, state = group["state_bits"], self.state
            states = [state[p] or self._state(p, bits) for p in ps]
            steps, avgs, sqs, *scales = zip(*map(_STATES[bits], states))
            adamw_step(ps, grads, avgs, sqs, steps, lr=group["lr"], betas=group["betas"], eps=group["eps"],
                       weight_decay=group["weight_decay"], grad_scale=scale,
                       **dict(zip(("exp_avg_scales", "exp_avg_sq_scales"), scales)))
        return loss
