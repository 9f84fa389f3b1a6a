"""Rows of an embedding by token, and the gradient of its weight, on the HIP path only (``csrc/embedding.hip``, host
side ``csrc/host_train.cpp``): where a model's forward pass begins and its backward pass ends."""
from __future__ import annotations

from typing import Optional

import torch

from . import _native as nat

MAX_ROWS = 1 << 23  # of a weight


def embedding(tokens: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0, padding_idx: Optional[int] = None,
              dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``weight[tokens] * scale``: [..., D] in ``dtype`` (the weight's unless given), computed in fp32 and rounded once.

    tokens [...] int64 (up to 2^30), weight [V, D] (V up to 2^23) fp32 or bf16, both on one ROCm device. The gradient of
    ``weight`` is dense, in its type: every row sums its tokens' gradients in fp32 in an order that the tokens alone
    decide, times ``scale``, rounded once, so that it is the same bits every time. Rows of no token are zeros. The row of
    ``padding_idx`` (from the end where negative) is read like any other and gets no gradient. A token outside 0 .. V - 1
    has a row of NaN and passes no gradient.

    Backward passes can themselves be differentiated. Under graph capture the backward pass is refused while a graph of
    the default stream holds the weight's leaves.
    """
    if padding_idx is None:
        padding = -1
    else:
        rows = weight.shape[0] if isinstance(weight, torch.Tensor) and weight.ndim == 2 else 0
        padding = int(padding_idx) + rows if padding_idx < 0 else int(padding_idx)
        if padding < 0:
            raise ValueError(f"padding_idx must be one of the weight's {rows} rows, got {padding_idx}")
    return nat.host().embedding(tokens, weight, scale, padding, dtype)
