"""The mixture-of-experts layer around the experts' products: the top-k router, the movement
of token rows to expert order and back, and their gradients.

    r = moe_route(logits, top_k)                       # weights, experts, rows, m_offsets
    xs = moe_dispatch(x, r)                            # token rows in expert order
    ys = linear_grouped(..., r.m_offsets ...)          # or quantize_grouped + gemm_grouped
    y = moe_combine(ys, r, residual=x)                 # weighted sum back in token order

Asynchronous on torch's current stream; nothing of the routing passes through the host.
These functions record no autograd graph; the operators of the same names in
torch.ops.nvfp4_b200 do.
"""
from typing import NamedTuple, Optional

import torch

from ._bind import native
from ._lib import SCORES


class Routing(NamedTuple):
    """What moe_route decides, all on the device."""
    weights: torch.Tensor    # fp32 [T, top_k]
    experts: torch.Tensor    # int32 [T, top_k], -1 where a token has no expert left
    rows: torch.Tensor       # int32 [T, top_k], the choice's row in expert order, or -1
    m_offsets: torch.Tensor  # int32 [E + 1], the experts' row offsets


def _scoring(name: str) -> int:
    code = SCORES.get(name)
    if code is None:
        raise ValueError(f"scoring must be one of {sorted(SCORES)}")
    return code


def moe_route(logits: torch.Tensor, top_k: int, scoring: str = "softmax", bias: Optional[torch.Tensor] = None,
              renormalize: bool = True, scale: float = 1.0) -> Routing:
    """The top_k experts of each token of logits [T, E] and their weights.

    scoring "softmax" or "sigmoid"; the experts are taken by highest logit, or with bias
    (fp32 [E], sigmoid only; it does not enter the weights) by highest score + bias, the
    lowest index first among equals.  weights = scores, divided by the sum of the chosen
    ones if renormalize, times scale.  An expert whose logit is -inf or NaN is never chosen;
    a choice that finds none left is -1 with weight 0.  E <= 256, top_k <= 32."""
    return Routing._make(native.moe_route(logits, top_k, _scoring(scoring), bias, renormalize, scale))


def moe_route_backward(dweights: torch.Tensor, logits: torch.Tensor, routing: Routing, scoring: str = "softmax",
                       renormalize: bool = True, scale: float = 1.0) -> torch.Tensor:
    """Gradient of the logits [T, E] from dweights fp32 [T, top_k]; the choice is constant."""
    return native.moe_route_backward(dweights, logits, routing[1], _scoring(scoring), renormalize, scale)


def moe_dispatch(x: torch.Tensor, routing: Routing) -> torch.Tensor:
    """x [T, K] -> [T * top_k, K] in expert order, a copy of a token's row for each of its
    choices; rows past m_offsets[-1] (masked choices) are zero."""
    return native.moe_dispatch(x, routing)


def moe_dispatch_backward(dx_rows: torch.Tensor, routing: Routing) -> torch.Tensor:
    """Gradient of moe_dispatch: dx[t] = the sum of the rows of t's choices."""
    return native.moe_combine(dx_rows, routing, None, False)


def moe_combine(x_rows: torch.Tensor, routing: Routing, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y[t] = residual[t] + sum_j weights[t, j] * x_rows[rows[t, j]], summed in fp32."""
    return native.moe_combine(x_rows, routing, residual, True)


def moe_combine_backward(dy: torch.Tensor, x_rows: torch.Tensor, routing: Routing):
    """Gradients (dx_rows [T * top_k, K], dweights fp32 [T, top_k]) of moe_combine; the
    residual's gradient is dy itself."""
    return native.moe_combine_backward(dy, x_rows, routing)
