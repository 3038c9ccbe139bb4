"""The mixture-of-experts layer around the experts' products: the top-k router, the movement
of token rows to expert order and back, and their gradients.

    r = moe_route(logits, top_k)                       # weights, experts, rows, m_offsets
    xs = moe_dispatch(x, r)                            # token rows in expert order
    ys = linear_grouped(..., r.m_offsets ...)          # or quantize_grouped + gemm_grouped
    y = moe_combine(ys, r, residual=x)                 # weighted sum back in token order

Asynchronous on torch's current stream; nothing of the routing passes through the host.
"""
from typing import NamedTuple, Optional, Tuple

import torch

from ._lib import SCORES, lib
from .layers import _DTYPES, _matrix, _ptr, call


class Routing(NamedTuple):
    """What moe_route decides, all on the device."""
    weights: torch.Tensor    # fp32 [T, top_k]
    experts: torch.Tensor    # int32 [T, top_k], -1 where a token has no expert left
    rows: torch.Tensor       # int32 [T, top_k], the choice's row in expert order, or -1
    m_offsets: torch.Tensor  # int32 [E + 1], the experts' row offsets


def _logits(logits: torch.Tensor) -> Tuple[int, int]:
    if not logits.is_cuda or logits.ndim != 2 or logits.dtype not in _DTYPES or not logits.is_contiguous():
        raise ValueError("logits must be a contiguous 2-D bf16, fp16 or fp32 CUDA tensor")
    return logits.shape


def _scoring(scoring: str) -> int:
    if scoring not in SCORES:
        raise ValueError(f"scoring must be one of {sorted(SCORES)}")
    return SCORES[scoring]


def moe_route(logits: torch.Tensor, top_k: int, scoring: str = "softmax", bias: Optional[torch.Tensor] = None,
              renormalize: bool = True, scale: float = 1.0) -> Routing:
    """The top_k experts of each token of logits [T, E] and their weights.

    scoring "softmax" or "sigmoid"; the experts are taken by highest logit, or with bias
    (fp32 [E], sigmoid only; it does not enter the weights) by highest score + bias, the
    lowest index first among equals.  weights = scores, divided by the sum of the chosen
    ones if renormalize, times scale.  An expert whose logit is -inf or NaN is never chosen;
    a choice that finds none left is -1 with weight 0.  E <= 256, top_k <= 32."""
    T, E = _logits(logits)
    score = _scoring(scoring)
    if bias is not None:
        if score != SCORES["sigmoid"]:
            raise ValueError("a selection bias needs sigmoid scoring")
        if bias.dtype != torch.float32 or bias.shape != (E,) or bias.device != logits.device or not bias.is_contiguous():
            raise ValueError(f"bias must be a contiguous float32 tensor of {E} entries on {logits.device}")
    weights = logits.new_empty((T, top_k), dtype=torch.float32)
    experts, rows = logits.new_empty((2, T, top_k), dtype=torch.int32).unbind(0)
    m_offsets = logits.new_empty(E + 1, dtype=torch.int32)
    ws, ws_bytes = None, 0
    if T > 64:
        ws_bytes = lib().nvfp4_moe_route_workspace_size(T, E)
        ws = logits.new_empty(ws_bytes // 4, dtype=torch.int32)
    call("nvfp4_moe_route", logits.get_device(), logits.data_ptr(), _DTYPES[logits.dtype], _ptr(bias), T, E, top_k, score,
         int(renormalize), scale, weights.data_ptr(), experts.data_ptr(), rows.data_ptr(), m_offsets.data_ptr(),
         _ptr(ws), ws_bytes)
    return Routing(weights, experts, rows, m_offsets)


def moe_route_backward(dweights: torch.Tensor, logits: torch.Tensor, routing: Routing, scoring: str = "softmax",
                       renormalize: bool = True, scale: float = 1.0) -> torch.Tensor:
    """Gradient of the logits [T, E] from dweights fp32 [T, top_k]; the choice is constant."""
    T, E = _logits(logits)
    experts = routing.experts
    k = experts.shape[1]
    _check_ints(experts, "experts", (T, k), logits.get_device())
    if dweights.dtype != torch.float32 or dweights.shape != (T, k) or \
            dweights.get_device() != logits.get_device() or \
            not dweights.is_contiguous():
        raise ValueError(f"dweights must be a contiguous float32 tensor ({T}, {k}) on {logits.device}")
    dl = torch.empty_like(logits)
    call("nvfp4_moe_route_backward", logits.get_device(), dweights.data_ptr(), logits.data_ptr(), _DTYPES[logits.dtype],
         experts.data_ptr(), T, E, k, _scoring(scoring), int(renormalize), scale, dl.data_ptr())
    return dl


def _check_ints(t: torch.Tensor, name: str, shape, index: int) -> None:
    if t.dtype != torch.int32 or t.shape != shape or t.get_device() != index or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor {tuple(shape)} on CUDA device {index}")


def _routed(routing: Routing, index: int) -> Tuple[int, int, int]:
    """(tokens, top_k, experts) of a routing on CUDA device `index`."""
    w, _, rows, offs = routing
    if rows.ndim != 2 or offs.ndim != 1:
        raise ValueError("routing.rows must be 2-D and routing.m_offsets 1-D")
    shape = rows.shape
    _check_ints(rows, "routing.rows", shape, index)
    _check_ints(offs, "routing.m_offsets", offs.shape, index)
    if w.dtype != torch.float32 or w.shape != shape or w.get_device() != index or not w.is_contiguous():
        raise ValueError(f"routing.weights must be a contiguous float32 tensor {tuple(shape)} on CUDA device {index}")
    return shape[0], shape[1], offs.numel() - 1


def _rows16(t: torch.Tensor, name: str, rows: int) -> int:
    if not t.is_cuda or t.ndim != 2 or _DTYPES.get(t.dtype, 2) == 2 or not t.is_contiguous() or t.shape[0] != rows:
        raise ValueError(f"{name} must be a contiguous 2-D bf16 or fp16 CUDA tensor of {rows} rows")
    K = t.shape[1]
    if K % 8 or not K:
        raise ValueError(f"{name} must have a multiple of 8 columns")
    return K


def moe_dispatch(x: torch.Tensor, routing: Routing) -> torch.Tensor:
    """x [T, K] -> [T * top_k, K] in expert order, a copy of a token's row for each of its
    choices; rows past m_offsets[-1] (masked choices) are zero."""
    T, k, E = _routed(routing, x.get_device())
    K = _rows16(x, "x", T)
    out = x.new_empty((T * k, K))
    call("nvfp4_moe_dispatch", x.get_device(), x.data_ptr(), routing.rows.data_ptr(), routing.m_offsets.data_ptr(), T, E, k,
         K, out.data_ptr())
    return out


def moe_dispatch_backward(dx_rows: torch.Tensor, routing: Routing) -> torch.Tensor:
    """Gradient of moe_dispatch: dx[t] = the sum of the rows of t's choices."""
    T, k, _ = _routed(routing, dx_rows.get_device())
    K = _rows16(dx_rows, "dx_rows", T * k)
    dx = dx_rows.new_empty((T, K))
    call("nvfp4_moe_combine", dx.get_device(), dx_rows.data_ptr(), _DTYPES[dx.dtype], routing.rows.data_ptr(), None, None, T,
         k, K, dx.data_ptr())
    return dx


def moe_combine(x_rows: torch.Tensor, routing: Routing, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y[t] = residual[t] + sum_j weights[t, j] * x_rows[rows[t, j]], summed in fp32."""
    T, k, _ = _routed(routing, x_rows.get_device())
    K = _rows16(x_rows, "x_rows", T * k)
    if residual is not None:
        _matrix(residual, "residual", (T, K), x_rows)
    y = x_rows.new_empty((T, K))
    call("nvfp4_moe_combine", y.get_device(), x_rows.data_ptr(), _DTYPES[y.dtype], routing.rows.data_ptr(),
         routing.weights.data_ptr(), _ptr(residual), T, k, K, y.data_ptr())
    return y


def moe_combine_backward(dy: torch.Tensor, x_rows: torch.Tensor, routing: Routing):
    """Gradients (dx_rows [T * top_k, K], dweights fp32 [T, top_k]) of moe_combine; the
    residual's gradient is dy itself."""
    T, k, E = _routed(routing, x_rows.get_device())
    K = _rows16(x_rows, "x_rows", T * k)
    _matrix(dy, "dy", (T, K), x_rows)
    dx_rows = torch.empty_like(x_rows)
    dweights = dy.new_empty((T, k), dtype=torch.float32)
    call("nvfp4_moe_combine_backward", dy.get_device(), dy.data_ptr(), x_rows.data_ptr(), _DTYPES[dy.dtype],
         routing.rows.data_ptr(), routing.weights.data_ptr(), routing.m_offsets.data_ptr(), T, E, k, K,
         dx_rows.data_ptr(), dweights.data_ptr())
    return dx_rows, dweights
