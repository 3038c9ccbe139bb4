"""PyTorch custom operators over the C ABI: torch.ops.nvfp4_b200.gemm, .quantize,
.gemm_epilogue (bias + activation fused) and .gemm_nvfp4_out (the epilogue's
result quantized to NVFP4 for the next layer).

Registered with torch.library, so they carry schemas, run under torch.compile /
FX tracing as opaque ops (fake implementations give output shapes without a GPU)
and can be called from TorchScript-free model code the way the reference's
harness calls torch._scaled_mm (matmul/sm100_nvfp4/main.py:25-34).  The CUDA
implementations are the library's kernels; there is no CPU implementation.
"""
from typing import Optional, Tuple

import torch

from ._bind import native
from .layers import _activation
from .layout import sf_bytes
from .moe import _scoring
from .ops import gemm as _gemm
from .ops import gemm_epilogue as _gemm_epilogue
from .ops import quantize as _quantize


@torch.library.custom_op("nvfp4_b200::gemm", mutates_args=(), device_types="cuda")
def gemm(a: torch.Tensor, sfa: torch.Tensor, b: torch.Tensor, sfb: torch.Tensor, alpha: float,
         fp16_out: bool = False) -> torch.Tensor:
    """D = alpha * A . B^T; A [M, K/2] and B [N, K/2] e2m1 codes, blocked e4m3 scales;
    bf16 (or fp16) [M, N]."""
    return _gemm(a, sfa, b, sfb, alpha, out_dtype=torch.float16 if fp16_out else torch.bfloat16)


@gemm.register_fake
def _gemm_fake(a, sfa, b, sfb, alpha, fp16_out=False):
    return a.new_empty((a.shape[0], b.shape[0]), dtype=torch.float16 if fp16_out else torch.bfloat16)


@torch.library.custom_op("nvfp4_b200::quantize", mutates_args=(), device_types="cuda")
def quantize(x: torch.Tensor, global_scale: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """bf16 [M, K] -> (e2m1 codes uint8 [M, K/2], blocked e4m3 scales uint8 [pad128(M)*K/16])."""
    return _quantize(x, global_scale)


@quantize.register_fake
def _quantize_fake(x, global_scale):
    M, K = x.shape
    return (x.new_empty((M, K // 2), dtype=torch.uint8), x.new_empty((sf_bytes(M, K),), dtype=torch.uint8))


@torch.library.custom_op("nvfp4_b200::gemm_epilogue", mutates_args=(), device_types="cuda")
def gemm_epilogue(a: torch.Tensor, sfa: torch.Tensor, b: torch.Tensor, sfb: torch.Tensor, alpha: float,
                  bias: Optional[torch.Tensor] = None, activation: str = "none") -> torch.Tensor:
    """bf16 D = act(alpha * A . B^T + bias) in one kernel."""
    return _gemm_epilogue(a, sfa, b, sfb, alpha, bias=bias, activation=activation)


@gemm_epilogue.register_fake
def _gemm_epilogue_fake(a, sfa, b, sfb, alpha, bias=None, activation="none"):
    N = b.shape[0] // 2 if activation == "swiglu" else b.shape[0]
    return a.new_empty((a.shape[0], N), dtype=torch.bfloat16)


@torch.library.custom_op("nvfp4_b200::gemm_nvfp4_out", mutates_args=(), device_types="cuda")
def gemm_nvfp4_out(a: torch.Tensor, sfa: torch.Tensor, b: torch.Tensor, sfb: torch.Tensor, alpha: float,
                   out_global_scale: torch.Tensor, bias: Optional[torch.Tensor] = None,
                   activation: str = "none") -> Tuple[torch.Tensor, torch.Tensor]:
    """act(alpha * A . B^T + bias) quantized to NVFP4 in the epilogue: (codes [M, N/2],
    blocked scales [pad128(M) * N/16]), the next layer's operand."""
    return _gemm_epilogue(a, sfa, b, sfb, alpha, bias=bias, activation=activation,
                          out_global_scale=out_global_scale)


@gemm_nvfp4_out.register_fake
def _gemm_nvfp4_out_fake(a, sfa, b, sfb, alpha, out_global_scale, bias=None, activation="none"):
    M, N = a.shape[0], b.shape[0] // 2 if activation == "swiglu" else b.shape[0]
    return (a.new_empty((M, N // 2), dtype=torch.uint8), a.new_empty((sf_bytes(M, N),), dtype=torch.uint8))


# ----------------------------------------------------------------------- 16-bit layers
# nvfp4_b200::linear / ::linear_preact (differentiable) and the mixture-of-experts router and
# row movement.  Optional results are empty tensors where they are not asked for.
def _out_columns(w, m_offsets, activation):
    groups = 1 if m_offsets is None else m_offsets.shape[0] - 1
    N = w.shape[0] // groups
    return groups, N, N // 2 if activation == "swiglu" else N


@torch.library.custom_op("nvfp4_b200::linear", mutates_args=(), device_types="cuda")
def linear(x: torch.Tensor, w: torch.Tensor, m_offsets: Optional[torch.Tensor] = None,
           bias: Optional[torch.Tensor] = None, activation: str = "none",
           residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """act(x @ w.T + bias) + residual, dense or (m_offsets) by row group; no gradient."""
    return native.linear(x, w, m_offsets, bias, _activation(activation), residual, None, False)


@linear.register_fake
def _linear_fake(x, w, m_offsets=None, bias=None, activation="none", residual=None):
    return x.new_empty((x.shape[0], _out_columns(w, m_offsets, activation)[2]))


@torch.library.custom_op("nvfp4_b200::linear_preact", mutates_args=(), device_types="cuda")
def linear_preact(x: torch.Tensor, w: torch.Tensor, m_offsets: Optional[torch.Tensor] = None,
                  bias: Optional[torch.Tensor] = None, activation: str = "none",
                  residual: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """linear with its gradient: (y, z), z the pre-activation kept for the backward pass (an
    empty tensor without an activation).  z carries no gradient: a loss on it alone raises."""
    if activation == "none":
        return native.linear(x, w, m_offsets, bias, 0, residual, None, False), x.new_empty(0)
    return native.linear(x, w, m_offsets, bias, _activation(activation), residual, None, True)


@linear_preact.register_fake
def _linear_preact_fake(x, w, m_offsets=None, bias=None, activation="none", residual=None):
    _, N, No = _out_columns(w, m_offsets, activation)
    return x.new_empty((x.shape[0], No)), x.new_empty((0,) if activation == "none" else (x.shape[0], N))


@torch.library.custom_op("nvfp4_b200::linear_backward", mutates_args=(), device_types="cuda")
def linear_backward(dy: torch.Tensor, x: torch.Tensor, w: torch.Tensor, m_offsets: Optional[torch.Tensor],
                    z: torch.Tensor, activation: str, bias_grad: bool, input_grad: bool = True,
                    weight_grad: bool = True) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, dw, db); empty where they are not wanted."""
    out = native.linear_backward(dy, x, w, m_offsets, None if activation == "none" else z, _activation(activation),
                                 bias_grad, input_grad, weight_grad)
    return tuple(x.new_empty(0) if t is None else t for t in out)


@linear_backward.register_fake
def _linear_backward_fake(dy, x, w, m_offsets, z, activation, bias_grad, input_grad=True, weight_grad=True):
    groups, N, _ = _out_columns(w, m_offsets, activation)
    db = (0,) if not bias_grad else (N,) if m_offsets is None else (groups, N)
    return x.new_empty(x.shape if input_grad else 0), w.new_empty(w.shape if weight_grad else 0), x.new_empty(db)


def _linear_context(ctx, inputs, output):
    x, w, m_offsets, bias, activation, residual = inputs
    ctx.save_for_backward(x, w, m_offsets, output[1])
    ctx.mark_non_differentiable(output[1])
    ctx.activation = activation
    ctx.bias_shape = None if bias is None else bias.shape  # dense: [N] or [1, N]
    ctx.set_materialize_grads(False)


def _linear_grad(ctx, dy, _dz):
    if dy is None:
        return None, None, None, None, None, None
    x, w, m_offsets, z = ctx.saved_tensors
    dy = dy.contiguous()
    for_x, for_w, _, for_bias, _, for_residual = (*ctx.needs_input_grad, *[False] * 6)[:6]  # trailing defaults are left out
    dx = dw = db = None
    if for_x or for_w or for_bias:
        dx, dw, db = torch.ops.nvfp4_b200.linear_backward(dy, x, w, m_offsets, z, ctx.activation, for_bias, for_x, for_w)
    return (dx if for_x else None, dw if for_w else None, None, db.view(ctx.bias_shape) if for_bias else None, None,
            dy if for_residual else None)


linear_preact.register_autograd(_linear_grad, setup_context=_linear_context)


@torch.library.custom_op("nvfp4_b200::moe_route", mutates_args=(), device_types="cuda")
def moe_route(logits: torch.Tensor, top_k: int, scoring: str = "softmax", bias: Optional[torch.Tensor] = None,
              renormalize: bool = True,
              scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(weights, experts, rows, m_offsets), the fields of a Routing; the weights carry a
    gradient to the logits."""
    return native.moe_route(logits, top_k, _scoring(scoring), bias, renormalize, scale)


@moe_route.register_fake
def _moe_route_fake(logits, top_k, scoring="softmax", bias=None, renormalize=True, scale=1.0):
    T, E = logits.shape

    def ints(*shape):
        return logits.new_empty(shape, dtype=torch.int32)

    return logits.new_empty((T, top_k), dtype=torch.float32), ints(T, top_k), ints(T, top_k), ints(E + 1)


@torch.library.custom_op("nvfp4_b200::moe_route_backward", mutates_args=(), device_types="cuda")
def moe_route_backward(dweights: torch.Tensor, logits: torch.Tensor, experts: torch.Tensor, scoring: str,
                       renormalize: bool, scale: float) -> torch.Tensor:
    return native.moe_route_backward(dweights, logits, experts, _scoring(scoring), renormalize, scale)


@moe_route_backward.register_fake
def _moe_route_backward_fake(dweights, logits, experts, scoring, renormalize, scale):
    return torch.empty_like(logits)


def _route_context(ctx, inputs, output):
    logits, _, scoring, _, renormalize, scale = inputs
    ctx.save_for_backward(logits, output[1])
    ctx.args = scoring, renormalize, scale
    ctx.set_materialize_grads(False)


def _route_grad(ctx, dweights, *_):
    if dweights is None:
        return None, None, None, None, None, None
    logits, experts = ctx.saved_tensors
    dl = torch.ops.nvfp4_b200.moe_route_backward(dweights.contiguous(), logits, experts, *ctx.args)
    return dl, None, None, None, None, None


moe_route.register_autograd(_route_grad, setup_context=_route_context)


@torch.library.custom_op("nvfp4_b200::moe_dispatch", mutates_args=(), device_types="cuda")
def moe_dispatch(x: torch.Tensor, weights: torch.Tensor, experts: torch.Tensor, rows: torch.Tensor,
                 m_offsets: torch.Tensor) -> torch.Tensor:
    """x [T, K] -> [T * top_k, K] in expert order; differentiable in x."""
    return native.moe_dispatch(x, (weights, experts, rows, m_offsets))


@moe_dispatch.register_fake
def _moe_dispatch_fake(x, weights, experts, rows, m_offsets):
    return x.new_empty((rows.shape[0] * rows.shape[1], x.shape[1]))


@torch.library.custom_op("nvfp4_b200::moe_dispatch_backward", mutates_args=(), device_types="cuda")
def moe_dispatch_backward(dx_rows: torch.Tensor, weights: torch.Tensor, experts: torch.Tensor, rows: torch.Tensor,
                          m_offsets: torch.Tensor) -> torch.Tensor:
    return native.moe_combine(dx_rows, (weights, experts, rows, m_offsets), None, False)


@moe_dispatch_backward.register_fake
def _moe_dispatch_backward_fake(dx_rows, weights, experts, rows, m_offsets):
    return dx_rows.new_empty((rows.shape[0], dx_rows.shape[1]))


def _dispatch_context(ctx, inputs, output):
    ctx.save_for_backward(*inputs[1:])


def _dispatch_grad(ctx, dx_rows):
    dx = torch.ops.nvfp4_b200.moe_dispatch_backward(dx_rows.contiguous(), *ctx.saved_tensors)
    return dx, None, None, None, None


moe_dispatch.register_autograd(_dispatch_grad, setup_context=_dispatch_context)


@torch.library.custom_op("nvfp4_b200::moe_combine", mutates_args=(), device_types="cuda")
def moe_combine(x_rows: torch.Tensor, weights: torch.Tensor, experts: torch.Tensor, rows: torch.Tensor,
                m_offsets: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """residual + the weighted sum of each token's rows; differentiable in x_rows, weights
    and residual."""
    return native.moe_combine(x_rows, (weights, experts, rows, m_offsets), residual, True)


@moe_combine.register_fake
def _moe_combine_fake(x_rows, weights, experts, rows, m_offsets, residual=None):
    return x_rows.new_empty((rows.shape[0], x_rows.shape[1]))


@torch.library.custom_op("nvfp4_b200::moe_combine_backward", mutates_args=(), device_types="cuda")
def moe_combine_backward(dy: torch.Tensor, x_rows: torch.Tensor, weights: torch.Tensor, experts: torch.Tensor,
                         rows: torch.Tensor, m_offsets: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    return native.moe_combine_backward(dy, x_rows, (weights, experts, rows, m_offsets))


@moe_combine_backward.register_fake
def _moe_combine_backward_fake(dy, x_rows, weights, experts, rows, m_offsets):
    return torch.empty_like(x_rows), torch.empty_like(weights)


def _combine_context(ctx, inputs, output):
    ctx.save_for_backward(*inputs[:5])
    ctx.has_residual = inputs[5] is not None


def _combine_grad(ctx, dy):
    dy = dy.contiguous()
    dx_rows, dweights = torch.ops.nvfp4_b200.moe_combine_backward(dy, *ctx.saved_tensors)
    return dx_rows, dweights, None, None, None, dy if ctx.has_residual else None


moe_combine.register_autograd(_combine_grad, setup_context=_combine_context)
