"""16-bit linear layers (bf16 / fp16), dense or grouped by expert, with their gradients:
the layers an NVFP4 model keeps in 16 bits, and the form in which it is trained and
calibrated.  torch tensors in, kernels of libnvfp4_b200.so underneath; asynchronous on
torch's current stream of the tensors' device.  ValueError for arguments of the wrong shape,
type or device, NVFP4Error for a bad status.

    z = x @ w.T + bias;  y = act(z) + residual          (fp32, rounded once)

These functions record no autograd graph: their results do not require grad, whatever their
inputs do.  torch.ops.nvfp4_b200.linear_preact is the differentiable form.

Row groups (mixture of experts) are given by m_offsets, as for gemm_grouped: group g is rows
m_offsets[g] .. m_offsets[g+1] and uses weight rows g*N .. (g+1)*N.
"""
from typing import Optional

import torch

from ._bind import native
from ._lib import ACTIVATIONS


def _activation(name: str) -> int:
    code = ACTIVATIONS.get(name)
    if code is None:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}")
    return code


def linear(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: str = "none",
           residual: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
           return_preact: bool = False):
    """y = act(x @ w.T + bias) + residual in one kernel.

    x [M, K] bf16 or fp16 (rows may be a slice of wider ones, 16-byte aligned), w [N, K],
    bias [N], residual [M, N]; activation "none", "relu", "silu", "gelu_tanh" or "swiglu"
    (rows of w and bias interleaved in blocks of 16 gate, 16 up: swiglu_interleave; N/2
    output columns).  out: where y goes; it may be the residual, and shares memory with no
    other input.  return_preact: also z = x @ w.T + bias [M, N], which linear_backward
    takes when there is an activation."""
    return native.linear(x, w, None, bias, _activation(activation), residual, out, return_preact)


def linear_grouped(x: torch.Tensor, w: torch.Tensor, m_offsets: torch.Tensor, bias: Optional[torch.Tensor] = None,
                   activation: str = "none", out: Optional[torch.Tensor] = None, return_preact: bool = False):
    """linear() by row group: rows m_offsets[g] .. m_offsets[g+1] of x [m_total, K] with
    weight rows g*N .. (g+1)*N of w [groups * N, K] and bias row g of [groups, N].
    m_offsets int32 [groups + 1] on the device (moe_route makes it); rows outside every
    group come out as zeros."""
    if m_offsets is None:
        raise ValueError("m_offsets must be a tensor")
    return native.linear(x, w, m_offsets, bias, _activation(activation), None, out, return_preact)


def linear_backward(dy: torch.Tensor, x: torch.Tensor, w: torch.Tensor, preact: Optional[torch.Tensor] = None,
                    activation: str = "none", bias_grad: bool = False, input_grad: bool = True,
                    weight_grad: bool = True):
    """Gradients (dx [M, K], dw [N, K], db [N]) of linear() for dy [M, Nout], None for those
    that are not wanted; the residual's gradient is dy itself.  preact: linear's z, needed
    with an activation.  dz = dy * act'(z) is rounded to the 16-bit type before the products
    (in fp16 an infinity past 65504); db sums it unrounded."""
    return native.linear_backward(dy, x, w, None, preact, _activation(activation), bias_grad, input_grad, weight_grad)


def linear_grouped_backward(dy: torch.Tensor, x: torch.Tensor, w: torch.Tensor, m_offsets: torch.Tensor,
                            preact: Optional[torch.Tensor] = None, activation: str = "none",
                            bias_grad: bool = False, input_grad: bool = True, weight_grad: bool = True):
    """Gradients (dx, dw [groups * N, K], db [groups, N], None for those that are not wanted)
    of linear_grouped(); zero for a group without rows and for rows outside every group."""
    if m_offsets is None:
        raise ValueError("m_offsets must be a tensor")
    return native.linear_backward(dy, x, w, m_offsets, preact, _activation(activation), bias_grad, input_grad,
                                  weight_grad)
