"""16-bit linear layers (bf16 / fp16), dense or grouped by expert, with their gradients:
the layers an NVFP4 model keeps in 16 bits, and the form in which it is trained and
calibrated.  torch tensors in, kernels of libnvfp4_b200.so underneath; asynchronous on
torch's current stream, errors as in ops.py.

    z = x @ w.T + bias;  y = act(z) + residual          (fp32, rounded once)

Row groups (mixture of experts) are given by m_offsets, as for gemm_grouped: group g is rows
m_offsets[g] .. m_offsets[g+1] and uses weight rows g*N .. (g+1)*N.
"""
from typing import Optional, Tuple

import torch

from ._lib import ACTIVATIONS, check, lib

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_raw_stream = torch._C._cuda_getCurrentRawStream
_device = torch._C._cuda_getDevice
_entries = {}  # entry points by name, bound on their first call


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def call(name: str, index: int, *args) -> None:
    """One entry point on the current stream of CUDA device `index` (the stream is the last
    argument of each of them).  A decode step is a few microseconds of GPU time a call, so
    the path from here to the launch is kept short."""
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = getattr(lib(), name)
    if index == _device():
        status = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, _raw_stream(index))
    if status:
        check(status, name)


def _matrix(t: torch.Tensor, name: str, shape, like: torch.Tensor) -> torch.Tensor:
    """A contiguous CUDA tensor of this shape, of `like`'s type and device."""
    if t.dtype != like.dtype or t.get_device() != like.get_device() or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {like.dtype} tensor {tuple(shape)} on {like.device}")
    return t


def _rows(x: torch.Tensor, name: str) -> Tuple[int, int, int]:
    """(rows, columns, row pitch) of a 2-D 16-bit CUDA tensor whose rows are contiguous."""
    if not x.is_cuda or x.ndim != 2 or _DTYPES.get(x.dtype, 2) == 2:
        raise ValueError(f"{name} must be a 2-D bf16 or fp16 CUDA tensor")
    M, K = x.shape
    if x.is_contiguous():
        pitch = K
    else:
        pitch, unit = x.stride()
        if M <= 1:
            pitch = max(K, pitch)
        if (K > 1 and unit != 1) or pitch < K:
            raise ValueError(f"{name} must have contiguous rows")
    if K % 8 or pitch % 8 or not K:
        raise ValueError(f"{name} must have a multiple of 8 columns, rows 16 bytes aligned")
    return M, K, pitch


def _weight(w: torch.Tensor, groups: int, K: int, x: torch.Tensor) -> int:
    """Rows N of one group's weight."""
    if w.ndim != 2 or w.shape[1] != K or w.shape[0] % groups:
        raise ValueError(f"w must be [{'groups * ' if groups > 1 else ''}N, {K}]")
    N = _matrix(w, "w", w.shape, x).shape[0] // groups
    if N % 8 or not N:
        raise ValueError("N must be a multiple of 8")
    return N


def _offsets(m_offsets: torch.Tensor, x: torch.Tensor) -> int:
    if m_offsets.dtype != torch.int32 or m_offsets.ndim != 1 or m_offsets.numel() < 2 or \
            m_offsets.get_device() != x.get_device() or not m_offsets.is_contiguous():
        raise ValueError("m_offsets must be a contiguous 1-D int32 tensor of groups + 1 entries on the device")
    if m_offsets.numel() > 257:
        raise ValueError("at most 256 groups")
    return m_offsets.numel() - 1


def _activation(name: str, N: int) -> Tuple[int, int]:
    """(code, output columns)."""
    if name not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}")
    if name == "swiglu":
        if N % 32:
            raise ValueError("swiglu: N must be a multiple of 32 (gate and up rows in blocks of 16)")
        return ACTIVATIONS[name], N // 2
    return ACTIVATIONS[name], N


def _forward(x, w, m_offsets, bias, activation, residual, out, return_preact):
    M, K, pitch = _rows(x, "x")
    G = 1 if m_offsets is None else _offsets(m_offsets, x)
    N = _weight(w, G, K, x)
    act, No = _activation(activation, N)
    if bias is not None:
        _matrix(bias, "bias", (N,) if bias.ndim == 1 and G == 1 else (G, N), x)
    if residual is not None:
        _matrix(residual, "residual", (M, No), x)
    y = x.new_empty((M, No)) if out is None else _matrix(out, "out", (M, No), x)
    z = x.new_empty((M, N)) if return_preact else None
    call("nvfp4_linear", x.get_device(), x.data_ptr(), pitch, w.data_ptr(), _ptr(bias), _ptr(residual), y.data_ptr(),
         _ptr(z), _ptr(m_offsets), G, M, N, K, act, _DTYPES[x.dtype])
    return (y, z) if return_preact else y


def linear(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: str = "none",
           residual: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
           return_preact: bool = False):
    """y = act(x @ w.T + bias) + residual in one kernel.

    x [M, K] bf16 or fp16 (rows may be a slice of wider ones, 16-byte aligned), w [N, K],
    bias [N], residual [M, N]; activation "none", "relu", "silu", "gelu_tanh" or "swiglu"
    (rows of w and bias interleaved in blocks of 16 gate, 16 up: swiglu_interleave; N/2
    output columns).  return_preact: also z = x @ w.T + bias [M, N], which linear_backward
    takes when there is an activation."""
    return _forward(x, w, None, bias, activation, residual, out, return_preact)


def linear_grouped(x: torch.Tensor, w: torch.Tensor, m_offsets: torch.Tensor, bias: Optional[torch.Tensor] = None,
                   activation: str = "none", out: Optional[torch.Tensor] = None, return_preact: bool = False):
    """linear() by row group: rows m_offsets[g] .. m_offsets[g+1] of x [m_total, K] with
    weight rows g*N .. (g+1)*N of w [groups * N, K] and bias row g of [groups, N].
    m_offsets int32 [groups + 1] on the device (moe_route makes it); rows outside every
    group come out as zeros."""
    return _forward(x, w, m_offsets, bias, activation, None, out, return_preact)


def _backward(dy, x, w, m_offsets, preact, activation, bias_grad):
    M, K, pitch = _rows(x, "x")
    G = 1 if m_offsets is None else _offsets(m_offsets, x)
    N = _weight(w, G, K, x)
    act, No = _activation(activation, N)
    _matrix(dy, "dy", (M, No), x)
    if act:
        if preact is None:
            raise ValueError("an activation's gradient needs preact")
        _matrix(preact, "preact", (M, N), x)
    dtype, dev, offs = _DTYPES[x.dtype], x.get_device(), _ptr(m_offsets)
    dz = x.new_empty((M, N)) if act else dy
    db = ws = None
    ws_bytes = 0
    if bias_grad:
        db = x.new_empty((N,) if m_offsets is None else (G, N))
        ws_bytes = lib().nvfp4_activation_backward_workspace_size(G, M, N)
        ws = x.new_empty(ws_bytes // 4, dtype=torch.float32)
    if act or bias_grad:
        call("nvfp4_activation_backward", dev, dy.data_ptr(), _ptr(preact) if act else None,
             dz.data_ptr() if act else None, _ptr(db), offs, G, M, N, act, dtype, _ptr(ws), ws_bytes)
    dx = x.new_empty((M, K))
    dw = torch.empty_like(w)
    call("nvfp4_linear_dgrad", dev, dz.data_ptr(), w.data_ptr(), dx.data_ptr(), offs, G, M, N, K, dtype)
    call("nvfp4_linear_wgrad", dev, dz.data_ptr(), x.data_ptr(), pitch, dw.data_ptr(), offs, G, M, N, K, dtype)
    return dx, dw, db


def linear_backward(dy: torch.Tensor, x: torch.Tensor, w: torch.Tensor, preact: Optional[torch.Tensor] = None,
                    activation: str = "none", bias_grad: bool = False):
    """Gradients (dx [M, K], dw [N, K], db [N] or None) of linear() for dy [M, Nout]; the
    residual's gradient is dy itself.  preact: linear's z, needed with an activation."""
    return _backward(dy, x, w, None, preact, activation, bias_grad)


def linear_grouped_backward(dy: torch.Tensor, x: torch.Tensor, w: torch.Tensor, m_offsets: torch.Tensor,
                            preact: Optional[torch.Tensor] = None, activation: str = "none",
                            bias_grad: bool = False):
    """Gradients (dx, dw [groups * N, K], db [groups, N] or None) of linear_grouped(); zero
    for a group without rows and for rows outside every group."""
    return _backward(dy, x, w, m_offsets, preact, activation, bias_grad)
