"""Dense layers in 8-bit floating point, with 8-bit activation checkpoints.

``fp8_dense(x, w, bias, act)`` is ``fused_dense``'s form in e4m3: x and w are
rounded to 8 bits with one power-of-two scale for each block of 128 (x: 128
neighbours along the contraction; w: tiles of 128 x 128) and multiplied by the
matrix cores. A result in 32 bits is added in 32 bits. One in 16 bits is added
in 32 too, but within eight neighbouring products with about 16 bits below the
largest of them, as the 8-bit instructions do; not so in front of a relu whose
gradient is asked for: the sign of each such sum decides a gradient, and all of
them are added in 32 bits.

In training the layer keeps its input for the backward pass in 8 bits
instead of 16: x^T in blocks of 128 rows of the batch, and one bit for each
output of a relu. The backward pass multiplies from these: with dz the
gradient before the activation and q() the rounding to blocks,

    db = sum over rows of dz
    dx = q(dz) q(w)               blocks along the outputs
    dw = q(dz^T) q(x^T)^T         blocks along the batch

For serving, ``quantize_fp8_weight`` lays a weight out once and ``fp8_dense``
takes the result in the weight's place.

On CUDA devices these are the kernels of csrc/fp8_kernels.hip; on the CPU the
same arithmetic in torch (ops/reference.py), to the bit in what is stored.
"""

from typing import Optional, Union

import torch
from torch.autograd.function import once_differentiable

from elasticdl_amd.ops import reference, require_native, use_native
from elasticdl_amd.ops.functional import _ACTS, ACT_RELU, ACT_SIGMOID

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


class Fp8Blocks:
    """A matrix [rows, cols] in e4m3 with a scale for each block of 128.

    ``data``: uint8 [rows, cols rounded up to 128], zeros behind cols;
    ``scale``: uint8 [blocks, rows rounded up to 256], a scale's exponent
    + 127 at ``reference.fp8_scale_slots``'s place for each row."""

    def __init__(self, data: torch.Tensor, scale: torch.Tensor, cols: int):
        self.data = data
        self.scale = scale
        self.shape = (data.shape[0], cols)

    @property
    def device(self):
        return self.data.device

    def dequantize(self) -> torch.Tensor:
        """The values that are stored, in float32."""
        return reference.fp8_values(self.data, self.scale, self.shape[1])

    def __repr__(self):
        return f"Fp8Blocks(shape={self.shape}, device={self.device})"


def _check_matrix(t: torch.Tensor, name: str) -> None:
    if t.dim() != 2:
        raise ValueError(f"{name} must have two dimensions, not {t.dim()}")
    if t.dtype not in _DTYPES:
        raise TypeError(
            f"{name} must be float32, bfloat16 or float16, not {t.dtype}")
    if t.shape[1] == 0:
        raise ValueError(f"{name} has no columns")


def quantize_fp8(x: torch.Tensor, tile: bool = False) -> Fp8Blocks:
    """x [rows, cols] in blocks of 128 neighbours in a row, or in tiles of
    128 x 128 (``tile``). Values that are not finite become NaN and leave
    their block's scale alone."""
    _check_matrix(x, "x")
    x = x.detach()
    if use_native(x.device):
        from elasticdl_amd.ops import _C

        q, s, _, _ = _C.fp8_quantize(x, tile, True, False)
    else:
        q, s = reference.fp8_quantize(x, tile)
    return Fp8Blocks(q, s, x.shape[1])


def quantize_fp8_weight(w: torch.Tensor) -> Fp8Blocks:
    """A weight [out, in] laid out for serving with ``fp8_dense``. Later
    changes of ``w`` do not reach it."""
    return quantize_fp8(w, tile=True)


class _Fp8DenseFn(torch.autograd.Function):
    """The CPU's; a GPU's is in csrc/fp8_bindings.cpp."""

    @staticmethod
    def forward(ctx, x, w, bias, act):
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        wtq = wts = None
        if need_x:
            wtq, wts = reference.fp8_quantize(w.t(), True)
        y, xtq, xts, mask = reference.fp8_dense_fwd(
            x, *reference.fp8_quantize(w, True), bias, act, need_w,
            act == ACT_RELU and (need_x or need_w or need_b))
        ctx.act = act
        ctx.k = x.shape[1]
        ctx.types = (w.dtype, None if bias is None else bias.dtype)
        ctx.save_for_backward(
            mask, y if act == ACT_SIGMOID else None, wtq, wts, xtq, xts)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        return (*reference.fp8_dense_bwd(
            dy, ctx.act, *ctx.saved_tensors, ctx.k, *ctx.needs_input_grad[:3],
            *ctx.types), None)


def fp8_dense(x: torch.Tensor, w: Union[torch.Tensor, Fp8Blocks],
              bias: Optional[torch.Tensor] = None,
              act: str = "none") -> torch.Tensor:
    """act(x @ w^T + bias), x [..., in], w [out, in], in e4m3 as above.

    x, w and bias are float32, bfloat16 or float16, each its own; y and dx
    have x's type, dw and db their parameter's. Gradients reach x, w and bias
    where w is a tensor. With a weight from ``quantize_fp8_weight`` the call
    serves only: it refuses inputs that require a gradient, and up to 16 rows
    are one launch that rounds x in registers.

    In code that is captured into a graph, take gradients with
    ``torch.autograd.grad`` (or drop eager graphs of the same leaves first):
    ``backward()`` accumulates on the stream of the eager graph's leaves,
    which ends the capture."""
    act_id = _ACTS.get(act)
    if act_id is None:
        raise ValueError(f"unknown activation {act!r}, not in {list(_ACTS)}")
    frozen = isinstance(w, Fp8Blocks)
    if x.is_cuda:
        C = require_native()
        if frozen:
            return C.fp8_dense_frozen(x, w.data, w.scale, w.shape[1], bias,
                                      act_id)
        return C.fp8_dense(x, w, bias, act_id)
    if not frozen:
        _check_matrix(w, "w")
    if x.dtype not in _DTYPES:
        raise TypeError(
            f"x must be float32, bfloat16 or float16, not {x.dtype}")
    n, k = w.shape
    if x.dim() < 1 or x.shape[-1] != k:
        raise ValueError(f"x is {tuple(x.shape)}, and the weight takes {k}")
    if w.device != x.device:
        raise ValueError(f"x is on {x.device}, and the weight on {w.device}")
    if n == 0:
        raise ValueError("the weight has no rows")
    if bias is not None:
        if bias.shape != (n,):
            raise ValueError(f"bias is {tuple(bias.shape)}, not ({n},)")
        if bias.dtype not in _DTYPES:
            raise TypeError("bias must be float32, bfloat16 or float16, "
                            f"not {bias.dtype}")
        if bias.device != x.device:
            raise ValueError(
                f"x is on {x.device}, and the bias on {bias.device}")
    x2 = x.reshape(-1, k)
    if not frozen:
        y = _Fp8DenseFn.apply(x2, w, bias, act_id)
    else:
        if torch.is_grad_enabled() and (
                x.requires_grad or (bias is not None and bias.requires_grad)):
            raise RuntimeError(
                "a weight from quantize_fp8_weight has no backward pass: call "
                "under torch.no_grad(), or pass the weight as a tensor")
        y = reference.fp8_dense_fwd(x2, w.data, w.scale, bias, act_id, False,
                                    False)[0]
    return y.reshape(*x.shape[:-1], n)
