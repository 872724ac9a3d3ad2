"""Block-scaled (microscaled) 4- and 8-bit floating point: quantisation, products and the norm that
feeds them.

Beside the INT4 path of :mod:`.linear` this module runs linears in the formats whose scales the
tensor cores apply themselves (``tcgen05`` block-scaled MMAs), so neither operand is converted on
the way:

========  ======  =====  ================================================
format    codes   block  scale
========  ======  =====  ================================================
nvfp4     e2m1    16     e4m3 per block, one fp32 per tensor
mxfp4     e2m1    32     power of two per block
mxfp8     e4m3    32     power of two per block (activations only)
========  ======  =====  ================================================

* :func:`quantize` / :func:`dequantize` / :func:`tensor_scale`: a matrix to :class:`MicroTensor` and back.
* :func:`matmul`: ``A @ W^T + bias`` of two of them (nvfp4 x nvfp4, mxfp4 x mxfp4, mxfp8 x mxfp4).
* :func:`linear`, :class:`MicroscaledLinear`: quantise the activations, then the product.
* :func:`rms_norm`: residual addition, root-mean-square norm and mxfp8 output in one pass, so that
  the linears which read a block's normed activations share one quantisation.

For inference, like :mod:`.linear`: outputs carry no gradient.

The reference has no counterpart: its weights are INT4 with bf16 group scales
(src/krea2_svdquant/quant/pack.py:6-70).
"""
from __future__ import annotations

from dataclasses import dataclass

import torch
from torch import nn

from . import _lib, ops

FORMATS = tuple(ops.MX_BLOCK)
_INTEGER = {2: torch.int16, 4: torch.int32, 8: torch.int64}  # by bytes
ACTIVATIONS = {act: w for act, w in ops.MX_PRODUCTS}  # activation format -> the weight format it multiplies


def _kernels():
    return ops if torch.compiler.is_compiling() else ops.eager


@dataclass(slots=True)
class MicroTensor:
    """A block-scaled matrix: ``codes`` and ``scales`` as ``ops.mx_quantize`` writes them, the format,
    the shape of the values (codes are the rows of ``shape`` flattened to 2-D), nvfp4's tensor scale and the
    type of the values it was made from (None where that is not known), which a linear's output takes."""

    codes: torch.Tensor
    scales: torch.Tensor
    fmt: str
    shape: tuple[int, ...]
    tensor_scale: torch.Tensor | None = None
    dtype: torch.dtype | None = None

    @property
    def device(self) -> torch.device:
        return self.codes.device


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x [..., K] as 2-D rows with unit column stride that do not overlap (a view where its strides
    allow one, otherwise a copy: a transposed or an expanded x)."""
    if x.dim() < 1:
        raise ValueError("expected a tensor with at least one dimension")
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    if x.is_contiguous() or (x.stride(1) == 1 and x.stride(0) >= x.shape[1]):
        return x
    return x.contiguous()


def tensor_scale(x: torch.Tensor) -> torch.Tensor:
    """The nvfp4 tensor scale of x: ``max |x| / (6 * 448)``, one fp32 value on x's device."""
    return _kernels().mx_tensor_scale(_rows(x))


def quantize(x: torch.Tensor, fmt: str = "nvfp4", *, tensor_scale: torch.Tensor | None = None) -> MicroTensor:
    """``x [..., K]`` (bf16, fp16, fp32) in format ``fmt``.  nvfp4 takes a calibrated ``tensor_scale``
    (None: 1); for weights use :func:`tensor_scale`.  Codes are those of the exact quotients, ties to
    even; a block with an infinity or a NaN reads back as NaN."""
    codes, scales = _kernels().mx_quantize(_rows(x), fmt, tensor_scale)
    return MicroTensor(codes, scales, fmt, x.shape, tensor_scale, x.dtype)


def dequantize(t: MicroTensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values of ``t`` (``code * scale * tensor scale`` in fp32, rounded once to ``dtype``)."""
    out = _kernels().mx_dequantize(t.codes, t.scales, t.fmt, t.shape[-1], t.tensor_scale, dtype)
    return out if len(t.shape) == 2 else out.reshape(t.shape)


def matmul(a: MicroTensor, w: MicroTensor, bias: torch.Tensor | None = None, *,
           out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``a @ w^T + bias``: activations ``a [..., K]``, weight ``w [N, K]``, bias [N] bf16."""
    if len(w.shape) != 2 or a.shape[-1] != w.shape[1]:
        raise ValueError(f"matmul: activations {a.shape} and weight {w.shape} do not match")
    out = _kernels().mx_gemm(a.codes, a.scales, a.fmt, a.tensor_scale, w.codes, w.scales, w.fmt, w.tensor_scale,
                             w.shape[1], bias, out_dtype)
    return out if len(a.shape) == 2 else out.reshape(*a.shape[:-1], w.shape[0])


def linear(x: torch.Tensor | MicroTensor, w: MicroTensor, bias: torch.Tensor | None = None, *, act: str | None = None,
           act_scale: torch.Tensor | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``x @ w^T + bias`` with x quantised to format ``act`` on the way (None: the weight's own format;
    ``act_scale``: its calibrated nvfp4 tensor scale).  An x that is a :class:`MicroTensor` already goes
    straight to the product.  The output has x's dtype (a MicroTensor's that of the values it was made from,
    bf16 where that is not known) unless ``out_dtype`` says otherwise."""
    if isinstance(x, MicroTensor):
        return matmul(x, w, bias, out_dtype=out_dtype or x.dtype or torch.bfloat16)
    if len(w.shape) != 2 or x.dim() < 1 or x.shape[-1] != w.shape[1]:
        raise ValueError(f"linear: activations {tuple(x.shape)} and weight {w.shape} do not match")
    out = _kernels().mx_linear(_rows(x), act or w.fmt, act_scale, w.codes, w.scales, w.fmt, w.tensor_scale, bias,
                               out_dtype or x.dtype)
    return out if x.dim() == 2 else out.reshape(*x.shape[:-1], w.shape[0])


def rms_norm(x: torch.Tensor, weight: torch.Tensor | None = None, *, residual: torch.Tensor | None = None,
             eps: float = 1e-6) -> tuple[MicroTensor, torch.Tensor]:
    """``(norm, h)``: ``h = x + residual`` in x's dtype (x itself without a residual) and the
    root-mean-square norm ``h * rsqrt(mean(h^2) + eps) * weight`` over the last dimension as mxfp8, with
    the codes and scales of its exact value (``eps`` as fp32)."""
    x2 = _rows(x)
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f"rms_norm: residual {tuple(residual.shape)} must have x's shape {tuple(x.shape)}")
    codes, scales, total = _kernels().rms_norm_mx(x2, weight, None if residual is None else _rows(residual), eps)
    if residual is None:
        total = x
    elif x.dim() != 2:
        total = total.reshape(x.shape)
    return MicroTensor(codes, scales, "mxfp8", x.shape, None, x.dtype), total


class MicroscaledLinear(nn.Module):
    """A linear with a block-scaled 4-bit weight: ``act`` is the format of its activations (``nvfp4``,
    ``mxfp4``, or ``mxfp8`` for 8-bit activations on an mxfp4 weight).  ``forward`` takes a tensor, which
    it quantises, or a :class:`MicroTensor` in ``act``'s format (:func:`rms_norm`'s output), which
    several layers can share (with calibrated nvfp4 scales, layers that are given one ``act_scale`` tensor).

    ``check_device_errors``: as on :class:`~krea2_svdquant_b200.linear.SVDQuantLinear`."""

    check_device_errors = False

    def __init__(self, weight: MicroTensor, bias: torch.Tensor | None = None, *, act: str = "nvfp4",
                 act_scale: torch.Tensor | None = None) -> None:
        super().__init__()
        if act not in ACTIVATIONS:
            raise ValueError(f"activation format must be one of {sorted(ACTIVATIONS)}, got {act!r}")
        if weight.fmt != ACTIVATIONS[act]:
            raise ValueError(f"{act} activations multiply a {ACTIVATIONS[act]} weight, got {weight.fmt}")
        if len(weight.shape) != 2:
            raise ValueError(f"the weight must be 2-D, got {weight.shape}")
        if act_scale is not None and act != "nvfp4":
            raise ValueError("only nvfp4 activations have a tensor scale")
        self.act = act
        self.out_features, self.in_features = (int(v) for v in weight.shape)
        self.register_buffer("codes", weight.codes)
        self.register_buffer("scales", weight.scales)
        self.register_buffer("weight_scale", weight.tensor_scale)
        self.register_buffer("act_scale", act_scale)
        self.register_buffer("bias", None if bias is None else bias.to(torch.bfloat16).contiguous())

    @classmethod
    def from_linear(cls, layer: nn.Linear, *, act: str = "nvfp4",
                    act_scale: torch.Tensor | None = None) -> "MicroscaledLinear":
        """Quantises a layer's weight (on its CUDA device)."""
        if act not in ACTIVATIONS:
            raise ValueError(f"activation format must be one of {sorted(ACTIVATIONS)}, got {act!r}")
        w = layer.weight.detach()
        fmt = ACTIVATIONS[act]
        packed = quantize(w, fmt, tensor_scale=tensor_scale(w) if fmt == "nvfp4" else None)
        return cls(packed, None if layer.bias is None else layer.bias.detach(), act=act, act_scale=act_scale)

    def _apply(self, fn, recurse=True):
        # .half() / .to(dtype) casts a model's floating buffers; these have one type each and only move, so
        # they go through fn as integers
        kept = {n: b for n in ("weight_scale", "act_scale", "bias") if (b := self._buffers[n]) is not None}
        views = {n: b.view(_INTEGER[b.element_size()]) for n, b in kept.items()}
        self._buffers.update(views)
        try:
            super()._apply(fn, recurse)
        finally:
            for n, b in kept.items():
                t = self._buffers[n]
                self._buffers[n] = b if t is views[n] else t.view(b.dtype)
        return self

    @property
    def weight(self) -> MicroTensor:
        return MicroTensor(self.codes, self.scales, ACTIVATIONS[self.act], (self.out_features, self.in_features),
                           self.weight_scale)

    def forward(self, x: torch.Tensor | MicroTensor) -> torch.Tensor:
        if isinstance(x, MicroTensor) and x.fmt != self.act:
            raise ValueError(f"this layer takes {self.act} activations, got {x.fmt}")
        y = linear(x, self.weight, self.bias, act=self.act, act_scale=self.act_scale)
        if self.check_device_errors:
            _lib.raise_on_device_error(f"MicroscaledLinear {(self.out_features, self.in_features)}")
        return y

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, out_features={self.out_features}, "
                f"weight={ACTIVATIONS[self.act]}, act={self.act}")
