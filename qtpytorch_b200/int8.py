"""Full-int8 layers with a scale a row: the norm that makes the codes, the product
that takes them.

    a, h = rms_norm_quantize(x, weight, residual=h)     # int8d codes, the new residual
    y = int8_matmul(a, w)                               # a @ w^T, bf16
    layer = int8_linear.from_linear(nn_linear)
    y = layer(a)                                        # or layer(x): quantized first

Activations hold one scale a token, weights [N, K] one a channel: the mx_tensors of
``dynamic_quantize(x, "int8d", "per_token")``.  The reference's counterpart is
``fused_int8_linear`` (mxtorch.py:3910-3960), whose fp32 result this product gives
for such operands; it has no norm.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
import torch.nn as nn

from . import _lib as L
from .dtypes import get_mx_dtype
from .tensor import mx_tensor, plain

_IO = {torch.float32: L.F32, torch.bfloat16: L.BF16}
_INT8 = get_mx_dtype("int8d")
MAX_K = 131071  # |a b| <= 2^14: sums that an int32 holds


def _rows(t: torch.Tensor, d: int) -> Tuple[torch.Tensor, int]:
    """A [rows, d] view (or copy) with adjacent elements, and its row stride."""
    if t.dim() != 2:
        t = t.reshape(-1, d)
    ld = t.stride(0) if t.shape[0] > 1 else d
    if (d > 1 and t.stride(1) != 1) or ld < d:
        t, ld = t.contiguous(), d
    return t, ld


def rms_norm_quantize(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None,
                      eps: float = 1e-6) -> Union[mx_tensor, Tuple[mx_tensor, torch.Tensor]]:
    """int8d codes, one scale a row of the last dim, of

        h = x + residual,  y = h * weight / sqrt(mean(h^2) + eps)

    with scale = max(amax|y|, 1e-12) / 127 and code = y / scale to the nearest, ties
    to even, as 64 bits give it: 127 u / amax|u| of u = h * weight, each step rounded to
    a double (a quotient that lies closer to a tie than that is taken for one).  x and
    residual fp32 or bf16 as they are (other and mixed types through fp32), weight [d]
    likewise.  With ``residual`` returns (codes, h), h in x's type.  A row with an infinity or NaN has codes of 0
    and a scale of NaN.  No gradient."""
    x, weight, residual = plain(x), plain(weight), plain(residual)
    L.require_cuda(x, "rms_norm_quantize")
    if x.dim() < 1:
        raise ValueError("rms_norm_quantize: x needs at least one dim")
    shape, dev, dtype = x.shape, x.device, x.dtype
    d = shape[-1]
    if d < 1 or weight.shape != (d,):
        raise ValueError(f"rms_norm_quantize: x {tuple(shape)} needs a weight [{d}] of at least one value, "
                         f"got {tuple(weight.shape)}")
    if not x.is_floating_point() or not weight.is_floating_point():
        raise ValueError("rms_norm_quantize: x and weight hold floating-point numbers")
    if not 0.0 <= eps <= 1e30:
        raise ValueError(f"rms_norm_quantize: eps must not be negative, got {eps}")
    if weight.device != dev or (residual is not None and residual.device != dev):
        raise ValueError(f"rms_norm_quantize: x, weight and residual must be on {dev}")
    if residual is not None:
        if residual.shape != shape or not residual.is_floating_point():
            raise ValueError(f"rms_norm_quantize: residual must be like x {tuple(shape)}, got "
                             f"{residual.dtype} {tuple(residual.shape)}")
        if residual.dtype != dtype:
            x, residual = x.float(), residual.float()
    if x.dtype not in _IO:
        x = x.float()
        residual = None if residual is None else residual.float()
    if weight.dtype not in _IO:
        weight = weight.float()
    weight = weight.contiguous()
    rows = x.numel() // d
    h = None if residual is None else torch.empty(shape, dtype=x.dtype, device=dev)
    codes = torch.empty(rows * d, dtype=torch.int8, device=dev)
    scales = torch.empty(rows, dtype=torch.float32, device=dev)
    ldr = 0
    if rows:
        x, ldx = _rows(x, d)
        if residual is not None:
            residual, ldr = _rows(residual, d)
        rc = L.call("mxb_rms_norm_quantize", dev, x.data_ptr(), L.ptr(residual), _IO[x.dtype], rows, d, ldx, ldr,
                    weight.data_ptr(), _IO[weight.dtype], eps, codes.data_ptr(), scales.data_ptr(), L.ptr(h))
        if rc:
            L.check(rc, f"mxb_rms_norm_quantize({rows}x{d})")
    q = mx_tensor(codes, scales, _INT8, shape, rows * d, d)
    return q if h is None else (q, h if h.dtype == dtype else h.to(dtype))


def _operand(t: mx_tensor, K: int, what: str) -> Tuple[torch.Tensor, torch.Tensor, int]:
    """Codes, scales and the step from a row's scale to the next (0: one scale for all)."""
    dt = t._mx_dtype
    if not (dt.is_int and dt.bits == 8 and dt.variant == ""):
        raise NotImplementedError(f"{what} takes int8 codes, not {dt.name}")
    codes, scales = t._mx_packed, t._mx_scales
    n = t._mx_orig_shape.numel()
    if t._mx_n != n or codes.numel() * codes.element_size() < n or scales.device != codes.device:
        raise ValueError(f"{what} takes whole tensors: {n} codes for {tuple(t._mx_orig_shape)} and their scales on one "
                         f"device, got {codes.numel()} on {codes.device} (n = {t._mx_n}) and scales on {scales.device}")
    rows = n // K if K else 0
    if t._mx_block == K and scales.numel() == rows:
        step = 1
    elif scales.numel() == 1:
        step = 0
    else:
        raise ValueError(f"{what} takes one scale a row of {K} or one for all, not blocks of {t._mx_block}")
    if not codes.is_contiguous():
        codes = codes.contiguous()
    if scales.dtype != torch.float32 or not scales.is_contiguous():
        scales = scales.float().contiguous()
    return codes, scales, step


def _product(a, b, M: int, K: int, N: int, bias: Optional[torch.Tensor], out: torch.Tensor) -> torch.Tensor:
    """a, b: (codes, scales, step) of rows of K; out [.., N] contiguous."""
    dev = out.device
    if K == 0:  # an empty sum
        out.zero_()
        return out if bias is None else out.add_(bias)
    ap, bp = a[0].data_ptr(), b[0].data_ptr()
    wsb = L.size("mxb_int8_matmul_workspace_size", M, K, N, int((ap | bp) % 16 == 0))
    ws = L.workspace(wsb, dev)
    rc = L.call("mxb_int8_matmul", dev, ap, a[1].data_ptr(), a[2], bp, b[1].data_ptr(), b[2], M, K, N,
                L.ptr(bias), out.data_ptr(), _IO[out.dtype], L.ptr(ws), wsb)
    if rc:
        L.check(rc, f"mxb_int8_matmul({M}x{K}x{N})")
    return out


def int8_matmul(a: mx_tensor, b: mx_tensor, bias: Optional[torch.Tensor] = None,
                out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """a [..., K] @ b [N, K]^T (+ bias [N]) of int8 codes with one scale a row (or one
    for all): the exact integer sum, times a's scale, times b's, plus the bias, each step
    (the sum itself past 2^24, too) rounded to fp32, the result to ``out_dtype`` (bf16 or
    fp32).  K at most 131071.  No
    gradient."""
    if not isinstance(a, mx_tensor) or not isinstance(b, mx_tensor):
        raise TypeError("int8_matmul takes two mx_tensors")
    sa, sb = a._mx_orig_shape, b._mx_orig_shape
    if len(sb) != 2 or len(sa) < 1 or sa[-1] != sb[1]:
        raise ValueError(f"int8_matmul: {tuple(sa)} @ {tuple(sb)}^T")
    if out_dtype not in _IO:
        raise ValueError(f"int8_matmul: float32 or bfloat16 out, not {out_dtype}")
    N, K = sb
    if K > MAX_K:
        raise NotImplementedError(f"int8_matmul: rows of at most {MAX_K} codes, not {K}")
    ta, tb = _operand(a, K, "int8_matmul"), _operand(b, K, "int8_matmul")
    L.require_cuda(ta[0], "int8_matmul")
    dev = ta[0].device
    if tb[0].device != dev:
        raise ValueError("int8_matmul: operands on different devices")
    bias = _bias(bias, N, dev, "int8_matmul")
    out = torch.empty((*sa[:-1], N), dtype=out_dtype, device=dev)
    return _product(ta, tb, sa[:-1].numel(), K, N, bias, out)


def _bias(bias: Optional[torch.Tensor], N: int, dev: torch.device, what: str) -> Optional[torch.Tensor]:
    if bias is None:
        return None
    bias = plain(bias)
    if bias.shape != (N,) or bias.device != dev:
        raise ValueError(f"{what}: bias must be [{N}] on {dev}")
    return bias if bias.dtype == torch.float32 and bias.is_contiguous() else bias.float().contiguous()


class int8_linear(nn.Module):
    """nn.Linear with an int8 weight, one scale an output channel.  Activations come
    quantized (``rms_norm_quantize``, ``dynamic_quantize`` per token) or are quantized
    per token on the way.  Inference only (no gradient).  Dtype casts of a model leave
    the codes, the scales and the fp32 bias as they are."""

    def __init__(self, weight: mx_tensor, bias: Optional[torch.Tensor] = None,
                 out_dtype: torch.dtype = torch.bfloat16):
        super().__init__()
        if not isinstance(weight, mx_tensor) or len(weight._mx_orig_shape) != 2:
            raise TypeError("int8_linear takes an mx_tensor [out, in]")
        if out_dtype not in _IO:
            raise ValueError(f"int8_linear: float32 or bfloat16 out, not {out_dtype}")
        self.out_features, self.in_features = weight._mx_orig_shape
        self.out_dtype = out_dtype
        codes, scales, _ = _operand(weight, self.in_features, "int8_linear")
        if scales.numel() != self.out_features:
            scales = scales.expand(self.out_features).contiguous()
        self.register_buffer("weight_codes", codes[:weight._mx_n].view(self.out_features, self.in_features))
        self.register_buffer("weight_scales", scales)
        bias = _bias(None if bias is None else bias.detach(), self.out_features, codes.device, "int8_linear")
        self.register_buffer("bias", bias)

    @classmethod
    def from_linear(cls, linear: nn.Linear, out_dtype: torch.dtype = torch.bfloat16) -> "int8_linear":
        from .dynamic import dynamic_quantize

        w = linear.weight.detach()
        if not w.is_cuda:
            w = w.cuda()
        bias = None if linear.bias is None else linear.bias.detach().to(w.device)
        return cls(dynamic_quantize(w, _INT8, "per_token"), bias, out_dtype)

    def _apply(self, fn, *args, **kwargs):
        # casts of the whole model (.bfloat16(), .half(), .to(dtype)) move these two but
        # leave them fp32: the scales belong to the codes
        kept = {n: self._buffers[n] for n in ("weight_scales", "bias")}
        super()._apply(fn, *args, **kwargs)
        for n, t in kept.items():
            if t is not None and self._buffers[n].dtype != torch.float32:
                self._buffers[n] = t.to(self._buffers[n].device)
        return self

    @property
    def weight(self) -> mx_tensor:
        return mx_tensor(self.weight_codes.view(-1), self.weight_scales, _INT8,
                         (self.out_features, self.in_features), self.weight_codes.numel(), self.in_features)

    def forward(self, x: Union[torch.Tensor, mx_tensor]) -> torch.Tensor:
        K, N = self.in_features, self.out_features
        if not isinstance(x, mx_tensor):
            from .dynamic import dynamic_quantize

            x = dynamic_quantize(x, _INT8, "per_token")
        shape = x._mx_orig_shape
        if len(shape) < 1 or shape[-1] != K:
            raise ValueError(f"int8_linear: {tuple(shape)} @ ({N}, {K})^T")
        if K > MAX_K:
            raise NotImplementedError(f"int8_linear: rows of at most {MAX_K} codes, not {K}")
        a = _operand(x, K, "int8_linear")
        L.require_cuda(a[0], "int8_linear")
        codes = self.weight_codes
        scales, bias = self.weight_scales, self.bias
        if codes.device != a[0].device or scales.device != codes.device:
            raise ValueError("int8_linear: activations and weight on different devices")
        # buffers that were assigned since
        if codes.dtype != torch.int8 or codes.shape != (N, K) or scales.dtype != torch.float32 or scales.shape != (N,):
            raise ValueError(f"int8_linear: int8 codes [{N}, {K}] and fp32 scales [{N}], got {codes.dtype} "
                             f"{tuple(codes.shape)} and {scales.dtype} {tuple(scales.shape)}")
        bias = _bias(bias, N, codes.device, "int8_linear")
        out = torch.empty((*shape[:-1], N), dtype=self.out_dtype, device=codes.device)
        return _product(a, (codes.contiguous(), scales.contiguous(), 1), shape[:-1].numel(), K, N, bias, out)

    def extra_repr(self):
        return f"in={self.in_features}, out={self.out_features}, bias={self.bias is not None}"
