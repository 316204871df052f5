"""Microscaled 4-bit floating point: matrices of E2M1 codes with block scales
along their rows, and their product on the block-scaled tensor-core kinds.

Two formats:

- ``"mxfp4"`` (the OCP microscaling format): blocks of 32, scales 2^e with
  e = floor(log2(amax)) - 2;
- ``"nvfp4"``: blocks of 16, E4M3 scales amax / (6 g) and one fp32 factor
  g = amax(tensor) / 2688 a tensor.

The reference has no counterpart: its ``float4d`` codes (mxtorch.py:1465-1528)
index a normalised grid under fp32 scales, which no tensor core reads.

    w = fp4_tensor.quantize(weight, "nvfp4")          # [N, K]
    y = fp4_matmul(fp4_tensor.quantize(x, "nvfp4"), w)  # x @ w^T, bf16
    layer = fp4_linear.from_linear(nn_linear, "mxfp4")
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn

from . import _lib as L

FORMATS = {"mxfp4": L.FP4_MX, "nvfp4": L.FP4_NV}
BLOCK = {"mxfp4": 32, "nvfp4": 16}
_IO = {torch.float32: L.F32, torch.bfloat16: L.BF16}


def _fmt(fmt: str) -> int:
    try:
        return FORMATS[fmt]
    except KeyError:
        raise ValueError(f"Unknown 4-bit format {fmt!r}: one of {sorted(FORMATS)}") from None


def _require_cuda(dev: torch.device, what: str) -> None:
    if dev.type != "cuda":
        raise L.MxbError(f"{what}: tensor is on {dev}; the mxb kernels run on CUDA only")


def code_row_bytes(K: int) -> int:
    """Bytes of one row of codes: two a byte, whole groups of 32."""
    return -(-K // 32) * 16


def scale_bytes(rows: int, K: int, fmt: str) -> int:
    """Bytes of the scale tiles (128 rows x 4 blocks, 512 bytes each)."""
    return -(-rows // 128) * -(-(-(-K // BLOCK[fmt])) // 4) * 512


class fp4_tensor:
    """A matrix [..., K] of E2M1 codes; leading dims are rows.

    ``codes``: uint8 [rows, ceil(K / 32) * 16], two codes a byte, low first,
    zero past K.  ``scales``: uint8, tiles of 128 rows x 4 blocks, tiles
    row-major, byte ((r % 32) * 4 + r // 32) * 4 + c of a tile, zero past the
    matrix.  ``global_scale``: fp32 [1] on the device (nvfp4) or None."""

    # _parts: (codes, scales, global_scale), or (buffer, rows, bytes of codes, offset
    # and bytes of scales, offset of the factor or the factor) as quantize made it.
    # Device and addresses are read off the tensors at each call, so that a copied,
    # unpickled or remapped object works on its own memory.
    __slots__ = ("fmt", "shape", "_parts")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, fmt: str, shape,
                 global_scale: Optional[torch.Tensor] = None):
        _fmt(fmt)
        shape = torch.Size(shape)
        if len(shape) < 1:
            raise ValueError("fp4_tensor: shape needs at least one dim")
        rows, K = shape[:-1].numel(), shape[-1]
        if (codes.dtype != torch.uint8 or scales.dtype != torch.uint8
                or codes.numel() != rows * code_row_bytes(K)
                or scales.numel() != scale_bytes(rows, K, fmt)
                or not codes.is_contiguous() or not scales.is_contiguous()):
            raise ValueError(
                f"fp4_tensor {tuple(shape)} {fmt}: codes must be {rows * code_row_bytes(K)} and "
                f"scales {scale_bytes(rows, K, fmt)} contiguous uint8 values")
        if (fmt == "nvfp4") != (global_scale is not None):
            raise ValueError("fp4_tensor: nvfp4 takes a global_scale, mxfp4 none")
        if global_scale is not None and (global_scale.dtype != torch.float32
                                         or global_scale.numel() != 1):
            raise ValueError("fp4_tensor: global_scale must be one fp32 value")
        if codes.device != scales.device or (global_scale is not None
                                             and global_scale.device != codes.device):
            raise ValueError("fp4_tensor: codes, scales and global_scale are on different devices")
        self.fmt, self.shape = fmt, shape
        self._parts = (codes, scales, global_scale)

    @classmethod
    def quantize(cls, x: torch.Tensor, fmt: str = "mxfp4",
                 global_scale: Optional[torch.Tensor] = None) -> "fp4_tensor":
        """Quantize along the last dim (fp32 and bf16 as they are, other types
        through fp32).  ``global_scale`` (nvfp4): a positive fp32 factor to
        use, e.g. a calibrated one; by default from the data.  No gradient."""
        f = _fmt(fmt)
        L.require_cuda(x, "fp4_tensor.quantize")
        if x.dim() < 1:
            raise ValueError("fp4_tensor.quantize: x needs at least one dim")
        io = _IO.get(x.dtype)
        if io is None:
            x, io = x.float(), L.F32
        shape = x.shape
        if len(shape) == 2:
            rows, K = shape
        else:
            rows, K = shape[:-1].numel(), shape[-1]
            x = x.reshape(rows, K)
        ldx = x.stride(0) if rows > 1 else K
        if x.stride(1) != 1 or ldx < K:
            x, ldx = x.contiguous(), K
        dev = x.device
        # one allocation: [codes][scales][factor, workspace]; the views are made
        # when they are asked for
        cb, sb = rows * code_row_bytes(K), scale_bytes(rows, K, fmt)
        at_s = -(-cb // 256) * 256
        at_g = at_s + sb
        derive = wsb = 0
        if f == L.FP4_NV and global_scale is None:
            derive, wsb = 1, L.size("mxb_fp4_quantize_workspace_size", rows, K, f, 1)
        elif f == L.FP4_NV:
            if (global_scale.dtype != torch.float32 or global_scale.numel() != 1
                    or global_scale.device != dev):
                raise ValueError("quantize: global_scale must be one fp32 value on x's device")
        elif global_scale is not None:
            raise ValueError("quantize: mxfp4 takes no global_scale")
        buf = torch.empty(at_g + (16 + wsb if derive else 0), dtype=torch.uint8, device=dev)
        base = buf.data_ptr()
        gp = base + at_g if derive else L.ptr(global_scale)
        if rows * K:
            rc = L.call("mxb_fp4_quantize", dev, x.data_ptr(), io, rows, K, ldx, f, gp, derive, base,
                        base + at_s, base + at_g + 16 if wsb else 0, wsb)
            if rc:
                L.check(rc, f"mxb_fp4_quantize({fmt}, {rows}x{K})")
        elif derive:
            buf[at_g:at_g + 4].view(torch.float32).fill_(1.0)
        self = cls.__new__(cls)
        self.fmt, self.shape = fmt, shape
        self._parts = (buf, rows, cb, at_s, sb, at_g if derive else global_scale)
        return self

    def __copy__(self) -> "fp4_tensor":
        other = type(self).__new__(type(self))
        other.fmt, other.shape, other._parts = self.fmt, self.shape, self._parts
        return other

    def __reduce__(self):
        # the factor in a storage of its own: torch.save takes no storage under two types
        codes, scales, g = self._views()
        return type(self), (codes, scales, self.fmt, tuple(self.shape), None if g is None else g.clone())

    @property
    def device(self) -> torch.device:
        return self._parts[0].device

    def _ptrs(self):
        """Addresses of codes, scales and factor (0: none)."""
        parts = self._parts
        if len(parts) == 3:
            return parts[0].data_ptr(), parts[1].data_ptr(), L.ptr(parts[2])
        buf, _, _, at_s, _, g = parts
        base = buf.data_ptr()
        return base, base + at_s, base + g if isinstance(g, int) else L.ptr(g)

    def _views(self):
        parts = self._parts  # read once: another thread may replace it
        if len(parts) != 3:
            buf, rows, cb, at_s, sb, g = parts
            if isinstance(g, int):
                g = buf[g:g + 4].view(torch.float32)
            parts = self._parts = (buf[:cb].view(rows, -1) if cb else buf[:0].view(rows, 0),
                                   buf[at_s:at_s + sb], g)
        return parts

    @property
    def codes(self) -> torch.Tensor:
        return self._views()[0]

    @property
    def scales(self) -> torch.Tensor:
        return self._views()[1]

    @property
    def global_scale(self) -> Optional[torch.Tensor]:
        return self._views()[2]

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values, fp32 or bf16."""
        io = _IO.get(dtype)
        if io is None:
            raise ValueError(f"dequantize: float32 or bfloat16, not {dtype}")
        dev, shape = self.device, self.shape
        _require_cuda(dev, "fp4_tensor.dequantize")
        rows, K = shape[:-1].numel(), shape[-1]
        out = torch.empty(shape, dtype=dtype, device=dev)
        rc = L.call("mxb_fp4_dequantize", dev, *self._ptrs(), rows, K, FORMATS[self.fmt],
                    out.data_ptr(), io)
        if rc:
            L.check(rc, f"mxb_fp4_dequantize({self.fmt}, {rows}x{K})")
        return out

    def block_scales(self) -> torch.Tensor:
        """The scale bytes in plain order, [rows, ceil(K / block)] (E8M0 or E4M3 bits)."""
        rows, nb = self.shape[:-1].numel(), -(-self.shape[-1] // BLOCK[self.fmt])
        t = self.scales.view(-(-rows // 128), -(-nb // 4), 32, 4, 4).permute(0, 3, 2, 1, 4)
        return t.reshape(-(-rows // 128) * 128, -(-nb // 4) * 4)[:rows, :nb].contiguous()

    @property
    def nbytes(self) -> int:
        return self.codes.nbytes + self.scales.nbytes + (4 if self.global_scale is not None else 0)

    def __repr__(self):
        return f"fp4_tensor({tuple(self.shape)}, {self.fmt}, {self.device})"


def fp4_matmul(a: fp4_tensor, b: fp4_tensor, bias: Optional[torch.Tensor] = None,
               out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """a [..., K] @ b [N, K]^T (+ bias [N]) of two matrices of one format, fp32
    accumulation, rounded once to ``out_dtype`` (bf16 or fp32).  No gradient."""
    if not isinstance(a, fp4_tensor) or not isinstance(b, fp4_tensor):
        raise TypeError("fp4_matmul takes two fp4_tensors")
    if a.fmt != b.fmt:
        raise ValueError(f"fp4_matmul: formats differ ({a.fmt}, {b.fmt})")
    if len(b.shape) != 2 or a.shape[-1] != b.shape[1]:
        raise ValueError(f"fp4_matmul: {tuple(a.shape)} @ {tuple(b.shape)}^T")
    if out_dtype not in _IO:
        raise ValueError(f"fp4_matmul: float32 or bfloat16 out, not {out_dtype}")
    dev = a.device
    _require_cuda(dev, "fp4_matmul")
    if b.device != dev:
        raise ValueError("fp4_matmul: operands on different devices")
    M, K, N = a.shape[:-1].numel(), a.shape[-1], b.shape[0]
    if bias is not None:
        if bias.shape != (N,) or bias.device != dev:
            raise ValueError(f"fp4_matmul: bias must be [{N}] on {dev}")
        if bias.dtype != torch.float32 or not bias.is_contiguous():
            bias = bias.float().contiguous()
    out = torch.empty((M, N) if len(a.shape) == 2 else (*a.shape[:-1], N), dtype=out_dtype, device=dev)
    if K == 0:  # an empty sum
        out.zero_()
        return out if bias is None else out.add_(bias)
    rc = L.call("mxb_fp4_matmul", dev, *a._ptrs(), *b._ptrs(), M, K, N, FORMATS[a.fmt], L.ptr(bias),
                out.data_ptr(), _IO[out_dtype])
    if rc:
        L.check(rc, f"mxb_fp4_matmul({M}x{K}x{N}, {a.fmt})")
    return out


class fp4_linear(nn.Module):
    """nn.Linear with a microscaled 4-bit weight; the activations are quantized
    to the same format on every call.  Inference only (no gradient).  Dtype casts
    of a model leave the codes, the factor and the fp32 bias as they are."""

    def __init__(self, weight: fp4_tensor, bias: Optional[torch.Tensor] = None,
                 out_dtype: torch.dtype = torch.bfloat16):
        super().__init__()
        self.out_features, self.in_features = weight.shape
        self.fmt, self.out_dtype = weight.fmt, out_dtype
        self.register_buffer("weight_codes", weight.codes)
        self.register_buffer("weight_scales", weight.scales)
        # in a storage of its own: torch.save takes no storage under two types
        g = weight.global_scale
        self.register_buffer("weight_global_scale", None if g is None else g.clone())
        self.register_buffer("bias", None if bias is None else bias.detach().float())

    @classmethod
    def from_linear(cls, linear: nn.Linear, fmt: str = "mxfp4",
                    out_dtype: torch.dtype = torch.bfloat16) -> "fp4_linear":
        w = linear.weight.data
        if not w.is_cuda:
            w = w.cuda()
        bias = None if linear.bias is None else linear.bias.data.to(w.device)
        return cls(fp4_tensor.quantize(w, fmt), bias, out_dtype)

    def _apply(self, fn, *args, **kwargs):
        # casts of the whole model (.bfloat16(), .half(), .to(dtype)) move these two but
        # leave them fp32: the factor belongs to the codes bit for bit
        kept = {n: self._buffers[n] for n in ("weight_global_scale", "bias")}
        super()._apply(fn, *args, **kwargs)
        for n, t in kept.items():
            if t is not None and self._buffers[n].dtype != torch.float32:
                self._buffers[n] = t.to(self._buffers[n].device)
        return self

    @property
    def weight(self) -> fp4_tensor:
        return fp4_tensor(self.weight_codes, self.weight_scales, self.fmt,
                          (self.out_features, self.in_features), self.weight_global_scale)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return fp4_matmul(fp4_tensor.quantize(x, self.fmt), self.weight, self.bias, self.out_dtype)

    def extra_repr(self):
        return (f"in={self.in_features}, out={self.out_features}, fmt={self.fmt}, "
                f"bias={self.bias is not None}")
