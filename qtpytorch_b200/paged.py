"""Paged quantized KV cache and attention over it.

``kv_cache_quantizer`` (mxtorch.py:2998-3119) keeps one slot a step for a whole
batch of equal lengths and is read back in fp32.  Here tokens of any sequence go
to any slot of a pool of pages, and attention reads the packed codes:

    cache = paged_kv_cache(n_pages=1024, n_heads=8, head_dim=128, dtype="int8d")
    cache.write(k, v, slots)                       # k, v [T, 8, 128]
    out = paged_attention(q, cache, table, lengths)  # q [B, T, Hq, 128] bf16
    out = paged_attention(q, cache, table, lengths, prefix_table=pages, prefix_len=5000)
    q = cache.append(k, v, slots, positions, inv_freq, q=q)  # rotated on the way
    out = paged_attention(q, cache, table, lengths, tree_mask=mask)  # a tree of drafts

A token's slot is page number * page_size + offset; ``table`` [B, width] holds
the page numbers of each sequence, ``lengths`` [B] its tokens.  A head row's codes
and scale are those of ``mx_tensor.quantize(row, dtype, head_dim)``.
"""
from __future__ import annotations

import ctypes
import functools
import math
from typing import Optional, Sequence, Tuple, Union

import torch

from . import _lib as L
from .dtypes import get_mx_dtype, mx_dtype
from .tensor import plain

_IO = {torch.float32: L.F32, torch.bfloat16: L.BF16}


def _cache_dtype(dtype: Union[str, mx_dtype]) -> mx_dtype:
    dt = get_mx_dtype(dtype)
    if not (dt.is_int and dt.variant == "" and dt.bits in (4, 8)):
        raise NotImplementedError(f"paged_kv_cache covers base int4 and int8 dtypes, not {dt.name}")
    return dt


class paged_kv_cache:
    """A pool of pages of quantized keys and values.

    ``k_codes`` / ``v_codes`` uint8 [n_pages, n_heads, page_size, head_dim * bits / 8],
    ``k_scales`` / ``v_scales`` fp32 [n_pages, n_heads, page_size].  head_dim 64 or
    128, page_size a power of two from 16 to 1024."""

    def __init__(self, n_pages: int, n_heads: int, head_dim: int,
                 dtype: Union[str, mx_dtype] = "int8d", page_size: int = 64, device="cuda"):
        dt = _cache_dtype(dtype)
        shape = (n_pages, n_heads, page_size)
        codes = [torch.zeros(*shape, head_dim * dt.bits // 8, dtype=torch.uint8, device=device)
                 for _ in range(2)]
        scales = [torch.zeros(shape, dtype=torch.float32, device=device) for _ in range(2)]
        self._bind(codes[0], scales[0], codes[1], scales[1], dt)

    @classmethod
    def from_buffers(cls, k_codes: torch.Tensor, k_scales: torch.Tensor, v_codes: torch.Tensor,
                     v_scales: torch.Tensor, dtype: Union[str, mx_dtype] = "int8d") -> "paged_kv_cache":
        """A cache over buffers that the caller owns (no copy)."""
        self = cls.__new__(cls)
        self._bind(k_codes, k_scales, v_codes, v_scales, _cache_dtype(dtype))
        return self

    def _bind(self, kc, ks, vc, vs, dt: mx_dtype) -> None:
        if kc.dim() != 4 or kc.shape != vc.shape or kc.shape[:3] != ks.shape or ks.shape != vs.shape:
            raise ValueError("paged_kv_cache: codes [pages, heads, page, bytes] and scales "
                             "[pages, heads, page] of K and V must agree")
        if (kc.dtype != torch.uint8 or vc.dtype != torch.uint8 or ks.dtype != torch.float32
                or vs.dtype != torch.float32):
            raise ValueError("paged_kv_cache: codes are uint8, scales fp32")
        if not kc.device == ks.device == vc.device == vs.device:
            raise ValueError("paged_kv_cache: buffers are on different devices")
        if not (kc.is_contiguous() and vc.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()):
            raise ValueError("paged_kv_cache: buffers must be contiguous")
        n_pages, heads, page, row = kc.shape
        dim = row * 8 // dt.bits
        if dim not in (64, 128):
            raise NotImplementedError(f"paged_kv_cache: head_dim 64 or 128, not {dim}")
        if page < 16 or page > 1024 or page & (page - 1):
            raise ValueError(f"paged_kv_cache: page_size must be a power of two from 16 to 1024, not {page}")
        if n_pages < 1 or heads < 1 or n_pages * heads * page >= 2 ** 31:
            raise ValueError("paged_kv_cache: needs pages and heads, fewer than 2^31 head rows")
        self._buffers = (kc, ks, vc, vs)
        self.dtype, self.n_pages, self.n_heads = dt, n_pages, heads
        self.page_size, self.head_dim = page, dim

    # The buffers are checked once, so they are not replaced; device and
    # addresses are read off them at each call, so that a copied, unpickled or
    # remapped cache works on its own memory.
    k_codes = property(lambda self: self._buffers[0])
    k_scales = property(lambda self: self._buffers[1])
    v_codes = property(lambda self: self._buffers[2])
    v_scales = property(lambda self: self._buffers[3])
    device = property(lambda self: self._buffers[0].device)

    def _pool(self):
        kc, ks, vc, vs = self._buffers
        return kc.data_ptr(), ks.data_ptr(), vc.data_ptr(), vs.data_ptr()

    def _cuda(self, what: str) -> torch.device:
        L.require_cuda(self.k_codes, what)
        return self.device

    def write(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """Quantize k, v [T, n_heads, head_dim] (fp32 or bf16, any token and
        head strides) into ``slots`` [T]; a negative slot skips its token.
        The slots of one call must be distinct."""
        dev = self._cuda("paged_kv_cache.write")
        k, v = plain(k), plain(v)
        H, D = self.n_heads, self.head_dim
        if k.dim() != 3 or k.shape != v.shape or k.shape[1:] != (H, D) or slots.shape != k.shape[:1]:
            raise ValueError(f"write: k and v must be [T, {H}, {D}] and slots [T]; got "
                             f"{tuple(k.shape)}, {tuple(v.shape)}, {tuple(slots.shape)}")
        if k.device != dev or v.device != dev or slots.device != dev:
            raise ValueError(f"write: k, v and slots must be on {dev}")
        if k.dtype != v.dtype or k.dtype not in _IO:
            k, v = k.float(), v.float()
        if k.stride(2) != 1:
            k = k.contiguous()
        if v.stride(2) != 1:
            v = v.contiguous()
        if slots.dtype != torch.int64 or not slots.is_contiguous():
            slots = slots.to(torch.int64).contiguous()
        rc = L.call("mxb_kv_write", dev, k.data_ptr(), v.data_ptr(), _IO[k.dtype], k.shape[0], H, D,
                    k.stride(0), k.stride(1), v.stride(0), v.stride(1), slots.data_ptr(),
                    self.n_pages, self.page_size, self.dtype.bits, *self._pool())
        if rc:
            L.check(rc, f"mxb_kv_write({self.dtype.name}, T={k.shape[0]})")

    def append(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, positions: torch.Tensor,
               inv_freq: torch.Tensor, q: Optional[torch.Tensor] = None,
               sections: Optional[Sequence[int]] = None, interleaved: bool = False) -> Optional[torch.Tensor]:
        """``write`` of keys rotated by their positions; ``q`` [T, heads of queries,
        head_dim] is rotated beside them and returned (contiguous, in its type).

        Pair i of a head row turns by ``positions[t] * inv_freq[i]`` (inv_freq fp32
        [pairs], pairs a multiple of 4, at most head_dim / 2): elements (i, i +
        pairs), or (2 i, 2 i + 1) where ``interleaved``; the others stay.  With
        ``sections`` (pairs of each axis, up to four, in order) positions are
        [axes, T], one row an axis.  Angles are found in 64 bits; a key's codes and
        scale are those of its rotation in 64 bits rounded to fp32.  The queries of
        skipped tokens are rotated too.  Slots of one call must be distinct.  No
        gradient."""
        dev = self._cuda("paged_kv_cache.append")
        k, v, q, inv_freq = plain(k), plain(v), plain(q), plain(inv_freq)
        H, D = self.n_heads, self.head_dim
        if k.dim() != 3 or k.shape != v.shape or k.shape[1:] != (H, D) or slots.shape != k.shape[:1]:
            raise ValueError(f"append: k and v must be [T, {H}, {D}] and slots [T]; got "
                             f"{tuple(k.shape)}, {tuple(v.shape)}, {tuple(slots.shape)}")
        T = k.shape[0]
        if q is not None and (q.dim() != 3 or q.shape[0] != T or q.shape[2] != D):
            raise ValueError(f"append: q must be [{T}, heads, {D}], got {tuple(q.shape)}")
        pairs = inv_freq.shape[0] if inv_freq.dim() == 1 else -1
        if pairs < 0 or pairs % 4 or pairs > D // 2 or not inv_freq.is_floating_point():
            raise ValueError(f"append: inv_freq must hold a multiple of 4 of at most {D // 2} frequencies, "
                             f"got {inv_freq.dtype} {tuple(inv_freq.shape)}")
        axes, c_sections = 1, None
        if sections is not None:
            sections = tuple(int(x) for x in sections)
            axes = len(sections)
            if not 1 <= axes <= 4 or min(sections) < 0 or sum(sections) != pairs:
                raise ValueError(f"append: sections must be one to four counts that add up to {pairs} pairs, "
                                 f"not {sections}")
            c_sections = _ints(sections)
        want = (T,) if sections is None else (axes, T)
        if positions.shape != want or positions.is_floating_point() or slots.is_floating_point():
            raise ValueError(f"append: positions must be integers {list(want)}, got {positions.dtype} "
                             f"{tuple(positions.shape)}")
        for t in (k, v, slots, positions, inv_freq) if q is None else (k, v, slots, positions, inv_freq, q):
            if t.device != dev:
                raise ValueError(f"append: tensors must be on {dev}")
        q_type = None if q is None else q.dtype
        if k.dtype not in _IO or k.dtype != v.dtype or (q is not None and q_type != k.dtype):
            k, v, q = k.float(), v.float(), None if q is None else q.float()
        k, v = _rows(k), _rows(v)
        if q is not None:
            q = _rows(q)
        if slots.dtype != torch.int64 or not slots.is_contiguous():
            slots = slots.to(torch.int64).contiguous()
        if positions.dtype != torch.int64 or (T > 1 and positions.stride(-1) != 1):
            positions = positions.to(torch.int64).contiguous()
        if inv_freq.dtype != torch.float32 or not inv_freq.is_contiguous():
            inv_freq = inv_freq.float().contiguous()
        out = None if q is None else torch.empty(q.shape, dtype=q.dtype, device=dev)
        Hq = 0 if q is None else q.shape[1]
        rc = L.call("mxb_kv_append", dev, L.ptr(q), k.data_ptr(), v.data_ptr(), _IO[k.dtype], T, Hq, H, D,
                    0 if q is None else q.stride(0), 0 if q is None else q.stride(1), k.stride(0), k.stride(1),
                    v.stride(0), v.stride(1), positions.data_ptr(), axes,
                    positions.stride(0) if axes > 1 else 0, inv_freq.data_ptr(), 2 * pairs, c_sections,
                    int(interleaved), slots.data_ptr(), self.n_pages, self.page_size, self.dtype.bits,
                    *self._pool(), L.ptr(out))
        if rc:
            L.check(rc, f"mxb_kv_append({self.dtype.name}, T={T}, heads={Hq}+{H})")
        return out if out is None or out.dtype == q_type else out.to(q_type)

    def read(self, table: torch.Tensor, lengths: torch.Tensor, max_len: int,
             dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
        """(k, v) [B, max_len, n_heads, head_dim] of the sequences' histories,
        fp32 or bf16; zero from each sequence's length on."""
        dev = self._cuda("paged_kv_cache.read")
        if dtype not in _IO:
            raise ValueError(f"read: float32 or bfloat16, not {dtype}")
        table, lengths = _tables(table, lengths, dev, "read")
        if max_len < 0:
            raise ValueError("read: max_len must not be negative")
        B = table.shape[0]
        k, v = torch.empty((2, B, max_len, self.n_heads, self.head_dim), dtype=dtype, device=dev).unbind()
        rc = L.call("mxb_kv_read", dev, *self._pool(), self.n_pages, self.n_heads, self.page_size,
                    self.head_dim, self.dtype.bits, table.data_ptr(), table.shape[1],
                    lengths.data_ptr(), B, max_len, k.data_ptr(), v.data_ptr(), _IO[dtype])
        if rc:
            L.check(rc, f"mxb_kv_read({self.dtype.name}, B={B}, max_len={max_len})")
        return k, v

    @property
    def nbytes(self) -> int:
        return (self.k_codes.nbytes + self.k_scales.nbytes + self.v_codes.nbytes
                + self.v_scales.nbytes)

    def __repr__(self):
        return (f"paged_kv_cache(pages={self.n_pages}, heads={self.n_heads}, dim={self.head_dim}, "
                f"page={self.page_size}, dtype={self.dtype.name})")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """[T, heads, dim] with adjacent elements and strides that 31 bits hold."""
    a, b, c = t.stride()
    return t if c == 1 and a < 2 ** 31 and b < 2 ** 31 else t.contiguous()


@functools.lru_cache(maxsize=256)
def _ints(values: Tuple[int, ...]):
    return (ctypes.c_int * len(values))(*values)


def _int32(t: torch.Tensor) -> torch.Tensor:
    """Contiguous int32 on the device; 64-bit values saturate, so that what lies
    outside every pool or table stays outside."""
    if not t.is_contiguous():
        t = t.contiguous()
    if t.dtype == torch.int32:
        return t
    if t.dtype != torch.int64:
        return t.to(torch.int32)
    out = torch.empty_like(t, dtype=torch.int32)
    rc = L.call("mxb_narrow_i64", t.device, t.data_ptr(), t.numel(), out.data_ptr())
    if rc:
        L.check(rc, f"mxb_narrow_i64({t.numel()})")
    return out


def _tables(table: torch.Tensor, lengths: torch.Tensor, dev, what: str):
    if table.dim() != 2 or lengths.shape != table.shape[:1]:
        raise ValueError(f"{what}: table must be [B, width] and lengths [B]")
    if table.device != dev or lengths.device != dev:
        raise ValueError(f"{what}: table and lengths must be on {dev}")
    if table.is_floating_point() or lengths.is_floating_point():
        raise ValueError(f"{what}: table and lengths hold integers")
    return _int32(table), _int32(lengths)


def paged_attention(q: torch.Tensor, cache: paged_kv_cache, table: torch.Tensor,
                    lengths: torch.Tensor, prefix_table: Optional[torch.Tensor] = None,
                    prefix_len: int = 0, scale: Optional[float] = None, return_lse: bool = False,
                    tree_mask: Optional[torch.Tensor] = None):
    """softmax(scale * q k^T) v over a paged quantized cache.

    q [B, T, Hq, head_dim] bf16, Hq a multiple of the cache's heads (query head i
    reads KV head i // (Hq / n_heads)).  ``lengths[b]`` counts sequence b's keys,
    its T newest tokens included: query t sees the keys before
    lengths[b] - (T - 1 - t).  ``prefix_table`` [pages] and ``prefix_len`` name
    keys that every query sees in front of its own; they are read once for the
    whole batch.  ``tree_mask`` [T, T] or [B, T, T] bool: the T newest tokens are a
    tree of drafts; query t sees all keys before them and of them those that row t
    names (its own among them, if it is to be seen).  ``scale`` defaults to 1 / sqrt(head_dim).  A row without keys
    gives zeros; a page number outside the pool holds no keys (recorded in the
    library's device error word).  Returns out (q's shape, bf16), with ``return_lse`` also the fp32
    log-sum-exp [B, T, Hq] of the scaled scores.  No gradient."""
    dev = cache._cuda("paged_attention")
    H, D = cache.n_heads, cache.head_dim
    if q.dim() != 4 or q.shape[3] != D or q.shape[2] % H or q.shape[2] == 0:
        raise ValueError(f"paged_attention: q must be [B, T, a multiple of {H} heads, {D}], "
                         f"got {tuple(q.shape)}")
    if q.dtype != torch.bfloat16:
        raise NotImplementedError(f"paged_attention takes bf16 queries, not {q.dtype}")
    if q.device != dev:
        raise ValueError(f"paged_attention: q must be on {dev}")
    table, lengths = _tables(table, lengths, dev, "paged_attention")
    B, T, Hq, _ = q.shape
    if table.shape[0] != B:
        raise ValueError(f"paged_attention: table has {table.shape[0]} rows for {B} sequences")
    if prefix_len < 0:
        raise ValueError("paged_attention: prefix_len must not be negative")
    width = 0
    if prefix_len > 0:
        if prefix_table is None or prefix_table.dim() != 1 or prefix_table.is_floating_point():
            raise ValueError("paged_attention: prefix_len needs a prefix_table [pages] of integers")
        if prefix_table.device != dev:
            raise ValueError(f"paged_attention: prefix_table must be on {dev}")
        width = prefix_table.shape[0]
        if prefix_len > width * cache.page_size:
            raise ValueError(f"paged_attention: prefix_len {prefix_len} needs more than the "
                             f"{width} pages of prefix_table")
        prefix_table = _int32(prefix_table)
    if tree_mask is not None:
        if tree_mask.dtype != torch.bool or tree_mask.shape not in ((T, T), (B, T, T)):
            raise ValueError(f"paged_attention: tree_mask must be bool [{T}, {T}] or [{B}, {T}, {T}], got "
                             f"{tree_mask.dtype} {tuple(tree_mask.shape)}")
        if tree_mask.device != dev:
            raise ValueError(f"paged_attention: tree_mask must be on {dev}")
        if tree_mask.stride(-1) != 1:
            tree_mask = tree_mask.contiguous()
    q = q.contiguous()
    if q.data_ptr() % 16:
        q = q.clone()
    out = torch.empty_like(q)
    lse = torch.empty(B, T, Hq, dtype=torch.float32, device=dev) if return_lse else None
    op = "mxb_paged_attention" if tree_mask is None else "mxb_tree_attention"
    tree = () if tree_mask is None else (tree_mask.data_ptr(), tree_mask.stride(0) if tree_mask.dim() == 3 else 0,
                                         tree_mask.stride(-2))
    wsb = L.size(op + "_workspace_size", B, T, H, Hq // H, D, cache.dtype.bits, cache.page_size,
                 table.shape[1], prefix_len)
    ws = L.workspace(wsb, dev)
    rc = L.call(op, dev, q.data_ptr(), B, T, H, Hq // H, D,
                *cache._pool(), cache.n_pages, cache.page_size, cache.dtype.bits,
                table.data_ptr(), table.shape[1], lengths.data_ptr(),
                prefix_table.data_ptr() if prefix_len else 0, width, prefix_len, *tree,
                1.0 / math.sqrt(D) if scale is None else float(scale), out.data_ptr(), L.ptr(lse),
                L.ptr(ws), wsb)
    if rc:
        L.check(rc, f"{op}(B={B}, T={T}, heads={H}x{Hq // H}, dim={D})")
    return (out, lse) if return_lse else out
