"""Paged quantized KV cache and attention over it, against 64 bits: ragged
batches, pages in any order, a shared prefix, rows without keys, hidden places
that hold NaN, strides, offsets past 32 bits; refusals.

The cache's codes and scales are those of ``mx_tensor.quantize`` with block =
head_dim (mxtorch.py:1426-1463); attention has no counterpart in the reference.
"""
import copy
import ctypes
import io
import math
import os
import pickle
import sys

import numpy as np
import pytest
import torch

import qtpytorch_b200 as mxb
from oracle import mx_oracle as O
from qtpytorch_b200 import _lib as L

CODE = {"int8d": 127.0, "int4d": 7.0}


# ── host ─────────────────────────────────────────────────────────────────────
def test_argument_errors_need_no_gpu():
    lib = L.load()
    p = ctypes.c_void_p(32)

    def write(T=2, heads=2, dim=128, pages=4, page=16, bits=8, dt=1, k=p, kc=p):
        return lib.mxb_kv_write(k, p, dt, T, heads, dim, 256, 128, 256, 128, p, pages, page, bits, kc, p, p,
                                p, None)

    assert write(bits=2) == -2 and write(dt=7) == -2
    assert write(dim=96) == -1 and write(page=24) == -1 and write(page=8) == -1 and write(page=2048) == -1
    assert write(pages=0) == -1 and write(heads=0) == -1 and write(T=-1) == -1
    assert write(pages=1 << 27, page=16) == -1  # 2^32 head rows
    assert write(k=None) == -6 and write(kc=None) == -6 and write(kc=ctypes.c_void_p(8)) == -3
    assert write(T=0) == 0

    def read(B=2, width=3, max_len=5, out=1, ko=p):
        return lib.mxb_kv_read(p, p, p, p, 4, 2, 16, 128, 8, p, width, p, B, max_len, ko, p, out, None)

    assert read(out=5) == -2 and read(B=-1) == -1 and read(B=1 << 16) == -1 and read(max_len=-1) == -1
    assert read(ko=None) == -6 and read(ko=ctypes.c_void_p(8)) == -3
    assert read(B=0) == 0 and read(max_len=0) == 0

    def attend(B=2, T=1, group=4, width=3, prefix=0, pw=0, q=p, pt=None, ws=None, n=0):
        return lib.mxb_paged_attention(q, B, T, 2, group, 128, p, p, p, p, 4, 16, 8, p, width, p, pt, pw,
                                       prefix, 0.1, p, None, ws, n, None)

    assert attend(B=-1) == -1 and attend(group=0) == -1 and attend(T=1 << 17) == -1
    assert attend(width=1 << 30) == -1
    assert attend(prefix=17, pw=1, pt=p) == -1 and attend(prefix=-1) == -1
    assert attend(q=None) == -6 and attend(prefix=16, pw=1) == -6 and attend(q=ctypes.c_void_p(8)) == -3
    need = lib.mxb_paged_attention_workspace_size(2, 1, 2, 4, 128, 8, 16, 1000, 0)
    assert need > 0 and attend(width=1000) == -7 and attend(width=1000, ws=p, n=need - 1) == -7
    assert lib.mxb_paged_attention_workspace_size(2, 1, 2, 4, 128, 8, 16, 3, 0) == 0  # short: one launch
    assert attend(B=0) == 0 and attend(T=0) == 0


def test_misaligned_pointers_are_refused():
    lib, p = L.load(), ctypes.c_void_p(32)
    need = lib.mxb_paged_attention_workspace_size(2, 1, 2, 4, 128, 8, 16, 1000, 0)

    def attend(ws):
        return lib.mxb_paged_attention(p, 2, 1, 2, 4, 128, p, p, p, p, 4, 16, 8, p, 1000, p, None, 0, 0, 0.1, p,
                                       None, ctypes.c_void_p(ws), need - 1, None)

    assert attend(48) == -3 and attend(64) == -7  # parts are stored 32 bytes at a time

    def write(k, v, dt):
        return lib.mxb_kv_write(ctypes.c_void_p(k), ctypes.c_void_p(v), dt, 2, 2, 128, 256, 128, 256, 128, p, 4, 16,
                                8, p, p, p, p, None)

    assert write(34, 32, 0) == -3 and write(32, 33, 1) == -3


def test_more_prefix_rows_than_a_grid_holds_are_refused():
    lib, p = L.load(), ctypes.c_void_p(32)

    def attend(B, prefix):
        return lib.mxb_paged_attention(p, B, 1, 2, 1024, 128, p, p, p, p, 4, 16, 8, p, 3, p, p, 1, prefix, 0.1, p,
                                       None, None, 0, None)

    assert attend(65535, 16) == -1            # 262140 groups of 256 rows a KV head
    assert attend(16383, 16) == -7            # 65532: the workspace is looked at next


def test_refusals():
    with pytest.raises(NotImplementedError):
        mxb.paged_kv_cache(4, 2, 128, "int2d", device="cpu")
    with pytest.raises(NotImplementedError):
        mxb.paged_kv_cache(4, 2, 128, "int8dh", device="cpu")
    with pytest.raises(NotImplementedError):
        mxb.paged_kv_cache(4, 2, 96, device="cpu")
    with pytest.raises(ValueError):
        mxb.paged_kv_cache(4, 2, 128, page_size=48, device="cpu")
    c = mxb.paged_kv_cache(4, 2, 64, "int4d", 16, device="cpu")
    assert c.k_codes.shape == (4, 2, 16, 32) and c.nbytes == 2 * (4 * 2 * 16 * 36)
    with pytest.raises(ValueError):
        mxb.paged_kv_cache.from_buffers(c.k_codes, c.k_scales[:3], c.v_codes, c.v_scales, "int4d")
    with pytest.raises(ValueError):
        mxb.paged_kv_cache.from_buffers(c.k_codes.int(), c.k_scales, c.v_codes, c.v_scales, "int4d")
    with pytest.raises(L.MxbError):
        c.write(torch.zeros(1, 2, 64), torch.zeros(1, 2, 64), torch.zeros(1, dtype=torch.long))
    with pytest.raises(L.MxbError):
        c.read(torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), 4)
    with pytest.raises(L.MxbError):
        mxb.paged_attention(torch.zeros(1, 1, 2, 64), c, torch.zeros(1, 1), torch.zeros(1))


def test_copies_own_their_addresses():
    """A copied, pickled or saved cache hands the kernels its own memory, on the
    device that this memory is on."""
    c = mxb.paged_kv_cache(4, 2, 64, "int4d", 16, device="cpu")
    c.k_codes.random_(0, 256)
    buf = io.BytesIO()
    torch.save(c, buf)
    buf.seek(0)

    def addresses(x):
        return tuple(t.data_ptr() for t in (x.k_codes, x.k_scales, x.v_codes, x.v_scales))

    for d in (copy.deepcopy(c), pickle.loads(pickle.dumps(c)), torch.load(buf, weights_only=False)):
        assert d._pool() == addresses(d) and not set(d._pool()) & set(c._pool())
        assert torch.equal(d.k_codes, c.k_codes) and d.page_size == 16 and d.dtype.bits == 4
    assert c._pool() == addresses(c) == copy.copy(c)._pool()
    buf.seek(0)
    assert torch.load(buf, map_location="meta", weights_only=False).device.type == "meta"
    with pytest.raises(AttributeError):
        c.k_codes = c.k_codes[:1]  # a smaller pool behind the geometry that was checked


@pytest.mark.gpu
def test_refusals_on_the_device():
    c = mxb.paged_kv_cache(4, 2, 64, "int8d", 16)
    z = torch.zeros(3, 2, 64, device="cuda")
    s = torch.zeros(3, dtype=torch.long, device="cuda")
    t, n = torch.zeros(1, 2, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    q = torch.zeros(1, 1, 4, 64, device="cuda", dtype=torch.bfloat16)
    for k, v, at in ((z, z[:2], s), (z, z, s[:2]), (z[..., :32], z[..., :32], s), (z, z, s.cpu())):
        with pytest.raises(ValueError):
            c.write(k, v, at)
    for a in ((t, n, -1), (t[0], n, 4), (t, n.float(), 4), (t.cpu(), n, 4)):
        with pytest.raises(ValueError):
            c.read(*a)
    with pytest.raises(ValueError):
        c.read(t, n, 4, torch.float16)
    with pytest.raises(NotImplementedError):
        mxb.paged_attention(q.float(), c, t, n)
    for kw in (dict(q=q[..., :3, :]), dict(q=q[0]), dict(table=t[:, :1].repeat(2, 1)), dict(lengths=n.cpu()),
               dict(prefix_len=5), dict(prefix_len=-1), dict(prefix_len=33, prefix_table=t[0])):
        a = dict(q=q, cache=c, table=t, lengths=n)
        a.update(kw)
        with pytest.raises(ValueError):
            mxb.paged_attention(**a)


# ── write and read ───────────────────────────────────────────────────────────
def pool(pages, heads, dim, dtype, page, seed):
    """A cache as an earlier run left it: any codes, positive scales."""
    g = torch.Generator("cuda").manual_seed(seed)
    c = mxb.paged_kv_cache(pages, heads, dim, dtype, page)
    for codes, scales in ((c.k_codes, c.k_scales), (c.v_codes, c.v_scales)):
        codes.random_(0, 256, generator=g)
        scales.copy_(torch.rand(scales.shape, generator=g, device="cuda") * 0.02 + 0.005)
    return c


def values(c, which):
    """fp64 [pages, heads, page, dim] of a cache's keys or values."""
    codes, scales = (c.k_codes, c.k_scales) if which == "k" else (c.v_codes, c.v_scales)
    if c.dtype.bits == 8:
        x = codes.view(torch.int8).double()
    else:
        x = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).to(torch.int16)
        x = torch.where(x > 7, x - 16, x).double()
    return x * scales.double()[..., None]


def history(c, which, pages, n):
    """fp64 [heads, n, dim] of the first n tokens behind a list of pages."""
    v = values(c, which)[pages.long()]
    return v.transpose(0, 1).flatten(1, 2)[:, :n]


def tables(lengths, page, pages, seed):
    wide = max(1, -(-max(lengths, default=1) // page))
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    assert len(lengths) * wide <= pages
    return order[:len(lengths) * wide].view(len(lengths), wide).cuda(), order[len(lengths) * wide:].cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["int8d", "int4d"])
@pytest.mark.parametrize("dim,page,heads,T", [(64, 16, 1, 1), (128, 64, 8, 5), (64, 128, 3, 200), (128, 16, 5, 67)])
@pytest.mark.parametrize("inp", [torch.float32, torch.bfloat16])
def test_write_matches_the_quantizer(dtype, dim, page, heads, T, inp):
    g = torch.Generator().manual_seed(T)
    k, v = torch.randn(T, heads, dim, generator=g), torch.randn(T, heads, dim, generator=g) * 50
    k[0, 0] = 0.0
    k, v = k.to(inp), v.to(inp)
    c = pool(2 * -(-T // page) + 1, heads, dim, dtype, page, 1)
    before = [t.clone() for t in (c.k_codes, c.k_scales, c.v_codes, c.v_scales)]
    slots = torch.randperm(c.n_pages * page, generator=g)[:T]
    slots[T // 2] = -1  # padding
    c.write(k.cuda(), v.cuda(), slots.cuda())
    keep = slots >= 0
    pg, off = slots[keep] // page, slots[keep] % page
    bits = c.dtype.bits
    for x, codes, scales, c0, s0 in ((k, c.k_codes, c.k_scales, before[0], before[1]),
                                     (v, c.v_codes, c.v_scales, before[2], before[3])):
        packed, sc, _ = O.quantize(x.float().numpy().reshape(-1, dim), bits, "int", dim)
        want_c, want_s = c0.cpu(), s0.cpu()
        want_c[pg, :, off] = torch.from_numpy(packed.view(np.uint8)).view(T, heads, -1)[keep]
        want_s[pg, :, off] = torch.from_numpy(sc).view(T, heads)[keep]
        assert torch.equal(codes.cpu(), want_c) and torch.equal(scales.cpu(), want_s)


@pytest.mark.gpu
def test_write_strides_types_and_bad_slots():
    c, d = (mxb.paged_kv_cache(4, 2, 64, "int8d", 16) for _ in range(2))
    qkv = torch.randn(10, 8, 64, generator=torch.Generator().manual_seed(0)).cuda().bfloat16()
    slots = torch.arange(3, 13, device="cuda")
    c.write(qkv[:, 4:6], qkv[:, 6:8], slots)  # slices of one projection
    d.write(qkv[:, 4:6].contiguous(), qkv[:, 6:8].transpose(0, 1).contiguous().transpose(0, 1), slots.int())
    assert torch.equal(c.k_codes, d.k_codes) and torch.equal(c.v_scales, d.v_scales)
    d.write(qkv[:, 4:6].half(), qkv[:, 6:8].half(), slots)
    assert torch.equal(c.v_codes, d.v_codes)
    d.write(qkv[:, 4:6], qkv[:, 6:8].float(), slots)  # mixed types go through fp32
    assert torch.equal(c.k_codes, d.k_codes) and torch.equal(c.v_codes, d.v_codes)
    L.load().mxb_device_error(1)
    before = c.k_codes.clone()
    c.write(qkv[:2, :2], qkv[:2, :2], torch.tensor([64, -5], device="cuda"))  # past the pool; skipped
    assert torch.equal(c.k_codes, before)
    assert L.load().mxb_device_error(1) == 8
    c.write(qkv[:0, :2], qkv[:0, :2], slots[:0])
    assert L.load().mxb_device_error(1) == 0


@pytest.mark.gpu
def test_write_infinity_and_nan_rows():
    c = mxb.paged_kv_cache(1, 1, 64, "int4d", 16)
    k = torch.randn(3, 1, 64, generator=torch.Generator().manual_seed(4)).cuda()
    k[0, 0, 5], k[1, 0, 7] = float("inf"), float("nan")
    c.write(k, k, torch.arange(3, device="cuda"))
    out, _ = c.read(torch.zeros(1, 1, dtype=torch.int32, device="cuda"),
                    torch.tensor([3], device="cuda"), 3, torch.float32)
    assert out[0, 0].isnan().all() and out[0, 1].isnan().all() and out[0, 2].isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["int8d", "int4d"])
@pytest.mark.parametrize("dim,page,heads,lengths,max_len", [
    (128, 16, 8, [1, 0, 40, 33], 40), (64, 64, 3, [130, 64, 65], 131), (128, 32, 1, [7], 3), (64, 16, 2, [0, 0], 5)])
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
def test_read(dtype, dim, page, heads, lengths, max_len, out):
    c = pool(40, heads, dim, dtype, page, 2)
    table, _ = tables(lengths, page, 40, 3)
    k, v = c.read(table, torch.tensor(lengths, device="cuda"), max_len, out)
    for got, which in ((k, "k"), (v, "v")):
        want = torch.zeros(len(lengths), max_len, heads, dim, dtype=torch.float32, device="cuda")
        for b, n in enumerate(lengths):
            n = min(n, max_len)
            want[b, :n] = history(c, which, table[b], n).transpose(0, 1).float()
        assert torch.equal(got, want.to(out))


@pytest.mark.gpu
def test_read_bad_pages_read_as_zero():
    c = pool(4, 2, 64, "int8d", 16, 5)
    L.load().mxb_device_error(1)
    table = torch.tensor([[0, 9], [-1, 1]], device="cuda")
    k, _ = c.read(table, torch.tensor([32, 40], device="cuda"), 48, torch.float32)
    assert L.load().mxb_device_error(1) == 8
    assert torch.equal(k[0, :16], history(c, "k", table[0, :1], 16).transpose(0, 1).float())
    assert not k[0, 16:].any() and not k[1, :16].any() and not k[1, 32:].any()


@pytest.mark.gpu
def test_read_through_tables_without_pages():
    """A batch whose sequences have no pages yet reads as zeros, as attention takes it."""
    c = pool(2, 2, 64, "int4d", 16, 5)
    L.load().mxb_device_error(1)
    for table in (torch.zeros(3, 0, dtype=torch.int32, device="cuda"), torch.zeros(3, 0, device="cuda").long()):
        for x in c.read(table, torch.zeros(3, dtype=torch.int32, device="cuda"), 4):
            assert x.shape == (3, 4, 2, 64) and not x.any()
        assert L.load().mxb_device_error(1) == 0
        c.read(table, torch.ones(3, dtype=torch.int32, device="cuda"), 4)
        assert L.load().mxb_device_error(1) == 8


# ── attention ────────────────────────────────────────────────────────────────
def attend64(q, c, table, lengths, prefix, prefix_len, scale):
    """(out, lse) in 64 bits, with sum_j p_j |v_j| for the tolerance."""
    B, T, Hq, D = q.shape
    H = c.n_heads
    q = q.double().view(B, T, H, Hq // H, D)
    out, mag = torch.zeros_like(q), torch.zeros_like(q)
    lse = torch.full(q.shape[:-1], float("-inf"), dtype=torch.float64, device=q.device)
    for b in range(B):
        n = lengths[b]
        ks, vs = (history(c, w, table[b], n) for w in "kv")
        if prefix_len:
            ks, vs = (torch.cat((history(c, w, prefix, prefix_len), x), 1) for w, x in (("k", ks), ("v", vs)))
        for t in range(T):
            live = prefix_len + max(0, n - (T - 1 - t))
            if live:
                s = torch.einsum("hgd,hld->hgl", q[b, t], ks[:, :live]) * scale
                p = torch.softmax(s, -1)
                out[b, t] = torch.einsum("hgl,hld->hgd", p, vs[:, :live])
                mag[b, t] = torch.einsum("hgl,hld->hgd", p, vs[:, :live].abs())
                lse[b, t] = torch.logsumexp(s, -1)
    return out.view(B, T, Hq, D), lse.view(B, T, Hq), mag.view(B, T, Hq, D)


def check_attention(got, lse, q, c, table, lengths, prefix, prefix_len, scale=None):
    """Tolerances, from the roundings:
    - a score: at most D / 16 + 4 fp32 additions (2^-23 each where the hardware
      truncates) of terms that sum to (offset + code) sum|q|, offset 1152 (int8)
      or 136 (int4), times the key's scale; e_s in units of log2;
    - a weight: fp16, 2^-11, and twice exp2 of a score that is e_s off (in the sum
      and in the product), each at most 2 e_s for e_s < 1 / 2, and 2^-20 of the
      exponentials and their sums;
    - weights under fp16's normal range: 2^-24 of the largest value each;
    - the output: bf16, 2^-8 (half an ulp is 2^-9, of a value that is itself off)."""
    D = q.shape[-1]
    scale = 1 / math.sqrt(D) if scale is None else scale
    out64, lse64, mag = attend64(q, c, table, lengths, prefix, prefix_len, scale)
    off, top = (1152, 127) if c.dtype.bits == 8 else (136, 8)
    ks = torch.nan_to_num(c.k_scales, nan=0.0).max().double()
    e_s = ((D / 16 + 4) * 2.0 ** -23 * (off + top) * q.double().abs().sum(-1) * ks * abs(scale) * 1.4427
           + 2.0 ** -22)[..., None]
    n = max(lengths, default=0) + prefix_len
    floor = n * 2.0 ** -24 * top * torch.nan_to_num(c.v_scales, nan=0.0).max().double()
    tol = (2.0 ** -11 + 4 * e_s + 2.0 ** -20) * mag + 2.0 ** -8 * out64.abs() + floor
    bad = (got.double() - out64).abs() > tol
    assert got.shape == q.shape and not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:3].tolist())
    if lse is not None:
        inf = lse64 == float("-inf")
        assert torch.equal(lse == float("-inf"), inf)
        d = (lse.double() - lse64).abs()[~inf]
        assert bool((d <= (2 * e_s[..., 0].expand_as(lse64) + 2.0 ** -18 * (1 + lse64.abs()))[~inf]).all())


def run_attention(dtype, dim, page, heads, group, T, lengths, prefix_len, seed=0, outlier=False):
    pages = len(lengths) * max(1, -(-max(lengths) // page)) + -(-prefix_len // page) + 3
    c = pool(pages, heads, dim, dtype, page, seed)
    table, rest = tables(lengths, page, pages, seed)
    g = torch.Generator("cuda").manual_seed(seed)
    q = torch.randn(len(lengths), T, heads * group, dim, generator=g, device="cuda")
    if outlier:
        q[..., 3] *= 30
    q = q.bfloat16()
    n = torch.tensor(lengths, device="cuda")
    out, lse = mxb.paged_attention(q, c, table, n, prefix_table=rest, prefix_len=prefix_len, return_lse=True)
    check_attention(out, lse, q, c, table, lengths, rest, prefix_len)
    assert L.load().mxb_device_error(1) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["int8d", "int4d"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page,heads,group,T,lengths", [
    (16, 1, 1, 1, [1]), (64, 2, 4, 1, [130]), (16, 3, 8, 1, [1, 17, 0, 256, 255]),
    (32, 2, 5, 3, [2, 40, 0, 1]), (64, 1, 8, 4, [300, 3]), (128, 2, 3, 5, [1000, 999, 33]),
    (16, 1, 16, 1, [513]), (1024, 1, 2, 1, [2050]), (32, 2, 40, 1, [70])])
def test_attention(dtype, dim, page, heads, group, T, lengths):
    run_attention(dtype, dim, page, heads, group, T, lengths, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["int8d", "int4d"])
@pytest.mark.parametrize("dim,page,heads,group,T,lengths,prefix", [
    (128, 16, 2, 4, 1, [5, 0, 33], 1), (64, 32, 1, 8, 2, [40, 1], 95),        # few rows
    (128, 64, 2, 8, 1, [3] * 6, 64), (64, 16, 1, 5, 3, [9] * 7, 131),         # one 128-row group
    (128, 64, 1, 8, 1, [20, 0] * 12, 1000), (64, 128, 2, 8, 1, [70] * 40, 640),  # two
    (128, 32, 1, 1, 1, [4] * 300, 200)])                                      # and more
def test_attention_with_a_shared_prefix(dtype, dim, page, heads, group, T, lengths, prefix):
    run_attention(dtype, dim, page, heads, group, T, lengths, prefix)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["int8d", "int4d"])
@pytest.mark.parametrize("dim,page,heads,group,T,lengths,prefix", [
    (128, 16, 2, 4, 16, [16, 40, 7, 0], 0), (64, 32, 1, 8, 70, [70, 200, 71, 3], 0),   # a unit a CTA
    (128, 64, 1, 5, 33, [33, 4500, 100], 0), (64, 64, 2, 1, 129, [5000, 129], 0),       # the shared list
    (128, 32, 2, 2, 40, [40, 90], 500), (64, 16, 1, 3, 7, [9, 7], 200)])                # behind a prefix
def test_attention_of_a_chunk_of_a_prompt(dtype, dim, page, heads, group, T, lengths, prefix):
    """Many query tokens a sequence: several row tiles, each row with a limit of its own."""
    run_attention(dtype, dim, page, heads, group, T, lengths, prefix)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["int8d", "int4d"])
def test_attention_long_skewed_batch(dtype):
    run_attention(dtype, 128, 64, 2, 4, 1, [20000, 3, 0, 700, 129], 0)
    run_attention(dtype, 64, 16, 1, 8, 3, [9000, 1, 0, 77], 3000, outlier=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["int8d", "int4d"])
@pytest.mark.parametrize("T,group,prefix", [(1, 4, 0), (3, 8, 0), (1, 4, 100)])
def test_attention_of_short_sequences_beside_a_long_one(dtype, T, group, prefix):
    """A table wide enough for 4200 keys, nearly all of it unused: many units of a
    tile or two in a CTA's run, empty ones between them."""
    run_attention(dtype, 64, 32, 2, group, T, [4200] + [0, 1, 31, 32, 33, 0, 65, 100] * 17, prefix)
    run_attention(dtype, 128, 64, 3, group, T, [1, 0, 40, 0, 4160, 64, 2], prefix)


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,width,prefix", [([70, 3], 2, 0), ([300, 1], 60, 0), ([70, 3], 2, 100),
                                                  ([70] * 130, 2, 0), ([70] * 130, 2, 100)])
def test_attention_of_zero_values_under_low_scores(lengths, width, prefix):
    """Value scales of zero leave no weight in range, wherever the scores lie."""
    c = pool(64, 2, 128, "int8d", 64, 5)
    c.v_scales.zero_()
    c.k_codes.fill_(100)
    c.k_scales.fill_(1.0)
    q = torch.full((len(lengths), 1, 8, 128), -1.0, device="cuda").bfloat16()
    table = torch.arange(width, device="cuda", dtype=torch.int32).repeat(len(lengths), 1)
    n = torch.tensor(lengths, device="cuda")
    out, lse = mxb.paged_attention(q, c, table, n, prefix_table=table[0], prefix_len=prefix, return_lse=True)
    assert not bool(out.any())
    want = torch.log(n + float(prefix)) - 100 * math.sqrt(128)
    assert torch.allclose(lse, want[:, None, None].expand_as(lse).float(), rtol=1e-5, atol=0)


@pytest.mark.gpu
def test_attention_scores_that_grow_and_values_of_any_scale():
    """Keys whose scores rise along the sequence move the running maximum again
    and again; value scales over six decades stay exact beside one another."""
    c = pool(40, 1, 128, "int8d", 64, 3)
    g = torch.Generator("cuda").manual_seed(3)
    ramp = torch.arange(40 * 64, device="cuda").float().view(40, 1, 64)
    c.k_scales.copy_(ramp * 2e-5)
    c.v_scales.copy_(10.0 ** (torch.rand(40, 1, 64, generator=g, device="cuda") * -6))
    table = torch.arange(40, device="cuda", dtype=torch.int32)
    q = torch.randn(12, 1, 8, 128, generator=g, device="cuda").bfloat16()
    for prefix in (0, 1500):
        own = table[None, 25:].repeat(12, 1)
        n = [900 - 7 * b for b in range(12)]
        out, lse = mxb.paged_attention(q, c, own, torch.tensor(n, device="cuda"), prefix_table=table[:25],
                                       prefix_len=prefix, return_lse=True)
        check_attention(out, lse, q, c, own, n, table[:25], prefix)


@pytest.mark.gpu
def test_attention_hidden_places_may_hold_anything():
    """NaN and infinite scales past the lengths, before the prefix's end and in
    keys that only later queries see reach no row that does not see them."""
    for dtype in ("int8d", "int4d"):
        c = pool(12, 2, 64, dtype, 16, 6)
        table = torch.tensor([[3, 1], [0, 2]], dtype=torch.int32, device="cuda")
        pre = torch.tensor([5, 6, 7, 8, 9], dtype=torch.int32, device="cuda")
        lengths, prefix = [21, 0], 70
        for s, bad in ((c.k_scales, float("nan")), (c.v_scales, float("inf"))):
            s[1, :, 5:], s[0], s[2], s[9, :, 6:] = bad, bad, bad, bad
            s[10], s[11], s[4] = bad, bad, bad
        g = torch.Generator("cuda").manual_seed(1)
        n = torch.tensor(lengths, device="cuda")
        for group, p in ((4, prefix), (4, 0), (40, prefix)):  # both prefix kernels, and none
            q = torch.randn(2, 2, 2 * group, 64, generator=g, device="cuda").bfloat16()
            out, lse = mxb.paged_attention(q, c, table, n, prefix_table=pre, prefix_len=p, return_lse=True)
            check_attention(out, lse, q, c, table, lengths, pre, p)
        # the newest key is NaN: only the newest query sees it
        c.k_scales[1, 0, 4] = float("nan")
        q = torch.randn(2, 2, 8, 64, generator=g, device="cuda").bfloat16()
        out = mxb.paged_attention(q, c, table, n)
        assert out[0, 1, :4].isnan().all() and out[0, 0].isfinite().all() and out[0, 1, 4:].isfinite().all()
        assert not out[1].any()


@pytest.mark.gpu
def test_attention_extreme_queries():
    """Query rows of any magnitude, zero rows, a NaN row."""
    c = pool(8, 1, 128, "int8d", 16, 8)
    table, lengths = torch.arange(8, device="cuda", dtype=torch.int32)[None], [100]
    q = torch.randn(1, 1, 6, 128, generator=torch.Generator().manual_seed(2)).cuda()
    q[0, 0, 1] *= 1e-30
    q[0, 0, 2] = 0
    q[0, 0, 3] *= 1e4
    q[0, 0, 4, 7] = float("nan")
    q = q.bfloat16()
    out = mxb.paged_attention(q, c, table, torch.tensor(lengths, device="cuda"))
    assert out[0, 0, 4].isnan().all()
    keep = [0, 1, 2, 5]
    check_attention(out[:, :, keep], None, q[:, :, keep], c, table, lengths, None, 0)
    # sharp: the largest score alone decides
    k = history(c, "k", table[0], 100)[0]
    best = (k @ q[0, 0, 3].double()).argmax()
    v = history(c, "v", table[0], 100)[0, best]
    assert bool(((out[0, 0, 3].double() - v).abs() <= 2.0 ** -7 * v.abs() + 1e-6).all())


@pytest.mark.gpu
def test_attention_repeats_on_any_stream_and_in_a_graph():
    """The same bits every time: no result depends on the order of CTAs."""
    c = pool(300, 2, 128, "int4d", 32, 9)
    table = torch.arange(160, device="cuda", dtype=torch.int32).view(32, 5)
    pre = torch.arange(160, 300, device="cuda", dtype=torch.int32)
    lengths = torch.arange(32, device="cuda", dtype=torch.int32) * 5
    q = torch.randn(32, 1, 16, 128, generator=torch.Generator().manual_seed(0)).cuda().bfloat16()
    run = lambda: mxb.paged_attention(q, c, table, lengths, prefix_table=pre, prefix_len=4470)  # noqa: E731
    want = run()
    for _ in range(30):
        assert torch.equal(run(), want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = run()
    s.synchronize()
    assert torch.equal(other, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run()
    lengths.copy_(torch.flip(lengths, (0,)))
    g.replay()
    assert torch.equal(out, run())
    assert L.load().mxb_device_error(1) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim,group,T", [
    ("int8d", 128, 4, 1), ("int8d", 128, 8, 2), ("int8d", 64, 8, 3), ("int4d", 128, 8, 3), ("int4d", 128, 8, 4)])
def test_attention_of_several_units_in_a_row_repeats(dtype, dim, group, T):
    """A CTA takes unit after unit, and the next unit's keys are copied over the
    buffer that the last one's rows were joined in."""
    lengths = [(29 * i) % 150 for i in range(150)]
    width = -(-4200 // 32)  # longer than one unit a CTA is used for
    c = pool(600, 4, dim, dtype, 32, 11)
    table = torch.randint(0, 600, (len(lengths), width), generator=torch.Generator().manual_seed(5),
                          dtype=torch.int32).cuda()
    q = torch.randn(len(lengths), T, 4 * group, dim, generator=torch.Generator().manual_seed(6)).cuda().bfloat16()
    n = torch.tensor(lengths, device="cuda")
    out, lse = mxb.paged_attention(q, c, table, n, return_lse=True)
    check_attention(out, lse, q, c, table, lengths, None, 0)
    for _ in range(20):
        again, _ = mxb.paged_attention(q, c, table, n, return_lse=True)
        assert torch.equal(again, out)
    assert L.load().mxb_device_error(1) == 0


@pytest.mark.gpu
def test_attention_bad_tables_are_recorded():
    c = pool(4, 1, 64, "int8d", 16, 1)
    q = torch.randn(1, 1, 2, 64, device="cuda").bfloat16()
    L.load().mxb_device_error(1)
    for table, n in (([[0, 99]], 20), ([[-3, 0]], 5)):
        mxb.paged_attention(q, c, torch.tensor(table, device="cuda"), torch.tensor([n], device="cuda"))
        assert L.load().mxb_device_error(1) == 8
    long = torch.zeros(1, 40, dtype=torch.int32, device="cuda")  # a table wide enough for the shared list
    a = mxb.paged_attention(q, c, long, torch.tensor([10 ** 6], device="cuda"))
    assert L.load().mxb_device_error(1) == 8
    assert torch.equal(a, mxb.paged_attention(q, c, long, torch.tensor([640], device="cuda")))
    assert L.load().mxb_device_error(1) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim,page,group,B,spare", [
    ("int8d", 128, 16, 4, 3, 0), ("int4d", 64, 64, 8, 3, 0),                 # a unit a CTA
    ("int8d", 64, 32, 4, 3, 300), ("int4d", 128, 128, 8, 3, 60),             # the shared list
    ("int8d", 128, 16, 8, 40, 0), ("int4d", 64, 32, 8, 40, 0), ("int4d", 128, 128, 8, 40, 0)])  # many rows
def test_attention_sees_no_keys_behind_bad_pages(dtype, dim, page, group, B, spare):
    """A page number outside the pool holds no keys, as in ``read``: the call gives
    what it gives without those pages, and page 0 is no stand-in."""
    c = pool(16, 2, dim, dtype, page, 12)
    c.k_scales[0] *= 20
    c.v_scales[0] *= 100
    rest = [0] * spare
    bad = torch.tensor([[4, 10 ** 6, 5, -7, 6, 7, 9] + rest] * B, device="cuda", dtype=torch.int32)
    good = torch.tensor([[4, 5, 6, 7, 9] + rest] * B, device="cuda", dtype=torch.int32)
    q = torch.randn(B, 1, 2 * group, dim, generator=torch.Generator().manual_seed(1)).cuda().bfloat16()
    n = [5 * page + 3] * B
    L.load().mxb_device_error(1)
    for own in (False, True):
        for pre in ((False, True) if own else (True,)):
            length = torch.tensor(n if own else [0] * B, device="cuda")
            out, lse = mxb.paged_attention(q, c, bad, length, prefix_table=bad[0], prefix_len=n[0] * pre,
                                           return_lse=True)
            assert L.load().mxb_device_error(1) == 8
            less = n[0] - 2 * page
            check_attention(out, lse, q, c, good, [less * own] * B, good[0], less * pre)
    none = torch.full_like(bad, 16)
    out, lse = mxb.paged_attention(q, c, none, torch.tensor(n, device="cuda"), prefix_table=none[0],
                                   prefix_len=n[0], return_lse=True)
    assert not out.any() and bool((lse == float("-inf")).all())
    assert L.load().mxb_device_error(1) == 8


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["int8d", "int4d"])
@pytest.mark.parametrize("B", [2, 12, 24])  # groups of 32 rows; 128-row tiles, one and two
@pytest.mark.parametrize("exponent", [-10, -20, -24, -40, -60])
@pytest.mark.parametrize("loud", [[3], [700], [1499], [64, 900]])
def test_attention_of_quiet_values_beside_loud_ones(dtype, B, exponent, loud):
    """Rows that rest on keys whose value scale lies far under another's, which
    they hardly see: the weights are held relative to the row's largest, so each
    is off by 2^-11 of itself or 2^-24 of that."""
    c = pool(24, 1, 128, dtype, 64, 13)
    top = 127 if dtype == "int8d" else 7
    c.v_scales.mul_(2.0 ** exponent)
    for j in loud:
        c.k_codes[j // 64, 0, j % 64] = 0x81 if dtype == "int8d" else 0x99  # -127, -7 and -7
        c.k_scales[j // 64, 0, j % 64] = 6.0 / top
        c.v_scales[j // 64, 0, j % 64] = 1.0
    g = torch.Generator("cuda").manual_seed(3)
    q = (1 + 0.5 * torch.randn(B, 1, 8, 128, generator=g, device="cuda")).bfloat16()
    pre = torch.arange(24, device="cuda", dtype=torch.int32)
    own, n, prefix = pre[None, :1].repeat(B, 1), [0] * B, 1500
    out, _ = mxb.paged_attention(q, c, own, torch.tensor(n, device="cuda"), prefix_table=pre,
                                 prefix_len=prefix, return_lse=True)
    out64, _, mag = attend64(q, c, own, n, pre, prefix, 128 ** -0.5)
    k, v = (history(c, w, pre, prefix)[0] for w in "kv")
    p = torch.softmax(torch.einsum("bgd,ld->bgl", q[:, 0].double(), k) * 128 ** -0.5, -1)
    largest = (p * c.v_scales[:, 0].flatten()[:prefix].double()).amax(-1)[:, None, :, None]
    off = 1152 + 127 if dtype == "int8d" else 136 + 8
    e_s = ((128 / 16 + 4) * 2.0 ** -23 * off * q.double().abs().sum(-1) * c.k_scales.max().double()
           * 128 ** -0.5 * 1.4427 + 2.0 ** -22)[..., None]
    tol = (2.0 ** -11 + 4 * e_s + 2.0 ** -20) * mag + 2.0 ** -8 * out64.abs() + prefix * 2.0 ** -24 * 128 * largest
    assert bool(((out.double() - out64).abs() <= tol).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["int8d", "int4d"])
@pytest.mark.parametrize("B,own", [(2, False), (12, False), (24, True)])
@pytest.mark.parametrize("span", [5, 14, 30])
def test_attention_of_value_scales_of_any_size(dtype, B, own, span):
    """Value scales over 2^-span, in no order: every weight is off by 2^-11 of itself
    or, below fp16's normal range, by 2^-17 of the row's largest at most, either way;
    over the keys that is held to 2^-20 each."""
    c = pool(30, 1, 64, dtype, 64, 16)
    g = torch.Generator("cuda").manual_seed(span)
    c.v_scales.copy_(2.0 ** (torch.rand(30, 1, 64, generator=g, device="cuda") * -span))
    q = (3 * torch.randn(B, 1, 8, 64, generator=g, device="cuda")).bfloat16()
    pages = torch.arange(30, device="cuda", dtype=torch.int32)
    table, n, prefix = pages[None, 24:].repeat(B, 1), [300 * own] * B, 1500
    out = mxb.paged_attention(q, c, table, torch.tensor(n, device="cuda"), prefix_table=pages[:24],
                              prefix_len=prefix)
    out64, _, mag = attend64(q, c, table, n, pages[:24], prefix, 0.125)
    k, s = history(c, "k", pages, 1920)[0], c.v_scales[:, 0].flatten().double()
    live = torch.arange(1920, device="cuda")
    live = (live < prefix) | ((live >= 24 * 64) & (live < 24 * 64 + n[0]))
    p = torch.softmax((torch.einsum("bgd,ld->bgl", q[:, 0].double(), k) * 0.125).masked_fill(~live, float("-inf")), -1)
    largest = (p * s).amax(-1)[:, None, :, None]
    off, top = (1152 + 127, 127) if dtype == "int8d" else (136 + 8, 8)
    e_s = ((64 / 16 + 4) * 2.0 ** -23 * off * q.double().abs().sum(-1) * c.k_scales.max().double()
           * 0.125 * 1.4427 + 2.0 ** -22)[..., None]
    tol = (2.0 ** -11 + 4 * e_s + 2.0 ** -20) * mag + 2.0 ** -8 * out64.abs() + 2.0 ** -20 * top * largest * int(live.sum())
    assert bool(((out.double() - out64).abs() <= tol).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["int8d", "int4d"])
@pytest.mark.parametrize("B", [1, 12, 40])
def test_attention_nan_query_has_a_nan_sum(dtype, B):
    """A NaN query's log-sum-exp is NaN, behind a prefix alone as with keys of its
    own; the other rows are untouched."""
    c = pool(4, 1, 64, dtype, 64, 14)
    q = torch.randn(B, 1, 8, 64, generator=torch.Generator().manual_seed(2)).cuda().bfloat16()
    q[0, 0, 3, 5] = float("nan")
    pre = torch.arange(4, device="cuda", dtype=torch.int32)
    for n in (0, 20):
        out, lse = mxb.paged_attention(q, c, pre[None, :1].repeat(B, 1), torch.full((B,), n, device="cuda"),
                                       prefix_table=pre, prefix_len=200, return_lse=True)
        want = torch.zeros(B, 1, 8, dtype=torch.bool, device="cuda")
        want[0, 0, 3] = True
        assert torch.equal(lse.isnan(), want) and torch.equal(out.isnan().all(-1), want)
        assert torch.equal(out.isnan().any(-1), want)


@pytest.mark.gpu
def test_64_bit_tables_and_lengths_do_not_wrap():
    """Page numbers and lengths past 32 bits are outside the pool and the table, not
    their low halves."""
    c = pool(4, 2, 64, "int8d", 16, 15)
    q = torch.randn(1, 1, 4, 64, generator=torch.Generator().manual_seed(0)).cuda().bfloat16()
    L.load().mxb_device_error(1)
    wide = torch.tensor([[1, 2 ** 32 + 2, -2 ** 32 + 3, 2]], device="cuda")
    n = torch.tensor([60], device="cuda")
    k, _ = c.read(wide, n, 64, torch.float32)
    assert L.load().mxb_device_error(1) == 8
    assert k[0, :16].any() and not k[0, 16:48].any() and k[0, 48:60].any()
    far = torch.tensor([2 ** 32 + 3], device="cuda")
    good = torch.tensor([[1, 2, 3, 2]], device="cuda")
    a = mxb.paged_attention(q, c, good, far)
    assert L.load().mxb_device_error(1) == 8
    assert torch.equal(a, mxb.paged_attention(q, c, good, torch.tensor([64], device="cuda")))
    none = mxb.paged_attention(q, c, good, torch.tensor([-2 ** 32 + 3], device="cuda"))
    assert not none.any() and L.load().mxb_device_error(1) == 0
    for rep in (1, 10):  # both prefix kernels
        qq = q.repeat(rep, 1, 4, 1)
        short = torch.tensor([[1, 2]] * rep, device="cuda")
        zero = torch.zeros(rep, dtype=torch.int32, device="cuda")
        out, lse = mxb.paged_attention(qq, c, short, zero, prefix_table=wide[0], prefix_len=60, return_lse=True)
        assert L.load().mxb_device_error(1) == 8
        check_attention(out, lse, qq, c, short, [0] * rep, short[0], 28)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """A pool of 5.4 GB of codes each for K and V: the last page works like the first."""
    pages, heads, dim, page = 41000, 8, 128, 128
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip("needs 16 GB")
    c = mxb.paged_kv_cache(pages, heads, dim, "int8d", page)
    small = mxb.paged_kv_cache(2, heads, dim, "int8d", page)
    g = torch.Generator("cuda").manual_seed(0)
    k, v = (torch.randn(200, heads, dim, generator=g, device="cuda").bfloat16() for _ in range(2))
    at = torch.arange(200, device="cuda")
    far = torch.tensor([pages - 1, pages - 2], device="cuda")
    c.write(k, v, far[at // page] * page + at % page)
    small.write(k, v, at)
    near = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda")
    n = torch.tensor([200], device="cuda")
    for x, y in zip(c.read(far[None], n, 200), small.read(near, n, 200)):
        assert torch.equal(x, y)
    q = torch.randn(1, 1, 32, dim, generator=g, device="cuda").bfloat16()
    assert torch.equal(mxb.paged_attention(q, c, far[None], n), mxb.paged_attention(q, small, near, n))
    q = q.expand(16, 1, 32, dim).contiguous()
    none, zero = far[None].expand(16, 2)[:, :0], torch.zeros(16, device="cuda", dtype=torch.int32)
    assert torch.equal(mxb.paged_attention(q, c, none, zero, prefix_table=far, prefix_len=200),
                       mxb.paged_attention(q, small, none, zero, prefix_table=near[0], prefix_len=200))


# ── together ─────────────────────────────────────────────────────────────────
@pytest.mark.gpu
def test_serving_example_matches_the_dequantized_layer():
    """The example's layer against the same layer in fp32 on what its cache and
    weights stand for."""
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
    import serve_step

    layer, y = serve_step.main(batch=6, document=300, steps=5)
    assert y.shape == (6, 5, 1024) and bool(y.isfinite().all())
    c = layer.cache
    page = c.page_size
    doc = torch.arange(-(-300 // page), device="cuda")
    for b in range(6):
        own = torch.tensor([len(doc) + b], device="cuda")
        k, _ = c.read(own[None].int(), torch.tensor([5], device="cuda"), 5, torch.float32)
        assert bool((k.abs().amax(-1) > 0).all())  # five tokens were written there
    x = torch.randn(6, 1, 1024, generator=torch.Generator("cuda").manual_seed(7), device="cuda").bfloat16()
    table = torch.arange(len(doc), len(doc) + 6, device="cuda")[:, None]
    slots = table * page + 5
    n = torch.full((6,), 6, dtype=torch.int32, device="cuda")
    got = layer.step(x, slots, table, n, doc, 300)
    q = layer.qkv(x.reshape(6, -1))[:, :1024].reshape(6, 1, layer.heads, layer.head_dim)
    out64, _, mag = attend64(q, c, table, [6] * 6, doc, 300, layer.head_dim ** -0.5)
    o = mxb.paged_attention(q, c, table, n, prefix_table=doc, prefix_len=300)
    check_attention(o, None, q, c, table, [6] * 6, doc, 300)
    assert torch.equal(got, layer.out(o.reshape(6, 1, 1024)))


@pytest.mark.gpu
def test_attention_of_a_batch_wider_than_a_block():
    """More sequences than threads in a CTA: the shared list is scanned in steps."""
    lengths = [(37 * i) % 300 for i in range(301)]
    run_attention("int8d", 64, 16, 2, 2, 1, lengths, 0)
    run_attention("int4d", 128, 64, 1, 4, 1, lengths[:129], 70)
