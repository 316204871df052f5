"""Microscaled 4-bit floating point (mxfp4, nvfp4): codes and scales bit for bit
against a numpy restatement of the formulas, values exactly, products within
the bound of fp32 accumulation against 64 bits; refusals.

The reference has no counterpart (its float4 grid, mxtorch.py:1465-1528, is
another format).
"""
import copy
import ctypes
import io
import pickle

import numpy as np
import pytest
import torch

import qtpytorch_b200 as mxb
from qtpytorch_b200 import _lib as L
from qtpytorch_b200 import fp4

F32 = np.float32
GRID = np.array([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=np.float64)


def e4m3_table():
    b = np.arange(128)
    v = np.where(b < 8, b / 8 * 2.0 ** -6, (1 + (b & 7) / 8) * 2.0 ** ((b >> 3) - 7.0))
    return v[:127]  # 127 is NaN


def nearest_even(v, table):
    """Index of the nearest table entry (non-negative, sorted), ties to the even index."""
    hi = np.clip(np.searchsorted(table, v), 1, len(table) - 1)
    lo = hi - 1
    dl, dh = v - table[lo], table[hi] - v
    return np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)


def ref_quantize(x, fmt, g=None):
    """(codes [rows, blocks, B], scale bytes [rows, blocks], g): the formulas with
    one fp32 rounding an operation."""
    B = fp4.BLOCK[fmt]
    rows, K = x.shape
    x = np.pad(x.astype(F32), ((0, 0), (0, -K % B))).reshape(rows, -1, B)
    with np.errstate(invalid="ignore"):
        amax = np.abs(x).max(-1)
    bad = ~np.isfinite(amax)
    safe = np.where(bad, F32(0), amax)
    if fmt == "mxfp4":
        _, ex = np.frexp(safe.astype(np.float64))
        e = np.clip(np.where(safe > 0, ex - 1 - 2, -127), -127, 127)
        byte = np.where(bad, 255, e + 127)
        scale = (2.0 ** e)[..., None]
        q = np.where(bad[..., None], 0, np.nan_to_num(x.astype(np.float64), posinf=0, neginf=0)) / scale
    else:
        if g is None:
            top = F32(np.nan) if bad.any() else amax.max()
            g = F32(top * F32(1.0 / 2688.0)) if np.isfinite(top) and top > 0 else F32(1)
        want = np.minimum((safe / (F32(6) * g)).astype(F32), F32(448))
        byte = nearest_even(want.astype(np.float64), e4m3_table())
        s = (e4m3_table()[byte].astype(F32) * g).astype(F32)[..., None]
        byte = np.where(bad, 127, byte)
        z = np.where(bad[..., None], F32(0), np.nan_to_num(x, posinf=0, neginf=0))
        q = np.where(s > 0, (z / np.where(s > 0, s, F32(1))).astype(F32), F32(0) * z).astype(np.float64)
    code = nearest_even(np.minimum(np.abs(q), 6.0), GRID)
    code = code + 8 * (np.signbit(x) & ~bad[..., None])
    return code.astype(np.uint8), byte.astype(np.uint8), g


def ref_values(code, byte, fmt, g, K):
    v = np.where(code & 8, -1.0, 1.0) * GRID[code & 7]
    if fmt == "mxfp4":
        s = np.where(byte == 255, np.nan, 2.0 ** (byte.astype(np.float64) - 127))
    else:
        s = np.where(byte == 127, np.nan, e4m3_table()[np.minimum(byte, 126)])
        s = (s.astype(F32) * F32(g)).astype(np.float64)
    return (v * s[..., None]).reshape(code.shape[0], -1)[:, :K].astype(F32)


def unpacked(t):
    """codes [rows, blocks, B] of an fp4_tensor, and the padding's bytes."""
    B, K = fp4.BLOCK[t.fmt], t.shape[-1]
    c = t.codes.cpu().numpy()
    flat = np.stack((c & 15, c >> 4), -1).reshape(c.shape[0], -1)
    n = -(-K // B) * B
    return flat[:, :n].reshape(c.shape[0], -1, B), flat[:, n:]


# ── host ─────────────────────────────────────────────────────────────────────
def test_sizes_agree_with_the_library():
    lib = L.load()
    for rows, K in ((1, 1), (1, 32), (3, 33), (128, 256), (129, 4100), (11008, 4096)):
        assert lib.mxb_fp4_code_bytes(rows, K) == rows * fp4.code_row_bytes(K)
        for fmt, f in fp4.FORMATS.items():
            assert lib.mxb_fp4_scale_bytes(rows, K, f) == fp4.scale_bytes(rows, K, fmt)


def test_argument_errors_need_no_gpu():
    lib = L.load()
    p, g = ctypes.c_void_p(32), ctypes.c_void_p(16)
    q = lib.mxb_fp4_quantize
    assert q(p, 0, 4, 64, 64, 7, None, 0, p, p, None, 0, None) == -2
    assert q(p, 5, 4, 64, 64, 0, None, 0, p, p, None, 0, None) == -2
    assert q(p, 0, 4, 64, 63, 0, None, 0, p, p, None, 0, None) == -1
    assert q(None, 0, 4, 64, 64, 0, None, 0, p, p, None, 0, None) == -6
    assert q(p, 0, 4, 64, 64, 1, None, 0, p, p, None, 0, None) == -6  # nvfp4 without a factor
    assert q(p, 0, 4, 64, 64, 0, g, 0, p, p, None, 0, None) == -6     # mxfp4 with one
    assert q(p, 0, 4, 64, 64, 0, None, 0, ctypes.c_void_p(8), p, None, 0, None) == -3
    assert q(p, 0, 4, 64, 64, 1, g, 1, p, p, None, 0, None) == -7
    assert q(p, 0, 0, 64, 64, 0, None, 0, p, p, None, 0, None) == 0
    d = lib.mxb_fp4_dequantize
    assert d(p, p, None, 4, 64, 0, p, 9, None) == -2
    assert d(p, p, None, 4, 64, 1, p, 0, None) == -6
    assert d(p, None, None, 4, 64, 0, p, 0, None) == -6
    m = lib.mxb_fp4_matmul
    assert m(p, p, None, p, p, None, 4, 64, 4, 3, None, p, 1, None) == -2
    assert m(p, p, None, p, p, None, 4, 0, 4, 0, None, p, 1, None) == -1
    assert m(p, p, g, p, p, None, 4, 64, 4, 1, None, p, 1, None) == -6
    assert m(p, p, None, p, p, None, 4, 64, 4, 0, None, None, 1, None) == -6
    assert m(p, ctypes.c_void_p(8), None, p, p, None, 4, 64, 4, 0, None, p, 1, None) == -3
    assert m(p, p, None, p, p, None, 0, 64, 4, 0, None, p, 1, None) == 0


def test_misaligned_pointers_are_refused():
    lib, p, g, odd = L.load(), ctypes.c_void_p(32), ctypes.c_void_p(16), ctypes.c_void_p(33)
    n = lib.mxb_fp4_quantize_workspace_size(4, 64, 1, 1)
    for dt in (0, 1):
        assert lib.mxb_fp4_quantize(odd, dt, 4, 64, 64, 0, None, 0, p, p, None, 0, None) == -3
        assert lib.mxb_fp4_dequantize(p, p, None, 4, 64, 0, odd, dt, None) == -3
    assert lib.mxb_fp4_quantize(p, 0, 4, 64, 64, 1, g, 1, p, p, odd, n - 1, None) == -3
    assert lib.mxb_fp4_quantize(p, 0, 4, 64, 64, 1, g, 1, p, p, p, n - 1, None) == -7


def test_refusals():
    with pytest.raises(L.MxbError):
        mxb.fp4_tensor.quantize(torch.zeros(4, 64))
    with pytest.raises(ValueError):
        mxb.fp4_tensor.quantize(torch.zeros(4, 64), "fp4")
    codes, scales = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8)
    t = mxb.fp4_tensor(codes, scales, "mxfp4", (4, 64))
    assert t.nbytes == 4 * 32 + 512 and t.block_scales().shape == (4, 2)
    for bad in (dict(shape=(4, 96)), dict(codes=codes.float()), dict(global_scale=torch.ones(1)),
                dict(fmt="nvfp4"), dict(scales=scales[:511])):
        a = dict(codes=codes, scales=scales, fmt="mxfp4", shape=(4, 64))
        a.update(bad)
        with pytest.raises(ValueError):
            mxb.fp4_tensor(**a)
    with pytest.raises(L.MxbError):
        t.dequantize()
    with pytest.raises(ValueError):
        t.dequantize(torch.float16)
    with pytest.raises(TypeError):
        mxb.fp4_matmul(t, codes)
    nv = mxb.fp4_tensor(codes, scales, "nvfp4", (4, 64), torch.ones(1))
    with pytest.raises(ValueError):
        mxb.fp4_matmul(t, nv)
    with pytest.raises(ValueError):
        mxb.fp4_matmul(t, mxb.fp4_tensor(codes, scales, "mxfp4", (4, 40)))
    with pytest.raises(ValueError):
        mxb.fp4_matmul(t, t, out_dtype=torch.float16)
    with pytest.raises(L.MxbError):
        mxb.fp4_matmul(t, t)


def one_buffer(fmt, rows=3, K=40):
    """An fp4_tensor as ``quantize`` leaves it (one allocation), on the host."""
    cb, sb = rows * fp4.code_row_bytes(K), fp4.scale_bytes(rows, K, fmt)
    at_s = -(-cb // 256) * 256
    nv = fmt == "nvfp4"
    t = mxb.fp4_tensor.__new__(mxb.fp4_tensor)
    t.fmt, t.shape = fmt, torch.Size((rows, K))
    t._parts = (torch.arange(at_s + sb + 16 * nv, dtype=torch.int64).to(torch.uint8), rows, cb, at_s, sb,
                at_s + sb if nv else None)
    return t


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("viewed", [False, True])
def test_copies_own_their_addresses(fmt, viewed):
    """A copied, pickled or saved tensor hands the kernels its own memory, on the
    device that this memory is on."""
    t = one_buffer(fmt)
    buf = io.BytesIO()
    torch.save(t, buf)
    buf.seek(0)
    if viewed:
        t.codes
    for u in (copy.deepcopy(t), pickle.loads(pickle.dumps(t)), torch.load(buf, weights_only=False)):
        g = u.global_scale
        assert u._ptrs() == (u.codes.data_ptr(), u.scales.data_ptr(), 0 if g is None else g.data_ptr())
        assert not set(u._ptrs()[:2]) & set(t._ptrs()[:2]) and u.device == u.codes.device
        assert torch.equal(u.codes, t.codes) and torch.equal(u.scales, t.scales) and u.shape == t.shape
    same = copy.copy(t)
    assert same._ptrs() == t._ptrs() == (t.codes.data_ptr(), t.scales.data_ptr(),
                                         0 if fmt == "mxfp4" else t.global_scale.data_ptr())
    buf.seek(0)
    assert torch.load(buf, map_location="meta", weights_only=False).device.type == "meta"


def test_parts_asked_for_by_two_threads():
    """Another thread makes the views between this one's look at the parts and its
    use of them."""
    t = one_buffer("nvfp4")
    made = one_buffer("nvfp4")._views()

    class Meanwhile(tuple):
        def __len__(self):
            n = super().__len__()
            t._parts = made
            return n

    t._parts = Meanwhile(t._parts)
    assert torch.equal(t.codes, made[0]) and torch.equal(t.scales, made[1])


def saved(x):
    buf = io.BytesIO()
    torch.save(x, buf)
    buf.seek(0)
    return torch.load(buf, weights_only=False)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_saved_after_its_parts_were_read(fmt):
    """The parts of one allocation go through torch.save: as a tensor, as a
    module's state and as a module."""
    t = one_buffer(fmt)
    t.codes
    m = mxb.fp4_linear(t)
    sd, u, n = saved(m.state_dict()), saved(t), saved(m)
    for w in (u, n.weight, mxb.fp4_tensor(sd["weight_codes"], sd["weight_scales"], fmt, t.shape,
                                          sd.get("weight_global_scale"))):
        assert torch.equal(w.codes, t.codes) and torch.equal(w.scales, t.scales)
        assert fmt == "mxfp4" or w.global_scale.view(torch.int32).equal(t.global_scale.view(torch.int32))


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("cast", [lambda m: m.bfloat16(), lambda m: m.half(), lambda m: m.double(),
                                  lambda m: m.to(torch.bfloat16), lambda m: m.to("cpu", torch.half)])
def test_linear_module_casts_leave_the_weight_alone(fmt, cast):
    t = one_buffer(fmt, 5, 64)
    bias = torch.randn(5, generator=torch.Generator().manual_seed(0))
    if fmt == "nvfp4":
        t = mxb.fp4_tensor(t.codes, t.scales, fmt, t.shape, torch.tensor([0.1234567]))
    m = cast(torch.nn.Sequential(torch.nn.Linear(64, 64), mxb.fp4_linear(t, bias)))
    w = m[1].weight  # raises where the factor's type changed
    assert m[0].weight.dtype != torch.float32
    assert torch.equal(w.codes, t.codes) and torch.equal(w.scales, t.scales)
    assert fmt == "mxfp4" or torch.equal(w.global_scale, t.global_scale)
    assert m[1].bias.dtype == torch.float32 and torch.equal(m[1].bias, bias)
    assert m.to("meta")[1].weight.device.type == "meta" and m[1].bias.dtype == torch.float32


# ── quantize ─────────────────────────────────────────────────────────────────
def special(rows, K, seed):
    """Normal values, with exact ties, zeros, a zero block, tiny and huge blocks."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, K, generator=g)
    x[torch.rand(rows, K, generator=g) < 0.1] = 0.0
    ties = torch.tensor([.25, .75, 1.25, 1.75, 2.5, 3.5, 5., 6.])
    n = min(K, 8)
    x[0, :n] = ties[:n]
    if rows > 2:
        x[1] = 0.0
        x[2] *= 1e-40
    if rows > 3:
        x[3] *= 2.0 ** 120
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,K", [(1, 1), (1, 32), (3, 17), (5, 100), (129, 250), (128, 256), (33, 4097), (300, 1500)])
def test_quantize_codes_scales_values(fmt, dtype, rows, K):
    x = special(rows, K, rows * 7919 + K).to(dtype)
    if fmt == "nvfp4" and rows > 3:
        x[3] = 1.0  # one factor a tensor: a huge row would flush the others
    t = mxb.fp4_tensor.quantize(x.cuda(), fmt)
    code, byte, g = ref_quantize(x.float().numpy(), fmt)
    got, pad = unpacked(t)
    assert np.array_equal(got, code) and not pad.any()
    assert np.array_equal(t.block_scales().cpu().numpy(), byte)
    if fmt == "nvfp4":
        assert t.global_scale.item() == g
    # bytes of the padding rows and blocks are zero
    total = int(t.scales.cpu().to(torch.int64).sum())
    assert total == int(byte.astype(np.int64).sum())
    v = ref_values(code, byte, fmt, g, K)
    assert np.array_equal(t.dequantize().cpu().numpy(), v)
    assert torch.equal(t.dequantize(torch.bfloat16).cpu(), torch.from_numpy(v).bfloat16())


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("rows,K", [(700, 1001), (700, 1002), (700, 1004), (700, 1000), (2, 1), (1100, 3)])
def test_rows_of_every_alignment(fmt, rows, K):
    x = special(rows, K, rows + K)
    x[rows - 1, K - 1] = 9.0  # the last value is the largest of nvfp4's blocks
    if rows > 3:
        x[3] = 1.0
    for s in (x.cuda(), torch.cat((x, x[:, :1]), 1).cuda()[:, :K]):  # rows with a gap as well
        t = mxb.fp4_tensor.quantize(s, fmt)
        code, byte, g = ref_quantize(x.numpy(), fmt)
        assert np.array_equal(unpacked(t)[0], code)
        assert fmt == "mxfp4" or t.global_scale.item() == g
        v = ref_values(code, byte, fmt, g, K)
        assert np.array_equal(t.dequantize().cpu().numpy(), v)
        assert torch.equal(t.dequantize(torch.bfloat16).cpu(), torch.from_numpy(v).bfloat16())


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_quantize_infinities_and_nan_stay_in_their_block(fmt):
    x = torch.randn(4, 96, generator=torch.Generator().manual_seed(3))
    x[1, 40], x[2, 3], x[3, 95] = float("inf"), float("nan"), float("-inf")
    t = mxb.fp4_tensor.quantize(x.cuda(), fmt, None if fmt == "mxfp4" else torch.tensor([0.01]).cuda())
    code, byte, _ = ref_quantize(x.numpy(), fmt, None if fmt == "mxfp4" else F32(0.01))
    assert np.array_equal(unpacked(t)[0], code)
    assert np.array_equal(t.block_scales().cpu().numpy(), byte)
    bad = torch.zeros(4, 96, dtype=torch.bool)
    b = fp4.BLOCK[fmt]
    bad[1, 40 // b * b:40 // b * b + b] = bad[2, :b] = bad[3, 96 - b:] = True
    assert torch.equal(t.dequantize().cpu().isnan(), bad)


@pytest.mark.gpu
def test_quantize_factor_rules():
    z = mxb.fp4_tensor.quantize(torch.zeros(3, 40, device="cuda"), "nvfp4")
    assert z.global_scale.item() == 1.0 and not z.dequantize().any()
    g = torch.tensor([0.5], device="cuda")
    x = torch.randn(3, 40, generator=torch.Generator().manual_seed(1))
    t = mxb.fp4_tensor.quantize(x.cuda(), "nvfp4", g)
    code, byte, _ = ref_quantize(x.numpy(), "nvfp4", F32(0.5))
    assert np.array_equal(unpacked(t)[0], code) and t.global_scale.item() == 0.5
    with pytest.raises(ValueError):
        mxb.fp4_tensor.quantize(x.cuda(), "mxfp4", g)
    with pytest.raises(ValueError):
        mxb.fp4_tensor.quantize(x.cuda(), "nvfp4", g.cpu())


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantize_keeps_the_sign_of_zero(fmt, dtype):
    x = torch.randn(40, 100, generator=torch.Generator().manual_seed(6)).to(dtype)
    x[:, ::3], x[:, 1::6] = -0.0, 0.0
    t = mxb.fp4_tensor.quantize(x.cuda(), fmt)
    code, _, _ = ref_quantize(x.float().numpy(), fmt)
    assert np.array_equal(unpacked(t)[0], code)


@pytest.mark.gpu
@pytest.mark.parametrize("g", [1e-20, 1e-25, 1e-30, 2e-33])
def test_quantize_under_a_factor_far_too_small_saturates(g):
    """Quotients past fp32 go to 6 with their sign, like smaller ones."""
    x = torch.randn(20, 96, generator=torch.Generator().manual_seed(7))
    x *= 10.0 ** torch.arange(-20, 40, 3)[:, None].float().clamp(max=37)
    t = mxb.fp4_tensor.quantize(x.cuda(), "nvfp4", torch.tensor([g], device="cuda"))
    with np.errstate(over="ignore"):
        code, byte, _ = ref_quantize(x.numpy(), "nvfp4", F32(g))
    assert np.array_equal(unpacked(t)[0], code)
    assert np.array_equal(t.block_scales().cpu().numpy(), byte)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_quantize_strides_types_and_empty(fmt):
    base = torch.randn(9, 3, 80, generator=torch.Generator().manual_seed(2)).cuda()
    want = mxb.fp4_tensor.quantize(base[:, 1].contiguous(), fmt)
    for x in (base[:, 1], base[:, 1].t().contiguous().t(), base.flatten(1)[:, 80:160]):
        t = mxb.fp4_tensor.quantize(x, fmt)
        assert torch.equal(t.codes, want.codes) and torch.equal(t.scales, want.scales)
    odd = torch.empty(9 * 80 + 1, device="cuda")[1:].view(9, 80).copy_(base[:, 1])  # 4-byte aligned
    assert torch.equal(mxb.fp4_tensor.quantize(odd, fmt).codes, want.codes)
    half = mxb.fp4_tensor.quantize(base[:, 1].half(), fmt)
    assert torch.equal(half.codes, mxb.fp4_tensor.quantize(base[:, 1].half().float(), fmt).codes)
    three = mxb.fp4_tensor.quantize(base, fmt)
    assert three.shape == (9, 3, 80) and three.dequantize().shape == (9, 3, 80)
    for shape in ((0, 64), (4, 0)):
        e = mxb.fp4_tensor.quantize(torch.empty(shape, device="cuda"), fmt)
        assert e.dequantize().shape == shape


# ── product ──────────────────────────────────────────────────────────────────
def product_case(m, k, n, fmt, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    x = torch.randn(m, k, generator=g, device="cuda")
    w = torch.randn(n, k, generator=g, device="cuda") * 0.02
    return mxb.fp4_tensor.quantize(x, fmt), mxb.fp4_tensor.quantize(w, fmt)


def check_product(y, a, b, bias=None):
    """|y - y64| <= (K + 4) 2^-23 (|a| |b|^T + |bias|): exact products of a few
    bits, at most one rounding (2^-23 where the hardware truncates) an addition,
    the factors and the bias; bf16 adds half an ulp of the result, 2^-9."""
    av, bv = a.dequantize().double(), b.dequantize().double()
    k = av.shape[-1]
    y64, mag = av @ bv.t(), av.abs() @ bv.abs().t()
    if bias is not None:
        y64, mag = y64 + bias.double(), mag + bias.double().abs()
    tol = (k + 4) * 2.0 ** -23 * mag + 1e-37
    if y.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * y64.abs()
    assert y.shape == y64.shape and bool(((y.double() - y64).abs() <= tol).all())


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("m,k,n", [
    (1, 1, 1), (1, 64, 128), (2, 31, 7), (16, 256, 128), (17, 300, 129), (32, 2048, 640), (33, 96, 130),
    (64, 1000, 1000), (65, 4096, 256), (128, 512, 384), (129, 257, 250), (300, 640, 1000), (515, 2050, 515)])
def test_product(fmt, m, k, n):
    a, b = product_case(m, k, n, fmt, m + k + n)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(n)).cuda()
    for out in (torch.float32, torch.bfloat16):
        check_product(mxb.fp4_matmul(a, b, out_dtype=out), a, b)
        check_product(mxb.fp4_matmul(a, b, bias, out), a, b, bias)
    assert L.load().mxb_device_error(1) == 0


@pytest.mark.gpu
def test_product_nan_stays_in_its_row_and_column():
    a, b = product_case(40, 200, 300, "mxfp4", 1)
    x = a.dequantize()
    x[5, 3] = float("nan")
    w = b.dequantize()
    w[290, 199] = float("inf")
    y = mxb.fp4_matmul(mxb.fp4_tensor.quantize(x), mxb.fp4_tensor.quantize(w))
    want = torch.zeros(40, 300, dtype=torch.bool, device="cuda")
    want[5], want[:, 290] = True, True
    assert torch.equal(y.isnan(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [3, 200])
@pytest.mark.parametrize("sx,sw", [(1e-18, 1e-18), (3e-19, 1e-17), (1e-30, 1e-6), (1e25, 1e25), (1e30, 1e15), (1e36, 1e-36)])
def test_product_of_factors_past_the_range(m, sx, sw):
    """Two nvfp4 factors whose product leaves fp32's normal range: the result is
    as near as any other where it lies in that range, and zeros stay zeros."""
    g = torch.Generator("cuda").manual_seed(1)
    x = torch.rand(m, 64, generator=g, device="cuda").add_(0.5).mul_(sx)
    w = torch.rand(130, 64, generator=g, device="cuda").add_(0.5).mul_(sw)
    x[1], w[129] = 0.0, 0.0
    a, b = mxb.fp4_tensor.quantize(x, "nvfp4"), mxb.fp4_tensor.quantize(w, "nvfp4")
    y = mxb.fp4_matmul(a, b, out_dtype=torch.float32)
    y64 = a.dequantize().double() @ b.dequantize().double().t()
    fits = y64 < 3e38
    # one rounding an addition and each of the factors' products, all terms positive
    assert bool(((y.double() - y64).abs() <= (64 + 6) * 2.0 ** -23 * y64)[fits].all())
    assert bool(y[~fits].isinf().all()) and not y[1].any() and not y[:, 129].any()


@pytest.mark.gpu
@pytest.mark.parametrize("m", [9, 40, 300])
def test_nvfp4_product_nan_stays_in_its_row_and_column(m):
    g = torch.Generator("cuda").manual_seed(m)
    x, w = torch.randn(m, 200, generator=g, device="cuda"), torch.randn(300, 200, generator=g, device="cuda")
    x[5, 3], w[290, 199] = float("nan"), float("-inf")
    one = torch.ones(1, device="cuda")  # a given factor: one from the data would be 1 here too
    y = mxb.fp4_matmul(mxb.fp4_tensor.quantize(x, "nvfp4", one / 100), mxb.fp4_tensor.quantize(w, "nvfp4"))
    want = torch.zeros(m, 300, dtype=torch.bool, device="cuda")
    want[5], want[:, 290] = True, True
    assert torch.equal(y.isnan(), want)


@pytest.mark.gpu
def test_product_repeats_bit_for_bit_on_any_stream_and_in_a_graph():
    a, b = product_case(20, 4096, 512, "nvfp4", 9)  # split over K
    y = mxb.fp4_matmul(a, b)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        z = mxb.fp4_matmul(a, b)
    s.synchronize()
    assert torch.equal(y, z)
    x = torch.randn(20, 4096, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c = mxb.fp4_matmul(mxb.fp4_tensor.quantize(x, "nvfp4"), b)
    for seed in (1, 2):
        x.copy_(torch.randn(20, 4096, generator=torch.Generator().manual_seed(seed)))
        g.replay()
        assert torch.equal(c, mxb.fp4_matmul(mxb.fp4_tensor.quantize(x, "nvfp4"), b))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_linear_module(fmt):
    lin = torch.nn.Linear(320, 200).cuda()
    m = mxb.fp4_linear.from_linear(lin, fmt)
    x = torch.randn(2, 5, 320, generator=torch.Generator().manual_seed(0)).cuda().bfloat16()
    a = mxb.fp4_tensor.quantize(x.reshape(10, 320), fmt)
    check_product(m(x).reshape(10, 200), a, m.weight, lin.bias)
    assert set(m.state_dict()) >= {"weight_codes", "weight_scales"}
    with pytest.raises(ValueError):
        mxb.fp4_matmul(a, m.weight, lin.bias[:7])
