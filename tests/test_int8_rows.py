"""int8 with a scale a row: norm into codes, product, linear; against 64 bits.

The norm's codes and the product's integer sums are exact, so both are compared
for equality; the reference's counterpart of the product is ``fused_int8_linear``
(mxtorch.py:3910-3960)."""
import copy
import ctypes
import io
import os
import subprocess
import sys

import pytest
import torch

import qtpytorch_b200 as mxb
from qtpytorch_b200 import _lib as L

P = ctypes.c_void_p(32)


# ── host ─────────────────────────────────────────────────────────────────────
def test_argument_errors_need_no_gpu():
    lib = L.load()

    def norm(x=P, r=None, dt=1, rows=2, d=64, w=P, wt=1, eps=1e-6, codes=P, scales=P, h=None):
        return lib.mxb_rms_norm_quantize(x, r, dt, rows, d, 64, 64, w, wt, eps, codes, scales, h, None)

    assert norm(dt=2) == -2 and norm(wt=5) == -2
    assert norm(rows=-1) == -1 and norm(d=0) == -1 and norm(d=(1 << 30) + 1) == -1 and norm(rows=1 << 31) == -1
    assert norm(eps=-1.0) == -6 and norm(eps=float("nan")) == -6 and norm(eps=float("inf")) == -6
    assert norm(x=None) == -6 and norm(w=None) == -6 and norm(codes=None) == -6 and norm(scales=None) == -6
    odd = ctypes.c_void_p(33)
    assert norm(x=odd) == -3 and norm(r=odd) == -3 and norm(h=odd) == -3 and norm(w=odd) == -3
    assert norm(scales=ctypes.c_void_p(34)) == -3 and norm(dt=0, x=ctypes.c_void_p(34)) == -3
    assert norm(rows=0) == 0
    # the sum lies over neither of its terms (rows 64 apart: 2 x 128 bytes of bf16)
    assert norm(h=P) == -6 and norm(h=ctypes.c_void_p(32 + 254)) == -6
    far = ctypes.c_void_p(4096)
    assert norm(r=far, h=far) == -6 and norm(r=far, h=ctypes.c_void_p(4096 - 254)) == -6

    def product(a=P, sa=P, sta=1, b=P, sb=P, stb=1, M=2, K=64, N=3, bias=None, out=P, od=1, ws=None, n=0):
        return lib.mxb_int8_matmul(a, sa, sta, b, sb, stb, M, K, N, bias, out, od, ws, n, None)

    assert product(od=2) == -2
    assert product(M=-1) == -1 and product(N=-1) == -1 and product(K=0) == -1 and product(K=131072) == -1
    assert product(M=65535 * 128 + 1) == -1 and product(N=1 << 30) == -1
    assert product(sta=2) == -6 and product(stb=-1) == -6
    assert product(a=None) == -6 and product(sb=None) == -6 and product(out=None) == -6
    assert product(out=odd) == -3 and product(sa=ctypes.c_void_p(34)) == -3 and product(bias=ctypes.c_void_p(34)) == -3
    assert product(M=0) == 0 and product(N=0) == 0
    size = lib.mxb_int8_matmul_workspace_size
    assert size(2, 64, 3, 1) == 0 and size(2, 64, 3, 0) == 5 * 64 and size(2, 65, 3, 1) == 5 * 80
    assert product(K=65) == -7 and product(K=65, ws=P, n=399) == -7 and product(a=odd) == -7
    assert product(K=65, ws=ctypes.c_void_p(40), n=400) == -3


def fake(rows, k, block=None, scales=None, dtype="int8d"):
    block = k if block is None else block
    n = -(-rows * k // block) if scales is None else scales
    return mxb.mx_tensor(torch.zeros(rows * k, dtype=torch.int8), torch.ones(n), mxb.get_mx_dtype(dtype), (rows, k),
                         rows * k, block)


def test_refusals():
    x, w = torch.zeros(2, 8), torch.ones(8)
    with pytest.raises(L.MxbError):
        mxb.rms_norm_quantize(x, w)  # on the CPU
    with pytest.raises(L.MxbError):
        mxb.int8_matmul(fake(2, 8), fake(3, 8))
    with pytest.raises(TypeError):
        mxb.int8_matmul(x, fake(3, 8))
    for a, b, kw in ((fake(2, 8), fake(3, 9), {}), (fake(2, 8), fake(3, 8), dict(out_dtype=torch.float16)),
                     (fake(2, 8, 4), fake(3, 8), {}), (fake(2, 8), fake(3, 8, 4), {})):
        with pytest.raises(ValueError):
            mxb.int8_matmul(a, b, **kw)
    with pytest.raises(NotImplementedError):
        mxb.int8_matmul(fake(2, 8, dtype="int4d"), fake(3, 8))
    with pytest.raises(NotImplementedError):
        mxb.int8_matmul(fake(2, 8, dtype="int8dh"), fake(3, 8))
    big = 131072
    with pytest.raises(NotImplementedError):
        mxb.int8_matmul(fake(1, big), fake(1, big))
    with pytest.raises(TypeError):
        mxb.int8_linear(torch.zeros(3, 8))


def test_linear_module_casts_and_copies():
    lin = mxb.int8_linear(fake(3, 8), torch.ones(3))
    for m in (copy.deepcopy(lin).bfloat16(), copy.deepcopy(lin).half(), copy.deepcopy(lin).to(torch.float64)):
        assert m.weight_codes.dtype == torch.int8
        assert m.weight_scales.dtype == torch.float32 and m.bias.dtype == torch.float32
    buf = io.BytesIO()
    torch.save(lin.state_dict(), buf)
    buf.seek(0)
    other = mxb.int8_linear(fake(3, 8), torch.zeros(3))
    other.load_state_dict(torch.load(buf))
    assert torch.equal(other.bias, lin.bias) and other.weight.shape == (3, 8)
    one = mxb.int8_linear(fake(3, 8, block=24))  # one scale for the whole weight
    assert one.weight_scales.shape == (3,)
    with pytest.raises(ValueError):
        lin(fake(2, 9))


def test_linear_module_checks_its_buffers():
    strided = torch.arange(6.0)[::2]
    assert torch.equal(mxb.int8_linear(fake(3, 8), strided).bias, strided)
    for bad in (torch.ones(2), torch.ones(3, 1), torch.ones(()), torch.ones(3, device="meta")):
        with pytest.raises(ValueError):
            mxb.int8_linear(fake(3, 8), bad)


def test_codes_made_in_inference_mode_leave_later_ones_usable():
    def inference(t):  # of the wrapper itself
        with torch._C.DisableTorchFunctionSubclass():
            return t.is_inference()

    with torch.inference_mode():
        fake(2, 8)
    later = fake(2, 8)
    assert not inference(later)
    with torch.inference_mode():
        assert not inference(mxb.mx_tensor(later.packed, later.mx_scales, mxb.int8d, (2, 8), 16, 8))
        assert inference(fake(2, 8))
    assert not inference(fake(2, 8))


@pytest.mark.gpu
def test_linear_module_with_assigned_buffers():
    lin = mxb.int8_linear.from_linear(torch.nn.Linear(64, 24, device="cuda"))
    x = rows(1, 5, 64)
    want = lin(x)
    state = {k: v.clone() for k, v in lin.state_dict().items()}
    wide = torch.zeros(48, device="cuda")
    wide[::2] = state["bias"]
    lin.bias = wide[::2]  # in steps
    assert torch.equal(lin(x), want)
    lin.bias = state["bias"].double()
    assert torch.equal(lin(x), want)
    lin.weight_codes = state["weight_codes"].t().contiguous().t()
    assert torch.equal(lin(x), want)
    for name, bad in (("bias", state["bias"][:23]), ("bias", state["bias"].cpu()),
                      ("weight_scales", state["weight_scales"].bfloat16()),
                      ("weight_scales", state["weight_scales"][:23]), ("weight_scales", state["weight_scales"].cpu()),
                      ("weight_codes", state["weight_codes"][:23]), ("weight_codes", state["weight_codes"].short())):
        for k, v in {**state, name: bad}.items():
            setattr(lin, k, v)
        with pytest.raises(ValueError):
            lin(x)
    for k, v in state.items():
        setattr(lin, k, v)
    assert torch.equal(lin(x), want)
    assert lin(x[:0]).shape == (0, 24) and torch.equal(lin(x[0]), want[0])
    with torch.inference_mode():
        assert torch.equal(lin(x), want)


# ── norm ─────────────────────────────────────────────────────────────────────
def norm64(x, w, r, eps):
    h = x.double() if r is None else x.double() + r.double()
    rms = torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    u = h * w.double()
    den = torch.maximum(u.abs().amax(-1, keepdim=True), 1e-12 * rms)
    return torch.round(127 * u / den), (den / rms / 127)[..., 0]


def check_norm(x, w, r=None, eps=1e-6):
    got = mxb.rms_norm_quantize(x, w, residual=r, eps=eps)
    if r is not None:
        got, h = got
        assert h.dtype == x.dtype and torch.equal(h, (x.float() + r.float()).to(x.dtype))
    code, scale = norm64(x, w, r, eps)
    assert got.shape == x.shape and got.mx_block == x.shape[-1] and got.mx_dtype.name == "int8d"
    codes = got.packed.view(x.shape)
    bad = codes.double() != code
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:3].tolist())
    # the sum of squares: at most 32 fused steps a thread and 10 of the tree, each
    # 2^-24, halved by the root; 2^-24 for the scale itself
    d = (got.mx_scales.view(scale.shape).double() - scale).abs()
    assert bool((d <= 2.0 ** -19 * scale).all())


def rows(seed, *shape, loud=True):
    g = torch.Generator("cuda").manual_seed(seed)
    x = torch.randn(*shape, generator=g, device="cuda")
    if loud:
        x *= 1 + 20 * (torch.rand(shape[-1], generator=g, device="cuda") < 0.02)
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,d", [(1, 1), (3, 7), (200, 8), (5, 64), (300, 100), (149, 256), (700, 512), (150, 1000),
                                 (2, 1024), (400, 1024), (33, 1999), (8, 4096), (500, 4096), (320, 8192), (3, 11008),
                                 (300, 11008), (297, 16384), (2, 16384), (299, 20000), (1, 20001), (300, 32768),
                                 (2, 32769)])
@pytest.mark.parametrize("residual", [False, True])
def test_norm(dtype, n, d, residual):
    x = rows(d, n, d).to(dtype)
    r = rows(d + 1, n, d).mul_(3).to(dtype) if residual else None
    w = (1 + 0.2 * rows(d + 2, d, loud=False)).to(dtype)
    check_norm(x, w, r)


@pytest.mark.gpu
def test_norm_many_values_next_to_borders():
    """Values k + 1/2 +- a few 2^-24 of a code, where fp32 alone rounds either way."""
    g = torch.Generator("cuda").manual_seed(0)
    k = torch.randint(-127, 127, (300, 4096), generator=g, device="cuda").double() + 0.5
    k = k * (1 + torch.randint(-4, 5, k.shape, generator=g, device="cuda") * 2.0 ** -24)
    k[:, 17] = 127.0
    w = 0.5 + torch.rand(4096, generator=g, device="cuda")
    check_norm((k / w.double()).float(), w)
    check_norm((k / w.double()).float(), w, rows(3, 300, 4096).mul_(1e-6))
    check_norm(k.float(), torch.ones(4096, device="cuda").bfloat16())  # ties among them


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(64, 24), (4, 3, 40)])
def test_norm_strides_types_and_alignment(shape):
    d = shape[-1]
    w = 1 + 0.2 * rows(1, d, loud=False)
    wide = rows(2, *shape[:-1], 3 * d)
    x, r = wide[..., d:2 * d], wide[..., 2 * d:]
    check_norm(x, w, r)
    check_norm(wide.bfloat16()[..., 1:d + 1], w.bfloat16(), wide.bfloat16()[..., 7:d + 7])  # unaligned
    check_norm(x, w.bfloat16())
    check_norm(wide.bfloat16()[..., :d], w)
    check_norm(x.transpose(0, -1).contiguous().transpose(0, -1), w)  # last dim strided
    check_norm(x[:1].expand(5, *shape[1:]), w)                       # rows that share memory
    h = x.half()
    a, b = mxb.rms_norm_quantize(h, w), mxb.rms_norm_quantize(h.float(), w)
    assert torch.equal(a.packed, b.packed) and torch.equal(a.mx_scales, b.mx_scales)
    a, s = mxb.rms_norm_quantize(h, w, residual=r)  # mixed types go through fp32
    b, t = mxb.rms_norm_quantize(h.float(), w, residual=r)
    assert torch.equal(a.packed, b.packed) and s.dtype == torch.float16 and torch.equal(s, t.half())
    a = mxb.rms_norm_quantize(x, w.double())
    assert torch.equal(a.packed, mxb.rms_norm_quantize(x, w).packed)
    e = mxb.rms_norm_quantize(x[..., :0, :] if len(shape) == 3 else x[:0], w)
    assert e.numel() == 0 and e.mx_scales.numel() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("n,d", [(3, 200), (400, 200), (2, 4096), (2, 40000)])
def test_norm_rows_outside_the_usual_range(n, d):
    w = torch.ones(d, device="cuda")
    base = rows(5, n, d)
    for size in (0.0, 1e-25, 1e-17, 1e-12, 1e15, 1e25, 1e36):
        check_norm(base * size, w)
        check_norm(base * size, w, eps=0.0) if size else None
    check_norm(base, w * 1e-20)     # under the scale's lower bound
    check_norm(base * 1e30, w * 1e30)  # products past fp32
    z = mxb.rms_norm_quantize(base * 0, w)
    assert not z.packed.any() and torch.equal(z.mx_scales, torch.full((n,), 1e-12 / 127, device="cuda"))
    x = base.clone()
    x[0, 3], x[1, d - 1] = float("nan"), float("-inf")
    z = mxb.rms_norm_quantize(x, w)
    assert z.mx_scales[:2].isnan().all() and not z.packed.view(n, d)[:2].any()
    if n > 2:
        assert z.mx_scales[2:].isfinite().all() and z.packed.view(n, d)[2:].any()
    assert mxb.rms_norm_quantize(base * 0, w, eps=0.0).mx_scales.isnan().all()  # 0 / 0


@pytest.mark.gpu
def test_norm_refusals_on_the_device():
    x, w = torch.zeros(2, 8, device="cuda"), torch.ones(8, device="cuda")
    for a in ((x, w[:7]), (x, w.cpu()), (x[0, 0], w), (x.int(), w), (x, w.int()), (x[:, :0], w[:0])):
        with pytest.raises(ValueError):
            mxb.rms_norm_quantize(*a)
    for kw in (dict(residual=x[:1]), dict(residual=x.cpu()), dict(residual=x.int()), dict(eps=-1e-6),
               dict(eps=float("nan"))):
        with pytest.raises(ValueError):
            mxb.rms_norm_quantize(x, w, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("n,d,dtype", [(8, 4096, torch.bfloat16), (500, 1000, torch.float32), (700, 512, torch.bfloat16)])
def test_norm_repeats_on_any_stream_and_in_a_graph(n, d, dtype):
    x, r, w = rows(1, n, d).to(dtype), rows(2, n, d).to(dtype), 1 + 0.1 * rows(3, d, loud=False)
    want, sum_ = mxb.rms_norm_quantize(x, w, residual=r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [mxb.rms_norm_quantize(x, w, residual=r) for _ in range(10)]
    here = [mxb.rms_norm_quantize(x, w, residual=r) for _ in range(10)]
    torch.cuda.synchronize()
    for q, s in got + here:
        assert torch.equal(q.packed, want.packed) and torch.equal(q.mx_scales, want.mx_scales)
        assert torch.equal(s, sum_)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, s = mxb.rms_norm_quantize(x, w, residual=r)
        y = q.dequantize()
    x0 = x.clone()
    x.copy_(r)
    graph.replay()
    other, _ = mxb.rms_norm_quantize(x, w, residual=r)
    assert torch.equal(q.packed, other.packed) and torch.equal(y, other.dequantize())
    x.copy_(x0)
    graph.replay()
    assert torch.equal(q.packed, want.packed) and torch.equal(s, sum_) and torch.equal(y, want.dequantize())


# ── product ──────────────────────────────────────────────────────────────────
def operand(n, k, seed, block=None, full=False):
    g = torch.Generator("cuda").manual_seed(seed)
    codes = torch.randint(-128 if full else -127, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
    count = n if block is None else 1
    scales = torch.rand(count, generator=g, device="cuda") * 0.02 + 1e-3
    return mxb.mx_tensor(codes.view(-1), scales, mxb.int8d, (n, k), n * k, k if block is None else max(n * k, 1))


def product_ref(a, b, bias, dtype):
    """The integer sum exactly, then the documented roundings."""
    (M, K), N = a.shape, b.shape[0]
    p = torch.mm(a.packed.view(M, K).double(), b.packed.view(N, K).double().t())
    y = p.float() * a.mx_scales.view(-1, 1) * b.mx_scales.view(1, -1)
    return (y if bias is None else y + bias).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,k,n", [
    (1, 1, 1), (2, 15, 5), (1, 16, 8), (3, 31, 127), (16, 128, 128), (17, 129, 130), (33, 257, 64), (1, 4096, 1000),
    (64, 1000, 96), (65, 640, 200), (5, 11008, 300), (128, 512, 256), (129, 130, 1), (200, 2048, 1000),
    (300, 4096, 130), (1000, 333, 257), (513, 1024, 640), (1, 2048, 11008), (2300, 64, 64), (700, 1600, 1928),
    (2048, 1024, 2048), (1111, 4096, 3000)])
def test_product(out, m, k, n):
    a, b = operand(m, k, m + k), operand(n, k, n, full=True)
    bias = torch.randn(n, generator=torch.Generator("cuda").manual_seed(1), device="cuda") if (m + n) % 2 else None
    y = mxb.int8_matmul(a, b, bias=bias, out_dtype=out)
    assert y.shape == (m, n) and torch.equal(y, product_ref(a, b, bias, out))
    assert L.load().mxb_device_error(1) == 0


@pytest.mark.gpu
def test_product_largest_sums():
    k = 131071
    a = mxb.mx_tensor(torch.full((2 * k,), -128, dtype=torch.int8, device="cuda"), torch.ones(2, device="cuda"),
                      mxb.int8d, (2, k), 2 * k, k)
    y = mxb.int8_matmul(a, a, out_dtype=torch.float32)
    assert torch.equal(y, torch.full((2, 2), float(2 ** 14 * k), device="cuda"))


@pytest.mark.gpu
def test_product_scales_layouts_and_empty():
    m, k, n = 40, 272, 100
    for ba, bb in ((None, 1), (1, None), (1, 1)):
        a, b = operand(m, k, 1, ba), operand(n, k, 2, bb)
        assert torch.equal(mxb.int8_matmul(a, b), product_ref(a, b, None, torch.bfloat16))
    a, b = operand(m, k, 1), operand(n, k, 2)
    want = mxb.int8_matmul(a, b)
    lead = mxb.mx_tensor(a.packed, a.mx_scales, mxb.int8d, (4, 10, k), m * k, k)
    assert torch.equal(mxb.int8_matmul(lead, b), want.view(4, 10, n))
    row = mxb.mx_tensor(a.packed[:k], a.mx_scales[:1], mxb.int8d, (k,), k, k)
    assert torch.equal(mxb.int8_matmul(row, b), want[0])
    for at in (1, 4, 8):  # codes that do not start at a multiple of 16 bytes
        moved = torch.empty(m * k + at, dtype=torch.int8, device="cuda")[at:].copy_(a.packed)
        am = mxb.mx_tensor(moved, a.mx_scales, mxb.int8d, (m, k), m * k, k)
        assert torch.equal(mxb.int8_matmul(am, b), want)
    bias = torch.arange(n, device="cuda").bfloat16()
    assert torch.equal(mxb.int8_matmul(a, b, bias=bias), product_ref(a, b, bias.float(), torch.bfloat16))
    assert mxb.int8_matmul(operand(0, k, 1), b).shape == (0, n) and mxb.int8_matmul(a, operand(0, k, 1)).shape == (m, 0)
    z = mxb.int8_matmul(operand(3, 0, 1, 1), operand(n, 0, 1, 1), bias=bias)
    assert torch.equal(z, bias.expand(3, n))
    for bad in (bias[:-1], bias.cpu()):
        with pytest.raises(ValueError):
            mxb.int8_matmul(a, b, bias=bad)


@pytest.mark.gpu
def test_product_odd_scales():
    """Scales that are infinite, NaN, zero or negative act on their rows alone."""
    a, b = operand(6, 64, 3), operand(130, 64, 4)
    for i, s in enumerate((float("inf"), float("nan"), 0.0, -1.0, 1e-40)):
        a.mx_scales[i] = s
        b.mx_scales[20 * i] = s
    y, want = mxb.int8_matmul(a, b, out_dtype=torch.float32), product_ref(a, b, None, torch.float32) + 0.0
    assert torch.equal(y.nan_to_num(7.0), want.nan_to_num(7.0)) and torch.equal(y.isnan(), want.isnan())


@pytest.mark.gpu
def test_product_repeats_on_any_stream_and_in_a_graph():
    a, b = operand(70, 4096, 1), operand(1000, 4096, 2)
    c, e = operand(600, 1003, 3), operand(700, 1003, 4)
    want, want2 = product_ref(a, b, None, torch.bfloat16), product_ref(c, e, None, torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ys = [mxb.int8_matmul(a, b) for _ in range(20)]
        zs = [mxb.int8_matmul(c, e) for _ in range(20)]
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in ys) and all(torch.equal(z, want2) for z in zs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, z = mxb.int8_matmul(a, b), mxb.int8_matmul(c, e)
    for _ in range(3):
        y.zero_()
        z.zero_()
        graph.replay()
        assert torch.equal(y, want) and torch.equal(z, want2)


@pytest.mark.gpu
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,k,n", [(2048, 2048, 2048), (2305, 1000, 2184)])
def test_product_of_many_tokens(out, m, k, n):
    """The kernel of CTA pairs: two at once on two streams, in a graph, one scale for all,
    and the operands that it leaves to the other one (scales and bias in steps of 4 bytes)."""
    a, b = operand(m, k, 1), operand(n, k, 2, full=True)
    bias = torch.randn(n, generator=torch.Generator("cuda").manual_seed(1), device="cuda")
    want = product_ref(a, b, bias, out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ys = [mxb.int8_matmul(a, b, bias=bias, out_dtype=out) for _ in range(5)]
    ys += [mxb.int8_matmul(a, b, bias=bias, out_dtype=out) for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in ys)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = mxb.int8_matmul(a, b, bias=bias, out_dtype=out)
    for _ in range(2):
        y.zero_()
        graph.replay()
        assert torch.equal(y, want)
    off = torch.empty(n + 1, device="cuda")[1:]
    assert torch.equal(mxb.int8_matmul(a, b, bias=off.copy_(bias), out_dtype=out), want)
    at = torch.empty(n + 1, device="cuda")[1:].copy_(b.mx_scales)
    moved = mxb.mx_tensor(b.packed, at, mxb.int8d, (n, k), n * k, k)
    assert torch.equal(mxb.int8_matmul(a, moved, bias=bias, out_dtype=out), want)
    one = mxb.mx_tensor(b.packed, b.mx_scales[:1], mxb.int8d, (n, k), n * k, n * k)
    for p, q in ((a, one), (mxb.mx_tensor(a.packed, a.mx_scales[5:6], mxb.int8d, (m, k), m * k, m * k), b)):
        assert torch.equal(mxb.int8_matmul(p, q, out_dtype=out), product_ref(p, q, None, out))
    assert L.load().mxb_device_error(1) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", [(5, 300, 70), (64, 1024, 512), (200, 2000, 130)])
def test_fused_int8_linear_of_row_scales(m, k, n):
    """The framework's fp32 linear of the same operands is this product."""
    x, w = rows(1, m, k), rows(2, n, k) * 0.02
    qx, qw = mxb.dynamic_quantize(x, "int8d", "per_token"), mxb.dynamic_quantize(w, "int8d", "per_token")
    bias = rows(3, n, loud=False)
    assert torch.equal(mxb.fused_int8_linear(qx, qw, bias), product_ref(qx, qw, bias, torch.float32))


@pytest.mark.gpu
def test_linear_module():
    lin = torch.nn.Linear(320, 200, device="cuda")
    layer = mxb.int8_linear.from_linear(lin)
    x = rows(4, 3, 7, 320).bfloat16()
    q = mxb.dynamic_quantize(x, "int8d", "per_token")
    y = layer(x)
    assert y.shape == (3, 7, 200) and y.dtype == torch.bfloat16 and torch.equal(y, layer(q))
    flat = mxb.mx_tensor(q.packed, q.mx_scales, mxb.int8d, (21, 320), 21 * 320, 320)
    assert torch.equal(y.view(21, 200), product_ref(flat, layer.weight, lin.bias.detach(), torch.bfloat16))
    want = lin(x.float())
    # each operand is off by half a code of its row's largest value
    ax, aw = x.float().abs(), lin.weight.abs()
    tol = (ax.amax(-1, keepdim=True) / 254 * aw.sum(1) + ax.sum(-1, keepdim=True) * aw.amax(1) / 254
           + 320 * ax.amax(-1, keepdim=True) * aw.amax(1) / 254 ** 2)
    assert bool(((y.float() - want).abs() <= 1.01 * tol + 2.0 ** -8 * want.abs() + 1e-5).all())


@pytest.mark.gpu
def test_norm_into_linear():
    """A layer's norm, its product and the residual that goes on."""
    x, h, w = (rows(i, 40, 512).bfloat16() for i in range(3))
    weight = 1 + 0.1 * rows(5, 512, loud=False).bfloat16()
    layer = mxb.int8_linear(mxb.dynamic_quantize(w, "int8d", "per_token"))
    a, h2 = mxb.rms_norm_quantize(x, weight, residual=h)
    code, scale = norm64(x, weight, h, 1e-6)
    y = layer(a)
    ref = torch.mm(code, layer.weight_codes.double().t()) * scale[:, None] * layer.weight_scales.double()
    # the scale is off by 2^-19, the roundings of the product are three of 2^-24 and one of 2^-8
    assert bool(((y.double() - ref).abs() <= (2.0 ** -8 + 2.0 ** -18) * ref.abs()).all())
    assert torch.equal(h2, x + h)


@pytest.mark.gpu
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,k,n", [(9, 128, 128), (16, 4096, 384), (17, 96, 640), (25, 8192, 256), (32, 256, 40000),
                                   (12, 2048, 19000)])
def test_product_of_narrow_tiles_beside_others(out, m, k, n):
    """Tiles of 16 and 32 tokens, with and without splits, while other products hold
    accumulators on the same SMs."""
    a, b = operand(m, k, 1), operand(n, k, 2, full=True)
    c, e = operand(100, 1024, 3), operand(900, 1024, 4)
    want, want2 = product_ref(a, b, None, out), product_ref(c, e, None, out)
    streams = [torch.cuda.Stream() for _ in range(3)]
    ys, zs = [], []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(8):
        for s in streams[:2]:
            with torch.cuda.stream(s):
                ys.append(mxb.int8_matmul(a, b, out_dtype=out))
        with torch.cuda.stream(streams[2]):
            zs.append(mxb.int8_matmul(c, e, out_dtype=out))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in ys) and all(torch.equal(z, want2) for z in zs)
    assert L.load().mxb_device_error(1) == 0


def plain_use(t):
    """Of the wrapper itself."""
    with torch._C.DisableTorchFunctionSubclass():
        return t.detach().untyped_storage().data_ptr(), t._version


@pytest.mark.parametrize("mode", ["fake", "grad", "jvp", "functionalize"])
def test_first_codes_made_under_a_mode_leave_later_ones_usable(mode):
    code = """if True:
    import sys, torch
    import qtpytorch_b200 as mxb
    from torch._subclasses.fake_tensor import FakeTensorMode

    codes, scales = torch.zeros(16, dtype=torch.int8), torch.ones(2)
    def make():
        return mxb.mx_tensor(codes, scales, mxb.int8d, (2, 8), 16, 8)
    def inside(x):
        make()
        return x.sum()
    def fake(x):
        with FakeTensorMode():
            try:
                make()
            except RuntimeError:  # real codes have no wrapper there
                pass
    modes = dict(fake=fake, grad=torch.func.grad(inside), functionalize=torch.func.functionalize(inside),
                 jvp=lambda x: torch.func.jvp(inside, (x,), (x,)))
    modes[sys.argv[1]](torch.ones(3))
    t = make()
    with torch._C.DisableTorchFunctionSubclass():
        t = t.detach()
        assert not torch._is_functional_tensor(t)
        t.untyped_storage().data_ptr()
    """
    subprocess.run([sys.executable, "-W", "ignore", "-c", code, mode], check=True, timeout=300,
                   cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


def test_wrappers_share_neither_memory_nor_versions():
    a, b = fake(2, 8), fake(2, 8)
    assert plain_use(a)[0] != plain_use(b)[0]
    with torch._C.DisableTorchFunctionSubclass():
        a.zero_()
    assert plain_use(a)[1] == 1 and plain_use(b)[1] == 0

    class keep(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, w):
            ctx.save_for_backward(w)
            return 2 * x

        @staticmethod
        def backward(ctx, g):
            assert ctx.saved_tensors[0].shape == (2, 8)
            return 2 * g, None

    x = torch.ones(2, requires_grad=True)
    y = keep.apply(x, b)
    with torch._C.DisableTorchFunctionSubclass():
        a.zero_()
    y.sum().backward()
    assert torch.equal(x.grad, torch.full((2,), 2.0))


def test_fused_int8_linear_refuses_the_cpu():
    for block in (None, 4):  # a scale a row, and blocks of K
        with pytest.raises(L.MxbError):
            mxb.fused_int8_linear(fake(2, 8, block), fake(3, 8, block))


def test_operands_that_are_not_whole_are_refused():
    """Before any device is looked at: their addresses would go to a kernel as they are."""
    codes, ones = torch.zeros(24, dtype=torch.int8), torch.ones(3)
    good = fake(3, 8)
    for bad in (mxb.mx_tensor(codes, ones.to("meta"), mxb.int8d, (3, 8), 24, 8),  # scales elsewhere
                mxb.mx_tensor(codes[:23], ones, mxb.int8d, (3, 8), 24, 8),        # a code short
                mxb.mx_tensor(codes, ones, mxb.int8d, (6, 8), 24, 8),             # another shape
                mxb.mx_tensor(codes, ones[:1], mxb.int8d, (3, 8), 48, 48)):
        for a, b in ((good, bad), (bad, good)):
            with pytest.raises(ValueError):
                mxb.int8_matmul(a, b)
        with pytest.raises(ValueError):
            mxb.int8_linear(bad)
        with pytest.raises(ValueError):
            mxb.int8_linear(good)(bad)


@pytest.mark.gpu
def test_fused_int8_linear_takes_scales_from_the_host():
    a, b = operand(5, 96, 1), operand(7, 96, 2)
    want = product_ref(a, b, None, torch.float32)
    for p, q in ((a, mxb.mx_tensor(b.packed, b.mx_scales.cpu(), mxb.int8d, (7, 96), 672, 96)),
                 (mxb.mx_tensor(a.packed, a.mx_scales.cpu(), mxb.int8d, (5, 96), 480, 96), b)):
        assert torch.equal(mxb.fused_int8_linear(p, q), want)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 2048, 40000])
def test_norm_codes_are_those_of_64_bits(d):
    """A residual too small for a double's sum makes a tie, as the documentation says; one
    that it holds does not."""
    x = torch.zeros(3, d, device="cuda")
    x[:, 0], x[:, 1], x[:, 2] = 127.0, 0.5, 2.5
    r = torch.zeros_like(x)
    r[0, 1:3], r[1, 1:3] = 2.0 ** -60, 2.0 ** -40
    for t in (torch.float32, torch.bfloat16):
        q, _ = mxb.rms_norm_quantize(x.to(t), torch.ones(d, device="cuda", dtype=t), residual=r.to(t))
        assert q.packed.view(3, d)[:, :3].tolist() == [[127, 0, 2], [127, 1, 3], [127, 0, 2]]
        check_norm(x.to(t), torch.ones(d, device="cuda", dtype=t), r.to(t))


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(3, 40), (300, 128), (2048, 2048)])
def test_product_rounds_sums_past_24_bits(m, n):
    """Each step of the documented formula by itself, P = 2^24 + 3 among the sums."""
    k = 4096
    code = torch.zeros(k, dtype=torch.int8, device="cuda")
    code[:2047] = 127
    p = int((code.long() ** 2).sum())  # under 2^25, and no multiple of 2
    a = code.repeat(m, 1)
    a[1:, 2047:] = torch.randint(-127, 128, (m - 1, k - 2047), generator=torch.Generator().manual_seed(3)).to(a)
    b = code.repeat(n, 1)
    b[:, 4095] = torch.arange(n) % 100
    sa, sb = (0.1 + torch.rand(x, generator=torch.Generator().manual_seed(x)).cuda() for x in (m, n))
    assert p > 1 << 24 and p % 2 == 1
    bias = torch.linspace(-3, 3, n, device="cuda")
    qa, qb = (mxb.mx_tensor(t.reshape(-1), s, mxb.int8d, t.shape, t.numel(), k) for t, s in ((a, sa), (b, sb)))
    y = mxb.int8_matmul(qa, qb, bias=bias, out_dtype=torch.float32)
    exact = torch.mm(a.double(), b.double().t())
    one = exact.to(torch.float32)
    assert bool((one.double() != exact).any())
    two = (one.double() * sa.double()[:, None]).to(torch.float32)
    three = (two.double() * sb.double()).to(torch.float32)
    assert torch.equal(y, (three.double() + bias.double()).to(torch.float32))


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", [(1, 4096, 4736), (30, 4000, 4700), (64, 8192, 4992), (2, 4096, 11520), (7, 4096, 11648),
                                   (1, 4096, 4224), (20, 4096, 7000), (1, 2048, 18944)])
def test_product_of_as_many_splits_as_clusters_fit(m, k, n):
    a, b = operand(m, k, 1), operand(n, k, 2, full=True)
    assert torch.equal(mxb.int8_matmul(a, b), product_ref(a, b, None, torch.bfloat16))


@pytest.mark.gpu
def test_quantized_tensors_are_taken_by_their_values():
    x, r, w, bias = (mxb.mx_tensor.quantize(rows(i, *s), "int8d", 64)
                     for i, s in enumerate([(40, 512), (40, 512), (512,), (24,)]))
    got, h = mxb.rms_norm_quantize(x, w, residual=r)
    want, h2 = mxb.rms_norm_quantize(x.dequantize(), w.dequantize(), residual=r.dequantize())
    assert torch.equal(got.packed, want.packed) and torch.equal(got.mx_scales, want.mx_scales) and torch.equal(h, h2)
    a, b = operand(5, 64, 1), operand(24, 64, 2)
    assert torch.equal(mxb.int8_matmul(a, b, bias=bias), mxb.int8_matmul(a, b, bias=bias.dequantize()))
    assert torch.equal(mxb.int8_linear(b, bias)(a), mxb.int8_matmul(a, b, bias=bias.dequantize()))


def test_norm_outputs_over_its_inputs_are_refused():
    """Values next to a border are read again after the codes are written."""
    lib = L.load()

    def norm(x, r, w, codes, scales, h, rows=2, d=64):
        x, r, w, codes, scales, h = (ctypes.c_void_p(p) if p else None for p in (x, r, w, codes, scales, h))
        return lib.mxb_rms_norm_quantize(x, r, 1, rows, d, 64, 64, w, 1, 1e-6, codes, scales, h, None)

    # x, residual: 256 bytes each; weight 128; codes 128, scales 8, sum 256
    at = dict(x=0x1000, r=0x2000, w=0x3000, codes=0x4000, scales=0x5000, h=0x6000)
    for over in (dict(codes=0x1000), dict(codes=0x10ff), dict(codes=0x0f81), dict(codes=0x2000), dict(codes=0x307f),
                 dict(scales=0x10fc), dict(scales=0x1ffc), dict(scales=0x3000), dict(h=0x2f02), dict(h=0x20fe)):
        assert norm(**{**at, **over}) == -6, over
