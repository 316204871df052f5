"""Keys and queries rotated on their way into the paged cache, against 64 bits: the
codes and scales are those of ``write`` fed the rotation in 64 bits rounded to fp32,
bit for bit."""
import ctypes

import pytest
import torch

import qtpytorch_b200 as mxb
from qtpytorch_b200 import _lib as L


# ── host ─────────────────────────────────────────────────────────────────────
def test_argument_errors_need_no_gpu():
    lib, p = L.load(), ctypes.c_void_p(32)

    def append(q=p, k=p, v=p, dt=1, T=2, Hq=4, heads=2, dim=128, pos=p, axes=1, freq=p, rot=128, sections=None,
               slots=p, pages=4, page=16, bits=8, kc=p, out=p):
        s = None if sections is None else (ctypes.c_int * len(sections))(*sections)
        return lib.mxb_kv_append(q, k, v, dt, T, Hq, heads, dim, 512, 128, 256, 128, 256, 128, pos, axes, 2, freq, rot,
                                 s, 0, slots, pages, page, bits, kc, p, p, p, out, None)

    assert append(dt=7) == -2 and append(bits=2) == -2
    assert append(dim=96) == -1 and append(page=24) == -1 and append(pages=0) == -1 and append(T=-1) == -1
    assert append(rot=130) == -1 and append(rot=12) == -1 and append(rot=-8) == -1 and append(Hq=-1) == -1
    assert append(axes=0) == -1 and append(axes=5) == -1 and append(Hq=65536) == -1
    assert append(axes=2) == -6 and append(axes=2, sections=[32, 31]) == -1 and append(axes=2, sections=[65, -1]) == -1
    big = 2 ** 31 - 1
    assert append(axes=4, sections=[big, big, 2, 64]) == -1
    for kw in (dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(pos=None), dict(freq=None),
               dict(slots=None), dict(kc=None)):
        assert append(**kw) == -6
    for kw in (dict(q=33), dict(k=33), dict(v=33), dict(out=40), dict(pos=36), dict(slots=36), dict(freq=34), dict(kc=8)):
        assert append(**{n: ctypes.c_void_p(x) for n, x in kw.items()}) == -3
    assert append(T=0) == 0 and append(T=0, axes=2, sections=[0, 64]) == 0


def test_refusals():
    c = mxb.paged_kv_cache(4, 2, 64, "int8d", 16, device="cpu")
    z = torch.zeros(1, 2, 64)
    with pytest.raises(L.MxbError):
        c.append(z, z, torch.zeros(1).long(), torch.zeros(1).long(), torch.ones(32))


@pytest.mark.gpu
def test_refusals_on_the_device():
    c = mxb.paged_kv_cache(4, 2, 64, "int8d", 16)
    z = torch.zeros(3, 2, 64, device="cuda")
    n = torch.zeros(3, dtype=torch.long, device="cuda")
    f = torch.ones(32, device="cuda")
    ok = dict(k=z, v=z, slots=n, positions=n, inv_freq=f, q=z)
    c.append(**dict(ok, slots=n - 1))
    for kw in (dict(k=z[:2]), dict(k=z[..., :32], v=z[..., :32]), dict(slots=n[:2]), dict(slots=n.float()),
               dict(positions=n[:2]), dict(positions=n.float()), dict(positions=n[None]), dict(inv_freq=f[:31]),
               dict(inv_freq=torch.ones(36, device="cuda")), dict(inv_freq=f.long()), dict(inv_freq=f[None]),
               dict(q=z[:2]), dict(q=z[..., :32]), dict(q=z[0]), dict(q=z.cpu()), dict(k=z.cpu(), v=z.cpu()),
               dict(positions=n.cpu()), dict(inv_freq=f.cpu()), dict(slots=n.cpu()), dict(sections=[16, 16]),
               dict(sections=[16, 15], positions=n.expand(2, 3)), dict(sections=[], positions=n[:0]),
               dict(sections=[33, -1], positions=n.expand(2, 3)),
               dict(sections=[8, 8, 8, 4, 4], positions=n.expand(5, 3))):
        with pytest.raises(ValueError):
            c.append(**dict(ok, **kw))


# ── rotation ─────────────────────────────────────────────────────────────────
def turned64(x, positions, inv_freq, sections, interleaved):
    """x [T, heads, dim] rotated in 64 bits, pair by pair."""
    x = x.double().clone()
    pairs = inv_freq.shape[0]
    where = positions.double().reshape(-1, x.shape[0])
    axis = [0] * pairs if sections is None else [a for a, n in enumerate(sections) for _ in range(n)]
    for i in range(pairs):
        t = where[axis[i]] * inv_freq[i].double()
        c, s = t.cos()[:, None], t.sin()[:, None]
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + pairs)
        x[..., a], x[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    return x


def same(c, d):
    return all(torch.equal(a, b) for a, b in ((c.k_codes, d.k_codes), (c.k_scales, d.k_scales),
                                              (c.v_codes, d.v_codes), (c.v_scales, d.v_scales)))


def check(k, v, q, slots, positions, inv_freq, dtype, page, pages, sections=None, interleaved=False):
    heads, dim = k.shape[1:]
    c, d = (mxb.paged_kv_cache(pages, heads, dim, dtype, page) for _ in range(2))
    got = c.append(k, v, slots, positions, inv_freq, q=q, sections=sections, interleaved=interleaved)
    d.write(turned64(k, positions, inv_freq, sections, interleaved).float(), v.float(), slots)
    assert same(c, d)
    if q is None:
        assert got is None
    else:
        want = turned64(q, positions, inv_freq, sections, interleaved)
        pairs = inv_freq.shape[0]
        size = q.double().abs().amax(-1, keepdim=True) * (2 if pairs else 0)
        # a cosine, a product and a sum of 2^-24 each on both elements, then the type's rounding
        eps = torch.finfo(q.dtype).eps / 2
        assert got.dtype == q.dtype and got.is_contiguous()
        assert bool(((got.double() - want).abs() <= eps * want.abs() + 4 * 2.0 ** -24 * size).all())
    assert L.load().mxb_device_error(1) == 0
    return c


def inputs(T, heads, group, dim, seed, dtype=torch.bfloat16):
    g = torch.Generator("cuda").manual_seed(seed)
    q, k, v = (torch.randn(T, h, dim, generator=g, device="cuda") for h in (heads * group, heads, heads))
    k *= 1 + 6 * (torch.rand(heads, dim, generator=g, device="cuda") < 0.05)
    return q.to(dtype), k.to(dtype), v.to(dtype), torch.randperm(2 * T + 16, generator=g, device="cuda")[:T]


def freqs(pairs, theta=500000.0):
    return (theta ** (-torch.arange(pairs, dtype=torch.float64) / max(pairs, 1))).float().cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["int8d", "int4d"])
@pytest.mark.parametrize("inp", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,heads,group,dim,pairs,page,far", [
    (1, 1, 1, 64, 32, 16, 0), (1, 8, 4, 128, 64, 64, 100), (5, 2, 3, 128, 64, 16, 1 << 20), (33, 4, 1, 64, 32, 32, 7),
    (70, 3, 5, 128, 32, 128, 30000), (600, 1, 4, 64, 20, 16, 0), (1300, 2, 2, 128, 52, 64, (1 << 31) - 5000),
    (9, 2, 2, 64, 0, 16, 3), (2500, 5, 1, 128, 64, 16, 100000)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append(dtype, inp, T, heads, group, dim, pairs, page, far, interleaved):
    q, k, v, slots = inputs(T, heads, group, dim, T, inp)
    pos = far + torch.arange(T, device="cuda")
    check(k, v, q, slots, pos, freqs(pairs), dtype, page, -(-(2 * T + 16) // page), interleaved=interleaved)


@pytest.mark.gpu
@pytest.mark.parametrize("sections", [[16, 24, 24], [64], [0, 64], [1, 2, 61], [30, 0, 17, 17], [63, 1]])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_of_several_axes(sections, interleaved):
    T = 300
    q, k, v, slots = inputs(T, 2, 3, 128, 5)
    g = torch.Generator("cuda").manual_seed(2)
    pos = torch.randint(-50, 5000, (len(sections), T), generator=g, device="cuda")
    check(k, v, q, slots, pos, freqs(64, 10000.0), "int8d", 32, 20, sections, interleaved)
    check(k, v, None, slots, pos, freqs(64, 10000.0), "int4d", 32, 20, sections, interleaved)


@pytest.mark.gpu
def test_append_strides_types_and_alignment():
    T, D = 21, 64
    g = torch.Generator("cuda").manual_seed(9)
    qkv = torch.randn(T, 8, D, generator=g, device="cuda").bfloat16()
    slots, pos = torch.arange(3, 3 + T, device="cuda"), torch.arange(T, device="cuda") * 31
    f = freqs(32)
    c = check(qkv[:, 4:6], qkv[:, 6:], qkv[:, :4], slots, pos, f, "int8d", 16, 4)  # slices of one projection
    heads_first = qkv.transpose(0, 1).contiguous().transpose(0, 1)
    last = qkv.transpose(1, 2).contiguous().transpose(1, 2)
    odd = torch.empty(T * 8 * D + 1, device="cuda", dtype=torch.bfloat16)[1:].view(T, 8, D).copy_(qkv)
    for x in (heads_first, last, odd):
        assert same(c, check(x[:, 4:6], x[:, 6:], x[:, :4], slots, pos, f, "int8d", 16, 4))
    assert same(c, check(qkv[:, 4:6], qkv[:, 6:], qkv[:, :4], slots.int(), pos.int(), f.double(), "int8d", 16, 4))
    assert same(c, check(qkv[:, 4:6].float(), qkv[:, 6:], qkv[:, :4], slots, pos, f, "int8d", 16, 4))
    d = mxb.paged_kv_cache(4, 2, D, "int8d", 16)
    q = d.append(qkv[:, 4:6], qkv[:, 6:], slots, pos, f, q=qkv[:, :4].half())
    assert q.dtype == torch.float16 and same(c, d)
    every = torch.stack((pos, pos, pos), -1).t()  # a row an axis, its elements apart
    assert same(c, check(qkv[:, 4:6], qkv[:, 6:], qkv[:, :4], slots, every, f, "int8d", 16, 4, [8, 8, 16]))
    one = pos[:1].expand(T)  # one position for all
    check(qkv[:, 4:6], qkv[:, 6:], qkv[:, :4], slots, one, f, "int4d", 16, 4)
    none = d.append(qkv[:0, 4:6], qkv[:0, 6:], slots[:0], pos[:0], f, q=qkv[:0, :4])
    assert none.shape == (0, 4, D)


@pytest.mark.gpu
def test_append_skips_padding_and_records_bad_slots():
    q, k, v, _ = inputs(6, 2, 2, 128, 4)
    pos, f = torch.arange(6, device="cuda"), freqs(64)
    c, d = (mxb.paged_kv_cache(4, 2, 128, "int8d", 16) for _ in range(2))
    L.load().mxb_device_error(1)
    slots = torch.tensor([5, -1, 64, 9, -(1 << 40), 1 << 40], device="cuda")
    got = c.append(k, v, slots, pos, f, q=q)
    assert L.load().mxb_device_error(1) == 8
    d.append(k[::3], v[::3], slots[::3], pos[::3], f)
    assert same(c, d)
    assert torch.equal(got, c.append(k, v, torch.full_like(slots, -1), pos, f, q=q)) and same(c, d)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["int8d", "int4d"])
def test_append_odd_rows(dtype):
    """Zero rows, tiny and huge ones; infinities and NaN stay in their rows."""
    T = 12
    q, k, v, _ = inputs(T, 1, 1, 64, 8, torch.float32)
    k[0], v[0] = 0, 0
    for i, s in enumerate((1e-38, 1e-20, 1e-13, 1e20, 1e37)):
        k[1 + i] *= s
    slots, pos, f = torch.arange(T, device="cuda"), torch.arange(T, device="cuda") + 3, freqs(32)
    check(k, v, q, slots, pos, f, dtype, 16, 1)
    k[7, 0, 5], k[8, 0, 40], v[9, 0, 1] = float("inf"), float("nan"), float("-inf")
    c = mxb.paged_kv_cache(1, 1, 64, dtype, 16)
    c.append(k, v, slots, pos, f)
    kk, vv = c.read(torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.tensor([T], device="cuda"), T,
                    torch.float32)
    assert kk[0, 7:9].isnan().all() and kk[0, :7].isfinite().all() and kk[0, 9:].isfinite().all()
    assert vv[0, 9].isnan().all() and vv[0, :9].isfinite().all() and vv[0, 10:].isfinite().all()


@pytest.mark.gpu
def test_append_keys_next_to_borders():
    """Rows whose rotated values lie within a few 2^-24 of a border between codes."""
    g = torch.Generator("cuda").manual_seed(0)
    T = 2000
    want = torch.randint(-127, 127, (T, 2, 128), generator=g, device="cuda").double() + 0.5
    want *= 1 + torch.randint(-4, 5, want.shape, generator=g, device="cuda") * 2.0 ** -24
    want[:, :, 9] = 127.0
    pos, f = torch.arange(T, device="cuda") + 77, freqs(64)
    k = turned64(want, -pos, f, None, False).float()  # turned back, so that the rotation gives it
    _, _, v, slots = inputs(T, 2, 1, 128, 3, torch.float32)
    check(k, v, None, slots, pos, f, "int8d", 64, 64)


@pytest.mark.gpu
def test_append_on_another_stream_and_in_a_graph():
    q, k, v, slots = inputs(50, 4, 2, 128, 6)
    pos, f = torch.arange(50, device="cuda"), freqs(64)
    c = mxb.paged_kv_cache(8, 4, 128, "int8d", 16)
    want = c.append(k, v, slots, pos, f, q=q)
    d, e = (mxb.paged_kv_cache(8, 4, 128, "int8d", 16) for _ in range(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = d.append(k, v, slots, pos, f, q=q)
    torch.cuda.synchronize()
    assert same(c, d) and torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = e.append(k, v, slots, pos, f, q=q)
    graph.replay()
    assert same(c, e) and torch.equal(got, want)


@pytest.mark.gpu
def test_quantized_keys_values_and_queries_are_taken_by_their_values():
    """Outputs of the packed product are such tensors."""
    g = torch.Generator("cuda").manual_seed(0)
    q, k, v = (mxb.mx_tensor.quantize(torch.randn(20, n, 64, generator=g, device="cuda"), "int8d", 64)
               for n in (4, 2, 2))
    slots, pos = torch.arange(20, device="cuda"), torch.arange(20, device="cuda") + 5
    freq = 10000.0 ** (-torch.arange(32, device="cuda") / 32)
    made = []
    for f in (lambda t: t, lambda t: t.dequantize()):
        c = mxb.paged_kv_cache(2, 2, 64, "int8d", 16)
        out = c.append(f(k), f(v), slots, pos, freq, q=f(q))
        d = mxb.paged_kv_cache(2, 2, 64, "int8d", 16)
        d.write(f(k), f(v), slots)
        made.append((out, c.k_codes, c.k_scales, c.v_codes, c.v_scales, d.k_codes, d.v_codes))
    assert all(torch.equal(x, y) for x, y in zip(*made))
