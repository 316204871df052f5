"""Attention of a tree of drafted tokens over the paged cache, against 64 bits: masks
that leave rows empty, sequences shorter than their trees, a shared prefix, hidden
places that hold NaN; and the layer in which it runs."""
import ctypes
import math

import pytest
import torch

import qtpytorch_b200 as mxb
from qtpytorch_b200 import _lib as L
from test_paged import history, pool, tables


# ── host ─────────────────────────────────────────────────────────────────────
def test_argument_errors_need_no_gpu():
    lib, p = L.load(), ctypes.c_void_p(32)

    def attend(B=2, T=3, group=4, width=3, mask=p, q=p, ws=None, n=0, prefix=0, pw=0, pt=None):
        return lib.mxb_tree_attention(q, B, T, 2, group, 128, p, p, p, p, 4, 16, 8, p, width, p, pt, pw, prefix, mask,
                                      9, 3, 0.1, p, None, ws, n, None)

    assert attend(mask=None) == -6 and attend(q=None) == -6 and attend(q=ctypes.c_void_p(8)) == -3
    assert attend(B=-1) == -1 and attend(group=0) == -1 and attend(T=1 << 17) == -1 and attend(width=1 << 30) == -1
    assert attend(prefix=17, pw=1, pt=p) == -1 and attend(prefix=16, pw=1) == -6
    need = lib.mxb_tree_attention_workspace_size(2, 3, 2, 4, 128, 8, 16, 1000, 0)
    assert need > 0 and attend(width=1000) == -7 and attend(width=1000, ws=p, n=need - 1) == -7
    assert attend(width=1000, ws=ctypes.c_void_p(48), n=need) == -3
    assert attend(B=0) == 0 and attend(T=0) == 0 and attend(B=0, mask=None) == 0


def test_histories_that_32_bit_positions_do_not_hold_are_refused():
    """A length within a tile of 2^31 wraps where it is rounded up to tiles of 128 keys.
    Shapes are looked at before the workspace, so that no call gets further than that."""
    lib, p = L.load(), ctypes.c_void_p(32)

    def attend(T, group, keys, page=16):
        return lib.mxb_tree_attention(p, 1, T, 2, group, 128, p, p, p, p, 4, page, 8, p, keys // page, p, None, 0, 0,
                                      p, T * T, T, 0.1, p, None, None, 0, None)

    most = 2 ** 31 - 1 - 512
    assert attend(64, 4, 2 ** 31 - 80) == -1 and attend(64, 1, most + 16) == -1
    assert attend(64, 4, most) == -7 and attend(64, 4, most, 1024) == -7
    assert attend(3, 4, 2 ** 31 - 80) == -7 and attend(3, 4, 2 ** 31 - 64) == -1  # few rows: tiles of 32


@pytest.mark.gpu
def test_refusals_on_the_device():
    c = mxb.paged_kv_cache(4, 2, 64, "int8d", 16)
    t, n = torch.zeros(2, 2, dtype=torch.int32, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda")
    q = torch.zeros(2, 3, 4, 64, device="cuda", dtype=torch.bfloat16)
    m = torch.ones(2, 3, 3, dtype=torch.bool, device="cuda")
    mxb.paged_attention(q, c, t, n, tree_mask=m)
    for bad in (m[:1], m[:, :2], m[..., :2], m.int(), m.float(), m.cpu(), m[0, 0], m[None]):
        with pytest.raises(ValueError):
            mxb.paged_attention(q, c, t, n, tree_mask=bad)


# ── attention ────────────────────────────────────────────────────────────────
def attend64(q, c, table, lengths, mask, prefix, prefix_len, scale):
    """(out, lse) in 64 bits, with sum_j p_j |v_j| for the tolerance."""
    B, T, Hq, D = q.shape
    H = c.n_heads
    q = q.double().view(B, T, H, Hq // H, D)
    out, mag = torch.zeros_like(q), torch.zeros_like(q)
    lse = torch.full(q.shape[:-1], float("-inf"), dtype=torch.float64, device=q.device)
    for b, n in enumerate(lengths):
        ks, vs = (history(c, w, table[b], n) for w in "kv")
        if prefix_len:
            ks, vs = (torch.cat((history(c, w, prefix, prefix_len), x), 1) for w, x in (("k", ks), ("v", vs)))
        for t in range(T):
            keep = [j for j in range(prefix_len + n)
                    if j < prefix_len + n - T or mask[b][t][j - (prefix_len + n - T)] or j < prefix_len]
            if keep:
                s = torch.einsum("hgd,hld->hgl", q[b, t], ks[:, keep]) * scale
                p = torch.softmax(s, -1)
                out[b, t] = torch.einsum("hgl,hld->hgd", p, vs[:, keep])
                mag[b, t] = torch.einsum("hgl,hld->hgd", p, vs[:, keep].abs())
                lse[b, t] = torch.logsumexp(s, -1)
    return out.view(B, T, Hq, D), lse.view(B, T, Hq), mag.view(B, T, Hq, D)


def check(got, lse, q, c, table, lengths, mask, prefix, prefix_len, scale=None):
    """The tolerances of the attention that this one is a form of (test_paged.py): a
    score's fp32 additions, fp16 weights, exponentials, and the rounding to bf16."""
    D = q.shape[-1]
    scale = 1 / math.sqrt(D) if scale is None else scale
    out64, lse64, mag = attend64(q, c, table, lengths, mask.tolist(), prefix, prefix_len, scale)
    off, top = (1152, 127) if c.dtype.bits == 8 else (136, 8)
    ks = torch.nan_to_num(c.k_scales, nan=0.0, posinf=0.0).max().double()
    e_s = ((D / 16 + 4) * 2.0 ** -23 * (off + top) * q.double().abs().sum(-1) * ks * abs(scale) * 1.4427
           + 2.0 ** -22)[..., None]
    n = max(lengths, default=0) + prefix_len
    floor = n * 2.0 ** -24 * top * torch.nan_to_num(c.v_scales, nan=0.0, posinf=0.0).max().double()
    tol = (2.0 ** -11 + 4 * e_s + 2.0 ** -20) * mag + 2.0 ** -8 * out64.abs() + floor
    bad = ~((got.double() - out64).abs() <= tol)
    assert got.shape == q.shape and not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:3].tolist())
    inf = lse64 == float("-inf")
    assert torch.equal(lse == float("-inf"), inf)
    d = (lse.double() - lse64).abs()[~inf]
    assert bool((d <= (2 * e_s[..., 0].expand_as(lse64) + 2.0 ** -18 * (1 + lse64.abs()))[~inf]).all())


def trees(B, T, seed):
    """Random trees: each token after the first hangs from one before it."""
    g = torch.Generator().manual_seed(seed)
    m = torch.eye(T, dtype=torch.bool).repeat(B, 1, 1)
    for b in range(B):
        for i in range(1, T):
            m[b, i] |= m[b, int(torch.rand((), generator=g) * i)]
    return m.cuda()


def run(dtype, dim, page, heads, group, T, lengths, prefix_len, mask=None, seed=0):
    B = len(lengths)
    pages = B * max(1, -(-max(lengths) // page)) + -(-prefix_len // page) + 3
    c = pool(pages, heads, dim, dtype, page, seed)
    table, rest = tables(lengths, page, pages, seed)
    g = torch.Generator("cuda").manual_seed(seed)
    q = torch.randn(B, T, heads * group, dim, generator=g, device="cuda").bfloat16()
    mask = trees(B, T, seed) if mask is None else mask
    n = torch.tensor(lengths, device="cuda")
    out, lse = mxb.paged_attention(q, c, table, n, prefix_table=rest, prefix_len=prefix_len, return_lse=True,
                                   tree_mask=mask)
    check(out, lse, q, c, table, lengths, mask.expand(B, T, T), rest, prefix_len)
    assert L.load().mxb_device_error(1) == 0
    return q, c, table, n, rest, out, lse


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["int8d", "int4d"])
@pytest.mark.parametrize("dim,page,heads,group,T,lengths,prefix", [
    (128, 64, 1, 1, 1, [1], 0), (64, 16, 2, 4, 2, [2, 40, 0, 1], 0), (128, 32, 2, 8, 5, [70, 5, 300], 0),
    (64, 64, 1, 5, 13, [13, 200, 64, 33], 0), (128, 16, 1, 4, 33, [100, 33, 34, 20], 0),
    (64, 128, 2, 8, 64, [64, 128, 700, 65], 0), (128, 64, 1, 4, 64, [1000, 63], 0), (128, 32, 1, 2, 130, [400, 131], 0),
    (64, 32, 2, 4, 7, [3000, 9, 0, 77], 0), (128, 64, 1, 8, 20, [5000, 21], 0), (64, 16, 1, 1, 70, [4500, 70, 71], 0),
    (128, 64, 2, 4, 6, [50, 6, 0], 100), (64, 32, 1, 8, 16, [40, 300], 1000), (128, 16, 1, 4, 40, [41, 90, 0], 333),
    (64, 64, 2, 2, 9, [9] * 20, 70)])
def test_tree_attention(dtype, dim, page, heads, group, T, lengths, prefix):
    run(dtype, dim, page, heads, group, T, lengths, prefix)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["int8d", "int4d"])
@pytest.mark.parametrize("dim,page,heads,group,T,lengths,prefix", [
    # short sequences of many rows, a unit a CTA: empty ones, shorter than their trees
    (128, 64, 2, 4, 16, [0, 3, 16, 17, 300, 900, 128, 127] * 5, 0), (64, 16, 2, 8, 12, [12, 0, 500, 5] * 10, 0),
    (64, 32, 4, 4, 40, [40, 41, 0, 170, 39] * 5, 90), (128, 128, 1, 8, 16, [16, 250] * 40, 0),
    # 25 to 63 rows in groups of the decode kernel
    (128, 16, 2, 4, 10, [600, 10, 0, 33] * 8, 0), (64, 32, 2, 4, 7, [640, 700, 9] * 9, 50),
    (128, 64, 4, 8, 5, [1500] * 5, 0)])
def test_many_units(dtype, dim, page, heads, group, T, lengths, prefix):
    run(dtype, dim, page, heads, group, T, lengths, prefix)


@pytest.mark.gpu
@pytest.mark.parametrize("group,T", [(1, 4), (8, 40)])
def test_no_keys_at_all(group, T):
    for B, prefix in ((2, 0), (60, 0), (2, 30)):
        run("int8d", 64, 16, 2, group, T, [0] * B, prefix)
    q, c, table, n, rest, _, _ = run("int8d", 64, 16, 2, group, T, [T, 2 * T], 0)
    mask = trees(2, T, 0)
    o, lse = mxb.paged_attention(q[:0], c, table[:0], n[:0], return_lse=True, tree_mask=mask[:0])
    assert o.shape == (0, T, 2 * group, 64) and lse.shape == (0, T, 2 * group)
    assert mxb.paged_attention(q[:, :0], c, table, n, tree_mask=mask[:, :0, :0]).shape == (2, 0, 2 * group, 64)
    o, lse = mxb.paged_attention(q, c, table[:, :0], n * 0, return_lse=True, tree_mask=mask)  # no pages
    assert not o.any() and bool((lse == float("-inf")).all())


@pytest.mark.gpu
@pytest.mark.parametrize("prefix", [0, 40])
def test_more_sequences_than_a_warp_adds_up(prefix):
    """The list of tiles of more than 512 sequences, one of them long."""
    lengths = [8 + i % 9 for i in range(700)]
    lengths[3], lengths[650], lengths[100], lengths[699] = 1500, 300, 0, 2
    run("int4d", 64, 16, 1, 8, 8, lengths, prefix)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["int8d", "int4d"])
@pytest.mark.parametrize("group,T,lengths,prefix", [(4, 5, [70, 5, 0], 0), (8, 40, [40, 300], 0), (4, 5, [70, 5, 0], 50),
                                                    (8, 40, [39, 300], 50), (2, 64, [3000, 64], 0)])
def test_masks_that_leave_rows_empty(dtype, group, T, lengths, prefix):
    """Rows that name none of the drafts, themselves included, see the history alone;
    where there is none they are zero."""
    none = torch.zeros(T, T, dtype=torch.bool, device="cuda")
    run(dtype, 64, 32, 2, group, T, lengths, prefix, none)
    some = torch.rand(len(lengths), T, T, generator=torch.Generator("cuda").manual_seed(1), device="cuda") < 0.1
    some[:, ::3] = False
    run(dtype, 128, 32, 1, group, T, lengths, prefix, some)


@pytest.mark.gpu
@pytest.mark.parametrize("group,T", [(1, 3), (4, 12), (8, 40)])
def test_a_chain_is_the_causal_order(group, T):
    """The mask of a chain gives what the call without a mask gives, row for row, up to
    the rounding of two orders of summation."""
    mask = torch.ones(T, T, dtype=torch.bool, device="cuda").tril()
    q, c, table, n, rest, out, lse = run("int8d", 128, 64, 2, group, T, [300, T, 65], 0, mask)
    causal, lse2 = mxb.paged_attention(q, c, table, n, return_lse=True)
    assert torch.allclose(out.float(), causal.float(), rtol=2 ** -7, atol=2 ** -9)
    assert torch.allclose(lse, lse2, rtol=1e-5, atol=1e-4)


@pytest.mark.gpu
def test_mask_layouts():
    T = 9
    q, c, table, n, rest, out, _ = run("int8d", 64, 16, 2, 4, T, [60, 9, 30], 0)
    m = trees(3, T, 0)
    wide = torch.zeros(3, T, 2 * T + 1, dtype=torch.bool, device="cuda")
    wide[:, :, 3:3 + T] = m
    same = mxb.paged_attention(q, c, table, n, tree_mask=wide[:, :, 3:3 + T])
    assert torch.equal(same, out)
    turned = m.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(mxb.paged_attention(q, c, table.long(), n.long(), tree_mask=turned), out)
    one = mxb.paged_attention(q, c, table, n, tree_mask=m[0])
    assert torch.equal(one, mxb.paged_attention(q, c, table, n, tree_mask=m[:1].expand(3, T, T)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["int8d", "int4d"])
@pytest.mark.parametrize("group,T,prefix", [(2, 6, 0), (8, 30, 0), (2, 6, 40), (8, 30, 40)])
def test_hidden_places_may_hold_anything(dtype, group, T, prefix):
    """Infinite and NaN scales of keys past the lengths, and of drafts that a row does
    not name, reach no row that does not see them."""
    page, heads = 16, 2
    lengths = [50, T, 0]
    c = pool(20, heads, 128, dtype, page, 6)
    table, rest = tables(lengths, page, 20, 6)
    mask = trees(3, T, 3)
    bad = 2 + T // 2  # a draft of the first sequence, and every key behind its end
    mask[0, :, bad] = False
    at = lengths[0] - T + bad
    for s, x in ((c.k_scales, float("nan")), (c.v_scales, float("inf"))):
        s[int(table[0, at // page]), :, at % page] = x
        s[int(table[0, 3]), :, 2:] = x       # 50 = 3 pages and 2 keys
        s[int(table[1, T // page]), :, T % page:] = x
        s[table[2].long()] = x
    g = torch.Generator("cuda").manual_seed(1)
    q = torch.randn(3, T, heads * group, 128, generator=g, device="cuda").bfloat16()
    n = torch.tensor(lengths, device="cuda")
    out, lse = mxb.paged_attention(q, c, table, n, prefix_table=rest, prefix_len=prefix, return_lse=True,
                                   tree_mask=mask)
    check(out, lse, q, c, table, lengths, mask, rest, prefix)
    mask[0, 3, bad] = True  # now one row sees it
    out = mxb.paged_attention(q, c, table, n, prefix_table=rest, prefix_len=prefix, tree_mask=mask)
    rows = torch.arange(T, device="cuda") != 3
    assert out[0, 3].isnan().all() and out[0, rows].isfinite().all() and out[1:].isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("group,T", [(2, 4), (8, 30)])
def test_bad_pages_hold_no_keys(group, T):
    c = pool(8, 2, 128, "int8d", 16, 5)
    L.load().mxb_device_error(1)
    table = torch.tensor([[1, 99, 2, 3], [4, -1, 5, 6]], dtype=torch.int32, device="cuda")
    lengths = [40, 64]
    mask = trees(2, T, 1)
    q = torch.randn(2, T, 2 * group, 128, generator=torch.Generator("cuda").manual_seed(2), device="cuda").bfloat16()
    out = mxb.paged_attention(q, c, table, torch.tensor(lengths, device="cuda"), tree_mask=mask)
    assert L.load().mxb_device_error(1) == 8
    for b, n in enumerate(lengths):
        k, v = (history(c, w, table[b].clamp(0, 7), n) for w in "kv")
        seen = torch.ones(T, n, dtype=torch.bool, device="cuda")
        seen[:, n - T:] = mask[b]
        seen[:, 16:32] = False
        s = torch.einsum("thgd,hld->thgl", q[b].double().view(T, 2, group, 128), k) / math.sqrt(128)
        p = torch.softmax(s.masked_fill(~seen[:, None, None], float("-inf")), -1)
        want = torch.einsum("thgl,hld->thgd", p, v).reshape(T, -1, 128)
        assert torch.allclose(out[b].double(), want, rtol=2 ** -7, atol=2e-2 * float(v.abs().max()))
    assert torch.isfinite(out).all()


@pytest.mark.gpu
@pytest.mark.parametrize("group,T", [(2, 4), (8, 30)])
def test_values_of_any_scale(group, T):
    """Value scales over six decades beside one another, scores that rise along the
    sequence."""
    c = pool(40, 1, 128, "int8d", 64, 3)
    g = torch.Generator("cuda").manual_seed(3)
    ramp = torch.arange(40 * 64, device="cuda").float().view(40, 1, 64)
    c.k_scales.copy_(ramp * 2e-5)
    c.v_scales.copy_(10.0 ** (torch.rand(40, 1, 64, generator=g, device="cuda") * -6))
    table = torch.arange(40, device="cuda", dtype=torch.int32)[None].repeat(3, 1)
    q = torch.randn(3, T, group, 128, generator=g, device="cuda").bfloat16()
    lengths, mask = [2500, 900, 77], trees(3, T, 2)
    out, lse = mxb.paged_attention(q, c, table, torch.tensor(lengths, device="cuda"), return_lse=True, tree_mask=mask)
    check(out, lse, q, c, table, lengths, mask, table[0], 0)


@pytest.mark.gpu
@pytest.mark.parametrize("group,T", [(4, 8), (8, 40)])
def test_repeats_on_any_stream_and_in_a_graph(group, T):
    q, c, table, n, rest, want, _ = run("int8d", 128, 64, 2, group, T, [700, 90, 300], 100)
    mask = trees(3, T, 0)

    def call():
        return mxb.paged_attention(q, c, table, n, prefix_table=rest, prefix_len=100, tree_mask=mask)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [call() for _ in range(10)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    n0 = n.clone()
    n.copy_(torch.tensor([T, T, T], device="cuda"))
    graph.replay()
    short = out.clone()
    assert torch.equal(short, call()) and not torch.equal(short, want)
    n.copy_(n0)
    graph.replay()
    assert torch.equal(out, want)


# ── together ─────────────────────────────────────────────────────────────────
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["int8d", "int4d"])
def test_a_layer_verifies_drafts(dtype):
    """Norm, projection, rotation into the cache, attention of the tree, projection: the
    drafts of a chain through the tree give what the same tokens give one by one."""
    dim, heads, kv, D, page, B, T, past = 256, 4, 2, 64, 16, 3, 5, 37
    g = torch.Generator("cuda").manual_seed(0)

    def weight(n, k):
        return mxb.int8_linear(mxb.dynamic_quantize(torch.randn(n, k, generator=g, device="cuda") * k ** -0.5,
                                                    "int8d", "per_token"))

    qkv, out = weight((heads + 2 * kv) * D, dim), weight(dim, heads * D)
    norm = 1 + 0.1 * torch.randn(dim, generator=g, device="cuda").bfloat16()
    inv_freq = (10000.0 ** (-torch.arange(D // 2, device="cuda") / (D // 2))).float()
    table = torch.randperm(16, generator=torch.Generator().manual_seed(1))[:B * 4].view(B, 4).cuda()

    def step(cache, x, h, at, mask):
        """x, h [B, t, dim] at slots `at` [B, t], positions by depth."""
        t = x.shape[1]
        a, h = mxb.rms_norm_quantize(x, norm, residual=h)
        q, k, v = qkv(a).flatten(0, 1).unflatten(-1, (-1, D)).split([heads, kv, kv], 1)
        depth = at if mask is None else at[:, :1] + mask.sum(-1) - 1
        slots = table.gather(1, at // page) * page + at % page
        q = cache.append(k, v, slots.flatten(), depth.flatten(), inv_freq, q=q)
        n = (at[:, -1] + 1).int()
        o = mxb.paged_attention(q.view(B, t, heads, D), cache, table, n, tree_mask=mask)
        return out(o.flatten(2)), h

    prompt = [torch.randn(B, past, dim, generator=g, device="cuda").bfloat16() for _ in range(2)]
    new = [torch.randn(B, T, dim, generator=g, device="cuda").bfloat16() for _ in range(2)]
    chain, single = (mxb.paged_kv_cache(16, kv, D, dtype, page) for _ in range(2))
    at = torch.arange(past, device="cuda").expand(B, past)
    for c in (chain, single):
        step(c, *prompt, at, None)
    at = past + torch.arange(T, device="cuda").expand(B, T)
    # tokens 0, 1, 3 are a chain; 2 hangs from 0, 4 from 2
    seen = torch.eye(T, dtype=torch.bool, device="cuda")
    for i, parent in ((1, 0), (2, 0), (3, 1), (4, 2)):
        seen[i] |= seen[parent]
    tree, h = step(chain, *new, at, seen.expand(B, T, T))
    assert torch.equal(h, new[0] + new[1])
    for path in ((0, 1, 3), (0, 2, 4)):
        for depth, i in enumerate(path):
            one, _ = step(single, *(x[:, i:i + 1] for x in new), at[:, depth:depth + 1], None)
            # the same keys in other places and orders: the attention's rounding to bf16,
            # and what it moves in the codes of the second product
            err = (one[:, 0].float() - tree[:, i].float()).abs().max()
            assert err <= 0.03 * tree[:, i].float().abs().max(), (path, i, float(err))
