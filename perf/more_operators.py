"""The operators of a quantized decoder layer that are measured beside those of
``perf/operators.py``: root-mean-square norm with the residual's addition into
int8 codes, the int8 product with a scale a token and a channel, keys and queries
rotated on their way into the paged cache, and attention of a tree of drafted
tokens over that cache.

``run`` computes each in its plain form (elementary torch operations) or, where
``own`` is true, through ``qtpytorch_b200``; ``exact`` gives the same outputs in
64 bits, written from the formulas on their own.

Formulas
- norm: h = x + residual; y = h w / sqrt(mean(h^2) + eps); scale = amax|y| / 127 a
  row (at least 1e-12 / 127), code = y / scale rounded to the nearest, ties to even;
  y / scale is 127 u / amax|u| of u = h w, whatever the root is.
- product: y[m, n] = sa[m] sb[n] sum_k a[m, k] b[n, k] (+ bias[n]), codes of 8 bits.
- append: pair i of a head row turns by position * inv_freq[i], the position taken
  from the axis that the pair's section names; a pair is (i, i + rot / 2), or
  (2 i, 2 i + 1) where interleaved; dims from rot on stay.  Queries return rotated;
  keys (rotated, then rounded to fp32) and values become codes by the cache's
  quantizer, which is defined by its steps in fp32: si = fl(fl(1 / max(amax, 1e-12)) m),
  code = rint(fl(x si)), scale = fl(1 / si), m = 127 or 7.
- tree: query t of a sequence sees its keys j < length - T and, of its T newest keys,
  those that row t of the mask names, behind a prefix that all see;
  softmax(scale * q k) v, zero where a row has no keys.
"""
import math

import torch

own = False

EPS = 1e-6


# ── cases ────────────────────────────────────────────────────────────────────
def listed():
    return [
        # a decode step's activations in front of a projection: latency
        dict(name="norm_step", op="norm", rows=8, cols=4096, dtype="bf16", residual=True),
        # an odd batch of an odd width at the start of a model, where no residual is yet
        dict(name="norm_odd", op="norm", rows=1001, cols=1999, dtype="f32", residual=False),
        # long prompts of a wide model
        dict(name="norm_prompt", op="norm", rows=4096, cols=8192, dtype="bf16", residual=True),
        # one token through an up projection (in 4096, out 11008)
        dict(name="product_token", op="product", m=1, k=4096, n=11008, bias=False, out="bf16"),
        # an odd batch through an odd layer with a bias, kept in fp32
        dict(name="product_odd", op="product", m=77, k=2000, n=1000, bias=True, out="f32"),
        # prompts through that projection
        dict(name="product_prompt", op="product", m=2048, k=4096, n=11008, bias=False, out="bf16"),
        # long prompts through a square layer of 8192
        dict(name="product_large", op="product", m=4096, k=8192, n=8192, bias=False, out="bf16"),
        # a decode step: one token a sequence into small pages; a short history is read back
        dict(name="append_step", op="append", dtype="int8d", q_heads=32, heads=8, dim=128, rot=128, page=16,
             batch=32, max_len=200, new=1, axes=1, interleaved=False),
        # prompts of images and text (time, height, width) are written whole and read back
        dict(name="append_images", op="append", dtype="int4d", q_heads=32, heads=8, dim=128, rot=128, page=64,
             batch=4, max_len=4096, new=4096, axes=3, interleaved=False),
        # a small tree behind one short sequence: latency
        dict(name="tree_short", op="tree", dtype="int8d", batch=1, tree=8, heads=8, group=4, dim=128, page=64,
             max_len=700, prefix=0, empty=0),
        # trees of a mid-sized batch behind a common instruction, some slots of the batch idle
        dict(name="tree_batch", op="tree", dtype="int4d", batch=24, tree=13, heads=4, group=8, dim=64, page=32,
             max_len=6000, prefix=1000, empty=2),
        # wide trees over long histories
        dict(name="tree_wide", op="tree", dtype="int8d", batch=16, tree=64, heads=8, group=4, dim=128, page=64,
             max_len=8192, prefix=0, empty=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: sizes log-uniform over the listed ranges, odd ones among them."""
    op = rng.choice(["norm", "product", "product", "append", "append", "tree", "tree", "tree"])
    if op == "norm":
        rows, cols = _log(rng, 1, 8192), _log(rng, 64, 16384)
        if rng.random() < 0.6:  # widths are mostly multiples of 64
            cols = -(-cols // 64) * 64
        return dict(op=op, rows=max(1, min(rows, 33_000_000 // cols)), cols=cols,
                    dtype=rng.choice(["bf16", "f32"]), residual=rng.random() < 0.6)
    if op == "product":
        k, n = _log(rng, 64, 11008), _log(rng, 64, 11008)
        if rng.random() < 0.6:
            k, n = -(-k // 64) * 64, -(-n // 64) * 64
        return dict(op=op, m=_log(rng, 1, 2300), k=k, n=n, bias=rng.random() < 0.3,
                    out=rng.choice(["bf16", "f32"]))
    if op == "append":
        batch, max_len = _log(rng, 1, 64), _log(rng, 1, 4096)
        max_len = min(max_len, max(1, 16384 // batch))
        heads, dim = rng.choice([1, 4, 8]), rng.choice([64, 128])
        return dict(op=op, dtype=rng.choice(["int8d", "int4d"]), q_heads=heads * rng.choice([1, 3, 4]),
                    heads=heads, dim=dim, rot=rng.choice([dim, dim, dim // 2, dim - 24]),
                    page=rng.choice([16, 32, 64, 128]), batch=batch, max_len=max_len,
                    new=rng.choice([1, max_len, max(1, max_len // 3)]), axes=rng.choice([1, 1, 2, 3]),
                    interleaved=rng.random() < 0.3)
    tree, group = _log(rng, 1, 64), rng.choice([1, 2, 4, 5, 8])
    heads, batch = rng.choice([1, 4, 8]), _log(rng, 1, 32)
    # the rows of all heads times the keys they see, at most half of tree_wide's
    most = min(200_000, 100_000_000 // (tree * group * heads))
    total = _log(rng, 1, most)
    return dict(op=op, dtype=rng.choice(["int8d", "int4d"]), batch=batch, tree=tree, heads=heads, group=group,
                dim=rng.choice([64, 128]), page=rng.choice([16, 32, 64, 128]), max_len=max(tree, total // batch),
                prefix=rng.choice([0, 0, _log(rng, 1, max(1, most // batch))]),
                empty=rng.choice([0, 0, batch // 8]))


# ── inputs ───────────────────────────────────────────────────────────────────
_TYPES = dict(bf16=torch.bfloat16, f32=torch.float32)


def _bits(case):
    return 8 if case["dtype"] == "int8d" else 4


def _gen(seed, device):
    return torch.Generator(device).manual_seed(seed)


def _lengths(case, gen):
    """Keys of each sequence: from the longest down to a quarter of it, in any order; `empty` idle slots."""
    b, top = case["batch"], case["max_len"]
    n = [max(1, top - (top - top // 4) * i // max(1, b - 1)) for i in range(b)]
    for i in range(case.get("empty", 0)):
        n[b - 1 - i] = 0
    return torch.tensor(n)[torch.randperm(b, generator=gen)]


def _tables(case, gen):
    """Page tables of the sequences and of the prefix, pages in any order; pages of the pool."""
    wide, shared = -(-case["max_len"] // case["page"]), -(-case.get("prefix", 0) // case["page"])
    pages = case["batch"] * wide + shared
    order = torch.randperm(pages, generator=gen).to(torch.int32)
    return order[shared:].view(case["batch"], wide).cuda(), order[:shared].cuda(), pages


def _pool(case, pages, rng):
    """Codes and scales of keys and values, as an earlier run left them."""
    bits, shape, pool = _bits(case), (pages, case["heads"], case["page"]), []
    for top in (3.0, 2.0):
        if bits == 8:
            c = torch.randn(*shape, case["dim"], generator=rng, device="cuda").mul_(40).clamp_(-127, 127)
            c = c.to(torch.int8).view(torch.uint8)
        else:
            c = torch.randint(1, 16, (2, *shape, case["dim"] // 2), generator=rng, device="cuda", dtype=torch.uint8)
            c = (c[0] + 8) % 16 | (c[1] + 8) % 16 << 4  # codes are -7..7
        s = torch.rand(shape, generator=rng, device="cuda").add_(0.5).mul_(top)
        pool += [c, s.div_(127.0 if bits == 8 else 7.0)]
    return pool


def _trees(case, gen):
    """[batch, T, T]: each token after the first hangs from one before it and sees its ancestors and itself."""
    t = case["tree"]
    seen = torch.eye(t, dtype=torch.bool).repeat(case["batch"], 1, 1)
    at = torch.arange(case["batch"])
    for i in range(1, t):
        parent = (torch.rand(case["batch"], generator=gen) * i).long()
        seen[:, i] |= seen[at, parent]
    return seen.cuda()


def _sections(case):
    """Pairs of each position axis: all of them, or the first quarter by time and the rest shared out."""
    pairs, axes = case["rot"] // 2, case["axes"]
    if axes == 1:
        return None
    first = pairs // 4
    rest = pairs - first
    return [first] + [rest // (axes - 1)] * (axes - 2) + [rest - rest // (axes - 1) * (axes - 2)]


def _positions(case, at):
    """Positions of the tokens `at` of their sequences: text, or (time, height, width) of images of 16 x 16."""
    if case["axes"] == 1:
        return at + 30000  # behind a long document that the cache holds elsewhere
    grid = torch.stack((at // 256, at // 16 % 16, at % 16))
    return (grid + 500)[:case["axes"]]


def prepare(case, seed):
    rng, gen = _gen(seed, "cuda"), _gen(seed, "cpu")
    s = dict(case=case)

    def normal(*shape):
        return torch.randn(*shape, generator=rng, device="cuda")

    if case["op"] == "norm":
        t, cols = _TYPES[case["dtype"]], case["cols"]
        loud = 1 + 20 * (torch.rand(cols, generator=rng, device="cuda") < 0.01)  # a few channels are far larger
        s["x"] = normal(case["rows"], cols).mul_(loud).to(t)
        s["residual"] = normal(case["rows"], cols).mul_(3 * loud).to(t) if case["residual"] else None
        s["weight"] = (1 + 0.2 * normal(cols)).to(t)
    elif case["op"] == "product":
        for name, rows, size in (("a", case["m"], 1.0), ("b", case["n"], 0.02)):
            x = normal(rows, case["k"]).mul_(size)
            scale = x.abs().amax(1) / 127
            s[name], s[name + "_scales"] = torch.round(x / scale[:, None]).to(torch.int8), scale
        s["bias"] = normal(case["n"]) if case["bias"] else None
        if own:  # the quantized tensors that the program holds
            s["tensors"] = _mx(s)
    else:
        s["table"], s["shared"], pages = _tables(case, gen)
        s["pool"] = _pool(case, pages, rng)
        n = _lengths(case, gen)
        s["lengths"] = n.to(torch.int32).cuda()
        if case["op"] == "append":
            # the last `new` tokens of every sequence (fewer where it is shorter), packed one after another
            at = torch.arange(case["max_len"]).repeat(case["batch"], 1)
            fresh = (at < n[:, None]) & (at >= n[:, None] - case["new"])
            where = s["table"].cpu().long().repeat_interleave(case["page"], 1)[:, :case["max_len"]]
            s["slots"] = (where * case["page"] + at % case["page"])[fresh].cuda()
            s["positions"] = _positions(case, at[fresh]).cuda()
            tokens, dim = int(fresh.sum()), case["dim"]
            s["q"] = normal(tokens, case["q_heads"], dim).bfloat16()
            s["k"] = normal(tokens, case["heads"], dim)
            s["k"] *= 1 + 6 * (torch.rand(case["heads"], dim, generator=rng, device="cuda") < 0.05)
            s["k"] = s["k"].bfloat16()
            s["v"] = normal(tokens, case["heads"], dim).bfloat16()
            i = torch.arange(case["rot"] // 2, dtype=torch.float64)
            s["inv_freq"] = (500000.0 ** (-2 * i / case["rot"])).float().cuda()
        else:
            s["q"] = normal(case["batch"], case["tree"], case["heads"] * case["group"], case["dim"]).bfloat16()
            s["tree"] = _trees(case, gen)
    return s


# ── the operators ────────────────────────────────────────────────────────────
def run(s):
    return (_run_own if own else _run_plain)(s)


def _mx(s):
    import qtpytorch_b200 as mxb

    k = s["case"]["k"]
    return [mxb.mx_tensor(s[x].view(-1), s[x + "_scales"], mxb.int8d, s[x].shape, s[x].numel(), k) for x in "ab"]


def _run_own(s):
    import qtpytorch_b200 as mxb

    case = s["case"]
    if case["op"] == "norm":
        if s["residual"] is None:
            return mxb.rms_norm_quantize(s["x"], s["weight"], eps=EPS).dequantize()
        codes, h = mxb.rms_norm_quantize(s["x"], s["weight"], residual=s["residual"], eps=EPS)
        return codes.dequantize(), h
    if case["op"] == "product":
        a, b = s["tensors"] if "tensors" in s else _mx(s)
        return mxb.int8_matmul(a, b, bias=s["bias"], out_dtype=_TYPES[case["out"]])
    cache = mxb.paged_kv_cache.from_buffers(*s["pool"], dtype=case["dtype"])
    if case["op"] == "append":
        q = cache.append(s["k"], s["v"], s["slots"], s["positions"], s["inv_freq"], q=s["q"],
                         sections=_sections(case), interleaved=case["interleaved"])
        return (q, *cache.read(s["table"], s["lengths"], case["max_len"]))
    return mxb.paged_attention(s["q"], cache, s["table"], s["lengths"], prefix_table=s["shared"],
                               prefix_len=case["prefix"], tree_mask=s["tree"])


def _run_plain(s):
    return dict(norm=_plain_norm, product=_plain_product, append=_plain_append, tree=_plain_tree)[s["case"]["op"]](s)


def _plain_norm(s):
    # codes of values next to a border, and the long sum: in 64 bits
    h = s["x"].double()
    if s["residual"] is not None:
        h = h + s["residual"].double()
    u = h * s["weight"].double()
    root = torch.sqrt(h.square().mean(1, keepdim=True) + EPS)
    top = torch.maximum(u.abs().amax(1, keepdim=True), 1e-12 * root)
    values = torch.round(u * 127 / top).float() * (top / root / 127).float()
    return values if s["residual"] is None else (values, h.to(s["x"].dtype))


def _plain_product(s):
    # sums of products of codes pass 2^24: parts of K whose sums fp32 holds, added up in 64
    acc = torch.zeros(s["a"].shape[0], s["b"].shape[0], dtype=torch.float64, device="cuda")
    for a, b in zip(s["a"].split(1024, 1), s["b"].split(1024, 1)):
        acc += torch.mm(a.float(), b.float().t())
    y = acc.float() * s["a_scales"][:, None] * s["b_scales"]
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(_TYPES[s["case"]["out"]])


def _pack(code, bits):
    code = code.to(torch.int32)
    if bits == 8:
        return (code & 255).to(torch.uint8)
    return ((code[..., 0::2] & 15) | (code[..., 1::2] & 15) << 4).to(torch.uint8)


def _values(packed, scales, bits):
    if bits == 8:
        code = packed.view(torch.int8).float()
    else:
        code = torch.stack(((packed & 15 ^ 8).float() - 8, (packed >> 4 ^ 8).float() - 8), -1).flatten(-2)
    return code * scales[..., None]


def _rotate(x, cos, sin, interleaved):
    """x [T, heads, dim] in 64 bits, cos and sin [T, pairs]."""
    pairs = cos.shape[1]
    first = slice(0, 2 * pairs, 2) if interleaved else slice(0, pairs)
    second = slice(1, 2 * pairs, 2) if interleaved else slice(pairs, 2 * pairs)
    c, n = cos[:, None], sin[:, None]
    out = x.clone()
    out[..., first] = x[..., first] * c - x[..., second] * n
    out[..., second] = x[..., first] * n + x[..., second] * c
    return out


def _plain_append(s):
    case, (kc, ks, vc, vs) = s["case"], s["pool"]
    bits, page, sections = _bits(case), case["page"], _sections(case)
    at = s["positions"].double()
    # angles of far positions, and keys next to a border between codes: in 64 bits
    if sections is None:
        angle = at[:, None] * s["inv_freq"].double()
    else:
        axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections)).cuda()
        angle = at[axis].t() * s["inv_freq"].double()
    cos, sin = angle.cos(), angle.sin()
    q = _rotate(s["q"].double(), cos, sin, case["interleaved"]).to(s["q"].dtype)
    m = 127.0 if bits == 8 else 7.0
    k = _rotate(s["k"].double(), cos, sin, case["interleaved"]).float()
    for codes, scales, x in ((kc, ks, k), (vc, vs, s["v"].float())):
        si = x.abs().amax(-1, keepdim=True).clamp(min=1e-12).reciprocal() * m
        codes[s["slots"] // page, :, s["slots"] % page] = _pack(torch.round(x * si), bits)
        scales[s["slots"] // page, :, s["slots"] % page] = si.reciprocal().squeeze(-1)
    live = torch.arange(case["max_len"], device="cuda") < s["lengths"][:, None]
    back = [q]
    for codes, scales in ((kc, ks), (vc, vs)):
        x = _values(codes[s["table"]], scales[s["table"]], bits)  # [b, pages, heads, page, dim]
        x = x.transpose(2, 3).flatten(1, 2)[:, :case["max_len"]]
        back.append(torch.where(live[:, :, None, None], x, 0.0).bfloat16())
    return tuple(back)


def _plain_tree(s):
    case, (kc, ks, vc, vs) = s["case"], s["pool"]
    bits, t, table = _bits(case), case["tree"], s["table"]
    q = s["q"].float().unflatten(2, (case["heads"], case["group"])) / math.sqrt(case["dim"])
    # which keys query t of a sequence sees: the history, then what its row of the mask names
    i = torch.arange(table.shape[1] * case["page"], device="cuda") - (s["lengths"][:, None] - t)  # [b, l]
    seen = s["tree"].gather(2, i.clamp(0, t - 1)[:, None].expand(-1, t, -1)) & (i < t)[:, None]
    seen = (seen | (i < 0)[:, None]) & (i < t)[:, None]
    k = _values(kc[table], ks[table], bits).transpose(2, 3).flatten(1, 2)
    score = torch.einsum("bthgd,blhd->bhgtl", q, k).masked_fill(~seen[:, None, None], float("-inf"))
    p, n = case["prefix"], score.shape[-1]
    if p:
        kp = _values(kc[s["shared"]], ks[s["shared"]], bits).transpose(1, 2).flatten(0, 1)[:p]
        score = torch.cat((score, torch.einsum("bthgd,lhd->bhgtl", q, kp)), -1)
    top = score.amax(-1, keepdim=True)
    w = torch.exp(score - torch.where(top == float("-inf"), 0.0, top))
    total = w.sum(-1, keepdim=True)
    w = torch.where(total > 0, w / total, 0.0)
    v = _values(vc[table], vs[table], bits).transpose(2, 3).flatten(1, 2)
    o = torch.einsum("bhgtl,blhd->bthgd", w[..., :n], v)
    if p:
        vp = _values(vc[s["shared"]], vs[s["shared"]], bits).transpose(1, 2).flatten(0, 1)[:p]
        o = o + torch.einsum("bhgtl,lhd->bthgd", w[..., n:], vp)
    return o.flatten(2, 3).bfloat16()


# ── what a pass cannot do without ────────────────────────────────────────────
def work(case):
    if case["op"] == "norm":
        n, size = case["rows"] * case["cols"], 2 if case["dtype"] == "bf16" else 4
        # x (and the residual) read, codes (and the sum) written; the codes read back, the values written
        return {"bytes": n * (size * (3 if case["residual"] else 1) + 2 + 4) + 8 * case["rows"] + size * case["cols"],
                "flops": 7 * n}
    if case["op"] == "product":
        m, k, n = case["m"], case["k"], case["n"]
        return {"bytes": (m + n) * (k + 4) + m * n * (2 if case["out"] == "bf16" else 4) + (4 * n if case["bias"] else 0),
                "flops": 2 * m * n * k}
    n = _lengths(case, _gen(0, "cpu"))
    row = case["dim"] * _bits(case) / 8 + 4  # a token's key or value in one head
    if case["op"] == "append":
        fresh, live = int(n.clamp(max=case["new"]).sum()), int(n.sum())
        heads, dim = case["heads"], case["dim"]
        dense = case["batch"] * case["max_len"] * dim * 2
        return {"bytes": fresh * case["q_heads"] * dim * 4 + 2 * heads * (fresh * (dim * 2 + row) + live * row + dense),
                "flops": fresh * dim * (3 * case["q_heads"] + 7 * heads) + 2 * live * heads * dim}
    rows = case["tree"] * case["group"] * case["heads"]
    keys = int(n.sum()) + case["prefix"]
    return {"bytes": 2 * case["heads"] * keys * row + 4 * case["batch"] * rows * case["dim"]
            + case["batch"] * case["tree"] ** 2,
            "flops": 4 * rows * case["dim"] * (int(n.sum()) + case["batch"] * case["prefix"])}


# ── 64 bits ──────────────────────────────────────────────────────────────────
def _exact_norm(s):
    h = s["x"].double() if s["residual"] is None else s["x"].double() + s["residual"].double()
    rms = torch.sqrt((h * h).sum(1, keepdim=True) / h.shape[1] + EPS)
    u = h * s["weight"].double()
    most = u.abs().max(1, keepdim=True).values
    # the quotient that is rounded: of whole products, so that ties are ties
    code = torch.round(torch.where(most >= 1e-12 * rms, 127 * u / most, u / rms * 127e12))
    values = code * torch.clamp(most / rms, min=1e-12) / 127
    return values if s["residual"] is None else (values, h)


def _exact_product(s):
    a, b = (s[x].double() * s[x + "_scales"].double()[:, None] for x in "ab")
    y = torch.mm(a, b.t())
    return y if s["bias"] is None else y + s["bias"].double()


def _exact_kv(codes, scales, bits):
    """[pages, heads, page, dim] values in 64 bits."""
    c = codes.to(torch.int16)
    if bits == 8:
        c = torch.where(c > 127, c - 256, c)
    else:
        both = torch.empty(*c.shape[:-1], 2 * c.shape[-1], dtype=torch.int16, device=c.device)
        both[..., 0::2], both[..., 1::2] = c % 16, c // 16
        c = torch.where(both > 7, both - 16, both)
    return c.double() * scales.double()[..., None]


def _exact_append(s):
    case, (kc, ks, vc, vs) = s["case"], s["pool"]
    bits, page, heads, dim, rot = _bits(case), case["page"], case["heads"], case["dim"], case["rot"]
    sections, where = _sections(case), s["positions"].double().reshape(case["axes"], -1)
    turn = torch.empty(where.shape[1], rot // 2, dtype=torch.float64, device="cuda")
    axis, left = 0, sections[0] if sections else rot
    for i in range(rot // 2):
        while left == 0:
            axis += 1
            left = sections[axis]
        turn[:, i] = where[axis] * s["inv_freq"][i].double()
        left -= 1

    def turned(x):  # as a product of complex numbers
        head = x.double()[..., :rot]
        z = (torch.view_as_complex(head.unflatten(-1, (-1, 2)).contiguous()) if case["interleaved"]
             else torch.complex(head[..., :rot // 2].contiguous(), head[..., rot // 2:].contiguous()))
        z = torch.view_as_real(z * torch.polar(torch.ones_like(turn), turn)[:, None])
        flat = z.flatten(-2) if case["interleaved"] else z.transpose(-1, -2).flatten(-2)
        return torch.cat((flat, x.double()[..., rot:]), -1)

    def fl(x):  # one step of the quantizer
        return x.to(torch.float32).to(torch.float64)

    back, top = [turned(s["q"])], 127.0 if bits == 8 else 7.0
    for codes, scales, x in ((kc, ks, fl(turned(s["k"]))), (vc, vs, s["v"].double())):
        si = fl(fl(1 / torch.clamp(x.abs().max(-1, keepdim=True).values, min=1e-12)) * top)
        pool = _exact_kv(codes, scales, bits).transpose(1, 2).reshape(-1, heads, dim)  # by slot
        pool[s["slots"]] = torch.round(fl(x * si)) / si
        out = torch.zeros(case["batch"], case["max_len"], heads, dim, dtype=torch.float64, device="cuda")
        for b, n in enumerate(s["lengths"].tolist()):
            at = torch.arange(n, device="cuda")
            out[b, :n] = pool[s["table"][b].long()[at // page] * page + at % page]
        back.append(out)
    return tuple(back)


def _exact_tree(s):
    case, (kc, ks, vc, vs) = s["case"], s["pool"]
    bits, heads, dim, t = _bits(case), case["heads"], case["dim"], case["tree"]
    q = s["q"].double().view(case["batch"], t, heads, case["group"], dim)
    out = torch.zeros_like(q)

    def keys(pages, n, codes, scales):  # [heads, n, dim]
        x = _exact_kv(codes[pages.long()], scales[pages.long()], bits)
        return x.transpose(0, 1).reshape(heads, -1, dim)[:, :n]

    first = [keys(s["shared"], case["prefix"], c, x) for c, x in ((kc, ks), (vc, vs))]
    for b, n in enumerate(s["lengths"].tolist()):
        k, v = (torch.cat((f, keys(s["table"][b], n, c, x)), 1) for f, (c, x) in zip(first, ((kc, ks), (vc, vs))))
        hidden = torch.zeros(t, k.shape[1], dtype=torch.bool, device="cuda")
        for i in range(max(0, t - n), t):  # key i of the tree, where the sequence holds it
            hidden[:, case["prefix"] + n - t + i] = ~s["tree"][b, :, i]
        if k.shape[1] == 0:
            continue
        a = torch.einsum("thgd,hld->hgtl", q[b], k) / dim ** 0.5
        a = torch.softmax(a.masked_fill(hidden, float("-inf")), -1).nan_to_num(0.0)  # a row without keys
        out[b] = torch.einsum("hgtl,hld->thgd", a, v)
    return out.flatten(2, 3)


def exact(case, seed):
    return dict(norm=_exact_norm, product=_exact_product, append=_exact_append,
                tree=_exact_tree)[case["op"]](prepare(case, seed))
