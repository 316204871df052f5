"""The serving operators that are measured: microscaled 4-bit floating point
(quantize, product), the paged quantized KV cache (write, read back) and
attention over that cache with a prefix shared by the whole batch.

``run`` computes each in its plain form (elementary torch operations, fp32)
or, where ``own`` is true, through ``qtpytorch_b200``; ``exact`` gives the
same outputs in 64 bits, written from the formulas on their own.

Formulas
- E2M1 holds 0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives.  mxfp4: blocks of
  32 along a row, scale 2^e with e = floor(log2(amax)) - 2 in [-127, 127];
  nvfp4: blocks of 16, scale s = e4m3(min(amax / (6 g), 448)) and one fp32
  factor g = amax(tensor) / 2688 a tensor.  The code is x / scale rounded to
  the nearest E2M1 value, ties to the even code, saturating.
- Scales of a [rows, blocks] matrix are kept in tiles of 128 rows x 4 blocks:
  byte ((r % 32) * 4 + r // 32) * 4 + c of the tile, tiles row-major.
- The product is dequant(quantize(x)) @ dequant(W)^T (+ bias).
- The cache holds int8 or int4 codes, one fp32 scale a token and head:
  si = m / max(amax, 1e-12), code = rint(x * si), scale = 1 / si, m = 127 or 7.
- Attention: query t of q_len sees the whole prefix and its sequence's keys
  j < length - (q_len - 1 - t); softmax(scale * q k) v, zero where a row has
  no keys.
"""
import math

import torch

own = False

HEADS = 8  # KV heads of the cache cases


# ── cases ────────────────────────────────────────────────────────────────────
def listed():
    return [
        # activations of a decode step on their way into a 4-bit product: latency
        dict(name="quantize_tokens", op="quantize", fmt="mxfp4", rows=8, cols=4096, dtype="bf16"),
        # a projection's fp32 weights quantized at load (in 4096, out 11008)
        dict(name="quantize_weight", op="quantize", fmt="nvfp4", rows=11008, cols=4096, dtype="f32"),
        # one token through that projection
        dict(name="linear_token", op="linear", fmt="mxfp4", m=1, k=4096, n=11008, bias=False),
        # an odd batch through an odd layer: ragged rows, blocks and columns, a bias
        dict(name="linear_odd", op="linear", fmt="nvfp4", m=77, k=2000, n=1000, bias=True),
        # prompts through the projection
        dict(name="linear_prompt", op="linear", fmt="nvfp4", m=2048, k=4096, n=11008, bias=False),
        # long prompts through a square layer of 8192
        dict(name="linear_large", op="linear", fmt="mxfp4", m=4096, k=8192, n=8192, bias=False),
        # a decode step writes one token a sequence into small pages; a short history is read back
        dict(name="cache_step", op="cache", dtype="int8d", heads=HEADS, dim=128, page=16, batch=32,
             max_len=200, new=1),
        # four prompts are written whole and read back for the next chunk
        dict(name="cache_prompt", op="cache", dtype="int4d", heads=HEADS, dim=128, page=64, batch=4,
             max_len=4096, new=4096),
        # one sequence that has just begun: latency
        dict(name="attend_short", op="attend", dtype="int8d", batch=1, q_len=1, heads=HEADS, group=4,
             dim=128, page=64, max_len=130, prefix=0, empty=0),
        # three drafted tokens a sequence behind a short instruction, some slots of the batch idle
        dict(name="attend_drafts", op="attend", dtype="int4d", batch=48, q_len=3, heads=4, group=8,
             dim=64, page=32, max_len=6000, prefix=1000, empty=3),
        # two very long contexts
        dict(name="attend_long", op="attend", dtype="int8d", batch=2, q_len=1, heads=HEADS, group=4,
             dim=128, page=64, max_len=131072, prefix=0, empty=0),
        # many conversations over one long document
        dict(name="attend_prefix", op="attend", dtype="int8d", batch=64, q_len=1, heads=HEADS, group=8,
             dim=128, page=64, max_len=512, prefix=8192, empty=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: sizes log-uniform over the listed ranges, odd ones among them."""
    op = rng.choice(["quantize", "linear", "linear", "cache", "attend", "attend", "attend"])
    if op == "quantize":
        rows = _log(rng, 1, 8192)
        return dict(op=op, fmt=rng.choice(["mxfp4", "nvfp4"]), rows=rows,
                    cols=min(_log(rng, 64, 16384), 40_000_000 // rows),
                    dtype=rng.choice(["bf16", "f32"]))
    if op == "linear":
        k, n = _log(rng, 256, 11008), _log(rng, 128, 11008)
        if rng.random() < 0.6:  # layers are mostly multiples of 64
            k, n = -(-k // 64) * 64, -(-n // 64) * 64
        return dict(op=op, fmt=rng.choice(["mxfp4", "nvfp4"]), m=_log(rng, 1, 2300), k=k, n=n,
                    bias=rng.random() < 0.3)
    if op == "cache":
        batch, max_len = _log(rng, 1, 64), _log(rng, 1, 4096)
        max_len = min(max_len, max(1, 16384 // batch))
        return dict(op=op, dtype=rng.choice(["int8d", "int4d"]), heads=rng.choice([1, 4, 8]),
                    dim=rng.choice([64, 128]), page=rng.choice([16, 32, 64, 128]), batch=batch,
                    max_len=max_len, new=rng.choice([1, max_len, max(1, max_len // 3)]))
    batch = _log(rng, 1, 64)
    total = _log(rng, 1, 200_000)  # keys of the sequences, together
    return dict(op="attend", dtype=rng.choice(["int8d", "int4d"]), batch=batch,
                q_len=rng.choice([1, 1, 1, 2, 4, 5]), heads=rng.choice([1, 4, 8]),
                group=rng.choice([1, 2, 4, 5, 8]), dim=rng.choice([64, 128]),
                page=rng.choice([16, 32, 64, 128]), max_len=max(1, total // batch),
                prefix=rng.choice([0, _log(rng, 1, 8192)]), empty=rng.choice([0, 0, batch // 8]))


# ── formats, in torch ────────────────────────────────────────────────────────
def _e2m1(device):
    return torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0.0, -.5, -1, -1.5, -2, -3, -4, -6],
                        device=device)


def _fp4_quantize(x, fmt):
    """(codes [rows, blocks, B] as 0..15, scale bytes [rows, blocks], g or None) of fp32 x."""
    size = 32 if fmt == "mxfp4" else 16
    rows, cols = x.shape
    x = torch.nn.functional.pad(x, (0, -cols % size)).view(rows, -1, size)
    amax = x.abs().amax(-1)
    g = None
    if fmt == "mxfp4":
        e = torch.where(amax > 0, torch.frexp(amax).exponent - 3, -127).clamp(-127, 127)
        byte = (e + 127).to(torch.uint8)
        q = torch.ldexp(x, -e[..., None])
    else:
        top = amax.amax()
        g = torch.where(top > 0, top / 2688.0, torch.ones_like(top))
        s = (amax / (6.0 * g)).clamp(max=448.0).to(torch.float8_e4m3fn)
        byte = s.view(torch.uint8)
        s = (s.float() * g)[..., None]
        q = torch.where(s > 0, x / s, torch.zeros_like(x))
    a = q.abs()
    code = ((a > .25).to(torch.uint8) + (a >= .75) + (a > 1.25) + (a >= 1.75) + (a > 2.5)
            + (a >= 3.5) + (a > 5))
    return code + 8 * torch.signbit(x).to(torch.uint8), byte, g


def _fp4_values(codes, byte, g, cols):
    """fp32 [rows, cols] of codes [rows, blocks, B] and scale bytes [rows, blocks]."""
    if g is None:
        s = torch.ldexp(torch.ones((), device=byte.device), byte.to(torch.int32) - 127)
    else:
        s = byte.contiguous().view(torch.float8_e4m3fn).float() * g
    return (_e2m1(codes.device)[codes.long()] * s[..., None]).flatten(1)[:, :cols]


def _fp4_pack(codes, byte):
    """Two codes a byte, low first, rows padded to 16 bytes; scales in 128 x 4 tiles."""
    rows, blocks = byte.shape
    flat = codes.flatten(1)
    flat = torch.nn.functional.pad(flat, (0, -flat.shape[1] % 32))
    t = torch.nn.functional.pad(byte, (0, -blocks % 4, 0, -rows % 128))
    t = t.view(t.shape[0] // 128, 4, 32, t.shape[1] // 4, 4).permute(0, 3, 2, 1, 4)
    return flat[:, 0::2] | flat[:, 1::2] << 4, t.contiguous().view(-1)


def _fp4_unpack(packed, tiles, rows, blocks, size):
    codes = torch.stack((packed & 15, packed >> 4), -1).flatten(1)[:, :blocks * size]
    t = tiles.view(-(-rows // 128), -(-blocks // 4), 32, 4, 4).permute(0, 3, 2, 1, 4)
    byte = t.reshape(-(-rows // 128) * 128, -1)[:rows, :blocks]
    return codes.view(rows, blocks, size), byte


def _kv_quantize(x, bits):
    """(packed uint8 [..., D * bits / 8], scales) of fp32 x [..., D]."""
    m = 127.0 if bits == 8 else 7.0
    si = x.abs().amax(-1, keepdim=True).clamp(min=1e-12).reciprocal() * m
    code = torch.round(x * si).to(torch.int32)
    if bits == 8:
        packed = (code & 255).to(torch.uint8)
    else:
        packed = ((code[..., 0::2] & 15) | (code[..., 1::2] & 15) << 4).to(torch.uint8)
    return packed, si.reciprocal().squeeze(-1)


def _kv_values(packed, scales, bits):
    if bits == 8:
        code = packed.view(torch.int8).float()
    else:
        code = torch.stack(((packed & 15 ^ 8).float() - 8, (packed >> 4 ^ 8).float() - 8), -1).flatten(-2)
    return code * scales[..., None]


# ── inputs ───────────────────────────────────────────────────────────────────
def _bits(case):
    return 8 if case["dtype"] == "int8d" else 4


def _lengths(case, gen):
    """Keys of each sequence: from the longest down to a quarter of it, in any order; `empty` idle slots."""
    b, top = case["batch"], case["max_len"]
    n = [max(1, top - (top - top // 4) * i // max(1, b - 1)) for i in range(b)]
    for i in range(case.get("empty", 0)):
        n[b - 1 - i] = 0
    return torch.tensor(n)[torch.randperm(b, generator=gen)]


def _gen(seed, device):
    return torch.Generator(device).manual_seed(seed)


def _pool(case, pages, rng):
    """Codes and scales as an earlier run left them: keys with a few strong channels."""
    bits, shape = _bits(case), (pages, case["heads"], case["page"])
    pool = []
    for kind in range(2):
        if bits == 8:
            c = torch.randn(*shape, case["dim"], generator=rng, device="cuda").mul_(40).clamp_(-127, 127)
            c = c.to(torch.int8).view(torch.uint8)
        else:
            c = torch.randint(0, 256, (*shape, case["dim"] // 2), generator=rng, device="cuda", dtype=torch.uint8)
            c = torch.where((c & 15) == 8, c - 7, c)  # codes are -7..7
            c = torch.where((c >> 4) == 8, c - 112, c)
        s = torch.rand(shape, generator=rng, device="cuda").add_(0.5).mul_(3.0 if kind == 0 else 2.0)
        pool += [c, s.div_(127.0 if bits == 8 else 7.0)]
    return pool


def _tables(case, gen):
    """Page tables of the sequences and of the prefix, pages in any order; pages of the pool."""
    wide, shared = -(-case["max_len"] // case["page"]), -(-case.get("prefix", 0) // case["page"])
    pages = case["batch"] * wide + shared
    order = torch.randperm(pages, generator=gen).to(torch.int32)
    return order[shared:].view(case["batch"], wide).cuda(), order[:shared].cuda(), pages


def prepare(case, seed):
    rng, gen = _gen(seed, "cuda"), _gen(seed, "cpu")
    s = dict(case=case)
    if case["op"] == "quantize":
        x = torch.randn(case["rows"], case["cols"], generator=rng, device="cuda")
        if case["dtype"] == "bf16":  # activations: a few channels are far larger
            x *= 1 + 20 * (torch.rand(case["cols"], generator=rng, device="cuda") < 0.01)
            s["x"] = x.bfloat16()
        else:
            s["x"] = x.mul_(0.02)
    elif case["op"] == "linear":
        w = torch.randn(case["n"], case["k"], generator=rng, device="cuda").mul_(0.02)
        codes, byte, s["w_g"] = _fp4_quantize(w, case["fmt"])
        s["w_codes"], s["w_scales"] = _fp4_pack(codes, byte)
        s["x"] = torch.randn(case["m"], case["k"], generator=rng, device="cuda").bfloat16()
        s["bias"] = torch.randn(case["n"], generator=rng, device="cuda") if case["bias"] else None
    else:
        table, shared, pages = _tables(case, gen)
        s["pool"] = _pool(case, pages, rng)
        s["table"], s["shared"] = table, shared
        n = _lengths(case, gen)
        s["lengths"] = n.to(torch.int32).cuda()
        if case["op"] == "cache":
            # the last `new` tokens of every sequence (fewer where it is shorter), packed one after another
            at = torch.arange(case["max_len"]).repeat(case["batch"], 1)
            fresh = (at < n[:, None]) & (at >= n[:, None] - case["new"])
            where = table.cpu().long().repeat_interleave(case["page"], 1)[:, :case["max_len"]]
            slots = where * case["page"] + at % case["page"]
            s["slots"] = slots[fresh].cuda()
            shape = (int(fresh.sum()), case["heads"], case["dim"])
            s["k"] = torch.randn(shape, generator=rng, device="cuda")
            s["k"] *= 1 + 6 * (torch.rand(shape[1:], generator=rng, device="cuda") < 0.05)
            s["k"] = s["k"].bfloat16()
            s["v"] = torch.randn(shape, generator=rng, device="cuda").bfloat16()
        else:
            s["q"] = torch.randn(case["batch"], case["q_len"], case["heads"] * case["group"], case["dim"],
                                 generator=rng, device="cuda").bfloat16()
    return s


# ── the operators ────────────────────────────────────────────────────────────
def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    import qtpytorch_b200 as mxb

    case = s["case"]
    if case["op"] == "quantize":
        t = mxb.fp4_tensor.quantize(s["x"], case["fmt"])
        return t.dequantize(s["x"].dtype)
    if case["op"] == "linear":
        w = mxb.fp4_tensor(s["w_codes"], s["w_scales"], case["fmt"], (case["n"], case["k"]), s["w_g"])
        x = mxb.fp4_tensor.quantize(s["x"], case["fmt"])
        return mxb.fp4_matmul(x, w, bias=s["bias"])
    cache = mxb.paged_kv_cache.from_buffers(*s["pool"], dtype=case["dtype"])
    if case["op"] == "cache":
        cache.write(s["k"], s["v"], s["slots"])
        return cache.read(s["table"], s["lengths"], case["max_len"])
    return mxb.paged_attention(s["q"], cache, s["table"], s["lengths"], prefix_table=s["shared"],
                               prefix_len=case["prefix"])


def _run_plain(s):
    case = s["case"]
    if case["op"] == "quantize":
        return _fp4_values(*_fp4_quantize(s["x"].float(), case["fmt"]), case["cols"]).to(s["x"].dtype)
    if case["op"] == "linear":
        x = _fp4_values(*_fp4_quantize(s["x"].float(), case["fmt"]), case["k"])
        size = 32 if case["fmt"] == "mxfp4" else 16
        codes, byte = _fp4_unpack(s["w_codes"], s["w_scales"], case["n"], -(-case["k"] // size), size)
        y = x @ _fp4_values(codes, byte, s["w_g"], case["k"]).t()
        return (y if s["bias"] is None else y + s["bias"]).bfloat16()
    return _plain_cache(s) if case["op"] == "cache" else _plain_attend(s)


def _plain_cache(s):
    case, (kc, ks, vc, vs) = s["case"], s["pool"]
    bits, page = _bits(case), case["page"]
    for codes, scales, x in ((kc, ks, s["k"]), (vc, vs, s["v"])):
        packed, sc = _kv_quantize(x.float(), bits)
        codes[s["slots"] // page, :, s["slots"] % page] = packed
        scales[s["slots"] // page, :, s["slots"] % page] = sc
    live = torch.arange(case["max_len"], device="cuda") < s["lengths"][:, None]
    back = []
    for codes, scales in ((kc, ks), (vc, vs)):
        x = _kv_values(codes[s["table"]], scales[s["table"]], bits)  # [b, pages, heads, page, dim]
        x = x.transpose(2, 3).flatten(1, 2)[:, :case["max_len"]]
        back.append(torch.where(live[:, :, None, None], x, 0.0).bfloat16())
    return back


def _plain_attend(s):
    case, (kc, ks, vc, vs) = s["case"], s["pool"]
    bits, t = _bits(case), case["q_len"]
    q = s["q"].float().unflatten(2, (case["heads"], case["group"])) / math.sqrt(case["dim"])
    at = torch.arange(s["table"].shape[1] * case["page"], device="cuda")
    seen = s["lengths"][:, None] - (t - 1 - torch.arange(t, device="cuda"))  # keys of query t
    k = _kv_values(kc[s["table"]], ks[s["table"]], bits).transpose(2, 3).flatten(1, 2)
    score = torch.einsum("bthgd,blhd->bhgtl", q, k)
    score = score.masked_fill((at >= seen[..., None])[:, None, None], float("-inf"))
    p, n = case["prefix"], score.shape[-1]
    if p:
        kp = _kv_values(kc[s["shared"]], ks[s["shared"]], bits).transpose(1, 2).flatten(0, 1)[:p]
        score = torch.cat((score, torch.einsum("bthgd,lhd->bhgtl", q, kp)), -1)
    top = score.amax(-1, keepdim=True)
    w = torch.exp(score - torch.where(top == float("-inf"), 0.0, top))
    total = w.sum(-1, keepdim=True)
    w = torch.where(total > 0, w / total, 0.0)
    v = _kv_values(vc[s["table"]], vs[s["table"]], bits).transpose(2, 3).flatten(1, 2)
    o = torch.einsum("bhgtl,blhd->bthgd", w[..., :n], v)
    if p:
        vp = _kv_values(vc[s["shared"]], vs[s["shared"]], bits).transpose(1, 2).flatten(0, 1)[:p]
        o = o + torch.einsum("bhgtl,lhd->bthgd", w[..., n:], vp)
    return o.flatten(2, 3).bfloat16()


# ── what a pass cannot do without ────────────────────────────────────────────
def work(case):
    if case["op"] == "quantize":
        n, size = case["rows"] * case["cols"], 2 if case["dtype"] == "bf16" else 4
        store = n / 2 + n / (32 if case["fmt"] == "mxfp4" else 16)
        # x is read, its codes are written; they are read back, the values written
        return {"bytes": 2 * n * size + 2 * store, "flops": 4 * n}
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        per = 0.5 + 1 / (32 if case["fmt"] == "mxfp4" else 16)
        return {"bytes": 2 * m * k + per * n * k + 2 * m * n + (4 * n if case["bias"] else 0),
                "flops": 2 * m * n * k}
    n = _lengths(case, _gen(0, "cpu"))
    row = case["dim"] * _bits(case) / 8 + 4  # a token's key or value in one head
    if case["op"] == "cache":
        fresh, live = int(n.clamp(max=case["new"]).sum()), int(n.sum())
        dense = case["batch"] * case["max_len"] * case["dim"] * 2
        return {"bytes": 2 * case["heads"] * (fresh * (case["dim"] * 2 + row) + live * row + dense),
                "flops": 2 * case["heads"] * case["dim"] * (4 * fresh + live)}
    rows = case["q_len"] * case["group"] * case["heads"]
    keys = int(n.sum()) + case["prefix"]
    return {"bytes": 2 * case["heads"] * keys * row + 4 * case["batch"] * rows * case["dim"],
            "flops": 4 * rows * case["dim"] * (int(n.sum()) + case["batch"] * case["prefix"])}


# ── 64 bits ──────────────────────────────────────────────────────────────────
def _exact_fp4(x, fmt):
    """The quantized x as the values it stands for: nearest grid point by distance, in 64 bits."""
    x = x.double()
    rows, cols = x.shape
    size = 32 if fmt == "mxfp4" else 16
    blocks = torch.zeros(rows, -(-cols // size) * size, dtype=torch.float64, device=x.device)
    blocks[:, :cols] = x
    blocks = blocks.view(-1, size)
    amax = blocks.abs().max(1, keepdim=True).values
    if fmt == "mxfp4":
        scale = torch.exp2((torch.floor(torch.log2(amax)) - 2).clamp(-127, 127))
    else:
        g = amax.max() / 2688
        want = torch.clamp(amax / (6 * g), max=448)  # e4m3: 3 bits after the point, 2^-9 steps below 2^-6
        step = torch.exp2(torch.floor(torch.log2(want)).clamp(min=-6) - 3)
        scale = torch.round(want / step) * step * g
    grid = torch.tensor([0, 1, 2, 4, 6, .5, 1.5, 3], dtype=torch.float64, device=x.device)  # even codes first
    u = blocks.abs() / torch.where(scale > 0, scale, 1)
    best, off = torch.zeros_like(u), u.clone()
    for value in grid[1:]:  # a later (odd) code has to be strictly nearer
        d = (u - value).abs()
        nearer = d < off
        best, off = torch.where(nearer, value, best), torch.where(nearer, d, off)
    out = torch.where(scale > 0, best * scale, 0) * torch.sign(blocks)
    return out.view(rows, -1)[:, :cols]


def _exact_weight(s, case):
    """The stored weight, by looking each byte up."""
    n, k = case["n"], case["k"]
    size = 32 if case["fmt"] == "mxfp4" else 16
    grid = [0, .5, 1, 1.5, 2, 3, 4, 6]
    value = torch.tensor(grid + [-v for v in grid], dtype=torch.float64, device="cuda")
    byte = s["w_codes"].long()
    w = torch.empty(n, 2 * byte.shape[1], dtype=torch.float64, device="cuda")
    w[:, 0::2], w[:, 1::2] = value[byte % 16], value[byte // 16]
    if case["fmt"] == "mxfp4":
        known = [2.0 ** (b - 127) for b in range(256)]
    else:
        known = [((b & 7) / 8 + (b >= 8)) * 2.0 ** (max(b >> 3, 1) - 7) for b in range(128)] + [0.0] * 128
    known = torch.tensor(known, dtype=torch.float64, device="cuda")
    r, c = torch.arange(n, device="cuda")[:, None], torch.arange(k, device="cuda")[None] // size
    place = ((r // 128) * -(-(-(-k // size)) // 4) + c // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + c % 4
    scale = known[s["w_scales"][place].long()]
    return w[:, :k] * scale * (1.0 if s["w_g"] is None else s["w_g"].double())


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


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantize":
        return _exact_fp4(s["x"], case["fmt"])
    if case["op"] == "linear":
        y = torch.mm(_exact_fp4(s["x"], case["fmt"]), _exact_weight(s, case).t())
        return y if s["bias"] is None else y + s["bias"].double()
    kc, ks, vc, vs = s["pool"]
    bits, page, heads, dim = _bits(case), case["page"], case["heads"], case["dim"]
    lengths = s["lengths"].tolist()
    if case["op"] == "cache":
        back, top = [], 127.0 if bits == 8 else 7.0
        for codes, scales, x in ((kc, ks, s["k"]), (vc, vs, s["v"])):
            x = x.double()
            si = top / x.abs().max(-1, keepdim=True).values.clamp(min=1e-12)
            pool = _exact_kv(codes, scales, bits).transpose(1, 2).reshape(-1, heads, dim)  # by slot
            pool[s["slots"]] = torch.round(x * si) / si
            out = torch.zeros(case["batch"], case["max_len"], heads, dim, dtype=torch.float64, device="cuda")
            for b, n in enumerate(lengths):
                at = torch.arange(n, device="cuda")
                out[b, :n] = pool[s["table"][b].long()[at // page] * page + at % page]
            back.append(out)
        return back
    out = torch.zeros(case["batch"], case["q_len"], heads, case["group"], dim, dtype=torch.float64, device="cuda")
    q = s["q"].double().view(out.shape)

    def keys(pages, n, codes, scales):  # [heads, n, dim]
        x = _exact_kv(codes[pages.long()], scales[pages.long()], bits)
        return x.transpose(0, 1).reshape(heads, -1, dim)[:, :n]

    first = [keys(s["shared"], case["prefix"], c, x) for c, x in ((kc, ks), (vc, vs))]
    for b, n in enumerate(lengths):
        k, v = (torch.cat((f, keys(s["table"][b], n, c, x)), 1) for f, (c, x) in zip(first, ((kc, ks), (vc, vs))))
        for t in range(case["q_len"]):
            live = case["prefix"] + max(0, n - (case["q_len"] - 1 - t))
            if live:
                a = torch.softmax(torch.matmul(q[b, t], k[:, :live].transpose(1, 2)) / dim ** 0.5, -1)
                out[b, t] = torch.matmul(a, v[:, :live])
    return out.flatten(2, 3)
