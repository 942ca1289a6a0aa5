"""The operators of the 4-bit state cache, in their plain form and through the framework.

A state's keys and values can be kept in 4 bits in pages of a pool. Five operators work on it:

``rotate``    per-head RMSNorm of queries and keys with a rotary embedding whose frequencies take
              their positions from several axes (time, height, width), in one pass;
``store``     quantise rows of K and V into slots of the pool, and read a sequence's rows back;
``decode``    attention of one or a few new tokens of many sequences, each over its own pages;
``question``  attention of question blocks over one state in pages and over each block's own keys;
``pages``     copy pages in every layer (a fork's last page), or move them and rewrite the tables.

The pool is uint8 [layers, pages, page_bytes]. A page holds, per kv head, page_tokens / 16 granules
of 16 tokens; a granule is

    K codes [16, D/2], K scales [16, D/16], K exponents [16],
    V codes [16, D/2], V scales [D/16, 16], V exponents [16]

with two e2m1 codes a byte (the even channel in the low half), one e4m3 scale for 16 channels and
one power of two (biased by 127; 255 marks a row that held a NaN or an infinity) for a token's row:
value = code * scale * 2^(exponent - 127).
"""

import math

import numpy as np
import torch

own = False

E_MIN = -64  # smallest row exponent
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one new token of one request at the model's attention shape: latency
        {"name": "rotate_1x1_d256", "op": "rotate", "rows": 1, "tokens": 1, "heads": 24, "kv_heads": 4, "dim": 256,
         "sections": "11,11,10", "far": 5000, "type": "bf16"},
        # the question pass: 255 blocks of 47 tokens behind a long state, image positions
        {"name": "rotate_255x47_d128", "op": "rotate", "rows": 255, "tokens": 47, "heads": 32, "kv_heads": 4, "dim": 128,
         "sections": "6,5,5", "far": 200000, "type": "bf16"},
        # a short block of a small model joins a cached sequence
        {"name": "store_33_d64", "op": "store", "tokens": 33, "kv_heads": 2, "dim": 64, "page": 16, "type": "fp16"},
        # a whole state goes into the cache after its pass, and is read for a pass in 16 bits
        {"name": "store_16384_d128", "op": "store", "tokens": 16384, "kv_heads": 4, "dim": 128, "page": 64,
         "type": "bf16"},
        # one token of one request over a short state: latency
        {"name": "decode_1x1_997_d256", "op": "decode", "rows": 1, "tokens": 1, "causal": False, "heads": 24,
         "kv_heads": 4, "dim": 256, "page": 16, "longest": 997, "type": "bf16"},
        # five proposed tokens of three requests, checked against long caches
        {"name": "decode_3x5_98765_d256", "op": "decode", "rows": 3, "tokens": 5, "causal": True, "heads": 24,
         "kv_heads": 4, "dim": 256, "page": 32, "longest": 98765, "type": "bf16"},
        # a full serving batch of ragged lengths
        {"name": "decode_64x1_16384_d128", "op": "decode", "rows": 64, "tokens": 1, "causal": False, "heads": 32,
         "kv_heads": 4, "dim": 128, "page": 64, "longest": 16384, "type": "bf16"},
        # one short question over a resident state
        {"name": "question_1x11_4096_d128", "op": "question", "rows": 1, "tokens": 11, "heads": 32, "kv_heads": 4,
         "dim": 128, "page": 64, "state": 4096, "type": "bf16"},
        # a ragged batch at the model's attention shape, a state that ends inside a page
        {"name": "question_31x37_3001_d256", "op": "question", "rows": 31, "tokens": 37, "heads": 24, "kv_heads": 4,
         "dim": 256, "page": 32, "state": 3001, "type": "fp16"},
        # the whole question batch over a 4096-token state
        {"name": "question_255x48_4096_d128", "op": "question", "rows": 255, "tokens": 48, "heads": 32, "kv_heads": 4,
         "dim": 128, "page": 64, "state": 4096, "type": "bf16"},
        # eight forks of a sequence copy its last page in each of 16 layers
        {"name": "pages_fork_8x16", "op": "pages", "moved": 8, "pages": 64, "layers": 16, "kv_heads": 4, "dim": 128,
         "page": 64, "rows": 0, "width": 0},
        # a cache that half emptied moves its live pages to the front, under 64 tables
        {"name": "pages_compact_700x16", "op": "pages", "moved": 700, "pages": 2000, "layers": 16, "kv_heads": 4,
         "dim": 128, "page": 64, "rows": 64, "width": 31},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over the logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    op = rng.choice(["rotate", "store", "decode", "decode", "question", "question", "pages"])
    kv = rng.choice([1, 2, 4, 8])
    dim = rng.choice([64, 128, 256])
    page = rng.choice([16, 32, 64, 128])
    kind = rng.choice(["bf16", "fp16"])
    group = rng.choice([1, 2, 3, 4, 6, 7, 8, 12, 16])
    if op == "rotate":
        half = rng.choice([n for n in (8, 16, 32, 64, 128) if 2 * n <= dim])
        axes = rng.choice([1, 2, 3])
        cuts = sorted(rng.sample(range(1, half), axes - 1))
        sections = [b - a for a, b in zip([0] + cuts, cuts + [half])]
        rows = _spread(rng, 1, 255)
        tokens = _spread(rng, 1, max(1, 30_000_000 // (rows * kv * (group + 1) * dim)))
        return {"op": op, "rows": rows, "tokens": min(tokens, 20000), "heads": kv * group, "kv_heads": kv, "dim": dim,
                "sections": ",".join(str(s) for s in sections), "far": _spread(rng, 10, 1000000), "type": kind}
    if op == "store":
        return {"op": op, "tokens": _spread(rng, 1, 8_000_000 // (kv * dim)), "kv_heads": kv, "dim": dim,
                "page": page, "type": kind}
    if op == "decode":
        tokens = rng.choice([1, 1, 1, 2, 3, 4, 8])
        rows = _spread(rng, 1, 64)
        longest = _spread(rng, tokens, 400_000_000 // (rows * kv * dim * max(1, group * tokens // 16)))
        return {"op": op, "rows": rows, "tokens": tokens, "causal": rng.random() < 0.5, "heads": kv * group,
                "kv_heads": kv, "dim": dim, "page": page, "longest": min(longest, 100000), "type": kind}
    if op == "question":
        state = _spread(rng, 1, 16384)
        rows = _spread(rng, 1, 255)
        most = 1_500_000_000 // ((state + 64) * rows * kv * group * max(1, dim // 128))
        return {"op": op, "rows": rows, "tokens": _spread(rng, 1, max(1, min(64, most))), "heads": kv * group,
                "kv_heads": kv, "dim": dim, "page": page, "state": state, "type": kind}
    moved = _spread(rng, 1, 400)
    rows = rng.choice([0, 1, 5, 33])
    return {"op": op, "moved": moved, "pages": 2 * moved + rng.randrange(1, 200), "layers": rng.choice([1, 3, 16]),
            "kv_heads": kv, "dim": dim, "page": page, "rows": rows, "width": rng.randrange(1, 60) if rows else 0}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _page_bytes(c):
    return c["kv_heads"] * (c["page"] // 16) * _granule(c["dim"])


def _granule(dim):
    return 32 * (dim // 2 + dim // 16 + 1)


def _quantise(x):
    """(codes [..., D/2], scales [..., D/16], exponents [...]), all uint8, of float32 rows [..., D]."""
    top = x.abs().amax(-1)
    bad = ~torch.isfinite(x).all(-1)
    part, power = torch.frexp(torch.where(bad, 0.0, top))
    # the smallest power of two that brings the row's largest magnitude to 6 * 448 or less
    power = torch.where(part <= 2688 / 4096, power - 12, power - 11)
    power = torch.where(top > 0, power, E_MIN).clamp(E_MIN, 127)
    rows = torch.where(bad[..., None], 0.0, torch.ldexp(x, -power[..., None]))
    groups = rows.unflatten(-1, (-1, 16))
    scale = (groups.abs().amax(-1) / 6).to(torch.float8_e4m3fn)
    wide = scale.float()[..., None]
    part = torch.where(wide > 0, groups / wide, 0.0)
    a = part.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
            + (part < 0).to(torch.uint8) * 8).flatten(-2)
    exponent = torch.where(bad, 255, power + 127).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale.view(torch.uint8), exponent


def _pack(k, v):
    """Granule bytes [..., granule] of float32 K and V [..., 16, D]."""
    kc, ks, ke = _quantise(k)
    vc, vs, ve = _quantise(v)
    return torch.cat([kc.flatten(-2), ks.flatten(-2), ke, vc.flatten(-2), vs.transpose(-1, -2).flatten(-2), ve], -1)


def _noise(shape, generator):
    return torch.randn(shape, generator=generator, device="cuda")


def _pool(c, pages, filled, generator):
    """A layer's pool [1, pages, page_bytes] whose tokens are real keys and values where ``filled`` [pages, page],
    and rows marked as not finite elsewhere (what a page's last owner left must not matter)."""
    heads, dim, grains = c["kv_heads"], c["dim"], c["page"] // 16
    out = torch.empty(1, pages, _page_bytes(c), dtype=torch.uint8, device="cuda")
    loud = 1 + 3 * (torch.rand(heads, 1, 1, dim, generator=generator, device="cuda") < 0.03).float()
    live = filled.view(pages, 1, grains, 16, 1)
    step = max(1, (1 << 27) // (heads * c["page"] * dim))
    for at in range(0, pages, step):
        n = min(step, pages - at)
        rows = live[at:at + n]
        k = torch.where(rows, _noise((n, heads, grains, 16, dim), generator) * loud, math.nan)
        v = torch.where(rows, _noise((n, heads, grains, 16, dim), generator) * 0.5, math.nan)
        out[0, at:at + n] = _pack(k, v).flatten(1)
    return out


def _tables(c, lengths, generator):
    """(page tables [rows, width] with -1 behind a row's last page, filled [pages, page])."""
    page = c["page"]
    lengths = torch.tensor(lengths)
    need = (lengths + page - 1) // page
    width = max(1, int(need.max()))
    pages = int(need.sum()) + 3
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(generator.initial_seed()))
    used = torch.arange(width)[None] < need[:, None]
    table = torch.full((len(need), width), -1, dtype=torch.int32)
    table[used] = order[:int(need.sum())].to(torch.int32)
    filled = torch.zeros(pages, page, dtype=torch.bool)
    tokens = torch.arange(width * page).view(1, width, page) < lengths[:, None, None]
    filled[table[used].long()] = tokens[used]
    return table.cuda(), filled.cuda()


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(seed)
    host = np.random.default_rng(seed)
    s = {"case": c, "op": c["op"]}
    dtype = TYPES.get(c.get("type"))
    if c["op"] == "rotate":
        rows, tokens, dim = c["rows"], c["tokens"], c["dim"]
        sections = [int(n) for n in c["sections"].split(",")]
        half = sum(sections)
        # the query half of a projection that also holds the output gate, as the model's layers leave it
        s["q"] = _noise((rows, tokens, c["heads"], 2 * dim), g).to(dtype)[..., :dim]
        s["k"] = _noise((rows, tokens, c["kv_heads"], dim), g).to(dtype)
        s["wq"], s["wk"] = (0.1 * _noise((dim,), g)).to(dtype), (0.1 * _noise((dim,), g)).to(dtype)
        s["freq"] = 1e7 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
        s["freq"] = s["freq"].float()
        start = torch.randint(0, c["far"], (len(sections), rows, 1), generator=g, device="cuda")
        s["at"] = start + torch.arange(tokens, device="cuda") // torch.tensor([1, 3, 2], device="cuda")[:len(sections), None, None]
        # axis 0 everywhere, the others each third frequency until their share is spent
        axes = [0] * half
        for a, n in enumerate(sections[1:], 1):
            for i in range(n):
                if a + 3 * i < half:
                    axes[a + 3 * i] = a
        s["axes"], s["axis"] = tuple(axes), torch.tensor(axes, device="cuda")
        s["eps"] = 1e-6
    elif c["op"] == "store":
        n, heads, dim, page = c["tokens"], c["kv_heads"], c["dim"], c["page"]
        pages = -(-n // page)
        table = torch.randperm(pages + 2, generator=g, device="cuda")[:pages]
        at = torch.arange(n, device="cuda")
        s["table"] = table.to(torch.int32)
        s["slots"] = table[at // page] * page + at % page
        s["pool"] = torch.randint(0, 256, (1, pages + 2, _page_bytes(c)), generator=g, device="cuda", dtype=torch.uint8)
        # K and V side by side, as one projection leaves them
        rows = _noise((n, 2 * heads, dim), g) * torch.exp(0.5 * _noise((n, 2 * heads, 1), g))
        rows = (rows * (1 + 5 * (torch.rand(2 * heads, dim, generator=g, device="cuda") < 0.02))).to(dtype)
        s["k"], s["v"] = rows[:, :heads], rows[:, heads:]
    elif c["op"] == "decode":
        low = c["tokens"]
        lengths = [int(x) for x in host.integers(max(low, c["longest"] // 2), c["longest"] + 1, c["rows"])]
        lengths[int(host.integers(0, c["rows"]))] = c["longest"]
        s["table"], filled = _tables(c, lengths, g)
        s["pool"] = _pool(c, filled.shape[0], filled, g)
        s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        s["q"] = _noise((c["rows"], c["tokens"], c["heads"], c["dim"]), g).to(dtype).transpose(1, 2)
        s["scale"] = c["dim"] ** -0.5
    elif c["op"] == "question":
        table, filled = _tables(c, [c["state"]], g)
        s["table"] = table[0]
        s["pool"] = _pool(c, filled.shape[0], filled, g)
        lengths = host.integers(max(1, c["tokens"] // 2), c["tokens"] + 1, c["rows"])
        lengths[int(host.integers(0, c["rows"]))] = c["tokens"]
        s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        s["q"], s["k"], s["v"] = ((_noise((c["rows"], c["tokens"], n, c["dim"]), g)).to(dtype).transpose(1, 2)
                                  for n in (c["heads"], c["kv_heads"], c["kv_heads"]))
        s["scale"] = c["dim"] ** -0.5
    else:
        pages, moved = c["pages"], c["moved"]
        s["pool"] = torch.randint(0, 256, (c["layers"], pages, _page_bytes(c)), generator=g, device="cuda",
                                  dtype=torch.uint8)
        order = host.permutation(pages)
        src, dst = np.sort(order[:moved]), order[moved:2 * moved]
        s["src"] = torch.tensor(src, dtype=torch.int32, device="cuda")
        s["dst"] = torch.tensor(dst, dtype=torch.int32, device="cuda")
        s["tables"] = None
        if c["rows"]:
            kept = np.concatenate([src, order[2 * moved:], [-1]])
            s["tables"] = torch.tensor(host.choice(kept, (c["rows"], c["width"])), dtype=torch.int32, device="cuda")
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    if own:
        return _framework(state)
    return {"rotate": _rotate, "store": _store, "decode": _decode, "question": _question, "pages": _pages}[state["op"]](state)


def _framework(s):
    from d3_turbo_trt_b200.kernels import kv4
    from d3_turbo_trt_b200.model import fused

    c = s["case"]
    if s["op"] == "rotate":
        return fused.qk_norm_mrope(s["q"], s["k"], s["wq"], s["wk"], s["at"], s["freq"], s["axes"], s["eps"])
    cache = kv4.Kv4Cache.over(s["pool"], kv_heads=c["kv_heads"], head_dim=c["dim"], page_tokens=c["page"])
    if s["op"] == "store":
        cache.append(0, s["k"], s["v"], s["slots"])
        return cache.read(0, s["table"], c["tokens"], dtype=s["k"].dtype)
    if s["op"] == "decode":
        return kv4.decode_attention(s["q"], cache, 0, s["table"], s["lengths"], scale=s["scale"], causal=c["causal"])
    if s["op"] == "question":
        return kv4.question_attention(s["q"], cache, 0, s["table"], c["state"], s["k"], s["v"], s["lengths"],
                                      scale=s["scale"])
    if s["tables"] is None:
        cache.copy_pages(s["src"], s["dst"])
        return s["pool"]
    cache.move_pages(s["src"], s["dst"], s["tables"])
    return s["pool"], s["tables"]


def _rotate(s):
    # angles in 64 bits: at position 200000 a 32-bit product is off by 0.008 rad
    angle = (s["at"].double().permute(1, 2, 0)[..., s["axis"]] * s["freq"].double())[:, :, None]
    cos, sin, half = angle.cos().float(), angle.sin().float(), s["freq"].numel()
    return _turned(s["q"], s["wq"], cos, sin, half, s["eps"]), _turned(s["k"], s["wk"], cos, sin, half, s["eps"])


def _turned(x, weight, cos, sin, half, eps):
    wide = x.float()
    y = wide * torch.rsqrt(wide.square().mean(-1, keepdim=True) + eps) * (1 + weight.float())
    a, b = y[..., :half], y[..., half:2 * half]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, y[..., 2 * half:]], -1).to(x.dtype)


def _parts(granules, dim):
    """K and V (codes [..., 16, D/2], scales [..., 16, D/16], exponents [..., 16]) of granule bytes."""
    sizes, at, out = [8 * dim, dim, 16] * 2, 0, []
    for n in sizes:
        out.append(granules[..., at:at + n])
        at += n
    return ((out[0].unflatten(-1, (16, -1)), out[1].unflatten(-1, (16, -1)), out[2]),
            (out[3].unflatten(-1, (16, -1)), out[4].unflatten(-1, (-1, 16)).transpose(-1, -2), out[5]))


def _values(codes, scales, exponents):
    """float32 rows [..., 16, D]."""
    steps = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    x = torch.stack([steps[(codes & 15).int()], steps[(codes >> 4).int()]], -1).flatten(-2)
    x = x.unflatten(-1, (-1, 16)) * scales.contiguous().view(torch.float8_e4m3fn).float()[..., None]
    power = torch.ldexp(torch.ones_like(exponents, dtype=torch.float32), exponents.int() - 127)
    return x.flatten(-2) * torch.where(exponents == 255, math.nan, power)[..., None]


def _rows(s, table):
    """float32 K and V [..., kv_heads, width * page, D] of the pages in ``table`` [..., width]."""
    c = s["case"]
    taken = s["pool"][0][table.clamp(min=0).long()]
    taken = taken.unflatten(-1, (c["kv_heads"], c["page"] // 16, _granule(c["dim"]))).movedim(-3, -4)
    return tuple(_values(*part).flatten(-4, -2) for part in _parts(taken, c["dim"]))


def _store(s):
    c = s["case"]
    (page, dim, heads, n) = c["page"], c["dim"], c["kv_heads"], c["tokens"]
    slot = s["slots"]
    grain, row = (slot // 16)[:, None], (slot % 16)[:, None, None]
    # [pages, heads, grains, granule] seen as [pages * grains, heads, granule] for whole-granule indexing
    pool = s["pool"][0].view(-1, heads, page // 16, _granule(dim))
    where = (grain // (page // 16), torch.arange(heads, device=slot.device)[None], grain % (page // 16))
    at = 0
    for x, turned in ((s["k"], False), (s["v"], True)):
        codes, scales, exponents = _quantise(x.float())
        wide = torch.arange(dim // 2, device=slot.device)
        pool[(*(w[..., None] for w in where), at + row * (dim // 2) + wide)] = codes
        small = torch.arange(dim // 16, device=slot.device)
        place = small * 16 + row if turned else row * (dim // 16) + small
        pool[(*(w[..., None] for w in where), at + 8 * dim + place)] = scales
        pool[(*where, at + 9 * dim + row[..., 0])] = exponents
        at += 9 * dim + 16
    k, v = _rows(s, s["table"])
    return k[:, :n].to(s["k"].dtype), v[:, :n].to(s["k"].dtype)


def _softmax_rows(scores, seen):
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top > -math.inf, top, 0.0))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total > 0, total, 1.0)


def _decode(s):
    c = s["case"]
    k, v = _rows(s, s["table"])
    at = torch.arange(k.shape[-2], device=k.device)
    held = (at < s["lengths"][:, None])[:, None, :, None]
    k, v = torch.where(held, k, 0.0), torch.where(held, v, 0.0)
    limit = s["lengths"][:, None].expand(-1, c["tokens"])
    if c["causal"]:  # token i of n sees what stands before it and itself
        limit = limit - torch.arange(c["tokens"] - 1, -1, -1, device=k.device)
    seen = at < limit[..., None]  # [rows, tokens, width]
    q = s["q"].float().unflatten(1, (c["kv_heads"], -1))  # [rows, kv, group, tokens, D]
    scores = (q.flatten(2, 3) @ k.transpose(-1, -2)).unflatten(2, (-1, c["tokens"]))
    p = _softmax_rows(scores * s["scale"], seen[:, None, None])
    out = (p.flatten(2, 3) @ v).unflatten(2, (-1, c["tokens"]))
    return out.flatten(1, 2).to(s["q"].dtype)


def _question(s):
    c, kv = s["case"], s["case"]["kv_heads"]
    k, v = (x[:, :c["state"]] for x in _rows(s, s["table"]))
    # rows of one kv head side by side: [kv, rows * group * tokens, D]
    q = s["q"].float().unflatten(1, (kv, -1))
    flat = q.transpose(0, 1).flatten(1, 3)
    far = (flat @ k.transpose(-1, -2)).unflatten(1, (c["rows"], -1))  # [kv, rows, group * tokens, state]
    near = (q.flatten(2, 3) @ s["k"].float().transpose(-1, -2)).transpose(0, 1)
    real = torch.arange(c["tokens"], device=q.device) < s["lengths"][:, None]
    seen = torch.cat([torch.ones(c["rows"], c["state"], dtype=torch.bool, device=q.device), real], -1)
    p = _softmax_rows(torch.cat([far, near], -1) * s["scale"], seen[:, None])
    out = (p[..., :c["state"]].flatten(1, 2) @ v).unflatten(1, (c["rows"], -1))
    out = out + p[..., c["state"]:] @ s["v"].float().transpose(0, 1)
    out = out.transpose(0, 1).unflatten(2, (-1, c["tokens"])).flatten(1, 2)
    return torch.where(real[:, None, :, None], out, 0.0).to(s["q"].dtype)


def _pages(s):
    s["pool"][:, s["dst"].long()] = s["pool"][:, s["src"].long()]
    if s["tables"] is None:
        return s["pool"]
    to = torch.arange(s["case"]["pages"], dtype=torch.int32, device=s["src"].device)
    to[s["src"].long()] = s["dst"]
    tables = s["tables"]
    tables.copy_(torch.where(tables >= 0, to[tables.clamp(min=0).long()], tables))
    return s["pool"], tables


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    c = case
    if c["op"] == "rotate":
        values = c["rows"] * c["tokens"] * (c["heads"] + c["kv_heads"]) * c["dim"]
        axes = c["sections"].count(",") + 1
        return {"bytes": 4 * values + 8 * axes * c["rows"] * c["tokens"], "flops": 10 * values}
    if c["op"] == "pages":
        return {"bytes": 2 * c["moved"] * c["layers"] * _page_bytes(c) + 8 * c["rows"] * c["width"] + 8 * c["moved"],
                "flops": 0}
    token = c["kv_heads"] * _granule(c["dim"]) / 16  # a token's bytes in the cache, K and V
    if c["op"] == "store":
        wide = 4 * c["tokens"] * c["kv_heads"] * c["dim"]  # K and V in 16 bits
        return {"bytes": 2 * wide + 2 * c["tokens"] * token + 8 * c["tokens"], "flops": 0}
    wide = c["rows"] * c["tokens"] * c["dim"]
    if c["op"] == "decode":
        # lengths are spread evenly over the upper half of the range
        keys = c["rows"] * 0.75 * c["longest"]
        return {"bytes": keys * token + 4 * wide * c["heads"],
                "flops": 4 * keys * c["tokens"] * c["heads"] * c["dim"]}
    keys = c["state"] + 0.75 * c["tokens"]
    return {"bytes": c["state"] * token + 4 * wide * (c["heads"] + c["kv_heads"]),
            "flops": 4 * 0.75 * wide * c["heads"] * keys}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"rotate": _exact_rotate, "store": _exact_store, "decode": _exact_decode, "question": _exact_question,
            "pages": lambda s: None}[s["op"]](s)


def _exact_rotate(s):
    half, out = s["freq"].numel(), []
    for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])):
        y = x.double()
        y = y / (y.pow(2).sum(-1, keepdim=True) / y.shape[-1] + s["eps"]).sqrt() * (w.double() + 1)
        turned = y.clone()
        for i in range(half):
            a = s["at"][s["axes"][i]].double() * float(s["freq"][i])
            z = torch.polar(torch.ones_like(a), a)[..., None] * torch.complex(y[..., i], y[..., i + half])
            turned[..., i], turned[..., i + half] = z.real, z.imag
        out.append(turned)
    return tuple(out)


def _exact_store(s):
    """What a row turns into: each magnitude goes to the nearest of the code's values times its group's scale."""
    if s["k"].numel() > 1 << 23:
        return None
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device="cuda", dtype=torch.float64)
    out = []
    for x in (s["k"], s["v"]):
        x = x.double()
        top = x.abs().amax(-1, keepdim=True)
        unit = torch.exp2(torch.ceil(torch.log2(top / 2688)).clamp(E_MIN, 127))
        unit = torch.where(top > 2688 * unit, 2 * unit, torch.where(2 * top <= 2688 * unit, unit / 2, unit))
        y = (x / unit).unflatten(-1, (-1, 16))
        scale = (y.abs().amax(-1) / 6).to(torch.float32).to(torch.float8_e4m3fn).double()[..., None]
        far = (y.abs()[..., None] - scale[..., None] * grid).abs()
        # of two codes equally near, the even one
        even = torch.tensor([0, 1] * 4, device="cuda", dtype=torch.float64)
        least = far.amin(-1, keepdim=True)
        code = torch.where(far == least, even, 2.0).argmin(-1)
        value = torch.where(scale > 0, grid[code] * scale, 0.0) * torch.sign(y)
        out.append((value.flatten(-2) * unit).transpose(0, 1))
    return tuple(out)


def _exact_cache(s, pages, count):
    """K and V [kv_heads, count, D] in 64 bits of one sequence, byte by byte from the layout."""
    c, dim = s["case"], s["case"]["dim"]
    t = torch.arange(count, device="cuda")
    page = pages.long()[t // c["page"]]
    bytes_ = s["pool"][0].view(-1, c["kv_heads"], c["page"] // 16, _granule(dim))
    grains = bytes_[page, :, (t % c["page"]) // 16].transpose(0, 1)  # [kv_heads, count, granule]
    row = (t % 16)[None, :, None].expand(c["kv_heads"], -1, -1)
    out = []
    for which in (0, 1):
        base = which * (9 * dim + 16)
        channel = torch.arange(dim, device="cuda")
        pair = grains.gather(2, (base + row * (dim // 2) + channel // 2))
        code = (pair.int() >> (4 * (channel % 2))) & 15
        low, high = code & 1, (code >> 1) & 3
        size = torch.where(high == 0, 0.5 * low, (1 + 0.5 * low) * 2.0 ** (high - 1)).double()
        group = channel // 16
        place = group * 16 + row if which else row * (dim // 16) + group
        byte = grains.gather(2, base + 8 * dim + place).int()
        power, tail = byte >> 3, (byte & 7).double()
        scale = torch.where(power == 0, tail / 8 * 2.0 ** -6, (1 + tail / 8) * 2.0 ** (power.double() - 7))
        unit = 2.0 ** (grains.gather(2, base + 9 * dim + row).double() - 127)
        out.append(torch.where(code >= 8, -size, size) * scale * unit)
    return out


def _exact_decode(s):
    c = s["case"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    group = c["heads"] // c["kv_heads"]
    for b in range(c["rows"]):
        n = int(s["lengths"][b])
        k, v = _exact_cache(s, s["table"][b], n)
        for i in range(c["tokens"]):
            m = n - (c["tokens"] - 1 - i) if c["causal"] else n
            q = s["q"][b, :, i].double().view(c["kv_heads"], group, -1)
            p = torch.softmax(torch.einsum("hgd,hsd->hgs", q, k[:, :m]) * s["scale"], -1)
            out[b, :, i] = torch.einsum("hgs,hsd->hgd", p, v[:, :m]).flatten(0, 1)
    return out


def _exact_question(s):
    c = s["case"]
    if c["rows"] * c["tokens"] * c["heads"] * c["state"] * c["dim"] > 1 << 39:
        return None
    k, v = _exact_cache(s, s["table"], c["state"])
    group = c["heads"] // c["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b in range(c["rows"]):
        n = int(s["lengths"][b])
        keys = torch.cat([k, s["k"][b, :, :n].double()], 1).repeat_interleave(group, 0)
        values = torch.cat([v, s["v"][b, :, :n].double()], 1).repeat_interleave(group, 0)
        p = torch.softmax(s["q"][b, :, :n].double() @ keys.transpose(1, 2) * s["scale"], -1)
        out[b, :, :n] = p @ values
    return out
