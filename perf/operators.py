"""The operators of token generation over a paged key-value cache, as cases to
time: rotary positions, the quantised cache's write and read, and the
attention of one new token over the cache.

``run`` computes them in their plain form (elementary torch operations) or,
with ``own`` set, through chimera_b200.attention.

Heads of width 128 are the framework's own vector width, and 64 and 96 the
other widths its build takes.  Lengths from 300 to 2,000 are its long
documents, 128 its batch of queries; the rest are generic serving sizes.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "int8": torch.int8,
         "e4m3": torch.float8_e4m3fn}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4, "int8": 1, "e4m3": 1}
TOP = {"int8": 127.0, "e4m3": 448.0}  # the largest code of an 8-bit cache
SMALLEST = 2.0 ** -96  # vectors whose largest value is below this are held as zeros


# ---- the cases ---------------------------------------------------------------

def listed():
    rope = {"op": "rotary", "batch": 1, "tokens": 1, "q_heads": 32, "k_heads": 8, "dim": 128, "rot": 128,
            "interleaved": False, "inverse": False, "type": "bf16", "stretch": 1.0, "far": 4096}
    cache = {"op": "cache", "tokens": 1, "heads": 8, "dim": 128, "page": 16, "in": "bf16", "held": "int8",
             "out": "bf16"}
    att = {"op": "attention", "batch": 1, "len": 97, "ragged": False, "q_heads": 32, "k_heads": 8, "dim": 128,
           "page": 16, "type": "bf16", "held": "bf16", "token_major": False}
    return [
        # one sequence generates its next token
        {**rope, "name": "rotary_one_token"},
        # a batch of 128 sequences at positions far past the trained length, frequencies stretched
        {**rope, "name": "rotary_batch_far", "batch": 128, "stretch": 8.0, "far": 131072},
        # a long prompt is read in
        {**rope, "name": "rotary_prompt", "tokens": 16384, "far": 16384},
        # the gradient in a training step: neighbouring pairs, two thirds of a 96-wide head, an odd length
        {**rope, "name": "rotary_gradient_part", "batch": 3, "tokens": 2047, "q_heads": 12, "k_heads": 12,
         "dim": 96, "rot": 64, "interleaved": True, "inverse": True, "type": "fp16", "far": 2047},
        # a batch's next tokens go into an int8 cache and are read back
        {**cache, "name": "cache_step_int8", "tokens": 32},
        # a batch of retrieved passages, odd count, fp32 vectors of width 64
        {**cache, "name": "cache_passages_int8", "tokens": 4999, "heads": 5, "dim": 64, "page": 48, "in": "fp32",
         "out": "fp32"},
        # a long prompt into an e4m3 cache and back
        {**cache, "name": "cache_prompt_e4m3", "tokens": 32768, "page": 64, "held": "e4m3"},
        # a prompt into a 16-bit cache and back (copied as it is)
        {**cache, "name": "cache_prompt_bf16", "tokens": 8192, "held": "bf16"},
        # one short sequence: latency
        {**att, "name": "attend_one_short"},
        # 64 conversations of all lengths up to 4,096, some of them empty slots of the batch
        {**att, "name": "attend_batch_bf16", "batch": 64, "len": 4096, "ragged": True},
        # one sequence over a very long int8 cache: split over its length
        {**att, "name": "attend_long_int8", "len": 262144, "q_heads": 28, "k_heads": 4, "page": 64, "held": "int8"},
        # 128 readers of one long document each, e4m3 cache of width 64 with the tokens outermost in a page
        {**att, "name": "attend_documents_e4m3", "batch": 128, "len": 2000, "ragged": True, "q_heads": 20,
         "k_heads": 4, "dim": 64, "page": 32, "type": "fp16", "held": "e4m3", "token_major": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "cache", "attention", "attention"])
    dim = rng.choice([64, 96, 128])
    if op == "rotary":
        q_heads, k_heads = rng.choice([(8, 8), (14, 2), (20, 4), (32, 8), (7, 1)])
        return {"op": op, "batch": _log(rng, 1, 128), "tokens": 1 if rng.random() < 0.4 else _log(rng, 1, 128),
                "q_heads": q_heads, "k_heads": k_heads, "dim": dim, "rot": rng.choice([dim, dim // 2, 20]),
                "interleaved": rng.random() < 0.5, "inverse": rng.random() < 0.5,
                "type": rng.choice(["bf16", "fp16", "fp32"]), "stretch": rng.choice([1.0, 4.0, 8.0]),
                "far": _log(rng, 256, 1 << 20)}
    held = rng.choice(["bf16", "fp16", "int8", "e4m3"])
    page = rng.choice([16, 32, 48, 64, 128])
    if op == "cache":
        # the cost bound is the 32,768-token prompt's: 8 heads of 128, six bytes a value
        return {"op": op, "tokens": _log(rng, 1, 12000), "heads": rng.choice([1, 2, 4, 5, 8]), "dim": dim,
                "page": page, "in": rng.choice(["bf16", "fp16", "fp32"]) if held in TOP else held, "held": held,
                "out": rng.choice(["bf16", "fp16", "fp32"]) if held in TOP else held}
    k_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 3, 4, 5, 7, 8, 16])
    batch = _log(rng, 1, 128)
    return {"op": op, "batch": batch, "len": _log(rng, 1, max(1, min(65536, 1048576 // (batch * k_heads)))),
            "ragged": rng.random() < 0.6, "q_heads": k_heads * group, "k_heads": k_heads, "dim": dim, "page": page,
            "type": held if held not in TOP else rng.choice(["bf16", "fp16"]), "held": held,
            "token_major": rng.random() < 0.5}


def _lens(c):
    """The sequences' lengths: all alike, or from nothing to the longest."""
    n, b = c["len"], c["batch"]
    return [n if not c["ragged"] or i == 0 else (i * 2654435761 >> 7) % (n + 1) for i in range(b)]


def work(c):
    if c["op"] == "rotary":
        n = c["batch"] * c["tokens"] * (c["q_heads"] + c["k_heads"])
        return {"bytes": 2 * n * c["dim"] * BYTES[c["type"]] + 8 * c["batch"] * c["tokens"] + 4 * c["rot"],
                "flops": 3 * n * c["rot"]}
    if c["op"] == "cache":
        n = 2 * c["tokens"] * c["heads"]
        scales = 4 if c["held"] in TOP else 0
        held = c["dim"] * BYTES[c["held"]] + scales
        return {"bytes": n * (c["dim"] * (BYTES[c["in"]] + BYTES[c["out"]]) + 2 * held) + 16 * c["tokens"],
                "flops": 4 * n * c["dim"]}
    tokens = sum(_lens(c))
    vector = c["dim"] * BYTES[c["held"]] + (4 if c["held"] in TOP else 0)
    rows = c["batch"] * c["q_heads"]
    return {"bytes": 2 * tokens * c["k_heads"] * vector + rows * (2 * c["dim"] * BYTES[c["type"]] + 4),
            "flops": 4 * tokens * c["q_heads"] * c["dim"]}


# ---- inputs ------------------------------------------------------------------

def _frequencies(rot, stretch, original=4096.0, base=10000.0):
    """base^(-2i/rot); where the context is stretched, frequencies that turn fewer than 32 times over the original
    length are lowered, the slowest by the whole factor."""
    f = base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if stretch > 1:
        keep = ((original * f / (2 * math.pi) - 1) / 31).clamp(0, 1)
        f = f * keep + f / stretch * (1 - keep)
    return f


def _codes(x, held):
    """The codes and scales of vectors (over the last axis) in an 8-bit type."""
    top = x.float().abs().amax(-1, keepdim=True)
    scale = torch.where(top < SMALLEST, torch.zeros_like(top), top / torch.full_like(top, TOP[held]))
    y = torch.where(scale > 0, x.double() / scale.double(), torch.zeros_like(x, dtype=torch.float64))
    if held == "int8":
        return y.round().to(torch.int8), scale.squeeze(-1)
    part = torch.frexp(y)[0]  # y over it is the power of two above y, without a rounding
    step = torch.where(y == 0, torch.ones_like(y), y / part).clamp(min=2.0 ** -5) / 16  # 3 bits behind the leading one
    return ((y / step).round() * step).float().to(torch.float8_e4m3fn), scale.squeeze(-1)


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if c["op"] == "rotary":
        b, s = c["batch"], c["tokens"]
        t = TYPES[c["type"]]
        # a prompt's positions follow one another; a batch's sequences are anywhere
        first = torch.randint(0, max(1, c["far"] - s + 1), (b, 1), generator=g, device="cuda")
        return {"c": c, "q": normal(b, s, c["q_heads"], c["dim"]).to(t), "k": normal(b, s, c["k_heads"], c["dim"]).to(t),
                "positions": first + torch.arange(s, device="cuda"),
                "freqs": _frequencies(c["rot"], c["stretch"]).cuda(),
                "scale": 0.1 * math.log(c["stretch"]) + 1.0}
    heads, dim, page, held = c.get("heads") or c["k_heads"], c["dim"], c["page"], c["held"]
    lens = _lens(c) if c["op"] == "attention" else [c["tokens"]]
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device="cuda")
    # some channels of real keys are much larger than the others
    loud = 1.0 + 3.0 * (torch.rand(heads, 1, dim, generator=g, device="cuda") > 0.95)

    def filled(by):
        shape = (pages, page, heads, dim) if c.get("token_major") else (pages, heads, page, dim)
        p = torch.empty(shape, dtype=TYPES[held], device="cuda")
        p = p.transpose(1, 2) if c.get("token_major") else p
        scale = torch.zeros(pages, heads, page, device="cuda") if held in TOP else None
        if c["op"] == "cache":
            p.copy_(torch.zeros((), device="cuda"))
            return p, scale
        for i in range(0, pages, 4096):  # a cache that was filled earlier
            x = normal(min(4096, pages - i), heads, page, dim) * by
            if held in TOP:
                codes, scale[i:i + 4096] = _codes(x.bfloat16(), held)
                p[i:i + 4096] = codes
            else:
                p[i:i + 4096] = x.to(TYPES[held])
        return p, scale

    k_pages, k_scale = filled(loud)
    v_pages, v_scale = filled(1.0)
    state = {"c": c, "k_pages": k_pages, "v_pages": v_pages, "k_scale": k_scale, "v_scale": v_scale}
    if c["op"] == "cache":
        t = torch.arange(c["tokens"], device="cuda")
        x = normal(2, c["tokens"], heads, dim).to(TYPES[c["in"]])
        x[0] *= loud[:, 0].to(x.dtype)
        return {**state, "k": x[0], "v": x[1], "slots": order[t // page] * page + t % page}
    width = max(1, max(need))
    tables = torch.full((c["batch"], width), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        tables[i, :n] = torch.arange(at, at + n)
        at += n
    tables = torch.where(tables.cuda() < 0, -1, order.int()[tables.cuda().clamp(min=0)])
    return {**state, "q": (1.5 * normal(c["batch"], c["q_heads"], dim)).to(TYPES[c["type"]]), "tables": tables,
            "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "scale": dim ** -0.5}


# ---- one pass ----------------------------------------------------------------

def _rotate(x, cos, sin, c):
    rot = c["rot"]
    y = x.float()
    if c["interleaved"]:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
    else:
        a, b = y[..., :rot // 2], y[..., rot // 2:rot]
    u, w = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((u, w), -1).flatten(-2) if c["interleaved"] else torch.cat((u, w), -1)
    return torch.cat((turned, y[..., rot:]), -1).to(x.dtype)


def _plain_rotary(s):
    c = s["c"]
    angle = s["positions"].double()[..., None] * s["freqs"]  # far positions lose their angle in 32 bits
    cos, sin = (s["scale"] * angle.cos()).float()[:, :, None], (s["scale"] * angle.sin()).float()[:, :, None]
    if c["inverse"]:
        sin = -sin
    return _rotate(s["q"], cos, sin, c), _rotate(s["k"], cos, sin, c)


def _plain_cache(s):
    c = s["c"]
    page = c["page"]
    at, within = s["slots"] // page, s["slots"] % page
    got = []
    for x, pages, scales in ((s["k"], s["k_pages"], s["k_scale"]), (s["v"], s["v_pages"], s["v_scale"])):
        if scales is None:
            pages[at, :, within] = x.to(pages.dtype)
            got.append(pages[at, :, within].to(TYPES[c["out"]]))
        else:
            codes, scale = _codes(x, c["held"])
            # 8-bit floats are moved as bytes
            pages.view(torch.uint8)[at, :, within] = codes.view(torch.uint8)
            scales[at, :, within] = scale
            read = pages.view(torch.uint8)[at, :, within].view(pages.dtype).float()
            got.append((read * scales[at, :, within][..., None]).to(TYPES[c["out"]]))
    return tuple(got)


def _plain_attention(s):
    c = s["c"]
    b, hk, dim, page = c["batch"], c["k_heads"], c["dim"], c["page"]
    tables = s["tables"].clamp(min=0).long()

    def values(pages, scales):
        x = pages.view(torch.uint8)[tables].view(pages.dtype) if scales is not None else pages[tables]
        x = x.float() if scales is None else x.float() * scales[tables][..., None]
        return x.transpose(1, 2).reshape(b, hk, -1, dim)  # [batch, heads, tokens, dim]

    k = values(s["k_pages"], s["k_scale"])
    q = s["q"].float().view(b, hk, -1, dim)
    score = q @ k.transpose(-1, -2) * s["scale"]
    del k
    seen = torch.arange(tables.shape[1] * page, device="cuda") < s["lens"][:, None]
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = (score - torch.where(top == -math.inf, torch.zeros_like(top), top)).exp()
    total = weight.sum(-1, keepdim=True)
    out = weight @ values(s["v_pages"], s["v_scale"]) / torch.where(total > 0, total, torch.ones_like(total))
    lse = (top + total.log()).masked_fill(total == 0, -math.inf)
    return out.reshape(b, -1, dim).to(s["q"].dtype), lse.reshape(b, -1)


def run(s):
    c = s["c"]
    if not own:
        return {"rotary": _plain_rotary, "cache": _plain_cache, "attention": _plain_attention}[c["op"]](s)
    from chimera_b200 import attention
    if c["op"] == "rotary":
        return attention.rotary(s["q"], s["k"], s["positions"], s["freqs"], interleaved=c["interleaved"],
                                inverse=c["inverse"], scale=s["scale"])
    cache = (s["k_pages"], s["v_pages"])
    if c["op"] == "cache":
        attention.cache_write(s["k"], s["v"], s["slots"], *cache, s["k_scale"], s["v_scale"])
        return attention.cache_read(s["slots"], *cache, s["k_scale"], s["v_scale"], dtype=TYPES[c["out"]])
    return attention.paged_attention(s["q"], *cache, s["tables"], s["lens"], s["k_scale"], s["v_scale"],
                                     scale=s["scale"])


# ---- the definitions in 64 bits ------------------------------------------------

def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "rotary":
        half = c["rot"] // 2
        turn = torch.polar(torch.full_like(s["freqs"], s["scale"]).expand(c["batch"], c["tokens"], half).contiguous(),
                           s["positions"].double()[..., None] * s["freqs"])[:, :, None]
        turn = turn.conj() if c["inverse"] else turn
        got = []
        for x in (s["q"], s["k"]):
            y = x.double().clone()
            where = (slice(0, c["rot"], 2), slice(1, c["rot"], 2)) if c["interleaved"] else \
                    (slice(0, half), slice(half, c["rot"]))
            z = torch.complex(y[..., where[0]].contiguous(), y[..., where[1]].contiguous()) * turn
            y[..., where[0]], y[..., where[1]] = z.real, z.imag
            got.append(y)
        return tuple(got)
    if c["op"] == "cache":
        got = []
        for x in (s["k"], s["v"]):
            y = x.double()
            if c["held"] in TOP:
                top = y.abs().max(-1, keepdim=True).values
                # a scale is a 32-bit number (and a divisor that is a plain number becomes a product)
                unit = torch.true_divide(top.float(), torch.full((1,), TOP[c["held"]], device="cuda")).double()
                z = torch.where(top >= SMALLEST, y / unit, 0.0)
                grid = 1.0
                if c["held"] == "e4m3":
                    bits = z.abs().clamp(min=2.0 ** -6).contiguous().view(torch.int64)
                    grid = (bits >> 52 << 52).view(torch.float64) / 8
                y = torch.round(z / grid) * grid * unit
            got.append(y)
        return tuple(got)
    out, lse = [], []
    group = c["q_heads"] // c["k_heads"]
    for i, n in enumerate(_lens(c)):
        if n == 0:
            out.append(torch.zeros(c["q_heads"], c["dim"], dtype=torch.float64, device="cuda"))
            lse.append(torch.full((c["q_heads"],), -math.inf, dtype=torch.float64, device="cuda"))
            continue
        used = s["tables"][i, :-(-n // c["page"])].tolist()
        at = torch.tensor(used, device="cuda")
        both = []
        for pages, scales in ((s["k_pages"], s["k_scale"]), (s["v_pages"], s["v_scale"])):
            x = (pages if scales is None else pages.view(torch.uint8))[at].view(pages.dtype).float()
            x = x.double() if scales is None else x.double() * scales.double()[at].unsqueeze(-1)
            x = x.permute(1, 0, 2, 3).flatten(1, 2)[:, :n]
            both.append(x.repeat_interleave(group, 0))
        score = torch.einsum("hd,hnd->hn", s["q"][i].double(), both[0]) * s["scale"]
        out.append(torch.einsum("hn,hnd->hd", torch.softmax(score, -1), both[1]))
        lse.append(torch.logsumexp(score, -1))
    return torch.stack(out), torch.stack(lse)
