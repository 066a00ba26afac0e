"""Keys and values held in 8 bits: the work of an attention layer whose cache is quantised as it is written.

A case is plain values.  ``kind`` says which calls a pass makes: ``write`` (the projected rows of a step: queries and keys
normed and rotated head by head, keys and values into the pages in 8 bits, and the touched pages read back, as a portion of
a prompt does before its attention), ``read`` (the pages of whole contexts read back) or ``attend`` (attention of a step's
queries over the pages: single tokens, a few tokens a request, portions of prompts, or these side by side).  ``hq``, ``hk``,
``dh``: query heads, key/value heads, head size; ``page``: tokens a page; ``requests``, ``new``: requests and tokens of each
in the step; ``context``: tokens of a request behind the step (the mean; ``ragged``: from a half to one and a half of it);
``singles``: further requests with one token each beside them; ``rule`` and ``span``: which keys a query reads (``all``,
``chunk``, ``window``); ``norm`` (``after``: weightless behind the rotation, ``before``: weighted in front of it, ``none``),
``pairs`` (``adjacent``, ``half``), ``rot`` (rotated elements of a head), ``tempered`` (queries scaled by their position).

A cached row of ``dh`` numbers is held as e4m3 numbers times a power of two of its own, the smallest with which the row's
largest magnitude stays within 448 (a byte: the exponent plus 127, from 1 on).  A page is ``[hk, 2, page, dh]`` codes and
``[hk, 2, page]`` scale bytes; the codes of sixteen keys lie together in pieces of 64 elements (a last piece of 32 where 64
does not divide the head), in the order in which a matrix instruction's lanes take them (:func:`places`).
"""
import math

import torch

own = False

DEVICE = "cuda:0"
EPS = 1e-5
FLOOR, TEMPER, THETA = 8192.0, 0.1, 500000.0


def case(name, kind, hq=40, hk=8, dh=128, page=16, requests=1, new=1, context=0, ragged=False, singles=0, rule="all", span=0,
         norm="after", pairs="adjacent", rot=128, tempered=False):
    return {"name": name, "kind": kind, "hq": hq, "hk": hk, "dh": dh, "page": page, "requests": requests, "new": new,
            "context": context, "ragged": ragged, "singles": singles, "rule": rule, "span": span, "norm": norm, "pairs": pairs,
            "rot": rot, "tempered": tempered}


def listed():
    return [
        # one user's next token on Llama 4 Scout's layers: what a launch costs
        case("write b1", "write", context=98),
        # a full server's step of single tokens, with learned norms and half of each head rotated in half-split pairs
        case("write b64 ragged", "write", hq=16, hk=8, requests=64, context=1100, ragged=True, norm="before", pairs="half", rot=64),
        # the benchmark's portion of a prompt, on a layer without rotation whose queries are scaled by their position
        case("write 2048", "write", new=2048, context=8192, rot=0, norm="none", tempered=True),
        # a portion of a long document on dense layers
        case("write 8191", "write", hq=32, new=8191, context=8191),
        # short chats whose caches are handed on
        case("read 8 x 333", "read", hq=16, hk=4, dh=64, requests=8, context=333, ragged=True),
        # one long context
        case("read 32768", "read", context=32768),
        # one user's next token behind a short question
        case("step b1 x 98", "attend", context=98),
        # a small server on Scout's chunked layers
        case("step b8 ragged", "attend", requests=8, context=2100, ragged=True, rule="chunk", span=8192),
        # one long context, bound by how fast its keys and values come
        case("step 1 x 32768", "attend", context=32768),
        # a full server with long contexts
        case("step b64 x 6100", "attend", hq=32, requests=64, context=6100, ragged=True),
        # eight requests check five drafted tokens each against windows, beside eight that go on by one token
        case("few 8 x 5", "attend", hq=16, requests=8, new=5, context=4100, ragged=True, singles=8, rule="window", span=2048),
        # the benchmark's portion of a prompt, the last of a chunk
        case("portion 2048", "attend", new=2048, context=8192, rule="chunk", span=8192),
    ]


def draw(rng):
    """Any of the three kinds, heads and pages of every supported form, lengths spread over their logarithms."""
    spread = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    kind = rng.choice(["write", "read", "attend", "attend", "attend"])
    hq, hk, dh = rng.choice([(40, 8, 128), (32, 8, 128), (16, 8, 128), (16, 4, 64), (32, 32, 64), (12, 4, 96), (8, 1, 256),
                             (16, 1, 128), (24, 2, 32)])
    c = case("", kind, hq, hk, dh, page=rng.choice([16, 16, 32, 48, 64, 128]), ragged=rng.random() < 0.7)
    c["rule"] = rng.choice(["all", "all", "chunk", "window"])
    c["span"] = 0 if c["rule"] == "all" else spread(100, 9000)
    c["norm"] = rng.choice(["after", "before", "none"])
    c["pairs"] = rng.choice(["adjacent", "half"])
    c["rot"] = rng.choice([0, dh // 2, dh, dh])
    c["tempered"] = rng.random() < 0.3
    step = rng.choice(["single", "single", "few", "portion", "mixed"])
    c["requests"] = spread(1, 64)
    if kind == "read":
        c["requests"] = spread(1, 16)
        c["context"] = spread(20, 32768 // c["requests"])
    elif step == "single":
        # (no more of the cache than the largest listed step reads)
        c["context"] = spread(20, min(32768, 64 * 6000 * 1024 // (hk * dh) // c["requests"]))
    elif step == "few":
        c["requests"], c["new"] = spread(1, 16), rng.randint(2, 12)
        c["context"] = spread(40, 32768 // c["requests"])
    else:
        c["requests"] = spread(1, 8)
        c["singles"] = rng.randint(1, 8) if step == "mixed" else 0
        c["new"] = spread(13, 2048 // (c["requests"] + c["singles"]))
        c["context"] = c["new"] * 2 + spread(10, 3000)
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------------ lengths
def segments(c):
    """``(tokens in the step, tokens of the request behind it)`` for every request, in the step's order."""
    out = []
    for i in range(c["requests"] + c["singles"]):
        new = c["new"] if i < c["requests"] else 1
        part = 0.5 + (0.381966 + 0.618034 * i) % 1.0 if c["ragged"] else 1.0
        out.append((new, max(new, int(c["context"] * part))))
    return out


def first_seen(c, pos):
    if c["rule"] == "chunk":
        return pos // c["span"] * c["span"]
    return max(0, pos - c["span"] + 1) if c["rule"] == "window" else 0


def touched(c):
    """Per request: the pages (by their place in its table) that a pass of this case reads back."""
    return [list(range((0 if c["kind"] == "read" else total - new) // c["page"], (total - 1) // c["page"] + 1))
            for new, total in segments(c)]


def work(c):
    hq, hk, dh, page = c["hq"], c["hk"], c["dh"], c["page"]
    segs = segments(c)
    n = sum(new for new, _ in segs)
    row = 2 * hk * (dh + 1)  # a token's codes and scale bytes
    if c["kind"] != "attend":
        back = sum(len(t) for t in touched(c)) * page * (row + 2 * 2 * hk * dh)
        rows = 0 if c["kind"] == "read" else n * (2 * (hq + 2 * hk) * dh + 2 * hq * dh + row)
        return {"bytes": back + rows, "flops": 0}
    keys = sum(total - first_seen(c, total - new) for new, total in segs)
    pairs = sum(p - first_seen(c, p) + 1 for new, total in segs for p in range(total - new, total))
    return {"bytes": keys * row + 2 * n * hq * dh * 2, "flops": 4 * pairs * hq * dh}


# ------------------------------------------------------------------------------------------------ what a program has in hand
class State:
    pass


def prepare(c, seed):
    dev = torch.device(DEVICE)
    g = torch.Generator(dev).manual_seed(seed)
    s = State()
    s.case, hq, hk, dh, page = c, c["hq"], c["hk"], c["dh"], c["page"]
    segs = segments(c)
    n, R = sum(new for new, _ in segs), len(segs)
    width = max(-(-total // page) for _, total in segs)
    pages = [-(-total // page) for _, total in segs]
    P = sum(pages) + 3
    ids = torch.randperm(P, generator=g, device=dev)[: sum(pages)].to(torch.int32).cpu().tolist()
    table, at = [], 0
    for (new, total), m in zip(segs, pages):
        row = ids[at: at + m]
        # (pages that no query of the step reads have been given back)
        gone = 0 if c["kind"] == "read" else first_seen(c, total - new) // page
        table.append([-1] * gone + row[gone:] + [-1] * (width - m))
        at += m
    s.new, s.total = [a for a, _ in segs], [b for _, b in segs]
    pos = [p for new, total in segs for p in range(total - new, total)]
    seg = [i for i, (new, _) in enumerate(segs) for _ in range(new)]
    put = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    s.table, s.positions, s.segment = put(table), put(pos), put(seg)
    s.slots = put([table[i][p // page] * page + p % page for i, p in zip(seg, pos)])
    s.page_ids = put([table[i][j] for i, t in enumerate(touched(c)) for j in t])
    s.scale = dh ** -0.5
    # what earlier steps left: rows of normal numbers, the largest of them between 224 and 448 before the row's scale
    shape = (P, hk, 2, page, dh)
    s.codes = torch.empty(shape, dtype=torch.uint8, device=dev)
    for i in range(0, P, 4096):
        x = torch.randn(s.codes[i: i + 4096].shape, generator=g, device=dev) * 110
        s.codes[i: i + 4096] = x.clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    s.scales = torch.randint(119, 122, shape[:-1], generator=g, device=dev, dtype=torch.uint8)
    s.inv_freq = s.wq = s.wk = None
    if c["kind"] == "write":
        s.qkv = torch.randn(n, (hq + 2 * hk) * dh, generator=g, device=dev).to(torch.bfloat16)
        if c["rot"]:
            s.inv_freq = (THETA ** (-torch.arange(0, c["rot"], 2, device=dev, dtype=torch.float64) / c["rot"])).float()
        if c["norm"] == "before":
            s.wq = torch.rand(dh, generator=g, device=dev) + 0.5
            s.wk = torch.rand(dh, generator=g, device=dev) + 0.5
    elif c["kind"] == "attend":
        s.q = torch.randn(n, hq, dh, generator=g, device=dev).to(torch.bfloat16)
    if own:
        from jax_llm_examples_amd.engine.batch import GroupContext, decode_bucket
        from jax_llm_examples_amd.engine.loading import get_ops
        from jax_llm_examples_amd.ops.quantized import QuantizedPages
        from jax_llm_examples_amd.parts.base import QKPreparation, Rotation

        s.ops = get_ops(DEVICE)
        s.kv = QuantizedPages(s.codes, s.scales)
        s.rule = (c["rule"],) if c["rule"] == "all" else (c["rule"], c["span"])
        s.prep = QKPreparation(
            rotation=None if s.inv_freq is None else Rotation(s.inv_freq, c["pairs"], c["rot"]),
            norm_eps=None if c["norm"] == "none" else EPS, norm_weight_q=s.wq, norm_weight_k=s.wk,
            norm_first=c["norm"] == "before", query_scale=(FLOOR, TEMPER) if c["tempered"] else None)
        s.step = GroupContext(block_table=s.table, slot_mapping=s.slots, width=width, retention=s.rule, seg_lens=s.new,
                              seg_starts=[b - a for a, b in segs],
                              decode_bucket=decode_bucket(max(s.total)) if max(s.new) == 1 else None)
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    c = s.case
    if own:
        if c["kind"] == "write":
            q = s.ops.qk_prepare_kv_write(s.qkv, c["hq"], c["hk"], c["dh"], s.positions, s.prep, s.kv, s.slots)
            return {"q": q, "pages": s.ops.read_pages(s.kv, s.page_ids)}
        if c["kind"] == "read":
            return {"pages": s.ops.read_pages(s.kv, s.page_ids)}
        return {"out": s.ops.paged_attention(s.q, s.kv, s.table, s.positions, s.segment, s.rule, s.scale, s.step)}
    if c["kind"] == "write":
        q, k, v = plain_prepare(s)
        plain_store(s, k, 0)
        plain_store(s, v, 1)
        return {"q": q, "pages": plain_pages(s)}
    if c["kind"] == "read":
        return {"pages": plain_pages(s)}
    return {"out": plain_attention(s)}


def places(dh, device):
    """Where element ``d`` of key ``j`` of sixteen lies among their ``16 * dh`` codes, ``[16, dh]``: keys, values."""
    j = torch.arange(16, device=device)[:, None]
    d = torch.arange(dh, device=device)[None, :]
    u = (dh - d // 64 * 64).clamp(max=64) // 4  # codes that a lane takes
    start = d // 64 * 1024
    return (start + d % 64 // u * 16 * u + j * u + d % u,
            start + j // 4 * 16 * u + d % 16 * u + d % 64 // 16 * 4 + j % 4)


def plain_rows(codes, scales):
    """float32 keys and values ``[..., page, dh]`` of pages ``[..., 2, page, dh]``."""
    *lead, _, page, dh = codes.shape
    x = codes.view(torch.float8_e4m3fn).float().reshape(*lead, 2, page // 16, 16 * dh)
    f = (scales.int() << 23).view(torch.float32).unsqueeze(-1)
    k, v = places(dh, codes.device)
    return (x[..., 0, :, :][..., k].reshape(*lead, page, dh) * f[..., 0, :, :],
            x[..., 1, :, :][..., v].reshape(*lead, page, dh) * f[..., 1, :, :])


def plain_pages(s):
    k, v = plain_rows(s.codes[s.page_ids.long()], s.scales[s.page_ids.long()])
    n, hk, page, dh = k.shape
    return torch.stack([k, v.transpose(-1, -2).reshape(n, hk, page, dh)], dim=1).to(torch.bfloat16)


def plain_prepare(s):
    c = s.case
    n, hq, hk, dh = s.qkv.shape[0], c["hq"], c["hk"], c["dh"]
    x = s.qkv.float().view(n, hq + 2 * hk, dh)
    heads, v = x[:, : hq + hk], x[:, hq + hk:]
    norm = lambda t: t * torch.rsqrt((t * t).mean(-1, keepdim=True) + EPS)
    if c["norm"] == "before":
        w = torch.cat([s.wq.expand(hq, dh), s.wk.expand(hk, dh)])
        heads = norm(heads) * w
    if s.inv_freq is not None:
        ang = s.positions.double()[:, None, None] * s.inv_freq.double()
        cos, sin = ang.cos().float(), ang.sin().float()
        turned, rest = heads[..., : c["rot"]], heads[..., c["rot"]:]
        if c["pairs"] == "adjacent":
            a, b = turned[..., 0::2], turned[..., 1::2]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = turned.chunk(2, -1)
            turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        heads = torch.cat([turned, rest], -1)
    if c["norm"] == "after":
        heads = norm(heads)
    q, k = heads[:, :hq], heads[:, hq:]
    if c["tempered"]:
        q = q * (1.0 + TEMPER * torch.log1p(torch.floor((s.positions.float() + 1.0) / FLOOR)))[:, None, None]
    return q.to(torch.bfloat16), k, v


def plain_store(s, x, which):
    """Rows ``[n, hk, dh]`` in 8 bits into their places (``which``: 0 keys, 1 values)."""
    c = s.case
    page, dh = c["page"], c["dh"]
    top = x.abs().amax(-1)
    # 448 is 1.75 times 2^8: the exponent, one more where the largest magnitude's fraction is beyond 1.75
    e = (((top.view(torch.int32) + 0x1FFFFF) >> 23) - 8).clamp(1, 254)
    codes = (x * ((254 - e) << 23).view(torch.float32).unsqueeze(-1)).to(torch.float8_e4m3fn).view(torch.uint8)
    slot = s.slots.long()
    s.scales[slot // page, :, which, slot % page] = e.to(torch.uint8)
    at = places(dh, x.device)[which][slot % 16] + (slot % page // 16 * 16 * dh)[:, None]
    flat = s.codes.view(*s.codes.shape[:3], page * dh)
    head = torch.arange(x.shape[1], device=x.device)
    flat[(slot // page)[:, None, None], head[None, :, None], which, at[:, None, :]] = codes


def plain_attention(s):
    c = s.case
    hq, hk, dh, page = c["hq"], c["hk"], c["dh"], c["page"]
    n, R, W = s.q.shape[0], s.table.shape[0], s.table.shape[1]
    k, v = plain_rows(s.codes[s.table.clamp(min=0).long()], s.scales[s.table.clamp(min=0).long()])
    k = k.transpose(1, 2).reshape(R, hk, W * page, dh)
    v = v.transpose(1, 2).reshape(R, hk, W * page, dh)
    # a request's queries in rows of their own, filled up to the longest
    T = max(s.new)
    seg = s.segment.long()
    lens = torch.bincount(seg, minlength=R)
    within = torch.arange(n, device=seg.device) - (lens.cumsum(0) - lens)[seg]
    q = s.q.new_zeros(R, T, hq, dh, dtype=torch.float32)
    q[seg, within] = s.q.float()
    pos = s.positions.new_zeros(R, T)
    pos[seg, within] = s.positions
    q = q.view(R, T, hk, hq // hk, dh).permute(0, 2, 3, 1, 4).reshape(R, hk, hq // hk * T, dh)
    score = (q @ k.transpose(-1, -2)).view(R, hk, hq // hk, T, W * page) * s.scale
    key = torch.arange(W * page, device=seg.device)
    seen = key <= pos[..., None]
    if c["rule"] == "chunk":
        seen &= key >= (pos // c["span"] * c["span"])[..., None]
    elif c["rule"] == "window":
        seen &= key > (pos - c["span"])[..., None]
    score = score.masked_fill_(~seen[:, None, None], float("-inf"))
    p = (score - score.amax(-1, keepdim=True)).exp_()
    p = p / p.sum(-1, keepdim=True)
    o = (p.view(R, hk, hq // hk * T, W * page) @ v).view(R, hk, hq // hk, T, dh)
    return o.permute(0, 3, 1, 2, 4)[seg, within].reshape(n, hq * dh).to(torch.bfloat16)


# ------------------------------------------------------------------------------------------------ the same in 64 bits
def exact(c, seed):
    s = prepare(c, seed)
    hq, hk, dh, page = c["hq"], c["hk"], c["dh"], c["page"]
    if c["kind"] == "attend":
        out = torch.empty(s.q.shape[0], hq, dh, dtype=torch.float64, device=DEVICE)
        at = 0
        for i, (new, total) in enumerate(zip(s.new, s.total)):
            first = first_seen(c, total - new) // page
            ids = s.table[i, first: -(-total // page)].long()
            for h in range(hk):
                k, v = (exact_rows(s, ids, h, which)[: total - first * page] for which in (0, 1))
                q = s.q[at: at + new, h * (hq // hk): (h + 1) * (hq // hk)].double()
                for a in range(0, new, 256):
                    w = torch.tensordot(q[a: a + 256], k, dims=([2], [1])) * s.scale
                    pos = torch.arange(total - new + a, min(total, total - new + a + 256), device=DEVICE)
                    key = torch.arange(first * page, total, device=DEVICE)
                    low = torch.tensor([first_seen(c, int(p)) for p in pos.tolist()], device=DEVICE)
                    hidden = (key[None] > pos[:, None]) | (key[None] < low[:, None])
                    w[hidden[:, None].expand_as(w)] = -math.inf
                    out[at + a: min(at + a + 256, at + new), h * (hq // hk): (h + 1) * (hq // hk)] = torch.softmax(w, -1) @ v
            at += new
        return {"out": out.view(-1, hq * dh)}
    res = {}
    if c["kind"] == "write":
        n = s.qkv.shape[0]
        x = s.qkv.double().view(n, hq + 2 * hk, dh)
        q, k, v = x[:, :hq], x[:, hq: hq + hk], x[:, hq + hk:]
        q, k = exact_turned(s, q, s.wq), exact_turned(s, k, s.wk)
        if c["tempered"]:
            q = q * (1 + TEMPER * torch.log1p(torch.floor((s.positions.double() + 1) / FLOOR))).view(-1, 1, 1)
        res["q"] = q
    pages = torch.empty(s.page_ids.numel(), 2, hk, page, dh, dtype=torch.float64, device=DEVICE)
    for h in range(hk):
        for which in (0, 1):
            rows = exact_rows(s, s.page_ids.long(), h, which).view(-1, page, dh)
            if c["kind"] == "write":
                new = exact_held((k, v)[which][:, h])
                where = torch.full((s.codes.shape[0],), -1, device=DEVICE)
                where[s.page_ids.long()] = torch.arange(s.page_ids.numel(), device=DEVICE)
                slot = s.slots.long()
                rows[where[slot // page], slot % page] = new
            pages[:, which, h] = rows if which == 0 else rows.transpose(1, 2).reshape(-1, page, dh)
    res["pages"] = pages
    return res


def exact_turned(s, x, w):
    c, rot = s.case, s.case["rot"]
    unit = lambda t: t / torch.sqrt((t ** 2).sum(-1, keepdim=True) / c["dh"] + EPS)
    x = unit(x) * w.double() if c["norm"] == "before" else x.clone()
    if rot:
        first = torch.arange(rot // 2, device=x.device)
        a, b = (2 * first, 2 * first + 1) if c["pairs"] == "adjacent" else (first, first + rot // 2)
        z = torch.polar(torch.ones(1, dtype=torch.float64, device=x.device),
                        torch.outer(s.positions.double(), s.inv_freq.double()))[:, None]
        z = z * torch.complex(x[..., a], x[..., b])
        x[..., a], x[..., b] = z.real, z.imag
    return unit(x) if c["norm"] == "after" else x


def exact_held(x):
    """What 8 bits a number and a power of two a row hold of rows ``[n, dh]``."""
    m, e = torch.frexp(x.abs().amax(-1, keepdim=True) / 448.0)
    e = torch.where(m == 0.5, e - 1, e).clamp(min=-126).double()
    return (x * torch.exp2(-e)).to(torch.float8_e4m3fn).double() * torch.exp2(e)


def exact_rows(s, ids, h, which):
    """Keys (or values) of head ``h`` in the pages ``ids``, one after the other, ``[tokens, dh]``."""
    page, dh = s.case["page"], s.case["dh"]
    x = s.codes[ids, h, which].view(torch.float8_e4m3fn).double().view(-1, 16 * dh)
    out = torch.empty(x.shape[0], 16, dh, dtype=torch.float64, device=x.device)
    for d0 in range(0, dh, 64):
        w = min(64, dh - d0)
        piece = x[:, 16 * d0: 16 * (d0 + w)]
        if which == 0:  # [a quarter of the elements, key, element]
            out[:, :, d0: d0 + w] = piece.view(-1, 4, 16, w // 4).transpose(1, 2).reshape(-1, 16, w)
        else:  # [key / 4, element % 16, element / 16, key % 4]
            out[:, :, d0: d0 + w] = piece.view(-1, 4, 16, w // 16, 4).permute(0, 1, 4, 3, 2).reshape(-1, 16, w)
    return out.view(-1, dh) * torch.exp2(s.scales[ids, h, which].double() - 127.0).reshape(-1, 1)
