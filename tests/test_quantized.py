"""A cache of keys and values in 8 bits: the format, writing, reading back, attention over it, and an engine that keeps its
cache so.  The oracles are plain 64-bit statements."""
import math

import pytest
import torch

from jax_llm_examples_amd.engine.batch import GroupContext, decode_bucket
from jax_llm_examples_amd.ops import quantized as Q
from jax_llm_examples_amd.ops.quantized import QuantizedPages
from jax_llm_examples_amd.ops.reference import ReferenceOps
from jax_llm_examples_amd.parts.base import QKPreparation, Rotation

gpu = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    from jax_llm_examples_amd.engine import get_ops
    return get_ops(DEV)


def _gen(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------------------------------------ the format
def held(x):
    """What a row of numbers is held as (64 bits): e4m3 times the smallest power of two that keeps it within 448."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    e = torch.full_like(top, -126.0)
    for k in range(-126, 129):  # (the smallest such power, by trying)
        e = torch.where((e == -126) & (top > 448.0 * 2.0 ** -126) & (top <= 448.0 * 2.0 ** k) & (top > 448.0 * 2.0 ** (k - 1)),
                        torch.full_like(e, float(k)), e)
    y = x * torch.exp2(-e)
    # e4m3: three bits of fraction, magnitudes below 2^-6 in steps of 2^-9, ties to even
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step * torch.exp2(e), e.squeeze(-1)


@pytest.mark.parametrize("dh", [32, 96, 128])
def test_rows_are_held_as_the_format_says(dh):
    x = torch.randn(300, dh, generator=_gen(1)) * torch.exp2(torch.randint(-60, 60, (300, 1), generator=_gen(2)).float())
    x[3], x[4, 1:] = 0.0, 0.0
    x[5, 0] = 1.75 * 2.0 ** 9  # the largest magnitude is exactly at a border, and just beyond it
    x[5, 1:] = 1.0
    x[6] = x[5]
    x[6, 0] = math.nextafter(1.75 * 2.0 ** 9, math.inf) * (1 + 2.0 ** -23)
    x[7] = x[7] / x[7].abs().max() * 3.3e38
    x[8] = x[8] / x[8].abs().max() * 2.0 ** -140
    codes, byte = Q.quantize_rows(x)
    want, e = held(x)
    assert torch.equal(byte.double() - 127, e)
    got = codes.view(torch.float8_e4m3fn).double() * torch.exp2(byte.double() - 127).unsqueeze(-1)
    assert torch.equal(got, want)
    # half a step: 2^-4 of a number's size, or 2^-10 of the codes' unit below 2^-6 of it
    assert ((got - x.double()).abs() <= torch.maximum(2.0 ** -4 * x.double().abs(), torch.exp2(e - 10).unsqueeze(-1))).all()


def test_rows_with_what_is_no_number_read_as_nan():
    x = torch.randn(4, 64, generator=_gen(1))
    x[1, 5], x[2, 0] = float("nan"), -float("inf")
    kv = QuantizedPages.empty(2, 1, 16, 64, "cpu")
    Q.store_rows(kv, x[:, None], x.flip(0)[:, None], torch.tensor([0, 17, 18, 3]))
    k, v = Q.read_rows(kv, torch.tensor([0, 1]))
    k, v = k.reshape(32, 64), v.reshape(32, 64)
    assert torch.isnan(k[[17, 18]]).all() and not torch.isnan(k[[0, 3]]).any()
    assert torch.isnan(v[[17, 18]]).all() and not torch.isnan(v[[0, 3]]).any()


@pytest.mark.parametrize("dh", Q.HEAD_DIMS)
def test_places_are_a_permutation_and_the_layout_that_the_lanes_take(dh):
    k, v = Q.places(dh)
    for at in (k, v):
        assert sorted(at.flatten().tolist()) == list(range(16 * dh))
    for piece in range(0, dh, 64):
        u = 16 if dh - piece >= 64 else 8
        for lane in (0, 5, 17, 40, 63):
            r, g = lane % 16, lane // 16
            assert [int(k[r, piece + u * g + i]) for i in range(u)] == [piece * 16 + lane * u + i for i in range(u)]
            assert [int(v[4 * g + i % 4, piece + 16 * (i // 4) + r]) for i in range(u)] == [piece * 16 + lane * u + i for i in range(u)]


def test_refusals():
    for hq, hk, dh, ps in ((4, 2, 48, 16), (4, 2, 64, 24), (4, 2, 64, 8), (5, 2, 64, 16), (66, 2, 64, 16)):
        with pytest.raises(ValueError, match="8 bits"):
            Q.check_sizes(hq, hk, dh, ps)
    with pytest.raises(ValueError, match="float8_e4m3"):
        Q.check_kv_dtype("int4")
    kv = QuantizedPages.empty(3, 2, 16, 64, "cpu")
    assert tuple(kv.shape) == (3, 2, 2, 16, 64)
    with pytest.raises(ValueError, match="uint8"):
        QuantizedPages(kv.codes.float(), kv.scales)
    with pytest.raises(ValueError, match="uint8"):
        QuantizedPages(kv.codes, kv.scales[:1])
    with pytest.raises(ValueError, match="contiguous"):
        QuantizedPages(kv.codes.transpose(0, 1).contiguous().transpose(0, 1), kv.scales)


# ------------------------------------------------------------------------------------------------ cases
class Case:
    """A step over pages in 8 bits: ``segs``: (tokens in the step, tokens of the request behind it)."""

    def __init__(self, segs, hq, hk, dh, ps, rule=("all",), seed=0, device=DEV, single=False):
        g = _gen(seed)
        self.segs, self.hq, self.hk, self.dh, self.ps, self.rule = segs, hq, hk, dh, ps, rule
        R = len(segs)
        pages = [-(-t // ps) for _, t in segs]
        width = max(pages)
        P = sum(pages) + 2
        ids = torch.randperm(P, generator=g).tolist()
        table = torch.full((R, width), -1, dtype=torch.int32)
        self.k = torch.full((P, hk, ps, dh), float("nan"), dtype=torch.float64)  # what is never written reads as NaN
        self.v = self.k.clone()
        kv = QuantizedPages.empty(P, hk, ps, dh, "cpu", poison=True)
        pos, seg, slots = [], [], []
        for i, (n, t) in enumerate(segs):
            first = self.first(t - n)
            for j in range(first // ps, pages[i]):  # (earlier pages were given back)
                table[i, j] = ids.pop()
            at = torch.arange(first // ps * ps, t)
            slot = table[i, at // ps].long() * ps + at % ps
            rows = [torch.randn(len(at), hk, dh, generator=g) * torch.exp2(torch.randint(-3, 4, (len(at), hk, 1), generator=g).float())
                    for _ in range(2)]
            Q.store_rows(kv, rows[0], rows[1], slot)
            pos += range(t - n, t)
            seg += [i] * n
            slots += slot[-n:].tolist()
        k, v = Q.read_rows(kv, torch.arange(P))
        self.k, self.v = k.double(), v.double()
        n = len(pos)
        self.q = torch.randn(n, hq, dh, generator=g).bfloat16()
        put = lambda x: torch.tensor(x, dtype=torch.int32, device=device)
        self.cpu = (table, pos, seg)
        self.kv = QuantizedPages(kv.codes.to(device), kv.scales.to(device))
        self.table, self.positions, self.segment, self.slots = table.to(device), put(pos), put(seg), put(slots)
        self.scale = dh ** -0.5
        self.meta = GroupContext(block_table=self.table, slot_mapping=self.slots, width=width, retention=rule,
                                 seg_lens=[a for a, _ in segs], seg_starts=[b - a for a, b in segs],
                                 decode_bucket=decode_bucket(max(t for _, t in segs)) if single else None)

    def first(self, pos):
        if self.rule[0] == "chunk":
            return pos // self.rule[1] * self.rule[1]
        return max(0, pos - self.rule[1] + 1) if self.rule[0] == "window" else 0

    def want(self, q=None):
        """Attention in 64 bits, and how far bfloat16 may be off it: the probabilities times the rows' scales and the result
        are rounded (half a step, 2^-8 each of the size); the scores are sums of dh products in float32, whose error moves a
        probability by as much of its size, and so does the base-2 exponential's argument."""
        table, pos, seg = self.cpu
        q = (self.q if q is None else q).double()
        out, tol = torch.empty_like(q), torch.empty_like(q)
        G = self.hq // self.hk
        for n, (p, i) in enumerate(zip(pos, seg)):
            at = torch.arange(self.first(p), p + 1)
            page = table[i, at // self.ps].long()
            k, v = self.k[page, :, at % self.ps], self.v[page, :, at % self.ps]  # [T, hk, dh]
            qi = q[n].view(self.hk, G, self.dh)
            s = torch.einsum("hgd,thd->hgt", qi, k) * self.scale
            size = (torch.einsum("hgd,thd->hgt", qi.abs(), k.abs()) * self.scale).amax(-1, keepdim=True)
            w = torch.softmax(s, -1)
            o = torch.einsum("hgt,thd->hgd", w, v)
            a = torch.einsum("hgt,thd->hgd", w, v.abs())
            out[n] = o.reshape(self.hq, self.dh)
            off = 2 * (self.dh + 16) * 2.0 ** -24 * size + 2.0 ** -18 + len(at) * 2.0 ** -24
            tol[n] = (2.0 ** -8 * (o.abs() + a) * (1 + 2.0 ** -8) + 2 * off * a).reshape(self.hq, self.dh)
        return out.view(len(pos), -1), tol.view(len(pos), -1)

    def run(self, ops, q=None):
        return ops.paged_attention((self.q if q is None else q).to(self.table.device), self.kv, self.table, self.positions,
                                   self.segment, self.rule, self.scale, self.meta)

    def check(self, got, q=None):
        want, tol = self.want(q)
        far = (got.cpu().double() - want).abs()
        assert (far <= tol).all(), f"off by {float((far / tol).max()):.3g} of what rounding allows"


SEGS = {
    "one token": [(1, 1)],
    "second page": [(1, 17), (1, 16), (1, 33)],
    "many": [(1, t) for t in (5, 700, 64, 333, 1025, 31, 32, 257)],
    "few": [(4, 4), (3, 50), (2, 531), (1, 90)],
    "portions": [(70, 70), (1, 300), (33, 215), (5, 12), (129, 400)],
    "long": [(1, 9000)],
}
SEGS["tens"] = [(17, 17), (40, 900), (1, 333), (100, 2100), (16, 16), (2, 700)]
HEADS = [(4, 2, 64), (10, 2, 128), (16, 1, 32), (17, 1, 64), (3, 3, 96), (32, 1, 128), (4, 2, 256), (20, 1, 256)]


@pytest.mark.parametrize("name", ["one token", "second page", "few"])
@pytest.mark.parametrize("rule", [("all",), ("chunk", 24), ("window", 19)], ids=str)
def test_plain_attention_over_codes(name, rule):
    c = Case(SEGS[name], 4, 2, 64, 16, rule, seed=3, device="cpu")
    c.check(c.run(ReferenceOps()))


# ------------------------------------------------------------------------------------------------ on the GPU
@gpu
@pytest.mark.parametrize("dh", Q.HEAD_DIMS)
def test_read_pages_gives_every_code_exactly(ops, dh):
    g = _gen(dh)
    for ps in (16, 48, 128):
        kv = QuantizedPages(torch.randint(0, 256, (5, 3, 2, ps, dh), generator=g, dtype=torch.uint8),
                            torch.randint(1, 248, (5, 3, 2, ps), generator=g, dtype=torch.uint8))
        ids = torch.tensor([4, 0, -1, 4, 2, 5], dtype=torch.int32)
        want = Q.read_pages(kv, ids)
        got = ops.read_pages(QuantizedPages(kv.codes.to(DEV), kv.scales.to(DEV)), ids.to(DEV)).cpu()
        # (numbers below bfloat16's smallest normal may be flushed)
        same = (got == want) | (got.isnan() & want.isnan()) | ((want.float().abs() < 2.0 ** -126) & (got.float().abs() < 2.0 ** -126))
        assert same.all() and got[[2, 5]].isnan().all()


def _prepared(qkv, hq, hk, dh, pos, prep):
    """Queries and keys in 64 bits, values."""
    x = qkv.double().view(len(pos), -1, dh)
    h, v = x[:, : hq + hk].clone(), x[:, hq + hk:]
    unit = lambda t: t / torch.sqrt((t * t).mean(-1, keepdim=True) + prep.norm_eps)
    weights = torch.ones(hq + hk, dh, dtype=torch.float64)
    if prep.norm_weight_q is not None:
        weights[:hq], weights[hq:] = prep.norm_weight_q.double(), prep.norm_weight_k.double()
    if prep.norm_eps is not None and prep.norm_first:
        h = unit(h) * weights
    r = prep.rotation
    if r is not None:
        ang = (torch.tensor(pos).double()[:, None] * r.inv_freq.double()[None])[:, None]
        half = r.rotary_dim // 2
        i = torch.arange(half)
        a, b = (2 * i, 2 * i + 1) if r.pairing == "adjacent" else (i, i + half)
        ha, hb = h[..., a], h[..., b]
        h[..., a], h[..., b] = ha * ang.cos() - hb * ang.sin(), hb * ang.cos() + ha * ang.sin()
    if prep.norm_eps is not None and not prep.norm_first:
        h = unit(h) * weights
    q = h[:, :hq]
    if prep.query_scale is not None:
        q = q * (1 + prep.query_scale[1] * torch.log1p(torch.floor((torch.tensor(pos).double() + 1) / prep.query_scale[0])))[:, None, None]
    return q, h[:, hq:], v


def _prep(kind, dh, device="cpu"):
    g = _gen(dh)
    rot = dh // 2 if kind in ("half part", "first") and dh >= 32 else dh
    pairing = "half" if kind in ("half part", "half") else "adjacent"
    freq = (10000.0 ** (-torch.arange(0, rot, 2).double() / rot)).float().to(device)
    weights = {} if kind not in ("first", "weighted") else dict(norm_weight_q=(torch.rand(dh, generator=g) + 0.5).to(device),
                                                               norm_weight_k=(torch.rand(dh, generator=g) + 0.5).to(device))
    return QKPreparation(rotation=None if kind == "none" else Rotation(freq, pairing, rot),
                         norm_eps=None if kind in ("none", "half") else 1e-5, norm_first=kind == "first",
                         query_scale=(16.0, 0.3) if kind == "plain" else None, **weights)


@gpu
@pytest.mark.parametrize("kind", ["none", "plain", "half", "half part", "first", "weighted"])
@pytest.mark.parametrize("hq,hk,dh", [(3, 1, 32), (4, 2, 64), (3, 3, 96), (10, 2, 128), (2, 1, 256)])
@pytest.mark.parametrize("ps", [16, 48])
def test_prepare_writes_rows_in_8_bits(ops, kind, hq, hk, dh, ps):
    for n in (1, 5, 75):
        g = _gen(n)
        start = 7 if n > 1 else 100
        pos = list(range(start, start + n))
        qkv = (torch.randn(n, (hq + 2 * hk) * dh, generator=g) * 3).bfloat16()
        qkv.view(n, -1, dh)[0, hq + hk] = 0.0  # a value of zeros
        P = 9
        kv = QuantizedPages.empty(P, hk, ps, dh, "cpu", poison=True)
        order = torch.randperm(P, generator=g)
        slots = torch.tensor([int(order[i // ps]) * ps + i % ps for i in range(3, 3 + n)], dtype=torch.int32)
        if n > 4:
            slots[2], slots[4] = -1, P * ps  # (rows without a place)
        dev = QuantizedPages(kv.codes.to(DEV), kv.scales.to(DEV))
        q = ops.qk_prepare_kv_write(qkv.to(DEV), hq, hk, dh, torch.tensor(pos, dtype=torch.int32, device=DEV),
                                    _prep(kind, dh, DEV), dev, slots.to(DEV)).cpu().double()
        prep = _prep(kind, dh)
        wq, wk, wv = _prepared(qkv, hq, hk, dh, pos, prep)
        # float32: two products and a sum a pair, sine and cosine to two units, the norm's sum and root: within 64 roundings
        # of the pair's size (no pair is longer than the head's longest numbers)
        slack = lambda x: 64 * 2.0 ** -24 * (x.abs() + x.abs().amax(-1, keepdim=True))
        assert ((q - wq).abs() <= 2.0 ** -8 * wq.abs() + slack(wq)).all()
        there = [i for i in range(n) if 0 <= slots[i] < P * ps]
        s = slots[there].long()
        k, v = (x.double().transpose(1, 2)[s // ps, s % ps] for x in Q.read_rows(QuantizedPages(dev.codes.cpu(), dev.scales.cpu()), torch.arange(P)))
        for got, want, which in ((k, wk[there], 0), (v, wv[there], 1)):
            full, e = held(want)
            byte = dev.scales.cpu()[s // ps, :, which, s % ps].double() - 127
            near = (torch.log2(want.abs().amax(-1) / 448) - e).abs() < 1e-5  # (at a border either scale is right)
            assert ((byte == e) | near).all()
            if which == 1:
                assert torch.equal(got, full)  # (values are rounded from what was given)
            assert ((got - want).abs() <= torch.maximum(2.0 ** -4 * want.abs(), torch.exp2(byte - 10).unsqueeze(-1)) + slack(want)).all()
        # nothing else changed
        untouched = torch.ones(P * ps, dtype=torch.bool)
        untouched[s] = False
        scales = dev.scales.cpu().permute(0, 3, 1, 2).reshape(P * ps, -1)
        assert (scales[untouched] == Q.NAN_CODE).all()
        rows = Q.read_rows(QuantizedPages(dev.codes.cpu(), torch.full_like(kv.scales, 127)), torch.arange(P))
        for x in rows:
            assert x.transpose(1, 2).reshape(P * ps, -1)[untouched].isnan().all()


@gpu
@pytest.mark.parametrize("kind", ["plain", "half", "first"])
@pytest.mark.parametrize("n", [3, 130])
def test_prepare_at_far_positions(ops, kind, n):
    """Positions of millions, where an angle that is a float32 product is off by a tenth and more: keys are the nearest codes
    of the 64-bit rows but where these lie within 2^-30 of their size of a border."""
    hq, hk, dh, ps = 4, 2, 128, 16
    g = _gen(n)
    pos = (4_000_001 + torch.arange(n) * 100_003).tolist()
    qkv = torch.randn(n, (hq + 2 * hk) * dh, generator=g).bfloat16()
    kv = QuantizedPages.empty(-(-n // ps), hk, ps, dh, DEV, poison=True)
    slots = torch.arange(n, dtype=torch.int32)
    q = ops.qk_prepare_kv_write(qkv.to(DEV), hq, hk, dh, torch.tensor(pos, dtype=torch.int32, device=DEV), _prep(kind, dh, DEV), kv,
                                slots.to(DEV)).cpu().double()
    wq, wk, _ = _prepared(qkv, hq, hk, dh, pos, _prep(kind, dh))
    assert ((q - wq).abs() <= 2.0 ** -8 * wq.abs() + 64 * 2.0 ** -24 * (wq.abs() + wq.abs().amax(-1, keepdim=True))).all()
    k, _ = Q.read_rows(QuantizedPages(kv.codes.cpu(), kv.scales.cpu()), torch.arange(kv.shape[0]))
    k = k.transpose(1, 2).reshape(-1, hk, dh)[:n].double()
    low, high = held(wk * (1 - 2.0 ** -30))[0], held(wk * (1 + 2.0 ** -30))[0]
    assert ((k == low) | (k == high)).all()


@gpu
@pytest.mark.parametrize("hq,hk,dh", HEADS)
@pytest.mark.parametrize("name", list(SEGS))
def test_attention_over_codes(ops, hq, hk, dh, name):
    c = Case(SEGS[name], hq, hk, dh, 16 if name != "many" else 48, seed=5)
    c.check(c.run(ops))


@gpu
@pytest.mark.parametrize("rule", [("chunk", 256), ("chunk", 100), ("window", 300), ("window", 1), ("window", 33)], ids=str)
@pytest.mark.parametrize("name", ["second page", "many", "few", "portions", "long", "tens"])
def test_attention_over_codes_by_rule(ops, rule, name):
    c = Case(SEGS[name], 10, 2, 128, 16, rule, seed=6)
    c.check(c.run(ops))


@gpu
@pytest.mark.parametrize("hq,hk,dh", HEADS + [(10, 2, 128)])
@pytest.mark.parametrize("name", ["portions", "tens", "portion"])
def test_either_way_of_a_portion(ops, monkeypatch, hq, hk, dh, name):
    """Segments of many tokens over the codes, and over pages read back, whatever the rule would choose."""
    c = Case({**SEGS, "portion": [(300, 1100), (1, 70), (600, 600)]}[name], hq, hk, dh, 16, seed=12)
    for tokens, over in (("QUANTIZED_TOKENS", 0), ("QUANTIZED_LONG_US", 1e9)):
        with monkeypatch.context() as m:
            m.setattr(type(ops), tokens, over)
            c.meta.meta.clear()
            got = c.run(ops)
            plan = next(v for k, v in c.meta.meta.items() if isinstance(k, tuple) and k[0] == "quantized_plan")
            assert (plan["long"] is not None) == (tokens == "QUANTIZED_TOKENS")
            c.check(got)


@gpu
@pytest.mark.parametrize("ps", [16, 32, 48, 64, 256])
@pytest.mark.parametrize("single", [False, True])
def test_single_tokens_by_page_size_and_layout(ops, ps, single):
    """A step of single tokens laid out for its own lengths, and for the next multiple of the recorded steps' bound."""
    c = Case([(1, t) for t in (1, 15, 16, 17, 2000, 1024, 1025, 511)], 8, 4, 64, ps, seed=7, single=single)
    c.check(c.run(ops))


@gpu
@pytest.mark.parametrize("hq,hk,dh", [(6, 2, 32), (16, 1, 64), (20, 1, 96), (5, 1, 128), (4, 2, 256)])
def test_every_number_of_ranges_is_joined(ops, hq, hk, dh):
    """One range to as many as a launch takes, counters that are zero again, and keys beyond what the launch was laid out
    for: NaN, and nothing waits."""
    from jax_llm_examples_amd.ops.hip import _p

    c = Case([(1, 4090), (1, 31), (1, 2049)], hq, hk, dh, 16, seed=11)
    q, n, cols = c.q.to(DEV), 3, hq // hk

    def run(span, ranges):
        out = torch.empty(n, hq * dh, dtype=torch.bfloat16, device=DEV)
        ml = torch.empty(n * hk * ranges * cols * 2, device=DEV)
        wo = torch.empty(n * hk * ranges * cols * dh, device=DEV)
        tickets = torch.zeros(n * hk, dtype=torch.int32, device=DEV)
        ops._call("jle_attention_quantized", _p(q), _p(c.kv.codes), _p(c.kv.scales), _p(out), _p(ml), _p(wo), _p(tickets),
                  _p(c.positions), _p(c.segment), _p(c.table), c.table.shape[1], c.kv.shape[0], None, n, cols, ranges, span,
                  0, 0, c.scale, hq, hk, dh, 16)
        assert not tickets.any()
        return out

    for span in (64, 96, 256, 1024, 2048, 4096):
        c.check(run(span, -(-4090 // span)))
    short = run(256, 7).cpu()  # (the second request has one range, the third nine, the first sixteen)
    want, _ = c.want()
    assert short[0].isnan().all() and short[2].isnan().all() and not short[1].isnan().any()


@gpu
def test_scores_far_apart_and_alike(ops):
    """Queries that make one key take all, and of zeros, where all keys weigh the same."""
    c = Case([(1, 600), (40, 300), (2, 40)], 4, 2, 64, 16, seed=8)
    q = c.q.clone()
    q[0] *= 300
    q[1:5] = 0
    q[-1] *= 100
    c.check(c.run(ops, q), q)


@gpu
@pytest.mark.parametrize("rule", [("all",), ("chunk", 24), ("window", 19)], ids=str)
@pytest.mark.parametrize("hq,hk,dh", [(4, 2, 32), (2, 1, 128), (6, 2, 96), (20, 1, 64), (8, 1, 256)])
@pytest.mark.parametrize("long", [False, True])
def test_rows_that_are_no_numbers_reach_only_queries_that_see_them(ops, monkeypatch, hq, hk, dh, rule, long):
    """A key's row that is NaN, another's values: tokens of the same step and tile that do not see them, those before the
    token and those whose window or chunk it is not in, have their results, the others NaN; over the codes and over pages read back."""
    monkeypatch.setattr(type(ops), *(("QUANTIZED_TOKENS", 0) if long else ("QUANTIZED_LONG_US", 1e9)))
    c = Case([(13, 61), (6, 40), (1, 33), (1, 64)], hq, hk, dh, 16, rule, seed=21)
    for request, at, which in ((0, 55, 1), (0, 30, 0), (1, 36, 0), (1, 38, 1), (2, 32, 1), (3, 20, 1), (3, 44, 1)):
        page = int(c.cpu[0][request, at // 16])
        if page < 0:
            continue
        where = Q.places(dh)[which][at % 16].to(DEV)
        c.kv.codes[page, :, which].view(hk, 16 * dh)[:, where] = Q.NAN_CODE
        c.kv.scales[page, :, which, at % 16] = 127
        (c.v if which else c.k)[page, :, at % 16] = float("nan")
    want, tol = c.want()
    got = c.run(ops).cpu().double()
    assert want.isnan().any() and not want.isnan().all()
    assert (got.isnan() == want.isnan()).all()
    fine = ~want.isnan()
    assert ((got - want).abs() <= tol)[fine].all()


@gpu
def test_missing_pages_give_nan_to_their_queries_alone(ops):
    for n in (1, 3, 40):
        c = Case([(n, 200), (n, 200)], 4, 2, 64, 16, seed=9)
        want, _ = c.want()
        c.table[1, 5] = -1
        got = c.run(ops).cpu()
        assert not got[:n].isnan().any() and got[n:].isnan().all()
        c.table[1, 5] = c.kv.shape[0]  # (a page that does not exist)
        c.meta.meta.clear()
        got = c.run(ops).cpu()
        assert not got[:n].isnan().any() and got[n:].isnan().all()


def _from_rows(ops, c, qkv, prep):
    return ops.attention_from_qkv(qkv, c.hq, c.hk, c.dh, c.positions, c.segment, prep, c.kv, True, c.slots, c.table, c.rule, c.scale,
                                  c.meta)


@gpu
def test_two_streams_with_one_plan_at_once(ops):
    """Calls that may run side by side on two streams, over ranges that are joined: each stream has its own counters and results."""
    c = Case([(1, 9000), (1, 4000), (3, 2500)], 16, 2, 128, 16, seed=14)
    alone = c.run(ops)
    c.check(alone)
    plan = next(v for k, v in c.meta.meta.items() if isinstance(k, tuple) and k[0] == "quantized_plan")
    assert any(ranges > 1 for _, _, _, ranges, _, _ in plan["few"])
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(c.run(ops))
    torch.cuda.synchronize()
    assert all(torch.equal(x, alone) for x in got)


@gpu
def test_two_recordings_of_one_plan_replayed_at_once(ops):
    """Two graphs recorded with the same step's plan, and the same calls launched one by one, on three streams at once: each
    has counters and results of its own.  Every replay gives the unrecorded call's bits, with other work in between."""
    cases = [Case([(1, t) for t in (3000, 2500, 17, 4000)], 10, 2, 128, 16, seed=s, single=True) for s in (1, 2, 3)]
    for c in cases[1:]:
        c.meta = cases[0].meta  # (the plan asks for lengths and bounds only, which are alike)
    want = [c.run(ops).clone() for c in cases]
    (plan,) = cases[0].meta.meta.values()
    assert plan["few"][0][3] > 1 and plan["tickets"] > 0
    streams = [torch.cuda.Stream() for _ in cases]
    qs = [c.q.to(DEV) for c in cases]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c, q, s in zip(cases[:2], qs, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append([ops.paged_attention(q, c.kv, c.table, c.positions, c.segment, c.rule, c.scale, c.meta) for _ in range(6)])
        graphs.append(g)
    for turn in range(5):
        for o in outs:
            for x in o:
                x.fill_(7.0)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[2]):
            loose = [ops.paged_attention(qs[2], cases[2].kv, cases[2].table, cases[2].positions, cases[2].segment, cases[2].rule,
                                         cases[2].scale, cases[2].meta) for _ in range(6)]
        torch.cuda.synchronize()
        for got, w in zip([*outs, loose], want):
            assert all(torch.equal(x, w) for x in got), turn
        torch.randn(1000, device=DEV).sum().item()


@gpu
def test_a_recorded_layer_writes_and_reads_what_the_next_replay_finds(ops):
    """From the projected rows, recorded once and replayed with other rows, positions and slots in the same buffers: what an
    unrecorded call of the same step gives, bit for bit, the pages included."""
    c = Case([(1, t) for t in (1000, 40, 1023, 333)], 8, 4, 64, 16, seed=4, single=True)
    prep = _prep("plain", 64, DEV)
    qkv = (torch.randn(4, 16 * 64, generator=_gen(1)) * 2).bfloat16().to(DEV)
    before = (c.kv.codes.clone(), c.kv.scales.clone())
    _from_rows(ops, c, qkv, prep)  # (its plan)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = _from_rows(ops, c, qkv, prep)
    rows = [(torch.randn(4, 16 * 64, generator=_gen(s)) * 2).bfloat16().to(DEV) for s in (5, 6, 7)]
    got = []
    for recorded in (True, False):
        c.kv.codes.copy_(before[0])
        c.kv.scales.copy_(before[1])
        c.positions.copy_(torch.tensor([999, 39, 1022, 332], dtype=torch.int32))
        mine = []
        for step, r in enumerate(rows):
            # (back by a token each step: its slot is the one before)
            page = c.table.gather(1, (c.positions.long() // 16)[:, None]).squeeze(1)
            c.slots.copy_(page * 16 + c.positions % 16)
            qkv.copy_(r)
            if recorded:
                g.replay()
                mine.append(out.clone())
            else:
                mine.append(_from_rows(ops, c, qkv, prep))
            torch.cuda.synchronize()
            c.positions.sub_(1)
        got.append((mine, c.kv.codes.clone(), c.kv.scales.clone()))
    assert all(torch.equal(a, b) for a, b in zip(got[0][0], got[1][0]))
    assert torch.equal(got[0][1], got[1][1]) and torch.equal(got[0][2], got[1][2])


@gpu
def test_pages_beyond_4_gib(ops):
    """Codes whose places pass 32 bits: rows written, read back and attended to at the end of a pool of 4.2 GiB."""
    hq, hk, dh, ps = 8, 8, 128, 16
    P = 140_000  # of 32 KiB
    kv = QuantizedPages(torch.zeros(P, hk, 2, ps, dh, dtype=torch.uint8, device=DEV),
                        torch.full((P, hk, 2, ps), 1, dtype=torch.uint8, device=DEV))
    n, prep = 40, _prep("plain", dh, DEV)
    put = lambda x: torch.tensor(list(x), dtype=torch.int32, device=DEV)
    pages = [P - 1, P - 7, P - 3]
    qkv = torch.randn(n, (hq + 2 * hk) * dh, generator=_gen(1)).bfloat16().to(DEV)
    slots = put([pages[i // ps] * ps + i % ps for i in range(n)])
    q = ops.qk_prepare_kv_write(qkv, hq, hk, dh, put(range(n)), prep, kv, slots)
    small = QuantizedPages.empty(3, hk, ps, dh, DEV)
    q2 = ops.qk_prepare_kv_write(qkv, hq, hk, dh, put(range(n)), prep, small, put(range(n)))
    assert torch.equal(q, q2)
    assert torch.equal(ops.read_pages(kv, put(pages))[:2], ops.read_pages(small, put([0, 1, 2]))[:2])
    out = []
    for pool, table in ((kv, pages), (small, [0, 1, 2])):
        meta = GroupContext(block_table=put([table]), slot_mapping=slots, width=3, retention=("all",), seg_lens=[n], seg_starts=[0])
        out.append(ops.paged_attention(q, pool, put([table]), put(range(n)), put([0] * n), ("all",), 0.1, meta))
    assert torch.equal(*out)


@gpu
def test_refused_on_the_gpu(ops):
    from jax_llm_examples_amd.ops.hip import KernelError

    c = Case([(2, 40)], 4, 2, 64, 16)
    q = c.q.to(DEV)
    args = (c.table, c.positions, c.segment)
    with pytest.raises(KernelError, match="score cap"):
        ops.paged_attention(q, c.kv, *args, ("all",), 0.1, c.meta, cap=3.0)
    with pytest.raises(KernelError, match="sinks"):
        ops.paged_attention(q, c.kv, *args, ("all",), 0.1, c.meta, sink=torch.zeros(4, device=DEV))
    with pytest.raises(KernelError, match="segments have"):
        short = GroupContext(block_table=c.table, slot_mapping=c.slots, width=3, retention=("all",), seg_lens=[3], seg_starts=[38])
        ops.paged_attention(q, c.kv, *args, ("all",), 0.1, short)
    with pytest.raises(KernelError, match="segments have"):
        short = GroupContext(block_table=c.table, slot_mapping=c.slots, width=3, retention=("all",), seg_lens=[1] * 3, decode_bucket=1024)
        ops.paged_attention(q, c.kv, *args, ("all",), 0.1, short)
    with pytest.raises(KernelError, match="rules"):
        ops.paged_attention(q, c.kv, *args, ("window_keep", 8, 2), 0.1, c.meta)
    with pytest.raises(KernelError, match="positive"):
        ops.paged_attention(q, c.kv, *args, ("all",), 0.0, c.meta)
    with pytest.raises(KernelError, match="bfloat16"):
        ops.paged_attention(q.float(), c.kv, *args, ("all",), 0.1, c.meta)
    with pytest.raises(KernelError, match="pages of"):
        ops.paged_attention(q.view(2, 2, 128), c.kv, *args, ("all",), 0.1, c.meta)
    rows = torch.zeros(2, 8 * 64, dtype=torch.bfloat16, device=DEV)
    pos = torch.zeros(2, dtype=torch.int32, device=DEV)
    with pytest.raises(KernelError, match="multiple"):
        ops.qk_prepare_kv_write(rows, 4, 2, 64, pos, QKPreparation(rotation=Rotation(torch.ones(12, device=DEV), "half", 24)), c.kv, pos)
    with pytest.raises(KernelError, match="as they are"):
        ops.qk_prepare_kv_write(rows, 4, 2, 64, pos, QKPreparation(rotation=Rotation(torch.ones(32, device=DEV), magnitude=2.0)), c.kv, pos)
    with pytest.raises(KernelError, match="bfloat16"):
        ops.qk_prepare_kv_write(rows.float(), 4, 2, 64, pos, QKPreparation(), c.kv, pos)
    with pytest.raises(KernelError, match="must be on the GPU that"):
        ops.read_pages(QuantizedPages(c.kv.codes.cpu(), c.kv.scales.cpu()), pos)
    with pytest.raises(KernelError, match="page ids"):
        ops.read_pages(c.kv, pos.long())


# ------------------------------------------------------------------------------------------------ the engine
def _engine(folder, device, kv_dtype="float8_e4m3", **kw):
    from jax_llm_examples_amd import Engine, load_model

    cpu = device == "cpu"
    return Engine(load_model(folder, "bfloat16", device), cache_tokens=1024, decode_batch_size=4,
                  **{"max_num_batched_tokens": 32, "kv_dtype": kv_dtype, "reference_ops": cpu, **kw})


def _prompts(vocab, lengths=(7, 40, 19)):
    return [torch.randint(0, vocab, (n,), generator=_gen(n)).tolist() for n in lengths]


def test_engine_keeps_its_cache_in_8_bits(model_dirs_bf16):
    """Tiny configuration B (heads of 32): pages of codes, their bytes, poisoned pages that nobody reads, and logits whose
    distance from the bfloat16 cache's is what 8 bits cost."""
    e = _engine(model_dirs_bf16["B"], "cpu", poison=True)
    for g in e.cache.groups:
        assert all(isinstance(t, QuantizedPages) and tuple(t.shape[1:]) == (2, 3, 16, 32) for t in g.tensors.values())
        assert g.bytes_per_token() == len(g.cache_ids) * 2 * 3 * 33
        assert sum(t.codes.numel() + t.scales.numel() for t in g.tensors.values()) == g.bytes_per_token() * 16 * g.pool.num_pages
    plain = _engine(model_dirs_bf16["B"], "cpu", kv_dtype=None)
    prompts = _prompts(1000)
    _, a, ids = e.prefill(prompts)
    _, b, ids_b = plain.prefill(prompts)
    for step in range(20):  # (past the chunk of 48 and several pages)
        far = float((a - b).norm() / b.norm())
        assert torch.isfinite(a).all() and far < 0.1, far
        a, b = e.decode_step([step] * 3, ids)[1], plain.decode_step([step] * 3, ids_b)[1]
    e.release(ids)
    e.cache.check()


def test_engine_with_8_bits_gives_the_same_logits_however_prompts_are_cut(model_dirs_bf16):
    got = []
    for budget in (5, 64):
        e = _engine(model_dirs_bf16["B"], "cpu", max_num_batched_tokens=budget, poison=True)
        got.append(e.prefill(_prompts(1000))[1])
    assert torch.allclose(got[0], got[1], rtol=1e-4, atol=1e-4)


def test_requests_that_lose_their_pages_and_start_again_give_the_same_tokens(model_dirs_bf16):
    from jax_llm_examples_amd import Engine, SamplingParams, load_model

    got = []
    for tokens in (1024, 96):  # (96: two of the three requests do not fit at once to their end)
        e = Engine(load_model(model_dirs_bf16["B"], "bfloat16", "cpu"), cache_tokens=tokens, decode_batch_size=4,
                   max_num_batched_tokens=32, kv_dtype="float8_e4m3", reference_ops=True, poison=True)
        got.append(e.generate(_prompts(1000), SamplingParams(max_decode_length=24)))
        e.cache.check()
    assert e.scheduler.stats["preemptions"] > 0 and got[0] == got[1]


def test_a_replay_holds_its_cache_in_8_bits(model_dirs_bf16, tmp_path):
    import json

    import numpy as np

    from jax_llm_examples_amd.engine.replay import make_runner, replay

    out = {}
    for kv in (None, "float8_e4m3"):
        runner = make_runner(model_dirs_bf16["B"], "bfloat16", 256, "cpu", reference_ops=True, poison=True, kv_dtype=kv)
        steps = [{"step": 0, "entries": [{"id": "a", "tokens": list(range(30)), "want": [29]}]},
                 {"step": 1, "entries": [{"id": "a", "tokens": [5], "want": [0]}], "end": ["a"]}]
        replay(runner, [json.dumps(s) for s in steps], str(tmp_path / str(kv)))
        assert isinstance(next(iter(runner.cache.groups[0].tensors.values())), QuantizedPages) == (kv is not None)
        out[kv] = np.fromfile(str(tmp_path / str(kv) / "1.f32"), "<f4")
    far = np.linalg.norm(out[None] - out["float8_e4m3"]) / np.linalg.norm(out[None])
    assert 0 < far < 0.1


def test_pool_sizes_by_memory_hold_about_twice_the_tokens(model_dirs_bf16):
    from jax_llm_examples_amd import load_model
    from jax_llm_examples_amd.cache import plan_groups, pool_sizes

    model = load_model(model_dirs_bf16["B"], "bfloat16", "cpu")
    kw = dict(page_size=16, itemsize=2, max_requests=4, max_step_tokens=64, memory_bytes=1 << 20)
    wide, narrow = pool_sizes(model.cache_needs(), **kw), pool_sizes(model.cache_needs("float8_e4m3"), **kw)
    everything = [i for i, (key, _) in enumerate(plan_groups(model.cache_needs())) if key[2] == ("all",)]
    assert len(everything) == 1 and narrow[everything[0]] > 1.9 * wide[everything[0]]


def test_engines_that_refuse_8_bits(model_dirs, model_dirs_bf16, tmp_path):
    from jax_llm_examples_amd import Engine, load_model

    with pytest.raises(ValueError, match="heads of"):
        _engine(model_dirs_bf16["A"], "cpu")  # (heads of 16)
    with pytest.raises(ValueError, match="multiple of 16 tokens"):
        _engine(model_dirs_bf16["B"], "cpu", page_size=8)
    with pytest.raises(ValueError, match="int8"):
        _engine(model_dirs_bf16["B"], "cpu", kv_dtype="int8")
    with pytest.raises(ValueError, match="beside a run dtype of bfloat16"):
        Engine(load_model(model_dirs["B"], "float32", "cpu"), cache_tokens=64, reference_ops=True, kv_dtype="float8_e4m3")


def test_designs_whose_attention_keeps_its_run_dtype_refuse_8_bits():
    import mazotar_configs
    import rovidra_configs
    from jax_llm_examples_amd.config import get_architecture
    from jax_llm_examples_amd.engine import build_model

    for configs, table, words in ((mazotar_configs, "MAZOTAR", "layer"), (rovidra_configs, "ROVIDRA", "no layer")):
        top = next(iter(getattr(configs, table).values()))
        top = {k: v for k, v in top.items() if k != "seed"}
        arch = get_architecture(top["architecture"])
        with pytest.raises(ValueError, match=words):
            build_model(arch, arch.parse_config(top), "bfloat16", "cpu").cache_needs("float8_e4m3")


@gpu
@pytest.mark.parametrize("name", ["B", "F"])
def test_engine_on_the_gpu_follows_the_plain_one(name, tmp_path):
    """Portions, single tokens, recorded steps: logits of the kernels beside those of the plain operations, both with a cache
    in 8 bits, over pages that are NaN until they are written."""
    from tiny_configs import write_tiny

    folder = write_tiny(name, str(tmp_path / name), torch.bfloat16)
    e, p = _engine(folder, DEV, poison=True), _engine(folder, "cpu", poison=True)
    prompts = _prompts(600, (7, 40, 90))
    _, a, ids = e.prefill(prompts)
    _, b, ids_p = p.prefill(prompts)
    for step in range(12):
        far = float((a.cpu() - b).norm() / b.norm())
        assert far < 0.03, (step, far)  # (bfloat16 activations through a few layers: each rounding 2^-9 on average)
        a, b = e.decode_step([step + 1] * 3, ids)[1], p.decode_step([step + 1] * 3, ids_p)[1]
    assert e.runner.graphs.replays > 0


@gpu
def test_recorded_steps_over_8_bits_equal_unrecorded_ones_bit_for_bit(tmp_path):
    from tiny_configs import write_tiny

    folder = write_tiny("F", str(tmp_path / "F"), torch.bfloat16)
    a, b = _engine(folder, DEV, poison=True), _engine(folder, DEV, decode_graphs=False)
    prompts = _prompts(600, (7, 40, 90, 1))
    _, la, ids = a.prefill(prompts)
    _, lb, ids_b = b.prefill(prompts)
    assert torch.equal(la, lb)
    for step in range(30):
        la, lb = a.decode_step([step] * 4, ids)[1], b.decode_step([step] * 4, ids_b)[1]
        assert torch.equal(la, lb), step
    assert a.runner.graphs.replays >= 28 and b.runner.graphs is None


@gpu
def test_a_layer_from_its_rows_writes_reads_and_attends(ops):
    """The calls of a layer one after the other, as a step makes them: a portion, then single tokens, then a few at once,
    each attending to what the steps before it wrote, against attention in 64 bits over the rows that the pages hold."""
    hq, hk, dh, ps, P = 10, 2, 128, 16, 40
    kv = QuantizedPages.empty(P, hk, ps, dh, DEV, poison=True)
    prep = _prep("plain", dh, DEV)
    table = torch.randperm(P, generator=_gen(1))[:20].to(torch.int32).view(1, -1)
    done = 0
    for n in (130, 1, 1, 4, 33, 1):
        c = Case.__new__(Case)
        c.segs, c.hq, c.hk, c.dh, c.ps, c.rule, c.scale = [(n, done + n)], hq, hk, dh, ps, ("chunk", 150), dh ** -0.5
        pos = list(range(done, done + n))
        put = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
        slots = put([int(table[0, p // ps]) * ps + p % ps for p in pos])
        qkv = (torch.randn(n, (hq + 2 * hk) * dh, generator=_gen(n)) * 2).bfloat16().to(DEV)
        meta = GroupContext(block_table=table.to(DEV), slot_mapping=slots, width=20, retention=c.rule, seg_lens=[n],
                            seg_starts=[done], decode_bucket=decode_bucket(done + n) if n == 1 else None)
        got = ops.attention_from_qkv(qkv, hq, hk, dh, put(pos), put([0] * n), prep, kv, True, slots, table.to(DEV), c.rule,
                                     c.scale, meta)
        done += n
        k, v = Q.read_rows(QuantizedPages(kv.codes.cpu(), kv.scales.cpu()), torch.arange(P))
        c.k, c.v, c.cpu = k.double(), v.double(), (table, pos, [0] * n)
        # (the queries, as a step that writes nothing prepares them)
        q = ops.qk_prepare_kv_write(qkv, hq, hk, dh, put(pos), prep, kv, torch.full_like(slots, -1)).cpu()
        c.check(got, q)


# ------------------------------------------------------------------------------------------------ a run that writes nothing
@pytest.mark.parametrize("device", ["cpu", pytest.param(DEV, marks=gpu)])
def test_queries_of_a_run_that_writes_nothing_are_turned_as_the_keys_are(device):
    """A run that shares another's cache attends to keys at positions in the millions with queries that those angles turned (a
    float32 product is off by a tenth there and more): the queries are those of a run that writes, and nothing is written."""
    if device == "cpu":
        ops = ReferenceOps()
    else:
        from jax_llm_examples_amd.engine import get_ops
        ops = get_ops(device)
    hq, hk, dh, ps, n = 4, 2, 64, 16, 3
    c = Case([(n, 40)], hq, hk, dh, ps, ("chunk", 64), seed=31, device=device)
    base = 64 * 62_501  # (a chunk's beginning: the pages in front of it were given back)
    table = torch.full((1, (base + 48) // ps), -1, dtype=torch.int32)
    table[0, base // ps:] = c.cpu[0][0]
    pos = [base + p for p in c.cpu[1]]
    positions, table = torch.tensor(pos, dtype=torch.int32, device=device), table.to(device)
    meta = GroupContext(block_table=table, slot_mapping=c.slots, width=table.shape[1], retention=c.rule, seg_lens=[n], seg_starts=[pos[0]])
    qkv = torch.randn(n, (hq + 2 * hk) * dh, generator=_gen(2)).bfloat16()
    prep, rows = _prep("plain", dh, device), qkv.to(device)
    before = (c.kv.codes.clone(), c.kv.scales.clone())
    got = ops.attention_from_qkv(rows, hq, hk, dh, positions, c.segment, prep, c.kv, False, c.slots, table, c.rule, c.scale, meta)
    q = ops.qk_prepare_kv_write(rows, hq, hk, dh, positions, prep, c.kv, torch.full_like(positions, -1))
    assert torch.equal(c.kv.codes, before[0]) and torch.equal(c.kv.scales, before[1])
    want = _prepared(qkv, hq, hk, dh, pos, _prep("plain", dh))[0]
    # (rounded to bfloat16, behind 64 roundings in float32: see the test of prepared rows)
    assert ((q.cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() + 64 * 2.0 ** -24 * (want.abs() + want.abs().amax(-1, keepdim=True))).all()
    assert torch.equal(got, ops.paged_attention(q, c.kv, table, positions, c.segment, c.rule, c.scale, meta))


# ------------------------------------------------------------------------------------------------ keys at the codes' borders
@gpu
@pytest.mark.parametrize("n", [1, 130])
@pytest.mark.parametrize("side", [-1, 0, 1])
def test_keys_that_float32_puts_on_a_border_are_rounded_once(ops, n, side):
    """Keys whose 64-bit numbers lie beside the border of two codes by less than float32 tells: the nearest code, not the even
    one.  ``side``: the row's largest magnitude lies as near to 448, below it or beyond it (another scale), or elsewhere (0)."""
    dh, hq, hk = 128, 2, 1
    for seed in range(1000):  # (until the largest magnitude lies on the asked side)
        g = _gen(seed)
        x = torch.randn(3 + hk, dh, generator=g).bfloat16()
        k = x[hq].double()
        k[k == 0] = 1.0
        x[hq] = k.bfloat16()
        border = (1 + (2 * torch.randint(0, 8, (dh,), generator=g) + 1) / 16).double() * torch.exp2(torch.randint(-5, 7, (dh,), generator=g).double())
        border[0] = 448.0 if side else 300.0
        inv = 1 / torch.sqrt((k * k).mean() + 1e-5)
        weight = (border / (k * inv).abs()).float()  # (a float32 step of the weight moves a key by up to 2^-23 of it)
        y = _prepared(x.view(1, -1), hq, hk, dh, [0], QKPreparation(norm_eps=1e-5, norm_weight_q=weight, norm_weight_k=weight))[1]
        off = (y.abs() / border - 1).view(-1)
        if side == 0 or (off[0] * side > 2.0 ** -45 and float(y.view(-1)[0].abs().float()) == 448.0):
            break
    else:
        raise AssertionError("no such row")
    clear = off.abs() > 2.0 ** -45  # (64-bit roundings are 2^-53 of the number, a dozen of them)
    assert int((clear & (y.view(-1).float().abs().double() == border)).sum()) > dh // 4
    want, e = held(y)
    assert float(e) == {-1: 0.0, 0: 0.0, 1: 1.0}[side]
    device = weight.to(DEV)
    kv = QuantizedPages.empty(-(-n // 16), hk, 16, dh, DEV, poison=True)
    rows = x.view(1, -1).expand(n, -1).contiguous().to(DEV)
    at = torch.arange(n, dtype=torch.int32, device=DEV)
    ops.qk_prepare_kv_write(rows, hq, hk, dh, at, QKPreparation(norm_eps=1e-5, norm_weight_q=device, norm_weight_k=device), kv, at)
    got = Q.read_rows(QuantizedPages(kv.codes.cpu(), kv.scales.cpu()), torch.arange(kv.shape[0]))[0]
    got = got.transpose(1, 2).reshape(-1, hk, dh)[:n].double()
    assert ((got == want) | ~clear).all()


# ------------------------------------------------------------------------------------------------ more tiles than a launch takes
@gpu
@pytest.mark.parametrize("kind", ["single", "bucket", "listed", "ranges"])
def test_more_tiles_than_one_launch_takes(ops, kind):
    """Sixteen requests 4,200 times over, a tile each: more than a grid's second dimension counts.  Single tokens, laid out for
    their own lengths or for a bound; beside segments of two tokens, where tiles are listed; in ranges that are joined.  The
    first sixteen against 64 bits, and all others like them bit for bit."""
    from jax_llm_examples_amd.ops.hip import _p

    many, hq, hk, dh = 4200, 2, 1, 32
    segs = [(1, t) for t in (300, 1, 17, 64, 555, 600, 33, 2, 16, 480, 31, 32, 99, 257, 256, 512)]
    if kind == "listed":
        segs[3] = (2, 64)
    c = Case(segs, hq, hk, dh, 16, seed=43, single=kind == "bucket")
    n, m = c.positions.numel(), c.meta
    again = lambda x: x.repeat(many, *[1] * (x.dim() - 1))
    q, positions, table = again(c.q.to(DEV)), again(c.positions), again(c.table)
    segment = (again(c.segment).view(many, n) + 16 * torch.arange(many, dtype=torch.int32, device=DEV)[:, None]).view(-1)
    meta = GroupContext(block_table=table, slot_mapping=again(c.slots), width=m.width, retention=c.rule, seg_lens=m.seg_lens * many,
                        seg_starts=m.seg_starts * many, decode_bucket=m.decode_bucket)
    if kind == "ranges":
        out = torch.empty(many * n, hq * dh, dtype=torch.bfloat16, device=DEV)
        ml, wo = torch.empty(many * 16 * 3 * 2 * 2, device=DEV), torch.empty(many * 16 * 3 * 2 * dh, device=DEV)
        tickets = torch.zeros(many * 16, dtype=torch.int32, device=DEV)
        ops._call("jle_attention_quantized", _p(q), _p(c.kv.codes), _p(c.kv.scales), _p(out), _p(ml), _p(wo), _p(tickets), _p(positions),
                  _p(segment), _p(table), table.shape[1], c.kv.shape[0], None, many * 16, 2, 3, 256, 0, 0, c.scale, hq, hk, dh, 16)
        assert not tickets.any()
    else:
        out = ops.paged_attention(q, c.kv, table, positions, segment, c.rule, c.scale, meta)
        plan = next(v for k, v in meta.meta.items() if isinstance(k, tuple) and k[0] == "quantized_plan")
        assert plan["long"] is None and plan["few"][0][1] == 16 * many > 65535
    c.check(out[:n])
    assert torch.equal(out, out[:n].repeat(many, 1))


# ------------------------------------------------------------------------------------------------ plans
def _planner(compute_units=256):
    """What plans steps, without a GPU."""
    from jax_llm_examples_amd.ops.hip import HipOps

    ops = HipOps.__new__(HipOps)
    ops._compute_units, ops._query = compute_units, lambda name, *a: 8
    return ops


@pytest.mark.parametrize("lens", [[0], [0, 0], [0, 300], [300, 0, 0], [0, 1], [0, 5000], [0, 5000, 1, 0, 40]], ids=str)
@pytest.mark.parametrize("rule", [("all",), ("chunk", 64), ("window", 100)], ids=str)
def test_segments_of_no_tokens_are_no_work(lens, rule):
    there = [i for i, n in enumerate(lens) if n]
    starts = [7 * i + 3 for i in range(len(lens))]
    table = lambda rows: torch.zeros(rows, 400, dtype=torch.int32)
    plan = _planner()._quantized_plan(lens, starts, rule, 2, 2, 128, 16, None, table(len(lens)))
    assert plan["tokens"] == sum(lens)
    alone = _planner()._quantized_plan([lens[i] for i in there], [starts[i] for i in there], rule, 2, 2, 128, 16, None,
                                       table(len(there))) if there else {"few": [], "long": None}
    assert [x[1:5] for x in plan["few"]] == [x[1:5] for x in alone["few"]] and (plan["long"] is None) == (alone["long"] is None)


@gpu
@pytest.mark.parametrize("long", [False, True])
def test_attention_beside_segments_of_no_tokens(ops, monkeypatch, long):
    monkeypatch.setattr(type(ops), *(("QUANTIZED_TOKENS", 0) if long else ("QUANTIZED_LONG_US", 1e9)))
    c = Case([(300, 1100), (1, 70)], 4, 2, 64, 16, seed=51)
    c.table = c.table[[0, 0, 0, 1, 1]].contiguous()
    c.segment = (2 * c.segment + 1).contiguous()
    c.meta = GroupContext(block_table=c.table, slot_mapping=c.slots, width=c.meta.width, retention=c.rule, seg_lens=[0, 300, 0, 1, 0],
                          seg_starts=[5, 800, 0, 69, 3])
    c.check(c.run(ops))


# ------------------------------------------------------------------------------------------------ rows at no position
@pytest.mark.parametrize("starts", [[-1], [-1, 40], [-1, -1, 700]], ids=str)
@pytest.mark.parametrize("rule", [("all",), ("chunk", 64), ("window", 100)], ids=str)
@pytest.mark.timeout(60)
def test_plans_with_rows_at_no_position(starts, rule):
    plan = _planner()._quantized_plan([1] * len(starts), starts, rule, 2, 2, 128, 16, None, torch.zeros(len(starts), 50, dtype=torch.int32))
    (_, num, cols, ranges, keys, _), = plan["few"]
    assert num == len(starts) and cols == 2 and ranges >= 1 and plan["long"] is None


@pytest.mark.parametrize("device", ["cpu", pytest.param(DEV, marks=gpu)])
@pytest.mark.parametrize("rule", [("all",), ("chunk", 24), ("window", 19)], ids=str)
@pytest.mark.parametrize("how", ["single", "lengths", "direct"])
@pytest.mark.parametrize("ps", [16, 48])
def test_rows_at_no_position_have_zeros(device, rule, how, ps):
    """A batch filled up with rows at position -1, of no segment and without a page: zeros, whether the step is laid out for a
    bound, for its lengths or from its arrays, and the other rows as they are without them."""
    if device == "cpu":
        ops = ReferenceOps()
    else:
        from jax_llm_examples_amd.engine import get_ops
        ops = get_ops(device)
    c = Case([(1, 1), (1, 700), (1, 40), (1, 333)], 4, 2, 64, ps, rule, seed=61, device=device)
    at = torch.tensor([0, 2, 3, 6], device=device)  # where the rows are among eight
    q = torch.randn(8, 4, 64, generator=_gen(1)).bfloat16().to(device)
    q[at] = c.q.to(device)
    positions, segment = (torch.full((8,), -1, dtype=torch.int32, device=device) for _ in range(2))
    table = torch.full((8, c.table.shape[1]), -1, dtype=torch.int32, device=device)
    positions[at], segment[at], table[at] = c.positions, at.to(torch.int32), c.table
    meta = None if how == "direct" else GroupContext(
        block_table=table, slot_mapping=positions, width=table.shape[1], retention=rule, seg_lens=[1] * 8,
        seg_starts=None if how == "single" else positions.tolist(), decode_bucket=1024 if how == "single" else None)
    if how == "direct":  # (the arrays alone: rows beside each other of one segment are told apart by its number)
        segment[1], segment[4], segment[5], segment[7] = 1, 4, 5, 7
    got = ops.paged_attention(q, c.kv, table, positions, segment, rule, c.scale, meta)
    c.check(got[at])
    none = torch.ones(8, dtype=torch.bool)
    none[at.cpu()] = False
    assert not got.cpu()[none].any()


@gpu
@pytest.mark.parametrize("rule", [("all",), ("chunk", 24), ("window", 19)], ids=str)
def test_tokens_in_front_of_the_first_position(ops, rule):
    """Segments of a few tokens of which the first lie in front of position 0: these have zeros, the others their results."""
    c = Case([(5, 5), (3, 40)], 4, 2, 64, 16, rule, seed=62)
    c.positions[:5] -= 2
    c.meta.seg_starts = [-2, 37]
    got = c.run(ops)
    assert not got[:2].any()
    c.cpu = (c.cpu[0], [0, 1, 2, 37, 38, 39], [0, 0, 0, 1, 1, 1])
    want, tol = c.want(c.q[2:])
    assert ((got[2:].cpu().double() - want).abs() <= tol).all()


# ------------------------------------------------------------------------------------------------ pages read back at once
LONG = [(300, 2000), (1, 70), (600, 600), (40, 9000), (5000, 5000), (33, 8000), (3, 20_000), (64, 700)]


@pytest.mark.parametrize("limit", [1 << 19, 1 << 21, 1 << 22, 1 << 24])
@pytest.mark.parametrize("rule", [("all",), ("chunk", 1024), ("window", 3000)], ids=str)
@pytest.mark.parametrize("codes", [0, 4096])
def test_plans_read_back_no_more_than_the_bound_at_once(limit, rule, codes):
    """What goes the long way is read back in passes of no more than the bound, several segments at once or some of a segment's
    heads; a segment of which one head's pages are more than that goes through the codes, whatever its length; every token and
    head is in one place."""
    ops = _planner()
    ops.QUANTIZED_READ_BYTES, ops.QUANTIZED_TOKENS = limit, codes
    hk, dh, ps = 3, 64, 16
    lens, starts = [n for n, _ in LONG], [t - n for n, t in LONG]
    table = torch.zeros(len(LONG), -(-20_000 // ps), dtype=torch.int32)
    plan = ops._quantized_plan(lens, starts, rule, hk, 4, dh, ps, None, table)
    done = torch.zeros(sum(lens), hk, dtype=torch.int32)
    for tiles, num, *_ in plan["few"]:
        for first, n in (tiles.tolist() if tiles is not None else [(i, 1) for i in range(num)]):
            done[first: first + n] += 1
    first_row = [sum(lens[:i]) for i in range(len(lens))]
    of = {i: Case.first(type("R", (), {"rule": rule})(), s) // ps for i, s in enumerate(starts)}
    head = {i: ((starts[i] + lens[i] - 1) // ps + 1 - of[i]) * ps * dh * 4 for i in of}
    for tiles, where, mapped, part in plan["long"] or ():
        low, high = (0, hk) if part is None else part[2:]
        assert 0 < where.numel() * (high - low) * ps * dh * 4 <= limit
        assert torch.equal(mapped.view(-1)[where.long()], torch.arange(where.numel(), dtype=torch.int32)) and int((mapped >= 0).sum()) == where.numel()
        for first, n in tiles["tiles"].view(-1, 2).tolist():
            done[first: first + n, low:high] += 1
            i = max(j for j in of if first_row[j] <= first)
            assert (mapped[i, of[i]: (starts[i] + lens[i] - 1) // ps + 1] >= 0).all()
            assert part is None or part[:2] == (first_row[i], first_row[i] + lens[i])
    assert (done == 1).all()
    if codes == 0:  # (only what is too much takes the codes, and single tokens and tiles of a few)
        few = {max(j for j in of if first_row[j] <= first) for first, _ in plan["few"][0][0].tolist()}
        assert few == {i for i in of if lens[i] <= 4 or head[i] > limit}


@gpu
@pytest.mark.parametrize("rule", [("all",), ("chunk", 256), ("window", 300)], ids=str)
@pytest.mark.parametrize("limit", [1 << 18, 1 << 19, 1 << 20])
@pytest.mark.parametrize("hq,hk,dh", [(10, 2, 128), (6, 3, 128), (8, 4, 32)])
def test_pages_read_back_in_passes(ops, monkeypatch, rule, limit, hq, hk, dh):
    """A bound that only some of the segments keep, one by one, and some in runs of heads: results as ever, bit for bit where
    the segments' tiles are the same, and no more memory than the bound at once (beside a run's queries and results)."""
    monkeypatch.setattr(type(ops), "QUANTIZED_TOKENS", 0)
    c = Case([(70, 70), (1, 300), (33, 215), (5, 12), (129, 400), (40, 2300), (17, 1000), (64, 64)], hq, hk, dh, 16, rule, seed=71)
    at_once = c.run(ops)
    c.check(at_once)
    monkeypatch.setattr(type(ops), "QUANTIZED_READ_BYTES", limit)
    c.meta.meta.clear()
    q = c.q.to(DEV)
    c.check(c.run(ops, q))  # (its plan)
    plan = next(v for k, v in c.meta.meta.items() if isinstance(k, tuple) and k[0] == "quantized_plan")
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = c.run(ops, q)
    assert torch.cuda.max_memory_allocated() - before <= limit + 3 * got.numel() * 2 + 8192
    c.check(got)
    many = [n for n, _ in c.segs]
    for _, where, table, part in plan["long"]:
        assert where.numel() * dh * 16 * 4 * (hk if part is None else part[3] - part[2]) <= limit
        for i in range(len(many)):
            if (table[i] >= 0).any():
                rows = slice(sum(many[:i]), sum(many[: i + 1]))
                assert torch.equal(got[rows], at_once[rows])


@gpu
def test_portions_of_a_growing_context_ask_for_few_sizes(ops):
    """Each portion reads back more pages than the one before: the allocator's memory grows by no more than twice the last's."""
    hq, hk, dh, ps, n, width = 8, 8, 128, 16, 600, 3000
    kv = QuantizedPages.empty(width, hk, ps, dh, DEV)
    table = torch.arange(width, dtype=torch.int32, device=DEV).view(1, -1)
    q = torch.randn(n, hq, dh, generator=_gen(1)).bfloat16().to(DEV)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    before = torch.cuda.memory_reserved()
    for start in range(0, width * ps - n, n):
        positions = torch.arange(start, start + n, dtype=torch.int32, device=DEV)
        meta = GroupContext(block_table=table, slot_mapping=positions, width=width, retention=("all",), seg_lens=[n], seg_starts=[start])
        with pytest.MonkeyPatch.context() as m:
            m.setattr(type(ops), "QUANTIZED_TOKENS", 0)
            ops.paged_attention(q, kv, table, positions, torch.zeros_like(positions), ("all",), 0.1, meta)
    last = width * ps * hk * dh * 4
    assert torch.cuda.memory_reserved() - before <= 4 * last + (64 << 20)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


def test_pool_sizes_by_memory_leave_room_for_what_is_read_back(model_dirs_bf16):
    """As many pages as the memory holds beside one run's pages in bfloat16, or beside the bound where that is less."""
    from jax_llm_examples_amd import load_model
    from jax_llm_examples_amd.cache import plan_groups, pool_sizes
    from jax_llm_examples_amd.cache.manager import row_bytes

    model = load_model(model_dirs_bf16["B"], "bfloat16", "cpu")
    for kv_dtype in (None, "float8_e4m3"):
        needs = model.cache_needs(kv_dtype)
        groups = plan_groups(needs)
        kw = dict(page_size=16, itemsize=2, max_requests=4, max_step_tokens=64)
        for memory in (1 << 20, 1 << 22):
            for bound in (0, 1 << 16, 1 << 30):
                def taken(n):
                    pools = sum(n[i] * 16 * len(cids) * row_bytes(kv, paged, 2) for i, ((kv, paged, _), cids) in enumerate(groups))
                    most = max(n[i] * 16 * 2 * kv[0] * kv[1] * 2 for i, ((kv, _, _), _) in enumerate(groups))
                    return pools + (min(bound, most) if kv_dtype else 0)
                n = pool_sizes(needs, memory_bytes=memory, read_back_bytes=bound, **kw)
                assert taken(n) <= memory < taken({i: k + 1 for i, k in n.items()})
                if kv_dtype is None:
                    assert n == pool_sizes(needs, memory_bytes=memory, **kw)


def test_engine_sizes_its_pools_with_room_for_what_is_read_back(model_dirs_bf16, monkeypatch):
    from jax_llm_examples_amd.engine import engine as module

    seen = []
    real = module.pool_sizes
    monkeypatch.setattr(module, "pool_sizes", lambda needs, **kw: seen.append(kw) or real(needs, **kw))
    monkeypatch.setattr(ReferenceOps, "QUANTIZED_READ_BYTES", 12_345, raising=False)
    _engine(model_dirs_bf16["B"], "cpu")
    assert seen[0]["read_back_bytes"] == 12_345
    from jax_llm_examples_amd.ops.hip import HipOps
    assert HipOps.QUANTIZED_READ_BYTES == 1 << 31


# ------------------------------------------------------------------------------------------------ rows of portions
def _check_written(ops, n, hq, hk, dh, ps, kind, seed, pos):
    """Rows in places that begin nowhere in particular, jump, run backwards and leave some out: every value's code and scale, a
    key's code but where its 64-bit number lies within 2^-44 of the row's longest of a border, queries, and nothing else."""
    g = _gen(seed)
    qkv = (torch.randn(n, hq + 2 * hk, dh, generator=g) * torch.exp2(torch.randint(-6, 7, (n, hq + 2 * hk, 1), generator=g).float())).bfloat16()
    qkv[0, hq + hk] = 0.0  # a value of zeros
    qkv[n // 2, hq + 2 * hk - 1, 3] = float("inf")  # one that is held as NaN
    P = (n + 3) // ps + 3
    order = torch.randperm(P, generator=g)
    slots = torch.tensor([int(order[i // ps]) * ps + i % ps for i in range(3, 3 + n)], dtype=torch.int32)
    slots[17:41] = slots[17:41].flip(0)  # (backwards)
    slots[60:70] = slots[60:70][torch.randperm(10, generator=g)]
    slots[2], slots[4], slots[9], slots[46], slots[90], slots[n - 1] = -1, P * ps, -5, -1, 2 ** 31 - 1, -1
    kv = QuantizedPages.empty(P, hk, ps, dh, DEV, poison=True)
    q = ops.qk_prepare_kv_write(qkv.view(n, -1).to(DEV), hq, hk, dh, torch.tensor(pos, dtype=torch.int32, device=DEV), _prep(kind, dh, DEV),
                                kv, slots.to(DEV)).cpu().double()
    wq, wk, wv = _prepared(qkv.view(n, -1), hq, hk, dh, pos, _prep(kind, dh))
    # (as in the test of a few rows: 64 roundings of float32 of the longest number, and bfloat16's)
    assert ((q - wq).abs() <= 2.0 ** -8 * wq.abs() + 64 * 2.0 ** -24 * (wq.abs() + wq.abs().amax(-1, keepdim=True))).all()
    codes, scales = kv.codes.cpu(), kv.scales.cpu()
    there = ((slots >= 0) & (slots < P * ps)).nonzero().view(-1)
    s = slots[there].long()
    assert s.unique().numel() == s.numel()
    k, v = (x.double().transpose(1, 2)[s // ps, s % ps] for x in Q.read_rows(QuantizedPages(codes, scales), torch.arange(P)))
    want, e = held(wv[there])
    bad = ~torch.isfinite(wv[there]).all(-1)
    assert bad.any() and v[bad].isnan().all() and torch.equal(v[~bad], want[~bad])
    assert torch.equal(scales[s // ps, :, 1, s % ps].double()[~bad] - 127, e[~bad])
    slack = 2.0 ** -44 * wk[there].abs().amax(-1, keepdim=True)
    low, high = held(wk[there] - slack)[0], held(wk[there] + slack)[0]
    assert ((k == low) | (k == high)).all()
    untouched = torch.ones(P * ps, dtype=torch.bool)
    untouched[s] = False
    assert (scales.permute(0, 3, 1, 2).reshape(P * ps, -1)[untouched] == Q.NAN_CODE).all()
    for x in Q.read_rows(QuantizedPages(codes, torch.full_like(scales, 127)), torch.arange(P)):
        assert x.transpose(1, 2).reshape(P * ps, -1)[untouched].isnan().all()


@gpu
@pytest.mark.parametrize("kind", ["none", "plain", "half", "half part", "first", "weighted"])
@pytest.mark.parametrize("hq,hk,dh", [(3, 1, 32), (4, 2, 64), (3, 3, 96), (10, 2, 128), (2, 1, 256), (16, 16, 128), (8, 8, 256)])
def test_portions_are_written_row_by_row(ops, kind, hq, hk, dh):
    """From 127 tokens, one a block, on 128, where a block takes eight (the last two: heads that do not fit there)."""
    for n, ps in ((127, 16), (128, 48), (131, 16), (200, 16)):
        _check_written(ops, n, hq, hk, dh, ps, kind, n + dh, list(range(5, 5 + n)))


@gpu
@pytest.mark.parametrize("kind,hq,hk,dh", [("plain", 3, 1, 32), ("half part", 4, 2, 64), ("first", 3, 3, 96), ("none", 4, 2, 128), ("weighted", 2, 1, 256)])
def test_portions_of_thousands_are_written_row_by_row(ops, kind, hq, hk, dh):
    """On both sides of the number of tokens from which a wavefront takes one by itself."""
    for n in (4096, 4097, 5003):
        _check_written(ops, n, hq, hk, dh, 16, kind, n, [(7919 * i) % 1_000_003 for i in range(n)])


# ------------------------------------------------------------------------------------------------ arguments on another device
@pytest.mark.parametrize("which", ["inv_freq", "q norm weight", "k norm weight"])
def test_preparation_refuses_what_lies_on_another_gpu(which):
    """What no launch may read: tensors of a second GPU (by what the checks look at of them)."""
    import types

    from jax_llm_examples_amd.ops.hip import KernelError

    def tensor(dtype, *shape, device=0):
        return types.SimpleNamespace(dtype=dtype, shape=torch.Size(shape), device=torch.device("cuda", device), is_cuda=True,
                                     get_device=lambda: device, is_contiguous=lambda: True, data_ptr=lambda: 4096)

    ops = _planner()
    ops._device_index, ops._tickets, ops._quantized_sizes = 0, tensor(torch.int32, 4), {(4, 2, 64, 16)}
    kv = types.SimpleNamespace(shape=(3, 2, 2, 16, 64), codes=tensor(torch.uint8, 3, 2, 2, 16, 64), scales=tensor(torch.uint8, 3, 2, 2, 16))
    there = lambda what, n: tensor(torch.float32, n, device=int(what == which))
    prep = QKPreparation(rotation=Rotation(there("inv_freq", 32)), norm_eps=1e-5, norm_weight_q=there("q norm weight", 64),
                         norm_weight_k=there("k norm weight", 64))
    rows, places = tensor(torch.bfloat16, 5, 8 * 64), tensor(torch.int32, 5)
    with pytest.raises(KernelError, match=which + " must be on the GPU that"):
        ops._qk_prepare_quantized(rows, 4, 2, 64, places, prep, kv, places)
