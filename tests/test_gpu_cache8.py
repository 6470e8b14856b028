"""The 8-bit cache: attention, write, page tables, and a run of them together, against plain restatements.

Tolerances.  A score is an fp32 sum of D products on the tensor cores; taking every addition as truncated (2^-23
of the partial sums) its error is at most d = D 2^-23 S + 2^-21 |s| with S = scale sum |q k| >= |s| (the second
part: the product with the scales, the exponent's argument).  A weight is then off by 2 d relative to the
normaliser, by 2^-20 from the exponential and the two 11-bit parts that hold it, and the sums over tokens and
blocks add (64 + blocks) 2^-23 of sum p |v|.  16-bit outputs add half a step (bf16 2^-8, fp16 2^-11)."""
import math

import numpy as np
import pytest
import torch

from kvskip_b200 import kvskip as K
from kvskip_b200.cache import PagedKV8
from kvskip_b200.graph import StepGraph
from tests import cache8_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
TILE = 64


def _cpu(t):
    return t.float().cpu() if t.dtype in (torch.float8_e4m3fn,) else t.cpu()


def _codes(shape, kind, gen):
    """Codes of values with a mean and a spread of their own per channel."""
    x = torch.randn(*shape, generator=gen) * torch.exp(0.5 * torch.randn(shape[-1], generator=gen)) \
        + 0.5 * torch.randn(shape[-1], generator=gen)
    x = x * (60.0 if kind == "e4m3" else 25.0)
    return x.clamp(-440, 440).to(torch.float8_e4m3fn) if kind == "e4m3" else x.round().clamp(-127, 127).to(torch.int8)


def _case(lens, Hkv, G, D, kind, qtype, layout, seed=0, T=None, poison=True):
    """CPU tensors of a case; rows behind a length hold NaN codes (e4m3) or 127s, spare pages and their scales NaN."""
    gen = torch.Generator().manual_seed(seed)
    B, T = len(lens), T or max(max(lens), 1)
    nb = -(-T // TILE)
    q = (1.5 * torch.randn(B, Hkv * G, D, generator=gen)).to(qtype)
    scale_of = lambda *s: torch.exp(0.3 * torch.randn(*s, generator=gen)) / (60.0 if kind == "e4m3" else 25.0)  # noqa: E731
    bad = 0x7F
    c = {"q": q, "lens": torch.tensor(lens, dtype=torch.int32), "scale": 1 / math.sqrt(D), "table": None, "nb": nb}
    if layout == "paged":
        n = sum(-(-x // TILE) for x in lens) + 3
        order = torch.randperm(n, generator=gen).tolist()
        table = torch.full((B, nb), -7, dtype=torch.int32)
        ends = []
        for b, x in enumerate(lens):
            for j in range(-(-x // TILE)):
                table[b, j] = order.pop()
            if x % TILE:
                ends.append((int(table[b, x // TILE]), x % TILE))
        c["table"] = table
        for name in ("k", "v"):
            codes, s = _codes((n, Hkv, TILE, D), kind, gen), scale_of(n, Hkv)
            if poison:
                for pg, r in ends:
                    codes.view(torch.uint8)[pg, :, r:] = bad
                codes.view(torch.uint8)[order] = bad
                s[order] = math.nan
            c[name], c[name + "s"] = codes, s
    else:
        for name in ("k", "v"):
            codes, s = _codes((B, Hkv, T, D), kind, gen), scale_of(B, Hkv, nb)
            if poison:
                for b, x in enumerate(lens):
                    codes.view(torch.uint8)[b, :, x:] = bad
                    s[b, :, -(-x // TILE):] = math.nan
            c[name], c[name + "s"] = codes, s
    return c


def _dev(c):
    return {n: (t.to(DEV) if isinstance(t, torch.Tensor) else t) for n, t in c.items()}


def _run(d, plan=None, stats=False, **kw):
    return K.decode8(d["q"], d["k"], d["v"], d["ks"], d["vs"], d["scale"], lens=d["lens"], page_table=d["table"],
                     plan=plan, stats=stats, out_f32=True, **kw)


def _check(r, ref, D, nb, qtype):
    qk = ref["qk"][..., None]
    live = torch.isfinite(ref["lse"])
    s_max = qk                                                   # |s| <= S
    d = D * 2.0 ** -23 * qk + 2.0 ** -21 * s_max
    rel = 2 * d + 2.0 ** -20 + (64 + nb) * 2.0 ** -23
    tol = rel * ref["mag"]
    o32, out, lse = r["out_f32"].double().cpu(), r["out"].double().cpu(), r["lse"].double().cpu()
    assert ((o32 - ref["out"]).abs() <= tol).all(), float(((o32 - ref["out"]).abs() - tol).max())
    half = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[qtype]
    assert ((out - ref["out"]).abs() <= tol + half * (ref["out"].abs() + tol) + 2.0 ** -25).all()
    assert r["out"].dtype == qtype
    assert torch.equal(torch.isneginf(lse), ~live)
    tl = (rel[..., 0] + 2.0 ** -22 * ref["lse"].abs())[live]
    assert ((lse - ref["lse"])[live].abs() <= tl).all()
    if "blk_max" in r:
        bm, bs = r["blk_max"].double().cpu(), r["blk_sum"].double().cpu()
        seen = torch.isfinite(ref["blk_max"])
        assert torch.equal(torch.isfinite(bm), seen) and (bs[~seen] == 0).all()
        dd = d.expand_as(bm)
        assert ((bm - ref["blk_max"])[seen].abs() <= dd[seen]).all()
        assert ((bs - ref["blk_sum"])[seen].abs() <= (rel.expand_as(bs) * ref["blk_sum"])[seen]).all()


LENS = [0, 1, 63, 64, 65, 128, 1000, 2047]


@pytest.mark.parametrize("layout", ["paged", "contiguous"])
@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("Hkv,G,D,qtype", [(8, 4, 128, torch.bfloat16), (2, 8, 64, torch.float16),
                                           (3, 5, 128, torch.float16), (1, 16, 64, torch.bfloat16),
                                           (2, 9, 128, torch.bfloat16), (4, 1, 64, torch.bfloat16)])
def test_decode8_lengths_and_head_layouts(layout, kind, Hkv, G, D, qtype):
    c = _case(LENS, Hkv, G, D, kind, qtype, layout, seed=Hkv * 100 + G)
    ref = R.decode_f64(c["q"], _cpu(c["k"]), _cpu(c["v"]), c["ks"], c["vs"], c["scale"], LENS, c["table"])
    r = _run(_dev(c), stats=True)
    _check(r, ref, D, c["nb"], qtype)
    a = _run(_dev(c), stats=True)
    assert all(torch.equal(r[n], a[n]) for n in ("out", "out_f32", "lse", "blk_max", "blk_sum"))
    if layout == "paged":     # the same lengths under a far larger bound: another form of the launch
        c["table"] = torch.cat([c["table"], torch.full((len(LENS), 3000), -1, dtype=torch.int32)], 1)
        w = _run(_dev(c), stats=True)
        assert torch.isneginf(w["blk_max"][..., c["nb"]:]).all() and (w["blk_sum"][..., c["nb"]:] == 0).all()
        _check({**w, **{n: w[n][..., :c["nb"]] for n in ("blk_max", "blk_sum")}}, ref, D, c["nb"], qtype)
    assert K.ext().device_status() == 0


@pytest.mark.parametrize("lens", [[1], [64], [65], [0], [0, 0, 5], [500], [1024], [2048], [4097], [8192], [20000],
                                  [300] * 70, [130, 0] * 300])
def test_decode8_work_split(lens):
    """One short request, one long one over every SM, many of a few blocks, batches larger than a CTA has threads."""
    Hkv = 2 if len(lens) > 4 else 8
    c = _case(lens, Hkv, 4, 128, "e4m3", torch.bfloat16, "paged", seed=len(lens))
    ref = R.decode_f64(c["q"], _cpu(c["k"]), _cpu(c["v"]), c["ks"], c["vs"], c["scale"], lens, c["table"])
    _check(_run(_dev(c)), ref, 128, c["nb"], torch.bfloat16)
    # a bound that is smaller than the table, and one-token clamps
    m = max(1, max(lens) - 3)
    short = [min(x, m) for x in lens]
    ref = R.decode_f64(c["q"], _cpu(c["k"]), _cpu(c["v"]), c["ks"], c["vs"], c["scale"], short, c["table"])
    _check(_run(_dev(c), max_len=m), ref, 128, c["nb"], torch.bfloat16)


@pytest.mark.parametrize("kind,layout,G", [("e4m3", "paged", 4), ("int8", "contiguous", 8), ("e4m3", "contiguous", 12)])
def test_decode8_block_lists(kind, layout, G):
    lens, Hkv, D = [1500, 64, 0, 777, 1], 3, 128
    c = _case(lens, Hkv, G, D, kind, torch.bfloat16, layout, seed=5)
    nb = c["nb"]
    gen = torch.Generator().manual_seed(3)
    keep = torch.rand(len(lens), Hkv, nb, generator=gen) < 0.4
    keep[0, 1] = False                                           # an empty list
    keep[0, 2] = True                                            # every block
    keep[3, :, nb - 1] = True                                    # a block behind the length: no tokens
    lists = {(b, h): torch.nonzero(keep[b, h])[:, 0].tolist() for b in range(len(lens)) for h in range(Hkv)}
    ref = R.decode_f64(c["q"], _cpu(c["k"]), _cpu(c["v"]), c["ks"], c["vs"], c["scale"], lens, c["table"], lists)
    d = _dev(c)
    plan = K.make_plan(keep.to(DEV))
    _check(_run(d, plan=plan, stats=True), ref, D, nb, torch.bfloat16)
    # entries behind the count are not used, whatever they hold
    idx = plan.block_idx.clone()
    idx[torch.arange(nb, device=DEV)[None, None] >= plan.block_cnt[..., None]] = 1 << 29
    _check(_run(d, plan=K.Plan(idx, plan.block_cnt, nb, nb), stats=True), ref, D, nb, torch.bfloat16)


@pytest.mark.parametrize("Hkv,T,masked", [(1, 45000 * 64 - 11, False), (2, 23000 * 64, True)])
def test_decode8_very_long_heads(Hkv, T, masked):
    """One or two heads over the whole GPU, dozens of blocks per warp.  The 64-bit sums are formed on the GPU, a stretch of
    the sequence at a time."""
    D, G, B = 64, 4, 1
    gen = torch.Generator(device=DEV).manual_seed(T)
    nb = -(-T // TILE)
    k, v = (torch.randint(-127, 128, (B, Hkv, T, D), generator=gen, device=DEV, dtype=torch.int8) for _ in range(2))
    ks, vs = (torch.exp(0.3 * torch.randn(B, Hkv, nb, generator=gen, device=DEV)) / 70 for _ in range(2))
    q = torch.randn(B, Hkv * G, D, generator=gen, device=DEV).to(torch.float16)
    scale, plan = 1 / math.sqrt(D), None
    keep = torch.ones(Hkv, nb, dtype=torch.bool, device=DEV)
    if masked:
        keep = torch.rand(Hkv, nb, generator=gen, device=DEV) < 0.98
        plan = K.make_plan(keep[None])
    r = K.decode8(q, k, v, ks, vs, scale, plan=plan, out_f32=True)
    out = {n: torch.zeros(B, Hkv * G, D, dtype=torch.float64) for n in ("out", "mag")}
    lse, qk = torch.zeros(B, Hkv * G, dtype=torch.float64), torch.zeros(B, Hkv * G, dtype=torch.float64)
    for h in range(Hkv):
        qh = q[0, h * G:(h + 1) * G].double()
        rows, parts = slice(h * G, (h + 1) * G), []
        for t0 in range(0, T, 1 << 18):
            t1 = min(T, t0 + (1 << 18))
            blk = torch.arange(t0, t1, device=DEV) // TILE
            kk, vv = k[0, h, t0:t1].double() * ks[0, h, blk].double()[:, None], v[0, h, t0:t1].double() * vs[0, h, blk].double()[:, None]
            s = (qh @ kk.T * scale).masked_fill(~keep[h, blk], -math.inf)
            m = s.amax(1, keepdim=True)
            p = torch.exp(s - m)
            parts.append((m, p.sum(1, keepdim=True), p @ vv, p @ vv.abs(), (qh.abs() @ kk.abs().T).amax(1) * scale))
        top = torch.cat([x[0] for x in parts], 1).amax(1, keepdim=True)
        w = [torch.exp(x[0] - top) for x in parts]
        total = sum(x[1] * f for x, f in zip(parts, w))
        out["out"][0, rows] = (sum(x[2] * f for x, f in zip(parts, w)) / total).cpu()
        out["mag"][0, rows] = (sum(x[3] * f for x, f in zip(parts, w)) / total).cpu()
        lse[0, rows] = (top + torch.log(total))[:, 0].cpu()
        qk[0, rows] = torch.stack([x[4] for x in parts]).amax(0).cpu()
    # (the sums run over a warp's chunks, then over the pieces: far fewer than nb additions one after the other)
    _check(r, {**out, "lse": lse, "qk": qk}, D, nb, torch.float16)
    again = K.decode8(q, k, v, ks, vs, scale, plan=plan, out_f32=True)
    assert torch.equal(again["out_f32"], r["out_f32"]) and torch.equal(again["lse"], r["lse"])


def test_decode8_strides_and_optional_lengths():
    B, Hkv, G, D, T = 2, 4, 4, 128, 333
    c = _case([T] * B, Hkv, G, D, "e4m3", torch.bfloat16, "contiguous", seed=9)
    ref = R.decode_f64(c["q"], _cpu(c["k"]), _cpu(c["v"]), c["ks"], c["vs"], c["scale"], [T] * B)
    d = _dev(c)
    # token-major cache, block-major scales, q as [B,Hq,1,D] out of a wider buffer, no lens
    def widen(t):
        w = torch.zeros(B, T + 5, Hkv, D, dtype=torch.uint8, device=DEV).view(t.dtype)
        w.view(torch.uint8)[:, :T] = t.transpose(1, 2).view(torch.uint8)
        return w.transpose(1, 2)[:, :, :T]
    ks = torch.zeros(6, B, Hkv, device=DEV).permute(1, 2, 0)
    vs = torch.zeros_like(ks)
    ks[:, :, :], vs[:, :, :] = d["ks"], d["vs"]
    wide = torch.zeros(B, Hkv * G, 2, 2 * D, dtype=torch.bfloat16, device=DEV)
    wide[:, :, 1, :D] = d["q"]
    q = wide[:, :, 1:, :D]
    assert q.dim() == 4 and not q.is_contiguous()
    r = K.decode8(q, widen(d["k"]), widen(d["v"]), ks, vs, c["scale"], out_f32=True)
    _check(r, ref, D, c["nb"], torch.bfloat16)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_decode8_extreme_values(kind):
    """Block scales far apart, a bf16 q far outside fp16, a query of zeros, one dominant token."""
    lens, Hkv, G, D = [500, 200], 2, 4, 64
    c = _case(lens, Hkv, G, D, kind, torch.bfloat16, "contiguous", seed=2)
    for b, x in enumerate(lens):
        n = -(-x // TILE)
        c["vs"][b, :, :n] *= torch.logspace(-12, 12, n)[None]
    c["q"][0, 0] *= 2.0 ** 60
    c["ks"][0, 0] *= 2.0 ** -60                                     # scores as before
    c["q"][0, 1:4] = c["q"][0, 1:4] * 2.0 ** 57
    c["q"][1, 2] = 0
    # a dominant token: its key along q
    c["k"][1, 1, 100] = (c["q"][1, 5].float().sign() * 100).to(c["k"].dtype)
    ref = R.decode_f64(c["q"], _cpu(c["k"]), _cpu(c["v"]), c["ks"], c["vs"], c["scale"], lens)
    _check(_run(_dev(c), stats=True), ref, D, c["nb"], torch.bfloat16)


@pytest.mark.parametrize("G,T", [(4, 700), (8, 700), (16, 700), (4, 40000)])
def test_decode8_values_near_the_end_of_the_type(G, T):
    """Values of 2^115, as bf16 has them: the sums of hundreds of tokens stay inside fp32, whose end is 2^128.  And what
    `write8` made of such values."""
    lens, Hkv, D = [T, 130], 2, 128
    c = _case(lens, Hkv, G, D, "e4m3", torch.bfloat16, "contiguous", seed=G)
    c["vs"] *= 2.0 ** 112 if T < 1000 else 2.0 ** 106
    ref = R.decode_f64(c["q"], _cpu(c["k"]), _cpu(c["v"]), c["ks"], c["vs"], c["scale"], lens)
    assert float(ref["mag"].max()) * T < 2.0 ** 127
    r = _run(_dev(c), stats=True)
    assert torch.isfinite(r["out"]).all()
    _check(r, ref, D, c["nb"], torch.bfloat16)
    cache = PagedKV8(4, 1, Hkv, D, 256, DEV)
    x = torch.randn(200, Hkv, D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(DEV)
    big = (x.float() * 2.0 ** 116).to(torch.bfloat16)
    cache.write(x, big, cache.extend(torch.tensor([200], dtype=torch.int32, device=DEV), n_tokens=200))
    r = cache.decode(c["q"][:1].to(DEV), c["scale"], out_f32=True)
    ref = R.decode_f64(c["q"][:1], _cpu(cache.k), _cpu(cache.v), cache.k_scale.cpu(), cache.v_scale.cpu(), c["scale"], [200],
                       cache.table.cpu())
    _check(r, ref, D, 4, torch.bfloat16)


def test_decode8_nan_stays_in_its_row():
    lens, Hkv, G, D = [300, 300], 2, 4, 128
    c = _case(lens, Hkv, G, D, "e4m3", torch.bfloat16, "paged", seed=4)
    d = _dev(c)
    clean = _run(d)
    d["k"].view(torch.uint8)[int(c["table"][0, 1]), 0, 7, 3] = 0x7F     # a NaN in a key that is read
    r = _run(d)
    assert torch.isnan(r["out_f32"][0, :G]).all() and torch.isnan(r["lse"][0, :G]).all()
    assert torch.equal(r["out_f32"][0, G:], clean["out_f32"][0, G:]) and torch.equal(r["out_f32"][1], clean["out_f32"][1])


@pytest.mark.parametrize("G,bound", [(4, 6), (8, 6), (4, 4000), (16, 6)])
def test_decode8_lists_without_a_token_and_negative_scale(G, bound):
    """A list of blocks behind the length reads nothing; the sign of the softmax scale is free."""
    lens, Hkv, D = [70, 300], 2, 128
    c = _case(lens, Hkv, G, D, "e4m3", torch.bfloat16, "paged", seed=G + bound, T=bound * TILE)
    c["scale"] = -0.05
    nb = c["nb"]
    keep = torch.zeros(2, Hkv, nb, dtype=torch.bool)
    keep[0, 0, 4:6] = True                                         # behind the length: nothing
    keep[0, 1, 0] = keep[0, 1, 5] = True
    keep[1] = True
    lists = {(b, h): torch.nonzero(keep[b, h])[:, 0].tolist() for b in range(2) for h in range(Hkv)}
    ref = R.decode_f64(c["q"], _cpu(c["k"]), _cpu(c["v"]), c["ks"], c["vs"], c["scale"], lens, c["table"], lists)
    r = _run(_dev(c), plan=K.make_plan(keep.to(DEV)), stats=True)
    _check(r, ref, D, nb, torch.bfloat16)
    assert (r["out_f32"][0, :G] == 0).all() and torch.isneginf(r["lse"][0, :G]).all()


@pytest.mark.parametrize("G,bound", [(4, 4), (4, 4000), (16, 4), (8, 4000)])
def test_decode8_batch_without_a_token(G, bound):
    """Every form of the launch: nothing is read, every output written."""
    c = _dev(_case([0, 0, 0], 2, G, 128, "e4m3", torch.bfloat16, "paged", seed=1, T=bound * TILE))
    junk = torch.full((1 << 22,), math.nan, device=DEV)
    del junk                                                          # (the outputs' memory)
    r = _run(c, stats=True)
    assert (r["out"] == 0).all() and (r["out_f32"] == 0).all() and torch.isneginf(r["lse"]).all()
    assert torch.isneginf(r["blk_max"]).all() and (r["blk_sum"] == 0).all()
    e = K.extend_pages(c["lens"], c["lens"], c["table"], torch.zeros(1, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV),
                       n_tokens=0)
    assert e["granted"].all() and e["slots"].numel() == 0 and e["lens"].tolist() == [0, 0, 0]


def test_c_entry_points_give_the_same_bits():
    from kvskip_b200.cabi import CAbi
    lib = CAbi()
    c = _dev(_case([200, 0, 65], 2, 4, 128, "int8", torch.float16, "paged", seed=3))
    out, lse = lib.decode8(c["q"], c["k"], c["v"], c["ks"], c["vs"], c["scale"], c["lens"], c["table"])
    r = _run(c)
    assert torch.equal(out, r["out"]) and torch.equal(lse, r["lse"])
    x = torch.randn(2, 70, 2, 128, device=DEV).to(torch.float16)
    slots = torch.arange(64, 134, device=DEV)
    a, b = ([t.clone() for t in (c["k"], c["v"], c["ks"], c["vs"])] for _ in range(2))
    lib.write8(x[0], x[1], slots, *a)
    K.write8(x[0], x[1], slots, *b)
    assert all(torch.equal(s.view(torch.uint8), t.view(torch.uint8)) for s, t in zip(a, b))


def test_decode8_pages_outside_the_pool_read_as_zeros():
    lens = [200, 70]
    c = _case(lens, 2, 4, 128, "e4m3", torch.bfloat16, "paged", seed=6)
    c["table"][0, 1] = -1
    c["table"][1, 0] = c["k"].shape[0]
    ref = R.decode_f64(c["q"], _cpu(c["k"]), _cpu(c["v"]), c["ks"], c["vs"], c["scale"], lens, c["table"])
    _check(_run(_dev(c), stats=True), ref, 128, c["nb"], torch.bfloat16)


def test_decode8_offsets_beyond_32_bits():
    """Pages whose byte offset, and a contiguous cache whose head offset, pass 2^32."""
    D, lens = 128, [150]
    c = _case(lens, 1, 4, D, "e4m3", torch.bfloat16, "paged", seed=8, poison=False)
    n = (1 << 32) // (TILE * D) + 64
    far = torch.tensor([n - 1, n - 9, n - 33], dtype=torch.int32)
    pools = {}
    for name in ("k", "v"):
        big = torch.empty(n, 1, TILE, D, dtype=torch.uint8, device=DEV)
        s = torch.zeros(n, 1, device=DEV)
        for j in range(3):
            big[int(far[j])] = c[name][int(c["table"][0, j])].view(torch.uint8).to(DEV)
            s[int(far[j])] = c[name + "s"][int(c["table"][0, j])].to(DEV)
        pools[name], pools[name + "s"] = big.view(torch.float8_e4m3fn), s
    ref = R.decode_f64(c["q"], _cpu(c["k"]), _cpu(c["v"]), c["ks"], c["vs"], c["scale"], lens, c["table"])
    d = {**_dev(c), **pools, "table": far[None].to(DEV).contiguous()}
    _check(_run(d), ref, D, 3, torch.bfloat16)
    # and the write: the same token again, far out
    x = torch.randn(2, 1, D, device=DEV, dtype=torch.bfloat16)
    slots = torch.tensor([int(far[0]) * TILE, int(far[0]) * TILE + 1], device=DEV)
    K.write8(x, -x, slots, d["k"], d["v"], d["ks"], d["vs"])
    got = d["k"][int(far[0]), 0, :2].float() * d["ks"][int(far[0]), 0]
    assert ((got - x[:, 0].float()).abs() <= 2.0 ** -4 * x[:, 0].float().abs() + 2.0 ** -10 * d["ks"][int(far[0]), 0]).all()
    assert torch.equal(d["v"][int(far[0]), 0, :2].float(), -d["k"][int(far[0]), 0, :2].float())


def test_decode8_streams_and_concurrent_graphs():
    """Calls on two streams, and two graphs captured on one stream and replayed side by side, do not share anything."""
    cs = [_dev(_case([20000, 30], 4, 4, 128, "e4m3", torch.bfloat16, "paged", seed=s)) for s in (1, 2)]
    want = [_run(d) for d in cs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        got = []
        for d, s in zip(cs, streams):
            with torch.cuda.stream(s):
                got.append(_run(d))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert torch.equal(g["out_f32"], w["out_f32"]) and torch.equal(g["lse"], w["lse"])
    graphs, outs = [], []
    for d in cs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_run(d))
        graphs.append(g)
    for _ in range(5):
        for o in outs:
            o["out_f32"].zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o["out_f32"], w["out_f32"]) and torch.equal(o["lse"], w["lse"])


# ------------------------------------------------------------------------------------------ write8
def _pool(n, Hkv, D, kind, gen):
    return _codes((n, Hkv, TILE, D), kind, gen), torch.exp2(torch.randint(-8, -2, (n, Hkv), generator=gen).float())


def _write_both(x, slots, codes, scales, kind, k4=None):
    """The call and the restatement on copies; the codes of K and V (= -x: the same scales) have to be equal."""
    want_c, want_s = codes.view(torch.uint8).numpy().copy(), scales.numpy().copy()
    R.write_ref(x.float().numpy(), slots.reshape(-1).tolist(), want_c, want_s, kind)
    k, v, ks, vs = codes.to(DEV), codes.clone().to(DEV), scales.to(DEV), scales.clone().to(DEV)
    xd = x.to(DEV)
    a, b = (xd, xd) if k4 is None else (k4(xd), k4(xd))
    K.write8(a, b, slots.to(DEV), k, v, ks, vs)
    for got_c, got_s in ((k, ks), (v, vs)):
        assert np.array_equal(got_s.cpu().numpy(), want_s, equal_nan=True)
        assert _same_codes(got_c.view(torch.uint8).cpu().numpy(), want_c, kind)
    return k, ks


def _same_codes(got, want, kind):
    """Equal bits; the two e4m3 codes of a NaN (0x7F, 0xFF) count as one, a NaN has no sign."""
    if kind == "e4m3":
        got, want = np.where(got == 0xFF, 0x7F, got), np.where(want == 0xFF, 0x7F, want)
    return bool(np.array_equal(got, want))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("qtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("runs", [[(0, 1)], [(0, 64)], [(3, 61)], [(63, 1)], [(5, 1), (0, 64), (0, 9), (60, 4), (0, 1)],
                                  [(r % 64, 1) for r in range(0, 200, 3)], [(0, 64)] * 20 + [(0, 7)],
                                  [(17, 30), (0, 50)] * 8])
def test_write8_matches_the_restatement(D, kind, qtype, runs):
    Hkv, gen = 3, torch.Generator().manual_seed(len(runs) * D)
    codes, scales = _pool(len(runs) + 2, Hkv, D, kind, gen)
    pages = torch.randperm(len(runs) + 2, generator=gen).tolist()
    slots = torch.tensor([pages[i] * TILE + r + j for i, (r, n) in enumerate(runs) for j in range(n)])
    x = torch.randn(len(slots), Hkv, D, generator=gen) * torch.exp2(torch.randint(-6, 7, (len(slots), 1, 1), generator=gen).float())
    _write_both(x.to(qtype), slots, codes, scales, kind)
    assert K.ext().device_status() == 0


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("qtype", [torch.bfloat16, torch.float16])
def test_write8_special_values(kind, qtype):
    Hkv, D, gen = 2, 64, torch.Generator().manual_seed(1)
    codes, scales = _pool(8, Hkv, D, kind, gen)
    x = torch.randn(40, Hkv, D, generator=gen)
    x[0, 0, :4] = torch.tensor([math.inf, -math.inf, math.nan, 0.0])
    x[1] = 0.0                                        # a block of zeros
    x[2, 0] = math.nan                                # nothing finite
    x[3, 1] = 2.0 ** -24                              # the smallest fp16 number
    x[4] = torch.finfo(qtype).max * (1 if qtype is torch.float16 else 0.9)
    x[5, :, :2] = torch.tensor([448.0, 127.0])        # exactly the largest code
    x[5, :, 2:] = 0.25
    x[6, :, :2] = torch.tensor([450.0, 128.0])        # just above
    x[7:20, 0, 5] = math.inf
    slots = torch.tensor([0, 64, 128, 192, 256, 320, 384 + 5] + list(range(448, 448 + 33)))
    scales[6, 0], scales[6, 1] = math.nan, -3.0       # a scale that is none, in front of row 5
    _write_both(x.to(qtype), slots, codes, scales, kind)


def test_write8_growing_a_block_token_by_token():
    """Every token of a block in a call of its own, larger and larger values: the scale grows and the codes of the earlier
    ones are rounded again; values stay within half a step of each rounding."""
    Hkv, D = 2, 128
    for kind in ("e4m3", "int8"):
        gen = torch.Generator().manual_seed(7)
        codes, scales = _pool(2, Hkv, D, kind, gen)
        want_c, want_s = codes.view(torch.uint8).numpy().copy(), scales.numpy().copy()
        k, ks = codes.to(DEV), scales.to(DEV)
        v, vs = k.clone(), ks.clone()
        x = torch.randn(64, Hkv, D, generator=gen).to(torch.bfloat16) * torch.exp2(torch.arange(64) / 9)[:, None, None]
        x = x.to(torch.bfloat16)
        for r in range(64):
            s = torch.tensor([64 + r], device=DEV)
            K.write8(x[r:r + 1].to(DEV), x[r:r + 1].to(DEV), s, k, v, ks, vs)
            R.write_ref(x[r:r + 1].float().numpy(), [64 + r], want_c, want_s, kind)
        assert np.array_equal(k.view(torch.uint8).cpu().numpy(), want_c) and np.array_equal(ks.cpu().numpy(), want_s)
        got = k[1].float().cpu() * ks[1].cpu()[:, None, None]
        err = (got - x.float().transpose(0, 1)).abs()
        s = ks[1].cpu()[:, None, None]
        if kind == "int8":      # half a step for each rounding, each time of at most half the next scale: < 1 step
            assert (err <= s).all()
        else:                   # one rounding of 2^-4; below 2^-6 of the scale, half a step 2^-10 and as much for the later ones
            assert (err <= 2.0 ** -4 * x.float().transpose(0, 1).abs() + 2.0 ** -9 * s).all()


def test_write8_layouts():
    """[B,Hkv,S,D] views into a contiguous cache whose capacity is no multiple of a block, and padding tokens."""
    B, Hkv, S, D, T = 3, 2, 70, 64, 200
    nb, gen = 4, torch.Generator().manual_seed(3)
    x = torch.randn(B, S, Hkv, D, generator=gen).to(torch.bfloat16)
    start = [0, 10, 129]
    slots = torch.full((B, S), -1)
    for b in range(B):
        n = S if b != 1 else 33                                  # row 1 is padded
        slots[b, :n] = b * nb * TILE + start[b] + torch.arange(n)
    codes, scales = _pool(B * nb, Hkv, D, "e4m3", gen)
    want_c, want_s = codes.view(torch.uint8).numpy().copy(), scales.numpy().copy()
    R.write_ref(x.reshape(-1, Hkv, D).float().numpy(), slots.reshape(-1).tolist(), want_c, want_s, "e4m3")
    cap = torch.zeros(B, Hkv, nb * TILE, D, dtype=torch.uint8, device=DEV)
    cap.view(B, Hkv, nb, TILE, D)[:] = codes.view(torch.uint8).view(B, nb, Hkv, TILE, D).transpose(1, 2).to(DEV)
    before = cap.clone()
    k = cap.view(torch.float8_e4m3fn)[:, :, :T]
    v = k.clone()
    ks = scales.view(B, nb, Hkv).transpose(1, 2).to(DEV)
    vs = ks.clone()
    xd = x.transpose(1, 2).to(DEV)
    wide = torch.zeros(B, Hkv, S, 2 * D, dtype=torch.bfloat16, device=DEV)
    wide[..., :D] = xd
    K.write8(wide[..., :D], xd.contiguous(), slots.to(DEV), k, v, ks, vs)
    want = torch.from_numpy(want_c).view(B, nb, Hkv, TILE, D).transpose(1, 2).reshape(B, Hkv, nb * TILE, D)
    assert torch.equal(cap[:, :, :T].cpu(), want[:, :, :T])
    assert torch.equal(cap[:, :, T:], before[:, :, T:])
    assert torch.equal(v.view(torch.uint8).cpu(), want[:, :, :T])
    assert np.array_equal(ks.cpu().numpy(), torch.from_numpy(want_s).view(B, nb, Hkv).transpose(1, 2).numpy())


def test_write8_skips_and_reports_bad_slots():
    Hkv, D, gen = 2, 128, torch.Generator().manual_seed(3)
    codes, scales = _pool(4, Hkv, D, "int8", gen)
    x = torch.randn(6, Hkv, D, generator=gen).to(torch.bfloat16)
    _write_both(x, torch.tensor([5, 4 * TILE, 70, -1, 1 << 40, 130]), codes, scales, "int8")
    assert K.ext().device_status() == 0x302
    _write_both(x, torch.tensor([5, 5, 6, 64, 130, 129]), codes, scales, "int8")         # a second run of one block
    assert K.ext().device_status() == 0x303
    assert K.ext().device_status() == 0
    # a contiguous cache: rows behind the last one it has room for
    k = torch.zeros(1, Hkv, 100, D, dtype=torch.int8, device=DEV)
    s = torch.ones(1, Hkv, 2, device=DEV)
    K.write8(x[:2].to(DEV), x[:2].to(DEV), torch.tensor([99, 100], device=DEV), k, k.clone(), s, s.clone())
    assert K.ext().device_status() == 0x302
    assert (k[:, :, :99] == 0).all() and (k[:, :, 99] != 0).any()


def test_write8_inputs_without_a_tensor_map():
    """One key for every head (a stride of 0), and a run that goes on in the next row of a padded list."""
    Hkv, D, gen = 4, 128, torch.Generator().manual_seed(8)
    codes, scales = _pool(5, Hkv, D, "e4m3", gen)
    x = torch.randn(80, 1, D, generator=gen).to(torch.bfloat16)
    slots = torch.cat([torch.arange(64, 128), torch.arange(128 + 40, 128 + 56)])
    _write_both(x.expand(80, Hkv, D), slots, codes, scales, "e4m3", k4=lambda t: t[:, :1].contiguous().expand(80, Hkv, D))
    x = torch.randn(80, Hkv, D, generator=gen).to(torch.bfloat16)
    rows = lambda t: t.view(4, 20, Hkv, D).transpose(1, 2)                      # noqa: E731
    want_c, want_s = codes.view(torch.uint8).numpy().copy(), scales.numpy().copy()
    R.write_ref(x.float().numpy(), slots.tolist(), want_c, want_s, "e4m3")
    k, ks = codes.to(DEV), scales.to(DEV)
    v, vs = k.clone(), ks.clone()
    K.write8(rows(x.to(DEV)), rows(x.to(DEV)), slots.view(4, 20).to(DEV), k, v, ks, vs)
    assert _same_codes(k.view(torch.uint8).cpu().numpy(), want_c, "e4m3") and np.array_equal(ks.cpu().numpy(), want_s)
    assert torch.equal(k.view(torch.uint8), v.view(torch.uint8)) and torch.equal(ks, vs)


@pytest.mark.parametrize("n", [300, 2500, 9000])
def test_write8_many_tokens_of_many_requests(n):
    """Single tokens and short runs in numbers that take every chunk size of the slot list, V unlike K."""
    Hkv, D, gen = 8, 64, torch.Generator().manual_seed(n)
    runs, left = [], n
    while left:
        m = min(left, int(torch.randint(1, 4, (1,), generator=gen)) if len(runs) % 7 else 1 + len(runs) % 64)
        runs.append(m)
        left -= m
    codes, scales = _pool(len(runs), Hkv, D, "int8", gen)
    order = torch.randperm(len(runs), generator=gen).tolist()
    start = [int(torch.randint(0, 65 - m, (1,), generator=gen)) for m in runs]
    slots = torch.tensor([order[i] * TILE + start[i] + j for i, m in enumerate(runs) for j in range(m)])
    x, y = (torch.randn(n, Hkv, D, generator=gen).to(torch.bfloat16) for _ in range(2))
    k, ks = codes.to(DEV), scales.to(DEV)
    v, vs = k.clone(), ks.clone()
    K.write8(x.to(DEV), y.to(DEV), slots.to(DEV), k, v, ks, vs)
    for t, c, s in ((x, k, ks), (y, v, vs)):
        want_c, want_s = codes.view(torch.uint8).numpy().copy(), scales.numpy().copy()
        R.write_ref(t.float().numpy(), slots.tolist(), want_c, want_s, "int8")
        assert np.array_equal(s.cpu().numpy(), want_s) and np.array_equal(c.view(torch.uint8).cpu().numpy(), want_c)


@pytest.mark.parametrize("n,D,kind", [(5, 128, "e4m3"), (300, 64, "e4m3"), (300, 128, "int8"), (2000, 128, "e4m3"),
                                      (2000, 64, "int8"), (7500, 64, "e4m3")])
def test_write8_single_tokens_that_grow_their_blocks(n, D, kind):
    """One token each for n blocks, every one larger than what its block holds: all lanes of a row round their channels of
    the earlier rows by the old scale, one of them stores the new one.  Every number of slots per warp, K and V unlike."""
    Hkv, gen = 8, torch.Generator().manual_seed(n + D)
    codes, scales = _pool(n, Hkv, D, kind, gen)
    rows = torch.randint(1, 6, (n,), generator=gen)
    slots = torch.randperm(n, generator=gen) * TILE + rows
    big = torch.exp2(torch.randint(0, 9, (n, Hkv, 1), generator=gen).float()) * {"e4m3": 448.0, "int8": 127.0}[kind] / 4
    x, y = (((torch.rand(n, Hkv, D, generator=gen) + 1) * big).to(torch.bfloat16) for _ in range(2))
    k, ks = codes.to(DEV), scales.to(DEV)
    v, vs = k.clone(), ks.clone()
    K.write8(x.to(DEV), y.to(DEV), slots.to(DEV), k, v, ks, vs)
    for t, c, s in ((x, k, ks), (y, v, vs)):
        want_c, want_s = codes.view(torch.uint8).numpy().copy(), scales.numpy().copy()
        R.write_ref(t.float().numpy(), slots.tolist(), want_c, want_s, kind)
        assert (want_s > scales.numpy()).all()
        assert np.array_equal(s.cpu().numpy(), want_s) and _same_codes(c.view(torch.uint8).cpu().numpy(), want_c, kind)


def test_both_status_words_are_reported():
    """A page outside the pool of the 16-bit cache, and a slot outside the 8-bit one: one call each."""
    k = torch.zeros(2, 1, 64, 128, dtype=torch.bfloat16, device=DEV)
    new = torch.ones(1, 1, 128, dtype=torch.bfloat16, device=DEV)
    x = torch.ones(1, 1, 128, dtype=torch.bfloat16, device=DEV)
    k8, s = torch.zeros(2, 1, 64, 128, dtype=torch.int8, device=DEV), torch.ones(2, 1, device=DEV)
    for first in (True, False):
        for paged in (first, not first):
            if paged:
                K.ext().append(k, k.clone(), new, new, 1, None, torch.full((1, 1), -1, dtype=torch.int32, device=DEV))
            else:
                K.write8(x, x, torch.tensor([128], device=DEV), k8, k8.clone(), s, s.clone())
        with pytest.raises(K.DeviceWaitError, match="page table entry"):
            K.check_status("append")
        with pytest.raises(K.DeviceWaitError, match="slot is outside"):
            K.check_status("write8")
        K.check_status("nothing")
    assert (k == 0).all() and (k8 == 0).all() and (s == 1).all()


def test_write8_refuses_shared_memory():
    x = torch.randn(2, 2, 64, device=DEV).to(torch.bfloat16)
    k = torch.zeros(3, 2, 64, 64, dtype=torch.int8, device=DEV)
    s = torch.ones(3, 2, device=DEV)
    slots = torch.tensor([0, 64], device=DEV)
    with pytest.raises(RuntimeError, match="same memory"):
        K.write8(x, x, slots, k, k, s, s.clone())
    with pytest.raises(RuntimeError, match="same memory"):
        K.write8(x, x, slots, k, k.clone(), s, s)
    with pytest.raises(RuntimeError, match="stride of 0"):
        K.write8(x, x, slots, k, k.clone(), s[:1].clone().expand(3, 2), s)
    both = torch.zeros(3, 2, 2, 64, 64, dtype=torch.int8, device=DEV)                              # K and V side by side
    scales = torch.ones(3, 2, 2, device=DEV)
    K.write8(x, 2 * x, slots, both[:, 0], both[:, 1], scales[:, 0], scales[:, 1])
    K.write8(x, 2 * x, slots, k, (v := torch.zeros_like(k)), s, (t := torch.ones_like(s)))
    assert torch.equal(both[:, 0], k) and torch.equal(both[:, 1], v) and torch.equal(scales[:, 0], s) and torch.equal(scales[:, 1], t)


# ------------------------------------------------------------------------------------------ pages
@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("B,hi,new_hi,pool,mode", [(1, 0, 1, 1.0, "packed"), (1, 130, 500, 1.0, "packed"),
                                                   (7, 300, 1, 1.0, "row"), (513, 700, 1, 1.0, "row"),
                                                   (100, 700, 90, 0.6, "packed"), (1500, 300, 70, 0.7, "packed"),
                                                   (2049, 300, 3, 0.9, "row"), (33, 100, 5000, 1.0, "packed"),
                                                   (40, 100, 4000, 0.5, "row")])
def test_extend_and_release_pages(B, hi, new_hi, pool, mode, inplace):
    gen = torch.Generator().manual_seed(B + new_hi)
    lens = torch.randint(0, hi + 1, (B,), generator=gen).tolist()
    new = torch.randint(0 if B > 1 else 1, new_hi + 1, (B,), generator=gen).tolist()
    if B > 8:
        new[3], new[5] = -4, 0
    cap = -(-(hi + new_hi) // TILE) - (1 if B > 50 else 0)          # some requests run into the table's end
    lens = [min(x, cap * TILE) for x in lens]
    have = sum(-(-x // TILE) for x in lens)
    extra = sum(-(-(x + max(0, n)) // TILE) for x, n in zip(lens, new)) - have
    pages = have + max(1, int(extra * pool))
    order = torch.randperm(pages, generator=gen).tolist()
    table = [[-1] * cap for _ in range(B)]
    for b in range(B):
        for j in range(-(-lens[b] // TILE)):
            table[b][j] = order.pop()
    n_free, free = len(order), order + [-9] * (pages - len(order))
    kw = {"per_row": max(max(new) - (1 if B > 1000 else 0), 1)} if mode == "row" else {"n_tokens": sum(max(0, n) for n in new) + (5 if B != 100 else -20)}
    want = R.extend_ref(lens, new, table, free, n_free, **kw)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    ld, td, fd, nd = i32(lens), i32(table), i32(free), i32([n_free])
    out = {"lens_out": ld, "n_free_out": nd} if inplace else {}
    r = K.extend_pages(ld, i32(new), td, fd, nd, **kw, **out)
    assert r["slots"].flatten().tolist() == want[0] and r["positions"].flatten().tolist() == want[1]
    assert r["granted"].tolist() == want[2] and r["lens"].tolist() == want[3] and r["n_free"].tolist() == [want[5]]
    assert td.tolist() == want[4] and fd.tolist() == free
    assert (ld.tolist() == lens or inplace) and (nd.tolist() == [n_free] or inplace)
    done = torch.rand(B, generator=gen) < 0.5
    back = R.release_ref(done.tolist(), want[3], want[4], free, want[5])
    ld, nd = r["lens"], r["n_free"]
    out = {"lens_out": ld, "n_free_out": nd} if inplace else {}
    r = K.release_pages(done.to(DEV), ld, td, fd, nd, **out)
    assert r["lens"].tolist() == back[0] and fd.tolist() == back[1] and r["n_free"].tolist() == [back[2]]
    assert td.tolist() == want[4]


@pytest.mark.parametrize("B", [5, 1030])
def test_extend_pages_grants_a_request_without_tokens_behind_a_full_list(B):
    """The slot list has room for the first request only; what asks for no token needs no place in it and keeps running,
    unless its length is beyond the table."""
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    lens, new = [10, 20, 30, 0, 200] + [70] * (B - 5), [4, 9, 0, -3, 0] + [0, 1] * ((B - 5) // 2) + [0] * ((B - 5) % 2)
    table = torch.full((B, 2), -1, dtype=torch.int32, device=DEV)
    table[:, 0] = torch.arange(B)
    free = torch.arange(B, B + 8, dtype=torch.int32, device=DEV)
    r = K.extend_pages(i32(lens), i32(new), table, free, i32([8]), n_tokens=6)
    assert r["granted"].tolist() == [True, False, True, True, False] + [n == 0 for n in new[5:]]
    assert r["slots"].tolist() == [10, 11, 12, 13, -1, -1] and r["positions"].tolist() == [10, 11, 12, 13, -1, -1]
    assert r["lens"].tolist() == [14] + lens[1:] and r["n_free"].tolist() == [8]
    assert torch.equal(table[:, 0].cpu(), torch.arange(B, dtype=torch.int32)) and (table[:, 1] == -1).all()


@pytest.mark.parametrize("kw", [dict(per_row=2), dict(n_tokens=7)])
def test_extend_pages_for_live_requests_only(kw):
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    lens, new, free = [64, 0, 5, -2, 127], [1, 2, 2, 1, 2], [9, 8, 7, 6]
    table = [[0, -1, -1], [-1] * 3, [1, -1, -1], [-1] * 3, [2, 3, -1]]
    want = R.extend_ref(lens, [n if x > 0 else 0 for x, n in zip(lens, new)], table, free, 4, **kw)
    td = i32(table)
    r = K.extend_pages(i32(lens), i32(new), td, i32(free), i32([4]), live_only=True, **kw)
    assert r["slots"].flatten().tolist() == want[0] and r["positions"].flatten().tolist() == want[1]
    assert r["granted"].tolist() == want[2] and td.tolist() == want[4] and r["n_free"].tolist() == [want[5]]
    assert r["lens"].tolist() == [max(0, x) for x in want[3]]


def test_overlapping_tables_are_refused():
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    lens, new, table, free, n = i32([3, 70]), i32([1, 1]), i32([[0, -1], [1, 2]]), i32([5, 4, 3]), i32([3])
    with pytest.raises(RuntimeError, match="lens_out and new overlap"):
        K.extend_pages(lens, new, table, free, n, per_row=1, lens_out=new)
    with pytest.raises(RuntimeError, match="lens_out and free_pages overlap"):
        K.release_pages(i32([1, 0]).bool(), lens, table, free, n, lens_out=free[1:])
    r = K.extend_pages(lens, lens, table, free, n, n_tokens=73, lens_out=lens, n_free_out=n)      # in place, twice the tokens
    assert r["lens"].tolist() == [6, 70] and r["granted"].tolist() == [True, False] and n.tolist() == [3]


def test_granted_and_positions_after_a_replay():
    """A captured extension that the pool refuses says so in the cache's attributes, an eager one in between or not."""
    cache = PagedKV8(3, 2, 1, 64, 256, DEV)
    one = torch.ones(2, dtype=torch.int32, device=DEV)
    step = StepGraph(lambda: cache.extend(one, per_row=1), [cache], eager=0)
    step.step()
    assert cache.granted.tolist() == [True, True] and cache.positions.flatten().tolist() == [0, 0]
    cache.extend(torch.tensor([63, 63], dtype=torch.int32, device=DEV), n_tokens=126)       # both pages full, one left
    assert cache.granted.tolist() == [True, True] and cache.lens.tolist() == [64, 64]
    step.step()
    assert cache.granted.tolist() == [True, False] and cache.positions.flatten().tolist() == [64, -1]
    assert cache.lens.tolist() == [65, 64] and cache.n_free.tolist() == [0]
    raw = torch.cuda.CUDAGraph()                                                             # a graph without StepGraph
    with torch.cuda.graph(raw):
        cache.extend(one, per_row=1)
    cache.extend(torch.zeros(2, dtype=torch.int32, device=DEV), per_row=1)
    assert cache.granted.tolist() == [True, True]
    raw.replay()
    assert cache.granted.tolist() == [True, False] and cache.lens.tolist() == [66, 64]


def test_one_table_for_the_pools_of_several_layers():
    """Slots, lengths and pages of one cache address another layer's pools too."""
    B, Hkv, G, D = 3, 2, 4, 128
    gen = torch.Generator().manual_seed(3)
    cache = PagedKV8(8, B, Hkv, D, 256, DEV)
    other = PagedKV8(8, B, Hkv, D, 256, DEV)                              # the same steps with tables of its own
    k2, v2 = (torch.zeros_like(cache.k.view(torch.uint8)).view(cache.k.dtype) for _ in range(2))
    ks2, vs2 = torch.ones_like(cache.k_scale), torch.ones_like(cache.v_scale)
    new = torch.tensor([100, 0, 65], dtype=torch.int32, device=DEV)
    x, y = (torch.randn(165, Hkv, D, generator=gen).to(torch.bfloat16).to(DEV) for _ in range(2))
    slots = cache.extend(new, n_tokens=165)
    cache.write(x, x, slots)
    K.write8(y, x, slots, k2, v2, ks2, vs2)
    other.write(y, x, other.extend(new, n_tokens=165))
    q = torch.randn(B, Hkv * G, D, generator=gen).to(torch.bfloat16).to(DEV)
    got = K.decode8(q, k2, v2, ks2, vs2, 0.1, lens=cache.lens, page_table=cache.table)
    want = other.decode(q, 0.1)
    assert torch.equal(got["out"], want["out"]) and torch.equal(got["lse"], want["lse"])
    assert not torch.equal(cache.decode(q, 0.1)["out"], got["out"])


def test_append_leaves_rows_without_a_request_alone():
    """After a release the row takes no page and no token until something is written for it."""
    B, Hkv, D = 4, 2, 64
    gen = torch.Generator().manual_seed(2)
    cache = PagedKV8(9, B, Hkv, D, 256, DEV)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    x = torch.randn(63 + 64 + 1, Hkv, D, generator=gen).to(torch.bfloat16).to(DEV)
    cache.write(x, x, cache.extend(i32([63, 64, 0, 1]), n_tokens=128))
    cache.release(torch.tensor([0, 1, 0, 0], dtype=torch.bool, device=DEV))
    new = torch.randn(3, B, Hkv, D, generator=gen).to(torch.bfloat16).to(DEV)
    codes, free = cache.k.view(torch.uint8).clone(), cache.free_pages.clone()
    for t in range(3):
        cache.append(new[t], new[t])
    assert cache.lens.tolist() == [66, 0, 0, 4] and cache.n_free.tolist() == [6] and cache.granted.all()
    mine = set(cache.table[0, :2].tolist() + cache.table[3, :1].tolist())
    others = [p for p in range(9) if p not in mine]
    assert len(mine) == 3 and torch.equal(cache.k.view(torch.uint8)[others], codes[others]) and torch.equal(cache.free_pages, free)
    q = torch.randn(B, Hkv, D, generator=gen).to(torch.bfloat16).to(DEV)
    r = cache.decode(q, 0.1)
    assert (r["out"][1:3] == 0).all() and torch.isneginf(r["lse"][1:3]).all() and torch.isfinite(r["lse"][[0, 3]]).all()
    cache.append(new[0], new[0], i32([0, 1, 0, 0]))                            # and a request that begins with one token
    assert cache.lens.tolist() == [66, 1, 0, 4]


# ------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("graph", [False, True], ids=["launches", "captured"])
@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_serving_loop(kind, graph):
    """Requests come and go: prompts are admitted, every live one grows by a token a step, finished ones give their
    pages back to later ones.  The captured form replays extend, write and attention from one graph."""
    B, Hkv, G, D, steps = 5, 2, 4, 128, 40
    gen = torch.Generator().manual_seed(11)
    cache = PagedKV8(24, B, Hkv, D, 512, DEV, dtype=R.KINDS[kind])
    truth = [torch.zeros(Hkv, 0, D) for _ in range(B)], [torch.zeros(Hkv, 0, D) for _ in range(B)]
    rand = lambda *s: torch.randn(*s, generator=gen).to(torch.bfloat16)  # noqa: E731

    def admit(prompts):
        new = torch.tensor(prompts, dtype=torch.int32)
        k, v = rand(sum(prompts), Hkv, D), rand(sum(prompts), Hkv, D)
        slots = cache.extend(new.to(DEV), n_tokens=sum(prompts))
        cache.write(k.to(DEV), v.to(DEV), slots)
        ok, at = cache.granted.tolist(), 0
        for b, n in enumerate(prompts):
            if ok[b]:
                for t, x in zip(truth, (k, v)):
                    t[b] = torch.cat([t[b], x[at:at + n].float().transpose(0, 1)], 1)
            at += n
        return ok

    assert admit([100, 0, 300, 64, 1]) == [True] * 5
    live = torch.tensor([1, 0, 1, 1, 1], dtype=torch.int32, device=DEV)
    kb, vb = (torch.zeros(B, Hkv, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    qb = torch.zeros(B, Hkv * G, D, dtype=torch.bfloat16, device=DEV)
    scale = 1 / math.sqrt(D)

    def launch():
        cache.append(kb, vb, live)
        return cache.decode(qb, scale, out_f32=True)

    step = StepGraph(launch, [cache]) if graph else None
    for t in range(steps):
        if t == 15:                                       # request 2 ends, request 1 begins in its place in the pool
            cache.release(torch.tensor([0, 0, 1, 0, 0], dtype=torch.uint8, device=DEV))
            for x in truth:
                x[2] = x[2][:, :0]
            assert admit([0, 333, 0, 0, 0]) == [True] * 5
            live.copy_(torch.tensor([1, 1, 0, 1, 1], dtype=torch.int32))
        if t == 25:                                       # a prompt that the pool has no room for
            assert admit([0, 0, 900, 0, 0])[2] is False
        k, v, q = rand(B, Hkv, D), rand(B, Hkv, D), rand(B, Hkv * G, D)
        kb.copy_(k), vb.copy_(v), qb.copy_(q)
        r = step.step() if graph else launch()
        ok = cache.granted.tolist()
        for b in range(B):
            if live[b] and ok[b]:
                for x, y in zip(truth, (k, v)):
                    x[b] = torch.cat([x[b], y[b].float()[:, None]], 1)
        lens = cache.lens.tolist()
        assert lens == [x.shape[1] for x in truth[0]]
        ref = R.decode_f64(q, _cpu(cache.k), _cpu(cache.v), cache.k_scale.cpu(), cache.v_scale.cpu(), scale, lens,
                           cache.table.cpu())
        _check(r, ref, D, cache.max_pages, torch.bfloat16)
    # what the pool holds is the tokens that went in, to 8 bits: int8 a step, e4m3 2^-4 and its smallest values
    for b in range(B):
        for got, t in zip(cache.gather(b), truth):
            if not t[b].numel():
                continue
            top = t[b].abs().max()
            bound = 2 * top / 127 if kind == "int8" else 2.0 ** -4 * t[b].abs() + top * 2.0 ** -16
            assert ((got.cpu() - t[b]).abs() <= bound).all()
    assert K.ext().device_status() == 0
    if graph:
        assert step.captures == 1 and step.replays == steps - 1
