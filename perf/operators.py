"""Cases for timing the operators of the 8-bit paged cache: the page and slot tables that are built on
the GPU from request lengths (`extend_pages`, `release_pages`), the write of new tokens into the
cache (`write8`), and the single-token attention that reads it (`decode8`).

`run` computes a case either in its plain form (elementary torch operations, fp32) or, with `own`,
through the calls a user of the package makes."""

import math

import torch

own = False

TILE = 64
DEV = "cuda"
KINDS = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
QMAX = {"e4m3": 448.0, "int8": 127.0}
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
MIN_EXP = -100                      # the smallest block scale is 2^-100


# ------------------------------------------------------------------------------------------- cases
def _decode(name, B, lo, hi, Hkv=8, G=4, D=128, kind="e4m3", qtype="bf16", layout="paged", keep=1.0, stats=False,
            empty=0.0):
    return {"name": name, "op": "decode", "B": B, "lo": lo, "hi": hi, "Hkv": Hkv, "G": G, "D": D, "kind": kind,
            "qtype": qtype, "layout": layout, "keep": keep, "stats": stats, "empty": empty}


def _write(name, B, lo, hi, new_lo, new_hi, Hkv=8, D=128, kind="e4m3", qtype="bf16", skip=0.0):
    return {"name": name, "op": "write", "B": B, "lo": lo, "hi": hi, "new_lo": new_lo, "new_hi": new_hi, "Hkv": Hkv,
            "D": D, "kind": kind, "qtype": qtype, "skip": skip}


def _tables(name, op, B, lo, hi, new_lo, new_hi, pool=1.2, done=0.0):
    return {"name": name, "op": op, "B": B, "lo": lo, "hi": hi, "new_lo": new_lo, "new_hi": new_hi, "pool": pool,
            "done": done}


def listed():
    return [
        # one request early in its answer: the call is as short as such a call gets, latency is all
        _decode("decode b1 1k", 1, 1000, 1000),
        # one request with a long context: the whole GPU on eight KV heads of one sequence
        _decode("decode b1 64k", 1, 65536, 65536),
        # the benchmark's largest batch at its longest context
        _decode("decode b16 64k", 16, 65536, 65536),
        # a serving batch: requests of all lengths, some rows of the batch without a request; int8 codes
        _decode("decode ragged b64", 64, 1, 16384, kind="int8", empty=0.1),
        # block lists with statistics, as a policy that reads a third of the blocks uses them
        _decode("decode masked b8 64k", 8, 60000, 65536, keep=0.3, stats=True),
        # small heads, eight query heads a KV head, fp16 queries, a contiguous cache
        _decode("decode d64 g8 contiguous", 12, 3, 5001, Hkv=4, G=8, D=64, kind="int8", qtype="fp16",
                layout="contiguous"),
        # a decode step writes one token a request, most of them in the middle of a block
        _write("write step b256", 256, 1, 8192, 1, 1),
        # prompts of a batch go into fresh pages
        _write("write prompts", 32, 0, 0, 200, 6000),
        # chunks of prompts that begin inside a block; int8 codes, fp16 inputs, some padding tokens
        _write("write chunks d64 int8", 9, 1, 700, 1, 500, Hkv=4, D=64, kind="int8", qtype="fp16", skip=0.05),
        # a decode step of a large batch: a few requests cross into a new page
        _tables("extend step b512", "extend", 512, 0, 8192, 1, 1),
        # admission of prompts, more than the pool can hold: the last ones are refused
        _tables("extend prompts", "extend", 300, 0, 4096, 0, 6000, pool=0.9),
        # finished requests give their pages back
        _tables("release b512", "release", 512, 0, 16384, 0, 0, done=0.3),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["decode", "decode", "decode", "write", "write", "extend", "release"])
    D = rng.choice([64, 128])
    kind, qtype = rng.choice(["e4m3", "int8"]), rng.choice(["bf16", "fp16"])
    if op == "decode":
        B = _log_int(rng, 1, 64)
        Hkv, G = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 4, 5, 8, 12, 16])
        hi = _log_int(rng, 2, max(2, min(65536, 1000000 // B)))
        lo = rng.choice([1, hi, max(1, hi // 2)])
        keep = rng.choice([1.0, 1.0, rng.uniform(0.05, 0.9)])
        c = _decode("", B, lo, hi, Hkv, G, D, kind, qtype, rng.choice(["paged", "paged", "contiguous"]), keep,
                    rng.random() < 0.4, rng.choice([0.0, 0.2]))
    elif op == "write":
        B, mode = _log_int(rng, 1, 300), rng.choice(["step", "prompt", "chunk"])
        hi = 0 if mode == "prompt" else _log_int(rng, 1, 4096)
        new = 1 if mode == "step" else _log_int(rng, 2, max(2, 60000 // B))
        c = _write("", B, min(hi, 1), hi, 1, new, rng.choice([1, 2, 5, 8]), D, kind, qtype, rng.choice([0.0, 0.1]))
    else:
        B = _log_int(rng, 1, 2000)
        hi = _log_int(rng, 1, 16384)
        new = rng.choice([1, _log_int(rng, 2, max(2, 1000000 // B))]) if op == "extend" else 0
        c = _tables("", op, B, 0, hi, 0, new, rng.choice([0.8, 1.0, 1.5]), rng.uniform(0.05, 1.0))
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------ inputs
def _spread(lo, hi, n):
    """n whole numbers that cover [lo, hi] evenly, over the logarithm where the range is wide."""
    u = [(i + 0.5) / n for i in range(n)]
    if hi > 10 * max(lo, 1):
        a = max(lo, 1)
        x = [a * math.exp(v * math.log((hi + 1) / a)) - (lo == 0) for v in u]
    else:
        x = [lo + v * (hi - lo + 1) for v in u]
    return [min(hi, max(lo, math.floor(v))) for v in x]


def _ints(lo, hi, n, gen):
    """The numbers of _spread in an order of the generator's: sizes do not depend on the seed."""
    x = torch.tensor(_spread(lo, hi, n), dtype=torch.int64, device=DEV)
    return x[torch.randperm(n, generator=gen, device=DEV)]


def _pages(x):
    return sum(-(-v // TILE) for v in x)


def _pow2_scale(amax, qmax):
    """Smallest power of two s >= 2^MIN_EXP with amax <= qmax * s (amax >= 0, finite), in fp32."""
    mq, eq = math.frexp(qmax)
    m, e = torch.frexp(amax)
    e = torch.where(amax > 0, e - eq + (m > mq).to(e.dtype), MIN_EXP).clamp(min=MIN_EXP)
    return torch.ldexp(torch.ones_like(amax), e)


def _codes(x, kind):
    """fp32 values in units of the scale -> 8-bit codes, round to nearest even, saturating."""
    if kind == "e4m3":
        return x.clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return torch.nan_to_num(x, nan=0.0, posinf=127.0, neginf=-127.0).round().clamp(-127, 127).to(torch.int8)


def _pool(n, Hkv, D, kind, gen, mean):
    """n blocks [n, Hkv, 64, D] of 8-bit codes with their scales, from values as keys and values have them: a mean
    and a spread of its own for each channel."""
    codes = torch.empty(n, Hkv, TILE, D, dtype=KINDS[kind], device=DEV)
    scales = torch.empty(n, Hkv, device=DEV)
    mu = mean * torch.randn(Hkv, 1, D, generator=gen, device=DEV)
    spread = torch.exp(0.5 * torch.randn(Hkv, 1, D, generator=gen, device=DEV))
    step = max(1, (1 << 26) // (Hkv * TILE * D))
    for i in range(0, n, step):
        x = torch.randn(min(step, n - i), Hkv, TILE, D, generator=gen, device=DEV) * spread + mu
        s = _pow2_scale(x.abs().amax((2, 3)), QMAX[kind])
        codes[i:i + step] = _codes(x / s[..., None, None], kind)
        scales[i:i + step] = s
    return codes, scales


def _table(lens, max_pages, num_pages, gen):
    """Shuffled pages for every block that `lens` fills (-1 behind them), and the free ones as a stack."""
    have = (lens + TILE - 1) // TILE
    order = torch.randperm(num_pages, generator=gen, device=DEV)
    j = torch.arange(max_pages, device=DEV)
    used = j[None] < have[:, None]
    table = torch.full((len(lens), max_pages), -1, dtype=torch.int64, device=DEV)
    n = int(have.sum())
    table[used] = order[:n]
    free = torch.full((num_pages,), -1, dtype=torch.int64, device=DEV)
    free[:num_pages - n] = order[n:]
    return table.to(torch.int32), free.to(torch.int32), torch.tensor([num_pages - n], dtype=torch.int32, device=DEV)


def _prepare_decode(c, gen):
    B, Hkv, G, D = c["B"], c["Hkv"], c["G"], c["D"]
    lens = _ints(c["lo"], c["hi"], B, gen)
    need = int(((lens + TILE - 1) // TILE).sum())
    lens[:int(c["empty"] * B)] = 0                       # rows of the batch without a request
    nb = math.ceil(c["hi"] / TILE)
    q = (1.5 * torch.randn(B, Hkv * G, D, generator=gen, device=DEV)).to(TYPES[c["qtype"]])
    s = {"case": c, "q": q, "lens": lens.to(torch.int32), "scale": 1.0 / math.sqrt(D), "nb": nb, "table": None}
    if c["layout"] == "paged":
        s["table"] = _table(lens, nb, need + 7, gen)[0]
        s["k"], s["ks"] = _pool(need + 7, Hkv, D, c["kind"], gen, 0.5)
        s["v"], s["vs"] = _pool(need + 7, Hkv, D, c["kind"], gen, 0.2)
    else:
        for n, mean in (("k", 0.5), ("v", 0.2)):
            codes, sc = _pool(B * nb, Hkv, D, c["kind"], gen, mean)
            s[n] = codes.view(B, nb, Hkv, TILE, D).transpose(1, 2).reshape(B, Hkv, nb * TILE, D)[:, :, :c["hi"]]
            s[n + "s"] = sc.view(B, nb, Hkv).transpose(1, 2).contiguous()
    s["plan"] = None
    if c["keep"] < 1:
        keep = torch.rand(B, Hkv, nb, generator=gen, device=DEV) < c["keep"]
        j, last = torch.arange(nb, device=DEV), (lens - 1) // TILE
        keep |= (j == 0) | (j[None, None] == last[:, None, None])
        keep &= j[None, None] < ((lens + TILE - 1) // TILE)[:, None, None]
        cnt = keep.sum(-1, dtype=torch.int32)
        idx = torch.argsort(keep.logical_not().to(torch.int8), dim=-1, stable=True).to(torch.int32).contiguous()
        s["plan"] = (idx, cnt, int(cnt.max()))
    return s


def _prepare_write(c, gen):
    B, Hkv, D = c["B"], c["Hkv"], c["D"]
    lens, new = _ints(c["lo"], c["hi"], B, gen), _ints(c["new_lo"], c["new_hi"], B, gen)
    total = lens + new
    pages = int(total.sum()) // TILE + B + 3
    table = _table(total, math.ceil((c["hi"] + c["new_hi"]) / TILE), pages, gen)[0].long()
    b = torch.repeat_interleave(torch.arange(B, device=DEV), new)
    pos = torch.arange(len(b), device=DEV) - (new.cumsum(0) - new)[b] + lens[b]
    slots = table[b, pos // TILE] * TILE + pos % TILE
    if c["skip"]:        # padding: whole requests whose tokens have no slot
        drop = torch.arange(B, device=DEV) % 16 < round(16 * c["skip"])
        slots = torch.where(drop[b], -1, slots)
    x = torch.randn(2, len(b), Hkv, D, generator=gen, device=DEV)
    x = x * torch.exp(0.5 * torch.randn(2, 1, Hkv, D, generator=gen, device=DEV))
    k_new, v_new = x.to(TYPES[c["qtype"]])
    k, ks = _pool(pages, Hkv, D, c["kind"], gen, 0.5)
    v, vs = _pool(pages, Hkv, D, c["kind"], gen, 0.2)
    return {"case": c, "k_new": k_new, "v_new": v_new, "slots": slots, "k": k, "v": v, "ks": ks, "vs": vs}


def _prepare_tables(c, gen):
    B = c["B"]
    lens = _ints(c["lo"], c["hi"], B, gen)
    new = _ints(c["new_lo"], c["new_hi"], B, gen)
    pages = int(((lens + TILE - 1) // TILE).sum()) + 1 + int(c["pool"] * int(new.sum()) / TILE)
    table, free, n_free = _table(lens, math.ceil((c["hi"] + c["new_hi"]) / TILE), pages, gen)
    s = {"case": c, "lens": lens.to(torch.int32), "new": new.to(torch.int32), "table": table, "free": free,
         "n_free": n_free, "tokens": int(new.sum())}
    if c["op"] == "release":
        s["done"] = torch.rand(B, generator=gen, device=DEV) < c["done"]
    return s


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    op = case["op"]
    return (_prepare_decode if op == "decode" else _prepare_write if op == "write" else _prepare_tables)(case, gen)


# ------------------------------------------------------------------------------- the plain forms
def _blocks(s, name):
    """Values [B, Hkv, nb, 64, D] of a cache in fp32, and which tokens [B, nb * 64] there are."""
    c, nb = s["case"], s["nb"]
    if s["table"] is not None:
        page = s["table"].long().clamp(min=0)
        x = s[name][page].transpose(1, 2).float()
        return x * s[name + "s"][page].transpose(1, 2)[..., None, None]
    x = s[name].float()
    pad = nb * TILE - x.shape[2]
    x = torch.cat([x, x.new_zeros(*x.shape[:2], pad, c["D"])], 2) if pad else x
    return x.view(c["B"], c["Hkv"], nb, TILE, c["D"]) * s[name + "s"][:, :, :nb, None, None]


def _plain_decode(s):
    c, nb = s["case"], s["nb"]
    B, Hkv, G, D = c["B"], c["Hkv"], c["G"], c["D"]
    ok = (torch.arange(nb * TILE, device=DEV)[None] < s["lens"][:, None]).view(B, 1, 1, nb, TILE)
    if s["plan"] is not None:
        idx, cnt, _ = s["plan"]
        listed_ = torch.arange(nb, device=DEV)[None, None] < cnt[..., None]
        read = torch.zeros(B, Hkv, nb, dtype=torch.bool, device=DEV).scatter_(2, idx.long(), listed_)
        ok = ok & read.view(B, Hkv, 1, nb, 1)
    q = s["q"].float().view(B, Hkv, G, D)
    sc = torch.matmul(q, _blocks(s, "k").reshape(B, Hkv, nb * TILE, D).transpose(2, 3)) * s["scale"]
    sc = sc.view(B, Hkv, G, nb, TILE).masked_fill(~ok, float("-inf"))
    top = sc.amax((3, 4), keepdim=True)
    p = torch.exp(sc - top.clamp(min=-3e38))
    total = p.sum((3, 4))
    out = torch.matmul(p.view(B, Hkv, G, nb * TILE), _blocks(s, "v").reshape(B, Hkv, nb * TILE, D))
    out = torch.where(total[..., None] > 0, out / total[..., None], 0.0)
    r = {"out": out.view(B, Hkv * G, D).to(TYPES[c["qtype"]]),
         "lse": (top[..., 0, 0] + torch.log(total)).view(B, Hkv * G)}
    if c["stats"]:
        bmax = sc.amax(4)
        r["blk_max"] = bmax.reshape(B, Hkv * G, nb)
        r["blk_sum"] = torch.exp(sc - bmax.clamp(min=-3e38)[..., None]).sum(4).reshape(B, Hkv * G, nb)
    return r


def _plain_write_one(x, codes, scales, slots, kind):
    n, Hkv = codes.shape[:2]
    live = slots >= 0
    page, row = torch.where(live, slots // TILE, n), torch.where(live, slots % TILE, 0)
    x = x.float()
    # each page's first row of this call, and the largest value that goes into it (a place for the padding at n)
    first = torch.full((n + 1,), TILE, dtype=torch.int64, device=DEV).scatter_reduce(0, page, row, "amin")[:n]
    big = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(2)
    amax = torch.zeros(n + 1, Hkv, device=DEV).scatter_reduce(0, page[:, None].expand(-1, Hkv), big, "amax")[:n]
    touched = (first < TILE)[:, None]
    low = 2.0 ** MIN_EXP
    old = torch.where((first > 0)[:, None] & (scales > 0) & torch.isfinite(scales), scales, low)
    now = torch.maximum(old, _pow2_scale(amax, QMAX[kind]))
    grown = touched & (now > old)
    again = _codes(codes.float() * (old / now)[..., None, None], kind)
    below = grown[..., None, None] & (torch.arange(TILE, device=DEV)[None] < first[:, None])[:, None, :, None]
    bits = codes.view(torch.uint8)
    bits.copy_(torch.where(below, again.view(torch.uint8), bits))
    scales.copy_(torch.where(touched, now, scales))
    code = _codes(x / scales[page.clamp(max=n - 1)][..., None], kind).view(torch.uint8)
    keep = torch.cat([bits.view(-1, *bits.shape[1:]), bits.new_zeros(1, *bits.shape[1:])])
    keep[page, :, row] = code
    bits.copy_(keep[:n])


def _plain_write(s):
    kind = s["case"]["kind"]
    _plain_write_one(s["k_new"], s["k"], s["ks"], s["slots"], kind)
    _plain_write_one(s["v_new"], s["v"], s["vs"], s["slots"], kind)


def _plain_extend(s):
    lens, new, table, n_free = s["lens"].long(), s["new"].long(), s["table"], s["n_free"].long()
    B, cap = table.shape
    have, want = (lens + TILE - 1) // TILE, (lens + new + TILE - 1) // TILE
    fits = want <= cap
    need = torch.where(fits, want - have, 0)
    upto = need.cumsum(0)
    granted = fits & ((need == 0) | (upto <= n_free))
    j = torch.arange(cap, device=DEV)[None]
    fresh = granted[:, None] & (j >= have[:, None]) & (j < want[:, None])
    place = n_free - 1 - ((upto - need)[:, None] + j - have[:, None])
    page = s["free"].long()[torch.where(fresh, place, 0)]
    table.copy_(torch.where(fresh, page, table).to(torch.int32))
    b = torch.repeat_interleave(torch.arange(B, device=DEV), new, output_size=s["tokens"])
    pos = torch.arange(s["tokens"], device=DEV) - (new.cumsum(0) - new)[b] + lens[b]
    slot = table[b, (pos // TILE).clamp(max=cap - 1)].long() * TILE + pos % TILE
    got = granted[b]
    return {"slots": torch.where(got, slot, -1), "positions": torch.where(got, pos, -1).to(torch.int32),
            "granted": granted, "lens": torch.where(granted, lens + new, lens).to(torch.int32),
            "n_free": n_free.sub((need * granted).sum()).to(torch.int32)}


def _plain_release(s):
    lens, table = s["lens"].long(), s["table"]
    cap = table.shape[1]
    have = torch.where(s["done"], (lens + TILE - 1) // TILE, 0)
    j = torch.arange(cap, device=DEV)[None]
    back = j < have[:, None]
    place = s["n_free"].long() + (have.cumsum(0) - have)[:, None] + j
    n = s["free"].shape[0]
    longer = torch.cat([s["free"], s["free"].new_zeros(1)])
    longer[torch.where(back, place, n).reshape(-1)] = table.reshape(-1)
    s["free"].copy_(longer[:n])
    return {"lens": torch.where(s["done"], 0, lens).to(torch.int32),
            "n_free": (s["n_free"] + have.sum()).to(torch.int32)}


def run(state):
    s, op = state, state["case"]["op"]
    if op == "decode":
        if not own:
            return _plain_decode(s)
        from kvskip_b200 import kvskip as K
        plan = None if s["plan"] is None else K.Plan(*s["plan"], s["nb"])
        r = K.decode8(s["q"], s["k"], s["v"], s["ks"], s["vs"], s["scale"], lens=s["lens"], page_table=s["table"],
                      plan=plan, stats=s["case"]["stats"])
        return {n: r[n] for n in ("out", "lse", "blk_max", "blk_sum") if n in r}
    if op == "write":
        if not own:
            _plain_write(s)
        else:
            from kvskip_b200 import kvskip as K
            K.write8(s["k_new"], s["v_new"], s["slots"], s["k"], s["v"], s["ks"], s["vs"])
        return {"k": s["k"], "v": s["v"], "k_scale": s["ks"], "v_scale": s["vs"]}
    if op == "extend":
        if not own:
            r = _plain_extend(s)
        else:
            from kvskip_b200 import kvskip as K
            r = K.extend_pages(s["lens"], s["new"], s["table"], s["free"], s["n_free"], n_tokens=s["tokens"])
        return {**{n: r[n] for n in ("slots", "positions", "granted", "lens", "n_free")}, "table": s["table"]}
    if not own:
        r = _plain_release(s)
    else:
        from kvskip_b200 import kvskip as K
        r = K.release_pages(s["done"], s["lens"], s["table"], s["free"], s["n_free"])
    return {"lens": r["lens"], "n_free": r["n_free"], "free": s["free"]}


# ------------------------------------------------------------------------------------------- work
def work(case):
    c, B = case, case["B"]
    lens = _spread(c["lo"], c["hi"], B)
    if c["op"] == "decode":
        # (which requests are the empty ones goes by the seed: their share of the tokens is the mean one)
        live = (B - int(c["empty"] * B)) / B
        tokens, blocks = live * sum(lens), live * _pages(lens)
        # a block list holds the first and the newest block too
        part = 1.0 if c["keep"] == 1 else min(1.0, c["keep"] + (1 - c["keep"]) * min(1.0, 2 * B * live / blocks))
        heads, nb = B * c["Hkv"] * c["G"], math.ceil(c["hi"] / TILE)
        read = c["Hkv"] * part
        return {"bytes": 2 * c["D"] * tokens * read + 8 * blocks * read + 4 * heads * c["D"] + 4 * heads
                + (8 * heads * nb if c["stats"] else 0), "flops": 4 * c["D"] * c["G"] * tokens * read}
    n = sum(_spread(c["new_lo"], c["new_hi"], B))
    if c["op"] == "write":
        n *= 1 - round(16 * c["skip"]) / 16
        return {"bytes": 6 * n * c["Hkv"] * c["D"] + 8 * n, "flops": 4 * n * c["Hkv"] * c["D"]}
    if c["op"] == "extend":
        return {"bytes": 12 * n + 17 * B + 8 * n / TILE, "flops": 0}
    return {"bytes": 8 * c["done"] * _pages(lens) + 9 * B + 8, "flops": 0}


# ---------------------------------------------------------------------------- the definition, in 64 bits
def _exact_decode(s):
    c, nb = s["case"], s["nb"]
    B, Hkv, G, D = c["B"], c["Hkv"], c["G"], c["D"]
    out = torch.zeros(B, Hkv * G, D, dtype=torch.float64, device=DEV)
    lse = torch.full((B, Hkv * G), -math.inf, dtype=torch.float64, device=DEV)
    bmax = torch.full((B, Hkv * G, nb), -math.inf, dtype=torch.float64, device=DEV)
    bsum = torch.zeros(B, Hkv * G, nb, dtype=torch.float64, device=DEV)
    lens = s["lens"].tolist()
    for b, T in enumerate(lens):
        n = -(-T // TILE)
        for h in range(Hkv if T else 0):
            if s["plan"] is not None:
                blocks = s["plan"][0][b, h, :int(s["plan"][1][b, h])].long()
            else:
                blocks = torch.arange(n, device=DEV)
            t = (blocks[:, None] * TILE + torch.arange(TILE, device=DEV)).reshape(-1)
            t = t[t < T]
            if not t.numel():
                continue
            if s["table"] is not None:
                pg = s["table"][b].long()[t // TILE]
                k, v = s["k"][pg, h, t % TILE].double(), s["v"][pg, h, t % TILE].double()
                k, v = k * s["ks"][pg, h].double()[:, None], v * s["vs"][pg, h].double()[:, None]
            else:
                k = s["k"][b, h, t].double() * s["ks"][b, h, t // TILE].double()[:, None]
                v = s["v"][b, h, t].double() * s["vs"][b, h, t // TILE].double()[:, None]
            x = s["q"][b, h * G:(h + 1) * G].double() @ k.T * s["scale"]
            z = torch.logsumexp(x, 1)
            rows = slice(h * G, (h + 1) * G)
            lse[b, rows] = z
            out[b, rows] = torch.exp(x - z[:, None]) @ v
            if c["stats"]:
                at = (t // TILE)[None].expand(G, -1)
                m = bmax[b, rows].scatter_reduce(1, at, x, "amax")
                bmax[b, rows] = m
                bsum[b, rows] = bsum[b, rows].scatter_add(1, at, torch.exp(x - m.gather(1, at)))
    r = {"out": out, "lse": lse}
    return {**r, "blk_max": bmax, "blk_sum": bsum} if c["stats"] else r


def _round_e4m3(x):
    """The nearest value of 4 exponent and 3 mantissa bits, ties to even: multiples of 2^(e-3) for 2^e <= |x| < 2^(e+1),
    of 2^-9 below 2^-6; at most 448."""
    step = torch.ldexp(torch.ones_like(x), torch.frexp(x.abs().clamp(min=2.0 ** -6))[1] - 4)
    return (torch.round(x / step) * step).clamp(-448, 448)


def _exact_write(s):
    c = s["case"]
    r = {}
    for n in ("k", "v"):
        codes, scales, x = s[n].double(), s[n + "s"].double(), s[n + "_new"].double()
        slots = s["slots"]
        live = slots >= 0
        x, page, row = x[live], slots[live] // TILE, slots[live] % TILE
        # groups of tokens that go into one page
        pages, group = torch.unique(page, return_inverse=True)
        H = x.shape[1]
        amax = torch.zeros(len(pages), H, dtype=torch.float64, device=DEV)
        amax = amax.scatter_reduce(0, group[:, None].expand(-1, H), x.abs().amax(2), "amax")
        first = torch.full((len(pages),), TILE, device=DEV).scatter_reduce(0, group, row, "amin")
        m, e = torch.frexp(amax / QMAX[c["kind"]])       # m = 0.5: a power of two by itself
        need = torch.where(amax > 0, torch.ldexp(torch.ones_like(m), e - (m == 0.5).to(e.dtype)), 0.0)
        need = need.clamp(min=2.0 ** MIN_EXP)
        old = torch.where(first[:, None] > 0, scales[pages], 2.0 ** MIN_EXP)
        now = torch.maximum(need, old)
        block = codes[pages]
        below = (torch.arange(TILE, device=DEV)[None] < first[:, None])[:, None, :, None]
        block = torch.where(below, _round_e4m3(block * (old / now)[..., None, None]), block)
        block[group, :, row] = _round_e4m3(x / now[group][..., None])
        codes[pages], scales[pages] = block, now
        # (int8 codes are whole numbers: they are equal or wrong)
        r[n], r[n + "_scale"] = codes if c["kind"] == "e4m3" else None, scales
    return r


def exact(case, seed):
    if case["op"] == "decode":
        return _exact_decode(prepare(case, seed))
    if case["op"] == "write":
        return _exact_write(prepare(case, seed))
    return None         # page numbers and lengths are whole numbers
