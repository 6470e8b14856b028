"""Python front end of the sm_100a decode-attention kernels.

Drop-in for the reference's `kernels/kvskip.py` (format37/kvskip kernels/kvskip.py:24-208): same
module-level names, signatures, defaults and return dictionaries, so `src/kvskip_attn.py` and the
`bench/` scripts of the reference run on top of it unchanged (`from kernels import kvskip` resolves
to this module through the `kernels/` package at the repository root).

    decode(q, k, v, scale)                                  dense
    decode(q, k, v, scale, plan=make_plan(keep))            only the listed blocks are read
    decode(q, k, v, scale, stats=True)                      + per-block max and sum-exp
    decode(q, k, v, scale, stats=True, load_v=False)        statistics only: K is read, V is not
    vskip_one_pass / vskip_two_pass / pv                    V-skip variants
    decode8 / write8 / extend_pages / release_pages         a cache of 8-bit codes with block scales, one
                                                            length per sequence, page tables on the device

q is [B, Hq, D] or [B, Hq, 1, D]; k, v are [B, Hkv, T, D] views with any batch/head/token strides
and D contiguous.  Blocks are 64 tokens counted from position 0.

There is no CPU path: every call needs the compiled extension and a CUDA device, and raises
otherwise.
"""

import importlib.util
import math
import os
from dataclasses import dataclass
from pathlib import Path

import torch

HERE = Path(__file__).resolve().parent
TILE = 64
_EXT = None


def ext():
    """The compiled extension module (decode, vskip1, pv, plan, update, read_bw, ...).

    Loaded from the in-tree `_kvskip_ext.so` (from the directory $KVSKIP_BUILD when that is set);
    if it is missing and a CUDA toolkit is present it is built once (`python -m kvskip_b200.build`).  Raises RuntimeError if it cannot be had: nothing
    in this package computes without it."""
    global _EXT
    if _EXT is None:
        from . import build as _build
        so = _build.EXT
        if not so.exists() or not _build.LIB.exists():
            if os.environ.get("KVSKIP_NO_BUILD"):
                raise RuntimeError(f"kvskip_b200: {so} is missing and KVSKIP_NO_BUILD is set")
            try:
                _build.build_all(verbose=bool(os.environ.get("KVSKIP_VERBOSE")))
            except Exception as e:  # noqa: BLE001
                raise RuntimeError("kvskip_b200: the CUDA extension is not built and building it failed "
                                   f"(run `python -m kvskip_b200.build`): {e}") from e
        spec = importlib.util.spec_from_file_location("_kvskip_ext", so)
        mod = importlib.util.module_from_spec(spec)
        try:
            spec.loader.exec_module(mod)
        except Exception as e:  # noqa: BLE001
            raise RuntimeError(f"kvskip_b200: cannot load {so}: {e}") from e
        _EXT = mod
    return _EXT


class DeviceWaitError(RuntimeError):
    """A bounded wait inside a kernel ran out (a load that never arrived, a peer GPU that never
    flagged its rows), or a kernel skipped what one of its tables pointed to (0x300 to 0x303).  `code` is the
    kernel's status word: 0x1xx to 0x4xx from 0x308 on, 0x6xx and 0x7xx waits on this GPU's own loads (0x700 / 0x720 + warp:
    K / V of decode8, 0x740 + warp: write8), 0x500 + r / 0x510 + r the exchange with rank r of a sequence-sharded step."""

    SKIPPED = {0x300: "a page table entry is outside the pool; the token was not read",
               0x301: "a page table entry is outside the pool; the token was not written",
               0x302: "a slot is outside the 8-bit cache; its token was not written",
               0x303: "two runs of one block stand next to each other in the slot list; the second was not written"}

    def __init__(self, code: int, what: str):
        why = self.SKIPPED.get(code)
        super().__init__(f"{what}: {why} (status word {code:#x})" if why else
                         f"{what}: a device-side wait gave up (status word {code:#x}); the results of that launch "
                         "are incomplete")
        self.code = code


def check_status(what: str = "kvskip") -> None:
    """Synchronise the current stream, read the kernels' status word and raise DeviceWaitError if a
    wait timed out or a table pointed outside (the word is cleared).  Blocks the host: call it where a synchronisation is
    acceptable (end of a decode step, after a failed exchange), or set KVSKIP_CHECK_STATUS=1 to
    have every front-end call do it (debugging)."""
    code = int(ext().device_status())
    if code:
        raise DeviceWaitError(code, what)


def _auto_check(what: str) -> None:
    if os.environ.get("KVSKIP_CHECK_STATUS", "") not in ("", "0"):
        check_status(what)


_SMS: dict = {}


def num_sms() -> int:
    """SMs of the current device (looked up once per device: the query costs microseconds of host
    time, and a decode loop asks on every step)."""
    dev = torch.cuda.current_device()
    n = _SMS.get(dev)
    if n is None:
        n = _SMS[dev] = torch.cuda.get_device_properties(dev).multi_processor_count
    return n


def num_splits_for(bh: int, n_tiles: int, sms: int | None = None, max_splits: int = 64,
                   min_tiles: int = 4) -> int:
    """Split count for bh = B*Hkv sequences of n_tiles blocks each, one CTA per SM.

    Candidates are scored by how full the last wave is (CTAs / (waves * SMs)) minus a small
    penalty per split, so that of two equally full layouts the one with fewer partials to merge
    wins; a split never gets fewer than `min_tiles` blocks."""
    sms = sms or num_sms()
    choice, top = 1, -1.0
    s = 1
    while s <= max_splits:
        if s > 1 and -(-n_tiles // s) < min_tiles:
            break
        ctas = bh * s
        fill = ctas / (-(-ctas // sms) * sms)
        score = fill - 0.002 * s
        if score > top + 1e-9:
            choice, top = s, score
        s += 1
    return choice


@dataclass
class Plan:
    """Block list of the masked kernel."""
    block_idx: torch.Tensor   # int32 [B, Hkv, >= max_cnt]: blocks to read first, ascending
    block_cnt: torch.Tensor   # int32 [B, Hkv]
    max_cnt: int              # longest list (sizes the split count)
    nb: int


def make_plan(keep: torch.Tensor, sync: bool = True) -> Plan:
    """bool [B, Hkv, nb] -> Plan.  sync=True reads the longest list length back to size the splits;
    sync=False sizes them for nb blocks and never touches the host."""
    nb = keep.shape[-1]
    cnt = keep.sum(-1, dtype=torch.int32).contiguous()
    # stable sort of "dropped" flags: kept blocks come first and stay in ascending order
    order = torch.argsort(keep.logical_not().to(torch.int8), dim=-1, stable=True).to(torch.int32).contiguous()
    return Plan(order, cnt, int(cnt.max()) if sync else nb, nb)


QUEUE_MIN_HEADS = 32      # (batch, kv head) pairs from which block lists go to the persistent queue kernel


def splits_for_unsynced_plan(bh: int, nb: int) -> int:
    """Split count (pieces provisioned per head) for a block list whose true lengths are not known
    on the host (sized for nb).  The tensor-core kernels cut every list into pieces of at least 24
    blocks, so a short list uses few of the provisioned pieces.
      * from 32 (batch, kv head) pairs on, the pieces are pulled from a queue by one persistent CTA
        per SM: 12 pieces per head measured best (a head that reads everything is cut into 12 long
        pieces, which are handed out first; more pieces make the merge of a head the tail of the
        launch);
      * below that every piece is a CTA of its own: enough splits for a head that reads every block
        to spread over many SMs."""
    if bh >= QUEUE_MIN_HEADS and ext().get_option("queue"):
        return max(1, min(12, -(-nb // 24)))
    base = num_splits_for(bh, nb)
    if bh * base <= 2 * num_sms():
        return min(64, max(base, -(-nb // 24)))
    return base


def _q3(q):
    return q.squeeze(2) if q.dim() == 4 else q


def decode(q, k, v, scale: float, *, plan: Plan | None = None, stats: bool = False, load_v: bool = True,
           num_splits: int | None = None, stages: int = 2, out_f32: bool = False, write_p: bool = False,
           t_dev: torch.Tensor | None = None, page_table: torch.Tensor | None = None,
           seq_len: int | None = None) -> dict:
    """One layer's decode attention.  Returns dict(out bf16 [B,Hq,D] (None without load_v),
    lse fp32 [B,Hq], num_splits[, blk_max, blk_sum fp32 [B,Hq,nb]][, out_f32][, p fp16 [B,Hq,nb*64]]).

    t_dev (one-element int32 CUDA tensor, not in the reference): the sequence length is read from
    it on the device; k and v are then views of the whole provisioned cache and their length is
    only a bound (it sizes the launch and the statistics rows).  For captured decode steps.

    page_table (int32 [B, max_pages], not in the reference) with seq_len: k and v are page pools
    [pages, Hkv, 64, D] and block j of sequence b is page page_table[b, j] (`kvskip_b200.cache.PagedKV`)."""
    q = _q3(q)
    B, Hkv, T = q.shape[0], k.shape[1], k.shape[2]
    if page_table is not None:
        if seq_len is None:
            raise ValueError("a paged cache needs seq_len")
        T = int(seq_len)
    if num_splits is None:
        n_items = math.ceil(T / TILE) if plan is None else plan.max_cnt
        # the tensor-core kernel owns an SM; three CTAs of the exact-order kernel share one
        tc = q.shape[-1] == 128 or (q.shape[-1] == 64 and not write_p)
        per_sm = 1 if (tc and ext().get_option("decode_path") != 1) else 3
        if plan is not None and per_sm == 1 and plan.max_cnt == plan.nb and load_v:
            num_splits = splits_for_unsynced_plan(B * Hkv, n_items)
        else:
            num_splits = num_splits_for(B * Hkv, n_items, sms=per_sm * num_sms())
            if (plan is not None and load_v and q.shape[-1] == 128 and per_sm == 1 and B * Hkv >= QUEUE_MIN_HEADS
                    and ext().get_option("queue")):
                # lists of known length on the persistent queue kernel: few, long pieces measured best
                # (every piece costs the consumers a reload of q and of the list, and the merger a merge)
                num_splits = min(num_splits, 8)
    bi, bc = (None, None) if plan is None else (plan.block_idx, plan.block_cnt)
    out, lse, bmax, bsum, o32, pbuf = ext().decode(q, k, v, float(scale), bi, bc, stats, load_v,
                                                   int(num_splits), int(stages), out_f32, write_p, t_dev,
                                                   page_table, int(seq_len or 0))
    _auto_check("decode")
    res = {"out": out if load_v else None, "lse": lse, "num_splits": num_splits}
    if stats:
        res["blk_max"], res["blk_sum"] = bmax, bsum
    if out_f32:
        res["out_f32"] = o32
    if write_p:
        res["p"] = pbuf
    return res


def block_weights(blk_max: torch.Tensor, blk_sum: torch.Tensor) -> torch.Tensor:
    """Softmax mass of every block, [B, Hq, nb], from the statistics outputs."""
    return torch.softmax(blk_max + torch.log(blk_sum), dim=-1)


def always_keep(nb: int, local: int, device) -> torch.Tensor:
    """Blocks every sparse mode reads: block 0 (sink) and the `local` newest."""
    a = torch.zeros(nb, dtype=torch.bool, device=device)
    a[0] = True
    a[-local:] = True
    return a


def select_blocks(logw: torch.Tensor, G: int, rule: str, value: float, local: int = 2) -> torch.Tensor:
    """Block selection per KV head (union over its G query heads) from unnormalised block
    log-weights [B, Hq, nb].  "tau": weight >= value; "topp": fewest blocks whose mass reaches
    value.  Sink and `local` newest blocks are always selected.  Returns bool [B, Hq//G, nb]."""
    B, Hq, nb = logw.shape
    w = torch.softmax(logw, dim=-1)
    if rule == "tau":
        per_head = w >= value
    elif rule == "topp":
        sorted_w, perm = w.sort(dim=-1, descending=True)
        before = sorted_w.cumsum(-1) - sorted_w            # mass of the heavier blocks
        per_head = torch.zeros_like(before, dtype=torch.bool).scatter(-1, perm, before < value)
    else:
        raise ValueError(rule)
    return per_head.view(B, Hq // G, G, nb).any(2) | always_keep(nb, local, logw.device)


def pv_splits(bh: int, max_cnt: int, sms: int | None = None) -> int:
    """Splits of the second pass of the two-pass V-skip (not in the reference, which uses
    num_splits_for): one wave of CTAs -- as many splits per (batch, kv head) as keep the grid within
    the SM count, pieces of at least 16 blocks.  Measured on B200 at 64k with 55 % of the blocks
    selected: batch 4, 4 splits 55 us against 61 us with the reference's 9; batch 8, 2 splits 100 us
    against 104 us with 16; batch 1 (18 splits) and batch 16 (1 split at 32k) as before or better."""
    sms = sms or num_sms()
    return max(1, min(sms // max(1, bh), math.ceil(max_cnt / 16)))


def pv(P, v, blk_scale, plan: Plan, num_splits: int | None = None, out_f32: bool = False,
       t_dev: torch.Tensor | None = None):
    if num_splits is None:
        num_splits = pv_splits(v.shape[0] * v.shape[1], plan.max_cnt)
    return ext().pv(P, v, blk_scale, plan.block_idx, plan.block_cnt, int(num_splits), out_f32, t_dev)


def vskip_two_pass(q, k, v, scale: float, rule: str = "topp", value: float = 0.99, local: int = 2,
                   sync: bool = True, out_f32: bool = False, device_select: bool = True,
                   t_dev: torch.Tensor | None = None) -> dict:
    """Two-pass V-skip: a statistics pass over all of K that also writes P = exp(s - block max) in
    fp16, block selection per GQA union, then a pass over P and V of the selected blocks.
    device_select (not in the reference): the selection between the passes runs as one kernel;
    False gives the reference's torch formulation (sort + cumulative sum).
    t_dev (not in the reference): the length is read on the device by all three launches (k, v are
    views of the whole provisioned cache, sync must be False): for captured decode steps."""
    q = _q3(q)
    B, Hq, _ = q.shape
    Hkv = k.shape[1]
    G = Hq // Hkv
    if t_dev is not None and (sync or not device_select or G != 4):
        raise ValueError("vskip_two_pass with t_dev: sync=False, device_select=True, G = 4")
    first = decode(q, k, v, scale, stats=True, load_v=False, write_p=True, t_dev=t_dev)
    if device_select and G == 4 and rule in ("topp", "tau"):
        # selection, block list and second-pass weights in one launch instead of a dozen torch ops
        keep8, bi, bc, weight = ext().select(first["blk_max"], first["blk_sum"], 0 if rule == "topp" else 1,
                                             float(value), int(local), t_dev, int(k.shape[2]) if t_dev is not None else 0)
        nb = keep8.shape[-1]
        plan = Plan(bi, bc, int(bc.max()) if sync else nb, nb)
        out, o32 = pv(first["p"], v, weight, plan, out_f32=out_f32, t_dev=t_dev)
        keep = keep8.bool()
        res = {"out": out, "keep": keep, "kept_frac": keep.float().mean().item() if sync else None}
        if out_f32:
            res["out_f32"] = o32
        return res
    logw = first["blk_max"] + torch.log(first["blk_sum"])
    keep = select_blocks(logw, G, rule, value, local)
    keep_q = keep.repeat_interleave(G, dim=1)
    lse_kept = logw.masked_fill(~keep_q, float("-inf")).logsumexp(-1, keepdim=True)
    weight = torch.exp(first["blk_max"] - lse_kept).masked_fill(~keep_q, 0.0)
    weight = weight.view(B, Hkv, G, -1).transpose(2, 3).contiguous()          # [B, Hkv, nb, G]
    out, o32 = pv(first["p"], v, weight, make_plan(keep, sync=sync), out_f32=out_f32)
    res = {"out": out, "keep": keep, "kept_frac": keep.float().mean().item() if sync else None}
    if out_f32:
        res["out_f32"] = o32
    return res


def vskip_one_pass(q, k, v, scale: float, tau: float = 1e-4, local: int = 2, num_splits: int | None = None,
                   out_f32: bool = False, count: bool = False, lse_prev: torch.Tensor | None = None,
                   sync: bool = True, page_table: torch.Tensor | None = None, seq_len: int | None = None,
                   t_dev: torch.Tensor | None = None) -> dict:
    """Single-pass V-skip: K is read once; the V block of a tile is read only if some query head of
    the group gives the block an estimated weight >= tau.  The normaliser estimate is `lse_prev`
    (per query head, e.g. the "lse" this function returned one step earlier); without it every
    CTA uses the sink block's log-sum-exp, a lower bound that keeps every block the exact rule
    keeps.  count=True adds "v_tiles" [B, Hkv] (and "kept_frac" when sync).
    page_table with seq_len (not in the reference): k and v are page pools, as in `decode`.
    t_dev (not in the reference): the length is read on the device (k, v views of the whole
    provisioned cache; count with sync=False only): for captured decode steps."""
    q = _q3(q)
    B, Hkv, T = q.shape[0], k.shape[1], k.shape[2]
    if page_table is not None:
        if seq_len is None:
            raise ValueError("a paged cache needs seq_len")
        T = int(seq_len)
    nb = math.ceil(T / TILE)
    if num_splits is None:
        num_splits = num_splits_for(B * Hkv, nb)
    out, lse, o32, cnt = ext().vskip1(q, k, v, float(scale), float(tau), int(local), int(num_splits),
                                      out_f32, count, lse_prev, page_table, int(seq_len or 0), t_dev)
    _auto_check("vskip_one_pass")
    res = {"out": out, "lse": lse, "num_splits": num_splits}
    if out_f32:
        res["out_f32"] = o32
    if count:
        res["v_tiles"] = cnt
        if sync:
            res["kept_frac"] = (cnt.sum() / (B * Hkv * nb)).item()
    return res


def decode8(q, k, v, k_scale, v_scale, scale: float, *, lens: torch.Tensor | None = None,
            page_table: torch.Tensor | None = None, max_len: int | None = None, plan: Plan | None = None,
            stats: bool = False, out_f32: bool = False) -> dict:
    """`decode` over a cache of 8-bit codes with one scale per 64-token block and KV head (value = code *
    scale), with one length per sequence.  Not in the reference.

    q bf16 or fp16 [B,Hq,D] or [B,Hq,1,D], Hq = 1 to 16 times Hkv, D 64 or 128.  k, v are float8_e4m3fn or
    int8: page pools [pages,Hkv,64,D] with page_table int32 [B,max_pages] and k_scale, v_scale fp32
    [pages,Hkv] (`kvskip_b200.cache.PagedKV8`), or contiguous views [B,Hkv,T,D] with scales
    [B,Hkv,ceil(T/64)].  lens int32 [B] is read on the device (clamped to what the cache holds, or to max_len,
    which bounds the launch and the statistics rows); without it every sequence of a contiguous
    cache has T tokens.  A sequence of length 0 gives out = 0, lse = -inf; rows behind a length may hold anything.
    plan: only the listed blocks are read (`make_plan`; its length is not read back).
    Returns dict(out of q's type, lse fp32 [B,Hq][, blk_max, blk_sum fp32 [B,Hq,nb]][, out_f32])."""
    if q.dim() == 4:
        q = q.squeeze(2)
    if max_len is not None and max_len < 1:
        raise ValueError("decode8: max_len >= 1")
    e = _EXT or ext()
    bi, bc = (None, None) if plan is None else (plan.block_idx, plan.block_cnt)
    out, lse, bmax, bsum, o32 = e.decode8(q, k, v, k_scale, v_scale, scale, lens, page_table, max_len or 0, bi, bc, stats,
                                          out_f32)
    if e.check_wanted():
        check_status("decode8")
    res = {"out": out, "lse": lse}
    if stats:
        res["blk_max"], res["blk_sum"] = bmax, bsum
    if out_f32:
        res["out_f32"] = o32
    return res


def write8(k_new, v_new, slots, k, v, k_scale, v_scale) -> None:
    """New tokens into an 8-bit cache (both forms of `decode8`), in place.  Not in the reference.

    k_new, v_new bf16 or fp16 [N,Hkv,D] with slots int64 [N], or [B,Hkv,S,D] with slots [B,S].  A slot is page *
    64 + row, or in a contiguous cache (sequence * ceil(T/64) + block) * 64 + row; a negative one skips its token
    (padding).  Tokens of one block stand next to each other with ascending rows, as `extend_pages` lists
    them.  The scale of a block is the smallest power of two that covers its values so far; when a token
    makes it grow, the codes already there are rounded to the new scale.  A token in row 0 starts its block
    afresh, whatever page and scale held before.  Infinities saturate; a NaN stays one in e4m3 and is 0 in int8.
    A slot outside the cache is skipped and sets the status word (`check_status`).  Two runs of one block in a call race
    for it unless they are neighbours (then the second is skipped, with the status word set); KVSKIP_CHECK_STATUS=1
    refuses them.  k and v, and k_scale and v_scale, are different memory, without strides of 0."""
    e = _EXT or ext()
    checked = e.check_wanted()
    if checked:
        _check_runs(slots)
    e.write8(k_new, v_new, slots, k, v, k_scale, v_scale)
    if checked:
        check_status("write8")


def _check_runs(slots) -> None:
    """Raises ValueError if a block's tokens are not one run of the slot list (reads the list back)."""
    s = slots.reshape(-1)
    before = torch.cat([s.new_full((1,), -1), s[:-1]])
    first = (s >= 0) & ~((before >= 0) & (s == before + 1) & (s % TILE != 0))
    blocks = s[first] // TILE
    if blocks.unique().numel() != blocks.numel():
        raise ValueError("write8: the tokens of a block must stand next to each other in `slots`, with ascending rows")


def extend_pages(lens, new, page_table, free_pages, n_free, *, n_tokens: int | None = None, per_row: int | None = None,
                 lens_out: torch.Tensor | None = None, n_free_out: torch.Tensor | None = None,
                 granted_out: torch.Tensor | None = None, live_only: bool = False) -> dict:
    """Pages and slots for `new` int32 [B] more tokens of requests that hold `lens` int32 [B] tokens, built on
    the device without a host synchronisation.  Not in the reference, whose caller counts on the host.

    page_table int32 [B,max_pages] receives the pages of new blocks, taken from the top of the stack
    free_pages int32 [pages] with n_free int32 [1] entries.  A request that does not fit (into max_pages, into
    the slot list, or into what earlier requests left of the stack) is refused as a whole.  live_only: requests of
    length 0 get nothing, whatever `new` says.
    Slots and positions: packed, request after request, in n_tokens places, or with per_row in a padded
    [B,per_row] list; -1 in places without a token.
    Returns dict(slots int64, positions int32, granted bool [B], lens, n_free); the last three are new tensors unless
    granted_out / lens_out / n_free_out are given; the latter two may be lens and n_free themselves, nothing else that is
    written may overlap another argument.  The new tensors of a call share one allocation: keeping one keeps them all."""
    if (n_tokens is None) == (per_row is None):
        raise ValueError("extend_pages: either n_tokens (packed) or per_row (padded)")
    if per_row is not None and per_row < 1:
        raise ValueError("extend_pages: per_row >= 1")
    slots, positions, granted, lens2, n2 = (_EXT or ext()).extend_pages(lens, new, page_table, free_pages, n_free, n_tokens or 0,
                                                              per_row or 0, lens_out, n_free_out, granted_out, live_only)
    return {"slots": slots, "positions": positions, "granted": granted, "lens": lens2, "n_free": n2}


def release_pages(done, lens, page_table, free_pages, n_free, *, lens_out: torch.Tensor | None = None,
                  n_free_out: torch.Tensor | None = None) -> dict:
    """The pages of the requests marked in `done` (bool or uint8 [B]) go back to the stack of
    `extend_pages` and their lengths become 0 (the table is left as it is).  Returns dict(lens, n_free), new
    tensors unless lens_out / n_free_out are given."""
    lens2, n2 = (_EXT or ext()).release_pages(done, lens, page_table, free_pages, n_free, lens_out, n_free_out)
    return {"lens": lens2, "n_free": n2}
