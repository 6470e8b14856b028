"""Plain restatements of the 8-bit cache's operators for the tests: attention in 64 bits on the CPU, the write
and the page tables one token and one request at a time."""
import math

import numpy as np
import torch

TILE = 64
KINDS = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
QMAX = {"e4m3": 448.0, "int8": 127.0}
MIN_SCALE = 2.0 ** -100


def decode_f64(q, k, v, ks, vs, scale, lens, table=None, lists=None, nb=None):
    """All arguments on the CPU.  k, v [pages,Hkv,64,D] with table, else [B,Hkv,T,D].  lists: {(b, h): [block, ...]}.
    Besides the results: `mag`, sum of p |v| per output element, and `qk`, the largest scale * sum |q k| per head."""
    B, Hq, D = q.shape
    Hkv = k.shape[1]
    G = Hq // Hkv
    if nb is None:
        nb = table.shape[1] if table is not None else -(-k.shape[2] // TILE)
    out, mag = torch.zeros(B, Hq, D, dtype=torch.float64), torch.zeros(B, Hq, D, dtype=torch.float64)
    lse = torch.full((B, Hq), -math.inf, dtype=torch.float64)
    qk = torch.zeros(B, Hq, dtype=torch.float64)
    bmax = torch.full((B, Hq, nb), -math.inf, dtype=torch.float64)
    bsum = torch.zeros(B, Hq, nb, dtype=torch.float64)
    for b in range(B):
        T = int(lens[b])
        for h in range(Hkv):
            blocks = range(-(-T // TILE)) if lists is None else lists[b, h]
            kk, vv, at = [], [], []
            for j in blocks:
                n = min(TILE, T - j * TILE)
                if n <= 0:
                    continue
                if table is not None:
                    pg = int(table[b, j])
                    if 0 <= pg < k.shape[0]:
                        x, y = k[pg, h, :n].double() * float(ks[pg, h]), v[pg, h, :n].double() * float(vs[pg, h])
                    else:
                        x = y = torch.zeros(n, D, dtype=torch.float64)
                else:
                    x = k[b, h, j * TILE:j * TILE + n].double() * float(ks[b, h, j])
                    y = v[b, h, j * TILE:j * TILE + n].double() * float(vs[b, h, j])
                kk.append(x)
                vv.append(y)
                at.append((j, n))
            if not kk:
                continue
            kk, vv = torch.cat(kk), torch.cat(vv)
            qh = q[b, h * G:(h + 1) * G].double()
            s = qh @ kk.T * scale
            z = torch.logsumexp(s, 1)
            p = torch.exp(s - z[:, None])
            rows = slice(h * G, (h + 1) * G)
            out[b, rows], mag[b, rows], lse[b, rows] = p @ vv, p @ vv.abs(), z
            qk[b, rows] = (qh.abs() @ kk.abs().T).amax(1) * abs(scale)
            o = 0
            for j, n in at:
                m = s[:, o:o + n].amax(1)
                bmax[b, rows, j], bsum[b, rows, j] = m, torch.exp(s[:, o:o + n] - m[:, None]).sum(1)
                o += n
    return {"out": out, "lse": lse, "blk_max": bmax, "blk_sum": bsum, "mag": mag, "qk": qk}


def needed_scale(amax, kind):
    """Smallest power of two s >= 2^-100 with amax <= qmax * s."""
    s = MIN_SCALE
    while QMAX[kind] * s < amax:
        s *= 2
    return s


def to_codes(x, kind):
    """fp32 array in units of the scale -> codes (numpy uint8 bit patterns)."""
    t = torch.from_numpy(np.asarray(x, dtype=np.float32))
    if kind == "e4m3":
        return t.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    r = torch.nan_to_num(t, nan=0.0, posinf=127.0, neginf=-127.0).round().clamp(-127, 127)
    return r.to(torch.int8).view(torch.uint8).numpy()


def write_ref(x, slots, codes, scales, kind):
    """In place, one run after the other.  x float32 [N,Hkv,D]; codes uint8 bit patterns [blocks,Hkv,64,D],
    scales float32 [blocks,Hkv].  Slots outside the cache and second runs of a block in a row are skipped."""
    slots = [int(s) if 0 <= int(s) < codes.shape[0] * TILE else -1 for s in slots]
    i = 0
    while i < len(slots):
        n = 1
        while i + n < len(slots) and slots[i] >= 0 and slots[i + n] == slots[i] + n and slots[i + n] % TILE:
            n += 1
        s = slots[i]
        again = i > 0 and s >= 0 and slots[i - 1] >= 0 and slots[i - 1] // TILE == s // TILE
        if s >= 0 and not again:
            page, row = divmod(s, TILE)
            for h in range(codes.shape[1]):
                vals = x[i:i + n, h]
                fin = np.abs(vals[np.isfinite(vals)])
                need = needed_scale(float(fin.max()) if fin.size else 0.0, kind)
                old = float(scales[page, h])
                if row == 0 or not (old > 0 and math.isfinite(old)):
                    old = MIN_SCALE
                now = max(old, need)
                if now > old and row:
                    t = torch.from_numpy(codes[page, h, :row].copy()).view(KINDS[kind]).float()
                    codes[page, h, :row] = to_codes(t.numpy() * np.float32(np.float32(old) / np.float32(now)), kind)
                with np.errstate(over="ignore", invalid="ignore"):
                    codes[page, h, row:row + n] = to_codes(vals / np.float32(now), kind)
                scales[page, h] = now
        i += n


def extend_ref(lens, new, table, free, n_free, n_tokens=None, per_row=None):
    """Lists of whole numbers; returns slots, positions, granted, lens, table, n_free."""
    lens, table = list(lens), [list(r) for r in table]
    B, cap = len(lens), len(table[0])
    total = n_tokens if per_row is None else B * per_row
    slots, pos, granted = [-1] * total, [-1] * total, []
    used, at, stuck = 0, 0, False
    for b in range(B):
        add = max(0, new[b])
        want, have = -(-(lens[b] + add) // TILE), -(-lens[b] // TILE)
        place = at if per_row is None else b * per_row
        at += add
        ok = want <= cap and (place + add <= total if per_row is None else add <= per_row)
        need = want - have
        if ok and need > 0:
            if stuck or used + need > n_free:
                ok, stuck = False, True
        granted.append(ok)
        if not ok:
            continue
        for j in range(have, want):
            table[b][j] = free[n_free - 1 - used]
            used += 1
        for i in range(add):
            p = lens[b] + i
            slots[place + i], pos[place + i] = table[b][p // TILE] * TILE + p % TILE, p
        lens[b] += add
    return slots, pos, granted, lens, table, n_free - used


def release_ref(done, lens, table, free, n_free):
    lens, free = list(lens), list(free)
    for b, d in enumerate(done):
        if d:
            for j in range(-(-lens[b] // TILE)):
                if n_free < len(free):
                    free[n_free] = table[b][j]
                    n_free += 1
            lens[b] = 0
    return lens, free, n_free
