"""Inputs of the 8-bit attention whose scores are exact in fp32, so that what is left of its error is the weights, the sums
and the last roundings, and can be bounded closely enough to tell a weight of 22 bits from one of 11.

q and the keys are small whole numbers, the key scales powers of two, and the softmax scale is ln 2 / 32: a score times
log2 e is a multiple of 2^-6 of a few units, in every step of the arithmetic.  Values and their scales are arbitrary.

The bound on |out - exact|, relative to sum p |v|, counts (u = 2^-22, the error of an fp32 base-2 exponential):
  weights      u each, in numerator and normaliser                                              2 u
  rescaling    blocks to a running maximum, pieces to a warp group's, groups to the head's:
               an exponential and two products each time, in both                               2 (nb + 2) (u + 2 u / 4)
  two parts    11 bits and 11 bits of what is left                                                u
  sums         n products of each part, every addition truncated (u / 2 of the sum so far):      n u
               the normaliser, n additions rounded (u / 4 each)                                  n u / 4
  blocks       nb additions of each, a product with the value scale                              (2 nb + 1) u / 4
  division     quotient and product                                                              2 u
with n the tokens of a block (an addition of 0 is exact) and nb the blocks."""
import math

import torch

TILE = 64
U = 2.0 ** -22
LENS = [12, 1, 64, 5, 130]
SCALE = math.log(2.0) / 32


def inputs(Hkv, G, D, kind, qtype, seed):
    """CPU tensors of a contiguous cache, [B,Hkv,T,D] codes with [B,Hkv,nb] scales."""
    gen = torch.Generator().manual_seed(seed)
    B, T = len(LENS), max(LENS)
    nb = -(-T // TILE)
    dtype = torch.float8_e4m3fn if kind == "e4m3" else torch.int8
    whole = lambda n, *s: torch.randint(-n, n + 1, s, generator=gen).float()  # noqa: E731
    width = 1 if D == 128 else 2                                # scores of the same spread for both head sizes
    q = whole(3, B, Hkv * G, D).to(qtype)
    k = (whole(4, B, Hkv, T, D) * width).to(dtype)
    v = torch.randn(B, Hkv, T, D, generator=gen) * 40
    v = v.to(dtype) if kind == "e4m3" else v.round().clamp(-127, 127).to(dtype)
    ks = torch.exp2(torch.randint(-1, 1, (B, Hkv, nb), generator=gen).float())
    vs = torch.exp(0.3 * torch.randn(B, Hkv, nb, generator=gen)) / 40
    return {"q": q, "k": k, "v": v, "ks": ks, "vs": vs, "nb": nb}


def log2_scores(c, b, h, G):
    """[G, n] scores of one sequence and KV head times log2 e, exactly."""
    n = LENS[b]
    k = c["k"][b, h, :n].double() * c["ks"][b, h].double().repeat_interleave(TILE)[:n, None]
    return c["q"][b, h * G:(h + 1) * G].double() @ k.T / 32


def rel_bound(n_tokens):
    """The bound on the error of out over sum p |v| for a sequence of that length."""
    n, nb = min(n_tokens, TILE), -(-n_tokens // TILE)
    return U * (2 + 3 * (nb + 2) + 1 + n + n / 4 + (2 * nb + 1) / 4 + 2)


def emulate(c, Hkv, G, weights):
    """out in 64 bits with the weights of a block, relative to its maximum and times 2^13, as `weights(p)` makes them
    ([G, tokens] in, the same out); and sum p |v|."""
    B, D = len(LENS), c["q"].shape[2]
    out, mag = (torch.zeros(B, Hkv * G, D, dtype=torch.float64) for _ in range(2))
    for b, n in enumerate(LENS):
        for h in range(Hkv):
            x = log2_scores(c, b, h, G)
            m = x.amax(1, keepdim=True)
            num, absolute, total = 0.0, 0.0, 0.0
            for j in range(0, n, TILE):
                xb, vb = x[:, j:j + TILE], c["v"][b, h, j:min(n, j + TILE)].double() * float(c["vs"][b, h, j // TILE])
                mb = xb.amax(1, keepdim=True)
                f = torch.exp2(mb - m)
                p = torch.exp2(xb - mb)
                num = num + f * (weights(p * 8192) / 8192 @ vb)
                absolute = absolute + f * (p @ vb.abs())
                total = total + f * p.sum(1, keepdim=True)
            rows = slice(h * G, (h + 1) * G)
            out[b, rows], mag[b, rows] = num / total, absolute / total
    return out, mag


def two_parts(p):
    """High and low fp16 part of an fp32 number, added up."""
    p = p.float()
    hi = p.half()
    return hi.double() + (p - hi.float()).half().double()


def one_part(p):
    return p.float().half().double()


def low_part_of_the_next_head(p):
    p = p.float()
    hi = p.half()
    return hi.double() + (p - hi.float()).half().double().roll(1, 0)


def low_part_of_half_the_tokens(p):
    p = p.float()
    hi = p.half()
    lo = (p - hi.float()).half().double()
    lo[:, 1::2] = 0
    return hi.double() + lo
