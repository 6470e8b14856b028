"""The 8-bit attention against 64 bits on inputs whose scores are exact, within bounds that weights of 11 bits break (see
`accuracy8.py`, and `test_accuracy8_cpu.py` for what the bounds tell)."""
import pytest
import torch

from kvskip_b200 import kvskip as K
from tests import accuracy8 as A
from tests import cache8_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _paged(c):
    """The same cache as a pool of pages under a table far wider than the lengths: the general form of the launch."""
    B, Hkv, T, D = c["k"].shape
    nb = c["nb"]
    d = {"table": torch.full((B, 3000), -1, dtype=torch.int32)}
    d["table"][:, :nb] = torch.arange(B * nb).view(B, nb)
    for n in ("k", "v"):
        x = torch.zeros(B, Hkv, nb * A.TILE, D, dtype=torch.uint8)
        x[:, :, :T] = c[n].view(torch.uint8)
        d[n] = x.view(B, Hkv, nb, A.TILE, D).transpose(1, 2).reshape(B * nb, Hkv, A.TILE, D).contiguous().view(c[n].dtype)
        d[n + "s"] = c[n + "s"].transpose(1, 2).reshape(B * nb, Hkv).contiguous()
    return {**c, **d}


@pytest.mark.parametrize("form", ["contiguous", "wide table"])
@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("qtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hkv,G,D", [(2, 4, 128), (3, 3, 64), (1, 1, 128), (2, 8, 128), (2, 5, 64), (1, 16, 128), (2, 12, 64)])
def test_decode8_keeps_the_weights_to_22_bits(Hkv, G, D, qtype, kind, form):
    c = A.inputs(Hkv, G, D, kind, qtype, seed=G * D + Hkv)
    f = lambda t: t.float() if kind == "e4m3" else t  # noqa: E731
    ref = R.decode_f64(c["q"], f(c["k"]), f(c["v"]), c["ks"], c["vs"], A.SCALE, A.LENS)
    d = {n: t.to(DEV) for n, t in (_paged(c) if form == "wide table" else c).items() if isinstance(t, torch.Tensor)}
    lens = torch.tensor(A.LENS, dtype=torch.int32, device=DEV)
    r = K.decode8(d["q"], d["k"], d["v"], d["ks"], d["vs"], A.SCALE, lens=lens, page_table=d.get("table"), stats=True, out_f32=True)
    o32, lse = r["out_f32"].double().cpu(), r["lse"].double().cpu()
    bm, bs = (r[n][..., :c["nb"]].double().cpu() for n in ("blk_max", "blk_sum"))
    for b, n in enumerate(A.LENS):
        rel, few = A.rel_bound(n), min(n, A.TILE)
        assert ((o32[b] - ref["out"][b]).abs() <= rel * ref["mag"][b]).all(), float(((o32[b] - ref["out"][b]).abs() / ref["mag"][b]).max())
        # lse: the logarithm to u of its value (8 bits at most), the sums' errors as in the bound, products and additions
        assert ((lse[b] - ref["lse"][b]).abs() <= A.U * (8 + ref["lse"][b].abs() + 3 * (c["nb"] + 2) + few / 4)).all()
        seen = torch.isfinite(ref["blk_max"][b])
        assert torch.equal(torch.isfinite(bm[b]), seen)
        assert ((bm[b] - ref["blk_max"][b])[seen].abs() <= A.U / 2 * ref["blk_max"][b][seen].abs()).all()
        assert ((bs[b] - ref["blk_sum"][b])[seen].abs() <= A.U * (1 + few / 4) * ref["blk_sum"][b][seen]).all()
    half = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[qtype]
    assert ((r["out"].double().cpu() - o32).abs() <= half * o32.abs() + 2.0 ** -25).all()
