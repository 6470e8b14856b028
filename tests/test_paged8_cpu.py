"""The 8-bit cache without a GPU: what is refused before anything runs, the C entry points' argument checks, and the
layout of their parameter blocks."""
import ctypes
import subprocess
import tempfile
from pathlib import Path

import pytest
import torch

from kvskip_b200 import cabi
from kvskip_b200 import kvskip as K
from kvskip_b200.cache import PagedKV8

ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture(scope="module")
def lib():
    from kvskip_b200 import build
    build.build_lib()
    lib = ctypes.CDLL(str(build.LIB))
    lib.kvskip_last_error.restype = ctypes.c_char_p
    lib.kvskip_decode8_work_bytes.restype = ctypes.c_int64
    return lib


def test_parameter_blocks_match_the_header():
    names = {"kvskip_decode8_params": cabi.Decode8Params, "kvskip_write8_params": cabi.Write8Params,
             "kvskip_pages_params": cabi.PagesParams}
    body = "".join(f'printf("%zu ", sizeof({n}));' for n in names)
    for n, c in names.items():
        for f, _ in c._fields_:
            body += f'printf("%zu ", offsetof({n}, {f}));'
    src = f'#include <stdio.h>\n#include <stddef.h>\n#include "kvskip_b200.h"\nint main(){{{body}return 0;}}\n'
    with tempfile.TemporaryDirectory() as d:
        c = Path(d) / "s.c"
        c.write_text(src)
        subprocess.run(["/usr/bin/gcc", "-I", str(ROOT / "include"), str(c), "-o", str(Path(d) / "s")], check=True)
        out = subprocess.run([str(Path(d) / "s")], capture_output=True, text=True, check=True).stdout.split()
    want = [ctypes.sizeof(c) for c in names.values()] + [getattr(c, f).offset for c in names.values() for f, _ in c._fields_]
    assert [int(x) for x in out] == want


def _decode_params(**kw):
    p = cabi.Decode8Params()
    base = dict(q=4096, k=4096, v=4096, k_scale=4096, v_scale=4096, out=4096, lse=4096, work=4096, q_sb=512, q_sh=128,
                k_sb=65536, k_sh=8192, k_st=128, v_sb=65536, v_sh=8192, v_st=128, kind=0, B=1, Hq=32, Hkv=8, D=128,
                T=100, nb=2, lens=4096)
    for n, x in {**base, **kw}.items():
        setattr(p, n, x)
    return p


@pytest.mark.parametrize("change,text", [
    (dict(D=96), b"head dim"), (dict(kind=2), b"kind"), (dict(B=0), b"bad B"), (dict(Hq=30), b"bad B"),
    (dict(Hq=17 * 8), b"at most 16"), (dict(Hkv=1 << 21, Hq=1 << 21), b"2^20"), (dict(T=0, nb=0), b"bad B"), (dict(q=0), b"required"), (dict(work=0), b"required"),
    (dict(nb=3), b"nb must be"), (dict(block_idx=4096), b"go together"), (dict(blk_max=4096), b"go together"),
    (dict(page_table=4096, max_pages=1, num_pages=9), b"page table"), (dict(page_table=4096, max_pages=2), b"page table"),
    (dict(page_table=4096, max_pages=2, num_pages=9, lens=0), b"needs lens"), (dict(q=4100), b"8-byte"),
    (dict(q_sh=130), b"8-byte"), (dict(k=4104), b"16-byte"), (dict(v_st=136), b"16"), (dict(work=4100), b"misaligned"),
    (dict(B=1 << 20, T=1 << 20, nb=1 << 14), b"2^29")])
def test_decode8_entry_refuses(lib, change, text):
    assert lib.kvskip_launch_decode8(ctypes.byref(_decode_params(**change)), None) < 0
    assert text in lib.kvskip_last_error()


def test_null_blocks_and_sizes(lib):
    for n in ("decode8", "write8", "extend_pages", "release_pages"):
        assert getattr(lib, f"kvskip_launch_{n}")(None, None) == -1 and b"null" in lib.kvskip_last_error()
    size = lambda **kw: lib.kvskip_decode8_work_bytes(ctypes.byref(_decode_params(**kw)))  # noqa: E731
    assert size(B=0) == 0 and size(nb=0) == 0 and size(block_idx=4096) == 0
    assert size(Hq=128, nb=4000) > size(nb=4000) > size() > 0


@pytest.mark.parametrize("change,text", [
    (dict(D=32), b"head dim"), (dict(kind=7), b"kind"), (dict(inner=0), b"bad n"), (dict(blocks=0), b"bad n"),
    (dict(slots=0), b"required"), (dict(k_new=4104), b"16-byte"), (dict(vn_sh=100), b"16-byte"), (dict(k=4100), b"8-byte"),
    (dict(v_st=132), b"8-byte"), (dict(Hkv=70000), b"grid")])
def test_write8_entry_refuses(lib, change, text):
    p = cabi.Write8Params()
    base = dict(k_new=4096, v_new=4096, kn_si=1024, kn_sh=128, vn_si=1024, vn_sh=128, n=4, inner=4, slots=4096, k=4096,
                v=4096, k_sb=65536, k_sh=8192, k_st=128, v_sb=65536, v_sh=8192, v_st=128, k_scale=4096, v_scale=4096,
                kind=0, Hkv=8, D=128, blocks=1, tokens=64, num_blocks=5)
    for n, x in {**base, **change}.items():
        setattr(p, n, x)
    assert lib.kvskip_launch_write8(ctypes.byref(p), None) < 0
    assert text in lib.kvskip_last_error()


@pytest.mark.parametrize("fn,change,text", [
    ("extend_pages", dict(lens=0), b"required"), ("extend_pages", dict(new_=0), b"required"),
    ("extend_pages", dict(slots=0), b"required"), ("extend_pages", dict(B=0), b">= 1"),
    ("extend_pages", dict(per_row=3), b"per_row"), ("extend_pages", dict(n_tokens=-1), b"n_tokens"),
    ("extend_pages", dict(max_pages=(1 << 20) + 1), b"2^26"),
    ("release_pages", dict(num_free=1 << 30), b"2^30"), ("release_pages", dict(done=0), b"done"),
    ("release_pages", dict(free_pages=0), b"required")])
def test_pages_entries_refuse(lib, fn, change, text):
    p = cabi.PagesParams()
    base = dict(lens=4096, new_=4096, done=4096, table=4096, free_pages=4096, n_free=4096, lens_out=4096,
                n_free_out=4096, slots=4096, positions=4096, granted=4096, n_tokens=4, B=2, max_pages=4, num_free=9)
    for n, x in {**base, **change}.items():
        setattr(p, n, x)
    assert getattr(lib, f"kvskip_launch_{fn}")(ctypes.byref(p), None) < 0
    assert text in lib.kvskip_last_error()


_APART = dict(lens=0x10000, new_=0x20000, done=0x30000, table=0x40000, free_pages=0x50000, n_free=0x60000,
              lens_out=0x70000, n_free_out=0x80000, slots=0x90000, positions=0xa0000, granted=0xb0000, n_tokens=9, B=7,
              max_pages=4, num_free=9)


@pytest.mark.parametrize("fn,change,text", [
    ("extend_pages", dict(lens_out=0x20000), b"lens_out and new"), ("extend_pages", dict(lens_out=0x10004), b"lens_out and lens"),
    ("extend_pages", dict(lens_out=0x10000, n_free_out=0x10000), b"lens_out and n_free_out"),
    ("extend_pages", dict(n_free_out=0x10018), b"n_free_out and lens"), ("extend_pages", dict(table=0x50000 - 4), b"table and free_pages"),
    ("extend_pages", dict(slots=0xa0000 - 64), b"slots and positions"), ("extend_pages", dict(granted=0x20000 + 27), b"granted and new"),
    ("release_pages", dict(lens_out=0x50000 + 32), b"lens_out and free_pages"), ("release_pages", dict(done=0x70000), b"lens_out and done"),
    ("release_pages", dict(free_pages=0x40000 + 108), b"free_pages and table"), ("release_pages", dict(n_free_out=0x10000), b"n_free_out and lens")])
def test_pages_entries_refuse_outputs_in_inputs(lib, fn, change, text):
    """The CTAs of one launch read all requests, and any of them may be the one that writes first."""
    p = cabi.PagesParams()
    for n, x in {**_APART, **change}.items():
        setattr(p, n, x)
    assert getattr(lib, f"kvskip_launch_{fn}")(ctypes.byref(p), None) == -1
    assert text in lib.kvskip_last_error() and b"overlap" in lib.kvskip_last_error()


def test_an_empty_slot_list_overlaps_nothing(lib):
    """Refused for what comes next: the zero-sized lists point into `new`, which does not matter."""
    p = cabi.PagesParams()
    for n, x in {**_APART, "slots": 0x20004, "positions": 0x20004, "n_tokens": 0, "granted": 0x20001}.items():
        setattr(p, n, x)
    assert lib.kvskip_launch_extend_pages(ctypes.byref(p), None) == -1
    assert b"granted and new overlap" in lib.kvskip_last_error()


@pytest.mark.parametrize("change,text", [
    (dict(v=0x10000), b"same memory"), (dict(v_scale=0x30000), b"same memory"), (dict(vs_sb=0), b"stride of 0"),
    (dict(k_sh=0), b"stride of 0"), (dict(ks_sh=0), b"stride of 0"), (dict(v_st=0), b"stride of 0"),
    (dict(blocks=5, tokens=300, vs_st=0), b"stride of 0")])
def test_write8_entry_refuses_shared_memory(lib, change, text):
    """K and V, the heads and the blocks are written by different warps at the same time."""
    p = cabi.Write8Params()
    base = dict(k_new=0x50000, v_new=0x60000, kn_si=1024, kn_sh=128, vn_si=1024, vn_sh=128, n=4, inner=4, slots=0x70000,
                k=0x10000, v=0x20000, k_sb=65536, k_sh=8192, k_st=128, v_sb=65536, v_sh=8192, v_st=128, k_scale=0x30000,
                v_scale=0x40000, ks_sb=8, ks_sh=1, ks_st=1, vs_sb=8, vs_sh=1, vs_st=1, kind=0, Hkv=8, D=128, blocks=1,
                tokens=64, num_blocks=10)
    for n, x in {**base, **change}.items():
        setattr(p, n, x)
    assert lib.kvskip_launch_write8(ctypes.byref(p), None) == -1
    assert text in lib.kvskip_last_error()


def test_front_end_refuses_cpu_tensors():
    k = torch.zeros(3, 2, 64, 64, dtype=torch.float8_e4m3fn)
    s = torch.ones(3, 2)
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.decode8(torch.zeros(1, 8, 64, dtype=torch.bfloat16), k, k, s, s, 1.0, lens=i, page_table=i[None])
    x = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.write8(x, x, torch.zeros(1, dtype=torch.int64), k, k.clone(), s, s.clone())
    with pytest.raises(RuntimeError, match="CUDA"):
        K.extend_pages(i, i, i[None], i, i, n_tokens=1)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.release_pages(i.bool(), i, i[None], i, i)


def test_front_end_argument_errors():
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="n_tokens"):
        K.extend_pages(i, i, i[None], i, i)
    with pytest.raises(ValueError, match="n_tokens"):
        K.extend_pages(i, i, i[None], i, i, n_tokens=1, per_row=1)
    with pytest.raises(ValueError, match="per_row"):
        K.extend_pages(i, i, i[None], i, i, per_row=0)
    with pytest.raises(ValueError, match="int8"):
        PagedKV8(1, 1, 1, 64, 64, "cpu", dtype=torch.uint8)
    with pytest.raises(ValueError, match="head dim"):
        PagedKV8(1, 1, 1, 96, 64, "cpu")
    with pytest.raises(ValueError, match="at least 1"):
        PagedKV8(0, 1, 1, 64, 64, "cpu")
    x = torch.zeros(1, 1, 64)
    for bad in (0, -1):
        with pytest.raises(ValueError, match="max_len"):
            K.decode8(x, x, x, x, x, 1.0, max_len=bad)


def test_a_replayed_step_says_what_it_granted(monkeypatch):
    """`granted` and `positions` of the cache are those of the replayed step, whatever was called in between."""
    from kvskip_b200 import cache as C
    from kvskip_b200 import graph as G

    def extend_pages(lens, new, table, free, n_free, *, n_tokens=None, per_row=None, lens_out=None, n_free_out=None,
                     granted_out=None, live_only=False):
        granted = torch.empty(len(lens), dtype=torch.bool) if granted_out is None else granted_out
        n = len(lens) * per_row if per_row else n_tokens
        r = {"slots": torch.zeros(n, dtype=torch.int64), "positions": torch.full((n,), -1, dtype=torch.int32),
             "granted": granted.fill_(True), "lens": lens, "n_free": n_free}
        seen.append((r["granted"], r["positions"]))
        return r

    class Graph:
        def replay(self):           # what the captured launch writes
            seen[at[id(self)]][0].copy_(torch.tensor([True, False]))
            seen[at[id(self)]][1].copy_(torch.tensor([7, -1]))

    class Capture:
        def __init__(self, g, **kw):
            at[id(g)] = len(seen)

        def __enter__(self):
            pass

        def __exit__(self, *a):
            return False

    seen, at = [], {}
    monkeypatch.setattr(C.K, "extend_pages", extend_pages)
    monkeypatch.setattr(torch.cuda, "CUDAGraph", Graph)
    monkeypatch.setattr(torch.cuda, "graph", Capture)
    cache = PagedKV8(4, 2, 1, 64, 128, "cpu")
    steps = [G.StepGraph(lambda: cache.extend(per_row=1), [cache], eager=0) for _ in range(2)]
    for g in [steps[0], steps[1], steps[0], steps[0]]:
        g.step()
        assert cache.granted.tolist() == [True, False] and cache.positions.tolist() == [7, -1]
        cache.extend(torch.tensor([3, 0], dtype=torch.int32), n_tokens=3)
        assert cache.granted.tolist() == [True, True] and cache.positions.tolist() == [-1] * 3
    assert steps[0].captures == steps[1].captures == 1


def test_status_codes_say_what_happened():
    for code, text in ((0x300, "page table"), (0x301, "page table"), (0x302, "slot is outside"), (0x303, "two runs")):
        e = K.DeviceWaitError(code, "write8")
        assert text in str(e) and hex(code) in str(e) and "wait" not in str(e) and e.code == code
    for code in (0x200, 0x308, 0x501, 0x700, 0x741):
        assert "wait gave up" in str(K.DeviceWaitError(code, "x"))


def test_debug_check_of_the_slot_list():
    K._check_runs(torch.tensor([5, 6, 7, -1, 64, 65, 128, -1, -1, 200]))
    K._check_runs(torch.tensor([[62, 63], [64, 65]]))
    K._check_runs(torch.tensor([], dtype=torch.int64))
    for bad in ([5, 5], [5, 7], [5, 64, 6], [7, -1, 8], [6, 5]):
        with pytest.raises(ValueError, match="next to each other"):
            K._check_runs(torch.tensor(bad))
