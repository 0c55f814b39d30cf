"""Attention over pages, writing and copying them, against 64-bit results."""
import math

import pytest
import torch

from elfa_b200 import native, ops

from paged_cases import attend64, close, make

pytestmark = pytest.mark.gpu


def _run(c, **kw):
    return ops.paged_attention(c["q"], c["pages"], c["table"], c["q_start"], c["kv_len"], **kw)


CASES = [
    # lens, H, Hkv, hd, page, window, sinks
    ([(1, 1)], 1, 1, 64, 16, None, 0),
    ([(1, 17), (1, 16), (1, 33)], 4, 2, 32, 16, None, 0),
    ([(1, 129)], 16, 16, 64, 16, None, 0),
    ([(1, 257), (1, 3000), (1, 1), (1, 800)], 8, 2, 128, 64, None, 0),
    ([(1, 5000)], 8, 1, 128, 32, None, 0),
    ([(1, 700), (1, 31), (1, 4100)], 10, 2, 80, 128, None, 0),
    ([(1, 300), (1, 299)], 2, 1, 8, 256, None, 0),
    ([(3, 300), (0, 77), (1, 1), (7, 7), (2, 64)], 8, 2, 64, 16, None, 0),
    ([(5, 1000), (4, 4)], 6, 2, 96, 32, None, 0),
    ([(40, 333), (17, 17), (1, 500)], 4, 4, 128, 64, None, 0),
    ([(130, 130)], 4, 1, 64, 16, None, 0),
    ([(150, 700), (300, 301)], 5, 1, 128, 64, None, 0),
    ([(1, 900), (1, 5), (1, 2000)], 8, 4, 64, 16, 100, 4),
    ([(1, 900), (1, 31)], 8, 4, 128, 32, 1, 0),
    ([(20, 900), (33, 33)], 4, 2, 128, 16, 16, 3),
    ([(200, 600), (7, 333)], 4, 4, 64, 128, 130, 70),
    ([(64, 400)], 2, 2, 64, 64, 50, 400),
    ([(300, 2500)], 16, 2, 128, 16, 700, 17),
    ([(9, 100)], 40, 1, 64, 16, None, 0),
    ([(2, 300)], 128, 1, 128, 16, None, 0),
    ([(1, 100), (2, 33)], 200, 1, 64, 16, None, 0),
    ([(1, 900 + 7 * i) for i in range(20)], 8, 4, 64, 16, None, 0),
    ([(8, 600)], 2, 1, 128, 32, 33, 5),
]


@pytest.mark.parametrize("lens,H,Hkv,hd,page,window,sinks", CASES)
def test_attention(cuda_device, lens, H, Hkv, hd, page, window, sinks):
    """Slots and pages that hold nothing are NaN."""
    c = make(lens, H, Hkv, hd, page, seed=hd + page)
    ref, mag = attend64(c, window, sinks)
    o = _run(c, max_new=max(n for n, _ in lens), window=window, sinks=sinks)
    assert native.status() == 0
    assert o.shape == ref.shape and close(o, ref, mag)
    assert torch.equal(o, _run(c, max_new=max(n for n, _ in lens), window=window, sinks=sinks))          # the same bits again
    assert close(_run(c, window=window, sinks=sinks), ref, mag)                                          # without a bound of the new tokens


LONG_TABLES = [
    # lens, H, Hkv, hd, page, pages that the table has room for, window, sinks: few rows, and items that several CTAs take together
    ([(1, 4000)], 16, 2, 64, 16, 250, None, 0),
    ([(2, 3999)], 16, 2, 128, 64, 63, None, 0),
    ([(1, 3)], 16, 2, 64, 16, 300, None, 0),
    ([(3, 40)], 5, 1, 128, 16, 300, None, 0),
    ([(1, 225)], 4, 1, 8, 32, 200, None, 0),
    ([(2, 2047), (0, 900), (1, 1), (16, 600)], 2, 2, 80, 128, 16, None, 0),
    ([(0, 0), (4, 1030), (1, 33), (0, 0), (2, 2)], 4, 1, 64, 16, 100, None, 0),
    ([(1, 5000), (1, 700), (1, 20), (1, 601)], 8, 2, 128, 16, 400, 600, 4),
    ([(4, 5000), (3, 3)], 8, 2, 64, 16, 400, 2000, 40),
    ([(1, 2500)], 6, 6, 96, 256, 10, 1000, 300),
]


@pytest.mark.parametrize("lens,H,Hkv,hd,page,room,window,sinks", LONG_TABLES)
def test_attention_with_room_in_the_table(cuda_device, lens, H, Hkv, hd, page, room, window, sinks):
    c = make(lens, H, Hkv, hd, page, seed=room)
    table = torch.full((len(lens), room), -1, dtype=torch.int32, device=cuda_device)
    table[:, :c["table"].shape[1]] = c["table"]
    c["table"] = table
    new = max(n for n, _ in lens)
    ref, mag = attend64(c, window, sinks)
    o = _run(c, max_new=new, window=window, sinks=sinks)
    assert native.status() == 0 and close(o, ref, mag)
    assert torch.equal(o, _run(c, max_new=new, window=window, sinks=sinks))
    # a value that is not finite reaches the rows that see it, and a page that is gone takes its keys with it
    kv = lens[0][1]
    if kv > 2 * page:
        at = kv // 2 if window is None else kv - min(window, kv) // 2 - new
        bad = {**c, "pages": c["pages"].clone()}
        bad["pages"][int(table[0, at // page]), 1, 0, at % page] = float("inf")
        o = _run(bad, max_new=new, window=window, sinks=sinks).view(-1, H, hd)
        sees = torch.zeros_like(o, dtype=torch.bool)
        sees[:lens[0][0], :H // Hkv] = True
        assert not torch.isfinite(o[sees]).any()
        assert close(o.masked_fill(sees, 0).view(ref.shape), ref.view(o.shape).masked_fill(sees, 0).view(ref.shape), mag)
        table[0, at // page] = -1
        ref, mag = attend64(c, window, sinks)
        assert close(_run(c, max_new=new, window=window, sinks=sinks), ref, mag)
    assert native.status() == 0


@pytest.mark.parametrize("hd,Hkv", [(64, 3), (128, 2)])
@pytest.mark.parametrize("B", [3, 17, 33, 70])
def test_shares_that_end_anywhere(cuda_device, B, hd, Hkv):
    """Few long sequences among many short ones: the work is cut into equal shares wherever that falls."""
    for step in range(5):
        lens = [(1 + (b + step) % 2, 2 + (b * 37 + step * 11) % 70 if b % 9 else 700 + 331 * step + 17 * b) for b in range(B)]
        c = make(lens, 2 * Hkv, Hkv, hd, 16, seed=B + step)
        ref, mag = attend64(c)
        o = _run(c, max_new=2)
        assert close(o, ref, mag) and torch.equal(o, _run(c, max_new=2))
    assert native.status() == 0


def test_scale_and_strides(cuda_device):
    c = make([(3, 400), (1, 90)], 8, 2, 64, 16)
    ref, mag = attend64(c, scale=0.3)
    assert close(_run(c, max_new=3, scale=0.3), ref, mag)
    odd = torch.empty(4, 8, 65, dtype=torch.bfloat16, device=cuda_device)[:, :, 1:]                      # rows that no kernel can take as they are
    odd.copy_(c["q"])
    base = torch.empty(4 * 8 * 64 + 1, dtype=torch.bfloat16, device=cuda_device)[1:].view(4, 8, 64)
    base.copy_(c["q"])
    for q in (odd, base, c["q"].contiguous()):
        assert close(_run({**c, "q": q}, max_new=3, scale=0.3), ref, mag)
    wide = torch.full((2, 100), -1, dtype=torch.int32, device=cuda_device)
    wide[:, :c["table"].shape[1]] = c["table"]
    assert close(_run({**c, "table": wide[:, :60]}, max_new=3, scale=0.3), ref, mag)


@pytest.mark.parametrize("new", [1, 40])
def test_pages_that_are_not_there(cuda_device, new):
    """Freed pages in front of a window, holes, and a sequence without any page at all."""
    c = make([(new, 500), (new, 90), (new, 200)], 8, 2, 64, 16)
    c["table"][0, 2:20] = -1
    c["table"][1] = -1
    c["table"][2, -1] = -7
    ref, mag = attend64(c)
    o = _run(c, max_new=new)
    assert native.status() == 0 and close(o, ref, mag)
    assert not o[new:2 * new].any() and mag[new:2 * new].sum() == 0


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("new,kv,window", [(4, 300, None), (4, 40, None), (50, 400, None), (300, 600, None), (1, 900, 64), (260, 900, 64)])
def test_what_is_hidden_does_not_reach_a_row(cuda_device, bad, new, kv, window):
    """A later token's key and value and those that left the window are not finite: rows that do not see them are as without, the others are not finite."""
    c = make([(new, kv)], 4, 2, 64, 16)
    ref, mag = attend64(c, window, 0)
    hit = kv - new // 2 - 1 if new > 1 else kv - window - 1
    page = int(c["table"][0, hit // 16])
    c["pages"][page, 1, :, hit % 16] = bad
    o = _run(c, max_new=new, window=window)
    pos = torch.arange(kv - new, kv, device=cuda_device)
    sees = pos >= hit if window is None else (pos >= hit) & (pos < hit + window)
    assert close(o[~sees], ref[~sees], mag[~sees])
    assert not torch.isfinite(o[sees]).any()
    c["pages"][page, 0, :, hit % 16] = bad
    o = _run(c, max_new=new, window=window)
    assert close(o[~sees], ref[~sees], mag[~sees])
    assert not torch.isfinite(o[sees]).any()


def test_many_sequences(cuda_device):
    lens = [(1 + i % 3 if i % 7 else 0, 3 + i % 50) for i in range(1100)]
    c = make(lens, 2, 1, 32, 16)
    ref, mag = attend64(c)
    o = _run(c, max_new=3)
    assert native.status() == 0 and close(o, ref, mag)


def test_offsets_past_32_bits(cuda_device):
    """A pool of 2.3e9 elements whose last pages are the ones in use."""
    P, Hkv, page, hd = 18000, 8, 64, 128
    pages = torch.zeros(P, 2, Hkv, page, hd, dtype=torch.bfloat16, device=cuda_device)
    assert pages.numel() > 2 ** 31
    c = make([(1, 640), (5, 100)], 8, 8, hd, page, unused=0.0, spare=0)
    n = c["pages"].shape[0]
    pages[-n:] = c["pages"]
    big = {**c, "pages": pages, "table": torch.where(c["table"] >= 0, c["table"] + (P - n), c["table"])}
    ref, mag = attend64(c)
    assert close(_run(big, max_new=5), ref, mag)
    ops.paged_write(c["k"], c["v"], big["pages"], big["table"], c["q_start"], c["kv_len"])
    ops.paged_write(c["k"], c["v"], c["pages"], c["table"], c["q_start"], c["kv_len"])
    assert torch.equal(pages[-n:], c["pages"])
    ops.copy_pages(pages, [P - 1], [0])
    assert torch.equal(pages[0], pages[-1]) and native.status() == 0


def test_another_stream(cuda_device):
    c = make([(1, 5000), (3, 700)], 8, 2, 128, 64)
    ref, mag = attend64(c)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        outs = [_run(c, max_new=3) for _ in range(20)]
    here = [_run(c, max_new=3) for _ in range(20)]
    torch.cuda.synchronize()
    assert all(close(o, ref, mag) and torch.equal(o, here[0]) for o in outs + here)


def test_captured_in_a_graph(cuda_device):
    c = make([(1, 900), (1, 3000)], 8, 2, 64, 16)
    _run(c, max_new=1)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = _run(c, max_new=1)
    c["kv_len"].copy_(torch.tensor([40, 2500]))                    # the lengths are read when it runs
    g.replay()
    torch.cuda.synchronize()
    ref, mag = attend64(c)
    assert close(o, ref, mag)


def test_bad_lengths_and_pages_are_recorded(cuda_device):
    """What the host cannot see without waiting: nothing is read or written outside, and the status word says so."""
    c = make([(2, 100), (1, 50)], 4, 2, 64, 16)
    native.status()
    for change in ({"kv_len": torch.tensor([100, 5000])}, {"kv_len": torch.tensor([1, 50])}, {"q_start": torch.tensor([0, 9, 3])},
                   {"q_start": torch.tensor([-4, 2, 3])}, {"table": c["table"] + 1000}):
        d = {**c, **{k: v.to(torch.int32).to(cuda_device) for k, v in change.items()}}
        _run(d, max_new=2)
        assert native.status() == native.ST_BAD_PAGE, change
        before = c["pages"].clone()
        ops.paged_write(c["k"], c["v"], d["pages"], d["table"], d["q_start"], d["kv_len"])
        assert native.status() & native.ST_BAD_PAGE, change
        c["pages"].copy_(before)
    _run(c, max_new=1)                                              # fewer than there are
    assert native.status() == native.ST_BAD_PAGE
    with pytest.raises(native.NativeError, match="paged cache"):
        _run({**c, "table": c["table"] + 1000}, max_new=2)
        native.check_status()


# ------------------------------------------------------------------------------------------------ pages
@pytest.mark.parametrize("lens,Hkv,hd,page", [([(1, 1)], 1, 8, 16), ([(1, 17), (0, 9), (1, 33)], 2, 64, 16), ([(700, 900), (3, 3), (1000, 1000)], 4, 128, 64),
                                              ([(5, 300)], 3, 80, 256)])
def test_write(cuda_device, lens, Hkv, hd, page):
    c = make(lens, 2 * Hkv, Hkv, hd, page)
    want = c["pages"].clone()
    at = 0
    for b, (n, kv) in enumerate(lens):
        for pos in range(kv - n, kv):
            p = int(c["table"][b, pos // page])
            want[p, 0, :, pos % page], want[p, 1, :, pos % page] = c["k"][at], c["v"][at]
            at += 1
    ops.paged_write(c["k"], c["v"], c["pages"], c["table"], c["q_start"], c["kv_len"])
    assert native.status() == 0
    assert torch.equal(c["pages"].view(torch.int16), want.view(torch.int16))                             # NaN and all
    ops.paged_write(c["k"].transpose(1, 2).contiguous().transpose(1, 2), c["v"].contiguous(), c["pages"], c["table"], c["q_start"], c["kv_len"])
    assert torch.equal(c["pages"].view(torch.int16), want.view(torch.int16))


def test_write_without_a_page(cuda_device):
    c = make([(3, 40)], 2, 1, 64, 16)
    c["table"][0, 2] = -1
    before = c["pages"].clone()
    native.status()
    ops.paged_write(c["k"], c["v"], c["pages"], c["table"], c["q_start"], c["kv_len"])
    assert native.status() == native.ST_BAD_PAGE and torch.equal(c["pages"].view(torch.int16), before.view(torch.int16))


@pytest.mark.parametrize("L,P,n,shape", [(1, 4, 1, (1, 16, 8)), (3, 50, 25, (2, 16, 80)), (2, 1500, 700, (1, 32, 64)), (0, 9, 2, (4, 128, 128))])
def test_copy(cuda_device, L, P, n, shape):
    """L 0: the pages of one layer, without the first dimension. 700 pairs are more than one launch carries."""
    pages = torch.randn(*([L] if L else []), P, 2, *shape, device=cuda_device).bfloat16()
    order = torch.randperm(P, generator=torch.Generator().manual_seed(P)).tolist()
    src, dst = order[:n], order[n:2 * n]
    src[-1] = src[0]                                                # one page may be copied to several places
    want = pages.clone()
    at = (slice(None),) if L else ()
    want[at + (torch.tensor(dst),)] = pages[at + (torch.tensor(src),)]
    ops.copy_pages(pages, src, dst)
    assert torch.equal(pages, want)
    for a, b in (([0], [P]), ([-1], [0]), ([0, 1], [2, 2]), ([0, 1], [1, 2])):
        with pytest.raises(native.NativeError, match="copy_pages"):
            ops.copy_pages(pages, a, b)
    ops.copy_pages(pages, [], [])
    assert torch.equal(pages, want)


def test_refusals(cuda_device):
    c = make([(2, 100)], 4, 2, 64, 16)
    with pytest.raises(TypeError, match="bf16"):
        _run({**c, "q": c["q"].float(), "pages": c["pages"].float()})
    with pytest.raises(ValueError, match="contiguous"):
        _run({**c, "pages": c["pages"].transpose(2, 3).contiguous().transpose(2, 3)})
    with pytest.raises(ValueError, match="multiple of 2"):
        _run({**c, "q": c["q"][:, :3]})
    with pytest.raises(ValueError, match="device"):
        _run({**c, "table": c["table"].cpu()})
    with pytest.raises(TypeError, match="int32"):
        _run({**c, "kv_len": c["kv_len"].long()})
    with pytest.raises(ValueError, match="tokens and head dimensions"):
        _run({**c, "pages": torch.zeros(4, 2, 2, 24, 64, dtype=torch.bfloat16, device=cuda_device)})
    with pytest.raises(ValueError, match="window"):
        _run(c, window=0)
    with pytest.raises(ValueError, match="max_new"):
        _run(c, max_new=0)
    with pytest.raises(RuntimeError, match="no backward"):
        _run({**c, "q": c["q"].detach().clone().requires_grad_(True)})
    assert _run({**c, "q": c["q"][:0], "q_start": torch.zeros(2, dtype=torch.int32, device=cuda_device)}).shape == (0, 256)
    assert math.isfinite(float(_run(c).float().sum()))
