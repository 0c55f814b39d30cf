"""Paged cache at the edges of what it takes, on the device."""
import pytest
import torch

from elfa_b200 import native, ops
from elfa_b200.runtime.paged_cache import PagedCache

from paged_cases import attend64, close, make

pytestmark = pytest.mark.gpu


def _run(c, **kw):
    return ops.paged_attention(c["q"], c["pages"], c["table"], c["q_start"], c["kv_len"], **kw)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("step", [0.0, 0.05])
def test_blocks_that_follow_each_other(cuda_device, hd, step):
    """Items of 24 blocks: the probabilities of one are written where the product of the block before has just read its own, and, with keys that grow, again when a row's
    maximum has moved. The same bits every time."""
    c = make([(128, 3000), (140, 140)], 4, 2, hd, 64, seed=hd)
    for b, kv in enumerate(c["kv_len"].tolist()):
        pos = torch.arange(kv, device=cuda_device)
        at = (c["table"][b, pos // 64].long(), 0, slice(None), pos % 64)
        c["pages"][at] = (c["pages"][at].float() * (0.5 + step * (pos // 128))[:, None, None]).bfloat16()
    ref, mag = attend64(c)
    outs = [_run(c, max_new=140) for _ in range(8)]
    assert close(outs[0], ref, mag) and all(torch.equal(o, outs[0]) for o in outs)
    assert native.status() == 0


@pytest.mark.parametrize("starts", [[0, 3, 0, 3], [0, 6, 2, 8], [0, 9, 3, 8], [-4, 2, 3, 8], [5, 2, 3, 8]])
@pytest.mark.parametrize("new,H", [(3, 2), (3, 64), (70, 8)])
def test_rows_that_several_sequences_claim(cuda_device, starts, new, H):
    """Few rows per sequence and many: recorded, and nothing outside is touched."""
    c = make([(new, 300), (new, 90), (new, 200)], H, 2, 64, 16)
    scale = c["q"].shape[0] // 8
    c["q_start"] = torch.tensor([x * scale for x in starts], dtype=torch.int32, device=cuda_device)
    before = c["pages"].clone()
    for _ in range(2):
        _run(c)
        assert native.status() == native.ST_BAD_PAGE
    assert torch.equal(c["pages"].view(torch.int16), before.view(torch.int16))


def test_more_claimed_rows_than_32_bits_of_units(cuda_device):
    """Every second of 1024 sequences claims all rows. Their units are 3 x 2^32 and 512 (256-row tiles, blocks of 128 keys): counted in 32 bits they would stand in a line
    that ends inside the first item, whose parts would be looked for behind the scratch."""
    T, H, Hkv, kv, other = 8192, 32, 8, 3149888, 3084416

    def units(n):
        return Hkv * sum(-(-(n - T + (t + 1) * 64) // 128) for t in range(T // 64))
    assert 511 * units(kv) + units(other) == 3 * 2 ** 32 + 512
    q = torch.zeros(T, H, 64, dtype=torch.bfloat16, device=cuda_device)
    pages = torch.zeros(1, 2, Hkv, 256, 64, dtype=torch.bfloat16, device=cuda_device)
    table = torch.zeros(1024, -(-kv // 256), dtype=torch.int32, device=cuda_device)
    start = torch.zeros(1025, dtype=torch.int32, device=cuda_device)
    start[1::2] = T
    lens = torch.full((1024,), kv, dtype=torch.int32, device=cuda_device)
    lens[0] = other
    assert ops.paged_attention(q, pages, table, start, lens).shape == (T, H * 64)
    assert native.status() == native.ST_BAD_PAGE


def test_writing_for_more_sequences_than_a_launch_of_the_attention_takes(cuda_device):
    lens = [(1 + i % 3 if i % 7 else 0, 3 + i % 50) for i in range(2500)]
    c = make(lens, 4, 2, 32, 16)
    want = c["pages"].clone()
    seq = torch.tensor([b for b, (n, _) in enumerate(lens) for _ in range(n)], device=cuda_device)
    pos = torch.tensor([p for n, kv in lens for p in range(kv - n, kv)], device=cuda_device)
    ids = c["table"][seq, pos // 16].long()
    want[ids, 0, :, pos % 16], want[ids, 1, :, pos % 16] = c["k"], c["v"]
    ops.paged_write(c["k"], c["v"], c["pages"], c["table"], c["q_start"], c["kv_len"])
    assert native.status() == 0 and torch.equal(c["pages"].view(torch.int16), want.view(torch.int16))


def test_a_step_of_many_sequences(cuda_device):
    """A prompt, 1100 forks of it, and a step of all of them: copied pages, written tokens and attention."""
    cache = PagedCache(1, 1300, 16, 1, 64, device=cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(0)
    root, q, k, v = cache.add(), *(torch.randn(20 + 1100, h, 64, generator=g, device=cuda_device).bfloat16() for h in (2, 1, 1))
    batch = cache.append([root], [20])
    cache.write(0, k[:20], v[:20], batch)
    seqs = [root] + cache.fork(root, 1099)
    batch = cache.append(seqs, [1] * 1100)
    cache.write(0, k[20:], v[20:], batch)
    o = cache.attend(0, q[20:], batch).view(1100, 2, 64).double()
    s = torch.cat([torch.einsum("nhd,kd->nhk", q[20:].double(), k[:20, 0].double()), torch.einsum("nhd,nd->nh", q[20:].double(), k[20:, 0].double())[..., None]], 2) / 8
    p = torch.softmax(s, -1)

    def mix(vals):
        return torch.einsum("nhk,kd->nhd", p[..., :20], vals[:20, 0]) + p[..., 20:] * vals[20:, 0][:, None]
    assert native.status() == 0 and close(o, mix(v.double()), mix(v.double().abs()))


@pytest.mark.parametrize("lens,H,Hkv,hd", [([(1, 60), (1, 33)], 4, 2, 64), ([(1, 2000)], 2, 2, 64), ([(1, 5000), (3, 900), (1, 1)], 8, 2, 128), ([(70, 300), (50, 90)], 8, 2, 64),
                                           ([(1 + i % 3, 3 + i % 50) for i in range(1100)], 2, 1, 32)])
@pytest.mark.parametrize("front,back", [(0, 3), (5, 0), (2, 40)])
def test_rows_of_no_sequence(cuda_device, lens, H, Hkv, hd, front, back):
    """Rows in front of the first sequence's and behind the last one's are zeros as on the host, and recorded; all forms of the attention."""
    c = make(lens, H, Hkv, hd, 16)
    ref, mag = attend64(c)
    new = max(n for n, _ in lens)
    n = c["q"].shape[0]
    d = {**c, "q": torch.cat([torch.ones(front, H, hd, device=cuda_device).bfloat16(), c["q"], torch.ones(back, H, hd, device=cuda_device).bfloat16()]),
         "q_start": c["q_start"] + front}
    torch.full((n + front + back, H * hd), float("nan"), dtype=torch.bfloat16, device=cuda_device)       # what the result's memory held before
    o = _run(d, max_new=new)
    assert native.status() == native.ST_BAD_PAGE
    assert close(o[front:front + n], ref, mag) and not o[:front].any() and not o[front + n:].any()
    assert close(_run(c, max_new=new), ref, mag) and native.status() == 0


def test_no_sequence_has_a_row(cuda_device):
    for new, H in ((1, 4), (200, 4)):
        c = make([(new, 300), (0, 20)], H, 2, 64, 16)
        torch.full((new, H * 64), float("nan"), dtype=torch.bfloat16, device=cuda_device)
        o = _run({**c, "q_start": torch.zeros_like(c["q_start"])})
        assert native.status() == native.ST_BAD_PAGE and not o.any()


@pytest.mark.parametrize("change", [dict(kv_len=[5000, 50, 20]), dict(kv_len=[113, 50, 20]), dict(kv_len=[3, 50, 20]), dict(kv_len=[-9, 50, 20]), dict(q_start=[-2, 4, 5, 7]),
                                    dict(q_start=[0, 4, 5, 9])])
def test_lengths_that_do_not_fit_write_nothing(cuda_device, change):
    """Tokens of such a sequence have no place: they must not land on those of others. The other sequences' are written."""
    c = make([(4, 100), (1, 50), (2, 20)], 4, 2, 64, 16, unused=0.0)
    for name, v in change.items():
        c[name] = torch.tensor(v, dtype=torch.int32, device=cuda_device)
    want = c["pages"].clone()
    st, kv = c["q_start"].tolist(), c["kv_len"].tolist()
    for b in range(3):
        n = st[b + 1] - st[b]
        if st[b] < 0 or st[b + 1] > 7 or not n <= kv[b] <= 112:
            continue
        for i in range(n):
            p, r = divmod(kv[b] - n + i, 16)
            want[c["table"][b, p].long(), 0, :, r], want[c["table"][b, p].long(), 1, :, r] = c["k"][st[b] + i], c["v"][st[b] + i]
    ops.paged_write(c["k"], c["v"], c["pages"], c["table"], c["q_start"], c["kv_len"])
    assert native.status() == native.ST_BAD_PAGE
    assert torch.equal(c["pages"], want)


@pytest.mark.parametrize("lens,H,Hkv,hd", [([(1, 60), (2, 33)], 4, 2, 64), ([(1, 4000)], 2, 2, 64), ([(2, 5000), (3, 900)], 8, 2, 128), ([(70, 300), (50, 90)], 8, 2, 64),
                                           ([(40, 3000)], 8, 1, 128)])
@pytest.mark.parametrize("value", [0.0, float("inf")])
def test_rows_that_see_only_scores_of_minus_infinity(cuda_device, lens, H, Hkv, hd, value):
    """The first sequence's rows see keys of minus infinity but for the last one's; zero, whatever the values are, as on the host."""
    c = make(lens, H, Hkv, hd, 16)
    n, kv = lens[0]
    c["q"] = c["q"].abs() + 0.1
    pos = torch.arange(kv if n == 1 else kv - 1, device=cuda_device)
    c["pages"][c["table"][0, pos // 16].long(), 0, :, pos % 16] = float("-inf")
    c["pages"][c["table"][0, 0].long(), 1, 0, 5, 3] += value
    o = _run(c, max_new=max(x for x, _ in lens)).view(-1, H, hd).float()
    host = ops.paged_attention(*(c[x].cpu() for x in ("q", "pages", "table", "q_start", "kv_len"))).view(-1, H, hd).float()
    assert native.status() == 0
    assert not o[:max(n - 1, 1)].any()
    assert torch.equal(o.isnan().cpu(), host.isnan()) and torch.allclose(o.cpu().nan_to_num(), host.nan_to_num(), atol=0.03)


def test_tangents_are_refused(cuda_device):
    """A forward-mode dual among the inputs, which the kernels would drop; inside a level, plain tensors are taken as ever."""
    import torch.autograd.forward_ad as fwd
    c = make([(2, 40)], 4, 2, 64, 16)
    args = ("table", "q_start", "kv_len")
    plain = _run(c)
    with torch.no_grad(), fwd.dual_level():
        def dual(name):
            return {**c, name: fwd.make_dual(c[name], torch.ones_like(c[name]))}
        for name in ("q", "pages"):
            with pytest.raises(RuntimeError, match="paged_attention has no forward"):
                _run(dual(name))
        for name in ("k", "v", "pages"):
            d = dual(name)
            with pytest.raises(RuntimeError, match="paged_write has no forward"):
                ops.paged_write(d["k"], d["v"], d["pages"], *(d[a] for a in args))
        with pytest.raises(RuntimeError, match="copy_pages has no forward"):
            ops.copy_pages(dual("pages")["pages"], [0], [1])
        assert torch.equal(_run(c), plain)
        ops.paged_write(c["k"], c["v"], c["pages"], *(c[a] for a in args))
    assert native.status() == 0


@pytest.mark.parametrize("new,H,Hkv,hd", [(1, 4, 2, 64), (6, 4, 2, 64), (1, 64, 2, 128), (90, 4, 2, 64)])
def test_broadcast_rows(cuda_device, new, H, Hkv, hd):
    """One row of queries, keys and values for all new tokens."""
    c = make([(new, 300)], H, Hkv, hd, 16)
    b = {**c, **{n: c[n][:1].contiguous()[0].expand(new, -1, -1) for n in ("q", "k", "v")}}
    own = {**c, **{n: b[n].contiguous() for n in ("q", "k", "v")}}
    for d in (b, own):
        d["pages"] = c["pages"].clone()
        ops.paged_write(d["k"], d["v"], d["pages"], d["table"], d["q_start"], d["kv_len"])
    assert torch.equal(b["pages"].view(torch.int16), own["pages"].view(torch.int16))
    assert torch.equal(_run(b), _run(own)) and close(_run(b), *attend64(own)) and native.status() == 0


def test_a_cache_that_no_kernel_can_read_is_refused(cuda_device):
    """When it is made, not by the first write, behind which it would count tokens that are not there."""
    for bad in (dict(head_dim=136), dict(head_dim=60), dict(head_dim=0), dict(dtype=torch.float32), dict(dtype=torch.float16)):
        with pytest.raises(ValueError, match="cache on the device"):
            PagedCache(1, 4, 16, 1, **{"head_dim": 64, "device": cuda_device, **bad})
    assert PagedCache(1, 4, 16, 1, 136, torch.float32, "cpu").free_pages == PagedCache(1, 4, 16, 1, 128, device=cuda_device).free_pages == 4
