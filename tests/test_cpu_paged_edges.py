"""Paged cache and sampling at the edges of what they take, as far as the host shows it."""
import re
from pathlib import Path

import pytest
import torch

from elfa_b200 import ops
from elfa_b200.config import Config
from elfa_b200.eval import Generator
from elfa_b200.models.gpt import GPTModel
from elfa_b200.runtime.paged_cache import PagedCache

from paged_cases import attend64, make

CSRC = Path(__file__).resolve().parent.parent / "elfa_b200" / "csrc"


def test_tensor_memory_is_touched_behind_a_fence():
    """A thread that has waited for a product may read or write tensor memory behind tcgen05.fence::after_thread_sync only: in the softmax warps' code every wait for S
    or O is followed by the fence before the next access, in the order of the source."""
    text = (CSRC / "paged_prefill.cu").read_text()
    text = re.sub(r"//[^\n]*", "", text[text.index("reg_inc"):text.index("paged_prefill_join_kernel")])
    seen, open_wait = 0, False
    for word in re.findall(r"mbar_wait\(bar\(PB_[SO]FULL|tc_fence_after|tmem_(?:ld|st)\d+", text):
        if word.startswith("mbar"):
            seen, open_wait = seen + 1, True
        elif word == "tc_fence_after":
            open_wait = False
        else:
            assert not open_wait, f"{word} behind a wait without a fence"
    assert seen >= 4


@pytest.mark.parametrize("change", [dict(kv_len=[5000, 50, 20]), dict(kv_len=[3, 50, 20]), dict(kv_len=[-9, 50, 20]), dict(q_start=[-2, 4, 5, 7]), dict(q_start=[0, 4, 5, 9]),
                                    dict(q_start=[0, 4, 5, 6]), dict(q_start=[1, 4, 5, 7]), dict(q_start=[0, 4, 3, 7])])
def test_lengths_that_do_not_fit_write_nothing(change):
    c = make([(4, 100), (1, 50), (2, 20)], 4, 2, 8, 16, device="cpu", dtype=torch.float32, unused=0.0)
    for name, v in change.items():
        c[name] = torch.tensor(v, dtype=torch.int32)
    before = c["pages"].clone()
    with pytest.raises(ValueError, match="paged_write"):
        ops.paged_write(c["k"], c["v"], c["pages"], c["table"], c["q_start"], c["kv_len"])
    assert torch.equal(c["pages"], before)


def test_a_sequence_without_new_tokens_is_not_looked_at():
    c = make([(4, 100), (0, 50)], 4, 2, 8, 16, device="cpu", dtype=torch.float32, unused=0.0)
    c["kv_len"][1] = 9000
    ops.paged_write(c["k"], c["v"], c["pages"], c["table"], c["q_start"], c["kv_len"])
    assert torch.equal(c["pages"][c["table"][0, 6].long(), 0, :, :4], c["k"].transpose(0, 1))


def test_rows_that_see_only_scores_of_minus_infinity():
    """Zero, as the kernels give; a row that sees one finite score too is as without the others, and scores of plus infinity or NaN are no reason for a zero."""
    c = make([(3, 40), (1, 17)], 4, 4, 8, 16, device="cpu", dtype=torch.float64)
    c["q"] = c["q"].abs() + 0.1
    ids = c["table"][0, :3].long()
    c["pages"][ids[:2], 0] = float("-inf")
    c["pages"][ids[2], 0, :, :6] = float("-inf")                   # tokens 0 to 37; 38 and 39 are finite
    o = ops.paged_attention(c["q"], c["pages"], c["table"], c["q_start"], c["kv_len"]).view(4, 4, 8)
    assert not o[0].any() and not o.isnan().any()
    assert torch.allclose(o[1], c["pages"][ids[2], 1, :, 6], atol=1e-12)
    ref, _ = attend64({**c, "q": c["q"][3:], "table": c["table"][1:], "q_start": torch.tensor([0, 1]), "kv_len": c["kv_len"][1:]})
    assert torch.allclose(o[3].view(1, -1), ref, atol=1e-12)
    c["pages"][ids[0], 1, 3, 5] = float("inf")                      # a value that a row with no weight at all sees
    assert torch.equal(ops.paged_attention(c["q"], c["pages"], c["table"], c["q_start"], c["kv_len"])[0], o[0].reshape(-1))
    c["pages"][ids[0], 1, 3, 5] = 0.0
    for bad in (float("inf"), float("nan")):
        c["pages"][ids[0], 0, 0, 3] = bad
        o = ops.paged_attention(c["q"], c["pages"], c["table"], c["q_start"], c["kv_len"]).view(4, 4, 8)
        assert o[:3, 0].isnan().all() and not o[0, 1:].any() and not o[3].isnan().any()


def _model(positions):
    cfg = Config.from_file("configs/bench/smoke_cpu.yaml")
    cfg.model.num_kv_heads, cfg.bench.learned_positions = 2, positions
    return GPTModel(cfg, device=torch.device("cpu")).eval()


@pytest.mark.parametrize("window,sinks,chunk,samples", [(20, 0, 16, 1), (20, 3, 16, 3), (33, 40, 7, 2), (1, 0, 1, 2), (16, 16, 16, 1)])
def test_a_window_bounds_the_pool_of_long_prompts(monkeypatch, window, sinks, chunk, samples):
    """Prompts far longer than the window take the pages that a window, the sinks and a piece of a prompt can hold, and no more; what is generated is what one that reserves
    for the whole prompts gives."""
    m = _model(False)
    asked, make_cache = [], GPTModel.new_paged_cache

    def new_paged_cache(self, pages, *args, **kw):
        asked.append(pages)
        return make_cache(self, pages * room, *args, **kw)
    monkeypatch.setattr(GPTModel, "new_paged_cache", new_paged_cache)
    prompts = [[(7 * i) % 90 for i in range(n)] for n in (600, 5, 333)]
    outs = []
    for room in (1, 8):
        outs.append(Generator(m).generate_batch(prompts, 30, temperature=0.0, samples=samples, window=window, sinks=sinks, page_size=16, chunk=chunk))
    assert outs[0] == outs[1] and all(len(o) == len(p) + 30 for p, s in zip(prompts, outs[0]) for o in s)
    live = -(-(window + sinks + chunk) // 16) + 2
    assert asked[0] <= len(prompts) * (1 + samples) * live < 600 // 16 + 333 // 16 + len(prompts) * samples * live


def test_rows_that_overlap_are_copied():
    """A tensor map wants rows apart: a broadcast query, or rows that begin inside the one before, are copied for the kernels; slices of a fused projection are not."""
    from elfa_b200.ops.paged import _rows
    base = torch.randn(6, 4, 8)
    for t in (base[0].expand(5, 4, 8), base.view(-1).as_strided((5, 4, 8), (8, 8, 1)), base.view(-1).as_strided((3, 4, 8), (24, 8, 1))):
        r = _rows(t, 8)
        assert r.is_contiguous() and r.data_ptr() != t.data_ptr() and torch.equal(r, t)
    for t in (base, base[:, :3], base[::2, 1:], base[:1], base[0].expand(1, 4, 8)):
        assert _rows(t, 8) is t


def test_top_k_beyond_32_bits():
    """Any number of tokens that is more than there are keeps all of them, negative ones too; no bit of it is dropped."""
    x = torch.arange(6.).repeat(4, 1)
    noise = torch.ones(4, 6)
    noise[:, 0] = 1e-9
    for k in (2 ** 32 + 1, 2 ** 40 + 2, 2 ** 31, 6, 10 ** 18, -(2 ** 40) + 3, -1, 0):
        assert ops.sample(x, noise, 1.0, k).tolist() == [0] * 4
        assert ops.sample(x, noise, 1.0, torch.full((4,), k, dtype=torch.int64)).tolist() == [0] * 4
    assert ops.sample(x, noise, 1.0, torch.tensor([1, 5, 6, 2 ** 33 + 1])).tolist() == [5, 5, 0, 0]
    assert ops.sample(x, noise, 1.0, torch.tensor([1, 5, 6, 7], dtype=torch.uint8)).tolist() == [5, 5, 0, 0]
    assert ops.sample(x, noise, 1.0, torch.tensor([1.0, 5.0, 6.0, 1e12])).tolist() == [5, 5, 0, 0]


def test_a_call_that_is_refused_counts_no_token():
    """Caches and ids that do not fit the model, and sequences that are not there: the cache is as it was."""
    m = _model(True)
    at, ids = m.blocks[0].attn, torch.zeros(3, dtype=torch.int64)
    L, Hkv, hd = len(m.blocks), at.n_kv_heads, at.head_dim
    for cache, bad in ((PagedCache(L + 1, 4, 16, Hkv, hd, torch.float32, "cpu"), ids), (PagedCache(L, 4, 16, Hkv * 2, hd, torch.float32, "cpu"), ids),
                       (PagedCache(L, 4, 16, Hkv, hd + 8, torch.float32, "cpu"), ids), (PagedCache(L, 4, 16, Hkv, hd, torch.float64, "cpu"), ids),
                       (m.new_paged_cache(4, 16), ids.float()), (m.new_paged_cache(4, 16), ids[:2]), (m.new_paged_cache(4, 16), ids.to("meta"))):
        s = cache.add()
        with pytest.raises(ValueError):
            m.forward_paged(bad, [s], [3], cache)
        assert cache.length(s) == 0 and cache.free_pages == 4
    cache = m.new_paged_cache(4, 16)
    s = cache.add()
    with pytest.raises(KeyError):
        m.forward_paged(ids, [s, 77], [2, 1], cache)
    assert cache.length(s) == 0 and m.forward_paged(ids.int(), [s], [3], cache).shape[0] == 1
