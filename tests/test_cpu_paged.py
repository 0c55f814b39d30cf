"""The paged cache on the host: who has which page, the formulas, the model on top of it and what is refused."""
import random

import pytest
import torch

from elfa_b200 import ops
from elfa_b200.config import Config
from elfa_b200.eval import Generator
from elfa_b200.models.gpt import GPTModel
from elfa_b200.runtime.paged_cache import OutOfPages, PagedCache

from paged_cases import attend64, make


def _model(kv_heads=4, positions=True, **kw):
    cfg = Config.from_file("configs/bench/smoke_cpu.yaml")
    cfg.model.num_kv_heads = kv_heads
    cfg.bench.learned_positions = positions
    for k, v in kw.items():
        setattr(cfg.model, k, v)
    return GPTModel(cfg, device=torch.device("cpu")).eval()


@pytest.mark.parametrize("window,sinks", [(None, 0), (5, 0), (16, 3), (1, 0), (40, 20)])
def test_formula(window, sinks):
    c = make([(3, 70), (0, 9), (1, 1), (33, 40)], 6, 2, 8, 16, device="cpu", dtype=torch.float64)
    c["table"][0, 1] = -1
    ref, _ = attend64(c, window, sinks)
    o = ops.paged_attention(c["q"], c["pages"], c["table"], c["q_start"], c["kv_len"], window=window, sinks=sinks)
    assert torch.allclose(o, ref, atol=1e-12)


def test_bookkeeping_against_lists():
    """Random adds, appends, forks, frees and compactions: every sequence reads back what a list of its tokens holds, pages are counted right."""
    rng = random.Random(0)
    for window, sinks in ((None, 0), (20, 0), (24, 5)):
        cache = PagedCache(2, 40, 16, 1, 1, torch.float64, "cpu", window, sinks)
        want, fresh = {}, 1.0
        for _ in range(400):
            op = rng.choice(["add", "append", "append", "append", "fork", "free", "compact"])
            if op == "add" and len(want) < 8:
                want[cache.add()] = []
            elif op == "fork" and want and len(want) < 10:
                s = rng.choice(list(want))
                for f in cache.fork(s, rng.choice([1, 2])):
                    want[f] = list(want[s])
            elif op == "free" and want:
                s = rng.choice(list(want))
                cache.free(s)
                del want[s]
            elif op == "compact":
                n = cache.compact()
                assert n == 40 - cache.free_pages and max([p for s in want for p in cache.pages_of(s)], default=-1) < n
            elif op == "append" and want:
                seqs = rng.sample(list(want), rng.randint(1, len(want)))
                new = [rng.choice([0, 1, 1, 3, 17, 40]) for _ in seqs]
                if not sum(new):
                    continue
                state = ([(list(x.pages), x.length) for x in cache._seqs.values()], list(cache._refs), sorted(cache._free))
                try:
                    batch = cache.append(seqs, new)
                except OutOfPages:
                    assert state == ([(list(x.pages), x.length) for x in cache._seqs.values()], list(cache._refs), sorted(cache._free))
                    continue
                assert batch.q_start.tolist() == [sum(new[:i]) for i in range(len(new) + 1)] and batch.max_new == max(new)
                for s, n in zip(seqs, new):
                    want[s] = want[s] + [fresh + j for j in range(n)]
                    fresh += n
                rows = torch.tensor([t for s, n in zip(seqs, new) for t in want[s][len(want[s]) - n:]], dtype=torch.float64).view(-1, 1, 1)
                for layer in range(2):
                    cache.write(layer, rows + layer, -rows, batch)
                assert batch.positions.tolist() == [p for s, n in zip(seqs, new) for p in range(len(want[s]) - n, len(want[s]))]
            for s, tokens in want.items():
                assert cache.length(s) == len(tokens)
                first = 0 if window is None else max(0, len(tokens) - window + 1)
                for p, t in enumerate(tokens):
                    page = cache.pages_of(s)[p // 16]
                    if p >= first or p < sinks:                  # all that a later token can see is there
                        assert page >= 0
                    if page >= 0:
                        assert cache.pool[0, page, 0, 0, p % 16, 0] == t and cache.pool[1, page, 0, 0, p % 16, 0] == t + 1
                        assert cache.pool[1, page, 1, 0, p % 16, 0] == -t
            held = {p for s in want for p in cache.pages_of(s) if p >= 0}
            assert cache.free_pages == 40 - len(held)
            if window is not None:
                assert all(sum(p >= 0 for p in cache.pages_of(s)) <= -(-(window + 40) // 16) + 2 + -(-sinks // 16) for s in want)


@pytest.mark.parametrize("kv_heads,positions", [(4, True), (2, True), (1, False)])
def test_model_equals_the_whole_context(kv_heads, positions):
    """Prompts in pieces, single tokens, sequences that fork and go apart, in any mixture: the logits of the whole context run at once. 2e-4 as for the other cache."""
    m = _model(kv_heads, positions)
    g = torch.Generator().manual_seed(3)
    ids = [torch.randint(0, m.cfg.model.vocab_size, (n,), generator=g) for n in (50, 7, 33)]
    with torch.no_grad():
        full = [m(x[None])[0] for x in ids]
    cache = m.new_paged_cache(20, 16)
    a, b, c = cache.add(), cache.add(), cache.add()
    lo = m.forward_paged(torch.cat([ids[0][:20], ids[2][:1]]), [a, c], [20, 1], cache)
    assert (lo - torch.stack([full[0][19], full[2][0]])).abs().max() < 2e-4
    lo = m.forward_paged(torch.cat([ids[0][20:21], ids[1], ids[2][1:30]]), [a, b, c], [1, 7, 29], cache, all_logits=True)
    assert (lo - torch.cat([full[0][20:21], full[1], full[2][1:30]])).abs().max() < 2e-4
    d, = cache.fork(a)
    other = torch.randint(0, m.cfg.model.vocab_size, (5,), generator=g)
    lo = m.forward_paged(torch.cat([other, ids[0][21:]]), [d, a], [5, 29], cache)
    with torch.no_grad():
        want = m(torch.cat([ids[0][:21], other])[None])[0, -1]
    assert (lo[0] - want).abs().max() < 2e-4 and (lo[1] - full[0][-1]).abs().max() < 2e-4
    cache.free(a)
    cache.free(b)
    cache.compact()
    lo = m.forward_paged(ids[2][30:], [c], [3], cache, all_logits=True)
    assert (lo - full[2][30:]).abs().max() < 2e-4
    lo = m.forward_paged(torch.cat([other[:1], ids[1][:1]]), [d, c], [1, 1], cache)
    with torch.no_grad():
        want = m(torch.cat([ids[0][:21], other, other[:1]])[None])[0, -1]
    assert (lo[0] - want).abs().max() < 2e-4


def test_window_frees_pages_and_keeps_the_result():
    """A windowed cache against an unbounded one that masks the same keys: layer outputs agree while pages go back."""
    g = torch.Generator().manual_seed(0)
    small, big = PagedCache(1, 8, 16, 2, 8, torch.float64, "cpu", 20, 3), PagedCache(1, 40, 16, 2, 8, torch.float64, "cpu")
    s, t = small.add(), big.add()
    for step in range(60):
        n = [1, 1, 5, 17][step % 4]
        q, k, v = (torch.randn(n, h, 8, generator=g, dtype=torch.float64) for h in (4, 2, 2))
        outs = []
        for cache, seq in ((small, s), (big, t)):
            batch = cache.append([seq], [n])
            cache.write(0, k, v, batch)
            outs.append(ops.paged_attention(q, cache.pool[0], batch.table, batch.q_start, batch.kv_len, window=20, sinks=3))
        assert torch.allclose(outs[0], outs[1], atol=1e-12)
    assert small.length(s) == 360 and small.free_pages >= 8 - 4


def test_generating_many():
    m = _model(2)
    gen = Generator(m)
    prompts = [[5, 6, 7], [9], list(range(40))]
    out = gen.generate_batch(prompts, 6, temperature=0.0, samples=2, page_size=16, chunk=16)
    for p, o in zip(prompts, out):
        assert o[0] == o[1] == gen.generate_greedy(p, 6)
    a = gen.generate_batch(prompts, 6, temperature=1.0, top_k=50, top_p=0.95, samples=3, seed=1, page_size=16)
    assert a == gen.generate_batch(prompts, 6, temperature=1.0, top_k=50, top_p=0.95, samples=3, seed=1, page_size=16)
    assert all(len(s) == len(p) + 6 and s[:len(p)] == p for p, o in zip(prompts, a) for s in o) and len({tuple(s) for s in a[0]}) > 1
    eos = a[0][0][3]
    b = gen.generate_batch(prompts, 6, temperature=1.0, top_k=50, top_p=0.95, samples=3, seed=1, page_size=16, eos_id=eos)
    assert b[0][0] == a[0][0][:4]
    full = gen.generate_batch([[1] * 125], 30, temperature=0.0)[0][0]           # the learned positions end at 128
    assert len(full) == 128
    long = Generator(_model(2, positions=False)).generate_batch([[3, 4]], 200, temperature=0.0, window=24, sinks=2, page_size=16)[0][0]
    assert len(long) == 202
    with pytest.raises(ValueError, match="positions"):
        gen.generate_batch([[1] * 129], 3)
    assert gen.generate_batch([], 3) == []


def test_command_line():
    from elfa_b200 import cli
    a = cli.build_parser().parse_args(["generate", "--checkpoint", "x", "--samples", "3", "--top-k", "5", "--window", "100", "--sinks", "4"])
    assert (a.samples, a.top_k, a.min_p, a.window, a.sinks, a.top_p) == (3, 5, 0.0, 100, 4, 0.9)


def test_sampling_on_the_host():
    x = torch.tensor([[0.0, 3.0, 1.0, 3.0], [float("-inf")] * 4, [float("nan"), 1.0, 0.5, float("-inf")]])
    assert ops.sample(x, None, 0.0).tolist() == [1, -1, 1]
    noise = torch.tensor([[1e-9, 1.0, 1.0, 0.9]] * 3)
    assert ops.sample(x, noise, 1.0).tolist() == [0, -1, 1]
    assert ops.sample(x, noise, 1.0, top_k=2).tolist() == [3, -1, 1]
    assert ops.sample(x, noise, 1.0, top_k=1).tolist() == [1, -1, 1]
    assert ops.sample(x, noise, 1.0, top_p=0.9).tolist() == [3, -1, 1]
    assert ops.sample(x, noise, 1.0, min_p=0.5).tolist() == [3, -1, 1]
    assert ops.sample(x, noise, torch.tensor([0.0, 1.0, 1.0]), torch.tensor([0, 0, 2], dtype=torch.int32)).tolist() == [1, -1, 1]


def test_refusals():
    c = make([(2, 20)], 4, 2, 8, 16, device="cpu", dtype=torch.float32)
    call = lambda **k: ops.paged_attention(**{**{n: c[n] for n in ("q", "pages", "table", "q_start", "kv_len")}, **k})        # noqa: E731
    for bad, kind in ((dict(q=c["q"][:, :3]), ValueError), (dict(pages=c["pages"][0]), ValueError), (dict(table=c["table"][0]), ValueError),
                      (dict(q_start=c["q_start"][:1]), ValueError), (dict(kv_len=c["kv_len"].long()), TypeError), (dict(q=c["q"].double()), TypeError),
                      (dict(window=0), ValueError), (dict(sinks=-1), ValueError), (dict(q=c["q"].clone().requires_grad_(True)), RuntimeError)):
        with pytest.raises(kind, match="paged_attention"):
            call(**bad)
    with pytest.raises(ValueError, match="without a page"):
        ops.paged_write(c["k"], c["v"], c["pages"], torch.full_like(c["table"], -1), c["q_start"], c["kv_len"])
    with pytest.raises(ValueError, match="paged_write"):
        ops.paged_write(c["k"][:, :1], c["v"][:, :1], c["pages"], c["table"], c["q_start"], c["kv_len"])
    for a, b in (([0], [9]), ([-1], [0]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([0], [1, 2])):
        with pytest.raises(ValueError, match="copy_pages"):
            ops.copy_pages(c["pages"], a, b)
    with pytest.raises(ValueError, match="page_size"):
        PagedCache(1, 4, 24, 1, 8)
    cache = PagedCache(1, 2, 16, 1, 8, torch.float32, "cpu")
    s = cache.add()
    with pytest.raises(OutOfPages):
        cache.append([s], [33])
    for seqs, new in (([s, s], [1, 1]), ([s], [0]), ([s], [-1]), ([], []), ([s], [1, 2])):
        with pytest.raises(ValueError):
            cache.append(seqs, new)
    m = _model()
    with pytest.raises(ValueError, match="ids must hold"):
        m.forward_paged(torch.zeros(3, dtype=torch.int64), [0], [2], m.new_paged_cache(4))
    with pytest.raises(ValueError, match="layers"):
        m.forward_paged(torch.zeros(2, dtype=torch.int64), [s], [2], PagedCache(9, 4, 16, 4, 32, torch.float32, "cpu"))
