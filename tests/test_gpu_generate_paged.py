"""The model on a paged cache, bf16 on the device."""
import pytest
import torch

from elfa_b200 import native
from elfa_b200.config import Config
from elfa_b200.eval import Generator
from elfa_b200.models.gpt import GPTModel

pytestmark = pytest.mark.gpu


def _model(kv_heads, positions=True):
    cfg = Config.from_file("configs/bench/gpt350m_zero1.yaml")
    m = cfg.model
    m.num_layers, m.hidden_dim, m.intermediate_dim, m.num_heads, m.num_kv_heads, m.head_dim, m.vocab_size, m.max_seq_len = 3, 512, 1024, 8, kv_heads, 64, 2048, 1024
    cfg.data.seq_len, cfg.bench.learned_positions = 1024, positions
    return GPTModel(cfg, device=torch.device("cuda")).eval()


@pytest.mark.parametrize("kv_heads", [8, 2])
def test_model_equals_the_whole_context(cuda_device, kv_heads):
    """bf16 activations, the whole context by another attention kernel: each of 3 layers rounds a residual stream of size about 1 a few times (2^-8 each), and the
    logits are sums of 512 products of it: a twentieth of their size holds with room (the whole context in fp32 against bf16 differs by a fiftieth)."""
    m = _model(kv_heads)
    g = torch.Generator().manual_seed(3)
    ids = [torch.randint(0, 2048, (n,), generator=g).cuda() for n in (700, 7, 333)]
    with torch.no_grad():
        full = [m(x[None])[0].float() for x in ids]
    cache = m.new_paged_cache(40, 32)
    a, b, c = cache.add(), cache.add(), cache.add()

    def near(got, want):
        return (got.float() - want).abs().max() < 0.05 * want.abs().max()
    lo = m.forward_paged(torch.cat([ids[0][:500], ids[2][:1]]), [a, c], [500, 1], cache)
    assert near(lo, torch.stack([full[0][499], full[2][0]]))
    lo = m.forward_paged(torch.cat([ids[0][500:501], ids[1], ids[2][1:300]]), [a, b, c], [1, 7, 299], cache, all_logits=True)
    assert near(lo, torch.cat([full[0][500:501], full[1], full[2][1:300]]))
    d, e = cache.fork(a, 2)
    for t in range(501, 540):
        lo = m.forward_paged(torch.stack([ids[0][t], ids[0][t]]), [a, e], [1, 1], cache)
        assert near(lo, full[0][t].expand(2, -1))                 # not the same bits: the line of work is cut through them in different places
    cache.free(a)
    cache.free(b)
    cache.compact()
    lo = m.forward_paged(torch.cat([ids[0][501:700], ids[2][300:]]), [d, c], [199, 33], cache)
    assert near(lo, torch.stack([full[0][-1], full[2][-1]]))
    native.check_status()


def test_generating_many(cuda_device):
    gen = Generator(_model(2))
    prompts = [[5, 6, 7], [9], list(range(700))]
    a = gen.generate_batch(prompts, 20, temperature=1.0, top_k=50, top_p=0.95, samples=4, seed=1, chunk=300)
    assert a == gen.generate_batch(prompts, 20, temperature=1.0, top_k=50, top_p=0.95, samples=4, seed=1, chunk=300)
    assert all(len(s) == len(p) + 20 and s[:len(p)] == p for p, o in zip(prompts, a) for s in o) and len({tuple(s) for s in a[2]}) > 1
    greedy = gen.generate_batch([prompts[2]], 8, temperature=0.0, samples=2)[0]
    assert greedy[0][:701] == greedy[1][:701]                     # drawn from the same row of logits
    native.check_status()


def test_window_keeps_the_cache_small(cuda_device):
    m = _model(2, positions=False)
    cache = m.new_paged_cache(14, 32, window=200, sinks=4)
    s = cache.add()
    g = torch.Generator().manual_seed(0)
    for n in [150] * 10 + [1] * 50:
        lo = m.forward_paged(torch.randint(0, 2048, (n,), generator=g).cuda(), [s], [n], cache)
    assert cache.length(s) == 1550 and torch.isfinite(lo).all()
    native.check_status()


@pytest.mark.parametrize("step", [0, 1, 5])
def test_what_kernels_record_is_raised(cuda_device, monkeypatch, step):
    """A table that names pages outside the pool, in the prompt or in one of the steps: an error, not tokens drawn from what was left."""
    from elfa_b200.runtime.paged_cache import PagedCache
    batch, calls = PagedCache._batch, []

    def broken(self, seqs, new):
        b = batch(self, seqs, new)
        if len(calls) == step:
            b.table.add_(1000)
        calls.append(new)
        return b
    gen = Generator(_model(2))
    native.status()
    monkeypatch.setattr(PagedCache, "_batch", broken)
    with pytest.raises(native.NativeError, match="paged cache"):
        gen.generate_batch([[5, 6, 7]], 7, temperature=0.0, samples=2)
    assert len(calls) == 7 if step else len(calls) == 1            # the prompt's is known before anything is drawn from it
    monkeypatch.undo()
    assert len(gen.generate_batch([[5, 6, 7]], 7, temperature=0.0, samples=2)[0][1]) == 10


@pytest.mark.parametrize("paged", [True, False])
def test_ids_of_other_types_and_places(cuda_device, paged):
    """Narrower whole numbers are taken for what they are; ids on the host and ids that are no whole numbers are refused before a kernel reads them."""
    m = _model(2)
    ids = torch.arange(40, 140)

    def call(x):
        if not paged:
            return m(x[None])
        cache = m.new_paged_cache(8, 32)
        return m.forward_paged(x, [cache.add()], [100], cache)
    with torch.no_grad():
        want = call(ids.cuda())
        for kind in (torch.int32, torch.int16, torch.uint8):
            assert torch.equal(call(ids.to(kind).cuda()), want)
        for bad in (ids, ids.int(), ids.cuda().float(), ids.cuda() > 50):
            with pytest.raises((ValueError, TypeError)):
                call(bad)
    native.check_status()
