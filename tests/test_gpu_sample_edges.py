"""Sampling at the edges of what it takes: the device against the host's form of the definition."""
import pytest
import torch

from elfa_b200 import native, ops

pytestmark = pytest.mark.gpu


def _draws(B, V, seed, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(B, V, generator=g, device="cuda") * 2.5).to(dtype)
    return x, torch.empty(B, V, device="cuda").exponential_(generator=g)


def _both(x, noise, *settings):
    host = [s.cpu() if isinstance(s, torch.Tensor) else s for s in settings]
    return ops.sample(x, noise, *settings).tolist(), ops.sample(x.cpu(), noise.cpu(), *host).tolist()


@pytest.mark.parametrize("B,V,dtype", [(1, 1, torch.float32), (4, 1000, torch.bfloat16), (3, 32000, torch.bfloat16), (2, 131072, torch.float32), (200, 9000, torch.float32)])
@pytest.mark.parametrize("k,p", [(0, 1.0), (5, 1.0), (6000, 1.0), (0, 0.7), (40, 0.7), (6000, 0.7), (1, 1.0)])
def test_rows_of_which_nothing_races(cuda_device, B, V, dtype, k, p):
    """min_p above 1 keeps no token, and a variate that is NaN keeps its token out of the race: the first largest logit, of equal ones the first."""
    x, noise = _draws(B, V, V + B, dtype)
    x[:, V // 3] = x[:, V // 2] = x.amax(1)
    first = x.float().cpu().numpy().argmax(1).tolist()                       # of equal ones the first
    nan = torch.full_like(noise, float("nan"))
    for e, m in ((noise, 1.5), (noise, float("inf")), (nan, 0.0), (nan, 0.1)):
        got, want = _both(x, e, 0.8, k, p, m)
        assert got == want == first
    rows = torch.where(torch.arange(B, device=cuda_device) % 2 == 0, 1.5, 0.0)
    got, want = _both(x, noise, 0.8, k, p, rows)
    assert got[::2] == want[::2] == first[::2]
    x[:] = float("-inf")
    assert _both(x, nan, 0.8, k, p, 1.5) == ([-1] * B, [-1] * B)
    assert native.status() == 0


def test_only_what_is_kept_counts(cuda_device):
    """The kept tokens' variates are NaN, those of the others are not."""
    x, noise = _draws(4, 20000, 7)
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    noise.scatter_(1, order[:, :10], float("nan"))
    for k, p, m in ((10, 1.0, 0.0), (10, 0.9, 0.0), (0, 1e-4, 0.0)):
        got, want = _both(x, noise, 1.0, k, p, m)
        assert got == want == order[:, 0].tolist()


@pytest.mark.parametrize("V,dtype", [(1000, torch.float32), (32000, torch.bfloat16), (131072, torch.float32)])
@pytest.mark.parametrize("name", ["temperature", "top_p", "min_p"])
@pytest.mark.parametrize("k", [0, 50, 6000])
def test_settings_that_are_nan(cuda_device, V, dtype, name, k):
    """Every test on a NaN is false: such a row takes its first largest logit, whether the setting is one for all rows or the row's own."""
    x, noise = _draws(6, V, V, dtype)
    s = dict(temperature=0.9, top_k=k, top_p=0.8, min_p=0.01)
    order = ("temperature", "top_k", "top_p", "min_p")
    got, want = _both(x, noise, *({**s, name: float("nan")}[n] for n in order))
    assert got == want == x.float().cpu().numpy().argmax(1).tolist()
    rows = torch.full((6,), s[name], device=cuda_device)
    rows[::2] = float("nan")
    for others in (s, dict(temperature=0.9, top_k=k, top_p=1.0, min_p=0.0)):
        mixed, want = _both(x, noise, *({**others, name: rows}[n] for n in order))
        assert mixed[::2] == want[::2] == got[::2]
    assert mixed[1::2] == ops.sample(x, noise, *({**others, name: s[name]}[n] for n in order)).tolist()[1::2]


def test_top_k_beyond_32_bits(cuda_device):
    x, noise = _draws(4, 3000, 2)
    for k in ([2 ** 32 + 1, 2 ** 40 + 2, 2 ** 31, -(2 ** 40) + 3], [1, 50, 2 ** 33 + 1, 0]):
        rows = torch.tensor(k, device=cuda_device)
        own = [x if 0 < x < 3000 else 0 for x in k]
        want = ops.sample(x, noise, 1.0, torch.tensor(own, dtype=torch.int32, device=cuda_device)).tolist()
        assert ops.sample(x, noise, 1.0, rows).tolist() == want
        assert [ops.sample(x, noise, 1.0, n).tolist()[i] for i, n in enumerate(k)] == want
