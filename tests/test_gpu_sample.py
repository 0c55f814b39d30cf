"""Sampling kernel against the definition in 64 bits. The result is a token: it has to be equal. Where the winner's score is within
2^-20 of the next one, or another token wins when a filter's line is moved by 2^-20, fp32 may choose either, and such rows are left out; more than half of them stay."""
import pytest
import torch

from elfa_b200 import native, ops

pytestmark = pytest.mark.gpu
NEG = float("-inf")


def _draws(B, V, seed, dtype=torch.float32, std=2.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(B, V, generator=g, device="cuda") * std).to(dtype)
    return x, torch.empty(B, V, device="cuda").exponential_(generator=g)


def exact_rows(x, noise, T, k, p, m):
    """(tokens, whether a row is clear of ties) of the definition, one row at a time in fp64."""
    ids, clear = [], []
    for b in range(x.shape[0]):
        v = x[b].double()
        v = torch.where(v.isnan(), torch.full_like(v, NEG), v)
        if v.max() == NEG:
            ids.append(-1), clear.append(True)
            continue
        val, idx = torch.sort(v, descending=True, stable=True)
        if not T > 0:
            ids.append(int(idx[0])), clear.append(True)
            continue
        w = torch.exp(torch.where(val == val[0], torch.zeros_like(val), (val - val[0]) / T))
        n0 = k if 0 < k < len(w) else len(w)
        mass = w[:n0].cumsum(0) / w[:n0].sum()

        def winner(dp, dm):                      # with the lines of top-p and min-p moved a little: (token, whether nothing comes near it)
            n = min(n0, 1 + int((mass[:-1] < p + dp).sum())) if p < 1 else n0
            n = min(n, max(1, int((w >= m * (1 + dm)).sum())))
            s = w[:n] / noise[b, idx[:n]].double()
            top = torch.topk(s, min(2, n)).values
            return int(idx[:n][s == s.max()].min()), n == 1 or bool(top[0] - top[1] >= 2 ** -20 * top[0]) or bool(top[0] == top[1])
        here, eps = winner(0, 0), 2 ** -20
        ids.append(here[0])
        clear.append(here[1] and all(winner(dp, dm)[0] == here[0] for dp in (-eps, eps if p > 0 else 0) for dm in (-eps, eps)))
    return torch.tensor(ids), torch.tensor(clear)


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.7, 50, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.3, 0, 1.0, 0.05), (0.8, 40, 0.9, 0.02), (1.0, 1, 1.0, 0.0), (2.0, 3000, 0.99, 0.0),
            (1.0, 0, 0.0, 0.0), (1.0, 7, 0.5, 0.0), (0.0, 5, 0.5, 0.1), (30.0, 0, 0.5, 0.0), (0.05, 0, 0.999, 0.0), (1.0, 0, 0.3, 1.0), (50.0, 100000, 0.97, 0.9)]


@pytest.mark.parametrize("T,k,p,m", SETTINGS)
@pytest.mark.parametrize("B,V,dtype", [(1, 1, torch.float32), (3, 2, torch.bfloat16), (2, 33, torch.float32), (4, 1000, torch.bfloat16), (3, 32000, torch.bfloat16),
                                       (5, 8192, torch.float32), (2, 50257, torch.float32), (1, 131072, torch.float32), (2, 300001, torch.bfloat16)])
def test_against_the_definition(cuda_device, B, V, dtype, T, k, p, m):
    x, noise = _draws(B, V, V + B, dtype)
    want, clear = exact_rows(x, noise, T, k, p, m)
    got = ops.sample(x, noise, T, k, p, m).cpu()
    assert got.dtype == torch.int64 and clear.float().mean() > 0.5
    assert torch.equal(got[clear], want[clear])
    rows = [torch.full((B,), float(s), device=cuda_device) for s in (T, k, p, m)]
    assert torch.equal(ops.sample(x, noise, *rows).cpu(), got)


def test_settings_of_each_row(cuda_device):
    x, noise = _draws(len(SETTINGS), 5000, 3)
    cols = list(zip(*SETTINGS))
    got = ops.sample(x, noise, torch.tensor(cols[0], device=cuda_device), torch.tensor(cols[1], device=cuda_device, dtype=torch.int32),
                     torch.tensor(cols[2], device=cuda_device), torch.tensor(cols[3], device=cuda_device)).cpu()
    for i, s in enumerate(SETTINGS):
        want, clear = exact_rows(x[i:i + 1], noise[i:i + 1], *s)
        assert not clear[0] or got[i] == want[0]


@pytest.mark.parametrize("V", [7, 3000, 40000, 131072])
def test_equal_logits_go_by_index(cuda_device, V):
    """bf16 logits of a few values: the filters' lines run through groups of equal ones."""
    g = torch.Generator(device="cuda").manual_seed(V)
    x = torch.randint(0, 3, (4, V), generator=g, device="cuda").bfloat16()
    noise = torch.empty(4, V, device="cuda").exponential_(generator=g)
    for s in ((1.0, 5, 1.0, 0.0), (1.0, V // 2, 1.0, 0.0), (1.0, 0, 0.31, 0.0), (0.5, V // 3 + 1, 0.77, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.2)):
        want, clear = exact_rows(x, noise, *s)
        assert torch.equal(ops.sample(x, noise, *s).cpu()[clear], want[clear]), s
    x.fill_(1.5)
    for s in ((1.0, 5, 1.0, 0.0), (1.0, 0, 0.31, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.2)):
        want, clear = exact_rows(x, noise, *s)
        assert torch.equal(ops.sample(x, noise, *s).cpu()[clear], want[clear]), s
    flat = torch.full((1, V), 0.5, device=cuda_device)             # equal scores: the lowest index
    assert int(ops.sample(x[:1], flat)) == 0
    flat[0, 3:] = 0.25
    assert int(ops.sample(x[:1], flat)) == 3


def test_masked_and_odd_values(cuda_device):
    x, noise = _draws(8, 4099, 1)
    low = torch.finfo(torch.bfloat16).min
    x[0, 100:] = NEG
    x[1, 1:] = NEG
    x[2] = NEG                                                      # nothing to draw
    x[3] = float("nan")
    x[4, ::2] = float("nan")
    x[5, 7] = float("inf")
    x[6] = low
    x[6, 4000:] = low / 2
    x[7, :] = torch.where(torch.arange(4099, device=cuda_device) % 5 == 0, x[7], torch.full_like(x[7], low))
    for s in SETTINGS:
        want, clear = exact_rows(x, noise, *s)
        got = ops.sample(x, noise, *s).cpu()
        assert torch.equal(got[clear], want[clear]), s
    assert ops.sample(x, noise).tolist()[2:4] == [-1, -1] and int(ops.sample(x, noise)[5]) == 7
    noise[:] = 0.0                                                  # no race is decided by it, but a token comes out
    assert 0 <= int(ops.sample(x, noise)[0]) < 100


def test_strides_types_and_streams(cuda_device):
    x, noise = _draws(3, 2000, 9)
    want = ops.sample(x, noise, 0.9, 60, 0.95)
    wide = torch.full((3, 2051), 99.0, device=cuda_device)
    wide[:, 5:2005] = x
    assert torch.equal(ops.sample(wide[:, 5:2005], noise, 0.9, 60, 0.95), want)
    assert torch.equal(ops.sample(x.t().contiguous().t(), noise.t().contiguous().t(), 0.9, 60, 0.95), want)
    half = x.bfloat16()
    odd = torch.full((3, 2051), 99.0, device=cuda_device, dtype=torch.bfloat16)
    odd[:, 3:2003] = half
    assert torch.equal(ops.sample(odd[:, 3:2003], noise, 0.9, 60, 0.95), ops.sample(half, noise, 0.9, 60, 0.95))
    assert torch.equal(ops.sample(x.double(), noise, 0.9, 60, 0.95), want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        outs = [ops.sample(x, noise, 0.9, 60, 0.95) for _ in range(10)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    assert ops.sample(x[:0], noise[:0]).shape == (0,)
    assert torch.equal(ops.sample(x, None, 0.0), x.argmax(1))


def test_frequencies(cuda_device):
    """20000 draws of one distribution: each token's count lies within five standard deviations of its share."""
    n, V = 20000, 12
    x = torch.linspace(0, 3, V, device=cuda_device).repeat(n, 1)
    noise = torch.empty(n, V, device=cuda_device).exponential_(generator=torch.Generator(device="cuda").manual_seed(4))
    for k, keep in ((0, V), (4, 4)):
        got = torch.bincount(ops.sample(x, noise, 0.8, k), minlength=V).double().cpu()
        p = torch.softmax(x[0, V - keep:].double() / 0.8, 0).cpu()
        assert not got[:V - keep].any()
        assert ((got[V - keep:] - n * p).abs() <= 5 * (n * p * (1 - p)).sqrt()).all()


def test_refusals(cuda_device):
    x, noise = _draws(2, 100, 0)
    for bad in (lambda: ops.sample(x[0], noise), lambda: ops.sample(x, noise[:1]), lambda: ops.sample(x, noise.double()), lambda: ops.sample(x, None),
                lambda: ops.sample(x, noise.cpu()), lambda: ops.sample(x, noise, torch.ones(3, device=cuda_device)), lambda: ops.sample(x, noise, torch.ones(2))):
        with pytest.raises(ValueError, match="sample"):
            bad()
    assert native.status() == 0


@pytest.mark.parametrize("V,dtype", [(1000, torch.float32), (32000, torch.bfloat16), (131072, torch.float32)])
@pytest.mark.parametrize("p,m", [(1.0, 0.0), (0.9, 0.0), (1.0, 0.02), (0.9, 0.02)])
def test_scores_that_are_nearly_alike(cuda_device, V, dtype, p, m):
    """All kept tokens' scores lie within 5e-5 of each other, the winner's 2e-5 in front: more than fp32 is off (exponents up to 12 are off by 2^-20, weights and quotients by
    2^-22). What the filters leave out has far better ones; tokens about a filter's line are out of the race."""
    B = 12
    x, u = _draws(B, V, V, dtype, std=1.2)
    w = torch.exp(x.double() - x.double().amax(1, keepdim=True))
    order = torch.sort(w, dim=1, descending=True, stable=True)
    mass = torch.zeros_like(w).scatter_(1, order.indices, (order.values.cumsum(1) - order.values) / w.sum(1, keepdim=True))       # in front of a token
    inside, outside = (mass < p - 0.02) & (w >= m * 1.02), (mass > p + 0.02) | (w < m * 0.98)
    if p == 1.0:
        inside, outside = w >= m * 1.02, w < m * 0.98
    score = 1 - 5e-5 * (1 - torch.exp(-u.double()))
    score[~inside] = 0.5
    score[outside] = 3.0
    best = torch.where(inside, torch.rand(B, V, device=cuda_device), -1.0).argmax(1)
    score[torch.arange(B, device=cuda_device), best] = 1 + 2e-5
    assert torch.equal(ops.sample(x, (w / score).float(), 1.0, 0, p, m), best)
    assert native.status() == 0


def test_variates_out_of_range(cuda_device):
    """Scores beyond fp32's largest, below its smallest, and of denormal variates."""
    x, noise = _draws(4, 40000, 5)
    for at, e in ((17, 1e-39), (30000, 0.0)):
        n = noise.clone()
        n[:, at] = e
        assert (ops.sample(x, n) == at).all()
    n = torch.full_like(noise, 3e38)
    n[:, 123] = 2e38
    x[:, 123] = x.amax(1)
    assert (ops.sample(x, n) == 123).all()
