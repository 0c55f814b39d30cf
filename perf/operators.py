"""Generation from a cache of pages: its operators, what they are measured on and their plain forms.

A cache keeps keys and values of all sequences in pages ``[P, 2, Hkv, page, hd]`` (one such tensor per layer, ``[L, P, ...]`` for all of
them); a table ``[B, N]`` names the pages of each sequence in order, -1 where there is none. A call brings new tokens for all sequences, one after
the other (``q_start [B + 1]``), and ``kv_len [B]``, the tokens that a sequence has with them.

* ``attend``: the new tokens' queries against the pages, causally, with a sliding window and first tokens that stay visible (sinks).
* ``write``: the new tokens' keys and values into their pages.
* ``copy``: pages to other places in all layers, what forking and compacting a cache do.
* ``sample``: one token per row of logits with temperature, top-k, top-p and min-p, from given exponential variates.

``listed()`` names the cases, ``draw`` makes more of the same ranges, ``prepare`` builds what a program holds before the call, ``run`` is one
pass, ``exact`` the same result in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False
BF = torch.bfloat16


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # the first steps of one generated sequence: nothing but latency
        dict(name="decode_one", kind="attend", B=1, new=1, kv=129, even=True, lens=0, H=16, Hkv=16, hd=64, page=16, window=0, sinks=0),
        # a step of a batch that is being served, sequences of all lengths, grouped heads
        dict(name="decode_batch", kind="attend", B=48, new=1, kv=8191, even=False, lens=1, H=32, Hkv=8, hd=128, page=64, window=0, sinks=0),
        # endless sequences in a bounded cache: a window and four sinks
        dict(name="decode_window", kind="attend", B=16, new=1, kv=50001, even=False, lens=2, H=16, Hkv=4, hd=64, page=32, window=4096, sinks=4),
        # a few proposed tokens per sequence, checked at once
        dict(name="chunk_few", kind="attend", B=8, new=7, kv=3001, even=False, lens=3, H=16, Hkv=16, hd=128, page=16, window=0, sinks=0),
        # a piece of a long prompt over what the pieces before it left
        dict(name="chunk_prompt", kind="attend", B=1, new=2048, kv=16384, even=True, lens=0, H=32, Hkv=8, hd=128, page=128, window=0, sinks=0),
        # prompts of several users beside running sequences, five query heads per key head, windowed
        dict(name="chunk_ragged", kind="attend", B=6, new=1531, kv=6001, even=False, lens=4, H=40, Hkv=8, hd=128, page=64, window=1024, sinks=16),
        # one new token of each sequence
        dict(name="write_step", kind="write", B=64, new=1, kv=4095, even=False, lens=5, H=32, Hkv=8, hd=128, page=64),
        # prompts of three users
        dict(name="write_prompt", kind="write", B=3, new=8191, kv=9001, even=False, lens=6, H=32, Hkv=8, hd=128, page=16),
        # eight samples of one prompt fork off: their last, half-filled page is copied in each layer
        dict(name="copy_fork", kind="copy", L=24, P=64, n=8, Hkv=16, hd=64, page=16),
        # a cache is compacted: pages move to the front
        dict(name="copy_compact", kind="copy", L=8, P=1000, n=300, Hkv=8, hd=128, page=64),
        # the next token of one sequence, everything switched on
        dict(name="sample_one", kind="sample", B=1, V=32000, dtype="bf16", temperature=0.8, top_k=50, top_p=0.9, min_p=0.02, masked=0, mixed=0),
        # a batch of a wide vocabulary, each row with settings of its own, a tenth of the vocabulary masked
        dict(name="sample_batch", kind="sample", B=96, V=131072, dtype="f32", temperature=1.0, top_k=0, top_p=0.95, min_p=0.0, masked=1, mixed=1),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "write", "copy", "sample", "sample"])
    page = rng.choice([16, 32, 64, 128])
    hd = rng.choice([32, 64, 64, 80, 128, 128])
    if kind == "attend":
        Hkv, rep = rng.choice([(16, 1), (4, 4), (8, 4), (8, 5), (16, 8), (1, 8)])
        c = dict(kind=kind, B=_log(rng, 1, 64), new=rng.choice([1, 1, rng.randint(2, 16), _log(rng, 16, 2048)]), kv=0, even=rng.random() < 0.3,
                 lens=rng.randrange(10 ** 6), H=Hkv * rep, Hkv=Hkv, hd=hd, page=page, window=0, sinks=0)
        c["kv"] = c["new"] + _log(rng, 1, 32768) - 1
        if rng.random() < 0.4:
            c["window"], c["sinks"] = _log(rng, 1, 8192), rng.choice([0, 1, 4, 17, 128])
        while c["B"] > 1 and (_pool_pages(c) * 4 * Hkv * page * hd > 1.2e9 or work(c)["flops"] > 4e11 or work(c)["bytes"] > 8e8):
            c["B"] //= 2
        while work(c)["flops"] > 4e11:
            c["kv"], c["new"] = c["kv"] - c["new"] // 2, c["new"] - c["new"] // 2
        return c
    if kind == "write":
        new = rng.choice([1, _log(rng, 2, 8192)])
        Hkv = rng.choice([1, 4, 8, 16])
        c = dict(kind=kind, B=_log(rng, 1, 64), new=new, kv=new + _log(rng, 1, 4096) - 1, even=rng.random() < 0.3, lens=rng.randrange(10 ** 6),
                 H=Hkv * rng.choice([1, 4]), Hkv=Hkv, hd=hd, page=page)
        while c["B"] > 1 and _pool_pages(c) * 4 * Hkv * page * hd > 3e8:
            c["B"] //= 2
        return c
    if kind == "copy":
        Hkv, L = rng.choice([1, 4, 8, 16]), _log(rng, 1, 32)
        P = max(8, min(_log(rng, 8, 2000), int(2e9 / (4 * L * Hkv * page * hd))))
        return dict(kind=kind, L=L, P=P, n=_log(rng, 1, P // 2), Hkv=Hkv, hd=hd, page=page)
    V = rng.choice([_log(rng, 100, 131072), 8192, 32000, 131072])
    B = max(1, min(_log(rng, 1, 256), 96 * 131072 // V))
    return dict(kind=kind, B=B, V=V, dtype=rng.choice(["bf16", "f32"]), temperature=rng.choice([0.0, 0.3, 0.8, 1.0, 1.7]),
                top_k=rng.choice([0, 0, 1, 40, _log(rng, 2, 20000)]), top_p=rng.choice([1.0, 1.0, 0.5, 0.9, 0.99]),
                min_p=rng.choice([0.0, 0.0, 0.05, 0.001]), masked=rng.choice([0, 0, 1, 2]), mixed=rng.choice([0, 0, 1]))


# ------------------------------------------------------------------------------------------------ inputs
def _lens(c):
    """[(new tokens, tokens with them)] of the sequences; in an uneven batch some bring none."""
    r = random.Random(c["lens"])
    if c["even"]:
        return [(c["new"], c["kv"])] * c["B"]
    out = []
    for i in range(c["B"]):
        n = r.randint(0 if i and c["new"] > 1 else 1, c["new"])
        out.append((n, n + r.randint(0, c["kv"] - c["new"])))
    return out


def _pages_of(c, kv):
    return -(-kv // c["page"])


def _pool_pages(c):
    return sum(_pages_of(c, kv) for _, kv in _lens(c)) + 3


class _Draw:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, *shape, std=1.0, dtype=BF):
        return (torch.randn(*shape, generator=self.g, device="cuda", dtype=torch.float32 if dtype != BF else BF) * std).to(dtype)

    def perm(self, n):
        return torch.randperm(n, generator=self.g, device="cuda")


def _inputs(c, seed):
    """The tensors of a case, from the seed alone (also what ``exact`` starts from)."""
    r = _Draw(seed)
    if c["kind"] in ("attend", "write"):
        lens, H, Hkv, hd, page = _lens(c), c["H"], c["Hkv"], c["hd"], c["page"]
        B, T, P = len(lens), sum(n for n, _ in lens), _pool_pages(c)
        perm = r.perm(P).to(torch.int32)
        table = torch.full((B, max(_pages_of(c, kv) for _, kv in lens)), -1, dtype=torch.int32, device="cuda")
        at = 0
        for b, (_, kv) in enumerate(lens):
            n = _pages_of(c, kv)
            table[b, :n] = perm[at:at + n]
            at += n
        start = [0]
        for n, _ in lens:
            start.append(start[-1] + n)
        i32 = dict(dtype=torch.int32, device="cuda")
        t = dict(pages=r.normal(P, 2, Hkv, page, hd), table=table, q_start=torch.tensor(start, **i32),
                 kv_len=torch.tensor([kv for _, kv in lens], **i32))
        qkv = r.normal(T, H + 2 * Hkv, hd)                            # what the fused projection of a layer gives
        t["q"], t["k"], t["v"] = qkv[:, :H], qkv[:, H:H + Hkv], qkv[:, H + Hkv:]
        return t
    if c["kind"] == "copy":
        order = random.Random(seed).sample(range(c["P"]), 2 * c["n"])
        return dict(pages=r.normal(c["L"], c["P"], 2, c["Hkv"], c["page"], c["hd"]), src=order[:c["n"]], dst=order[c["n"]:])
    B, V = c["B"], c["V"]
    x = torch.randn(B, V, generator=r.g, device="cuda") * 2.5
    x.scatter_add_(1, torch.randint(0, V, (B, 8), generator=r.g, device="cuda"), torch.full((B, 8), 6.0, device="cuda"))   # what the model is sure of
    if c["masked"]:
        low = float("-inf") if c["masked"] == 1 else torch.finfo(BF).min
        hide = torch.rand(B, V, generator=r.g, device="cuda") < 0.1
        x = x.masked_fill(hide, low)
    if c["dtype"] == "bf16":
        x = x.to(BF)
    noise = torch.empty(B, V, device="cuda").exponential_(generator=r.g)
    rows = torch.arange(B, device="cuda")
    par = {}
    for name, kind, other in (("temperature", torch.float32, 0.7), ("top_k", torch.int32, 100), ("top_p", torch.float32, 0.8), ("min_p", torch.float32, 0.1)):
        p = torch.full((B,), c[name], dtype=kind, device="cuda")
        if c["mixed"]:                                                # every second, third, ... row has settings of its own
            p = torch.where(rows % (2 + len(par)) == 1, torch.full_like(p, other), p)
        par[name] = p
    return dict(logits=x, noise=noise, **par)


def prepare(case, seed):
    t = _inputs(case, seed)
    s = dict(c=case, t=t)
    if case["kind"] == "attend":
        s["lens"] = _lens(case)
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    c, t = state["c"], state["t"]
    if own:
        from elfa_b200 import ops
        if c["kind"] == "attend":
            return ops.paged_attention(t["q"], t["pages"], t["table"], t["q_start"], t["kv_len"], max_new=c["new"], window=c["window"] or None,
                                       sinks=c["sinks"])
        if c["kind"] == "write":
            ops.paged_write(t["k"], t["v"], t["pages"], t["table"], t["q_start"], t["kv_len"])
            return t["pages"]
        if c["kind"] == "copy":
            ops.copy_pages(t["pages"], t["src"], t["dst"])
            return t["pages"]
        return ops.sample(t["logits"], t["noise"], t["temperature"], t["top_k"], t["top_p"], t["min_p"])
    return {"attend": _attend, "write": _write, "copy": _copy, "sample": _sample}[c["kind"]](state)


def _seen(c, n, kv):
    """First key of the window of the first new token, and the sinks before it."""
    lo = max(0, kv - n + 1 - c["window"]) if c["window"] else 0
    return min(c["sinks"], lo) if c["window"] else 0, lo


def _attend(state):
    """Sequence by sequence: the keys that any of its new tokens sees, softmax, sum of the values."""
    c, t = state["c"], state["t"]
    H, Hkv, hd, page = c["H"], c["Hkv"], c["hd"], c["page"]
    out = torch.empty(t["q"].shape[0], H * hd, dtype=BF, device="cuda")
    at = 0
    for b, (n, kv) in enumerate(state["lens"]):
        if not n:
            continue
        s, lo = _seen(c, n, kv)
        key = torch.cat([torch.arange(s, device="cuda"), torch.arange(lo, kv, device="cuda")])
        kvs = t["pages"][t["table"][b].long()[key // page], :, :, key % page].float()          # [keys, 2, Hkv, hd]
        k, v = kvs[:, 0].permute(1, 2, 0), kvs[:, 1].permute(1, 0, 2)
        for i in range(0, n, 1024):
            m = min(1024, n - i)
            pos = torch.arange(kv - n + i, kv - n + i + m, device="cuda")[:, None]
            hidden = key[None] > pos
            if c["window"]:
                hidden = hidden | ((key[None] <= pos - c["window"]) & (key[None] >= c["sinks"]))
            q = t["q"][at + i:at + i + m].float().view(m, Hkv, H // Hkv, hd).permute(1, 2, 0, 3).reshape(Hkv, -1, hd)
            x = (torch.matmul(q, k) * hd ** -0.5).view(Hkv, -1, m, key.numel()).masked_fill(hidden, float("-inf"))
            x = torch.exp(x - x.amax(-1, keepdim=True))
            x = (x / x.sum(-1, keepdim=True)).view(Hkv, -1, key.numel())
            out[at + i:at + i + m] = torch.matmul(x, v).view(Hkv, -1, m, hd).permute(2, 0, 1, 3).reshape(m, -1).to(BF)
        at += n
    return out


def _write(state):
    c, t = state["c"], state["t"]
    T = t["k"].shape[0]
    tok = torch.arange(T, device="cuda")
    b = torch.searchsorted(t["q_start"][1:].long(), tok, right=True)
    pos = t["kv_len"].long()[b] - t["q_start"].long()[b + 1] + tok
    pg = t["table"][b, pos // c["page"]].long()
    t["pages"][pg, 0, :, pos % c["page"]] = t["k"]
    t["pages"][pg, 1, :, pos % c["page"]] = t["v"]
    return t["pages"]


def _copy(state):
    t = state["t"]
    src, dst = torch.tensor(t["src"], device="cuda"), torch.tensor(t["dst"], device="cuda")
    t["pages"][:, dst] = t["pages"][:, src]
    return t["pages"]


def _sample(state):
    """All filters keep a prefix of the tokens by falling logit (equal ones by index); the race x / noise is won by token i with its share of the
    probability. Running sums in 64 bits: which token ends the nucleus must not depend on the order of a sum."""
    t = state["t"]
    x = t["logits"].float()
    V = x.shape[1]
    T = t["temperature"][:, None]
    greedy = T <= 0
    best = x.amax(1, keepdim=True)
    d = torch.where(x == best, torch.zeros_like(x), (x - best) / torch.where(greedy, torch.ones_like(T), T))
    w = torch.exp(d)
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    rank = torch.arange(V, device="cuda")
    k = t["top_k"][:, None]
    k = torch.where((k > 0) & (k < V), k, torch.full_like(k, V))
    keep = rank < k
    mass = torch.where(keep, ws, torch.zeros_like(ws)).cumsum(1, dtype=torch.float64)
    before = torch.cat([torch.zeros_like(mass[:, :1]), mass[:, :-1]], 1)
    p = t["top_p"][:, None]
    keep = keep & ((p >= 1) | (before < p.double() * mass[:, -1:]) | (rank == 0)) & (ws >= t["min_p"][:, None])
    keep = keep & (~greedy | (rank == 0))
    kept = torch.zeros_like(keep).scatter(1, order, keep)
    score = torch.where(kept, w / t["noise"], torch.full_like(w, -1.0))
    top = score.amax(1, keepdim=True)
    return torch.where(score == top, torch.arange(V, device="cuda"), V).amin(1)


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    c, t = case, _inputs(case, seed)
    if c["kind"] == "copy":
        out = t["pages"].double() if t["pages"].numel() < 2 ** 31 else None
        if out is None:
            return None
        for a, b in zip(t["src"], t["dst"]):
            out[:, b] = out[:, a]
        return out
    if c["kind"] == "write":
        out, at = t["pages"].double(), 0
        for b, (n, kv) in enumerate(_lens(c)):
            ids = t["table"][b].tolist()
            for pos in range(kv - n, kv):
                if pos == kv - n or pos % c["page"] == 0:            # a run of tokens inside one page
                    m, r = min(c["page"] - pos % c["page"], kv - pos), pos % c["page"]
                    for j, name in enumerate(("k", "v")):
                        out[ids[pos // c["page"]], j, :, r:r + m] = t[name][at:at + m].double().transpose(0, 1)
                    at += m
        return out
    if c["kind"] == "attend":
        H, Hkv, hd, page = c["H"], c["Hkv"], c["hd"], c["page"]
        rep, at = H // Hkv, 0
        out = torch.zeros(t["q"].shape[0], H, hd, dtype=torch.float64, device="cuda")
        for b, (n, kv) in enumerate(_lens(c)):
            if not n:
                continue
            rows = t["pages"][t["table"][b, :_pages_of(c, kv)].long()]                             # [pages, 2, Hkv, page, hd]
            pos = torch.arange(kv - n, kv, device="cuda").view(-1, 1)
            key = torch.arange(kv, device="cuda").view(1, -1)
            sees = key <= pos
            if c["window"]:
                sees &= (key > pos - c["window"]) | (key < c["sinks"])
            for h in range(Hkv):
                k = rows[:, 0, h].reshape(-1, hd)[:kv].double()
                v = rows[:, 1, h].reshape(-1, hd)[:kv].double()
                for i in range(h * rep, (h + 1) * rep):
                    s = t["q"][at:at + n, i].double() @ k.T / math.sqrt(hd)
                    out[at:at + n, i] = torch.softmax(s.masked_fill(~sees, -math.inf), -1) @ v
            at += n
        return out.reshape(-1, H * hd)
    ids = []
    for b in range(c["B"]):
        x = t["logits"][b].double()
        temp, k, p, m = (t[n][b].item() for n in ("temperature", "top_k", "top_p", "min_p"))
        if temp <= 0:
            ids.append(int((x == x.max()).nonzero()[0]))
            continue
        val, idx = torch.sort(x, descending=True, stable=True)
        w = torch.exp((val - val[0]) / temp)
        n = k if 0 < k < c["V"] else c["V"]
        if p < 1:
            mass = w[:n].cumsum(0)
            n = min(n, 1 + int((mass[:-1] < p * mass[-1]).sum()))
        n = min(n, int((w >= m).sum()))
        score = w[:n] / t["noise"][b, idx[:n]].double()
        ids.append(int(idx[:n][score == score.max()].min()))
    return torch.tensor(ids, device="cuda")


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    if c["kind"] == "attend":
        keys = pairs = tokens = 0
        for n, kv in _lens(c):
            if not n:
                continue
            s, lo = _seen(c, n, kv)
            keys += s + kv - lo
            tokens += n
            for pos in range(kv - n, kv):
                first = max(0, pos + 1 - c["window"]) if c["window"] else 0
                pairs += pos + 1 - first + (min(c["sinks"], first) if c["window"] else 0)
        return dict(bytes=2 * c["hd"] * (2 * keys * c["Hkv"] + 2 * tokens * c["H"]), flops=4 * c["hd"] * c["H"] * pairs)
    if c["kind"] == "write":
        return dict(bytes=8 * c["Hkv"] * c["hd"] * sum(n for n, _ in _lens(c)), flops=0)
    if c["kind"] == "copy":
        return dict(bytes=8 * c["L"] * c["n"] * c["Hkv"] * c["page"] * c["hd"], flops=0)
    # every logit; the variates of the tokens that are left are few where a filter is on
    filtered = c["top_k"] > 0 or c["top_p"] < 1 or c["min_p"] > 0 or c["temperature"] <= 0
    return dict(bytes=c["B"] * c["V"] * ((2 if c["dtype"] == "bf16" else 4) + (0 if filtered else 4)), flops=2 * c["B"] * c["V"])
