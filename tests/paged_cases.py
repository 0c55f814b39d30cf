"""Inputs and 64-bit results for the tests of the paged cache."""
import math

import torch

BF = torch.bfloat16


def make(lens, H, Hkv, hd, page, seed=0, device="cuda", dtype=BF, unused=float("nan"), spare=2):
    """Pages in random order, a table and the queries of ``lens`` = [(new, tokens with them)], as slices of a fused projection. Slots that hold no token
    and pages that belong to nobody are filled with ``unused``."""
    g = torch.Generator(device=device).manual_seed(seed)
    counts = [-(-kv // page) for _, kv in lens]
    P, N = sum(counts) + spare, max(max(counts), 1)
    perm = torch.randperm(P, generator=g, device=device).to(torch.int32)
    table = torch.full((len(lens), N), -1, dtype=torch.int32, device=device)
    pages = torch.full((P, 2, Hkv, page, hd), unused, dtype=dtype, device=device)
    at = 0
    for b, (_, kv) in enumerate(lens):
        table[b, :counts[b]] = perm[at:at + counts[b]]
        at += counts[b]
        pos = torch.arange(kv, device=device)
        pages[table[b, pos // page].long(), :, :, pos % page] = torch.randn(kv, 2, Hkv, hd, generator=g, device=device).to(dtype)
    start = torch.tensor([0] + [n for n, _ in lens]).cumsum(0).to(torch.int32).to(device)
    T = int(start[-1])
    qkv = torch.randn(T, H + 2 * Hkv, hd, generator=g, device=device).to(dtype)
    return dict(q=qkv[:, :H], k=qkv[:, H:H + Hkv], v=qkv[:, H + Hkv:], pages=pages, table=table, q_start=start,
                kv_len=torch.tensor([kv for _, kv in lens], dtype=torch.int32, device=device))


def attend64(c, window=None, sinks=0, scale=None):
    """(result, sum of probability times |value|) in fp64, one query head at a time, from the visible keys alone."""
    T, H, hd = c["q"].shape
    Hkv, page = c["pages"].shape[2:4]
    sc = scale if scale is not None else 1 / math.sqrt(hd)
    out = torch.zeros(T, H, hd, dtype=torch.float64, device=c["q"].device)
    mag = torch.zeros_like(out)
    st = c["q_start"].tolist()
    for b, kv in enumerate(c["kv_len"].tolist()):
        for i in range(st[b], st[b + 1]):
            pos = kv - (st[b + 1] - i)
            key = torch.arange(max(pos + 1, 0), device=out.device)
            if window is not None:
                key = key[(key > pos - window) | (key < sinks)]
            ids = c["table"][b, key // page].long()
            key, ids = key[ids >= 0], ids[ids >= 0]
            if not key.numel():
                continue
            rows = c["pages"][ids, :, :, key % page].double().repeat_interleave(H // Hkv, 2)     # [keys, 2, H, hd]
            s = torch.einsum("hd,khd->hk", c["q"][i].double(), rows[:, 0]) * sc
            p = torch.softmax(s, -1)
            out[i] = torch.einsum("hk,khd->hd", p, rows[:, 1])
            mag[i] = torch.einsum("hk,khd->hd", p, rows[:, 1].abs())
    return out.reshape(T, -1), mag.reshape(T, -1)


def close(got, ref, mag):
    """Probabilities are rounded to bf16 (2^-8 of each) and the result once more: 2^-7 of sum p |v|, and a fiftieth of that for the fp32 arithmetic (scores of
    up to 30 with 2^-20 of error change a probability by 3e-5)."""
    return bool(((got.double() - ref).abs() <= 2 ** -7 * 1.02 * mag).all())
