"""Drawing tokens from logits on the device.

reference: ``src/eval/evaluator.zig:472-529`` (nucleus sampling of one row on the host: softmax in f64, sort, smallest prefix with mass >= top_p).
"""
from __future__ import annotations

from typing import Optional, Union

import torch

from ..native import lib, stream_ptr

_Setting = Union[float, int, torch.Tensor]


def sample_ref(logits: torch.Tensor, noise: Optional[torch.Tensor], temperature: torch.Tensor, top_k: torch.Tensor, top_p: torch.Tensor,
               min_p: torch.Tensor) -> torch.Tensor:
    """:func:`sample` by sorting; the settings one per row. fp32, running sums in fp64 (fp64 throughout for fp64 logits)."""
    x = logits if logits.dtype == torch.float64 else logits.float()
    B, V = x.shape
    x = torch.where(x.isnan(), torch.full_like(x, float("-inf")), x)
    best = x.amax(1, keepdim=True)
    empty = (best == float("-inf")).squeeze(1)
    T = temperature.to(x.dtype)[:, None]
    greedy = ~(T > 0)
    w = torch.exp(torch.where(x == best, torch.zeros_like(x), (x - best) / torch.where(greedy, torch.ones_like(T), T)))
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    rank = torch.arange(V, device=x.device)[None]
    k = top_k[:, None]
    k = torch.where((k > 0) & (k < V), k, torch.full_like(k, V))
    keep = rank < k
    mass = torch.where(keep, ws, torch.zeros_like(ws)).cumsum(1, dtype=torch.float64)
    before = torch.cat([torch.zeros_like(mass[:, :1]), mass[:, :-1]], 1)
    p = top_p[:, None]
    keep = keep & ((p >= 1) | (before < p.double() * mass[:, -1:]) | (rank == 0)) & (ws >= min_p[:, None])
    keep = (keep & ~greedy) | (rank == 0)
    kept = torch.zeros_like(keep).scatter(1, order, keep)
    score = w / noise.to(x.dtype) if noise is not None else w
    score = torch.where(kept & (score >= 0), score, torch.full_like(w, -1.0))
    top = score.amax(1, keepdim=True)
    ids = torch.where(score == top, rank, V).amin(1)
    return torch.where(empty, torch.full_like(ids, -1), torch.where((top.squeeze(1) < 0) | greedy.squeeze(1), order[:, 0], ids))


def _setting(value: _Setting, name: str, dtype: torch.dtype, rows: torch.Size, dev: int, most: int = 0):
    """(tensor or None, number) of a setting that is one number for all rows or a tensor with one per row. ``most``: a bound of whole numbers, whose bits a narrower
    type would drop."""
    if not isinstance(value, torch.Tensor):
        return None, max(0, min(int(value), most)) if most else value
    if value.shape != rows or value.get_device() != dev:
        raise ValueError(f"sample: {name} must be a number or one per row, {list(rows)} on device {dev} (-1: host)")
    if most and value.dtype in (torch.int64, torch.float32, torch.float64):
        value = value.clamp(0, most)
    if value.dtype is not dtype or not value.is_contiguous():
        value = value.to(dtype).contiguous()
    return value, 0


def sample(logits: torch.Tensor, noise: Optional[torch.Tensor], temperature: _Setting = 1.0, top_k: _Setting = 0, top_p: _Setting = 1.0,
           min_p: _Setting = 0.0) -> torch.Tensor:
    """One token id per row of ``logits [B, V]`` (bf16 or fp32, other types are cast to fp32; rows may be strided), int64 ``[B]``. ``noise [B, V]`` fp32: independent
    exponential variates (``torch.empty(B, V).exponential_()``), the only source of chance; it may be ``None`` where ``temperature`` is the number 0.

    With ``w_i = exp((x_i - max x) / temperature)`` and the tokens by falling logit (equal ones by index): the first ``top_k`` (0: all), of those the shortest
    prefix with at least ``top_p`` of their mass (1: all), of those the ones with ``w_i >= min_p``. The token with the largest ``w_i / noise_i`` is returned, which is
    token ``i`` with probability ``w_i / sum w``; the lowest index where two are equal. ``temperature <= 0``: the first largest logit, and so where no token races (``min_p`` above 1, variates that are
    NaN). A NaN counts as -inf; a row
    with nothing above -inf gives -1. Each setting is a number or a tensor with one per row. Runs on the current stream without a host synchronisation."""
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError(f"sample: logits must be [B, V], got {tuple(logits.shape)}")
    B, V = logits.shape
    rows, dev = logits.shape[:1], logits.get_device()
    if noise is None:
        if isinstance(temperature, torch.Tensor) or temperature > 0:
            raise ValueError("sample: noise may be left out where temperature is 0 for all rows")
    elif noise.shape != logits.shape or noise.dtype is not torch.float32 or noise.get_device() != dev:
        raise ValueError(f"sample: noise must be fp32 {tuple(logits.shape)} on {logits.device}")
    t, tn = _setting(temperature, "temperature", torch.float32, rows, dev)
    k, kn = _setting(top_k, "top_k", torch.int32, rows, dev, V)
    p, pn = _setting(top_p, "top_p", torch.float32, rows, dev)
    m, mn = _setting(min_p, "min_p", torch.float32, rows, dev)
    if B == 0:
        return torch.empty(0, dtype=torch.int64, device=logits.device)
    if dev < 0:
        each = [s if s is not None else torch.full((B,), n, dtype=d)
                for s, n, d in ((t, tn, torch.float32), (k, kn, torch.int32), (p, pn, torch.float32), (m, mn, torch.float32))]
        return sample_ref(logits, noise, *each)
    if logits.dtype is not torch.bfloat16 and logits.dtype is not torch.float32:
        logits = logits.float()
    if logits.stride(1) != 1:
        logits = logits.contiguous()
    if noise is not None and noise.stride(1) != 1:
        noise = noise.contiguous()
    out = logits.new_empty(B, dtype=torch.int64)
    pt, pk, pp, pm, pe = (s.data_ptr() if s is not None else None for s in (t, k, p, m, noise))
    lib.call_plain("elfa_sample", logits.data_ptr(), int(logits.dtype is torch.float32), logits.stride(0), pe, noise.stride(0) if pe else 0, pt, pk, pp, pm, tn, kn,
                   pn, mn, out.data_ptr(), B, V, stream_ptr(logits))
    return out
