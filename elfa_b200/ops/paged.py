"""Attention over a cache of pages, and moving keys and values into and between them.

A layer's cache is ``pages [P, 2, Hkv, page, hd]`` (keys, then values; ``page`` tokens of 16, 32, 64, 128 or 256), ``table [B, N]`` int32 names the
pages of each sequence in order (negative: not there). A call takes new tokens of all sequences one after the other: those of sequence ``b`` are rows
``q_start[b]`` to ``q_start[b + 1]`` (``q_start [B + 1]`` int32 from 0 to the number of rows), and ``kv_len [B]`` int32 counts its tokens with them. The i-th of
``n`` new tokens stands at ``kv_len - n + i``.

CUDA tensors run the kernels of ``csrc/paged_decode.cu`` and ``csrc/pages.cu``: bf16, on the current stream, nothing is read back; lengths or
page numbers that do not fit are recorded in the device status word (``native.check_status``). CPU tensors run the formula. There is no backward
pass, nor forward mode on CUDA: sequences are generated, not trained, from a cache. :class:`elfa_b200.runtime.paged_cache.PagedCache` keeps pools, tables and lengths.

reference: ``src/eval/evaluator.zig:419-470`` (generation runs the whole context of one sequence again for every token).
"""
from __future__ import annotations

import array
import functools
import math
from typing import Optional, Sequence

import torch
from torch.autograd import forward_ad

from ..native import lib, stream_ptr

PAGE_SIZES = (16, 32, 64, 128, 256)


def paged_attention_ref(q: torch.Tensor, pages: torch.Tensor, table: torch.Tensor, q_start: torch.Tensor, kv_len: torch.Tensor,
                        window: Optional[int] = None, sinks: int = 0, scale: Optional[float] = None) -> torch.Tensor:
    """The formula in fp32 (fp64 for fp64 pages), sequence by sequence."""
    T, H, hd = q.shape
    Hkv, page = pages.shape[2], pages.shape[3]
    acc = torch.float64 if pages.dtype == torch.float64 else torch.float32
    sc = scale if scale is not None else 1.0 / math.sqrt(hd)
    out = torch.zeros(T, H, hd, dtype=acc, device=q.device)
    starts = q_start.tolist()
    for b, kv in enumerate(kv_len.tolist()):
        n = starts[b + 1] - starts[b]
        if n <= 0:
            continue
        key = torch.arange(kv, device=q.device)
        ids = table[b, key // page].long()
        there = (ids >= 0) & (ids < pages.shape[0])
        rows = pages[ids.clamp(0, pages.shape[0] - 1), :, :, key % page].to(acc)             # [kv, 2, Hkv, hd]
        pos = torch.arange(kv - n, kv, device=q.device)[:, None]
        sees = (key <= pos) & there
        if window is not None:
            sees = sees & ((key > pos - window) | (key < sinks))
        qb = q[starts[b]:starts[b + 1]].to(acc).view(n, Hkv, H // Hkv, hd)
        s = torch.einsum("nhrd,khd->hrnk", qb, rows[:, 0]) * sc
        s = s.masked_fill(~sees, float("-inf"))
        nothing = (s == float("-inf")).all(-1, keepdim=True) | ~sees                         # a row that sees nothing, or only scores of -inf: zeros
        p = torch.softmax(s, -1).masked_fill(nothing, 0.0)
        # what a row does not see must not reach it, not even as 0 times infinity
        v = rows[:, 1]
        if bool(torch.isfinite(v).all()):
            o = torch.einsum("hrnk,khd->nhrd", p, v)
        else:
            o = torch.stack([torch.einsum("hrk,khd->hrd", p[:, :, i][..., sees[i]], v[sees[i]]) for i in range(n)])
        out[starts[b]:starts[b + 1]] = o.masked_fill(nothing.all(-1).permute(2, 0, 1)[..., None], 0.0).reshape(n, H, hd)
    return out.reshape(T, H * hd).to(q.dtype)


def _check(pages: torch.Tensor, table: torch.Tensor, q_start: torch.Tensor, kv_len: torch.Tensor, what: str):
    """The shapes ``(P, Hkv, page, hd, B, N)`` of arguments that fit each other. A decoding step is issued in the time that its kernel takes: the tests of
    good arguments are few and cheap."""
    ps, ts = pages.shape, table.shape
    if len(ps) != 5 or ps[1] != 2:
        raise ValueError(f"{what}: pages must be [P, 2, Hkv, page, hd], got {tuple(ps)}")
    if len(ts) != 2 or kv_len.shape != ts[:1] or q_start.shape != (ts[0] + 1,):
        raise ValueError(f"{what}: table [B, N], q_start [B + 1] and kv_len [B] do not fit each other: "
                         f"{tuple(ts)}, {tuple(q_start.shape)}, {tuple(kv_len.shape)}")
    dev = pages.get_device()
    if not table.get_device() == q_start.get_device() == kv_len.get_device() == dev:
        raise ValueError(f"{what}: table, q_start and kv_len must be on the pages' device, {pages.device}")
    if not (table.dtype is q_start.dtype is kv_len.dtype is torch.int32):
        raise TypeError(f"{what}: table, q_start and kv_len must be int32")
    if dev >= 0:
        if pages.dtype is not torch.bfloat16:
            raise TypeError(f"{what}: bf16 required on CUDA, got {pages.dtype}")
        if ps[3] not in PAGE_SIZES or ps[4] % 8 or not 8 <= ps[4] <= 128:
            raise ValueError(f"{what}: pages of {PAGE_SIZES} tokens and head dimensions that are multiples of 8 up to 128, got {ps[3]} and {ps[4]}")
        if not pages.is_contiguous() or pages.data_ptr() % 16:
            raise ValueError(f"{what}: pages must be contiguous and 16-byte aligned")
    return ps[0], ps[2], ps[3], ps[4], ts[0], ts[1]


def _no_tangent(what: str, *tensors: torch.Tensor) -> None:
    """Kernels read addresses: the tangent of a forward-mode dual would be lost without a word."""
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{what} has no forward-mode derivative on CUDA: call it without tangents")


def _rows(t: torch.Tensor, hd: int) -> torch.Tensor:
    """``t [T, heads, hd]`` with packed heads on 16-byte boundaries and rows that do not overlap (a tensor map's must not): itself (a slice of a fused projection
    is), or a copy."""
    st = t.stride()
    if st[2] == 1 and st[1] == hd and st[0] % 8 == 0 and st[0] >= t.shape[1] * hd and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


@functools.lru_cache(maxsize=256)
def _scratch_floats(*sizes: int) -> int:
    return lib.raw("elfa_paged_attention_scratch")(*sizes)


def paged_attention(q: torch.Tensor, pages: torch.Tensor, table: torch.Tensor, q_start: torch.Tensor, kv_len: torch.Tensor,
                    max_new: Optional[int] = None, window: Optional[int] = None, sinks: int = 0, scale: Optional[float] = None) -> torch.Tensor:
    """The new tokens' queries ``q [T, H, hd]`` (rows may be strided) against the pages, which hold the new tokens' keys and values already
    (:func:`paged_write`). A query at position ``p`` sees the keys up to ``p``; with a ``window`` the last ``window`` of them and the first ``sinks``; never those of
    pages that are not there. A row that sees nothing (or only scores of -inf) is zero, and what a row does not see cannot reach it whatever it holds; so is a row that
    no sequence has, which the status word tells of. ``H`` is a
    multiple of ``Hkv``. ``max_new``: an upper bound of the new tokens of one sequence, known to the host; without it the number of rows. Returns ``[T, H * hd]``."""
    P, Hkv, page, hd, B, N = _check(pages, table, q_start, kv_len, "paged_attention")
    qs = q.shape
    if len(qs) != 3 or qs[2] != hd or qs[1] < 1 or qs[1] % Hkv:
        raise ValueError(f"paged_attention: q must be [T, H, {hd}] with H a multiple of {Hkv}, got {tuple(qs)}")
    dev = q.get_device()
    if q.dtype is not pages.dtype or dev != pages.get_device():
        raise TypeError("paged_attention: q and pages differ in type or device")
    if window is not None and window < 1:
        raise ValueError("paged_attention: a window holds at least the token itself")
    if sinks < 0:
        raise ValueError("paged_attention: negative sinks")
    if torch.is_grad_enabled() and (q.requires_grad or pages.requires_grad):
        raise RuntimeError("paged_attention has no backward pass: call it without gradients")
    T, H = qs[0], qs[1]
    if dev < 0:
        return paged_attention_ref(q, pages, table, q_start, kv_len, window, sinks, scale)
    _no_tangent("paged_attention", q, pages)
    out = q.new_empty((T, H * hd))
    if T == 0:
        return out
    if B == 0 or N == 0:
        return out.zero_()
    max_new = T if max_new is None else min(int(max_new), T)
    if max_new < 1:
        raise ValueError("paged_attention: max_new must be positive where there are new tokens")
    q = _rows(q, hd)
    if not (table.is_contiguous() and q_start.is_contiguous() and kv_len.is_contiguous()):
        table, q_start, kv_len = table.contiguous(), q_start.contiguous(), kv_len.contiguous()
    window, sinks = min(window or 0, 1 << 30), min(sinks, 1 << 30)
    n = _scratch_floats(B, N, page, H, Hkv, hd, max_new, window, sinks)
    scratch = q.new_empty(n, dtype=torch.float32) if n else None
    lib.call_plain("elfa_paged_attention", q.data_ptr(), q.stride(0), pages.data_ptr(), table.data_ptr(), q_start.data_ptr(), kv_len.data_ptr(), out.data_ptr(),
                   scratch.data_ptr() if n else None, B, N, P, page, T, H, Hkv, hd, max_new, window, sinks, scale if scale is not None else hd ** -0.5, stream_ptr(q))
    return out


def paged_write(k: torch.Tensor, v: torch.Tensor, pages: torch.Tensor, table: torch.Tensor, q_start: torch.Tensor, kv_len: torch.Tensor) -> None:
    """Writes the new tokens' keys and values ``k, v [T, Hkv, hd]`` (rows may be strided) into their places, in place. Every new token needs a page;
    of a sequence whose lengths do not fit nothing is written."""
    P, Hkv, page, hd, B, N = _check(pages, table, q_start, kv_len, "paged_write")
    ks, dev = k.shape, k.get_device()
    if len(ks) != 3 or ks != v.shape or ks[1] != Hkv or ks[2] != hd:
        raise ValueError(f"paged_write: k and v must be [T, {Hkv}, {hd}], got {tuple(ks)} and {tuple(v.shape)}")
    if not (k.dtype is v.dtype is pages.dtype) or not dev == v.get_device() == pages.get_device():
        raise TypeError("paged_write: k, v and pages differ in type or device")
    if torch.is_grad_enabled() and (k.requires_grad or v.requires_grad or pages.requires_grad):
        raise RuntimeError("paged_write has no backward pass: call it without gradients")
    T = ks[0]
    if T == 0:
        return
    if B == 0 or N == 0:
        raise ValueError("paged_write: new tokens without a sequence or a page")
    if dev < 0:
        starts, lens, places = q_start.tolist(), kv_len.tolist(), []
        if starts[0] != 0 or starts[-1] != T or sorted(starts) != starts:
            raise ValueError(f"paged_write: q_start must rise from 0 to the {T} rows, got {starts}")
        for b, kv in enumerate(lens):
            n = starts[b + 1] - starts[b]
            if n and not n <= kv <= N * page:
                raise ValueError(f"paged_write: sequence {b} of {kv} tokens, {n} of them new, does not fit its table of {N * page}")
            pos = torch.arange(kv - n, kv) if n else torch.empty(0, dtype=torch.int64)
            ids = table[b, pos // page].long()                 # none of a sequence without new tokens
            if bool(((ids < 0) | (ids >= P)).any()):
                raise ValueError("paged_write: a new token without a page")
            places.append((ids, pos % page))
        for b, (ids, at) in enumerate(places):                 # nothing is written where a test fails
            pages[ids, 0, :, at] = k[starts[b]:starts[b + 1]]
            pages[ids, 1, :, at] = v[starts[b]:starts[b + 1]]
        return
    _no_tangent("paged_write", k, v, pages)
    k, v = _rows(k, hd), _rows(v, hd)
    if not (table.is_contiguous() and q_start.is_contiguous() and kv_len.is_contiguous()):
        table, q_start, kv_len = table.contiguous(), q_start.contiguous(), kv_len.contiguous()
    lib.call_plain("elfa_paged_write", k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), pages.data_ptr(), table.data_ptr(), q_start.data_ptr(),
                   kv_len.data_ptr(), B, N, P, page, T, Hkv, hd, stream_ptr(k))


def copy_pages(pages: torch.Tensor, src: Sequence[int], dst: Sequence[int]) -> None:
    """Copies page ``src[i]`` over page ``dst[i]`` for all ``i`` at once, in place: ``pages [P, ...]`` of one layer (5 dimensions) or ``[L, P, ...]`` of all
    (6). The page numbers come from the host, which knows them; they travel with the launch. No page may be written twice, or read and written."""
    if pages.dim() not in (5, 6):
        raise ValueError(f"copy_pages: pages must be [P, 2, Hkv, page, hd] or [L, P, 2, Hkv, page, hd], got {tuple(pages.shape)}")
    if len(src) != len(dst):
        raise ValueError("copy_pages: as many pages to read as to write")
    if not pages.is_contiguous():
        raise ValueError("copy_pages: pages must be contiguous")
    if torch.is_grad_enabled() and pages.requires_grad:
        raise RuntimeError("copy_pages has no backward pass: call it without gradients")
    n = len(src)
    if n == 0:
        return
    P = pages.shape[-5]
    if not pages.is_cuda:
        if min(min(src), min(dst)) < 0 or max(max(src), max(dst)) >= P:
            raise ValueError("copy_pages: a page outside the pool")
        if len(set(dst)) != n or not set(dst).isdisjoint(src):
            raise ValueError("copy_pages: a page is written twice, or both read and written")
        at = (slice(None),) * (pages.dim() - 5)
        pages[at + (torch.tensor(list(dst)),)] = pages[at + (torch.tensor(list(src)),)]
        return
    _no_tangent("copy_pages", pages)
    L = pages.shape[0] if pages.dim() == 6 else 1
    if L == 0:
        return
    size = pages.stride(-5) * pages.element_size()
    a, b = array.array("i", src), array.array("i", dst)
    lib.call_plain("elfa_copy_pages", pages.data_ptr(), P * size, size, L, P, a.buffer_info()[0], b.buffer_info()[0], n, stream_ptr(pages))
