"""Perplexity, long-context sweep, generation and the forward-throughput micro-benchmark.

reference: ``src/eval/evaluator.zig:269-319`` (perplexity = exp of the token-weighted mean loss over
non-shuffled windows of ``seq_len``), ``:321-377`` (sweep over context lengths), ``:419-470`` (greedy and
temperature / top-p generation, which re-runs the whole prefix for every token), ``:472-529``
(nucleus sampling: softmax(logits / T) in f64, sort descending, smallest prefix with mass >= top_p,
sample proportionally inside it), ``:532-590`` (2 warm-up + 10 timed forward passes → tokens/s).
Generation here reuses per-layer state for the EFLA family (constant cost per token) and falls
back to prefix recomputation for the attention family.
"""
from __future__ import annotations

import math
import time
from typing import Dict, List, Optional

import torch

from .. import native, ops
from ..data import BinaryDataset, DataLoader


def sample_top_p(logits: torch.Tensor, temperature: float = 1.0, top_p: float = 0.9,
                 generator: Optional[torch.Generator] = None) -> int:
    """Nucleus sampling of one token id from a 1-D logits vector."""
    if temperature <= 0:
        return int(torch.argmax(logits))
    probs = torch.softmax(logits.double() / temperature, -1)
    sp, si = torch.sort(probs, descending=True)
    cum = torch.cumsum(sp, 0)
    cutoff = int(torch.searchsorted(cum, torch.tensor(top_p, dtype=cum.dtype, device=cum.device)).item()) + 1
    cutoff = max(1, min(cutoff, sp.numel()))
    head = sp[:cutoff] / sp[:cutoff].sum()
    idx = torch.multinomial(head, 1, generator=generator)
    return int(si[idx])


class Evaluator:
    def __init__(self, model, cfg, device):
        self.model, self.cfg, self.device = model, cfg, device

    @torch.no_grad()
    def _loss(self, ids: torch.Tensor, tgt: torch.Tensor) -> float:
        self.model.eval()
        loss = self.model(ids.to(self.device), tgt.to(self.device))
        return float(loss)

    def evaluate_perplexity(self, data_path_or_dataset, seq_len: Optional[int] = None, max_tokens: Optional[int] = None) -> Dict[str, float]:
        ds = BinaryDataset.open(data_path_or_dataset) if isinstance(data_path_or_dataset, str) else data_path_or_dataset
        S = seq_len or self.cfg.data.seq_len
        loader = DataLoader(ds, 1, S, shuffle=False, pin_memory=False)
        tot_loss, tot_tok = 0.0, 0
        for b in loader:
            tot_loss += self._loss(b.input, b.target) * b.num_tokens
            tot_tok += b.num_tokens
            if max_tokens is not None and tot_tok >= max_tokens:
                break
        mean = tot_loss / max(tot_tok, 1)
        return {"loss": mean, "perplexity": math.exp(min(mean, 50.0)), "tokens": tot_tok}

    def evaluate_long_context(self, dataset, lengths: List[int]) -> List[Dict[str, float]]:
        out = []
        for n in lengths:
            if n + 1 > len(dataset):
                break
            r = self.evaluate_perplexity(dataset, seq_len=n, max_tokens=n)
            r["context"] = n
            out.append(r)
        return out


class Generator:
    def __init__(self, model, tokenizer=None, device=None):
        self.model, self.tok = model, tokenizer
        self.device = device or next(model.parameters()).device

    @torch.no_grad()
    def generate_ids(self, prompt_ids: List[int], max_new_tokens: int = 256, temperature: float = 1.0, top_p: float = 0.9,
                     seed: Optional[int] = None, eos_id: Optional[int] = None) -> List[int]:
        self.model.eval()
        gen = None
        if seed is not None:
            gen = torch.Generator(device="cpu").manual_seed(seed)
        ids = list(prompt_ids) or [0]
        stateful = hasattr(self.model, "forward_with_states")
        if stateful and len(ids) + max_new_tokens > getattr(self.model, "max_positions", 1 << 62):
            stateful = False        # learned positions run out: slide a window over the context instead
        states = None
        if stateful:
            logits, states = self.model.forward_with_states(torch.tensor([ids], device=self.device), None)
            last = logits[0, -1]
        max_ctx = self.model.cfg.data.seq_len
        for _ in range(max_new_tokens):
            if not stateful:
                ctx = ids[-max_ctx:]
                last = self.model(torch.tensor([ctx], device=self.device))[0, -1]
            nxt = sample_top_p(last.float().cpu(), temperature, top_p, gen)
            ids.append(nxt)
            if eos_id is not None and nxt == eos_id:
                break
            if stateful:
                logits, states = self.model.forward_with_states(torch.tensor([[nxt]], device=self.device), states)
                last = logits[0, -1]
        return ids

    @torch.no_grad()
    def generate_batch(self, prompts: List[List[int]], max_new_tokens: int = 256, temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0,
                       min_p: float = 0.0, samples: int = 1, seed: Optional[int] = None, eos_id: Optional[int] = None, window: Optional[int] = None,
                       sinks: int = 0, page_size: int = 64, chunk: int = 2048) -> List[List[List[int]]]:
        """``samples`` continuations of each prompt, all at once, from a cache of pages (softmax-attention family): a prompt runs once, in pieces of at most ``chunk``
        tokens, its samples fork off and share its pages, every step brings one token of each unfinished sequence, and tokens are drawn on the device
        (:func:`elfa_b200.ops.sample`). With a ``window`` tokens see the last ``window`` ones and the first ``sinks``, and pages out of sight are used again. Ends a
        sequence behind ``eos_id``, or before the model's positions run out. Raises what kernels have recorded in the device status word. Returns prompt and
        continuation of ``[prompt][sample]``."""
        if not hasattr(self.model, "forward_paged"):
            raise ValueError("generate_batch wants a model with a paged cache (the softmax-attention family)")
        if samples < 1 or chunk < 1:
            raise ValueError("at least one sample, and at least one token in a piece of a prompt")
        self.model.eval()
        dev = self.device
        prompts = [list(p) or [0] for p in prompts]
        limit = self.model.pos_embed.shape[0] if self.model.pos_embed is not None else 1 << 62
        longest = [min(len(p) + max_new_tokens, limit) for p in prompts]
        if any(len(p) > limit for p in prompts):
            raise ValueError(f"a prompt is longer than the model's {limit} positions")
        live = -(-min(max(longest, default=0), (window or limit) + sinks + chunk) // page_size) + 2        # pages of one sequence that are in use
        pages = sum(min(-(-len(p) // page_size), live) + samples * min(-(-n // page_size) - len(p) // page_size + 1, live) for p, n in zip(prompts, longest))
        cache = self.model.new_paged_cache(max(pages, 1), page_size, window, sinks)
        gen = torch.Generator(device=dev)
        if seed is not None:
            gen.manual_seed(seed)
        else:
            gen.seed()
        roots, last = [cache.add() for _ in prompts], [None] * len(prompts)
        done = [0] * len(prompts)
        while any(d < len(p) for d, p in zip(done, prompts)):                     # prompts, up to `chunk` tokens of them in a call
            part, room = [], chunk
            for i, p in enumerate(prompts):
                n = min(len(p) - done[i], room)
                if n > 0:
                    part.append((i, n))
                    room -= n
            ids = torch.tensor([t for i, n in part for t in prompts[i][done[i]:done[i] + n]], device=dev)
            logits = self.model.forward_paged(ids, [roots[i] for i, _ in part], [n for _, n in part], cache)
            for row, (i, n) in zip(logits, part):
                done[i] += n
                last[i] = row
        self._check_device()
        out = [[list(p) for _ in range(samples)] for p in prompts]
        seqs = [(i, j, s) for i, r in enumerate(roots) for j, s in enumerate([r] + cache.fork(r, samples - 1))]
        logits = torch.stack([last[i] for i, _, _ in seqs]) if seqs else None
        for step in range(max_new_tokens):
            seqs_left = [x for x in range(len(seqs)) if len(out[seqs[x][0]][seqs[x][1]]) < limit]
            if len(seqs_left) < len(seqs):
                for x in set(range(len(seqs))) - set(seqs_left):
                    cache.free(seqs[x][2])
                seqs, logits = [seqs[x] for x in seqs_left], logits[seqs_left]
            if not seqs:
                break
            noise = torch.empty(logits.shape, dtype=torch.float32, device=dev).exponential_(generator=gen) if temperature > 0 else None
            ids = ops.sample(logits, noise, temperature, top_k, top_p, min_p)
            keep = []
            for x, ((i, j, s), t) in enumerate(zip(seqs, ids.tolist())):
                if t < 0:
                    self._check_device()
                    raise FloatingPointError("logits without a finite number: nothing to draw from")
                out[i][j].append(t)
                if t == eos_id:
                    cache.free(s)
                else:
                    keep.append(x)
            if len(keep) < len(seqs):
                seqs, ids = [seqs[x] for x in keep], ids[keep]
            if not seqs or step + 1 == max_new_tokens:
                break
            logits = self.model.forward_paged(ids, [s for _, _, s in seqs], [1] * len(seqs), cache)
        self._check_device()
        return out

    def _check_device(self) -> None:
        """What kernels could only record (a wait that ran out, lengths or ids that do not fit) is an error here, not tokens drawn from what they left."""
        if torch.device(self.device).type == "cuda":
            native.check_status()

    def generate_greedy(self, prompt_ids, max_new_tokens=256):
        return self.generate_ids(prompt_ids, max_new_tokens, temperature=0.0)

    def generate(self, prompt: str, max_new_tokens: int = 256, temperature: float = 1.0, top_p: float = 0.9, seed=None) -> str:
        if self.tok is None:
            raise ValueError("a tokenizer is required for text generation")
        ids = self.generate_ids(self.tok.encode(prompt), max_new_tokens, temperature, top_p, seed)
        return self.tok.decode(ids)


@torch.no_grad()
def benchmark_throughput(model, batch: int, seq_len: int, vocab: int, device, warmup: int = 2, iters: int = 10) -> float:
    """Forward-only tokens/s, timed on the device when it is a GPU."""
    model.eval()
    ids = torch.randint(0, vocab, (batch, seq_len), device=device)
    tgt = torch.randint(0, vocab, (batch, seq_len), device=device)
    for _ in range(warmup):
        model(ids, tgt)
    if device.type == "cuda":
        torch.cuda.synchronize()
        e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        e0.record()
        for _ in range(iters):
            model(ids, tgt)
        e1.record()
        torch.cuda.synchronize()
        dt = e0.elapsed_time(e1) / 1e3
    else:
        t0 = time.time()
        for _ in range(iters):
            model(ids, tgt)
        dt = time.time() - t0
    return batch * seq_len * iters / max(dt, 1e-9)
