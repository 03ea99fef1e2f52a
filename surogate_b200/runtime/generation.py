"""Answers of a model that is loaded for training: prompts in, sampled completions with their log-probabilities out.

``generate`` (public as ``Trainer.generate``) runs the prompts once, keeps their keys and values in a paged cache (``ops.PagedKVCache``) and
then one token of every unfinished completion per step: embed, attend over the pages, draw (``ops.sample_tokens``).  Completions of one prompt
share its pages; only the last, partly filled one is copied when they part.  The uniform numbers of step ``i`` are row ``i`` of one generator's
stream, one for each completion, so a completion's draws do not depend on when its neighbours end.  (Its logits may, within their rounding: products over
other numbers of rows add up in another order, and a recipe with one scale for a whole tensor takes it from all rows.)  What recipes
measure here does not reach the scales of training.

Models whose layers mix positions by other means than attention (short convolutions, state-space and delta-rule mixers, attention that keeps
values of other layers) have no such cache: for them every step runs the whole prefix again, with the same draws.
"""
from __future__ import annotations

from dataclasses import dataclass, field
from typing import List, Optional, Sequence

import torch

from ..ops.paged_kv import ATTENTION_DIMS, PagedKVCache
from ..ops.sampling import sample_tokens

# ``torch_fn`` ops that mix positions; attention_general runs on the cache, the others keep what a cache of keys and values does not hold
_MIXERS = ("attention_general", "short_conv", "mamba2_mixer", "qwen35_gated_attention", "qwen35_gated_delta_net", "gated_delta_rule")


@dataclass
class Completion:
    """One answer: the drawn tokens (an end token among them), each one's log-probability under the model's softmax, and why it ended."""
    tokens: List[int] = field(default_factory=list)
    logprobs: List[float] = field(default_factory=list)
    finish_reason: str = "length"       # "stop": the end token was drawn


class CacheStep:
    """What the attention ops of one forward pass need of the cache (``ExecContext.kv``): the batch rows' pages, where their new tokens go
    and how many keys they then have.  ``prompt``: the pass brings whole prompts, which attend within themselves."""

    def __init__(self, cache: PagedKVCache, table: torch.Tensor, start: torch.Tensor, count: Optional[torch.Tensor], prompt: bool):
        self.cache, self.table, self.start, self.count, self.prompt = cache, table, start, count, prompt
        self.lengths = start + 1

    def attend(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, **kw) -> Optional[torch.Tensor]:
        """Append the new tokens of ``layer``; the attention of one new token a row, or None for a prompt (attend as without a cache)."""
        self.cache.append(layer, k, v, self.table, self.start, self.count)
        if self.prompt:
            return None
        B, _, Hq, D = q.shape
        return self.cache.attend(layer, q[:, 0], self.table, self.lengths, **kw).reshape(B, 1, Hq * D)


def cache_layout(cm, device: torch.device):
    """(kv heads, head size) of the cache that the model's attention layers can share, or None if it has none."""
    found = set()
    for bt in set(cm.layer_types):
        for op in cm.block_fwd[bt].ops:
            a = op.attrs
            if op.kind == "flash_attention" or (op.kind == "torch_fn" and a.get("fn") == "attention_general"):
                if not a.get("causal", True) or a.get("v_head_dim") not in (None, a["head_dim"]) or a["num_q_heads"] % a["num_kv_heads"]:
                    return None
                found.add((a["num_kv_heads"], a["head_dim"]))
            elif op.kind == "torch_fn" and a.get("fn") in _MIXERS:
                return None
    if len(found) != 1:
        return None
    heads, dim = found.pop()
    return (heads, dim) if device.type != "cuda" or dim in ATTENTION_DIMS else None


def _padded(rows: Sequence[Sequence[int]], device: torch.device) -> torch.Tensor:
    """Token rows padded on the right (attention and the other mixers are causal: padding reaches no token before it); on a GPU to whole
    tiles of the attention kernels."""
    T = max(len(r) for r in rows)
    T = (T + 127) // 128 * 128 if device.type == "cuda" else T
    out = torch.zeros(len(rows), T, dtype=torch.int32)
    for i, r in enumerate(rows):
        out[i, :len(r)] = torch.tensor(r, dtype=torch.int32)
    return out.to(device)


@torch.no_grad()
def generate(trainer, prompts: Sequence[Sequence[int]], *, n: int = 1, max_new_tokens: int = 64, temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0,
             min_p: float = 0.0, seed: int = 0, eos_id: Optional[int] = None, page_size: int = 64, cache_dtype: Optional[torch.dtype] = None,
             prompt_rows: int = 8) -> List[List[Completion]]:
    """See ``Trainer.generate``."""
    prompts = [[int(t) for t in p] for p in prompts]
    if any(not p for p in prompts):
        raise ValueError("generate: a prompt needs at least one token")
    vocab = trainer.model.vocab_size
    if any(not 0 <= t < vocab for p in prompts for t in p):
        raise ValueError(f"generate: a prompt has a token outside the vocabulary of {vocab}")
    if n < 1 or max_new_tokens < 0 or prompt_rows < 1:
        raise ValueError("generate: n and prompt_rows must be positive, max_new_tokens not negative")
    if trainer.world > 1 and (trainer.cfg.zero_level >= 3 or trainer.cfg.ep_size > 1):
        raise NotImplementedError("generate: weights spread over ranks (ZeRO-3, expert parallelism) would need every rank to take the same steps")
    if trainer._visual is not None:
        raise NotImplementedError("generate answers text: clear the visual inputs first (set_visual_inputs without arguments)")
    out = [[Completion() for _ in range(n)] for _ in prompts]
    if not prompts or max_new_tokens == 0:
        return out
    device, ex = trainer.device, trainer.executor
    gen = torch.Generator(device=device).manual_seed(int(seed))
    draw = dict(temperature=float(temperature), top_k=int(top_k), top_p=float(top_p), min_p=float(min_p))
    trainer.drain_optimizer()
    layout = cache_layout(trainer.cm, device)
    cache = None
    dtype = cache_dtype or ex.options.act_dtype
    if device.type == "cuda" and dtype not in (torch.bfloat16, torch.float16, torch.float8_e4m3fn):
        if cache_dtype is not None:
            raise ValueError(f"generate: a cache of {dtype} has no attention kernel")
        layout = None                                                  # fp32 activations on a GPU: whole passes
    if layout is not None:
        # a prompt's pages once, and for each completion those behind the prompt's last full page
        pages = sum((len(p) + page_size - 1) // page_size + n * ((len(p) + max_new_tokens + page_size - 1) // page_size - len(p) // page_size) for p in prompts)
        cache = PagedKVCache(trainer.cm.n_layers, pages, page_size, layout[0], layout[1], len(prompts) * n, dtype=dtype, device=device)
    elif cache_dtype is not None:
        raise ValueError("generate: this model has no key/value cache")
    trainer.store.grads_enabled = False
    try:
        with trainer.recipe.inference():
            run = _Cached(trainer, cache, prompts, n, prompt_rows) if cache is not None else _Uncached(trainer, prompts, n, prompt_rows)
            alive = list(range(len(prompts) * n))                          # completion c of prompt i is number i * n + c
            tokens = None
            for step in range(max_new_tokens):
                u = torch.rand(len(prompts) * n, generator=gen, device=device)
                logits = run.first() if step == 0 else run.next(alive, tokens)
                tokens, logprobs = sample_tokens(logits, u[torch.tensor(alive, device=device)] if len(alive) < len(u) else u, **draw)
                got, lp = tokens.tolist(), logprobs.tolist()
                if min(got) < 0:
                    _check_device(device)
                    raise FloatingPointError("generate: a row of logits has no finite value")
                going = []
                for row, s in enumerate(alive):
                    c = out[s // n][s % n]
                    c.tokens.append(got[row])
                    c.logprobs.append(lp[row])
                    if eos_id is not None and got[row] == eos_id:
                        c.finish_reason = "stop"
                        run.drop(s)
                    else:
                        going.append(row)
                if not going:
                    break
                if len(going) < len(alive):
                    tokens = tokens[torch.tensor(going, device=device)]
                    alive = [alive[r] for r in going]
        _check_device(device)
    finally:
        trainer.store.grads_enabled = True
    return out


def _check_device(device: torch.device) -> None:
    """Raise if a kernel gave up or left something out (a wait, a page, a token): the answers would look like any others."""
    if device.type == "cuda":
        from ..ops import check_device_errors

        check_device_errors()


class _Cached:
    """Steps over a paged cache."""

    def __init__(self, trainer, cache: PagedKVCache, prompts, n: int, prompt_rows: int):
        self.tr, self.cache, self.prompts, self.n, self.prompt_rows = trainer, cache, prompts, n, prompt_rows

    def first(self) -> torch.Tensor:
        """All prompts, ``prompt_rows`` at a time: the logits behind each, once for each of its completions."""
        dev, outs = self.tr.device, []
        for a in range(0, len(self.prompts), self.prompt_rows):
            part = self.prompts[a:a + self.prompt_rows]
            seqs = [(a + i) * self.n for i in range(len(part))]
            self.cache.reserve({s: len(p) for s, p in zip(seqs, part)})
            ids = _padded(part, dev)
            count = torch.tensor([len(p) for p in part], dtype=torch.int32).to(dev)
            step = CacheStep(self.cache, self.cache.table(seqs), torch.zeros_like(count), count, prompt=True)
            pos = torch.arange(ids.shape[1], dtype=torch.int32, device=dev).expand(ids.shape).contiguous()
            outs.append(self.tr.executor.last_logits(ids, pos, count.long() - 1, kv=step))
            for s in seqs:
                self.cache.fork(s, range(s + 1, s + self.n))
        return torch.cat(outs).repeat_interleave(self.n, dim=0)

    def next(self, alive: Sequence[int], tokens: torch.Tensor) -> torch.Tensor:
        dev = self.tr.device
        start = torch.tensor([self.cache.length(s) for s in alive], dtype=torch.int32).to(dev)
        self.cache.reserve({s: 1 for s in alive})
        step = CacheStep(self.cache, self.cache.table(alive), start, None, prompt=False)
        return self.tr.executor.last_logits(tokens.view(-1, 1), start.view(-1, 1), torch.zeros(len(alive), dtype=torch.int64, device=dev), kv=step)

    def drop(self, s: int) -> None:
        self.cache.free(s)


class _Uncached:
    """Steps that run every row's whole prefix again."""

    def __init__(self, trainer, prompts, n: int, prompt_rows: int):
        self.tr, self.n, self.prompt_rows = trainer, n, prompt_rows
        self.rows = [list(p) for p in prompts for _ in range(n)]

    def _logits(self, rows) -> torch.Tensor:
        dev, outs = self.tr.device, []
        for a in range(0, len(rows), self.prompt_rows):
            part = rows[a:a + self.prompt_rows]
            ids = _padded(part, dev)
            pos = torch.arange(ids.shape[1], dtype=torch.int32, device=dev).expand(ids.shape).contiguous()
            outs.append(self.tr.executor.last_logits(ids, pos, torch.tensor([len(p) - 1 for p in part]).to(dev)))
        return torch.cat(outs)

    def first(self) -> torch.Tensor:
        return self._logits(self.rows[::self.n]).repeat_interleave(self.n, dim=0)

    def next(self, alive: Sequence[int], tokens: torch.Tensor) -> torch.Tensor:
        for s, t in zip(alive, tokens.tolist()):
            self.rows[s].append(t)
        return self._logits([self.rows[s] for s in alive])

    def drop(self, s: int) -> None:
        pass
