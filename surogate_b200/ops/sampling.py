"""Drawing the next token of each row from its logits: ``sample_tokens``.

On a GPU one kernel (``csrc/sampling_kernels.cu``) reads each row once; elsewhere the PyTorch form below, in fp64, which is also the oracle of
the kernel tests.
"""
from __future__ import annotations

from typing import Tuple, Union

import torch

from .paged_kv import _kernels

Number = Union[float, torch.Tensor]


def sample_tokens_reference(logits: torch.Tensor, u: torch.Tensor, temperature: torch.Tensor, top_k: torch.Tensor, top_p: torch.Tensor, min_p: torch.Tensor
                            ) -> Tuple[torch.Tensor, torch.Tensor]:
    """The definition, row by row, in fp64 (parameters: one value a row)."""
    B, V = logits.shape
    lf = logits.double().nan_to_num(nan=-float("inf"), posinf=float("inf"), neginf=-float("inf")) + 0.0
    token, logprob = torch.full((B,), -1, dtype=torch.int32, device=logits.device), torch.full((B,), -float("inf"), device=logits.device)
    for b in range(B):
        l = lf[b]
        top = l.max()
        if top == -float("inf"):
            continue
        d = torch.where(l == top, torch.zeros_like(l), l - top)
        z = torch.exp(d).sum()
        T, k, p, m, x = float(temperature[b]), int(top_k[b]), float(top_p[b]), float(min_p[b]), float(u[b])
        if not T > 0:
            i = int((l == top).nonzero()[0])
        else:
            w = torch.where(d == 0, torch.ones_like(d), torch.where(d == -float("inf"), torch.zeros_like(d), torch.exp(d / T)))   # (T may be infinite)
            order = torch.sort(l, descending=True, stable=True).indices          # equal logits in the order of their indices
            s = w[order]
            keep = s >= min(m, 1.0) if m > 0 else torch.ones_like(s, dtype=torch.bool)
            if 0 < k < V:
                keep[k:] = False
            s = torch.where(keep, s, torch.zeros_like(s))
            if p < 1:
                before = torch.cumsum(s, 0) - s
                keep = keep & (before < max(p, 0.0) * s.sum())
                keep[0] = True
            kept = torch.zeros_like(w)
            kept[order[keep]] = w[order[keep]]
            c = torch.cumsum(kept, 0)
            over = (c > min(max(x, 0.0), 1.0 - 2.0 ** -53) * c[-1]).nonzero()
            i = int(over[0])
        token[b], logprob[b] = i, d[i] - torch.log(z)
    return token, logprob


def _each(value: Number, B: int, dtype: torch.dtype, device) -> torch.Tensor:
    if torch.is_tensor(value):
        if value.shape != (B,) or value.dtype != dtype:
            raise RuntimeError(f"sample_tokens: a parameter given as a tensor must be {dtype} [{B}]")
        return value
    return torch.full((B,), value, dtype=dtype, device=device)


def sample_tokens(logits: torch.Tensor, u: torch.Tensor, *, temperature: Number = 1.0, top_k: Union[int, torch.Tensor] = 0, top_p: Number = 1.0, min_p: Number = 0.0
                  ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Draw one token of each row of ``logits [rows, vocabulary]`` (fp32, bf16 or fp16; at most 2^20 - 1 tokens) by ``u`` fp32 ``[rows]``, uniform in [0, 1).

    Weights are ``exp((logit - largest) / temperature)``.  In the order of falling logit (equal ones: rising index) tokens are kept while fewer
    than ``top_k`` come before (0: no limit), the weight is at least ``min_p``, and the mass before is below ``top_p`` of the mass that the other
    two leave; at least one stays.  The token is the first, in the order of the indices, at which the kept mass exceeds ``u`` of the whole.
    ``temperature`` 0: the lowest index of the largest logit.  Each parameter is a number for all rows or a tensor ``[rows]`` on the logits'
    device (fp32; ``top_k`` int32).

    Returns (tokens int32, log-probabilities fp32): the latter under the softmax of the logits as they are, without temperature and filters (what
    ``Trainer.token_logprobs`` recomputes).  NaN counts as -inf; a row without a logit above -inf gives token -1 and -inf."""
    if logits.dim() == 2 and not 0 < logits.shape[1] < 1 << 20:
        raise RuntimeError("sample_tokens: the vocabulary must have 1 to 2^20 - 1 tokens")
    if logits.dim() != 2 or u.shape != (logits.shape[0],) or logits.dtype not in (torch.float32, torch.bfloat16, torch.float16) or u.dtype != torch.float32:
        raise RuntimeError("sample_tokens: logits must be fp32, bf16 or fp16 [rows, vocabulary], u fp32 [rows]")
    if not torch.is_tensor(temperature) and not temperature >= 0:
        raise RuntimeError("sample_tokens: the temperature must not be negative")
    if logits.is_cuda:
        t, k, p, m = torch.is_tensor(temperature), torch.is_tensor(top_k), torch.is_tensor(top_p), torch.is_tensor(min_p)
        return _kernels().sample_tokens(logits, u, temperature if t else None, top_k if k else None, top_p if p else None, min_p if m else None,
                                        1.0 if t else temperature, 0 if k else top_k, 1.0 if p else top_p, 0.0 if m else min_p)
    B = logits.shape[0]
    f = lambda x: _each(x, B, torch.float32, logits.device)  # noqa: E731
    return sample_tokens_reference(logits, u, f(temperature), _each(top_k, B, torch.int32, logits.device), f(top_p), f(min_p))
