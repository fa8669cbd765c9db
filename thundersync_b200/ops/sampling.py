"""Sampling from logits with temperature, top-k, top-p and min-p, from given random numbers.

:func:`sample_tokens` draws one token per row of ``logits`` [B, V] and returns it with its log-prob, so an on-policy
loop has the behaviour log-prob beside the token. Per row, with ``p = softmax(logits / temperature)`` and tokens ranked
by logit (equal logits: the lower token first), a token is kept when all of these hold, or when it ranks first:

    fewer than ``top_k`` tokens rank before it          (0 or less: no limit)
    the tokens ranked before it have mass < ``top_p``   (1 or more: no limit)
    its probability is at least ``min_p`` of the largest one

Each condition looks at the full distribution ``p``. The token is the kept one with the largest ``p_i / noise_i``: with
independent Exp(1) ``noise`` [B, V] (``torch.empty_like(...).exponential_()``) it is a draw from ``p`` restricted to
the kept tokens, and two models given the same noise draw coupled samples. The result depends on its arguments alone.

The log-prob is the token's under ``p``, the whole softmax at the row's temperature, which is what a trainer
recomputes; it is not renormalised to the kept tokens. Temperature 0 (anything below 1e-6) takes the first-ranked token
and reports its log-prob at temperature 1. A row without a distribution (it holds NaN or +inf, or nothing but -inf)
gives token -1 and log-prob NaN.
"""

from __future__ import annotations

import math

import torch

from thundersync_b200.ops._ext import native

__all__ = ["sample_tokens"]

_NATIVE = (torch.float32, torch.bfloat16, torch.float16)
_COLDEST = 1e-6


def _setting(value, name: str, n: int, device, dtype, low: float, high: float):
    """(tensor or None, number) of a setting; a number is checked here, a tensor's values are the caller's."""
    if isinstance(value, torch.Tensor):
        if tuple(value.shape) != (n,) or value.device != device:
            raise ValueError(f"{name} must be a number or a tensor [{n}] on {device}, got {tuple(value.shape)} on "
                             f"{value.device}")
        return value.to(dtype).contiguous(), 0
    if not low <= value <= high:
        raise ValueError(f"{name} must be in [{low}, {high}], got {value}")
    return None, value


def _whole(top_k, v: int) -> int:
    """A number of tokens in [0, v]: 0 and v are no limit, and what is below or above them none either."""
    if math.isnan(top_k) or (math.isfinite(top_k) and top_k != int(top_k)):
        raise ValueError(f"top_k must be a whole number, got {top_k}")
    return int(min(max(top_k, 0), v))


def sample_tokens(logits: torch.Tensor, noise: torch.Tensor | None, *, temperature: float | torch.Tensor = 1.0,
                  top_k: int | torch.Tensor = 0, top_p: float | torch.Tensor = 1.0,
                  min_p: float | torch.Tensor = 0.0) -> tuple[torch.Tensor, torch.Tensor]:
    """(tokens int64 [B], log-probs fp32 [B]) drawn from ``logits`` [B, V] (fp32, bf16 or fp16).

    ``noise``: fp32 [B, V], positive Exp(1) draws; None where ``temperature`` is the number 0. Each setting is a number
    or a tensor [B]."""
    if logits.dim() != 2 or not logits.is_floating_point() or logits.shape[1] < 1:
        raise ValueError(f"logits must be a floating-point [B, V], got {logits.dtype} {tuple(logits.shape)}")
    n = logits.shape[0]
    dev = logits.device
    if noise is None:
        if isinstance(temperature, torch.Tensor) or temperature != 0:
            raise ValueError("noise may be left out at temperature 0 only")
    elif noise.shape != logits.shape or noise.dtype != torch.float32 or noise.device != dev:
        raise ValueError(f"noise must be fp32 {tuple(logits.shape)} on {dev}, got {noise.dtype} {tuple(noise.shape)} "
                         f"on {noise.device}")
    t = _setting(temperature, "temperature", n, dev, torch.float32, 0.0, math.inf)
    k = _setting(top_k if isinstance(top_k, torch.Tensor) else _whole(top_k, logits.shape[1]), "top_k", n, dev,
                 torch.int64, 0, math.inf)
    p = _setting(top_p, "top_p", n, dev, torch.float32, 0.0, math.inf)
    mp = _setting(min_p, "min_p", n, dev, torch.float32, 0.0, 1.0)
    logits = logits.detach()
    if logits.is_cuda and logits.dtype in _NATIVE:
        if logits.stride(1) != 1 and logits.shape[1] > 1:
            logits = logits.contiguous()
        if noise is not None and noise.stride(1) != 1 and noise.shape[1] > 1:
            noise = noise.contiguous()
        tok, lp = native().sample_tokens(logits, noise, t[0], float(t[1]), k[0], int(k[1]), p[0], float(p[1]), mp[0],
                                         float(mp[1]))
        return tok, lp
    return _sample_reference(logits, noise, *(x if x is not None else y for x, y in (t, k, p, mp)))


def _sample_reference(logits, noise, temperature, top_k, top_p, min_p):
    z = logits.to(torch.float64 if logits.dtype == torch.float64 else torch.float32)
    n, v = z.shape
    t, k, p, mp = (torch.as_tensor(x, device=z.device).expand(n)[:, None] for x in (temperature, top_k, top_p, min_p))
    greedy = ~(t >= _COLDEST)
    t = torch.where(greedy, torch.ones_like(t, dtype=z.dtype), t.to(z.dtype))
    m = z.amax(-1, keepdim=True)
    a = (z - m) / t
    w = torch.exp(a)
    s = w.sum(-1, keepdim=True)
    order = z.sort(dim=-1, descending=True, stable=True)[1]
    ws = w.gather(-1, order)
    before = ws.cumsum(-1) - ws
    rank = torch.arange(v, device=z.device)[None]
    keep = ((k <= 0) | (rank < k)) & ((p >= 1) | (before < p * s)) & (ws >= mp.clamp(max=1))
    keep = (keep & ~greedy) | (rank == 0)
    race = torch.where(greedy, torch.ones_like(w), w if noise is None else w / noise)
    key = torch.where(torch.zeros_like(keep).scatter_(-1, order, keep), race, torch.full_like(race, -1.0))
    tok = key.argmax(-1)
    lp = (a.gather(-1, tok[:, None]) - torch.log(s)).squeeze(-1)
    ok = ((s > 0) & (s < math.inf)).squeeze(-1)
    return torch.where(ok, tok, -1), torch.where(ok, lp, math.nan).to(torch.float32)
