"""Distillation from a teacher's top logits: the teacher's entries, and the loss against them with its gradient.

A teacher that scores a position with its ``k`` most likely tokens (ids and log-probs, :func:`topk_logprobs`) says far
more about it than the log-prob of the one sampled token, at a few hundred bytes per position. The loss compares them
with the student's distribution ``p = softmax(z / temperature)`` over the whole vocabulary. Per row, with the entries'
set ``S``, ``q = exp(teacher log-prob)``, and ``P``, ``Q`` what ``p`` and ``q`` give to all other tokens together:

    direction "forward":  sum_S q (log q - log p)  [+ Q (log Q - log P)]      KL(teacher || student)
    direction "reverse":  sum_S p (log p - log q)  [+ P (log P - log Q)]      KL(student || teacher)

``tail=True`` adds the bracketed term (all other tokens as one class; ``Q`` is held at 1e-7 at least, and the term is
left out where ``P`` is 0 in 64 bits: the others are masked, or some 744 nats and more below the entries). The teacher is
a constant: no gradient reaches it.

An entry with id -1 or log-prob -inf is no entry, so rows may have fewer than ``K``; of entries with the same id the
first counts. A row without entries has loss 0 and gradient 0, whatever its logits are. A row whose logits hold NaN,
+inf, or nothing but -inf has loss NaN.

:func:`topk_distill_loss` takes logits that are in memory; :func:`lm_head_topk_distill` takes hidden states and the
LM-head weight. Sums, softmax statistics and the entries' arithmetic are fp32 or wider; the gradient is rounded once,
to the logits' type.
"""

from __future__ import annotations

import math
import threading
import weakref

import torch

from thundersync_b200.ops import sink as _sink
from thundersync_b200.ops._ext import native
from thundersync_b200.ops.gemm import gemm, gemm_accumulate
from thundersync_b200.ops.logprob import _logits_fp32, _row_block

__all__ = ["topk_logprobs", "topk_distill_loss", "lm_head_topk_distill", "MAX_ENTRIES"]

MAX_ENTRIES = 256  # teacher entries of a row (one per thread of a row's block)
_TAIL_FLOOR = 1e-7
_NATIVE = (torch.float32, torch.bfloat16, torch.float16)


def _native_rows(logits: torch.Tensor) -> bool:
    return logits.is_cuda and logits.dtype in _NATIVE


def _rows_contiguous(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _check_logits(logits: torch.Tensor) -> None:
    if logits.dim() != 2 or not logits.is_floating_point():
        raise ValueError(f"logits must be a floating-point [N, V], got {logits.dtype} {tuple(logits.shape)}")
    if logits.shape[1] < 1:
        raise ValueError("logits must have a vocabulary")


def _check_teacher(n: int, ids, logprobs, temperature: float, direction: str, device):
    if ids.dim() != 2 or ids.shape[0] != n or not 1 <= ids.shape[1] <= MAX_ENTRIES:
        raise ValueError(f"teacher_ids must be [N, K] with N = {n} and K in [1, {MAX_ENTRIES}], got {tuple(ids.shape)}")
    if ids.is_floating_point() or ids.dtype == torch.bool:
        raise ValueError("teacher_ids must be integers")
    if logprobs.shape != ids.shape or not logprobs.is_floating_point():
        raise ValueError(f"teacher_logprobs must be floating-point {tuple(ids.shape)}, got {logprobs.dtype} "
                         f"{tuple(logprobs.shape)}")
    if logprobs.requires_grad:
        raise ValueError("teacher_logprobs must be detached")
    if ids.device != device or logprobs.device != device:
        raise ValueError("the teacher's entries must be on the student's device")
    if not (temperature > 0 and math.isfinite(temperature)):
        raise ValueError(f"temperature must be positive, got {temperature}")
    if direction not in ("forward", "reverse"):
        raise ValueError(f"direction must be 'forward' or 'reverse', got {direction!r}")
    wide = torch.float64 if logprobs.dtype == torch.float64 and not ids.is_cuda else torch.float32
    return ids.to(torch.int64).contiguous(), logprobs.to(wide).contiguous()


# ------------------------------------------------------------------ the teacher's side
def topk_logprobs(logits: torch.Tensor, k: int, *, temperature: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """The ``k`` most likely tokens of each row of ``logits`` [N, V], most likely first: (ids int64 [N, k], log-probs
    fp32 [N, k] under ``softmax(logits / temperature)``).

    Equal logits: the lower token comes first. NaN counts as less than -inf, and a row that holds NaN or +inf has
    log-probs NaN; a row of -inf alone has log-probs -inf.
    """
    _check_logits(logits)
    k = int(k)
    if not 1 <= k <= min(MAX_ENTRIES, logits.shape[1]):
        raise ValueError(f"k must be in [1, {min(MAX_ENTRIES, logits.shape[1])}], got {k}")
    if not (temperature > 0 and math.isfinite(temperature)):
        raise ValueError(f"temperature must be positive, got {temperature}")
    logits = logits.detach()
    if _native_rows(logits):
        ids, lp = native().topk_logprobs(_rows_contiguous(logits), k, float(temperature))
        return ids, lp
    return _topk_reference(logits, k, temperature)


def _topk_reference(logits, k, temperature):
    z = logits.to(torch.float64 if logits.dtype == torch.float64 else torch.float32)
    order = torch.where(z.isnan(), -math.inf, z)
    top, ids = order.sort(dim=-1, descending=True, stable=True)
    if bool(z.isnan().any()):  # NaN after -inf
        last = z.isnan().gather(-1, ids)
        ids = ids.gather(-1, last.to(torch.int8).sort(dim=-1, stable=True)[1])
    ids = ids[:, :k].contiguous()
    m = z.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    total = torch.exp((z - m) / temperature).sum(-1, keepdim=True)
    lp = (z.gather(-1, ids) - m) / temperature - torch.where(total == 0, 0.0, torch.log(total))
    return ids, lp.to(torch.float32)


# ------------------------------------------------------------------ the loss on logits
def _slots(ids, logprobs, v: int):
    """Which entries count: inside the vocabulary, with a probability, first of their id."""
    have = (ids >= 0) & (ids < v) & (logprobs != -math.inf)
    k = ids.shape[1]
    same = (ids[:, :, None] == ids[:, None, :]) & have[:, None, :]
    earlier = torch.ones(k, k, dtype=torch.bool, device=ids.device).tril(-1)
    return have & ~(same & earlier).any(-1)


def _loss_reference(z, ids, logprobs, temperature, direction, tail):
    """The definition in plain torch, differentiable in ``z`` [N, V]; computed in 64 bits, as the kernels do the entries'
    arithmetic, so both leave the tail out of the same rows. fp32 [N] (fp64 for fp64 logits)."""
    n, v = z.shape
    wide = torch.float64
    have = _slots(ids, logprobs, v)
    used = have.any(-1)
    out = torch.float64 if z.dtype == torch.float64 else torch.float32
    z = torch.where(used[:, None], z.to(wide), torch.zeros((), dtype=wide, device=z.device))
    logp = torch.log_softmax(z / temperature, -1)
    at = torch.where(have, ids, 0)
    t = torch.where(have, logprobs.to(wide), torch.zeros((), dtype=wide, device=z.device))
    a = logp.gather(-1, at)
    if direction == "forward":
        loss = torch.where(have, t.exp() * (t - a), torch.zeros_like(a)).sum(-1)
    else:
        p = a.exp()
        on = have & ((p > 0) | p.isnan())
        a = torch.where(on, a, torch.zeros_like(a))
        loss = torch.where(on, a.exp() * (a - t), torch.zeros_like(a)).sum(-1)
    if tail:
        inside = torch.zeros(n, v, dtype=torch.bool, device=z.device)
        rows = torch.arange(n, device=z.device)[:, None].expand_as(at)
        inside[rows[have], at[have]] = True
        rest = logp.masked_fill(inside, -math.inf)
        some = used & (rest.exp().sum(-1) != 0)  # (NaN stays)
        lpt = torch.logsumexp(torch.where(some[:, None], rest, torch.zeros_like(rest)), -1)
        qt = (1.0 - torch.where(have, t.exp(), torch.zeros_like(t)).sum(-1)).clamp(min=_TAIL_FLOOR)
        more = qt * (qt.log() - lpt) if direction == "forward" else lpt.exp() * (lpt - qt.log())
        loss = loss + torch.where(some, more, torch.zeros_like(more))
    return loss.to(out)


def topk_distill_loss(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logprobs: torch.Tensor, *,
                      temperature: float = 1.0, direction: str = "forward", tail: bool = True) -> torch.Tensor:
    """Loss [N] (fp32) of student ``logits`` [N, V] against the teacher's entries [N, K], differentiable in ``logits``.

    ``teacher_logprobs`` are under the teacher's distribution at the same ``temperature``."""
    _check_logits(logits)
    ids, lp = _check_teacher(logits.shape[0], teacher_ids, teacher_logprobs, temperature, direction, logits.device)
    if _native_rows(logits):
        return native().distill_rows(_rows_contiguous(logits), ids, lp, float(temperature), direction == "reverse",
                                     bool(tail))
    return _loss_reference(logits, ids, lp, temperature, direction, tail)


# ------------------------------------------------------------------ the loss from hidden states
# Rows of a block, where the caller names none: a block's buffers are its fp32 logits (2.5 GB at 4096 rows of a
# 151,936-token vocabulary) and the two bf16 halves of its dlogits (as much again). One block writes the weight gradient
# in bf16 at once; several add fp32 products and round at the end.
BLOCK_ROWS = 4096
# The forwards' fp32 logits that a process keeps on a device for their backwards, in bytes, of all graphs that are alive
# together. A block past it computes them again, which at 2048 rows x 2048 x 151,936 takes a third of the backward's time
# on top; keeping them holds that memory from the forward to the backward.
KEEP_LOGITS_BYTES = 3 << 30
_kept_lock = threading.Lock()


class _KeptLogits:
    """A block's logits from its forward to its backward; they count as kept until they are taken or the graph is gone."""

    _alive: "weakref.WeakSet[_KeptLogits]" = weakref.WeakSet()

    def __init__(self, device: torch.device, size: int) -> None:
        self.device, self.size, self.logits = device, size, None

    @classmethod
    def room(cls, device: torch.device, size: int) -> "_KeptLogits | None":
        """A place for ``size`` bytes of logits, or None."""
        with _kept_lock:
            if size + sum(k.size for k in cls._alive if k.device == device) > KEEP_LOGITS_BYTES:
                return None
            kept = cls(device, size)
            cls._alive.add(kept)
            return kept

    def take(self) -> torch.Tensor | None:
        """The logits, once."""
        logits, self.logits, self.size = self.logits, None, 0
        return logits


def _fused_ok(hidden: torch.Tensor, weight: torch.Tensor) -> bool:
    return (hidden.is_cuda and hidden.dtype == torch.bfloat16 and weight.dtype == torch.bfloat16
            and hidden.shape[1] % 8 == 0 and hidden.shape[1] > 0 and weight.shape[0] % 8 == 0 and weight.shape[0] > 0
            and weight.is_contiguous())


def _to_eight(d: torch.Tensor, h: torch.Tensor):
    """Zero rows up to a multiple of 8 for the accumulating GEMM's contraction."""
    pad = (-d.shape[0]) % 8
    if not pad:
        return d, h
    return (torch.cat((d, d.new_zeros(pad, d.shape[1]))), torch.cat((h, h.new_zeros(pad, h.shape[1]))))


class _DifferentiatedOnce(torch.autograd.Function):
    """A gradient as the end of what can be differentiated: asking how it depends on the inputs is an error."""

    @staticmethod
    def forward(ctx, gradient, *inputs):
        return gradient

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("lm_head_topk_distill is differentiable once: its gradients have no gradients of their own")


class _HeadTopkDistill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, ids, logprobs, rows, temperature, direction, tail, round_dlogits,
                differentiated):
        n = hidden.shape[0]
        ctx.conf = (rows, temperature, direction, tail, round_dlogits)
        ctx.param = weight  # for the sink, which knows its parameters by identity
        ctx.kept = []  # logits of the blocks that keep theirs: a first backward uses them up, another computes them again
        saved = []  # four small tensors of each block
        fused = _fused_ok(hidden, weight)
        reverse = direction == "reverse"
        loss = []
        for r0 in range(0, n, rows):
            r1 = min(n, r0 + rows)
            if fused:
                kept = _KeptLogits.room(hidden.device, 4 * (r1 - r0) * weight.shape[0]) if differentiated else None
                part, *small, logits = native().distill_head_fwd(hidden[r0:r1], weight, ids[r0:r1], logprobs[r0:r1],
                                                                 temperature, reverse, tail, kept is not None)
                if kept is not None:
                    kept.logits = logits
                saved += small
                ctx.kept.append(kept)
                loss.append(part)
                continue
            logits = _logits_fp32(hidden[r0:r1], weight)
            if _native_rows(logits):
                part, *small = native().distill_rows_fwd(logits, ids[r0:r1], logprobs[r0:r1], temperature, reverse, tail)
                saved += small
            else:
                part = _loss_reference(logits, ids[r0:r1], logprobs[r0:r1], temperature, direction, tail)
            loss.append(part)
        ctx.save_for_backward(hidden, weight, ids, logprobs, *saved)
        if len(loss) == 1:
            return loss[0]
        return torch.cat(loss) if loss else hidden.new_zeros(0, dtype=torch.float32)

    @staticmethod
    def backward(ctx, g):
        hidden, weight = ctx.saved_tensors[:2]
        with torch.no_grad():
            grads = _HeadTopkDistill._gradients(ctx, g)
        if torch.is_grad_enabled():  # (create_graph)
            grads = [None if d is None else _DifferentiatedOnce.apply(d, hidden, weight, g) for d in grads]
        return (*grads, None, None, None, None, None, None, None, None)

    @staticmethod
    def _gradients(ctx, g):
        hidden, weight, ids, logprobs, *saved = ctx.saved_tensors
        rows, temperature, direction, tail, round_dlogits = ctx.conf
        n = hidden.shape[0]
        need_h, need_w = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        fused = _fused_ok(hidden, weight)
        dh = torch.empty_like(hidden) if need_h else None
        s = _sink.active()
        sink_w = need_w and s is not None and s.owns(ctx.param)
        at_once = fused and need_w and not sink_w and 0 < n <= rows  # one block: no fp32 sum of blocks
        dw = None
        if need_w and not sink_w and not at_once:
            wide = torch.float32 if weight.dtype != torch.float64 else torch.float64
            dw = torch.zeros(weight.shape, dtype=wide, device=weight.device)
        g = g.contiguous()
        for i, r0 in enumerate(range(0, n, rows)):
            r1 = min(n, r0 + rows)
            h = hidden[r0:r1]
            logits = ctx.kept[i].take() if ctx.kept and ctx.kept[i] is not None else None
            if logits is None:
                logits = native().distill_head_logits(h, weight) if fused else _logits_fp32(h, weight)
            parts = []  # of the dlogits, which are their sum
            if _native_rows(logits):
                dtype = hidden.dtype if fused or round_dlogits else torch.float32
                parts.append(torch.empty(logits.shape, dtype=dtype, device=hidden.device))
                if fused and not round_dlogits:
                    parts.append(torch.empty_like(parts[0]))
                native().distill_rows_bwd(logits, *saved[4 * i:4 * i + 4], g[r0:r1].float(), temperature, parts[0],
                                          parts[1] if len(parts) > 1 else None)
            else:
                with torch.enable_grad():
                    z = logits.requires_grad_(True)
                    part = _loss_reference(z, ids[r0:r1], logprobs[r0:r1], temperature, direction, tail)
                (d,) = torch.autograd.grad(part, z, g[r0:r1].to(part.dtype))
                parts.append(d.to(hidden.dtype) if round_dlogits else d)
            del logits
            if need_h:
                if fused:
                    native().distill_head_dh(parts[0], parts[1] if len(parts) > 1 else None, weight, dh[r0:r1])
                elif parts[0].dtype == weight.dtype:
                    gemm(parts[0], weight, b_t=False, out=dh[r0:r1])
                else:
                    dh[r0:r1] = torch.mm(parts[0], weight.to(parts[0].dtype))
            if at_once:
                dw = native().distill_head_dw(parts[0], parts[1] if len(parts) > 1 else None, h)
            elif need_w:
                for d in parts:
                    d8, h8 = _to_eight(d, h) if d.is_cuda else (d, h)
                    if sink_w:
                        s.addmm_(s.view(ctx.param), d8, h8)
                    else:
                        gemm_accumulate(dw, d8, h8, a_t=True, b_t=False)
        return dh, None if dw is None else dw.to(weight.dtype)


def lm_head_topk_distill(hidden: torch.Tensor, weight: torch.Tensor, teacher_ids: torch.Tensor,
                         teacher_logprobs: torch.Tensor, *, temperature: float = 1.0, direction: str = "forward",
                         tail: bool = True, rows: int | None = None, round_dlogits: bool = False) -> torch.Tensor:
    """Loss [N] (fp32) of the student ``hidden`` [N, D] · ``weight`` [V, D]ᵀ against the teacher's entries [N, K],
    differentiable in ``hidden`` and ``weight`` (whose gradient honours an active gradient sink).

    ``rows`` rows are worked at a time (default ``BLOCK_ROWS``), and up to ``KEEP_LOGITS_BYTES`` of fp32 logits, of all
    graphs of a process on a device together, stay from their forwards to their backwards; both are attributes of this
    module. Hidden rows must be finite: a row without entries gives no gradient, but its zeros meet the hidden row in the
    weight gradient.

    The tensor cores take both operands of a product in one type, and the weight is bf16. So the dlogits go into the two
    gradient products as two bf16 halves (16 bits), and the gradients are rounded once, to their type: about 1.7e-3 of
    their norm in bf16. ``round_dlogits=True`` rounds the dlogits to the hidden states' type instead, as
    :func:`lm_head_logprob` does, for half the arithmetic: the gradients are then 1.9e-3 to 3.3e-3 from 64 bits, and more
    where the dlogits of a row cancel in ``d · weight`` (1.1e-2 where the entries' weight rows are nearly the same)."""
    if hidden.dim() != 2:
        raise ValueError(f"hidden must be [N, D], got {tuple(hidden.shape)}")
    if weight.dim() != 2 or weight.shape[1] != hidden.shape[1]:
        raise ValueError(f"weight {tuple(weight.shape)} does not match hidden dim {hidden.shape[1]}")
    if weight.dtype != hidden.dtype or weight.device != hidden.device:
        raise ValueError("hidden and weight must have one dtype and device")
    ids, lp = _check_teacher(hidden.shape[0], teacher_ids, teacher_logprobs, temperature, direction, hidden.device)
    rows = _row_block(BLOCK_ROWS if rows is None else rows, hidden.is_cuda)
    h = hidden.contiguous()
    if h.is_cuda and h.data_ptr() % 16:  # the GEMMs' loads begin on 16-byte boundaries
        h = h.clone()
    differentiated = torch.is_grad_enabled() and (h.requires_grad or weight.requires_grad)
    return _HeadTopkDistill.apply(h, weight, ids, lp, rows, float(temperature), direction, bool(tail),
                                  bool(round_dlogits), differentiated)
