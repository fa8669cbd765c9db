"""Sampling, top-k and the distillation loss where single roundings, masks and scales decide: against 64 bits.

Log-probs and losses go by the tolerances of ``tests/test_distill_ops.py`` (fp32 roundings of log-probs of up to ~40);
where a test has larger log-probs, they add 4e-7 of the value.
"""

from __future__ import annotations

import math

import pytest
import torch

from thundersync_b200.ops.distill import topk_distill_loss
from thundersync_b200.ops.sampling import sample_tokens

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _near(got: float, want: float, rtol: float = 4e-7, atol: float = 4e-6) -> bool:
    return got == want or abs(got - want) <= atol + rtol * abs(want)


def _loss_64(z, ids, lp, temperature, direction):
    """One row from the definition, with the tail where its mass is not 0 in 64 bits."""
    logp = torch.log_softmax(z / temperature, -1)
    a, t = logp[ids], lp.double()
    rest = torch.ones_like(z, dtype=torch.bool)
    rest[ids] = False
    lpt = torch.logsumexp(logp[rest], -1)
    q = max(1.0 - float(t.exp().sum()), 1e-7)
    if direction == "forward":
        loss, more = (t.exp() * (t - a)).sum(), q * (math.log(q) - lpt)
    else:
        loss, more = (a.exp() * (a - t)).sum(), lpt.exp() * (lpt - math.log(q))
    return loss + more if float(lpt.detach().exp()) > 0 else loss


# ------------------------------------------------------------------ top-p at the edge of a token's mass
@pytest.mark.gpu
@pytest.mark.parametrize("n,v,width", [(1300, 32000, 2.5), (700, 40000, 3.5), (140, 32000, 1.5), (400, 20001, 2.5)])
def test_sample_top_p_one_rounding_apart(n, v, width):
    """Equal rows, and a top-p of each that is one unit in the last place past its neighbour's, around the mass before
    the race's winner. All threads of a row have to come to one answer; the answer changes once, from the second to the
    winner, within what fp32 sums of positive terms carry (a relative 2^-24 * 2 for each of about 17 levels of adding
    and 2^-22 for each exponential: 3e-6)."""
    g = torch.Generator().manual_seed(v + n)
    z = torch.randn(v, generator=g) * width
    order = z.double().sort(descending=True, stable=True)[1]
    p = torch.softmax(z.double(), -1)[order]
    rank = int((p.cumsum(0) < 0.8).sum())
    mass = float(p[:rank].sum())
    noise = torch.ones(v)
    noise[order[rank]] = 1e-20  # wins where it is kept
    noise[order[0]] = 1e-6  # and this one where it is not
    p0 = torch.tensor(mass, dtype=torch.float32).view(torch.int32)
    top_p = (p0 + torch.arange(-(n // 2), n - n // 2, dtype=torch.int32)).view(torch.float32)
    top_p[0], top_p[-1] = mass * (1 - 1e-4), mass * (1 + 1e-4)
    for dtype in (torch.float32, torch.bfloat16):
        zd = z.to(dtype)
        if dtype == torch.bfloat16:  # other logits: another order and mass; any top-p will do
            assert set(sample_tokens(zd.expand(n, v).cuda(), noise.expand(n, v).cuda(), top_p=top_p.cuda())[0]
                       .tolist()) <= {int(order[0]), int(order[rank])}
            continue
        tok, _ = sample_tokens(zd.expand(n, v).cuda(), noise.expand(n, v).cuda(), top_p=top_p.cuda())
        kept = (tok.cpu() == order[rank])
        assert bool((kept | (tok.cpu() == order[0])).all())
        assert not bool(kept[0]) and bool(kept[-1])
        inner = kept[1:-1].int()
        assert bool((inner.diff() >= 0).all())
        far = (top_p.double() / mass - 1).abs() > 3e-6
        assert torch.equal(kept[far], (top_p.double() > mass)[far])


def _sample_rows_64(z, noise, top_p):
    """(tokens, whether the kept set is clear of the rounding of sums) of rows at temperature 1, on their device."""
    zd = z.double()
    order = zd.sort(dim=-1, descending=True, stable=True)[1]
    p = torch.softmax(zd, -1).gather(-1, order)
    before = p.cumsum(-1) - p
    kept = before < top_p
    kept[:, 0] = True
    race = torch.where(kept, noise.double().gather(-1, order) / p, math.inf)
    # the winner among twice the kept tokens: where it is the same, the edge of the set does not decide
    wide = torch.where(before < top_p + 1e-5, noise.double().gather(-1, order) / p, math.inf)
    narrow = torch.where((before < top_p - 1e-5) | (torch.arange(z.shape[1], device=z.device) == 0),
                         noise.double().gather(-1, order) / p, math.inf)
    at = race.argmin(-1)
    clear = (wide.argmin(-1) == at) & (narrow.argmin(-1) == at)
    return order.gather(-1, at[:, None]).squeeze(-1), clear


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,v,top_p", [(600, 32000, 0.9), (1300, 32000, 0.5), (60, 32000, 0.95), (1300, 50257, 0.9)])
def test_sample_top_p_rows_in_one_part(dtype, n, v, top_p):
    g = torch.Generator(device="cuda").manual_seed(n + v)
    z = (torch.randn(n, v, generator=g, device="cuda") * (1.5 + 2 * torch.rand(n, 1, generator=g, device="cuda"))).to(dtype)
    noise = torch.empty(n, v, device="cuda").exponential_(generator=g)
    tok, _ = sample_tokens(z, noise, top_p=top_p)
    settings = torch.full((n,), top_p, device="cuda")
    again, _ = sample_tokens(z, noise, top_p=settings)
    p = float(torch.tensor(top_p))  # as fp32 holds it
    for r0 in range(0, n, 200):
        want, clear = _sample_rows_64(z[r0:r0 + 200], noise[r0:r0 + 200], p)
        assert int(clear.sum()) >= 0.95 * len(want)
        assert torch.equal(tok[r0:r0 + 200][clear], want[clear])
        assert torch.equal(again[r0:r0 + 200][clear], want[clear])


# ------------------------------------------------------------------ students that give the other tokens next to nothing
GAPS = [30.0, 80.0, 85.0, 88.0, 95.0, 100.0, 300.0, 700.0, 800.0, 1e4]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("direction", ["forward", "reverse"])
@pytest.mark.parametrize("temperature", [1.0, 0.1])
def test_gradient_of_a_far_tail(device, dtype, direction, temperature):
    """Logits outside the entries lie `gap` nats below: their gradient is about Q in all, as long as their mass is not 0
    in 64 bits; on the CPU as in the kernels."""
    n, v, k = len(GAPS), 3001, 4
    g = torch.Generator().manual_seed(0)
    z = torch.randn(n, v, generator=g) * temperature - torch.tensor(GAPS)[:, None] * temperature
    ids = torch.tensor([5, 700, 2047, 3000]).expand(n, k).contiguous()
    z[:, ids[0]] = torch.tensor([0.0, -1.0, -0.5, -2.0]) * temperature
    z = z.to(dtype)
    lp = torch.log(torch.tensor([0.5, 0.25, 0.15, 0.05])).expand(n, k).contiguous()
    x = z.to(device).requires_grad_(True)
    loss = topk_distill_loss(x, ids.to(device), lp.to(device), temperature=temperature, direction=direction)
    (dz,) = torch.autograd.grad(loss.sum(), x)
    outside = torch.ones(v, dtype=torch.bool)
    outside[ids[0]] = False
    t32 = float(torch.tensor(temperature))
    for i in range(n):
        z64 = z[i].double().requires_grad_(True)
        want = _loss_64(z64, ids[i], lp[i], t32, direction)
        (dwant,) = torch.autograd.grad(want, z64)
        assert _near(float(loss[i].detach()), float(want.detach()), 2e-6, 1e-5), (GAPS[i], loss[i], want)
        got = dz[i].double().cpu()
        unit = 2e-5 if dtype == torch.float32 else 2.0 ** -8
        for part in (outside, ~outside):  # each against its own largest
            err = (got[part] - dwant[part]).abs()
            allowed = 2e-5 * dwant[part].abs().max() + unit * dwant[part].abs() + 1e-37
            assert bool((err <= allowed).all()), (GAPS[i], float((err - allowed).max()))
