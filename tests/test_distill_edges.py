"""Sampling, top-k and the distillation loss where single roundings, masks and scales decide: against 64 bits.

Log-probs and losses go by the tolerances of ``tests/test_distill_ops.py`` (fp32 roundings of log-probs of up to ~40);
where a test has larger log-probs, they add 4e-7 of the value.
"""

from __future__ import annotations

import math

import pytest
import torch

from thundersync_b200.ops.sampling import sample_tokens


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
