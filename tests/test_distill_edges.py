"""Sampling, top-k and the distillation loss where single roundings, masks and scales decide: against 64 bits.

Log-probs and losses go by the tolerances of ``tests/test_distill_ops.py`` (fp32 roundings of log-probs of up to ~40);
where a test has larger log-probs, they add 4e-7 of the value.
"""

from __future__ import annotations

import math

import pytest
import torch

from thundersync_b200.ops.distill import lm_head_topk_distill, topk_distill_loss, topk_logprobs
from thundersync_b200.ops.sampling import sample_tokens

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _near(got: float, want: float, rtol: float = 4e-7, atol: float = 4e-6) -> bool:
    """`got` is an fp32 number: -5e38 can only be -inf there."""
    return got == float(torch.tensor(want, dtype=torch.float32)) or abs(got - want) <= atol + rtol * abs(want)


def _sample_64(z, noise, t, k=0, p=1.0, mp=0.0):
    """One row in 64 bits: (token, log-prob, whether the edge of the kept set leaves the token as it is when it moves by
    1e-5 of the mass or of a weight, which fp32 sums may do)."""
    logp = torch.log_softmax(z.double() / t, -1)
    order = z.double().sort(descending=True, stable=True)[1]
    ps = logp[order].exp()
    race = noise[order].double().log() - logp[order]  # the order of noise / p, without its underflow
    found = []
    for off in (0.0, 1e-5, -1e-5):
        kept = torch.ones_like(ps, dtype=torch.bool)
        if k > 0:
            kept[k:] = False
        if p < 1:
            kept &= ps.cumsum(0) - ps < p + off
        kept &= ps >= mp * (1 - off) * ps[0]
        kept[0] = True
        found.append(int(order[torch.where(kept, race, math.inf).argmin()]))
    return found[0], float(logp[found[0]]), len(set(found)) == 1


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


@pytest.mark.gpu
@pytest.mark.parametrize("temperature,top", [(0.05, 60.0), (0.01, 60.0), (1e-4, 60.0), (1e-4, 0.0), (1.0, 9000.0), (1.0, -2e4)])
def test_sample_top_p_of_cold_and_offset_rows(temperature, top):
    """The edge of the kept set where the scaled logits are large: the winner is kept from a top-p of the mass before it
    on, within 6e-6 (3e-6 as above, and 2^-24 of exponents of up to 40 for the rounded log2(e) / temperature)."""
    n, v = 900, 9001
    g = torch.Generator().manual_seed(2)
    z = (top + temperature * 2.5 * torch.randn(v, generator=g).double()).float()
    order = z.double().sort(descending=True, stable=True)[1]
    p = torch.softmax(z.double() / float(torch.tensor(temperature)), -1)[order]
    rank = int((p.cumsum(0) < 0.8).sum())
    mass = float(p[:rank].sum())
    noise = torch.ones(v)
    noise[order[rank]] = 1e-20  # wins where it is kept
    noise[order[0]] = 1e-6  # and this one where it is not
    top_p = (mass * (1 + torch.cat([torch.linspace(-1e-2, 1e-2, 300).double(), torch.linspace(-1e-4, 1e-4, 600).double()]))).float()
    for parts in (z.expand(n, v), z.expand(n, v)[:100]):  # rows in one part, and in several
        tok, _ = sample_tokens(parts.cuda(), noise.expand(n, v)[:len(parts)].cuda(), temperature=temperature,
                               top_p=top_p[:len(parts)].cuda())
        kept = tok.cpu() == order[rank]
        assert bool((kept | (tok.cpu() == order[0])).all())
        far = (top_p[:len(parts)].double() / mass - 1).abs() > 6e-6
        assert torch.equal(kept[far], (top_p[:len(parts)].double() > mass)[far])


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


@pytest.mark.gpu
@pytest.mark.parametrize("direction", ["forward", "reverse"])
@pytest.mark.parametrize("temperature", [1.0, 0.125])
def test_head_gradient_of_a_far_tail(direction, temperature):
    """The same through the LM head: logits of the entries are a column of the weight times the gap, exact in bf16.
    Tolerances of the bf16 head: 5e-3 of the norm, for the entries' rows of the weight gradient and for the others'."""
    n, d, v, k = len(GAPS), 64, 2056, 4
    g = torch.Generator().manual_seed(1)
    w = torch.randn(v, d, generator=g) * 0.1
    ids = torch.tensor([5, 700, 1535, v - 1])
    w[:, 0] = 0.0
    w[ids] = 0.0
    w[ids, 0] = torch.tensor([1.0, 0.984375, 0.9921875, 0.96875])
    h = torch.randn(n, d, generator=g)
    h[:, 0] = torch.tensor(GAPS)
    h = h * temperature
    w, h = w.to(torch.bfloat16), h.to(torch.bfloat16)
    ids = ids.expand(n, k).contiguous()
    lp = torch.log(torch.tensor([0.5, 0.25, 0.15, 0.05])).expand(n, k).contiguous()
    for r in range(n):  # one row at a time: each row's own part of the weight gradient
        hr, wr = h[r:r + 1].cuda().requires_grad_(True), w.cuda().requires_grad_(True)
        loss = lm_head_topk_distill(hr, wr, ids[:1].cuda(), lp[:1].cuda(), temperature=temperature,
                                    direction=direction)
        got = torch.autograd.grad(loss.sum(), (hr, wr))
        h64, w64 = h[r:r + 1].double().requires_grad_(True), w.double().requires_grad_(True)
        want = _loss_64((h64 @ w64.t())[0], ids[0], lp[0], temperature, direction)
        ref = torch.autograd.grad(want, (h64, w64))
        assert _near(float(loss.detach()), float(want.detach()), 5e-6, 3e-5), (GAPS[r], loss, want)
        outside = torch.ones(v, dtype=torch.bool)
        outside[ids[0]] = False
        for a, b in ((got[0], ref[0]), (got[1].cpu()[outside], ref[1][outside]), (got[1].cpu()[~outside], ref[1][~outside])):
            off = float((a.cpu().double() - b).norm())
            assert off <= 5e-3 * float(b.norm()) + 1e-36, (GAPS[r], off, float(b.norm()))


# ------------------------------------------------------------------ masks of finite values, offsets, cold rows
def _teacher_64(v, k, seed):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randperm(v, generator=g)[:k]
    lp = torch.log_softmax(torch.randn(k, generator=g).double(), -1) + math.log(0.9)
    return ids, lp.float()


def _check_rows(z, temperature, directions=("forward", "reverse"), settings=None):
    """topk_logprobs, sample_tokens and topk_distill_loss on rows z [N, V] against 64 bits."""
    n, v = z.shape
    host = z.cpu().double()
    t32 = float(torch.tensor(temperature))  # the kernels hold it in fp32
    k = 20
    ids, lp = topk_logprobs(z, k, temperature=temperature)
    want = host.sort(dim=-1, descending=True, stable=True)[1][:, :k]
    assert torch.equal(ids.cpu(), want)
    for i in range(n):
        ref = torch.log_softmax(host[i] / t32, -1)[want[i]]
        assert all(_near(float(a), float(b)) for a, b in zip(lp[i], ref)), (i, lp[i], ref)
    noise = torch.empty(n, v).exponential_(generator=torch.Generator().manual_seed(11))
    for kw in settings or (dict(), dict(top_k=20, top_p=0.95), dict(top_p=0.9), dict(top_k=700), dict(min_p=0.01)):
        tok, lps = sample_tokens(z, noise.to(z.device), temperature=temperature, **kw)
        for i in range(n):
            a, b, clear = _sample_64(host[i], noise[i], t32, kw.get("top_k", 0), kw.get("top_p", 1.0),
                                     kw.get("min_p", 0.0))
            assert int(tok[i]) == a or not clear, (i, kw, int(tok[i]), a)
            if int(tok[i]) == a:
                assert _near(float(lps[i]), b), (i, kw, float(lps[i]), b)
    pairs = [_teacher_64(v, 12, i) for i in range(n)]
    tid = torch.stack([a for a, _ in pairs])
    tlp = torch.stack([b for _, b in pairs])
    tid[:, 0] = host.argmax(-1)  # one likely entry, all different
    for i in range(n):
        tlp[i, 1:][tid[i, 1:] == tid[i, 0]] = -math.inf
    for direction in directions:
        x = z.detach().clone().requires_grad_(True)
        loss = topk_distill_loss(x, tid.to(z.device), tlp.to(z.device), temperature=temperature, direction=direction)
        (dz,) = torch.autograd.grad(loss.sum(), x)
        for i in range(n):
            on = tlp[i] != -math.inf
            z64 = host[i].clone().requires_grad_(True)
            ref = _loss_64(z64, tid[i][on], tlp[i][on], t32, direction)
            (dref,) = torch.autograd.grad(ref, z64)
            ref = float(ref.detach())
            assert _near(float(loss[i].detach()), ref, 2e-6, 1e-5), (i, direction, float(loss[i].detach()), ref)
            unit = 2e-5 if z.dtype == torch.float32 else 2.0 ** -8
            dref = dref.float().double()  # (1e-204 is 0 there)
            err = (dz[i].cpu().double() - dref).abs()
            # a certain row's gradient is a difference of numbers of about 8 in 64 bits, in the reference too
            allowed = 2e-5 * dref.abs().max() + unit * dref.abs() + 2.0 ** -47 / temperature
            assert bool((err <= allowed).all()), (i, direction, float((err - allowed).max()))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mask", [-1e4, -1e9, -1e10, -1e18, -1e20, -3e38])
@pytest.mark.parametrize("temperature", [1.0, 0.6, 0.3])
def test_masks_of_finite_values(device, dtype, mask, temperature):
    v = 20003
    g = torch.Generator().manual_seed(4)
    z = torch.randn(5, v, generator=g) * 2.5
    z[0, :v // 2] = mask  # every thread's first steps
    z[1] = torch.where(torch.rand(v, generator=g) < 0.95, mask, z[1])
    z[2] = mask  # a row that is nothing else: uniform
    z[3, :-1] = mask
    z[4, 1::2] = mask
    _check_rows(z.to(dtype).to(device), temperature)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masks_of_finite_values_in_several_parts(dtype):
    v = 151936
    z = torch.randn(3, v, generator=torch.Generator().manual_seed(5)) * 2.5
    z[0, :140000] = -1e10  # whole slices of the row
    z[1] = -1e9
    z[2, 7:] = -1e20
    _check_rows(z.to(dtype).cuda(), 0.6)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("offset", [1e3, -1e5, 1e6, -3e7])
def test_logits_with_an_offset(device, offset):
    z = torch.randn(3, 9001, generator=torch.Generator().manual_seed(6)) * 2.5 + offset
    _check_rows(z.to(device), 1.0)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("temperature", [0.05, 1e-2, 1e-3, 1e-4, 1e-5, 2e-6, 1.01e-6])
def test_cold_rows(device, temperature):
    """One token holds the mass, or a few that are nearly equal: its log-prob is 0 and its draws are its own."""
    g = torch.Generator().manual_seed(7)
    z = torch.randn(6, 8009, generator=g) * 2.5 + torch.tensor([0.0, 3.0, 10.0, 20.0, 30.0, -30.0])[:, None]
    z[0, 17] = 20.0
    z[4, [40, 4000, 8000]] = 60.0
    _check_rows(z.to(device), temperature, settings=(dict(), dict(top_k=20, top_p=0.95), dict(top_p=0.9),
                                                     dict(top_p=0.4), dict(min_p=0.05)))


# ------------------------------------------------------------------ the LM head's products at more shapes
def _head_shape(n, d, v, k, dtype, seed):
    """Random rows with entries at the edges of the products' tiles, some short, some without any."""
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(v, d, generator=g) * (2.5 / math.sqrt(d))).to(dtype).cuda()
    h = torch.randn(n, d, generator=g).to(dtype).cuda()
    z = h.double() @ w.double().t()
    lp, ids = torch.log_softmax(z + torch.randn(n, v, generator=g).cuda(), -1).topk(k)
    edges = torch.tensor([0, 127, 128, 255, 256, v - 1], device="cuda")
    ids[::2, -6:], lp[::2, -6:] = edges, -6.0
    for j in range(k - 6):  # (an edge that was among the others already counts once)
        ids[::2, j] = torch.where((ids[::2, j, None] == edges).any(-1), -1, ids[::2, j])
    ids[1::5, k // 2:] = -1
    ids[3::7] = -1
    lp[4::9, 1] = -math.inf
    up = torch.rand(n, generator=g).cuda()
    return h.requires_grad_(True), w.requires_grad_(True), ids, lp.float(), up


def _head_64(h, w, ids, lp, up, temperature, direction):
    """(loss, d hidden, d weight) in 64 bits, from the definition."""
    h, w = (x.detach().double().requires_grad_(True) for x in (h, w))
    logp = torch.log_softmax(h @ w.t() / temperature, -1)
    have = (ids >= 0) & (lp > -math.inf)
    t = torch.where(have, lp.double(), 0.0)
    at = ids.clamp(min=0)
    a = torch.where(have, logp.gather(-1, at), 0.0)
    weight = torch.where(have, (t if direction == "forward" else a).exp(), 0.0)
    inside = torch.zeros_like(logp, dtype=torch.bool)
    rows = torch.arange(len(ids), device=ids.device)[:, None].expand_as(ids)
    inside[rows[have], ids[have]] = True
    lpt = torch.logsumexp(logp.masked_fill(inside, -math.inf), -1)
    q = (1.0 - torch.where(have, t.exp(), 0.0).sum(-1)).clamp(min=1e-7)
    if direction == "forward":
        loss = (weight * (t - a)).sum(-1) + q * (q.log() - lpt)
    else:
        loss = (weight * (a - t)).sum(-1) + lpt.exp() * (lpt - q.log())
    loss = torch.where(have.any(-1), loss, 0.0)
    return (loss.detach(), *torch.autograd.grad(loss, (h, w), up.double()))


HEADS = [  # rows by pairs of CTAs (512, 2100, 2304, 1024) and by single ones, contractions of several chunks, odd tiles
    (300, 1032, 5008, 16), (257, 2048, 4104, 32), (512, 1000, 4104, 16), (600, 1024, 2056, 8), (2304, 264, 1032, 8),
    (2100, 520, 2056, 16), (97, 2560, 4104, 64), (40, 4096, 8200, 256), (1024, 1304, 1288, 12), (1, 2048, 12296, 8)]


@pytest.mark.gpu
@pytest.mark.parametrize("n,d,v,k", HEADS)
@pytest.mark.parametrize("direction,temperature", [("forward", 1.0), ("reverse", 1.4)])
@pytest.mark.parametrize("rounded", [False, True])
def test_head_products(n, d, v, k, direction, temperature, rounded):
    """The loss as in ``test_head_gpu``. Gradients: the dlogits' halves hold 2^-17 of them, so what counts is the rounding
    to bf16, a relative 2^-8 / sqrt(3) of a norm at most where all its values lie at the foot of their binade, and 2^-8
    for the worst value; rounded dlogits add as much again, and are held to 5e-3 as there."""
    h, w, ids, lp, up = _head_shape(n, d, v, k, torch.bfloat16, n + d)
    loss = lm_head_topk_distill(h, w, ids, lp, temperature=temperature, direction=direction, round_dlogits=rounded)
    got = torch.autograd.grad(loss, (h, w), up)
    want, *grads = _head_64(h, w, ids, lp, up, temperature, direction)
    torch.testing.assert_close(loss.detach().double(), want, rtol=5e-6, atol=3e-5)
    for a, b in zip(got, grads):
        assert a.dtype == torch.bfloat16 and a.shape == b.shape
        rel = float((a.double() - b).norm() / b.norm())
        assert rel <= (5e-3 if rounded else 2.3e-3), rel
        if not rounded:
            off, size = (a.double() - b).norm(dim=-1), b.norm(dim=-1)
            assert bool((off <= 2.0 ** -8 * size).all()), float((off / size).nan_to_num().max())
            assert not bool(a[size == 0].any())


@pytest.mark.gpu
@pytest.mark.parametrize("n,d,v,rows", [(700, 264, 2056, 256), (60, 256, 1003, 2048), (300, 1032, 1003, 128)])
@pytest.mark.parametrize("sink", [False, True])
def test_head_in_blocks_and_odd_vocabularies(n, d, v, rows, sink):
    """Several blocks, and vocabularies that are no multiple of 8, whose gradients are formed in fp32. A sink holds the
    weight gradient in fp32: 2^-17 of each dlogit, and fp32 sums."""
    from thundersync_b200.ops.sink import GradSink, ParamArena, grad_sink

    h, w, ids, lp, up = _head_shape(n, d, v, 16, torch.bfloat16, n + v)
    _, dh, dw = _head_64(h, w, ids, lp, up, 1.0, "forward")
    if not sink:
        got = torch.autograd.grad(lm_head_topk_distill(h, w, ids, lp, rows=rows), (h, w), up)
        for a, b in zip(got, (dh, dw)):
            assert float((a.double() - b).norm() / b.norm()) <= 2.3e-3
        return
    lin = torch.nn.Linear(d, v, bias=False, device="cuda", dtype=torch.bfloat16)
    lin.weight.data.copy_(w.detach())
    arena = ParamArena(list(lin.parameters()))
    into = GradSink(arena, arena.new_buffer(torch.float32))
    with grad_sink(into):
        lm_head_topk_distill(h, lin.weight, ids, lp, rows=rows).backward(up)
    assert float((into.view(lin.weight).double() - dw).norm() / dw.norm()) <= 2e-5
    assert float((h.grad.double() - dh).norm() / dh.norm()) <= 2.3e-3


@pytest.mark.gpu
def test_head_fp16():
    """Gradients rounded once to fp16: 2^-11 / sqrt(3) of the norm, and half of the least subnormal number a value."""
    h, w, ids, lp, up = _head_shape(90, 128, 1000, 16, torch.float16, 3)
    loss = lm_head_topk_distill(h, w, ids, lp)
    got = torch.autograd.grad(loss, (h, w), up)
    want, *grads = _head_64(h, w, ids, lp, up, 1.0, "forward")
    torch.testing.assert_close(loss.detach().double(), want, rtol=5e-6, atol=3e-5)
    for a, b in zip(got, grads):
        assert a.dtype == torch.float16
        allowed = 2.0 ** -11 / math.sqrt(3) * float(b.norm()) + 2.0 ** -25 * math.sqrt(b.numel())
        assert float((a.double() - b).norm()) <= allowed


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_head_cpu_rounds_gradients_once(dtype):
    h, w, ids, lp = _head_inputs(9, 40, 203, 6, "cpu", dtype)
    got = torch.autograd.grad(lm_head_topk_distill(h, w, ids, lp).sum(), (h, w))
    _, *grads = _head_64(h, w, ids, lp, torch.ones(9), 1.0, "forward")
    eps = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    for a, b in zip(got, grads):
        assert bool(((a.double() - b).abs() <= 0.51 * eps * 2 * b.abs() + 1e-6 * b.abs().max() + 2.0 ** -25).all())


# ------------------------------------------------------------------ what the LM head's node holds
def _head_inputs(n, d, v, k, device, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(v, d, generator=g) * (2.5 / math.sqrt(d))).to(dtype).to(device)
    h = torch.randn(n, d, generator=g).to(dtype).to(device)
    ids = torch.stack([torch.randperm(v, generator=g)[:k] for _ in range(n)]).to(device)
    lp = (torch.log_softmax(torch.randn(n, k, generator=g), -1) + math.log(0.9)).to(device)
    return h.requires_grad_(True), torch.nn.Parameter(w), ids, lp


@pytest.mark.gpu
def test_head_without_a_graph_holds_no_logits():
    n, v = 640, 20480
    h, w, ids, lp = _head_inputs(n, 64, v, 4, "cuda", torch.bfloat16)
    logits = 4 * n * v
    used = {}
    for name in ("graph", "no graph"):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        with torch.set_grad_enabled(name == "graph"):
            loss = lm_head_topk_distill(h, w, ids, lp)
        used[name] = torch.cuda.max_memory_allocated() - before
        assert loss.requires_grad == (name == "graph")
        del loss
    # a few numbers per row and 128 columns beside them
    assert used["graph"] >= logits and used["no graph"] <= logits // 8, used


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("change", ["weight", "hidden"])
def test_head_operands_changed_before_the_backward(device, change):
    """The backward reads hidden rows and weight again: one that has been changed in place is refused."""
    h, w, ids, lp = _head_inputs(6, 64, 104, 4, device, torch.bfloat16 if device == "cuda" else torch.float32)
    loss = lm_head_topk_distill(h, w, ids, lp)
    with torch.no_grad():
        (w if change == "weight" else h).mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.sum().backward()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows", [128, 4096])
def test_head_second_backward(device, rows):
    """A retained graph gives the same gradients again; one that was not retained says so."""
    h, w, ids, lp = _head_inputs(300, 64, 104, 4, device, torch.bfloat16 if device == "cuda" else torch.float32)
    loss = lm_head_topk_distill(h, w, ids, lp, rows=rows).sum()
    first = torch.autograd.grad(loss, (h, w), retain_graph=True)
    second = torch.autograd.grad(loss, (h, w))
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    with pytest.raises(RuntimeError, match="backward through the graph a second time"):
        torch.autograd.grad(loss, (h, w))


@pytest.mark.gpu
def test_head_graphs_share_the_room_for_logits(monkeypatch):
    """Several losses before one backward hold no more logits than one may, and their gradients do not depend on it."""
    from thundersync_b200.ops import distill

    n, v = 256, 20480
    size = 4 * n * v
    monkeypatch.setattr(distill, "KEEP_LOGITS_BYTES", 2 * size + 1000)
    h, w, ids, lp = _head_inputs(n, 64, v, 4, "cuda", torch.bfloat16)

    def six():
        return [lm_head_topk_distill(h * (1.0 + 0.25 * i), w, ids, lp) for i in range(6)]

    one = torch.autograd.grad(six()[0].sum(), (h, w))
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    losses = six()
    held = torch.cuda.memory_allocated() - before
    assert 2 * size <= held <= 2 * size + size // 2, held / size
    grads = [torch.autograd.grad(x.sum(), (h, w)) for x in losses]
    assert all(torch.equal(a, b) for a, b in zip(grads[0], one))
    monkeypatch.setattr(distill, "KEEP_LOGITS_BYTES", 0)
    for a, b in zip(grads, [torch.autograd.grad(x.sum(), (h, w)) for x in six()]):
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    del losses
    monkeypatch.setattr(distill, "KEEP_LOGITS_BYTES", 2 * size + 1000)
    losses = six()[:1]  # the others' room is free again
    assert torch.cuda.memory_allocated() - before >= size
    again = lm_head_topk_distill(h, w, ids, lp)
    assert torch.cuda.memory_allocated() - before >= 2 * size
    del losses, again


# ------------------------------------------------------------------ derivatives of derivatives
@pytest.mark.gpu
@pytest.mark.parametrize("head", [False, True])
def test_a_second_derivative_is_refused_on_cuda(head):
    """With create_graph the gradient is the same; what depends on it cannot be differentiated as if it were constant."""
    h, w, ids, lp = _head_inputs(5, 64, 104, 4, "cuda", torch.bfloat16)
    if head:
        x, loss = h, lambda: lm_head_topk_distill(h, w, ids, lp).sum()
    else:
        x = torch.randn(5, 104, device="cuda", requires_grad=True)
        loss = lambda: topk_distill_loss(x, ids, lp).sum()  # noqa: E731
    (plain,) = torch.autograd.grad(loss(), x)
    (d,) = torch.autograd.grad(loss(), x, create_graph=True)
    assert torch.equal(d, plain) and d.requires_grad
    with pytest.raises(RuntimeError, match="differentia"):
        (d.float() ** 2).sum().backward()
    # a penalty on other terms of the same graph is not in the way
    (d,) = torch.autograd.grad(loss() + (x ** 3).sum(), x, create_graph=True)
    assert torch.allclose(d.detach(), plain + 3 * x.detach() ** 2, rtol=1e-2, atol=1e-2)


def test_a_second_derivative_through_the_head_is_refused():
    h, w, ids, lp = _head_inputs(5, 64, 104, 4, "cpu", torch.float32)
    loss = lm_head_topk_distill(h, w, ids, lp).sum()
    plain = torch.autograd.grad(loss, (h, w), retain_graph=True)
    dh, dw = torch.autograd.grad(loss, (h, w), create_graph=True)
    assert torch.equal(dh, plain[0]) and torch.equal(dw, plain[1])
    with pytest.raises(RuntimeError, match="differentiable once"):
        dw.sum().backward()


def test_second_derivative_on_the_cpu():
    z = torch.randn(2, 9, dtype=torch.float64, generator=torch.Generator().manual_seed(0)).requires_grad_(True)
    ids = torch.tensor([[0, 3, 5], [8, 2, 1]])
    lp = torch.log(torch.tensor([[0.5, 0.2, 0.1], [0.3, 0.3, 0.2]]))
    assert torch.autograd.gradgradcheck(lambda x: topk_distill_loss(x, ids, lp), (z,))


# ------------------------------------------------------------------ counted launches
@pytest.mark.gpu
def test_launch_counts():
    from thundersync_b200.ops._ext import launch_counts, reset_launch_counts

    def kernels(fn):
        reset_launch_counts()
        fn()
        torch.cuda.synchronize()
        return launch_counts()["kernels"]

    h, w, ids, lp = _head_inputs(5, 64, 8 * 64 * 64, 4, "cuda", torch.bfloat16)  # a contraction that is worth slicing
    z = torch.randn(5, 300, device="cuda", requires_grad=True)
    loss = topk_distill_loss(z, ids % 300, lp)
    assert kernels(lambda: topk_distill_loss(z, ids % 300, lp)) == 1
    assert kernels(lambda: loss.sum().backward()) == 1
    head = lm_head_topk_distill(h, w, ids, lp)
    assert kernels(lambda: lm_head_topk_distill(h, w, ids, lp)) == 3  # entries, logits, the rows' end
    assert kernels(lambda: torch.autograd.grad(head.sum(), (h, w))) == 4  # dlogits, dH and the sum of its slices, dW
    h1, w1, ids1, lp1 = _head_inputs(5, 64, 1024, 4, "cuda", torch.bfloat16)  # 16 K blocks: one slice
    head = lm_head_topk_distill(h1, w1, ids1, lp1)
    assert kernels(lambda: torch.autograd.grad(head.sum(), (h1, w1))) == 3


# ------------------------------------------------------------------ a top-k that is no usual whole number
@pytest.mark.parametrize("device", DEVICES)
def test_sample_top_k_values(device):
    g = torch.Generator().manual_seed(1)
    z = (torch.randn(4, 700, generator=g) * 2).to(device)
    noise = torch.empty(4, 700).exponential_(generator=g).to(device)
    free = sample_tokens(z, noise)[0]
    for none in (0, -3, 700, 10 ** 6, 1 << 70, math.inf, -math.inf):
        assert torch.equal(sample_tokens(z, noise, top_k=none)[0], free)
    assert torch.equal(sample_tokens(z, noise, top_k=3.0)[0], sample_tokens(z, noise, top_k=3)[0])
    for bad in (2.5, math.nan):
        with pytest.raises(ValueError, match="top_k"):
            sample_tokens(z, noise, top_k=bad)
