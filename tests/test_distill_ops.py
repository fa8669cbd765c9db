"""Teacher's top entries, the distillation loss against them, and sampling: against definitions in 64 bits.

Tolerances. A log-prob is (z - m)/tau - log s: three fp32 roundings of a value up to ~40 (3 * 2^-24 * 40 = 7e-6 at
most, 4e-7 relative) and the error of log s, whose terms carry 2^-22 from the exponential and up to ~2^-23 * 30 from
its argument's scale: 4e-6 in all. The loss is a sum of such log-probs with weights that sum to one. The gradient is
a probability times coefficients of order one, relative to the row's largest entry: 2e-5, and half a unit in the last
place of the output's type on top (bf16 2^-9, fp16 2^-12, given as rtol of a whole unit).
"""

from __future__ import annotations

import math

import pytest
import torch

from thundersync_b200.ops.distill import (MAX_ENTRIES, _loss_reference, lm_head_topk_distill, topk_distill_loss,
                                          topk_logprobs)
from thundersync_b200.ops.sampling import sample_tokens

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
UNIT = {torch.float32: 2e-5, torch.bfloat16: 2 ** -8, torch.float16: 2 ** -11}


def _logits(n, v, dtype, device, seed=0, width=2.5):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(n, v, generator=g) * width
    return z.to(dtype).to(device)


def _teacher(z, k, temperature, seed=0, ragged=True):
    g = torch.Generator().manual_seed(seed)
    n, v = z.shape
    other = z.double().cpu() + torch.randn(n, v, generator=g)
    lp, ids = torch.log_softmax(other / temperature, -1).topk(k)
    if ragged:
        for i in range(0, n, 3):
            keep = int(torch.randint(0, k + 1, (1,), generator=g))
            ids[i, keep:] = -1
        if k > 2:
            lp[n // 2, 1] = -math.inf  # an entry without probability
    return ids.to(z.device), lp.float().to(z.device)


# ------------------------------------------------------------------ top-k
def _topk_64(z, k, temperature):
    z = z.double().cpu()
    ids = z.sort(dim=-1, descending=True, stable=True)[1][:, :k]
    return ids, torch.log_softmax(z / temperature, -1).gather(-1, ids)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,v,k", [(1, 1, 1), (3, 7, 7), (5, 256, 256), (2, 4099, 33), (4, 20001, 64), (300, 5003, 5),
                                   (2, 151936, 256), (1, 70000, 1)])
def test_topk_logprobs(device, dtype, n, v, k):
    z = _logits(n, v, dtype, device, seed=n + v)
    for temperature in (1.0, 0.7):
        ids, lp = topk_logprobs(z, k, temperature=temperature)
        want_ids, want = _topk_64(z, k, temperature)
        assert ids.dtype == torch.int64 and lp.dtype == torch.float32
        assert torch.equal(ids.cpu(), want_ids)
        torch.testing.assert_close(lp.cpu().double(), want, rtol=4e-7, atol=4e-6)


@pytest.mark.parametrize("device", DEVICES)
def test_topk_ties_masks_and_orders(device):
    v, k = 30011, 100
    rising = torch.arange(v, dtype=torch.float32) / 1000.0
    rows = [torch.zeros(v), rising, -rising, torch.full((v,), -math.inf),
            torch.where(torch.arange(v) % 1000 == 7, 1.0, -math.inf),  # fewer finite logits than k
            torch.full((v,), torch.finfo(torch.float32).min), torch.where(torch.arange(v) >= v - 3, 2.0, -3.4e38),
            torch.where(torch.arange(v) % 2 == 0, -0.0, 0.0), (torch.arange(v) % 17).float()]
    z = torch.stack(rows).to(device)
    ids, lp = topk_logprobs(z, k)
    want_ids, want = _topk_64(z, k, 1.0)
    assert torch.equal(ids.cpu(), want_ids)
    lp = lp.cpu().double()
    assert bool((lp[3] == -math.inf).all())
    keep = [0, 1, 2, 4, 5, 6, 7, 8]
    a, b = lp[keep], want[keep]
    assert torch.equal(a == -math.inf, b.float() == -math.inf)
    fin = (b > -1e6)
    torch.testing.assert_close(a[fin], b[fin], rtol=4e-7, atol=4e-6)


@pytest.mark.parametrize("device", DEVICES)
def test_topk_nan_rows(device):
    z = torch.zeros(3, 9000, device=device)
    z[0, 4000] = math.nan
    z[1, 8999] = math.inf
    z[2] = math.nan
    ids, lp = topk_logprobs(z, 3)
    assert bool(lp.isnan().all())
    assert ids.cpu().tolist() == [[0, 1, 2], [8999, 0, 1], [0, 1, 2]]
    few = torch.full((1, 5), math.nan, device=device)
    few[0, 3] = -math.inf
    assert topk_logprobs(few, 3)[0].cpu().tolist() == [[3, 0, 1]]


@pytest.mark.parametrize("device", DEVICES)
def test_topk_strided_rows_and_no_rows(device):
    base = _logits(6, 5000, torch.bfloat16, device)
    view = base[::2, 13:4710]
    got = topk_logprobs(view, 20)
    want = topk_logprobs(view.contiguous(), 20)
    assert torch.equal(got[0], want[0])
    torch.testing.assert_close(got[1], want[1], rtol=4e-7, atol=4e-6)
    turned = topk_logprobs(base.t().contiguous().t(), 4)
    assert torch.equal(turned[0], topk_logprobs(base, 4)[0])
    ids, lp = topk_logprobs(base[:0], 4)
    assert tuple(ids.shape) == (0, 4) and tuple(lp.shape) == (0, 4)


# ------------------------------------------------------------------ loss and gradient on logits
def _loss_64(z, ids, lp, temperature, direction, tail):
    """One row after the other, straight from the definition."""
    out = []
    for i in range(z.shape[0]):
        logp = torch.log_softmax(z[i].double() / temperature, -1)
        seen, pairs = set(), []
        for j, t in zip(ids[i].tolist(), lp[i].double().tolist()):
            if 0 <= j < z.shape[1] and t != -math.inf and j not in seen:
                seen.add(j)
                pairs.append((j, t))
        if not pairs:
            out.append(z[i].double().sum() * 0.0)
            continue
        js = torch.tensor([j for j, _ in pairs])
        t = torch.tensor([t for _, t in pairs], dtype=torch.float64)
        a = logp[js]
        loss = (t.exp() * (t - a)).sum() if direction == "forward" else (a.exp() * (a - t)).sum()
        others = torch.ones(z.shape[1], dtype=torch.bool)
        others[js] = False
        if tail and bool(others.any()):
            lpt = torch.logsumexp(logp[others], -1)
            q = max(1.0 - float(t.exp().sum()), 1e-7)
            loss = loss + (q * (math.log(q) - lpt) if direction == "forward" else lpt.exp() * (lpt - math.log(q)))
        out.append(loss)
    return torch.stack(out)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("direction", ["forward", "reverse"])
@pytest.mark.parametrize("n,v,k,temperature,tail", [(1, 9, 9, 1.0, True), (7, 1003, 1, 1.0, True), (5, 4099, 64, 0.7, True),
                                                    (6, 20001, 256, 2.0, False), (2, 151936, 100, 1.0, True)])
def test_distill_rows(device, dtype, direction, n, v, k, temperature, tail):
    z = _logits(n, v, dtype, device, seed=v).requires_grad_(True)
    ids, lp = _teacher(z.detach(), k, temperature, seed=k)
    g = torch.rand(n, generator=torch.Generator().manual_seed(1)).to(device)
    loss = topk_distill_loss(z, ids, lp, temperature=temperature, direction=direction, tail=tail)
    (dz,) = torch.autograd.grad(loss, z, g)
    assert loss.dtype == torch.float32 and dz.dtype == dtype
    z64 = z.detach().cpu().double().requires_grad_(True)
    want = _loss_64(z64, ids.cpu(), lp.cpu(), temperature, direction, tail)
    (dwant,) = torch.autograd.grad(want, z64, g.cpu().double())
    torch.testing.assert_close(loss.detach().cpu().double(), want.detach(), rtol=2e-6, atol=1e-5)
    top = dwant.abs().amax(-1, keepdim=True)
    err = (dz.cpu().double() - dwant).abs()
    allowed = 2e-5 * top + UNIT[dtype] * dwant.abs() + (2 ** -24 if dtype == torch.float16 else 0.0)
    assert bool((err <= allowed).all()), float((err - allowed).max())


@pytest.mark.parametrize("direction", ["forward", "reverse"])
@pytest.mark.parametrize("tail", [True, False])
def test_distill_gradient_by_differences(direction, tail):
    z = _logits(4, 23, torch.float64, "cpu")
    ids, lp = _teacher(z, 5, 1.3)
    fn = lambda x: topk_distill_loss(x, ids, lp.double(), temperature=1.3, direction=direction, tail=tail)  # noqa: E731
    assert torch.autograd.gradcheck(fn, (z.requires_grad_(True),), eps=1e-6, atol=1e-7, rtol=1e-6)


@pytest.mark.gpu
@pytest.mark.parametrize("direction", ["forward", "reverse"])
def test_distill_rows_gradient_by_differences_on_gpu(direction):
    # central differences of the loss along random directions, 1e-2 apart: the loss carries 1e-5 (5e-4 in the
    # quotient), the second order of a step of 1e-2 is below it
    z = _logits(3, 301, torch.float32, "cuda").requires_grad_(True)
    ids, lp = _teacher(z.detach(), 20, 1.0, ragged=False)
    (dz,) = torch.autograd.grad(topk_distill_loss(z, ids, lp, direction=direction).sum(), z)
    for seed in range(3):
        u = torch.randn(z.shape, generator=torch.Generator().manual_seed(seed)).to("cuda")
        h = 1e-2
        up = topk_distill_loss(z.detach() + h * u, ids, lp, direction=direction).double()
        down = topk_distill_loss(z.detach() - h * u, ids, lp, direction=direction).double()
        torch.testing.assert_close((up - down) / (2 * h), (dz.double() * u).sum(-1), rtol=2e-3, atol=2e-3)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("direction", ["forward", "reverse"])
def test_distill_special_rows(device, direction):
    v = 5000
    z = _logits(8, v, torch.float32, device, seed=3)
    ids, lp = _teacher(z, 8, 1.0, ragged=False)
    z[0] = math.nan  # no entries: the row is not looked at
    ids[0] = -1
    z[1, 100:] = -math.inf  # a masked vocabulary around the entries
    ids[1], lp[1] = torch.arange(8, device=device), math.log(1 / 9)
    z[2, :] = -math.inf
    z[3, 17] = math.nan
    ids[4, 3] = ids[4, 2]  # the same token twice: the first counts
    z[5, ids[5, 1]] = -math.inf  # the student cannot give an entry
    z[6, 300:] = torch.finfo(torch.float32).min
    ids[6], lp[6] = torch.arange(8, device=device), math.log(1 / 9)
    z.requires_grad_(True)
    loss = topk_distill_loss(z, ids, lp, direction=direction)
    (dz,) = torch.autograd.grad(loss[[0, 1, 4, 6, 7]].sum(), z)
    got = loss.detach().cpu().double()
    ref = _loss_64(z.detach().cpu(), ids.cpu(), lp.cpu(), 1.0, direction, True)
    assert float(got[0]) == 0.0 and math.isnan(got[2]) and math.isnan(got[3])
    for i in (1, 4, 6, 7):
        torch.testing.assert_close(got[i], ref[i], rtol=2e-6, atol=1e-5)
    assert float(got[5]) == math.inf if direction == "forward" else math.isfinite(got[5])
    assert not bool(dz[0].any()) and bool(torch.isfinite(dz[[0, 1, 4, 6, 7]]).all())
    assert not bool(dz[1, 100:].any())


@pytest.mark.parametrize("device", DEVICES)
def test_distill_whole_vocabulary_is_the_kl(device):
    # all V tokens as entries: no tail is left, and the loss is the full divergence with gradient p - q
    z = _logits(3, 200, torch.float32, device).requires_grad_(True)
    q = torch.log_softmax(_logits(3, 200, torch.float64, "cpu", seed=9), -1)
    ids = torch.arange(200, device=device).expand(3, 200)
    loss = topk_distill_loss(z, ids, q.float().to(device))
    (dz,) = torch.autograd.grad(loss.sum(), z)
    p = torch.log_softmax(z.detach().cpu().double(), -1)
    torch.testing.assert_close(loss.detach().cpu().double(), (q.exp() * (q - p)).sum(-1), rtol=2e-6, atol=1e-5)
    torch.testing.assert_close(dz.cpu().double(), p.exp() - q.exp(), rtol=0, atol=2e-5 * float(q.exp().max()))


@pytest.mark.parametrize("device", DEVICES)
def test_distill_student_nearly_certain(device):
    # the entries hold all but 1e-9 of the student's mass: the rest of it must not come out of a difference of ones
    v = 3000
    z = torch.full((1, v), -30.0, device=device)
    z[0, :4] = torch.tensor([5.0, 4.0, 3.0, 2.0], device=device)
    z.requires_grad_(True)
    ids = torch.arange(4, device=device)[None]
    lp = torch.log(torch.tensor([[0.6, 0.2, 0.1, 0.05]], device=device))
    loss = topk_distill_loss(z, ids, lp)
    (dz,) = torch.autograd.grad(loss.sum(), z)
    z64 = z.detach().cpu().double().requires_grad_(True)
    want = _loss_64(z64, ids.cpu(), lp.cpu(), 1.0, "forward", True)
    (dwant,) = torch.autograd.grad(want.sum(), z64)
    torch.testing.assert_close(loss.detach().cpu().double(), want.detach(), rtol=2e-6, atol=1e-5)
    torch.testing.assert_close(dz.cpu().double(), dwant, rtol=2e-5, atol=2e-5 * float(dwant.abs().max()))


@pytest.mark.gpu
def test_distill_rows_strided_and_other_stream():
    base = _logits(12, 6000, torch.bfloat16, "cuda")
    view = base[1::3, 5:5990].requires_grad_(True)
    ids, lp = _teacher(view.detach(), 12, 1.0)
    loss = topk_distill_loss(view, ids, lp)
    (d,) = torch.autograd.grad(loss.sum(), view)
    flat = view.detach().clone().requires_grad_(True)
    want = topk_distill_loss(flat, ids, lp)
    (dw,) = torch.autograd.grad(want.sum(), flat)
    # other slices and vectors, so other orders of summation
    torch.testing.assert_close(loss, want, rtol=2e-6, atol=1e-5)
    torch.testing.assert_close(d.float(), dw.float(), rtol=2 ** -7, atol=2e-5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = topk_distill_loss(flat, ids, lp)
        (d2,) = torch.autograd.grad(again.sum(), flat)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(again, want) and torch.equal(d2, dw)


@pytest.mark.gpu
def test_teacher_id_outside_the_vocabulary_is_recorded():
    from thundersync_b200.ops._ext import native

    native().bounds_status(True)
    z = _logits(2, 500, torch.float32, "cuda")
    ids = torch.tensor([[1, 500], [2, 3]], device="cuda")
    lp = torch.full((2, 2), math.log(0.25), device="cuda")
    got = topk_distill_loss(z, ids, lp)
    ids[0, 1] = -1
    assert native().bounds_status(True)["distill"][1] == 500
    assert torch.equal(got, topk_distill_loss(z, ids, lp))
    assert "distill" not in native().bounds_status(True)


def test_distill_refusals():
    z = torch.zeros(3, 10)
    ids, lp = torch.zeros(3, 2, dtype=torch.long), torch.zeros(3, 2)
    ok = dict(logits=z, teacher_ids=ids, teacher_logprobs=lp)
    for bad, word in [(dict(logits=z[0]), "logits"), (dict(logits=z.long()), "logits"), (dict(logits=z[:, :0]), "vocab"),
                      (dict(teacher_ids=ids[:2]), "teacher_ids"), (dict(teacher_ids=ids.float()), "integers"),
                      (dict(teacher_ids=ids[:, :0]), "teacher_ids"), (dict(teacher_logprobs=lp[:, :1]), "teacher_logprobs"),
                      (dict(teacher_logprobs=lp.long()), "teacher_logprobs"),
                      (dict(teacher_logprobs=lp.clone().requires_grad_(True)), "detached"),
                      (dict(temperature=0.0), "temperature"), (dict(temperature=math.nan), "temperature"),
                      (dict(direction="both"), "direction"),
                      (dict(teacher_ids=torch.zeros(3, MAX_ENTRIES + 1, dtype=torch.long),
                            teacher_logprobs=torch.zeros(3, MAX_ENTRIES + 1)), "teacher_ids")]:
        with pytest.raises(ValueError, match=word):
            topk_distill_loss(**{**ok, **bad})
    for k in (0, 11, MAX_ENTRIES + 1):
        with pytest.raises(ValueError, match="k must"):
            topk_logprobs(z, k)
    with pytest.raises(ValueError, match="temperature"):
        topk_logprobs(z, 2, temperature=-1.0)
    h, w = torch.zeros(3, 4), torch.zeros(10, 4)
    for args, word in [((h[0], w, ids, lp), "hidden"), ((h, w[:, :3], ids, lp), "match"),
                       ((h, w.double(), ids, lp), "dtype"), ((h, w, ids[:2], lp), "teacher_ids")]:
        with pytest.raises(ValueError, match=word):
            lm_head_topk_distill(*args)


# ------------------------------------------------------------------ loss and gradients from hidden states
@pytest.mark.parametrize("direction", ["forward", "reverse"])
@pytest.mark.parametrize("rows", [3, 2048])
def test_head_cpu(direction, rows):
    torch.manual_seed(0)
    h = torch.randn(7, 6, dtype=torch.float64, requires_grad=True)
    w = torch.randn(40, 6, dtype=torch.float64, requires_grad=True)
    ids, lp = _teacher((h @ w.t()).detach(), 5, 1.0)
    g = torch.rand(7, dtype=torch.float64)
    loss = lm_head_topk_distill(h, w, ids, lp.double(), direction=direction, rows=rows)
    got = torch.autograd.grad(loss, (h, w), g)
    want = _loss_64(h @ w.t(), ids, lp.double(), 1.0, direction, True)
    torch.testing.assert_close(loss, want)
    for a, b in zip(got, torch.autograd.grad(want, (h, w), g)):
        torch.testing.assert_close(a, b)


def _head_case(n, d, v, k, dtype, temperature, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = (torch.randn(v, d, device="cuda", generator=g) * (2.5 / math.sqrt(d))).to(dtype).requires_grad_(True)
    h = torch.randn(n, d, device="cuda", generator=g).to(dtype).requires_grad_(True)
    ids, lp = _teacher(h.detach().double() @ w.detach().double().t(), k, temperature)
    return h, w, ids, lp, torch.rand(n, device="cuda", generator=g)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("direction,tail", [("forward", True), ("reverse", True), ("forward", False)])
@pytest.mark.parametrize("n,d,v,k,temperature,rows", [(1, 64, 512, 4, 1.0, 2048), (97, 128, 5008, 33, 0.7, 2048),
                                                      (300, 256, 5003, 256, 1.0, 128), (515, 64, 12344, 16, 2.0, 256)])
def test_head_gpu(dtype, direction, tail, n, d, v, k, temperature, rows):
    """bf16: logits from fp32 accumulation (error 2^-24 sqrt(d) or so), dlogits rounded to bf16 before the products and
    the gradients rounded to bf16 again: two independent relative errors of at most 2^-9 a term, so at most 2^-8 of
    the gradient's norm, and 5e-3 covers it with what the fp32 sums add."""
    h, w, ids, lp, g = _head_case(n, d, v, k, dtype, temperature)
    loss = lm_head_topk_distill(h, w, ids, lp, temperature=temperature, direction=direction, tail=tail, rows=rows)
    got = torch.autograd.grad(loss, (h, w), g)
    h64, w64 = (x.detach().double().requires_grad_(True) for x in (h, w))
    want = _loss_reference(h64 @ w64.t(), ids, lp, temperature, direction, tail)
    torch.testing.assert_close(loss.detach().double(), want.detach(), rtol=5e-6, atol=3e-5)
    for a, b in zip(got, torch.autograd.grad(want, (h64, w64), g.double())):
        assert a.dtype == dtype
        rel = float((a.double() - b).norm() / b.norm())
        assert rel <= (5e-3 if dtype == torch.bfloat16 else 1e-4), rel


@pytest.mark.gpu
def test_head_needs_only_what_is_asked_and_honours_the_sink():
    from thundersync_b200.ops.sink import GradSink, ParamArena, grad_sink

    h, w, ids, lp, g = _head_case(130, 64, 1024, 8, torch.bfloat16, 1.0)
    full = torch.autograd.grad(lm_head_topk_distill(h, w, ids, lp), (h, w), g)
    only_h = torch.autograd.grad(lm_head_topk_distill(h, w.detach(), ids, lp), h, g)[0]
    only_w = torch.autograd.grad(lm_head_topk_distill(h.detach(), w, ids, lp), w, g)[0]
    assert torch.equal(full[0], only_h) and torch.equal(full[1], only_w)
    lin = torch.nn.Linear(64, 1024, bias=False, device="cuda", dtype=torch.bfloat16)
    lin.weight.data.copy_(w.detach())
    arena = ParamArena(list(lin.parameters()))
    sink = GradSink(arena, arena.new_buffer(torch.float32))
    with grad_sink(sink):
        lm_head_topk_distill(h, lin.weight, ids, lp).backward(g)
    got = sink.view(lin.weight)
    rel = float((got.float() - full[1].float()).norm() / full[1].float().norm())
    assert rel <= 2 ** -8, rel  # the sink is not rounded to bf16


@pytest.mark.gpu
def test_head_kept_and_computed_again_are_the_same(monkeypatch):
    from thundersync_b200.ops import distill

    h, w, ids, lp, g = _head_case(300, 128, 2056, 8, torch.bfloat16, 1.0)
    got = []
    for room in (distill.KEEP_LOGITS_BYTES, 0):
        monkeypatch.setattr(distill, "KEEP_LOGITS_BYTES", room)
        loss = lm_head_topk_distill(h, w, ids, lp)
        got.append([loss.detach(), *torch.autograd.grad(loss, (h, w), g)])
    assert all(torch.equal(a, b) for a, b in zip(*got))
    with torch.no_grad():
        assert torch.equal(lm_head_topk_distill(h, w, ids, lp), got[0][0])


# ------------------------------------------------------------------ sampling
def _sample_64(z, noise, t, k, p, mp):
    """One row: (token, log-prob) from the sorted tokens in 64 bits."""
    z = z.double()
    logp = torch.log_softmax(z / (t or 1.0), -1)
    order = z.sort(dim=-1, descending=True, stable=True)[1]
    ps = logp[order].exp()
    kept = torch.ones_like(ps, dtype=torch.bool)
    if t == 0:
        kept[1:] = False
    if k > 0:
        kept[k:] = False
    if p < 1:
        kept &= ps.cumsum(0) - ps < p
    kept &= ps >= mp * ps[0]
    kept[0] = True
    race = noise[order].double() / ps
    tok = int(order[torch.where(kept, race, math.inf).argmin()]) if t else int(order[0])
    return tok, float(logp[tok])


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.6, 20, 0.95, 0.0), (1.0, 0, 0.9, 0.0), (1.3, 0, 0.999, 0.0), (1.0, 300, 1.0, 0.0),
            (1.5, 5000, 0.99, 0.0), (1.0, 0, 1.0, 0.2), (2.0, 0, 1.0, 1e-4), (0.0, 50, 0.5, 0.1), (1.0, 1, 1.0, 0.0),
            (1.0, 256, 0.0, 0.0), (0.8, 50, 0.9, 0.05)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,v", [(1, 1), (4, 300), (3, 20001), (2, 151936), (320, 1027)])
def test_sample_tokens(device, dtype, n, v):
    z = _logits(n, v, dtype, device, seed=v)
    noise = torch.empty(n, v).exponential_(generator=torch.Generator().manual_seed(n)).to(device)
    for t, k, p, mp in SETTINGS:
        tok, lp = sample_tokens(z, noise, temperature=t, top_k=k, top_p=p, min_p=mp)
        assert tok.dtype == torch.int64 and lp.dtype == torch.float32
        for i in range(0, n, max(1, n // 16)):
            want = _sample_64(z[i].cpu(), noise[i].cpu(), t, k, p, mp)
            assert int(tok[i]) == want[0], (t, k, p, mp, i)
            assert abs(float(lp[i]) - want[1]) <= 4e-6 + 4e-7 * abs(want[1])


@pytest.mark.parametrize("device", DEVICES)
def test_sample_settings_of_each_row(device):
    n, v = len(SETTINGS), 9001
    z = _logits(n, v, torch.float32, device, seed=5)
    noise = torch.empty(n, v).exponential_(generator=torch.Generator().manual_seed(2)).to(device)
    cols = [torch.tensor(c, device=device) for c in zip(*SETTINGS)]
    tok, lp = sample_tokens(z, noise, temperature=cols[0], top_k=cols[1], top_p=cols[2], min_p=cols[3])
    for i, (t, k, p, mp) in enumerate(SETTINGS):
        p = float(torch.tensor(p))  # as fp32 holds it
        assert int(tok[i]) == _sample_64(z[i].cpu(), noise[i].cpu(), t, k, p, mp)[0], i
    one = [sample_tokens(z[i:i + 1], noise[i:i + 1], temperature=t, top_k=k, top_p=p, min_p=mp)[0]
           for i, (t, k, p, mp) in enumerate(SETTINGS)]
    assert torch.equal(tok, torch.cat(one))


@pytest.mark.parametrize("device", DEVICES)
def test_sample_flat_rows_and_ties(device):
    """Equal logits: the kept set is the lowest tokens, and the smallest exponential among them wins."""
    n, v = 6, 12000
    z = torch.zeros(n, v, device=device)
    noise = torch.empty(n, v).exponential_(generator=torch.Generator().manual_seed(3)).to(device)
    for k in (1, 3, 256, 257, 5000):
        tok, lp = sample_tokens(z, noise, top_k=k)
        assert torch.equal(tok.cpu(), noise[:, :k].argmin(-1).cpu())
        torch.testing.assert_close(lp.cpu(), torch.full((n,), -math.log(v)), rtol=4e-7, atol=4e-6)
    # a share of p that no rounding of the sum decides: 0.25 of 12000 equal tokens, half a token further
    tok, _ = sample_tokens(z, noise, top_p=(3000 - 0.5) / v)
    assert torch.equal(tok.cpu(), noise[:, :3000].argmin(-1).cpu())


@pytest.mark.parametrize("device", DEVICES)
def test_sample_masked_and_broken_rows(device):
    v = 7000
    z = torch.full((8, v), -math.inf, device=device)
    z[0, 4321] = 2.0  # one token left
    z[1, [5, 6000]] = torch.tensor([1.0, 1.5], device=device)
    z[3] = 0.0
    z[3, 77] = math.nan
    z[4] = 0.0
    z[4, 78] = math.inf
    z[5] = torch.finfo(torch.float32).min  # masked with the type's lowest value, all but one
    z[5, 123] = -4.0
    z[6] = torch.finfo(torch.float32).min  # all of it: equal tokens
    z[7] = math.nan
    noise = torch.ones(8, v, device=device)
    noise[1, 6000], noise[6, 99] = 100.0, 0.5
    for kw in (dict(), dict(top_k=20, top_p=0.95), dict(top_p=0.99), dict(top_k=1000), dict(min_p=0.01)):
        tok, lp = sample_tokens(z, noise, **kw)
        tok, lp = tok.cpu().tolist(), lp.cpu()
        assert tok[0] == 4321 and abs(float(lp[0])) <= 4e-6
        assert tok[1] == 5
        assert [tok[i] for i in (2, 3, 4, 7)] == [-1] * 4
        assert all(math.isnan(lp[i]) for i in (2, 3, 4, 7))
        assert tok[5] == 123
        assert tok[6] == (0 if kw.get("top_k") == 20 else 99)
    greedy, _ = sample_tokens(z, None, temperature=0.0)
    assert greedy.cpu().tolist() == [4321, 6000, -1, -1, -1, 123, 0, -1]


@pytest.mark.parametrize("device", DEVICES)
def test_sample_with_numbers_that_are_not_random(device):
    """Falling numbers put the best key on the last-ranked token each time: the kept set must not be found one token a
    pass. Distinct logits, so that ranks are the tokens' order, in both directions."""
    n, v = 2, 12000
    noise = torch.linspace(2.0, 1.0, v, device=device).expand(n, v).contiguous()
    flat = torch.zeros(n, v, device=device)
    slope = torch.stack([-torch.arange(v), torch.arange(v)]).to(device) * 2.0 ** -26  # hardly any slope
    for z in (flat, flat + 1.0 + slope):
        tok, _ = sample_tokens(z, noise, top_k=300)
        first = z.cpu().sort(dim=-1, descending=True, stable=True)[1][:, :300]
        want = first.gather(-1, noise.cpu().gather(-1, first).argmin(-1, keepdim=True)).squeeze(-1)
        assert torch.equal(tok.cpu(), want)
    # half a token past a quarter of the mass: 3000 tokens
    tok, _ = sample_tokens(flat, noise, top_p=(3000 - 0.5) / v)
    assert tok.cpu().tolist() == [2999, 2999]


@pytest.mark.gpu
def test_sample_numbers_that_are_none():
    z = _logits(3, 9000, torch.float32, "cuda")
    nan = torch.full((3, 9000), math.nan, device="cuda")
    for kw in (dict(), dict(top_k=20), dict(top_p=0.5), dict(top_k=1000, min_p=0.1)):
        assert torch.equal(sample_tokens(z, nan, **kw)[0], z.argmax(-1))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_topk_crowded_groups(dtype):
    """Far more large logits than k, all in a few threads' vectors, so that the groups that are read again hold more
    candidates than there is room for; and rows whose k-th largest lies among them or below them."""
    n, v = 230, 151936
    z = torch.randn(n, v, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    i = torch.arange(v, device="cuda")
    per = 4 if dtype == torch.float32 else 8
    crowd = ((i // per) % 256 < 200) & (i < 12288)
    z = torch.where(crowd, 20.0 + z, z).to(dtype)
    for k in (64, 200, 256):
        ids, _ = topk_logprobs(z, k)
        for r in range(0, n, 37):
            want = z[r].float().sort(descending=True, stable=True)[1][:k]
            assert torch.equal(ids[r], want), (k, r)


@pytest.mark.gpu
def test_sample_strided_and_repeatable():
    base = _logits(9, 8000, torch.float16, "cuda")
    nb = torch.empty(9, 9001, device="cuda").exponential_()
    z, noise = base[::2, 3:7777], nb[::2, 1:7775]
    for kw in (dict(), dict(top_p=0.9), dict(top_k=40), dict(top_p=0.9995, temperature=1.4)):
        a = sample_tokens(z, noise, **kw)
        b = sample_tokens(z.contiguous(), noise.contiguous(), **kw)
        c = sample_tokens(z, noise, **kw)
        assert torch.equal(a[0], b[0]) and torch.equal(a[0], c[0]) and torch.equal(a[1], c[1])
    tok, lp = sample_tokens(base[:0], nb[:0, :8000])
    assert tok.numel() == 0 and lp.numel() == 0


def test_sample_distribution():
    """The draws follow the restricted softmax: with 20000 of them a frequency is within five deviations."""
    n, v = 20000, 6
    z = torch.tensor([2.0, 1.0, 0.5, 0.0, -1.0, -3.0]).expand(n, v).contiguous()
    noise = torch.empty(n, v).exponential_(generator=torch.Generator().manual_seed(7))
    tok, _ = sample_tokens(z, noise, top_k=4)
    p = torch.softmax(z[0, :4], -1)
    freq = torch.bincount(tok, minlength=v)[:4] / n
    assert bool(((freq - p).abs() <= 5 * (p * (1 - p) / n).sqrt()).all()) and int(tok.max()) < 4


def test_sample_refusals():
    z, e = torch.zeros(3, 10), torch.ones(3, 10)
    for args, kw, word in [((z[0], e), {}, "logits"), ((z.long(), e), {}, "logits"), ((z, e[:, :5]), {}, "noise"),
                           ((z, e.double()), {}, "noise"), ((z, None), {}, "noise"),
                           ((z, e), dict(temperature=-1.0), "temperature"), ((z, e), dict(top_p=-0.1), "top_p"),
                           ((z, e), dict(min_p=1.5), "min_p"), ((z, e), dict(top_p=math.nan), "top_p"),
                           ((z, e), dict(top_k=torch.ones(2, dtype=torch.long)), "top_k"),
                           ((z, None), dict(temperature=torch.zeros(3)), "noise")]:
        with pytest.raises(ValueError, match=word):
            sample_tokens(*args, **kw)
