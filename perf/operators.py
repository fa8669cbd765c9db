"""Cases of the on-policy distillation operators: a teacher's top logits, the loss against them, and sampling.

Four calls are covered, in the order a distillation step makes them:

``sample``  draw the next token of each sequence from logits [B, V] (temperature, top-k, top-p, min-p) with given
            exponential random numbers, and return its log-probability
``topk``    a teacher's k largest logits per row, as token ids and log-probabilities
``rows``    the distillation loss of student logits [N, V] against a teacher's top entries, and the logits' gradient
``head``    the same loss from hidden states and LM-head weight, and the gradients of both

Inputs are random with the shape of language-model outputs: a row's logits are normal with a width of 1.5 to 3.5
(from thousands of likely tokens down to a handful), and the teacher is the student plus noise.
"""

from __future__ import annotations

import math

import torch

own = False

_FLOAT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # one packed turn of scored tokens through a 151,936-token head: the ordinary training call
        {"name": "head_pack_2048", "op": "head", "n": 2048, "d": 2048, "v": 151936, "k": 64, "direction": "forward",
         "tail": True, "temperature": 1.0, "ragged": False},
        # one short action of one trajectory, scored as soon as it exists (a wider model): bound by the weight
        {"name": "head_action_97", "op": "head", "n": 97, "d": 2560, "v": 151936, "k": 16, "direction": "reverse",
         "tail": True, "temperature": 1.0, "ragged": True},
        # a long trajectory's close, in several row blocks; the teacher's entries as plain partial sums
        {"name": "head_close_4096", "op": "head", "n": 4096, "d": 2048, "v": 151936, "k": 32, "direction": "forward",
         "tail": False, "temperature": 2.0, "ragged": True},
        # logits already in memory, half precision
        {"name": "rows_bf16_1000", "op": "rows", "n": 1000, "v": 151936, "dtype": "bf16", "k": 64,
         "direction": "forward", "tail": True, "temperature": 1.0, "ragged": False},
        # a few rows of fp32 logits with many teacher entries, some rows short or empty
        {"name": "rows_fp32_33", "op": "rows", "n": 33, "v": 151936, "dtype": "fp32", "k": 128,
         "direction": "reverse", "tail": True, "temperature": 1.5, "ragged": True},
        # a teacher's scores for a whole pack
        {"name": "topk_pack_2048", "op": "topk", "n": 2048, "v": 151936, "dtype": "fp32", "k": 64,
         "temperature": 1.0},
        # an odd vocabulary: no row but the first begins on a 16-byte boundary; half precision has many equal logits
        {"name": "topk_odd_517", "op": "topk", "n": 517, "v": 50257, "dtype": "bf16", "k": 20, "temperature": 1.0},
        # one token's scores: latency
        {"name": "topk_one", "op": "topk", "n": 1, "v": 151936, "dtype": "fp32", "k": 8, "temperature": 1.0},
        # one sequence, nucleus only: latency
        {"name": "sample_one", "op": "sample", "n": 1, "v": 151936, "dtype": "fp32", "temperature": 1.0, "top_k": 0,
         "top_p": 0.9, "min_p": 0.0, "per_row": False},
        # a serving batch with the usual reasoning settings
        {"name": "sample_serve_64", "op": "sample", "n": 64, "v": 151936, "dtype": "bf16", "temperature": 0.6,
         "top_k": 20, "top_p": 0.95, "min_p": 0.0, "per_row": False},
        # on-policy rollouts: the untruncated distribution
        {"name": "sample_policy_512", "op": "sample", "n": 512, "v": 151936, "dtype": "fp32", "temperature": 1.0,
         "top_k": 0, "top_p": 1.0, "min_p": 0.0, "per_row": False},
        # requests with settings of their own, some greedy
        {"name": "sample_mixed_200", "op": "sample", "n": 200, "v": 151936, "dtype": "bf16", "temperature": 0.8,
         "top_k": 50, "top_p": 0.9, "min_p": 0.05, "per_row": True},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["head", "rows", "topk", "sample"])
    if op == "head":
        v = rng.choice([32000, 50304, 128256, 151936])
        d = rng.choice([1024, 2048, 2560, 4096])
        most = min(4096, 4096 * 2048 * 151936 // (d * v))
        return {"op": op, "n": _log_int(rng, 1, most), "d": d, "v": v, "k": _log_int(rng, 4, 128),
                "direction": rng.choice(["forward", "reverse"]), "tail": rng.random() < 0.75,
                "temperature": rng.choice([1.0, 1.0, 2.0]), "ragged": rng.random() < 0.5}
    v = rng.choice([32000, 50257, 128256, 151936, 248320, rng.randrange(1000, 160001)])
    dtype = rng.choice(["bf16", "fp32", "fp32", "fp16"])
    case = {"op": op, "n": _log_int(rng, 1, min(2048, 2048 * 151936 // v // (2 if op == "rows" else 1))), "v": v,
            "dtype": dtype}
    if op == "rows":
        case |= {"k": _log_int(rng, 4, 256), "direction": rng.choice(["forward", "reverse"]),
                 "tail": rng.random() < 0.75, "temperature": rng.choice([1.0, 1.0, 0.7, 2.0]),
                 "ragged": rng.random() < 0.5}
    elif op == "topk":
        case |= {"k": _log_int(rng, 1, 256), "temperature": rng.choice([1.0, 1.0, 0.7, 2.0])}
    else:
        case["n"] = min(case["n"], 512)
        case |= {"temperature": rng.choice([1.0, 0.6, 0.8, 1.3]), "top_k": rng.choice([0, 0, 20, 50, 200, 2000]),
                 "top_p": rng.choice([1.0, 0.95, 0.9, 0.5]), "min_p": rng.choice([0.0, 0.0, 0.05]),
                 "per_row": rng.random() < 0.4}
    return case


def _logits(case, g):
    n, v = case["n"], case["v"]
    width = 1.5 + 2.0 * torch.rand(n, 1, device="cuda", generator=g)
    return torch.randn(n, v, device="cuda", generator=g).mul_(width)


def _teacher(z, k, temperature, ragged, g):
    """The k largest entries of teacher logits z, as (ids, log-probs); short rows end in id -1."""
    n = z.shape[0]
    top, ids = z.topk(k, dim=-1)
    lp = top / temperature - torch.logsumexp(z / temperature, -1, keepdim=True)
    if ragged:
        length = torch.randint(0, k + 1, (n, 1), device="cuda", generator=g)
        length = torch.where(torch.rand(n, 1, device="cuda", generator=g) < 0.5, length.new_tensor(k), length)
        off = torch.arange(k, device="cuda") >= length
        ids, lp = ids.masked_fill(off, -1), lp.masked_fill(off, -math.inf)
    return ids, lp


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    state = {"case": dict(case)}
    if op == "head":
        n, d, v, k = case["n"], case["d"], case["v"], case["k"]
        weight = torch.randn(v, d, device="cuda", generator=g).mul_(2.5 / math.sqrt(d)).to(torch.bfloat16)
        hidden = torch.randn(n, d, device="cuda", generator=g)
        other = (hidden + 0.4 * torch.randn(n, d, device="cuda", generator=g)).to(torch.bfloat16)
        parts = [_teacher(torch.mm(o, weight.t()).float(), k, case["temperature"], case["ragged"], g)
                 for o in other.split(1024)]
        state["ids"], state["lp"] = (torch.cat(p) for p in zip(*parts))
        state["hidden"] = hidden.to(torch.bfloat16).requires_grad_(True)
        state["weight"] = weight.requires_grad_(True)
        state["grad"] = torch.rand(n, device="cuda", generator=g)  # token weights
        return state
    z = _logits(case, g)
    if op == "rows":
        other = z + 0.7 * torch.randn(z.shape, device="cuda", generator=g)
        state["ids"], state["lp"] = _teacher(other, case["k"], case["temperature"], case["ragged"], g)
        del other
        state["grad"] = torch.rand(case["n"], device="cuda", generator=g)
    state["logits"] = z.to(_FLOAT[case["dtype"]])
    if op == "rows":
        state["logits"].requires_grad_(True)
    if op == "sample":
        n = case["n"]
        state["noise"] = torch.empty(n, case["v"], device="cuda").exponential_(generator=g)
        if case["per_row"]:  # a quarter of the rows greedy, the others around the case's settings, some without a filter
            u = torch.rand(4, n, device="cuda", generator=g)
            state["temperature"] = torch.where(u[0] < 0.25, 0.0, case["temperature"] * (0.75 + 0.5 * u[0]))
            state["top_k"] = torch.where(u[1] < 0.3, 0, case["top_k"])
            state["top_p"] = torch.where(u[2] < 0.3, 1.0, case["top_p"])
            state["min_p"] = torch.where(u[3] < 0.3, 0.0, case["min_p"])
        else:
            for name in ("temperature", "top_k", "top_p", "min_p"):
                state[name] = case[name]
    return state


# ---------------------------------------------------------------- plain forms
def _plain_loss(z, ids, lp, temperature, direction, tail):
    """(loss [N], d loss / d z [N, V]) for fp32 logits z."""
    a = z / temperature
    m = a.amax(-1, keepdim=True)
    e = torch.exp(a - m)
    s = e.sum(-1, keepdim=True)
    p = e / s
    have = (ids >= 0) & (lp > -math.inf)
    at = ids.clamp(min=0)
    t = torch.where(have, lp, 0.0)
    q = torch.where(have, torch.exp(t), 0.0)
    pk = torch.where(have, p.gather(-1, at), 0.0)
    ak = torch.where(have, a.gather(-1, at) - m - torch.log(s), 0.0)
    inside = torch.zeros_like(p).scatter_add_(-1, at, have.to(p.dtype))
    if tail:
        pt = torch.where(inside > 0, 0.0, p).sum(-1, keepdim=True)
        qt = (1.0 - q.sum(-1, keepdim=True)).clamp(min=1e-7)
        some = have.any(-1, keepdim=True) & (pt > 0)
        lpt, lqt = torch.log(torch.where(some, pt, 1.0)), torch.log(qt)
        pt = torch.where(some, pt, 1.0)
    if direction == "forward":
        loss = (q * (t - ak)).sum(-1)
        g = -q
        if tail:
            loss = loss + torch.where(some, qt * (lqt - lpt), 0.0).squeeze(-1)
            g = g + torch.where(some, qt * pk / pt, 0.0)
    else:
        loss = (pk * (ak - t)).sum(-1)
        g = pk * (ak - t + 1.0)
        if tail:
            loss = loss + torch.where(some, pt * (lpt - lqt), 0.0).squeeze(-1)
            g = g - torch.where(some, pk * (lpt - lqt + 1.0), 0.0)
    g = torch.where(have, g, 0.0)
    d = torch.zeros_like(p).scatter_add_(-1, at, g) - g.sum(-1, keepdim=True) * p
    return loss, d / temperature


def _plain(state):
    case = state["case"]
    op = case["op"]
    with torch.no_grad():
        if op == "head":
            h, w = state["hidden"].float(), state["weight"].float()
            loss, dz = _plain_loss(h @ w.t(), state["ids"], state["lp"], case["temperature"], case["direction"],
                                   case["tail"])
            dz = dz * state["grad"][:, None]
            return {"loss": loss, "d_hidden": (dz @ w).to(torch.bfloat16), "d_weight": (dz.t() @ h).to(torch.bfloat16)}
        z = state["logits"].float()
        if op == "rows":
            loss, dz = _plain_loss(z, state["ids"], state["lp"], case["temperature"], case["direction"], case["tail"])
            return {"loss": loss, "d_logits": (dz * state["grad"][:, None]).to(state["logits"].dtype)}
        if op == "topk":
            m = z.amax(-1, keepdim=True)
            t = case["temperature"]
            s = torch.exp((z - m) / t).sum(-1, keepdim=True)
            top, ids = z.sort(dim=-1, descending=True, stable=True)
            top, ids = top[:, :case["k"]], ids[:, :case["k"]].contiguous()
            return {"ids": ids, "logprobs": (top - m) / t - torch.log(s)}
        n, v = z.shape
        row = [torch.as_tensor(state[x], device=z.device).expand(n)[:, None] for x in
               ("temperature", "top_k", "top_p", "min_p")]
        t, top_k, top_p, min_p = row[0].float(), row[1], row[2].float(), row[3].float()
        greedy = t == 0
        m = z.amax(-1, keepdim=True)
        a = (z - m) / torch.where(greedy, 1.0, t)
        w = torch.exp(a)
        s = w.sum(-1, keepdim=True)
        key = w / state["noise"]
        if case["top_k"] > 0 or case["top_p"] < 1 or case["min_p"] > 0:
            order = z.sort(dim=-1, descending=True, stable=True)[1]  # equal logits: the lower token first
            ws = w.gather(-1, order)
            before = ws.cumsum(-1) - ws
            rank = torch.arange(v, device=z.device)[None]
            keep = ((top_k <= 0) | (rank < top_k)) & ((top_p >= 1) | (before < top_p * s)) & (ws >= min_p)
            keep |= rank == 0
            key = torch.where(torch.zeros_like(keep).scatter_(-1, order, keep), key, -1.0)
        tok = torch.where(greedy[:, 0], z.argmax(-1), key.argmax(-1))
        return {"tokens": tok, "logprobs": (a.gather(-1, tok[:, None]) - torch.log(s)).squeeze(-1)}


def _own(state):
    from thundersync_b200.ops.distill import lm_head_topk_distill, topk_distill_loss, topk_logprobs
    from thundersync_b200.ops.sampling import sample_tokens

    case = state["case"]
    op = case["op"]
    if op == "head":
        loss = lm_head_topk_distill(state["hidden"], state["weight"], state["ids"], state["lp"],
                                    temperature=case["temperature"], direction=case["direction"], tail=case["tail"])
        dh, dw = torch.autograd.grad(loss, (state["hidden"], state["weight"]), state["grad"])
        return {"loss": loss.detach(), "d_hidden": dh, "d_weight": dw}
    if op == "rows":
        loss = topk_distill_loss(state["logits"], state["ids"], state["lp"], temperature=case["temperature"],
                                 direction=case["direction"], tail=case["tail"])
        (dz,) = torch.autograd.grad(loss, (state["logits"],), state["grad"])
        return {"loss": loss.detach(), "d_logits": dz}
    if op == "topk":
        ids, lp = topk_logprobs(state["logits"], case["k"], temperature=case["temperature"])
        return {"ids": ids, "logprobs": lp}
    tok, lp = sample_tokens(state["logits"], state["noise"], temperature=state["temperature"], top_k=state["top_k"],
                            top_p=state["top_p"], min_p=state["min_p"])
    return {"tokens": tok, "logprobs": lp}


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    n, v = case["n"], case["v"]
    if case["op"] == "head":
        # logits, d_hidden and d_weight: three products; hidden and weight in, their gradients out
        d, k = case["d"], case["k"]
        return {"bytes": 4 * n * d + 4 * v * d + 12 * n * k + 8 * n, "flops": 6 * n * v * d}
    size = _SIZE[case["dtype"]]
    if case["op"] == "rows":
        return {"bytes": 2 * n * v * size + 12 * n * case["k"] + 8 * n, "flops": 6 * n * v}
    if case["op"] == "topk":
        return {"bytes": n * v * size + 12 * n * case["k"], "flops": 4 * n * v}
    # the random numbers of tokens that a filter takes out are not needed: all of them without a filter, else few
    free = case["top_k"] == 0 and case["top_p"] >= 1 and case["min_p"] == 0
    return {"bytes": n * v * (size + (4 if free else 0)) + 12 * n, "flops": 4 * n * v}


# ---------------------------------------------------------------- the definition, in 64 bits
def _exact_loss(z, ids, lp, temperature, direction, tail):
    logp = torch.log_softmax(z / temperature, -1)
    have = (ids >= 0) & torch.isfinite(lp)
    at = ids.clamp(min=0)
    t = torch.where(have, lp.double(), 0.0)
    ak = logp.gather(-1, at)
    rest = torch.ones_like(z, dtype=torch.bool)
    rows = torch.arange(z.shape[0], device=z.device)[:, None].expand_as(ids)
    rest[rows[have], ids[have]] = False
    lpt = torch.logsumexp(logp.masked_fill(~rest, -math.inf), -1)
    qt = (1.0 - (t.exp() * have).sum(-1)).clamp(min=1e-7)
    some = have.any(-1) & (lpt > -math.inf)
    if direction == "forward":
        loss = torch.where(have, t.exp() * (t - ak), 0.0).sum(-1)
        more = qt * (qt.log() - lpt)
    else:
        loss = torch.where(have, ak.exp() * (ak - t), 0.0).sum(-1)
        more = lpt.exp() * (lpt - qt.log())
    return loss + torch.where(some, more, 0.0) if tail else loss


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    how = (case.get("temperature"), case.get("direction"), case.get("tail"))
    if op == "head":
        w = state["weight"].detach().double()
        loss, dh, dw = [], [], torch.zeros_like(w)
        for i in range(0, case["n"], 512):
            j = min(case["n"], i + 512)
            h = state["hidden"].detach()[i:j].double()
            z = (h @ w.t()).requires_grad_(True)
            part = _exact_loss(z, state["ids"][i:j], state["lp"][i:j], *how)
            (dz,) = torch.autograd.grad(part, z, state["grad"][i:j].double())
            loss.append(part.detach())
            dh.append(dz @ w)
            dw.addmm_(dz.t(), h)
        return {"loss": torch.cat(loss), "d_hidden": torch.cat(dh), "d_weight": dw}
    logits = state["logits"].detach()
    if op == "rows":
        loss, grad = [], []
        for i in range(0, case["n"], 256):
            j = min(case["n"], i + 256)
            z = logits[i:j].double().requires_grad_(True)
            part = _exact_loss(z, state["ids"][i:j], state["lp"][i:j], *how)
            grad.append(torch.autograd.grad(part, z, state["grad"][i:j].double())[0])
            loss.append(part.detach())
        return {"loss": torch.cat(loss), "d_logits": torch.cat(grad)}
    if op == "topk":
        ids, lps = [], []
        for z in logits.split(256):
            z = z.double()
            order = torch.argsort(z, dim=-1, descending=True, stable=True)[:, :case["k"]]
            ids.append(order)
            lps.append(torch.log_softmax(z / case["temperature"], -1).gather(-1, order))
        return {"ids": torch.cat(ids), "logprobs": torch.cat(lps)}
    n, v = logits.shape
    named = {x: torch.as_tensor(state[x], device="cuda").double().expand(n) for x in
             ("temperature", "top_k", "top_p", "min_p")}
    tokens, lps = [], []
    for i in range(n):  # one row after the other, from its sorted tokens
        t, k, p, mp = (float(named[x][i]) for x in ("temperature", "top_k", "top_p", "min_p"))
        z = logits[i].double()
        logp = torch.log_softmax(z / (t or 1.0), -1)
        order = torch.argsort(z, descending=True, stable=True)
        if t == 0:
            tok = order[0]
        else:
            ps = logp[order].exp()
            kept = torch.ones(v, dtype=torch.bool, device="cuda")
            if k > 0:
                kept[int(k):] = False
            if p < 1:
                kept &= torch.cumsum(ps, 0) - ps < p
            kept &= ps >= mp * ps[0]
            kept[0] = True
            race = state["noise"][i][order].double() / ps
            tok = order[torch.where(kept, race, math.inf).argmin()]
        tokens.append(tok)
        lps.append(logp[tok])
    return {"tokens": torch.stack(tokens), "logprobs": torch.stack(lps)}
