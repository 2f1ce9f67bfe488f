"""Cases of the operators over a vocabulary: scores of tokens with their gradient, and distillation from a
teacher's top alternatives with its gradient.

A case is one call.  ``prepare`` makes what a program holds before the call (logits, tokens, the teacher's
alternatives, the buffers that the results go to) and ``run`` makes the call: the plain form in elementary torch
operations in 32 bits (64 where 32 lose what matters), or, with ``own`` set, the library's operators.

The vocabularies are powers of two and odd sizes beside them; rows go from one token being sampled to a whole batch
of training rows.
"""
import math
import os
import sys

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # one token being sampled: its score and the 20 best alternatives; latency counts
        _score("logprobs_sample_1x131072_bf16_top20", 1, 131072, "bf16", top=20, entropy=False),
        # a batch of sequences, one token each, odd vocabulary in padded rows, some tokens forbidden
        _score("logprobs_batch_37x50001_f32_top5", 37, 50001, "f32", top=5, entropy=True, pad=15, banned=0.3, scale=1.25),
        # the tokens of a whole prompt with the 20 best alternatives of each
        _score("logprobs_prompt_4096x131072_bf16_top20", 4096, 131072, "bf16", top=20, entropy=True),
        # scoring a batch of answers: no alternatives asked for
        _score("logprobs_answers_2048x100003_f16", 2048, 100003, "f16", top=0, entropy=True),
        # gradient of a small batch with an entropy bonus
        _score_grad("logprobs_grad_16x32000_f32", 16, 32000, "f32", entropy=True),
        # ragged training rows: odd vocabulary in padded rows, some rows without a target, some tokens forbidden
        _score_grad("logprobs_grad_1001x50001_bf16", 1001, 50001, "bf16", entropy=False, pad=63, banned=0.3, scale=0.8),
        # the gradient of a training batch, cross entropy with an entropy term
        _score_grad("logprobs_grad_4096x131072_bf16", 4096, 131072, "bf16", entropy=True),
        # validation loss of a student
        _distill("distill_loss_512x65536_bf16_top64", "distill_loss", 512, 65536, "bf16", 64, tail=True),
        # one long sequence's loss on odd rows, the teacher's alternatives renormalised
        _distill("distill_loss_99x100003_f32_top20", "distill_loss", 99, 100003, "f32", 20, tail=False, scale=0.5),
        # a small step: loss and gradient of a few rows
        _distill("distill_grad_8x32000_f32_top16", "distill_grad", 8, 32000, "f32", 16, tail=False),
        # ragged rows: odd vocabulary, lists of different lengths, some tokens forbidden
        _distill("distill_grad_777x50001_bf16_top32", "distill_grad", 777, 50001, "bf16", 32, tail=True, pad=63, banned=0.3),
        # a training batch of a student
        _distill("distill_grad_4096x131072_bf16_top64", "distill_grad", 4096, 131072, "bf16", 64, tail=True),
    ]


def _score(name, *args, **more):
    return {"name": name} | _score_case(*args, **more)


def _score_grad(name, *args, **more):
    return {"name": name} | _score_grad_case(*args, **more)


def _distill(name, *args, **more):
    return {"name": name} | _distill_case(*args, **more)


def _score_case(rows, vocab, dtype, top, entropy, pad=0, banned=0.0, scale=1.0):
    return {"op": "logprobs", "rows": rows, "vocab": vocab, "dtype": dtype, "top": top, "entropy": entropy,
            "pad": pad, "banned": banned, "scale": scale}


def _score_grad_case(rows, vocab, dtype, entropy, pad=0, banned=0.0, scale=1.0):
    return {"op": "logprobs_grad", "rows": rows, "vocab": vocab, "dtype": dtype, "entropy": entropy,
            "pad": pad, "banned": banned, "scale": scale}


def _distill_case(op, rows, vocab, dtype, top, tail, pad=0, banned=0.0, scale=1.0):
    return {"op": op, "rows": rows, "vocab": vocab, "dtype": dtype, "top": top, "tail": tail,
            "pad": pad, "banned": banned, "scale": scale}


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["logprobs", "logprobs_grad", "distill_loss", "distill_grad"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    vocab = spread(300, 160000)
    most = (1 << 28) // (2 if dtype == "f32" else 1)
    rows = spread(1, max(1, min(8192, most // vocab)))
    pad = rng.choice([0, 0, 1, 7, 64 - vocab % 64])
    banned = rng.choice([0.0, 0.0, 0.3, 0.9])
    scale = rng.choice([1.0, 1.0, 0.5, 1.4])
    if op == "logprobs":
        return _score_case(rows, vocab, dtype, rng.choice([0, 1, 5, 20, 64]), rng.random() < 0.7, pad, banned, scale)
    if op == "logprobs_grad":
        return _score_grad_case(rows, vocab, dtype, rng.random() < 0.5, pad, banned, scale)
    return _distill_case(op, rows, vocab, dtype, rng.choice([1, 8, 32, 64, 128]), rng.random() < 0.5, pad, banned, scale)


# ---- inputs ------------------------------------------------------------------------------------------------------


def _logits(case, gen, sharp):
    """Rows as an output layer makes them: a spread of a few units around an offset of the row, with some forbidden
    tokens in a part of the rows (minus infinity) where the case has any.  Rows lie in a wider buffer where it pads."""
    n, v, dtype = case["rows"], case["vocab"], _TYPES[case["dtype"]]
    buf = torch.empty(n, v + case["pad"], dtype=dtype, device="cuda")
    x = buf[:, :v]
    offset = torch.randn(n, 1, generator=gen, device="cuda") * 4
    step = max(1, (1 << 27) // v)
    for a in range(0, n, step):
        r = torch.randn(min(step, n - a), v, generator=gen, device="cuda")
        if case["banned"]:
            gone = torch.rand(r.shape, generator=gen, device="cuda") < case["banned"]
            gone &= torch.rand(r.shape[0], 1, generator=gen, device="cuda") < 0.5
            gone[:, : min(v, 8)] = False
            r = torch.where(gone, float("-inf"), r)
        x[a:a + step] = r * sharp + offset[a:a + step]
    if case["pad"]:
        buf[:, v:] = 0
    return x


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    n, v, op, s = case["rows"], case["vocab"], case["op"], case["scale"]
    x = _logits(case, gen, 2.5)
    dev = {"device": "cuda"}
    st = {"op": op, "scale": s, "logits": x}
    if op in ("logprobs", "logprobs_grad"):
        # tokens: a likely one in most rows, any other in the rest, and none (-1) in a few
        t = torch.randint(0, v, (n,), generator=gen, **dev)
        rows = torch.arange(n, **dev)
        likely = torch.rand(n, generator=gen, **dev) < 0.7
        top = torch.finfo(x.dtype).max
        x[rows[likely], t[likely]] = (x[rows, t].float().clamp(-20, 20) + 9).clamp(-top, top).to(x.dtype)[likely]
        t[torch.rand(n, generator=gen, **dev) < (0.05 if n > 8 else 0.0)] = -1
        st["targets"] = t.int()
        st["entropy"] = torch.empty(n, **dev) if case["entropy"] else None
    if op == "logprobs":
        k = case["top"]
        st["top"] = k
        st["logprob"] = torch.empty(n, **dev)
        st["stats"] = torch.empty(n, 2, **dev)
        st["top_logprobs"] = torch.empty(n, k, **dev) if k else None
        st["top_ids"] = torch.empty(n, k, dtype=torch.int32, **dev) if k else None
    elif op == "logprobs_grad":
        # what the forward call left: the row's largest logit and the log of its sum, and the entropy
        m, total, ent = [], [], []
        for a in range(0, n, max(1, (1 << 26) // v)):
            y = x[a:a + max(1, (1 << 26) // v)].double()
            top = y.amax(1, keepdim=True)
            d = (y - top) * s
            e = d.exp()
            z = e.sum(1)
            m.append(top[:, 0])
            total.append(z.log())
            ent.append(z.log() - (e * d.clamp(min=-1e4)).sum(1) / z)
        st["stats"] = torch.stack([torch.cat(m), torch.cat(total)], 1).float()
        st["d_logprob"] = -torch.rand(n, generator=gen, **dev) / n
        if case["entropy"]:
            st["entropy"] = torch.cat(ent).float()
            st["d_entropy"] = torch.full((n,), -0.01 / n, **dev)
        else:
            st["d_entropy"] = None
        st["dlogits"] = torch.empty(n, v, dtype=x.dtype, **dev)
    else:
        # a teacher near the student: the best of the student's logits after a disturbance, as log probabilities; the
        # lists of some rows end early (-1)
        k = min(case["top"], v)
        ids, lp = [], []
        step = max(1, (1 << 26) // v)
        for a in range(0, n, step):
            y = x[a:a + step].float() * s
            y = y + torch.randn(y.shape, generator=gen, **dev)
            y = y - y.amax(1, keepdim=True)
            y = y - y.exp().sum(1, keepdim=True).log()
            best, at = y.topk(k, 1)
            ids.append(at)
            lp.append(best)
        ids, lp = torch.cat(ids), torch.cat(lp)
        length = torch.randint(k // 2, k + 1, (n, 1), generator=gen, **dev)
        short = torch.rand(n, 1, generator=gen, **dev) < (0.2 if n > 8 else 0.0)
        ids = torch.where(short & (torch.arange(k, **dev) >= length), -1, ids)
        st["ids"] = ids.int()
        st["teacher"] = lp if case["tail"] else lp / s + 3
        st["tail"] = case["tail"]
        st["loss"] = torch.empty(n, **dev)
        if op == "distill_grad":
            st["d_loss"] = torch.rand(n, generator=gen, **dev) / n
            st["dlogits"] = torch.empty(n, v, dtype=x.dtype, **dev)
    return st


# ---- one pass ----------------------------------------------------------------------------------------------------


def run(state):
    if own:
        return _own(state)
    return _PLAIN[state["op"]](state)


def _plain_softmax(x, s):
    """The scaled distance of each logit from the row's largest, the log of the sum, and the row's largest."""
    m = x.amax(1, keepdim=True)
    d = (x - m) * s
    total = d.exp().sum(1, keepdim=True).log()
    return d, total, m


def _plain_logprobs(st):
    x = st["logits"].float()
    t = st["targets"].long()
    d, total, m = _plain_softmax(x, st["scale"])
    lp = d - total
    out = {"logprob": torch.where(t >= 0, lp.gather(1, t.clamp(min=0)[:, None])[:, 0], 0.0),
           "stats": torch.cat([m, total], 1)}
    if st["entropy"] is not None:
        out["entropy"] = total[:, 0] - (d.exp() * d.clamp(min=-1e4)).sum(1) / total[:, 0].exp()
    if st["top"]:
        # order by value, the lower index first among equal values: one 64-bit key per logit
        b = (x + 0.0).view(torch.int32).long()
        key = (torch.where(b < 0, b ^ 0x7FFFFFFF, b) << 32) | (0xFFFFFFFF - torch.arange(x.shape[1], device=x.device))
        ids = 0xFFFFFFFF - (key.topk(st["top"], 1).values & 0xFFFFFFFF)
        out["top_ids"] = ids.int()
        out["top_logprobs"] = lp.gather(1, ids)
    return out


def _plain_logprobs_grad(st):
    x = st["logits"].float()
    t = st["targets"].long()
    s = st["scale"]
    lp = (x - st["stats"][:, :1]) * s - st["stats"][:, 1:]
    p = lp.exp()
    g = torch.where(t >= 0, st["d_logprob"], 0.0)[:, None]
    dx = p * -g
    if st["d_entropy"] is not None:
        dx = dx - st["d_entropy"][:, None] * p * (lp.clamp(min=-1e4) + st["entropy"][:, None])
    dx = dx.scatter_add(1, t.clamp(min=0)[:, None], g)
    return {"dlogits": (dx * s).to(st["logits"].dtype)}


def _plain_distill(st):
    x = st["logits"].float()
    n, v = x.shape
    s = st["scale"]
    ids, z = st["ids"].long(), st["teacher"].double()
    k = ids.shape[1]
    valid = (ids >= 0) & (ids < v)
    again = ((ids[:, :, None] == ids[:, None, :]) & torch.ones(k, k, dtype=torch.bool, device=x.device).tril(-1)).any(2)
    valid &= ~again
    if st["tail"]:
        logp = torch.where(valid, z, float("-inf"))
        p = logp.exp()
        r = (1 - p.sum(1, keepdim=True)).clamp(min=0)
    else:
        z = torch.where(valid, z * s, float("-inf"))
        z = z - z.amax(1, keepdim=True)
        logp = z - z.exp().sum(1, keepdim=True).log()
        p = logp.exp()
        r = torch.zeros(n, 1, dtype=torch.float64, device=x.device)
    at = torch.where(valid, ids, v)
    inside = torch.zeros(n, v + 1, dtype=torch.bool, device=x.device).scatter(1, at, True)[:, :v]
    d, total, _ = _plain_softmax(x, s)
    logq = d - total
    q = logq.exp()
    logq_k = logq.gather(1, ids.clamp(min=0)).double()
    rest = torch.where(inside, 0.0, q).sum(1, keepdim=True).double()
    r = torch.where(rest > 0, r, 0.0)
    loss = torch.where(p > 0, p * (logp - logq_k), 0.0).sum(1, keepdim=True)
    loss = loss + torch.where(r > 0, r * (r.log() - rest.log()), 0.0)
    out = {"loss": loss[:, 0].float()}
    if st["op"] == "distill_grad":
        c = p.sum(1, keepdim=True) + r
        share = torch.where(r > 0, r / rest, 0.0)
        dx = q * torch.where(inside, c.float(), (c - share).float())
        dx = dx.scatter_add(1, ids.clamp(min=0), torch.where(valid, -p, 0.0).float())
        out["dlogits"] = (dx * (st["d_loss"][:, None] * s)).to(st["logits"].dtype)
    return out


_PLAIN = {"logprobs": _plain_logprobs, "logprobs_grad": _plain_logprobs_grad, "distill_loss": _plain_distill,
          "distill_grad": _plain_distill}


def _library():
    """The library's package, which lies in a folder of its own under the repository's root."""
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pipeline-parallelism-deep-learning-library_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import linalg_b200 as lb

    return lb


def _own(st):
    lb = _library()
    ctx = lb.context()
    # torch's default stream is the legacy one, whose handle 0 the library reads as its own stream: name it (1) instead
    stream = torch.cuda.current_stream().cuda_stream or 1
    op, s = st["op"], st["scale"]
    if op == "logprobs":
        lb.encode_token_logprobs(ctx, stream, st["logits"], st["targets"], s, logprob=st["logprob"], entropy=st["entropy"],
                                 stats=st["stats"], top_logprobs=st["top_logprobs"], top_ids=st["top_ids"])
        out = {"logprob": st["logprob"], "stats": st["stats"]}
        if st["entropy"] is not None:
            out["entropy"] = st["entropy"]
        if st["top"]:
            out["top_ids"] = st["top_ids"]
            out["top_logprobs"] = st["top_logprobs"]
        return out
    if op == "logprobs_grad":
        lb.encode_token_logprobs_backward(ctx, stream, st["logits"], st["targets"], s, st["stats"], st["d_logprob"],
                                          st["dlogits"], entropy=st["entropy"], d_entropy=st["d_entropy"])
        return {"dlogits": st["dlogits"]}
    if op == "distill_loss":
        lb.encode_distill_loss(ctx, stream, st["logits"], st["ids"], st["teacher"], s, st["loss"], tail=st["tail"])
        return {"loss": st["loss"]}
    lb.encode_distill_grad(ctx, stream, st["logits"], st["ids"], st["teacher"], s, st["dlogits"], d_loss=st["d_loss"],
                           loss=st["loss"], tail=st["tail"])
    return {"loss": st["loss"], "dlogits": st["dlogits"]}


# ---- work and exact values ---------------------------------------------------------------------------------------


def work(case):
    n, v = case["rows"], case["vocab"]
    e = 4 if case["dtype"] == "f32" else 2
    row = v * e
    if case["op"] == "logprobs":
        # logits and token in; score, the two statistics, entropy and alternatives out; a difference, a scaling, an
        # exponential and a sum per logit, a product and a sum more for the entropy
        per = row + 4 + 4 + 8 + (4 if case["entropy"] else 0) + 8 * case["top"]
        flops = v * (6 if case["entropy"] else 4)
    elif case["op"] == "logprobs_grad":
        per = 2 * row + 4 + 8 + 4 + (8 if case["entropy"] else 0)
        flops = v * (7 if case["entropy"] else 5)
    else:
        k = min(case["top"], v)
        per = row + 8 * k + 4
        flops = v * 4
        if case["op"] == "distill_grad":
            per += row + 4
            flops += v * 2
    return {"bytes": n * per, "flops": n * flops}


def exact(case, seed):
    st = prepare(case, seed)
    n, v = case["rows"], case["vocab"]
    parts = []
    step = max(1, (1 << 26) // v)
    for a in range(0, n, step):
        rows = {key: (val[a:a + step] if isinstance(val, torch.Tensor) else val) for key, val in st.items()}
        parts.append(_EXACT[case["op"]](rows))
    return {key: torch.cat([p[key] for p in parts]) for key in parts[0]}


def _exact_logprobs(st):
    y = st["logits"].double() * st["scale"]
    logz = torch.logsumexp(y, 1)
    logp = y - logz[:, None]
    p = logp.exp()
    t = st["targets"].long()
    picked = logp[torch.arange(len(t), device=y.device), t.clamp(min=0)]
    picked[t < 0] = 0.0
    top = st["logits"].double().amax(1)
    out = {"logprob": picked, "stats": torch.stack([top, logz - top * st["scale"]], 1)}
    if st["entropy"] is not None:
        out["entropy"] = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(1)
    if st["top"]:
        order = torch.sort(st["logits"].double(), dim=1, descending=True, stable=True).indices[:, : st["top"]]
        out["top_ids"] = order.int()
        out["top_logprobs"] = torch.take_along_dim(logp, order, 1)
    return out


def _exact_logprobs_grad(st):
    # the gradient for the statistics as they are given (in 32 bits), which are inputs of this call
    y = st["logits"].double()
    stats = st["stats"].double()
    logp = st["scale"] * (y - stats[:, 0:1]) - stats[:, 1:2]
    p = logp.exp()
    t = st["targets"].long()
    hot = torch.zeros_like(p)
    has = (t >= 0).nonzero()[:, 0]
    hot[has, t[has]] = 1.0
    g = (st["d_logprob"].double() * (t >= 0))[:, None]
    dx = g * (hot - p)
    if st["d_entropy"] is not None:
        inner = torch.where(p > 0, p * (logp + st["entropy"].double()[:, None]), torch.zeros_like(p))
        dx -= st["d_entropy"].double()[:, None] * inner
    return {"dlogits": dx * st["scale"]}


def _exact_distill(st):
    y = st["logits"].double() * st["scale"]
    logq = torch.log_softmax(y, 1)
    q = logq.exp()
    n, v = y.shape
    # the teacher's distribution laid out over the vocabulary; prepare's lists hold no index twice
    ids = st["ids"].long()
    row, col = (ids >= 0).nonzero(as_tuple=True)
    teacher = torch.full_like(y, float("-inf"))
    teacher[row, ids[row, col]] = st["teacher"].double()[row, col]
    listed_ = torch.isfinite(teacher)
    if not st["tail"]:
        teacher = torch.log_softmax(teacher * st["scale"], 1)
    p = teacher.exp()
    rest = (q * ~listed_).sum(1)
    r = (1 - p.sum(1)).clamp(min=0) * (rest > 0) if st["tail"] else torch.zeros_like(rest)
    loss = torch.where(p > 0, p * (teacher - logq), torch.zeros_like(p)).sum(1)
    loss = loss + torch.where(r > 0, r * (r / rest).log(), torch.zeros_like(r))
    out = {"loss": loss}
    if st["op"] == "distill_grad":
        total = (p.sum(1) + r)[:, None]
        outside = torch.where(listed_, torch.zeros_like(q), q) * torch.where(r > 0, r / rest, torch.zeros_like(r))[:, None]
        out["dlogits"] = (total * q - p - outside) * (st["d_loss"].double() * st["scale"])[:, None]
    return out


_EXACT = {"logprobs": _exact_logprobs, "logprobs_grad": _exact_logprobs_grad, "distill_loss": _exact_distill,
          "distill_grad": _exact_distill}
