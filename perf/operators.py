"""Cases that measure the operators on vocabulary rows (``hikoboshi_b200.vocab``).

A vocabulary row is one position's logits over V tokens.  Four operators work
on N such rows:

* ``sample``   draws a token of each row after temperature, top-k, top-p and
  min-p, from a uniform number that the caller gives;
* ``top``      takes the k largest logits of each row in order, with the row's
  log-sum-exp: what a teacher stores of its answer;
* ``distill``  is the divergence of a student's rows from such stored answers
  (mode "loss"), its gradient by autograd (mode "step"), or both in one pass
  over the rows (mode "fused").

Here, with ``own`` false, they are computed with elementary torch operations.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # one sequence that is being written token by token: latency alone
        dict(name="sample-one-row", op="sample", rows=1, vocab=32768, type="f32",
             per_row=False, temperature=0.8, top_k=50, top_p=0.95, min_p=0.0),
        # a serving batch whose requests each bring their own settings
        dict(name="sample-serving-batch", op="sample", rows=64, vocab=131072, type="bf16",
             per_row=True, temperature=0.8, top_k=50, top_p=0.9, min_p=0.05),
        # sampling without a filter, from rows that start at any address
        dict(name="sample-unfiltered", op="sample", rows=192, vocab=50001, type="f16",
             per_row=False, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0),
        # sequence design: 64 backbones of 256 residues, 32 sequences each, 21 letters
        dict(name="sample-design-rows", op="sample", rows=524288, vocab=21, type="f32",
             per_row=False, temperature=0.3, top_k=0, top_p=0.95, min_p=0.02),
        # a teacher that scores 128 backbones of 384 residues with 16 sequences each
        dict(name="top-design-rows", op="top", rows=786432, vocab=21, type="f32", k=8,
             temperature=1.0),
        # alternatives shown for a handful of positions
        dict(name="top-few-rows", op="top", rows=5, vocab=100003, type="f32", k=256,
             temperature=1.0),
        # a teacher's pass over a training batch
        dict(name="top-teacher-batch", op="top", rows=2048, vocab=131072, type="bf16", k=64,
             temperature=2.0),
        # evaluation of a student: the loss alone
        dict(name="distill-loss", op="distill", mode="loss", rows=1024, vocab=32768, type="f32",
             k=32, teacher="f32", tail=False, temperature=1.0),
        # a small training step of odd sizes
        dict(name="distill-small-step", op="distill", mode="step", rows=48, vocab=1009,
             type="f16", k=17, teacher="f16", tail=True, temperature=2.0),
        # a training step through autograd, forward and backward
        dict(name="distill-step", op="distill", mode="step", rows=2000, vocab=50001, type="bf16",
             k=50, teacher="bf16", tail=True, temperature=1.5),
        # a student of the design model, loss and gradient at once
        dict(name="distill-design-rows", op="distill", mode="fused", rows=524288, vocab=21,
             type="f32", k=8, teacher="f32", tail=True, temperature=2.0),
        # the largest training step, loss and gradient at once
        dict(name="distill-large-fused", op="distill", mode="fused", rows=4096, vocab=131072,
             type="bf16", k=64, teacher="bf16", tail=False, temperature=1.0),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["sample", "sample", "top", "distill", "distill"])
    vocab = 21 if rng.random() < 0.2 else _log_uniform(rng, 22, 131072)
    rows = _log_uniform(rng, 1, max(2, min(524288, (1 << 27) // vocab)))
    case = dict(op=op, rows=rows, vocab=vocab, type=rng.choice(["f32", "f16", "bf16"]))
    if op == "sample":
        case.update(per_row=rng.random() < 0.4,
                    temperature=round(rng.uniform(0.2, 1.5), 3),
                    top_k=rng.choice([0, 0, 1, _log_uniform(rng, 2, 1000)]),
                    top_p=rng.choice([1.0, round(rng.uniform(0.1, 0.99), 3)]),
                    min_p=rng.choice([0.0, 0.0, round(rng.uniform(0.001, 0.2), 4)]))
    elif op == "top":
        case.update(k=_log_uniform(rng, 1, min(vocab, 512)), temperature=rng.choice([1.0, 2.0]))
    else:
        case.update(mode=rng.choice(["loss", "step", "fused"]),
                    k=_log_uniform(rng, 1, min(vocab, 256)),
                    teacher=rng.choice(["f32", "f16", "bf16"]), tail=rng.random() < 0.5,
                    temperature=round(rng.uniform(0.7, 3.0), 3))
    return case


def _chunks(rows, vocab, elements=1 << 26):
    step = max(1, elements // vocab)
    return [(r, min(rows, r + step)) for r in range(0, rows, step)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows, vocab, dtype = case["rows"], case["vocab"], _TYPES[case["type"]]
    state = dict(case=case)

    def logits_of(r0, r1):
        # a broad body of unlikely tokens and an exponential spread of likely ones
        x = torch.randn(r1 - r0, vocab, generator=gen, device="cuda") * 2.0
        e = torch.rand(r1 - r0, vocab, generator=gen, device="cuda")
        return x.sub_(e.clamp_(min=1e-7).log_(), alpha=0.7)

    x = torch.empty(rows, vocab, dtype=dtype, device="cuda")
    if case["op"] != "distill":
        for r0, r1 in _chunks(rows, vocab):
            x[r0:r1] = logits_of(r0, r1)
        state["logits"] = x
        if case["op"] == "sample":
            state["uniforms"] = torch.rand(rows, generator=gen, device="cuda")
            s = dict(temperature=case["temperature"], top_k=case["top_k"], top_p=case["top_p"],
                     min_p=case["min_p"])
            if case["per_row"]:
                def around(v, lo):
                    r = torch.rand(rows, generator=gen, device="cuda")
                    return (v * (lo + (1.0 - lo) * r)).float()
                pick = torch.rand(rows, generator=gen, device="cuda")
                # some requests are greedy, some switch a filter off
                t = around(case["temperature"], 0.5)
                s["temperature"] = torch.where(pick < 0.1, torch.zeros_like(t), t)
                k = torch.randint(0, max(1, case["top_k"]) + 1, (rows,), generator=gen,
                                  device="cuda", dtype=torch.int32)
                s["top_k"] = torch.where(pick > 0.5, torch.zeros_like(k), k)
                p = around(case["top_p"], 0.7)
                s["top_p"] = torch.where(pick > 0.9, torch.ones_like(p), p)
                s["min_p"] = around(case["min_p"], 0.0)
            state["settings"] = s
        return state

    k, tau = case["k"], case["temperature"]
    values = torch.empty(rows, k, dtype=_TYPES[case["teacher"]], device="cuda")
    tokens = torch.empty(rows, k, dtype=torch.int32, device="cuda")
    norm = torch.empty(rows, device="cuda")
    for r0, r1 in _chunks(rows, vocab):
        s = logits_of(r0, r1)
        x[r0:r1] = s
        teacher = s.add_(torch.randn(s.shape, generator=gen, device="cuda"))
        v, t = teacher.topk(k, dim=1)
        values[r0:r1], tokens[r0:r1] = v, t
        norm[r0:r1] = torch.logsumexp(teacher / tau, dim=1)
    weights = torch.rand(rows, generator=gen, device="cuda") + 0.5
    # rows of the prompt and of padding do not train
    weights = torch.where(weights < 0.6, torch.zeros_like(weights), weights)
    state.update(logits=x, values=values, tokens=tokens, norm=norm if case["tail"] else None,
                 weights=weights)
    return state


def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    if case["op"] == "sample":
        return _plain_sample(state["logits"], state["uniforms"], **state["settings"])
    if case["op"] == "top":
        return _plain_top(state["logits"], case["k"], case["temperature"])
    loss, grad = _plain_distill(state["logits"], state["values"], state["tokens"], state["norm"],
                                case["temperature"],
                                None if case["mode"] == "loss" else state["weights"])
    return loss if case["mode"] == "loss" else (loss, grad)


def _run_own(case, state):
    from hikoboshi_b200 import vocab

    if case["op"] == "sample":
        r = vocab.sample_tokens(state["logits"], state["uniforms"], **state["settings"])
        return r.tokens, r.log_probs, r.kept
    if case["op"] == "top":
        r = vocab.top_logits(state["logits"], case["k"], temperature=case["temperature"])
        return r.values, r.tokens, r.log_norm
    args = dict(teacher_log_norm=state["norm"], temperature=case["temperature"])
    x, values, tokens = state["logits"], state["values"], state["tokens"]
    if case["mode"] == "loss":
        return vocab.distill_loss(x, values, tokens, **args)
    if case["mode"] == "fused":
        return vocab.distill_loss_and_grad(x, values, tokens, row_weights=state["weights"], **args)
    x = x.detach().requires_grad_()
    loss = vocab.distill_loss(x, values, tokens, **args)
    (grad,) = torch.autograd.grad(loss, x, state["weights"])
    return loss.detach(), grad


def _column(v, rows, dtype):
    return torch.as_tensor(v, device="cuda").to(dtype).reshape(-1, 1).expand(rows, 1)


def _plain_sample(x, u, temperature, top_k, top_p, min_p):
    # in 64 bits: the token is decided by values next to a border
    rows, vocab = x.shape
    t = _column(temperature, rows, torch.float64)
    k = _column(top_k, rows, torch.int64)
    p = _column(top_p, rows, torch.float64)
    m = _column(min_p, rows, torch.float64)
    greedy = t == 0
    sx, order = x.double().sort(dim=1, descending=True, stable=True)
    w = ((sx - sx[:, :1]) / torch.where(greedy, torch.ones_like(t), t)).exp()
    place = torch.arange(vocab, device=x.device)[None, :]
    keep = (place < torch.where(k > 0, k, vocab)) & (~greedy | (place == 0))
    w = w * keep
    before = w.cumsum(1) - w
    keep &= (p >= 1) | (before < p * w.sum(1, keepdim=True)) | (place == 0)
    keep &= (w >= m) | (place == 0)
    w = w * keep
    kept = keep.sum(1).int()
    total = w.sum(1)
    weight = torch.zeros_like(w).scatter_(1, order, w)
    cum = weight.cumsum(1)
    token = (cum > (u.double() * total)[:, None]).int().argmax(1)
    log_prob = (weight.gather(1, token[:, None])[:, 0] / total).log()
    return token.int(), log_prob.float(), kept


def _plain_top(x, k, temperature):
    v, t = x.sort(dim=1, descending=True, stable=True)
    z = x.float() / temperature
    top = z.max(1, keepdim=True).values
    norm = (z - top).exp().sum(1).log() + top[:, 0]
    return v[:, :k].contiguous(), t[:, :k].int().contiguous(), norm


def _plain_distill(x, values, tokens, norm, tau, weights):
    z = x.float() / tau
    a = values.float() / tau
    idx = tokens.long()
    z = z - z.max(1, keepdim=True).values
    e = z.exp()
    total = e.sum(1, keepdim=True)
    log_total = total.log()
    zk = z.gather(1, idx)
    if norm is None:
        a = a - a.max(1, keepdim=True).values
        log_q = a - a.exp().sum(1, keepdim=True).log()
        loss = (log_q.exp() * (log_q - zk + log_total)).sum(1)
    else:
        log_q = a - norm[:, None]
        rest = e.scatter(1, idx, 0.0).sum(1, keepdim=True)
        q_rest = (1.0 - log_q.double().exp().sum(1, keepdim=True)).clamp(min=0).float()
        q_rest = torch.where(rest > 0, q_rest, torch.zeros_like(q_rest))
        tail = q_rest * (q_rest.log() - rest.log() + log_total)
        loss = (log_q.exp() * (log_q - zk + log_total)).sum(1)
        loss = loss + torch.where(q_rest > 0, tail, torch.zeros_like(tail))[:, 0]
    loss = loss * (tau * tau)
    if weights is None:
        return loss, None
    q = log_q.exp()
    if norm is None:
        mass = q.sum(1, keepdim=True)
        grad = (e / total) * mass
    else:
        mass = q.sum(1, keepdim=True) + q_rest
        # p_i (mass - q_rest / p_rest) off the list, p_i mass - q_i on it
        part = torch.where(q_rest > 0, q_rest / rest, torch.zeros_like(rest))
        grad = e * (mass / total - part)
        grad.scatter_(1, idx, zk.exp() * (mass / total))
    grad.scatter_add_(1, idx, -q)
    return loss, (grad * (tau * weights[:, None])).to(x.dtype)


def work(case):
    n, v, b = case["rows"], case["vocab"], _BYTES[case["type"]]
    row = n * v * b
    if case["op"] == "sample":
        settings = 16 * n if case["per_row"] else 0
        return {"bytes": row + settings + 4 * n + 12 * n, "flops": 4 * n * v}
    if case["op"] == "top":
        return {"bytes": row + n * case["k"] * (b + 4) + 4 * n, "flops": 4 * n * v}
    listing = n * case["k"] * (_BYTES[case["teacher"]] + 4) + (4 * n if case["tail"] else 0)
    if case["mode"] == "loss":
        return {"bytes": row + listing + 4 * n, "flops": 4 * n * v}
    # in a step the backward pass comes after the whole forward pass: it has to
    # read the rows again unless they are kept, so one reading counts here
    return {"bytes": 2 * row + listing + 8 * n, "flops": 8 * n * v}


def exact(case, seed):
    state = prepare(case, seed)
    x = state["logits"]
    rows, vocab = x.shape
    parts = []
    for r0, r1 in _chunks(rows, vocab, 1 << 25):
        if case["op"] == "sample":
            s = {n: (v[r0:r1] if torch.is_tensor(v) else v)
                 for n, v in state["settings"].items()}
            parts.append(_exact_sample(x[r0:r1], state["uniforms"][r0:r1], **s))
        elif case["op"] == "top":
            parts.append(_exact_top(x[r0:r1], case["k"], case["temperature"]))
        else:
            norm = state["norm"]
            parts.append(_exact_distill(x[r0:r1], state["values"][r0:r1],
                                        state["tokens"][r0:r1],
                                        None if norm is None else norm[r0:r1],
                                        case["temperature"], state["weights"][r0:r1],
                                        case["mode"] != "loss"))
    out = tuple(torch.cat(p) for p in zip(*parts))
    return out[0] if case["op"] == "distill" and case["mode"] == "loss" else out


def _exact_sample(x, u, temperature, top_k, top_p, min_p):
    # every filter keeps the head of the row's order (value down, index up), so
    # the kept tokens are a number per row: the least of the filters' numbers
    rows, vocab = x.shape

    def per_row(v):
        return (v.double().cpu() if torch.is_tensor(v) else torch.full((rows,), float(v)).double()
                ).to(x.device)

    def setting(v):
        # a number is the 32-bit float that the operator is given
        return per_row(v if torch.is_tensor(v) else torch.tensor(v, dtype=torch.float32).item())

    t, k, p, m = setting(temperature), per_row(top_k), setting(top_p), setting(min_p)
    rank_of = (-x.double()).argsort(dim=1, stable=True).argsort(dim=1)
    best = x.double().amax(1)
    z = (x.double() - best[:, None]) / torch.where(t > 0, t, 1.0)[:, None]
    weight = torch.exp(z)
    by_rank = torch.empty_like(weight).scatter_(1, rank_of, weight)
    n = torch.where(k > 0, k.clamp(max=vocab), float(vocab)).long()
    n = torch.where(t > 0, n, 1)
    running = by_rank.cumsum(1)
    in_k = running.gather(1, n[:, None] - 1)[:, 0]
    # first place whose running mass reaches the share p of the top-k mass
    n_p = torch.searchsorted(running, (p * in_k)[:, None].contiguous())[:, 0] + 1
    n = torch.where(p < 1, torch.minimum(n, n_p), n)
    n_m = (by_rank >= m[:, None]).sum(1)
    n = torch.minimum(n, n_m).clamp(min=1)
    weight = weight * (rank_of < n[:, None])
    cum = weight.cumsum(1)
    total = weight.sum(1)
    token = torch.searchsorted(cum, (u.double() * total)[:, None], right=True)[:, 0]
    token = token.clamp(max=vocab - 1)
    log_prob = z.gather(1, token[:, None])[:, 0] - total.log()
    return token.int(), log_prob, n.int()


def _exact_top(x, k, temperature):
    # the place of a token is the number of tokens before it
    xd = x.double()
    norm = torch.logsumexp(xd / float(torch.tensor(temperature, dtype=torch.float32)), dim=1)
    order = (-xd).argsort(dim=1, stable=True)[:, :k]
    return x.gather(1, order).double(), order.int(), norm


def _exact_distill(x, values, tokens, norm, tau, weights, with_grad):
    tau = float(torch.tensor(tau, dtype=torch.float32))
    log_p = torch.log_softmax(x.double() / tau, dim=1)
    idx = tokens.long()
    a = values.double() / tau
    log_q = torch.log_softmax(a, dim=1) if norm is None else a - norm.double()[:, None]
    q = log_q.exp()
    loss = (q * (log_q - log_p.gather(1, idx))).sum(1)
    rest_q = torch.zeros_like(loss)
    if norm is not None:
        log_rest = torch.logsumexp(log_p.scatter(1, idx, -math.inf), dim=1)
        rest_q = (1.0 - q.sum(1)).clamp(min=0)
        rest_q = torch.where(torch.isinf(log_rest), torch.zeros_like(rest_q), rest_q)
        loss = loss + torch.where(rest_q > 0, rest_q * (rest_q.log() - log_rest), 0.0)
    loss = loss * tau * tau
    if not with_grad:
        return (loss,)
    p = log_p.exp()
    target = torch.zeros_like(p)
    if norm is not None:
        share = torch.where(rest_q[:, None] > 0, (log_p - log_rest[:, None]).exp(), 0.0)
        target = (share * rest_q[:, None]).scatter(1, idx, 0.0)
    target = target.scatter_add(1, idx, q)
    mass = (q.sum(1) + rest_q)[:, None]
    return loss, (p * mass - target) * (tau * weights.double()[:, None])
