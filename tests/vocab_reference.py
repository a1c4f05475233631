"""The operators on vocabulary rows in 64 bits, row by row, from their
definitions; and the error bounds the kernels are held to."""
import numpy as np
import torch

STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
# half of the smallest number above zero: what rounding near zero may add
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}


def to64(t):
    return t.detach().double().cpu().numpy()


def sample_row(x, u, temperature, top_k, top_p, min_p, drawn=None):
    """(token, log-probability, kept) of one row of 64-bit logits.

    A sum of V weights in 64 bits is off by at most V * 2^-53 of itself, here
    and in any other order of adding.  So where the target u * mass lies within
    V * 2^-52 of the mass of a border between two tokens (exactly on it when a
    row repeats itself and u is the matching fraction), either neighbour is the
    formula's: ``drawn`` is then returned if it is the other one."""
    settings = np.array([temperature, top_p, min_p, u], np.float64)
    if (np.isnan(settings).any() or not 0 <= temperature < np.inf or top_k < 0
            or not 0 <= top_p <= 1 or not 0 <= min_p <= 1 or not 0 <= u <= 1):
        return -1, np.nan, 0
    x = np.where(np.isnan(x), -np.inf, x)
    best = x.max()
    if best == -np.inf:
        return -1, -np.inf, 0
    if temperature == 0:
        return int(x.argmax()), 0.0, 1
    with np.errstate(invalid="ignore"):
        z = np.where(x == best, 0.0, (x - best) / temperature)
    w = np.exp(z)
    order = np.argsort(-x, kind="stable")
    n = int((x > -np.inf).sum())
    if top_k:
        n = min(n, top_k)
    run = np.cumsum(w[order[:n]])
    if top_p < 1:
        n = min(n, 1 + int((run < top_p * run[-1]).sum()))
    n = max(1, min(n, int((w >= min_p).sum())))
    keep = np.zeros(len(x), bool)
    keep[order[:n]] = True
    cum = np.cumsum(np.where(keep, w, 0.0))
    over = np.nonzero(cum > u * cum[-1])[0]
    token = int(over[0]) if len(over) else int(np.nonzero(keep & (w > 0))[0][-1])
    if drawn is not None and 0 <= drawn < len(x) and keep[drawn] and w[drawn] > 0:
        slack = len(x) * 2.0 ** -52 * cum[-1]
        if cum[drawn] - w[drawn] - slack <= u * cum[-1] <= cum[drawn] + slack:
            token = int(drawn)
    return token, float(z[token] - np.log(cum[-1])), n


def top_row(x, k, temperature):
    """(order of the k largest with -1 past the end, log-norm, bound of its error)."""
    x = np.where(np.isnan(x), -np.inf, x)
    order = np.argsort(-x, kind="stable")
    n = int((x > -np.inf).sum())
    tokens = np.full(k, -1)
    tokens[:min(k, n)] = order[:min(k, n)]
    if n == 0:
        return tokens, -np.inf, 0.0
    best = x.max()
    if best == np.inf:
        return tokens, np.inf, 0.0
    z = (x - best) / temperature
    w = np.exp(z)
    total = w.sum()
    norm = best / temperature + np.log(total)
    return tokens, norm, sum_error(z, w) + 2.0 ** -24 * abs(norm)


def sum_error(z, w):
    """Relative error of a 32-bit sum of 32-bit exp(z): each exponent takes three
    roundings (difference, constant, product), the function 2 ulp = 2^-22, and a
    thread adds at most 160 terms one after another (the rest is in 64 bits)."""
    mean = float((np.where(w > 0, -z, 0.0) * w).sum() / w.sum())
    return 2.0 ** -24 * (3 * mean + 4 + 160)


def distill_row(x, values, tokens, norm, tau, dtype):
    """(loss, gradient, bound of the loss's error, bounds of the gradient's)
    of one row, for weight 1."""
    vocab = len(x)
    listed = (tokens >= 0) & (values > -np.inf)
    zero = np.zeros(vocab)
    if (tokens[listed] >= vocab).any():
        return np.nan, np.full(vocab, np.nan), 0.0, zero
    if not listed.any():
        return 0.0, zero, 0.0, zero
    a, t = values[listed] / tau, tokens[listed]
    if norm is None:
        norm = a.max() + np.log(np.exp(a - a.max()).sum())
        tail = False
    else:
        tail = True
    log_q = a - norm
    q = np.exp(log_q)
    best = x.max()
    z = (x - best) / tau
    w = np.exp(z)
    total = w.sum()
    log_p = z - np.log(total)
    p = np.exp(log_p)
    term = q > 0
    loss = float((q[term] * (log_q[term] - log_p[t[term]])).sum())
    err = sum_error(z, w)
    loss_err = q.sum() * err
    rest_q = 0.0
    target = np.zeros(vocab)
    if tail:
        off = np.ones(vocab, bool)
        off[t] = False
        off &= x > -np.inf
        if off.any():
            rest_q = max(0.0, 1.0 - q.sum())
            zr = z[off] - z[off].max()
            wr = np.exp(zr)
            log_rest = z[off].max() + np.log(wr.sum()) - np.log(total)
            if rest_q > 0:
                loss += rest_q * (np.log(rest_q) - log_rest)
                target[off] = rest_q * wr / wr.sum()
                err = max(err, sum_error(zr, wr))
            loss_err += 2 * rest_q * sum_error(zr, wr)
    mass = q.sum() + rest_q
    share = target.copy()
    np.add.at(target, t, q)
    grad = tau * (mass * p - target)
    with np.errstate(invalid="ignore"):
        each = err + 2.0 ** -24 * (4 + 4 * np.where(p > 0, -z, 0.0))
    grad_err = tau * ((mass * p + share) * each + 2.0 ** -40 * target) + 2.0 ** -100
    grad_err = grad_err + STEP[dtype] * (np.abs(grad) + grad_err) + TINY[dtype]
    loss *= tau * tau
    loss_err = tau * tau * (loss_err + 1e-13 * (1 + abs(np.log(total)))) + 2.0 ** -24 * abs(loss)
    return loss, grad, loss_err, grad_err
