"""Operators on two models' class distributions in 64 bits on the CPU, row by row from their definitions: the k largest
logits of a row, distillation from them (loss and gradient) and the verification of drafted classes."""
import numpy as np

NEG = -np.inf


def _lse(y):
    y = np.asarray(y, np.float64)
    if y.size == 0 or np.max(y) == NEG:
        return NEG
    m = np.max(y)
    return m + np.log(np.sum(np.exp(y - m)))


def _log_softmax(y):
    """Of the values as they are: the largest is taken off first, so that -1.7e308 and its like keep their share."""
    y = np.asarray(y, np.float64)
    top = np.max(y)
    if top == NEG:
        return np.full(y.shape, NEG)
    return (y - top) - np.log(np.sum(np.exp(y - top)))


def top_row(z, k, temperature=1.0):
    """z (K,) -> (classes of the k largest, log-sum-exp of the others / T)."""
    z = np.asarray(z, np.float64)
    order = sorted(range(len(z)), key=lambda c: (-(np.inf if np.isnan(z[c]) else z[c]), c))
    left = np.array([np.inf if np.isnan(z[c]) else z[c] for c in order[k:]])
    rest = np.inf if np.any(left == np.inf) else _lse(left / temperature)
    return np.array(order[:k]), rest


def distill_row(z, values, index, rest=None, temperature=1.0):
    """-> (loss, dloss/dz (K,), counted).  Also correct where classes or slots are -inf."""
    z, t = np.asarray(z, np.float64) / temperature, np.asarray(values, np.float64) / temperature
    index = np.asarray(index, np.int64)
    K = len(z)
    filled = t > NEG
    if not filled.any():
        return 0.0, np.zeros(K), False
    if np.any((index[filled] < 0) | (index[filled] >= K)):
        return np.nan, np.full(K, np.nan), True
    r = NEG if rest is None else float(rest)
    log_p = _log_softmax(np.append(t, r))
    log_p, log_pr = log_p[:-1], log_p[-1]
    log_q = _log_softmax(z)
    loss, grad = 0.0, np.exp(log_q)
    listed = np.zeros(K, bool)
    listed[index[filled]] = True
    for j in np.nonzero(filled)[0]:
        p = np.exp(log_p[j])
        if p > 0:
            loss += p * (log_p[j] - log_q[index[j]])
            grad[index[j]] -= p
    pr = np.exp(log_pr)
    if rest is not None and pr > 0:
        lr = _lse(log_q[~listed])
        loss += pr * (log_pr - lr)
        if lr > NEG:
            grad[~listed] -= pr * np.exp(log_q[~listed] - lr)
    return temperature ** 2 * loss, temperature * grad, True


def distill_scale(z, values, index, rest=None, temperature=1.0):
    """Per class: the sum of the magnitudes whose difference the gradient is (what its rounding errors scale with)."""
    z, t = np.asarray(z, np.float64) / temperature, np.asarray(values, np.float64) / temperature
    q = np.exp(_log_softmax(z))
    out = q.copy()
    filled = t > NEG
    r = NEG if rest is None else float(rest)
    p = np.exp(_log_softmax(np.append(t, r)))
    listed = np.zeros(len(z), bool)
    for j in np.nonzero(filled)[0]:
        out[index[j]] += p[j]
        listed[index[j]] = True
    left = q[~listed].sum()
    if left > 0:
        out[~listed] += p[-1] * q[~listed] / left
    return temperature * out


def verify_row(tokens, target, draft, accept_u, sample_u, length):
    """One sequence: tokens (T,), target (Tp, K), draft (T, K) | None -> (tokens (Tp,), accepted)."""
    target = np.asarray(target, np.float64)
    steps, K = target.shape
    n = int(min(max(length, 0), len(tokens)))
    a = 0
    while a < n:
        d = int(tokens[a])
        if not 0 <= d < K:
            break
        q = 1.0 if draft is None else float(draft[a][d])
        if not float(accept_u[a]) * q < target[a][d]:
            break
        a += 1
    out = np.full(steps, -1, np.int64)
    out[:a] = tokens[:a]
    if a < steps:
        w = target[a].copy()
        if a < n:
            if draft is not None:
                w = w - np.asarray(draft[a], np.float64)
            elif 0 <= int(tokens[a]) < K:
                w[int(tokens[a])] = 0.0
        w = np.where(w > 0, w, 0.0)
        if not w.sum() > 0:
            w = np.where(target[a] > 0, target[a], 0.0)
        if w.sum() > 0:
            run = np.cumsum(w)
            past = np.nonzero(run > float(sample_u) * run[-1])[0]
            out[a] = past[0] if len(past) else np.nonzero(w > 0)[0][-1]
    return out, a
