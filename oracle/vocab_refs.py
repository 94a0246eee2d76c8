"""64-bit CPU references of the vocabulary operators (filtered sampling, top-k with log-normaliser, distillation from a
teacher's top logits, 8-bit products).  TEST INFRASTRUCTURE ONLY.  Written from the formulas in include/icrl_a2c.h."""
import numpy as np


def row_order(x):
    """Indices of x in the row's order: larger first, ties by lowest index, NaN after everything."""
    x = np.asarray(x, dtype=np.float64)
    return np.lexsort((np.arange(x.size), np.where(np.isnan(x), np.inf, -x), np.isnan(x)))


def sample_filtered(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, log_prob) of one row."""
    x = np.asarray(x, dtype=np.float64)
    bad = (not (np.isfinite(temperature) and temperature >= 0) or top_k < 0 or not 0 <= top_p <= 1 or not 0 <= min_p <= 1
           or np.isnan(u) or np.isnan(x).any() or x.max() == -np.inf)
    if bad:
        return -1, np.nan
    order = row_order(x)
    if temperature == 0 or top_k == 1 or top_p == 0:
        return int(order[0]), 0.0
    order = order[x[order] == np.inf] if x.max() == np.inf else order[x[order] > -np.inf]
    if top_k > 0:
        order = order[:top_k]
    with np.errstate(invalid="ignore"):
        z = np.where(x[order] == x[order[0]], 0.0, (x[order] - x[order[0]]) / temperature)
    w = np.exp(z)
    before = np.concatenate(([0.0], np.cumsum(w)[:-1]))
    last = 0 if top_p == 0 else int(np.nonzero(before < top_p * w.sum())[0].max())
    order, w = order[:last + 1], w[:last + 1]
    order, w = order[w >= min_p], w[w >= min_p]
    by_index = np.argsort(order)
    order, w = order[by_index], w[by_index]
    cdf = np.cumsum(w) / w.sum()
    live = np.nonzero(w > 0)[0]
    at = int((cdf <= u).sum())
    at = int(live[-1]) if at > live[-1] else max(at, int(live[0]))
    return int(order[at]), float(np.log(w[at] / w.sum()))


def topk_lse(x, k, temperature=1.0):
    """(values, indices, lse) of one row in float64."""
    x = np.asarray(x, dtype=np.float64)
    order = row_order(x)[:k]
    m = x.max() if not np.isnan(x).any() else np.nan
    if not np.isfinite(m):
        lse = m
    else:
        lse = m / temperature + np.log(np.exp((x - m) / temperature).sum())
    return x[order], order, lse


def distill(x, values, indices, lse=None, temperature=1.0, weight=1.0):
    """(row_loss, gradient, parts) of one row in float64; parts: z - max z, p, and the ratio q_rest / p_rest."""
    x = np.asarray(x, dtype=np.float64)
    if weight == 0:
        return 0.0, np.zeros_like(x), dict(z=np.zeros_like(x), p=np.zeros_like(x), ratio=0.0, total=0.0)
    there = np.asarray(indices) >= 0
    idx, val = np.asarray(indices)[there], np.asarray(values, dtype=np.float64)[there]
    z = x / temperature
    z = z - z.max()
    e = np.exp(z)
    p = e / e.sum()
    log_p = z - np.log(e.sum())
    nothing = dict(z=z, p=p, ratio=0.0, total=0.0)
    if lse is None:
        if val.size == 0 or val.max() == -np.inf:
            return 0.0, np.zeros_like(x), nothing
        log_q = val / temperature - val.max() / temperature
        log_q = log_q - np.log(np.exp(log_q).sum())
    else:
        log_q = val / temperature - lse
    q = np.exp(log_q)
    live = q > 0
    loss = float((q[live] * (log_q[live] - log_p[idx][live])).sum())
    total, ratio = float(q.sum()), 0.0
    outside = np.ones(x.size, dtype=bool)
    outside[idx] = False
    if lse is not None:
        left, p_rest = 1.0 - q.sum(), p[outside].sum()
        if left > 0 and p_rest > 0:
            loss += left * (np.log(left) - np.log(p_rest))
            total += left
            ratio = left / p_rest
    grad = p * np.where(outside, total - ratio, total)
    grad[idx] -= q
    return weight * loss, weight / temperature * grad, dict(z=z, p=p, ratio=ratio, total=total)


def fp8_values(x):
    """x [rows, K] float32 -> (values an 8-bit operand stands for, float64; the scales' exponents [rows, blocks])."""
    x = np.asarray(x, dtype=np.float64)
    rows, k = x.shape
    out, exps = np.zeros((rows, k)), np.zeros((rows, -(-k // 128)), dtype=np.int64)
    for b in range(0, k, 128):
        part = x[:, b:b + 128]
        top = np.abs(part).max(1)
        with np.errstate(divide="ignore"):
            exp = np.where(top > 0, np.ceil(np.log2(np.where(top > 0, top, 1.0)) - np.log2(448.0) - 1e-12), 0)
        exp = np.where((top > 0) & (top > 448.0 * 2.0 ** exp), exp + 1, exp)
        exp = np.maximum(exp, -127).astype(np.int64)
        y = part / 2.0 ** exp[:, None]
        # e4m3: 3 bits after the leading one, down to 2^-6; steps of 2^-9 below
        step = 2.0 ** (np.maximum(np.floor(np.log2(np.maximum(np.abs(y), 2.0 ** -6))), -6) - 3)
        out[:, b:b + 128] = np.rint(y / step) * step * 2.0 ** exp[:, None]
        exps[:, b // 128] = exp
    return out, exps


