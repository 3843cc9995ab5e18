"""Plain 64-bit definitions of the operators around gated mixtures of kernels (spnc.mixture), in NumPy, from their formulas.
Test infrastructure only."""
import numpy as np


def gate(z, k, over="chosen", log=False):
    """index, weight of the k largest logits a row; ties to the lowest index, NaN above everything, -inf never chosen."""
    z = np.asarray(z, dtype=np.float64)
    n, experts = z.shape
    index, weight = np.full((n, k), -1, dtype=np.int32), np.full((n, k), -np.inf if log else 0.0)
    for i in range(n):
        order = sorted(range(experts), key=lambda e: (not np.isnan(z[i, e]), 0.0 if np.isnan(z[i, e]) else -z[i, e], e))
        chosen = [e for e in order if not z[i, e] == -np.inf][:k]
        if not chosen:
            continue
        pool = z[i, chosen] if over == "chosen" else z[i]
        with np.errstate(all="ignore"):
            top = np.nan if np.isnan(pool).any() else pool.max()
            log_total = top + np.log(np.exp(pool - top).sum())
            w = z[i, chosen] - log_total
        index[i, :len(chosen)] = chosen
        weight[i, :len(chosen)] = w if log else np.exp(w)
    return index, weight


def gate_gradient(z, index, grad, over="chosen", log=False):
    """d sum(grad * weight) / dz from d log w_j / dz_e = [e is j's expert] - p_e, p over the chosen or over all experts."""
    z, grad = np.asarray(z, dtype=np.float64), np.asarray(grad, dtype=np.float64)
    dz = np.zeros_like(z)
    for i in range(z.shape[0]):
        slots = [j for j in range(index.shape[1]) if index[i, j] >= 0]
        if not slots:
            continue
        pool = index[i, slots] if over == "chosen" else np.arange(z.shape[1])
        e = np.exp(z[i, pool] - z[i, pool].max())
        p = np.zeros(z.shape[1])
        p[pool] = e / e.sum()
        for j in slots:
            dlog = grad[i, j] * (1.0 if log else p[index[i, j]])
            dz[i] -= p * dlog
            dz[i, index[i, j]] += dlog
    return dz


def gate_many(z, k, over, log, grad):
    """index, weight and the logits' gradient of many rows without NaN at once."""
    order = np.argsort(-z, axis=1, kind="stable")[:, :k]
    chosen = np.take_along_axis(z, order, axis=1)
    is_open = chosen > -np.inf
    with np.errstate(all="ignore"):
        total = np.logaddexp.reduce(chosen if over == "chosen" else z, axis=1, keepdims=True)
        log_weight = np.where(is_open, chosen - total, -np.inf)
        p = np.where(z > -np.inf, np.exp(z - total), 0.0)
    weight = np.exp(log_weight)
    dlog = np.where(is_open, grad, 0.0) * (1.0 if log else weight)
    dz = -p * dlog.sum(axis=1, keepdims=True) if over == "all" else np.zeros_like(z)
    if over == "chosen":
        dlog = dlog - weight * dlog.sum(axis=1, keepdims=True)
    np.add.at(dz, (np.arange(z.shape[0])[:, None], order), np.where(is_open, dlog, 0.0))
    return np.where(is_open, order, -1), log_weight if log else weight, dz


def route(index, experts, align=1):
    """position, starts, counts by going through the slots in order."""
    flat = np.asarray(index).reshape(-1)
    counts = np.array([(flat == e).sum() for e in range(experts)], dtype=np.int32)
    starts = np.concatenate([[0], np.cumsum((counts + align - 1) // align * align)]).astype(np.int32)
    position, taken = np.full(flat.shape, -1, dtype=np.int32), starts.copy()
    for s, e in enumerate(flat):
        if 0 <= e < experts:
            position[s] = taken[e]
            taken[e] += 1
    return position.reshape(np.shape(index)), starts, counts


def dispatch(rows, position, capacity):
    out = np.zeros((capacity, rows.shape[1]), dtype=rows.dtype)
    for i, j in zip(*np.nonzero(position >= 0)):
        out[position[i, j]] = rows[i]
    return out


def combine(values, position, weights=None):
    values = np.asarray(values, dtype=np.float64)
    out = np.zeros((position.shape[0], values.shape[1]))
    for i, j in zip(*np.nonzero(position >= 0)):
        out[i] += (1.0 if weights is None else float(weights[i, j])) * values[position[i, j]]
    return out


def combine_gradient(values, position, weights, grad):
    values, grad = np.asarray(values, dtype=np.float64), np.asarray(grad, dtype=np.float64)
    grad_values, grad_weights = np.zeros_like(values), np.zeros(position.shape)
    for i, j in zip(*np.nonzero(position >= 0)):
        grad_values[position[i, j]] = float(weights[i, j]) * grad[i]
        grad_weights[i, j] = grad[i] @ values[position[i, j]]
    return grad_values, grad_weights


def combine_log(values, position, log_weights, grad=None):
    """The mixture's log-likelihoods, and with grad [n] the gradients of sum(grad * out) for the values and the log weights.
    In extended precision: a sum of a log weight and a value near -900, rounded to 64 bits, is off by 900 / 2^53, and a share
    by as much relative to itself, which is more than kernels that subtract first are."""
    values, log_weights = np.asarray(values, dtype=np.longdouble), np.asarray(log_weights, dtype=np.longdouble)
    out = np.full(position.shape[0], -np.inf, dtype=np.longdouble)
    grad_values, grad_weights = np.zeros_like(values), np.zeros(position.shape, dtype=np.longdouble)
    for i in range(position.shape[0]):
        slots = [j for j in range(position.shape[1]) if position[i, j] >= 0 and log_weights[i, j] != -np.inf]
        t = np.array([log_weights[i, j] + values[position[i, j]] for j in slots])
        if not slots or (t == -np.inf).all():
            continue
        with np.errstate(all="ignore"):
            top = np.nan if np.isnan(t).any() else t.max()
            e = np.exp(t - top) if not np.isinf(top) else np.full(t.shape, np.nan)
            out[i] = top + np.log(e.sum()) if not np.isinf(top) else top
            if grad is not None:
                for j, share in zip(slots, e / e.sum()):
                    grad_values[position[i, j]] = grad_weights[i, j] = float(grad[i]) * share
    return out if grad is None else (out, grad_values, grad_weights)


def philox(block, offset, seed):
    """Four 32-bit words of Philox4x32-10 (Salmon et al., SC 2011) in Python integers."""
    low = 2 ** 32 - 1
    c = [block & low, block >> 32, offset & low, offset >> 32]
    k = [seed & low, seed >> 32]
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & low, (a >> 32) ^ c[3] ^ k[1], a & low]
        k = [(k[0] + 0x9E3779B9) & low, (k[1] + 0xBB67AE85) & low]
    return c


def keep(count, p, seed, offset=0, first=0):
    """Which of `count` elements from `first` on dropout keeps."""
    words = [philox(e // 4, offset, seed)[e % 4] for e in range(first, first + count)]
    return np.array([w >= round(p * 2 ** 32) for w in words], dtype=bool)
