"""The token-policy operators in 64 bits, from their definitions (include/cleanba_mi.h), row by row with numpy: what the HIP kernels are held to."""
import math

import numpy as np

EPS32 = 2.0 ** -24                     # half a step of fp32, relative
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
TINY = {"f32": 2.0 ** -126, "bf16": 2.0 ** -126, "f16": 2.0 ** -25}   # what flushing / subnormal rounding may take


def lse64(x, tau):
    x = np.asarray(x, np.float64) / tau
    if np.isnan(x).any():
        return math.nan
    m = x.max() if x.size else -math.inf
    if not math.isfinite(m):
        return m
    return m + math.log(np.exp(x - m).sum())


def top(row, k, tau):
    """(idx, values, lse) of one row of fp32-exact logits."""
    row = np.asarray(row, np.float64)
    order = sorted((j for j in range(row.size) if row[j] > -math.inf), key=lambda j: (-row[j], j)) if row.size < 4096 else \
        [j for j in np.lexsort((np.arange(row.size), -np.where(np.isnan(row), -math.inf, row)))[:k] if row[j] > -math.inf]
    idx = np.full(k, -1, np.int32)
    val = np.full(k, -math.inf, np.float32)
    n = min(k, len(order))
    idx[:n] = order[:n]
    val[:n] = row[order[:n]] + 0.0
    return idx, val, math.inf if np.isposinf(row).any() else lse64(row, tau)


def distill(z, idx, v, tlse, w, tau):
    """(loss, gradient, s, t_T s_j / s_T) of one row."""
    z = np.asarray(z, np.float64)
    V = z.size
    zero = (0.0, np.zeros(V), np.zeros(V), np.zeros(V))
    if w == 0.0 or (z == -math.inf).all():
        return zero
    slots = [(int(i), float(x)) for i, x in zip(idx, v) if 0 <= i < V]
    if tlse is None:
        peak = max((x for _, x in slots), default=-math.inf)
        if peak == -math.inf:
            return zero
        e = [math.exp((x - peak) / tau) for _, x in slots]
        t = [x / sum(e) for x in e]
        rest = 0.0
    else:
        t = [math.exp(x / tau - tlse) if x > -math.inf else 0.0 for _, x in slots]
        rest = max(0.0, 1.0 - math.fsum(t))
    total = lse64(z, tau)
    s = np.exp(z / tau - total)
    outside = np.ones(V, bool)
    for i, _ in slots:
        outside[i] = False
    other = lse64(np.where(outside, z, -math.inf), tau)
    if other == -math.inf:
        rest = 0.0
    loss = 0.0
    g = s * (math.fsum(t) + rest)
    for (i, _), p in zip(slots, t):
        if p > 0.0:
            loss += p * (math.log(p) - (z[i] / tau - total)) if z[i] > -math.inf else math.inf
            g[i] -= p
    share = np.zeros(V)
    if rest > 0.0:
        loss += rest * (math.log(rest) - (other - total))
        share = np.where(outside, rest * np.exp(z / tau - other), 0.0)
        g = g - share
    return w * tau * tau * loss, w * tau * g, s, share


def _dist(row, tau):
    """Probabilities of a row, or None where it is no distribution."""
    row = np.asarray(row, np.float64)
    if np.isnan(row).any() or np.isposinf(row).any() or (row == -math.inf).all():
        return None
    if tau == 0.0:
        p = np.zeros(row.size)
        p[int(np.argmax(row))] = 1.0
        return p
    e = np.exp((row - row.max()) / tau)
    return e / e.sum()


def verify(target, draft, tokens, n, u_accept, u_sample, tau):
    """One sequence: (tokens, accepted, logprobs, margin): margin is how near, relatively, the nearest decision was to falling the other way."""
    K = len(tokens)
    V = target.shape[1]
    out, logs, margin = [], [], math.inf
    left = None
    a = 0
    n = min(max(int(n), 0), K)
    while a < n:
        x = int(tokens[a])
        p = _dist(target[a], tau)
        if tau == 0.0:
            if p is not None and 0 <= x < V and p[x] == 1.0:
                out.append(x); logs.append(0.0); a += 1
                continue
            left = p
            break
        if draft is not None:
            q = _dist(draft[a], tau)
        else:
            q = np.zeros(V)
            if 0 <= x < V:
                q[x] = 1.0
        if p is not None and q is not None and 0 <= x < V:
            u = float(u_accept[a])
            if u * q[x] < p[x]:
                out.append(x); logs.append(math.log(p[x])); a += 1
                margin = min(margin, (p[x] - u * q[x]) / p[x])
                continue
            if u * q[x] > 0.0:
                margin = min(margin, (u * q[x] - p[x]) / (u * q[x]))
        left = p
        if p is not None and q is not None:
            r = np.maximum(p - q, 0.0)
            if r.sum() > 0.0:
                left = r
        break
    if a == n:
        left = _dist(target[n], tau)
    at = a
    if left is None:
        return out + [-1] * (K + 1 - at), a, logs + [0.0] * (K + 1 - at), margin
    if tau == 0.0:
        token, lp = int(np.argmax(left)), 0.0
    else:
        c = np.cumsum(left)
        goal = float(u_sample) * c[-1]
        token = int(np.argmax(c > goal))
        below = c[token - 1] if token else 0.0
        margin = min(margin, 1e6 * (c[token] - goal) / c[-1], 1e6 * (goal - below) / c[-1] if below > 0.0 else math.inf)   # (summed in fp64: the scale of what may flip is a million times smaller)
        lp = math.log(_dist(target[at], tau)[token])
    return out + [token] + [-1] * (K - at), a, logs + [lp] + [0.0] * (K - at), margin
