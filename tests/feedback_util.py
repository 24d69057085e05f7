"""Plain float64 forms of the feedback losses, and the error bounds that
follow from the arithmetic of the library's kernels."""
import numpy as np

U32 = 2.0 ** -24  # half a step of float32, relative


def softmax_rows(z, actions, weights=None):
    """(logp, stats, p, one minus p, part) of [n, K] float64 scores."""
    n, K = z.shape
    part = (actions >= 0) & ~np.all(z == -np.inf, axis=1)
    if weights is not None:
        part &= weights != 0
    zs = np.where(part[:, None], z, 0.0)
    m = zs.max(1)
    with np.errstate(invalid="ignore"):
        e = np.exp(zs - m[:, None])
    top = zs.argmax(1)
    rows = np.arange(n)
    e_others = e.copy()
    e_others[rows, top] = 0.0
    rest = e_others.sum(1)
    p = e / (1 + rest)[:, None]
    left = 1 - p
    left[rows, top] = rest / (1 + rest)
    a = np.clip(actions, 0, K - 1)
    with np.errstate(divide="ignore"):
        logp = zs[rows, a] - m - np.log1p(rest)
    logp = np.where(part, logp, 0.0)
    stats = np.stack([np.where(part, m, 0.0), np.where(part, rest, -1.0)], 1)
    return logp, stats, p, left, part


def to_scores(p, left, actions, part, g, h):
    """Derivatives with respect to the scores."""
    rows = np.arange(len(p))
    q = -p
    a = np.clip(actions, 0, p.shape[1] - 1)
    q[rows, a] = left[rows, a]
    g = np.where(part, g, 0.0)[:, None]
    h = np.where(part, h, 0.0)[:, None]
    return g * q, h * q * q + np.abs(g) * p * left, q


def policy_rows(logp, part, adv, old, ref, w, low, high, kl):
    """Loss per row and its first and second derivative in the log probability."""
    part = part & (logp != -np.inf)
    l = np.where(part, logp, 0.0)
    with np.errstate(over="ignore", invalid="ignore"):
        ra = np.exp(l - old) * adv
        ca = np.clip(np.exp(l - old), 1 - low, 1 + high) * adv
    active = np.where(adv >= 0, np.exp(l - old) <= 1 + high, np.exp(l - old) >= 1 - low)
    loss = -np.minimum(ra, ca)
    g = np.where(active, -ra, 0.0)
    h = np.maximum(g, 0.0)
    if ref is not None:
        e = np.expm1(ref - l)
        loss = loss + kl * (e - (ref - l))
        g = g - kl * e
        h = h + kl * (e + 1)
    w = np.ones(len(l)) if w is None else w
    return [np.where(part, w * v, 0.0) for v in (loss, g, h)] + [part]


def exp_error(d, f64):
    """Bound of the relative error of exp(d): __expf is documented within
    2 + 1.173 |d| steps of 2^-23, and d itself is rounded; float64's exp is
    within 1 step."""
    d = np.abs(np.where(np.isfinite(d), d, 0.0))
    return 2.0 ** -52 * (2 + d) if f64 else (2 + 1.173 * d) * 2.0 ** -23 + d * U32


def sum_error(K, p, d, f64):
    """Bound of the relative error of a row's sum: each term's own, and the
    additions of n positive terms one after the other in the scores'
    arithmetic, which change the sum by at most (n - 1) half steps.  Rows of up
    to 128 (float64: 512) classes: at most 16 terms in a lane, then 5 sums of lanes; longer
    rows: ceil(K / 256) in a thread, and float64 across threads."""
    terms = (p * exp_error(d, f64)).sum(1)
    return terms + (min(K, 16) + K // 256 + 4) * (2.0 ** -53 if f64 else U32)


def pairs_loss(s, ref, i, j, w, beta, eps, kind):
    """Loss per pair, and its derivatives in the difference of scores."""
    lean = s if ref is None else s - ref
    u = lean[i] - lean[j]
    if kind == "squared":
        d = u - 1 / (2 * beta)
        loss, g, h = d * d, 2 * d, np.full_like(d, 2.0)
    else:
        x = beta * u
        soft = np.log1p(np.exp(-np.abs(x)))
        loss = (1 - eps) * (soft + np.maximum(-x, 0)) + eps * (soft + np.maximum(x, 0))
        up, down = 1 / (1 + np.exp(-x)), 1 / (1 + np.exp(x))
        g, h = beta * (eps * up - (1 - eps) * down), beta * beta * up * down
    w = np.ones(len(u)) if w is None else np.asarray(w, np.float64)
    return w * loss, w * g, w * h
