"""Measured cases of the feedback losses: log probabilities of taken classes, the clipped policy loss and the paired
preference loss, each with its gradient.

A case is one call (the log probabilities' forward and backward pass are two calls of one case) on inputs like those of a
boosting round (float64 raw scores of a few classes, many rows, gradients and hessians) or of token scores (16-bit scores
of thousands of classes, fewer rows, gradients alone).  Where `own` is false the operators are computed in plain torch
operations, in 32 bits for scores of 32 and 16 bits and in 64 for float64 scores.  The sums over a row and the scalars of
a row are always in 64 bits, since a row next to the clipping border has a gradient on one side of it and none on the
other; with millions of rows of a few float32 scores some rows come that near to it, and the policy loss takes their
exponentials in 64 bits too.
"""
import math

import torch

own = False

DTYPES = {"float64": torch.float64, "float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
BYTES = {"float64": 8, "float32": 4, "float16": 2, "bfloat16": 2}


# ---------------------------------------------------------------------------------------------------------- the cases

def _logprobs(name, n, k, dtype, hess, mask=False, pad=0, ids="int32"):
    return {"name": name, "op": "logprobs", "n": n, "k": k, "dtype": dtype, "hess": hess, "mask": mask, "pad": pad, "ids": ids}


def _policy(name, n, k, dtype, hess, mask=False, pad=0, ids="int32", weights=False, ref=True, grad=True):
    return {"name": name, "op": "policy", "n": n, "k": k, "dtype": dtype, "hess": hess, "mask": mask, "pad": pad, "ids": ids,
            "weights": weights, "ref": ref, "grad": grad, "low": 0.2, "high": 0.28, "kl": 0.04 if ref else 0.0}


def _preference(name, n, pairs, dtype, layout, loss="logistic", weights=False, ref=True, beta=0.5, smoothing=0.0):
    return {"name": name, "op": "preference", "n": n, "pairs": pairs, "dtype": dtype, "layout": layout, "loss": loss,
            "weights": weights, "ref": ref, "beta": beta, "smoothing": smoothing}


def listed():
    return [
        # the reference log probabilities of 4M logged decisions among 10 classes (the multiclass configuration's rows),
        # and the way back to the scores with hessians, as the preference objective of a 10-class model takes it
        _logprobs("logprobs 4M x 10 f64", 4_000_000, 10, "float64", True),
        # one small batch of logged decisions, some classes not allowed
        _logprobs("logprobs 300 x 5 f64 masked", 300, 5, "float64", True, mask=True),
        # a training batch of token scores with an odd number of classes
        _logprobs("logprobs 2047 x 50001 bf16", 2047, 50_001, "bfloat16", False, ids="int64"),
        # one boosting round of a 10-class policy at the multiclass configuration's rows
        _policy("policy 4M x 10 f64", 4_000_000, 10, "float64", True),
        # single precision scores, an odd number of rows and classes, classes that are not allowed, weighted rows
        _policy("policy 1000003 x 7 f32 masked", 1_000_003, 7, "float32", True, mask=True, weights=True),
        # a training batch of token scores
        _policy("policy 8192 x 32768 bf16", 8192, 32_768, "bfloat16", False, ids="int64"),
        # few rows of many classes in a padded buffer: the last part of a batch
        _policy("policy 37 x 131072 f16 padded", 37, 131_072, "float16", False, pad=64, ids="int64", weights=True),
        # the loss alone (no gradient) of a handful of rows: latency
        _policy("policy 16 x 64 f32 loss", 16, 64, "float32", False, grad=False),
        # every item in one pair: chosen and rejected answers, or rows, of a large preference set
        _preference("preference 1M apart f64", 2_000_000, 1_000_000, "float64", "apart"),
        # every pair within groups of 64: ranked candidates of 65536 items
        _preference("preference groups of 64 f64", 65_536, 65_536 // 64 * 2016, "float64", "groups64", smoothing=0.1),
        # popular items win against many others: degrees from none to hundreds of thousands
        _preference("preference popular f32", 300_001, 4_000_000, "float32", "popular", weights=True),
        # a batch of answer pairs with their reference log probabilities: latency
        _preference("preference 48 apart f32", 96, 48, "float32", "apart", loss="squared", beta=0.1),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["logprobs", "policy", "policy", "preference"])
    if op == "preference":
        layout = rng.choice(["apart", "groups", "popular"])
        dtype = rng.choice(["float64", "float32"])
        more = {"loss": rng.choice(["logistic", "logistic", "squared"]), "weights": rng.random() < 0.5, "ref": rng.random() < 0.7,
                "beta": round(rng.uniform(0.05, 2.0), 3), "smoothing": rng.choice([0.0, 0.0, 0.1])}
        if layout == "apart":
            pairs = _spread(rng, 1, 1_000_000)
            n = 2 * pairs + rng.randrange(3)
        elif layout == "groups":
            g = rng.randrange(2, 100)
            groups = _spread(rng, 1, max(1, 4_000_000 // (g * (g - 1) // 2)))
            n, pairs, layout = groups * g, groups * (g * (g - 1) // 2), "groups%d" % g
        else:
            n, pairs = _spread(rng, 3, 1_000_000), _spread(rng, 1, 4_000_000)
        case = _preference("", n, pairs, dtype, layout, **more)
    else:
        if rng.random() < 0.5:  # raw scores of a boosting round
            k = rng.randrange(2, 65)
            n = _spread(rng, 1, min(4_000_000, 39_000_000 // k))
            dtype, hess, ids = rng.choice(["float64", "float32"]), True, "int32"
        else:  # token scores
            k = _spread(rng, 65, 131_072)
            n = _spread(rng, 1, min(65_536, 260_000_000 // k))
            dtype, hess, ids = rng.choice(["bfloat16", "float16", "float32"]), False, "int64"
            if dtype == "float32":
                n = max(1, n // 2)
        common = {"mask": rng.random() < 0.4, "pad": rng.choice([0, 0, 0, 1, 8, 64]), "ids": ids}
        if op == "logprobs":
            case = _logprobs("", n, k, dtype, hess, **common)
        else:
            grad = rng.random() < 0.85
            case = _policy("", n, k, dtype, hess and grad, weights=rng.random() < 0.5, ref=rng.random() < 0.7, grad=grad, **common)
    del case["name"]
    return case


# --------------------------------------------------------------------------------------------------------- the inputs

def _scores(case, gen):
    """Scores, taken classes and their log probabilities (64 bits).  With "mask": a fifth of the classes is not allowed
    (-inf), every 50th row takes no part (class -1, scores NaN), some rows have no class that is allowed, or take one
    that is not."""
    n, k, dtype = case["n"], case["k"], DTYPES[case["dtype"]]
    buf = torch.empty(n, k + case["pad"], dtype=dtype, device="cuda")
    x = buf[:, :k]
    a = torch.randint(0, k, (n,), generator=gen, device="cuda")
    for r0 in range(0, n, max(1, (1 << 26) // k)):
        r1 = min(n, r0 + max(1, (1 << 26) // k))
        t = torch.randn(r1 - r0, k, generator=gen, device="cuda") * (1.5 if k <= 64 else 2.5)
        if k > 64:  # a model's choice stands out among thousands of classes
            t.scatter_add_(1, a[r0:r1, None], torch.rand(r1 - r0, 1, generator=gen, device="cuda") * 12)
        if case["mask"]:
            off = torch.rand(r1 - r0, k, generator=gen, device="cuda") < 0.2
            row = torch.rand(r1 - r0, 1, generator=gen, device="cuda")
            off.scatter_(1, a[r0:r1, None], row < 0.02)
            off |= row < 0.01
            t.masked_fill_(off, -math.inf)
            t[torch.arange(r0, r1, device="cuda") % 50 == 49] = math.nan
        x[r0:r1] = t.to(dtype)
    logp = torch.empty(n, dtype=torch.float64, device="cuda")
    for r0 in range(0, n, max(1, (1 << 25) // k)):
        xs = x[r0:r0 + max(1, (1 << 25) // k)].double()
        logp[r0:r0 + len(xs)] = torch.log_softmax(xs, 1).gather(1, a[r0:r0 + len(xs), None])[:, 0]
    logp = torch.nan_to_num(logp, nan=-1.0, posinf=-1.0, neginf=-1.0)
    if case["mask"]:
        a[49::50] = -1
    return x, a.to(torch.int32 if case["ids"] == "int32" else torch.int64), logp


def _pair_list(case, gen):
    n, p, layout = case["n"], case["pairs"], case["layout"]
    if layout == "apart":
        at = torch.randperm(n, generator=gen, device="cuda")
        return at[:p].clone(), at[p:2 * p].clone()
    if layout == "popular":
        win = (n * torch.rand(p, generator=gen, device="cuda", dtype=torch.float64) ** 4).long().clamp_(max=n - 1)
        lose = torch.randint(0, n - 1, (p,), generator=gen, device="cuda")
        return win, lose + (lose >= win)
    g = int(layout[len("groups"):])
    i, j = torch.triu_indices(g, g, 1, device="cuda")
    first = torch.arange(n // g, device="cuda")[:, None] * g
    i, j = (first + i).reshape(-1), (first + j).reshape(-1)
    turn = torch.rand(len(i), generator=gen, device="cuda") < 0.5
    return torch.where(turn, i, j), torch.where(turn, j, i)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    if case["op"] == "preference":
        dtype = DTYPES[case["dtype"]]
        n, p = case["n"], case["pairs"]
        s["winners"], s["losers"] = _pair_list(case, gen)
        s["pair_weights"] = None
        if case["weights"]:  # some pairs weigh nothing
            w = torch.rand(p, generator=gen, device="cuda") * 2
            s["pair_weights"] = torch.where(w < 0.1, torch.zeros_like(w), w)
        # log probabilities of whole answers, or raw scores, and the reference's near them
        s["reference"] = torch.randn(n, generator=gen, device="cuda", dtype=dtype) * 6 - 40 if case["ref"] else None
        s["scores"] = torch.randn(n, generator=gen, device="cuda", dtype=dtype) * 1.5
        if case["ref"]:
            s["scores"] += s["reference"]
        if own:  # the pairs' plan is kept while the scores change from round to round
            import mojoboost_b200 as mb
            w = s["pair_weights"]
            s["plan"] = mb.PreferencePlan(s["winners"].cpu().numpy(), s["losers"].cpu().numpy(), n,
                                          weights=None if w is None else w.cpu().numpy())
        return s
    s["scores"], s["actions"], logp = _scores(case, gen)
    n = case["n"]
    per_row = torch.float64 if case["dtype"] == "float64" else torch.float32
    if case["op"] == "logprobs":
        s["grad_logp"] = torch.randn(n, generator=gen, device="cuda")
        s["hess_logp"] = torch.rand(n, generator=gen, device="cuda") if case["hess"] else None
        return s
    noise = torch.randn(n, generator=gen, device="cuda", dtype=torch.float64)
    s["old_logp"] = (logp + 0.2 * noise).clamp_(max=0).to(per_row)
    s["advantages"] = torch.randn(n, generator=gen, device="cuda", dtype=torch.float64).to(per_row)
    noise = torch.randn(n, generator=gen, device="cuda", dtype=torch.float64)
    s["ref_logp"] = (logp + 0.4 * noise).clamp_(max=0).to(per_row) if case["ref"] else None
    s["weights"] = None
    if case["weights"]:  # padding weighs nothing
        w = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64) * 2
        s["weights"] = torch.where(w < 0.2, torch.zeros_like(w), w).to(per_row)
    return s


# ------------------------------------------------------------------------------------------------------ the plain form

def _row_sums(x, a, border=False):
    """exp(x - max), max, sum in 64 bits, the taken class, its score less the max, whether the row takes part."""
    wide = x.dtype == torch.float64 or (border and x.dtype == torch.float32 and x.shape[1] <= 64)
    xw = x.double() if wide else x.float()
    m = xw.amax(1)
    part = (a >= 0) & (m != -math.inf)
    m = torch.where(part, m, torch.zeros_like(m))
    e = torch.exp(xw - m[:, None])
    total = e.sum(1, dtype=torch.float64)
    at = a.clamp(min=0).long()[:, None]
    return e, m, total, at, (xw.gather(1, at)[:, 0] - m).double(), part


def _to_scores(e, total, at, part, g, h, dtype, hess):
    """The gradient and hessian of the taken class's log probability, taken back to the scores."""
    p = torch.where(part[:, None], e / total.to(e.dtype)[:, None], torch.zeros((), dtype=e.dtype, device=e.device))
    g, h = g.to(e.dtype)[:, None], h.to(e.dtype)[:, None] if hess else None
    q = -p
    q.scatter_add_(1, at, part[:, None].to(e.dtype))
    grad = (g * q).to(dtype)
    return grad, (h * q * q + g.abs() * p * (1 - p)).to(dtype) if hess else None


def _plain_logprobs(s):
    x, a = s["scores"], s["actions"]
    e, m, total, at, xa, part = _row_sums(x, a)
    row = torch.float64 if x.dtype == torch.float64 else torch.float32
    zero = torch.zeros((), dtype=torch.float64, device="cuda")
    logp = torch.where(part, xa - torch.log(total), zero).to(row)
    stats = torch.stack([m.to(row), (torch.where(part, total, zero) - 1).to(row)], 1)
    g = torch.where(part, s["grad_logp"], 0.0)
    h = torch.where(part, s["hess_logp"], 0.0) if s["hess"] else None
    grad, hess = _to_scores(e, total, at, part, g, h, torch.float32 if x.dtype == torch.float64 else x.dtype, s["hess"])
    return {"logp": logp, "stats": stats, "grad": grad, "hess": hess}


def _plain_policy(s):
    x, a = s["scores"], s["actions"]
    e, m, total, at, xa, part = _row_sums(x, a, border=True)
    row = torch.float64 if x.dtype == torch.float64 else torch.float32
    zero = torch.zeros((), dtype=torch.float64, device="cuda")
    w = torch.ones(s["n"], dtype=torch.float64, device="cuda") if s["weights"] is None else s["weights"].double()
    part = part & (w != 0)
    logp = torch.where(part, xa - torch.log(total), zero)
    part = part & (xa != -math.inf)
    safe = torch.where(part, logp, zero)
    adv = s["advantages"].double()
    r = torch.exp(safe - s["old_logp"].double())
    ra, ca = r * adv, r.clamp(1 - s["low"], 1 + s["high"]) * adv
    active = torch.where(adv >= 0, r <= 1 + s["high"], r >= 1 - s["low"])
    loss, g = -torch.minimum(ra, ca), torch.where(active, -ra, zero)
    h = g.clamp(min=0)
    if s["ref"]:
        t = s["ref_logp"].double() - safe
        et = torch.exp(t)
        loss, g, h = loss + s["kl"] * (et - t - 1), g + s["kl"] * (1 - et), h + s["kl"] * et
    loss, g, h = (torch.where(part, w * v, zero) for v in (loss, g, h))
    out = {"loss": loss.to(row), "logp": logp.to(row)}
    if s["grad"]:
        to = torch.float32 if x.dtype == torch.float64 else x.dtype
        out["grad"], out["hess"] = _to_scores(e, total, at, part, g, h, to, s["hess"])
    return out


def _plain_preference(s):
    i, j, x = s["winners"], s["losers"], s["scores"].double()
    m = x[i] - x[j]
    if s["ref"]:
        r = s["reference"].double()
        m = m - (r[i] - r[j])
    beta, eps = s["beta"], s["smoothing"]
    if s["loss"] == "squared":
        d = m - 1 / (2 * beta)
        loss, g, h = d * d, 2 * d, torch.full_like(d, 2.0)
    else:
        z = beta * m
        e = torch.exp(-z.abs())
        big, small = 1 / (1 + e), e / (1 + e)
        up, down = torch.where(z >= 0, big, small), torch.where(z >= 0, small, big)
        soft = torch.log1p(e)
        loss = (1 - eps) * (soft + (-z).clamp(min=0)) + eps * (soft + z.clamp(min=0))
        g, h = beta * (eps * up - (1 - eps) * down), beta * beta * up * down
    if s["pair_weights"] is not None:
        w = s["pair_weights"].double()
        loss, g, h = w * loss, w * g, w * h
    grad = torch.zeros_like(x).index_add_(0, i, g).index_add_(0, j, -g)
    hess = torch.zeros_like(x).index_add_(0, i, h).index_add_(0, j, h)
    return {"loss": loss.to(s["scores"].dtype), "grad": grad.float(), "hess": hess.float()}


# ------------------------------------------------------------------------------------------------------------ one pass

def run(state):
    s = state
    if not own:
        return {"logprobs": _plain_logprobs, "policy": _plain_policy, "preference": _plain_preference}[s["op"]](s)
    import mojoboost_b200 as mb
    if s["op"] == "logprobs":
        logp, stats = mb.action_logprobs(s["scores"], s["actions"])
        grad, hess = mb.action_logprobs_grad(s["scores"], s["actions"], stats, s["grad_logp"], s["hess_logp"])
        return {"logp": logp, "stats": stats, "grad": grad, "hess": hess}
    if s["op"] == "policy":
        loss, logp, grad, hess = mb.policy_loss(s["scores"], s["actions"], s["advantages"], s["old_logp"], ref_logp=s["ref_logp"],
                                                weights=s["weights"], clip_low=s["low"], clip_high=s["high"], kl_coef=s["kl"],
                                                grad=s["grad"], hess=s["hess"])
        return {"loss": loss, "logp": logp, "grad": grad, "hess": hess} if s["grad"] else {"loss": loss, "logp": logp}
    loss, grad, hess = mb.preference_loss(s["plan"], s["scores"], reference=s["reference"], beta=s["beta"],
                                          label_smoothing=s["smoothing"], loss=s["loss"])
    return {"loss": loss, "grad": grad, "hess": hess}


def work(case):
    size = BYTES[case["dtype"]]
    if case["op"] == "preference":
        n, p = case["n"], case["pairs"]
        return {"bytes": p * (8 + (4 if case["weights"] else 0) + size) + n * (size * (2 if case["ref"] else 1) + 8), "flops": 40 * p + 2 * n}
    n, k = case["n"], case["k"]
    back = min(size, 4) * (2 if case["hess"] else 1)
    row = 8 if case["dtype"] == "float64" else 4
    ids = 4 if case["ids"] == "int32" else 8
    if case["op"] == "logprobs":
        return {"bytes": n * k * (size + back) + n * (ids + 3 * row + 4 + (4 if case["hess"] else 0)), "flops": n * k * (8 if case["hess"] else 5)}
    per = ids + row * (4 + (1 if case["ref"] else 0) + (1 if case["weights"] else 0))
    return {"bytes": n * k * (size + (back if case["grad"] else 0)) + n * per, "flops": n * k * (8 if case["hess"] else 5 if case["grad"] else 3)}


# ------------------------------------------------------------------------------------------- the definition in 64 bits

def _exact_rows(s, r0, r1):
    """Rows [r0, r1) by differentiation of the definition in 64 bits; the hessian's two factors from the probabilities."""
    take = lambda v: None if v is None else v[r0:r1]  # noqa: E731
    x, a = s["scores"][r0:r1].double(), s["actions"][r0:r1].long()
    live = (a >= 0) & ~(x == -math.inf).all(1)
    if s["op"] == "policy" and s["weights"] is not None:
        live = live & (take(s["weights"]) != 0)
    rows = live.nonzero()[:, 0]
    xs, at = x[rows].requires_grad_(True), a[rows]
    lp_all = torch.log_softmax(xs, 1)
    lp = lp_all.gather(1, at[:, None])[:, 0]
    n, k = r1 - r0, x.shape[1]
    out = {"logp": x.new_zeros(n).index_put((rows,), lp.detach())}
    if s["op"] == "logprobs":
        top = torch.where(live, x.nan_to_num(nan=0.0, neginf=-math.inf).amax(1), 0.0)
        less_one = torch.where(live, torch.expm1(torch.logsumexp(x, 1) - top), -1.0)
        out["stats"] = torch.stack([top, less_one], 1)
        d1 = take(s["grad_logp"]).double()[rows]
        d2 = take(s["hess_logp"]).double()[rows] if s["hess"] else None
        value, want = (lp * d1).sum(), True
    else:
        fine = (lp.detach() != -math.inf)
        lps = torch.where(fine, lp, lp.new_zeros(()))
        adv, old = take(s["advantages"]).double()[rows], take(s["old_logp"]).double()[rows]
        w = torch.ones_like(adv) if s["weights"] is None else take(s["weights"]).double()[rows]
        w = torch.where(fine, w, 0.0)
        ratio = (lps - old).exp()
        each = torch.maximum(-adv * ratio, -adv * ratio.clamp(1 - s["low"], 1 + s["high"]))
        bent = torch.where(-adv * ratio.detach() >= each.detach(), (-adv * ratio.detach()).clamp(min=0), 0.0)
        if s["ref"]:
            t = take(s["ref_logp"]).double()[rows] - lps
            each = each + s["kl"] * (torch.expm1(t) - t)
            bent = bent + s["kl"] * t.detach().exp()
        each = torch.where(fine, w * each, 0.0)
        out["loss"] = x.new_zeros(n).index_put((rows,), each.detach())
        d2, value, want = w * bent, each.sum(), s["grad"]
        d1 = torch.autograd.grad(each.sum(), lp, retain_graph=True)[0] if want else None
    if want:
        out["grad"] = x.new_zeros(n, k).index_put((rows,), torch.autograd.grad(value, xs)[0].nan_to_num(nan=0.0))
        if s["hess"]:
            p = lp_all.detach().exp()
            lean = torch.nn.functional.one_hot(at, k) - p
            out["hess"] = x.new_zeros(n, k).index_put((rows,), d2[:, None] * lean ** 2 + d1.abs()[:, None] * (p - p * p))
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "preference":
        z = s["scores"].double().requires_grad_(True)
        lean = z - s["reference"].double() if case["ref"] else z * 1.0
        gap = lean[s["winners"]] - lean[s["losers"]]
        b, eps = case["beta"], case["smoothing"]
        if case["loss"] == "squared":
            each = (gap - 0.5 / b).square()
            curve = torch.full_like(gap, 2.0).detach()
        else:
            each = -(1 - eps) * torch.nn.functional.logsigmoid(b * gap) - eps * torch.nn.functional.logsigmoid(-b * gap)
            curve = (b / (2 * torch.cosh((b * gap.detach() / 2)))).square()
        if s["pair_weights"] is not None:
            each, curve = each * s["pair_weights"].double(), curve * s["pair_weights"].double()
        hess = torch.zeros_like(lean).detach().scatter_add_(0, s["winners"], curve).scatter_add_(0, s["losers"], curve)
        return {"loss": each.detach(), "grad": torch.autograd.grad(each.sum(), z)[0], "hess": hess}
    n, step, parts = case["n"], max(1, (1 << 25) // case["k"]), []
    for r0 in range(0, n, step):
        parts.append(_exact_rows(s, r0, min(n, r0 + step)))
    out = {key: torch.cat([p[key] for p in parts]) for key in parts[0]}
    for key in ("grad", "hess"):
        if key not in out and (case["op"] == "logprobs" or case["grad"]):
            out[key] = None
    return out
