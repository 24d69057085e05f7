"""Losses from feedback where they can go wrong: plans used at once, masks of
finite values, log ratios at the end of float64's range, and the like, against
plain float64 forms (feedback_util)."""
import math

import numpy as np
import pytest

import feedback_util as fu
from test_feedback import DTYPES, HALF_STEP, TINY, _close

gpu = pytest.mark.gpu


# ------------------------------------------------------------------- plans

@gpu
@pytest.mark.parametrize("n,P,turns", [(96, 48, 200), (3000, 4000, 60), (60_000, 200_000, 12)])
def test_plan_is_there_for_any_stream(mtlib, n, P, turns):
    """A plan made from recycled memory and used at once on a stream that
    does not wait for the legacy one, which has work of its own meanwhile.
    Per pair, in float64: x rounds to |x| steps, exp is within 2 + |x| steps,
    then 1 + e, its inverse and three products, or a log1p within 2 steps and a
    sum; both here and there, so 4 (14 + 4 |x|) half steps of a value below
    1 + |x| hold.  A gradient adds a pair's in any order and rounds to float32."""
    import torch
    rng = np.random.default_rng(n)
    side = torch.cuda.Stream()
    s = torch.from_numpy(rng.normal(size=n)).cuda()
    sd = s.cpu().numpy()
    x = 2 * np.abs(sd).max()
    term = 4 * (14 + 4 * x) * 2.0 ** -53
    busy = torch.zeros(1 << 26, device="cuda")
    torch.cuda.synchronize()
    for turn in range(turns):
        i = rng.integers(0, n, size=P)
        j = (i + 1 + rng.integers(0, n - 1, size=P)) % n
        busy.add_(1.0)  # the legacy stream is behind
        plan = mtlib.PreferencePlan(i, j, n)
        with torch.cuda.stream(side):
            loss, grad, hess = mtlib.preference_loss(plan, s)
        side.synchronize()
        L, g, h = fu.pairs_loss(sd, None, i, j, None, 1.0, 0.0, "logistic")
        assert np.abs(loss.cpu().numpy() - L).max() <= term * (1 + x), turn
        G = np.zeros(n)
        np.add.at(G, i, g)
        np.add.at(G, j, -g)
        degree = np.bincount(np.concatenate([i, j]), minlength=n)
        tol = np.abs(G) * fu.U32 * 1.01 + degree * (term + degree * 2.0 ** -52)
        assert (np.abs(grad.cpu().numpy() - G) <= tol).all(), turn


@gpu
def test_recycled_memory_keeps_its_size():
    """A plan that takes a somewhat larger block of recycled memory gives all
    of it back: the next plan of the larger size needs no new memory."""
    import os
    import subprocess
    import sys
    code = """
import numpy as np, torch
import mojoboost_b200 as mb
def plan(pairs):  # 16 bytes a pair: 9 and 8 units of 2 MB
    i = np.arange(pairs) % 999
    mb.PreferencePlan(i, i + 1, 1000)
    torch.cuda.synchronize()
    return torch.cuda.mem_get_info()[0]
torch.zeros(1, device="cuda")
large = plan(1_150_000)
assert plan(1_000_000) == large, "the block was not recycled"
print("free", large - plan(1_150_000))
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.split() == ["free", "0"], r.stdout + r.stderr


# -------------------------------------------------------------- parameters

def test_refused_bytes_in_a_message(mtlib):
    """A parameter that is not UTF-8 is refused as any other wrong one."""
    with pytest.raises(mtlib.MojoTreesError, match="integer"):
        mtlib.train_dense(np.arange(8.0).reshape(4, 2), np.zeros(4), b"num_leaves=\xff")

@pytest.mark.parametrize("params,k", [
    (None, 1), ("num_iterations=3", 1), ("num_class=3", 3), ({"num_classes": 3}, 3), (b"NUM_CLASS=3", 3), ("num_class=+3", 3),
    ("num_class=-3", -3), ("num_class=003", 3), ("num_class=3.0", None), ("num_class=--3", None), ("num_class=", None),
    ("num_class=\u0663", None), (b"num_class=\xff", None), ("verbosity=1\x0bnum_class=3", 3)])
def test_num_class_is_read_as_the_library_does(mtlib, params, k):
    from mojoboost_b200 import _feedback
    assert _feedback._num_class(params) == k
    X, zeros = np.arange(8.0).reshape(4, 2), np.zeros((4, 3))
    if k == 3:  # initial scores of that width are accepted (what remains is a device)
        if not mtlib.gpu_available():
            with pytest.raises(mtlib.UnsupportedError, match="CUDA"):
                mtlib.train_dense_policy(X, [0, 1, 2, 0], np.ones(4), params, initial_scores=zeros)
    else:
        with pytest.raises(mtlib.MojoTreesError, match="initial_scores" if k is not None else "integer") as e:
            mtlib.train_dense_policy(X, [0, 1, 2, 0], np.ones(4), params, initial_scores=zeros)
        assert e.value.code == -1


# ------------------------------------------------------------------- masks

def _bounds(z, a, f64):
    """(logp, stats, p, left, part) of float64 scores z, and error bounds from
    the kernels' arithmetic: of a log probability (absolute), each p, the
    others' sum and the largest class's complement (relative).

    A lane adds at most 16 terms (up to 128 classes, float64 512) or 33 (a
    lane's 8 vectors of 16 bytes in pairs, and an element at the row's edge),
    then 5 sums of lanes; warps are joined in float64.  float64 rows of more
    than 512 classes: ceil(K / 256) in a thread.  An exponential's own error is
    fu.exp_error; a row's statistics and scalars round up to 10 times on the way
    to a gradient."""
    logp, stats, p, left, part = fu.softmax_rows(z, a)
    K = z.shape[1]
    unit = 2.0 ** -53 if f64 else fu.U32
    adds = 16 if K <= (512 if f64 else 128) else -(-K // 256) if f64 else 33
    with np.errstate(invalid="ignore"):
        d = np.where(np.isfinite(z), z - stats[:, :1], -np.inf)
    e_exp = np.where(p > 0, fu.exp_error(d, f64), 0.0)
    e_sum = (p * e_exp).sum(1) + (adds + 5) * unit
    others = p.copy()
    others[np.arange(len(z)), z.argmax(1)] = 0.0
    total = others.sum(1)
    e_rest = np.where(total > 0, (others * e_exp).sum(1) / np.where(total > 0, total, 1.0), 0.0) + (adds + 5) * unit
    e_rest = 2 * e_rest + 2 * unit  # the sum less 1, where it is 1 and more
    e_l = e_sum + np.where(np.isfinite(logp), np.abs(logp), 0.0) * (2 * unit) + 2.0 ** -52
    e_p = e_exp + e_sum[:, None] + 10 * unit
    return logp, stats, p, left, part, e_l, e_p, e_rest, e_rest + 10 * unit + (2.0 ** -42 if f64 else 0.0)


def _check_logprobs(mtlib, x, a_t, z, a, dtype):
    """action_logprobs and its way back on scores x (z in float64) within _bounds."""
    import torch
    f64 = dtype == "float64"
    n, K = z.shape
    logp, stats, p, left, part, e_l, e_p, e_rest, e_left = _bounds(z, a, f64)
    got_l, got_s = mtlib.action_logprobs(x, a_t)
    _close(got_l, logp, e_l, "logp")
    _close(got_s[:, 0], stats[:, 0], 0.0, "maximum")
    _close(got_s[:, 1], stats[:, 1], np.abs(stats[:, 1]) * e_rest + TINY[dtype] * K, "sum less 1")
    rng = np.random.default_rng(K)
    g, h = rng.normal(size=n).astype(np.float32), rng.random(n).astype(np.float32)
    got_g, got_h = mtlib.action_logprobs_grad(x, a_t, got_s, torch.from_numpy(g).cuda(), torch.from_numpy(h).cuda())
    G, H, q = fu.to_scores(p, left, a, part, g.astype(np.float64), h.astype(np.float64))
    tol_q = np.where(q > 0, np.maximum(e_left[:, None], e_p), e_p)
    # 1 - p of the largest class by the others' share, of the rest within p's error of a value of at least a half
    tol_h = 2 * tol_q + e_p + e_left[:, None]
    half, tiny = HALF_STEP[dtype], TINY[dtype] * 4
    _close(got_g, G, np.abs(G) * (tol_q + half) * 1.01 + tiny, "grad")
    _close(got_h, H, H * (tol_h + half) * 1.01 + tiny, "hess")


def _check_policy(got, z, a, adv, old, ref, low, high, kl, dtype):
    """policy_loss's four outputs within _bounds: with e the bound of l, the
    loss is off by |dloss/dl| e and a few roundings of its float64 terms, and
    dloss/dl by its own derivative times e (away from the clip range's ends)."""
    n, f64 = len(z), dtype == "float64"
    logp, stats, p, left, part, e_l, e_p, e_rest, e_left = _bounds(z, a, f64)
    loss, g, h, part = fu.policy_rows(logp, part, adv.astype(np.float64), old.astype(np.float64),
                                      None if ref is None else ref.astype(np.float64), None, low, high, kl)
    unit = 2.0 ** -53 if f64 else fu.U32
    l = np.where(part, logp, 0.0)
    ra = np.abs(np.exp(l - old) * adv)
    et = np.zeros(n) if ref is None else np.exp(ref - l)
    far = 0.0 if ref is None else 1 + np.abs(ref - l)
    step = 2.0 ** -50 * (1 + np.abs(l) + np.abs(old))
    e_g = np.where(part, (ra + kl * et) * (e_l * 1.01 + step), 0.0)
    _close(got[1], logp, e_l, "logp")
    _close(got[0], loss, np.where(part, (np.abs(g) + e_g) * e_l + (ra + kl * (et + far)) * step, 0.0) + np.abs(loss) * 2 * unit
           + TINY["float32"], "loss")
    G, H, q = fu.to_scores(p, left, a, part, g, h)
    tol_q = np.where(q > 0, np.maximum(e_left[:, None], e_p), e_p)
    tol_h = 2 * tol_q + e_p + e_left[:, None]
    half, tiny, e_g = HALF_STEP[dtype], TINY[dtype] * 4, e_g[:, None]
    _close(got[2], G, (np.abs(q) * e_g + np.abs(G) * (tol_q + half)) * 1.01 + tiny, "grad")
    _close(got[3], H, ((q * q + p * left) * 2 * e_g + H * (tol_h + half)) * 1.01 + tiny, "hess")


MASKS = ["-inf", -1e4, -1e7, -1e9, -1e10, -1e12, -1e20, -1e30, "lowest"]


def _masked_rows(seed, K, dtype, mask):
    """Rows with masked classes: none, single ones, all but three next to one
    another, all but one, all but the first or last, all; the class taken
    allowed but in one row."""
    import torch
    rng = np.random.default_rng(seed)
    t = getattr(torch, dtype)
    low = -math.inf if mask == "-inf" else torch.finfo(t).min if mask == "lowest" else max(mask, torch.finfo(t).min)
    allowed = [np.ones(K, bool), rng.random(K) < 0.7, np.zeros(K, bool), np.zeros(K, bool), np.zeros(K, bool), np.zeros(K, bool),
               np.zeros(K, bool), rng.random(K) < 0.5]
    at = int(rng.integers(0, K - 3))
    allowed[2][at:at + 3] = True
    allowed[3][at] = True
    allowed[4][0] = allowed[5][K - 1] = True
    z = rng.normal(size=(len(allowed), K)) * 2
    a = np.zeros(len(allowed), np.int64)
    for r, ok in enumerate(allowed):
        z[r, ~ok] = low
        a[r] = rng.choice(np.flatnonzero(ok)) if ok.any() else 1
    a[7] = np.flatnonzero(~allowed[7])[0]
    x = torch.from_numpy(z).to(t).cuda()
    return x, x.double().cpu().numpy(), torch.from_numpy(a).cuda(), a


WIDTHS = [5, 64, 128, 129, 300, 600, 1025, 5000, 20_001, 50_001, 131_072]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K", WIDTHS)
def test_masks_of_any_value(mtlib, K, dtype):
    """A mask is as good as -inf from where its probability is 0 on, and a row
    that holds nothing else is uniform (of -inf: takes no part)."""
    import torch
    t = torch.float64 if dtype == "float64" else torch.float32
    for mask in MASKS:
        x, z, a_t, a = _masked_rows(K, K, dtype, mask)
        _check_logprobs(mtlib, x, a_t, z, a, dtype)
        rng = np.random.default_rng(1)
        logp = fu.softmax_rows(z, a)[0]
        near = np.where(np.isfinite(logp), logp, -1.0)
        near = np.maximum(near, -80)  # the masked class that a row took: a ratio of 0
        adv = rng.normal(size=len(z))
        old, ref = near + 0.2 * rng.normal(size=len(z)), near + 0.3 * rng.normal(size=len(z))
        rows = [torch.from_numpy(v).to(t).cuda() for v in (adv, old, ref)]
        back = [v.cpu().numpy() for v in rows]
        for n, kl in ((len(z), 0.0), (7, 0.3)):  # exp(ref - l) of a masked class that was taken has no end
            got = mtlib.policy_loss(x[:n], a_t[:n], rows[0][:n], rows[1][:n], ref_logp=rows[2][:n], kl_coef=kl, clip_high=0.3, hess=True)
            _check_policy(got, z[:n], a[:n], back[0][:n], back[1][:n], back[2][:n] if kl else None, 0.2, 0.3, kl, dtype)


@gpu
@pytest.mark.parametrize("dtype", ["float64", "float32", "bfloat16"])
@pytest.mark.parametrize("K", WIDTHS)
def test_scores_of_any_size(mtlib, K, dtype):
    """Rows that lie far from 0 as a whole, on both sides of where the kernels
    take the maximum out first, and up to the ends of the type."""
    import torch
    t = getattr(torch, dtype)
    rng = np.random.default_rng(K)
    far = [0.0, 1e3, 2.0 ** 22, 2.0 ** 23 - 4, 2.0 ** 23 + 4, 2.0 ** 24 - 8, 2.0 ** 24 + 8, 2.0 ** 26, 1e9, 1e10, 1e20, 1e30]
    far = far + [-v for v in far[1:]] + [torch.finfo(t).max, torch.finfo(t).min]
    z = rng.normal(size=(len(far), K)) * 3
    for r, v in enumerate(far):
        at = np.float64(torch.tensor(v, dtype=t))
        step = abs(at) * torch.finfo(t).eps if v else 1.0  # a class now and then is a step or two below
        if step > 1e30:  # the type's ends: the row's other classes are at 0
            z[r] = np.where(rng.random(K) < 0.5, at, 0.0) if v > 0 else at
            z[r, 0] = at
        else:
            z[r] = np.where(rng.random(K) < 0.5, at, at - max(step, 1.0) * rng.integers(1, 3, size=K))
    x = torch.from_numpy(z).to(t).cuda()
    z = x.double().cpu().numpy()
    a = z.argmax(1)
    a[::2] = rng.integers(0, K, size=len(a[::2]))
    a_t = torch.from_numpy(a).cuda()
    _check_logprobs(mtlib, x, a_t, z, a, dtype)
    row = torch.float64 if dtype == "float64" else torch.float32
    logp = fu.softmax_rows(z, a)[0]
    rows = [torch.from_numpy(v).to(row).cuda() for v in (rng.normal(size=len(z)), np.maximum(logp, -80) + 0.2 * rng.normal(size=len(z)))]
    back = [v.cpu().numpy() for v in rows]
    got = mtlib.policy_loss(x, a_t, *rows, clip_high=0.3, hess=True)
    _check_policy(got, z, a, *back, None, 0.2, 0.3, 0.0, dtype)


@gpu
@pytest.mark.parametrize("dtype,K", [("float32", 129), ("float32", 40_000), ("bfloat16", 200), ("bfloat16", 131_072)])
def test_clip_border_of_far_rows(mtlib, dtype, K):
    """As test_clip_border_is_decided_in_float64, for rows at 1e12 whose
    classes lie apart by more than an exponential tells, so that 1 to 64 of them
    share the probability."""
    import torch
    n = 64
    rng = np.random.default_rng(K)
    top = float(torch.tensor(1e12, dtype=getattr(torch, dtype)))
    z = np.full((n, K), 0.0)
    for r in range(n):
        z[r, rng.permutation(K)[:r + 1]] = top
    a = z.argmax(1)
    x = torch.from_numpy(z).to(getattr(torch, dtype)).cuda()
    adv = np.where(np.arange(n) % 2 == 0, 1.0, -1.0)
    logp = -np.log(np.arange(n) + 1.0)
    end = np.where(adv > 0, math.log1p(0.3), math.log1p(-0.2))
    old = (logp - end - rng.choice([-1, 1], size=n) * 10.0 ** rng.uniform(-9, -6, size=n)).astype(np.float32)
    d = logp - old.astype(np.float64)
    clear = np.abs(d - end) > 1e-12
    t = [torch.from_numpy(v.astype(np.float32)).cuda() for v in (adv, old)]
    grad = mtlib.policy_loss(x, torch.from_numpy(a).cuda(), *t, clip_low=0.2, clip_high=0.3)[2]
    moved = (grad != 0).any(1).cpu().numpy()
    active = np.where(adv > 0, d <= end, d >= end)
    active[0] = False  # one class has it all: a gradient of 0 either way
    np.testing.assert_array_equal(moved[clear], active[clear])


# ------------------------------------------------------- the end of float64's range

FAR_RATIOS = [-800.0, -708.5, -707.5, 600.0, 708.9, 709.1, 709.7, 709.77, 709.7773, 709.779, 709.78, 709.781, 709.7827, 709.783, 709.79, 710.0, 1e4]


@gpu
@pytest.mark.parametrize("K", [3, 40, 600])
@pytest.mark.parametrize("end", ["ratio", "reference"])
def test_log_ratios_up_to_the_end_of_float64(mtlib, K, end):
    """e^d of a log ratio or of the reference's distance is right up to
    float64's largest and infinite beyond; a clipped row keeps its finite loss."""
    import torch
    rng = np.random.default_rng(K)
    d = np.repeat(FAR_RATIOS, 2)
    n = len(d)
    x, a = rng.normal(size=(n, K)), rng.integers(0, K, size=n)
    logp = fu.softmax_rows(x, a)[0]
    adv, old, ref, kl = np.where(np.arange(n) % 2 == 0, -1e-300, 1e-300), logp - d, None, 0.0
    if end == "reference":
        adv, old, ref, kl = np.zeros(n), logp.copy(), logp + d, 1e-300
    t = [None if v is None else torch.from_numpy(v).cuda() for v in (x, a, adv, old, ref)]
    got = mtlib.policy_loss(t[0], t[1], t[2], t[3], ref_logp=t[4], clip_low=0.2, clip_high=0.3, kl_coef=kl, hess=True)
    with np.errstate(over="ignore"):
        loss, g, h, part = fu.policy_rows(logp, np.ones(n, bool), adv, old, ref, None, 0.2, 0.3, kl)
        # where the oracle's own d decides between finite and infinite
        clear = np.isfinite(np.exp(np.abs(d) + 1e-9)) | ~np.isfinite(np.exp(np.abs(d) - 1e-9))
    step = 2.0 ** -50 * (1 + np.abs(logp) + np.abs(logp - d))
    have = got[0].cpu().numpy()
    assert not np.isnan(have).any() and not any(v.isnan().any() for v in got[1:3])
    fine = clear & np.isfinite(loss)
    np.testing.assert_array_equal(have[clear & ~fine], loss[clear & ~fine])
    # exp is 0 below -708: off by at most e^-708 there
    tol = np.abs(loss) * step + (np.abs(adv) + kl) * (np.exp(-708) + 2.0 ** -52 * (1 + np.abs(d)))
    assert (np.abs(have[fine] - loss[fine]) <= tol[fine]).all()
    grad = got[2].double().cpu().numpy()[np.arange(n), a]
    q = 1 - np.exp(logp)
    small = fine & (np.abs(g) < 1e38)
    tol = np.abs(g) * q * (fu.U32 * 1.01 + step + 2.0 ** -40) + 2.0 ** -149
    assert (np.abs(grad[small] - (g * q)[small]) <= tol[small]).all()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K", [3, 10, 40, 128, 300, 600, 5000])
def test_infinite_derivatives(mtlib, K, dtype):
    """A ratio beyond the derivatives' type: the row's gradient and hessian are
    infinite, with the gradient's signs, and not NaN; other rows are theirs."""
    import torch
    t = torch.float64 if dtype == "float64" else torch.float32
    rng = np.random.default_rng(K)
    x = torch.from_numpy(rng.normal(size=(4, K))).to(getattr(torch, dtype)).cuda()
    a = torch.tensor([0, 1, 2, K - 1], device="cuda")
    logp, _ = mtlib.action_logprobs(x, a)
    # minus an advantage of 1: every class has probability, and the ratio is e^150 or 1
    old = logp - torch.tensor([150.0, 0.0, 150.0, 0.0], device="cuda", dtype=t)
    loss, _, G, H = mtlib.policy_loss(x, a, -torch.ones(4, device="cuda", dtype=t), old, hess=True)
    taken = torch.zeros(4, K, dtype=torch.bool, device="cuda").scatter_(1, a[:, None], True)
    for r in (0, 2):
        assert (H[r] == math.inf).all()
        assert torch.equal(G[r], torch.where(taken[r], math.inf, -math.inf).to(G.dtype))
    assert torch.isfinite(G[1::2]).all() and torch.isfinite(H[1::2]).all()
    assert torch.isfinite(loss[1::2]).all() and (loss[::2] > 1e38).all()


# ------------------------------------------------------------------- pairs

@gpu
@pytest.mark.parametrize("beta", [0.1, 0.37, 3.0])
@pytest.mark.parametrize("size", [1.0, 40.0, 900.0])
def test_squared_loss_next_to_its_target(mtlib, beta, size):
    """float32 scores and references whose difference is next to 1 / (2 beta):
    u is known to its parts' rounding errors (2^-46 of the items' distances to
    their references), u - 1 / (2 beta) is rounded once, and its square and
    double once more each; float32 holds the results."""
    import torch
    rng = np.random.default_rng(int(size))
    P = 4000
    target = 1 / (2 * beta)
    ref = (rng.normal(size=2 * P) * size - size).astype(np.float32)
    s = (ref + rng.normal(size=2 * P)).astype(np.float32)
    i, j = np.arange(P), P + np.arange(P)
    lean = s.astype(np.float64) - ref
    s[:P] = (target + lean[j] + ref[:P]).astype(np.float32)
    step = np.abs(np.spacing(s[:P])).astype(np.float64)
    s[:P] = (s[:P] + step * rng.integers(-3, 4, size=P)).astype(np.float32)
    lean = s.astype(np.float64) - ref
    plan = mtlib.PreferencePlan(i, j, 2 * P)
    got = mtlib.preference_loss(plan, torch.from_numpy(s).cuda(), reference=torch.from_numpy(ref).cuda(), beta=beta, loss="squared")
    d = (lean[i] - lean[j]) - target
    off = 2.0 ** -46 * (np.abs(lean[i]) + np.abs(lean[j])) + 2.0 ** -52 * target
    e = np.abs(d) * fu.U32 + off
    _close(got[0], d * d, 2 * np.abs(d) * e + e * e + d * d * 2 * fu.U32 + 2.0 ** -126, "loss")
    _close(got[1][:P], 2 * d, 2 * e + 2.0 ** -126, "grad of the winners")
    assert torch.equal(got[1][P:], -got[1][:P]) and (got[2] == 2).all()


@gpu
@pytest.mark.parametrize("dtype,beta", [("float64", 1e160), ("float64", 1e307), ("float32", 1e20), ("float32", 1e37)])
def test_logistic_loss_of_large_beta(mtlib, dtype, beta):
    """A beta whose square is beyond the type: pairs that are told apart have
    a hessian of 0 and a gradient of 0 or -beta, equal ones log 2 and -beta / 2."""
    import torch
    s = torch.tensor([1.0, 0.0, 0.0, 1.0, 2.0, 2.0], dtype=getattr(torch, dtype), device="cuda")
    loss, grad, hess = mtlib.preference_loss(mtlib.PreferencePlan([0, 2, 4], [1, 3, 5], 6), s, beta=beta)
    want = [0.0, beta, math.log(2)]
    assert np.allclose(loss.double().cpu().numpy(), want, rtol=2.0 ** -22, atol=0)
    big = beta if beta < 3e38 else math.inf
    assert np.allclose(grad.double().cpu().numpy(), [0, 0, -big, big, -big / 2, big / 2], rtol=2.0 ** -22, atol=0)
    assert hess[:4].tolist() == [0.0] * 4 and (hess[4:] > 1e38).all()
    if dtype == "float32":
        with pytest.raises(mtlib.MojoTreesError, match="beyond float32"):
            mtlib.preference_loss(mtlib.PreferencePlan([0], [1], 6), s, beta=1e39)


# -------------------------------------------------------------------- fits

@gpu
@pytest.mark.parametrize("K", [2, 5, 20])
def test_first_round_lies_inside_any_clip_range(mtlib, K):
    """Without old_logp the first round's ratios are 1: no row is clipped, a
    range of no width included, and the reference is no distance away."""
    n = 3000
    rng = np.random.default_rng(K)
    bins = rng.integers(0, 32, size=(5, n)).astype(np.uint8)
    actions, adv, init = rng.integers(0, K, size=n), rng.normal(size=n), rng.normal(size=(n, K)) * 3
    params = {"num_class": K, "num_iterations": 1, "num_leaves": 15, "min_data_in_leaf": 5, "gpu_histogram_precision": "int64"}
    wide = mtlib.train_binned_policy(bins, 32, actions, adv, params, initial_scores=init)
    none = mtlib.train_binned_policy(bins, 32, actions, adv, dict(params, policy_clip_low=0, policy_clip_high=0), initial_scores=init)
    for k in range(K):
        for name in ("feature", "threshold_bin", "count", "value"):
            np.testing.assert_array_equal(wide.tree(k)[name], none.tree(k)[name])
