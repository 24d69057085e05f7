"""Losses from feedback on device scores: log probabilities of taken classes,
clipped policy loss, paired preference loss, against plain float64 forms.

Tolerances follow from the kernels' arithmetic (feedback_util: exp_error,
sum_error): with e the bound on a log probability's absolute error, a value
f(l) is held to |f'(l)| e and its own rounding.
"""
import ctypes
import math

import numpy as np
import pytest

import feedback_util as fu

gpu = pytest.mark.gpu

DTYPES = ["float64", "float32", "float16", "bfloat16"]
# half a step of each type, relative; the smallest subnormal's half for float16
HALF_STEP = {"float64": 2.0 ** -24, "float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
TINY = {"float64": 2.0 ** -149, "float32": 2.0 ** -126, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -126}


# ------------------------------------------------------------------ refusals

@pytest.fixture
def err(mtlib):
    e = mtlib.lib().mojotrees_error_create()
    yield e
    mtlib.lib().mojotrees_error_free(e)


# a host address: every refusal below comes before any array is looked at
HOST = np.zeros(64)
P = HOST.ctypes.data


def _logprobs(lib, e, scores=P, kind=1, n=2, k=3, stride=3, actions=P, bytes_=4, logp=P, stats=P):
    return lib.mojotrees_b200_action_logprobs(scores, kind, n, k, stride, actions, bytes_, logp, stats, None, e)


@pytest.mark.parametrize("kw,needle", [
    (dict(scores=None), "null"), (dict(actions=None), "null"), (dict(logp=None), "null"), (dict(stats=None), "null"),
    (dict(kind=4), "score type"), (dict(kind=-1), "score type"), (dict(n=-1), "n_rows"), (dict(k=0), "n_classes"),
    (dict(k=262145, stride=262145), "n_classes"), (dict(stride=2), "row_stride"), (dict(bytes_=2), "actions"),
    (dict(n=1 << 40, stride=1 << 20), "too large"), (dict(scores=P + 2), "aligned"), (dict(actions=P + 4, bytes_=8), "aligned"),
    (dict(logp=P + 2), "aligned"), (dict(stats=P + 1), "aligned"), (dict(kind=0, logp=P + 4), "aligned"),
])
def test_logprobs_refusals(mtlib, err, kw, needle):
    assert _logprobs(mtlib.lib(), err, **kw) == -1
    assert needle in mtlib.lib().mojotrees_error_message(err).decode()


def _back(lib, e, stats=P, g=P, h=None, og=P, oh=None, ostride=3):
    return lib.mojotrees_b200_action_logprobs_grad(P, 1, 2, 3, 3, P, 4, stats, g, h, og, oh, ostride, None, e)


@pytest.mark.parametrize("kw,needle", [
    (dict(stats=None), "null"), (dict(g=None), "null"), (dict(og=None), "null"), (dict(h=P), "go together"),
    (dict(oh=P), "go together"), (dict(ostride=2), "out_stride"), (dict(g=P + 2), "aligned"), (dict(og=P + 1), "aligned"),
])
def test_logprobs_grad_refusals(mtlib, err, kw, needle):
    assert _back(mtlib.lib(), err, **kw) == -1
    assert needle in mtlib.lib().mojotrees_error_message(err).decode()


def _policy(lib, e, adv=P, old=P, ref=P, low=0.2, high=0.2, kl=0.1, loss=P, og=P, oh=None, ostride=3, n=2):
    return lib.mojotrees_b200_policy_loss(P, 1, n, 3, 3, P, 4, adv, old, ref, None, low, high, kl, loss, None, og, oh,
                                          ostride, None, e)


@pytest.mark.parametrize("kw,needle", [
    (dict(adv=None), "null"), (dict(old=None), "null"), (dict(loss=None), "null"), (dict(ref=None), "ref_logp"),
    (dict(low=-0.1), "clip_low"), (dict(low=1.1), "clip_low"), (dict(low=math.nan), "clip_low"),
    (dict(high=-0.1), "clip_high"), (dict(high=math.nan), "clip_high"), (dict(kl=-1.0), "kl_coef"),
    (dict(kl=math.inf), "kl_coef"), (dict(kl=math.nan), "kl_coef"), (dict(og=None, oh=P), "out_grad"),
    (dict(ostride=1), "out_stride"), (dict(adv=P + 2), "aligned"), (dict(og=P + 2), "aligned"),
])
def test_policy_refusals(mtlib, err, kw, needle):
    assert _policy(mtlib.lib(), err, **kw) == -1
    assert needle in mtlib.lib().mojotrees_error_message(err).decode()


@pytest.mark.parametrize("w,l,n,weights,needle", [
    ([0, 1], [1, 2], 2, None, "out of range"), ([0, -1], [1, 0], 2, None, "out of range"),
    ([0, 1], [1, 1], 2, None, "paired with itself"), ([0], [1], 2, [-1.0], "weights"),
    ([0], [1], 2, [math.nan], "weights"), ([0], [1], 2, [math.inf], "weights"), ([0], [1], -1, None, "non-negative"),
    ([0, 1], [1], 2, None, "one length"), ([[0]], [[1]], 2, None, "one-dimensional"), ([0.5], [1], 2, None, "integers"),
    ([0], [1], 2, [1.0, 1.0], "one length"), ([0], [1], 1 << 31, None, "items"),
])
def test_plan_refusals(mtlib, w, l, n, weights, needle):
    with pytest.raises(mtlib.MojoTreesError, match=needle):
        mtlib.PreferencePlan(w, l, n, weights=weights)


def test_no_device_is_unsupported(mtlib, err):
    if mtlib.gpu_available():
        pytest.skip("a GPU is present")
    lib = mtlib.lib()
    assert _logprobs(lib, err) == -4 and _back(lib, err) == -4 and _policy(lib, err) == -4
    assert b"CUDA" in lib.mojotrees_error_message(err)
    with pytest.raises(mtlib.UnsupportedError):
        mtlib.PreferencePlan([0], [1], 2)
    assert lib.mojotrees_b200_preference_loss(None, P, None, 0, 1.0, 0.0, 0, P, P, P, None, err) == -1
    lib.mojotrees_b200_preference_plan_free(None)


def test_python_refuses_host_tensors(mtlib):
    import torch
    with pytest.raises(mtlib.MojoTreesError, match="CUDA device"):
        mtlib.action_logprobs(torch.zeros(2, 3), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(mtlib.MojoTreesError, match="float64"):
        mtlib.policy_loss(torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), None, None)


# ------------------------------------------------------------- row operators

def _inputs(seed, n, K, dtype, mask=False, ids="int32", pad=0, spread=2.0):
    """Scores (a torch view with `pad` columns behind it) with their float64
    values, and actions.  mask: classes of -inf, rows without a class, rows
    that took a masked class, rows of NaN that take no part."""
    import torch
    rng = np.random.default_rng(seed)
    z = rng.normal(size=(n, K)) * spread
    a = rng.integers(0, K, size=n)
    if K > 64:
        z[np.arange(n), a] += rng.uniform(0, 12, size=n)
    if mask:
        off = rng.random((n, K)) < 0.3
        off[np.arange(n), a] = rng.random(n) < 0.1
        off |= rng.random((n, 1)) < 0.05
        z[off] = -np.inf
        dead = rng.random(n) < 0.1
        z[dead] = np.nan
        a[dead] = -1 - rng.integers(0, 100, size=dead.sum())
    buf = torch.zeros((n, K + pad), dtype=getattr(torch, dtype))
    buf[:, :K] = torch.from_numpy(z).to(buf.dtype)
    buf = buf.cuda()
    x = buf[:, :K]
    return x, x.double().cpu().numpy(), torch.from_numpy(a).to(getattr(torch, ids)).cuda(), a


def _close(got, want, tol, what):
    got = got.double().cpu().numpy()
    fine = np.isfinite(want)
    np.testing.assert_array_equal(got[~fine], want[~fine], err_msg=what)
    off = np.abs(got[fine] - want[fine])
    tol = np.broadcast_to(tol, want.shape)[fine]
    assert np.all(off <= tol), f"{what}: {np.max(off - tol)} over the bound {tol[np.argmax(off - tol)]}"


def _row_bounds(z, p, stats, logp, f64):
    """Bounds: of a log probability (absolute), of each p (relative), of rest/(1+rest) (relative)."""
    with np.errstate(invalid="ignore"):
        d = np.where(np.isfinite(z), z - stats[:, :1], -np.inf)
    e_sum = fu.sum_error(z.shape[1], p, d, f64)
    unit = 2.0 ** -53 if f64 else fu.U32
    l = np.where(np.isfinite(logp), np.abs(logp), 0.0)
    e_l = e_sum + 2 * l * unit + 2.0 ** -52
    e_p = fu.exp_error(d, f64) + e_sum[:, None] + 4 * unit
    # the largest class's complement sums the others: each term's own error
    with np.errstate(invalid="ignore"):
        far = np.where(p > 0, fu.exp_error(d, f64), 0.0).max(1)
    e_left = far + (min(z.shape[1], 16) + z.shape[1] // 256 + 4) * unit + e_sum + 4 * unit
    return e_l, e_p, e_left


SIZES = [(1, 1), (3, 2), (37, 5), (64, 10), (33, 31), (40, 32), (41, 33), (16, 64), (17, 65), (9, 127), (9, 128),
         (9, 129), (5, 175), (7, 255), (6, 512), (5, 1000), (3, 1025), (3, 4099), (2, 16384), (2, 16391), (2, 50001),
         (1, 131072), (1, 262144), (0, 7), (300, 7), (257, 3), (1025, 10)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,K", SIZES)
def test_logprobs_and_gradient(mtlib, n, K, dtype):
    import torch
    f64 = dtype == "float64"
    for mask, pad, ids in ((False, 0, "int32"), (True, 0, "int64"), (True, 1, "int32"), (False, 8, "int64")):
        x, z, a_t, a = _inputs(n * 31 + K, n, K, dtype, mask, ids, pad)
        logp, stats, p, left, part = fu.softmax_rows(z, a)
        got_l, got_s = mtlib.action_logprobs(x, a_t)
        assert got_l.dtype == (torch.float64 if f64 else torch.float32) and got_s.shape == (n, 2)
        if n == 0:
            continue
        unit = 2.0 ** -53 if f64 else fu.U32
        e_l, e_p, e_left = _row_bounds(z, p, stats, logp, f64)
        _close(got_l, logp, e_l, "logp")
        _close(got_s[:, 0], stats[:, 0], 0.0, "maximum")
        _close(got_s[:, 1], stats[:, 1], np.abs(stats[:, 1]) * (e_left + e_l + 2 * unit) * (1 + np.maximum(stats[:, 1], 0)), "sum less 1")
        rng = np.random.default_rng(K)
        g = rng.normal(size=n).astype(np.float32)
        h = rng.random(n).astype(np.float32)
        g_t, h_t = torch.from_numpy(g).cuda(), torch.from_numpy(h).cuda()
        G, H, q = fu.to_scores(p, left, a, part, g.astype(np.float64), h.astype(np.float64))
        tol_q = np.where(q > 0, np.maximum(e_left[:, None], e_p), e_p)
        half, tiny = HALF_STEP[dtype], TINY[dtype]
        for with_h in (True, False):
            got_g, got_h = mtlib.action_logprobs_grad(x, a_t, got_s, g_t, h_t if with_h else None)
            _close(got_g, G, np.abs(G) * (tol_q + half) * 1.01 + tiny, "grad")
            if with_h:
                _close(got_h, H, H * (2 * tol_q + e_p + e_left[:, None] + half) * 1.01 + tiny, "hess")
            else:
                assert got_h is None


def _policy_rows(seed, n, f64, logp, with_ref, with_w):
    rng = np.random.default_rng(seed)
    t = np.float64 if f64 else np.float32
    l = np.where(np.isfinite(logp), logp, -1.0)
    adv = rng.normal(size=n).astype(t)
    old = np.minimum(l + 0.25 * rng.normal(size=n), 0).astype(t)
    ref = np.minimum(l + 0.4 * rng.normal(size=n), 0).astype(t) if with_ref else None
    w = None
    if with_w:
        w = (rng.random(n) * 2).astype(t)
        w[rng.random(n) < 0.2] = 0
    return adv, old, ref, w


def _check_policy(got, z, a, adv, old, ref, w, low, high, kl, dtype):
    """policy_loss's four outputs against the plain form on float64 scores z."""
    n, f64 = len(z), dtype == "float64"
    wide = [None if v is None else v.astype(np.float64) for v in (adv, old, ref, w)]
    logp, stats, p, left, part = fu.softmax_rows(z, a, wide[3])
    loss, g, h, part2 = fu.policy_rows(logp, part, *wide, low, high, kl)
    e_l, e_p, e_left = _row_bounds(z, p, stats, logp, f64)
    unit = 2.0 ** -53 if f64 else fu.U32
    l = np.where(part2, logp, 0.0)
    ww = np.where(part2, 1.0 if w is None else wide[3], 0.0)
    ra = np.abs(np.exp(l - wide[1]) * wide[0])
    et = np.exp(wide[2] - l) if ref is not None else np.zeros(n)
    # a rounded step of the float64 scalars: exp of a sum of a few units
    step = 2.0 ** -50 * (1 + np.abs(l) + np.abs(wide[1]))
    e_g = ww * ((ra + kl * et) * (e_l * 1.01 + step))
    _close(got[1], logp, e_l, "logp")
    _close(got[0], loss, (np.abs(g) + e_g) * e_l + ww * (ra + kl * (et + 1 + np.abs(l) + np.abs(wide[2] if ref is not None else 0))) * step
           + np.abs(loss) * unit * 2 + TINY["float32"], "loss")
    G, H, q = fu.to_scores(p, left, a, part2, g, h)
    tol_q = np.where(q > 0, np.maximum(e_left[:, None], e_p), e_p)
    half, tiny = HALF_STEP[dtype], TINY[dtype]
    eg, unit_c = e_g[:, None] * 1.01, 4 * unit
    _close(got[2], G, (np.abs(q) * eg + np.abs(G) * (tol_q + half + unit_c)) * 1.01 + tiny, "grad")
    if got[3] is not None:
        _close(got[3], H, ((q * q + p * left) * 2 * eg + H * (2 * tol_q + e_p + e_left[:, None] + half + unit_c)) * 1.02 + tiny, "hess")


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,K", SIZES)
def test_policy_loss(mtlib, n, K, dtype):
    import torch
    f64 = dtype == "float64"
    low, high = 0.2, 0.3
    for mask, pad, with_ref, with_w, kl in ((False, 0, True, False, 0.04), (True, 0, True, True, 0.5),
                                            (True, 3, False, True, 0.0), (False, 8, True, False, 0.0)):
        x, z, a_t, a = _inputs(n * 37 + K, n, K, dtype, mask, "int64" if pad else "int32", pad)
        adv, old, ref, w = _policy_rows(K, n, f64, fu.softmax_rows(z, a)[0], with_ref, with_w)
        args = [torch.from_numpy(v).cuda() if v is not None else None for v in (adv, old, ref, w)]
        got = mtlib.policy_loss(x, a_t, args[0], args[1], ref_logp=args[2], weights=args[3], clip_low=low,
                                clip_high=high, kl_coef=kl, grad=True, hess=True)
        if n == 0:
            assert got[2].shape == (0, K)
            continue
        _check_policy(got, z, a, adv, old, ref, w, low, high, kl, dtype)
        alone = mtlib.policy_loss(x, a_t, args[0], args[1], ref_logp=args[2], weights=args[3], clip_low=low,
                                  clip_high=high, kl_coef=kl, grad=False)
        assert alone[2] is None and alone[3] is None
        assert torch.equal(alone[0], got[0]) and torch.equal(alone[1], got[1])
        no_h = mtlib.policy_loss(x, a_t, args[0], args[1], ref_logp=args[2], weights=args[3], clip_low=low,
                                 clip_high=high, kl_coef=kl)
        assert torch.equal(no_h[2], got[2]) and no_h[3] is None


@gpu
def test_policy_gradient_by_differences(mtlib):
    """Central differences of the summed loss in float64: error (step^2 / 6)
    times the third derivative (below 8 |A| r + kl e^t ~ 40) and 2^-52 |L| / step."""
    import torch
    n, K, step = 64, 6, 2.0 ** -13
    x, z, a_t, a = _inputs(5, n, K, "float64")
    adv, old, ref, w = [torch.from_numpy(v).cuda() for v in _policy_rows(1, n, True, fu.softmax_rows(z, a)[0], True, True)]
    ends = [math.log1p(-0.2), math.log1p(0.3)]

    def run(v):
        return mtlib.policy_loss(v, a_t, adv, old, ref_logp=ref, weights=w, clip_low=0.2, clip_high=0.3, kl_coef=0.1)

    loss, logp, grad, _ = run(x)
    smooth = torch.stack([(logp - old - e).abs() for e in ends]).amin(0) > 4 * step
    assert smooth.sum() > n // 2
    for k in range(K):
        up, down = x.clone(), x.clone()
        up[:, k] += step
        down[:, k] -= step
        diff = (run(up)[0] - run(down)[0]) / (2 * step)
        assert (diff - grad[:, k].double()).abs()[smooth].max() < 40 * step ** 2 / 6 + 2.0 ** -52 * 10 / step + 2.0 ** -22


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K", [3, 64, 200, 5000, 40000])
def test_clip_border_is_decided_in_float64(mtlib, dtype, K):
    """Rows whose log ratio lies 1e-9 to 1e-6 to either side of an end of the
    clip range (for float32 rows: where old_logp's own steps put it) get the
    gradient of their side."""
    import torch
    n = 64
    f64 = dtype == "float64"
    x, z, a_t, a = _inputs(K, n, K, dtype)
    logp, stats, p, left, part = fu.softmax_rows(z, a)
    rng = np.random.default_rng(3)
    adv = np.where(np.arange(n) % 2 == 0, 1.0, -1.0)
    end = np.where(adv > 0, math.log1p(0.3), math.log1p(-0.2))
    off = rng.choice([-1, 1], size=n) * 10.0 ** rng.uniform(-9, -6, size=n)
    old = (logp - end - off).astype(np.float64 if f64 else np.float32)
    d = logp - old.astype(np.float64)
    clear = np.abs(d - end) > 1e-12  # float64's own accuracy of a log probability
    t = [torch.from_numpy(v.astype(old.dtype)).cuda() for v in (adv, old)]
    _, _, grad, _ = mtlib.policy_loss(x, a_t, t[0], t[1], clip_low=0.2, clip_high=0.3)
    active = np.where(adv > 0, d <= end, d >= end)
    moved = (grad != 0).any(1).cpu().numpy()
    np.testing.assert_array_equal(moved[clear], active[clear])


@gpu
def test_special_values(mtlib):
    """An action of n_classes or more, NaN and +inf scores make their own row
    NaN; neighbours keep their values."""
    import torch
    for K in (5, 200, 3000):
        x, z, a_t, a = _inputs(K, 6, K, "float32")
        x[1, 2], x[3, 0] = math.nan, math.inf
        a_t[4] = K + 7
        x[5] = math.nan
        logp, stats = mtlib.action_logprobs(x, a_t)
        one = torch.ones(6, device="cuda")
        loss, l2, G, H = mtlib.policy_loss(x, a_t, one, logp.nan_to_num(-1.0), ref_logp=logp.nan_to_num(-1.0), kl_coef=0.1, hess=True)
        G2, H2 = mtlib.action_logprobs_grad(x, a_t, stats, one, one)
        bad = torch.tensor([False, True, False, True, True, True])
        for v in (logp, l2, loss):
            assert torch.equal(v.isnan().cpu(), bad)
        for v in (G, H, G2, H2):
            assert torch.equal(v.isnan().any(1).cpu(), bad)
            assert not v[~bad.cuda()].isnan().any()


@gpu
def test_extreme_scores(mtlib):
    """Scores of +-1e4 and float16's largest: the maximum is taken out first."""
    import torch
    for K in (4, 300, 2000):
        x, z, a_t, a = _inputs(K, 8, K, "float32")
        x += 1e4
        x[0] = -1e4
        z = x.double().cpu().numpy()
        want = fu.softmax_rows(z, a)
        e_l = _row_bounds(z, want[2], want[1], want[0], False)[0]
        _close(mtlib.action_logprobs(x, a_t)[0], want[0], e_l, "logp")
        y = torch.full((2, K), 65504.0, dtype=torch.float16, device="cuda")
        got = mtlib.action_logprobs(y, a_t[:2])[0]
        assert (got.double() + math.log(K)).abs().max() < 1e-5


@gpu
def test_rows_do_not_depend_on_their_neighbours(mtlib):
    """A row's outputs are the same bits at any place of a batch and in any
    buffer whose rows are aligned alike."""
    import torch
    for K, dtype in ((7, "float32"), (10, "float64"), (64, "bfloat16"), (136, "bfloat16"), (4096, "float16")):
        x, z, a_t, a = _inputs(K, 50, K, dtype)
        t = torch.float64 if dtype == "float64" else torch.float32
        adv, old = torch.randn(50, device="cuda", dtype=t), torch.full((50,), -1.0, device="cuda", dtype=t)
        all_ = mtlib.policy_loss(x, a_t, adv, old, hess=True)
        for r0, r1 in ((0, 1), (17, 18), (13, 29)):
            some = mtlib.policy_loss(x[r0:r1].clone(), a_t[r0:r1], adv[r0:r1], old[r0:r1], hess=True)
            for u, v in zip(all_, some):
                assert torch.equal(u[r0:r1], v)


@gpu
def test_streams_graphs_and_unaligned_buffers(mtlib):
    import torch
    n, K = 33, 1001
    buf = torch.randn(n * K + 8, device="cuda").to(torch.bfloat16)
    a = torch.randint(0, K, (n,), device="cuda")
    adv, old = torch.randn(n, device="cuda"), torch.full((n,), -6.0, device="cuda")
    for off in range(1, 8):  # rows that start off 16-byte boundaries
        x = buf[off:off + n * K].view(n, K)
        want = mtlib.policy_loss(x.clone().float(), a, adv, old)
        got = mtlib.policy_loss(x, a, adv, old)
        assert torch.allclose(got[0], want[0], rtol=1e-5, atol=1e-6)
        assert (got[2].float() - want[2]).abs().max() <= want[2].abs().max() * 2.0 ** -7
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = mtlib.policy_loss(x, a, adv, old)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for u, v in zip(got[:3], on_side[:3]):
        assert torch.equal(u, v)
    plan = mtlib.PreferencePlan([0, 2, 4], [1, 3, 0], 7)
    s = torch.randn(7, device="cuda")
    mtlib.preference_loss(plan, s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        logp, stats = mtlib.action_logprobs(x, a)
        back = mtlib.action_logprobs_grad(x, a, stats, adv)
        pol = mtlib.policy_loss(x, a, adv, old)
        pref = mtlib.preference_loss(plan, s)
    for seed in (1, 2):
        x.copy_(torch.randn(n, K, device="cuda").to(torch.bfloat16))
        s.copy_(torch.randn(7, device="cuda"))
        g.replay()
        torch.cuda.synchronize()
        now = (*mtlib.action_logprobs(x, a), mtlib.action_logprobs_grad(x, a, stats, adv)[0],
               *mtlib.policy_loss(x, a, adv, old)[:3], *mtlib.preference_loss(plan, s))
        for u, v in zip((logp, stats, back[0], *pol[:3], *pref), now):
            assert torch.equal(u, v)


@gpu
def test_mixed_and_host_arrays_are_refused(mtlib):
    import torch
    x, a = torch.randn(4, 3, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    one = torch.ones(4, device="cuda")
    logp, stats = mtlib.action_logprobs(x, a)
    bad = [lambda: mtlib.action_logprobs(x, a.cpu()), lambda: mtlib.action_logprobs(x, a[:3]),
           lambda: mtlib.action_logprobs(x, a.long()[::1].to(torch.int16)), lambda: mtlib.action_logprobs(x.t(), a[:3]),
           lambda: mtlib.action_logprobs(x[0], a), lambda: mtlib.action_logprobs(x[:1].expand(4, 3), a),
           lambda: mtlib.policy_loss(x, a, one.double(), one), lambda: mtlib.policy_loss(x, a, one, one[:2]),
           lambda: mtlib.policy_loss(x, a, one, one, kl_coef=0.1), lambda: mtlib.policy_loss(x, a, one, one, grad=False, hess=True),
           lambda: mtlib.action_logprobs_grad(x, a, stats[:, :1], one), lambda: mtlib.action_logprobs_grad(x, a, stats, one.double()),
           lambda: mtlib.policy_loss(x, a, torch.ones(8, device="cuda")[::2], one)]
    for f in bad:
        with pytest.raises(mtlib.MojoTreesError) as e:
            f()
        assert e.value.code == -1
    plan = mtlib.PreferencePlan([0], [1], 4)
    for f in (lambda: mtlib.preference_loss(plan, one[:3]), lambda: mtlib.preference_loss(plan, one.half()),
              lambda: mtlib.preference_loss(plan, one, beta=0.0), lambda: mtlib.preference_loss(plan, one, label_smoothing=0.6),
              lambda: mtlib.preference_loss(plan, one, label_smoothing=-0.1), lambda: mtlib.preference_loss(plan, one, loss="x"),
              lambda: mtlib.preference_loss(plan, one, reference=one.double()), lambda: mtlib.preference_loss(plan, one.cpu())):
        with pytest.raises(mtlib.MojoTreesError) as e:
            f()
        assert e.value.code == -1
    lib = mtlib.lib()  # a host address reaches no kernel
    e = lib.mojotrees_error_create()
    assert lib.mojotrees_b200_action_logprobs(P, 1, 4, 3, 3, a.data_ptr(), 4, logp.data_ptr(), stats.data_ptr(), None, e) == -1
    assert b"device memory" in lib.mojotrees_error_message(e)
    lib.mojotrees_error_free(e)


# ------------------------------------------------------------- paired losses

def _pairs(seed, n, P_, how):
    rng = np.random.default_rng(seed)
    if how == "apart":
        at = rng.permutation(n)
        return at[:P_], at[P_:2 * P_]
    if how == "star":  # one item in every pair
        j = 1 + rng.integers(0, n - 1, size=P_)
        turn = rng.random(P_) < 0.5
        return np.where(turn, 0, j), np.where(turn, j, 0)
    i = (n * rng.random(P_) ** 3).astype(np.int64)
    j = rng.integers(0, n - 1, size=P_)
    return i, j + (j >= i)


@gpu
@pytest.mark.parametrize("dtype", ["float64", "float32"])
@pytest.mark.parametrize("n,P_,how", [(2, 1, "apart"), (7, 3, "apart"), (1001, 500, "apart"), (3, 0, "any"), (2, 5000, "any"),
                                      (70, 3, "any"), (100, 5000, "any"), (300, 40_000, "star"), (5000, 20_001, "any"),
                                      (40, 100_000, "any"), (20_000, 300_000, "star"), (0, 0, "apart")])
def test_preference_loss(mtlib, n, P_, how, dtype):
    import torch
    i, j = _pairs(n + P_, n, P_, how) if P_ else (np.zeros(0, np.int64), np.zeros(0, np.int64))
    rng = np.random.default_rng(P_)
    for loss, beta, eps, with_ref, with_w in (("logistic", 0.5, 0.0, True, False), ("logistic", 2.0, 0.1, False, True),
                                              ("squared", 0.1, 0.0, True, True), ("squared", 0.3, 0.1, False, False)):
        w = rng.random(P_).astype(np.float32) if with_w else None
        if with_w:
            w[rng.random(P_) < 0.2] = 0
        s = torch.from_numpy(rng.normal(size=n) * 3 - 40).to(getattr(torch, dtype)).cuda()
        ref = torch.from_numpy(rng.normal(size=n) - 40).to(s.dtype).cuda() if with_ref else None
        plan = mtlib.PreferencePlan(i, j, n, weights=w)
        got = mtlib.preference_loss(plan, s, reference=ref, beta=beta, label_smoothing=eps, loss=loss)
        assert got[0].dtype == s.dtype and got[0].shape == (P_,) and got[1].shape == (n,)
        sd = s.double().cpu().numpy()
        rd = None if ref is None else ref.double().cpu().numpy()
        L, g, h = fu.pairs_loss(sd, rd, i, j, w, beta, eps, loss)
        unit = 2.0 ** -53 if dtype == "float64" else fu.U32
        # Each term in the scores' arithmetic, with half a step `unit`.  The pair's difference u: a rounding of each
        # item's distance to its reference (up to 60 here) and of their difference in float64; in float32 that
        # distance keeps its rounding error, which leaves one rounding of u itself.  Then x = beta u, exp within 2 + |x|
        # steps, 1 + e, its inverse, three products; the loss a log1p within 2 steps and a sum.
        u = np.abs(sd - (0 if rd is None else rd))
        u = (u[i] + u[j]) if P_ else np.zeros(0)
        x = beta * u
        # The plain form rounds alike in float64: beside a float64 kernel its error counts too.
        sides = 2 if dtype == "float64" else 1
        du = sides * (u + (1 / (2 * beta) if loss == "squared" else 0)) * 2 * unit  # absolute
        term = sides * 2 * (14 + 4 * x) * unit  # relative, a full step being 2 unit
        _close(got[0], L, np.abs(L) * (term + 2 * unit) + (np.abs(g) + h * du) * du + 2.0 ** -126, "loss")
        G, H, E, A, B = (np.zeros(n) for _ in range(5))
        np.add.at(G, i, g)
        np.add.at(G, j, -g)
        for v, at in ((h, H), (np.abs(g), A), (np.abs(g) * term + h * du * 1.1, E), (h * (term + 2 * beta * du), B)):
            np.add.at(at, i, v)
            np.add.at(at, j, v)
        degree = np.bincount(np.concatenate([i, j]), minlength=n)[:n]
        lane = 2 * degree * 2.0 ** -53  # sums in float64, in any order, both here and there
        _close(got[1], G, np.abs(G) * fu.U32 * 1.01 + E + A * lane + 2.0 ** -126, "grad")
        _close(got[2], H, H * (fu.U32 * 1.01 + lane) + B + 2.0 ** -126, "hess")
        again = mtlib.preference_loss(plan, s, reference=ref, beta=beta, label_smoothing=eps, loss=loss)
        for u, v in zip(got, again):
            assert torch.equal(u, v)


@gpu
def test_preference_special_values(mtlib):
    """NaN of an item reaches its own pairs alone, and none through pairs of
    weight 0; an infinite difference saturates."""
    import torch
    i, j = np.array([0, 2, 4, 6, 8]), np.array([1, 3, 5, 7, 0])
    s = torch.tensor([0.0, 1.0, math.nan, 0.0, math.inf, 0.0, -math.inf, 0.0, 1.0, math.nan], dtype=torch.float64, device="cuda")
    loss, grad, hess = mtlib.preference_loss(mtlib.PreferencePlan(i, j, 10), s)
    assert torch.equal(loss.isnan().cpu(), torch.tensor([False, True, False, False, False]))
    assert loss[2] == 0 and loss[3] == math.inf
    assert torch.equal(grad.isnan().cpu(), torch.tensor([False] * 2 + [True] * 2 + [False] * 6))
    assert grad[4] == 0 and grad[5] == 0 and grad[6] == -1 and grad[7] == 1 and grad[9] == 0 and hess[9] == 0
    plan = mtlib.PreferencePlan(i, j, 10, weights=[1, 0, 1, 1, 1])
    loss, grad, hess = mtlib.preference_loss(plan, s)
    assert loss[1] == 0 and not grad.isnan().any() and not hess.isnan().any()


@gpu
def test_two_plans_and_two_streams_at_once(mtlib):
    """One plan used by overlapping calls on two streams gives what it gives alone."""
    import torch
    i, j = _pairs(1, 5000, 200_000, "any")
    plan = mtlib.PreferencePlan(i, j, 5000)
    s = [torch.randn(5000, device="cuda", dtype=torch.float64) for _ in range(2)]
    alone = [mtlib.preference_loss(plan, v) for v in s]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(10):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                got[k].append(mtlib.preference_loss(plan, s[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for out in got[k]:
            for u, v in zip(out, alone[k]):
                assert torch.equal(u, v)


@gpu
def test_preference_through_class_scores(mtlib):
    """Preference over answers of one decision each, as a model of K classes
    is trained: log probabilities, the paired loss of their difference to a
    reference's, and back to the scores; against differentiating the whole in
    float64."""
    import torch
    n, K = 600, 9
    x, z, a_t, a = _inputs(8, n, K, "float64")
    ref, _ = mtlib.action_logprobs(torch.randn(n, K, dtype=torch.float64, device="cuda"), a_t)
    i, j = _pairs(2, n, 3000, "any")
    logp, stats = mtlib.action_logprobs(x, a_t)
    loss, g, h = mtlib.preference_loss(mtlib.PreferencePlan(i, j, n), logp, reference=ref, beta=0.7)
    G, H = mtlib.action_logprobs_grad(x, a_t, stats, g, h)
    y = x.clone().requires_grad_(True)
    l = torch.log_softmax(y, 1).gather(1, a_t.long()[:, None])[:, 0] - ref
    ti, tj = torch.from_numpy(i).cuda(), torch.from_numpy(j).cuda()
    want = -torch.nn.functional.logsigmoid(0.7 * (l[ti] - l[tj]))
    want.sum().backward()
    assert (loss - want).abs().max() < 1e-13
    # g and G are rounded to float32 one after the other
    size = g.abs().double()[:, None].expand(n, K)
    assert ((G.double() - y.grad).abs() <= 2.1 * fu.U32 * size + 1e-12).all()
    assert (H >= 0).all()


# --------------------------------------------- calls that the ones above leave out

@gpu
@pytest.mark.parametrize("dtype,n,K,out_stride", [
    ("float64", 70, 10, 13), ("float64", 33, 200, 203), ("float32", 65, 7, 8), ("float32", 9, 300, 304), ("float32", 5, 5000, 5001),
    ("bfloat16", 40, 50, 57), ("bfloat16", 9, 1000, 1003), ("float16", 7, 4096, 4104), ("float16", 3, 20001, 20011)])
def test_strided_derivatives_leave_the_rest_alone(mtlib, dtype, n, K, out_stride):
    """Derivatives written at a row stride of their own: the same values, and
    what lies between the rows and behind the last keeps its bits."""
    import torch
    x, z, a_t, a = _inputs(K, n, K, dtype, mask=True)
    row = torch.float64 if dtype == "float64" else torch.float32
    adv = torch.randn(n, device="cuda", dtype=row)
    old = torch.full((n,), -2.0, device="cuda", dtype=row)
    loss, logp, want_g, want_h = mtlib.policy_loss(x, a_t, adv, old, hess=True)
    got = [torch.full((n + 2, out_stride), 7.0, dtype=want_g.dtype, device="cuda") for _ in range(2)]
    out_loss = torch.full((n + 5,), 7.0, dtype=row, device="cuda")
    lib = mtlib.lib()
    e = lib.mojotrees_error_create()
    kind = DTYPES.index(dtype)
    rc = lib.mojotrees_b200_policy_loss(x.data_ptr(), kind, n, K, x.stride(0), a_t.data_ptr(), 4, adv.data_ptr(), old.data_ptr(),
                                        None, None, 0.2, 0.2, 0.0, out_loss.data_ptr(), None, got[0].data_ptr(), got[1].data_ptr(),
                                        out_stride, torch.cuda.current_stream().cuda_stream, e)
    assert rc == 0, lib.mojotrees_error_message(e)
    lib.mojotrees_error_free(e)
    assert torch.equal(out_loss[:n], loss) and (out_loss[n:] == 7).all()
    for u, want in zip(got, (want_g, want_h)):
        assert torch.equal(u[:n, :K], want)
        assert (u[:n, K:] == 7).all() and (u[n:] == 7).all()


@gpu
def test_first_call_inside_a_capture():
    """A process whose first calls are captured into a graph, items of many
    pairs among them; the graph is replayed twice without a wait between."""
    import os
    import subprocess
    import sys
    code = """
import numpy as np, torch
import mojoboost_b200 as mb
rng = np.random.default_rng(0)
n = 3000
i = np.concatenate([np.zeros(40000, int), np.ones(3000, int), rng.integers(2, n, 20000)])
j = 2 + rng.integers(0, n - 3, i.size); j += j == i
plan = mb.PreferencePlan(i, j, n)
s = torch.randn(n, dtype=torch.float64, device="cuda")
x = torch.randn(300, 1000, device="cuda").half(); a = torch.randint(0, 1000, (300,), device="cuda")
y = torch.randn(300, 9, dtype=torch.float64, device="cuda"); b = torch.randint(0, 9, (300,), device="cuda", dtype=torch.int32)
adv = torch.randn(300, device="cuda"); old = torch.full((300,), -7.0, device="cuda")
torch.cuda.synchronize()
def run():
    l, st = mb.action_logprobs(y, b)
    return [l, *mb.policy_loss(x, a, adv, old)[:3], *mb.preference_loss(plan, s), mb.action_logprobs_grad(y, b, st, adv, adv.abs())[0]]
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = run()
for seed in range(3):
    s.normal_(); y.normal_(); x.normal_()
    g.replay(); g.replay()
    torch.cuda.synchronize()
    for u, v in zip(out, run()):
        assert torch.equal(u, v)
print("captured")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stdout + r.stderr


@gpu
@pytest.mark.parametrize("n,K,dtype", [(66_000, 32_769, "bfloat16"), (270_000_000, 8, "float16")])
def test_offsets_beyond_32_bits(mtlib, n, K, dtype):
    """Scores of more than 2^31 elements: the last rows as in a call of their own."""
    import torch
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    x = torch.zeros((n, K), dtype=getattr(torch, dtype), device="cuda")
    x[-40:] = torch.randn((40, K), device="cuda").to(x.dtype)
    a = torch.zeros(n, dtype=torch.int32, device="cuda")
    a[-40:] = torch.randint(0, K, (40,), device="cuda", dtype=torch.int32)
    adv, old = torch.ones(n, device="cuda"), torch.full((n,), -math.log(K), device="cuda")
    loss, logp, grad, _ = mtlib.policy_loss(x, a, adv, old)
    l2, stats = mtlib.action_logprobs(x, a)
    back, _ = mtlib.action_logprobs_grad(x, a, stats, adv)
    t = slice(n - 40, n)
    z, at = x[t].double().cpu().numpy(), a[t].cpu().numpy()
    rows = [v[t].cpu().numpy() for v in (adv, old)]
    _check_policy((loss[t], logp[t], grad[t], None), z, at, *rows, None, None, 0.2, 0.2, 0.0, dtype)
    want_l, want_s, p, left, part = fu.softmax_rows(z, at)
    e_l, e_p, e_left = _row_bounds(z, p, want_s, want_l, False)
    _close(l2[t], want_l, e_l, "logp")
    G, _, q = fu.to_scores(p, left, at, part, rows[0].astype(np.float64), np.zeros(40))
    tol_q = np.where(q > 0, np.maximum(e_left[:, None], e_p), e_p)
    _close(back[t], G, np.abs(G) * (tol_q + HALF_STEP[dtype]) * 1.01 + TINY[dtype], "grad")
    assert (logp[:-40] + math.log(K)).abs().max() < 1e-5
    del grad, back
    torch.cuda.empty_cache()


@gpu
@pytest.mark.parametrize("n,P_", [(1500, 200_000), (40_000, 30_000)])
def test_preference_loss_alone_and_derivatives_alone(mtlib, n, P_):
    """The C entry's optional outputs: the loss without derivatives, and the
    derivatives without the loss (as a fit takes them)."""
    import torch
    i, j = _pairs(n, n, P_, "any")
    i[: P_ // 4], j[: P_ // 4] = 0, 1 + np.arange(P_ // 4) % (n - 1)  # an item of many pairs
    w = np.random.default_rng(1).random(P_).astype(np.float32)
    w[::7] = 0
    plan = mtlib.PreferencePlan(i, j, n, weights=w)
    s = torch.randn(n, dtype=torch.float64, device="cuda")
    want = mtlib.preference_loss(plan, s)
    loss = torch.full_like(want[0], 7)
    g, h = torch.full_like(want[1], 7), torch.full_like(want[2], 7)
    lib = mtlib.lib()
    e = lib.mojotrees_error_create()
    st = torch.cuda.current_stream().cuda_stream
    assert lib.mojotrees_b200_preference_loss(plan.h, s.data_ptr(), None, 0, 1.0, 0.0, 0, loss.data_ptr(), None, None, st, e) == 0
    assert lib.mojotrees_b200_preference_loss(plan.h, s.data_ptr(), None, 0, 1.0, 0.0, 0, None, g.data_ptr(), h.data_ptr(), st, e) == 0
    assert lib.mojotrees_b200_preference_loss(plan.h, s.data_ptr(), None, 0, 1.0, 0.0, 0, None, None, h.data_ptr(), st, e) == -1
    lib.mojotrees_error_free(e)
    assert torch.equal(loss, want[0]) and torch.equal(g, want[1]) and torch.equal(h, want[2])
