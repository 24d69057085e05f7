"""Fits of objective=policy and objective=preference: the trees' leaf values
against the losses' derivatives in float64, the multiclass objective as a
special case, refusals, model files.
"""
import ctypes
import math

import numpy as np
import pytest

import feedback_util as fu

gpu = pytest.mark.gpu

# ------------------------------------------------------------------ refusals

X4 = np.arange(8.0).reshape(4, 2)


def _policy(mtlib, **kw):
    a = dict(X=X4, actions=[0, 1, 2, 0], advantages=[1.0, -1.0, 0.5, 0.0], params={"num_class": 3})
    a.update(kw)
    return mtlib.train_dense_policy(a.pop("X"), a.pop("actions"), a.pop("advantages"), a.pop("params"), **a)


@pytest.mark.parametrize("kw,code,needle", [
    (dict(actions=[0, 1, 2, 3]), -1, "num_class-1"), (dict(actions=[0, 1, 2, -2]), -1, "num_class-1"),
    (dict(actions=[0, 1, 2]), -1, "shape"), (dict(actions=[0.0, 1.0, 2.0, 0.0]), -1, "integers"),
    (dict(actions=[0, 1, 2, 2 ** 40]), -1, "32 bits"), (dict(actions=None), -1, "null"), (dict(advantages=None), -1, "null"),
    (dict(advantages=[1.0, math.nan, 0, 0]), -1, "advantages"), (dict(advantages=[1.0, 2.0]), -1, "shape"),
    (dict(old_logp=[0, 0, 0, -math.inf]), -1, "old_logp"), (dict(ref_logp=[0, 0, 0, math.nan]), -1, "ref_logp"),
    (dict(weights=[1, 1, 1, -1]), -1, "weights"), (dict(weights=[1, 1, 1, math.inf]), -1, "weights"),
    (dict(initial_scores=np.zeros((4, 2))), -1, "initial_scores"), (dict(initial_scores=np.zeros(4)), -1, "initial_scores"),
    (dict(initial_scores=np.full((4, 3), math.inf)), -1, "initial_scores"),
    (dict(params={}), -1, "num_class"), (dict(params={"num_class": 1}), -1, "num_class"),
    (dict(params={"num_class": 3, "objective": "binary"}), -1, "objective=policy"),
    (dict(params={"num_class": 3, "objective": "preference"}), -1, "objective=policy"),
    (dict(params={"num_class": 3, "policy_clip_low": 1.5}), -1, "policy_clip_low"),
    (dict(params={"num_class": 3, "policy_clip_low": "nan"}), -1, "policy_clip_low"),
    (dict(params={"num_class": 3, "policy_clip_high": -1}), -1, "policy_clip_high"),
    (dict(params={"num_class": 3, "policy_kl": "inf"}), -1, "policy_kl"),
    (dict(X=np.zeros(4)), -1, "n_features"),
])
def test_policy_fit_refusals(mtlib, kw, code, needle):
    with pytest.raises(mtlib.MojoTreesError, match=needle) as e:
        _policy(mtlib, **kw)
    assert e.value.code == code


def _preference(mtlib, **kw):
    a = dict(X=X4, winners=[0, 1], losers=[2, 3], params=None)
    a.update(kw)
    return mtlib.train_dense_preference(a.pop("X"), a.pop("winners"), a.pop("losers"), a.pop("params"), **a)


@pytest.mark.parametrize("kw,code,needle", [
    (dict(winners=[0, 4]), -1, "out of range"), (dict(losers=[2, -1]), -1, "out of range"), (dict(losers=[2, 1]), -1, "itself"),
    (dict(winners=[0]), -1, "one length"), (dict(winners=[], losers=[]), -1, "n_pairs"), (dict(winners=[0.5, 1.0]), -1, "integers"),
    (dict(pair_weights=[1.0, -1.0]), -1, "weights"), (dict(pair_weights=[1.0]), -1, "one length"),
    (dict(actions=[0, 1, 1, 0]), -1, "num_class"), (dict(params={"num_class": 2}), -1, "actions"),
    (dict(params={"num_class": 2}, actions=[0, 1, 1, -1]), -1, "actions"), (dict(params={"num_class": 2}, actions=[0, 1, 1, 2]), -1, "actions"),
    (dict(reference=[0, 0, 0, math.nan]), -1, "reference"), (dict(reference=[0.0]), -1, "shape"),
    (dict(initial_scores=np.zeros((4, 2))), -1, "initial_scores"), (dict(initial_scores=np.zeros(3)), -1, "initial_scores"),
    (dict(params={"preference_beta": 0}), -1, "preference_beta"), (dict(params={"preference_label_smoothing": 0.7}), -1, "smoothing"),
    (dict(params={"preference_loss": "hinge"}), -1, "preference_loss"),
    (dict(params={"preference_loss": "squared", "preference_label_smoothing": -0.1}), -1, "smoothing"),
    (dict(params={"objective": "regression"}), -1, "objective=preference"),
])
def test_preference_fit_refusals(mtlib, kw, code, needle):
    with pytest.raises(mtlib.MojoTreesError, match=needle) as e:
        _preference(mtlib, **kw)
    assert e.value.code == code


@pytest.mark.parametrize("objective", ["policy", "preference"])
def test_label_fits_refuse_feedback_objectives(mtlib, objective):
    for fit in (lambda p: mtlib.train_dense(X4, np.zeros(4), p),
                lambda p: mtlib.train_binned(np.zeros((2, 4), np.uint8), 4, np.zeros(4), p)):
        with pytest.raises(mtlib.UnsupportedError, match="feedback"):
            fit({"objective": objective, "num_class": 3})


def test_binned_fits_check_their_bins(mtlib):
    for bins, n_bins, kw in ((np.zeros((2, 4), np.uint8), 1, {}), (np.zeros((2, 4), np.uint8), 257, {}),
                             (np.zeros((2, 4), np.uint8), 4, dict(missing_bin=[4, -1])), (np.zeros(4, np.uint8), 4, {}),
                             (np.zeros((2, 4), np.uint8), 4, dict(n_categories=[1]))):
        with pytest.raises(mtlib.MojoTreesError) as e:
            mtlib.train_binned_preference(bins, n_bins, [0], [1], **kw)
        assert e.value.code == -1
        with pytest.raises(mtlib.MojoTreesError) as e:
            mtlib.train_binned_policy(bins, n_bins, [0, 1, 1, 0], np.zeros(4), {"num_class": 2}, **kw)
        assert e.value.code == -1


def test_fits_need_a_device(mtlib):
    if mtlib.gpu_available():
        pytest.skip("a GPU is present")
    for fit in (_policy, _preference):
        with pytest.raises(mtlib.UnsupportedError, match="CUDA"):
            fit(mtlib)


def test_null_pointers(mtlib):
    lib = mtlib.lib()
    e = lib.mojotrees_error_create()
    h = ctypes.c_void_p()
    P = np.zeros(16).ctypes.data
    I = np.zeros(4, np.int64).ctypes.data
    try:
        assert lib.mojotrees_b200_train_dense_policy(None, 4, 2, I, P, None, None, None, None, b"num_class=2", ctypes.byref(h), e) == -1
        assert lib.mojotrees_b200_train_dense_policy(P, 4, 2, I, P, None, None, None, None, b"num_class=2", None, e) == -1
        assert lib.mojotrees_b200_train_dense_policy(P, 0, 2, I, P, None, None, None, None, b"num_class=2", ctypes.byref(h), e) == -1
        assert lib.mojotrees_b200_train_dense_preference(P, 4, 2, None, I, None, 1, None, None, None, None, ctypes.byref(h), e) == -1
        assert lib.mojotrees_b200_train_binned_u8_preference(None, 4, 2, 4, None, None, I, I, None, 1, None, None, None, None, ctypes.byref(h), e) == -1
    finally:
        lib.mojotrees_error_free(e)


# ------------------------------------------------------------------- fits

N_BINS = 32


def _bins(seed, n, F):
    return np.random.default_rng(seed).integers(0, N_BINS, size=(F, n)).astype(np.uint8)


def _leaves(tree, bins):
    """The leaf node of every row (numeric features, no missing values)."""
    node = np.zeros(bins.shape[1], np.int64)
    while True:
        f = tree["feature"][node]
        inner = f >= 0
        if not inner.any():
            return node
        b = bins[np.maximum(f, 0), np.arange(len(node))]
        to = np.where(b <= tree["threshold_bin"][node], tree["left"][node], tree["right"][node])
        node = np.where(inner, to, node)


def _check_tree(tree, bins, G, H, lam, floor=1e-16):
    """Every leaf's value is -sum G / (sum H + lambda).  G and H are narrowed
    to float32 (half a step each; their float64 forms agree to 1e-12), and the
    int64 histogram mode rounds each row's to units of at most 2^-51 of the
    absolute total: half a unit a row."""
    at = _leaves(tree, bins)
    H = np.maximum(H, floor)
    assert (tree["feature"][0] >= 0) and tree["count"][0] == len(G)
    for leaf in np.unique(at):
        rows = at == leaf
        g, h = G[rows].sum(), H[rows].sum() + lam
        eg = np.abs(G[rows]).sum() * 1.01 * fu.U32 + np.abs(G).sum() * 2.0 ** -52 * rows.sum() + 2.0 ** -149 * rows.sum()
        eh = H[rows].sum() * 1.01 * fu.U32 + H.sum() * 2.0 ** -52 * rows.sum()
        tol = eg / h + np.abs(g) / h * eh / h
        assert abs(tree["value"][leaf] + g / h) <= 1.05 * tol + 1e-15, (leaf, tree["value"][leaf], -g / h, tol)
        assert tree["count"][leaf] == rows.sum()


FIT = {"num_leaves": 15, "learning_rate": 0.3, "lambda_l2": 0.7, "min_data_in_leaf": 5, "min_sum_hessian_in_leaf": 1e-6,
       "gpu_histogram_precision": "int64", "keep_training_scores": True}


def _policy_case(seed, n, K, with_old, with_ref, with_w, with_init):
    rng = np.random.default_rng(seed)
    init = rng.normal(size=(n, K)) if with_init else None
    actions = rng.integers(0, K, size=n).astype(np.int32)
    actions[rng.random(n) < 0.05] = -1
    lp0 = fu.softmax_rows(np.zeros((n, K)) if init is None else init, actions)[0]
    return dict(initial_scores=init, actions=actions, advantages=rng.normal(size=n),
                old_logp=np.minimum(lp0 + 0.2 * rng.normal(size=n), 0) if with_old else None,
                ref_logp=np.minimum(lp0 + 0.3 * rng.normal(size=n), 0) if with_ref else None,
                weights=rng.random(n) * (rng.random(n) > 0.1) if with_w else None)


@gpu
@pytest.mark.parametrize("K,with_old,with_ref,with_w,with_init", [
    (2, True, True, True, True), (3, False, False, False, False), (10, True, False, True, True), (64, True, True, False, False)])
def test_policy_trees(mtlib, K, with_old, with_ref, with_w, with_init):
    n, F, low, high, kl = 3000, 6, 0.15, 0.25, 0.3
    bins = _bins(K, n, F)
    case = _policy_case(K, n, K, with_old, with_ref, with_w, with_init)
    params = dict(FIT, num_class=K, policy_clip_low=low, policy_clip_high=high, policy_kl=kl)
    raw = np.zeros((n, K)) if case["initial_scores"] is None else case["initial_scores"].copy()
    lp0 = fu.softmax_rows(raw, case["actions"])[0]
    old = lp0 if case["old_logp"] is None else case["old_logp"]
    ref = lp0 if case["ref_logp"] is None else case["ref_logp"]
    rounds = 3
    model = mtlib.train_binned_policy(bins, N_BINS, case["actions"], case["advantages"], dict(params, num_iterations=rounds),
                                      **{k: case[k] for k in ("old_logp", "ref_logp", "weights", "initial_scores")})
    assert model.num_classes == K and model.num_iterations == rounds and np.all(model.base_scores() == 0)
    for it in range(rounds):
        logp, stats, p, left, part = fu.softmax_rows(raw, case["actions"], case["weights"])
        if it == 0:
            assert with_old or np.allclose(logp[part], old[part])
        loss, g, h, part = fu.policy_rows(logp, part, case["advantages"], old, ref, case["weights"], low, high, kl)
        # rows on the border within float64's accuracy could lie on either side
        d = np.where(part, logp, 0) - old
        assert min(np.abs(d - math.log1p(high)).min(), np.abs(d - math.log1p(-low)).min()) > 1e-12
        G, H, _ = fu.to_scores(p, left, case["actions"], part, g, h)
        for k in range(K):
            tree = model.tree(it * K + k)
            _check_tree(tree, bins, G[:, k], H[:, k], FIT["lambda_l2"])
            raw[:, k] += FIT["learning_rate"] * tree["value"][_leaves(tree, bins)]
    np.testing.assert_allclose(model.training_scores(n).reshape(n, K), raw, rtol=1e-12, atol=1e-12)
    # predictions are what the fit added
    np.testing.assert_allclose(model.predict_binned(bins), raw - (0 if case["initial_scores"] is None else case["initial_scores"]),
                               rtol=1e-11, atol=1e-11)


@gpu
def test_policy_of_one_round_is_the_multiclass_step(mtlib):
    """With advantage 1 and the ratio at 1 the gradient is softmax's and the
    hessian p (1 - p): the multiclass objective's without its factor K / (K -
    1), so lambda and the least hessian scaled by (K - 1) / K give the same
    trees with values K / (K - 1) as large."""
    n, F, K = 4000, 5, 4
    bins = _bins(1, n, F)
    y = (bins[0].astype(int) + bins[1] + np.random.default_rng(0).integers(0, 12, size=n)) % K
    common = dict(FIT, num_class=K, num_iterations=1, num_leaves=7)
    multi = mtlib.train_binned(bins, N_BINS, y, dict(common, objective="multiclass"))
    init = np.tile(multi.base_scores(), (n, 1))
    scale = (K - 1) / K
    policy = mtlib.train_binned_policy(bins, N_BINS, y, np.ones(n),
                                       dict(common, lambda_l2=FIT["lambda_l2"] * scale,
                                            min_sum_hessian_in_leaf=FIT["min_sum_hessian_in_leaf"] * scale),
                                       initial_scores=init)
    for k in range(K):
        a, b = multi.tree(k), policy.tree(k)
        for name in ("feature", "threshold_bin", "left", "right", "count"):
            np.testing.assert_array_equal(a[name], b[name])
        np.testing.assert_allclose(b["value"], a["value"] / scale, rtol=1e-5, atol=1e-9)


@gpu
@pytest.mark.parametrize("K", [1, 2, 5])
@pytest.mark.parametrize("loss,beta,eps", [("logistic", 0.8, 0.0), ("logistic", 1.5, 0.2), ("squared", 0.4, 0.0)])
def test_preference_trees(mtlib, K, loss, beta, eps):
    n, F, P = 2500, 6, 9000
    bins = _bins(K, n, F)
    rng = np.random.default_rng(K)
    i = rng.integers(0, n, size=P)
    j = (i + 1 + rng.integers(0, n - 1, size=P)) % n
    w = rng.random(P).astype(np.float32)
    w[rng.random(P) < 0.1] = 0
    actions = rng.integers(0, K, size=n).astype(np.int32) if K > 1 else None
    ref = rng.normal(size=n) * 0.5
    init = rng.normal(size=(n, K)) if K > 1 else rng.normal(size=n)
    params = dict(FIT, preference_beta=beta, preference_label_smoothing=eps, preference_loss=loss, num_iterations=2)
    if K > 1:
        params["num_class"] = K
    model = mtlib.train_binned_preference(bins, N_BINS, i, j, params, pair_weights=w, actions=actions, reference=ref,
                                          initial_scores=init)
    raw = init.copy().reshape(n, K)
    for it in range(2):
        if K > 1:
            s, stats, p, left, part = fu.softmax_rows(raw, actions)
        else:
            s = raw[:, 0]
        L, g, h = fu.pairs_loss(s, ref, i, j, w, beta, eps, loss)
        gi, hi = np.zeros(n), np.zeros(n)
        np.add.at(gi, i, g)
        np.add.at(gi, j, -g)
        np.add.at(hi, i, h)
        np.add.at(hi, j, h)
        if K > 1:  # narrowed between the two losses
            G, H, _ = fu.to_scores(p, left, actions, part, gi.astype(np.float32).astype(np.float64),
                                   hi.astype(np.float32).astype(np.float64))
        else:
            G, H = gi[:, None], hi[:, None]
        for k in range(K):
            tree = model.tree(it * K + k)
            _check_tree(tree, bins, G[:, k], H[:, k], FIT["lambda_l2"])
            raw[:, k] += FIT["learning_rate"] * tree["value"][_leaves(tree, bins)]
    np.testing.assert_allclose(model.training_scores(n).reshape(n, K), raw, rtol=1e-12, atol=1e-12)


@gpu
@pytest.mark.parametrize("quant", [False, True])
def test_dense_fits_and_model_files(mtlib, quant, tmp_path):
    """Dense fits bin as train_dense does, repeat bit for bit, and save, load
    and predict as regression and multiclass models."""
    rng = np.random.default_rng(2)
    n, K = 3000, 3
    X = rng.normal(size=(n, 5))
    X[rng.random((n, 5)) < 0.05] = np.nan
    params = {"num_iterations": 4, "num_leaves": 15, "min_data_in_leaf": 5, "use_quantized_grad": quant}
    actions, adv = rng.integers(0, K, size=n), rng.normal(size=n)
    i = rng.integers(0, n, size=5000)
    j = (i + 1 + rng.integers(0, n - 1, size=5000)) % n
    bins, mb, nc, nb = mtlib.bin_dense(X)
    for dense, binned in (
            (lambda: mtlib.train_dense_policy(X, actions, adv, dict(params, num_class=K, objective="policy")),
             lambda: mtlib.train_binned_policy(bins, nb, actions, adv, dict(params, num_class=K), missing_bin=mb, n_categories=nc)),
            (lambda: mtlib.train_dense_preference(X, i, j, params),
             lambda: mtlib.train_binned_preference(bins, nb, i, j, params, missing_bin=mb, n_categories=nc))):
        m, again, b = dense(), dense(), binned()
        out = m.predict(X, raw_score=True)
        assert out.std() > 0
        np.testing.assert_array_equal(out, again.predict(X, raw_score=True))
        np.testing.assert_array_equal(out, b.predict_binned(bins))
        np.testing.assert_array_equal(out, m.predict(X, raw_score=True, device="gpu"))
        path = str(tmp_path / "m.mbst")
        m.save(path)
        back = mtlib.Model.load(path)
        np.testing.assert_array_equal(back.predict(X), m.predict(X))
        if m.num_classes > 1:
            assert m.objective_name == "multiclass"
            np.testing.assert_allclose(m.predict(X).sum(1), 1, rtol=1e-12)
        else:
            assert m.objective_name == "regression"
            np.testing.assert_array_equal(m.predict(X), out)
        s = m.stats()
        assert s["kernel_launches"] > 0 and s["rounds"] == 4


@gpu
def test_behaviour_policy_then_policy_fit(mtlib):
    """The losses as they are used together: a multiclass model logs
    decisions, their log probabilities on the device are the fit's defaults,
    and the improved policy's loss is evaluated on the device."""
    import torch
    rng = np.random.default_rng(5)
    n, K = 2000, 4
    X = rng.normal(size=(n, 6))
    y = np.argmax(X[:, :K] + rng.gumbel(size=(n, K)), axis=1)
    behaviour = mtlib.train_dense(X, y, {"objective": "multiclass", "num_class": K, "num_iterations": 5, "num_leaves": 7})
    raw = behaviour.predict(X, raw_score=True)
    prob = behaviour.predict(X)
    actions = np.array([rng.choice(K, p=q / q.sum()) for q in prob])
    reward = (actions == np.argmax(X[:, :K], 1)).astype(float)
    adv = (reward - reward.mean()) / reward.std()
    t_raw, t_a = torch.from_numpy(raw).cuda(), torch.from_numpy(actions.astype(np.int32)).cuda()
    logp, _ = mtlib.action_logprobs(t_raw, t_a)
    np.testing.assert_allclose(logp.cpu().numpy(), np.log(prob[np.arange(n), actions]), rtol=1e-9)
    params = {"num_class": K, "num_iterations": 3, "num_leaves": 7, "policy_kl": 0.05, "keep_training_scores": True}
    given = mtlib.train_dense_policy(X, actions, adv, params, old_logp=logp.cpu().numpy(), ref_logp=logp.cpu().numpy(),
                                     initial_scores=raw)
    default = mtlib.train_dense_policy(X, actions, adv, params, initial_scores=raw)
    np.testing.assert_allclose(given.training_scores(n), default.training_scores(n), rtol=1e-6, atol=1e-6)
    new = torch.from_numpy(default.training_scores(n).reshape(n, K)).cuda()
    loss, l2, grad, _ = mtlib.policy_loss(new, t_a, torch.from_numpy(adv).cuda(), logp, ref_logp=logp, kl_coef=0.05)
    assert torch.isfinite(loss).all() and torch.isfinite(grad).all()
    np.testing.assert_allclose(default.predict(X, raw_score=True) + raw, new.cpu().numpy(), rtol=1e-9, atol=1e-9)


@gpu
@pytest.mark.parametrize("quant", [False, True])
def test_derivatives_beyond_float32_are_refused(mtlib, quant):
    bins = _bins(0, 500, 3)
    with pytest.raises(mtlib.MojoTreesError, match="not finite"):
        mtlib.train_binned_policy(bins, N_BINS, np.zeros(500, int), -np.ones(500),
                                  {"num_class": 2, "num_iterations": 1, "use_quantized_grad": quant}, old_logp=np.full(500, -200.0))
    # and the next fit is as ever
    mtlib.train_binned_policy(bins, N_BINS, np.zeros(500, int), np.ones(500), {"num_class": 2, "num_iterations": 1})


@gpu
def test_rows_without_a_part(mtlib):
    """A policy fit in which no row takes part grows nothing; rows that take
    none leave the others' leaf sums as they are (checked in the trees' test)."""
    bins = _bins(0, 500, 3)
    m = mtlib.train_binned_policy(bins, N_BINS, np.full(500, -1), np.ones(500), {"num_class": 2, "num_iterations": 5})
    assert m.num_trees == 0
    m = mtlib.train_binned_preference(bins, N_BINS, [0], [1], {"num_iterations": 1, "min_data_in_leaf": 1}, pair_weights=[0.0])
    assert m.num_trees == 0
