"""Losses that learn from feedback instead of labels: fits, and their losses on
device scores.

train_dense_policy and train_dense_preference (and their train_binned_ twins)
fit trees to logged decisions with advantages and to pairs of which one row
was preferred.  The other calls are the losses behind them, for callers whose
scores are torch tensors on a CUDA device: the log probabilities of taken classes,
the clipped policy loss of logged decisions and the paired preference loss,
each with its first and second derivative (include/mojotrees.h has the
formulas).  Calls run on torch's current stream of the scores' device, do not
wait for the device and can be captured into a CUDA graph.  They are not
recorded by autograd: the derivatives that a call returns are what a caller
hands on, as in scores.backward(grad).

A row takes no part, with outputs 0, when its action is negative, its weight
is 0 or every score is -inf; an action of n_classes or more gives NaN there.
torch is imported by the first call on device scores.
"""
import ctypes
import re
import threading

import numpy as np

from . import _capi
from ._capi import Model, MojoTreesError, _Err, _ptr, lib, params_string

PREFERENCE_LOSSES = {"logistic": 0, "squared": 1}

_types = None
_local = threading.local()


def _torch_types():
    """{score dtype: (C code, per-row dtype, derivatives' dtype)}, torch, and
    the function that gives a device's current stream as an integer."""
    global _types
    if _types is None:
        import torch
        # without the Stream object that torch.cuda.current_stream makes, where this torch has it
        raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        stream = raw or (lambda index: torch.cuda.current_stream(index).cuda_stream)
        _types = ({torch.float64: (0, torch.float64, torch.float32), torch.float32: (1, torch.float32, torch.float32),
                   torch.float16: (2, torch.float32, torch.float16), torch.bfloat16: (3, torch.float32, torch.bfloat16)},
                  torch, stream)
    return _types


def _err():
    """This thread's error object."""
    e = getattr(_local, "err", None)
    if e is None:
        e = _local.err = _Err()
    return e


def _invalid(message):
    return MojoTreesError(_capi.ERROR_INVALID_ARGUMENT, message)


def _vector(name, t, shape, dtype, device):
    """The address of a contiguous tensor (None: none)."""
    if t is None:
        return None
    if t.dtype is not dtype or t.shape != shape or t.device != device or not t.is_contiguous():
        raise _invalid(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)} on {device}, got "
                       f"{t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _rows(scores, actions):
    """The arguments that describe scores and actions, and what follows from them."""
    types, torch, stream = _torch_types()
    dev = scores.device
    if scores.dtype not in types:
        raise _invalid(f"scores must be float64, float32, float16 or bfloat16, got {scores.dtype}")
    if scores.dim() != 2 or dev.type != "cuda":
        raise _invalid(f"scores must be [n_rows, n_classes] on a CUDA device, got {tuple(scores.shape)} on {dev}")
    n, k = scores.shape
    stride, inner = scores.stride()
    if n <= 1:
        stride = k
    if (k > 1 and inner != 1) or stride < k:
        raise _invalid("scores must hold a row's classes next to each other and rows that do not overlap")
    if actions.dtype is torch.int32:
        width = 4
    elif actions.dtype is torch.int64:
        width = 8
    else:
        raise _invalid(f"actions must be int32 or int64, got {actions.dtype}")
    code, row, out = types[scores.dtype]
    head = (scores.data_ptr(), code, n, k, stride, _vector("actions", actions, (n,), actions.dtype, dev), width)
    return torch, head, row, out, dev, stream(dev.index)


def action_logprobs(scores, actions):
    """log softmax(scores)[actions] of [n_rows, n_classes] scores, and the row
    statistics its gradient needs: (logp [n_rows], stats [n_rows, 2]), float64
    for float64 scores and else float32."""
    torch, head, row, _, dev, stream = _rows(scores, actions)
    n = head[2]
    logp = torch.empty(n, dtype=row, device=dev)
    stats = torch.empty((n, 2), dtype=row, device=dev)
    e = _err()
    e.check(lib().mojotrees_b200_action_logprobs(*head, logp.data_ptr(), stats.data_ptr(), stream, e.h))
    return logp, stats


def action_logprobs_grad(scores, actions, stats, grad_logp, hess_logp=None):
    """Derivatives of a loss with respect to the scores from those with respect
    to action_logprobs' log probabilities (float32 [n_rows]): (grad, hess), hess
    None without hess_logp.  float32 for float64 and float32 scores, else the
    scores' type."""
    torch, head, row, out, dev, stream = _rows(scores, actions)
    n, k = head[2], head[3]
    st = _vector("stats", stats, (n, 2), row, dev)
    g = _vector("grad_logp", grad_logp, (n,), torch.float32, dev)
    h = _vector("hess_logp", hess_logp, (n,), torch.float32, dev)
    grad = torch.empty((n, k), dtype=out, device=dev)
    hess = None if hess_logp is None else torch.empty((n, k), dtype=out, device=dev)
    e = _err()
    e.check(lib().mojotrees_b200_action_logprobs_grad(*head, st, g, h, grad.data_ptr(),
                                                      None if hess is None else hess.data_ptr(), k, stream, e.h))
    return grad, hess


def policy_loss(scores, actions, advantages, old_logp, ref_logp=None, weights=None, clip_low=0.2, clip_high=0.2,
                kl_coef=0.0, grad=True, hess=False):
    """Clipped policy loss per row, with a KL term to a reference policy:
    weight * (-min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef * (exp(t) - t - 1)),
    r = exp(logp - old_logp), t = ref_logp - logp.  Per-row tensors are float64
    for float64 scores and else float32.  Returns (loss, logp, grad, hess); the
    derivatives with respect to the scores are None where not asked for."""
    torch, head, row, out, dev, stream = _rows(scores, actions)
    n, k = shape = head[2], head[3]
    if hess and not grad:
        raise _invalid("hess needs grad")
    per_row = (n,)
    rows = (_vector("advantages", advantages, per_row, row, dev), _vector("old_logp", old_logp, per_row, row, dev),
            _vector("ref_logp", ref_logp, per_row, row, dev), _vector("weights", weights, per_row, row, dev))
    loss = torch.empty(n, dtype=row, device=dev)
    logp = torch.empty(n, dtype=row, device=dev)
    dg = torch.empty(shape, dtype=out, device=dev) if grad else None
    dh = torch.empty(shape, dtype=out, device=dev) if hess else None
    e = _err()
    e.check(lib().mojotrees_b200_policy_loss(*head, *rows, clip_low, clip_high, kl_coef, loss.data_ptr(),
                                             logp.data_ptr(), None if dg is None else dg.data_ptr(),
                                             None if dh is None else dh.data_ptr(), k, stream, e.h))
    return loss, logp, dg, dh


def _index_array(name, v):
    v = np.asarray(v)
    if v.dtype.kind not in "iu" and v.size:
        raise _invalid(f"{name} must be integers, got {v.dtype}")
    return np.ascontiguousarray(v, dtype=np.int64)


class PreferencePlan:
    """The pairs of a preference loss on a device: item winners[p] was
    preferred to losers[p], with weights[p] (default 1).  Made once from host
    arrays; any number of preference_loss calls may use it, and it has to
    outlive them and the CUDA graphs that hold one.  It takes 16 bytes a pair
    (24 with weights) and 4 an item of device memory, 2 MB at least."""

    def __init__(self, winners, losers, n_items, weights=None, device=None):
        w, l = _index_array("winners", winners), _index_array("losers", losers)
        ws = None if weights is None else np.ascontiguousarray(weights, dtype=np.float32)
        if w.ndim != 1 or w.shape != l.shape or (ws is not None and ws.shape != w.shape):
            raise _invalid("winners, losers and weights must be one-dimensional and of one length")
        self.n_items, self.n_pairs = int(n_items), w.size
        e = _Err()
        h = ctypes.c_void_p()
        e.check(lib().mojotrees_b200_preference_plan_create(_ptr(w), _ptr(l), _ptr(ws), w.size, self.n_items,
                                                            -1 if device is None else int(device), ctypes.byref(h),
                                                            e.h))
        self.h = h.value

    def __del__(self):
        if getattr(self, "h", None) and _capi is not None and _capi._lib is not None:
            _capi._lib.mojotrees_b200_preference_plan_free(self.h)
            self.h = None


def preference_loss(plan, scores, reference=None, beta=1.0, label_smoothing=0.0, loss="logistic"):
    """Paired preference loss of the items' scores (raw scores or log
    probabilities of whole answers, float64 or float32 [n_items]) relative to
    a reference model's.  loss "logistic": -log sigmoid(beta u), with label
    smoothing; "squared": (u - 1 / (2 beta))^2, without; for a pair's difference u of
    score - reference.  Returns (loss [n_pairs], grad [n_items], hess
    [n_items]); the derivatives are float32."""
    types, torch, stream = _torch_types()
    dtype, dev = scores.dtype, scores.device
    if dtype not in (torch.float64, torch.float32) or dev.type != "cuda":
        raise _invalid(f"scores must be float64 or float32 on a CUDA device, got {dtype} on {dev}")
    if loss not in PREFERENCE_LOSSES:
        raise _invalid(f"loss must be one of {', '.join(PREFERENCE_LOSSES)}, got {loss!r}")
    items = (plan.n_items,)
    s = _vector("scores", scores, items, dtype, dev)
    r = _vector("reference", reference, items, dtype, dev)
    out = torch.empty(plan.n_pairs, dtype=dtype, device=dev)
    grad = torch.empty(items, dtype=torch.float32, device=dev)
    hess = torch.empty(items, dtype=torch.float32, device=dev)
    e = _err()
    e.check(lib().mojotrees_b200_preference_loss(plan.h, s, r, types[dtype][0], beta, label_smoothing,
                                                 PREFERENCE_LOSSES[loss], out.data_ptr(), grad.data_ptr(),
                                                 hess.data_ptr(), stream(dev.index), e.h))
    return out, grad, hess


def _row_array(name, v, shape, dtype=np.float64):
    if v is None:
        return None
    v = np.asarray(v)
    if dtype != np.float64 and v.dtype.kind not in "iu" and v.size:
        raise _invalid(f"{name} must be integers, got {v.dtype}")
    if v.shape != shape:
        raise _invalid(f"{name} must have shape {shape}, got {v.shape}")
    if dtype == np.int32 and v.size and (v.min() < -2 ** 31 or v.max() >= 2 ** 31):
        raise _invalid(f"{name} must fit 32 bits")
    return np.ascontiguousarray(v, dtype=dtype)


def _scores_array(v, n):
    if v is None:
        return None
    v = np.asarray(v)
    return _row_array("initial_scores", v, (n,) if v.ndim == 1 else (n, v.shape[-1]))


def _num_class(params):
    """num_class of the parameters as the library reads it: 1 when they do not
    give it, None when it is not an integer (which the library refuses)."""
    for token in params_string(params).split():
        key, _, value = token.partition(b"=")
        if key.lower() in (b"num_class", b"num_classes"):
            return int(value) if re.fullmatch(rb"[+-]?[0-9]+", value) else None
    return 1


def _check_initial(initial, params):
    k = _num_class(params)
    if initial is not None and k is not None and (1 if initial.ndim == 1 else initial.shape[1]) != max(k, 1):
        raise _invalid(f"initial_scores must have num_class = {max(k, 1)} values a row, got shape {initial.shape}")
    return initial


def _dense(X):
    X = np.asarray(X, dtype=np.float64)
    if X.ndim != 2:
        raise _invalid(f"X must be [n_rows, n_features], got shape {X.shape}")
    n, f = X.shape
    Xc = np.asfortranarray(X)
    return n, (Xc.ctypes.data_as(ctypes.c_void_p), n, f), Xc


def _binned(bins_fm, n_bins, missing_bin, n_categories):
    bins = np.ascontiguousarray(bins_fm, dtype=np.uint8)
    if bins.ndim != 2:
        raise _invalid(f"bins must be [n_features, n_rows], got shape {bins.shape}")
    f, n = bins.shape
    mb = None if missing_bin is None else _row_array("missing_bin", missing_bin, (f,), np.int32)
    nc = None if n_categories is None else _row_array("n_categories", n_categories, (f,), np.int32)
    return n, (_ptr(bins), n, f, n_bins, _ptr(mb), _ptr(nc)), (bins, mb, nc)


def _fit(fn, data, keep, args, params):
    e = _Err()
    h = ctypes.c_void_p()
    e.check(fn(*data, *args, params_string(params), ctypes.byref(h), e.h))
    del keep
    return Model(h.value)


def _preference_args(n, winners, losers, pair_weights, actions, reference, initial_scores, params):
    w, l = _index_array("winners", winners), _index_array("losers", losers)
    pw = None if pair_weights is None else np.ascontiguousarray(pair_weights, dtype=np.float32)
    if w.ndim != 1 or w.shape != l.shape or (pw is not None and pw.shape != w.shape):
        raise _invalid("winners, losers and pair_weights must be one-dimensional and of one length")
    a = _row_array("actions", actions, (n,), np.int32)
    r = _row_array("reference", reference, (n,))
    s = _check_initial(_scores_array(initial_scores, n), params)
    return (_ptr(w), _ptr(l), _ptr(pw), w.size, _ptr(a), _ptr(r), _ptr(s)), (w, l, pw, a, r, s)


def _policy_args(n, actions, advantages, old_logp, ref_logp, weights, initial_scores, params):
    a = _row_array("actions", actions, (n,), np.int32)
    rows = [_row_array(name, v, (n,)) for name, v in (("advantages", advantages), ("old_logp", old_logp),
                                                      ("ref_logp", ref_logp), ("weights", weights))]
    s = _check_initial(_scores_array(initial_scores, n), params)
    return (_ptr(a), *[_ptr(v) for v in rows], _ptr(s)), (a, rows, s)


def train_dense_preference(X, winners, losers, params=None, pair_weights=None, actions=None, reference=None,
                           initial_scores=None):
    """Fit a float64 matrix [n_rows, n_features] to pairs of rows, row
    winners[p] preferred to row losers[p].  With num_class > 1 in params a row
    stands for the class actions says it took.  The model adds to
    initial_scores ([n_rows] or [n_rows, num_class]; default 0)."""
    n, data, keep = _dense(X)
    args, more = _preference_args(n, winners, losers, pair_weights, actions, reference, initial_scores, params)
    return _fit(lib().mojotrees_b200_train_dense_preference, data, (keep, more), args, params)


def train_binned_preference(bins_fm, n_bins, winners, losers, params=None, pair_weights=None, actions=None,
                            reference=None, initial_scores=None, missing_bin=None, n_categories=None):
    """train_dense_preference on feature-major uint8 bins [n_features, n_rows]."""
    n, data, keep = _binned(bins_fm, n_bins, missing_bin, n_categories)
    args, more = _preference_args(n, winners, losers, pair_weights, actions, reference, initial_scores, params)
    return _fit(lib().mojotrees_b200_train_binned_u8_preference, data, (keep, more), args, params)


def train_dense_policy(X, actions, advantages, params=None, old_logp=None, ref_logp=None, weights=None,
                       initial_scores=None):
    """Fit a policy over params' num_class classes to logged decisions: row r
    took actions[r] (-1: takes no part) with advantage advantages[r].
    old_logp and ref_logp are the actions' log probabilities under the policy
    that took them and under the reference; by default both are the policy
    that the fit starts from, softmax(initial_scores [n_rows, num_class])."""
    n, data, keep = _dense(X)
    args, more = _policy_args(n, actions, advantages, old_logp, ref_logp, weights, initial_scores, params)
    return _fit(lib().mojotrees_b200_train_dense_policy, data, (keep, more), args, params)


def train_binned_policy(bins_fm, n_bins, actions, advantages, params=None, old_logp=None, ref_logp=None, weights=None,
                        initial_scores=None, missing_bin=None, n_categories=None):
    """train_dense_policy on feature-major uint8 bins [n_features, n_rows]."""
    n, data, keep = _binned(bins_fm, n_bins, missing_bin, n_categories)
    args, more = _policy_args(n, actions, advantages, old_logp, ref_logp, weights, initial_scores, params)
    return _fit(lib().mojotrees_b200_train_binned_u8_policy, data, (keep, more), args, params)
