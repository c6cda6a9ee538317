"""Operators over class scores against plain 64-bit numpy, on the host and on the GPU.

Tolerances. The device takes exponentials of (z - high) * s with s = log2(e) / T in 32 bits
(64 for float64 scores), eps = 2^-24 (2^-53) being half a step. One term of a softmax with
exponent x (base two) is off by at most eps * (3 |x| + 4) of itself: the roundings of s, of the
difference and of the product, and one step of the exponential; as 2^-x (3 |x| + 4) <= 5.7, that
is below 8 eps of the row's largest term, and below (2 * 64 + 4) eps of the term for every term
above 2^-42; of up to 2^20 classes, what is smaller adds up to 2^-22. A sum of n terms adds at
most one rounding for each addition along its longest chain: n / 64 + 32 (a lane's own terms,
then the tree). `_rel` is the sum of these; a result's own rounding to
its type is added where it is compared. The 32-bit gradients of float64 scores are allowed the
32-bit terms: the device computes them in 64 and needs less.
"""
import math
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest

import lightgbm_amd as lgb
from lightgbm_amd import ops
from lightgbm_amd.basic import LightGBMError

torch = pytest.importorskip("torch")

PLACES = ["numpy", "torch", pytest.param("gpu", marks=pytest.mark.gpu)]
INF = math.inf
HALF_STEP = {"f64": 2.0 ** -53, "f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f64": 0.0, "f32": 2.0 ** -126, "f16": 2.0 ** -25, "bf16": 2.0 ** -126}
TORCH = {"f64": torch.float64, "f32": torch.float32, "f16": torch.float16,
         "bf16": torch.bfloat16, "i32": torch.int32, "i64": torch.int64}


def _rel(classes, dtype):
    return (2 * 64 + 4 + 2 * (classes / 64 + 32)) * HALF_STEP["f64" if dtype == "f64" else "f32"]


def _round(x, dtype):
    """x (float64) rounded to a type, as float64."""
    return torch.from_numpy(np.ascontiguousarray(x)).to(TORCH[dtype]).double().numpy()


def _put(place, x, dtype=None, order="C", pad=0):
    """A numpy array as an array of the place, row- or class-major; `pad` columns of NaN (or -7)
    stand between its rows."""
    if x is None:
        return None
    x = np.asarray(x)
    if pad and x.ndim == 2:
        wide = np.full((x.shape[0], x.shape[1] + pad), np.nan if x.dtype.kind == "f" else -7,
                       dtype=x.dtype)
        wide[:, :x.shape[1]] = x
        return _put(place, wide, dtype, order)[:, :x.shape[1]]
    if place == "numpy":
        kind = {"f64": np.float64, "f32": np.float32, "f16": np.float16, "i32": np.int32,
                "i64": np.int64, None: x.dtype}[dtype]
        return np.array(x, dtype=kind, order=order)
    t = torch.from_numpy(np.array(x))
    if dtype is not None:
        t = t.to(TORCH[dtype])
    if order == "F":
        t = t.t().contiguous().t()
    return t.cuda() if place == "gpu" else t


def _get(x):
    if x is None or isinstance(x, np.ndarray):
        return x
    x = x.cpu()
    return (x.double() if x.dtype.is_floating_point else x).numpy()


def _types(place):
    return ["f64", "f32", "f16"] + ([] if place == "numpy" else ["bf16"])


# ------------------------------------------------------------------ plain forms, 64 bits
def _lse(v):
    v = np.asarray(v, dtype=np.float64)
    high = v.max() if v.size else -INF
    if not np.isfinite(high):
        return high
    return high + math.log(np.exp(v - high).sum())


def _plain_top(x, k, t):
    n, c = x.shape
    classes = np.full((n, k), -1)
    logits = np.full((n, k), -INF)
    rest = np.empty(n)
    for i in range(n):
        able = [j for j in range(c) if x[i, j] > -INF]
        order = sorted(able, key=lambda j: (-x[i, j], j))
        classes[i, :len(order[:k])] = order[:k]
        logits[i, :len(order[:k])] = x[i, order[:k]]
        rest[i] = _lse([x[i, j] / t for j in order[k:]])
    return classes, logits, rest


def _plain_distill(z, classes, logits, rest, labels, weight, t, alpha):
    """loss, gradient, hessian, and the scale that the gradient's error is relative to."""
    n, c = z.shape
    loss, grad, hess = np.zeros(n), np.zeros((n, c)), np.zeros((n, c))
    size_l, size_g = np.zeros(n), np.zeros((n, c))
    factor = c / (c - 1) if c > 1 else 1.0
    for i in range(n):
        w = 1.0 if weight is None else weight[i]
        if w == 0 or z[i].max() == -INF:
            continue
        with np.errstate(all="ignore"):
            # against the row's maximum: of z = 5000 alone, 64 bits keep 5e-13
            d = z[i] - (z[i].max() if z[i].max() < INF else 0.0)
            log_q = d / t - _lse(d / t)
            log_1 = d - _lse(d)
        q, q1 = np.exp(log_q), np.exp(log_1)
        slot = {}
        for j in range(classes.shape[1]):
            if 0 <= classes[i, j] < c:
                slot.setdefault(int(classes[i, j]), logits[i, j] / t)
        r = -INF if rest is None else rest[i]
        norm = _lse(list(slot.values()) + [r])
        others = np.array([j not in slot for j in range(c)])
        if norm > -INF and alpha > 0:
            log_rho = _lse(log_q[others])
            want = np.zeros(c)
            total = 0.0
            spread = 0.0
            for j, v in slot.items():
                lp = v - norm
                want[j] = math.exp(lp)
                if want[j] > 0:
                    total += want[j] * (lp - log_q[j])
                    spread += want[j] * (abs(lp) + abs(log_q[j]))
            share = math.exp(r - norm)
            if share > 0:
                total += share * (r - norm - log_rho)
                spread += share * (abs(r - norm) + abs(log_rho))
                if log_rho > -INF:
                    want[others] = share * np.exp(log_q[others] - log_rho)
            loss[i] += alpha * t * t * total
            size_l[i] += alpha * t * t * (2 + spread)
            grad[i] += alpha * t * (q - want)
            size_g[i] += alpha * t * (q + want)
            hess[i] += alpha * q * (1 - q)
        if alpha < 1 and 0 <= labels[i] < c:
            y = int(labels[i])
            loss[i] -= (1 - alpha) * log_1[y]
            size_l[i] += (1 - alpha) * (2 + abs(log_1[y]))
            grad[i] += (1 - alpha) * (q1 - (np.arange(c) == y))
            size_g[i] += (1 - alpha) * (q1 + (np.arange(c) == y))
            hess[i] += (1 - alpha) * q1 * (1 - q1)
        loss[i] *= w
        size_l[i] *= abs(w)
        grad[i] *= w
        size_g[i] *= abs(w)
        hess[i] *= w * factor
    return loss, grad, hess, size_l, size_g


def _plain_verify(p, drafts, q, u, v, lengths):
    b, t1, c = p.shape
    mass = lambda a: np.where((a > 0) & np.isfinite(a), a, 0.0)  # noqa: E731
    p = mass(p)
    q = None if q is None else mass(q)
    classes = np.full((b, t1), -1)
    accepted = np.zeros(b, dtype=int)
    for i in range(b):
        length = t1 - 1 if lengths is None else min(max(int(lengths[i]), 0), t1 - 1)
        s = 0
        while s < length:
            x = int(drafts[i, s])
            if not 0 <= x < c:
                break
            if not u[i, s] * (1.0 if q is None else q[i, s, x]) < p[i, s, x]:
                break
            classes[i, s] = x
            s += 1
        left = p[i, s].copy()
        if s < length:
            if q is not None:
                left = np.maximum(left - q[i, s], 0)
            elif 0 <= drafts[i, s] < c:
                left[drafts[i, s]] = 0
        if left.sum() == 0:
            left = p[i, s]
        accepted[i] = s
        if left.sum() > 0:
            reach = np.cumsum(left)
            # a class without mass is never drawn, not for a sample below zero either
            over = np.nonzero((reach > v[i] * reach[-1]) & (left > 0))[0]
            classes[i, s] = over[0] if len(over) else np.nonzero(left)[0][-1]
    return classes, accepted


# ------------------------------------------------------------------ top logits
def _top_case(place, x, dtype, k, t=1.0, order="C", pad=0):
    x = _round(x, dtype)
    got = ops.top_logits(_put(place, x, dtype, order, pad), k, temperature=t)
    classes, logits, rest = _plain_top(x, k, t)
    np.testing.assert_array_equal(_get(got.classes), classes)
    np.testing.assert_array_equal(_get(got.logits), logits)
    out = "f64" if dtype == "f64" else "f32"
    where = np.isfinite(rest)
    # the maximum over T is rounded, and scaled by a rounded s
    far = _rel(x.shape[1], dtype) * (1 + np.abs(rest[where]))
    assert np.all(np.abs(_get(got.log_rest)[where] - rest[where]) <=
                  far + 2 * HALF_STEP[out] * np.abs(rest[where]))
    np.testing.assert_array_equal(_get(got.log_rest)[~where], rest[~where])
    return got


@pytest.mark.parametrize("place", PLACES)
@pytest.mark.parametrize("rows,classes,k", [
    (1, 1, 1), (3, 2, 1), (5, 7, 3), (70, 10, 10), (130, 33, 4), (3, 64, 64), (2, 65, 20),
    (37, 100, 10), (9, 300, 9), (4, 257, 256), (20, 512, 100), (9, 1000, 17), (2, 1025, 100),
    (3, 4099, 64), (2, 20011, 256), (1, 70001, 33), (1, 200003, 40)])
def test_top_logits_sizes(place, rows, classes, k):
    rng = np.random.default_rng(rows * classes + k)
    for dtype in _types(place):
        _top_case(place, 3 * rng.standard_normal((rows, classes)), dtype, k, t=1.7)
        _top_case(place, 3 * rng.standard_normal((rows, classes)), dtype, k, order="F", pad=1)
        _top_case(place, 3 * rng.standard_normal((rows, classes)), dtype, k, t=0.5, pad=3)


@pytest.mark.parametrize("place", PLACES)
@pytest.mark.parametrize("classes", [6, 100, 300, 5000, 40001])
def test_top_logits_ties(place, classes):
    """Constant rows, rows of few values, signed zeros, sorted rows: the lowest classes win."""
    rng = np.random.default_rng(classes)
    k = min(50, classes - 1)
    rows = [np.zeros(classes), np.full(classes, -3.25), np.arange(classes) * 0.0 - 0.0,
            rng.integers(0, 3, classes).astype(float), np.arange(classes) / 8.0,
            -np.arange(classes) / 8.0, np.where(np.arange(classes) % 2, 0.0, -0.0),
            np.where(np.arange(classes) == classes - 1, 50.0, -80.0),
            np.minimum(np.arange(classes), 7.0)]
    for dtype in _types(place):
        for order in "CF":
            _top_case(place, np.stack(rows), dtype, k, order=order)


@pytest.mark.parametrize("place", PLACES)
@pytest.mark.parametrize("classes", [5, 90, 3000, 33000])
def test_top_logits_masked(place, classes):
    rng = np.random.default_rng(classes)
    x = rng.standard_normal((8, classes))
    x[0] = -INF
    x[1] = np.nan
    x[2, 1:] = -INF
    x[3, ::2] = np.nan
    x[4, 3:] = -INF
    x[5, -1] = INF
    x[6, :classes // 2] = np.finfo(np.float16).min
    x[7, :] = np.where(np.arange(classes) < 2, x[7], np.nan)
    for dtype in _types(place):
        for order in "CF":
            _top_case(place, x, dtype, 4, order=order)


@pytest.mark.parametrize("place", PLACES)
def test_top_logits_confident(place):
    """What is left stands far below the best: it is summed against its own maximum."""
    for classes in (12, 400, 9000):
        x = np.random.default_rng(1).standard_normal((3, classes))
        x[:, 2] = 400.0
        x[1, 3] = 300.0
        for dtype in _types(place):
            _top_case(place, x, dtype, 1)
            _top_case(place, x, dtype, 2, t=0.25)


# ------------------------------------------------------------------ distillation
def _teacher(rng, rows, classes, k, rest, masked=False):
    ids = np.stack([rng.permutation(max(classes, k))[:k] for _ in range(rows)])
    logits = np.sort(8 * rng.random((rows, k)), axis=1)[:, ::-1].astype(np.float32)
    ids = np.where(ids < classes, ids, -1)
    r = (1 + 3 * rng.random(rows)).astype(np.float32) if rest else None
    if masked:
        ids[::3, (k + 1) // 2:] = -1
        logits = np.where(ids < 0, np.nan, logits).astype(np.float32)
        ids[1::5] = -1
        if rest:
            r[1::5] = -INF
    return ids, logits, r


def _distill_case(place, z, teacher, dtype, labels=None, weight=None, t=1.0, alpha=1.0,
                  order="C", pad=0, int_type="i32"):
    z = _round(z, dtype)
    ids, logits, rest = teacher
    put_teacher = ops.TopLogits(_put(place, ids, int_type), _put(place, logits, "f32"),
                                _put(place, rest, "f32"))
    args = (_put(place, z, dtype, order, pad), put_teacher)
    mix = {"labels": _put(place, labels, int_type), "weight": _put(place, weight, "f32"),
           "temperature": t, "alpha": alpha}
    w = None if weight is None else np.asarray(weight, np.float32).astype(np.float64)
    loss, grad, hess, size_l, size_g = _plain_distill(
        z, ids, logits.astype(np.float64), None if rest is None else rest.astype(np.float64),
        labels, w, t, alpha)
    rel = _rel(z.shape[1], dtype)
    out = "f32" if dtype == "f64" else dtype
    got_loss = _get(ops.distill_loss(*args, **mix))
    got = ops.distill_gradients(*args, hessian=True, loss=True, **mix)
    alone = ops.distill_gradients(*args, **mix)
    with np.errstate(invalid="ignore"):
        close = np.abs(got_loss - loss) <= 3 * rel * size_l + HALF_STEP[
            "f64" if dtype == "f64" else "f32"] * np.abs(loss)
    same = (got_loss == loss) | (np.isnan(got_loss) & np.isnan(loss))
    assert np.all(close | same)
    np.testing.assert_array_equal(got_loss, _get(got.loss))
    np.testing.assert_array_equal(_get(got.gradient), _get(alone.gradient))
    assert alone.hessian is None and alone.loss is None
    rel = _rel(z.shape[1], "f32")
    for a, b, size in ((_get(got.gradient), grad, size_g), (_get(got.hessian), hess, size_g)):
        # a hessian q (1 - q) is off by what q is, relative to q at most
        far = 3 * rel * size * (z.shape[1] / max(1, z.shape[1] - 1)) / min(t, 1.0)
        far = far + (1 + rel) * HALF_STEP[out] * np.abs(b) + TINY[out]
        with np.errstate(invalid="ignore"):
            close = np.abs(a - b) <= far
        assert np.all(close | (np.isnan(a) & np.isnan(b))), np.nanmax(np.abs(a - b) - far)
    return got


SIZES = [(1, 1, 1), (2, 2, 1), (5, 3, 2), (70, 7, 3), (200, 10, 10), (65, 33, 9), (3, 64, 20),
         (66, 65, 64), (3, 300, 150), (4, 1000, 8), (2, 1025, 256), (3, 4099, 50), (2, 20011, 17),
         (20, 512, 30), (1, 70001, 64), (1, 200003, 40)]


@pytest.mark.parametrize("place", PLACES)
@pytest.mark.parametrize("rows,classes,k", SIZES)
@pytest.mark.parametrize("rest", [False, True])
def test_distill_sizes(place, rows, classes, k, rest):
    rng = np.random.default_rng(rows + classes + k)
    teacher = _teacher(rng, rows, classes, k, rest and classes > k)
    labels = rng.integers(0, classes, rows)
    for dtype in _types(place):
        z = 3 * rng.standard_normal((rows, classes))
        _distill_case(place, z, teacher, dtype, t=2.0)
        _distill_case(place, z, teacher, dtype, labels=labels, t=1.0, alpha=0.25, order="F",
                      int_type="i64")
        _distill_case(place, z, teacher, dtype, labels=labels, t=3.0, alpha=0.5, pad=3)
        _distill_case(place, z, teacher, dtype, labels=labels, t=1.5, alpha=0.0, order="F", pad=1)


@pytest.mark.parametrize("place", PLACES)
@pytest.mark.parametrize("classes", [9, 130, 1500, 17000])
def test_distill_masked(place, classes):
    """Masked classes, rows with nothing in them, padding of any contents, empty slots, rows
    without a teacher or a label, the same class twice, ids out of range."""
    rng = np.random.default_rng(classes)
    rows, k = 21, 6
    ids, logits, rest = _teacher(rng, rows, classes, k, True, masked=True)
    ids[6, 2] = ids[6, 0] = 1
    ids[6, 1] = 2
    logits[6] = [1, 2, 3, 4, 5, 6]
    ids[9] = [3, 3, 3, 3, 3, 3]
    logits[9] = [0, 1, np.nan, INF, 2, 3]
    ids[12] = [classes, -5, 2 ** 31 - 1, 0, -1, 1]
    logits[12] = [9, 9, 9, 1, np.nan, 2]
    z = 2 * rng.standard_normal((rows, classes))
    z[rng.random((rows, classes)) < 0.2] = -INF
    np.put_along_axis(z, np.clip(ids, 0, classes - 1), 0.5, axis=1)
    z[10] = -INF
    z[13, classes // 2:] = np.finfo(np.float16).min
    weight = rng.random(rows).astype(np.float32) + 0.5
    weight[4] = 0.0
    z[4] = np.nan
    weight[5] = -1.5
    labels = rng.integers(0, classes, rows)
    labels[2], labels[3], labels[8] = -1, classes, -100
    z[np.arange(rows), np.clip(labels, 0, classes - 1)] = np.where(
        np.arange(rows) == 4, np.nan, 1.0)
    z[10] = -INF
    for dtype in _types(place):
        for order in "CF":
            for r in (rest, None):
                _distill_case(place, z, (ids, logits, r), dtype, labels=labels, weight=weight,
                              t=2.0, alpha=0.5, order=order)
                _distill_case(place, z, (ids, logits, r), dtype, weight=weight, t=1.0,
                              order=order, pad=2)


@pytest.mark.parametrize("place", PLACES)
@pytest.mark.parametrize("classes", [8, 200, 6000])
def test_distill_far_apart(place, classes):
    """A student sure of its class: the others' share underflows, and is summed again."""
    rng = np.random.default_rng(3)
    z = rng.standard_normal((4, classes))
    z[:, 2] = 30.0
    z[1, 2] = 120.0
    z[2, 2] = 900.0
    z[3] += 5000.0
    ids = np.full((4, 3), -1)
    ids[:, 0] = 2
    logits = np.zeros((4, 3), np.float32)
    rest = np.zeros(4, np.float32)
    for dtype in _types(place):
        for order in "CF":
            _distill_case(place, z, (ids, logits, rest), dtype, order=order)
            _distill_case(place, z, (ids, logits, rest), dtype, t=0.5, order=order)


@pytest.mark.parametrize("place", PLACES)
@pytest.mark.parametrize("classes", [6, 150, 5000])
def test_distill_infinite(place, classes):
    """A teacher's class that the student masks costs an infinite loss and a finite gradient;
    NaN and +inf among the scores make NaN of their row alone."""
    rng = np.random.default_rng(4)
    z = rng.standard_normal((5, classes))
    z[0, 1] = -INF
    z[1, 4] = np.nan
    z[2, 4] = INF
    z[3, 3:] = -INF
    ids = np.tile([1, 0, 2], (5, 1))
    logits = np.tile(np.float32([3, 2, 1]), (5, 1))
    rest = np.float32([0.5, 0.5, 0.5, 0.5, 0.5])
    for dtype in _types(place):
        for order in "CF":
            args = (_put(place, z, dtype, order),
                    ops.TopLogits(_put(place, ids, "i32"), _put(place, logits, "f32"),
                                  _put(place, rest, "f32")))
            loss = _get(ops.distill_loss(*args))
            grad = _get(ops.distill_gradients(*args).gradient)
            assert loss[0] == INF and loss[3] == INF and np.isfinite(loss[4])
            assert np.isnan(loss[1]) and np.isnan(loss[2])
            assert np.all(np.isfinite(grad[[0, 3, 4]]))
            assert np.all(np.isnan(grad[[1, 2]]))
            assert grad[0, 1] < 0 and np.all(grad[3, 3:] == 0)


@pytest.mark.parametrize("place", PLACES)
@pytest.mark.parametrize("order", ["C", "F"])
@pytest.mark.parametrize("classes", [5, 140])
def test_distill_gradient_is_the_slope(place, order, classes):
    """Central differences of the float64 loss: the third derivative of the loss is at most
    2 alpha / T + 1, so a step h leaves h^2 / 3 and the loss's rounding over h. The gradient
    itself is computed in 32 bits."""
    rng = np.random.default_rng(11)
    rows, k, h = 4, 3, 1e-5
    ids, logits, rest = _teacher(rng, rows, classes, k, True)
    labels = rng.integers(0, classes, rows)
    weight = np.float32([1.0, 0.5, 2.0, 1.0])
    z = rng.standard_normal((rows, classes))
    teacher = ops.TopLogits(_put(place, ids, "i32"), _put(place, logits, "f32"),
                            _put(place, rest, "f32"))
    mix = {"labels": _put(place, labels, "i32"), "weight": _put(place, weight, "f32"),
           "temperature": 2.0, "alpha": 0.6}
    grad = _get(ops.distill_gradients(_put(place, z, "f64", order), teacher, **mix).gradient)

    def loss(x):
        return _get(ops.distill_loss(_put(place, x, "f64", order), teacher, **mix))

    top = np.abs(loss(z)).max()
    size_g = _plain_distill(z, ids, logits.astype(float), rest.astype(float), labels,
                            weight.astype(float), 2.0, 0.6)[4]
    for c in range(0, classes, max(1, classes // 7)):
        up, down = z.copy(), z.copy()
        up[:, c] += h
        down[:, c] -= h
        slope = (loss(up) - loss(down)) / (2 * h)
        far = 2 * 3 * h * h + 2 * 3 * _rel(classes, "f64") * (10 + top) / h
        far = far + 3 * _rel(classes, "f32") * size_g[:, c]
        assert np.all(np.abs(slope - grad[:, c]) <= far + HALF_STEP["f32"] * np.abs(grad[:, c]))


@pytest.mark.parametrize("place", PLACES)
def test_distill_broadcast_and_strides(place):
    """One row of scores for all teachers, teachers in any order of memory, every second row."""
    rng = np.random.default_rng(5)
    ids, logits, rest = _teacher(rng, 6, 40, 5, True)
    z = np.float32(rng.standard_normal((1, 40)))
    many = np.repeat(z, 6, 0)
    want = ops.distill_gradients(_put(place, many, "f32"), ops.TopLogits(
        _put(place, ids, "i32"), _put(place, logits, "f32"), _put(place, rest, "f32")), loss=True)
    if place == "numpy":
        one = np.broadcast_to(z, (6, 40))
    else:
        one = _put(place, z, "f32").expand(6, 40)
    twice = _put(place, np.repeat(ids, 2, 0), "i64")[::2]
    got = ops.distill_gradients(one, (twice, _put(place, logits, "f32", "F"),
                                      _put(place, rest, "f64")), loss=True)
    np.testing.assert_array_equal(_get(got.gradient), _get(want.gradient))
    np.testing.assert_array_equal(_get(got.loss), _get(want.loss))


# ------------------------------------------------------------------ verification
def _softmax(x):
    e = np.exp(x - x.max(-1, keepdims=True))
    return e / e.sum(-1, keepdims=True)


def _verify_case(place, p, drafts, q, u, v, lengths, dtype, int_type="i32", uniform="f32"):
    p = _round(p, dtype)
    q = None if q is None else _round(q, dtype)
    u, v = _round(u, uniform), _round(v, uniform)
    got = ops.verify_drafts(_put(place, p, dtype), _put(place, drafts, int_type),
                            _put(place, q, dtype), _put(place, u, uniform),
                            _put(place, v, uniform), lengths=_put(place, lengths, int_type))
    classes, accepted = _plain_verify(p, drafts, q, u, v, lengths)
    np.testing.assert_array_equal(_get(got.accepted), accepted)
    np.testing.assert_array_equal(_get(got.classes), classes)


@pytest.mark.parametrize("place", PLACES)
@pytest.mark.parametrize("rows,t,classes", [
    (1, 1, 1), (1, 4, 2), (300, 3, 10), (67, 1, 63), (40, 5, 64), (33, 2, 65), (20, 70, 130),
    (9, 3, 1000), (5, 2, 4099), (3, 4, 20011), (2, 1, 70001), (1, 2, 131072)])
def test_verify_sizes(place, rows, t, classes):
    rng = np.random.default_rng(rows + t + classes)
    x = 2 * rng.standard_normal((rows, t + 1, classes))
    p = _softmax(x)
    q = _softmax(x[:, :t] + 0.7 * rng.standard_normal((rows, t, classes)))
    drafts = (q / rng.exponential(size=q.shape)).argmax(-1)
    u, v = rng.random((rows, t)), rng.random(rows)
    lengths = rng.integers(0, t + 1, rows)
    for dtype in _types(place):
        _verify_case(place, p, drafts, q, u, v, None, dtype)
        _verify_case(place, p, drafts, q, u, v, lengths, dtype, "i64", "f64")
        _verify_case(place, p, p[:, :t].argmax(-1), None, u, v, lengths, dtype)


@pytest.mark.parametrize("place", PLACES)
@pytest.mark.parametrize("classes", [4, 70, 5000])
def test_verify_borders(place, classes):
    """Sums that are exact in every order, numbers that stand on a border or outside [0, 1),
    entries that are no probability, lengths and ids out of range, rows with no mass."""
    rows, t = 16, 2
    p = np.zeros((rows, t + 1, classes))
    p[..., 1], p[..., 3], p[..., classes - 1] = 0.25, 0.25, 0.5
    q = np.zeros((rows, t, classes))
    q[..., 1], q[..., 3], q[..., 0] = 0.5, 0.25, 0.25
    drafts = np.tile([1, 3], (rows, 1))
    u = np.full((rows, t), 0.25)
    v = np.zeros(rows)
    lengths = np.full(rows, t)
    u[0] = 0.5                # 0.5 * 0.5 < 0.25 is false: refused
    u[1, 1] = 1.0             # 1 * 0.25 < 0.25 is false
    v[2], v[3], v[4], v[5] = 0.25, 0.5, 1.0, 2.0
    v[6] = np.nan
    drafts[7, 0], drafts[8, 1] = -1, classes
    lengths[9], lengths[10] = -3, 99
    p[11, :, 1], q[11, :, 0] = np.nan, INF
    p[12] = 0.0
    q[13] = np.maximum(p[13, :t], q[13])   # nothing of the target is left
    u[13] = 1.0
    p[14, :, 0] = -1.0
    v[15], u[15] = -0.5, np.nan
    for dtype in _types(place):
        for uniform in ("f32", "f64"):
            _verify_case(place, p, drafts, q, u, v, lengths, dtype, uniform=uniform)
            _verify_case(place, p, drafts, None, u, v, lengths, dtype, uniform=uniform)


@pytest.mark.parametrize("place", PLACES)
def test_verify_strides(place):
    rng = np.random.default_rng(8)
    p = _softmax(rng.standard_normal((6, 4, 50))).astype(np.float32)
    q = _softmax(rng.standard_normal((6, 3, 50))).astype(np.float32)
    drafts = rng.integers(0, 50, (6, 3))
    u, v = rng.random((6, 3)).astype(np.float32), rng.random(6).astype(np.float32)
    want = ops.verify_drafts(*[_put(place, x) for x in (p, drafts, q, u, v)])
    turn = lambda x: _put(place, np.ascontiguousarray(x.transpose(2, 0, 1)))  # noqa: E731
    moved = [turn(p), turn(q)]
    moved = [x.transpose(1, 2, 0) if place == "numpy" else x.permute(1, 2, 0) for x in moved]
    got = ops.verify_drafts(moved[0], _put(place, np.repeat(drafts, 2, 1))[:, ::2], moved[1],
                            _put(place, u, order="F"), _put(place, np.repeat(v, 2))[::2])
    np.testing.assert_array_equal(_get(got.classes), _get(want.classes))
    np.testing.assert_array_equal(_get(got.accepted), _get(want.accepted))


@pytest.mark.parametrize("place", PLACES)
def test_verify_distribution(place):
    """The first class of every sequence is distributed as the target, whatever the draft: over
    n sequences a frequency is off by at most 5 standard deviations of sqrt(p (1 - p) / n)."""
    rng = np.random.default_rng(9)
    n, c = 40000, 8
    p0 = _softmax(rng.standard_normal(c))
    q0 = _softmax(rng.standard_normal(c))
    p = np.broadcast_to(p0, (n, 2, c))
    q = np.broadcast_to(q0, (n, 1, c))
    drafts = (q / rng.exponential(size=(n, 1, c))).argmax(-1)
    got = ops.verify_drafts(*[_put(place, np.ascontiguousarray(x)) for x in
                              (p, drafts, q, rng.random((n, 1)), rng.random(n))])
    seen = np.bincount(_get(got.classes)[:, 0], minlength=c) / n
    assert np.all(np.abs(seen - p0) <= 5 * np.sqrt(p0 * (1 - p0) / n))


# ------------------------------------------------------------------ the set together, refusals
@pytest.mark.parametrize("place", PLACES)
@pytest.mark.parametrize("classes", [12, 3000])
def test_teacher_to_student(place, classes):
    """A student that starts from zero scores follows its gradient to the teacher: its loss does
    not rise, and a student that has the teacher's scores has no loss and no gradient."""
    rng = np.random.default_rng(12)
    scores = _put(place, 2 * rng.standard_normal((5, classes)).astype(np.float32))
    teacher = ops.top_logits(scores, 5, temperature=2.0)
    loss = _get(ops.distill_loss(scores, teacher, temperature=2.0))
    # KL of two roundings of one distribution: first order terms cancel up to their error
    assert np.all(np.abs(loss) <= 4 * 3 * _rel(classes, "f32") * 20)
    grad = _get(ops.distill_gradients(scores, teacher, temperature=2.0).gradient)
    assert np.all(np.abs(grad) <= 2 * 6 * _rel(classes, "f32"))


@pytest.mark.parametrize("place", PLACES)
def test_no_rows(place):
    top = ops.top_logits(_put(place, np.zeros((0, 5), np.float32)), 2)
    assert tuple(top.classes.shape) == (0, 2) and tuple(top.log_rest.shape) == (0,)
    z = _put(place, np.zeros((0, 5), np.float32))
    got = ops.distill_gradients(z, top, hessian=True, loss=True)
    assert tuple(got.gradient.shape) == (0, 5) and tuple(got.loss.shape) == (0,)
    p = _put(place, np.zeros((0, 3, 5), np.float32))
    got = ops.verify_drafts(p, _put(place, np.zeros((0, 2), np.int32)), None,
                            _put(place, np.zeros((0, 2), np.float32)),
                            _put(place, np.zeros(0, np.float32)))
    assert tuple(got.classes.shape) == (0, 3)


@pytest.mark.parametrize("place", PLACES)
def test_refusals(place):
    f = lambda *shape: _put(place, np.ones(shape, np.float32))  # noqa: E731
    i = lambda *shape: _put(place, np.ones(shape, np.int32))  # noqa: E731
    teacher = (i(3, 2), f(3, 2))
    bad = [
        lambda: ops.top_logits(f(3, 4), 0),
        lambda: ops.top_logits(f(3, 4), 5),
        lambda: ops.top_logits(f(3, 400), 257),
        lambda: ops.top_logits(f(4), 1),
        lambda: ops.top_logits(f(3, 0), 1),
        lambda: ops.top_logits(i(3, 4), 1),
        lambda: ops.top_logits(f(3, 4), 1, temperature=0.0),
        lambda: ops.top_logits(f(3, 4), 1, temperature=-1.0),
        lambda: ops.top_logits(f(3, 4), 1, temperature=math.nan),
        lambda: ops.top_logits(f(3, 4), 1, temperature=math.inf),
        lambda: ops.distill_loss(f(3, 4), (i(2, 2), f(2, 2))),
        lambda: ops.distill_loss(f(3, 4), (i(3, 2), f(3, 3))),
        lambda: ops.distill_loss(f(3, 4), (f(3, 2), f(3, 2))),
        lambda: ops.distill_loss(f(3, 4), (i(3, 2), i(3, 2))),
        lambda: ops.distill_loss(f(3, 4), (i(3, 2),)),
        lambda: ops.distill_loss(f(3, 4), (i(3, 2), f(3, 2), f(3, 1))),
        lambda: ops.distill_loss(f(3, 4), (i(3, 257), f(3, 257))),
        lambda: ops.distill_loss(f(3, 4), (i(3, 0), f(3, 0))),
        lambda: ops.distill_loss(f(3, 4), teacher, alpha=0.5),
        lambda: ops.distill_loss(f(3, 4), teacher, alpha=1.5),
        lambda: ops.distill_loss(f(3, 4), teacher, alpha=math.nan),
        lambda: ops.distill_loss(f(3, 4), teacher, temperature=0.0),
        lambda: ops.distill_loss(f(3, 4), teacher, labels=i(2), alpha=0.5),
        lambda: ops.distill_loss(f(3, 4), teacher, weight=f(4)),
        lambda: ops.distill_loss(f(3, 4), teacher, weight=i(3)),
        lambda: ops.distill_gradients(f(3, 4, 1), teacher),
        lambda: ops.verify_drafts(f(2, 1, 4), i(2, 0), None, f(2, 0), f(2)),
        lambda: ops.verify_drafts(f(2, 3, 4), i(2, 3), None, f(2, 3), f(2)),
        lambda: ops.verify_drafts(f(2, 3, 4), i(2, 2), f(2, 3, 4), f(2, 2), f(2)),
        lambda: ops.verify_drafts(f(2, 3, 4), f(2, 2), None, f(2, 2), f(2)),
        lambda: ops.verify_drafts(f(2, 3, 4), i(2, 2), None, i(2, 2), f(2)),
        lambda: ops.verify_drafts(f(2, 3, 4), i(2, 2), None, f(2, 2), f(3)),
        lambda: ops.verify_drafts(f(2, 3, 4), i(2, 2), None, f(2, 2), f(2), lengths=f(2)),
        lambda: ops.verify_drafts(f(2, 3), i(2, 2), None, f(2, 2), f(2)),
    ]
    for k, call in enumerate(bad):
        with pytest.raises(LightGBMError):
            call()
            pytest.fail(f"call {k} was not refused")
    other = ops.verify_drafts
    with pytest.raises(LightGBMError):
        other(f(2, 3, 4), i(2, 2), _put(place, np.ones((2, 2, 4))), f(2, 2), f(2))


@pytest.mark.gpu
def test_refuses_mixed_places():
    z, ids, t = np.ones((3, 4), np.float32), np.ones((3, 2), np.int32), np.ones((3, 2), np.float32)
    with pytest.raises(LightGBMError):
        ops.distill_loss(_put("gpu", z), (ids, t))
    with pytest.raises(LightGBMError):
        ops.distill_loss(_put("torch", z), (_put("gpu", ids), _put("torch", t)))


# ------------------------------------------------------------------ on the device
def _set(rows, classes, dtype, seed, order="C", drafts=2):
    """Inputs of one call of each operator, on the GPU."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    z = 3 * torch.randn((rows, classes), generator=g, device="cuda", dtype=torch.float64)
    z = z.to(TORCH[dtype])
    if order == "F":
        z = z.t().contiguous().t()
    p = torch.softmax(torch.randn((rows, drafts + 1, classes), generator=g, device="cuda"), 2)
    q = torch.softmax(torch.randn((rows, drafts, classes), generator=g, device="cuda"), 2)
    return {"z": z, "labels": torch.randint(0, classes, (rows,), generator=g, device="cuda"),
            "p": p, "q": q,
            "drafts": torch.randint(0, classes, (rows, drafts), generator=g, device="cuda"),
            "u": torch.rand((rows, drafts), generator=g, device="cuda"),
            "v": torch.rand((rows,), generator=g, device="cuda")}


def _run_set(s, k):
    """The operators one after the other, as a training and serving program calls them."""
    top = ops.top_logits(s["z"], k, temperature=2.0)
    got = ops.distill_gradients(s["z"] * 0.5, top, labels=s["labels"], temperature=2.0, alpha=0.5,
                                hessian=True, loss=True)
    loss = ops.distill_loss(s["z"] * 0.5, top, temperature=2.0)
    drawn = ops.verify_drafts(s["p"], s["drafts"], s["q"], s["u"], s["v"])
    return [*top, *got, loss, *drawn]


def _same(a, b):
    for x, y in zip(a, b):
        assert torch.equal(x, y)


DEVICE_SETS = [(5, 9, "f64", "F", 3), (70, 200, "f32", "F", 40), (6, 40, "bf16", "C", 7),
               (4, 3001, "f16", "C", 33), (2, 70001, "f32", "C", 20), (3, 3000, "f64", "C", 9),
               (600, 20011, "bf16", "C", 64), (600, 40001, "f32", "C", 9)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,classes,dtype,order,k", DEVICE_SETS)
def test_repeats_bit_for_bit(rows, classes, dtype, order, k):
    s = _set(rows, classes, dtype, 0, order)
    want = _run_set(s, k)
    for _ in range(5):
        _same(_run_set(s, k), want)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,classes,dtype,order,k", DEVICE_SETS)
def test_graphs(rows, classes, dtype, order, k):
    """Two graphs of the same calls, replayed in turn on new inputs with the program's own eager
    work between: every replay is the eager result."""
    graphs = []
    for seed in (1, 2):
        s = _set(rows, classes, dtype, seed, order)
        _run_set(s, k)  # the kernels are loaded before the capture
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _run_set(s, k)
        graphs.append((g, s, out))
    for turn in range(4):
        for g, s, out in graphs:
            new = _set(rows, classes, dtype, 10 + turn, order)
            for name, x in new.items():
                s[name].copy_(x)
            want = _run_set(new, k)
            g.replay()
            torch.cuda.synchronize()
            _same(out, want)
    for g, s, out in graphs:  # both on their way at once
        g.replay()
    torch.cuda.synchronize()
    _same(graphs[0][2], graphs[1][2])


@pytest.mark.gpu
@pytest.mark.parametrize("rows,classes,dtype,order,k", DEVICE_SETS)
def test_streams(rows, classes, dtype, order, k):
    """Calls on two streams at once, inputs made and results used on the call's own stream."""
    want = [_run_set(_set(rows, classes, dtype, seed, order), k) for seed in (1, 2)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [None, None]
    for turn in range(3):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                s = _set(rows, classes, dtype, i + 1, order)
                got[i] = [x.clone() for x in _run_set(s, k)]
    torch.cuda.synchronize()
    for i in range(2):
        _same(got[i], want[i])


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """The last rows of an array of more than 2^31 elements are what they are alone."""
    rows, classes = 66000, 32768
    z = torch.empty((rows, classes), dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda")
    g.manual_seed(0)
    z.normal_(generator=g)
    last = z[-3:].clone()
    top = ops.top_logits(z, 9)
    alone = ops.top_logits(last, 9)
    _same([x[-3:] for x in top[:2]], alone[:2])
    # few rows are shared among more threads than many, so sums have another order
    rel = _rel(classes, "f32")
    rest = _get(alone.log_rest)
    assert np.all(np.abs(_get(top.log_rest[-3:]) - rest) <= 2 * rel * (1 + np.abs(rest)))
    got = ops.distill_gradients(z, top, loss=True)
    loss, grad, _, size_l, size_g = _plain_distill(
        _get(last), _get(alone.classes), _get(alone.logits), _get(top.log_rest[-3:]), None, None,
        1.0, 1.0)
    assert np.all(np.abs(_get(got.loss[-3:]) - loss) <= 3 * rel * size_l +
                  HALF_STEP["f32"] * np.abs(loss))
    assert np.all(np.abs(_get(got.gradient[-3:]) - grad) <= 3 * rel * size_g +
                  (1 + rel) * HALF_STEP["bf16"] * np.abs(grad) + TINY["bf16"])
    del got, top
    turned = torch.empty((300, 7200000), dtype=torch.float32, device="cuda")
    turned.normal_(generator=g)
    end = turned.t()[-2:].contiguous().t().contiguous().t()  # class-major too
    _same([x[-2:] for x in ops.top_logits(turned.t(), 5)], ops.top_logits(end, 5))
    p = torch.softmax(z[-4:].float(), 1).view(2, 2, classes)
    wide = torch.zeros((33000, 2, classes), dtype=torch.float32, device="cuda")
    wide[-2:] = p
    wide[:-2, :, 3] = 1.0
    drafts = torch.zeros((33000, 1), dtype=torch.int64, device="cuda")
    u = torch.full((33000, 1), 0.5, device="cuda")
    v = torch.rand(33000, generator=g, device="cuda")
    got = ops.verify_drafts(wide, drafts, None, u, v)
    want = ops.verify_drafts(p, drafts[-2:], None, u[-2:], v[-2:])
    _same([x[-2:] for x in got], want)
    assert bool((got.classes[:-2, 0] == 3).all())


@pytest.mark.gpu
@pytest.mark.parametrize("rows,classes,dtype,k", [
    (1100, 2500, "f32", 30), (600, 9001, "bf16", 64), (520, 24001, "f32", 100),
    (520, 60001, "f32", 64), (520, 110003, "f16", 33)])
def test_many_rows_of_many_classes(rows, classes, dtype, k):
    """Shapes that only many rows take, some of whose rows are held against the plain forms."""
    rng = np.random.default_rng(classes)
    some = [0, 1, 255, 256, rows - 1]
    s = _set(rows, classes, dtype, 5)
    top = ops.top_logits(s["z"], k, temperature=2.0)
    z = _get(s["z"])[some]
    ids, logits, rest = _plain_top(z, k, 2.0)
    np.testing.assert_array_equal(_get(top.classes)[some], ids)
    np.testing.assert_array_equal(_get(top.logits)[some], logits)
    rel = _rel(classes, dtype)
    assert np.all(np.abs(_get(top.log_rest)[some] - rest) <= 2 * rel * (1 + np.abs(rest)))
    student = _put("gpu", _round(rng.permutation(z.T).T, dtype), dtype)
    student = student[torch.arange(rows, device="cuda") % len(some)]
    teacher = ops.TopLogits(*[x[some][torch.arange(rows) % len(some)] for x in top])
    labels = torch.arange(rows, device="cuda") % classes
    mix = {"labels": labels, "temperature": 2.0, "alpha": 0.5}
    here = list(range(len(some)))
    loss, grad, _, size_l, size_g = _plain_distill(
        _get(student)[here], _get(teacher.classes)[here], _get(teacher.logits)[here],
        _get(teacher.log_rest)[here].astype(float), _get(labels)[here], None, 2.0, 0.5)
    got = ops.distill_gradients(student, teacher, **mix)
    for x in (ops.distill_loss(student, teacher, **mix),
              ops.distill_gradients(student, teacher, loss=True, **mix).loss):
        assert np.all(np.abs(_get(x)[here] - loss) <= 3 * rel * size_l +
                      HALF_STEP["f32"] * np.abs(loss))
    assert np.all(np.abs(_get(got.gradient)[here] - grad) <= 3 * rel * size_g +
                  (1 + rel) * HALF_STEP[dtype] * np.abs(grad) + TINY[dtype])
    # the same row again and again has the same results
    again = _get(got.gradient)[len(some):2 * len(some)] - _get(got.gradient)[here]
    assert np.count_nonzero(again) <= 2 * len(some)  # but for the classes of the labels


@pytest.mark.gpu
def test_more_rows_than_a_launch_has():
    """Rows past a part's end are what they are alone, and so are the last of the part before."""
    rows = (1 << 21) + 5
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    for order, classes in (("C", 3), ("F", 2)):
        z = torch.randn((rows, classes), generator=g, device="cuda")
        z = z if order == "C" else z.t().contiguous().t()
        end = slice(rows - 9, rows)
        few = z[end].clone() if order == "C" else z[end].t().contiguous().t()
        top, alone = ops.top_logits(z, 1), ops.top_logits(few, 1)
        _same([x[end] for x in top], alone)
        labels = torch.randint(0, classes, (rows,), generator=g, device="cuda")
        got = ops.distill_gradients(z, top, labels=labels, alpha=0.5, hessian=True, loss=True)
        want = ops.distill_gradients(few, alone, labels=labels[end], alpha=0.5, hessian=True,
                                     loss=True)
        _same([x[end] for x in got], want)
    for rows, classes in (((1 << 21) + 5, 2), (32768 + 5, 300)):
        end = slice(rows - 9, rows)
        p = torch.rand((rows, 2, classes), generator=g, device="cuda")
        q = torch.rand((rows, 1, classes), generator=g, device="cuda")
        x = torch.randint(0, classes, (rows, 1), generator=g, device="cuda")
        u = torch.rand((rows, 1), generator=g, device="cuda")
        v = torch.rand((rows,), generator=g, device="cuda")
        got = ops.verify_drafts(p, x, q, u, v)
        want = ops.verify_drafts(p[end], x[end], q[end], u[end], v[end])
        _same([r[end] for r in got], want)


def _padded(shape, dtype, value):
    """A tensor inside a larger one of a single value, and the larger one."""
    big = torch.full([n + 6 for n in shape], value, dtype=dtype, device="cuda")
    return big[tuple(slice(3, 3 + n) for n in shape)], big


@pytest.mark.gpu
@pytest.mark.parametrize("rows,classes,dtype,order,k", DEVICE_SETS)
def test_nothing_else_is_written(rows, classes, dtype, order, k):
    """Through the C ABI, results into views of larger tensors: what is around them stays."""
    s = _set(rows, classes, dtype, 3, order)
    want = _run_set(s, k)
    wide = TORCH["f64" if dtype == "f64" else "f32"]
    out = TORCH["f32" if dtype == "f64" else dtype]
    made = [_padded((rows, k), torch.int32, -9), _padded((rows, k), TORCH[dtype], 7.0),
            _padded((rows,), wide, 7.0), _padded((rows, classes), out, 7.0),
            _padded((rows, classes), out, 7.0), _padded((rows,), wide, 7.0),
            _padded((rows, 3), torch.int32, -9), _padded((rows,), torch.int32, -9)]
    f = lambda x: ops._fields(x, "")  # noqa: E731
    view = [m[0] for m in made]
    stream = torch.cuda.current_stream().cuda_stream
    lib = ops._LIB
    ops._safe_call(lib.LGBM_TopLogits(ops._TOP.pack(
        rows, classes, k, 2.0, *f(s["z"]), *f(view[0]), *f(view[1]), *f(view[2])), 0, stream))
    student = s["z"] * 0.5
    ops._safe_call(lib.LGBM_Distill(ops._DISTILL.pack(
        rows, classes, k, 2.0, 0.5, *f(student), *f(view[0]), *f(view[1]), *f(view[2]),
        *f(s["labels"]), *ops._NONE, *f(view[5]), *f(view[3]), *f(view[4])), 0, stream))
    verify = (rows, classes, 2, *f(s["p"]), *f(s["q"]), *f(s["drafts"]), *f(s["u"]), *f(s["v"]),
              *ops._NONE, *f(view[6]), *f(view[7]))
    need = ops.ctypes.c_int64(0)
    ops._safe_call(lib.LGBM_VerifyDraftsWorkspace(ops._VERIFY.pack(*verify, 0, 0),
                                                  ops.ctypes.byref(need)))
    space = torch.full((need.value + 64,), 77, dtype=torch.uint8, device="cuda")
    if need.value:
        with pytest.raises(LightGBMError):
            ops._safe_call(lib.LGBM_VerifyDrafts(ops._VERIFY.pack(
                *verify, space.data_ptr(), need.value - 1), 0, stream))
        with pytest.raises(LightGBMError):
            ops._safe_call(lib.LGBM_VerifyDrafts(ops._VERIFY.pack(*verify, 0, need.value), 0,
                                                 stream))
    ops._safe_call(lib.LGBM_VerifyDrafts(ops._VERIFY.pack(*verify, space.data_ptr(), need.value),
                                         0, stream))
    torch.cuda.synchronize()
    assert bool((space[need.value:] == 77).all())
    order_of = [0, 1, 2, 3, 4, 5, 7, 8]
    for (got, big), w in zip(made, [want[i] for i in order_of]):
        # the C ABI's gradients are in row order here, whatever the scores' order is
        assert torch.equal(got, w)
        keep = big.flatten()[0].item()
        big[tuple(slice(3, 3 + n) for n in got.shape)] = keep
        assert bool((big == keep).all())


@pytest.mark.gpu
def test_torch_first():
    """This process has loaded lightgbm_amd first; the other order of import serves too."""
    code = ("import torch, numpy as np; x = torch.randn(4, 300, device='cuda')\n"
            "import lightgbm_amd as lgb\n"
            "t = lgb.ops.top_logits(x, 3); assert torch.equal(t.logits, x.topk(3)[0])\n"
            "X = np.random.RandomState(0).randn(500, 4)\n"
            "b = lgb.train({'objective': 'regression', 'device_type': 'gpu', 'verbosity': -1},"
            " lgb.Dataset(X, label=X[:, 0]), 2)\n"
            "assert b.num_trees() == 2; print('both')")
    root = Path(__file__).resolve().parent.parent
    got = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True,
                         timeout=100)
    assert got.returncode == 0 and "both" in got.stdout, got.stderr[-2000:]


def test_lgb_exports_ops():
    assert lgb.ops is ops


# ------------------------------------------------------------------ lists
def test_lists_are_their_arrays():
    """Every argument may be a list; the array made of it lives until the call has returned.
    Large enough that memory freed before would be used again."""
    rng = np.random.default_rng(21)
    rows, classes, k = 5000, 10, 3
    z = rng.standard_normal((rows, classes))
    ids, logits, rest = _teacher(rng, rows, classes, k, True)
    args = [ids, logits.astype(float), rest.astype(float), rng.integers(0, classes, rows),
            0.5 + rng.random(rows)]

    def distill(turn):
        c, t, r, y, w = map(turn, args)
        got = ops.distill_gradients(turn(z), (c, t, r), labels=y, weight=w, alpha=0.5, loss=True,
                                    hessian=True)
        return [*got, ops.distill_loss(turn(z), (c, t, r), labels=y, weight=w, alpha=0.5)]

    p = _softmax(rng.standard_normal((rows, 3, classes)))
    q = _softmax(rng.standard_normal((rows, 2, classes)))
    drafts = rng.integers(0, classes, (rows, 2))
    u, v, lengths = rng.random((rows, 2)), rng.random(rows), rng.integers(0, 3, rows)
    for call in (distill, lambda turn: ops.top_logits(turn(z), k),
                 lambda turn: ops.verify_drafts(*map(turn, (p, drafts, q, u, v)),
                                                lengths=turn(lengths))):
        for got, want in zip(call(lambda x: x.tolist()), call(lambda x: x)):
            np.testing.assert_array_equal(got, want)


@pytest.mark.parametrize("place", PLACES[1:])
def test_views_that_negate(place):
    """The imaginary part of a conjugate is a real tensor whose memory holds the other sign."""
    rng = np.random.default_rng(22)

    def turned(x):
        x = _put(place, -np.asarray(x), "f32")
        x = torch.complex(torch.zeros_like(x), x).conj().imag
        assert x.is_neg()
        return x

    z = rng.standard_normal((6, 9)).astype(np.float32)
    ids, logits, rest = _teacher(rng, 6, 9, 3, True)
    weight = np.float32(0.5 + rng.random(6))
    results = []
    for f in (turned, lambda x: _put(place, x, "f32")):
        teacher = (_put(place, ids, "i32"), f(logits), f(rest))
        results.append([*ops.top_logits(f(z), 3),
                        *ops.distill_gradients(f(z), teacher, weight=f(weight), loss=True,
                                               hessian=True),
                        ops.distill_loss(f(z), teacher, weight=f(weight))])
        p = np.float32(_softmax(rng.standard_normal((6, 3, 9)))) if not results[1:] else p
        u, v = (np.full((6, 2), 0.5), np.full(6, 0.5))
        results[-1] += [*ops.verify_drafts(f(p), _put(place, ids[:, :2], "i32"),
                                           f(p[:, ::-1][:, :2]), f(u), f(v))]
        ds = lgb.Dataset(np.zeros((6, 1)), params={"min_data_in_bin": 1, "verbosity": -1},
                         teacher=teacher).construct().get_teacher()
        results[-1] += [torch.from_numpy(x) for x in ds]
    _same(*results)


@pytest.mark.parametrize("place", PLACES)
def test_refuses_what_is_no_number(place):
    """Whole numbers and numbers of other kinds than an argument's, and ones of no size."""
    f = lambda *shape: _put(place, np.ones(shape, np.float32))  # noqa: E731
    teacher = (_put(place, np.ones((3, 2), np.int32)), f(3, 2))
    for k in (2.9, 2.0, "2", None, 10 ** 12, -1):
        with pytest.raises(LightGBMError):
            ops.top_logits(f(3, 4), k)
    for bad in (None, "1", 1j, [1.0]):
        with pytest.raises(LightGBMError):
            ops.top_logits(f(3, 4), 1, temperature=bad)
        with pytest.raises(LightGBMError):
            ops.distill_loss(f(3, 4), teacher, temperature=bad)
        with pytest.raises(LightGBMError):
            ops.distill_gradients(f(3, 4), teacher, labels=teacher[0][:, 0], alpha=bad)
    got = ops.top_logits(f(3, 4), np.int64(2), temperature=np.float32(1.5))
    assert tuple(got.classes.shape) == (3, 2)


@pytest.mark.parametrize("place", PLACES[1:])
def test_refuses_to_lose_gradients(place):
    """Of each argument in turn, where gradients are recorded, and nowhere else."""
    rng = np.random.default_rng(23)
    p = np.float32(_softmax(rng.standard_normal((6, 3, 9))))
    f32 = lambda x: _put(place, x, "f32")  # noqa: E731
    ids = _put(place, rng.integers(0, 9, (6, 2)), "i32")
    top = (f32(p[:, 0]),)
    distill = (f32(p[:, 0]), f32(p[:, 0, :2]), f32(p[:, 0, 0]), f32(p[:, 0, 0]))
    verify = (f32(p), f32(p[:, :2]), f32(p[:, 0, :2]), f32(p[:, 0, 0]))
    calls = [(lambda z: ops.top_logits(z, 3), top),
             (lambda z, t, r, w: ops.distill_loss(z, (ids, t, r), weight=w), distill),
             (lambda z, t, r, w: ops.distill_gradients(z, (ids, t, r), weight=w, hessian=True),
              distill),
             (lambda p, q, u, v: ops.verify_drafts(p, ids, q, u, v), verify)]
    forward = torch.autograd.forward_ad
    for call, args in calls:
        want = call(*args)
        want = [want] if torch.is_tensor(want) else [x for x in want if x is not None]
        for i in range(len(args)):
            asking = [x.clone().requires_grad_(i == j) for j, x in enumerate(args)]
            with pytest.raises(LightGBMError):
                call(*asking)
            for quiet in (torch.no_grad, torch.inference_mode):
                with quiet():
                    got = call(*asking)
                _same([got] if torch.is_tensor(got) else [x for x in got if x is not None], want)
            with forward.dual_level():
                dual = [forward.make_dual(x, x) if i == j else x for j, x in enumerate(args)]
                with pytest.raises(LightGBMError):
                    call(*dual)
                call(*args)


@pytest.mark.parametrize("place", PLACES)
@pytest.mark.parametrize("classes", [6, 150, 5000])
def test_distill_teacher_of_no_number(place, classes):
    """NaN or +inf among a teacher's logits, or as its rest, makes NaN of all that its row wants:
    of the slots, and of the other classes where it speaks of them. Other rows keep theirs."""
    rng = np.random.default_rng(24)
    z = rng.standard_normal((5, classes))
    ids = np.tile([1, 0, 2], (5, 1))
    logits = np.tile(np.float32([3, 2, 1]), (5, 1))
    rest = np.full(5, 0.5, np.float32)
    clean = logits.copy(), rest.copy()
    logits[0, 1], logits[1, 0], rest[2], rest[3] = np.nan, INF, np.nan, INF
    labels = np.full(5, 4)
    for dtype in _types(place):
        for order in "CF":
            for alpha in (1.0, 0.5):
                for with_rest in (True, False):
                    def call(t, r):
                        got = ops.distill_gradients(
                            _put(place, z, dtype, order),
                            (_put(place, ids, "i32"), _put(place, t, "f32"),
                             _put(place, r, "f32") if with_rest else None),
                            labels=_put(place, labels, "i32"), alpha=alpha, loss=True)
                        return _get(got.gradient), _get(got.loss)
                    grad, loss = call(logits, rest)
                    want, want_loss = call(*clean)
                    bad = 4 if with_rest else 2
                    assert np.all(np.isnan(loss[:bad])) and np.all(np.isnan(grad[:bad, :3]))
                    if with_rest:
                        assert np.all(np.isnan(grad[:bad]))
                    else:
                        np.testing.assert_array_equal(grad[:bad, 3:], want[:bad, 3:])
                    np.testing.assert_array_equal(grad[bad:], want[bad:])
                    np.testing.assert_array_equal(loss[bad:], want_loss[bad:])


def test_refuses_tensors_without_memory():
    """A weight that holds no values is not a weight that is absent."""
    z, ids, t = torch.ones(3, 4), torch.ones((3, 2), dtype=torch.int32), torch.ones(3, 2)
    with pytest.raises(LightGBMError):
        ops.distill_loss(z, (ids, t), weight=torch.ones(3, device="meta"))
    with pytest.raises(LightGBMError):
        ops.top_logits(z.to("meta"), 1)


# ------------------------------------------------------------------ scores of any size
# The device's exponents are (z - high) * s: the difference, s and the product are rounded, so a
# term 2^-x is off by (3 x + 4) eps of itself, and by less than 8 eps of the row's largest: `_rel`
# covers that, being applied three times over. How large z itself is does not come in.
def _plain_gradient(z, classes, logits, rest, labels, t, alpha):
    """Gradient, hessian and their scale in 64 bits, for scores so far apart that even there a
    logarithm of a sum keeps nothing of the sum: every softmax is taken against a maximum of its
    own, of differences."""
    def softmax(x):
        e = np.exp(x - x.max())
        return e / e.sum()

    n, c = z.shape
    grad, hess, size = np.zeros((n, c)), np.zeros((n, c)), np.zeros((n, c))
    for i in range(n):
        with np.errstate(over="ignore"):
            q, q1 = softmax((z[i] - z[i].max()) / t), softmax(z[i] - z[i].max())
        slot = {}
        for j, x in enumerate(classes[i]):
            if 0 <= x < c:
                slot.setdefault(int(x), logits[i, j] / t)
        p = softmax(np.array([*slot.values(), -INF if rest is None else rest[i]]))
        want = np.zeros(c)
        others = np.ones(c, bool)
        others[list(slot)] = False
        if p[-1] > 0:
            own = z[i][others]
            with np.errstate(over="ignore"):
                want[others] = p[-1] * softmax((own - own.max()) / t)
        want[list(slot)] = p[:-1]
        grad[i] = alpha * t * (q - want)
        hess[i] = alpha * q * (1 - q)
        size[i] = alpha * t * (q + want)
        if alpha < 1:
            hit = np.arange(c) == labels[i]
            grad[i] += (1 - alpha) * (q1 - hit)
            hess[i] += (1 - alpha) * q1 * (1 - q1)
            size[i] += (1 - alpha) * (q1 + hit)
    return grad, hess * (c / (c - 1)), size


def _gradient_case(place, z, teacher, dtype, labels=None, t=1.0, alpha=1.0, order="C", rel=None,
                   rows=None):
    """Gradient and hessian of the rows (all of them, or the first few)."""
    z = _round(z, dtype)
    ids, logits, rest = teacher
    many = slice(None) if rows is None else np.arange(rows) % len(z)
    pick = lambda x: None if x is None else x[many]  # noqa: E731
    got = ops.distill_gradients(
        _put(place, pick(z), dtype, order),
        (_put(place, pick(ids), "i32"), _put(place, pick(logits), "f32"),
         _put(place, pick(rest), "f32")),
        labels=_put(place, pick(labels), "i32"), temperature=t, alpha=alpha, hessian=True)
    grad, hess, size = _plain_gradient(z, ids, logits.astype(np.float64),
                                       None if rest is None else rest.astype(np.float64),
                                       labels, t, alpha)
    out = "f32" if dtype == "f64" else dtype
    rel = rel or 3 * _rel(z.shape[1], "f32")
    for a, b, far in ((got.gradient, grad, rel * size),
                      (got.hessian, hess, 2 * rel * size / min(t, 1.0))):
        a = _get(a[:len(z)])
        far = far + (1 + rel) * HALF_STEP[out] * np.abs(b) + TINY[out] * max(t, 1.0)
        assert np.all(np.abs(a - b) <= far), np.nanmax(np.abs(a - b) - far)


@pytest.mark.parametrize("place", PLACES)
@pytest.mark.parametrize("classes", [6, 40, 150, 600, 5000, 90001, 200003])
def test_distill_masked_by_the_lowest(place, classes):
    """Masks of the type's lowest value: whole rows, which are uniform, all unnamed classes, with a
    rest that wants something of them and without, and half of a row; rows of the highest value."""
    rng = np.random.default_rng(classes)
    ids = np.tile([1, 0, 2], (7, 1))
    logits = np.tile(np.float32([3, 2, 1]), (7, 1))
    rest = np.full(7, 0.5, np.float32)
    rest[3] = -INF
    labels = np.array([4, 4, 1, 4, 0, 4, 4])
    for dtype in _types(place):
        low = torch.finfo(TORCH[dtype]).min
        z = rng.standard_normal((7, classes))
        z[0] = low
        z[1, 3:] = z[2, 3:] = z[3, 3:] = low
        z[4, 1::2] = low
        z[5] = -low
        z[6] = low
        z[6, 0] = 1.0
        for order in "CF" if classes < 20000 else "C":
            for t in (1.0, 0.5):
                _gradient_case(place, z, (ids, logits, rest), dtype, t=t, order=order)
                _gradient_case(place, z, (ids, logits, rest), dtype, labels=labels, t=t, alpha=0.5,
                               order=order)


@pytest.mark.parametrize("place", PLACES)
@pytest.mark.parametrize("classes", [6, 150, 600, 5000, 90001])
def test_distill_of_small_temperature(place, classes):
    """Large scores over a small temperature: every row has a largest score, so all are live."""
    rng = np.random.default_rng(classes)
    ids = np.tile([1, 0, 2], (4, 1))
    logits = np.tile(np.float32([3e-6, 2e-6, 1e-6]), (4, 1))
    rest = np.full(4, 2.5, np.float32)
    labels = np.array([4, 1, 0, 4])
    for dtype in _types(place):
        z = rng.standard_normal((4, classes))
        z[0] += 60000.0
        z[1] -= 60000.0
        z[2] = 50000.0
        for order in "CF" if classes < 20000 else "C":
            for alpha in (1.0, 0.5):
                _gradient_case(place, z, (ids, logits, rest), dtype, labels=labels, t=1e-6,
                               alpha=alpha, order=order)


@pytest.mark.parametrize("place", PLACES)
@pytest.mark.parametrize("classes,dtype", [(131077, "f32"), (200003, "f32"), (200003, "f16"),
                                           (200003, "bf16")])
@pytest.mark.parametrize("offset", [0.0, -1000.0, 50000.0])
def test_distill_large_rows_with_an_offset(place, classes, dtype, offset):
    """Rows of which a part is read again: what is held and what is not have sums of their own. A
    term that matters, 2^-x with x below 64, is off by (3 * 64 + 4) eps, a sum of a thread's 200
    terms in chunks and the tree by 64 more; a quotient has two of them."""
    if place != "gpu" and classes > 100000:
        pytest.skip("of the device's shapes; the host has one way")
    rng = np.random.default_rng(classes)
    teacher = _teacher(rng, 3, classes, 20, True)
    z = 3 * rng.standard_normal((3, classes)) + offset
    labels = rng.integers(0, classes, 3)
    for t, alpha in ((1.0, 1.0), (2.0, 0.5)):
        _gradient_case(place, z, teacher, dtype, labels=labels, t=t, alpha=alpha,
                       rel=2 * 260 * HALF_STEP["f32"])
    if place == "gpu":  # as many rows as share a compute unit, where they are only read
        z = _round(z, dtype)
        loss, _, _, size, _ = _plain_distill(z, teacher[0], teacher[1].astype(float),
                                             teacher[2].astype(float), None, None, 1.0, 1.0)
        many = torch.arange(600) % 3
        got = ops.distill_loss(_put("gpu", z, dtype)[many], ops.TopLogits(
            *[_put("gpu", x)[many] for x in (teacher[0].astype(np.int32), *teacher[1:])]))
        far = 2 * 260 * HALF_STEP["f32"] * size + HALF_STEP["f32"] * np.abs(loss)
        assert np.all(np.abs(_get(got)[:3] - loss) <= far)


@pytest.mark.parametrize("place", PLACES)
@pytest.mark.parametrize("classes", [6, 40, 150, 600, 5000])
@pytest.mark.parametrize("offset", [-1e3, 1e4, -1e5])
def test_distill_teacher_with_an_offset(place, classes, offset):
    """What all logits and the rest have in common changes nothing, and neither does its size. The
    exponents are formed in 64 bits, where an offset of 1e5 over T leaves 1e-10."""
    rng = np.random.default_rng(classes)
    ids, logits, rest = _teacher(rng, 4, classes, 5, True)
    logits = (logits + offset).astype(np.float32)
    labels = rng.integers(0, classes, 4)
    for t in (1.0, 0.75):
        r = (rest + offset / t).astype(np.float32)
        for dtype in _types(place):
            z = 3 * rng.standard_normal((4, classes))
            for order in "CF":
                for far in (r, None):
                    _gradient_case(place, z, (ids, logits, far), dtype, labels=labels, t=t,
                                   alpha=0.5, order=order)


@pytest.mark.parametrize("place", PLACES)
@pytest.mark.parametrize("classes", [6, 150, 5000])
def test_distill_teacher_of_the_lowest_value(place, classes):
    """Slots of the type's lowest logit are alike, and nothing beside a rest or a better slot."""
    rng = np.random.default_rng(classes)
    ids = np.tile([1, 0, 2], (3, 1))
    low = torch.finfo(torch.float32).min
    logits = np.tile(np.float32([low, low, low]), (3, 1))
    logits[1, 2] = 5.0
    z = rng.standard_normal((3, classes))
    labels = np.full(3, 3)
    for t in (1.0, 0.5):
        for rest in (None, np.float32([0.5, 0.5, -INF])):
            for order in "CF":
                for dtype in _types(place):
                    _gradient_case(place, z, (ids, logits, rest), dtype, labels=labels, t=t,
                                   alpha=0.5, order=order)


@pytest.mark.parametrize("place", PLACES)
@pytest.mark.parametrize("classes", [6, 150, 5000])
def test_distill_teacher_in_64_bits(place, classes):
    """Logits that 32 bits would round: what a float64 teacher says is read as it is, beside scores
    of any type."""
    rng = np.random.default_rng(classes)
    ids, logits, rest = _teacher(rng, 4, classes, 5, True)
    logits = logits.astype(np.float64) / 3 + 1e6
    rest = rest.astype(np.float64) / 3 + 1e6
    for dtype in _types(place):
        z = _round(rng.standard_normal((4, classes)), dtype)
        for order in "CF":
            got = _get(ops.distill_gradients(_put(place, z, dtype, order),
                                             (_put(place, ids, "i32"), _put(place, logits, "f64"),
                                              _put(place, rest, "f64"))).gradient)
            want, _, size = _plain_gradient(z, ids, logits, rest, None, 1.0, 1.0)
            out = HALF_STEP["f32" if dtype == "f64" else dtype]
            far = 3 * _rel(classes, "f32") * size + 2 * out * np.abs(want)
            assert np.all(np.abs(got - want) <= far + TINY["f32" if dtype == "f64" else dtype])


def _plain_loss(z, classes, logits, rest, labels, t, alpha):
    """The loss in 64 bits from differences, for scores of any size."""
    loss = np.zeros(len(z))
    for i, x in enumerate(z):
        with np.errstate(over="ignore"):
            d = (x - x.max()) / t
        log_all = math.log(np.exp(d).sum())
        names = [int(j) for j in classes[i]]
        p = np.array([*(logits[i] / t), rest[i]])
        log_p = p - _lse(p)
        others = np.ones(len(x), bool)
        others[names] = False
        own = x[others].max()
        with np.errstate(over="ignore"):
            left = math.log(np.exp((x[others] - own) / t).sum()) + (own - x.max()) / t
        log_q = np.array([*d[names], left]) - log_all
        loss[i] = alpha * t * t * (np.exp(log_p) * (log_p - log_q)).sum()
        if alpha < 1:
            loss[i] += (1 - alpha) * (math.log(np.exp(x - x.max()).sum()) - (
                x[labels[i]] - x.max()))
    return loss


@pytest.mark.parametrize("place", PLACES)
@pytest.mark.parametrize("classes", [6, 40, 150, 600, 5000, 90001])
def test_distill_loss_of_the_lowest(place, classes):
    """Where the student masks with the type's lowest value what the teacher or the label wants, the
    loss is large and finite. It has one term of that size, off by what the probability and the
    logarithms beside it are."""
    rng = np.random.default_rng(classes)
    ids = np.tile([1, 0, 2], (4, 1))
    logits = np.tile(np.float32([3, 2, 1]), (4, 1))
    rest = np.full(4, 0.5, np.float32)
    labels = np.array([4, 4, 4, 0])
    for dtype in _types(place):
        z = rng.standard_normal((4, classes))
        low = torch.finfo(TORCH[dtype]).min
        z[0] = low
        z[1, 3:] = low     # the rest
        z[2, 2] = low      # a slot
        z[3, 4] = z[3, 0] = low
        z = _round(z, dtype)
        for order in "CF" if classes < 20000 else "C":
            for t, alpha in ((1.0, 1.0), (1.0, 0.5), (2.0, 0.75)):
                got = _get(ops.distill_loss(
                    _put(place, z, dtype, order),
                    (_put(place, ids, "i32"), _put(place, logits, "f32"), _put(place, rest, "f32")),
                    labels=_put(place, labels, "i32"), temperature=t, alpha=alpha))
                want = _plain_loss(z, ids, logits.astype(float), rest.astype(float), labels, t,
                                   alpha)
                far = 3 * _rel(classes, dtype) * (20 * t * t + np.abs(want))
                assert np.all(np.abs(got - want) <= far), (got, want)


@pytest.mark.parametrize("place", PLACES)
@pytest.mark.parametrize("classes", [8, 100, 400, 600, 1000, 5000, 90001, 200003])
def test_top_logits_masked_by_the_lowest(place, classes):
    """Masks of the type's lowest value are scores: they are chosen after all others, and what is
    not chosen of them has a logarithm of their size. Exactly k others, fewer, none, one more."""
    if place != "gpu" and classes > 50000:
        pytest.skip("of the device's shapes; the host has one way")
    rng = np.random.default_rng(classes)
    k = 5
    for dtype in _types(place):
        low = torch.finfo(TORCH[dtype]).min
        x = np.full((5, classes), low)
        for i, many in enumerate((k, k - 2, 0, k + 1, classes // 2)):
            x[i, rng.permutation(classes)[:many]] = rng.standard_normal(many)
        for order in "CF" if classes < 20000 else "C":
            _top_case(place, x, dtype, k, order=order)
            _top_case(place, x, dtype, k, t=2.0, order=order)


@pytest.mark.parametrize("place", PLACES)
@pytest.mark.parametrize("classes", [8, 100, 400, 600, 5000, 90001])
def test_top_logits_of_small_temperature(place, classes):
    """Large scores over a small temperature, and scores with a large offset: the rest's logarithm
    is that of a size, with the same few roundings."""
    if place != "gpu" and classes > 50000:
        pytest.skip("of the device's shapes; the host has one way")
    rng = np.random.default_rng(classes)
    for dtype in _types(place):
        x = rng.standard_normal((3, classes))
        x[0] += 60000.0
        x[1] -= 60000.0
        for order in "CF" if classes < 20000 else "C":
            for t in (1e-6, 0.01, 1.0):
                _top_case(place, x, dtype, 3, t=t, order=order)


@pytest.mark.parametrize("place", PLACES)
@pytest.mark.parametrize("classes", [6, 40, 150, 600, 5000])
@pytest.mark.parametrize("less", [1e-3, 1e-6, 1e-12])
def test_distill_alpha_next_to_one(place, classes, less):
    """The labels' weight is what alpha leaves, however little: of rows without a teacher it is all
    there is, and relative to it the errors are those of any softmax."""
    rng = np.random.default_rng(classes)
    alpha = 1.0 - less
    ids = np.full((4, 2), -1)
    logits = np.zeros((4, 2), np.float32)
    labels = rng.integers(0, classes, 4)
    for dtype in _types(place):
        z = _round(rng.standard_normal((4, classes)), dtype)
        for order in "CF":
            got = ops.distill_gradients(
                _put(place, z, dtype, order), (_put(place, ids, "i32"), _put(place, logits, "f32")),
                labels=_put(place, labels, "i32"), alpha=alpha, loss=True)
            q = _softmax(z)
            hit = np.arange(classes) == labels[:, None]
            want, size = (1.0 - alpha) * (q - hit), (1.0 - alpha) * (q + hit)
            out = "f32" if dtype == "f64" else dtype
            far = 3 * _rel(classes, "f32") * size + 2 * HALF_STEP[out] * np.abs(want) + TINY[out]
            assert np.all(np.abs(_get(got.gradient) - want) <= far)
            loss = (1.0 - alpha) * -np.log(q[hit])
            assert np.all(np.abs(_get(got.loss) - loss) <= 3 * _rel(classes, dtype) * (
                (1.0 - alpha) * (2 + np.abs(np.log(q[hit])))) + HALF_STEP["f32"] * loss)


# ------------------------------------------------------------------ rows that registers do not hold
# 81920 float32 or 163840 16-bit classes stand in a workgroup of 1024 threads, half of them in one
# of 512; what is beyond is read again in each pass.
LARGE = [(90001, "f32"), (200003, "f32"), (200003, "f16"), (200003, "bf16")]


@pytest.mark.parametrize("place", PLACES)
@pytest.mark.parametrize("classes,dtype", LARGE)
def test_distill_large_rows_masked(place, classes, dtype):
    """Masks, NaN and infinities, a rest that underflows, in what is held and what is read again."""
    if place != "gpu" and classes > 100000:
        pytest.skip("of the device's shapes; the host has one way")
    rng = np.random.default_rng(classes)
    rows = 10
    ids, logits, rest = _teacher(rng, rows, classes, 9, True)
    labels = rng.integers(0, classes, rows)
    z = 2 * rng.standard_normal((rows, classes))
    z[0, rng.random(classes) < 0.3] = -INF
    z[1, :classes - 100] = -INF            # only the end is there
    z[2, 100:] = -INF                      # only the beginning
    z[3] = -INF
    z[4, classes // 2:] = -INF
    np.put_along_axis(z, ids, 1.0, axis=1)
    z[3] = -INF
    z[np.arange(rows), labels] = np.where(np.arange(rows) == 3, -INF, 1.0)
    z[5], z[6] = z[5] - 300.0, z[6] - 300.0
    z[5, ids[5, 0]] = 0.0                  # the others underflow
    z[6, ids[6, 0]] = 100.0
    z[7, classes - 1] = np.nan
    z[8, classes - 2] = INF
    z[9, 3] = np.nan
    labels[7:] = -1
    clean = np.arange(rows) < 7
    for t, alpha in ((1.0, 1.0), (2.0, 0.5)):
        teacher = ids, logits, rest
        _distill_case(place, z[clean], tuple(x[clean] for x in teacher), dtype,
                      labels=labels[clean], t=t, alpha=alpha)
        got = ops.distill_gradients(_put(place, z, dtype), (
            _put(place, ids, "i32"), _put(place, logits, "f32"), _put(place, rest, "f32")),
            labels=_put(place, labels, "i32"), temperature=t, alpha=alpha, loss=True, hessian=True)
        bad = np.isnan(_get(got.loss))
        np.testing.assert_array_equal(bad, ~clean)
        for x in (_get(got.gradient), _get(got.hessian)):
            assert np.all(np.isnan(x[7:])) and np.all(np.isfinite(x[:7]))


@pytest.mark.parametrize("place", PLACES)
@pytest.mark.parametrize("classes,dtype", LARGE)
def test_top_logits_large_rows(place, classes, dtype):
    """Ties, masks and NaN, scores that stand out at the row's ends, and a rest that underflows."""
    if place != "gpu" and classes > 100000:
        pytest.skip("of the device's shapes; the host has one way")
    rng = np.random.default_rng(classes)
    x = rng.standard_normal((9, classes))
    x[0] = 1.5
    x[1] = rng.integers(0, 3, classes)
    x[2, :classes - 30] = -INF
    x[3, 30:] = np.nan
    x[4, rng.random(classes) < 0.5] = -INF
    x[5] = np.arange(classes) // 4096
    x[6, -3:], x[6, :3] = 200.0, 200.0
    x[7, classes - 5] = INF
    x[8] = np.where(np.arange(classes) % 2, 0.0, -0.0)
    for k in (1, 40, 256):
        _top_case(place, x, dtype, k)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,classes,dtype", [
    (1100, 2500, "f32"), (1100, 7001, "f32"), (600, 9001, "bf16"), (600, 20011, "f16"),
    (520, 24001, "f32"), (520, 60001, "f16"), (600, 3000, "bf16")])
def test_hessians_of_many_rows(rows, classes, dtype):
    """The shapes that only many rows take, against the plain form."""
    rng = np.random.default_rng(classes)
    teacher = _teacher(rng, 3, classes, 20, True)
    z = 3 * rng.standard_normal((3, classes))
    labels = rng.integers(0, classes, 3)
    for t, alpha in ((2.0, 0.5), (1.0, 1.0)):
        _gradient_case("gpu", z, teacher, dtype, labels=labels, t=t, alpha=alpha, rows=rows)


@pytest.mark.parametrize("call", [
    "ops.top_logits(z, 1)",
    "ops.distill_loss(z, (ids, f(64, 1)))",
    "ops.verify_drafts(f(64, 2, 1 << 20), ids, None, f(64, 1), f(64))"])
def test_host_memory_that_is_not_there(call):
    """Scratch of a call that does not fit is a LightGBMError, not the end of the process."""
    code = (
        "import resource, numpy as np, lightgbm_amd as lgb\n"
        "from lightgbm_amd import ops\n"
        "f = lambda *s: np.broadcast_to(np.float32(0.5), s)\n"
        "ids, z = np.zeros((64, 1), np.int32), f(64, 1 << 20)\n"
        "ops.distill_loss(f(64, 4), (ids, f(64, 1)))  # the threads are there\n"
        "size = int(open('/proc/self/statm').read().split()[0]) * 4096\n"
        "resource.setrlimit(resource.RLIMIT_AS, (size + (6 << 20),) * 2)\n"
        f"try:\n    {call}\nexcept lgb.LightGBMError:\n    print('refused')\n")
    root = Path(__file__).resolve().parent.parent
    got = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True,
                         timeout=100)
    assert got.returncode == 0 and "refused" in got.stdout, got.stderr[-2000:]


def test_first_calls_at_once(monkeypatch):
    """A call of another thread, while the first one looks torch up, finds all of it or looks it up
    itself."""
    z = torch.arange(6.0).reshape(2, 3)
    want = ops.top_logits(z, 2)

    class Types(dict):
        def __setitem__(self, key, value):
            super().__setitem__(key, value)
            if not seen:
                seen.append(0)
                _same(ops.top_logits(z, 2), want)

    seen = []
    for name, value in (("_torch", None), ("_Tensor", ()), ("_raw_stream", None),
                        ("_forward", None), ("_TORCH_TYPES", Types()), ("_TORCH_OF", {})):
        monkeypatch.setattr(ops, name, value)
    _same(ops.top_logits(z, 2), want)
    assert seen


# ------------------------------------------------------------------ the largest sizes
MOST = 1 << 20


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f64", "f32", "f16", "bf16"])
@pytest.mark.parametrize("step", [1, 2])
def test_most_classes(dtype, step):
    """2^20 classes, next to each other and every second one; one row and as many as share units."""
    rng = np.random.default_rng(MOST + step)
    z = _round(3 * rng.standard_normal((2, MOST)), dtype)
    wide = torch.zeros((2, MOST * step), dtype=TORCH[dtype], device="cuda")
    x = wide[:, ::step]
    x.copy_(_put("gpu", z, dtype))
    for rows in (1, 2):
        got = ops.top_logits(x[:rows], 100, temperature=2.0)
        classes, logits, rest = _plain_top(z[:rows], 100, 2.0)
        np.testing.assert_array_equal(_get(got.classes), classes)
        np.testing.assert_array_equal(_get(got.logits), logits)
        assert np.all(np.abs(_get(got.log_rest) - rest) <=
                      _rel(MOST, dtype) * (1 + np.abs(rest)))
    ids, logits, rest = _teacher(rng, 2, MOST, 256, True)
    ids[1, 0] = MOST - 1
    labels = np.array([MOST - 1, 0])
    mix = {"labels": _put("gpu", labels, "i32"), "temperature": 2.0, "alpha": 0.5}
    got = ops.distill_gradients(x, (_put("gpu", ids, "i32"), _put("gpu", logits, "f32"),
                                    _put("gpu", rest, "f32")), hessian=True, loss=True, **mix)
    grad, hess, size = _plain_gradient(z, ids, logits.astype(float), rest.astype(float), labels,
                                       2.0, 0.5)
    loss = _plain_loss(z, ids, logits.astype(float), rest.astype(float), labels, 2.0, 0.5)
    out = "f32" if dtype == "f64" else dtype
    rel = 3 * _rel(MOST, "f32")
    for a, b in ((got.gradient, grad), (got.hessian, hess)):
        far = 2 * rel * size + (1 + rel) * HALF_STEP[out] * np.abs(b) + TINY[out]
        assert np.all(np.abs(_get(a) - b) <= far)
    assert np.all(np.abs(_get(got.loss) - loss) <= 3 * _rel(MOST, dtype) * (20 + loss))
    p = torch.softmax(x.double(), 1)[None]
    drafts = torch.tensor([[MOST - 1]], device="cuda")
    p[0, 0, MOST - 1] = 0.25
    p = p.to(TORCH[dtype])
    u, v = torch.zeros((1, 1), device="cuda"), torch.full((1,), 0.999, device="cuda")
    for accept in (u, u + 0.999):
        got = ops.verify_drafts(p, drafts, None, accept, v)
        classes, accepted = _plain_verify(_get(p), _get(drafts), None, _get(accept), _get(v), None)
        np.testing.assert_array_equal(_get(got.accepted), accepted)
        # next to a border the order of the sums decides: the class's own sum is the check
        mass = np.where(np.arange(MOST) == (MOST - 1 if not accepted[0] else -1), 0.0,
                        _get(p)[0, accepted[0]])
        reach, at = np.cumsum(mass), int(_get(got.classes)[0, accepted[0]])
        goal, slack = float(_get(v)[0]) * reach[-1], MOST * HALF_STEP["f64"] * reach[-1]
        assert mass[at] > 0 and reach[at] > goal - slack and reach[at] - mass[at] <= goal + slack


@pytest.mark.parametrize("place", PLACES)
@pytest.mark.parametrize("classes", [3, 64, 300, 2500])
def test_most_drafts(place, classes):
    """1024 drafts a sequence, refused nowhere, at the end, in the middle, at once."""
    rng = np.random.default_rng(classes)
    p = _softmax(rng.standard_normal((4, 1025, classes)))
    drafts = p[:, :-1].argmax(-1)
    u = np.zeros((4, 1024))
    u[1, 1023] = u[2, 500] = u[3, 0] = 2.0
    v = rng.random(4)
    _verify_case(place, p, drafts, None, u, v, None, "f32")
    _verify_case(place, p, drafts, p[:, :-1], u, v, np.array([1024, 1024, 700, 5]), "f64", "i64")


@pytest.mark.parametrize("place", ["numpy", "torch"])
def test_more_than_the_most_is_refused(place):
    wide = np.broadcast_to(np.float32(1.0), (1, MOST + 1))
    z = wide if place == "numpy" else torch.ones(1, 1).expand(1, MOST + 1)
    teacher = _put(place, np.zeros((1, 1), np.int32)), _put(place, np.ones((1, 1), np.float32))
    with pytest.raises(LightGBMError):
        ops.top_logits(z, 1)
    with pytest.raises(LightGBMError):
        ops.distill_loss(z, teacher)
    p = np.broadcast_to(np.float32(0.5), (1, 1026, 2))
    with pytest.raises(LightGBMError):
        ops.verify_drafts(p, np.zeros((1, 1025), np.int32), None, p[:, :-1, 0], p[:, 0, 0])
