"""KeyedEstimator(keySolver="grouped") and KeyedModel.transform(device=...)
against the host's loop over keys."""

import numpy as np
import pandas as pd
import pytest
import torch

import spark_sklearn_amd as ska
from spark_sklearn_amd.models import (LinearRegression, LinearSVC,
                                      LogisticRegression, Ridge,
                                      SGDClassifier)

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def frame(n_keys, n_classes, F=9, seed=0, low=30, high=90):
    """n_classes 0: a regression target."""
    rng = np.random.default_rng(seed)
    parts = []
    for k in range(n_keys):
        n = int(rng.integers(low, high))
        X = rng.standard_normal((n, F)).astype(np.float32)
        z = X @ rng.standard_normal((F, max(n_classes, 1)))
        if n_classes == 0:
            y = z[:, 0] + 0.1 * rng.standard_normal(n)
        elif n_classes == 2:
            y = (z[:, 0] > 0).astype(int)
            y[:2] = 0, 1
        else:
            y = z.argmax(1)
            y[:n_classes] = np.arange(n_classes)
        parts.append(pd.DataFrame({"k": k, "features": list(X), "y": y}))
    df = pd.concat(parts, ignore_index=True)
    return df.sample(frac=1.0, random_state=seed).reset_index(drop=True)


def host_loop(est, df):
    from sklearn.base import clone

    from spark_sklearn_amd.models._solver_ref import BatchPlan, linear_fit_ref

    out = {}
    for key, g in df.groupby("k"):
        X = np.stack(g["features"].values).astype(np.float32)
        y = g["y"].values
        msq = float(np.mean(np.sum(X.astype(np.float64) ** 2, axis=1)))
        spec = est._column_spec(len(X), msq)
        classes = np.unique(df["y"]) if hasattr(est, "_estimator_type") and \
            est._estimator_type == "classifier" else None
        n_classes = 0 if classes is None else len(classes)
        C = n_classes if n_classes > 2 else 1
        plan = BatchPlan(
            loss=np.full(C, spec["loss"], np.int32),
            **{v: np.full(C, spec[v], np.float32)
               for v in ("lr", "l1", "l2", "momentum", "tol")},
            max_iter=np.full(C, spec["max_iter"], np.int32),
            target_class=(np.arange(C) if C > 1 else np.array(
                [1 if n_classes else -1])).astype(np.int32),
            col_to_cand=np.zeros(C, np.int32), n_classes=C,
            fit_intercept=np.full(C, spec["fit_intercept"], np.uint8))
        yy = y.astype(np.float32) if classes is None else \
            np.searchsorted(classes, y)
        W, b, n_iter, _ = linear_fit_ref(X, yy, plan)
        out[key] = clone(est)._finalize_fit(W, b, n_iter, classes)
    return out




def tagged(est):
    from sklearn.base import is_classifier

    est._estimator_type = "classifier" if is_classifier(est) else "regressor"
    return est


FITS = [
    (LogisticRegression(max_iter=40, tol=0.0), 2),
    (LogisticRegression(max_iter=25, tol=0.0, C=0.1), 4),
    (LogisticRegression(max_iter=40, tol=1e-2), 2),
    (LinearSVC(max_iter=15, tol=0.0, C=0.05), 2),
    (SGDClassifier(loss="squared_error", max_iter=20, tol=0.0), 3),
    (LinearRegression(max_iter=30, tol=0.0), 0),
    (Ridge(alpha=3.0, max_iter=30, tol=0.0, fit_intercept=False), 0),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("case", range(len(FITS)))
def test_grouped_fit_follows_the_reference(device, case, monkeypatch):
    """Weights after the same steps of gradient descent.  A step's gradient
    sums some 90 rows of some 9 products in float32 on both sides, off by
    about 100 * 2^-24 each and carried over at most 40 steps whose momentum
    weighs an error at most 1 / (1 - 0.9) times: 40 * 10 * 100 * 2^-24 =
    2.4e-3 of the largest weight."""
    est, n_classes = FITS[case]
    df = frame(7, n_classes, seed=case)
    import spark_sklearn_amd.engine as engine

    monkeypatch.setattr(
        engine, "_device_or_none",
        lambda d: torch.device(device) if device == "cuda" else None)
    model = ska.KeyedEstimator(sklearnEstimator=est, keyCols=["k"],
                               yCol="y", keySolver="grouped").fit(df)
    want = host_loop(tagged(est), df)
    assert len(model.keyedModels) == 7
    for _, row in model.keyedModels.iterrows():
        got, ref = row["estimator"].estimator, want[row["k"]]
        assert got.coef_.shape == ref.coef_.shape
        scale = np.abs(ref.coef_).max()
        assert np.abs(got.coef_ - ref.coef_).max() <= 2.4e-3 * scale
        assert np.abs(np.atleast_1d(got.intercept_ - ref.intercept_)
                      ).max() <= 2.4e-3 * scale
        if est.tol == 0.0:
            assert np.array_equal(got.n_iter_, ref.n_iter_)
        else:
            assert np.all(np.abs(got.n_iter_ - ref.n_iter_) <= 1)


def test_grouped_fit_leaves_other_keys_to_the_host():
    """Keys without all classes, other estimators, class weights."""
    from sklearn.linear_model import LogisticRegression as Host

    df = frame(4, 3)
    df.loc[(df["k"] == 2) & (df["y"] == 1), "y"] = 0
    for est in (LogisticRegression(max_iter=5), Host(max_iter=50)):
        model = ska.KeyedEstimator(sklearnEstimator=est, keyCols=["k"],
                                   yCol="y", keySolver="grouped").fit(df)
        assert len(model.keyedModels) == 4
        missing = model.keyedModels.iloc[2]["estimator"]
        assert list(missing.classes_) == [0, 2]
    with pytest.raises(ValueError):
        ska.KeyedEstimator(sklearnEstimator=Host(), yCol="y",
                           keySolver="rows")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("est,n_classes", [
    (LogisticRegression(max_iter=20), 2), (LinearSVC(max_iter=20), 5),
    (Ridge(max_iter=20), 0)], ids=["binary", "multiclass", "ridge"])
def test_device_transform_equals_the_host(device, est, n_classes):
    df = frame(12, n_classes, seed=3)
    model = ska.KeyedEstimator(sklearnEstimator=est, keyCols=["k"],
                               yCol="y", keySolver="grouped").fit(df)
    host = model.transform(df)
    got = model.transform(df, device=device)
    assert list(got.columns) == list(host.columns)
    assert got.index.equals(host.index)
    assert got["prediction"].dtype == host["prediction"].dtype
    if n_classes:
        # scores in float32: only a row whose two best are equal to
        # rounding could differ, and random rows are not
        assert (got["prediction"] == host["prediction"]).all()
    else:
        np.testing.assert_allclose(got["prediction"], host["prediction"],
                                   rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("device", DEVICES)
def test_device_transform_keys(device):
    """Several key columns, keys without a model or without a value, models
    of different classes, a class label that is a text."""
    df = frame(6, 3, seed=8)
    df["a"] = np.where(df["k"] % 2, "odd", "even")
    names = np.array(["x", "y", "z"])
    df["y"] = names[df["y"]]
    df.loc[(df["k"] == 4) & (df["y"] == "y"), "y"] = "x"   # two classes
    model = ska.KeyedEstimator(
        sklearnEstimator=LogisticRegression(max_iter=15), keyCols=["a", "k"],
        yCol="y").fit(df)
    df["a"] = df["a"].astype(object)
    df.loc[df.index[3], "a"] = None
    df.loc[df.index[5], "k"] = 77
    with pytest.raises(KeyError):
        model.transform(df, device=device)
    host = model.transform(df, unseenKeys="drop")
    got = model.transform(df, unseenKeys="drop", device=device)
    assert len(got) == len(df) - 2
    assert got.index.equals(host.index)
    assert (got["prediction"] == host["prediction"]).all()
    none = df[df["k"] == 77]
    empty = model.transform(none, unseenKeys="drop", device=device)
    assert len(empty) == 0 and "prediction" in empty.columns


def test_device_transform_refuses():
    from sklearn.linear_model import LogisticRegression as Host
    from sklearn.preprocessing import StandardScaler

    df = frame(3, 2)
    for est, y in ((Host(), "y"), (StandardScaler(), None)):
        model = ska.KeyedEstimator(sklearnEstimator=est, keyCols=["k"],
                                   yCol=y).fit(df)
        with pytest.raises(ValueError):
            model.transform(df, device="cpu")
    model = ska.KeyedEstimator(
        sklearnEstimator=Ridge(max_iter=3), keyCols=["k"], yCol="y").fit(df)
    wide = df.copy()
    wide["features"] = [np.append(v, 1.0) for v in wide["features"]]
    with pytest.raises(ValueError):
        model.transform(wide, device="cpu")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan, 3e38])
def test_device_transform_of_rows_that_are_not_finite(device, value):
    """A key without all classes answers with one of its own, whatever the
    row holds, as on the host."""
    df = frame(5, 4, seed=2)
    df.loc[(df["k"] == 3) & (df["y"] == 3), "y"] = 0      # three classes
    df.loc[(df["k"] == 4) & (df["y"] > 1), "y"] = 0       # two
    model = ska.KeyedEstimator(
        sklearnEstimator=LogisticRegression(max_iter=15), keyCols=["k"],
        yCol="y").fit(df)
    odd = df.groupby("k").head(4).copy()
    odd["features"] = [np.where(np.arange(9) == i % 9, value, v).astype(
        np.float32) for i, v in enumerate(odd["features"])]
    with np.errstate(all="ignore"):
        host = model.transform(odd)
        got = model.transform(odd, device=device)
    assert got["prediction"].dtype == host["prediction"].dtype
    known = {k: set(g["y"]) for k, g in df.groupby("k")}
    assert all(p in known[k] for k, p in zip(got["k"], got["prediction"]))
    if abs(value) == np.inf or np.isnan(value):
        assert (got["prediction"] == host["prediction"]).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("est,n_classes", [
    (LogisticRegression(max_iter=20), 3), (LinearSVC(max_iter=20), 2),
    (Ridge(max_iter=20), 0)], ids=["logistic", "hinge", "ridge"])
def test_grouped_fit_under_another_default_type(device, est, n_classes,
                                                monkeypatch):
    import spark_sklearn_amd.engine as engine

    monkeypatch.setattr(
        engine, "_device_or_none",
        lambda d: torch.device(device) if device == "cuda" else None)
    df = frame(5, n_classes, seed=6)

    def fit():
        model = ska.KeyedEstimator(sklearnEstimator=est, keyCols=["k"],
                                   yCol="y", keySolver="grouped").fit(df)
        scored = model.transform(df, device=device)["prediction"].to_numpy()
        return [e.estimator.coef_ for e in
                model.keyedModels["estimator"]] + [scored]

    want = fit()
    before = torch.get_default_dtype()
    torch.set_default_dtype(torch.float64)
    try:
        got = fit()
    finally:
        torch.set_default_dtype(before)
    for a, b in zip(got, want):
        assert a.dtype == b.dtype and np.array_equal(a, b)


@pytest.mark.parametrize("default", ["meta", pytest.param(
    "cuda", marks=pytest.mark.gpu)])
def test_grouped_fit_under_another_default_device(default, monkeypatch):
    import spark_sklearn_amd.engine as engine

    monkeypatch.setattr(engine, "_device_or_none", lambda d: None)
    df = frame(4, 3, seed=6)

    def fit():
        model = ska.KeyedEstimator(
            sklearnEstimator=LogisticRegression(max_iter=9), keyCols=["k"],
            yCol="y", keySolver="grouped").fit(df)
        scored = model.transform(df, device="cpu")["prediction"].to_numpy()
        return [e.estimator.coef_ for e in
                model.keyedModels["estimator"]] + [scored]

    want = fit()
    with torch.device(default):
        got = fit()
    assert all(np.array_equal(a, b) for a, b in zip(got, want))


def test_an_estimator_pickled_without_a_key_solver_fits():
    """As one that was saved before there was a choice."""
    import pickle

    est = ska.KeyedEstimator(sklearnEstimator=Ridge(max_iter=3),
                             keyCols=["k"], yCol="y")
    del est.keySolver
    est = pickle.loads(pickle.dumps(est))
    assert "keySolver" not in vars(est)
    assert len(est.fit(frame(3, 0)).keyedModels) == 3


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("labels", ["same", "few", "own"])
def test_device_transform_has_the_hosts_row_order(device, labels):
    """Also where rows share their index label."""
    df = frame(6, 2, seed=5)
    model = ska.KeyedEstimator(sklearnEstimator=LogisticRegression(
        max_iter=9), keyCols=["k"], yCol="y").fit(df)
    df["row"] = np.arange(len(df))
    df.loc[df.index[4], "k"] = 99
    if labels != "own":
        df.index = np.zeros(len(df), int) if labels == "same" else \
            np.arange(len(df))[::-1] // 7
    host = model.transform(df, unseenKeys="drop")
    got = model.transform(df, unseenKeys="drop", device=device)
    pd.testing.assert_frame_equal(got, host)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("change", [
    lambda k: k.astype(float), lambda k: k == 1, lambda k: k.astype("Int64"),
    lambda k: k.astype("category"), lambda k: k.astype(object),
    lambda k: k.astype("int8")],
    ids=["float", "bool", "nullable", "category", "object", "int8"])
def test_device_transform_finds_the_keys_that_the_host_finds(device, change):
    """Keys of another type that equal the models'."""
    df = frame(2, 2, seed=9)
    model = ska.KeyedEstimator(sklearnEstimator=LogisticRegression(
        max_iter=9), keyCols=["k"], yCol="y").fit(df)
    df["k"] = change(df["k"])
    pd.testing.assert_frame_equal(model.transform(df, device=device),
                                  model.transform(df))
