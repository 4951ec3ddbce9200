"""Grouped-row operators against their definition in 64 bits.

Tolerances.  A value that is computed as a sum of K products in 32 bits and
then rounded to type t is off by at most

    eps_t / 2 * |value|  +  (K + 1) * 2^-23 * sum |a_i * b_i|

whatever the order of the sum (2^-24 an addition that rounds, 2^-23 one that
truncates, as a matrix unit may), plus the least step of the type below its
normal range.  Copies are exact.
"""

import numpy as np
import pytest
import torch

import spark_sklearn_amd as ska

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
TYPES = [torch.float32, torch.bfloat16, torch.float16]
SHORT = {torch.float32: "fp32", torch.bfloat16: "bf16",
         torch.float16: "fp16"}


def ids_of(case, T, k, G, seed=0):
    rng = np.random.default_rng(seed)
    shape = (T, k)
    if case == "uniform":
        return rng.integers(0, G, shape)
    if case == "skewed":
        return np.minimum((rng.pareto(0.7, shape)).astype(np.int64), G - 1)
    if case == "one":
        return np.full(shape, G // 2)
    if case == "none":
        return np.full(shape, -1)
    if case == "dropped":
        ids = rng.integers(0, G, shape)
        ids[rng.random(shape) < 0.3] = -1
        ids[rng.random(shape) < 0.1] = G
        return ids
    raise AssertionError(case)


def plan64(ids, G):
    flat = np.asarray(ids).astype(np.int64).ravel()
    flat = np.where((flat < 0) | (flat >= G), G, flat)
    order = np.argsort(flat, kind="stable")
    slots = np.empty_like(order)
    slots[order] = np.arange(order.size)
    counts = np.bincount(flat, minlength=G + 1)[:G]
    return np.concatenate([[0], np.cumsum(counts)]), slots, order


def check(got, want, scale, K):
    """`want` and `scale` (the sum of absolute products) in float64."""
    info = torch.finfo(got.dtype)
    got = got.double().cpu()
    tol = (info.eps / 2 * want.abs() + (K + 1) * 2.0 ** -23 * scale
           + info.tiny * info.eps)
    # the rounding of a value that is itself off
    tol = tol * (1 + info.eps)
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (
        f"{int(bad.sum())} of {bad.numel()} off, worst "
        f"{float(((got - want).abs() / tol.clamp_min(1e-300))[bad].max())} "
        f"times the tolerance, first at {bad.nonzero()[0].tolist()}")


def randn(gen, *shape, dtype=torch.float32, device="cpu"):
    return torch.randn(*shape, generator=gen).to(dtype).to(device)


# -- group_rows ---------------------------------------------------------------

SORTS = [
    (0, 1, 5, "uniform"), (1, 1, 1, "uniform"), (1, 2, 64, "uniform"),
    (7, 3, 2, "dropped"), (64, 1, 64, "uniform"), (65, 1, 300, "skewed"),
    (1024, 2, 37, "dropped"), (2049, 1, 37, "uniform"),
    (683, 3, 100, "one"), (5000, 1, 1, "uniform"), (5000, 1, 8, "none"),
    (9001, 2, 60, "skewed"), (40000, 1, 4096, "dropped"),
    (30011, 1, 8191, "uniform"), (30011, 1, 8192, "dropped"),
    (2500, 1, 70000, "uniform"), (300, 1, 65537, "dropped"),
    (100, 1, 65536, "dropped"), (3000, 2, 1 << 20, "uniform"),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("itype", [torch.int32, torch.int64])
@pytest.mark.parametrize("T,k,G,case", SORTS)
def test_group_rows(device, itype, T, k, G, case):
    ids = ids_of(case, T, k, G)
    offsets, slots, order = plan64(ids, G)
    plan = ska.group_rows(torch.as_tensor(ids).to(itype).to(device), G)
    assert all(v.dtype == torch.int32 for v in plan)
    assert plan.slots.shape == (T, k)
    assert np.array_equal(plan.offsets.cpu().numpy(), offsets)
    assert np.array_equal(plan.order.cpu().numpy(), order)
    assert np.array_equal(plan.slots.cpu().numpy().ravel(), slots)


@pytest.mark.gpu
@pytest.mark.parametrize("M,G", [
    (3_000_000, 1000), (2_300_001, 100_000), (60_001, 4096), (10_000, 3000),
    (9_999, 3000), (217_640, 8191), (250_007, 8191), (250_007, 8192)])
def test_group_rows_many(M, G):
    ids = ids_of("dropped", M, 1, G)
    offsets, slots, order = plan64(ids, G)
    plan = ska.group_rows(torch.as_tensor(ids[:, 0]).cuda(), G)
    assert np.array_equal(plan.offsets.cpu().numpy(), offsets)
    assert np.array_equal(plan.order.cpu().numpy(), order)
    assert np.array_equal(plan.slots.cpu().numpy(), slots)


@pytest.mark.parametrize("device", DEVICES)
def test_group_rows_far_ids_and_strides(device):
    """Ids that only look valid in 32 bits, and ids that lie apart."""
    wide = torch.tensor([[1 << 32, 9], [(1 << 32) + 1, 9], [1, 9],
                         [-(1 << 33), 9], [0, 9], [2 ** 63 - 1, 9]])
    ids = wide.to(device)[:, 0]
    plan = ska.group_rows(ids, 2)
    assert plan.offsets.tolist() == [0, 1, 2]
    assert plan.order.tolist() == [4, 2, 0, 1, 3, 5]
    assert plan.slots.tolist() == [2, 3, 1, 4, 0, 5]


# -- gather and combine -------------------------------------------------------

MOVES = [  # T, k, G, F, ids
    (1, 1, 1, 1, "uniform"), (1, 2, 64, 256, "uniform"),
    (5, 1, 3, 3, "dropped"), (33, 2, 4, 8, "uniform"),
    (100, 3, 7, 65, "dropped"), (257, 2, 16, 250, "skewed"),
    (64, 8, 8, 1032, "dropped"), (31, 4, 5, 2047, "uniform"),
    (1000, 1, 100, 17, "none"), (130, 5, 3, 64, "one"),
    (2100, 2, 33, 127, "dropped"),
]


def spread64(v, slots, kept, w=None):
    """v[t] (scaled) to the places of the kept entries, in float64."""
    T, k = slots.shape
    out = torch.zeros(T * k, v.shape[1], dtype=torch.float64)
    for j in range(k):
        at = kept[:, j]
        part = v.double()[at]
        if w is not None:
            part = part * w.double()[at, j][:, None]
        out[slots[at, j]] = part
    return out


def collect64(v, slots, kept, w=None):
    T, k = slots.shape
    out = torch.zeros(T, v.shape[1], dtype=torch.float64)
    for j in range(k):
        at = kept[:, j]
        part = v.double()[slots[at, j]]
        if w is not None:
            part = part * w.double()[at, j][:, None]
        out[at] += part
    return out


def move_case(T, k, G, case):
    ids = ids_of(case, T, k, G, seed=T)
    offsets, slots, _ = plan64(ids, G)
    slots = torch.as_tensor(slots).reshape(T, k)
    return torch.as_tensor(ids), slots, slots < int(offsets[-1])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES, ids=SHORT.get)
@pytest.mark.parametrize("T,k,G,F,case", MOVES)
def test_gather_rows(device, dtype, T, k, G, F, case):
    ids, slots, kept = move_case(T, k, G, case)
    gen = torch.Generator().manual_seed(F)
    # every other column block of a wider matrix, from an odd address
    wide = randn(gen, T, F + 5, dtype=dtype, device=device)
    x = wide[:, 3:3 + F].detach().requires_grad_()
    plan = ska.group_rows(ids.to(device), G)
    rows = ska.gather_rows(x, plan)
    xc = x.detach().cpu()
    assert torch.equal(rows.detach().double().cpu(),
                       spread64(xc, slots, kept))
    grad = randn(gen, T * k, F, dtype=dtype, device=device)
    dx, = torch.autograd.grad(rows, x, grad)
    check(dx, collect64(grad.cpu(), slots, kept),
          collect64(grad.abs().cpu(), slots, kept), k)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES, ids=SHORT.get)
@pytest.mark.parametrize("weights", ["none", "same", "float32"])
@pytest.mark.parametrize("T,k,G,F,case", MOVES)
def test_combine_rows(device, dtype, weights, T, k, G, F, case):
    ids, slots, kept = move_case(T, k, G, case)
    gen = torch.Generator().manual_seed(F)
    wide = randn(gen, T * k, F + 5, dtype=dtype, device=device)
    rows = wide[:, 2:2 + F].detach()
    w = None
    if weights != "none":
        w = randn(gen, T, k, device=device,
                  dtype=torch.float32 if weights == "float32" else dtype)
        # an entry without a group takes no part, whatever it holds
        w = torch.where(kept.to(device), w, float("nan"))
    rows = torch.where(
        (torch.arange(T * k) < int(kept.sum()))[:, None].to(device), rows,
        float("inf")).requires_grad_()
    if w is not None:
        w.requires_grad_()
    plan = ska.group_rows(ids.to(device), G)
    y = ska.combine_rows(rows, plan, w)
    rc = rows.detach().cpu()
    wc = None if w is None else w.detach().cpu()
    check(y.detach(), collect64(rc, slots, kept, wc),
          collect64(rc.abs(), slots, kept, None if wc is None else wc.abs()),
          k + 1)
    grad = randn(gen, T, F, dtype=dtype, device=device)
    leaves = [rows] if w is None else [rows, w]
    got = torch.autograd.grad(y, leaves, grad)
    gc = grad.cpu()
    want = spread64(gc, slots, kept, wc)
    check(got[0], want, want.abs(), 1)
    if w is not None:
        clean = torch.where(torch.isfinite(rc), rc, 0)
        pick = clean.double()[slots] * kept[..., None]
        check(got[1], (pick * gc.double()[:, None]).sum(-1),
              (pick * gc.double()[:, None]).abs().sum(-1), F)


# -- grouped_linear -----------------------------------------------------------

def offsets_of(case, M, G, seed=0):
    rng = np.random.default_rng(seed)
    if case == "even":
        cut = np.linspace(0, M, G + 1).astype(np.int64)
    elif case == "ragged":
        cut = np.sort(rng.integers(0, M + 1, G + 1))
        cut[0], cut[-1] = 0, M
    elif case == "tail":      # rows behind the last group
        cut = np.sort(rng.integers(0, M // 2 + 1, G + 1))
        cut[0] = 0
    elif case == "first":     # all in the first group
        cut = np.full(G + 1, M)
        cut[0] = 0
    elif case == "last":
        cut = np.zeros(G + 1, np.int64)
        cut[-1] = M
    elif case == "nobody":
        cut = np.zeros(G + 1, np.int64)
    return torch.as_tensor(cut).int()


PRODUCTS = [  # M, G, N, F, offsets
    (1, 1, 1, 1, "even"), (1, 5, 3, 7, "last"), (2, 64, 33, 64, "ragged"),
    (8, 64, 256, 512, "ragged"), (16, 4, 17, 16, "even"),
    (63, 3, 64, 32, "ragged"), (64, 1, 64, 64, "even"),
    (65, 2, 65, 65, "ragged"), (130, 7, 10, 256, "ragged"),
    (300, 9, 1, 250, "tail"), (300, 4, 131, 250, "ragged"),
    (257, 300, 40, 24, "ragged"), (500, 3, 200, 130, "first"),
    (200, 6, 72, 96, "nobody"), (1025, 5, 129, 257, "tail"),
    (900, 2, 264, 520, "last"), (700, 11, 384, 136, "ragged"),
    (1500, 3, 5, 70, "ragged"), (3000, 40, 3, 260, "ragged"),
    (2000, 2, 40, 33, "first"), (1100, 600, 20, 9, "tail"),
    (40, 90, 300, 48, "ragged"), (1030, 1, 61, 2056, "even"),
]


def linear64(rows, weight, offsets, bias, grad):
    """y, drows, dweight, dbias, each with its sum of absolute products."""
    M, (G, N, F) = rows.shape[0], weight.shape
    r, w, b, d = (v.double().cpu() for v in (rows, weight, bias, grad))
    shapes = [(M, N), (M, F), (G, N, F), (G, N)]
    out = [[torch.zeros(s, dtype=torch.float64) for s in shapes]
           for _ in range(2)]
    edges = offsets.tolist()
    for g, (lo, hi) in enumerate(zip(edges, edges[1:])):
        for o, (rr, ww, bb, dd) in zip(out, (
                (r[lo:hi], w[g], b[g], d[lo:hi]),
                (r[lo:hi].abs(), w[g].abs(), b[g].abs(), d[lo:hi].abs()))):
            o[0][lo:hi] = rr @ ww.t() + bb
            o[1][lo:hi] = dd @ ww
            o[2][g] = dd.t() @ rr
            o[3][g] = dd.sum(0)
    return out


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES, ids=SHORT.get)
@pytest.mark.parametrize("apart", [False, True], ids=["packed", "apart"])
@pytest.mark.parametrize("M,G,N,F,case", PRODUCTS)
def test_grouped_linear(device, dtype, apart, M, G, N, F, case):
    gen = torch.Generator().manual_seed(M + N)
    offsets = offsets_of(case, M, G, seed=M)
    pad = 3 if apart else 0
    rows = randn(gen, M, F + pad, dtype=dtype, device=device)[:, pad:]
    rows = rows.detach().requires_grad_()
    weight = randn(gen, G, N, F, dtype=dtype,
                   device=device).requires_grad_()
    bias = randn(gen, G, N, dtype=dtype, device=device).requires_grad_()
    grad = randn(gen, M, N + pad, dtype=dtype, device=device)[:, pad:]
    y = ska.grouped_linear(rows, weight, offsets.to(device), bias)
    got = (y.detach(),) + torch.autograd.grad(y, [rows, weight, bias], grad)
    want, scale = linear64(rows.detach(), weight.detach(), offsets,
                           bias.detach(), grad)
    for name, v, u, s, K in zip(("y", "drows", "dweight", "dbias"), got,
                                want, scale, (F + 1, N, M, M)):
        assert v.dtype == dtype and v.shape == u.shape, name
        check(v, u, s, K)


def check_there(got, want, scale, K):
    """check(), where the operands are."""
    info = torch.finfo(got.dtype)
    tol = (info.eps / 2 * want.abs() + (K + 1) * 2.0 ** -23 * scale
           + info.tiny * info.eps) * (1 + info.eps)
    off = (got.double() - want).abs() - tol
    assert bool((off <= 0).all()), float(off.max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=SHORT.get)
@pytest.mark.parametrize("M,G,N,F", [
    (24000, 20, 1200, 1250),    # the largest tiles, in all three products
    (24000, 20, 1200, 1251),    # the same with rows at odd addresses
    (6000, 16, 700, 300),       # middle tiles, two steps in LDS
    (20000, 60, 520, 200),      # and one
    (9000, 100, 520, 140),      # low tiles, one step
    (6000, 90, 520, 700),       # and two
    (5000, 3, 37, 600),         # few outputs
])
def test_grouped_linear_tiles(dtype, M, G, N, F):
    """Sizes at which each of the tiles is taken, ragged everywhere."""
    gen = torch.Generator().manual_seed(N)
    offsets = offsets_of("ragged", M, G, seed=F)
    offsets[-1] -= 3            # rows behind the last group
    rows, weight, bias, grad = (
        randn(gen, *shape, dtype=dtype, device="cuda")
        for shape in ((M, F), (G, N, F), (G, N), (M, N)))
    leaves = [v.requires_grad_() for v in (rows, weight, bias)]
    y = ska.grouped_linear(rows, weight, offsets.cuda(), bias)
    dr, dw, db = torch.autograd.grad(y, leaves, grad)
    y = y.detach()
    edges = offsets.tolist()
    for g, (a, b) in enumerate(zip(edges, edges[1:])):
        r, w, c, d = (v.detach().double() for v in (
            rows[a:b], weight[g], bias[g], grad[a:b]))
        R, W, C, D = (v.abs() for v in (r, w, c, d))
        check_there(y[a:b], r @ w.t() + c, R @ W.t() + C, F + 1)
        check_there(dr[a:b], d @ w, D @ W, N)
        check_there(dw[g], d.t() @ r, D.t() @ R, M)
        check_there(db[g], d.sum(0), D.sum(0), M)
    assert not y[M - 3:].any() and not dr[M - 3:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=SHORT.get)
def test_grouped_linear_most_outputs(dtype):
    """As many outputs as there may be, for a few rows."""
    M, N, F = 3, 2 ** 21 - 1, 4
    gen = torch.Generator().manual_seed(5)
    rows, weight, bias, grad = (
        randn(gen, *shape, dtype=dtype, device="cuda")
        for shape in ((M, F), (1, N, F), (1, N), (M, N)))
    offsets = torch.tensor([0, M], dtype=torch.int32, device="cuda")
    leaves = [v.requires_grad_() for v in (rows, weight, bias)]
    y = ska.grouped_linear(rows, weight, offsets, bias)
    dr, dw, db = torch.autograd.grad(y, leaves, grad)
    r, w, c, d = (v.detach().double() for v in (
        rows, weight[0], bias[0], grad))
    R, W, C, D = (v.abs() for v in (r, w, c, d))
    check_there(y.detach(), r @ w.t() + c, R @ W.t() + C, F + 1)
    check_there(dr, d @ w, D @ W, N)
    check_there(dw[0], d.t() @ r, D.t() @ R, M)
    check_there(db[0], d.sum(0), D.sum(0), M)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES, ids=SHORT.get)
def test_grouped_linear_keeps_groups_apart(device, dtype):
    """What one group's rows and weights hold, and what lies behind the last
    group, reaches no other group: neither NaN nor infinity."""
    M, G, N, F = 150, 5, 70, 90
    gen = torch.Generator().manual_seed(3)
    offsets = torch.tensor([0, 31, 64, 64, 101, 140], dtype=torch.int32)
    rows = randn(gen, M, F, dtype=dtype)
    weight = randn(gen, G, N, F, dtype=dtype)
    grad = randn(gen, M, N, dtype=dtype)
    clean = [v.clone() for v in (rows, weight, grad)]
    for v in (rows, grad):
        v[31:64] = float("nan")
        v[140:] = float("inf")
    weight[1] = float("inf")
    weight[2] = float("nan")
    out = []
    for r, w, d in ((rows, weight, grad), clean):
        r, w = (v.to(device).requires_grad_() for v in (r, w))
        y = ska.grouped_linear(r, w, offsets.to(device))
        out.append([y.detach().cpu()] + [
            v.cpu() for v in torch.autograd.grad(y, [r, w], d.to(device))])
    for a, b, rowwise in zip(*out, (True, True, False)):
        if rowwise:
            assert torch.isnan(a[31:64]).all()
            a, b = (torch.cat([v[:31], v[64:]]) for v in (a, b))
            assert (a[140 - 33:] == 0).all()
        else:
            assert torch.isnan(a[1]).all() and (a[2] == 0).all()
            a, b = a[[0, 2, 3, 4]], b[[0, 2, 3, 4]]
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("M,G,N,F", [(8192, 1, 2048, 2048),
                                     (30000, 2, 70, 100), (30000, 1, 9, 64)])
def test_long_sums_in_parts(M, G, N, F):
    """float32 weight gradients sum at most 512 terms, and then those sums:
    a term passes 512 + M / 512 + 1 additions."""
    gen = torch.Generator().manual_seed(M)
    offsets = offsets_of("even", M, G)
    rows, grad = (randn(gen, M, v, device="cuda") for v in (F, N))
    weight = torch.zeros(G, N, F, device="cuda", requires_grad=True)
    bias = torch.zeros(G, N, device="cuda", requires_grad=True)
    y = ska.grouped_linear(rows, weight, offsets.cuda(), bias)
    dweight, dbias = torch.autograd.grad(y, [weight, bias], grad)
    r, d = rows.double(), grad.double()
    edges = offsets.tolist()
    for g, (a, b) in enumerate(zip(edges, edges[1:])):
        check(dweight[g], (d[a:b].t() @ r[a:b]).cpu(),
              (d[a:b].t().abs() @ r[a:b].abs()).cpu(), 513 + M // 512)
        check(dbias[g], d[a:b].sum(0).cpu(), d[a:b].abs().sum(0).cpu(),
              513 + M // 512)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("M,G,N,F", [(0, 3, 4, 5), (7, 3, 0, 5),
                                     (7, 3, 4, 0), (0, 1, 0, 0)])
def test_grouped_linear_empty(device, M, G, N, F):
    offsets = torch.tensor([0] + [M] * G, dtype=torch.int32, device=device)
    rows = torch.ones(M, F, device=device, requires_grad=True)
    weight = torch.ones(G, N, F, device=device, requires_grad=True)
    bias = torch.full((G, N), 2.0, device=device, requires_grad=True)
    y = ska.grouped_linear(rows, weight, offsets, bias)
    assert y.shape == (M, N) and bool((y == 2.0 + F).all())
    dr, dw, db = torch.autograd.grad(y, [rows, weight, bias],
                                     torch.ones_like(y))
    assert dr.shape == rows.shape and bool((dr == N).all())
    assert dw.shape == weight.shape and db.shape == bias.shape
    if N:
        assert db[0].tolist() == [float(M)] * N and not db[1:].any()
    if N and F:
        assert bool((dw[0] == M).all()) and not dw[1:].any()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("wrt", [(0,), (1,), (2,), (0, 2), (1, 2)])
def test_grouped_linear_some_gradients(device, wrt):
    """Only the gradients that are asked for, the same as all together."""
    gen = torch.Generator().manual_seed(1)
    offsets = torch.tensor([0, 5, 5, 40], dtype=torch.int32, device=device)
    data = [randn(gen, 44, 33, device=device),
            randn(gen, 3, 20, 33, device=device),
            randn(gen, 3, 20, device=device)]
    grad = randn(gen, 44, 20, device=device)

    def grads(which):
        leaves = [v.detach().requires_grad_(i in which)
                  for i, v in enumerate(data)]
        y = ska.grouped_linear(leaves[0], leaves[1], offsets, leaves[2])
        return torch.autograd.grad(y, [leaves[i] for i in which], grad)

    every = grads((0, 1, 2))
    for got, i in zip(grads(wrt), wrt):
        assert torch.equal(got, every[i])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("wrt", [(0,), (1,), (2,), (3,), (1, 3)])
def test_gradients_asked_for_one_by_one(device, wrt):
    """Some gradients of a run in which all inputs require theirs."""
    x, ids, weight, bias, w, dy = chain_data(device, T=50)
    leaves = [v.requires_grad_() for v in (x, weight, bias, w)]
    every = torch.autograd.grad(
        chain(x, ids, weight.shape[0], weight, bias, w), leaves, dy)
    some = torch.autograd.grad(
        chain(x, ids, weight.shape[0], weight, bias, w),
        [leaves[i] for i in wrt], dy)
    for got, i in zip(some, wrt):
        assert torch.equal(got, every[i])


def test_gradcheck_reference():
    """The reference's gradients against differences, in 64 bits."""
    gen = torch.Generator().manual_seed(5)
    ids = torch.tensor([[0, 2], [2, 2], [-1, 0], [3, 1], [0, 9]])
    x = torch.randn(5, 3, generator=gen, dtype=torch.float64)
    weight = torch.randn(4, 2, 3, generator=gen, dtype=torch.float64)
    bias = torch.randn(4, 2, generator=gen, dtype=torch.float64)
    w = torch.randn(5, 2, generator=gen, dtype=torch.float64)
    plan = ska.group_rows(ids, 4)

    def whole(x, weight, bias, w):
        rows = ska.gather_rows(x, plan)
        out = ska.grouped_linear(rows, weight, plan.offsets, bias)
        return ska.combine_rows(out, plan, w)

    assert torch.autograd.gradcheck(
        whole, [v.requires_grad_() for v in (x, weight, bias, w)])


@pytest.mark.parametrize("device", DEVICES)
def test_differentiates_once_only(device):
    """A second differentiation is an error, never a silent zero."""
    x, ids, weight, bias, w, dy = chain_data(device, T=20)
    for i in range(4):
        leaves = [v.detach().requires_grad_(j == i)
                  for j, v in enumerate((x, weight, bias, w))]
        y = chain(leaves[0], ids, weight.shape[0], *leaves[1:])
        g, = torch.autograd.grad((y * y).sum(), leaves[i], create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.sum(), leaves[i])


def chain(x, ids, G, weight, bias, w):
    plan = ska.group_rows(ids, G)
    rows = ska.gather_rows(x, plan)
    out = ska.grouped_linear(rows, weight, plan.offsets, bias)
    return ska.combine_rows(out, plan, w)


def chain_data(device, T=203, k=2, G=9, F=70, N=41, seed=0):
    gen = torch.Generator().manual_seed(seed)
    ids = torch.as_tensor(ids_of("dropped", T, k, G, seed=seed)).to(device)
    return (randn(gen, T, F, device=device), ids,
            randn(gen, G, N, F, device=device) * F ** -0.5,
            randn(gen, G, N, device=device),
            torch.rand(T, k, generator=gen).to(device),
            randn(gen, T, N, device=device))


@pytest.mark.parametrize("device", DEVICES)
def test_whole_run_gradients(device):
    """Sort, gather, product and weighted sum together: each gradient against
    a difference.  The run is linear in each input by itself, so that a step
    of any size gives <grad, step> = <dy, f(v + step) - f(v)>; both sides are
    sums of about 10^4 products in float32, whose errors stay under
    10^4 * 2^-23 of the sum of their absolute values."""
    x, ids, weight, bias, w, dy = chain_data(device)
    G = weight.shape[0]
    leaves = [v.requires_grad_() for v in (x, weight, bias, w)]
    y = chain(x, ids, G, weight, bias, w)
    grads = torch.autograd.grad(y, leaves, dy)
    gen = torch.Generator().manual_seed(9)
    with torch.no_grad():
        for i, g in enumerate(grads):
            step = randn(gen, *g.shape, device=device)
            moved = [v + step if j == i else v
                     for j, v in enumerate(leaves)]
            y2 = chain(moved[0], ids, G, *moved[1:])
            lhs = (g.double() * step.double()).sum()
            diff = dy.double() * (y2.double() - y.double())
            bound = 1e4 * 2.0 ** -23 * float(
                (g.double() * step.double()).abs().sum()
                + (dy.double().abs() * (y2.double().abs()
                                        + y.double().abs())).sum())
            assert abs(float(lhs - diff.sum())) <= bound


@pytest.mark.gpu
def test_whole_run_repeats_and_other_streams():
    """Bit-equal from run to run and on a stream of the user's own."""
    data = chain_data("cuda", T=3001, G=40)

    def once():
        x, ids, weight, bias, w, dy = data
        leaves = [v.detach().requires_grad_() for v in (x, weight, bias, w)]
        y = chain(leaves[0], ids, weight.shape[0], *leaves[1:])
        return (y.detach(),) + torch.autograd.grad(y, leaves, dy)

    first = once()
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        second = once()
    torch.cuda.current_stream().wait_stream(other)
    for a, b in zip(first, second):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_whole_run_captured():
    """Two captured graphs, replayed in turn with new inputs and eager work
    between them: each replay equals the eager result of its inputs."""
    sets = [chain_data("cuda", T=t, G=g, seed=t)
            for t, g in ((301, 12), (2501, 33))]
    graphs = []
    for x, ids, weight, bias, w, dy in sets:
        G = weight.shape[0]
        held = [v.clone() for v in (x, weight, bias, w)]
        ids, dy = ids.clone(), dy.clone()

        def once(held=held, ids=ids, dy=dy, G=G):
            leaves = [v.detach().requires_grad_() for v in held]
            y = chain(leaves[0], ids, G, *leaves[1:])
            return (y.detach(),) + torch.autograd.grad(y, leaves, dy)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            once()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = once()
        graphs.append((graph, out, once, held, ids, dy, G))
    for turn in range(4):
        for i, (graph, out, once, held, ids, dy, G) in enumerate(graphs):
            gen = torch.Generator().manual_seed(100 + turn)
            for v in held + [dy]:
                v.copy_(randn(gen, *v.shape))
            ids.copy_(torch.as_tensor(ids_of(
                ("uniform", "dropped", "one", "none")[turn], *ids.shape, G,
                seed=turn)))
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, once()):
                assert torch.equal(a, b), (turn, i)


@pytest.mark.gpu
def test_far_rows():
    """Rows whose addresses pass 32 bits: 2^31 elements and more."""
    F, T = 4096, (1 << 19) + 77
    x = torch.zeros(T, F, dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator().manual_seed(0)
    ends = torch.tensor([0, 1, T // 2, T - 2, T - 1])
    x[ends] = randn(gen, 5, F, dtype=torch.bfloat16, device="cuda")
    ids = torch.zeros(T, dtype=torch.int32, device="cuda")
    ids[ends] = 1
    plan = ska.group_rows(ids, 2)
    rows = ska.gather_rows(x, plan)
    assert torch.equal(rows[T - 5:], x[ends]) and not rows[0].any()
    weight = randn(gen, 2, 5, F, dtype=torch.bfloat16, device="cuda")
    y = ska.grouped_linear(rows, weight, plan.offsets)
    near = ska.grouped_linear(
        rows[T - 5:].contiguous(), weight[1:],
        torch.tensor([0, 5], dtype=torch.int32, device="cuda"))
    want = rows[T - 5:].double() @ weight[1].double().t()
    scale = rows[T - 5:].double().abs() @ weight[1].double().abs().t()
    check(y[T - 5:], want.cpu(), scale.cpu(), F)
    check(near, want.cpu(), scale.cpu(), F)
    back = ska.combine_rows(rows, plan)
    assert torch.equal(back[ends], x[ends])
    assert int(back.any(1).sum()) == 5


@pytest.mark.gpu
def test_plan_of_wild_values_stays_in_bounds():
    """Slots and offsets that no sort made: an entry outside the rows is
    skipped and an offset is clamped, so that nothing faults and the rows
    that are well described come out right."""
    big = 2 ** 31 - 1
    offsets = torch.tensor([0, 2, big], dtype=torch.int32, device="cuda")
    slots = torch.tensor([[0], [-7], [big], [3]], dtype=torch.int32,
                         device="cuda")
    plan = ska.GroupPlan(offsets, slots, slots.reshape(-1))
    x = torch.arange(8.0, device="cuda").reshape(4, 2)
    rows = ska.gather_rows(x, plan)
    assert torch.equal(rows[0], x[0]) and torch.equal(rows[3], x[3])
    y = ska.combine_rows(x, plan)
    assert torch.equal(y[0], x[0]) and not y[1].any() and not y[2].any()
    weight = torch.ones(2, 3, 2, device="cuda")
    out = ska.grouped_linear(x, weight, offsets)
    assert torch.equal(out[:, 0], x.sum(1))


@pytest.mark.gpu
def test_far_products():
    """The tile kernels where row addresses pass 32 bits, in both operands
    and in the gradients; the last rows are compared."""
    F, N, M = 4096, 72, (1 << 19) + 77
    gen = torch.Generator().manual_seed(1)
    rows = torch.zeros(M, F, dtype=torch.bfloat16, device="cuda")
    rows[M - 90:] = randn(gen, 90, F, dtype=torch.bfloat16, device="cuda")
    dy = torch.zeros(M, N, dtype=torch.bfloat16, device="cuda")
    dy[M - 90:] = randn(gen, 90, N, dtype=torch.bfloat16, device="cuda")
    weight = randn(gen, 2, N, F, dtype=torch.bfloat16, device="cuda")
    offsets = torch.tensor([0, M - 80, M], dtype=torch.int32, device="cuda")
    leaves = [rows.requires_grad_(), weight.requires_grad_()]
    y = ska.grouped_linear(*leaves, offsets)
    drows, dweight = torch.autograd.grad(y, leaves, dy)
    r, d = (v[M - 80:].detach().double() for v in (rows, dy))
    w = weight[1].detach().double()
    for got, a, b, K in ((y[M - 80:].detach(), r, w.t(), F),
                         (drows[M - 80:], d, w, N),
                         (dweight[1], d.t(), r, 80)):
        check(got, (a @ b).cpu(), (a.abs() @ b.abs()).cpu(), K)
    assert not y[:M - 90].any() and not drows[:M - 90].any()


@pytest.mark.gpu
def test_far_strides():
    """Rows of a view that lie further apart than a tile's offsets reach."""
    gen = torch.Generator().manual_seed(2)
    wide = torch.zeros(300, 1 << 23, dtype=torch.bfloat16, device="cuda")
    wide[:, :96] = randn(gen, 300, 96, dtype=torch.bfloat16, device="cuda")
    rows = wide[:, :96]
    weight = randn(gen, 2, 80, 96, dtype=torch.bfloat16, device="cuda")
    offsets = torch.tensor([0, 150, 300], dtype=torch.int32, device="cuda")
    got = ska.grouped_linear(rows, weight, offsets)
    assert torch.equal(got, ska.grouped_linear(rows.contiguous(), weight,
                                               offsets))


@pytest.mark.gpu
def test_two_threads_at_once():
    """Two threads on streams of their own, as often as each likes."""
    import threading

    datas = [chain_data("cuda", T=t, G=g, seed=t)
             for t, g in ((900, 7), (2600, 21))]

    def once(data):
        x, ids, weight, bias, w, dy = data
        leaves = [v.detach().requires_grad_() for v in (x, weight, bias, w)]
        y = chain(leaves[0], ids, weight.shape[0], *leaves[1:])
        return (y.detach(),) + torch.autograd.grad(y, leaves, dy)

    want = [once(d) for d in datas]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = once(datas[i])
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not bad and not any(t.is_alive() for t in threads)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("T,k,F", [(5, 0, 4), (0, 2, 4), (3, 2, 0)])
def test_moves_of_nothing(device, T, k, F):
    plan = ska.group_rows(torch.zeros(T, k, dtype=torch.int64,
                                      device=device), 3)
    assert plan.offsets.tolist() == [0] + [T * k] * 3
    x = torch.ones(T, F, device=device, requires_grad=True)
    w = torch.ones(T, k, device=device, requires_grad=True)
    y = ska.combine_rows(ska.gather_rows(x, plan), plan, w)
    assert y.shape == (T, F) and (k or not y.any())
    dx, dw = torch.autograd.grad(y, [x, w], torch.ones_like(y))
    assert dx.shape == (T, F) and dw.shape == (T, k) and not dw[:, :0].any()
    assert F or not dw.any()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("k", [1, 17])
def test_one_dimension_and_many_entries_a_row(device, k):
    """ids [T] are ids [T, 1]; a row may go to many groups, to one twice."""
    gen = torch.Generator().manual_seed(k)
    T, G, F = 90, 11, 24
    ids = torch.randint(-1, G, (T, k), generator=gen).to(device)
    if k == 1:
        ids = ids[:, 0]
    x = randn(gen, T, F, device=device).requires_grad_()
    w = randn(gen, *ids.shape, device=device).requires_grad_()
    plan = ska.group_rows(ids, G)
    assert plan.slots.shape == ids.shape
    y = ska.combine_rows(ska.gather_rows(x, plan), plan, w)
    kept = (ids >= 0).double()
    total = (w.detach().double() * kept).reshape(T, -1).sum(1, keepdim=True)
    size = (w.detach().double().abs() * kept).reshape(T, -1).sum(
        1, keepdim=True)
    xd = x.detach().double()
    check(y.detach(), (xd * total).cpu(), (xd.abs() * size).cpu(), k + 1)
    dy = randn(gen, T, F, device=device)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    assert dw.shape == w.shape
    dots = (xd * dy.double()).sum(1, keepdim=True)
    mags = (xd * dy.double()).abs().sum(1, keepdim=True)
    shape = (T, -1)
    check(dw.reshape(shape), (dots * kept.reshape(shape)).cpu(),
          (mags * kept.reshape(shape)).cpu(), F)
    check(dx, (dy.double() * total).cpu(),
          (dy.double().abs() * size).cpu(), k + 1)


# -- refusals -----------------------------------------------------------------

def small():
    ids = torch.tensor([[0, 1], [1, 1], [0, 2]])
    return (ids, ska.group_rows(ids, 3), torch.ones(3, 4),
            torch.ones(6, 4), torch.ones(3, 2, 4))


@pytest.mark.parametrize("ids,G,error", [
    ([0, 1], 2, TypeError),
    (torch.tensor([0.0]), 2, TypeError),
    (torch.tensor([0], dtype=torch.int16), 2, TypeError),
    (torch.zeros(1, 1, 1, dtype=torch.int32), 2, ValueError),
    (torch.tensor(3), 2, ValueError),
    (torch.tensor([0]), 0, ValueError),
    (torch.tensor([0]), 1 << 24, ValueError),
    (torch.tensor([0]), 2.0, TypeError),
    (torch.tensor([0]), True, TypeError),
])
def test_group_rows_refuses(ids, G, error):
    with pytest.raises(error):
        ska.group_rows(ids, G)


def test_gather_and_combine_refuse():
    ids, plan, x, rows, _ = small()
    for bad, error in [(x.numpy(), TypeError), (x.int(), TypeError),
                       (x[0], ValueError), (x[:2], ValueError),
                       (x.to("meta"), ValueError)]:
        with pytest.raises(error):
            ska.gather_rows(bad, plan)
    with pytest.raises(TypeError):
        ska.gather_rows(x, tuple(plan))
    with pytest.raises(TypeError):
        ska.gather_rows(x, plan._replace(slots=plan.slots.long()))
    with pytest.raises(ValueError):
        ska.gather_rows(x, plan._replace(offsets=plan.offsets[:1]))
    with pytest.raises(ValueError):
        ska.gather_rows(x, plan._replace(slots=plan.slots.reshape(1, 3, 2)))
    for bad, error in [(rows[:5], ValueError), (rows.double().int(),
                                                TypeError)]:
        with pytest.raises(error):
            ska.combine_rows(bad, plan)
    for bad, error in [(torch.ones(3), ValueError),
                       (torch.ones(2, 3), ValueError),
                       (torch.ones(3, 2).half(), TypeError),
                       ([[1.0]], TypeError)]:
        with pytest.raises(error):
            ska.combine_rows(rows, plan, bad)


def test_grouped_linear_refuses():
    _, plan, _, rows, weight = small()
    ok = dict(rows=rows, weight=weight, offsets=plan.offsets, bias=None)
    assert ska.grouped_linear(**ok).shape == (6, 2)
    for change, error in [
            (dict(rows=rows.numpy()), TypeError),
            (dict(rows=rows[:, :3]), ValueError),
            (dict(rows=rows.bfloat16()), TypeError),
            (dict(weight=weight[0]), ValueError),
            (dict(weight=weight[:0]), ValueError),
            (dict(weight=weight.numpy()), TypeError),
            (dict(offsets=plan.offsets.long()), TypeError),
            (dict(offsets=plan.offsets[:3]), ValueError),
            (dict(offsets=plan.offsets[None]), ValueError),
            (dict(bias=torch.ones(3)), ValueError),
            (dict(bias=torch.ones(3, 2).half()), TypeError),
            (dict(bias=1.0), TypeError)]:
        with pytest.raises(error):
            ska.grouped_linear(**{**ok, **change})


@pytest.mark.gpu
def test_refuses_the_same_on_the_gpu():
    """The kernels' checks raise what the reference's raise."""
    ids, plan, x, rows, weight = small()
    w = torch.ones(3, 2)
    calls = [
        lambda c: ska.group_rows(c(ids).float(), 3),
        lambda c: ska.group_rows(c(ids).short(), 3),
        lambda c: ska.group_rows(c(ids), 0),
        lambda c: ska.group_rows(c(ids), 1 << 24),
        lambda c: ska.group_rows(c(ids), 1 << 70),
        lambda c: ska.group_rows(c(ids), 2.0),
        lambda c: ska.group_rows(c(ids)[None], 3),
        lambda c: ska.gather_rows(c(x).int(), p(c)),
        lambda c: ska.gather_rows(c(x)[0], p(c)),
        lambda c: ska.gather_rows(c(x)[:2], p(c)),
        lambda c: ska.gather_rows(c(x), tuple(p(c))),
        lambda c: ska.gather_rows(c(x), None),
        lambda c: ska.gather_rows(c(x), p(c)._replace(
            slots=p(c).slots.long())),
        lambda c: ska.gather_rows(c(x), p(c)._replace(
            offsets=p(c).offsets[:1])),
        lambda c: ska.gather_rows(c(x), p(c)._replace(offsets=3)),
        lambda c: ska.combine_rows(c(rows)[:5], p(c)),
        lambda c: ska.combine_rows(c(rows), p(c), c(w)[:2]),
        lambda c: ska.combine_rows(c(rows), p(c), c(w).half()),
        lambda c: ska.combine_rows(c(rows), p(c), c(w)[:, 0]),
        lambda c: ska.combine_rows(c(rows), p(c), [[1.0]]),
        lambda c: ska.combine_rows(c(rows), None),
        lambda c: ska.grouped_linear(c(rows)[:, :3], c(weight),
                                     p(c).offsets),
        lambda c: ska.grouped_linear(c(rows).bfloat16(), c(weight),
                                     p(c).offsets),
        lambda c: ska.grouped_linear(c(rows), c(weight)[0], p(c).offsets),
        lambda c: ska.grouped_linear(c(rows), c(weight)[:0], p(c).offsets),
        lambda c: ska.grouped_linear(c(rows), c(weight), p(c).offsets[:3]),
        lambda c: ska.grouped_linear(c(rows), c(weight),
                                     p(c).offsets.long()),
        lambda c: ska.grouped_linear(c(rows), c(weight), p(c).offsets,
                                     torch.ones(3)),
        lambda c: ska.grouped_linear(c(rows), c(weight), p(c).offsets,
                                     c(torch.ones(3, 2)).half()),
        lambda c: ska.grouped_linear(c(rows), weight.numpy(), p(c).offsets),
        lambda c: ska.grouped_linear(c(rows), c(weight), p(c).offsets, 1.0),
    ]

    def p(c):
        return ska.GroupPlan(*(c(v) for v in plan))

    for i, call in enumerate(calls):
        raised = []
        for c in (lambda v: v, lambda v: v.cuda()):
            with pytest.raises((TypeError, ValueError)) as info:
                call(c)
            raised.append(info.type)
        assert raised[0] is raised[1], (i, raised)


@pytest.mark.gpu
def test_refuses_mixed_devices():
    _, plan, x, rows, weight = small()
    with pytest.raises(ValueError):
        ska.gather_rows(x.cuda(), plan)
    with pytest.raises(ValueError):
        ska.grouped_linear(rows.cuda(), weight.cuda(), plan.offsets)
    with pytest.raises(ValueError):
        ska.grouped_linear(rows.cuda(), weight, plan.offsets.cuda())
    with pytest.raises(TypeError):
        ska.gather_rows(x.cuda().double(), plan)


# -- derivatives of derivatives -----------------------------------------------

def second_orders(device):
    """(leaf, loss) pairs whose losses hold a gradient and, beside it, a term
    that is differentiable once: the error may not be passed by."""
    for i in range(4):
        for where in (0, 1, 2):
            x, ids, weight, bias, w, dy = chain_data(device, T=20)
            leaves = [v.detach().requires_grad_(j == i)
                      for j, v in enumerate((x, weight, bias, w))]
            y = chain(leaves[0], ids, weight.shape[0], *leaves[1:])
            g, = torch.autograd.grad((y * y).sum(), leaves[i],
                                     create_graph=True)
            assert g.requires_grad
            yield leaves[i], (y.sum() + (g * g).sum(),
                              leaves[i].sum() + g.sum(),
                              y.square().sum() + g.sum())[where]


@pytest.mark.gpu
def test_second_derivatives_raise_on_the_gpu():
    for leaf, loss in second_orders("cuda"):
        with pytest.raises(RuntimeError, match="once only"):
            torch.autograd.grad(loss, leaf, retain_graph=True)
        with pytest.raises(RuntimeError, match="once only"):
            loss.backward()


@pytest.mark.gpu
def test_a_gradients_other_sources_raise_on_the_gpu():
    """A gradient is linear in the incoming one and in the saved operand; it
    raises for these and is a constant for the rest."""
    x, ids, weight, bias, w, dy = chain_data("cuda", T=20)
    plan = ska.group_rows(ids, weight.shape[0])
    rows = ska.gather_rows(x, plan).requires_grad_()
    weight.requires_grad_()
    bias.requires_grad_()
    out = ska.grouped_linear(rows, weight, plan.offsets, bias)
    drows, dweight, dbias = torch.autograd.grad(
        out.sum(), [rows, weight, bias], create_graph=True)
    for got, raises, constant in ((drows, weight, rows),
                                  (dweight, rows, weight)):
        with pytest.raises(RuntimeError, match="once only"):
            torch.autograd.grad(raises.sum() + got.sum(), raises,
                                retain_graph=True)
        plain, = torch.autograd.grad(constant.sum() + got.sum(), constant,
                                     retain_graph=True)
        assert bool((plain == 1).all())
    assert not dbias.requires_grad
    w.requires_grad_()
    y = ska.combine_rows(rows, plan, w)
    drows, dw = torch.autograd.grad(y.sum(), [rows, w], create_graph=True)
    for got, raises, constant in ((drows, w, rows), (dw, rows, w)):
        with pytest.raises(RuntimeError, match="once only"):
            torch.autograd.grad(raises.sum() + got.sum(), raises,
                                retain_graph=True)
        plain, = torch.autograd.grad(constant.sum() + got.sum(), constant,
                                     retain_graph=True)
        assert bool((plain == 1).all())


@pytest.mark.gpu
def test_gradients_are_the_same_with_a_graph_of_them():
    for i in range(2):
        x, ids, weight, bias, w, dy = chain_data("cuda", T=333)
        leaves = [v.requires_grad_() for v in (x, weight, bias, w)]
        y = chain(leaves[0], ids, weight.shape[0], *leaves[1:])
        a = torch.autograd.grad(y, leaves, dy, retain_graph=True)
        b = torch.autograd.grad(y, leaves, dy, create_graph=True)
        assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_second_derivatives_raise_on_the_cpu():
    for leaf, loss in second_orders("cpu"):
        with pytest.raises(RuntimeError, match="once only"):
            torch.autograd.grad(loss, leaf, retain_graph=True)
        with pytest.raises(RuntimeError, match="once only"):
            loss.backward()


def test_gradients_are_the_same_with_a_graph_of_them_on_the_cpu():
    x, ids, weight, bias, w, dy = chain_data("cpu", T=99)
    leaves = [v.requires_grad_() for v in (x, weight, bias, w)]
    y = chain(leaves[0], ids, weight.shape[0], *leaves[1:])
    a = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    b = torch.autograd.grad(y, leaves, dy, create_graph=True)
    assert all(torch.equal(u, v) for u, v in zip(a, b))


# -- row numbers near 2^31 ----------------------------------------------------

@pytest.mark.gpu
def test_group_rows_beyond_half_of_the_row_numbers():
    """More than 2^30 entries in more groups than one pass takes: entry i has
    the group i % G, so that its place is known."""
    M, G = (1 << 30) + 12345, 10007
    ids = torch.arange(M, dtype=torch.int32, device="cuda").remainder_(G)
    plan = ska.group_rows(ids, G)
    g = torch.arange(G + 1, device="cuda")
    offsets = g * (M // G) + g.clamp(max=M % G)
    assert torch.equal(plan.offsets, offsets.int())
    for lo in range(0, M, 1 << 28):
        i = torch.arange(lo, min(M, lo + (1 << 28)), device="cuda")
        place = offsets[i % G] + i // G
        assert torch.equal(plan.slots[lo:lo + (1 << 28)], place.int())
        assert torch.equal(plan.order[place], i.int())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16],
                         ids=SHORT.get)
def test_gradients_of_a_group_of_all_row_numbers(dtype):
    """As many rows as there may be, in one group.  Sums of ones: whole
    numbers, exact in 32 bits up to 2^24 and in fewer than 2^12 parts, each of
    whose additions is off by half a step of the sum so far, 2^-24 of it."""
    M = 2 ** 31 - 65537
    rows = torch.ones(M, 1, dtype=dtype, device="cuda")
    weight = torch.ones(1, 1, 1, dtype=dtype, device="cuda",
                        requires_grad=True)
    bias = torch.ones(1, 1, dtype=dtype, device="cuda", requires_grad=True)
    offsets = torch.tensor([0, M], dtype=torch.int32, device="cuda")
    y = ska.grouped_linear(rows, weight, offsets, bias)
    assert bool((y[-70000:] == 2).all())
    dweight, dbias = torch.autograd.grad(y, [weight, bias], rows)
    tol = M * (2.0 ** -12 + torch.finfo(dtype).eps / 2)
    assert abs(float(dweight) - M) <= tol and abs(float(dbias) - M) <= tol


# -- calls that the kernels refuse ----------------------------------------------

@pytest.mark.parametrize("device", DEVICES)
def test_forward_mode_raises(device):
    """A tangent is refused, in the inputs and in an incoming gradient: it
    would come back as none, which stands for zero."""
    import torch.autograd.forward_ad as fw

    x, ids, weight, bias, w, dy = chain_data(device, T=20)
    G = weight.shape[0]
    plan = ska.group_rows(ids, G)
    rows = ska.gather_rows(x, plan)
    out = ska.grouped_linear(rows, weight, plan.offsets, bias)
    with fw.dual_level():
        def dual(v):
            return fw.make_dual(v.detach().clone(), torch.ones_like(v))

        for call in (
                lambda: ska.gather_rows(dual(x), plan),
                lambda: ska.grouped_linear(dual(rows), weight, plan.offsets),
                lambda: ska.grouped_linear(rows, dual(weight), plan.offsets),
                lambda: ska.grouped_linear(rows, weight, plan.offsets,
                                           dual(bias)),
                lambda: ska.combine_rows(dual(out), plan, w),
                lambda: ska.combine_rows(out, plan, dual(w))):
            with pytest.raises(NotImplementedError):
                call()
        for i in range(4):
            leaves = [v.detach().requires_grad_(j == i)
                      for j, v in enumerate((x, weight, bias, w))]
            y = chain(leaves[0], ids, G, *leaves[1:])
            with pytest.raises(NotImplementedError):
                torch.autograd.grad(y, leaves[i], dual(dy))


@pytest.mark.gpu
def test_tracing_raises_on_the_gpu():
    """A trace would hold the outputs' allocations and not the kernels."""
    x, ids, weight, bias, w, dy = chain_data("cuda", T=20)
    plan = ska.group_rows(ids, weight.shape[0])
    out = ska.grouped_linear(ska.gather_rows(x, plan), weight, plan.offsets)
    for call, given in (
            (lambda v: ska.group_rows(v, 3).order, ids),
            (lambda v: ska.gather_rows(v, plan), x),
            (lambda v: ska.grouped_linear(v, weight, plan.offsets),
             ska.gather_rows(x, plan)),
            (lambda v: ska.combine_rows(v, plan), out)):
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(call, given, check_trace=False)
        call(given)


def test_tracing_on_the_cpu_follows_its_inputs():
    """The reference's calls are part of a trace."""
    x, ids, weight, bias, w, dy = chain_data("cpu", T=20)
    G = weight.shape[0]

    def run(x, ids):
        return chain(x, ids, G, weight, bias, w)

    traced = torch.jit.trace(run, (x, ids), check_trace=False)
    other = torch.as_tensor(ids_of("skewed", *ids.shape, G, seed=4))
    assert torch.equal(traced(x + 1, other), run(x + 1, other))


class Wrapped(torch.Tensor):
    """A tensor that stands for another and has no memory of its own."""

    @staticmethod
    def __new__(cls, shape, dtype):
        return torch.Tensor._make_wrapper_subclass(cls, shape, dtype=dtype,
                                                   device="cuda")

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise AssertionError(f"{func} was called")


def memoryless_calls(make):
    """Each operator with one tensor that has no memory; make(shape, dtype)
    gives one, and real(...) an ordinary one if there is a device."""
    f, i = torch.float32, torch.int32
    plan = ska.GroupPlan(make((4,), i), make((3, 2), i), make((6,), i))
    return [
        lambda: ska.group_rows(make((3, 2), i), 3),
        lambda: ska.gather_rows(make((3, 4), f), plan),
        lambda: ska.combine_rows(make((6, 4), f), plan),
        lambda: ska.combine_rows(make((6, 4), f), plan, make((3, 2), f)),
        lambda: ska.grouped_linear(make((6, 4), f), make((3, 2, 4), f),
                                   plan.offsets),
    ]


def test_refuses_tensors_without_memory():
    """Before anything else is done with them: the device is not touched,
    which this machine may not have."""
    from spark_sklearn_amd.ops import extension_available

    if not extension_available():
        pytest.skip("the extension is not built")
    for call in memoryless_calls(Wrapped):
        with pytest.raises(TypeError, match="memory"):
            call()


@pytest.mark.gpu
def test_refuses_tensors_without_memory_beside_real_ones():
    x, ids, weight, bias, w, dy = chain_data("cuda", T=20)
    plan = ska.group_rows(ids, weight.shape[0])
    rows = ska.gather_rows(x, plan)
    out = ska.grouped_linear(rows, weight, plan.offsets, bias)

    def without(t):
        return Wrapped(t.shape, t.dtype)

    def zeros(t):
        return torch._efficientzerotensor(t.shape, device="cuda")

    calls = memoryless_calls(Wrapped) + [
        lambda: ska.gather_rows(x, plan._replace(slots=without(plan.slots))),
        lambda: ska.gather_rows(x, plan._replace(
            offsets=without(plan.offsets))),
        lambda: ska.gather_rows(zeros(x), plan),
        lambda: ska.combine_rows(out, plan, without(w)),
        lambda: ska.combine_rows(out, plan, zeros(w)),
        lambda: ska.combine_rows(zeros(out), plan, w),
        lambda: ska.grouped_linear(zeros(rows), weight, plan.offsets),
        lambda: ska.grouped_linear(rows, without(weight), plan.offsets),
        lambda: ska.grouped_linear(rows, zeros(weight), plan.offsets),
        lambda: ska.grouped_linear(rows, weight, without(plan.offsets)),
        lambda: ska.grouped_linear(rows, weight, plan.offsets,
                                   without(bias)),
        lambda: ska.grouped_linear(rows, weight, plan.offsets, zeros(bias)),
    ]
    for call in calls:
        with pytest.raises(TypeError, match="memory"):
            call()


@pytest.mark.gpu
def test_refuses_under_a_mode_that_makes_fake_outputs():
    from torch._subclasses.fake_tensor import FakeTensorMode

    x, ids, weight, bias, w, dy = chain_data("cuda", T=20)
    plan = ska.group_rows(ids, weight.shape[0])
    rows = ska.gather_rows(x, plan)
    want = ska.grouped_linear(rows, weight, plan.offsets, bias)
    many = torch.zeros(5000, dtype=torch.int64, device="cuda")
    with FakeTensorMode(allow_non_fake_inputs=True):
        for call in (lambda: ska.group_rows(ids, 9),
                     lambda: ska.group_rows(many, 9),
                     lambda: ska.gather_rows(x, plan),
                     lambda: ska.combine_rows(rows, plan, w),
                     lambda: ska.grouped_linear(rows, weight, plan.offsets)):
            with pytest.raises(TypeError, match="memory"):
                call()
    with pytest.raises(TypeError, match="memory"):
        torch.func.functionalize(lambda v: ska.gather_rows(v, plan))(x)
    assert torch.equal(
        ska.grouped_linear(rows, weight, plan.offsets, bias), want)


@pytest.mark.parametrize("device", DEVICES)
def test_lazily_negated_tensors(device):
    """A tensor whose memory holds the negative of its values, as the
    imaginary part of a conjugate does: in every place, and as a gradient."""
    x, ids, weight, bias, w, dy = chain_data(device, T=20)
    G = weight.shape[0]

    def negated(v):
        out = torch._neg_view(-v)
        assert out.is_neg() and torch.equal(out, v)
        return out

    def run(make):
        leaves = [v.clone().requires_grad_() for v in (x, weight, bias, w)]
        a, b, c, d = (make(v) for v in leaves)
        plan = ska.GroupPlan(*(make(v) for v in ska.group_rows(make(ids), G)))
        out = ska.grouped_linear(ska.gather_rows(a, plan), b, plan.offsets,
                                 c)
        y = ska.combine_rows(out, plan, d)
        return [y.detach()] + list(torch.autograd.grad(y, leaves, make(dy)))

    for got, want in zip(run(negated), run(lambda v: v)):
        assert torch.equal(got, want)
    # a column of such a part, which is a matrix whose rows lie apart
    z = torch.complex(x[:, :1], dy[:, :1]).conj().imag
    assert z.is_neg()
    plan = ska.group_rows(ids, G)
    assert torch.equal(ska.gather_rows(z, plan),
                       ska.gather_rows(-dy[:, :1], plan))


# -- long sums ----------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("M,N,F", [
    (1 << 24, 1, 1), (1 << 21, 3, 65), (1 << 21, 20, 8)])
@pytest.mark.parametrize("at", [0, 12345])
def test_no_accumulator_takes_more_than_512_rows(M, N, F, at):
    """One term of 2^30 among ones: an accumulator of 32 bits that holds it
    loses what is added after it, four ones at a time.  All other partial sums
    are whole numbers of 512s below 2^25, so exact, and 2^30 and such numbers
    add exactly (the spacing there is 128): what is lost is at most the other
    511 rows of one accumulator."""
    grad = torch.ones(M, N, device="cuda")
    grad[at] = 2.0 ** 30
    rows = torch.ones(M, F, device="cuda")
    weight = torch.zeros(1, N, F, device="cuda", requires_grad=True)
    bias = torch.zeros(1, N, device="cuda", requires_grad=True)
    offsets = torch.tensor([0, M], dtype=torch.int32, device="cuda")
    y = ska.grouped_linear(rows, weight, offsets, bias)
    for got in torch.autograd.grad(y, [weight, bias], grad):
        off = (got.double() - (2.0 ** 30 + M - 1)).abs().max()
        assert float(off) <= 511
    alone, = torch.autograd.grad(
        ska.grouped_linear(rows, weight, offsets, bias), [bias], grad)
    assert float((alone.double() - (2.0 ** 30 + M - 1)).abs().max()) <= 511


@pytest.mark.gpu
def test_threads_on_streams_of_their_own_all_succeed():
    """Four threads, two for each set of inputs, forward and backward: every
    call of every thread returns, with the result it has alone."""
    from concurrent.futures import ThreadPoolExecutor

    datas = [chain_data("cuda", T=t, G=g, seed=t)
             for t, g in ((900, 7), (2600, 21))]

    def once(data):
        x, ids, weight, bias, w, dy = data
        leaves = [v.detach().requires_grad_() for v in (x, weight, bias, w)]
        y = chain(leaves[0], ids, weight.shape[0], *leaves[1:])
        return (y.detach(),) + torch.autograd.grad(y, leaves, dy)

    want = [once(d) for d in datas]
    torch.cuda.synchronize()

    def work(i):
        equal = 0
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = once(datas[i])
                torch.cuda.current_stream().synchronize()
                equal += all(torch.equal(a, b)
                             for a, b in zip(got, want[i]))
        return equal

    with ThreadPoolExecutor(4) as pool:
        # result() raises what a thread raised
        done = [pool.submit(work, i) for i in (0, 1, 0, 1)]
        assert [d.result(timeout=60) for d in done] == [20] * 4


def test_the_reference_stays_on_its_tensors_device():
    """Whatever the program's default device is."""
    x, ids, weight, bias, w, dy = chain_data("cpu", T=20)

    def run():
        leaves = [v.detach().requires_grad_() for v in (x, weight, bias, w)]
        y = chain(leaves[0], ids, weight.shape[0], *leaves[1:])
        return [y.detach()] + list(torch.autograd.grad(y, leaves, dy))

    want = run()
    with torch.device("meta"):
        got = run()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


class WrappedView(Wrapped):
    """The same as a view that begins behind its storage's first values: its
    pointer is not null."""

    @staticmethod
    def __new__(cls, shape, dtype):
        strides = [1] * len(shape)
        for i in range(len(shape) - 1, 0, -1):
            strides[i - 1] = strides[i] * shape[i]
        return torch.Tensor._make_wrapper_subclass(
            cls, shape, strides, 8, dtype=dtype, device="cuda")


def test_refuses_views_without_memory():
    from spark_sklearn_amd.ops import extension_available

    if not extension_available():
        pytest.skip("the extension is not built")
    for call in memoryless_calls(WrappedView):
        with pytest.raises(TypeError, match="memory"):
            call()


@pytest.mark.gpu
@pytest.mark.parametrize("left", [0, 64])
def test_refuses_tensors_whose_storage_was_given_back(left):
    """A storage made smaller than the tensor (all of it, or all but 64
    bytes), as freed parameters have; the tensor itself and a view."""
    x, ids, weight, bias, w, dy = chain_data("cuda", T=20)
    plan = ska.group_rows(ids, weight.shape[0])
    rows = ska.gather_rows(x, plan)
    out = ska.grouped_linear(rows, weight, plan.offsets, bias)

    def freed(v, view):
        if view:
            v = torch.cat([v.reshape(-1)[:8], v.reshape(-1)])[8:].view(
                v.shape)
        else:
            v = v.clone()
        v.untyped_storage().resize_(left)
        return v

    for view in (False, True):
        for call in (
                lambda: ska.group_rows(freed(ids, view), 9),
                lambda: ska.gather_rows(freed(x, view), plan),
                lambda: ska.gather_rows(x, plan._replace(
                    slots=freed(plan.slots, view))),
                lambda: ska.combine_rows(freed(out, view), plan, w),
                lambda: ska.combine_rows(out, plan, freed(w, view)),
                lambda: ska.grouped_linear(freed(rows, view), weight,
                                           plan.offsets),
                lambda: ska.grouped_linear(rows, freed(weight, view),
                                           plan.offsets),
                lambda: ska.grouped_linear(rows, weight, plan.offsets,
                                           freed(bias, view))):
            with pytest.raises(TypeError, match="memory"):
                call()


@pytest.mark.gpu
def test_refuses_meta_tensors_the_same_on_the_gpu():
    """Beside tensors of either device they are on another one: ValueError."""
    ids, plan, x, rows, weight = small()
    bias, w = torch.ones(3, 2), torch.ones(3, 2)

    def meta(v):
        return v.to("meta")

    for c in (lambda v: v, lambda v: v.cuda()):
        p = ska.GroupPlan(*(c(v) for v in plan))
        for call in (
                lambda: ska.gather_rows(c(x), p._replace(
                    slots=meta(p.slots))),
                lambda: ska.gather_rows(c(x), p._replace(
                    offsets=meta(p.offsets))),
                lambda: ska.combine_rows(c(rows), p, meta(w)),
                lambda: ska.grouped_linear(c(rows), meta(weight), p.offsets),
                lambda: ska.grouped_linear(c(rows), c(weight),
                                           meta(p.offsets)),
                lambda: ska.grouped_linear(c(rows), c(weight), p.offsets,
                                           meta(bias))):
            with pytest.raises(ValueError):
                call()
