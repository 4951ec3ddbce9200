"""Cases that measure the grouped-row operators.

Rows that belong to groups (the keys of a keyed model, the experts of a
routed layer) are sorted by group, multiplied by their own group's weights
and put back in row order:

    group_rows      ids -> offsets, slots, order         (a stable sort)
    gather_rows     rows into group order                (and its gradient)
    grouped_linear  each run of rows times its weights   (and its gradients)
    combine_rows    back to row order, weighted          (and its gradients)

``run`` computes them with elementary torch operations in 32 bits, or, where
``own`` is true, through spark_sklearn_amd's entry points.
"""

import math

import numpy as np
import torch

own = False

_TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16,
          "float16": torch.float16}


def _case(op, dtype, rows, k, groups, features, outputs=0, train=False,
          wrt="all", skew=0.0, dropped=0.0, weights="", index="int32",
          name=None):
    """op: dispatch (group_rows + gather_rows), combine, linear, or chain (all
    of them).  wrt: "all" gradients, or those of the "weights" alone (rows
    that are data and not activations).  skew: exponent of the groups'
    shares.  dropped: share of entries that belong to no group."""
    case = dict(op=op, dtype=dtype, rows=rows, k=k, groups=groups,
                features=features, outputs=outputs, train=train, wrt=wrt,
                skew=skew, dropped=dropped, weights=weights, index=index)
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # one row on its way to two of 64 groups: nothing but latency
        _case("dispatch", "bfloat16", 1, 2, 64, 256, name="dispatch_1"),
        # a million-row data matrix laid out by key before a keyed fit, ids
        # as pandas gives them, popular keys and rows whose key is unknown
        _case("dispatch", "float32", 1000000, 1, 4096, 256, skew=0.8,
              dropped=0.01, index="int64", name="dispatch_1M"),
        # activations to two of 60 experts, forward and backward
        _case("dispatch", "bfloat16", 12289, 2, 60, 1032, train=True,
              skew=0.5, name="dispatch_train"),
        # a prompt's rows back from four of 128 experts
        _case("combine", "bfloat16", 16384, 4, 128, 2048, weights="bfloat16",
              skew=0.5, name="combine_16k"),
        # the same in training, at an odd width and with dropped entries
        _case("combine", "float16", 8191, 2, 33, 1001, train=True,
              weights="float32", skew=0.5, dropped=0.05,
              name="combine_train"),
        # eight rows of a serving step, each with another of 64 experts
        _case("linear", "bfloat16", 8, 1, 64, 2048, 2048, name="linear_8"),
        # scoring a million rows with their keys' 10-class models
        _case("linear", "float32", 1000000, 1, 1000, 256, 10, skew=0.6,
              dropped=0.01, name="linear_score_1M"),
        # one epoch's products of a keyed fit; the rows are data
        _case("linear", "float32", 400003, 1, 512, 256, 3, train=True,
              wrt="weights", skew=0.6, name="linear_fit_400k"),
        # small ragged groups at odd sizes, all gradients
        _case("linear", "float16", 5003, 1, 37, 250, 131, train=True,
              skew=0.7, dropped=0.02, name="linear_odd_train"),
        # a long prompt's rows through an expert's projection
        _case("linear", "bfloat16", 65536, 1, 64, 2048, 1024, skew=0.4,
              name="linear_64k"),
        # the largest: a training step's projection, all gradients
        _case("linear", "bfloat16", 65536, 1, 32, 1024, 4096, train=True,
              skew=0.4, name="linear_64k_train"),
        # sort, gather, product and weighted sum as they are used together
        _case("chain", "bfloat16", 4099, 2, 48, 768, 768, train=True,
              weights="bfloat16", skew=0.5, dropped=0.02,
              name="chain_train"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _size(rng, low, high):
    """Half of the sizes are whole multiples of 8, the others fall anywhere."""
    n = _log(rng, low, high)
    return max(8, n // 8 * 8) if rng.random() < 0.5 else n


def draw(rng):
    op = rng.choice(["dispatch", "combine", "linear", "linear", "chain"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    k = 1 if op == "linear" else rng.choice([1, 2, 2, 3, 4, 8])
    groups = _log(rng, 2, 4096)
    skew = rng.choice([0.0, 0.4, 0.8])
    dropped = rng.choice([0.0, 0.0, 0.03])
    train = rng.random() < 0.5
    weights = rng.choice([dtype, "float32"])
    index = rng.choice(["int32", "int64"])
    features = _size(rng, 16, 2048)
    outputs = 0
    if op in ("linear", "chain"):
        outputs = _size(rng, 1, 4096)
        # weights of all groups stay within half a billion values
        while groups * features * outputs > 1 << 29:
            groups = max(2, groups // 2)
            outputs = max(1, outputs // 2)
        rows = _log(rng, 1, 65536)
        if op == "chain":
            rows = max(1, rows // k)
            weights = dtype
        while rows * k * features * outputs > 1 << 38:
            rows //= 2
    else:
        rows = max(1, _log(rng, 1, 1 << 20) // k)
        while rows * k * features > 1 << 28:
            rows //= 2
    wrt = rng.choice(["all", "weights"]) if op == "linear" else "all"
    return _case(op, dtype, rows, k, groups, features, outputs, train, wrt,
                 skew, dropped, weights if op in ("combine", "chain") else "",
                 index)


def _sorted_plan(ids, groups):
    """offsets [groups + 1], slots (like ids) and order of the stable sort by
    group; ids outside the groups come last and count nowhere."""
    flat = ids.reshape(-1)
    key = torch.where((flat >= 0) & (flat < groups), flat, groups).long()
    ranked, order = torch.sort(key, stable=True)
    slots = torch.empty_like(order)
    slots[order] = torch.arange(order.numel(), device=order.device)
    offsets = torch.searchsorted(
        ranked, torch.arange(groups + 1, device=ids.device))
    return (offsets.int(), slots.int().reshape(ids.shape), order.int())


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed * 1000003 + 17)
    dtype = _TYPES[case["dtype"]]
    t, k, g = case["rows"], case["k"], case["groups"]
    f, n = case["features"], case["outputs"]

    def normal(*shape, scale=1.0, to=dtype):
        return (torch.randn(*shape, device=dev, generator=gen)
                * scale).to(to)

    share = torch.arange(1, g + 1, device=dev,
                         dtype=torch.float64) ** -case["skew"]
    share = share[torch.randperm(g, device=dev, generator=gen)]
    edges = torch.cumsum(share, 0) / share.sum()
    pick = torch.rand(t, k, device=dev, generator=gen, dtype=torch.float64)
    ids = torch.searchsorted(edges, pick).clamp_(max=g - 1)
    if case["dropped"]:
        lost = torch.rand(t, k, device=dev, generator=gen) < case["dropped"]
        ids = torch.where(lost, -1, ids)
    ids = ids.to(getattr(torch, case["index"]))
    state = {"case": case}
    op, train = case["op"], case["train"]
    if op in ("dispatch", "chain"):
        state["ids"] = ids
        state["x"] = normal(t, f).requires_grad_(train)
    if op == "dispatch" and train:
        state["grad"] = normal(t * k, f)
    if op in ("combine", "linear"):
        offsets, slots, order = _sorted_plan(ids, g)
        state["offsets"] = offsets
        state["rows"] = normal(t * k, f).requires_grad_(
            train and case["wrt"] == "all")
    if op == "combine":
        state["slots"], state["order"] = slots, order
        state["grad"] = normal(t, f)
    if op in ("combine", "chain"):
        w = torch.rand(t, k, device=dev, generator=gen) + 0.05
        w = (w / w.sum(1, keepdim=True)).to(_TYPES[case["weights"]])
        state["weights"] = w.requires_grad_(train)
    if op in ("linear", "chain"):
        state["weight"] = normal(g, n, f, scale=f ** -0.5).requires_grad_(
            train)
        state["bias"] = normal(g, n).requires_grad_(train)
        state["grad"] = normal(t, n)
    return state


# -- the plain form ----------------------------------------------------------

def _blocks(offsets, m, step):
    """Splits each group's run of rows into blocks of `step` rows: the block's
    group, its rows' indices, and which of them are the group's."""
    g = offsets.numel() - 1
    start = offsets.long()
    counts = start[1:] - start[:-1]
    per = (counts + step - 1) // step
    ends = torch.cumsum(per, 0)
    block = torch.arange(min(m, m // step + g), device=offsets.device)
    group = torch.searchsorted(ends, block, right=True)
    used = group < g
    group = group.clamp(max=g - 1)
    first = start[group] + (block - ends[group] + per[group]) * step
    index = first[:, None] + torch.arange(step, device=offsets.device)
    mine = used[:, None] & (index < start[group + 1][:, None])
    return group, torch.where(mine, index, m), mine


def _step(m, groups):
    return 1 << max(0, min(7, (m // groups).bit_length()))


def _plain_linear(rows, weight, bias, offsets, grad, wrt):
    """y, and with `grad` the gradients, all in 32 bits."""
    m, (g, n, f) = rows.shape[0], weight.shape
    group, index, mine = _blocks(offsets, m, _step(m, g))
    some = index.clamp(max=max(m - 1, 0))
    x = rows.float()[some] * mine[..., None]
    w = weight.float()[group]
    y = rows.new_zeros(m + 1, n, dtype=torch.float32)
    y[index] = (torch.bmm(x, w.transpose(1, 2)) + bias.float()[group][:, None]
                ) * mine[..., None]
    if grad is None:
        return (y[:m],)
    dy = grad.float()[some] * mine[..., None]
    dw = torch.zeros(g, n, f, device=rows.device)
    dw.index_add_(0, group, torch.bmm(dy.transpose(1, 2), x))
    db = torch.zeros(g, n, device=rows.device)
    db.index_add_(0, group, dy.sum(1))
    if wrt == "weights":
        return y[:m], dw, db
    dx = rows.new_zeros(m + 1, f, dtype=torch.float32)
    dx[index] = torch.bmm(dy, w)
    return y[:m], dx[:m], dw, db


def _plain_gather(x, order, offsets, k):
    kept = torch.arange(order.numel(), device=x.device) < offsets[-1]
    return x[order.long() // k] * kept[:, None]


def _plain_combine(rows, slots, offsets, weights):
    kept = (slots < offsets[-1])[..., None]
    taken = torch.where(kept, rows[slots.long()], 0.0)
    return taken if weights is None else taken * weights[..., None]


def _plain(state):
    case = state["case"]
    dtype, k = _TYPES[case["dtype"]], case["k"]
    grad = state.get("grad") if case["train"] else None
    if case["op"] == "linear":
        out = _plain_linear(state["rows"], state["weight"], state["bias"],
                            state["offsets"], grad, case["wrt"])
        return tuple(v.to(dtype) for v in out)
    if case["op"] == "combine":
        rows, w = state["rows"].float(), state["weights"].float()
        slots, offsets = state["slots"], state["offsets"]
        y = _plain_combine(rows, slots, offsets, w).sum(1)
        if grad is None:
            return (y.to(dtype),)
        dy = grad.float()
        drows = (_plain_gather(dy, state["order"], offsets, k)
                 * w.reshape(-1)[state["order"].long()][:, None])
        dw = (_plain_combine(rows, slots, offsets, None)
              * dy[:, None]).sum(-1)
        return (y.to(dtype), drows.to(dtype),
                dw.to(_TYPES[case["weights"]]))
    offsets, slots, order = _sorted_plan(state["ids"], case["groups"])
    x = state["x"].float()
    rows = _plain_gather(x, order, offsets, k)
    if case["op"] == "dispatch":
        out = (offsets, slots, order, rows.to(dtype))
        if grad is None:
            return out
        dx = _plain_combine(grad.float(), slots, offsets, None).sum(1)
        return out + (dx.to(dtype),)
    w = state["weights"].float()
    if grad is None:
        (ys,) = _plain_linear(rows, state["weight"], state["bias"], offsets,
                              None, "all")
        return (_plain_combine(ys, slots, offsets, w).sum(1).to(dtype),)
    dy = grad.float()
    dys = (_plain_gather(dy, order, offsets, k)
           * w.reshape(-1)[order.long()][:, None])
    ys, drows, dweight, dbias = _plain_linear(
        rows, state["weight"], state["bias"], offsets, dys, "all")
    y = _plain_combine(ys, slots, offsets, w).sum(1)
    dw = (_plain_combine(ys, slots, offsets, None) * dy[:, None]).sum(-1)
    dx = _plain_combine(drows, slots, offsets, None).sum(1)
    return tuple(v.to(dtype) for v in (y, dx, dweight, dbias, dw))


# -- the framework's operators -----------------------------------------------

def _own(state):
    import spark_sklearn_amd as ska

    case = state["case"]
    grad = state.get("grad") if case["train"] else None
    if case["op"] == "linear":
        y = ska.grouped_linear(state["rows"], state["weight"],
                               state["offsets"], state["bias"])
        leaves = [state["rows"]] if case["wrt"] == "all" else []
        leaves += [state["weight"], state["bias"]]
        head = (y.detach(),)
    elif case["op"] == "combine":
        plan = ska.GroupPlan(state["offsets"], state["slots"],
                             state["order"])
        y = ska.combine_rows(state["rows"], plan, state["weights"])
        leaves = [state["rows"], state["weights"]]
        head = (y.detach(),)
    elif case["op"] == "dispatch":
        plan = ska.group_rows(state["ids"], case["groups"])
        y = ska.gather_rows(state["x"], plan)
        leaves = [state["x"]]
        head = (plan.offsets, plan.slots, plan.order, y.detach())
    else:
        plan = ska.group_rows(state["ids"], case["groups"])
        rows = ska.gather_rows(state["x"], plan)
        rows = ska.grouped_linear(rows, state["weight"], plan.offsets,
                                  state["bias"])
        y = ska.combine_rows(rows, plan, state["weights"])
        leaves = [state["x"], state["weight"], state["bias"],
                  state["weights"]]
        head = (y.detach(),)
    if grad is None:
        return head
    return head + torch.autograd.grad(y, leaves, grad)


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _plain(state)


# -- what a pass cannot do without -------------------------------------------

def work(case):
    e = 4 if case["dtype"] == "float32" else 2
    t, k, f, n = (case[v] for v in ("rows", "k", "features", "outputs"))
    m, g = t * k, case["groups"]
    train = case["train"]
    we = 4 if case["weights"] == "float32" else 2
    ints = m * (12 if case["index"] == "int32" else 16) + 4 * (g + 1)
    if case["op"] == "dispatch":
        move = (t + m) * f * e
        return {"bytes": ints + move * (2 if train else 1),
                "flops": m * f if train else 0}
    if case["op"] == "combine":
        fwd = (t + m) * f * e + m * (4 + we)
        bwd = (t + m) * f * e + m * we
        return {"bytes": fwd + (bwd if train else 0),
                "flops": 2 * m * f * (3 if train else 1)}
    products = 1
    if train:
        products = 3 if case["wrt"] == "all" else 2
    used = min(g, m)
    if case["op"] == "linear":
        size = m * (f + n) + used * n * (f + 1)
        if train:
            size += m * n + g * n * (f + 1)
            size += m * f if case["wrt"] == "all" else 0
        return {"bytes": size * e + 4 * (g + 1),
                "flops": 2 * m * n * f * products}
    size = t * (f + n) + used * n * (f + 1)
    if train:
        size += t * (f + n) + g * n * (f + 1)
    return {"bytes": size * e + m * we * (2 if train else 1)
            + m * (4 if case["index"] == "int32" else 8),
            "flops": 2 * m * n * f * products + 2 * m * n}


# -- the definition in 64 bits -----------------------------------------------

def _exact_plan(ids, groups):
    flat = ids.detach().cpu().numpy().astype(np.int64).ravel()
    flat = np.where((flat < 0) | (flat >= groups), groups, flat)
    order = np.argsort(flat, kind="stable")
    slots = np.empty_like(order)
    slots[order] = np.arange(order.size)
    offsets = np.concatenate(
        [[0], np.cumsum(np.bincount(flat, minlength=groups + 1))[:groups]])
    return offsets, slots.reshape(tuple(ids.shape)), order


def _exact_linear(rows, weight, bias, offsets, grad):
    y = torch.zeros(rows.shape[0], weight.shape[1], dtype=torch.float64,
                    device=rows.device)
    dx, dw, db = (torch.zeros_like(v, dtype=torch.float64)
                  for v in (rows, weight, bias))
    edges = [int(v) for v in offsets]
    for i, (a, b) in enumerate(zip(edges[:-1], edges[1:])):
        if a == b:
            continue
        w = weight[i].double()
        y[a:b] = rows[a:b].double() @ w.t() + bias[i].double()
        if grad is not None:
            d = grad[a:b].double()
            dx[a:b] = d @ w
            dw[i] = d.t() @ rows[a:b].double()
            db[i] = d.sum(0)
    return y, dx, dw, db


def exact(case, seed):
    with torch.no_grad():
        return _exact(case, prepare(case, seed))


def _exact(case, state):
    grad = state.get("grad") if case["train"] else None
    t, k = case["rows"], case["k"]
    if case["op"] == "linear":
        y, dx, dw, db = _exact_linear(
            state["rows"], state["weight"], state["bias"], state["offsets"],
            grad)
        if grad is None:
            return (y,)
        return (y, dx, dw, db) if case["wrt"] == "all" else (y, dw, db)
    dev = (state["x"] if "x" in state else state["rows"]).device
    if case["op"] == "combine":
        offsets, slots = state["offsets"].cpu().numpy(), state["slots"]
        slots = slots.cpu().numpy()
    else:
        offsets, slots, order = _exact_plan(state["ids"], case["groups"])
    where = torch.as_tensor(slots.astype(np.int64), device=dev).reshape(t, k)
    kept = where < int(offsets[-1])

    def spread(v, scale=None):
        """Row t of v to the slots of its kept entries, scaled."""
        out = torch.zeros(t * k, v.shape[1], dtype=torch.float64, device=dev)
        for j in range(k):
            at = kept[:, j].nonzero().squeeze(1)
            part = v[at].double()
            if scale is not None:
                part = part * scale[at, j].double()[:, None]
            out[where[at, j]] = part
        return out

    def collect(v, scale=None):
        """The kept entries' rows of v summed for each t, scaled."""
        out = torch.zeros(t, v.shape[1], dtype=torch.float64, device=dev)
        for j in range(k):
            at = kept[:, j].nonzero().squeeze(1)
            part = v[where[at, j]].double()
            if scale is not None:
                part = part * scale[at, j].double()[:, None]
            out[at] += part
        return out

    def dots(v, d):
        out = torch.zeros(t, k, dtype=torch.float64, device=dev)
        for j in range(k):
            at = kept[:, j].nonzero().squeeze(1)
            out[at, j] = (v[where[at, j]].double() * d[at].double()).sum(1)
        return out

    if case["op"] == "combine":
        y = collect(state["rows"], state["weights"])
        if grad is None:
            return (y,)
        return (y, spread(grad, state["weights"]),
                dots(state["rows"], grad))
    rows = spread(state["x"])
    if case["op"] == "dispatch":
        ints = tuple(torch.as_tensor(v.astype(np.int32), device=dev)
                     for v in (offsets, slots, order))
        return ints + ((rows,) if grad is None else (rows, collect(grad)))
    d = None if grad is None else spread(grad, state["weights"])
    ys, drows, dweight, dbias = _exact_linear(
        rows, state["weight"], state["bias"], offsets, d)
    y = collect(ys, state["weights"])
    if grad is None:
        return (y,)
    return y, collect(drows), dweight, dbias, dots(ys, grad)
