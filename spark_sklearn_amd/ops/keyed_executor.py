"""Per-key linear models through the grouped-row operators.

The other batched form of a keyed fit makes every key a column of one launch,
in which each column reads the rows of all keys.  Here the rows are sorted by
key once, and an epoch multiplies each key's rows by that key's weights alone:
an epoch reads the matrix twice whatever the number of keys.  The matrix stays
in float32, so that a fit follows the reference solver's steps
(``models/_solver_ref.py``) to float32 rounding.
"""

from __future__ import annotations

import numpy as np

from ..grouped_rows import (_kernels, combine_rows, gather_rows, group_rows,
                            grouped_linear)

__all__ = ["KeyedLinearExecutor", "keyed_scores"]


def _tensor(array, dtype):
    """On the CPU, whatever the program's default device is; a copy only if
    the array is not writable, of another type or not contiguous."""
    import torch

    array = np.ascontiguousarray(array, dtype)
    return torch.from_numpy(array if array.flags.writeable
                            else array.copy())


def _sums(values, offsets):
    """The sum of each group's run of rows [G, C]."""
    _, total = _kernels(values).grouped_linear_dweight(
        values, values, offsets, False, True)
    return total


class KeyedLinearExecutor:
    """Fits one linear model a key, all keys at once."""

    def __init__(self, X, y, row_key, n_keys, device=None):
        import torch

        self.torch = torch
        self.device = torch.device("cpu") if device is None else device
        self.n_keys = n_keys
        ids = _tensor(row_key, np.int64).to(self.device)
        self.plan = group_rows(ids, n_keys)
        x = _tensor(X, np.float32)
        self.rows = gather_rows(x.to(self.device), self.plan)
        self.y = gather_rows(
            _tensor(y, np.float32)[:, None].to(self.device), self.plan)
        counts = np.bincount(row_key, minlength=n_keys)
        self.counts = counts
        sq = np.sum(np.asarray(X, np.float32).astype(np.float64) ** 2, axis=1)
        self.msq = np.bincount(row_key, weights=sq, minlength=n_keys) \
            / np.maximum(counts, 1)

    def fit(self, specs, n_classes):
        """``specs``: one column spec a key.  Returns W [G, C, F], b [G, C],
        n_iter [G, C]."""
        from ..models._solver_ref import LOSS_HINGE, LOSS_LOGISTIC

        torch = self.torch
        G, F = self.n_keys, self.rows.shape[1]
        C = n_classes if n_classes > 2 else 1
        offsets, rows = self.plan.offsets, self.rows

        def per_key(name, dtype=torch.float32):
            return torch.tensor([s[name] for s in specs], dtype=dtype,
                                device=self.device)[:, None]

        lr, l1, l2 = (per_key(v) for v in ("lr", "l1", "l2"))
        momentum, tol = per_key("momentum"), per_key("tol")
        limit = per_key("max_iter", torch.int32)
        intercept = per_key("fit_intercept")
        inv_n = _tensor(1.0 / np.maximum(self.counts, 1), np.float32).to(
            self.device)[:, None]
        loss = specs[0]["loss"]
        if n_classes:
            target = torch.arange(C, device=self.device) if C > 1 else \
                torch.ones(1, device=self.device)
            hit = self.y == target
            t = hit.float() if loss == LOSS_LOGISTIC else \
                torch.where(hit, 1.0, -1.0).float()
        else:
            t = self.y

        # the types are said, since the program may have other defaults
        W = torch.zeros(G, C, F, dtype=torch.float32, device=self.device)
        b = torch.zeros(G, C, dtype=torch.float32, device=self.device)
        V, Vb = torch.zeros_like(W), torch.zeros_like(b)
        active = torch.ones(G, C, dtype=torch.bool, device=self.device)
        prev = torch.full((G, C), float("inf"), dtype=torch.float32,
                          device=self.device)
        n_iter = torch.zeros(G, C, dtype=torch.int32, device=self.device)
        k = _kernels(rows)
        for epoch in range(int(max(s["max_iter"] for s in specs))):
            z = k.grouped_linear(rows, W, offsets, b)
            if loss == LOSS_LOGISTIC:
                p = 1.0 / (1.0 + torch.exp(-z))
                d = p - t
                le = -(t * torch.log(p + 1e-12)
                       + (1 - t) * torch.log(1 - p + 1e-12))
            elif loss == LOSS_HINGE:
                margin = t * z
                d = torch.where(margin < 1.0, -t, 0.0)
                le = (1.0 - margin).clamp_min(0.0)
            else:
                d = z - t
                le = 0.5 * d * d
            cur = _sums(le, offsets) * inv_n
            now = active & (epoch < limit)
            n_iter = torch.where(now, epoch + 1, n_iter)
            g, gb = k.grouped_linear_dweight(d, rows, offsets, True, True)
            g = g * inv_n[..., None] + l2[..., None] * W \
                + l1[..., None] * torch.sign(W)
            gb = gb * inv_n * intercept
            # a column that has converged keeps its weights and momentum
            V = torch.where(now[..., None],
                            momentum[..., None] * V - lr[..., None] * g, V)
            Vb = torch.where(now, momentum * Vb - lr * gb, Vb)
            W = W + V * now[..., None]
            b = b + Vb * now
            done = (prev - cur).abs() <= tol * cur.clamp_min(1.0)
            active = active & ~(done & now)
            prev = torch.where(now, cur, prev)
            # the host looks now and then only: frozen columns do not move
            if epoch % 32 == 31 and not bool(active.any()):
                break
        return (W.cpu().numpy(), b.cpu().numpy(), n_iter.cpu().numpy())


def keyed_scores(X, row_key, coef, intercept, device):
    """Each row's scores [n, C] under its own key's ``coef`` [G, C, F] and
    ``intercept`` [G, C]; a row whose key is outside the models scores 0."""
    x = _tensor(X, np.float32).to(device)
    ids = _tensor(row_key, np.int64).to(device)
    w = _tensor(coef, np.float32).to(device)
    b = _tensor(intercept, np.float32).to(device)
    plan = group_rows(ids, w.shape[0])
    out = grouped_linear(gather_rows(x, plan), w, plan.offsets, b)
    return combine_rows(out, plan).cpu().numpy()
