"""Reference grouped-row operators (torch on the CPU).

Defines the semantics of the kernels in ``ops/csrc/ska_grouped.hip``; the
CPU tier of :mod:`spark_sklearn_amd.grouped_rows` runs it directly.

M = T * k entries, entry ``t * k + j`` with the group ``ids[t, j]``; an id
outside ``[0, n_groups)`` belongs to no group:

  offsets[g]           entries with a group below g
  slots[t, j]          place of the entry in the stable sort by group, the
                       entries without a group last; order is its inverse
  rows[slots[t, j]]  = x[t], 0 where slots[t, j] >= offsets[G]
  y[t]               = sum over kept j of w[t, j] * rows[slots[t, j]]
  out[s]             = weight[g] @ rows[s] + bias[g] for
                       offsets[g] <= s < offsets[g + 1], 0 behind the last

Sums are held in 32 bits (64 for float64) and rounded once.
"""

from __future__ import annotations

import torch

__all__ = ["group_rows_ref", "gather_rows_ref", "combine_rows_ref",
           "combine_rows_backward_ref", "grouped_linear_ref",
           "grouped_linear_drows_ref", "grouped_linear_dweight_ref"]


def _wide(t):
    return t if t.dtype == torch.float64 else t.float()


def _runs(offsets):
    edges = offsets.tolist()
    return [(g, a, b) for g, (a, b) in enumerate(zip(edges, edges[1:]))
            if a < b]


def group_rows_ref(ids, n_groups):
    flat = ids.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < n_groups), flat, n_groups)
    ranked, order = torch.sort(key, stable=True)
    slots = torch.empty_like(order)
    slots[order] = torch.arange(order.numel(), device=ids.device)
    offsets = torch.searchsorted(
        ranked, torch.arange(n_groups + 1, device=ids.device))
    return offsets.int(), slots.int().reshape(ids.shape), order.int()


def gather_rows_ref(x, offsets, slots):
    T, k = slots.shape
    out = x.new_empty(T * k, x.shape[1])
    out[slots.long().reshape(-1)] = x.repeat_interleave(k, 0)
    out[int(offsets[-1]):] = 0
    return out


def _kept(rows, offsets, slots):
    """The rows of the kept entries [T, k, F], zero for the others."""
    kept = (slots < offsets[-1])[..., None]
    picked = _wide(rows)[slots.long()]
    return torch.where(kept, picked, picked.new_zeros(()))


def combine_rows_ref(rows, offsets, slots, weights):
    kept = _kept(rows, offsets, slots)
    if weights is not None:
        w = torch.where(slots < offsets[-1], weights, 0).to(kept.dtype)
        kept = kept * w[..., None]
    return kept.sum(1).to(rows.dtype)


def combine_rows_backward_ref(dy, rows, offsets, slots, weights, need_rows,
                              need_weights):
    T, k = slots.shape
    d = _wide(dy)
    drows = dw = None
    if need_rows:
        spread = d[:, None].expand(T, k, d.shape[1])
        if weights is not None:
            spread = spread * weights.to(d.dtype)[..., None]
        drows = dy.new_empty(T * k, dy.shape[1])
        drows[slots.long().reshape(-1)] = spread.reshape(
            T * k, dy.shape[1]).to(dy.dtype)
        drows[int(offsets[-1]):] = 0
    if need_weights:
        dot = (_kept(rows, offsets, slots) * d[:, None]).sum(-1)
        dw = torch.where(slots < offsets[-1], dot, 0).to(weights.dtype)
    return drows, dw


def grouped_linear_ref(rows, weight, offsets, bias):
    out = rows.new_zeros(rows.shape[0], weight.shape[1])
    for g, a, b in _runs(offsets):
        y = _wide(rows[a:b]) @ _wide(weight[g]).t()
        if bias is not None:
            y = y + _wide(bias[g])
        out[a:b] = y.to(rows.dtype)
    return out


def grouped_linear_drows_ref(dy, weight, offsets):
    out = dy.new_zeros(dy.shape[0], weight.shape[2])
    for g, a, b in _runs(offsets):
        out[a:b] = (_wide(dy[a:b]) @ _wide(weight[g])).to(dy.dtype)
    return out


def grouped_linear_dweight_ref(dy, rows, offsets, need_weight, need_bias):
    G = offsets.numel() - 1
    dw = dy.new_zeros(G, dy.shape[1], rows.shape[1]) if need_weight else None
    db = dy.new_zeros(G, dy.shape[1]) if need_bias else None
    for g, a, b in _runs(offsets):
        d = _wide(dy[a:b])
        if need_weight:
            dw[g] = (d.t() @ _wide(rows[a:b])).to(dy.dtype)
        if need_bias:
            db[g] = d.sum(0).to(dy.dtype)
    return dw, db
