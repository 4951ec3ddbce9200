"""Rows in groups: sort by group, per-group products, and back.

The device form of what ``gapply`` and ``KeyedModel`` do one group at a time
on the host (reference ``group_apply.py`` ~L20 and ``keyed_models.py`` ~L300
[R]): every row belongs to a group -- the key of a keyed model, the expert
of a routed layer -- and each group has its own weights.

>>> import torch
>>> from spark_sklearn_amd import (combine_rows, gather_rows, group_rows,
...                                grouped_linear)
>>> ids = torch.tensor([1, 0, 1])                  # row -> group
>>> x = torch.tensor([[1., 2.], [3., 4.], [5., 6.]])
>>> weight = torch.tensor([[[1., 0.]], [[0., 1.]]])        # [G, N, F]
>>> plan = group_rows(ids, n_groups=2)
>>> rows = gather_rows(x, plan)                    # in group order
>>> out = grouped_linear(rows, weight, plan.offsets)
>>> combine_rows(out, plan).tolist()               # in row order again
[[2.0], [3.0], [6.0]]

GPU tensors (float32, bfloat16, float16) run the kernels of
``ops/csrc/ska_grouped.hip``; CPU tensors (float64 too) run
``models/_grouped_ref.py``, which defines their semantics.  Everything is
enqueued on the current stream of the tensors' device, nothing waits for the
host, and results do not change from run to run.  All calls can be captured
into a HIP graph.  As for any torch operation, a backward pass is captured
only while no eager autograd graph of the same leaves is alive.
"""

from __future__ import annotations

from typing import Any, NamedTuple, Optional

__all__ = ["GroupPlan", "group_rows", "gather_rows", "combine_rows",
           "grouped_linear"]

_MAX_GROUPS = (1 << 24) - 1
_NO_PLAN = "plan must be a GroupPlan (see group_rows)"
_MAX_WIDTH = (1 << 21) - 1
_reference: Any = None
_ext: Any = None


class GroupPlan(NamedTuple):
    """Where each row goes: the result of :func:`group_rows`.

    offsets : int32 [n_groups + 1]; group g's rows are
        ``offsets[g] : offsets[g + 1]`` in group order, and
        ``offsets[n_groups]`` entries belong to a group at all.
    slots : int32, shaped like the ids; the place of each entry in group
        order.  Entries without a group come behind all others.
    order : int32 [ids.numel()]; the entry at each place.
    """

    offsets: Any
    slots: Any
    order: Any


def _require(ok: bool, error, message: str):
    if not ok:
        raise error(message)


def _is_tensor(t):
    import torch

    return isinstance(t, torch.Tensor)


def _check_rows(name, t):
    import torch

    _require(_is_tensor(t), TypeError, f"{name} must be a torch.Tensor")
    allowed = (torch.float64, torch.float32, torch.bfloat16, torch.float16)
    _require(t.device.type == "cpu", ValueError,
             f"{name} must be on a GPU or the CPU, got {t.device}")
    _require(t.dtype in allowed, TypeError,
             f"{name} must be one of {allowed}, got {t.dtype}")
    _require(t.dim() == 2, ValueError,
             f"{name} must be a matrix, got shape {tuple(t.shape)}")
    _require(t.shape[1] <= _MAX_WIDTH, ValueError,
             f"{name} must have at most {_MAX_WIDTH} columns")
    _require(t.shape[0] < (1 << 31) - (1 << 16), ValueError,
             f"{name} has too many rows")


def _check_ints(name, t, device, dim=None):
    import torch

    _require(_is_tensor(t), TypeError, f"{name} must be a torch.Tensor")
    _require(t.dtype == torch.int32, TypeError,
             f"{name} must be int32, got {t.dtype}")
    _require(t.device == device, ValueError,
             f"{name} is on {t.device}, the rows are on {device}")
    _require(dim is None or t.dim() == dim, ValueError,
             f"{name} must have {dim} dimensions, got {t.dim()}")


def _check_plan(plan, device):
    _check_ints("plan.offsets", plan.offsets, device, 1)
    _check_ints("plan.slots", plan.slots, device)
    _require(plan.offsets.numel() >= 2, ValueError,
             "plan.offsets must have n_groups + 1 values")
    _require(plan.slots.dim() in (1, 2), ValueError,
             "plan.slots must have one or two dimensions")
    slots = plan.slots
    if slots.dim() == 1:
        slots = slots[:, None]
    return plan.offsets.contiguous(), slots.contiguous()


def _native(t):
    """The kernels, where the tensor is on a GPU.  They make the checks that
    are made here for the reference, with the same exceptions."""
    global _ext
    if getattr(t, "is_cuda", False):
        if _ext is None:
            from .ops import load_extension

            _ext = load_extension()
        return _ext
    return None


def _kernels(t):
    """The functions that serve the tensor, each with its gradients: native
    kernels on a GPU, the reference on the CPU."""
    global _reference
    if _reference is None:
        _reference = _make_reference()
    return _native(t) or _reference


def _make_reference():
    """The reference as autograd functions (torch is imported late throughout
    the package)."""
    from types import SimpleNamespace

    import torch

    from .models import _grouped_ref as ref

    class Once(torch.autograd.Function):
        """A gradient between the tensors it is a product of, the incoming
        gradient and a saved operand: a second differentiation that comes
        through it is an error, whatever else the loss holds."""

        @staticmethod
        def forward(ctx, make, grad, operand=None):
            return make()

        @staticmethod
        def backward(ctx, grad):
            raise RuntimeError(
                "grouped-row operators can be differentiated once only")

    class Gather(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, offsets, slots):
            ctx.save_for_backward(offsets, slots)
            return ref.gather_rows_ref(x, offsets, slots)

        @staticmethod
        def backward(ctx, grad):
            # a row's gradient is the sum over its places
            return Once.apply(lambda: ref.combine_rows_ref(
                grad, *ctx.saved_tensors, None), grad), None, None

    class Combine(torch.autograd.Function):
        @staticmethod
        def forward(ctx, rows, offsets, slots, weights):
            ctx.save_for_backward(rows, offsets, slots, weights)
            return ref.combine_rows_ref(rows, offsets, slots, weights)

        @staticmethod
        def backward(ctx, grad):
            rows, offsets, slots, weights = ctx.saved_tensors
            drows = dw = None
            if ctx.needs_input_grad[0]:
                drows = Once.apply(lambda: ref.combine_rows_backward_ref(
                    grad, rows, offsets, slots, weights, True, False)[0],
                    grad, weights)
            if ctx.needs_input_grad[3]:
                dw = Once.apply(lambda: ref.combine_rows_backward_ref(
                    grad, rows, offsets, slots, weights, False, True)[1],
                    grad, rows)
            return drows, None, None, dw

    class Linear(torch.autograd.Function):
        @staticmethod
        def forward(ctx, rows, weight, offsets, bias):
            ctx.save_for_backward(rows, weight, offsets)
            return ref.grouped_linear_ref(rows, weight, offsets, bias)

        @staticmethod
        def backward(ctx, grad):
            rows, weight, offsets = ctx.saved_tensors
            drows = dweight = dbias = None
            if ctx.needs_input_grad[0]:
                drows = Once.apply(lambda: ref.grouped_linear_drows_ref(
                    grad, weight, offsets), grad, weight)
            if ctx.needs_input_grad[1]:
                dweight = Once.apply(lambda: ref.grouped_linear_dweight_ref(
                    grad, rows, offsets, True, False)[0], grad, rows)
            if ctx.needs_input_grad[3]:
                dbias = Once.apply(lambda: ref.grouped_linear_dweight_ref(
                    grad, rows, offsets, False, True)[1], grad)
            return drows, dweight, None, dbias

    return SimpleNamespace(
        group_rows=ref.group_rows_ref, gather_rows=Gather.apply,
        combine_rows=Combine.apply, grouped_linear=Linear.apply,
        grouped_linear_dweight=ref.grouped_linear_dweight_ref)


def group_rows(ids, n_groups: int) -> GroupPlan:
    """Sort entries by group, stably.

    Parameters
    ----------
    ids : int32 or int64 tensor [T] or [T, k]
        Row t belongs to group ``ids[t]``, or to the k groups ``ids[t, :]``
        (the same one twice is allowed).  An id outside ``[0, n_groups)``
        belongs to no group: its entry takes no part in what follows.
    n_groups : int
        Up to 2^24 - 1.
    """
    if type(n_groups) is int:
        native = _native(ids)
        if native is not None and n_groups.bit_length() < 64:
            return GroupPlan(*native.group_rows(ids, n_groups))
    import torch

    _require(_is_tensor(ids), TypeError, "ids must be a torch.Tensor")
    _require(ids.dtype in (torch.int32, torch.int64), TypeError,
             f"ids must be int32 or int64, got {ids.dtype}")
    _require(ids.dim() in (1, 2), ValueError,
             "ids must have one or two dimensions")
    _require(ids.device.type in ("cpu", "cuda"), ValueError,
             f"ids must be on a GPU or the CPU, got {ids.device}")
    _require(isinstance(n_groups, int) and not isinstance(n_groups, bool),
             TypeError, "n_groups must be an int")
    _require(1 <= n_groups <= _MAX_GROUPS, ValueError,
             f"n_groups must be in [1, {_MAX_GROUPS}], got {n_groups}")
    _require(ids.numel() < (1 << 31) - (1 << 16), ValueError,
             "too many entries")
    return GroupPlan(*_kernels(ids).group_rows(ids, n_groups))


def gather_rows(x, plan: GroupPlan):
    """Rows into group order: ``out[plan.slots[t, j]] = x[t]``.

    ``x`` is [T, F]; the result is [T * k, F].  Places behind
    ``plan.offsets[-1]`` (entries without a group) are zero.  Differentiable
    in ``x``.
    """
    native = _native(x)
    if native is not None and isinstance(plan, GroupPlan):
        return native.gather_rows(x, plan.offsets, plan.slots)
    _require(isinstance(plan, GroupPlan), TypeError, _NO_PLAN)
    _check_rows("x", x)
    offsets, slots = _check_plan(plan, x.device)
    _require(slots.shape[0] == x.shape[0], ValueError,
             f"x has {x.shape[0]} rows, the plan {slots.shape[0]}")
    return _kernels(x).gather_rows(x, offsets, slots)


def combine_rows(rows, plan: GroupPlan, weights=None):
    """Rows back from group order: ``out[t]`` is the sum over j of
    ``weights[t, j] * rows[plan.slots[t, j]]``.

    ``rows`` is [T * k, F] in group order, ``weights`` (float32 or the rows'
    type) is shaped like the ids, or None for ones.  Entries without a group
    are left out, whatever their rows and weights hold; a row without any is
    zero.  Sums run over j in order, in 32 bits.  Differentiable in ``rows``
    and ``weights``.
    """
    native = _native(rows)
    if native is not None and isinstance(plan, GroupPlan):
        return native.combine_rows(rows, plan.offsets, plan.slots, weights)
    import torch

    _require(isinstance(plan, GroupPlan), TypeError, _NO_PLAN)
    _check_rows("rows", rows)
    offsets, slots = _check_plan(plan, rows.device)
    _require(slots.numel() == rows.shape[0], ValueError,
             f"rows has {rows.shape[0]} rows, the plan {slots.numel()}")
    if weights is not None:
        _require(_is_tensor(weights), TypeError,
                 "weights must be a torch.Tensor")
        _require(weights.dtype in (torch.float32, rows.dtype), TypeError,
                 f"weights must be float32 or {rows.dtype}, got "
                 f"{weights.dtype}")
        _require(weights.device == rows.device, ValueError,
                 f"weights are on {weights.device}, the rows on "
                 f"{rows.device}")
        _require(weights.shape == plan.slots.shape, ValueError,
                 f"weights must have the ids' shape "
                 f"{tuple(plan.slots.shape)}, got {tuple(weights.shape)}")
        weights = weights.reshape(slots.shape).contiguous()
    return _kernels(rows).combine_rows(rows, offsets, slots, weights)


def grouped_linear(rows, weight, offsets, bias: Optional[Any] = None):
    """Each group's run of rows times that group's weights.

    ``out[s] = weight[g] @ rows[s] + bias[g]`` for
    ``offsets[g] <= s < offsets[g + 1]``; rows behind ``offsets[-1]`` are
    zero.

    Parameters
    ----------
    rows : [M, F] in group order
    weight : [G, N, F], one matrix a group in the layout of ``coef_``
    offsets : int32 [G + 1] that begins with 0 and does not decrease
        (``GroupPlan.offsets``); groups may be empty
    bias : [G, N] or None

    All of one type; sums are in 32 bits and rounded once.  Differentiable
    in ``rows``, ``weight`` and ``bias``; an empty group's gradients are
    zero.
    """
    native = _native(rows)
    if native is not None:
        return native.grouped_linear(rows, weight, offsets, bias)
    _check_rows("rows", rows)
    _require(_is_tensor(weight) and (bias is None or _is_tensor(bias)),
             TypeError, "weight and bias must be torch.Tensors")
    _check_ints("offsets", offsets, rows.device, 1)
    _require(weight.dim() == 3, ValueError,
             f"weight must be [G, N, F], got shape {tuple(weight.shape)}")
    G, N, F = weight.shape
    _require(1 <= G <= _MAX_GROUPS, ValueError,
             f"between 1 and {_MAX_GROUPS} groups, got {G}")
    _require(N <= _MAX_WIDTH, ValueError,
             f"at most {_MAX_WIDTH} outputs, got {N}")
    _require(F == rows.shape[1], ValueError,
             f"rows have {rows.shape[1]} columns, weight takes {F}")
    _require(offsets.numel() == G + 1, ValueError,
             f"offsets must have {G + 1} values, got {offsets.numel()}")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        _require(t.dtype == rows.dtype, TypeError,
                 f"{name} must be {rows.dtype} like the rows, got {t.dtype}")
        _require(t.device == rows.device, ValueError,
                 f"{name} is on {t.device}, the rows on {rows.device}")
    if bias is not None:
        _require(tuple(bias.shape) == (G, N), ValueError,
                 f"bias must be {(G, N)}, got {tuple(bias.shape)}")
        bias = bias.contiguous()
    return _kernels(rows).grouped_linear(rows, weight.contiguous(),
                                         offsets.contiguous(), bias)
