"""Tokens into expert order and back, with gradients.

The permutation of the MoE block as operators of their own, for programs that run their own computation between the two
- experts in another format, an adapter, a training step: ``permute_tokens`` takes over ``permute_tokens``
(src/blackwell_moe/kernels/permute.py:12-39), ``unpermute_tokens`` takes over ``unpermute_and_combine``
(src/blackwell_moe/kernels/permute.py:42-59).  bf16, fp16 and fp32; sums are held in fp32, added in a fixed order and
rounded once.  Both are differentiable (once, forwards or backwards): in the tokens and the rows, and in the routing weights.
"""

from __future__ import annotations

import functools
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from . import _lib
from .moe import _contig, _on_device, _require_cuda, _stream

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


class PermutePlan(NamedTuple):
    """Where every slot (token, k) of a batch goes in expert order; int32 tensors of one device.

    ``offsets[E+1]``: expert e's rows are ``offsets[e] .. offsets[e+1]-1``; ``pos[T,K]``: the row of each slot;
    ``row_slot[M]``: the slot of each row, ``t*K + k``; ``row_expert[M]``: its expert.  A slot whose expert id is
    outside ``[0, E)`` has no row (``pos`` -1), and the rows past ``offsets[E]`` then have no slot (-1).  The operators
    read ``offsets`` and ``pos`` only: a plan made elsewhere, or one with slots dropped (``pos`` set to -1), may leave the
    other two out, and may leave any row without a slot.  Two slots never have the same row.  (A plan of this package that
    was written to without torch counting it, through ``.data`` or by another library, is to be passed as a new
    ``PermutePlan`` of its tensors.)"""
    offsets: torch.Tensor
    pos: torch.Tensor
    row_slot: Optional[torch.Tensor] = None
    row_expert: Optional[torch.Tensor] = None


class _OwnPlan(PermutePlan):
    """A plan as the library wrote it: the rows without a slot are those past ``offsets[E]``.  Copies, of whose tensors nobody
    knows what they went through, are plain plans, as is what ``_replace`` returns; see :func:`_own_plan`."""
    __slots__ = ()
    _make = PermutePlan._make

    def __new__(cls, *args, **kwargs):
        return PermutePlan(*args, **kwargs)


def _own_plan(*tensors):
    return tuple.__new__(_OwnPlan, tensors)


def _is_own(plan) -> bool:
    if type(plan) is not _OwnPlan:
        return False
    offsets, pos = plan[0], plan[1]
    return not (pos.is_inference() or offsets.is_inference()) and pos._version == 0 and offsets._version == 0


def _row_owners(offsets, pos, own):
    """What tells the rows without a slot: the segments of the library's own plan, or each row's slot.  The tensor, and its
    number of experts (0)."""
    if own:
        return offsets, offsets.numel() - 1
    slots = pos.new_empty(pos.numel())
    _lib.check(_lib.lib().bwmoe_plan_row_slots(pos.data_ptr(), *pos.shape, slots.data_ptr(), _stream(pos.device)))
    return slots, 0


_MAX_SIZE = 2 ** 31 - 4096      # sizes reach the library as 32-bit integers: a larger one would wrap on the way


def _check_sizes(name, *sizes):
    if max(sizes) > _MAX_SIZE:
        raise ValueError(f"{name}: sizes {sizes}, at most {_MAX_SIZE} each")


def _dtype_code(t: torch.Tensor, name: str) -> int:
    if t.numel() > _MAX_SIZE:        # (a size that large, or only their product)
        _check_sizes(name, *t.shape)
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"{name}: {t.dtype} is not one of bfloat16, float16, float32")
    return code


@functools.lru_cache(maxsize=256)
def _plan_scratch_bytes(T, num_experts, K):
    return _lib.lib().bwmoe_plan_scratch_bytes(T, num_experts, K)


def _empty_plan(indices, T, K, num_experts, scratch_bytes):
    """The plan's tensors, and the addresses of its status word and scratch behind them: one allocation."""
    M, extra = T * K, 4 + (scratch_bytes + 3) // 4
    # (not views of one another: each has its own version, as tensors that were allocated apart)
    o, p, s, e, rest = torch.unsafe_split_with_sizes(indices.new_empty(num_experts + 1 + 3 * M + extra), (num_experts + 1, M, M, M, extra))
    status = rest.data_ptr()
    return _own_plan(o, p.view(T, K), s, e), status, status + 16


def _check_indices(indices, num_experts):
    assert indices.dim() == 2 and indices.shape[1] >= 1, indices.shape
    assert indices.dtype == torch.int32, indices.dtype
    if not 1 <= num_experts <= 256 or indices.shape[1] > 32:
        raise ValueError(f"{num_experts} experts and {indices.shape[1]} slots per token: at most 256 and 32")
    _check_sizes("indices", indices.numel())
    return _contig(indices, "indices")


def _check_plan(plan, name="plan"):
    offsets, pos = plan[0], plan[1]
    assert pos.dim() == 2 and offsets.dim() == 1 and offsets.numel() >= 2, (name, pos.shape, offsets.shape)
    assert pos.dtype == torch.int32 and offsets.dtype == torch.int32, (name, pos.dtype, offsets.dtype)
    if pos.numel() > _MAX_SIZE or offsets.numel() > _MAX_SIZE:
        _check_sizes(name, pos.numel(), offsets.numel())
    _contig(pos, "plan.pos"), _contig(offsets, "plan.offsets")
    return offsets, pos


def _elsewhere(dev):
    """Whether a call has to make its tensors' device the current one first.  (The usual answer costs a tenth of a context
    manager, and small batches are bound by the host.)"""
    return dev.index != torch.cuda.current_device()


def permute_plan(indices: torch.Tensor, num_experts: int) -> PermutePlan:
    """The stable sort of all slots of ``indices[T,K]`` int32 by expert id."""
    indices = _check_indices(indices, num_experts)
    dev = _require_cuda(indices)
    T, K = indices.shape
    lib = _lib.lib()
    with _on_device(dev):
        plan, status, scratch = _empty_plan(indices, T, K, num_experts, _plan_scratch_bytes(T, num_experts, K))
        if T == 0:
            plan.offsets.zero_()
            return plan
        _lib.check(lib.bwmoe_permute_plan(indices.data_ptr(), None, T, num_experts, K, plan.offsets.data_ptr(),
                                          plan.pos.data_ptr(), plan.row_slot.data_ptr(), plan.row_expert.data_ptr(), None,
                                          status, scratch, _stream(dev)))
    return plan


def _permute_new(x, indices, num_experts):
    """The plan and the rows in one call."""
    dev = x.device
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return _permute_new(x, indices, num_experts)
    (T, K), D = indices.shape, x.shape[1]
    lib = _lib.lib()
    plan, status, scratch = _empty_plan(indices, T, K, num_experts, _plan_scratch_bytes(T, num_experts, K))
    rows = x.new_empty((T * K, D))
    pos = plan.pos.data_ptr()
    _lib.check(lib.bwmoe_permute_tokens(x.data_ptr(), indices.data_ptr(), T, D, num_experts, K, _DTYPES[x.dtype],
                                        plan.offsets.data_ptr(), pos, pos + 4 * T * K, pos + 8 * T * K, rows.data_ptr(),
                                        status, scratch, _stream(dev)))
    return rows, plan


def _permute(x, offsets, pos, own):
    """rows[pos[t,k]] = x[t]"""
    dev = x.device
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return _permute(x, offsets, pos, own)
    (T, K), D = pos.shape, x.shape[1]
    rows = x.new_empty((T * K, D))
    if T and D:
        owners, E = _row_owners(offsets, pos, own)
        _lib.check(_lib.lib().bwmoe_permute_rows(x.data_ptr(), pos.data_ptr(), owners.data_ptr(), T, D, E,
                                                 K, _DTYPES[x.dtype], rows.data_ptr(), _stream(dev)))
    return rows


def _unpermute(rows, pos, weights):
    """sum over k of w[t,k] * rows[pos[t,k]]"""
    dev = rows.device
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return _unpermute(rows, pos, weights)
    (T, K), D = pos.shape, rows.shape[1]
    out = rows.new_empty((T, D))
    if T and D:
        _lib.check(_lib.lib().bwmoe_unpermute_rows(rows.data_ptr(), pos.data_ptr(), None if weights is None else weights.data_ptr(),
                                                   T, D, K, _DTYPES[rows.dtype], out.data_ptr(), _stream(dev)))
    return out


def _unpermute_backward(dout, rows, offsets, pos, own, weights, rows_grad, weights_grad):
    T, K = pos.shape
    D, dev = dout.shape[1], dout.device
    with _on_device(dev):
        drows = dout.new_empty((T * K, D)) if rows_grad else None
        dweights = torch.empty_like(weights) if weights_grad else None
        if T and D:
            if rows_grad or weights_grad:
                owners, E = _row_owners(offsets, pos, own or not rows_grad)
                _lib.check(_lib.lib().bwmoe_unpermute_rows_backward(
                    dout.data_ptr(), rows.data_ptr() if weights_grad else None, pos.data_ptr(), owners.data_ptr(),
                    weights.data_ptr(), T, D, E, K, _DTYPES[dout.dtype], drows.data_ptr() if rows_grad else None,
                    dweights.data_ptr() if weights_grad else None, _stream(dev)))
        elif weights_grad:
            dweights.zero_()
    return drows, dweights


def _has_tangent(*tensors):
    """Whether one of them is a dual tensor, for which ``requires_grad`` need not be set: the launches know nothing of tangents."""
    return forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _once(backward):
    """``once_differentiable`` where a second derivative could be asked for (``create_graph``): its bookkeeping costs as
    much as a small batch's backward pass."""
    guarded = torch.autograd.function.once_differentiable(backward)

    def call(ctx, grad):
        if forward_ad._current_level >= 0 and _has_tangent(grad, *ctx.saved_tensors):
            raise NotImplementedError("the gradients of permute_tokens and unpermute_tokens have no derivative themselves")
        return guarded(ctx, grad) if torch.is_grad_enabled() else backward(ctx, grad)
    return staticmethod(call)


def _permute_backward(ctx, drows):
    return _unpermute(drows.contiguous(), ctx.saved_tensors[0], None), None, None, None


def _permute_jvp(ctx, dx, *_):
    return _permute(dx.contiguous(), *ctx.saved_tensors, ctx.own)


class _PermuteRows(torch.autograd.Function):
    backward, jvp = _once(_permute_backward), staticmethod(_permute_jvp)

    @staticmethod
    def forward(ctx, x, offsets, pos, own):
        ctx.save_for_backward(pos)
        if forward_ad._current_level >= 0:
            ctx.save_for_forward(offsets, pos)
            ctx.own = own
        return _permute(x, offsets, pos, own)


class _PermuteTokens(torch.autograd.Function):
    backward, jvp = _once(_permute_backward), staticmethod(_permute_jvp)

    @staticmethod
    def forward(ctx, x, args, found):        # args: (indices, num_experts); the plan leaves through the list `found`
        rows, plan = _permute_new(x, *args)
        ctx.save_for_backward(plan.pos)
        if forward_ad._current_level >= 0:
            ctx.save_for_forward(plan.offsets, plan.pos)
            ctx.own = True
        found.append(plan)
        return rows


def _unpermute_rows_backward(ctx, dout):
    rows, offsets, pos, weights = ctx.saved_tensors
    dout = dout.contiguous()
    if weights is None:
        return _permute(dout, offsets, pos, ctx.own), None, None, None, None
    drows, dweights = _unpermute_backward(dout, rows, offsets, pos, ctx.own, weights, ctx.needs_input_grad[0], ctx.needs_input_grad[3])
    return drows, None, None, dweights, None


def _unpermute_rows_jvp(ctx, drows, _offsets, _pos, dweights, _own):
    rows, pos, weights = ctx.saved_tensors
    # (a sum of two results that are rounded to the type each)
    terms = [] if drows is None else [_unpermute(drows.contiguous(), pos, weights)]
    if dweights is not None:
        terms.append(_unpermute(rows, pos, dweights.contiguous()))
    return sum(terms[1:], start=terms[0])


class _UnpermuteRows(torch.autograd.Function):
    backward, jvp = _once(_unpermute_rows_backward), staticmethod(_unpermute_rows_jvp)

    @staticmethod
    def forward(ctx, rows, offsets, pos, weights, own):
        # the rows are kept for the weights' derivative only
        ctx.save_for_backward(rows if ctx.needs_input_grad[3] else None, offsets, pos, weights)
        if forward_ad._current_level >= 0:
            ctx.save_for_forward(rows, pos, weights)
        ctx.own = own
        return _unpermute(rows, pos, weights)


def permute_tokens(x: torch.Tensor, indices: torch.Tensor = None, num_experts: int = None, *, plan: PermutePlan = None):
    """``x[T,D]`` -> ``(rows[T*K,D], plan)``: a copy of token t in the row of each of its slots, rows sorted by expert
    (stable).  ``indices[T,K]`` int32 are the tokens' experts; or pass the ``plan`` of an earlier call.  Rows that no slot
    owns are zero.  The gradient of a token is the sum of its rows' gradients."""
    assert x.dim() == 2, x.shape
    _dtype_code(x, "x")
    _contig(x, "x")
    if (indices is None) == (plan is None) or (indices is None) != (num_experts is None):
        raise ValueError("permute_tokens takes indices and num_experts, or a plan")
    wants_grad = (x.requires_grad and torch.is_grad_enabled()) or _has_tangent(x)
    if plan is None:
        _check_indices(indices, num_experts)
        assert indices.shape[0] == x.shape[0], (indices.shape, x.shape)
        _require_cuda(x, indices)
        if x.numel():
            if not wants_grad:
                return _permute_new(x, indices, num_experts)
            found = []
            return _PermuteTokens.apply(x, (indices, num_experts), found), found[0]
        plan = permute_plan(indices, num_experts)
    offsets, pos = _check_plan(plan)
    assert pos.shape[0] == x.shape[0], (pos.shape, x.shape)
    _require_cuda(x, offsets, pos)
    own = _is_own(plan)
    return (_PermuteRows.apply(x, offsets, pos, own) if wants_grad else _permute(x, offsets, pos, own)), plan


def _check_unpermute(rows, plan, weights):
    assert rows.dim() == 2, rows.shape
    _dtype_code(rows, "rows")
    offsets, pos = _check_plan(plan)
    assert rows.shape[0] == pos.numel(), (rows.shape, pos.shape)
    _contig(rows, "rows")
    if weights is None:
        _require_cuda(rows, offsets, pos)
    else:
        assert weights.shape == pos.shape and weights.dtype == torch.float32, (weights.shape, weights.dtype)
        _require_cuda(rows, offsets, pos, _contig(weights, "weights"))
    return offsets, pos


def unpermute_tokens(rows: torch.Tensor, plan: PermutePlan, weights: torch.Tensor = None) -> torch.Tensor:
    """``rows[T*K,D]`` in expert order -> ``out[T,D]``, ``out[t] = sum_k weights[t,k] * rows[plan.pos[t,k]]`` with
    ``weights[T,K]`` fp32 (absent: 1).  Slots without a row add nothing.  Differentiable in ``rows`` and ``weights``."""
    offsets, pos = _check_unpermute(rows, plan, weights)
    if (torch.is_grad_enabled() and (rows.requires_grad or (weights is not None and weights.requires_grad))) \
            or _has_tangent(rows, weights):
        return _UnpermuteRows.apply(rows, offsets, pos, weights, _is_own(plan))
    return _unpermute(rows, pos, weights)


def unpermute_tokens_backward(dout: torch.Tensor, rows: torch.Tensor, plan: PermutePlan, weights: torch.Tensor, *,
                              rows_grad: bool = True, weights_grad: bool = True):
    """The gradients of :func:`unpermute_tokens` without autograd, for programs that run (or capture) their backward pass
    themselves: ``(drows, dweights)``, ``None`` where not asked for.  ``rows`` may be ``None`` without ``weights_grad``."""
    assert dout.dim() == 2, dout.shape
    _dtype_code(dout, "dout")
    offsets, pos = _check_plan(plan)
    (T, K), D = pos.shape, dout.shape[1]
    assert dout.shape[0] == T, (dout.shape, pos.shape)
    assert weights.shape == pos.shape and weights.dtype == torch.float32, (weights.shape, weights.dtype)
    tensors = [_contig(dout, "dout"), offsets, pos, _contig(weights, "weights")]
    if weights_grad:
        assert rows is not None and rows.shape == (T * K, D) and rows.dtype == dout.dtype, (None if rows is None else rows.shape)
        tensors.append(_contig(rows, "rows"))
    _require_cuda(*tensors)
    return _unpermute_backward(dout, rows, offsets, pos, _is_own(plan), weights, rows_grad, weights_grad)
