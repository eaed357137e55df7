"""Experts in 8-bit integers: a scale for each token's row and for each channel of the weights.

``value = code * scale`` on both sides.  Weights keep the package's ``[E, in, out]`` layout, int8, with scales
``[E, out]`` fp32 (``quantize_expert_weights_int8`` makes them at load time); activations are quantised token by token
on every call.  The products are summed in 32-bit integers, exactly, on the tensor cores, so a token's result does not
depend on the batch around it.  Inference only: the operators have no derivative, and a backward pass that reaches one
raises.

The reference has no counterpart (its integer path, src/blackwell_moe/kernels/int4_moe.py, is 4-bit and weights only);
``int8_moe_forward`` keeps the argument order of ``fp8_moe_forward`` (src/blackwell_moe/kernels/fp8_moe.py:111-121).
"""

from __future__ import annotations

import functools
import inspect

import torch
from torch.autograd import forward_ad

from . import _lib
from .moe import _contig, _int32_ids, _on_device, _require_cuda, _stream, _thread_workspace
from .permute import _DTYPES, _MAX_SIZE, _check_plan, _check_sizes, _dtype_code, _has_tangent, _is_own, _row_owners

_I8 = torch.int8


class _WithoutDerivative(torch.autograd.Function):
    """A call among differentiable ones.  Without a node of its own its result would look like a constant, and the gradients of
    what is in front of it would be wrong without a word."""

    @staticmethod
    def forward(ctx, fn, *args):
        ctx.name = fn.__name__
        return fn(*args)

    @staticmethod
    def backward(ctx, *grads):
        raise NotImplementedError(f"{ctx.name} has no gradient: call it under torch.no_grad(), or with detached tensors")


def _inference_only(fn):
    signature = inspect.signature(fn)

    def checked(args, kwargs):
        tensors = [a for a in (*args, *kwargs.values()) if isinstance(a, torch.Tensor)]
        if (torch.is_grad_enabled() and any(t.requires_grad for t in tensors)) or (forward_ad._current_level >= 0 and _has_tangent(*tensors)):
            bound = signature.bind(*args, **kwargs)
            bound.apply_defaults()
            return _WithoutDerivative.apply(fn, *bound.args)
        return fn(*args, **kwargs)

    @functools.wraps(fn)
    def call(*args, **kwargs):
        for a in args:                       # (the usual call at a third of the cost: small products are bound by the host)
            if getattr(a, "requires_grad", False):
                break
        else:
            if forward_ad._current_level < 0 and not any(getattr(a, "requires_grad", False) for a in kwargs.values()):
                return fn(*args, **kwargs)
        return checked(args, kwargs)
    return call


def _out_code(dtype) -> int:
    if dtype not in _DTYPES:
        raise ValueError(f"out_dtype {dtype} is not one of bfloat16, float16, float32")
    return _DTYPES[dtype]


@_inference_only
def quantize_tokens_int8(x: torch.Tensor, plan=None):
    """``x[T,D]`` (bf16, fp16 or fp32; D a multiple of 16) -> ``(codes[T,D] int8, scales[T] fp32)``:
    ``scale = max|x| / 127`` of the row, codes rounded to nearest, ties to even.  A row of zeros has scale 0; a row with an
    infinity or a NaN has scale NaN and codes 0.

    With the ``plan`` of :func:`permute_tokens` the rows come out in expert order, ``(codes[T*K,D], scales[T*K])`` -
    each token is quantised once and written to all of its rows; rows that no slot owns are zero."""
    assert x.dim() == 2, x.shape
    code = _dtype_code(x, "x")
    T, D = x.shape
    if D == 0 or D % 16:
        raise ValueError(f"D={D} must be a multiple of 16")
    tensors, K = [_contig(x, "x")], 1
    if plan is not None:
        offsets, pos = _check_plan(plan)
        assert pos.shape[0] == T, (pos.shape, x.shape)
        tensors += [offsets, pos]
        K = pos.shape[1]
    dev = _require_cuda(*tensors)
    codes = torch.empty((T * K, D), dtype=_I8, device=dev)
    scales = torch.empty(T * K, dtype=torch.float32, device=dev)
    if T:
        with _on_device(dev):
            owners, E = _row_owners(offsets, pos, _is_own(plan)) if plan is not None else (None, 1)
            _lib.check(_lib.lib().bwmoe_int_quant(x.data_ptr(), pos.data_ptr() if plan is not None else None,
                                                  owners.data_ptr() if plan is not None else None, T, D, E, K, code,
                                                  codes.data_ptr(), scales.data_ptr(), _stream(dev)))
    return codes, scales


def _check_grouped(codes, scales, offsets, weights, w_scales):
    assert codes.dim() == 2 and codes.dtype == _I8, (codes.shape, codes.dtype)
    M, D = codes.shape
    assert scales.shape == (M,) and scales.dtype == torch.float32, (scales.shape, scales.dtype)
    assert weights[0].dim() == 3, weights[0].shape
    E, _, N = weights[0].shape
    assert offsets.shape == (E + 1,) and offsets.dtype == torch.int32, (offsets.shape, offsets.dtype, E)
    for w, s in zip(weights, w_scales):
        assert tuple(w.shape) == (E, D, N) and w.dtype == _I8, (w.shape, w.dtype)
        assert tuple(s.shape) == (E, N) and s.dtype == torch.float32, (s.shape, s.dtype)
    _check_sizes("codes and weights", M, D, N, E)
    names = ["codes", "scales", "offsets"] + ["weights"] * len(weights) + ["weight scales"] * len(w_scales)
    dev = _require_cuda(*[_contig(t, n) for t, n in zip([codes, scales, offsets, *weights, *w_scales], names)])
    return dev, M, D, N, E


def _grouped(fn_name, codes, scales, offsets, weights, w_scales, out_dtype):
    dev, M, D, N, E = _check_grouped(codes, scales, offsets, weights, w_scales)
    code = _out_code(out_dtype)
    out = torch.empty((M, N), dtype=out_dtype, device=dev)
    if M:
        lib = _lib.lib()
        with _on_device(dev):
            ws = _thread_workspace(dev, lib.bwmoe_int_scratch_bytes(M, D, N, E))
            _lib.check(getattr(lib, fn_name)(codes.data_ptr(), scales.data_ptr(), offsets.data_ptr(),
                                             *[w.data_ptr() for w in weights], *[s.data_ptr() for s in w_scales], M, D, N, E,
                                             code, out.data_ptr(), ws.data_ptr(), ws.numel(), _stream(dev)))
    return out


@_inference_only
def int8_grouped_gemm(codes, scales, offsets, w, w_scales, out_dtype=torch.bfloat16) -> torch.Tensor:
    """``out[M,N]``: the rows ``offsets[e] .. offsets[e+1]-1`` of ``codes[M,K]`` int8 (scales ``[M]``) times ``w[e]`` of
    ``w[E,K,N]`` int8 (scales ``[E,N]``); K and N multiples of 16.  Rows of no segment are zero."""
    return _grouped("bwmoe_int_grouped_gemm", codes, scales, offsets, (w,), (w_scales,), out_dtype)


@_inference_only
def int8_grouped_swiglu(codes, scales, offsets, w_gate, w_up, s_gate, s_up, out_dtype=torch.bfloat16) -> torch.Tensor:
    """``silu(gate) * up`` of the two grouped products with ``w_gate`` and ``w_up``, in one pass over the rows."""
    return _grouped("bwmoe_int_gateup_swiglu", codes, scales, offsets, (w_gate, w_up), (s_gate, s_up), out_dtype)


@functools.lru_cache(maxsize=256)
def _matmul_workspace_bytes(device_index, T, K, N):         # (sizes go by the device's SMs)
    return _lib.lib().bwmoe_workspace_bytes_int_matmul(T, K, N)


@_inference_only
def int8_matmul(x: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor) -> torch.Tensor:
    """``x[T,K]`` (bf16, fp16 or fp32), quantised token by token, times ``w[K,N]`` int8 with scales ``[N]``, in x's type."""
    assert x.dim() == 2 and w.dim() == 2 and x.shape[1] == w.shape[0], (x.shape, w.shape)
    assert w.dtype == _I8 and w_scales.dtype == torch.float32 and w_scales.shape == (w.shape[1],), (w.dtype, w_scales.shape)
    code = _dtype_code(x, "x")
    _check_sizes("w", *w.shape)
    dev = _require_cuda(_contig(x, "x"), _contig(w, "w"), _contig(w_scales, "w_scales"))
    (T, K), N = x.shape, w.shape[1]
    out = x.new_empty((T, N))
    if T == 0:
        return out
    lib = _lib.lib()
    with _on_device(dev):
        need = _matmul_workspace_bytes(dev.index, T, K, N)
        if need == 0:
            raise ValueError(f"unsupported shape T={T} K={K} N={N} (K and N must be multiples of 16)")
        ws = _thread_workspace(dev, need)
        _lib.check(lib.bwmoe_int_matmul(x.data_ptr(), w.data_ptr(), w_scales.data_ptr(), T, K, N, code, out.data_ptr(),
                                        ws.data_ptr(), ws.numel(), _stream(dev)))
    return out


def _check_int8_experts(x, w_gate, w_up, w_down, s_gate, s_up, s_down):
    assert x.dim() == 2, x.shape
    T, D = x.shape
    assert w_gate.dim() == 3 and w_gate.shape[1] == D, (w_gate.shape, D)
    E, _, H = w_gate.shape
    assert tuple(w_up.shape) == (E, D, H) and tuple(w_down.shape) == (E, H, D), (w_up.shape, w_down.shape)
    for w in (w_gate, w_up, w_down):
        assert w.dtype == _I8, w.dtype
    for s, n in ((s_gate, H), (s_up, H), (s_down, D)):
        assert tuple(s.shape) == (E, n) and s.dtype == torch.float32, (s.shape, s.dtype)
    _check_sizes("x and weights", T, D, H, E)
    tensors = [_contig(t, "tensor") for t in (x, w_gate, w_up, w_down, s_gate, s_up, s_down)]
    return _require_cuda(*tensors), T, D, H, E


def _int8_workspace(lib, dev, T, D, H, E, K):
    need = lib.bwmoe_workspace_bytes_int(T, D, H, E, min(K, _MAX_SIZE))
    if need == 0:
        raise ValueError(f"unsupported shape T={T} D={D} H={H} E={E} top_k={K} "
                         "(D and H must be multiples of 16, E <= 256, top_k <= min(E, 32))")
    return _thread_workspace(dev, need)


@_inference_only
def int8_moe_forward_routed(x, router_weights, expert_indices, experts_w_gate, experts_w_up, experts_w_down,
                            scales_gate, scales_up, scales_down) -> torch.Tensor:
    """The block over experts in 8-bit integers, with the caller's routing (``router_weights[T,K]`` fp32,
    ``expert_indices[T,K]`` int32 or int64): ``x[T,D]`` bf16 or fp16 -> ``out[T,D]``.  Equal, bit for bit, to
    :func:`permute_tokens`' plan, :func:`quantize_tokens_int8`, :func:`int8_grouped_swiglu`, :func:`quantize_tokens_int8`,
    :func:`int8_grouped_gemm` and :func:`unpermute_tokens` in a row, every result in x's type."""
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"x is {x.dtype}: bfloat16 or float16")
    dev, T, D, H, E = _check_int8_experts(x, experts_w_gate, experts_w_up, experts_w_down, scales_gate, scales_up, scales_down)
    assert router_weights.shape == expert_indices.shape and expert_indices.dim() == 2 and expert_indices.shape[0] == T, \
        (router_weights.shape, expert_indices.shape)
    K = expert_indices.shape[1]
    weights, indices = (_contig(t, "routing") for t in (router_weights.to(torch.float32), _int32_ids(expert_indices, E)))
    _require_cuda(x, weights, indices)
    lib = _lib.lib()
    with _on_device(dev):
        out = torch.empty_like(x)
        if T == 0:
            return out
        ws = _int8_workspace(lib, dev, T, D, H, E, K)
        _lib.check(lib.bwmoe_moe_forward_int_routed(
            x.data_ptr(), weights.data_ptr(), indices.data_ptr(), experts_w_gate.data_ptr(), experts_w_up.data_ptr(),
            experts_w_down.data_ptr(), scales_gate.data_ptr(), scales_up.data_ptr(), scales_down.data_ptr(), T, D, H, E, K,
            _DTYPES[x.dtype], out.data_ptr(), ws.data_ptr(), ws.numel(), _stream(dev)))
    return out


@_inference_only
def int8_moe_forward(x, w_gate, experts_w_gate, experts_w_up, experts_w_down, scales_gate, scales_up, scales_down,
                     top_k: int = 8) -> torch.Tensor:
    """:func:`int8_moe_forward_routed` behind :func:`top_k_router`: ``x[T,D]`` bf16, ``w_gate[D,E]`` bf16."""
    assert x.dtype == torch.bfloat16, x.dtype
    dev, T, D, H, E = _check_int8_experts(x, experts_w_gate, experts_w_up, experts_w_down, scales_gate, scales_up, scales_down)
    assert w_gate.shape == (D, E) and w_gate.dtype == torch.bfloat16, (w_gate.shape, w_gate.dtype)
    _require_cuda(x, _contig(w_gate, "w_gate"))
    lib = _lib.lib()
    with _on_device(dev):
        out = torch.empty_like(x)
        if T == 0:
            return out
        ws = _int8_workspace(lib, dev, T, D, H, E, top_k)
        _lib.check(lib.bwmoe_moe_forward_int(
            x.data_ptr(), w_gate.data_ptr(), experts_w_gate.data_ptr(), experts_w_up.data_ptr(), experts_w_down.data_ptr(),
            scales_gate.data_ptr(), scales_up.data_ptr(), scales_down.data_ptr(), T, D, H, E, top_k, out.data_ptr(),
            ws.data_ptr(), ws.numel(), _stream(dev)))
    return out
