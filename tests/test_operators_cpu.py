"""Refusals of the permutation and of the 8-bit integer operators, and sizes: nothing here reaches a GPU."""

import pytest
import torch

import blackwell_moe_b200 as bw
from blackwell_moe_b200 import _lib

I8, I32, F32, BF16 = torch.int8, torch.int32, torch.float32, torch.bfloat16


def test_permute_refusals():
    x, idx = torch.zeros(4, 32), torch.zeros(4, 2, dtype=I32)
    plan = bw.PermutePlan(torch.zeros(9, dtype=I32), torch.zeros(4, 2, dtype=I32), None, None)
    for call in (lambda: bw.permute_tokens(x, idx, 8), lambda: bw.permute_plan(idx, 8), lambda: bw.permute_tokens(x, plan=plan),
                 lambda: bw.unpermute_tokens(torch.zeros(8, 32), plan),                     # no CPU path
                 lambda: bw.permute_tokens(x), lambda: bw.permute_tokens(x, idx), lambda: bw.permute_tokens(x, idx, 8, plan=plan),
                 lambda: bw.permute_tokens(x.double(), idx, 8), lambda: bw.permute_tokens(x.t(), torch.zeros(32, 2, dtype=I32), 8),
                 lambda: bw.permute_tokens(x, idx.t().contiguous().t(), 8),
                 lambda: bw.permute_tokens(x, idx, 257), lambda: bw.permute_tokens(x, idx, 0),
                 lambda: bw.permute_plan(torch.zeros(4, 33, dtype=I32), 64)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: bw.permute_tokens(x, idx.long(), 8), lambda: bw.permute_tokens(x[0], idx, 8),
                 lambda: bw.permute_tokens(x[:3], idx, 8), lambda: bw.permute_tokens(x[:3], plan=plan),
                 lambda: bw.unpermute_tokens(torch.zeros(7, 32), plan), lambda: bw.unpermute_tokens(torch.zeros(8, 32), plan, torch.zeros(4, 3)),
                 lambda: bw.unpermute_tokens(torch.zeros(8, 32), plan, torch.zeros(4, 2, dtype=BF16)),
                 lambda: bw.unpermute_tokens_backward(torch.zeros(4, 32), None, plan, torch.zeros(4, 2))):
        with pytest.raises(AssertionError):
            call()


def test_int8_refusals():
    codes, s, off = torch.zeros(4, 32, dtype=I8), torch.zeros(4), torch.zeros(3, dtype=I32)
    w, ws = torch.zeros(2, 32, 48, dtype=I8), torch.zeros(2, 48)
    x = torch.zeros(4, 32, dtype=BF16)
    for call in (lambda: bw.int8_grouped_gemm(codes, s, off, w, ws), lambda: bw.int8_grouped_gemm(codes, s, off, w, ws, out_dtype=torch.float64),
                 lambda: bw.quantize_tokens_int8(x), lambda: bw.quantize_tokens_int8(x.double()), lambda: bw.quantize_tokens_int8(x[:, :24]),
                 lambda: bw.quantize_tokens_int8(torch.zeros(4, 40)), lambda: bw.int8_matmul(x, w[0], ws[0]),
                 lambda: bw.int8_matmul(x, w[0].t().contiguous().t(), ws[0]), lambda: bw.int8_matmul(x.double(), w[0], ws[0]),
                 lambda: bw.int8_moe_forward_routed(x.float(), s[:, None], off[:, None], w, w, w, ws, ws, ws)):
        with pytest.raises(ValueError):
            call()
    down, ds = torch.zeros(2, 48, 32, dtype=I8), torch.zeros(2, 32)
    for call in (lambda: bw.int8_grouped_gemm(codes.float(), s, off, w, ws), lambda: bw.int8_grouped_gemm(codes, s[:3], off, w, ws),
                 lambda: bw.int8_grouped_gemm(codes, s, off[:2], w, ws), lambda: bw.int8_grouped_gemm(codes, s, off.long(), w, ws),
                 lambda: bw.int8_grouped_gemm(codes, s, off, w, ws[:, :32]), lambda: bw.int8_grouped_gemm(codes, s, off, w.float(), ws),
                 lambda: bw.int8_grouped_gemm(codes[:, :16].contiguous(), s, off, w, ws), lambda: bw.int8_matmul(x, w[0], ws),
                 lambda: bw.int8_grouped_swiglu(codes, s, off, w, w[:, :, :32].contiguous(), ws, ws),
                 lambda: bw.int8_moe_forward(x.half(), x, w, w, down, ws, ws, ds),
                 lambda: bw.int8_moe_forward_routed(x, torch.zeros(4, 2), torch.zeros(4, 2, dtype=I32), w, w, w, ws, ws, ds),
                 lambda: bw.int8_moe_forward_routed(x, torch.zeros(4, 2), torch.zeros(4, 2, dtype=I32), w, w, down, ws, ws, ws)):
        with pytest.raises(AssertionError):
            call()


def test_entry_points_refuse_before_any_device_work():
    lib, p = bw.lib(), 4096                       # an aligned address that nothing reads
    bad = lambda rc, code, word: rc == code and word in _lib.last_error()                    # noqa: E731
    assert bad(lib.bwmoe_permute_rows(p, p, p, 0, 16, 8, 2, 0, p, None), -1, "permute_rows")
    assert bad(lib.bwmoe_permute_rows(p, p, p, 4, 16, 8, 33, 0, p, None), -4, "permute_rows")
    assert bad(lib.bwmoe_permute_rows(p, p, p, 4, 16, 8, 2, 3, p, None), -4, "permute_rows")
    assert bad(lib.bwmoe_permute_rows(p, None, p, 4, 16, 8, 2, 0, p, None), -6, "permute_rows")
    assert bad(lib.bwmoe_permute_rows(p + 2, p, p, 4, 16, 8, 2, 2, p, None), -2, "permute_rows")
    assert bad(lib.bwmoe_permute_rows(p, p, p, 2 ** 30, 16, 8, 2, 0, p, None), -4, "too large")
    for n in (2 ** 31 - 1, 2 ** 31 - 4095):       # sizes that round up to a tile would leave 32 bits
        assert bad(lib.bwmoe_unpermute_rows(p, p, None, n, 16, 1, 0, p, None), -4, "too large")
        assert bad(lib.bwmoe_permute_tokens(p, p, n, 16, 8, 1, 0, p, p, p, p, p, p, p, None), -4, "too large")
        assert bad(lib.bwmoe_int_quant(p, None, None, n, 32, 1, 1, 0, p, p, None), -4, "too large")
        assert bad(lib.bwmoe_int_grouped_gemm(p, p, p, p, p, n, 32, 48, 2, 0, p, p, 1 << 40, None), -4, "rows")
    assert bad(lib.bwmoe_permute_tokens(p, p, 4, 16, 300, 2, 0, p, p, p, p, p, p, p, None), -4, "plan")
    assert bad(lib.bwmoe_unpermute_rows(p, p, None, 4, 0, 2, 0, p, None), -1, "unpermute_rows")
    assert bad(lib.bwmoe_unpermute_rows_backward(p, p, p, p, p, 4, 16, 8, 2, 0, None, None, None), -6, "backward")
    assert bad(lib.bwmoe_unpermute_rows_backward(p, None, p, p, p, 4, 16, 8, 2, 0, None, p, None), -6, "backward")
    assert bad(lib.bwmoe_unpermute_rows_backward(p, None, p, p, None, 4, 16, 8, 2, 0, p, None, None), -6, "backward")
    assert bad(lib.bwmoe_int_quant(p, None, None, 4, 24, 1, 1, 0, p, p, None), -1, "int_quant")
    assert bad(lib.bwmoe_int_quant(p, None, None, 4, 32, 1, 2, 0, p, p, None), -1, "int_quant")
    assert bad(lib.bwmoe_int_quant(p + 8, None, None, 4, 32, 1, 1, 0, p, p, None), -2, "int_quant")
    n = lib.bwmoe_int_scratch_bytes(4, 32, 48, 2)
    assert n > 0
    assert bad(lib.bwmoe_int_grouped_gemm(p, p, p, p, p, 4, 32, 48, 2, 0, p, p, n - 1, None), -3, "int_grouped_gemm")
    assert bad(lib.bwmoe_int_grouped_gemm(p, p, p, p, p, 4, 32, 48, 2, 0, p, None, n, None), -3, "int_grouped_gemm")
    assert bad(lib.bwmoe_int_gateup_swiglu(p, p, p, p, None, p, p, 4, 32, 48, 2, 0, p, p, n, None), -6, "int_gateup_swiglu")
    for K, N, E, code in ((24, 48, 2, -1), (32, 40, 2, -1), (32, 48, 257, -4), (1 << 17, 48, 2, -4)):
        assert bad(lib.bwmoe_int_grouped_gemm(p, p, p, p, p, 4, K, N, E, 0, p, p, 1 << 40, None), code, "int_grouped_gemm")
    assert bad(lib.bwmoe_int_grouped_gemm(p, p, None, p, p, 4, 32, 48, 2, 0, p, p, 1 << 40, None), -6, "offsets")
    assert bad(lib.bwmoe_int_grouped_gemm(p, p, p, p, p + 4, 4, 32, 48, 2, 0, p, p, 1 << 40, None), -2, "int_grouped_gemm")
    assert lib.bwmoe_workspace_bytes_int_matmul(4, 40, 16) == 0 and lib.bwmoe_workspace_bytes_int_matmul(4, 32, 48) > 0
    assert bad(lib.bwmoe_int_matmul(p, p, p, 4, 32, 48, 0, p, p, 16, None), -3, "int_matmul")
    assert lib.bwmoe_workspace_bytes_int(4, 40, 48, 2, 2) == 0 and lib.bwmoe_workspace_bytes_int(4, 32, 48, 2, 3) == 0
    ws = lib.bwmoe_workspace_bytes_int(4, 32, 48, 2, 2)
    assert ws > 0
    assert bad(lib.bwmoe_moe_forward_int_routed(*[p] * 9, 4, 32, 48, 2, 2, 2, p, p, ws, None), -4, "bf16 or fp16")
    assert bad(lib.bwmoe_moe_forward_int_routed(*[p] * 9, 4, 32, 48, 2, 2, 0, p, p, ws - 1, None), -3, "moe_forward_int_routed")
    assert bad(lib.bwmoe_moe_forward_int(*[None] * 8, 4, 32, 48, 2, 2, None, None, 0, None), -6, "moe_forward_int")


def test_weights_in_8_bit_integers():
    g = torch.Generator().manual_seed(0)
    w = torch.randn(3, 64, 48, generator=g) * 0.02
    w[1, :, 5] = 0
    codes, scales = bw.quantize_expert_weights_int8(w.to(BF16))
    assert codes.dtype == I8 and codes.shape == w.shape and scales.shape == (3, 48) and scales.dtype == F32
    assert (codes[1, :, 5] == 0).all() and scales[1, 5] == 0
    err = (codes.double() * scales[:, None].double() - w.to(BF16).double()).abs()
    assert (err <= scales[:, None].double() * (0.5 + 127 * 2.0 ** -23)).all()       # half a step, and the quotient's rounding
    live = scales > 0
    assert (codes.abs().amax(1)[live] == 127).all()


def test_sizes_past_32_bits_are_refused():
    """They would reach the library modulo 2^32."""
    big, m = 2 ** 32 + 16, lambda *shape, dtype=BF16: torch.empty(shape, dtype=dtype, device="meta")      # noqa: E731
    plan = lambda T, K, E=8: bw.PermutePlan(m(E + 1, dtype=I32), m(T, K, dtype=I32))                       # noqa: E731
    w, ws = m(2, 16, big, dtype=I8), m(2, big, dtype=F32)
    for call in (lambda: bw.permute_tokens(m(big, 1), m(big, 1, dtype=I32), 8), lambda: bw.permute_tokens(m(1, big), m(1, 1, dtype=I32), 8),
                 lambda: bw.permute_plan(m(big, 1, dtype=I32), 8), lambda: bw.permute_tokens(m(1, 16), plan=plan(1, big)),
                 lambda: bw.permute_tokens(m(1, 16), plan=plan(1, 2, big)), lambda: bw.unpermute_tokens(m(big, 16), plan(big, 1)),
                 lambda: bw.unpermute_tokens_backward(m(1, big), m(2, big), plan(1, 2), m(1, 2, dtype=F32)),
                 lambda: bw.quantize_tokens_int8(m(big, 16)), lambda: bw.int8_matmul(m(1, 16), m(16, big, dtype=I8), m(big, dtype=F32)),
                 lambda: bw.int8_grouped_gemm(m(4, 16, dtype=I8), m(4, dtype=F32), m(3, dtype=I32), w, ws),
                 lambda: bw.int8_grouped_swiglu(m(big, 16, dtype=I8), m(big, dtype=F32), m(3, dtype=I32), *[m(2, 16, 16, dtype=I8)] * 2, *[m(2, 16, dtype=F32)] * 2),
                 lambda: bw.int8_moe_forward(m(4, 16), m(16, 2), w, w, m(2, big, 16, dtype=I8), ws, ws, m(2, 16, dtype=F32)),
                 lambda: bw.int8_moe_forward_routed(m(4, 16), m(4, 2, dtype=F32), m(4, 2, dtype=I32), w, w, m(2, big, 16, dtype=I8), ws, ws, m(2, 16, dtype=F32))):
        with pytest.raises(ValueError, match="sizes"):
            call()


def test_row_slots_and_negative_expert_counts_are_refused():
    lib, p = bw.lib(), 4096
    bad = lambda rc, code, word: rc == code and word in _lib.last_error()                    # noqa: E731
    assert bad(lib.bwmoe_plan_row_slots(p, 0, 2, p, None), -1, "plan_row_slots")
    assert bad(lib.bwmoe_plan_row_slots(p, 4, 0, p, None), -1, "plan_row_slots")
    assert bad(lib.bwmoe_plan_row_slots(p, 2 ** 31 - 1, 1, p, None), -4, "too large")
    assert bad(lib.bwmoe_plan_row_slots(None, 4, 2, p, None), -6, "plan_row_slots")
    assert bad(lib.bwmoe_plan_row_slots(p, 4, 2, None, None), -6, "plan_row_slots")
    assert bad(lib.bwmoe_permute_rows(p, p, p, 4, 16, -1, 2, 0, p, None), -1, "permute_rows")
    assert bad(lib.bwmoe_unpermute_rows_backward(p, p, p, p, p, 4, 16, -1, 2, 0, p, None, None), -6, "backward")
    assert bad(lib.bwmoe_int_quant(p, p, p, 4, 32, -1, 2, 0, p, p, None), -1, "int_quant")


def test_channels_without_a_representation():
    w = torch.randn(2, 32, 16, generator=torch.Generator().manual_seed(1))
    want = bw.quantize_expert_weights_int8(w)
    bad = w.clone()
    bad[0, 3, 1], bad[0, 4, 2], bad[1, 5, 3], bad[1, 6, 3] = float("nan"), float("inf"), -float("inf"), float("nan")
    codes, scales = bw.quantize_expert_weights_int8(bad)
    none = torch.zeros(2, 16, dtype=torch.bool)
    none[0, 1] = none[0, 2] = none[1, 3] = True
    assert torch.equal(scales.isnan(), none) and torch.equal(scales[~none], want[1][~none])
    assert (codes.transpose(1, 2)[none] == 0).all() and torch.equal(codes.transpose(1, 2)[~none], want[0].transpose(1, 2)[~none])
