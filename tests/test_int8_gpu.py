"""Experts in 8-bit integers: the row quantiser, the grouped products and the block, against the definitions in 64 bits."""

import pytest
import torch

import blackwell_moe_b200 as bw

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16, F32, I8 = torch.bfloat16, torch.float16, torch.float32, torch.int8
U32 = 2.0 ** -24                                 # half a step of fp32


def half_step(dtype):
    return 0.0 if dtype == F32 else torch.finfo(dtype).eps / 2


def smallest_step(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def exact_codes(x):
    """Codes and scales by the definition; the quotients in 64 bits are exact enough to tell a tie from its neighbours
    (they differ from n + 1/2 by 2^-33 at least, or not at all).  A row with an infinity or a NaN has none."""
    x = x.double()
    amax = x.abs().amax(1)
    scale = (torch.where(amax.isfinite(), amax, torch.full_like(amax, float("nan"))) / 127).float().double()
    q = torch.where(scale[:, None] > 0, x / scale[:, None], torch.zeros_like(x))
    return torch.round(q).clamp(-127, 127).to(I8), scale.float()


def assert_codes(codes, scales, x):
    want, scale = exact_codes(x)
    torch.testing.assert_close(scales.cpu(), scale, rtol=0, atol=0, equal_nan=True)
    assert torch.equal(codes.cpu(), want), torch.nonzero(codes.cpu() != want)[:8].tolist()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("T,D", [(1, 16), (3, 48), (64, 2048), (517, 1408), (5, 14336), (2, 16384), (3, 20000), (6000, 64)])
def test_codes_are_exact(T, D, dtype):
    g = torch.Generator().manual_seed(T + D)
    x = (torch.randn(T, D, generator=g) * torch.exp(3 * torch.randn(T, 1, generator=g))).to(dtype)
    codes, scales = bw.quantize_tokens_int8(x.to(DEV))
    assert_codes(codes, scales, x)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_codes_on_borders_and_of_small_rows(dtype):
    D = 1024
    n = torch.arange(D) % 255 - 127
    ties = (n.float() + 0.5).clamp(-127, 127)
    rows = [ties * 2.0 ** -4, ties * 2.0 ** -8, n.float(), torch.zeros(D)]     # the largest is 127 steps: the scale is exact
    g = torch.Generator().manual_seed(3)
    tiny = torch.finfo(dtype).smallest_normal
    rows += [torch.randn(D, generator=g) * s for s in (tiny, tiny * 2 ** -4, tiny * 2 ** -6, tiny * 2 ** -7, tiny * 200)]
    rows += [torch.randn(D, generator=g).clamp(-1, 1) * torch.finfo(dtype).max * 0.99]
    one = torch.zeros(D)
    one[700] = -smallest_step(dtype)
    rows += [one, -0.0 * one]
    x = torch.stack(rows).to(dtype)
    if dtype != F32:
        x[0, 0] = 127 * 2.0 ** -4
    # fp32: values next to the borders of a scale that is not a power of two
    s = torch.tensor(0.0123).float()
    near = ((torch.arange(D) % 127).double() + 0.5) * s.double()
    near = near.float() if dtype == F32 else near.to(dtype).float()
    if dtype == F32:
        near[1::3] = torch.nextafter(near[1::3], torch.tensor(9e9))
        near[2::3] = torch.nextafter(near[2::3], torch.tensor(-9e9))
    near[5] = 127 * s
    x = torch.cat([x, near[None].to(dtype), -near[None].to(dtype)])
    codes, scales = bw.quantize_tokens_int8(x.to(DEV))
    assert_codes(codes, scales, x)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_rows_without_a_representation(dtype):
    x = torch.ones(6, 64, dtype=dtype)
    x[1, 3], x[2, 63], x[3, 0] = float("nan"), float("inf"), -float("inf")
    codes, scales = bw.quantize_tokens_int8(x.to(DEV))
    assert scales.isnan().tolist() == [False, True, True, True, False, False]
    assert (codes[1:4] == 0).all() and (codes[0] == 127).all() and (codes[4:] == 127).all()
    w = torch.ones(64, 32, dtype=I8, device=DEV)
    out = bw.int8_matmul(x.to(DEV), w, torch.ones(32, device=DEV))
    assert out.isnan().any(1).tolist() == out.isnan().all(1).tolist() == [False, True, True, True, False, False]


@pytest.mark.parametrize("T,D,E,K,bad", [(1, 16, 4, 2, 0), (37, 2048, 64, 6, 5), (700, 144, 16, 3, 11)])
def test_codes_in_expert_order(T, D, E, K, bad):
    g = torch.Generator().manual_seed(T)
    idx = torch.rand(T, E, generator=g).topk(K, 1).indices.to(torch.int32)
    idx.view(-1)[torch.randperm(T * K, generator=g)[:bad]] = E
    x = torch.randn(T, D, generator=g).to(BF16).to(DEV)
    plan = bw.permute_plan(idx.to(DEV), E)
    codes, scales = bw.quantize_tokens_int8(x, plan)
    alone, s = bw.quantize_tokens_int8(x)
    n = T * K - bad
    tok = plan.row_slot[:n].long() // K
    assert torch.equal(codes[:n], alone[tok]) and torch.equal(scales[:n], s[tok])
    assert (codes[n:] == 0).all() and (scales[n:] == 0).all()


def make_segments(counts, M):
    return torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32), M - sum(counts)


def make_codes(shape, seed, extreme=False):
    g = torch.Generator().manual_seed(seed)
    if extreme:
        return torch.full(shape, -128, dtype=I8)
    return torch.randint(-128, 128, shape, generator=g, dtype=torch.int16).to(I8)


# rows of each expert, rows without one, K, N
GROUPED = [([1], 0, 16, 16), ([3], 0, 4096, 512), ([0, 2, 0, 1], 2, 48, 32), ([130, 0, 5], 0, 144, 272), ([128, 256, 17], 40, 384, 1040),
           ([1, 300, 7, 0, 90], 3, 1408, 528), ([0, 0], 4, 64, 64), ([2] * 64, 0, 2048, 1408), ([33, 1, 64, 65, 31], 0, 2064, 256),
           ([600], 0, 512, 4112), ([0] * 255 + [9], 1, 128, 128), ([700] * 3, 0, 256, 768)]


@pytest.mark.parametrize("counts,loose,K,N", GROUPED)
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_grouped_product(counts, loose, K, N, dtype):
    M, E = sum(counts) + loose, len(counts)
    offsets, _ = make_segments(counts, M)
    a, w = make_codes((M, K), 1), make_codes((E, K, N), 2)
    g = torch.Generator().manual_seed(3)
    rs = torch.rand(M, generator=g) * 1e-2
    cs = torch.rand(E, N, generator=g) * 1e-3
    out = bw.int8_grouped_gemm(a.to(DEV), rs.to(DEV), offsets.to(DEV), w.to(DEV), cs.to(DEV), out_dtype=dtype).cpu()
    assert out.dtype == dtype and out.shape == (M, N)
    n = sum(counts)
    expert = torch.repeat_interleave(torch.arange(E), torch.tensor(counts))
    for e in range(E):
        rows = torch.nonzero(expert == e).flatten()
        if len(rows):
            acc = (a[rows].to(DEV).double() @ w[e].to(DEV).double()).cpu()             # whole numbers below 2^53: exact
            ref = acc * rs[rows, None].double() * cs[e].double()
            # the sum's conversion and two products, then the rounding to the type
            bound = ref.abs() * (3.01 * U32 + half_step(dtype) * 1.001) + smallest_step(dtype)
            assert ((out[rows].double() - ref).abs() <= bound).all(), e
    assert (out[n:] == 0).all()


def swiglu_bound(g, u, dtype):
    """silu(g) * u in fp32 from a gate and an up product that are 3 roundings off: the gate's error counts (1 + |g|) times in
    silu; the exponential is off by (2 + 1.16 |g|) steps, the quotient by 2, four more roundings."""
    ref = g * torch.sigmoid(g) * u
    rel = (3 * (1 + g.abs()) + 3 + 2 * (2 + 1.16 * g.abs()) + 4 + 4) * U32
    # below exp(-87) the quotient of the fast form is 0 instead of a number below 2^-118
    return ref, ref.abs() * (rel * 1.01 + half_step(dtype) * 1.001) + smallest_step(dtype) + u.abs() * 2.0 ** -118


@pytest.mark.parametrize("counts,loose,K,N", GROUPED)
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_grouped_swiglu(counts, loose, K, N, dtype):
    M, E = sum(counts) + loose, len(counts)
    offsets, _ = make_segments(counts, M)
    a, wg, wu = make_codes((M, K), 1), make_codes((E, K, N), 2), make_codes((E, K, N), 5)
    g = torch.Generator().manual_seed(3)
    rs = torch.rand(M, generator=g) * 1e-2
    sg, su = (torch.rand(E, N, generator=g) * 2e-2 / K ** 0.5 for _ in range(2))
    sg[:, ::7] *= 20                                # gates far on either side
    out = bw.int8_grouped_swiglu(a.to(DEV), rs.to(DEV), offsets.to(DEV), wg.to(DEV), wu.to(DEV), sg.to(DEV), su.to(DEV),
                                 out_dtype=dtype).cpu()
    expert = torch.repeat_interleave(torch.arange(E), torch.tensor(counts))
    for e in range(E):
        rows = torch.nonzero(expert == e).flatten()
        if len(rows):
            x = a[rows].to(DEV).double()
            gate, up = (((x @ w[e].to(DEV).double()).cpu() * rs[rows, None].double() * s[e].double()) for w, s in ((wg, sg), (wu, su)))
            ref, bound = swiglu_bound(gate, up, dtype)
            assert ((out[rows].double() - ref).abs() <= bound).all(), e
    assert (out[sum(counts):] == 0).all()


@pytest.mark.parametrize("K", [16, 2048, 131056])
@pytest.mark.parametrize("M", [1, 200])
def test_largest_sums(M, K):
    """-128 * -128 everywhere: 2^14 K, which for the largest K is just below 2^31."""
    a, w = make_codes((M, K), 0, True).to(DEV), make_codes((1, K, 32), 0, True).to(DEV)
    offsets = torch.tensor([0, M], dtype=torch.int32, device=DEV)
    out = bw.int8_grouped_gemm(a, torch.ones(M, device=DEV), offsets, w, torch.ones(1, 32, device=DEV), out_dtype=F32)
    assert (out == float(2 ** 14 * K)).all()      # 2^18 times a 13-bit number: exact in fp32


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("T,K,N", [(1, 16, 16), (1, 4096, 1024), (7, 2064, 272), (64, 1408, 2064), (517, 1408, 2064), (1500, 256, 640)])
def test_matmul(T, K, N, dtype):
    g = torch.Generator().manual_seed(T + K)
    x = torch.randn(T, K, generator=g).to(dtype)
    w, s = bw.quant_int8_channels(torch.randn(K, N, generator=g) * 0.02)
    out = bw.int8_matmul(x.to(DEV), w.to(DEV), s.to(DEV)).cpu()
    codes, scale = exact_codes(x)
    ref = (codes.to(DEV).double() @ w.to(DEV).double()).cpu() * scale[:, None].double() * s.double()
    assert ((out.double() - ref).abs() <= ref.abs() * (3.01 * U32 + half_step(dtype) * 1.001) + smallest_step(dtype)).all()


def make_block(T, D, H, E, K, dtype, seed, zipf=False):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(T, D, generator=g, device=DEV).to(dtype)
    logits = torch.randn(T, E, generator=g, device=DEV)
    if zipf:
        logits -= 1.1 * torch.log(torch.arange(1, E + 1, device=DEV).float())
    top, idx = logits.topk(K, 1)
    ws, ss = zip(*(bw.quantize_expert_weights_int8(torch.randn(E, a, b, generator=g, device=DEV) * 0.02)
                   for a, b in ((D, H), (D, H), (H, D))))
    return x, top.softmax(1), idx.to(torch.int32), ws, ss


BLOCKS = [(1, 64, 48, 4, 2, BF16, False), (64, 2048, 1408, 64, 6, BF16, False), (37, 256, 400, 16, 4, F16, True),
          (1003, 512, 768, 128, 8, F16, True), (3000, 256, 512, 8, 2, BF16, False), (300, 128, 16384 + 32, 2, 1, BF16, False)]


@pytest.mark.parametrize("T,D,H,E,K,dtype,zipf", BLOCKS)
def test_block_is_its_operators_in_a_row(T, D, H, E, K, dtype, zipf):
    x, weights, idx, (wg, wu, wd), (sg, su, sd) = make_block(T, D, H, E, K, dtype, T, zipf)
    if T > 5:
        idx[3, 0], idx[4, K - 1] = E, -1            # no expert: contributes nothing
    out = bw.int8_moe_forward_routed(x, weights, idx, wg, wu, wd, sg, su, sd)
    rows, plan = bw.permute_tokens(x, idx, E)
    codes, s = bw.quantize_tokens_int8(rows)
    assert all(torch.equal(a, b) for a, b in zip((codes, s), bw.quantize_tokens_int8(x, plan)))
    h = bw.int8_grouped_swiglu(codes, s, plan.offsets, wg, wu, sg, su, out_dtype=dtype)
    hq, sh = bw.quantize_tokens_int8(h)
    y = bw.int8_grouped_gemm(hq, sh, plan.offsets, wd, sd, out_dtype=dtype)
    assert torch.equal(out, bw.unpermute_tokens(y, plan, weights))
    # and against the definition in 64 bits, h and y rounded to the type.  Where the fp32 h lies next to a border of the
    # type (2^-20 of the 2^-8 between two bf16 numbers) it may round the other way, and move codes by one: far below the
    # rounding of the result, half a step at most.
    ref = torch.zeros(T, D, dtype=torch.float64, device=DEV)
    for e in range(E):
        t, k = torch.nonzero(idx == e, as_tuple=True)
        if len(t) == 0:
            continue
        c, sc = (v.to(DEV) for v in exact_codes(x[t]))
        gate, up = (c.double() @ w[e].double() * sc[:, None].double() * ws[e].double() for w, ws in ((wg, sg), (wu, su)))
        c, sc = (v.to(DEV) for v in exact_codes((gate * torch.sigmoid(gate) * up).to(dtype)))
        y64 = (c.double() @ wd[e].double() * sc[:, None].double() * sd[e].double()).to(dtype).double()
        ref.index_add_(0, t, y64 * weights[t, k, None].double())
    assert (out.double() - ref).norm() <= ref.norm() * (half_step(dtype) + 1e-3)


@pytest.mark.parametrize("T,E,K", [(1, 8, 2), (130, 16, 2), (700, 64, 6), (2100, 8, 1)])
def test_block_with_its_router(T, E, K):
    D, H = 256, 512
    x, _, _, ws, ss = make_block(T, D, H, E, K, BF16, 3)
    gate = (torch.randn(D, E, device=DEV) * 0.02).to(BF16)
    out = bw.int8_moe_forward(x, gate, *ws, *ss, top_k=K)
    assert torch.equal(out, bw.int8_moe_forward_routed(x, *bw.top_k_router(x, gate, K), *ws, *ss))


@pytest.mark.parametrize("T", [20, 1500])
def test_status_words_and_reserved_sms(T):
    """The C entry points: the workspace's status word tells of an expert id out of range, and of nothing else; SMs left free
    change no result."""
    import ctypes
    from blackwell_moe_b200 import _lib
    lib, stream = bw.lib(), torch.cuda.current_stream().cuda_stream
    D, H, E, K = 256, 512, 8, 2
    x, weights, idx, ws, ss = make_block(T, D, H, E, K, BF16, 2)
    n = lib.bwmoe_workspace_bytes_int(T, D, H, E, K)
    space = torch.full((n,), 0xff, dtype=torch.uint8, device=DEV)          # whatever was there before
    status = ctypes.c_int32(-1)

    def call(ids):
        out = torch.empty_like(x)
        _lib.check(lib.bwmoe_moe_forward_int_routed(x.data_ptr(), weights.data_ptr(), ids.data_ptr(), *[t.data_ptr() for t in ws],
                                                    *[t.data_ptr() for t in ss], T, D, H, E, K, 0, out.data_ptr(),
                                                    space.data_ptr(), n, stream))
        _lib.check(lib.bwmoe_read_status(space.data_ptr(), stream, ctypes.byref(status)))
        return out

    want = call(idx)
    assert status.value == 0
    bad = idx.clone()
    bad[7, 1] = E
    call(bad)
    assert status.value == 2
    for reserve in (100, 127):
        assert lib.bwmoe_set_sm_reserve(reserve) == 0
        try:
            got = call(idx)
        finally:
            lib.bwmoe_set_sm_reserve(0)
        assert status.value == 0 and torch.equal(got, want)


def test_block_beside_the_reference_in_bf16():
    """Four quantisations (x, gate/up, h, down), each off by scale / sqrt(12) with scale = amax / 127: about 0.9 % where the
    largest is 4 standard deviations, 2 % for the heavier tails of h.  Together below 4 %."""
    import oracle
    from helpers import make_inputs
    inp = make_inputs(96, 512, 8, 2, 256, seed=2)
    ref = oracle.moe_forward_bf16(inp["x"], inp["w_gate"], inp["bf_gate"], inp["bf_up"], inp["bf_down"], top_k=2)
    ws, ss = zip(*(bw.quantize_expert_weights_int8(inp[k].to(DEV)) for k in ("bf_gate", "bf_up", "bf_down")))
    out = bw.int8_moe_forward(inp["x"].to(DEV), inp["w_gate"].to(DEV), *ws, *ss, top_k=2).cpu()
    assert oracle.rel_l1(out, ref) < 0.04


def test_empty_batches():
    x, w, idx, ws, ss = make_block(4, 64, 48, 4, 2, BF16, 0)
    assert bw.int8_moe_forward_routed(x[:0], w[:0], idx[:0], *ws, *ss).shape == (0, 64)
    assert bw.int8_matmul(x[:0], ws[0][0], ss[0][0]).shape == (0, 48)
    codes, s = bw.quantize_tokens_int8(x[:0])
    assert codes.shape == (0, 64) and s.shape == (0,)
    none = torch.zeros(5, dtype=torch.int32, device=DEV)
    assert bw.int8_grouped_gemm(codes, s, none, ws[0], ss[0]).shape == (0, 48)


@pytest.mark.parametrize("T", [1, 9, 700])
def test_streams_and_captured_graphs(T):
    D, H, E, K = 256, 512, 16, 4
    x, weights, idx, ws, ss = make_block(T, D, H, E, K, BF16, 5)

    def step():
        return bw.int8_moe_forward_routed(x, weights, idx, *ws, *ss), bw.int8_matmul(x, ws[0][0], ss[0][0])

    want = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step()
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for _ in range(4):
        x.normal_()
        weights.copy_(torch.rand_like(weights))
        idx.copy_(torch.rand(T, E, device=DEV).topk(K, 1).indices)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(captured, step()))


@pytest.mark.parametrize("T", [3, 40, 600])
def test_graphs_that_are_replayed_side_by_side(T):
    """Two graphs captured on one stream, replayed on two at once: they have no workspace in common."""
    D, H, E, K = 512, 1024, 8, 2
    sets = [make_block(T, D, H, E, K, BF16, seed) for seed in (1, 2)]
    graphs, outs = [], []
    for x, weights, idx, ws, ss in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append((bw.int8_moe_forward_routed(x, weights, idx, *ws, *ss), bw.int8_matmul(x, ws[0][0], ss[0][0])))
    want = [(bw.int8_moe_forward_routed(x, weights, idx, *ws, *ss), bw.int8_matmul(x, ws[0][0], ss[0][0]))
            for x, weights, idx, ws, ss in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for got, ref in zip(outs, want):
        assert all(torch.equal(a, b) for a, b in zip(got, ref))


def test_two_streams_at_once():
    x, weights, idx, ws, ss = make_block(50, 512, 1024, 8, 2, BF16, 4)
    want = bw.int8_moe_forward_routed(x, weights, idx, *ws, *ss)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(20):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(bw.int8_moe_forward_routed(x, weights, idx, *ws, *ss))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_two_threads_on_one_stream():
    """Calls are several launches: those of two threads interleave on the stream, and their workspaces must not be one."""
    import threading
    sets = [make_block(T, 512, 1024, 8, 2, BF16, T) for T in (5, 90)]
    call = lambda s: (bw.int8_moe_forward_routed(*s[:3], *s[3], *s[4]), bw.int8_matmul(s[0], s[3][0][0], s[4][0][0]))      # noqa: E731
    want = [call(s) for s in sets]
    torch.cuda.synchronize()
    got, threads = [[], []], []
    for i, s in enumerate(sets):
        threads.append(threading.Thread(target=lambda i=i, s=s: [got[i].append(call(s)) for _ in range(150)]))
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for outs, ref in zip(got, want):
        assert len(outs) == 150 and all(torch.equal(a, b) for out in outs for a, b in zip(out, ref))


def test_workspaces_go_with_their_thread():
    import threading
    w, s = bw.quant_int8_channels(torch.randn(2048, 4096, device=DEV))
    x = torch.randn(3, 2048, device=DEV).to(BF16)
    want = bw.int8_matmul(x, w, s)
    torch.cuda.synchronize()
    before, together, same = torch.cuda.memory_allocated(), threading.Barrier(4, timeout=60), []
    kept = []

    def work():
        same.append(bool(torch.equal(bw.int8_matmul(x, w, s), want)))
        together.wait()                          # all live at once: every one has its own
        kept.append(torch.cuda.memory_allocated())
        together.wait()

    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert same == [True] * 4 and min(kept) >= before + 4 * bw.lib().bwmoe_workspace_bytes_int_matmul(3, 2048, 4096)
    assert torch.cuda.memory_allocated() == before
    bw.moe.release_workspaces()
    assert torch.cuda.memory_allocated() < before
    assert torch.equal(bw.int8_matmul(x, w, s), want)


def test_the_same_workspace_for_batches_of_all_sizes():
    """The stream's workspace carries what the call before left in it: sizes up and down, cut tiles and uncut ones."""
    D, H, E, K = 512, 2048, 8, 2
    x, weights, idx, ws, ss = make_block(1500, D, H, E, K, BF16, 6)
    first = {}
    for T in (1, 1500, 7, 130, 1, 513, 40, 1500, 130, 7, 513, 40):
        out = bw.int8_moe_forward_routed(x[:T].contiguous(), weights[:T].contiguous(), idx[:T].contiguous(), *ws, *ss)
        lin = bw.int8_matmul(x[:T].contiguous(), ws[0][3], ss[0][3])
        if T in first:
            assert torch.equal(out, first[T][0]) and torch.equal(lin, first[T][1])
        first[T] = (out, lin)
    # a token's row does not depend on the rows beside it, nor on the kernel that its batch got
    assert torch.equal(first[1][1], first[1500][1][:1]) and torch.equal(first[130][0], first[1500][0][:130])


def test_segments_from_elsewhere_stay_inside_the_rows():
    """Offsets past the rows, negative or falling: clamped, nothing is read or written out of range."""
    M, K, N, E = 40, 64, 64, 3
    a, w = make_codes((M, K), 1).to(DEV), make_codes((E, K, N), 2).to(DEV)
    rs, cs = torch.ones(M, device=DEV), torch.ones(E, N, device=DEV)
    for offsets in ([0, 10, 30, 4000], [-7, 10, 30, 40], [0, 2 ** 31 - 1, 30, 40], [40, 40, 40, 40], [40, 10, 5, 0]):
        out = bw.int8_grouped_gemm(a, rs, torch.tensor(offsets, dtype=torch.int32, device=DEV), w, cs, out_dtype=F32)
        torch.cuda.synchronize()
        if offsets[0] > 0:
            assert (out == 0).all()
        if offsets[1:3] == [10, 30]:
            for e, (lo, hi) in enumerate(((0, 10), (10, 30), (30, 40))):
                assert torch.equal(out[lo:hi].double(), a[lo:hi].double() @ w[e].double())


@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("counts,loose,K,N", [([5000, 4000], 7, 4096, 8192), ([8200], 0, 8192, 6144), ([0, 3001, 257, 9000, 1], 300, 4096, 7680),
                                                ([900, 1, 0, 2500, 700, 1111, 890, 1500], 5, 1408, 8192)])
def test_long_products(counts, loose, K, N, swiglu):
    """Products long enough for CTA pairs, with segments that end anywhere in a pair's tile; some rows are compared."""
    M, E = sum(counts) + loose, len(counts)
    offsets, _ = make_segments(counts, M)
    g = torch.Generator(device=DEV).manual_seed(9)
    codes = lambda *shape: torch.randint(-128, 128, shape, generator=g, device=DEV, dtype=torch.int16).to(I8)     # noqa: E731
    a, w, w2 = codes(M, K), codes(E, K, N), codes(E, K, N)
    rs = torch.rand(M, generator=g, device=DEV) * 1e-2
    cs, cs2 = (torch.rand(E, N, generator=g, device=DEV) * 2e-4 for _ in range(2))
    if swiglu:
        out = bw.int8_grouped_swiglu(a, rs, offsets.to(DEV), w, w2, cs, cs2)
    else:
        out = bw.int8_grouped_gemm(a, rs, offsets.to(DEV), w, cs)
    for e in range(E):
        lo, hi = int(offsets[e]), int(offsets[e + 1])
        rows = sorted({r for r in (lo, lo + 1, lo + 127, lo + 128, lo + 255, lo + 256, (lo + hi) // 2, hi - 129, hi - 2, hi - 1) if lo <= r < hi})
        if not rows:
            continue
        x, r = a[rows].double(), rs[rows, None].double()
        gate = (x @ w[e].double()) * r * cs[e].double()
        if swiglu:
            ref, bound = swiglu_bound(gate, (x @ w2[e].double()) * r * cs2[e].double(), BF16)
        else:
            ref, bound = gate, gate.abs() * (3.01 * U32 + half_step(BF16) * 1.001) + smallest_step(BF16)
        assert ((out[rows].double() - ref).abs() <= bound).all(), e
    assert (out[sum(counts):] == 0).all()


def test_a_long_matmul():
    """Quantisation in front of a product on CTA pairs."""
    T, K, N = 8200, 4096, 12288
    g = torch.Generator(device=DEV).manual_seed(2)
    x = torch.randn(T, K, generator=g, device=DEV).to(BF16)
    w, s = bw.quant_int8_channels(torch.randn(K, N, generator=g, device=DEV) * 0.02)
    out = bw.int8_matmul(x, w, s)
    rows = [0, 1, 127, 128, 255, 256, 4000, 8191, 8192, 8198, 8199]
    codes, scale = (v.to(DEV) for v in exact_codes(x[rows].cpu()))
    ref = (codes.double() @ w.double()) * scale[:, None].double() * s.double()
    assert ((out[rows].double() - ref).abs() <= ref.abs() * (3.01 * U32 + half_step(BF16) * 1.001) + smallest_step(BF16)).all()


def test_rows_in_front_of_the_first_segment_are_zero():
    a, w = make_codes((300, 64), 1).to(DEV), make_codes((2, 64, 48), 2).to(DEV)
    rs, cs = torch.ones(300, device=DEV), torch.ones(2, 48, device=DEV)
    out = bw.int8_grouped_gemm(a, rs, torch.tensor([9, 100, 290], dtype=torch.int32, device=DEV), w, cs, out_dtype=F32)
    assert (out[:9] == 0).all() and (out[290:] == 0).all()
    for e, (lo, hi) in enumerate(((9, 100), (100, 290))):
        assert torch.equal(out[lo:hi].double(), a[lo:hi].double() @ w[e].double())


def test_quotients_of_all_pairs_of_16_bit_numbers():
    """Rows whose largest value runs through every significand, with every smaller value from a 512th of it on: all the ties,
    and all that lies next to one."""
    for dtype, bits in ((BF16, 8), (F16, 11)):
        ints = torch.arange(2 ** (bits - 1), 2 ** bits).float()
        values = torch.cat([ints * 2.0 ** -s for s in range(1, 10)] + [ints])
        x = values.repeat(len(ints), 1)
        x[x > ints[:, None]] = 0
        x[:, 1::2] *= -1
        x[torch.arange(len(ints)), len(values) - len(ints) + torch.arange(len(ints))] = ints
        for scale in (1.0, 2.0 ** -9):
            y = (x * scale).to(dtype)
            assert_codes(*bw.quantize_tokens_int8(y.to(DEV)), y)


def test_more_tiles_than_22_bits_count():
    """More than 2^22 tiles of 128 short rows: the ones at the end, too."""
    M, K, N = 2 ** 29 + 40000, 16, 16
    codes = torch.zeros(M, K, dtype=I8, device=DEV)
    w = make_codes((1, K, N), 2).to(DEV)
    rs, cs = torch.ones(M, device=DEV), torch.ones(1, N, device=DEV)
    places = [slice(0, 300), slice(2 ** 28 - 200, 2 ** 28 + 200), slice(2 ** 29 - 200, 2 ** 29 + 200), slice(M - 300, M)]
    for i, rows in enumerate(places):
        codes[rows] = make_codes((rows.stop - rows.start, K), 3 + i).to(DEV)
    for offsets in ([0, M], [0, M - 7]):
        out = bw.int8_grouped_gemm(codes, rs, torch.tensor(offsets, dtype=torch.int32, device=DEV), w, cs, out_dtype=F32)
        for rows in places:
            want = codes[rows].double() @ w[0].double()
            if rows.stop > offsets[1]:
                want[offsets[1] - rows.start:] = 0
            assert torch.equal(out[rows].double(), want), (offsets, rows)
        assert int(torch.count_nonzero(out[300:2 ** 28 - 200])) + int(torch.count_nonzero(out[2 ** 29 + 200:M - 300])) == 0
        del out
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M", [5, 300])
def test_scales_of_any_size(M, dtype):
    """Infinity only where the product itself is that large: sums of 2^20 and more times a scale of 1e33 on either side, the other
    one small.  Rows and channels of every size meet; both kernels, plain and SwiGLU."""
    K, N, E = 4096, 320, 2
    a, w = make_codes((M, K), 1), make_codes((E, K, N), 2)
    a[:, :64], w[:, :64] = 127, 127                     # no sum near zero
    a[0], w[1, :, 3] = 0, 0                             # but these are
    offsets = torch.tensor([0, M // 2, M], dtype=torch.int32)
    rs = torch.tensor([1.0, 1e33, 1e-4, 3e-39, 1e-33, 2e29])[torch.arange(M) % 6]
    cs = torch.tensor([1e-4, 1e33, 1.0, 1e-33, 3e-39, 2e29])[torch.arange(E * N) % 6].view(E, N)
    args = [t.to(DEV) for t in (a, rs, offsets, w, cs)]
    out = bw.int8_grouped_gemm(*args, out_dtype=dtype)
    ones = torch.full((E, N), 1e-3, device=DEV)         # gates of ordinary rows; up products of every size
    h = bw.int8_grouped_swiglu(args[0], args[1], args[2], args[3], args[3], ones, args[4], out_dtype=dtype)
    seen = 0
    top = torch.finfo(dtype).max
    for e, (lo, hi) in enumerate(((0, M // 2), (M // 2, M))):
        acc = args[0][lo:hi].double() @ args[3][e].double()
        ref = acc * args[1][lo:hi, None].double() * args[4][e].double()
        fits, past = ref.abs() <= top * (1 - 2.0 ** -7), ref.abs() > top * (1 + 2.0 ** -7)
        bound = ref.abs() * (3.01 * U32 + half_step(dtype) * 1.001) + smallest_step(dtype)
        seen += int(past.sum())
        assert ((out[lo:hi].double() - ref).abs() <= bound)[fits].all(), e
        assert (out[lo:hi].isinf() & (out[lo:hi].double().sign() == ref.sign()))[past].all(), e
        gate = acc * args[1][lo:hi, None].double() * ones[0, 0].double()
        want, bound = swiglu_bound(gate, ref, dtype)
        live = fits & (want.abs() <= top * (1 - 2.0 ** -7)) & (gate.abs() < 1e3)
        assert live.any() and ((h[lo:hi].double() - want).abs() <= bound)[live].all(), e
    assert seen


@pytest.mark.parametrize("counts,loose,K,N", GROUPED)
def test_swiglu_is_rounded_to_16_bits_once(counts, loose, K, N):
    """bf16 and fp16 results are the fp32 results rounded, and those are within the accurate functions' errors: the gate's three
    roundings times (1 + |g|), the exponential's 2 steps, the sum, the quotient, the product, and up's three - a bound that does not
    grow with |g| otherwise."""
    M, E = sum(counts) + loose, len(counts)
    offsets, _ = make_segments(counts, M)
    a, wg, wu = make_codes((M, K), 1), make_codes((E, K, N), 2), make_codes((E, K, N), 5)
    g = torch.Generator().manual_seed(3)
    rs = torch.rand(M, generator=g) * 1e-2
    sg, su = (torch.rand(E, N, generator=g) * 2e-2 / K ** 0.5 for _ in range(2))
    sg[:, ::7] *= 20
    args = [t.to(DEV) for t in (a, rs, offsets, wg, wu, sg, su)]
    out = {t: bw.int8_grouped_swiglu(*args, out_dtype=t) for t in (BF16, F16, F32)}
    expert = torch.repeat_interleave(torch.arange(E), torch.tensor(counts)).to(DEV)
    for e in range(E):
        rows = torch.nonzero(expert == e).flatten()
        if len(rows):
            x, r = args[0][rows].double(), args[1][rows, None].double()
            gate, up = ((x @ w[e].double()) * r * s[e].double() for w, s in ((args[3], args[5]), (args[4], args[6])))
            near = gate > -87
            ref = gate * torch.sigmoid(gate) * up
            rel = (3 * (1 + gate.abs()) + 2 * 2 + 1 + 1 + 1 + 3) * U32 * 1.001
            got = out[F32][rows].double()
            assert ((got - ref).abs() <= ref.abs() * rel + 2.0 ** -149)[near].all(), e
            for t in (BF16, F16):
                bits = out[t][rows], out[F32][rows].to(t)
                # once in a million the quotient is rounded the other way; with that, once in 2^8 or less the 16 bits
                assert int((bits[0] != bits[1])[near].sum()) <= 1, (e, t)


def test_ids_of_64_bits_do_not_wrap_around():
    """2^32 + 1 is no expert, not expert 1; valid ids in 64 bits are what they are in 32."""
    x, weights, idx, ws, ss = make_block(30, 256, 512, 8, 2, BF16, 1)
    assert torch.equal(bw.int8_moe_forward_routed(x, weights, idx.long(), *ws, *ss), bw.int8_moe_forward_routed(x, weights, idx, *ws, *ss))
    wide, none = idx.long(), idx.clone()
    for t, id64 in enumerate((2 ** 32 + 1, -2 ** 32, 2 ** 40 + 3, -2 ** 63, 2 ** 63 - 1, 8, -1)):
        wide[t, t % 2], none[t, t % 2] = id64, -1
    assert torch.equal(bw.int8_moe_forward_routed(x, weights, wide, *ws, *ss), bw.int8_moe_forward_routed(x, weights, none, *ws, *ss))


def test_a_backward_pass_through_the_integers_says_that_there_is_none():
    """The operators stand among differentiable ones: a gradient that ends in them must not do so silently."""
    from torch.autograd import forward_ad as fw
    x, weights, idx, (wg, wu, wd), (sg, su, sd) = make_block(6, 64, 64, 4, 2, BF16, 0)
    gate = torch.randn(64, 4, device=DEV).to(BF16)
    rows, plan = bw.permute_tokens(x, idx, 4)
    codes, s = bw.quantize_tokens_int8(rows)
    calls = [(lambda x: bw.quantize_tokens_int8(x)[1], x), (lambda x: bw.quantize_tokens_int8(x, plan)[1], x),
             (lambda s: bw.int8_grouped_gemm(codes, s, plan.offsets, wg, sg), s), (lambda sg: bw.int8_grouped_gemm(codes, s, plan.offsets, wg, w_scales=sg), sg),
             (lambda s: bw.int8_grouped_swiglu(codes, s, plan.offsets, wg, wu, sg, su, out_dtype=F32), s),
             (lambda x: bw.int8_matmul(x, wg[0], sg[0]), x), (lambda x: bw.int8_moe_forward_routed(x, weights, idx, wg, wu, wd, sg, su, sd), x),
             (lambda w: bw.int8_moe_forward_routed(x, w, idx, wg, wu, wd, sg, su, scales_down=sd), weights),
             (lambda x: bw.int8_moe_forward(x, gate, wg, wu, wd, sg, su, sd, top_k=2), x)]
    for call, t in calls:
        want, leaf = call(t), t.clone().requires_grad_()
        out = call(leaf)
        assert torch.equal(out.detach(), want) and not want.requires_grad
        with pytest.raises(NotImplementedError, match="has no gradient"):
            (leaf.float().sum() + out.float().sum()).backward()
        with torch.no_grad():
            assert torch.equal(call(leaf), want) and not call(leaf).requires_grad
        with fw.dual_level():
            with pytest.raises(NotImplementedError):
                call(fw.make_dual(t, torch.ones_like(t)))
            assert torch.equal(call(t), want)
    assert not bw.quantize_tokens_int8(x.clone().requires_grad_())[0].requires_grad


def test_the_same_rows_in_tiles_of_both_heights():
    """One tensor of codes, read by the kernel of 32-row tiles and by that of 128-row tiles in turn: the descriptors of its rows
    are kept by address and shape, and by the tile's height."""
    M, K = 300, 512
    a, rs = make_codes((M, K), 1).to(DEV), torch.ones(M, device=DEV)
    few, many = make_codes((16, K, 256), 2).to(DEV), make_codes((1, K, 16384), 3).to(DEV)
    bounds = [19 * e for e in range(16)] + [M]
    for _ in range(2):
        out = bw.int8_grouped_gemm(a, rs, torch.tensor(bounds, dtype=torch.int32, device=DEV), few, torch.ones(16, 256, device=DEV), out_dtype=F32)
        for e in range(16):
            assert torch.equal(out[bounds[e]:bounds[e + 1]].double(), a[bounds[e]:bounds[e + 1]].double() @ few[e].double())
        out = bw.int8_grouped_gemm(a, rs, torch.tensor([0, M], dtype=torch.int32, device=DEV), many, torch.ones(1, 16384, device=DEV), out_dtype=F32)
        assert torch.equal(out.double(), a.double() @ many[0].double())


def check_rows_against_64_bits(out, rows_of, a, rs, offsets, ws, ss, dtype):
    """Rows rows_of(lo, hi) of each segment against the definition: one product, or SwiGLU of two."""
    for e in range(len(offsets) - 1):
        rows = rows_of(offsets[e], offsets[e + 1])
        if not len(rows):
            continue
        x, r = a[rows].double(), rs[rows, None].double()
        products = [(x @ w[e].double()) * r * s[e].double() for w, s in zip(ws, ss)]
        if len(products) == 2:
            ref, bound = swiglu_bound(*products, dtype)
        else:
            ref, bound = products[0], products[0].abs() * (3.01 * U32 + half_step(dtype) * 1.001) + smallest_step(dtype)
        assert ((out[rows].double() - ref).abs() <= bound).all(), e


def random_product(counts, loose, K, N, swiglu, seed=9):
    M, E = sum(counts) + loose, len(counts)
    offsets, _ = make_segments(counts, M)
    g = torch.Generator(device=DEV).manual_seed(seed)
    codes = lambda *shape: torch.randint(-128, 128, shape, generator=g, device=DEV, dtype=torch.int16).to(I8)     # noqa: E731
    a, ws = codes(M, K), [codes(E, K, N) for _ in range(1 + swiglu)]
    rs = torch.rand(M, generator=g, device=DEV) * 1e-2
    ss = [torch.rand(E, N, generator=g, device=DEV) * 2e-2 / K ** 0.5 for _ in ws]
    return a, rs, offsets, ws, ss


def product(a, rs, offsets, ws, ss, dtype):
    call = bw.int8_grouped_swiglu if len(ws) == 2 else bw.int8_grouped_gemm
    return call(a, rs, offsets.to(DEV), *ws, *ss, out_dtype=dtype)


# (rows of each expert, rows of none, K, N, SwiGLU): 128-row tiles so few, and K so long, that their K loops are cut on 148 SMs - into
# 3, 2, 2 and 5 slices, and into 2, 3 and 2 with two products; the last tiles of some have one weight box, or one that hangs over N
CUT = [([256], 0, 14336, 4096, False), ([300], 0, 8192, 3984, False), ([200, 0, 130], 5, 8192, 3216, False), ([256], 0, 14336, 2064, False),
       ([300], 0, 8192, 2048, True), ([300], 9, 14336, 1488, True), ([250, 3, 140], 0, 12288, 1040, True)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("counts,loose,K,N,swiglu", CUT)
def test_cut_tiles_of_128_rows(counts, loose, K, N, swiglu, dtype):
    case = random_product(counts, loose, K, N, swiglu)
    out = product(*case, dtype)
    a, rs, offsets, ws, ss = case
    check_rows_against_64_bits(out, lambda lo, hi: list(range(lo, hi)), a, rs, offsets.tolist(), ws, ss, dtype)
    assert (out[sum(counts):] == 0).all()


def test_cut_tiles_one_after_the_other():
    """Products of other tiles and slices in a row, with the slabs and counters that the one before left; twice each, and
    inside a graph."""
    cases = [random_product(*c) for c in CUT]
    first = [product(*c, F32) for c in cases]
    again = [product(*c, F32) for c in cases for _ in range(2)]
    assert all(torch.equal(x, first[i // 2]) for i, x in enumerate(again))
    graph = torch.cuda.CUDAGraph()
    dev = [(a, rs, offsets.to(DEV), ws, ss) for a, rs, offsets, ws, ss in cases]
    with torch.cuda.graph(graph):
        captured = [product(*c, F32) for c in dev]
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(captured, first))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("counts,loose,K,N,swiglu", [([5000, 4000], 7, 4096, 8192, False), ([5000, 4000], 7, 4096, 8192, True), ([4200], 0, 8192, 5904, True),
                                                     ([2100, 2200], 3, 4096, 12304, True), ([8200], 0, 8192, 6144, False)])
def test_long_products_in_every_type(counts, loose, K, N, swiglu, dtype):
    """CTA pairs; with SwiGLU also where the last weight box of a pair's tile hangs over N."""
    a, rs, offsets, ws, ss = random_product(counts, loose, K, N, swiglu)
    out = product(a, rs, offsets, ws, ss, dtype)
    ends = lambda lo, hi: sorted({r for r in (lo, lo + 1, lo + 127, lo + 128, lo + 255, lo + 256, (lo + hi) // 2, hi - 129, hi - 2, hi - 1) if lo <= r < hi})      # noqa: E731
    check_rows_against_64_bits(out, ends, a, rs, offsets.tolist(), ws, ss, dtype)
    assert (out[sum(counts):] == 0).all()


@pytest.mark.parametrize("dtype,code", [(BF16, 0), (F16, 1), (F32, 2)])
@pytest.mark.parametrize("counts,loose,K,N,swiglu", [([3, 20], 1, 256, 272, False), ([200, 150], 3, 256, 272, False), ([200, 150], 3, 256, 272, True),
                                                     ([256], 0, 14336, 2064, False), ([5000, 4000], 7, 4096, 8192, False)])
def test_results_at_16_byte_aligned_addresses(counts, loose, K, N, swiglu, dtype, code):
    """Through the C entries a result may lie at any multiple of 16 bytes: nothing around it is written."""
    from blackwell_moe_b200 import _lib
    lib = bw.lib()
    a, rs, offsets, ws, ss = random_product(counts, loose, K, N, swiglu)
    offsets = offsets.to(DEV)
    want, (M, E) = product(a, rs, offsets, ws, ss, dtype), (a.shape[0], len(counts))
    n = lib.bwmoe_int_scratch_bytes(M, K, N, E)
    scratch = torch.empty(n, dtype=torch.uint8, device=DEV)
    pad = 16 * 8 // torch.finfo(dtype).bits
    space = torch.full((M * N + 2 * pad,), 7.0, dtype=dtype, device=DEV)
    fn = lib.bwmoe_int_gateup_swiglu if swiglu else lib.bwmoe_int_grouped_gemm
    _lib.check(fn(a.data_ptr(), rs.data_ptr(), offsets.data_ptr(), *[w.data_ptr() for w in ws], *[s.data_ptr() for s in ss], M, K, N, E,
                  code, space.data_ptr() + 16, scratch.data_ptr(), n, torch.cuda.current_stream().cuda_stream))
    assert space.data_ptr() % 32 == 0
    assert torch.equal(space[pad:-pad].view(M, N), want) and (space[:pad] == 7).all() and (space[-pad:] == 7).all()


def test_codes_into_more_rows_than_the_permutation_takes():
    """A plan made elsewhere with 40 slots per token: the quantiser has no limit of 32."""
    T, D, K = 9, 64, 40
    g = torch.Generator().manual_seed(4)
    x = torch.randn(T, D, generator=g).to(BF16).to(DEV)
    pos = torch.randperm(T * K, generator=g).to(DEV, torch.int32).view(T, K)
    plan = bw.PermutePlan(torch.tensor([0, T * K], dtype=torch.int32, device=DEV), pos)
    codes, s = bw.quantize_tokens_int8(x, plan)
    alone, scale = bw.quantize_tokens_int8(x)
    assert torch.equal(codes[pos.long()], alone[:, None].expand(T, K, D)) and torch.equal(s[pos.long()], scale[:, None].expand(T, K))
