"""Tokens into expert order and back (permute_tokens, unpermute_tokens) against the definition in 64 bits, and their
gradients against the formulas and against differences."""

import pytest
import torch

import blackwell_moe_b200 as bw

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U32 = 2.0 ** -24                                 # half a step of fp32


def routing(T, E, K, seed, bad=0):
    g = torch.Generator().manual_seed(seed)
    idx = torch.rand(T, E, generator=g).topk(K, dim=1).indices.to(torch.int32)
    flat = idx.view(-1)
    for i, v in zip(torch.randperm(flat.numel(), generator=g)[:bad].tolist(), [-1, E, 2 ** 30, -2 ** 31] * bad):
        flat[i] = v
    return idx, torch.rand(T, K, generator=g)


def reference_plan(idx, E):
    """Stable sort by expert on the CPU; ids out of range have no row."""
    flat = idx.reshape(-1).long()
    ok = (flat >= 0) & (flat < E)
    slots = torch.nonzero(ok).flatten()
    order = slots[torch.sort(flat[slots], stable=True).indices]
    pos = torch.full_like(flat, -1)
    pos[order] = torch.arange(order.numel())
    offsets = torch.zeros(E + 1, dtype=torch.int64)
    offsets[1:] = torch.bincount(flat[slots], minlength=E).cumsum(0)
    return pos.view(idx.shape), offsets, order


CASES = [(1, 16, 8, 1, BF16, 0), (1, 1, 1, 1, F32, 0), (5, 33, 8, 3, F16, 2), (64, 2048, 64, 6, BF16, 0), (37, 100, 60, 32, F32, 9),
         (1003, 130, 128, 8, F32, 0), (171, 2050, 16, 6, BF16, 40), (2100, 264, 256, 1, F16, 0), (400, 1024, 8, 2, BF16, 800),
         (9, 4100, 12, 9, F16, 1), (4096, 64, 200, 5, BF16, 3)]


@pytest.mark.parametrize("T,D,E,K,dtype,bad", CASES)
def test_forward_and_gradients(T, D, E, K, dtype, bad):
    idx, w = routing(T, E, K, T + D, bad)
    g = torch.Generator().manual_seed(7)
    x = torch.randn(T, D, generator=g).to(dtype)
    drows, dout = torch.randn(T * K, D, generator=g).to(dtype), torch.randn(T, D, generator=g).to(dtype)
    pos, offsets, order = reference_plan(idx, E)
    n = order.numel()
    M, half = T * K, torch.finfo(dtype).eps / 2 if dtype != F32 else 0.0

    xg = x.to(DEV).requires_grad_()
    rows, plan = bw.permute_tokens(xg, idx.to(DEV), E)
    assert torch.equal(plan.pos.cpu().long(), pos) and torch.equal(plan.offsets.cpu().long(), offsets)
    assert torch.equal(plan.row_slot.cpu().long()[:n], order) and (plan.row_slot.cpu()[n:] == -1).all()
    want = torch.zeros(M, D, dtype=dtype)
    want[:n] = x[order // K]
    assert torch.equal(rows.detach().cpu(), want)
    rows2, _ = bw.permute_tokens(xg, plan=plan)
    assert torch.equal(rows2, rows)
    alone = bw.permute_plan(idx.to(DEV), E)
    assert all(torch.equal(a, b) for a, b in zip(alone, plan))

    # dx: K fp32 additions, one rounding
    dx, = torch.autograd.grad(rows, xg, drows.to(DEV))
    d64 = torch.cat([drows.double(), torch.zeros(1, D, dtype=torch.float64)])[pos]          # pos -1: the zero row
    ref, size = d64.sum(1), d64.abs().sum(1)
    assert ((dx.cpu().double() - ref).abs() <= ref.abs() * half * (1 + 2 * K * U32) + 2 * K * U32 * size).all()

    # out and its gradients
    rg, wg = rows.detach().clone(), w.to(DEV).requires_grad_()
    rg[n:] = float("nan")                         # rows that no slot owns are never read
    rg.requires_grad_()
    out = bw.unpermute_tokens(rg, plan, wg)
    r64 = torch.cat([want.double(), torch.zeros(1, D, dtype=torch.float64)])[pos]
    terms = w.double().unsqueeze(2) * r64
    ref, size = terms.sum(1), terms.abs().sum(1)
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps      # a step below the normal numbers
    assert ((out.detach().cpu().double() - ref).abs() <= ref.abs() * half * (1 + 2 * K * U32) + 2 * K * U32 * size + tiny).all()
    drg, dwg = torch.autograd.grad(out, (rg, wg), dout.to(DEV))
    live = w.double().reshape(-1)[order].unsqueeze(1) * dout.double()[order // K]
    err = (drg.cpu().double()[:n] - live).abs()
    assert (err <= live.abs() * (half + U32) * 1.001 + tiny).all() and (drg[n:] == 0).all()
    prod = r64 * dout.double().unsqueeze(1)
    steps = D / 32 + 8 + 5 + 8                    # additions that follow one another: a lane's, the lanes', the warps'
    assert ((dwg.cpu().double() - prod.sum(2)).abs() <= (steps + 1) * U32 * 1.01 * prod.abs().sum(2)).all()
    assert (dwg.cpu()[pos < 0] == 0).all()

    # one gradient at a time gives the same; and without weights
    only_r, none = bw.unpermute_tokens_backward(dout.to(DEV), None, plan, wg.detach(), weights_grad=False)
    assert none is None and torch.equal(only_r, drg)
    none, only_w = bw.unpermute_tokens_backward(dout.to(DEV), rg.detach(), plan, wg.detach(), rows_grad=False)
    assert none is None and torch.equal(only_w, dwg)
    plain = bw.unpermute_tokens(rg, plan)
    dplain, = torch.autograd.grad(plain, rg, dout.to(DEV))
    assert torch.equal(plain, bw.unpermute_tokens(rg, plan, torch.ones_like(wg)))
    assert torch.equal(dplain.cpu()[:n], dout[order // K]) and (dplain[n:] == 0).all()


def test_gradients_are_differences():
    """Both operators are linear in each input: with whole numbers all sums are exact, and so are the differences."""
    T, D, E, K = 19, 48, 8, 3
    idx, _ = routing(T, E, K, 3, bad=2)
    g = torch.Generator().manual_seed(5)

    def whole(*shape):
        return torch.randint(-8, 9, shape, generator=g).float().to(DEV)

    x, v, c = whole(T, D), whole(T, D), whole(T * K, D)
    f = lambda t: (bw.permute_tokens(t, idx.to(DEV), E)[0].double() * c.double()).sum().item()          # noqa: E731
    xg = x.clone().requires_grad_()
    rows, plan = bw.permute_tokens(xg, idx.to(DEV), E)
    dx, = torch.autograd.grad(rows, xg, c)
    assert (dx.double() * v.double()).sum().item() == (f(x + v) - f(x - v)) / 2

    r, w, vr, vw, c = whole(T * K, D), whole(T, K), whole(T * K, D), whole(T, K), whole(T, D)
    f = lambda a, b: (bw.unpermute_tokens(a, plan, b).double() * c.double()).sum().item()               # noqa: E731
    rg, wg = r.clone().requires_grad_(), w.clone().requires_grad_()
    dr, dw = torch.autograd.grad(bw.unpermute_tokens(rg, plan, wg), (rg, wg), c)
    assert (dr.double() * vr.double()).sum().item() == (f(r + vr, w) - f(r - vr, w)) / 2
    assert (dw.double() * vw.double()).sum().item() == (f(r, w + vw) - f(r, w - vw)) / 2


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D", [8, 66, 1024])
def test_pointers_aligned_to_their_type_only(dtype, D):
    T, E, K = 23, 8, 2
    idx, w = routing(T, E, K, 11)
    base = torch.randn(T * K * D + 1, generator=torch.Generator().manual_seed(2)).to(dtype).to(DEV)
    x = base[1:1 + T * D].view(T, D)
    rows, plan = bw.permute_tokens(x, idx.to(DEV), E)
    assert torch.equal(rows, x[plan.row_slot.long() // K])
    r = base[1:].view(T * K, D)
    assert torch.equal(bw.unpermute_tokens(r, plan, w.to(DEV)), bw.unpermute_tokens(r.clone(), plan, w.to(DEV)))
    dout = base[1:1 + T * D].view(T, D)
    a = bw.unpermute_tokens_backward(dout, r, plan, w.to(DEV))
    b = bw.unpermute_tokens_backward(dout.clone(), r.clone(), plan, w.to(DEV))
    assert torch.equal(a[0], b[0])
    torch.testing.assert_close(a[1], b[1], rtol=0, atol=2 * (D / 32 + 22) * U32 * float((r.double().abs().amax() ** 2) * D))


def test_a_round_trip_inside_a_step():
    """permute -> the experts' own torch computation -> unpermute, forward and backward, against autograd over indexing."""
    T, D, E, K = 50, 64, 8, 2
    idx, w = routing(T, E, K, 1)
    g = torch.Generator().manual_seed(4)
    x0, A0 = torch.randn(T, D, generator=g).to(DEV), (torch.randn(E, D, D, generator=g) / 8).to(DEV)

    def step(own):
        x, A, wt = (t.clone().requires_grad_() for t in (x0, A0, w.to(DEV)))
        if own:
            rows, plan = bw.permute_tokens(x, idx.to(DEV), E)
            bounds = plan.offsets.tolist()
            y = torch.cat([torch.tanh(rows[bounds[e]:bounds[e + 1]].double() @ A[e].double()) for e in range(E)]).float()
            out = bw.unpermute_tokens(y, plan, wt)
        else:
            out = sum((torch.tanh(torch.einsum("td,tdf->tf", x.double(), A.double()[idx[:, k].long().to(DEV)]))
                       * wt[:, k:k + 1].double()) for k in range(K)).float()
        return (out, *torch.autograd.grad((out.double() ** 2).sum(), (x, A, wt)))

    for a, b in zip(step(True), step(False)):
        torch.testing.assert_close(a, b, rtol=0, atol=float(64 * U32 * b.detach().abs().max()))


def test_gradient_of_an_expanded_sum():
    idx, w = routing(6, 4, 2, 0)
    r = torch.ones(12, 40, device=DEV, requires_grad=True)
    wt = w.to(DEV).requires_grad_()
    bw.unpermute_tokens(r, bw.permute_plan(idx.to(DEV), 4), wt).sum().backward()       # its gradient has strides of zero
    assert (wt.grad == 40).all()
    x = torch.ones(6, 40, device=DEV, requires_grad=True)
    bw.permute_tokens(x, idx.to(DEV), 4)[0].sum().backward()
    assert (x.grad == 2).all()


def test_empty_batches():
    for T, D in ((0, 16), (3, 0)):
        x = torch.empty(T, D, device=DEV, dtype=BF16, requires_grad=True)
        idx = torch.zeros(T, 2, dtype=torch.int32, device=DEV)
        idx[:, 1] = 1
        rows, plan = bw.permute_tokens(x, idx, 4)
        assert rows.shape == (2 * T, D) and plan.offsets.tolist() == [0, T, 2 * T, 2 * T, 2 * T]
        out = bw.unpermute_tokens(rows, plan, torch.ones(T, 2, device=DEV))
        out.sum().backward()
        assert out.shape == (T, D) and x.grad.shape == (T, D)


def test_another_stream_and_a_captured_graph():
    T, D, E, K = 300, 512, 16, 4
    idx, w = routing(T, E, K, 8)
    idx, w = idx.to(DEV), w.to(DEV)
    x = torch.randn(T, D, device=DEV).to(BF16)
    dout = torch.randn(T, D, device=DEV).to(BF16)

    def step():
        rows, plan = bw.permute_tokens(x, idx, E)
        out = bw.unpermute_tokens(rows, plan, w)
        return (rows, out, *bw.unpermute_tokens_backward(dout, rows, plan, w))

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
    for seed in range(3):
        new, w2 = routing(T, E, K, 20 + seed)
        idx.copy_(new), w.copy_(w2), x.normal_(), dout.normal_()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(captured, step()))


def test_a_captured_training_step():
    """Forward and backward through autograd inside a graph, replayed on new values."""
    T, D, E, K = 200, 128, 16, 2
    idx, w = routing(T, E, K, 9)
    idx = idx.to(DEV)
    x, wt = torch.randn(T, D, device=DEV).to(BF16).requires_grad_(), w.to(DEV).requires_grad_()
    grad = torch.randn(T, D, device=DEV).to(BF16)

    def step():
        rows, plan = bw.permute_tokens(x, idx, E)
        out = bw.unpermute_tokens(rows * 2, plan, wt)
        return (out.detach(), *torch.autograd.grad(out, (x, wt), grad))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in range(3):
        new, w2 = routing(T, E, K, 40 + seed)
        with torch.no_grad():
            idx.copy_(new), wt.copy_(w2), x.normal_(), grad.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, step()))


def test_no_second_derivative():
    idx, w = routing(6, 4, 2, 0)
    x, wt = torch.randn(6, 40, device=DEV, requires_grad=True), w.to(DEV).requires_grad_()
    rows, plan = bw.permute_tokens(x, idx.to(DEV), 4)
    dx, = torch.autograd.grad(rows.square().sum(), x, create_graph=True)
    assert torch.equal(dx.detach(), 4 * x.detach())
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dx.sum(), x)
    out = bw.unpermute_tokens(rows.detach(), plan, wt)
    dw, = torch.autograd.grad(out.square().sum(), wt, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dw.sum(), wt)


def test_a_value_changed_before_the_backward_pass_is_noticed():
    idx, w = routing(6, 4, 2, 0)
    r, wt = torch.randn(12, 40, device=DEV, requires_grad=True), w.to(DEV).requires_grad_()
    plan = bw.permute_plan(idx.to(DEV), 4)
    out = bw.unpermute_tokens(r, plan, wt)
    with torch.no_grad():
        wt.mul_(2)
    with pytest.raises(RuntimeError):
        out.sum().backward()
    rows, plan = bw.permute_tokens(r, torch.zeros(12, 1, dtype=torch.int32, device=DEV), 2)
    plan.offsets.zero_()                          # not needed by the backward pass: each tensor of a plan stands for itself
    rows.sum().backward()
    rows, plan = bw.permute_tokens(r, torch.zeros(12, 1, dtype=torch.int32, device=DEV), 2)
    plan.pos.zero_()
    with pytest.raises(RuntimeError):
        rows.sum().backward()


def test_rows_beyond_two_to_the_thirty_one_values():
    T, D, E, K = 34000, 8192, 8, 8
    idx, w = routing(T, E, K, 6)
    x = torch.randn(T, D, device=DEV, dtype=BF16)
    rows, plan = bw.permute_tokens(x, idx.to(DEV), E)
    assert rows.numel() > 2 ** 31
    for m in (0, 1, 131071, 262143, 262144, T * K // 2, T * K - 1):
        assert torch.equal(rows[m], x[int(plan.row_slot[m]) // K])
    out = bw.unpermute_tokens(rows, plan)
    assert torch.equal(out, (x.float() * K).to(BF16))        # eight equal terms: exact
    drows, dw = bw.unpermute_tokens_backward(x, rows, plan, w.to(DEV))
    for t in (0, 17000, T - 1):
        for k in (0, 7):
            want = (w[t, k].to(DEV) * x[t].float()).to(BF16)
            assert torch.equal(drows[int(plan.pos[t, k])], want)
        sq = (x[t].double() ** 2).sum()
        assert ((dw[t].double() - sq).abs() <= (D / 32 + 22) * U32 * sq).all()


def test_places_outside_the_rows_are_no_rows():
    """A plan made elsewhere: places past the rows or negative add nothing and are never written through."""
    T, D, K = 4, 32, 2
    pos = torch.tensor([[0, 99], [-5, 3], [2 ** 31 - 1, 1], [2, -2 ** 31]], dtype=torch.int32, device=DEV)
    plan = bw.PermutePlan(torch.tensor([0, 8], dtype=torch.int32, device=DEV), pos)
    rows = torch.randn(8, D, device=DEV)
    out = bw.unpermute_tokens(rows, plan)
    assert torch.equal(out, rows[[0, 3, 1, 2]])
    back, _ = bw.permute_tokens(out, plan=plan)
    assert torch.equal(back[:4], rows[:4])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_forward_mode_derivatives(dtype):
    """Dual tensors, which need not require a gradient.  Whole numbers: every sum is exact, and so is the derivative."""
    from torch.autograd import forward_ad as fw
    T, D, E, K = 19, 40, 8, 3
    idx, _ = routing(T, E, K, 3, bad=2)
    idx = idx.to(DEV)
    g = torch.Generator().manual_seed(5)
    whole = lambda *shape: torch.randint(-2, 3, shape, generator=g).float().to(DEV)                     # noqa: E731
    x, dx, r, dr = (whole(*s).to(dtype) for s in ((T, D), (T, D), (T * K, D), (T * K, D)))
    w, dw = whole(T, K), whole(T, K)
    want, plan = bw.permute_tokens(dx, idx, E)
    for grad in (False, True):
        with fw.dual_level():
            dual = fw.make_dual(x.clone().requires_grad_(grad), dx)
            for rows in (bw.permute_tokens(dual, idx, E)[0], bw.permute_tokens(dual, plan=plan)[0]):
                assert torch.equal(fw.unpack_dual(rows).tangent, want)
                assert torch.equal(rows.detach(), bw.permute_tokens(x, plan=plan)[0])
            rd, wd = fw.make_dual(r.clone().requires_grad_(grad), dr), fw.make_dual(w.clone().requires_grad_(grad), dw)
            tangent = lambda *a: fw.unpack_dual(bw.unpermute_tokens(*a)).tangent                        # noqa: E731
            assert torch.equal(tangent(rd, plan), bw.unpermute_tokens(dr, plan))
            assert torch.equal(tangent(rd, plan, w), bw.unpermute_tokens(dr, plan, w))
            assert torch.equal(tangent(r, plan, wd), bw.unpermute_tokens(r, plan, dw))
            assert torch.equal(tangent(rd, plan, wd), bw.unpermute_tokens(dr, plan, w) + bw.unpermute_tokens(r, plan, dw))
            # a tensor that is no dual inside the level
            assert fw.unpack_dual(bw.unpermute_tokens(r, plan, w)).tangent is None
    assert torch.equal(bw.unpermute_tokens(r, plan, w), bw.unpermute_tokens(r.clone(), plan, w.clone()))


def test_no_derivative_of_a_gradient():
    """Forward over reverse: the gradients are not differentiable themselves, and say so."""
    from torch.autograd import forward_ad as fw
    idx, w = routing(6, 4, 2, 0)
    x, v = torch.randn(6, 40, device=DEV), torch.randn(6, 40, device=DEV)
    with fw.dual_level():
        leaf = x.clone().requires_grad_()
        rows, plan = bw.permute_tokens(fw.make_dual(leaf, v), idx.to(DEV), 4)
        with pytest.raises(NotImplementedError):
            torch.autograd.grad(rows.square().sum(), leaf)
        r, wt = torch.randn(12, 40, device=DEV, requires_grad=True), fw.make_dual(w.to(DEV), torch.ones(6, 2, device=DEV))
        out = bw.unpermute_tokens(r, plan, wt)
        with pytest.raises(NotImplementedError):
            torch.autograd.grad(out.sum(), r)


def test_the_largest_number_of_rows():
    """As many slots as are accepted: the plan's blocks have 2^23 slots each, which takes the sum in a rounded-up quotient past
    32 bits."""
    T, E = 2 ** 31 - 4096, 3
    idx = torch.zeros(T, 1, dtype=torch.int32, device=DEV)
    idx[-5000:] = 1
    idx[5], idx[2 ** 30], idx[T - 3] = 2, -1, 2
    x = torch.zeros(T, 1, dtype=BF16, device=DEV)
    for i, t in enumerate((0, 5, 6, 2 ** 30 - 1, 2 ** 30, 2 ** 30 + 1, T - 5001, T - 5000, T - 3, T - 1)):
        x[t] = i + 1
    rows, plan = bw.permute_tokens(x, idx, E)
    zeros, ones = T - 5000 - 2, 4999
    assert plan.offsets.tolist() == [0, zeros, zeros + ones, T - 1]
    places = {0: 0, 5: T - 3, 6: 5, 2 ** 30 - 1: 2 ** 30 - 2, 2 ** 30: -1, 2 ** 30 + 1: 2 ** 30 - 1, T - 5001: zeros - 1,
              T - 5000: zeros, T - 3: T - 2, T - 1: zeros + ones - 1}
    for t, p in places.items():
        assert int(plan.pos[t, 0]) == p, t
        if p >= 0:
            assert int(plan.row_slot[p]) == t and float(rows[p]) == float(x[t]), t
    assert int(plan.row_slot[T - 1]) == -1 and float(rows[T - 1]) == 0 and int(torch.count_nonzero(rows)) == 9
    assert torch.equal(bw.unpermute_tokens(rows, plan)[:7], x[:7])
    del idx, x, rows, plan
    torch.cuda.empty_cache()


def in_used_memory(shape, dtype, call):
    """The call's result where the allocator hands it memory that holds NaN (in 8-bit integers: -1)."""
    torch.cuda.synchronize()
    block = torch.full(shape, float("nan"), dtype=dtype, device=DEV) if dtype.is_floating_point else torch.full(shape, -1, dtype=dtype, device=DEV)
    del block
    return call()


@pytest.mark.parametrize("how", ["dropped", "elsewhere", "in place", "inference"])
@pytest.mark.parametrize("T,D,E,K,dtype", [(4, 32, 2, 1, F32), (90, 1024, 16, 2, BF16), (37, 50, 8, 3, F16), (300, 2048, 32, 8, BF16), (41, 66, 64, 11, F32)])
def test_rows_that_no_slot_of_a_plan_from_elsewhere_owns(T, D, E, K, dtype, how):
    """Slots dropped from a plan leave rows in the middle of a segment without an owner: zeros, in every operator that writes
    rows."""
    idx, w = routing(T, E, K, T)
    g = torch.Generator().manual_seed(K)
    with torch.inference_mode(how == "inference"):
        made = bw.permute_plan(idx.to(DEV), E)
        gone = (torch.rand(T, K, generator=g) < 0.4).to(DEV)
        gone[0, 0], gone[1, 0] = True, False
        if how in ("in place", "inference"):
            made.pos[gone] = -1
            plan = made
        else:
            pos = torch.where(gone, -1, made.pos)
            if how == "dropped":
                plan = made._replace(pos=pos)
            else:                                           # other segments, rows in another order, places past the rows
                other = torch.randperm(T * K, generator=g).to(DEV, torch.int32)
                pos = torch.where(gone, T * K + 5, other[made.pos.long()])
                plan = bw.PermutePlan(torch.tensor([0, 3 * T * K], dtype=torch.int32, device=DEV), pos)
        x, dout = (torch.randn(T, D, generator=g).to(dtype).to(DEV) for _ in range(2))
        rows, _ = in_used_memory((T * K, D), dtype, lambda: bw.permute_tokens(x, plan=plan))
        pos = plan.pos
        owned = torch.zeros(T * K, dtype=torch.bool, device=DEV)
        owned[pos[~gone].long()] = True
        token = torch.arange(T, device=DEV)[:, None].expand(T, K)[~gone]
        want = torch.zeros_like(rows)
        want[pos[~gone].long()] = x[token]
        assert torch.equal(rows, want)
        wt = w.to(DEV)
        drows, dw = in_used_memory((T * K, D), dtype, lambda: bw.unpermute_tokens_backward(dout, rows, plan, wt))
        want[pos[~gone].long()] = (wt[~gone][:, None] * dout[token].float()).to(dtype)
        assert torch.equal(drows, want) and (dw[gone] == 0).all() and not dw.isnan().any()
        if D % 16 == 0:
            alone, scale = bw.quantize_tokens_int8(x)
            codes, scales = in_used_memory((T * K, D), torch.int8, lambda: bw.quantize_tokens_int8(x, plan))
            want, ws = torch.zeros_like(codes), torch.zeros_like(scales)
            want[pos[~gone].long()], ws[pos[~gone].long()] = alone[token], scale[token]
            assert torch.equal(codes, want) and torch.equal(scales, ws)
    if how != "inference":
        rg = rows.detach().clone().requires_grad_()
        d, = in_used_memory((T * K, D), dtype, lambda: torch.autograd.grad(bw.unpermute_tokens(rg, plan), rg, dout))
        assert torch.equal(d[~owned], torch.zeros_like(d[~owned])) and torch.equal(d[pos[~gone].long()], dout[token])
        d, = in_used_memory((T * K, D), dtype, lambda: torch.autograd.grad(bw.unpermute_tokens(rg, plan, wt), rg, dout))
        assert torch.equal(d, drows)


def test_the_librarys_own_plans_need_no_owners():
    """One launch, as long as nothing was written to them."""
    idx, _ = routing(40, 8, 2, 0)
    x = torch.randn(40, 64, device=DEV)
    _, plan = bw.permute_tokens(x, idx.to(DEV), 8)
    lib = bw.lib()

    def launches(p):
        n = lib.bwmoe_launch_count()
        bw.permute_tokens(x, plan=p)
        return lib.bwmoe_launch_count() - n
    assert launches(plan) == 1 and launches(bw.PermutePlan(*plan)) == 2
    plan.pos[3, 1] = -1
    assert launches(plan) == 2


def test_copies_of_a_plan_are_plans_from_elsewhere():
    """Slots dropped, then copied: the copies' tensors are as new, but not as the library wrote them."""
    import copy
    import pickle
    from torch.utils._pytree import tree_map
    T, D, K = 30, 64, 2
    idx, _ = routing(T, 8, K, 0)
    x = torch.randn(T, D, device=DEV)
    plan = bw.permute_plan(idx.to(DEV), 8)
    gone = int(plan.pos[3, 1])
    plan.pos[3, 1] = -1
    for made in (copy.copy(plan), copy.deepcopy(plan), pickle.loads(pickle.dumps(plan)), tree_map(torch.clone, plan), type(plan)(*[t.clone() for t in plan]),
                 plan._replace(pos=plan.pos.clone()), type(plan)._make(t.clone() for t in plan)):
        assert isinstance(made, bw.PermutePlan) and torch.equal(made.pos, plan.pos)
        rows, back = in_used_memory((T * K, D), F32, lambda: bw.permute_tokens(x, plan=made))
        assert back is made and (rows[gone] == 0).all() and torch.equal(rows[made.pos[0, 0]], x[0])


def test_a_captured_step_with_a_plan_from_elsewhere():
    """Every operator that writes rows, replayed on other places and values: rows without a slot are zeros each time."""
    T, D, K = 60, 128, 3
    g = torch.Generator().manual_seed(1)

    def places():
        pos = torch.randperm(T * K, generator=g).to(torch.int32).view(T, K)
        return torch.where(torch.rand(T, K, generator=g) < 0.3, -1, pos)
    plan = bw.PermutePlan(torch.tensor([0, T * K], dtype=torch.int32, device=DEV), places().to(DEV))
    x, dout = (torch.randn(T, D, generator=g).to(BF16).to(DEV) for _ in range(2))
    w = torch.rand(T, K, generator=g).to(DEV)

    def step():
        rows, _ = bw.permute_tokens(x, plan=plan)
        return (rows, *bw.unpermute_tokens_backward(dout, rows, plan, w), *bw.quantize_tokens_int8(x, plan))
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for _ in range(3):
        plan.pos.copy_(places()), x.normal_(), dout.normal_(), w.uniform_()
        for t in captured:
            t.fill_(3)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, step()))
        free = torch.ones(T * K, dtype=torch.bool, device=DEV)
        free[plan.pos[plan.pos >= 0].long()] = False
        assert free.any() and all((t[free] == 0).all() for t in (captured[0], captured[1], captured[3], captured[4]))
