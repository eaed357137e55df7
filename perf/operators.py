"""The operators around and inside experts of 8-bit integers, as cases that can be timed and compared.

A case is one pass through one operator:

* ``permute``:   ``permute_tokens`` - a batch's tokens sorted by expert; in training also the gradient of the tokens;
* ``unpermute``: ``unpermute_tokens`` - the experts' rows back in token order, summed with the routing weights; in
  training also the gradients of the rows and of the weights;
* ``linear``:    ``int8_matmul`` - activations quantised token by token, times a matrix of 8-bit integers with a scale
  for each channel;
* ``grouped``:   ``int8_grouped_gemm`` - the product of rows in expert order with their experts' matrices;
* ``experts``:   ``int8_moe_forward_routed`` - all of it together: a batch with its routing through experts of 8-bit
  integers, SwiGLU between the products.

``own`` false: the operators' plain form, elementary torch operations.  ``own`` true: this package's calls.  The shapes
are the benchmark configurations of this repository (see cases.py beside this file) and odd ones of the same range.
"""

import math

import numpy as np
import torch

own = False

# hidden size, expert intermediate size, experts, experts per token
MIXTRAL_8X7B = dict(D=4096, H=14336, E=8, K=2)
DEEPSEEK_V2_LITE = dict(D=2048, H=1408, E=64, K=6)
QWEN3_30B = dict(D=2048, H=768, E=128, K=8)
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _case(name, op, T, D, H=0, E=1, K=1, dtype="bf16", train=False, zipf=False):
    return dict(name=name, op=op, T=T, D=D, H=H, E=E, K=K, dtype=dtype, train=train, zipf=zipf)


def listed():
    return [
        # a server's decode batch: launches and latency count
        _case("permute-64", "permute", 64, 2048, E=64, K=6),
        # a training step of full size, forward and backward
        _case("permute-train-16384", "permute", 16384, 4096, E=8, K=2, train=True),
        # a ragged micro-batch in 32 bits with a hidden size of no round length, skewed popularity
        _case("permute-train-1003-f32", "permute", 1003, 2050, E=128, K=8, dtype="f32", train=True, zipf=True),
        # a decode batch's sum
        _case("unpermute-37", "unpermute", 37, 2048, E=64, K=6, dtype="f16"),
        # prefill
        _case("unpermute-4096", "unpermute", 4096, 2048, E=64, K=6),
        # a training step over many small experts, forward and backward with the routing weights' gradient
        _case("unpermute-train-8192", "unpermute", 8192, 2048, E=128, K=8, train=True),
        # one token through a large matrix: the weights are all that counts
        _case("linear-1", "linear", 1, 4096, 14336),
        # an odd batch in 32 bits, a ragged number of channels
        _case("linear-517-f32", "linear", 517, 1408, 2064, dtype="f32"),
        # the rows of a prefill batch through their experts' matrices
        _case("grouped-8192", "grouped", 8192, 2048, 1408, E=64, K=6),
        # a decode batch through a layer of small experts
        _case("experts-64", "experts", 64, **DEEPSEEK_V2_LITE),
        # a chunk of a prompt, skewed popularity, 16-bit floats
        _case("experts-1003-f16", "experts", 1003, **QWEN3_30B, dtype="f16", zipf=True),
        # full prefill over large experts
        _case("experts-16384", "experts", 16384, **MIXTRAL_8X7B),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _multiple(rng, unit, lo, hi):
    return max(1, round(_log_uniform(rng, lo, max(lo, hi)) / unit)) * unit


def draw(rng):
    """One more case of the same ranges: any operator, odd batch sizes, every type."""
    op = rng.choice(["permute", "permute", "unpermute", "unpermute", "linear", "grouped", "experts", "experts"])
    dtype = rng.choice(["bf16", "bf16", "f16"] if op == "experts" else ["bf16", "f16", "f32"])
    zipf = op != "linear" and rng.random() < 0.3
    if op in ("permute", "unpermute"):
        E = rng.choice([8, 16, 60, 64, 128, 200, 256])
        K = rng.randint(1, 8)
        D = _multiple(rng, rng.choice([1, 8, 64]), 512, 8192)
        T = _log_uniform(rng, 1, 16384 * 2 * 4096 / (K * D))
        case = _case("", op, T, D, E=E, K=K, dtype=dtype, train=rng.random() < 0.6, zipf=zipf)
    elif op == "linear":
        D, H = _multiple(rng, 16, 512, 8192), _multiple(rng, 16, 512, 16384)
        case = _case("", op, _log_uniform(rng, 1, 8192), D, H, dtype=dtype)
    else:
        if rng.random() < 0.4:
            shape = dict(rng.choice([MIXTRAL_8X7B, DEEPSEEK_V2_LITE, QWEN3_30B]))
        else:
            E = rng.choice([8, 16, 64, 128, 160])
            D = _multiple(rng, 64, 1024, 4096)
            H = _multiple(rng, 16, 320, min(14336, 1.2e9 / (3.0 * D * E)))
            shape = dict(D=D, H=H, E=E, K=rng.randint(1, 8))
        t_max = min(16384, 6e12 / (6.0 * shape["K"] * shape["D"] * shape["H"]))
        case = _case("", op, _log_uniform(rng, 1, t_max), dtype=dtype, zipf=zipf, **shape)
    del case["name"]
    return case


# ---------------------------------------------------------------- inputs
def _generator(seed, tensor):
    # one stream per tensor, made from the seed alone
    return torch.Generator(device="cuda").manual_seed(int(seed) * 1009 + tensor)


def _normal(shape, seed, stream, std=1.0, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=_generator(seed, stream))


def _quantised_weights(case, seed, stream, rows, cols):
    """Weights ~N(0, 0.02^2) of every expert in 8-bit integers, a scale for each output channel: what a loader keeps."""
    w = _normal((case["E"], rows, cols), seed, stream, 0.02, torch.bfloat16)
    scales = w.abs().amax(dim=1).float() / 127.0
    return w.float().div_(scales.unsqueeze(1)).round_().clamp_(-127, 127).to(torch.int8), scales


def _routing(case, seed):
    """Each token's K experts and their weights: the largest of random logits, which where popularity is skewed carry
    the experts' log rank (Zipf 1.1)."""
    T, E, K = case["T"], case["E"], case["K"]
    logits = _normal((T, E), seed, 1)
    if case["zipf"]:
        logits -= 1.1 * torch.log(torch.randperm(E, generator=_generator(seed, 2), device="cuda").float() + 1.0)
    top, indices = torch.topk(logits, K, dim=1)
    return torch.softmax(top, dim=1), indices.to(torch.int32)


def _plan(indices, E):
    """The stable sort of all slots (token, k) by expert: where each expert's rows begin, the row of every slot, the
    slot and the expert of every row."""
    flat = indices.reshape(-1).long()
    experts, slots = torch.sort(flat, stable=True)
    pos = torch.empty_like(slots)
    pos[slots] = torch.arange(slots.numel(), device=slots.device)
    offsets = torch.searchsorted(experts, torch.arange(E + 1, device=slots.device))
    i32 = torch.int32
    return offsets.to(i32), pos.view(indices.shape).to(i32), slots.to(i32), experts.to(i32)


def prepare(case, seed):
    case = dict(case)
    T, D, H, E, K, dtype = (case[k] for k in ("T", "D", "H", "E", "K", "dtype"))
    state, M = dict(case=case), T * K
    if case["op"] == "linear":
        state["x"] = _normal((T, D), seed, 8).to(TYPES[dtype])
        w, s = _quantised_weights(case, seed, 10, D, H)
        state["w"], state["scales"] = w[0], s[0]
        return state
    weights, indices = _routing(case, seed)
    if case["op"] == "permute":
        state["x"] = _normal((T, D), seed, 8).to(TYPES[dtype]).requires_grad_(case["train"])
        state["indices"] = indices
        if case["train"]:
            state["grad"] = _normal((M, D), seed, 9).to(TYPES[dtype])
    elif case["op"] == "unpermute":
        state["plan"] = _plan(indices, E)
        state["rows"] = _normal((M, D), seed, 8).to(TYPES[dtype]).requires_grad_(case["train"])
        state["weights"] = weights.requires_grad_(case["train"])
        if case["train"]:
            state["grad"] = _normal((T, D), seed, 9).to(TYPES[dtype])
    elif case["op"] == "grouped":
        # rows as an earlier step of the program quantised them
        state["plan"] = _plan(indices, E)
        state["codes"] = _normal((M, D), seed, 8, 32.0).round_().clamp_(-127, 127).to(torch.int8)
        state["row_scales"] = torch.rand(M, generator=_generator(seed, 9), device="cuda") * 0.02 + 0.02
        state["w"], state["scales"] = _quantised_weights(case, seed, 10, D, H)
    else:
        state["x"] = _normal((T, D), seed, 8).to(TYPES[dtype])
        state["weights"], state["indices"] = weights, indices
        state["experts"] = [_quantised_weights(case, seed, 10 + n, *shape) for n, shape in enumerate(((D, H), (D, H), (H, D)))]
    return state


# ---------------------------------------------------------------- the operators
def _run_own(state):
    import blackwell_moe_b200 as bw

    case = state["case"]
    if case["op"] == "permute":
        rows, plan = bw.permute_tokens(state["x"], state["indices"], case["E"])
        out = dict(rows=rows, pos=plan.pos, offsets=plan.offsets)
        if case["train"]:
            out["dx"], = torch.autograd.grad(rows, state["x"], state["grad"])
        return out
    if case["op"] == "unpermute":
        out = dict(out=bw.unpermute_tokens(state["rows"], bw.PermutePlan(*state["plan"]), state["weights"]))
        if case["train"]:
            out["drows"], out["dweights"] = torch.autograd.grad(out["out"], (state["rows"], state["weights"]), state["grad"])
        return out
    if case["op"] == "linear":
        return bw.int8_matmul(state["x"], state["w"], state["scales"])
    if case["op"] == "grouped":
        return bw.int8_grouped_gemm(state["codes"], state["row_scales"], state["plan"][0], state["w"], state["scales"],
                                    out_dtype=TYPES[case["dtype"]])
    (g, sg), (u, su), (d, sd) = state["experts"]
    return bw.int8_moe_forward_routed(state["x"], state["weights"], state["indices"], g, u, d, sg, su, sd)


def _quantise(x):
    """Row by row: scale = max|x| / 127 in 32 bits, codes = x / scale rounded to the nearest, ties to even.  The
    quotients are formed in 64 bits: in 32, one next to a border between two codes may fall on it."""
    amax = x.float().abs().amax(dim=1)
    scale = amax / torch.full_like(amax, 127.0)
    safe = torch.where(scale > 0, scale, torch.ones_like(scale))
    return torch.round(x.double() / safe.double().unsqueeze(1)).float(), scale


def _product(codes, row_scales, offsets, w, scales):
    """Each expert's rows times its matrix, in 32 bits: the codes' product, times the row's and the channel's scale."""
    bounds = offsets.tolist()
    out = torch.zeros((codes.shape[0], w.shape[2]), dtype=torch.float32, device="cuda")
    for e in range(w.shape[0]):
        if bounds[e + 1] > bounds[e]:
            torch.matmul(codes[bounds[e]:bounds[e + 1]].float(), w[e].float(), out=out[bounds[e]:bounds[e + 1]])
            out[bounds[e]:bounds[e + 1]] *= scales[e]
    return out.mul_(row_scales.unsqueeze(1))


def _run_plain(state):
    case = state["case"]
    E, K, dtype = case["E"], case["K"], TYPES[case["dtype"]]
    with torch.no_grad():
        if case["op"] == "permute":
            offsets, pos, slots, _ = _plan(state["indices"], E)
            out = dict(rows=state["x"][slots.long() // K], pos=pos, offsets=offsets)
            if case["train"]:
                out["dx"] = state["grad"][pos.long()].float().sum(dim=1).to(dtype)
            return out
        if case["op"] == "unpermute":
            _, pos, slots, _ = state["plan"]
            rows = state["rows"][pos.long()].float()
            out = dict(out=(rows * state["weights"].unsqueeze(2)).sum(dim=1).to(dtype))
            if case["train"]:
                grad = state["grad"].float()
                out["drows"] = (grad[slots.long() // K] * state["weights"].reshape(-1)[slots.long()].unsqueeze(1)).to(dtype)
                out["dweights"] = (rows * grad.unsqueeze(1)).sum(dim=2)
            return out
        if case["op"] == "linear":
            codes, row_scales = _quantise(state["x"])
            return (torch.matmul(codes, state["w"].float()) * state["scales"] * row_scales.unsqueeze(1)).to(dtype)
        if case["op"] == "grouped":
            return _product(state["codes"], state["row_scales"], state["plan"][0], state["w"], state["scales"]).to(dtype)
        # the experts: every step's result in the activations' type, as one step hands it to the next
        (g, sg), (u, su), (d, sd) = state["experts"]
        offsets, pos, slots, _ = _plan(state["indices"], E)
        codes, row_scales = _quantise(state["x"])
        codes, row_scales = codes[slots.long() // K], row_scales[slots.long() // K]
        gate = _product(codes, row_scales, offsets, g, sg)
        up = _product(codes, row_scales, offsets, u, su)
        h = (gate / (1.0 + torch.exp(-gate)) * up).to(dtype)
        y = _product(*_quantise(h), offsets, d, sd).to(dtype)
        return (y[pos.long()].float() * state["weights"].unsqueeze(2)).sum(dim=1).to(dtype)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------- what a pass cannot do without
def _experts_used(case):
    """Distinct experts that a batch reaches, counted on a draw of the logits' distribution."""
    rng = np.random.default_rng(0)
    logits = rng.standard_normal((min(case["T"], 2048), case["E"]))
    if case["zipf"]:
        logits -= 1.1 * np.log(rng.permutation(case["E"]) + 1.0)
    return len(np.unique(np.argsort(-logits, axis=1)[:, : case["K"]]))


def work(case):
    T, D, H, E, K = (case[k] for k in ("T", "D", "H", "E", "K"))
    size, M = (4.0 if case["dtype"] == "f32" else 2.0), T * K
    if case["op"] == "permute":       # tokens in, rows out, ids in, places out; backward: the rows' gradient in, the tokens' out
        moved = (T + M) * D * size
        return {"bytes": moved * (2.0 if case["train"] else 1.0) + 8.0 * M + 4.0 * E, "flops": float(M) * D if case["train"] else 0.0}
    if case["op"] == "unpermute":     # rows in, sums out, places and weights in; backward: the sums' gradient in, the rows' out
        moved = (T + M) * D * size
        return {"bytes": moved * (2.0 if case["train"] else 1.0) + (12.0 if case["train"] else 8.0) * M,
                "flops": M * D * (5.0 if case["train"] else 2.0)}
    if case["op"] == "linear":        # activations, codes and scales of the matrix in, result out
        return {"bytes": T * (D + H) * size + D * H + 4.0 * H, "flops": 2.0 * T * D * H}
    used = _experts_used(case)
    if case["op"] == "grouped":
        return {"bytes": M * (D + H * size + 4.0) + used * (D * H + 4.0 * H), "flops": 2.0 * M * D * H}
    return {"bytes": 2.0 * T * D * size + 8.0 * M + used * (3.0 * D * H + 8.0 * H + 4.0 * D), "flops": 6.0 * M * D * H}


# ---------------------------------------------------------------- the definition, in 64 bits
def _exact_codes(x):
    """Row by row: the scale is the 32-bit number nearest to max|x| / 127, the codes are the whole numbers nearest to
    x / scale."""
    x = x.double()
    scale = (x.abs().max(dim=1).values / 127.0).float().double()
    quotient = torch.where(scale[:, None] > 0, x / scale[:, None], torch.zeros_like(x))
    low = torch.floor(quotient)
    rest = quotient - low
    up = (rest > 0.5) | ((rest == 0.5) & (torch.remainder(low, 2) == 1))
    return torch.where(up, low + 1, low), scale


def _exact_experts(codes, row_scales, expert_of_row, w, scales):
    out = torch.zeros((codes.shape[0], w.shape[2]), dtype=torch.float64, device="cuda")
    for e in torch.unique(expert_of_row).tolist():
        mine = torch.nonzero(expert_of_row == e).flatten()
        out[mine] = (codes[mine] * row_scales[mine, None]) @ (w[e].double() * scales[e].double())
    return out


def exact(case, seed):
    state = prepare(case, seed)
    T, E, K, dtype = case["T"], case["E"], case["K"], TYPES[case["dtype"]]
    with torch.no_grad():
        if case["op"] == "linear":
            codes, scale = _exact_codes(state["x"])
            return (codes * scale[:, None]) @ (state["w"].double() * state["scales"].double())
        if case["op"] == "grouped":
            return _exact_experts(state["codes"].double(), state["row_scales"].double(), state["plan"][3], state["w"], state["scales"])
        if case["op"] == "unpermute":
            weights, rows, pos = state["weights"].double(), state["rows"].double(), state["plan"][1].long()
            out = torch.zeros((T, case["D"]), dtype=torch.float64, device="cuda")
            for k in range(K):
                out += weights[:, k, None] * rows[pos[:, k]]
            out = dict(out=out)
            if case["train"]:
                grad = state["grad"].double()
                out["drows"] = torch.empty_like(rows)
                out["dweights"] = torch.empty_like(weights)
                for k in range(K):
                    out["drows"][pos[:, k]] = weights[:, k, None] * grad
                    out["dweights"][:, k] = (rows[pos[:, k]] * grad).sum(dim=1)
            return out
        # rows in expert order: by expert, then by slot
        slot = torch.arange(T * K, device="cuda")
        key = state["indices"].reshape(-1).long() * (T * K) + slot
        slot_of_row = torch.argsort(key)
        token = slot_of_row // K
        if case["op"] == "permute":
            out = dict(rows=state["x"].double()[token], pos=None, offsets=None)
            if case["train"]:
                out["dx"] = torch.zeros((T, case["D"]), dtype=torch.float64, device="cuda").index_add_(0, token, state["grad"].double())
            return out
        (g, sg), (u, su), (d, sd) = state["experts"]
        expert = state["indices"].reshape(-1)[slot_of_row]
        codes, scale = _exact_codes(state["x"])
        gate = _exact_experts(codes[token], scale[token], expert, g, sg)
        up = _exact_experts(codes[token], scale[token], expert, u, su)
        h = (gate * torch.sigmoid(gate) * up).to(dtype)
        del gate, up
        y = _exact_experts(*_exact_codes(h), expert, d, sd).to(dtype)
        weight = state["weights"].reshape(-1)[slot_of_row].double()
        return torch.zeros((T, case["D"]), dtype=torch.float64, device="cuda").index_add_(0, token, y.double() * weight[:, None])
