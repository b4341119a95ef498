"""Cases of the 8-bit integer grouped product and of the gradient clip: inputs, a plain torch form, the package's own calls.

Two operators:

``linear``  rows of bf16 activations -> int8 codes with one scale per row -> grouped product with int8 weights that carry
            one scale per output channel -> bf16.  The rows may be gathered from tokens by a router's sort (each token
            goes to ``top_k`` experts), and an activation may stand in front of the quantisation (the second layer of
            an expert reads the first layer's bf16 pre-activation).

                v[r, :]  = act(x[indices[r] // top_k, :])
                s[r]     = max_k |v[r, k]| / 127             q[r, k] = round_half_even(127 v[r, k] / max_k |v[r, k]|)
                out[r,n] = s[r] * w_scale[g, n] * sum_k q[r, k] w[g, n, k]          (row r belongs to group g)

``clip``    global 2-norm over a list of gradients of mixed sizes and types, and the clipped gradients.

                norm = sqrt(sum_i sum_j g_i[j]^2)            out_i = g_i * min(1, max_norm / (norm + 1e-6))

Where ``own`` is false ``run`` computes them with elementary torch operations, otherwise with fp8_gmm_b200.
"""
import math

import torch

own = False

MAX_NORM = 1.0
_MOST_WEIGHTS = 8 * 28672 * 4096          # bytes of int8 weights of the largest case
_MOST_FLOPS = 2 * 32768 * 28672 * 4096
_MOST_GRADS = 8 * 3 * 14336 * 4096        # gradient elements of the largest case


def _linear(tokens, top_k, experts, k, n, gather=True, act="none", device_sizes=False, zipf=False):
    return {"op": "linear", "tokens": tokens, "top_k": top_k, "experts": experts, "k": k, "n": n, "gather": gather, "act": act,
            "device_sizes": device_sizes, "zipf": zipf}


def _clip(layers, experts, hidden, ffn, grads="bf16", out="same"):
    return {"op": "clip", "layers": layers, "experts": experts, "hidden": hidden, "ffn": ffn, "grads": grads, "out": out}


def listed():
    return [
        # one token through one small expert: nothing but latency
        dict(_linear(1, 1, 4, 768, 1024, device_sizes=True), name="linear_tiny"),
        # one generated token, second layer of two of eight experts: SwiGLU of its pre-activation, 117 MB of weights
        dict(_linear(1, 2, 8, 14336, 4096, gather=False, act="swiglu", device_sizes=True), name="linear_decode_1_fc2"),
        # a batch of 64 sequences generating one token each, first layer, all eight experts hit: 940 MB of weights
        dict(_linear(64, 2, 8, 4096, 28672, device_sizes=True), name="linear_decode_64_fc1"),
        # a short prompt over many small experts with Zipf popularity: ragged and empty groups, odd sizes
        dict(_linear(777, 6, 64, 2080, 1424, zipf=True), name="linear_ragged_64"),
        # a medium prompt, second layer with the GELU of the default expert
        dict(_linear(1481, 1, 5, 4096, 1024, gather=False, act="gelu"), name="linear_gelu_5"),
        # a training-sized batch (evaluation pass), first layer: the largest product
        dict(_linear(16384, 2, 8, 4096, 28672), name="linear_large_fc1"),
        # the same batch, second layer: long contraction behind the SwiGLU
        dict(_linear(16384, 2, 8, 14336, 4096, gather=False, act="swiglu"), name="linear_large_fc2"),
        # the gradients of a two-layer toy: latency of a clip over ten small tensors
        dict(_clip(2, 4, 128, 256), name="clip_small"),
        # many tensors of odd sizes and both types, as a model with several MoE layers leaves them
        dict(_clip(12, 5, 677, 1481, "mixed", "same"), name="clip_ragged_60"),
        # the gradients of eight full-size experts, clipped into the optimizer's fp32 gradients
        dict(_clip(1, 8, 4096, 14336, "bf16", "fp32"), name="clip_experts_fp32"),
        # one rank's share of them, bf16 throughout
        dict(_clip(1, 2, 4096, 14336, "bf16", "same"), name="clip_experts_bf16"),
        # the norm alone, as a training loop logs it
        dict(_clip(1, 8, 4096, 14336, "bf16", "norm"), name="norm_experts"),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    if rng.random() < 0.6:
        while True:
            experts = _spread(rng, 1, 64)
            act = rng.choice(["none", "none", "swiglu", "gelu"])
            c = _linear(_spread(rng, 1, 16384), rng.randint(1, min(experts, 8)), experts, 16 * _spread(rng, 8, 896), 16 * _spread(rng, 8, 1792),
                        gather=act == "none" and rng.random() < 0.7, act=act, device_sizes=rng.random() < 0.5, zipf=rng.random() < 0.5)
            rows = c["tokens"] * c["top_k"]
            if experts * c["k"] * c["n"] <= _MOST_WEIGHTS and 2 * rows * c["k"] * c["n"] <= _MOST_FLOPS and rows <= 32768:
                return c
    while True:
        c = _clip(rng.randint(1, 12), _spread(rng, 1, 64), _spread(rng, 33, 4096), _spread(rng, 40, 14336),
                  rng.choice(["bf16", "fp32", "mixed"]), rng.choice(["same", "same", "fp32", "norm"]))
        if sum(math.prod(s) for s in _shapes(c)) <= _MOST_GRADS // 2:
            return c


# ------------------------------------------------------------------------------------------------ inputs
def _shapes(case):
    """Gradients of one MoE layer: gate|up weights, down weights, router, a norm's weight, the experts' biases."""
    e, h, f = case["experts"], case["hidden"], case["ffn"]
    return [(e, 2 * f, h), (e, h, f), (e, h), (h,), (e, 2 * f + 1)] * case["layers"]


def _grad_types(case):
    both = {"bf16": (torch.bfloat16,), "fp32": (torch.float32,), "mixed": (torch.bfloat16, torch.bfloat16, torch.float32)}[case["grads"]]
    return [both[i % len(both)] for i in range(5 * case["layers"])]


def _prepare_clip(case, gen, dev):
    grads, outs = [], []
    for i, (shape, dtype) in enumerate(zip(_shapes(case), _grad_types(case))):
        g = torch.empty(shape, dtype=dtype, device=dev)
        g.normal_(0.0, 0.02 / (1 + i % 7), generator=gen)
        grads.append(g)
        if case["out"] != "norm":
            outs.append(torch.empty(shape, dtype=torch.float32 if case["out"] == "fp32" else dtype, device=dev))
    return {"op": "clip", "out": case["out"], "grads": grads, "outs": outs}


def _route(case, gen, dev):
    """Router of ``tokens`` tokens: flat expert ids, the rows sorted by expert, and the group sizes."""
    e, t, k = case["experts"], case["tokens"], case["top_k"]
    logits = torch.randn(1, e, generator=gen, device=dev)
    if case["zipf"]:
        logits = -1.1 * torch.log(torch.arange(1, e + 1, device=dev, dtype=torch.float32))[None]
    noise = -torch.log(-torch.log(torch.rand(t, e, generator=gen, device=dev).clamp(1e-6, 1 - 1e-6)))
    ids = torch.topk(logits + noise, k, dim=1).indices.reshape(-1)
    return torch.argsort(ids, stable=True).to(torch.int32), torch.bincount(ids, minlength=e)


def _prepare_linear(case, gen, dev):
    e, k, n, rows = case["experts"], case["k"], case["n"], case["tokens"] * case["top_k"]
    indices, sizes = _route(case, gen, dev)
    width = 2 * k if case["act"] == "swiglu" else k
    x = torch.empty(case["tokens"] if case["gather"] else rows, width, dtype=torch.bfloat16, device=dev).normal_(0.0, 1.0, generator=gen)
    # a few large activations per thousand, as trained models have them: they set the row's scale
    x *= 1 + 19 * (torch.rand(x.shape[0], width, generator=gen, device=dev, dtype=torch.bfloat16) < 0.002)
    w = torch.randint(-127, 128, (e, n, k), generator=gen, device=dev, dtype=torch.int8)
    w_scales = (torch.rand(e, n, generator=gen, device=dev) * 0.2 + 0.9) / (127 * math.sqrt(k))
    host = sizes.cpu()
    return {"op": "linear", "x": x, "w": w, "w_scales": w_scales, "indices": indices if case["gather"] else None, "top_k": case["top_k"],
            "act": case["act"], "sizes": host.tolist(), "group_sizes": sizes if case["device_sizes"] else host}


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    return (_prepare_linear if case["op"] == "linear" else _prepare_clip)(case, gen, dev)


# ------------------------------------------------------------------------------------------------ the plain form
def _activate(x, act):
    if act == "swiglu":
        gate, up = x.chunk(2, dim=1)
        return gate / (1 + torch.exp(-gate)) * up
    if act == "gelu":
        return 0.5 * x * (1 + torch.tanh(0.79788456 * x * (1 + 0.044715 * x * x)))
    return x


def _plain_linear(s):
    x = s["x"] if s["indices"] is None else s["x"][s["indices"].long() // s["top_k"]]
    v = _activate(x.float(), s["act"])
    top = v.abs().amax(dim=1, keepdim=True)
    # the codes in 64 bits: values next to a rounding border
    q = torch.round(v.double() * 127 / torch.where(top > 0, top, 1).double()).float()
    parts = [(rows @ w.float().t()) * ws for rows, w, ws in zip(q.split(s["sizes"]), s["w"], s["w_scales"]) if rows.shape[0]]
    return (torch.cat(parts) * (top / 127)).to(torch.bfloat16)


def _plain_clip(s):
    squares = torch.stack([g.float().square().sum(dtype=torch.float64) for g in s["grads"]])
    norm = squares.sum().sqrt()
    coef = (MAX_NORM / (norm + 1e-6)).clamp(max=1.0).float()
    return [norm.float()] + [o.copy_(g.float() * coef) for g, o in zip(s["grads"], s["outs"])]


def run(state):
    if own:
        from fp8_gmm_b200 import backend

        if state["op"] == "clip":
            if state["out"] == "norm":
                return backend.multi_grad_norm(state["grads"])
            return [backend.multi_clip_grad_norm(state["grads"], MAX_NORM, outputs=state["outs"])] + state["outs"]
        return backend.int8_linear(state["x"], state["w"], state["group_sizes"], state["w_scales"], indices=state["indices"],
                                   top_k=state["top_k"], activation=None if state["act"] == "none" else state["act"])
    if state["op"] == "clip":
        return _plain_clip(state)[0] if state["out"] == "norm" else _plain_clip(state)
    return _plain_linear(state)


# ------------------------------------------------------------------------------------------------ work and exact values
def work(case):
    if case["op"] == "clip":
        numel = [math.prod(s) for s in _shapes(case)]
        size = [2 if t == torch.bfloat16 else 4 for t in _grad_types(case)]
        read = sum(a * b for a, b in zip(numel, size))
        write = {"same": read, "fp32": 4 * sum(numel), "norm": 0}[case["out"]] + 4
        return {"bytes": read + write, "flops": (2 if case["out"] == "norm" else 3) * sum(numel)}
    rows, k, n = case["tokens"] * case["top_k"], case["k"], case["n"]
    x = 2 * (case["tokens"] if case["gather"] else rows) * k * (2 if case["act"] == "swiglu" else 1)
    experts = min(case["experts"], rows)  # experts that a row can name
    return {"bytes": x + experts * (n * k + 4 * n) + 2 * rows * n + (4 * rows if case["gather"] else 0), "flops": 2 * rows * n * k}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "clip":
        norm = math.sqrt(sum(float((g.double() ** 2).sum()) for g in s["grads"]))
        if case["out"] == "norm":
            return torch.tensor(norm, dtype=torch.float64)
        factor = min(1.0, MAX_NORM / (norm + 1e-6))
        return [torch.tensor(norm, dtype=torch.float64)] + [g.double().mul_(factor) for g in s["grads"]]
    out = torch.empty(case["tokens"] * case["top_k"], case["n"], dtype=torch.float64, device=s["x"].device)
    row = 0
    for g, m in enumerate(s["sizes"]):
        if m == 0:
            continue
        weights = s["w"][g].double() * s["w_scales"][g].double()[:, None]
        for first in range(row, row + m, 4096):
            last = min(first + 4096, row + m)
            x = s["x"][first:last] if s["indices"] is None else s["x"][torch.div(s["indices"][first:last].long(), s["top_k"], rounding_mode="floor")]
            v = x.double()
            if case["act"] == "swiglu":
                v = v[:, : case["k"]] * torch.sigmoid(v[:, : case["k"]]) * v[:, case["k"]:]
            elif case["act"] == "gelu":
                v = v * torch.sigmoid(2 * 0.79788456 * (v + 0.044715 * v ** 3))
            top = v.abs().max(dim=1).values[:, None].clamp_min(1e-300)
            out[first:last] = (torch.round(127 * v / top) @ weights.t()) * (top / 127)
        row += m
    return out
