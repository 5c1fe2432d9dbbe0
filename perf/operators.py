"""Operators of a decoder layer around this package's quantised GEMMs, as cases that can be timed.

A case is a dict of plain values; `what` says which operator one pass goes through:

  norm_quant  root-mean-square norm of (tokens, cols) rows, with the residual's addition before it and 8-bit codes with
              one scale a token behind it: what the 8-bit GEMMs read.  ops.rms_norm_per_token_quant
  int8_mm     product of int8 activations (m, k) and int8 weights (n, k) with a scale for each token and channel.
              ops.scaled_mm_int8
  router      the experts of each token from the router's logits (tokens, experts), and their weights: what
              fused_marlin_moe reads.  ops.topk_routing

`own` false: the same from elementary torch operations.  `own` true: the calls of this package."""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CODES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
EPSILON = 1e-5
#: The most elements of a drawn norm, multiply-adds of a drawn product and logits of a drawn router: those of the largest listed ones.
MOST_ELEMENTS = 16384 * 4096
MOST_PRODUCTS = 8192 * 4096 * 28672
MOST_LOGITS = 16384 * 256


def listed():
    return [
        # one sequence being decoded: the norm in front of a projection of an 8B decoder, where latency counts
        {"name": "norm_1_row", "what": "norm_quant", "tokens": 1, "cols": 4096, "dtype": "bf16", "codes": "int8",
         "residual": True, "norm": False},
        # a mixed batch of decodes and a prompt in front of an expert layer: the router reads the norm's 16-bit copy
        {"name": "norm_333_rows", "what": "norm_quant", "tokens": 333, "cols": 2880, "dtype": "fp16", "codes": "fp8",
         "residual": True, "norm": True},
        # a long prefill: the largest norm
        {"name": "norm_16384_rows", "what": "norm_quant", "tokens": 16384, "cols": 4096, "dtype": "bf16", "codes": "int8",
         "residual": True, "norm": False},
        # one sequence being decoded: the attention output projection of an 8B decoder
        {"name": "mm_1_row", "what": "int8_mm", "m": 1, "k": 4096, "n": 4096, "dtype": "bf16", "bias": False, "one_scale": False},
        # a small decode batch on the widest projection
        {"name": "mm_16_rows", "what": "int8_mm", "m": 16, "k": 4096, "n": 28672, "dtype": "bf16", "bias": False,
         "one_scale": False},
        # a short prompt on a qkv projection with a bias
        {"name": "mm_200_rows", "what": "int8_mm", "m": 200, "k": 4096, "n": 6144, "dtype": "fp16", "bias": True,
         "one_scale": False},
        # sizes that no tile divides and rows that no vector is aligned to
        {"name": "mm_odd_77_rows", "what": "int8_mm", "m": 77, "k": 1003, "n": 1537, "dtype": "bf16", "bias": True,
         "one_scale": True},
        # a chunk of a prompt on the down projection
        {"name": "mm_2048_rows", "what": "int8_mm", "m": 2048, "k": 14336, "n": 4096, "dtype": "bf16", "bias": False,
         "one_scale": False},
        # a long prefill on the widest projection: the largest product
        {"name": "mm_8192_rows", "what": "int8_mm", "m": 8192, "k": 4096, "n": 28672, "dtype": "bf16", "bias": False,
         "one_scale": False},
        # a decode step of a Mixtral-8x7B-shaped layer
        {"name": "router_16_tokens", "what": "router", "tokens": 16, "experts": 8, "topk": 2, "dtype": "bf16",
         "scoring": "softmax", "renormalize": True, "bias": False, "groups": 1, "kept_groups": 1, "factor": 1.0, "masked": 0},
        # a prefill of an expert layer of the shape of gpt-oss, logits in 32 bits
        {"name": "router_2000_tokens", "what": "router", "tokens": 2000, "experts": 32, "topk": 4, "dtype": "fp32",
         "scoring": "softmax", "renormalize": True, "bias": False, "groups": 1, "kept_groups": 1, "factor": 1.0, "masked": 0},
        # a long prefill with many small experts: sigmoid scores, a bias for balance, groups of experts; some are switched off
        {"name": "router_16384_tokens", "what": "router", "tokens": 16384, "experts": 256, "topk": 8, "dtype": "fp32",
         "scoring": "sigmoid", "renormalize": True, "bias": True, "groups": 8, "kept_groups": 4, "factor": 2.5, "masked": 5},
    ]


def _between(rng, low, high, step=1):
    """A whole number from low to high, spread over its logarithm, `step` apart."""
    x = int(round(math.exp(rng.uniform(math.log(low), math.log(high))) / step)) * step
    return min(high // step * step, max(-(-low // step) * step, x))


def draw(rng):
    what = rng.choice(["norm_quant", "int8_mm", "int8_mm", "router"])
    if what == "norm_quant":
        cols = _between(rng, 64, 16384, rng.choice([1, 8, 64]))
        return {"what": what, "tokens": min(_between(rng, 1, 16384), MOST_ELEMENTS // cols), "cols": cols,
                "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "codes": rng.choice(["int8", "int8", "fp8"]),
                "residual": rng.random() < 0.7, "norm": rng.random() < 0.3}
    if what == "int8_mm":
        step = rng.choice([1, 16, 64, 128])
        k, n = _between(rng, 256, 14336, step), _between(rng, 256, 28672, step)
        return {"what": what, "m": max(1, min(_between(rng, 1, 8192), MOST_PRODUCTS // (k * n))), "k": k, "n": n,
                "dtype": rng.choice(["bf16", "fp16"]), "bias": rng.random() < 0.4, "one_scale": rng.random() < 0.2}
    groups = rng.choice([1, 1, 2, 4, 8])
    experts = groups * _between(rng, 4, 512 // groups)
    kept = rng.randint(1, groups)
    topk = rng.randint(1, min(16, kept * (experts // groups)))
    return {"what": what, "tokens": min(_between(rng, 1, 16384), MOST_LOGITS // experts), "experts": experts, "topk": topk,
            "dtype": rng.choice(["fp32", "bf16", "fp16"]), "scoring": rng.choice(["softmax", "sigmoid"]),
            "renormalize": rng.random() < 0.7, "bias": rng.random() < 0.5, "groups": groups, "kept_groups": kept,
            "factor": rng.choice([1.0, 1.0, 2.5]), "masked": rng.choice([0, 0, 1])}


# ---------------------------------------------------------------- inputs
def _codes(gen, rows, cols):
    """int8 codes of normally distributed numbers whose row or column maximum is near 4 standard deviations."""
    x = torch.randn((rows, cols), device="cuda", generator=gen, dtype=torch.float16)
    return x.mul_(32).round_().clamp_(-127, 127).to(torch.int8)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, device="cuda", generator=gen)

    def rand(*shape):
        return torch.rand(shape, device="cuda", generator=gen)

    state = {"case": dict(case)}
    dtype = DTYPES[case["dtype"]]
    if case["what"] == "norm_quant":
        tokens, cols = case["tokens"], case["cols"]
        # a few channels of the residual stream carry values far above the others
        wide = 1 + 20 * (rand(cols) < 0.004)
        state["x"] = randn(tokens, cols).to(dtype)
        state["residual"] = (randn(tokens, cols) * 2 * wide).to(dtype) if case["residual"] else None
        state["weight"] = (1 + 0.2 * randn(cols)).to(dtype)
    elif case["what"] == "int8_mm":
        m, k, n = case["m"], case["k"], case["n"]
        state["a"] = _codes(gen, m, k)
        state["b"] = _codes(gen, n, k).t()   # a checkpoint's (n, k) weight, as the operator names it: (k, n)
        state["a_scales"] = rand(*((1, 1) if case["one_scale"] else (m, 1))) * 0.03 + 0.005
        state["b_scales"] = rand(n) * 4e-4 + 1e-4
        state["bias"] = (0.2 * randn(n)).to(dtype) if case["bias"] else None
    else:
        tokens, experts = case["tokens"], case["experts"]
        logits = randn(tokens, experts) * 1.5 + 0.5 * randn(experts)
        if case["masked"]:   # experts that are switched off for the whole batch
            logits[:, torch.randperm(experts, device="cuda", generator=gen)[:case["masked"]]] = -math.inf
        state["logits"] = logits.to(dtype)
        state["bias"] = 0.1 * randn(experts) if case["bias"] else None
    return state


# ---------------------------------------------------------------- the plain forms
def _norm_quant(x, weight, residual, codes, with_norm):
    z = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    # the mean in 64 bits: a code next to a border between two goes by its last bit
    inverse = torch.rsqrt(z.double().square().mean(-1, keepdim=True) + EPSILON).float()
    y = z.float() * inverse * weight.float()
    most = y.abs().amax(-1, keepdim=True)
    if codes == "int8":
        most = most.clamp(min=1e-10)
        limit = torch.full_like(most, 127.0)
        scales = most / limit
        t = y * (limit / most)
        q = torch.copysign(torch.floor(t.abs() + 0.5), t).to(torch.int8)
    else:
        scales = (most / torch.full_like(most, 448.0)).clamp(min=1 / (448.0 * 512.0))
        q = (y * (torch.ones_like(scales) / scales)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return q, scales, None if residual is None else z, y.to(x.dtype) if with_norm else None


def _int8_mm(a, b, a_scales, b_scales, dtype, bias):
    c = (a.float() @ b.float()) * (a_scales * b_scales)
    return (c if bias is None else c + bias.float()).to(dtype)


def _router(logits, case, bias):
    x = logits.float()
    x = torch.where(x.isnan(), -math.inf, x)
    # sigmoids far from 0 and sums with the bias next to each other: in 64 bits
    wide = x.double() if bias is not None or case["scoring"] == "sigmoid" else x
    if case["scoring"] == "sigmoid":
        scores = 1 / (1 + torch.exp(-wide))
    else:
        e = torch.exp(wide - wide.amax(-1, keepdim=True).clamp(min=-3e38))
        scores = e / e.sum(-1, keepdim=True).clamp(min=1e-300 if wide.dtype == torch.float64 else 1e-38)
    choice = x if bias is None else scores + bias.double()   # (without a bias the scores have the order of the logits)
    order = torch.sort(choice, dim=-1, descending=True, stable=True).indices
    groups, size = case["groups"], case["experts"] // case["groups"]
    if groups > 1:
        best = torch.sort(choice.view(-1, groups, size), dim=-1, descending=True).values
        of_group = best[..., 0] if bias is None or size == 1 else best[..., 0] + best[..., 1]
        chosen = torch.sort(of_group, dim=-1, descending=True, stable=True).indices[:, :case["kept_groups"]]
        kept = torch.zeros_like(of_group, dtype=torch.int8).scatter_(1, chosen, 1)
        of_order = kept.gather(1, order // size)
        order = order.gather(1, torch.sort(of_order, dim=-1, descending=True, stable=True).indices)
    ids = order[:, :case["topk"]]
    w = scores.gather(1, ids)
    if case["renormalize"]:
        total = w.sum(-1, keepdim=True)
        w = w / torch.where(total > 0, total, torch.ones_like(total))
    return (w * case["factor"]).float(), ids.to(torch.int32)


def _outputs(*values):
    return [v for v in values if v is not None]


def run(state):
    case = state["case"]
    if case["what"] == "norm_quant":
        if own:
            from sonar_amd import ops
            return _outputs(*ops.rms_norm_per_token_quant(state["x"], state["weight"], EPSILON, CODES[case["codes"]],
                                                          residual=state["residual"], with_norm=case["norm"]))
        return _outputs(*_norm_quant(state["x"], state["weight"], state["residual"], case["codes"], case["norm"]))
    if case["what"] == "int8_mm":
        if own:
            from sonar_amd import ops
            return ops.scaled_mm_int8(state["a"], state["b"], state["a_scales"], state["b_scales"], DTYPES[case["dtype"]],
                                      state["bias"])
        return _int8_mm(state["a"], state["b"], state["a_scales"], state["b_scales"], DTYPES[case["dtype"]], state["bias"])
    if own:
        from sonar_amd import ops
        return list(ops.topk_routing(state["logits"], case["topk"], case["scoring"], renormalize=case["renormalize"],
                                     bias=state["bias"], num_expert_group=case["groups"], topk_group=case["kept_groups"],
                                     routed_scaling_factor=case["factor"]))
    return list(_router(state["logits"], case, state["bias"]))


# ---------------------------------------------------------------- the definitions in 64 bits
def _exact_norm(state, case):
    x = state["x"].double()
    z = x if state["residual"] is None else (x + state["residual"].double()).to(state["x"].dtype).double()
    y = z / torch.sqrt((z * z).sum(-1, keepdim=True) / case["cols"] + EPSILON) * state["weight"].double()
    most = y.abs().max(-1, keepdim=True).values
    if case["codes"] == "int8":
        scales, q = torch.clamp(most, min=1e-10) / 127, None   # (codes are whole numbers)
    else:
        scales = torch.clamp(most / 448, min=1 / (448 * 512))
        q = y / scales
    out = [q, scales]
    if state["residual"] is not None:
        out.append(z)
    if case["norm"]:
        out.append(y)
    return out


def _exact_router(state, case):
    x = state["logits"].double().cpu().numpy()
    tokens, experts = x.shape
    x = np.where(np.isnan(x), -np.inf, x)
    with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
        if case["scoring"] == "sigmoid":
            scores = np.where(x >= 0, 1 / (1 + np.exp(-np.abs(x))), np.exp(-np.abs(x)) / (1 + np.exp(-np.abs(x))))
        else:
            top = x.max(axis=1)
            e = np.where(np.isneginf(x), 0.0, np.exp(x - np.where(np.isneginf(top), 0.0, top)[:, None]))
            total = e.sum(axis=1)
            scores = e / np.where(total > 0, total, 1.0)[:, None]
    choice = x if state["bias"] is None else scores + state["bias"].double().cpu().numpy()[None]
    size = experts // case["groups"]
    per_group = np.sort(choice.reshape(tokens, case["groups"], size), axis=2)[:, :, ::-1]
    of_group = per_group[:, :, 0] if state["bias"] is None or size == 1 else per_group[:, :, :2].sum(axis=2)
    best_groups = np.argsort(-of_group, axis=1, kind="stable")[:, :case["kept_groups"]]
    left_out = np.ones((tokens, case["groups"]), dtype=np.int8)
    np.put_along_axis(left_out, best_groups, 0, axis=1)
    left_out = np.repeat(left_out, size, axis=1)
    index = np.broadcast_to(np.arange(experts), x.shape)
    ids = np.lexsort((index, -choice, left_out), axis=1)[:, :case["topk"]]
    w = np.take_along_axis(scores, ids, axis=1)
    if case["renormalize"]:
        total = w.sum(axis=1, keepdims=True)
        w = w / np.where(total > 0, total, 1.0)
    return [w * case["factor"], None]   # (expert numbers are whole numbers)


def exact(case, seed):
    state = prepare(case, seed)
    if case["what"] == "norm_quant":
        return _exact_norm(state, case)
    if case["what"] == "int8_mm":
        scale = state["a_scales"].double() * state["b_scales"].double()
        c = torch.matmul(state["a"].double(), state["b"].double()).mul_(scale)
        return c if state["bias"] is None else c.add_(state["bias"].double())
    return _exact_router(state, case)


def work(case):
    if case["what"] == "norm_quant":
        size, n = 4 if case["dtype"] == "fp32" else 2, case["tokens"] * case["cols"]
        per_element = size + (2 * size if case["residual"] else 0) + 1 + (size if case["norm"] else 0)
        return {"bytes": n * per_element + case["cols"] * size + case["tokens"] * 4, "flops": 8 * n}
    if case["what"] == "int8_mm":
        m, k, n = case["m"], case["k"], case["n"]
        return {"bytes": m * k + k * n + 2 * m * n + 4 * n + (4 if case["one_scale"] else 4 * m) + (2 * n if case["bias"] else 0),
                "flops": 2 * m * k * n}
    size, n = 4 if case["dtype"] == "fp32" else 2, case["tokens"] * case["experts"]
    return {"bytes": n * size + case["tokens"] * case["topk"] * 8 + (4 * case["experts"] if case["bias"] else 0), "flops": 4 * n}
