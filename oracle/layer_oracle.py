"""Plain 64-bit implementations of the operators around the GEMMs (test infrastructure only): the norm with 8-bit
codes, the product of 8-bit integers, the router.  numpy only."""
import numpy as np


def round_to(x, dtype):
    """float64 -> the nearest number of `dtype` ("fp16", "bf16", "fp32"), as float64."""
    with np.errstate(over="ignore"):
        if dtype == "fp32":
            return x.astype(np.float32).astype(np.float64)
        if dtype == "fp16":
            return x.astype(np.float16).astype(np.float64)
        # bf16: round to nearest even at 8 bits of the significand (one rounding, not by way of float32)
        m, e = np.frexp(x)
        step = np.ldexp(1.0, np.maximum(e - 8, -133))
        out = np.rint(x / step) * step
        return np.where(np.isfinite(x), out, x)


def rms_norm(x, weight, epsilon, residual=None, dtype="fp32"):
    """(z, y): the sum of x and the residual in `dtype`, and its norm, in 64 bits.  Inputs: float64 numbers of `dtype`."""
    z = x if residual is None else round_to(x + residual, dtype)
    y = z / np.sqrt(np.mean(z * z, axis=-1, keepdims=True) + epsilon) * weight
    return z, y


def scales_of(y, code):
    most = np.abs(y).max(axis=-1, keepdims=True)
    return np.maximum(most, 1e-10) / 127 if code == "int8" else np.maximum(most / 448, 1 / (448 * 512))


def scaled_mm_int8(a, b, a_scales, b_scales, bias=None):
    """a (M, K), b (N, K) int8 -> float64 (M, N).  Products of float64 integers: exact."""
    c = (a.astype(np.float64) @ b.astype(np.float64).T) * (np.reshape(a_scales, (-1, 1)).astype(np.float64) *
                                                          np.reshape(b_scales, (1, -1)).astype(np.float64))
    return c if bias is None else c + bias


def topk_routing(logits, topk, scoring="softmax", renormalize=False, bias=None, groups=1, kept_groups=1, factor=1.0):
    """(weights float64, ids), token after token, expert after expert."""
    logits = np.asarray(logits, dtype=np.float64)
    tokens, experts = logits.shape
    size = experts // groups
    weights, ids = np.zeros((tokens, topk)), np.zeros((tokens, topk), dtype=np.int64)
    for t in range(tokens):
        x = np.where(np.isnan(logits[t]), -np.inf, logits[t])
        with np.errstate(over="ignore", invalid="ignore"):
            if scoring == "sigmoid":
                s = np.where(x < 0, np.exp(np.minimum(x, 0)) / (1 + np.exp(np.minimum(x, 0))), 1 / (1 + np.exp(-np.abs(x))))
            else:
                top = x.max()
                e = np.where(x == -np.inf, 0.0, np.where(x == top, 1.0, np.exp(x - top)))
                s = e / e.sum() if e.sum() > 0 else e
        c = x if bias is None else s + np.asarray(bias, dtype=np.float64)
        c = np.where(np.isnan(c), -np.inf, c)
        per_group = -np.sort(-c.reshape(groups, size), axis=1)
        best = per_group[:, :1 if bias is None else 2].sum(axis=1)
        kept = sorted(range(groups), key=lambda g: (-best[g], g))[:kept_groups]
        chosen = sorted((e for e in range(experts) if e // size in kept), key=lambda e: (-c[e], e))[:topk]
        w = s[chosen]
        if renormalize and w.sum() > 0:
            w = w / w.sum()
        weights[t], ids[t] = w * factor, chosen
    return weights, ids


__all__ = ["rms_norm", "scales_of", "scaled_mm_int8", "topk_routing", "round_to"]
