"""The serving operators from their definitions in 64 bits (numpy), for the tests."""
import numpy as np
import torch


def as64(t):
    return t.detach().double().cpu().numpy()


def quantize(x):
    """(q, scale) of float64 rows: ties to even, scale in FP32."""
    largest = np.abs(x).max(axis=-1, keepdims=True)
    finite = np.isfinite(largest)
    unit = np.where(finite & (largest > 0), largest, 1.0)
    q = np.where(finite, np.rint(127.0 * np.where(finite, x, 0.0) / unit), 0.0)
    scale = np.where(finite, (np.where(finite, largest, 0.0).astype(np.float32) / np.float32(127.0)), np.float32(np.nan))
    return q, scale[..., 0].astype(np.float64)


def projection(q, scale, weight, weight_scale, bias=None):
    """The product, and the magnitude its roundings in 32 bits are relative to."""
    with np.errstate(invalid="ignore"):
        y = (q @ weight.T) * scale[:, None] * weight_scale[None, :]
    size = np.abs(y)
    if bias is not None:
        y, size = y + bias, size + np.abs(bias)
    return y, size


def silu(x):
    with np.errstate(over="ignore"):
        return x / (1.0 + np.exp(-x))


def projection_bound(y, size, eps, swiglu):
    """(result, bound).  FP32: the sum's conversion, two scales and the bias are four roundings of 2^-24 of at most
    ``size``; the store is half a step, ``eps`` / 2, of the result.  SwiGLU: |silu'| < 1.1, and the sigmoid's exponential
    and reciprocal are 2^-22 + 1.5 |x| 2^-24 and 2^-23 off; two products more."""
    off = 4 * 2.0 ** -24 * size
    if swiglu:
        half = y.shape[1] // 2
        g, v, dg, dv = y[:, :half], y[:, half:], off[:, :half], off[:, half:]
        s = silu(g)
        off = np.abs(v) * (1.1 * dg + np.abs(s) * (2.0 ** -21 + (1.5 * np.abs(g) + 2) * 2.0 ** -24)) + np.abs(s) * dv
        y = s * v
    return y, 1.01 * (off + eps / 2 * (np.abs(y) + off)) + 1e-37


def token(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, empty=-1):
    """One row, rule by rule."""
    logits = np.where(np.isnan(logits), -np.inf, logits)
    if not (logits > -np.inf).any():
        return empty
    if (logits == np.inf).any():
        logits = np.where(logits == np.inf, 0.0, -np.inf)
    order = np.lexsort((np.arange(logits.size), -logits))
    order = order[logits[order] > -np.inf]
    if not temperature > 1e-30 or top_p <= 0:
        return int(order[0])
    if top_k > 0:
        order = order[:top_k]
    w = np.exp((logits[order] - logits[order[0]]) / temperature)
    if top_p < 1:
        last = int(np.searchsorted(np.cumsum(w), top_p * w.sum(), side="left"))
        order, w = order[:last + 1], w[:last + 1]
    stays = w >= min(min_p, 1.0) if min_p > 0 else np.ones(w.size, bool)
    order, w = order[stays], w[stays]
    by_index = np.argsort(order)
    order, w = order[by_index], w[by_index]
    return int(order[min(np.searchsorted(np.cumsum(w), u * w.sum(), side="right"), order.size - 1)])


def tokens(logits, uniform, **settings):
    x, u = as64(logits), as64(uniform)
    # settings are FP32 numbers, whether one for all rows or a tensor
    rows = {k: (v.detach().cpu().tolist() if torch.is_tensor(v) else [v if k == "top_k" else float(np.float32(v))] * len(x))
            for k, v in settings.items()}
    return [token(x[i], u[i], **{k: v[i] for k, v in rows.items()}) for i in range(len(x))]
