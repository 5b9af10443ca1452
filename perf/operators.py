"""The operators of a quantised serving step: what is measured of them, and over which sizes.

Kinds of case (``kind``):

* ``linear``  ``int8_linear``: BF16 rows, quantised row by row, times an 8-bit weight with a scale for each output channel
* ``shared``  ``quantize_rows`` once, then two ``int8_matmul`` products of the same rows
* ``sample``  ``sample_tokens``: temperature, top-k, top-p and min-p on a batch of logits, from given uniform numbers

Widths are those of the package's models (hidden 1024 and 2048, gated MLPs of 2816 and 5632, vocabulary 32000, the fused
projection row of 7488 columns) and odd ones in between.

The plain forms follow the definitions.  A row is quantised as ``q = round(127 x / a)`` to nearest even with
``a = max |x|`` and stands for ``q * scale`` with ``scale = a / 127`` rounded to FP32; the quotient is taken in 64 bits,
since a value next to a half would otherwise depend on the order of two roundings.  Sampling is in 64 bits throughout: a
cumulative sum next to the drawn number decides a whole number.
"""
from __future__ import annotations

import math

import torch

own = False

VOCAB = 32000


def _linear(rows, width, columns, swiglu=False, bias=False, out="bf16"):
    return {"kind": "linear", "rows": rows, "width": width, "columns": columns, "swiglu": swiglu, "bias": bias, "out": out}


def _shared(rows, width, first, second):
    return {"kind": "shared", "rows": rows, "width": width, "first": first, "second": second}


def _sample(rows, vocab, dtype, temperature, top_k, top_p, min_p, mixed=False, banned=0.0):
    return {"kind": "sample", "rows": rows, "vocab": vocab, "dtype": dtype, "temperature": temperature, "top_k": top_k,
            "top_p": top_p, "min_p": min_p, "mixed": mixed, "banned": banned}


def listed():
    return [
        # one cached token through the gate/up projection of the 1024-wide model: the weight is read once
        dict(_linear(1, 1024, 5632, swiglu=True), name="token_gate_up"),
        # the down projection of a small serving batch: few output columns, a long sum
        dict(_linear(16, 2816, 1024), name="batch_down"),
        # nothing is a multiple of anything: rows that do not fill a tile, odd sums, odd rows in the result, with a bias
        dict(_linear(203, 1531, 2731, bias=True, out="fp32"), name="ragged_linear"),
        # the logits of 64 sequences, in FP32 for the sampler
        dict(_linear(64, 1024, VOCAB, out="fp32"), name="logits"),
        # a prompt of 4096 tokens through the gate/up projection of the 1024-wide model
        dict(_linear(4096, 1024, 5632, swiglu=True), name="prompt_gate_up"),
        # four prompts of 4096 tokens through the gate/up projection of the 2048-wide model
        dict(_linear(16384, 2048, 11264, swiglu=True), name="long_prompts_gate_up"),
        # the same rows for two projections of a serving batch: the fused projection row and the gate/up row
        dict(_shared(48, 1024, 7488, 5632), name="shared_rows_batch"),
        # the same for two prompts, with square weights
        dict(_shared(8192, 2048, 2048, 2048), name="shared_rows_prompts"),
        # one sequence, the usual settings of a chat
        dict(_sample(1, VOCAB, "bf16", 0.8, 50, 0.95, 0.0), name="sample_one"),
        # a serving batch whose requests each bring their own settings (greedy ones among them)
        dict(_sample(64, VOCAB, "bf16", 0.9, 0, 0.9, 0.02, mixed=True), name="sample_batch"),
        # odd vocabulary in FP32 (rows start at any 4 bytes), a grammar that bans most tokens, one row without any token
        dict(_sample(9, 50021, "fp32", 1.0, 0, 1.0, 0.05, banned=0.7), name="sample_banned"),
        # a large batch on a large vocabulary, nucleus sampling alone
        dict(_sample(512, 128000, "fp32", 0.7, 0, 0.95, 0.0), name="sample_large"),
    ]


def _between(rng, low, high):
    """A whole number, spread evenly over the logarithm of the range."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(("linear", "linear", "linear", "shared", "sample", "sample", "sample"))
    if kind == "sample":
        vocab = _between(rng, 200, 131072)
        rows = _between(rng, 1, max(1, min(512, 512 * 128000 // vocab)))
        return _sample(rows, vocab, rng.choice(("bf16", "bf16", "fp32")), round(rng.uniform(0.5, 1.5), 2),
                       rng.choice((0, 0, 1, 20, 50, 200, 1000)), rng.choice((1.0, 1.0, 0.95, 0.9, 0.5)),
                       rng.choice((0.0, 0.0, 0.02, 0.1)), mixed=rng.random() < 0.3, banned=rng.choice((0.0, 0.0, 0.5, 0.9)))
    rows = rng.choice((_between(rng, 1, 32), _between(rng, 1, 512), _between(rng, 64, 16384)))
    width, columns = _between(rng, 64, 8192), _between(rng, 64, 16384)
    if rng.random() < 0.6:   # model widths come in whole groups; the others end anywhere
        width, columns = max(64, width // 64 * 64), max(64, columns // 64 * 64)
    most = 16384 * 2048 * 11264
    while rows * width * columns > most or rows * columns > 16384 * 11264:
        rows = max(1, rows // 2)
    if kind == "shared":
        first = max(1, columns // rng.choice((2, 3)))
        return _shared(rows, width, first, columns - first)
    swiglu = rng.random() < 0.4
    return _linear(rows, width, columns - columns % 2 if swiglu else columns, swiglu=swiglu, bias=rng.random() < 0.3,
                   out=rng.choice(("bf16", "bf16", "fp32")))


# ---- inputs -------------------------------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _weight(gen, columns, width):
    """An 8-bit weight as a loaded model holds it: values drawn row by row, rows padded to whole groups of 16 bytes."""
    pitch = (width + 15) // 16 * 16
    store = torch.zeros(columns, pitch, dtype=torch.int8, device="cuda")
    values = torch.randn(columns, width, generator=gen, device="cuda").mul_(127 / 4.2).round_().clamp_(-127, 127)
    store[:, :width] = values.to(torch.int8)
    scale = (1 + 0.3 * torch.rand(columns, generator=gen, device="cuda")) * (4.2 / 127 / math.sqrt(width))
    return store[:, :width], scale


def _rows(gen, rows, width):
    """Normalised activations with a few channels that are much larger, as a residual stream has them."""
    x = torch.randn(rows, width, generator=gen, device="cuda")
    loud = torch.randint(0, width, (max(1, width // 200),), generator=gen, device="cuda")
    x[:, loud] *= 8
    return x.to(torch.bfloat16)


def _settings(case, gen):
    """Temperature, top-k, top-p and min-p: numbers for the whole batch, or a tensor each where requests differ."""
    names = ("temperature", "top_k", "top_p", "min_p")
    if not case["mixed"]:
        return {name: case[name] for name in names}
    rows = case["rows"]
    pick = torch.randint(0, 4, (rows,), generator=gen, device="cuda")
    temperature = torch.tensor([0.0, 0.6, case["temperature"], 1.3], device="cuda")[pick]
    pick = torch.randint(0, 4, (rows,), generator=gen, device="cuda")
    top_k = torch.tensor([0, 0, max(1, case["top_k"]), 40], dtype=torch.int32, device="cuda")[pick]
    pick = torch.randint(0, 3, (rows,), generator=gen, device="cuda")
    top_p = torch.tensor([1.0, 0.8, case["top_p"]], device="cuda")[pick]
    pick = torch.randint(0, 2, (rows,), generator=gen, device="cuda")
    min_p = torch.tensor([0.0, case["min_p"]], device="cuda")[pick]
    return {"temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p}


def prepare(case, seed):
    gen = _generator(seed)
    state = {"kind": case["kind"]}
    if case["kind"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        logits = 2.2 * torch.randn(rows, vocab, generator=gen, device="cuda")
        # a few likely continuations stand out of the bulk
        likely = torch.randint(0, vocab, (rows, 12), generator=gen, device="cuda")
        logits.scatter_add_(1, likely, 4 + 5 * torch.rand(rows, 12, generator=gen, device="cuda"))
        if case["banned"]:
            logits[torch.rand(rows, vocab, generator=gen, device="cuda") < case["banned"]] = -math.inf
            if rows > 2:
                logits[rows // 2] = -math.inf
        state["logits"] = logits.to(torch.float32 if case["dtype"] == "fp32" else torch.bfloat16)
        state["uniform"] = torch.rand(rows, generator=gen, device="cuda")
        state["settings"] = _settings(case, gen)
        return state
    state["x"] = _rows(gen, case["rows"], case["width"])
    if case["kind"] == "shared":
        state["weights"] = [_weight(gen, case[name], case["width"]) for name in ("first", "second")]
        return state
    state["weight"], state["scale"] = _weight(gen, case["columns"], case["width"])
    state["bias"] = torch.randn(case["columns"], generator=gen, device="cuda").to(torch.bfloat16) if case["bias"] else None
    state["swiglu"] = case["swiglu"]
    state["out"] = torch.float32 if case["out"] == "fp32" else torch.bfloat16
    return state


# ---- plain forms --------------------------------------------------------------------------------------------------
def _plain_quantize(x):
    """What the 8-bit rows hold, as FP32 whole numbers, and the rows' scales."""
    largest = x.abs().amax(dim=1, keepdim=True).double()
    q = (127.0 * x.double() / largest.clamp_min(torch.finfo(torch.float64).tiny)).round()
    return q.float(), largest.float() / 127.0


def _plain_product(q, scale, weight, weight_scale):
    # whole numbers up to 127 * 127 a term: FP32 products are exact and the sums lose no more than FP32 rounding
    return (q @ weight.float().t()) * scale * weight_scale


def _plain_linear(state):
    y = _plain_product(*_plain_quantize(state["x"]), state["weight"], state["scale"])
    if state["bias"] is not None:
        y = y + state["bias"].float()
    if state["swiglu"]:
        gate, value = y.chunk(2, dim=1)
        y = gate / (1 + torch.exp(-gate)) * value
    return y.to(state["out"])


def _plain_sample(state):
    logits, u, given = state["logits"], state["uniform"].double(), state["settings"]
    rows, vocab = logits.shape

    def column(name):
        return torch.as_tensor(given[name], device=logits.device).double().reshape(-1, 1).expand(rows, 1)

    temperature, top_k, top_p, min_p = (column(name) for name in ("temperature", "top_k", "top_p", "min_p"))
    greedy = temperature <= 0
    values, index = torch.sort(logits.double(), dim=1, descending=True, stable=True)   # ties: the lowest index first
    largest = values[:, :1]
    mass = torch.exp((values - largest) / torch.where(greedy, 1.0, temperature))
    rank = torch.arange(vocab, device=logits.device)
    k = torch.where(top_k <= 0, float(vocab), top_k)
    k = torch.where(greedy, 1.0, k)
    mass = torch.where(rank < k, mass, 0.0)
    before = torch.cumsum(mass, dim=1) - mass
    keep = (before < top_p * mass.sum(dim=1, keepdim=True)) | (top_p >= 1) | (rank == 0)
    keep &= (mass >= min_p) | (rank == 0)
    kept = torch.zeros_like(mass).scatter_(1, index, torch.where(keep, mass, 0.0))
    summed = torch.cumsum(kept, dim=1)
    token = (summed <= u[:, None] * summed[:, -1:]).sum(dim=1)
    return torch.where(torch.isneginf(largest[:, 0]), -1, token)


def run(state):
    if own:
        import solvedelta_b200 as sd

        if state["kind"] == "sample":
            return sd.sample_tokens(state["logits"], state["uniform"], **state["settings"])
        if state["kind"] == "shared":
            q, scale = sd.quantize_rows(state["x"])
            return [sd.int8_matmul(q, scale, weight, weight_scale) for weight, weight_scale in state["weights"]]
        return sd.int8_linear(state["x"], state["weight"], state["scale"], state["bias"], swiglu=state["swiglu"],
                              out_dtype=state["out"])
    if state["kind"] == "sample":
        return _plain_sample(state)
    if state["kind"] == "shared":
        q, scale = _plain_quantize(state["x"])
        return [_plain_product(q, scale, weight, weight_scale).to(torch.bfloat16) for weight, weight_scale in state["weights"]]
    return _plain_linear(state)


def work(case):
    if case["kind"] == "sample":
        size = 4 if case["dtype"] == "fp32" else 2
        entries = case["rows"] * case["vocab"]
        # every logit is read once and compared once; the draw's numbers and the tokens are a few bytes a row
        return {"bytes": entries * size + case["rows"] * 12, "flops": entries}
    rows, width = case["rows"], case["width"]
    columns = case["first"] + case["second"] if case["kind"] == "shared" else case["columns"]
    moved = 2 * rows * width + columns * width + 4 * columns
    if case["kind"] == "linear":
        moved += 2 * columns if case["bias"] else 0
        moved += rows * (columns // 2 if case["swiglu"] else columns) * (4 if case["out"] == "fp32" else 2)
    else:
        moved += 2 * rows * columns
    return {"bytes": moved, "flops": 2 * rows * width * columns}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------
def _exact_projection(x, weight, weight_scale):
    """sum over k of q[i,k] W[j,k], whole numbers that 64 bits hold, times both scales (which are kept in FP32)."""
    x = x.to(torch.float64)
    top = x.abs().max(dim=1).values
    unit = torch.where(top > 0, top, torch.ones_like(top))
    q = torch.round(x * 127 / unit[:, None])
    scale = (top / 127).to(torch.float32).to(torch.float64)
    return torch.matmul(q, weight.to(torch.float64).t()) * weight_scale.to(torch.float64) * scale[:, None]


def _exact_token(logits, u, temperature, top_k, top_p, min_p):
    """One row, step by step as the definition goes, on the host."""
    import numpy as np

    if not np.isfinite(logits).any():
        return -1
    if temperature == 0:
        return int(np.argmax(logits))
    order = np.lexsort((np.arange(logits.size), -logits))
    if top_k > 0:
        order = order[:top_k]
    p = np.exp((logits[order] - logits[order[0]]) / temperature)
    if top_p < 1:
        last = int(np.searchsorted(np.cumsum(p), top_p * p.sum(), side="left"))
        order, p = order[:last + 1], p[:last + 1]
    stays = p >= min_p
    stays[0] = True
    by_index = np.argsort(order[stays])
    chosen, p = order[stays][by_index], p[stays][by_index]
    return int(chosen[np.searchsorted(np.cumsum(p), u * p.sum(), side="right")])


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "sample":
        logits, u = state["logits"].double().cpu().numpy(), state["uniform"].double().cpu().numpy()
        if logits.size > 80_000_000:
            return None
        rows = [[float(v) for v in (s.cpu().tolist() if torch.is_tensor(s) else [s] * case["rows"])]
                for s in (state["settings"][n] for n in ("temperature", "top_k", "top_p", "min_p"))]
        return torch.tensor([_exact_token(logits[i], u[i], rows[0][i], int(rows[1][i]), rows[2][i], rows[3][i])
                             for i in range(case["rows"])])
    if case["kind"] == "shared":
        return [_exact_projection(state["x"], *pair) for pair in state["weights"]]
    y = _exact_projection(state["x"], state["weight"], state["scale"])
    if state["bias"] is not None:
        y += state["bias"].to(torch.float64)
    if state["swiglu"]:
        half = y.shape[1] // 2
        y = y[:, :half] * torch.sigmoid(y[:, :half]) * y[:, half:]
    return y
