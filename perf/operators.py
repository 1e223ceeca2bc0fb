"""The decode step's operators and the cases that measure them: the draw from given uniforms, the
quantisation to 8-bit floating point with a scale per block of 128, and the language-model head's
product of such codes.

  draw          rows of logits (f32, bf16, fp16) and one uniform a row -> a token a row, under
                temperature, top-k, top-p and min-p
  quant_rows    activations -> e4m3 codes, one f32 scale per row and 128 columns
  quant_blocks  weights -> e4m3 codes, one f32 scale per 128 x 128 block
  logits        codes of hidden states times codes of the head's weights -> logits

`own` false computes them in elementary torch operations; true makes the framework's calls.
"""
import os
import sys

import torch

own = False

BLOCK = 128
E4M3_MAX = 448.0
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
_lrs = None


def _package():
    """The framework's package (llama.rs_b200/ holds it)."""
    global _lrs
    if _lrs is None:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        sys.path.insert(0, os.path.join(root, "llama.rs_b200"))
        import lrs
        _lrs = lrs
    return _lrs


# ------------------------------------------------------------------------------- cases ----
def listed():
    return [
        # one stream at the full vocabulary, the sampler's default filters: latency
        {"name": "draw_one", "op": "draw", "rows": 1, "n": 151936, "dtype": "f32", "values": "normal", "filters": "default"},
        # the benchmark's headline batch: Zipf-like rows, mixed parameters
        {"name": "draw_headline", "op": "draw", "rows": 1024, "n": 151936, "dtype": "f32", "values": "zipf", "filters": "mixed"},
        # the pruned vocabulary (odd rows, no row after the first on a 16-byte boundary) in 16 bits, min-p
        {"name": "draw_pruned", "op": "draw", "rows": 256, "n": 109051, "dtype": "bf16", "values": "normal", "filters": "min_p"},
        # nuclei of tens of thousands of tokens: flat and spiked rows under top-p alone
        {"name": "draw_nucleus", "op": "draw", "rows": 512, "n": 151936, "dtype": "f32", "values": "flat", "filters": "top_p"},
        # no filter: the plain inverse of the distribution function, 16 bits, a short odd row
        {"name": "draw_plain", "op": "draw", "rows": 48, "n": 32003, "dtype": "f16", "values": "normal", "filters": "none"},
        # a decode step's hidden states, one stream
        {"name": "quant_rows_one", "op": "quant_rows", "rows": 1, "k": 1024, "dtype": "bf16"},
        # a prompt's hidden states, odd width: the last block is short
        {"name": "quant_rows_prompt", "op": "quant_rows", "rows": 8191, "k": 5000, "dtype": "f16"},
        # the head's weights, laid out once when a model is loaded
        {"name": "quant_head", "op": "quant_blocks", "rows": 151936, "k": 1024, "dtype": "bf16"},
        # one stream's logits: the weights' bytes are all there is
        {"name": "logits_one", "op": "logits", "rows": 1, "n": 151936, "k": 1024, "dtype": "f32"},
        # a batch of streams on the pruned vocabulary, 16-bit logits
        {"name": "logits_batch", "op": "logits", "rows": 64, "n": 109051, "k": 2048, "dtype": "bf16"},
        # odd everything: rows, vocabulary and width
        {"name": "logits_odd", "op": "logits", "rows": 237, "n": 109051, "k": 1000, "dtype": "f32"},
        # the headline batch from a wide model
        {"name": "logits_headline", "op": "logits", "rows": 1024, "n": 151936, "k": 4096, "dtype": "f32"},
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(lo * (hi / lo) ** rng.random() + 0.5)))


def draw(rng):
    op = rng.choice(["draw", "draw", "draw", "quant_rows", "quant_blocks", "logits", "logits", "logits"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "draw":
        n = _log(rng, 40, 200000)
        rows = _log(rng, 1, min(2048, max(1, 1024 * 151936 // n)))
        return {"op": op, "rows": rows, "n": n, "dtype": dtype, "values": rng.choice(["normal", "zipf", "flat", "masked"]),
                "filters": rng.choice(["default", "mixed", "min_p", "top_p", "top_k", "none", "greedy"])}
    if op == "quant_rows":
        return {"op": op, "rows": _log(rng, 1, 8191), "k": _log(rng, 100, 8000), "dtype": dtype}
    if op == "quant_blocks":
        return {"op": op, "rows": _log(rng, 500, 151936), "k": _log(rng, 100, 2000), "dtype": dtype}
    return {"op": op, "rows": _log(rng, 1, 1024), "n": _log(rng, 500, 151936), "k": _log(rng, 100, 4096), "dtype": dtype}


# ------------------------------------------------------------------------------ inputs ----
def _padded(rows, cols, dtype, device, unit=16):
    """An uninitialised [rows, cols] view whose row stride is a multiple of `unit` elements."""
    return torch.empty(rows, -(-cols // unit) * unit, dtype=dtype, device=device)[:, :cols]


def _values(case, g, device):
    """Rows of logits with the distributions of the samplers' workloads."""
    rows, n, kind = case["rows"], case["n"], case["values"]
    if kind == "zipf":  # Gumbel noise under a Zipf-like head, in random order
        x = -torch.log(-torch.log(torch.rand(rows, n, generator=g, device=device).clamp(1e-30, 1 - 2.0 ** -24)))
        x -= 2.2 * torch.log(torch.rand(rows, n, generator=g, device=device).argsort(dim=1).float() + 1)
    else:
        x = torch.randn(rows, n, generator=g, device=device)
    if kind == "flat":  # even rows flat, odd rows wide with one token far above the others
        odd = (torch.arange(rows, device=device) % 2)[:, None]
        x *= 0.5 + 1.5 * odd
        x.scatter_add_(1, torch.randint(0, n, (rows, 1), generator=g, device=device), 12.0 * odd)
    elif kind != "zipf":
        x *= 3.0
    if kind == "masked":  # a grammar's mask: most tokens are closed, the last one is open
        shut = torch.rand(rows, n, generator=g, device=device) < 0.95
        shut[:, -1] = False
        x = x.masked_fill_(shut, -float("inf"))
    return x.to(TYPES[case["dtype"]])


def _filters(case, g, device):
    """Temperature, top-k (0: off), top-p (1: off) and min-p (0: off) of every row."""
    rows, kind = case["rows"], case["filters"]
    u = torch.rand(4, rows, generator=g, device=device)
    t = torch.full((rows,), 1.0, device=device)
    k = torch.zeros(rows, dtype=torch.int32, device=device)
    p = torch.ones(rows, device=device)
    m = torch.zeros(rows, device=device)
    if kind == "default":
        t, k, p = t * 0.7, k + 40, p * 0.95
    elif kind == "mixed":
        t, p = 0.5 + u[0], 0.8 + 0.2 * u[1]
        k = torch.tensor([0, 20, 40, 100], dtype=torch.int32, device=device)[(u[2] * 4).long()]
        m = torch.tensor([0.0, 0.02, 0.05, 0.1], device=device)[(u[3] * 4).long()]
    elif kind == "min_p":
        t, m = 0.5 + u[0], 0.02 + 0.08 * u[1]
    elif kind == "top_p":
        p = 0.85 + 0.1 * u[1]
    elif kind == "top_k":
        k = torch.tensor([1, 5, 50, 1000], dtype=torch.int32, device=device)[(u[2] * 4).long()]
    elif kind == "greedy":
        t = t * 0
    return t, k, p, m


def _quantize(x, tall):
    """e4m3 codes and scales of x in blocks of 1 x 128 (scales [block][row]) or 128 x 128."""
    rows, k = x.shape
    kb, rb = -(-k // BLOCK), -(-rows // BLOCK)
    y = torch.nn.functional.pad(x.float(), (0, kb * BLOCK - k, 0, rb * BLOCK - rows if tall else 0))
    y = y.view(rb, BLOCK, kb, BLOCK) if tall else y.view(rows, 1, kb, BLOCK)
    scale = (y.abs().amax(dim=(1, 3)) / E4M3_MAX).clamp_min(2.0 ** -126)
    code = (y * (1.0 / scale)[:, None, :, None]).to(torch.float8_e4m3fn)
    code = code.view(-1, kb * BLOCK)[:rows, :k]
    return code, (scale if tall else scale.t().contiguous())


def prepare(case, seed):
    device = torch.device("cuda:0")
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    rows, op = case["rows"], case["op"]
    s = {"op": op}
    if op == "draw":
        s["logits"] = _values(case, g, device)
        s["temperature"], s["top_k"], s["top_p"], s["min_p"] = _filters(case, g, device)
        # the same as records of {f32 temperature, u32 top_k, f32 top_p, f32 min_p}
        s["params"] = torch.stack([s["temperature"].view(torch.int32), s["top_k"], s["top_p"].view(torch.int32),
                                   s["min_p"].view(torch.int32)], dim=1).contiguous()
        s["uniform"] = torch.rand(rows, generator=g, device=device)
        for name in ("tokens", "kept", "status"):
            s[name] = torch.zeros(rows, dtype=torch.int32, device=device)
        s["probs"] = torch.zeros(rows, device=device)
    elif op in ("quant_rows", "quant_blocks"):
        k = case["k"]
        # hidden states with a few wide columns, or weights whose rows differ in size
        x = torch.randn(rows, k, generator=g, device=device)
        if op == "quant_rows":
            x *= torch.exp(torch.randn(k, generator=g, device=device))
        else:
            x *= 0.02 * torch.exp(0.5 * torch.randn(rows, 1, generator=g, device=device))
        s["x"] = x.to(TYPES[case["dtype"]])
        s["codes"] = _padded(rows, k, torch.float8_e4m3fn, device)
        kb = -(-k // BLOCK)
        s["scales"] = torch.zeros((kb, rows) if op == "quant_rows" else (-(-rows // BLOCK), kb), device=device)
    else:
        n, k = case["n"], case["k"]
        h = torch.randn(rows, k, generator=g, device=device) * torch.exp(0.5 * torch.randn(k, generator=g, device=device))
        w = torch.randn(n, k, generator=g, device=device) * (2.0 / k ** 0.5)
        for name, x, tall in (("hidden", h, False), ("weight", w, True)):
            code, scale = _quantize(x, tall)
            s[name] = _padded(*x.shape, torch.float8_e4m3fn, device)
            s[name].copy_(code)
            s[name + "_scales"] = scale
        s["out"] = torch.zeros(rows, n, dtype=TYPES[case["dtype"]], device=device)
    return s


# ----------------------------------------------------------------------- the operators ----
def _plain_draw(s):
    x = s["logits"].float()
    rows, n = x.shape
    t = s["temperature"].double()[:, None]
    greedy = t <= 0
    k = s["top_k"].long()[:, None]
    k = torch.where(greedy, 1, torch.where(k == 0, n, k))
    p, m = s["top_p"].double()[:, None], s["min_p"].double()[:, None]
    v, at = torch.sort(x, dim=1, descending=True, stable=True)  # ties: the lowest index first
    v = v.double()
    w = torch.exp((v - v[:, :1]) / torch.where(greedy, 1.0, t))
    c = torch.cumsum(w, dim=1)
    before = torch.nn.functional.pad(c[:, :-1], (1, 0))
    keep = (torch.arange(n, device=x.device)[None] < k) & (w >= m) & ((before < p * c[:, -1:]) | (p >= 1) | (p <= 0))
    keep &= v > -float("inf")
    w = torch.where(keep, w, 0.0)
    w = torch.zeros_like(w).scatter_(1, at, w)  # back in the vocabulary's order
    c = torch.cumsum(w, dim=1)
    total = c[:, -1:]
    token = (c <= s["uniform"].double()[:, None] * total).sum(dim=1, keepdim=True)
    prob = (w.gather(1, token) / total)[:, 0].float()
    return [token[:, 0].int(), prob, keep.sum(dim=1).int(), torch.zeros(rows, dtype=torch.int32, device=x.device)]


def _plain_logits(s):
    def values(code, scale, tall):
        rows, k = code.shape
        wide = scale.repeat_interleave(BLOCK, dim=1)[:, :k]
        return code.float() * (wide.repeat_interleave(BLOCK, dim=0)[:rows] if tall else wide)
    a = values(s["hidden"], s["hidden_scales"].t(), False)
    w = values(s["weight"], s["weight_scales"], True)
    return (a @ w.t()).to(s["out"].dtype)


def run(s):
    op = s["op"]
    if own:
        L = _package()
        if op == "draw":
            L.BatchSampler.draw_device(s["logits"], s["params"], s["uniform"], s["tokens"], probs=s["probs"],
                                       kept=s["kept"], status=s["status"])
            return [s["tokens"], s["probs"], s["kept"], s["status"]]
        if op == "quant_rows":
            L.quantize_rows(s["x"], s["codes"], s["scales"])
            return [s["codes"], s["scales"]]
        if op == "quant_blocks":
            L.quantize_blocks(s["x"], s["codes"], s["scales"])
            return [s["codes"], s["scales"]]
        L.fp8_logits(s["hidden"], s["hidden_scales"], s["weight"], s["weight_scales"], s["out"])
        return [s["out"]]
    if op == "draw":
        return _plain_draw(s)
    if op in ("quant_rows", "quant_blocks"):
        return list(_quantize(s["x"], op == "quant_blocks"))
    return [_plain_logits(s)]


def work(case):
    rows, op = case["rows"], case["op"]
    if op == "draw":
        n = case["n"]  # the logits once, the parameters, uniforms and results of every row; one exp an element
        return {"bytes": rows * (n * SIZE[case["dtype"]] + 36), "flops": 4.0 * rows * n}
    k = case["k"]
    kb = -(-k // BLOCK)
    if op in ("quant_rows", "quant_blocks"):
        scales = kb * (rows if op == "quant_rows" else -(-rows // BLOCK))
        return {"bytes": rows * k * (SIZE[case["dtype"]] + 1) + 4 * scales, "flops": 3.0 * rows * k}
    n = case["n"]
    scales = kb * (rows + -(-n // BLOCK))
    return {"bytes": (rows + n) * k + 4 * scales + rows * n * SIZE[case["dtype"]], "flops": 2.0 * rows * n * k}


# ----------------------------------------------------------------- the definition, 64 bits ----
def _exact_draw(s):
    """By normalised probabilities: the filters as a number of ranks, the token by a search of the
    kept distribution function."""
    x = s["logits"].double()
    rows, n = x.shape
    t, m, p, u = (s[f].double()[:, None] for f in ("temperature", "min_p", "top_p", "uniform"))
    k = s["top_k"].long()[:, None]
    k = torch.where(t <= 0, 1, torch.where((k <= 0) | (k > n), n, k))
    t = torch.where(t <= 0, 1.0, t)
    prob = torch.softmax(x / t, dim=1)
    order = torch.argsort(-x, dim=1, stable=True)  # ties: ascending index
    reach = torch.cumsum(prob.gather(1, order), dim=1)
    count = torch.where((p > 0) & (p < 1), (reach < p * reach[:, -1:]).sum(dim=1, keepdim=True) + 1, n)
    near = ((x - x.amax(dim=1, keepdim=True)) / t >= torch.log(m)).sum(dim=1, keepdim=True)
    count = torch.minimum(torch.minimum(count, near), torch.minimum(k, torch.isfinite(x).sum(dim=1, keepdim=True)))
    rank = torch.empty_like(order).scatter_(1, order, torch.arange(n, device=x.device).repeat(rows, 1))
    kept = prob * (rank < count)
    cdf = torch.cumsum(kept, dim=1)
    token = torch.searchsorted(cdf, u * cdf[:, -1:], right=True)
    return [token[:, 0].int(), (kept.gather(1, token) / cdf[:, -1:])[:, 0], count[:, 0].int(),
            torch.zeros(rows, dtype=torch.int32, device=x.device)]


def _exact_quant(x, tall):
    """Codes as values in 64 bits: x over its block's scale, rounded to 4 significant bits (to the
    multiples of 2^-9 below 2^-6), ties to even."""
    x = x.double()
    rows, k = x.shape
    high = BLOCK if tall else 1
    scale = torch.stack([b.abs().amax(dim=1) for b in x.split(BLOCK, dim=1)])  # [kb][rows]
    if tall:
        scale = torch.stack([b.amax(dim=1) for b in scale.split(high, dim=1)])  # [rb][kb]
    scale = (scale / E4M3_MAX).clamp_min(2.0 ** -126)
    wide = (scale.repeat_interleave(high, dim=0)[:rows] if tall else scale.t()).repeat_interleave(BLOCK, dim=1)[:, :k]
    v = x / wide
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
    return [(torch.round(v / step) * step).clamp(-E4M3_MAX, E4M3_MAX), scale]


def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op == "draw":
        return _exact_draw(s)
    if op in ("quant_rows", "quant_blocks"):
        return _exact_quant(s["x"], op == "quant_blocks")
    n, k = s["weight"].shape
    out = torch.zeros(s["hidden"].shape[0], n, dtype=torch.float64, device=s["out"].device)
    for j in range(-(-k // BLOCK)):  # block by block, scaled after each block's sum
        at = slice(j * BLOCK, min(k, (j + 1) * BLOCK))
        part = s["hidden"][:, at].double() @ s["weight"][:, at].double().t()
        column = s["weight_scales"][:, j].double().repeat_interleave(BLOCK)[:n]
        out += part * s["hidden_scales"][j].double()[:, None] * column[None]
    return [out]
