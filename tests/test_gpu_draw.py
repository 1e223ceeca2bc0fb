"""GPU tests of lrs_draw_device: tokens, probabilities, kept counts and statuses against the 64-bit
definition.  Tokens, counts and statuses are equal; a probability is the real one rounded once to
f32, so it is off by at most half a step (2^-24 relative), plus 2^-38 for the 64-bit sums of up to
2^18 weights (each good to a few 2^-52) and 2^-149 where it is subnormal."""
import numpy as np
import pytest

import lrs
from draw_ref import NONE, draw_row

pytestmark = pytest.mark.gpu

FILTERS = {
    "none": (1.0, 0, 1.0, 0.0),
    "default": (0.7, 40, 0.95, 0.0),
    "top_k": (1.0, 7, 1.0, 0.0),
    "top_k_big": (1.3, 900, 1.0, 0.0),
    "top_p": (1.0, 0, 0.9, 0.0),
    "top_p_low": (1.0, 0, 0.02, 0.0),
    "min_p": (0.8, 0, 1.0, 0.05),
    "all": (1.2, 60, 0.93, 0.01),
    "greedy": (0.0, 40, 0.95, 0.1),
}


def types():
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def records(rows, filters):
    p = np.zeros(rows, lrs.DRAW_PARAMS_DTYPE)
    for r in range(rows):
        p[r] = tuple(filters[r % len(filters)])
    return p


def run(x, params, u, rows=None, **kw):
    """x a CUDA tensor; returns (tokens, probs, kept, status) as numpy, with a sentinel row behind."""
    import torch
    rows = len(u) if rows is None else rows
    d = x.device
    out = dict(probs=torch.full((rows + 1,), -7.0, device=d))
    for name in ("tokens", "kept", "status"):
        out[name] = torch.full((rows + 1,), -77, dtype=torch.int32, device=d)
    lrs.BatchSampler.draw_device(x, torch.from_numpy(params.view(np.uint8)).to(d),
                                 torch.from_numpy(np.asarray(u, np.float32)).to(d), out["tokens"], probs=out["probs"],
                                 kept=out["kept"], status=out["status"], rows=rows, **kw)
    torch.cuda.synchronize()
    o = {k: v.cpu().numpy() for k, v in out.items()}
    assert o["tokens"][rows] == o["kept"][rows] == o["status"][rows] == -77 and o["probs"][rows] == -7.0
    return o["tokens"][:rows].view(np.uint32), o["probs"][:rows], o["kept"][:rows].view(np.uint32), o["status"][:rows]


def check(got, x, params, u, label=""):
    """x: the rows as float64."""
    for r in range(len(u)):
        st, token, prob, kept = draw_row(x[r], *params[r], u[r])
        g = tuple(a[r] for a in got)
        assert (g[3], g[0], g[2]) == (st, token, kept), (label, r, params[r], u[r], g, (st, token, prob, kept))
        assert abs(float(g[1]) - prob) <= prob * (2.0 ** -24 + 2.0 ** -38) + 2.0 ** -149, (label, r, g, prob)


def matrix(rng, rows, n, kind):
    if kind == "flat":
        return rng.standard_normal((rows, n)) * 0.5
    if kind == "ties":  # a dozen levels: every cut falls inside a run of equal logits
        return rng.integers(0, 12, (rows, n)) * 0.5
    if kind == "masked":
        x = rng.standard_normal((rows, n)) * 3
        x[rng.random((rows, n)) < 0.97] = -np.inf
        x[:, rng.integers(0, n)] = 0.0
        return x
    return rng.standard_normal((rows, n)) * 3


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kind", ["normal", "flat", "ties", "masked"])
@pytest.mark.parametrize("n", [1, 2, 3, 31, 33, 127, 128, 129, 1000, 1025, 4099, 9001])
def test_against_the_definition(dtype, kind, n):
    import torch
    rng = np.random.default_rng([n, len(kind), len(dtype)])
    rows = 2 * len(FILTERS)
    x = torch.from_numpy(matrix(rng, rows, n, kind)).to(types()[dtype]).cuda()
    params, u = records(rows, list(FILTERS.values())), rng.random(rows, np.float32)
    check(run(x, params, u), x.double().cpu().numpy(), params, u, (dtype, kind, n))


@pytest.mark.parametrize("dtype,n,rows", [("f32", 151936, 18), ("bf16", 109051, 18), ("f16", 32003, 150),
                                          ("f32", 151936, 1), ("bf16", 151936, 3), ("f32", 5000, 700)])
@pytest.mark.parametrize("kind", ["normal", "flat", "ties"])
def test_vocabularies_and_batches(dtype, n, rows, kind):
    import torch
    rng = np.random.default_rng([n, rows, len(kind)])
    x = torch.from_numpy(matrix(rng, rows, n, kind)).to(types()[dtype]).cuda()
    names = list(FILTERS.values()) if rows > 1 else [FILTERS["default"]]
    for f in [names] if rows > 1 else [[v] for v in FILTERS.values()]:
        params, u = records(rows, f), rng.random(rows, np.float32)
        check(run(x, params, u), x.double().cpu().numpy(), params, u, (dtype, n, kind))


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("offset,pad", [(0, 0), (1, 0), (3, 5), (2, 1), (7, 9)])
def test_strides_and_alignments(dtype, offset, pad):
    import torch
    rng = np.random.default_rng([offset, pad])
    rows, n = 9, 2049
    flat = torch.full((offset + rows * (n + pad),), float("nan"), dtype=types()[dtype], device="cuda")  # (pads never read)
    x = flat[offset:].view(rows, n + pad)[:, :n]
    x.copy_(torch.from_numpy(matrix(rng, rows, n, "normal")))
    params, u = records(rows, list(FILTERS.values())), rng.random(rows, np.float32)
    check(run(x, params, u), x.double().cpu().numpy(), params, u, (offset, pad))


def test_every_row_may_read_one_row():
    import torch
    rng = np.random.default_rng(5)
    x = torch.from_numpy(matrix(rng, 1, 3001, "normal")).float().cuda()
    params, u = records(40, list(FILTERS.values())), rng.random(40, np.float32)
    want = np.repeat(x.double().cpu().numpy(), 40, axis=0)
    check(run(x, params, u), want, params, u)
    check(run(x.expand(40, 3001), params, u), want, params, u)
    check(run(x, params, u, ld=0), want, params, u)


def test_rows_without_a_distribution_and_bad_parameters():
    import torch
    rng = np.random.default_rng(6)
    n, good = 700, FILTERS["all"]
    x = rng.standard_normal((16, n))
    x[0] = -np.inf
    x[1, 0], x[2, n - 1], x[3, 350] = np.nan, np.nan, np.inf
    x[4, :] = np.inf
    x[5, 1:] = -np.inf
    params, u = records(16, [good]), rng.random(16, np.float32)
    params[6]["temperature"], params[7]["temperature"] = np.nan, np.inf
    params[8]["top_p"], params[9]["min_p"], params[10]["min_p"], params[11]["min_p"] = np.nan, -0.5, 1.5, np.nan
    u[12], u[13], u[14] = 1.0, -0.25, np.nan
    params[15] = (0.0, 9, np.nan, 7.0)  # greedy reads none of the others
    u[15] = 5.0
    t = torch.from_numpy(x).float().cuda()
    got = run(t, params, u)
    check(got, t.double().cpu().numpy(), params, u)
    assert list(got[3]) == [-2] * 5 + [0] + [-1] * 9 + [0] and (got[0][:5] == NONE).all()
    params["temperature"] = -1.0  # greedy rows see a NaN too
    got = run(t, params, u)
    assert list(got[3][:6]) == [-2] * 5 + [0]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_masks_of_the_types_lowest_value(dtype):
    """Masked entries are finite here: they count among the kept where no filter drops them, and have a
    weight of 0 in 64 bits."""
    import torch
    rng = np.random.default_rng(7)
    x = torch.from_numpy(matrix(rng, 18, 5003, "normal")).to(types()[dtype]).cuda()
    x[:, torch.from_numpy(rng.random(5003) < 0.999).cuda()] = torch.finfo(x.dtype).min
    x[4] = torch.finfo(x.dtype).min  # nothing but the mask: every entry alike
    params, u = records(18, list(FILTERS.values())), rng.random(18, np.float32)
    check(run(x, params, u), x.double().cpu().numpy(), params, u, dtype)


def test_equal_logits_are_cut_by_index():
    import torch
    n = 1003
    x = torch.full((12, n), 1.25, device="cuda")
    params = records(12, [(0.9, 10, 1.0, 0.0), (1.0, 0, 0.5, 0.0), (2.0, 0, 1.0, 1.0), (1.0, 100, 0.25, 1.0)])
    u = np.linspace(0, 1 - 2.0 ** -24, 12).astype(np.float32)
    got = run(x, params, u)
    check(got, np.full((12, n), 1.25), params, u)
    assert list(got[2][:4]) == [10, 502, 1003, 100]


@pytest.mark.parametrize("t", [1e-45, 1e-30, 1e-3, 1e3, 1e30, 3e38])
def test_temperatures(t):
    import torch
    rng = np.random.default_rng(8)
    x = torch.from_numpy(matrix(rng, 8, 3000, "ties")).float().cuda()
    x[3] *= 1e30
    x[4, 5:] = -3e38
    x[4, :5] = 3e38
    params, u = records(8, [(t, 0, 1.0, 0.0), (t, 50, 0.9, 0.0), (t, 0, 0.5, 0.0), (t, 0, 1.0, 0.5)]), rng.random(8, np.float32)
    check(run(x, params, u), x.double().cpu().numpy(), params, u, t)


def test_uniforms_at_their_ends_and_tiny_filters():
    import torch
    rng = np.random.default_rng(9)
    x = torch.from_numpy(matrix(rng, 24, 2500, "normal")).float().cuda()
    params = records(24, [(1.0, 0, 1.0, 0.0), (1.0, 0, 1e-30, 0.0), (1.0, 0, 1 - 2.0 ** -24, 0.0), (1.0, 2500, 1.0, 0.0),
                          (1.0, 2499, 0.99999, 1e-30), (1.0, 1, 0.5, 0.5), (1.0, 0xFFFFFFFF, 0.0, 1.0), (1.0, 0, -1.0, 1e-6)])
    u = np.resize(np.array([0.0, 1 - 2.0 ** -24, 2.0 ** -149], np.float32), 24)
    check(run(x, params, u), x.double().cpu().numpy(), params, u)


@pytest.mark.parametrize("rows", [2, 40, 200])
def test_long_rows_of_every_make(rows):
    """Rows longer than a list, under every filter with many survivors: all alike (cut inside one run of
    equal logits, at whole and half counts), two levels, sorted up and down, closed but for a few."""
    import torch
    rng = np.random.default_rng([14, rows])
    n = 40960
    kinds = [np.full(n, 2.5), np.where(np.arange(n) % 3 == 0, 1.0, -1.0), np.sort(rng.standard_normal(n) * 3),
             np.sort(rng.standard_normal(n))[::-1], np.where(rng.random(n) < 0.999, -np.inf, rng.standard_normal(n)),
             np.where(rng.random(n) < 0.5, -3e38, rng.standard_normal(n) * 0.1), rng.standard_normal(n) * 1e-20,
             np.round(rng.standard_normal(n) * 4) / 4, rng.standard_cauchy(n)]
    filters = [(1.0, 0, 0.5, 0.0), (1.0, 0, 0.25, 0.0), (1.0, 20480, 1.0, 0.0), (1.0, 5000, 0.9, 0.0), (1.0, 4097, 1.0, 0.0),
               (1.0, 0, 1 - 2.0 ** -24, 0.0), (0.7, 0, 0.9999, 0.0), (2.0, 0, 1.0, 1e-30), (1.0, 0, 0.99, 1e-6),
               (1.0, 3000, 0.999, 0.0), (1.0, 0, 1.0, 0.0), (1.0, 40959, 1.0, 0.0), (1.0, 0, 1e-30, 0.0)]
    x = torch.from_numpy(np.stack([kinds[r % len(kinds)] for r in range(rows)])).float().cuda()
    want = x.double().cpu().numpy()
    for shift in range(0, len(filters), 1 if rows < 100 else 5):
        params = records(rows, filters[shift:] + filters[:shift])
        u = np.where(rng.random(rows) < 0.3, 0.5, rng.random(rows)).astype(np.float32)
        check(run(x, params, u), want, params, u, shift)


@pytest.mark.parametrize("t", [1e-45, 1e-39, 1e-20, 1e20, 3e38])
def test_temperatures_of_long_rows(t):
    import torch
    rng = np.random.default_rng(15)
    x = torch.from_numpy(matrix(rng, 10, 20000, "normal")).float().cuda()
    x[3] *= 1e30
    x[4] = 7.0
    x[5, ::2] = -3e38
    params = records(10, [(t, 0, 0.9, 0.0), (t, 5000, 1.0, 0.0), (t, 0, 0.5, 0.0), (t, 0, 1.0, 0.5), (t, 0, 1.0, 0.0), (t, 6000, 0.99, 0.0)])
    u = rng.random(10, np.float32)
    check(run(x, params, u), x.double().cpu().numpy(), params, u, t)


def test_widest_row_and_offsets_past_32_bits():
    import torch
    rng = np.random.default_rng(10)
    n = 1 << 22
    x = torch.randn(2, n, device="cuda") * 2
    params, u = records(2, [FILTERS["default"], (1.0, 0, 0.9, 0.0)]), rng.random(2, np.float32)
    check(run(x, params, u), x.double().cpu().numpy(), params, u)
    ld = (1 << 31) + 3
    wide = torch.empty(2 * ld + 5000, dtype=torch.float16, device="cuda")
    y = wide.as_strided((3, 4999), (ld, 1))
    y.copy_(torch.from_numpy(matrix(rng, 3, 4999, "normal")))
    params, u = records(3, [FILTERS["all"]]), rng.random(3, np.float32)
    check(run(y, params, u), y.double().cpu().numpy(), params, u)


def test_streams_graphs_and_optional_outputs():
    """Calls on two streams at once, and a call captured once and replayed on new inputs, beside an
    eager call; every optional output may be absent."""
    import torch
    rng = np.random.default_rng(11)
    rows, n = 64, 40000
    params, dev = records(rows, list(FILTERS.values())), torch.device("cuda")
    tp = torch.from_numpy(params.view(np.uint8)).to(dev)
    xs = [torch.from_numpy(matrix(rng, rows, n, k)).float().to(dev) for k in ("normal", "flat")]
    us = [rng.random(rows, np.float32) for _ in xs]
    tu = [torch.from_numpy(u).to(dev) for u in us]
    want = [[draw_row(r, *p, w) for r, p, w in zip(x.double().cpu().numpy(), params, u)] for x, u in zip(xs, us)]
    toks = [torch.zeros(rows, dtype=torch.int32, device=dev) for _ in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(3):
        for x, u, t, s in zip(xs, tu, toks, streams):
            lrs.BatchSampler.draw_device(x, tp, u, t, stream=s.cuda_stream)
    torch.cuda.synchronize()
    for t, w in zip(toks, want):
        assert list(t.cpu().numpy()) == [v[1] for v in w]
    sx, su, st = xs[0].clone(), tu[0].clone(), torch.zeros(rows, dtype=torch.int32, device=dev)
    sp = torch.zeros(rows, device=dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lrs.BatchSampler.draw_device(sx, tp, su, st, probs=sp)
    for i in (1, 0):
        sx.copy_(xs[i])
        su.copy_(tu[i])
        graph.replay()
        lrs.BatchSampler.draw_device(xs[1 - i], tp, tu[1 - i], toks[1 - i])
        torch.cuda.synchronize()
        assert list(st.cpu().numpy()) == [v[1] for v in want[i]]
        assert list(toks[1 - i].cpu().numpy()) == [v[1] for v in want[1 - i]]
        assert np.allclose(sp.cpu().numpy(), [v[2] for v in want[i]], rtol=2.0 ** -23, atol=0)


def test_the_same_call_gives_the_same_bits():
    import torch
    rng = np.random.default_rng(12)
    x = torch.from_numpy(matrix(rng, 300, 30011, "flat")).float().cuda()
    params, u = records(300, list(FILTERS.values())), rng.random(300, np.float32)
    a = run(x, params, u)
    for _ in range(3):
        b = run(x, params, u)
        assert all(np.array_equal(p.view(np.uint32), q.view(np.uint32)) for p, q in zip(a, b))
