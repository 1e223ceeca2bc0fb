"""GPU tests of the 8-bit head: lrs_quantize_rows and lrs_quantize_blocks bit for bit against the
three f32 operations that define them, and lrs_fp8_logits against the product in 64 bits.

Tolerance of the product: products of e4m3 values are exact in f32; a block's 128 of them are added in
f32 in an order of the hardware's, each addition off by at most one step (2^-23, rounded or cut); the
scaling takes two roundings and the sum over B blocks B more, half a step each.  So a value is within
((128 + 2 + B) 2^-23) of the sum of its terms' magnitudes, and the output's rounding adds
eps(out) / 2 of the value."""
import numpy as np
import pytest

import lrs
from draw_ref import blocks_of, draw_row, e4m3_values, head

pytestmark = pytest.mark.gpu


def types():
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def plain_codes(x, tall):
    """The definition in torch's f32 operations on the CPU: codes (uint8) and scales."""
    import torch
    rows, k = x.shape
    kb, rb = -(-k // 128), -(-rows // 128)
    y = torch.nn.functional.pad(x.float(), (0, kb * 128 - k, 0, rb * 128 - rows if tall else 0))
    y = y.view(rb, 128, kb, 128) if tall else y.view(rows, 1, kb, 128)
    s = (y.abs().amax(dim=(1, 3)) / 448.0).clamp_min(2.0 ** -126)
    c = (y * (1.0 / s)[:, None, :, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    return c.reshape(-1, kb * 128)[:rows, :k], s if tall else s.t()


def quantize(x, tall, ldq=None, ld_scale=0):
    """Codes and scales of the library, in buffers whose padding must stay as it was."""
    import torch
    rows, k = x.shape
    a, b = (-(-rows // 128), -(-k // 128)) if tall else (-(-k // 128), rows)
    qbuf = torch.full((rows, ldq or (k + 15) // 16 * 16), 0x55, dtype=torch.uint8, device="cuda")
    sbuf = torch.full((a, b + ld_scale), -3.0, device="cuda")
    (lrs.quantize_blocks if tall else lrs.quantize_rows)(x, qbuf[:, :k], sbuf[:, :b])
    torch.cuda.synchronize()
    assert (qbuf[:, k:] == 0x55).all() and (sbuf[:, b:] == -3.0).all()
    return qbuf[:, :k], sbuf[:, :b]


@pytest.mark.parametrize("tall", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,k,offset,pad,ldq,lds", [
    (1, 1, 0, 0, None, 0), (1, 1024, 0, 0, None, 0), (3, 127, 0, 0, None, 2), (7, 128, 0, 0, 128, 0),
    (8, 129, 1, 0, 129, 0), (9, 1000, 3, 5, 1003, 1), (127, 384, 0, 8, None, 0), (128, 256, 0, 0, None, 0),
    (130, 300, 0, 4, None, 3), (300, 77, 2, 1, 80, 0), (1029, 520, 0, 0, None, 0),
])
def test_codes_and_scales(tall, dtype, rows, k, offset, pad, ldq, lds):
    import torch
    g = torch.Generator().manual_seed(rows * k + offset)
    x = torch.randn(rows, k, generator=g) * torch.exp(2 * torch.randn(rows, 1, generator=g))
    if rows > 2:
        x[rows // 2] = 0
    flat = torch.full((offset + rows * (k + pad),), float("nan"), dtype=types()[dtype], device="cuda")
    v = flat[offset:].view(rows, k + pad)[:, :k]
    v.copy_(x)
    q, s = quantize(v, tall, ldq, lds)
    want_q, want_s = plain_codes(v.cpu(), tall)
    assert torch.equal(s.cpu().contiguous().view(torch.int32), want_s.contiguous().view(torch.int32))
    assert torch.equal(q.cpu() & 127, want_q & 127) and torch.equal((q.cpu() - want_q) & 127, torch.zeros_like(want_q))
    # and against 64 bits: every value within half a step of its code, the step of e4m3 at that size
    val = e4m3_values()[q.cpu().numpy()]
    big = blocks_of(v.double().cpu().numpy(), 128 if tall else 1)
    scale = np.maximum(big / 448, 2.0 ** -126)
    at = np.repeat(np.repeat(scale, 128, axis=1)[:, :k], 128 if tall else 1, axis=0)[:rows]
    real = v.double().cpu().numpy() / at
    step = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(real), 2.0 ** -6))) - 3)
    assert (np.abs(val - real) <= step / 2 + np.abs(real) * 2.0 ** -22).all()


@pytest.mark.parametrize("tall", [False, True])
def test_subnormal_zero_and_non_finite_blocks(tall):
    import torch
    x = torch.zeros(256, 512)
    x[0, :128] = 1e-42
    x[1, 128:256] = 2.0 ** -126
    x[2, 300] = 3e38
    x[200, 5] = float("nan")
    x[201, 130] = float("inf")
    x[202, 400] = -float("inf")
    q, s = quantize(x.cuda(), tall)
    want_q, want_s = plain_codes(x, tall)
    q, s = q.cpu(), s.cpu()
    assert torch.equal(s.isnan(), want_s.isnan()) and torch.equal(s.nan_to_num(7, 8, 9), want_s.nan_to_num(7, 8, 9))
    v = e4m3_values()
    assert np.array_equal(v[q.numpy()], v[want_q.numpy()], equal_nan=True)


def codes(rng, rows, k):
    c = rng.integers(0, 256, (rows, k)).astype(np.uint8)
    c[(c & 127) == 127] = 0x38  # (no NaN codes)
    return c


def product(a, sa, w, sw, dtype, ldo=None, offset=0):
    """Through the library, on padded buffers; sa (blocks, rows)."""
    import torch

    def put(c):
        t = lrs.empty_codes(c.shape[0], c.shape[1], "cuda")
        t.view(torch.uint8).copy_(torch.from_numpy(c))
        return t
    rows, n = a.shape[0], w.shape[0]
    ldo = ldo or n
    buf = torch.full((offset + rows * ldo + 9,), -9.0, dtype=types()[dtype], device="cuda")
    out = buf[offset:offset + rows * ldo].view(rows, ldo)[:, :n]
    lrs.fp8_logits(put(a), torch.from_numpy(sa).cuda(), put(w), torch.from_numpy(sw).cuda(), out)
    torch.cuda.synchronize()
    rest = buf.clone()
    rest[offset:offset + rows * ldo].view(rows, ldo)[:, :n] = -9.0
    assert (rest == -9.0).all()
    return out.double().cpu().numpy()


def within(got, a, sa, w, sw, dtype, label):
    import torch
    v = e4m3_values()
    want, size = head(v[a], sa.T, v[w], sw)
    blocks = sa.shape[0]
    tol = size * ((130 + blocks) * 2.0 ** -23) + np.abs(want) * (torch.finfo(types()[dtype]).eps / 2) + torch.finfo(types()[dtype]).tiny
    worst = (np.abs(got - want) / tol).max()
    assert worst <= 1, (label, worst)


def scales(rng, a, b):
    return np.exp(rng.standard_normal((a, b))).astype(np.float32) * np.float32(2.0 ** -10)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,n,k", [
    (1, 1, 1), (1, 128, 128), (1, 1000, 1024), (2, 129, 127), (3, 300, 129), (15, 127, 500), (16, 256, 256),
    (17, 1031, 384), (33, 640, 1000), (64, 777, 2048), (65, 128, 130), (127, 511, 640), (128, 384, 96),
    (129, 1030, 257), (200, 300, 16), (256, 512, 512), (257, 900, 1100), (700, 1290, 260),
])
def test_product(dtype, rows, n, k):
    rng = np.random.default_rng([rows, n, k])
    a, w = codes(rng, rows, k), codes(rng, n, k)
    sa, sw = scales(rng, -(-k // 128), rows), scales(rng, -(-n // 128), -(-k // 128))
    within(product(a, sa, w, sw, dtype), a, sa, w, sw, dtype, (rows, n, k))


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("rows,n,k,ldo,offset", [(5, 333, 200, 340, 0), (5, 333, 200, 333, 1), (40, 1001, 130, 1003, 3), (300, 257, 384, 260, 2)])
def test_product_strides(dtype, rows, n, k, ldo, offset):
    rng = np.random.default_rng([rows, n, k, ldo])
    a, w = codes(rng, rows, k), codes(rng, n, k)
    sa, sw = scales(rng, -(-k // 128), rows), scales(rng, -(-n // 128), -(-k // 128))
    within(product(a, sa, w, sw, dtype, ldo, offset), a, sa, w, sw, dtype, (rows, n, k, ldo))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,n,k,ldo,offset", [(65, 64, 100, 65, 0), (129, 256, 128, 259, 7), (130, 333, 200, 333, 1),
                                                 (130, 333, 200, 338, 6), (131, 515, 140, 517, 5), (97, 640, 130, 644, 4), (200, 1281, 40, 1281, 3)])
def test_product_rows_of_every_alignment(dtype, rows, n, k, ldo, offset):
    """Row starts that walk through the 16-byte boundaries, whole and ragged runs of columns."""
    rng = np.random.default_rng([rows, n, k, ldo, offset])
    a, w = codes(rng, rows, k), codes(rng, n, k)
    sa, sw = scales(rng, -(-k // 128), rows), scales(rng, -(-n // 128), -(-k // 128))
    within(product(a, sa, w, sw, dtype, ldo, offset), a, sa, w, sw, dtype, (rows, n, k, ldo, offset))


def test_product_of_exact_sums_is_exact():
    """Small whole numbers and scales of 1: every partial sum is exact in f32, so the product is too,
    whatever the order; each output then names its row, column and every block's part in it."""
    rng = np.random.default_rng(4)
    v = e4m3_values()
    small = np.array([c for c in range(256) if v[c] == np.round(v[c]) and abs(v[c]) <= 8], np.uint8)
    for rows, n, k in ((1, 151936, 1024), (70, 2000, 1152), (300, 700, 4096)):
        a, w = rng.choice(small, (rows, k)), rng.choice(small, (n, k))
        sa, sw = np.ones((-(-k // 128), rows), np.float32), np.ones((-(-n // 128), -(-k // 128)), np.float32)
        sa *= (2.0 ** (np.arange(rows) % 4))[None].astype(np.float32)
        sw *= (2.0 ** (np.arange(len(sw)) % 3))[:, None].astype(np.float32)
        want, _ = head(v[a], sa.T, v[w], sw)
        assert np.abs(want).max() < 2 ** 24
        assert np.array_equal(product(a, sa, w, sw, "f32"), want), (rows, n, k)


def test_a_bad_hidden_state_spoils_its_row_alone():
    import torch
    rng = np.random.default_rng(5)
    h = torch.from_numpy(rng.standard_normal((6, 400))).float().cuda()
    h[1, 3], h[4, 399] = float("nan"), float("inf")
    lm = lrs.LmHead(torch.from_numpy(rng.standard_normal((900, 400))).bfloat16().cuda())
    y = lm.logits(h)
    bad = torch.tensor([False, True, False, False, True, False], device="cuda")
    assert y[bad].isnan().all() and y[~bad].isfinite().all()
    p = torch.zeros(6, 4, dtype=torch.int32, device="cuda")
    p[:, 0] = torch.ones(6, device="cuda").view(torch.int32)
    p[:, 2] = torch.ones(6, device="cuda").view(torch.int32)
    tok, st = torch.zeros(6, dtype=torch.int32, device="cuda"), torch.zeros(6, dtype=torch.int32, device="cuda")
    lrs.BatchSampler.draw_hidden(lm, h, p, torch.full((6,), 0.5, device="cuda"), tok, status=st)
    assert st.tolist() == [0, -2, 0, 0, -2, 0] and tok[bad].tolist() == [-1, -1]


@pytest.mark.parametrize("rows,n,k,dtype", [(1, 5000, 256, "f32"), (19, 3011, 400, "bf16"), (150, 1999, 300, "f16")])
def test_a_decode_step(rows, n, k, dtype):
    """Hidden states to tokens as a serving loop runs it: quantise, multiply, draw, append, on the head's
    own logits; captured into a graph and replayed on new hidden states."""
    import torch
    rng = np.random.default_rng([rows, n])
    dev = torch.device("cuda")
    w = torch.from_numpy(rng.standard_normal((n, k)) * 3 / k ** 0.5).bfloat16().to(dev)
    lm = lrs.LmHead(w)
    params = np.zeros(rows, lrs.DRAW_PARAMS_DTYPE)
    for r in range(rows):
        params[r] = [(0.8, 40, 0.95, 0.0), (1.0, 0, 0.9, 0.0), (1.1, 0, 1.0, 0.02), (0.0, 0, 1.0, 0.0)][r % 4]
    tp = torch.from_numpy(params.view(np.uint8)).to(dev)
    h, u = torch.zeros(rows, k, device=dev, dtype=torch.bfloat16), torch.zeros(rows, device=dev)
    tok, st = torch.zeros(rows, dtype=torch.int32, device=dev), torch.zeros(rows, dtype=torch.int32, device=dev)
    prob = torch.zeros(rows, device=dev)
    hist, hist_len = torch.zeros(rows, 16, dtype=torch.int32, device=dev), torch.zeros(rows, dtype=torch.int32, device=dev)

    def step():
        y = lrs.BatchSampler.draw_hidden(lm, h, tp, u, tok, probs=prob, status=st, dtype=types()[dtype])
        lrs.BatchSampler.history_append(tok, hist, hist_len, status=st)
        return y
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    hist_len.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step()
    drawn = []
    for _ in range(3):
        h.copy_(torch.from_numpy(rng.standard_normal((rows, k))))
        uu = rng.random(rows, np.float32)
        u.copy_(torch.from_numpy(uu))
        graph.replay()
        torch.cuda.synchronize()
        drawn.append(tok.tolist())
        rowsf = y.double().cpu().numpy()
        # the logits: codes of both sides by the definition, then the product in 64 bits
        (qa, sa), (qw, sw) = plain_codes(h.cpu(), False), plain_codes(w.cpu(), True)
        v = e4m3_values()
        want, size = head(v[qa.numpy()], sa.t().numpy(), v[qw.numpy()], sw.numpy())
        eps = torch.finfo(types()[dtype]).eps
        assert (np.abs(rowsf - want) <= size * (133 * 2.0 ** -23) + np.abs(want) * eps / 2 + 1e-6).all()
        for r in range(rows):
            status, token, p, _ = draw_row(rowsf[r], *params[r], uu[r])
            assert (st[r].item(), tok[r].item()) == (status, token), r
            assert abs(prob[r].item() - p) <= p * 2.0 ** -23
    assert hist_len.tolist() == [3] * rows
    assert hist[:, :3].t().tolist() == drawn


def test_the_exact_sampler_on_the_heads_logits():
    """sample_hidden: the exact sampler on the head's logits gives what sample_device gives on them, and a
    vocabulary-sharded rank that holds the whole head gives the same tokens."""
    import torch
    from lrs import workloads as W
    from lrs.sharded import VocabShardedSampler
    rng = np.random.default_rng(13)
    rows, n, k = 12, 4000, 320
    dev = torch.device("cuda")
    lm = lrs.LmHead(torch.from_numpy(rng.standard_normal((n, k)) * 0.2).half().to(dev))
    h = torch.from_numpy(rng.standard_normal((rows, k))).half().to(dev)
    p = np.zeros(rows, W.PARAMS_DTYPE)
    p["temperature"], p["top_k"], p["top_p"], p["repetition_penalty"], p["repeat_last_n"] = 0.8, 40, 0.95, 1.0, 64
    tp = torch.from_numpy(p.view(np.uint8)).to(dev)
    states = [torch.arange(1, 2 * rows, 2, dtype=torch.int64, device=dev) for _ in range(3)]
    toks = [torch.zeros(rows, dtype=torch.int32, device=dev) for _ in range(3)]
    bs = lrs.BatchSampler(rows, n)
    y = bs.sample_hidden(lm, h, tp, states[0], toks[0])
    bs.sample_device(y, tp, states[1], toks[1])
    vs = VocabShardedSampler(rows, n)
    vs.sample_hidden(lm, h, tp, states[2], toks[2])
    torch.cuda.synchronize()
    assert toks[0].tolist() == toks[1].tolist() == toks[2].tolist()
    assert states[0].tolist() == states[1].tolist() == states[2].tolist()
    bs.close()
    vs.close()
