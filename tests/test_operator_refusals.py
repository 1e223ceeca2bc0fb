"""CPU tests of the decode step's operators: what they refuse, before any GPU work, and the plain
64-bit forms that the GPU tests compare with."""
import ctypes

import numpy as np
import pytest

import lrs
from draw_ref import draw_row, e4m3_values

P = 1 << 20  # an address that is aligned and never read: every call here is refused


def draw(**kw):
    a = dict(logits=P, dtype=0, rows=2, n=100, ld=100, params=P, uniform=P, tokens=P, probs=None, kept=None,
             status=None, stream=None)
    a.update(kw)
    return lrs.lib().lrs_draw_device(*a.values())


def quant(name="lrs_quantize_rows", **kw):
    a = dict(x=P, dtype=1, rows=4, k=200, ld_x=200, q=P, ld_q=200, scale=P, ld_scale=4, stream=None)
    a.update(kw)
    return getattr(lrs.lib(), name)(*a.values())


def logits(**kw):
    a = dict(a=P, ld_a=208, sa=P, ld_as=4, w=P, ld_w=208, sw=P, ld_ws=2, rows=4, n=300, k=200, out=P, dtype=0,
             ld_out=300, stream=None)
    a.update(kw)
    return lrs.lib().lrs_fp8_logits(*a.values())


@pytest.mark.parametrize("bad", [
    dict(dtype=3), dict(dtype=-1), dict(logits=None), dict(params=None), dict(uniform=None), dict(tokens=None),
    dict(n=0), dict(n=(1 << 22) + 1), dict(rows=(1 << 24) + 1), dict(ld=99), dict(logits=P + 2),
    dict(dtype=1, logits=P + 1), dict(params=P + 2), dict(uniform=P + 1), dict(tokens=P + 2), dict(probs=P + 3),
    dict(kept=P + 1), dict(status=P + 2),
])
def test_draw_refuses(built_lib, bad):
    assert draw(**bad) == lrs.LRS_E_INVALID
    assert lrs.lib().lrs_last_error(None).startswith(b"lrs_draw_device")


@pytest.mark.parametrize("name", ["lrs_quantize_rows", "lrs_quantize_blocks"])
@pytest.mark.parametrize("bad", [
    dict(dtype=3), dict(x=None), dict(q=None), dict(scale=None), dict(k=0), dict(k=(1 << 18) + 1, ld_x=1 << 20, ld_q=1 << 20),
    dict(rows=(1 << 24) + 1, ld_scale=1 << 25), dict(ld_x=199), dict(ld_q=199), dict(ld_scale=1), dict(x=P + 1),
    dict(scale=P + 2), dict(dtype=0, x=P + 2),
])
def test_quantize_refuses(built_lib, name, bad):
    assert quant(name, **bad) == lrs.LRS_E_INVALID
    assert lrs.lib().lrs_last_error(None).startswith(name.encode())


@pytest.mark.parametrize("bad", [
    dict(dtype=3), dict(a=None), dict(sa=None), dict(w=None), dict(sw=None), dict(out=None), dict(n=0), dict(k=0),
    dict(n=(1 << 24) + 1, ld_out=1 << 25), dict(rows=(1 << 24) + 1, ld_as=1 << 25),
    dict(k=(1 << 18) + 1, ld_a=1 << 20, ld_w=1 << 20, ld_ws=1 << 12), dict(ld_a=192), dict(ld_w=192), dict(ld_as=3),
    dict(ld_ws=1), dict(ld_out=299), dict(a=P + 8), dict(w=P + 8), dict(ld_a=216), dict(ld_w=216), dict(sa=P + 2),
    dict(sw=P + 1), dict(out=P + 2), dict(dtype=1, out=P + 1),
])
def test_logits_refuses(built_lib, bad):
    assert logits(**bad) == lrs.LRS_E_INVALID
    assert lrs.lib().lrs_last_error(None).startswith(b"lrs_fp8_logits")


def test_no_rows_is_no_work(built_lib):
    assert draw(rows=0, logits=None) == lrs.LRS_OK
    assert quant(rows=0, x=None) == lrs.LRS_OK
    assert quant("lrs_quantize_blocks", rows=0, x=None) == lrs.LRS_OK
    assert logits(rows=0, a=None) == lrs.LRS_OK


def test_python_calls_refuse_host_tensors_and_wrong_shapes(built_lib):
    import torch
    f, i = torch.zeros(2, 100), torch.zeros(2, dtype=torch.int32)
    p, u = torch.zeros(32, dtype=torch.uint8), torch.zeros(2)
    for args in ((f, p, u, i), (f[0], p, u, i), (f.t(), p, u, i), (f, p[:16], u, i), (f, p, u[:1], i),
                 (f, p, u.double(), i), (f[:, ::2], p, u, i)):
        with pytest.raises(lrs.SamplerError) as e:
            lrs.BatchSampler.draw_device(*args)
        assert e.value.code == lrs.LRS_E_INVALID
    q, s = torch.zeros(2, 100, dtype=torch.uint8), torch.zeros(1, 2)
    for args in ((f, q, s), (f, q[:, :99], s), (f, q, s.t()), (f, f, s), (f.t(), q, s)):
        for call in (lrs.quantize_rows, lrs.quantize_blocks):
            with pytest.raises(lrs.SamplerError):
                call(*args)
    with pytest.raises(lrs.SamplerError):
        lrs.fp8_logits(q, s, q, torch.zeros(1, 1), torch.zeros(2, 3))
    with pytest.raises(lrs.SamplerError):
        lrs.fp8_logits(q, s, q, torch.zeros(1, 1), torch.zeros(2, 2))


def test_record_layout_matches_header():
    assert lrs.DRAW_PARAMS_DTYPE.itemsize == 16
    assert ctypes.sizeof(ctypes.c_float) * 4 == lrs.DRAW_PARAMS_DTYPE.itemsize


def test_plain_draw_follows_its_definition():
    x = np.log(np.array([0.1, 0.4, 0.3, 0.2]))
    assert draw_row(x, 1, 0, 1, 0, 0.05)[1:] == (0, pytest.approx(0.1), 4)
    assert draw_row(x, 1, 0, 1, 0, 0.11)[1] == 1
    assert draw_row(x, 1, 2, 1, 0, 0.6)[1:] == (2, pytest.approx(3 / 7), 2)
    assert draw_row(x, 1, 0, 0.65, 0, 0.99)[1:] == (2, pytest.approx(3 / 7), 2)
    assert draw_row(x, 1, 0, 1, 0.4, 0.99)[1:] == (3, pytest.approx(2 / 9), 3)
    assert draw_row(np.zeros(5), 1, 3, 1, 0, 0.9)[1:] == (2, pytest.approx(1 / 3), 3)
    assert draw_row(x, 0, 0, 1, 0, 0.9) == (0, 1, 1.0, 1)


def test_e4m3_values_are_torchs():
    import torch
    v = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(v, e4m3_values(), equal_nan=True)
