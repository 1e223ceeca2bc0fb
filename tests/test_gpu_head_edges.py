"""GPU tests of the 8-bit head beside test_gpu_head.py: codes compared as whole bytes, and the product on both
sides of the border between its forms.  Tolerances are that file's."""
import numpy as np
import pytest

from test_gpu_head import codes, plain_codes, product, quantize, scales, types, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tall", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,k", [(1, 1024), (9, 1000), (130, 300), (1029, 520)])
def test_codes_are_the_definitions_bytes(tall, dtype, rows, k):
    """Signs too: what rounds to 0 from below is -0, as e4m3 has it."""
    import torch
    g = torch.Generator().manual_seed(rows + k)
    x = torch.randn(rows, k, generator=g) * torch.exp(3 * torch.randn(rows, k, generator=g))
    x = x.clamp(-6e4, 6e4).to(types()[dtype])  # (finite in every type: a NaN's code may have either sign)
    q, s = quantize(x.cuda(), tall)
    want_q, want_s = plain_codes(x, tall)
    assert torch.equal(q.cpu(), want_q)
    assert torch.equal(s.cpu().contiguous().view(torch.int32), want_s.contiguous().view(torch.int32))
    assert (want_q == 0x80).any() and (want_q >= 0x81).any()  # (-0 and negative ones among them)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows", [31, 32, 33, 47, 48, 49, 63, 64, 65])
@pytest.mark.parametrize("n,k,ldo,offset", [(640, 300, 640, 0), (515, 300, 520, 0), (515, 300, 517, 3)])
def test_product_around_the_forms_border(dtype, rows, n, k, ldo, offset):
    rng = np.random.default_rng([rows, n, k, ldo])
    a, w = codes(rng, rows, k), codes(rng, n, k)
    sa, sw = scales(rng, -(-k // 128), rows), scales(rng, -(-n // 128), -(-k // 128))
    within(product(a, sa, w, sw, dtype, ldo, offset), a, sa, w, sw, dtype, (rows, n, k, ldo, offset))
