"""GPU tests of how the decode step's operators are called: what their statuses report."""
import ctypes

import numpy as np
import pytest

import lrs

pytestmark = pytest.mark.gpu


def test_an_earlier_calls_error_is_not_the_launches():
    """A context that could not be allocated leaves an error behind in the thread; the operators' launches
    after it are sound and say so."""
    import torch
    L, h = lrs.lib(), ctypes.c_void_p()
    x = torch.ones(130, 256, device="cuda")

    def fail():
        assert L.lrs_create(0, 1 << 16, 1000, 0xFFFFFFFF, ctypes.byref(h)) == lrs.LRS_E_NOMEM and h.value is None
    codes, scales = lrs.empty_codes(130, 256, "cuda"), torch.zeros(2, 130, device="cuda")
    fail()
    lrs.quantize_rows(x, codes, scales)
    weight, weights = lrs.empty_codes(130, 256, "cuda"), torch.zeros(2, 2, device="cuda")
    fail()
    lrs.quantize_blocks(x, weight, weights)
    out = torch.zeros(130, 130, device="cuda")
    fail()
    lrs.fp8_logits(codes, scales, weight, weights, out)
    p = torch.from_numpy(np.array([(0.0, 0, 1.0, 0.0)] * 130, lrs.DRAW_PARAMS_DTYPE).view(np.uint8)).cuda()
    tok = torch.full((130,), -5, dtype=torch.int32, device="cuda")
    fail()
    lrs.BatchSampler.draw_device(out, p, torch.zeros(130, device="cuda"), tok)
    torch.cuda.synchronize()
    # (448 * (1 / 448) rounded once is 1 but for a last bit, and so is the sum of 256 of its squares)
    assert ((out - 256).abs() <= 256 * 2.0 ** -22).all() and (tok == 0).all()
