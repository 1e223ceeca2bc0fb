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


@pytest.mark.parametrize("rows,tile_r,tile_v", [(5, 16, 128), (64, 64, 128), (300, 128, 256)])
@pytest.mark.parametrize("steps", [0, 1, 2])
def test_the_products_waits_run_out_and_the_launch_ends(rows, tile_r, tile_v, steps):
    """Copies that never come (lrs_test_fp8_logits_timeout: bounds of 20 million cycles, about 10 ms; no copy in
    flight): the tiles that wait for them are NaN, those whose two steps had come are right, nothing is written
    beside them, and the next call is sound."""
    import torch
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    k, row_tiles = 256, -(-rows // tile_r)
    n = -(-(sms + 37) // row_tiles) * tile_v - 5  # (37 CTAs or more have a second tile)
    g = torch.Generator(device="cuda").manual_seed(rows)
    whole = lambda *shape: torch.randint(-4, 5, shape, generator=g, device="cuda").float()  # (e4m3 holds them, every sum is exact)
    a, w = lrs.empty_codes(rows, k, "cuda"), lrs.empty_codes(n, k, "cuda")
    x, y = whole(rows, k), whole(n, k)
    a.copy_(x)
    w.copy_(y)
    sa, sw = torch.ones(2, rows, device="cuda"), torch.ones(-(-n // 128), 2, device="cuda")
    want = (x.double() @ y.double().t()).float()
    buf = torch.full((rows, n + 3), -9.0, device="cuda")
    lrs.head.test_wait_timeout(a, sa, w, sw, buf[:, :n], steps, 20_000_000)
    torch.cuda.synchronize()
    tile = torch.arange(n, device="cuda") // tile_v * row_tiles + (torch.arange(rows, device="cuda") // tile_r)[:, None]
    right = (tile < sms) & (steps == 2)
    out = buf[:, :n]
    assert torch.equal(out[right], want[right]) and out[~right].isnan().all() and (buf[:, n:] == -9.0).all()
    assert (~right).any()
    lrs.fp8_logits(a, sa, w, sw, out)
    torch.cuda.synchronize()
    assert torch.equal(out, want)
