"""CPU tests of what the decode step's operators check, each refusal by its message (a refusal for another
reason does not count)."""
import ctypes

import pytest

import lrs

P = 1 << 20  # an address that is aligned and never read: every call here is refused


def test_the_test_of_the_products_waits_checks_its_arguments(built_lib):
    call, args = lrs.lib().lrs_test_fp8_logits_timeout, [P, 208, P, 4, P, 208, P, 2, 4, 300, 200, P, 0, 300]
    assert call(*args, 1, 0, None) == lrs.LRS_E_INVALID
    assert lrs.lib().lrs_last_error(None) == b"lrs_test_fp8_logits_timeout: bound is 0"
    assert call(*args[:-1], 299, 1, 1000, None) == lrs.LRS_E_INVALID
    assert b"leading dimension" in lrs.lib().lrs_last_error(None)
