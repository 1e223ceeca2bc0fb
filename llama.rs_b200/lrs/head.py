"""The language-model head in 8-bit floating point: the product whose rows the samplers read.

rust-llama computes it as ops::matmul over the vocabulary (src/model.rs:579-582, 733-737) on its GGML
weight formats; here the weights are e4m3 codes with one f32 scale per 128 x 128 block, laid out
once, and the hidden states are quantised per row and 128 columns in front of each product.

  quantize_rows, quantize_blocks   codes and scales (lrs_quantize_rows, lrs_quantize_blocks)
  fp8_logits                       the product of codes (lrs_fp8_logits)
  LmHead                           a head's weights, with logits(hidden)

All are asynchronous on the tensors' device: on torch's current stream there, or on `stream` (a
cudaStream_t handle of that device) where one is given.
"""
from __future__ import annotations

from .sampler import LRS_E_INVALID, SamplerError, check_kind, dtype_code, kinds, launch, lib

BLOCK = 128


def _lead(t, rows: int, cols: int, kind, what: str) -> int:
    """The leading dimension of a rows x cols tensor of contiguous rows (rows of one have none) and a kind of type
    (check_kind; None: the caller has looked)."""
    if kind and t.dtype not in kinds[kind]:
        check_kind(t, kind, what)
    step, inner = t.stride()
    if inner != 1 and cols > 1:
        raise SamplerError(LRS_E_INVALID, f"{what}: contiguous rows are needed")
    return step if rows > 1 else cols


def _matrix(t, rows: int, cols: int, kind, what: str) -> int:
    """_lead() of a tensor that has to be rows x cols."""
    if t.shape != (rows, cols):
        raise SamplerError(LRS_E_INVALID, f"{what}: a tensor of {rows} x {cols} is needed")
    return _lead(t, rows, cols, kind, what)


def _blocks(k: int) -> int:
    return (k + BLOCK - 1) // BLOCK


def _two(t, what: str):
    shape = t.shape
    if len(shape) != 2:
        raise SamplerError(LRS_E_INVALID, f"{what}: a 2-d tensor is needed")
    if (shape[0] | shape[1]) >> 32:  # (ctypes would cut them)
        raise SamplerError(LRS_E_INVALID, f"{what}: {shape[0]} x {shape[1]} is larger than 2^32 a side")
    return shape


def _quantize(call, x, codes, scales, a: int, b: int, stream) -> None:
    rows, k = x.shape
    launch(call, stream,
           (x.data_ptr(), dtype_code(x), rows, k, _lead(x, rows, k, None, "x"), codes.data_ptr(),
            _matrix(codes, rows, k, "codes", "codes"), scales.data_ptr(), _matrix(scales, a, b, "f32", "scales")),
           x, codes, scales)


def quantize_rows(x, codes, scales, stream=None) -> None:
    """x (rows, k) float32 / bfloat16 / float16 -> codes (rows, k) e4m3 (float8_e4m3fn or uint8) and
    scales (ceil(k / 128), rows) float32, one per row and 128 columns.  For lrs_fp8_logits let the
    codes start on 16-byte boundaries (see `empty_codes`)."""
    rows, k = _two(x, "x")
    _quantize(lib().lrs_quantize_rows, x, codes, scales, _blocks(k), rows, stream)


def quantize_blocks(x, codes, scales, stream=None) -> None:
    """x (rows, k) -> codes (rows, k) e4m3 and scales (ceil(rows / 128), ceil(k / 128)) float32, one per
    128 x 128 block."""
    rows, k = _two(x, "x")
    _quantize(lib().lrs_quantize_blocks, x, codes, scales, _blocks(rows), _blocks(k), stream)


def _product(a, a_scales, w, w_scales, out) -> tuple:
    rows, k = _two(a, "a")
    n, kb = _two(w, "w")[0], _blocks(k)
    return (a.data_ptr(), _lead(a, rows, k, "codes", "a"), a_scales.data_ptr(), _matrix(a_scales, kb, rows, "f32", "a_scales"),
            w.data_ptr(), _matrix(w, n, k, "codes", "w"), w_scales.data_ptr(), _matrix(w_scales, _blocks(n), kb, "f32", "w_scales"),
            rows, n, k, out.data_ptr(), dtype_code(out), _matrix(out, rows, n, None, "out"))


def fp8_logits(a, a_scales, w, w_scales, out, stream=None) -> None:
    """out (rows, n) = a (rows, k) times w (n, k) transposed, both e4m3 codes with the scales of
    quantize_rows and quantize_blocks; out is float32, bfloat16 or float16."""
    launch(lib().lrs_fp8_logits, stream, _product(a, a_scales, w, w_scales, out), a, a_scales, w, w_scales, out)


def test_wait_timeout(a, a_scales, w, w_scales, out, steps: int, bound_cycles: int, stream=None) -> None:
    """fp8_logits whose waits run out after every CTA's first `steps` steps (lrs_test_fp8_logits_timeout)."""
    launch(lib().lrs_test_fp8_logits_timeout, stream, (*_product(a, a_scales, w, w_scales, out), steps, bound_cycles),
           a, a_scales, w, w_scales, out)


def empty_codes(rows: int, k: int, device):
    """An uninitialised (rows, k) code tensor whose rows start on 16-byte boundaries."""
    import torch
    return torch.empty(rows, (k + 15) // 16 * 16, dtype=torch.float8_e4m3fn, device=device)[:, :k]


class LmHead:
    """A head's weights (vocab, k), quantised once to e4m3 with a scale per 128 x 128 block, on torch's current stream of
    their device: a product on another stream has to be ordered after that one, as any tensor's first use is."""

    def __init__(self, weight):
        import torch
        n, k = _two(weight, "weight")
        self.vocab, self.k, self.device = n, k, weight.device
        self.codes = empty_codes(n, k, weight.device)
        self.scales = torch.empty(_blocks(n), _blocks(k), dtype=torch.float32, device=weight.device)
        quantize_blocks(weight, self.codes, self.scales)

    def logits(self, hidden, out=None, dtype=None):
        """hidden (rows, k) float32 / bfloat16 / float16 -> logits (rows, vocab), into `out` or a new
        tensor of `dtype` (float32).  On torch's current stream of the head's device; the codes of
        the hidden states come from torch's allocator, so calls on several streams and captured
        calls do not share them."""
        import torch
        rows, k = _two(hidden, "hidden")
        if k != self.k:
            raise SamplerError(LRS_E_INVALID, f"hidden: {k} columns, the head has {self.k}")
        if out is None:
            out = torch.empty(rows, self.vocab, dtype=dtype or torch.float32, device=self.device)
        if rows == 0:
            return out
        with torch.cuda.device(self.device):
            codes = empty_codes(rows, k, self.device)
            scales = torch.empty(_blocks(k), rows, dtype=torch.float32, device=self.device)
            quantize_rows(hidden, codes, scales)
            fp8_logits(codes, scales, self.codes, self.scales, out)
        return out
