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

from .sampler import LRS_E_INVALID, SamplerError, _check, _Launch, dtype_code, lib

BLOCK = 128


def _matrix(t, what: str):
    """A 2-d CUDA tensor of contiguous rows: its leading dimension (rows of one have none)."""
    if t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1):
        raise SamplerError(LRS_E_INVALID, f"{what}: a 2-d tensor with contiguous rows is needed")
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _codes(t, rows: int, k: int, what: str):
    if t.element_size() != 1 or tuple(t.shape) != (rows, k):
        raise SamplerError(LRS_E_INVALID, f"{what}: codes are 8-bit tensors of {rows} x {k}")
    return _matrix(t, what)


def _scales(t, a: int, b: int, what: str):
    if dtype_code(t) != 0 or tuple(t.shape) != (a, b):
        raise SamplerError(LRS_E_INVALID, f"{what}: scales are a float32 tensor of {a} x {b}")
    return _matrix(t, what)


def _blocks(k: int) -> int:
    return (k + BLOCK - 1) // BLOCK


def quantize_rows(x, codes, scales, stream=None) -> None:
    """x (rows, k) float32 / bfloat16 / float16 -> codes (rows, k) e4m3 (float8_e4m3fn or uint8) and
    scales (ceil(k / 128), rows) float32, one per row and 128 columns.  For lrs_fp8_logits let the
    codes start on 16-byte boundaries (see `empty_codes`)."""
    rows, k = x.shape
    ld, ldq, lds = _matrix(x, "x"), _codes(codes, rows, k, "codes"), _scales(scales, _blocks(k), rows, "scales")
    with _Launch(stream, x, codes, scales) as s:
        _check(lib().lrs_quantize_rows(x.data_ptr(), dtype_code(x), rows, k, ld, codes.data_ptr(), ldq,
                                       scales.data_ptr(), max(lds, rows), s))


def quantize_blocks(x, codes, scales, stream=None) -> None:
    """x (rows, k) -> codes (rows, k) e4m3 and scales (ceil(rows / 128), ceil(k / 128)) float32, one per
    128 x 128 block."""
    rows, k = x.shape
    kb = _blocks(k)
    ld, ldq, lds = _matrix(x, "x"), _codes(codes, rows, k, "codes"), _scales(scales, _blocks(rows), kb, "scales")
    with _Launch(stream, x, codes, scales) as s:
        _check(lib().lrs_quantize_blocks(x.data_ptr(), dtype_code(x), rows, k, ld, codes.data_ptr(), ldq,
                                         scales.data_ptr(), max(lds, kb), s))


def fp8_logits(a, a_scales, w, w_scales, out, stream=None) -> None:
    """out (rows, n) = a (rows, k) times w (n, k) transposed, both e4m3 codes with the scales of
    quantize_rows and quantize_blocks; out is float32, bfloat16 or float16."""
    rows, k = a.shape
    n = w.shape[0]
    lda, ldw = _codes(a, rows, k, "a"), _codes(w, n, k, "w")
    kb = _blocks(k)
    ldas, ldws = _scales(a_scales, kb, rows, "a_scales"), _scales(w_scales, _blocks(n), kb, "w_scales")
    if tuple(out.shape) != (rows, n):
        raise SamplerError(LRS_E_INVALID, f"out: a tensor of {rows} x {n} is needed")
    ldo = _matrix(out, "out")
    with _Launch(stream, a, a_scales, w, w_scales, out) as s:
        _check(lib().lrs_fp8_logits(a.data_ptr(), lda, a_scales.data_ptr(), max(ldas, rows), w.data_ptr(), ldw,
                                    w_scales.data_ptr(), max(ldws, kb), rows, n, k, out.data_ptr(), dtype_code(out),
                                    ldo, s))


def empty_codes(rows: int, k: int, device):
    """An uninitialised (rows, k) code tensor whose rows start on 16-byte boundaries."""
    import torch
    return torch.empty(rows, (k + 15) // 16 * 16, dtype=torch.float8_e4m3fn, device=device)[:, :k]


class LmHead:
    """A head's weights (vocab, k), quantised once to e4m3 with a scale per 128 x 128 block."""

    def __init__(self, weight):
        import torch
        n, k = weight.shape
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
        rows, k = hidden.shape
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
