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


def refused(message, call, *args, **kw):
    with pytest.raises(lrs.SamplerError, match=message) as e:
        call(*args, **kw)
    assert e.value.code == lrs.LRS_E_INVALID


def draw_args(rows=2, n=100, **kw):
    """draw_device's arguments, right but for lying on the CPU."""
    import torch
    a = dict(logits=torch.zeros(rows, n), params=torch.zeros(16 * rows, dtype=torch.uint8), uniform=torch.zeros(rows),
             tokens=torch.zeros(rows, dtype=torch.int32), probs=torch.zeros(rows), kept=torch.zeros(rows, dtype=torch.int32),
             status=torch.zeros(rows, dtype=torch.int32))
    a.update(kw)
    return a


def product_args(rows=3, n=300, k=200):
    import torch
    return dict(a=lrs.empty_codes(rows, k, "cpu"), a_scales=torch.zeros(2, rows), w=lrs.empty_codes(n, k, "cpu"),
                w_scales=torch.zeros(3, 2), out=torch.zeros(rows, n))


def test_calls_on_the_cpu_get_as_far_as_the_device(built_lib):
    """What the refusals below differ from."""
    import torch
    refused("CUDA tensors are needed", lrs.BatchSampler.draw_device, **draw_args())
    refused("CUDA tensors are needed", lrs.BatchSampler.draw_device, **draw_args(tokens=torch.zeros(2, dtype=torch.uint32)))
    refused("CUDA tensors are needed", lrs.fp8_logits, **product_args())
    for call, scales in ((lrs.quantize_rows, (2, 3)), (lrs.quantize_blocks, (1, 2))):
        for codes in (torch.zeros(3, 200, dtype=torch.uint8), lrs.empty_codes(3, 200, "cpu")):
            refused("CUDA tensors are needed", call, torch.zeros(3, 200), codes, torch.zeros(scales))


@pytest.mark.parametrize("name,dtype", [("uniform", "int32"), ("uniform", "float64"), ("tokens", "float32"), ("tokens", "int64"),
                                        ("probs", "int32"), ("probs", "bfloat16"), ("kept", "float32"), ("status", "int16")])
def test_a_draws_buffers_have_the_types_that_they_are_read_as(built_lib, name, dtype):
    import torch
    bad = torch.zeros(4, dtype=getattr(torch, dtype))
    refused(f"{name}: torch.{dtype}, ", lrs.BatchSampler.draw_device, rows=2, **draw_args(**{name: bad}))


@pytest.mark.parametrize("dtype", ["float8_e5m2", "int8", "bool", "float32"])
def test_codes_are_e4m3(built_lib, dtype):
    import torch
    bad = lambda *shape: torch.zeros(shape, dtype=getattr(torch, dtype))
    message = f"torch.{dtype}, float8_e4m3fn or uint8 is needed"
    refused("codes: " + message, lrs.quantize_rows, torch.zeros(3, 200), bad(3, 200), torch.zeros(2, 3))
    refused("codes: " + message, lrs.quantize_blocks, torch.zeros(3, 200), bad(3, 200), torch.zeros(1, 2))
    refused("a: " + message, lrs.fp8_logits, **{**product_args(), "a": bad(3, 208)[:, :200]})
    refused("w: " + message, lrs.fp8_logits, **{**product_args(), "w": bad(300, 208)[:, :200]})


@pytest.mark.parametrize("dtype", ["int32", "float64", "bfloat16"])
def test_scales_are_f32(built_lib, dtype):
    import torch
    bad = lambda *shape: torch.zeros(shape, dtype=getattr(torch, dtype))
    message = f"scales: torch.{dtype}, float32 is needed"
    refused(message, lrs.quantize_rows, torch.zeros(3, 200), lrs.empty_codes(3, 200, "cpu"), bad(2, 3))
    refused(message, lrs.quantize_blocks, torch.zeros(3, 200), lrs.empty_codes(3, 200, "cpu"), bad(1, 2))
    refused("a_" + message, lrs.fp8_logits, **{**product_args(), "a_scales": bad(2, 3)})
    refused("w_" + message, lrs.fp8_logits, **{**product_args(), "w_scales": bad(3, 2)})


def test_shapes_and_strides_are_named_where_they_are_wrong(built_lib):
    import torch
    f, z = torch.zeros, lambda *s: torch.zeros(s, dtype=torch.uint8)
    draw = lrs.BatchSampler.draw_device
    refused("logits: a 2-d tensor", draw, **draw_args(logits=f(200)))
    refused("contiguous rows", draw, **draw_args(logits=f(100, 2).t()))
    refused("contiguous rows", draw, **draw_args(logits=f(2, 200)[:, ::2]))
    refused("fewer than 2 rows", draw, **draw_args(params=z(31)))
    refused("parameters are not contiguous", draw, **draw_args(params=f(2, 8)[:, ::2]))
    refused("uniform: not 2 values", draw, **draw_args(uniform=f(1)))
    refused("kept: not 2 values", draw, **draw_args(kept=torch.zeros(4, dtype=torch.int32)[::2]))
    refused("float64: float32, bfloat16 or float16", draw, **draw_args(logits=f(2, 100).double()))
    refused("x: a 2-d tensor", lrs.quantize_rows, f(200), z(1, 200), f(2, 1))
    refused("codes: a tensor of 3 x 200", lrs.quantize_rows, f(3, 200), z(3, 199), f(2, 3))
    refused("scales: a tensor of 2 x 3", lrs.quantize_rows, f(3, 200), z(3, 200), f(3, 2))
    refused("scales: a tensor of 1 x 2", lrs.quantize_blocks, f(3, 200), z(3, 200), f(2, 3))
    refused("x: contiguous rows", lrs.quantize_blocks, f(200, 3).t(), z(3, 200), f(1, 2))
    refused("float64: float32, bfloat16 or float16", lrs.quantize_rows, f(3, 200).double(), z(3, 200), f(2, 3))
    refused("w: a tensor of 300 x 200", lrs.fp8_logits, **{**product_args(), "w": z(300, 199)})
    refused("w_scales: a tensor of 3 x 2", lrs.fp8_logits, **{**product_args(), "w_scales": f(2, 3)})
    refused("out: a tensor of 3 x 300", lrs.fp8_logits, **{**product_args(), "out": f(3, 301)})
    refused("out: contiguous rows", lrs.fp8_logits, **{**product_args(), "out": f(300, 3).t()})


def test_a_leading_dimension_stays_within_the_tensor(built_lib):
    import torch
    draw, padded = lrs.BatchSampler.draw_device, torch.zeros(4, 128)[:, :100]
    for rows, kw in ((4, dict(ld=129)), (4, dict(ld=1 << 40)), (4, dict(ld=-128)), (1, dict(ld=-1)), (2, dict(ld=385, n=100)),
                     (5, dict()), (5, dict(ld=128)), (4, dict(ld=100)), (4, dict(n=101)), (4, dict(n=-1)),
                     (4, dict(n=(1 << 32) + 5)), (-1, dict()), (-(1 << 32) + 4, dict())):
        if (rows, kw) == (4, dict(ld=100)):  # (rows closer together than the tensor's are within it)
            refused("CUDA tensors are needed", draw, **draw_args(4, logits=padded), rows=rows, **kw)
            continue
        refused("draw_device: ", draw, **draw_args(8, logits=padded), rows=rows, **kw)
    # what the last row reaches, and row 0 for every row
    for rows, kw in ((4, dict(ld=128)), (2, dict(ld=384)), (2, dict(ld=384, n=7)), (2, dict(ld=477, n=7)), (9, dict(ld=0)),
                     (1, dict(ld=1 << 40)), (0, dict()), (0, dict(ld=1 << 40))):
        refused("CUDA tensors are needed", draw, **draw_args(9, logits=padded), rows=rows, **kw)
    refused("draw_device: ", draw, **draw_args(9, logits=padded), rows=2, ld=478, n=7)


def test_sizes_past_32_bits_are_refused(built_lib):
    """They would reach the library cut to 32 bits."""
    import torch
    tall, long, u8 = (1 << 32) + 3, (1 << 32) + 200, torch.uint8
    for call in (lrs.quantize_rows, lrs.quantize_blocks):
        for shape in ((tall, 1), (3, long)):
            refused("larger than 2\\^32", call, torch.zeros(1, 1).expand(shape), torch.zeros(1, 1, dtype=u8).expand(shape), torch.zeros(1, 1))
    a = product_args()
    refused("larger than 2\\^32", lrs.fp8_logits, **{**a, "w": torch.zeros(1, 1, dtype=u8).expand(tall, 200)})
    refused("larger than 2\\^32", lrs.fp8_logits, **{**a, "a": torch.zeros(1, 1, dtype=u8).expand(tall, 200)})
    refused("draw_device: ", lrs.BatchSampler.draw_device, **draw_args(logits=torch.empty(2, long, device="meta")))


class StandInHead:
    """A head of 5 tokens on a device of one's choice."""
    vocab = 5

    def __init__(self, device):
        import torch
        self.device = torch.device(device)

    def logits(self, hidden, out=None, dtype=None):
        import torch
        return torch.zeros(hidden.shape[0], self.vocab, device="meta")


def sampler_without_a_gpu(device=0):
    bs = lrs.BatchSampler.__new__(lrs.BatchSampler)
    bs._h, bs.device, bs.calls = None, device, []
    bs.sample_device = lambda *args, **kw: bs.calls.append((args, kw))
    return bs


def hidden_args(rows=3, **kw):
    """sample_hidden's arguments (meta tensors: only shapes and devices count)."""
    import torch
    t = lambda *shape, dtype=torch.int32: torch.empty(shape, dtype=dtype, device="meta")
    a = dict(hidden=t(rows, 8, dtype=torch.float32), params=t(rows * 24, dtype=torch.uint8), state=t(rows, dtype=torch.int64),
             tokens=t(rows), hist=t(rows, 16), hist_len=t(rows), probs=t(rows, dtype=torch.float32), status=t(rows))
    a.update(kw)
    return a


def test_the_head_and_the_sampler_lie_on_one_device(built_lib):
    import torch
    from lrs.sharded import VocabShardedSampler
    bs = sampler_without_a_gpu(0)
    refused("the head lies on cuda:1, the sampler on cuda:0", bs.sample_hidden, StandInHead("cuda:1"), **hidden_args())
    refused("the head lies on cpu, the sampler on cuda:0", bs.sample_hidden, StandInHead("cpu"), **hidden_args())
    vs = VocabShardedSampler.__new__(VocabShardedSampler)
    vs.shard_n, vs.rows, vs.bs, vs.calls = 5, 3, bs, []
    vs.sample = lambda *args, **kw: vs.calls.append(args)
    a = hidden_args()
    refused("the head lies on cuda:1, the sampler on cuda:0", vs.sample_hidden, StandInHead("cuda:1"), **a)
    assert not bs.calls and not vs.calls
    vs.sample_hidden(StandInHead("cuda:0"), **a)
    assert len(vs.calls) == 1


def test_sample_hidden_has_a_buffer_for_every_row(built_lib):
    import torch
    bs, head = sampler_without_a_gpu(), StandInHead("cuda:0")
    whole = hidden_args()
    for name, t in whole.items():
        if name == "hidden":
            continue
        short = torch.empty((t.shape[0] - 1, *t.shape[1:]), dtype=t.dtype, device="meta")
        refused(f"{name}: fewer than 3 rows", bs.sample_hidden, head, **{**whole, name: short})
    assert not bs.calls
    bs.sample_hidden(head, **whole)
    for name in ("hist", "hist_len", "probs", "status"):
        bs.sample_hidden(head, **{**whole, name: None})
    assert len(bs.calls) == 5 and bs.calls[0][1]["rows"] == 3


def test_sample_hiddens_buffers_lie_on_the_gpu(built_lib):
    """Their addresses go to the kernels as they are."""
    import torch
    from lrs.sharded import VocabShardedSampler
    bs, head = sampler_without_a_gpu(), StandInHead("cuda:0")
    vs = VocabShardedSampler.__new__(VocabShardedSampler)
    vs.shard_n, vs.rows, vs.bs = 5, 3, bs
    vs.sample = lambda *args, **kw: bs.calls.append((args, kw))
    whole = hidden_args()
    for name, t in whole.items():
        host = {**whole, name: torch.zeros(t.shape, dtype=t.dtype)}
        if name != "hidden":  # (LmHead.logits refuses those)
            refused(f"{name}: not on cuda:0", bs.sample_hidden, head, **host)
        if name in ("params", "hist", "hist_len"):  # (the others are copied by torch there)
            refused(f"{name}: not on cuda:0", vs.sample_hidden, head, **host)
    assert not bs.calls


def test_the_crates_product_compares_every_size_of_its_matrices():
    """rust/src/ops.rs is not compiled here: the sizes that its safe types carry and the C call does not are looked
    for in its text (w.cols, out.rows, out.cols went unread)."""
    import os
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rust", "src", "ops.rs")).read()
    body = text[text.index("pub unsafe fn fp8_logits("):]
    guard = body[:body.index("lrs_fp8_logits(")]
    assert "if w.cols != a.cols || out.rows != a.rows || out.cols != w.rows {" in guard and "ffi::LRS_E_INVALID" in guard
