"""CPU-side checks of the dense operators: what the entry points refuse, in Python before anything reaches the library and
in the C ABI before anything is launched.  No GPU is touched."""
import ctypes as C

import pytest
import torch

import okc_muse_kernels_b200 as okc
from okc_muse_kernels_b200 import _lib, dense

OK, BAD, LARGE, NO_DEVICE = _lib.OKC_OK, _lib.OKC_ERR_BAD_ARG, _lib.OKC_ERR_TOO_LARGE, _lib.OKC_ERR_NO_DEVICE


def _weight(rows=8, cols=64):
    return torch.zeros((rows, cols), dtype=torch.int8), torch.ones(rows)


def test_cpu_tensors_are_refused():
    x = torch.zeros((2, 64), dtype=torch.bfloat16)
    for call in (lambda: okc.quantize_rows(x), lambda: okc.int8_linear(x, _weight()), lambda: okc.int8_gated(x, _weight()),
                 lambda: okc.block_norm(x, x), lambda: okc.block_norm(x, pre_gain=torch.ones(64)), lambda: okc.int8_rows(*_weight())):
        with pytest.raises(ValueError, match="CUDA"):
            call()


@pytest.mark.parametrize("weight,word", [
    ((torch.zeros((8, 64)), torch.ones(8)), "int8"),
    ((torch.zeros((8, 64), dtype=torch.int8), torch.ones(7)), "int8"),
    ((torch.zeros((8, 64), dtype=torch.int8), torch.ones(8, dtype=torch.float64)), "int8"),
    ((torch.zeros((8, 60), dtype=torch.int8), torch.ones(8)), "int8_rows"),              # rows 60 bytes apart
    ((torch.zeros((8, 128), dtype=torch.int8)[:, ::2], torch.ones(8)), "int8_rows"),     # columns two bytes apart
    ((torch.zeros((8, 80), dtype=torch.int8)[:, 1:65], torch.ones(8)), "int8_rows"),     # starts off a 16-byte boundary
    ((torch.zeros((1, 64), dtype=torch.int8).expand(8, 64), torch.ones(8)), "int8_rows"),
    ((torch.zeros((0, 64), dtype=torch.int8), torch.ones(0)), "weight"),
])
def test_weights_that_the_products_refuse(weight, word):
    for fn in (okc.int8_linear, okc.int8_gated):
        with pytest.raises(ValueError, match=word):
            fn(torch.zeros((2, 64), dtype=torch.bfloat16), weight)


def test_product_arguments_that_are_refused():
    x = torch.zeros((2, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="columns"):
        okc.int8_linear(x[:, :63], _weight())
    with pytest.raises(ValueError, match="bf16 or f32"):
        okc.int8_linear(x.half(), _weight())
    with pytest.raises(ValueError, match="bf16 or f32"):
        okc.int8_linear(x[0], _weight())
    with pytest.raises(ValueError, match="as many up rows"):
        okc.int8_gated(x, _weight(rows=7))
    with pytest.raises(ValueError, match="131071"):
        okc.int8_linear(torch.zeros((1, 131072), dtype=torch.bfloat16), _weight(1, 131072))
    with pytest.raises(ValueError, match="131071"):
        okc.quantize_rows(torch.zeros((1, 131072)))
    with pytest.raises(ValueError, match="131071"):
        okc.quantize_rows(torch.zeros((1, 0)))
    with pytest.raises(ValueError, match="bf16 or f32"):
        okc.quantize_rows(torch.zeros((2, 64), dtype=torch.float64))


def test_block_norm_arguments_that_are_refused():
    x, g = torch.zeros((2, 64)), torch.ones(64)
    for kw, word in ((dict(out="fp8"), "out is"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps")):
        with pytest.raises(ValueError, match=word):
            okc.block_norm(x, x, pre_gain=g, **kw)
    with pytest.raises(ValueError, match="bf16 or f32"):
        okc.block_norm(x.half(), x)
    with pytest.raises(ValueError, match="16384"):
        okc.block_norm(torch.zeros((1, 16385)), pre_gain=torch.ones(16385))


def test_overlap_of_memory():
    b = torch.zeros(1000)
    a = b[:640].view(10, 64)
    assert dense._overlap(a, b[639:]) and not dense._overlap(a, b[640:])
    assert dense._overlap(a, a) and not dense._overlap(a[:0], a)
    view = b[:630].view(10, 63)[:, 10:20]        # its last element is 9 * 63 + 19
    assert dense._overlap(view, b[586:]) and not dense._overlap(view, b[587:])


def _norm_args(**kw):
    a = dict(residual=0x1000, block=0x2000, residual_out=0x3000, out=0x4000, pre_gain=0x5000, post_gain=0x6000, rows=4, hidden=64,
             residual_stride=64, block_stride=64, residual_out_stride=64, out_stride=64, residual_scale=1.0, block_scale=1.0, eps=1e-5)
    a.update(kw)
    return _lib.BlockNormArgs(**a)


@pytest.mark.parametrize("kw,rc", [
    (dict(rows=0), OK), (dict(rows=-1), BAD), (dict(hidden=0), BAD), (dict(hidden=16385, residual_stride=20000), LARGE),
    (dict(residual=None), BAD), (dict(residual_stride=63), BAD), (dict(block_stride=63), BAD), (dict(residual_out=None), BAD),
    (dict(residual_out_stride=10), BAD), (dict(out=None), BAD), (dict(out_stride=1), BAD), (dict(out_kind=3), BAD),
    (dict(out_kind=2), BAD), (dict(eps=-1e-3), BAD), (dict(gate=0x7000), BAD), (dict(gate_kind=1), BAD),
    (dict(gate=0x7000, gate_kind=3, gate_stride=63), BAD), (dict(block=None), BAD), (dict(block=None, post_gain=None, pre_gain=None), BAD),
    (dict(residual=0x1001), BAD), (dict(residual=0x1002, residual_f32=1), BAD), (dict(block=0x2001), BAD), (dict(out=0x4002, out_kind=1), BAD),
    (dict(pre_gain=0x5002), BAD), (dict(gate=0x7001, gate_kind=1), BAD),
])
def test_block_norm_abi_checks(kw, rc):
    assert _lib.lib().okc_moe_block_norm(C.byref(_norm_args(**kw)), None) == rc


def _int8_args(**kw):
    a = dict(x=0x1000, w=0x2000, w_scale=0x3000, out=0x4000, scratch=0x5000, x_stride=64, w_stride=64, out_stride=32, tokens=16, k=64, n=32)
    a.update(kw)
    return _lib.Int8Args(**a)


@pytest.mark.parametrize("kw,rc", [
    (dict(tokens=0), OK), (dict(tokens=-1), BAD), (dict(k=0), BAD), (dict(n=0), BAD), (dict(k=131072, x_stride=131072, w_stride=131072), LARGE),
    (dict(tokens=(1 << 30) + 1), LARGE), (dict(n=(1 << 30) + 1, out_stride=1 << 31), LARGE),
    (dict(x=None), BAD), (dict(w=None), BAD), (dict(w_scale=None), BAD), (dict(out=None), BAD), (dict(scratch=None), BAD),
    (dict(w=0x2008), BAD), (dict(w_stride=72), BAD), (dict(w_stride=48), BAD), (dict(x_stride=63), BAD), (dict(out_stride=31), BAD),
    (dict(x=0x1001), BAD), (dict(x=0x1002, x_kind=1), BAD), (dict(out=0x4001), BAD), (dict(out=0x4002, out_f32=1), BAD), (dict(w_scale=0x3002), BAD),
    (dict(bias=0x7002), BAD), (dict(x_kind=3), BAD), (dict(x_kind=2), BAD), (dict(x_kind=2, x_scale=0x6000, x=0x1004), BAD), (dict(x_kind=2, x_scale=0x6000, x_stride=72), BAD),
])
def test_int8_product_abi_checks(kw, rc):
    lib = _lib.lib()
    assert lib.okc_moe_int8_linear(C.byref(_int8_args(**kw)), None) == rc
    assert lib.okc_moe_int8_gated(C.byref(_int8_args(**kw)), None) == rc
    assert lib.okc_moe_int8_gated(C.byref(_int8_args(bias=0x7000)), None) == BAD


def test_quantize_rows_abi_checks_and_scratch():
    lib = _lib.lib()
    q = lambda rows=4, cols=64, xs=64, qs=64, x=0x1000: lib.okc_moe_quantize_rows(x, 0, xs, rows, cols, 0x2000, qs, 0x3000, None)  # noqa: E731
    assert q(rows=0) == OK and q(rows=-1) == BAD and q(cols=0) == BAD and q(cols=131072) == LARGE
    assert q(xs=63) == BAD and q(qs=63) == BAD and q(x=None) == BAD
    assert lib.okc_moe_block_norm(None, None) == BAD and lib.okc_moe_int8_linear(None, None) == BAD
    assert lib.okc_moe_int8_scratch_bytes(0, 1, 4096) == 0 and lib.okc_moe_int8_scratch_bytes(2, 4096, 4096) == 0
    assert lib.okc_moe_int8_scratch_bytes(0, 1, dense.INT8_ONE_MAX_K) == 0 and lib.okc_moe_int8_scratch_bytes(0, 1, dense.INT8_ONE_MAX_K + 1) == 16400 + 4
    assert lib.okc_moe_int8_scratch_bytes(1, 2, 1000) == 2 * (1008 + 4)


@pytest.mark.skipif(torch.cuda.is_available(), reason="a GPU is there")
def test_calls_without_a_device_are_errors_not_crashes():
    lib = _lib.lib()
    assert lib.okc_moe_block_norm(C.byref(_norm_args()), None) == NO_DEVICE
    assert lib.okc_moe_int8_linear(C.byref(_int8_args()), None) == NO_DEVICE
    assert lib.okc_moe_quantize_rows(0x1000, 0, 64, 4, 64, 0x2000, 64, 0x3000, None) == NO_DEVICE


def test_packed_arguments_are_the_structs():
    """The byte strings the Python side passes are the ctypes (and so the C) structs, field for field."""
    for cls, pack in ((_lib.BlockNormArgs, _lib.pack_block_norm), (_lib.Int8Args, _lib.pack_int8)):
        n = len(cls._fields_)
        values = [float(i + 1) if t is C.c_float else i + 1 for i, (_, t) in enumerate(cls._fields_)]
        assert bytes(cls(*values)) == pack(*values) and len(pack(*values)) == C.sizeof(cls), n
