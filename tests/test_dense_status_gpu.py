"""What the dense operators report of device waits that ran out (run with -m gpu on a B200).  The waits are probes with a short
limit on a barrier that nothing completes: their kernels return normally."""
import threading
import time

import pytest
import torch

import okc_muse_kernels_b200 as okc
from okc_muse_kernels_b200 import _lib

pytestmark = pytest.mark.gpu

CODES = (0x7D, 0x7C)       # a norm's, a product's


def _probe(product, stream):
    assert _lib.lib().okc_moe_probe_dense_timeout(product, stream.cuda_stream) == _lib.OKC_OK


@pytest.mark.parametrize("product", [0, 1])
def test_a_wait_that_ran_out_is_reported_once_and_the_operators_go_on(product):
    assert torch.cuda.is_available(), "these tests need a CUDA device"
    assert okc.dense_status() == (0, 0)
    _probe(product, torch.cuda.current_stream())
    assert okc.dense_status() == (_lib.OKC_ERR_TIMEOUT, CODES[product])
    assert okc.dense_status() == (0, 0)
    x = torch.randn((9, 256), device="cuda")
    w = okc.quantize_rows(torch.randn((64, 256), device="cuda"))
    r, n = okc.block_norm(x, x, pre_gain=torch.ones(256, device="cuda"))
    assert torch.isfinite(r).all() and torch.isfinite(n).all() and torch.isfinite(okc.int8_linear(x, w)).all()
    assert okc.dense_status() == (0, 0)
    assert _lib.lib().okc_moe_probe_dense_timeout(2, None) == _lib.OKC_ERR_BAD_ARG


def test_a_norm_and_a_product_are_both_reported():
    for product in (0, 1):
        _probe(product, torch.cuda.current_stream())
    got = [okc.dense_status() for _ in range(3)]
    assert sorted(got[:2]) == [(_lib.OKC_ERR_TIMEOUT, c) for c in sorted(CODES)] and got[2] == (0, 0)


@pytest.mark.parametrize("product", [0, 1])
def test_nothing_is_lost_to_a_reader_on_another_stream(product):
    """A thread reads the status all the time; each of the waits that run out beside it has to show up there."""
    assert okc.dense_status() == (0, 0)
    seen, stop = [], threading.Event()

    def read():
        with torch.cuda.stream(torch.cuda.Stream()):
            while not stop.is_set():
                rc, code = okc.dense_status()
                if rc:
                    seen.append((rc, code))

    reader = threading.Thread(target=read)
    reader.start()
    stream = torch.cuda.Stream()
    lost = 0
    try:
        for k in range(300):
            before = len(seen)
            _probe(product, stream)
            stream.synchronize()
            end = time.monotonic() + 2.0
            while len(seen) == before and time.monotonic() < end:
                time.sleep(0)
            if len(seen) == before:
                lost += 1
                if lost == 3:
                    break
    finally:
        stop.set()
        reader.join()
    assert lost == 0 and set(seen) == {(_lib.OKC_ERR_TIMEOUT, CODES[product])}
    assert okc.dense_status() == (0, 0)
