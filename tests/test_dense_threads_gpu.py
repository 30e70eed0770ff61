"""Calls of one kernel with different amounts of shared memory, from two host threads on two streams and side by side in one
captured graph (run with -m gpu on a B200).  A thread's call may not depend on what the other one asks for."""
import sys
import threading

import pytest
import torch

import okc_muse_kernels_b200 as okc

pytestmark = pytest.mark.gpu


def _gen(seed):
    assert torch.cuda.is_available(), "these tests need a CUDA device"
    return torch.Generator(device="cuda").manual_seed(seed)


def _product(T, K, N, gated=False):
    """A call on bf16 tokens."""
    g = _gen(T + K + N)
    x = torch.randn((T, K), generator=g, device="cuda").bfloat16()
    w = okc.quantize_rows(torch.randn((2 * N if gated else N, K), generator=g, device="cuda") * 0.02)
    return lambda: (okc.int8_gated if gated else okc.int8_linear)(x, w)


def _norm(T, H, out, lo=0):
    """A call on rows that start `lo` elements into their buffer."""
    g = _gen(T + H)
    r, y = (torch.randn((T, H + lo), generator=g, device="cuda").bfloat16()[:, lo:] for _ in range(2))
    gain = torch.ones(H, device="cuda")
    def run():
        r2, x = okc.block_norm(r, y, post_gain=gain, pre_gain=gain, out=out)
        return (r2, *x) if out == "int8" else (r2, x)
    return run


def _tensors(result):
    return result if isinstance(result, tuple) else (result,)


PAIRS = {
    "one": lambda: (_product(1, 4096, 7168), _product(1, 4096, 1024)),
    "one-gated": lambda: (_product(1, 7168, 2048, True), _product(1, 300, 200, True)),
    "mid": lambda: (_product(40, 7168, 2048), _product(40, 1408, 2048)),
    "mid-gated": lambda: (_product(100, 7168, 2048, True), _product(16, 4096, 2048, True)),
    "norm": lambda: (_norm(700, 8192, "bf16"), _norm(700, 4096, "bf16")),
    "norm-int8": lambda: (_norm(700, 8192, "int8"), _norm(700, 4096, "int8")),
    "norm-odd": lambda: (_norm(700, 8001, "bf16", 1), _norm(700, 4001, "bf16", 1)),
}


@pytest.mark.parametrize("name", PAIRS)
def test_two_threads_on_two_streams(name):
    calls = PAIRS[name]()
    want = [_tensors(call()) for call in calls]
    torch.cuda.synchronize()
    failed = []

    def work(call, ref):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(40):
                    got = [_tensors(call()) for _ in range(50)]
                    torch.cuda.current_stream().synchronize()
                    for one in got:
                        assert all(torch.equal(a, b) for a, b in zip(one, ref))
        except BaseException as e:      # (an assertion in a thread would be lost)
            failed.append(e)

    switch = sys.getswitchinterval()
    sys.setswitchinterval(1e-5)
    try:
        threads = [threading.Thread(target=work, args=pair) for pair in zip(calls, want)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    finally:
        sys.setswitchinterval(switch)
    assert not failed, failed
    assert okc.dense_status() == (0, 0)


@pytest.mark.parametrize("name", PAIRS)
def test_one_graph_of_two_sizes(name):
    """The larger call first, the smaller behind it, as often as they come."""
    calls = PAIRS[name]()
    want = [_tensors(call()) for call in calls]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [_tensors(calls[k % 2]()) for k in range(6)]
    for _ in range(3):
        for one in got:
            for t in one:
                t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for k, one in enumerate(got):
            assert all(torch.equal(a, b) for a, b in zip(one, want[k % 2])), k
