"""The router and sort kernels from two host threads on two streams, each with its own state, with different numbers of
tokens and so different amounts of shared memory (run with -m gpu on a B200)."""
import ctypes as C
import sys
import threading

import pytest
import torch

import okc_muse_kernels_b200 as okc
from okc_muse_kernels_b200 import _lib, synth

pytestmark = pytest.mark.gpu

E, K, H = 256, 8, 256


@pytest.fixture(scope="module")
def states():
    assert torch.cuda.is_available(), "these tests need a CUDA device"
    dev = torch.device("cuda")
    weights = synth.make_weights(synth.Workload("router", 4, H, 256, E, K), seed=3, device=dev)
    return [okc.prepare(weights, okc.MoEPlan(hidden=H, inter=256, n_experts=E, top_k=K, max_tokens=512)) for _ in range(2)]


def _calls(kind, state, T):
    g = torch.Generator(device="cuda").manual_seed(T)
    logits = torch.randn((T, E), generator=g, device="cuda")
    hidden = torch.randn((T, H), generator=g, device="cuda").bfloat16()
    w = torch.randn((E, H), generator=g, device="cuda")
    if kind == "logits":      # straight at the C entry: next to nothing of the thread's time is outside it
        plan, lib = C.byref(state["plan"].c_plan()), _lib.lib()
        at = [state[k].data_ptr() for k in ("ids", "wts", "workspace")]

        def call():
            assert lib.okc_moe_route(plan, logits.data_ptr(), T, 0, 0, *at, torch.cuda.current_stream().cuda_stream) == _lib.OKC_OK
            return state["ids"][:T], state["wts"][:T]

        return call
    if kind == "given":
        ids = logits.topk(K, dim=1).indices.int()
        data = {"hidden_states": hidden, "topk_ids": ids, "topk_weights": torch.full((T, K), 0.125, device="cuda")}
        return lambda: (okc.kernel_fn(data, state),)
    split = okc.split_router(w)
    return lambda: okc.route_hidden(hidden, split if kind == "split" else w, state)


@pytest.mark.parametrize("kind,tokens", [("logits", (32, 1)), ("logits", (512, 40)), ("given", (512, 1)), ("hidden", (256, 2)), ("split", (256, 2))])
def test_two_threads_route_different_batches(states, kind, tokens):
    calls = [_calls(kind, s, T) for s, T in zip(states, tokens)]
    want = [[t.clone() for t in call()] for call in calls]
    torch.cuda.synchronize()
    failed = []

    def work(call, ref):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(40):
                    for _ in range(100):
                        got = call()
                    torch.cuda.current_stream().synchronize()
                    assert all(torch.equal(a, b) for a, b in zip(got, ref))
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
    assert all(okc.read_status(s)[0] == 0 for s in states)
