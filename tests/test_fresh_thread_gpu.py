"""Calls that are the first of their host thread: nothing has been launched from it, so it has no current CUDA context yet
(run with -m gpu on a B200)."""
import threading

import pytest
import torch

import okc_muse_kernels_b200 as okc
from okc_muse_kernels_b200 import synth

pytestmark = pytest.mark.gpu


def _gen(seed):
    assert torch.cuda.is_available(), "these tests need a CUDA device"
    return torch.Generator(device="cuda").manual_seed(seed)


def _in_a_fresh_thread(call):
    """The call's result, made by a thread that has done nothing else."""
    box = []

    def go():
        try:
            box.append(call())
        except BaseException as e:
            box.append(e)

    t = threading.Thread(target=go)
    t.start()
    t.join()
    if isinstance(box[0], BaseException):
        raise box[0]
    torch.cuda.synchronize()
    return box[0]


@pytest.mark.parametrize("T", [1, 5, 40, 900])
@pytest.mark.parametrize("rows", ["int8", "bf16"])
def test_products(T, rows):
    g = _gen(T)
    x = torch.randn((T, 512), generator=g, device="cuda").bfloat16()
    if rows == "int8":
        x = okc.quantize_rows(x)
    w = okc.quantize_rows(torch.randn((256, 512), generator=g, device="cuda"))
    for fn in (okc.int8_linear, okc.int8_gated):
        want = fn(x, w)
        torch.cuda.synchronize()
        assert torch.equal(_in_a_fresh_thread(lambda: fn(x, w)), want)


@pytest.mark.parametrize("T", [3, 700])
def test_norm_and_quantiser(T):
    g = _gen(T)
    r = torch.randn((T, 512), generator=g, device="cuda")
    gain = torch.ones(512, device="cuda")
    want = okc.block_norm(r, r, pre_gain=gain)
    torch.cuda.synchronize()
    got = _in_a_fresh_thread(lambda: okc.block_norm(r, r, pre_gain=gain))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    want = okc.quantize_rows(r)
    torch.cuda.synchronize()
    got = _in_a_fresh_thread(lambda: okc.quantize_rows(r))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert _in_a_fresh_thread(okc.dense_status) == (0, 0)


def test_router_and_experts():
    g = _gen(7)
    weights = synth.make_weights(synth.Workload("small", 5, 512, 256, 16, 2), seed=11, device=torch.device("cuda"))
    state = okc.prepare(weights, okc.MoEPlan(hidden=512, inter=256, n_experts=16, top_k=2, max_tokens=64))
    hidden = torch.randn((40, 512), generator=g, device="cuda").bfloat16()
    router = torch.randn((16, 512), generator=g, device="cuda")
    logits = torch.randn((40, 16), generator=g, device="cuda")
    for call in (lambda: okc.moe_layer_step(hidden, okc.split_router(router), state), lambda: okc.moe_layer_step(hidden, router, state),
                 lambda: okc.moe_step(hidden, logits, state), lambda: okc.moe_block_step(hidden, router, state, pre_gain=router[0])[0]):
        want = call()
        torch.cuda.synchronize()
        assert torch.equal(_in_a_fresh_thread(call), want)
    split = okc.split_router(router)
    want = okc.moe_layer_step(hidden, split, state)
    torch.cuda.synchronize()
    assert torch.equal(_in_a_fresh_thread(lambda: okc.moe_layer_step(hidden, split, state)), want)
