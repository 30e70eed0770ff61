"""moe_block_step and int8_ffn captured in CUDA graphs, in place, and two of them at once (run with -m gpu on a B200)."""
import pytest
import torch

import okc_muse_kernels_b200 as okc
from okc_muse_kernels_b200 import synth

pytestmark = pytest.mark.gpu

H, E = 512, 16


@pytest.fixture(scope="module")
def layer():
    assert torch.cuda.is_available(), "these tests need a CUDA device"
    g = torch.Generator(device="cuda").manual_seed(2)
    weights = synth.make_weights(synth.Workload("small", 5, H, 256, E, 2), seed=11, device=torch.device("cuda"))
    states = [okc.prepare(weights, okc.MoEPlan(hidden=H, inter=256, n_experts=E, top_k=2, max_tokens=64)) for _ in range(2)]
    router, gain, post = (torch.randn(s, generator=g, device="cuda") for s in ((E, H), (H,), (H,)))
    w13, w2 = (okc.quantize_rows(0.05 * torch.randn(s, generator=g, device="cuda")) for s in ((2 * 320, H), (H, 320)))

    def step(r, state, split=None):
        """Two layers on the stream r, in place: an expert block, and a dense feed-forward on its int8 rows."""
        _, x = okc.moe_block_step(r, router if split is None else split, state, pre_gain=gain, post_gain=post, next_gain=gain, residual_scale=0.9, out="int8", residual_out=r)
        y = okc.int8_ffn(x, w13, w2)
        return okc.block_norm(r, y, post_gain=post, gate=gain, pre_gain=gain, residual_out=r)[1]

    return states, step, okc.split_router(router)


@pytest.mark.parametrize("T", [1, 7, 64])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_in_place_and_two_graphs_at_once(layer, T, dtype):
    states, step, split = layer
    def rows(seed):
        return torch.randn((T, H), generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)
    streams = [torch.cuda.Stream() for _ in range(2)]
    held, outs, graphs = [rows(0), rows(1)], [], []
    for r, state in zip(held, states):
        step(r, state, split)
    torch.cuda.synchronize()
    for r, state in zip(held, states):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(r, state, split))
        graphs.append(graph)
    for k in range(5):
        fresh = [rows(10 * k + i) for i in range(2)]
        want = []
        for f, state in zip(fresh, states):
            r = f.clone()
            x = step(r, state, split).clone()
            x2 = step(r, state, split).clone()
            want.append((r, x2, x))
        for r, f in zip(held, fresh):
            r.copy_(f)
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
                graph.replay()
        torch.cuda.synchronize()
        for r, x, (wr, wx, first) in zip(held, outs, want):
            assert torch.equal(r, wr) and torch.equal(x, wx) and not torch.equal(x, first)
        assert all(okc.read_status(s)[0] == 0 for s in states)
    assert okc.dense_status() == (0, 0)


@pytest.mark.parametrize("T", [1, 5, 64, 700])
def test_feed_forward_over_its_own_input(layer, T):
    """The second product writes where the tokens of the first one lay: only the activations between them are its input."""
    g = torch.Generator(device="cuda").manual_seed(T)
    w13, w2 = (okc.quantize_rows(0.05 * torch.randn(s, generator=g, device="cuda")) for s in ((2 * 320, H), (H, 320)))
    x = torch.randn((T, H), generator=g, device="cuda").bfloat16()
    want = okc.int8_ffn(x, w13, w2)
    for _ in range(3):
        y = x.clone()
        assert okc.int8_ffn(y, w13, w2, out=y) is y and torch.equal(y, want)
