"""moe_block_step: its arguments are checked before the first of its launches, and all of them go to the state's device."""
import contextlib

import pytest
import torch

import okc_muse_kernels_b200 as okc
from okc_muse_kernels_b200 import moe, synth


def test_tensors_and_state_have_to_be_on_one_device():
    state = {"plan": okc.MoEPlan(hidden=256, inter=256, n_experts=16, top_k=2, max_tokens=8), "workspace": torch.empty(0, device="meta")}
    r, w = torch.zeros((2, 256), device="meta"), torch.zeros((16, 256), device="meta")
    for args, kw in (((torch.zeros((2, 256)), w), {}), ((r, torch.zeros((16, 256))), {}), ((r, w), {"bias": torch.zeros(16)})):
        with pytest.raises(ValueError, match="state on"):
            okc.moe_block_step(*args, state, pre_gain=torch.ones(256, device="meta"), **kw)


def test_every_launch_goes_to_the_states_device(monkeypatch):
    entered, launched = [], []

    @contextlib.contextmanager
    def device(d):
        entered.append(d)
        yield
        entered.pop()

    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(moe, "check_norm", lambda r, *a: (r, r.bfloat16(), 0, None, ()))
    monkeypatch.setattr(moe, "_check_hidden", lambda h, plan: (h, 0))
    monkeypatch.setattr(moe, "_check_router", lambda *a: False)
    monkeypatch.setattr(moe, "launch_norm", lambda n: launched.append(("norm", list(entered))) or n[:2])
    monkeypatch.setattr(moe, "moe_layer_step", lambda *a, **k: launched.append(("layer", list(entered))))
    where = torch.device("meta")
    r = torch.zeros((2, 256), device=where)
    okc.moe_block_step(r, torch.zeros((16, 256), device=where), {"plan": None, "workspace": torch.empty(0, device=where)}, pre_gain=None)
    assert launched == [("norm", [where]), ("layer", [where]), ("norm", [where])]


@pytest.mark.gpu
def test_wrong_arguments_are_refused_before_anything_is_launched(monkeypatch):
    assert torch.cuda.is_available(), "these tests need a CUDA device"
    plan = okc.MoEPlan(hidden=512, inter=256, n_experts=16, top_k=2, max_tokens=16)
    weights = synth.make_weights(synth.Workload("small", 5, 512, 256, 16, 2), seed=11, device=torch.device("cuda"))
    state = okc.prepare(weights, plan)
    r, w, gain = torch.randn((4, 512), device="cuda"), torch.randn((16, 512), device="cuda"), torch.ones(512, device="cuda")
    bad = [dict(post_gain=gain[:511]), dict(gate=gain[:5]), dict(gate=gain.double()), dict(next_gain=gain.bfloat16()), dict(out="fp8"), dict(eps=-1.0),
           dict(residual_out=r.bfloat16()), dict(residual_out=r[:3]), dict(pre_gain=gain[:4]), dict(pre_gain=None), dict(mode="other"), dict(bias=gain),
           dict(router_w=w[:15]), dict(router_w=w.half()), dict(residual=r[:, :256].contiguous()), dict(residual=torch.randn((17, 512), device="cuda")), dict(residual=r[:0])]
    launched = []
    with monkeypatch.context() as m:
        m.setattr(moe, "launch_norm", lambda n: launched.append(n) or n[:2])
        m.setattr(moe, "moe_layer_step", lambda *a, **k: launched.append(a))
        for kw in bad:
            kw = dict(dict(residual=r, router_w=w, pre_gain=gain), **kw)
            with pytest.raises(ValueError):
                okc.moe_block_step(kw.pop("residual"), kw.pop("router_w"), state, **kw)
        assert not launched
    r2, x = okc.moe_block_step(r, w, state, pre_gain=gain, post_gain=gain, next_gain=gain)
    assert torch.isfinite(r2).all() and torch.isfinite(x).all()
