"""What a token's result may depend on besides its own row (run with -m gpu on a B200): of the quantiser and the products nothing,
not a bit; of block_norm the number of rows and where they start (the order of a row's sum goes by both), never their values."""
import pytest
import torch

import okc_muse_kernels_b200 as okc

pytestmark = pytest.mark.gpu


def _gen(seed):
    assert torch.cuda.is_available(), "these tests need a CUDA device"
    return torch.Generator(device="cuda").manual_seed(seed)


@pytest.mark.parametrize("T", [2, 295, 296, 591, 592, 900])
@pytest.mark.parametrize("H", [1000, 1001])
@pytest.mark.parametrize("out", ["f32", "int8"])
def test_a_norms_bits_do_not_depend_on_the_other_rows_values(T, H, out):
    g = _gen(T + H)
    r, y = torch.randn((T, H), generator=g, device="cuda"), torch.randn((T, H), generator=g, device="cuda").bfloat16()
    gate, gain = torch.randn((T, H), generator=g, device="cuda"), torch.ones(H, device="cuda")

    def run():
        r2, x = okc.block_norm(r, y, post_gain=gain, gate=gate, pre_gain=gain, out=out)
        return [t.clone() for t in (r2, *(x if out == "int8" else (x,)))]

    first = run()
    keep = torch.arange(T, device="cuda") % 3 == 1
    for t in (r, y, gate):
        t[~keep] = (t[~keep].float() * 1000 + 7).to(t.dtype)
    r[0, 0] = float("nan")
    for a, b in zip(run(), first):
        assert torch.equal(a[keep], b[keep])


@pytest.mark.parametrize("K", [500, 1504, 1505])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantised_rows_do_not_depend_on_the_batch(K, dtype):
    """The same row alone, among few and among many, and from any address: the same integers, scale and products."""
    g = _gen(K)
    wide = torch.randn((900, K + 3), generator=g, device="cuda").to(dtype)
    w, both = (okc.quantize_rows(torch.randn((n, K), generator=g, device="cuda")) for n in (130, 260))
    x = wide[:, 3:]
    full, y, h = okc.quantize_rows(x), okc.int8_linear(x, w), okc.int8_gated(x, both)
    for T in (1, 2, 40, 295, 296, 591, 592):
        for rows, at in ((x[:T], slice(0, T)), (x[:T].contiguous(), slice(0, T)), (x[900 - T:], slice(900 - T, 900))):
            got = okc.quantize_rows(rows)
            assert torch.equal(got.q, full.q[at]) and torch.equal(got.scale, full.scale[at]), T
            assert torch.equal(okc.int8_linear(rows, w), y[at]) and torch.equal(okc.int8_gated(rows, both), h[at]), T
