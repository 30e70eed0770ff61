"""Values that are not finite, rows of zeros, the ends of the int8 range and far gates, for the kernels of one token and of rows
off the 16-byte grid, against the definitions (run with -m gpu on a B200).

U = 2^-24 is half a step of f32.  What is compared exactly is exact: integer sums, powers of two, NaN and zeros."""
import pytest
import torch

import okc_muse_kernels_b200 as okc

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
INF, NAN = float("inf"), float("nan")


def _gen(seed):
    assert torch.cuda.is_available(), "these tests need a CUDA device"
    return torch.Generator(device="cuda").manual_seed(seed)


def _weight(rows, cols, g):
    q = torch.randint(-127, 128, (rows, cols), generator=g, device="cuda", dtype=torch.int8)
    return okc.int8_rows(q, torch.rand(rows, generator=g, device="cuda") * 1e-2 + 1e-4)


@pytest.mark.parametrize("K", [1, 15, 200, 4096, 9001, 16384])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_one_token_that_is_not_finite_or_zero(K, dtype):
    g = _gen(K)
    w, both, bias = _weight(150, K, g), _weight(2 * 150, K, g), torch.randn(150, generator=g, device="cuda")
    for value, at in ((INF, 0), (-INF, K - 1), (NAN, K // 2), (NAN, K - 1)):
        x = torch.randn((1, K), generator=g, device="cuda").to(dtype)
        x[0, at] = value
        for out_f32 in (False, True):
            assert okc.int8_linear(x, w, bias=bias, out_f32=out_f32).isnan().all() and okc.int8_gated(x, both, out_f32=out_f32).isnan().all()
    for x in (torch.zeros((1, K), device="cuda", dtype=dtype), torch.full((1, K), -0.0, device="cuda", dtype=dtype),
              torch.full((1, K), 2.0 ** -121, device="cuda", dtype=dtype)):
        assert torch.equal(okc.int8_linear(x, w, bias=bias, out_f32=True)[0], bias) and not okc.int8_gated(x, both, out_f32=True).any()
    assert okc.dense_status() == (0, 0)


@pytest.mark.parametrize("T", [1, 2, 40, 600])
def test_int8_tokens_with_scales_that_are_not_finite(T):
    g = _gen(T)
    w, both = _weight(70, 130, g), _weight(140, 130, g)
    q = torch.randint(-128, 128, (T, 130), generator=g, device="cuda", dtype=torch.int8)
    for value in (NAN, 0.0):
        scale = torch.full((T,), 0.25, device="cuda")
        scale[T // 2] = value
        x = okc.int8_rows(q, scale)
        y, h = okc.int8_linear(x, w, out_f32=True), okc.int8_gated(x, both, out_f32=True)
        here = torch.arange(T, device="cuda") == T // 2
        for out in (y, h):
            assert out[here].isnan().all() if value != 0.0 else not out[here].any()
            assert torch.isfinite(out[~here]).all()


@pytest.mark.parametrize("K", [1, 130, 5000, 16384])
def test_one_token_of_the_lowest_value(K):
    """-128 (made elsewhere; the quantiser stops at -127) against -128 and 127: sums of up to 2^28, exact in f32 as a power of two
    times K, or of 127 * 128 * K below 2^24."""
    low = okc.int8_rows(torch.full((1, K), -128, dtype=torch.int8, device="cuda"), torch.ones(1, device="cuda"))
    rows = torch.cat([torch.full((3, K), -128, dtype=torch.int8, device="cuda"), torch.full((3, K), 127, dtype=torch.int8, device="cuda")])
    y = okc.int8_linear(low, okc.int8_rows(rows, torch.ones(6, device="cuda")), out_f32=True)
    want = torch.tensor([16384.0 * K] * 3 + [float(-127 * 128 * K)] * 3, device="cuda")      # the second: a conversion rounds once, as here
    assert torch.equal(y[0], want)


def test_one_token_with_far_gates():
    """Gate values of thousands: silu is g or 0, never NaN.  g = u = 64 * 127 * s with s the token's f32 scale times 127."""
    w = okc.int8_rows(torch.full((64, 64), 127, dtype=torch.int8, device="cuda"), torch.ones(64, device="cuda"))
    for sign in (1.0, -1.0):
        for dtype in (torch.bfloat16, torch.float32):
            h = okc.int8_gated(torch.full((1, 64), sign, device="cuda", dtype=dtype), w, out_f32=True)
            if sign < 0:
                assert not h.any()
            else:
                # g is 64 * 127 (1 / 127 rounded, then 127 * 127 * 64 times it): off by 3 U; e^-g is 0; the division by 1 is
                # off by 4 U at most, the product by U and both factors
                g = 64 * 127.0
                assert ((h.double() - g * g).abs() <= 12 * U * g * g).all()


@pytest.mark.parametrize("res,blk", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("T", [5, 300, 640])
@pytest.mark.parametrize("H", [501, 2051, 5121, 12289])
def test_norm_rows_off_the_grid_that_are_not_finite(res, blk, T, H):
    """A NaN or an infinity stays in its own row, and makes it NaN (int8: zeros with scale NaN)."""
    g = _gen(T + H)
    r, y = torch.randn((T, H), generator=g, device="cuda").to(res), torch.randn((T, H), generator=g, device="cuda").to(blk)
    gain = torch.ones(H, device="cuda")
    clean = okc.block_norm(r, y, post_gain=gain, pre_gain=gain, out="f32")
    clean_q = okc.block_norm(r, y, post_gain=gain, pre_gain=gain, out="int8")[1]
    r, y = r.clone(), y.clone()
    r[0, 0], r[1, H - 1], y[2, H - 1], y[3, 0] = NAN, INF, INF, NAN
    bad = torch.arange(T, device="cuda") < 4
    r2, x = okc.block_norm(r, y, post_gain=gain, pre_gain=gain, out="f32")
    assert torch.equal(r2[4:], clean[0][4:]) and torch.equal(x[4:], clean[1][4:])
    assert r2[0].isnan().sum() == 1 and torch.isinf(r2[1]).sum() == 1 and not r2[1].isnan().any()
    # y[2]: inf * rsqrt(inf) = NaN in its column, 0 beside it; y[3]: the norm is NaN
    assert r2[2].isnan().sum() == 1 and torch.equal(r2[2, :-1], r[2, :-1]) and r2[3].isnan().all()
    assert x[0].isnan().all() and x[2].isnan().all() and x[3].isnan().all()
    assert x[1, -1].isnan() and not x[1, :-1].any()                 # inf * rsqrt(inf), and 0 * r' beside it
    _, q = okc.block_norm(r, y, post_gain=gain, pre_gain=gain, out="int8")
    assert torch.equal(q.scale.isnan(), bad) and not q.q[:4].any()
    assert torch.equal(q.q[4:], clean_q.q[4:]) and torch.equal(q.scale[4:], clean_q.scale[4:])
    # without the norm after the block, and without a block
    r2, x = okc.block_norm(r, y, pre_gain=gain, out="bf16")
    assert torch.isinf(r2[2, -1]) and r2[3, 0].isnan() and torch.isfinite(r2[2:4, 1:-1]).all() and torch.isfinite(x[4:]).all()
    _, x = okc.block_norm(r, pre_gain=gain, out="int8")
    assert x.scale.isnan().tolist() == [i < 2 for i in range(T)] and not x.q[:2].any()
    # an infinite gate per channel makes that column's values infinite in every row, and x NaN there
    gate = torch.ones(H, device="cuda")
    gate[H - 1] = INF
    r2, x = okc.block_norm(r[4:], y[4:], gate=gate, pre_gain=gain, out="f32")
    assert torch.isinf(r2[:, -1]).all() and torch.isfinite(r2[:, :-1]).all() and x[:, -1].isnan().all() and not x[:, :-1].any()
    assert okc.dense_status() == (0, 0)


@pytest.mark.parametrize("T", [3, 640])
@pytest.mark.parametrize("H", [520, 521])
def test_norm_rows_of_zeros_and_extremes(T, H):
    r, y = torch.zeros((T, H), device="cuda"), torch.zeros((T, H), device="cuda")
    gain = torch.ones(H, device="cuda")
    r2, x = okc.block_norm(r, y, post_gain=gain, pre_gain=gain, out="int8")
    assert not r2.any() and not x.q.any() and not x.scale.any()
    # the same number in every column: x is 1 / sqrt(1 + eps / r'^2); eps = 0 and a power of two give 1 up to the roundings of
    # a mean (H adds of equal squares, at most H / 2 + 10 U), a root and two products
    r += 2.0 ** 40
    _, x = okc.block_norm(r, pre_gain=gain, eps=0.0, out="f32")
    assert ((x.double() - 1).abs() <= (H / 2 + 20) * U).all()
    _, x = okc.block_norm(r, pre_gain=gain, eps=0.0, out="int8")
    assert (x.q == 127).all()
